// k_attn.hip -- the key-value cache's write and attention over it.
#include "attn_internal.hpp"
#include "moe_device.hpp"

namespace moe {

namespace {

typedef __bf16 bf16_t;
typedef _Float16 f16_t;

// The sequence that a packed row belongs to, or -1: the last b with row_start[b] <= row, checked
// against its end (so a row_start that does not ascend finds no wrong memory).
__device__ __forceinline__ int row_sequence(const AttnArgs &a, int row) {
    if (!a.row_start) return row < a.n_seqs ? row : -1;
    int lo = 0, hi = a.n_seqs - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (a.row_start[mid] <= row) lo = mid;
        else hi = mid - 1;
    }
    return a.row_start[lo] <= row && row < a.row_start[lo + 1] ? lo : -1;
}

// Rows of a sequence and the position of its row `row`.
__device__ __forceinline__ int64_t row_position(const AttnArgs &a, int b, int row) {
    if (!a.row_start) return (int64_t)a.kv_len[b] - 1;
    return (int64_t)a.kv_len[b] - a.row_start[b + 1] + row;
}

__device__ __forceinline__ void raise(uint32_t *flags, uint32_t bit) {
    if (!(__hip_atomic_load(flags, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) & bit)) atomicOr(flags, bit);
}

template <typename T, int N>
struct alignas(sizeof(T) * N) Vec {
    T v[N];
};

// 8 elements a thread, keys then values of a row: one 16-byte store each.
template <typename IN, typename T, int D>
__global__ __launch_bounds__(256) void k_kv_append(AppendArgs p) {
    const AttnArgs &a = p.c;
    const int per_row = 2 * a.hkv * (D / 8);
    const int64_t n = (int64_t)a.n_rows * per_row;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
        const int row = (int)(i / per_row), e = (int)(i - (int64_t)row * per_row);
        const int b = row_sequence(a, row);
        if (b < 0) continue;
        const int64_t pos = row_position(a, b, row);
        if (pos < 0 || (pos >> a.page_shift) >= a.max_pages) {
            raise(a.flags, MOE_DEVFLAG_BAD_SEQ);
            continue;
        }
        const int page = a.pages[b * a.pages_stride + (pos >> a.page_shift)];
        if ((unsigned)page >= (unsigned)a.n_pages) {
            raise(a.flags, MOE_DEVFLAG_BAD_PAGE);
            continue;
        }
        const int which = e >= a.hkv * (D / 8);
        const int he = e - which * a.hkv * (D / 8);
        const int h = he / (D / 8), d = he % (D / 8) * 8;
        const IN *src = (const IN *)(p.src[which] + row * p.src_stride[which]) + h * D + d;
        const Vec<IN, 8> x = *(const Vec<IN, 8> *)src;
        Vec<T, 8> y;
        for (int j = 0; j < 8; ++j) y.v[j] = (T)x.v[j];
        T *dst = (T *)p.dst[which] + page * a.page_stride + h * a.head_stride +
                 (pos & ((1 << a.page_shift) - 1)) * a.token_stride + d;
        *(Vec<T, 8> *)dst = y;
    }
}

// One wave per (row, query head), the cached tokens one after the other.
template <typename T, int D>
__global__ __launch_bounds__(256) void k_attn(AttnArgs a) {
    constexpr int N = D / 64;
    const int lane = threadIdx.x & 63;
    const int64_t unit = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (unit >= (int64_t)a.n_rows * a.hq) return;
    const int row = (int)(unit / a.hq), h = (int)(unit - (int64_t)row * a.hq);
    const int b = row_sequence(a, row);
    if (b < 0) return;
    const int64_t cap = (int64_t)a.max_pages << a.page_shift;
    const int64_t len = a.kv_len[b];
    if (len < 0 || len > cap) raise(a.flags, MOE_DEVFLAG_BAD_SEQ);
    int64_t seen = row_position(a, b, row) + 1;
    if (seen > cap) seen = cap;
    const Vec<T, N> qv = *(const Vec<T, N> *)((const T *)a.q + row * a.q_stride + h * D + lane * N);
    float q[N], acc[N], m = -INFINITY, l = 0.f;
    for (int i = 0; i < N; ++i) q[i] = (float)qv.v[i], acc[i] = 0.f;
    const int hk = h / a.group;
    for (int64_t j = 0; j < seen; ++j) {
        const int page = a.pages[b * a.pages_stride + (j >> a.page_shift)];
        if ((unsigned)page >= (unsigned)a.n_pages) {
            raise(a.flags, MOE_DEVFLAG_BAD_PAGE);
            continue;
        }
        const int64_t at = page * a.page_stride + hk * a.head_stride +
                           (j & ((1 << a.page_shift) - 1)) * a.token_stride + lane * N;
        const Vec<T, N> kv = *(const Vec<T, N> *)((const T *)a.k + at);
        const Vec<T, N> vv = *(const Vec<T, N> *)((const T *)a.v + at);
        float s = 0.f;
        for (int i = 0; i < N; ++i) s += q[i] * (float)kv.v[i];
        for (int o = 1; o < 64; o <<= 1) s += __shfl_xor(s, o);
        s *= a.scale_log2;
        const float mn = fmaxf(m, s);
        const float f = mn == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - mn);
        const float e = mn == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(s - mn);
        l = l * f + e;
        for (int i = 0; i < N; ++i) acc[i] = acc[i] * f + e * (float)vv.v[i];
        m = mn;
    }
    Vec<T, N> y;
    for (int i = 0; i < N; ++i) y.v[i] = (T)(l == 0.f ? 0.f : acc[i] / l);
    *(Vec<T, N> *)((T *)a.o + row * a.o_stride + h * D + lane * N) = y;
    if (a.lse && lane == 0) a.lse[(int64_t)row * a.hq + h] = l == 0.f ? -INFINITY : (m + __log2f(l)) * 0.69314718055994531f;
}

__global__ void k_attn_flags(uint32_t *flags, uint32_t *dst) { *dst = atomicExch(flags, 0u); }

template <typename IN, typename T>
hipError_t append_d(const AppendArgs &a, int d, hipStream_t st) {
    const int64_t n = (int64_t)a.c.n_rows * 2 * a.c.hkv * (d / 8);
    const unsigned grid = (unsigned)(n / 256 + 1 < 8192 ? n / 256 + 1 : 8192);
    if (d == 64) k_kv_append<IN, T, 64><<<grid, 256, 0, st>>>(a);
    else if (d == 128) k_kv_append<IN, T, 128><<<grid, 256, 0, st>>>(a);
    else k_kv_append<IN, T, 256><<<grid, 256, 0, st>>>(a);
    return hipGetLastError();
}

template <typename T>
hipError_t attn_d(const AttnArgs &a, int d, hipStream_t st) {
    const unsigned grid = (unsigned)(((int64_t)a.n_rows * a.hq + 3) / 4);
    if (d == 64) k_attn<T, 64><<<grid, 256, 0, st>>>(a);
    else if (d == 128) k_attn<T, 128><<<grid, 256, 0, st>>>(a);
    else k_attn<T, 256><<<grid, 256, 0, st>>>(a);
    return hipGetLastError();
}

} // namespace

hipError_t launch_kv_append(const AppendArgs &a, int type, int in_type, int d, hipStream_t st) {
    if (type == MOE_T_F16)
        return in_type == MOE_T_F32 ? append_d<float, f16_t>(a, d, st) : append_d<f16_t, f16_t>(a, d, st);
    return in_type == MOE_T_F32 ? append_d<float, bf16_t>(a, d, st) : append_d<bf16_t, bf16_t>(a, d, st);
}

hipError_t launch_attn(const AttnArgs &a, int type, int d, hipStream_t st) {
    return type == MOE_T_F16 ? attn_d<f16_t>(a, d, st) : attn_d<bf16_t>(a, d, st);
}

hipError_t launch_attn_flags(uint32_t *flags, uint32_t *dst, hipStream_t st) {
    k_attn_flags<<<1, 1, 0, st>>>(flags, dst);
    return hipGetLastError();
}

} // namespace moe
