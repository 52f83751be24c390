// k_attn.hip -- the key-value cache's write, and the attention's flags.
#include "attn_device.hpp"

namespace moe {

namespace {

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

} // namespace

hipError_t launch_kv_append(const AppendArgs &a, int type, int in_type, int d, hipStream_t st) {
    if (type == MOE_T_F16)
        return in_type == MOE_T_F32 ? append_d<float, f16_t>(a, d, st) : append_d<f16_t, f16_t>(a, d, st);
    return in_type == MOE_T_F32 ? append_d<float, bf16_t>(a, d, st) : append_d<bf16_t, bf16_t>(a, d, st);
}

hipError_t launch_attn_flags(uint32_t *flags, uint32_t *dst, hipStream_t st) {
    k_attn_flags<<<1, 1, 0, st>>>(flags, dst);
    return hipGetLastError();
}

} // namespace moe
