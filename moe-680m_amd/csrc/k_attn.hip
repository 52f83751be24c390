// k_attn.hip -- the key-value cache's write, and the attention's flags.
#include "attn_device.hpp"

namespace moe {

namespace {

// 8 elements, as 32-bit words.
template <typename T>
struct Eight {
    uint32_t w[2 * sizeof(T)];
};
__device__ __forceinline__ uint32_t pack2(float a, float b, f16_t) { return Elem<f16_t>::pack(a, b); }
__device__ __forceinline__ uint32_t pack2(float a, float b, bf16_t) { return Elem<bf16_t>::pack(a, b); }

// New keys and values to their places, a wave a row.  A copy: bound by its bytes, and for few rows by
// the chain row -> sequence -> length -> page -> place, whose links are looked up by the wave as one
// (64 sequences at a time) while the row's first 4 KB (8 KB of f32) are loaded.  9976 rows of two heads
// of 256, bf16: 9.6 us (41 MB, 4.3 TB/s); a thread for each 16 bytes, each with its own search, 11.5 us.
template <typename IN, typename T, int D>
__global__ __launch_bounds__(256) void k_kv_append(AppendArgs p) {
    constexpr int AHEAD = 4; // of a lane's 8-element units
    const AttnArgs &a = p.c;
    const int lane = threadIdx.x & 63, row = blockIdx.x * 4 + uniform(threadIdx.x >> 6);
    if (row >= a.n_rows) return;
    const int half = a.hkv * (D / 8), units = 2 * half; // keys' units, then values'
    const uint8_t *src[2] = {p.src[0] + row * p.src_stride[0], p.src[1] + row * p.src_stride[1]};
    auto load = [&](int e) {
        Eight<IN> x;
        const uint8_t *at = e < half ? src[0] + e * (8 * sizeof(IN)) : src[1] + (e - half) * (8 * sizeof(IN));
#pragma unroll
        for (int i = 0; i < (int)sizeof(IN) / 2; ++i) {
            const u32x4 w = ldg<u32x4>(at + 16 * i);
            for (int j = 0; j < 4; ++j) x.w[4 * i + j] = w[j];
        }
        return x;
    };
    Eight<IN> x[AHEAD];
#pragma unroll
    for (int i = 0; i < AHEAD; ++i)
        if (lane + 64 * i < units) x[i] = load(lane + 64 * i);

    // the sequence, or none
    int b = row;
    int64_t pos; // place in it
    if (a.row_start) {
        int lo = 0, hi = (a.n_seqs - 1) >> 6; // 64 sequences: the last ones that begin at the row or before it
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (ldc(a.row_start + 64 * mid) <= row) lo = mid;
            else hi = mid - 1;
        }
        const int i = 64 * lo + lane;
        const bool here = i < a.n_seqs && ldg<int>(a.row_start + i) <= row && row < ldg<int>(a.row_start + i + 1);
        const uint64_t in = __ballot(here);
        if (!in) return;
        b = 64 * lo + __builtin_ctzll(in);
        pos = (int64_t)ldc(a.kv_len + b) - ldc(a.row_start + b + 1) + row;
    } else pos = (int64_t)ldc(a.kv_len + b) - 1;
    if (pos < 0 || (pos >> a.page_shift) >= a.max_pages) {
        if (lane == 0) raise(a.flags, MOE_DEVFLAG_BAD_SEQ);
        return;
    }
    const int page = ldc(a.pages + b * a.pages_stride + (pos >> a.page_shift));
    if ((unsigned)page >= (unsigned)a.n_pages) {
        if (lane == 0) raise(a.flags, MOE_DEVFLAG_BAD_PAGE);
        return;
    }
    const int64_t place = page * a.page_stride + (pos & ((1 << a.page_shift) - 1)) * a.token_stride;
    auto store = [&](int e, const Eight<IN> &x) {
        const int which = e >= half, he = e - which * half, h = he / (D / 8), d = he % (D / 8) * 8;
        u32x4 y;
        if constexpr (sizeof(IN) == sizeof(T)) y = u32x4{x.w[0], x.w[1], x.w[2], x.w[3]};
        else
            for (int j = 0; j < 4; ++j)
                y[j] = pack2(__builtin_bit_cast(float, x.w[2 * j]), __builtin_bit_cast(float, x.w[2 * j + 1]), T{});
        *(u32x4 *)((T *)p.dst[which] + place + h * a.head_stride + d) = y;
    };
#pragma unroll
    for (int i = 0; i < AHEAD; ++i)
        if (lane + 64 * i < units) store(lane + 64 * i, x[i]);
    for (int e = lane + 64 * AHEAD; e < units; e += 64) store(e, load(e));
}

__global__ void k_attn_flags(uint32_t *flags, uint32_t *dst) { *dst = atomicExch(flags, 0u); }

template <typename IN, typename T>
hipError_t append_d(const AppendArgs &a, int d, hipStream_t st) {
    const unsigned grid = (unsigned)((a.c.n_rows + 3) / 4);
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
