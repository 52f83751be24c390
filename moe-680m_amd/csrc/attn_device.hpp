// attn_device.hpp -- device helpers of the attention kernels.
#pragma once

#include "attn_internal.hpp"
#include "moe_device.hpp"

namespace moe {

typedef __bf16 bf16_t;
typedef _Float16 f16_t;
typedef f16_t f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef bf16_t bf16x2 __attribute__((ext_vector_type(2)));

// Softmax weights meet the values in the cache's type.  They are taken relative to the running
// maximum and, for f16, 2^15 above it: f16 keeps all its bits down to 2^-14, so a weight loses bits
// only below 2^-29 of the largest (unshifted below 2^-14, where thousands of such keys can hold most
// of the mass).  bf16 has f32's range.
template <typename T>
struct Elem;
template <>
struct Elem<f16_t> {
    typedef f16x8 x8;
    static constexpr float SHIFT = 15.f;
    static __device__ __forceinline__ uint32_t pack(float a, float b) {
        return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{a, b}), f16x2));
    }
    static __device__ __forceinline__ f32x4 mfma16(x8 a, x8 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
    }
    static __device__ __forceinline__ f32x16 mfma32(x8 a, x8 b, f32x16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
    }
};
template <>
struct Elem<bf16_t> {
    typedef bf16x8 x8;
    static constexpr float SHIFT = 0.f;
    static __device__ __forceinline__ uint32_t pack(float a, float b) {
        return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{a, b}), bf16x2));
    }
    static __device__ __forceinline__ f32x4 mfma16(x8 a, x8 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
    }
    static __device__ __forceinline__ f32x16 mfma32(x8 a, x8 b, f32x16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
    }
};

__device__ __forceinline__ float exp2_(float x) { return __builtin_amdgcn_exp2f(x); }
// The maximum to subtract: 0 while no score was seen (every score -inf: all weights 0).
__device__ __forceinline__ float base_of(float m) { return m == -INFINITY ? 0.f : m; }

__device__ __forceinline__ void raise(uint32_t *flags, uint32_t bit) {
    __hip_atomic_fetch_or((MOE_GLOBAL uint32_t *)flags, bit, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// A load from an address that is the same in all lanes, of memory that no launch under way writes:
// through the scalar cache, so it waits for no vector load in flight.
template <typename T>
__device__ __forceinline__ T ldc(const T *p) {
    return *(const __attribute__((address_space(4))) T *)p;
}

// A load at a lane's 32-bit offset (and a constant) from an address that is the same in all lanes.
template <typename T>
__device__ __forceinline__ T ldo(const uint8_t *base, uint32_t off, int imm = 0) {
    return *(const MOE_GLOBAL T *)((const MOE_GLOBAL uint8_t *)base + off + imm);
}

// The kernel's argument block (its only argument), read again: where only an epilogue uses them, the
// arguments are not held in scalar registers through the loop before it.
__device__ __forceinline__ const __attribute__((address_space(4))) AttnArgs &fresh_args() {
    auto p = (const __attribute__((address_space(4))) AttnArgs *)__builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(p));
    return *p;
}

// Inclusive sum over the wave's lanes.
__device__ __forceinline__ uint32_t wave_scan(uint32_t x) {
    x += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x111, 0xf, 0xf, false); // row_shr:1
    x += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x112, 0xf, 0xf, false); // row_shr:2
    x += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x114, 0xf, 0xf, false); // row_shr:4
    x += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x118, 0xf, 0xf, false); // row_shr:8
    x += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x142, 0xa, 0xf, false); // row_bcast:15
    x += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x143, 0xc, 0xf, false); // row_bcast:31
    return x;
}

// 2^shift sets of 64 sequences make a group, of which there are up to 64.
__device__ __forceinline__ int group_shift(int n_seqs) {
    int shift = 0;
    while ((n_seqs - 1) >> (12 + shift)) ++shift;
    return shift;
}
// Something counted for each sequence (count(b) for any b, 0 behind the last one): of up to 64 sequences lane b has
// sequence b's, of more lane c those of the c-th of up to 64 groups; incl: with all in front.  All four waves
// of a workgroup call it, and share the sequences where they are many.  Neighbours' loads lie side by side
// (each lane of every wave a run of sequences, the run searched one by one: 4096 prompts of 16 rows 541 us, so
// 142; 1024 of them 42, 25).
template <typename Count>
__device__ __forceinline__ void count_seqs(int n_seqs, int lane, int wave, Count count, uint32_t &mine, uint32_t &incl) {
    if (n_seqs <= 64) mine = count(lane);
    else {
        constexpr int AT_ONCE = 4;
        __shared__ uint32_t s_mine[4][64];
        const int sets = (n_seqs + 63) / 64, shift = group_shift(n_seqs);
        mine = 0;
        for (int k = wave * AT_ONCE; k < sets; k += 4 * AT_ONCE) {
            uint32_t n[AT_ONCE];
#pragma unroll
            for (int i = 0; i < AT_ONCE; ++i) n[i] = count((k + i) * 64 + lane);
#pragma unroll
            for (int i = 0; i < AT_ONCE; ++i) {
                const uint32_t sum = (uint32_t)__builtin_amdgcn_readlane((int)wave_scan(n[i]), 63);
                mine += lane == (k + i) >> shift ? sum : 0u;
            }
        }
        s_mine[wave][lane] = mine;
        __syncthreads();
        mine = (s_mine[0][lane] + s_mine[1][lane]) + (s_mine[2][lane] + s_mine[3][lane]);
    }
    incl = wave_scan(mine);
}
// The sequence that has the want-th of what was counted, and what is in front of it; `from`: the lane that
// counted it last.
template <typename Count>
__device__ __forceinline__ int find_seq(int n_seqs, int lane, Count count, uint32_t mine, uint32_t incl, uint32_t want,
                                        uint32_t &before, int &from) {
    from = __builtin_ctzll(__ballot(incl > want));
    before = (uint32_t)__builtin_amdgcn_readlane((int)(incl - mine), from);
    if (n_seqs <= 64) return from;
    const int shift = group_shift(n_seqs), last = ((from + 1) << shift) - 1;
    for (int k = from << shift;; ++k) {
        const uint32_t n = count(k * 64 + lane), upto = before + wave_scan(n);
        const uint64_t in = __ballot(upto > want);
        if (in || k >= last) { // (none: the counts changed during the call)
            from = in ? __builtin_ctzll(in) : 0;
            before = (uint32_t)__builtin_amdgcn_readlane((int)(upto - n), from);
            return min(k * 64 + from, n_seqs - 1);
        }
        before = (uint32_t)__builtin_amdgcn_readlane((int)upto, 63);
    }
}

// The largest of the wave's lanes.
__device__ __forceinline__ uint32_t wave_most(uint32_t x) {
    x = max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x111, 0xf, 0xf, false)); // as above
    x = max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x112, 0xf, 0xf, false));
    x = max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x114, 0xf, 0xf, false));
    x = max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x118, 0xf, 0xf, false));
    x = max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x142, 0xa, 0xf, false));
    x = max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x143, 0xc, 0xf, false));
    return (uint32_t)__builtin_amdgcn_readlane((int)x, 63);
}

__device__ __forceinline__ float wave_max(float x) {
    for (int o = 1; o < 64; o <<= 1) x = fmaxf(x, __shfl_xor(x, o));
    return x;
}
#define MOE_LDS __attribute__((address_space(3)))
// 16 bytes a lane straight to LDS: lane i's to lds + 16 i.  They are there behind lds_loaded() (and, for
// other waves, a barrier).
__device__ __forceinline__ void lds_load16(const uint8_t *base, uint32_t off, void *lds) {
    __builtin_amdgcn_global_load_lds((const MOE_GLOBAL void *)((const MOE_GLOBAL uint8_t *)base + off), (MOE_LDS void *)lds,
                                     16, 0, 0);
}
__device__ __forceinline__ void lds_loaded() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

// The transposing LDS read: among 16 lanes, lane 4 j + c addresses elements 4c..4c+3 of row j, lane i gets
// element i of rows 0..3.
typedef short s16x4 __attribute__((ext_vector_type(4)));
__device__ __forceinline__ u32x2 lds_read_tr(const MOE_LDS uint8_t *p) {
    return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((MOE_LDS s16x4 *)p));
}
// An LDS address held in a register: reads add their constants (16 bits) to it in the instruction.
__device__ __forceinline__ const MOE_LDS uint8_t *lds_at(const void *base, uint32_t off) {
    const MOE_LDS uint8_t *p = (const MOE_LDS uint8_t *)base + off;
    asm("" : "+v"(p));
    return p;
}

__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }

// Four elements of a finished row: x / L, and with the first ones the log of the sum; the weights were
// 2^(score - M + shift).
template <typename T, typename Args>
__device__ __forceinline__ void put_row(const Args &a, int row, int h, int D, int d, f32x4 x, float M, float L,
                                        float shift) {
    typedef Elem<T> E;
    const float inv = 1.f / L;
    x = L == 0.f ? f32x4{0.f, 0.f, 0.f, 0.f} : x * inv;
    *(u32x2 *)((T *)a.o + row * a.o_stride + (int64_t)h * D + d) = u32x2{E::pack(x[0], x[1]), E::pack(x[2], x[3])};
    if (a.lse && d == 0)
        a.lse[(int64_t)row * a.hq + h] =
            L == 0.f ? -INFINITY : (base_of(M) - shift + __log2f(L)) * 0.69314718055994531f;
}

} // namespace moe
