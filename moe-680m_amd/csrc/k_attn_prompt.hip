// k_attn_prompt.hip -- packed causal prompts over the paged cache.
//
//   o[i][h] = sum_{j <= p_i} e^(s_ij - m_i) V_j / sum_j e^(s_ij - m_i),   s_ij = scale * q[i][h] . K_j,
//   p_i the row's position (kv_len - rows + i)
//
// Bound by the matrix cores: 4 D operations for each (row, head, seen token).  A workgroup's rows are
// 128 NQ (token, head) pairs of one key-value head, the heads of a token side by side, so the
// group's heads share each tile of K and V and the causal edge crosses few of them.
//   * A wave takes NQ blocks of 32 rows, a row to a lane pair:
//       S^T[token][row] = K Q^T      32x32x16 products; a row's scores lie in the lanes r and r + 32,
//                                    so maximum, sum and rescaling are a lane's own (and one swap)
//       O^T[d][row] += V^T P^T       S^T's register layout is P^T's operand layout with the tokens of 16
//                                    in the order {0-3, 8-11}, {4-7, 12-15}; V^T is stored in that order
//   * K and V tiles of BN tokens go straight to LDS (no registers), two buffers, one barrier a tile; the
//     next tile's loads are under way while this one is worked on.  V^T is read by the transposing LDS
//     load: of 16 lanes, lane 4 j + c gives the address of elements 4c..4c+3 of token j, lane d gets
//     element d of tokens 0..3.  A row's 16-byte chunks are stored at chunk ^ f(token), f = token & 7 for K
//     and 2 (token & 3) for V, so that all reads are free of bank conflicts.
//   * A fragment read from LDS serves the NQ row blocks of a wave.
//   * The running maximum is only raised when a row's new one exceeds it by more than 2^8: until then
//     the weights stay below 2^(8 + SHIFT) and no output is rescaled.
#include "attn_device.hpp"

namespace moe {

namespace {

constexpr float LAZY = 8.f;     // log2 of what a weight may exceed 1 by

struct Rows {
    int r0, n;
    bool bad;
};
// The packed rows of sequence b, inside the arrays whatever row_start holds.
__device__ __forceinline__ Rows seq_rows(const AttnArgs &a, int b) {
    const int s = a.row_start[b], e = a.row_start[b + 1];
    const int r0 = min(max(s, 0), a.n_rows), r1 = min(max(e, r0), a.n_rows);
    return {r0, r1 - r0, r0 != s || r1 != e};
}

// Of two elements in a word: whether one is an infinity or NaN; the word with those as 0.
template <typename T>
constexpr uint32_t EXP = __is_same(T, f16_t) ? 0x7c00u : 0x7f80u;
template <typename T>
__device__ __forceinline__ bool not_finite(uint32_t w) {
    return (w & EXP<T>) == EXP<T> || (w >> 16 & EXP<T>) == EXP<T>;
}
template <typename T>
__device__ __forceinline__ uint32_t finite_only(uint32_t w) {
    if ((w & EXP<T>) == EXP<T>) w &= 0xffff0000u;
    if ((w >> 16 & EXP<T>) == EXP<T>) w &= 0xffffu;
    return w;
}

// Products of N fragments, each read from LDS DEPTH products before its own.  The order is kept as written
// (by itself the compiler reads, waits, multiplies).
template <int N, int DEPTH, typename Frag, typename Read, typename Product>
__device__ __forceinline__ void products(Read read, Product product) {
    Frag f[DEPTH];
#pragma unroll
    for (int i = 0; i < DEPTH; ++i) f[i] = read(i);
#pragma unroll
    for (int i = 0; i < N; ++i) {
        product(i, f[i % DEPTH]);
        if (i + DEPTH < N) f[i % DEPTH] = read(i + DEPTH);
        __builtin_amdgcn_sched_barrier(0);
    }
}

template <typename T, int D, int NQ, int BN>
__global__ __launch_bounds__(256, NQ * D >= 256 ? 1 : 2) void k_attn_prompt(AttnArgs a) {
    typedef Elem<T> E;
    typedef typename E::x8 x8;
    constexpr int KS = D / 16;           // products of a score tile
    constexpr int NB = BN / 16;          // blocks of 16 tokens, each in one page
    constexpr int NS = BN / 32;          // score tiles
    constexpr int RI = 512 / D;          // tokens of one wave load
    constexpr int NL = BN / 4 / RI;      // loads of a wave and tile, for K and for V
    constexpr int ROWS = 128 * NQ;
    constexpr int DEPTH = D == 64 ? 4 : 6; // fragments read ahead
    constexpr float SHIFT = E::SHIFT > 0.f ? 7.f : 0.f; // f16: 2^(SHIFT + LAZY) is in range
    __shared__ __attribute__((aligned(16))) T s_k[2][BN * D];
    __shared__ __attribute__((aligned(16))) T s_v[2][BN * D];
    __shared__ int s_bad;

    const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6);
    const int r = lane & 31, h = lane >> 5;
    const int cap = a.max_pages << a.page_shift;

    // ---- this workgroup's rows: tile numbers run over the sequences, the last one first (it sees the
    // most tokens); the key-value head is the fastest index, so that a head's tiles share an XCD's L2
    const int per = (a.n_seqs + 63) / 64;
    uint32_t mine = 0;
    bool bad_rows = false;
    for (int i = 0; i < per; ++i) {
        const int b = lane * per + i;
        if (b < a.n_seqs) {
            const Rows w = seq_rows(a, b);
            bad_rows |= w.bad;
            mine += (uint32_t)(((int64_t)w.n * a.group + ROWS - 1) / ROWS);
        }
    }
    if (blockIdx.x == 0 && bad_rows) raise(a.flags, MOE_DEVFLAG_BAD_SEQ);
    const uint32_t incl = wave_scan(mine);
    const uint32_t total = (uint32_t)__builtin_amdgcn_readlane((int)incl, 63);
    const uint32_t nth = blockIdx.x / a.hkv;
    if (nth >= total) return;
    const int hk = blockIdx.x - nth * a.hkv;
    uint32_t want = total - 1 - nth;
    // All at work at once, two on some CUs: there the lighter one is to lie beside the heavier one.
    const uint32_t first = a.n_cu / a.hkv; // (head groups of) tiles that take a CU each
    if (D < 256 && total > first && total * a.hkv <= 2u * a.n_cu && nth >= first) want = nth - first;
    const int owner = __builtin_ctzll(__ballot(incl > want));
    uint32_t at = (uint32_t)__builtin_amdgcn_readlane((int)(incl - mine), owner);
    int b = owner * per;
    Rows sr;
    for (;; ++b) {
        sr = seq_rows(a, uniform(b));
        const uint32_t n = (uint32_t)(((int64_t)sr.n * a.group + ROWS - 1) / ROWS);
        if (want < at + n) break;
        at += n;
    }
    b = uniform(b);
    sr.r0 = uniform(sr.r0);
    sr.n = uniform(sr.n);
    if (tid == 0) s_bad = 0;

    // ---- rows: number f of the sequence's (token, head) pairs, position
    const int64_t f0 = (int64_t)(want - at) * ROWS, nf = (int64_t)sr.n * a.group;
    const int len = ldc(a.kv_len + b);
    if ((len < 0 || len > cap) && tid == 0) raise(a.flags, MOE_DEVFLAG_BAD_SEQ);
    const int64_t first_pos = (int64_t)len - ldc(a.row_start + b + 1) + sr.r0; // of the sequence's first row
    auto seen_by = [&](int64_t f) { // tokens that pair f's row sees
        const int64_t p = first_pos + f / a.group + 1;
        return (int)(p < 0 ? 0 : p > cap ? cap : p);
    };
    const int64_t wf0 = f0 + wave * (32 * NQ);
    const int64_t f_last = f0 + ROWS < nf ? f0 + ROWS : nf;
    const int ext = uniform(seen_by(f_last - 1));  // tokens that some row of the workgroup sees
    const int full = uniform(seen_by(f0));         // ... that all see
    // a lane's rows: pair wf0 + 32 n + r; one behind the last reads the last one's query and sees nothing
    auto pair = [&](int n) { return wf0 + 32 * n + r; };
    auto q_at = [&](int n, int64_t stride) {
        const int64_t f = pair(n) < nf ? pair(n) : nf - 1, tok = f / a.group;
        return (sr.r0 + tok) * stride + (hk * a.group + (f - tok * a.group)) * D;
    };
    int seen[NQ];
    x8 qf[NQ][KS];
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
        seen[n] = pair(n) < nf ? seen_by(pair(n)) : 0;
        const T *q = (const T *)a.q + q_at(n, a.q_stride) + h * 8;
        const uint32_t flip = a.scale_log2 < 0.f ? 0x80008000u : 0u; // a negative scale: -q, exactly
#pragma unroll
        for (int k = 0; k < KS; ++k) {
            u32x4 w = ldg<u32x4>(q + k * 16);
            for (int i = 0; i < 4; ++i) w[i] ^= flip;
            qf[n][k] = __builtin_bit_cast(x8, w);
        }
    }
    // Scale 0: the smallest normal number, so that -inf (not seen) stays -inf; any finite score times it
    // is 0 beside the exponential's 1.
    const float scale = fmaxf(fabsf(a.scale_log2), 1.17549435e-38f);

    // ---- tiles
    const int nt = (ext + BN - 1) / BN;
    const int32_t *pages = a.pages + b * a.pages_stride;
    const uint8_t *kb = a.k + 2 * hk * a.head_stride, *vb = a.v + 2 * hk * a.head_stride;
    const int ts2 = (int)(2 * a.token_stride), mask = (1 << a.page_shift) - 1;
    // Lane i has the page of block i of the tile to be staged next (-1: none); okay: the blocks of the tile
    // staged last that have a page of the cache, or no token to be seen.
    bool bad_page = false;
    uint32_t okay = 0;
    auto look_up = [&](int t) {
        const int key = t * BN + 16 * lane;
        return lane < NB && key < ext ? ldg<int>(pages + (key >> a.page_shift)) : -1;
    };
    int pg_next = look_up(0);
    int64_t off = 0; // of this wave's quarter of the tile: one block's, or a part of it; tokens there
    int toks = 0;
    auto stage = [&](int t) {
        const int blk = wave * NB / 4, key = t * BN + 16 * blk;
        const uint64_t in = __ballot((unsigned)pg_next < (unsigned)a.n_pages);
        const uint64_t none = __ballot(t * BN + 16 * lane >= ext);
        okay = (uint32_t)(in | none);
        bad_page |= (okay & ((1u << NB) - 1)) != (1u << NB) - 1;
        const bool here = in >> blk & 1;
        const int pg = here ? __builtin_amdgcn_readlane(pg_next, blk) : 0;
        toks = here ? min(16, ext - key) : 0;
        off = 2 * (pg * a.page_stride + (key & mask) * a.token_stride);
        if (t + 1 < nt) pg_next = look_up(t + 1);
    };
    // Every wave loads its quarter.  Tokens that are not there are taken from a place that is (masked below).
    auto stage_load = [&](const uint8_t *base, T *lds, bool values) {
#pragma unroll
        for (int p = 0; p < NL; ++p) {
            const int key = (wave * NL + p) * RI + lane / (D / 8), ch = lane % (D / 8); // of the tile
            const int tok = max(0, min(key & 15, toks - 1));
            lds_load16(base + off, (uint32_t)(tok * ts2 + (ch ^ (values ? 2 * (key & 3) : key & 7)) * 16),
                       lds + (wave * NL + p) * 512);
        }
    };

    f32x16 o[NQ][D / 32];
    float m[NQ], l[NQ]; // the maximum that weights are taken against, and this lane's sum
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
#pragma unroll
        for (int i = 0; i < D / 32; ++i) o[n][i] = f32x16{};
        m[n] = -INFINITY;
        l[n] = 0.f;
    }
    uint32_t ko[4], vo[2];
#pragma unroll
    for (int i = 0; i < 4; ++i) ko[i] = r * (D * 2) + (((2 * i + h) ^ (r & 7)) * 16);
    {
        const int j = (lane & 15) >> 2, c = 2 * (r >> 4) + ((lane & 3) >> 1); // token, chunk of its first 64 bytes
        vo[0] = (4 * h + j) * (D * 2) + ((c ^ (2 * j)) * 16) + 8 * (lane & 1);
        vo[1] = vo[0] ^ 64;
    }

    if (nt > 0) {
        stage(0);
        stage_load(kb, s_k[0], false);
        stage_load(vb, s_v[0], true);
    }
    bool fresh = true, part = false;
    uint32_t ok = 0;
    for (int t = 0; t < nt;) {
        // Tiles until a row's maximum grows past what its weights allow for; then the outputs are rescaled
        // and the tile's scores computed again.  (Two loops, so that the inner one's outputs are the
        // products' own and stay where those put them.)
        float mx[NQ];
        for (;;) {
            const int buf = t & 1;
            const uint8_t *lk = (const uint8_t *)s_k[buf], *lv = (const uint8_t *)s_v[buf];
            if (fresh) {
                ok = okay;
                // a tile that some row does not see all of
                part = (t + 1) * BN > full || (ok & ((1u << NB) - 1)) != (1u << NB) - 1;
                lds_loaded();
                __syncthreads(); // tile t is there, and nobody works on tile t - 1
                // A value that a row does not see meets a weight of 0, which an infinity or NaN would survive:
                                // in such a tile those are 0 for the products, and the rows that see them get them at the end.
                                if (part) {
                                    bool bad = false;
                #pragma unroll 1
                                    for (int i = tid; i < BN * D / 8; i += 256) {
                                        u32x4 *p = (u32x4 *)s_v[buf] + i;
                                        u32x4 w = *p;
                                        bool any = false;
                                        for (int j = 0; j < 4; ++j) any |= not_finite<T>(w[j]);
                                        if (any) {
                                            for (int j = 0; j < 4; ++j) w[j] = finite_only<T>(w[j]);
                                            *p = w;
                                            bad = true;
                                        }
                                    }
                                    if (bad) s_bad = 1;
                                    __syncthreads();
                                }
                if (t + 1 < nt) {
                    stage(t + 1);
                    stage_load(kb, s_k[buf ^ 1], false);
                    stage_load(vb, s_v[buf ^ 1], true);
                }
            }
            f32x16 s[NQ][NS];
            auto read_k = [&](int x) { // the score tiles in turn: two chains of sums
                const int i = x % NS, k = x / NS;
                return *(const x8 *)(lk + ko[k & 3] + i * (32 * D * 2) + (k >> 2) * 128);
            };
            auto mul_k = [&](int x, x8 kf) {
                const int i = x % NS, k = x / NS;
#pragma unroll
                for (int n = 0; n < NQ; ++n) s[n][i] = E::mfma32(kf, qf[n][k], k ? s[n][i] : f32x16{});
            };
            products<NS * KS, DEPTH, x8>(read_k, mul_k);
            if (part)
#pragma unroll
                for (int n = 0; n < NQ; ++n)
#pragma unroll
                    for (int i = 0; i < NS; ++i)
#pragma unroll
                        for (int j = 0; j < 16; ++j) {
                            const int key = 32 * i + 8 * (j >> 2) + 4 * h + (j & 3);
                            if (t * BN + key >= seen[n] || !(ok >> (2 * i + (j >> 3)) & 1)) s[n][i][j] = -INFINITY;
                        }
            bool grows = false;
#pragma unroll
            for (int n = 0; n < NQ; ++n) {
                mx[n] = s[n][0][0];
#pragma unroll
                for (int i = 0; i < NS; ++i)
#pragma unroll
                    for (int j = 0; j < 16; ++j) mx[n] = fmaxf(mx[n], s[n][i][j]);
                mx[n] = fmaxf(mx[n], __shfl_xor(mx[n], 32)) * scale;
                grows |= mx[n] > m[n] + LAZY;
            }
            fresh = !__any(grows);
            if (!fresh) break;
            u32x4 pw[NQ][2 * NS]; // the weights, in P^T's operand layout
#pragma unroll
            for (int n = 0; n < NQ; ++n) {
                const float base = base_of(m[n]) - SHIFT;
                float sum = 0.f;
#pragma unroll
                for (int i = 0; i < NS; ++i)
#pragma unroll
                    for (int j = 0; j < 16; j += 2) {
                        const float p0 = exp2_(__builtin_fmaf(s[n][i][j], scale, -base));
                        const float p1 = exp2_(__builtin_fmaf(s[n][i][j + 1], scale, -base));
                        sum += p0 + p1;
                        pw[n][2 * i + (j >> 3)][(j & 7) >> 1] = E::pack(p0, p1);
                    }
                l[n] += sum;
            }
            auto read_v = [&](int x) {
                const int k = x / (D / 32), i = x % (D / 32);
                const uint8_t *p = lv + vo[i & 1] + k * (16 * D * 2) + (i >> 1) * 128;
                const u32x2 v0 = lds_read_tr(p), v1 = lds_read_tr(p + 8 * D * 2);
                return __builtin_bit_cast(x8, (u32x4{v0.x, v0.y, v1.x, v1.y}));
            };
            auto mul_v = [&](int x, x8 vf) {
                const int k = x / (D / 32), i = x % (D / 32);
#pragma unroll
                for (int n = 0; n < NQ; ++n) o[n][i] = E::mfma32(vf, __builtin_bit_cast(x8, pw[n][k]), o[n][i]);
            };
            products<NS * D / 16, DEPTH, x8>(read_v, mul_v);
            if (++t == nt) break;
        }
        if (t < nt)
#pragma unroll
            for (int n = 0; n < NQ; ++n) {
                const float mn = fmaxf(m[n], mx[n]);
                const float alpha = exp2_(m[n] - base_of(mn));
                m[n] = mn;
                l[n] *= alpha;
#pragma unroll
                for (int i = 0; i < D / 32; ++i) o[n][i] *= alpha;
            }
    }
    if (bad_page && lane == 0) raise(a.flags, MOE_DEVFLAG_BAD_PAGE);

    // ---- the infinities and NaN that were 0 for the products, token by token
    __syncthreads();
    if (*(volatile int *)&s_bad)
#pragma unroll
        for (int n = 0; n < NQ; ++n)
#pragma unroll 1
            for (int key = full / BN * BN; key < seen[n]; ++key) {
                const int pg = pages[key >> a.page_shift];
                if ((unsigned)pg >= (unsigned)a.n_pages) continue;
                const uint8_t *v = vb + 2 * (pg * a.page_stride + (key & mask) * a.token_stride) + 8 * h;
#pragma unroll
                for (int i = 0; i < D / 32; ++i)
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const u32x2 w = ldg<u32x2>(v + 64 * i + 16 * j);
#pragma unroll
                        for (int x = 0; x < 4; ++x) {
                            const uint32_t e = x & 1 ? w[x >> 1] >> 16 : w[x >> 1] & 0xffffu;
                            if (not_finite<T>(e)) o[n][i][4 * j + x] += (float)__builtin_bit_cast(T, (uint16_t)e);
                        }
                    }
            }

    // ---- rows out
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
        const float sum = l[n] + __shfl_xor(l[n], 32);
        if (pair(n) >= nf) continue;
        const float inv = sum == 0.f ? 0.f : 1.f / sum;
        T *op = (T *)a.o + q_at(n, a.o_stride) + 4 * h;
#pragma unroll
        for (int i = 0; i < D / 32; ++i)
#pragma unroll
            for (int j = 0; j < 16; j += 4) {
                u32x2 w = {E::pack(o[n][i][j] * inv, o[n][i][j + 1] * inv),
                           E::pack(o[n][i][j + 2] * inv, o[n][i][j + 3] * inv)};
                if (sum == 0.f) w = u32x2{0u, 0u};
                *(u32x2 *)(op + 32 * i + 2 * j) = w;
            }
        if (a.lse && h == 0)
            a.lse[q_at(n, a.hq * D) / D] =
                sum == 0.f ? -INFINITY : (base_of(m[n]) - SHIFT + __log2f(sum)) * 0.69314718055994531f;
    }
}

template <typename T>
hipError_t prompt_t(const AttnArgs &a, int d, hipStream_t st) {
    // tiles of the rows however they are divided: each sequence's last one may be short
    const int64_t tiles = (int64_t)a.n_rows * a.group / 128 + a.n_seqs;
    const unsigned grid = (unsigned)(tiles * a.hkv);
    if (d == 64) k_attn_prompt<T, 64, 1, 64><<<grid, 256, 0, st>>>(a);
    else if (d == 128) k_attn_prompt<T, 128, 1, 64><<<grid, 256, 0, st>>>(a);
    else k_attn_prompt<T, 256, 1, 64><<<grid, 256, 0, st>>>(a);
    return hipGetLastError();
}

} // namespace

hipError_t launch_attn_prompt(const AttnArgs &a, int type, int d, hipStream_t st) {
    return type == MOE_T_F16 ? prompt_t<f16_t>(a, d, st) : prompt_t<bf16_t>(a, d, st);
}

} // namespace moe
