// k_attn_prompt.hip -- packed causal prompts over the paged cache.
//
//   o[i][h] = sum_{j <= p_i} e^(s_ij - m_i) V_j / sum_j e^(s_ij - m_i),   s_ij = scale * q[i][h] . K_j,
//   p_i the row's position (kv_len - rows + i)
//
// Bound by the matrix cores: 4 D operations for each (row, head, seen token).  A workgroup's rows are
// PR_ROWS (token, head) pairs of one key-value head, the heads of a token side by side, so the
// group's heads share each tile of K and V and the causal edge crosses few of them.
//   * A wave takes 32 rows, one to a lane pair:
//       S^T[token][row] = K Q^T      32x32x16 products; a row's scores lie in the lanes r and r + 32,
//                                    so maximum, sum and rescaling are a lane's own (and one swap)
//       O^T[d][row] += V^T P^T       S^T's register layout is P^T's operand layout with the tokens of 16
//                                    in the order {0-3, 8-11}, {4-7, 12-15}; V^T is stored in that order
//   * K and V tiles of 64 tokens go through LDS, two buffers, one barrier a tile; the next tile's loads
//     are under way while this one is worked on.  K rows are stored with their 16-byte chunks XORed by
//     the row, V transposed in registers (two v_perm a dword pair) and XORed likewise: reads and writes
//     are free of bank conflicts.
//   * The running maximum is only raised when a row's new one exceeds it by more than 2^8: until then
//     the weights stay below 2^(8 + SHIFT) and no output is rescaled.
#include "attn_device.hpp"

namespace moe {

namespace {

constexpr int BN = 64;          // tokens of a tile
constexpr int NB = BN / 16;     // ... in blocks that lie in one page
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

template <typename T>
__device__ __forceinline__ bool not_finite(uint32_t w);
template <>
__device__ __forceinline__ bool not_finite<f16_t>(uint32_t w) {
    return (w & 0x7c00u) == 0x7c00u || (w & 0x7c000000u) == 0x7c000000u;
}
template <>
__device__ __forceinline__ bool not_finite<bf16_t>(uint32_t w) {
    return (w & 0x7f80u) == 0x7f80u || (w & 0x7f800000u) == 0x7f800000u;
}

template <typename T, int D>
__global__ __launch_bounds__(256, D == 256 ? 1 : 2) void k_attn_prompt(AttnArgs a) {
    typedef Elem<T> E;
    typedef typename E::x8 x8;
    constexpr int KS = D / 16;           // products of a score tile
    constexpr int RP = 2048 / D;         // tokens of a pass of the workgroup's K loads
    constexpr int VW = D / 32;           // elements of a lane's V load
    constexpr float SHIFT = E::SHIFT > 0.f ? 7.f : 0.f; // f16: 2^(SHIFT + LAZY) is in range
    typedef uint32_t vload __attribute__((ext_vector_type(VW / 2)));
    __shared__ __attribute__((aligned(16))) T s_k[2][BN * D];
    __shared__ __attribute__((aligned(16))) T s_v[2][D * BN];
    __shared__ int s_bad[2];

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
            mine += (uint32_t)(((int64_t)w.n * a.group + PR_ROWS - 1) / PR_ROWS);
        }
    }
    if (blockIdx.x == 0 && bad_rows) raise(a.flags, MOE_DEVFLAG_BAD_SEQ);
    const uint32_t incl = wave_scan(mine);
    const uint32_t total = (uint32_t)__builtin_amdgcn_readlane((int)incl, 63);
    const uint32_t nth = blockIdx.x / a.hkv;
    if (nth >= total) return;
    const int hk = blockIdx.x - nth * a.hkv;
    const uint32_t want = total - 1 - nth;
    const int owner = __builtin_ctzll(__ballot(incl > want));
    uint32_t at = (uint32_t)__builtin_amdgcn_readlane((int)(incl - mine), owner);
    int b = owner * per;
    Rows sr;
    for (;; ++b) {
        sr = seq_rows(a, uniform(b));
        const uint32_t n = (uint32_t)(((int64_t)sr.n * a.group + PR_ROWS - 1) / PR_ROWS);
        if (want < at + n) break;
        at += n;
    }
    b = uniform(b);
    sr.r0 = uniform(sr.r0);
    sr.n = uniform(sr.n);
    if (tid < 2) s_bad[tid] = 0;

    // ---- rows: number f of the sequence's (token, head) pairs, position
    const int64_t f0 = (int64_t)(want - at) * PR_ROWS, nf = (int64_t)sr.n * a.group;
    const int len = ldc(a.kv_len + b);
    if ((len < 0 || len > cap) && tid == 0) raise(a.flags, MOE_DEVFLAG_BAD_SEQ);
    const int64_t first_pos = (int64_t)len - ldc(a.row_start + b + 1) + sr.r0; // of the sequence's first row
    auto seen_by = [&](int64_t f) { // tokens that pair f's row sees
        const int64_t p = first_pos + f / a.group + 1;
        return (int)(p < 0 ? 0 : p > cap ? cap : p);
    };
    const int64_t f = f0 + wave * 32 + r;
    const bool mine_valid = f < nf;
    const int tok = (int)((mine_valid ? f : nf - 1) / a.group);
    const int head = hk * a.group + (int)((mine_valid ? f : nf - 1) - (int64_t)tok * a.group);
    const int row = sr.r0 + tok;
    const int seen = mine_valid ? seen_by(f) : 0;
    const int64_t f_last = f0 + PR_ROWS < nf ? f0 + PR_ROWS : nf;
    const int ext = uniform(seen_by(f_last - 1));  // tokens that some row of the workgroup sees
    const int full = uniform(seen_by(f0));         // ... that all see
    const int64_t wf = f0 + wave * 32 + 32;
    const int wave_ext = f0 + wave * 32 < nf ? uniform(seen_by((wf < nf ? wf : nf) - 1)) : 0;

    x8 qf[KS];
    {
        const T *q = (const T *)a.q + row * a.q_stride + head * D + h * 8;
        const uint32_t flip = a.scale_log2 < 0.f ? 0x80008000u : 0u; // a negative scale: -q, exactly
#pragma unroll
        for (int k = 0; k < KS; ++k) {
            u32x4 w = ldg<u32x4>(q + k * 16);
            for (int i = 0; i < 4; ++i) w[i] ^= flip;
            qf[k] = __builtin_bit_cast(x8, w);
        }
    }
    // Scale 0: the smallest normal number, so that -inf (not seen) stays -inf; any finite score times it
    // is 0 beside the exponential's 1.
    const float scale = fmaxf(fabsf(a.scale_log2), 1.17549435e-38f);

    // ---- tiles
    const int32_t *pages = a.pages + b * a.pages_stride;
    const uint8_t *kb = a.k + 2 * hk * a.head_stride, *vb = a.v + 2 * hk * a.head_stride;
    const int ts2 = (int)(2 * a.token_stride), mask = (1 << a.page_shift) - 1;
    bool bad_page = false;
    int64_t off[NB]; // of the staged tile: a block's first token, and how many tokens it has
    int have[NB];
    auto place = [&](int t) {
#pragma unroll
        for (int i = 0; i < NB; ++i) {
            const int key = t * BN + 16 * i;
            int pg = 0;
            have[i] = min(16, max(0, ext - key));
            if (have[i] > 0) {
                pg = ldc(pages + (key >> a.page_shift));
                if ((unsigned)pg >= (unsigned)a.n_pages) bad_page = true, pg = 0, have[i] = 0;
            }
            off[i] = 2 * (pg * a.page_stride + (key & mask) * a.token_stride);
        }
    };
    u32x4 kr[BN / RP];
    vload vr[8];
    const int vblk = wave; // this wave's V block of 16 tokens: its lanes r hold VW elements of half of them
    auto load = [&]() {
#pragma unroll
        for (int p = 0; p < BN / RP; ++p) {
            const int key = p * RP + tid / (D / 8);
            const int i = D == 64 ? 2 * p + (wave >> 1) : p * RP / 16;
            const int t = max(0, min(key & 15, have[i] - 1));
            kr[p] = ldo<u32x4>(kb + off[i], (uint32_t)(t * ts2 + tid % (D / 8) * 16));
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int t = max(0, min(8 * (j >> 2) + 4 * h + (j & 3), have[vblk] - 1));
            vr[j] = ldo<vload>(vb + off[vblk], (uint32_t)(t * ts2 + r * (VW * 2)));
        }
    };
    // A value that a row does not see meets a weight of 0, which an infinity or NaN would survive: those
    // in tiles that some row does not see all of are noted (s_bad), those that none sees are 0.
    auto store = [&](int t, int buf) {
        if (have[vblk] < 16)
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (8 * (j >> 2) + 4 * h + (j & 3) >= have[vblk]) vr[j] = vload{};
        if ((t + 1) * BN > full) {
            bool bad = false;
#pragma unroll
            for (int j = 0; j < 8; ++j)
#pragma unroll
                for (int w = 0; w < VW / 2; ++w) bad |= not_finite<T>(vr[j][w]);
            if (bad) s_bad[buf] = t + 1;
        }
        uint8_t *lk = (uint8_t *)s_k[buf], *lv = (uint8_t *)s_v[buf];
#pragma unroll
        for (int p = 0; p < BN / RP; ++p) {
            const int key = p * RP + tid / (D / 8), ch = tid % (D / 8);
            *(u32x4 *)(lk + key * (D * 2) + ((ch ^ (key & 7)) * 16)) = kr[p];
        }
#pragma unroll
        for (int w = 0; w < VW / 2; ++w)
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                u32x4 e;
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    e[i] = __builtin_amdgcn_perm(vr[2 * i + 1][w], vr[2 * i][w], x ? 0x07060302u : 0x05040100u);
                const int d = r * VW + 2 * w + x;
                *(u32x4 *)(lv + d * (BN * 2) + (((2 * vblk + h) ^ ((d ^ (d >> 3)) & 7)) * 16)) = e;
            }
    };

    f32x16 o[D / 32];
#pragma unroll
    for (int i = 0; i < D / 32; ++i) o[i] = f32x16{};
    float m = -INFINITY, l = 0.f; // the maximum that weights are taken against, and this lane's sum
    uint32_t ko[4], vo[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        ko[i] = r * (D * 2) + (((2 * i + h) ^ (r & 7)) * 16);
        vo[i] = r * (BN * 2) + (((2 * i + h) ^ ((r ^ (r >> 3)) & 7)) * 16);
    }

    const int nt = (ext + BN - 1) / BN;
    if (nt > 0) {
        place(0);
        load();
        __syncthreads(); // s_bad
        store(0, 0);
        __syncthreads();
    }
    for (int t = 0; t < nt; ++t) {
        const int buf = t & 1;
        int hv[NB];
        bool part = (t + 1) * BN > full;
#pragma unroll
        for (int i = 0; i < NB; ++i) {
            hv[i] = have[i];
            part |= hv[i] < 16;
        }
        if (t + 1 < nt) {
            place(t + 1);
            load();
        }
        const bool slow = part && *(volatile int *)&s_bad[buf] == t + 1;
        const bool active = t * BN < wave_ext;
        u32x4 pw[4]; // the weights, in P^T's operand layout
        if (active) {
            f32x16 s[2];
            const uint8_t *lk = (const uint8_t *)s_k[buf], *lv = (const uint8_t *)s_v[buf];
#pragma unroll
            for (int k = 0; k < KS; ++k)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const x8 kf = *(const x8 *)(lk + ko[k & 3] + i * (32 * D * 2) + (k >> 2) * 128);
                    s[i] = E::mfma32(kf, qf[k], k ? s[i] : f32x16{});
                }
            if (part)
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int j = 0; j < 16; ++j) {
                        const int key = 32 * i + 8 * (j >> 2) + 4 * h + (j & 3);
                        if (t * BN + key >= seen || (key & 15) >= hv[2 * i + (j >> 3)]) s[i][j] = -INFINITY;
                    }
            float mx = s[0][0];
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int j = 0; j < 16; ++j) mx = fmaxf(mx, s[i][j]);
            mx = fmaxf(mx, __shfl_xor(mx, 32)) * scale;
            if (__any(mx > m + LAZY)) {
                const float mn = fmaxf(m, mx);
                const float alpha = exp2_(m - base_of(mn));
                m = mn;
                l *= alpha;
#pragma unroll
                for (int i = 0; i < D / 32; ++i) o[i] *= alpha;
            }
            const float base = base_of(m) - SHIFT;
            float sum = 0.f;
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int j = 0; j < 16; j += 2) {
                    const float p0 = exp2_(__builtin_fmaf(s[i][j], scale, -base));
                    const float p1 = exp2_(__builtin_fmaf(s[i][j + 1], scale, -base));
                    sum += p0 + p1;
                    pw[2 * i + (j >> 3)][(j & 7) >> 1] = E::pack(p0, p1);
                }
            l += sum;
            if (!slow)
#pragma unroll
                for (int k = 0; k < 4; ++k)
#pragma unroll
                    for (int i = 0; i < D / 32; ++i) {
                        const x8 vf = *(const x8 *)(lv + vo[i & 1 ? k ^ 2 : k] + i * (32 * BN * 2));
                        o[i] = E::mfma32(vf, __builtin_bit_cast(x8, pw[k]), o[i]);
                    }
        }
        if (slow) { // token by token, each only where it is seen
            __syncthreads(); // K of both buffers is free
            T *sp = &s_k[0][0] + (wave * 32 + r) * BN;
            if (active) {
#pragma unroll
                for (int k = 0; k < 4; ++k)
#pragma unroll
                    for (int i = 0; i < 4; ++i) // tokens 16 k + 8 (i / 2) + 4 h + 2 (i % 2) and the next
                        *(uint32_t *)(sp + 16 * k + 8 * (i >> 1) + 4 * h + 2 * (i & 1)) = pw[k][i];
                lds_fence();
                const uint8_t *lv = (const uint8_t *)s_v[buf];
#pragma unroll 1
                for (int key = 0; key < BN; ++key) {
                    const int in = key & 15;
                    const int ch = 2 * (key >> 4) + ((in >> 2) & 1), el = 4 * (in >> 3) + (in & 3);
                    const bool sees = t * BN + key < seen;
                    const float p = (float)sp[key];
#pragma unroll
                    for (int i = 0; i < D / 32; ++i)
#pragma unroll
                        for (int j = 0; j < 16; ++j) {
                            const int d = 32 * i + 8 * (j >> 2) + 4 * h + (j & 3);
                            const T v = *(const T *)(lv + d * (BN * 2) + ((ch ^ ((d ^ (d >> 3)) & 7)) * 16) + el * 2);
                            if (sees) o[i][j] += p * (float)v;
                        }
                }
            }
            __syncthreads();
        }
        if (t + 1 < nt) store(t + 1, buf ^ 1);
        __syncthreads();
    }
    if (bad_page && lane == 0) raise(a.flags, MOE_DEVFLAG_BAD_PAGE);

    // ---- rows out
    l += __shfl_xor(l, 32);
    if (!mine_valid) return;
    const float inv = l == 0.f ? 0.f : 1.f / l;
    T *op = (T *)a.o + row * a.o_stride + head * D + 4 * h;
#pragma unroll
    for (int i = 0; i < D / 32; ++i)
#pragma unroll
        for (int j = 0; j < 16; j += 4) {
            u32x2 w = {E::pack(o[i][j] * inv, o[i][j + 1] * inv), E::pack(o[i][j + 2] * inv, o[i][j + 3] * inv)};
            if (l == 0.f) w = u32x2{0u, 0u};
            *(u32x2 *)(op + 32 * i + 2 * j) = w;
        }
    if (a.lse && h == 0)
        a.lse[(int64_t)row * a.hq + head] =
            l == 0.f ? -INFINITY : (base_of(m) - SHIFT + __log2f(l)) * 0.69314718055994531f;
}

template <typename T>
hipError_t prompt_t(const AttnArgs &a, int d, hipStream_t st) {
    // tiles of the rows however they are divided: each sequence's last one may be short
    const int64_t tiles = (int64_t)a.n_rows * a.group / PR_ROWS + a.n_seqs;
    const unsigned grid = (unsigned)(tiles * a.hkv);
    if (d == 64) k_attn_prompt<T, 64><<<grid, 256, 0, st>>>(a);
    else if (d == 128) k_attn_prompt<T, 128><<<grid, 256, 0, st>>>(a);
    else k_attn_prompt<T, 256><<<grid, 256, 0, st>>>(a);
    return hipGetLastError();
}

} // namespace

hipError_t launch_attn_prompt(const AttnArgs &a, int type, int d, hipStream_t st) {
    return type == MOE_T_F16 ? prompt_t<f16_t>(a, d, st) : prompt_t<bf16_t>(a, d, st);
}

} // namespace moe
