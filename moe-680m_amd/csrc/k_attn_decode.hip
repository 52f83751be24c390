// k_attn_decode.hip -- one new token of every sequence over its paged cache.
//
//   o[h] = sum_j e^(s_j - m) V_j / sum_j e^(s_j - m),   s_j = scale * q[h] . K_j
//
// Bound by reading K and V once (4 bytes of K and V for 4 * group operations a head element, far
// below the matrix rate), so all that matters is to keep every CU's loads in flight:
//
//   * A unit is one (sequence, key-value head, up to 16 of its query heads), a step of it
//     DEC_STEP tokens, 32 for each wave of a workgroup.
//   * Work is cut by the lengths as they are in device memory, not by the host's bound: the units'
//     steps are numbered through and each of the n_wg resident workgroups takes an equal run of
//     them.  A run that ends inside a unit leaves partial rows (maximum, sum, unnormalised
//     output), which a second launch joins in their order (same bits every time).
//   * A wave works by itself, no barrier until the run leaves the unit:
//       S^T[token][head] = K Q^T       16x16x32 products, A rows = tokens straight from memory
//                                      (a lane's 16 bytes = 8 elements of one token)
//       O^T[d][head] += V^T P^T        B = P^T is S^T's own register layout: lane (head, g) holds
//                                      tokens 4g..4g+3 and 16+4g..16+4g+3, and V's tokens are taken in
//                                      that order, so P never moves between lanes
//     V^T: a lane loads 8 tokens x 8 consecutive elements (whole rows are contiguous over 16
//     lanes) and swaps them in registers, two v_perm a dword pair; the matrix row m of product j
//     is element 8 m + j, which only the output's addressing sees.
//   * A wave's loads of the next 32 tokens' K are issued before the softmax, those of V after the
//     products.
// 64 sequences of 202 to 16384 tokens, 16/2 heads of 256: 90 us, 4.9 TB/s of K and V; one of 128k tokens 57 us,
// 4.7 TB/s (this launch alone 5.3 TB/s; a kernel that only reads reaches 6.1).  256 sequences of 1 to 2048, 32/8 heads of
// 128: 66 us, 4.1 TB/s.  One of 512 tokens: 11 us, two launches and the chain lengths -> pages -> K -> V.
// The same kernel with one workgroup a unit and no cut: 128k tokens 102 ms, 64 sequences 12.6 ms.
#include "attn_device.hpp"

namespace moe {

namespace {

constexpr int DEC_STEP = DEC_WAVES * DEC_WAVE_TOK;

// Steps of a sequence's units: one at least, so that an empty one's rows are written too.
__device__ __forceinline__ int steps(int len, int cap) {
    return max(1, (min(max(len, 0), cap) + DEC_STEP - 1) / DEC_STEP);
}

// A partial row's maximum and sum: those of a row place lie together, so that a wave loads many
// pieces' at once.
template <typename Args>
__device__ __forceinline__ size_t ml_at(const Args &a, int place, size_t slot) {
    return (size_t)place * (4 * a.n_wg) + 2 * slot;
}

template <typename T, int D>
__global__ __launch_bounds__(256, 2) void k_attn_decode(AttnArgs a) {
    typedef Elem<T> E;
    typedef typename E::x8 x8;
    constexpr int KS = D / 32;               // products of a score tile
    constexpr int VW = D >= 128 ? 8 : 4;     // elements of a lane's V load
    constexpr int VS = D / (16 * VW);        // loads a token
    typedef uint32_t vload __attribute__((ext_vector_type(VW / 2)));
    // the waves' rows, 4 floats apart so that 16 lanes' rows start in different banks
    __shared__ float s_o[DEC_WAVES][DEC_HEADS][D + 4];
    __shared__ f32x2 s_ml[DEC_WAVES][DEC_HEADS];

    const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6);
    const int c = lane & 15, g = lane >> 4;
    const int cap = a.max_pages << a.page_shift;
    const int gb = (a.group + DEC_HEADS - 1) / DEC_HEADS; // head blocks of a key-value head
    const int ng = a.hkv * gb;                            // units of a sequence

    // ---- this workgroup's run of steps [lo, hi): every wave has the sequences' steps and finds the sequence
    // that lo lies in
    auto steps_of = [&](int b) {
        const int n = steps(ldg<int>(a.kv_len + min(b, a.n_seqs - 1)), cap);
        return b < a.n_seqs ? (uint32_t)n : 0u;
    };
    uint32_t mine, incl;
    count_seqs(a.n_seqs, lane, wave, steps_of, mine, incl);
    const uint32_t total = (uint32_t)__builtin_amdgcn_readlane((int)incl, 63) * ng;
    const uint32_t share = (total + gridDim.x - 1) / gridDim.x;
    const uint32_t lo = blockIdx.x * share;
    // For the join: of every unit the pieces it was cut into, or (more units than workgroups) of every
    // workgroup those of the unit that it begins and others go on with.
    const bool by_unit = (int64_t)a.n_seqs * ng <= a.n_wg;
    Piece tail = {0, 0, 0, 0};
    if (lo >= total) {
        if (!by_unit && tid == 0) a.piece[blockIdx.x] = tail;
        return;
    }
    const uint32_t hi = min(lo + share, total);
    uint32_t at; // steps before b, of one unit each
    int from, b = find_seq(a.n_seqs, lane, steps_of, mine, incl, lo / ng, at, from);
    int nt = steps(ldc(a.kv_len + b), cap);
    // (a head block or sequence out of range, here and below: the lengths changed during the call)
    int hb = min((int)((lo - at * ng) / (uint32_t)nt), ng - 1);
    uint32_t unit = at * ng + hb * nt; // first step of unit (b, hb)

    // a unit's first query head and heads
    auto head0 = [&](int hb) { return hb / gb * a.group + hb % gb * DEC_HEADS; };
    auto heads = [&](int hb) { return min(DEC_HEADS, a.group - hb % gb * DEC_HEADS); };

    const int ts2 = (int)(2 * a.token_stride), mask = (1 << a.page_shift) - 1;
    bool bad = false;
    for (uint32_t pos = lo;;) {
        // ---- the unit at work: steps t0..t1 of it
        const int t0 = (int)(pos - unit), t1 = (int)(min(hi, unit + nt) - unit);
        const int len = ldc(a.kv_len + b), seen = min(max(len, 0), cap);
        if (seen != len && tid == 0) raise(a.flags, MOE_DEVFLAG_BAD_SEQ);
        const int end = min(seen, t1 * DEC_STEP); // of the tokens
        const int hk = hb / gb, nh = heads(hb);
        const int32_t *pages = a.pages + b * a.pages_stride;
        const uint8_t *kb = a.k + 2 * hk * a.head_stride, *vb = a.v + 2 * hk * a.head_stride;
        const T *q = (const T *)a.q + b * a.q_stride + (int64_t)(head0(hb) + min(c, nh - 1)) * D;
        x8 qf[KS], kf[2][KS];
        vload vf[8][VS];
#pragma unroll
        for (int k = 0; k < KS; ++k) qf[k] = ldg<x8>(q + k * 32 + g * 8);
        int64_t off[2]; // the two 16-token halves of a step: byte offset of the first token, tokens there
        int have[2];
        auto place = [&](int tok) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int t = tok + 16 * i;
                have[i] = min(16, end - t);
                int pg = 0;
                if (have[i] > 0) {
                    pg = ldc(pages + (t >> a.page_shift));
                    if ((unsigned)pg >= (unsigned)a.n_pages) bad = true, pg = 0, have[i] = 0;
                } else have[i] = 0;
                off[i] = 2 * (pg * a.page_stride + (t & mask) * a.token_stride);
            }
        };
        // a lane whose token is not there reads the last one that is (the first place if none is)
        auto lane_off = [&](int t, int i, int byte) {
            if (have[i] < 16) t = max(0, min(t, have[i] - 1));
            return (uint32_t)(t * ts2 + byte);
        };
        auto load_k = [&]() {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const uint32_t lo = lane_off(c, i, g * 16);
#pragma unroll
                for (int k = 0; k < KS; ++k) kf[i][k] = ldo<x8>(kb + off[i], lo, k * 64);
            }
        };
        auto load_v = [&]() {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const uint32_t lo = lane_off(4 * g + (j & 3), j >> 2, c * (VW * 2));
#pragma unroll
                for (int s = 0; s < VS; ++s) vf[j][s] = ldo<vload>(vb + off[j >> 2], lo, s * (32 * VW));
            }
        };
        int tok = t0 * DEC_STEP + wave * DEC_WAVE_TOK;
        if (tok < end) {
            place(tok);
            load_k();
            load_v();
        }
        // The queries' fragments stay in registers; at D = 256, where those are short, in the wave's own
        // part of s_o, every lane reading back what it wrote.
        x8 *const ql = (x8 *)&s_o[wave][0][0] + lane;
        if (D == 256)
#pragma unroll
            for (int k = 0; k < KS; ++k) ql[64 * k] = qf[k];
        f32x4 acc[D / 16];
#pragma unroll
        for (int i = 0; i < D / 16; ++i) acc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
        float m = -INFINITY, l = 0.f;
        for (; tok < end; tok += DEC_STEP) {
            const int hv[2] = {have[0], have[1]};
            f32x4 st[2];
#pragma unroll
            for (int k = 0; k < KS; ++k) {
                const x8 qk = D == 256 ? ql[64 * k] : qf[k];
                if (D == 256 && k % 2 == 0) __builtin_amdgcn_sched_barrier(0); // not all of them at once
#pragma unroll
                for (int i = 0; i < 2; ++i)
                    st[i] = E::mfma16(kf[i][k], qk, k ? st[i] : f32x4{0.f, 0.f, 0.f, 0.f});
            }
            const bool more = tok + DEC_STEP < end;
            if (more) {
                place(tok + DEC_STEP);
                load_k();
            }
            float mx = m;
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    st[i][r] = 4 * g + r < hv[i] ? st[i][r] * a.scale_log2 : -INFINITY;
                    mx = fmaxf(mx, st[i][r]);
                }
            mx = fmaxf(mx, __shfl_xor(mx, 16));
            mx = fmaxf(mx, __shfl_xor(mx, 32));
            const float mb = base_of(mx);
            const float alpha = exp2_(m - mb);
            m = mx;
            float p[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) p[i] = exp2_(st[i >> 2][i & 3] - (mb - E::SHIFT));
            l = l * alpha + (((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7])));
            const u32x4 pw = {E::pack(p[0], p[1]), E::pack(p[2], p[3]), E::pack(p[4], p[5]), E::pack(p[6], p[7])};
            const x8 pf = __builtin_bit_cast(x8, pw);
#pragma unroll
            for (int i = 0; i < D / 16; ++i) acc[i] *= alpha;
            if (hv[0] < 16 || hv[1] < 16) { // values that are not seen: 0 (0 * inf would be NaN)
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (4 * g + (j & 3) >= hv[j >> 2])
#pragma unroll
                        for (int s = 0; s < VS; ++s) vf[j][s] = vload{};
            }
#pragma unroll
            for (int s = 0; s < VS; ++s)
#pragma unroll
                for (int w = 0; w < VW / 2; ++w) {
                    u32x4 e0, e1;
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        e0[i] = __builtin_amdgcn_perm(vf[2 * i + 1][s][w], vf[2 * i][s][w], 0x05040100u);
                        e1[i] = __builtin_amdgcn_perm(vf[2 * i + 1][s][w], vf[2 * i][s][w], 0x07060302u);
                    }
                    f32x4 &a0 = acc[s * VW + 2 * w], &a1 = acc[s * VW + 2 * w + 1];
                    a0 = E::mfma16(__builtin_bit_cast(x8, e0), pf, a0);
                    a1 = E::mfma16(__builtin_bit_cast(x8, e1), pf, a1);
                }
            if (more) load_v();
        }

        // ---- join the four waves: row (head c) of O^T's register layout to s_o[wave][head][d]
        l += __shfl_xor(l, 16);
        l += __shfl_xor(l, 32);
        if (g == 0) s_ml[wave][c] = f32x2{m, l};
        // the row's elements 16 VW s + VW (4 g + r) + j, j = 0..VW-1
#pragma unroll
        for (int s = 0; s < VS; ++s)
#pragma unroll
            for (int r = 0; r < 4; ++r)
#pragma unroll
                for (int j = 0; j < VW; j += 4)
                    *(f32x4 *)&s_o[wave][c][16 * VW * s + VW * (4 * g + r) + j] =
                        f32x4{acc[s * VW + j][r], acc[s * VW + j + 1][r], acc[s * VW + j + 2][r], acc[s * VW + j + 3][r]};
        const bool begins = t0 == 0, whole = begins && t1 == nt;
        const Piece pc = {b, hb, (int)blockIdx.x, (int)((unit + nt - 1) / share - blockIdx.x + 1)};
        lds_barrier();
        // Partial rows: slot 0 of a workgroup holds the piece of a unit that began before it, slot 1 that
        // of one which goes on behind it.
        const size_t slot = 2 * (size_t)blockIdx.x + (begins ? 1 : 0);
        int et = tid; // opaque, so that no item's index is computed before the loop and held through it
        asm volatile("" : "+v"(et));
        {
            const auto &a = fresh_args();
            for (int i = et; i < nh * (D / 4); i += 256) {
                const int hh = i / (D / 4), d = i % (D / 4) * 4;
                f32x2 ml[DEC_WAVES];
                f32x4 y[DEC_WAVES], x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int w = 0; w < DEC_WAVES; ++w) {
                    ml[w] = s_ml[w][hh];
                    y[w] = *(const f32x4 *)&s_o[w][hh][d];
                }
                float M = -INFINITY, L = 0.f;
#pragma unroll
                for (int w = 0; w < DEC_WAVES; ++w) M = fmaxf(M, ml[w].x);
#pragma unroll
                for (int w = 0; w < DEC_WAVES; ++w) {
                    const float f = exp2_(ml[w].x - base_of(M));
                    L += f * ml[w].y;
                    x += f * y[w];
                }
                if (whole) put_row<T>(a, b, head0(hb) + hh, D, d, x, M, L, E::SHIFT);
                else {
                    *(f32x4 *)(a.part + (slot * DEC_HEADS + hh) * D + d) = x;
                    if (d == 0) *(f32x2 *)(a.part_ml + ml_at(a, hh, slot)) = f32x2{M, L};
                }
            }
            if (begins) {
                if (by_unit) {
                    if (tid == 0) a.piece[b * ng + hb] = pc;
                } else if (!whole) tail = pc;
            }
        }
        pos = unit + t1;
        if (pos >= hi) break;
        lds_barrier(); // s_o is free again
        unit += nt; // the next unit
        if (++hb == ng) {
            hb = 0;
            if (++b >= a.n_seqs) break;
            nt = steps(ldc(a.kv_len + b), cap);
        }
    }
    if (bad && lane == 0) raise(a.flags, MOE_DEVFLAG_BAD_PAGE);
    if (!by_unit && tid == 0) a.piece[blockIdx.x] = tail;
}

// The partial rows of a unit that several runs share: out = sum_p f_p x_p / sum_p f_p l_p,
// f_p = 2^(m_p - max m), in the pieces' order.  Up to JOIN_FEW pieces: a thread takes four elements of a
// row through all of them.  More: a row at a time, a thread four elements of every PG-th piece, JOIN_B of
// them under way.
constexpr int JOIN_FEW = 16, JOIN_B = 16;
template <typename T, int D, int W, int THREADS>
__global__ __launch_bounds__(THREADS) void k_attn_join(AttnArgs a, int rows_per_wg) {
    constexpr int TPR = W / 4, PG = THREADS / TPR; // W elements of a row, gridDim.z times
    const int d0 = (int)blockIdx.z * W;
    __shared__ float s_f[DEC_MAX_WG];
    __shared__ f32x4 s_x[PG][TPR];
    const Piece pc = {ldc(&a.piece[blockIdx.x].b), ldc(&a.piece[blockIdx.x].hb), ldc(&a.piece[blockIdx.x].w0),
                      ldc(&a.piece[blockIdx.x].n)};
    const int n = pc.n;
    if (n < 2 || pc.b >= a.n_seqs) return; // (an earlier call's: the lengths changed during this one)
    const int tid = threadIdx.x, lane = tid & 63;
    const int gb = (a.group + DEC_HEADS - 1) / DEC_HEADS;
    const int h0 = pc.hb / gb * a.group + pc.hb % gb * DEC_HEADS; // the unit's first query head, and its heads
    const int nh = min(DEC_HEADS, a.group - pc.hb % gb * DEC_HEADS);
    const int r0 = blockIdx.y * rows_per_wg, r1 = min(nh, r0 + rows_per_wg);
    // row r of piece p: of the first workgroup the later slot, of the others the earlier one
    auto slot = [&](int p) { return 2 * (size_t)(pc.w0 + p) + (p == 0 ? 1 : 0); };
    auto row = [&](int r, int p) { return slot(p) * DEC_HEADS + r; };
    if (n <= JOIN_FEW) {
        for (int i = r0 * TPR + tid; i < r1 * TPR; i += THREADS) {
            const int r = i / TPR, d = d0 + i % TPR * 4;
            f32x2 ml[JOIN_FEW];
            f32x4 v[JOIN_FEW];
#pragma unroll
            for (int p = 0; p < JOIN_FEW; ++p) {
                ml[p] = p < n ? ldg<f32x2>(a.part_ml + ml_at(a, r, slot(p))) : f32x2{-INFINITY, 0.f};
                v[p] = p < n ? ldg<f32x4>(a.part + row(r, p) * D + d) : f32x4{};
            }
            float M = -INFINITY, L = 0.f;
#pragma unroll
            for (int p = 0; p < JOIN_FEW; ++p) M = fmaxf(M, ml[p].x);
            f32x4 x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int p = 0; p < JOIN_FEW; ++p) {
                const float f = exp2_(ml[p].x - base_of(M));
                L += f * ml[p].y;
                x += f * v[p];
            }
            put_row<T>(a, pc.b, h0 + r, D, d, x, M, L, Elem<T>::SHIFT);
        }
        return;
    }
    const int pg = tid / TPR, d = d0 + tid % TPR * 4;
    for (int r = r0; r < r1; ++r) {
        f32x4 v[JOIN_B];
        auto load = [&](int p) {
#pragma unroll
            for (int j = 0; j < JOIN_B; ++j)
                v[j] = p + j * PG < n ? ldg<f32x4>(a.part + row(r, p + j * PG) * D + d) : f32x4{};
        };
        load(pg);
        float M = -INFINITY, L = 0.f;
        for (int p = lane; p < n; p += 64) M = fmaxf(M, ldg<f32x2>(a.part_ml + ml_at(a, r, slot(p))).x);
        M = wave_max(M);
        for (int p = lane; p < n; p += 64) {
            const f32x2 ml = ldg<f32x2>(a.part_ml + ml_at(a, r, slot(p)));
            const float f = exp2_(ml.x - base_of(M));
            L += f * ml.y;
            if (tid < 64) s_f[p] = f;
        }
        L = wave_sum(L);
        lds_barrier();
        f32x4 x = {0.f, 0.f, 0.f, 0.f};
        for (int p = pg;;) {
#pragma unroll
            for (int j = 0; j < JOIN_B; ++j)
                if (p + j * PG < n) x += s_f[p + j * PG] * v[j];
            if ((p += JOIN_B * PG) >= n) break;
            load(p);
        }
        s_x[pg][tid % TPR] = x;
        lds_barrier();
        if (pg == 0) {
            for (int i = 1; i < PG; ++i) x += s_x[i][tid];
            put_row<T>(a, pc.b, h0 + r, D, d, x, M, L, Elem<T>::SHIFT);
        }
        lds_barrier(); // s_f and s_x are free again
    }
}

template <typename T, int D>
hipError_t decode_d(const AttnArgs &a, hipStream_t st) {
    k_attn_decode<T, D><<<a.n_wg, 256, 0, st>>>(a);
    // Few units, so possibly many pieces each: one row a workgroup, or 64 elements of it where the page lists
    // hold more than 64 steps.  (One sequence of 128k tokens, 16/2 heads of 256: 58.8 us by rows, 56.7 by 64
    // elements with the decode; of 512 tokens 10.7 and 10.9; 256 sequences, as many slices as 4096, 66 and 69.)
    // Many units, so a few pieces of each mostly: the rows that 256 threads hold.
    const int gb = (a.group + DEC_HEADS - 1) / DEC_HEADS, rows = a.group < DEC_HEADS ? a.group : DEC_HEADS;
    const int64_t units = (int64_t)a.n_seqs * a.hkv * gb;
    const int x = units <= a.n_wg ? (int)units : a.n_wg, per = 1024 / D;
    const bool longer = (int64_t)a.max_pages << a.page_shift > 64 * DEC_STEP;
    if (longer && x * rows * (D / 64) <= 256) k_attn_join<T, D, 64, 256><<<dim3(x, rows, D / 64), 256, 0, st>>>(a, 1);
    else if (x * rows <= 512) k_attn_join<T, D, D, 512><<<dim3(x, rows), 512, 0, st>>>(a, 1);
    else if (x * rows <= 2048) k_attn_join<T, D, D, 256><<<dim3(x, rows), 256, 0, st>>>(a, 1);
    else k_attn_join<T, D, D, 256><<<dim3(x, (rows + per - 1) / per), 256, 0, st>>>(a, per);
    return hipGetLastError();
}

template <typename T>
hipError_t decode_t(const AttnArgs &a, int d, hipStream_t st) {
    return d == 64 ? decode_d<T, 64>(a, st) : d == 128 ? decode_d<T, 128>(a, st) : decode_d<T, 256>(a, st);
}

} // namespace

hipError_t launch_attn_decode(const AttnArgs &a, int type, int d, hipStream_t st) {
    return type == MOE_T_F16 ? decode_t<f16_t>(a, d, st) : decode_t<bf16_t>(a, d, st);
}

} // namespace moe
