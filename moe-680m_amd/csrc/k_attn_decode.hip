// k_attn_decode.hip -- one new token of every sequence over its paged cache.
//
//   o[h] = sum_j e^(s_j - m) V_j / sum_j e^(s_j - m),   s_j = scale * q[h] . K_j
//
// Bound by reading K and V once (4 bytes of K and V for 4 * group operations a head element, far
// below the matrix rate), so all that matters is to keep every CU's loads in flight:
//
//   * A unit is one (sequence, key-value head, up to 16 of its query heads).  Each wave of a
//     workgroup takes 32 tokens of a unit at a step; `wpu` waves share a unit, so a workgroup has
//     U = 4 / wpu units of one sequence at work (a group).  wpu = 4 splits a unit the widest;
//     wpu = 1 leaves nothing to join between waves and has the longest runs.
//   * Work is cut by the lengths as they are in device memory, not by the host's bound: the groups'
//     steps are numbered through and each of the n_wg resident workgroups takes an equal run of
//     them.  A run that ends inside a group leaves partial rows (maximum, sum, unnormalised
//     output).  They are joined inside the launch, in their order (same bits every time): of each
//     16 consecutive workgroups the last one to arrive joins theirs, of those the last one all.
//   * A wave works by itself, no barrier until the run leaves the group:
//       S^T[token][head] = K Q^T       16x16x32 products, A rows = tokens straight from memory
//                                      (a lane's 16 bytes = 8 elements of one token)
//       O^T[d][head] += V^T P^T        B = P^T is S^T's own register layout: lane (head, g) holds
//                                      tokens 4g..4g+3 and 16+4g..16+4g+3, and V's tokens are taken in
//                                      that order, so P never moves between lanes
//     V^T: a lane loads 8 tokens x 8 consecutive elements (whole rows are contiguous over 16
//     lanes) and swaps them in registers, two v_perm a dword pair; the matrix row m of product j
//     is element 8 m + j, which only the output's addressing sees.
//   * A wave's loads of the next 32 tokens' K are issued before the softmax, those of V after the
//     products: some 16 KB a wave are always under way.
#include "attn_device.hpp"

namespace moe {

namespace {

constexpr int JOIN = 16; // workgroups whose partial rows one workgroup joins
constexpr int JOIN_MAX = 64; // pieces of one join: JOIN, or the groups of JOIN of a launch
static_assert(DEC_MAX_WG <= JOIN * JOIN_MAX, "two levels join all");

// Steps of a sequence's group: one at least, so that an empty one's rows are written too.
__device__ __forceinline__ int seq_steps(const AttnArgs &a, int b, int cap, int shift) {
    const int n = min(max(a.kv_len[b], 0), cap);
    return max(1, (n + (1 << shift) - 1) >> shift);
}

template <typename T, int D>
__global__ __launch_bounds__(256, 2) void k_attn_decode(AttnArgs a) {
    typedef Elem<T> E;
    typedef typename E::x8 x8;
    constexpr int KS = D / 32;               // products of a score tile
    constexpr int VW = D >= 128 ? 8 : 4;     // elements of a lane's V load
    constexpr int VS = D / (16 * VW);        // loads a token
    typedef uint32_t vload __attribute__((ext_vector_type(VW / 2)));
    // the waves' rows; in a join the pieces' maxima and sums, then their factors
    __shared__ float s_o[DEC_WAVES][DEC_HEADS][D];
    __shared__ float s_ml[DEC_WAVES][DEC_HEADS][2];
    __shared__ uint32_t s_scan[DEC_WAVES], s_find[2];
    __shared__ uint32_t s_last;
    static_assert(sizeof s_o >= JOIN_MAX * DEC_WAVES * DEC_HEADS * 4, "a join's factors");

    const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6);
    const int c = lane & 15, g = lane >> 4;
    const int cap = a.max_pages << a.page_shift;
    const int gb = (a.group + DEC_HEADS - 1) / DEC_HEADS; // head blocks of a key-value head
    const int wpu = 1 << a.wpu_shift, U = DEC_WAVES >> a.wpu_shift;
    const int shift = 5 + a.wpu_shift;                    // log2 of a step's tokens
    const int ng = a.hkv * gb / U;                        // groups of a sequence
    const int sub = wave >> a.wpu_shift, wsub = wave & (wpu - 1);
    const int rows = min(DEC_HEADS, a.group);             // row places of a unit

    // ---- this workgroup's run of steps [lo, hi): prefix sums over the sequences
    const int per = (a.n_seqs + 255) / 256;
    uint32_t mine = 0;
    for (int i = 0; i < per; ++i) {
        const int b = tid * per + i;
        if (b < a.n_seqs) mine += (uint32_t)seq_steps(a, b, cap, shift);
    }
    uint32_t incl = mine;
    for (int o = 1; o < 64; o <<= 1) {
        const uint32_t v = __shfl_up(incl, o);
        if (lane >= o) incl += v;
    }
    if (lane == 63) s_scan[wave] = incl;
    __syncthreads();
    uint32_t before = 0, total_seq = 0;
    for (int w = 0; w < DEC_WAVES; ++w) {
        if (w < wave) before += s_scan[w];
        total_seq += s_scan[w];
    }
    before += incl - mine;
    const uint64_t total = (uint64_t)total_seq * ng;
    const uint32_t share = (uint32_t)((total + gridDim.x - 1) / gridDim.x);
    const uint64_t lo = (uint64_t)blockIdx.x * share;
    if (lo >= total) return;
    const uint64_t hi = lo + share < total ? lo + share : total;
    {
        const uint64_t first = (uint64_t)before * ng;
        if (first <= lo && lo < first + (uint64_t)mine * ng) {
            uint32_t p = before;
            int b = tid * per;
            for (;; ++b) {
                const uint32_t n = (uint32_t)seq_steps(a, b, cap, shift);
                if (lo < (uint64_t)(p + n) * ng) break;
                p += n;
            }
            s_find[0] = (uint32_t)b;
            s_find[1] = p;
        }
    }
    __syncthreads();
    int b = uniform((int)s_find[0]);
    const uint64_t at = (uint64_t)(uint32_t)uniform((int)s_find[1]) * ng; // first step of sequence b
    int nt = uniform(seq_steps(a, b, cap, shift));
    int sg = (int)((lo - at) / (uint32_t)nt);
    uint64_t unit = at + (uint64_t)sg * nt; // first step of group (b, sg)

    for (uint64_t pos = lo; pos < hi;) {
        const int t0 = (int)(pos - unit);
        const int t1 = (int)((hi < unit + nt ? hi : unit + nt) - unit);
        const int len = ldc(a.kv_len + b);
        const int seen = min(max(len, 0), cap);
        if (seen != len && tid == 0) raise(a.flags, MOE_DEVFLAG_BAD_SEQ);
        // a unit's key-value head, first query head and heads
        auto head0 = [&](int hb) { return hb / gb * a.group + hb % gb * DEC_HEADS; };
        auto heads = [&](int hb) { return min(DEC_HEADS, a.group - hb % gb * DEC_HEADS); };
        const int hb = sg * U + sub, hk = hb / gb;
        const T *q = (const T *)a.q + b * a.q_stride + (int64_t)(head0(hb) + min(c, heads(hb) - 1)) * D;
        // The queries' fragments stay in registers; at D = 256, where those are short, in the wave's own
        // part of s_o, every lane reading back what it wrote.
        x8 qf[KS];
        x8 *const ql = (x8 *)&s_o[wave][0][0] + lane;
#pragma unroll
        for (int k = 0; k < KS; ++k) {
            qf[k] = ldg<x8>(q + k * 32 + g * 8);
            if (D == 256) ql[64 * k] = qf[k];
        }

        f32x4 acc[D / 16];
#pragma unroll
        for (int i = 0; i < D / 16; ++i) acc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
        float m = -INFINITY, l = 0.f;
        const int32_t *pages = a.pages + b * a.pages_stride;
        const uint8_t *kb = a.k + 2 * hk * a.head_stride, *vb = a.v + 2 * hk * a.head_stride;
        const int ts2 = (int)(2 * a.token_stride);
        const int mask = (1 << a.page_shift) - 1;
        const int end = min(seen, t1 << shift); // of this piece
        bool bad = false;

        // the two 16-token halves of a step: byte offset of the first token, tokens there
        int64_t off[2];
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
        x8 kf[2][KS];
        vload vf[8][VS];
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
                for (int k = 0; k < KS; ++k) kf[i][k] = ldo<x8>(kb + off[i], lo + k * 64);
            }
        };
        auto load_v = [&]() {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int i = j >> 2;
                const uint32_t lo = lane_off(4 * g + (j & 3), i, c * (VW * 2));
#pragma unroll
                for (int s = 0; s < VS; ++s) vf[j][s] = ldo<vload>(vb + off[i], lo + s * (32 * VW));
            }
        };
        int tok = (t0 << shift) + wsub * DEC_WAVE_TOK;
        const int step = 1 << shift;
        if (tok < end) {
            place(tok);
            load_k();
            load_v();
        }
        for (; tok < end; tok += step) {
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
            const bool more = tok + step < end;
            if (more) {
                place(tok + step);
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
        if (bad && lane == 0) raise(a.flags, MOE_DEVFLAG_BAD_PAGE);

        // ---- join the four waves: row (head c) of O^T's register layout to s_o[wave][head][d]
        l += __shfl_xor(l, 16);
        l += __shfl_xor(l, 32);
        if (g == 0) {
            s_ml[wave][c][0] = m;
            s_ml[wave][c][1] = l;
        }
        // the row's elements 16 VW s + VW (4 g + r) + j, j = 0..VW-1
#pragma unroll
        for (int s = 0; s < VS; ++s)
#pragma unroll
            for (int r = 0; r < 4; ++r)
#pragma unroll
                for (int j = 0; j < VW; j += 4)
                    *(f32x4 *)&s_o[wave][c][16 * VW * s + VW * (4 * g + r) + j] =
                        f32x4{acc[s * VW + j][r], acc[s * VW + j + 1][r], acc[s * VW + j + 2][r], acc[s * VW + j + 3][r]};
        __syncthreads();
        const bool whole = t0 == 0 && t1 == nt;
        // Partial rows: slot 0 of a workgroup holds the piece of a group that began before it, slot 1
        // that of one which goes on behind it.
        const size_t prow = DEC_WAVES * DEC_HEADS; // rows of a slot
        const size_t slot = 2 * (size_t)blockIdx.x + (t0 == 0 ? 1 : 0);
        const int items = U * rows * (D / 4);
        auto put = [&](int u, int hh, int d, f32x4 x, float M, float L) {
            const float inv = L == 0.f ? 0.f : 1.f / L;
            if (L == 0.f) x = f32x4{0.f, 0.f, 0.f, 0.f};
            const int h = head0(sg * U + u) + hh;
            *(u32x2 *)((T *)a.o + b * a.o_stride + (int64_t)h * D + d) =
                u32x2{E::pack(x[0] * inv, x[1] * inv), E::pack(x[2] * inv, x[3] * inv)};
            if (a.lse && d == 0)
                a.lse[(int64_t)b * a.hq + h] =
                    L == 0.f ? -INFINITY : (base_of(M) - E::SHIFT + __log2f(L)) * 0.69314718055994531f;
        };
        for (int i = tid; i < items; i += 256) {
            const int r = i / (D / 4), d = i % (D / 4) * 4, u = r / rows, hh = r % rows;
            if (hh >= heads(sg * U + u)) continue;
            const int w0 = u << a.wpu_shift;
            float M = -INFINITY, L = 0.f;
            for (int w = 0; w < wpu; ++w) M = fmaxf(M, s_ml[w0 + w][hh][0]);
            f32x4 x = {0.f, 0.f, 0.f, 0.f};
            for (int w = 0; w < wpu; ++w) {
                const float f = exp2_(s_ml[w0 + w][hh][0] - base_of(M));
                L += f * s_ml[w0 + w][hh][1];
                x += f * *(const f32x4 *)&s_o[w0 + w][hh][d];
            }
            if (whole) put(u, hh, d, x, M, L);
            else {
                publish(a.part + (slot * prow + u * DEC_HEADS + hh) * D + d, x);
                if (d == 0) publish(a.part_ml + (slot * prow + u * DEC_HEADS + hh) * 2, f32x2{M, L});
            }
        }
        if (!whole) {
            // the group's pieces: workgroups w0 (slot 1) to w1 (slot 0)
            const uint32_t w0 = (uint32_t)(unit / share), w1 = (uint32_t)((unit + nt - 1) / share);
            uint32_t wa = blockIdx.x / JOIN * JOIN;
            const uint32_t wb = min(wa + JOIN - 1, w1);
            wa = max(wa, w0);
            uint32_t first = wa, stride = 1, n = wb - wa + 1;
            uint32_t *count = a.arrived + 2 * wa + (wa == w0 ? 1 : 0);
            for (int level = 0;; ++level) {
                __syncthreads(); // waits for this piece's stores
                if (tid == 0) {
                    s_last = __hip_atomic_fetch_add(count, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                    if (s_last == n - 1) __hip_atomic_store(count, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                }
                __syncthreads();
                if (s_last != n - 1) break;
                // piece p's slot: workgroup first + p stride, of w0 the later one, and of a joined
                // group of JOIN its first workgroup's
                auto at_piece = [&](uint32_t p) {
                    uint32_t w = first + p * stride;
                    if (level) w = p == 0 ? w0 : w / JOIN * JOIN;
                    return 2 * (size_t)w + (w == w0 ? 1 : 0);
                };
                const int R = U * rows;
                float *fac = &s_o[0][0][0];                     // [n][R]
                f32x2 *ml = (f32x2 *)&s_ml[0][0][0];            // [R]: the joined maximum and sum
                for (int r = tid; r < R; r += 256) {
                    const int u = r / rows, hh = r % rows;
                    const float *src = a.part_ml + (size_t)(u * DEC_HEADS + hh) * 2;
                    float M = -INFINITY, L = 0.f;
                    for (uint32_t p = 0; p < n; p += 8) {
                        f32x2 v[8];
#pragma unroll
                        for (int j = 0; j < 8; ++j)
                            v[j] = p + j < n ? remote2(src + at_piece(p + j) * prow * 2) : f32x2{-INFINITY, 0.f};
                        float mx = M;
#pragma unroll
                        for (int j = 0; j < 8; ++j) mx = fmaxf(mx, v[j].x);
                        L *= exp2_(M - base_of(mx));
                        M = mx;
#pragma unroll
                        for (int j = 0; j < 8; ++j) {
                            L += v[j].y * exp2_(v[j].x - base_of(M));
                            if (p + j < n) fac[(p + j) * R + r] = v[j].x;
                        }
                    }
                    for (uint32_t p = 0; p < n; ++p) fac[p * R + r] = exp2_(fac[p * R + r] - base_of(M));
                    ml[r] = f32x2{M, L};
                }
                __syncthreads();
                const bool final = level || w0 / JOIN == w1 / JOIN;
                for (int i = tid; i < items; i += 256) {
                    const int r = i / (D / 4), d = i % (D / 4) * 4, u = r / rows, hh = r % rows;
                    if (hh >= heads(sg * U + u)) continue;
                    f32x4 x = {0.f, 0.f, 0.f, 0.f};
                    const float *src = a.part + (size_t)(u * DEC_HEADS + hh) * D + d;
                    for (uint32_t p = 0; p < n; p += 8) {
                        f32x4 v[8];
#pragma unroll
                        for (int j = 0; j < 8; ++j)
                            v[j] = p + j < n ? remote4(src + at_piece(p + j) * prow * D) : f32x4{};
#pragma unroll
                        for (int j = 0; j < 8; ++j) x += (p + j < n ? fac[(p + j) * R + r] : 0.f) * v[j];
                    }
                    if (final) put(u, hh, d, x, ml[r].x, ml[r].y);
                    else publish(a.part + (at_piece(0) * prow + u * DEC_HEADS + hh) * D + d, x);
                }
                if (final) break;
                for (int r = tid; r < R; r += 256)
                    publish(a.part_ml + (at_piece(0) * prow + r / rows * DEC_HEADS + r % rows) * 2, ml[r]);
                first = w0 / JOIN * JOIN;
                stride = JOIN;
                n = w1 / JOIN - w0 / JOIN + 1;
                count = a.arrived + 2 * gridDim.x + w0;
            }
        }
        pos = unit + t1;
        if (pos < hi) { // the next (sequence, heads)
            __syncthreads(); // s_o is free again
            unit += nt;
            if (++sg == ng) {
                sg = 0;
                ++b;
                nt = uniform(seq_steps(a, b, cap, shift));
            }
        }
    }
}

template <typename T>
hipError_t decode_d(const AttnArgs &a, int d, hipStream_t st) {
    const unsigned grid = (unsigned)a.n_wg;
    if (d == 64) k_attn_decode<T, 64><<<grid, 256, 0, st>>>(a);
    else if (d == 128) k_attn_decode<T, 128><<<grid, 256, 0, st>>>(a);
    else k_attn_decode<T, 256><<<grid, 256, 0, st>>>(a);
    return hipGetLastError();
}

} // namespace

hipError_t launch_attn_decode(const AttnArgs &args, int type, int d, hipStream_t st) {
    AttnArgs a = args;
    // Units enough for every workgroup to have several at once: let fewer waves share one.
    const int hb = a.hkv * ((a.group + DEC_HEADS - 1) / DEC_HEADS);
    const int64_t units = (int64_t)a.n_seqs * hb;
    a.wpu_shift = 2;
    if (hb % 4 == 0 && units >= 4 * a.n_wg) a.wpu_shift = 0;
    else if (hb % 2 == 0 && units >= 2 * a.n_wg) a.wpu_shift = 1;
    return type == MOE_T_F16 ? decode_d<f16_t>(a, d, st) : decode_d<bf16_t>(a, d, st);
}

} // namespace moe
