// k_attn_prompt.hip -- packed causal prompts over the paged cache.
//
//   o[i][h] = sum_{j <= p_i} e^(s_ij - m_i) V_j / sum_j e^(s_ij - m_i),   s_ij = scale * q[i][h] . K_j,
//   p_i the row's position (kv_len - rows + i)
//
// Bound by the matrix cores: 4 D operations for each (row, head, seen token).  A workgroup's rows are
// PR_ROWS (token, head) pairs of one key-value head, the heads of a token side by side, so the
// group's heads share each tile of K and V and the causal edge crosses few of them.
//   * A wave takes 32 rows, a row to a lane pair:
//       S^T[token][row] = K Q^T      32x32x16 products; a row's scores lie in the lanes r and r + 32,
//                                    so maximum, sum and rescaling are a lane's own (and one swap)
//       O^T[d][row] += V^T P^T       S^T's register layout is P^T's operand layout with the tokens of 16
//                                    in the order {0-3, 8-11}, {4-7, 12-15}; V^T is stored in that order
//   * K and V tiles of BN tokens go straight to LDS (no registers), two buffers, one barrier a tile; the
//     next tile's loads go out between this one's score products.  V^T is read by the transposing LDS
//     load: of 16 lanes, lane 4 j + c gives the address of elements 4c..4c+3 of token j, lane d gets
//     element d of tokens 0..3.  A row's 16-byte chunks are stored at chunk ^ f(token), f = token & 15 for K
//     (& 7 at D = 64) and 2 (token & 3) for V, so that all reads are free of bank conflicts.
//   * Of the weights only those of the first 16 tokens are computed before the output's products, the others
//     between these.
//   * The running maximum is only raised when a row's new one exceeds it by more than 2^8: until then
//     the weights stay below 2^(8 + SHIFT) and no output is rescaled.
//   * Too few rows to fill the card (a piece of a prompt over a long cache, short prompts): the tokens of
//     the longest rows are cut into pieces, whose partial rows a second launch joins.
// At D = 256 a wave has a SIMD for itself (128 registers of outputs, 64 of queries), so what it does between
// the products adds to their time: a prompt of 4096 rows of 16/2 heads 142 us, 969 TFLOP/s, where a matrix
// product of 8192^3 reaches 1221.  At D <= 128 two workgroups share a CU: 8192 rows of 32/8 heads of 128 529 us,
// 1039 TFLOP/s.  (All loads before the products, all weights before theirs, the maximum's swap through
// LDS: 167 and 553 us.)
#include "attn_device.hpp"

namespace moe {

namespace {

constexpr int BN = 64;           // tokens of a tile
constexpr float LAZY = 8.f;      // log2 of what a weight may exceed 1 by
constexpr int PR_MIN_CHUNK = 4;  // tiles of a piece at least
constexpr int PR_CUT_FROM = 9;   // tiles of the longest rows from which on they are cut
constexpr int PR_MAX_SPLITS = 128;

// A sequence's packed rows, inside the arrays whatever row_start holds, and its length.
struct Rows {
    int r0, n, end, len; // end: row_start's own
    bool bad;
};
__device__ __forceinline__ Rows seq_rows(const AttnArgs &a, int b) {
    const int s = ldg<int>(a.row_start + b), e = ldg<int>(a.row_start + b + 1), len = ldg<int>(a.kv_len + b);
    const int r0 = min(max(s, 0), a.n_rows), r1 = min(max(e, r0), a.n_rows);
    return {r0, r1 - r0, e, len, r0 != s || r1 != e};
}

// Workgroups that are on the card at once.
template <int D>
__host__ __device__ __forceinline__ uint32_t slots_of(const AttnArgs &a) {
    return a.n_cu * (D == 256 ? 1u : 2u);
}

// Tokens that the f-th (token, head) pair's row of a sequence sees, its first row's position given.
__device__ __forceinline__ int seen_by(const AttnArgs &a, int64_t first_pos, int f) {
    const int64_t p = first_pos + f / a.group + 1, cap = (int64_t)a.max_pages << a.page_shift;
    return (int)(p < 0 ? 0 : p > cap ? cap : p);
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

// Products of N fragments, each read from LDS DEPTH products before its own.  The order is kept four products
// by four (by itself the compiler reads, waits, multiplies; one by one is 2 to 5 % slower).
template <int N, int DEPTH, typename Frag, typename Read, typename Product>
__device__ __forceinline__ void products(Read read, Product product) {
    Frag f[DEPTH];
#pragma unroll
    for (int i = 0; i < DEPTH; ++i) f[i] = read(i);
#pragma unroll
    for (int i = 0; i < N; ++i) {
        product(i, f[i % DEPTH]);
        if (i + DEPTH < N) f[i % DEPTH] = read(i + DEPTH);
        if (i % 4 == 3) __builtin_amdgcn_sched_barrier(0);
    }
}

// The values of lanes r and r + 32, to both.
__device__ __forceinline__ f32x2 both_halves(float x) {
    // (of the builtin's two results this compiler uses the first one for both; the wait is for the registers'
    // writes just before)
    float lo = x, hi = x;
    asm("s_nop 1\n\tv_permlane32_swap_b32 %0, %1" : "+v"(lo), "+v"(hi));
    return f32x2{lo, hi};
}

// A workgroup's place: PR_ROWS (token, head) pairs of sequence b, from its f0-th of nf on, of which the
// last one sees ext tokens and the first one `full`; piece `piece` of n at most, `chunk` tiles each.
struct Place {
    int b, r0, hk;
    int f0, nf;
    int64_t first_pos; // of the sequence's first row
    int ext, full, chunk;
    int nth, piece, n; // nth: place number
};

// This workgroup's place, or (join) place number blockIdx.x; false where there is none.  Whole rows: the
// tiles that see the most tokens first, where not all are at work at once (8 prompts of 100 to 2001 rows, the
// longest one first, 103.5 -> 97.6 us; of more than 64 sequences the last one first), the key-value head as the
// fastest index, so that a head's tiles share an XCD's L2.  Rows in pieces: the tiles that read the same
// tokens lie on one XCD (workgroups go round the XCDs in turn), side by side.  (No loop runs on and no
// index leaves its array if the lengths and rows should change under the call.)
template <int D, bool JOIN>
__device__ __forceinline__ bool find_place(const AttnArgs &a, int lane, int wave, bool flag, Place &pl) {
    const int cap = a.max_pages << a.page_shift;
    uint32_t mine, incl;
    int most = 0; // tokens that a row sees
    bool bad = false;
    Rows sr = {}; // of the sequence that the lane looked at last
    auto tiles_of = [&](int b) {
        sr = seq_rows(a, min(b, a.n_seqs - 1));
        if (b >= a.n_seqs) sr.n = 0;
        bad |= sr.bad || (sr.n > 0 && (sr.len < 0 || sr.len > cap));
        most = max(most, sr.n > 0 ? min(sr.len, cap) : 0);
        return ((uint32_t)sr.n * a.group + PR_ROWS - 1) / PR_ROWS;
    };
    count_seqs(a.n_seqs, lane, wave, tiles_of, mine, incl);
    if (flag && bad) raise(a.flags, MOE_DEVFLAG_BAD_SEQ);
    if (a.n_seqs > 64 && a.splits > 1) { // each wave has looked at some
        __shared__ int s_most[4];
        most = (int)wave_most((uint32_t)most);
        if (lane == 0) s_most[wave] = most;
        __syncthreads();
        most = max(max(s_most[0], s_most[1]), max(s_most[2], s_most[3]));
    }
    const uint32_t total = (uint32_t)__builtin_amdgcn_readlane((int)incl, 63);
    if (total == 0) return false;
    uint32_t nth = blockIdx.x / a.hkv; // tile number, from the end
    pl.hk = blockIdx.x - nth * a.hkv;
    pl.piece = 0;
    pl.n = 1;
    pl.chunk = 1 << 30;
    if (a.splits > 1 && total <= a.splits_below && __any(most > (PR_CUT_FROM - 1) * BN)) {
        const int n = min(a.splits, (int)(slots_of<D>(a) / (total * a.hkv))), tiles = ((int)wave_most((uint32_t)most) + BN - 1) / BN;
        pl.chunk = max(PR_MIN_CHUNK, (tiles + n - 1) / n);
        pl.n = max(1, (tiles + pl.chunk - 1) / pl.chunk);
        if (!JOIN) {
            const uint32_t jobs = total * a.hkv * pl.n, per_xcd = (jobs + 7) / 8;
            const uint32_t y = blockIdx.x / 8, job = blockIdx.x % 8 * per_xcd + y;
            if (y >= per_xcd || job >= jobs) return false;
            const uint32_t s = job / total;
            nth = job - s * total;
            pl.piece = s / a.hkv;
            pl.hk = s - pl.piece * a.hkv;
        }
    }
    if (nth >= total) return false;
    pl.nth = nth * a.hkv + pl.hk;
    // The heaviest first; all at work at once, two on some CUs: there the lighter one is to lie beside the
    // heavier one.
    const uint32_t first = a.n_cu / a.hkv; // (head groups of) tiles that take a CU each
    if (D < 256 && pl.n == 1 && total > first && total * a.hkv <= 2u * a.n_cu && nth >= first)
        nth = total - 1 - (nth - first);
    int from; // the lane that has the sequence
    uint32_t before; // the sequence's tiles before this one
    if (a.n_seqs <= 64 && a.n_seqs > 1 && pl.n == 1 && total > first) {
        // Tile j of a sequence, from its end, weighs `top` - j (in tiles of seen tokens).  The nth heaviest
        // one: of weight w, the largest one that more than nth reach, and among those of the same weight by
        // sequence.
        const int len = min(max(sr.len, 0), min(cap, 1 << 28)); // (of more, no order)
        const int top = (len / PR_ROWS) * a.group + (len % PR_ROWS * a.group) / PR_ROWS;
        auto reach = [&](int w) { // tiles of weight w or more
            const uint32_t n = top >= w ? min((uint32_t)(top - w) + 1, mine) : 0u;
            return (uint32_t)__builtin_amdgcn_readlane((int)wave_scan(n), 63);
        };
        int w = -(int)total, above = (int)wave_most((uint32_t)top) + 1;
        while (above - w > 1) {
            const int mid = w + (above - w) / 2;
            if (reach(mid) > nth) w = mid;
            else above = mid;
        }
        uint64_t same = __ballot(top >= w && (uint32_t)(top - w) < mine);
        for (uint32_t i = nth - reach(above); i > 0; --i) same &= same - 1;
        from = __builtin_ctzll(same);
        pl.b = from;
        before = (uint32_t)__builtin_amdgcn_readlane((int)(mine - 1 - (uint32_t)(top - w)), from);
    } else {
        const uint32_t want = total - 1 - nth;
        pl.b = find_seq(a.n_seqs, lane, tiles_of, mine, incl, want, before, from);
        before = want - before;
    }
    auto of = [&](int v) { return __builtin_amdgcn_readlane(v, from); };
    pl.r0 = of(sr.r0);
    pl.f0 = (int)before * PR_ROWS;
    pl.nf = of(sr.n) * a.group;
    if (pl.f0 >= pl.nf) return false; // (the arrays changed during the call)
    pl.first_pos = (int64_t)min(max(of(sr.len), 0), cap) - of(sr.end) + pl.r0;
    pl.full = uniform(seen_by(a, pl.first_pos, pl.f0));
    pl.ext = uniform(seen_by(a, pl.first_pos, min(pl.f0 + PR_ROWS, pl.nf) - 1));
    return true;
}

// A place's partial rows of piece `piece`.
__device__ __forceinline__ size_t part_row(const Place &pl, int piece) {
    return ((size_t)pl.nth * pl.n + piece) * PR_ROWS;
}

// f16: 2^(SHIFT + LAZY) is in range.
template <typename T>
constexpr float SHIFT = Elem<T>::SHIFT > 0.f ? 7.f : 0.f;

template <typename T, int D>
__global__ __launch_bounds__(256, D == 256 ? 1 : 2) void k_attn_prompt(AttnArgs a) {
    typedef Elem<T> E;
    typedef typename E::x8 x8;
    constexpr int KS = D / 16;             // products of a score tile
    constexpr int NB = BN / 16;            // blocks of 16 tokens, each in one page: one a wave
    constexpr int NS = BN / 32;            // score tiles
    constexpr int RI = 512 / D;            // tokens of one wave load
    constexpr int NL = 16 / RI;            // loads of a wave and tile, for K and for V
    constexpr int DEPTH = D == 64 ? 4 : 6; // fragments read ahead
    constexpr int NP = NS * KS;            // products of a tile's scores; as many of its outputs
    static_assert(NP == 4 * NL && NP == NS * D / 16, "a load every other product");
    constexpr int KM = D == 64 ? 7 : 15, KQ = (KM + 1) / 2; // K's chunks: swizzle, offsets of a lane
    constexpr uint32_t ALL = (1u << NB) - 1;
    static_assert(NB == 4, "a block a wave");
    // Two tiles, each an array of its own: the compiler has reads wait for loads to the same array.
    __shared__ __attribute__((aligned(16))) T s_k0[BN * D], s_k1[BN * D], s_v0[BN * D], s_v1[BN * D];
    __shared__ int s_bad;

    const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6);
    const int r = lane & 31, h = lane >> 5;
    Place pl;
    if (!find_place<D, false>(a, lane, wave, blockIdx.x == 0, pl)) return;
    // this piece's tiles [t, nt); the first one also where no token is seen, to write the rows
    const int tiles = (pl.ext + BN - 1) / BN, first_t = pl.piece * pl.chunk;
    if (pl.piece > 0 && first_t >= tiles) return;
    const int nt = min(tiles, first_t + pl.chunk), ext = pl.ext;
    const bool whole = tiles <= pl.chunk;
    if (tid == 0) s_bad = 0;

    // this lane's row; one behind the last reads the last one's query and sees nothing
    const int pair = pl.f0 + wave * 32 + r;
    const bool valid = pair < pl.nf;
    const int tok = min(pair, pl.nf - 1) / a.group;
    const int row = pl.r0 + tok, head = pl.hk * a.group + min(pair, pl.nf - 1) - tok * a.group;
    const int seen = valid ? seen_by(a, pl.first_pos, pair) : 0;
    // Scale 0: the smallest normal number, so that -inf (not seen) stays -inf; any finite score times it
    // is 0 beside the exponential's 1.
    const float scale = fmaxf(fabsf(a.scale_log2), 1.17549435e-38f);

    // ---- tiles
    const int32_t *pages = a.pages + pl.b * a.pages_stride;
    const uint8_t *kb = a.k + 2 * pl.hk * a.head_stride, *vb = a.v + 2 * pl.hk * a.head_stride;
    const uint32_t ts2 = (uint32_t)(2 * a.token_stride); // (below 2^24)
    const int mask = (1 << a.page_shift) - 1;
    // Lane i has the page of block i of the tile to be staged next (-1: none); okay: the blocks of the tile
    // staged last that have a page of the cache, or no token to be seen.
    bool bad_page = false;
    uint32_t okay = 0;
    auto look_up = [&](int t) {
        const int key = t * BN + 16 * lane;
        return lane < NB && key < ext ? ldg<int>(pages + (key >> a.page_shift)) : -1;
    };
    int pg_next = look_up(first_t);
    u32x4 qw[KS];
#pragma unroll
    for (int k = 0; k < KS; ++k) qw[k] = ldg<u32x4>((const T *)a.q + row * a.q_stride + head * D + h * 8 + k * 16);
    int64_t off = 0; // of this wave's block of the tile; tokens there
    int toks = 0;
    auto stage = [&](int t) {
        const int key = t * BN + 16 * wave;
        const uint64_t in = __ballot((unsigned)pg_next < (unsigned)a.n_pages);
        const uint64_t none = __ballot(t * BN + 16 * lane >= ext);
        okay = (uint32_t)(in | none) & ALL;
        bad_page |= okay != ALL;
        const bool here = in >> wave & 1;
        const int pg = here ? __builtin_amdgcn_readlane(pg_next, wave) : 0;
        toks = here ? min(16, ext - key) : 0;
        off = 2 * (pg * a.page_stride + (key & mask) * a.token_stride);
        if (t + 1 < nt) pg_next = look_up(t + 1);
    };
    // Every wave loads its block.  Tokens that are not there are taken from a place that is (masked below).
    // Load x of 2 NL: the keys', then the values'.
    auto stage_load = [&](T *to_k, T *to_v, int x) {
        const bool values = x >= NL;
        const int p = x % NL, key = p * RI + lane / (D / 8), ch = lane % (D / 8); // of the block
        const int t = max(0, min(key, toks - 1));
        lds_load16((values ? vb : kb) + off, __umul24(t, ts2) + (ch ^ (values ? 2 * (key & 3) : key & KM)) * 16,
                   (values ? to_v : to_k) + (wave * NL + p) * 512);
    };

    f32x16 o[D / 32];
#pragma unroll
    for (int i = 0; i < D / 32; ++i) o[i] = f32x16{};
    float m = -INFINITY, l = 0.f; // the maximum that weights are taken against, and this lane's sum
    uint32_t ko[KQ], vo[2];
#pragma unroll
    for (int i = 0; i < KQ; ++i) ko[i] = r * (D * 2) + (((2 * i + h) ^ (r & KM)) * 16);
    {
        const int j = (lane & 15) >> 2, c = 2 * (r >> 4) + ((lane & 3) >> 1); // token, chunk of its first 64 bytes
        vo[0] = (4 * h + j) * (D * 2) + ((c ^ (2 * j)) * 16) + 8 * (lane & 1);
        vo[1] = vo[0] ^ 64;
    }

    if (first_t < nt) {
        stage(first_t);
#pragma unroll
        for (int x = 0; x < 2 * NL; ++x) stage_load(s_k0, s_v0, x);
    }
    x8 qf[KS];
    const uint32_t flip = a.scale_log2 < 0.f ? 0x80008000u : 0u; // a negative scale: -q, exactly
#pragma unroll
    for (int k = 0; k < KS; ++k) qf[k] = __builtin_bit_cast(x8, qw[k] ^ flip);
    bool fresh = true, part = false;
    uint32_t ok = 0;
    int first_part = nt; // the first tile that some row does not see all of
    int t = first_t;
    float mx;
    // Works on tile t; true: it is done, and another one follows.
    auto tile = [&](T *k_now, T *v_now, T *k_next, T *v_next) {
        const uint8_t *lk = (const uint8_t *)k_now;
        if (fresh) {
            ok = okay;
            part = (t + 1) * BN > pl.full || ok != ALL;
            lds_loaded();
            __syncthreads(); // tile t is there, and nobody works on tile t - 1
            // A value that a row does not see meets a weight of 0, which an infinity or NaN would survive:
            // in such a tile those are 0 for the products, and the rows that see them get them at the end.
            if (part) {
                first_part = min(first_part, t);
                constexpr int NW = BN * D / 8 / 256;
                u32x4 w[NW];
                bool bad = false;
#pragma unroll
                for (int i = 0; i < NW; ++i) w[i] = ((const u32x4 *)v_now)[tid + 256 * i];
#pragma unroll
                for (int i = 0; i < NW; ++i) {
                    bool any = false;
                    for (int j = 0; j < 4; ++j) any |= not_finite<T>(w[i][j]);
                    if (any) {
                        for (int j = 0; j < 4; ++j) w[i][j] = finite_only<T>(w[i][j]);
                        ((u32x4 *)v_now)[tid + 256 * i] = w[i];
                        bad = true;
                    }
                }
                if (bad) s_bad = 1;
                __syncthreads();
            }
        }
        f32x16 s[NS];
        auto read_k = [&](int x) { // the score tiles in turn: two chains of sums
            const int i = x % NS, k = x / NS;
            return *(const x8 *)(lk + ko[k % KQ] + i * (32 * D * 2) + (k / KQ) * (32 * KQ));
        };
        auto score = [&](int x, x8 kf) { s[x % NS] = E::mfma32(kf, qf[x / NS], x < NS ? f32x16{} : s[x % NS]); };
        // The next tile's loads go out between the products: all at once would hold the wave up.
        if (fresh && t + 1 < nt) {
            stage(t + 1);
            products<NP, DEPTH, x8>(read_k, [&](int x, x8 kf) {
                score(x, kf);
                if (x % 2 == 0) stage_load(k_next, v_next, x / 2);
            });
        } else products<NP, DEPTH, x8>(read_k, score);
        if (part)
#pragma unroll
            for (int i = 0; i < NS; ++i)
#pragma unroll
                for (int j = 0; j < 16; ++j) {
                    const int key = 32 * i + 8 * (j >> 2) + 4 * h + (j & 3);
                    if (t * BN + key >= seen || !(ok >> (2 * i + (j >> 3)) & 1)) s[i][j] = -INFINITY;
                }
        mx = s[0][0];
#pragma unroll
        for (int i = 0; i < NS; ++i)
#pragma unroll
            for (int j = 0; j < 16; ++j) mx = fmaxf(mx, s[i][j]);
        const f32x2 mb = both_halves(mx);
        mx = fmaxf(mb.x, mb.y) * scale;
        if (t == first_t) m = fmaxf(m, mx); // nothing to rescale yet
        fresh = !__any(mx > m + LAZY);
        if (!fresh) return false;
        const float base = base_of(m) - SHIFT<T>;
        float sum = 0.f;
        u32x4 pw[2 * NS]; // the weights, in P^T's operand layout
        auto weights = [&](int k, int w) { // of block k's word w
            const int i = k / 2, j = k % 2 * 8 + 2 * w;
            const float p0 = exp2_(__builtin_fmaf(s[i][j], scale, -base));
            const float p1 = exp2_(__builtin_fmaf(s[i][j + 1], scale, -base));
            sum += p0 + p1;
            pw[k][w] = E::pack(p0, p1);
        };
#pragma unroll
        for (int w = 0; w < 4; ++w) weights(0, w);
        const MOE_LDS uint8_t *const lv[2] = {lds_at(v_now, vo[0]), lds_at(v_now, vo[1])};
        auto read_v = [&](int x) {
            const int k = x / (D / 32), i = x % (D / 32);
            const MOE_LDS uint8_t *p = lv[i & 1] + k * (16 * D * 2) + (i >> 1) * 128;
            const u32x2 v0 = lds_read_tr(p), v1 = lds_read_tr(p + 8 * D * 2);
            return __builtin_bit_cast(x8, (u32x4{v0.x, v0.y, v1.x, v1.y}));
        };
        products<NP, DEPTH, x8>(read_v, [&](int x, x8 vf) {
            const int k = x / (D / 32), i = x % (D / 32);
            o[i] = E::mfma32(vf, __builtin_bit_cast(x8, pw[k]), o[i]);
            // the next block's weights, beside this one's products
            for (int w = 4 * i / (D / 32); k + 1 < NB && w < 4 * (i + 1) / (D / 32); ++w) weights(k + 1, w);
        });
        l += sum;
        return ++t < nt;
    };
    while (t < nt) {
        // Tiles until a row's maximum grows past what its weights allow for; then the outputs are rescaled
        // and the tile's scores computed again.  (Two loops, so that the inner one's outputs are the
        // products' own and stay where those put them.)
        for (;;) {
            if (((t - first_t) & 1) == 0 && !tile(s_k0, s_v0, s_k1, s_v1)) break;
            if (!tile(s_k1, s_v1, s_k0, s_v0)) break;
        }
        if (t < nt) {
            const float mn = fmaxf(m, mx);
            const float alpha = exp2_(m - base_of(mn));
            m = mn;
            l *= alpha;
#pragma unroll
            for (int i = 0; i < D / 32; ++i) o[i] *= alpha;
        }
    }
    if (bad_page && lane == 0) raise(a.flags, MOE_DEVFLAG_BAD_PAGE);

    // ---- the infinities and NaN that were 0 for the products, token by token
    __syncthreads();
    if (*(volatile int *)&s_bad)
#pragma unroll 1
        for (int key = first_part * BN; key < min(seen, nt * BN); ++key) {
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
                        if (not_finite<T>(e)) o[i][4 * j + x] += (float)__builtin_bit_cast(T, (uint16_t)e);
                    }
                }
        }

    // ---- rows out, or their part
    const f32x2 lb = both_halves(l);
    const float sum = lb.x + lb.y;
    if (!whole) {
        if (!valid) return;
        const size_t pr = part_row(pl, pl.piece) + wave * 32 + r;
        if (h == 0) *(f32x2 *)(a.part_ml + 2 * pr) = f32x2{m, sum};
#pragma unroll
        for (int i = 0; i < D / 32; ++i)
#pragma unroll
            for (int j = 0; j < 16; j += 4)
                *(f32x4 *)(a.part + pr * D + 4 * h + 32 * i + 2 * j) =
                    f32x4{o[i][j], o[i][j + 1], o[i][j + 2], o[i][j + 3]};
        return;
    }
    // Through LDS, so that whole rows are stored: a wave's rows in a part of its own, 16 bytes between them.
    // (The tiles are done with: the barrier before the infinities.)
    constexpr int OS = D + 8;
    static_assert(32 * OS <= BN * D, "the rows in the tiles' place");
    T *so = (wave == 0 ? s_k0 : wave == 1 ? s_k1 : wave == 2 ? s_v0 : s_v1);
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
    for (int i = 0; i < D / 32; ++i)
#pragma unroll
        for (int j = 0; j < 16; j += 4) {
            u32x2 w = {E::pack(o[i][j] * inv, o[i][j + 1] * inv), E::pack(o[i][j + 2] * inv, o[i][j + 3] * inv)};
            if (sum == 0.f) w = u32x2{0u, 0u};
            *(u32x2 *)(so + r * OS + 4 * h + 32 * i + 2 * j) = w;
        }
    if (a.lse && valid && h == 0)
        a.lse[(int64_t)row * a.hq + head] =
            sum == 0.f ? -INFINITY : (base_of(m) - SHIFT<T> + __log2f(sum)) * 0.69314718055994531f;
    constexpr int LR = D / 8; // lanes of a row
    const int f0 = pl.f0 + wave * 32, n = min(32, pl.nf - f0);
    const int t0 = f0 / a.group, y0 = f0 - t0 * a.group; // the first row's token and head
    const float by_group = 1.f / (float)a.group;
#pragma unroll
    for (int i = 0; i < LR / 2; ++i) { // 64 / LR rows at a time
        const int x = i * (64 / LR) + lane / LR;
        const u32x4 w = *(const u32x4 *)(so + x * OS + lane % LR * 8);
        if (x < n) {
            // (y0 + x) / group, below 256 + 32: exact in f32
            const int t = (int)(((float)(y0 + x) + 0.5f) * by_group), hd = pl.hk * a.group + y0 + x - t * a.group;
            *(u32x4 *)((T *)a.o + (pl.r0 + t0 + t) * a.o_stride + hd * D + lane % LR * 8) = w;
        }
    }
}

// The partial rows of places that were cut into pieces: sum_p f_p x_p / sum_p f_p l_p, f_p = 2^(m_p - max m),
// the same order every time.  One row a workgroup (gridDim.y = PR_ROWS): a thread takes four elements of
// every PG-th piece, and the threads' sums are joined through LDS.  More rows: a thread takes four
// elements of a row through all pieces.
constexpr int JOIN_ROWS = 8, JOIN_B = 8;
template <typename T, int D>
__global__ __launch_bounds__(256) void k_attn_prompt_join(AttnArgs a) {
    constexpr int TPR = D / 4, PG = 256 / TPR;
    __shared__ f32x4 s_x[PG][TPR];
    __shared__ f32x2 s_ml[PG];
    const int tid = threadIdx.x, i = tid % TPR, g = tid / TPR;
    Place pl;
    if (!find_place<D, true>(a, tid & 63, uniform(tid >> 6), false, pl)) return;
    const int tiles = (pl.ext + BN - 1) / BN, n = min(pl.n, (tiles + pl.chunk - 1) / pl.chunk);
    if (n < 2) return;
    const bool one = gridDim.y == PR_ROWS;
    const int rows = PR_ROWS / gridDim.y, step = one ? PG : 1;
    for (int x0 = one ? 0 : g; x0 < rows; x0 += PG) {
        const int r = blockIdx.y * rows + x0, pair = pl.f0 + r;
        if (pair >= pl.nf) return; // (one: all threads)
        float M = -INFINITY, L = 0.f;
        f32x4 x = {0.f, 0.f, 0.f, 0.f};
        for (int p = one ? g : 0; p < n; p += JOIN_B * step) {
            f32x2 ml[JOIN_B];
            f32x4 v[JOIN_B];
#pragma unroll
            for (int j = 0; j < JOIN_B; ++j) {
                const int q = p + j * step;
                ml[j] = q < n ? ldg<f32x2>(a.part_ml + 2 * (part_row(pl, q) + r)) : f32x2{-INFINITY, 0.f};
                v[j] = q < n ? ldg<f32x4>(a.part + (part_row(pl, q) + r) * D + 4 * i) : f32x4{};
            }
            float mn = M;
#pragma unroll
            for (int j = 0; j < JOIN_B; ++j) mn = fmaxf(mn, ml[j].x);
            const float f = exp2_(M - base_of(mn));
            M = mn;
            L *= f;
            x *= f;
#pragma unroll
            for (int j = 0; j < JOIN_B; ++j) {
                const float w = exp2_(ml[j].x - base_of(M));
                L += w * ml[j].y;
                x += w * v[j];
            }
        }
        if (one) {
            s_x[g][i] = x;
            if (i == 0) s_ml[g] = f32x2{M, L};
            __syncthreads();
            if (g) return;
            const float m0 = M;
            for (int k = 1; k < PG; ++k) M = fmaxf(M, s_ml[k].x);
            const float f = exp2_(m0 - base_of(M));
            L *= f;
            x *= f;
            for (int k = 1; k < PG; ++k) {
                const float w = exp2_(s_ml[k].x - base_of(M));
                L += w * s_ml[k].y;
                x += w * s_x[k][i];
            }
        }
        const int tok = pair / a.group, head = pl.hk * a.group + pair - tok * a.group;
        put_row<T>(a, pl.r0 + tok, head, D, 4 * i, x, M, L, SHIFT<T>);
    }
}

template <typename T, int D>
hipError_t prompt_d(const AttnArgs &args, hipStream_t st) {
    AttnArgs a = args;
    const int64_t places = prompt_places(a), slots = slots_of<D>(a), cap = (int64_t)a.max_pages << a.page_shift;
    // A quarter of the card's workgroup slots or less, and PR_CUT_FROM tiles: the rows are cut into pieces, as
    // many as fill the slots once.  64 rows of 16/2 heads of 256 over 32k tokens: 1144 -> 62 us (99 us cut to
    // fill them twice, by an earlier join).  With more places the partial rows cost what the pieces gain:
    // 1024 rows of 32/8 heads of 128 (half the slots) 32 us whole, 44 us cut in two.  Of 9 tiles (64 rows
    // after 512) 28.0 -> 24.4 us and, 32/8 heads of 128, 18.3 -> 16.7 us; of 8 (512 rows) 26.6 -> 27.9 and 17.4 ->
    // 23.2 us.  (The worst that the rule does: 512 rows after 256 of 32/8 heads of 128, 22.8 -> 27.9 us; after
    // 2048, 61 -> 42 us.)  The kernels count the tiles themselves, so sequences without rows do not matter;
    // whether it can be is known here, and the second launch left out otherwise.
    a.splits_below = (unsigned)(slots / 4 / a.hkv);
    const int64_t useful = (cap + BN * PR_MIN_CHUNK - 1) / (BN * PR_MIN_CHUNK);
    a.splits = 1;
    if (cap > (PR_CUT_FROM - 1) * BN && (int64_t)a.n_rows * a.group <= (int64_t)a.splits_below * PR_ROWS)
        a.splits = (int)(useful < PR_MAX_SPLITS ? useful : PR_MAX_SPLITS);
    k_attn_prompt<T, D><<<(unsigned)(a.splits > 1 && places < slots + 7 ? slots + 7 : places), 256, 0, st>>>(a);
    if (a.splits > 1) {
        const int64_t cut = (int64_t)a.splits_below * a.hkv, x = places < cut ? places : cut;
        k_attn_prompt_join<T, D><<<dim3((unsigned)x, PR_ROWS / (x > 16 ? JOIN_ROWS : 1)), 256, 0, st>>>(a);
    }
    return hipGetLastError();
}

template <typename T>
hipError_t prompt_t(const AttnArgs &a, int d, hipStream_t st) {
    return d == 64 ? prompt_d<T, 64>(a, st) : d == 128 ? prompt_d<T, 128>(a, st) : prompt_d<T, 256>(a, st);
}

} // namespace

hipError_t launch_attn_prompt(const AttnArgs &a, int type, int d, hipStream_t st) {
    return type == MOE_T_F16 ? prompt_t<f16_t>(a, d, st) : prompt_t<bf16_t>(a, d, st);
}

} // namespace moe
