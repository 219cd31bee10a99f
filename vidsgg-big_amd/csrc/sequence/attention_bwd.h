// Backward of the attention over ordered rows: two kernels, each with one side's gradients in registers and every product recomputed there, so that no
// sum crosses workgroups (seven products of 2 head_dim flops a pair where one kernel with atomics would do five, and the same bits every time).
//
//   dq:     lanes are queries.  S = K q, dP = V dO, dS = P (dP - delta), dq += K^T dS; the sums of dS along the diagonals of equal distance (the
//           bias table's gradient); first the rows' delta = dO . o, which it also leaves, with m and 1 / l, for the other kernel.
//   dk, dv: lanes are keys.  S = Q k, dP = dO v, dv += dO^T P, dk += Q^T dS, over all query heads of the key head.
//
// Half types round P and dS once each, to their own type, for the products that they enter (errors of the gradients 1.4 times those of an f32 computation rounded at its end, of the
// kind that the outputs' own rounding makes; a second part of each would be two more products of seven); scores, statistics, delta and every sum, the bias table's among them, are f32.
//
// Bound by vector instructions and the matrix instructions between them (16 heads of 64 with a learned bias over sequences of up to 2048 rows, bf16: dq and
// the diagonals' sums 207 us, dk and dv 187, the forward before them 182); with few sequences by the longest one's own chain of tiles (two packed rows of
// 4096 of documents, f16: 93 and 146 us, the forward 76).
#pragma once
#include "attention_fwd.h"

namespace {

// f16 holds dS scaled by a power of two: the largest so far at 2^14 .. 2^15, the accumulator rescaled when a larger one comes.  dS is as small as the loss's
// gradient makes it, and f16 ends at 2^-14; bf16 and f32 have f32's range.
template <typename T> struct GradScale {
    __device__ __forceinline__ void fit(f32x16&, f32x16*, int) {}
    __device__ __forceinline__ float back() const { return 1.f; }
};
template <> struct GradScale<f16_t> {
    float s = 0.f;
    __device__ __forceinline__ void fit(f32x16& v, f32x16* acc, int n) {
        float top = fabsf(v[0]);
        for (int e = 1; e < 16; ++e) top = fmaxf(top, fabsf(v[e]));
        if (__ballot(s == 0.f ? top > 0.f : top * s > 32768.f)) {
            if (__ballot(top == INFINITY)) {                    // of finite values: a row of Inf takes its neighbours in the wave nothing
                top = 0.f;
                for (int e = 0; e < 16; ++e) top = fmaxf(top, fabsf(v[e]) < INFINITY ? fabsf(v[e]) : 0.f);
            }
            for (int m = 32; m; m >>= 1) top = fmaxf(top, __shfl_xor(top, m));
            if (s == 0.f ? top > 0.f : top * s > 32768.f) {
                const float now = ldexpf(1.f, min(14 - ilogbf(top), 120));
                if (s != 0.f) {
                    const float c = now / s;
                    for (int d = 0; d < n; ++d) for (int e = 0; e < 16; ++e) acc[d][e] *= c;
                }
                s = now;
            }
        }
        for (int e = 0; e < 16; ++e) v[e] *= s == 0.f ? 1.f : s;
    }
    __device__ __forceinline__ float back() const { return s == 0.f ? 1.f : 1.f / s; }
};

struct BwdShape {
    int q_split, k_split;                                       // which form of the kernels (see BwdTile)
    int q_tiles, k_tiles;                                       // of a block's rows, of the longest sequence
    int q_pairs, k_pairs;                                       // (sequence, head), (sequence, key head)
    size_t q_lds, k_lds;
    size_t rows, q_ranges, k_ranges, bins, total;               // workspace: [3][n_head][n_q] -m, 2^P_LIFT / l, delta; document ranges; sums by distance
};

// SPLIT: for launches of few blocks.  A block then has 32 rows instead of 128, and its waves take the streamed tiles of the same rows in turn, each through
// LDS of its own; their sums are joined at the end, in order.  Not for f32s, where every wave would have to take its tiles apart by itself (clips of 8
// videos, 256 whole blocks: 93 and 74 us whole, 152 and 95 us split).
template <typename T, int HD, bool SPLIT, bool KV> struct BwdTile {
    static constexpr int ROWS = sizeof(T) == 4 || SPLIT || (KV && HD > 64) ? 32 : 64, SUBS = ROWS / 32;          // streamed rows of a tile
    typedef Tile<T, HD, ROWS> TL;
    static constexpr int WAVES = 4, BLOCK_ROWS = SPLIT ? 32 : 128, NW = SPLIT ? 1 : 4, NBUF = 2;
    static constexpr int TILE = TL::BYTES, BUF = 2 * TILE, STAGES = (SPLIT ? WAVES : 1) * NBUF * BUF;
    static constexpr int SIDE = KV ? 1024 : 256, SIDES = (SPLIT ? WAVES : 1) * NBUF * SIDE;            // beside a tile: the streamed queries' -m, 2^P_LIFT / l, delta, documents; keys' documents
    static constexpr int PAD = 33, JOIN = WAVES * HD * PAD * 4;
    static_assert(!SPLIT || (JOIN <= STAGES && STAGES <= 140 * 1024), "");
};
constexpr int DIAG_PAD = BIAS_PAD;                              // bins beyond the radius on both sides

// the place of a block among `pairs` x `tiles`, tiles of a pair on one XCD (see fwd_place)
__device__ __forceinline__ bool bwd_place(int pairs, int tiles, int& pair, int& tile) {
    const int xcd = blockIdx.x & 7, k = blockIdx.x >> 3;
    long id;
    if ((pairs & 7) == 0) id = (long)(xcd + 8 * (k / tiles)) * tiles + k % tiles;
    else {
        const long n = (long)pairs * tiles, q = n >> 3, rest = n & 7;
        id = xcd * q + min((long)xcd, rest) + k;
    }
    pair = (int)(id / tiles); tile = (int)(id % tiles);
    return pair < pairs;
}

// document range of the block's live lanes: [min of those >= 0, max], and of the wave's: [min with -1 for padding, max]
__device__ __forceinline__ void doc_bounds(int doc, bool live, int wave, int2* shared, int& wave_min, int& wave_max, int& block_min, int& block_max, int waves = 4) {
    int lo = live ? max(doc, -1) : 0x7fffffff, some = live && doc >= 0 ? doc : 0x7fffffff, most = live ? doc : -1;
    for (int m = 32; m; m >>= 1) { lo = min(lo, __shfl_xor(lo, m)); some = min(some, __shfl_xor(some, m)); most = max(most, __shfl_xor(most, m)); }
    wave_min = __builtin_amdgcn_readfirstlane(lo); wave_max = __builtin_amdgcn_readfirstlane(most);
    if ((threadIdx.x & 63) == 0) shared[wave] = make_int2(some, most);
    __syncthreads();
    block_min = shared[0].x; block_max = shared[0].y;
    for (int w = 1; w < waves; ++w) { block_min = min(block_min, shared[w].x); block_max = max(block_max, shared[w].y); }
}

// whether a lane of any of the block's four waves has `x`
__device__ __forceinline__ bool any_wave(bool x, int wave, int* shared) {
    x = __ballot(x) != 0;
    if ((threadIdx.x & 63) == 0) shared[wave] = x;
    wait_block();
    x = shared[0] | shared[1] | shared[2] | shared[3];
    wait_block();
    return x;
}


// Joins the waves' sums for the same 32 rows (`f` times each wave's own) through LDS and stores them as rows of T
template <typename T, typename B>
__device__ __forceinline__ void join_rows(char* lds, const f32x16* acc, float f, int n, int hd, T* out, long ld) {
    const int wave = threadIdx.x / 64, l = threadIdx.x & 63, hi = l >> 5, col = l & 31;
    float* const all = (float*)lds;
    __syncthreads();
    for (int d = 0; d < B::TL::HD / 32; ++d) for (int e = 0; e < 16; ++e) all[(wave * B::TL::HD + 32 * d + mfma_row(e, hi)) * B::PAD + col] = acc[d][e] * f;
    __syncthreads();
    for (int e = threadIdx.x; e < n * hd; e += 64 * B::WAVES) {
        const int r = e / hd, c = e % hd;
        float x = 0.f;
        for (int w = 0; w < B::WAVES; ++w) x += all[(w * B::TL::HD + c) * B::PAD + r];
        out[r * ld + c] = (T)x;
    }
}

// Adds the 32 x 32 sums of `v` along its diagonals to bins (a wave's own): lane c of column c, register e of key e.  Lane s takes column (s + key) mod 32 of
// every key, so that it holds diagonal -s where that did not wrap and 32 - s where it did.
__device__ __forceinline__ void add_diagonals(const f32x16& v, float* bins, int base /* d of key 0, column 0 */, int low /* d of bin 0 */) {
    const int lane = threadIdx.x & 63, s = lane & 31, hi = lane >> 5;
    float a = 0.f, b = 0.f;
    for (int e = 0; e < 16; ++e) {
        const int k = reg_row(e) + 4 * hi;
        const float x = __shfl(v[e], ((s + k) & 31) + 32 * hi);
        if (s + k < 32) a += x; else b += x;
    }
    a += __shfl_xor(a, 32);
    b += __shfl_xor(b, 32);
    if (hi == 0) {
        float* at = bins + base - s - low;
        at[0] += a;
        if (s) at[32] += b;                                     // (diagonal 32 has no element)
    }
}

// P reaches the product with dO as P 2^P_LIFT (f16 ends at 2^-14).  The lift goes with 1 / l, a power of two on a factor, and not into the exponent beside -m, where it would be
// rounded away once a row's scores pass 2^24 (biases of -1e9 and the like on all that a row sees).
template <typename T> constexpr float P_LIFT = 0.f;
template <> constexpr float P_LIFT<f16_t> = 14.f;

template <typename T, int HD, bool SPLIT>
__global__ __launch_bounds__(256, (SPLIT || HD > 96 || (sizeof(T) == 4 && HD > 32) ? 1 : 2)) void attn_bwd_q(bigc_seq_attn a, BwdShape sh, float* row_data, const int2* ranges, float* by_dist) {
    typedef BwdTile<T, HD, SPLIT, false> B;
    typedef typename B::TL TL;
    constexpr int DT = HD / 32, KEYS = B::ROWS, SUBS = B::SUBS, TILE = B::TILE, BUF = B::BUF;
    extern __shared__ __attribute__((aligned(16))) char lds[];
    __shared__ int2 shared_docs[4];
    __shared__ int shared_bad[4];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), lane = threadIdx.x & 63, col = lane & 31, hi = lane >> 5;
    if (a.zero_rest) zero_outside((T*)a.dq, a.lddq, a.hsdq, a.n_q, a.n_head, a.head_dim, a.q_off, a.n_seq, a.max_q);
    int pair, tile;
    if (!bwd_place(sh.q_pairs, sh.q_tiles, pair, tile)) return;
    if (a.causal) tile = sh.q_tiles - 1 - tile;                 // the longest first
    const int s = pair / a.n_head, head = pair % a.n_head, hk = head / (a.n_head / a.n_kv_head);
    const SeqSpan sp = seq_span(a, s);
    const int first = tile * B::BLOCK_ROWS, nb = a.d_rel_table ? 2 * a.bias_radius + 1 : 0, nbins = nb ? nb + 2 * DIAG_PAD : 0;
    float* const out_bins = nb ? by_dist + ((long)(s * sh.q_tiles + tile) * a.n_head + head) * nb : nullptr;
    if (first >= sp.nq) {
        for (int e = threadIdx.x; e < nb; e += 64 * B::WAVES) out_bins[e] = 0.f;
        return;
    }
    const int i0 = first + (SPLIT ? 0 : wave * 32), i = min(i0 + col, sp.nq - 1), shift = sp.nk - sp.nq, pos = i + shift;
    const bool live = i0 + col < sp.nq, wave_live = i0 < sp.nq;
    const long row = sp.q0 + i;
    const ScoreRule rule(a, T());
    const Reach reach(a);
    const int prefix = a.prefix_len ? min(a.prefix_len[s], sp.nk) : 0;
    LaneRow me;
    me.lo = reach.lo; me.hi = min(reach.hi, sp.nk - 1 - pos);
    me.prefix = prefix - pos; me.doc = 0; me.bias = 0;
    me.slope2 = rule.slopes ? a.slopes[head] * LOG2E : 0.f;

    char* const docs_lds = lds + B::STAGES;
    float* const biases = (float*)(docs_lds + (a.q_doc ? B::SIDES : 0));
    float* const all_bins = biases + (rule.table ? bias_entries(a) : 0);
    float* const bins = all_bins + wave * nbins;
    if (rule.table) load_biases(a, biases, head, 1);
    int doc_min = 0, doc_max = 0, block_doc_min = 0, block_doc_max = 0;
    if (a.q_doc) {
        me.doc = live ? a.q_doc[row] : -1;
        doc_bounds(me.doc, live, wave, shared_docs, doc_min, doc_max, block_doc_min, block_doc_max, B::WAVES);
    }
    __syncthreads();

    // the rows' statistics and delta
    typename Mat<T>::frag q[TL::STEPS], go[TL::STEPS];
    load_lane_rows<T, HD>(q, (const T*)a.q + row * a.ldq + head * a.hsq, live, a.head_dim);
    load_lane_rows<T, HD>(go, (const T*)a.d_o + row * a.lddo + head * a.hsdo, live, a.head_dim);
    const long rh = row * a.n_head + head;
    const float2 ml = live ? *(const float2*)(a.stats + 2 * rh) : make_float2(0.f, 0.f);
    // A lane without a query has P = 0 by a maximum of Inf: its scores, a bias at most, would otherwise have none taken off, and the table's sums add all lanes up.
    const float m = !live ? INFINITY : ml.x == -INFINITY ? 0.f : ml.x, inv_l = ml.y == 0.f ? 0.f : 1.f / ml.y;
    double total = 0.;                                          // (the table's gradient adds delta's error up over all keys)
    if (a.o32) {
        for (int c = 0; c < TL::STEPS; ++c)
            for (int e = 0; e < TL::E; ++e) {
                const int at = (2 * c + hi) * TL::E + e;
                if (live && at < a.head_dim) total += (double)(float)go[c][e] * a.o32[rh * a.head_dim + at];
            }
    } else {
        typename Mat<T>::frag o[TL::STEPS];
        load_lane_rows<T, HD>(o, (const T*)a.o + row * a.ldo + head * a.hso, live, a.head_dim);
        for (int c = 0; c < TL::STEPS; ++c)
            for (int e = 0; e < TL::E; ++e) total += (double)(float)go[c][e] * (float)o[c][e];
    }
    total += __shfl_xor(total, 32);
    float delta = (float)total;
    if (ml.y == 0.f) delta = 0.f;
    if (live && hi == 0 && (!SPLIT || wave == 0)) {
        const long plane = a.n_q * a.n_head, at = head * a.n_q + row;
        row_data[at] = -m; row_data[plane + at] = inv_l * (P_LIFT<T> == 0.f ? 1.f : 16384.f); row_data[2 * plane + at] = delta;
    }
    const float minus = -delta * inv_l;                         // dS = p (dP / l - delta / l)
    // Every other row's dP is taken negated: the matrix instructions cut off a sum's last bits downwards, and the table's gradient, which adds such errors up over all rows
    // and keys where dP - delta itself cancels, would have them all with one sign (2000 keys of 32 columns, 64 of
    // them near: f32 12e-6 of the table with one sign, 0.7e-6 with both; f16 1.9e-6 and 0.4e-6).
    const bool odd = col & 1;
    const float sign_l = odd ? -inv_l : inv_l;
    if (odd) for (int c = 0; c < TL::STEPS; ++c) go[c] = -go[c];

    TileList list;
    list.end = (sp.nk + KEYS - 1) / KEYS;
    list.ahead = (prefix + KEYS - 1) / KEYS;
    list.first = max(0, tile_floor((long)first + shift + reach.lo, KEYS));
    list.last = tile_floor((long)min(first + B::BLOCK_ROWS - 1, sp.nq - 1) + shift + reach.hi, KEYS);
    list.ranges = a.q_doc ? ranges + (long)s * ((a.max_k + 63) / 64) : nullptr;
    list.per64 = 64 / KEYS; list.doc_min = block_doc_min; list.doc_max = block_doc_max; list.stride = SPLIT ? B::WAVES : 1;
    list.wave_min = doc_min; list.wave_max = doc_max;
    const int p_min = min(i0, sp.nq - 1) + shift, p_max = min(i0 + 31, sp.nq - 1) + shift;

    const int sw = SPLIT ? 0 : wave;
    Stage<TL, B::NW> stage_k, stage_v;
    stage_k.init(a.ldk, a.head_dim, sw);
    stage_v.init(a.ldv, a.head_dim, sw);
    const T* const k_rows = (const T*)a.k + sp.k0 * a.ldk + hk * a.hsk;
    const T* const v_rows = (const T*)a.v + sp.k0 * a.ldv + hk * a.hsv;
    char* const mine = lds + (SPLIT ? wave * B::NBUF * BUF : 0);
    int* const docs = (int*)docs_lds + (SPLIT ? wave * B::NBUF * 64 : 0);
    const auto arrived = [&] { if (SPLIT) wait_copies(); else wait_block(); };
    const auto copy_tile = [&](int k, int buf) {
        stage_k.load(mine + buf * BUF, k_rows, k * KEYS, sp.nk, sw);
        stage_v.load(mine + buf * BUF + TILE, v_rows, k * KEYS, sp.nk, sw);
    };
    const auto copy_side = [&](int k, int buf) {
        if (a.q_doc && sw == 0)
            __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(a.k_doc + sp.k0 + min(k * KEYS + lane, sp.nk - 1)), LDS_PTR(void, docs + buf * 64), 4, 0, 0);
    };
    const auto finish_tile = [&](int buf) {
        stage_k.finish(mine + buf * BUF, sw);
        stage_v.finish(mine + buf * BUF + TILE, sw);
    };
    const int low = -a.bias_radius - DIAG_PAD;                  // d of the first bin

    f32x16 acc[DT];
    GradScale<T> scale;
    float below = 0.f, above = 0.f;                             // dS of distances at or beyond the radius, of 32 x 32s that lie there whole
    const auto pass = [&](auto careful_) {
        constexpr bool careful = decltype(careful_)::value;
        for (int d = 0; d < DT; ++d) for (int e = 0; e < 16; ++e) acc[d][e] = 0.f;
        scale = GradScale<T>();
        below = above = 0.f;
        for (int e = lane; e < nbins; e += 64) bins[e] = 0.f;
        list.restart();
        int k = list.next(SPLIT ? wave : 0), buf = 0;
        bool whole = list.whole;
        if (k < list.end) { copy_tile(k, 0); copy_side(k, 0); finish_tile(0); }
        arrived();
        while (k < list.end) {
            const int after = list.next(k + list.stride), other = buf ^ 1;
            const bool after_whole = list.whole;
            if (after < list.end) {
                copy_tile(after, other);
                copy_side(after, other);
            }
            const char* const kt = mine + buf * BUF;
            const char* const vt = kt + TILE;
            if constexpr (careful) {
                stage_k.clear_tail((char*)kt, sw);
                stage_v.clear_tail((char*)vt, sw);
                arrived();
            }
            const int kb = k * KEYS, ke = min(kb + KEYS, sp.nk), d_min = kb - p_max, d_max = kb + KEYS - 1 - p_min;
            const bool seen = wave_live && (kb < prefix || (d_max >= reach.lo && d_min <= reach.hi));
            bool full = kb + KEYS <= sp.nk && (ke <= prefix || (d_min >= reach.lo && d_max <= reach.hi));
            full &= whole;
            if (seen) {
                for (int u = 0; u < SUBS; ++u) {
                    f32x16 x, y, t;
                    for (int e = 0; e < 16; ++e) x[e] = y[e] = 0.f;
                    if constexpr (careful) {
                        add_products_seen<TL>(x, kt, 32 * u, q);
                        add_products_seen<TL>(y, vt, 32 * u, go);
                    } else {
                        add_products<TL>(x, kt, 32 * u, q);
                        add_products<TL>(y, vt, 32 * u, go);
                    }
                    const int d0 = kb + 32 * u + 4 * hi - pos;
                    const Linear sc = make_scores<T, true, true>(x, &t, rule, me, biases, d0, d_min + 32 * u, d_max - 32 * (SUBS - 1 - u));
                    if (!full) hide_scores<true>(x, sc, me, d0, a.q_doc ? docs + buf * 64 + 32 * u + 4 * hi : nullptr);
                    const float base = sc.c - m;
                    for (int e = 0; e < 16; ++e) {
                        const float p = __builtin_amdgcn_exp2f(fmaf(x[e], sc.a, base)), ds = p * fmaf(y[e], sign_l, minus);
                        x[e] = careful && (p == 0.f || !live) ? 0.f : ds;
                    }
                    if (nb) {
                        const int lo = d_min + 32 * u, up = d_max - 32 * (SUBS - 1 - u);
                        if (lo >= a.bias_radius || up <= -a.bias_radius) {
                            float sum = x[0];
                            for (int e = 1; e < 16; ++e) sum += x[e];
                            if (lo >= a.bias_radius) above += sum; else below += sum;
                        } else {
                            add_diagonals(x, bins, kb + 32 * u - (i0 + shift), low);
                        }
                    }
                    if (rule.cap) for (int e = 0; e < 16; ++e) x[e] = careful && x[e] == 0.f ? 0.f : x[e] * t[e];     // (the slope of a hidden place's score may be NaN)
                    scale.fit(x, acc, DT);
                    if constexpr (careful) accumulate_seen<TL>(acc, kt, 32 * u, x);
                    else accumulate<TL>(acc, kt, 32 * u, x);
                }
            }
            if (after < list.end) finish_tile(other);
            arrived();
            k = after; buf = other; whole = after_whole;
        }
    };
    pass(std::false_type());
    float check = 0.f;                                          // NaN or Inf: again, value by value (see attn_fwd)
    for (int d = 0; d < DT; ++d) for (int e = 0; e < 16; ++e) check += acc[d][e] * 0.f;
    if (SPLIT ? __ballot(check != 0.f && live) != 0 : any_wave(check != 0.f && live, wave, shared_bad)) pass(std::true_type());
    if (nb) {
        for (int w = 32; w; w >>= 1) { below += __shfl_xor(below, w); above += __shfl_xor(above, w); }
        if (lane == 0) { bins[0] += below; bins[nbins - 1] += above; }
        __syncthreads();
        for (int e = threadIdx.x; e < nb; e += 64 * B::WAVES) { // waves in order; the bins beyond the radius belong to the two ends
            float sum = 0.f;
            const int from = e == 0 ? 0 : e + DIAG_PAD, to = e == nb - 1 ? nbins : e + DIAG_PAD + 1;
            for (int w = 0; w < B::WAVES; ++w)
                for (int b = from; b < to; ++b) sum += all_bins[w * nbins + b];
            out_bins[e] = sum;
        }
    }
    const float f = a.scale * scale.back() * slope_unit<T>(rule);
    if constexpr (SPLIT) {
        join_rows<T, B>(lds, acc, f, min(32, sp.nq - first), a.head_dim, (T*)a.dq + (sp.q0 + first) * a.lddq + head * a.hsdq, a.lddq);
        return;
    }
    if (!live) return;
    for (int d = 0; d < DT; ++d)
        for (int g = 0; g < 4; ++g) {
            const int c = 32 * d + 8 * g + 4 * hi;
            if (c >= a.head_dim) continue;
            struct alignas(4 * sizeof(T)) Four { T v[4]; } z;
            for (int e = 0; e < 4; ++e) z.v[e] = (T)(acc[d][4 * g + e] * f);
            *(Four*)((T*)a.dq + row * a.lddq + head * a.hsdq + c) = z;
        }
}

template <typename T, int HD, bool SPLIT>
__global__ __launch_bounds__(256, (SPLIT || HD > 64 || sizeof(T) == 4 ? 1 : 2)) void attn_bwd_kv(bigc_seq_attn a, BwdShape sh, const float* row_data, const int2* ranges) {
    typedef BwdTile<T, HD, SPLIT, true> B;
    typedef typename B::TL TL;
    constexpr int DT = HD / 32, ROWS = B::ROWS, SUBS = B::SUBS, TILE = B::TILE, BUF = B::BUF;
    extern __shared__ __attribute__((aligned(16))) char lds[];
    __shared__ int2 shared_docs[4];
    __shared__ int shared_bad[4];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), lane = threadIdx.x & 63, col = lane & 31, hi = lane >> 5;
    if (a.zero_rest) {
        zero_outside((T*)a.dk, a.lddk, a.hsdk, a.n_k, a.n_kv_head, a.head_dim, a.k_off, a.n_seq, a.max_k);
        zero_outside((T*)a.dv, a.lddv, a.hsdv, a.n_k, a.n_kv_head, a.head_dim, a.k_off, a.n_seq, a.max_k);
    }
    int pair, tile;
    if (!bwd_place(sh.k_pairs, sh.k_tiles, pair, tile)) return;
    const int s = pair / a.n_kv_head, hk = pair % a.n_kv_head, group = a.n_head / a.n_kv_head;
    const SeqSpan sp = seq_span(a, s);
    const int first = tile * B::BLOCK_ROWS;
    if (first >= sp.nk) return;
    const int j0 = first + (SPLIT ? 0 : wave * 32), j = min(j0 + col, sp.nk - 1), shift = sp.nk - sp.nq;
    const bool live = j0 + col < sp.nk, wave_live = j0 < sp.nk;
    const long row = sp.k0 + j;
    const ScoreRule rule(a, T());
    const Reach reach(a);
    const int prefix = a.prefix_len ? min(a.prefix_len[s], sp.nk) : 0;
    LaneRow me;                                                 // streamed queries behind the last are hidden by their distance
    me.lo = j < prefix ? j - (sp.nk - 1) : max(reach.lo, j - (sp.nk - 1));
    me.hi = j < prefix ? 0x7fffffff : reach.hi;
    me.prefix = 0; me.doc = 0; me.bias = 0;
    // A lane without a key has P = 0 by an offset of -Inf: its score of 0 may be far above a row's maximum, and would set the wave's GradScale.
    const float none = live ? 0.f : -INFINITY;

    // LDS: two buffers of Q and dO tiles; per buffer the rows' -m, 2^P_LIFT / l, delta and documents (64 places each); biases of a head
    char* const mine = lds + (SPLIT ? wave * B::NBUF * BUF : 0);
    char* const side = lds + B::STAGES + (SPLIT ? wave * B::NBUF * B::SIDE : 0);
    float* const biases = (float*)(lds + B::STAGES + B::SIDES);
    const auto arrived = [&] { if (SPLIT) wait_copies(); else wait_block(); };
    int doc_min = 0, doc_max = 0, block_doc_min = 0, block_doc_max = 0;
    if (a.q_doc) {
        me.doc = live ? a.k_doc[row] : -1;
        doc_bounds(me.doc, live, wave, shared_docs, doc_min, doc_max, block_doc_min, block_doc_max, B::WAVES);
    }
    if (SPLIT && rule.table) { load_biases(a, biases, hk * group, group); __syncthreads(); }
    typename Mat<T>::frag kf[TL::STEPS], vf[TL::STEPS];
    load_lane_rows<T, HD>(kf, (const T*)a.k + row * a.ldk + hk * a.hsk, live, a.head_dim);
    load_lane_rows<T, HD>(vf, (const T*)a.v + row * a.ldv + hk * a.hsv, live, a.head_dim);

    // queries that see a key of the block: all, where it holds keys of the prefix
    TileList list;
    list.end = (sp.nq + ROWS - 1) / ROWS;
    list.ahead = first < prefix ? list.end : 0;
    list.first = max(0, tile_floor((long)first - reach.hi - shift, ROWS));
    list.last = tile_floor((long)min(first + B::BLOCK_ROWS - 1, sp.nk - 1) - reach.lo - shift, ROWS);
    list.ranges = a.q_doc ? ranges + (long)s * ((a.max_q + 63) / 64) : nullptr;
    list.per64 = 64 / ROWS; list.doc_min = block_doc_min; list.doc_max = block_doc_max; list.stride = SPLIT ? B::WAVES : 1;
    list.wave_min = doc_min; list.wave_max = doc_max;
    const int j_min = min(j0, sp.nk - 1), j_max = min(j0 + 31, sp.nk - 1);
    const long plane = a.n_q * a.n_head;
    const int sw = SPLIT ? 0 : wave;
    Stage<TL, B::NW> stage_q, stage_o;
    stage_q.init(a.ldq, a.head_dim, sw);
    stage_o.init(a.lddo, a.head_dim, sw);

    f32x16 dk[DT], dv[DT];
    GradScale<T> scale;
    const auto pass = [&](auto careful_) {
        constexpr bool careful = decltype(careful_)::value;
        for (int d = 0; d < DT; ++d) for (int e = 0; e < 16; ++e) dk[d][e] = dv[d][e] = 0.f;
        scale = GradScale<T>();
#pragma unroll 1
        for (int head = hk * group; head < (hk + 1) * group; ++head) {
            me.slope2 = rule.slopes ? a.slopes[head] * LOG2E : 0.f;
            if (SPLIT) me.bias = (head - hk * group) * bias_entries(a);
            else if (rule.table) { __syncthreads(); load_biases(a, biases, head, 1); }     // (readable behind the first wait below)
            const T* const q_rows = (const T*)a.q + sp.q0 * a.ldq + head * a.hsq;
            const T* const o_rows = (const T*)a.d_o + sp.q0 * a.lddo + head * a.hsdo;
            const auto copy_tile = [&](int k, int buf) {
                stage_q.load(mine + buf * BUF, q_rows, k * ROWS, sp.nq, sw);
                stage_o.load(mine + buf * BUF + TILE, o_rows, k * ROWS, sp.nq, sw);
            };
            const auto copy_side = [&](int k, int buf) {
                const int at = min(k * ROWS + lane, sp.nq - 1);                            // -m, 2^P_LIFT / l, delta and the documents, one a wave (SPLIT: all by each)
                for (int what = SPLIT ? 0 : wave; what < (a.q_doc ? 4 : 3); what += SPLIT ? 1 : 4) {
                    const void* from = what < 3 ? (const void*)(row_data + what * plane + head * a.n_q + sp.q0 + at) : (const void*)(a.q_doc + sp.q0 + at);
                    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)from, LDS_PTR(void, side + buf * B::SIDE + what * 256), 4, 0, 0);
                }
            };
            const auto finish_tile = [&](int buf) {
                stage_q.finish(mine + buf * BUF, sw);
                stage_o.finish(mine + buf * BUF + TILE, sw);
            };
            list.restart();
            int k = list.next(SPLIT ? (wave + head) % B::WAVES : 0), buf = 0;
            bool whole = list.whole;
            if (k < list.end) { copy_tile(k, 0); copy_side(k, 0); finish_tile(0); }
            arrived();
            while (k < list.end) {
                const int after = list.next(k + list.stride), other = buf ^ 1;
            const bool after_whole = list.whole;
                if (after < list.end) {
                    copy_tile(after, other);
                    copy_side(after, other);
                }
                const char* const qt = mine + buf * BUF;
                const char* const ot = qt + TILE;
                if constexpr (careful) {
                    stage_q.clear_tail((char*)qt, sw);
                    stage_o.clear_tail((char*)ot, sw);
                    arrived();
                }
                const int ib = k * ROWS, p_min = ib + shift, p_max = ib + ROWS - 1 + shift, d_min = j_min - p_max, d_max = j_max - p_min;
                const bool seen = wave_live && (j_min < prefix || (d_max >= reach.lo && d_min <= reach.hi));
                bool full = ib + ROWS <= sp.nq && (j_max < prefix || (d_min >= reach.lo && d_max <= reach.hi));
                full &= whole;
                if (seen) {
                    for (int u = 0; u < SUBS; ++u) {
                        const float* const rows = (const float*)(side + buf * B::SIDE) + 32 * u + 4 * hi;
                        f32x16 x, y, t;
                        for (int e = 0; e < 16; ++e) x[e] = y[e] = 0.f;
                        if constexpr (careful) {
                            add_products_seen<TL>(x, qt, 32 * u, kf);
                            add_products_seen<TL>(y, ot, 32 * u, vf);
                        } else {
                            add_products<TL>(x, qt, 32 * u, kf);
                            add_products<TL>(y, ot, 32 * u, vf);
                        }
                        const int d0 = j - shift - ib - 32 * u - 4 * hi;
                        const Linear sc = make_scores<T, false, true>(x, &t, rule, me, biases, d0, d_min + 32 * (SUBS - 1 - u), d_max - 32 * u);
                        if (!full) hide_scores<false>(x, sc, me, d0, a.q_doc ? (const int*)rows + 192 : nullptr);
                        const float offset = sc.c + none;
                        for (int g = 0; g < 4; ++g) {
                            const f32x4 m4 = *LDS_PTR(const f32x4, rows + 8 * g), l4 = *LDS_PTR(const f32x4, rows + 64 + 8 * g);
                            for (int e = 0; e < 4; ++e) {
                                const float p = __builtin_amdgcn_exp2f(fmaf(x[4 * g + e], sc.a, offset + m4[e]));
                                x[4 * g + e] = careful && p == 0.f ? 0.f : p * l4[e];
                            }
                        }
                        if constexpr (careful) accumulate_seen<TL>(dv, ot, 32 * u, x);
                        else accumulate<TL>(dv, ot, 32 * u, x);
                        for (int g = 0; g < 4; ++g) {
                            const f32x4 d4 = *LDS_PTR(const f32x4, rows + 128 + 8 * g);
                            for (int e = 0; e < 4; ++e) {
                                const float p = x[4 * g + e];
                                x[4 * g + e] = careful && p == 0.f ? 0.f : p * (y[4 * g + e] - d4[e]);
                            }
                        }
                        if (rule.cap) for (int e = 0; e < 16; ++e) x[e] = careful && x[e] == 0.f ? 0.f : x[e] * t[e];     // (the slope of a hidden place's score may be NaN)
                        scale.fit(x, dk, DT);
                        if constexpr (careful) accumulate_seen<TL>(dk, qt, 32 * u, x);
                        else accumulate<TL>(dk, qt, 32 * u, x);
                    }
                }
                if (after < list.end) finish_tile(other);
                arrived();
                k = after; buf = other; whole = after_whole;
            }
        }
    };
    pass(std::false_type());
    float check = 0.f;
    for (int d = 0; d < DT; ++d) for (int e = 0; e < 16; ++e) check += (dk[d][e] + dv[d][e]) * 0.f;
    if (SPLIT ? __ballot(check != 0.f && live) != 0 : any_wave(check != 0.f && live, wave, shared_bad)) pass(std::true_type());
    const float unlift = P_LIFT<T> == 0.f ? 1.f : 1.f / 16384.f, f = a.scale * scale.back() * unlift * slope_unit<T>(rule);
    if constexpr (SPLIT) {
        const int n = min(32, sp.nk - first);
        join_rows<T, B>(lds, dk, f, n, a.head_dim, (T*)a.dk + (sp.k0 + first) * a.lddk + hk * a.hsdk, a.lddk);
        join_rows<T, B>(lds, dv, unlift, n, a.head_dim, (T*)a.dv + (sp.k0 + first) * a.lddv + hk * a.hsdv, a.lddv);
        return;
    }
    if (!live) return;
    static_assert(P_LIFT<f16_t> == 14.f, "");
    for (int d = 0; d < DT; ++d)
        for (int g = 0; g < 4; ++g) {
            const int c = 32 * d + 8 * g + 4 * hi;
            if (c >= a.head_dim) continue;
            struct alignas(4 * sizeof(T)) Four { T v[4]; } z, w;
            for (int e = 0; e < 4; ++e) { z.v[e] = (T)(dk[d][4 * g + e] * f); w.v[e] = (T)(dv[d][4 * g + e] * unlift); }
            *(Four*)((T*)a.dk + row * a.lddk + hk * a.hsdk + c) = z;
            *(Four*)((T*)a.dv + row * a.lddv + hk * a.hsdv + c) = w;
        }
}

// The table's gradient of one head: the blocks' sums by distance, added in order by four threads a bin (eight loads on their way at a time), then
// the bins of every bucket by 32 threads each
__global__ __launch_bounds__(1024) void rel_table_grad(bigc_seq_attn a, const float* by_dist, int blocks) {
    extern __shared__ float total[];                            // [nb] sums, [nb] buckets, then [4][256]
    const int nb = 2 * a.bias_radius + 1, h = blockIdx.x, lane = threadIdx.x & 255, part = threadIdx.x >> 8;
    int* const bucket = (int*)(total + nb);
    float* const parts = total + 2 * nb;
    for (int b = threadIdx.x; b < nb; b += 1024) bucket[b] = min(max(a.rel_map[b], 0), a.n_bucket - 1);
    for (int b0 = 0; b0 < nb; b0 += 256) {
        const int b = b0 + lane;
        float x = 0.f;
        for (int k0 = part; k0 < blocks; k0 += 32) {
            float v[8];
            for (int i = 0; i < 8; ++i) v[i] = b < nb && k0 + 4 * i < blocks ? by_dist[((long)(k0 + 4 * i) * a.n_head + h) * nb + b] : 0.f;
            for (int i = 0; i < 8; ++i) x += v[i];
        }
        parts[part * 256 + lane] = x;
        __syncthreads();
        if (part == 0 && b < nb) total[b] = (parts[lane] + parts[256 + lane]) + (parts[512 + lane] + parts[768 + lane]);
        __syncthreads();
    }
    for (int k = threadIdx.x >> 5; k < a.n_bucket; k += 32) {
        float x = 0.f;
        for (int b = threadIdx.x & 31; b < nb; b += 32) x += bucket[b] == k ? total[b] : 0.f;
        for (int m = 16; m; m >>= 1) x += __shfl_xor(x, m);
        if ((threadIdx.x & 31) == 0) a.d_rel_table[(long)k * a.n_head + h] = x;
    }
}

BwdShape bwd_shape(const bigc_seq_attn& a) {
    BwdShape sh = {};
    const bool f32 = a.dtype == BIGC_F32;
    const int nb = a.rel_table ? 2 * a.bias_radius + 1 : 0, be = a.rel_table ? bias_entries(a) : 0, hd = tile_dim(a.head_dim), group = a.n_head / a.n_kv_head;
    sh.q_pairs = a.n_seq * a.n_head; sh.k_pairs = a.n_seq * a.n_kv_head;
    // Blocks of 128 rows until they are fewer than two a CU; then of 32 (two packed rows of 4096, f16, 256 blocks of dk, dv: 210 us whole, 150 us split).  The dk, dv
    // form keeps the biases of all heads of a group in LDS.
    sh.q_split = !f32 && (long)sh.q_pairs * cdiv(a.max_q, 128) < 512;
    sh.k_split = !f32 && (long)sh.k_pairs * cdiv(a.max_k, 128) < 512 && (long)group * be <= 4096;
    sh.q_tiles = cdiv(a.max_q, sh.q_split ? 32 : 128); sh.k_tiles = cdiv(a.max_k, sh.k_split ? 32 : 128);
    sh.q_lds = (sh.q_split ? 4 * 2 * (2 * tile_bytes(a, 32, false) + (a.q_doc ? 256 : 0)) : 2 * (2 * tile_bytes(a, f32 ? 32 : 64, f32) + (a.q_doc ? 256 : 0)))
             + sizeof(float) * (be + (a.d_rel_table ? 4 * (nb + 2 * DIAG_PAD) : 0));
    sh.k_lds = (sh.k_split ? 4 * 2 * (2 * tile_bytes(a, 32, false) + 1024) : 2 * (2 * tile_bytes(a, !f32 && hd <= 64 ? 64 : 32, f32) + 1024)) + sizeof(float) * be * (sh.k_split ? group : 1);
    // what does not fit with the bins of a wide bias goes whole
    if (sh.q_lds > 160 * 1024 - 512 && sh.q_split) {
        sh.q_split = 0; sh.q_tiles = cdiv(a.max_q, 128);
        sh.q_lds = 2 * (2 * tile_bytes(a, f32 ? 32 : 64, f32) + (a.q_doc ? 256 : 0)) + sizeof(float) * (be + (a.d_rel_table ? 4 * (nb + 2 * DIAG_PAD) : 0));
    }
    sh.rows = 0;
    sh.q_ranges = round_up(sizeof(float) * 3 * (size_t)a.n_q * a.n_head, 256);
    sh.k_ranges = sh.q_ranges + (a.q_doc ? round_up(sizeof(int2) * (size_t)a.n_seq * ((a.max_q + 63) / 64), 256) : 0);
    sh.bins = sh.k_ranges + (a.q_doc ? round_up(sizeof(int2) * (size_t)a.n_seq * ((a.max_k + 63) / 64), 256) : 0);
    sh.total = sh.bins + (a.d_rel_table ? round_up(sizeof(float) * (size_t)a.n_seq * sh.q_tiles * a.n_head * nb, 256) : 0);
    return sh;
}

template <typename T, int HD>
void launch_bwd(hipStream_t s, const bigc_seq_attn& a, const BwdShape& sh, char* ws) {
    float* rows = (float*)(ws + sh.rows);
    const long nq = (long)sh.q_pairs * sh.q_tiles, nk = (long)sh.k_pairs * sh.k_tiles;
    const int2 *kr = (const int2*)(ws + sh.k_ranges), *qr = (const int2*)(ws + sh.q_ranges);
    float* bins = (float*)(ws + sh.bins);
    constexpr bool CAN = sizeof(T) == 2;
    if (nq && a.n_q) {
        if (CAN && sh.q_split) attn_bwd_q<T, HD, CAN><<<(unsigned)nq, 256, sh.q_lds, s>>>(a, sh, rows, kr, bins);
        else attn_bwd_q<T, HD, false><<<(unsigned)nq, 256, sh.q_lds, s>>>(a, sh, rows, kr, bins);
    }
    if (nk && a.n_k) {
        if (CAN && sh.k_split) attn_bwd_kv<T, HD, CAN><<<(unsigned)nk, 256, sh.k_lds, s>>>(a, sh, rows, qr);
        else attn_bwd_kv<T, HD, false><<<(unsigned)nk, 256, sh.k_lds, s>>>(a, sh, rows, qr);
    }
}
template <typename T>
void launch_bwd_dim(hipStream_t s, const bigc_seq_attn& a, const BwdShape& sh, char* ws) {
    switch (tile_dim(a.head_dim)) {
        case 32: launch_bwd<T, 32>(s, a, sh, ws); break;
        case 64: launch_bwd<T, 64>(s, a, sh, ws); break;
        case 96: launch_bwd<T, 96>(s, a, sh, ws); break;
        default: launch_bwd<T, 128>(s, a, sh, ws); break;
    }
}
}  // namespace
