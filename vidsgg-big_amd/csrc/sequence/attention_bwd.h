// Backward of the attention over ordered rows: two kernels, each with one side's gradients in registers and every product recomputed there, so that no
// sum crosses workgroups (seven products of 2 head_dim flops a pair where one kernel with atomics would do five, and the same bits every time).
//
//   dq:     lanes are queries.  S = K q, dP = V dO, dS = P (dP - delta), dq += K^T dS; the sums of dS along the diagonals of equal distance (the
//           bias table's gradient); first the rows' delta = dO . o, which it also leaves, with m and 1 / l, for the other kernel.
//   dk, dv: lanes are keys.  S = Q k, dP = dO v, dv += dO^T P, dk += Q^T dS, over all query heads of the key head.
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
            for (int m = 32; m; m >>= 1) top = fmaxf(top, __shfl_xor(top, m));
            if (top > 0.f && top < INFINITY) {
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
    int q_tiles, k_tiles;                                       // of 128 rows, of the longest sequence
    int q_pairs, k_pairs;                                       // (sequence, head), (sequence, key head)
    size_t q_lds, k_lds;
    size_t rows, q_ranges, k_ranges, bins, total;               // workspace: [3][n_head][n_q] P_LIFT - m, 1 / l, delta; document ranges; sums by distance
};

template <typename T, int HD> struct BwdTile {
    static constexpr int KEYS = sizeof(T) == 4 ? 32 : 64;                       // streamed rows of the dq kernel
    static constexpr int ROWS = sizeof(T) == 2 && HD <= 64 ? 64 : 32;          // and of the dk, dv kernel
};
constexpr int DIAG_PAD = 64;                                    // bins beyond the radius on both sides: a 32 x 32 that touches the radius reaches so far

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
__device__ __forceinline__ void doc_bounds(int doc, bool live, int wave, int2* shared, int& wave_min, int& wave_max, int& block_min, int& block_max) {
    int lo = live ? max(doc, -1) : 0x7fffffff, some = live && doc >= 0 ? doc : 0x7fffffff, most = live ? doc : -1;
    for (int m = 32; m; m >>= 1) { lo = min(lo, __shfl_xor(lo, m)); some = min(some, __shfl_xor(some, m)); most = max(most, __shfl_xor(most, m)); }
    wave_min = __builtin_amdgcn_readfirstlane(lo); wave_max = __builtin_amdgcn_readfirstlane(most);
    if ((threadIdx.x & 63) == 0) shared[wave] = make_int2(some, most);
    __syncthreads();
    block_min = shared[0].x; block_max = shared[0].y;
    for (int w = 1; w < 4; ++w) { block_min = min(block_min, shared[w].x); block_max = max(block_max, shared[w].y); }
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

// a block's streamed tiles: those before `ahead`, or in [first, last], and of a document the block has
struct TileList {
    int end, ahead, first, last;
    const int2* ranges;                                         // by 64 rows, or null
    int per64, doc_min, doc_max;                                // tiles of 64 rows
    __device__ __forceinline__ int next(int k) const {
        if (k >= ahead && k < first) k = first;
        if (!ranges) return k >= end || (k >= ahead && k > last) ? end : k;
        while (k < end) {
            const int c = k + (int)(threadIdx.x & 63);
            bool ok = c < end && (c < ahead || (c >= first && c <= last));
            if (ok && ranges) {
                const int2 r = ranges[c / per64];
                ok = r.x <= doc_max && r.y >= doc_min;
            }
            const unsigned long long m = __ballot(ok);
            if (m) return __builtin_amdgcn_readfirstlane(k + (int)__builtin_ctzll(m));
            k += 64;
        }
        return end;
    }
};
__device__ __forceinline__ int tile_floor(long row, int rows) { return row < 0 ? -1 : (int)min(row / rows, 0x3fffffffl); }

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

template <typename T> constexpr float P_LIFT = 0.f;             // P reaches the product with dO as P 2^P_LIFT (f16 ends at 2^-14)
template <> constexpr float P_LIFT<f16_t> = 14.f;

template <typename T, int HD>
__global__ __launch_bounds__(256, (HD > 96 || (sizeof(T) == 4 && HD > 32) ? 1 : 2)) void attn_bwd_q(bigc_seq_attn a, BwdShape sh, float* row_data, const int2* ranges, float* by_dist) {
    constexpr int DT = HD / 32, KEYS = BwdTile<T, HD>::KEYS, SUBS = KEYS / 32;
    typedef Tile<T, HD, KEYS> TL;
    constexpr int TILE = TL::BYTES, BUF = 2 * TILE;
    extern __shared__ __attribute__((aligned(16))) char lds[];
    __shared__ int2 shared_docs[4];
    __shared__ int shared_bad[4];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), lane = threadIdx.x & 63, col = lane & 31, hi = lane >> 5;
    if (a.zero_rest) zero_outside((T*)a.dq, a.lddq, a.hsdq, a.n_q, a.n_head, a.head_dim, a.q_off, a.n_seq);
    int pair, tile;
    if (!bwd_place(sh.q_pairs, sh.q_tiles, pair, tile)) return;
    if (a.causal) tile = sh.q_tiles - 1 - tile;                 // the longest first
    const int s = pair / a.n_head, head = pair % a.n_head, hk = head / (a.n_head / a.n_kv_head);
    const SeqSpan sp = seq_span(a, s);
    const int first = tile * 128, nb = a.d_rel_table ? 2 * a.bias_radius + 1 : 0, nbins = nb ? nb + 2 * DIAG_PAD : 0;
    float* const out_bins = nb ? by_dist + ((long)(s * sh.q_tiles + tile) * a.n_head + head) * nb : nullptr;
    if (first >= sp.nq) {
        for (int e = threadIdx.x; e < nb; e += 256) out_bins[e] = 0.f;
        return;
    }
    const int i0 = first + wave * 32, i = min(i0 + col, sp.nq - 1), shift = sp.nk - sp.nq, pos = i + shift;
    const bool live = i0 + col < sp.nq, wave_live = i0 < sp.nq;
    const long row = sp.q0 + i;
    const ScoreRule rule(a, T());
    const Reach reach(a);
    const int prefix = a.prefix_len ? min(a.prefix_len[s], sp.nk) : 0;
    LaneRow me;
    me.lo = reach.lo; me.hi = min(reach.hi, sp.nk - 1 - pos);
    me.prefix = prefix - pos; me.doc = 0; me.bias = 0;
    me.slope2 = rule.slopes ? a.slopes[head] * LOG2E : 0.f;

    char* const docs_lds = lds + 2 * BUF;
    float* const biases = (float*)(docs_lds + (a.q_doc ? 512 : 0));
    float* const bins = biases + (rule.table ? 2 * a.bias_radius + 1 : 0) + wave * nbins;
    if (rule.table) load_biases(a, biases, head, 1);
    int doc_min = 0, doc_max = 0, block_doc_min = 0, block_doc_max = 0;
    if (a.q_doc) {
        me.doc = live ? a.q_doc[row] : -1;
        doc_bounds(me.doc, live, wave, shared_docs, doc_min, doc_max, block_doc_min, block_doc_max);
    }
    __syncthreads();

    // the rows' statistics and delta
    typename Mat<T>::frag q[TL::STEPS], go[TL::STEPS];
    load_lane_rows<T, HD>(q, (const T*)a.q + row * a.ldq + head * a.hsq, live, a.head_dim);
    load_lane_rows<T, HD>(go, (const T*)a.d_o + row * a.lddo + head * a.hsdo, live, a.head_dim);
    const long rh = row * a.n_head + head;
    const float2 ml = live ? *(const float2*)(a.stats + 2 * rh) : make_float2(0.f, 0.f);
    const float m = ml.x == -INFINITY ? 0.f : ml.x, inv_l = ml.y == 0.f ? 0.f : 1.f / ml.y;
    float delta = 0.f;
    if (a.o32) {
        for (int c = 0; c < TL::STEPS; ++c)
            for (int e = 0; e < TL::E; ++e) {
                const int at = (2 * c + hi) * TL::E + e;
                if (live && at < a.head_dim) delta += (float)go[c][e] * a.o32[rh * a.head_dim + at];
            }
    } else {
        typename Mat<T>::frag o[TL::STEPS];
        load_lane_rows<T, HD>(o, (const T*)a.o + row * a.ldo + head * a.hso, live, a.head_dim);
        for (int c = 0; c < TL::STEPS; ++c)
            for (int e = 0; e < TL::E; ++e) delta += (float)go[c][e] * (float)o[c][e];
    }
    delta += __shfl_xor(delta, 32);
    if (ml.y == 0.f) delta = 0.f;
    if (live && hi == 0) {
        const long plane = a.n_q * a.n_head, at = head * a.n_q + row;
        row_data[at] = P_LIFT<T> - m; row_data[plane + at] = inv_l; row_data[2 * plane + at] = delta;
    }
    const float minus = -delta * inv_l;                         // dS = p (dP / l - delta / l)

    TileList list;
    list.end = (sp.nk + KEYS - 1) / KEYS;
    list.ahead = (prefix + KEYS - 1) / KEYS;
    list.first = max(0, tile_floor((long)first + shift + reach.lo, KEYS));
    list.last = tile_floor((long)min(first + 127, sp.nq - 1) + shift + reach.hi, KEYS);
    list.ranges = a.q_doc ? ranges + (long)s * ((a.max_k + 63) / 64) : nullptr;
    list.per64 = 64 / KEYS; list.doc_min = block_doc_min; list.doc_max = block_doc_max;
    const int p_min = min(i0, sp.nq - 1) + shift, p_max = min(i0 + 31, sp.nq - 1) + shift;

    Stage<TL, 4> stage_k, stage_v;
    stage_k.init(a.ldk, a.head_dim, wave);
    stage_v.init(a.ldv, a.head_dim, wave);
    const T* const k_rows = (const T*)a.k + sp.k0 * a.ldk + hk * a.hsk;
    const T* const v_rows = (const T*)a.v + sp.k0 * a.ldv + hk * a.hsv;
    int* const docs = (int*)docs_lds;
    const auto copy_tile = [&](int k, int buf) {
        stage_k.load(lds + buf * BUF, k_rows, k * KEYS, sp.nk, wave);
        stage_v.load(lds + buf * BUF + TILE, v_rows, k * KEYS, sp.nk, wave);
        if (a.q_doc && wave == 0)
            __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(a.k_doc + sp.k0 + min(k * KEYS + lane, sp.nk - 1)), LDS_PTR(void, docs + buf * 64), 4, 0, 0);
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
        int k = list.next(0), buf = 0;
        const auto finish_tile = [&](int buf) { stage_k.finish(lds + buf * BUF, wave); stage_v.finish(lds + buf * BUF + TILE, wave); };
        if (k < list.end) { copy_tile(k, 0); finish_tile(0); }
        wait_block();
        while (k < list.end) {
            const int after = list.next(k + 1);
            if (after < list.end) copy_tile(after, buf ^ 1);
            const char* const kt = lds + buf * BUF;
            const char* const vt = kt + TILE;
            if constexpr (careful) {
                stage_k.clear_tail((char*)kt, wave);
                stage_v.clear_tail((char*)vt, wave);
                wait_block();
            }
            const int kb = k * KEYS, ke = min(kb + KEYS, sp.nk), d_min = kb - p_max, d_max = kb + KEYS - 1 - p_min;
            const bool seen = wave_live && (kb < prefix || (d_max >= reach.lo && d_min <= reach.hi));
            bool full = kb + KEYS <= sp.nk && (ke <= prefix || (d_min >= reach.lo && d_max <= reach.hi));
            if (a.q_doc && full) {
                const int2 r = list.ranges[kb / 64];
                full = __builtin_amdgcn_readfirstlane(r.x >= 0 && r.x == r.y && doc_min == r.x && doc_max == r.x);
            }
            if (seen) {
                for (int u = 0; u < SUBS; ++u) {
                    f32x16 x, y, t;
                    for (int e = 0; e < 16; ++e) x[e] = y[e] = 0.f;
                    for (int c = 0; c < TL::STEPS; ++c) x = Mat<T>::mul(rows_frag<TL>(kt, 32 * u, c), q[c], x);
                    for (int c = 0; c < TL::STEPS; ++c) y = Mat<T>::mul(rows_frag<TL>(vt, 32 * u, c), go[c], y);
                    const int d0 = kb + 32 * u + 4 * hi - pos;
                    const Linear sc = make_scores<T, true, true>(x, &t, rule, me, biases, d0, d_min + 32 * u, d_max - 32 * (SUBS - 1 - u));
                    if (!full) hide_scores<true>(x, sc, me, d0, a.q_doc ? docs + buf * 64 + 32 * u + 4 * hi : nullptr);
                    const float base = sc.c - m;
                    for (int e = 0; e < 16; ++e) {              // rows that are not there: 0 (1 / l is 0)
                        const float p = __builtin_amdgcn_exp2f(fmaf(x[e], sc.a, base)), ds = p * fmaf(y[e], inv_l, minus);
                        x[e] = careful && p == 0.f ? 0.f : ds;
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
                    if (rule.cap) for (int e = 0; e < 16; ++e) x[e] *= cap_slope<T>(t[e]);
                    scale.fit(x, acc, DT);
                    if constexpr (careful) accumulate_seen<TL>(acc, kt, 32 * u, x);
                    else accumulate<TL>(acc, kt, 32 * u, x);
                }
            }
            if (after < list.end) finish_tile(buf ^ 1);
            wait_block();
            k = after; buf ^= 1;
        }
    };
    pass(std::false_type());
    float check = 0.f;                                          // NaN or Inf: again, value by value (see attn_fwd)
    for (int d = 0; d < DT; ++d) for (int e = 0; e < 16; ++e) check += acc[d][e] * 0.f;
    if (any_wave(check != 0.f && live, wave, shared_bad)) pass(std::true_type());
    if (nb) {
        for (int w = 32; w; w >>= 1) { below += __shfl_xor(below, w); above += __shfl_xor(above, w); }
        if (lane == 0) { bins[0] += below; bins[nbins - 1] += above; }
        __syncthreads();
        const float* all = biases + nb;
        for (int e = threadIdx.x; e < nb; e += 256) {           // waves in order; the bins beyond the radius belong to the two ends
            float sum = 0.f;
            const int from = e == 0 ? 0 : e + DIAG_PAD, to = e == nb - 1 ? nbins : e + DIAG_PAD + 1;
            for (int w = 0; w < 4; ++w)
                for (int b = from; b < to; ++b) sum += all[w * nbins + b];
            out_bins[e] = sum;
        }
    }
    if (!live) return;
    const float f = a.scale * scale.back() * (rule.cap ? CAP_SLOPE<T> : 1.f);
    for (int d = 0; d < DT; ++d)
        for (int g = 0; g < 4; ++g) {
            const int c = 32 * d + 8 * g + 4 * hi;
            if (c >= a.head_dim) continue;
            struct alignas(4 * sizeof(T)) Four { T v[4]; } z;
            for (int e = 0; e < 4; ++e) z.v[e] = (T)(acc[d][4 * g + e] * f);
            *(Four*)((T*)a.dq + row * a.lddq + head * a.hsdq + c) = z;
        }
}

template <typename T, int HD>
__global__ __launch_bounds__(256, HD > 64 || sizeof(T) == 4 ? 1 : 2) void attn_bwd_kv(bigc_seq_attn a, BwdShape sh, const float* row_data, const int2* ranges) {
    constexpr int DT = HD / 32, ROWS = BwdTile<T, HD>::ROWS, SUBS = ROWS / 32;
    typedef Tile<T, HD, ROWS> TL;
    constexpr int TILE = TL::BYTES, BUF = 2 * TILE;
    extern __shared__ __attribute__((aligned(16))) char lds[];
    __shared__ int2 shared_docs[4];
    __shared__ int shared_bad[4];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), lane = threadIdx.x & 63, col = lane & 31, hi = lane >> 5;
    if (a.zero_rest) {
        zero_outside((T*)a.dk, a.lddk, a.hsdk, a.n_k, a.n_kv_head, a.head_dim, a.k_off, a.n_seq);
        zero_outside((T*)a.dv, a.lddv, a.hsdv, a.n_k, a.n_kv_head, a.head_dim, a.k_off, a.n_seq);
    }
    int pair, tile;
    if (!bwd_place(sh.k_pairs, sh.k_tiles, pair, tile)) return;
    const int s = pair / a.n_kv_head, hk = pair % a.n_kv_head, group = a.n_head / a.n_kv_head;
    const SeqSpan sp = seq_span(a, s);
    const int first = tile * 128;
    if (first >= sp.nk) return;
    const int j0 = first + wave * 32, j = min(j0 + col, sp.nk - 1), shift = sp.nk - sp.nq;
    const bool live = j0 + col < sp.nk, wave_live = j0 < sp.nk;
    const long row = sp.k0 + j;
    const ScoreRule rule(a, T());
    const Reach reach(a);
    const int prefix = a.prefix_len ? min(a.prefix_len[s], sp.nk) : 0;
    LaneRow me;                                                 // streamed queries behind the last are hidden by their distance
    me.lo = j < prefix ? j - (sp.nk - 1) : max(reach.lo, j - (sp.nk - 1));
    me.hi = j < prefix ? 0x7fffffff : reach.hi;
    me.prefix = 0; me.doc = 0; me.bias = 0;

    // LDS: two buffers of Q and dO tiles; per buffer the rows' -m, 1 / l, delta and documents (64 places each); biases of a head
    char* const side = lds + 2 * BUF;
    float* const biases = (float*)(side + 2 * 4 * 256);
    int doc_min = 0, doc_max = 0, block_doc_min = 0, block_doc_max = 0;
    if (a.q_doc) {
        me.doc = live ? a.k_doc[row] : -1;
        doc_bounds(me.doc, live, wave, shared_docs, doc_min, doc_max, block_doc_min, block_doc_max);
    }
    typename Mat<T>::frag kf[TL::STEPS], vf[TL::STEPS];
    load_lane_rows<T, HD>(kf, (const T*)a.k + row * a.ldk + hk * a.hsk, live, a.head_dim);
    load_lane_rows<T, HD>(vf, (const T*)a.v + row * a.ldv + hk * a.hsv, live, a.head_dim);

    // queries that see a key of the block: all, where it holds keys of the prefix
    TileList list;
    list.end = (sp.nq + ROWS - 1) / ROWS;
    list.ahead = first < prefix ? list.end : 0;
    list.first = max(0, tile_floor((long)first - reach.hi - shift, ROWS));
    list.last = tile_floor((long)min(first + 127, sp.nk - 1) - reach.lo - shift, ROWS);
    list.ranges = a.q_doc ? ranges + (long)s * ((a.max_q + 63) / 64) : nullptr;
    list.per64 = 64 / ROWS; list.doc_min = block_doc_min; list.doc_max = block_doc_max;
    const int j_min = min(j0, sp.nk - 1), j_max = min(j0 + 31, sp.nk - 1);
    const long plane = a.n_q * a.n_head;
    Stage<TL, 4> stage_q, stage_o;
    stage_q.init(a.ldq, a.head_dim, wave);
    stage_o.init(a.lddo, a.head_dim, wave);

    f32x16 dk[DT], dv[DT];
    GradScale<T> scale;
    const auto pass = [&](auto careful_) {
        constexpr bool careful = decltype(careful_)::value;
        for (int d = 0; d < DT; ++d) for (int e = 0; e < 16; ++e) dk[d][e] = dv[d][e] = 0.f;
        scale = GradScale<T>();
#pragma unroll 1
        for (int head = hk * group; head < (hk + 1) * group; ++head) {
            me.slope2 = rule.slopes ? a.slopes[head] * LOG2E : 0.f;
            if (rule.table) { __syncthreads(); load_biases(a, biases, head, 1); }          // (readable behind the first wait below)
            const T* const q_rows = (const T*)a.q + sp.q0 * a.ldq + head * a.hsq;
            const T* const o_rows = (const T*)a.d_o + sp.q0 * a.lddo + head * a.hsdo;
            const auto copy_tile = [&](int k, int buf) {
                stage_q.load(lds + buf * BUF, q_rows, k * ROWS, sp.nq, wave);
                stage_o.load(lds + buf * BUF + TILE, o_rows, k * ROWS, sp.nq, wave);
                const int at = min(k * ROWS + lane, sp.nq - 1);                            // one of -m, 1 / l, delta and the documents a wave
                if (wave < 3 || a.q_doc) {
                    const void* from = wave < 3 ? (const void*)(row_data + wave * plane + head * a.n_q + sp.q0 + at) : (const void*)(a.q_doc + sp.q0 + at);
                    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)from, LDS_PTR(void, side + (buf * 4 + wave) * 256), 4, 0, 0);
                }
            };
            int k = list.next(0), buf = 0;
            const auto finish_tile = [&](int buf) { stage_q.finish(lds + buf * BUF, wave); stage_o.finish(lds + buf * BUF + TILE, wave); };
            if (k < list.end) { copy_tile(k, 0); finish_tile(0); }
            wait_block();
            while (k < list.end) {
                const int after = list.next(k + 1);
                if (after < list.end) copy_tile(after, buf ^ 1);
                const char* const qt = lds + buf * BUF;
                const char* const ot = qt + TILE;
                if constexpr (careful) {
                    stage_q.clear_tail((char*)qt, wave);
                    stage_o.clear_tail((char*)ot, wave);
                    wait_block();
                }
                const int ib = k * ROWS, p_min = ib + shift, p_max = ib + ROWS - 1 + shift, d_min = j_min - p_max, d_max = j_max - p_min;
                const bool seen = wave_live && (j_min < prefix || (d_max >= reach.lo && d_min <= reach.hi));
                bool full = ib + ROWS <= sp.nq && (j_max < prefix || (d_min >= reach.lo && d_max <= reach.hi));
                if (a.q_doc && full) {
                    const int2 r = list.ranges[ib / 64];
                    full = __builtin_amdgcn_readfirstlane(r.x >= 0 && r.x == r.y && doc_min == r.x && doc_max == r.x);
                }
                if (seen) {
                    for (int u = 0; u < SUBS; ++u) {
                        const float* const rows = (const float*)(side + buf * 1024) + 32 * u + 4 * hi;
                        f32x16 x, y, t;
                        for (int e = 0; e < 16; ++e) x[e] = y[e] = 0.f;
                        for (int c = 0; c < TL::STEPS; ++c) x = Mat<T>::mul(rows_frag<TL>(qt, 32 * u, c), kf[c], x);
                        for (int c = 0; c < TL::STEPS; ++c) y = Mat<T>::mul(rows_frag<TL>(ot, 32 * u, c), vf[c], y);
                        const int d0 = j - shift - ib - 32 * u - 4 * hi;
                        const Linear sc = make_scores<T, false, true>(x, &t, rule, me, biases, d0, d_min + 32 * (SUBS - 1 - u), d_max - 32 * u);
                        if (!full) hide_scores<false>(x, sc, me, d0, a.q_doc ? (const int*)rows + 192 : nullptr);
                        for (int g = 0; g < 4; ++g) {
                            const f32x4 m4 = *LDS_PTR(const f32x4, rows + 8 * g), l4 = *LDS_PTR(const f32x4, rows + 64 + 8 * g);
                            for (int e = 0; e < 4; ++e) {
                                const float p = __builtin_amdgcn_exp2f(fmaf(x[4 * g + e], sc.a, sc.c + m4[e]));
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
                        if (rule.cap) for (int e = 0; e < 16; ++e) x[e] *= cap_slope<T>(t[e]);
                        scale.fit(x, dk, DT);
                        if constexpr (careful) accumulate_seen<TL>(dk, qt, 32 * u, x);
                        else accumulate<TL>(dk, qt, 32 * u, x);
                    }
                }
                if (after < list.end) finish_tile(buf ^ 1);
                wait_block();
                k = after; buf ^= 1;
            }
        }
    };
    pass(std::false_type());
    float check = 0.f;
    for (int d = 0; d < DT; ++d) for (int e = 0; e < 16; ++e) check += (dk[d][e] + dv[d][e]) * 0.f;
    if (any_wave(check != 0.f && live, wave, shared_bad)) pass(std::true_type());
    if (!live) return;
    const float unlift = P_LIFT<T> == 0.f ? 1.f : 1.f / 16384.f, f = a.scale * scale.back() * unlift * (rule.cap ? CAP_SLOPE<T> : 1.f);
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
    const bool split = a.dtype == BIGC_F32;
    const int nb = a.rel_table ? 2 * a.bias_radius + 1 : 0;
    sh.q_tiles = cdiv(a.max_q, 128); sh.k_tiles = cdiv(a.max_k, 128);
    sh.q_pairs = a.n_seq * a.n_head; sh.k_pairs = a.n_seq * a.n_kv_head;
    sh.q_lds = (size_t)4 * tile_bytes(a, split ? 32 : 64, split) + (a.q_doc ? 512 : 0) + sizeof(float) * (nb + (a.d_rel_table ? 4 * (nb + 2 * DIAG_PAD) : 0));
    sh.k_lds = (size_t)4 * tile_bytes(a, !split && tile_dim(a.head_dim) <= 64 ? 64 : 32, split) + 2048 + sizeof(float) * nb;
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
    if (nq && a.n_q) attn_bwd_q<T, HD><<<(unsigned)nq, 256, sh.q_lds, s>>>(a, sh, rows, (const int2*)(ws + sh.k_ranges), (float*)(ws + sh.bins));
    if (nk && a.n_k) attn_bwd_kv<T, HD><<<(unsigned)nk, 256, sh.k_lds, s>>>(a, sh, rows, (const int2*)(ws + sh.q_ranges));
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
