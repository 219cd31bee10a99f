// Forward of the attention over ordered rows.
#pragma once
#include "attention_tiles.h"

namespace {

// The streamed tiles of a block (or of one of its waves): of those with the right remainder by the stride the ones before `ahead` or in [first, last] whose documents
// the block has.  64 tiles' document ranges are looked at together and kept as bits, so that a step costs no trip to memory.
struct TileList {
    int end, ahead, first, last, stride;
    const int2* ranges;                                         // by 64 rows, or null
    int per64;                                                  // tiles of 64 rows
    int doc_min, doc_max, wave_min, wave_max;                   // the block's documents; the wave's, -1 with padding
    int base;                                                   // the tile that bit 0 stands for
    unsigned long long some, one;                               // tiles to visit; those of the wave's only document throughout
    bool whole;                                                 // of the tile found: nothing of it is another document's
    __device__ __forceinline__ void restart() { base = -1; some = one = 0; whole = true; }
    __device__ __forceinline__ int next(int k) {                // the first of k, k + stride, ... that is one
        if (k >= ahead && k < first) k += (first - k + stride - 1) / stride * stride;
        if (!ranges) return k >= end || (k >= ahead && k > last) ? end : k;
        while (k < end) {
            if (base < 0 || k >= base + 64 * stride) {
                base = k;
                const int c = k + (int)(threadIdx.x & 63) * stride;
                const bool in = c < end && (c < ahead || (c >= first && c <= last));
                const int2 r = in ? ranges[c / per64] : make_int2(0x7fffffff, -1);
                some = __ballot(r.x <= doc_max && r.y >= doc_min);
                one = __ballot(r.x >= 0 && r.x == r.y && r.x == wave_min && r.x == wave_max);
            }
            const int at = (k - base) / stride;
            const unsigned long long m = some >> at;
            if (m) {
                const int f = (int)__builtin_ctzll(m);
                whole = one >> (at + f) & 1;
                return __builtin_amdgcn_readfirstlane(k + f * stride);
            }
            k = base + 64 * stride;
        }
        return end;
    }
};
__device__ __forceinline__ int tile_floor(long row, int rows) { return row < 0 ? -1 : (int)min(row / rows, 0x3fffffffl); }

// How a forward call is cut.  A tile's rows are (query, head) pairs of one key head: `pack` of a group's heads side by side, so that a key is read once
// for all of them and a single token still fills rows.  many: four waves of 32 rows share every tile of keys; few (at most 32 rows in the
// longest sequence): the four waves take the key tiles of the same 32 rows in turn, each through LDS of its own.
struct FwdShape {
    int pack, sub;                                              // heads a tile packs; packs of a group
    int few, tiles, pairs;                                      // row tiles of the longest sequence; (sequence, key head, pack) triples
    int chunk, splits;                                          // keys a block takes; chunks of the longest sequence
    long blocks;
    size_t lds, part_o, part_ml, total;                         // LDS; workspace (document ranges first): offsets of the parts and its size
};

template <typename T, int HD, bool FEW> struct FwdTile {
    static constexpr int KEYS = FEW || sizeof(T) == 4 ? 32 : 64, SUBS = KEYS / 32;
    typedef Tile<T, HD, KEYS> TL;
    static constexpr int WAVES = FEW && TL::ROW > 256 ? 2 : 4;                      // (rows of 512 bytes: 160 KB of LDS hold the buffers of two)
    static constexpr int TILE = TL::BYTES, BUF = 2 * TILE;                          // bytes: one tile, K and V
    static constexpr int STAGES = (FEW ? WAVES : 1) * 2 * BUF;                      // two buffers of a block (many) or of each wave (few)
    static constexpr int DOCS = (FEW ? WAVES : 1) * 2 * 64 * 4;
};

// (pair, tile, chunk) of a block.  Blocks go to the eight XCDs in turn, each with an L2 of its own: all tiles of a pair, which read the same keys, are
// put on one XCD; the pairs go round the XCDs when they are a multiple of eight, else every XCD gets one piece of the list.
struct FwdPlace { int pair, tile, split; };
__device__ __forceinline__ FwdPlace fwd_place(const FwdShape& sh, bool last_first) {
    const int per = sh.tiles * sh.splits, xcd = blockIdx.x & 7, k = blockIdx.x >> 3;
    long id;
    if ((sh.pairs & 7) == 0) id = (long)(xcd + 8 * (k / per)) * per + k % per;
    else {
        const long q = sh.blocks >> 3, rest = sh.blocks & 7;
        id = xcd * q + min((long)xcd, rest) + k;
    }
    const int pair = (int)(id / per), in = (int)(id % per), tile = in % sh.tiles;
    return {pair, last_first ? sh.tiles - 1 - tile : tile, in / sh.tiles};
}

// rows of `t` outside every sequence -> 0: those before the first and behind the last, and what of a sequence lies behind its first `longest` rows, to which it is cut
template <typename T>
__device__ __forceinline__ void zero_outside(T* t, long ld, long hs, long n, int heads, int hd, const int* off, int n_seq, int longest) {
    const long first = n_seq ? min(max((long)off[0], 0l), n) : 0, last = n_seq ? min(max((long)off[n_seq], first), n) : 0;
    const int chunks = hd / (16 / (int)sizeof(T));
    const auto zero = [&](long r, long e) { *(uint4*)(t + r * ld + e / chunks % heads * hs + e % chunks * (16 / sizeof(T))) = make_uint4(0, 0, 0, 0); };
    const long all = (first + n - last) * heads * chunks;
    for (long e = (long)blockIdx.x * blockDim.x + threadIdx.x; e < all; e += (long)gridDim.x * blockDim.x) {
        const long r = e / chunks / heads;
        zero(r < first ? r : r - first + last, e);
    }
    for (int s = blockIdx.x; s < n_seq; s += gridDim.x) {
        const long begin = min(max((long)off[s], 0l), n), cut = begin + longest, rest = (min((long)off[s + 1], n) - cut) * heads * chunks;
        for (long e = threadIdx.x; e < rest; e += blockDim.x) zero(cut + e / chunks / heads, e);
    }
}

// Least and greatest document of every 64 keys (or queries) of a sequence; -1: padding among them
__global__ __launch_bounds__(256) void doc_ranges(bigc_seq_attn a, bool keys, int tiles, int2* ranges) {
    const long w = (long)blockIdx.x * 4 + threadIdx.x / 64;
    if (w >= (long)a.n_seq * tiles) return;
    const SeqSpan sp = seq_span(a, (int)(w / tiles));
    const int j = (int)(w % tiles) * 64 + (threadIdx.x & 63);
    int lo = 0x7fffffff, hi = -1;
    if (j < (keys ? sp.nk : sp.nq)) lo = hi = max(keys ? a.k_doc[sp.k0 + j] : a.q_doc[sp.q0 + j], -1);
    for (int m = 32; m; m >>= 1) { lo = min(lo, __shfl_xor(lo, m)); hi = max(hi, __shfl_xor(hi, m)); }
    if ((threadIdx.x & 63) == 0) ranges[w] = make_int2(lo, hi);
}

// place of a chunk's result for query i of sequence s, head h
__device__ __forceinline__ long part_row(const bigc_seq_attn& a, int split, int s, int i, int h) {
    return (((long)split * a.n_seq + s) * a.max_q + i) * a.n_head + h;
}

// One pass over the keys with the running maximum m and sum l of every row:  o = sum 2^(s - m) v / l.
//
// A row's maximum is only moved when a score passes it by more than SLACK, so that the accumulators are rarely rescaled (and p is what the backward's will be,
// bit for bit: next to another maximum the exponent is rounded differently); p then lies in (0, 2^SLACK].
// Bound: few rows over long caches by memory (48 tokens over caches of 1 to 16384, 8 key heads of 128, bf16: 378 us for 1.75 GB, 4.6 TB/s of the 5.1 that a
// copy reaches); many rows by vector instructions beside the matrix instructions (some ten a score of 2 head_dim x 2 flops; of a SIMD's cycles about half
// issue those and a quarter of them feed the matrix unit, the two adding up rather than overlapping): 8192 causal rows, 32 + 8 heads of 128, bf16: 790 us, 696
// TFLOP/s.
//
// p is rounded to the tensors' type for its product with v (the one rounding inside; sums and statistics are f32 before it).  f16 ends at 2^-14, so that its p is
// scaled by 2^LIFT (o32, which the exact gradient of the bias table is taken from, has p in two parts): with 2^(SLACK + LIFT) the largest, values down to 2^-39 of the row's largest still arrive.
template <typename T> constexpr float SLACK = 8.f;
template <> constexpr float SLACK<f16_t> = 4.f;
template <typename T> constexpr float LIFT = 0.f;
template <> constexpr float LIFT<f16_t> = 11.f;
// What p is taken beside: the maximum less the lift.  From 2^20 on, where f32 holds no more than eighths of a score and soon rounds the lift itself (by 5 at 2^27: p would pass f16's
// end), without one.  The running maximum, the chunks' and waves' statistics and `stats` are all this.
template <typename T> __device__ __forceinline__ float lifted(float top) { return LIFT<T> != 0.f && fabsf(top) < 0x1p20f ? top - LIFT<T> : top; }

// PARTS: of p (see o32).
template <typename T, int HD, bool FEW, int PARTS>
__global__ __launch_bounds__((64 * FwdTile<T, HD, FEW>::WAVES), (FEW || (sizeof(T) == 4 && HD > 96) ? 1 : 2)) void attn_fwd(bigc_seq_attn a, FwdShape sh, const int2* ranges, float* part_o, float2* part_ml) {
    typedef FwdTile<T, HD, FEW> F;
    typedef typename F::TL TL;
    constexpr int DT = HD / 32;
    extern __shared__ __attribute__((aligned(16))) char lds[];
    __shared__ int shared_bad[4];
    __shared__ int2 shared_docs[4];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), lane = threadIdx.x & 63, col = lane & 31, hi = lane >> 5;
    if (a.zero_rest) zero_outside((T*)a.o, a.ldo, a.hso, a.n_q, a.n_head, a.head_dim, a.q_off, a.n_seq, a.max_q);

    const FwdPlace at = fwd_place(sh, a.causal);
    if (at.pair >= sh.pairs) return;
    const int group = a.n_head / a.n_kv_head, s = at.pair / (a.n_kv_head * sh.sub), hk = at.pair / sh.sub % a.n_kv_head, head0 = hk * group + at.pair % sh.sub * sh.pack;
    const SeqSpan sp = seq_span(a, s);
    const int rows = sp.nq * sh.pack, first = at.tile * (FEW ? 32 : 128);
    if (first >= rows || (at.split && at.split * sh.chunk >= sp.nk)) return;

    // the wave's rows and the lane's
    const int t0 = first + (FEW ? 0 : wave * 32), t = t0 + col;
    const bool live = t < rows, wave_live = t0 < rows;
    const int i = min(t, rows - 1) / sh.pack, head = head0 + min(t, rows - 1) % sh.pack, shift = sp.nk - sp.nq;
    const long row = sp.q0 + i;
    const ScoreRule rule(a, T());
    const Reach reach(a);
    const int prefix = a.prefix_len ? min(a.prefix_len[s], sp.nk) : 0;
    const int pos = i + shift;
    LaneRow me;
    me.lo = reach.lo; me.hi = min(reach.hi, sp.nk - 1 - pos);   // keys behind the last are hidden by their distance
    me.prefix = prefix - pos;
    me.doc = 0;
    me.slope2 = rule.slopes ? a.slopes[head] * LOG2E : 0.f;
    me.bias = (head - head0) * bias_entries(a);

    char* docs_lds = lds + F::STAGES;
    float* biases = (float*)(docs_lds + (a.q_doc ? F::DOCS : 0));
    if (rule.table) load_biases(a, biases, head0, sh.pack);

    // the wave's and the block's range of positions, and of documents
    const int p_min = min(t0, rows - 1) / sh.pack + shift, p_max = min(t0 + 31, rows - 1) / sh.pack + shift;
    const int b_min = first / sh.pack + shift, b_max = min(first + (FEW ? 31 : 127), rows - 1) / sh.pack + shift;
    int doc_min = 0, doc_max = 0, block_doc_min = 0, block_doc_max = 0;
    if (a.q_doc) {
        me.doc = live ? a.q_doc[row] : -1;
        int lo = live ? max(me.doc, -1) : 0x7fffffff, some = me.doc >= 0 ? me.doc : 0x7fffffff, most = me.doc;
        for (int m = 32; m; m >>= 1) { lo = min(lo, __shfl_xor(lo, m)); some = min(some, __shfl_xor(some, m)); most = max(most, __shfl_xor(most, m)); }
        doc_min = __builtin_amdgcn_readfirstlane(lo); doc_max = __builtin_amdgcn_readfirstlane(most);
        if (lane == 0) shared_docs[wave] = make_int2(some, most);
        __syncthreads();
        block_doc_min = shared_docs[0].x; block_doc_max = shared_docs[0].y;
        for (int w = 1; w < F::WAVES; ++w) { block_doc_min = min(block_doc_min, shared_docs[w].x); block_doc_max = max(block_doc_max, shared_docs[w].y); }
    }
    if (rule.table) __syncthreads();

    // the block's key tiles: of its chunk those in the prefix or in reach of any of its rows
    const int tile_begin = at.split * sh.chunk / F::KEYS;
    TileList list;
    list.end = min((sp.nk + F::KEYS - 1) / F::KEYS, (at.split + 1) * (sh.chunk / F::KEYS));
    list.ahead = (prefix + F::KEYS - 1) / F::KEYS;
    list.first = max(0, tile_floor((long)b_min + reach.lo, F::KEYS));
    list.last = tile_floor((long)b_max + reach.hi, F::KEYS);
    list.stride = FEW ? F::WAVES : 1;
    list.ranges = a.q_doc ? ranges + (long)s * ((a.max_k + 63) / 64) : nullptr;
    list.per64 = 64 / F::KEYS; list.doc_min = block_doc_min; list.doc_max = block_doc_max; list.wave_min = doc_min; list.wave_max = doc_max;

    typename Mat<T>::frag q[TL::STEPS];
    Stage<TL, FEW ? 1 : F::WAVES> stage_k, stage_v;
    const int sw = FEW ? 0 : wave;
    stage_k.init(a.ldk, a.head_dim, sw);
    stage_v.init(a.ldv, a.head_dim, sw);
    const T* const k_rows = (const T*)a.k + sp.k0 * a.ldk + hk * a.hsk;
    const T* const v_rows = (const T*)a.v + sp.k0 * a.ldv + hk * a.hsv;
    char* const mine = lds + (FEW ? wave * 2 * F::BUF : 0);
    int* const my_docs = (int*)(docs_lds) + (FEW ? wave * 128 : 0);
    const auto copy_tile = [&](int k, int buf) {
        stage_k.load(mine + buf * F::BUF, k_rows, k * F::KEYS, sp.nk, sw);
        stage_v.load(mine + buf * F::BUF + F::TILE, v_rows, k * F::KEYS, sp.nk, sw);
        if (a.q_doc && sw == 0)
            __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(a.k_doc + sp.k0 + min(k * F::KEYS + lane, sp.nk - 1)),
                                             LDS_PTR(void, my_docs + buf * 64), 4, 0, 0);
    };
    const auto finish_tile = [&](int buf) {
        stage_k.finish(mine + buf * F::BUF, sw);
        stage_v.finish(mine + buf * F::BUF + F::TILE, sw);
    };
    const auto arrived = [&] { if (FEW) wait_copies(); else wait_block(); };

    f32x16 acc[DT];
    float m = -INFINITY, l = 0.f;
    const auto pass = [&](auto careful_) {
        constexpr bool careful = decltype(careful_)::value;
        for (int d = 0; d < DT; ++d) for (int e = 0; e < 16; ++e) acc[d][e] = 0.f;
        m = -INFINITY; l = 0.f;
        list.restart();
        int k = list.next(tile_begin + (FEW ? wave : 0)), buf = 0;
        bool whole = list.whole;
        if (k < list.end) copy_tile(k, 0);
        if (!careful) load_lane_rows<T, HD>(q, (const T*)a.q + row * a.ldq + head * a.hsq, live, a.head_dim);       // (behind the first tile's copies)
        if (k < list.end) finish_tile(0);
        arrived();
        while (k < list.end) {
            const int after = list.next(k + list.stride);
            const bool after_whole = list.whole;
            if (after < list.end) copy_tile(after, buf ^ 1);
            const char* const kt = mine + buf * F::BUF;
            const char* const vt = kt + F::TILE;
            if constexpr (careful) {                             // products with the zeros behind head_dim stay zeros
                stage_k.clear_tail((char*)kt, sw);
                if (FEW) wait_copies(); else wait_block();
            }
            // what the wave sees of the tile: nothing, everything, or part
            const int kb = k * F::KEYS, ke = min(kb + F::KEYS, sp.nk);
            const int d_min = kb - p_max, d_max = kb + F::KEYS - 1 - p_min;
            const bool seen = wave_live && (kb < prefix || (d_max >= reach.lo && d_min <= reach.hi));
            bool full = kb + F::KEYS <= sp.nk && (ke <= prefix || (d_min >= reach.lo && d_max <= reach.hi));
            full &= whole;
            if (seen) {
                for (int u = 0; u < F::SUBS; ++u) {                 // 32 keys at a time
                    f32x16 x;
                    for (int e = 0; e < 16; ++e) x[e] = 0.f;
                    if constexpr (careful) add_products_seen<TL>(x, kt, 32 * u, q);
                    else add_products<TL>(x, kt, 32 * u, q);
                    const int d0 = kb + 32 * u + 4 * hi - pos;
                    const Linear s = make_scores<T, true, false>(x, nullptr, rule, me, biases, d0, d_min + 32 * u, d_max - 32 * (F::SUBS - 1 - u));
                    if (!full) hide_scores<true>(x, s, me, d0, a.q_doc ? my_docs + buf * 64 + 32 * u + 4 * hi : nullptr);
                    float top = x[0];
                    if (s.a < 0.f) { for (int e = 1; e < 16; ++e) top = fminf(top, x[e]); }
                    else { for (int e = 1; e < 16; ++e) top = fmaxf(top, x[e]); }
                    top = fmaf(top, s.a, s.c);
                    top = lifted<T>(fmaxf(top, __shfl_xor(top, 32)));
                    const bool move = top > m + SLACK<T>;
                    if (__ballot(move)) {
                        const float c = move ? __builtin_amdgcn_exp2f(m - top) : 1.f;
                        m = move ? top : m;
                        l *= c;
                        for (int d = 0; d < DT; ++d) for (int e = 0; e < 16; ++e) acc[d][e] *= c;
                    }
                    const float base = s.c - (m == -INFINITY ? 0.f : m);
                    for (int e = 0; e < 16; ++e) x[e] = __builtin_amdgcn_exp2f(fmaf(x[e], s.a, base));
                    float sum = x[0];
                    for (int e = 1; e < 16; ++e) sum += x[e];
                    l += sum;
                    if constexpr (careful) accumulate_seen<TL>(acc, vt, 32 * u, x);
                    else accumulate<TL>(acc, vt, 32 * u, x, PARTS);
                }
            }
            if (after < list.end) finish_tile(buf ^ 1);
            arrived();
            k = after; buf ^= 1; whole = after_whole;
        }
    };
    pass(std::false_type());
    // NaN or Inf in the result: it may come from a hidden place (0 times it is NaN), so that the rows are done again value by value
    float check = 0.f;
    for (int d = 0; d < DT; ++d) for (int e = 0; e < 16; ++e) check += acc[d][e] * 0.f;
    bool bad = __ballot(check != 0.f && live) != 0;             // NaN differs from 0
    if (!FEW) {
        if (lane == 0) shared_bad[wave] = bad;
        wait_block();
        bad = shared_bad[0] | shared_bad[1] | shared_bad[2] | shared_bad[3];
        wait_block();
    }
    if (bad) pass(std::true_type());
    l += __shfl_xor(l, 32);

    if constexpr (FEW) {                                        // the waves' results of the same rows, joined in LDS: [wave][column][row], rows padded against bank conflicts
        constexpr int PAD = 33;
        __syncthreads();
        float* const o_all = (float*)lds;
        float* const ml_all = o_all + F::WAVES * HD * PAD;
        static_assert(!FEW || ((F::WAVES * (HD * PAD + 2 * 32)) * 4 <= F::STAGES && F::STAGES <= 136 * 1024), "");
        for (int d = 0; d < DT; ++d) for (int e = 0; e < 16; ++e) o_all[(wave * HD + 32 * d + mfma_row(e, hi)) * PAD + col] = acc[d][e];
        if (hi == 0) { ml_all[wave * 32 + col] = m; ml_all[(F::WAVES + wave) * 32 + col] = l; }
        __syncthreads();
        const int n = min(32, rows - first);
        for (int e = threadIdx.x; e < n * a.head_dim; e += 64 * F::WAVES) {
            const int r = e / a.head_dim, c = e % a.head_dim, rt = first + r;
            float top = -INFINITY, sum = 0.f, o = 0.f;
            for (int w = 0; w < F::WAVES; ++w) top = fmaxf(top, ml_all[w * 32 + r]);
            const float base = top == -INFINITY ? 0.f : top;
            for (int w = 0; w < F::WAVES; ++w) {
                const float f = __builtin_amdgcn_exp2f(ml_all[w * 32 + r] - base);
                if (f == 0.f && !isnan(ml_all[(F::WAVES + w) * 32 + r])) continue;
                sum += f * ml_all[(F::WAVES + w) * 32 + r];
                o += f * o_all[(w * HD + c) * PAD + r];
            }
            const long qrow = sp.q0 + rt / sh.pack;
            const int h = head0 + rt % sh.pack;
            const long rh = qrow * a.n_head + h;
            if (sh.splits > 1) {
                const long part = part_row(a, at.split, s, rt / sh.pack, h);
                part_o[part * a.head_dim + c] = o;
                if (c == 0) part_ml[part] = make_float2(top, sum);
            } else {
                o *= sum == 0.f ? 0.f : 1.f / sum;
                ((T*)a.o)[qrow * a.ldo + h * a.hso + c] = (T)o;
                if (a.o32) a.o32[rh * a.head_dim + c] = o;
                if (a.stats && c == 0) *(float2*)(a.stats + 2 * rh) = make_float2(top, sum);
            }
        }
        return;
    }
    if (!live) return;
    const long rh = row * a.n_head + head;
    if (sh.splits > 1) {
        const long part = part_row(a, at.split, s, i, head);
        float* o = part_o + part * a.head_dim;
        for (int d = 0; d < DT; ++d)
            for (int g = 0; g < 4; ++g) {
                const int c = 32 * d + 8 * g + 4 * hi;
                if (c < a.head_dim) *(float4*)(o + c) = make_float4(acc[d][4 * g], acc[d][4 * g + 1], acc[d][4 * g + 2], acc[d][4 * g + 3]);
            }
        if (hi == 0) part_ml[part] = make_float2(m, l);
        return;
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    for (int d = 0; d < DT; ++d)
        for (int g = 0; g < 4; ++g) {
            const int c = 32 * d + 8 * g + 4 * hi;
            if (c >= a.head_dim) continue;
            float y[4];
            T z[4];
            for (int e = 0; e < 4; ++e) { y[e] = acc[d][4 * g + e] * inv; z[e] = (T)y[e]; }
            struct alignas(4 * sizeof(T)) Four { T v[4]; };
            *(Four*)((T*)a.o + row * a.ldo + head * a.hso + c) = *(const Four*)z;
            if (a.o32) *(float4*)(a.o32 + rh * a.head_dim + c) = make_float4(y[0], y[1], y[2], y[3]);
        }
    if (a.stats && hi == 0) *(float2*)(a.stats + 2 * rh) = make_float2(m, l);
}

// Joins the chunks of every (row, head): a wave each
template <typename T>
__global__ __launch_bounds__(256) void attn_join(bigc_seq_attn a, FwdShape sh, const float* part_o, const float2* part_ml) {
    const long w = (long)blockIdx.x * 4 + threadIdx.x / 64;
    const int lane = threadIdx.x & 63, h = (int)(w % a.n_head);
    const long r = w / a.n_head;
    if (r >= (long)a.n_seq * a.max_q) return;
    const int s = (int)(r / a.max_q), i = (int)(r % a.max_q);
    const SeqSpan sp = seq_span(a, s);
    if (i >= sp.nq) return;
    const long row = sp.q0 + i, rh = row * a.n_head + h, part = part_row(a, 0, s, i, h), stride = part_row(a, 1, 0, 0, 0);
    const int n = max(1, (int)(((long)sp.nk + sh.chunk - 1) / sh.chunk));
    // 64 chunks at a time: their statistics by a lane each, then their sums with four loads on their way
    float top = -INFINITY, sum = 0.f, o[2] = {0.f, 0.f};
    for (int k0 = 0; k0 < n; k0 += 64) {
        const int m = min(64, n - k0);
        const float2 ml = lane < m ? part_ml[(k0 + lane) * stride + part] : make_float2(-INFINITY, 0.f);
        float now = ml.x;
        for (int w = 32; w; w >>= 1) now = fmaxf(now, __shfl_xor(now, w));
        now = fmaxf(now, top);
        const float base = now == -INFINITY ? 0.f : now, old = __builtin_amdgcn_exp2f(top - base);
        const float f = __builtin_amdgcn_exp2f(ml.x - base);
        float l = f == 0.f && !isnan(ml.y) ? 0.f : f * ml.y;
        for (int w = 32; w; w >>= 1) l += __shfl_xor(l, w);
        sum = sum * old + l;
        o[0] *= old; o[1] *= old;
        top = now;
        const bool none = f == 0.f && !isnan(ml.y);
        const unsigned long long skip = __ballot(none);
#pragma unroll 4
        for (int k = 0; k < m; ++k) {
            const float w = __shfl(f, k);
            for (int t = 0; t < 2; ++t) {
                const float x = lane + 64 * t < a.head_dim ? part_o[((k0 + k) * stride + part) * a.head_dim + lane + 64 * t] : 0.f;
                o[t] += skip >> k & 1 ? 0.f : w * x;
            }
        }
    }
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    for (int t = 0; t < 2; ++t) {
        const int c = lane + 64 * t;
        if (c >= a.head_dim) continue;
        ((T*)a.o)[row * a.ldo + h * a.hso + c] = (T)(o[t] * inv);
        if (a.o32) a.o32[rh * a.head_dim + c] = o[t] * inv;
    }
    if (a.stats && lane == 0) *(float2*)(a.stats + 2 * rh) = make_float2(top, sum);
}

template <typename T>
__global__ __launch_bounds__(256) void zero_rows(T* t, long ld, long hs, long n, int heads, int hd, const int* off, int n_seq, int longest) {
    zero_outside(t, ld, hs, n, heads, hd, off, n_seq, longest);
}

int tile_dim(int hd) { return hd <= 32 ? 32 : hd <= 64 ? 64 : hd <= 96 ? 96 : 128; }
// bytes of a tile in LDS (see Tile); split: f32 in its three parts
int tile_bytes(const bigc_seq_attn& a, int rows, bool split) {
    const int hd = tile_dim(a.head_dim), columns = hd == 96 ? 128 : hd;
    return (split ? 3 : 1) * (rows * columns * (split ? 2 : seq_size(a.dtype)) / 1024 * (1024 + 32));
}
size_t round_up(size_t n, size_t m) { return (n + m - 1) / m * m; }

FwdShape fwd_shape(const bigc_seq_attn& a) {
    FwdShape sh = {};
    const int group = a.n_head / a.n_kv_head, nb = a.rel_table ? bias_entries(a) : 0;
    // heads packed in a tile: all of a group; with a bias by distance as many as have their biases in 4096 LDS entries (one head's may be 4223)
    sh.pack = 1;
    for (int p = 1; p <= group; ++p)
        if (group % p == 0 && (long)p * nb <= 4096 && (long)p * a.max_q < (1l << 30)) sh.pack = p;
    sh.sub = group / sh.pack;
    sh.few = (long)a.max_q * sh.pack <= 32;
    const int rows = sh.few ? 32 : 128, keys = sh.few || a.dtype == BIGC_F32 ? 32 : 64;
    sh.tiles = (int)(((long)a.max_q * sh.pack + rows - 1) / rows);
    sh.pairs = a.n_seq * a.n_kv_head * sh.sub;
    // Keys a block takes.  While the row tiles alone do not give every CU its blocks (two; four for few rows, where a block is a stream through memory and sequences differ
    // in length: 48 tokens over caches of 1 to 16384, 8 key heads of 128: 377 us with four, 418 with eight, 471 with sixteen), the keys are cut: to blocks of
    // equal work over all sequences, none under 512 keys.
    const long row_blocks = (long)sh.pairs * sh.tiles, want = sh.few ? 1024 : 512;
    sh.chunk = (int)round_up(a.max_k > 0 ? a.max_k : 1, 64);
    if (row_blocks && row_blocks < want) {
        const long total = a.n_k < (long)a.n_seq * a.max_k ? a.n_k : (long)a.n_seq * a.max_k;        // keys of all sequences together, at most
        long chunk = (total * (row_blocks / a.n_seq) + want - 1) / want;
        chunk = chunk < 512 ? 512 : chunk;
        if (chunk < sh.chunk) sh.chunk = (int)round_up(chunk, 4 * keys);
    }
    sh.splits = (int)(((long)a.max_k + sh.chunk - 1) / sh.chunk);
    if (sh.splits < 1) sh.splits = 1;
    sh.blocks = row_blocks * sh.splits;
    const int tile = tile_bytes(a, keys, a.dtype == BIGC_F32 && !sh.few), row = tile_dim(a.head_dim) * seq_size(a.dtype);
    sh.lds = (size_t)(!sh.few ? 1 : row > 256 ? 2 : 4) * (4 * tile + (a.q_doc ? 512 : 0)) + sizeof(float) * sh.pack * nb;
    sh.part_o = a.q_doc ? round_up(sizeof(int2) * (size_t)a.n_seq * ((a.max_k + 63) / 64), 256) : 0;
    sh.part_ml = sh.part_o + (sh.splits > 1 ? round_up(sizeof(float) * (size_t)sh.splits * a.n_seq * a.max_q * a.n_head * a.head_dim, 256) : 0);
    sh.total = sh.part_ml + (sh.splits > 1 ? round_up(sizeof(float2) * (size_t)sh.splits * a.n_seq * a.max_q * a.n_head, 256) : 0);
    return sh;
}

// p in as many parts as the use of o32 needs, which the backward takes delta from: two, or for the f32 gradient of a bias table what adds up to f32's bits
// (f32s: products from zero for every 32 keys, see accumulate).  Two also for few rows whose keys are not cut (about 512 at most): the roundings of p do not average out over few
// keys (an f16 token over 257 keys: 1.3 - 1.5 times the error of o's own rounding with one part, 1.0 with two), and the time is the launch's; over long caches
// they do (1.1 - 1.4), and two parts cost 376 -> 386 us (48 tokens).
template <typename T, int HD>
void launch_fwd(hipStream_t s, const bigc_seq_attn& a, const FwdShape& sh, const int2* ranges, float* part_o, float2* part_ml) {
    const int threads = sh.few ? 64 * FwdTile<T, HD, true>::WAVES : 256;
    // (f32: few rows wait for memory, which is then copied as it is; many for the products, which then run on its parts)
    typedef typename std::conditional<std::is_same<T, float>::value, f32s, T>::type Many;
#define LAUNCH(PARTS) do { \
        if (sh.few) attn_fwd<T, HD, true, (sizeof(T) == 4 ? 1 : PARTS)><<<(unsigned)sh.blocks, threads, sh.lds, s>>>(a, sh, ranges, part_o, part_ml); \
        else attn_fwd<Many, HD, false, PARTS><<<(unsigned)sh.blocks, threads, sh.lds, s>>>(a, sh, ranges, part_o, part_ml); \
    } while (0)
    if constexpr (sizeof(T) == 4) { LAUNCH(2); return; }
    else {
        if (!a.o32 && !(sh.few && sh.splits == 1)) LAUNCH(1);
        else if (std::is_same<T, bf16_t>::value && a.o32 && a.rel_table) LAUNCH((std::is_same<T, bf16_t>::value ? 3 : 2));
        else LAUNCH(2);
    }
#undef LAUNCH
}
template <typename T>
void launch_fwd_dim(hipStream_t s, const bigc_seq_attn& a, const FwdShape& sh, const int2* ranges, float* part_o, float2* part_ml) {
    switch (tile_dim(a.head_dim)) {
        case 32: launch_fwd<T, 32>(s, a, sh, ranges, part_o, part_ml); break;
        case 64: launch_fwd<T, 64>(s, a, sh, ranges, part_o, part_ml); break;
        case 96: launch_fwd<T, 96>(s, a, sh, ranges, part_o, part_ml); break;
        default: launch_fwd<T, 128>(s, a, sh, ranges, part_o, part_ml); break;
    }
}
}  // namespace
