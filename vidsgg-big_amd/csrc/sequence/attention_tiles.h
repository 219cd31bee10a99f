// The parts that the attention kernels share: tiles of rows in LDS, matrix fragments, and the scores of a tile.
//
// Every kernel keeps one side of the attention in lanes (32 rows a wave, a row a lane and its twin 32 lanes on) and streams the other side through LDS:
// the product of a streamed row-major tile (A operand, 32 rows) with the lanes' side (B operand) leaves element (streamed row, lane's row) in
// register r of lane l at streamed row (r & 3) + 8 (r >> 2) + 4 (l >> 5).  That is already the B operand of the next product, whose A operand is the
// streamed tile TRANSPOSED -- the order of a contraction is free, so the transposed tile is read in the register's order of rows and no value
// changes lanes between the two products.
#pragma once
#include "sequence.h"
#include <math.h>
#include <type_traits>

namespace {

typedef __attribute__((ext_vector_type(8))) bf16_t bf16x8;
typedef __attribute__((ext_vector_type(8))) f16_t f16x8;
typedef __attribute__((ext_vector_type(4))) short s16x4;
typedef __attribute__((ext_vector_type(4))) int i32x4;

#define LDS_PTR(T, ...) ((__attribute__((address_space(3))) T*)(__VA_ARGS__))

constexpr float LOG2E = 1.44269504088896340736f;

// Matrix instructions by type: f16 / bf16 contract 16 rows a step, f32 two.
template <typename T> struct Mat;
template <> struct Mat<bf16_t> {
    typedef bf16x8 frag;
    static __device__ __forceinline__ f32x16 mul(frag a, frag b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
};
template <> struct Mat<f16_t> {
    typedef f16x8 frag;
    static __device__ __forceinline__ f32x16 mul(frag a, frag b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
};
template <> struct Mat<float> {
    typedef f32x4 frag;                                         // four steps of two: lane l's four values go with l's twin's four
    static __device__ __forceinline__ f32x16 mul(frag a, frag b, f32x16 c) {
        c = mfma32(a.x, b.x, c);
        c = mfma32(a.y, b.y, c);
        c = mfma32(a.z, b.z, c);
        return mfma32(a.w, b.w, c);
    }
};

// f32 whose products run on the bf16 matrix instructions: a value is the sum of three bf16 (its first, second and third eight bits: the parts are cut
// off, not rounded, so that nothing is lost), a product of two the sum of the six of their parts' products that reach 2^-16 of it; what is left out is under
// 2^-21, on average 2^-24, of the product.  192 cycles for 16 steps of a 32 x 32 product, where the f32 instructions take 512; no range is lost (bf16 has f32's).
struct f32s {
    float x;
    f32s() = default;
    __device__ __forceinline__ f32s(float y) : x(y) {}
    __device__ __forceinline__ operator float() const { return x; }
};
struct Parts {
    bf16x8 h, m, l;
    __device__ __forceinline__ float operator[](int e) const { return (float)h[e] + (float)m[e] + (float)l[e]; }
    __device__ __forceinline__ Parts operator-() const { return {-h, -m, -l}; }
};
// two values' parts, in pairs
__device__ __forceinline__ void split_pair(float a, float b, unsigned& h, unsigned& m, unsigned& l) {
    constexpr unsigned HIGH = 0xffff0000u, BOTH = 0x07060302u;
    const float ra = a - __uint_as_float(__float_as_uint(a) & HIGH), rb = b - __uint_as_float(__float_as_uint(b) & HIGH);
    const float sa = ra - __uint_as_float(__float_as_uint(ra) & HIGH), sb = rb - __uint_as_float(__float_as_uint(rb) & HIGH);
    h = __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), BOTH);
    m = __builtin_amdgcn_perm(__float_as_uint(rb), __float_as_uint(ra), BOTH);
    l = __builtin_amdgcn_perm(__float_as_uint(sb), __float_as_uint(sa), BOTH);
}
// The same for four values that may be Inf or NaN, which are their own first part: looked for at a fourth of the cost of taking care of them
__device__ __forceinline__ void split_four(f32x4 v, unsigned* h, unsigned* m, unsigned* l) {
    split_pair(v.x, v.y, h[0], m[0], l[0]);
    split_pair(v.z, v.w, h[1], m[1], l[1]);
    const float odd = fmaf(v.x, 0.f, fmaf(v.y, 0.f, fmaf(v.z, 0.f, v.w * 0.f)));
    if (__ballot(odd != 0.f)) {
        for (int p = 0; p < 2; ++p) {
            const float a = v[2 * p], b = v[2 * p + 1];
            const unsigned keep = (isfinite(a) ? 0xffffu : 0u) | (isfinite(b) ? 0xffff0000u : 0u);
            m[p] &= keep;
            l[p] &= keep;
            if (isnan(a)) h[p] |= 0x40u;
            if (isnan(b)) h[p] |= 0x400000u;
        }
    }
}
template <> struct Mat<f32s> {
    typedef Parts frag;
    static __device__ __forceinline__ f32x16 mul(const frag& a, const frag& b, f32x16 c) {
        return Mat<bf16_t>::mul(a.h, b.h, mul_rest(a, b, c));
    }
    static __device__ __forceinline__ f32x16 mul_rest(const frag& a, const frag& b, f32x16 c) {                 // all but the largest
        c = Mat<bf16_t>::mul(a.l, b.h, c);
        c = Mat<bf16_t>::mul(a.h, b.l, c);
        c = Mat<bf16_t>::mul(a.m, b.m, c);
        c = Mat<bf16_t>::mul(a.m, b.h, c);
        return Mat<bf16_t>::mul(a.h, b.m, c);
    }
};

// A tile of ROWS rows of HD columns in LDS, as the copies of 64 lanes x 16 bytes lay it down: copy b holds rows b, b + B, b + 2 B, ... one after the other
// (B copies in all, 1024 bytes each, 32 bytes apart).  Eight rows' chunks of one column, which a row-major fragment reads together, and four rows' pairs
// of chunks, which a transposed one does, then lie in different banks, and the place of a fragment is the lane's own plus a constant -- an address register for
// each kind of fragment and no arithmetic in the loops (chunks swizzled by row, which do the same for the banks, took one per fragment, and spilled).
// 96 columns lie in rows of 128.
template <typename T_, int HD_, int ROWS_>
struct Tile {
    typedef T_ T;
    static constexpr int HD = HD_, ROWS = ROWS_;
    static constexpr int E = 16 / (int)sizeof(T), ROW = (HD == 96 ? 128 : HD) * (int)sizeof(T), CH = ROW / 16, STEPS = HD / E / 2;      // chunk's elements; bytes and chunks of a row; fragments of it
    static constexpr int B = ROWS * ROW / 1024, PITCH = 1024 + 32, BYTES = B * PITCH;
    static_assert(B >= 2 && B <= 16 && 32 % B == 0 && ROWS % B == 0, "");
    static __device__ __forceinline__ int place(int row, int chunk) { return row % B * PITCH + row / B * ROW + chunk * 16; }
};

// f32s: a tile of each part
template <int HD_, int ROWS_>
struct Tile<f32s, HD_, ROWS_> {
    typedef f32s T;
    typedef Tile<bf16_t, HD_, ROWS_> Part;
    static constexpr int HD = HD_, ROWS = ROWS_, E = Part::E, ROW = Part::ROW, STEPS = Part::STEPS, BYTES = 3 * Part::BYTES;
};

// A operand, row-major: rows row0 .. row0 + 31 (row0 a multiple of 32), columns of step `s`
template <typename TL>
__device__ __forceinline__ typename Mat<typename TL::T>::frag rows_frag(const char* tile, int row0, int s) {
    const int l = threadIdx.x & 63;
    if constexpr (std::is_same<typename TL::T, f32s>::value) {
        typedef typename TL::Part P;
        return {rows_frag<P>(tile, row0, s), rows_frag<P>(tile + P::BYTES, row0, s), rows_frag<P>(tile + 2 * P::BYTES, row0, s)};
    } else
    return *LDS_PTR(const typename Mat<typename TL::T>::frag, tile + TL::place(l & 31, l >> 5) + (row0 / TL::B * TL::ROW + 32 * s));
}

// x += the products of 32 streamed rows with the lanes' rows.  f32s: the small products of all columns first, so that the sum is rounded at its full size once
// a step and not six times (o over 2048 keys of 64 columns: error 4.5e-7 of its size otherwise, 3.0e-7 so, in the same time).
template <typename TL>
__device__ __forceinline__ void add_products(f32x16& x, const char* tile, int row0, const typename Mat<typename TL::T>::frag* lanes) {
    if constexpr (std::is_same<typename TL::T, f32s>::value) {
        for (int c = 0; c < TL::STEPS; ++c) x = Mat<f32s>::mul_rest(rows_frag<TL>(tile, row0, c), lanes[c], x);
        for (int c = 0; c < TL::STEPS; ++c) x = Mat<bf16_t>::mul(rows_frag<typename TL::Part>(tile, row0, c), lanes[c].h, x);
    } else
    for (int c = 0; c < TL::STEPS; ++c) x = Mat<typename TL::T>::mul(rows_frag<TL>(tile, row0, c), lanes[c], x);
}

// The same for tiles or lanes that may hold Inf (x was 0 before).  f32s: Inf times a second or third part that is 0 is NaN where Inf times the value is Inf; the products of the
// first parts, which no nonzero value lacks, have then what the sum comes to.
template <typename TL>
__device__ __forceinline__ void add_products_seen(f32x16& x, const char* tile, int row0, const typename Mat<typename TL::T>::frag* lanes) {
    add_products<TL>(x, tile, row0, lanes);
    if constexpr (std::is_same<typename TL::T, f32s>::value) {
        f32x16 first;
        for (int e = 0; e < 16; ++e) first[e] = 0.f;
        for (int c = 0; c < TL::STEPS; ++c) first = Mat<bf16_t>::mul(rows_frag<typename TL::Part>(tile, row0, c), lanes[c].h, first);
        for (int e = 0; e < 16; ++e) x[e] = isnan(x[e]) ? first[e] : x[e];
    }
}

// A operand, transposed: columns col0 .. col0 + 31, the 16 rows from row0 on (a multiple of 16) in the order in which a product's registers 8 u .. 8 u + 7
// hold them (half types)
template <typename TL>
__device__ __forceinline__ typename Mat<typename TL::T>::frag cols_frag(const char* tile, int row0, int col0) {
    const int l = threadIdx.x & 63, i = l & 15, r = 4 * (l >> 5) + (i >> 2);           // lanes 4 k .. 4 k + 3 of 16 point at row k's 16 columns, and get a column of the four rows each
    const char* const at = tile + TL::place(r, ((l >> 4) & 1) * 2 + ((i >> 1) & 1)) + (i & 1) * 8;
    const int first = row0 % TL::B * TL::PITCH + row0 / TL::B * TL::ROW + col0 * 2, second = (row0 + 8) % TL::B * TL::PITCH + (row0 + 8) / TL::B * TL::ROW + col0 * 2;
    static_assert(8 % TL::B == 0 || TL::B == 16, "");                                  // row0 and row0 + 8 add to a lane's place without a carry
    union { s16x4 v[2]; typename Mat<typename TL::T>::frag f; } u;
    u.v[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(LDS_PTR(s16x4, at + first));
    u.v[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(LDS_PTR(s16x4, at + second));
    return u.f;
}

// acc[d columns of a block of 32][lane's row] += sum over the 32 streamed rows from row0 of tile^T x values; `values` in a product's register order.
// Half types round the values; what that leaves goes through further products (of k parts 2^-8k (bf16) or 2^-11k (f16) of a value remain).
template <typename TL>
__device__ __forceinline__ void accumulate(f32x16* acc, const char* tile, int row0, const f32x16& v, int parts = 1) {
    typedef typename TL::T T;
    if constexpr (std::is_same<T, f32s>::value) {
        typedef typename TL::Part P;
        Parts b[2];
        for (int u = 0; u < 2; ++u) {
            union { unsigned w[4]; bf16x8 f; } h, m, l;
            for (int e = 0; e < 4; ++e) split_pair(v[8 * u + 2 * e], v[8 * u + 2 * e + 1], h.w[e], m.w[e], l.w[e]);
            b[u] = {h.f, m.f, l.f};
        }
        // parts > 1: the 32 rows' sum from zero, small products first, then one addition to what has come so far, whose size has one rounding instead of twelve
        for (int dt = 0; dt < TL::HD / 32; ++dt) {
            f32x16 sum;
            for (int e = 0; e < 16; ++e) sum[e] = parts > 1 ? 0.f : acc[dt][e];
            Parts t[2];
            for (int u = 0; u < 2; ++u) {
                t[u] = {cols_frag<P>(tile, row0 + 16 * u, 32 * dt), cols_frag<P>(tile + P::BYTES, row0 + 16 * u, 32 * dt), cols_frag<P>(tile + 2 * P::BYTES, row0 + 16 * u, 32 * dt)};
                sum = Mat<f32s>::mul_rest(t[u], b[u], sum);
            }
            for (int u = 0; u < 2; ++u) sum = Mat<bf16_t>::mul(t[u].h, b[u].h, sum);
            for (int e = 0; e < 16; ++e) acc[dt][e] = parts > 1 ? acc[dt][e] + sum[e] : sum[e];
        }
    } else if constexpr (sizeof(T) == 4) {
        const int l = threadIdx.x & 63, hi = l >> 5, c = l & 31;
        for (int r = 0; r < 16; ++r) {
            const int row = mfma_row(r, 0);                     // + 4 (l >> 5), without a carry
            const char* const at = tile + TL::place(4 * hi, c >> 2) + (c & 3) * 4 + (row0 + row) % TL::B * TL::PITCH + (row0 + row) / TL::B * TL::ROW;
            for (int dt = 0; dt < TL::HD / 32; ++dt) acc[dt] = mfma32(*LDS_PTR(const float, at + 128 * dt), v[r], acc[dt]);
        }
    } else {
        typename Mat<T>::frag b[2];
        for (int e = 0; e < 8; ++e) { b[0][e] = (T)v[e]; b[1][e] = (T)v[8 + e]; }
        for (int u = 0; u < 2; ++u)
            for (int dt = 0; dt < TL::HD / 32; ++dt) acc[dt] = Mat<T>::mul(cols_frag<TL>(tile, row0 + 16 * u, 32 * dt), b[u], acc[dt]);
        if (parts == 1) return;
        f32x16 rest = v;
#pragma unroll 1
        for (int k = 1; k < parts; ++k) {
            for (int u = 0; u < 2; ++u)
                for (int e = 0; e < 8; ++e) { rest[8 * u + e] -= (float)b[u][e]; b[u][e] = (T)rest[8 * u + e]; }
            for (int u = 0; u < 2; ++u)
                for (int dt = 0; dt < TL::HD / 32; ++dt) acc[dt] = Mat<T>::mul(cols_frag<TL>(tile, row0 + 16 * u, 32 * dt), b[u], acc[dt]);
        }
    }
}

// The same, one value at a time: a value of 0 takes no part, whatever its row of the tile holds.  For the calls whose tiles hold NaN or Inf in hidden places.
template <typename TL>
__device__ __forceinline__ void accumulate_seen(f32x16* acc, const char* tile, int row0, const f32x16& v) {
    typedef typename TL::T T;
    const int l = threadIdx.x & 63, hi = l >> 5;
#pragma unroll 1
    for (int r = 0; r < 16; ++r) {
        float mine = v[0];
        for (int q = 1; q < 16; ++q) mine = r == q ? v[q] : mine;
#pragma unroll 1
        for (int half = 0; half < 2; ++half) {
            const float p = __shfl(mine, (l & 31) + 32 * half);
            const int row = row0 + mfma_row(r, half);
            for (int dt = 0; dt < TL::HD / 32; ++dt)
                for (int e = 0; e < 16; ++e) {
                    const int col = 32 * dt + mfma_row(e, hi);
                    float x;
                    if constexpr (std::is_same<T, f32s>::value) {
                        typedef typename TL::Part P;
                        const char* const at = tile + P::place(row, 0) + col * 2;
                        x = (float)*LDS_PTR(const bf16_t, at) + (float)*LDS_PTR(const bf16_t, at + P::BYTES) + (float)*LDS_PTR(const bf16_t, at + 2 * P::BYTES);
                    } else {
                        x = (float)*LDS_PTR(const T, tile + TL::place(row, 0) + col * (int)sizeof(T));
                    }
                    acc[dt][e] += p != 0.f ? p * x : 0.f;
                }
        }
    }
}

// B operand: the lane's row, all steps, from memory (zeros behind head_dim and for rows that are not there)
template <typename T, int HD>
__device__ __forceinline__ void load_lane_rows(typename Mat<T>::frag* f, const T* row, bool live, int hd) {
    const int hi = (threadIdx.x & 63) >> 5;
    if constexpr (std::is_same<T, f32s>::value) {
        for (int s = 0; s < HD / 16; ++s) {
            const int c = 16 * s + 8 * hi;
            union { unsigned w[4]; bf16x8 f; } h, m, l;
            for (int q = 0; q < 2; ++q)
                split_four(live && c < hd ? *(const f32x4*)((const float*)row + c + 4 * q) : f32x4{0.f, 0.f, 0.f, 0.f}, h.w + 2 * q, m.w + 2 * q, l.w + 2 * q);
            f[s] = {h.f, m.f, l.f};
        }
        return;
    }
    constexpr int E = 16 / (int)sizeof(T);
    if constexpr (!std::is_same<T, f32s>::value)
    for (int s = 0; s < HD / E / 2; ++s) {
        const int c = (2 * s + hi) * E;
        union { i32x4 raw; typename Mat<T>::frag f; } u;
        u.raw = live && c < hd ? *(const i32x4*)(row + c) : i32x4{0, 0, 0, 0};
        f[s] = u.f;
    }
}

// Copies tiles into LDS straight from memory, 16 bytes a lane; NW waves share the work.  A lane's offset from the tile's first row is the same for every
// tile that is whole.  Behind head_dim the columns repeat the row's first chunk (their products are with zeros, or not stored).
template <typename TL, int NW>
struct Stage {
    typedef typename TL::T T;
    static constexpr int N = TL::B / NW;
    static_assert(TL::B % NW == 0, "");
    unsigned off;                                               // of the first copy's rows; copy i's lie i NW rows on
    long step;                                                  // bytes from row to row
    int row, chunk, hd;                                         // the lane's place in the first copy

    __device__ __forceinline__ void init(long ld, int head_dim, int wave) {
        const int lane = threadIdx.x & 63;
        step = ld * (long)sizeof(T);
        hd = head_dim;
        row = lane / TL::CH * TL::B + wave;
        chunk = lane % TL::CH;
        off = (unsigned)(row * step) + (chunk * TL::E < hd ? chunk : 0) * 16;
    }
    // rows row0 .. row0 + ROWS - 1 of the n from first_row on: those behind the last repeat it (n > 0)
    __device__ __forceinline__ void load(char* tile, const T* first_row, int row0, int n, int wave) const {
        const char* from = (const char*)first_row + row0 * step;
        if (row0 + TL::ROWS <= n) {
            for (int i = 0; i < N; ++i)
                __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(from + i * NW * step + off), LDS_PTR(void, tile + (i * NW + wave) * TL::PITCH), 16, 0, 0);
        } else {
            for (int i = 0; i < N; ++i) {
                const int r = min(row + i * NW, n - 1 - row0);
                __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(from + r * step + (chunk * TL::E < hd ? chunk : 0) * 16),
                                                 LDS_PTR(void, tile + (i * NW + wave) * TL::PITCH), 16, 0, 0);
            }
        }
    }
    // what is left to do between the copies' arrival and the barrier
    __device__ __forceinline__ void finish(char*, int) const {}
    // zeros behind head_dim (for tiles that may hold Inf, which a product with 0 would make NaN)
    __device__ __forceinline__ void clear_tail(char* tile, int wave) const {
        if (chunk * TL::E < hd) return;
        for (int i = 0; i < N; ++i) *LDS_PTR(i32x4, tile + (i * NW + wave) * TL::PITCH + (threadIdx.x & 63) * 16) = i32x4{0, 0, 0, 0};
    }
};

// f32s: through registers, where the values fall into their parts; a thread has 16 bytes of a row at a time
template <int HD, int ROWS, int NW>
struct Stage<Tile<f32s, HD, ROWS>, NW> {
    typedef typename Tile<f32s, HD, ROWS>::Part P;
    static constexpr int PER_ROW = HD / 4, N = ROWS * PER_ROW / (64 * NW);
    static_assert(ROWS * PER_ROW % (64 * NW) == 0, "");
    long step;
    int hd;
    f32x4 v[N];
    __device__ __forceinline__ int row_of(int i, int wave) const { return ((i * NW + wave) * 64 + (int)(threadIdx.x & 63)) / PER_ROW; }
    __device__ __forceinline__ int col_of(int i, int wave) const { return ((i * NW + wave) * 64 + (int)(threadIdx.x & 63)) % PER_ROW * 4; }
    __device__ __forceinline__ void init(long ld, int head_dim, int) { step = ld; hd = head_dim; }
    __device__ __forceinline__ void load(char*, const f32s* first_row, int row0, int n, int wave) {
        for (int i = 0; i < N; ++i) {
            const int r = min(row0 + row_of(i, wave), n - 1), c = col_of(i, wave);
            v[i] = c < hd ? *(const f32x4*)((const float*)first_row + r * step + c) : f32x4{0.f, 0.f, 0.f, 0.f};
        }
    }
    __device__ __forceinline__ void finish(char* tile, int wave) const {
        typedef __attribute__((ext_vector_type(2))) unsigned u32x2;
        for (int i = 0; i < N; ++i) {
            unsigned h[2], m[2], l[2];
            split_four(v[i], h, m, l);
            char* const at = tile + P::place(row_of(i, wave), 0) + col_of(i, wave) * 2;
            *LDS_PTR(u32x2, at) = u32x2{h[0], h[1]};
            *LDS_PTR(u32x2, at + P::BYTES) = u32x2{m[0], m[1]};
            *LDS_PTR(u32x2, at + 2 * P::BYTES) = u32x2{l[0], l[1]};
        }
    }
    __device__ __forceinline__ void clear_tail(char*, int) const {}
};

// own copies have arrived / and everybody's, and nobody reads the buffer any more that the next copies go to
__device__ __forceinline__ void wait_copies() { asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory"); }
__device__ __forceinline__ void wait_block() {
    wait_copies();
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

// ---- scores -----------------------------------------------------------------------------------------------------------------------------

// What every score of a call has in common; scores are kept times log2 e (exp is then one instruction).  Without a bias by distance a score is linear,
// a v + c, in a value v: the product itself, or what the cap makes of it.
constexpr float COARSE_CAP = 64.f, MAX_CAP = 0x1p100f;         // (a larger cap leaves every score under 2^88 as it is)
struct ScoreRule {
    float a, c;
    float cap_in, cap_y;                                        // 2 scale log2 e / cap: the argument of tanh doubled, for 2^x; scale / cap
    bool cap, coarse, slopes, table;                            // coarse: see cap_values
    int radius;
    template <typename T> __device__ __forceinline__ ScoreRule(const bigc_seq_attn& q, T)
        : a(q.scale * LOG2E), c(0.f), cap_in(0.f), cap_y(0.f), cap(q.softcap > 0.f && q.softcap < MAX_CAP), coarse(sizeof(T) < 4 && q.softcap <= COARSE_CAP), slopes(q.slopes != nullptr), table(q.rel_table != nullptr), radius(q.bias_radius) {
        if (!cap) return;
        cap_in = 2.f * q.scale / q.softcap * LOG2E;
        cap_y = q.scale / q.softcap;
        a = q.softcap * LOG2E;
        if (coarse) { c = a; a = -2.f * a; }
    }
};

// The capped products' values.  f32: v = tanh y, small arguments through the odd series (to y^13: 2^-26 of the value at 0.5), the others with a division in full.
// Half types under caps of up to 64 (coarse): v = 1 / (e^2y + 1), tanh y = 1 - 2 v -- its error is a step of 1, not of the value, so that a score is off by up to 2^-23 of the
// cap: 8e-6 at 64, which scores of half operands live with, 0.1 at a million.  Larger caps: v = tanh y, by the series to y^7 up to 0.25, where both are off by 2^-21 of the value.
// KEEP: the cap's slopes 1 - tanh^2 too, coarse a fourth of them (slope_unit).
template <typename T, bool KEEP>
__device__ __forceinline__ void cap_values(f32x16& x, f32x16* slopes, const ScoreRule& r) {
    if (sizeof(T) < 4 && r.coarse) {
        for (int e = 0; e < 16; ++e) {
            const float v = __builtin_amdgcn_rcpf(__builtin_amdgcn_exp2f(x[e] * r.cap_in) + 1.f);
            if (KEEP) (*slopes)[e] = v - v * v;
            x[e] = v;
        }
        return;
    }
    for (int e = 0; e < 16; ++e) {
        const float y = x[e] * r.cap_y, z = y * y, f = __builtin_amdgcn_exp2f(x[e] * r.cap_in) + 1.f;
        float v;
        if (sizeof(T) < 4) {
            const float p = y * (1.f + z * (-1.f / 3 + z * (2.f / 15 + z * (-17.f / 315))));
            v = fabsf(y) < 0.25f ? p : 1.f - 2.f * __builtin_amdgcn_rcpf(f);
        } else {
            const float p = 1.f + z * (-1.f / 3 + z * (2.f / 15 + z * (-17.f / 315 + z * (62.f / 2835 + z * (-1382.f / 155925 + z * (21844.f / 6081075))))));
            v = fabsf(y) < 0.5f ? y * p : 1.f - 2.f / f;
        }
        if (KEEP) (*slopes)[e] = 1.f - v * v;
        x[e] = v;
        if (sizeof(T) < 4) __builtin_amdgcn_sched_barrier(0);    // one value after the other: side by side they would take registers that the other calls' loop is short of
    }
}
template <typename T> __device__ __forceinline__ float slope_unit(const ScoreRule& r) { return sizeof(T) < 4 && r.cap && r.coarse ? 4.f : 1.f; }

// What a call lets a row see, by d = key - position of the query: [lo, hi] (wide enough for any two int32 places), and a prefix
struct Reach {
    int lo, hi;
    __device__ __forceinline__ Reach(const bigc_seq_attn& a) {
        lo = a.window_left < 0 ? -0x7fffffff : -a.window_left;
        hi = a.causal ? 0 : a.window_right < 0 ? 0x7fffffff : a.window_right;
        if (a.causal && a.window_right >= 0) hi = 0;
    }
};

// A lane's row.  LANE_IS_QUERY: the key at distance d is seen when lo <= d <= hi or d < prefix; else (the lane is a key) when lo <= d <= hi.
struct LaneRow {
    int lo, hi, prefix, doc;
    float slope2;                                               // slope log2 e
    int bias;                                                   // first entry of its head's biases by distance
};

// Bias by distance of `heads` heads from h0 on, times log2 e: the lowest finite value stays finite (it hides nothing), -inf stays -inf.  Beyond the radius the ends
// go on for BIAS_PAD entries on both sides, as far as a 32 x 32 that touches the radius reaches: the registers' entries then lie at constants from the lane's.
constexpr int BIAS_PAD = 64;
__host__ __device__ __forceinline__ int bias_entries(const bigc_seq_attn& a) { return 2 * (a.bias_radius + BIAS_PAD) + 1; }
__device__ __forceinline__ void load_biases(const bigc_seq_attn& a, float* biases, int h0, int heads) {
    const int nb = bias_entries(a), r = a.bias_radius;
    for (int e = threadIdx.x; e < heads * nb; e += blockDim.x) {
        const int at = min(max(e % nb - BIAS_PAD, 0), 2 * r);
        const float b = a.rel_table[(long)min(max(a.rel_map[at], 0), a.n_bucket - 1) * a.n_head + h0 + e / nb];
        const float s = b * LOG2E;
        biases[e] = isinf(s) && !isinf(b) ? copysignf(3.402823466e38f, b) : s;
    }
}

// place of register e's streamed row among the lane's half of 32, without the 4 (l >> 5)
__device__ __forceinline__ constexpr int reg_row(int e) { return (e & 3) + 8 * (e >> 2); }

// Products of 32 streamed rows with the lanes' rows -> values v with score = a v + c (c the lane's own).  d0: d of register 0; streamed keys count d up,
// streamed queries down.  d_min, d_max: the least and the greatest d of the 32 x 32: where all are beyond the radius one bias serves and goes into c; else the
// biased scores themselves become the values.  slopes: the cap's, for the backward (KEEP).
struct Linear { float a, c; };
template <typename T, bool LANE_IS_QUERY, bool KEEP>
__device__ __forceinline__ Linear make_scores(f32x16& x, f32x16* slopes, const ScoreRule& r, const LaneRow& l, const float* biases, int d0, int d_min, int d_max) {
    if (r.cap) cap_values<T, KEEP>(x, slopes, r);
    Linear s = {r.a, r.c};
    const float* const b = biases + l.bias + r.radius + BIAS_PAD;                          // of distance 0
    bool one_by_one = r.slopes || r.a == 0.f;
    const bool far = d_min >= r.radius || d_max <= -r.radius;
    if (r.table) {
        one_by_one |= !far;
        if (far) {                                              // (a bias so low that it swallows the score must do so)
            const float v = *LDS_PTR(const float, b + (d_min >= r.radius ? r.radius : -r.radius));
            s.c += v;
            one_by_one |= __ballot(!(fabsf(s.c) < 1e30f)) != 0;
        }
    }
    if (one_by_one) {
        for (int e = 0; e < 16; ++e) x[e] = r.table && far ? x[e] * s.a + r.c : x[e] * s.a + s.c;
        if (r.slopes) {
            for (int e = 0; e < 16; ++e) x[e] -= l.slope2 * fabsf((float)(LANE_IS_QUERY ? d0 + reg_row(e) : d0 - reg_row(e)));
        }
        if (r.table && far) {
            const float v = *LDS_PTR(const float, b + (d_min >= r.radius ? r.radius : -r.radius));
            for (int e = 0; e < 16; ++e) x[e] += v;
        } else if (r.table) {
            const float* const at = b + (LANE_IS_QUERY ? d0 : d0 - reg_row(15));
            for (int e = 0; e < 16; ++e) x[e] += *LDS_PTR(const float, at + (LANE_IS_QUERY ? reg_row(e) : reg_row(15) - reg_row(e)));
        }
        s = {1.f, 0.f};
    }
    return s;
}

// values of hidden scores -> those of the score -inf; docs: the streamed rows' documents from register 0's row on, or null
template <bool LANE_IS_QUERY>
__device__ __forceinline__ void hide_scores(f32x16& x, const Linear& s, const LaneRow& l, int d0, const int* docs) {
    const float hidden = s.a < 0.f ? INFINITY : -INFINITY;
    for (int g = 0; g < 4; ++g) {
        i32x4 doc = {l.doc, l.doc, l.doc, l.doc};
        if (docs) doc = *LDS_PTR(const i32x4, docs + 8 * g);
        for (int e = 0; e < 4; ++e) {
            const int d = LANE_IS_QUERY ? d0 + reg_row(4 * g + e) : d0 - reg_row(4 * g + e);
            const bool near = ((d >= l.lo) & (d <= l.hi)) | (LANE_IS_QUERY & (d < l.prefix));
            x[4 * g + e] = near & (doc[e] == l.doc) & (l.doc >= 0) ? x[4 * g + e] : hidden;
        }
    }
}
}  // namespace
