// RMS norm of every query / key head and the position rotation of its columns, forward and backward.
//
// Bound by memory: an element is read once and written once (the backward reads two and writes one) for some ten operations.  A lane holds 16
// bytes of one head's columns (E = 4 f32 or 8 half values), LPH = 2^n lanes hold a head, so that the mean of squares is a butterfly of
// log2 LPH steps inside a wave and no head leaves its wave.  What is not a head's own value lies in LDS as coefficients per column, built once per
// row: the forward's y = r (x A + partner B) with A = w cos, B = +- w_partner sin (two multiplies and one fma an element), the backward's cos,
// +- sin and w.  With few registers (many waves on a CU) rather than loads ahead: prefetching the next head, or two heads in flight with
// weights and angles in registers, measured 139 - 142 us where this order of work takes 76: 335 MB at 4.4 TB/s (16384 rows of
// 32 + 8 heads of 128, f16).
#include "sequence.h"
#include <math.h>

namespace {
constexpr int MAX_WAVES = 8, THREADS = 64 * MAX_WAVES;         // of a block at most
constexpr int MAX_FREQ = 128;
constexpr int ROWS_PER_BLOCK = 4;
constexpr int BWD_BLOCKS = 768;                                 // of the backward, each summing its rows' weight gradients: three of 8 waves on every CU

enum { TURN_NONE, TURN_HALVES, TURN_PAIRS, TURN_ANY };          // how a chunk meets its partner columns: none; a whole chunk n_freq columns away; inside the chunk; column by column

// cosine and sine of t = pos * inv_freq.  The angle is taken in turns, in 64 bits (t has up to 31 bits before the point), cut to an eighth of a turn
// around the nearest quarter, and only that rest, which 32 bits hold to 2^-27 of a turn, goes through the f32 functions.
__device__ __forceinline__ float2 turn(int pos, double inv_freq) {
    const double x = (double)pos * (inv_freq * 0.15915494309189533577);
    const double rest = x - rint(x), quarter = rint(rest * 4.0);
    float s, c;
    sincospif(2.0f * (float)(rest - quarter * 0.25), &s, &c);
    const int k = (int)quarter & 3;
    const float a = k & 1 ? s : c, b = k & 1 ? c : s;
    return make_float2(k == 1 || k == 2 ? -a : a, k >= 2 ? -b : b);
}

template <typename T> struct Chunk {
    static constexpr int E = 16 / sizeof(T);
    uint4 raw;
    __device__ __forceinline__ float operator[](int e) const { return (float)((const T*)&raw)[e]; }
};

template <typename T>
__device__ __forceinline__ Chunk<T> load_chunk(const T* p, bool live) {
    Chunk<T> c;
    c.raw = live ? *(const uint4*)p : make_uint4(0, 0, 0, 0);
    return c;
}

template <typename T>
__device__ __forceinline__ void store_chunk(T* p, const float* y) {
    T v[16 / sizeof(T)];
    for (int e = 0; e < (int)(16 / sizeof(T)); ++e) v[e] = (T)y[e];
    *(uint4*)p = *(const uint4*)v;
}

// The column a column is turned with, and whether it is the first of the pair (itself, where nothing turns)
__device__ __forceinline__ int partner_of(const bigc_head_norm& a, int col) {
    if (col >= 2 * a.n_freq) return col;
    return a.interleaved ? col ^ 1 : col < a.n_freq ? col + a.n_freq : col - a.n_freq;
}

// place of a column's coefficient in LDS: lanes read the four of a quarter chunk side by side
template <int E> __device__ __forceinline__ int slot(int col, int chunks) { return (col % E / 4 * chunks + col / E) * 4 + col % 4; }

template <int E>
__device__ __forceinline__ void coefficients(const float* table, int ch, int chunks, float* out) {
    for (int p = 0; p < E / 4; ++p) *(float4*)(out + 4 * p) = *(const float4*)(table + (p * chunks + ch) * 4);
}

// the partners' values of a chunk that the head's lanes hold
template <typename T, int TURN>
__device__ __forceinline__ void partners(const bigc_head_norm& a, const Chunk<T>& x, const T* head, int ch, bool live, float* o) {
    constexpr int E = 16 / sizeof(T);
    if (TURN == TURN_HALVES) {
        Chunk<T> y;
        const int half = a.n_freq / E, from = (threadIdx.x & 63) + (ch < half ? half : ch < 2 * half ? -half : 0);
        y.raw.x = __shfl(x.raw.x, from); y.raw.y = __shfl(x.raw.y, from); y.raw.z = __shfl(x.raw.z, from); y.raw.w = __shfl(x.raw.w, from);
        for (int e = 0; e < E; ++e) o[e] = y[e];
    } else {
        for (int e = 0; e < E; ++e) o[e] = TURN == TURN_PAIRS ? x[e ^ 1] : TURN == TURN_ANY && live ? (float)head[partner_of(a, ch * E + e)] : 0.f;
    }
}

__device__ __forceinline__ float head_sum(float x, int lph) {
    for (int m = lph >> 1; m; m >>= 1) x += __shfl_xor(x, m);
    return x;
}

// Forward: `rows` rows in a block, whose threads take the heads of a row in turn (blockIdx.y: a part of them).
// LDS: per row A and B of the queries and of the keys.
template <typename T, int TURN>
__global__ __launch_bounds__(THREADS) void head_norm_fwd(bigc_head_norm a, int lph, int rows) {
    constexpr int E = 16 / sizeof(T);
    extern __shared__ float4 lds4[];
    __shared__ float2 angle[ROWS_PER_BLOCK][MAX_FREQ];
    float* tables = (float*)lds4;                               // [row][q, k][A, B][head_dim]
    const long row0 = (long)blockIdx.x * rows;
    const int n = (int)min((long)rows, a.n_rows - row0), heads = a.n_q_head + a.n_k_head, per = blockDim.x / lph, hd = a.head_dim, chunks = hd / E;
    if (TURN != TURN_NONE) {
        for (int i = threadIdx.x; i < n * a.n_freq; i += blockDim.x) angle[i / a.n_freq][i % a.n_freq] = turn(a.pos[row0 + i / a.n_freq], a.inv_freq[i % a.n_freq]);
        __syncthreads();
    }
    for (int i = threadIdx.x; i < n * 2 * hd; i += blockDim.x) {
        const int c = i % hd, of = i / hd;                      // of = 2 row + (key)
        const float* w = of & 1 ? a.wk : a.wq;
        float A = w ? w[c] : 1.f, B = 0.f;
        if (TURN != TURN_NONE && c < 2 * a.n_freq) {
            const int o = partner_of(a, c);
            const float2 t = angle[of >> 1][a.interleaved ? c >> 1 : min(c, o)];
            B = (w ? w[o] : 1.f) * (c < o ? -t.y : t.y);
            A *= t.x;
        }
        tables[of * 2 * hd + slot<E>(c, chunks)] = A;
        tables[of * 2 * hd + hd + slot<E>(c, chunks)] = B;
    }
    __syncthreads();
    const int ch = threadIdx.x % lph;
    const float inv_d = 1.f / hd;
    for (int r = 0; r < n; ++r) {
        const long row = row0 + r;
        for (int h0 = blockIdx.y * per; h0 < heads; h0 += gridDim.y * per) {
            const int h = h0 + threadIdx.x / lph;               // the wave stays together: lanes without a head hold zeros
            const bool key = h >= a.n_q_head, live = ch < chunks && h < heads;
            const T* head = key ? (const T*)a.k + row * a.ldk + (h - a.n_q_head) * a.hsk : (const T*)a.q + row * a.ldq + h * a.hsq;
            const Chunk<T> x = load_chunk(head + ch * E, live);
            float y[E], o[E], A[E], B[E], ss = 0.f;
            partners<T, TURN>(a, x, head, ch, live, o);
            for (int e = 0; e < E; ++e) ss += x[e] * x[e];
            const float f = 1.f / sqrtf(head_sum(ss, lph) * inv_d + a.eps);
            if (!live) continue;                                // (whole heads: the other lanes of the wave need nothing of these any more)
            const float* t = tables + (2 * r + key) * 2 * hd;
            coefficients<E>(t, ch, chunks, A);
            if (TURN != TURN_NONE) coefficients<E>(t + hd, ch, chunks, B);
            for (int e = 0; e < E; ++e) y[e] = f * (TURN == TURN_NONE ? x[e] * A[e] : x[e] * A[e] + o[e] * B[e]);
            store_chunk((key ? (T*)a.k_out + row * a.ldko + (h - a.n_q_head) * a.hsko : (T*)a.q_out + row * a.ldqo + h * a.hsqo) + ch * E, y);
        }
    }
}

// Backward: dn = dy turned back, dw += dn xhat, dx = r (dn w - xhat mean(dn w xhat)), xhat = x r.  Block b takes rows b, b + gridDim.x, ...
// LDS: w of queries and keys, two rows' cos and +- sin (the next row's are written while the last one's may still be read).
// Held to the registers of six waves a SIMD, so that all blocks run at once (8192 rows x 24 + 8 heads of 128, bf16, forward and backward: 87 us; 95 - 101
// at four waves, 146 at eight, which spill).
template <typename T, int TURN>
__global__ __launch_bounds__(THREADS) __attribute__((amdgpu_waves_per_eu(6))) void head_norm_bwd(bigc_head_norm a, int lph, float* part) {
    constexpr int E = 16 / sizeof(T);
    extern __shared__ float4 lds4[];
    float* weights = (float*)lds4;                              // [q, k][head_dim]
    const int heads = a.n_q_head + a.n_k_head, per = blockDim.x / lph, hd = a.head_dim, chunks = hd / E;
    float* turns = weights + 2 * hd;                            // [2][cos, sin][head_dim]
    float* sums = turns + 4 * hd;                               // [threads][E]
    for (int i = threadIdx.x; i < 2 * hd; i += blockDim.x) {
        const float* w = i >= hd ? a.wk : a.wq;
        weights[(i >= hd ? hd : 0) + slot<E>(i % hd, chunks)] = w ? w[i % hd] : 1.f;
    }
    for (int i = threadIdx.x; i < 2 * hd; i += blockDim.x) {    // what does not turn
        turns[i / hd * 2 * hd + slot<E>(i % hd, chunks)] = 1.f;
        turns[i / hd * 2 * hd + hd + slot<E>(i % hd, chunks)] = 0.f;
    }
    __syncthreads();
    float dwq[E], dwk[E];
    for (int e = 0; e < E; ++e) dwq[e] = dwk[e] = 0.f;
    const int ch = threadIdx.x % lph;
    const float inv_d = 1.f / hd;
    int flip = 0;
    for (long row = blockIdx.x; row < a.n_rows; row += gridDim.x, flip ^= 1) {
        float* t = turns + flip * 2 * hd;
        if (TURN != TURN_NONE) {
            for (int f = threadIdx.x; f < a.n_freq; f += blockDim.x) {
                const float2 v = turn(a.pos[row], a.inv_freq[f]);
                const int c = slot<E>(a.interleaved ? 2 * f : f, chunks), o = slot<E>(a.interleaved ? 2 * f + 1 : f + a.n_freq, chunks);
                t[c] = t[o] = v.x;
                t[hd + c] = v.y;
                t[hd + o] = -v.y;
            }
            __syncthreads();
        }
        for (int h0 = 0; h0 < heads; h0 += per) {
            const int h = h0 + threadIdx.x / lph;
            const bool key = h >= a.n_q_head, live = ch < chunks && h < heads;
            const int hh = key ? h - a.n_q_head : h;
            const Chunk<T> x = load_chunk((key ? (const T*)a.k + row * a.ldk + hh * a.hsk : (const T*)a.q + row * a.ldq + hh * a.hsq) + ch * E, live);
            const T* up = key ? (const T*)a.dk_out + row * a.lddko + hh * a.hsdko : (const T*)a.dq_out + row * a.lddqo + hh * a.hsdqo;
            const Chunk<T> g = load_chunk(up + ch * E, live);
            float dn[E], o[E], c[E], s[E], w[E], ss = 0.f, dot = 0.f;
            partners<T, TURN>(a, g, up, ch, live, o);
            const int at = min(ch, chunks - 1);
            coefficients<E>(weights + key * hd, at, chunks, w);
            if (TURN != TURN_NONE) { coefficients<E>(t, at, chunks, c); coefficients<E>(t + hd, at, chunks, s); }
            for (int e = 0; e < E; ++e) {
                dn[e] = TURN == TURN_NONE ? g[e] : g[e] * c[e] + o[e] * s[e];       // 0 in lanes without a head
                ss += x[e] * x[e];
            }
            const float r = 1.f / sqrtf(head_sum(ss, lph) * inv_d + a.eps);
            for (int e = 0; e < E; ++e) {
                const float hat = x[e] * r, d = dn[e] * hat;
                if (key) dwk[e] += live ? d : 0.f; else dwq[e] += live ? d : 0.f;
                dn[e] *= w[e];
                dot += dn[e] * hat;
            }
            dot = head_sum(dot, lph) * inv_d;
            for (int e = 0; e < E; ++e) dn[e] = r * (dn[e] - x[e] * r * dot);
            if (live) store_chunk((key ? (T*)a.dk + row * a.lddk + hh * a.hsdk : (T*)a.dq + row * a.lddq + hh * a.hsdq) + ch * E, dn);
        }
    }
    if (!part) return;
    for (int i = 0; i < 2; ++i) {                               // the block's threads of one chunk, in their order
        __syncthreads();
        for (int e = 0; e < E; ++e) sums[threadIdx.x * E + e] = i ? dwk[e] : dwq[e];
        __syncthreads();
        for (int cc = threadIdx.x; cc < a.head_dim; cc += blockDim.x) {
            float x = 0.f;
            for (int t = cc / E; t < (int)blockDim.x; t += lph) x += sums[t * E + cc % E];
            part[((long)blockIdx.x * 2 + i) * a.head_dim + cc] = x;
        }
    }
}

// 32 columns of one weight (blockIdx.y: 0 wq, 1 wk) in a block: 32 threads a column, each every 32nd partial sum (eight of them on their way at a
// time: with eight threads a column, one after the other, this took 35 us, as long as the backward itself), joined in order
__global__ __launch_bounds__(1024) void head_weight_grad(bigc_head_norm a, const float* part, int blocks) {
    __shared__ float sums[32][33];
    const int c = blockIdx.x * 32 + threadIdx.x % 32, g = threadIdx.x / 32;
    float x = 0.f;
    for (int b0 = g; b0 < blocks; b0 += 32 * 8) {
        float v[8];
        for (int i = 0; i < 8; ++i) v[i] = b0 + 32 * i < blocks && c < a.head_dim ? part[((long)(b0 + 32 * i) * 2 + blockIdx.y) * a.head_dim + c] : 0.f;
        for (int i = 0; i < 8; ++i) x += v[i];
    }
    sums[g][threadIdx.x % 32] = x;
    __syncthreads();
    x = sums[threadIdx.x % 32][g];                              // now column g of the block, one partial sum a lane
    for (int m = 16; m; m >>= 1) x += __shfl_xor(x, m);
    float* dw = blockIdx.y ? a.dwk : a.dwq;
    if (threadIdx.x % 32 == 0 && blockIdx.x * 32 + g < a.head_dim && dw) dw[blockIdx.x * 32 + g] = x;
}

// Lanes of a head, how its columns are turned, and the waves of a block: of 4 to 8 waves the number that leaves fewest of them without a head in
// a row's last round (40 heads, four to a wave: five waves, two rounds).
struct Shape { int lph, turn, rounds, waves; };
Shape shape_of(const bigc_head_norm& a) {
    const int e = 16 / seq_size(a.dtype);
    int lph = 1;
    while (lph * e < a.head_dim) lph *= 2;
    const int need = cdiv((a.n_q_head + a.n_k_head) * lph, 64);
    int waves = need < 4 ? need : 4;
    for (int w = 5; w <= MAX_WAVES && w <= need; ++w)
        if (cdiv(need, w) * w < cdiv(need, waves) * waves || w == need) waves = w;
    return {lph, a.n_freq == 0 ? TURN_NONE : a.interleaved ? TURN_PAIRS : a.n_freq % e == 0 ? TURN_HALVES : TURN_ANY, cdiv(need, waves), waves};
}

int check_rows(const bigc_head_norm& a, const char* who, const char* what, const void* p, int64_t ld, int64_t hs, int heads) {
    const int64_t e = 16 / seq_size(a.dtype);
    if (a.n_rows == 0 || heads == 0) return BIGC_OK;
    BIGC_CHECK_ARG(p, "%s: %s is NULL", who, what);
    BIGC_CHECK_ARG((uintptr_t)p % 16 == 0 && (a.n_rows == 1 || ld % e == 0) && (heads == 1 || hs % e == 0),
                   "%s: %s: address, row stride %ld and head stride %ld have to be multiples of 16 bytes", who, what, (long)ld, (long)hs);
    BIGC_CHECK_ARG((a.n_rows == 1 || ld >= 0) && (heads == 1 || hs >= 0), "%s: %s: negative stride", who, what);
    return BIGC_OK;
}

// an output: no two of its rows and heads share a place, and one that is its input's place has its strides (a row's partner columns are read before it is written, other rows' not)
int check_out(const bigc_head_norm& a, const char* who, const char* what, const void* p, int64_t ld, int64_t hs, int heads, const void* in, int64_t ldi, int64_t hsi) {
    const int rc = check_rows(a, who, what, p, ld, hs, heads);
    if (rc != BIGC_OK || a.n_rows == 0 || heads == 0) return rc;
    BIGC_CHECK_ARG(!rows_overlap(ld, hs, a.head_dim, a.n_rows, heads), "%s: %s: rows or heads overlap (row stride %ld, head stride %ld)", who, what, (long)ld, (long)hs);
    BIGC_CHECK_ARG(p != in || ((a.n_rows == 1 || ld == ldi) && (heads == 1 || hs == hsi)), "%s: %s: in place of its input with other strides", who, what);
    return BIGC_OK;
}

int check_args(const bigc_head_norm* ap, const char* who) {
    BIGC_CHECK_ARG(ap, "%s: arguments are NULL", who);
    const bigc_head_norm& a = *ap;
    BIGC_CHECK_ARG(a.dtype == BIGC_F32 || a.dtype == BIGC_F16 || a.dtype == BIGC_BF16, "%s: dtype %d", who, a.dtype);
    BIGC_CHECK_ARG(a.n_q_head >= 0 && a.n_k_head >= 0 && a.n_q_head + a.n_k_head > 0 && a.n_q_head <= 65536 && a.n_k_head <= 65536, "%s: %d and %d heads", who, a.n_q_head, a.n_k_head);
    BIGC_CHECK_ARG(a.head_dim > 0 && a.head_dim <= 256 && a.head_dim % 8 == 0, "%s: head_dim %d (a multiple of 8 up to 256)", who, a.head_dim);
    BIGC_CHECK_ARG(a.n_rows >= 0 && a.n_rows < (1ll << 31), "%s: %ld rows", who, (long)a.n_rows);
    BIGC_CHECK_ARG(a.n_freq >= 0 && 2 * (long)a.n_freq <= a.head_dim, "%s: %d frequencies on head_dim %d", who, a.n_freq, a.head_dim);
    BIGC_CHECK_ARG(a.n_freq == 0 || a.n_rows == 0 || (a.pos && a.inv_freq), "%s: pos or inv_freq is NULL", who);
    BIGC_CHECK_ARG(isfinite(a.eps) && a.eps >= 0.f, "%s: eps %g", who, a.eps);
    return BIGC_OK;
}

int bwd_blocks(const bigc_head_norm& a) { return (int)(a.n_rows < 1 ? 1 : a.n_rows < BWD_BLOCKS ? a.n_rows : BWD_BLOCKS); }

#define TURNS(turn, T, kernel, grid, threads, lds, stream, ...) do { \
    if (turn == TURN_NONE) kernel<T, TURN_NONE><<<grid, threads, lds, stream>>>(__VA_ARGS__); \
    else if (turn == TURN_HALVES) kernel<T, TURN_HALVES><<<grid, threads, lds, stream>>>(__VA_ARGS__); \
    else if (turn == TURN_PAIRS) kernel<T, TURN_PAIRS><<<grid, threads, lds, stream>>>(__VA_ARGS__); \
    else kernel<T, TURN_ANY><<<grid, threads, lds, stream>>>(__VA_ARGS__); } while (0);
#define SEQ_DISPATCH(dtype, F) do { if ((dtype) == BIGC_F32) { F(float) } else if ((dtype) == BIGC_F16) { F(f16_t) } else { F(bf16_t) } } while (0)
}  // namespace

extern "C" int bigc_head_norm_rope_fwd(void* stream, const bigc_head_norm* ap) {
    const char* who = "head_norm_rope_fwd";
    int rc = check_args(ap, who);
    if (rc != BIGC_OK) return rc;
    const bigc_head_norm a = *ap;
    if ((rc = check_rows(a, who, "q", a.q, a.ldq, a.hsq, a.n_q_head)) != BIGC_OK) return rc;
    if ((rc = check_rows(a, who, "k", a.k, a.ldk, a.hsk, a.n_k_head)) != BIGC_OK) return rc;
    if ((rc = check_out(a, who, "q_out", a.q_out, a.ldqo, a.hsqo, a.n_q_head, a.q, a.ldq, a.hsq)) != BIGC_OK) return rc;
    if ((rc = check_out(a, who, "k_out", a.k_out, a.ldko, a.hsko, a.n_k_head, a.k, a.ldk, a.hsk)) != BIGC_OK) return rc;
    if (a.n_rows == 0) return BIGC_OK;
    // Four rows a block, all heads of each; while that would leave CUs without a block, one row and one round of heads a block instead (a call of a
    // few rows is latency: its threads then make one trip through memory).
    const Shape sh = shape_of(a);
    const bool few = a.n_rows < ROWS_PER_BLOCK * 1024;
    const int rows = few ? 1 : ROWS_PER_BLOCK;
    const dim3 grid((unsigned)((a.n_rows + rows - 1) / rows), few ? sh.rounds : 1);
    BIGC_CHECK_ARG((double)grid.x * grid.y * 64 * sh.waves < 4294967296.0, "%s: %ld rows of %d heads are too many for one launch", who, (long)a.n_rows, a.n_q_head + a.n_k_head);
    ProfScope prof(stream, FAM_LAYERNORM, 0, 0);
#define F(T) TURNS(sh.turn, T, head_norm_fwd, grid, 64 * sh.waves, sizeof(float) * rows * 4 * a.head_dim, (hipStream_t)stream, a, sh.lph, rows)
    SEQ_DISPATCH(a.dtype, F);
#undef F
    BIGC_LAUNCH_CHECK("head_norm_rope_fwd");
    return BIGC_OK;
}

extern "C" size_t bigc_head_norm_rope_workspace_bytes(const bigc_head_norm* a) {
    if (check_args(a, "head_norm_rope_workspace_bytes") != BIGC_OK) return 0;
    return sizeof(float) * bwd_blocks(*a) * 2 * a->head_dim;
}

extern "C" int bigc_head_norm_rope_bwd(void* stream, const bigc_head_norm* ap, void* workspace, size_t workspace_bytes) {
    const char* who = "head_norm_rope_bwd";
    int rc = check_args(ap, who);
    if (rc != BIGC_OK) return rc;
    const bigc_head_norm a = *ap;
    if ((rc = check_rows(a, who, "q", a.q, a.ldq, a.hsq, a.n_q_head)) != BIGC_OK) return rc;
    if ((rc = check_rows(a, who, "k", a.k, a.ldk, a.hsk, a.n_k_head)) != BIGC_OK) return rc;
    if ((rc = check_rows(a, who, "dq_out", a.dq_out, a.lddqo, a.hsdqo, a.n_q_head)) != BIGC_OK) return rc;
    if ((rc = check_rows(a, who, "dk_out", a.dk_out, a.lddko, a.hsdko, a.n_k_head)) != BIGC_OK) return rc;
    if ((rc = check_out(a, who, "dq", a.dq, a.lddq, a.hsdq, a.n_q_head, a.dq_out, a.lddqo, a.hsdqo)) != BIGC_OK) return rc;
    if ((rc = check_out(a, who, "dk", a.dk, a.lddk, a.hsdk, a.n_k_head, a.dk_out, a.lddko, a.hsdko)) != BIGC_OK) return rc;
    const size_t need = bigc_head_norm_rope_workspace_bytes(ap);
    if (workspace_bytes < need || !workspace || (uintptr_t)workspace % 16)
        return bigc_fail(BIGC_ERR_WORKSPACE, "%s: workspace of %zu bytes, %zu needed", who, workspace_bytes, need);
    ProfScope prof(stream, FAM_BACKWARD, 0, 0);
    float* part = (float*)workspace;
    const Shape sh = shape_of(a);
    const bool weights = a.dwq || a.dwk;
    const int blocks = bwd_blocks(a);
#define F(T) TURNS(sh.turn, T, head_norm_bwd, blocks, 64 * sh.waves, sizeof(float) * (6 * a.head_dim + 64 * sh.waves * (16 / seq_size(a.dtype))), (hipStream_t)stream, a, sh.lph, weights ? part : nullptr)
    SEQ_DISPATCH(a.dtype, F);
#undef F
    if (weights) head_weight_grad<<<dim3(cdiv(a.head_dim, 32), 2), 1024, 0, (hipStream_t)stream>>>(a, part, blocks);
    BIGC_LAUNCH_CHECK("head_norm_rope_bwd");
    return BIGC_OK;
}
