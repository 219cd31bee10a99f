// RMS norm of every query / key head and the position rotation of its columns, forward and backward.
#include "sequence.h"
#include <math.h>

namespace {
constexpr int ROW_BLOCKS = 256;                                // blocks of the backward: each sums its rows' weight gradients

__device__ __forceinline__ float wave_sum(float x) {
    for (int m = 32; m; m >>= 1) x += __shfl_xor(x, m);
    return x;
}

// One wave per head row; columns in LDS.  back: x = dy, rotated by -t.
__device__ void rotate(const bigc_head_norm& a, float* y, int pos, bool back) {
    for (int f = threadIdx.x; f < a.n_freq; f += 64) {
        double sn, cs;
        sincos((double)pos * a.inv_freq[f], &sn, &cs);
        const float c = (float)cs, s = back ? -(float)sn : (float)sn;
        const int i = a.interleaved ? 2 * f : f, j = a.interleaved ? 2 * f + 1 : f + a.n_freq;
        const float u = y[i], v = y[j];
        y[i] = u * c - v * s;
        y[j] = v * c + u * s;
    }
    __syncthreads();
}

template <typename T>
__global__ __launch_bounds__(64) void head_rows_fwd(bigc_head_norm a) {
    __shared__ float y[256];
    const int lane = threadIdx.x, heads = a.n_q_head + a.n_k_head;
    int h = blockIdx.x % heads;
    const long row = blockIdx.x / heads;
    const bool key = h >= a.n_q_head;
    if (key) h -= a.n_q_head;
    const T* x = key ? (const T*)a.k + row * a.ldk + h * a.hsk : (const T*)a.q + row * a.ldq + h * a.hsq;
    T* o = key ? (T*)a.k_out + row * a.ldko + h * a.hsko : (T*)a.q_out + row * a.ldqo + h * a.hsqo;
    const float* w = key ? a.wk : a.wq;
    float ss = 0.f;
    for (int c = lane; c < a.head_dim; c += 64) { const float v = (float)x[c]; y[c] = v; ss += v * v; }
    const float r = 1.f / sqrtf(wave_sum(ss) / a.head_dim + a.eps);
    for (int c = lane; c < a.head_dim; c += 64) y[c] *= r * (w ? w[c] : 1.f);
    __syncthreads();
    rotate(a, y, a.pos ? a.pos[row] : 0, false);
    for (int c = lane; c < a.head_dim; c += 64) o[c] = (T)y[c];
}

template <typename T>
__global__ __launch_bounds__(64) void head_rows_bwd(bigc_head_norm a, float* part) {
    __shared__ float y[256];
    const int lane = threadIdx.x, heads = a.n_q_head + a.n_k_head;
    float dw[2][4] = {};
    for (long e = blockIdx.x; e < a.n_rows * heads; e += ROW_BLOCKS) {
        int h = (int)(e % heads);
        const long row = e / heads;
        const bool key = h >= a.n_q_head;
        if (key) h -= a.n_q_head;
        const T* x = key ? (const T*)a.k + row * a.ldk + h * a.hsk : (const T*)a.q + row * a.ldq + h * a.hsq;
        const T* g = key ? (const T*)a.dk_out + row * a.lddko + h * a.hsdko : (const T*)a.dq_out + row * a.lddqo + h * a.hsdqo;
        T* o = key ? (T*)a.dk + row * a.lddk + h * a.hsdk : (T*)a.dq + row * a.lddq + h * a.hsdq;
        const float* w = key ? a.wk : a.wq;
        float ss = 0.f, dot = 0.f, xv[4];
        __syncthreads();
        for (int t = 0; t < 4; ++t) {
            const int c = lane + 64 * t;
            xv[t] = c < a.head_dim ? (float)x[c] : 0.f;
            if (c < a.head_dim) y[c] = (float)g[c];
            ss += xv[t] * xv[t];
        }
        __syncthreads();
        rotate(a, y, a.pos ? a.pos[row] : 0, true);
        const float r = 1.f / sqrtf(wave_sum(ss) / a.head_dim + a.eps);
        for (int t = 0; t < 4; ++t) {
            const int c = lane + 64 * t;
            if (c < a.head_dim) { dw[key][t] += y[c] * xv[t] * r; dot += y[c] * (w ? w[c] : 1.f) * xv[t] * r; }
        }
        dot = wave_sum(dot) / a.head_dim;
        for (int t = 0; t < 4; ++t) {
            const int c = lane + 64 * t;
            if (c < a.head_dim) o[c] = (T)(r * (y[c] * (w ? w[c] : 1.f) - xv[t] * r * dot));
        }
    }
    for (int i = 0; i < 2; ++i)
        for (int t = 0; t < 4; ++t) part[((long)blockIdx.x * 2 + i) * 256 + lane + 64 * t] = dw[i][t];
}

__global__ __launch_bounds__(256) void head_weight_grad(bigc_head_norm a, const float* part) {
    float x = 0.f;
    for (int b = 0; b < ROW_BLOCKS; ++b) x += part[((long)b * 2 + blockIdx.x) * 256 + threadIdx.x];
    float* dw = blockIdx.x ? a.dwk : a.dwq;
    if (dw && threadIdx.x < a.head_dim) dw[threadIdx.x] = x;
}

int check_rows(const bigc_head_norm& a, const char* who, const char* what, const void* p, int64_t ld, int64_t hs, int heads) {
    const int64_t e = 16 / seq_size(a.dtype);
    if (a.n_rows == 0 || heads == 0) return BIGC_OK;
    BIGC_CHECK_ARG(p, "%s: %s is NULL", who, what);
    BIGC_CHECK_ARG((uintptr_t)p % 16 == 0 && ld % e == 0 && (heads == 1 || hs % e == 0),
                   "%s: %s: address, row stride %ld and head stride %ld have to be multiples of 16 bytes", who, what, (long)ld, (long)hs);
    BIGC_CHECK_ARG(ld >= 0 && (heads == 1 || hs >= 0), "%s: %s: negative stride", who, what);
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
    BIGC_CHECK_ARG((double)a.n_rows * (a.n_q_head + a.n_k_head) < 2147483648.0, "%s: %ld rows of %d heads are too many for one launch", who, (long)a.n_rows,
                   a.n_q_head + a.n_k_head);
    return BIGC_OK;
}

#define SEQ_DISPATCH(dtype, F) do { if ((dtype) == BIGC_F32) { F(float) } else if ((dtype) == BIGC_F16) { F(f16_t) } else { F(bf16_t) } } while (0)
}  // namespace

extern "C" int bigc_head_norm_rope_fwd(void* stream, const bigc_head_norm* ap) {
    const char* who = "head_norm_rope_fwd";
    int rc = check_args(ap, who);
    if (rc != BIGC_OK) return rc;
    const bigc_head_norm a = *ap;
    if ((rc = check_rows(a, who, "q", a.q, a.ldq, a.hsq, a.n_q_head)) != BIGC_OK) return rc;
    if ((rc = check_rows(a, who, "k", a.k, a.ldk, a.hsk, a.n_k_head)) != BIGC_OK) return rc;
    if ((rc = check_rows(a, who, "q_out", a.q_out, a.ldqo, a.hsqo, a.n_q_head)) != BIGC_OK) return rc;
    if ((rc = check_rows(a, who, "k_out", a.k_out, a.ldko, a.hsko, a.n_k_head)) != BIGC_OK) return rc;
    if (a.n_rows == 0) return BIGC_OK;
    ProfScope prof(stream, FAM_LAYERNORM, 0, 0);
#define F(T) head_rows_fwd<T><<<(unsigned)(a.n_rows * (a.n_q_head + a.n_k_head)), 64, 0, (hipStream_t)stream>>>(a);
    SEQ_DISPATCH(a.dtype, F);
#undef F
    BIGC_LAUNCH_CHECK("head_norm_rope_fwd");
    return BIGC_OK;
}

extern "C" size_t bigc_head_norm_rope_workspace_bytes(const bigc_head_norm* a) {
    if (check_args(a, "head_norm_rope_workspace_bytes") != BIGC_OK) return 0;
    return sizeof(float) * ROW_BLOCKS * 2 * 256;
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
    if ((rc = check_rows(a, who, "dq", a.dq, a.lddq, a.hsdq, a.n_q_head)) != BIGC_OK) return rc;
    if ((rc = check_rows(a, who, "dk", a.dk, a.lddk, a.hsdk, a.n_k_head)) != BIGC_OK) return rc;
    const size_t need = bigc_head_norm_rope_workspace_bytes(ap);
    if (workspace_bytes < need || !workspace || (uintptr_t)workspace % 16)
        return bigc_fail(BIGC_ERR_WORKSPACE, "%s: workspace of %zu bytes, %zu needed", who, workspace_bytes, need);
    ProfScope prof(stream, FAM_BACKWARD, 0, 0);
    float* part = (float*)workspace;
#define F(T) head_rows_bwd<T><<<ROW_BLOCKS, 64, 0, (hipStream_t)stream>>>(a, part);
    SEQ_DISPATCH(a.dtype, F);
#undef F
    if (a.dwq || a.dwk) head_weight_grad<<<2, 256, 0, (hipStream_t)stream>>>(a, part);
    BIGC_LAUNCH_CHECK("head_norm_rope_bwd");
    return BIGC_OK;
}
