// Attention over ordered rows: entry points, checks, and the kernels.
#include "attention_fwd.h"

namespace {

// ---- row kernels: one wave per (row, head), the definition read out directly ----------------------------------------------------

__device__ __forceinline__ float wave_sum(float x) {
    for (int m = 32; m; m >>= 1) x += __shfl_xor(x, m);
    return x;
}
__device__ __forceinline__ float wave_max(float x) {
    for (int m = 32; m; m >>= 1) x = fmaxf(x, __shfl_xor(x, m));
    return x;
}

struct Score { float s, dcap; int bin; bool seen; };          // dcap: d score / d (scale q.k)

template <typename T>
__device__ Score score_of(const bigc_seq_attn& a, const float* qrow, const T* krow, int h, int prefix, int pos, int j, int qdoc, int kdoc) {
    Score r;
    r.seen = seq_near(a, prefix, pos, j) && (!a.q_doc || (qdoc == kdoc && kdoc >= 0));
    r.s = -INFINITY; r.dcap = 1.f; r.bin = 0;
    if (!r.seen) return r;
    float x = 0.f;
    for (int c = 0; c < a.head_dim; ++c) x += qrow[c] * (float)krow[c];
    x *= a.scale;
    if (a.softcap > 0.f) { const float t = tanhf(x / a.softcap); x = a.softcap * t; r.dcap = 1.f - t * t; }
    const int d = j - pos;
    if (a.slopes) x -= a.slopes[h] * fabsf((float)d);
    if (a.rel_table) {
        r.bin = min(max(d, -a.bias_radius), a.bias_radius) + a.bias_radius;
        x += a.rel_table[(long)min(max(a.rel_map[r.bin], 0), a.n_bucket - 1) * a.n_head + h];
    }
    r.s = x;
    return r;
}

// delta = dO . O per (row, head)
template <typename T>
__global__ __launch_bounds__(64) void rows_delta(bigc_seq_attn a, float* delta) {
    const int lane = threadIdx.x, h = blockIdx.x % a.n_head;
    const long row = blockIdx.x / a.n_head;
    float x = 0.f;
    for (int c = lane; c < a.head_dim; c += 64) {
        const float o = a.o32 ? a.o32[(row * a.n_head + h) * a.head_dim + c] : (float)((const T*)a.o)[row * a.ldo + h * a.hso + c];
        x += o * (float)((const T*)a.d_o)[row * a.lddo + h * a.hsdo + c];
    }
    x = wave_sum(x);
    if (lane == 0) delta[row * a.n_head + h] = x;
}

constexpr int BIN_BLOCKS = 64;

// dq of the rows of one head, and the sums of dS by distance of this block's rows
template <typename T>
__global__ __launch_bounds__(64) void rows_dq(bigc_seq_attn a, const float* delta, float* by_dist) {
    __shared__ float qs[128], go[128];
    extern __shared__ float bins[];
    const int lane = threadIdx.x, h = blockIdx.x % a.n_head, blk = blockIdx.x / a.n_head;
    const int nbin = a.d_rel_table ? 2 * a.bias_radius + 1 : 0;
    for (int b = lane; b < nbin; b += 64) bins[b] = 0.f;
    const int hk = h / (a.n_head / a.n_kv_head);
    for (long r = blk; r < (long)a.n_seq * a.max_q; r += BIN_BLOCKS) {
        const int s = (int)(r / a.max_q), i = (int)(r % a.max_q);
        const SeqSpan sp = seq_span(a, s);
        if (i >= sp.nq) continue;
        const long row = sp.q0 + i;
        __syncthreads();
        for (int c = lane; c < a.head_dim; c += 64) {
            qs[c] = (float)((const T*)a.q)[row * a.ldq + h * a.hsq + c];
            go[c] = (float)((const T*)a.d_o)[row * a.lddo + h * a.hsdo + c];
        }
        __syncthreads();
        const int pos = i + sp.nk - sp.nq, prefix = a.prefix_len ? a.prefix_len[s] : 0, qdoc = a.q_doc ? a.q_doc[row] : 0;
        const float m = a.stats[2 * (row * a.n_head + h)], l = a.stats[2 * (row * a.n_head + h) + 1], dl = delta[row * a.n_head + h];
        float g[2] = {0.f, 0.f};
        for (int j0 = 0; j0 < sp.nk; j0 += 64) {
            const int j = j0 + lane;
            float ds = 0.f, dx = 0.f;
            int bin = 0;
            if (j < sp.nk) {
                const Score e = score_of<T>(a, qs, (const T*)a.k + (long)(sp.k0 + j) * a.ldk + hk * a.hsk, h, prefix, pos, j, qdoc, a.k_doc ? a.k_doc[sp.k0 + j] : 0);
                if (e.seen && l != 0.f) {
                    const T* v = (const T*)a.v + (long)(sp.k0 + j) * a.ldv + hk * a.hsv;
                    float dp = 0.f;
                    for (int c = 0; c < a.head_dim; ++c) dp += go[c] * (float)v[c];
                    ds = exp2f(e.s * LOG2E - m) / l * (dp - dl);
                    dx = ds * e.dcap * a.scale;
                    bin = e.bin;
                    if (bin > 0 && bin < nbin - 1) bins[bin] += ds;      // the lanes' distances differ
                }
            }
            if (nbin) {                                                  // the clipped ends: many keys of one bin
                const float lo = wave_sum(bin == 0 ? ds : 0.f), hi = wave_sum(bin == nbin - 1 && bin > 0 ? ds : 0.f);
                if (lane == 0) { bins[0] += lo; bins[nbin - 1] += hi; }
            }
            for (int jj = 0; jj < 64 && j0 + jj < sp.nk; ++jj) {
                const float x = __shfl(dx, jj);
                if (x == 0.f) continue;
                const T* k = (const T*)a.k + (long)(sp.k0 + j0 + jj) * a.ldk + hk * a.hsk;
                for (int t = 0; t < 2; ++t) if (lane + 64 * t < a.head_dim) g[t] += x * (float)k[lane + 64 * t];
            }
        }
        for (int t = 0; t < 2; ++t)
            if (lane + 64 * t < a.head_dim) ((T*)a.dq)[row * a.lddq + h * a.hsdq + lane + 64 * t] = (T)g[t];
    }
    __syncthreads();
    for (int b = lane; b < nbin; b += 64) by_dist[((long)blk * a.n_head + h) * nbin + b] = bins[b];
}

// dk, dv of one key row and key head, summed over the rows and the query heads that read it
template <typename T>
__global__ __launch_bounds__(64) void rows_dkv(bigc_seq_attn a, const float* delta) {
    __shared__ float ks[128], vs[128];
    const int lane = threadIdx.x, hk = blockIdx.x % a.n_kv_head, group = a.n_head / a.n_kv_head;
    const long r = blockIdx.x / a.n_kv_head;
    const int s = (int)(r / a.max_k), j = (int)(r % a.max_k);
    const SeqSpan sp = seq_span(a, s);
    if (j >= sp.nk) return;
    const long row = sp.k0 + j;
    for (int c = lane; c < a.head_dim; c += 64) {
        ks[c] = (float)((const T*)a.k)[row * a.ldk + hk * a.hsk + c];
        vs[c] = (float)((const T*)a.v)[row * a.ldv + hk * a.hsv + c];
    }
    __syncthreads();
    const int prefix = a.prefix_len ? a.prefix_len[s] : 0, kdoc = a.k_doc ? a.k_doc[row] : 0;
    float gk[2] = {0.f, 0.f}, gv[2] = {0.f, 0.f};
    for (int h = hk * group; h < (hk + 1) * group; ++h)
        for (int i0 = 0; i0 < sp.nq; i0 += 64) {
            const int i = i0 + lane;
            float p = 0.f, ds = 0.f;
            if (i < sp.nq) {
                const long qr = sp.q0 + i;
                const float m = a.stats[2 * (qr * a.n_head + h)], l = a.stats[2 * (qr * a.n_head + h) + 1];
                const Score e = score_of<T>(a, ks, (const T*)a.q + qr * a.ldq + h * a.hsq, h, prefix, i + sp.nk - sp.nq, j, a.q_doc ? a.q_doc[qr] : 0, kdoc);
                if (e.seen && l != 0.f) {
                    const T* go = (const T*)a.d_o + qr * a.lddo + h * a.hsdo;
                    float dp = 0.f;
                    for (int c = 0; c < a.head_dim; ++c) dp += vs[c] * (float)go[c];
                    p = exp2f(e.s * LOG2E - m) / l;
                    ds = p * (dp - delta[qr * a.n_head + h]) * e.dcap * a.scale;
                }
            }
            for (int ii = 0; ii < 64 && i0 + ii < sp.nq; ++ii) {
                const float pi = __shfl(p, ii), di = __shfl(ds, ii);
                if (pi == 0.f && di == 0.f) continue;
                const long qr = sp.q0 + i0 + ii;
                for (int t = 0; t < 2; ++t) {
                    const int c = lane + 64 * t;
                    if (c >= a.head_dim) continue;
                    gv[t] += pi * (float)((const T*)a.d_o)[qr * a.lddo + h * a.hsdo + c];
                    gk[t] += di * (float)((const T*)a.q)[qr * a.ldq + h * a.hsq + c];
                }
            }
        }
    for (int t = 0; t < 2; ++t) {
        const int c = lane + 64 * t;
        if (c >= a.head_dim) continue;
        ((T*)a.dk)[row * a.lddk + hk * a.hsdk + c] = (T)gk[t];
        ((T*)a.dv)[row * a.lddv + hk * a.hsdv + c] = (T)gv[t];
    }
}

// table gradient: the sums by distance of all blocks, added per bucket in order
__global__ __launch_bounds__(256) void rel_table_grad(bigc_seq_attn a, const float* by_dist, int blocks) {
    __shared__ float part[256];
    const int h = blockIdx.x % a.n_head, b = blockIdx.x / a.n_head, nbin = 2 * a.bias_radius + 1;
    float x = 0.f;
    for (long e = threadIdx.x; e < (long)blocks * nbin; e += 256) {
        const int bin = (int)(e % nbin);
        if (min(max(a.rel_map[bin], 0), a.n_bucket - 1) == b) x += by_dist[(e / nbin * a.n_head + h) * nbin + bin];
    }
    part[threadIdx.x] = x;
    for (int m = 128; m; m >>= 1) {
        __syncthreads();
        if (threadIdx.x < m) part[threadIdx.x] += part[threadIdx.x + m];
    }
    if (threadIdx.x == 0) a.d_rel_table[(long)b * a.n_head + h] = part[0];
}

// ---- host -----------------------------------------------------------------------------------------------------------------------

size_t up(size_t n) { return (n + 255) & ~(size_t)255; }

struct Plan { size_t delta, by_dist, total; };
Plan plan_of(const bigc_seq_attn& a) {
    Plan p = {0, 0, 0};
    p.by_dist = up(sizeof(float) * (size_t)a.n_q * a.n_head);
    p.total = p.by_dist + (a.d_rel_table ? up(sizeof(float) * BIN_BLOCKS * (size_t)a.n_head * (2 * a.bias_radius + 1)) : 0);
    return p;
}

int check_rows(const bigc_seq_attn& a, const char* who, const char* what, const void* p, int64_t ld, int64_t hs, int64_t rows, int heads) {
    const int64_t e = 16 / seq_size(a.dtype);
    if (rows == 0) return BIGC_OK;
    BIGC_CHECK_ARG(p, "%s: %s is NULL", who, what);
    BIGC_CHECK_ARG((uintptr_t)p % 16 == 0 && ld % e == 0 && (heads == 1 || hs % e == 0),
                   "%s: %s: address, row stride %ld and head stride %ld have to be multiples of 16 bytes", who, what, (long)ld, (long)hs);
    BIGC_CHECK_ARG(ld >= 0 && ld <= (1 << 22) && (heads == 1 || hs >= 0), "%s: %s: row stride %ld (0 to 2^22 elements), head stride %ld", who, what, (long)ld, (long)hs);
    return BIGC_OK;
}

int check_args(const bigc_seq_attn* ap, const char* who) {
    BIGC_CHECK_ARG(ap, "%s: arguments are NULL", who);
    const bigc_seq_attn& a = *ap;
    BIGC_CHECK_ARG(a.dtype == BIGC_F32 || a.dtype == BIGC_F16 || a.dtype == BIGC_BF16, "%s: dtype %d", who, a.dtype);
    BIGC_CHECK_ARG(a.n_seq >= 0 && a.n_head > 0 && a.n_kv_head > 0 && a.n_head % a.n_kv_head == 0, "%s: %d sequences, %d heads over %d key heads", who, a.n_seq,
                   a.n_head, a.n_kv_head);
    BIGC_CHECK_ARG(a.head_dim > 0 && a.head_dim <= 128 && a.head_dim % 8 == 0, "%s: head_dim %d (a multiple of 8 up to 128)", who, a.head_dim);
    BIGC_CHECK_ARG(a.n_q >= 0 && a.n_k >= 0 && a.n_q < (1ll << 31) && a.n_k < (1ll << 31) && a.max_q >= 0 && a.max_k >= 0, "%s: %ld query and %ld key rows, longest %d and %d",
                   who, (long)a.n_q, (long)a.n_k, a.max_q, a.max_k);
    BIGC_CHECK_ARG((long)a.max_q + a.max_k < (1l << 31), "%s: %d queries and %d keys are too far apart", who, a.max_q, a.max_k);
    BIGC_CHECK_ARG((double)a.n_q * a.n_head < 2147483648.0, "%s: %ld rows of %d heads are too many", who, (long)a.n_q, a.n_head);
    BIGC_CHECK_ARG(a.n_seq == 0 || (a.q_off && a.k_off), "%s: offsets are NULL", who);
    BIGC_CHECK_ARG(a.window_left >= -1 && a.window_right >= -1, "%s: window (%d, %d)", who, a.window_left, a.window_right);
    BIGC_CHECK_ARG(isfinite(a.scale) && isfinite(a.softcap) && a.softcap >= 0.f, "%s: scale %g, softcap %g", who, a.scale, a.softcap);
    BIGC_CHECK_ARG(!a.q_doc == !a.k_doc || a.n_q == 0 || a.n_k == 0, "%s: q_doc and k_doc come together", who);
    BIGC_CHECK_ARG(!a.rel_table == !a.rel_map, "%s: rel_table and rel_map come together", who);
    if (a.rel_table) BIGC_CHECK_ARG(a.n_bucket > 0 && a.bias_radius >= 0 && a.bias_radius <= 2047, "%s: %d buckets, radius %d (at most 2047)", who, a.n_bucket, a.bias_radius);
    BIGC_CHECK_ARG((double)a.n_seq * a.max_q * a.n_head < 2147483648.0 && (double)a.n_seq * a.max_k * a.n_head < 2147483648.0,
                   "%s: %d sequences of up to %d queries and %d keys with %d heads are too many for one launch", who, a.n_seq, a.max_q, a.max_k, a.n_head);
    return BIGC_OK;
}

#define SEQ_DISPATCH(dtype, F) do { if ((dtype) == BIGC_F32) { F(float) } else if ((dtype) == BIGC_F16) { F(f16_t) } else { F(bf16_t) } } while (0)
}  // namespace

extern "C" size_t bigc_seq_attn_workspace_bytes(const bigc_seq_attn* a, int backward) {
    if (check_args(a, "seq_attn_workspace_bytes") != BIGC_OK) return 0;
    return backward ? plan_of(*a).total : fwd_shape(*a).total;
}

extern "C" int bigc_seq_attn_fwd(void* stream, const bigc_seq_attn* ap, void* workspace, size_t workspace_bytes) {
    const char* who = "seq_attn_fwd";
    int rc = check_args(ap, who);
    if (rc != BIGC_OK) return rc;
    const bigc_seq_attn a = *ap;
    if ((rc = check_rows(a, who, "q", a.q, a.ldq, a.hsq, a.n_q, a.n_head)) != BIGC_OK) return rc;
    if ((rc = check_rows(a, who, "k", a.k, a.ldk, a.hsk, a.n_k, a.n_kv_head)) != BIGC_OK) return rc;
    if ((rc = check_rows(a, who, "v", a.v, a.ldv, a.hsv, a.n_k, a.n_kv_head)) != BIGC_OK) return rc;
    if ((rc = check_rows(a, who, "o", a.o, a.ldo, a.hso, a.n_q, a.n_head)) != BIGC_OK) return rc;
    BIGC_CHECK_ARG((uintptr_t)a.stats % 8 == 0 && (uintptr_t)a.o32 % 16 == 0, "%s: stats has to lie at a multiple of 8 bytes, o32 of 16", who);
    const FwdShape sh = fwd_shape(a);
    if (workspace_bytes < sh.total || (sh.total && (!workspace || (uintptr_t)workspace % 16)))
        return bigc_fail(BIGC_ERR_WORKSPACE, "%s: workspace of %zu bytes, %zu needed", who, workspace_bytes, sh.total);
    if (a.n_q == 0) return BIGC_OK;
    hipStream_t hs = (hipStream_t)stream;
    ProfScope prof(stream, FAM_MHA, 0, 0);
    if (sh.blocks == 0) {                                       // no sequence, or none with a query
        if (a.zero_rest) {
#define F(T) zero_rows<T><<<256, 256, 0, hs>>>((T*)a.o, a.ldo, a.hso, a.n_q, a.n_head, a.head_dim, a.q_off, a.n_seq);
            SEQ_DISPATCH(a.dtype, F);
#undef F
        }
    } else {
        int2* ranges = (int2*)workspace;
        float* part_o = (float*)((char*)workspace + sh.part_o);
        float2* part_ml = (float2*)((char*)workspace + sh.part_ml);
        const int range_tiles = (a.max_k + 63) / 64;
        if (a.q_doc && range_tiles) doc_ranges<<<(unsigned)(((long)a.n_seq * range_tiles + 3) / 4), 256, 0, hs>>>(a, range_tiles, ranges);
#define F(T) launch_fwd_dim<T>(hs, a, sh, ranges, part_o, part_ml); \
        if (sh.splits > 1) attn_join<T><<<(unsigned)(((long)a.n_seq * a.max_q * a.n_head + 3) / 4), 256, 0, hs>>>(a, sh, part_o, part_ml);
        SEQ_DISPATCH(a.dtype, F);
#undef F
    }
    BIGC_LAUNCH_CHECK("seq_attn_fwd");
    return BIGC_OK;
}

extern "C" int bigc_seq_attn_bwd(void* stream, const bigc_seq_attn* ap, void* workspace, size_t workspace_bytes) {
    const char* who = "seq_attn_bwd";
    int rc = check_args(ap, who);
    if (rc != BIGC_OK) return rc;
    const bigc_seq_attn a = *ap;
    if ((rc = check_rows(a, who, "q", a.q, a.ldq, a.hsq, a.n_q, a.n_head)) != BIGC_OK) return rc;
    if ((rc = check_rows(a, who, "k", a.k, a.ldk, a.hsk, a.n_k, a.n_kv_head)) != BIGC_OK) return rc;
    if ((rc = check_rows(a, who, "v", a.v, a.ldv, a.hsv, a.n_k, a.n_kv_head)) != BIGC_OK) return rc;
    if (!a.o32 && (rc = check_rows(a, who, "o", a.o, a.ldo, a.hso, a.n_q, a.n_head)) != BIGC_OK) return rc;
    if ((rc = check_rows(a, who, "d_o", a.d_o, a.lddo, a.hsdo, a.n_q, a.n_head)) != BIGC_OK) return rc;
    if ((rc = check_rows(a, who, "dq", a.dq, a.lddq, a.hsdq, a.n_q, a.n_head)) != BIGC_OK) return rc;
    if ((rc = check_rows(a, who, "dk", a.dk, a.lddk, a.hsdk, a.n_k, a.n_kv_head)) != BIGC_OK) return rc;
    if ((rc = check_rows(a, who, "dv", a.dv, a.lddv, a.hsdv, a.n_k, a.n_kv_head)) != BIGC_OK) return rc;
    BIGC_CHECK_ARG(a.n_q == 0 || (a.stats && (uintptr_t)a.stats % 8 == 0), "%s: stats is NULL or not a multiple of 8 bytes", who);
    BIGC_CHECK_ARG(!a.d_rel_table || a.rel_table, "%s: d_rel_table without rel_table", who);
    const Plan p = plan_of(a);
    if (workspace_bytes < p.total || (p.total && (!workspace || (uintptr_t)workspace % 16)))
        return bigc_fail(BIGC_ERR_WORKSPACE, "%s: workspace of %zu bytes, %zu needed", who, workspace_bytes, p.total);
    hipStream_t hs = (hipStream_t)stream;
    ProfScope prof(stream, FAM_ATTN_BWD, 0, 0);
    float* delta = (float*)workspace;
    float* by_dist = (float*)((char*)workspace + p.by_dist);
    const long nk = (long)a.n_seq * a.max_k * a.n_kv_head;
    const size_t lds = a.d_rel_table ? sizeof(float) * (2 * a.bias_radius + 1) : 0;
#define F(T) \
    if (a.zero_rest && a.n_q) zero_rows<T><<<256, 256, 0, hs>>>((T*)a.dq, a.lddq, a.hsdq, a.n_q, a.n_head, a.head_dim, a.q_off, a.n_seq); \
    if (a.zero_rest && a.n_k) zero_rows<T><<<256, 256, 0, hs>>>((T*)a.dk, a.lddk, a.hsdk, a.n_k, a.n_kv_head, a.head_dim, a.k_off, a.n_seq); \
    if (a.zero_rest && a.n_k) zero_rows<T><<<256, 256, 0, hs>>>((T*)a.dv, a.lddv, a.hsdv, a.n_k, a.n_kv_head, a.head_dim, a.k_off, a.n_seq); \
    if (a.n_q) rows_delta<T><<<(unsigned)(a.n_q * a.n_head), 64, 0, hs>>>(a, delta); \
    if ((a.n_q && a.n_seq) || a.d_rel_table) rows_dq<T><<<BIN_BLOCKS * a.n_head, 64, lds, hs>>>(a, delta, by_dist); \
    if (nk && a.n_k) rows_dkv<T><<<(unsigned)nk, 64, 0, hs>>>(a, delta);
    SEQ_DISPATCH(a.dtype, F);
#undef F
    if (a.d_rel_table) rel_table_grad<<<a.n_bucket * a.n_head, 256, 0, hs>>>(a, by_dist, BIN_BLOCKS);
    BIGC_LAUNCH_CHECK("seq_attn_bwd");
    return BIGC_OK;
}
