// Attention over ordered rows: entry points and checks.
#include "attention_bwd.h"

namespace {

// ---- host -----------------------------------------------------------------------------------------------------------------------

int check_rows(const bigc_seq_attn& a, const char* who, const char* what, const void* p, int64_t ld, int64_t hs, int64_t rows, int heads) {
    const int64_t e = 16 / seq_size(a.dtype);
    if (rows == 0) return BIGC_OK;
    BIGC_CHECK_ARG(p, "%s: %s is NULL", who, what);
    BIGC_CHECK_ARG((uintptr_t)p % 16 == 0 && (rows == 1 || ld % e == 0) && (heads == 1 || hs % e == 0),
                   "%s: %s: address, row stride %ld and head stride %ld have to be multiples of 16 bytes", who, what, (long)ld, (long)hs);
    BIGC_CHECK_ARG((rows == 1 || (ld >= 0 && ld <= (1 << 22))) && (heads == 1 || hs >= 0), "%s: %s: row stride %ld (0 to 2^22 elements), head stride %ld", who, what, (long)ld, (long)hs);
    return BIGC_OK;
}

int check_out(const bigc_seq_attn& a, const char* who, const char* what, const void* p, int64_t ld, int64_t hs, int64_t rows, int heads) {
    const int rc = check_rows(a, who, what, p, ld, hs, rows, heads);
    if (rc != BIGC_OK || rows == 0) return rc;
    BIGC_CHECK_ARG(!rows_overlap(ld, hs, a.head_dim, rows, heads), "%s: %s: rows or heads overlap (row stride %ld, head stride %ld)", who, what, (long)ld, (long)hs);
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
    // (places, their distances and what a tile or a chunk adds to them are int32)
    BIGC_CHECK_ARG((long)a.max_q + a.max_k <= (1l << 31) - (1 << 20), "%s: %d queries and %d keys are too far apart", who, a.max_q, a.max_k);
    BIGC_CHECK_ARG((double)a.n_q * a.n_head < 2147483648.0, "%s: %ld rows of %d heads are too many", who, (long)a.n_q, a.n_head);
    BIGC_CHECK_ARG(a.n_seq == 0 || (a.q_off && a.k_off), "%s: offsets are NULL", who);
    BIGC_CHECK_ARG(a.window_left >= -1 && a.window_right >= -1, "%s: window (%d, %d)", who, a.window_left, a.window_right);
    BIGC_CHECK_ARG(isfinite(a.scale) && isfinite(a.softcap) && a.softcap >= 0.f, "%s: scale %g, softcap %g", who, a.scale, a.softcap);
    BIGC_CHECK_ARG(a.softcap == 0.f || isfinite(a.scale / a.softcap * 4.f), "%s: softcap %g too small for scale %g", who, a.softcap, a.scale);
    BIGC_CHECK_ARG(!a.q_doc == !a.k_doc || a.n_q == 0 || a.n_k == 0, "%s: q_doc and k_doc come together", who);
    BIGC_CHECK_ARG(!a.rel_table == !a.rel_map, "%s: rel_table and rel_map come together", who);
    if (a.rel_table) BIGC_CHECK_ARG(a.n_bucket > 0 && a.bias_radius >= 0 && a.bias_radius <= 2047, "%s: %d buckets, radius %d (at most 2047)", who, a.n_bucket, a.bias_radius);
    BIGC_CHECK_ARG((double)a.n_seq * a.n_head < 2147483648.0 && (double)a.n_seq * a.max_q < 4294967296.0 && (double)a.n_seq * a.max_k < 4294967296.0,
                   "%s: %d sequences of up to %d queries and %d keys with %d heads are too many", who, a.n_seq, a.max_q, a.max_k, a.n_head);
    return BIGC_OK;
}

// the launches of a call: a grid holds less than 2^32 threads, 2^24 blocks of 256
int check_blocks(const bigc_seq_attn& a, const char* who, long blocks) {
    const long ranges = a.q_doc ? ((long)a.n_seq * cdiv(a.max_q > a.max_k ? a.max_q : a.max_k, 64) + 3) / 4 : 0;
    BIGC_CHECK_ARG(blocks < (1 << 24) && ranges < (1 << 24), "%s: %d sequences of up to %d queries and %d keys with %d heads need %ld blocks, too many for one launch", who,
                   a.n_seq, a.max_q, a.max_k, a.n_head, blocks > ranges ? blocks : ranges);
    return BIGC_OK;
}
int check_blocks(const bigc_seq_attn& a, const char* who, const FwdShape& sh) { return check_blocks(a, who, sh.blocks); }
int check_blocks(const bigc_seq_attn& a, const char* who, const BwdShape& sh) {
    const long q = (long)sh.q_pairs * sh.q_tiles, k = (long)sh.k_pairs * sh.k_tiles, table = a.d_rel_table ? 4l * a.n_head : 0, most = q > k ? q : k;    // (the table's blocks are of 1024)
    return check_blocks(a, who, most > table ? most : table);
}
template <typename Shape>
size_t workspace_of(const bigc_seq_attn& a, const Shape& sh) { return check_blocks(a, "seq_attn_workspace_bytes", sh) == BIGC_OK ? sh.total : 0; }

#define SEQ_DISPATCH(dtype, F) do { if ((dtype) == BIGC_F32) { F(float) } else if ((dtype) == BIGC_F16) { F(f16_t) } else { F(bf16_t) } } while (0)
}  // namespace

extern "C" size_t bigc_seq_attn_workspace_bytes(const bigc_seq_attn* a, int backward) {
    if (check_args(a, "seq_attn_workspace_bytes") != BIGC_OK) return 0;
    return backward ? workspace_of(*a, bwd_shape(*a)) : workspace_of(*a, fwd_shape(*a));
}

extern "C" int bigc_seq_attn_fwd(void* stream, const bigc_seq_attn* ap, void* workspace, size_t workspace_bytes) {
    const char* who = "seq_attn_fwd";
    int rc = check_args(ap, who);
    if (rc != BIGC_OK) return rc;
    const bigc_seq_attn a = *ap;
    if ((rc = check_rows(a, who, "q", a.q, a.ldq, a.hsq, a.n_q, a.n_head)) != BIGC_OK) return rc;
    if ((rc = check_rows(a, who, "k", a.k, a.ldk, a.hsk, a.n_k, a.n_kv_head)) != BIGC_OK) return rc;
    if ((rc = check_rows(a, who, "v", a.v, a.ldv, a.hsv, a.n_k, a.n_kv_head)) != BIGC_OK) return rc;
    if ((rc = check_out(a, who, "o", a.o, a.ldo, a.hso, a.n_q, a.n_head)) != BIGC_OK) return rc;
    BIGC_CHECK_ARG((uintptr_t)a.stats % 8 == 0 && (uintptr_t)a.o32 % 16 == 0, "%s: stats has to lie at a multiple of 8 bytes, o32 of 16", who);
    const FwdShape sh = fwd_shape(a);
    if ((rc = check_blocks(a, who, sh)) != BIGC_OK) return rc;
    if (workspace_bytes < sh.total || (sh.total && (!workspace || (uintptr_t)workspace % 16)))
        return bigc_fail(BIGC_ERR_WORKSPACE, "%s: workspace of %zu bytes, %zu needed", who, workspace_bytes, sh.total);
    if (a.n_q == 0) return BIGC_OK;
    hipStream_t hs = (hipStream_t)stream;
    ProfScope prof(stream, FAM_MHA, 0, 0);
    if (sh.blocks == 0) {                                       // no sequence, or none with a query
        if (a.zero_rest) {
#define F(T) zero_rows<T><<<256, 256, 0, hs>>>((T*)a.o, a.ldo, a.hso, a.n_q, a.n_head, a.head_dim, a.q_off, a.n_seq, a.max_q);
            SEQ_DISPATCH(a.dtype, F);
#undef F
        }
    } else {
        int2* ranges = (int2*)workspace;
        float* part_o = (float*)((char*)workspace + sh.part_o);
        float2* part_ml = (float2*)((char*)workspace + sh.part_ml);
        const int range_tiles = (a.max_k + 63) / 64;
        if (a.q_doc && range_tiles) doc_ranges<<<(unsigned)(((long)a.n_seq * range_tiles + 3) / 4), 256, 0, hs>>>(a, true, range_tiles, ranges);
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
    if ((rc = check_out(a, who, "dq", a.dq, a.lddq, a.hsdq, a.n_q, a.n_head)) != BIGC_OK) return rc;
    if ((rc = check_out(a, who, "dk", a.dk, a.lddk, a.hsdk, a.n_k, a.n_kv_head)) != BIGC_OK) return rc;
    if ((rc = check_out(a, who, "dv", a.dv, a.lddv, a.hsdv, a.n_k, a.n_kv_head)) != BIGC_OK) return rc;
    BIGC_CHECK_ARG(a.n_q == 0 || (a.stats && (uintptr_t)a.stats % 8 == 0), "%s: stats is NULL or not a multiple of 8 bytes", who);
    BIGC_CHECK_ARG(!a.d_rel_table || a.rel_table, "%s: d_rel_table without rel_table", who);
    BIGC_CHECK_ARG(!a.d_rel_table || a.dtype != BIGC_F32 || a.head_dim <= 64 || a.bias_radius <= 1023, "%s: d_rel_table of f32 heads over 64 columns: radius %d (at most 1023)", who, a.bias_radius);
    const BwdShape sh = bwd_shape(a);
    if ((rc = check_blocks(a, who, sh)) != BIGC_OK) return rc;
    if (workspace_bytes < sh.total || (sh.total && (!workspace || (uintptr_t)workspace % 16)))
        return bigc_fail(BIGC_ERR_WORKSPACE, "%s: workspace of %zu bytes, %zu needed", who, workspace_bytes, sh.total);
    hipStream_t hs = (hipStream_t)stream;
    char* ws = (char*)workspace;
    ProfScope prof(stream, FAM_ATTN_BWD, 0, 0);
    const long q_blocks = a.n_q ? (long)sh.q_pairs * sh.q_tiles : 0, k_blocks = a.n_k ? (long)sh.k_pairs * sh.k_tiles : 0;
    if (a.q_doc && q_blocks && k_blocks) {
        const int qt = cdiv(a.max_q, 64), kt = cdiv(a.max_k, 64);
        doc_ranges<<<(unsigned)(((long)a.n_seq * qt + 3) / 4), 256, 0, hs>>>(a, false, qt, (int2*)(ws + sh.q_ranges));
        doc_ranges<<<(unsigned)(((long)a.n_seq * kt + 3) / 4), 256, 0, hs>>>(a, true, kt, (int2*)(ws + sh.k_ranges));
    }
#define F(T) \
    launch_bwd_dim<typename std::conditional<std::is_same<T, float>::value, f32s, T>::type>(hs, a, sh, ws); \
    if (a.zero_rest && a.n_q && !q_blocks) zero_rows<T><<<256, 256, 0, hs>>>((T*)a.dq, a.lddq, a.hsdq, a.n_q, a.n_head, a.head_dim, a.q_off, a.n_seq, a.max_q); \
    if (a.zero_rest && a.n_k && !k_blocks) { \
        zero_rows<T><<<256, 256, 0, hs>>>((T*)a.dk, a.lddk, a.hsdk, a.n_k, a.n_kv_head, a.head_dim, a.k_off, a.n_seq, a.max_k); \
        zero_rows<T><<<256, 256, 0, hs>>>((T*)a.dv, a.lddv, a.hsdv, a.n_k, a.n_kv_head, a.head_dim, a.k_off, a.n_seq, a.max_k); \
    }
    SEQ_DISPATCH(a.dtype, F);
#undef F
    if (a.d_rel_table)
        rel_table_grad<<<a.n_head, 1024, sizeof(float) * (2 * (2 * a.bias_radius + 1) + 1024), hs>>>(a, (const float*)(ws + sh.bins), q_blocks ? a.n_seq * sh.q_tiles : 0);
    BIGC_LAUNCH_CHECK("seq_attn_bwd");
    return BIGC_OK;
}
