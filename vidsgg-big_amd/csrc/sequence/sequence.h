// Shared parts of the sequence operators (attention over ordered rows, head norm + rotation).
#pragma once
#include "../common.h"
#include "../prof.h"

typedef __bf16 bf16_t;
typedef _Float16 f16_t;

static inline int seq_size(int dtype) { return dtype == BIGC_F32 ? 4 : 2; }

// whether two of `rows` x `heads` pieces of hd elements at r ld + h hs share a place, as outputs must not (strides not negative; one row's or one head's is not looked at)
static inline bool rows_overlap(int64_t ld, int64_t hs, int hd, int64_t rows, int heads) {
    if (rows > 1 && ld < hd) return true;
    if (heads == 1) return false;
    if (hs < hd) return true;
    if (rows <= 1 || ld >= (heads - 1) * hs + hd || hs >= (rows - 1) * ld + hd) return false;       // heads inside rows, or rows inside heads
    for (int64_t h = 1; h < heads; ++h)
        for (int64_t r = h * hs / ld, end = r + 2; r < end && r < rows; ++r)
            if (r * ld - h * hs < hd && h * hs - r * ld < hd) return true;
    return false;
}

// the place of sequence s: rows cut to what the tensors hold and lengths to what the launch was sized for, so that no offset leads outside
struct SeqSpan { int q0, nq, k0, nk; };
__device__ __forceinline__ SeqSpan seq_span(const bigc_seq_attn& a, int s) {
    const int q0 = min(max(a.q_off[s], 0), (int)a.n_q), q1 = min(max(a.q_off[s + 1], q0), (int)a.n_q);
    const int k0 = min(max(a.k_off[s], 0), (int)a.n_k), k1 = min(max(a.k_off[s + 1], k0), (int)a.n_k);
    return {q0, min(q1 - q0, a.max_q), k0, min(k1 - k0, a.max_k)};
}
