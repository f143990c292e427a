// qms_paged.cuh - the paged KV cache as the kernels see it (qms_paged*.cu). Not part of the C ABI.
#pragma once

#include "qms_kv.cuh"

namespace qms {

// A pool of pages and a batch of new tokens, flattened (QmsCudaPages, QmsCudaPagedBatch).
struct Paged {
    const int *q_start, *kv_len, *table;
    int n_seq, n_tok, table_stride, max_q, max_kv, prefix;
    char *k, *v;
    int64_t page_stride, pos_stride, head_stride;    // bytes
    int n_pages, page_log;
    int H, Hk, G;                                    // q heads, kv heads, q heads per kv head
    int *err;
};

__device__ __forceinline__ void paged_err(const Paged &a, int bit) {
    if (a.err) atomicOr(a.err, bit);
}

// The sequence that token row t belongs to, by the whole warp: how many sequences end at or before t
// (independent loads: one round trip up to 32 sequences, not a chain of dependent ones).
__device__ __forceinline__ int paged_seq_of(const Paged &a, int t) {
    int n = 0;
    for (int b = threadIdx.x & 31; b < a.n_seq; b += 32) n += __ldg(a.q_start + b + 1) <= t;
    return __reduce_add_sync(kFull, n);
}

// Sequence b's rows [t0, t0 + n) and cache length. False (n = kv = 0) when the batch arrays do not make
// sense for it; such a sequence counts as idle.
__device__ __forceinline__ bool paged_seq(const Paged &a, int b, int &t0, int &n, int &kv) {
    t0 = __ldg(a.q_start + b);
    n = __ldg(a.q_start + b + 1) - t0;
    kv = __ldg(a.kv_len + b);
    if (t0 >= 0 && n >= 0 && n <= a.max_q && n <= a.n_tok - t0 && kv >= 0 && kv <= a.max_kv) return true;
    n = kv = 0;
    return false;
}

// Byte offset of position p of table row `row` in the K / V pool, or -1 on a bad page id.
// 0 <= p < table_stride * page_size.
__device__ __forceinline__ int64_t paged_at(const Paged &a, const int *row, int p) {
    const int page = __ldg(row + (p >> a.page_log));
    if ((unsigned)page >= (unsigned)a.n_pages) return -1;
    return page * a.page_stride + (p & ((1 << a.page_log) - 1)) * a.pos_stride;
}

}  // namespace qms
