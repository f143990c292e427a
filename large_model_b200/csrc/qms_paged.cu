// qms_paged.cu - a paged KV cache on B200 (sm_100a): the append of new tokens with QK-norm and rotation
// (src/model.c:436-462 on one contiguous cache), and the C entries of the paged operators.
#include <math.h>
#include <string.h>

#include "qms_moe.cuh"
#include "qms_paged.cuh"

namespace qms {

// ---- append --------------------------------------------------------------------------------------
// One warp per (token, head row of q | k | v): y = R(pos) (w * x / sqrt(mean x^2 + eps)) for q and k, v
// unchanged. The mean's sum is held in double and the steps are k_qk_rope's, so a paged cache
// holds the same values as the model's contiguous one.
template <int D, typename KT>
__global__ void __launch_bounds__(256) k_paged_append(const Paged a, const float *qkv, int64_t ldqkv, const float *q_norm,
                                                      const float *k_norm, float eps, const float *rope_cos,
                                                      const float *rope_sin, int n_rope, float *q, int64_t ldq) {
    constexpr int J = D / 32, JH = J / 2;
    const int lane = threadIdx.x & 31, hh = blockIdx.y * 8 + (threadIdx.x >> 5), t = blockIdx.x;
    pdl_trigger();
    pdl_wait();
    if (hh >= a.H + 2 * a.Hk) return;
    const int b = paged_seq_of(a, t);
    if (b >= a.n_seq) return;                                   // padding
    int t0, n, kv;
    const bool ok = paged_seq(a, b, t0, n, kv);
    if (ok && (t < t0 || t >= t0 + n)) return;                  // before the first sequence's rows
    const int p = kv - n + (t - t0);
    if (!ok || p < 0 || p >= n_rope) {
        if (lane == 0 && hh == 0) paged_err(a, QMS_PAGED_ELEN);
        return;
    }
    const int64_t at = paged_at(a, a.table + (int64_t)b * a.table_stride, p);
    if (at < 0) {
        if (lane == 0 && hh == 0) paged_err(a, QMS_PAGED_EPAGE);
        return;
    }
    const float *row = qkv + t * ldqkv + hh * D;
    float x[J];
#pragma unroll
    for (int j = 0; j < J; j++) x[j] = row[lane + 32 * j];
    if (hh < a.H + a.Hk) {
        const float *nw = hh < a.H ? q_norm : k_norm;
        float w[J], c[JH], s[JH];
#pragma unroll
        for (int j = 0; j < J; j++) w[j] = nw[lane + 32 * j];
#pragma unroll
        for (int j = 0; j < JH; j++) {
            c[j] = rope_cos[(int64_t)p * (D / 2) + lane + 32 * j];
            s[j] = rope_sin[(int64_t)p * (D / 2) + lane + 32 * j];
        }
        norm_rope_pre<D>(x, w, c, s, eps);
    }
    if (hh < a.H) {
#pragma unroll
        for (int j = 0; j < J; j++) q[t * ldq + hh * D + lane + 32 * j] = x[j];
        return;
    }
    const int kh = hh < a.H + a.Hk ? hh - a.H : hh - a.H - a.Hk;
    KT *dst = reinterpret_cast<KT *>((hh < a.H + a.Hk ? a.k : a.v) + at + kh * a.head_stride);
#pragma unroll
    for (int j = 0; j < J; j++) kv_st(dst + lane + 32 * j, x[j]);
}

// ---- host ----------------------------------------------------------------------------------------
// The two descriptors, checked, as the kernels take them.
static int paged_args(const char *who, const QmsCudaPages *pg, const QmsCudaPagedBatch *bt, int n_head, int *err, Paged &a) {
    QMS_REQUIRE(pg && bt, QMS_CUDA_EINVAL, "%s: NULL descriptor", who);
    QMS_REQUIRE(pg->type == QMS_T_F32 || pg->type == QMS_T_F16, QMS_CUDA_EUNSUPPORTED, "%s: cache type %d (F32 or F16)",
                who, pg->type);
    QMS_REQUIRE(pg->head_dim == 64 || pg->head_dim == 128, QMS_CUDA_EUNSUPPORTED, "%s: head_dim %d (64 or 128 supported)",
                who, pg->head_dim);
    QMS_REQUIRE(pg->n_pages > 0 && pg->n_head_kv > 0 && pg->page_size > 0 && (pg->page_size & (pg->page_size - 1)) == 0,
                QMS_CUDA_EINVAL, "%s: pages need n_pages > 0, n_head_kv > 0 and a page size that is a power of two", who);
    QMS_REQUIRE(n_head > 0 && n_head % pg->n_head_kv == 0 && n_head <= 1024, QMS_CUDA_EINVAL,
                "%s: %d q heads over %d kv heads", who, n_head, pg->n_head_kv);
    const int64_t es = pg->type == QMS_T_F16 ? 2 : 4;
    QMS_REQUIRE(pg->k && pg->v && ((uintptr_t)pg->k & 15) == 0 && ((uintptr_t)pg->v & 15) == 0, QMS_CUDA_EINVAL,
                "%s: K and V must be 16-byte aligned device memory", who);
    QMS_REQUIRE(pg->page_stride >= 0 && pg->pos_stride >= 0 && pg->head_stride >= 0 && pg->page_stride * es % 16 == 0 &&
                    pg->pos_stride * es % 16 == 0 && pg->head_stride * es % 16 == 0,
                QMS_CUDA_EINVAL, "%s: strides must be multiples of 16 bytes, none negative", who);
    QMS_REQUIRE(bt->n_seq >= 0 && bt->n_tok >= 0 && bt->n_tok <= (1 << 20) && bt->n_seq <= (1 << 20), QMS_CUDA_EINVAL,
                "%s: n_seq %d, n_tok %d", who, bt->n_seq, bt->n_tok);
    QMS_REQUIRE(bt->max_q >= 0 && bt->max_kv >= 0 && bt->prefix_len >= 0 && bt->table_stride >= 0, QMS_CUDA_EINVAL,
                "%s: negative max_q, max_kv, prefix_len or table_stride", who);
    const int64_t cap = (int64_t)bt->table_stride * pg->page_size;
    QMS_REQUIRE(bt->max_kv <= cap && bt->prefix_len <= cap, QMS_CUDA_EINVAL,
                "%s: max_kv %d and prefix_len %d need pages in the table (%d of %d positions)", who, bt->max_kv,
                bt->prefix_len, bt->table_stride, pg->page_size);
    QMS_REQUIRE(bt->n_seq == 0 || (bt->q_start && bt->kv_len && (bt->table || bt->table_stride == 0)), QMS_CUDA_EINVAL,
                "%s: NULL q_start, kv_len or table", who);
    QMS_REQUIRE((((uintptr_t)bt->q_start | (uintptr_t)bt->kv_len | (uintptr_t)bt->table | (uintptr_t)err) & 3) == 0,
                QMS_CUDA_EINVAL, "%s: misaligned int array", who);
    a.q_start = bt->q_start;
    a.kv_len = bt->kv_len;
    a.table = bt->table;
    a.n_seq = bt->n_seq;
    a.n_tok = bt->n_tok;
    a.table_stride = bt->table_stride;
    a.max_q = bt->max_q;
    a.max_kv = bt->max_kv;
    a.prefix = bt->n_seq > 0 ? bt->prefix_len : 0;
    a.k = (char *)pg->k;
    a.v = (char *)pg->v;
    a.page_stride = pg->page_stride * es;
    a.pos_stride = pg->pos_stride * es;
    a.head_stride = pg->head_stride * es;
    a.n_pages = pg->n_pages;
    a.page_log = 0;
    while ((1 << a.page_log) < pg->page_size) a.page_log++;
    a.H = n_head;
    a.Hk = pg->n_head_kv;
    a.G = n_head / pg->n_head_kv;
    a.err = err;
    return QMS_CUDA_OK;
}

static int paged_rows(const char *who, const char *what, const void *p, int64_t ld, int64_t cols) {
    QMS_REQUIRE(p && ((uintptr_t)p & 15) == 0 && ld >= cols && ld % 4 == 0, QMS_CUDA_EINVAL,
                "%s: %s rows must be 16-byte aligned device memory, at least %lld floats apart", who, what, (long long)cols);
    return QMS_CUDA_OK;
}

}  // namespace qms

using namespace qms;

extern "C" {

int qms_cuda_paged_append(const QmsCudaPages *pages, const QmsCudaPagedBatch *batch, const float *qkv, int64_t ldqkv,
                          int n_head, const float *q_norm, const float *k_norm, float eps, const float *rope_cos,
                          const float *rope_sin, int n_rope, float *q, int64_t ldq, int *err, void *stream) {
    clear_error();
    Paged a;
    int rc = paged_args("paged_append", pages, batch, n_head, err, a);
    if (rc) return rc;
    if (a.n_tok == 0 || a.n_seq == 0) return QMS_CUDA_OK;
    const int D = pages->head_dim;
    if ((rc = paged_rows("paged_append", "qkv", qkv, ldqkv, (int64_t)(n_head + 2 * a.Hk) * D))) return rc;
    if ((rc = paged_rows("paged_append", "q", q, ldq, (int64_t)n_head * D))) return rc;
    QMS_REQUIRE(q_norm && k_norm && rope_cos && rope_sin && n_rope > 0, QMS_CUDA_EINVAL,
                "paged_append: NULL norm weights or rotation tables");
    const dim3 grid(a.n_tok, (n_head + 2 * a.Hk + 7) / 8);
#define QMS_APPEND(D_, KT)                                                                                        \
    QMS_CK(launch_pdl(k_paged_append<D_, KT>, grid, dim3(256), 0, (cudaStream_t)stream, a, qkv, ldqkv, q_norm, k_norm, \
                      eps, rope_cos, rope_sin, n_rope, q, ldq))
    if (pages->type == QMS_T_F16) {
        if (D == 128) QMS_APPEND(128, __half); else QMS_APPEND(64, __half);
    } else {
        if (D == 128) QMS_APPEND(128, float); else QMS_APPEND(64, float);
    }
#undef QMS_APPEND
    return QMS_CUDA_OK;
}

int64_t qms_cuda_paged_attention_ws(const QmsCudaPages *pages, const QmsCudaPagedBatch *batch, int n_head) {
    Paged a;
    const int rc = paged_args("paged_attention_ws", pages, batch, n_head, nullptr, a);
    if (rc) return rc;
    PagedPlan p;
    paged_plan(a, pages->type, pages->head_dim, p);
    return paged_ws_bytes(a, pages->head_dim, p);
}

int qms_cuda_paged_attention(const QmsCudaPages *pages, const QmsCudaPagedBatch *batch, const float *q, int64_t ldq,
                             int n_head, float scale, float *out, int64_t ldo, void *ws, int64_t ws_bytes, int *err,
                             void *stream) {
    clear_error();
    Paged a;
    int rc = paged_args("paged_attention", pages, batch, n_head, err, a);
    if (rc) return rc;
    if (a.n_tok == 0) return QMS_CUDA_OK;
    const int D = pages->head_dim;
    if ((rc = paged_rows("paged_attention", "q", q, ldq, (int64_t)n_head * D))) return rc;
    if ((rc = paged_rows("paged_attention", "out", out, ldo, (int64_t)n_head * D))) return rc;
    PagedPlan p;
    paged_plan(a, pages->type, D, p);
    const int64_t need = paged_ws_bytes(a, D, p);
    QMS_REQUIRE(need == 0 || (ws && ((uintptr_t)ws & 255) == 0 && ws_bytes >= need), QMS_CUDA_EINVAL,
                "paged_attention: needs a 256-byte aligned workspace of %lld bytes", (long long)need);
    return launch_paged_attention(a, pages->type, D, p, q, ldq, scale, out, ldo, ws, (cudaStream_t)stream);
}

}  // extern "C"
