// qms_paged.cu - a paged KV cache on B200 (sm_100a): the append of new tokens with QK-norm and rotation
// (src/model.c:436-462 on one contiguous cache), and the C entries of the paged operators.
#include <math.h>
#include <string.h>

#include "qms_moe.cuh"
#include "qms_paged.cuh"

namespace qms {

// ---- append --------------------------------------------------------------------------------------
// A warp takes R head rows of q | k | v of one token: y = R(pos) (w * x / sqrt(mean x^2 + eps)) for q and k, v unchanged.
// The mean's sum is held in double and the steps are k_qk_rope's, each in its order, so a paged cache holds the same
// values as the model's contiguous one.
// Bound by latency for few rows (R = 1: 2.5 us for one token) and by instructions for many, most of them for the 64-bit
// mean: R = 4 rows share the exchanges of their sums and one square root and division (a lane each).
template <int R>
__device__ __forceinline__ void sum_rows(double (&v)[R], int lane) {      // the sum of v[r] over the lanes; R = 4: v[0] of row lane / 8
    if constexpr (R == 1) {
        v[0] = warp_sum_d(v[0]);
    } else {
        const bool hi = lane & 16, mid = lane & 8;
        const double a = __shfl_xor_sync(kFull, hi ? v[0] : v[2], 16), b = __shfl_xor_sync(kFull, hi ? v[1] : v[3], 16);
        const double x = (hi ? v[2] : v[0]) + a, y = (hi ? v[3] : v[1]) + b;
        v[0] = (mid ? y : x) + __shfl_xor_sync(kFull, mid ? x : y, 8);
#pragma unroll
        for (int o = 4; o > 0; o >>= 1) v[0] += __shfl_xor_sync(kFull, v[0], o);
    }
}

template <int D, typename KT, int R>
__global__ void __launch_bounds__(256) k_paged_append(const Paged a, const float *qkv, int64_t ldqkv, const float *q_norm,
                                                      const float *k_norm, float eps, const float *rope_cos,
                                                      const float *rope_sin, int n_rope, float *q, int64_t ldq) {
    static_assert(R == 1 || R == 4, "rows per warp");
    constexpr int J = D / 32, JH = J / 2;
    const int lane = threadIdx.x & 31, groups = (a.H + 2 * a.Hk + R - 1) / R, nq = a.H + a.Hk;
    const unsigned unit = blockIdx.x * 8 + (threadIdx.x >> 5);
    const int t = unit / groups, h0 = (unit - t * groups) * R;
    pdl_trigger();
    pdl_wait();
    if (t >= a.n_tok) return;
    const float *row = qkv + t * ldqkv + h0 * D;
    float x[R][J], w[J];
#pragma unroll
    for (int r = 0; r < R; r++)
#pragma unroll
        for (int j = 0; j < J; j++) x[r][j] = h0 + r < nq + a.Hk ? row[r * D + lane + 32 * j] : 0.0f;
#pragma unroll
    for (int j = 0; j < J; j++) w[j] = (h0 < a.H ? q_norm : k_norm)[lane + 32 * j];
    const int b = paged_seq_of(a, t);
    if (b >= a.n_seq) return;                                   // padding
    int t0, n, kv;
    const bool ok = paged_seq(a, b, t0, n, kv);
    if (ok && (t < t0 || t >= t0 + n)) return;                  // before the first sequence's rows
    const int p = kv - n + (t - t0);
    if (!ok || p < 0 || p >= n_rope) {
        if (lane == 0 && h0 == 0) paged_err(a, QMS_PAGED_ELEN);
        return;
    }
    const int64_t at = paged_at(a, a.table + (int64_t)b * a.table_stride, p);
    if (at < 0) {
        if (lane == 0 && h0 == 0) paged_err(a, QMS_PAGED_EPAGE);
        return;
    }
    float c[JH], s[JH];
    double inv = 0.0;
    if (h0 < nq) {
#pragma unroll
        for (int j = 0; j < JH; j++) {
            c[j] = rope_cos[(int64_t)p * (D / 2) + lane + 32 * j];
            s[j] = rope_sin[(int64_t)p * (D / 2) + lane + 32 * j];
        }
        double ss[R];
#pragma unroll
        for (int r = 0; r < R; r++) {
            ss[r] = 0.0;
#pragma unroll
            for (int j = 0; j < J; j++) ss[r] = fma((double)x[r][j], (double)x[r][j], ss[r]);
        }
        sum_rows<R>(ss, lane);
        inv = 1.0 / sqrt(ss[0] / D + (double)eps);
    }
#pragma unroll
    for (int r = 0; r < R; r++) {
        const int hh = h0 + r;
        if (hh >= nq + a.Hk) return;
        if (hh < nq) {
            if (r > 0 && hh == a.H)                             // from q to k
#pragma unroll
                for (int j = 0; j < J; j++) w[j] = k_norm[lane + 32 * j];
            rope_scaled<D>(x[r], w, c, s, R == 1 ? inv : __shfl_sync(kFull, inv, 8 * r));
        }
        if (hh < a.H) {
#pragma unroll
            for (int j = 0; j < J; j++) q[t * ldq + hh * D + lane + 32 * j] = x[r][j];
        } else {
            KT *dst = reinterpret_cast<KT *>((hh < nq ? a.k : a.v) + at + (hh < nq ? hh - a.H : hh - nq) * a.head_stride);
#pragma unroll
            for (int j = 0; j < J; j++) kv_st(dst + lane + 32 * j, x[r][j]);
        }
    }
}

template <int D, typename KT>
static int launch_append(const Paged &a, const float *qkv, int64_t ldqkv, const float *q_norm, const float *k_norm, float eps,
                         const float *rope_cos, const float *rope_sin, int n_rope, float *q, int64_t ldq, cudaStream_t s) {
    const int heads = a.H + 2 * a.Hk;
    // Four rows per warp once there are 48 for each SM. Both in us at 40 or 72 head rows per token: 4608 rows 3.56 one,
    // 3.59 four; 5120 3.4, 3.8; 9216 5.2, 4.2; 10240 5.6, 4.8; 144000 50, 29 (4.9 TB/s).
    const bool four = (int64_t)a.n_tok * heads >= 148 * 48;
    const int64_t units = (int64_t)a.n_tok * (four ? (heads + 3) / 4 : heads);
    QMS_REQUIRE(units < (1ll << 31), QMS_CUDA_EUNSUPPORTED, "paged_append: too many rows");
    const dim3 grid((unsigned)((units + 7) / 8));
    if (four) QMS_CK(launch_pdl(k_paged_append<D, KT, 4>, grid, dim3(256), 0, s, a, qkv, ldqkv, q_norm, k_norm, eps, rope_cos, rope_sin, n_rope, q, ldq));
    else QMS_CK(launch_pdl(k_paged_append<D, KT, 1>, grid, dim3(256), 0, s, a, qkv, ldqkv, q_norm, k_norm, eps, rope_cos, rope_sin, n_rope, q, ldq));
    return QMS_CUDA_OK;
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
    QMS_REQUIRE(q != qkv || ldq == ldqkv || a.n_tok == 1, QMS_CUDA_EINVAL,
                "paged_append: in place, q and qkv need rows at one distance (%lld, %lld)", (long long)ldq, (long long)ldqkv);
    QMS_REQUIRE(q_norm && k_norm && rope_cos && rope_sin && n_rope > 0, QMS_CUDA_EINVAL,
                "paged_append: NULL norm weights or rotation tables");
#define QMS_APPEND(D_, KT) \
    return launch_append<D_, KT>(a, qkv, ldqkv, q_norm, k_norm, eps, rope_cos, rope_sin, n_rope, q, ldq, (cudaStream_t)stream)
    if (pages->type == QMS_T_F16) {
        if (D == 128) QMS_APPEND(128, __half); else QMS_APPEND(64, __half);
    } else {
        if (D == 128) QMS_APPEND(128, float); else QMS_APPEND(64, float);
    }
#undef QMS_APPEND
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
