// qms_verify.cu - probabilities of logits rows and the verification of drafted tokens on B200 (sm_100a).
//
// The reference draws one token from one row on the host (sample(), src/chat.c:36-69); it has no drafts.
#include <math.h>
#include <string.h>

#include "qms_moe.cuh"

namespace qms {

constexpr int kRowThreads = 1024;

// ---- probabilities -------------------------------------------------------------------------------
// p = exp((l - max) / temp) / sum, one CTA per row.
__global__ void __launch_bounds__(kRowThreads) k_probs(const float *l, int64_t ldl, int V, float temp, float *p, int64_t ldp) {
    __shared__ float s_v[32];
    __shared__ int s_i[32];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    pdl_trigger();
    pdl_wait();
    l += blockIdx.x * ldl;
    p += blockIdx.x * ldp;
    float m = -INFINITY;
    int at = V;                                            // first index of the maximum (NaN never is)
    for (int i = tid; i < V; i += kRowThreads) {
        const float x = l[i];
        if (x > m || (at == V && x == m)) {
            m = x;
            at = i;
        }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const float om = __shfl_xor_sync(0xffffffffu, m, o);
        const int oi = __shfl_xor_sync(0xffffffffu, at, o);
        if (om > m || (om == m && oi < at)) {
            m = om;
            at = oi;
        }
    }
    if (lane == 0) {
        s_v[warp] = m;
        s_i[warp] = at;
    }
    __syncthreads();
    for (int w = 0; w < 32; w++)
        if (s_v[w] > m || (s_v[w] == m && s_i[w] < at)) {
            m = s_v[w];
            at = s_i[w];
        }
    if (!(temp > 0.0f)) {
        const bool none = m == -INFINITY;
        __syncthreads();
        for (int i = tid; i < V; i += kRowThreads) p[i] = i == at && !none ? 1.0f : 0.0f;
        return;
    }
    const float base = m == -INFINITY ? 0.0f : m;
    float z = 0.0f;                                        // in groups of 32: no long chain of roundings
    for (int i = tid; i < V; i += 32 * kRowThreads) {
        float g = 0.0f;
        for (int j = i; j < V && j < i + 32 * kRowThreads; j += kRowThreads) g += expf(__fdiv_rn(l[j] - base, temp));
        z += g;
    }
    z = warp_sum(z);
    __syncthreads();
    if (lane == 0) s_v[warp] = z;
    __syncthreads();
    z = 0.0f;
    for (int w = 0; w < 32; w++) z += s_v[w];
    for (int i = tid; i < V; i += kRowThreads) p[i] = z == 0.0f ? 0.0f : __fdiv_rn(expf(__fdiv_rn(l[i] - base, temp)), z);
}

// ---- verification --------------------------------------------------------------------------------
struct VerifyArgs {
    const float *p, *q, *u;
    int64_t ldp, ldq;
    int p_rows, n_seq, max_draft, V;
    const int *row_start, *draft, *n_draft;
    int *n_accept, *tokens, *err;
};

__device__ __forceinline__ void verify_err(const VerifyArgs &a, int bit) {
    if (a.err) atomicOr(a.err, bit);
}

// A probability as a whole number of 2^-40 (round half to even; NaN and negative: 0, above 1: 2^40).
__device__ __forceinline__ unsigned long long verify_weight(float r) {
    return r > 0.0f ? (unsigned long long)__float2ll_rn(fminf(r, 1.0f) * 1099511627776.0f) : 0ull;
}

// One CTA per sequence: the drafts in order, then the next token by inversion of the cumulative weights.
__global__ void __launch_bounds__(kRowThreads) k_verify(const VerifyArgs a) {
    __shared__ unsigned long long s_w[kRowThreads];
    __shared__ int s_n, s_pick;
    const int b = blockIdx.x, tid = threadIdx.x, N = a.max_draft;
    pdl_trigger();
    pdl_wait();
    const int nd = a.n_draft ? a.n_draft[b] : N;
    const int r0 = a.row_start ? a.row_start[b] : b * (N + 1);
    int *tok = a.tokens + (int64_t)b * (N + 1);
    if (nd < 0 || nd > N || r0 < 0 || r0 > a.p_rows - nd - 1) {
        if (tid == 0) {
            verify_err(a, QMS_PAGED_ELEN);
            a.n_accept[b] = 0;
        }
        for (int i = tid; i <= N; i += kRowThreads) tok[i] = -1;
        return;
    }
    if (tid == 0) {
        int n = 0;
        for (; n < nd; n++) {
            const int x = a.draft[(int64_t)b * N + n];
            if (x < 0 || x >= a.V) {
                verify_err(a, QMS_PAGED_ETOKEN);
                break;
            }
            const float qx = a.q ? a.q[((int64_t)b * N + n) * a.ldq + x] : 1.0f;
            if (!(__fmul_rn(a.u[(int64_t)b * (N + 1) + n], qx) < a.p[(int64_t)(r0 + n) * a.ldp + x])) break;
        }
        s_n = n;
        s_pick = -1;
    }
    __syncthreads();
    const int n = s_n, x = n < nd ? a.draft[(int64_t)b * N + n] : -1;
    const float *p = a.p + (int64_t)(r0 + n) * a.ldp;
    const float *q = x >= 0 && x < a.V && a.q ? a.q + ((int64_t)b * N + n) * a.ldq : nullptr;
    const int per = (a.V + kRowThreads - 1) / kRowThreads, i0 = min(a.V, tid * per), i1 = min(a.V, i0 + per);
    const float u = a.u[(int64_t)b * (N + 1) + N];
    for (int pass = 0; pass < 2; pass++) {                  // the remainder of p over q; then p itself
        auto weight = [&](int i) {
            float r = p[i];
            if (pass == 0 && q) r = __fsub_rn(r, q[i]);
            if (pass == 0 && !a.q && i == x) r = 0.0f;
            return verify_weight(r);
        };
        unsigned long long w = 0, before = 0, total = 0;
        for (int i = i0; i < i1; i++) w += weight(i);
        s_w[tid] = w;
        __syncthreads();
        for (int i = 0; i < kRowThreads; i++) {
            if (i < tid) before += s_w[i];
            total += s_w[i];
        }
        __syncthreads();
        if (total == 0) continue;
        const unsigned long long m = (unsigned long long)floorf(fminf(fmaxf(u, 0.0f), 0.99999994f) * 16777216.0f);
        const unsigned long long want = (total >> 24) * m + (((total & 0xFFFFFFull) * m) >> 24);     // floor(total u)
        if (before <= want && want < before + w) {
            int i = i0;
            for (; i < i1; i++) {
                before += weight(i);
                if (before > want) break;
            }
            s_pick = i;
        }
        break;
    }
    __syncthreads();
    if (tid == 0) {
        a.n_accept[b] = n;
        if (s_pick < 0) verify_err(a, QMS_PAGED_EMASS);
    }
    for (int i = tid; i <= N; i += kRowThreads) tok[i] = i < n ? a.draft[(int64_t)b * N + i] : i == n ? s_pick : -1;
}

}  // namespace qms

using namespace qms;

extern "C" {

int qms_cuda_probs(const float *logits, int64_t ldl, int rows, int vocab, float temp, float *p, int64_t ldp, void *stream) {
    clear_error();
    QMS_REQUIRE(logits && p && vocab > 0 && rows >= 0, QMS_CUDA_EINVAL, "probs: NULL logits or p, vocab <= 0 or rows < 0");
    QMS_REQUIRE(ldl >= vocab && ldp >= vocab && (p != logits || ldp == ldl), QMS_CUDA_EINVAL,
                "probs: rows of %d need ldl and ldp of at least that (in place: equal ones)", vocab);
    QMS_REQUIRE(!isnan(temp), QMS_CUDA_EINVAL, "probs: temp is NaN");
    if (rows == 0) return QMS_CUDA_OK;
    QMS_CK(launch_pdl(k_probs, dim3(rows), dim3(kRowThreads), 0, (cudaStream_t)stream, logits, ldl, vocab, temp, p, ldp));
    return QMS_CUDA_OK;
}

int qms_cuda_verify(const float *p, int64_t ldp, int p_rows, const int *row_start, const float *q, int64_t ldq,
                    const int *draft, const int *n_draft, int n_seq, int max_draft, int vocab, const float *u,
                    int *n_accept, int *tokens, int *err, void *stream) {
    clear_error();
    QMS_REQUIRE(p && u && n_accept && tokens && (draft || max_draft == 0), QMS_CUDA_EINVAL, "verify: NULL argument");
    QMS_REQUIRE(n_seq >= 0 && max_draft >= 0 && max_draft <= 1024 && p_rows >= 0 && vocab > 0 && vocab <= (1 << 22),
                QMS_CUDA_EINVAL, "verify: n_seq %d, max_draft %d (at most 1024), p_rows %d, vocab %d (at most %d)", n_seq,
                max_draft, p_rows, vocab, 1 << 22);
    QMS_REQUIRE((int64_t)n_seq * (max_draft + 1) < (1ll << 31), QMS_CUDA_EINVAL, "verify: too many sequences");
    QMS_REQUIRE(ldp >= vocab && (!q || ldq >= vocab), QMS_CUDA_EINVAL, "verify: rows of %d need ldp and ldq of at least that",
                vocab);
    if (n_seq == 0) return QMS_CUDA_OK;
    VerifyArgs a;
    memset(&a, 0, sizeof a);
    a.p = p;
    a.q = q;
    a.u = u;
    a.ldp = ldp;
    a.ldq = ldq;
    a.p_rows = p_rows;
    a.n_seq = n_seq;
    a.max_draft = max_draft;
    a.V = vocab;
    a.row_start = row_start;
    a.draft = draft;
    a.n_draft = n_draft;
    a.n_accept = n_accept;
    a.tokens = tokens;
    a.err = err;
    QMS_CK(launch_pdl(k_verify, dim3(n_seq), dim3(kRowThreads), 0, (cudaStream_t)stream, a));
    return QMS_CUDA_OK;
}

}  // extern "C"
