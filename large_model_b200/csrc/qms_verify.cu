// qms_verify.cu - probabilities of logits rows and the verification of drafted tokens on B200 (sm_100a).
//
// The reference draws one token from one row on the host (sample(), src/chat.c:36-69); it has no drafts.
#include <cooperative_groups.h>
#include <math.h>
#include <string.h>

#include "qms_rows.cuh"

namespace cg = cooperative_groups;

namespace qms {

// ---- probabilities -------------------------------------------------------------------------------
// (m, i): a maximum and its first index
__device__ __forceinline__ void join_mi(float &m, int &i, float om, int oi) {
    if (om > m || (om == m && oi < i)) {
        m = om;
        i = oi;
    }
}

// p = 2^((l - max) c) / sum, c = log2(e) / temp; GREEDY: 1 at the first maximum. Grid: rows x
// cluster. A slice comes into shared memory by cp.async (16 bytes at a time where the row is aligned); its
// weights replace it there, relative to the slice's own maximum, and one exchange over the cluster gives every
// CTA the common factor. The order of the additions does not depend on the row's address.
// Bound by memory: 320 rows of 151,936 move 389 MB in 84 us, 4.6 TB/s, 0.72 of a plain copy (reading all of a row comes before
// writing any of it; three CTAs per SM overlap). One row: 6.3 us, launch, one round trip, the exchange.
template <bool GREEDY>
__global__ void __launch_bounds__(kProbsThreads, 3) k_probs(const float *l, int64_t ldl, int V, float c, float *p, int64_t ldp) {
    extern __shared__ __align__(16) float x[];
    __shared__ float s_m[kProbsWarps], s_z[kProbsWarps], s_cm[kRowCtas], s_cz[kRowCtas];
    __shared__ int s_i[kProbsWarps], s_ci[kRowCtas];
    cg::cluster_group cl = cg::this_cluster();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, rank = (int)cl.block_rank(), nc = (int)cl.num_blocks();
    auto started = cl.barrier_arrive();                    // waited for before the first write to another CTA
    pdl_trigger();
    pdl_wait();
    const int64_t r = blockIdx.x / nc;
    const int groups = (V + 3) >> 2;                       // slices start at multiples of 4 values
    const int lo = (int)((int64_t)groups * rank / nc) * 4, n = min(V, (int)((int64_t)groups * (rank + 1) / nc) * 4) - lo;
    l += r * ldl + lo;
    p += r * ldp + lo;
    const int kept = min(n, kProbsKeep), n4 = (kept + 3) >> 2;
    float4 *x4 = reinterpret_cast<float4 *>(x);
    const bool vec = ((uintptr_t)l & 15) == 0;
    if (vec) {
        for (int i = tid; i < kept >> 2; i += kProbsThreads) cp_async16(x + 4 * i, l + 4 * i);
        if (tid < (kept & 3)) cp_async4(x + (kept & ~3) + tid, l + (kept & ~3) + tid);
    } else {
#pragma unroll 4
        for (int i = tid; i < kept; i += kProbsThreads) cp_async4(x + i, l + i);
    }
    if (tid >= kept && tid < 4 * n4) x[tid] = -INFINITY;   // (a slice below one group)
    for (int i = max(kept, kProbsThreads) + tid; i < 4 * n4; i += kProbsThreads) x[i] = -INFINITY;
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncthreads();

    float m = -INFINITY;
    int at = 0x7fffffff;
    auto maximum = [&](float y, int i) {
        if constexpr (GREEDY) {
            if (y > m) at = lo + i;
        }
        m = fmaxf(m, y);
    };
#pragma unroll 4
    for (int i = tid; i < n4; i += kProbsThreads) {
        const float4 y = x4[i];
        maximum(y.x, 4 * i);
        maximum(y.y, 4 * i + 1);
        maximum(y.z, 4 * i + 2);
        maximum(y.w, 4 * i + 3);
    }
    for (int i = kept + tid; i < n; i += kProbsThreads) maximum(l[i], i);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const float om = __shfl_xor_sync(kFull, m, o);
        if constexpr (GREEDY) join_mi(m, at, om, __shfl_xor_sync(kFull, at, o));
        else m = fmaxf(m, om);
    }
    if (lane == 0) s_m[warp] = m, s_i[warp] = at;
    __syncthreads();
    m = s_m[lane & (kProbsWarps - 1)], at = s_i[lane & (kProbsWarps - 1)];
#pragma unroll
    for (int o = kProbsWarps / 2; o > 0; o >>= 1) {
        const float om = __shfl_xor_sync(kFull, m, o);
        if constexpr (GREEDY) join_mi(m, at, om, __shfl_xor_sync(kFull, at, o));
        else m = fmaxf(m, om);
    }
    // the slice's weights under its own maximum
    const float M = m == -INFINITY ? 0.0f : m;
    float z = 0.0f;
    if constexpr (!GREEDY) {
        for (int i0 = tid; i0 < n4; i0 += 8 * kProbsThreads) {      // sums of 32: no long chain of roundings
            float g = 0.0f;
#pragma unroll
            for (int k = 0; k < 8; k++) {
                const int i = i0 + k * kProbsThreads;
                if (i < n4) {
                    float4 y = x4[i];
                    y = make_float4(ex2f((y.x - M) * c), ex2f((y.y - M) * c), ex2f((y.z - M) * c), ex2f((y.w - M) * c));
                    x4[i] = y;
                    g += (y.x + y.y) + (y.z + y.w);
                }
            }
            z += g;
        }
        for (int i0 = kept + tid; i0 < n; i0 += 32 * kProbsThreads) {
            float g = 0.0f;
            for (int i = i0; i < n && i < i0 + 32 * kProbsThreads; i += kProbsThreads) g += ex2f((l[i] - M) * c);
            z += g;
        }
        z = warp_sum(z);
        if (lane == 0) s_z[warp] = z;
        __syncthreads();
        z = s_z[lane & (kProbsWarps - 1)];
#pragma unroll
        for (int o = kProbsWarps / 2; o > 0; o >>= 1) z += __shfl_xor_sync(kFull, z, o);
    }
    cl.barrier_wait(std::move(started));
    if (tid < nc) {                                        // to every CTA of the row
        *cl.map_shared_rank(&s_cm[rank], tid) = m;
        *cl.map_shared_rank(&s_cz[rank], tid) = z;
        *cl.map_shared_rank(&s_ci[rank], tid) = at;
    }
    cl.sync();
    if constexpr (GREEDY) {
        m = s_cm[0], at = s_ci[0];
        for (int k = 1; k < nc; k++) join_mi(m, at, s_cm[k], s_ci[k]);
        for (int i = tid; i < n; i += kProbsThreads) p[i] = lo + i == at ? 1.0f : 0.0f;
    } else {
        m = -INFINITY;
        for (int k = 0; k < nc; k++) m = fmaxf(m, s_cm[k]);
        const float top = m == -INFINITY ? 0.0f : m;
        z = 0.0f;
        for (int k = 0; k < nc; k++) {                     // a slice of -inf alone has no weight (0, or NaN)
            const float zk = s_cz[k];
            z += s_cm[k] == -INFINITY ? zk : zk * ex2f((s_cm[k] - top) * c);
        }
        const float inv = z == 0.0f ? 0.0f : __fdiv_rn(1.0f, z), f = s_cm[rank] == -INFINITY ? inv : ex2f((M - top) * c) * inv;
        if (((uintptr_t)p & 15) == 0) {
#pragma unroll 4
            for (int i = tid; i < kept >> 2; i += kProbsThreads) {
                const float4 y = x4[i];
                *reinterpret_cast<float4 *>(p + 4 * i) = make_float4(y.x * f, y.y * f, y.z * f, y.w * f);
            }
            if (tid < (kept & 3)) p[(kept & ~3) + tid] = x[(kept & ~3) + tid] * f;
        } else {
#pragma unroll 4
            for (int i = tid; i < kept; i += kProbsThreads) p[i] = x[i] * f;
        }
        for (int i = kept + tid; i < n; i += kProbsThreads) p[i] = ex2f((l[i] - top) * c) * inv;
    }
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

typedef unsigned long long u64;

// A probability as a whole number of 2^-40 (round half to even; NaN and negative: 0, above 1: 2^40). Whole
// numbers add up to the same sum in any order, so the drawn token does not depend on the split.
__device__ __forceinline__ u64 verify_weight(float r) {
    return r > 0.0f ? (u64)__float2ll_rn(fminf(r, 1.0f) * 1099511627776.0f) : 0ull;
}

__device__ __forceinline__ u64 warp_sum_u64(u64 v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(kFull, v, o);
    return v;
}
// Which lane's interval of the cumulative sums holds `want` (31 bits set where none), and `before` up to it.
__device__ __forceinline__ int warp_find_u64(u64 mine, u64 want, u64 &before) {
    u64 inc = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const u64 t = __shfl_up_sync(kFull, inc, o);
        if ((threadIdx.x & 31) >= o) inc += t;
    }
    const unsigned hit = __ballot_sync(kFull, before + inc > want);
    const int at = hit ? __ffs(hit) - 1 : -1;
    const u64 e = __shfl_sync(kFull, inc - mine, at < 0 ? 0 : at), all = __shfl_sync(kFull, inc, 31);
    before += at < 0 ? all : e;
    return at;
}

constexpr int kVerBatch = 8;          // loads in flight per lane: a batch is 256 values of a warp's segment

// What is left of p behind the rejected draft: p - q, p without token x, or p.
struct Remains {
    const float *p, *q;
    int x;
    __device__ __forceinline__ void load(int i0, int end, float (&r)[kVerBatch]) const {
        float w[kVerBatch];
#pragma unroll
        for (int k = 0; k < kVerBatch; k++) r[k] = i0 + 32 * k < end ? __ldcg(p + i0 + 32 * k) : 0.0f;
        if (q) {
#pragma unroll
            for (int k = 0; k < kVerBatch; k++) w[k] = i0 + 32 * k < end ? __ldcg(q + i0 + 32 * k) : 0.0f;
#pragma unroll
            for (int k = 0; k < kVerBatch; k++) r[k] = __fsub_rn(r[k], w[k]);
        } else if (x >= 0) {
#pragma unroll
            for (int k = 0; k < kVerBatch; k++)
                if (i0 + 32 * k == x) r[k] = 0.0f;
        }
    }
};

constexpr int kVerifyThreads = 256;

// One cluster per sequence: the drafts first (every CTA finds the same count), then the next token by
// inversion of the cumulative weights of the row. Every warp adds up its segment, 256 values at a time, and keeps
// those sums; the one warp whose segment holds the wanted weight finds the 256, then the 32, then the value.
// Bound by the latencies of that chain (drafts, their probabilities, the row, the exchange, the search) for one sequence
// (8.8 us), by memory for many: 64 sequences with the draft's probabilities, 78 MB in 16.8 us, 4.6 TB/s. 256 threads, so that
// many clusters are resident: with 1024, 16 sequences took 16.1 us against 10.0, 128 sequences 76 against 32.
__global__ void __launch_bounds__(kVerifyThreads, 4) k_verify(const VerifyArgs a) {
    constexpr int NT = kVerifyThreads, kWarps = NT / 32;
    extern __shared__ u64 s_sum[];                         // [kWarps][batches] sums of 256 values
    __shared__ u64 s_w[kWarps], s_c[2][kRowCtas];
    __shared__ int s_n;
    cg::cluster_group cl = cg::this_cluster();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, N = a.max_draft, V = a.V;
    const int rank = (int)cl.block_rank(), nc = (int)cl.num_blocks(), b = blockIdx.x / nc;
    auto started = cl.barrier_arrive();
    pdl_trigger();
    pdl_wait();
    const int nd = a.n_draft ? a.n_draft[b] : N;
    const int r0 = a.row_start ? a.row_start[b] : b * (N + 1);
    int *tok = a.tokens + (int64_t)b * (N + 1);
    const int *draft = a.draft + (int64_t)b * N;
    const float *u = a.u + (int64_t)b * (N + 1);
    if (nd < 0 || nd > N || r0 < 0 || r0 > a.p_rows - nd - 1) {         // the same for the whole cluster
        if (rank == 0) {
            if (tid == 0) {
                verify_err(a, QMS_PAGED_ELEN);
                a.n_accept[b] = 0;
            }
            for (int i = tid; i <= N; i += NT) tok[i] = -1;
        }
        cl.barrier_wait(std::move(started));
        return;
    }
    if (warp == 0) {
        int n = 0;
        for (int i0 = 0; i0 < nd; i0 += 32) {              // 32 drafts at a time, up to the first that falls
            const int i = i0 + lane;
            bool fell = false;
            if (i < nd) {
                const int x = draft[i];
                fell = x < 0 || x >= V;
                if (!fell) {
                    const float px = a.p[(int64_t)(r0 + i) * a.ldp + x];
                    const float qx = a.q ? a.q[((int64_t)b * N + i) * a.ldq + x] : 1.0f;
                    fell = !(__fmul_rn(u[i], qx) < px);
                }
            }
            const unsigned f = __ballot_sync(kFull, fell);
            n = min(nd, f ? i0 + __ffs(f) - 1 : i0 + 32);
            if (f) break;
        }
        if (lane == 0) s_n = n;
    }
    __syncthreads();
    const int n = s_n, x = n < nd ? draft[n] : -1;
    const bool known = x >= 0 && x < V;
    Remains rem;
    rem.p = a.p + (int64_t)(r0 + n) * a.ldp;
    rem.q = known && a.q ? a.q + ((int64_t)b * N + n) * a.ldq : nullptr;
    rem.x = known ? x : -1;
    const int seg = rank * kWarps + warp, segs = nc * kWarps, batches = (V / segs + 256) / 256;
    const int lo = (int)((int64_t)V * seg / segs), hi = (int)((int64_t)V * (seg + 1) / segs);
    const u64 m = (u64)floorf(fminf(fmaxf(u[N], 0.0f), 0.99999994f) * 16777216.0f);
    bool found = false;
    for (int pass = 0; pass < 2 && !found; pass++) {        // what p has over q; where that is nothing, p itself
        u64 w = 0;
        for (int k = 0; lo + 256 * k < hi; k++) {
            float r[kVerBatch];
            rem.load(lo + 256 * k + lane, hi, r);
            u64 t = 0;
#pragma unroll
            for (int j = 0; j < kVerBatch; j++) t += verify_weight(r[j]);
            t = warp_sum_u64(t);
            if (lane == 0) s_sum[warp * batches + k] = t;
            w += t;
        }
        __syncthreads();                                   // the last pass is done with s_w
        if (lane == 0) s_w[warp] = w;
        __syncthreads();
        u64 cta = 0, before = 0;
        for (int k = 0; k < kWarps; k++) {
            if (k < warp) before += s_w[k];
            cta += s_w[k];
        }
        if (pass == 0) cl.barrier_wait(std::move(started));
        if (tid < nc) *cl.map_shared_rank(&s_c[pass][rank], tid) = cta;
        cl.sync();
        u64 total = 0;
        for (int k = 0; k < nc; k++) {
            if (k < rank) before += s_c[pass][k];
            total += s_c[pass][k];
        }
        if (total == 0) {
            rem.q = nullptr;
            rem.x = -1;
            continue;
        }
        found = true;
        const u64 want = (total >> 24) * m + (((total & 0xFFFFFFull) * m) >> 24);        // floor(total * u)
        if (before > want || want >= before + w) continue;                             // in another warp's segment
        int at = -1, k0 = 0;
        for (; at < 0 && k0 < batches; k0 += 32)
            at = warp_find_u64(k0 + lane < batches && lo + 256 * (k0 + lane) < hi ? s_sum[warp * batches + k0 + lane] : 0, want, before);
        if (at < 0) continue;                              // not reached: the segment holds it
        const int i0 = lo + 256 * (k0 - 32 + at);
        float r[kVerBatch];
        u64 t[kVerBatch];
        rem.load(i0 + lane, hi, r);                        // the batch once more, from L2
#pragma unroll
        for (int j = 0; j < kVerBatch; j++) t[j] = warp_sum_u64(verify_weight(r[j]));
        bool done = false;
#pragma unroll
        for (int j = 0; j < kVerBatch; j++) {
            if (done) continue;
            if (before + t[j] <= want) {
                before += t[j];
                continue;
            }
            done = true;
            const int e = warp_find_u64(verify_weight(r[j]), want, before);
            if (lane == 0) tok[n] = i0 + 32 * j + e;
        }
    }
    if (rank == 0) {
        if (tid == 0) {
            a.n_accept[b] = n;
            if (!found) {
                verify_err(a, QMS_PAGED_EMASS);
                tok[n] = -1;
            }
            if (n < nd && !known) verify_err(a, QMS_PAGED_ETOKEN);
        }
        for (int i = tid; i <= N; i += NT)
            if (i != n) tok[i] = i < n ? draft[i] : -1;
    }
}

static int launch_probs(const float *l, int64_t ldl, int rows, int V, float temp, float *p, int64_t ldp, cudaStream_t s) {
    static std::atomic<unsigned long long> done[2];
    int rc = allow_smem(done[0], k_probs<true>, kProbsKeep * 4);
    if (rc || (rc = allow_smem(done[1], k_probs<false>, kProbsKeep * 4))) return rc;
    const int nc = row_ctas(rows, V, 74), slice = ((V + 3) / 4 / nc + 1) * 4;
    const size_t smem = (size_t)(slice < kProbsKeep ? slice : kProbsKeep) * 4;
    if (!(temp > 0.0f)) return launch_rows(k_probs<true>, kProbsThreads, rows, nc, smem, s, l, ldl, V, 0.0f, p, ldp);
    // a scale of 0 or infinity would make NaN of the logits -inf and of the maximum
    const float c = fminf(fmaxf(1.4426950408889634f / temp, 1e-37f), 1e37f);
    return launch_rows(k_probs<false>, kProbsThreads, rows, nc, smem, s, l, ldl, V, c, p, ldp);
}

static int launch_verify(const VerifyArgs &a, cudaStream_t s) {
    const int nc = row_ctas(a.n_seq, a.V, 148), warps = kVerifyThreads / 32;
    const size_t smem = (size_t)warps * ((a.V / (nc * warps) + 256) / 256) * 8;
    return launch_rows(k_verify, kVerifyThreads, a.n_seq, nc, smem, s, a);
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
    return launch_probs(logits, ldl, rows, vocab, temp, p, ldp, (cudaStream_t)stream);
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
    return launch_verify(a, (cudaStream_t)stream);
}

}  // extern "C"
