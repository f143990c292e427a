// qms_logprobs.cu - log probabilities of given tokens, the entropy and the likeliest tokens of rows of logits on B200
// (sm_100a). The reference prints the ten likeliest tokens of a row it holds on the host (src/main.c, --top); it has no entropy.
#include <cooperative_groups.h>
#include <float.h>
#include <math.h>

#include "qms_rows.cuh"

namespace cg = cooperative_groups;

namespace qms {

typedef unsigned long long u64;

constexpr int kLpThreads = 512, kLpWarps = kLpThreads / 32, kLpTop = 32, kLpList = 2048;

struct LogprobArgs {
    const float *l;
    int64_t ldl;
    int V, n_ids, n_top;
    const int *ids;
    float c, temp;                   // log2(e) / temp
    float *lp, *entropy, *top_lp;
    int *top_id, *err;
};

// A value and its index as one number that grows with the value and, among equals, falls with the index. Never 0 for a value that
// is not NaN.
__device__ __forceinline__ u64 lp_key(float x, int i) {
    const uint32_t b = __float_as_uint(x + 0.0f);                   // (-0 counts as 0)
    return (u64)(b ^ ((uint32_t)((int)b >> 31) | 0x80000000u)) << 32 | (uint32_t)~i;
}
__device__ __forceinline__ float lp_value(u64 key) {
    const uint32_t b = (uint32_t)(key >> 32);
    return __uint_as_float(b & 0x80000000u ? b ^ 0x80000000u : ~b);
}

// What one CTA knows of its slice: the maximum m; z, t: sums of w and w log2(w), w = 2^((l - m) c), without one value that is m.
struct LpPart {
    float m, z, t;
};

// With x = (l - max) / temp: log p = x - log Z and the entropy log Z - sum p x, where Z = 1 + z and z leaves out one value that is the
// maximum: of a sure row z is what matters, and 1 + z would round it away. Grid: rows x cluster, a slice per CTA, kept in shared memory
// as in k_probs. First pass over a slice: every lane's maximum. From these a bound that at least n_top values of the slice
// reach: the least over the warps of each warp's r-th largest lane maximum, r n_top over the number of warps. Second
// pass: z and t, and the values at or above the bound go to a list, some 50 of 19,000; a value's rank is the number of list entries
// above it. A list that overflows (thousands of equal values) is not used: n_top rounds of the largest below the last one.
// The cluster's first CTA joins the parts and the lists.
__global__ void __launch_bounds__(kLpThreads, 2) k_logprobs(const LogprobArgs a) {
    extern __shared__ __align__(16) float x[];
    __shared__ u64 s_list[kLpList], s_all[kRowCtas * kLpTop], s_key[kLpWarps];
    __shared__ float s_m[kLpWarps], s_r[kLpWarps], s_z[kLpWarps], s_t[kLpWarps];
    __shared__ LpPart s_part[kRowCtas];
    __shared__ int s_n, s_most;
    cg::cluster_group cl = cg::this_cluster();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, rank = (int)cl.block_rank(), nc = (int)cl.num_blocks();
    if (tid < nc * kLpTop) s_all[tid] = 0;
    if (tid == 0) s_n = s_most = 0;
    auto started = cl.barrier_arrive();                    // waited for before the first write to another CTA
    pdl_trigger();
    pdl_wait();
    const int64_t r = blockIdx.x / nc;
    const int groups = (a.V + 3) >> 2;                     // slices start at multiples of 4 values
    const int lo = (int)((int64_t)groups * rank / nc) * 4, n = min(a.V, (int)((int64_t)groups * (rank + 1) / nc) * 4) - lo;
    const float *row = a.l + r * a.ldl, *l = row + lo;
    const int kept = min(n, kProbsKeep), n4 = (kept + 3) >> 2;
    const float4 *x4 = reinterpret_cast<const float4 *>(x);
    if (((uintptr_t)l & 15) == 0) {
        for (int i = tid; i < kept >> 2; i += kLpThreads) cp_async16(x + 4 * i, l + 4 * i);
        if (tid < (kept & 3)) cp_async4(x + (kept & ~3) + tid, l + (kept & ~3) + tid);
    } else {
#pragma unroll 4
        for (int i = tid; i < kept; i += kLpThreads) cp_async4(x + i, l + i);
    }
    if (tid >= kept && tid < 4 * n4) x[tid] = -INFINITY;   // (a slice below one group)
    for (int i = max(kept, kLpThreads) + tid; i < 4 * n4; i += kLpThreads) x[i] = -INFINITY;
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncthreads();

    // ---- first pass: maxima
    float m = -INFINITY;
#pragma unroll 4
    for (int i = tid; i < n4; i += kLpThreads) {
        const float4 y = x4[i];
        m = fmaxf(m, fmaxf(fmaxf(y.x, y.y), fmaxf(y.z, y.w)));
    }
    for (int i = kept + tid; i < n; i += kLpThreads) m = fmaxf(m, l[i]);
    const int busy = min(kLpWarps, (n4 + 31) >> 5);        // warps with values
    const int rounds = (a.n_top + max(busy, 1) - 1) / max(busy, 1);
    {
        uint32_t k = __float_as_uint(m + 0.0f);
        k ^= (uint32_t)((int)k >> 31) | 0x80000000u;
        uint32_t best = __reduce_max_sync(kFull, k), top = best;
        for (int i = 1; i < rounds; i++) {                 // the next largest lane
            const unsigned hit = __ballot_sync(kFull, k == best);
            if (lane == __ffs(hit) - 1) k = 0;
            best = __reduce_max_sync(kFull, k);
        }
        if (lane == 0) {
            s_m[warp] = lp_value((u64)top << 32);
            s_r[warp] = best == 0 ? -INFINITY : lp_value((u64)best << 32);
        }
    }
    __syncthreads();
    m = s_m[lane & (kLpWarps - 1)];
    float bound = (lane & (kLpWarps - 1)) < busy ? s_r[lane & (kLpWarps - 1)] : INFINITY;
#pragma unroll
    for (int o = kLpWarps / 2; o > 0; o >>= 1) {
        m = fmaxf(m, __shfl_xor_sync(kFull, m, o));
        bound = fminf(bound, __shfl_xor_sync(kFull, bound, o));
    }
    bound = a.n_top == 0 ? m : fmaxf(fminf(bound, m), -FLT_MAX);
    const float M = m == -INFINITY ? 0.0f : m;

    // ---- second pass: sums, and the list
    float z = 0.0f, t = 0.0f;
    auto add = [&](float v, float &gz, float &gt) {
        const float y = (v - M) * a.c, w = ex2f(y);
        gz += w;
        gt = fmaf(w, fmaxf(y, -256.0f), gt);               // (weights below 2^-126 are 0; 0 * inf is not)
    };
    // a value at the bound or above: listed; the maxima are counted and left out of the sums
    auto look = [&](float v, int i) {
        if (v >= bound && v > -INFINITY) {
            if (a.n_top > 0) {
                const int k = atomicAdd(&s_n, 1);
                if (k < kLpList) s_list[k] = lp_key(v, lo + i);
            }
            if (v == m) {
                atomicAdd(&s_most, 1);
                return -INFINITY;
            }
        }
        return v;
    };
    for (int i0 = tid; i0 < n4; i0 += 8 * kLpThreads) {    // sums of 32: no long chain of roundings
        float gz = 0.0f, gt = 0.0f;
#pragma unroll
        for (int k = 0; k < 8; k++) {
            const int i = i0 + k * kLpThreads;
            if (i < n4) {
                float4 y = x4[i];
                if (fmaxf(fmaxf(y.x, y.y), fmaxf(y.z, y.w)) >= bound)
                    y = make_float4(look(y.x, 4 * i), look(y.y, 4 * i + 1), look(y.z, 4 * i + 2), look(y.w, 4 * i + 3));
                add(y.x, gz, gt), add(y.y, gz, gt), add(y.z, gz, gt), add(y.w, gz, gt);
            }
        }
        z += gz;
        t += gt;
    }
    for (int i0 = kept + tid; i0 < n; i0 += 32 * kLpThreads) {
        float gz = 0.0f, gt = 0.0f;
        for (int i = i0; i < n && i < i0 + 32 * kLpThreads; i += kLpThreads) add(look(l[i], i), gz, gt);
        z += gz;
        t += gt;
    }
    z = warp_sum(z);
    t = warp_sum(t);
    if (lane == 0) s_z[warp] = z, s_t[warp] = t;
    __syncthreads();
    const int listed = s_n;
    u64 *all = cl.map_shared_rank(s_all, 0) + rank * kLpTop;
    if (tid < 32) {
        z = lane < kLpWarps ? s_z[lane] : 0.0f;
        t = lane < kLpWarps ? s_t[lane] : 0.0f;
        z = warp_sum(z) + (float)max(s_most - 1, 0);
        t = warp_sum(t);
    }
    cl.barrier_wait(std::move(started));
    if (tid == 0) {
        if (m == INFINITY) z = NAN;
        *cl.map_shared_rank(&s_part[rank], 0) = LpPart{m, z, t};
    }
    if (listed <= kLpList) {
        for (int i = tid; i < listed; i += kLpThreads) {
            const u64 k = s_list[i];
            int above = 0;
            for (int j = 0; j < listed; j++) above += s_list[j] > k;
            if (above < a.n_top) all[above] = k;
        }
    } else {
        u64 last = ~0ull;
        for (int q = 0; q < a.n_top; q++) {
            u64 best = 0;
            auto offer = [&](float v, int i) {
                if (v >= bound) {                          // (NaN is not)
                    const u64 k = lp_key(v, lo + i);
                    if (k < last && k > best) best = k;
                }
            };
            for (int i = tid; i < kept; i += kLpThreads) offer(x[i], i);
            for (int i = kept + tid; i < n; i += kLpThreads) offer(l[i], i);
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) {
                const u64 other = __shfl_xor_sync(kFull, best, o);
                best = other > best ? other : best;
            }
            if (lane == 0) s_key[warp] = best;
            __syncthreads();
            for (int w = 0; w < kLpWarps; w++) best = s_key[w] > best ? s_key[w] : best;
            __syncthreads();
            if (tid == 0) all[q] = best;
            last = best;
        }
    }
    cl.sync();
    if (rank != 0) return;

    // ---- the row: parts and lists joined
    m = -INFINITY;
    int first = 0;
    for (int k = nc - 1; k >= 0; k--)
        if (s_part[k].m >= m) m = s_part[k].m, first = k;
    z = t = 0.0f;
    for (int k = 0; k < nc; k++) {
        const LpPart p = s_part[k];
        if (k == first || p.m == -INFINITY) {              // (of a slice of -inf alone z is 0, or NaN)
            z += p.z;
            t += p.t;
        } else {
            const float d = (p.m - m) * a.c, f = ex2f(d), one = p.z + 1.0f;
            z = fmaf(one, f, z);
            t = fmaf(f, fmaf(one, fmaxf(d, -256.0f), p.t), t);
        }
    }
    const bool none = m == -INFINITY && !isnan(z);         // a row of -inf
    const float lz = log1pf(z);
    auto logp = [&](float v) { return none || v == -INFINITY ? (isnan(z) ? NAN : -INFINITY) : __fdiv_rn(v - m, a.temp) - lz; };
    for (int i = tid; i < a.n_ids; i += kLpThreads) {
        const int id = a.ids[r * a.n_ids + i];
        const bool good = (unsigned)id < (unsigned)a.V;
        if (!good && a.err) atomicOr(a.err, QMS_PAGED_ETOKEN);
        a.lp[r * a.n_ids + i] = good ? logp(__ldcg(row + id)) : NAN;
    }
    if (tid == 0 && a.entropy) a.entropy[r] = none ? 0.0f : lz - 0.69314718056f * t / (1.0f + z);
    if (a.n_top == 0) return;
    const u64 k = tid < nc * kLpTop ? s_all[tid] : 0;
    const int found = __syncthreads_count(k != 0);
    if (k != 0) {
        int above = 0;
        for (int i = 0; i < nc; i++)
            for (int j = 0; j < a.n_top; j++) above += s_all[i * kLpTop + j] > k;
        if (above < a.n_top) {
            a.top_id[r * a.n_top + above] = (int)~(uint32_t)k;
            a.top_lp[r * a.n_top + above] = logp(lp_value(k));
        }
    }
    if (tid >= found && tid < a.n_top) {
        a.top_id[r * a.n_top + tid] = -1;
        a.top_lp[r * a.n_top + tid] = isnan(z) ? NAN : -INFINITY;
    }
}

static int launch_logprobs(const LogprobArgs &a, int rows, cudaStream_t s) {
    static std::atomic<unsigned long long> done{0};
    const int rc = allow_smem(done, k_logprobs, kProbsKeep * 4);
    if (rc) return rc;
    const int nc = row_ctas(rows, a.V, 74), slice = ((a.V + 3) / 4 / nc + 1) * 4;
    const size_t smem = (size_t)(slice < kProbsKeep ? slice : kProbsKeep) * 4;
    return launch_rows(k_logprobs, kLpThreads, rows, nc, smem, s, a);
}

}  // namespace qms

using namespace qms;

extern "C" {

int qms_cuda_logprobs(const float *logits, int64_t ldl, int rows, int vocab, float temp, const int *ids, int n_ids, float *logp,
                      float *entropy, int n_top, int *top_id, float *top_logp, int *err, void *stream) {
    clear_error();
    QMS_REQUIRE(logits && vocab > 0 && vocab <= (1 << 22) && rows >= 0, QMS_CUDA_EINVAL,
                "logprobs: NULL logits, rows %d or vocab %d (at most %d)", rows, vocab, 1 << 22);
    QMS_REQUIRE(ldl >= vocab, QMS_CUDA_EINVAL, "logprobs: rows of %d need ldl of at least that", vocab);
    QMS_REQUIRE(temp > 0.0f && temp <= FLT_MAX, QMS_CUDA_EINVAL, "logprobs: temp must be positive and finite");
    QMS_REQUIRE(n_ids >= 0 && (n_ids == 0 || (ids && logp)), QMS_CUDA_EINVAL, "logprobs: %d ids per row need ids and logp", n_ids);
    QMS_REQUIRE(n_top >= 0 && n_top <= kLpTop && (n_top == 0 || (top_id && top_logp)), n_top > kLpTop ? QMS_CUDA_EUNSUPPORTED : QMS_CUDA_EINVAL,
                "logprobs: %d likeliest tokens (at most %d) need top_id and top_logp", n_top, kLpTop);
    QMS_REQUIRE((((uintptr_t)logits | (uintptr_t)ids | (uintptr_t)logp | (uintptr_t)entropy | (uintptr_t)top_id | (uintptr_t)top_logp |
                  (uintptr_t)err) & 3) == 0, QMS_CUDA_EINVAL, "logprobs: misaligned pointer");
    if (rows == 0) return QMS_CUDA_OK;
    LogprobArgs a;
    memset(&a, 0, sizeof a);
    a.l = logits;
    a.ldl = ldl;
    a.V = vocab;
    a.n_ids = n_ids;
    a.n_top = n_top;
    a.ids = ids;
    // a scale of 0 or infinity would make NaN of the maximum and of -inf
    a.c = fminf(fmaxf(1.4426950408889634f / temp, 1e-37f), 1e37f);
    a.temp = temp;
    a.lp = logp;
    a.entropy = entropy;
    a.top_lp = top_logp;
    a.top_id = top_id;
    a.err = err;
    return launch_logprobs(a, rows, (cudaStream_t)stream);
}

}  // extern "C"
