// qms_logprobs.cu - log probabilities of given tokens, the entropy and the likeliest tokens of rows of logits on B200
// (sm_100a). The reference prints the ten likeliest tokens of a row it holds on the host (src/main.c, --top); it has no entropy.
#include <cooperative_groups.h>
#include <float.h>
#include <math.h>

#include "qms_rows.cuh"

namespace cg = cooperative_groups;

namespace qms {

typedef unsigned long long u64;

constexpr int kLpThreads = 256, kLpWarps = kLpThreads / 32, kLpTop = 32;
// a warp's groups of 4 values per lane, values per chunk, chunks in flight, or kept; entries of the list, what is short for one
constexpr int kLpQuads = 4, kLpChunk = 128 * kLpQuads, kLpRing = 2, kLpKeep = 6, kLpShort = 256, kLpList = 512;
constexpr uint32_t kLpSpin = 1u << 22;
constexpr int kLpFew = 74;            // CTAs up to which a row's slices are kept in shared memory (launch_logprobs)

struct LogprobArgs {
    const float *l;
    int64_t ldl;
    int V, n_ids, n_top;
    const int *ids;
    float h, c, temp;                // (l h - max h) c is (l - max) log2(e) / temp; temp: h times the temperature
    float *lp, *entropy, *top_lp;
    int *top_id, *err;
};

// A value and its index as one number that grows with the value and, among equals, falls with the index. Never 0 for a value that
// is not NaN.
__device__ __forceinline__ uint32_t lp_order(float x) {
    const uint32_t b = __float_as_uint(x + 0.0f);                   // (-0 counts as 0)
    return b ^ ((uint32_t)((int)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ u64 lp_key(float x, int i) { return (u64)lp_order(x) << 32 | (uint32_t)~i; }
__device__ __forceinline__ float lp_unorder(uint32_t b) { return __uint_as_float(b & 0x80000000u ? b ^ 0x80000000u : ~b); }
__device__ __forceinline__ float lp_value(u64 key) { return lp_unorder((uint32_t)(key >> 32)); }
__device__ __forceinline__ float min_nan(float a, float b) {
    float d;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
    return d;
}

// Two fp32 at once.
__device__ __forceinline__ u64 two(float a, float b) {
    u64 d;
    asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(a), "f"(b));
    return d;
}
__device__ __forceinline__ float2 of_two(u64 x) {
    float2 d;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(d.x), "=f"(d.y) : "l"(x));
    return d;
}
__device__ __forceinline__ u64 add_two(u64 a, u64 b) {
    u64 d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ u64 mul_two(u64 a, u64 b) {
    u64 d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ u64 fma_two(u64 a, u64 b, u64 c) {
    u64 d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}

__device__ __forceinline__ u64 max_key(u64 key) {                   // of a warp's lanes
    const uint32_t hi = __reduce_max_sync(kFull, (uint32_t)(key >> 32));
    return (u64)hi << 32 | __reduce_max_sync(kFull, (uint32_t)(key >> 32) == hi ? (uint32_t)key : 0u);
}

// How many entries of `lists` lists, each of kLpTop in falling order, are above the key.
__device__ __forceinline__ int lp_above(const u64 *list, int lists, u64 key) {
    static_assert(kLpTop == 32, "5 steps to one of 32, a sixth for none or all");
    int at[kRowCtas] = {};
#pragma unroll
    for (int step = 16; step > 0; step >>= 1)
#pragma unroll
        for (int w = 0; w < kRowCtas; w++)
            if (w < lists && list[w * kLpTop + at[w] + step - 1] > key) at[w] += step;
    int above = 0;
#pragma unroll
    for (int w = 0; w < kRowCtas; w++)
        if (w < lists) above += at[w] + (at[w] == 31 && list[w * kLpTop + 31] > key);
    return above;
}

// What is known of some values: the maximum m; z, t: sums of w and w log2(w), w = 2^((l - m) c), without one value that is m.
struct LpPart {
    float m, z, t;
};
// p under the maximum M of several parts; `first`: it is the one whose m is left out. Nothing seen: z is 0, or NaN.
__device__ __forceinline__ LpPart lp_under(const LpPart &p, float M, bool first, float h, float c) {
    if (first) return p;
    const float d = p.m == -INFINITY ? -INFINITY : (p.m * h - M * h) * c, f = ex2f(d), one = p.z + 1.0f;
    return LpPart{M, one * f, f * fmaf(one, fmaxf(d, -256.0f), p.t)};
}

// With x = (l - max) / temp: log p = x - log Z and the entropy log Z - sum p x, where Z = 1 + z and z leaves out one value that is the
// maximum: of a sure row z is what matters, and 1 + z would round it away. One pass, and no warp waits for another before its end: a row
// is cut over a cluster, the warps of a CTA take its chunks in turn, each into its part of shared memory by bulk copies. A lane keeps two
// running maxima apart from its sums (what is no longer the largest is added), under a base that follows them at a distance of 2^4 at
// most, and adds two values by one instruction (512 rows 84 us, one by one 88).
// The likeliest: lane i holds the i-th largest of its warp's so far. Values that reach a bound are put in their place: first one that n_top
// lanes' largest of the first chunk reach, then the n_top-th itself, of this warp or of another that is further. Some 40 of 19,000 values
// reach it, in 14 chunks of 37; those of a chunk are put in together. The first CTA of the cluster joins all.
// KEEP: for few rows, where that chain of steps is what the row takes: all of a slice stays in shared memory, the bound comes from all lanes'
// largest (the least over the warps of each one's r-th, r = n_top over the number of warps), and a second look lists what reaches it, some
// 60 of 19,000, whose places are the numbers of entries above them.
// Bound by instructions for many rows, some 17 per value and lane (0.7 per cycle and scheduler), a third more with ten alternatives: 512 rows of 151,936 84 us,
// 3.7 TB/s, without alternatives 57, 5.5 TB/s, 0.83 of a plain copy. One row by the chain of its steps: 10.2 us, without alternatives 5.2.
template <bool KEEP>
__global__ void __launch_bounds__(kLpThreads, KEEP ? 2 : 4) k_logprobs(const LogprobArgs a) {
    constexpr int RING = KEEP ? kLpKeep : kLpRing;
    extern __shared__ __align__(128) float rings[];        // [kLpWarps][RING][kLpChunk], then (KEEP) the list
    __shared__ u64 s_all[kRowCtas * kLpTop], s_list[kLpWarps * kLpTop], s_some[kLpWarps][48];
    __shared__ uint64_t s_full[kLpWarps][RING];
    __shared__ LpPart s_warp[kLpWarps], s_part[kRowCtas];
    __shared__ uint32_t s_bound, s_r[kLpWarps];            // the highest bound of a warp, by lp_order
    __shared__ u64 s_lowest;
    __shared__ int s_abort, s_n;
    cg::cluster_group cl = cg::this_cluster();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, rank = (int)cl.block_rank(), nc = (int)cl.num_blocks();
    float *ring = rings + warp * RING * kLpChunk;
    for (int i = tid; i < nc * kLpTop; i += kLpThreads) s_all[i] = 0;
    if (tid == 0) s_abort = 0, s_bound = 0;
    if (lane == 0) {
        for (int i = 0; i < RING; i++) mbar_init(&s_full[warp][i], 1);
        fence_mbar_init();
    }
    auto started = cl.barrier_arrive();                    // waited for before the first write to another CTA
    pdl_wait();
    pdl_trigger();
    // the row: up to 3 values before a 16-byte boundary, groups of 4 that are cut over all warps, up to 3 behind them
    const int64_t r = blockIdx.x / nc;
    const float *row = a.l + r * a.ldl;
    const int head = min(a.V, (int)(-((uintptr_t)row >> 2) & 3)), groups = (a.V - head) >> 2, tail = head + 4 * groups;
    const int lo = head + (int)((int64_t)groups * rank / nc) * 4, hi = head + (int)((int64_t)groups * (rank + 1) / nc) * 4;
    const int chunks = ((hi - lo + kLpChunk - 1) / kLpChunk - warp + kLpWarps - 1) / kLpWarps;     // in turn over the warps
    auto load = [&](int k) {                               // by one lane
        const int base = lo + (k * kLpWarps + warp) * kLpChunk, n = min(kLpChunk, hi - base);
        mbar_arrive_expect_tx(&s_full[warp][k % RING], n * 4);
        bulk_load(smem_u32(ring + k % RING * kLpChunk), row + base, n * 4, &s_full[warp][k % RING]);
    };
    if (lane == 0)
        for (int k = 0; k < min(chunks, RING); k++) load(k);
    const float mine = tid < a.n_ids && rank == 0 && (unsigned)a.ids[r * a.n_ids + tid] < (unsigned)a.V ? row[a.ids[r * a.n_ids + tid]] : 0.0f;
    __syncthreads();                                       // s_bound, s_abort

    float B = -FLT_MAX, m[2] = {-INFINITY, -INFINITY};
    u64 z2 = 0, t2 = 0;                                     // (two sums each)
    const u64 h2 = two(a.h, a.h), c2 = two(a.c, a.c);
    float bound = -FLT_MAX;                                // a value has to reach it
    u64 best = 0;                                          // the lane-th largest of the warp's
    // new values, up to 32 in s_new, take their places among the n_top largest: a key's place is the number of keys above it
    u64 *s_new = s_some[warp], *s_mine = s_list + warp * kLpTop;
    auto merge = [&](int n) {
        __syncwarp();
        const u64 key = lane < n ? s_new[lane] : 0;
        int at = 0, down = lane;
        for (int i = 0; i < n; i++) {
            const u64 k = s_new[i];
            at += k > key;
            down += k > best;
        }
        for (int i = 0; i < a.n_top; i++) at += __shfl_sync(kFull, best, i) > key;
        s_mine[lane] = 0;
        __syncwarp();
        if (best != 0 && down < a.n_top) s_mine[down] = best;
        if (key != 0 && at < a.n_top) s_mine[at] = key;
        __syncwarp();
        best = s_mine[lane];
    };
    int news = 0;
    auto look = [&](float v, int i) {                      // v: a value of each lane
        const unsigned hit = __ballot_sync(kFull, v >= bound);
        if (hit == 0) return;
        if (v >= bound) s_new[news + __popc(hit & ((1u << lane) - 1u))] = lp_key(v, i);
        news += __popc(hit);
        if (news > 16) {
            merge(min(news, 32));
            news = max(news - 32, 0);
            const u64 rest = lane < news ? s_new[32 + lane] : 0;
            __syncwarp();
            if (lane < news) s_new[lane] = rest;
        }
    };
    // between chunks: what comes later has a higher index, and has to be more than the n_top-th
    auto raise = [&]() {
        if (news > 4) {
            merge(news);
        } else {                                           // (one costs a third of a merge)
            __syncwarp();
            for (int i = 0; i < news; i++) {
                const u64 key = s_new[i], up = __shfl_up_sync(kFull, best, 1);
                const int at = __popc(__ballot_sync(kFull, best > key));
                if (lane > at) best = up;
                if (lane == at) best = key;
                if (lane >= a.n_top) best = 0;
            }
            __syncwarp();
        }
        news = 0;
        const uint32_t own = __shfl_sync(kFull, (uint32_t)(best >> 32), a.n_top - 1);     // (0: there are not so many yet)
        if (own == 0) return;
        if (lane == 0) atomicMax(&s_bound, own);
        bound = fmaxf(bound, lp_unorder(own + 1));           // (the next number above; of the largest finite one inf)
    };
    auto rebase = [&](float top) {                         // (B is h times a value)
        top *= a.h;
        if ((top - B) * a.c > 4.0f) {
            const float d = fmaxf((B - top) * a.c, -256.0f), f = ex2f(d);
            B = top;
            t2 = mul_two(two(f, f), fma_two(z2, two(d, d), t2));
            z2 = mul_two(z2, two(f, f));
        }
    };
    auto add = [&](float v0, float v1) {                   // to the sums: each value, or the largest so far that it replaces
        const float2 y = of_two(mul_two(fma_two(two(min_nan(m[0], v0), min_nan(m[1], v1)), h2, two(-B, -B)), c2));
        const u64 w = two(ex2f(y.x), ex2f(y.y));
        m[0] = fmaxf(m[0], v0), m[1] = fmaxf(m[1], v1);
        z2 = add_two(z2, w);
        t2 = fma_two(w, two(fmaxf(y.x, -256.0f), fmaxf(y.y, -256.0f)), t2);          // (weights below 2^-126 are 0; 0 * inf is not)
    };
    if (rank == 0 && warp == 0) {                                      // the values before the first boundary
        const float v = lane < head ? row[lane] : -INFINITY;
        rebase(v);
        if (!KEEP && a.n_top > 0) {
            look(v, lane);
            raise();
        }
        add(v, -INFINITY);
    }
    bool gave_up = false;
    for (int k = 0, slot = 0, phase = 0; k < chunks; k++) {
        for (uint32_t n = 0; !gave_up && !mbar_try_wait(&s_full[warp][slot], phase); n++) {
            gave_up = n == kLpSpin;
            if (n > 64) __nanosleep(32);
        }
        if ((gave_up = __any_sync(kFull, gave_up))) {      // the copies have 0.1 s to land before this CTA's memory goes
            for (int n = 0; n < 1 << 20; n++) __nanosleep(100);
            if (lane == 0) s_abort = 1;
            break;
        }
        const int base = lo + (k * kLpWarps + warp) * kLpChunk, n4 = min(kLpChunk, hi - base) >> 2;
        const float4 *x4 = reinterpret_cast<const float4 *>(ring + slot * kLpChunk);
        float4 y[kLpQuads];
        float top[kLpQuads];
#pragma unroll
        for (int e = 0; e < kLpQuads; e++) {
            const int i = lane + e * 32;
            y[e] = i < n4 ? x4[i] : make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
            top[e] = fmaxf(fmaxf(y[e].x, y[e].y), fmaxf(y[e].z, y[e].w));
        }
        static_assert(kLpQuads == 4, "the largest of 4 groups");
        const float most = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
        rebase(most);
#pragma unroll
        for (int e = 0; e < kLpQuads; e++) add(y[e].x, y[e].y), add(y[e].z, y[e].w);
        if (!KEEP && a.n_top > 0) {
            if (k == 0) {                                  // the n_top-th of the lanes' largest (NaN is none)
                uint32_t o = lp_order(fmaxf(most, -INFINITY)), at = __reduce_max_sync(kFull, o);
                for (int i = 1; i < a.n_top; i++) {
                    if (lane == __ffs(__ballot_sync(kFull, o == at)) - 1) o = 0;
                    at = __reduce_max_sync(kFull, o);
                }
                bound = fmaxf(bound, at == 0 ? -FLT_MAX : lp_unorder(at));
            }
            const uint32_t others = *(volatile uint32_t *)&s_bound;      // what another warp has found
            if (others != 0) bound = fmaxf(bound, lp_unorder(others));
            if (__any_sync(kFull, most >= bound)) {
#pragma unroll
                for (int e = 0; e < kLpQuads; e++) {
                    if (!__any_sync(kFull, top[e] >= bound)) continue;
                    const int i = base + 4 * (lane + e * 32);
                    look(y[e].x, i), look(y[e].y, i + 1), look(y[e].z, i + 2), look(y[e].w, i + 3);
                }
                raise();
            }
        }
        __syncwarp();
        if (!KEEP && lane == 0 && k + RING < chunks) {
            fence_async_smem();
            load(k + RING);
        }
        if (++slot == RING) slot = 0, phase ^= 1;
    }
    if (rank == nc - 1 && warp == kLpWarps - 1) {                             // the values behind the last group
        const float v = tail + lane < a.V ? row[tail + lane] : -INFINITY;
        rebase(v);
        if (!KEEP && a.n_top > 0) {
            look(v, tail + lane);
            raise();
        }
        add(v, -INFINITY);
    }

    // ---- lanes to warps, warps to the CTA
    LpPart p;
    {
        const float2 z = of_two(z2), t = of_two(t2);
        const bool second = m[1] > m[0];                   // of the two maxima one joins the sums
        const float y = ((second ? m[0] : m[1]) * a.h - B) * a.c, w = ex2f(y);
        p.m = second ? m[1] : m[0];
        p.z = z.x + z.y + w;
        p.t = fmaf(w, fmaxf(y, -256.0f), t.x + t.y);
        const float d = p.m == -INFINITY ? 0.0f : (B - p.m * a.h) * a.c, f = ex2f(d);            // from the base to the maximum
        p.t = f * fmaf(p.z, d, p.t);
        p.z *= f;
    }
    auto join = [&](LpPart p) {                            // of a warp's lanes
        const uint32_t k = lp_order(p.m), most = __reduce_max_sync(kFull, k);
        const int first = __ffs(__ballot_sync(kFull, k == most)) - 1;
        p = lp_under(p, lp_unorder(most), lane == first, a.h, a.c);
        p.z = warp_sum(p.z);
        p.t = warp_sum(p.t);
        p.m = lp_unorder(most);
        return p;
    };
    p = join(p);
    if (lane == 0) s_warp[warp] = p;
    s_list[tid] = best;
    u64 *list = reinterpret_cast<u64 *>(rings + kLpWarps * RING * kLpChunk);
    int listed = 0;
    if constexpr (KEEP) {
        if (a.n_top > 0) {
            // warps without a value do not count
            const int busy = max(1, min(kLpWarps, (hi - lo + kLpChunk - 1) / kLpChunk)), rounds = (a.n_top + busy - 1) / busy;
            uint32_t o = lp_order(fmaxf(m[0], m[1])), at = __reduce_max_sync(kFull, o);
            for (int i = 1; i < rounds; i++) {
                if (lane == __ffs(__ballot_sync(kFull, o == at)) - 1) o = 0;
                at = __reduce_max_sync(kFull, o);
            }
            if (lane == 0) s_r[warp] = at;
            if (tid == 0) s_n = 0;
            __syncthreads();
            uint32_t least = s_r[0];
            for (int w = 1; w < busy; w++) least = min(least, s_r[w]);
            bound = fmaxf(least == 0 ? -FLT_MAX : lp_unorder(least), -FLT_MAX);
            u64 lowest = 0;                                // a key has to reach it
            auto take = [&](float v, int i) {
                if (v >= bound && lp_key(v, i) >= lowest) {
                    const int n = atomicAdd(&s_n, 1);
                    if (n < kLpList) list[n] = lp_key(v, i);
                }
            };
            auto all_values = [&](auto &&f) {              // of this thread
                for (int k = 0; k < chunks; k++) {
                    const int base = lo + (k * kLpWarps + warp) * kLpChunk, n4 = min(kLpChunk, hi - base) >> 2;
                    const float4 *x4 = reinterpret_cast<const float4 *>(ring + k * kLpChunk);
#pragma unroll
                    for (int e = 0; e < kLpQuads; e++) {
                        const int i = lane + e * 32;
                        if (i >= n4) break;
                        const float4 y = x4[i];
                        if (fmaxf(fmaxf(y.x, y.y), fmaxf(y.z, y.w)) >= bound) {
                            f(y.x, base + 4 * i), f(y.y, base + 4 * i + 1), f(y.z, base + 4 * i + 2), f(y.w, base + 4 * i + 3);
                        }
                    }
                }
                if (rank == 0 && tid < head) f(row[tid], tid);
                if (rank == nc - 1 && tail + tid < a.V && tid < 4) f(row[tail + tid], tail + tid);
            };
            for (bool again = false;; again = true) {
                all_values(take);
                __syncthreads();
                listed = s_n;
                if (listed <= kLpShort || again) break;
                // A warp whose values are few, masked away or equal lets the bound be anything: then the n_top-th of all lanes' largest
                // keys. (All of them listed and ranked: one row of 1540 values 100 us, so 9.0; one of 151,936 with 60,000 masked 152, so 13.7.)
                u64 own = 0, key = 0;
                all_values([&](float v, int i) {
                    if (v >= bound) own = max(own, lp_key(v, i));
                });
                for (int i = 0; i < a.n_top; i++) {        // the warp's, in falling order
                    const u64 most = max_key(own);
                    if (lane == i) key = most;
                    if (own == most) own = 0;
                }
                s_list[tid] = key;
                __syncthreads();
                if (tid == 0) s_n = 0, s_lowest = 0;
                __syncthreads();
                if (key != 0 && lp_above(s_list, kLpWarps, key) == a.n_top - 1) s_lowest = key;
                __syncthreads();
                lowest = s_lowest;
            }
            if (listed > kLpList) {                        // fewer lanes than n_top have all the values: one after the other
                u64 last = ~0ull;
                for (int q = 0; q < a.n_top; q++) {
                    u64 most = 0;
                    all_values([&](float v, int i) {
                        if (v >= bound) {
                            const u64 k = lp_key(v, i);
                            if (k < last && k > most) most = k;
                        }
                    });
                    most = max_key(most);
                    if (lane == 0) s_list[warp] = most;
                    __syncthreads();
                    for (int w = 0; w < kLpWarps; w++) most = s_list[w] > most ? s_list[w] : most;
                    __syncthreads();
                    if (tid == 0) list[q] = most;
                    last = most;
                }
                listed = a.n_top;
            }
        }
    }
    cl.barrier_wait(std::move(started));
    __syncthreads();
    if (warp == 0) {
        p = join(lane < kLpWarps ? s_warp[lane] : LpPart{-INFINITY, 0.0f, 0.0f});
        if (s_abort || p.m == INFINITY) p.z = NAN;
        if (lane == 0) *cl.map_shared_rank(&s_part[rank], 0) = p;
    }
    if constexpr (KEEP) {
        for (int i = tid; i < listed; i += kLpThreads) {
            const u64 k = list[i];
            int above = 0;
#pragma unroll 8
            for (int j = 0; j < listed; j++) above += list[j] > k;
            if (k != 0 && above < a.n_top) cl.map_shared_rank(s_all, 0)[rank * kLpTop + above] = k;
        }
    } else if (best != 0) {
        const int above = lp_above(s_list, kLpWarps, best);
        if (above < a.n_top) cl.map_shared_rank(s_all, 0)[rank * kLpTop + above] = best;
    }
    cl.sync();
    if (s_abort && tid == 0 && a.err) atomicOr(a.err, QMS_PAGED_ETIMEOUT);
    if (rank != 0) return;

    // ---- the row: parts and lists joined
    p = join(lane < nc ? s_part[lane] : LpPart{-INFINITY, 0.0f, 0.0f});
    const bool none = p.m == -INFINITY && !isnan(p.z);     // a row of -inf
    const float lz = log1pf(p.z);
    auto logp = [&](float v) { return none || v == -INFINITY ? (isnan(p.z) ? NAN : -INFINITY) : __fdiv_rn(v * a.h - p.m * a.h, a.temp) - lz; };
    for (int i = tid; i < a.n_ids; i += kLpThreads) {
        const int id = a.ids[r * a.n_ids + i];
        const bool good = (unsigned)id < (unsigned)a.V;
        if (!good && a.err) atomicOr(a.err, QMS_PAGED_ETOKEN);
        a.lp[r * a.n_ids + i] = good ? logp(i < kLpThreads ? mine : row[id]) : NAN;
    }
    if (tid == 0 && a.entropy) a.entropy[r] = none ? 0.0f : lz - 0.69314718056f * p.t / (1.0f + p.z);
    if (a.n_top == 0) return;
    const u64 k = tid < nc * kLpTop ? s_all[tid] : 0;
    const int found = __syncthreads_count(k != 0);
    if (k != 0) {
        const int above = lp_above(s_all, nc, k);
        if (above < a.n_top) {
            a.top_id[r * a.n_top + above] = (int)~(uint32_t)k;
            a.top_lp[r * a.n_top + above] = logp(lp_value(k));
        }
    }
    if (tid >= found && tid < a.n_top) {
        a.top_id[r * a.n_top + tid] = -1;
        a.top_lp[r * a.n_top + tid] = isnan(p.z) ? NAN : -INFINITY;
    }
}

static int launch_logprobs(const LogprobArgs &a, int rows, cudaStream_t s) {
    constexpr int ring = kLpWarps * kLpRing * kLpChunk * 4, keep = kLpWarps * kLpKeep * kLpChunk * 4 + kLpList * 8;
    static std::atomic<unsigned long long> done[2];
    int rc = allow_smem(done[0], k_logprobs<false>, ring);
    if (rc || (rc = allow_smem(done[1], k_logprobs<true>, keep))) return rc;
    // CTAs per row: at most 8, a warp's piece a chunk at least, and as many as fill the device
    int nc = 1;
    while (nc < kRowCtas && a.V > nc * kLpWarps * kLpChunk && (int64_t)rows * nc < 500) nc *= 2;
    // Kept in shared memory for few CTAs. Both in us, not kept and kept: 1 row of 151,936 14.3, 10.2; 8 rows 14.8, 11.3; 19 rows 16.9, 18.5; 64
    // rows of 4096 8.4, 7.2; 16 rows of 32,003 9.1, 11.7.
    const bool few = (int64_t)rows * nc <= kLpFew && a.V / nc + 8 <= kLpWarps * kLpKeep * kLpChunk;
    if (few) return launch_rows(k_logprobs<true>, kLpThreads, rows, nc, keep, s, a);
    return launch_rows(k_logprobs<false>, kLpThreads, rows, nc, ring, s, a);
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
    QMS_REQUIRE(temp >= FLT_MIN && temp <= FLT_MAX, QMS_CUDA_EINVAL, "logprobs: temp must be positive and finite, at least 2^-126");
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
    // From a temperature of 1 on a difference is taken of the halves: of two values of fp32's whole range it may be past that range where x is
    // not. (Below 1 x is then too.) c is neither 0 nor infinite, which would make NaN of the maximum and of -inf.
    a.h = temp >= 1.0f ? 0.5f : 1.0f;
    a.temp = temp * a.h;
    a.c = 1.4426950408889634f / a.temp;
    a.lp = logp;
    a.entropy = entropy;
    a.top_lp = top_logp;
    a.top_id = top_id;
    a.err = err;
    return launch_logprobs(a, rows, (cudaStream_t)stream);
}

}  // extern "C"
