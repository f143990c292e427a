// qms_paged_wide.cu - paged attention where one K / V tile meets many rows (a shared prompt against a batch, drafted
// tokens, a chunk of a prompt): tcgen05 tensor cores, fp16 cache, on B200 (sm_100a).
//
// A unit is 256 rows (two tiles of 128) of one kv head against a chunk of positions, 128 at a time:
//   S = Q K^T   tcgen05.mma kind::f16 from shared memory, M 128 x N 128, K = head_dim, twice: Q = hi + lo
//               in fp16 (22 bits, each row scaled by a power of two into fp16's range), K exact
//   softmax     one thread per row reads its S from TMEM, keeps the running base B and sum l, writes the
//               weights 2^(s f - B) back over S as two fp16 terms
//   O += P V    tcgen05.mma with P from TMEM (hi, then lo) and V as it lies in shared memory (MN-major)
// O stays in TMEM over the whole chunk. It is rescaled only when a row's maximum rises by more than 2^7
// since its base was set, which a base 2^8 below the first maximum and fp16's range of 2^16 allow; the
// result does not depend on it beyond rounding.
//
// Warps 0-3 and 4-7 are the softmax of the two row tiles, warps 8-11 bring K and V in by cp.async (any page size,
// layout and length; positions past the chunk or on bad pages are zeros), one thread of warp 12 issues the
// MMAs: while it works on one row tile, the other's softmax runs. Shared memory: Q 128 KB, a ring of 3
// tiles of 32 KB; TMEM: S 2 x 128, O 2 x 128 columns (head_dim 128).
// Bound by the tensor cores: 4 * 128 * 128 * head_dim flop per tile and product pair, twice for the split.
#include <math.h>
#include <string.h>

#include "qms_moe.cuh"
#include "qms_paged.cuh"
#include "qms_tcgen05.cuh"

namespace qms {

constexpr int kWTile = 128, kWThreads = 416;
constexpr uint32_t kWSpin = 1u << 22;
constexpr float kWLow = 8.0f, kWHigh = 15.0f;       // a new base is 2^8 below the maximum; weights stay below 2^15

template <int D>
struct WideCfg {
    static constexpr int HALVES = D / 64;                       // 64 values = 128 bytes: one swizzle row
    static constexpr uint32_t HALF = kWTile * 128;              // bytes of 128 rows x 64 values
    static constexpr uint32_t TILE = HALVES * HALF;             // a K or V tile; one term of a Q tile
    static constexpr int SLOTS = 3, CH = D / 8;                 // CH: 16-byte pieces per row
    static constexpr uint32_t RING = 4 * TILE, META = RING + SLOTS * TILE;
    // meta: page offsets [2][128] int64, bad-page masks [4][4], barriers, flags
    static constexpr uint32_t BAD = META + 2 * kWTile * 8, BARS = BAD + 64, SMEM = BARS + 16 * 8 + 64;
    static constexpr uint32_t O_COL = 256;                      // TMEM columns: S0, S1, O0, O1
};

__device__ __forceinline__ uint64_t desc_sw128(uint32_t saddr, uint32_t lbo, uint32_t sbo) { return umma_desc(saddr, lbo, sbo) | (2ull << 61); }

// D[tmem] (+)= A B^T, fp16 in, fp32 out: A from shared memory / from TMEM
__device__ __forceinline__ void umma_f16_ss(uint32_t d, uint64_t da, uint64_t db, uint32_t idesc, bool acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(da), "l"(db), "r"(idesc), "r"((uint32_t)acc)
        : "memory");
}
__device__ __forceinline__ void umma_f16_ts(uint32_t d, uint32_t a, uint64_t db, uint32_t idesc, bool acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d), "r"(a), "l"(db), "r"(idesc), "r"((uint32_t)acc)
        : "memory");
}
// M 128 x N, f16 x f16 -> f32, A K-major, B K-major or MN-major
__host__ __device__ constexpr uint32_t idesc_f16(int N, bool b_mn) {
    return (1u << 4) | ((uint32_t)b_mn << 16) | ((uint32_t)(N >> 3) << 17) | ((128u >> 4) << 24);
}

// The loads into r are complete, and no use of r may move before this.
__device__ __forceinline__ void tmem_wait_ld(uint32_t (&r)[32]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]),
                   "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]), "+r"(r[16]), "+r"(r[17]), "+r"(r[18]),
                   "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]),
                   "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31])::"memory");
}
__device__ __forceinline__ void tmem_st32(uint32_t addr, const uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,"
        "%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(addr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]),
        "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]),
        "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
        : "memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Bounded wait for a phase of a barrier; a wait that gives up ends the CTA's work (flag) and is reported.
struct WideSync {
    volatile int *abort;
    const Paged *a;
    __device__ bool wait(uint64_t *bar, uint32_t parity) const {
        for (uint32_t n = 0; !mbar_try_wait(bar, parity); n++) {
            if (*abort) return false;
            if (n == kWSpin) {
                *abort = 1;
                paged_err(*a, QMS_PAGED_ETIMEOUT);
                return false;
            }
            if (n > 64) __nanosleep(32);
        }
        return true;
    }
};

// One unit of work; every role derives it from the unit's number.
struct WideUnit {
    bool any;                        // there is something to do
    int kh, b, t0, n, kv, slot, k0, k1, r0, rows, nt, tiles, lo;
    // kv head; sequence, its first row, rows and length (own); slot of the partial result; positions [k0, k1) in
    // nt tiles; first row and number of rows of the segment; row tiles (1 or 2); every row of the unit sees
    // the positions up to lo
    __device__ WideUnit(const PagedAttn &A, bool own, int lo_p, int u) {
        const Paged &a = A.a;
        kh = u % a.Hk;
        u /= a.Hk;
        const int nt_rows = own ? A.p.tiles_s : A.p.tiles_p, tile = u % nt_rows;
        u /= nt_rows;
        r0 = tile * 2 * kWTile;
        b = t0 = n = kv = 0;
        if (own) {
            b = u % a.n_seq;
            slot = u / a.n_seq;
            paged_seq(a, b, t0, n, kv);
            rows = n * a.G;
            k0 = a.prefix + slot * A.p.chunk_s;
            k1 = min(kv, k0 + A.p.chunk_s);
            lo = kv - n + r0 / a.G;
            k1 = min(k1, kv - n + min(n - 1, (r0 + 2 * kWTile - 1) / a.G) + 1);     // nobody sees the rest
            slot += A.p.slots_p;
        } else {
            slot = u;
            rows = a.n_tok * a.G;
            k0 = slot * A.p.chunk_p;
            k1 = min(a.prefix, k0 + A.p.chunk_p);
            lo = lo_p;
        }
        any = r0 < rows && k0 < k1;
        nt = (k1 - k0 + kWTile - 1) / kWTile;
        tiles = rows - r0 > kWTile ? 2 : 1;
    }
};

template <int D>
__global__ void __launch_bounds__(kWThreads, 1) k_paged_wide(const PagedAttn A, const bool own, const bool last) {
    using C = WideCfg<D>;
    extern __shared__ __align__(1024) unsigned char sm[];
    const Paged &a = A.a;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const uint32_t sm0 = smem_u32(sm);
    int64_t *s_off = reinterpret_cast<int64_t *>(sm + C::META);
    uint32_t *s_bad = reinterpret_cast<uint32_t *>(sm + C::BAD);
    uint64_t *full = reinterpret_cast<uint64_t *>(sm + C::BARS), *empty = full + C::SLOTS;
    uint64_t *q_full = empty + C::SLOTS, *s_full = q_full + 2, *p_full = s_full + 2, *drain = p_full + 2;
    int *s_int = reinterpret_cast<int *>(drain + 1);              // abort, V set aside, TMEM base, least position
    volatile int *s_abort = s_int, *s_flag = s_int + 1;
    int *s_lo = s_int + 3;
    uint32_t *s_tmem = reinterpret_cast<uint32_t *>(s_int + 2);
    if (sm0 & 1023) {                             // the swizzled tiles need it; never seen
        if (tid == 0) paged_err(a, QMS_PAGED_ETIMEOUT);
        pdl_wait();
        return;
    }
    if (tid == 0) {
        for (int i = 0; i < C::SLOTS; i++) {
            mbar_init(&full[i], 128);
            mbar_init(&empty[i], 1);
        }
        for (int i = 0; i < 2; i++) {
            mbar_init(&q_full[i], 128);
            mbar_init(&s_full[i], 1);
            mbar_init(&p_full[i], 4);
        }
        mbar_init(drain, 1);
        s_int[0] = s_int[1] = 0;
        *s_lo = 0x7fffffff;
        fence_mbar_init();
    }
    if (warp == 12) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(s_tmem)), "r"(512) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    if (!last) pdl_wait();
    pdl_trigger();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *s_tmem;
    if (!own) {                                   // the least position among all rows: what lies below needs no mask
        int lo = 0x7fffffff;
        for (int b = tid; b < a.n_seq; b += kWThreads) {
            int t0, n, kv;
            if (paged_seq(a, b, t0, n, kv) && n > 0) lo = min(lo, kv - n);
        }
        lo = __reduce_min_sync(kFull, lo);
        if (lane == 0) atomicMin(s_lo, lo);
        __syncthreads();
    }
    const int lo_p = *s_lo;
    const int n_unit = (own ? A.p.slots_s * a.n_seq * A.p.tiles_s : A.p.slots_p * A.p.tiles_p) * a.Hk;
    const WideSync sy{s_abort, &a};

    if (warp < 8) {
        // ---- softmax of row tile i: thread = row = TMEM lane
        const int i = warp >> 2, row = (warp & 3) * 32 + lane;
        const uint32_t lanes = tmem + ((uint32_t)((warp & 3) * 32) << 16);
        const uint32_t s_col = lanes + i * kWTile, o_col = lanes + C::O_COL + i * D;
        uint32_t ns = 0, tiles_done = 0;          // phases of s_full; tiles seen by the CTA (for s_bad)
        bool ok = true;
        for (int u = blockIdx.x; u < n_unit && ok; u += gridDim.x) {
            const WideUnit w(A, own, lo_p, u);
            if (!w.any) continue;
            if (i >= w.tiles) {
                tiles_done += w.nt;
                continue;
            }
            // this row: position, token row * H + head (-1: none)
            const int r = w.r0 + i * kWTile + row;
            int pos = -1, tok = -1;
            if (own) {
                const int t = r / a.G;
                if (r < w.rows) pos = w.kv - w.n + t, tok = (w.t0 + t) * a.H + w.kh * a.G + (r - t * a.G);
            } else {
                const int t = r / a.G, t_end = min(a.n_tok - 1, __shfl_sync(kFull, t, 31));
                for (int x = __shfl_sync(kFull, t, 0); x <= t_end; x++) {
                    int s0 = 0, sn = 0, skv = 0;
                    const int sb = paged_seq_of(a, x);
                    if (sb < a.n_seq) paged_seq(a, sb, s0, sn, skv);
                    if (t == x && r < w.rows) {
                        pos = x >= s0 && x < s0 + sn ? skv - sn + (x - s0) : -1;
                        tok = x * a.H + w.kh * a.G + (r - x * a.G);
                    }
                }
            }
            // q: 8 lanes per row, 4 rows at a time: row maximum, power-of-two scale, two fp16 terms, swizzled rows
            float f = 0.0f;
            const float sign = A.scale2 < 0.0f ? -1.0f : 1.0f;     // f >= 0: the largest s f has the largest s
            const uint32_t qb = sm0 + i * 2 * C::TILE;
#pragma unroll 2
            for (int g = 0; g < 8; g++) {
                const int src = 4 * g + (lane >> 3), part = lane & 7;
                const int tk = __shfl_sync(kFull, tok, src);
                float4 x[D / 32];
                float mx = 0.0f;
#pragma unroll
                for (int k = 0; k < D / 32; k++) {
                    x[k] = tk < 0 ? make_float4(0.0f, 0.0f, 0.0f, 0.0f)
                                  : __ldcg(reinterpret_cast<const float4 *>(A.q + (tk / a.H) * A.ldq + (int64_t)(tk % a.H) * D + part * 4 + k * 32));
                    mx = fmaxf(mx, fmaxf(fmaxf(fabsf(x[k].x), fabsf(x[k].y)), fmaxf(fabsf(x[k].z), fabsf(x[k].w))));
                }
                mx = fmaxf(mx, __shfl_xor_sync(kFull, mx, 1));
                mx = fmaxf(mx, __shfl_xor_sync(kFull, mx, 2));
                mx = fmaxf(mx, __shfl_xor_sync(kFull, mx, 4));
                const int e = mx > 0.0f && mx < INFINITY ? ilogbf(mx) - 9 : 0;
                const float fr = ldexpf(fabsf(A.scale2), e), got = __shfl_sync(kFull, fr, (lane & 3) * 8);
                if (lane >> 2 == g) f = got;
                const float d1 = ldexpf(sign, -e / 2), d2 = ldexpf(1.0f, -e - -e / 2);
                const int rr = (warp & 3) * 32 + src;
#pragma unroll
                for (int k = 0; k < D / 32; k++) {
                    const float y[4] = {x[k].x * d1 * d2, x[k].y * d1 * d2, x[k].z * d1 * d2, x[k].w * d1 * d2};
                    uint32_t h[2], l[2];
                    split_h2(y[0], y[1], h[0], l[0]);
                    split_h2(y[2], y[3], h[1], l[1]);
                    const int d = part * 4 + k * 32;
                    const uint32_t at = qb + (d >> 6) * C::HALF + rr * 128 + ((((d & 63) >> 3) ^ (rr & 7)) << 4) + (d & 4) * 2;
                    asm volatile("st.shared.v2.b32 [%0], {%1, %2};" ::"r"(at), "r"(h[0]), "r"(h[1]) : "memory");
                    asm volatile("st.shared.v2.b32 [%0], {%1, %2};" ::"r"(at + C::TILE), "r"(l[0]), "r"(l[1]) : "memory");
                }
            }
            fence_async_smem();
            mbar_arrive(&q_full[i]);

            const int lim = min(pos, w.k1 - 1);   // last position that this row sees
            float B = -INFINITY, l = 0.0f;
            for (int j = 0; j < w.nt; j++, tiles_done++) {
                if (!(ok = __all_sync(kFull, sy.wait(&s_full[i], ns & 1)))) break;    // the whole warp or none of it
                ns++;
                tc_fence_after();
                const int base = w.k0 + j * kWTile;
                const uint32_t *bad = s_bad + (tiles_done & 3) * 4;
                const uint32_t bads[4] = {bad[0], bad[1], bad[2], bad[3]};
                // rows that see nothing of this chunk are not read from its slot: no mask for them
                const bool mask = __any_sync(kFull, lim >= w.k0 && lim < base + kWTile - 1) || (bads[0] | bads[1] | bads[2] | bads[3]);
                uint32_t vis[4];
#pragma unroll
                for (int c = 0; c < 4; c++) {
                    const int d = lim - base - 32 * c;
                    vis[c] = (d < 0 ? 0u : d >= 31 ? 0xffffffffu : (2u << d) - 1u) & ~bads[c];
                }
                float mx = -INFINITY;
#pragma unroll
                for (int c = 0; c < 4; c++) {
                    uint32_t s[32];
                    tmem_ld<32>(s_col + 32 * c, s);
                    tmem_wait_ld(s);
                    if (mask) {
#pragma unroll
                        for (int e = 0; e < 32; e++) mx = fmaxf(mx, vis[c] >> e & 1 ? __uint_as_float(s[e]) : -INFINITY);
                    } else {
#pragma unroll
                        for (int e = 0; e < 32; e++) mx = fmaxf(mx, __uint_as_float(s[e]));
                    }
                }
                mx = mx == -INFINITY ? mx : mx * f;
                const bool rise = mx > B + kWHigh;
                if (__any_sync(kFull, rise)) {
                    const float nb = rise ? mx - kWLow : B, fac = B == -INFINITY ? 0.0f : ex2(B - nb);
                    B = nb;
                    l *= fac;
                    if (j > 0) {                  // the MMAs up to tile j - 1 ended before S of tile j was announced
#pragma unroll
                        for (int c = 0; c < D / 32; c++) {
                            uint32_t o[32];
                            tmem_ld<32>(o_col + 32 * c, o);
                            tmem_wait_ld(o);
#pragma unroll
                            for (int e = 0; e < 32; e++) o[e] = __float_as_uint(__uint_as_float(o[e]) * fac);
                            tmem_st32(o_col + 32 * c, o);
                        }
                    }
                }
                const float nB = B == -INFINITY ? 0.0f : -B;
#pragma unroll
                for (int c = 0; c < 4; c++) {
                    uint32_t s[32], o[32];
                    tmem_ld<32>(s_col + 32 * c, s);
                    tmem_wait_ld(s);
                    float g = 0.0f;
#pragma unroll
                    for (int e = 0; e < 32; e += 2) {
                        float p0 = ex2(fmaf(__uint_as_float(s[e]), f, nB)), p1 = ex2(fmaf(__uint_as_float(s[e + 1]), f, nB));
                        if (mask) {
                            p0 = vis[c] >> e & 1 ? p0 : 0.0f;
                            p1 = vis[c] >> e & 2 ? p1 : 0.0f;
                        }
                        g += p0 + p1;
                        split_h2(p0, p1, o[e / 2], o[16 + e / 2]);
                    }
                    l += g;
                    tmem_st32(s_col + 32 * c, o); // hi of 32 positions in 16 columns, lo in the next 16
                }
                tmem_wait_st();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&p_full[i]);
            }
            if (!ok || !(ok = __all_sync(kFull, sy.wait(&s_full[i], ns & 1)))) break;     // O is complete
            ns++;
            tc_fence_after();
            if (isnan(l) && B == -INFINITY) B = 0.0f;
            const bool put = tok >= 0 && lim >= w.k0, none = l == 0.0f, fix = *s_flag != 0;
            float *dst = A.part_o + ((int64_t)w.slot * a.n_tok * a.H + (put ? tok : 0)) * D;
#pragma unroll
            for (int c = 0; c < D / 32; c++) {
                uint32_t o[32];
                tmem_ld<32>(o_col + 32 * c, o);
                tmem_wait_ld(o);
                if (fix && put) {
                    // V that were set aside: added where the row sees them (inf and NaN are not changed by a weight)
                    for (int p = max(w.k0, w.lo + 1); p <= lim; p++) {
                        const int64_t at = paged_at(a, a.table + (own ? (int64_t)w.b * a.table_stride : 0), p);
                        if (at < 0) continue;
                        const __half *vr = reinterpret_cast<const __half *>(a.v + at + w.kh * a.head_stride) + 32 * c;
#pragma unroll
                        for (int e = 0; e < 32; e++) {
                            const float v = kv_ld(vr + e);
                            if (!isfinite(v)) o[e] = __float_as_uint(__uint_as_float(o[e]) + v);
                        }
                    }
                }
                if (put) {
#pragma unroll
                    for (int e = 0; e < 32; e += 4)
                        *reinterpret_cast<float4 *>(dst + 32 * c + e) =
                            none ? make_float4(0.0f, 0.0f, 0.0f, 0.0f)
                                 : make_float4(__uint_as_float(o[e]), __uint_as_float(o[e + 1]), __uint_as_float(o[e + 2]), __uint_as_float(o[e + 3]));
                }
            }
            if (put) A.part_ml[(int64_t)w.slot * a.n_tok * a.H + tok] = make_float2(none ? -INFINITY : B, l);
            tc_fence_before();
        }
    } else if (warp < 12) {
        // ---- K and V: load c = 2 t (K), 2 t + 1 (V) of the CTA's tile t into ring slot c % SLOTS
        const int pt = tid - 256, pw = warp - 8, piece = pt % C::CH, row0 = pt / C::CH;
        constexpr int RS = 128 / C::CH;           // rows between a thread's pieces
        uint32_t c = 0, t = 0;
        int pend = -1;                            // the load that is issued but not announced
        bool pend_scan = false, ok = true;
        int pend_base = 0, pend_lo = 0;
        auto announce = [&]() {
            const uint32_t dst = sm0 + C::RING + (pend % C::SLOTS) * C::TILE;
            if (pend_scan) {                      // V behind the causal mask: a weight of 0 does not cancel inf
#pragma unroll 4
                for (int k = 0; k < kWTile / RS; k++) {
                    const int r = row0 + k * RS;
                    if (pend_base + r <= pend_lo) continue;
                    const uint32_t at = dst + (piece >> 3) * C::HALF + r * 128 + (((piece & 7) ^ (r & 7)) << 4);
                    uint4 *pv = reinterpret_cast<uint4 *>(sm + (at - sm0));
                    uint4 v = *pv;
                    if (drop_nonfinite((const __half *)nullptr, v)) {
                        *pv = v;
                        *s_flag = 1;
                    }
                }
            }
            fence_async_smem();
            mbar_arrive(&full[pend % C::SLOTS]);
            pend = -1;
        };
        auto issue = [&](const int64_t *off, const char *pool, int kh, bool scan, int base, int lo) {
            const uint32_t slot = c % C::SLOTS;
            if (c >= C::SLOTS) {
                const uint32_t ph = (c / C::SLOTS - 1) & 1;
                if (!mbar_test_wait(&empty[slot], ph)) {
                    if (pend >= 0) {              // do not hold back what has landed
                        cp_wait<0>();
                        announce();
                    }
                    if (!sy.wait(&empty[slot], ph)) return false;
                }
            }
            const uint32_t dst = sm0 + C::RING + slot * C::TILE;
#pragma unroll 4
            for (int k = 0; k < kWTile / RS; k++) {
                const int r = row0 + k * RS;
                const int64_t at = off[r];
                cp_async16_or0(dst + (piece >> 3) * C::HALF + r * 128 + (((piece & 7) ^ (r & 7)) << 4),
                               pool + (at < 0 ? 0 : at + kh * a.head_stride + piece * 16), at >= 0);
            }
            cp_commit();
            if (pend >= 0) {
                cp_wait<1>();
                announce();
            }
            pend = (int)c++;
            pend_scan = scan;
            pend_base = base;
            pend_lo = lo;
            return true;
        };
        for (int u = blockIdx.x; u < n_unit; u += gridDim.x) {     // after a failed wait: the barriers, no copies
            const WideUnit w(A, own, lo_p, u);
            if (!w.any) continue;
            const int *table = a.table + (own ? (int64_t)w.b * a.table_stride : 0);
            for (int j = 0; j < w.nt; j++, t++) {
                const int base = w.k0 + j * kWTile, p = base + pt;
                int64_t *off = s_off + (t & 1) * kWTile;
                int64_t at = -1;
                if (p < w.k1) {
                    at = paged_at(a, table, p);
                    if (at < 0) paged_err(a, QMS_PAGED_EPAGE);
                }
                off[pt] = at;
                const uint32_t bad = __ballot_sync(kFull, p < w.k1 && at < 0);
                if (lane == 0) s_bad[(t & 3) * 4 + pw] = bad;
                asm volatile("bar.sync 1, 128;" ::: "memory");
                ok = ok && issue(off, a.k, w.kh, false, 0, 0) && issue(off, a.v, w.kh, base + kWTile - 1 > w.lo, base, w.lo);
                ok = __all_sync(kFull, ok) && !*s_abort;
            }
        }
        cp_wait<0>();
        if (pend >= 0) announce();
    } else {
        // ---- the MMAs, by one thread
        if (lane == 0) {
            constexpr uint32_t id_s = idesc_f16(kWTile, false), id_o = idesc_f16(D, true);
            uint32_t c = 0, nq[2] = {0, 0}, np[2] = {0, 0};
            bool ok = true;
            auto score = [&](int i, uint32_t kc) {             // S_i = (hi + lo of Q_i) K^T
                const uint32_t k = sm0 + C::RING + (kc % C::SLOTS) * C::TILE, q = sm0 + i * 2 * C::TILE;
#pragma unroll
                for (int term = 0; term < 2; term++)
#pragma unroll
                    for (int ks = 0; ks < D / 16; ks++) {
                        const uint32_t o = (ks >> 2) * C::HALF + (ks & 3) * 32;
                        umma_f16_ss(tmem + i * kWTile, desc_sw128(q + term * C::TILE + o, 16, 1024), desc_sw128(k + o, 16, 1024), id_s, term || ks);
                    }
            };
            auto weigh = [&](int i, uint32_t vc, bool first) { // O_i (+)= (hi + lo of P_i) V
                const uint32_t v = sm0 + C::RING + (vc % C::SLOTS) * C::TILE;
#pragma unroll
                for (int term = 0; term < 2; term++)
#pragma unroll
                    for (int ks = 0; ks < kWTile / 16; ks++)
                        umma_f16_ts(tmem + C::O_COL + i * D, tmem + i * kWTile + (ks >> 1) * 32 + term * 16 + (ks & 1) * 8,
                                    desc_sw128(v + ks * 2048, C::HALF, 1024), id_o, !first || term || ks);
            };
            auto full_at = [&](uint32_t x) { return sy.wait(&full[x % C::SLOTS], (x / C::SLOTS) & 1); };
            for (int u = blockIdx.x; u < n_unit && ok; u += gridDim.x) {
                const WideUnit w(A, own, lo_p, u);
                if (!w.any) continue;
                if (!(ok = full_at(c))) break;
                for (int i = 0; i < w.tiles && ok; i++) {
                    if (!(ok = sy.wait(&q_full[i], nq[i]++ & 1))) break;
                    tc_fence_after();
                    score(i, c);
                    umma_commit(&s_full[i]);
                }
                if (!ok) break;
                umma_commit(&empty[c % C::SLOTS]);
                for (int j = 0; j < w.nt && ok; j++, c += 2) {
                    if (!(ok = full_at(c + 1))) break;
                    const bool more = j + 1 < w.nt;
                    for (int i = 0; i < w.tiles && ok; i++) {
                        if (!(ok = sy.wait(&p_full[i], np[i]++ & 1))) break;
                        tc_fence_after();
                        weigh(i, c + 1, j == 0);
                        if (i == w.tiles - 1) umma_commit(&empty[(c + 1) % C::SLOTS]);
                        if (more) {
                            if (i == 0 && !(ok = full_at(c + 2))) break;
                            score(i, c + 2);
                        }
                        umma_commit(&s_full[i]);
                    }
                    if (ok && more) umma_commit(&empty[(c + 2) % C::SLOTS]);
                }
            }
            if (!ok) {                                          // nothing of this CTA's is in flight when TMEM goes
                umma_commit(drain);
                for (uint32_t n = 0; n < kWSpin && !mbar_try_wait(drain, 0); n++) __nanosleep(32);
            }
        }
        __syncwarp();
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 12) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
    }
    if (last) pdl_wait();
}

template <int D>
static int launch_wide(const PagedAttn &A, bool own, bool last, cudaStream_t s) {
    using C = WideCfg<D>;
    static_assert(C::SMEM <= 232448, "shared memory per CTA");
    const int64_t units = own ? (int64_t)A.p.slots_s * A.a.n_seq * A.p.tiles_s * A.a.Hk : (int64_t)A.p.slots_p * A.p.tiles_p * A.a.Hk;
    QMS_REQUIRE(units < (1ll << 30), QMS_CUDA_EUNSUPPORTED, "paged_attention: too many units of work");
    static unsigned long long set = 0;                          // per device
    int dev = 0;
    QMS_CK(cudaGetDevice(&dev));
    if (!(set >> (dev & 63) & 1)) {
        QMS_CK(cudaFuncSetAttribute(k_paged_wide<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM));
        set |= 1ull << (dev & 63);
    }
    const int grid = (int)(units < 148 ? units : 148);
    QMS_CK(launch_pdl(k_paged_wide<D>, dim3(grid), dim3(kWThreads), C::SMEM, s, A, own, last));
    return QMS_CUDA_OK;
}

int launch_paged_wide(const PagedAttn &A, int D, bool own, bool last, cudaStream_t s) {
    return D == 128 ? launch_wide<128>(A, own, last, s) : launch_wide<64>(A, own, last, s);
}

}  // namespace qms
