// qms_paged_wide.cu - paged attention on tcgen05 tensor cores (B200, sm_100a): for many rows per K / V tile (a shared
// prompt against a batch, drafted tokens, a chunk of a prompt), and for fp32 caches.
//
// A unit is a run of positions, a tile at a time, of one kv head against rows; two streams of tiles take turns, so
// that the tensor cores work on one while the other's softmax runs:
//   PAIR   fp16 cache, 256 rows: a stream per 128 rows, both over every tile of 128 positions
//   SPLIT  fp16 cache, 128 rows: the even and the odd tiles, joined at the end of the unit
//   F32    fp32 cache, 128 rows: the same with tiles of 64 positions, split into fp16 terms on the way
//   NIB    cache in 4 bits, 128 rows: as F32, tiles of 128 positions, to fp16 on the way, exact (one term); for up to 256 rows on a
//          position or several sequences' own ones (beyond that the positions go to fp16 in the workspace first, and PAIR reads them)
// For each tile of a stream
//   S = Q K^T   tcgen05.mma kind::f16 from shared memory, M 128, N the positions, K = head_dim, with 22-bit operands: Q =
//               hi + lo in fp16 (each row scaled by a power of two into fp16's range), K exact in fp16 (two
//               products) or K = hi + lo under a scale of its tile (three: lo * lo is below 2^-22)
//   softmax     one thread per row reads its S from TMEM, keeps the running base B and sum l, writes the
//               weights 2^(s f - B) back over S as two fp16 terms
//   O += P V    tcgen05.mma with P from TMEM (hi, lo) and V as it lies in shared memory (MN-major), fp32 V = hi + lo
//               under the largest scale so far (O is in its units)
// O stays in TMEM over the whole unit. A base is set 2^8 below a maximum and stays until a score lies 2^15 above it
// (fp16 holds weights to 2^16), so that the maximum needs no pass of its own; the result does not depend on
// it beyond rounding. In PAIR O is taken out after every 8 tiles and added to the unit's partial result in global memory
// (tensor cores add by cutting bits off, the longer the more); the other units are that short.
//
// Warps 0-3 and 4-7 are the softmax of the two streams. One warp brings K and V in by TMA, a box per page: 64 swizzled
// values x the page's positions (fp32: whole rows, into a staging ring, from which four warps write the terms). Tiles
// start on page boundaries, so a tile may begin before the first position of its unit: such rows are masked. V
// values that are not finite in rows that some row does not see are set aside (a weight of 0 does not cancel
// them), by one warp or by the four. One thread each of two warps issues the MMAs of a stream, a product at a time
// under a lock: one thread for both leaves the tensor cores idle while it waits and commits (some 1200 of 6150 cycles
// per pair of tiles: hardly one MMA is queued), two that interleave slow every MMA down.
// Shared memory at head_dim 128: Q 128 KB and a ring of 3 tiles of 32 KB (PAIR), Q 64 KB and a ring of 2 for each stream
// (SPLIT), Q 64 KB, 2 stages and a ring of 3 (F32, NIB); TMEM: S 2 x 128, O 2 x 128 columns.
// Bound by the tensor cores, 4 * 128 * 128 * head_dim flop per 128 rows and positions, times 2 (fp16) or 3, and by the softmax
// between a tile's two products where the other stream does not cover it: 64 sequences of 5 tokens (64 q heads, 4 kv heads)
// over 8192 shared and 640 own fp16 positions take 235 us, 394 TFLOP/s by the definition and 788 with the split; tensor
// cores 45% active. A prompt chunk of 256 tokens over 4096 positions: 85 us, 394 TFLOP/s. Over 4 bits by way of the workspace 251 and 86 us
// (the step to fp16 some 8 of the 251); NIB for the same 348 and 119: its four warps convert each tile for 128 rows, some 2000 cycles.
#include <math.h>
#include <string.h>

#include <type_traits>

#include "qms_moe.cuh"
#include "qms_paged.cuh"
#include "qms_tcgen05.cuh"

namespace qms {

enum { PAIR, SPLIT, F32, NIB };
constexpr float kWLow = 8.0f, kWHigh = 15.0f;       // a new base is 2^8 below the maximum; weights stay below 2^15

template <int D, int MODE>
struct WideCfg {
    static constexpr bool CONV = MODE == F32 || MODE == NIB;    // K and V are written by four warps, from stages
    static constexpr int TP = MODE == F32 ? 64 : 128, ROWS = MODE == PAIR ? 256 : 128;     // positions per tile, rows per unit
    static constexpr int THREADS = CONV ? 480 : 384, REGS = CONV ? 128 : 168;    // (4, 3 warps per scheduler)
    static constexpr int TMA_WARP = CONV ? 12 : 8, MMA_WARP = CONV ? 13 : 10;
    static constexpr int PIECE = MODE == PAIR ? 8 : 1 << 30;    // tiles that O adds up before it is taken out
    static constexpr int HALVES = D / 64;                       // 64 values = 128 bytes: one swizzle row
    static constexpr uint32_t QHALF = 128 * 128, QTILE = HALVES * QHALF;     // one term of 128 rows of Q
    static constexpr uint32_t HALF = TP * 128, TILE = HALVES * HALF;         // one term of a K or V tile
    static constexpr uint32_t SLOT = (MODE == F32 ? 2 : 1) * TILE;
    static constexpr int SLOTS = MODE == SPLIT ? 4 : 3;
    static constexpr uint32_t RING = (MODE == PAIR ? 4 : 2) * QTILE, STAGE = RING + SLOTS * SLOT;
    static constexpr uint32_t STAGED = MODE == F32 ? TP * D * 4 : MODE == NIB ? TP * q4_row(D) : 0;
    // then: bad-page masks [8][4]; scales of K and V tiles [2][4], maxima [2][4]; a stream's (B, l, V scale) by row;
    // barriers; flags
    static constexpr uint32_t BAD = STAGE + 2 * STAGED, UP = BAD + 128, JOIN = UP + 64,
                              BARS = JOIN + (MODE == PAIR ? 256 * 8 : 128 * 12), SMEM = BARS + 24 * 8 + 32;
    static constexpr uint32_t O_COL = 256;                      // TMEM columns: S0, S1, O0, O1
    // The tensor cores add into fp32 by cutting bits off, towards 0: an addition takes CUT of the sum away on average, 2^-24
    // E[1 / mantissa] = 0.72 * 2^-24 where the terms have bits behind the sum's last (fp32 caches); products of fp16 values
    // have few (0.6 * 2^-24 measured). A sum o = sum p v grows with l = sum p, so that what a tile's ADDS additions take of o is,
    // for given o, expected at ADDS * CUT * o * (l then) / (l at the end), and at half the tile's own weights at most: that is given
    // back at the end. (RISE: while l grows within a tile, of the hi terms.) Nothing is given back where nothing was cut: where l
    // has so few bits that all weights are alike (fp16 values add up exactly then; of fp32 values those whose o has few bits too).
    // What is left, of an output: 1 to 2e-6 for values of either sign, as a plain fp32 softmax; up to 6e-6 for values of one sign (every
    // product is cut at the sum's last bits by itself; the low terms have either sign and lose nothing by that). A row whose
    // first weight is 2^14 to 2^26 times each other one is up to 5e-6 too large, or with values of one sign 9e-6 too small. Half
    // the additions per sum would leave half of that, for 1.12 times the time (F32: 1.19).
    static constexpr float CUT = MODE == F32 ? 4.3e-8f : 3.6e-8f, ADDS = MODE == F32 ? 12.0f : 16.0f, RISE = MODE == F32 ? 2.0f : 4.0f;
    // Load n of a ring (K, V, K, ...): its slot. One ring for both streams; in SPLIT a ring per stream.
    static __device__ __forceinline__ uint32_t slot(int stream, uint32_t n) { return MODE == SPLIT ? 2 * stream + (n & 1) : n % 3; }
    static constexpr uint32_t RINGLEN = MODE == SPLIT ? 2 : 3;
    static __device__ __forceinline__ uint32_t phase(uint32_t n) { return n / RINGLEN & 1; }
};

__device__ __forceinline__ void red4(float *to, const uint32_t *v) {
    asm volatile("red.relaxed.gpu.global.add.v4.f32 [%0], {%1, %2, %3, %4};" ::"l"(to), "f"(__uint_as_float(v[0])), "f"(__uint_as_float(v[1])),
                 "f"(__uint_as_float(v[2])), "f"(__uint_as_float(v[3]))
                 : "memory");
}

// One unit of work, as every role derives it.
struct WideUnit {
    int kh, b, t0, n, kv, slot, k0, k1, kmin, r0, rows, nt, lo;
    // kv head; sequence, its first row, rows and length (own); slot of the partial result; positions
    // [k0, k1) in nt tiles, of which those below kmin belong to another unit; first row and number of rows of the
    // segment; every row of the unit sees the positions up to lo
};

// The units of this CTA in order. Own positions: units blockIdx.x, + gridDim.x, ... of (chunk, sequence, row tile, kv
// head). Shared positions: all (row tile, kv head, position tile) triples in one line, cut into equal runs, the
// same number for each CTA; a run is one unit per row tile and kv head that it crosses.
template <class C>
struct WideWork {
    const PagedAttn &A;
    const bool own;
    const int lo_p;
    unsigned x, end;
    __device__ WideWork(const PagedAttn &A_, bool own_, int lo_p_) : A(A_), own(own_), lo_p(lo_p_) {
        if (own) {
            x = blockIdx.x;
            end = (unsigned)A.p.chunks_s * A.a.n_seq * A.p.tiles_s * A.a.Hk;
        } else {
            x = line_start(A.p, blockIdx.x * A.p.line_per);
            end = line_start(A.p, (blockIdx.x + 1) * A.p.line_per);
        }
    }
    __device__ bool next(WideUnit &w) {
        const Paged &a = A.a;
        while (x < end) {
            w.b = w.t0 = w.n = w.kv = 0;
            if (own) {
                unsigned u = x, d = u / a.Hk;
                x += gridDim.x;
                w.kh = u - d * a.Hk;
                u = d;
                d = u / (unsigned)A.p.tiles_s;
                w.r0 = (u - d * A.p.tiles_s) * C::ROWS;
                u = d;
                d = u / a.n_seq;
                w.b = u - d * a.n_seq;
                paged_seq(a, w.b, w.t0, w.n, w.kv);
                w.k0 = A.p.base_s + d * A.p.chunk_s;
                w.kmin = max(w.k0, a.prefix);
                w.k1 = min(w.kv, w.k0 + A.p.chunk_s);
                w.k1 = min(w.k1, w.kv - w.n + min(w.n - 1, (w.r0 + C::ROWS - 1) / a.G) + 1);     // nobody sees the rest
                w.slot = A.p.slots_p + d;
                w.rows = w.n * a.G;
                w.lo = w.kv - w.n + w.r0 / a.G;
            } else {
                const unsigned nt = A.p.line_nt, u = x / nt, j = x - u * nt, tile = u / a.Hk;
                const unsigned run = line_run(A.p, x), c = min(nt - j, line_start(A.p, run + 1) - x);
                x += c;
                w.kh = u - tile * a.Hk;
                w.r0 = tile * C::ROWS;
                w.slot = run - line_run(A.p, u * nt);
                w.k0 = w.kmin = j * C::TP;
                w.k1 = min(a.prefix, (int)(j + c) * C::TP);
                w.rows = a.n_tok * a.G;
                w.lo = lo_p;
            }
            w.nt = (w.k1 - w.k0 + C::TP - 1) / C::TP;
            if (w.r0 < w.rows && w.kmin < w.k1) return true;
        }
        return false;
    }
};

template <int D, int MODE>
__global__ void __maxnreg__((WideCfg<D, MODE>::REGS)) k_paged_wide(const PagedAttn A, const __grid_constant__ CUtensorMap mk,
                                                                 const __grid_constant__ CUtensorMap mv, const bool own, const bool last) {
    using C = WideCfg<D, MODE>;
    extern __shared__ __align__(1024) unsigned char sm[];
    const Paged &a = A.a;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const uint32_t sm0 = smem_u32(sm);
    uint32_t *s_bad = reinterpret_cast<uint32_t *>(sm + C::BAD);
    uint32_t *s_up = reinterpret_cast<uint32_t *>(sm + C::UP), *s_max = s_up + 8;     // F32: scales of K, of V (4 +), at tile & 3
    float *s_join = reinterpret_cast<float *>(sm + C::JOIN);
    // full, empty: of the ring's slots (F32: `full` is of stream i's K, i, and V, 2 + i); landed: V tiles that go on
    // after a look, or (F32) the stages, at 2 + i when they are free again
    uint64_t *full = reinterpret_cast<uint64_t *>(sm + C::BARS), *empty = full + 4, *landed = empty + 4;
    uint64_t *joined = landed + 4, *q_full = joined + 1, *s_full = q_full + 2, *p_full = s_full + 2, *drain = p_full + 2;
    int *s_int = reinterpret_cast<int *>(drain + 1);              // abort, V set aside, TMEM base, least position, lock
    volatile int *s_abort = s_int, *s_flag = s_int + 1;
    uint32_t *s_tmem = reinterpret_cast<uint32_t *>(s_int + 2);
    int *s_lo = s_int + 3, *s_lock = s_int + 4;
    if (sm0 & 1023) {                             // the swizzled tiles need it; never seen
        if (tid == 0) paged_err(a, QMS_PAGED_ETIMEOUT);
        pdl_wait();
        return;
    }
    if (tid == 0) {
        for (int i = 0; i < 4; i++) {
            mbar_init(&full[i], C::CONV ? 128 : 1);
            mbar_init(&empty[i], MODE == PAIR ? 2 : 1);
            mbar_init(&landed[i], C::CONV && i >= 2 ? 4 : 1);
        }
        for (int i = 0; i < 2; i++) {
            mbar_init(&q_full[i], 128);
            mbar_init(&s_full[i], 1);
            mbar_init(&p_full[i], 4);
        }
        mbar_init(drain, 2);
        mbar_init(joined, 4);
        s_int[0] = s_int[1] = *s_lock = 0;
        *s_lo = 0x7fffffff;
        fence_mbar_init();
    }
    if (warp == C::MMA_WARP) {
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
        for (int b = tid; b < a.n_seq; b += C::THREADS) {
            int t0, n, kv;
            if (paged_seq(a, b, t0, n, kv) && n > 0) lo = min(lo, kv - n);
        }
        lo = __reduce_min_sync(kFull, lo);
        if (lane == 0) atomicMin(s_lo, lo);
        __syncthreads();
    }
    const int lo_p = *s_lo;
    const WideSync sy{s_abort, &a};
    WideWork<C> work(A, own, lo_p);
    WideUnit w = {};
    // The tiles of stream i in a unit of nt: all (PAIR, where it has rows), or every second one, from first_of(i). In F32
    // the streams alternate over all tiles of the CTA (`before` those of earlier units), not from the start of each
    // unit: the one ring keeps a stream's barriers at most a phase ahead of who waits for them only if its tiles
    // never follow one another.
    auto first_of = [&](int i, uint32_t before) { return C::CONV ? (int)((i ^ before) & 1) : MODE == SPLIT ? i : 0; };
    auto tiles_of = [&](int i, uint32_t before) {
        return MODE == PAIR ? (w.rows - w.r0 > 128 * i ? w.nt : 0) : (w.nt + 1 - first_of(i, before)) / 2;
    };

    if (warp < 8) {
        // ---- softmax of stream i: thread = row = TMEM lane
        const int i = warp >> 2, row = (warp & 3) * 32 + lane;
        const uint32_t lanes = tmem + ((uint32_t)((warp & 3) * 32) << 16);
        float2 *s_sum = reinterpret_cast<float2 *>(s_join) + (MODE == PAIR ? i * 128 + row : 0);
        const uint32_t s_col = lanes + i * 128, o_col = lanes + C::O_COL + i * D;
        uint32_t ns = 0, nv = 0, before = 0, unit_no = 0;      // phases of s_full, of V; position tiles, units before
        bool ok = true;
        for (; ok && work.next(w); before += w.nt, unit_no++) {
            const int nt = tiles_of(i, before);
            if (MODE == PAIR && nt == 0) continue;
            const int r = w.r0 + (MODE == PAIR ? i * 128 : 0) + row, t = r / a.G;    // this row: its token, position below
            int tok = -1;                                                        // token row * H + head (-1: none)
            int64_t qo = -1;                                                     // where its q is
            if (r < w.rows) {
                const int h = w.kh * a.G + (r - t * a.G);
                tok = (w.t0 + t) * a.H + h;
                qo = (w.t0 + t) * A.ldq + (int64_t)h * D;
            }
            // q: 8 lanes per row, 4 rows at a time: row maximum, power-of-two scale, two fp16 terms, swizzled
            // rows (one tile: stream 0 writes them, stream 1 only wants the scales)
            float f = 0.0f;
            const uint32_t sign = A.scale2 < 0.0f ? 0x80000000u : 0u;  // f >= 0: the largest s f has the largest s
            auto fetch = [&](float4 (&z)[4][D / 32], int g0) {         // 16 rows of the warp
#pragma unroll
                for (int g = 0; g < 4; g++) {
                    const int64_t from = __shfl_sync(kFull, qo, 4 * (g0 + g) + (lane >> 3));
                    const float4 *src = reinterpret_cast<const float4 *>(A.q + from) + (lane & 7);
#pragma unroll
                    for (int k = 0; k < D / 32; k++) z[g][k] = from < 0 ? make_float4(0.0f, 0.0f, 0.0f, 0.0f) : __ldcg(src + 8 * k);
                }
            };
            auto place = [&](float4 (&z)[4][D / 32], int g0) {
#pragma unroll
                for (int g = 0; g < 4; g++) {
                    float mx = 0.0f;
#pragma unroll
                    for (int k = 0; k < D / 32; k++) mx = fmaxf(mx, fmaxf(fmaxf(fabsf(z[g][k].x), fabsf(z[g][k].y)), fmaxf(fabsf(z[g][k].z), fabsf(z[g][k].w))));
                    mx = fmaxf(mx, __shfl_xor_sync(kFull, mx, 1));
                    mx = fmaxf(mx, __shfl_xor_sync(kFull, mx, 2));
                    mx = fmaxf(mx, __shfl_xor_sync(kFull, mx, 4));
                    const uint32_t up = scale_up(__float_as_uint(mx) >> 23);
                    const float got = __shfl_sync(kFull, (MODE == F32 ? 1.0f : fabsf(A.scale2)) * pow2_bits(254u - up), (lane & 3) * 8);
                    if (lane >> 2 == g0 + g) f = got;
                    if (MODE != PAIR && i == 1) continue;
                    const float m = __uint_as_float(up << 23 | sign);
                    const int rr = (warp & 3) * 32 + 4 * (g0 + g) + (lane >> 3);
                    const uint32_t at = sm0 + (MODE == PAIR ? i * 2 * C::QTILE : 0) + rr * 128 + (lane & 1) * 8;
#pragma unroll
                    for (int k = 0; k < D / 32; k++) {
                        const float2 y0 = f2_mul(make_float2(z[g][k].x, z[g][k].y), make_float2(m, m)), y1 = f2_mul(make_float2(z[g][k].z, z[g][k].w), make_float2(m, m));
                        const float2 h0 = make_float2(tf32_hi(y0.x), tf32_hi(y0.y)), h1 = make_float2(tf32_hi(y1.x), tf32_hi(y1.y));
                        const float2 l0 = f2_fma(h0, make_float2(-1.0f, -1.0f), y0), l1 = f2_fma(h1, make_float2(-1.0f, -1.0f), y1);
                        // values 4 (lane & 7) + 32 k .. + 3: 16-byte piece (lane & 7) / 2 + 4 (k & 1) of half k / 2
                        const uint32_t to = at + (k >> 1) * C::QHALF + (((((lane & 7) >> 1) + 4 * (k & 1)) ^ (rr & 7)) << 4);
                        asm volatile("st.shared.v2.b32 [%0], {%1, %2};" ::"r"(to), "r"(pack_h2(h0.x, h0.y)), "r"(pack_h2(h1.x, h1.y)) : "memory");
                        asm volatile("st.shared.v2.b32 [%0], {%1, %2};" ::"r"(to + C::QTILE), "r"(pack_h2(l0.x, l0.y)), "r"(pack_h2(l1.x, l1.y)) : "memory");
                    }
                }
            };
            if constexpr (MODE != F32) {
                float4 x[2][4][D / 32];
                fetch(x[0], 0);
                fetch(x[1], 4);
                place(x[0], 0);
                place(x[1], 4);
            } else {
#pragma unroll 1
                for (int g = 0; g < 8; g += 4) {
                    float4 x[4][D / 32];
                    fetch(x, g);
                    place(x, g);
                }
            }
            f = fmaxf(f, 1.17549435e-38f);        // (0 would make NaN of a masked score, -inf)
            fence_async_smem();
            if (MODE == PAIR || i == 0) mbar_arrive(&q_full[i]);
            int pos = -1;
            if (own) {
                if (r < w.rows) pos = w.kv - w.n + t;
            } else {
                const int t_end = min(a.n_tok - 1, __shfl_sync(kFull, t, 31));
                for (int x = __shfl_sync(kFull, t, 0); x <= t_end; x++) {
                    int s0 = 0, sn = 0, skv = 0;
                    const int sb = paged_seq_of(a, x);
                    if (sb < a.n_seq) paged_seq(a, sb, s0, sn, skv);
                    if (t == x && r < w.rows && x >= s0 && x < s0 + sn) pos = skv - sn + (x - s0);
                }
            }

            const int lim = min(pos, w.k1 - 1);   // last position that this row sees
            uint32_t vup = 0;                     // F32: the scale of V that O is in
            // O times a power of 2 (the MMAs on it ended before the S at hand was announced)
            auto scale_o = [&](float fac) {
#pragma unroll 1
                for (int k = 0; k < D / 32; k++) {
                    uint32_t o[32];
                    tmem_ld<32>(o_col + 32 * k, o);
                    tmem_wait_ld(o);
#pragma unroll
                    for (int e = 0; e < 32; e++) o[e] = __float_as_uint(__uint_as_float(o[e]) * fac);
                    tmem_st32(o_col + 32 * k, o);
                }
            };
            // O adds up the tiles from position kp on, up to tile n1
            int n = 0, n1 = min(nt, C::PIECE), kp = w.kmin;
            if (MODE == PAIR) *s_sum = make_float2(-INFINITY, 0.0f);
            float B = -INFINITY, l = 0.0f, cut = 0.0f;
        next_part:                                // (as a loop around all this, 1 us more per call)
            for (; n < n1; n++) {
                const int j = MODE == PAIR ? n : 2 * n + first_of(i, before), base = w.k0 + j * C::TP;
                if (MODE != PAIR || n == 0 || base > kp) {           // (else waited for already)
                    if (!(ok = __all_sync(kFull, sy.wait(&s_full[i], ns & 1)))) break;       // the whole warp or none of it
                    ns++;
                    tc_fence_after();
                }
                const uint32_t *bad = s_bad + ((before + j) & 7) * 4;
                uint32_t any_bad = bad[0] | bad[1];
                if constexpr (C::TP == 128) any_bad |= bad[2] | bad[3];
                // rows that see nothing of this unit are not read from its slot: no mask for them
                if (__any_sync(kFull, lim >= w.kmin && lim < base + C::TP - 1) || base < w.kmin || any_bad) {
#pragma unroll 1
                    for (int c = 0; c < C::TP / 32; c++) {
                        const int d = lim - base - 32 * c, below = w.kmin - base - 32 * c;
                        const uint32_t vis = (d < 0 ? 0u : d >= 31 ? 0xffffffffu : (2u << d) - 1u) & ~bad[c] &
                                             (below <= 0 ? 0xffffffffu : below >= 32 ? 0u : 0xffffffffu << below);
                        uint32_t x[32];
                        tmem_ld<32>(s_col + 32 * c, x);
                        tmem_wait_ld(x);
#pragma unroll
                        for (int e = 0; e < 32; e++) x[e] = vis >> e & 1 ? x[e] : 0xff800000u;
                        tmem_st32(s_col + 32 * c, x);
                    }
                    tmem_wait_st();
                }
                // scores of 32 positions in z become weights, hi terms in the first 16 columns, lo in the next 16. The
                // base of the weights is a whole number and stays, unless a score lies 2^kWHigh above it: then
                // what was computed with the old one (o; this tile's weights so far) is scaled by a power of 2.
                // (F32: the powers of 2 of q and K first: small q may meet large K)
                const float fk = MODE == F32 ? fmaxf(fabsf(A.scale2) * (f * pow2_bits(254u - s_up[(before + j) & 3])), 1.17549435e-38f) : f;
                const float2 f2 = make_float2(fk, fk);
                float S = 0.0f;                   // the tile's weights
                auto weights = [&](uint32_t (&z)[32], int c, uint32_t done) {
                    float mx = max3(__uint_as_float(z[0]), __uint_as_float(z[1]), __uint_as_float(z[2]));
#pragma unroll
                    for (int e = 3; e < 31; e += 2) mx = max3(mx, __uint_as_float(z[e]), __uint_as_float(z[e + 1]));
                    mx = fmaxf(mx, __uint_as_float(z[31]));
                    mx = mx == -INFINITY ? mx : mx * fk;
                    if (__any_sync(kFull, mx > B + kWHigh)) {
                        const float nb = mx > B + kWHigh ? ceilf(mx) - kWLow : B, fac = B == nb ? 1.0f : B == -INFINITY ? 0.0f : ex2(B - nb);
                        B = nb;
                        S *= fac;
                        l *= fac;
                        cut *= fac;
                        if (n > 0 && (MODE != PAIR || base > kp)) scale_o(fac);
#pragma unroll 1
                        for (int k = 0; k < 4; k++) {
                            if (!(done >> k & 1)) continue;
                            uint32_t o[32];
                            tmem_wait_st();
                            tmem_ld<32>(s_col + 32 * k, o);
                            tmem_wait_ld(o);
#pragma unroll
                            for (int e = 0; e < 16; e++) {           // (in fp32: in fp16 a factor below 2^-24 is 0, and 2^15 times it is not)
                                const float2 h = __half22float2(*reinterpret_cast<const __half2 *>(&o[e]));
                                const float2 lo = __half22float2(*reinterpret_cast<const __half2 *>(&o[16 + e]));
                                const float2 y = f2_mul(f2_add(h, lo), make_float2(fac, fac));
                                split_h2(y.x, y.y, o[e], o[16 + e]);
                            }
                            tmem_st32(s_col + 32 * k, o);
                        }
                    }
                    const float2 nB = B == -INFINITY ? make_float2(0.0f, 0.0f) : make_float2(-B, -B);
                    uint32_t o[32];
                    float2 l2 = make_float2(0.0f, 0.0f);             // (sums of 16: a weight far above the others hides few)
#pragma unroll
                    for (int e = 0; e < 32; e += 2) {
                        const float2 q = f2_fma(make_float2(__uint_as_float(z[e]), __uint_as_float(z[e + 1])), f2, nB);
                        const float2 w2 = make_float2(ex2(q.x), ex2(q.y));
                        l2 = f2_add(l2, w2);
                        split_h2(w2.x, w2.y, o[e / 2], o[16 + e / 2]);
                    }
                    tmem_st32(s_col + 32 * c, o);
                    S += l2.x + l2.y;
                };
                uint32_t x[32], y[32];
                tmem_ld<32>(s_col, x);
                tmem_wait_ld(x);
                tmem_ld<32>(s_col + 32, y);       // the next 32 come while these are worked on
                weights(x, 0, 0);
                tmem_wait_ld(y);
                if constexpr (C::TP == 128) {
                    tmem_ld<32>(s_col + 64, x);
                    weights(y, 1, 1);
                    tmem_wait_ld(x);
                    tmem_ld<32>(s_col + 96, y);
                    weights(x, 2, 3);
                    tmem_wait_ld(y);
                    weights(y, 3, 7);
                } else {
                    weights(y, 1, 1);
                    if (!(ok = __all_sync(kFull, sy.wait(&full[2 + i], nv++ & 1)))) break;     // V's scale is known
                    const uint32_t up = s_up[4 + ((before + j) & 3)];
                    if (up != vup && n > 0) scale_o(vup - up > 126 ? 0.0f : pow2_bits(127u - (vup - up)));
                    vup = up;
                }
                tmem_wait_st();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&p_full[i]);
                const float sum = l + S;          // (and what rounding takes of l itself)
                cut += fminf(C::ADDS * C::CUT * sum, 0.5f * S) - (S - (sum - l));
                l = sum;
            }
            if (!ok) break;
            // O is complete (no tiles at all: not before the last unit is read)
            if (nt > 0) {
                if (!(ok = __all_sync(kFull, sy.wait(&s_full[i], ns & 1)))) break;
                ns++;
                tc_fence_after();
            } else if (!(ok = __all_sync(kFull, sy.wait(&q_full[0], unit_no & 1)))) {
                break;
            }
            if (isnan(l) && B == -INFINITY) B = 0.0f;
            auto alike = [](float x) { return (__float_as_uint(x) & 0xfffu) == 0; };
            float w0 = l > 0.0f && l < INFINITY && (MODE == F32 || !alike(l)) ? 1.0f + fmaxf(__fdividef(cut, l) - C::RISE * C::CUT, 0.0f) : 1.0f, w1 = 0.0f;
            float even0 = 1.0f, even1 = 1.0f;     // F32: what undoes the giving back, for streams whose weights are all alike
            if (MODE == F32 && nt > 0) w0 *= pow2_bits(254u - vup);
            if constexpr (MODE != PAIR) {
                // stream 1 leaves its (B, l, scale); stream 0 reads both O (the same TMEM lanes) and writes the rows
                if (i == 1) {
                    s_join[row] = B;
                    s_join[128 + row] = l;
                    s_join[256 + row] = w0;
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(joined);
                    continue;                     // (its O stays until the next unit's q is written, by stream 0 after this)
                }
                if (!(ok = __all_sync(kFull, sy.wait(joined, unit_no & 1)))) break;
                tc_fence_after();
                const float B1 = s_join[row], l1 = s_join[128 + row], M = fmaxf(B, B1);
                const float c0 = B == -INFINITY ? 0.0f : ex2(B - M), c1 = B1 == -INFINITY ? 0.0f : ex2(B1 - M);
                auto undo = [&](float x, float w) { return alike(x) && x > 0.0f ? __fdividef(__uint_as_float(__float_as_uint(w) & 0x7f800000u), w) : 1.0f; };
                w1 = s_join[256 + row];
                if (MODE == F32) even0 = undo(l, w0), even1 = undo(l1, w1);
                w1 *= c1;
                w0 *= c0;
                l = c0 * l + c1 * l1;
                B = M;
            }
            const bool put = tok >= 0 && lim >= w.kmin, none = l == 0.0f, fix = *s_flag != 0;
            const int64_t first = (int64_t)w.slot * a.n_tok * a.H;
            const int row_out = put ? tok : -1;
            float *part = A.part_o + first * D + (lane & 7) * 4;
            // PAIR: the unit's earlier sums are in the slot, with their base and l in *s_sum: this one joins them in that base, or,
            // where it is far above (and for the first), takes their place, but for what is not finite: no weight makes that nothing
            bool over = true;
            if (MODE == PAIR && put) {
                const float2 sum = *s_sum;
                over = !(B - sum.x <= 40.0f);
                const float f = over || none ? 1.0f : ex2(B - sum.x);
                *s_sum = over ? make_float2(B, l + (sum.y == 0.0f ? 0.0f : sum.y * ex2(sum.x - B))) : make_float2(sum.x, fmaf(l, f, sum.y));
                w0 *= f;
            }
            uint32_t fresh = __ballot_sync(kFull, over);
            if (MODE == PAIR && kp > w.kmin) {    // of earlier sums that lose their place 0 is left, or NaN; the new ones are added to that
                uint32_t later = __ballot_sync(kFull, over && put);
                for (fresh &= ~later; later; later &= later - 1) {
                    float *to = A.part_o + (first + __shfl_sync(kFull, tok, __ffs(later) - 1)) * D + lane;
#pragma unroll
                    for (int d = 0; d < D; d += 32) to[d] = __ldcg(to + d) * 0.0f;
                }
                __syncwarp();
            }
            const bool any_even = MODE == F32 && __any_sync(kFull, even0 != 1.0f || even1 != 1.0f);
            auto uncut = [](uint32_t (&o)[32], float f) {     // o's sums of few bits
#pragma unroll
                for (int e = 0; e < 32; e++)
                    if ((o[e] & 0xffu) == 0) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
            };
            // (the O of a stream without tiles may be anything: the other's, 0 times)
            const uint32_t o0_col = nt > 0 ? o_col : o_col + D, o1_col = tiles_of(1, before) > 0 ? o_col + D : o_col;
            // the rows leave by way of shared memory (where this warp's rows of Q are), 128 bytes of a row per 8 lanes; while Q is
            // still wanted, by shuffles
            unsigned char *stage = sm + (MODE == PAIR ? i * 2 * C::QTILE : 0) + (warp & 3) * 4096;
#pragma unroll 1
            for (int c = 0; c < D / 32; c++) {
                uint32_t o[32];
                tmem_ld<32>(o0_col + 32 * c, o);
                tmem_wait_ld(o);
                if (any_even) uncut(o, even0);
#pragma unroll
                for (int e = 0; e < 32; e++) o[e] = __float_as_uint(__uint_as_float(o[e]) * w0);
                if constexpr (MODE != PAIR) {
                    uint32_t o1[32];
                    tmem_ld<32>(o1_col + 32 * c, o1);
                    tmem_wait_ld(o1);
                    if (any_even) uncut(o1, even1);
#pragma unroll
                    for (int e = 0; e < 32; e++) o[e] = __float_as_uint(fmaf(__uint_as_float(o1[e]), w1, __uint_as_float(o[e])));
                }
                if (fix && put) {
                    // V that were set aside: added where the row sees them (inf and NaN are not changed by a weight)
                    typedef typename std::conditional<MODE == F32, float, __half>::type KT;
                    const int past = MODE == PAIR ? min(lim + 1, w.k0 + n1 * C::TP) : lim + 1;
                    for (int p = kp; p < past; p++) {
                        const int64_t at = paged_at(a, a.table + (own ? (int64_t)w.b * a.table_stride : 0), p);
                        if (at < 0) continue;
                        const char *vr = a.v + at + w.kh * a.head_stride;
#pragma unroll
                        for (int e = 0; e < 32; e++) {
                            float v;
                            if constexpr (MODE == NIB) v = q4_ld<D>(vr, q4_scales<D>(a, p & ((1 << a.page_log) - 1)), 32 * c + e);
                            else v = kv_ld(reinterpret_cast<const KT *>(vr) + 32 * c + e);
                            if (!isfinite(v)) o[e] = __float_as_uint(__uint_as_float(o[e]) + v);
                        }
                    }
                }
                if (none)
#pragma unroll
                    for (int e = 0; e < 32; e++) o[e] = 0;
                if (MODE == PAIR && n < nt) {
                    transpose8(o, lane);
#pragma unroll
                    for (int k = 0; k < 8; k++) {
                        const int rr = (lane & 24) + k, to = __shfl_sync(kFull, row_out, rr);
                        float *dst = part + (int64_t)to * D + 32 * c;
                        if (to >= 0 && (fresh >> rr & 1)) *reinterpret_cast<uint4 *>(dst) = make_uint4(o[4 * k], o[4 * k + 1], o[4 * k + 2], o[4 * k + 3]);
                        else if (to >= 0) red4(dst, o + 4 * k);
                    }
                    continue;
                }
                __syncwarp();
#pragma unroll
                for (int e = 0; e < 32; e += 4)   // 16-byte piece e / 4 of row `lane`, XOR-placed against bank conflicts
                    *reinterpret_cast<uint4 *>(stage + lane * 128 + (((e >> 2) ^ (lane & 7)) << 4)) =
                        make_uint4(o[e], o[e + 1], o[e + 2], o[e + 3]);
                __syncwarp();
#pragma unroll
                for (int k = 0; k < 8; k++) {     // 4 rows of 128 bytes at a time
                    const int rr = 4 * k + (lane >> 3), to = __shfl_sync(kFull, row_out, rr);
                    const uint4 v = *reinterpret_cast<const uint4 *>(stage + rr * 128 + (((lane & 7) ^ (rr & 7)) << 4));
                    float *dst = part + (int64_t)to * D + 32 * c;
                    if (to >= 0 && (MODE != PAIR || (fresh >> rr & 1))) *reinterpret_cast<uint4 *>(dst) = v;
                    else if (MODE == PAIR && to >= 0) red4(dst, reinterpret_cast<const uint32_t *>(&v));
                }
            }
            if constexpr (MODE == PAIR) {
                __syncwarp();                     // (other lanes may add to a row later)
                if (put && n == nt) A.part_ml[first + tok] = make_float2(s_sum->y == 0.0f ? -INFINITY : s_sum->x, s_sum->y);
            } else if (put) {
                A.part_ml[first + tok] = make_float2(none ? -INFINITY : B, l);
            }
            tc_fence_before();
            if (MODE == PAIR && n < nt) {
                kp = w.k0 + n * C::TP;
                n1 = min(nt, n + C::PIECE);
                B = -INFINITY;
                l = cut = 0.0f;
                goto next_part;
            }
        }
        tmem_wait_st();
    } else if (warp == C::TMA_WARP || (!C::CONV && warp == 9)) {
        // ---- K and V, in the order of their use: K, V of each position tile, or (SPLIT) K, K, V, V of two. One warp
        // issues them; V tiles with rows that not every row sees (or that were not loaded) land on a barrier of their
        // own and are passed on by the other (F32: all go to the stages, and the converting warps look at them).
        uint32_t c[2] = {0, 0}, t = 0, phases = 0;       // loads so far (SPLIT: of each stream); tiles; of `landed`
        bool ok = true;
        const int R = min(1 << a.page_log, C::TP), boxes = C::TP / R;          // positions per box, boxes per half of a row
        constexpr int STEP = MODE == SPLIT ? 2 : 1, PER = MODE == F32 ? 2 : 1;  // boxes per lane (F32: pages of any size)
        while (ok && work.next(w)) {
            const int *table = a.table + (own ? (int64_t)w.b * a.table_stride : 0);
            for (int j0 = 0; ok && j0 < w.nt; j0 += STEP) {
                const int m = min(STEP, w.nt - j0);
                for (int k = 0; ok && k < 2 * m; k++) {
                    const bool is_v = k >= m;
                    const int jj = is_v ? k - m : k, base = w.k0 + (j0 + jj) * C::TP;
                    const uint32_t n = MODE == SPLIT && jj ? c[1]++ : c[0]++, slot = C::slot(jj, n);
                    // lane x: page of box x (positions base + x R ..), and x + 32; boxes past the unit are not loaded
                    int page[PER];
                    uint32_t have = 0, missing[PER];
#pragma unroll
                    for (int h = 0; h < PER; h++) {
                        const int i = lane + 32 * h, p = base + i * R;
                        const bool want = i < boxes && p < w.k1;
                        page[h] = want ? table[p >> a.page_log] : -1;
                        const bool good = want && (unsigned)page[h] < (unsigned)a.n_pages;
                        if (!good) page[h] = -1;
                        if (want && !good && warp == C::TMA_WARP) paged_err(a, QMS_PAGED_EPAGE);
                        have += __popc(__ballot_sync(kFull, good));
                        missing[h] = __ballot_sync(kFull, want && !good);
                    }
                    uint32_t any_missing = missing[0];
                    if constexpr (PER > 1) any_missing |= missing[PER - 1];
                    const int seen = min(w.lo, w.k1 - 1);
                    const bool scan = !C::CONV && is_v && (base + C::TP - 1 > seen || base < w.kmin || any_missing);
                    if (warp == C::TMA_WARP) {
                        if (!is_v && lane < C::TP / 32) {     // bits of the tile's positions on bad pages
                            uint32_t bits = 0;
                            if (any_missing)
                                for (int e = 0; e < 32; e++) {
                                    const int i = (lane * 32 + e) / R;
                                    bits |= ((PER > 1 && i >= 32 ? missing[PER - 1] : missing[0]) >> (i & 31) & 1u) << e;
                                }
                            s_bad[((t + jj) & 7) * 4 + lane] = bits;
                        }
                        __syncwarp();
                        uint64_t *bar;
                        if constexpr (C::CONV) {
                            if (n >= 2) ok = __all_sync(kFull, sy.wait(&landed[2 + (n & 1)], (n / 2 - 1) & 1));
                            bar = &landed[n & 1];
                        } else {
                            if (n >= C::RINGLEN) ok = __all_sync(kFull, sy.wait(&empty[slot], C::phase(n) ^ 1));
                            bar = scan ? &landed[slot] : &full[slot];
                        }
                        if (!ok) break;
                        if (lane == 0) mbar_arrive_expect_tx(bar, have * (uint32_t)(R * (MODE == NIB ? q4_row(D) : D * (MODE == F32 ? 4 : 2))));
                        __syncwarp();
#pragma unroll
                        for (int h = 0; h < PER; h++) {
                            const int i = lane + 32 * h, y = (base + i * R) & ((1 << a.page_log) - 1);
                            if (page[h] < 0) continue;
                            if constexpr (MODE == NIB) {
                                const char *src = (is_v ? a.v : a.k) + page[h] * a.page_stride + w.kh * a.head_stride;
                                const uint32_t to = sm0 + C::STAGE + (n & 1) * C::STAGED;
                                bulk_load(to + i * R * (D / 2), src + y * (D / 2), R * (D / 2), bar);
                                bulk_load(to + C::TP * (D / 2) + i * R * (D / 16), src + (D / 2 << a.page_log) + y * (D / 16), R * (D / 16), bar);
                            } else if constexpr (MODE == F32)
                                tma_load4(sm0 + C::STAGE + (n & 1) * C::STAGED + i * R * (D * 4), is_v ? &mv : &mk, 0, w.kh, y, page[h], bar);
                            else
#pragma unroll
                                for (int x = 0; x < C::HALVES; x++)
                                    tma_load4(sm0 + C::RING + slot * C::SLOT + x * C::HALF + i * R * 128, is_v ? &mv : &mk, x * 64, w.kh, y, page[h], bar);
                        }
                    } else if (scan) {
                        ok = __all_sync(kFull, sy.wait(&landed[slot], phases >> slot & 1));
                        phases ^= 1u << slot;
                        for (int x = lane; ok && x < C::TP * (D / 8); x += 32) {
                            const int r = x / (D / 8), piece = x % (D / 8), p = base + r;
                            if (p >= w.kmin && p <= seen && !any_missing) continue;
                            uint4 *pv = reinterpret_cast<uint4 *>(sm + C::RING + slot * C::SLOT + (piece >> 3) * C::HALF + r * 128 +
                                                                  (((piece & 7) ^ (r & 7)) << 4));
                            uint4 v = *pv;
                            if (drop_nonfinite((const __half *)nullptr, v)) {
                                *pv = v;
                                if (p >= w.kmin && p < w.k1) *s_flag = 1;      // (else left over: nobody's)
                            }
                        }
                        fence_async_smem();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(&full[slot]);
                    }
                }
                t += m;
            }
        }
    } else if (MODE == NIB && warp < 12) {
        // ---- nibbles from the stages to fp16 tiles, 32 values with one scale at a time: what the unit holds, V that is not finite
        // where some row does not see it set aside. A group's pieces go out in an order that lets 8 lanes write to all banks.
        constexpr int GR = D / 32, N = C::TP * GR / 128;
        const int ct = tid - 256;
        uint32_t c = 0, t = 0;                    // loads, tiles so far
        bool ok = true;
        while (work.next(w)) {                    // (after a failed wait: the barriers, no work)
            const int seen0 = min(w.lo, w.k1 - 1);
            for (int j = 0; j < w.nt; j++, t++)
#pragma unroll 1
                for (int is_v = 0; is_v < 2; is_v++, c++) {
                    const int base = w.k0 + j * C::TP;
                    const unsigned char *src = sm + C::STAGE + (c & 1) * C::STAGED;
                    ok = __all_sync(kFull, ok && sy.wait(&landed[c & 1], c / 2 & 1));
                    const uint32_t *bad = s_bad + (t & 7) * 4;
                    const int seen = bad[0] | bad[1] | bad[2] | bad[3] ? -1 : seen0;
                    const bool look = base + C::TP - 1 > seen || base < w.kmin;
                    ok = __all_sync(kFull, ok && (c < 3 || sy.wait(&empty[c % 3], (c / 3 - 1) & 1)));
                    if (ok) {
                        unsigned char *dst = sm + C::RING + c % 3 * C::SLOT;
#pragma unroll 1
                        for (int i = 0; i < N; i++) {          // (in line four times, the warps waited for instructions)
                            const int at = ct + 128 * i, r = at / GR, g = at % GR, turn = g & 2;
                            uint4 x = *reinterpret_cast<const uint4 *>(src + at * 16);
                            const __half2 d = __half2half2(reinterpret_cast<const __half *>(src + C::TP * (D / 2))[at]), m24 = __hmul2(d, __float2half2_rn(-24.0f));
                            if (turn) x = make_uint4(x.z, x.w, x.x, x.y);
                            const uint32_t xx[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
                            for (int k = 0; k < 4; k++) {
                                const int q = 4 * g + (k ^ turn);
                                *reinterpret_cast<uint4 *>(dst + (q >> 3) * C::HALF + r * 128 + (((q & 7) ^ (r & 7)) << 4)) = q4_dequant(xx[k], d, m24);
                            }
                        }
                        if (look)                              // what this thread wrote, again
#pragma unroll 1
                            for (int i = 0; i < 4 * N; i++) {
                                const int at = ct + 128 * (i >> 2), r = at / GR, q = at % GR * 4 + (i & 3), p = base + r;
                                const bool in = p >= w.kmin && p < w.k1 && !(bad[r >> 5] >> (r & 31) & 1);
                                uint4 *py = reinterpret_cast<uint4 *>(dst + (q >> 3) * C::HALF + r * 128 + (((q & 7) ^ (r & 7)) << 4));
                                uint4 y = in ? *py : make_uint4(0, 0, 0, 0);
                                if (in && is_v && p > seen && drop_nonfinite((const __half *)nullptr, y)) *s_flag = 1;
                                *py = y;
                            }
                    }
                    fence_async_smem();
                    mbar_arrive(&full[2 * is_v + (t & 1)]);
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&landed[2 + (c & 1)]);
                }
        }
    } else if (MODE == F32 && warp < 12) {
        // ---- fp32 rows from the stages into hi and lo tiles, under one scale: K under the tile's, V under the largest so
        // far, of what somebody sees. A 16-byte piece of a row per lane at a time.
        constexpr int CH = D / 4, N = C::TP * CH / 128;
        const int ct = tid - 256, cw = warp - 8;
        uint32_t c = 0, t = 0;                    // loads, tiles so far
        bool ok = true;
        while (work.next(w)) {                    // (after a failed wait: the barriers, no work)
            uint32_t v_exp = 0;
            const int seen0 = min(w.lo, w.k1 - 1);
            for (int j = 0; j < w.nt; j++, t++)
#pragma unroll 1
                for (int is_v = 0; is_v < 2; is_v++, c++) {
                    const int base = w.k0 + j * C::TP;
                    const float4 *src = reinterpret_cast<const float4 *>(sm + C::STAGE + (c & 1) * C::STAGED) + ct;
                    ok = __all_sync(kFull, ok && sy.wait(&landed[c & 1], c / 2 & 1));
                    const uint32_t bad[2] = {s_bad[(t & 7) * 4], s_bad[(t & 7) * 4 + 1]};
                    const int seen = bad[0] | bad[1] ? -1 : seen0;
                    float4 x[N];
#pragma unroll
                    for (int i = 0; i < N; i++) x[i] = src[128 * i];
                    if (base + C::TP - 1 > seen || base < w.kmin)
#pragma unroll
                        for (int i = 0; i < N; i++) {
                            const int r = (ct + 128 * i) / CH, p = base + r;
                            if (p >= w.kmin && p <= seen) continue;
                            const bool in = p >= w.kmin && p < w.k1 && !(bad[r >> 5] >> (r & 31) & 1);
                            if (is_v) {
                                uint4 v = *reinterpret_cast<const uint4 *>(&x[i]);
                                if (drop_nonfinite((const float *)nullptr, v)) {
                                    x[i] = *reinterpret_cast<const float4 *>(&v);
                                    if (in) *s_flag = 1;
                                }
                            }
                            if (!in) x[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);   // no part of the unit
                        }
                    // largest finite |value|: by float maxima, looked at again where it is inf (NaN is no maximum)
                    float m[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                    for (int i = 0; i < N; i++) m[i & 3] = max3(m[i & 3], max3(fabsf(x[i].x), fabsf(x[i].y), fabsf(x[i].z)), fabsf(x[i].w));
                    uint32_t mb = __float_as_uint(fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3])));
                    if (mb == 0x7f800000u) {
                        mb = 0;
#pragma unroll
                        for (int i = 0; i < N; i++) mb = max(mb, max(max(finite_bits(x[i].x), finite_bits(x[i].y)), max(finite_bits(x[i].z), finite_bits(x[i].w))));
                    }
                    mb = __reduce_max_sync(kFull, mb);
                    uint32_t *s_m = s_max + (c & 1) * 4;
                    if (lane == 0) s_m[cw] = mb;
                    asm volatile("bar.sync 1, 128;" ::: "memory");
                    uint32_t exp = max(max(s_m[0], s_m[1]), max(s_m[2], s_m[3])) >> 23;
                    if (is_v) exp = v_exp = max(v_exp, exp);
                    const uint32_t up = scale_up(exp);
                    if (ct == 0) s_up[4 * is_v + (t & 3)] = up;
                    ok = __all_sync(kFull, ok && (c < 3 || sy.wait(&empty[c % 3], (c / 3 - 1) & 1)));
                    if (ok) {
                        const float2 u2 = make_float2(pow2_bits(up), pow2_bits(up));
                        unsigned char *dst = sm + C::RING + c % 3 * C::SLOT;
#pragma unroll
                        for (int i = 0; i < N; i++) {
                            const int r = (ct + 128 * i) / CH, q = ct % CH;   // values 4 q .. + 3 of row r
                            const float2 y0 = f2_mul(make_float2(x[i].x, x[i].y), u2), y1 = f2_mul(make_float2(x[i].z, x[i].w), u2);
                            uint32_t h0, h1, l0, l1;
                            split_h2(y0.x, y0.y, h0, l0);
                            split_h2(y1.x, y1.y, h1, l1);
                            unsigned char *to = dst + (q >> 4) * C::HALF + r * 128 + ((((q & 15) >> 1) ^ (r & 7)) << 4) + (q & 1) * 8;
                            *reinterpret_cast<uint2 *>(to) = make_uint2(h0, h1);
                            *reinterpret_cast<uint2 *>(to + C::TILE) = make_uint2(l0, l1);
                        }
                    }
                    fence_async_smem();
                    mbar_arrive(&full[2 * is_v + (t & 1)]);
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&landed[2 + (c & 1)]);
                }
        }
    } else {
        // ---- the MMAs of stream i, by one thread
        const int i = warp - C::MMA_WARP;
        if (lane == 0 && i < 2) {
            constexpr uint32_t id_s = idesc_f16(C::TP, false), id_o = idesc_f16(D, true);
            constexpr int TERMS = MODE == F32 ? 3 : 2;          // hi hi, lo hi, (fp32) hi lo
            uint32_t c = 0, nf = 0, nq = 0, np = 0;             // loads of the ring so far; phases of (CONV) full, of q_full, p_full
            bool ok = true;
            auto score = [&](uint32_t n) {                     // S_i = Q_i K^T
                const uint32_t k = sm0 + C::RING + C::slot(i, n) * C::SLOT, q = sm0 + (MODE == PAIR ? i * 2 * C::QTILE : 0);
#pragma unroll
                for (int x = 0; x < TERMS; x++)                 // (the large one last)
#pragma unroll
                    for (int ks = 0, term = TERMS - 1 - x; ks < D / 16; ks++)
                        umma_f16_ss(tmem + i * 128, desc_sw128(q + (term == 1) * C::QTILE + (ks >> 2) * C::QHALF + (ks & 3) * 32, 16, 1024),
                                    desc_sw128(k + (term == 2) * C::TILE + (ks >> 2) * C::HALF + (ks & 3) * 32, 16, 1024), id_s, x || ks);
            };
            auto weigh = [&](uint32_t n, bool first) {         // O_i (+)= P_i V
                const uint32_t v = sm0 + C::RING + C::slot(i, n) * C::SLOT;
#pragma unroll
                for (int term = 0; term < TERMS; term++)
#pragma unroll
                    for (int ks = 0; ks < C::TP / 16; ks++)
                        umma_f16_ts(tmem + C::O_COL + i * D, tmem + i * 128 + (ks >> 1) * 32 + (term == 1) * 16 + (ks & 1) * 8,
                                    desc_sw128(v + (term == 2) * C::TILE + ks * 2048, C::HALF, 1024), id_o, !first || term || ks);
            };
            auto lock = [&]() {
                uint32_t x = 0;
                do {                                            // (reading costs less than trying)
                    while (*(volatile int *)s_lock != 0 && ++x < kWSpin) {}
                } while (atomicCAS(s_lock, 0, 1) != 0 && x < kWSpin);
            };
            auto unlock = [&]() { *(volatile int *)s_lock = 0; };
            // K, V of this stream's tile at load n (K) or n + 1 of the ring; nf: tiles of the stream so far
            auto k_bar = [&](uint32_t n) { return C::CONV ? &full[i] : &full[C::slot(i, n)]; };
            auto v_bar = [&](uint32_t n) { return C::CONV ? &full[2 + i] : &full[C::slot(i, n)]; };
            constexpr uint32_t NEXT = C::CONV ? 4 : 2;      // loads to the stream's next tile
            while (ok && work.next(w)) {
                const int nt = tiles_of(i, c / 2);
                const uint32_t c1 = c + (MODE == SPLIT ? 2 * nt : 2 * w.nt);
                if (C::CONV) c += 2 * first_of(i, c / 2);
                if (MODE != PAIR || nt > 0) {
                    ok = sy.wait(&q_full[MODE == PAIR ? i : 0], nq++ & 1);
                    if (ok && nt > 0 && (ok = sy.wait(k_bar(c), C::CONV ? nf & 1 : C::phase(c)))) {
                        tc_fence_after();
                        lock();
                        score(c);
                        unlock();
                        umma_commit(&s_full[i]);
                        umma_commit(&empty[C::slot(i, c)]);
                    }
                    for (int j = 0; ok && j < nt; j++, c += NEXT, nf++) {
                        const bool more = j + 1 < nt;
                        if (!(ok = sy.wait(v_bar(c + 1), C::CONV ? nf & 1 : C::phase(c + 1)) && sy.wait(&p_full[i], np++ & 1))) break;
                        tc_fence_after();
                        lock();
                        weigh(c + 1, MODE == PAIR ? j % C::PIECE == 0 : j == 0);
                        if (more) {
                            const uint32_t ph = C::CONV ? (nf + 1) & 1 : C::phase(c + NEXT);
                            if (!mbar_test_wait(k_bar(c + NEXT), ph)) {      // K is late: not at the other's cost
                                unlock();
                                umma_commit(&empty[C::slot(i, c + 1)]);
                                if (!(ok = sy.wait(k_bar(c + NEXT), ph))) break;
                                lock();
                                score(c + NEXT);
                                unlock();
                                umma_commit(&s_full[i]);
                                umma_commit(&empty[C::slot(i, c + NEXT)]);
                                continue;
                            }
                            score(c + NEXT);
                        }
                        unlock();
                        umma_commit(&s_full[i]);
                        umma_commit(&empty[C::slot(i, c + 1)]);
                        if (more) umma_commit(&empty[C::slot(i, c + NEXT)]);
                    }
                } else {                                        // one row tile: the other stream's loads are read once
                    for (uint32_t x = c; ok && x < c1; x++)
                        if ((ok = sy.wait(&full[C::slot(i, x)], C::phase(x)))) mbar_arrive(&empty[C::slot(i, x)]);
                }
                c = c1;
            }
            if (!ok) *s_abort = 1;
            umma_commit(drain);                                 // nothing of this CTA's is in flight when TMEM goes
            for (uint32_t n = 0; n < kWSpin && !mbar_try_wait(drain, 0); n++) __nanosleep(32);
        }
        __syncwarp();
    }
    tc_fence_before();
    __syncthreads();
    if (*s_abort)                                 // copies in flight have 0.1 s to land before the CTA's memory goes
        for (int n = 0; n < 1 << 20; n++) __nanosleep(100);
    if (warp == C::MMA_WARP) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
    }
    if (last) pdl_wait();
}

template <int D, int MODE>
static int launch_wide(const PagedAttn &A, bool own, bool last, cudaStream_t s) {
    using C = WideCfg<D, MODE>;
    static_assert(C::SMEM <= 232448, "shared memory per CTA");
    const int64_t units = own ? (int64_t)A.p.chunks_s * A.a.n_seq * A.p.tiles_s * A.a.Hk : (int64_t)(A.p.line_runs / A.p.line_per);
    QMS_REQUIRE(units < (1ll << 30), QMS_CUDA_EUNSUPPORTED, "paged_attention: too many units of work");
    static std::atomic<unsigned long long> done{0};
    int rc = allow_smem(done, k_paged_wide<D, MODE>, C::SMEM);
    if (rc) return rc;
    CUtensorMap mk, mv;
    if constexpr (MODE == NIB) {
        memset(&mk, 0, sizeof mk);                // (its copies need none)
        mv = mk;
    } else {
        rc = paged_map(A.a, D, MODE != F32, C::TP, A.a.k, &mk);
        if (rc || (rc = paged_map(A.a, D, MODE != F32, C::TP, A.a.v, &mv))) return rc;
    }
    const int grid = (int)(units < 148 ? units : 148);
    QMS_CK(launch_pdl(k_paged_wide<D, MODE>, dim3(grid), dim3(C::THREADS), C::SMEM, s, A, mk, mv, own, last));
    return QMS_CUDA_OK;
}

int launch_paged_wide(const PagedAttn &A, int D, bool own, bool last, cudaStream_t s) {
    const int kind = own ? A.p.wr_s : A.p.wr_p;
    if (kind == kPaWideQ4) return D == 128 ? launch_wide<128, NIB>(A, own, last, s) : launch_wide<64, NIB>(A, own, last, s);
    if (D == 128)
        return kind == kPaWidePair ? launch_wide<128, PAIR>(A, own, last, s) : kind == kPaWideSplit ? launch_wide<128, SPLIT>(A, own, last, s)
                                                                                                  : launch_wide<128, F32>(A, own, last, s);
    return kind == kPaWidePair ? launch_wide<64, PAIR>(A, own, last, s) : kind == kPaWideSplit ? launch_wide<64, SPLIT>(A, own, last, s)
                                                                                             : launch_wide<64, F32>(A, own, last, s);
}

}  // namespace qms
