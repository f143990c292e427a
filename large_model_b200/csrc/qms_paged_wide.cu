// qms_paged_wide.cu - paged attention where one K / V tile meets many rows (a shared prompt against a batch, drafted
// tokens, a chunk of a prompt): tcgen05 tensor cores, fp16 cache, on B200 (sm_100a).
//
// A unit is a run of positions, 128 at a time, of one kv head against 256 rows (two tiles of 128: PAIR) or, where there
// are no more than 128 rows, against one tile whose even and odd position tiles are two streams with an O and
// a softmax of their own (SPLIT): either way the tensor cores have one stream to work on while the other's
// softmax runs.
//   S = Q K^T   tcgen05.mma kind::f16 from shared memory, M 128 x N 128, K = head_dim, twice: Q = hi + lo
//               in fp16 (22 bits, each row scaled by a power of two into fp16's range), K exact
//   softmax     one thread per row reads its S from TMEM, keeps the running base B and sum l, writes the
//               weights 2^(s f - B) back over S as two fp16 terms
//   O += P V    tcgen05.mma with P from TMEM (hi, then lo) and V as it lies in shared memory (MN-major)
// O stays in TMEM over the whole unit. A base is set 2^8 below a maximum and stays until a score lies 2^15 above it
// (fp16 holds weights to 2^16), so that the maximum needs no pass of its own; the result does not depend on
// it beyond rounding.
//
// Warps 0-3 and 4-7 are the softmax of the two streams, warp 8 brings K and V in by TMA (a box of 64 values x up to 128
// positions per page, swizzled), warp 9 clears values that are not finite out of V rows that some row does
// not see (a weight of 0 does not cancel them), one thread each of warps 10 and 11 issues the MMAs of a stream, 16 or
// 32 at a time under a lock: one thread for both leaves the tensor cores idle while it waits and commits (some
// 1200 of 6150 cycles per pair of tiles: hardly one MMA is queued), two that interleave slow every MMA down. Tiles start on a
// page boundary (or, in larger pages, a multiple of 128), so a tile may begin before the first position of its
// unit; such rows are masked. Shared memory at head_dim 128: Q 128 KB and a ring of 3 tiles of 32 KB, or (SPLIT) Q 64 KB and a
// ring of 2 for each stream; TMEM: S 2 x 128, O 2 x 128 columns.
// Bound by the tensor cores: 4 * 128 * 128 * head_dim flop per tile and product pair, twice for the split.
#include <math.h>
#include <string.h>

#include "qms_moe.cuh"
#include "qms_paged.cuh"
#include "qms_tcgen05.cuh"

namespace qms {

constexpr int kWTile = 128, kWThreads = 384;         // 12 warps: 168 registers each
constexpr uint32_t kWSpin = 1u << 22;
constexpr float kWLow = 8.0f, kWHigh = 15.0f;       // a new base is 2^8 below the maximum; weights stay below 2^15

template <int D, bool SPLIT>
struct WideCfg {
    static constexpr int HALVES = D / 64;                       // 64 values = 128 bytes: one swizzle row
    static constexpr uint32_t HALF = kWTile * 128;              // bytes of 128 rows x 64 values
    static constexpr uint32_t TILE = HALVES * HALF;             // a K or V tile; one term of a Q tile
    static constexpr int SLOTS = SPLIT ? 4 : 3, CH = D / 8;     // CH: 16-byte pieces per row
    static constexpr uint32_t RING = (SPLIT ? 2 : 4) * TILE, META = RING + SLOTS * TILE;
    // meta: bad-page masks [8][4], barriers, flags
    static constexpr uint32_t BAD = META, BARS = BAD + 128, SMEM = BARS + (3 * SLOTS + 9) * 8 + 32;
    static constexpr uint32_t O_COL = 256;                      // TMEM columns: S0, S1, O0, O1
    // load n of a ring: its slot and the parity of that slot's phase. (A ring per stream in SPLIT: whoever waits
    // for a slot waits for each of its phases.)
    static constexpr uint32_t RINGLEN = SPLIT ? 2 : 3;
    static __device__ __forceinline__ uint32_t slot(int stream, uint32_t n) { return SPLIT ? 2 * stream + (n & 1) : n % 3; }
    static __device__ __forceinline__ uint32_t phase(uint32_t n) { return n / RINGLEN & 1; }
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

__device__ __forceinline__ void tmem_tie(uint32_t (&r)[32]) {      // the same for a second array of that wait
    asm volatile("" : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]),
                   "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]), "+r"(r[16]), "+r"(r[17]), "+r"(r[18]),
                   "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]),
                   "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31]));
}

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

// One unit of work, as every role derives it.
struct WideUnit {
    int kh, b, t0, n, kv, slot, k0, k1, kmin, r0, rows, nt, tiles, lo;
    // kv head; sequence, its first row, rows and length (own); slot of the partial result; positions [k0, k1) in
    // nt tiles, of which those below kmin belong to another unit; first row and number of rows of the
    // segment; row tiles (1 or 2); every row of the unit sees the positions up to lo
};

// The units of this CTA in order. Own positions: units blockIdx.x, + gridDim.x, ... of (chunk, sequence, row tile, kv
// head). Shared positions against pairs of row tiles: all (row tile, kv head, position tile) triples in one line, cut
// into equal runs, one per CTA; a run is one unit per row tile and kv head that it crosses.
struct WideWork {
    const PagedAttn &A;
    const bool own, line;
    const int lo_p;
    unsigned x, end;
    __device__ WideWork(const PagedAttn &A_, bool own_, int lo_p_) : A(A_), own(own_), line(!own_ && A_.p.line > 0), lo_p(lo_p_) {
        if (line) {
            x = line_start(blockIdx.x, A.p.line, gridDim.x);
            end = line_start(blockIdx.x + 1, A.p.line, gridDim.x);
        } else {
            x = blockIdx.x;
            end = (unsigned)(own ? A.p.chunks_s * A.a.n_seq * A.p.tiles_s : A.p.chunks_p * A.p.tiles_p) * A.a.Hk;
        }
    }
    __device__ bool next(WideUnit &w) {
        const Paged &a = A.a;
        const unsigned rows_tile = (own ? A.p.wr_s : A.p.wr_p) == kPaWideSplit ? kWTile : 2 * kWTile;
        for (; x < end;) {
            w.b = w.t0 = w.n = w.kv = 0;
            if (line) {
                const unsigned nt = (a.prefix + kWTile - 1) / kWTile, u = x / nt, j = x - u * nt, c = min(nt - j, end - x);
                const unsigned tile = u / a.Hk;
                w.kh = u - tile * a.Hk;
                w.r0 = tile * rows_tile;
                w.slot = blockIdx.x - line_run(u * nt, A.p.line, gridDim.x);
                w.k0 = w.kmin = j * kWTile;
                w.k1 = min(a.prefix, (int)(j + c) * kWTile);
                x += c;
            } else {
                unsigned u = x;
                x += gridDim.x;
                unsigned d = u / a.Hk;
                w.kh = u - d * a.Hk;
                u = d;
                const unsigned nr = own ? A.p.tiles_s : A.p.tiles_p;
                d = u / nr;
                w.r0 = (u - d * nr) * rows_tile;
                u = d;
                if (own) {
                    d = u / a.n_seq;
                    w.b = u - d * a.n_seq;
                    u = d;
                    paged_seq(a, w.b, w.t0, w.n, w.kv);
                    w.k0 = A.p.base_s + u * A.p.chunk_s;
                    w.kmin = max(w.k0, a.prefix);
                    w.k1 = min(w.kv, w.k0 + A.p.chunk_s);
                    w.k1 = min(w.k1, w.kv - w.n + min(w.n - 1, (int)(w.r0 + rows_tile - 1) / a.G) + 1);     // nobody sees the rest
                } else {
                    w.k0 = w.kmin = u * A.p.chunk_p;
                    w.k1 = min(a.prefix, w.k0 + A.p.chunk_p);
                }
                w.slot = (own ? A.p.slots_p : 0) + u * (rows_tile == kWTile ? 2 : 1);
            }
            w.rows = own ? w.n * a.G : a.n_tok * a.G;
            w.lo = own ? w.kv - w.n + w.r0 / a.G : lo_p;
            w.nt = (w.k1 - w.k0 + kWTile - 1) / kWTile;
            w.tiles = w.rows - w.r0 > kWTile ? 2 : 1;
            if (w.r0 < w.rows && w.kmin < w.k1) return true;
        }
        return false;
    }
};

template <int D, bool SPLIT>
__global__ void __maxnreg__(168) k_paged_wide(const PagedAttn A, const __grid_constant__ CUtensorMap mk, const __grid_constant__ CUtensorMap mv,
                                             const bool own, const bool last) {
    using C = WideCfg<D, SPLIT>;
    extern __shared__ __align__(1024) unsigned char sm[];
    const Paged &a = A.a;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const uint32_t sm0 = smem_u32(sm);
    uint32_t *s_bad = reinterpret_cast<uint32_t *>(sm + C::BAD);
    uint64_t *full = reinterpret_cast<uint64_t *>(sm + C::BARS), *empty = full + C::SLOTS, *landed = empty + C::SLOTS;
    uint64_t *staged = landed + C::SLOTS, *q_free = staged + 1, *q_full = q_free + 1, *s_full = q_full + 2, *p_full = s_full + 2, *drain = p_full + 2;
    int *s_int = reinterpret_cast<int *>(drain + 1);              // abort, V set aside, TMEM base, least position
    volatile int *s_abort = s_int, *s_flag = s_int + 1;
    int *s_lo = s_int + 3, *s_lock = s_int + 4;
    uint32_t *s_tmem = reinterpret_cast<uint32_t *>(s_int + 2);
    if (sm0 & 1023) {                             // the swizzled tiles need it; never seen
        if (tid == 0) paged_err(a, QMS_PAGED_ETIMEOUT);
        pdl_wait();
        return;
    }
    if (tid == 0) {
        for (int i = 0; i < C::SLOTS; i++) {
            mbar_init(&full[i], 1);
            mbar_init(&empty[i], SPLIT ? 1 : 2);
            mbar_init(&landed[i], 1);
        }
        for (int i = 0; i < 2; i++) {
            mbar_init(&q_full[i], 128);
            mbar_init(&s_full[i], 1);
            mbar_init(&p_full[i], 4);
        }
        mbar_init(drain, 2);
        mbar_init(staged, 4);
        mbar_init(q_free, 2);
        s_int[0] = s_int[1] = *s_lock = 0;
        *s_lo = 0x7fffffff;
        fence_mbar_init();
    }
    if (warp == 11) {
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
    const WideSync sy{s_abort, &a};
    WideWork work(A, own, lo_p);
    WideUnit w;

    if (warp < 8) {
        // ---- softmax of stream i: thread = row = TMEM lane
        const int i = warp >> 2, row = (warp & 3) * 32 + lane;
        const uint32_t lanes = tmem + ((uint32_t)((warp & 3) * 32) << 16);
        const uint32_t s_col = lanes + i * kWTile, o_col = lanes + C::O_COL + i * D;
        uint32_t ns = 0, before = 0, unit_no = 0; // phases of s_full; position tiles of the CTA's earlier units (for s_bad)
        bool ok = true;
        for (; ok && work.next(w); before += w.nt, unit_no++) {
            if (!SPLIT && i >= w.tiles) continue;
            const int r = w.r0 + (SPLIT ? 0 : i * kWTile) + row, t = r / a.G;    // this row: its token, position below
            int tok = -1;                                                        // token row * H + head (-1: none)
            int64_t qo = -1;                                                     // where its q is
            if (r < w.rows) {
                const int h = w.kh * a.G + (r - t * a.G);
                tok = (w.t0 + t) * a.H + h;
                qo = (w.t0 + t) * A.ldq + (int64_t)h * D;
            }
            // q: 8 lanes per row, 4 rows at a time: row maximum, power-of-two scale, two fp16 terms, swizzled
            // rows (SPLIT: one stream writes them for both, the other one only wants the scales)
            float f = 0.0f;
            const uint32_t sign = A.scale2 < 0.0f ? 0x80000000u : 0u;  // f >= 0: the largest s f has the largest s
            float4 x[2][4][D / 32];
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
                    // the maximum goes to 2^9 .. 2^10: times 2^(up - 127), undone by 2^(127 - up) in the score
                    const uint32_t up = mx == 0.0f ? 127u : min(263u - (__float_as_uint(mx) >> 23), 253u);
                    const float got = __shfl_sync(kFull, fabsf(A.scale2) * __uint_as_float((254u - up) << 23), (lane & 3) * 8);
                    if (lane >> 2 == g0 + g) f = got;
                    if (SPLIT && i == 1) continue;
                    const float m = __uint_as_float(up << 23 | sign);
                    const int rr = (warp & 3) * 32 + 4 * (g0 + g) + (lane >> 3);
                    const uint32_t at = sm0 + (SPLIT ? 0 : i * 2 * C::TILE) + rr * 128 + (lane & 1) * 8;
#pragma unroll
                    for (int k = 0; k < D / 32; k++) {
                        const float2 y0 = f2_mul(make_float2(z[g][k].x, z[g][k].y), make_float2(m, m)), y1 = f2_mul(make_float2(z[g][k].z, z[g][k].w), make_float2(m, m));
                        const float2 h0 = make_float2(tf32_hi(y0.x), tf32_hi(y0.y)), h1 = make_float2(tf32_hi(y1.x), tf32_hi(y1.y));
                        const float2 l0 = f2_fma(h0, make_float2(-1.0f, -1.0f), y0), l1 = f2_fma(h1, make_float2(-1.0f, -1.0f), y1);
                        // values 4 (lane & 7) + 32 k .. + 3: 16-byte piece (lane & 7) / 2 + 4 (k & 1) of half k / 2
                        const uint32_t to = at + (k >> 1) * C::HALF + (((((lane & 7) >> 1) + 4 * (k & 1)) ^ (rr & 7)) << 4);
                        asm volatile("st.shared.v2.b32 [%0], {%1, %2};" ::"r"(to), "r"(pack_h2(h0.x, h0.y)), "r"(pack_h2(h1.x, h1.y)) : "memory");
                        asm volatile("st.shared.v2.b32 [%0], {%1, %2};" ::"r"(to + C::TILE), "r"(pack_h2(l0.x, l0.y)), "r"(pack_h2(l1.x, l1.y)) : "memory");
                    }
                }
            };
            fetch(x[0], 0);
            fetch(x[1], 4);
            if (SPLIT && i == 0 && unit_no > 0 && !(ok = __all_sync(kFull, sy.wait(staged, (unit_no - 1) & 1)))) break;
            place(x[0], 0);
            place(x[1], 4);
            fence_async_smem();
            if (!SPLIT || i == 0) mbar_arrive(&q_full[i]);
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
            float B = -INFINITY;
            float2 l2 = make_float2(0.0f, 0.0f);
            for (int j = SPLIT ? i : 0; j < w.nt; j += SPLIT ? 2 : 1) {
                if (!(ok = __all_sync(kFull, sy.wait(&s_full[i], ns & 1)))) break;    // the whole warp or none of it
                ns++;
                tc_fence_after();
                const int base = w.k0 + j * kWTile;
                const uint32_t *bad = s_bad + ((before + j) & 7) * 4;
                // rows that see nothing of this unit are not read from its slot: no mask for them
                if (__any_sync(kFull, lim >= w.kmin && lim < base + kWTile - 1) || base < w.kmin || (bad[0] | bad[1] | bad[2] | bad[3])) {
#pragma unroll 1
                    for (int c = 0; c < 4; c++) {
                        const int d = lim - base - 32 * c;
                        const int below = w.kmin - base - 32 * c;
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
                const float2 f2 = make_float2(f, f);
                auto weights = [&](uint32_t (&z)[32], int c, uint32_t done) {
                    float mx = max3(__uint_as_float(z[0]), __uint_as_float(z[1]), __uint_as_float(z[2]));
#pragma unroll
                    for (int e = 3; e < 31; e += 2) mx = max3(mx, __uint_as_float(z[e]), __uint_as_float(z[e + 1]));
                    mx = fmaxf(mx, __uint_as_float(z[31]));
                    mx = mx == -INFINITY ? mx : mx * f;
                    if (__any_sync(kFull, mx > B + kWHigh)) {
                        const float nb = mx > B + kWHigh ? ceilf(mx) - kWLow : B, fac = B == nb ? 1.0f : B == -INFINITY ? 0.0f : ex2(B - nb);
                        B = nb;
                        l2.x *= fac;
                        l2.y *= fac;
                        if (j > 1 || (!SPLIT && j > 0)) {      // (the MMAs on O ended before this tile's S was announced)
#pragma unroll 1
                            for (int k = 0; k < D / 32; k++) {
                                uint32_t o[32];
                                tmem_ld<32>(o_col + 32 * k, o);
                                tmem_wait_ld(o);
#pragma unroll
                                for (int e = 0; e < 32; e++) o[e] = __float_as_uint(__uint_as_float(o[e]) * fac);
                                tmem_st32(o_col + 32 * k, o);
                            }
                        }
                        const __half2 fh = __float2half2_rn(fac);
#pragma unroll 1
                        for (int k = 0; k < 4; k++) {
                            if (!(done >> k & 1)) continue;
                            uint32_t o[32];
                            tmem_wait_st();
                            tmem_ld<32>(s_col + 32 * k, o);
                            tmem_wait_ld(o);
#pragma unroll
                            for (int e = 0; e < 32; e++) {
                                const __half2 p2 = __hmul2(*reinterpret_cast<const __half2 *>(&o[e]), fh);
                                o[e] = *reinterpret_cast<const uint32_t *>(&p2);
                            }
                            tmem_st32(s_col + 32 * k, o);
                        }
                    }
                    const float2 nB = B == -INFINITY ? make_float2(0.0f, 0.0f) : make_float2(-B, -B);
                    uint32_t o[32];
#pragma unroll
                    for (int e = 0; e < 32; e += 2) {
                        const float2 q = f2_fma(make_float2(__uint_as_float(z[e]), __uint_as_float(z[e + 1])), f2, nB);
                        const float2 w2 = make_float2(ex2(q.x), ex2(q.y));
                        const float2 h = make_float2(tf32_hi(w2.x), tf32_hi(w2.y));        // 11 bits: an fp16 value
                        const float2 lo = f2_fma(h, make_float2(-1.0f, -1.0f), w2);
                        l2 = f2_add(l2, w2);
                        o[e / 2] = pack_h2(h.x, h.y);
                        o[16 + e / 2] = pack_h2(lo.x, lo.y);
                    }
                    tmem_st32(s_col + 32 * c, o);
                };
                uint32_t x[32], y[32];
                tmem_ld<32>(s_col, x);
                tmem_wait_ld(x);
                tmem_ld<32>(s_col + 32, y);       // the next 32 come while these are worked on
                weights(x, 0, 0);
                tmem_wait_ld(y);
                tmem_ld<32>(s_col + 64, x);
                weights(y, 1, 1);
                tmem_wait_ld(x);
                tmem_ld<32>(s_col + 96, y);
                weights(x, 2, 3);
                tmem_wait_ld(y);
                weights(y, 3, 7);
                tmem_wait_st();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&p_full[i]);
            }
            if (SPLIT && i >= w.nt) {             // no position tile for this stream
                if (lane == 0) mbar_arrive(staged);
                continue;
            }
            if (!ok || !(ok = __all_sync(kFull, sy.wait(&s_full[i], ns & 1)))) break;     // O is complete
            ns++;
            tc_fence_after();
            // SPLIT: Q, where the rows are staged, is both streams'
            if (SPLIT && !(ok = __all_sync(kFull, sy.wait(q_free, unit_no & 1)))) break;
            const float l = l2.x + l2.y;
            if (isnan(l) && B == -INFINITY) B = 0.0f;
            const bool put = tok >= 0 && lim >= (SPLIT && i ? w.k0 + kWTile : w.kmin), none = l == 0.0f, fix = *s_flag != 0;
            const int64_t first = (int64_t)(w.slot + (SPLIT ? i : 0)) * a.n_tok * a.H;
            const int row_out = put ? tok : -1;
            float *part = A.part_o + first * D + (lane & 7) * 4;
            // the rows leave by way of shared memory (where this warp's rows of Q are; SPLIT's second stream: of
            // their low terms), 128 bytes of a row per 8 lanes
            unsigned char *stage = sm + i * (SPLIT ? 1 : 2) * C::TILE + (warp & 3) * 4096;
#pragma unroll 1
            for (int c = 0; c < D / 32; c++) {
                uint32_t o[32];
                tmem_ld<32>(o_col + 32 * c, o);
                tmem_wait_ld(o);
                if (fix && put) {
                    // V that were set aside: added where the row sees them (inf and NaN are not changed by a weight)
                    for (int p = w.kmin; p <= lim; p++) {
                        if (SPLIT && ((p - w.k0) / kWTile & 1) != i) continue;
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
                __syncwarp();
#pragma unroll
                for (int e = 0; e < 32; e += 4)   // 16-byte piece e / 4 of row `lane`, XOR-placed against bank conflicts
                    *reinterpret_cast<uint4 *>(stage + lane * 128 + (((e >> 2) ^ (lane & 7)) << 4)) =
                        none ? make_uint4(0, 0, 0, 0) : make_uint4(o[e], o[e + 1], o[e + 2], o[e + 3]);
                __syncwarp();
#pragma unroll
                for (int k = 0; k < 8; k++) {     // 4 rows of 128 bytes at a time
                    const int rr = 4 * k + (lane >> 3), to = __shfl_sync(kFull, row_out, rr);
                    const uint4 v = *reinterpret_cast<const uint4 *>(stage + rr * 128 + (((lane & 7) ^ (rr & 7)) << 4));
                    if (to >= 0) *reinterpret_cast<uint4 *>(part + (int64_t)to * D + 32 * c) = v;
                }
            }
            if (SPLIT && i == 1) {
                __syncwarp();
                if (lane == 0) mbar_arrive(staged);
            }
            if (put) A.part_ml[first + tok] = make_float2(none ? -INFINITY : B, l);
            tc_fence_before();
        }
    } else if (warp < 10) {
        // ---- K and V, in the order of their use: K, V of each position tile, or (SPLIT) K, K, V, V of two. Warp 8 issues them; V tiles with rows that not every row sees (or that were
        // not loaded) land on a barrier of their own and are passed on by warp 9.
        uint32_t c[2] = {0, 0}, t = 0, phases = 0;       // loads so far (SPLIT: of each stream); tiles; of `landed`
        bool ok = true;
        const int R = min(1 << a.page_log, kWTile), boxes = kWTile / R;        // positions per box, boxes per 64 values
        while (ok && work.next(w)) {
            const int *table = a.table + (own ? (int64_t)w.b * a.table_stride : 0);
            constexpr int STEP = SPLIT ? 2 : 1;
            for (int j0 = 0; ok && j0 < w.nt; j0 += STEP) {
                const int m = min(STEP, w.nt - j0);
                for (int k = 0; ok && k < 2 * m; k++) {
                    const bool is_v = k >= m;
                    const int jj = is_v ? k - m : k, base = w.k0 + (j0 + jj) * kWTile;
                    const uint32_t n = SPLIT && jj ? c[1]++ : c[0]++, slot = C::slot(jj, n);
                    // lane x: page of box x (positions base + x R ..); boxes past the unit are not loaded
                    const int p = base + lane * R;
                    int page = -1;
                    if (lane < boxes && p < w.k1) {
                        page = table[p >> a.page_log];
                        if ((unsigned)page >= (unsigned)a.n_pages) {
                            page = -1;
                            if (warp == 8) paged_err(a, QMS_PAGED_EPAGE);
                        }
                    }
                    const uint32_t have = __ballot_sync(kFull, page >= 0), want = __ballot_sync(kFull, lane < boxes && p < w.k1);
                    const int seen = min(w.lo, w.k1 - 1);
                    const bool scan = is_v && (base + kWTile - 1 > seen || base < w.kmin || want != have);
                    if (warp == 8) {
                        if (!is_v && lane < 4) {  // bits of the tile's positions on bad pages
                            uint32_t bits = 0;
                            if (want != have)
                                for (int e = 0; e < 32; e++) bits |= ((want & ~have) >> ((lane * 32 + e) / R) & 1u) << e;
                            s_bad[((t + jj) & 7) * 4 + lane] = bits;
                        }
                        __syncwarp();
                        if (n >= C::RINGLEN) ok = __all_sync(kFull, sy.wait(&empty[slot], C::phase(n) ^ 1));
                        if (!ok) break;
                        uint64_t *bar = scan ? &landed[slot] : &full[slot];
                        if (lane == 0) mbar_arrive_expect_tx(bar, __popc(have) * (uint32_t)(R * 128 * C::HALVES));
                        __syncwarp();
                        const uint32_t dst = sm0 + C::RING + slot * C::TILE + lane * R * 128;
                        if (page >= 0)
#pragma unroll
                            for (int h = 0; h < C::HALVES; h++) tma_load4(dst + h * C::HALF, is_v ? &mv : &mk, h * 64, w.kh, p & ((1 << a.page_log) - 1), page, bar);
                    } else if (scan) {
                        ok = __all_sync(kFull, ok && sy.wait(&landed[slot], phases >> slot & 1));
                        phases ^= 1u << slot;
                        for (int x = lane; ok && x < kWTile * C::CH; x += 32) {
                            const int r = x / C::CH, piece = x % C::CH;
                            if (base + r >= w.kmin && base + r <= seen && want == have) continue;
                            uint4 *pv = reinterpret_cast<uint4 *>(sm + C::RING + slot * C::TILE + (piece >> 3) * C::HALF + r * 128 +
                                                                  (((piece & 7) ^ (r & 7)) << 4));
                            uint4 v = *pv;
                            if (drop_nonfinite((const __half *)nullptr, v)) {
                                *pv = v;
                                if (base + r >= w.kmin && base + r < w.k1) *s_flag = 1;      // (else left over: nobody's)
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
    } else {
        // ---- the MMAs of stream i, by one thread
        const int i = warp - 10;
        if (lane == 0) {
            constexpr uint32_t id_s = idesc_f16(kWTile, false), id_o = idesc_f16(D, true);
            uint32_t c = 0, nq = 0, np = 0;                     // loads of the ring so far; phases of q_full, p_full
            bool ok = true;
            auto score = [&](uint32_t n) {                     // S_i = (hi + lo of Q_i) K^T
                const uint32_t k = sm0 + C::RING + C::slot(i, n) * C::TILE, q = sm0 + (SPLIT ? 0 : i * 2 * C::TILE);
#pragma unroll
                for (int term = 0; term < 2; term++)
#pragma unroll
                    for (int ks = 0; ks < D / 16; ks++) {
                        const uint32_t o = (ks >> 2) * C::HALF + (ks & 3) * 32;
                        umma_f16_ss(tmem + i * kWTile, desc_sw128(q + term * C::TILE + o, 16, 1024), desc_sw128(k + o, 16, 1024), id_s, term || ks);
                    }
            };
            auto weigh = [&](uint32_t n, bool first) {         // O_i (+)= (hi + lo of P_i) V
                const uint32_t v = sm0 + C::RING + C::slot(i, n) * C::TILE;
#pragma unroll
                for (int term = 0; term < 2; term++)
#pragma unroll
                    for (int ks = 0; ks < kWTile / 16; ks++)
                        umma_f16_ts(tmem + C::O_COL + i * D, tmem + i * kWTile + (ks >> 1) * 32 + term * 16 + (ks & 1) * 8,
                                    desc_sw128(v + ks * 2048, C::HALF, 1024), id_o, !first || term || ks);
            };
            auto lock = [&]() {
                uint32_t x = 0;
                do {                                            // (reading costs less than trying)
                    while (*(volatile int *)s_lock != 0 && ++x < kWSpin) {}
                } while (atomicCAS(s_lock, 0, 1) != 0 && x < kWSpin);
            };
            auto unlock = [&]() { *(volatile int *)s_lock = 0; };
            auto full_at = [&](uint32_t n) { return sy.wait(&full[C::slot(i, n)], C::phase(n)); };
            while (ok && work.next(w)) {
                // this stream's position tiles; loads c + 2 j (K) and c + 2 j + 1 (V) of its ring are tile j of them
                const int nt = SPLIT ? (w.nt + 1 - i) / 2 : w.nt;
                if (SPLIT || i < w.tiles) {
                    ok = sy.wait(&q_full[SPLIT ? 0 : i], nq++ & 1);
                    if (ok && nt > 0 && (ok = full_at(c))) {
                        tc_fence_after();
                        lock();
                        score(c);
                        unlock();
                        umma_commit(&s_full[i]);
                        umma_commit(&empty[C::slot(i, c)]);
                    }
                    if (SPLIT && ok && nt == 0) mbar_arrive(q_free);
                    if (SPLIT && ok && nt == 1) umma_commit(q_free);
                    for (int j = 0; ok && j < nt; j++, c += 2) {
                        const bool more = j + 1 < nt;
                        if (!(ok = full_at(c + 1) && sy.wait(&p_full[i], np++ & 1))) break;
                        tc_fence_after();
                        lock();
                        weigh(c + 1, j == 0);
                        if (more) {
                            if (!mbar_test_wait(&full[C::slot(i, c + 2)], C::phase(c + 2))) {      // K is late: not at the other's cost
                                unlock();
                                if (!(ok = full_at(c + 2))) break;
                                lock();
                            }
                            score(c + 2);
                        }
                        unlock();
                        umma_commit(&s_full[i]);
                        umma_commit(&empty[C::slot(i, c + 1)]);
                        if (more) umma_commit(&empty[C::slot(i, c + 2)]);
                        if (SPLIT && j + 2 == nt) umma_commit(q_free);          // the last of the unit's reads of Q
                    }
                } else {                                        // one row tile: the other stream's loads are read once
                    for (int x = 0; ok && x < 2 * nt; x++, c++)
                        if ((ok = full_at(c))) mbar_arrive(&empty[C::slot(i, c)]);
                }
            }
            if (!ok) {                                          // nothing of this CTA's is in flight when TMEM goes
                umma_commit(drain);
                *s_abort = 1;
                for (uint32_t n = 0; n < kWSpin && !mbar_try_wait(drain, 0); n++) __nanosleep(32);
            }
        }
        __syncwarp();
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 11) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
    }
    if (last) pdl_wait();
}

template <int D, bool SPLIT>
static int launch_wide(const PagedAttn &A, bool own, bool last, cudaStream_t s) {
    using C = WideCfg<D, SPLIT>;
    static_assert(C::SMEM <= 232448, "shared memory per CTA");
    const int64_t units = !own && A.p.line > 0 ? A.p.line
                          : own                ? (int64_t)A.p.chunks_s * A.a.n_seq * A.p.tiles_s * A.a.Hk
                                               : (int64_t)A.p.chunks_p * A.p.tiles_p * A.a.Hk;
    QMS_REQUIRE(units < (1ll << 30), QMS_CUDA_EUNSUPPORTED, "paged_attention: too many units of work");
    static unsigned long long set = 0;                          // per device
    int dev = 0;
    QMS_CK(cudaGetDevice(&dev));
    if (!(set >> (dev & 63) & 1)) {
        QMS_CK(cudaFuncSetAttribute(k_paged_wide<D, SPLIT>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM));
        set |= 1ull << (dev & 63);
    }
    CUtensorMap mk, mv;
    int rc = paged_map(A.a, D, true, kWTile, A.a.k, &mk);
    if (rc || (rc = paged_map(A.a, D, true, kWTile, A.a.v, &mv))) return rc;
    const int grid = (int)(units < 148 ? units : 148);
    QMS_CK(launch_pdl(k_paged_wide<D, SPLIT>, dim3(grid), dim3(kWThreads), C::SMEM, s, A, mk, mv, own, last));
    return QMS_CUDA_OK;
}

int launch_paged_wide(const PagedAttn &A, int D, bool own, bool last, cudaStream_t s) {
    const bool split = (own ? A.p.wr_s : A.p.wr_p) == kPaWideSplit;
    if (D == 128) return split ? launch_wide<128, true>(A, own, last, s) : launch_wide<128, false>(A, own, last, s);
    return split ? launch_wide<64, true>(A, own, last, s) : launch_wide<64, false>(A, own, last, s);
}

}  // namespace qms
