// qms_prompt.cu - causal grouped-query attention over whole prompts, packed one after another, in 16 bits, on tcgen05 tensor cores
// (B200, sm_100a). The reference attends one position of one sequence at a time in fp32 (src/model.c:465-492).
//
// A unit of work is two tiles of up to 128 rows of one sequence and kv head; a row is a (token, q head of the kv head's group)
// pair, row = token * G + head, so that a tile of 16 heads holds 8 tokens, hardly more positions than each of them sees, and a
// prompt of a few tokens fills a tile. Both tiles go over the sequence's positions in tiles of 128, two streams that take turns:
// the tensor cores work on one while the other's softmax runs. For each tile of a stream
//   S = Q K^T   tcgen05.mma kind::f16 from shared memory, M 128, K = head_dim, N the tile's positions (rounded up to 16)
//   softmax     one thread per row: base-2 exponents, the running base B and sum l in fp32; the weights 2^(s f - B), rounded to the
//               type once, go back over S. (The rounding of a weight is the type's half step of itself, as the output's own rounding
//               is; l adds up what was rounded, so that rows of few positions hardly have it.)
//   O += P V    P from TMEM, V as it lies in shared memory (MN-major), in fp32 over the whole unit
// B is a whole number and stays until a score lies 2^15 above it. S is read twice, for its maximum and for the weights: one vote per
// tile, nothing that the exponentials wait for, and short loops (a row's 128 scores in registers, all in line: 1.03 times as fast over 8192
// positions, 0.87 over 1500).
// Bound by the two products and the exponentials in turn (16 of a row's 128 per cycle and SM), and by what is between them where two streams
// do not cover it: 8192 tokens of 64 q heads and 4 kv heads 1060 to 1190 us with the clock, 0.93 to 1.03 PFLOP/s, 0.55 to 0.62 of the library's rate
// for one large product; 17 prompts of up to 1500 tokens 152, 0.63 PFLOP/s: of some 20,000 cycles per unit 5000 are its first S, its last
// product and its rows. Short ones by the chain of one unit: 100 tokens 8.7 us, 64 prompts of up to 333 tokens with 8 heads of 64 values 24.4 for
// three units per SM.
#include <cuda_bf16.h>
#include <math.h>
#include <string.h>

#include <algorithm>

#include "qms_moe.cuh"
#include "qms_paged.cuh"
#include "qms_tcgen05.cuh"

namespace qms {

constexpr float kPrLow = 8.0f, kPrHigh = 15.0f;     // a new base is 2^8 below the maximum; weights stay below 2^15

struct PromptAttn {
    Paged a;                         // q_start, n_seq, n_tok, max_q, H, Hk, G, err
    const char *v;
    char *out;
    int64_t v_tok, v_head, o_tok, o_head;           // elements
    float f;                         // scale * log2(e)
    int tq;                          // tokens per tile: 128 / G
    int share;                       // sequences per unit number
    int out32, whole;                // fp32 rows out; rows out on 32-byte boundaries
};

template <int D>
struct PrCfg {
    static constexpr int THREADS = 384, TMA_WARP = 8, SCAN_WARP = 9, MMA_WARP = 10, UNIT_WARP = 11;
    static constexpr int HALVES = D / 64;                       // 64 values = 128 bytes: one swizzle row
    static constexpr uint32_t HALF = 128 * 128, TILE = HALVES * HALF;
    static constexpr uint32_t SLOTS = D == 128 ? 5 : 8;
    // then: the unit at hand and the answer of who asked for the next; barriers; flags
    static constexpr uint32_t RING = 2 * TILE, UNIT = RING + SLOTS * TILE, BARS = UNIT + 32, SMEM = BARS + (3 * SLOTS + 14) * 8 + 16;
    static constexpr uint32_t O_COL = 256;                      // TMEM columns: S0, S1, O0, O1
};

// 32 bytes of a row; whole: one sector.
__device__ __forceinline__ void put32(char *dst, const uint32_t *x, bool whole) {
    if (whole) {
        asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(dst), "r"(x[0]), "r"(x[1]), "r"(x[2]), "r"(x[3]), "r"(x[4]), "r"(x[5]),
                     "r"(x[6]), "r"(x[7])
                     : "memory");
    } else {
        *reinterpret_cast<uint4 *>(dst) = make_uint4(x[0], x[1], x[2], x[3]);
        *reinterpret_cast<uint4 *>(dst + 16) = make_uint4(x[4], x[5], x[6], x[7]);
    }
}

// Place in a ring: slot and the parity of its phase.
template <uint32_t SLOTS>
struct RingAt {
    uint32_t slot = 0, phase = 0;
    __device__ __forceinline__ void next() {
        if (++slot == SLOTS) slot = 0, phase ^= 1;
    }
    __device__ __forceinline__ void skip(uint32_t n) { slot = (slot + n) % SLOTS; }        // (the slot alone)
};

__device__ __forceinline__ void tmem_st16(uint32_t addr, const uint32_t (&r)[16]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(addr), "r"(r[0]),
                 "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]),
                 "r"(r[13]), "r"(r[14]), "r"(r[15])
                 : "memory");
}
__device__ __forceinline__ void tma_load3(uint32_t dst, const CUtensorMap *map, int x, int head, int tok, uint64_t *bar) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst), "l"(map),
                 "r"(x), "r"(head), "r"(tok), "r"(smem_u32(bar))
                 : "memory");
}

// The MMAs by the low words of the operands' descriptors; the high word is the same for all: 1024 bytes between groups of 8 rows,
// 128-byte swizzle.
__device__ __forceinline__ uint32_t desc_lo(uint32_t saddr, uint32_t lbo) { return (uint32_t)desc_sw128(saddr, lbo, 1024); }
constexpr uint32_t kDescHi = 1024u >> 4 | 1u << 14 | 2u << 29;
__device__ __forceinline__ void umma_ss_lo(uint32_t d, uint32_t da, uint32_t db, uint32_t idesc, bool acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 a, b;\n\tsetp.ne.b32 p, %4, 0;\n\tmov.b64 a, {%1, %5};\n\tmov.b64 b, {%2, %5};\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, p;\n\t}" ::"r"(d), "r"(da), "r"(db), "r"(idesc), "r"((uint32_t)acc), "n"(kDescHi)
        : "memory");
}
__device__ __forceinline__ void umma_ts_lo(uint32_t d, uint32_t a, uint32_t db, uint32_t idesc, bool acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 b;\n\tsetp.ne.b32 p, %4, 0;\n\tmov.b64 b, {%2, %5};\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %3, p;\n\t}" ::"r"(d), "r"(a), "r"(db), "r"(idesc), "r"((uint32_t)acc), "n"(kDescHi)
        : "memory");
}

// Two fp32 as a pair of the 16-bit type, and back.
template <bool BF>
__device__ __forceinline__ uint32_t pack16(float x, float y) {
    if constexpr (BF) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
        return *reinterpret_cast<const uint32_t *>(&h);
    } else {
        return pack_h2(x, y);
    }
}
template <bool BF>
__device__ __forceinline__ float2 unpack16(uint32_t v) {
    if constexpr (BF) return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
    else return __half22float2(*reinterpret_cast<const __half2 *>(&v));
}
template <bool BF>
__device__ __forceinline__ bool drop_nonfinite16(uint4 &v) {        // zero what is not finite; true if something was
    constexpr uint32_t E = BF ? 0x7F80u : 0x7C00u;
    uint32_t w[4] = {v.x, v.y, v.z, v.w};
    bool any = false;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        if ((w[i] & E) == E) {
            w[i] &= 0xFFFF0000u;
            any = true;
        }
        if ((w[i] & E << 16) == E << 16) {
            w[i] &= 0x0000FFFFu;
            any = true;
        }
    }
    v = make_uint4(w[0], w[1], w[2], w[3]);
    return any;
}

// x += the first, y += the second of a pair of the 16-bit type, in fp32.
template <bool BF>
__device__ __forceinline__ void add16(uint32_t v, float &x, float &y) {
    if constexpr (BF)
        asm("{\n\t.reg .b16 a, b, o;\n\tmov.b32 {a, b}, %2;\n\tmov.b16 o, 0x3F80;\n\tfma.rn.f32.bf16 %0, a, o, %0;\n\tfma.rn.f32.bf16 %1, b, o, %1;\n\t}"
            : "+f"(x), "+f"(y)
            : "r"(v));
    else
        asm("{\n\t.reg .b16 a, b, o;\n\tmov.b32 {a, b}, %2;\n\tmov.b16 o, 0x3C00;\n\tfma.rn.f32.f16 %0, a, o, %0;\n\tfma.rn.f32.f16 %1, b, o, %1;\n\t}"
            : "+f"(x), "+f"(y)
            : "r"(v));
}
// One unit of work: kv head; the sequence's first token row and length (-1: there are no more units); the unit's first token.
struct PromptUnit {
    int kh, t0, n, tok0;
    __device__ __forceinline__ int last(int i, int tq) const { return min(n, tok0 + (i + 1) * tq) - 1; }      // of stream i
    __device__ __forceinline__ bool there(int i, int tq) const { return tok0 + i * tq < n; }
    __device__ __forceinline__ int tiles(int i, int tq) const { return there(i, tq) ? last(i, tq) / 128 + 1 : 0; }
};

// The search for a unit's rows goes on from where the last one was found, since a CTA's unit numbers grow but for chance: otherwise n_seq
// prompts would take n_seq^2 / 64 steps (65,536 of a token each took 160 ms so, 1.6 as it is).
struct UnitSearch {
    int b0 = 0, before = 0;          // 32 sequences from b0 on, and the units (of a kv head) of those before them
};

// Unit u of the call, by the whole warp: kv heads in the innermost, a sequence's tiles from its end (long ones first). False: there
// are not so many.
__device__ __forceinline__ bool prompt_unit(const PromptAttn &A, unsigned u, UnitSearch &s, PromptUnit &w) {
    const Paged &a = A.a;
    const int lane = threadIdx.x & 31;
    const int v = u / a.Hk;
    w.kh = u - v * a.Hk;
    if (v < s.before) s = UnitSearch();
    for (; s.b0 < a.n_seq; s.b0 += 32) {
        int t0 = 0, n = 0, kv;
        if (s.b0 + lane < a.n_seq) prompt_seq(a, s.b0 + lane, t0, n, kv);
        const int mine = (n + 2 * A.tq - 1) / (2 * A.tq);
        int upto = s.before + mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int x = __shfl_up_sync(kFull, upto, o) - s.before;
            if (lane >= o) upto += x;
        }
        const unsigned hit = __ballot_sync(kFull, upto > v);
        if (hit) {
            const int at = __ffs(hit) - 1;
            w.t0 = __shfl_sync(kFull, t0, at);
            w.n = __shfl_sync(kFull, n, at);
            w.tok0 = (__shfl_sync(kFull, upto, at) - 1 - v) * 2 * A.tq;
            return true;
        }
        s.before = __shfl_sync(kFull, upto, 31);
    }
    return false;
}

template <int D, bool BF>
__global__ void __launch_bounds__(384, 1) k_prompt_attn(const PromptAttn A, const __grid_constant__ CUtensorMap mq, const __grid_constant__ CUtensorMap mk,
                                                        const __grid_constant__ CUtensorMap mv) {
    using C = PrCfg<D>;
    extern __shared__ __align__(1024) unsigned char sm[];
    const Paged &a = A.a;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, tq = A.tq, G = a.G;
    const uint32_t sm0 = smem_u32(sm);
    // full, empty: of the ring's slots; landed: V tiles that go on after a look
    uint64_t *full = reinterpret_cast<uint64_t *>(sm + C::BARS), *empty = full + C::SLOTS, *landed = empty + C::SLOTS, *q_full = landed + C::SLOTS;
    uint64_t *q_empty = q_full + 2, *s_full = q_empty + 2, *p_full = s_full + 2, *o_full = p_full + 2, *drain = o_full + 2;
    uint64_t *u_full = drain + 1, *u_empty = u_full + 1, *u_got = u_empty + 1;
    int *s_int = reinterpret_cast<int *>(u_got + 1);            // abort, V set aside, TMEM base
    volatile int *s_abort = s_int, *s_flag = s_int + 1;
    uint32_t *s_tmem = reinterpret_cast<uint32_t *>(s_int + 2);
    if (sm0 & 1023) {                             // the swizzled tiles need it; never seen
        if (tid == 0) paged_err(a, QMS_PAGED_ETIMEOUT);
        return;
    }
    if (tid == 0) {
        for (uint32_t i = 0; i < C::SLOTS; i++) {
            mbar_init(&full[i], 1);
            mbar_init(&empty[i], 1);
            mbar_init(&landed[i], 1);
        }
        for (int i = 0; i < 2; i++) {
            mbar_init(&q_full[i], 1);
            mbar_init(&q_empty[i], 1);
            mbar_init(&s_full[i], 1);
            mbar_init(&p_full[i], 4);
            mbar_init(&o_full[i], 1);
        }
        mbar_init(drain, 1);
        mbar_init(u_full, 1);
        mbar_init(u_empty, 11);
        mbar_init(u_got, 1);
        s_int[0] = s_int[1] = 0;
        fence_mbar_init();
    }
    if (warp == C::MMA_WARP) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(s_tmem)), "r"(512) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    // rows of a tile that no token fills stay zero
    for (int x = tid; x < (128 - tq * G) * 8 * C::HALVES * 2; x += C::THREADS) {
        const int per = (128 - tq * G) * 8, half = x / per, r = tq * G + x % per / 8;
        *reinterpret_cast<uint4 *>(sm + half * C::HALF + r * 128 + (x & 7) * 16) = make_uint4(0, 0, 0, 0);
    }
    fence_async_smem();
    pdl_wait();
    pdl_trigger();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *s_tmem;
    const WideSync sy{s_abort, &a};
    PromptUnit w;
    // the next unit, by each warp but the one that finds them; false: a wait gave up
    uint32_t units = 0;
    auto next_unit = [&]() {
        if (!__all_sync(kFull, sy.wait(u_full, units++ & 1))) return false;
        const volatile int *x = reinterpret_cast<const int *>(sm + C::UNIT);
        w = PromptUnit{x[0], x[1], x[2], x[3]};
        __syncwarp();
        if (lane == 0) mbar_arrive(u_empty);
        return true;
    };

    if (warp < 8) {
        // ---- softmax of stream i: thread = row = TMEM lane
        const int i = warp >> 2, row = (warp & 3) * 32 + lane;
        const uint32_t lanes = tmem + ((uint32_t)((warp & 3) * 32) << 16), s_col = lanes + i * 128, o_col = lanes + C::O_COL + i * D;
        const int my_tok = row / G, my_head = row - my_tok * G;
        const float f = A.f;
        uint32_t ns = 0, no = 0;
        RingAt<C::SLOTS> at;
        const bool gives = (warp & 3) == 0 && lane == 0;
        bool ok = true;
        while (ok && (ok = next_unit()) && w.n >= 0) {
            const int nt = w.tiles(i, tq);
            const bool gives_kv = gives && w.there(1, tq) == (i == 1);             // the stream that uses a tile last (it has as many, or more)
            if (nt == 0) {
                at.skip(2 * w.tiles(0, tq));
                continue;
            }
            const int lo = w.tok0 + i * tq, last = w.last(i, tq), tok = lo + my_tok;       // every row sees the positions up to lo
            const bool there = my_tok < tq && tok <= last;
            const int pos = there ? tok : -1;
            auto scale_o = [&](float fac) {       // O times a power of 2 (the MMAs on it ended before the S at hand was announced)
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
            float B = -INFINITY, l = 0.0f;
            for (int j = 0; j < nt; j++) {
                if (!(ok = __all_sync(kFull, sy.wait(&s_full[i], ns & 1)))) break;
                ns++;
                tc_fence_after();
                // what the MMAs that ended before this S read can be written again: K of this tile, V of the last, Q
                if (gives_kv) {
                    mbar_arrive(&empty[at.slot]);
                    if (j > 0) mbar_arrive(&empty[at.slot == 0 ? C::SLOTS - 1 : at.slot - 1]);
                }
                if (gives && j + 1 == nt) mbar_arrive(&q_empty[i]);
                at.skip(2);
                uint32_t x[32], y[32];
                const int chunks = min(4, (last - j * 128) / 32 + 1);
                float mx0 = -INFINITY, mx1 = -INFINITY;
                auto most = [&](const uint32_t (&z)[32], int e) {
                    mx0 = max3(mx0, __uint_as_float(z[e]), __uint_as_float(z[e + 1]));
                    mx1 = max3(mx1, __uint_as_float(z[e + 2]), __uint_as_float(z[e + 3]));
                };
                if (j * 128 + 127 > lo) {         // some row does not see the whole tile
#pragma unroll 1
                    for (int c = 0; c < chunks; c++) {
                        const int d = pos - j * 128 - 32 * c;
                        const uint32_t vis = d < 0 ? 0u : d >= 31 ? 0xffffffffu : (2u << d) - 1u;
                        tmem_ld<32>(s_col + 32 * c, x);
                        tmem_wait_ld(x);
#pragma unroll
                        for (int e = 0; e < 32; e++) x[e] = vis >> e & 1 ? x[e] : 0xff800000u;
                        tmem_st32(s_col + 32 * c, x);
#pragma unroll
                        for (int e = 0; e < 32; e += 4) most(x, e);
                    }
                    tmem_wait_st();
                } else {
                    tmem_ld<32>(s_col, x);
#pragma unroll 1
                    for (int c = 0; c < 4; c += 2) {
                        tmem_wait_ld(x);
                        tmem_ld<32>(s_col + 32 * c + 32, y);
#pragma unroll
                        for (int e = 0; e < 32; e += 4) most(x, e);
                        tmem_wait_ld(y);
                        if (c == 0) tmem_ld<32>(s_col + 64, x);
#pragma unroll
                        for (int e = 0; e < 32; e += 4) most(y, e);
                    }
                }
                tmem_ld<32>(s_col, x);
                const float top = fmaxf(mx0, mx1) * f;
                // the base stays unless a score lies 2^kPrHigh above it: then what was computed with the old one is scaled
                if (__any_sync(kFull, top - B > kPrHigh)) {
                    // (from 2^24 on a score's own rounding would move the weights by powers of 2: NaN says so)
                    const float far = fabsf(top) < 16777216.0f ? ceilf(top) - kPrLow : NAN, nb = top - B > kPrHigh ? far : B;
                    const float fac = B == nb ? 1.0f : B == -INFINITY ? 0.0f : ex2(B - nb);
                    B = nb;
                    l *= fac;
                    if (j > 0) scale_o(fac);
                }
                const float2 f2 = make_float2(f, f), nB = B == -INFINITY ? make_float2(0.0f, 0.0f) : make_float2(-B, -B);
                float l0 = 0.0f, l1 = 0.0f, l2 = 0.0f, l3 = 0.0f;
                auto weights = [&](uint32_t (&z)[32], int c) {
                    uint32_t o[16];
#pragma unroll
                    for (int e = 0; e < 32; e += 2) {
                        const float2 q = f2_fma(make_float2(__uint_as_float(z[e]), __uint_as_float(z[e + 1])), f2, nB);
                        o[e / 2] = pack16<BF>(ex2(q.x), ex2(q.y));
                        if (e & 2) add16<BF>(o[e / 2], l0, l1);
                        else add16<BF>(o[e / 2], l2, l3);
                    }
                    tmem_st16(s_col + 16 * c, o);
                };
#pragma unroll 1
                for (int c = 0; c < chunks; c += 2) {
                    tmem_wait_ld(x);
                    tmem_ld<32>(s_col + 32 * c + 32, y);
                    weights(x, c);
                    tmem_wait_ld(y);
                    if (c == 0) tmem_ld<32>(s_col + 64, x);
                    if (c + 1 < chunks) weights(y, c + 1);
                }
                tmem_wait_ld(x);
                l += (l0 + l1) + (l2 + l3);
                tmem_wait_st();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&p_full[i]);
            }
            if (!ok) break;
            if (!(ok = __all_sync(kFull, sy.wait(&o_full[i], no & 1)))) break;
            no++;
            tc_fence_after();
            if (gives_kv) mbar_arrive(&empty[at.slot == 0 ? C::SLOTS - 1 : at.slot - 1]);      // V of the last tile
            at.skip(2 * (max(w.tiles(0, tq), w.tiles(1, tq)) - nt));
            // ---- the rows: O / l, each thread its own, a sector of 32 bytes by one store. (Few instructions: they are new to the
            // instructions' cache at the end of every unit. 64 prompts of up to 333 tokens: rows exchanged between 8 threads, for whole lines, 27 us;
            // between 4 26.5; so 24.6.)
            const float inv = l == 0.0f ? 0.0f : __fdividef(1.0f, l);
            const bool none = l == 0.0f, fix = *s_flag != 0;
            char *dst = A.out + ((int64_t)(w.t0 + tok) * A.o_tok + (int64_t)(w.kh * G + my_head) * A.o_head) * (A.out32 ? 4 : 2);
#pragma unroll 1
            for (int c = 0; c < D / 32; c++) {
                uint32_t o[32];
                tmem_ld<32>(o_col + 32 * c, o);
                tmem_wait_ld(o);
                if (there) {
                    if (fix) {
                        // V that were set aside: added where the row sees them (inf and NaN are not changed by a weight)
                        for (int p = w.tok0 + 1; p <= pos; p++) {
                            const char *vr = A.v + ((int64_t)(w.t0 + p) * A.v_tok + w.kh * A.v_head + 32 * c) * 2;
#pragma unroll
                            for (int e = 0; e < 16; e++) {
                                const float2 y = unpack16<BF>(__ldcg(reinterpret_cast<const unsigned int *>(vr) + e));
                                if (!isfinite(y.x)) o[2 * e] = __float_as_uint(__uint_as_float(o[2 * e]) + y.x);
                                if (!isfinite(y.y)) o[2 * e + 1] = __float_as_uint(__uint_as_float(o[2 * e + 1]) + y.y);
                            }
                        }
                    }
#pragma unroll
                    for (int e = 0; e < 32; e++) o[e] = none ? 0u : __float_as_uint(__uint_as_float(o[e]) * inv);
                    if (A.out32) {
#pragma unroll
                        for (int e = 0; e < 32; e += 8) put32(dst + 128 * c + 4 * e, o + e, A.whole);
                    } else {
#pragma unroll
                        for (int e = 0; e < 16; e++) o[e] = pack16<BF>(__uint_as_float(o[2 * e]), __uint_as_float(o[2 * e + 1]));
                        put32(dst + 64 * c, o, A.whole), put32(dst + 64 * c + 32, o + 8, A.whole);
                    }
                }
                __syncwarp();
            }
            tc_fence_before();
        }
        tmem_wait_st();
    } else if (warp == C::TMA_WARP) {
        // ---- Q of both tiles, then K and V of every tile of positions. What lies behind the sequence in a box is masked, or read as 0.
        RingAt<C::SLOTS> at;
        uint32_t n = 0, nq[2] = {0, 0};
        bool ok = true;
        while (ok && (ok = next_unit()) && w.n >= 0) {
            const int nt = max(w.tiles(0, tq), w.tiles(1, tq));
#pragma unroll
            for (int i = 0; i < 2; i++) {
                if (!ok || !w.there(i, tq)) continue;
                if (nq[i] > 0) ok = __all_sync(kFull, sy.wait(&q_empty[i], (nq[i] - 1) & 1));
                nq[i]++;
                if (ok && lane == 0) {
                    mbar_arrive_expect_tx(&q_full[i], tq * G * 128 * C::HALVES);
                    for (int x = 0; x < C::HALVES; x++) tma_load3(sm0 + i * C::TILE + x * C::HALF, &mq, x * 64, w.kh * G, w.t0 + w.tok0 + i * tq, &q_full[i]);
                }
            }
            for (int j = 0; ok && j < 2 * nt; j++, n++, at.next()) {
                const bool is_v = j & 1;
                const int base = j / 2 * 128;
                if (n >= C::SLOTS && !(ok = __all_sync(kFull, sy.wait(&empty[at.slot], at.phase ^ 1)))) break;
                if (lane == 0) {
                    uint64_t *bar = is_v && base + 127 > w.tok0 ? &landed[at.slot] : &full[at.slot];
                    mbar_arrive_expect_tx(bar, C::TILE);
                    for (int x = 0; x < C::HALVES; x++)
                        tma_load3(sm0 + C::RING + at.slot * C::TILE + x * C::HALF, is_v ? &mv : &mk, x * 64, w.kh, w.t0 + base, bar);
                }
                __syncwarp();
            }
        }
    } else if (warp == C::SCAN_WARP) {
        // ---- V tiles with rows that not every row of the unit sees: behind the mask a weight is 0, but 0 * inf is not
        RingAt<C::SLOTS> at;
        uint32_t phases = 0;                      // of `landed`
        bool ok = true;
        while (ok && (ok = next_unit()) && w.n >= 0) {
            const int nt = max(w.tiles(0, tq), w.tiles(1, tq)), end = max(w.last(0, tq), w.last(1, tq)) + 1;
            for (int j = 0; ok && j < nt; j++) {
                at.next();
                const int base = j * 128;
                if (base + 127 > w.tok0) {
                    ok = __all_sync(kFull, sy.wait(&landed[at.slot], phases >> at.slot & 1));
                    phases ^= 1u << at.slot;
                    const int r0 = max(0, w.tok0 + 1 - base), r1 = min(128, (end - base + 15) & ~15);        // (the products read 16 at a time)
                    for (int x = r0 * (D / 8) + lane; ok && x < r1 * (D / 8); x += 32) {
                        const int r = x / (D / 8), piece = x % (D / 8);
                        uint4 *pv = reinterpret_cast<uint4 *>(sm + C::RING + at.slot * C::TILE + (piece >> 3) * C::HALF + r * 128 +
                                                              (((piece & 7) ^ (r & 7)) << 4));
                        uint4 v = *pv;
                        if (drop_nonfinite16<BF>(v)) {
                            *pv = v;
                            if (base + r < end) *s_flag = 1;       // (else the next sequence's: nobody's)
                        }
                    }
                    fence_async_smem();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&full[at.slot]);
                }
                at.next();
            }
        }
    } else if (warp == C::MMA_WARP) {
        // ---- the MMAs of both streams in turn, by one thread. An instruction runs 64 cycles, so what leads to the next one has to be
        // little: descriptors of which only the low word changes, by a constant. (Made anew for each they took 100 cycles, in loops
        // that are not unrolled 130; two threads, one per stream and under a lock, were no better.)
        constexpr uint32_t kind = BF ? 1u << 7 | 1u << 10 : 0u, id_o = idesc_f16(D, true) | kind;
        RingAt<C::SLOTS> at;
        uint32_t np = 0, nq = 0;                               // phases of p_full, q_full
        bool ok = true;
        auto wait = [&](uint64_t *bar, uint32_t parity) {      // (no sleep: what follows is late by as much)
            for (uint32_t n = 0; !mbar_test_wait(bar, parity); n++) {
                if (*s_abort) return false;
                if (n == kWSpin) {
                    *s_abort = 1;
                    paged_err(a, QMS_PAGED_ETIMEOUT);
                    return false;
                }
            }
            return true;
        };
        auto score = [&](int i, uint32_t slot, int cnt) {      // S_i = Q_i K^T
            const uint32_t id_s = idesc_f16((cnt + 15) & ~15, false) | kind;
            const uint32_t dq = desc_lo(sm0 + i * C::TILE, 16), dk = desc_lo(sm0 + C::RING + slot * C::TILE, 16);
#pragma unroll
            for (int ks = 0; ks < D / 16; ks++) {
                const uint32_t off = ((ks >> 2) * C::HALF + (ks & 3) * 32) >> 4;
                umma_ss_lo(tmem + i * 128, dq + off, dk + off, id_s, ks > 0);
            }
        };
        auto weigh = [&](int i, uint32_t slot, int cnt, bool first) {      // O_i (+)= P_i V
            const uint32_t dv = desc_lo(sm0 + C::RING + slot * C::TILE, C::HALF);
#pragma unroll
            for (int ks = 0; ks < 8; ks++)
                if (ks * 16 < cnt) umma_ts_lo(tmem + C::O_COL + i * D, tmem + i * 128 + ks * 8, dv + ks * 128, id_o, ks > 0 || !first);
        };
        while (ok && (ok = next_unit()) && w.n >= 0) {
            if (lane == 0) {
                const int nt0 = w.tiles(0, tq), nt1 = w.tiles(1, tq), all = max(nt0, nt1);
                ok = wait(&full[at.slot], at.phase);
#pragma unroll 1
                for (int i = 0; i < 2; i++) {
                    if (!ok || (i && nt1 == 0)) break;
                    if (!(ok = wait(&q_full[i], nq >> i & 1))) break;
                    nq ^= 1u << i;
                    tc_fence_after();
                    score(i, at.slot, min(128, w.last(i, tq) + 1));
                    umma_commit(&s_full[i]);
                }
                for (int j = 0; ok && j < all; j++) {
                    at.next();                                 // V of tile j
                    const RingAt<C::SLOTS> va = at;
                    at.next();                                 // K of the next (or of the next unit)
                    if (!(ok = wait(&full[va.slot], va.phase))) break;
                    if (j + 1 < all && !(ok = wait(&full[at.slot], at.phase))) break;
#pragma unroll 1
                    for (int i = 0; i < 2; i++) {
                        if (j >= (i ? nt1 : nt0)) continue;
                        if (!(ok = wait(&p_full[i], np >> i & 1))) break;
                        np ^= 1u << i;
                        tc_fence_after();
                        const int cnt = w.last(i, tq) + 1 - 128 * j;
                        weigh(i, va.slot, cnt, j == 0);
                        if (cnt > 128) {
                            score(i, at.slot, min(128, cnt - 128));
                            umma_commit(&s_full[i]);
                        } else {
                            umma_commit(&o_full[i]);
                        }
                    }
                }
            }
            ok = __shfl_sync(kFull, (int)ok, 0);
        }
        if (lane == 0) {
            if (!ok) *s_abort = 1;
            umma_commit(drain);                                // nothing of this CTA's is in flight when TMEM goes
            for (uint32_t n = 0; n < kWSpin && !mbar_try_wait(drain, 0); n++) __nanosleep(32);
        }
        __syncwarp();
    } else {
        // ---- which unit is next: the CTA's own, then those of CTAs of the grid that have not started, one ahead of the softmax
        uint32_t k = 0;
        bool ok = true;
        auto publish = [&](const PromptUnit &x) {
            if (k > 0 && !__all_sync(kFull, sy.wait(u_empty, (k - 1) & 1))) return false;
            k++;
            if (lane == 0) {
                volatile int *to = reinterpret_cast<int *>(sm + C::UNIT);
                to[0] = x.kh, to[1] = x.t0, to[2] = x.n, to[3] = x.tok0;
                mbar_arrive(u_full);
            }
            __syncwarp();
            return true;
        };
        unsigned u = blockIdx.x;
        UnitSearch search;
        for (uint32_t asked = 0;; asked++) {
            if (prompt_unit(A, u, search, w) && !(ok = publish(w))) break;
            if (lane == 0) {
                fence_async_smem();
                mbar_arrive_expect_tx(u_got, 16);
                asm volatile("clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];" ::"r"(sm0 + C::UNIT + 16),
                             "r"(smem_u32(u_got))
                             : "memory");
            }
            // the batch's arrays, checked once: a share of them goes with each unit number, by whoever takes it (no CTA is sure to start),
            // while the answer is on its way
            const int64_t b1 = min((int64_t)a.n_seq, ((int64_t)u + 1) * A.share);
            for (int64_t b = (int64_t)u * A.share + lane; b < b1; b += 32) {
                int t0, cnt, kv;
                if (!prompt_seq(a, (int)b, t0, cnt, kv)) paged_err(a, QMS_PAGED_ELEN);
            }
            __syncwarp();
            uint32_t n = 0;                       // (not given up before the answer is there, abort or not: it is written to this CTA's memory)
            while (!mbar_try_wait(u_got, asked & 1) && ++n < kWSpin) {}
            if (!__all_sync(kFull, n < kWSpin)) {
                *s_abort = 1;
                if (lane == 0) paged_err(a, QMS_PAGED_ETIMEOUT);
                ok = false;
                break;
            }
            uint32_t got, x;
            asm volatile(
                "{\n\t.reg .b128 r;\n\t.reg .pred p;\n\tld.shared.b128 r, [%2];\n\t"
                "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, r;\n\tselp.u32 %0, 1, 0, p;\n\tmov.u32 %1, 0;\n\t"
                "@p clusterlaunchcontrol.query_cancel.get_first_ctaid::x.b32.b128 %1, r;\n\t}"
                : "=r"(got), "=r"(x)
                : "r"(sm0 + C::UNIT + 16)
                : "memory");
            __syncwarp();
            if (!got) break;
            u = x;
        }
        if (ok) publish(PromptUnit{0, 0, -1, 0});
    }
    tc_fence_before();
    __syncthreads();
    if (*s_abort)                                 // copies in flight have 0.1 s to land before the CTA's memory goes
        for (int n = 0; n < 1 << 20; n++) __nanosleep(100);
    if (warp == C::MMA_WARP) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
    }
}

// ---- host ------------------------------------------------------------------------------------------
// Rows of heads as a tensor [token][head][value], in boxes of 64 values x heads x tokens, 128-byte swizzled.
static int heads_map(const QmsCudaHeads &h, bool bf, int D, int heads, int n_tok, int box_heads, int box_tok, CUtensorMap *map) {
    TensorEncode encode;
    const int rc = tensor_encode(&encode);
    if (rc) return rc;
    const cuuint64_t dim[3] = {(cuuint64_t)D, (cuuint64_t)heads, (cuuint64_t)n_tok};
    // (the stride of a dimension of one has no meaning, and may be one that the encoder does not take)
    const cuuint64_t stride[2] = {heads > 1 ? (cuuint64_t)h.head_stride * 2 : (cuuint64_t)D * 2, n_tok > 1 ? (cuuint64_t)h.tok_stride * 2 : (cuuint64_t)heads * D * 2};
    const cuuint32_t box[3] = {64, (cuuint32_t)box_heads, (cuuint32_t)box_tok}, one[3] = {1, 1, 1};
    const CUresult ru = encode(map, bf ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, h.data, dim, stride, box, one,
                               CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                               CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    QMS_REQUIRE(ru == CUDA_SUCCESS, QMS_CUDA_EINVAL, "prompt_attention: the rows' strides do not make a tensor map (%d)", (int)ru);
    return QMS_CUDA_OK;
}

template <int D, bool BF>
static int launch_prompt(PromptAttn &A, const QmsCudaHeads &q, const QmsCudaHeads &k, const QmsCudaHeads &v, cudaStream_t s) {
    using C = PrCfg<D>;
    static_assert(C::SMEM <= 232448, "shared memory per CTA");
    static std::atomic<unsigned long long> done{0};
    int rc = allow_smem(done, k_prompt_attn<D, BF>, C::SMEM);
    if (rc) return rc;
    CUtensorMap mq, mk, mv;
    if ((rc = heads_map(q, BF, D, A.a.H, A.a.n_tok, A.a.G, A.tq, &mq)) || (rc = heads_map(k, BF, D, A.a.Hk, A.a.n_tok, 1, 128, &mk)) ||
        (rc = heads_map(v, BF, D, A.a.Hk, A.a.n_tok, 1, 128, &mv)))
        return rc;
    const int64_t most = ((int64_t)A.a.n_tok / (2 * A.tq) + std::min(A.a.n_seq, A.a.n_tok)) * A.a.Hk;      // units there can be
    QMS_REQUIRE(most < (1ll << 31), QMS_CUDA_EUNSUPPORTED, "prompt_attention: too many units of work");
    const unsigned grid = (unsigned)most;          // (those that have not started are taken over by CTAs that have)
    A.share = (int)((A.a.n_seq + most - 1) / most);
    QMS_CK(launch_pdl(k_prompt_attn<D, BF>, dim3(grid), dim3(C::THREADS), C::SMEM, s, A, mq, mk, mv));
    return QMS_CUDA_OK;
}

static int heads_args(const char *what, const QmsCudaHeads *h, int D, int es) {
    QMS_REQUIRE(h && h->data && ((uintptr_t)h->data & 15) == 0, QMS_CUDA_EINVAL, "prompt_attention: %s must be 16-byte aligned device memory", what);
    QMS_REQUIRE(h->tok_stride >= D && h->head_stride >= D && h->tok_stride * es % 16 == 0 && h->head_stride * es % 16 == 0 &&
                    h->tok_stride < (1ll << 36) && h->head_stride < (1ll << 36),
                QMS_CUDA_EINVAL, "prompt_attention: %s strides must be multiples of 16 bytes, at least a head's %d values", what, D);
    return QMS_CUDA_OK;
}

}  // namespace qms

using namespace qms;

extern "C" {

int qms_cuda_prompt_attention(const QmsCudaPagedBatch *batch, int type, const QmsCudaHeads *q, const QmsCudaHeads *k, const QmsCudaHeads *v,
                              int n_head, int n_head_kv, int head_dim, float scale, int out_type, const QmsCudaHeads *out, int *err, void *stream) {
    clear_error();
    QMS_REQUIRE(batch, QMS_CUDA_EINVAL, "prompt_attention: NULL descriptor");
    QMS_REQUIRE(type == QMS_T_F16 || type == QMS_CUDA_T_BF16, QMS_CUDA_EUNSUPPORTED, "prompt_attention: type %d (F16 or BF16)", type);
    QMS_REQUIRE(out_type == type || out_type == QMS_T_F32, QMS_CUDA_EUNSUPPORTED, "prompt_attention: rows out of type %d (that of q, or F32)", out_type);
    QMS_REQUIRE(head_dim == 64 || head_dim == 128, QMS_CUDA_EUNSUPPORTED, "prompt_attention: head_dim %d (64 or 128 supported)", head_dim);
    QMS_REQUIRE(n_head > 0 && n_head_kv > 0 && n_head % n_head_kv == 0 && n_head <= 1024, QMS_CUDA_EINVAL, "prompt_attention: %d q heads over %d kv heads",
                n_head, n_head_kv);
    QMS_REQUIRE(n_head / n_head_kv <= 128, QMS_CUDA_EUNSUPPORTED, "prompt_attention: %d q heads per kv head (at most 128)", n_head / n_head_kv);
    QMS_REQUIRE(batch->n_seq >= 0 && batch->n_tok >= 0 && batch->n_tok <= (1 << 20) && batch->n_seq <= (1 << 20) && batch->max_q >= 0, QMS_CUDA_EINVAL,
                "prompt_attention: n_seq %d, n_tok %d, max_q %d", batch->n_seq, batch->n_tok, batch->max_q);
    QMS_REQUIRE(batch->n_seq == 0 || batch->q_start, QMS_CUDA_EINVAL, "prompt_attention: NULL q_start");
    QMS_REQUIRE((((uintptr_t)batch->q_start | (uintptr_t)err) & 3) == 0, QMS_CUDA_EINVAL, "prompt_attention: misaligned int array");
    QMS_REQUIRE(scale > 0.0f && scale <= 1e30f, QMS_CUDA_EINVAL, "prompt_attention: scale must be positive and finite");
    if (batch->n_tok == 0 || batch->n_seq == 0) return QMS_CUDA_OK;
    int rc;
    if ((rc = heads_args("q", q, head_dim, 2)) || (rc = heads_args("k", k, head_dim, 2)) || (rc = heads_args("v", v, head_dim, 2)) ||
        (rc = heads_args("out", out, head_dim, out_type == QMS_T_F32 ? 4 : 2)))
        return rc;
    PromptAttn A;
    memset(&A, 0, sizeof A);
    A.a.q_start = batch->q_start;
    A.a.n_seq = batch->n_seq;
    A.a.n_tok = batch->n_tok;
    A.a.max_q = batch->max_q;
    A.a.H = n_head;
    A.a.Hk = n_head_kv;
    A.a.G = n_head / n_head_kv;
    A.a.err = err;
    A.v = (const char *)v->data;
    A.out = (char *)out->data;
    A.v_tok = v->tok_stride;
    A.v_head = v->head_stride;
    A.o_tok = out->tok_stride;
    A.o_head = out->head_stride;
    A.f = fmaxf(scale * 1.4426950408889634f, 1.17549435e-38f);
    A.tq = 128 / A.a.G;
    A.out32 = out_type == QMS_T_F32;
    const int64_t es = A.out32 ? 4 : 2;
    A.whole = (((uintptr_t)out->data | (uintptr_t)(out->tok_stride * es) | (uintptr_t)(out->head_stride * es)) & 31) == 0;
    const cudaStream_t s = (cudaStream_t)stream;
    if (type == QMS_T_F16) return head_dim == 128 ? launch_prompt<128, false>(A, *q, *k, *v, s) : launch_prompt<64, false>(A, *q, *k, *v, s);
    return head_dim == 128 ? launch_prompt<128, true>(A, *q, *k, *v, s) : launch_prompt<64, true>(A, *q, *k, *v, s);
}

}  // extern "C"
