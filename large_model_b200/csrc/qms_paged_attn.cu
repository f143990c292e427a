// qms_paged_attn.cu - causal grouped-query attention of a batch of new tokens over a paged KV cache on B200
// (sm_100a); src/model.c:465-492 is the reference's, of one sequence over one contiguous cache.
//
// One pass over the positions with the running maximum and sum of the softmax, the two products on the tensor
// cores with 22-bit operands: an fp32 operand x, scaled by a power of two into fp16's range, is split as x = hi + lo
// into two fp16 terms (one alone would leave an error of 2^-12), and their products are added in fp32.
// Over an fp16 cache K and V are exact: two mma.sync m16n8k16 per product. Over an fp32 cache K and V are split too,
// once per stage in shared memory, and three products kept (lo * lo is below 2^-22); the tf32 form of the same
// (m16n8k8, three products, split in every warp) took about twice as long.
#include <math.h>
#include <string.h>

#include <algorithm>

#include "qms_moe.cuh"
#include "qms_paged.cuh"

namespace qms {

constexpr uint32_t kPaSpin = 1u << 22;
constexpr float kPaShift = 8.0f;      // weights reach 2^8: their fp16 low terms stay clear of the subnormals
constexpr int pa_stage(int type) { return type == QMS_T_F16 ? 64 : 32; }       // positions per stage: 32 KB of K and V

__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
__device__ __forceinline__ void mma_f16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// The same from 0.
__device__ __forceinline__ void mma_f16_first(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
                 : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));
}
// ---- the kernel over mma.sync ----------------------------------------------------------------------
// A CTA of 4 warps takes units of (16 WR rows, one chunk of positions): WR row groups of 16 rows x WK groups of
// positions x WD parts of head_dim (in the second product; the first is done by each). K and V come in
// by TMA, a stage of positions at a time, one box per page (cp.async cost some 2000 of 4300 cycles per stage in
// issuing alone); stages start on page boundaries, so the first may begin before the unit's first position, and boxes
// past the unit or on bad pages are not loaded: all that is masked. Each warp scores its rows against its share
// of the stage, keeps its own running (m, l, o), and the position groups are joined in shared memory at the end.
// One token each of 64 sequences of 4096 positions (64 q heads, 4 kv heads): fp16 104 us, 5.2 TB/s, 0.80 of a plain copy;
// fp32 308 us, 3.5 TB/s. What is left goes to the chain of each stage: the barrier, the scores, the softmax and (fp32) the
// split before them; issue slots are 36% (31%) used, tensor cores 31% (22%). One sequence of 1100 positions: 12 us, of which some 4
// are the launch and 4 the join of the slots.
template <int D, typename KT, int WR>
struct PaCfg {
    static constexpr bool F16 = sizeof(KT) == 2;
    static constexpr int PS = F16 ? 64 : 32;
    static constexpr int WD = !F16 && WR == 1 ? 2 : 1, WK = 4 / WR / WD;
    static constexpr int KW = PS / WK, NT = KW / 8, DW = D / WD;             // positions, 8-position tiles, output dims per warp
    static constexpr int CH = D * (int)sizeof(KT) / 16, ROW = D * (int)sizeof(KT);      // a row as it comes: 16-byte pieces, bytes
    static constexpr int STAGE = 2 * ROW * PS;                               // K, then V
    // The tiles that the MMAs read: fp16 rows in halves of 64 values (128 bytes), their 16-byte pieces XOR-swizzled by the
    // row (ldmatrix reads 8 rows at one piece): the stages themselves, or (fp32) hi and lo of K, hi and lo of V
    // after the ring.
    static constexpr int HTILE = 2 * D * PS, HALF = 128 * PS;
    static __device__ __forceinline__ uint32_t piece(int r, int c) { return (c >> 3) * HALF + r * 128 + (((c & 7) ^ (r & 7)) << 4); }
    static constexpr int NS = WR == 1 || !F16 ? 2 : 3, MINB = WR == 1 && F16 ? 3 : 2;    // stages; CTAs per SM
    static constexpr int CONV = NS * STAGE;
    static constexpr int RED = WK > 1 ? WK * WR * 16 * (D + 4) * 4 : 0;      // the position groups' o, m, l
    static constexpr int USED = CONV + (F16 ? 0 : 4 * HTILE), SMEM = (USED > RED ? USED : RED) + 1024;    // (1024: alignment)
    static constexpr int QROWS = 16 * WR, QHALF = 128 * QROWS;               // the tile's q, as HTILE: hi, lo
};

// OWN: the sequences' own positions; else the shared ones. LAST: launched beside the kernel of the other kind,
// whose end it waits for at its own end, so that what follows this kernel follows both.
template <int D, typename KT, int WR>
__global__ void __launch_bounds__(128, PaCfg<D, KT, WR>::MINB) k_paged_attn(const PagedAttn A, const __grid_constant__ CUtensorMap mk,
                                                                               const __grid_constant__ CUtensorMap mv, const bool own, const bool last) {
    using C = PaCfg<D, KT, WR>;
    extern __shared__ unsigned char sm_[];
    __shared__ uint64_t s_full[C::NS];
    __shared__ int s_pos[64];                     // position of each row of the tile (-1: none)
    __shared__ int s_tok[64];                     // token row * H + q head (-1: none)
    __shared__ float s_f[64];                     // score factor of each row
    __shared__ int s_bad[4][2];                   // stage c's positions on bad pages, as a bit mask, at c % 4
    __shared__ __align__(8) float s_fk[C::F16 ? 1 : C::PS];    // what undoes the scale of each K row of a stage (fp32)
    __shared__ uint32_t s_max[4];                 // largest |V| of a stage (fp32), by warp
    __shared__ int s_flag;                        // V had values that are not finite behind the mask
    __shared__ volatile int s_abort;
    const Paged &a = A.a;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, tq = lane & 3;
    const int wr = warp % WR, wk = warp / WR % C::WK, wd = warp / WR / C::WK;
    unsigned char *sm = sm_ + (-smem_u32(sm_) & 1023);
    const uint32_t sm0 = smem_u32(sm);
    if (tid == 0) {
        for (int i = 0; i < C::NS; i++) mbar_init(&s_full[i], 1);
        s_abort = 0;
        fence_mbar_init();
    }
    uint32_t c0 = 0;                              // stages of the CTA's earlier units
    // the trigger comes after the wait: a kernel that starts on it may read what this one waited for
    if (!last) pdl_wait();
    pdl_trigger();
    const int n_unit = (own ? A.p.chunks_s * a.n_seq * A.p.tiles_s : A.p.chunks_p * A.p.tiles_p) * a.Hk;
    for (int unit = blockIdx.x; unit < n_unit; unit += gridDim.x) {
        // ---- which rows, which positions
        int u = unit;
        const int kh = u % a.Hk;
        u /= a.Hk;
        const int tile = u % (own ? A.p.tiles_s : A.p.tiles_p);
        u /= own ? A.p.tiles_s : A.p.tiles_p;
        int b = 0, slot, k0, k1, t0 = 0, n = 0, kv = 0;
        if (own) {
            b = u % a.n_seq;
            slot = u / a.n_seq;
            paged_seq(a, b, t0, n, kv);
            k0 = A.p.base_s + slot * A.p.chunk_s;
            k1 = min(kv, k0 + A.p.chunk_s);
            if (max(k0, a.prefix) >= k1 || tile * 16 * WR >= n * a.G) continue;
            slot += A.p.slots_p;
        } else {
            slot = u;
            k0 = slot * A.p.chunk_p;
            k1 = min(a.prefix, k0 + A.p.chunk_p);
        }
        const int *table = a.table + (own ? (int64_t)b * a.table_stride : 0);
        const int kmin = own ? max(k0, a.prefix) : k0;
        const int r0 = tile * 16 * WR;
        fence_async_smem();
        __syncthreads();                          // the previous unit is done with shared memory
        if (tid == 0) s_flag = 0;
        // rows of the tile: the sequence's own, or all tokens' (each token's sequence found by a warp)
        if (own) {
            if (tid < 16 * WR) {
                const int r = r0 + tid, i = r / a.G;
                s_pos[tid] = i < n ? kv - n + i : -1;
                s_tok[tid] = i < n ? (t0 + i) * a.H + kh * a.G + (r - i * a.G) : -1;
            }
        } else {
            const int first = r0 / a.G, end = min(a.n_tok, (r0 + 16 * WR + a.G - 1) / a.G);
            for (int t = first + warp; t < end; t += 4) {
                int s0 = 0, sn = 0, skv = 0;
                const int sb = paged_seq_of(a, t);
                if (sb < a.n_seq) paged_seq(a, sb, s0, sn, skv);
                const int pos = t >= s0 && t < s0 + sn ? skv - sn + (t - s0) : -1;
                for (int j = lane; j < a.G; j += 32) {
                    const int r = t * a.G + j - r0;
                    if (r >= 0 && r < 16 * WR) {
                        s_pos[r] = pos;
                        s_tok[r] = t * a.H + kh * a.G + j;
                    }
                }
            }
            if (tid < 16 * WR && r0 + tid >= a.n_tok * a.G) s_pos[tid] = s_tok[tid] = -1;
        }
        // A stage's boxes (of K and V, by halves of a row where those are boxes of their own) in turn over the four warps, one
        // lane each: a lane issues a box in some 90 cycles. Page ids are fetched a stage ahead; warp 0 also looks at
        // all of them (box i in lane i, and i + 32) for what to expect and what is bad.
        const int R = min(1 << a.page_log, C::PS), boxes = C::PS / R;
        constexpr int KINDS = C::F16 ? D / 32 : 2;                 // tensors x halves
        int pages[2], every[2];
        auto page_of = [&](int st, int i) {
            const int p = k0 + st * C::PS + i * R;
            return i < boxes && p < k1 ? table[p >> a.page_log] : -2;                          // -2: past the unit
        };
        auto look_up = [&](int st) {
#pragma unroll
            for (int h = 0; h < 2; h++) {
                pages[h] = page_of(st, ((lane + 32 * h) * 4 + warp) / KINDS);
                every[h] = warp == 0 ? page_of(st, lane + 32 * h) : -2;
            }
        };
        auto load = [&](int st) {                 // (its pages have been looked up)
            const uint32_t c = c0 + st, dst = sm0 + c % C::NS * C::STAGE;
            uint64_t *bar = &s_full[c % C::NS];
            if (warp == 0) {
                uint32_t have = 0, bad[2];
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    const bool b = every[h] != -2 && (unsigned)every[h] >= (unsigned)a.n_pages;
                    have += __popc(__ballot_sync(kFull, every[h] != -2 && !b));
                    bad[h] = __ballot_sync(kFull, b);
                    if (b) paged_err(a, QMS_PAGED_EPAGE);
                }
                if (lane < 2) {                   // bits of the stage's positions
                    uint32_t bits = 0;
                    if (bad[0] | bad[1])
                        for (int e = 0; e < 32; e++) {
                            const int i = (lane * 32 + e) / R;
                            bits |= (lane * 32 + e < C::PS ? bad[i >> 5 & 1] >> (i & 31) & 1u : 0u) << e;
                        }
                    s_bad[c & 3][lane] = (int)bits;
                }
                if (lane == 0) mbar_arrive_expect_tx(bar, have * (uint32_t)(2 * R * C::ROW));
            }
#pragma unroll
            for (int h = 0; h < 2; h++)
                if ((unsigned)pages[h] < (unsigned)a.n_pages) {
                    const int item = (lane + 32 * h) * 4 + warp, i = item / KINDS, kind = item % KINDS;
                    const int y = (k0 + st * C::PS + i * R) & ((1 << a.page_log) - 1);
                    const uint32_t to = dst + (kind & 1) * (C::STAGE / 2) + (C::F16 ? (kind >> 1) * C::HALF + i * R * 128 : i * R * C::ROW);
                    tma_load4(to, kind & 1 ? &mv : &mk, (kind >> 1) * 64, kh, y, pages[h], bar);
                }
        };
        look_up(0);
        __syncthreads();
        int lo_pos = 0x7fffffff, hi_pos = -1;     // least and largest position among the tile's rows
        for (int r = lane; r < 16 * WR; r += 32) {
            const int p = s_pos[r];
            if (p >= 0) lo_pos = min(lo_pos, p);
            hi_pos = max(hi_pos, p);
        }
        lo_pos = __reduce_min_sync(kFull, lo_pos);
        hi_pos = __reduce_max_sync(kFull, hi_pos);
        if (kmin > hi_pos) continue;              // nobody sees any of it
        const int k_end = min(k1, hi_pos + 1), nst = (k_end - k0 + C::PS - 1) / C::PS;
#pragma unroll
        for (int st = 0; st < C::NS - 1; st++) {
            if (st < nst) load(st);
            look_up(st + 1);
        }

        // ---- q: 8 lanes per row; each row scaled by a power of two into fp16's range (exact; undone in the score's factor)
        // and split, into the stage slot that is filled last; from there as mma A fragments
        unsigned char *qs = sm + (c0 + C::NS - 1) % C::NS * C::STAGE;
#pragma unroll
        for (int i = 0; i < WR; i++) {
            const int r = (warp * WR + i) * 4 + (lane >> 3), tok = s_tok[r], t = tok < 0 ? 0 : tok / a.H;
            const float4 *src = reinterpret_cast<const float4 *>(A.q + t * A.ldq + (int64_t)(tok < 0 ? 0 : tok - t * a.H) * D) + (lane & 7);
            float4 x[D / 32];
            uint32_t mx = 0;
#pragma unroll
            for (int k = 0; k < D / 32; k++) x[k] = tok < 0 ? make_float4(0.0f, 0.0f, 0.0f, 0.0f) : __ldcg(src + 8 * k);
#pragma unroll
            for (int k = 0; k < D / 32; k++) mx = max(mx, max(max(finite_bits(x[k].x), finite_bits(x[k].y)), max(finite_bits(x[k].z), finite_bits(x[k].w))));
            mx = max(mx, __shfl_xor_sync(kFull, mx, 1));
            mx = max(mx, __shfl_xor_sync(kFull, mx, 2));
            mx = max(mx, __shfl_xor_sync(kFull, mx, 4));
            const uint32_t up = scale_up(mx >> 23);
            if ((lane & 7) == 0) s_f[r] = A.scale2 * pow2_bits(254u - up);
            const float m = pow2_bits(up);
#pragma unroll
            for (int k = 0; k < D / 32; k++) {    // values 4 (lane & 7) + 32 k .. + 3
                const int c = 4 * k + ((lane & 7) >> 1);
                unsigned char *to = qs + (c >> 3) * C::QHALF + r * 128 + (((c & 7) ^ (r & 7)) << 4) + (lane & 1) * 8;
                uint32_t h[2], l[2];
                split_h2(x[k].x * m, x[k].y * m, h[0], l[0]);
                split_h2(x[k].z * m, x[k].w * m, h[1], l[1]);
                *reinterpret_cast<uint2 *>(to) = make_uint2(h[0], h[1]);
                *reinterpret_cast<uint2 *>(to + C::QROWS * D * 2) = make_uint2(l[0], l[1]);
            }
        }
        __syncthreads();
        const int pos0 = s_pos[wr * 16 + g], pos1 = s_pos[wr * 16 + g + 8];
        const float f0 = s_f[wr * 16 + g], f1 = s_f[wr * 16 + g + 8];
        uint32_t qh[D / 16][4], ql[D / 16][4];
#pragma unroll
        for (int ks = 0; ks < D / 16; ks++) {
            const int r = wr * 16 + (lane & 15), c = 2 * ks + (lane >> 4);
            const uint32_t at = smem_u32(qs) + (c >> 3) * C::QHALF + r * 128 + (((c & 7) ^ (r & 7)) << 4);
            ldsm4(qh[ks], at);
            ldsm4(ql[ks], at + C::QROWS * D * 2);
        }
        fence_async_smem();

        float o[C::DW / 8][4];
#pragma unroll
        for (int i = 0; i < C::DW / 8; i++) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.0f;
        float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.0f, l1 = 0.0f;
        uint32_t v_exp = 0;                       // fp32: largest exponent of V so far; o is in units of its scale

        bool gave_up = false;
        for (int st = 0; st < nst; st++) {
            const uint32_t c = c0 + st;
            for (uint32_t n = 0; !mbar_try_wait(&s_full[c % C::NS], c / C::NS & 1) && !s_abort; n++) {
                if (n == kPaSpin) s_abort = 1;
                if (n > 64) __nanosleep(32);
            }
            __syncthreads();                      // the stage has landed; the slot before it is free
            if (s_abort) {                        // reported; the CTA's results are not valid. Its copies have 0.1 s to land before its memory goes.
                if (tid == 0) paged_err(a, QMS_PAGED_ETIMEOUT);
                for (int n = 0; n < 1 << 20; n++) __nanosleep(100);
                gave_up = true;
                break;
            }
            const int base = k0 + st * C::PS;
            if (st + C::NS - 1 < nst) {
                load(st + C::NS - 1);
                look_up(st + C::NS);
            }
            const int bad0 = s_bad[c & 3][0], bad1 = C::PS > 32 ? s_bad[c & 3][1] : 0;
            // some row does not see all of it: rows [first, seen] of the stage are seen by every row of the tile
            const int first = kmin, seen = bad0 | bad1 ? -1 : min(lo_pos, k1 - 1);
            const bool masked = base + C::PS - 1 > seen || base < first;
            unsigned char *raw = sm + c % C::NS * C::STAGE;
            uint32_t kb = sm0 + c % C::NS * C::STAGE, vb = kb + C::STAGE / 2;
            if constexpr (C::F16) {
                if (masked) {                     // behind the mask a weight is 0, but 0 * inf is not
                    for (int i = tid; i < C::PS * C::CH; i += 128) {
                        const int r = i / C::CH, p = base + r;
                        if (p >= first && p <= seen) continue;
                        uint4 *pv = reinterpret_cast<uint4 *>(raw + C::STAGE / 2 + C::piece(r, i % C::CH));
                        uint4 v = *pv;
                        if (drop_nonfinite((const KT *)nullptr, v)) {
                            *pv = v;
                            if (p >= first && p < k1) s_flag = 1;      // (else left over from before: nobody's)
                        }
                    }
                    fence_async_smem();
                    __syncthreads();
                }
            } else {
                // hi and lo: K by rows, each with a scale of its own (undone in its scores), V with the largest scale so
                // far of what somebody sees (o is in its units)
                constexpr int N = C::PS * C::CH / 128;             // 16-byte pieces of K (and of V) per thread
                const float4 *rk = reinterpret_cast<const float4 *>(raw), *rv = reinterpret_cast<const float4 *>(raw + C::STAGE / 2);
                // largest finite |value|: by float maxima, looked at again where one is inf (NaN is no maximum)
                auto largest = [](const float4 &y) { return fmaxf(max3(0.0f, fabsf(y.x), fabsf(y.y)), fmaxf(fabsf(y.z), fabsf(y.w))); };
                auto finite4 = [](const float4 &y) { return max(max(finite_bits(y.x), finite_bits(y.y)), max(finite_bits(y.z), finite_bits(y.w))); };
                float4 x[N];
                float mx = 0.0f;
#pragma unroll
                for (int i = 0; i < N; i++) x[i] = rv[tid + 128 * i];
                if (masked)
#pragma unroll
                    for (int i = 0; i < N; i++) {
                        const int r = (tid + 128 * i) / C::CH, p = base + r;
                        if (p >= first && p <= seen) continue;
                        uint4 v = *reinterpret_cast<const uint4 *>(&x[i]);
                        if (drop_nonfinite((const KT *)nullptr, v)) {
                            x[i] = *reinterpret_cast<const float4 *>(&v);
                            if (p >= first && p < k1) s_flag = 1;
                        }
                        if (p < first || p >= k1 || (bad0 >> r & 1)) x[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);    // no part of the unit
                    }
#pragma unroll
                for (int i = 0; i < N; i++) mx = fmaxf(mx, largest(x[i]));
                uint32_t mb = __float_as_uint(mx);
                if (mx == INFINITY) {
                    mb = 0;
#pragma unroll
                    for (int i = 0; i < N; i++) mb = max(mb, finite4(x[i]));       // (of what is part of the unit, as above)
                }
                mb = __reduce_max_sync(kFull, mb);
                if (lane == 0) s_max[warp] = mb;
                auto put = [&](int w, int at, float4 y, float up) {
                    const int r = at / C::CH, c = at % C::CH;      // values 4 c .. + 3 of row r
                    const float2 y0 = f2_mul(make_float2(y.x, y.y), make_float2(up, up)), y1 = f2_mul(make_float2(y.z, y.w), make_float2(up, up));
                    uint32_t h[2], l[2];
                    split_h2(y0.x, y0.y, h[0], l[0]);
                    split_h2(y1.x, y1.y, h[1], l[1]);
                    unsigned char *to = sm + C::CONV + w * 2 * C::HTILE + C::piece(r, c >> 1) + (c & 1) * 8;
                    *reinterpret_cast<uint2 *>(to) = make_uint2(h[0], h[1]);
                    *reinterpret_cast<uint2 *>(to + C::HTILE) = make_uint2(l[0], l[1]);
                };
                const unsigned peers = C::CH == 32 ? kFull : 0xffffu << (lane & 16);             // the lanes of a row
#pragma unroll
                for (int h = 0; h < N; h += 4) {
                    float4 y[4];
                    uint32_t ky[4];
#pragma unroll
                    for (int i = 0; i < 4; i++) y[i] = rk[tid + 128 * (h + i)];
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const float t = largest(y[i]);
                        ky[i] = __reduce_max_sync(peers, t == INFINITY ? finite4(y[i]) : __float_as_uint(t));
                    }
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const int at = tid + 128 * (h + i);
                        const uint32_t up = scale_up(ky[i] >> 23);
                        if (at % C::CH == 0) s_fk[at / C::CH] = pow2_bits(254u - up);
                        put(0, at, y[i], pow2_bits(up));
                    }
                }
                __syncthreads();
                const uint32_t ve = max(max(max(s_max[0], s_max[1]), max(s_max[2], s_max[3])) >> 23, v_exp);
                if (ve != v_exp) {
                    const uint32_t down = scale_up(v_exp) - scale_up(ve);
                    const float d = down > 126 ? 0.0f : pow2_bits(127u - down);
                    if (v_exp != 0)               // (before, o is 0)
#pragma unroll
                        for (int i = 0; i < C::DW / 8; i++) o[i][0] *= d, o[i][1] *= d, o[i][2] *= d, o[i][3] *= d;
                    v_exp = ve;
                }
#pragma unroll
                for (int i = 0; i < N; i++) put(1, tid + 128 * i, x[i], pow2_bits(scale_up(ve)));
                __syncthreads();
                kb = sm0 + C::CONV;
                vb = kb + 2 * C::HTILE;
            }

            // ---- scores
            float s[C::NT][4], s2[C::NT][4];
#pragma unroll
            for (int i = 0; i < C::NT; i++)
#pragma unroll
                for (int j = 0; j < 4; j++) s[i][j] = s2[i][j] = 0.0f;
#pragma unroll
            for (int ks = 0; ks < D / 16; ks++)
#pragma unroll
                for (int i = 0; i < C::NT / 2; i++) {
                    const int r = wk * C::KW + i * 16 + ((lane >> 4) << 3) + (lane & 7), c = 2 * ks + ((lane >> 3) & 1);
                    const uint32_t at = kb + C::piece(r, c);
                    uint32_t kf[4];
                    ldsm4(kf, at);
                    mma_f16(s[2 * i], qh[ks], kf[0], kf[1]);
                    mma_f16(s[2 * i + 1], qh[ks], kf[2], kf[3]);
                    mma_f16(s2[2 * i], ql[ks], kf[0], kf[1]);
                    mma_f16(s2[2 * i + 1], ql[ks], kf[2], kf[3]);
                    if constexpr (!C::F16) {
                        ldsm4(kf, at + C::HTILE);
                        mma_f16(s2[2 * i], qh[ks], kf[0], kf[1]);
                        mma_f16(s2[2 * i + 1], qh[ks], kf[2], kf[3]);
                    }
                }
            // ---- softmax of the stage: s becomes the weights
            float n0 = m0, n1 = m1;
#pragma unroll
            for (int i = 0; i < C::NT; i++) {
                const int r = wk * C::KW + i * 8 + tq * 2, p = base + r;
                const float2 fk = C::F16 ? make_float2(1.0f, 1.0f) : *reinterpret_cast<const float2 *>(s_fk + (C::F16 ? 0 : r));
                s[i][0] = (s[i][0] + s2[i][0]) * (f0 * fk.x), s[i][1] = (s[i][1] + s2[i][1]) * (f0 * fk.y);
                s[i][2] = (s[i][2] + s2[i][2]) * (f1 * fk.x), s[i][3] = (s[i][3] + s2[i][3]) * (f1 * fk.y);
                if (masked) {
                    const int bm = (r < 32 ? bad0 : bad1) >> (r & 31);
                    const bool ok0 = p >= first && p < k1 && !(bm & 1), ok1 = p + 1 >= first && p + 1 < k1 && !(bm & 2);
                    if (!ok0 || p > pos0) s[i][0] = -INFINITY;
                    if (!ok1 || p + 1 > pos0) s[i][1] = -INFINITY;
                    if (!ok0 || p > pos1) s[i][2] = -INFINITY;
                    if (!ok1 || p + 1 > pos1) s[i][3] = -INFINITY;
                }
                n0 = fmaxf(n0, fmaxf(s[i][0], s[i][1]));
                n1 = fmaxf(n1, fmaxf(s[i][2], s[i][3]));
            }
            n0 = fmaxf(n0, __shfl_xor_sync(kFull, n0, 1));
            n1 = fmaxf(n1, __shfl_xor_sync(kFull, n1, 1));
            n0 = fmaxf(n0, __shfl_xor_sync(kFull, n0, 2));
            n1 = fmaxf(n1, __shfl_xor_sync(kFull, n1, 2));
            const float b0 = n0 == -INFINITY ? 0.0f : n0 - kPaShift, b1 = n1 == -INFINITY ? 0.0f : n1 - kPaShift;
            if (n0 != m0 || n1 != m1) {
                const float d0 = m0 == -INFINITY ? 0.0f : ex2(m0 - n0), d1 = m1 == -INFINITY ? 0.0f : ex2(m1 - n1);
                l0 *= d0;
                l1 *= d1;
#pragma unroll
                for (int i = 0; i < C::DW / 8; i++) o[i][0] *= d0, o[i][1] *= d0, o[i][2] *= d1, o[i][3] *= d1;
            }
            m0 = n0;
            m1 = n1;
#pragma unroll
            for (int i = 0; i < C::NT; i++) {
                s[i][0] = ex2(s[i][0] - b0), s[i][1] = ex2(s[i][1] - b0);
                s[i][2] = ex2(s[i][2] - b1), s[i][3] = ex2(s[i][3] - b1);
                l0 += s[i][0] + s[i][1];
                l1 += s[i][2] + s[i][3];
            }
            // ---- o += weights * V. The tensor cores add by cutting bits off, towards 0; so they add up one stage, from 0, and its
            // sums join o by additions that round to nearest. In us, against sums over a whole unit (off by up to 8e-6): 64 tokens
            // over 4096 positions fp16 104, 105; 64 on a prompt of 1024 37.7, 37.5; 16 x 4 on 1000 29.4, 28.1; 8 x 4 on 2000 fp32
            // 42.4, 40.0.
            uint32_t ph[C::NT / 2][4], pl[C::NT / 2][4];
#pragma unroll
            for (int kk = 0; kk < C::NT / 2; kk++) {
                split_h2(s[2 * kk][0], s[2 * kk][1], ph[kk][0], pl[kk][0]);
                split_h2(s[2 * kk][2], s[2 * kk][3], ph[kk][1], pl[kk][1]);
                split_h2(s[2 * kk + 1][0], s[2 * kk + 1][1], ph[kk][2], pl[kk][2]);
                split_h2(s[2 * kk + 1][2], s[2 * kk + 1][3], ph[kk][3], pl[kk][3]);
            }
            constexpr int JS = C::F16 ? 2 : 1;    // 16-value columns at a time
#pragma unroll
            for (int j0 = 0; j0 < C::DW / 16; j0 += JS) {
                float t[2 * JS][4];
#pragma unroll
                for (int kk = 0; kk < C::NT / 2; kk++) {
                    const int r = wk * C::KW + kk * 16 + (((lane >> 3) & 1) << 3) + (lane & 7), c = wd * (C::DW / 8) + 2 * j0 + (lane >> 4);
                    uint32_t vf[JS][4];
#pragma unroll
                    for (int j = 0; j < JS; j++) ldsm4t(vf[j], vb + C::piece(r, c + 2 * j));
#pragma unroll
                    for (int j = 0; j < 2 * JS; j++) {
                        if (kk == 0) mma_f16_first(t[j], pl[kk], vf[j / 2][j % 2 * 2], vf[j / 2][j % 2 * 2 + 1]);
                        else mma_f16(t[j], pl[kk], vf[j / 2][j % 2 * 2], vf[j / 2][j % 2 * 2 + 1]);
                    }
#pragma unroll
                    for (int j = 0; j < 2 * JS; j++) mma_f16(t[j], ph[kk], vf[j / 2][j % 2 * 2], vf[j / 2][j % 2 * 2 + 1]);
                    if constexpr (!C::F16) {
#pragma unroll
                        for (int j = 0; j < JS; j++) ldsm4t(vf[j], vb + C::piece(r, c + 2 * j) + C::HTILE);
#pragma unroll
                        for (int j = 0; j < 2 * JS; j++) mma_f16(t[j], ph[kk], vf[j / 2][j % 2 * 2], vf[j / 2][j % 2 * 2 + 1]);
                    }
                }
#pragma unroll
                for (int j = 0; j < 2 * JS; j++) {
                    float(&x)[4] = o[2 * j0 + j];
                    const float2 lo = f2_add(make_float2(x[0], x[1]), make_float2(t[j][0], t[j][1])), hi = f2_add(make_float2(x[2], x[3]), make_float2(t[j][2], t[j][3]));
                    x[0] = lo.x, x[1] = lo.y, x[2] = hi.x, x[3] = hi.y;
                }
            }
        }
        if (gave_up) break;
        c0 += nst;
        __syncthreads();                          // every warp is done with the stages
        l0 += __shfl_xor_sync(kFull, l0, 1);
        l1 += __shfl_xor_sync(kFull, l1, 1);
        l0 += __shfl_xor_sync(kFull, l0, 2);
        l1 += __shfl_xor_sync(kFull, l1, 2);
        if constexpr (!C::F16) {                  // out of V's scale
            const float d = pow2_bits(254u - scale_up(v_exp));
#pragma unroll
            for (int i = 0; i < C::DW / 8; i++) o[i][0] *= d, o[i][1] *= d, o[i][2] *= d, o[i][3] *= d;
        }
        // dims of this thread's o[i][0..1] (row g) and o[i][2..3] (row g + 8)
        auto dim = [&](int i, int j) { return wd * C::DW + i * 8 + tq * 2 + (j & 1); };
        if (s_flag) {
            // V that were set aside: added where the row sees them (inf and NaN are not changed by a weight), by the group that
            // scored the position: the join leaves out groups that saw nothing
            for (int p = kmin; p < k1; p++) {
                if ((p - k0) % C::PS / C::KW != wk) continue;
                const int64_t at = paged_at(a, table, p);
                if (at < 0) continue;
                const KT *vr = reinterpret_cast<const KT *>(a.v + at + kh * a.head_stride);
#pragma unroll
                for (int i = 0; i < C::DW / 8; i++)
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        const float v = kv_ld(vr + dim(i, j));
                        if (!isfinite(v) && p <= (j < 2 ? pos0 : pos1)) o[i][j] += v;
                    }
            }
        }
        if (isnan(l0)) m0 = 0.0f;                 // scores that are all NaN leave no maximum, but are not nothing
        if (isnan(l1)) m1 = 0.0f;
        const int64_t po = (int64_t)slot * a.n_tok * a.H;
        const int tok0 = s_tok[wr * 16 + g], tok1 = s_tok[wr * 16 + g + 8];
        if constexpr (C::WK == 1) {
#pragma unroll
            for (int r = 0; r < 2; r++) {
                const int tok = r ? tok1 : tok0;
                const float m = r ? m1 : m0, l = r ? l1 : l0;
                if (tok < 0) continue;
                float *dst = A.part_o + (po + tok) * D;
#pragma unroll
                for (int i = 0; i < C::DW / 8; i++)
                    *reinterpret_cast<float2 *>(dst + dim(i, 0)) =
                        m == -INFINITY ? make_float2(0.0f, 0.0f) : make_float2(o[i][2 * r], o[i][2 * r + 1]);
                if (tq == 0) A.part_ml[po + tok] = make_float2(m == -INFINITY ? m : m - kPaShift, l);
            }
        } else {
            // join the position groups: group w's row r at red[(w * 16 WR + r)][D + 4]
            float *red = reinterpret_cast<float *>(sm);
            constexpr int LD = D + 4;            // rows on different banks; 8-byte pieces
#pragma unroll
            for (int r = 0; r < 2; r++) {
                float *dst = red + ((wk * WR + wr) * 16 + g + 8 * r) * LD;
#pragma unroll
                for (int i = 0; i < C::DW / 8; i++) *reinterpret_cast<float2 *>(dst + dim(i, 0)) = make_float2(o[i][2 * r], o[i][2 * r + 1]);
                if (tq == 0 && wd == 0) {
                    dst[D] = r ? m1 : m0;
                    dst[D + 1] = r ? l1 : l0;
                }
            }
            __syncthreads();
#pragma unroll
            for (int q = 0; q < 4 * WR; q++) {
                const int r = warp + 4 * q, tok = s_tok[r];
                float m = -INFINITY, l = 0.0f, x[D / 32], mk_[C::WK], w[C::WK];
#pragma unroll
                for (int k = 0; k < C::WK; k++) {
                    mk_[k] = red[(k * 16 * WR + r) * LD + D];
                    m = fmaxf(m, mk_[k]);
                }
#pragma unroll
                for (int k = 0; k < C::WK; k++) {
                    w[k] = mk_[k] == -INFINITY ? 0.0f : ex2(mk_[k] - m);
                    l = fmaf(w[k], red[(k * 16 * WR + r) * LD + D + 1], l);
                }
#pragma unroll
                for (int d = 0; d < D / 32; d++) {
                    x[d] = 0.0f;
#pragma unroll
                    for (int k = 0; k < C::WK; k++)            // (a group that saw nothing: its o may be 0 * inf)
                        x[d] = fmaf(w[k], mk_[k] == -INFINITY ? 0.0f : red[(k * 16 * WR + r) * LD + lane + 32 * d], x[d]);
                }
                if (tok < 0) continue;
#pragma unroll
                for (int d = 0; d < D / 32; d++) A.part_o[(po + tok) * D + lane + 32 * d] = x[d];
                if (lane == 0) A.part_ml[po + tok] = make_float2(m == -INFINITY ? m : m - kPaShift, l);
            }
        }
    }
    if (last) pdl_wait();
}

// ---- a row as it is defined --------------------------------------------------------------------------
// Row `row` (token * H + q head) of the output in plain fp32, by one warp: for rows whose weights' sum came out NaN. The two fp16
// terms of an operand make NaN of an infinite value (inf - inf, 0 * inf) also where the score is -inf and the weight 0. Reached by
// values that are not finite alone; a q that is not makes the row NaN in any case, and is left. False then.
template <typename T>
__device__ __forceinline__ void fetch_part(const T *src, float (&v)[4]) { *reinterpret_cast<float4 *>(v) = kv_ldg4(src); }
template <typename T>
__device__ __forceinline__ void fetch_part(const T *src, float (&v)[2]) { *reinterpret_cast<float2 *>(v) = kv_ldg2(src); }

template <int D>
__device__ __noinline__ bool plain_row(const PagedAttn &A, unsigned row) {
    constexpr int J = D / 32;
    float x[J];
    const Paged &a = A.a;
    const int lane = threadIdx.x & 31, t = row / (unsigned)a.H, h = row - t * a.H;
    float q[J], m = -INFINITY, l = 0.0f;
    int b = 0, t0, n, kv;
    while (b < a.n_seq && a.q_start[b + 1] <= t) b++;           // (one by one: paged_seq_of twice in a kernel costs each row)
    if (b == a.n_seq || !paged_seq(a, b, t0, n, kv) || t < t0) return false;
    fetch_part(A.q + t * A.ldq + (int64_t)h * D + lane * J, q);
    bool finite = true;
#pragma unroll
    for (int j = 0; j < J; j++) finite = finite && isfinite(q[j]), x[j] = 0.0f;
    if (!__all_sync(kFull, finite)) return false;
#pragma unroll 1
    for (int p = 0; p < kv - n + (t - t0) + 1; p++) {
        const int64_t at = paged_at(a, a.table + (p < a.prefix ? 0 : (int64_t)b * a.table_stride), p);
        if (at < 0) continue;
        const int64_t head = at + h / a.G * a.head_stride;
        float k[J], v[J], s = 0.0f;
        if (A.f16) {
            fetch_part(reinterpret_cast<const __half *>(a.k + head) + lane * J, k);
            fetch_part(reinterpret_cast<const __half *>(a.v + head) + lane * J, v);
        } else {
            fetch_part(reinterpret_cast<const float *>(a.k + head) + lane * J, k);
            fetch_part(reinterpret_cast<const float *>(a.v + head) + lane * J, v);
        }
#pragma unroll
        for (int j = 0; j < J; j++) s = fmaf(q[j], k[j], s);
        s = warp_sum(s) * A.scale2;
        const float f = s > m ? ex2(m - s) : 1.0f;              // (from -inf: 0)
        m = fmaxf(m, s);
        const float w = m == -INFINITY && !isnan(s) ? 0.0f : ex2(s - m);
        l = fmaf(l, f, w);
#pragma unroll
        for (int j = 0; j < J; j++) x[j] = fmaf(w, v[j], x[j] * f);
    }
#pragma unroll
    for (int j = 0; j < J; j++) A.out[t * A.ldo + (int64_t)h * D + lane * J + j] = x[j] / l;
    return true;
}

// ---- joining the slots of a row --------------------------------------------------------------------
// out = sum_s 2^(m_s - M) o_s / sum_s 2^(m_s - M) l_s over the slots of a (token, q head) row in their order; 0 where
// nothing was seen. WPR warps per row, each with every WPR-th slot; the loads of (m, l) and of the first slots go out
// before the row's length is known (what was not written is not used), so that the chain is one round trip.
// Bound by that latency for few rows, by the partial results' traffic (L2) for many.
template <int D, int WPR>
__global__ void __launch_bounds__(256) k_paged_merge(const __grid_constant__ PagedAttn A) {
    constexpr int J = D / 32, AHEAD = 4;
    __shared__ float s_x[WPR > 1 ? 8 : 1][D], s_l[8];
    const Paged &a = A.a;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, sub = warp % WPR;
    const unsigned row = blockIdx.x * (8 / WPR) + warp / WPR, t = row / (unsigned)a.H;
    const int64_t rows = (int64_t)a.n_tok * a.H;
    const int slots = A.p.slots_p + A.p.slots_s;
    pdl_trigger();
    pdl_wait();
    const bool there = row < rows;
    // the batch arrays, checked once for all kernels (rows or not: a sequence without any counts too)
    if (blockIdx.x == gridDim.x - 1)
        for (int b = threadIdx.x; b < a.n_seq; b += 256) {
            int t0, n, kv;
            if (!paged_seq(a, b, t0, n, kv)) paged_err(a, QMS_PAGED_ELEN);
        }
    // slot s of the row in the order of its use is at `at`; np: how many are of the shared positions
    int np = 0;
    auto at = [&](int s) { return (s < np ? s : s - np + A.p.slots_p) * rows + row; };
    auto fetch = [&](int64_t i, float (&v)[J]) {
        const float *src = A.part_o + i * D + lane * J;
        if constexpr (J == 4) *reinterpret_cast<float4 *>(v) = __ldcg(reinterpret_cast<const float4 *>(src));
        else *reinterpret_cast<float2 *>(v) = __ldcg(reinterpret_cast<const float2 *>(src));
    };
    float x[J], l = 0.0f;
#pragma unroll
    for (int j = 0; j < J; j++) x[j] = 0.0f;
    if (there) {
        // whatever the row's length: slot `lane`'s (m, l), and the first values of this warp's slots
        const float2 first = lane < slots ? __ldcg(&A.part_ml[lane * rows + row]) : make_float2(-INFINITY, 0.0f);
        float v[AHEAD][J];
#pragma unroll
        for (int i = 0; i < AHEAD; i++)
            if (sub + WPR * i < slots) fetch((sub + WPR * i) * rows + row, v[i]);
        int t0 = 0, n = 0, kv = 0;
        const int b = paged_seq_of(a, t);
        if (b < a.n_seq) paged_seq(a, b, t0, n, kv);
        const int pos = (int)t >= t0 && (int)t < t0 + n ? kv - n + ((int)t - t0) : -1;
        if (pos >= 0) {                           // the slots of chunks that begin past the row's position are not written
            if (a.prefix > 0) {
                const int d = min(pos, a.prefix - 1);
                if (A.p.line > 0) {
                    const unsigned h = row - t * a.H, kh = h / a.G;
                    const unsigned y = ((t * a.G + h - kh * a.G) / (unsigned)A.p.line_rows * a.Hk + kh) * A.p.line_nt;
                    np = line_run(A.p, y + d / (unsigned)A.p.line_tp) - line_run(A.p, y) + 1;
                } else {
                    np = d / A.p.chunk_p + 1;
                }
            }
            const int ns = np + (pos < a.prefix ? 0 : (pos - A.p.base_s) / A.p.chunk_s + 1);
            const bool dense = np == A.p.slots_p || ns == np;              // slot s is where the fetch above took it
            float M = -INFINITY;
            float2 ml = make_float2(-INFINITY, 0.0f);
            for (int s0 = 0; s0 < ns; s0 += 32) {
                const float2 y = s0 + lane >= ns ? make_float2(-INFINITY, 0.0f) : s0 == 0 && dense ? first : __ldcg(&A.part_ml[at(s0 + lane)]);
                if (s0 == 0) ml = y;
                M = fmaxf(M, y.x);
            }
            M = warp_max(M);
            if (M != -INFINITY) {
                for (int s0 = 0; s0 < ns; s0 += 32) {
                    if (s0 > 0) ml = s0 + lane < ns ? __ldcg(&A.part_ml[at(s0 + lane)]) : make_float2(-INFINITY, 0.0f);
                    const float w = ex2(ml.x - M);
                    if (sub == 0) l += w * (ml.x == -INFINITY ? 0.0f : ml.y);
                    const int ne = min(32, ns - s0);
                    int i = sub;
                    if (s0 == 0 && dense) {
#pragma unroll
                        for (int k = 0; k < AHEAD; k++, i += WPR) {
                            const float wi = __shfl_sync(kFull, w, i & 31);
                            if (i < ne)
#pragma unroll
                                for (int j = 0; j < J; j++) x[j] = fmaf(wi, v[k][j], x[j]);
                        }
                    }
#pragma unroll 8
                    for (; i < ne; i += WPR) {
                        const float wi = __shfl_sync(kFull, w, i);
                        float y[J];
                        fetch(at(s0 + i), y);
#pragma unroll
                        for (int j = 0; j < J; j++) x[j] = fmaf(wi, y[j], x[j]);
                    }
                }
            }
        }
    }
    if (sub == 0) l = warp_sum(l);
    if constexpr (WPR > 1) {
#pragma unroll
        for (int j = 0; j < J; j++) s_x[warp][lane * J + j] = x[j];
        if (sub == 0 && lane == 0) s_l[warp] = l;
        __syncthreads();
        if (sub != 0) return;
#pragma unroll
        for (int k = 1; k < WPR; k++)
#pragma unroll
            for (int j = 0; j < J; j++) x[j] += s_x[warp + k][lane * J + j];
    }
    if (!there) return;
    float *dst = A.out + t * A.ldo + (int64_t)(row - t * a.H) * D + lane * J;
    if (__any_sync(kFull, isnan(l)) && plain_row<D>(A, row)) return;
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    if constexpr (J == 4) *reinterpret_cast<float4 *>(dst) = l == 0.0f ? make_float4(0.0f, 0.0f, 0.0f, 0.0f) : make_float4(x[0] * inv, x[1] * inv, x[2] * inv, x[3] * inv);
    else *reinterpret_cast<float2 *>(dst) = l == 0.0f ? make_float2(0.0f, 0.0f) : make_float2(x[0] * inv, x[1] * inv);
}

// ---- host ------------------------------------------------------------------------------------------
// Rows per tile: 16, 32 or 64 for k_paged_attn, as tall as the rows there are (more rows per K / V read); k_paged_wide
// from 65 on (fp16: in pages of 8 positions or more, a swizzle unit of its tiles) and from so many rows x positions (`rows`
// by the 64, over all units) that its longer start pays. Narrow against wide in us, 16 q heads per kv head, 4 of these:
// 80 rows x 16 sequences x 1000 positions 40.9, 26.5 (fp32 74.2, 47.1); 64 rows of the same 27.8, 26.1 (44.6, 45.6). By millions
// of rows x positions: 8 sequences of 5 tokens, own positions 1.2 narrow 17.6, wide 19.5 (22.2, 21.4); 1.8 19.5, 19.2 (26.1, 28.1); 2.5
// 21.8, 18.4 (29.8, 27.2); 4.1 25.9, 19.6 (42.3, 31.0); 20 tokens on a prompt, shared ones 1.6 23.4, 25.1 (35.4, 36.9); 2.0 27.8, 27.2 (38.0,
// 37.7); 3.1 31.3, 35.1 (45.7, 46.5); 6.3 39.8, 43.5 (65.8, 58.2); 16.8 69, 63 (139, 96).
static int row_groups(int type, int page_log, int64_t rows, int64_t positions, bool shared) {
    const bool f16 = type == QMS_T_F16;
    if (rows > 64 && (!f16 || page_log >= 3) && (rows + 63) / 64 * 64 * positions > (f16 || shared ? 2600000 : 1200000))
        return !f16 ? kPaWideF32 : rows > 128 ? kPaWidePair : kPaWideSplit;
    return rows > 32 ? 4 : rows > 16 ? 2 : 1;
}
static int tile_rows(int wr) { return wr == kPaWidePair ? 256 : wr < 0 ? 128 : 16 * wr; }
static int tile_positions(int type, int wr) { return wr > 0 ? pa_stage(type) : wr == kPaWideF32 ? 64 : 128; }

// Positions that one unit of k_paged_wide may cover, by the additions into an accumulator (its CUT): fp16 144 of them, 2 per 16
// positions; fp32 192, 3 per 16, by two streams. (kPaWidePair takes its own out in time; k_paged_attn adds up single stages.)
static int most_positions(int wr) { return wr == kPaWideSplit ? 2304 : wr == kPaWideF32 ? 2048 : 1 << 30; }

// Chunks of `len` positions for `tiles` units of rows: the number of chunks with the least estimated time, from waves
// of resident CTAs, stages of `stage` positions (us each, us_unit once per unit) and 1 KB of partial results
// written and read back per row and chunk.
static int chunk_of(int len, int64_t tiles, int64_t rows, int stage, int resident, double us_stage, double us_unit, int cap) {
    const int st = (len + stage - 1) / stage, most = std::min(st, cap / stage);
    int best = most;
    double least = 1e30;
    for (int per = most; per >= 1; per = per > 64 ? per - per / 16 : per - 1) {
        const int n = (st + per - 1) / per;
        const int64_t waves = (tiles * n + resident - 1) / resident;
        const double us = (double)waves * (per * us_stage + us_unit) + (double)rows * n * 2.0e-4;
        if (us < least) least = us, best = per;
    }
    return (best > 0 ? best : 1) * stage;
}

// share: what these units have of the SMs' room beside those of the other kind
static int chunk_for(int type, int wr, int len, int64_t tiles, int64_t rows, double share) {
    const int tp = tile_positions(type, wr), most = most_positions(wr);
    if (wr == kPaWidePair) return chunk_of(len, tiles, rows, tp, 148, 3.0, 8.0, most);
    if (wr <= 0) return chunk_of(len, tiles, rows, tp, 148, 1.5, 8.0, most);
    const int per_sm = type == QMS_T_F16 && wr == 1 ? 3 : 2;
    return chunk_of(len, tiles, rows, tp, std::max(1, (int)(148 * per_sm * share)), wr == 4 ? 2.0 : 1.2, 4.0, most);
}

void paged_plan(const Paged &a, int type, int D, PagedPlan &p) {
    const int64_t rows_p = (int64_t)a.n_tok * a.G, rows_s = (int64_t)a.max_q * a.G, all = (int64_t)a.n_tok * a.H;
    memset(&p, 0, sizeof p);
    p.wr_p = row_groups(type, a.page_log, rows_p, (int64_t)a.prefix * a.Hk, true);
    p.wr_s = row_groups(type, a.page_log, rows_s, (int64_t)std::max(0, a.max_kv - a.prefix) * a.Hk * a.n_seq, false);
    p.base_s = a.prefix & ~(std::min(1 << a.page_log, tile_positions(type, p.wr_s)) - 1);
    const int own = std::max(0, a.max_kv - p.base_s);
    p.tiles_p = (int)((rows_p + tile_rows(p.wr_p) - 1) / tile_rows(p.wr_p));
    p.tiles_s = (int)((rows_s + tile_rows(p.wr_s) - 1) / tile_rows(p.wr_s));
    // k_paged_attn for both kinds: they run beside each other, and each is cut for its share of the SMs by the work, though not
    // less than 0.35 (its tail would hold the other up). With a share of 1 each, and so, in us: 23 x 3 tokens on 1001 + 701
    // positions, fp32, 53.0, 47.5; 8 tokens on 1000 + 1000 26.5, 20.7; 4 x 3 on 2000 + 2000 35.1, 27.3; 48 tokens on 200 + 2000
    // 65.3, 65.3 (73.0 without the 0.35).
    const double work_p = (double)p.tiles_p * a.prefix * (p.wr_p == 4 ? 2.0 : 1.2), work_s = (double)p.tiles_s * a.n_seq * own * (p.wr_s == 4 ? 2.0 : 1.2);
    const double share = p.wr_p > 0 && p.wr_s > 0 && work_p > 0 && work_s > 0 ? work_p / (work_p + work_s) : -1.0;
    p.chunk_p = chunk_for(type, p.wr_p, a.prefix, (int64_t)p.tiles_p * a.Hk, all, share < 0 ? 1.0 : std::max(share, 0.35));
    p.chunk_s = chunk_for(type, p.wr_s, own, (int64_t)p.tiles_s * a.Hk * a.n_seq, all, share < 0 ? 1.0 : std::max(1.0 - share, 0.35));
    p.slots_p = p.chunks_p = (a.prefix + p.chunk_p - 1) / p.chunk_p;
    p.slots_s = p.chunks_s = (own + p.chunk_s - 1) / p.chunk_s;
    if (p.wr_p <= 0 && p.chunks_p > 0 && p.tiles_p > 0) {
        p.line_tp = tile_positions(type, p.wr_p);
        p.line_rows = tile_rows(p.wr_p);
        const int64_t nt = (a.prefix + p.line_tp - 1) / p.line_tp, line = nt * p.tiles_p * a.Hk;
        const int64_t ctas = std::min<int64_t>(148, line), most = most_positions(p.wr_p) / p.line_tp;
        p.line = (unsigned)line;
        p.line_nt = (unsigned)nt;
        p.line_per = (unsigned)((line + ctas * most - 1) / (ctas * most));
        p.line_runs = (unsigned)(p.line_per * ctas);
        p.line_q = p.line / p.line_runs;
        p.line_r = p.line % p.line_runs;
        // a row tile's positions meet at most this many runs
        p.slots_p = (int)std::min<int64_t>(nt, (nt - 1) / p.line_q + 2);
    }
}

static int64_t al256(int64_t x) { return (x + 255) & ~(int64_t)255; }

int64_t paged_ws_bytes(const Paged &a, int D, const PagedPlan &p) {
    const int64_t n = (int64_t)(p.slots_p + p.slots_s) * a.n_tok * a.H;
    return al256(n * D * 4) + al256(n * 8);
}

int paged_map(const Paged &a, int D, bool f16, int rows, const char *pool, CUtensorMap *map) {
    typedef CUresult (*Encode)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *, const cuuint32_t *,
                               const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
    static std::atomic<Encode> known{nullptr};
    Encode encode = known.load();
    if (!encode) {
        cudaDriverEntryPointQueryResult found;
        void *f = nullptr;
        QMS_CK(cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &found));
        QMS_REQUIRE(f, QMS_CUDA_ECUDA, "paged_attention: the driver has no cuTensorMapEncodeTiled");
        known = encode = (Encode)f;
    }
    const cuuint64_t ps = 1ull << a.page_log, row = (cuuint64_t)D * (f16 ? 2 : 4);
    const cuuint64_t dim[4] = {(cuuint64_t)D, (cuuint64_t)a.Hk, ps, (cuuint64_t)a.n_pages};
    // (the stride of a dimension of one has no meaning, and 0 none that the encoder takes)
    const cuuint64_t stride[3] = {a.Hk > 1 ? (cuuint64_t)a.head_stride : row, ps > 1 ? (cuuint64_t)a.pos_stride : row,
                                  a.n_pages > 1 ? (cuuint64_t)a.page_stride : row};
    const cuuint32_t box[4] = {f16 ? 64u : (cuuint32_t)D, 1, (cuuint32_t)std::min<cuuint64_t>(ps, rows), 1}, one[4] = {1, 1, 1, 1};
    const CUresult rc = encode(map, f16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 4, (void *)pool, dim, stride, box, one,
                               CU_TENSOR_MAP_INTERLEAVE_NONE, f16 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_NONE,
                               CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    QMS_REQUIRE(rc == CUDA_SUCCESS, QMS_CUDA_EINVAL, "paged_attention: the pool's strides do not make a tensor map (%d)", (int)rc);
    return QMS_CUDA_OK;
}

template <int D, typename KT, int WR>
static int launch_attn_wr(const PagedAttn &A, bool own, bool last, cudaStream_t s) {
    using C = PaCfg<D, KT, WR>;
    const int64_t units = own ? (int64_t)A.p.chunks_s * A.a.n_seq * A.p.tiles_s * A.a.Hk : (int64_t)A.p.chunks_p * A.p.tiles_p * A.a.Hk;
    QMS_REQUIRE(units < (1ll << 30), QMS_CUDA_EUNSUPPORTED, "paged_attention: too many units of work");
    static std::atomic<unsigned long long> done{0};
    int rc = allow_smem(done, k_paged_attn<D, KT, WR>, C::SMEM);
    if (rc) return rc;
    CUtensorMap mk, mv;
    rc = paged_map(A.a, D, C::F16, C::PS, A.a.k, &mk);
    if (rc || (rc = paged_map(A.a, D, C::F16, C::PS, A.a.v, &mv))) return rc;
    const int grid = (int)std::min<int64_t>(units, 148 * 8);
    QMS_CK(launch_pdl(k_paged_attn<D, KT, WR>, dim3(grid), dim3(128), C::SMEM, s, A, mk, mv, own, last));
    return QMS_CUDA_OK;
}

template <int D, typename KT>
static int launch_attn(const PagedAttn &A, cudaStream_t s) {
    bool before = false;
    for (int kind = 0; kind < 2; kind++) {
        const bool own = kind == 1;
        if (own ? !(A.p.chunks_s && A.p.tiles_s && A.a.n_seq) : !(A.p.chunks_p && A.p.tiles_p)) continue;
        const int wr = own ? A.p.wr_s : A.p.wr_p;
        const int rc = wr <= 0   ? launch_paged_wide(A, D, own, before, s)
                       : wr == 4 ? launch_attn_wr<D, KT, 4>(A, own, before, s)
                       : wr == 2 ? launch_attn_wr<D, KT, 2>(A, own, before, s)
                                 : launch_attn_wr<D, KT, 1>(A, own, before, s);
        if (rc) return rc;
        before = true;
    }
    return QMS_CUDA_OK;
}

int launch_paged_attention(const Paged &a, int type, int D, const PagedPlan &p, const float *q, int64_t ldq, float scale,
                           float *out, int64_t ldo, void *ws, cudaStream_t s) {
    PagedAttn A;
    memset(&A, 0, sizeof A);
    A.a = a;
    A.p = p;
    A.q = q;
    A.out = out;
    A.ldq = ldq;
    A.ldo = ldo;
    A.scale2 = scale * 1.4426950408889634f;
    A.f16 = type == QMS_T_F16;
    A.part_o = (float *)ws;
    // (32-bit run arithmetic)
    QMS_REQUIRE((int64_t)p.tiles_p * a.Hk * ((a.prefix + 63) / 64) < (1ll << 31), QMS_CUDA_EUNSUPPORTED, "paged_attention: too many units of work");
    A.part_ml = (float2 *)((char *)ws + al256((int64_t)(p.slots_p + p.slots_s) * a.n_tok * a.H * D * 4));
    int rc;
    if (type == QMS_T_F16) rc = D == 128 ? launch_attn<128, __half>(A, s) : launch_attn<64, __half>(A, s);
    else rc = D == 128 ? launch_attn<128, float>(A, s) : launch_attn<64, float>(A, s);
    if (rc) return rc;
    // Four warps per row while there are few rows, or many slots for each. Four against one in us: 320 rows (5 tokens, 2000
    // positions) 14.9, 16.1; 512 rows on a prompt of 4096 positions 24.7, 28.9; 1024 rows of 100 positions 11.5, 9.1; 3072 rows
    // of 1000 positions 28.3, 25.2.
    const int64_t rows = (int64_t)a.n_tok * a.H;
    const int wpr = rows <= 4 * 148 || p.slots_p + p.slots_s > 32 ? 4 : 1;
    const dim3 grid((unsigned)((rows * wpr + 7) / 8));
    if (D == 128) {
        if (wpr == 4) QMS_CK(launch_pdl(k_paged_merge<128, 4>, grid, dim3(256), 0, s, A));
        else QMS_CK(launch_pdl(k_paged_merge<128, 1>, grid, dim3(256), 0, s, A));
    } else {
        if (wpr == 4) QMS_CK(launch_pdl(k_paged_merge<64, 4>, grid, dim3(256), 0, s, A));
        else QMS_CK(launch_pdl(k_paged_merge<64, 1>, grid, dim3(256), 0, s, A));
    }
    return QMS_CUDA_OK;
}

}  // namespace qms
