// qms_paged_q4.cu - attention of few rows over a paged KV cache in 4 bits on B200 (sm_100a): up to 16 rows per tile (one token of
// 16 q heads on a kv head), several tiles while they are few. More rows: qms_paged_attn.cu, qms_paged_wide.cu.
//
// K and V go from nibbles straight into the registers that mma.sync m16n8k16 wants them in, never to fp16 in shared memory. A product's
// operands may have the head's values, and the positions, in any order that is the same on both sides, so that
//   K (B operand, 8 positions x 16 values)  a thread takes 32 values (16 at head_dim 64) of one position that lie together: one load
//       of 16 bytes, one scale, and the 16 pairs that come out of it are its registers for all steps; q has that order too
//   V (B operand, 16 positions x 8 values)  a thread takes 16 values (8) of four positions; pairs of two positions' values are made
//       by a byte permutation before the nibbles are cut out
// A nibble becomes d (n - 8) by a shift, a mask and one fused step, exact in fp16 (q4_dequant). q and the weights have two terms,
// sums join by rounded additions, as in k_paged_attn. Each warp has positions of its own, in tiles of 16 in turn, its own copies in
// flight and its own (m, l, o); they meet at the end of a unit.
// Bound by instructions: some 1140 per warp for 32 positions (4.6 KB), 128 of them MMAs (the tensor pipe is busy for 41 % of the time), 350 for what
// comes out of the nibbles, where most steps wait for the one before them. 64 sequences of 4096 positions (64 q heads, 4 kv heads) 89 us, 1.69 TB/s; one
// of 131,072 (32 q heads) 48.0, 1.57 TB/s; one of 1100 9.8, of which some 4 are the launch and 4 the join of the slots. A third stage of copies changed nothing.
// The same with K and V's transpose as tcgen05's M operand, 128 positions or values, and the rows as its N: 110 us and 55, by the way of K and
// V through shared memory in fp16 (164 KB in and out for 18 that are read).
#include <math.h>
#include <string.h>

#include "qms_moe.cuh"
#include "qms_paged.cuh"

namespace qms {

constexpr float kQ4Shift = 8.0f, kQ4High = 7.0f;      // weights reach 2^8, from there up to 2^15: their fp16 low terms stay clear of the subnormals

__device__ __forceinline__ void mma_16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_16_first(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));
}
// The pair of nibbles at bits 4 e and 16 + 4 e as d (n - 8). six: 0x4C004C00, in a register (two constants in one step need one).
__device__ __forceinline__ uint32_t q4_pair(uint32_t w, int e, __half2 d, __half2 m24, uint32_t six) {
    uint32_t x;
    asm("lop3.b32 %0, %1, 0x03C003C0, %2, 0xEA;" : "=r"(x) : "r"(e == 0 ? w << 6 : e == 1 ? w << 2 : e == 2 ? w >> 2 : w >> 6), "r"(six));
    const __half2 y = __hfma2(*reinterpret_cast<const __half2 *>(&x), d, m24);
    return *reinterpret_cast<const uint32_t *>(&y);
}

template <int D>
struct Q4Cfg {
    static constexpr int NIB = 16 * (D / 2), SC = 16 * (D / 16), TILE = NIB + SC;      // bytes of a tile of 16 positions, of K or of V
    static constexpr int STAGE = 4 * TILE, NS = 2;                                      // two tiles of K and V; stages per warp
    static constexpr int RING = 4 * NS * STAGE;
    static constexpr int LD = D / 8 * 9 + 2;                                            // the warps' o, m, l: 9 per 8 values (banks)
    static constexpr int RED = 4 * 16 * LD * 4, Q = (RING > RED ? RING : RED) + 127 & ~127;
    static constexpr int SMEM = Q + D / 16 * 2 * 512 + 128;                             // q as A operands: [step][hi, lo][lane]
};

template <int D, int PER_SM>
__global__ void __launch_bounds__(128, PER_SM) k_paged_q4(const PagedAttn A, const bool own, const bool last) {
    using C = Q4Cfg<D>;
    constexpr int KS = D / 16, W = D / 32, VW = D / 64;      // steps of 16 values; words of K per thread and position, of V
    extern __shared__ unsigned char sm_[];
    __shared__ int s_pos[16], s_tok[16];          // position of each row of the tile; token row * H + q head (-1: none)
    __shared__ int s_flag;                        // V had values that are not finite behind the mask
    const Paged &a = A.a;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, tq = lane & 3;
    unsigned char *sm = sm_ + (-smem_u32(sm_) & 127);
    unsigned char *ring = sm + warp * C::NS * C::STAGE;
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
        int b = 0, part, k0, k1, t0 = 0, n = 0, kv = 0;
        if (own) {
            b = u % a.n_seq;
            part = u / a.n_seq;
            paged_seq(a, b, t0, n, kv);
            k0 = A.p.base_s + part * A.p.chunk_s;
            k1 = min(kv, k0 + A.p.chunk_s);
            if (max(k0, a.prefix) >= k1 || tile * 16 >= n * a.G) continue;
            part += A.p.slots_p;
        } else {
            part = u;
            k0 = part * A.p.chunk_p;
            k1 = min(a.prefix, k0 + A.p.chunk_p);
        }
        const int *table = a.table + (own ? (int64_t)b * a.table_stride : 0);
        const int kmin = own ? max(k0, a.prefix) : k0, r0 = tile * 16;
        __syncthreads();                          // the previous unit is done with shared memory
        if (tid == 0) s_flag = 0;
        if (own) {
            if (tid < 16) {
                const int r = r0 + tid, i = r / a.G;
                s_pos[tid] = i < n ? kv - n + i : -1;
                s_tok[tid] = i < n ? (t0 + i) * a.H + kh * a.G + (r - i * a.G) : -1;
            }
        } else {
            const int first = r0 / a.G, end = min(a.n_tok, (r0 + 16 + a.G - 1) / a.G);
            for (int t = first + warp; t < end; t += 4) {
                int s0 = 0, sn = 0, skv = 0;
                const int sb = paged_seq_of(a, t);
                if (sb < a.n_seq) paged_seq(a, sb, s0, sn, skv);
                const int pos = t >= s0 && t < s0 + sn ? skv - sn + (t - s0) : -1;
                for (int j = lane; j < a.G; j += 32) {
                    const int r = t * a.G + j - r0;
                    if (r >= 0 && r < 16) {
                        s_pos[r] = pos;
                        s_tok[r] = t * a.H + kh * a.G + j;
                    }
                }
            }
            if (tid < 16 && r0 + tid >= a.n_tok * a.G) s_pos[tid] = s_tok[tid] = -1;
        }
        __syncthreads();
        const int pos_l = s_pos[lane & 15];
        const int hi_pos = __reduce_max_sync(kFull, pos_l), lo_pos = __reduce_min_sync(kFull, pos_l < 0 ? 0x7fffffff : pos_l);
        if (kmin > hi_pos) continue;              // nobody sees any of it (the same for all warps)
        const int k_end = min(k1, hi_pos + 1), nst = (k_end - k0 - warp * 16 + 127) / 128;       // stages in which this warp has positions
        // A stage: tile 0, positions k0 + 128 st + 16 warp .. + 15, and tile 1, 64 further; each lies in one page. Which tiles there are,
        // and on good pages, is kept in bits 2 (st % 16) on. Plain asynchronous copies: eight bulk copies of 128 bytes to 1 KB per stage
        // were what the kernel waited for.
        uint32_t tiles = 0;
        int page = -1;                            // lane x: of tile x
        auto look_up = [&](int st) {
            const int p = k0 + st * 128 + (lane & 1) * 64 + warp * 16;
            page = lane < 2 && st < nst && p < k_end ? table[p >> a.page_log] : -2;            // -2: nothing there
        };
        auto load = [&](int st, uint32_t at) {    // (its pages have been looked up)
            const bool there = (unsigned)page < (unsigned)a.n_pages;
            if (page != -2 && !there) paged_err(a, QMS_PAGED_EPAGE);
            const uint32_t two = __ballot_sync(kFull, there) & 3;
            tiles = (tiles & ~(3u << 2 * (st & 15))) | two << 2 * (st & 15);
            unsigned char *to = ring + at * C::STAGE;
            int64_t from[2];                      // where a tile's page and head start
            int y[2];
#pragma unroll
            for (int x = 0; x < 2; x++) {
                from[x] = __shfl_sync(kFull, page, x) * a.page_stride + kh * a.head_stride;
                y[x] = (k0 + st * 128 + x * 64 + warp * 16) & ((1 << a.page_log) - 1);
                if (!(two >> x & 1)) continue;
#pragma unroll
                for (int v = 0; v < 2; v++)
#pragma unroll
                    for (int c = 0; c < C::NIB / 512; c++)
                        cp_async16(to + (2 * x + v) * C::TILE + c * 512 + lane * 16, (v ? a.v : a.k) + from[x] + y[x] * (D / 2) + c * 512 + lane * 16);
            }
            constexpr int N = C::SC / 16;         // 16-byte pieces of a tile's scales
            const int x = lane / (2 * N), v = lane / N & 1, c = lane % N;
            if (lane < 4 * N && (two >> x & 1))
                cp_async16(to + (2 * x + v) * C::TILE + C::NIB + c * 16, (v ? a.v : a.k) + from[x] + (D / 2 << a.page_log) + y[x] * (D / 16) + c * 16);
        };
        look_up(0);
        if (nst > 0) load(0, 0);
        asm volatile("cp.async.commit_group;" ::: "memory");
        look_up(1);
        // ---- q: rows g and g + 8, this thread's D / 4 values of each; a row scaled by a power of two into fp16's range (undone in the
        // score's factor) and split
        // (warp w: steps w, w + 4)
        float f[2];
        int pos[2];
        uint32_t qs[KS / 4][2][4];
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const int tok = s_tok[g + 8 * h], t = tok < 0 ? 0 : tok / a.H;
            const float4 *src = reinterpret_cast<const float4 *>(A.q + t * A.ldq + (int64_t)(tok < 0 ? 0 : tok - t * a.H) * D + tq * (D / 4));
            pos[h] = s_pos[g + 8 * h];
            float4 x[KS];
            uint32_t mx = 0;
#pragma unroll
            for (int k = 0; k < KS; k++) x[k] = tok < 0 ? make_float4(0.0f, 0.0f, 0.0f, 0.0f) : __ldcg(src + (k + warp) % KS);
#pragma unroll
            for (int k = 0; k < KS; k++) mx = max(mx, max(max(finite_bits(x[k].x), finite_bits(x[k].y)), max(finite_bits(x[k].z), finite_bits(x[k].w))));
            mx = max(mx, __shfl_xor_sync(kFull, mx, 1));
            mx = max(mx, __shfl_xor_sync(kFull, mx, 2));
            const uint32_t up = scale_up(mx >> 23);
            f[h] = A.scale2 * pow2_bits(254u - up);
            const float m = pow2_bits(up);
#pragma unroll
            for (int k = 0; k < KS / 4; k++) {    // values 4 k .. 4 k + 3 of step k: its two pairs
                split_h2(x[4 * k].x * m, x[4 * k].y * m, qs[k][0][h], qs[k][1][h]);
                split_h2(x[4 * k].z * m, x[4 * k].w * m, qs[k][0][2 + h], qs[k][1][2 + h]);
            }
        }
        uint4 *s_q = reinterpret_cast<uint4 *>(sm + C::Q);
#pragma unroll
        for (int k = 0; k < KS / 4; k++)
#pragma unroll
            for (int e = 0; e < 2; e++) s_q[((4 * k + warp) * 2 + e) * 32 + lane] = make_uint4(qs[k][e][0], qs[k][e][1], qs[k][e][2], qs[k][e][3]);
        __syncthreads();
        s_q += lane;
        float o[D / 8][4];                        // value 16 n + i (D 64: 8 n + i) of rows g, g + 8 in o[i], n = 2 tq, 2 tq + 1
#pragma unroll
        for (int i = 0; i < D / 8; i++) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.0f;
        float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.0f, l1 = 0.0f;
        uint32_t six;
        asm volatile("mov.b32 %0, 0x4C004C00;" : "=r"(six));
#pragma unroll 1
        for (int st = 0; st < nst; st++) {
            __syncwarp();                         // (the other slot was read in the last round)
            if (st + 1 < nst) {
                load(st + 1, st + 1 & 1);
                look_up(st + 2);
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
            asm volatile("cp.async.wait_group 1;" ::: "memory");
            __syncwarp();
            const uint32_t there = tiles >> 2 * (st & 15);
            const int base = k0 + st * 128 + warp * 16;        // tile x: positions base + 64 x ..
            const unsigned char *stage = ring + (st & 1) * C::STAGE;
            // ---- scores: column c of 8-position tile i is position 64 (i / 2) + 8 (i % 2) + (c >> 1) + 4 (c & 1) from base on
            float s[4][4], s2[4][4];
            {
                uint32_t w[4][W];
                __half2 d[4], m24[4];
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const unsigned char *kn = stage + (i >> 1) * 2 * C::TILE;
                    const int r = 8 * (i & 1) + (g >> 1) + 4 * (g & 1);
                    if constexpr (D == 128) *reinterpret_cast<uint4 *>(w[i]) = *reinterpret_cast<const uint4 *>(kn + r * 64 + tq * 16);
                    else *reinterpret_cast<uint2 *>(w[i]) = *reinterpret_cast<const uint2 *>(kn + r * 32 + tq * 8);
                    d[i] = __half2half2(reinterpret_cast<const __half *>(kn + C::NIB)[r * (D / 32) + (D == 128 ? tq : tq >> 1)]);
                    m24[i] = __hmul2(d[i], __float2half2_rn(-24.0f));
                }
#pragma unroll
                for (int k = 0; k < KS; k++) {
                    const uint4 h4 = s_q[(2 * k) * 32], l4 = s_q[(2 * k + 1) * 32];
                    const uint32_t qh[4] = {h4.x, h4.y, h4.z, h4.w}, ql[4] = {l4.x, l4.y, l4.z, l4.w};
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const uint32_t b0 = q4_pair(w[i][k / 2], 2 * (k & 1), d[i], m24[i], six);
                        const uint32_t b1 = q4_pair(w[i][k / 2], 2 * (k & 1) + 1, d[i], m24[i], six);
                        if (k == 0) {
                            mma_16_first(s[i], qh, b0, b1);
                            mma_16_first(s2[i], ql, b0, b1);
                        } else {
                            mma_16(s[i], qh, b0, b1);
                            mma_16(s2[i], ql, b0, b1);
                        }
                    }
                }
            }
            // some row does not see all of it
            const int seen = (there & 3) == 3 ? min(lo_pos, k1 - 1) : -1;
            const bool masked = base + 79 > seen || base < kmin;
            auto gone = [&](int x, int p) { return !(there >> x & 1) || p < kmin || p >= k1; };      // a position of tile x that is no part of it
            float n0 = -INFINITY, n1 = -INFINITY;
#pragma unroll
            for (int i = 0; i < 4; i++) {
#pragma unroll
                for (int j = 0; j < 4; j++) s[i][j] = (s[i][j] + s2[i][j]) * f[j >> 1];
                if (masked) {
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        const int p = base + 64 * (i >> 1) + 8 * (i & 1) + tq + 4 * (j & 1);
                        if (gone(i >> 1, p) || p > pos[j >> 1]) s[i][j] = -INFINITY;
                    }
                }
                n0 = fmaxf(n0, fmaxf(s[i][0], s[i][1]));
                n1 = fmaxf(n1, fmaxf(s[i][2], s[i][3]));
            }
            // the base of the weights stays until a score lies 2^kQ4High above it (in short units nearly every stage holds some row's
            // new maximum)
            if (__any_sync(kFull, n0 > m0 + kQ4High || n1 > m1 + kQ4High)) {
                n0 = fmaxf(n0, __shfl_xor_sync(kFull, n0, 1));
                n1 = fmaxf(n1, __shfl_xor_sync(kFull, n1, 1));
                n0 = fmaxf(m0, fmaxf(n0, __shfl_xor_sync(kFull, n0, 2)));
                n1 = fmaxf(m1, fmaxf(n1, __shfl_xor_sync(kFull, n1, 2)));
                const float d0 = m0 == -INFINITY ? 0.0f : ex2(m0 - n0), d1 = m1 == -INFINITY ? 0.0f : ex2(m1 - n1);
                l0 *= d0;
                l1 *= d1;
#pragma unroll
                for (int i = 0; i < D / 8; i++) o[i][0] *= d0, o[i][1] *= d0, o[i][2] *= d1, o[i][3] *= d1;
                m0 = n0;
                m1 = n1;
            }
            const float b0 = m0 == -INFINITY ? 0.0f : m0 - kQ4Shift, b1 = m1 == -INFINITY ? 0.0f : m1 - kQ4Shift;
            uint32_t ph[2][4], pl[2][4];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                s[i][0] = ex2(s[i][0] - b0), s[i][1] = ex2(s[i][1] - b0);
                s[i][2] = ex2(s[i][2] - b1), s[i][3] = ex2(s[i][3] - b1);
                l0 += s[i][0] + s[i][1];
                l1 += s[i][2] + s[i][3];
                split_h2(s[i][0], s[i][1], ph[i >> 1][2 * (i & 1)], pl[i >> 1][2 * (i & 1)]);
                split_h2(s[i][2], s[i][3], ph[i >> 1][2 * (i & 1) + 1], pl[i >> 1][2 * (i & 1) + 1]);
            }
            // ---- o += weights * V: of each tile positions tq, 4 + tq (a pair), 8 + tq, 12 + tq; the tensor cores add up a stage, from 0
            // (they cut bits off), and its sums join o by additions that round
            uint32_t w[2][4][VW];
            __half2 d[2][2], m24[2][2];
#pragma unroll
            for (int x = 0; x < 2; x++) {
                const unsigned char *vn = stage + (2 * x + 1) * C::TILE;
                __half e[4];
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const int r = 4 * i + tq;
                    if constexpr (D == 128) *reinterpret_cast<uint2 *>(w[x][i]) = *reinterpret_cast<const uint2 *>(vn + r * 64 + g * 8);
                    else w[x][i][0] = *reinterpret_cast<const uint32_t *>(vn + r * 32 + g * 4);
                    e[i] = reinterpret_cast<const __half *>(vn + C::NIB)[r * (D / 32) + (D == 128 ? g >> 1 : g >> 2)];
                }
                if (masked)                       // behind the mask a weight is 0, but 0 * inf is not
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const int p = base + 64 * x + 4 * i + tq;
                        const bool none = gone(x, p);
                        if (none || (p > seen && !(fabsf(__half2float(e[i])) <= kQ4Finite))) {
                            if (!none) s_flag = 1;         // (else nobody's)
                            e[i] = __float2half(0.0f);
                        }
                    }
                d[x][0] = __halves2half2(e[0], e[1]);
                d[x][1] = __halves2half2(e[2], e[3]);
                m24[x][0] = __hmul2(d[x][0], __float2half2_rn(-24.0f));
                m24[x][1] = __hmul2(d[x][1], __float2half2_rn(-24.0f));
            }
#pragma unroll
            for (int i = 0; i < VW; i++)
#pragma unroll
                for (int h = 0; h < 2; h++) {     // values 0, 2, 4, 6 and 1, 3, 5, 7 of a word
                    uint32_t v[2][2];
#pragma unroll
                    for (int x = 0; x < 2; x++) {
                        v[x][0] = __byte_perm(w[x][0][i], w[x][1][i], h ? 0x7632 : 0x5410);
                        v[x][1] = __byte_perm(w[x][2][i], w[x][3][i], h ? 0x7632 : 0x5410);
                    }
#pragma unroll
                    for (int e = 0; e < 4; e += 2) {             // two products at a time
                        float sum[2][4];
#pragma unroll
                        for (int x = 0; x < 2; x++) {
                            uint32_t b[2][2];
#pragma unroll
                            for (int k = 0; k < 2; k++)
#pragma unroll
                                for (int z = 0; z < 2; z++) b[k][z] = q4_pair(v[x][z], e + k, d[x][z], m24[x][z], six);
#pragma unroll
                            for (int k = 0; k < 2; k++) {
                                if (x == 0) mma_16_first(sum[k], pl[x], b[k][0], b[k][1]);
                                else mma_16(sum[k], pl[x], b[k][0], b[k][1]);
                            }
#pragma unroll
                            for (int k = 0; k < 2; k++) mma_16(sum[k], ph[x], b[k][0], b[k][1]);
                        }
#pragma unroll
                        for (int k = 0; k < 2; k++) {
                            float(&y)[4] = o[8 * i + 2 * (e + k) + h];
                            const float2 lo = f2_add(make_float2(y[0], y[1]), make_float2(sum[k][0], sum[k][1]));
                            const float2 hi = f2_add(make_float2(y[2], y[3]), make_float2(sum[k][2], sum[k][3]));
                            y[0] = lo.x, y[1] = lo.y, y[2] = hi.x, y[3] = hi.y;
                        }
                    }
                }
        }
        l0 += __shfl_xor_sync(kFull, l0, 1);
        l1 += __shfl_xor_sync(kFull, l1, 1);
        l0 += __shfl_xor_sync(kFull, l0, 2);
        l1 += __shfl_xor_sync(kFull, l1, 2);
        if (isnan(l0)) m0 = 0.0f;                 // scores that are all NaN leave no maximum, but are not nothing
        if (isnan(l1)) m1 = 0.0f;
        __syncthreads();                          // every warp is done with its stages
        if (s_flag) {
            // V that were set aside: added where the row sees them (inf and NaN are not changed by a weight), by the warp that scored the
            // position: the join leaves out warps that saw nothing
            for (int p = kmin; p < k_end; p++) {
                if (((p - k0) >> 4 & 3) != warp) continue;
                const int64_t at = paged_at(a, table, p);
                if (at < 0) continue;
                const char *vr = a.v + at + kh * a.head_stride;
                const int64_t sc = q4_scales<D>(a, p & ((1 << a.page_log) - 1));
#pragma unroll
                for (int i = 0; i < D / 8; i++)
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        const float v = q4_ld<D>(vr, sc, (2 * tq + (j & 1)) * (D / 8) + i);
                        if (!isfinite(v) && p <= pos[j >> 1]) o[i][j] += v;
                    }
            }
        }
        // ---- the warps' o, m, l joined: value n (D / 8) + i of a row at 9 i + n
        float *red = reinterpret_cast<float *>(sm);
#pragma unroll
        for (int h = 0; h < 2; h++) {
            float *dst = red + (warp * 16 + g + 8 * h) * C::LD;
#pragma unroll
            for (int i = 0; i < D / 8; i++) dst[9 * i + 2 * tq] = o[i][2 * h], dst[9 * i + 2 * tq + 1] = o[i][2 * h + 1];
            if (tq == 0) {
                dst[C::LD - 2] = h ? m1 : m0;
                dst[C::LD - 1] = h ? l1 : l0;
            }
        }
        __syncthreads();
        const int64_t po = (int64_t)part * a.n_tok * a.H;
#pragma unroll
        for (int h = 0; h < 4; h++) {
            const int r = warp + 4 * h, tok = s_tok[r];
            float m = -INFINITY, l = 0.0f, mk[4], wk[4];
#pragma unroll
            for (int k = 0; k < 4; k++) {
                mk[k] = red[(k * 16 + r) * C::LD + C::LD - 2];
                m = fmaxf(m, mk[k]);
            }
#pragma unroll
            for (int k = 0; k < 4; k++) {
                wk[k] = mk[k] == -INFINITY ? 0.0f : ex2(mk[k] - m);
                l = fmaf(wk[k], red[(k * 16 + r) * C::LD + C::LD - 1], l);
            }
            if (tok < 0) continue;
#pragma unroll
            for (int d = 0; d < D / 32; d++) {
                const int v = lane + 32 * d, at = 9 * (v % (D / 8)) + v / (D / 8);
                float y = 0.0f;
#pragma unroll
                for (int k = 0; k < 4; k++)       // (a warp that saw nothing: its o may be 0 * inf)
                    y = fmaf(wk[k], mk[k] == -INFINITY ? 0.0f : red[(k * 16 + r) * C::LD + at], y);
                A.part_o[(po + tok) * D + v] = y;
            }
            if (lane == 0) A.part_ml[po + tok] = make_float2(m == -INFINITY ? m : m - kQ4Shift, l);
        }
    }
    if (last) pdl_wait();
}

template <int D, int PER_SM>
static int launch_q4(const PagedAttn &A, bool own, bool last, cudaStream_t s) {
    using C = Q4Cfg<D>;
    const int64_t units = own ? (int64_t)A.p.chunks_s * A.a.n_seq * A.p.tiles_s * A.a.Hk : (int64_t)A.p.chunks_p * A.p.tiles_p * A.a.Hk;
    QMS_REQUIRE(units < (1ll << 30), QMS_CUDA_EUNSUPPORTED, "paged_attention: too many units of work");
    static std::atomic<unsigned long long> done{0};
    const int rc = allow_smem(done, k_paged_q4<D, PER_SM>, C::SMEM);
    if (rc) return rc;
    const int grid = (int)(units < 148 * 8 ? units : 148 * 8);
    QMS_CK(launch_pdl(k_paged_q4<D, PER_SM>, dim3(grid), dim3(128), C::SMEM, s, A, own, last));
    return QMS_CUDA_OK;
}

int launch_paged_q4(const PagedAttn &A, int D, bool own, bool last, cudaStream_t s) {
    const int64_t tiles = own ? (int64_t)A.p.tiles_s * A.a.Hk * A.a.n_seq : (int64_t)A.p.tiles_p * A.a.Hk;
    if (q4_per_sm(tiles) == 2) return D == 128 ? launch_q4<128, 2>(A, own, last, s) : launch_q4<64, 2>(A, own, last, s);
    return D == 128 ? launch_q4<128, 3>(A, own, last, s) : launch_q4<64, 3>(A, own, last, s);
}

}  // namespace qms
