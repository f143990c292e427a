// qms_paged.cuh - the paged KV cache as the kernels see it (qms_paged*.cu). Not part of the C ABI.
#pragma once

#include <cuda.h>

#include "qms_kv.cuh"

namespace qms {

// A pool of pages and a batch of new tokens, flattened (QmsCudaPages, QmsCudaPagedBatch).
struct Paged {
    const int *q_start, *kv_len, *table;
    int n_seq, n_tok, table_stride, max_q, max_kv, prefix;
    char *k, *v;
    int64_t page_stride, pos_stride, head_stride;    // bytes
    int n_pages, page_log;
    int H, Hk, G;                                    // q heads, kv heads, q heads per kv head
    int *err;
};

__device__ __forceinline__ void paged_err(const Paged &a, int bit) {
    if (a.err) atomicOr(a.err, bit);
}

// The sequence that token row t belongs to, by the whole warp: how many sequences end at or before t
// (independent loads: one round trip up to 32 sequences, not a chain of dependent ones).
__device__ __forceinline__ int paged_seq_of(const Paged &a, int t) {
    int n = 0;
    for (int b = threadIdx.x & 31; b < a.n_seq; b += 32) n += a.q_start[b + 1] <= t;
    return __reduce_add_sync(kFull, n);
}

// Sequence b's rows [t0, t0 + n) and cache length. False (n = kv = 0) when the batch arrays do not make
// sense for it; such a sequence counts as idle.
__device__ __forceinline__ bool paged_seq(const Paged &a, int b, int &t0, int &n, int &kv) {
    t0 = a.q_start[b];
    n = a.q_start[b + 1] - t0;
    kv = a.kv_len[b];
    if (t0 >= 0 && n >= 0 && n <= a.max_q && n <= a.n_tok - t0 && kv >= 0 && kv <= a.max_kv) return true;
    n = kv = 0;
    return false;
}

// The same for whole prompts, whose rows are all there is of them: kv_len is not looked at.
__device__ __forceinline__ bool prompt_seq(const Paged &a, int b, int &t0, int &n, int &kv) {
    t0 = a.q_start[b];
    n = kv = a.q_start[b + 1] - t0;
    if (t0 >= 0 && n >= 0 && n <= a.max_q && n <= a.n_tok - t0) return true;
    n = kv = 0;
    return false;
}

// Byte offset of position p of table row `row` in the K / V pool, or -1 on a bad page id.
// 0 <= p < table_stride * page_size.
__device__ __forceinline__ int64_t paged_at(const Paged &a, const int *row, int p) {
    const int page = row[p >> a.page_log];
    if ((unsigned)page >= (unsigned)a.n_pages) return -1;
    return page * a.page_stride + (p & ((1 << a.page_log) - 1)) * a.pos_stride;
}

// ---- a cache in 4 bits ----
// Of a (page, kv head) lie first the positions' nibbles, D / 2 bytes each, then their scales, an fp16 number for 32 values. A value
// is d (n - 8): d has 8 significant bits and |d| <= 2720, so that the value is exact in fp16, and so are its 24 d below. (Of a larger
// scale 24 d is finite up to 2728; the values of one beyond that are not finite, all 32 of them.)
// (Paged: pos_stride is D / 2, and paged_at leads to the position's nibbles.)
struct Q4 {};
constexpr float kQ4Most = 2720.0f, kQ4Finite = 2728.0f;

__host__ __device__ constexpr int q4_row(int D) { return D / 2 + D / 16; }
// Byte distance from the nibbles of position `off` of a page to its scales.
template <int D>
__device__ __forceinline__ int64_t q4_scales(const Paged &a, int off) {
    return (int64_t)((1 << a.page_log) - off) * (D / 2) + off * (D / 16);
}
// 8 values of a word: value i in bits 4 (i / 2) + 16 (i % 2). A nibble in the upper bits of a mantissa is 16 + n, from there one
// fused step, d (16 + n) - 24 d, exact. m24: -24 d.
__device__ __forceinline__ uint4 q4_dequant(uint32_t w, __half2 d, __half2 m24) {
    uint32_t x[4] = {w << 6, w << 2, w >> 2, w >> 6};
#pragma unroll
    for (int i = 0; i < 4; i++) {
        x[i] = (x[i] & 0x03C003C0u) | 0x4C004C00u;
        const __half2 y = __hfma2(*reinterpret_cast<const __half2 *>(&x[i]), d, m24);
        x[i] = *reinterpret_cast<const uint32_t *>(&y);
    }
    return make_uint4(x[0], x[1], x[2], x[3]);
}
// One value of a row.
template <int D>
__device__ __forceinline__ float q4_ld(const char *nibbles, int64_t scales, int i) {
    const __half d = __ldcg(reinterpret_cast<const __half *>(nibbles + scales) + (i >> 5));
    const uint32_t w = __ldcg(reinterpret_cast<const unsigned int *>(nibbles) + (i >> 3));
    const int n = w >> (4 * ((i & 7) >> 1) + 16 * (i & 1)) & 15;
    return __half2float(__hfma(__int2half_rn(16 + n), d, __hmul(d, __float2half(-24.0f))));
}

// ---- pieces of the attention kernels ----
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}

__device__ __forceinline__ uint32_t pack_h2(float x, float y) {
    const __half2 h = __floats2half2_rn(x, y);
    return *reinterpret_cast<const uint32_t *>(&h);
}
// (x, y) = hi + lo in fp16 pairs, hi to nearest (so that lo has either sign: the tensor cores cut every product at the last bits
// of the sum, towards 0, and cuts of either sign cancel)
__device__ __forceinline__ void split_h2(float x, float y, uint32_t &hi, uint32_t &lo) {
    hi = pack_h2(x, y);
    asm("{\n\t.reg .b16 a, b, m;\n\t.reg .f32 x, y;\n\tmov.b32 {a, b}, %1;\n\tmov.b16 m, 0xBC00;\n\t"
        "fma.rn.f32.f16 x, a, m, %2;\n\tfma.rn.f32.f16 y, b, m, %3;\n\tcvt.rn.f16x2.f32 %0, y, x;\n\t}"
        : "=r"(lo)
        : "r"(hi), "f"(x), "f"(y));
}
// x = hi + lo, hi the 11 leading bits (what a tf32 operand keeps)
__device__ __forceinline__ float tf32_hi(float x) { return __uint_as_float(__float_as_uint(x) & 0xffffe000u); }

// Bits of the largest finite |value|, as an ordered integer: of one value (0 if it is not finite).
__device__ __forceinline__ uint32_t finite_bits(float x) {
    const uint32_t b = __float_as_uint(x) & 0x7fffffffu;
    return b < 0x7f800000u ? b : 0u;
}
// Values whose largest has the biased exponent e go to 2^9 .. 2^10 when multiplied by 2^(up - 127), which
// 2^(127 - up) undoes; both are normal numbers.
__device__ __forceinline__ uint32_t scale_up(uint32_t e) { return e == 0 ? 127u : min(263u - e, 253u); }
__device__ __forceinline__ float pow2_bits(uint32_t biased) { return __uint_as_float(biased << 23); }

// A box of a paged pool: values from x of one head, the positions of the map's box from y of a page.
__device__ __forceinline__ void tma_load4(uint32_t dst, const CUtensorMap *map, int x, int head, int y, int page, uint64_t *bar) {
    asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(dst),
                 "l"(map), "r"(x), "r"(head), "r"(y), "r"(page), "r"(smem_u32(bar))
                 : "memory");
}

// Zero what is not finite in a 16-byte piece of V; true if something was.
__device__ __forceinline__ bool drop_nonfinite(const __half *, uint4 &v) {
    uint32_t w[4] = {v.x, v.y, v.z, v.w};
    bool any = false;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        if ((w[i] & 0x7C00u) == 0x7C00u) {
            w[i] &= 0xFFFF0000u;
            any = true;
        }
        if ((w[i] & 0x7C000000u) == 0x7C000000u) {
            w[i] &= 0x0000FFFFu;
            any = true;
        }
    }
    v = make_uint4(w[0], w[1], w[2], w[3]);
    return any;
}
__device__ __forceinline__ bool drop_nonfinite(const float *, uint4 &v) {
    uint32_t w[4] = {v.x, v.y, v.z, v.w};
    bool any = false;
#pragma unroll
    for (int i = 0; i < 4; i++)
        if ((w[i] & 0x7F800000u) == 0x7F800000u) {
            w[i] = 0;
            any = true;
        }
    v = make_uint4(w[0], w[1], w[2], w[3]);
    return any;
}

// ---- attention: the work and its split ----------------------------------------------------------
// Two kinds of units, per kv head: the shared positions [0, prefix) against tiles of all token rows, and
// a sequence's own positions [prefix, kv_len) against tiles of its rows. A row is a (token, q head of the
// kv head's group) pair, row = token * G + head. Positions are cut into chunks; every (chunk, row) writes a
// partial result to its slot of the workspace (prefix chunks first) and k_paged_merge joins a row's
// slots: part_o [slots][n_tok * H][D] (not divided by l), part_ml [slots][n_tok * H] of (m, l),
// m the base-2 exponent of the weights' common factor.
struct PagedPlan {
    int wr_p, wr_s;                  // shared, own: row groups of 16 per tile (k_paged_attn), or kPaWide...
    int chunk_p, chunk_s;            // positions per chunk
    int base_s;                      // where the own positions' chunks start: prefix, or the tile boundary before it
    int chunks_p, chunks_s;          // chunks of each kind
    int slots_p, slots_s;            // slots of each kind
    int tiles_p, tiles_s;            // row tiles of each kind
    // k_paged_wide's runs over the shared positions: total length (0: none), runs, runs per CTA, places of the line per
    // run (the first line_r runs have one more), position tiles; positions per place, rows per row tile
    unsigned line, line_runs, line_per, line_q, line_r, line_nt;
    int line_tp, line_rows;
    int flat;                        // 4 bits: positions that go to the workspace in fp16 (0: none), for every kind that is kPaWidePair
};
// CTAs of k_paged_q4 per SM for so many tiles of rows: two have more products in flight each, three even out sequences of
// unlike lengths, and waves. Two and three in us: 4 tiles (one token on 131,072 positions) 48.0, 53.3; on 16,384 18.7, 22.7; 32 19.7, 22.6; 160 28.5, 25.9; 256 81.1,
// 89.1, of lengths up to that 60 to 77, 57; 512 150.6, 145.7.
inline int q4_per_sm(int64_t tiles) { return tiles < 148 ? 2 : 3; }

// k_paged_wide: 256 rows; 128; 128 over an fp32 cache; 128 over one in 4 bits
constexpr int kPaWidePair = 0, kPaWideSplit = -1, kPaWideF32 = -2, kPaWideQ4 = -3;

// Where run i starts, and which run holds place x. (Divisions are what a short kernel's start waits for: few, of 32 bits.)
__device__ __forceinline__ unsigned line_start(const PagedPlan &p, unsigned i) { return i * p.line_q + min(i, p.line_r); }
__device__ __forceinline__ unsigned line_run(const PagedPlan &p, unsigned x) {
    const unsigned longer = p.line_r * (p.line_q + 1);
    return x < longer ? x / (p.line_q + 1) : p.line_r + (x - longer) / p.line_q;
}

struct PagedAttn {
    Paged a;
    PagedPlan p;
    const float *q;
    float *out;
    int64_t ldq, ldo;
    float scale2;                    // scale * log2(e)
    int type;                        // the cache's
    float *part_o;
    float2 *part_ml;
};

constexpr uint32_t kWSpin = 1u << 22;

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

// The driver's cuTensorMapEncodeTiled, looked up once.
typedef CUresult (*TensorEncode)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *, const cuuint32_t *,
                                 const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
int tensor_encode(TensorEncode *encode);                                                   // qms_paged_attn.cu

// The pool as a tensor [page][position][head][value], in boxes of up to `rows` positions of a page: 64 fp16 values, 128-byte
// swizzled, or a whole fp32 row.
int paged_map(const Paged &a, int D, bool f16, int rows, const char *pool, CUtensorMap *map);
void paged_plan(const Paged &a, int type, int D, PagedPlan &p);
int64_t paged_ws_bytes(const Paged &a, int D, const PagedPlan &p);
int launch_paged_wide(const PagedAttn &A, int D, bool own, bool last, cudaStream_t s);     // qms_paged_wide.cu
int launch_paged_q4(const PagedAttn &A, int D, bool own, bool last, cudaStream_t s);       // qms_paged_q4.cu
int launch_paged_attention(const Paged &a, int type, int D, const PagedPlan &p, const float *q, int64_t ldq, float scale,
                           float *out, int64_t ldo, void *ws, cudaStream_t s);

}  // namespace qms
