// qms_paged.cu - a paged KV cache on B200 (sm_100a): the append of new tokens with QK-norm and rotation
// (src/model.c:436-462 on one contiguous cache), and the C entries of the paged operators.
#include <cuda_bf16.h>
#include <math.h>
#include <string.h>

#include <algorithm>

#include "qms_moe.cuh"
#include "qms_paged.cuh"

namespace qms {

// ---- append --------------------------------------------------------------------------------------
// A warp takes R head rows of q | k | v of one token: y = R(pos) (w * x / sqrt(mean x^2 + eps)) for q and k, v unchanged.
// The mean's sum is held in double and the steps are k_qk_rope's, each in its order, so a paged cache holds the same
// values as the model's contiguous one.
// Bound by latency for few rows (R = 1: 2.5 us for one token) and by instructions for many, most of them for the 64-bit
// mean: R = 4 rows share the exchanges of their sums and one square root and division (a lane each).
template <int R>
__device__ __forceinline__ void sum_rows(double (&v)[R], int lane) {      // the sum of v[r] over the lanes; R = 4: v[0] of row lane / 8
    if constexpr (R == 1) {
        v[0] = warp_sum_d(v[0]);
    } else {
        const bool hi = lane & 16, mid = lane & 8;
        const double a = __shfl_xor_sync(kFull, hi ? v[0] : v[2], 16), b = __shfl_xor_sync(kFull, hi ? v[1] : v[3], 16);
        const double x = (hi ? v[2] : v[0]) + a, y = (hi ? v[3] : v[1]) + b;
        v[0] = (mid ? y : x) + __shfl_xor_sync(kFull, mid ? x : y, 8);
#pragma unroll
        for (int o = 4; o > 0; o >>= 1) v[0] += __shfl_xor_sync(kFull, v[0], o);
    }
}

template <int D, typename KT, int R>
__global__ void __launch_bounds__(256) k_paged_append(const Paged a, const float *qkv, int64_t ldqkv, const float *q_norm,
                                                      const float *k_norm, float eps, const float *rope_cos,
                                                      const float *rope_sin, int n_rope, float *q, int64_t ldq) {
    static_assert(R == 1 || R == 4, "rows per warp");
    constexpr int J = D / 32, JH = J / 2;
    const int lane = threadIdx.x & 31, groups = (a.H + 2 * a.Hk + R - 1) / R, nq = a.H + a.Hk;
    const unsigned unit = blockIdx.x * 8 + (threadIdx.x >> 5);
    const int t = unit / groups, h0 = (unit - t * groups) * R;
    pdl_trigger();
    pdl_wait();
    if (t >= a.n_tok) return;
    const float *row = qkv + t * ldqkv + h0 * D;
    float x[R][J], w[J];
#pragma unroll
    for (int r = 0; r < R; r++)
#pragma unroll
        for (int j = 0; j < J; j++) x[r][j] = h0 + r < nq + a.Hk ? row[r * D + lane + 32 * j] : 0.0f;
#pragma unroll
    for (int j = 0; j < J; j++) w[j] = (h0 < a.H ? q_norm : k_norm)[lane + 32 * j];
    const int b = paged_seq_of(a, t);
    if (b >= a.n_seq) return;                                   // padding
    int t0, n, kv;
    const bool ok = paged_seq(a, b, t0, n, kv);
    if (ok && (t < t0 || t >= t0 + n)) return;                  // before the first sequence's rows
    const int p = kv - n + (t - t0);
    if (!ok || p < 0 || p >= n_rope) {
        if (lane == 0 && h0 == 0) paged_err(a, QMS_PAGED_ELEN);
        return;
    }
    const int64_t at = paged_at(a, a.table + (int64_t)b * a.table_stride, p);
    if (at < 0) {
        if (lane == 0 && h0 == 0) paged_err(a, QMS_PAGED_EPAGE);
        return;
    }
    float c[JH], s[JH];
    double inv = 0.0;
    if (h0 < nq) {
#pragma unroll
        for (int j = 0; j < JH; j++) {
            c[j] = rope_cos[(int64_t)p * (D / 2) + lane + 32 * j];
            s[j] = rope_sin[(int64_t)p * (D / 2) + lane + 32 * j];
        }
        double ss[R];
#pragma unroll
        for (int r = 0; r < R; r++) {
            ss[r] = 0.0;
#pragma unroll
            for (int j = 0; j < J; j++) ss[r] = fma((double)x[r][j], (double)x[r][j], ss[r]);
        }
        sum_rows<R>(ss, lane);
        inv = 1.0 / sqrt(ss[0] / D + (double)eps);
    }
#pragma unroll
    for (int r = 0; r < R; r++) {
        const int hh = h0 + r;
        if (hh >= nq + a.Hk) return;
        if (hh < nq) {
            if (r > 0 && hh == a.H)                             // from q to k
#pragma unroll
                for (int j = 0; j < J; j++) w[j] = k_norm[lane + 32 * j];
            rope_scaled<D>(x[r], w, c, s, R == 1 ? inv : __shfl_sync(kFull, inv, 8 * r));
        }
        if (hh < a.H) {
#pragma unroll
            for (int j = 0; j < J; j++) q[t * ldq + hh * D + lane + 32 * j] = x[r][j];
        } else {
            KT *dst = reinterpret_cast<KT *>((hh < nq ? a.k : a.v) + at + (hh < nq ? hh - a.H : hh - nq) * a.head_stride);
#pragma unroll
            for (int j = 0; j < J; j++) kv_st(dst + lane + 32 * j, x[r][j]);
        }
    }
}

template <int D, typename KT>
static int launch_append(const Paged &a, const float *qkv, int64_t ldqkv, const float *q_norm, const float *k_norm, float eps,
                         const float *rope_cos, const float *rope_sin, int n_rope, float *q, int64_t ldq, cudaStream_t s) {
    const int heads = a.H + 2 * a.Hk;
    // Four rows per warp once there are 48 for each SM. Both in us at 40 or 72 head rows per token: 4608 rows 3.56 one,
    // 3.59 four; 5120 3.4, 3.8; 9216 5.2, 4.2; 10240 5.6, 4.8; 144000 50, 29 (4.9 TB/s).
    const bool four = (int64_t)a.n_tok * heads >= 148 * 48;
    const int64_t units = (int64_t)a.n_tok * (four ? (heads + 3) / 4 : heads);
    QMS_REQUIRE(units < (1ll << 31), QMS_CUDA_EUNSUPPORTED, "paged_append: too many rows");
    const dim3 grid((unsigned)((units + 7) / 8));
    if (four) QMS_CK(launch_pdl(k_paged_append<D, KT, 4>, grid, dim3(256), 0, s, a, qkv, ldqkv, q_norm, k_norm, eps, rope_cos, rope_sin, n_rope, q, ldq));
    else QMS_CK(launch_pdl(k_paged_append<D, KT, 1>, grid, dim3(256), 0, s, a, qkv, ldqkv, q_norm, k_norm, eps, rope_cos, rope_sin, n_rope, q, ldq));
    return QMS_CUDA_OK;
}

// ---- append to a cache in 4 bits, rows in 16 bits ----------------------------------------------------
// 32 values, one per lane, as they are held: the scale is the value m of largest magnitude (the first of equals) over -8, rounded to 8
// significant bits; n = floor(y / d + 8.5) within 0 .. 15. In double, as y is: a K value next to a border between two steps goes to
// the side that the formula has it on, whatever order the sums were added in. (y r + 8.5, r = 1 / d rounded: the 2^-40 more keeps a
// quotient that is a tie, such as 2.5, from falling below it, and is less than what lies between a tie and the next quotient of an
// fp32 value.) A group with a value that is not finite is NaN.
struct Q4Group {
    uint32_t n;
    __half d;
};
__device__ __noinline__ Q4Group q4_quantize_exact(double y) {
    const unsigned long long bits = __double_as_longlong(y) & 0x7fffffffffffffffull;
    const uint32_t hi = (uint32_t)(bits >> 32), lo = (uint32_t)bits, mh = __reduce_max_sync(kFull, hi);
    const uint32_t ml = __reduce_max_sync(kFull, hi == mh ? lo : 0u);
    const int first = __ffs(__ballot_sync(kFull, hi == mh && lo == ml)) - 1;
    const double m = __shfl_sync(kFull, y, first);
    Q4Group q;
    if (mh >= 0x7ff00000u) {
        q.n = 8;
        q.d = __ushort_as_half(0x7fff);
        return q;
    }
    unsigned long long db = __double_as_longlong(m * -0.125);
    db = (db + (1ull << 44) - 1 + (db >> 45 & 1)) & ~((1ull << 45) - 1);        // half to even
    const double d = fmin(fmax(__longlong_as_double(db), -(double)kQ4Most), (double)kQ4Most);
    q.d = __double2half(d);
    const double held = (double)__half2float(q.d);
    if (held == 0.0) q.n = 8;
    else q.n = (uint32_t)min(max(__double2int_rd(fma(y, 1.0 / held, 8.5 + 0x1p-40)), 0), 15);
    return q;
}

// The same in fp32 where that is certain to give the same: one value of largest magnitude, by more than 2 in its last place; a scale
// that is not within 8 of the border between two of 8 bits; quotients (off by some 2e-6) that are 2e-5 from a border. One group in 1000
// of random values is not, and takes 5 times as long.
__device__ __forceinline__ Q4Group q4_quantize(double y) {
    const float yf = (float)y;
    const uint32_t b = __float_as_uint(yf) & 0x7fffffffu, most = __reduce_max_sync(kFull, b);
    const unsigned near = __ballot_sync(kFull, b + 2 >= most);
    const float m = __shfl_sync(kFull, yf, __ffs(near) - 1);
    const uint32_t db = __float_as_uint(m * -0.125f);
    Q4Group q;
    q.d = __float2half_rn(fminf(fmaxf(__uint_as_float((db + 0x7fffu + (db >> 16 & 1)) & 0xffff0000u), -kQ4Most), kQ4Most));
    const float held = __half2float(q.d), t = fmaf(yf, __frcp_rn(held), 8.5f);
    q.n = (uint32_t)min(max(__float2int_rd(t), 0), 15);
    const bool sure = most < 0x7f800000u && most >= 0x01000000u && (near & (near - 1)) == 0 && (uint32_t)((int)(db & 0xffffu) - 0x7ff8) > 16u && held != 0.0f;
    if (!sure || __any_sync(kFull, fabsf(t - rintf(t)) < 2e-5f)) return q4_quantize_exact(y);
    return q;
}

// A row's values (lane + 32 j: y[j]) to their place in a page.
template <int D>
__device__ __forceinline__ void q4_store(const Paged &a, char *nibbles, int off, const double (&y)[D / 32], int lane) {
    constexpr int J = D / 32;
    uint32_t word = 0;
    __half d = __float2half(0.0f);
#pragma unroll
    for (int j = 0; j < J; j++) {
        const Q4Group q = q4_quantize(y[j]);
        uint32_t w = q.n << (4 * ((lane & 7) >> 1) + 16 * (lane & 1));
        w |= __shfl_xor_sync(kFull, w, 1);
        w |= __shfl_xor_sync(kFull, w, 2);
        w |= __shfl_xor_sync(kFull, w, 4);
        if ((lane & 7) == j) word = w;
        if (lane == j) d = q.d;
    }
    if ((lane & 7) < J) reinterpret_cast<uint32_t *>(nibbles)[4 * (lane & 7) + (lane >> 3)] = word;
    if (lane < J) reinterpret_cast<__half *>(nibbles + q4_scales<D>(a, off))[lane] = d;
}

__device__ __forceinline__ void row_st(float *p, float v) { *p = v; }
__device__ __forceinline__ void row_st(__half *p, float v) { *p = __float2half_rn(v); }
__device__ __forceinline__ void row_st(__nv_bfloat16 *p, float v) { *p = __float2bfloat16_rn(v); }
__device__ __forceinline__ void row_st2(float *p, float x, float y) { *reinterpret_cast<float2 *>(p) = make_float2(x, y); }
__device__ __forceinline__ void row_st2(__half *p, float x, float y) { *reinterpret_cast<__half2 *>(p) = __floats2half2_rn(x, y); }
__device__ __forceinline__ void row_st2(__nv_bfloat16 *p, float x, float y) { *reinterpret_cast<__nv_bfloat162 *>(p) = __floats2bfloat162_rn(x, y); }

// R q heads of one token to 16 bits, in fp32: y = R(pos) (w x / sqrt(mean x^2 + eps)). (The mean too: 9 roundings on the way of a square, half
// of them after the root, are 2^-21 of y, 2^-10 of fp16's half step.) Of 128 values a lane has 2 l, 2 l + 1 and the two 64 further, which
// they are rotated with.
template <typename OT, int R>
__device__ __forceinline__ void q_rows16(const float2 (&x)[R][2], int cnt, const float *norm, float eps, const float *cos, const float *sin, OT *out, int lane) {
    auto two = [&](const float *v) { return make_float2(v[2 * lane], v[2 * lane + 1]); };       // (of any alignment)
    const float2 w0 = two(norm), w1 = two(norm + 64), c = two(cos), s = two(sin);
    float ss[R];
#pragma unroll
    for (int r = 0; r < R; r++) ss[r] = fmaf(x[r][0].x, x[r][0].x, x[r][0].y * x[r][0].y) + fmaf(x[r][1].x, x[r][1].x, x[r][1].y * x[r][1].y);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
#pragma unroll
        for (int r = 0; r < R; r++) ss[r] += __shfl_xor_sync(kFull, ss[r], o);
#pragma unroll
    for (int r = 0; r < R; r++) {
        if (r >= cnt) return;
        const float inv = 1.0f / sqrtf(fmaf(ss[r], 1.0f / 128.0f, eps));
        const float a0 = x[r][0].x * inv * w0.x, a1 = x[r][0].y * inv * w0.y, b0 = x[r][1].x * inv * w1.x, b1 = x[r][1].y * inv * w1.y;
        OT *to = out + r * 128 + 2 * lane;
        row_st2(to, a0 * c.x - b0 * s.x, a1 * c.y - b1 * s.y);
        row_st2(to + 64, b0 * c.x + a0 * s.x, b1 * c.y + a1 * s.y);
    }
}

// k_paged_append's steps where the cache or the rows that go out are of another kind: a cache in 4 bits (K normalised and rotated in
// double, see above), or none; rows out of fp32, the q heads, or of 16 bits, all heads q | k | v as the prompt attention reads
// them, each value rounded once from fp32. (What is stored in 4 bits: q4_quantize. Rows of 16 bits next to a cache of fp32 or fp16: that cache's values are k_paged_append's.)
// A warp takes R q heads, or one K or V head: what is stored in 4 bits takes as long as four q heads.
// Bound by latency for few rows (64 tokens of 72 heads 4.1 us, one token 3.1), by instructions for many, those of the exchanges within 32
// values and, for K, of double up to the rotated value: 700 tokens of 40 heads 9.9 us with rows in 16 bits, 2.5 TB/s.
template <int D, typename OT, int R>
__global__ void __launch_bounds__(256) k_rows_append(const Paged a, const int type, const float *qkv, int64_t ldqkv, const float *q_norm,
                                                     const float *k_norm, float eps, const float *rope_cos, const float *rope_sin, int n_rope,
                                                     OT *out, int64_t ldo) {
    static_assert(R == 1 || R == 4, "rows per warp");
    constexpr bool ALL = sizeof(OT) == 2;
    constexpr int J = D / 32, JH = J / 2;
    const int lane = threadIdx.x & 31, gq = (a.H + R - 1) / R, groups = gq + 2 * a.Hk, nq = a.H + a.Hk;
    const unsigned unit = blockIdx.x * 8 + (threadIdx.x >> 5);
    const int t = unit / groups, j0 = unit - t * groups, h0 = j0 < gq ? j0 * R : a.H + j0 - gq, cnt = j0 < gq ? min(R, a.H - h0) : 1;
    pdl_trigger();
    pdl_wait();
    if (t >= a.n_tok) return;
    const float *row = qkv + t * ldqkv + h0 * D;
    constexpr bool Q16 = ALL && D == 128;
    float x[R][J], w[J];
    float2 x2[R][2];
    if (Q16 && h0 < a.H) {
#pragma unroll
        for (int r = 0; r < R; r++)
#pragma unroll
            for (int j = 0; j < 2; j++) x2[r][j] = r < cnt ? reinterpret_cast<const float2 *>(row + r * D)[lane + 32 * j] : make_float2(0.0f, 0.0f);
    } else {
#pragma unroll
        for (int r = 0; r < R; r++)
#pragma unroll
            for (int j = 0; j < J; j++) x[r][j] = r < cnt ? row[r * D + lane + 32 * j] : 0.0f;
    }
#pragma unroll
    for (int j = 0; j < J; j++) w[j] = (h0 < a.H ? q_norm : k_norm)[lane + 32 * j];
    const int b = paged_seq_of(a, t);
    if (b >= a.n_seq) return;                                   // padding
    int t0, n, kv;
    const bool ok = a.n_pages == 0 ? prompt_seq(a, b, t0, n, kv) : paged_seq(a, b, t0, n, kv);
    if (ok && (t < t0 || t >= t0 + n)) return;                  // before the first sequence's rows
    const int p = kv - n + (t - t0);
    if (!ok || p < 0 || p >= n_rope) {
        if (lane == 0 && h0 == 0) paged_err(a, QMS_PAGED_ELEN);
        return;
    }
    const int64_t at = a.n_pages == 0 ? 0 : paged_at(a, a.table + (int64_t)b * a.table_stride, p);
    if (at < 0) {
        if (lane == 0 && h0 == 0) paged_err(a, QMS_PAGED_EPAGE);
        return;
    }
    if constexpr (Q16) {
        if (h0 < a.H) {
            q_rows16<OT, R>(x2, cnt, q_norm, eps, rope_cos + (int64_t)p * (D / 2), rope_sin + (int64_t)p * (D / 2), out + t * ldo + h0 * D, lane);
            return;
        }
    }
    float c[JH], s[JH];
    double inv = 0.0;
    if (h0 < nq) {
#pragma unroll
        for (int j = 0; j < JH; j++) {
            c[j] = rope_cos[(int64_t)p * (D / 2) + lane + 32 * j];
            s[j] = rope_sin[(int64_t)p * (D / 2) + lane + 32 * j];
        }
        double ss[R];
#pragma unroll
        for (int r = 0; r < R; r++) {
            ss[r] = 0.0;
#pragma unroll
            for (int j = 0; j < J; j++) ss[r] = fma((double)x[r][j], (double)x[r][j], ss[r]);
        }
        sum_rows<R>(ss, lane);
        inv = 1.0 / sqrt(ss[0] / D + (double)eps);
    }
    if (h0 >= a.H) {                                            // a K or V head
        const double iv = R == 1 ? inv : __shfl_sync(kFull, inv, 0);
        const bool is_k = h0 < nq;
        char *dst = a.n_pages == 0 ? nullptr : (is_k ? a.k : a.v) + at + (is_k ? h0 - a.H : h0 - nq) * a.head_stride;
        if (dst && type == QMS_T_Q4_0) {
            double y[J];
#pragma unroll
            for (int j = 0; j < J; j++) y[j] = is_k ? (double)x[0][j] * iv * (double)w[j] : (double)x[0][j];
            if (is_k) {
#pragma unroll
                for (int j = 0; j < JH; j++) {
                    const double y1 = y[j], y2 = y[j + JH];
                    y[j] = y1 * (double)c[j] - y2 * (double)s[j];
                    y[j + JH] = y2 * (double)c[j] + y1 * (double)s[j];
                }
            }
            q4_store<D>(a, dst, p & ((1 << a.page_log) - 1), y, lane);
        }
        if (is_k && (ALL || type != QMS_T_Q4_0)) rope_scaled<D>(x[0], w, c, s, iv);
        if (dst && type != QMS_T_Q4_0) {
#pragma unroll
            for (int j = 0; j < J; j++) {
                if (type == QMS_T_F16) kv_st(reinterpret_cast<__half *>(dst) + lane + 32 * j, x[0][j]);
                else kv_st(reinterpret_cast<float *>(dst) + lane + 32 * j, x[0][j]);
            }
        }
        if (ALL)
#pragma unroll
            for (int j = 0; j < J; j++) row_st(out + t * ldo + h0 * D + lane + 32 * j, x[0][j]);
        return;
    }
#pragma unroll
    for (int r = 0; r < R; r++) {
        if (r >= cnt) return;
        rope_scaled<D>(x[r], w, c, s, R == 1 ? inv : __shfl_sync(kFull, inv, 8 * r));
#pragma unroll
        for (int j = 0; j < J; j++) row_st(out + t * ldo + (h0 + r) * D + lane + 32 * j, x[r][j]);
    }
}

template <int D, typename OT>
static int launch_rows_append(const Paged &a, int type, const float *qkv, int64_t ldqkv, const float *q_norm, const float *k_norm, float eps,
                              const float *rope_cos, const float *rope_sin, int n_rope, OT *out, int64_t ldo, cudaStream_t s) {
    const int heads = a.H + 2 * a.Hk;
    // Four q heads per warp from 32 head rows for each SM on. Both in us, one and four: 2304 rows 3.6, 3.6; 4608 4.1, 4.1; 5120 5.3, 4.1; 7200 5.6, 4.3;
    // 28,000 14.6, 11.3; 160,000 78, 55 (rows in 16 bits 69, 45).
    const bool four = (int64_t)a.n_tok * heads >= 148 * 32;
    const int64_t units = (int64_t)a.n_tok * (four ? (a.H + 3) / 4 + 2 * a.Hk : heads);
    QMS_REQUIRE(units < (1ll << 31), QMS_CUDA_EUNSUPPORTED, "append: too many rows");
    const dim3 grid((unsigned)((units + 7) / 8));
    const auto k = four ? k_rows_append<D, OT, 4> : k_rows_append<D, OT, 1>;
    QMS_CK(launch_pdl(k, grid, dim3(256), 0, s, a, type, qkv, ldqkv, q_norm, k_norm, eps, rope_cos, rope_sin, n_rope, out, ldo));
    return QMS_CUDA_OK;
}

// ---- what a pool's pages hold, as fp32 ---------------------------------------------------------------
// 8 values per thread, in the order of the result [page][position][head][value]: whole lines are written. Grid y: K, V. Bound by
// those writes: 64 pages of 16 positions and 4 heads 3.6 us.
template <int D>
__global__ void __launch_bounds__(256) k_paged_values(const Paged a, const int type, float *ko, float *vo) {
    pdl_trigger();
    pdl_wait();
    const int64_t total = ((int64_t)a.n_pages << a.page_log) * a.Hk * (D / 8);
    const char *pool = blockIdx.y ? a.v : a.k;
    float *out = blockIdx.y ? vo : ko;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
        const int w = (int)(i % (D / 8));
        const int64_t row = i / (D / 8), pos = row / a.Hk;
        const int h = (int)(row - pos * a.Hk), off = (int)(pos & ((1 << a.page_log) - 1));
        const char *src = pool + (pos >> a.page_log) * a.page_stride + off * a.pos_stride + h * a.head_stride;
        float x[8];
        if (type == QMS_T_Q4_0) {
            const __half2 d = __half2half2(reinterpret_cast<const __half *>(src + q4_scales<D>(a, off))[w / 4]);
            const uint4 y = q4_dequant(reinterpret_cast<const uint32_t *>(src)[w], d, __hmul2(d, __float2half2_rn(-24.0f)));
            const uint32_t yy[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&yy[e]));
                x[2 * e] = f.x, x[2 * e + 1] = f.y;
            }
        } else {
#pragma unroll
            for (int e = 0; e < 8; e += 4) {
                const float4 f = type == QMS_T_F16 ? kv_ldg4(reinterpret_cast<const __half *>(src) + 8 * w + e)
                                                   : kv_ldg4(reinterpret_cast<const float *>(src) + 8 * w + e);
                x[e] = f.x, x[e + 1] = f.y, x[e + 2] = f.z, x[e + 3] = f.w;
            }
        }
        *reinterpret_cast<float4 *>(out + 8 * i) = make_float4(x[0], x[1], x[2], x[3]);
        *reinterpret_cast<float4 *>(out + 8 * i + 4) = make_float4(x[4], x[5], x[6], x[7]);
    }
}

// ---- host ----------------------------------------------------------------------------------------
// The two descriptors, checked, as the kernels take them.
// (may_lack: the call can do without a pool, where n_pages is 0 and k and v are NULL)
static int paged_args(const char *who, const QmsCudaPages *pg, const QmsCudaPagedBatch *bt, int n_head, int *err, Paged &a, bool may_lack = false) {
    QMS_REQUIRE(pg && bt, QMS_CUDA_EINVAL, "%s: NULL descriptor", who);
    const bool pool = !may_lack || pg->n_pages != 0 || pg->k || pg->v, packed = pool && pg->type == QMS_T_Q4_0;
    QMS_REQUIRE(!pool || pg->type == QMS_T_F32 || pg->type == QMS_T_F16 || packed, QMS_CUDA_EUNSUPPORTED, "%s: cache type %d (F32, F16 or Q4_0)",
                who, pg->type);
    QMS_REQUIRE(pg->head_dim == 64 || pg->head_dim == 128, QMS_CUDA_EUNSUPPORTED, "%s: head_dim %d (64 or 128 supported)",
                who, pg->head_dim);
    QMS_REQUIRE(pg->n_head_kv > 0 && (!pool || (pg->n_pages > 0 && pg->page_size > 0 && (pg->page_size & (pg->page_size - 1)) == 0)),
                QMS_CUDA_EINVAL, "%s: pages need n_pages > 0, n_head_kv > 0 and a page size that is a power of two", who);
    QMS_REQUIRE(n_head > 0 && n_head % pg->n_head_kv == 0 && n_head <= 1024, QMS_CUDA_EINVAL,
                "%s: %d q heads over %d kv heads", who, n_head, pg->n_head_kv);
    QMS_REQUIRE(!packed || (pg->page_size >= 16 && pg->page_size <= (1 << 20) && pg->pos_stride == 0), QMS_CUDA_EINVAL,
                "%s: pages in 4 bits need 16 to 2^20 positions and pos_stride 0 (a head's positions lie together)", who);
    const int64_t es = packed ? 1 : pg->type == QMS_T_F16 ? 2 : 4;
    QMS_REQUIRE(!pool || (pg->k && pg->v), QMS_CUDA_EINVAL, "%s: NULL K or V", who);
    QMS_REQUIRE(((uintptr_t)pg->k & 15) == 0 && ((uintptr_t)pg->v & 15) == 0, QMS_CUDA_EINVAL,
                "%s: K and V must be 16-byte aligned device memory", who);
    QMS_REQUIRE(!pool || (pg->page_stride >= 0 && pg->pos_stride >= 0 && pg->head_stride >= 0 && pg->page_stride * es % 16 == 0 &&
                    pg->pos_stride * es % 16 == 0 && pg->head_stride * es % 16 == 0),
                QMS_CUDA_EINVAL, "%s: strides must be multiples of 16 bytes, none negative", who);
    QMS_REQUIRE(bt->n_seq >= 0 && bt->n_tok >= 0 && bt->n_tok <= (1 << 20) && bt->n_seq <= (1 << 20), QMS_CUDA_EINVAL,
                "%s: n_seq %d, n_tok %d", who, bt->n_seq, bt->n_tok);
    QMS_REQUIRE(bt->max_q >= 0 && bt->max_kv >= 0 && bt->prefix_len >= 0 && bt->table_stride >= 0, QMS_CUDA_EINVAL,
                "%s: negative max_q, max_kv, prefix_len or table_stride", who);
    const int64_t cap = (int64_t)bt->table_stride * pg->page_size;
    QMS_REQUIRE(!pool || (bt->max_kv <= cap && bt->prefix_len <= cap), QMS_CUDA_EINVAL,
                "%s: max_kv %d and prefix_len %d need pages in the table (%d of %d positions)", who, bt->max_kv,
                bt->prefix_len, bt->table_stride, pg->page_size);
    QMS_REQUIRE(bt->n_seq == 0 || (bt->q_start && (!pool || (bt->kv_len && (bt->table || bt->table_stride == 0)))), QMS_CUDA_EINVAL,
                "%s: NULL q_start, kv_len or table", who);
    QMS_REQUIRE((((uintptr_t)bt->q_start | (uintptr_t)bt->kv_len | (uintptr_t)bt->table | (uintptr_t)err) & 3) == 0,
                QMS_CUDA_EINVAL, "%s: misaligned int array", who);
    a.q_start = bt->q_start;
    a.kv_len = bt->kv_len;
    a.table = bt->table;
    a.n_seq = bt->n_seq;
    a.n_tok = bt->n_tok;
    a.table_stride = bt->table_stride;
    a.max_q = bt->max_q;
    a.max_kv = bt->max_kv;
    a.prefix = bt->n_seq > 0 ? bt->prefix_len : 0;
    a.k = (char *)pg->k;
    a.v = (char *)pg->v;
    a.page_stride = pg->page_stride * es;
    a.pos_stride = packed ? pg->head_dim / 2 : pg->pos_stride * es;
    a.head_stride = pg->head_stride * es;
    a.n_pages = pg->n_pages;
    a.page_log = 0;
    while (pool && (1 << a.page_log) < pg->page_size) a.page_log++;
    a.H = n_head;
    a.Hk = pg->n_head_kv;
    a.G = n_head / pg->n_head_kv;
    a.err = err;
    return QMS_CUDA_OK;
}

static int paged_rows(const char *who, const char *what, const void *p, int64_t ld, int64_t cols) {
    QMS_REQUIRE(p && ((uintptr_t)p & 15) == 0 && ld >= cols && ld % 4 == 0, QMS_CUDA_EINVAL,
                "%s: %s rows must be 16-byte aligned device memory, at least %lld floats apart", who, what, (long long)cols);
    return QMS_CUDA_OK;
}

}  // namespace qms

using namespace qms;

extern "C" {

int qms_cuda_paged_append(const QmsCudaPages *pages, const QmsCudaPagedBatch *batch, const float *qkv, int64_t ldqkv,
                          int n_head, const float *q_norm, const float *k_norm, float eps, const float *rope_cos,
                          const float *rope_sin, int n_rope, float *q, int64_t ldq, int *err, void *stream) {
    clear_error();
    Paged a;
    int rc = paged_args("paged_append", pages, batch, n_head, err, a);
    if (rc) return rc;
    if (a.n_tok == 0 || a.n_seq == 0) return QMS_CUDA_OK;
    const int D = pages->head_dim;
    if ((rc = paged_rows("paged_append", "qkv", qkv, ldqkv, (int64_t)(n_head + 2 * a.Hk) * D))) return rc;
    if ((rc = paged_rows("paged_append", "q", q, ldq, (int64_t)n_head * D))) return rc;
    QMS_REQUIRE(q != qkv || ldq == ldqkv || a.n_tok == 1, QMS_CUDA_EINVAL,
                "paged_append: in place, q and qkv need rows at one distance (%lld, %lld)", (long long)ldq, (long long)ldqkv);
    QMS_REQUIRE(q_norm && k_norm && rope_cos && rope_sin && n_rope > 0, QMS_CUDA_EINVAL,
                "paged_append: NULL norm weights or rotation tables");
    if (pages->type == QMS_T_Q4_0) {
        if (D == 128) return launch_rows_append<128>(a, pages->type, qkv, ldqkv, q_norm, k_norm, eps, rope_cos, rope_sin, n_rope, q, ldq, (cudaStream_t)stream);
        return launch_rows_append<64>(a, pages->type, qkv, ldqkv, q_norm, k_norm, eps, rope_cos, rope_sin, n_rope, q, ldq, (cudaStream_t)stream);
    }
#define QMS_APPEND(D_, KT) \
    return launch_append<D_, KT>(a, qkv, ldqkv, q_norm, k_norm, eps, rope_cos, rope_sin, n_rope, q, ldq, (cudaStream_t)stream)
    if (pages->type == QMS_T_F16) {
        if (D == 128) QMS_APPEND(128, __half); else QMS_APPEND(64, __half);
    } else {
        if (D == 128) QMS_APPEND(128, float); else QMS_APPEND(64, float);
    }
#undef QMS_APPEND
}

int qms_cuda_prompt_append(const QmsCudaPages *pages, const QmsCudaPagedBatch *batch, const float *qkv, int64_t ldqkv, int n_head,
                           const float *q_norm, const float *k_norm, float eps, const float *rope_cos, const float *rope_sin, int n_rope,
                           int type, void *rows, int64_t ldrows, int *err, void *stream) {
    clear_error();
    Paged a;
    int rc = paged_args("prompt_append", pages, batch, n_head, err, a, true);
    if (rc) return rc;
    QMS_REQUIRE(type == QMS_T_F16 || type == QMS_CUDA_T_BF16, QMS_CUDA_EUNSUPPORTED, "prompt_append: rows of type %d (F16 or BF16)", type);
    if (a.n_tok == 0 || a.n_seq == 0) return QMS_CUDA_OK;
    const int D = pages->head_dim;
    const int64_t cols = (int64_t)(n_head + 2 * a.Hk) * D;
    if ((rc = paged_rows("prompt_append", "qkv", qkv, ldqkv, cols))) return rc;
    QMS_REQUIRE(rows && ((uintptr_t)rows & 15) == 0 && ldrows >= cols && ldrows % 8 == 0, QMS_CUDA_EINVAL,
                "prompt_append: rows must be 16-byte aligned device memory, at least %lld values and a multiple of 8 apart", (long long)cols);
    QMS_REQUIRE(q_norm && k_norm && rope_cos && rope_sin && n_rope > 0, QMS_CUDA_EINVAL,
                "prompt_append: NULL norm weights or rotation tables");
#define QMS_ROWS(D_, OT) \
    return launch_rows_append<D_>(a, pages->type, qkv, ldqkv, q_norm, k_norm, eps, rope_cos, rope_sin, n_rope, (OT *)rows, ldrows, (cudaStream_t)stream)
    if (type == QMS_T_F16) {
        if (D == 128) QMS_ROWS(128, __half); else QMS_ROWS(64, __half);
    } else {
        if (D == 128) QMS_ROWS(128, __nv_bfloat16); else QMS_ROWS(64, __nv_bfloat16);
    }
#undef QMS_ROWS
}

int qms_cuda_paged_values(const QmsCudaPages *pages, float *k, float *v, void *stream) {
    clear_error();
    const QmsCudaPagedBatch none = {};
    Paged a;
    const int rc = paged_args("paged_values", pages, &none, pages ? pages->n_head_kv : 1, nullptr, a);
    if (rc) return rc;
    QMS_REQUIRE(k && v && (((uintptr_t)k | (uintptr_t)v) & 15) == 0, QMS_CUDA_EINVAL, "paged_values: k and v must be 16-byte aligned device memory");
    const int D = pages->head_dim;
    const int64_t ctas = (((int64_t)a.n_pages << a.page_log) * a.Hk * (D / 8) + 255) / 256;
    const dim3 grid((unsigned)std::min<int64_t>(ctas, 148 * 8), 2);
    if (D == 128) QMS_CK(launch_pdl(k_paged_values<128>, grid, dim3(256), 0, (cudaStream_t)stream, a, pages->type, k, v));
    else QMS_CK(launch_pdl(k_paged_values<64>, grid, dim3(256), 0, (cudaStream_t)stream, a, pages->type, k, v));
    return QMS_CUDA_OK;
}

int64_t qms_cuda_paged_attention_ws(const QmsCudaPages *pages, const QmsCudaPagedBatch *batch, int n_head) {
    Paged a;
    const int rc = paged_args("paged_attention_ws", pages, batch, n_head, nullptr, a);
    if (rc) return rc;
    PagedPlan p;
    paged_plan(a, pages->type, pages->head_dim, p);
    return paged_ws_bytes(a, pages->head_dim, p);
}

int qms_cuda_paged_attention(const QmsCudaPages *pages, const QmsCudaPagedBatch *batch, const float *q, int64_t ldq,
                             int n_head, float scale, float *out, int64_t ldo, void *ws, int64_t ws_bytes, int *err,
                             void *stream) {
    clear_error();
    Paged a;
    int rc = paged_args("paged_attention", pages, batch, n_head, err, a);
    if (rc) return rc;
    if (a.n_tok == 0) return QMS_CUDA_OK;
    const int D = pages->head_dim;
    if ((rc = paged_rows("paged_attention", "q", q, ldq, (int64_t)n_head * D))) return rc;
    if ((rc = paged_rows("paged_attention", "out", out, ldo, (int64_t)n_head * D))) return rc;
    PagedPlan p;
    paged_plan(a, pages->type, D, p);
    const int64_t need = paged_ws_bytes(a, D, p);
    QMS_REQUIRE(need == 0 || (ws && ((uintptr_t)ws & 255) == 0 && ws_bytes >= need), QMS_CUDA_EINVAL,
                "paged_attention: needs a 256-byte aligned workspace of %lld bytes", (long long)need);
    return launch_paged_attention(a, pages->type, D, p, q, ldq, scale, out, ldo, ws, (cudaStream_t)stream);
}

}  // extern "C"
