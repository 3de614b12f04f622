// The INT8 key/value cache (include/sgq_decoder.h): rows of head_dim codes with one fp32 scale per (sequence, head,
// position), written with the rotary embedding, read back as fp32, and read by the decode attention.
//
// A row is quantized by the library's per-row INT8 quantizer, bit for bit: a = max(1e-8, max |r|), scale = a / 127,
// code = clamp(round_half_away(r * (127 / a))), every operation rounded to fp32 (NaN -> +127, an infinity makes the scale
// infinite).  The rotation in front of it rounds every product and sum to fp32 (no contraction), so codes and scales are a
// function of the inputs alone: the prompt's store, the decode step's append and a host restatement agree in every bit.
#include "sgq_common.cuh"
#include "gemv_prepare.cuh"
#include "sm100_ptx.cuh"

#include "../../include/sgq_decoder.h"

#include <cooperative_groups.h>
#include <math_constants.h>

namespace sgq {

namespace {

constexpr int kMaxHeadDim = 256;
constexpr int64_t kMaxPositions = 1ll << 30;       // of the attention: positions and strides between tiles in 32 bits

// (x1, x2) of a rotary pair, every operation rounded (src/ops.cpp:1737-1738)
__device__ __forceinline__ void rotate_pair(float& x1, float& x2, float c, float s) {
    const float a = __fsub_rn(__fmul_rn(x1, c), __fmul_rn(x2, s));
    x2 = __fadd_rn(__fmul_rn(x2, c), __fmul_rn(x1, s));
    x1 = a;
}

__device__ __forceinline__ float4 ld4(const float* p) { return *reinterpret_cast<const float4*>(p); }

// ---- store ------------------------------------------------------------------------------------------------------------
// One group of LPR lanes per row (a head of q, k or v of one token); a lane owns the values 4l .. 4l+3 of the first half of the
// row and of the second half, so that a rotary pair sits in one lane and only the absmax crosses lanes.
constexpr int kStoreThreads = 256;
template <int LPR>
__global__ void __launch_bounds__(kStoreThreads) rope_kv_store_int8_kernel(const float* qkv, int64_t qkv_stride, int t_new, int n_heads, int n_kv,
                                                                           int head_dim, const float* __restrict__ cos_t,
                                                                           const float* __restrict__ sin_t, int64_t table_rows,
                                                                           const int32_t* __restrict__ pos_p, int64_t pos_stride,
                                                                           const int32_t* __restrict__ n_new,
                                                                           const int32_t* __restrict__ rope_offset, float* q_out, int64_t q_stride,
                                                                           int8_t* __restrict__ kc, float* __restrict__ ks, int8_t* __restrict__ vc,
                                                                           float* __restrict__ vs, int64_t max_seq) {
    pdl_launch_dependents();
    pdl_wait();
    const int64_t m = blockIdx.x;
    const int b = static_cast<int>(m / t_new), i = static_cast<int>(m - static_cast<int64_t>(b) * t_new);
    const int r = blockIdx.y * (kStoreThreads / LPR) + threadIdx.x / LPR;      // row of the token: q heads, k heads, v heads
    const int l = threadIdx.x % LPR;
    const int half = head_dim >> 1;
    const bool in = r < n_heads + 2 * n_kv && 4 * l < half;
    const float* row = qkv + m * qkv_stride + static_cast<int64_t>(r) * head_dim + 4 * l;
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f), c = a;
    if (in) { a = ld4(row); c = ld4(row + half); }
    const int64_t pos = static_cast<int64_t>(pos_p[b * pos_stride]) + i;
    const int64_t turn = pos + (rope_offset ? *rope_offset : 0);
    // a token behind the sequence's own count, outside the cache or outside the tables leaves everything as it was
    if (pos < 0 || pos >= max_seq || turn < 0 || turn >= table_rows || (n_new && i >= n_new[b])) return;         // uniform over the block
    if (r < n_heads + n_kv && in) {
        const int64_t at = turn * half + 4 * l;
        const float4 co = ld4(cos_t + at), si = ld4(sin_t + at);
        rotate_pair(a.x, c.x, co.x, si.x);
        rotate_pair(a.y, c.y, co.y, si.y);
        rotate_pair(a.z, c.z, co.z, si.z);
        rotate_pair(a.w, c.w, co.w, si.w);
    }
    float top = 1e-8f;
    top = absmax_step(absmax_step(absmax_step(absmax_step(top, a.x), a.y), a.z), a.w);
    top = absmax_step(absmax_step(absmax_step(absmax_step(top, c.x), c.y), c.z), c.w);
#pragma unroll
    for (int o = LPR / 2; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    if (!in) return;
    if (r < n_heads) {
        float* o = q_out + m * q_stride + static_cast<int64_t>(r) * head_dim + 4 * l;
        *reinterpret_cast<float4*>(o) = a;
        *reinterpret_cast<float4*>(o + half) = c;
        return;
    }
    const bool is_v = r >= n_heads + n_kv;
    const int h = r - n_heads - (is_v ? n_kv : 0);
    const int64_t at = (static_cast<int64_t>(b) * n_kv + h) * max_seq + pos;
    const float inv = __fdiv_rn(127.0f, top);
    auto q4 = [&](const float4& v) {
        return make_char4(quantize_code<127, -127>(v.x, inv), quantize_code<127, -127>(v.y, inv), quantize_code<127, -127>(v.z, inv),
                          quantize_code<127, -127>(v.w, inv));
    };
    int8_t* codes = (is_v ? vc : kc) + at * head_dim + 4 * l;
    *reinterpret_cast<char4*>(codes) = q4(a);
    *reinterpret_cast<char4*>(codes + half) = q4(c);
    if (l == 0) (is_v ? vs : ks)[at] = __fdiv_rn(top, 127.0f);
}

// ---- read back --------------------------------------------------------------------------------------------------------
constexpr int kLoadThreads = 256, kLoadPerThread = 4;
__global__ void __launch_bounds__(kLoadThreads) kv_load_int8_kernel(const int8_t* __restrict__ kc, const float* __restrict__ ks,
                                                                    const int8_t* __restrict__ vc, const float* __restrict__ vs, int64_t max_seq,
                                                                    int head_dim, int64_t vecs, int64_t chunks, int64_t src_heads,
                                                                    float* __restrict__ k_out, float* __restrict__ v_out, int64_t out_max_seq,
                                                                    int64_t out_row0) {
    pdl_launch_dependents();
    pdl_wait();
    const int64_t bh = blockIdx.x / chunks, chunk = blockIdx.x - bh * chunks;
    const int64_t src = (bh % src_heads) * max_seq;               // src_heads: heads of all source sequences, or of the one shared
    const bool is_v = blockIdx.y != 0;
    const int8_t* codes = (is_v ? vc : kc) + src * head_dim;
    const float* scales = (is_v ? vs : ks) + src;
    float* out = (is_v ? v_out : k_out) + (bh * out_max_seq + out_row0) * head_dim;
    const uint32_t per_row = static_cast<uint32_t>(head_dim) / 4;
    char4 c[kLoadPerThread];
    float s[kLoadPerThread];
#pragma unroll
    for (int u = 0; u < kLoadPerThread; ++u) {
        const int64_t v = (chunk * kLoadPerThread + u) * kLoadThreads + threadIdx.x;
        if (v < vecs) {
            c[u] = *reinterpret_cast<const char4*>(codes + 4 * v);
            s[u] = scales[v / per_row];
        }
    }
#pragma unroll
    for (int u = 0; u < kLoadPerThread; ++u) {
        const int64_t v = (chunk * kLoadPerThread + u) * kLoadThreads + threadIdx.x;
        if (v < vecs) *reinterpret_cast<float4*>(out + 4 * v) = make_float4(c[u].x * s[u], c[u].y * s[u], c[u].z * s[u], c[u].w * s[u]);
    }
}

// ---- decode attention -------------------------------------------------------------------------------------------------
// Both products of the attention run on the tensor cores as exact integer products (mma.sync m16n8k32, s8 x s8 -> s32): the
// codes go in as they lie in memory, the query and the softmax weights as 24-bit fixed point split into three balanced
// base-256 digits (the arithmetic of gemv_prepare.cuh), one digit per column of the small operand.
//
//   scores   A = 16 rows of the cache x 32 values, B = 32 values x 8 columns.  A lane (g, t) = (lane / 4, lane % 4) of the
//            warp loads the 16-byte chunks t (and 4 + t) of the rows 4g .. 4g+3 of a tile of 32 positions: these ARE the A
//            fragments, the order of the head dimension inside them being the same in the query's digits.  Columns 2t, 2t+1
//            of a "main" column set hold digits 2 and 1 of query t, those of the "low" set digit 0 of queries t and
//            t + 4, so a lane finds all digits of its one or two queries in its own accumulators.
//   weights  w = p * value scale, relative to the largest |w| of the tile and query: their digits cross the warp by shuffles
//            (rows of the accumulators become the contraction index).
//   output   A = 16 values x 32 positions: a lane loads HD/8 consecutive values of 8 positions and transposes 4 x 4 bytes
//            with byte permutes.  B = 32 positions x 8 columns of weight digits.
//
// Scores and outputs leave the integer domain once per tile (sum of 32 or HD products below 2^22, exact as fp32), scaled
// and added in fp32 with the running maximum and sum of the softmax.  A lane holds the scores of positions 4g .. 4g+3 and
// the values [HD/8 g, HD/8 (g+1)) of the outputs of queries t and t + 4.
struct CacheView {
    int8_t* kc;
    float* ks;
    int8_t* vc;
    float* vs;
    int64_t max_seq;
};

// D = A(16x32, s8) * B(32x8, s8) + magic (see gemv_prepare.cuh: the sum read as fp32 bits is 12582912 + S), and D += A * B
__device__ __forceinline__ void mma_first(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "r"(kMagicBits));
}
__device__ __forceinline__ void mma_next(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// digit sums (2: highest) of one exact sum, as fp32
__device__ __forceinline__ float join_digits(int d2, int d1, int d0) {
    const float f2 = __int_as_float(d2) - kMagicF, f1 = __int_as_float(d1) - kMagicF, f0 = __int_as_float(d0) - kMagicF;
    return fmaf(f2, 65536.0f, fmaf(f1, 256.0f, f0));
}
__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float exp2_approx(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

constexpr int kTile = 32;              // positions per step of a warp

// One warp's running attention of up to NQ (4 or 8) queries over tiles of one kv head's rows.
template <int HD, int NQ>
struct WarpAttention {
    static constexpr int KW = HD / 16;         // 32-bit words of a key row per lane
    static constexpr int VB = HD / 8;          // values per lane and position
    static constexpr int VW = VB / 4;
    static constexpr int NS = NQ / 4, NT = NS + 1;
    static constexpr int kQueryBytes = 3 * HD; // digit planes of one query: [digit][HD]

    uint32_t k[4][KW], v[8][VW], bq[NT][KW];
    float ks[4], vs[4];
    float qu[NS], m[NS], l[NS], o[NS][VB];
    int g, t;

    __device__ __forceinline__ void init(int lane) {
        g = lane >> 2;
        t = lane & 3;
#pragma unroll
        for (int s = 0; s < NS; ++s) {
            m[s] = -CUDART_INF_F;
            l[s] = 0.f;
#pragma unroll
            for (int j = 0; j < VB; ++j) o[s][j] = 0.f;
        }
    }
    // the digit planes and units of NQ queries, written by query_digits below
    __device__ __forceinline__ void load_queries(const uint8_t* planes, const float* units) {
        auto rd = [&](uint32_t (&w)[KW], int query, int digit, bool zero) {
            const uint8_t* p = planes + query * kQueryBytes + digit * HD + 16 * t;
#pragma unroll
            for (int c = 0; c < KW / 4; ++c) {
                const uint4 x = *reinterpret_cast<const uint4*>(p + 64 * c);
                w[4 * c] = zero ? 0u : x.x; w[4 * c + 1] = zero ? 0u : x.y; w[4 * c + 2] = zero ? 0u : x.z; w[4 * c + 3] = zero ? 0u : x.w;
            }
        };
#pragma unroll
        for (int s = 0; s < NS; ++s) {
            rd(bq[s], 4 * s + (g >> 1), 2 - (g & 1), false);
            qu[s] = units[4 * s + t];
        }
        if (NS == 2) rd(bq[NS], (g >> 1) + 4 * (g & 1), 0, false);
        else rd(bq[NS], g >> 1, 0, (g & 1) != 0);
    }
    __device__ __forceinline__ void load_k(const int8_t* kc, const float* ksc, int t0, int t1) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            int key = t0 + 4 * g + i;
            key = key < t1 ? key : t1 - 1;                    // clamped: masked in step()
            const uint4* p = reinterpret_cast<const uint4*>(kc + static_cast<int64_t>(key) * HD + 16 * t);
#pragma unroll
            for (int c = 0; c < KW / 4; ++c) {
                const uint4 x = p[4 * c];
                k[i][4 * c] = x.x; k[i][4 * c + 1] = x.y; k[i][4 * c + 2] = x.z; k[i][4 * c + 3] = x.w;
            }
            ks[i] = ksc[key];
        }
    }
    __device__ __forceinline__ void load_v(const int8_t* vc, const float* vsc, int t0, int t1) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            int key = t0 + 4 * g + i;
            key = key < t1 ? key : t1 - 1;
            vs[i] = vsc[key];
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            int key = t0 + 4 * t + (i & 3) + 16 * (i >> 2);
            key = key < t1 ? key : t1 - 1;
            const int8_t* p = vc + static_cast<int64_t>(key) * HD + VB * g;
            if constexpr (VW == 4) {
                const uint4 x = *reinterpret_cast<const uint4*>(p);
                v[i][0] = x.x; v[i][1] = x.y; v[i][2] = x.z; v[i][3] = x.w;
            } else {
                const uint2 x = *reinterpret_cast<const uint2*>(p);
                v[i][0] = x.x; v[i][1] = x.y;
            }
        }
    }
    // scores of the loaded keys: sc[s][i] of position t0 + 4g + i and query t + 4s, in base-2 units
    __device__ __forceinline__ void scores(float (&sc)[NS][4], int t0, int t1) {
        int acc[2][NT][4];
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                mma_first(acc[h][n], k[2 * h][0], k[2 * h + 1][0], k[2 * h][1], k[2 * h + 1][1], bq[n][0], bq[n][1]);
#pragma unroll
                for (int c = 1; c < KW / 2; ++c)
                    mma_next(acc[h][n], k[2 * h][2 * c], k[2 * h + 1][2 * c], k[2 * h][2 * c + 1], k[2 * h + 1][2 * c + 1], bq[n][2 * c], bq[n][2 * c + 1]);
            }
#pragma unroll
        for (int s = 0; s < NS; ++s)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int h = i >> 1, r = 2 * (i & 1);
                const float x = join_digits(acc[h][s][r], acc[h][s][r + 1], acc[h][NS][r + s]) * qu[s];
                const float y = fmaf(x, ks[i], ks[i] - ks[i]);          // NaN for a row whose scale is not finite
                sc[s][i] = t0 + 4 * g + i < t1 ? y : -CUDART_INF_F;
            }
    }
    // the tile's weights into the running softmax, and its values into the outputs
    __device__ __forceinline__ void accumulate(float (&sc)[NS][4], int t0, int t1) {
        uint32_t bw[NT][2];
        float corr[NS], unit[NS];
        uint32_t w0[NS], w1[NS], w2[NS];
#pragma unroll
        for (int s = 0; s < NS; ++s) {
            float top = fmaxf(fmaxf(sc[s][0], sc[s][1]), fmaxf(sc[s][2], sc[s][3]));
#pragma unroll
            for (int d = 4; d < 32; d <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
            const float mn = fmaxf(m[s], top);
            corr[s] = m[s] == mn ? 1.0f : exp2_approx(m[s] - mn);
            m[s] = mn;
            float w[4], sum = 0.f, most = 0.f;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float p = sc[s][i] == -CUDART_INF_F ? 0.f : exp2_approx(sc[s][i] - mn);
                sum += p;
                w[i] = p * (t0 + 4 * g + i < t1 ? vs[i] : 0.f);
                most = max_nan(most, fabsf(w[i]));
            }
            l[s] = fmaf(l[s], corr[s], sum);
#pragma unroll
            for (int d = 4; d < 32; d <<= 1) most = max_nan(most, __shfl_xor_sync(0xffffffffu, most, d));
            // a tile whose weights vanish against the running maximum contributes nothing; NaN and infinity pass
            const float per = most < 1e-30f ? 0.f : __fdividef(kDigitRange, most);
            unit[s] = most * (1.0f / kDigitRange);
            uint32_t d[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) d[i] = digit_bytes(__float2int_rn(w[i] * per));
            const uint32_t x = __byte_perm(d[0], d[1], 0x5140), y = __byte_perm(d[2], d[3], 0x5140);
            w0[s] = __byte_perm(x, y, 0x5410);
            w1[s] = __byte_perm(x, y, 0x7632);
            w2[s] = __byte_perm(__byte_perm(d[0], d[1], 0x0062), __byte_perm(d[2], d[3], 0x0062), 0x5410);
        }
        // B fragments: lane (column g, position quad t or t + 4) takes the digit words that lane (quad, query) holds
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const int from = 4 * (t + 4 * half) + (g >> 1);
#pragma unroll
            for (int s = 0; s < NS; ++s) {
                const uint32_t hi = __shfl_sync(0xffffffffu, w2[s], from), mid = __shfl_sync(0xffffffffu, w1[s], from);
                bw[s][half] = (g & 1) ? mid : hi;
            }
            const uint32_t lo = __shfl_sync(0xffffffffu, w0[0], from);
            const uint32_t lo2 = NS == 2 ? __shfl_sync(0xffffffffu, w0[NS - 1], from) : 0u;
            bw[NS][half] = (g & 1) ? lo2 : lo;
        }
#pragma unroll
        for (int wd = 0; wd < VW; ++wd) {
            uint32_t a[2][4];                   // [quad half][value 4 wd + r]: four positions each
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                const uint32_t x0 = v[4 * q][wd], x1 = v[4 * q + 1][wd], x2 = v[4 * q + 2][wd], x3 = v[4 * q + 3][wd];
                const uint32_t p0 = __byte_perm(x0, x1, 0x5140), p1 = __byte_perm(x0, x1, 0x7362);
                const uint32_t p2 = __byte_perm(x2, x3, 0x5140), p3 = __byte_perm(x2, x3, 0x7362);
                a[q][0] = __byte_perm(p0, p2, 0x5410);
                a[q][1] = __byte_perm(p0, p2, 0x7632);
                a[q][2] = __byte_perm(p1, p3, 0x5410);
                a[q][3] = __byte_perm(p1, p3, 0x7632);
            }
#pragma unroll
            for (int pr = 0; pr < 2; ++pr) {    // values 4 wd + 2 pr (rows g) and 4 wd + 2 pr + 1 (rows g + 8)
                int acc[NT][4];
#pragma unroll
                for (int n = 0; n < NT; ++n) mma_first(acc[n], a[0][2 * pr], a[0][2 * pr + 1], a[1][2 * pr], a[1][2 * pr + 1], bw[n][0], bw[n][1]);
#pragma unroll
                for (int s = 0; s < NS; ++s)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        float& out = o[s][4 * wd + 2 * pr + e];
                        out = fmaf(out, corr[s], join_digits(acc[s][2 * e], acc[s][2 * e + 1], acc[NS][2 * e + s]) * unit[s]);
                    }
            }
        }
    }
    // tiles t0, t0 + stride, ... below t1 of the rows at kc / vc; the first one's loads may be under way (`loaded`)
    __device__ __forceinline__ void run(const int8_t* kc, const float* ksc, const int8_t* vc, const float* vsc, int t0, int t1, int stride) {
        for (; t0 < t1; t0 += stride) {
            float sc[NS][4];
            scores(sc, t0, t1);
            const bool more = t1 - t0 > stride;
            if (more) load_k(kc, ksc, t0 + stride, t1);       // on their way while this tile's values are added up
            accumulate(sc, t0, t1);
            if (more) load_v(vc, vsc, t0 + stride, t1);
        }
    }
    // (max, sum, value) of every query into sm_ml[NQ][2], sm_o[NQ][HD]
    __device__ __forceinline__ void store(float* sm_ml, float* sm_o) {
#pragma unroll
        for (int s = 0; s < NS; ++s) {
#pragma unroll
            for (int d = 4; d < 32; d <<= 1) l[s] += __shfl_xor_sync(0xffffffffu, l[s], d);
            const int q = t + 4 * s;
            if (g == 0) { sm_ml[2 * q] = m[s]; sm_ml[2 * q + 1] = l[s]; }
#pragma unroll
            for (int j = 0; j < VB; j += 4)
                *reinterpret_cast<float4*>(sm_o + q * HD + VB * g + j) = make_float4(o[s][j], o[s][j + 1], o[s][j + 2], o[s][j + 3]);
        }
    }
};

// One warp, one row of HD values (VEC consecutive per lane), rotated if `turn`.
template <int HD>
__device__ __forceinline__ void load_row(float (&v)[HD / 32], const float* row, const float* cos_row, const float* sin_row, bool turn, int lane) {
    constexpr int VEC = HD / 32;
#pragma unroll
    for (int j = 0; j < VEC; ++j) v[j] = row[lane * VEC + j];
    if (!turn) return;
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
        const float other = __shfl_xor_sync(0xffffffffu, v[j], 16);
        const float c = cos_row[(lane & 15) * VEC + j], s = sin_row[(lane & 15) * VEC + j];
        float x1 = lane < 16 ? v[j] : other, x2 = lane < 16 ? other : v[j];
        rotate_pair(x1, x2, c, s);
        v[j] = lane < 16 ? x1 : x2;
    }
}

// The rotated query as digit planes [3][HD] and its unit, which carries 1/sqrt(HD) and log2(e).  A NaN or an infinity in the
// query makes the unit NaN or infinite and the digits zero: every score is NaN.
template <int HD>
__device__ __forceinline__ void query_digits(const float (&v)[HD / 32], uint8_t* planes, float* unit, int lane) {
    constexpr int VEC = HD / 32;
    uint32_t top = 0;
#pragma unroll
    for (int j = 0; j < VEC; ++j) top = max(top, __float_as_uint(v[j]) & 0x7FFFFFFFu);
    top = __reduce_max_sync(0xffffffffu, top);
    const float most = __uint_as_float(top);
    const bool fine = top < 0x7F800000u && most >= 1e-30f;
    const float per = fine ? __fdiv_rn(kDigitRange, most) : 0.f;
    uint32_t d[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) d[j] = fine ? digit_bytes(__float2int_rn(__fmul_rn(v[j], per))) : 0u;
#pragma unroll
    for (int j = 0; j < 3; ++j) {
        if constexpr (VEC == 4)
            *reinterpret_cast<uint32_t*>(planes + j * HD + lane * 4) = gather_byte(d[0], d[1], d[2], d[3], j);
        else
            *reinterpret_cast<uint16_t*>(planes + j * HD + lane * 2) = static_cast<uint16_t>(__byte_perm(d[0], d[1], 0x0040 + 0x11 * j));
    }
    if (lane == 0) *unit = top >= 0x7F800000u ? CUDART_NAN_F : (fine ? __fmul_rn(__fdiv_rn(most, kDigitRange), rsqrtf(static_cast<float>(HD)) * 1.4426950408889634f) : 0.f);
}

// One warp quantizes a row into the cache.
template <int HD>
__device__ __forceinline__ void append_row(const float (&v)[HD / 32], int8_t* codes, float* scale, int lane) {
    constexpr int VEC = HD / 32;
    float top = 1e-8f;
#pragma unroll
    for (int j = 0; j < VEC; ++j) top = absmax_step(top, v[j]);
    top = warp_max(top);
    const float inv = __fdiv_rn(127.0f, top);
    if constexpr (VEC == 4)
        *reinterpret_cast<char4*>(codes + lane * 4) = make_char4(quantize_code<127, -127>(v[0], inv), quantize_code<127, -127>(v[1], inv),
                                                                 quantize_code<127, -127>(v[2], inv), quantize_code<127, -127>(v[3], inv));
    else
        *reinterpret_cast<char2*>(codes + lane * 2) = make_char2(quantize_code<127, -127>(v[0], inv), quantize_code<127, -127>(v[1], inv));
    if (lane == 0) *scale = __fdiv_rn(top, 127.0f);
}

struct DecodeArgs {
    const float* qkv;
    int64_t qkv_stride;
    int n_heads, n_kv, batch;
    const float* cos_t;
    const float* sin_t;
    const int32_t* pos;
    int64_t pos_stride;
    CacheView own, first;              // first: the shared prefix (prefix_len != NULL)
    const int32_t* prefix_len;
    float* out;
    int64_t out_stride;
    int pmode, nmain, nlow;
    uint8_t* planes;
    const float* part_ml;              // prefix partial results [kv head][row][split][2] and [...][HD]
    const float* part_o;
    int parts;
};

__device__ __forceinline__ int64_t prefix_rows(const DecodeArgs& a) {
    if (!a.prefix_len) return 0;
    const int64_t p = *a.prefix_len;
    return p < 0 ? 0 : (p > a.first.max_seq ? a.first.max_seq : p);
}

constexpr int kWarps = 8;

// Joins `n` partial results (max, sum at ml[2 i stride_ml], value at o[i * stride_o]) of one output value into (M, L, A)
struct Joined {
    float M, L, A;
};
__device__ __forceinline__ void join_part(Joined& j, float m, float l, float a) {
    const float mn = fmaxf(j.M, m);
    const float x = j.M == mn ? 1.0f : exp2_approx(j.M - mn), y = m == mn ? 1.0f : exp2_approx(m - mn);
    j.L = fmaf(j.L, x, l * y);
    j.A = fmaf(j.A, x, a * y);
    j.M = mn;
}

// grid (batch * kv heads, query blocks, S) in clusters of S along z: the S CTAs of a cluster split the positions of one (sequence,
// kv head); the warp that owns the last position appends the new token's row first.  Warps are joined through shared memory and
// CTAs through distributed shared memory, head g by CTA g % S.
template <int HD, int NQ>
__global__ void __launch_bounds__(kWarps * 32) attn_decode_int8_kernel(const DecodeArgs a) {
    namespace cg = cooperative_groups;
    using Attn = WarpAttention<HD, NQ>;
    __shared__ __align__(16) uint8_t sm_q[NQ * Attn::kQueryBytes];
    __shared__ float sm_unit[NQ];
    __shared__ float sm_ml[kWarps][NQ][2];
    __shared__ __align__(16) float sm_o[kWarps][NQ][HD];
    __shared__ float sm_part_ml[NQ][2];
    __shared__ __align__(16) float sm_part[NQ][HD];
    pdl_launch_dependents();
    pdl_wait();
    const int b = blockIdx.x / a.n_kv, hk = blockIdx.x - b * a.n_kv, G = a.n_heads / a.n_kv;
    const int q0 = blockIdx.y * NQ, nq = min(NQ, G - q0);             // this block's queries of the group
    const int split = blockIdx.z, S = gridDim.z;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int64_t pos = a.pos[b * a.pos_stride];
    const bool live = pos >= 0 && pos < a.own.max_seq;
    const int64_t P = prefix_rows(a);
    const int n = live ? static_cast<int>(pos) + 1 : 0;
    const int chunk = ((n + S - 1) / S + kTile - 1) / kTile * kTile;
    const int t0 = min(static_cast<int64_t>(split) * chunk, static_cast<int64_t>(n)), t1 = min(static_cast<int64_t>(t0) + chunk, static_cast<int64_t>(n));
    const int64_t base = (static_cast<int64_t>(b) * a.n_kv + hk) * a.own.max_seq;
    const int8_t* kc = a.own.kc + base * HD;
    const int8_t* vc = a.own.vc + base * HD;
    const float* ks = a.own.ks + base;
    const float* vs = a.own.vs + base;
    const float* row = a.qkv + b * a.qkv_stride;
    const float* cos_row = a.cos_t + (live ? P + pos : 0) * (HD / 2);
    const float* sin_row = a.sin_t + (live ? P + pos : 0) * (HD / 2);

    Attn w;
    w.init(lane);
    const int first = t0 + warp * kTile;
    const bool owner = t1 == n && n > 0 && t1 > t0 && (n - 1 - t0) / kTile % kWarps == warp;
    if (owner) {
        // every query block of the group attends to the new row, so every one's owner writes it (the same bits)
        float v[HD / 32];
        load_row<HD>(v, row + static_cast<int64_t>(a.n_heads + hk) * HD, cos_row, sin_row, true, lane);
        append_row<HD>(v, a.own.kc + (base + pos) * HD, a.own.ks + base + pos, lane);
        load_row<HD>(v, row + static_cast<int64_t>(a.n_heads + a.n_kv + hk) * HD, cos_row, sin_row, false, lane);
        append_row<HD>(v, a.own.vc + (base + pos) * HD, a.own.vs + base + pos, lane);
        __syncwarp();
    }
    if (first < t1) {
        w.load_k(kc, ks, first, t1);
        w.load_v(vc, vs, first, t1);
    }
    for (int q = warp; q < NQ; q += kWarps) {
        float v[HD / 32];
        if (q < nq && live) {
            load_row<HD>(v, row + static_cast<int64_t>(hk * G + q0 + q) * HD, cos_row, sin_row, true, lane);
        } else {
#pragma unroll
            for (int j = 0; j < HD / 32; ++j) v[j] = 0.f;
        }
        query_digits<HD>(v, sm_q + q * Attn::kQueryBytes, sm_unit + q, lane);
    }
    __syncthreads();
    w.load_queries(sm_q, sm_unit);
    w.run(kc, ks, vc, vs, first, t1, kWarps * kTile);
    w.store(&sm_ml[warp][0][0], &sm_o[warp][0][0]);
    __syncthreads();
    for (int i = threadIdx.x; i < nq * HD; i += kWarps * 32) {
        const int q = i / HD, d = i % HD;
        Joined j = {-CUDART_INF_F, 0.f, 0.f};
#pragma unroll
        for (int u = 0; u < kWarps; ++u) join_part(j, sm_ml[u][q][0], sm_ml[u][q][1], sm_o[u][q][d]);
        sm_part[q][d] = j.A;
        if (d == 0) { sm_part_ml[q][0] = j.M; sm_part_ml[q][1] = j.L; }
    }
    cg::cluster_group cluster = cg::this_cluster();
    cluster.sync();
    const int64_t R = static_cast<int64_t>(a.batch) * G;
    for (int q = split; q < nq; q += S) {
        if (threadIdx.x < HD) {
            const int d = threadIdx.x;
            Joined j = {-CUDART_INF_F, 0.f, 0.f};
            for (int r = 0; r < S; ++r) {
                const float* ml = cluster.map_shared_rank(&sm_part_ml[q][0], r);
                join_part(j, ml[0], ml[1], cluster.map_shared_rank(&sm_part[q][0], r)[d]);
            }
            if (live) {
                const int64_t at = (hk * R + static_cast<int64_t>(b) * G + q0 + q) * a.parts;
                for (int p = 0; p < a.parts; ++p) join_part(j, a.part_ml[2 * (at + p)], a.part_ml[2 * (at + p) + 1], a.part_o[(at + p) * HD + d]);
            }
            const float o = j.L == 0.f ? 0.f : j.A / j.L;
            a.out[b * a.out_stride + static_cast<int64_t>(hk * G + q0 + q) * HD + d] = o;
            sm_o[0][0][d] = o;
        }
        if (a.planes != nullptr) {
            // the same values as prepared activations of the [batch, n_heads * HD] matrix: a head is HD / 32 whole groups
            __syncthreads();
            if (warp == 0) {
                const bool in = lane < HD / 8;
                float v[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) v[j] = in ? sm_o[0][0][lane * 8 + j] : 0.f;
                const PreparedParts pp = prepared_parts(a.planes, static_cast<size_t>(a.n_heads) * (HD / 32), a.nmain, a.nlow);
                convert_groups<kOrderNibble>(v, b, a.batch, static_cast<size_t>(hk * G + q0 + q) * (HD / 32), a.pmode, a.nmain, a.nlow, 0.0625f, pp, in);
            }
            __syncthreads();
        }
    }
    cluster.sync();                                                    // keeps shared memory alive until it has been read
}

// Partial attention of every sequence's queries to the shared prefix.  grid (kv heads, splits of the prefix, blocks of 8 QW rows),
// the rows of a kv head being its queries (b, g) in the order b * G + g.  A warp carries 8 rows; QW warps of a block take
// the same positions (their loads meet in L1) and the KW = 8 / QW groups of warps take alternate tiles.
template <int HD>
__global__ void __launch_bounds__(kWarps * 32) attn_prefix_int8_kernel(const DecodeArgs a, int QW, float* __restrict__ part_ml, float* __restrict__ part_o) {
    constexpr int NQ = 8;
    using Attn = WarpAttention<HD, NQ>;
    constexpr int kDigits = kWarps * NQ * Attn::kQueryBytes, kOuts = kWarps * NQ * HD * 4;
    __shared__ __align__(16) uint8_t sm[kDigits > kOuts ? kDigits : kOuts];      // the queries' digits, then the warps' outputs
    __shared__ float sm_unit[kWarps * NQ];
    __shared__ float sm_ml[kWarps][NQ][2];
    pdl_launch_dependents();
    pdl_wait();
    const int hk = blockIdx.x, split = blockIdx.y, splits = gridDim.y, G = a.n_heads / a.n_kv;
    const int64_t R = static_cast<int64_t>(a.batch) * G, r0 = static_cast<int64_t>(blockIdx.z) * QW * NQ;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, KW = kWarps / QW, qg = warp % QW, kw = warp / QW;
    const int n = static_cast<int>(prefix_rows(a));
    const int chunk = ((n + splits - 1) / splits + kTile - 1) / kTile * kTile;
    const int t0 = min(static_cast<int64_t>(split) * chunk, static_cast<int64_t>(n)), t1 = min(static_cast<int64_t>(t0) + chunk, static_cast<int64_t>(n));
    const int64_t base = static_cast<int64_t>(hk) * a.first.max_seq;
    const int8_t* kc = a.first.kc + base * HD;
    const int8_t* vc = a.first.vc + base * HD;
    const float* ks = a.first.ks + base;
    const float* vs = a.first.vs + base;
    Attn w;
    w.init(lane);
    const int first = t0 + kw * kTile;
    if (first < t1) {
        w.load_k(kc, ks, first, t1);
        w.load_v(vc, vs, first, t1);
    }
    for (int i = warp; i < QW * NQ; i += kWarps) {
        const int64_t r = r0 + i;
        const int64_t b = r < R ? r / G : 0;
        const int64_t pos = a.pos[b * a.pos_stride];
        float v[HD / 32];
        if (r < R && pos >= 0 && pos < a.own.max_seq) {
            load_row<HD>(v, a.qkv + b * a.qkv_stride + (hk * G + r - b * G) * HD, a.cos_t + (n + pos) * (HD / 2), a.sin_t + (n + pos) * (HD / 2), true, lane);
        } else {
#pragma unroll
            for (int j = 0; j < HD / 32; ++j) v[j] = 0.f;
        }
        query_digits<HD>(v, sm + i * Attn::kQueryBytes, sm_unit + i, lane);
    }
    __syncthreads();
    w.load_queries(sm + qg * NQ * Attn::kQueryBytes, sm_unit + qg * NQ);
    w.run(kc, ks, vc, vs, first, t1, KW * kTile);
    __syncthreads();                                                    // everyone has read the digits
    float* sm_o = reinterpret_cast<float*>(sm);
    w.store(&sm_ml[warp][0][0], sm_o + warp * NQ * HD);
    __syncthreads();
    for (int i = threadIdx.x; i < QW * NQ * HD; i += kWarps * 32) {
        const int q = i / HD, d = i % HD;
        if (r0 + q >= R) break;
        Joined j = {-CUDART_INF_F, 0.f, 0.f};
        for (int u = 0; u < KW; ++u) {
            const int wi = q / NQ + u * QW;
            join_part(j, sm_ml[wi][q % NQ][0], sm_ml[wi][q % NQ][1], sm_o[(wi * NQ + q % NQ) * HD + d]);
        }
        const int64_t at = (hk * R + r0 + q) * splits + split;
        part_o[at * HD + d] = j.A;
        if (d == 0) { part_ml[2 * at] = j.M; part_ml[2 * at + 1] = j.L; }
    }
}

// ---- host -------------------------------------------------------------------------------------------------------------
int check_cache(const sgqd_cache_int8* c) {
    if (!c) return bad(SGQ_ERR_NULL_POINTER, "cache is NULL");
    if (c->batch < 0 || c->batch > 0x7fffffff || c->n_kv_heads <= 0 || c->n_kv_heads > 65535 || c->max_seq <= 0 || c->max_seq > 0x7fffffff ||
        c->head_dim <= 0 || c->batch * c->n_kv_heads > 0x7fffffff)
        return bad(SGQ_ERR_BAD_SHAPE, "bad cache shape");
    if (c->head_dim % 8 || c->head_dim > kMaxHeadDim) return bad(SGQ_ERR_BAD_SHAPE, "head_dim must be a multiple of 8, at most 256");
    return SGQ_OK;
}
int check_cache_pointers(const sgqd_cache_int8* c) {
    if (!c->k_codes || !c->k_scales || !c->v_codes || !c->v_scales) return bad(SGQ_ERR_NULL_POINTER, "a cache pointer is NULL");
    if (!aligned(c->k_codes, 16) || !aligned(c->v_codes, 16) || !aligned(c->k_scales, 4) || !aligned(c->v_scales, 4))
        return bad(SGQ_ERR_ALIGNMENT, "codes must be 16-byte aligned");
    return SGQ_OK;
}
CacheView view(const sgqd_cache_int8* c) { return CacheView{c->k_codes, c->k_scales, c->v_codes, c->v_scales, c->max_seq}; }

// Splits of a shared prefix and rows per block of its kernel: a function of the sizes alone, so that the workspace's size is one
// too.  148 SMs, one block each.
constexpr int kPrefixBlocks = 148;
struct PrefixPlan {
    int qw, blocks, splits;
    int64_t rows;                        // (kv head, query row) pairs
    size_t off_o, bytes;
};
PrefixPlan prefix_plan(int64_t batch, int64_t n_heads, int64_t n_kv, int64_t head_dim, int64_t prefix_max) {
    PrefixPlan p = {};
    const int64_t R = batch * (n_heads / n_kv);
    p.qw = R <= 8 ? 1 : (R <= 16 ? 2 : (R <= 32 ? 4 : 8));
    p.blocks = static_cast<int>(ceil_div(R, 8 * p.qw));
    const int64_t most = ceil_div(prefix_max, kTile * (kWarps / p.qw));              // a tile for every warp
    int64_t s = kPrefixBlocks / (n_kv * p.blocks);
    s = s < 1 ? 1 : (s > most ? most : s);
    p.splits = static_cast<int>(s > 65535 ? 65535 : s);
    p.rows = n_kv * R;
    p.off_o = (static_cast<size_t>(p.rows) * p.splits * 8 + 255) / 256 * 256;
    p.bytes = p.off_o + static_cast<size_t>(p.rows) * p.splits * head_dim * 4;
    return p;
}

template <int HD, int NQ>
int launch_decode(const DecodeArgs& a, int64_t batch, cudaStream_t s) {
    const int G = a.n_heads / a.n_kv, blocks = (G + NQ - 1) / NQ;
    const int64_t units = batch * a.n_kv * blocks;
    // splits of the positions: a block per SM slot, at least a tile for each of its warps, at most the portable cluster size
    int64_t S = 2 * static_cast<int64_t>(sm_count()) / units;
    const int64_t most = ceil_div(a.own.max_seq, kTile * kWarps);
    S = S > most ? most : S;
    S = S > 8 ? 8 : (S < 1 ? 1 : S);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(batch * a.n_kv), static_cast<unsigned>(blocks), static_cast<unsigned>(S));
    cfg.blockDim = dim3(kWarps * 32);
    cfg.stream = s;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 1;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = static_cast<unsigned>(S);
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    SGQ_CUDA_TRY(cudaLaunchKernelEx(&cfg, attn_decode_int8_kernel<HD, NQ>, a));
    return SGQ_OK;
}

int attn_decode(const float* qkv, int64_t qkv_stride, int64_t n_heads, const float* cos_table, const float* sin_table, int64_t table_rows,
                const int32_t* pos, int64_t pos_stride, const sgqd_cache_int8* cache, const sgqd_cache_int8* prefix, const int32_t* prefix_len,
                float* out, int64_t out_stride, void* prepared_out, size_t prepared_bytes, void* workspace, size_t workspace_bytes, cudaStream_t s) {
    int rc = check_cache(cache);
    if (rc != SGQ_OK) return rc;
    const int64_t hd = cache->head_dim, kv = cache->n_kv_heads, batch = cache->batch;
    if (hd != 64 && hd != 128) return bad(SGQ_ERR_UNSUPPORTED, "head_dim must be 64 or 128");
    if (n_heads <= 0 || n_heads > 65535 || n_heads % kv) return bad(SGQ_ERR_BAD_SHAPE, "n_heads must be a multiple of the cache's heads");
    if (qkv_stride < (n_heads + 2 * kv) * hd || out_stride < n_heads * hd) return bad(SGQ_ERR_BAD_SHAPE, "row stride too small");
    if (pos_stride != 0 && pos_stride != 1) return bad(SGQ_ERR_BAD_ARGUMENT, "pos_stride must be 0 or 1");
    if (prefix) {
        if ((rc = check_cache(prefix)) != SGQ_OK) return rc;
        if (prefix->batch != 1 || prefix->n_kv_heads != kv || prefix->head_dim != hd)
            return bad(SGQ_ERR_BAD_SHAPE, "the prefix is one sequence with the cache's heads");
    }
    if (cache->max_seq > kMaxPositions || (prefix && prefix->max_seq > kMaxPositions)) return bad(SGQ_ERR_BAD_SHAPE, "more than 2^30 positions");
    if (table_rows < cache->max_seq + (prefix ? prefix->max_seq : 0)) return bad(SGQ_ERR_BAD_SHAPE, "the cos / sin tables are too short");
    if (batch == 0) return SGQ_OK;
    if (!qkv || !cos_table || !sin_table || !pos || !out || (prefix && !prefix_len)) return bad(SGQ_ERR_NULL_POINTER, "NULL argument");
    if ((rc = check_cache_pointers(cache)) != SGQ_OK || (prefix && (rc = check_cache_pointers(prefix)) != SGQ_OK)) return rc;
    if (!aligned(qkv, 16) || (qkv_stride & 3) || !aligned(cos_table, 16) || !aligned(sin_table, 16))
        return bad(SGQ_ERR_ALIGNMENT, "qkv rows and tables must be 16-byte aligned");
    PreparedLayout L = {};
    if ((rc = check_prepared(prepared_out, prepared_bytes, batch, n_heads * hd, &L)) != SGQ_OK) return rc;
    PrefixPlan plan = {};
    if (prefix) {
        plan = prefix_plan(batch, n_heads, kv, hd, prefix->max_seq);
        if (plan.blocks > 65535) return bad(SGQ_ERR_BAD_SHAPE, "too many query rows for one call");
        if (!workspace || workspace_bytes < plan.bytes || !aligned(workspace, 256)) return bad(SGQ_ERR_WORKSPACE, "workspace too small or not 256-byte aligned");
    }
    if ((rc = check_device()) != SGQ_OK) return rc;
    DecodeArgs a = {};
    a.qkv = qkv; a.qkv_stride = qkv_stride; a.n_heads = static_cast<int>(n_heads); a.n_kv = static_cast<int>(kv); a.batch = static_cast<int>(batch);
    a.cos_t = cos_table; a.sin_t = sin_table; a.pos = pos; a.pos_stride = pos_stride; a.own = view(cache);
    a.out = out; a.out_stride = out_stride; a.pmode = L.mode; a.nmain = L.nmain; a.nlow = L.nlow; a.planes = static_cast<uint8_t*>(prepared_out);
    if (prefix) {
        a.first = view(prefix);
        a.prefix_len = prefix_len;
        float* ml = static_cast<float*>(workspace);
        float* o = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + plan.off_o);
        const dim3 grid(static_cast<unsigned>(kv), static_cast<unsigned>(plan.splits), static_cast<unsigned>(plan.blocks));
        if (hd == 128) SGQ_CUDA_TRY(launch_kernel(attn_prefix_int8_kernel<128>, grid, dim3(kWarps * 32), 0, s, true, a, plan.qw, ml, o));
        else SGQ_CUDA_TRY(launch_kernel(attn_prefix_int8_kernel<64>, grid, dim3(kWarps * 32), 0, s, true, a, plan.qw, ml, o));
        a.part_ml = ml;
        a.part_o = o;
        a.parts = plan.splits;
    }
    // four queries per warp where the group has no more: 2 column sets in the place of 3 and half the outputs in registers
    const bool four = n_heads / kv <= 4;
    if (hd == 128) return four ? launch_decode<128, 4>(a, batch, s) : launch_decode<128, 8>(a, batch, s);
    return four ? launch_decode<64, 4>(a, batch, s) : launch_decode<64, 8>(a, batch, s);
}

}  // namespace
}  // namespace sgq

using namespace sgq;

extern "C" {

int sgqd_rope_kv_store_int8(const float* qkv, int64_t qkv_stride, int64_t t_new, int64_t n_heads, const float* cos_table,
                            const float* sin_table, int64_t table_rows, const int32_t* pos, int64_t pos_stride, const int32_t* n_new,
                            const int32_t* rope_offset, float* q_out, int64_t q_stride, const sgqd_cache_int8* cache, void* stream) {
    int rc = check_cache(cache);
    if (rc != SGQ_OK) return rc;
    const int64_t hd = cache->head_dim, kv = cache->n_kv_heads;
    if (n_heads <= 0 || n_heads > 65535 || n_heads % kv) return bad(SGQ_ERR_BAD_SHAPE, "n_heads must be a multiple of the cache's heads");
    if (t_new < 0 || t_new > 0x7fffffff || cache->batch * t_new > 0x7fffffff) return bad(SGQ_ERR_BAD_SHAPE, "bad token count");
    if (qkv_stride < (n_heads + 2 * kv) * hd || q_stride < n_heads * hd) return bad(SGQ_ERR_BAD_SHAPE, "row stride too small");
    if (pos_stride != 0 && pos_stride != 1) return bad(SGQ_ERR_BAD_ARGUMENT, "pos_stride must be 0 or 1");
    if (q_out == qkv && q_stride != qkv_stride && qkv) return bad(SGQ_ERR_BAD_ARGUMENT, "in place, q_stride must be qkv_stride");
    if (table_rows < cache->max_seq) return bad(SGQ_ERR_BAD_SHAPE, "the cos / sin tables are too short");
    if (cache->batch * t_new == 0) return SGQ_OK;
    if (!qkv || !cos_table || !sin_table || !pos || !q_out) return bad(SGQ_ERR_NULL_POINTER, "NULL argument");
    if ((rc = check_cache_pointers(cache)) != SGQ_OK) return rc;
    if (!aligned(qkv, 16) || (qkv_stride & 3) || !aligned(q_out, 16) || (q_stride & 3) || !aligned(cos_table, 16) || !aligned(sin_table, 16))
        return bad(SGQ_ERR_ALIGNMENT, "rows and tables must be 16-byte aligned");
    if ((rc = check_device()) != SGQ_OK) return rc;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const int64_t rows = n_heads + 2 * kv;
#define SGQ_STORE(LPR)                                                                                                                    \
    SGQ_CUDA_TRY(launch_kernel(rope_kv_store_int8_kernel<LPR>,                                                                            \
                               dim3(static_cast<unsigned>(cache->batch * t_new), static_cast<unsigned>(ceil_div(rows, kStoreThreads / LPR))), \
                               dim3(kStoreThreads), 0, s, true, qkv, qkv_stride, static_cast<int>(t_new), static_cast<int>(n_heads),       \
                               static_cast<int>(kv), static_cast<int>(hd), cos_table, sin_table, table_rows, pos, pos_stride, n_new, rope_offset,       \
                               q_out, q_stride, cache->k_codes, cache->k_scales, cache->v_codes, cache->v_scales, cache->max_seq))
    if (hd <= 32) SGQ_STORE(4);
    else if (hd <= 64) SGQ_STORE(8);
    else if (hd <= 128) SGQ_STORE(16);
    else SGQ_STORE(32);
#undef SGQ_STORE
    return SGQ_OK;
}

int sgqd_kv_load_int8(const sgqd_cache_int8* cache, int64_t rows, int64_t batch, float* k_out, float* v_out, int64_t out_max_seq,
                      int64_t out_row0, void* stream) {
    int rc = check_cache(cache);
    if (rc != SGQ_OK) return rc;
    if (rows < 0 || rows > cache->max_seq) return bad(SGQ_ERR_BAD_SHAPE, "rows must lie inside the cache");
    if (batch < 0 || batch > 0x7fffffff || (cache->batch != batch && cache->batch != 1))
        return bad(SGQ_ERR_BAD_SHAPE, "batch must be the cache's, or the cache one sequence");
    if (out_row0 < 0 || out_max_seq > 0x7fffffff || out_row0 > out_max_seq - rows) return bad(SGQ_ERR_BAD_SHAPE, "the rows do not fit behind out_row0");
    if (batch * rows == 0) return SGQ_OK;
    if (!k_out || !v_out) return bad(SGQ_ERR_NULL_POINTER, "an output is NULL");
    if ((rc = check_cache_pointers(cache)) != SGQ_OK) return rc;
    if (!aligned(k_out, 16) || !aligned(v_out, 16)) return bad(SGQ_ERR_ALIGNMENT, "outputs must be 16-byte aligned");
    const int64_t vecs = rows * cache->head_dim / 4, chunks = ceil_div(vecs, kLoadThreads * kLoadPerThread);
    const int64_t heads = batch * cache->n_kv_heads;
    if (heads > 0x7fffffff / chunks) return bad(SGQ_ERR_BAD_SHAPE, "too many rows for one call");
    if ((rc = check_device()) != SGQ_OK) return rc;
    SGQ_CUDA_TRY(launch_kernel(kv_load_int8_kernel, dim3(static_cast<unsigned>(heads * chunks), 2), dim3(kLoadThreads), 0,
                               static_cast<cudaStream_t>(stream), true, cache->k_codes, cache->k_scales, cache->v_codes, cache->v_scales,
                               cache->max_seq, static_cast<int>(cache->head_dim), vecs, chunks, cache->batch * cache->n_kv_heads, k_out, v_out,
                               out_max_seq, out_row0));
    return SGQ_OK;
}

int sgqd_attn_decode_int8(const float* qkv, int64_t qkv_stride, int64_t n_heads, const float* cos_table, const float* sin_table,
                          int64_t table_rows, const int32_t* pos, int64_t pos_stride, const sgqd_cache_int8* cache, float* out, int64_t out_stride,
                          void* prepared_out, size_t prepared_bytes, void* stream) {
    return attn_decode(qkv, qkv_stride, n_heads, cos_table, sin_table, table_rows, pos, pos_stride, cache, nullptr, nullptr, out, out_stride, prepared_out,
                       prepared_bytes, nullptr, 0, static_cast<cudaStream_t>(stream));
}

size_t sgqd_attn_decode_prefix_int8_workspace_bytes(int64_t batch, int64_t n_heads, int64_t n_kv_heads, int64_t head_dim, int64_t prefix_max) {
    if (batch <= 0 || batch > 0x7fffffff || n_heads <= 0 || n_heads > 65535 || n_kv_heads <= 0 || n_heads % n_kv_heads || prefix_max <= 0 ||
        prefix_max > kMaxPositions || (head_dim != 64 && head_dim != 128))
        return 0;
    return prefix_plan(batch, n_heads, n_kv_heads, head_dim, prefix_max).bytes;
}

int sgqd_attn_decode_prefix_int8(const float* qkv, int64_t qkv_stride, int64_t n_heads, const float* cos_table, const float* sin_table,
                                 int64_t table_rows, const int32_t* pos, int64_t pos_stride, const sgqd_cache_int8* cache, const sgqd_cache_int8* prefix,
                                 const int32_t* prefix_len, float* out, int64_t out_stride, void* prepared_out, size_t prepared_bytes,
                                 void* workspace, size_t workspace_bytes, void* stream) {
    if (!prefix) return bad(SGQ_ERR_NULL_POINTER, "prefix is NULL");
    return attn_decode(qkv, qkv_stride, n_heads, cos_table, sin_table, table_rows, pos, pos_stride, cache, prefix, prefix_len, out, out_stride, prepared_out,
                       prepared_bytes, workspace, workspace_bytes, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
