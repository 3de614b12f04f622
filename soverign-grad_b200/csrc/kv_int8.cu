// The INT8 key/value cache (include/sgq_decoder.h): rows of head_dim codes with one fp32 scale per (sequence, head,
// position), written with the rotary embedding, read back as fp32, and read by the decode attention.
//
// A row is quantized by the library's per-row INT8 quantizer, bit for bit: a = max(1e-8, max |r|), scale = a / 127,
// code = clamp(round_half_away(r * (127 / a))), every operation rounded to fp32 (NaN -> +127, an infinity makes the scale
// infinite).  The rotation in front of it rounds every product and sum to fp32 (no contraction), so codes and scales are a
// function of the inputs alone: the prompt's store, the decode step's append and a host restatement agree in every bit.
#include "kv_int8.cuh"

#include <algorithm>
#include <cooperative_groups.h>
#include <math.h>
#include <math_constants.h>
#include <stdint.h>

namespace sgq {

namespace {

constexpr int kMaxHeadDim = 256;
constexpr int64_t kMaxPositions = 1ll << 30;       // of the attention: positions and strides between tiles in 32 bits

// ---- store ------------------------------------------------------------------------------------------------------------
// One group of LPR lanes per row (a head of q, k or v of one token); a lane owns VEC values of the first half of the row and the
// same VEC of the second half, so that a rotary pair sits in one lane and only the absmax crosses lanes.  grid (tokens, row blocks).
// What bounds it is memory: 8 x 512 tokens of 16 + 2 x 16 heads of 128 move 154 MB in 26.7 us, 88% of the rate of a plain copy.
// VEC 8, where rows and tables allow 32-byte accesses, against 4: 26.3 / 28.9 us.  The row is read behind the token's check, not
// next to it: 26.9 / 26.5 us where every token exists, 5.4 / 7.3 where 3 x 777 are padded to about half.
constexpr int kStoreThreads = 256;                   // at most; the rows of a token are dealt out evenly to its blocks
template <int LPR, int VEC>
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
    const int b = static_cast<int>(blockIdx.x / static_cast<unsigned>(t_new)), i = static_cast<int>(m - static_cast<int64_t>(b) * t_new);
    const int r = blockIdx.y * (blockDim.x / LPR) + threadIdx.x / LPR;          // row of the token: q heads, k heads, v heads
    const int l = threadIdx.x % LPR;
    const int half = head_dim >> 1;
    const bool in = r < n_heads + 2 * n_kv && VEC * l < half;
    const float* row = qkv + m * qkv_stride + static_cast<int64_t>(r) * head_dim + VEC * l;
    const int64_t pos = static_cast<int64_t>(pos_p[b * pos_stride]) + i;
    const int64_t turn = pos + (rope_offset ? *rope_offset : 0);
    // a token behind the sequence's own count, outside the cache or outside the tables leaves everything as it was
    if (pos < 0 || pos >= max_seq || turn < 0 || turn >= table_rows || (n_new && i >= n_new[b])) return;         // uniform over the block
    float x[VEC] = {}, y[VEC] = {};
    if (in) {
        load_floats<VEC>(x, row);
        load_floats<VEC>(y, row + half);
    }
    if (in && r < n_heads + n_kv) {
        float co[VEC], si[VEC];
        load_floats<VEC>(co, cos_t + turn * half + VEC * l);
        load_floats<VEC>(si, sin_t + turn * half + VEC * l);
#pragma unroll
        for (int j = 0; j < VEC; ++j) rotate_pair(x[j], y[j], co[j], si[j]);
    }
    float top = 1e-8f;
#pragma unroll
    for (int j = 0; j < VEC; ++j) top = absmax_step(absmax_step(top, x[j]), y[j]);
#pragma unroll
    for (int o = LPR / 2; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    if (!in) return;
    if (r < n_heads) {
        float* o = q_out + m * q_stride + static_cast<int64_t>(r) * head_dim + VEC * l;
        store_floats<VEC>(o, x);
        store_floats<VEC>(o + half, y);
        return;
    }
    const bool is_v = r >= n_heads + n_kv;
    const int h = r - n_heads - (is_v ? n_kv : 0);
    const int64_t at = (static_cast<int64_t>(b) * n_kv + h) * max_seq + pos;
    const float inv = __fdiv_rn(127.0f, top);
    auto put = [&](int8_t* to, const float (&v)[VEC]) {
        union { char4 c[VEC / 4]; uint2 w; } q;
#pragma unroll
        for (int j = 0; j < VEC / 4; ++j)
            q.c[j] = make_char4(quantize_code<127, -127>(v[4 * j], inv), quantize_code<127, -127>(v[4 * j + 1], inv),
                                quantize_code<127, -127>(v[4 * j + 2], inv), quantize_code<127, -127>(v[4 * j + 3], inv));
        if constexpr (VEC == 8) *reinterpret_cast<uint2*>(to) = q.w;
        else *reinterpret_cast<char4*>(to) = q.c[0];
    };
    int8_t* codes = (is_v ? vc : kc) + at * head_dim + VEC * l;
    put(codes, x);
    put(codes + half, y);
    if (l == 0) (is_v ? vs : ks)[at] = __fdiv_rn(top, 127.0f);
}

// ---- read back --------------------------------------------------------------------------------------------------------
// A lane turns 8 codes of a row into 8 floats, kLoadRows times.  grid (heads * row blocks, keys | values).  WIDE: the outputs are
// 32-byte aligned, and a lane's floats leave as one 32-byte store (8 x 16 x 512 rows of 128, 84 MB: 14.7 us, 88% of the rate of a
// plain copy; four codes and a 16-byte store per lane: 19.7; 1 / 2 / 4 rows of a shared prefix per lane: 4.75 / 4.3 / 5.1).
constexpr int kLoadThreads = 256, kLoadRows = 2;
template <bool WIDE>
__global__ void __launch_bounds__(kLoadThreads) kv_load_int8_kernel(const int8_t* __restrict__ kc, const float* __restrict__ ks,
                                                                    const int8_t* __restrict__ vc, const float* __restrict__ vs, int64_t max_seq,
                                                                    int head_dim, int rows, int chunks, int step, int64_t src_heads,
                                                                    float* __restrict__ k_out, float* __restrict__ v_out, int64_t out_max_seq,
                                                                    int64_t out_row0) {
    pdl_launch_dependents();
    pdl_wait();
    const int per_row = head_dim >> 3;
    const int64_t bh = blockIdx.x / static_cast<unsigned>(chunks);
    const int chunk = static_cast<int>(blockIdx.x - bh * chunks);
    const int row = threadIdx.x / per_row, col = (threadIdx.x - row * per_row) * 8;
    if (row >= step) return;                                      // step: rows that the block's threads cover at once
    const int64_t src = (bh % src_heads) * max_seq;               // src_heads: heads of all source sequences, or of the one shared
    const bool is_v = blockIdx.y != 0;
    const int8_t* codes = (is_v ? vc : kc) + src * head_dim + col;
    const float* scales = (is_v ? vs : ks) + src;
    float* out = (is_v ? v_out : k_out) + (bh * out_max_seq + out_row0) * head_dim + col;
    const int64_t first = static_cast<int64_t>(chunk) * (kLoadRows * step) + row;
    uint2 c[kLoadRows];
    float s[kLoadRows];
#pragma unroll
    for (int u = 0; u < kLoadRows; ++u) {
        const int64_t r = first + u * step;
        if (r < rows) {
            c[u] = *reinterpret_cast<const uint2*>(codes + r * head_dim);
            s[u] = scales[r];
        }
    }
#pragma unroll
    for (int u = 0; u < kLoadRows; ++u) {
        const int64_t r = first + u * step;
        if (r >= rows) break;
        const char4 a = *reinterpret_cast<const char4*>(&c[u].x), d = *reinterpret_cast<const char4*>(&c[u].y);
        const float lo[4] = {a.x * s[u], a.y * s[u], a.z * s[u], a.w * s[u]}, hi[4] = {d.x * s[u], d.y * s[u], d.z * s[u], d.w * s[u]};
        float* o = out + r * head_dim;
        if constexpr (WIDE) {
            store_floats<8>(o, {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]});
        } else {
            store_floats<4>(o, lo);
            store_floats<4>(o + 4, hi);
        }
    }
}

// ---- decode attention -------------------------------------------------------------------------------------------------
// Both products of the attention run on the tensor cores as exact integer products (mma.sync m16n8k32, s8 x s8 -> s32): the
// codes go in as they lie in memory, the query and the softmax weights as 24-bit fixed point split into three balanced
// base-256 digits (the arithmetic of gemv_prepare.cuh), one digit per column of the small operand.  A query has one scale, that of its
// largest value: a value far below it keeps as many bits less.  (Scales per 32 values, as the linears have, would end the integer
// sums, and the conversions behind them, four times as often; a fourth digit would take eight queries a fourth column set and the
// tcgen05 kernel more columns than tensor memory has.)
//
//   scores   A = 16 rows of the cache x 32 values, B = 32 values x 8 columns.  A lane (g, t) = (lane / 4, lane % 4) of the
//            warp reads the 16-byte chunks t (and 4 + t) of the rows 4g .. 4g+3 of a tile of 32 positions: these ARE the A
//            fragments, the order of the head dimension inside them being the same in the query's digits.  Columns 2t, 2t+1
//            of a "main" column set hold digits 2 and 1 of query t, those of the "low" set digit 0 of queries t and
//            t + 4, so a lane finds all digits of its one or two queries in its own accumulators.
//   weights  w = p * value scale, relative to the largest |w| of the tile and query: their digits cross the warp by shuffles
//            (rows of the accumulators become the contraction index).
//   output   A = 16 values x 32 positions: a lane reads HD/8 consecutive values of 8 positions and transposes 4 x 4 bytes
//            with byte permutes.  B = 32 positions x 8 columns of weight digits.
//
// Scores and outputs leave the integer domain once per tile or step (sums of at most 128 products, below 2^21.1), scaled
// and added in fp32 with the running reference and sum of the softmax.  A lane holds the scores of positions 4g .. 4g+3 and
// the values [HD/8 g, HD/8 (g+1)) of the outputs of queries t and t + 4.
// D = A(16x32, s8) * B(32x8, s8), and D += A * B
__device__ __forceinline__ void mma_first(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "r"(0));
}
__device__ __forceinline__ void mma_next(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
constexpr int kTile = 32;              // positions per step of a warp

// ---- half tiles in shared memory: the 32 rows of keys or of values and their scales, fetched by cp.async -------------------
// Rows lie in 128-byte lines of eight 16-byte chunks whose place is permuted by the row, so that the fragment reads (for keys
// the chunks t of rows 4g + i, for values the chunk g of rows 4t + i) touch all banks.
template <int HD>
struct Half {
    static constexpr int kScales = kTile * HD, kBytes = kScales + kTile * 4;
    static __device__ __forceinline__ int place(int row, int chunk, int turn) {
        if constexpr (HD == 128) return row * 128 + ((chunk ^ turn) << 4);
        else return (row >> 1) * 128 + ((((row & 1) * 4 + chunk) ^ turn) << 4);
    }
    static __device__ __forceinline__ int key_at(int row, int chunk) { return place(row, chunk, ((row >> 2) & 1) * 4); }
    static __device__ __forceinline__ int value_at(int row, int chunk) { return place(row, chunk, ((row >> 2) & 3) * 2); }
    template <bool KEYS>
    static __device__ __forceinline__ int at(int row, int chunk) { return KEYS ? key_at(row, chunk) : value_at(row, chunk); }
};
__device__ __forceinline__ void cp_async_4(uint32_t dst, const void* src) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}

// `THREADS` threads (this one is number i) ask for the rows codes[t ..] and their scales; rows from t1 on repeat the last one
// (their positions are masked).
template <int HD, int THREADS, bool KEYS>
__device__ __forceinline__ void request_half(uint32_t dst, const int8_t* codes, const float* scales, int t, int t1, int i) {
    constexpr int CH = HD / 16, USED = THREADS < kTile * CH ? THREADS : kTile * CH, STEP = USED / CH;
    const int last = t1 - 1 - t, row0 = i / CH, c = i % CH;
    if (USED == THREADS || i < USED) {
        const int8_t* from = codes + static_cast<int64_t>(t) * HD + c * 16;
        // where the row's chunk goes differs from row to row by a multiple of the line and by which bits of the place are flipped
        uint32_t to[kTile / STEP];
#pragma unroll
        for (int x = 0; x < kTile / STEP; ++x) to[x] = dst + Half<HD>::template at<KEYS>(row0 + x * STEP, c);
        if (last >= kTile - 1) {
            from += row0 * HD;
#pragma unroll
            for (int x = 0; x < kTile / STEP; ++x) cp_async_16(to[x], from + x * STEP * HD);
        } else {
#pragma unroll
            for (int x = 0; x < kTile / STEP; ++x) cp_async_16(to[x], from + min(row0 + x * STEP, last) * HD);
        }
    }
    if (THREADS == 32 || i < 32) cp_async_4(dst + Half<HD>::kScales + 4 * (i & 31), scales + t + min(i & 31, last));
}
// A group: ST half tiles `step` positions apart, the first one at position t
template <int HD, int THREADS, int ST, bool KEYS>
__device__ __forceinline__ void request_group(uint32_t dst, const int8_t* codes, const float* scales, int t, int step, int t1, int i) {
#pragma unroll
    for (int j = 0; j < ST; ++j)
        if (t + j * step < t1) request_half<HD, THREADS, KEYS>(dst + j * Half<HD>::kBytes, codes, scales, t + j * step, t1, i);
}
// A warp's ring holds three groups: keys, values, keys of the next step, values of the next step, ... in turn.  While one of them
// is in use the two behind it are on their way.
constexpr int kGroups = 3;
__device__ __forceinline__ int next_slot(int s) { return s + 1 == kGroups ? 0 : s + 1; }

// One warp's running attention of up to NQ (4 or 8) queries over tiles of one kv head's rows, ST tiles per step.
template <int HD, int NQ, int ST>
struct WarpAttention {
    static constexpr int KW = HD / 16;         // 32-bit words of a key row per lane
    static constexpr int VB = HD / 8;          // values per lane and position
    static constexpr int VW = VB / 4;
    static constexpr int NS = NQ / 4, NT = NS + 1;
    static constexpr int kQueryBytes = 3 * HD; // digit planes of one query: [digit][HD]

    const uint8_t* planes;                     // the queries' digits, in shared memory
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
    // the digit planes and units of NQ queries, written by query_planes below
    __device__ __forceinline__ void use_queries(const uint8_t* digits, const float* units) {
        planes = digits;
#pragma unroll
        for (int s = 0; s < NS; ++s) qu[s] = units[4 * s + t];
    }
    // B fragments of the digits: 16 to 24 registers that are read again for every step rather than kept through the products
    // behind it (kept, the kernels do not fit three CTAs per SM)
    __device__ __forceinline__ void load_queries(uint32_t (&bq)[NT][KW]) const {
        auto rd = [&](uint32_t (&w)[KW], int query, int digit, bool zero) {
            const uint8_t* p = planes + query * kQueryBytes + digit * HD + 16 * t;
#pragma unroll
            for (int c = 0; c < KW / 4; ++c) {
                const uint4 x = *reinterpret_cast<const uint4*>(p + 64 * c);
                w[4 * c] = zero ? 0u : x.x; w[4 * c + 1] = zero ? 0u : x.y; w[4 * c + 2] = zero ? 0u : x.z; w[4 * c + 3] = zero ? 0u : x.w;
            }
        };
#pragma unroll
        for (int s = 0; s < NS; ++s) rd(bq[s], 4 * s + (g >> 1), 2 - (g & 1), false);
        if (NS == 2) rd(bq[NS], (g >> 1) + 4 * (g & 1), 0, false);
        else rd(bq[NS], g >> 1, 0, (g & 1) != 0);
    }
    // scores of a tile's keys: sc[s][i] of position 4g + i and query t + 4s, in base-2 units; positions from `n` on are masked
    __device__ __forceinline__ void scores(float (&sc)[NS][4], const uint32_t (&bq)[NT][KW], const uint8_t* tile, int n) {
        uint32_t k[4][KW];
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int c = 0; c < KW / 4; ++c) {
                const uint4 x = *reinterpret_cast<const uint4*>(tile + Half<HD>::key_at(4 * g + i, t + 4 * c));
                k[i][4 * c] = x.x; k[i][4 * c + 1] = x.y; k[i][4 * c + 2] = x.z; k[i][4 * c + 3] = x.w;
            }
        const float4 ks4 = *reinterpret_cast<const float4*>(tile + Half<HD>::kScales + 16 * g);
        const float ks[4] = {ks4.x, ks4.y, ks4.z, ks4.w};
        int acc[2][NT][4];
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int n2 = 0; n2 < NT; ++n2) {
                mma_first(acc[h][n2], k[2 * h][0], k[2 * h + 1][0], k[2 * h][1], k[2 * h + 1][1], bq[n2][0], bq[n2][1]);
#pragma unroll
                for (int c = 1; c < KW / 2; ++c)
                    mma_next(acc[h][n2], k[2 * h][2 * c], k[2 * h + 1][2 * c], k[2 * h][2 * c + 1], k[2 * h + 1][2 * c + 1], bq[n2][2 * c], bq[n2][2 * c + 1]);
            }
#pragma unroll
        for (int s = 0; s < NS; ++s)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int h = i >> 1, r = 2 * (i & 1);
                const float x = join_digits(acc[h][s][r], acc[h][s][r + 1], acc[h][NS][r + s]) * (ks[i] * kKeyDown);
                sc[s][i] = fmaf(x, qu[s], ks[i] - ks[i]);               // NaN for a row whose scale is not finite
            }
        if (n < kTile) {
#pragma unroll
            for (int s = 0; s < NS; ++s)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (4 * g + i >= n) sc[s][i] = -CUDART_INF_F;
        }
    }
    __device__ __forceinline__ void scores_of(float (&sc)[ST][NS][4], const uint8_t* keys, const int (&n)[ST]) {
        uint32_t bq[NT][KW];
        load_queries(bq);
#pragma unroll
        for (int j = 0; j < ST; ++j) scores(sc[j], bq, keys + j * Half<HD>::kBytes, n[j]);
    }
    // A group of values, of which tile j has n[j] positions, with the scores: into the running sums and the outputs.  The
    // weights are taken against a reference that follows the maximum only when a score exceeds it by kAhead (weights up to
    // 2^kAhead): most steps then neither wait for a maximum to cross the warp nor rescale anything.
    __device__ __forceinline__ void accumulate(float (&sc)[ST][NS][4], const uint8_t* values, const int (&n)[ST]) {
        uint32_t bw[ST][NT][2];
        float unit[NS];
        uint32_t w0[ST][NS], w1[ST][NS], w2[ST][NS];
        float top[NS];
        bool ahead = false;
#pragma unroll
        for (int s = 0; s < NS; ++s) {
            top[s] = -CUDART_INF_F;
#pragma unroll
            for (int j = 0; j < ST; ++j) top[s] = fmaxf(top[s], fmaxf(fmaxf(sc[j][s][0], sc[j][s][1]), fmaxf(sc[j][s][2], sc[j][s][3])));
            ahead |= top[s] > m[s] + kAhead;
        }
        if (__any_sync(0xffffffffu, ahead)) {
#pragma unroll
            for (int s = 0; s < NS; ++s) {
#pragma unroll
                for (int d = 4; d < 32; d <<= 1) top[s] = fmaxf(top[s], __shfl_xor_sync(0xffffffffu, top[s], d));
                const float mn = fmaxf(m[s], top[s]), corr = m[s] == mn ? 1.0f : exp2_approx(m[s] - mn);
                m[s] = mn;
                l[s] *= corr;
#pragma unroll
                for (int j = 0; j < VB; ++j) o[s][j] *= corr;
            }
        }
#pragma unroll
        for (int s = 0; s < NS; ++s) {
            float most = 0.f;
            const float ref = m[s] == -CUDART_INF_F ? 0.f : m[s];        // nothing but masked positions so far: weights of zero
#pragma unroll
            for (int j = 0; j < ST; ++j) {
                const float4 v4 = *reinterpret_cast<const float4*>(values + j * Half<HD>::kBytes + Half<HD>::kScales + 16 * g);
                float vs[4] = {v4.x, v4.y, v4.z, v4.w};
                if (n[j] < kTile) {
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (4 * g + i >= n[j]) vs[i] = 0.f;               // whatever a masked position's scale is
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float p = exp2_approx(sc[j][s][i] - ref);
                    l[s] += p;
                    sc[j][s][i] = p * vs[i];
                    most = max_nan(most, fabsf(sc[j][s][i]));
                }
            }
#pragma unroll
            for (int d = 4; d < 32; d <<= 1) most = max_nan(most, __shfl_xor_sync(0xffffffffu, most, d));
            // weights that vanish against the reference contribute nothing; NaN and infinity make the unit NaN
            const float down = most * kValueDown;                         // far below 2^126, where __fdividef ends
            const float per = most < kVanishing ? 0.f : __fdividef(kWeightRange * kValueDown, down);
            unit[s] = fmaf(down, 1.0f / kWeightRange, most - most);
#pragma unroll
            for (int j = 0; j < ST; ++j) {
                uint32_t d[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) d[i] = weight_digits(sc[j][s][i], per);
                gather_digits(d, w0[j][s], w1[j][s], w2[j][s]);
            }
        }
        // B fragments: lane (column g, position quad t or t + 4) takes the digit words that lane (quad, query) holds
#pragma unroll
        for (int j = 0; j < ST; ++j)
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const int from = 4 * (t + 4 * half) + (g >> 1);
#pragma unroll
                for (int s = 0; s < NS; ++s) {
                    const uint32_t hi = __shfl_sync(0xffffffffu, w2[j][s], from), mid = __shfl_sync(0xffffffffu, w1[j][s], from);
                    bw[j][s][half] = (g & 1) ? mid : hi;
                }
                const uint32_t lo = __shfl_sync(0xffffffffu, w0[j][0], from);
                const uint32_t lo2 = NS == 2 ? __shfl_sync(0xffffffffu, w0[j][NS - 1], from) : 0u;
                bw[j][NS][half] = (g & 1) ? lo2 : lo;
            }
        int acc[2 * VW][NT][4];                 // values 2 x (rows g) and 2 x + 1 (rows g + 8) of this lane
#pragma unroll
        for (int j = 0; j < ST; ++j) {
            uint32_t v[8][VW];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int row = 4 * t + (i & 3) + 16 * (i >> 2);
                if constexpr (VW == 4) {
                    const uint4 x = *reinterpret_cast<const uint4*>(values + j * Half<HD>::kBytes + Half<HD>::value_at(row, g));
                    v[i][0] = x.x; v[i][1] = x.y; v[i][2] = x.z; v[i][3] = x.w;
                } else {
                    const uint2 x = *reinterpret_cast<const uint2*>(values + j * Half<HD>::kBytes + Half<HD>::value_at(row, g >> 1) + 8 * (g & 1));
                    v[i][0] = x.x; v[i][1] = x.y;
                }
            }
#pragma unroll
            for (int wd = 0; wd < VW; ++wd) {
                uint32_t a[2][4];               // [quad half][value 4 wd + r]: four positions each
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
                for (int pr = 0; pr < 2; ++pr) {
                    const int x = 2 * wd + pr;
#pragma unroll
                    for (int n2 = 0; n2 < NT; ++n2) {
                        if (j == 0) mma_first(acc[x][n2], a[0][2 * pr], a[0][2 * pr + 1], a[1][2 * pr], a[1][2 * pr + 1], bw[j][n2][0], bw[j][n2][1]);
                        else mma_next(acc[x][n2], a[0][2 * pr], a[0][2 * pr + 1], a[1][2 * pr], a[1][2 * pr + 1], bw[j][n2][0], bw[j][n2][1]);
                    }
                    if (j < ST - 1) continue;
#pragma unroll
                    for (int s = 0; s < NS; ++s)
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            float& out = o[s][2 * x + e];
                            out = fmaf(join_digits(acc[x][s][2 * e], acc[x][s][2 * e + 1], acc[x][NS][2 * e + s]), unit[s], out);
                        }
                }
            }
        }
    }
    // (reference, sum, value) of the first nq queries into to_ml[NQ][2], to_o[NQ][HD]
    __device__ __forceinline__ void store(float* to_ml, float* to_o, int nq = NQ) {
#pragma unroll
        for (int s = 0; s < NS; ++s) {
#pragma unroll
            for (int d = 4; d < 32; d <<= 1) l[s] += __shfl_xor_sync(0xffffffffu, l[s], d);
            const int q = t + 4 * s;
            if (q >= nq) continue;
            if (g == 0) { to_ml[2 * q] = m[s]; to_ml[2 * q + 1] = l[s]; }
#pragma unroll
            for (int j = 0; j < VB; j += 4)
                *reinterpret_cast<float4*>(to_o + q * HD + VB * g + j) = make_float4(o[s][j], o[s][j + 1], o[s][j + 2], o[s][j + 3]);
        }
    }
};

// Digit planes [3][HD] of a query for WarpAttention::load_queries
template <int HD>
__device__ __forceinline__ void query_planes(const float (&v)[HD / 32], uint8_t* planes, float* unit, int lane) {
    query_digits<HD>(v, [&](int j, int d) { return planes + j * HD + d; }, unit, lane);
}

// One warp quantizes a row: its lane's codes (HD / 32 bytes) and the scale.
template <int HD>
struct HeldRow {
    uint32_t codes;
    float scale;
    __device__ __forceinline__ void make(const float (&v)[HD / 32]) {
        float top = 1e-8f;
#pragma unroll
        for (int j = 0; j < HD / 32; ++j) top = absmax_step(top, v[j]);
        top = warp_max(top);
        const float inv = __fdiv_rn(127.0f, top);
        codes = 0;
#pragma unroll
        for (int j = 0; j < HD / 32; ++j) codes |= (static_cast<uint32_t>(quantize_code<127, -127>(v[j], inv)) & 0xFFu) << (8 * j);
        scale = __fdiv_rn(top, 127.0f);
    }
    __device__ __forceinline__ void put(void* row) const {               // row: where the lane's codes go
        if constexpr (HD == 128) *static_cast<uint32_t*>(row) = codes;
        else *static_cast<uint16_t*>(row) = static_cast<uint16_t>(codes);
    }
};

// The rows a new token brings to a kv head: one warp makes them and keeps them in shared memory until it puts them into the
// half tiles whose copies of the rows are older.
template <int HD>
struct NewRows {
    static constexpr int kBytes = 2 * HD + 16;                             // codes of the key and of the value, their scales
    static constexpr int VEC = HD / 32;
    static __device__ __forceinline__ void load(const DecodeArgs& a, int b, int hk, float (&x)[VEC], float (&y)[VEC], int lane) {
        const float* from = a.qkv + b * a.qkv_stride + static_cast<int64_t>(a.n_heads + hk) * HD + lane * VEC;
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            x[j] = from[j];
            y[j] = from[static_cast<int64_t>(a.n_kv) * HD + j];
        }
    }
    static __device__ __forceinline__ void make(const DecodeArgs& a, float (&x)[VEC], float (&y)[VEC], const float* cos_row, const float* sin_row,
                                                uint8_t* keep, int64_t row, bool append, int lane) {
        rotate_row<HD>(x, cos_row, sin_row, lane);
        HeldRow<HD> k, v;
        k.make(x);
        v.make(y);
        k.put(keep + lane * VEC);
        v.put(keep + HD + lane * VEC);
        float* scales = reinterpret_cast<float*>(keep + 2 * HD);
        if (lane == 0) { scales[0] = k.scale; scales[1] = v.scale; }
        if (append) {
            k.put(a.own.kc + row * HD + lane * VEC);
            v.put(a.own.vc + row * HD + lane * VEC);
            if (lane == 0) { a.own.ks[row] = k.scale; a.own.vs[row] = v.scale; }
        }
        __syncwarp();
    }
    template <bool KEYS>
    static __device__ __forceinline__ void bring_in(const uint8_t* keep, uint8_t* half, int r, int lane) {
        if (lane < HD / 16)
            *reinterpret_cast<uint4*>(half + Half<HD>::template at<KEYS>(r, lane)) = *reinterpret_cast<const uint4*>(keep + (KEYS ? 0 : HD) + lane * 16);
        if (lane == 31) *reinterpret_cast<float*>(half + Half<HD>::kScales + 4 * r) = reinterpret_cast<const float*>(keep + 2 * HD)[KEYS ? 0 : 1];
        __syncwarp();
    }
};

// One warp: a finished head as prepared activations of the [batch, n_heads * HD] matrix (a head is HD / 32 whole groups)
template <int HD>
__device__ __forceinline__ void prepare_head(const DecodeArgs& a, const float* head, int b, int h, int lane) {
    const bool in = lane < HD / 8;
    float v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = in ? head[lane * 8 + j] : 0.f;
    const PreparedParts pp = prepared_parts(a.planes, static_cast<size_t>(a.n_heads) * (HD / 32), a.nmain, a.nlow);
    convert_groups<kOrderNibble>(v, b, a.batch, static_cast<size_t>(h) * (HD / 32), a.pmode, a.nmain, a.nlow, 0.0625f, pp, in);
}

// One warp's share of a head: the partial result of HD / 32 values per lane.
template <int HD>
struct JoinedHead {
    static constexpr int VEC = HD / 32;
    float M, L, A[VEC];
    __device__ __forceinline__ JoinedHead() : M(-HUGE_VALF), L(0.f) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) A[i] = 0.f;
    }
    // the partial results i < n of which `load` gives reference, sum and this lane's values; U of them are asked for together
    template <int U, typename Load>
    __device__ __forceinline__ void join(int n, Load load) {
        for (int p = 0; p < n; p += U) {
            float m[U], l[U], v[U][VEC];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                m[u] = -CUDART_INF_F;
                l[u] = 0.f;
#pragma unroll
                for (int i = 0; i < VEC; ++i) v[u][i] = 0.f;
                if (p + u < n) load(p + u, m[u], l[u], v[u]);
            }
            float mn = M;
#pragma unroll
            for (int u = 0; u < U; ++u) mn = fmaxf(mn, m[u]);
            const float x = M == mn ? 1.0f : exp2_approx(M - mn);
            L *= x;
#pragma unroll
            for (int i = 0; i < VEC; ++i) A[i] *= x;
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const float y = m[u] == mn ? 1.0f : exp2_approx(m[u] - mn);
                L = fmaf(l[u], y, L);
#pragma unroll
                for (int i = 0; i < VEC; ++i) A[i] = fmaf(v[u][i], y, A[i]);
            }
            M = mn;
        }
    }
    // joins the prefix's partial results, divides, stores query head h of sequence b (`head`: HD floats of shared memory)
    template <bool PREFIX>
    __device__ __forceinline__ void finish(const DecodeArgs& a, int b, int h, bool live, float* head, int lane) {
        if (PREFIX && live) {
            const int G = a.n_heads / a.n_kv, hk = h / G;
            const int64_t p0 = (static_cast<int64_t>(hk) * a.batch * G + static_cast<int64_t>(b) * G + h - hk * G) * a.parts;
            join<6>(a.parts, [&](int p, float& m, float& l, float (&v)[VEC]) {
                m = a.part_ml[2 * (p0 + p)];
                l = a.part_ml[2 * (p0 + p) + 1];
                load_values_of(a.part_o + (p0 + p) * HD + lane * VEC, v);
            });
        }
        float* to = a.out + b * a.out_stride + static_cast<int64_t>(h) * HD + lane * VEC;
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
            const float o = live ? A[i] / L * (1.0f / kValueDown) : 0.f;          // L == 0: every score is -infinity, and the output NaN
            to[i] = o;
            head[lane * VEC + i] = o;
        }
        if (a.planes != nullptr) {
            __syncwarp();
            prepare_head<HD>(a, head, b, h, lane);
            __syncwarp();
        }
    }
};

constexpr int kWarps = 8;
// Short caches.  grid (batch * kv heads, query blocks, S) in clusters of S along z: the W warps of the S CTAs of a cluster take
// the tiles of one (sequence, kv head) in turn, each through a ring of its own (nothing but warp barriers in the loop).
// The warp of the last tile brings in the new token's row.  Warps are joined through shared memory; every CTA then stores its
// partial result of head q into the shared memory of CTA q % S of the cluster, which finishes it.
constexpr int kDecodeWarps = 4, kMaxSplits = 8;
template <int HD, int NQ>
struct DecodeShape {
    static constexpr int ST = 128 / HD, kStep = ST * kTile, kGroup = ST * Half<HD>::kBytes;
    static constexpr int kRecv = NQ + kMaxSplits - 1;                     // (head, sender) rows a CTA can receive: ceil(NQ / S) * S
    static constexpr int kRing = kDecodeWarps * kGroups * kGroup;
    static constexpr int kOuts = kDecodeWarps * NQ * HD * 4;
    static constexpr int kQ = kRing > kOuts ? kRing : kOuts;              // the warps' outputs take the ring's place at the end
    static constexpr int kPart = kQ + NQ * 3 * HD;
    static constexpr int kSmall = kPart + kRecv * HD * 4;                 // units [NQ], received [kRecv][2], ml [warps][NQ][2]
    static constexpr int kNew = (kSmall + (NQ + 2 * kRecv + 2 * kDecodeWarps * NQ) * 4 + 15) / 16 * 16;
    static constexpr int kBytes = kNew + NewRows<HD>::kBytes;
};
// What bounds it: bytes where caches are long (32 x 8 kv heads x 4 queries, up to 8192 positions, 287 MB: 53.8 to 57.1 us from box to box, 0.77
// to 0.81 of the rate of a plain copy; all of 4096: 49.4, 0.86), a chain of latencies where they are short: position, cosines,
// digits, first tile, merge (1 x 16 heads, 130 positions: 5.1 us; 8 x 16, 576: 7.9).  Groups of more than eight queries read the rows once for
// every eight (32 x 8 kv heads, 4096 positions: 57.5 us with 8 queries, 104 with 16, 184 with 32).
// PER_SM: CTAs that an SM has to hold.  With three the kernel keeps within 168 registers, where the compiler spills a few that it
// needs at the end; with 2 it uses 175.
template <int HD, int NQ, bool PREFIX, int PER_SM>
__global__ void __launch_bounds__(kDecodeWarps * 32, PER_SM) attn_decode_int8_kernel(const DecodeArgs a) {
    namespace cg = cooperative_groups;
    using Shape = DecodeShape<HD, NQ>;
    constexpr int VEC = HD / 32, W = kDecodeWarps, ST = Shape::ST, STEP = Shape::kStep, GROUP = Shape::kGroup;
    using Attn = WarpAttention<HD, NQ, ST>;
    constexpr int QPW = (NQ + W - 1) / W;                                  // queries that a warp prepares
    extern __shared__ __align__(128) uint8_t sm[];
    uint8_t* sm_q = sm + Shape::kQ;
    float* sm_part = reinterpret_cast<float*>(sm + Shape::kPart);         // [kRecv][HD]
    float* sm_unit = reinterpret_cast<float*>(sm + Shape::kSmall);
    float* sm_part_ml = sm_unit + NQ;                                     // [kRecv][2]
    float* sm_ml = sm_part_ml + 2 * Shape::kRecv;
    float* sm_o = reinterpret_cast<float*>(sm);                           // [W][NQ][HD]
    cg::cluster_group cluster = cg::this_cluster();
    const int S = gridDim.z;
    pdl_launch_dependents();
    // Behind a prefix kernel only its partial results have to be waited for: that kernel lets this one start when
    // everything older than the two is complete.
    if (!PREFIX) pdl_wait();
    if (S > 1) cluster_arrive();                                           // every CTA is there when it comes to storing into it
    const int b = blockIdx.x / a.n_kv, hk = blockIdx.x - b * a.n_kv, G = a.n_heads / a.n_kv;
    const int q0 = blockIdx.y * NQ, nq = min(NQ, G - q0);             // this block's queries of the group
    const int split = blockIdx.z;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int64_t base = (static_cast<int64_t>(b) * a.n_kv + hk) * a.own.max_seq;
    uint8_t* ring = sm + warp * kGroups * GROUP;
    const uint32_t ring_u = smem_u32(ring);
    const int first = (split * W + warp) * STEP, stride = S * W * STEP, rows = static_cast<int>(a.own.max_seq);
    auto keys = [&](int to, int t, int end) {                              // asks for the step's keys, or values, at position t
        request_group<HD, 32, ST, true>(ring_u + to * GROUP, a.own.kc + base * HD, a.own.ks + base, t, kTile, end, lane);
        cp_async_commit();
    };
    auto values = [&](int to, int t, int end) {
        request_group<HD, 32, ST, false>(ring_u + to * GROUP, a.own.vc + base * HD, a.own.vs + base, t, kTile, end, lane);
        cp_async_commit();
    };
    // The first tile is asked for before the position is known: its rows lie inside the cache in any case.
    keys(0, first, rows);
    values(1, first, rows);
    const float* row = a.qkv + b * a.qkv_stride + static_cast<int64_t>(hk * G + q0) * HD + lane * VEC;
    float qv[QPW][VEC];
#pragma unroll
    for (int i = 0; i < QPW; ++i)
#pragma unroll
        for (int j = 0; j < VEC; ++j) qv[i][j] = warp + i * W < nq ? row[(warp + i * W) * HD + j] : 0.f;
    float new_k[VEC], new_v[VEC];
    if (warp == W - 1) NewRows<HD>::load(a, b, hk, new_k, new_v, lane);
    const int64_t pos = a.pos[b * a.pos_stride];
    const bool live = pos >= 0 && pos < a.own.max_seq;
    const int64_t P = PREFIX ? prefix_rows(a) : 0;
    const int n = live ? static_cast<int>(pos) + 1 : 0;
    const float* cos_row = a.cos_t + (live ? P + pos : 0) * (HD / 2);
    const float* sin_row = a.sin_t + (live ? P + pos : 0) * (HD / 2);
    keys(2, first + stride, n);
#pragma unroll
    for (int i = 0; i < QPW; ++i) {
        rotate_row<HD>(qv[i], cos_row, sin_row, lane);
        query_planes<HD>(qv[i], sm_q + (warp + i * W) * Attn::kQueryBytes, sm_unit + warp + i * W, lane);
    }
    // The CTA whose warp takes the last tile makes the new token's rows (and stores them, in one query block of the group): its last
    // warp, which has no query of its own where the group has fewer than four.
    const int last_warp = n > 0 ? (n - 1) / STEP % (S * W) - split * W : -1;
    const bool owner = last_warp == warp;
    uint8_t* fresh = sm + Shape::kNew;
    if (warp == W - 1 && last_warp >= 0 && last_warp < W) NewRows<HD>::make(a, new_k, new_v, cos_row, sin_row, fresh, base + pos, blockIdx.y == 0, lane);
    __syncthreads();
    Attn w;
    w.init(lane);
    w.use_queries(sm_q, sm_unit);
    int slot = 0;
    for (int t = first; t < n; t += stride) {
        int left[ST];
#pragma unroll
        for (int j = 0; j < ST; ++j) left[j] = n - t - j * kTile;
        const bool last = owner && t + STEP >= n;
        const int r = n - 1 - t;                                           // the new row's place in the last step
        float sc[ST][Attn::NS][4];
        cp_async_wait<kGroups - 1>();
        __syncwarp();                                                      // the keys are there
        uint8_t* group = ring + slot * GROUP;
        if (last) NewRows<HD>::template bring_in<true>(fresh, group + r / kTile * Half<HD>::kBytes, r % kTile, lane);
        w.scores_of(sc, group, left);
        __syncwarp();                                                      // everyone is through with them
        values(slot, t + stride, n);
        slot = next_slot(slot);
        cp_async_wait<kGroups - 1>();
        __syncwarp();
        group = ring + slot * GROUP;
        if (last) NewRows<HD>::template bring_in<false>(fresh, group + r / kTile * Half<HD>::kBytes, r % kTile, lane);
        w.accumulate(sc, group, left);
        __syncwarp();
        keys(slot, t + 2 * stride, n);
        slot = next_slot(slot);
    }
    cp_async_wait<0>();
    __syncthreads();                                                       // the rings are free
    w.store(sm_ml + warp * 2 * NQ, sm_o + warp * NQ * HD);
    __syncthreads();
    if (S > 1) cluster_wait();
    for (int i = threadIdx.x; i < nq * HD; i += W * 32) {
        const int q = i / HD, d = i % HD;
        Joined j = {-CUDART_INF_F, 0.f, 0.f};
#pragma unroll
        for (int u = 0; u < W; ++u) join_part(j, sm_ml[(u * NQ + q) * 2], sm_ml[(u * NQ + q) * 2 + 1], sm_o[(u * NQ + q) * HD + d]);
        const int to = q % S, at = q / S * S + split;                      // row `at` of CTA `to`
        cluster.map_shared_rank(sm_part, to)[at * HD + d] = j.A;
        if (d == 0) {
            float* ml = cluster.map_shared_rank(sm_part_ml, to) + 2 * at;
            ml[0] = j.M;
            ml[1] = j.L;
        }
    }
    if (PREFIX) pdl_wait();
    if (S > 1) {
        cluster_arrive();
        cluster_wait();
    } else {
        __syncthreads();
    }
    for (int i = warp; split + i * S < nq; i += W) {                       // a warp finishes every W-th of this CTA's heads
        JoinedHead<HD> j;
        j.template join<4>(S, [&](int r, float& m, float& l, float (&v)[VEC]) {
            m = sm_part_ml[2 * (i * S + r)];
            l = sm_part_ml[2 * (i * S + r) + 1];
            load_values_of(sm_part + (i * S + r) * HD + lane * VEC, v);
        });
        j.template finish<PREFIX>(a, b, hk * G + q0 + split + i * S, live, sm_o + warp * HD, lane);
    }
}

// Long caches.  The steps (ST tiles) of all units (sequence, kv head, query block) in a row are dealt out evenly to all warps of
// one CTA per SM: a warp works on one run of steps, which may end one unit and begin others, and writes a partial result for
// each unit it touches.  How many steps a unit has follows from `pos` alone, so every warp (and the kernel that joins the
// results) finds its place by itself: nothing is handed out at run time and the result does not depend on timing.
// The partial result of warp w for unit u goes to slot w + u: from one part of the row to the next w or u grows.
// What bounds it: bytes; 11 us are spent around a stream that runs at the rate of a plain copy (1 x 8 kv heads x 4 queries: 131072
// positions 52.8 us with the joining kernel, each further 131072 another 42.2).  A warp with a ring of its own, one CTA of 8 per SM:
// 201 KB of tiles under way, no barrier between warps.
constexpr int kFlatWarpsPerSm = 8, kFlatWarps = kSms * kFlatWarpsPerSm;
template <int HD, int NQ>
struct FlatShape {
    static constexpr int ST = HD == 128 ? 2 : 4, kStep = ST * kTile, kGroup = ST * Half<HD>::kBytes;
    static constexpr int kQ = kFlatWarpsPerSm * kGroups * kGroup;         // digits [W][NQ][3][HD]
    static constexpr int kSmall = kQ + kFlatWarpsPerSm * NQ * 3 * HD;     // units [W][NQ]
    static constexpr int kNew = kSmall + kFlatWarpsPerSm * NQ * 4;        // new rows [W]
    static constexpr int kBytes = kNew + kFlatWarpsPerSm * NewRows<HD>::kBytes;
};
// How the row of steps is dealt out.  Every warp works it out, from 32 sequences at a time.
struct FlatPlan {
    int total, per;
    static __device__ __forceinline__ int steps(const DecodeArgs& a, int64_t b, int step) {
        const int64_t pos = a.pos[b * a.pos_stride];
        return pos >= 0 && pos < a.own.max_seq ? static_cast<int>(pos / step) + 1 : 0;
    }
    // steps of all sequences (for one head and query block), and of those in front of sequence b
    __device__ __forceinline__ int make(const DecodeArgs& a, int units_per_seq, int b, int step, int lane) {
        int all = 0, front = 0;
        for (int i = lane; i < a.batch; i += 32) {
            const int t = steps(a, i, step);
            all += t;
            front += i < b ? t : 0;
        }
        total = __reduce_add_sync(0xffffffffu, all) * units_per_seq;
        per = max((total + kFlatWarps - 1) / kFlatWarps, 1);
        return __reduce_add_sync(0xffffffffu, front);
    }
};
template <int HD, int NQ, bool PREFIX>
__global__ void __launch_bounds__(kFlatWarpsPerSm * 32) attn_flat_int8_kernel(const DecodeArgs a, int blocks) {
    using Shape = FlatShape<HD, NQ>;
    constexpr int ST = Shape::ST, VEC = HD / 32, STEP = Shape::kStep;
    using Attn = WarpAttention<HD, NQ, ST>;
    extern __shared__ __align__(128) uint8_t sm[];
    if (!PREFIX) pdl_wait();                                          // else at the end: see attn_decode_int8_kernel
    pdl_launch_dependents();                                          // behind the wait: the joining kernel reads `pos` at once
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, G = a.n_heads / a.n_kv, units_per_seq = a.n_kv * blocks;
    const int gw = blockIdx.x * kFlatWarpsPerSm + warp;
    uint8_t* ring = sm + warp * kGroups * Shape::kGroup;
    uint8_t* sm_q = sm + Shape::kQ + warp * NQ * Attn::kQueryBytes;
    float* sm_unit = reinterpret_cast<float*>(sm + Shape::kSmall) + warp * NQ;
    const uint32_t ring_u = smem_u32(ring);
    FlatPlan plan;
    plan.make(a, units_per_seq, 0, STEP, lane);
    const int64_t lo = static_cast<int64_t>(gw) * plan.per;
    int left = static_cast<int>(min(static_cast<int64_t>(plan.per), plan.total - lo));
    if (left > 0) {
        // the sequence, unit and step this warp's run begins with
        int b = 0, before = 0, T = 0;
        for (int b0 = 0; b0 < a.batch; b0 += 32) {
            const int mine = b0 + lane < a.batch ? FlatPlan::steps(a, b0 + lane, STEP) * units_per_seq : 0;
            int up = mine;
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) {
                const int x = __shfl_up_sync(0xffffffffu, up, d);
                if (lane >= d) up += x;
            }
            const uint32_t past = __ballot_sync(0xffffffffu, before + up > lo);
            if (past) {
                const int at = __ffs(past) - 1;
                T = __shfl_sync(0xffffffffu, mine, at) / units_per_seq;
                before += __shfl_sync(0xffffffffu, up - mine, at);
                b = b0 + at;
                break;
            }
            before += __shfl_sync(0xffffffffu, up, 31);
        }
        if (T == 0) left = 0;                                              // cannot be, unless somebody writes `pos` meanwhile
        T = max(T, 1);
        const int off = static_cast<int>(lo - before);
        // A place in the row of steps: step s of T of unit j of sequence b, which has n positions
        struct Place {
            int b, j, s, T, n;
        };
        auto positions = [&](int seq) { return static_cast<int>(a.pos[seq * a.pos_stride]) + 1; };
        auto advance = [&](Place& p) {                                     // only called while the run goes on: there is a next step
            if (++p.s < p.T) return;
            p.s = 0;
            if (++p.j < units_per_seq) return;
            p.j = 0;
            do { p.T = FlatPlan::steps(a, ++p.b, STEP); } while (p.T == 0 && p.b + 1 < a.batch);
            p.n = positions(p.b);
        };
        Place use = {b, off / T, off % T, T, positions(b)}, ask = use;
        int to_ask = left;                                                 // steps whose values have not been asked for
        int slot_ask = 0;
        auto request = [&](bool keys) {
            if (to_ask > 0) {
                const int64_t base = (static_cast<int64_t>(ask.b) * a.n_kv + ask.j / blocks) * a.own.max_seq;
                const uint32_t dst = ring_u + slot_ask * Shape::kGroup;
                if (keys) {
                    request_group<HD, 32, ST, true>(dst, a.own.kc + base * HD, a.own.ks + base, ask.s * STEP, kTile, ask.n, lane);
                } else {
                    request_group<HD, 32, ST, false>(dst, a.own.vc + base * HD, a.own.vs + base, ask.s * STEP, kTile, ask.n, lane);
                    if (--to_ask > 0) advance(ask);
                }
            }
            cp_async_commit();
            slot_ask = next_slot(slot_ask);
        };
        request(true);
        request(false);
        request(true);
        Attn w;
        uint8_t* fresh = sm + Shape::kNew + warp * NewRows<HD>::kBytes;
        bool begin = true;
        int slot = 0;
        for (; left > 0; --left) {
            const int hk = use.j / blocks, qb = use.j - hk * blocks, q0 = qb * NQ, nq = min(NQ, G - q0);
            const bool end = use.s + 1 == use.T;                           // of the unit
            if (begin) {
                const int64_t turn = ((PREFIX ? prefix_rows(a) : 0) + use.n - 1) * (HD / 2);
                const float* row = a.qkv + use.b * a.qkv_stride + static_cast<int64_t>(hk * G + q0) * HD + lane * VEC;
                float qv[NQ][VEC];
#pragma unroll
                for (int q = 0; q < NQ; ++q)
#pragma unroll
                    for (int j = 0; j < VEC; ++j) qv[q][j] = q < nq ? row[q * HD + j] : 0.f;
#pragma unroll
                for (int q = 0; q < NQ; ++q) {
                    rotate_row<HD>(qv[q], a.cos_t + turn, a.sin_t + turn, lane);
                    query_planes<HD>(qv[q], sm_q + q * Attn::kQueryBytes, sm_unit + q, lane);
                }
                if (use.s + left >= use.T) {                               // the run holds the unit's last step
                    float x[VEC], y[VEC];
                    NewRows<HD>::load(a, use.b, hk, x, y, lane);
                    NewRows<HD>::make(a, x, y, a.cos_t + turn, a.sin_t + turn, fresh,
                                      (static_cast<int64_t>(use.b) * a.n_kv + hk) * a.own.max_seq + use.n - 1, qb == 0, lane);
                }
                __syncwarp();
                w.init(lane);
                w.use_queries(sm_q, sm_unit);
                begin = false;
            }
            int in[ST];
#pragma unroll
            for (int j = 0; j < ST; ++j) in[j] = use.n - use.s * STEP - j * kTile;
            const int r = (use.n - 1) % STEP;                              // the new row's place in the last step
            float sc[ST][Attn::NS][4];
            cp_async_wait<kGroups - 1>();
            __syncwarp();                                                  // the keys are there
            uint8_t* group = ring + slot * Shape::kGroup;
            if (end) NewRows<HD>::template bring_in<true>(fresh, group + r / kTile * Half<HD>::kBytes, r % kTile, lane);
            w.scores_of(sc, group, in);
            __syncwarp();                                                  // everyone is through with them
            request(false);
            slot = next_slot(slot);
            cp_async_wait<kGroups - 1>();
            __syncwarp();
            group = ring + slot * Shape::kGroup;
            if (end) NewRows<HD>::template bring_in<false>(fresh, group + r / kTile * Half<HD>::kBytes, r % kTile, lane);
            w.accumulate(sc, group, in);
            __syncwarp();
            request(true);
            slot = next_slot(slot);
            if (end || left == 1) {
                const int64_t to = gw + static_cast<int64_t>(use.b) * units_per_seq + use.j;
                w.store(a.flat_ml + to * NQ * 2, a.flat_o + to * NQ * HD, nq);
                begin = true;
            }
            if (left > 1) advance(use);
        }
    }
    cp_async_wait<0>();
    if (PREFIX) pdl_wait();
}

constexpr int kJoinWarps = 16;         // of a block (8 / 16 / 32: 1 x 8 heads, 131072 positions 54.6 / 53.2 / 53.6 us, 16384 16.6 / 15.5 / 14.9)
// Joins the partial results of attn_flat_int8_kernel (and of a prefix).  WIDE: a block per (sequence, query head), whose warps take
// the slots in turn; else a warp per (sequence, query head).  A lane holds HD / 32 values.  Where the slots are follows from
// `pos`, which is older than the kernel in front: that is worked out before its results are waited for.
template <int HD, int NQ, bool WIDE, bool PREFIX>
__global__ void __launch_bounds__((WIDE ? kJoinWarps : kWarps) * 32) attn_flat_join_kernel(const DecodeArgs a, int blocks) {
    constexpr int VEC = HD / 32, STEP = FlatShape<HD, NQ>::kStep, W = WIDE ? kJoinWarps : kWarps, BY = WIDE ? W : 1;
    __shared__ float sm_ml[W][2];
    __shared__ __align__(16) float sm_o[W][HD];
    pdl_launch_dependents();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, G = a.n_heads / a.n_kv, units_per_seq = a.n_kv * blocks;
    const int64_t bh = WIDE ? blockIdx.x : static_cast<int64_t>(blockIdx.x) * W + warp;
    const bool there = bh < static_cast<int64_t>(a.batch) * a.n_heads;
    const int b = there ? static_cast<int>(bh / a.n_heads) : 0, h = there ? static_cast<int>(bh - static_cast<int64_t>(b) * a.n_heads) : 0;
    const int hk = h / G, g = h - hk * G, j = hk * blocks + g / NQ;
    FlatPlan plan;
    const int front = plan.make(a, units_per_seq, b, STEP, lane) * units_per_seq, T = FlatPlan::steps(a, b, STEP);
    const int start = front + j * T, w0 = start / plan.per, w1 = T > 0 ? (start + T - 1) / plan.per : w0 - 1;
    const int64_t unit = static_cast<int64_t>(b) * units_per_seq + j;
    JoinedHead<HD> t;
    pdl_wait();
    const int w_first = w0 + (WIDE ? warp : 0);
    t.template join<6>(w_first <= w1 ? (w1 - w_first) / BY + 1 : 0, [&](int p, float& m, float& l, float (&v)[VEC]) {
        const int64_t at = (unit + w_first + p * BY) * NQ + g % NQ;
        m = a.flat_ml[2 * at];
        l = a.flat_ml[2 * at + 1];
        load_values_of(a.flat_o + at * HD + lane * VEC, v);
    });
    if constexpr (WIDE) {
        if (lane == 0) { sm_ml[warp][0] = t.M; sm_ml[warp][1] = t.L; }
#pragma unroll
        for (int i = 0; i < VEC; ++i) sm_o[warp][lane * VEC + i] = t.A[i];
        __syncthreads();
        if (warp != 0) return;
        t = JoinedHead<HD>();
        t.template join<4>(W, [&](int u, float& m, float& l, float (&v)[VEC]) {
            m = sm_ml[u][0];
            l = sm_ml[u][1];
            load_values_of(&sm_o[u][lane * VEC], v);
        });
        __syncwarp();
    }
    if (there) t.template finish<PREFIX>(a, b, h, T > 0, &sm_o[warp][0], lane);
}

// Partial attention of every sequence's queries to the shared prefix.  grid (kv heads, splits of the prefix, blocks of 8 QW rows),
// the rows of a kv head being its queries (b, g) in the order b * G + g.  A warp carries 8 rows; the QW warps of a group
// take the same tiles, which they fetch together into the group's ring, and the KW = 8 / QW groups take alternate tiles.
// What bounds it: the s8 products of mma.sync, 8 cycles each on an SM's quarter, from 16 rows on (32 rows x 8 heads behind 16384
// positions: 35.2 us with the decode behind it); below, start, digits and the hand-over (8 rows x 16 heads behind 2048: 11.4).
template <int HD, int QW>
struct PrefixShape {
    static constexpr int NQ = 8, KW = kWarps / QW;
    // tiles per step: 4 x 8 rows behind 16384 positions 22.6 / 24.9 us with 1 / 2, 24 x 16 behind 4096 25.8 / 24.1
    static constexpr int ST = (QW == 4 ? 2 : 1) * (128 / HD);
    static constexpr int kGroup = ST * Half<HD>::kBytes, kRing = KW * kGroups * kGroup;
    static constexpr int kOuts = kWarps * NQ * HD * 4;
    static constexpr int kQ = kRing > kOuts ? kRing : kOuts;
    static constexpr int kSmall = kQ + QW * NQ * 3 * HD;                  // units [QW][NQ], ml [warps][NQ][2]
    static constexpr int kBytes = kSmall + (QW * NQ + kWarps * NQ * 2) * 4;
};
template <int HD, int QW>
__global__ void __launch_bounds__(kWarps * 32) attn_prefix_int8_kernel(const DecodeArgs a) {
    using Shape = PrefixShape<HD, QW>;
    constexpr int NQ = Shape::NQ, KW = Shape::KW, ST = Shape::ST;
    using Attn = WarpAttention<HD, NQ, ST>;
    extern __shared__ __align__(128) uint8_t sm[];
    uint8_t* sm_q = sm + Shape::kQ;
    float* sm_unit = reinterpret_cast<float*>(sm + Shape::kSmall);
    float* sm_ml = sm_unit + QW * NQ;
    float* sm_o = reinterpret_cast<float*>(sm);
    pdl_wait();
    pdl_launch_dependents();                                                // behind the wait: see attn_decode_int8_kernel
    const int hk = blockIdx.x, split = blockIdx.y, splits = gridDim.y, G = a.n_heads / a.n_kv;
    const int64_t R = static_cast<int64_t>(a.batch) * G, r0 = static_cast<int64_t>(blockIdx.z) * QW * NQ;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, qg = warp % QW, kw = warp / QW, in_group = threadIdx.x % (QW * 32);
    const int n = static_cast<int>(prefix_rows(a));
    const int chunk = ((n + splits - 1) / splits + kTile - 1) / kTile * kTile;
    const int t0 = min(static_cast<int64_t>(split) * chunk, static_cast<int64_t>(n)), t1 = min(static_cast<int64_t>(t0) + chunk, static_cast<int64_t>(n));
    const int64_t base = static_cast<int64_t>(hk) * a.first.max_seq;
    const int8_t* kc = a.first.kc + base * HD;
    const int8_t* vc = a.first.vc + base * HD;
    const float* ks = a.first.ks + base;
    const float* vs = a.first.vs + base;

    uint8_t* ring = sm + kw * kGroups * Shape::kGroup;
    const uint32_t ring_u = smem_u32(ring);
    constexpr int BETWEEN = KW * kTile, STRIDE = ST * BETWEEN;              // tiles of a step, steps
    auto request = [&](int slot, int t, bool keys) {
        const uint32_t dst = ring_u + slot * Shape::kGroup;
        if (keys) request_group<HD, QW * 32, ST, true>(dst, kc, ks, t, BETWEEN, t1, in_group);
        else request_group<HD, QW * 32, ST, false>(dst, vc, vs, t, BETWEEN, t1, in_group);
        cp_async_commit();
    };
    auto group_sync = [&] {
        if constexpr (QW == 1) __syncwarp();
        else named_barrier_sync(1 + kw, QW * 32);
    };
    const int first = t0 + kw * kTile;
    request(0, first, true);
    request(1, first, false);
    request(2, first + STRIDE, true);
    float v[QW][HD / 32];                                                   // this warp's rows: warp, warp + 8, ...
#pragma unroll
    for (int i = 0; i < QW; ++i) {
        const int64_t r = r0 + warp + i * kWarps;
        const int64_t b = r < R ? r / G : 0;
        const int64_t pos = a.pos[b * a.pos_stride];
        const bool live = r < R && pos >= 0 && pos < a.own.max_seq;
        const int64_t turn = (live ? n + pos : 0) * (HD / 2);
#pragma unroll
        for (int j = 0; j < HD / 32; ++j) v[i][j] = live ? a.qkv[b * a.qkv_stride + (hk * G + r - b * G) * HD + lane * (HD / 32) + j] : 0.f;
        rotate_row<HD>(v[i], a.cos_t + turn, a.sin_t + turn, lane);
    }
#pragma unroll
    for (int i = 0; i < QW; ++i) {
        const int q = warp + i * kWarps;
        query_planes<HD>(v[i], sm_q + q * Attn::kQueryBytes, sm_unit + q, lane);
    }
    __syncthreads();
    Attn w;
    w.init(lane);
    w.use_queries(sm_q + qg * NQ * Attn::kQueryBytes, sm_unit + qg * NQ);
    int slot = 0;
    for (int t = first; t < t1; t += STRIDE) {
        int left[ST];
#pragma unroll
        for (int j = 0; j < ST; ++j) left[j] = t1 - t - j * BETWEEN;
        float sc[ST][Attn::NS][4];
        cp_async_wait<kGroups - 1>();
        group_sync();                                                       // the keys are there
        w.scores_of(sc, ring + slot * Shape::kGroup, left);
        group_sync();                                                       // everyone is through with them
        request(slot, t + STRIDE, false);
        slot = next_slot(slot);
        cp_async_wait<kGroups - 1>();
        group_sync();
        w.accumulate(sc, ring + slot * Shape::kGroup, left);
        group_sync();
        request(slot, t + 2 * STRIDE, true);
        slot = next_slot(slot);
    }
    cp_async_wait<0>();
    __syncthreads();                                                        // the rings are free
    w.store(sm_ml + warp * 2 * NQ, sm_o + warp * NQ * HD);
    __syncthreads();
    for (int i = threadIdx.x; i < QW * NQ * HD; i += kWarps * 32) {
        const int q = i / HD, d = i % HD;
        if (r0 + q >= R) break;
        Joined j = {-CUDART_INF_F, 0.f, 0.f};
#pragma unroll
        for (int u = 0; u < KW; ++u) {
            const int at = (q / NQ + u * QW) * NQ + q % NQ;
            join_part(j, sm_ml[2 * at], sm_ml[2 * at + 1], sm_o[at * HD + d]);
        }
        const int64_t to = (hk * R + r0 + q) * splits + split;
        a.part_o[to * HD + d] = j.A;
        if (d == 0) { a.part_ml[2 * to] = j.M; a.part_ml[2 * to + 1] = j.L; }
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
// Do `rows` rows of wx floats, sx apart, and of wy floats, sy apart, share memory?  (Columns of one wider matrix do not.)
bool rows_overlap(const float* x, int64_t sx, int64_t wx, const float* y, int64_t sy, int64_t wy, int64_t rows) {
    using wide = __int128;
    const wide a = reinterpret_cast<uintptr_t>(x) / 4, b = reinterpret_cast<uintptr_t>(y) / 4, steps = rows - 1;
    if (a + steps * sx + wx <= b || b + steps * sy + wy <= a) return false;
    if (sx != sy || rows == 1) return true;
    const wide d = ((b - a) % sx + sx) % sx;
    return d < wx || d + wy > sx;
}
// Memory that a call reads or writes
struct Span {
    uintptr_t from, to;
    bool meets(const Span& other) const { return from < other.to && other.from < to; }
};
Span span(const void* p, int64_t a, int64_t b, int64_t c, int64_t d) {      // a * b * c * d bytes at p, none where p is NULL
    const uintptr_t from = reinterpret_cast<uintptr_t>(p);
    const unsigned __int128 most = UINTPTR_MAX - from, bytes = static_cast<unsigned __int128>(a * b) * static_cast<uint64_t>(c * d);
    return Span{from, p ? from + static_cast<uintptr_t>(std::min(bytes, most)) : from};
}
Span span_of_rows(const float* p, int64_t rows, int64_t stride, int64_t width) {
    const __int128 floats = static_cast<__int128>(rows - 1) * stride + width;
    return span(p, 1, 1, 4, static_cast<int64_t>(std::min<__int128>(floats, INT64_MAX / 4)));
}
struct CacheSpans {
    Span s[4];
    explicit CacheSpans(const sgqd_cache_int8* c)
        : s{span(c->k_codes, c->batch, c->n_kv_heads, c->max_seq, c->head_dim), span(c->k_scales, c->batch, c->n_kv_heads, c->max_seq, 4),
            span(c->v_codes, c->batch, c->n_kv_heads, c->max_seq, c->head_dim), span(c->v_scales, c->batch, c->n_kv_heads, c->max_seq, 4)} {}
    bool meets(const Span& other) const { return s[0].meets(other) || s[1].meets(other) || s[2].meets(other) || s[3].meets(other); }
    bool meets(const CacheSpans& other) const { return meets(other.s[0]) || meets(other.s[1]) || meets(other.s[2]) || meets(other.s[3]); }
    bool apart() const {                                                    // the four arrays from one another
        for (int i = 0; i < 4; ++i)
            for (int j = 0; j < i; ++j)
                if (s[i].meets(s[j])) return false;
        return true;
    }
};
CacheView view(const sgqd_cache_int8* c) { return CacheView{c->k_codes, c->k_scales, c->v_codes, c->v_scales, c->max_seq}; }

// Splits of a shared prefix and rows per block of its kernel: a function of the sizes alone, so that the workspace's size is one
// too: the plans count 148 SMs, whatever the device has.
struct PrefixPlan {
    int qw;                              // warps side by side on 8 rows each, 0: the tcgen05 kernel
    int blocks, splits;
    int64_t rows;                        // (kv head, query row) pairs
    size_t off_o, bytes;
};
PrefixPlan prefix_plan(int64_t batch, int64_t n_heads, int64_t n_kv, int64_t head_dim, int64_t prefix_max) {
    PrefixPlan p = {};
    const int64_t R = batch * (n_heads / n_kv);
    // Up to 32 rows the tcgen05 kernel's 128 are mostly idle.  Measured, decode included (us, warps / tcgen05): 20 rows x 16 heads, 1024
    // positions 15.1 / 20.2; 24 x 8, 4096 18.9 / 23.3; 24 x 16 heads of 64, 8192 24.7 / 33.5; 32 x 8, 16384 35.9 / 40.6.  More
    // rows would take the warps a second pass over the prefix (48 x 8, 4096 on tcgen05: 21.8).
    p.qw = R <= 8 ? 1 : (R <= 16 ? 2 : (R <= 32 ? 4 : 0));
    const int64_t per_block = p.qw ? 8 * p.qw : kPrefixTcRows;
    p.blocks = static_cast<int>(ceil_div(R, per_block));
    const int64_t most = ceil_div(prefix_max, p.qw ? kTile * (kWarps / p.qw) : kPrefixTcTile);        // a tile for every group of warps
    // Splits: the least of steps of a CTA (1 us, 2.6 of the tcgen05 kernel) and 0.1 us for each part that is joined.  Measured against as
    // many as there are SMs or steps: 68 rows x 1 head, 14354 positions 24.4 -> 21.9 us, 8 x 1 of 64, 30437 14.7 -> 10.4, 30 x 1, 9000 23.5 ->
    // 15.7; 6 x 2, 20685 11.7 -> 12.0.
    const int64_t room = std::max<int64_t>(std::min(kSms / (n_kv * p.blocks), most), 1), step = p.qw ? 10 : 26;
    int64_t least = 0;
    for (int64_t s = 1; s <= room; ++s) {
        const int64_t cost = ceil_div(most, s) * step + s;
        if (s == 1 || cost < least) { least = cost; p.splits = static_cast<int>(s); }
    }
    p.rows = n_kv * R;
    p.off_o = (static_cast<size_t>(p.rows) * p.splits * 8 + 255) / 256 * 256;
    p.bytes = p.off_o + static_cast<size_t>(p.rows) * p.splits * head_dim * 4;
    return p;
}

template <int HD, int QW>
int launch_prefix(const DecodeArgs& a, const PrefixPlan& plan, cudaStream_t s) {
    static SmemOptIn opt_in;
    constexpr int bytes = PrefixShape<HD, QW>::kBytes;
    SGQ_CUDA_TRY(opt_in.ensure(attn_prefix_int8_kernel<HD, QW>, bytes));
    const dim3 grid(static_cast<unsigned>(a.n_kv), static_cast<unsigned>(plan.splits), static_cast<unsigned>(plan.blocks));
    SGQ_CUDA_TRY(launch_kernel(attn_prefix_int8_kernel<HD, QW>, grid, dim3(kWarps * 32), bytes, s, true, a));
    return SGQ_OK;
}
template <int HD>
int launch_prefix(const DecodeArgs& a, const PrefixPlan& plan, cudaStream_t s) {
    if (plan.qw == 0) return launch_prefix_tc(a, HD, plan.splits, plan.blocks, s);
    if (plan.qw == 4) return launch_prefix<HD, 4>(a, plan, s);
    return plan.qw == 1 ? launch_prefix<HD, 1>(a, plan, s) : launch_prefix<HD, 2>(a, plan, s);
}

// Which kernel reads the sequences' own rows.  `flat`: few units over long caches, where clusters cannot fill the device (one
// sequence x 8 heads: 18.8 -> 15.4 us at 16384 positions, 110 -> 53 us at 131071); its second launch costs 3 us.
struct DecodePlan {
    int nq, blocks, splits;
    int64_t units;                       // (sequence, kv head, query block)
    bool flat;
    size_t off_o, bytes;                 // of the flat kernel's partial results
};
DecodePlan decode_plan(int64_t batch, int64_t n_heads, int64_t n_kv, int64_t head_dim, int64_t max_seq) {
    DecodePlan p = {};
    const int64_t G = n_heads / n_kv;
    // four queries per warp where the group has no more: 2 column sets in the place of 3 and half the outputs in registers
    p.nq = G <= 4 ? 4 : 8;
    p.blocks = static_cast<int>(ceil_div(G, p.nq));
    p.units = batch * n_kv * p.blocks;
    const int64_t units = p.units, tiles = ceil_div(max_seq, kTile);
    p.flat = units * kMaxSplits < 3 * kSms && units * tiles >= 16 * kSms && units * tiles < (1 << 30);
    if (p.flat) {
        const size_t slots = static_cast<size_t>(units + kFlatWarps);
        p.off_o = (slots * p.nq * 8 + 255) / 256 * 256;
        p.bytes = p.off_o + slots * p.nq * head_dim * 4;
    }
    // Splits: the least of waves x (what a CTA costs beside its steps, in steps: 3, and 1 for each CTA that shares the SM, + steps of a
    // warp).  Measured (us): batch 8 x 16 heads, 576 positions 9.6 / 8.8 / 10.8 / 12.7 with 1 / 2 / 3 / 4 splits; batch 32 x 8
    // heads, 512 positions 9 / 16 with 1 / 2, of up to 8192 76 / 58 / 56 / 55 / 62 with 1 / 2 / 3 / 4 / 8; batch 37 x 16, 2048
    // positions 63 / 57 / 65 with 1 / 2 / 4.
    const int64_t steps = ceil_div(max_seq, (128 / head_dim) * kTile);
    int64_t least = 0;
    for (int S = 1; S <= kMaxSplits; ++S) {
        const int64_t ctas = units * S, waves = ceil_div(ctas, 3 * kSms), shared = std::min<int64_t>(ceil_div(ctas, kSms), 3);
        const int64_t cost = waves * (3 + shared + ceil_div(steps, kDecodeWarps * S));
        if (S == 1 || cost < least) { least = cost; p.splits = S; }
    }
    return p;
}

template <int HD, int NQ, bool PREFIX, int PER_SM>
int launch_clusters(const DecodeArgs& a, const DecodePlan& plan, cudaStream_t s) {
    static SmemOptIn opt_in;
    constexpr int bytes = DecodeShape<HD, NQ>::kBytes;
    SGQ_CUDA_TRY(opt_in.ensure(attn_decode_int8_kernel<HD, NQ, PREFIX, PER_SM>, bytes));
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(a.batch * a.n_kv), static_cast<unsigned>(plan.blocks), static_cast<unsigned>(plan.splits));
    cfg.blockDim = dim3(kDecodeWarps * 32);
    cfg.dynamicSmemBytes = bytes;
    cfg.stream = s;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 1;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = static_cast<unsigned>(plan.splits);
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    SGQ_CUDA_TRY(cudaLaunchKernelEx(&cfg, attn_decode_int8_kernel<HD, NQ, PREFIX, PER_SM>, a));
    return SGQ_OK;
}
template <int HD, int NQ, bool PREFIX>
int launch_decode(const DecodeArgs& a, const DecodePlan& plan, cudaStream_t s) {
    if (plan.flat) {
        static SmemOptIn opt_in;
        constexpr int bytes = FlatShape<HD, NQ>::kBytes;
        SGQ_CUDA_TRY(opt_in.ensure(attn_flat_int8_kernel<HD, NQ, PREFIX>, bytes));
        SGQ_CUDA_TRY(launch_kernel(attn_flat_int8_kernel<HD, NQ, PREFIX>, dim3(kSms), dim3(kFlatWarpsPerSm * 32), bytes, s, true, a, plan.blocks));
        const int64_t heads = static_cast<int64_t>(a.batch) * a.n_heads;
        // a head has about kFlatWarps / units slots: with more than a warp asks for at once, a block takes it
        if (plan.units * 6 < kFlatWarps)
            SGQ_CUDA_TRY(launch_kernel(attn_flat_join_kernel<HD, NQ, true, PREFIX>, dim3(static_cast<unsigned>(heads)), dim3(kJoinWarps * 32), 0, s, true, a, plan.blocks));
        else
            SGQ_CUDA_TRY(launch_kernel(attn_flat_join_kernel<HD, NQ, false, PREFIX>, dim3(static_cast<unsigned>(ceil_div(heads, kWarps))), dim3(kWarps * 32), 0, s, true,
                                       a, plan.blocks));
        return SGQ_OK;
    }
    // Where two per SM take the whole grid, the form that spills nothing (8 x 16 heads, 576 positions: 8.9 -> 8.2 us; 32 x 8 heads,
    // 512 positions 11.4 -> 9.9); else three (32 x 8 heads, 8192 positions: 59 -> 57).
    if constexpr ((HD == 128) == (NQ == 4)) {
        if (plan.units * plan.splits <= 2 * kSms) return launch_clusters<HD, NQ, PREFIX, 2>(a, plan, s);
    }
    return launch_clusters<HD, NQ, PREFIX, 3>(a, plan, s);
}

template <bool PREFIX>
int launch_decode(const DecodeArgs& a, int64_t head_dim, const DecodePlan& plan, cudaStream_t s) {
    if (head_dim == 128) return plan.nq == 4 ? launch_decode<128, 4, PREFIX>(a, plan, s) : launch_decode<128, 8, PREFIX>(a, plan, s);
    return plan.nq == 4 ? launch_decode<64, 4, PREFIX>(a, plan, s) : launch_decode<64, 8, PREFIX>(a, plan, s);
}

size_t decode_workspace(int64_t batch, int64_t n_heads, int64_t n_kv, int64_t head_dim, int64_t max_seq, int64_t prefix_max) {
    if (batch <= 0 || batch > 0x7fffffff || n_heads <= 0 || n_heads > 65535 || n_kv <= 0 || n_heads % n_kv || max_seq <= 0 || max_seq > kMaxPositions ||
        prefix_max < 0 || prefix_max > kMaxPositions || (head_dim != 64 && head_dim != 128))
        return 0;
    const size_t flat = decode_plan(batch, n_heads, n_kv, head_dim, max_seq).bytes;
    return (flat + 255) / 256 * 256 + (prefix_max ? prefix_plan(batch, n_heads, n_kv, head_dim, prefix_max).bytes : 0);
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
    if (!aligned(pos, 4) || !aligned(out, 4) || !aligned(prefix_len, 4)) return bad(SGQ_ERR_ALIGNMENT, "pos, prefix_len and out must be 4-byte aligned");
    if (rows_overlap(qkv, qkv_stride, (n_heads + 2 * kv) * hd, out, out_stride, n_heads * hd, batch))
        return bad(SGQ_ERR_BAD_ARGUMENT, "out overlaps qkv");
    PreparedLayout L = {};
    if ((rc = check_prepared(prepared_out, prepared_bytes, batch, n_heads * hd, &L)) != SGQ_OK) return rc;
    const DecodePlan plan = decode_plan(batch, n_heads, kv, hd, cache->max_seq);
    PrefixPlan first = {};
    if (prefix) {
        first = prefix_plan(batch, n_heads, kv, hd, prefix->max_seq);
        if (first.blocks > 65535) return bad(SGQ_ERR_BAD_SHAPE, "too many query rows for one call");
    }
    const size_t need = decode_workspace(batch, n_heads, kv, hd, cache->max_seq, prefix ? prefix->max_seq : 0);
    if (need && (!workspace || workspace_bytes < need || !aligned(workspace, 256)))
        return bad(SGQ_ERR_WORKSPACE, "workspace too small or not 256-byte aligned");
    if (batch * n_heads > 0x7fffff00) return bad(SGQ_ERR_BAD_SHAPE, "too many query rows for one call");
    // The kernels run next to one another and store rows, scratch and outputs while others are still reading.
    const CacheSpans own(cache);
    const Span results = span_of_rows(out, batch, out_stride, n_heads * hd), rows = span_of_rows(qkv, batch, qkv_stride, (n_heads + 2 * kv) * hd),
               scratch = span(workspace, 1, 1, 1, static_cast<int64_t>(need)),
               planes = span(prepared_out, 1, 1, 1, prepared_out ? static_cast<int64_t>(gemv_prepared_bytes(batch, n_heads * hd)) : 0);
    if (!own.apart()) return bad(SGQ_ERR_BAD_ARGUMENT, "the cache's arrays overlap one another");
    if (prefix && CacheSpans(prefix).meets(own)) return bad(SGQ_ERR_BAD_ARGUMENT, "prefix and cache share memory");
    for (const Span& written : {results, scratch, planes})
        if (own.meets(written) || (prefix && CacheSpans(prefix).meets(written))) return bad(SGQ_ERR_BAD_ARGUMENT, "an output or the workspace overlaps a cache");
    if (scratch.meets(results) || scratch.meets(planes) || scratch.meets(rows) || planes.meets(results) || planes.meets(rows) || own.meets(rows))
        return bad(SGQ_ERR_BAD_ARGUMENT, "outputs, workspace, cache and qkv overlap");
    if ((rc = check_device()) != SGQ_OK) return rc;
    DecodeArgs a = {};
    a.qkv = qkv; a.qkv_stride = qkv_stride; a.n_heads = static_cast<int>(n_heads); a.n_kv = static_cast<int>(kv); a.batch = static_cast<int>(batch);
    a.cos_t = cos_table; a.sin_t = sin_table; a.pos = pos; a.pos_stride = pos_stride; a.own = view(cache);
    a.out = out; a.out_stride = out_stride; a.pmode = L.mode; a.nmain = L.nmain; a.nlow = L.nlow; a.planes = static_cast<uint8_t*>(prepared_out);
    uint8_t* ws = static_cast<uint8_t*>(workspace);
    if (plan.flat) {
        a.flat_ml = reinterpret_cast<float*>(ws);
        a.flat_o = reinterpret_cast<float*>(ws + plan.off_o);
    }
    if (prefix) {
        uint8_t* at = ws + (plan.bytes + 255) / 256 * 256;
        a.first = view(prefix);
        a.prefix_len = prefix_len;
        a.part_ml = reinterpret_cast<float*>(at);
        a.part_o = reinterpret_cast<float*>(at + first.off_o);
        a.parts = first.splits;
        rc = hd == 128 ? launch_prefix<128>(a, first, s) : launch_prefix<64>(a, first, s);
        if (rc != SGQ_OK) return rc;
    }
    return prefix ? launch_decode<true>(a, hd, plan, s) : launch_decode<false>(a, hd, plan, s);
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
    if (!aligned(pos, 4) || !aligned(n_new, 4) || !aligned(rope_offset, 4)) return bad(SGQ_ERR_ALIGNMENT, "pos, n_new and rope_offset must be 4-byte aligned");
    if (q_out != qkv && rows_overlap(qkv, qkv_stride, (n_heads + 2 * kv) * hd, q_out, q_stride, n_heads * hd, cache->batch * t_new))
        return bad(SGQ_ERR_BAD_ARGUMENT, "q_out overlaps qkv and is not qkv itself");
    const CacheSpans own(cache);
    const int64_t tokens = cache->batch * t_new;
    if (!own.apart()) return bad(SGQ_ERR_BAD_ARGUMENT, "the cache's arrays overlap one another");
    if (own.meets(span_of_rows(qkv, tokens, qkv_stride, (n_heads + 2 * kv) * hd)) || own.meets(span_of_rows(q_out, tokens, q_stride, n_heads * hd)))
        return bad(SGQ_ERR_BAD_ARGUMENT, "the cache overlaps the rows");
    if ((rc = check_device()) != SGQ_OK) return rc;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const int64_t rows = n_heads + 2 * kv;
#define SGQ_STORE(LPR, VEC)                                                                                                                \
    do {                                                                                                                                   \
        const int64_t blocks = ceil_div(rows * LPR, kStoreThreads), threads = ceil_div(ceil_div(rows * LPR, blocks), 32) * 32;             \
        SGQ_CUDA_TRY(launch_kernel(rope_kv_store_int8_kernel<LPR, VEC>, dim3(static_cast<unsigned>(cache->batch * t_new),                  \
                                   static_cast<unsigned>(ceil_div(rows * LPR, threads))), dim3(static_cast<unsigned>(threads)), 0, s,      \
                                   true, qkv, qkv_stride, static_cast<int>(t_new), static_cast<int>(n_heads), static_cast<int>(kv),        \
                                   static_cast<int>(hd), cos_table, sin_table, table_rows, pos, pos_stride, n_new, rope_offset, q_out,     \
                                   q_stride, cache->k_codes, cache->k_scales, cache->v_codes, cache->v_scales, cache->max_seq));           \
    } while (0)
    const bool wide = hd % 16 == 0 && aligned(qkv, 32) && qkv_stride % 8 == 0 && aligned(q_out, 32) && q_stride % 8 == 0 &&
                      aligned(cos_table, 32) && aligned(sin_table, 32);
    if (wide) {
        if (hd <= 32) SGQ_STORE(2, 8);
        else if (hd <= 64) SGQ_STORE(4, 8);
        else if (hd <= 128) SGQ_STORE(8, 8);
        else SGQ_STORE(16, 8);
    } else {
        if (hd <= 32) SGQ_STORE(4, 4);
        else if (hd <= 64) SGQ_STORE(8, 4);
        else if (hd <= 128) SGQ_STORE(16, 4);
        else SGQ_STORE(32, 4);
    }
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
    const int64_t step = kLoadThreads / (cache->head_dim / 8), chunks = ceil_div(rows, step * kLoadRows);
    const int64_t heads = batch * cache->n_kv_heads;
    if (heads > 0x7fffffff / chunks) return bad(SGQ_ERR_BAD_SHAPE, "too many rows for one call");
    const int64_t hd = cache->head_dim, apart = out_max_seq * hd;          // floats between the written rows of two heads
    if (rows_overlap(k_out + out_row0 * hd, apart, rows * hd, v_out + out_row0 * hd, apart, rows * hd, heads))
        return bad(SGQ_ERR_BAD_ARGUMENT, "the outputs overlap");
    const CacheSpans own(cache);
    if (own.meets(span(k_out, heads, out_max_seq, hd, 4)) || own.meets(span(v_out, heads, out_max_seq, hd, 4)))
        return bad(SGQ_ERR_BAD_ARGUMENT, "an output overlaps the cache");
    if ((rc = check_device()) != SGQ_OK) return rc;
    const bool wide = aligned(k_out, 32) && aligned(v_out, 32);
    SGQ_CUDA_TRY(launch_kernel(wide ? kv_load_int8_kernel<true> : kv_load_int8_kernel<false>, dim3(static_cast<unsigned>(heads * chunks), 2), dim3(kLoadThreads), 0,
                               static_cast<cudaStream_t>(stream), true, cache->k_codes, cache->k_scales, cache->v_codes, cache->v_scales,
                               cache->max_seq, static_cast<int>(cache->head_dim), static_cast<int>(rows), static_cast<int>(chunks),
                               static_cast<int>(step), cache->batch * cache->n_kv_heads, k_out, v_out,
                               out_max_seq, out_row0));
    return SGQ_OK;
}

size_t sgqd_attn_decode_int8_workspace_bytes(int64_t batch, int64_t n_heads, int64_t n_kv_heads, int64_t head_dim, int64_t max_seq) {
    return decode_workspace(batch, n_heads, n_kv_heads, head_dim, max_seq, 0);
}

int sgqd_attn_decode_int8(const float* qkv, int64_t qkv_stride, int64_t n_heads, const float* cos_table, const float* sin_table,
                          int64_t table_rows, const int32_t* pos, int64_t pos_stride, const sgqd_cache_int8* cache, float* out, int64_t out_stride,
                          void* prepared_out, size_t prepared_bytes, void* workspace, size_t workspace_bytes, void* stream) {
    return attn_decode(qkv, qkv_stride, n_heads, cos_table, sin_table, table_rows, pos, pos_stride, cache, nullptr, nullptr, out, out_stride,
                       prepared_out, prepared_bytes, workspace, workspace_bytes, static_cast<cudaStream_t>(stream));
}

size_t sgqd_attn_decode_prefix_int8_workspace_bytes(int64_t batch, int64_t n_heads, int64_t n_kv_heads, int64_t head_dim, int64_t max_seq,
                                                    int64_t prefix_max) {
    return prefix_max > 0 ? decode_workspace(batch, n_heads, n_kv_heads, head_dim, max_seq, prefix_max) : 0;
}

int sgqd_attn_decode_prefix_int8(const float* qkv, int64_t qkv_stride, int64_t n_heads, const float* cos_table, const float* sin_table,
                                 int64_t table_rows, const int32_t* pos, int64_t pos_stride, const sgqd_cache_int8* cache,
                                 const sgqd_cache_int8* prefix, const int32_t* prefix_len, float* out, int64_t out_stride, void* prepared_out,
                                 size_t prepared_bytes, void* workspace, size_t workspace_bytes, void* stream) {
    if (!prefix) return bad(SGQ_ERR_NULL_POINTER, "prefix is NULL");
    return attn_decode(qkv, qkv_stride, n_heads, cos_table, sin_table, table_rows, pos, pos_stride, cache, prefix, prefix_len, out, out_stride,
                       prepared_out, prepared_bytes, workspace, workspace_bytes, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
