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

#include <math_constants.h>

namespace sgq {

namespace {

constexpr int kMaxHeadDim = 256;

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
struct CacheView {
    int8_t* kc;
    float* ks;
    int8_t* vc;
    float* vs;
    int64_t max_seq;
};

// One block per (sequence, kv head).  The block appends the new token's row, then its warps walk the positions (the prefix's,
// then the sequence's own) with a running maximum and sum, one query head after the other.
constexpr int kSimpleWarps = 8;
template <int HD>
__global__ void __launch_bounds__(kSimpleWarps * 32) attn_decode_int8_kernel(const float* __restrict__ qkv, int64_t qkv_stride, int n_heads, int n_kv,
                                                                             const float* __restrict__ cos_t, const float* __restrict__ sin_t,
                                                                             const int32_t* __restrict__ pos_p, int64_t pos_stride, CacheView own,
                                                                             CacheView first, const int32_t* __restrict__ prefix_len,
                                                                             float* __restrict__ out, int64_t out_stride) {
    constexpr int VEC = HD / 32;
    __shared__ float sm_m[kSimpleWarps], sm_l[kSimpleWarps], sm_acc[kSimpleWarps][HD];
    pdl_launch_dependents();
    pdl_wait();
    const int b = blockIdx.x / n_kv, hk = blockIdx.x - b * n_kv, G = n_heads / n_kv;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int64_t pos = pos_p[b * pos_stride];
    const bool live = pos >= 0 && pos < own.max_seq;
    int64_t P = prefix_len ? *prefix_len : 0;
    P = P < 0 ? 0 : (prefix_len && P > first.max_seq ? first.max_seq : P);
    const float* row = qkv + b * qkv_stride + lane * VEC;
    const int64_t base = (static_cast<int64_t>(b) * n_kv + hk) * own.max_seq;
    float* orow = out + b * out_stride + static_cast<int64_t>(hk) * G * HD;
    if (!live) {
        for (int i = threadIdx.x; i < G * HD; i += kSimpleWarps * 32) orow[i] = 0.f;
        return;
    }
    auto rotated = [&](int64_t at, float (&v)[VEC], bool turn) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) v[j] = row[at + j];
        if (!turn) return;
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            const float other = __shfl_xor_sync(0xffffffffu, v[j], 16);
            const float c = cos_t[(P + pos) * (HD / 2) + (lane & 15) * VEC + j], s = sin_t[(P + pos) * (HD / 2) + (lane & 15) * VEC + j];
            float x1 = lane < 16 ? v[j] : other, x2 = lane < 16 ? other : v[j];
            rotate_pair(x1, x2, c, s);
            v[j] = lane < 16 ? x1 : x2;
        }
    };
    if (warp < 2) {                       // warp 0 appends the key, warp 1 the value
        float v[VEC];
        rotated(static_cast<int64_t>(n_heads + (warp ? n_kv : 0) + hk) * HD, v, warp == 0);
        float top = 1e-8f;
#pragma unroll
        for (int j = 0; j < VEC; ++j) top = absmax_step(top, v[j]);
        top = warp_max(top);
        const float inv = __fdiv_rn(127.0f, top);
        int8_t* codes = (warp ? own.vc : own.kc) + (base + pos) * HD + lane * VEC;
#pragma unroll
        for (int j = 0; j < VEC; ++j) codes[j] = static_cast<int8_t>(quantize_code<127, -127>(v[j], inv));
        if (lane == 0) (warp ? own.vs : own.ks)[base + pos] = __fdiv_rn(top, 127.0f);
    }
    __syncthreads();
    for (int g = 0; g < G; ++g) {
        float q[VEC], acc[VEC];
        rotated(static_cast<int64_t>(hk * G + g) * HD, q, true);
#pragma unroll
        for (int j = 0; j < VEC; ++j) { q[j] *= rsqrtf(static_cast<float>(HD)); acc[j] = 0.f; }
        float m = -CUDART_INF_F, l = 0.f;
        for (int64_t t = warp; t < P + pos + 1; t += kSimpleWarps) {
            const CacheView& c = t < P ? first : own;
            const int64_t at = t < P ? hk * first.max_seq + t : base + (t - P);
            float d = 0.f;
#pragma unroll
            for (int j = 0; j < VEC; ++j) d = fmaf(q[j], static_cast<float>(c.kc[at * HD + lane * VEC + j]), d);
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) d += __shfl_xor_sync(0xffffffffu, d, o);
            const float ksc = c.ks[at], vsc = c.vs[at];
            const float s = fmaf(d, ksc, ksc - ksc);                 // NaN for a row whose scale is not finite
            const float mn = fmaxf(m, s);
            const float corr = m == -CUDART_INF_F ? 0.f : expf(m - mn);
            const float p = s == -CUDART_INF_F ? 0.f : expf(s - mn);
            l = fmaf(l, corr, p + (vsc - vsc));
#pragma unroll
            for (int j = 0; j < VEC; ++j) acc[j] = fmaf(acc[j], corr, p * vsc * static_cast<float>(c.vc[at * HD + lane * VEC + j]));
            m = mn;
        }
        if (lane == 0) { sm_m[warp] = m; sm_l[warp] = l; }
#pragma unroll
        for (int j = 0; j < VEC; ++j) sm_acc[warp][lane * VEC + j] = acc[j];
        __syncthreads();
        if (threadIdx.x < HD) {
            float M = -CUDART_INF_F, L = 0.f, A = 0.f;
            for (int w = 0; w < kSimpleWarps; ++w) M = fmaxf(M, sm_m[w]);
            for (int w = 0; w < kSimpleWarps; ++w) {
                const float wgt = sm_m[w] == -CUDART_INF_F ? 0.f : expf(sm_m[w] - M);
                L += sm_l[w] * wgt;
                A += sm_acc[w][threadIdx.x] * wgt;
            }
            orow[g * HD + threadIdx.x] = L == 0.f ? 0.f : A / L;
        }
        __syncthreads();
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

int attn_decode(const float* qkv, int64_t qkv_stride, int64_t n_heads, const float* cos_table, const float* sin_table, int64_t table_rows,
                const int32_t* pos, int64_t pos_stride, const sgqd_cache_int8* cache, const sgqd_cache_int8* prefix, const int32_t* prefix_len, float* out,
                int64_t out_stride, void* prepared_out, size_t prepared_bytes, cudaStream_t s) {
    int rc = check_cache(cache);
    if (rc != SGQ_OK) return rc;
    const int64_t hd = cache->head_dim, kv = cache->n_kv_heads;
    if (hd != 64 && hd != 128) return bad(SGQ_ERR_UNSUPPORTED, "head_dim must be 64 or 128");
    if (n_heads <= 0 || n_heads > 65535 || n_heads % kv) return bad(SGQ_ERR_BAD_SHAPE, "n_heads must be a multiple of the cache's heads");
    if (qkv_stride < (n_heads + 2 * kv) * hd || out_stride < n_heads * hd) return bad(SGQ_ERR_BAD_SHAPE, "row stride too small");
    if (pos_stride != 0 && pos_stride != 1) return bad(SGQ_ERR_BAD_ARGUMENT, "pos_stride must be 0 or 1");
    if (prefix) {
        if ((rc = check_cache(prefix)) != SGQ_OK) return rc;
        if (prefix->batch != 1 || prefix->n_kv_heads != kv || prefix->head_dim != hd)
            return bad(SGQ_ERR_BAD_SHAPE, "the prefix is one sequence with the cache's heads");
    }
    if (table_rows < cache->max_seq + (prefix ? prefix->max_seq : 0)) return bad(SGQ_ERR_BAD_SHAPE, "the cos / sin tables are too short");
    if (cache->batch == 0) return SGQ_OK;
    if (!qkv || !cos_table || !sin_table || !pos || !out || (prefix && !prefix_len)) return bad(SGQ_ERR_NULL_POINTER, "NULL argument");
    if ((rc = check_cache_pointers(cache)) != SGQ_OK || (prefix && (rc = check_cache_pointers(prefix)) != SGQ_OK)) return rc;
    if (!aligned(qkv, 16) || (qkv_stride & 3) || !aligned(cos_table, 16) || !aligned(sin_table, 16))
        return bad(SGQ_ERR_ALIGNMENT, "qkv rows and tables must be 16-byte aligned");
    PreparedLayout L = {};
    if ((rc = check_prepared(prepared_out, prepared_bytes, cache->batch, n_heads * hd, &L)) != SGQ_OK) return rc;
    if ((rc = check_device()) != SGQ_OK) return rc;
    const CacheView own = view(cache), first = prefix ? view(prefix) : CacheView{};
    const dim3 grid(static_cast<unsigned>(cache->batch * kv));
    if (hd == 128)
        SGQ_CUDA_TRY(launch_kernel(attn_decode_int8_kernel<128>, grid, dim3(kSimpleWarps * 32), 0, s, true, qkv, qkv_stride, static_cast<int>(n_heads),
                                   static_cast<int>(kv), cos_table, sin_table, pos, pos_stride, own, first, prefix_len, out, out_stride));
    else
        SGQ_CUDA_TRY(launch_kernel(attn_decode_int8_kernel<64>, grid, dim3(kSimpleWarps * 32), 0, s, true, qkv, qkv_stride, static_cast<int>(n_heads),
                                   static_cast<int>(kv), cos_table, sin_table, pos, pos_stride, own, first, prefix_len, out, out_stride));
    if (prepared_out) return sgq_prepare_x(out, cache->batch, n_heads * hd, prepared_out, prepared_bytes, s);
    return SGQ_OK;
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
                       prepared_bytes, static_cast<cudaStream_t>(stream));
}

size_t sgqd_attn_decode_prefix_int8_workspace_bytes(int64_t batch, int64_t n_heads, int64_t n_kv_heads, int64_t head_dim, int64_t prefix_max) {
    (void)batch; (void)n_heads; (void)n_kv_heads; (void)head_dim; (void)prefix_max;
    return 0;
}

int sgqd_attn_decode_prefix_int8(const float* qkv, int64_t qkv_stride, int64_t n_heads, const float* cos_table, const float* sin_table,
                                 int64_t table_rows, const int32_t* pos, int64_t pos_stride, const sgqd_cache_int8* cache, const sgqd_cache_int8* prefix,
                                 const int32_t* prefix_len, float* out, int64_t out_stride, void* prepared_out, size_t prepared_bytes,
                                 void* workspace, size_t workspace_bytes, void* stream) {
    (void)workspace; (void)workspace_bytes;
    if (!prefix) return bad(SGQ_ERR_NULL_POINTER, "prefix is NULL");
    return attn_decode(qkv, qkv_stride, n_heads, cos_table, sin_table, table_rows, pos, pos_stride, cache, prefix, prefix_len, out, out_stride, prepared_out,
                       prepared_bytes, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
