// What the kernels of the INT8 key/value cache share (kv_int8.cu, kv_int8_prefix.cu): the rotation, the fixed-point query, the
// joining of partial results, the arguments of a decode step.
#pragma once

#include "gemv_prepare.cuh"
#include "sm100_ptx.cuh"

#include "../../include/sgq_decoder.h"

#include <math_constants.h>

namespace sgq {

constexpr int kSms = 148;                     // what the plans count on, whatever the device has

struct CacheView {
    int8_t* kc;
    float* ks;
    int8_t* vc;
    float* vs;
    int64_t max_seq;
};

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
    float* part_ml;                    // partial results of the prefix: [kv head][row][split][2] and [...][HD]
    float* part_o;
    int parts;                         // splits of the prefix, 0: none
    float* flat_ml;                    // partial results of attn_flat_int8_kernel: [slot][NQ][2] and [slot][NQ][HD]
    float* flat_o;
};

#ifdef __CUDACC__

__device__ __forceinline__ int64_t prefix_rows(const DecodeArgs& a) {
    if (!a.prefix_len) return 0;
    const int64_t p = *a.prefix_len;
    return p < 0 ? 0 : (p > a.first.max_seq ? a.first.max_seq : p);
}

// (x1, x2) of a rotary pair, every operation rounded (src/ops.cpp:1737-1738)
__device__ __forceinline__ void rotate_pair(float& x1, float& x2, float c, float s) {
    const float a = __fsub_rn(__fmul_rn(x1, c), __fmul_rn(x2, s));
    x2 = __fadd_rn(__fmul_rn(x2, c), __fmul_rn(x1, s));
    x1 = a;
}

// The exact sum whose digit sums (2: highest; each below 2^21.1) these are, as fp32.  256 d2 + d1 fits an int32.
__device__ __forceinline__ float join_digits(int d2, int d1, int d0) {
    return fmaf(static_cast<float>(d2 * 256 + d1), 256.0f, static_cast<float>(d0));
}
// A softmax weight w as fixed point: rint(w * per), at most kWeightRange, 23 bits in steps of the 1.5 * 2^23 trick, as
// balanced digits (bytes 0 .. 2; see digit_bytes)
constexpr float kWeightRange = 4194000.0f;    // below 2^22, where fp32 behind the added constant is exact to one
__device__ __forceinline__ uint32_t weight_digits(float w, float per) {
    return (__float_as_uint(fmaf(w, per, kMagicF)) + (0x00808080u - static_cast<uint32_t>(kMagicBits))) ^ 0x00808080u;
}
// digit j of four numbers side by side in w_j
__device__ __forceinline__ void gather_digits(const uint32_t (&d)[4], uint32_t& w0, uint32_t& w1, uint32_t& w2) {
    const uint32_t x = __byte_perm(d[0], d[1], 0x5140), y = __byte_perm(d[2], d[3], 0x5140);
    w0 = __byte_perm(x, y, 0x5410);
    w1 = __byte_perm(x, y, 0x7632);
    w2 = __byte_perm(__byte_perm(d[0], d[1], 0x0062), __byte_perm(d[2], d[3], 0x0062), 0x5410);
}
// The reference that weights are taken against follows the maximum only when a score exceeds it by kAhead: weights of up to 2^kAhead.
constexpr float kAhead = 6.0f;
// Outputs are summed before they are divided by the sum of the weights, which are up to 2^6 each: they are carried times 2^-24, so
// that values of any size hold behind 2^18 positions (and of FLT_MAX * 2^18 / n behind n).  What a tile adds is taken as nothing
// where the largest weight times value scale is below 2^-80, with units of sums still in the fp32 range.
constexpr float kValueDown = 0x1p-24f, kVanishing = 0x1p-80f;
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

__device__ __forceinline__ void cp_async_16(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// N = 4 or 8 consecutive floats, aligned to their own size
template <int N>
__device__ __forceinline__ void load_floats(float (&v)[N], const float* p) {
    if constexpr (N == 8)
        asm volatile("ld.global.v8.f32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                     : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7])
                     : "l"(p)
                     : "memory");
    else {
        const float4 x = *reinterpret_cast<const float4*>(p);
        v[0] = x.x; v[1] = x.y; v[2] = x.z; v[3] = x.w;
    }
}
template <int N>
__device__ __forceinline__ void store_floats(float* p, const float (&v)[N]) {
    if constexpr (N == 8)
        asm volatile("st.global.v8.f32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]),
                     "f"(v[6]), "f"(v[7])
                     : "memory");
    else *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
}

// A lane's HD / 32 consecutive values of a row
template <int N>
__device__ __forceinline__ void load_values_of(const float* from, float (&v)[N]) {
    static_assert(N == 2 || N == 4, "head sizes of 64 and 128");
    if constexpr (N == 4) {
        const float4 x = *reinterpret_cast<const float4*>(from);
        v[0] = x.x; v[1] = x.y; v[2] = x.z; v[3] = x.w;
    } else {
        const float2 x = *reinterpret_cast<const float2*>(from);
        v[0] = x.x; v[1] = x.y;
    }
}

// Joins partial results (maximum, sum, value) of one output value
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

// One warp rotates a row of HD values, VEC consecutive per lane: lane l < 16 holds the first ones of the pairs of lane l + 16.  c, s:
// the cosines and sines of pairs (lane & 15) VEC ..
template <int HD>
__device__ __forceinline__ void rotate_values(float (&v)[HD / 32], const float (&c)[HD / 32], const float (&s)[HD / 32], int lane) {
#pragma unroll
    for (int j = 0; j < HD / 32; ++j) {
        const float other = __shfl_xor_sync(0xffffffffu, v[j], 16);
        float x1 = lane < 16 ? v[j] : other, x2 = lane < 16 ? other : v[j];
        rotate_pair(x1, x2, c[j], s[j]);
        v[j] = lane < 16 ? x1 : x2;
    }
}
template <int HD>
__device__ __forceinline__ void rotate_row(float (&v)[HD / 32], const float* cos_row, const float* sin_row, int lane) {
    float c[HD / 32], s[HD / 32];
#pragma unroll
    for (int j = 0; j < HD / 32; ++j) {
        c[j] = cos_row[(lane & 15) * (HD / 32) + j];
        s[j] = sin_row[(lane & 15) * (HD / 32) + j];
    }
    rotate_values<HD>(v, c, s, lane);
}

// What a rotated query is multiplied with on the way to its digits, from the bits of its largest |value|, and the unit of its
// scores, which carries 1/sqrt(HD) and log2(e).  A NaN or an infinity in the query makes the unit NaN and the digits zero: every
// score is NaN.
//
// A score is (digit sum * key scale) * unit, in this order in every kernel, so that equal rows have equal scores whichever kernel
// reads them.  Digit sums reach 2^37, key scales 2^121 and units without kKeyDown 2^102: the key scale is taken times 2^-31 and the
// unit times 2^31, so that no factor overflows where the score is of ordinary size (queries of up to 2^122, keys of any size).
constexpr float kKeyDown = 0x1p-31f;
// A query below 2^-64 is lifted by 2^64 on the way, so that neither factor leaves the fp32 range however small it is.
__device__ __forceinline__ float query_lift(uint32_t top) { return top < 0x1F800000u ? 0x1p64f : 1.0f; }
__device__ __forceinline__ float query_scale(uint32_t top) {                 // of the lifted values
    return top == 0u || top >= 0x7F800000u ? 0.f : __fdiv_rn(kDigitRange, __uint_as_float(top) * query_lift(top));
}
template <int HD>
__device__ __forceinline__ float query_unit(uint32_t top) {
    if (top - 1u >= 0x7F800000u - 1u) return top == 0u ? 0.f : CUDART_NAN_F;      // rows that a block does not have: no division of zero (0.2 us)
    const float per = rsqrtf(static_cast<float>(HD)) * 1.4426950408889634f * (1.0f / kKeyDown);
    return __fmul_rn(__fdiv_rn(__uint_as_float(top) * query_lift(top), kDigitRange), top < 0x1F800000u ? per * 0x1p-64f : per);
}
template <int HD>
__device__ __forceinline__ uint32_t largest_bits(const float (&v)[HD / 32]) {
    uint32_t top = 0;
#pragma unroll
    for (int j = 0; j < HD / 32; ++j) top = max(top, __float_as_uint(v[j]) & 0x7FFFFFFFu);
    return __reduce_max_sync(0xffffffffu, top);
}
// A query's digits from its lifted values, `per` being its query_scale (at(j, d): where digit j of value d goes)
template <int HD, typename At>
__device__ __forceinline__ void put_digits(const float (&v)[HD / 32], float per, At at, int lane) {
    constexpr int VEC = HD / 32;
    uint32_t d[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) d[j] = per != 0.f ? digit_bytes(__float2int_rn(__fmul_rn(v[j], per))) : 0u;
#pragma unroll
    for (int j = 0; j < 3; ++j) {
        if constexpr (VEC == 4)
            *reinterpret_cast<uint32_t*>(at(j, lane * 4)) = gather_byte(d[0], d[1], d[2], d[3], j);
        else
            *reinterpret_cast<uint16_t*>(at(j, lane * 2)) = static_cast<uint16_t>(__byte_perm(d[0], d[1], 0x0040 + 0x11 * j));
    }
}
// The rotated query as digits and its unit
template <int HD, typename At>
__device__ __forceinline__ void query_digits(const float (&v)[HD / 32], At at, float* unit, int lane) {
    const uint32_t top = largest_bits<HD>(v);
    float x[HD / 32];
#pragma unroll
    for (int j = 0; j < HD / 32; ++j) x[j] = v[j] * query_lift(top);
    put_digits<HD>(x, query_scale(top), at, lane);
    if (lane == 0) *unit = query_unit<HD>(top);
}

#endif  // __CUDACC__

// kv_int8_prefix.cu: partial results of up to 128 query rows per block to the prefix on the tcgen05 tensor cores
constexpr int kPrefixTcRows = 128, kPrefixTcTile = 128;
int launch_prefix_tc(const DecodeArgs& a, int head_dim, int splits, int blocks, cudaStream_t s);

}  // namespace sgq
