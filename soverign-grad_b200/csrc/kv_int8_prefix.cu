// Partial attention of many query rows to a shared prefix in the INT8 cache, on the tcgen05 tensor cores.
//
// Scores as in kv_int8.cu: codes as they lie in memory, queries as fixed point split into three balanced base-256 digits, exact
// integer products.  With 33 query rows and more per kv head they are worth the large MMA: a block takes 128 rows (sequence,
// query of the group) and walks its part of the prefix in tiles of 128 positions,
//   S_j = Q_j K^T      kind::i8, 128 x 128 x HD for each digit plane j, into columns 128 j of tensor memory
//   softmax            a thread holds a quarter of a row: 32 scores; the quarters exchange their maxima through shared memory
//   O = (P_lo + P_hi) V     kind::f16, 128 x HD x 128 twice, into columns 384 ..: codes are exact in 16-bit floats, a weight is the
//                      sum of two (22 bits), relative to the largest of the tile and row
// and adds O into fp32 registers once per tile: 16 additions in the tensor core between two roundings that are known.  (The
// weights as digit planes, as in kv_int8.cu, need 384 columns for O and five more instructions per weight: 52 us for 32
// sequences x 8 kv heads x 4 queries behind 16384 positions, decode included, where this form takes 45.  Queries as 16-bit floats
// would save as much again, but a score then carries the rounding of the tensor core's sums, 16 of them, where an exact one
// has one.)  Keys are copied as they are (K-major, 128-byte-swizzled rows), values are widened on the way and read MN-major, so
// nothing is transposed.  The next tile's scores run while a tile's weights are made, its outputs while the next scores are read.
// What bounds it: 3.1 us a tile (6000 cycles, of which the MMAs take 1800 behind the softmax), sixteen warps in step, so that exponentials,
// conversions and shared memory (which the MMAs' operands alone hold for 1800 cycles) take turns; and what stands beside the tiles.  32
// sequences x 8 kv heads x 4 queries with room for 16384 positions, decode included: 23.4 / 26.6 / 32.5 / 45.4 us with 1 / 2 / 4 / 8 tiles a
// CTA, so 20 us are start, digits (each split makes those of its 128 rows again), partial results and the sequences' own rows.
// Measured without effect: products issued by several warps or a few at a time, one more warp to issue them (96 registers are
// too few), magic-number conversions of the digits; packed fp32 arithmetic took 44.2 us to 43.3, the weights' unit by row 43.3 to 45.
#include <cuda_fp16.h>

#include <type_traits>

#include "kv_int8.cuh"

namespace sgq {

__device__ uint32_t g_status_kv = 0;

cudaError_t read_status_kv(uint32_t* v, bool clear) {
    cudaError_t e = cudaMemcpyFromSymbol(v, g_status_kv, sizeof(uint32_t));
    if (e == cudaSuccess && clear && *v != 0) {
        const uint32_t zero = 0;
        e = cudaMemcpyToSymbol(g_status_kv, &zero, sizeof(zero));
    }
    return e;
}

namespace {

constexpr int kThreads = 512, kRows = kPrefixTcRows, kTile = kPrefixTcTile;
constexpr int kPlane = 128 * 128;              // an operand: 128 rows of 128 bytes
constexpr int kTmemCols = 512;
constexpr int kWeightBits = 13;                // a row's weights reach about 2^13 before they are split: below the largest 16-bit float
// Up to this reference a score may be a product that is not rounded: what the rounding would change, 2^-14, is what a score of an
// fp32 evaluation is off by.  Beyond, the row's largest score has to be the reference exactly, and scores that are equal stay equal.
constexpr float kFar = 1024.0f;

template <int HD>
struct Shape {
    static constexpr int kVBytes = kTile * HD * 2;                    // values in 16 bits: [half of the positions][64 values][64 positions]
    static constexpr int kPPlane = kRows * kTile * 2;                 // weights in 16 bits: [half of the positions][row][64 positions]
    static constexpr int kQ = 0, kK = kQ + 3 * kPlane, kV = kK + 2 * kPlane, kP = kV + 2 * kVBytes, kSmall = kP + 2 * kPPlane;
    static constexpr int kFloats = 128 + 6 * kTile + 8 * kRows + 8;  // units, scales of keys, values, log2 of these (twice), maxima, tiles' value units
    static constexpr int kBars = kSmall + kFloats * 4, kBytes = kBars + 32 + 1024;   // 1024: alignment of the base
    static_assert(kBytes <= 227 * 1024 && 2 * kPPlane >= kRows * HD * 4, "shared memory");
};

// 16-byte chunk c of row r of a 128-byte-swizzled operand
__device__ __forceinline__ int swizzled(int r, int c) { return r * 128 + ((c ^ (r & 7)) << 4); }

// Two fp32 operations in one instruction
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;"
        : "=l"(reinterpret_cast<unsigned long long&>(d))
        : "l"(reinterpret_cast<unsigned long long&>(a)), "l"(reinterpret_cast<unsigned long long&>(b)), "l"(reinterpret_cast<unsigned long long&>(c)));
    return d;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
    float2 d;
    asm("mul.rn.f32x2 %0, %1, %2;"
        : "=l"(reinterpret_cast<unsigned long long&>(d))
        : "l"(reinterpret_cast<unsigned long long&>(a)), "l"(reinterpret_cast<unsigned long long&>(b)));
    return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    float2 d;
    asm("add.rn.f32x2 %0, %1, %2;"
        : "=l"(reinterpret_cast<unsigned long long&>(d))
        : "l"(reinterpret_cast<unsigned long long&>(a)), "l"(reinterpret_cast<unsigned long long&>(b)));
    return d;
}
__device__ __forceinline__ float2 both(float x) { return make_float2(x, x); }
// join_digits of two
__device__ __forceinline__ float2 join_two(const int* d2, const int* d1, const int* d0) {
    return fma2(make_float2(static_cast<float>(d2[0] * 256 + d1[0]), static_cast<float>(d2[1] * 256 + d1[1])), both(256.f),
                make_float2(static_cast<float>(d0[0]), static_cast<float>(d0[1])));
}

// Codes 2 H and 2 H + 1 of four as 16-bit floats: 1152 + code is read off the bits of 1024 + (code + 128)
template <int H>
__device__ __forceinline__ uint32_t half2_of(uint32_t codes) {
    const uint32_t x = __byte_perm(codes ^ 0x80808080u, 0x64646464u, H == 0 ? 0x4140 : 0x4342);
    const __half2 y = __hsub2(*reinterpret_cast<const __half2*>(&x), __half2half2(__ushort_as_half(0x6480)));
    return *reinterpret_cast<const uint32_t*>(&y);
}
// Two weights as sums of two 16-bit floats (22 bits)
__device__ __forceinline__ void split_weights(float2 w, uint32_t& hi, uint32_t& lo) {
    const __half2 x = __float22half2_rn(w), y = __float22half2_rn(fma2(__half22float2(x), both(-1.f), w));
    hi = *reinterpret_cast<const uint32_t*>(&x);
    lo = *reinterpret_cast<const uint32_t*>(&y);
}

// grid (kv heads, splits of the prefix, blocks of 128 rows)
template <int HD>
__global__ void __launch_bounds__(kThreads, 1) attn_prefix_tc_int8_kernel(const DecodeArgs a) {
    using S = Shape<HD>;
    constexpr int VEC = HD / 32, KEYS = kTile / 4, COLS = HD / 4;         // a thread's part of a row: positions, output columns
    extern __shared__ uint8_t raw[];
    uint8_t* sm = raw + ((1024u - (smem_u32(raw) & 1023u)) & 1023u);
    float* sm_unit = reinterpret_cast<float*>(sm + S::kSmall);
    float* sm_ks = sm_unit + 128;                                     // [2][kTile], times kKeyDown
    float* sm_vs = sm_ks + 2 * kTile;                                 // [2][kTile], relative to the tile's largest
    float* sm_lv = sm_vs + 2 * kTile;                                 // [2][kTile]: log2 of these
    float2* sm_top = reinterpret_cast<float2*>(sm_lv + 2 * kTile);    // [4][128]: a quarter's largest score, and score + sm_lv
    float* sm_vtop = reinterpret_cast<float*>(sm_top + 4 * kRows);    // [4]: the largest of 32 value scales
    float* sm_vunit = sm_vtop + 4;                                    // [4]: what a tile's outputs are scaled by, of tile i in i % 4
    uint64_t* bars = reinterpret_cast<uint64_t*>(sm + S::kBars);      // scores done, outputs done
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 2);
    volatile uint32_t* gave_up = tmem_slot + 1;                       // a wait ran out: everyone leaves at the next tile
    const int tid = threadIdx.x, warp = warp_index(), lane = tid & 31;
    if (warp == 0) {
        tmem_alloc(tmem_slot, kTmemCols);
        tmem_relinquish();
    }
    if (tid == 0) {
        mbar_init(&bars[0], 1);
        mbar_init(&bars[1], 1);
        mbar_fence_init();
        *gave_up = 0;
    }
    pdl_wait();
    pdl_launch_dependents();                                          // behind the wait: see attn_decode_int8_kernel
    const int hk = blockIdx.x, split = blockIdx.y, splits = gridDim.y, G = a.n_heads / a.n_kv;
    const int R = a.batch * G, r0 = blockIdx.z * kRows;
    const uint32_t sm_u = smem_u32(sm);
    // the raw rows of this warp's queries are asked for before anything is known of the prefix
    constexpr int QR = kRows / (kThreads / 32);
    float* rows = reinterpret_cast<float*>(sm + S::kP) + warp * QR * HD;
    float* turns = reinterpret_cast<float*>(sm + S::kV) + warp * QR * HD;      // HD / 2 cosines and HD / 2 sines of each
    int at = -1;                                                      // lane i: position of the warp's row i, -1: no such row, or idle
    {
        long long from = 0;
        if (lane < QR) {
            const int r = min(r0 + warp * QR + lane, R - 1), b = r / G;
            from = b * a.qkv_stride + static_cast<int64_t>(hk * G + r - b * G) * HD;
            const int64_t pos = r0 + warp * QR + lane < R ? a.pos[b * a.pos_stride] : -1;
            at = pos >= 0 && pos < a.own.max_seq ? static_cast<int>(pos) : -1;
        }
#pragma unroll
        for (int i = 0; i < QR; ++i) {
            const long long f = __shfl_sync(0xffffffffu, from, i);
            if (lane < HD / 4) cp_async_16(smem_u32(rows + i * HD + lane * 4), a.qkv + f + lane * 4);
        }
    }
    const int n = static_cast<int>(prefix_rows(a));
    const int chunk = ((n + splits - 1) / splits + kTile - 1) / kTile * kTile;
    const int t0 = static_cast<int>(min(static_cast<int64_t>(split) * chunk, static_cast<int64_t>(n)));
    const int t1 = static_cast<int>(min(static_cast<int64_t>(t0) + chunk, static_cast<int64_t>(n)));
    const int64_t base = static_cast<int64_t>(hk) * a.first.max_seq;
    const int8_t* kc = a.first.kc + base * HD;
    const int8_t* vc = a.first.vc + base * HD;
    const float* scales = (tid < kTile ? a.first.ks : a.first.vs) + base;      // threads 0 .. 255 bring the scales
    {
        const int turn = at >= 0 ? n + at : 0, x = lane & 15;
#pragma unroll
        for (int i = 0; i < QR; ++i) {
            const int64_t from = static_cast<int64_t>(__shfl_sync(0xffffffffu, turn, i)) * (HD / 2);
            if (x < HD / 8) cp_async_16(smem_u32(turns + i * HD + (lane >> 4) * (HD / 2) + x * 4), (lane < 16 ? a.cos_t : a.sin_t) + from + x * 4);
        }
    }
    // A group of their own: a CTA without a tile (t0 == t1) commits no other, and a wait covers committed copies alone.
    cp_async_commit();

    auto request_keys = [&](int slot, int t) {
        constexpr int CH = HD / 16;
#pragma unroll
        for (int u = 0; u < kTile * CH / kThreads; ++u) {
            const int x = tid + u * kThreads, r = x / CH, c = x % CH;
            cp_async_16(sm_u + S::kK + slot * kPlane + swizzled(r, c), kc + static_cast<int64_t>(t) * HD + min(r, t1 - 1 - t) * HD + c * 16);
        }
        cp_async_commit();
    };
    // values: 8 codes of a row per load, which are a 16-byte chunk of the operand
    constexpr int VCH = HD / 8, VN = kTile * VCH / kThreads;
    uint2 vr[VN];
    float scale = 0.f;
    auto load_values = [&](int t) {
        const int8_t* from = vc + static_cast<int64_t>(t) * HD;
        const int last = t1 - 1 - t;
#pragma unroll
        for (int u = 0; u < VN; ++u) {
            const int x = tid + u * kThreads;
            vr[u] = *reinterpret_cast<const uint2*>(from + min(x / VCH, last) * HD + x % VCH * 8);
        }
        if (tid < 2 * kTile) scale = scales[t + min(tid & (kTile - 1), last)];
    };
    auto store_values = [&](int i_tile, int left) {                  // vr and scale, of a tile with `left` positions
        const int slot = i_tile & 1;
#pragma unroll
        for (int u = 0; u < VN; ++u) {
            const int x = tid + u * kThreads, r = x / VCH, c = x % VCH;
            *reinterpret_cast<uint4*>(sm + S::kV + slot * S::kVBytes + (r >> 6) * (HD * 128) + (c >> 3) * 8192 + swizzled(r & 63, c & 7)) =
                make_uint4(half2_of<0>(vr[u].x), half2_of<1>(vr[u].x), half2_of<0>(vr[u].y), half2_of<1>(vr[u].y));
        }
        // a scale that is not finite counts as NaN; positions that do not exist weigh nothing
        if (tid < kTile) sm_ks[slot * kTile + tid] = fmaf(scale, kKeyDown, scale - scale);
        else if (tid < 2 * kTile) {
            const int i = tid - kTile;
            const bool finite = scale - scale == 0.f;
            const uint32_t of_warp = __reduce_max_sync(0xffffffffu, finite && i < left ? __float_as_uint(fabsf(scale)) : 0u);
            if (lane == 0) sm_vtop[i >> 5] = __uint_as_float(of_warp);
            named_barrier_sync(5, kTile);
            const float top = fmaxf(fmaxf(sm_vtop[0], sm_vtop[1]), fmaxf(sm_vtop[2], sm_vtop[3]));
            const float per = top < 1e-30f ? 0.f : __fdiv_rn(1.0f, top);
            const float v = i < left && finite ? scale * per : 0.f;
            sm_vs[slot * kTile + i] = i < left && !finite ? CUDART_NAN_F : v;
            sm_lv[slot * kTile + i] = __log2f(fabsf(v));              // -inf where nothing is added
            if (i == 0) sm_vunit[i_tile & 3] = top * kValueDown;
        }
    };
    if (t0 < t1) {
        request_keys(0, t0);
        load_values(t0);
    }
    // Queries: every warp turns eight raw rows, which lie where the weights will, with cosines and sines where the values will, into
    // digits, four at a time.  (All unrolled with everything in registers this took 12000 cycles, most of them for code.)
    {
        cp_async_wait<0>();
        __syncwarp();
        uint32_t top = 0;                                             // lane i: the largest of row i
#pragma unroll 1
        for (int i0 = 0; i0 < QR; i0 += 4) {
#pragma unroll
            for (int i = i0; i < i0 + 4; ++i) {
                float q[VEC], co[VEC], si[VEC];
                load_values_of(rows + i * HD + lane * VEC, q);
                load_values_of(turns + i * HD + (lane & 15) * VEC, co);
                load_values_of(turns + i * HD + HD / 2 + (lane & 15) * VEC, si);
                rotate_values<HD>(q, co, si, lane);
                if (__shfl_sync(0xffffffffu, at, i) < 0) {
#pragma unroll
                    for (int j = 0; j < VEC; ++j) q[j] = 0.f;
                }
                const uint32_t largest = largest_bits<HD>(q);
                if (lane == i) top = largest;
#pragma unroll
                for (int j = 0; j < VEC; ++j) rows[i * HD + lane * VEC + j] = q[j] * query_lift(largest);
            }
        }
        const float per = query_scale(top);
        if (lane < QR) sm_unit[warp * QR + lane] = query_unit<HD>(top);
#pragma unroll 1
        for (int i0 = 0; i0 < QR; i0 += 4) {
#pragma unroll
            for (int i = i0; i < i0 + 4; ++i) {
                const int r = warp * QR + i;
                float q[VEC];
                load_values_of(rows + i * HD + lane * VEC, q);
                put_digits<HD>(q, __shfl_sync(0xffffffffu, per, i), [&](int j, int d) { return sm + S::kQ + j * kPlane + swizzled(r, d >> 4) + (d & 15); }, lane);
            }
        }
    }
    __syncthreads();                                                  // the cosines and sines have been read
    if (t0 < t1) {
        store_values(0, t1 - t0);
        if (t0 + kTile < t1) {
            request_keys(1, t0 + kTile);
            load_values(t0 + kTile);
        }
    }
    fence_proxy_async_smem();
    tcgen05_fence_before();
    __syncthreads();
    tcgen05_fence_after();
    const uint32_t tmem = *tmem_slot;
    const uint64_t qd = umma_desc_sw128(sm_u + S::kQ), kd = umma_desc_sw128(sm_u + S::kK), vd = umma_desc_sw128_mn(sm_u + S::kV),
                   pd = umma_desc_sw128(sm_u + S::kP);
    const int row = (warp & 3) * 32 + lane, h = warp >> 2;            // this thread: quarter h of the row
    const uint32_t tmem_row = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16);
    const float qu = sm_unit[row];
    float m = -CUDART_INF_F, unit = 0.f;                              // unit: of the last tile's weights
    float2 l2 = both(0.f), o[COLS / 2];
#pragma unroll
    for (int d = 0; d < COLS / 2; ++d) o[d] = both(0.f);
    // Columns: scores of digit j at 128 j, outputs at 384.
    auto multiply_keys = [&](int slot) {                              // by one thread
        const uint32_t idesc = umma_idesc(2u, 1u, kRows, kTile);
#pragma unroll
        for (int j = 0; j < 3; ++j)
#pragma unroll
            for (int k = 0; k < HD / 32; ++k)
                tcgen05_mma_i8(tmem + 128 * j, qd + j * (kPlane >> 4) + 2 * k, kd + slot * (kPlane >> 4) + 2 * k, idesc, k != 0 ? 1u : 0u);
        tcgen05_commit(&bars[0]);
    };
    auto multiply_values = [&](int slot) {                            // by one thread; the smaller parts of the weights first
        const uint32_t idesc = umma_idesc(1u, 0u, kRows, HD) | kIdescBMajorMN;
#pragma unroll
        for (int j = 1; j >= 0; --j)
#pragma unroll
            for (int k = 0; k < kTile / 16; ++k)
                tcgen05_mma_f16(tmem + 384, pd + (j * S::kPPlane + (k >> 2) * (kRows * 128) + (k & 3) * 32 >> 4),
                                vd + (slot * S::kVBytes + (k >> 2) * (HD * 128) + (k & 3) * 2048 >> 4), idesc, j != 1 || k != 0 ? 1u : 0u);
        tcgen05_commit(&bars[1]);
    };
    auto add_outputs = [&](int i_tile) {
        tcgen05_fence_after();
        const float vunit = sm_vunit[i_tile & 3] * unit;
#pragma unroll
        for (int q = 0; q < COLS / 16; ++q) {
            int s0[16];
            tmem_ld_32x32b_x16(tmem_row + 384 + COLS * h + 16 * q, s0);
            tmem_ld_wait();
#pragma unroll
            for (int x = 0; x < 16; x += 2)
                o[8 * q + x / 2] = fma2(make_float2(__int_as_float(s0[x]), __int_as_float(s0[x + 1])), both(vunit), o[8 * q + x / 2]);
        }
    };
    bool fine = true;
    int i_tile = 0;                                                   // tiles alternate between the two buffers of everything
    if (t0 < t1 && warp == 0 && elect_one()) multiply_keys(0);
    __syncwarp();
    for (int t = t0; t < t1; t += kTile, ++i_tile) {
        const int left = t1 - t, slot = i_tile & 1;
        // scores of a quarter of the positions, without the query's unit
        fine = mbar_wait(&bars[0], slot) && fine;
        tcgen05_fence_after();
        float2 c[KEYS / 2];
        float top = -CUDART_INF_F;
#pragma unroll
        for (int q = 0; q < KEYS / 8; ++q) {                          // (16 columns at a time spill: 44.2 us where 8 take 43.2)
            int s2[8], s1[8], s0[8];
            tmem_ld_32x32b_x8(tmem_row + KEYS * h + 8 * q, s0);
            tmem_ld_32x32b_x8(tmem_row + 128 + KEYS * h + 8 * q, s1);
            tmem_ld_32x32b_x8(tmem_row + 256 + KEYS * h + 8 * q, s2);
            tmem_ld_wait();
#pragma unroll
            for (int x = 0; x < 8; x += 4) {
                const float4 k4 = *reinterpret_cast<const float4*>(sm_ks + slot * kTile + KEYS * h + 8 * q + x);
                c[4 * q + x / 2] = mul2(join_two(&s2[x], &s1[x], &s0[x]), make_float2(k4.x, k4.y));
                c[4 * q + x / 2 + 1] = mul2(join_two(&s2[x + 2], &s1[x + 2], &s0[x + 2]), make_float2(k4.z, k4.w));
            }
        }
        if (left < kTile) {
#pragma unroll
            for (int x = 0; x < KEYS; x += 2) {
                if (KEYS * h + x >= left) c[x / 2].x = -CUDART_INF_F;
                if (KEYS * h + x + 1 >= left) c[x / 2].y = -CUDART_INF_F;
            }
        }
        float most = -CUDART_INF_F;                                   // log2 of the row's largest weight, as top is of exp2(score)
#pragma unroll
        for (int x = 0; x < KEYS / 2; x += 2) {
            const float4 lv = *reinterpret_cast<const float4*>(sm_lv + slot * kTile + KEYS * h + 2 * x);
            const float2 w = fma2(c[x], both(qu), make_float2(lv.x, lv.y)), z = fma2(c[x + 1], both(qu), make_float2(lv.z, lv.w));
            top = fmaxf(top, fmaxf(fmaxf(c[x].x, c[x].y), fmaxf(c[x + 1].x, c[x + 1].y)));
            most = fmaxf(most, fmaxf(fmaxf(w.x, w.y), fmaxf(z.x, z.y)));
        }
        top *= qu;
        sm_top[h * kRows + row] = make_float2(top, most);
        if (!fine) *gave_up = 1;
        cp_async_wait<0>();
        fence_proxy_async_smem();
        tcgen05_fence_before();
        __syncthreads();                                              // the scores have been read, the next keys are there
        if (*gave_up != 0) break;
        if (left > kTile && warp == 0 && elect_one()) {
            tcgen05_fence_after();
            multiply_keys(slot ^ 1);                                  // the next tile's, while this one's weights are made
        }
        __syncwarp();
        if (left > 2 * kTile) request_keys(slot, t + 2 * kTile);
        if (t > t0) {
            fine = mbar_wait(&bars[1], slot ^ 1) && fine;
            add_outputs(i_tile - 1);
        }
#pragma unroll
        for (int x = 0; x < 4; ++x) {
            const float2 other = sm_top[x * kRows + row];
            top = fmaxf(top, other.x);
            most = fmaxf(most, other.y);
        }
        if (top > m + kAhead) {
            const float mn = fmaxf(m, top), corr = exp2_approx(m - mn);
            m = mn;
            l2 = mul2(l2, both(corr));
#pragma unroll
            for (int d = 0; d < COLS / 2; ++d) o[d] = mul2(o[d], both(corr));
        }
        // The weights are taken times a power of two that brings the row's largest to about 2^13.  (Relative to the tile's largest
        // value scale alone, rows that look past this tile would keep few bits of it: beside a token that takes the weight and
        // has small values, the outputs live on weights of 2^-17.)
        // (A far row's largest weight is not known to a power of two: the value scales count as the tile's largest.)
        const float ref = m == -CUDART_INF_F ? 0.f : m;
        const bool far = fabsf(ref) > kFar;
        const int up = kWeightBits - __float2int_rn(fminf(fmaxf((far ? top : most) - ref, -100.f), 100.f));
        const float shifted = static_cast<float>(up) - ref;
        unit = __int_as_float((127 - up) << 23);
        float2 sum = both(0.f);
        auto weights = [&](auto plain) {                              // plain: the tile has all its positions and the warp no far row
#pragma unroll
            for (int q = 0; q < KEYS / 8; ++q) {
                uint32_t hi[4], lo[4];
#pragma unroll
                for (int y = 0; y < 4; ++y) {
                    const int x = 4 * q + y;
                    float2 p;
                    if constexpr (plain.value) p = fma2(c[x], both(qu), both(shifted));
                    else p = make_float2(__fadd_rn(__fsub_rn(__fmul_rn(c[x].x, qu), ref), static_cast<float>(up)),
                                         __fadd_rn(__fsub_rn(__fmul_rn(c[x].y, qu), ref), static_cast<float>(up)));      // (packed, ptxas fuses product and sum)
                    p.x = exp2_approx(p.x);
                    p.y = exp2_approx(p.y);
                    if (!plain.value && KEYS * h + 2 * x >= left) p.x = 0.f;              // whatever the unit is
                    if (!plain.value && KEYS * h + 2 * x + 1 >= left) p.y = 0.f;
                    sum = add2(sum, p);
                    const float4 v4 = *reinterpret_cast<const float4*>(sm_vs + slot * kTile + KEYS * h + 2 * (x & ~1));
                    split_weights(mul2(p, y & 1 ? make_float2(v4.z, v4.w) : make_float2(v4.x, v4.y)), hi[y], lo[y]);
                }
                uint8_t* to = sm + S::kP + (h >> 1) * (kRows * 128) + swizzled(row, KEYS / 8 * (h & 1) + q);
                *reinterpret_cast<uint4*>(to) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
                *reinterpret_cast<uint4*>(to + S::kPPlane) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
            }
        };
        if (left >= kTile && !__any_sync(0xffffffffu, far)) weights(std::true_type{});
        else weights(std::false_type{});
        l2 = fma2(sum, both(unit), l2);
        if (left > kTile) {
            store_values(i_tile + 1, left - kTile);
            if (left > 2 * kTile) load_values(t + 2 * kTile);
        }
        fence_proxy_async_smem();
        tcgen05_fence_before();
        __syncthreads();                                              // weights and the next values are there, the outputs have been read
        if (warp == 0 && elect_one()) {
            tcgen05_fence_after();
            multiply_values(slot);
        }
        __syncwarp();
    }
    if (t0 < t1 && *gave_up == 0) {
        fine = mbar_wait(&bars[1], (i_tile - 1) & 1) && fine;
        add_outputs(i_tile - 1);
    }
    if (!fine) {                                                      // a wait that ran out: report, give the MMAs time
        atomicCAS(&g_status_kv, 0u, (static_cast<uint32_t>(kDevErrMmaWait) << 24) | 1u);
        for (int i = 0; i < 1000; ++i) __nanosleep(1000);
    }
    cp_async_wait<0>();
    const float l = l2.x + l2.y;
    float* sm_sum = reinterpret_cast<float*>(sm_top);                // [4][128]
    sm_sum[h * kRows + row] = l;
    __syncthreads();
    if (r0 + row < R) {
        float* out = a.part_o + ((static_cast<int64_t>(hk) * R + r0 + row) * splits + split) * HD + COLS * h;
#pragma unroll
        for (int x = 0; x < COLS / 2; x += 4) store_floats<8>(out + 2 * x, {o[x].x, o[x].y, o[x + 1].x, o[x + 1].y, o[x + 2].x, o[x + 2].y, o[x + 3].x, o[x + 3].y});
    }
    if (h == 0 && r0 + row < R) {
        const int64_t to = (static_cast<int64_t>(hk) * R + r0 + row) * splits + split;
        a.part_ml[2 * to] = m;
        a.part_ml[2 * to + 1] = (l + sm_sum[kRows + row]) + (sm_sum[2 * kRows + row] + sm_sum[3 * kRows + row]);
    }
    tcgen05_fence_before();
    __syncthreads();
    if (warp == 0) {
        tcgen05_fence_after();
        tmem_dealloc(tmem, kTmemCols);
    }
}

template <int HD>
int launch(const DecodeArgs& a, int splits, int blocks, cudaStream_t s) {
    static SmemOptIn opt_in;
    SGQ_CUDA_TRY(opt_in.ensure(attn_prefix_tc_int8_kernel<HD>, Shape<HD>::kBytes));
    SGQ_CUDA_TRY(launch_kernel(attn_prefix_tc_int8_kernel<HD>, dim3(static_cast<unsigned>(a.n_kv), static_cast<unsigned>(splits), static_cast<unsigned>(blocks)),
                               dim3(kThreads), Shape<HD>::kBytes, s, true, a));
    return SGQ_OK;
}

}  // namespace

int launch_prefix_tc(const DecodeArgs& a, int head_dim, int splits, int blocks, cudaStream_t s) {
    return head_dim == 128 ? launch<128>(a, splits, blocks, s) : launch<64>(a, splits, blocks, s);
}

}  // namespace sgq
