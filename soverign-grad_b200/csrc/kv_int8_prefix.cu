// Partial attention of many query rows to a shared prefix in the INT8 cache, on the tcgen05 tensor cores (kind::i8).
//
// The arithmetic is that of kv_int8.cu: codes as they lie in memory, queries and softmax weights as fixed point split into three
// balanced base-256 digits, exact integer products, fp32 in between.  With 17 query rows and more per kv head the products
// are worth the large MMA: a block takes 128 rows (sequence, query of the group) and walks its part of the prefix in tiles of
// 128 positions,
//   S_j = Q_j K^T      three MMAs of 128 x 128 x HD, one per digit plane, into 3 x 128 columns of tensor memory
//   softmax            a thread holds a quarter of a row: 32 scores; the quarters exchange their maxima through shared memory
//   O_j = P_j V        three MMAs of 128 x HD x 128 over the weights' digit planes, into the same columns
// and adds O into fp32 registers once per tile, scaled by the row's unit.  K-major operands in 128-byte-swizzled rows: the keys
// are copied as they are, the values are transposed on the way (4 x 4 bytes by byte permutes, while the tile before is in its
// second product), the weights are written as rows.  What bounds it: the fp32 work between the two products, about 20
// instructions per (row, position), 4700 cycles of a tile; its MMAs take 1500, of which 1300 are not hidden.
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
constexpr float kAhead = 6.0f;                 // see WarpAttention in kv_int8.cu

template <int HD>
struct Shape {
    static constexpr int kVPlane = HD * 128;
    static constexpr int kQ = 0, kK = kQ + 3 * kPlane, kV = kK + 2 * kPlane, kP = kV + 2 * HD * 128, kSmall = kP + 3 * kPlane;
    static constexpr int kFloats = 128 + 2 * kTile + 8 * kRows;      // units, key and value scales, the quarters' maxima (twice)
    static constexpr int kBars = kSmall + kFloats * 4, kBytes = kBars + 32 + 1024;   // 1024: alignment of the base
    static constexpr int kOutStride = HD + 4;                         // staging of the results over Q and K
};

// 16-byte chunk c of row r of a 128-byte-swizzled operand
__device__ __forceinline__ int swizzled(int r, int c) { return r * 128 + ((c ^ (r & 7)) << 4); }

__device__ __forceinline__ void cp_async_16(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}

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

// grid (kv heads, splits of the prefix, blocks of 128 rows)
template <int HD>
__global__ void __launch_bounds__(kThreads, 1) attn_prefix_tc_int8_kernel(const DecodeArgs a) {
    using S = Shape<HD>;
    constexpr int VEC = HD / 32, DW = HD / 4, KEYS = kTile / 4, COLS = HD / 4;         // a thread's part of a row: positions, output columns
    extern __shared__ uint8_t raw[];
    uint8_t* sm = raw + ((1024u - (smem_u32(raw) & 1023u)) & 1023u);
    float* sm_unit = reinterpret_cast<float*>(sm + S::kSmall);
    float* sm_ks = sm_unit + 128;
    float* sm_vs = sm_ks + kTile;
    float* sm_top = sm_vs + kTile;                                    // [4][128]
    float* sm_most = sm_top + 4 * kRows;                              // [4][128]
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
    const int n = static_cast<int>(prefix_rows(a));
    const int chunk = ((n + splits - 1) / splits + kTile - 1) / kTile * kTile;
    const int t0 = static_cast<int>(min(static_cast<int64_t>(split) * chunk, static_cast<int64_t>(n)));
    const int t1 = static_cast<int>(min(static_cast<int64_t>(t0) + chunk, static_cast<int64_t>(n)));
    const int64_t base = static_cast<int64_t>(hk) * a.first.max_seq;
    const int8_t* kc = a.first.kc + base * HD;
    const int8_t* vc = a.first.vc + base * HD;
    const float* scales = (tid < kTile ? a.first.ks : a.first.vs) + base;      // threads 0 .. 255 bring the scales
    const uint32_t sm_u = smem_u32(sm);

    auto request_keys = [&](int slot, int t) {
        constexpr int CH = HD / 16;
#pragma unroll
        for (int u = 0; u < kTile * CH / kThreads; ++u) {
            const int x = tid + u * kThreads, r = x / CH, c = x % CH;
            cp_async_16(sm_u + S::kK + slot * kPlane + swizzled(r, c), kc + static_cast<int64_t>(t) * HD + min(r, t1 - 1 - t) * HD + c * 16);
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    // A thread transposes the values 4 dw .. 4 dw + 3 of VN positions: row i DW + dw of the operand is value 4 dw + i.
    constexpr int VN = HD == 128 ? 8 : 4;
    static_assert(kTile / VN * DW == kThreads, "one unit per thread");
    const int vch = tid / DW, dw = tid % DW;                          // chunk of positions, word of values
    uint32_t vr[VN];
    float scale = 0.f;
    auto load_values = [&](int t) {
        const int8_t* from = vc + static_cast<int64_t>(t) * HD + 4 * dw;
        const int last = t1 - 1 - t;
#pragma unroll
        for (int x = 0; x < VN; ++x) vr[x] = *reinterpret_cast<const uint32_t*>(from + min(VN * vch + x, last) * HD);
        if (tid < 2 * kTile) scale = scales[t + min(tid & (kTile - 1), last)];
    };
    auto store_values = [&](int slot, int left) {                    // vr and scale, of a tile with `left` positions
        uint32_t y[4][VN / 4];                                        // [value][quad of positions]
#pragma unroll
        for (int q = 0; q < VN / 4; ++q) {
            const uint32_t p0 = __byte_perm(vr[4 * q], vr[4 * q + 1], 0x5140), p1 = __byte_perm(vr[4 * q], vr[4 * q + 1], 0x7362);
            const uint32_t p2 = __byte_perm(vr[4 * q + 2], vr[4 * q + 3], 0x5140), p3 = __byte_perm(vr[4 * q + 2], vr[4 * q + 3], 0x7362);
            y[0][q] = __byte_perm(p0, p2, 0x5410);
            y[1][q] = __byte_perm(p0, p2, 0x7632);
            y[2][q] = __byte_perm(p1, p3, 0x5410);
            y[3][q] = __byte_perm(p1, p3, 0x7632);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            uint8_t* to = sm + S::kV + slot * S::kVPlane + swizzled(i * DW + dw, VN * vch >> 4) + (VN * vch & 15);
            if constexpr (VN == 8) *reinterpret_cast<uint2*>(to) = make_uint2(y[i][0], y[i][1]);
            else *reinterpret_cast<uint32_t*>(to) = y[i][0];
        }
        // a scale that is not finite counts as NaN; positions that do not exist weigh nothing
        if (tid < kTile) sm_ks[tid] = scale + (scale - scale);
        else if (tid < 2 * kTile) sm_vs[tid - kTile] = tid - kTile < left ? scale + (scale - scale) : 0.f;
    };
    if (t0 < t1) {
        request_keys(0, t0);
        load_values(t0);
    }
    // Queries: every warp brings eight raw rows to where the second tile's values and the weights will lie and turns them into
    // digits, four at a time.  (All unrolled with everything in registers this took 12000 cycles, most of them for code.)
    {
        constexpr int QR = kRows / (kThreads / 32);
        float* rows = reinterpret_cast<float*>(sm + S::kV + S::kVPlane) + warp * QR * HD;
        int turn = -1;                                                // lane i: position of the warp's row i, -1: no such row, or idle
        for (int i = 0; i < QR; ++i) {
            const int r = min(r0 + warp * QR + i, R - 1), b = r / G;
            if (lane < HD / 4)
                cp_async_16(smem_u32(rows + i * HD + lane * 4), a.qkv + b * a.qkv_stride + static_cast<int64_t>(hk * G + r - b * G) * HD + lane * 4);
            if (lane == i) turn = b;
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
        if (lane < QR) {
            const int64_t pos = r0 + warp * QR + lane < R ? a.pos[turn * a.pos_stride] : -1;
            turn = pos >= 0 && pos < a.own.max_seq ? n + static_cast<int>(pos) : -1;
        }
        asm volatile("cp.async.wait_group 0;" ::: "memory");
        __syncwarp();
#pragma unroll 1
        for (int i0 = 0; i0 < QR; i0 += 4) {
            float q[4][VEC], co[4][VEC], si[4][VEC];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int at = __shfl_sync(0xffffffffu, turn, i0 + i);
                const int64_t from = static_cast<int64_t>(max(at, 0)) * (HD / 2) + (lane & 15) * VEC;
                load_values_of(a.cos_t + from, co[i]);
                load_values_of(a.sin_t + from, si[i]);
                load_values_of(rows + (i0 + i) * HD + lane * VEC, q[i]);
                if (at < 0) {
#pragma unroll
                    for (int j = 0; j < VEC; ++j) q[i][j] = 0.f;
                }
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int r = warp * QR + i0 + i;
                rotate_values<HD>(q[i], co[i], si[i], lane);
                query_digits<HD>(q[i], [&](int j, int d) { return sm + S::kQ + j * kPlane + swizzled(r, d >> 4) + (d & 15); }, sm_unit + r, lane);
            }
        }
    }
    if (t0 < t1) {
        store_values(0, t1 - t0);
        if (t0 + kTile < t1) {
            request_keys(1, t0 + kTile);
            load_values(t0 + kTile);
        }
    }
    tcgen05_fence_before();
    __syncthreads();
    tcgen05_fence_after();
    const uint32_t tmem = *tmem_slot;
    const uint64_t qd = umma_desc_sw128(sm_u + S::kQ), kd = umma_desc_sw128(sm_u + S::kK), vd = umma_desc_sw128(sm_u + S::kV),
                   pd = umma_desc_sw128(sm_u + S::kP);
    const int row = (warp & 3) * 32 + lane, h = warp >> 2;            // this thread: quarter h of the row
    const uint32_t tmem_row = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16);
    const float qu = sm_unit[row];
    float m = -CUDART_INF_F, l = 0.f, o[COLS];
#pragma unroll
    for (int d = 0; d < COLS; ++d) o[d] = 0.f;
    // Columns: outputs of digit j at 128 j; scores of digits 1, 2 at 0, 128 and of digit 0 at 384, where no output lies.
    auto score_cols = [](int j) { return j == 0 ? 384u : (j - 1) * 128u; };
    auto multiply_keys = [&](int j, int slot) {                       // by one thread: scores of digit j of the keys in `slot`
        const uint32_t idesc = umma_idesc(2u, 1u, kRows, kTile);
#pragma unroll
        for (int k = 0; k < HD / 32; ++k)
            tcgen05_mma_i8(tmem + score_cols(j), qd + j * (kPlane >> 4) + 2 * k, kd + slot * (kPlane >> 4) + 2 * k, idesc, k != 0 ? 1u : 0u);
    };
    auto row_sync = [&] { named_barrier_sync(1 + (warp & 3), 128); };     // the four warps that share 32 rows
    bool fine = true;
    uint32_t phase = 0;
    int slot = 0;
    for (int t = t0; t < t1; t += kTile, phase ^= 1u, slot ^= 1) {
        const int left = t1 - t;
        fence_proxy_async_smem();
        tcgen05_fence_before();
        __syncthreads();                                              // keys and values are there, the outputs have been read
        if (*gave_up != 0) break;
        if (warp == 0 && elect_one()) {
            tcgen05_fence_after();
            if (t == t0) multiply_keys(0, slot);
            multiply_keys(1, slot);
            multiply_keys(2, slot);
            tcgen05_commit(&bars[0]);
        }
        __syncwarp();
        // scores of a quarter of the positions, without the query's unit
        fine = mbar_wait(&bars[0], phase);
        tcgen05_fence_after();
        float c[KEYS], top = -CUDART_INF_F;
#pragma unroll
        for (int q = 0; q < KEYS / 16; ++q) {
            int s2[16], s1[16], s0[16];
            tmem_ld_32x32b_x16(tmem_row + score_cols(0) + KEYS * h + 16 * q, s0);
            tmem_ld_32x32b_x16(tmem_row + score_cols(1) + KEYS * h + 16 * q, s1);
            tmem_ld_32x32b_x16(tmem_row + score_cols(2) + KEYS * h + 16 * q, s2);
            tmem_ld_wait();
#pragma unroll
            for (int x = 0; x < 16; x += 4) {
                const float4 k4 = *reinterpret_cast<const float4*>(sm_ks + KEYS * h + 16 * q + x);
                c[16 * q + x] = join_digits(s2[x], s1[x], s0[x]) * k4.x;
                c[16 * q + x + 1] = join_digits(s2[x + 1], s1[x + 1], s0[x + 1]) * k4.y;
                c[16 * q + x + 2] = join_digits(s2[x + 2], s1[x + 2], s0[x + 2]) * k4.z;
                c[16 * q + x + 3] = join_digits(s2[x + 3], s1[x + 3], s0[x + 3]) * k4.w;
            }
        }
        if (left < kTile) {
#pragma unroll
            for (int x = 0; x < KEYS; ++x)
                if (KEYS * h + x >= left) c[x] = -CUDART_INF_F;
        }
#pragma unroll
        for (int x = 0; x < KEYS; ++x) top = fmaxf(top, c[x]);
        top *= qu;
        sm_top[h * kRows + row] = top;
        row_sync();
#pragma unroll
        for (int x = 0; x < 4; ++x) top = fmaxf(top, sm_top[x * kRows + row]);
        if (top > m + kAhead) {
            const float mn = fmaxf(m, top), corr = exp2_approx(m - mn);
            m = mn;
            l *= corr;
#pragma unroll
            for (int d = 0; d < COLS; ++d) o[d] *= corr;
        }
        const float ref = m == -CUDART_INF_F ? 0.f : m;
        float most = 0.f;
#pragma unroll
        for (int x = 0; x < KEYS; ++x) c[x] = exp2_approx(fmaf(c[x], qu, -ref));
        if (left < kTile) {
#pragma unroll
            for (int x = 0; x < KEYS; ++x)
                if (KEYS * h + x >= left) c[x] = 0.f;                 // whatever the unit is
        }
#pragma unroll
        for (int x = 0; x < KEYS; x += 4) {
            const float4 v4 = *reinterpret_cast<const float4*>(sm_vs + KEYS * h + x);
            l += (c[x] + c[x + 1]) + (c[x + 2] + c[x + 3]);
            c[x] *= v4.x; c[x + 1] *= v4.y; c[x + 2] *= v4.z; c[x + 3] *= v4.w;
            most = max_nan(max_nan(most, fabsf(c[x])), max_nan(fabsf(c[x + 1]), max_nan(fabsf(c[x + 2]), fabsf(c[x + 3]))));
        }
        sm_most[h * kRows + row] = most;
        row_sync();
#pragma unroll
        for (int x = 0; x < 4; ++x) most = max_nan(most, sm_most[x * kRows + row]);
        const float per = most < 1e-30f ? 0.f : __fdividef(kWeightRange, most), unit = fmaf(most, 1.0f / kWeightRange, most - most);
#pragma unroll
        for (int q = 0; q < KEYS / 16; ++q) {
            uint32_t w[3][4];
#pragma unroll
            for (int y = 0; y < 4; ++y) {
                uint32_t d[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) d[i] = weight_digits(c[16 * q + 4 * y + i], per);
                gather_digits(d, w[0][y], w[1][y], w[2][y]);
            }
#pragma unroll
            for (int j = 0; j < 3; ++j)
                *reinterpret_cast<uint4*>(sm + S::kP + j * kPlane + swizzled(row, KEYS / 16 * h + q)) = make_uint4(w[j][0], w[j][1], w[j][2], w[j][3]);
        }
        asm volatile("cp.async.wait_group 0;" ::: "memory");
        fence_proxy_async_smem();
        tcgen05_fence_before();
        __syncthreads();                                              // weights and the next keys are there, the scores have been read
        if (warp == 0 && elect_one()) {
            tcgen05_fence_after();
            const uint32_t idesc = umma_idesc(2u, 1u, kRows, HD);
#pragma unroll
            for (int j = 0; j < 3; ++j)
#pragma unroll
                for (int k = 0; k < kTile / 32; ++k)
                    tcgen05_mma_i8(tmem + j * 128, pd + j * (kPlane >> 4) + 2 * k, vd + slot * (S::kVPlane >> 4) + 2 * k, idesc, k != 0 ? 1u : 0u);
            tcgen05_commit(&bars[1]);
            if (left > kTile) multiply_keys(0, slot ^ 1);             // the next tile's, while the outputs are read
        }
        __syncwarp();
        if (left > kTile) {
            store_values(slot ^ 1, left - kTile);
            if (left > 2 * kTile) {
                request_keys(slot, t + 2 * kTile);
                load_values(t + 2 * kTile);
            }
        }
        fine = mbar_wait(&bars[1], phase) && fine;
        tcgen05_fence_after();
#pragma unroll
        for (int q = 0; q < COLS / 16; ++q) {
            int s2[16], s1[16], s0[16];
            tmem_ld_32x32b_x16(tmem_row + 0 * 128 + COLS * h + 16 * q, s0);
            tmem_ld_32x32b_x16(tmem_row + 1 * 128 + COLS * h + 16 * q, s1);
            tmem_ld_32x32b_x16(tmem_row + 2 * 128 + COLS * h + 16 * q, s2);
            tmem_ld_wait();
#pragma unroll
            for (int x = 0; x < 16; ++x) o[16 * q + x] = fmaf(join_digits(s2[x], s1[x], s0[x]), unit, o[16 * q + x]);
        }
        tcgen05_fence_before();
        if (!fine) *gave_up = 1;
    }
    if (!fine) {                                                      // a wait that ran out: report, give the MMAs time
        atomicCAS(&g_status_kv, 0u, (static_cast<uint32_t>(kDevErrMmaWait) << 24) | 1u);
        for (int i = 0; i < 1000; ++i) __nanosleep(1000);
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    // results: columns n = COLS h + x of the operand order, value 4 (n % DW) + n / DW
    sm_top[h * kRows + row] = l;
    __syncthreads();
    float* out = reinterpret_cast<float*>(sm);
#pragma unroll
    for (int x = 0; x < COLS; ++x) {
        const int c = COLS * h + x;
        out[row * S::kOutStride + 4 * (c % DW) + c / DW] = o[x];
    }
    __syncthreads();
    for (int i = tid; i < kRows * DW; i += kThreads) {
        const int r = i / DW, d = 4 * (i % DW);
        if (r0 + r >= R) break;
        *reinterpret_cast<float4*>(a.part_o + ((static_cast<int64_t>(hk) * R + r0 + r) * splits + split) * HD + d) =
            *reinterpret_cast<const float4*>(out + r * S::kOutStride + d);
    }
    if (h == 0 && r0 + row < R) {
        const int64_t to = (static_cast<int64_t>(hk) * R + r0 + row) * splits + split;
        a.part_ml[2 * to] = m;
        a.part_ml[2 * to + 1] = (l + sm_top[kRows + row]) + (sm_top[2 * kRows + row] + sm_top[3 * kRows + row]);
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
