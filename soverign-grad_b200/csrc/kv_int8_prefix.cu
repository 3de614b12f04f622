// Partial attention of many query rows to a shared prefix in the INT8 cache, on the tcgen05 tensor cores (kind::i8).
//
// The arithmetic is that of kv_int8.cu: codes as they lie in memory, queries and softmax weights as fixed point split into three
// balanced base-256 digits, exact integer products, fp32 in between.  With 17 query rows and more per kv head the products
// are worth the large MMA: a block takes 128 rows (sequence, query of the group) and walks its part of the prefix in tiles of
// 128 positions,
//   S_j = Q_j K^T      three MMAs of 128 x 128 x HD, one per digit plane, into 3 x 128 columns of tensor memory
//   softmax            a thread holds half a row: 64 scores; the two halves exchange their maxima through shared memory
//   O_j = P_j V        three MMAs of 128 x HD x 128 over the weights' digit planes, into the same columns
// and adds O into fp32 registers once per tile, scaled by the row's unit.  K-major operands in 128-byte-swizzled rows: the keys
// are copied as they are, the values are transposed on the way (4 x 4 bytes by byte permutes), the weights are written as rows.
// What bounds it: the fp32 work between the two products, about 20 instructions per (row, position); the MMAs of a tile take
// about 1500 cycles and do not overlap it.
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

constexpr int kThreads = 256, kRows = kPrefixTcRows, kTile = kPrefixTcTile;
constexpr int kPlane = 128 * 128;              // an operand: 128 rows of 128 bytes
constexpr int kTmemCols = 512;
constexpr float kAhead = 6.0f;                 // see WarpAttention in kv_int8.cu

template <int HD>
struct Shape {
    static constexpr int kQ = 0, kK = kQ + 3 * kPlane, kV = kK + 2 * kPlane, kP = kV + HD * 128, kSmall = kP + 3 * kPlane;
    static constexpr int kFloats = 128 + 2 * kTile + 4 * kRows;      // units, key and value scales, the halves' maxima (twice)
    static constexpr int kBars = kSmall + kFloats * 4, kBytes = kBars + 32 + 1024;   // 1024: alignment of the base
    static constexpr int kOutStride = HD + 4;                         // staging of the results over Q, K and V
};

// 16-byte chunk c of row r of a 128-byte-swizzled operand
__device__ __forceinline__ int swizzled(int r, int c) { return r * 128 + ((c ^ (r & 7)) << 4); }

__device__ __forceinline__ void cp_async_16(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}

// grid (kv heads, splits of the prefix, blocks of 128 rows)
template <int HD>
__global__ void __launch_bounds__(kThreads, 1) attn_prefix_tc_int8_kernel(const DecodeArgs a) {
    using S = Shape<HD>;
    constexpr int VEC = HD / 32, DW = HD / 4, HALF = HD / 2;
    extern __shared__ uint8_t raw[];
    uint8_t* sm = raw + ((1024u - (smem_u32(raw) & 1023u)) & 1023u);
    float* sm_unit = reinterpret_cast<float*>(sm + S::kSmall);
    float* sm_ks = sm_unit + 128;
    float* sm_vs = sm_ks + kTile;
    float* sm_top = sm_vs + kTile;                                    // [2][128]
    float* sm_most = sm_top + 2 * kRows;                              // [2][128]
    uint64_t* bars = reinterpret_cast<uint64_t*>(sm + S::kBars);      // scores done, outputs done
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 2);
    const int tid = threadIdx.x, warp = warp_index(), lane = tid & 31;
    if (warp == 0) {
        tmem_alloc(tmem_slot, kTmemCols);
        tmem_relinquish();
    }
    if (tid == 0) {
        mbar_init(&bars[0], 1);
        mbar_init(&bars[1], 1);
        mbar_fence_init();
    }
    pdl_wait();
    pdl_launch_dependents();                                          // behind the wait: see attn_decode_int8_kernel
    const int hk = blockIdx.x, split = blockIdx.y, splits = gridDim.y, G = a.n_heads / a.n_kv;
    const int64_t R = static_cast<int64_t>(a.batch) * G, r0 = static_cast<int64_t>(blockIdx.z) * kRows;
    const int n = static_cast<int>(prefix_rows(a));
    const int chunk = ((n + splits - 1) / splits + kTile - 1) / kTile * kTile;
    const int t0 = static_cast<int>(min(static_cast<int64_t>(split) * chunk, static_cast<int64_t>(n)));
    const int t1 = static_cast<int>(min(static_cast<int64_t>(t0) + chunk, static_cast<int64_t>(n)));
    const int64_t base = static_cast<int64_t>(hk) * a.first.max_seq;
    const int8_t* kc = a.first.kc + base * HD;
    const int8_t* vc = a.first.vc + base * HD;
    const float* scales = (tid < kTile ? a.first.ks : a.first.vs) + base;
    const uint32_t sm_u = smem_u32(sm);

    auto request_keys = [&](int slot, int t) {
        constexpr int CH = HD / 16;
#pragma unroll
        for (int u = 0; u < kTile * CH / kThreads; ++u) {
            const int x = tid + u * kThreads, r = x / CH, c = x % CH;
            cp_async_16(sm_u + S::kK + slot * kPlane + swizzled(r, c), kc + static_cast<int64_t>(min(t + r, t1 - 1)) * HD + c * 16);
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    // A thread transposes the values 4 dw .. 4 dw + 3 of 16 positions: row i DW + dw of the operand is value 4 dw + i.
    const int vch = tid / DW, dw = tid % DW;                          // chunk of positions, word of values
    const bool has_v = vch < kTile / 16;
    uint32_t vr[16];
    float scale = 0.f;
    auto load_values = [&](int t) {
        if (has_v) {
#pragma unroll
            for (int x = 0; x < 16; ++x)
                vr[x] = *reinterpret_cast<const uint32_t*>(vc + static_cast<int64_t>(min(t + 16 * vch + x, t1 - 1)) * HD + 4 * dw);
        }
        scale = scales[min(t + (tid & (kTile - 1)), t1 - 1)];
    };
    if (t0 < t1) {
        request_keys(0, t0);
        load_values(t0);
    }
    // queries: 16 rows per warp, four at a time
    for (int i0 = 0; i0 < 16; i0 += 4) {
        float q[4][VEC];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int64_t r = r0 + warp * 16 + i0 + i, b = r < R ? r / G : 0, pos = a.pos[b * a.pos_stride];
            const bool live = r < R && pos >= 0 && pos < a.own.max_seq;
            const int64_t turn = (live ? n + pos : 0) * HALF;
#pragma unroll
            for (int j = 0; j < VEC; ++j) q[i][j] = live ? a.qkv[b * a.qkv_stride + (hk * G + r - b * G) * HD + lane * VEC + j] : 0.f;
            rotate_row<HD>(q[i], a.cos_t + turn, a.sin_t + turn, lane);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int r = warp * 16 + i0 + i;
            query_digits<HD>(q[i], [&](int j, int d) { return sm + S::kQ + j * kPlane + swizzled(r, d >> 4) + (d & 15); }, sm_unit + r, lane);
        }
    }
    tcgen05_fence_before();
    __syncthreads();
    tcgen05_fence_after();
    const uint32_t tmem = *tmem_slot;
    const int row = (warp & 3) * 32 + lane, h = warp >> 2;            // this thread: half h of the row
    const uint32_t tmem_row = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16);
    const float qu = sm_unit[row];
    float m = -CUDART_INF_F, l = 0.f, o[HALF];
#pragma unroll
    for (int d = 0; d < HALF; ++d) o[d] = 0.f;
    const uint64_t qd = umma_desc_sw128(sm_u + S::kQ), kd = umma_desc_sw128(sm_u + S::kK), vd = umma_desc_sw128(sm_u + S::kV),
                   pd = umma_desc_sw128(sm_u + S::kP);
    bool fine = true;
    uint32_t phase = 0;
    int slot = 0;
    for (int t = t0; t < t1; t += kTile, phase ^= 1u, slot ^= 1) {
        const int left = t1 - t;
        // a scale that is not finite counts as NaN; positions that do not exist weigh nothing
        if (tid < kTile) sm_ks[tid] = scale + (scale - scale);
        else sm_vs[tid - kTile] = tid - kTile < left ? scale + (scale - scale) : 0.f;
        asm volatile("cp.async.wait_group 0;" ::: "memory");
        fence_proxy_async_smem();
        __syncthreads();                                              // keys (and the queries) are there, the columns are free
        if (warp == 0 && elect_one()) {
            tcgen05_fence_after();
            const uint32_t idesc = umma_idesc(2u, 1u, kRows, kTile);
            for (int j = 0; j < 3; ++j)
                for (int k = 0; k < HD / 32; ++k)
                    tcgen05_mma_i8(tmem + j * 128, qd + j * (kPlane >> 4) + 2 * k, kd + slot * (kPlane >> 4) + 2 * k, idesc, k != 0 ? 1u : 0u);
            tcgen05_commit(&bars[0]);
        }
        __syncwarp();
        if (has_v) {
            uint32_t y[4][4];                                         // [value][quad of positions]
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const uint32_t p0 = __byte_perm(vr[4 * q], vr[4 * q + 1], 0x5140), p1 = __byte_perm(vr[4 * q], vr[4 * q + 1], 0x7362);
                const uint32_t p2 = __byte_perm(vr[4 * q + 2], vr[4 * q + 3], 0x5140), p3 = __byte_perm(vr[4 * q + 2], vr[4 * q + 3], 0x7362);
                y[0][q] = __byte_perm(p0, p2, 0x5410);
                y[1][q] = __byte_perm(p0, p2, 0x7632);
                y[2][q] = __byte_perm(p1, p3, 0x5410);
                y[3][q] = __byte_perm(p1, p3, 0x7632);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i)
                *reinterpret_cast<uint4*>(sm + S::kV + swizzled(i * DW + dw, vch)) = make_uint4(y[i][0], y[i][1], y[i][2], y[i][3]);
        }
        if (left > kTile) {
            request_keys(slot ^ 1, t + kTile);
            load_values(t + kTile);
        }
        // scores of 64 positions, without the query's unit
        fine = mbar_wait(&bars[0], phase);
        tcgen05_fence_after();
        float c[64], top = -CUDART_INF_F;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            int s2[16], s1[16], s0[16];
            tmem_ld_32x32b_x16(tmem_row + 0 * 128 + 64 * h + 16 * q, s0);
            tmem_ld_32x32b_x16(tmem_row + 1 * 128 + 64 * h + 16 * q, s1);
            tmem_ld_32x32b_x16(tmem_row + 2 * 128 + 64 * h + 16 * q, s2);
            tmem_ld_wait();
#pragma unroll
            for (int x = 0; x < 16; ++x) c[16 * q + x] = join_digits(s2[x], s1[x], s0[x]) * sm_ks[64 * h + 16 * q + x];
        }
        if (left < kTile) {
#pragma unroll
            for (int x = 0; x < 64; ++x)
                if (64 * h + x >= left) c[x] = -CUDART_INF_F;
        }
#pragma unroll
        for (int x = 0; x < 64; ++x) top = fmaxf(top, c[x]);
        top *= qu;
        sm_top[h * kRows + row] = top;
        __syncthreads();
        top = fmaxf(top, sm_top[(h ^ 1) * kRows + row]);
        if (top > m + kAhead) {
            const float mn = fmaxf(m, top), corr = exp2_approx(m - mn);
            m = mn;
            l *= corr;
#pragma unroll
            for (int d = 0; d < HALF; ++d) o[d] *= corr;
        }
        const float ref = m == -CUDART_INF_F ? 0.f : m;
        float most = 0.f;
#pragma unroll
        for (int x = 0; x < 64; ++x) {
            float p = exp2_approx(fmaf(c[x], qu, -ref));
            if (left < kTile && 64 * h + x >= left) p = 0.f;
            l += p;
            c[x] = p * sm_vs[64 * h + x];
            most = max_nan(most, fabsf(c[x]));
        }
        sm_most[h * kRows + row] = most;
        __syncthreads();
        most = max_nan(most, sm_most[(h ^ 1) * kRows + row]);
        const float per = most < 1e-30f ? 0.f : __fdividef(kWeightRange, most), unit = fmaf(most, 1.0f / kWeightRange, most - most);
#pragma unroll
        for (int q = 0; q < 4; ++q) {
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
                *reinterpret_cast<uint4*>(sm + S::kP + j * kPlane + swizzled(row, 4 * h + q)) = make_uint4(w[j][0], w[j][1], w[j][2], w[j][3]);
        }
        fence_proxy_async_smem();
        tcgen05_fence_before();
        __syncthreads();                                              // weights and values are there, the scores have been read
        if (warp == 0 && elect_one()) {
            tcgen05_fence_after();
            const uint32_t idesc = umma_idesc(2u, 1u, kRows, HD);
            for (int j = 0; j < 3; ++j)
                for (int k = 0; k < kTile / 32; ++k)
                    tcgen05_mma_i8(tmem + j * 128, pd + j * (kPlane >> 4) + 2 * k, vd + 2 * k, idesc, k != 0 ? 1u : 0u);
            tcgen05_commit(&bars[1]);
        }
        __syncwarp();
        fine = mbar_wait(&bars[1], phase) && fine;
        tcgen05_fence_after();
#pragma unroll
        for (int q = 0; q < HALF / 16; ++q) {
            int s2[16], s1[16], s0[16];
            tmem_ld_32x32b_x16(tmem_row + 0 * 128 + HALF * h + 16 * q, s0);
            tmem_ld_32x32b_x16(tmem_row + 1 * 128 + HALF * h + 16 * q, s1);
            tmem_ld_32x32b_x16(tmem_row + 2 * 128 + HALF * h + 16 * q, s2);
            tmem_ld_wait();
#pragma unroll
            for (int x = 0; x < 16; ++x) o[16 * q + x] = fmaf(join_digits(s2[x], s1[x], s0[x]), unit, o[16 * q + x]);
        }
        tcgen05_fence_before();
        if (__syncthreads_or(!fine)) {                                // a wait that ran out: report, give the MMAs time, leave
            if (tid == 0) atomicCAS(&g_status_kv, 0u, (static_cast<uint32_t>(kDevErrMmaWait) << 24) | 1u);
            for (int i = 0; i < 1000; ++i) __nanosleep(1000);
            break;
        }
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    // results: columns n = HALF h + x of the operand order, value 4 (n % DW) + n / DW
    sm_top[h * kRows + row] = l;
    __syncthreads();
    float* out = reinterpret_cast<float*>(sm);
#pragma unroll
    for (int x = 0; x < HALF; ++x) {
        const int c = HALF * h + x;
        out[row * S::kOutStride + 4 * (c % DW) + c / DW] = o[x];
    }
    __syncthreads();
    for (int i = tid; i < kRows * HD; i += kThreads) {
        const int r = i / HD, d = i % HD;
        if (r0 + r >= R) break;
        a.part_o[((hk * R + r0 + r) * splits + split) * HD + d] = out[r * S::kOutStride + d];
    }
    if (h == 0 && r0 + row < R) {
        const int64_t to = (hk * R + r0 + row) * splits + split;
        a.part_ml[2 * to] = m;
        a.part_ml[2 * to + 1] = l + sm_top[kRows + row];
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
