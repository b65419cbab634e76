// Products of few rows (1 to 128) with quantised weights:
//     y[m, n] = leaky(alpha * sum_k x[m, k] w[n, k] + bias[n]) + residual[m, n]
//
// Reading the weights bounds these calls, so the roles of the operands are
// swapped: 128 weight rows fill the tensor core's M, the few rows of x are its
// N (a multiple of 8), and nothing is padded to 128 but what is in memory
// anyway.  Where there are fewer weight tiles than SMs, the panels of k are
// split over the CTAs of a cluster; their sums meet through distributed shared
// memory, in rank order, so results do not depend on timing.
//
// Dense rows are quantised here, by every CTA for its share of k, into the
// swizzled tiles that the tensor core reads: that work (16 values a lane) runs
// while the first weight panels are on their way, and saves a launch and a
// round trip of x through memory.  Rows quantised beforehand come by TMA beside
// each weight panel.
//
// Warps: 0 copies, 1 MMA and TMEM, 2..9 quantise and then finish the sums.
#include "mx.cuh"

namespace mlvc_b200 {

constexpr int kMxRowsThreads = 320;
constexpr int kMxRowsMaxStages = 12;
constexpr int kMxRowsMaxGroups = 32;  // of panels of x (see MxRowsParams::group)
constexpr int kMxRowsHeader = 1024;

struct MxRowsShared {
    uint64_t full[kMxRowsMaxStages];
    uint64_t empty[kMxRowsMaxStages];
    uint64_t x_full[kMxRowsMaxGroups];
    uint64_t sums;
    uint64_t drain;
    uint32_t tmem_base;
    int abort_flag;
};
static_assert(sizeof(MxRowsShared) <= kMxRowsHeader, "header");

__device__ __forceinline__ float4 load_cluster(uint32_t saddr, uint32_t rank)
{
    float4 v;
    asm volatile(
        "{\n\t.reg .u32 a;\n\tmapa.shared::cluster.u32 a, %4, %5;\n\t"
        "ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [a];\n\t}"
        : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
        : "r"(saddr), "r"(rank));
    return v;
}

// One result.
__device__ __forceinline__ void mx_finish_one(const MxEpilogue& e, int m, int n, float sum, float bias)
{
    const float t = fmaf(sum, e.alpha, bias);
    float v = t >= 0.0f ? t : t * e.slope;
    const long long at = m * e.y_stride + n, res = m * e.residual_stride + n;
    if (e.y_dtype == kMxF16) {
        if (e.residual)
            v += __half2float(static_cast<const __half*>(e.residual)[res]);
        static_cast<__half*>(e.y)[at] = __float2half_rn(v);
    } else if (e.y_dtype == kMxBf16) {
        if (e.residual)
            v += __bfloat162float(static_cast<const __nv_bfloat16*>(e.residual)[res]);
        static_cast<__nv_bfloat16*>(e.y)[at] = __float2bfloat16_rn(v);
    } else {
        if (e.residual)
            v += static_cast<const float*>(e.residual)[res];
        static_cast<float*>(e.y)[at] = v;
    }
}

// DT < 0: x is already quantised.
template <int F, int DT>
__device__ __forceinline__ void mx_rows(const MxRowsParams& p)
{
    constexpr bool kDense = DT >= 0;
    constexpr int kWords = Mx<F>::kWords;
    constexpr uint32_t kW = 128 * 128, kS = kWords * 512;
    extern __shared__ __align__(1024) uint8_t smem_dyn[];
    uint8_t* base = align_smem_1024(smem_dyn);
    MxRowsShared* sh = reinterpret_cast<MxRowsShared*>(base);
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const uint32_t rank = blockIdx.x % p.splits;
    const int n0 = blockIdx.x / p.splits * 128;
    const int k0 = static_cast<int>(static_cast<long long>(p.k.count) * rank / p.splits);
    const int k1 = static_cast<int>(static_cast<long long>(p.k.count) * (rank + 1) / p.splits);
    const int panels = k1 - k0;
    const int M = p.e.M;

    // shared memory: dense: x tiles and their scales of all panels, then the
    // ring of weight panels; else the ring holds both operands
    const uint32_t x_bytes = static_cast<uint32_t>(p.row_tile) * 128u;
    uint8_t* x_tiles = base + kMxRowsHeader;
    const int most = (p.k.count + p.splits - 1) / p.splits;
    uint8_t* x_scales = x_tiles + (kDense ? most * x_bytes : 0);
    uint8_t* ring = x_scales + (kDense ? (most * kS + 1023) / 1024 * 1024 : 0);
    const uint32_t stage_bytes = (kW + kS + (kDense ? 0 : x_bytes + kS) + 1023) / 1024 * 1024;
    const uint32_t x_at = kW, sw_at = kDense ? kW : kW + x_bytes, sx_at = sw_at + kS;

    if (threadIdx.x == 0) {
        for (int s = 0; s < p.stages; ++s) {
            mbar_init(&sh->full[s], 1);
            mbar_init(&sh->empty[s], 1);
        }
        if constexpr (kDense)
            for (int g = 0; g * p.group < panels; ++g)
                mbar_init(&sh->x_full[g], 256);
        mbar_init(&sh->sums, 1);
        mbar_init(&sh->drain, 1);
        sh->abort_flag = 0;
        fence_barrier_init();
    }
    // TMEM is taken once the kernel before has ended: one that allocates after
    // it let this one start would otherwise wait for columns held here.  The
    // columns hold the sums, then the scales of both operands.
    const uint32_t cols_needed = p.row_tile + 8 * kWords;
    const uint32_t tmem_cols = cols_needed <= 64 ? 64 : cols_needed <= 128 ? 128 : 256;
    pdl_wait();
    if (warp == 1)
        tmem_alloc(&sh->tmem_base, tmem_cols);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    pdl_launch_dependents();
    const uint32_t tmem = sh->tmem_base;
    bool issuer = false;
    uint32_t issued = 0;

    if (warp == 0) {
        if (elect_one()) {
            uint32_t armed = 0, parity = 0;
            int stage = 0;
            uint32_t phase = 0;
            for (int k = k0; k < k1; ++k) {
                if (!mbar_wait(&sh->empty[stage], phase ^ 1u, &sh->abort_flag, kErrMxProducer))
                    break;
                uint8_t* s = ring + stage * stage_bytes;
                uint64_t* bar = &sh->full[stage];
                const uint32_t sbytes = 512u * (k + 1 == p.k.count ? p.k.last_words : kWords);
                const long long word = static_cast<long long>(k) * kWords;
                mbar_arrive_expect_tx(bar, kW + sbytes + (kDense ? 0 : x_bytes + sbytes));
                tma_load_2d(s, &p.map_w, bar, k * 128, n0);
                bulk_load(s + sw_at, p.scales_w + (static_cast<long long>(n0 / 128) * p.k.k_tiles + word) * 512, sbytes, bar);
                if constexpr (!kDense) {
                    tma_load_2d(s + x_at, &p.map_x, bar, k * 128, 0);
                    bulk_load(s + sx_at, p.scales_x + word * 512, sbytes, bar);
                }
                armed |= 1u << stage;
                parity = (parity & ~(1u << stage)) | (phase << stage);
                if (++stage == p.stages) {
                    stage = 0;
                    phase ^= 1u;
                }
            }
            if (sh->abort_flag) {  // no copy may land after this CTA has gone
                volatile int never = 0;
                for (int s = 0; s < p.stages; ++s)
                    if ((armed >> s) & 1u)
                        mbar_wait(&sh->full[s], (parity >> s) & 1u, &never, kErrMxProducer);
            }
        }
        __syncwarp();
    } else if (warp == 1) {
        if (elect_one()) {
            issuer = true;
            const uint32_t idesc = mx_idesc<F>(128, p.row_tile);
            const uint32_t tmem_sw = tmem + p.row_tile, tmem_sx = tmem_sw + 4 * kWords;
            int stage = 0;
            uint32_t phase = 0;
            bool ok = true;
            for (int k = k0, g = 0; ok && k < k1; ++k) {
                if (kDense && k - k0 == g * p.group &&
                    !mbar_wait(&sh->x_full[g++], 0, &sh->abort_flag, kErrMxMma)) {
                    ok = false;
                    break;
                }
                if (!mbar_wait(&sh->full[stage], phase, &sh->abort_flag, kErrMxMma)) {
                    ok = false;
                    break;
                }
                tc_fence_after();
                const uint32_t s = smem_u32(ring + stage * stage_bytes);
                const uint32_t x = kDense ? smem_u32(x_tiles) + (k - k0) * x_bytes : s + x_at;
                const uint32_t sx = kDense ? smem_u32(x_scales) + (k - k0) * kS : s + sx_at;
                const bool last = k + 1 == p.k.count;
                const int words = last ? p.k.last_words : kWords, steps = last ? p.k.last_steps : 4;
                for (int w = 0; w < words; ++w) {
                    tmem_copy_scales(tmem_sw + 4 * w, s + sw_at + 512 * w);
                    tmem_copy_scales(tmem_sx + 4 * w, sx + 512 * w);
                }
#pragma unroll
                for (int ks = 0; ks < 4; ++ks) {
                    if (ks >= steps)
                        break;
                    const uint32_t w = ks * kWords / 4, id = kWords == 4 ? 0 : kWords == 2 ? (ks & 1) * 2 : ks;
                    umma_mx<F>(tmem, smem_desc(s + ks * 32, 16, 1024, 2), smem_desc(x + ks * 32, 16, 1024, 2), idesc, id,
                               tmem_sw + 4 * w, tmem_sx + 4 * w, (k - k0) | ks);
                    ++issued;
                }
                umma_commit(&sh->empty[stage]);
                if (++stage == p.stages) {
                    stage = 0;
                    phase ^= 1u;
                }
            }
            if (ok)
                umma_commit(&sh->sums);
        }
        __syncwarp();
    } else {
        const int t = threadIdx.x - 64;  // 0..255
        if constexpr (kDense) {
            // a group of panels at a time, four chunks a thread under way at once
            constexpr int kChunks = Mx<F>::kPanelValues / 16;  // of a panel
            constexpr int kBatch = 4;
            for (int g = 0; g * p.group < panels; ++g) {
                const int first = g * p.group;  // panel
                const int row_chunks = min(p.group, panels - first) * kChunks, items = M * row_chunks;
                for (int i0 = t; i0 < ((items + 31) & ~31); i0 += 256 * kBatch) {
                    Raw<DT> x[kBatch];
#pragma unroll
                    for (int b = 0; b < kBatch; ++b) {
                        const int i = i0 + 256 * b, m = i / row_chunks, c = i - m * row_chunks;
                        if (i < items)
                            load_raw<DT>(static_cast<const typename Dense<DT>::T*>(p.x) + m * p.row_stride, p.col_stride,
                                         ((k0 + first) * kChunks + c) * 16, p.cols, p.vec, x[b]);
                        else
                            x[b] = Raw<DT>{};
                    }
#pragma unroll
                    for (int b = 0; b < kBatch; ++b) {
                        const int i = i0 + 256 * b, m = i / row_chunks, c = i - m * row_chunks;
                        if ((i & ~31) >= items)  // whole warps
                            break;
                        uint32_t codes[4], scale;
                        quantise_chunk<F, DT>(x[b], p.tensor_scale, p.inv_six_scale, codes, scale);
                        if (i >= items)
                            continue;
                        const int panel = first + c / kChunks, in = c % kChunks;
                        const int byte = in * Mx<F>::kChunkBytes;
                        uint8_t* to = x_tiles + panel * x_bytes + m * 128 + (((byte >> 4) ^ (m & 7)) << 4) + (byte & 15);
                        if constexpr (Mx<F>::kIs8)
                            *reinterpret_cast<uint4*>(to) = make_uint4(codes[0], codes[1], codes[2], codes[3]);
                        else
                            *reinterpret_cast<uint2*>(to) = make_uint2(codes[0], codes[1]);
                        const int column = Mx<F>::kIsNv ? in : in >> 1;
                        if (Mx<F>::kIsNv || !(in & 1))
                            x_scales[panel * kS + (column >> 2) * 512 + (m & 31) * 16 + (m >> 5) * 4 + (column & 3)] =
                                static_cast<uint8_t>(scale);
                    }
                }
                fence_proxy_async_smem();  // the tensor core reads through the async proxy
                mbar_arrive(&sh->x_full[g]);
            }
        }
        // the warp's quadrant of the 128 weight rows, half of the columns (rows
        // of x, 32 at a time)
        const int quadrant = warp & 3, group = (warp - 2) / 4, n = quadrant * 32 + lane;
        const bool ok = __all_sync(0xFFFFFFFFu, mbar_wait(&sh->sums, 0, &sh->abort_flag, kErrMxEpilogue));
        tc_fence_after();
        if (ok) {
            float* part = reinterpret_cast<float*>(ring);  // [row of x][128], once the weights are consumed
            const float bias = p.e.bias && n0 + n < p.e.N ? p.e.bias[n0 + n] : 0.0f;
            for (int c = group * 32; c < M; c += 64) {
                uint32_t v[32];
                const uint32_t at = tmem + c + (static_cast<uint32_t>(quadrant * 32) << 16);
                tmem_ld32_nowait(at, v);
                tmem_wait_ld();
#pragma unroll
                for (int i = 0; i < 32; ++i) {
                    if (c + i >= M)
                        break;
                    if (p.splits > 1)
                        part[(c + i) * 128 + n] = __uint_as_float(v[i]);
                    else if (n0 + n < p.e.N)
                        mx_finish_one(p.e, c + i, n0 + n, __uint_as_float(v[i]), bias);
                }
                __syncwarp();
            }
        }
    }
    if (issuer && sh->abort_flag && issued) {  // MMAs in flight end before TMEM is freed
        umma_commit(&sh->drain);
        volatile int never = 0;
        mbar_wait(&sh->drain, 0, &never, kErrMxMma);
    }
    tc_fence_before();
    __syncthreads();
    if (p.splits > 1) {
        cluster_barrier();  // every CTA's part is written
        if (warp >= 2) {
            // a warp takes a row of x: four columns a lane, all parts under way at once
            const uint32_t part = smem_u32(ring) + lane * 16;
            for (int m = static_cast<int>(rank) + p.splits * (warp - 2); m < M; m += 8 * p.splits) {
                float4 v[8];
#pragma unroll
                for (int r = 0; r < 8; ++r)
                    if (r < p.splits)
                        v[r] = load_cluster(part + m * 512, r);
                float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
                for (int r = 0; r < 8; ++r)
                    if (r < p.splits)
                        sum = make_float4(sum.x + v[r].x, sum.y + v[r].y, sum.z + v[r].z, sum.w + v[r].w);
                const float s[4] = {sum.x, sum.y, sum.z, sum.w};
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int n = n0 + lane * 4 + i;
                    if (n < p.e.N)
                        mx_finish_one(p.e, m, n, s[i], p.e.bias ? p.e.bias[n] : 0.0f);
                }
            }
        }
        __syncwarp();
        cluster_barrier();  // no CTA leaves while its part is being read
    }
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem, tmem_cols);
    }
}

#define MLVC_MX_ROWS(NAME, F, DT)                                                                              \
    extern "C" __global__ void __launch_bounds__(kMxRowsThreads) NAME(const __grid_constant__ MxRowsParams p) \
    {                                                                                                          \
        mx_rows<F, DT>(p);                                                                                     \
    }
#define MLVC_MX_ROWS_ALL(FN, F)                          \
    MLVC_MX_ROWS(mlvc_mx_rows_quantised_##FN, F, -1)     \
    MLVC_MX_ROWS(mlvc_mx_rows_f16_##FN, F, kMxF16)       \
    MLVC_MX_ROWS(mlvc_mx_rows_bf16_##FN, F, kMxBf16)     \
    MLVC_MX_ROWS(mlvc_mx_rows_f32_##FN, F, kMxF32)
MLVC_MX_ROWS_ALL(mxfp4, kMxFp4)
MLVC_MX_ROWS_ALL(nvfp4, kNvFp4)
MLVC_MX_ROWS_ALL(mxfp8, kMxFp8)

}  // namespace mlvc_b200
