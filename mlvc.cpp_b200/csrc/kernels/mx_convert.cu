// Quantising dense rows into a microscaled matrix or a paged cache, and
// reading them back.
//
// One lane holds a chunk of 16 values: one 32-byte access of 16-bit values,
// one block of nvfp4, half a block of the 32-value formats (the halves sit in
// neighbouring lanes and exchange their maxima with one shuffle).  Bytes moved
// are what bounds these kernels: 2 or 4 bytes a dense value and 0.53 to 1.03 a
// quantised one.
#include "mx.cuh"

namespace mlvc_b200 {

constexpr int kMxThreads = 256;

// The place of packed row t in the cache, or -1 (no page, or no such row); by
// one warp.  The sequence is the last one that begins at or before t: each
// round asks 32 offsets at once, so 1024 sequences take two dependent loads.
__device__ __forceinline__ long long cache_slot(const MxConvertParams& p, long long t)
{
    const int lane = threadIdx.x & 31;
    int lo = 0, hi = p.sequences;
    if (t < p.offsets[0] || t >= p.offsets[hi])
        return -1;
    while (hi - lo > 1) {
        const int step = (hi - lo + 31) / 32;
        const long long at = lo + static_cast<long long>(lane + 1) * step;
        const int below = __popc(__ballot_sync(0xFFFFFFFFu, at < hi && p.offsets[at] <= t));
        lo += below * step;
        hi = min(hi, lo + step);
    }
    const long long position = (p.starts ? p.starts[lo] : 0) + (t - p.offsets[lo]);
    const long long place = position >= 0 ? position / p.page_rows : -1;
    int page = 0;
    const bool inside = place >= 0 && place < p.pages_per_sequence;
    if (inside)
        page = p.pages[static_cast<long long>(lo) * p.pages_per_sequence + place];
    if (!inside || page >= p.page_count) {
        if (lane == 0)
            atomicOr(&mlvc_b200_status, kStatusCachePage);
        return -1;
    }
    return page < 0 ? -1 : static_cast<long long>(page) * p.page_rows + (position - place * p.page_rows);
}

template <int DT, int F, bool kCache, bool kRead>
__device__ __forceinline__ void mx_convert(const MxConvertParams& p)
{
    pdl_launch_dependents();
    pdl_wait();
    __shared__ long long slots[kCache ? kMxCacheRowsMax : 1];
    const long long row0 = static_cast<long long>(blockIdx.x) * p.cta_rows;
    const int rows = static_cast<int>(min(static_cast<long long>(p.cta_rows), p.rows - row0));
    const int chunk0 = blockIdx.y * p.cta_chunks;
    const int chunks = min(p.cta_chunks, p.chunks - chunk0);
    if constexpr (kCache) {
        for (int r = threadIdx.x / 32; r < rows; r += kMxThreads / 32) {
            const long long s = cache_slot(p, row0 + r);
            if (threadIdx.x % 32 == 0)
                slots[r] = s;
        }
        __syncthreads();
    }
    const int items = rows * chunks;
    // whole warps: the shuffle of the 32-value formats
    for (int i = threadIdx.x; i < ((items + 31) & ~31); i += kMxThreads) {
        const int r = i / chunks, c = chunk0 + i - r * chunks;
        const long long row = row0 + r;
        const bool valid = i < items;
        long long held = row;  // row of the quantised form
        if constexpr (kCache)
            held = valid ? slots[r] : -1;
        const int column = Mx<F>::kIsNv ? c : c >> 1;
        uint32_t codes[4] = {0, 0, 0, 0}, scale = 0;
        uint8_t* data = p.data + held * p.pitch + c * Mx<F>::kChunkBytes;
        uint8_t* at = p.scales + (kCache ? held * p.scale_pitch + column : scale_at(held, column, p.k_tiles));
        if constexpr (kRead) {
            if (!valid)
                continue;
            if (!kCache || held >= 0) {
                if constexpr (Mx<F>::kIs8)
                    *reinterpret_cast<uint4*>(codes) = *reinterpret_cast<const uint4*>(data);
                else
                    *reinterpret_cast<uint2*>(codes) = *reinterpret_cast<const uint2*>(data);
                scale = *at;
            }
            float v[16];
            read_chunk<F>(codes, scale, p.tensor_scale, v);
            store_chunk<DT>(p.dense, row * p.row_stride, p.col_stride, c * 16, p.cols, p.vec, v);
        } else {
            Raw<DT> x{};
            if (valid)
                load_raw<DT>(p.dense, row * p.row_stride, p.col_stride, c * 16, p.cols, p.vec, x);
            quantise_chunk<F, DT>(x, p.tensor_scale, p.inv_six_scale, codes, scale);
            if (!valid || (kCache && held < 0))
                continue;
            if constexpr (Mx<F>::kIs8)
                *reinterpret_cast<uint4*>(data) = *reinterpret_cast<const uint4*>(codes);
            else
                *reinterpret_cast<uint2*>(data) = *reinterpret_cast<const uint2*>(codes);
            if (Mx<F>::kIsNv || !(c & 1))
                *at = static_cast<uint8_t>(scale);
            // the rest of the last scale tile: the product reads whole words
            if (!kCache && c == p.chunks - 1)
                for (int k = column + 1; k < 4 * p.k_tiles; ++k)
                    p.scales[scale_at(held, k, p.k_tiles)] = 0;
        }
    }
}

#define MLVC_MX_CONVERT(NAME, DT, F, CACHE, READ)                                                       \
    extern "C" __global__ void __launch_bounds__(kMxThreads) NAME(const __grid_constant__ MxConvertParams p) \
    {                                                                                                   \
        mx_convert<DT, F, CACHE, READ>(p);                                                              \
    }
#define MLVC_MX_CONVERT_ALL(T, DT, FN, F)                              \
    MLVC_MX_CONVERT(mlvc_mx_quantise_##T##_##FN, DT, F, false, false)  \
    MLVC_MX_CONVERT(mlvc_mx_dequantise_##T##_##FN, DT, F, false, true) \
    MLVC_MX_CONVERT(mlvc_mx_cache_write_##T##_##FN, DT, F, true, false) \
    MLVC_MX_CONVERT(mlvc_mx_cache_read_##T##_##FN, DT, F, true, true)

MLVC_MX_CONVERT_ALL(f16, kMxF16, mxfp4, kMxFp4)
MLVC_MX_CONVERT_ALL(f16, kMxF16, nvfp4, kNvFp4)
MLVC_MX_CONVERT_ALL(f16, kMxF16, mxfp8, kMxFp8)
MLVC_MX_CONVERT_ALL(bf16, kMxBf16, mxfp4, kMxFp4)
MLVC_MX_CONVERT_ALL(bf16, kMxBf16, nvfp4, kNvFp4)
MLVC_MX_CONVERT_ALL(bf16, kMxBf16, mxfp8, kMxFp8)
MLVC_MX_CONVERT_ALL(f32, kMxF32, mxfp4, kMxFp4)
MLVC_MX_CONVERT_ALL(f32, kMxF32, nvfp4, kNvFp4)
MLVC_MX_CONVERT_ALL(f32, kMxF32, mxfp8, kMxFp8)

}  // namespace mlvc_b200
