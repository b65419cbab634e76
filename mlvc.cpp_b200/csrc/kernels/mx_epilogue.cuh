// What follows a product's sums: y = leaky(alpha * sum + bias) + residual, from
// TMEM to memory, 32 x 32 results of one warp at a time.
//
// In TMEM a lane holds a row; rows of y are far apart, so stores straight from
// there would touch 32 lines for 16 bytes each and compete with the operands'
// loads for the way to L2 (they cost 33 of 279 us at 8192 x 8192 x 8192).  The
// chunk is turned in shared memory (4 KB a warp, 16-byte pieces exchanged
// within a row by row % 8, so that neither side meets a bank twice), and then
// consecutive lanes hold consecutive columns.  Residual and bias are asked for
// before the sums are waited for.
#pragma once

#include "mx.cuh"

namespace mlvc_b200 {

constexpr int kMxTurnBytes = 4096;  // of a warp

template <int DT>
struct MxTurn {
    static constexpr int kCols = DT == kMxF32 ? 4 : 8;  // a lane's columns: 16 bytes of y
    static constexpr int kLanes = 32 / kCols;           // of a row
    static constexpr int kRounds = kLanes;              // each of 32 / kLanes rows
};

// `after` is called once the sums are in registers.
template <int DT, typename After>
__device__ __forceinline__ void mx_empty_chunk(const MxEpilogue& e, float4* turn, uint32_t taddr, long long row0, int col0,
                                               After&& after)
{
    using D = Dense<DT>;
    using T = typename D::T;
    using S = MxTurn<DT>;
    const int lane = threadIdx.x & 31;
    const int col = col0 + (lane % S::kLanes) * S::kCols, sub = lane / S::kLanes;
    const bool wide = e.vec && col + S::kCols <= e.N;
    uint4 res[S::kRounds];
    float bias[S::kCols];
#pragma unroll
    for (int i = 0; i < S::kRounds; ++i) {
        res[i] = make_uint4(0, 0, 0, 0);
        const long long row = row0 + sub + i * S::kCols;
        if (e.residual && wide && row < e.M)
            res[i] = *reinterpret_cast<const uint4*>(static_cast<const T*>(e.residual) + row * e.residual_stride + col);
    }
#pragma unroll
    for (int k = 0; k < S::kCols; ++k)
        bias[k] = e.bias && wide ? e.bias[col + k] : 0.0f;

    uint32_t v[32];
    tmem_ld32_nowait(taddr, v);
    tmem_wait_ld();
    after();
#pragma unroll
    for (int q = 0; q < 8; ++q)
        turn[lane * 8 + (q ^ (lane & 7))] = make_float4(__uint_as_float(v[4 * q]), __uint_as_float(v[4 * q + 1]),
                                                        __uint_as_float(v[4 * q + 2]), __uint_as_float(v[4 * q + 3]));
    __syncwarp();
    auto finish = [&](float sum, float b) {
        const float t = fmaf(sum, e.alpha, b);
        return t >= 0.0f ? t : t * e.slope;
    };
    if (__all_sync(0xFFFFFFFFu, wide)) {
#pragma unroll
        for (int i = 0; i < S::kRounds; ++i) {
            const int r = sub + i * S::kCols;
            const int q = (lane % S::kLanes) * (S::kCols / 4);
            float f[S::kCols];
#pragma unroll
            for (int k = 0; k < S::kCols; k += 4) {
                const float4 s = turn[r * 8 + ((q + k / 4) ^ (r & 7))];
                f[k] = finish(s.x, bias[k]);
                f[k + 1] = finish(s.y, bias[k + 1]);
                f[k + 2] = finish(s.z, bias[k + 2]);
                f[k + 3] = finish(s.w, bias[k + 3]);
            }
            const uint32_t u[4] = {res[i].x, res[i].y, res[i].z, res[i].w};
            uint32_t o[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                if constexpr (DT == kMxF32) {
                    o[k] = __float_as_uint(f[k] + __uint_as_float(u[k]));
                } else {
                    float a, b;
                    D::unpack(u[k], a, b);
                    o[k] = D::pack2(f[2 * k] + a, f[2 * k + 1] + b);
                }
            }
            if (row0 + r < e.M)
                *reinterpret_cast<uint4*>(static_cast<T*>(e.y) + (row0 + r) * e.y_stride + col) =
                    make_uint4(o[0], o[1], o[2], o[3]);
        }
    } else if (col0 + lane < e.N) {
        // off 16-byte boundaries or at the last columns: a lane takes a column
        const float b = e.bias ? e.bias[col0 + lane] : 0.0f;
        const float* sums = reinterpret_cast<const float*>(turn);
        const int rows = static_cast<int>(min(e.M - row0, 32ll));
        T* y = static_cast<T*>(e.y) + row0 * e.y_stride + col0 + lane;
        const T* from = static_cast<const T*>(e.residual) + row0 * e.residual_stride + col0 + lane;
#pragma unroll 8
        for (int r = 0; r < rows; ++r) {
            float f = finish(sums[r * 32 + (((lane >> 2) ^ (r & 7)) << 2) + (lane & 3)], b);
            if (e.residual)
                f += D::load(from + r * e.residual_stride);
            y[r * e.y_stride] = D::pack(f);
        }
    }
    __syncwarp();
}

template <typename After>
__device__ __forceinline__ void mx_empty(const MxEpilogue& e, float4* turn, uint32_t taddr, long long row0, int col0,
                                         After&& after)
{
    if (e.y_dtype == kMxF16)
        mx_empty_chunk<kMxF16>(e, turn, taddr, row0, col0, after);
    else if (e.y_dtype == kMxBf16)
        mx_empty_chunk<kMxBf16>(e, turn, taddr, row0, col0, after);
    else
        mx_empty_chunk<kMxF32>(e, turn, taddr, row0, col0, after);
}

}  // namespace mlvc_b200
