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

__device__ __forceinline__ uint4 load16(const void* p)
{
    uint4 v;
    asm volatile("ld.global.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p) : "memory");
    return v;
}
__device__ __forceinline__ void store16(void* p, const uint4& v)
{
    asm volatile("st.global.v4.b32 [%0], {%1, %2, %3, %4};" ::"l"(p), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}

// A lane's part of 32 rows of y: a piece of 16 bytes (kCols columns) of each
// kCols-th row.  Warps work alone here, so what a chunk waits for one after the
// other is what it takes: addresses are made once for the rows, and all that a
// chunk reads is asked for before any of it is used.
template <int DT>
struct MxOut {
    using D = Dense<DT>;
    using T = typename D::T;
    static constexpr int kCols = DT == kMxF32 ? 4 : 8;
    static constexpr int kLanes = 32 / kCols;  // of a row
    static constexpr int kRounds = kLanes;     // each of kCols rows

    struct Asked {  // what a chunk needs from memory
        // residual: the lane's pieces, or, off 16-byte boundaries, 32 rows' values
        // of one column (16-bit: two a word)
        uint4 res[kRounds];
        float bias[kCols];
    };

    T* y;
    const T* res;
    long long y_step, res_step;  // bytes
    uint32_t there;              // bit i: the row of round i exists
    long long row0;
    int rows;

    // The value at p, 0 where it is not there: no branch and no conversion, so
    // that many can be under way.
    static __device__ __forceinline__ uint32_t bits(const T* p, bool there)
    {
        uint32_t v;
        if constexpr (DT == kMxF32)
            asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %2, 0;\n\tmov.b32 %0, 0;\n\t@p ld.global.b32 %0, [%1];\n\t}"
                         : "=&r"(v) : "l"(p), "r"(static_cast<int>(there)) : "memory");
        else
            asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %2, 0;\n\tmov.b32 %0, 0;\n\t@p ld.global.u16 %0, [%1];\n\t}"
                         : "=&r"(v) : "l"(p), "r"(static_cast<int>(there)) : "memory");
        return v;
    }

    // Rows row0 .. row0 + 32, none from `end` on.
    __device__ __forceinline__ void set_rows(const MxEpilogue& e, long long first, long long end)
    {
        const int sub = (threadIdx.x & 31) / kLanes;
        row0 = first;
        rows = static_cast<int>(max(min(end - first, 32ll), 0ll));
        y = static_cast<T*>(e.y) + (first + sub) * e.y_stride;
        res = static_cast<const T*>(e.residual) + (first + sub) * e.residual_stride;
        y_step = e.y_stride * (kCols * static_cast<long long>(sizeof(T)));
        res_step = e.residual_stride * (kCols * static_cast<long long>(sizeof(T)));
        there = 0;
#pragma unroll
        for (int i = 0; i < kRounds; ++i)
            there |= (sub + i * kCols < rows ? 1u : 0u) << i;
    }

    __device__ __forceinline__ void ask(const MxEpilogue& e, int col0, Asked& a) const
    {
        const int col = col0 + (threadIdx.x & 31) % kLanes * kCols;
        const bool wide = e.vec && col + kCols <= e.N;
        if (__all_sync(0xFFFFFFFFu, wide)) {
            const uint8_t* from = reinterpret_cast<const uint8_t*>(res + col);
#pragma unroll
            for (int i = 0; i < kRounds; ++i, from += res_step)
                a.res[i] = e.residual && (there >> i & 1u) ? load16(from) : make_uint4(0, 0, 0, 0);
        } else {
            const int lane = threadIdx.x & 31;
            const T* from = static_cast<const T*>(e.residual) + row0 * e.residual_stride + col0 + lane;
            const int n = e.residual && col0 + lane < e.N ? rows : 0;
            uint32_t* w = reinterpret_cast<uint32_t*>(a.res);
            uint32_t each[32];  // all under way before two become one
#pragma unroll
            for (int r = 0; r < 32; ++r, from += e.residual_stride)
                each[r] = bits(from, r < n);
#pragma unroll
            for (int r = 0; r < 32; ++r)
                if constexpr (DT == kMxF32)
                    w[r] = each[r];
                else if (r & 1)
                    w[r / 2] = each[r - 1] | each[r] << 16;
        }
#pragma unroll
        for (int k = 0; k < kCols; k += 4) {
            const uint4 b = e.bias && wide ? load16(e.bias + col + k) : make_uint4(0, 0, 0, 0);
            a.bias[k] = __uint_as_float(b.x);
            a.bias[k + 1] = __uint_as_float(b.y);
            a.bias[k + 2] = __uint_as_float(b.z);
            a.bias[k + 3] = __uint_as_float(b.w);
        }
    }

    // The chunk at `taddr` to columns col0 ...; `after` is called once the sums
    // are in registers.
    template <typename After>
    __device__ __forceinline__ void empty(const MxEpilogue& e, const Asked& a, float4* turn, uint32_t taddr, int col0,
                                          After&& after) const
    {
        const int lane = threadIdx.x & 31;
        const int col = col0 + lane % kLanes * kCols, sub = lane / kLanes;
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
        if (__all_sync(0xFFFFFFFFu, e.vec && col + kCols <= e.N)) {
            float f[kRounds][kCols];
#pragma unroll
            for (int i = 0; i < kRounds; ++i) {
                const int r = sub + i * kCols, q = lane % kLanes * (kCols / 4);
#pragma unroll
                for (int k = 0; k < kCols; k += 4) {
                    const float4 s = turn[r * 8 + ((q + k / 4) ^ (r & 7))];
                    f[i][k] = s.x;
                    f[i][k + 1] = s.y;
                    f[i][k + 2] = s.z;
                    f[i][k + 3] = s.w;
                }
            }
            uint8_t* to = reinterpret_cast<uint8_t*>(y + col);
#pragma unroll
            for (int i = 0; i < kRounds; ++i, to += y_step) {
#pragma unroll
                for (int k = 0; k < kCols; ++k)
                    f[i][k] = finish(f[i][k], a.bias[k]);
                const uint32_t u[4] = {a.res[i].x, a.res[i].y, a.res[i].z, a.res[i].w};
                uint32_t o[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    if constexpr (DT == kMxF32) {
                        o[k] = __float_as_uint(f[i][k] + __uint_as_float(u[k]));
                    } else {
                        float r0, r1;
                        D::unpack(u[k], r0, r1);
                        o[k] = D::pack2(f[i][2 * k] + r0, f[i][2 * k + 1] + r1);
                    }
                }
                if (there >> i & 1u)
                    store16(to, make_uint4(o[0], o[1], o[2], o[3]));
            }
        } else if (col0 + lane < e.N) {
            // off 16-byte boundaries or at the last columns: a lane takes a column
            const float b = e.bias ? e.bias[col0 + lane] : 0.0f;
            const float* sums = reinterpret_cast<const float*>(turn);
            const uint32_t* w = reinterpret_cast<const uint32_t*>(a.res);
            T* to = static_cast<T*>(e.y) + row0 * e.y_stride + col0 + lane;
#pragma unroll
            for (int r = 0; r < 32; ++r, to += e.y_stride) {
                float g = finish(sums[r * 32 + (((lane >> 2) ^ (r & 7)) << 2) + (lane & 3)], b);
                if constexpr (DT == kMxF32) {
                    g += __uint_as_float(w[r]);
                } else {
                    float lo, hi;
                    D::unpack(w[r / 2], lo, hi);
                    g += r & 1 ? hi : lo;
                }
                if (r < rows)
                    *to = D::pack(g);
            }
        }
        __syncwarp();
    }
};

template <int DT>
struct MxType {
    static constexpr int value = DT;
};

// fn(MxType<DT>) of y's type.
template <typename Fn>
__device__ __forceinline__ void mx_by_type(int y_dtype, Fn&& fn)
{
    if (y_dtype == kMxF16)
        fn(MxType<kMxF16>{});
    else if (y_dtype == kMxBf16)
        fn(MxType<kMxBf16>{});
    else
        fn(MxType<kMxF32>{});
}

}  // namespace mlvc_b200
