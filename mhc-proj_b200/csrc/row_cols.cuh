// A thread's columns of a row that a group of threads holds: pieces p of K
// columns, in pairs.
//   VecCols     16-byte pieces, the group's next to each other.  For rows whose
//               starts are 16-byte aligned and whose width is whole pieces (kFull:
//               all the pieces that the group's threads take).
//   LooseCols   single columns, the group's threads next to each other; any
//               width and alignment, each column in the row or not.
// What is not in the row reads as zero (or what the caller names) and is not
// written.
#pragma once

#include "row_ops.cuh"

namespace mhcp {

template <class Elem, bool kFull>
struct VecCols {
    static constexpr bool kVec = true;
    static constexpr int K = 16 / sizeof(Elem);
    int C, t, threads;

    __device__ __forceinline__ int col(int p, int j) const { return (p * threads + t) * K + j; }
    __device__ __forceinline__ bool has(int p, int = 0) const { return kFull || col(p, 0) < C; }

    static __device__ __forceinline__ void unpack(const uint4& q, float2 (&v)[K / 2])
    {
#pragma unroll
        for (int i = 0; i < K / 2; ++i) v[i] = pair_of<Elem>(q, i);
    }

    __device__ __forceinline__ void load(int p, const Elem* __restrict__ row, float2 (&v)[K / 2]) const
    {
        unpack(has(p) ? __ldg(reinterpret_cast<const uint4*>(row + col(p, 0))) : make_uint4(0, 0, 0, 0), v);
    }

    __device__ __forceinline__ void store(int p, Elem* __restrict__ row, const float2 (&v)[K / 2]) const
    {
        const uint4 q = piece_of<Elem>(v);
        if (has(p)) *reinterpret_cast<uint4*>(row + col(p, 0)) = q;
    }

    // A norm's weight or bias: of the rows' own type or fp32, aligned (the launcher's rule).
    __device__ __forceinline__ void param(int p, const void* a, int dtype, float none, float2 (&v)[K / 2]) const
    {
        if (!a) {
#pragma unroll
            for (int i = 0; i < K / 2; ++i) v[i] = both(none);
        } else if (sizeof(Elem) == 4 || dtype != MHC_DTYPE_F32) {
            load(p, static_cast<const Elem*>(a), v);
        } else {
            const float4* q = reinterpret_cast<const float4*>(static_cast<const float*>(a) + col(p, 0));
#pragma unroll
            for (int i = 0; i < K / 4; ++i) {
                const float4 f = has(p) ? __ldg(q + i) : make_float4(0, 0, 0, 0);
                v[2 * i] = make_float2(f.x, f.y);
                v[2 * i + 1] = make_float2(f.z, f.w);
            }
        }
    }

    // Pairs of v that are in the row, the others zero.
    __device__ __forceinline__ void clear_rest(int p, float2 (&v)[K / 2]) const
    {
#pragma unroll
        for (int i = 0; i < K / 2; ++i) v[i] = has(p) ? v[i] : both(0.0f);
    }
    // Sum of squares of the pairs that are in the row.
    __device__ __forceinline__ float2 squares(int p, const float2 (&v)[K / 2], float2 sum) const
    {
        float2 d = both(0.0f);
#pragma unroll
        for (int i = 0; i < K / 2; ++i) d = fma2(v[i], v[i], d);
        return has(p) ? add2(sum, d) : sum;
    }
};

template <class Elem>
struct LooseCols {
    static constexpr bool kVec = false;
    static constexpr int K = 8;
    int C, t, threads;

    __device__ __forceinline__ int col(int p, int j) const { return (p * K + j) * threads + t; }
    __device__ __forceinline__ bool has(int p, int j) const { return col(p, j) < C; }

    __device__ __forceinline__ void load(int p, const Elem* row, float2 (&v)[K / 2]) const
    {
#pragma unroll
        for (int i = 0; i < K / 2; ++i) {
            v[i].x = has(p, 2 * i) ? to_f32(row[col(p, 2 * i)]) : 0.0f;
            v[i].y = has(p, 2 * i + 1) ? to_f32(row[col(p, 2 * i + 1)]) : 0.0f;
        }
    }

    __device__ __forceinline__ void store(int p, Elem* __restrict__ row, const float2 (&v)[K / 2]) const
    {
#pragma unroll
        for (int i = 0; i < K / 2; ++i) {
            if (has(p, 2 * i)) row[col(p, 2 * i)] = from_f32<Elem>(v[i].x);
            if (has(p, 2 * i + 1)) row[col(p, 2 * i + 1)] = from_f32<Elem>(v[i].y);
        }
    }

    __device__ __forceinline__ void param(int p, const void* a, int dtype, float none, float2 (&v)[K / 2]) const
    {
#pragma unroll
        for (int i = 0; i < K / 2; ++i) {
            v[i].x = a && has(p, 2 * i) ? load_any(a, col(p, 2 * i), dtype) : none;
            v[i].y = a && has(p, 2 * i + 1) ? load_any(a, col(p, 2 * i + 1), dtype) : none;
        }
    }

    __device__ __forceinline__ void clear_rest(int p, float2 (&v)[K / 2]) const
    {
#pragma unroll
        for (int i = 0; i < K / 2; ++i) {
            if (!has(p, 2 * i)) v[i].x = 0.0f;
            if (!has(p, 2 * i + 1)) v[i].y = 0.0f;
        }
    }
    __device__ __forceinline__ float2 squares(int p, const float2 (&v)[K / 2], float2 sum) const
    {
#pragma unroll
        for (int i = 0; i < K / 2; ++i) {
            const float2 d = make_float2(has(p, 2 * i) ? v[i].x : 0.0f, has(p, 2 * i + 1) ? v[i].y : 0.0f);
            sum = fma2(d, d, sum);
        }
        return sum;
    }
};

// The three forms that the kernels are built for.  kWhole: pieces, and exactly
// as many as the group's threads take, so that nothing is asked per piece.
enum RowForm { kLoose, kPieces, kWhole };

template <class Elem, RowForm kForm>
using RowCols = typename std::conditional<kForm == kLoose, LooseCols<Elem>, VecCols<Elem, kForm == kWhole>>::type;

}  // namespace mhcp
