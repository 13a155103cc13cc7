// A thread's kElems columns of a row that a group of threads holds: pieces of K
// columns, in pairs.  The forms of rows that the kernels are built for:
//   kLoose    any rows: single columns, a warp's threads next to each other
//   kSkewed   16-byte pieces as they lie in memory, where a row's first and
//             last piece may be shared with its neighbours.  For rows that lie
//             the same way in all of their tensors; a group takes rows that
//             lie `skew` elements into their first piece, all of them
//   kPieces   rows of whole, aligned pieces
//   kWhole    the same, and exactly as many as the group's threads take, so
//             that nothing is asked per piece
// What is not in the row reads as zero (or what the caller names) and is not
// written.
#pragma once

#include "ring_plan.h"
#include "row_ops.cuh"

namespace mhcp {

// An array of Param at single columns of a thread.
template <class Param, class Cols, int kPairs>
__device__ __forceinline__ void load_columns(const Cols& cols, int p, const void* a, float none, float2 (&v)[kPairs])
{
    const Param* q = static_cast<const Param*>(a);
#pragma unroll
    for (int i = 0; i < kPairs; ++i) {
        v[i].x = cols.in(p, 2 * i) ? to_f32(q[cols.col(p, 2 * i)]) : none;
        v[i].y = cols.in(p, 2 * i + 1) ? to_f32(q[cols.col(p, 2 * i + 1)]) : none;
    }
}

template <class Cols, int kPairs>
__device__ __forceinline__ void load_columns(const Cols& cols, int p, const void* a, int dtype, float none,
                                             float2 (&v)[kPairs])
{
    if (dtype == MHC_DTYPE_F32)
        load_columns<float>(cols, p, a, none, v);
    else if (dtype == MHC_DTYPE_BF16)
        load_columns<__nv_bfloat16>(cols, p, a, none, v);
    else
        load_columns<__half>(cols, p, a, none, v);
}

template <class Elem, RowForm kForm, int kElems>
struct RowCols {  // in pieces
    static constexpr int K = 16 / sizeof(Elem);
    int C, t, threads, skew;
    int end;     // elements of the last piece, where they are not all of it
    bool edge;   // one of this thread's pieces is only partly in the row

    __device__ __forceinline__ RowCols(int width, int thread, int of, int skewed)
        : C(width), t(thread), threads(of), skew(kForm == kSkewed ? skewed : 0), end(0), edge(false)
    {
        if constexpr (kForm == kSkewed) {
            end = (C + skew) % K;
            edge = (t == 0 && skew) || last();
        }
    }
    // Whether the last piece is this thread's and not whole.
    __device__ __forceinline__ bool last() const { return end && t == (C + skew) / K % threads; }
    __device__ __forceinline__ int col(int p, int j) const
    {
        return (p * threads + t) * K + j - (kForm == kSkewed ? skew : 0);
    }
    // Whether something of piece p is in the row, and whether all of it is.
    __device__ __forceinline__ bool has(int p) const { return kForm == kWhole || col(p, 0) < C; }
    __device__ __forceinline__ bool all(int p) const
    {
        return kForm != kSkewed || (col(p, 0) >= 0 && col(p, 0) + K <= C);
    }
    __device__ __forceinline__ bool in(int p, int j) const
    {
        if constexpr (kForm != kSkewed) return has(p);
        return static_cast<unsigned>(col(p, j)) < static_cast<unsigned>(C);
    }

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
        if (!has(p)) return;
        if (!edge || all(p)) {
            *reinterpret_cast<uint4*>(row + col(p, 0)) = piece_of<Elem>(v);
        } else {
#pragma unroll
            for (int j = 0; j < K; ++j)
                if (in(p, j)) row[col(p, j)] = from_f32<Elem>(j & 1 ? v[j / 2].y : v[j / 2].x);
        }
    }
    // A norm's weight or bias: in pieces of the rows' own type or fp32, aligned (the launcher's rule).
    __device__ __forceinline__ void param(int p, const void* a, int dtype, float none, float2 (&v)[K / 2]) const
    {
        if (!a) {
#pragma unroll
            for (int i = 0; i < K / 2; ++i) v[i] = both(none);
        } else if constexpr (kForm == kSkewed) {
            load_columns(*this, p, a, dtype, none, v);
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
    __device__ __forceinline__ void clear_rest(int p, float2 (&v)[K / 2]) const
    {
        if constexpr (kForm == kWhole) return;
        if (has(p) && (!edge || all(p))) return;
#pragma unroll
        for (int i = 0; i < K / 2; ++i) {
            if (!in(p, 2 * i)) v[i].x = 0.0f;
            if (!in(p, 2 * i + 1)) v[i].y = 0.0f;
        }
    }
};

template <class Elem, int kElems>
struct RowCols<Elem, kLoose, kElems> {
    static constexpr int K = 8;
    int C, t, threads;
    int first, rest;  // this thread's first column, and the row's columns from there

    __device__ __forceinline__ RowCols(int width, int thread, int of, int)
        : C(width), t(thread), threads(of), first((thread >> 5) * (32 * kElems) + (thread & 31)), rest(width - first)
    {
    }
    // a warp's columns are next to each other, a thread's 32 apart
    __device__ __forceinline__ int col(int p, int j) const { return first + (p * K + j) * 32; }
    __device__ __forceinline__ bool in(int p, int j) const { return (p * K + j) * 32 < rest; }

    __device__ __forceinline__ void load(int p, const Elem* row, float2 (&v)[K / 2]) const
    {
#pragma unroll
        for (int i = 0; i < K / 2; ++i) {
            v[i].x = in(p, 2 * i) ? to_f32((row + first)[(p * K + 2 * i) * 32]) : 0.0f;
            v[i].y = in(p, 2 * i + 1) ? to_f32((row + first)[(p * K + 2 * i + 1) * 32]) : 0.0f;
        }
    }
    __device__ __forceinline__ void store(int p, Elem* __restrict__ row, const float2 (&v)[K / 2]) const
    {
#pragma unroll
        for (int i = 0; i < K / 2; ++i) {
            if (in(p, 2 * i)) (row + first)[(p * K + 2 * i) * 32] = from_f32<Elem>(v[i].x);
            if (in(p, 2 * i + 1)) (row + first)[(p * K + 2 * i + 1) * 32] = from_f32<Elem>(v[i].y);
        }
    }
    __device__ __forceinline__ void param(int p, const void* a, int dtype, float none, float2 (&v)[K / 2]) const
    {
        if (a) {
            load_columns(*this, p, a, dtype, none, v);
        } else {
#pragma unroll
            for (int i = 0; i < K / 2; ++i) v[i] = both(none);
        }
    }
    __device__ __forceinline__ void clear_rest(int p, float2 (&v)[K / 2]) const
    {
#pragma unroll
        for (int i = 0; i < K / 2; ++i) {
            if (!in(p, 2 * i)) v[i].x = 0.0f;
            if (!in(p, 2 * i + 1)) v[i].y = 0.0f;
        }
    }
};

}  // namespace mhcp
