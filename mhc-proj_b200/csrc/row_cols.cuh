// A thread's columns of a row that a group of threads holds: P pieces of K
// columns, in pairs.  The forms of rows that the kernels are built for:
//   kLoose    any rows: single columns, the group's threads next to each other
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

#include "row_ops.cuh"

namespace mhcp {

enum RowForm { kLoose, kSkewed, kPieces, kWhole };

template <class Elem, RowForm kForm>
struct RowCols {  // in pieces
    static constexpr int K = 16 / sizeof(Elem);
    int C, t, threads, skew;

    __device__ __forceinline__ RowCols(int width, int thread, int of, int skewed)
        : C(width), t(thread), threads(of), skew(kForm == kSkewed ? skewed : 0)
    {
    }
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

    __device__ __forceinline__ void unpack(int p, const uint4& q, float2 (&v)[K / 2]) const
    {
#pragma unroll
        for (int i = 0; i < K / 2; ++i) v[i] = pair_of<Elem>(q, i);
        if constexpr (kForm == kSkewed) clear_rest(p, v);
    }
    __device__ __forceinline__ void load(int p, const Elem* __restrict__ row, float2 (&v)[K / 2]) const
    {
        unpack(p, has(p) ? __ldg(reinterpret_cast<const uint4*>(row + col(p, 0))) : make_uint4(0, 0, 0, 0), v);
    }
    __device__ __forceinline__ void store(int p, Elem* __restrict__ row, const float2 (&v)[K / 2]) const
    {
        if (!has(p)) return;
        if (all(p)) {
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
#pragma unroll
            for (int j = 0; j < K; ++j) {
                const float f = in(p, j) ? load_any(a, col(p, j), dtype) : none;
                (j & 1 ? v[j / 2].y : v[j / 2].x) = f;
            }
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
        if (has(p) && all(p)) return;
#pragma unroll
        for (int i = 0; i < K / 2; ++i) {
            if (!in(p, 2 * i)) v[i].x = 0.0f;
            if (!in(p, 2 * i + 1)) v[i].y = 0.0f;
        }
    }
};

template <class Elem>
struct RowCols<Elem, kLoose> {
    static constexpr int K = 8;
    int C, t, threads;
    int steps, mine;  // columns of the first and of this thread

    __device__ __forceinline__ RowCols(int width, int thread, int of, int)
        : C(width), t(thread), threads(of), steps((width + of - 1) / of), mine((width - thread + of - 1) / of)
    {
    }
    __device__ __forceinline__ int col(int p, int j) const { return (p * K + j) * threads + t; }
    __device__ __forceinline__ bool in(int p, int j) const { return p * K + j < mine; }

    __device__ __forceinline__ void load(int p, const Elem* row, float2 (&v)[K / 2]) const
    {
#pragma unroll
        for (int i = 0; i < K / 2; ++i) {
            v[i] = both(0.0f);
            if (p * K + 2 * i >= steps) continue;
            if (in(p, 2 * i)) v[i].x = to_f32(row[col(p, 2 * i)]);
            if (in(p, 2 * i + 1)) v[i].y = to_f32(row[col(p, 2 * i + 1)]);
        }
    }
    __device__ __forceinline__ void store(int p, Elem* __restrict__ row, const float2 (&v)[K / 2]) const
    {
#pragma unroll
        for (int i = 0; i < K / 2; ++i) {
            if (p * K + 2 * i >= steps) continue;
            if (in(p, 2 * i)) row[col(p, 2 * i)] = from_f32<Elem>(v[i].x);
            if (in(p, 2 * i + 1)) row[col(p, 2 * i + 1)] = from_f32<Elem>(v[i].y);
        }
    }
    __device__ __forceinline__ void param(int p, const void* a, int dtype, float none, float2 (&v)[K / 2]) const
    {
#pragma unroll
        for (int i = 0; i < K / 2; ++i) {
            v[i].x = a && in(p, 2 * i) ? load_any(a, col(p, 2 * i), dtype) : none;
            v[i].y = a && in(p, 2 * i + 1) ? load_any(a, col(p, 2 * i + 1), dtype) : none;
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
