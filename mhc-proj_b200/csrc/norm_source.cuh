// What the layer norm kernels share.
#pragma once

#include "row_ops.cuh"

namespace mhcp {

// Where a row's u comes from: one row, or four weighted ones.
template <class Elem, int kStreams>
struct NormSource {
    const Elem* x;
    int64_t stride, stream_stride;
    const void* h;
    int h_dtype;
};

template <class Elem, int kStreams>
struct NormRow {
    const Elem* x;
    int64_t stream_stride;
    float h[kStreams];

    NormRow() = default;
    __device__ __forceinline__ NormRow(const NormSource<Elem, kStreams>& s, int64_t r)
        : x(s.x + r * s.stride), stream_stride(s.stream_stride)
    {
        if constexpr (kStreams == 1) {
            h[0] = 1.0f;
        } else {
#pragma unroll
            for (int i = 0; i < kStreams; ++i) h[i] = load_any(s.h, r * kStreams + i, s.h_dtype);
        }
    }

    __device__ __forceinline__ float at(int64_t c) const
    {
        if constexpr (kStreams == 1) return to_f32(x[c]);
        float u = 0.0f;
#pragma unroll
        for (int i = 0; i < kStreams; ++i) u = fmaf(h[i], to_f32(x[i * stream_stride + c]), u);
        return u;
    }
};

struct NormAffine {
    const void *w, *b;
    int dtype;
};

}  // namespace mhcp
