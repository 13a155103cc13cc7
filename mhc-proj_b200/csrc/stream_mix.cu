// The residual update of an mHC layer with n = 4 streams, forward and
// backward: per token, with T its 4x4 mixing matrix (a projection's output),
// h its four output weights and y the sublayer's output,
//   X'[i] = sum_j T[i, j] X[j] + h[i] drop(y)
// and given G = dL/dX'
//   dX[j] = sum_i T[i, j] G[i]         dT[i, j] = sum_c G[i] X[j]
//   dy = drop(sum_i h[i] G[i])         dh[i] = sum_c G[i] drop(y)
// drop is dropout.cu's with the element's index in the (tokens, C) array y, so
// the fused form is the composition with dropout's output left unrounded.
// Arithmetic and sums are fp32; outputs are rounded once.
#include <algorithm>

#include "philox.cuh"
#include "row_ops.cuh"

namespace mhcp {

constexpr int kMixBlock = 256;

template <class Elem>
struct MixIn {
    const Elem* x;
    int64_t stride, stream_stride;
    const Elem* y;
    int64_t y_stride;
    const void *T, *h;
    int T_dtype, h_dtype;
};

// A token's coefficients.
struct MixCoef {
    float t[16], h[4];
};

template <class Elem>
__device__ __forceinline__ MixCoef mix_coef(const MixIn<Elem>& in, int64_t r)
{
    MixCoef k;
#pragma unroll
    for (int i = 0; i < 16; ++i) k.t[i] = load_any(in.T, 16 * r + i, in.T_dtype);
#pragma unroll
    for (int i = 0; i < 4; ++i) k.h[i] = load_any(in.h, 4 * r + i, in.h_dtype);
    return k;
}

// drop's factor of element e.
__device__ __forceinline__ float drop_factor(int64_t e, const Dropout& d, uint2 key)
{
    if (!d.limit) return 1.0f;
    return (keep_bits(e >> 3, d.offset, key, d.limit) >> (e & 7) & 1) ? d.scale : 0.0f;
}

template <class Elem>
__global__ void __launch_bounds__(kMixBlock)
mix_fwd_rows(MixIn<Elem> in, Elem* __restrict__ out, Dropout d, int64_t N, int64_t C)
{
    const uint2 key = dropout_key(d);
    for (int64_t r = blockIdx.x; r < N; r += gridDim.x) {
        const MixCoef k = mix_coef(in, r);
        const Elem* x = in.x + r * in.stride;
        for (int64_t c = threadIdx.x; c < C; c += kMixBlock) {
            const float f = drop_factor(r * C + c, d, key);
            const float y = f != 0.0f ? to_f32(in.y[r * in.y_stride + c]) * f : 0.0f;
            float v[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] = to_f32(x[j * in.stream_stride + c]);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float s = k.h[i] * y;
#pragma unroll
                for (int j = 0; j < 4; ++j) s = fmaf(k.t[4 * i + j], v[j], s);
                out[(4 * r + i) * C + c] = from_f32<Elem>(s);
            }
        }
    }
}

template <class Elem>
__global__ void __launch_bounds__(kMixBlock)
mix_bwd_rows(const Elem* __restrict__ g, int64_t g_stride, int64_t g_stream_stride, MixIn<Elem> in,
             Elem* __restrict__ dx, void* __restrict__ dT, Elem* __restrict__ dy, void* __restrict__ dh, Dropout d,
             int64_t N, int64_t C)
{
    __shared__ float buf[20 * kMixBlock / 32];
    const uint2 key = dropout_key(d);
    for (int64_t r = blockIdx.x; r < N; r += gridDim.x) {
        const MixCoef k = mix_coef(in, r);
        const Elem* x = in.x + r * in.stride;
        const Elem* gr = g + r * g_stride;
        float acc[20];
#pragma unroll
        for (int i = 0; i < 20; ++i) acc[i] = 0.0f;
        for (int64_t c = threadIdx.x; c < C; c += kMixBlock) {
            const float f = drop_factor(r * C + c, d, key);
            const float y = f != 0.0f ? to_f32(in.y[r * in.y_stride + c]) * f : 0.0f;
            float v[4], gv[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                v[j] = to_f32(x[j * in.stream_stride + c]);
                gv[j] = to_f32(gr[j * g_stream_stride + c]);
            }
            float s = 0.0f;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                s = fmaf(k.h[i], gv[i], s);
                acc[16 + i] = fmaf(gv[i], y, acc[16 + i]);
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[4 * i + j] = fmaf(gv[i], v[j], acc[4 * i + j]);
            }
            dy[r * C + c] = from_f32<Elem>(f != 0.0f ? s * f : 0.0f);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                float t = 0.0f;
#pragma unroll
                for (int i = 0; i < 4; ++i) t = fmaf(k.t[4 * i + j], gv[i], t);
                dx[(4 * r + j) * C + c] = from_f32<Elem>(t);
            }
        }
        block_sum(acc, buf);
        if (threadIdx.x == 0) {
#pragma unroll
            for (int i = 0; i < 16; ++i) store_any(dT, 16 * r + i, in.T_dtype, acc[i]);
#pragma unroll
            for (int i = 0; i < 4; ++i) store_any(dh, 4 * r + i, in.h_dtype, acc[16 + i]);
        }
        __syncthreads();  // buf is written again
    }
}

constexpr int64_t kMaxMixGrid = int64_t{1} << 20;

template <class Elem>
static int mix_forward(const MixIn<Elem>& in, void* out, const Dropout& d, int64_t N, int64_t C, cudaStream_t stream)
{
    mix_fwd_rows<Elem><<<static_cast<unsigned>(std::min(N, kMaxMixGrid)), kMixBlock, 0, stream>>>(
        in, static_cast<Elem*>(out), d, N, C);
    return static_cast<int>(cudaGetLastError());
}

template <class Elem>
static int mix_backward(const void* g, int64_t g_stride, int64_t g_stream_stride, const MixIn<Elem>& in, void* dx,
                        void* dT, void* dy, void* dh, const Dropout& d, int64_t N, int64_t C, cudaStream_t stream)
{
    mix_bwd_rows<Elem><<<static_cast<unsigned>(std::min(N, kMaxMixGrid)), kMixBlock, 0, stream>>>(
        static_cast<const Elem*>(g), g_stride, g_stream_stride, in, static_cast<Elem*>(dx), dT,
        static_cast<Elem*>(dy), dh, d, N, C);
    return static_cast<int>(cudaGetLastError());
}

static bool mix_args_ok(const void* X, int64_t token_stride, int64_t stream_stride, const void* y, int64_t y_stride,
                        int dtype, const void* T, int T_dtype, const void* h, int h_dtype, double p, int64_t N,
                        int64_t C)
{
    return N >= 0 && C >= 1 && token_stride >= 0 && stream_stride >= 0 && y_stride >= 0 && known_dtype(dtype) &&
           known_dtype(T_dtype) && known_dtype(h_dtype) && p >= 0.0 && p <= 1.0 && (N == 0 || (X && y && T && h));
}

}  // namespace mhcp

using namespace mhcp;

extern "C" int mhc_stream_mix_n4(const void* d_X, int64_t token_stride, int64_t stream_stride, const void* d_y,
                                 int64_t y_stride, int dtype, const void* d_T, int T_dtype, const void* d_h,
                                 int h_dtype, void* d_out, double p, int64_t seed, const int64_t* d_seed,
                                 int64_t offset, int64_t N, int64_t C, cudaStream_t stream)
{
    if (!mix_args_ok(d_X, token_stride, stream_stride, d_y, y_stride, dtype, d_T, T_dtype, d_h, h_dtype, p, N, C) ||
        (N > 0 && !d_out))
        return MHC_ERR_INVALID_VALUE;
    if (N == 0) return MHC_OK;
    const Dropout d = make_dropout(p, seed, d_seed, offset);
    auto run = [&](auto elem) {
        using Elem = decltype(elem);
        const MixIn<Elem> in{static_cast<const Elem*>(d_X), token_stride, stream_stride, static_cast<const Elem*>(d_y),
                             y_stride, d_T, d_h, T_dtype, h_dtype};
        return mix_forward(in, d_out, d, N, C, stream);
    };
    switch (dtype) {
        case MHC_DTYPE_BF16: return run(__nv_bfloat16{});
        case MHC_DTYPE_F16: return run(__half{});
        default: return run(float{});
    }
}

extern "C" int mhc_stream_mix_n4_backward(const void* d_G, int64_t g_token_stride, int64_t g_stream_stride,
                                          const void* d_X, int64_t token_stride, int64_t stream_stride,
                                          const void* d_y, int64_t y_stride, int dtype, const void* d_T, int T_dtype,
                                          const void* d_h, int h_dtype, void* d_dX, void* d_dT, void* d_dy, void* d_dh,
                                          double p, int64_t seed, const int64_t* d_seed, int64_t offset, int64_t N,
                                          int64_t C, cudaStream_t stream)
{
    if (!mix_args_ok(d_X, token_stride, stream_stride, d_y, y_stride, dtype, d_T, T_dtype, d_h, h_dtype, p, N, C) ||
        g_token_stride < 0 || g_stream_stride < 0 || (N > 0 && (!d_G || !d_dX || !d_dT || !d_dy || !d_dh)))
        return MHC_ERR_INVALID_VALUE;
    if (N == 0) return MHC_OK;
    const Dropout d = make_dropout(p, seed, d_seed, offset);
    auto run = [&](auto elem) {
        using Elem = decltype(elem);
        const MixIn<Elem> in{static_cast<const Elem*>(d_X), token_stride, stream_stride, static_cast<const Elem*>(d_y),
                             y_stride, d_T, d_h, T_dtype, h_dtype};
        return mix_backward(d_G, g_token_stride, g_stream_stride, in, d_dX, d_dT, d_dy, d_dh, d, N, C, stream);
    };
    switch (dtype) {
        case MHC_DTYPE_BF16: return run(__nv_bfloat16{});
        case MHC_DTYPE_F16: return run(__half{});
        default: return run(float{});
    }
}
