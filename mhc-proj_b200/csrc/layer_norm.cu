// Layer norm of rows, and of the weighted sum of a token's four residual
// streams, forward and backward.
//
//   u = x                              (layer_norm)
//   u = sum_i h[i] X[i]                (stream_norm_n4; never in memory)
//   mean = sum(u) / C,  rstd = 1 / sqrt(sum((u - mean)^2) / C + eps)
//   y = (u - mean) rstd w + b
// Backward, with xhat = (u - mean) rstd and gw = g w:
//   du = rstd (gw - sum(gw) / C - xhat sum(gw xhat) / C)
//   dw = sum over rows of g xhat,  db = sum over rows of g
//   dX[i] = h[i] du,  dh[i] = sum(du X[i])
// Sums are fp32 whatever the storage type; the variance is the mean of the
// squared distances from the mean (never a difference of squares, which
// cancels for rows far from zero).
#include <algorithm>

#include "row_ops.cuh"

namespace mhcp {

constexpr int kNormBlock = 256;

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

// One block per row, which it reads three times (the second and third come
// from L1 or L2).
template <class Elem, int kStreams>
__global__ void __launch_bounds__(kNormBlock)
norm_fwd_rows(NormSource<Elem, kStreams> src, NormAffine aff, Elem* __restrict__ y, float* __restrict__ mean_out,
              float* __restrict__ rstd_out, float eps, int64_t N, int64_t C)
{
    __shared__ float buf[2][kNormBlock / 32];
    for (int64_t r = blockIdx.x; r < N; r += gridDim.x) {
        const NormRow<Elem, kStreams> row(src, r);
        float s[1] = {0.0f};
        for (int64_t c = threadIdx.x; c < C; c += kNormBlock) s[0] += row.at(c);
        block_sum(s, buf[0]);
        const float mean = s[0] / static_cast<float>(C);
        s[0] = 0.0f;
        for (int64_t c = threadIdx.x; c < C; c += kNormBlock) {
            const float d = row.at(c) - mean;
            s[0] = fmaf(d, d, s[0]);
        }
        block_sum(s, buf[1]);
        const float rstd = 1.0f / sqrtf(s[0] / static_cast<float>(C) + eps);
        for (int64_t c = threadIdx.x; c < C; c += kNormBlock) {
            float v = (row.at(c) - mean) * rstd;
            if (aff.w) v *= load_any(aff.w, c, aff.dtype);
            if (aff.b) v += load_any(aff.b, c, aff.dtype);
            y[r * C + c] = from_f32<Elem>(v);
        }
        if (threadIdx.x == 0) {
            if (mean_out) mean_out[r] = mean;
            if (rstd_out) rstd_out[r] = rstd;
        }
    }
}

template <class Elem, int kStreams>
__global__ void __launch_bounds__(kNormBlock)
norm_bwd_rows(const Elem* __restrict__ g, int64_t g_stride, NormSource<Elem, kStreams> src,
              const float* __restrict__ mean_in, const float* __restrict__ rstd_in, NormAffine aff,
              Elem* __restrict__ dx, void* __restrict__ dh, int64_t N, int64_t C)
{
    __shared__ float buf[2 * kNormBlock / 32];
    __shared__ float buf_h[4 * kNormBlock / 32];
    for (int64_t r = blockIdx.x; r < N; r += gridDim.x) {
        const NormRow<Elem, kStreams> row(src, r);
        const Elem* gr = g + r * g_stride;
        const float mean = mean_in[r], rstd = rstd_in[r];
        float s[2] = {0.0f, 0.0f};
        for (int64_t c = threadIdx.x; c < C; c += kNormBlock) {
            const float gw = to_f32(gr[c]) * (aff.w ? load_any(aff.w, c, aff.dtype) : 1.0f);
            s[0] += gw;
            s[1] = fmaf(gw, (row.at(c) - mean) * rstd, s[1]);
        }
        block_sum(s, buf);
        const float m1 = s[0] / static_cast<float>(C), m2 = s[1] / static_cast<float>(C);
        float a[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        for (int64_t c = threadIdx.x; c < C; c += kNormBlock) {
            const float gw = to_f32(gr[c]) * (aff.w ? load_any(aff.w, c, aff.dtype) : 1.0f);
            const float du = rstd * (gw - m1 - (row.at(c) - mean) * rstd * m2);
            if constexpr (kStreams == 1) {
                dx[r * C + c] = from_f32<Elem>(du);
            } else {
#pragma unroll
                for (int i = 0; i < kStreams; ++i) {
                    a[i] = fmaf(du, to_f32(row.x[i * row.stream_stride + c]), a[i]);
                    dx[(r * kStreams + i) * C + c] = from_f32<Elem>(row.h[i] * du);
                }
            }
        }
        if constexpr (kStreams > 1) {
            block_sum(a, buf_h);
            if (threadIdx.x == 0) {
#pragma unroll
                for (int i = 0; i < kStreams; ++i) store_any(dh, r * kStreams + i, src.h_dtype, a[i]);
            }
        }
        __syncthreads();  // buf is written again
    }
}

// Partial sums of dw and db over one chunk of rows: partials[chunk][0 or 1][C].
constexpr int kParamRows = 8;  // rows a block works on at once, 32 columns wide

template <class Elem, int kStreams>
__global__ void __launch_bounds__(32 * kParamRows)
norm_param_partials(const Elem* __restrict__ g, int64_t g_stride, NormSource<Elem, kStreams> src,
                    const float* __restrict__ mean_in, const float* __restrict__ rstd_in, float* __restrict__ partials,
                    int64_t N, int64_t C, int64_t chunk_rows)
{
    __shared__ float part[2][kParamRows][32];
    const int lane = threadIdx.x & 31, line = threadIdx.x >> 5;
    const int64_t chunk = blockIdx.y, end = min(N, (chunk + 1) * chunk_rows);
    for (int64_t c0 = static_cast<int64_t>(blockIdx.x) * 32; c0 < C; c0 += static_cast<int64_t>(gridDim.x) * 32) {
        const int64_t c = c0 + lane;
        float dw = 0.0f, db = 0.0f;
        if (c < C) {
            for (int64_t r = chunk * chunk_rows + line; r < end; r += kParamRows) {
                const NormRow<Elem, kStreams> row(src, r);
                const float gv = to_f32(g[r * g_stride + c]);
                dw = fmaf(gv, (row.at(c) - mean_in[r]) * rstd_in[r], dw);
                db += gv;
            }
        }
        part[0][line][lane] = dw;
        part[1][line][lane] = db;
        __syncthreads();
        if (line < 2 && c < C) {
            float v = part[line][0][lane];
#pragma unroll
            for (int k = 1; k < kParamRows; ++k) v += part[line][k][lane];
            partials[(chunk * 2 + line) * C + c] = v;
        }
        __syncthreads();
    }
}

// dw and db from `rows` rows of partial sums.
__global__ void __launch_bounds__(32 * kParamRows)
norm_param_fold(const float* __restrict__ partials, int64_t rows, void* __restrict__ dw, void* __restrict__ db,
                int dtype, int64_t C)
{
    __shared__ float part[kParamRows][32];
    const int lane = threadIdx.x & 31, line = threadIdx.x >> 5;
    void* out = blockIdx.y == 0 ? dw : db;
    if (!out) return;
    for (int64_t c0 = static_cast<int64_t>(blockIdx.x) * 32; c0 < C; c0 += static_cast<int64_t>(gridDim.x) * 32) {
        const int64_t c = c0 + lane;
        float v = 0.0f;
        if (c < C) {
            for (int64_t k = line; k < rows; k += kParamRows) v += partials[(k * 2 + blockIdx.y) * C + c];
        }
        part[line][lane] = v;
        __syncthreads();
        if (line == 0 && c < C) {
#pragma unroll
            for (int k = 1; k < kParamRows; ++k) v += part[k][lane];
            store_any(out, c, dtype, v);
        }
        __syncthreads();
    }
}

constexpr int64_t kMaxRowGrid = int64_t{1} << 20;
constexpr int64_t kParamChunks = 64;

static int64_t norm_workspace(int64_t N, int64_t C)
{
    return std::max<int64_t>(1, std::min(ceil_div(N, kParamRows), kParamChunks)) * 2 * C *
           static_cast<int64_t>(sizeof(float));
}

template <class Elem, int kStreams>
static int norm_forward(const void* x, int64_t stride, int64_t stream_stride, const void* h, int h_dtype,
                        const NormAffine& aff, void* y, float* mean, float* rstd, float eps, int64_t N, int64_t C,
                        cudaStream_t stream)
{
    const NormSource<Elem, kStreams> src{static_cast<const Elem*>(x), stride, stream_stride, h, h_dtype};
    norm_fwd_rows<Elem, kStreams><<<static_cast<unsigned>(std::min(N, kMaxRowGrid)), kNormBlock, 0, stream>>>(
        src, aff, static_cast<Elem*>(y), mean, rstd, eps, N, C);
    return static_cast<int>(cudaGetLastError());
}

template <int kStreams>
static int norm_forward(const void* x, int64_t stride, int64_t stream_stride, int dtype, const void* h, int h_dtype,
                        const void* w, const void* b, int w_dtype, void* y, float* mean, float* rstd, float eps,
                        int64_t N, int64_t C, cudaStream_t stream)
{
    if (N < 0 || C < 1 || stride < 0 || stream_stride < 0 || !known_dtype(dtype) || !known_dtype(h_dtype) ||
        !known_dtype(w_dtype) || !(eps >= 0.0f) || (N > 0 && (!x || !y || (kStreams > 1 && !h))))
        return MHC_ERR_INVALID_VALUE;
    if (N == 0) return MHC_OK;
    const NormAffine aff{w, b, w_dtype};
    switch (dtype) {
        case MHC_DTYPE_BF16:
            return norm_forward<__nv_bfloat16, kStreams>(x, stride, stream_stride, h, h_dtype, aff, y, mean, rstd, eps,
                                                         N, C, stream);
        case MHC_DTYPE_F16:
            return norm_forward<__half, kStreams>(x, stride, stream_stride, h, h_dtype, aff, y, mean, rstd, eps, N, C,
                                                  stream);
        default:
            return norm_forward<float, kStreams>(x, stride, stream_stride, h, h_dtype, aff, y, mean, rstd, eps, N, C,
                                                 stream);
    }
}

template <class Elem, int kStreams>
static int norm_backward(const void* g, int64_t g_stride, const void* x, int64_t stride, int64_t stream_stride,
                         const void* h, int h_dtype, const float* mean, const float* rstd, const NormAffine& aff,
                         void* dx, void* dh, void* dw, void* db, int64_t N, int64_t C, float* partials,
                         cudaStream_t stream)
{
    const NormSource<Elem, kStreams> src{static_cast<const Elem*>(x), stride, stream_stride, h, h_dtype};
    const Elem* gp = static_cast<const Elem*>(g);
    if (N > 0)
        norm_bwd_rows<Elem, kStreams><<<static_cast<unsigned>(std::min(N, kMaxRowGrid)), kNormBlock, 0, stream>>>(
            gp, g_stride, src, mean, rstd, aff, static_cast<Elem*>(dx), dh, N, C);
    if (dw || db) {
        const unsigned cols = static_cast<unsigned>(std::min<int64_t>(ceil_div(C, 32), int64_t{1} << 20));
        int64_t chunks = 0;
        if (N > 0) {
            chunks = std::min(ceil_div(N, kParamRows), kParamChunks);
            const int64_t chunk_rows = ceil_div(N, chunks);
            norm_param_partials<Elem, kStreams>
                <<<dim3(cols, static_cast<unsigned>(chunks)), 32 * kParamRows, 0, stream>>>(
                    gp, g_stride, src, mean, rstd, partials, N, C, chunk_rows);
        }
        norm_param_fold<<<dim3(cols, 2), 32 * kParamRows, 0, stream>>>(partials, chunks, dw, db, aff.dtype, C);
    }
    return static_cast<int>(cudaGetLastError());
}

template <int kStreams>
static int norm_backward(const void* g, int64_t g_stride, const void* x, int64_t stride, int64_t stream_stride,
                         int dtype, const void* h, int h_dtype, const float* mean, const float* rstd, const void* w,
                         int w_dtype, void* dx, void* dh, void* dw, void* db, int64_t N, int64_t C, void* workspace,
                         int64_t workspace_bytes, cudaStream_t stream)
{
    if (N < 0 || C < 1 || g_stride < 0 || stride < 0 || stream_stride < 0 || !known_dtype(dtype) ||
        !known_dtype(h_dtype) || !known_dtype(w_dtype) ||
        (N > 0 && (!g || !x || !mean || !rstd || !dx || (kStreams > 1 && (!h || !dh)))))
        return MHC_ERR_INVALID_VALUE;
    if (N > 0 && (dw || db) && (!workspace || workspace_bytes < norm_workspace(N, C))) return MHC_ERR_INVALID_VALUE;
    if (N == 0 && !dw && !db) return MHC_OK;
    const NormAffine aff{w, nullptr, w_dtype};
    float* partials = static_cast<float*>(workspace);
    switch (dtype) {
        case MHC_DTYPE_BF16:
            return norm_backward<__nv_bfloat16, kStreams>(g, g_stride, x, stride, stream_stride, h, h_dtype, mean, rstd,
                                                          aff, dx, dh, dw, db, N, C, partials, stream);
        case MHC_DTYPE_F16:
            return norm_backward<__half, kStreams>(g, g_stride, x, stride, stream_stride, h, h_dtype, mean, rstd, aff,
                                                   dx, dh, dw, db, N, C, partials, stream);
        default:
            return norm_backward<float, kStreams>(g, g_stride, x, stride, stream_stride, h, h_dtype, mean, rstd, aff, dx,
                                                  dh, dw, db, N, C, partials, stream);
    }
}

}  // namespace mhcp

using namespace mhcp;

extern "C" int mhc_layer_norm(const void* d_x, int64_t x_stride, int dtype, const void* d_w, const void* d_b,
                              int w_dtype, void* d_y, float* d_mean, float* d_rstd, float eps, int64_t N, int64_t C,
                              cudaStream_t stream)
{
    return norm_forward<1>(d_x, x_stride, 0, dtype, nullptr, MHC_DTYPE_F32, d_w, d_b, w_dtype, d_y, d_mean, d_rstd, eps,
                           N, C, stream);
}

extern "C" int mhc_layer_norm_backward_workspace(int64_t N, int64_t C, int64_t* bytes)
{
    if (N < 0 || C < 1 || !bytes) return MHC_ERR_INVALID_VALUE;
    *bytes = norm_workspace(N, C);
    return MHC_OK;
}

extern "C" int mhc_layer_norm_backward(const void* d_g, int64_t g_stride, const void* d_x, int64_t x_stride, int dtype,
                                       const float* d_mean, const float* d_rstd, const void* d_w, int w_dtype,
                                       void* d_dx, void* d_dw, void* d_db, int64_t N, int64_t C, void* d_workspace,
                                       int64_t workspace_bytes, cudaStream_t stream)
{
    return norm_backward<1>(d_g, g_stride, d_x, x_stride, 0, dtype, nullptr, MHC_DTYPE_F32, d_mean, d_rstd, d_w,
                            w_dtype, d_dx, nullptr, d_dw, d_db, N, C, d_workspace, workspace_bytes, stream);
}

extern "C" int mhc_stream_norm_n4(const void* d_X, int64_t token_stride, int64_t stream_stride, int dtype,
                                  const void* d_h, int h_dtype, const void* d_w, const void* d_b, int w_dtype,
                                  void* d_y, float* d_mean, float* d_rstd, float eps, int64_t N, int64_t C,
                                  cudaStream_t stream)
{
    return norm_forward<4>(d_X, token_stride, stream_stride, dtype, d_h, h_dtype, d_w, d_b, w_dtype, d_y, d_mean,
                           d_rstd, eps, N, C, stream);
}

extern "C" int mhc_stream_norm_n4_backward_workspace(int64_t N, int64_t C, int64_t* bytes)
{
    if (N < 0 || C < 1 || !bytes) return MHC_ERR_INVALID_VALUE;
    *bytes = norm_workspace(N, C);
    return MHC_OK;
}

extern "C" int mhc_stream_norm_n4_backward(const void* d_g, int64_t g_stride, const void* d_X, int64_t token_stride,
                                           int64_t stream_stride, int dtype, const void* d_h, int h_dtype,
                                           const float* d_mean, const float* d_rstd, const void* d_w, int w_dtype,
                                           void* d_dX, void* d_dh, void* d_dw, void* d_db, int64_t N, int64_t C,
                                           void* d_workspace, int64_t workspace_bytes, cudaStream_t stream)
{
    return norm_backward<4>(d_g, g_stride, d_X, token_stride, stream_stride, dtype, d_h, h_dtype, d_mean, d_rstd, d_w,
                            w_dtype, d_dX, d_dh, d_dw, d_db, N, C, d_workspace, workspace_bytes, stream);
}
