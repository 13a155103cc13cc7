// Layer norm kernels for rows that the ring kernels do not hold, one block per
// row in loops over its columns, and the fold of the parameters' partial sums.
// Such rows are wider than 16384 elements; in the backward also skewed ones from
// 16378 (fp32 16382), and four streams in fp32 from 10244 (loose ones 10237), a
// stage of which does not fit in a block's shared memory.  Bound by latency:
// every pass reads single elements, from L1 or L2 after the first.
#pragma once

#include "norm_source.cuh"
#include "ring_plan.h"

namespace mhcp {

constexpr int kNormBlock = 256;

// Adds up a thread's columns c of a row, K sums of what term(c, sums) adds to
// them: in 32 bits over runs of 64 columns and in 64 bits over the runs, so that
// the rounding of a row of 2^30 columns (4 million a thread) is that of a short
// one.  4096 rows of 32768: forward fp32 1132 us for 1091 with one sum in 32 bits,
// backward bf16 820 (1442 without the loop's unrolling).
constexpr int kNormRun = 64;

template <int K, class Term>
__device__ __forceinline__ void column_sums(int64_t C, float (&s)[K], Term term)
{
    double total[K] = {};
    for (int64_t c = threadIdx.x; c < C;) {
        float run[K] = {};
        const int64_t end = min(C, c + kNormRun * kNormBlock);
#pragma unroll 4
        for (; c < end; c += kNormBlock) term(c, run);
#pragma unroll
        for (int k = 0; k < K; ++k) total[k] += run[k];
    }
#pragma unroll
    for (int k = 0; k < K; ++k) s[k] = static_cast<float>(total[k]);
}

// One block per row, which it reads three times (the second and third come
// from L1 or L2).
template <class Elem, int kStreams>
__global__ void __launch_bounds__(kNormBlock)
norm_fwd_rows(NormSource<Elem, kStreams> src, NormAffine aff, Elem* __restrict__ y, float* __restrict__ mean_out,
              float* __restrict__ rstd_out, float eps, int64_t N, int64_t C)
{
    __shared__ __align__(16) float buf[2][32];
    const Group group;
    group_sum_init<1>(group, buf[0]);
    group_sum_init<1>(group, buf[1]);
    for (int64_t r = blockIdx.x; r < N; r += gridDim.x) {
        const NormRow<Elem, kStreams> row(src, r);
        float s[1];
        column_sums(C, s, [&](int64_t c, float (&run)[1]) { run[0] += row.at(c); });
        group_sum(group, s, buf[0]);
        const float mean = s[0] / static_cast<float>(C);
        column_sums(C, s, [&](int64_t c, float (&run)[1]) {
            const float d = row.at(c) - mean;
            run[0] = fmaf(d, d, run[0]);
        });
        group_sum(group, s, buf[1]);
        const float rstd = rsqrtf(s[0] / static_cast<float>(C) + eps);
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
    __shared__ __align__(16) float buf[2 * 32];
    __shared__ __align__(16) float buf_h[4 * 32];
    const Group group;
    group_sum_init<2>(group, buf);
    group_sum_init<4>(group, buf_h);
    for (int64_t r = blockIdx.x; r < N; r += gridDim.x) {
        const NormRow<Elem, kStreams> row(src, r);
        const Elem* gr = g + r * g_stride;
        const float mean = mean_in[r], rstd = rstd_in[r];
        float s[2];
        column_sums(C, s, [&](int64_t c, float (&run)[2]) {
            const float gw = to_f32(gr[c]) * (aff.w ? load_any(aff.w, c, aff.dtype) : 1.0f);
            run[0] += gw;
            run[1] = fmaf(gw, (row.at(c) - mean) * rstd, run[1]);
        });
        group_sum(group, s, buf);
        const float m1 = s[0] / static_cast<float>(C), m2 = s[1] / static_cast<float>(C);
        float a[4];
        column_sums(C, a, [&](int64_t c, float (&run)[4]) {
            const float gw = to_f32(gr[c]) * (aff.w ? load_any(aff.w, c, aff.dtype) : 1.0f);
            const float du = rstd * (gw - m1 - (row.at(c) - mean) * rstd * m2);
            if constexpr (kStreams == 1) {
                dx[r * C + c] = from_f32<Elem>(du);
            } else {
#pragma unroll
                for (int i = 0; i < kStreams; ++i) {
                    run[i] = fmaf(du, to_f32(row.x[i * row.stream_stride + c]), run[i]);
                    dx[(r * kStreams + i) * C + c] = from_f32<Elem>(row.h[i] * du);
                }
            }
        });
        if constexpr (kStreams > 1) {
            group_sum(group, a, buf_h);
            if (threadIdx.x == 0) {
#pragma unroll
                for (int i = 0; i < kStreams; ++i) store_any(dh, r * kStreams + i, src.h_dtype, a[i]);
            }
        }
        __syncthreads();  // buf is written again
    }
}

// Partial sums of dw and db over one chunk of rows: partials[chunk][0 or 1][C].
// A block works on kParamRows rows at once, 32 columns wide.
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

// dw and db from `rows` rows of partial sums, 32 columns a block.
constexpr int kFoldLines = 32;

__global__ void __launch_bounds__(32 * kFoldLines)
norm_param_fold(const float* __restrict__ partials, int64_t rows, void* __restrict__ dw, void* __restrict__ db,
                int dtype, int64_t C)
{
    __shared__ float part[kFoldLines][33];
    const int lane = threadIdx.x & 31, line = threadIdx.x >> 5;
    void* out = blockIdx.y == 0 ? dw : db;
    if (!out) return;
    cudaGridDependencySynchronize();  // launched while the kernel that sums is still running
    for (int64_t c0 = static_cast<int64_t>(blockIdx.x) * 32; c0 < C; c0 += static_cast<int64_t>(gridDim.x) * 32) {
        const int64_t c = c0 + lane;
        float v = 0.0f;
        if (c < C) {
#pragma unroll 8
            for (int64_t k = line; k < rows; k += kFoldLines) v += partials[(k * 2 + blockIdx.y) * C + c];
        }
        part[line][lane] = v;
        __syncthreads();
        // warp l folds column c0 + l
        v = part[lane][line];
#pragma unroll
        for (int m = 16; m > 0; m >>= 1) v += __shfl_xor_sync(0xffffffffu, v, m);
        if (lane == 0 && c0 + line < C) store_any(out, c0 + line, dtype, v);
        __syncthreads();
    }
}

}  // namespace mhcp
