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
#include <type_traits>

#include "norm_ring.cuh"
#include "norm_source.cuh"
#include "row_copy.cuh"

namespace mhcp {

#ifndef MHC_RING_N
#define MHC_RING_N 1024
#endif
#ifndef MHC_SMEM
#define MHC_SMEM 204
#endif
#ifndef MHC_BE
#define MHC_BE 16
#endif
#ifndef MHC_BES
#define MHC_BES 8
#endif
#ifndef MHC_BHS
#define MHC_BHS true
#endif
#ifndef MHC_BB
#define MHC_BB 1
#endif
#ifndef MHC_BBS
#define MHC_BBS 1
#endif
#ifndef MHC_BT
#define MHC_BT 2
#endif
#ifndef MHC_BTS
#define MHC_BTS 1
#endif
#ifndef MHC_BTH
#define MHC_BTH 512
#endif
#ifndef MHC_BTHS
#define MHC_BTHS 512
#endif
constexpr int kNormBlock = 256;

// One block per row, which it reads three times (the second and third come
// from L1 or L2).
template <class Elem, int kStreams>
__global__ void __launch_bounds__(kNormBlock)
norm_fwd_rows(NormSource<Elem, kStreams> src, NormAffine aff, Elem* __restrict__ y, float* __restrict__ mean_out,
              float* __restrict__ rstd_out, float eps, int64_t N, int64_t C)
{
    __shared__ __align__(16) float buf[2][32];
    const Group group{kNormBlock, static_cast<int>(threadIdx.x), 0};
    group_sum_init<1>(group, buf[0]);
    group_sum_init<1>(group, buf[1]);
    for (int64_t r = blockIdx.x; r < N; r += gridDim.x) {
        const NormRow<Elem, kStreams> row(src, r);
        float s[1] = {0.0f};
        for (int64_t c = threadIdx.x; c < C; c += kNormBlock) s[0] += row.at(c);
        group_sum(group, s, buf[0]);
        const float mean = s[0] / static_cast<float>(C);
        s[0] = 0.0f;
        for (int64_t c = threadIdx.x; c < C; c += kNormBlock) {
            const float d = row.at(c) - mean;
            s[0] = fmaf(d, d, s[0]);
        }
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
    const Group group{kNormBlock, static_cast<int>(threadIdx.x), 0};
    group_sum_init<2>(group, buf);
    group_sum_init<4>(group, buf_h);
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
        group_sum(group, s, buf);
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

constexpr int64_t kMaxRowGrid = int64_t{1} << 20;
constexpr int64_t kParamChunks = 64;

// Rows of partial sums at most: the row kernels' chunks, or the ring kernel's blocks.
constexpr int64_t kMaxPartials = 1024;

static int64_t norm_workspace(int64_t N, int64_t C)
{
    return std::max<int64_t>(1, std::min(N, kMaxPartials)) * 2 * C * static_cast<int64_t>(sizeof(float));
}

// Whether rows move in 16-byte pieces: whole pieces, aligned, and the
// parameters of a type that load_param reads in pieces.
template <class Elem, int kStreams>
static bool norm_in_pieces(const NormSource<Elem, kStreams>& src, const NormAffine& aff, int64_t C)
{
    constexpr int e = sizeof(Elem);
    const int own = e == 4 ? MHC_DTYPE_F32 : std::is_same<Elem, __half>::value ? MHC_DTYPE_F16 : MHC_DTYPE_BF16;
    return ((C * e) & 15) == 0 && aligned16(src.x, src.stride, e) && ((src.stream_stride * e) & 15) == 0 &&
           aligned16(aff.w) && aligned16(aff.b) &&
           ((!aff.w && !aff.b) || aff.dtype == own || aff.dtype == MHC_DTYPE_F32);
}

// Elements of a row per thread and the most threads of a block, for rows of C
// elements: more elements as the rows get wider.
constexpr int64_t kHeldMax = 32 * 512;

template <class Elem, int kStreams, RowForm kForm, int kElems>
static void norm_forward_held(const NormSource<Elem, kStreams>& src, const NormAffine& aff, Elem* y, float* mean,
                              float* rstd, float eps, int64_t N, int64_t C, cudaStream_t stream)
{
    const int t = 32 * static_cast<int>(ceil_div(C, 32 * kElems));
    const int per_block = t == 32 ? 4 : 1;
    norm_fwd_held<Elem, kStreams, kForm, kElems, 512>
        <<<static_cast<unsigned>(ceil_div(N, per_block)), dim3(t, per_block), 0, stream>>>(
            src, aff, y, mean, rstd, eps, N, static_cast<int>(C));
}

// Calls `launch` with the form of the rows.
template <class Launch>
static cudaError_t by_form(bool pieces, bool whole, Launch launch)
{
    if (!pieces) return launch(std::integral_constant<RowForm, kLoose>{});
    if (!whole) return launch(std::integral_constant<RowForm, kPieces>{});
    return launch(std::integral_constant<RowForm, kWhole>{});
}

// The ring kernels' shape for rows of C elements.
struct RingPlan {
    int threads, groups, stages, blocks_per_sm, smem;
};

// Elements of a row per thread, rows a turn and whether the parameters stay in
// registers: rows of up to 8192 elements, and wider ones.
template <int kStreams, bool kWide>
struct FwdShape {
    static constexpr int kElems = kWide ? 32 : 16, kTurn = kStreams == 1 && !kWide ? 2 : 1;
    static constexpr bool kHold = true;
};
template <class Elem, int kStreams, bool kWide>
struct BwdShape {
    static constexpr int kNarrow = kStreams == 1 ? MHC_BE : MHC_BES;
    static constexpr int kElems = kWide ? 2 * kNarrow : kNarrow;
    static constexpr bool kHold = kWide ? false : kStreams == 1 ? true : MHC_BHS;
    static constexpr int kMaxThreads = 512;
};
constexpr int64_t kNarrowMax = 16 * 512, kWideMax = 32 * 512;
#ifndef MHC_MINST
#define MHC_MINST 2
#endif
constexpr int kMinStages = MHC_MINST;
constexpr int kRingSmem = MHC_SMEM * 1024;         // of an SM's 227 KB, for the ring

static RingPlan ring_plan(int64_t C, int elem, bool vec, int rows, int per_thread, int threads_per_sm)
{
    RingPlan p;
    p.threads = 32 * static_cast<int>(ceil_div(C, 32 * per_thread));
    p.groups = p.threads == 32 ? 8 : std::max(1, 256 / p.threads);
    const int stage = rows * ring_row_bytes(static_cast<int>(C), elem, vec, p.threads, per_thread) * p.groups;
    p.blocks_per_sm = std::max(1, std::min(threads_per_sm / (p.threads * p.groups), kRingSmem / (kMinStages * stage)));
    p.stages = std::min(kRingStages, std::max(1, kRingSmem / p.blocks_per_sm / stage));
    p.smem = std::max(p.stages * stage, p.groups > 1 ? static_cast<int>(8 * C) : 0);
    if (stage > 225 * 1024) p.stages = 0;  // one row does not fit
    return p;
}

template <class Elem, int kStreams, RowForm kForm, bool kWide>
static cudaError_t norm_forward_ring(const RingPlan& p, const NormSource<Elem, kStreams>& src, const NormAffine& aff,
                                     Elem* y, float* mean, float* rstd, float eps, int64_t N, int64_t C,
                                     cudaStream_t stream)
{
    using S = FwdShape<kStreams, kWide>;
    const auto kernel = norm_fwd_ring<Elem, kStreams, kForm, S::kElems, S::kTurn, S::kHold, 512>;
    const cudaError_t e = allow_smem(kernel, p.smem);
    if (e != cudaSuccess) return e;
    const int64_t grid = std::min<int64_t>(ceil_div(ceil_div(N, S::kTurn), p.groups), static_cast<int64_t>(p.blocks_per_sm) * sm_count());
    kernel<<<static_cast<unsigned>(grid), dim3(p.threads, p.groups), p.smem, stream>>>(
        src, span_of(src.x, N, src.stride, kStreams, src.stream_stride, C), aff, y, mean, rstd, eps, N,
        static_cast<int>(C), p.stages);
    return cudaSuccess;
}

template <class Elem, int kStreams>
static int norm_forward(const void* x, int64_t stride, int64_t stream_stride, const void* h, int h_dtype,
                        const NormAffine& aff, void* y, float* mean, float* rstd, float eps, int64_t N, int64_t C,
                        cudaStream_t stream)
{
    const NormSource<Elem, kStreams> src{static_cast<const Elem*>(x), stride, stream_stride, h, h_dtype};
    Elem* yp = static_cast<Elem*>(y);
    const bool pieces = norm_in_pieces(src, aff, C) && aligned16(y);
    const bool wide = C > kNarrowMax;
    const int elems = wide ? FwdShape<kStreams, true>::kElems : FwdShape<kStreams, false>::kElems;
    const int turn = wide ? FwdShape<kStreams, true>::kTurn : FwdShape<kStreams, false>::kTurn;
    const RingPlan plan = ring_plan(C, sizeof(Elem), pieces, kStreams * turn, elems, 512);
    if (C <= kWideMax && plan.stages > 0 && N >= MHC_RING_N) {
        const auto launch = [&](auto form) {
            constexpr RowForm f = decltype(form)::value;
            return wide ? norm_forward_ring<Elem, kStreams, f, true>(plan, src, aff, yp, mean, rstd, eps, N, C, stream)
                        : norm_forward_ring<Elem, kStreams, f, false>(plan, src, aff, yp, mean, rstd, eps, N, C, stream);
        };
        const cudaError_t e = by_form(pieces, plan.threads * elems == C, launch);
        if (e != cudaSuccess) return static_cast<int>(e);
    } else if (C > kHeldMax)
        norm_fwd_rows<Elem, kStreams><<<static_cast<unsigned>(std::min(N, kMaxRowGrid)), kNormBlock, 0, stream>>>(
            src, aff, yp, mean, rstd, eps, N, C);
    else if (C > 8 * 512)
        pieces ? norm_forward_held<Elem, kStreams, kPieces, 32>(src, aff, yp, mean, rstd, eps, N, C, stream)
               : norm_forward_held<Elem, kStreams, kLoose, 32>(src, aff, yp, mean, rstd, eps, N, C, stream);
    else
        pieces ? norm_forward_held<Elem, kStreams, kPieces, 8>(src, aff, yp, mean, rstd, eps, N, C, stream)
               : norm_forward_held<Elem, kStreams, kLoose, 8>(src, aff, yp, mean, rstd, eps, N, C, stream);
    return static_cast<int>(cudaGetLastError());
}

template <int kStreams>
static int norm_forward(const void* x, int64_t stride, int64_t stream_stride, int dtype, const void* h, int h_dtype,
                        const void* w, const void* b, int w_dtype, void* y, float* mean, float* rstd, float eps,
                        int64_t N, int64_t C, cudaStream_t stream)
{
    if (N < 0 || N >= (int64_t{1} << 31) || C < 1 || C > kMaxWidth || stride < 0 || stream_stride < 0 || !known_dtype(dtype) || !known_dtype(h_dtype) ||
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

template <class Elem, int kStreams, RowForm kForm, bool kWide>
static cudaError_t norm_backward_ring(const RingPlan& p, int64_t grid, const Elem* g, int64_t g_stride,
                                      const NormSource<Elem, kStreams>& src, const float* mean, const float* rstd,
                                      const NormAffine& aff, Elem* dx, void* dh, float* partials, int64_t N, int64_t C,
                                      cudaStream_t stream)
{
    using S = BwdShape<Elem, kStreams, kWide>;
    const auto kernel = norm_bwd_ring<Elem, kStreams, kForm, S::kElems, S::kHold, S::kMaxThreads>;
    const cudaError_t e = allow_smem(kernel, p.smem);
    if (e != cudaSuccess) return e;
    kernel<<<static_cast<unsigned>(grid), dim3(p.threads, p.groups), p.smem, stream>>>(
        g, g_stride, span_of(g, N, g_stride, 1, 0, C), src,
        span_of(src.x, N, src.stride, kStreams, src.stream_stride, C), mean, rstd, aff, dx, dh, partials, N,
        static_cast<int>(C), p.stages);
    return cudaSuccess;
}

template <class Elem, int kStreams>
static int norm_backward(const void* g, int64_t g_stride, const void* x, int64_t stride, int64_t stream_stride,
                         const void* h, int h_dtype, const float* mean, const float* rstd, const NormAffine& aff,
                         void* dx, void* dh, void* dw, void* db, int64_t N, int64_t C, float* partials,
                         cudaStream_t stream)
{
    const NormSource<Elem, kStreams> src{static_cast<const Elem*>(x), stride, stream_stride, h, h_dtype};
    const Elem* gp = static_cast<const Elem*>(g);
    const unsigned cols = static_cast<unsigned>(std::min<int64_t>(ceil_div(C, 32), int64_t{1} << 20));
    const bool pieces = norm_in_pieces(src, aff, C) && aligned16(g, g_stride, sizeof(Elem)) && aligned16(dx);
    const bool wide = C > BwdShape<Elem, kStreams, false>::kElems * 512;
    const int elems = wide ? BwdShape<Elem, kStreams, true>::kElems : BwdShape<Elem, kStreams, false>::kElems;
    const RingPlan plan = ring_plan(C, sizeof(Elem), pieces, kStreams + 1, elems, kStreams == 1 ? MHC_BTH : MHC_BTHS);
    if (N > 0 && plan.threads <= 512 && plan.stages > 0) {
        const int64_t grid = std::min({ceil_div(N, plan.groups),
                                       static_cast<int64_t>(plan.blocks_per_sm) * sm_count(), kMaxPartials});
        float* part = dw || db ? partials : nullptr;
        Elem* dxp = static_cast<Elem*>(dx);
        const auto launch = [&](auto form) {
            constexpr RowForm f = decltype(form)::value;
            return wide ? norm_backward_ring<Elem, kStreams, f, true>(plan, grid, gp, g_stride, src, mean, rstd, aff, dxp,
                                                                      dh, part, N, C, stream)
                        : norm_backward_ring<Elem, kStreams, f, false>(plan, grid, gp, g_stride, src, mean, rstd, aff, dxp,
                                                                       dh, part, N, C, stream);
        };
        const cudaError_t e = by_form(pieces, plan.threads * elems == C, launch);
        if (e != cudaSuccess) return static_cast<int>(e);
        if (part) norm_param_fold<<<dim3(cols, 2), 32 * kFoldLines, 0, stream>>>(partials, grid, dw, db, aff.dtype, C);
        return static_cast<int>(cudaGetLastError());
    }
    if (N > 0)
        norm_bwd_rows<Elem, kStreams><<<static_cast<unsigned>(std::min(N, kMaxRowGrid)), kNormBlock, 0, stream>>>(
            gp, g_stride, src, mean, rstd, aff, static_cast<Elem*>(dx), dh, N, C);
    if (dw || db) {
        int64_t chunks = 0;
        if (N > 0) {
            chunks = std::min(ceil_div(N, kParamRows), kParamChunks);
            const int64_t chunk_rows = ceil_div(N, chunks);
            norm_param_partials<Elem, kStreams>
                <<<dim3(cols, static_cast<unsigned>(chunks)), 32 * kParamRows, 0, stream>>>(
                    gp, g_stride, src, mean, rstd, partials, N, C, chunk_rows);
        }
        norm_param_fold<<<dim3(cols, 2), 32 * kFoldLines, 0, stream>>>(partials, chunks, dw, db, aff.dtype, C);
    }
    return static_cast<int>(cudaGetLastError());
}

template <int kStreams>
static int norm_backward(const void* g, int64_t g_stride, const void* x, int64_t stride, int64_t stream_stride,
                         int dtype, const void* h, int h_dtype, const float* mean, const float* rstd, const void* w,
                         int w_dtype, void* dx, void* dh, void* dw, void* db, int64_t N, int64_t C, void* workspace,
                         int64_t workspace_bytes, cudaStream_t stream)
{
    if (N < 0 || N >= (int64_t{1} << 31) || C < 1 || C > kMaxWidth || g_stride < 0 || stride < 0 || stream_stride < 0 || !known_dtype(dtype) ||
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
    if (N < 0 || N >= (int64_t{1} << 31) || C < 1 || C > kMaxWidth || !bytes) return MHC_ERR_INVALID_VALUE;
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
    if (N < 0 || N >= (int64_t{1} << 31) || C < 1 || C > kMaxWidth || !bytes) return MHC_ERR_INVALID_VALUE;
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
