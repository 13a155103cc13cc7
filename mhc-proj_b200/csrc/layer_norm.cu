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
#include "norm_rows.cuh"
#include "norm_source.cuh"
#include "row_copy.cuh"

namespace mhcp {

constexpr int64_t kMaxRowGrid = int64_t{1} << 20;
static int64_t norm_workspace(int64_t N, int64_t C)
{
    return norm_partial_rows(N, C) * 2 * C * static_cast<int64_t>(sizeof(float));
}

// Whether rows move in 16-byte pieces: whole pieces, aligned, and the
// parameters of a type that RowCols::param reads in pieces.
template <class Elem, int kStreams>
static bool norm_in_pieces(const NormSource<Elem, kStreams>& src, const NormAffine& aff, int64_t C)
{
    constexpr int e = sizeof(Elem);
    const int own = e == 4 ? MHC_DTYPE_F32 : std::is_same<Elem, __half>::value ? MHC_DTYPE_F16 : MHC_DTYPE_BF16;
    return ((C * e) & 15) == 0 && aligned16(src.x, src.stride, e) && ((src.stream_stride * e) & 15) == 0 &&
           aligned16(aff.w) && aligned16(aff.b) &&
           ((!aff.w && !aff.b) || aff.dtype == own || aff.dtype == MHC_DTYPE_F32);
}

// Whether every row of x starts as far into 16 bytes as the same row of the
// contiguous output does.
template <class Elem>
static bool lies_alike(const Elem* x, int64_t stride, const Elem* out, int64_t C)
{
    return ((reinterpret_cast<uintptr_t>(x) - reinterpret_cast<uintptr_t>(out)) & 15) == 0 &&
           (((stride - C) * static_cast<int64_t>(sizeof(Elem))) & 15) == 0;
}

// Fewer rows than this go to the held kernel (bf16, 4096 wide: 8 rows 2.4 us; 300
// rows 4.5 us held, 3.8 in the ring; 800 rows 7.1 and 5.0).
constexpr int64_t kRingRows = 256;

// The widest row that the held kernel takes, 512 threads with 32 elements each.
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
template <int kStreams, class Launch>
static cudaError_t by_form(RowForm form, Launch launch)
{
    if constexpr (kStreams == 1) {
        if (form == kSkewed) return launch(std::integral_constant<RowForm, kSkewed>{});
    }
    if (form == kWhole) return launch(std::integral_constant<RowForm, kWhole>{});
    if (form == kPieces) return launch(std::integral_constant<RowForm, kPieces>{});
    return launch(std::integral_constant<RowForm, kLoose>{});
}

template <class Elem, int kStreams, RowForm kForm, int kWidth>
static cudaError_t norm_forward_ring(const RingPlan& p, const NormSource<Elem, kStreams>& src, const NormAffine& aff,
                                     Elem* y, float* mean, float* rstd, float eps, int64_t N, int64_t C,
                                     cudaStream_t stream)
{
    using S = FwdShape<kStreams, kWidth>;
    const auto kernel = norm_fwd_ring<Elem, kStreams, kForm, S::kElems, S::kTurn, S::kHold>;
    const cudaError_t e = allow_smem<sizeof(typename S::Sums)>(kernel, p.smem);
    if (e != cudaSuccess) return e;
    const int64_t grid = p.grid(ceil_div(N, S::kTurn), sizeof(Elem), sm_count());
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
    const RowForm form = norm_in_pieces(src, aff, C) && aligned16(y)            ? kPieces
                         : kStreams == 1 && lies_alike(src.x, stride, yp, C) ? kSkewed
                                                                                : kLoose;
    const RingPlan plan = ring_plan<FwdShape, kStreams, 2>(C, sizeof(Elem), form);
    if (plan.stages > 0 && N >= kRingRows) {
        const cudaError_t e = by_form<kStreams>(plan.form, [&](auto f) {
            constexpr RowForm form = decltype(f)::value;
            return plan.width ? norm_forward_ring<Elem, kStreams, form, 1>(plan, src, aff, yp, mean, rstd, eps, N, C, stream)
                              : norm_forward_ring<Elem, kStreams, form, 0>(plan, src, aff, yp, mean, rstd, eps, N, C, stream);
        });
        if (e != cudaSuccess) return static_cast<int>(e);
    } else if (C > kHeldMax) {
        norm_fwd_rows<Elem, kStreams><<<static_cast<unsigned>(std::min(N, kMaxRowGrid)), kNormBlock, 0, stream>>>(
            src, aff, yp, mean, rstd, eps, N, C);
    } else if (C > 8 * 512) {
        form == kPieces ? norm_forward_held<Elem, kStreams, kPieces, 32>(src, aff, yp, mean, rstd, eps, N, C, stream)
                        : norm_forward_held<Elem, kStreams, kLoose, 32>(src, aff, yp, mean, rstd, eps, N, C, stream);
    } else {
        form == kPieces ? norm_forward_held<Elem, kStreams, kPieces, 8>(src, aff, yp, mean, rstd, eps, N, C, stream)
                        : norm_forward_held<Elem, kStreams, kLoose, 8>(src, aff, yp, mean, rstd, eps, N, C, stream);
    }
    return static_cast<int>(cudaGetLastError());
}

template <int kStreams>
static int norm_forward(const void* x, int64_t stride, int64_t stream_stride, int dtype, const void* h, int h_dtype,
                        const void* w, const void* b, int w_dtype, void* y, float* mean, float* rstd, float eps,
                        int64_t N, int64_t C, cudaStream_t stream)
{
    if (!rows_ok(N, C) || stride < 0 || stream_stride < 0 || !known_dtype(dtype) || !known_dtype(h_dtype) ||
        !known_dtype(w_dtype) || !(eps >= 0.0f) || (N > 0 && (!x || !y || (kStreams > 1 && !h))) ||
        !at_elements(dtype, x, y) || !at_elements(h_dtype, h) || !at_elements(w_dtype, w, b) ||
        !at_elements(MHC_DTYPE_F32, mean, rstd))
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

template <class Elem, int kStreams, RowForm kForm, int kWidth>
static cudaError_t norm_backward_ring(const RingPlan& p, int64_t grid, const Elem* g, int64_t g_stride,
                                      const NormSource<Elem, kStreams>& src, const float* mean, const float* rstd,
                                      const NormAffine& aff, Elem* dx, void* dh, float* partials, int64_t N, int64_t C,
                                      cudaStream_t stream)
{
    using S = BwdShape<kStreams, kWidth>;
    const auto kernel = norm_bwd_ring<Elem, kStreams, kForm, S::kElems, S::kHold>;
    const cudaError_t e = allow_smem<sizeof(typename S::Sums)>(kernel, p.smem);
    if (e != cudaSuccess) return e;
    kernel<<<static_cast<unsigned>(grid), dim3(p.threads, p.groups), p.smem, stream>>>(
        g, g_stride, span_of(g, N, g_stride, 1, 0, C), src,
        span_of(src.x, N, src.stride, kStreams, src.stream_stride, C), mean, rstd, aff, dx, dh, partials, N,
        static_cast<int>(C), p.stages);
    return cudaSuccess;
}

// Launched so that its blocks may be set up while the kernel before it, which
// makes the partial sums, still runs; they wait for its end.
static cudaError_t fold_params(const float* partials, int64_t rows, void* dw, void* db, int dtype, int64_t C,
                               cudaStream_t stream)
{
    cudaLaunchConfig_t config{};
    config.gridDim = dim3(static_cast<unsigned>(std::min<int64_t>(ceil_div(C, 32), int64_t{1} << 20)), 2);
    config.blockDim = dim3(32 * kFoldLines);
    config.stream = stream;
    cudaLaunchAttribute early{};
    early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    early.val.programmaticStreamSerializationAllowed = 1;
    config.attrs = &early;
    config.numAttrs = 1;
    return cudaLaunchKernelEx(&config, norm_param_fold, partials, rows, dw, db, dtype, C);
}

template <class Elem, int kStreams>
static int norm_backward(const void* g, int64_t g_stride, const void* x, int64_t stride, int64_t stream_stride,
                         const void* h, int h_dtype, const float* mean, const float* rstd, const NormAffine& aff,
                         void* dx, void* dh, void* dw, void* db, int64_t N, int64_t C, float* partials,
                         cudaStream_t stream)
{
    const NormSource<Elem, kStreams> src{static_cast<const Elem*>(x), stride, stream_stride, h, h_dtype};
    const Elem* gp = static_cast<const Elem*>(g);
    Elem* dxp = static_cast<Elem*>(dx);
    float* part = dw || db ? partials : nullptr;
    const RowForm form =
        norm_in_pieces(src, aff, C) && aligned16(g, g_stride, sizeof(Elem)) && aligned16(dx)                  ? kPieces
        : kStreams == 1 && lies_alike(src.x, stride, dxp, C) && lies_alike(gp, g_stride, dxp, C) ? kSkewed
                                                                                                              : kLoose;
    const RingPlan plan = ring_plan<BwdShape, kStreams, 3>(C, sizeof(Elem), form);
    int64_t rows = 0;  // of partial sums
    if (N > 0 && plan.stages > 0) {
        rows = std::min(plan.grid(N, sizeof(Elem), sm_count()), kMaxPartials);
        const cudaError_t e = by_form<kStreams>(plan.form, [&](auto f) {
            constexpr RowForm form = decltype(f)::value;
            switch (plan.width) {
                case 0:
                    return norm_backward_ring<Elem, kStreams, form, 0>(plan, rows, gp, g_stride, src, mean, rstd, aff, dxp,
                                                                       dh, part, N, C, stream);
                case 1:
                    return norm_backward_ring<Elem, kStreams, form, 1>(plan, rows, gp, g_stride, src, mean, rstd, aff, dxp,
                                                                       dh, part, N, C, stream);
                default:
                    return norm_backward_ring<Elem, kStreams, form, 2>(plan, rows, gp, g_stride, src, mean, rstd, aff, dxp,
                                                                       dh, part, N, C, stream);
            }
        });
        if (e != cudaSuccess) return static_cast<int>(e);
    } else if (N > 0) {
        norm_bwd_rows<Elem, kStreams><<<static_cast<unsigned>(std::min(N, kMaxRowGrid)), kNormBlock, 0, stream>>>(
            gp, g_stride, src, mean, rstd, aff, dxp, dh, N, C);
        if (dw || db) {
            rows = param_chunks(N);
            const unsigned cols = static_cast<unsigned>(std::min<int64_t>(ceil_div(C, 32), int64_t{1} << 20));
            norm_param_partials<Elem, kStreams><<<dim3(cols, static_cast<unsigned>(rows)), 32 * kParamRows, 0, stream>>>(
                gp, g_stride, src, mean, rstd, partials, N, C, ceil_div(N, rows));
        }
    }
    if (dw || db) {
        const cudaError_t e = fold_params(partials, rows, dw, db, aff.dtype, C, stream);
        if (e != cudaSuccess) return static_cast<int>(e);
    }
    return static_cast<int>(cudaGetLastError());
}

template <int kStreams>
static int norm_backward(const void* g, int64_t g_stride, const void* x, int64_t stride, int64_t stream_stride,
                         int dtype, const void* h, int h_dtype, const float* mean, const float* rstd, const void* w,
                         int w_dtype, void* dx, void* dh, void* dw, void* db, int64_t N, int64_t C, void* workspace,
                         int64_t workspace_bytes, cudaStream_t stream)
{
    if (!rows_ok(N, C) || g_stride < 0 || stride < 0 || stream_stride < 0 || !known_dtype(dtype) ||
        !known_dtype(h_dtype) || !known_dtype(w_dtype) ||
        (N > 0 && (!g || !x || !mean || !rstd || !dx || (kStreams > 1 && (!h || !dh)))) ||
        !at_elements(dtype, g, x, dx) || !at_elements(h_dtype, h, dh) || !at_elements(w_dtype, w, dw, db) ||
        !at_elements(MHC_DTYPE_F32, mean, rstd, workspace))
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
    if (!rows_ok(N, C) || !bytes) return MHC_ERR_INVALID_VALUE;
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
    if (!rows_ok(N, C) || !bytes) return MHC_ERR_INVALID_VALUE;
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
