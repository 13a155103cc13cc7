// Layer norm over rows that pass through a ring of stages in shared memory.
//
// A group of threads (one warp, or the whole block) takes row after row.  The
// rows to come are copied into the ring by asynchronous copies of 16-byte
// pieces that need no registers, so the bytes in flight do not depend on the
// occupancy and the copies go on while the group reduces and stores a row.
//
// Rows of aligned, whole pieces (kVec): every thread copies the pieces that it
// reads itself, so that the wait for its own copies is all the
// synchronisation a stage needs.  Any other rows: a stage keeps a row at the
// offset within 16 bytes that it has in memory, the group copies all the
// pieces that the row touches, and a barrier stands between that and the
// reading of single elements, `threads` apart.  Pieces that reach beyond the
// first or last byte of the tensor are copied element by element.
#pragma once

#include "norm_source.cuh"
#include "row_ops.cuh"

namespace mhcp {

__device__ __forceinline__ void copy_piece_async(void* smem, const void* global)
{
    const unsigned s = static_cast<unsigned>(__cvta_generic_to_shared(smem));
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(s), "l"(global) : "memory");
}

__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }

// Waits until at most `stages` - 1 of this thread's batches of copies are under way.
__device__ __forceinline__ void copies_wait(int stages)
{
    if (stages >= 4)
        asm volatile("cp.async.wait_group 3;" ::: "memory");
    else if (stages == 3)
        asm volatile("cp.async.wait_group 2;" ::: "memory");
    else if (stages == 2)
        asm volatile("cp.async.wait_group 1;" ::: "memory");
    else
        asm volatile("cp.async.wait_group 0;" ::: "memory");
}

constexpr int kRingStages = 4;  // at most

// A tensor of rows: the row's address is base + r * stride, and [lo, hi) are
// the bytes from its first to its last element.
struct RowSpan {
    const char *lo, *hi;
};

template <class Elem>
inline RowSpan span_of(const Elem* p, int64_t N, int64_t stride, int streams, int64_t stream_stride, int64_t C)
{
    return {reinterpret_cast<const char*>(p),
            reinterpret_cast<const char*>(p + (N - 1) * stride + (streams - 1) * stream_stride + C)};
}

// Bytes of one row's place in a stage.
__host__ __device__ inline int ring_row_bytes(int C, int elem, bool vec, int threads, int per_thread)
{
    return vec ? threads * per_thread * elem : (C * elem + 15) / 16 * 16 + 16;
}

// The ring of one group: kRows rows a stage, kElems elements of a row a thread.
template <class Elem, int kRows, bool kVec, int kElems>
struct RowRing {
    static constexpr int kPiece = 16 / sizeof(Elem);
    static constexpr int K = kVec ? kPiece : 8;
    static constexpr int P = kElems / K;

    char* base;
    int row_bytes, C, t, threads;

    __device__ __forceinline__ char* place(int stage, int row) const { return base + (stage * kRows + row) * row_bytes; }

    __device__ __forceinline__ void copy(int stage, int row, const Elem* from, const RowSpan& span) const
    {
        char* to = place(stage, row);
        if constexpr (kVec) {
#pragma unroll
            for (int p = 0; p < P; ++p) {
                const int piece = p * threads + t;
                if (piece * kPiece < C) copy_piece_async(to + piece * 16, from + piece * kPiece);
            }
        } else {
            const char* start = reinterpret_cast<const char*>(from);
            const char* end = reinterpret_cast<const char*>(from + C);
            const int shift = static_cast<int>(reinterpret_cast<uintptr_t>(start) & 15);
            const char* first = start - shift;
            const int pieces = (shift + C * static_cast<int>(sizeof(Elem)) + 15) >> 4;
            for (int q = t; q < pieces; q += threads) {
                const char* src = first + 16 * q;
                if (src >= span.lo && src + 16 <= span.hi) {
                    copy_piece_async(to + 16 * q, src);
                } else {
#pragma unroll
                    for (int i = 0; i < kPiece; ++i) {
                        const char* e = src + i * sizeof(Elem);
                        if (e >= start && e < end)
                            reinterpret_cast<Elem*>(to + 16 * q)[i] = *reinterpret_cast<const Elem*>(e);
                    }
                }
            }
        }
    }

    // Columns of piece p of this thread: col(p, j), j < K.
    __device__ __forceinline__ int col(int p, int j) const
    {
        if constexpr (kVec) return (p * threads + t) * K + j;
        return (p * K + j) * threads + t;
    }
    __device__ __forceinline__ bool has(int p, int j) const { return col(p, kVec ? 0 : j) < C; }

    // Piece p of a row of a stage; `from` is where the row came from.
    __device__ __forceinline__ void get(int stage, int row, int p, const Elem* from, float (&v)[K]) const
    {
        const char* at = place(stage, row);
        if constexpr (kVec) {
            uint4 q = make_uint4(0, 0, 0, 0);
            if (has(p, 0)) q = *reinterpret_cast<const uint4*>(at + (p * threads + t) * 16);
            const Elem* e = reinterpret_cast<const Elem*>(&q);
#pragma unroll
            for (int j = 0; j < K; ++j) v[j] = to_f32(e[j]);
        } else {
            const Elem* e = reinterpret_cast<const Elem*>(at + (reinterpret_cast<uintptr_t>(from) & 15));
#pragma unroll
            for (int j = 0; j < K; ++j) v[j] = has(p, j) ? to_f32(e[col(p, j)]) : 0.0f;
        }
    }

    __device__ __forceinline__ void put(Elem* __restrict__ row, int p, const float (&v)[K]) const
    {
        if constexpr (kVec) {
            uint4 q;
            Elem* e = reinterpret_cast<Elem*>(&q);
#pragma unroll
            for (int j = 0; j < K; ++j) e[j] = from_f32<Elem>(v[j]);
            if (has(p, 0)) *reinterpret_cast<uint4*>(row + col(p, 0)) = q;
        } else {
#pragma unroll
            for (int j = 0; j < K; ++j)
                if (has(p, j)) row[col(p, j)] = from_f32<Elem>(v[j]);
        }
    }

    // w or b at this thread's piece p; `none` where there is no such array.
    __device__ __forceinline__ void param(const void* a, int dtype, int p, float none, float (&v)[K]) const
    {
        if (!a) {
#pragma unroll
            for (int j = 0; j < K; ++j) v[j] = none;
        } else if constexpr (kVec) {
            const Elem* own = static_cast<const Elem*>(a);
            if (sizeof(Elem) == 4 || dtype != MHC_DTYPE_F32) {  // of the rows' own type (the launcher's rule)
                uint4 q = make_uint4(0, 0, 0, 0);
                if (has(p, 0)) q = __ldg(reinterpret_cast<const uint4*>(own + col(p, 0)));
                const Elem* e = reinterpret_cast<const Elem*>(&q);
#pragma unroll
                for (int j = 0; j < K; ++j) v[j] = to_f32(e[j]);
            } else {
                const float4* q = reinterpret_cast<const float4*>(static_cast<const float*>(a) + col(p, 0));
#pragma unroll
                for (int i = 0; i < K / 4; ++i) {
                    const float4 f = has(p, 0) ? __ldg(q + i) : make_float4(0, 0, 0, 0);
                    v[4 * i] = f.x;
                    v[4 * i + 1] = f.y;
                    v[4 * i + 2] = f.z;
                    v[4 * i + 3] = f.w;
                }
            }
        } else {
#pragma unroll
            for (int j = 0; j < K; ++j) v[j] = has(p, j) ? load_any(a, col(p, j), dtype) : none;
        }
    }

    // A barrier of the group.
    __device__ __forceinline__ void sync() const
    {
        if (threads == 32)
            __syncwarp();
        else
            __syncthreads();
    }
};

// Block: (threads of a row's group, groups); more groups than one only where a
// group is a warp.  first + k * step are a group's rows.
template <class Elem, int kStreams, bool kVec, int kElems>
__global__ void __launch_bounds__(1024)
norm_fwd_ring(NormSource<Elem, kStreams> src, RowSpan span, NormAffine aff, Elem* __restrict__ y,
              float* __restrict__ mean_out, float* __restrict__ rstd_out, float eps, int64_t N, int C, int stages)
{
    extern __shared__ __align__(16) char ring_memory[];
    __shared__ float buf[2][32];
    using Ring = RowRing<Elem, kStreams, kVec, kElems>;
    constexpr int K = Ring::K, P = Ring::P;
    const int threads = blockDim.x, t = threadIdx.x;
    const int row_bytes = ring_row_bytes(C, sizeof(Elem), kVec, threads, kElems);
    const Ring ring{ring_memory + static_cast<size_t>(threadIdx.y) * stages * kStreams * row_bytes, row_bytes, C, t, threads};
    const int64_t first = blockIdx.x * static_cast<int64_t>(blockDim.y) + threadIdx.y;
    const int64_t step = static_cast<int64_t>(gridDim.x) * blockDim.y;
    auto fill = [&](int stage, int64_t r) {
        if (r < N) {
#pragma unroll
            for (int i = 0; i < kStreams; ++i) ring.copy(stage, i, src.x + r * src.stride + i * src.stream_stride, span);
        }
        copies_commit();
    };
    for (int s = 0; s < stages; ++s) fill(s, first + s * step);
    const float inv = 1.0f / static_cast<float>(C);
    int stage = 0;
    NormRow<Elem, kStreams> next(src, min(first, N - 1));  // a row's weights are loaded one row ahead
    for (int64_t r = first; r < N; r += step) {
        const NormRow<Elem, kStreams> row = next;
        next = NormRow<Elem, kStreams>(src, min(r + step, N - 1));
        copies_wait(stages);
        if constexpr (!kVec) ring.sync();
        float u[P][K];
        float s[1] = {0.0f};
#pragma unroll
        for (int p = 0; p < P; ++p) {
            ring.get(stage, 0, p, row.x, u[p]);
            if constexpr (kStreams > 1) {
#pragma unroll
                for (int j = 0; j < K; ++j) u[p][j] *= row.h[0];
#pragma unroll
                for (int i = 1; i < kStreams; ++i) {
                    float v[K];
                    ring.get(stage, i, p, row.x + i * row.stream_stride, v);
#pragma unroll
                    for (int j = 0; j < K; ++j) u[p][j] = fmaf(row.h[i], v[j], u[p][j]);
                }
            }
#pragma unroll
            for (int j = 0; j < K; ++j) s[0] += u[p][j];
        }
        block_sum(s, buf[0]);
        fill(stage, r + stages * step);  // all of the group have read the stage
        stage = stage + 1 == stages ? 0 : stage + 1;
        const float mean = s[0] * inv;
        s[0] = 0.0f;
#pragma unroll
        for (int p = 0; p < P; ++p) {
#pragma unroll
            for (int j = 0; j < K; ++j) {
                u[p][j] = ring.has(p, j) ? u[p][j] - mean : 0.0f;
                s[0] = fmaf(u[p][j], u[p][j], s[0]);
            }
        }
        block_sum(s, buf[1]);
        const float rstd = 1.0f / sqrtf(s[0] * inv + eps);
#pragma unroll
        for (int p = 0; p < P; ++p) {
            float w[K], b[K];
            ring.param(aff.w, aff.dtype, p, 1.0f, w);
            ring.param(aff.b, aff.dtype, p, 0.0f, b);
#pragma unroll
            for (int j = 0; j < K; ++j) w[j] = fmaf(u[p][j] * rstd, w[j], b[j]);
            ring.put(y + r * C, p, w);
        }
        if (t == 0) {
            if (mean_out) mean_out[r] = mean;
            if (rstd_out) rstd_out[r] = rstd;
        }
    }
}

// The backward pass, with each block's part of dw and db in registers over
// all its rows: partials[block][0 or 1][C] (null: neither is wanted).
template <class Elem, int kStreams, bool kVec, int kElems, int kMaxThreads>
__global__ void __launch_bounds__(kMaxThreads)
norm_bwd_ring(const Elem* __restrict__ g, int64_t g_stride, RowSpan g_span, NormSource<Elem, kStreams> src,
              RowSpan span, const float* __restrict__ mean_in, const float* __restrict__ rstd_in, NormAffine aff,
              Elem* __restrict__ dx, void* __restrict__ dh, float* __restrict__ partials, int64_t N, int C, int stages)
{
    extern __shared__ __align__(16) char ring_memory[];
    __shared__ float buf[2][64];
    __shared__ float buf_h[2][32 * 4];
    using Ring = RowRing<Elem, kStreams + 1, kVec, kElems>;  // the row of g is the last of a stage
    constexpr int K = Ring::K, P = Ring::P;
    const int threads = blockDim.x, t = threadIdx.x, warps = threads >> 5;
    const int row_bytes = ring_row_bytes(C, sizeof(Elem), kVec, threads, kElems);
    const Ring ring{ring_memory + static_cast<size_t>(threadIdx.y) * stages * (kStreams + 1) * row_bytes, row_bytes, C, t,
                    threads};
    const int64_t first = blockIdx.x * static_cast<int64_t>(blockDim.y) + threadIdx.y;
    const int64_t step = static_cast<int64_t>(gridDim.x) * blockDim.y;
    auto fill = [&](int stage, int64_t r) {
        if (r < N) {
#pragma unroll
            for (int i = 0; i < kStreams; ++i) ring.copy(stage, i, src.x + r * src.stride + i * src.stream_stride, span);
            ring.copy(stage, kStreams, g + r * g_stride, g_span);
        }
        copies_commit();
    };
    for (int s = 0; s < stages; ++s) fill(s, first + s * step);
    float dw[P][K], db[P][K], w[P][K];
#pragma unroll
    for (int p = 0; p < P; ++p) {
        ring.param(aff.w, aff.dtype, p, 1.0f, w[p]);
#pragma unroll
        for (int j = 0; j < K; ++j) dw[p][j] = db[p][j] = 0.0f;
    }
    const float inv = 1.0f / static_cast<float>(C);
    // dh of the group's last row: its warps' parts, put together one row later
    auto put_dh = [&](int64_t r, int which) {
        if (t < kStreams) {
            float v = 0.0f;
            for (int k = 0; k < warps; ++k) v += buf_h[which][k * 4 + t];
            store_any(dh, r * kStreams + t, src.h_dtype, v);
        }
    };
    int stage = 0, parity = 0;
    // a row's weights and statistics are loaded one row ahead
    int64_t ahead = min(first, N - 1);
    NormRow<Elem, kStreams> next(src, ahead);
    float mean_next = mean_in[ahead], rstd_next = rstd_in[ahead];
    for (int64_t r = first; r < N; r += step) {
        const NormRow<Elem, kStreams> row = next;
        const Elem* gr = g + r * g_stride;
        const float mean = mean_next, rstd = rstd_next;
        ahead = min(r + step, N - 1);
        next = NormRow<Elem, kStreams>(src, ahead);
        mean_next = mean_in[ahead];
        rstd_next = rstd_in[ahead];
        copies_wait(stages);
        if constexpr (!kVec) ring.sync();
        // gw and xhat of a piece
        auto piece = [&](int p, float (&gv)[K], float (&xhat)[K]) {
            ring.get(stage, kStreams, p, gr, gv);
            ring.get(stage, 0, p, row.x, xhat);
            if constexpr (kStreams > 1) {
#pragma unroll
                for (int j = 0; j < K; ++j) xhat[j] *= row.h[0];
#pragma unroll
                for (int i = 1; i < kStreams; ++i) {
                    float v[K];
                    ring.get(stage, i, p, row.x + i * row.stream_stride, v);
#pragma unroll
                    for (int j = 0; j < K; ++j) xhat[j] = fmaf(row.h[i], v[j], xhat[j]);
                }
            }
#pragma unroll
            for (int j = 0; j < K; ++j) xhat[j] = (xhat[j] - mean) * rstd;
        };
        float s[2] = {0.0f, 0.0f};
#pragma unroll
        for (int p = 0; p < P; ++p) {
            float gv[K], xhat[K];
            piece(p, gv, xhat);
#pragma unroll
            for (int j = 0; j < K; ++j) {  // g is zero beyond the row
                dw[p][j] = fmaf(gv[j], xhat[j], dw[p][j]);
                db[p][j] += gv[j];
                const float gw = gv[j] * w[p][j];
                s[0] += gw;
                s[1] = fmaf(gw, xhat[j], s[1]);
            }
        }
        block_sum(s, buf[parity]);
        if constexpr (kStreams > 1) {
            if (warps > 1 && r != first) put_dh(r - step, parity ^ 1);
        }
        const float m1 = s[0] * inv, m2 = s[1] * inv;
        float a[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int p = 0; p < P; ++p) {
            float du[K], xhat[K];
            piece(p, du, xhat);
#pragma unroll
            for (int j = 0; j < K; ++j) du[j] = rstd * (fmaf(du[j], w[p][j], -m1) - xhat[j] * m2);
            if constexpr (kStreams == 1) {
                ring.put(dx + r * C, p, du);
            } else {
#pragma unroll
                for (int j = 0; j < K; ++j)
                    if (!ring.has(p, j)) du[j] = 0.0f;
#pragma unroll
                for (int i = 0; i < kStreams; ++i) {
                    float v[K];
                    ring.get(stage, i, p, row.x + i * row.stream_stride, v);
#pragma unroll
                    for (int j = 0; j < K; ++j) {
                        a[i] = fmaf(du[j], v[j], a[i]);
                        v[j] = row.h[i] * du[j];
                    }
                    ring.put(dx + (r * kStreams + i) * C, p, v);
                }
            }
        }
        if constexpr (kStreams > 1) {
#pragma unroll
            for (int i = 0; i < kStreams; ++i) {
#pragma unroll
                for (int m = 16; m > 0; m >>= 1) a[i] += __shfl_xor_sync(0xffffffffu, a[i], m);
            }
            if (warps == 1) {
                if (t == 0) {
#pragma unroll
                    for (int i = 0; i < kStreams; ++i) store_any(dh, r * kStreams + i, src.h_dtype, a[i]);
                }
            } else if ((t & 31) == 0) {
#pragma unroll
                for (int i = 0; i < kStreams; ++i) buf_h[parity][(t >> 5) * 4 + i] = a[i];
            }
        }
        if constexpr (!kVec) ring.sync();  // others read what this thread copies over
        fill(stage, r + stages * step);
        stage = stage + 1 == stages ? 0 : stage + 1;
        parity ^= 1;
    }
    if constexpr (kStreams > 1) {
        if (warps > 1) {
            __syncthreads();
            const int64_t rows = first < N ? (N - 1 - first) / step + 1 : 0;
            if (rows > 0) put_dh(first + (rows - 1) * step, static_cast<int>((rows - 1) & 1));
        }
    }
    if (!partials) return;
    float* out = partials + static_cast<int64_t>(blockIdx.x) * 2 * C;
    if (blockDim.y > 1) {
        // the groups' parts, added one group after another
        float* sum = reinterpret_cast<float*>(ring_memory);
        for (int k = 0; k < static_cast<int>(blockDim.y); ++k) {
            __syncthreads();
            if (static_cast<int>(threadIdx.y) != k) continue;
#pragma unroll
            for (int p = 0; p < P; ++p) {
#pragma unroll
                for (int j = 0; j < K; ++j) {
                    if (!ring.has(p, j)) continue;
                    const int c = ring.col(p, j);
                    if (k > 0) {
                        dw[p][j] += sum[c];
                        db[p][j] += sum[C + c];
                    }
                    sum[c] = dw[p][j];
                    sum[C + c] = db[p][j];
                }
            }
        }
        if (static_cast<int>(threadIdx.y) != static_cast<int>(blockDim.y) - 1) return;
    }
#pragma unroll
    for (int p = 0; p < P; ++p) {
#pragma unroll
        for (int j = 0; j < K; ++j) {
            if (!ring.has(p, j)) continue;
            out[ring.col(p, j)] = dw[p][j];
            out[C + ring.col(p, j)] = db[p][j];
        }
    }
}

}  // namespace mhcp
