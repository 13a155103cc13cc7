// Layer norm over rows that pass through a ring of stages in shared memory.
//
// A group of threads (some lanes of a warp, a warp, or several warps) takes row
// after row.  The rows to come are copied into the ring by asynchronous copies of
// 16-byte pieces that need no registers, so the bytes in flight do not depend
// on the occupancy and the copies go on while the group reduces and stores a
// row.
//
// Rows in pieces (row_cols.cuh): every thread copies the pieces that it reads
// itself, so that the wait for its own copies is all the synchronisation a
// stage needs.  Loose rows: a stage keeps a row at the offset within 16 bytes
// that it has in memory, the group copies all the pieces that the row touches,
// and a barrier stands between that and the reading of single elements.  Pieces
// that reach beyond the first or last byte of the tensor are copied element by
// element.
//
// Bound by HBM: a row is read once and written once, its sums are taken from
// registers, and the parameters stay in registers over all rows.  Forward, 65536
// x 4096 bf16: 168 us, 6.4 TB/s (a block per row with the row in registers 342;
// the ring with the parameters read for each row 283).  The backward pass has
// three tensors and twice the sums: 252 us, 6.4 TB/s (1762 with three readings
// and separate sums of the parameters' gradients; the ring alone 393, with
// packed arithmetic 320, with the parameters held 303, with the pieces held as
// they are so that a stage is refilled at once 264, with blocks' sums in whole
// lines 251, with xhat from the distance to the mean 252).  Under a load of seconds
// the clock falls and its instructions show: 270 to 291 us, by the box.
#pragma once

#include "norm_source.cuh"
#include "ring_plan.h"
#include "row_cols.cuh"
#include "row_copy.cuh"

namespace mhcp {

// The ring of one group: kRows rows a stage, kElems elements of a row a thread.
template <class Elem, int kRows, RowForm kForm, int kElems>
struct RowRing {
    using Cols = RowCols<Elem, kForm, kElems>;
    static constexpr int K = Cols::K, P = kElems / K;

    char* base;
    int row_bytes;
    const Cols& cols;

    __device__ __forceinline__ char* place(int stage, int row) const { return base + (stage * kRows + row) * row_bytes; }
    __device__ __forceinline__ int piece(int p) const { return p * cols.threads + cols.t; }

    // amid: the tensor has 32 bytes on both sides of the row
    __device__ __forceinline__ void copy(int stage, int row, const Elem* from, const RowSpan& span, bool amid) const
    {
        char* to = place(stage, row);
        if constexpr (kForm != kLoose) {
            const char* src = reinterpret_cast<const char*>(from - (kForm == kSkewed ? cols.skew : 0));
#pragma unroll
            for (int p = 0; p < P; ++p) {
                if (!cols.has(p)) continue;
                if (kForm != kSkewed || amid || cols.all(p))
                    copy_piece_async(to + piece(p) * 16, src + piece(p) * 16);
                else
                    copy_checked_piece(to + piece(p) * 16, src + piece(p) * 16, from, from + cols.C, span);
            }
        } else {
            const int skew = offset_in_piece(from);
            const int pieces = (skew + cols.C * static_cast<int>(sizeof(Elem)) + 15) >> 4;
            const char* src = reinterpret_cast<const char*>(from) - skew;
            if (amid) {
                for (int q = cols.t; q < pieces; q += cols.threads) copy_piece_async(to + 16 * q, src + 16 * q);
            } else {
                for (int q = cols.t; q < pieces; q += cols.threads)
                    copy_checked_piece(to + 16 * q, src + 16 * q, from, from + cols.C, span);
            }
        }
    }

    // What a skewed row's first and last pieces have of its neighbours, to
    // zero: once per row, by the threads that read them.
    __device__ __forceinline__ void trim(int stage, int row) const
    {
        if constexpr (kForm == kSkewed) {
            if (!cols.edge) return;
            if (cols.t == 0) {
                Elem* e = reinterpret_cast<Elem*>(place(stage, row));
#pragma unroll
                for (int j = 0; j < K - 1; ++j)
                    if (j < cols.skew) e[j] = from_f32<Elem>(0.0f);
            }
            if (cols.last()) {
                Elem* e = reinterpret_cast<Elem*>(place(stage, row) + (cols.C + cols.skew) / K * 16);
#pragma unroll
                for (int j = 1; j < K; ++j)
                    if (j >= cols.end) e[j] = from_f32<Elem>(0.0f);
            }
        }
    }

    // The 16 bytes of piece p of a row of a stage, of rows in pieces.
    __device__ __forceinline__ uint4 raw(int stage, int row, int p) const
    {
        return cols.has(p) ? *reinterpret_cast<const uint4*>(place(stage, row) + piece(p) * 16) : make_uint4(0, 0, 0, 0);
    }

    // Piece p of a row of a stage; `from` is where the row came from.
    __device__ __forceinline__ void get(int stage, int row, int p, const Elem* from, float2 (&v)[K / 2]) const
    {
        if constexpr (kForm != kLoose)
            cols.unpack(raw(stage, row, p), v);
        else
            cols.load(p, reinterpret_cast<const Elem*>(place(stage, row) + offset_in_piece(from)), v);
    }
};

// How far into its first piece of 16 bytes a skewed row starts, in elements.
template <class Elem, RowForm kForm>
__device__ __forceinline__ int row_skew(const Elem* row)
{
    return kForm == kSkewed ? offset_in_piece(row) / static_cast<int>(sizeof(Elem)) : 0;
}

// Block: (threads of a row's group, groups).  A group takes kTurn rows at a time,
// so that their sums share their barriers; its turns are first + k * step, where
// step is a whole number of kTurn rows' period: rows `period` apart are skewed
// alike.
template <class Elem, int kStreams, RowForm kForm, int kElems, int kTurn, bool kHold>
__global__ void __launch_bounds__(kRingThreads, 1)
norm_fwd_ring(NormSource<Elem, kStreams> src, RowSpan span, NormAffine aff, Elem* __restrict__ y,
              float* __restrict__ mean_out, float* __restrict__ rstd_out, float eps, int64_t N, int C, int stages)
{
    extern __shared__ __align__(16) char ring_memory[];
    __shared__ GroupSums<kStreams, kTurn> buf;
    using Ring = RowRing<Elem, kStreams * kTurn, kForm, kElems>;
    constexpr int K = Ring::K, P = Ring::P;
    const Group group;
    constexpr int64_t period = kForm == kSkewed ? 16 / sizeof(Elem) : 1;
    auto row_of = [&](int64_t turn, int q) { return turn / period * (period * kTurn) + turn % period + q * period; };
    const int64_t turns = (N + period * kTurn - 1) / (period * kTurn) * period;
    const int64_t first = blockIdx.x * static_cast<int64_t>(blockDim.y) + threadIdx.y;
    const int64_t step = static_cast<int64_t>(gridDim.x) * blockDim.y;
    const int row_bytes = ring_row_bytes(C, sizeof(Elem), kForm == kLoose, group.threads, kElems);
    const typename Ring::Cols cols(C, group.t, group.threads, row_skew<Elem, kForm>(src.x + row_of(first, 0) * src.stride));
    const Ring ring{ring_memory + static_cast<size_t>(group.id) * stages * kStreams * kTurn * row_bytes, row_bytes, cols};
    float(*sums)[kTurn * 32] = buf.of[group.one_warp() ? 0 : group.id];  // a warp's group needs none
    group_sum_init<kTurn>(group, sums[0]);
    group_sum_init<kTurn>(group, sums[1]);
    auto fill = [&](int stage, int64_t turn) {
#pragma unroll
        for (int q = 0; q < kTurn; ++q) {
            const int64_t r = row_of(turn, q);
            if (r < N) {
#pragma unroll
                for (int i = 0; i < kStreams; ++i)
                    ring.copy(stage, q * kStreams + i, src.x + r * src.stride + i * src.stream_stride, span, span.amid(r, N));
            }
        }
        copies_commit();
    };
    for (int s = 0; s < stages; ++s) fill(s, first + s * step);
    const float inv = 1.0f / static_cast<float>(C);
    float2 held_w[kHold ? P : 1][K / 2], held_b[kHold ? P : 1][K / 2];
    if constexpr (kHold) {
#pragma unroll
        for (int p = 0; p < P; ++p) {
            cols.param(p, aff.w, aff.dtype, 1.0f, held_w[p]);
            cols.param(p, aff.b, aff.dtype, 0.0f, held_b[p]);
            keep(held_w[p]);
            keep(held_b[p]);
        }
    }
    int stage = 0;
    NormRow<Elem, kStreams> next[kTurn];  // rows' weights are loaded one turn ahead
    auto look_ahead = [&](int64_t turn) {
#pragma unroll
        for (int q = 0; q < kTurn; ++q) next[q] = NormRow<Elem, kStreams>(src, min(row_of(turn, q), N - 1));
    };
    look_ahead(first);
    for (int64_t turn = first; turn < turns; turn += step) {
        NormRow<Elem, kStreams> row[kTurn];
#pragma unroll
        for (int q = 0; q < kTurn; ++q) row[q] = next[q];
        look_ahead(turn + step);
        copies_wait(stages);
        if constexpr (kForm == kLoose) group.sync();
        float2 u[kTurn][P][K / 2];
        float s[kTurn];
#pragma unroll
        for (int q = 0; q < kTurn; ++q) {
            ring.trim(stage, q * kStreams);
            float2 s2 = both(0.0f);
#pragma unroll
            for (int p = 0; p < P; ++p) {
                ring.get(stage, q * kStreams, p, row[q].x, u[q][p]);
                if constexpr (kStreams > 1) {
#pragma unroll
                    for (int j = 0; j < K / 2; ++j) u[q][p][j] = mul2(u[q][p][j], both(row[q].h[0]));
#pragma unroll
                    for (int i = 1; i < kStreams; ++i) {
                        float2 v[K / 2];
                        ring.get(stage, q * kStreams + i, p, row[q].x + i * row[q].stream_stride, v);
#pragma unroll
                        for (int j = 0; j < K / 2; ++j) u[q][p][j] = fma2(v[j], both(row[q].h[i]), u[q][p][j]);
                    }
                }
#pragma unroll
                for (int j = 0; j < K / 2; ++j) s2 = add2(s2, u[q][p][j]);
            }
            s[q] = s2.x + s2.y;
        }
        group_sum(group, s, sums[0]);
        fill(stage, turn + stages * step);  // all of the group have read the stage
        stage = stage + 1 == stages ? 0 : stage + 1;
        float mean[kTurn], rstd[kTurn];
#pragma unroll
        for (int q = 0; q < kTurn; ++q) {
            mean[q] = s[q] * inv;
            float2 s2 = both(0.0f);
#pragma unroll
            for (int p = 0; p < P; ++p) {
#pragma unroll
                for (int j = 0; j < K / 2; ++j) u[q][p][j] = add2(u[q][p][j], both(-mean[q]));
                cols.clear_rest(p, u[q][p]);
#pragma unroll
                for (int j = 0; j < K / 2; ++j) s2 = fma2(u[q][p][j], u[q][p][j], s2);
            }
            s[q] = s2.x + s2.y;
        }
        group_sum(group, s, sums[1]);
#pragma unroll
        for (int q = 0; q < kTurn; ++q) rstd[q] = rsqrtf(fmaf(s[q], inv, eps));
#pragma unroll
        for (int p = 0; p < P; ++p) {
            float2 w[K / 2], b[K / 2];
            if constexpr (kHold) {
#pragma unroll
                for (int j = 0; j < K / 2; ++j) {
                    w[j] = held_w[p][j];
                    b[j] = held_b[p][j];
                }
            } else {
                cols.param(p, aff.w, aff.dtype, 1.0f, w);
                cols.param(p, aff.b, aff.dtype, 0.0f, b);
            }
#pragma unroll
            for (int q = 0; q < kTurn; ++q) {
                float2 o[K / 2];
#pragma unroll
                for (int j = 0; j < K / 2; ++j) o[j] = fma2(mul2(u[q][p][j], both(rstd[q])), w[j], b[j]);
                if (row_of(turn, q) < N) cols.store(p, y + row_of(turn, q) * C, o);
            }
        }
        if (group.t == 0) {
#pragma unroll
            for (int q = 0; q < kTurn; ++q) {
                const int64_t r = row_of(turn, q);
                if (r < N && mean_out) mean_out[r] = mean[q];
                if (r < N && rstd_out) rstd_out[r] = rstd[q];
            }
        }
    }
}

// Sums of 16 values over a warp: each step hands half of the values a lane
// still holds to its partner and takes the partner's other half (16 shuffles
// for the 16 values instead of 80).  Lane l ends with the sum of value l % 16.
__device__ __forceinline__ float warp_sum16(float (&v)[16])
{
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int m = 8; m >= 1; m >>= 1) {
        const bool up = lane & m;
#pragma unroll
        for (int i = 0; i < m; ++i) {
            const float give = up ? v[i] : v[i + m];
            const float mine = up ? v[i + m] : v[i];
            v[i] = mine + __shfl_xor_sync(0xffffffffu, give, m);
        }
    }
    return v[0] + __shfl_xor_sync(0xffffffffu, v[0], 16);
}

// The backward pass of layer norm, with each block's part of dw and db in
// registers over all its rows: partials[block][0 or 1][C] (null: neither is
// wanted).
//
// xhat is formed from the distance u - mean.  u rstd - (mean rstd) would be one
// operation a pair of columns less (250 us for 252, 65536 x 4096 bf16; four
// streams, 65536 x 1024 fp16, 203 for 205), but the product's rounding is an error
// of all of a row's xhat that grows with |mean| rstd: 6e-5 at a centre 1024
// times the spread, and a gradient for the weight from rows of one value.
//
// All that a row's gradients need is summed in one go over the row, so that
// its stage is free again before the sums are known: sum(gw) and
// sum(gw xhat), and for the streams' weights
//   dh[i] = sum(du X[i]) = rstd (sum(gw X[i]) - m1 sum(X[i]) - m2 sum(xhat X[i])),
// m1 = sum(gw) / C, m2 = sum(gw xhat) / C.  A thread keeps its elements' gw and
// xhat until then (of one stream: the 16-byte pieces of g and x as they are).
// Four streams, 65536 x 2048 bf16: 400 us, 6.0 TB/s, 447 under a load of seconds
// (498 with dh in a second pass over the stage, 506 with 16 elements a thread,
// which spill).
template <class Elem, int kStreams, RowForm kForm, int kElems, bool kHold>
__global__ void __launch_bounds__(kRingThreads, 1)
norm_bwd_ring(const Elem* __restrict__ g, int64_t g_stride, RowSpan g_span, NormSource<Elem, kStreams> src,
              RowSpan span, const float* __restrict__ mean_in, const float* __restrict__ rstd_in, NormAffine aff,
              Elem* __restrict__ dx, void* __restrict__ dh, float* __restrict__ partials, int64_t N, int C, int stages)
{
    extern __shared__ __align__(16) char ring_memory[];
    constexpr int kSums = kStreams == 1 ? 2 : 16;
    __shared__ GroupSums<kStreams, kSums> buf;
    constexpr int kRows = kStreams + 1;  // of a stage: the streams, then g
    using Ring = RowRing<Elem, kRows, kForm, kElems>;
    constexpr int K = Ring::K, P = Ring::P;
    const Group group;
    const int64_t first = blockIdx.x * static_cast<int64_t>(blockDim.y) + threadIdx.y;
    const int64_t step = static_cast<int64_t>(gridDim.x) * blockDim.y;
    const int row_bytes = ring_row_bytes(C, sizeof(Elem), kForm == kLoose, group.threads, kElems);
    const typename Ring::Cols cols(C, group.t, group.threads, row_skew<Elem, kForm>(src.x + first * src.stride));
    const Ring ring{ring_memory + static_cast<size_t>(group.id) * stages * kRows * row_bytes, row_bytes, cols};
    float(*sums)[kSums * 32] = buf.of[group.one_warp() ? 0 : group.id];  // a warp's group needs none
    group_sum_init<2>(group, sums[0]);
    group_sum_init<2>(group, sums[1]);
    auto fill = [&](int stage, int64_t r) {
        if (r < N) {
#pragma unroll
            for (int i = 0; i < kStreams; ++i) ring.copy(stage, i, src.x + r * src.stride + i * src.stream_stride, span, span.amid(r, N));
            ring.copy(stage, kStreams, g + r * g_stride, g_span, g_span.amid(r, N));
        }
        copies_commit();
    };
    for (int s = 0; s < stages; ++s) fill(s, first + s * step);
    float2 dw[P][K / 2], db[P][K / 2], held[kHold ? P : 1][K / 2];
#pragma unroll
    for (int p = 0; p < P; ++p) {
        if constexpr (kHold) {
            cols.param(p, aff.w, aff.dtype, 1.0f, held[p]);
            keep(held[p]);
        }
#pragma unroll
        for (int j = 0; j < K / 2; ++j) dw[p][j] = db[p][j] = both(0.0f);
    }
    auto weight = [&](int p, float2 (&w)[K / 2]) {
        if constexpr (kHold) {
#pragma unroll
            for (int j = 0; j < K / 2; ++j) w[j] = held[p][j];
        } else {
            cols.param(p, aff.w, aff.dtype, 1.0f, w);
        }
    };
    const float inv = 1.0f / static_cast<float>(C);
    cudaTriggerProgrammaticLaunchCompletion();  // the fold may get ready
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
        if constexpr (kForm == kLoose) group.sync();
        if constexpr (kStreams == 1) {
            // Rows in pieces are kept as they are; other rows are read from the stage twice.
            uint4 kept[kForm != kLoose ? 2 : 1][P];
            if constexpr (kForm != kLoose) {
                ring.trim(stage, 0);
                ring.trim(stage, 1);
#pragma unroll
                for (int p = 0; p < P; ++p) {
                    kept[0][p] = ring.raw(stage, 0, p);
                    kept[1][p] = ring.raw(stage, 1, p);
                }
                fill(stage, r + stages * step);
            }
            auto piece = [&](int p, float2 (&gv)[K / 2], float2 (&u)[K / 2]) {
                if constexpr (kForm != kLoose) {
                    cols.unpack(kept[0][p], u);
                    cols.unpack(kept[1][p], gv);
                } else {
                    ring.get(stage, 0, p, row.x, u);
                    ring.get(stage, 1, p, gr, gv);
                }
            };
            float2 s0 = both(0.0f), s1 = both(0.0f);
#pragma unroll
            for (int p = 0; p < P; ++p) {
                float2 gv[K / 2], u[K / 2], w[K / 2];
                piece(p, gv, u);
                weight(p, w);
#pragma unroll
                for (int j = 0; j < K / 2; ++j) {  // g is zero beyond the row
                    const float2 xhat = mul2(add2(u[j], both(-mean)), both(rstd));
                    const float2 gw = mul2(gv[j], w[j]);
                    s0 = add2(s0, gw);
                    s1 = fma2(gw, xhat, s1);
                    dw[p][j] = fma2(gv[j], xhat, dw[p][j]);
                    db[p][j] = add2(db[p][j], gv[j]);
                }
            }
            float s[2] = {s0.x + s0.y, s1.x + s1.y};
            group_sum(group, s, sums[parity]);
            // du = rstd (gw - m1 - (u - mean) rstd m2)
            const float m1 = s[0] * inv, m2 = -s[1] * inv * rstd;
#pragma unroll
            for (int p = 0; p < P; ++p) {
                float2 du[K / 2], u[K / 2], w[K / 2];
                piece(p, du, u);
                weight(p, w);
#pragma unroll
                for (int j = 0; j < K / 2; ++j)
                    du[j] = mul2(both(rstd), fma2(add2(u[j], both(-mean)), both(m2), fma2(du[j], w[j], both(-m1))));
                cols.store(p, dx + r * C, du);
            }
            if constexpr (kForm == kLoose) {
                group.sync();  // others read what this thread copies over
                fill(stage, r + stages * step);
            }
        } else {
            float2 gw[P][K / 2], xhat[P][K / 2];
            float2 s0 = both(0.0f), s1 = both(0.0f), sx[kStreams], sg[kStreams], sh[kStreams];
#pragma unroll
            for (int i = 0; i < kStreams; ++i) sx[i] = sg[i] = sh[i] = both(0.0f);
#pragma unroll
            for (int p = 0; p < P; ++p) {
                float2 v[kStreams][K / 2], gv[K / 2], w[K / 2];
#pragma unroll
                for (int i = 0; i < kStreams; ++i) ring.get(stage, i, p, row.x + i * row.stream_stride, v[i]);
                ring.get(stage, kStreams, p, gr, gv);
                weight(p, w);
#pragma unroll
                for (int j = 0; j < K / 2; ++j) {  // g and X are zero beyond the row
                    float2 u = mul2(v[0][j], both(row.h[0]));
#pragma unroll
                    for (int i = 1; i < kStreams; ++i) u = fma2(v[i][j], both(row.h[i]), u);
                    const float2 x = mul2(add2(u, both(-mean)), both(rstd)), y = mul2(gv[j], w[j]);
                    s0 = add2(s0, y);
                    s1 = fma2(y, x, s1);
                    dw[p][j] = fma2(gv[j], x, dw[p][j]);
                    db[p][j] = add2(db[p][j], gv[j]);
#pragma unroll
                    for (int i = 0; i < kStreams; ++i) {
                        sg[i] = fma2(y, v[i][j], sg[i]);
                        sx[i] = add2(sx[i], v[i][j]);
                        sh[i] = fma2(x, v[i][j], sh[i]);
                    }
                    gw[p][j] = y;
                    xhat[p][j] = x;
                }
            }
            if constexpr (kForm != kLoose) fill(stage, r + stages * step);
            float all[16] = {s0.x + s0.y, s1.x + s1.y};
#pragma unroll
            for (int i = 0; i < kStreams; ++i) {
                all[2 + i] = sg[i].x + sg[i].y;
                all[6 + i] = sx[i].x + sx[i].y;
                all[10 + i] = sh[i].x + sh[i].y;
            }
            all[14] = all[15] = 0.0f;
            float m1, m2, a = 0.0f, b = 0.0f, c = 0.0f;  // a, b, c: of stream t, in the group's first threads
            if (group.threads < 32) {
                group.lane_sum(all);
                m1 = all[0];
                m2 = all[1];
#pragma unroll
                for (int i = 0; i < kStreams; ++i) {
                    if (group.t == i) {
                        a = all[2 + i];
                        b = all[6 + i];
                        c = all[10 + i];
                    }
                }
            } else if (group.threads == 32) {
                const float mine = warp_sum16(all);
                m1 = __shfl_sync(0xffffffffu, mine, 0);
                m2 = __shfl_sync(0xffffffffu, mine, 1);
                a = __shfl_sync(0xffffffffu, mine, 2 + (group.t & 3));
                b = __shfl_sync(0xffffffffu, mine, 6 + (group.t & 3));
                c = __shfl_sync(0xffffffffu, mine, 10 + (group.t & 3));
            } else {
                // value k of warp w at [k][w]
                float* part = sums[parity];
                const float mine = warp_sum16(all);
                if ((group.t & 31) < 14) part[(group.t & 31) * 32 + (group.t >> 5)] = mine;
                group.sync();
                m1 = m2 = 0.0f;
                for (int k = 0; k < group.warps(); k += 4) {  // parts of warps that the group does not have are zero
                    const float4 f = *reinterpret_cast<const float4*>(part + k);
                    const float4 h = *reinterpret_cast<const float4*>(part + 32 + k);
                    m1 += (f.x + f.y) + (f.z + f.w);
                    m2 += (h.x + h.y) + (h.z + h.w);
                }
                if (group.t < kStreams) {
                    for (int k = 0; k < group.warps(); ++k) {
                        a += part[(2 + group.t) * 32 + k];
                        b += part[(6 + group.t) * 32 + k];
                        c += part[(10 + group.t) * 32 + k];
                    }
                }
            }
            if constexpr (kForm == kLoose) fill(stage, r + stages * step);  // all of the group have read the stage
            m1 *= inv;
            m2 *= inv;
            if (group.t < kStreams) store_any(dh, r * kStreams + group.t, src.h_dtype, rstd * (a - m1 * b - m2 * c));
#pragma unroll
            for (int p = 0; p < P; ++p) {
#pragma unroll
                for (int j = 0; j < K / 2; ++j)
                    gw[p][j] = fma2(gw[p][j], both(rstd), fma2(xhat[p][j], both(-m2 * rstd), both(-m1 * rstd)));
#pragma unroll
                for (int i = 0; i < kStreams; ++i) {
                    float2 v[K / 2];
#pragma unroll
                    for (int j = 0; j < K / 2; ++j) v[j] = mul2(both(row.h[i]), gw[p][j]);
                    cols.store(p, dx + (r * kStreams + i) * C, v);
                }
            }
        }
        stage = stage + 1 == stages ? 0 : stage + 1;
        parity ^= 1;
    }
    if (!partials) return;
    // The groups' parts go through shared memory: one row of the workspace a
    // block, written in whole lines.  A skewed row's pieces keep their places.
    int2 me, of;  // read again: kept through the loop they cost registers that it has not
    asm volatile("mov.u32 %0, %%tid.x; mov.u32 %1, %%tid.y;" : "=r"(me.x), "=r"(me.y));
    asm volatile("mov.u32 %0, %%ntid.x; mov.u32 %1, %%ntid.y;" : "=r"(of.x), "=r"(of.y));
    float* part = reinterpret_cast<float*>(ring_memory) + static_cast<size_t>(me.y) * 2 * part_pitch(C);
    __syncthreads();  // the rings have been read
    auto put = [&](float* to, int p, const float2 (&v)[K / 2]) {
        if constexpr (kForm == kLoose) {
#pragma unroll
            for (int j = 0; j < K; ++j)
                if (cols.in(p, j)) to[cols.col(p, j)] = j & 1 ? v[j / 2].y : v[j / 2].x;
        } else if (cols.has(p)) {
#pragma unroll
            for (int j = 0; j < K / 2; j += 2)
                *reinterpret_cast<float4*>(to + ring.piece(p) * K + 2 * j) = make_float4(v[j].x, v[j].y, v[j + 1].x, v[j + 1].y);
        }
    };
#pragma unroll
    for (int p = 0; p < P; ++p) {
        put(part, p, dw[p]);
        put(part + part_pitch(C), p, db[p]);
    }
    __syncthreads();
    float* out = partials + static_cast<int64_t>(blockIdx.x) * 2 * C;
    const float* from = reinterpret_cast<const float*>(ring_memory);
    for (int c = me.y * of.x + me.x; c < C; c += of.x * of.y) {
        float w = 0.0f, b = 0.0f;
#pragma unroll 4
        for (int k = 0; k < of.y; ++k) {
            const int64_t r = blockIdx.x * static_cast<int64_t>(of.y) + k;
            const float* at = from + k * 2 * part_pitch(C) + c + row_skew<Elem, kForm>(src.x + r * src.stride);
            w += at[0];
            b += at[part_pitch(C)];
        }
        out[c] = w;
        out[C + c] = b;
    }
}

// A row held in the registers of its group, read once and directly: for
// batches that do not fill the GPU, where the way from the first load to the
// last store counts (8 rows of 4096 bf16: 2.4 us on the device, about an empty
// kernel's time and three trips to memory).
template <class Elem, int kStreams, RowForm kForm, int kElems, int kMaxThreads>
__global__ void __launch_bounds__(kMaxThreads)
norm_fwd_held(NormSource<Elem, kStreams> src, NormAffine aff, Elem* __restrict__ y, float* __restrict__ mean_out,
              float* __restrict__ rstd_out, float eps, int64_t N, int C)
{
    using Cols = RowCols<Elem, kForm, kElems>;
    constexpr int K = Cols::K, P = kElems / K;
    __shared__ __align__(16) float buf[2][32];
    const Group group;  // of whole warps; more than one in the block only where it is one warp
    group_sum_init<1>(group, buf[0]);
    group_sum_init<1>(group, buf[1]);
    const int64_t r = blockIdx.x * static_cast<int64_t>(blockDim.y) + threadIdx.y;
    if (r >= N) return;
    const Cols cols(C, group.t, group.threads, 0);
    const NormRow<Elem, kStreams> row(src, r);
    float2 u[P][K / 2];
    float2 s2 = both(0.0f);
#pragma unroll
    for (int p = 0; p < P; ++p) {
        cols.load(p, row.x, u[p]);
        if constexpr (kStreams > 1) {
            float2 v[kStreams - 1][K / 2];
#pragma unroll
            for (int i = 1; i < kStreams; ++i) cols.load(p, row.x + i * row.stream_stride, v[i - 1]);
#pragma unroll
            for (int j = 0; j < K / 2; ++j) {
                u[p][j] = mul2(u[p][j], both(row.h[0]));
#pragma unroll
                for (int i = 1; i < kStreams; ++i) u[p][j] = fma2(v[i - 1][j], both(row.h[i]), u[p][j]);
            }
        }
    }
    float2 w[P][K / 2], b[P][K / 2];
#pragma unroll
    for (int p = 0; p < P; ++p) {
        cols.param(p, aff.w, aff.dtype, 1.0f, w[p]);
        cols.param(p, aff.b, aff.dtype, 0.0f, b[p]);
    }
#pragma unroll
    for (int p = 0; p < P; ++p) {
#pragma unroll
        for (int j = 0; j < K / 2; ++j) s2 = add2(s2, u[p][j]);
    }
    float s[1] = {s2.x + s2.y};
    group_sum(group, s, buf[0]);
    const float inv = 1.0f / static_cast<float>(C), mean = s[0] * inv;
    s2 = both(0.0f);
#pragma unroll
    for (int p = 0; p < P; ++p) {
#pragma unroll
        for (int j = 0; j < K / 2; ++j) u[p][j] = add2(u[p][j], both(-mean));
        cols.clear_rest(p, u[p]);
#pragma unroll
        for (int j = 0; j < K / 2; ++j) s2 = fma2(u[p][j], u[p][j], s2);
    }
    s[0] = s2.x + s2.y;
    group_sum(group, s, buf[1]);
    const float rstd = rsqrtf(fmaf(s[0], inv, eps));
#pragma unroll
    for (int p = 0; p < P; ++p) {
#pragma unroll
        for (int j = 0; j < K / 2; ++j) b[p][j] = fma2(mul2(u[p][j], both(rstd)), w[p][j], b[p][j]);
        cols.store(p, y + r * C, b[p]);
    }
    if (threadIdx.x == 0) {
        if (mean_out) mean_out[r] = mean;
        if (rstd_out) rstd_out[r] = rstd;
    }
}

}  // namespace mhcp
