// The mix over chunks of tokens' columns that pass through private rings in
// shared memory: each warp copies the chunks it will take next, without
// registers, while it works on one; no barrier of a block stands anywhere.  A
// lane works on a piece of K consecutive columns, 16 bytes of each row.
// Bound by HBM.  65536 tokens of 2048 bf16: forward 375 us, 6.4 TB/s (a block per
// token with direct loads 643, a warp per token 458, this ring without packed
// arithmetic 420); backward 595 us, 6.3 TB/s (a block per token 3220 with a sum
// over it for each of the 20 coefficients' gradients, a warp per token with
// direct loads 633), 631 under a load of seconds, when the clock falls.
//   kVec   rows of aligned, whole pieces: `lanes` lanes (a power of two) share a
//          token, 32 / lanes tokens a warp, and each lane copies what it reads.
//   else   any rows of any width: the warp copies the aligned pieces that a
//          row's part of the chunk touches, waits together, and a lane reads and
//          writes single elements, 32 apart.  Chunks go by y's element index
//          (whole groups of draws), so a token's first and last one may reach
//          beyond its row; only there is each column asked for.
#pragma once

#include "mix_source.cuh"
#include "row_copy.cuh"

namespace mhcp {

constexpr int kMixRingBlock = 128;
// Blocks of an SM and their stages: as many bytes under way as keep HBM busy; more
// (forward 4 stages: 429 us for 375) meet one another in the memory system.
constexpr int kMixFwdStages = 2, kMixBwdStages = 2, kMixFwdBlocks = 4;

// What of a chunk is kept, by warp: the ring kernels' static memory.
struct MixMasks {
    alignas(16) unsigned char of[kMixRingBlock / 32][32];
};

template <class Elem, bool kVec>
struct MixChunk {
    static constexpr int K = 16 / sizeof(Elem);
    static constexpr int kPlace = kVec ? 512 : 528;  // bytes of a row's part of a chunk
    int C, lane, lanes;

    // Chunks of a token (of a row that starts in the middle of a group of eight, too).
    static __host__ __device__ __forceinline__ int count(int C, int lanes)
    {
        return kVec ? (C / K + lanes - 1) / lanes : (C + 7 + 32 * K - 1) / (32 * K);
    }
    // First column of this lane in chunk i of a token whose row of y starts at element `first`.
    __device__ __forceinline__ int start(int i, int64_t first) const
    {
        if constexpr (kVec) return (i * lanes + (lane & (lanes - 1))) * K;
        return i * (32 * K) + lane - static_cast<int>(first & 7);
    }
    // Work goes step by step, kPairs pairs of columns at a time; what of the
    // row's columns lies beyond a chunk's last step is not touched.
    static constexpr int kPairs = kVec ? K / 2 : 1, kSteps = kVec ? 1 : K / 2;
    __device__ __forceinline__ int steps(int c) const
    {
        if constexpr (kVec) return 1;
        return min(kSteps, (C - (c - lane) + 63) / 64);
    }
    // Whether columns x and y of pair 0 of a step are in the row.
    __device__ __forceinline__ bool has_x(int c, int step) const
    {
        if constexpr (kVec) return c < C;
        return static_cast<unsigned>(c + 64 * step) < static_cast<unsigned>(C);
    }
    __device__ __forceinline__ bool has_y(int c, int step) const
    {
        if constexpr (kVec) return c < C;
        return static_cast<unsigned>(c + 64 * step + 32) < static_cast<unsigned>(C);
    }

    // This chunk of a row to a place; c is the lane's first column.  amid: the
    // tensor has 32 bytes on both sides of the row.
    __device__ __forceinline__ void copy(char* to, const Elem* row, int c, const RowSpan& span, bool amid) const
    {
        if constexpr (kVec) {
            if (c < C) copy_piece_async(to + lane * 16, row + c);
        } else {
            const Elem* from = row + (c - lane);
            const int skew = offset_in_piece(from);
            const char* src = reinterpret_cast<const char*>(from) - skew + 16 * lane;
            to += 16 * lane;
            if (amid) {
                // to the piece that holds the chunk's or the row's last column
                const int bytes = skew + min(32 * K, C - (c - lane)) * static_cast<int>(sizeof(Elem));
                if (16 * lane < bytes) copy_piece_async(to, src);
                if (lane == 31 && 512 < bytes) copy_piece_async(to + 16, src + 16);
            } else {
                copy_checked_piece(to, src, row, row + C, span);
                if (lane == 31) copy_checked_piece(to + 16, src + 16, row, row + C, span);
            }
        }
    }
    // Where this lane's columns of a row lie in a place.
    __device__ __forceinline__ const char* at(const char* place, const Elem* row, int c) const
    {
        if constexpr (kVec) return place + lane * 16;
        return place + offset_in_piece(row + (c - lane)) + lane * sizeof(Elem);
    }
    // What is not in the row may be anything.
    __device__ __forceinline__ void get(const char* at, int step, float2 (&v)[kPairs]) const
    {
        if constexpr (kVec) {
            const uint4 q = *reinterpret_cast<const uint4*>(at);
#pragma unroll
            for (int j = 0; j < kPairs; ++j) v[j] = pair_of<Elem>(q, j);
        } else {
            const Elem* e = reinterpret_cast<const Elem*>(at);
            v[0] = make_float2(to_f32(e[64 * step]), to_f32(e[64 * step + 32]));
        }
    }
    __device__ __forceinline__ void put(Elem* __restrict__ to, int step, bool x, bool y, const float2 (&v)[kPairs]) const
    {
        if constexpr (kVec) {
            const uint4 q = piece_of<Elem>(v);
            if (x) *reinterpret_cast<uint4*>(to) = q;
        } else {
            if (x) to[64 * step] = from_f32<Elem>(v[0].x);
            if (y) to[64 * step + 32] = from_f32<Elem>(v[0].y);
        }
    }
    static __device__ __forceinline__ void clear_rest(bool x, bool y, float2 (&v)[kPairs])
    {
#pragma unroll
        for (int j = 0; j < kPairs; ++j) v[j] = make_float2(x ? v[j].x : 0.0f, y ? v[j].y : 0.0f);
    }
    // What of a lane's columns is kept.
    struct Keep {
        uint32_t w[kVec ? 1 : K];  // bit of column j: kVec w[0] >> j, else w[j] >> lane
    };
    // `masks`: 32 bytes of the warp.
    __device__ __forceinline__ Keep keep(int64_t first, int c, const Dropout& d, uint2 key, unsigned char* masks) const
    {
        Keep k;
        if constexpr (kVec) {
            const int64_t e = first + c;
            k.w[0] = keep_bits(e >> 3, d.offset, key, d.limit) >> (e & 7);
        } else {
            // lane l draws for the chunk's columns 8 l .. 8 l + 7: the masks' bytes, four to the 32 columns of a step
            masks[lane] = static_cast<unsigned char>(keep_bits(((first + c - lane) >> 3) + lane, d.offset, key, d.limit));
            __syncwarp();
#pragma unroll
            for (int j = 0; j < K; ++j) k.w[j] = reinterpret_cast<const uint32_t*>(masks)[j];
            __syncwarp();  // the masks are written again
        }
        return k;
    }
    __device__ __forceinline__ void drop(float2 (&y)[kPairs], const Keep& k, int step, float scale) const
    {
#pragma unroll
        for (int j = 0; j < kPairs; ++j) {
            y[j] = mul2(y[j], both(scale));
            if (!(kVec ? k.w[0] >> (2 * j) & 1u : k.w[kVec ? 0 : 2 * step] >> lane & 1u)) y[j].x = 0.0f;
            if (!(kVec ? k.w[0] >> (2 * j + 1) & 1u : k.w[kVec ? 0 : 2 * step + 1] >> lane & 1u)) y[j].y = 0.0f;
        }
    }
};

// A walk over (token group, chunk) items in steps of `groups` groups and `rest` chunks.
struct MixWalk {
    int64_t group;
    int chunk;

    __device__ __forceinline__ MixWalk(int64_t item, int chunks)
        : group(item / chunks), chunk(static_cast<int>(item % chunks))
    {
    }
    __device__ __forceinline__ void advance(int64_t groups, int rest, int chunks)
    {
        group += groups;
        chunk += rest;
        if (chunk >= chunks) {
            chunk -= chunks;
            ++group;
        }
    }
};

template <class Elem, bool kVec, bool kWide>
__global__ void __launch_bounds__(kMixRingBlock)
mix_fwd_ring(MixIn<Elem> in, RowSpan x_span, RowSpan y_span, Elem* __restrict__ out, Dropout d, int64_t N, int C, int lanes)
{
    extern __shared__ __align__(16) char ring_memory[];
    __shared__ MixMasks masks;
    using Chunk = MixChunk<Elem, kVec>;
    constexpr int kPairs = Chunk::kPairs, kPlace = Chunk::kPlace;
    constexpr int kStage = 5 * kPlace;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    const Chunk ch{C, lane, lanes};
    char* ring = ring_memory + warp * (kMixFwdStages * kStage);
    const uint2 key = dropout_key(d);
    const int chunks = Chunk::count(C, lanes);
    const int per_warp = kVec ? 32 / lanes : 1;  // tokens
    const int mine = kVec ? lane / lanes : 0;
    const int64_t items = (N + per_warp - 1) / per_warp * chunks;
    const int64_t first = blockIdx.x * static_cast<int64_t>(warps) + warp, step = static_cast<int64_t>(gridDim.x) * warps;
    const int64_t step_groups = step / chunks;
    const int step_rest = static_cast<int>(step % chunks);
    MixWalk walk(first, chunks), ahead = walk;
    int64_t ahead_item = first;
    auto fill = [&](int stage) {
        const int64_t r = ahead.group * per_warp + mine;
        if (ahead_item < items && r < N) {
            const int c = ch.start(ahead.chunk, r * C);
            const bool x_amid = x_span.amid(r, N), y_amid = y_span.amid(r, N);
            char* to = ring + stage * kStage;
#pragma unroll
            for (int j = 0; j < 4; ++j) ch.copy(to + j * kPlace, in.x + r * in.stride + j * in.stream_stride, c, x_span, x_amid);
            ch.copy(to + 4 * kPlace, in.y + r * in.y_stride, c, y_span, y_amid);
        }
        copies_commit();
        ahead.advance(step_groups, step_rest, chunks);
        ahead_item += step;
    };
#pragma unroll
    for (int s = 0; s < kMixFwdStages; ++s) fill(s);
    int stage = 0;
    MixCoef next = mix_coef<kWide>(in, min(walk.group * per_warp + mine, N - 1));  // loaded one item ahead
    for (int64_t item = first; item < items; item += step) {
        const int64_t r = walk.group * per_warp + mine;
        const int c = ch.start(walk.chunk, r * C);
        const MixCoef k = next;
        walk.advance(step_groups, step_rest, chunks);
        next = mix_coef<kWide>(in, min(walk.group * per_warp + mine, N - 1));
        copies_wait(kMixFwdStages);
        if constexpr (!kVec) __syncwarp();
        const char* place = ring + stage * kStage;
        const char *at_x[4], *at_y = ch.at(place + 4 * kPlace, in.y + r * in.y_stride, c);
#pragma unroll
        for (int j = 0; j < 4; ++j) at_x[j] = ch.at(place + j * kPlace, in.x + r * in.stride + j * in.stream_stride, c);
        typename Chunk::Keep keep;
        if (d.limit) keep = ch.keep(r * C, c, d, key, masks.of[warp]);
        Elem* to = out + r * 4 * C + c;
        const int steps = ch.steps(c);
#pragma unroll
        for (int s = 0; s < Chunk::kSteps; ++s) {
            if (s >= steps) break;
            float2 v[4][kPairs], y[kPairs];
#pragma unroll
            for (int j = 0; j < 4; ++j) ch.get(at_x[j], s, v[j]);
            ch.get(at_y, s, y);
            if constexpr (kVec) fill(stage);  // a lane reads what it copied
            if (d.limit) ch.drop(y, keep, s, d.scale);
            const bool has_x = r < N && ch.has_x(c, s), has_y = r < N && ch.has_y(c, s);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float2 a[kPairs];
#pragma unroll
                for (int p = 0; p < kPairs; ++p) {
                    a[p] = mul2(both(k.h[i]), y[p]);
#pragma unroll
                    for (int j = 0; j < 4; ++j) a[p] = fma2(both(k.t[4 * i + j]), v[j][p], a[p]);
                }
                ch.put(to + static_cast<int64_t>(i) * C, s, has_x, has_y, a);
            }
        }
        if constexpr (!kVec) {
            __syncwarp();  // others have read what is copied over
            fill(stage);
        }
        stage = (stage + 1) % kMixFwdStages;
    }
}

// The backward pass: a warp takes whole tokens (of kVec 32 / lanes at a time),
// chunk after chunk.  kLong: tokens of more than a run of chunks (a kernel of its own:
// the sums over runs cost registers, and with them the third block of an SM:
// 20000 tokens of 512 bf16 73 us for 49).
template <class Elem, bool kVec, bool kWide, bool kLong>
__global__ void __launch_bounds__(kMixRingBlock)
mix_bwd_ring(const Elem* __restrict__ g, int64_t g_stride, int64_t g_stream_stride, RowSpan g_span, MixIn<Elem> in,
             RowSpan x_span, RowSpan y_span, Elem* __restrict__ dx, void* __restrict__ dT, Elem* __restrict__ dy,
             void* __restrict__ dh, Dropout d, int64_t N, int C, int lanes)
{
    extern __shared__ __align__(16) char ring_memory[];
    __shared__ MixMasks masks;
    using Chunk = MixChunk<Elem, kVec>;
    constexpr int kPairs = Chunk::kPairs, kPlace = Chunk::kPlace;
    constexpr int kStage = 9 * kPlace;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    const Chunk ch{C, lane, lanes};
    char* ring = ring_memory + warp * (kMixBwdStages * kStage);
    const uint2 key = dropout_key(d);
    const int chunks = Chunk::count(C, lanes);
    const int per_warp = kVec ? 32 / lanes : 1;  // tokens
    const int mine = kVec ? lane / lanes : 0;
    const int64_t groups = (N + per_warp - 1) / per_warp;
    const int64_t first = blockIdx.x * static_cast<int64_t>(warps) + warp, step = static_cast<int64_t>(gridDim.x) * warps;
    int64_t ahead = first;
    int ahead_chunk = 0;
    auto fill = [&](int stage) {
        const int64_t r = ahead * per_warp + mine;
        if (r < N) {
            const int c = ch.start(ahead_chunk, r * C);
            const bool x_amid = x_span.amid(r, N), y_amid = y_span.amid(r, N), g_amid = g_span.amid(r, N);
            char* to = ring + stage * kStage;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                ch.copy(to + j * kPlace, in.x + r * in.stride + j * in.stream_stride, c, x_span, x_amid);
                ch.copy(to + (5 + j) * kPlace, g + r * g_stride + j * g_stream_stride, c, g_span, g_amid);
            }
            ch.copy(to + 4 * kPlace, in.y + r * in.y_stride, c, y_span, y_amid);
        }
        copies_commit();
        if (++ahead_chunk == chunks) {
            ahead_chunk = 0;
            ahead += step;
        }
    };
#pragma unroll
    for (int s = 0; s < kMixBwdStages; ++s) fill(s);
    int stage = 0;
    for (int64_t group = first; group < groups; group += step) {
        const int64_t r = group * per_warp + mine;
        const MixCoef k = mix_coef<kWide>(in, min(r, N - 1));
        float2 acc[20];
        float sums[20];
        double total = 0.0;  // of the runs before
#pragma unroll
        for (int i = 0; i < 20; ++i) acc[i] = both(0.0f);
        for (int s = 0; s < chunks; ++s) {
            const int c = ch.start(s, r * C);
            copies_wait(kMixBwdStages);
            if constexpr (!kVec) __syncwarp();
            const char* place = ring + stage * kStage;
            const char *at_x[4], *at_g[4], *at_y = ch.at(place + 4 * kPlace, in.y + r * in.y_stride, c);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                at_x[j] = ch.at(place + j * kPlace, in.x + r * in.stride + j * in.stream_stride, c);
                at_g[j] = ch.at(place + (5 + j) * kPlace, g + r * g_stride + j * g_stream_stride, c);
            }
            typename Chunk::Keep keep;
            if (d.limit) keep = ch.keep(r * C, c, d, key, masks.of[warp]);
            Elem *to = dx + r * 4 * C + c, *to_y = dy + r * C + c;
            const int steps = ch.steps(c);
#pragma unroll
            for (int t = 0; t < Chunk::kSteps; ++t) {
                if (t >= steps) break;
                const bool has_x = r < N && ch.has_x(c, t), has_y = r < N && ch.has_y(c, t);
                const bool some = !(has_x && has_y);
                float2 gv[4][kPairs], y[kPairs], b[kPairs];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    ch.get(at_g[i], t, gv[i]);
                    if (some) ch.clear_rest(has_x, has_y, gv[i]);
                }
                ch.get(at_y, t, y);
                if (some) ch.clear_rest(has_x, has_y, y);
#pragma unroll
                for (int p = 0; p < kPairs; ++p) {
                    b[p] = mul2(both(k.h[0]), gv[0][p]);
#pragma unroll
                    for (int i = 1; i < 4; ++i) b[p] = fma2(both(k.h[i]), gv[i][p], b[p]);
                }
                if (d.limit) {
                    ch.drop(y, keep, t, d.scale);
                    ch.drop(b, keep, t, d.scale);
                }
                ch.put(to_y, t, has_x, has_y, b);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
#pragma unroll
                    for (int p = 0; p < kPairs; ++p) acc[16 + i] = fma2(gv[i][p], y[p], acc[16 + i]);
                }
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    float2 v[kPairs];
                    ch.get(at_x[j], t, v);
                    if (some) ch.clear_rest(has_x, has_y, v);
#pragma unroll
                    for (int p = 0; p < kPairs; ++p) {
                        b[p] = mul2(both(k.t[j]), gv[0][p]);
#pragma unroll
                        for (int i = 1; i < 4; ++i) b[p] = fma2(both(k.t[4 * i + j]), gv[i][p], b[p]);
#pragma unroll
                        for (int i = 0; i < 4; ++i) acc[4 * i + j] = fma2(gv[i][p], v[p], acc[4 * i + j]);
                    }
                    ch.put(to + static_cast<int64_t>(j) * C, t, has_x, has_y, b);
                }
            }
            if constexpr (!kVec) __syncwarp();  // others have read what is copied over
            fill(stage);
            stage = (stage + 1) % kMixBwdStages;
            if constexpr (kLong) {
                constexpr int run = kMixRun / (Chunk::kPairs * Chunk::kSteps);  // chunks
                if (s % run == run - 1 && s + 1 < chunks) {
#pragma unroll
                    for (int i = 0; i < 20; ++i) {
                        sums[i] = acc[i].x + acc[i].y;
                        acc[i] = both(0.0f);
                    }
                    total += warp_sum20(sums);
                }
            }
        }
#pragma unroll
        for (int i = 0; i < 20; ++i) sums[i] = acc[i].x + acc[i].y;
        put_token_sums<kLong>(in, r, r < N, lane, lanes, sums, dT, dh, total);
    }
}

}  // namespace mhcp
