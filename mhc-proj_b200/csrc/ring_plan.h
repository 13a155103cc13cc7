// The launches of the norms' ring kernels (norm_ring.cuh) by width, type and
// form of the rows: host arithmetic without CUDA, so that a host compiler can
// check it for every width.
#pragma once

#include <algorithm>
#include <cstdint>

#ifdef __CUDACC__
#define MHCP_BOTH __host__ __device__
#else
#define MHCP_BOTH
#endif

namespace mhcp {

// How a kernel takes rows (row_cols.cuh):
//   kLoose    any rows: single columns
//   kSkewed   16-byte pieces as they lie in memory
//   kPieces   rows of whole, aligned pieces
//   kWhole    the same, and exactly as many as the group's threads take
enum RowForm { kLoose, kSkewed, kPieces, kWhole };

// Shared memory of a block: what a kernel may take without asking, static and
// dynamic together, what it may take at all, and the dynamic part that every
// launch which has to ask asks for (row_copy.cuh).
constexpr int kDefaultSmem = 48 * 1024, kLargestSmem = 227 * 1024, kMostSmem = 200 * 1024;

// Whether a launch has to ask.
constexpr bool asks_for_smem(int static_bytes, int dynamic_bytes) { return static_bytes + dynamic_bytes > kDefaultSmem; }

constexpr int kRingThreads = 512;  // of an SM, in its rings' blocks
constexpr int kRingStages = 4;     // at most

// Groups of more than a warp in a block, at most (the memory for their sums).
template <int kStreams>
constexpr int kMaxGroups = kStreams == 1 ? 8 : 5;

// Where the groups of a block exchange kSums sums, twice: the ring kernels' static memory.
template <int kStreams, int kSums>
struct GroupSums {
    alignas(16) float of[kMaxGroups<kStreams>][2][kSums * 32];
};

// Bytes of one row's place in a stage.
MHCP_BOTH inline int ring_row_bytes(int C, int elem, bool loose, int threads, int per_thread)
{
    return loose ? (C * elem + 15) / 16 * 16 + 16 : threads * per_thread * elem;
}

// Floats of a row of partial sums in shared memory: the columns, from the start of
// a skewed row's first piece, in whole pieces.
MHCP_BOTH inline int part_pitch(int C) { return (C + 15) / 8 * 8; }

// The ring kernels' shapes by width: elements of a row per thread, the most
// threads of a group (their product is the widest row), rows a turn, and
// whether the parameters stay in registers.  512 threads of an SM have 128
// registers each.  One stream's shapes of up to 8192 columns and four streams' of
// up to 4096 fit in them (16 elements a thread for the four streams' gradients
// spill, so narrower rows do not take them: 506 us against 440, 65536 x 2048 bf16);
// wider rows spill what they need.
template <int kStreams, int kWidth>
struct FwdShape {
    static constexpr int kElems = kWidth ? 32 : 16, kTurn = kStreams == 1 && !kWidth ? 2 : 1;
    static constexpr int kMaxThreads = kStreams == 1 && !kWidth ? 256 : 512;
    static constexpr bool kHold = true;
    static constexpr int kRows = kStreams * kTurn;  // of a stage
    static constexpr bool kParts = false;           // of the parameters' gradients, in shared memory at the end
    static constexpr int64_t kWidest = kElems * kMaxThreads;
    using Sums = GroupSums<kStreams, kTurn>;
};
template <int kStreams, int kWidth>
struct BwdShape {
    static constexpr int kElems = kWidth == 2 ? 32 : kStreams == 1 || kWidth == 1 ? 16 : 8;
    static constexpr int kMaxThreads = kStreams == 1 && !kWidth ? 256 : 512;
    static constexpr bool kHold = kWidth == 0 || (kStreams == 1 && kWidth == 1);
    static constexpr int kRows = kStreams + 1;
    static constexpr bool kParts = true;
    static constexpr int64_t kWidest = kElems * kMaxThreads;
    using Sums = GroupSums<kStreams, kStreams == 1 ? 2 : 16>;
};

// A ring kernel's launch.
struct RingPlan {
    RowForm form;
    int width, elems, threads, groups, stages, blocks_per_sm, smem;

    // Blocks for `turns` turns of the groups.
    int64_t grid(int64_t turns, int elem, int sms) const
    {
        const int64_t blocks = std::min((turns + groups - 1) / groups, static_cast<int64_t>(blocks_per_sm) * sms);
        if (form != kSkewed) return blocks;
        // the groups' turns go in steps of whole periods of 16 / elem rows
        const int period = 16 / elem, unit = period / std::min(period, groups & -groups);
        return std::max<int64_t>(unit, blocks / unit * unit);
    }
};

// Of an SM's 227 KB, for the rings: more bytes under way are slower again (one
// stream, fp32, 16384 x 4096 forward: 100 KB 90 us, 204 KB 98; four streams, fp32,
// 16384 x 2048 backward: 150 KB 184 us, 204 KB 219).
constexpr int ring_smem(int streams) { return (streams == 1 ? 100 : 150) * 1024; }

// The shape (of kWidths) and launch for rows of C elements in `form`; stages 0: too wide.
template <template <int, int> class Shape, int kStreams, int kWidths>
inline RingPlan ring_plan(int64_t C, int elem, RowForm form)
{
    RingPlan p{};
    const int64_t span = C + (form == kSkewed ? 16 / elem - 1 : 0);  // columns from a piece's start
    if (span > Shape<kStreams, kWidths - 1>::kWidest) return p;
    int rows = Shape<kStreams, 0>::kRows;
    p.elems = Shape<kStreams, 0>::kElems;
    if (span > Shape<kStreams, 0>::kWidest) {
        p.width = 1;
        rows = Shape<kStreams, 1>::kRows;
        p.elems = Shape<kStreams, 1>::kElems;
    }
    if (kWidths > 2 && span > Shape<kStreams, 1>::kWidest) {
        p.width = 2;
        rows = Shape<kStreams, kWidths - 1>::kRows;
        p.elems = Shape<kStreams, kWidths - 1>::kElems;
    }
    const int64_t want = (span + p.elems - 1) / p.elems;
    p.threads = form == kLoose ? 32 : 4;
    while (p.threads < 32 && p.threads < want) p.threads *= 2;
    if (want > 32) p.threads = 32 * static_cast<int>((want + 31) / 32);
    p.form = form == kPieces && p.threads * p.elems == C ? kWhole : form;
    const int row_stage = rows * ring_row_bytes(static_cast<int>(C), elem, form == kLoose, p.threads, p.elems);
    const int least = kStreams == 1 ? 1 : 2;  // stages
    // Blocks of about 256 threads, or of up to 512 where two of the smaller leave
    // threads of the SM without work (groups of 96, bf16, 20003 x 1025: forward 39
    // us in blocks of five, 43 in two of two; backward 57 and 61.  65536 x 4096
    // backward, as many threads either way: 269 in one block, 263 in two).
    p.groups = std::max(1, 256 / p.threads);
    if (kRingThreads / p.threads > kRingThreads / (p.threads * p.groups) * p.groups) p.groups = kRingThreads / p.threads;
    if (p.threads > 32) p.groups = std::min(p.groups, kMaxGroups<kStreams>);
    // two stages of all groups' rows have to fit (four streams in fp32)
    while (p.groups > 1 && least * row_stage * p.groups > ring_smem(kStreams)) p.groups /= 2;
    const int stage = row_stage * p.groups;
    p.blocks_per_sm = std::max(1, std::min(kRingThreads / (p.threads * p.groups), ring_smem(kStreams) / (least * stage)));
    p.stages = std::min(kRingStages, std::max(1, ring_smem(kStreams) / p.blocks_per_sm / stage));
    p.smem = std::max(p.stages * stage, Shape<kStreams, 0>::kParts ? p.groups * 8 * part_pitch(static_cast<int>(C)) : 0);
    if (p.smem > kMostSmem) p.stages = 0;
    return p;
}

// Rows of partial sums of the parameters' gradients: one for every block of a
// ring kernel (three for each of 160 SMs, whole periods of skewed rows), or of
// the wide rows' kernels one for every chunk of rows.
constexpr int64_t kMaxPartials = 3 * 160;
constexpr int kParamRows = 8;
constexpr int64_t kParamChunks = 64;

inline int64_t param_chunks(int64_t N) { return std::min((N + kParamRows - 1) / kParamRows, kParamChunks); }

// At most, for N rows of C elements of any type in any form.
inline int64_t norm_partial_rows(int64_t N, int64_t C)
{
    return C > BwdShape<1, 2>::kWidest ? std::max<int64_t>(1, param_chunks(N)) : std::min(std::max<int64_t>(N, 16), kMaxPartials);
}

}  // namespace mhcp
