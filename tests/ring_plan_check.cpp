// Host check of the norms' ring launches (ring_plan.h) for every width: a
// launch fits in a block's shared memory, by default or after asking for more, and its
// groups hold a row.
#include "ring_plan.h"

#include <cstdio>
#include <cstdlib>

using namespace mhcp;

#define CHECK(cond)                                                                                        \
    do {                                                                                                   \
        if (!(cond)) {                                                                                     \
            std::printf("%s: streams %d backward %d bytes %d form %d width %d\n", #cond, kStreams,         \
                        static_cast<int>(kWidths == 3), elem, static_cast<int>(form), static_cast<int>(C)); \
            std::exit(1);                                                                                  \
        }                                                                                                  \
    } while (0)

// The first width whose rows the ring does not take.
template <template <int, int> class Shape, int kStreams, int kWidths>
int64_t check(int elem, RowForm form)
{
    int64_t end = 0;
    for (int64_t C = 1; C < 17000; ++C) {
        if (form == kPieces && C * elem % 16) continue;
        const RingPlan p = ring_plan<Shape, kStreams, kWidths>(C, elem, form);
        if (p.stages == 0) {
            if (!end) end = C;
            continue;
        }
        CHECK(!end);
        const int static_bytes = static_cast<int>(p.width == 0   ? sizeof(typename Shape<kStreams, 0>::Sums)
                                                  : p.width == 1 ? sizeof(typename Shape<kStreams, 1>::Sums)
                                                                 : sizeof(typename Shape<kStreams, kWidths - 1>::Sums));
        // the documented limits, not the header's own constants
        CHECK(asks_for_smem(static_bytes, p.smem) || static_bytes + p.smem <= 48 * 1024);
        CHECK(p.smem <= kMostSmem && static_bytes + kMostSmem <= 227 * 1024);
        // what the plan counts as resident on an SM, with the 1 KB the system takes of each block
        CHECK(p.blocks_per_sm == 1 || p.blocks_per_sm * (static_bytes + p.smem + 1024) <= 228 * 1024);
        CHECK(p.threads * p.groups <= kRingThreads && p.threads * p.groups * p.blocks_per_sm <= kRingThreads);
        CHECK(p.threads > 32 ? p.threads % 32 == 0 : 32 % p.threads == 0);
        CHECK(p.threads <= 32 || (p.groups <= kMaxGroups<kStreams> && p.groups < 16));  // a named barrier each
        CHECK(p.threads * p.elems >= C + (form == kSkewed ? 16 / elem - 1 : 0));
        CHECK(p.stages >= 1 && p.stages <= kRingStages);
        const int rows = kWidths == 3 || p.width ? Shape<kStreams, 1>::kRows : Shape<kStreams, 0>::kRows;
        CHECK(p.smem >= p.stages * p.groups * rows *
                            ring_row_bytes(static_cast<int>(C), elem, form == kLoose, p.threads, p.elems));
        CHECK(kWidths == 2 || p.smem >= p.groups * 2 * part_pitch(static_cast<int>(C)) * 4);
        for (int64_t turns : {1, 7, 1000, 1 << 30}) {
            const int64_t grid = p.grid(turns, elem, 148);
            CHECK(grid >= 1 && grid <= std::max<int64_t>(8, static_cast<int64_t>(p.blocks_per_sm) * 148));
            CHECK(form != kSkewed || grid * p.groups % (16 / elem) == 0);
        }
        // the backward's blocks each have a row of the workspace
        for (int64_t N : {1, 3, 17, 300, 500, 1 << 20}) {
            const int64_t blocks = std::min(p.grid(N, elem, 148), kMaxPartials);
            CHECK(blocks == p.grid(N, elem, 148) && blocks <= norm_partial_rows(N, C));
            CHECK(param_chunks(N) <= norm_partial_rows(N, C));
            const int64_t most = std::min(p.grid(N, elem, 1000), kMaxPartials);
            CHECK(most <= norm_partial_rows(N, C) && (form != kSkewed || most * p.groups % (16 / elem) == 0));
        }
    }
    return end;
}

int main()
{
    for (int elem : {2, 4}) {
        for (RowForm form : {kLoose, kSkewed, kPieces}) {
            const int64_t widest = form == kSkewed ? 16384 - 16 / elem + 2 : form == kPieces ? 16384 + 16 / elem : 16385;
            if (check<FwdShape, 1, 2>(elem, form) != widest || check<BwdShape, 1, 3>(elem, form) != widest) {
                std::printf("one stream leaves the ring elsewhere\n");
                return 1;
            }
            if (form == kSkewed) continue;
            // in 32 bits four streams, and G with them in the backward, outgrow a block earlier
            const int64_t f = check<FwdShape, 4, 2>(elem, form), b = check<BwdShape, 4, 3>(elem, form);
            const bool loose = form == kLoose;
            if (elem == 2 ? f != widest || b != widest : f != (loose ? 12797 : 12292) || b != (loose ? 10237 : 10244)) {
                std::printf("four streams leave the ring at %d and %d\n", static_cast<int>(f), static_cast<int>(b));
                return 1;
            }
        }
    }
    std::printf("ok\n");
    return 0;
}
