// Every vector that the delta rule's scans fetch of a chunk's record lies inside the planes
// of its matrix, or is one that the hardware's range check drops. Compiled only.
#include "delta.h"

using namespace snhip;

template <int Q, int NTH> constexpr bool inside(int at) {
    for (int i = 0; i < MatFetch<Q, NTH>::N * NTH; i++) {
        const int o = MatFetch<Q, NTH>::offset(i, at);
        if (o != kNowhere && (o < at * 4 || o + 16 > (at + Q * 512) * 4)) return false;
    }
    return (at + Q * 512) * 4 <= kDeltaChunk * 4;
}

constexpr int kThreads = 64 * kDeltaW;
static_assert(inside<3, kThreads>(0) && inside<3, kThreads>(kDeltaP), "three planes of M and P");
static_assert(inside<2, kThreads>(0) && inside<2, kThreads>(kDeltaP), "two planes");
static_assert(inside<3, 512>(kDeltaP) && inside<3, 128>(kDeltaP) && inside<3, 64>(kDeltaP), "other block sizes");
