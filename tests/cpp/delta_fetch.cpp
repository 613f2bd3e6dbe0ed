// Every vector that the delta rule's scans fetch of a chunk's record lies inside the planes
// of its matrix, or is one that the hardware's range check drops. Compiled only.
#include "delta.h"

using namespace snhip;

template <int NTH> constexpr bool inside(int at) {
    constexpr int bytes = 3 * kDC * kDC * 2;       // of a matrix
    for (int i = 0; i < MatFetch<NTH>::N * NTH; i++) {
        const int o = MatFetch<NTH>::offset(i, at);
        if (o != kNowhere && (o < at * 4 || o + 16 > at * 4 + bytes)) return false;
    }
    return at * 4 + bytes <= kDeltaChunk * 4;
}

static_assert(inside<64 * kDeltaW>(0) && inside<64 * kDeltaW>(kDeltaP), "M and P");
static_assert(inside<512>(kDeltaP) && inside<128>(kDeltaP) && inside<64>(kDeltaP), "other block sizes");
