// Linear attention's recurrence for float operands (a file per type: they compile at once).
#include "linscan.h"

namespace snhip {

snhip_status lin_run_f32(const LinShape& d, const LinPass& a, bool rev, int kind, hipStream_t st) {
    return lin_run<float>(d, a, rev, kind, st);
}

}  // namespace snhip
