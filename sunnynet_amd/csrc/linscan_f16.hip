// Linear attention's recurrence for _Float16 operands (a file per type: they compile at once).
#include "linscan.h"

namespace snhip {

snhip_status lin_run_f16(const LinShape& d, const LinPass& a, bool rev, int kind, hipStream_t st) {
    return lin_run<_Float16>(d, a, rev, kind, st);
}

}  // namespace snhip
