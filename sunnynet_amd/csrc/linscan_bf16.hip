// Linear attention's recurrence for __bf16 operands (a file per type: they compile at once).
#include "linscan.h"

namespace snhip {

snhip_status lin_run_bf16(const LinShape& d, const LinPass& a, bool rev, int kind, hipStream_t st) {
    return lin_run<__bf16>(d, a, rev, kind, st);
}

}  // namespace snhip
