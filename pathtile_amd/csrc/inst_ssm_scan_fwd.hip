// Instantiates the selective scan's forward.
#include "ssm_scan.hpp"
#include "ssm_tables.hpp"

namespace pt {
#define ROW(T, BCT, NS) {&scan_fwd_kernel<T, BCT, NS, false>, &scan_fwd_kernel<T, BCT, NS, true>}
#define TYPES(T, BCT) {ROW(T, BCT, 4), ROW(T, BCT, 8), ROW(T, BCT, 16)}
const ScanFwdFn kScanFwd[3][3][2] = {TYPES(float, float), TYPES(__bf16, __bf16), TYPES(__bf16, float)};
}  // namespace pt
