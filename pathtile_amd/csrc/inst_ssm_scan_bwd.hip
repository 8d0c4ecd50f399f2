// Instantiates the selective scan's backward.
#include "ssm_scan.hpp"
#include "ssm_tables.hpp"

namespace pt {
#define ROW(T, BCT, R) {&scan_bwd_kernel<T, BCT, R, false>, &scan_bwd_kernel<T, BCT, R, true>}
#define TYPES(T, BCT) {ROW(T, BCT, 1), ROW(T, BCT, 2), ROW(T, BCT, 4)}
const ScanBwdFn kScanBwd[3][3][2] = {TYPES(float, float), TYPES(__bf16, __bf16), TYPES(__bf16, float)};
}  // namespace pt
