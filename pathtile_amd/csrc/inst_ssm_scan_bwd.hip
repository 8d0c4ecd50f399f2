// Instantiates the selective scan's backward and its chunks' states.
#include "ssm_scan.hpp"
#include "ssm_tables.hpp"

namespace pt {
#define ROW(T, MANY) {&scan_bwd_kernel<T, MANY, false>, &scan_bwd_kernel<T, MANY, true>}
const ScanBwdFn kScanBwd[2][2][2] = {{ROW(float, false), ROW(float, true)},
                                    {ROW(__bf16, false), ROW(__bf16, true)}};
#undef ROW
#define ROW(T, MANY) \
  {&scan_chunk_kernel<T, MANY, false, true>, &scan_chunk_kernel<T, MANY, true, true>}
const ScanChunkFn kScanChunkBwd[2][2][2] = {{ROW(float, false), ROW(float, true)},
                                         {ROW(__bf16, false), ROW(__bf16, true)}};
}  // namespace pt
