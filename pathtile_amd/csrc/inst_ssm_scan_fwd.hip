// Instantiates the selective scan's forward and its chunks' states.
#include "ssm_scan.hpp"
#include "ssm_tables.hpp"

namespace pt {
#define ROW(T, MANY) {&scan_fwd_kernel<T, MANY, false>, &scan_fwd_kernel<T, MANY, true>}
const ScanFwdFn kScanFwd[2][2][2] = {{ROW(float, false), ROW(float, true)},
                                    {ROW(__bf16, false), ROW(__bf16, true)}};
#undef ROW
#define ROW(T, MANY) \
  {&scan_chunk_kernel<T, MANY, false, false>, &scan_chunk_kernel<T, MANY, true, false>}
const ScanChunkFn kScanChunkFwd[2][2][2] = {{ROW(float, false), ROW(float, true)},
                                         {ROW(__bf16, false), ROW(__bf16, true)}};
}  // namespace pt
