// ssm_tables.hpp — dispatch tables of the selective scan, each defined in its
// own translation unit (inst_ssm_scan_*.hip).
#pragma once

namespace pt {

struct ScanFwdArgs;
struct ScanBwdArgs;
struct ScanChunkArgs;
using ScanFwdFn = void (*)(ScanFwdArgs);
using ScanBwdFn = void (*)(ScanBwdArgs);
using ScanChunkFn = void (*)(ScanChunkArgs);

// [FP32, BF16][up to 16 states, more][single, vector loads]
extern const ScanFwdFn kScanFwd[2][2][2];
extern const ScanBwdFn kScanBwd[2][2][2];
extern const ScanChunkFn kScanChunkFwd[2][2][2];
extern const ScanChunkFn kScanChunkBwd[2][2][2];

}  // namespace pt
