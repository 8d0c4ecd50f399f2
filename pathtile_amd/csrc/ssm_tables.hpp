// ssm_tables.hpp — dispatch tables of the selective scan, each defined in its
// own translation unit (inst_ssm_scan_*.hip).
#pragma once

namespace pt {

struct ScanFwdArgs;
struct ScanBwdArgs;
using ScanFwdFn = void (*)(ScanFwdArgs);
using ScanBwdFn = void (*)(ScanBwdArgs);

// [FP32; BF16; BF16 with B and C as FP32][16, 32, 64 states][single, vector]
extern const ScanFwdFn kScanFwd[3][3][2];
extern const ScanBwdFn kScanBwd[3][3][2];

}  // namespace pt
