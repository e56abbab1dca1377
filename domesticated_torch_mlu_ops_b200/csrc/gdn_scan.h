// Internal interface between the scan's C entry points (gdn_scan.cu) and its
// tensor-core kernels (gdn_scan_tc.cu).
#pragma once

#include "gdn_internal.h"

namespace gdn {
namespace scan {

struct ScanParams;

inline bool tc_applies(const gdn_scan_args&) { return false; }
inline int64_t tc_slices(const gdn_scan_args&) { return 1; }
// The states that segments start from, from those they add.
void launch_pass(const ScanParams& p, cudaStream_t s);

}  // namespace scan
}  // namespace gdn
