// Internal interface between the scan's C entry points (gdn_scan.cu) and its
// tensor-core kernels (gdn_scan_tc.cu).
#pragma once

#include "gdn_internal.h"

namespace gdn {
namespace scan {

struct ScanParams;

// Whether types and sizes suit the tensor-core kernels, and whether the
// buffers' alignment does (the recurrent kernels run otherwise).
bool tc_shape(const gdn_scan_args& a);
bool tc_layout(const gdn_scan_args& a);
int64_t tc_slices(const gdn_scan_args& a);
// Per-token scalars of the tensor-core kernels: so many bytes of workspace.
size_t tc_scratch_bytes(const gdn_scan_args& a);
cudaError_t launch_tc(const ScanParams& p, const gdn_scan_args& a, float* scratch, cudaStream_t s);
// The states that segments start from, from those they add.
void launch_pass(const ScanParams& p, cudaStream_t s);

}  // namespace scan
}  // namespace gdn
