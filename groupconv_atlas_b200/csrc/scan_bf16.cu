// The selective scan's kernels for one element type (see kernel_scan.cuh).
#include "kernel_scan.cuh"

namespace gcb {

template ScanLaunch scan_launch<__nv_bfloat16>(ScanKernel, int);

}  // namespace gcb
