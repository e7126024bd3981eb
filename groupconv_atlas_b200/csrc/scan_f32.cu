// The selective scan's kernels for one element type (see kernel_scan.cuh).
#include "kernel_scan.cuh"

namespace gcb {

template ScanLaunch scan_launch<float>(ScanKernel, int);

}  // namespace gcb
