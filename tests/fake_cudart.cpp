// A stand-in for the CUDA runtime calls that the library makes around its
// launches, preloaded into a process without a GPU: every pointer is device
// memory of device 0, a B200's limits, and launches that do nothing or fail.
//   fake_launch_error  what cudaLaunchKernelExC returns
//   fake_throw         cudaGetDevice throws what a failed allocation throws
//   fake_no_memory     operator new throws
//   fake_launches      launches so far
//   fake_live          allocations that live
#include <cuda_runtime.h>

#include <cstdlib>
#include <new>

extern "C" {
int fake_launch_error = 0, fake_throw = 0, fake_no_memory = 0, fake_launches = 0, fake_live = 0;

cudaError_t cudaGetDevice(int *device) {
    if (fake_throw) throw std::bad_alloc();
    *device = 0;
    return cudaSuccess;
}
cudaError_t cudaDeviceGetAttribute(int *value, cudaDeviceAttr attr, int) {
    *value = attr == cudaDevAttrMultiProcessorCount             ? 148
             : attr == cudaDevAttrMaxSharedMemoryPerBlockOptin ? 232448
                                                                : 233472;
    return cudaSuccess;
}
cudaError_t cudaPointerGetAttributes(cudaPointerAttributes *attr, const void *) {
    attr->type = cudaMemoryTypeDevice;
    attr->device = 0;
    return cudaSuccess;
}
cudaError_t cudaStreamIsCapturing(cudaStream_t, cudaStreamCaptureStatus *status) {
    *status = cudaStreamCaptureStatusNone;
    return cudaSuccess;
}
cudaError_t cudaFuncSetAttribute(const void *, cudaFuncAttribute, int) { return cudaSuccess; }
cudaError_t cudaGetLastError(void) { return cudaSuccess; }
cudaError_t cudaMemsetAsync(void *, int, size_t, cudaStream_t) { return cudaSuccess; }
cudaError_t cudaLaunchKernelExC(const cudaLaunchConfig_t *, const void *, void **) {
    if (fake_launch_error) return static_cast<cudaError_t>(fake_launch_error);
    ++fake_launches;
    return cudaSuccess;
}
}

void *operator new(size_t bytes) {
    void *p = fake_no_memory ? nullptr : std::malloc(bytes);
    if (p == nullptr) throw std::bad_alloc();
    __atomic_add_fetch(&fake_live, 1, __ATOMIC_RELAXED);
    return p;
}
void operator delete(void *p) noexcept {
    if (p != nullptr) __atomic_sub_fetch(&fake_live, 1, __ATOMIC_RELAXED);
    std::free(p);
}
void operator delete(void *p, size_t) noexcept { operator delete(p); }
