// Host-side helpers shared by the entry points: launch-plan records, cached
// device facts, the launch wrapper, and the pointer and stream checks of the
// ABI contract.
#pragma once
#include "groupconv.h"

#include <cuda_runtime.h>

#include <cstdint>
#include <string>

namespace gcb {

// The last launch's plan on this thread, kept as numbers and formatted only
// when gc_b200_last_plan asks for it (formatting costs about a third of a
// microsecond, a tenth of the host time of a call).
struct PlanRecord {
    enum Kind { kNone, kDirect, kWide, kTf32, kSmall, kGeneral, kDw, kDwS2, kNhwc, kNorm, kDropout } kind = kNone;
    const char *name = "";  // variant name, static storage
    bool tma = false;
    long long v[14] = {};
};
PlanRecord &last_plan();  // this thread's record
std::string format_plan(const PlanRecord &r);

template <class... T>
void record_plan(PlanRecord::Kind kind, const char *name, bool tma, T... values) {
    PlanRecord &last = last_plan();
    last.kind = kind;
    last.name = name;
    last.tma = tma;
    const long long vals[] = {static_cast<long long>(values)...};
    for (size_t i = 0; i < sizeof...(T); ++i) last.v[i] = vals[i];
}

inline long long round_up(long long v, long long m) { return (v + m - 1) / m * m; }
inline long long ceil_div(long long a, long long b) { return (a + b - 1) / b; }
inline bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

struct DeviceFacts {
    int sms = 0;
    int smem_optin = 0;   // max dynamic shared memory per block (opt-in)
    int smem_per_sm = 0;  // shared memory per multiprocessor
};
int device_facts(int dev, DeviceFacts &out);  // cached per device

// Opt a kernel into the device's full dynamic shared memory once, then ask
// the occupancy calculator (cached) how many CTAs fit per SM.
int kernel_occupancy(int dev, const void *fn, int threads, size_t smem, int smem_optin, int &ctas);

// Launch on the caller's stream with programmatic stream serialization: the
// kernel may start its prologue while the previous kernel in the stream
// drains, and waits (griddepcontrol.wait) before touching global memory.
// cluster > 1 launches clusters of that many CTAs along x.
cudaError_t launch_pdl(const void *fn, dim3 grid, dim3 block, void **args, size_t smem, cudaStream_t stream,
                       int cluster = 1);

// Device memory on the descriptor's device, which must be the current device
// (reference groupconv.cu:130-139).  Managed and mapped host memory are
// outside the contract.
int check_pointer(const gc_tensor *t, int current);
int check_device_memory(const void *p, int device_index, int current);

}  // namespace gcb
