// Host-side helpers shared by the entry points (see host_util.h).
#include "host_util.h"

#include <cstdio>
#include <cstring>
#include <map>
#include <mutex>
#include <tuple>

namespace gcb {

namespace {
std::mutex g_mutex;
std::map<int, DeviceFacts> g_facts;
std::map<std::pair<int, const void *>, bool> g_attr_done;
std::map<std::tuple<int, const void *, int, size_t>, int> g_occupancy;
}  // namespace

PlanRecord &last_plan() {
    thread_local PlanRecord record;
    return record;
}

std::string format_plan(const PlanRecord &r) {
    char buf[400];
    const long long *v = r.v;
    switch (r.kind) {
    case PlanRecord::kDirect:
        std::snprintf(buf, sizeof(buf),
                      "kernel=direct_%s engine=group variant=%s grid=%lld block=%lld smem=%lld ctas_per_sm=%lld "
                      "cb=%lld bh=%lld items=%lld cells=%lld stages=%lld pitch=%lld rows=%lld bulk_w=%lld "
                      "vec_store=%lld",
                      r.tma ? "tma" : "ldg", r.name, v[0], v[1], v[2], v[3], v[4], v[5], v[6], v[7], v[8], v[9],
                      v[10], v[11], v[12]);
        break;
    case PlanRecord::kWide:
        std::snprintf(buf, sizeof(buf),
                      "kernel=direct_%s engine=wide variant=%s grid=%lld block=%lld smem=%lld ctas_per_sm=%lld "
                      "kc=%lld chunks=%lld co_item=%lld bh=%lld items=%lld cells=%lld pitch=%lld rows=%lld "
                      "vec_store=%lld",
                      r.tma ? "tma" : "ldg", r.name, v[0], v[1], v[2], v[3], v[4], v[5], v[6], v[7], v[8], v[9],
                      v[10], v[11], v[12]);
        break;
    case PlanRecord::kTf32:
        std::snprintf(buf, sizeof(buf),
                      "kernel=tf32x3 engine=tcgen05 n_cta=%lld block=320 smem=%lld M=%lld N=%lld nb=%lld sp=%lld "
                      "strips=%lld items=%lld chunks=%lld rows_b=%lld ks=%lld layout=%s",
                      v[0], v[1], v[2], v[3], v[4], v[5], v[6], v[7], v[8], v[9], v[10], r.name);
        break;
    case PlanRecord::kSmall:
        std::snprintf(buf, sizeof(buf),
                      "kernel=small grid=%lld block=%lld smem=%lld ctas_per_sm=%lld cob=%lld cb=%lld items=%lld "
                      "vec=%lld stages=%lld",
                      v[0], v[1], v[2], v[3], v[4], v[5], v[6], v[7], v[8]);
        break;
    case PlanRecord::kDw:
        std::snprintf(buf, sizeof(buf),
                      "kernel=general engine=depthwise k=%lld grid=%lld block=%lld smem=%lld bh=%lld bands=%lld "
                      "pitch=%lld items=%lld",
                      v[0], v[1], v[7], v[2], v[3], v[4], v[5], v[6]);
        break;
    case PlanRecord::kDwS2:
        std::snprintf(buf, sizeof(buf),
                      "kernel=general engine=depthwise_cells k=%lld stride=%lld grid=%lld block=256 cells=%lld "
                      "vec_in=%lld vec_out=%lld",
                      v[0], v[5], v[1], v[2], v[3], v[4]);
        break;
    case PlanRecord::kNhwc:
        std::snprintf(buf, sizeof(buf), "kernel=nhwc engine=%s grid=%lld block=%lld cpg=%lld bias=%lld rows=%lld",
                      r.name, v[0], v[1], v[2], v[3], v[4]);
        break;
    case PlanRecord::kNorm:
        std::snprintf(buf, sizeof(buf),
                      "kernel=group_norm engine=%s grid=%lld block=%lld smem=%lld cluster=%lld channels=%lld rows=%lld "
                      "vec=%lld launches=%lld rounds=%lld",
                      r.name, v[0], v[1], v[2], v[3], v[4], v[5], v[6], v[7], v[8]);
        break;
    case PlanRecord::kDropout:
        std::snprintf(buf, sizeof(buf), "kernel=dropout engine=%s grid=%lld block=%lld vec=%lld", r.name, v[0], v[1],
                      v[2]);
        break;
    case PlanRecord::kGeneral:
        std::snprintf(buf, sizeof(buf), "kernel=general grid=%lld block=%lld run=%lld cob=%lld index=%s runs=%lld",
                      v[0], v[1], v[2], v[3], v[4] ? "32" : "64", v[5]);
        break;
    default:
        buf[0] = '\0';
    }
    return buf;
}

int device_facts(int dev, DeviceFacts &out) {
    std::lock_guard<std::mutex> lock(g_mutex);
    auto it = g_facts.find(dev);
    if (it != g_facts.end()) {
        out = it->second;
        return GC_OK;
    }
    DeviceFacts f;
    cudaError_t e = cudaDeviceGetAttribute(&f.sms, cudaDevAttrMultiProcessorCount, dev);
    if (e == cudaSuccess)
        e = cudaDeviceGetAttribute(&f.smem_optin, cudaDevAttrMaxSharedMemoryPerBlockOptin, dev);
    if (e == cudaSuccess)
        e = cudaDeviceGetAttribute(&f.smem_per_sm, cudaDevAttrMaxSharedMemoryPerMultiprocessor, dev);
    if (e != cudaSuccess) return gc_error(GC_DEVICE_ERROR, cudaGetErrorString(e));
    g_facts[dev] = f;
    out = f;
    return GC_OK;
}

int kernel_occupancy(int dev, const void *fn, int threads, size_t smem, int smem_optin,
                     int &ctas) {
    std::lock_guard<std::mutex> lock(g_mutex);
    auto key = std::make_tuple(dev, fn, threads, smem);
    auto it = g_occupancy.find(key);
    if (it != g_occupancy.end()) {
        ctas = it->second;
        return GC_OK;
    }
    auto akey = std::make_pair(dev, fn);
    if (!g_attr_done[akey]) {
        cudaError_t e =
            cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, smem_optin);
        if (e != cudaSuccess) return gc_error(GC_DEVICE_ERROR, cudaGetErrorString(e));
        g_attr_done[akey] = true;
    }
    int n = 0;
    cudaError_t e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, fn, threads, smem);
    if (e != cudaSuccess) return gc_error(GC_DEVICE_ERROR, cudaGetErrorString(e));
    g_occupancy[key] = n;
    ctas = n;
    return GC_OK;
}

cudaError_t launch_pdl(const void *fn, dim3 grid, dim3 block, void **args, size_t smem, cudaStream_t stream,
                       int cluster) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if (cluster > 1) {
        attr[1].id = cudaLaunchAttributeClusterDimension;
        attr[1].val.clusterDim.x = static_cast<unsigned>(cluster);
        attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
        cfg.numAttrs = 2;
    }
    return cudaLaunchKernelExC(&cfg, fn, args);
}

int check_device_memory(const void *p, int device_index, int current) {
    cudaPointerAttributes attr;
    std::memset(&attr, 0, sizeof(attr));
    cudaError_t e = cudaPointerGetAttributes(&attr, p);
    if (e != cudaSuccess) {
        cudaGetLastError();  // the failed query must not poison the next launch check
        return gc_error(GC_DEVICE_ERROR, cudaGetErrorString(e));
    }
    if (attr.type != cudaMemoryTypeDevice || attr.device != device_index || attr.device != current)
        return gc_error(GC_INVALID, "CUDA pointer must be device memory on descriptor/current device");
    return GC_OK;
}

int check_pointer(const gc_tensor *t, int current) { return check_device_memory(t->data, t->device_index, current); }

}  // namespace gcb
