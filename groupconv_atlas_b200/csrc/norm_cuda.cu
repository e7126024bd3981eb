// gc_b200_group_norm, its gradient, and gc_b200_dropout: descriptor checks,
// plans and launches.  As in the convolution backend nothing here allocates
// device memory or synchronizes, and a call can be captured into a CUDA graph.
// What is kept between calls: the plans of shapes, as many as kPlans, and which
// kernels have been opted into their shared memory.
#include "groupconv.h"

#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <initializer_list>
#include <map>
#include <mutex>
#include <numeric>
#include <tuple>

#include "host_util.h"
#include "kernel_dropout.cuh"
#include "kernel_norm.cuh"
#include "tensor_checks.cuh"

namespace {

using gcb::ceil_div;
using gcb::DropParams;
using gcb::DropoutParams;
using gcb::NormParams;
using gcb::PlanRecord;
using gcb::Range;
using gcb::wide;
using gcb::check_call;
using gcb::check_fields;
using gcb::check_workspace;
using gcb::elem_size;
using gcb::elem_type;
using gcb::internal_error;
using gcb::launched;
using gcb::outputs_meet;
using gcb::range_of;
using gcb::ranges_meet;
using gcb::same_dims;
using gcb::up16;

// ---- descriptors ------------------------------------------------------------------------
// A channels-last tensor as images of evenly spaced pixels.
struct View {
    char *data = nullptr;
    long long n = 0, c = 0, px = 0;
    long long ldn = 0, ldp = 0;  // element strides of an image and of a pixel
    int type = 0;
    uint64_t span = 0;  // bytes from the first to the end of the last element
};

int view_of(const gc_tensor *t, View &v) {
    const int64_t *d = t->dims, *s = t->strides;
    if (t->dtype == GC_F64) return gc_error(GC_UNSUPPORTED, "FP64 tensors are not supported here");
    v.data = static_cast<char *>(t->data);
    v.type = elem_type(t->dtype);
    v.n = d[0];
    v.c = d[1];
    v.px = 1;
    v.ldp = v.c;
    bool even = true;
    for (int i = t->rank - 1; i >= 2; --i) {  // axes of one image, innermost first
        if (d[i] > 1) {
            if (v.px == 1) v.ldp = s[i];
            else even = even && s[i] >= 0 && static_cast<wide>(v.ldp) * v.px == s[i];
        }
        v.px *= d[i];
    }
    if (v.n == 0 || v.px == 0) return GC_OK;
    if (v.ldp < v.c || (v.c > 1 && s[1] != 1) || !even)
        return gc_error(GC_UNSUPPORTED, "tensor is not channels last with evenly spaced pixels");
    const wide image = static_cast<wide>(v.px - 1) * v.ldp + v.c;
    wide total = image;
    v.ldn = 0;
    if (v.n > 1) {
        if (s[0] < image) return gc_error(GC_UNSUPPORTED, "tensor's images overlap or interleave");
        v.ldn = s[0];
        total += static_cast<wide>(v.n - 1) * v.ldn;
    }
    total *= elem_size(v.type);
    if (total > static_cast<wide>(t->bytes)) return gc_error(GC_INVALID, "tensor buffer is too small");
    v.span = static_cast<uint64_t>(total);
    return GC_OK;
}

// A nullable vector of one parameter per channel.
int check_channel_vector(const gc_tensor *t, const gc_tensor *x) {
    if (t == nullptr) return GC_OK;
    int64_t count = 0;
    int st = check_fields(t, 1, 1, count);
    if (st != GC_OK) return st;
    if (count != x->dims[1]) return gc_error(GC_INVALID, "channel parameters must have C elements");
    if (t->dtype != GC_F32 && t->dtype != x->dtype)
        return gc_error(GC_INVALID, "channel parameters must be F32 or of the data's type");
    if (t->device_index != x->device_index) return gc_error(GC_INVALID, "tensor device indices differ");
    return GC_OK;
}
int check_channel_layout(const gc_tensor *t) {
    if (t != nullptr && t->dims[0] > 1 && t->strides[0] != 1)
        return gc_error(GC_UNSUPPORTED, "channel parameters must be dense");
    return GC_OK;
}
int check_stats(const gc_tensor *t, const gc_tensor *x, int64_t groups) {
    int64_t count = 0;
    int st = check_fields(t, 3, 3, count);
    if (st != GC_OK) return st;
    if (t->dtype != GC_F32 || t->dims[0] != x->dims[0] || t->dims[1] != groups || t->dims[2] != 2)
        return gc_error(GC_INVALID, "stats must be an F32 tensor of dims (N, groups, 2)");
    if (t->device_index != x->device_index) return gc_error(GC_INVALID, "tensor device indices differ");
    if (reinterpret_cast<uintptr_t>(t->data) % 8 != 0) return gc_error(GC_INVALID, "stats must be 8-byte aligned");
    return GC_OK;
}
bool dense_stats(const gc_tensor *t) {
    return t->strides[2] == 1 && (t->dims[1] == 1 || t->strides[1] == 2) &&
           (t->dims[0] <= 1 || t->strides[0] == 2 * t->dims[1]);
}

int check_dropout(const gc_b200_dropout_args *d, DropParams &out) {
    out = DropParams{};
    if (d == nullptr) return GC_OK;
    if (!(d->p >= 0.0 && d->p <= 1.0)) return gc_error(GC_INVALID, "dropout probability must be in 0..1");
    if (d->scope != GC_B200_DROP_ELEMENT && d->scope != GC_B200_DROP_CHANNEL)
        return gc_error(GC_INVALID, "unknown dropout scope");
    for (const void *p : {static_cast<const void *>(d->seed_ptr), static_cast<const void *>(d->offset_ptr),
                          static_cast<const void *>(d->used)})
        if (reinterpret_cast<uintptr_t>(p) % 8 != 0) return gc_error(GC_INVALID, "dropout words are not 8-byte aligned");
    if (d->used != nullptr)
        for (const uint64_t *p : {d->seed_ptr, d->offset_ptr})
            if (p != nullptr && ranges_meet(d->used, 16, p, 8))
                return gc_error(GC_INVALID, "the words in use must not overwrite the given ones");
    out.threshold = static_cast<uint32_t>(std::nearbyint(65536.0 * d->p));
    out.limit = out.threshold != 0 ? (out.threshold << 16) - 1u : 0u;  // 65536 wraps to all ones: nothing is above
    out.scale = out.threshold < 65536 ? static_cast<float>(65536.0 / (65536.0 - out.threshold)) : 0.0f;
    out.channel = d->scope == GC_B200_DROP_CHANNEL;
    out.seed = d->seed;
    out.offset = d->offset;
    out.seed_ptr = d->seed_ptr;
    out.offset_ptr = d->offset_ptr;
    out.used = d->used;
    return GC_OK;
}

Range used_words(const DropParams &d) { return {d.used, d.used != nullptr ? 16u : 0u}; }
Range given_word(const uint64_t *p) { return {p, p != nullptr ? 8u : 0u}; }

// ---- group norm: plan ---------------------------------------------------------------------
int vector_of(const View &v) { return v.type == gcb::kElemF32 ? 4 : 8; }

// Every pixel of every given view starts on a 16-byte boundary.
bool vector_access(std::initializer_list<const View *> views) {
    for (const View *v : views) {
        const int e = vector_of(*v);
        if (v->c % e || v->ldp % e || v->ldn % e || !gcb::aligned16(v->data)) return false;
    }
    return true;
}

// The split path's work split: blocks of up to 256 vector columns and chunks
// of pixels such that one wave of blocks streams everything, but at least eight
// pixels for each thread.  Two waves where a thread has 64 vectors even then,
// because the SMs are not served alike (N64 C128 112x112 FP32 forward: 211 us
// in one wave, 200 in two; N8 C128 256x256 bf16: 71 and 77).  Launching sets of
// images small enough for the second pass to find them in the L2 cache was
// slower: a set's three launches cost about 10 us beside its data (the latter
// shape: 78 us in one set, 108 in four).  In the gradient a thread takes at most
// kNormRun runs of kNormRun vectors, for the sake of its sums.
void plan_split(NormParams &P, int v, bool backward, int sms) {
    P.vcols = P.c / v;
    P.cblocks = static_cast<int>(ceil_div(P.vcols, gcb::kNormThreads));
    P.vb = static_cast<int>(ceil_div(P.vcols, P.cblocks));
    P.lanes = gcb::kNormThreads / P.vb;
    const long long wave = static_cast<long long>(gcb::split_blocks(v, backward)) * sms;
    // vectors of a thread if one wave of blocks takes everything
    const long long each = ceil_div(P.n * P.px, wave * P.lanes) * P.cblocks;
    const long long wanted = std::max<long long>(1, (each >= 128 ? 2 : 1) * wave / (P.n * P.cblocks));
    P.chunk_rows = std::min(P.px, std::max<long long>(ceil_div(P.px, wanted), 8LL * P.lanes));
    const long long most = static_cast<long long>(gcb::kNormRun) * gcb::kNormRun * P.lanes;
    if (backward && P.chunk_rows > most) P.chunk_rows = ceil_div(P.px, ceil_div(P.px, most));
    P.chunks = static_cast<int>(ceil_div(P.px, P.chunk_rows));
    P.items = P.n * P.chunks * P.cblocks;
}

// Shared memory of the split path's kernels: the ring, and in its place after
// the data what the sums need.
size_t split_smem(const NormParams &P, int v, bool sums, bool backward) {
    size_t after = 0;
    if (sums) after += gcb::channel_sums_space(gcb::kNormThreads, P.vb, P.lanes, P.vb * v) * sizeof(float2);
    if (sums && !backward) after += ceil_div(P.vb * v, 2) * 2 * sizeof(float);
    return std::max(gcb::ring_space(v), after);
}

struct NormPlan {
    bool vec = false;
    int type = 0;
    bool resident = false, small = false;
    int threads = gcb::kNormThreads;
    size_t smem = 0;
    int width() const { return !vec ? 1 : type == gcb::kElemF32 ? 4 : 8; }  // elements of a vector
    int slot() const { return vec ? 16 : elem_size(type); }                 // its bytes
};

struct NormSpace {  // the workspace's parts, in this order
    uint64_t stats = 0, part = 0, chan = 0, gsum = 0;
    uint64_t total() const { return stats + part + chan + gsum; }
};

// Bytes of the workspace for a plan that is already in P.
NormSpace space_of(const NormParams &P, const NormPlan &plan, bool backward) {
    NormSpace s;
    const uint64_t n = P.n;
    if (plan.small) {
        if (backward) s.part = up16(static_cast<uint64_t>(P.nblocks) * P.c * sizeof(float2));
        return s;
    }
    if (plan.resident) {
        if (backward) s.part = up16(static_cast<uint64_t>(P.stride * P.cluster) * P.c * sizeof(float2));
        return s;
    }
    s.part = up16(n * P.chunks * P.c * sizeof(float2));
    if (backward) {
        s.chan = up16(n * P.c * sizeof(float2));
        s.gsum = up16(n * P.groups * sizeof(float2));
    } else {
        s.stats = up16(n * P.groups * sizeof(float2));
    }
    return s;
}

// Checks shared by the workspace queries and the calls: data tensors that
// have the same dims and type, then their layout.  views[0] is x's.
int check_data(std::initializer_list<const gc_tensor *> tensors, int64_t groups, View *views, NormParams &P,
               NormPlan &plan) {
    const gc_tensor *first = *tensors.begin();
    int64_t count = 0;
    for (const gc_tensor *t : tensors) {
        const int st = check_fields(t, 2, 4, count);
        if (st != GC_OK) return st;
        if (!same_dims(t, first)) return gc_error(GC_INVALID, "tensor dimensions differ");
        if (t->dtype != first->dtype) return gc_error(GC_INVALID, "tensor dtypes differ");
        if (t->device_index != first->device_index) return gc_error(GC_INVALID, "tensor device indices differ");
    }
    if (first->dims[1] < 1 || first->dims[1] > INT32_MAX) return gc_error(GC_INVALID, "channel count out of range");
    if (groups < 1 || first->dims[1] % groups != 0) return gc_error(GC_INVALID, "channels must be divisible by groups");
    P = NormParams{};
    int i = 0;
    plan.vec = true;
    for (const gc_tensor *t : tensors) {
        const int st = view_of(t, views[i]);
        if (st != GC_OK) return st;
        plan.vec = plan.vec && vector_access({&views[i]});
        ++i;
    }
    P.n = views[0].n;
    P.px = views[0].px;
    P.c = static_cast<int>(views[0].c);
    P.groups = static_cast<int>(groups);
    P.cpg = P.c / P.groups;
    plan.type = views[0].type;
    return GC_OK;
}

bool empty(const NormParams &P) { return P.n == 0 || P.px == 0; }

// ---- resident path: plan --------------------------------------------------------------------
// What a plan depends on.
struct ResidentKey {
    int dev, type, backward, vec;
    long long n, px;
    int c, groups;
    bool operator<(const ResidentKey &o) const {
        return std::tie(dev, type, backward, vec, n, px, c, groups) <
               std::tie(o.dev, o.type, o.backward, o.vec, o.n, o.px, o.c, o.groups);
    }
};
struct ResidentPlan {
    bool ok = false, small = false;
    double cost = 0.0;  // of the resident or split path
    int cb = 0, threads = 0, cluster = 0;
    size_t smem = 0;
};

// Fills the resident fields of P for a choice; false when it does not apply.
bool set_resident(NormParams &P, int v, int slot, int cb, int cluster, int threads, bool backward, bool bits,
                  size_t limit, size_t &smem) {
    P.cb = cb;
    P.vr = cb / v;
    if (P.vr > threads) return false;
    P.lanes = threads / P.vr;
    P.sub = v % P.cpg == 0 ? v / P.cpg : P.cpg % v == 0 ? 1 : v;
    P.gcols = static_cast<int>(static_cast<long long>(P.cpg) * P.sub / v);
    P.gb = cb / P.cpg;
    P.bundles = P.c / cb;
    P.cluster = cluster;
    const long long rows = ceil_div(P.px, cluster);
    if (rows > (1 << 20)) return false;
    P.rows = static_cast<int>(rows);
    P.iters = static_cast<int>(ceil_div(rows, P.lanes));
    smem = gcb::tile_bytes((backward ? 2 : 1) * P.iters, threads, slot) + gcb::resident_extra(P, threads, backward) +
           (bits ? static_cast<size_t>(P.iters) * threads : 0);
    return smem <= limit;
}

// Clusters per bundle: as many as the device holds at once, evenly loaded.
long long resident_stride(const NormParams &P, int threads, size_t smem, const gcb::DeviceFacts &f, int &occ) {
    // 128 registers a thread allow 512 threads per SM
    occ = static_cast<int>(std::min<size_t>(gcb::kResidentThreads / threads, f.smem_per_sm / (smem + 1024)));
    occ = std::max(1, occ);
    const long long most = std::max(1LL, static_cast<long long>(occ) * f.sms / (static_cast<long long>(P.bundles) * P.cluster));
    return ceil_div(P.n, ceil_div(P.n, most));
}

// Estimated cost of a resident choice that is set in P: its phases (load; for
// each image of a cluster the first pass, the sums, the second pass).  The
// constants are fitted, to 5765 choices of 112 shapes timed on a B200, so that
// the cheapest choice is the fastest one; they follow the times in
// microseconds only roughly.  Clusters are counted as if any SMs could make one
// up, though one is placed within a GPC.  On those shapes the choice is 5 % slower than the
// best on average, and at most 1.25 times where a call takes more than 6 us
// (once 1.39, with 255 channels of FP32).
double resident_cost(const NormParams &P, int v, int slot, int threads, size_t smem, bool backward,
                     const gcb::DeviceFacts &f) {
    int occ = 1;
    const long long stride = resident_stride(P, threads, smem, f, occ);
    const double rounds = static_cast<double>(ceil_div(P.n, stride));
    const double per_sm = std::ceil(static_cast<double>(stride) * P.bundles * P.cluster / f.sms);  // CTAs of the fullest SM
    const double run = P.cb * static_cast<double>(slot) / v;  // bytes of a pixel that lie together
    const double kb = per_sm * P.iters * P.lanes * P.vr * static_cast<double>(slot) * (backward ? 2 : 1) / 1024.0 /
                      (run >= 64 ? 1.0 : run >= 32 ? 0.51 : 0.26);
    double sums = 1.13 + (P.cluster > 1 ? 2.61 : 0.0) + (P.cluster > 8 ? 1.73 : 0.0) + 1.48 * per_sm * threads / 512;
    if (backward) sums += 0.35 + (32 % P.vr != 0 ? 0.14 : 0.0);
    else sums += 0.05 * P.vr * P.lanes * P.sub / 512;
    // per vector of a thread: latency with few warps, issue slots with many
    const double crowd = P.iters * std::max(1.0, per_sm * threads / 32 / 11.1);
    const double first = std::max(kb / 103.0, crowd * (v == 1 ? 0.047 : v == 4 ? 0.027 : 0.0125) * (backward ? 10.7 : 1.0));
    const double second = std::max(kb / (backward ? 237.0 : 38.0),
                                   crowd * (v == 1 ? 0.147 : v == 4 ? 0.112 : 0.225) * (backward ? 1.33 : 1.0));
    return 0.4 + kb / 190.0 + rounds * (first + sums + second) + (backward ? 1.0 : 0.0);
}
// The same for the split path.  Images that are more than a wave of blocks
// cost a block's fixed time for each further wave, in both data passes.
double split_cost(const NormParams &P, int v, int slot, bool backward, const gcb::DeviceFacts &f) {
    const double blocks = static_cast<double>(P.n) * ceil_div(P.c / v, gcb::kNormThreads);
    const double extra = 5.0 * std::max(0.0, blocks / (gcb::split_blocks(v, backward) * f.sms) - 1.0);
    const double elements = static_cast<double>(P.n) * P.px * P.c, mb = elements * slot / v * 1e-6;
    if (v == 1) return extra + (backward ? 10.0 + elements * 4.76e-6 : 15.3 + elements * (slot == 4 ? 6.4e-6 : 2.1e-6));
    return extra + (backward ? 10.0 + 2 * mb / 6.0 + 3 * mb / 6.6 : 15.3 + mb / 5.5 + 2 * mb / 6.6);
}

// Plans that are kept; a program whose shapes never repeat starts anew there.
constexpr size_t kPlans = 4096;
std::mutex g_mutex;
std::map<ResidentKey, ResidentPlan> g_resident;

ResidentPlan choose_resident(const NormParams &base, int v, int slot, bool backward, bool bits,
                             const gcb::DeviceFacts &f) {
    ResidentPlan best;
    double best_cost = split_cost(base, v, slot, backward, f);
    const int unit = std::lcm(base.cpg, v);  // channels: whole groups and whole vectors
    const int units = base.c / unit;
    for (int m = 1; m <= units && static_cast<long long>(m) * unit / v <= gcb::kNormThreads; ++m) {
        if (units % m) continue;
        for (int cluster = 1; cluster <= 16; cluster *= 2)
            for (int threads = 64; threads <= gcb::kResidentThreads; threads *= 2) {
                NormParams P = base;
                size_t smem = 0;
                if (!set_resident(P, v, slot, m * unit, cluster, threads, backward, bits, f.smem_optin, smem)) continue;
                if (P.n * P.bundles * cluster > INT32_MAX) continue;
                const double cost = resident_cost(P, v, slot, threads, smem, backward, f);
                if (cost < best_cost) {
                    best_cost = cost;
                    best.ok = true;
                    best.cb = m * unit;
                    best.threads = threads;
                    best.cluster = cluster;
                    best.smem = smem;
                }
            }
    }
    best.cost = best_cost;
    return best;
}

// The small path: threads per group so that each holds about four elements, and
// at most kNormRun images in turn.  False where a group is too large for a warp.
bool set_small(NormParams &P, int sms) {
    if (static_cast<wide>(P.px) * P.cpg > 32 * 16) return false;
    const int elements = static_cast<int>(P.px) * P.cpg;
    P.team = 1;
    while (P.team < 32 && 4 * P.team < elements) P.team *= 2;
    P.gb = std::min(P.groups, gcb::kNormThreads / P.team);
    P.gblocks = static_cast<int>(ceil_div(P.groups, P.gb));
    const long long images = gcb::kNormThreads / P.team / P.gb;
    P.nblocks = std::min(ceil_div(P.n, images), std::max<long long>(1, ceil_div(8LL * sms, P.gblocks)));
    P.nblocks = std::max(P.nblocks, ceil_div(P.n, images * gcb::kNormRun));
    return P.nblocks * P.gblocks <= INT32_MAX;
}
// Its time in the same units: element accesses reach about 2 TB/s.
double small_cost(const NormParams &P, int v, int slot, bool backward) {
    const double mb = static_cast<double>(P.n) * P.px * P.c * slot / v * 1e-6;
    return (backward ? 5.0 : 3.0) + (backward ? 3.0 : 2.0) * mb / 2.0;
}

int plan_norm(NormParams &P, NormPlan &plan, bool backward) {
    int dev = -1;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return gc_error(GC_DEVICE_ERROR, cudaGetErrorString(e));
    gcb::DeviceFacts facts;
    const int st = gcb::device_facts(dev, facts);
    if (st != GC_OK) return st;
    const int v = plan.width();
    {
        // room for the decision bytes is planned for whether they are needed
        // or not, so that a tensor's workspace does not depend on the dropout
        const ResidentKey key{dev, plan.type, backward, plan.vec, P.n, P.px, P.c, P.groups};
        ResidentPlan r;
        bool known = false;
        {
            std::lock_guard<std::mutex> lock(g_mutex);
            const auto it = g_resident.find(key);
            if (it != g_resident.end()) {
                r = it->second;
                known = true;
            }
        }
        if (!known) {
            r = choose_resident(P, v, plan.slot(), backward, backward, facts);
            NormParams Q = P;
            r.small = set_small(Q, facts.sms) && small_cost(P, v, plan.slot(), backward) < r.cost;
            std::lock_guard<std::mutex> lock(g_mutex);
            if (g_resident.size() >= kPlans) g_resident.clear();
            g_resident[key] = r;
        }
        if (r.small) {
            plan.small = set_small(P, facts.sms);
            return GC_OK;
        }
        if (r.ok) {
            set_resident(P, v, plan.slot(), r.cb, r.cluster, r.threads, backward, backward, facts.smem_optin, plan.smem);
            plan.resident = true;
            plan.threads = r.threads;
            int occ = 1;
            P.stride = resident_stride(P, r.threads, plan.smem, facts, occ);
            return GC_OK;
        }
    }
    plan_split(P, v, backward, facts.sms);
    if (P.items > INT32_MAX) return gc_error(GC_UNSUPPORTED, "more images than a grid has blocks");
    return GC_OK;
}

void set_param(const gc_tensor *t, const void *&p, int &type) {
    p = t != nullptr ? t->data : nullptr;
    type = t != nullptr ? elem_type(t->dtype) : 0;
}

// ---- kernel tables --------------------------------------------------------------------------
// The vector kernels without dropout are compiled for each activation, those
// with dropout for SiLU: N8 C128 256x256 bf16 92 us and gradient 150 instead of
// 96 and 167 with the activation chosen at run time, N32 C256 28x28 12.7 and 25
// instead of 13.4 and 29 (FP32 19 and 30 instead of 21 and 35).  The others
// choose it at run time (ReLU, gradient of the first: 154 us).
enum NormKernel { kMoments, kApply, kGradSums, kGradApply };

template <class T, int V, int ACT, bool DROP>
const void *norm_instance(NormKernel k) {
    switch (k) {
    case kApply: return reinterpret_cast<const void *>(&gcb::norm_apply_kernel<T, V, ACT, DROP>);
    case kGradSums: return reinterpret_cast<const void *>(&gcb::norm_grad_sums_kernel<T, V, ACT, DROP>);
    case kGradApply: return reinterpret_cast<const void *>(&gcb::norm_grad_apply_kernel<T, V, ACT, DROP>);
    default: return reinterpret_cast<const void *>(&gcb::norm_moments_kernel<T, V>);
    }
}
template <class T>
const void *norm_typed(NormKernel k, bool vec, int act, bool drop) {
    constexpr int V = gcb::kVec<T>;
    if (!vec) return drop ? norm_instance<T, 1, -1, true>(k) : norm_instance<T, 1, -1, false>(k);
    if (drop && act == gcb::kActSilu) return norm_instance<T, V, gcb::kActSilu, true>(k);
    if (drop) return norm_instance<T, V, -1, true>(k);
    if (act == gcb::kActRelu) return norm_instance<T, V, gcb::kActRelu, false>(k);
    if (act == gcb::kActRelu6) return norm_instance<T, V, gcb::kActRelu6, false>(k);
    if (act == gcb::kActSilu) return norm_instance<T, V, gcb::kActSilu, false>(k);
    return norm_instance<T, V, gcb::kActNone, false>(k);
}
const void *norm_kernel(NormKernel k, const NormPlan &plan, const NormParams &P) {
    const bool drop = P.drop.threshold != 0;
    if (plan.type == gcb::kElemF16) return norm_typed<__half>(k, plan.vec, P.act, drop);
    if (plan.type == gcb::kElemBF16) return norm_typed<__nv_bfloat16>(k, plan.vec, P.act, drop);
    return norm_typed<float>(k, plan.vec, P.act, drop);
}

template <class T, int V, int ACT, bool DROP>
const void *resident_instance(bool backward) {
    return backward ? reinterpret_cast<const void *>(&gcb::norm_resident_grad_kernel<T, V, ACT, DROP>)
                    : reinterpret_cast<const void *>(&gcb::norm_resident_kernel<T, V, ACT, DROP>);
}
template <class T>
const void *resident_typed(bool backward, bool vec, int act, bool drop) {
    constexpr int V = gcb::kVec<T>;
    if (!vec) return drop ? resident_instance<T, 1, -1, true>(backward) : resident_instance<T, 1, -1, false>(backward);
    if (drop && act == gcb::kActSilu) return resident_instance<T, V, gcb::kActSilu, true>(backward);
    if (drop) return resident_instance<T, V, -1, true>(backward);
    if (act == gcb::kActRelu) return resident_instance<T, V, gcb::kActRelu, false>(backward);
    if (act == gcb::kActRelu6) return resident_instance<T, V, gcb::kActRelu6, false>(backward);
    if (act == gcb::kActSilu) return resident_instance<T, V, gcb::kActSilu, false>(backward);
    return resident_instance<T, V, gcb::kActNone, false>(backward);
}
const void *resident_kernel(const NormPlan &plan, bool backward, int act, bool drop) {
    if (plan.type == gcb::kElemF16) return resident_typed<__half>(backward, plan.vec, act, drop);
    if (plan.type == gcb::kElemBF16) return resident_typed<__nv_bfloat16>(backward, plan.vec, act, drop);
    return resident_typed<float>(backward, plan.vec, act, drop);
}

template <class T>
const void *small_typed(bool backward, bool four) {
    return backward ? (four ? reinterpret_cast<const void *>(&gcb::norm_small_kernel<T, 4, true>)
                            : reinterpret_cast<const void *>(&gcb::norm_small_kernel<T, 16, true>))
                    : (four ? reinterpret_cast<const void *>(&gcb::norm_small_kernel<T, 4, false>)
                            : reinterpret_cast<const void *>(&gcb::norm_small_kernel<T, 16, false>));
}
const void *small_kernel(const NormParams &P, const NormPlan &plan, bool backward) {
    const bool four = P.px * P.cpg <= 4LL * P.team;
    if (plan.type == gcb::kElemF16) return small_typed<__half>(backward, four);
    if (plan.type == gcb::kElemBF16) return small_typed<__nv_bfloat16>(backward, four);
    return small_typed<float>(backward, four);
}

// Opts a kernel into the shared memory and the cluster sizes it may be
// launched with, once per device.
int prepare_kernel(const void *fn, int dev, int smem_optin) {
    static std::map<std::pair<int, const void *>, bool> done;
    std::lock_guard<std::mutex> lock(g_mutex);
    bool &flag = done[{dev, fn}];
    if (flag) return GC_OK;
    cudaError_t e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, smem_optin);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(fn, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e != cudaSuccess) {
        cudaGetLastError();
        return gc_error(GC_DEVICE_ERROR, cudaGetErrorString(e));
    }
    flag = true;
    return GC_OK;
}

int launch_resident(NormParams &P, const NormPlan &plan, bool backward, int dev, cudaStream_t s, cudaError_t &e) {
    gcb::DeviceFacts facts;
    int st = gcb::device_facts(dev, facts);
    if (st != GC_OK) return st;
    const void *fn = resident_kernel(plan, backward, P.act, P.drop.threshold != 0);
    if ((st = prepare_kernel(fn, dev, facts.smem_optin)) != GC_OK) return st;
    void *args[] = {&P};
    const unsigned grid = static_cast<unsigned>(static_cast<long long>(P.stride) * P.bundles * P.cluster);
    e = gcb::launch_pdl(fn, dim3(grid), dim3(plan.threads), args, plan.smem, s, P.cluster);
    return GC_OK;
}

// Images that a cluster (resident path) or a team of threads (small path) takes
// in turn, at most; 1 on the split path.
long long rounds_of(const NormParams &P, const NormPlan &plan) {
    if (plan.small) return ceil_div(P.n, P.nblocks * (gcb::kNormThreads / P.team / P.gb));
    return plan.resident ? ceil_div(P.n, P.stride) : 1;
}

unsigned grid_of(long long items) { return static_cast<unsigned>(std::min<long long>(items, INT32_MAX)); }

cudaError_t launch(const void *fn, long long blocks, NormParams &P, cudaStream_t s, size_t smem = 0) {
    void *args[] = {&P};
    return gcb::launch_pdl(fn, dim3(grid_of(blocks)), dim3(gcb::kNormThreads), args, smem, s);
}

// A kernel of the split path that streams data.
int launch_split(NormKernel k, NormParams &P, const NormPlan &plan, int dev, cudaStream_t s, cudaError_t &e) {
    gcb::DeviceFacts facts;
    int st = gcb::device_facts(dev, facts);
    if (st != GC_OK) return st;
    const void *fn = norm_kernel(k, plan, P);
    if ((st = prepare_kernel(fn, dev, facts.smem_optin)) != GC_OK) return st;
    e = launch(fn, P.items, P, s, split_smem(P, plan.width(), k == kMoments || k == kGradSums, k == kGradSums));
    return GC_OK;
}

// The kernels that join partial results per group: a warp per group, or a
// block where a group has more than 256 entries.
cudaError_t launch_finalize(bool backward, NormParams &P, cudaStream_t s) {
    const bool block = static_cast<long long>(P.chunks) * P.cpg > 256;
    const void *fn = backward ? (block ? reinterpret_cast<const void *>(&gcb::norm_grad_finalize_kernel<gcb::kNormThreads>)
                                       : reinterpret_cast<const void *>(&gcb::norm_grad_finalize_kernel<32>))
                              : (block ? reinterpret_cast<const void *>(&gcb::norm_finalize_kernel<gcb::kNormThreads>)
                                       : reinterpret_cast<const void *>(&gcb::norm_finalize_kernel<32>));
    return launch(fn, block ? P.n * P.groups : ceil_div(P.n * P.groups, gcb::kNormThreads / 32), P, s);
}

bool known_activation(int a) {
    return a == GC_B200_ACT_NONE || a == GC_B200_ACT_RELU || a == GC_B200_ACT_RELU6 || a == GC_B200_ACT_SILU;
}

// ---- dropout ----------------------------------------------------------------------------------
// Whether the axes, taken in some order, fill memory without gaps or overlap.
bool dense_any_order(const gc_tensor *t) {
    bool used[4] = {false, false, false, false};
    wide expect = 1;
    for (int step = 0; step < t->rank; ++step) {
        int pick = -1;
        for (int i = 0; i < t->rank; ++i)
            if (!used[i] && (t->dims[i] == 1 || t->strides[i] == expect) && (pick < 0 || t->dims[i] == 1)) pick = i;
        if (pick < 0) return false;
        used[pick] = true;
        expect *= t->dims[pick];
    }
    return true;
}

// (N, C, ..) in plain order, the innermost axis last?
bool plain_order(const gc_tensor *t) {
    wide expect = 1;
    for (int i = t->rank - 1; i >= 0; --i) {
        if (t->dims[i] > 1 && t->strides[i] != expect) return false;
        expect *= t->dims[i];
    }
    return true;
}
bool channels_last_order(const gc_tensor *t) {
    if (t->dims[1] > 1 && t->strides[1] != 1) return false;
    wide expect = t->dims[1];
    for (int i = t->rank - 1; i >= 2; --i) {
        if (t->dims[i] > 1 && t->strides[i] != expect) return false;
        expect *= t->dims[i];
    }
    return t->dims[0] <= 1 || t->strides[0] == expect;
}

enum DropoutKernel { kElements, kChannels, kPlanes, kMapped };
template <class T, int V>
const void *dropout_instance(DropoutKernel k) {
    return k == kElements   ? reinterpret_cast<const void *>(&gcb::dropout_kernel<T, V, false>)
           : k == kMapped   ? reinterpret_cast<const void *>(&gcb::dropout_kernel<T, V, true>)
           : k == kChannels ? reinterpret_cast<const void *>(&gcb::channel_dropout_kernel<T, V>)
                            : reinterpret_cast<const void *>(&gcb::plane_dropout_kernel<T, V>);
}
template <class T>
const void *dropout_typed(DropoutKernel k, bool vec) {
    return vec ? dropout_instance<T, gcb::kVec<T>>(k) : dropout_instance<T, 1>(k);
}

}  // namespace

extern "C" {

int gc_b200_group_norm_workspace(const gc_tensor *x, const gc_tensor *y, int64_t groups, uint64_t *bytes) try {
    if (bytes == nullptr) return gc_error(GC_INVALID, "null size pointer");
    View v[2];
    NormParams P;
    NormPlan plan;
    int st = check_data({x, y}, groups, v, P, plan);
    if (st != GC_OK) return st;
    *bytes = 0;
    if (empty(P)) return gc_error(GC_OK, "");
    st = plan_norm(P, plan, false);
    if (st != GC_OK) return st;
    *bytes = space_of(P, plan, false).total();
    return gc_error(GC_OK, "");
} catch (...) {
    return internal_error();
}

int gc_b200_group_norm(const gc_tensor *x, const gc_tensor *gamma, const gc_tensor *beta, gc_tensor *y,
                       gc_tensor *stats, int64_t groups, double eps, int activation,
                       const gc_b200_dropout_args *dropout, void *workspace, uint64_t workspace_bytes, void *stream) try {
    View v[2];
    NormParams P;
    NormPlan plan;
    int st = check_data({x, y}, groups, v, P, plan);
    if (st != GC_OK) return st;
    if (!(eps >= 0.0) || !std::isfinite(eps)) return gc_error(GC_INVALID, "eps must be finite and not negative");
    for (const gc_tensor *t : {gamma, beta})
        if ((st = check_channel_vector(t, x)) != GC_OK) return st;
    if (stats != nullptr && (st = check_stats(stats, x, groups)) != GC_OK) return st;
    DropParams drop;
    if ((st = check_dropout(dropout, drop)) != GC_OK) return st;
    if (outputs_meet({{y->data, v[1].span}, range_of(stats), used_words(drop), {workspace, workspace_bytes}},
                     {{x->data, v[0].span}, range_of(gamma), range_of(beta), given_word(drop.seed_ptr),
                      given_word(drop.offset_ptr)}))
        return gc_error(GC_INVALID, "outputs and workspace must not overlap inputs or one another");
    if (!known_activation(activation)) return gc_error(GC_UNSUPPORTED, "unknown activation");
    for (const gc_tensor *t : {gamma, beta})
        if ((st = check_channel_layout(t)) != GC_OK) return st;
    if (stats != nullptr && !dense_stats(stats)) return gc_error(GC_UNSUPPORTED, "stats must be dense");
    if (empty(P)) return gc_error(GC_OK, "");
    int dev = -1;
    st = check_call({x, y, gamma, beta, stats}, {drop.seed_ptr, drop.offset_ptr, drop.used}, x->device_index, stream,
                    dev);
    if (st != GC_OK) return st;
    if ((st = plan_norm(P, plan, false)) != GC_OK) return st;
    const NormSpace space = space_of(P, plan, false);
    if ((st = check_workspace(workspace, workspace_bytes, space.total())) != GC_OK) return st;
    if (space.total() != 0 && (st = gcb::check_device_memory(workspace, x->device_index, dev)) != GC_OK) return st;
    P.x = v[0].data;
    P.x_ldn = v[0].ldn;
    P.x_ldp = v[0].ldp;
    P.y = v[1].data;
    P.y_ldn = v[1].ldn;
    P.y_ldp = v[1].ldp;
    set_param(gamma, P.gamma, P.gamma_type);
    set_param(beta, P.beta, P.beta_type);
    P.eps = static_cast<float>(eps);
    P.act = activation;
    P.drop = drop;
    char *w = static_cast<char *>(workspace);
    P.stats = reinterpret_cast<float2 *>(stats != nullptr ? static_cast<char *>(stats->data) : w);
    P.part = reinterpret_cast<float2 *>(w + space.stats);
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    cudaError_t e = cudaSuccess;
    if (plan.small) {
        if (stats == nullptr) P.stats = nullptr;
        e = launch(small_kernel(P, plan, false), P.nblocks * P.gblocks, P, s);
        return launched(e, PlanRecord::kNorm, "small", P.nblocks * P.gblocks, gcb::kNormThreads, 0, 1,
                         P.gb * P.cpg, P.px, 0, 1, rounds_of(P, plan));
    }
    if (plan.resident) {
        if (stats == nullptr) P.stats = nullptr;
        if ((st = launch_resident(P, plan, false, dev, s, e)) != GC_OK) return st;
        return launched(e, PlanRecord::kNorm, "resident", static_cast<long long>(P.stride) * P.bundles * P.cluster,
                         plan.threads, plan.smem, P.cluster, P.cb, P.rows, plan.vec ? 1 : 0, 1, rounds_of(P, plan));
    }
    if ((st = launch_split(kMoments, P, plan, dev, s, e)) != GC_OK) return st;
    if (e == cudaSuccess) e = launch_finalize(false, P, s);
    if (e == cudaSuccess && (st = launch_split(kApply, P, plan, dev, s, e)) != GC_OK) return st;
    return launched(e, PlanRecord::kNorm, "split", P.items, gcb::kNormThreads, 0, 1, P.vb, P.chunk_rows,
                     plan.vec ? 1 : 0, 3, 1);
} catch (...) {
    return internal_error();
}

int gc_b200_group_norm_backward_workspace(const gc_tensor *dy, const gc_tensor *x, const gc_tensor *dx,
                                          int64_t groups, uint64_t *bytes) try {
    if (bytes == nullptr) return gc_error(GC_INVALID, "null size pointer");
    View v[3];
    NormParams P;
    NormPlan plan;
    int st = check_data({x, dy, dx}, groups, v, P, plan);
    if (st != GC_OK) return st;
    *bytes = 0;
    if (empty(P)) return gc_error(GC_OK, "");
    st = plan_norm(P, plan, true);
    if (st != GC_OK) return st;
    *bytes = space_of(P, plan, true).total();
    return gc_error(GC_OK, "");
} catch (...) {
    return internal_error();
}

int gc_b200_group_norm_backward(const gc_tensor *dy, const gc_tensor *x, const gc_tensor *gamma,
                                const gc_tensor *beta, const gc_tensor *stats, gc_tensor *dx, gc_tensor *dgamma,
                                gc_tensor *dbeta, int64_t groups, int activation,
                                const gc_b200_dropout_args *dropout, void *workspace, uint64_t workspace_bytes,
                                void *stream) try {
    View v[3];
    NormParams P;
    NormPlan plan;
    int st = check_data({x, dy, dx}, groups, v, P, plan);
    if (st != GC_OK) return st;
    for (const gc_tensor *t : {gamma, beta, static_cast<const gc_tensor *>(dgamma),
                               static_cast<const gc_tensor *>(dbeta)})
        if ((st = check_channel_vector(t, x)) != GC_OK) return st;
    if ((st = check_stats(stats, x, groups)) != GC_OK) return st;
    DropParams drop;
    if ((st = check_dropout(dropout, drop)) != GC_OK) return st;
    if (outputs_meet({{dx->data, v[2].span}, range_of(dgamma), range_of(dbeta), used_words(drop),
                      {workspace, workspace_bytes}},
                     {{x->data, v[0].span}, {dy->data, v[1].span}, range_of(gamma), range_of(beta), range_of(stats),
                      given_word(drop.seed_ptr), given_word(drop.offset_ptr)}))
        return gc_error(GC_INVALID, "outputs and workspace must not overlap inputs or one another");
    if (!known_activation(activation)) return gc_error(GC_UNSUPPORTED, "unknown activation");
    for (const gc_tensor *t : {gamma, beta, static_cast<const gc_tensor *>(dgamma),
                               static_cast<const gc_tensor *>(dbeta)})
        if ((st = check_channel_layout(t)) != GC_OK) return st;
    if (!dense_stats(stats)) return gc_error(GC_UNSUPPORTED, "stats must be dense");
    int dev = -1;
    st = check_call({x, dy, dx, gamma, beta, stats, dgamma, dbeta}, {drop.seed_ptr, drop.offset_ptr, drop.used},
                    x->device_index, stream, dev);
    if (st != GC_OK) return st;
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    if (empty(P)) {  // sums over nothing
        cudaError_t e = cudaSuccess;
        for (const gc_tensor *t : {dgamma, dbeta})
            if (t != nullptr && e == cudaSuccess) e = cudaMemsetAsync(t->data, 0, range_of(t).bytes, s);
        return launched(e);
    }
    if ((st = plan_norm(P, plan, true)) != GC_OK) return st;
    const NormSpace space = space_of(P, plan, true);
    if ((st = check_workspace(workspace, workspace_bytes, space.total())) != GC_OK) return st;
    if (space.total() != 0 && (st = gcb::check_device_memory(workspace, x->device_index, dev)) != GC_OK) return st;
    P.x = v[0].data;
    P.x_ldn = v[0].ldn;
    P.x_ldp = v[0].ldp;
    P.dy = v[1].data;
    P.dy_ldn = v[1].ldn;
    P.dy_ldp = v[1].ldp;
    P.y = v[2].data;
    P.y_ldn = v[2].ldn;
    P.y_ldp = v[2].ldp;
    set_param(gamma, P.gamma, P.gamma_type);
    set_param(beta, P.beta, P.beta_type);
    const void *q = nullptr;
    set_param(dgamma, q, P.dgamma_type);
    P.dgamma = const_cast<void *>(q);
    set_param(dbeta, q, P.dbeta_type);
    P.dbeta = const_cast<void *>(q);
    P.act = activation;
    P.drop = drop;
    P.stats = static_cast<float2 *>(stats->data);
    char *w = static_cast<char *>(workspace);
    P.part = reinterpret_cast<float2 *>(w);
    P.chan = reinterpret_cast<float2 *>(w + space.part);
    P.gsum = reinterpret_cast<float2 *>(w + space.part + space.chan);
    cudaError_t e = cudaSuccess;
    const bool params = P.dgamma != nullptr || P.dbeta != nullptr;
    const void *sums = reinterpret_cast<const void *>(&gcb::norm_grad_params_kernel);
    if (plan.small) {
        if (!params) P.part = nullptr;
        e = launch(small_kernel(P, plan, true), P.nblocks * P.gblocks, P, s);
        P.chan = P.part;
        P.sum_rows = P.nblocks;
        if (e == cudaSuccess && params) e = launch(sums, ceil_div(P.c, 32), P, s);
        return launched(e, PlanRecord::kNorm, "small_backward", P.nblocks * P.gblocks, gcb::kNormThreads, 0, 1,
                         P.gb * P.cpg, P.px, 0, params ? 2 : 1, rounds_of(P, plan));
    }
    if (plan.resident) {
        if (!params) P.part = nullptr;
        if ((st = launch_resident(P, plan, true, dev, s, e)) != GC_OK) return st;
        P.chan = P.part;
        P.sum_rows = static_cast<long long>(P.stride) * P.cluster;
        if (e == cudaSuccess && params) e = launch(sums, ceil_div(P.c, 32), P, s);
        return launched(e, PlanRecord::kNorm, "resident_backward",
                         static_cast<long long>(P.stride) * P.bundles * P.cluster, plan.threads, plan.smem, P.cluster,
                         P.cb, P.rows, plan.vec ? 1 : 0, params ? 2 : 1, rounds_of(P, plan));
    }
    P.sum_rows = P.n;
    if ((st = launch_split(kGradSums, P, plan, dev, s, e)) != GC_OK) return st;
    if (e == cudaSuccess) e = launch_finalize(true, P, s);
    if (e == cudaSuccess && (st = launch_split(kGradApply, P, plan, dev, s, e)) != GC_OK) return st;
    if (e == cudaSuccess && params) e = launch(sums, ceil_div(P.c, 32), P, s);
    return launched(e, PlanRecord::kNorm, "split_backward", P.items, gcb::kNormThreads, 0, 1, P.vb, P.chunk_rows,
                     plan.vec ? 1 : 0, params ? 4 : 3, 1);
} catch (...) {
    return internal_error();
}

int gc_b200_dropout(const gc_tensor *x, const gc_tensor *residual, gc_tensor *y,
                    const gc_b200_dropout_args *dropout, void *stream) try {
    int64_t count = 0;
    for (const gc_tensor *t : {x, static_cast<const gc_tensor *>(y), residual}) {
        if (t == nullptr && t == residual && x != nullptr && y != nullptr) continue;
        const int st = check_fields(t, 1, 4, count);
        if (st != GC_OK) return st;
        if (!same_dims(t, x)) return gc_error(GC_INVALID, "tensor dimensions differ");
        if (t->dtype != x->dtype) return gc_error(GC_INVALID, "tensor dtypes differ");
        if (t->device_index != x->device_index) return gc_error(GC_INVALID, "tensor device indices differ");
    }
    if (dropout == nullptr) return gc_error(GC_INVALID, "null dropout arguments");
    DropParams drop;
    int st = check_dropout(dropout, drop);
    if (st != GC_OK) return st;
    if (outputs_meet({range_of(y), used_words(drop)}, {range_of(x), range_of(residual), given_word(drop.seed_ptr),
                                                       given_word(drop.offset_ptr)}))
        return gc_error(GC_INVALID, "outputs must not overlap inputs");
    if (drop.channel && x->rank < 2) return gc_error(GC_INVALID, "channel dropout needs a channel axis");
    if (x->dtype == GC_F64) return gc_error(GC_UNSUPPORTED, "FP64 tensors are not supported here");
    if (count == 0) return gc_error(GC_OK, "");
    for (const gc_tensor *t : {static_cast<const gc_tensor *>(y), residual})
        if (t != nullptr)
            for (int i = 0; i < x->rank; ++i)
                if (x->dims[i] > 1 && t->strides[i] != x->strides[i])
                    return gc_error(GC_UNSUPPORTED, "tensors must have the same strides");
    if (!dense_any_order(x)) return gc_error(GC_UNSUPPORTED, "tensors must be dense");
    const bool plain = plain_order(x);
    if (drop.channel && !plain && !channels_last_order(x))
        return gc_error(GC_UNSUPPORTED, "channel dropout needs plain or channels-last order");
    int dev = -1;
    st = check_call({x, y, residual}, {drop.seed_ptr, drop.offset_ptr, drop.used}, x->device_index, stream, dev);
    if (st != GC_OK) return st;
    gcb::DeviceFacts facts;
    if ((st = gcb::device_facts(dev, facts)) != GC_OK) return st;
    DropoutParams P{};
    P.x = x->data;
    P.residual = residual != nullptr ? residual->data : nullptr;
    P.y = y->data;
    P.count = static_cast<uint64_t>(count);
    P.drop = drop;
    bool vec = gcb::aligned16(P.x) && gcb::aligned16(P.y) && gcb::aligned16(P.residual);
    const int type = elem_type(x->dtype), per_vector = type == gcb::kElemF32 ? 4 : 8;
    DropoutKernel kind = kElements;
    // Blocks: up to four waves of them, so that the SMs that are served faster
    // take more, but for more than one wave at least eight vectors a thread
    // (N32 C256 56x56 FP32 40 us in one wave, 35 in four).
    const long long wave = 3LL * facts.sms, threads = gcb::kStreamThreads;
    const long long vectors = ceil_div(count, vec ? per_vector : 1);
    long long grid = std::max(std::min(ceil_div(vectors, threads), wave), std::min(ceil_div(vectors, 8 * threads), 4 * wave));
    // A channel of one pixel is an element: one kernel for many rows instead of
    // a block for each.
    const long long px = drop.channel ? count / x->dims[0] / x->dims[1] : 1;
    if (px > 1) {
        const long long images = x->dims[0], channels = x->dims[1];
        if (channels > INT32_MAX) return gc_error(GC_UNSUPPORTED, "channel count out of range");
        P.decisions = static_cast<uint64_t>(images * channels);
        P.channels = static_cast<int>(channels);
        P.row = static_cast<uint64_t>(px);
        // Small planes and small images leave a warp or a block of the kernels
        // below little to do (N64 C512 7x7 bf16, plain: 17 us there, 5 us here;
        // N16384 C64 4x4 channels last: 57 and 21); from 512 bytes a plane and
        // 8 KB an image on, one decision per thread and a plain loop win
        // (N128 C256 14x14 FP32, plain: 15 us there, 16 here).
        const long long bytes = px * (16 / per_vector);
        if (plain ? bytes < 512 : bytes * channels <= 8192) {
            kind = kMapped;
            P.image = plain ? 0 : static_cast<uint64_t>(px * channels);
            if (!plain && vec && channels % per_vector != 0) {
                vec = false;
                grid = std::max(std::min(ceil_div(count, threads), wave), std::min(ceil_div(count, 8 * threads), 4 * wave));
            }
        } else if (plain) {
            kind = kPlanes;
            const long long warps = threads / 32, least = 32LL * (vec ? 4 * per_vector : gcb::kAhead);
            const long long wanted = std::max<long long>(1, 4 * wave * warps / (images * channels));
            P.chunk = static_cast<uint64_t>(gcb::round_up(ceil_div(px, wanted), least));
            P.chunks = (P.row + P.chunk - 1) / P.chunk;
            grid = static_cast<long long>(
                std::min<uint64_t>((P.decisions * P.chunks + warps - 1) / warps, static_cast<uint64_t>(4 * wave)));
        } else {
            kind = kChannels;
            vec = vec && channels % per_vector == 0;
            P.vcols = static_cast<int>(vec ? channels / per_vector : channels);
            P.cblocks = static_cast<int>(ceil_div(P.vcols, threads));
            P.vb = static_cast<int>(ceil_div(P.vcols, P.cblocks));
            P.lanes = static_cast<int>(threads / P.vb);
            const long long wanted = std::max<long long>(1, (vec ? 4 : 1) * wave / (images * P.cblocks));
            P.chunk = static_cast<uint64_t>(std::max<long long>(ceil_div(px, wanted), (vec ? 8LL : 4LL) * P.lanes));
            P.chunks = (P.row + P.chunk - 1) / P.chunk;
            const wide blocks = static_cast<wide>(images) * static_cast<wide>(P.chunks) * P.cblocks;
            if (blocks > INT32_MAX) return gc_error(GC_UNSUPPORTED, "more images than a grid has blocks");
            grid = static_cast<long long>(blocks);
        }
    }
    const void *fn = type == gcb::kElemF16    ? dropout_typed<__half>(kind, vec)
                     : type == gcb::kElemBF16 ? dropout_typed<__nv_bfloat16>(kind, vec)
                                              : dropout_typed<float>(kind, vec);
    if ((st = prepare_kernel(fn, dev, facts.smem_optin)) != GC_OK) return st;
    void *args[] = {&P};
    const cudaError_t e = gcb::launch_pdl(fn, dim3(static_cast<unsigned>(grid)), dim3(gcb::kStreamThreads), args,
                                          gcb::ring_space(vec ? per_vector : 1), reinterpret_cast<cudaStream_t>(stream));
    static const char *const names[] = {"element", "channels_last", "planes", "small_images"};
    return launched(e, PlanRecord::kDropout, names[kind], grid, gcb::kStreamThreads, vec ? 1 : 0);
} catch (...) {
    return internal_error();
}

}  // extern "C"
