// layer_host.h — host side that the layer operators (layernorm.cu, linear.cu, muon.cu) share.
#pragma once
#include <stdint.h>
#include "state.h"

namespace thc {

// The buffers of one call: the first `n_required` of each list must be given (id != 0), all given ones must be live and hold
// at least need[i] bytes, and no output may be another output or an input — except that the first output may be the input j
// whose bit j is set in `inplace`.  False, with the reason in the sticky error, if not.
bool layer_buffers(const char *who, const uint32_t *ins, const uint64_t *in_need, int n_in, int in_required,
                   const uint32_t *outs, const uint64_t *out_need, int n_out, int out_required, uint32_t inplace);

// Scratch of an operator, or null where a captured step would need more than there is (the reason is in the sticky error; the capture
// is refused at its end).
void *layer_scratch(const char *who, uint64_t bytes);

// Whether this is the first call for the current device with this `seen` (-1 at first): kernel attributes belong to a device.
static inline bool first_on_device(int &seen) { if (seen == g.device) return false; seen = g.device; return true; }

// what profile_report says of the launch that comes next
static inline void layer_estimate(double ops, double bytes) { if (g.profile) { g.prof_ops = (unsigned long long)ops; g.prof_bytes = (unsigned long long)bytes; } }

// Launches a kernel that begins with depend() (layer_common.cuh) on the backend's stream.  The set-up of a kernel and its blocks' start
// overlap the end of the kernel before it, which is worth some 2 us of the 4 that a launch in a chain costs.
// cluster_y: blocks of a cluster along y, where the kernel does not say itself.
template <class... P, class... A>
static void chain_cluster(uint32_t cluster_y, void (*kernel)(P...), dim3 grid, uint32_t threads, size_t smem, A... args) {
    cudaLaunchConfig_t c;
    cudaLaunchAttribute a[2];
    a[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    a[0].val.programmaticStreamSerializationAllowed = 1;
    a[1].id = cudaLaunchAttributeClusterDimension;
    a[1].val.clusterDim.x = 1; a[1].val.clusterDim.y = cluster_y; a[1].val.clusterDim.z = 1;
    c.gridDim = grid; c.blockDim = dim3(threads); c.dynamicSmemBytes = smem; c.stream = g.stream;
    c.attrs = a; c.numAttrs = cluster_y ? 2 : 1;
    THC_CUDA_OK(cudaLaunchKernelEx(&c, kernel, static_cast<P>(args)...));
}
template <class... P, class... A>
static void chain(void (*kernel)(P...), dim3 grid, uint32_t threads, size_t smem, A... args) { chain_cluster(0, kernel, grid, threads, smem, args...); }

}  // namespace thc
