// layer_host.h — host side that the layer operators (layernorm.cu, linear.cu, muon.cu) share.
#pragma once
#include <stdint.h>

namespace thc {

// The buffers of one call: the first `n_required` of each list must be given (id != 0), all given ones must be live and hold
// at least need[i] bytes, and no output may be another output or an input — except that the first output may be the input j
// whose bit j is set in `inplace`.  False, with the reason in the sticky error, if not.
bool layer_buffers(const char *who, const uint32_t *ins, const uint64_t *in_need, int n_in, int in_required,
                   const uint32_t *outs, const uint64_t *out_need, int n_out, int out_required, uint32_t inplace);

}  // namespace thc
