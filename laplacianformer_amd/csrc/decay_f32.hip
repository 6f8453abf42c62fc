// decay_attention's kernels for f32 (decay_common.h; the C entries are in decay_host.hip).
#include "decay_common.h"

namespace lfamd {

int decay_run_f32(const DecayArgs& a, int out, hipStream_t st) {
  return out ? decay_dispatch<float, true>(a, st) : decay_dispatch<float, false>(a, st);
}

}  // namespace lfamd
