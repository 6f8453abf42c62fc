// decay_attention's kernels for f16 (decay_common.h; the C entries are in decay_host.hip).
#include "decay_common.h"

namespace lfamd {

int decay_run_f16(const DecayArgs& a, int out, hipStream_t st) {
  return out ? decay_dispatch<f16s, true>(a, st) : decay_dispatch<f16s, false>(a, st);
}

}  // namespace lfamd
