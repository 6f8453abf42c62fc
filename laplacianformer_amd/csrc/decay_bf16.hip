// decay_attention's kernels for bf16 (decay_common.h; the C entries are in decay_host.hip).
#include "decay_common.h"

namespace lfamd {

int decay_run_bf16(const DecayArgs& a, int out, hipStream_t st) {
  return out ? decay_dispatch<bf16s, true>(a, st) : decay_dispatch<bf16s, false>(a, st);
}

}  // namespace lfamd
