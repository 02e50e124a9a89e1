// Attention over the paged KV cache behind a sliding window, with sinks: the
// kernels of paged_attn.hpp for that scope.
#include "paged_attn.hpp"

namespace mtp {

int launch_window(const char* who, const PAttn& p, const AttnPlan& a, int D, int bits, hipStream_t st) {
  return launch_scope<kWindow>(who, p, a, D, bits, st);
}

}  // namespace mtp
