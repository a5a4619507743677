// The kernels of qph_mask4.h for float32 queries and results.
#include "qph_mask4.h"

namespace qph {

int launch_mask4_f32(const Mask4& g, const Mask4Plan& p, int dh, hipStream_t s) {
  return launch_mask4<F32>(g, p, dh, s);
}

}  // namespace qph
