// The kernels of qph_mask4.h for float16 queries and results.
#include "qph_mask4.h"

namespace qph {

int launch_mask4_f16(const Mask4& g, const Mask4Plan& p, int dh, hipStream_t s) {
  return launch_mask4<F16>(g, p, dh, s);
}

}  // namespace qph
