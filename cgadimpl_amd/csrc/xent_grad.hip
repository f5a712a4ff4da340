// xent_grad.hip -- kernels of xent_gemm.hpp: the backward's z^T = w x^T, which leaves as the
// gradient of the logits.
#define AGK_RING_KERNELS
#define AGK_XENT_KERNELS
#include "xent_gemm.hpp"

namespace agk_xent {

int launch_grad(int shape, const Product& p, const GradEpi<1>& e) {
    return launch_logits(shape, p, e);
}
int launch_grad(int shape, const Product& p, const GradEpi<2>& e, const PlanesK& k) {
    return launch_product<false, false>(shape, p, e, k);
}

}  // namespace agk_xent
