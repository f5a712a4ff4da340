// xent_lse.hip -- kernels of xent_gemm.hpp: the forward's product z^T = w x^T (both
// k-contiguous), reduced in its epilogue.
#define AGK_RING_KERNELS
#define AGK_XENT_KERNELS
#include "xent_gemm.hpp"

namespace agk_xent {

int launch_lse(int shape, const Product& p, const LseEpi<false>& e) {
    return launch_logits(shape, p, e);
}
int launch_lse(int shape, const Product& p, const LseEpi<true>& e, const PlanesK& k) {
    return launch_product<false, false>(shape, p, e, k);
}

}  // namespace agk_xent
