// xent_dx.hip -- kernels of xent_gemm.hpp: dx = G w: G^T [vocab][tokens] and w [vocab][cols] are
// both k-strided.
#define AGK_RING_KERNELS
#define AGK_XENT_KERNELS
#include "xent_gemm.hpp"

namespace agk_xent {

int launch_dx(int shape, const Product& p, const AddEpi<true>& e) {
    return launch_product<true, true>(shape, p, e);
}
int launch_dx(int shape, const Product& p, const AddEpi<true>& e, const PlanesK& k) {
    return launch_product<true, true>(shape, p, e, k);
}

}  // namespace agk_xent
