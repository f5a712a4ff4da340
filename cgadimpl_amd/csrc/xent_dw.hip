// xent_dw.hip -- kernels of xent_gemm.hpp: dw = G^T x, G^T [vocab][tokens] k-contiguous
// and x [tokens][cols] k-strided.
#define AGK_RING_KERNELS
#define AGK_XENT_KERNELS
#include "xent_gemm.hpp"

namespace agk_xent {

int launch_dw(int shape, const Product& p, const AddEpi<true>& e) {
    return launch_product<false, true>(shape, p, e);
}
int launch_dw(int shape, const Product& p, const AddEpi<false>& e) {
    return launch_product<false, true>(shape, p, e);
}
int launch_dw(int shape, const Product& p, const AddEpi<true>& e, const PlanesK& k) {
    return launch_product<false, true>(shape, p, e, k);
}

}  // namespace agk_xent
