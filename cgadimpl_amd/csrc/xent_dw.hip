// xent_dw.hip -- kernels of xent_gemm.hpp: dw = G^T x, G^T [vocab][tokens] k-contiguous
// and x [tokens][cols] k-strided.
#define AGK_RING_KERNELS
#define AGK_XENT_KERNELS
#include "xent_gemm.hpp"

namespace agk_xent {

// Few tokens: the short kernel, where its tiles (the smallest) fit a grid.
bool is_short(const Product& p) {
    const int64_t tiles = static_cast<int64_t>((p.M + kShortM - 1) / kShortM) *
                          ((p.N + kShortN - 1) / kShortN);
    return p.K <= kShortK && agk::grid_fits(tiles, 256);
}

int launch_dw(int shape, const Product& p, const AddEpi<true>& e) {
    if (is_short(p)) return launch_short<false, true>(p, e);
    return launch_product<false, true>(shape, p, e);
}
int launch_dw(int shape, const Product& p, const AddEpi<false>& e) {
    if (is_short(p)) return launch_short<false, true>(p, e);
    return launch_product<false, true>(shape, p, e);
}
int launch_dw(int shape, const Product& p, const AddEpi<true>& e, const PlanesK& k) {
    return launch_product<false, true>(shape, p, e, k);
}

}  // namespace agk_xent
