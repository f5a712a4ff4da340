// xent_f32.hip -- the vocabulary head's products of few fp32 tokens on the fp32 matrix
// instruction (gemm_f32.hpp): w is read as it lies, where planes (PlanesK) would first be written
// and read again, more than the few tokens' products take.
#include "xent_gemm.hpp"

#include "gemm_f32.hpp"

namespace agk_xent {

namespace {

template <int BM, int BN, int WVM, bool A_KC, bool B_KC, class Epi>
__global__ __launch_bounds__(256, 2) void xent_f32_kernel(
    const float* __restrict__ A, int64_t lda, const float* __restrict__ B, int64_t ldb, int M,
    int N, int K, int k_slice, const Epi epi, int tiles_m, int tiles_n) {
    const int k0 = static_cast<int>(blockIdx.y) * k_slice;
    A += A_KC ? k0 : static_cast<int64_t>(k0) * lda;
    B += B_KC ? k0 : static_cast<int64_t>(k0) * ldb;
    const int k = blockIdx.y + 1 < gridDim.y ? k_slice : K - k0;
    agk_sgemm::f32_body<BM, BN, WVM, A_KC, B_KC>(A, lda, B, ldb, M, N, k, tiles_m, tiles_n, epi);
}

template <int BM, int BN, int WVM, bool A_KC, bool B_KC, class Epi>
int launch(const ProductF32& p, const Epi& e) {
    const int tiles_m = (p.M + BM - 1) / BM, tiles_n = (p.N + BN - 1) / BN;
    hipLaunchKernelGGL((xent_f32_kernel<BM, BN, WVM, A_KC, B_KC, Epi>),
                       dim3(tiles_m * tiles_n, p.slices), dim3(256), 0, p.st, p.A, p.lda, p.B,
                       p.ldb, p.M, p.N, p.K, p.k_slice, e, tiles_m, tiles_n);
    return agk::check_launch();
}

}  // namespace

// Logits: w [vocab][cols] along M, x [tokens][cols] along N, both k-contiguous.
template <class Epi>
int launch_logits32(const ProductF32& p, const Epi& e) {
    return p.N <= 32 ? launch<128, 32, 4, true, true>(p, e) : launch<64, 64, 2, true, true>(p, e);
}
int launch_lse(const ProductF32& p, const LseEpi<false>& e) { return launch_logits32(p, e); }
int launch_grad(const ProductF32& p, const GradEpiF32& e) { return launch_logits32(p, e); }
// dx = G w: G^T [vocab][tokens] and w [vocab][cols], both k-strided.
int launch_dx(const ProductF32& p, const AddEpi<true>& e) {
    return p.M <= 32 ? launch<32, 128, 1, false, false>(p, e)
                     : launch<64, 64, 2, false, false>(p, e);
}
// dw = G^T x: G^T [vocab][tokens] k-contiguous, x [tokens][cols] k-strided.
int launch_dw(const ProductF32& p, const AddEpi<true>& e) {
    return launch<64, 64, 2, true, false>(p, e);
}

}  // namespace agk_xent
