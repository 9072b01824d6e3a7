// Paged decode attention over affine codes, K of 4 bits.
#include "paged_attn.cuh"

namespace rec {

namespace {
template <int VB>
struct CfgCodes {
  template <int DP, int NT>
  struct of {
    // two m tiles a step keep as many bytes on their way as one of 16-bit rows
    using type = PagedCfg<4, VB, true, DP, NT, DP == 256 ? 1 : 2, paged_warps(DP, NT), 1>;
  };
};
}  // namespace

cudaError_t paged_attn_codes4(const PagedView& p, const PagedAttnArgs& a, int sms, cudaStream_t st) {
  return p.v_bits == 8 ? paged_attn_by_shape<CfgCodes<8>::of>(p, a, sms, st)
                       : paged_attn_by_shape<CfgCodes<4>::of>(p, a, sms, st);
}

}  // namespace rec
