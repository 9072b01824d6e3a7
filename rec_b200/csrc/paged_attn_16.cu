// Paged decode attention over 16-bit rows.
#include "paged_attn.cuh"

namespace rec {

namespace {
template <bool F16>
struct Cfg16 {
  template <int DP, int NT>
  struct of {
    using type = PagedCfg<16, 16, F16, DP, NT, 1, paged_warps(DP, NT), 1>;
  };
};
}  // namespace

cudaError_t paged_attn_bf16(const PagedView& p, const PagedAttnArgs& a, int sms, cudaStream_t st) {
  return paged_attn_by_shape<Cfg16<false>::of>(p, a, sms, st);
}
cudaError_t paged_attn_fp16(const PagedView& p, const PagedAttnArgs& a, int sms, cudaStream_t st) {
  return paged_attn_by_shape<Cfg16<true>::of>(p, a, sms, st);
}

}  // namespace rec
