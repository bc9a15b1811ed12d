// kv_attn4.cu — decode attention instances of 4-bit pools (templates in kv_attn.cuh), over whole
// sequences and over picked blocks.
#include "kv_attn.cuh"

namespace krill {
namespace {

template <int D, int NG>
cudaError_t launch4(const AttnParams& p, int grid, cudaStream_t stream) {
  if (p.sel != nullptr) return launch_tc_r<D, NG, 8, kFmtInt4, true>(p, grid, stream);
  return launch_tc_r<D, NG, 8, kFmtInt4>(p, grid, stream);
}

}  // namespace

cudaError_t launch_attention4(const Geom& g, const AttnParams& p, int grid, cudaStream_t stream) {
  if (g.D == 64 && g.NG == 1) return launch4<64, 1>(p, grid, stream);
  if (g.D == 128 && g.NG == 2) return launch4<128, 2>(p, grid, stream);
  if (g.D == 128 && g.NG == 1) return launch4<128, 1>(p, grid, stream);
  if (g.D == 256 && g.NG == 4) return launch4<256, 4>(p, grid, stream);
  if (g.D == 256 && g.NG == 1) return launch4<256, 1>(p, grid, stream);
  return cudaErrorInvalidValue;
}

int describe_attention4(const Geom& g, const AttnParams& p, char* buf, size_t cap) {
  if (g.D == 64) return tc_desc_r<64, 1, kFmtInt4>(p, buf, cap);
  if (g.D == 128 && g.NG == 2) return tc_desc_r<128, 2, kFmtInt4>(p, buf, cap);
  if (g.D == 128) return tc_desc_r<128, 1, kFmtInt4>(p, buf, cap);
  if (g.NG == 4) return tc_desc_r<256, 4, kFmtInt4>(p, buf, cap);
  return tc_desc_r<256, 1, kFmtInt4>(p, buf, cap);
}

}  // namespace krill
