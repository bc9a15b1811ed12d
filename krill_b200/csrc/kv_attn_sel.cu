// kv_attn_sel.cu — decode attention over picked blocks of int8 pools (templates in kv_attn.cuh).
#include "kv_attn.cuh"

namespace krill {

cudaError_t launch_attention_sel8(const Geom& g, const AttnParams& p, int grid, cudaStream_t stream) {
  if (g.D == 64 && g.NG == 1) return launch_tc_r<64, 1, 8, kFmtInt8, true>(p, grid, stream);
  if (g.D == 128 && g.NG == 2) return launch_tc_r<128, 2, 8, kFmtInt8, true>(p, grid, stream);
  if (g.D == 128 && g.NG == 1) return launch_tc_r<128, 1, 8, kFmtInt8, true>(p, grid, stream);
  if (g.D == 256 && g.NG == 4) return launch_tc_r<256, 4, 8, kFmtInt8, true>(p, grid, stream);
  if (g.D == 256 && g.NG == 1) return launch_tc_r<256, 1, 8, kFmtInt8, true>(p, grid, stream);
  return cudaErrorInvalidValue;
}

}  // namespace krill
