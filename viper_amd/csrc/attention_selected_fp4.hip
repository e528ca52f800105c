// Attention over selected pages of an FP4 cache.
#include "attention.h"
namespace vq {
AttnFn attn_selected_fp4(int D, int qt, int W) { return attn_fn<VIPER_KV_FP4, true>(D, qt, W); }
}  // namespace vq
