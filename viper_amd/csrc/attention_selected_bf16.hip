// Attention over selected pages of a bf16 cache.
#include "attention.h"
namespace vq {
AttnFn attn_selected_bf16(int D, int qt, int W) { return attn_fn<VIPER_KV_BF16, true>(D, qt, W); }
}  // namespace vq
