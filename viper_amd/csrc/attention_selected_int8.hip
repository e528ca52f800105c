// Attention over selected pages of an int8 cache.
#include "attention.h"
namespace vq {
AttnFn attn_selected_int8(int D, int qt, int W) { return attn_fn<VIPER_KV_INT8, true>(D, qt, W); }
}  // namespace vq
