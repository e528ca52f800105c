// Attention over an int8 cache.
#include "attention.h"
namespace vq {
AttnFn attn_kernels_int8(int D, int qt, int W) { return attn_fn<VIPER_KV_INT8>(D, qt, W); }
}  // namespace vq
