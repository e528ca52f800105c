// Attention over a bf16 cache.
#include "attention.h"
namespace vq {
AttnFn attn_kernels_bf16(int D, int qt, int W) { return attn_fn<VIPER_KV_BF16>(D, qt, W); }
}  // namespace vq
