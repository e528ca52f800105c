// Attention over an int8 cache.
#include "attention.h"
namespace vq {
AttnFn attn_kernels_int8(int D, int qt, int W) { return attn_fn<true>(D, qt, W); }
}  // namespace vq
