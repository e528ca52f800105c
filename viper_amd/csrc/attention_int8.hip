// Attention over an int8 cache.
#include "attention.h"
namespace vq {
const void* attn_kernel_int8(int D, int qt) { return attn_fn<true>(D, qt); }
}  // namespace vq
