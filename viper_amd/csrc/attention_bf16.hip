// Attention over a bf16 cache.
#include "attention.h"
namespace vq {
const void* attn_kernel_bf16(int D, int qt) { return attn_fn<false>(D, qt); }
}  // namespace vq
