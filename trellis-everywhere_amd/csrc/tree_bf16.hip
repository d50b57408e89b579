// Attention of several new tokens over bf16 caches.
#include <hip/hip_runtime.h>

#include "tree.h"

namespace trellis {

void launch_tree_bf16(const TreeLaunch& l) { launch_tree<bf16_t>(l); }

}  // namespace trellis
