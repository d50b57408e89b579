// Attention of several new tokens over f16 caches.
#include <hip/hip_runtime.h>

#include "tree.h"

namespace trellis {

void launch_tree_f16(const TreeLaunch& l) { launch_tree<_Float16>(l); }

}  // namespace trellis
