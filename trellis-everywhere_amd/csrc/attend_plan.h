// attend_plan.h — the attention's arithmetic on sizes, as plain functions that the host and the kernels share.
#pragma once

namespace trellis {

// The dim at which a lane begins to load 8 dims of a query head for k-step j: 32 j + 8 g, or the row's last 8 where it
// has none there (head dims that do not fill the last step's lane groups g; the values then count as zeros).
constexpr int att_q_dim(int j, int g, int d) { return 32 * j + 8 * g < d ? 32 * j + 8 * g : d - 8; }

}  // namespace trellis
