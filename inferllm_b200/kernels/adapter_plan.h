// The plan of a step's tokens among low-rank adapters (csrc/adapters.h), made on the host once per step.
#pragma once
#include <vector>

#include "csrc/adapters.h"

namespace illm {
namespace ops {

// The smallest sizes that hold the plan of these tokens.  index[t] is a token's adapter, -1 for none; ranks[a] the rank of
// adapter a.  KernelError for an index outside the adapters, a rank outside [0, 256] or too many tokens.
AdapterPlanSizes adapter_plan_sizes(const int* index, int T, const int* ranks, int count);
// Sizes that hold any plan of T tokens over `count` adapters of ranks up to max_rank (for captured steps, whose arrays must
// not move): of one sequence, which has one adapter, or of any.
AdapterPlanSizes adapter_plan_bound(int T, int count, int max_rank, bool one_sequence);
// Fills out[0 .. layout(sizes).total).
void adapter_plan_fill(const int* index, int T, const int* ranks, int count, const AdapterPlanSizes& sizes, int* out);

}  // namespace ops
}  // namespace illm
