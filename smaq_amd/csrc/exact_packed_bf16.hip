// The bf16 kernels of exact_packed.h.
#include "exact_packed.h"

namespace smaq {

void launch_packed_bf16(const smaq_packed_params& p, const ScoreRule& rule, unsigned grid, int blocks, hipStream_t st) {
  launch_packed<bf16>(p, rule, grid, blocks, st);
}

}  // namespace smaq
