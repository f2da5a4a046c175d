// The chunked walk of linear attention for one operand type (linattn_walk.h).
#include "linattn_walk.h"

namespace lsh {
int la_launch_f16(const LaWalks& all, bool sums, hipStream_t st) { return la_launch<f16_t, f16_t>(all, sums, st); }
}  // namespace lsh
