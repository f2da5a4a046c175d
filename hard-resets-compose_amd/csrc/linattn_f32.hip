// The chunked walk of linear attention for one operand type (linattn_walk.h).
#include "linattn_walk.h"

namespace lsh {
int la_launch_f32(const LaWalks& all, bool sums, hipStream_t st) { return la_launch<float, float>(all, sums, st); }
}  // namespace lsh
