// Products of fp32 queries with four-bit rows (mx4_scores.h).
#include "mx4_scores.h"

namespace rag {

int mx4_launch_f32(const Mx4Shape& p, const Mx4ScoreArgs& a, long long grid, int device, hipStream_t s) { return mx4_launch_nd<5>(p, a, grid, device, s); }

}  // namespace rag
