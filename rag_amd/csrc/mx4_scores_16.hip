// Products of bf16 and fp16 queries with four-bit rows (mx4_scores.h).
#include "mx4_scores.h"

namespace rag {

int mx4_launch_16(const Mx4Shape& p, const Mx4ScoreArgs& a, long long grid, int device, hipStream_t s) { return mx4_launch_nd<4>(p, a, grid, device, s); }

}  // namespace rag
