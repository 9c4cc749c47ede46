// Products of fp32 queries with four-bit rows (mx4_scores.h).
#include "mx4_scores.h"

namespace rag {

int mx4_launch_f32(const Mx4Shape& p, const Mx4ScoreArgs& a, long long grid, int device, hipStream_t s) {
    MX4_MANY(3, 16, 3, 2);
    MX4_MANY(3, 16, 6, 3);
    MX4_FEW(3, 4, 1);
    MX4_FEW(3, 4, 2);
    MX4_CASE(3, 4, 1, 8, 8, 8, 0);
    return fail(RAG_ERR_INVALID, "internal: no four-bit product kernel for this shape");
}

}  // namespace rag
