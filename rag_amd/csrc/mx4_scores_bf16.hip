// Products of bf16 queries with four-bit rows (mx4_scores.h).
#include "mx4_scores.h"

namespace rag {

int mx4_launch_bf16(const Mx4Shape& p, const Mx4ScoreArgs& a, long long grid, int device, hipStream_t s) {
    MX4_MANY(1, 16, 4, 4);
    MX4_FEW(1, 4, 1);
    MX4_FEW(1, 8, 1);
    MX4_FEW(1, 16, 1);
    MX4_FEW(1, 16, 2);
    MX4_CASE(1, 16, 1, 8, 8, 8, 0);
    return fail(RAG_ERR_INVALID, "internal: no four-bit product kernel for this shape");
}

}  // namespace rag
