// What the kernels over four-bit rows share: vector types, elements of the three float types, small reductions.
#pragma once
#include <float.h>
#include <math.h>

#include <type_traits>

#include "index.h"
#include "mx4.h"

namespace rag {

typedef int v4i __attribute__((ext_vector_type(4)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef float v2f __attribute__((ext_vector_type(2)));
typedef unsigned v2u __attribute__((ext_vector_type(2)));
typedef __bf16 v2bf __attribute__((ext_vector_type(2)));
typedef __bf16 v8bf __attribute__((ext_vector_type(8)));
typedef v4i v4i_apart __attribute__((aligned(2)));               // wide loads from addresses that are only aligned to their elements

template <int N, typename F>
__device__ __forceinline__ void static_for(F f) {
    if constexpr (N > 0) {
        static_for<N - 1>(f);
        f(std::integral_constant<int, N - 1>{});
    }
}

__device__ __forceinline__ float mx4_pow2(int e) { return __uint_as_float((unsigned)(e + 127) << 23); }   // -126 <= e <= 127
__device__ __forceinline__ float bf16_f32(unsigned h) { return __uint_as_float(h << 16); }
__device__ __forceinline__ float f16_f32(unsigned short h) {
    _Float16 v;
    __builtin_memcpy(&v, &h, 2);
    return (float)v;
}
// element i of a row of the given type (RAG_MX4_F32 / BF16 / F16)
__device__ __forceinline__ float mx4_elem(const void* row, int type, long long i) {
    if (type == RAG_MX4_F32) return static_cast<const float*>(row)[i];
    const unsigned short h = static_cast<const unsigned short*>(row)[i];
    return type == RAG_MX4_BF16 ? bf16_f32(h) : f16_f32(h);
}
// Eight consecutive elements from i on; past `dim` zero.  VEC: rows start on 16-byte boundaries.  Read past the caches' retention:
// nobody reads these rows again (writing 100k rows of 384 fp32: 43 -> 35 us).
template <int TYPE, bool VEC>
__device__ __forceinline__ void mx4_load8(const void* row, int i, int dim, float* v) {
    if (VEC && i + 8 <= dim) {
        if constexpr (TYPE == RAG_MX4_F32) {
#pragma unroll
            for (int j = 0; j < 8; j += 4) {
                const v4f x = __builtin_nontemporal_load(reinterpret_cast<const v4f*>(static_cast<const float*>(row) + i + j));
                v[j] = x.x; v[j + 1] = x.y; v[j + 2] = x.z; v[j + 3] = x.w;
            }
        } else {
            const v4i x = __builtin_nontemporal_load(reinterpret_cast<const v4i*>(static_cast<const unsigned short*>(row) + i));
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const unsigned w = (unsigned)x[j];
                v[2 * j] = TYPE == RAG_MX4_BF16 ? bf16_f32(w & 0xffffu) : f16_f32((unsigned short)w);
                v[2 * j + 1] = TYPE == RAG_MX4_BF16 ? __uint_as_float(w & 0xffff0000u) : f16_f32((unsigned short)(w >> 16));
            }
        }
        return;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = i + j < dim ? mx4_elem(row, TYPE, i + j) : 0.f;
}

__device__ __forceinline__ unsigned dpp_max_u32(unsigned v, unsigned o) { return v > o ? v : o; }
// the largest of |v| (as ordered bits) over each aligned group of 4 lanes
__device__ __forceinline__ unsigned quad_max(unsigned v) {
    v = dpp_max_u32(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0xB1, 0xF, 0xF, true));
    return dpp_max_u32(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0x4E, 0xF, 0xF, true));
}
__device__ __forceinline__ double wave_sum_f64(double v) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off, 64);
    return v;
}
// 1 / |x| of one row by one wave, as a power of two and a factor: |2^k x| lies in [1/2, 1) whatever the norm, and the factor, in (1, 2],
// is rounded once.  The sum of squares is one of fp64; a zero row keeps its zeros, one that is not finite becomes NaN.
__device__ __forceinline__ float wave_inv_norm(const void* row, int type, int dim, int lane, int& k) {
    double ss = 0.0;
    for (int i = lane; i < dim; i += 64) {
        const double x = (double)mx4_elem(row, type, i);
        ss = fma(x, x, ss);
    }
    ss = wave_sum_f64(ss);
    k = 0;
    if (ss == 0.0) return 1.f;
    if (!(ss <= DBL_MAX)) return NAN;
    int e;
    const double m = frexp(sqrt(ss), &e);
    k = -e;
    return (float)(1.0 / m);
}

}  // namespace rag
