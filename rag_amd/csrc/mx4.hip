// Rows kept at four bits (e2m1 values, one power-of-two scale per group of 32 consecutive elements: the MX layout):
// quantising rows as they are written, reading them back, and multiplying them with queries.
//
// value(row, i) = sign * T[code & 7] * 2^(scale[i / 32] - 127),  T = {0, 0.5, 1, 1.5, 2, 3, 4, 6};  scale 255: NaN.
//
// Products run on the scaled matrix instruction, which reads four-bit values and their scales as they are stored: nothing
// is unpacked.  Its other operand is eight bits wide (e4m3, scaled per 32 as well), so a query is split into digits first:
// with 2^E the power of two that brings the largest element of a group of 32 into [8, 16),
//     x = 2^E * (d0 + d1 / 32 + d2 / 32^2 + ...),   dj a whole number in [-16, 16],
// and a whole number up to 16 is exact in e4m3.  Each digit is a row of the matrix tile of its own, with the scale
// 2^(E - 5j), so one instruction multiplies all digits; the digits' sums are added at the end.  fp32 queries take five
// digits (what is left is at most 2^-24 of the group's largest element), bf16 and fp16 four (at most 2^-19 of it: every
// element down to 2^-12 (bf16) / 2^-9 (fp16) of the largest one is exact).  Products of such digits with four-bit values
// are multiples of 1/2 up to 96, which the instruction adds without loss; it adds across groups and to the accumulator in
// fp32.  One query fills four or five of the tile's sixteen rows, so three (fp32) or four queries cost what one does.
#include <float.h>
#include <limits.h>
#include <math.h>
#include <stdlib.h>

#include <algorithm>
#include <type_traits>

#include "index.h"
#include "mx4.h"
#include "topk_keys.h"

namespace rag {

typedef int v4i __attribute__((ext_vector_type(4)));
typedef int v8i __attribute__((ext_vector_type(8)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef float v2f __attribute__((ext_vector_type(2)));
typedef unsigned v2u __attribute__((ext_vector_type(2)));

struct Mx4DeviceGuard {
    int prev = -1;
    bool ok = true, moved = false;
    explicit Mx4DeviceGuard(int dev) {
        if (hipGetDevice(&prev) != hipSuccess) prev = -1;
        if (prev != dev) {
            moved = true;
            ok = hipSetDevice(dev) == hipSuccess;
        }
    }
    ~Mx4DeviceGuard() {
        if (moved && prev >= 0) (void)hipSetDevice(prev);
    }
};

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
// N (4 or 8) consecutive elements from i on; past `dim` zero.  vec: rows start on 16-byte boundaries.  ONCE: read past the
// caches' retention, for rows that nobody reads again (writing 100k rows of 384 fp32: 43 -> 35 us).
template <int N, bool ONCE = false>
__device__ __forceinline__ void mx4_load(const void* row, int type, int i, int dim, int vec, float* v) {
    if (vec && i + N <= dim) {
        if (type == RAG_MX4_F32) {
#pragma unroll
            for (int j = 0; j < N; j += 4) {
                const v4f* p = reinterpret_cast<const v4f*>(static_cast<const float*>(row) + i + j);
                const v4f x = ONCE ? __builtin_nontemporal_load(p) : *p;
                v[j] = x.x; v[j + 1] = x.y; v[j + 2] = x.z; v[j + 3] = x.w;
            }
        } else {
            unsigned w[N / 2];
            if constexpr (N == 8) {
                const v4i* p = reinterpret_cast<const v4i*>(static_cast<const unsigned short*>(row) + i);
                const v4i x = ONCE ? __builtin_nontemporal_load(p) : *p;
                w[0] = x.x; w[1] = x.y; w[2] = x.z; w[3] = x.w;
            } else {
                const v2u x = *reinterpret_cast<const v2u*>(static_cast<const unsigned short*>(row) + i);
                w[0] = x.x; w[1] = x.y;
            }
#pragma unroll
            for (int j = 0; j < N / 2; ++j) {
                v[2 * j] = type == RAG_MX4_BF16 ? bf16_f32(w[j] & 0xffffu) : f16_f32((unsigned short)w[j]);
                v[2 * j + 1] = type == RAG_MX4_BF16 ? __uint_as_float(w[j] & 0xffff0000u) : f16_f32((unsigned short)(w[j] >> 16));
            }
        }
        return;
    }
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] = i + j < dim ? mx4_elem(row, type, i + j) : 0.f;
}

__device__ __forceinline__ unsigned dpp_max_u32(unsigned v, unsigned o) { return v > o ? v : o; }
// the largest of |v| (as ordered bits) over each aligned group of 4 / 8 lanes
__device__ __forceinline__ unsigned quad_max(unsigned v) {
    v = dpp_max_u32(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0xB1, 0xF, 0xF, true));
    return dpp_max_u32(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0x4E, 0xF, 0xF, true));
}
__device__ __forceinline__ unsigned oct_max(unsigned v) {
    v = quad_max(v);
    return dpp_max_u32(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0x141, 0xF, 0xF, true));   // row_half_mirror
}
__device__ __forceinline__ double wave_sum_f64(double v) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off, 64);
    return v;
}
// 1 / |x| of one row by one wave: the sum of squares in fp64, rounded once (a zero row keeps its zeros)
__device__ __forceinline__ float wave_inv_norm(const void* row, int type, int dim, int lane) {
    double ss = 0.0;
    for (int i = lane; i < dim; i += 64) {
        const double x = (double)mx4_elem(row, type, i);
        ss = fma(x, x, ss);
    }
    ss = wave_sum_f64(ss);
    return ss > 0.0 ? (float)(1.0 / sqrt(ss)) : ss == 0.0 ? 1.f : (float)ss;      // NaN stays NaN
}

// ------------------------------------------------------------------------------------------------ writing rows
// Bound by HBM: dim * size bytes in, 0.53 dim bytes out per row.  A lane takes 8 consecutive elements, four lanes a group:
// loads of 16 (two for fp32) and stores of 4 bytes per lane, both contiguous over the wave; the loads of four such units
// are under way at once.
struct Mx4WriteArgs {
    uint8_t* codes;
    uint8_t* scales;
    long long n;                 // rows of the store
    const long long* rows;       // nullptr: row `first + i`
    int* owner;                  // nullptr, or owner[r] = 1 + the last i that names row r (mx4_claim_kernel)
    long long first;
    long long count;
    const void* x;
    long long ldx;               // elements
    int dim, code_ld, scale_ld, normalize;
    int upr;                     // units of 8 elements per (padded) row
    unsigned per;                // ceil(2^32 / upr): u / upr == (u * per) >> 32 for the units of a workgroup
    int per_block;               // rows a workgroup takes
};
constexpr int MX4_ROWS = 64;                 // most rows of one workgroup
constexpr int MX4_FEW = 256;                 // up to so many positions a workgroup looks for repeated ones itself
constexpr int MX4_UNITS = 4;

// A position that is named twice keeps the last of its rows: the highest index wins the claim, whatever the order of arrival.
__global__ __launch_bounds__(256) void mx4_claim_kernel(const long long* rows, long long count, long long n, int* owner) {
    const long long i = blockIdx.x * 256ll + threadIdx.x;
    if (i >= count) return;
    const long long r = rows[i];
    if (r >= 0 && r < n) atomicMax(&owner[r], (int)(i + 1));
}

// AT: rows go to named positions, and those that are skipped are not fetched (for consecutive rows the test would cost 10 %)
template <int TYPE, bool VEC, bool AT>
__global__ __launch_bounds__(256) void mx4_write_kernel(Mx4WriteArgs a) {
    __shared__ long long s_to[MX4_ROWS];
    __shared__ float s_inv[MX4_ROWS];
    __shared__ int s_late[MX4_ROWS];
    const long long i0 = (long long)blockIdx.x * a.per_block;
    const int nr = (int)(a.count - i0 < a.per_block ? a.count - i0 : a.per_block);
    const int tid = threadIdx.x, lane = tid & 63;
    constexpr size_t ESIZE = TYPE == RAG_MX4_F32 ? 4 : 2;
    const char* x = static_cast<const char*>(a.x) + (size_t)i0 * a.ldx * ESIZE;
    if (tid < nr) {
        long long to = a.first + i0 + tid;
        if (AT) {
            to = a.rows[i0 + tid];
            if (to < 0 || to >= a.n) to = -1;
            else if (a.owner) {
                if (a.owner[to] != (int)(i0 + tid + 1)) to = -1;
                else a.owner[to] = 0;       // only the winner sees its own number here, so no other row is misled by the reset
            }
        }
        s_to[tid] = to;
        s_inv[tid] = 1.f;
        s_late[tid] = 0;
    }
    __syncthreads();
    if (AT && !a.owner && a.count > 1) {                     // at most MX4_FEW positions: does a later row name the same one?
        const long long mine = tid < a.count ? a.rows[tid] : -1;
        for (int r = 0; r < nr; ++r)
            if (mine >= 0 && mine == s_to[r] && tid > i0 + r) s_late[r] = 1;
        __syncthreads();
        if (tid < nr && s_late[tid]) s_to[tid] = -1;
        __syncthreads();
    }
    if (a.normalize) {
        for (int r = tid >> 6; r < nr; r += 4) {
            const float inv = wave_inv_norm(x + (size_t)r * a.ldx * ESIZE, TYPE, a.dim, lane);
            if (lane == 0) s_inv[r] = inv;
        }
        __syncthreads();
    }
    const int units = nr * a.upr;
    for (int u0 = tid; u0 < units; u0 += 256 * MX4_UNITS) {
        float v[MX4_UNITS][8];
#pragma unroll
        for (int j = 0; j < MX4_UNITS; ++j) {
            const int u = u0 + 256 * j < units ? u0 + 256 * j : u0;
            const int r = (int)__umulhi((unsigned)u, a.per), c = u - r * a.upr;
            if (!AT || s_to[r] >= 0) mx4_load<8, true>(x + (size_t)r * a.ldx * ESIZE, TYPE, c * 8, a.dim, VEC, v[j]);
        }
#pragma unroll
        for (int j = 0; j < MX4_UNITS; ++j) {
            const int u = u0 + 256 * j;
            if (u >= units) break;
            const int r = (int)__umulhi((unsigned)u, a.per), c = u - r * a.upr;
            const long long to = s_to[r];
            if (AT && to < 0) continue;                                // uniform over the four lanes of a group
            const float inv = s_inv[r];
            unsigned most = 0;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                v[j][i] *= inv;
                const unsigned m = __float_as_uint(v[j][i]) & 0x7fffffffu;
                most = m > most ? m : most;
            }
            most = quad_max(most);
            // scale: floor(log2(most)) - 2, one more where most / 2^floor > 1.75 (then 6 is nearer than the 8 that four bits lack)
            int e = (int)(most >> 23) - 129 + ((most & 0x7fffffu) > 0x600000u ? 1 : 0);
            e = e < -126 ? -126 : e > 125 ? 125 : e;
            const bool bad = most >= 0x7f800000u;                // a NaN or an infinity: the group is NaN
            const float scale = mx4_pow2(e);
            unsigned w = 0;
            w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[j][0], v[j][1], scale, 0);
            w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[j][2], v[j][3], scale, 1);
            w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[j][4], v[j][5], scale, 2);
            w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[j][6], v[j][7], scale, 3);
            *reinterpret_cast<unsigned*>(a.codes + mx4_code_at(to, a.code_ld, c >> 4) + (c & 15) * 4) = bad ? 0u : w;
            if ((c & 3) == 0) a.scales[(size_t)to * a.scale_ld + mx4_scale_at(c >> 2)] = bad ? 255 : (uint8_t)(e + 127);
        }
    }
}

// ------------------------------------------------------------------------------------------------ reading rows
// Bound by HBM, mostly by what it writes.  A lane makes 8 elements from 4 bytes of codes and a scale; four such units are under
// way at once, behind one fetch of the workgroup's positions.
struct Mx4ReadArgs {
    const uint8_t* codes;
    const uint8_t* scales;
    long long n;
    const long long* rows;
    long long count;
    void* out;                   // [count][dim]
    int dim, code_ld, scale_ld;
    int upr;
    unsigned per;                // as for writing; not used where upr is 1
    int per_block;
};

__device__ __forceinline__ unsigned pack16(int type, float lo, float hi) {
    if (type == RAG_MX4_BF16) {                                  // four-bit values fit bf16 exactly (subnormal ones round to even)
        unsigned a = __float_as_uint(lo), b = __float_as_uint(hi);
        const unsigned ra = lo != lo ? 0x7fc0u : (a + 0x7fffu + ((a >> 16) & 1u)) >> 16;
        const unsigned rb = hi != hi ? 0x7fc0u : (b + 0x7fffu + ((b >> 16) & 1u)) >> 16;
        return ra | (rb << 16);
    }
    const _Float16 x = (_Float16)lo, y = (_Float16)hi;           // to nearest even
    unsigned short a, b;
    __builtin_memcpy(&a, &x, 2);
    __builtin_memcpy(&b, &y, 2);
    return (unsigned)a | ((unsigned)b << 16);
}

template <int TYPE, bool VEC>
__global__ __launch_bounds__(256) void mx4_read_kernel(Mx4ReadArgs a) {
    __shared__ long long s_from[MX4_ROWS];
    const long long i0 = (long long)blockIdx.x * a.per_block;
    const int nr = (int)(a.count - i0 < a.per_block ? a.count - i0 : a.per_block);
    const int tid = threadIdx.x;
    if (tid < nr) {
        const long long from = a.rows[i0 + tid];
        s_from[tid] = from >= 0 && from < a.n ? from : -1;
    }
    __syncthreads();
    const int units = nr * a.upr;
    for (int u0 = tid; u0 < units; u0 += 256 * MX4_UNITS) {
        unsigned w[MX4_UNITS];
        int b[MX4_UNITS];
#pragma unroll
        for (int j = 0; j < MX4_UNITS; ++j) {
            const int u = u0 + 256 * j < units ? u0 + 256 * j : u0;
            const int r = a.upr == 1 ? u : (int)__umulhi((unsigned)u, a.per), c = u - r * a.upr;
            const long long from = s_from[r];
            w[j] = 0;
            b[j] = 127;
            if (from >= 0) {
                w[j] = *reinterpret_cast<const unsigned*>(a.codes + mx4_code_at(from, a.code_ld, c >> 4) + (c & 15) * 4);
                b[j] = a.scales[(size_t)from * a.scale_ld + mx4_scale_at(c >> 2)];
            }
        }
#pragma unroll
        for (int j = 0; j < MX4_UNITS; ++j) {
            const int u = u0 + 256 * j;
            if (u >= units) break;
            const int r = a.upr == 1 ? u : (int)__umulhi((unsigned)u, a.per), c = u - r * a.upr;
            const float f = b[j] == 255 ? NAN : b[j] == 0 ? __uint_as_float(0x00400000u) : __uint_as_float((unsigned)b[j] << 23);
            float v[8];
            v2f p;
            p = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[j], 1.f, 0); v[0] = p.x * f; v[1] = p.y * f;
            p = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[j], 1.f, 1); v[2] = p.x * f; v[3] = p.y * f;
            p = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[j], 1.f, 2); v[4] = p.x * f; v[5] = p.y * f;
            p = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[j], 1.f, 3); v[6] = p.x * f; v[7] = p.y * f;
            const size_t at = (size_t)(i0 + r) * a.dim + (size_t)c * 8;
            if constexpr (VEC) {
                if constexpr (TYPE == RAG_MX4_F32) {
                    v4f* o = reinterpret_cast<v4f*>(static_cast<float*>(a.out) + at);
                    o[0] = (v4f){v[0], v[1], v[2], v[3]};
                    o[1] = (v4f){v[4], v[5], v[6], v[7]};
                } else {
                    *reinterpret_cast<v4i*>(static_cast<unsigned short*>(a.out) + at) =
                        (v4i){(int)pack16(TYPE, v[0], v[1]), (int)pack16(TYPE, v[2], v[3]), (int)pack16(TYPE, v[4], v[5]),
                              (int)pack16(TYPE, v[6], v[7])};
                }
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    if (c * 8 + i < a.dim) {
                        if constexpr (TYPE == RAG_MX4_F32) static_cast<float*>(a.out)[at + i] = v[i];
                        else static_cast<unsigned short*>(a.out)[at + i] = (unsigned short)pack16(TYPE, v[i], 0.f);
                    }
            }
        }
    }
}

// ------------------------------------------------------------------------------------------------ products
struct Mx4ScoreArgs {
    const uint8_t* codes;        // of the store's first row
    const uint8_t* scales;
    const void* q;
    long long ldq;               // elements
    int q_type, q_vec, dim, ks, ksu, code_ld, scale_ld, normalize;
    size_t code_bytes, scale_bytes;      // of the whole store
    float* out;
    // grouped: one workgroup per item
    const Mx4Item* items;
    // dense: rows [row0, row0 + rows) cut into slabs, every slab against blocks of QB queries
    long long row0, rows, slab, slabs, out_ld;
    long long total;             // grouped: scores in out (and rows = the store's)
    int nq, nqb;
};

// Layout of the instruction (checked on the card): lane l, column c = l / 16.  Four-bit operand: row l % 16, elements
// 32 c .. 32 c + 31 of the block of 128.  Eight-bit operand: row l % 16, bytes 0..15 = elements 16 c .., bytes 16..31 =
// elements 64 + 16 c ..; scale of lane l (either operand): elements 32 c .. 32 c + 31.  Result register r of lane l:
// (eight-bit row 4 c + r, four-bit row l % 16).
//
// Digit j < 4 of query s of a tile is eight-bit row 4 s + j: the four registers of column s, added without leaving the lane.
// Fifth digits (fp32): up to three queries share their tile with them -- rows 12 + s: register s of column 3, fetched from
// there by fifth_digits().  More queries put four to a tile and have the fifth digits of each four tiles in one more tile, query s
// of tile t in row 4 s + t: register t of column s, where they are wanted.
template <int ND, int MT>
struct Mx4Digits {
    static constexpr bool INSIDE = ND == 5 && MT == 1;           // fifth digits in the tile itself
    static constexpr int EX = ND == 5 && !INSIDE ? (MT + 3) / 4 : 0;
    static constexpr int TILES = MT + EX;
    static constexpr int QPT = INSIDE ? 3 : 4;                   // queries per tile of 16 eight-bit rows
};

// queries [q0, q0 + nqh) -> digit fragments in LDS.  frag[(block * TILES + tile) * 2 + half][place of lane][16 bytes], then the scales
// sc[(block / 4) * TILES + tile][lane][block % 4], then 1 / |q|.  Blocks past the row's are zero: they meet a real block of the
// row again.  A lane's place: its row number exclusive-or'ed with column and half, so that the lanes that write one digit of
// consecutive elements meet different banks (with the rows in order sixteen lanes shared four).  What the fragments of absent queries hold does not matter: it stays in result rows that nobody reads.
template <int ND, int MT, int NT>
__device__ __forceinline__ void mx4_stage_queries(const Mx4ScoreArgs& a, long long q0, int nqh, uint8_t* frag, uint8_t* sc, float* inv) {
    typedef Mx4Digits<ND, MT> L;
    constexpr int QPT = L::QPT, TILES = L::TILES;
    const int tid = threadIdx.x;
    if (a.ksu > a.ks) {
        const v4i zero = {0, 0, 0, 0};
        v4i* f = reinterpret_cast<v4i*>(frag + (size_t)a.ks * TILES * 2048);
        for (int i = tid; i < (a.ksu - a.ks) * TILES * 128; i += NT) f[i] = zero;
        v4i* s = reinterpret_cast<v4i*>(sc + (size_t)(a.ks / 4) * TILES * 256);
        for (int i = tid; i < ((a.ksu + 3) / 4 - a.ks / 4) * TILES * 16; i += NT) s[i] = zero;
        __syncthreads();
    }
    const size_t esize = a.q_type == RAG_MX4_F32 ? 4 : 2;
    const char* q = static_cast<const char*>(a.q) + (size_t)q0 * a.ldq * esize;
    for (int s = tid >> 6; s < MT * QPT; s += NT / 64) {
        float f = 1.f;
        if (a.normalize && s < nqh) f = wave_inv_norm(q + (size_t)s * a.ldq * esize, a.q_type, a.dim, tid & 63);
        if ((tid & 63) == 0) inv[s] = f;
    }
    const int upq = a.ks * 32;                                  // units of 4 elements per query
    for (int s = 0, c = tid;; c += NT) {
        while (c >= upq && s < nqh) { c -= upq; ++s; }
        if (s >= nqh) break;
        float v[4];
        mx4_load<4>(q + (size_t)s * a.ldq * esize, a.q_type, c * 4, a.dim, a.q_vec, v);
        unsigned most = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const unsigned m = __float_as_uint(v[j]) & 0x7fffffffu;
            most = m > most ? m : most;
        }
        most = oct_max(most);                                   // eight lanes hold a group of 32
        const bool bad = most >= 0x7f800000u;
        int e = (int)(most >> 23) - 130;                        // the largest element / 2^e lies in [8, 16)
        e = e < -100 ? -100 : e;                                // (a group below 2^-97 has its digits cut instead)
        e = bad ? 0 : e;
        const float down = mx4_pow2(-e);
        const int block = c >> 5, in = c & 31;                  // 4 elements `in` of the block
        const int col = (in >> 2) & 3, half = in >> 4;
        const int tile = s / QPT, slot = s - tile * QPT;
        uint8_t* to = frag + (size_t)(block * TILES * 2 + half) * 1024 + col * 256 + (in & 3) * 4;
        const int turn = col | half << 2;
        uint8_t* ts = sc + (size_t)((block >> 2) * TILES) * 256 + (in >> 3) * 64 + (block & 3);
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] *= down;
#pragma unroll
        for (int d = 0; d < ND; ++d) {
            float w[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                w[j] = rintf(v[j]);
                v[j] = (v[j] - w[j]) * 32.f;                    // both steps exact
            }
            int p = __builtin_amdgcn_cvt_pk_fp8_f32(w[0], w[1], 0, false);
            p = __builtin_amdgcn_cvt_pk_fp8_f32(w[2], w[3], p, true);
            if (bad) p = d == 0 ? 0x7f7f7f7f : 0;               // NaN: every score of the query is NaN
            const int m = d < 4 ? 4 * slot + d : L::INSIDE ? 12 + slot : 4 * slot + (tile & 3);
            const int at = d < 4 || L::INSIDE ? tile : MT + (tile >> 2);
            *reinterpret_cast<int*>(to + at * 2048 + (m ^ turn) * 16) = p;
            if ((in & 7) == 0) ts[at * 256 + m * 4] = (uint8_t)(127 + e - 5 * d);
        }
    }
    __syncthreads();
}

// four values over four columns of lanes, transposed: column c of v_s goes to column s of v_c
__device__ __forceinline__ void columns_transpose(float* v) {
    const v2u a = __builtin_bit_cast(v2u, __builtin_amdgcn_permlane32_swap(__float_as_uint(v[0]), __float_as_uint(v[2]), false, false));
    const v2u b = __builtin_bit_cast(v2u, __builtin_amdgcn_permlane32_swap(__float_as_uint(v[1]), __float_as_uint(v[3]), false, false));
    const v2u c = __builtin_bit_cast(v2u, __builtin_amdgcn_permlane16_swap(a.x, b.x, false, false));
    const v2u d = __builtin_bit_cast(v2u, __builtin_amdgcn_permlane16_swap(a.y, b.y, false, false));
    v[0] = __uint_as_float(c.x);
    v[1] = __uint_as_float(c.y);
    v[2] = __uint_as_float(d.x);
    v[3] = __uint_as_float(d.y);
}
// lanes of column s (0, 1, 2) receive v_s of column 3
__device__ __forceinline__ float fifth_digits(float v0, float v1, float v2) {
    const v2u a = __builtin_bit_cast(v2u, __builtin_amdgcn_permlane32_swap(__float_as_uint(v0), __float_as_uint(v2), false, false));
    const v2u b = __builtin_bit_cast(v2u, __builtin_amdgcn_permlane32_swap(__float_as_uint(v1), __float_as_uint(v1), false, false));
    // a.y: columns 2, 3 of v0, then 2, 3 of v2; b.y: columns 2, 3 of v1, twice
    const v2u r = __builtin_bit_cast(v2u, __builtin_amdgcn_permlane16_swap(a.y, b.y, false, false));
    return __uint_as_float(r.y);                                // the odd columns of both in turn: v0, v1, v2, v1 of column 3
}

// ND digits, MT tiles of queries, NB blocks of 16 rows per wave, U blocks of 128 along the row fetched together, NW waves.
// STEPS 1 or 2: that many fetches are a row; 0: as many as it takes.
//
// A wave takes 16 NB rows at a time and keeps the next U blocks of them in flight while the present ones go through the
// matrix unit; nothing but the query fragments goes through LDS, and there is no barrier after they are staged.  The wave's
// memory operations are the same whatever the data: the fetch ahead is made past the last rows too (of the last ones again), and
// lanes without a score to store address nothing behind a buffer descriptor's end.  Behind a branch the compiler would have to
// wait for all of them at every turn, stores too (256 fp32 queries x 200k x 768: 160 us with branches around the stores, 156 without).
//
// BIG, for stores larger than the caches: rows are fetched past them (4M x 768, one query: 299 -> 264 us), and where up to 8
// queries meet a row a wave takes four tiles of sixteen rows in a row and stores their scores together, 256 contiguous bytes
// per query instead of 64 (264 -> 255).
//
// Where it stands.  Few queries: bound by HBM.  4M x 768, one query: 255 us, 6.6 TB/s of rows, scales and scores; reading the same
// rows alone takes 220 us (7.0 TB/s), and with one 256-byte store per 24 KB 236 to 247.  16 bf16 queries x 1M x 1024: 113 us, 5.4 TB/s
// (100 without the stores).  Many queries: bound by the matrix unit and the LDS that feeds it (a tile's fragments serve NB row blocks):
// 256 fp32 queries x 200k x 768: 156 us, 2.5e15 eight-bit operations a second, against 2.8e15 of a large library product of eight-bit matrices.
template <int ND, int MT, int NB, int U, int NW, int STEPS, bool BIG>
__global__ __launch_bounds__(NW * 64) void mx4_scores_kernel(Mx4ScoreArgs a) {
    typedef Mx4Digits<ND, MT> L;
    constexpr int QPT = L::QPT, TILES = L::TILES, QB = MT * QPT;
    constexpr bool LONG = BIG && MT <= 2;
    static_assert(!LONG || NB == 1, "four tiles of one row block each are stored together");
    const int ks = STEPS ? STEPS * U : a.ks, ksu = STEPS ? STEPS * U : a.ksu;
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    uint8_t* frag = smem;
    uint8_t* sc = frag + (size_t)ksu * TILES * 2048;
    float* inv = reinterpret_cast<float*>(sc + (size_t)((ksu + 3) / 4) * TILES * 256);

    // rows [row0, row0 + rows) against queries [q0, q0 + nqh); this wave takes the tiles of 16 NB rows first, first + stride, ...
    // (LONG: four from each)
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    long long row0, at, ld;
    int rows, q0, nqh, first = wave, stride = NW;
    if (a.items) {
        const Mx4Item it = a.items[blockIdx.x];
        row0 = it.row0; at = it.at; ld = it.ld; rows = it.rows; q0 = it.q0; nqh = it.nq;
        // a piece that was not made for this store, these queries or this result is left out
        if (rows < 1 || row0 < 0 || row0 > a.rows - rows || nqh < 1 || nqh > QB || q0 < 0 || q0 > a.nq - nqh || ld < rows || at < 0 ||
            at > a.total - (long long)(nqh - 1) * ld - rows)
            return;
    } else if (a.nqb == 1) {
        row0 = a.row0; at = 0; ld = a.out_ld; rows = (int)a.rows; q0 = 0; nqh = a.nq;
        first = (int)blockIdx.x * NW + wave;
        stride = (int)gridDim.x * NW;
    } else {
        // workgroups go to the eight dies in turn: each die takes a contiguous part of the (slab, query block) pairs, so the
        // query blocks of a slab stay on one die, whose L2 then holds the slab's rows for all of them
        const long long pairs = a.slabs * a.nqb, id = (blockIdx.x & 7) * ((pairs + 7) >> 3) + (blockIdx.x >> 3);
        if (id >= pairs || (blockIdx.x >> 3) >= (pairs + 7) >> 3) return;
        const long long s = id / a.nqb;
        const int qb = (int)(id % a.nqb);
        const long long lo = s * a.slab;
        rows = (int)(a.rows - lo < a.slab ? a.rows - lo : a.slab);
        q0 = qb * QB;
        nqh = a.nq - q0 < QB ? a.nq - q0 : QB;
        row0 = a.row0 + lo;
        at = (long long)q0 * a.out_ld + lo;
        ld = a.out_ld;
    }
    if (LONG) first *= 4;
    const int n16 = lane & 15, col = lane >> 4;
    const int tiles = rows / (16 * NB) + (rows % (16 * NB) != 0);
    const int end = LONG ? (tiles + 3) & ~3 : tiles;
    const int sd = (ks + 3) / 4;                                // scale dwords of a lane per row
    float* out = a.out + at;

    constexpr int SW = (U + 3) / 4 + (STEPS == 2 && U % 4 ? 1 : 0);     // scale dwords per fetch
    struct Buf {
        v4i w[NB][U];
        int s[NB][SW];
    };
    // Rows are fetched through buffer descriptors that end with the store: rows past the last one of a piece are fetched and
    // never stored, what would lie behind the store comes back as zeros.  (The check is lane offset >= size - uniform offset: the
    // uniform part, a block or scale dword of the tile's first row, always lies inside the store.)
    const int l0 = (int)(row0 & 15) + n16;                      // tiles start at multiples of 16 from row0
    const int wo = (l0 >> 4) * 16 * a.code_ld + (l0 & 15) * 64 + col * 16, so = n16 * a.scale_ld + col * 4;
    constexpr int AUX = BIG ? 2 : 0;                            // 2: not to be kept in the caches
    auto load = [&](Buf& b, int tile, auto ks0c) {              // ks0c: a constant where STEPS is 1 or 2
        const int ks0 = ks0c;
        tile = tile < tiles ? tile : tiles - 1;
        const long long r0 = row0 + (long long)tile * (16 * NB);
        const size_t wat = (size_t)(r0 >> 4) * 16 * a.code_ld, sat = (size_t)r0 * a.scale_ld;
        const size_t wleft = a.code_bytes - wat, sleft = a.scale_bytes - sat;
        const auto wr = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(a.codes) + wat, 0, (int)(wleft < 0x7fffffffu ? wleft : 0x7fffffffu), 0x00027000);
        const auto sr = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(a.scales) + sat, 0, (int)(sleft < 0x7fffffffu ? sleft : 0x7fffffffu), 0x00027000);
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int k = STEPS || ks0 + u < ks ? ks0 + u : ks - 1;          // blocks past the row's meet zero digits
                b.w[nb][u] = __builtin_bit_cast(v4i, __builtin_amdgcn_raw_buffer_load_b128(wr, wo + nb * 16 * a.code_ld, k * 1024, AUX));
            }
#pragma unroll
            for (int d = 0; d < SW; ++d) {
                const int k = (ks0 >> 2) + d < sd ? (ks0 >> 2) + d : sd - 1;
                b.s[nb][d] = (int)__builtin_amdgcn_raw_buffer_load_b32(sr, so + nb * 16 * a.scale_ld, k * 16, 0);
            }
        }
    };
    v4f acc[TILES][NB];
    auto multiply = [&](const Buf& b, auto ks0c, auto first_of_row) {
        const int ks0 = ks0c;
        constexpr bool FIRST = decltype(first_of_row)::value;   // begins the sums at zero
        constexpr bool SHIFT = STEPS == 0 && U < 4;             // the fetch may begin inside a scale dword
        constexpr int K0 = [] { if constexpr (STEPS) return decltype(ks0c)::value; else return 0; }();
        const uint8_t* f = frag + (size_t)ks0 * TILES * 2048;
        int fl = (col * 16 + (n16 ^ col)) * 16, sl = lane * 4;  // places of the first half; the second half's differ in bit 2 of the row
        if constexpr (TILES > 1) asm volatile("" : "+v"(fl), "+v"(sl));      // more than one tile's fragments do not fit the registers: read from LDS each time
        // query fragments AHEAD tiles ahead: the LDS latency passes under the products of the tiles before
        constexpr int AHEAD = 2, RING = AHEAD + 1;
        v4i lo[RING], hi[RING];
        int xs[RING];
        auto fetch = [&](auto ic) {
            constexpr int i = decltype(ic)::value, u = i / TILES, mt = i % TILES;
            lo[i % RING] = *reinterpret_cast<const v4i*>(f + i * 2048 + fl);
            hi[i % RING] = *reinterpret_cast<const v4i*>(f + i * 2048 + 1024 + (fl ^ 64));
            const int x = *reinterpret_cast<const int*>(sc + (size_t)(((ks0 + (SHIFT ? 0 : u)) >> 2) * TILES + mt) * 256 + sl);
            xs[i % RING] = SHIFT ? (int)((unsigned)x >> ((ks0 & 3) * 8)) : x;
        };
        int ys[NB][SW];
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
            for (int d = 0; d < SW; ++d) ys[nb][d] = SHIFT ? (int)((unsigned)b.s[nb][d] >> ((ks0 & 3) * 8)) : b.s[nb][d];
        static_for<AHEAD>([&](auto ic) {
            if constexpr (decltype(ic)::value < U * TILES) fetch(ic);
        });
        static_for<U * TILES>([&](auto ic) {
            constexpr int i = decltype(ic)::value, u = i / TILES, mt = i % TILES;
            constexpr int kk = K0 + u;                          // (K0 is a multiple of 4, or shifted away, where STEPS is 0)
            if constexpr (i + AHEAD < U * TILES) fetch(std::integral_constant<int, i + AHEAD>{});
            if constexpr (TILES > 1) __builtin_amdgcn_sched_barrier(0);
            const v8i x = __builtin_shufflevector(lo[i % RING], hi[i % RING], 0, 1, 2, 3, 4, 5, 6, 7);
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) {
                const v8i y = __builtin_shufflevector(b.w[nb][u], b.w[nb][u], 0, 1, 2, 3, -1, -1, -1, -1);
                const v4f c = FIRST && u == 0 ? (v4f){0.f, 0.f, 0.f, 0.f} : acc[mt][nb];
                acc[mt][nb] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(x, y, c, 0, 4, kk & 3, xs[i % RING], kk & 3,
                                                                               ys[nb][(kk >> 2) - (K0 >> 2)]);
            }
        });
    };
    float iv[MT];
    unsigned place[MT];                                         // of this lane's score from the tile's first one; past the end where there is none
    constexpr unsigned NOWHERE = 0x80000000u;
    float held[MT][4];                                          // LONG: the scores of the tiles since the last store
    auto total = [&](int mt, int nb) -> float {
        // column c of lanes holds query c of the tile; the order of the additions is the same for every query, so a score does
        // not depend on what it is computed together with
        const v4f v = acc[mt][nb];
        float y = (v[0] + v[1]) + (v[2] + v[3]);
        if constexpr (L::INSIDE) y += fifth_digits(v[0], v[1], v[2]);
        else if constexpr (ND == 5) y += acc[MT + mt / 4][nb][mt & 3];
        y *= iv[mt];
        if constexpr (STEPS == 0) asm volatile("" : "+v"(y));   // here: else the products sink into the branch that asks whether a row is done
        return y;
    };
    auto put = [&](float v, float* base, int bytes, unsigned offset) {
        __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(v), __builtin_amdgcn_make_buffer_rsrc(base, 0, bytes, 0x00027000), offset, 0, 0);
    };
    auto store = [&](int tile) {
        if constexpr (LONG) {
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
                columns_transpose(held[mt]);
                const int r = (tile - 3) * 16, left = (rows - r) * 4 < 256 && rows - r < 64 ? (rows - r) * 4 : 256;
#pragma unroll
                for (int s = 0; s < QPT; ++s)
                    put(held[mt][s], out + (mt * QPT + s) * ld + r, mt * QPT + s < nqh ? left : 0, lane * 4);
            }
        } else {
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) {
                const int r = (tile * NB + nb) * 16;
                const bool there = r + n16 < rows;
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) put(total(mt, nb), out + mt * QPT * ld + r, 0x7fffffff, there ? place[mt] : NOWHERE);
            }
        }
    };

    Buf x, y;
    typedef std::integral_constant<int, 0> Zero;
    typedef std::integral_constant<int, U> Half;
    int t = first;
    if constexpr (STEPS) load(x, t, Zero{});                    // on its way while the queries are split
    else load(x, t, 0);
    mx4_stage_queries<ND, MT, NW * 64>(a, q0, nqh, frag, sc, inv);
    if (first >= end) return;
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
        iv[mt] = inv[col < QPT ? mt * QPT + col : 0];
        place[mt] = col < QPT && mt * QPT + col < nqh ? (unsigned)(col * ld + n16) * 4u : NOWHERE;
    }
    auto hold = [&](auto sub) {
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) held[mt][decltype(sub)::value] = total(mt, 0);
    };
    if constexpr (STEPS == 1) {
        // pairs of tiles: x and y in turn (LONG: two pairs to a store)
        for (;;) {
            static_for<LONG ? 2 : 1>([&](auto pair) {
                constexpr int p = decltype(pair)::value * 2;
                const int t1 = LONG ? t + p + 1 : t + stride;
                const int t2 = LONG ? (p == 0 ? t + 2 : t + 4 * stride) : t + 2 * stride;
                load(y, t1, Zero{});
                __builtin_amdgcn_sched_barrier(0);              // the fetch goes out before the products wait for theirs
                multiply(x, Zero{}, std::true_type{});
                if constexpr (LONG) hold(std::integral_constant<int, p>{});
                else store(t);
                if (!LONG && t1 >= end) return;
                load(x, t2, Zero{});
                __builtin_amdgcn_sched_barrier(0);
                multiply(y, Zero{}, std::true_type{});
                if constexpr (LONG) hold(std::integral_constant<int, p + 1>{});
                else store(t1);
            });
            if constexpr (LONG) store(t + 3);
            t += LONG ? 4 * stride : 2 * stride;
            if (t >= end) break;
        }
    } else if constexpr (STEPS == 2 && !LONG) {
        for (;;) {
            load(y, t, Half{});
            __builtin_amdgcn_sched_barrier(0);
            multiply(x, Zero{}, std::true_type{});
            load(x, t + stride, Zero{});
            __builtin_amdgcn_sched_barrier(0);
            multiply(y, Half{}, std::false_type{});
            store(t);
            t += stride;
            if (t >= end) break;
        }
    } else {
        int k = 0;
        auto piece = [&](const Buf& b, int ks0) {
            if (ks0 == 0) multiply(b, ks0, std::true_type{});
            else multiply(b, ks0, std::false_type{});
        };
        // where the piece behind this one lies
        auto next = [&](int& t2, int& k2) {
            k2 += U;
            if (k2 < ksu) return;
            k2 = 0;
            t2 += !LONG ? stride : (t2 & 3) != 3 ? 1 : 4 * stride - 3;
        };
        auto done = [&](int tile) {
            if constexpr (LONG) {
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) {
                    held[mt][0] = held[mt][1];
                    held[mt][1] = held[mt][2];
                    held[mt][2] = held[mt][3];
                    held[mt][3] = total(mt, 0);
                }
                if ((tile & 3) != 3) return;
            }
            store(tile);
        };
        for (;;) {
            int t2 = t, k2 = k;
            next(t2, k2);
            load(y, t2, k2);
            __builtin_amdgcn_sched_barrier(0);
            piece(x, k);
            if (k2 == 0) done(t);
            if (t2 >= end) break;
            t = t2;
            k = k2;
            next(t, k);
            load(x, t, k);
            __builtin_amdgcn_sched_barrier(0);
            piece(y, k2);
            if (k == 0) done(t2);
            if (t >= end) break;
        }
    }
}

// Which kernel a product takes: from the queries that meet a row, and the row's length.
struct Mx4Shape {
    int nd, mt, nb, u, nw, steps, ksu, qb;
    bool big;
    size_t lds;
};
static int mx4_tiles(int nd, int mt) { return nd == 5 && mt > 1 ? mt + (mt + 3) / 4 : mt; }        // Mx4Digits::TILES
static size_t mx4_lds(int ks, int u, int tiles) {
    const int ksu = (ks + u - 1) / u * u;
    return (size_t)ksu * tiles * 2048 + (size_t)(ksu + 3) / 4 * tiles * 256 + (size_t)tiles * 4 * sizeof(float);
}
// wide: the scores of two queries may lie further apart than a lane's 32-bit offset reaches (LONG kernels have none)
static Mx4Shape mx4_shape(int type, int dim, long long nq, bool wide) {
    Mx4Shape p = {};
    const int ks = mx4_blocks(dim);
    p.nd = type == RAG_MX4_F32 ? 5 : 4;
    // rows of up to 8 blocks: one fetch, or two of half the row where more tiles need the registers
    auto fetch = [&](int mt, int* steps) {
        *steps = mt <= 2 ? ks <= 8 : ks <= 3 ? 1 : ks == 4 || ks == 6 || ks == 8 ? 2 : 0;
        if (mt == 8 && ks == 8) *steps = 0;
        if (*steps) return ks / *steps;
        if (mt <= 2) return (ks & 7) == 0 || (ks & 7) > 4 ? 8 : 4;
        return mt == 4 && (ks & 3) == 0 ? 4 : (ks & 1) == 0 ? 2 : 1;
    };
    p.mt = nq <= (p.nd == 5 ? 3 : 4) ? 1 : nq <= 8 ? 2 : nq <= 16 ? 4 : 8;
    if (wide) p.mt = std::min(p.mt, 2);
    while (p.mt > 1 && mx4_lds(ks, fetch(p.mt, &p.steps), mx4_tiles(p.nd, p.mt)) > 160 * 1024) p.mt /= 2;
    p.u = fetch(p.mt, &p.steps);
    p.big = wide;
    p.nb = p.mt <= 4 ? 1 : 2;
    p.nw = p.mt >= 4 ? 8 : 4;
    p.ksu = (ks + p.u - 1) / p.u * p.u;
    p.qb = p.nd == 5 && p.mt == 1 ? 3 : 4 * p.mt;
    p.lds = mx4_lds(ks, p.u, mx4_tiles(p.nd, p.mt));
    return p;
}
constexpr long long MX4_WIDE = 100 * 1000 * 1000;        // 3 * 4 bytes * this, and a tile, stay below 2^31

template <int ND, int MT, int NB, int U, int NW, int STEPS, bool BIG>
static int mx4_launch(const Mx4ScoreArgs& a, long long grid, size_t lds, int device, hipStream_t s) {
    static bool attr_set[64] = {};          // per device: the attribute belongs to the device's code object
    auto kern = mx4_scores_kernel<ND, MT, NB, U, NW, STEPS, BIG>;
    if (lds > 48 * 1024 && !attr_set[device & 63]) {
        RAG_HIP_CHECK(hipFuncSetAttribute(reinterpret_cast<const void*>(kern), hipFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024));
        attr_set[device & 63] = true;
    }
    hipLaunchKernelGGL(kern, dim3((unsigned)grid), dim3(NW * 64), lds, s, a);
    RAG_HIP_CHECK(hipGetLastError());
    return RAG_OK;
}
template <int ND>
static int mx4_launch_nd(const Mx4Shape& p, const Mx4ScoreArgs& a, long long grid, int device, hipStream_t s) {
#define MX4_CASE(MT, NB, U, NW, STEPS) \
    if (p.mt == MT && p.u == U && p.steps == STEPS) \
        return p.big ? mx4_launch<ND, MT, NB, U, NW, STEPS, true>(a, grid, p.lds, device, s) : mx4_launch<ND, MT, NB, U, NW, STEPS, false>(a, grid, p.lds, device, s)
#define MX4_FEW(MT) \
    MX4_CASE(MT, 1, 1, 4, 1); MX4_CASE(MT, 1, 2, 4, 1); MX4_CASE(MT, 1, 3, 4, 1); MX4_CASE(MT, 1, 4, 4, 1); MX4_CASE(MT, 1, 5, 4, 1); \
    MX4_CASE(MT, 1, 6, 4, 1); MX4_CASE(MT, 1, 7, 4, 1); MX4_CASE(MT, 1, 8, 4, 1); MX4_CASE(MT, 1, 4, 4, 0); MX4_CASE(MT, 1, 8, 4, 0)
    MX4_FEW(1);
    MX4_FEW(2);
    MX4_CASE(4, 1, 1, 8, 1); MX4_CASE(4, 1, 2, 8, 1); MX4_CASE(4, 1, 3, 8, 1); MX4_CASE(4, 1, 2, 8, 2); MX4_CASE(4, 1, 3, 8, 2); MX4_CASE(4, 1, 4, 8, 2);
    MX4_CASE(4, 1, 1, 8, 0); MX4_CASE(4, 1, 2, 8, 0); MX4_CASE(4, 1, 4, 8, 0);
    MX4_CASE(8, 2, 1, 8, 1); MX4_CASE(8, 2, 2, 8, 1); MX4_CASE(8, 2, 3, 8, 1); MX4_CASE(8, 2, 2, 8, 2); MX4_CASE(8, 2, 3, 8, 2);
    MX4_CASE(8, 2, 1, 8, 0); MX4_CASE(8, 2, 2, 8, 0);
#undef MX4_FEW
#undef MX4_CASE
    return fail(RAG_ERR_INVALID, "internal: no four-bit product kernel for this shape");
}
static int mx4_launch_any(const Mx4Shape& p, const Mx4ScoreArgs& a, long long grid, int device, hipStream_t s) {
    if (grid < 1 || grid > 0x7fffffffLL) return fail(RAG_ERR_INVALID, "four-bit product: grid out of range");
    return p.nd == 5 ? mx4_launch_nd<5>(p, a, grid, device, s) : mx4_launch_nd<4>(p, a, grid, device, s);
}

static int mx4_check_store(const rag_mx4_store_t* st) {
    if (!st) return fail(RAG_ERR_INVALID, "store is NULL");
    if (st->dim < 1 || st->dim > MX4_MAX_DIM) return fail(RAG_ERR_INVALID, "dim must be in [1, " + std::to_string(MX4_MAX_DIM) + "]");
    if (st->n < 0 || st->n > 0x7fffffffLL) return fail(RAG_ERR_INVALID, "a store holds 0 to 2^31 - 1 rows");
    if (st->n > 0 && (!st->codes || !st->scales)) return fail(RAG_ERR_INVALID, "store without buffers");
    if ((reinterpret_cast<uintptr_t>(st->codes) & 15) || (reinterpret_cast<uintptr_t>(st->scales) & 15))
        return fail(RAG_ERR_INVALID, "the store's buffers must lie on 16-byte boundaries");
    return RAG_OK;
}
static int mx4_check_type(int type) {
    if (type != RAG_MX4_F32 && type != RAG_MX4_BF16 && type != RAG_MX4_F16) return fail(RAG_ERR_INVALID, "unknown element type");
    return RAG_OK;
}
static size_t mx4_esize(int type) { return type == RAG_MX4_F32 ? 4 : 2; }
static int mx4_aligned(const void* p, long long ld, int type) {
    return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && (size_t)ld * mx4_esize(type) % 16 == 0;
}
// rows of a workgroup that writes or reads rows: four units a thread, fewer where that would leave compute units without work
static int mx4_rows_per_block(long long count, int upr) {
    const long long full = std::max(1, std::min(MX4_ROWS, 256 * MX4_UNITS / upr));
    return (int)std::max<long long>(1, std::min<long long>(full, count / 512));
}
static Mx4ScoreArgs mx4_score_args(const rag_mx4_store_t* st, const Mx4Shape& p, const void* q, int q_type, long long ldq, int normalize, float* out) {
    Mx4ScoreArgs a = {};
    a.codes = static_cast<const uint8_t*>(st->codes);
    a.scales = static_cast<const uint8_t*>(st->scales);
    a.q = q;
    a.ldq = ldq;
    a.q_type = q_type;
    a.q_vec = mx4_aligned(q, ldq, q_type);
    a.dim = st->dim;
    a.ks = mx4_blocks(st->dim);
    a.ksu = p.ksu;
    a.code_ld = mx4_code_bytes(st->dim);
    a.scale_ld = mx4_scale_bytes(st->dim);
    a.code_bytes = (size_t)((st->n + 15) / 16 * 16) * a.code_ld;
    a.scale_bytes = (size_t)st->n * a.scale_ld;
    a.normalize = normalize;
    a.out = out;
    return a;
}

// scores of rows [row0, row0 + rows) (checked by the caller)
static int mx4_scores(const rag_mx4_store_t* st, long long row0, long long rows, long long nq, const void* q, int q_type, long long ldq,
                      int normalize, float* out, long long out_ld, hipStream_t s) {
    Mx4Shape p = mx4_shape(q_type, st->dim, nq, out_ld > MX4_WIDE);
    Mx4ScoreArgs a = mx4_score_args(st, p, q, q_type, ldq, normalize, out);
    p.big = p.big || (nq <= p.qb && rows * a.code_ld > 64LL << 20);
    a.row0 = row0;
    a.rows = rows;
    a.out_ld = out_ld;
    a.nq = (int)nq;
    a.nqb = (int)((nq + p.qb - 1) / p.qb);
    const long long unit = 16LL * p.nb * p.nw;                  // rows of one step of a workgroup
    const long long units = (rows + unit - 1) / unit;
    if (a.nqb == 1) return mx4_launch_any(p, a, std::min<long long>(units, p.mt == 8 ? 256 : p.mt == 4 ? 512 : 1024), st->device, s);
    // Slabs: as many as make the workgroups come out even over the chip's compute units, each long against the staging of
    // its queries (about two units of work)
    const long long seats = 256LL * (p.mt == 8 ? 1 : 2);
    long long best = 1, least = LLONG_MAX;
    for (long long n = 1; n <= std::min<long long>(units, std::max<long long>(64, 8 * seats / a.nqb)); ++n) {
        const long long cost = (n * a.nqb + seats - 1) / seats * ((units + n - 1) / n + 2);
        if (cost < least) { least = cost; best = n; }
    }
    a.slab = (units + best - 1) / best * unit;
    a.slabs = (rows + a.slab - 1) / a.slab;
    return mx4_launch_any(p, a, (a.slabs * a.nqb + 7) / 8 * 8, st->device, s);
}

int direct_select_segments(long long nq, long long n_row, long long seg_rows, int k, float min_score, const uint8_t* mask,
                           const long long* row_ids, long long id_base, const float* scores, float* D, long long* I, long long out_stride,
                           const float* floor, long long floor_stride, hipStream_t s);   // direct_topk.hip
int merge_lists_device(int nlists, long long nq, int k, const float* D_dev, long long d_list_stride, const long long* I_dev,
                       long long i_list_stride, float* D_out, long long* I_out, u64* keys, hipStream_t s);      // api.hip
void launch_fill_results(float* D, long long* I, long long n, hipStream_t s);                // api.hip

__global__ void mx4_copy_lists_kernel(const float* D, const long long* I, long long n, float* Dto, long long* Ito) {
    for (long long i = blockIdx.x * (long long)blockDim.x + threadIdx.x; i < n; i += (long long)gridDim.x * blockDim.x) {
        Dto[i] = D[i];
        Ito[i] = I[i];
    }
}

__global__ void mx4_and_masks_kernel(const uint8_t* a, const uint8_t* b, long long n, uint8_t* out) {
    for (long long i = blockIdx.x * (long long)blockDim.x + threadIdx.x; i < n; i += (long long)gridDim.x * blockDim.x)
        out[i] = (a[i] != 0 && b[i] != 0) ? 1 : 0;
}

// A search walks the rows in spans whose scores fit 256 MiB: score matrix, the k best of every 32768 rows, merge.
constexpr long long MX4_SEG = 32768;
struct Mx4Plan {
    long long qc, span;          // queries and rows of one step
    size_t scores, d, i, keys, mask;     // bytes of the workspace's parts
    size_t total() const { return scores + d + i + keys + mask; }
};
static Mx4Plan mx4_plan(long long n, long long nq, int k) {
    Mx4Plan p;
    const long long segs = std::max<long long>(1, (n + MX4_SEG - 1) / MX4_SEG);
    p.qc = std::min<long long>(std::max<long long>(nq, 1), 512);
    p.span = std::max<long long>(1, std::min<long long>(std::min<long long>(segs, 256), (256LL << 20) / (p.qc * MX4_SEG * 4)));
    // the merge reads (span + 1) lists of k keys per query
    while (p.span > 1 && (p.span + 1) * p.qc * k > (16LL << 20)) p.span /= 2;
    auto al = [](size_t b) { return (b + 255) & ~(size_t)255; };
    p.scores = al((size_t)p.qc * std::min<long long>(std::max<long long>(n, 1), p.span * MX4_SEG) * sizeof(float));
    p.d = al((size_t)(p.span + 1) * p.qc * k * sizeof(float));
    p.i = al((size_t)(p.span + 1) * p.qc * k * sizeof(long long));
    p.keys = al((size_t)(p.span + 1) * p.qc * k * sizeof(u64));
    p.mask = al((size_t)std::max<long long>(n, 1));
    return p;
}

}  // namespace rag

using namespace rag;

extern "C" {

int rag_mx4_layout(int dim, int64_t* code_bytes, int64_t* scale_bytes) {
    if (dim < 1 || dim > MX4_MAX_DIM) return fail(RAG_ERR_INVALID, "dim must be in [1, " + std::to_string(MX4_MAX_DIM) + "]");
    if (!code_bytes || !scale_bytes) return fail(RAG_ERR_INVALID, "NULL output");
    *code_bytes = mx4_code_bytes(dim);
    *scale_bytes = mx4_scale_bytes(dim);
    return RAG_OK;
}

int rag_mx4_write_device(const rag_mx4_store_t* st, int64_t first, const int64_t* rows_dev, int32_t* owner_dev, int64_t count,
                         const void* x_dev, int x_type, int64_t x_stride, int normalize, void* stream) {
    if (int rc = mx4_check_store(st)) return rc;
    if (int rc = mx4_check_type(x_type)) return rc;
    if (count < 0 || count >= 0x7fffffffLL) return fail(RAG_ERR_INVALID, "count out of range");
    if (count == 0) return RAG_OK;
    if (!x_dev) return fail(RAG_ERR_INVALID, "NULL buffer");
    if (x_stride < st->dim) return fail(RAG_ERR_INVALID, "x_stride smaller than dim");
    if ((reinterpret_cast<uintptr_t>(x_dev) & (mx4_esize(x_type) - 1))) return fail(RAG_ERR_INVALID, "x is not aligned to its elements");
    if (rows_dev) {
        if (!owner_dev) return fail(RAG_ERR_INVALID, "positions need the store's owner array");
        if (st->n == 0) return RAG_OK;                  // every position lies outside
    } else if (first < 0 || first > st->n || count > st->n - first) {
        return fail(RAG_ERR_INVALID, "rows [first, first + count) do not lie inside the store");
    }
    Mx4DeviceGuard g(st->device);
    if (!g.ok) return fail(RAG_ERR_HIP, "hipSetDevice failed");
    hipStream_t s = static_cast<hipStream_t>(stream);
    Mx4WriteArgs a = {};
    a.codes = static_cast<uint8_t*>(st->codes);
    a.scales = static_cast<uint8_t*>(st->scales);
    a.n = st->n;
    a.rows = reinterpret_cast<const long long*>(rows_dev);
    a.first = first;
    a.count = count;
    a.x = x_dev;
    a.ldx = x_stride;
    a.dim = st->dim;
    a.code_ld = mx4_code_bytes(st->dim);
    a.scale_ld = mx4_scale_bytes(st->dim);
    a.normalize = normalize ? 1 : 0;
    a.upr = mx4_blocks(st->dim) * 16;
    a.per = (unsigned)((0x100000000ull + a.upr - 1) / a.upr);
    a.per_block = mx4_rows_per_block(count, a.upr);
    if (rows_dev && count > MX4_FEW) {
        hipLaunchKernelGGL(mx4_claim_kernel, dim3((unsigned)((count + 255) / 256)), dim3(256), 0, s, a.rows, (long long)count, a.n, owner_dev);
        RAG_HIP_CHECK(hipGetLastError());
        a.owner = owner_dev;
    }
    const dim3 grid((unsigned)((count + a.per_block - 1) / a.per_block));
    const int vec = mx4_aligned(x_dev, x_stride, x_type);
#define MX4_WRITE(T) \
    if (x_type == T) { \
        if (rows_dev && vec) hipLaunchKernelGGL((mx4_write_kernel<T, true, true>), grid, dim3(256), 0, s, a); \
        else if (rows_dev) hipLaunchKernelGGL((mx4_write_kernel<T, false, true>), grid, dim3(256), 0, s, a); \
        else if (vec) hipLaunchKernelGGL((mx4_write_kernel<T, true, false>), grid, dim3(256), 0, s, a); \
        else hipLaunchKernelGGL((mx4_write_kernel<T, false, false>), grid, dim3(256), 0, s, a); \
    }
    MX4_WRITE(RAG_MX4_F32) MX4_WRITE(RAG_MX4_BF16) MX4_WRITE(RAG_MX4_F16)
#undef MX4_WRITE
    RAG_HIP_CHECK(hipGetLastError());
    return RAG_OK;
}

int rag_mx4_read_device(const rag_mx4_store_t* st, const int64_t* rows_dev, int64_t count, void* out_dev, int out_type, void* stream) {
    if (int rc = mx4_check_store(st)) return rc;
    if (int rc = mx4_check_type(out_type)) return rc;
    if (count < 0 || count >= 0x7fffffffLL) return fail(RAG_ERR_INVALID, "count out of range");
    if (count == 0) return RAG_OK;
    if (!rows_dev || !out_dev) return fail(RAG_ERR_INVALID, "NULL buffer");
    if ((reinterpret_cast<uintptr_t>(out_dev) & (mx4_esize(out_type) - 1))) return fail(RAG_ERR_INVALID, "out is not aligned to its elements");
    Mx4DeviceGuard g(st->device);
    if (!g.ok) return fail(RAG_ERR_HIP, "hipSetDevice failed");
    Mx4ReadArgs a = {};
    a.codes = static_cast<const uint8_t*>(st->codes);
    a.scales = static_cast<const uint8_t*>(st->scales);
    a.n = st->n;
    a.rows = reinterpret_cast<const long long*>(rows_dev);
    a.count = count;
    a.out = out_dev;
    a.dim = st->dim;
    a.code_ld = mx4_code_bytes(st->dim);
    a.scale_ld = mx4_scale_bytes(st->dim);
    a.upr = (st->dim + 7) / 8;
    a.per = (unsigned)((0x100000000ull + a.upr - 1) / a.upr);
    a.per_block = mx4_rows_per_block(count, a.upr);
    const dim3 grid((unsigned)((count + a.per_block - 1) / a.per_block));
    const int vec = st->dim % 8 == 0 && mx4_aligned(out_dev, st->dim, out_type);
    hipStream_t s = static_cast<hipStream_t>(stream);
#define MX4_READ(T) \
    if (out_type == T) { \
        if (vec) hipLaunchKernelGGL((mx4_read_kernel<T, true>), grid, dim3(256), 0, s, a); \
        else hipLaunchKernelGGL((mx4_read_kernel<T, false>), grid, dim3(256), 0, s, a); \
    }
    MX4_READ(RAG_MX4_F32) MX4_READ(RAG_MX4_BF16) MX4_READ(RAG_MX4_F16)
#undef MX4_READ
    RAG_HIP_CHECK(hipGetLastError());
    return RAG_OK;
}

static int mx4_check_queries(const rag_mx4_store_t* st, int64_t nq, const void* q_dev, int q_type, int64_t q_stride) {
    if (int rc = mx4_check_store(st)) return rc;
    if (int rc = mx4_check_type(q_type)) return rc;
    if (nq < 0 || nq > 0x7fffffffLL) return fail(RAG_ERR_INVALID, "nq out of range");
    if (nq > 0 && !q_dev) return fail(RAG_ERR_INVALID, "NULL buffer");
    if (nq > 0 && q_stride < st->dim) return fail(RAG_ERR_INVALID, "q_stride smaller than dim");
    if ((reinterpret_cast<uintptr_t>(q_dev) & (mx4_esize(q_type) - 1))) return fail(RAG_ERR_INVALID, "q is not aligned to its elements");
    return RAG_OK;
}

int rag_mx4_scores_device(const rag_mx4_store_t* st, int64_t row_begin, int64_t row_end, int64_t nq, const void* q_dev, int q_type,
                          int64_t q_stride, int normalize, float* out_dev, int64_t out_stride, void* stream) {
    if (int rc = mx4_check_queries(st, nq, q_dev, q_type, q_stride)) return rc;
    if (row_begin < 0 || row_end < row_begin || row_end > st->n) return fail(RAG_ERR_INVALID, "rows [row_begin, row_end) do not lie inside the store");
    const long long rows = row_end - row_begin;
    if (nq == 0 || rows == 0) return RAG_OK;
    if (!out_dev) return fail(RAG_ERR_INVALID, "NULL buffer");
    if (out_stride < rows) return fail(RAG_ERR_INVALID, "out_stride smaller than the number of rows");
    Mx4DeviceGuard g(st->device);
    if (!g.ok) return fail(RAG_ERR_HIP, "hipSetDevice failed");
    return mx4_scores(st, row_begin, rows, nq, q_dev, q_type, q_stride, normalize ? 1 : 0, out_dev, out_stride, static_cast<hipStream_t>(stream));
}

int rag_mx4_plan_groups(int dim, int q_type, int64_t nq, int64_t n, int64_t ngroups, const int64_t* groups, int64_t max_items,
                        void* items_out, int64_t* n_items, int64_t* out_begin, int64_t* total, int32_t* widest) {
    if (dim < 1 || dim > MX4_MAX_DIM) return fail(RAG_ERR_INVALID, "dim must be in [1, " + std::to_string(MX4_MAX_DIM) + "]");
    if (int rc = mx4_check_type(q_type)) return rc;
    if (ngroups < 0 || nq < 0 || nq > 0x7fffffffLL || n < 0 || n > 0x7fffffffLL || max_items < 0) return fail(RAG_ERR_INVALID, "size out of range");
    if ((ngroups > 0 && !groups) || !n_items || !total || !widest || (max_items > 0 && !items_out)) return fail(RAG_ERR_INVALID, "NULL buffer");
    long long most_q = 0, sum = 0;
    __int128 pairs = 0;
    for (long long g = 0; g < ngroups; ++g) {
        const int64_t* d = groups + 4 * g;
        if (d[0] < 0 || d[1] < d[0] || d[1] > nq) return fail(RAG_ERR_INVALID, "group " + std::to_string(g) + ": queries do not lie inside [0, nq)");
        if (d[2] < 0 || d[3] < d[2] || d[3] > n) return fail(RAG_ERR_INVALID, "group " + std::to_string(g) + ": rows do not lie inside the store");
        if (out_begin) out_begin[g] = sum;
        pairs += (__int128)(d[1] - d[0]) * (d[3] - d[2]);
        if (pairs > (__int128)1 << 60) return fail(RAG_ERR_INVALID, "too many scores");
        sum = (long long)pairs;
        if (d[3] > d[2]) most_q = std::max<long long>(most_q, d[1] - d[0]);
    }
    *total = sum;
    *widest = (int32_t)most_q;
    const Mx4Shape p = mx4_shape(q_type, dim, std::max<long long>(most_q, 1), sum > MX4_WIDE);       // (no group has more rows than scores)
    // rows of an item: enough items to fill the chip several times over, each long enough to pay for staging its queries
    long long work = 0;
    for (long long g = 0; g < ngroups; ++g)
        work += (groups[4 * g + 1] - groups[4 * g] + p.qb - 1) / p.qb * (groups[4 * g + 3] - groups[4 * g + 2]);
    const long long unit = 16LL * p.nb * p.nw;
    const long long part = std::max<long long>(4 * unit, std::min<long long>(8192, (work / 1024 + unit - 1) / unit * unit));
    long long m = 0;
    Mx4Item* items = static_cast<Mx4Item*>(items_out);
    long long at = 0;
    for (long long g = 0; g < ngroups; ++g) {
        const int64_t* d = groups + 4 * g;
        const long long gq = d[1] - d[0], gr = d[3] - d[2];
        for (long long r = 0; r < gr && gq > 0; r += part)
            for (long long q = 0; q < gq; q += p.qb, ++m)
                if (m < max_items) {
                    Mx4Item it;
                    it.row0 = d[2] + r;
                    it.at = at + q * gr + r;
                    it.rows = (int)std::min(part, gr - r);
                    it.ld = (int)gr;
                    it.q0 = (int)(d[0] + q);
                    it.nq = (int)std::min<long long>(p.qb, gq - q);
                    items[m] = it;
                }
        at += gq * gr;
    }
    *n_items = m;
    return RAG_OK;
}

int rag_mx4_scores_grouped_device(const rag_mx4_store_t* st, int64_t nq, const void* q_dev, int q_type, int64_t q_stride, int normalize,
                                  const void* items_dev, int64_t n_items, int32_t widest, float* out_dev, int64_t total, void* stream) {
    if (int rc = mx4_check_queries(st, nq, q_dev, q_type, q_stride)) return rc;
    if (n_items < 0 || n_items > 0x7fffffffLL) return fail(RAG_ERR_INVALID, "n_items out of range");
    if (n_items == 0) return RAG_OK;
    if (nq == 0 || !items_dev || !out_dev) return fail(RAG_ERR_INVALID, "NULL buffer");
    if ((reinterpret_cast<uintptr_t>(items_dev) & 15)) return fail(RAG_ERR_INVALID, "items must lie on a 16-byte boundary");
    if (widest < 1 || widest > nq) return fail(RAG_ERR_INVALID, "widest is not what rag_mx4_plan_groups gave for these queries");
    Mx4DeviceGuard g(st->device);
    if (!g.ok) return fail(RAG_ERR_HIP, "hipSetDevice failed");
    const Mx4Shape p = mx4_shape(q_type, st->dim, widest, total > MX4_WIDE);
    Mx4ScoreArgs a = mx4_score_args(st, p, q_dev, q_type, q_stride, normalize ? 1 : 0, out_dev);
    a.items = static_cast<const Mx4Item*>(items_dev);
    a.nq = (int)nq;
    a.rows = st->n;
    a.total = total;
    return mx4_launch_any(p, a, n_items, st->device, static_cast<hipStream_t>(stream));
}

int64_t rag_mx4_search_workspace(int64_t n, int64_t nq, int k) {
    if (n < 0 || nq < 0 || k < 1 || k > 1024) return -1;
    return (int64_t)mx4_plan(n, nq, k).total();
}

int rag_mx4_search_device(const rag_mx4_store_t* st, int64_t nq, const void* q_dev, int q_type, int64_t q_stride, int normalize, int k,
                          float min_score, const uint8_t* row_mask_dev, const uint8_t* active_dev, float* D_dev, int64_t* I_dev, void* workspace_dev,
                          int64_t workspace_bytes, void* stream) {
    if (int rc = mx4_check_queries(st, nq, q_dev, q_type, q_stride)) return rc;
    if (k < 1 || k > 1024) return fail(RAG_ERR_INVALID, "k must be in [1, 1024]");
    if (min_score != min_score) return fail(RAG_ERR_INVALID, "min_score is NaN");
    if (nq == 0) return RAG_OK;
    if (!D_dev || !I_dev) return fail(RAG_ERR_INVALID, "NULL buffer");
    Mx4DeviceGuard g(st->device);
    if (!g.ok) return fail(RAG_ERR_HIP, "hipSetDevice failed");
    hipStream_t s = static_cast<hipStream_t>(stream);
    long long* I = reinterpret_cast<long long*>(I_dev);
    if (st->n == 0) {
        launch_fill_results(D_dev, I, (long long)nq * k, s);
        RAG_HIP_CHECK(hipGetLastError());
        return RAG_OK;
    }
    const Mx4Plan p = mx4_plan(st->n, nq, k);
    if (!workspace_dev || (reinterpret_cast<uintptr_t>(workspace_dev) & 255) || workspace_bytes < (int64_t)p.total())
        return fail(RAG_ERR_INVALID, "workspace: " + std::to_string(p.total()) + " bytes on a 256-byte boundary are needed");
    char* w = static_cast<char*>(workspace_dev);
    float* scores = reinterpret_cast<float*>(w);
    float* Dl = reinterpret_cast<float*>(w + p.scores);
    long long* Il = reinterpret_cast<long long*>(w + p.scores + p.d);
    u64* keys = reinterpret_cast<u64*>(w + p.scores + p.d + p.i);
    const uint8_t* mask = row_mask_dev ? row_mask_dev : active_dev;
    if (row_mask_dev && active_dev) {
        uint8_t* both = reinterpret_cast<uint8_t*>(w + p.scores + p.d + p.i + p.keys);
        hipLaunchKernelGGL(mx4_and_masks_kernel, dim3((unsigned)std::min<long long>(4096, (st->n + 255) / 256)), dim3(256), 0, s, row_mask_dev,
                           active_dev, (long long)st->n, both);
        RAG_HIP_CHECK(hipGetLastError());
        mask = both;
    }
    for (long long q0 = 0; q0 < nq; q0 += p.qc) {
        const long long qc = std::min<long long>(p.qc, nq - q0);
        const long long lists = qc * k;                       // hits of one list per query
        const char* q = static_cast<const char*>(q_dev) + (size_t)q0 * q_stride * mx4_esize(q_type);
        // list 0 is the answer so far; its k-th score is a floor for the rows behind it
        launch_fill_results(Dl, Il, lists, s);
        for (long long lo = 0; lo < st->n; lo += p.span * MX4_SEG) {
            const long long rows = std::min<long long>(p.span * MX4_SEG, st->n - lo);
            const int segs = (int)((rows + MX4_SEG - 1) / MX4_SEG);
            if (int rc = mx4_scores(st, lo, rows, qc, q, q_type, q_stride, normalize ? 1 : 0, scores, rows, s)) return rc;
            if (int rc = direct_select_segments(qc, rows, MX4_SEG, k, min_score, mask ? mask + lo : nullptr, nullptr, lo, scores,
                                                Dl + lists, Il + lists, lists, lo > 0 ? Dl + (k - 1) : nullptr, k, s))
                return rc;
            float* Do = D_dev + (size_t)q0 * k;
            long long* Io = I + (size_t)q0 * k;
            if (int rc = merge_lists_device(segs + 1, qc, k, Dl, lists, Il, lists, Do, Io, keys, s)) return rc;
            if (lo + rows < st->n) {
                hipLaunchKernelGGL(mx4_copy_lists_kernel, dim3((unsigned)std::min<long long>(256, (lists + 255) / 256)), dim3(256), 0, s, Do, Io,
                                   lists, Dl, Il);
                RAG_HIP_CHECK(hipGetLastError());
            }
        }
    }
    return RAG_OK;
}

}  // extern "C"
