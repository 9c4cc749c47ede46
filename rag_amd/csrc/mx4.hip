// Rows kept at four bits (e2m1 values, one power-of-two scale per group of 32 consecutive elements: the MX layout):
// quantising rows as they are written, reading them back, and multiplying them with queries.
//
// value(row, i) = sign * T[code & 7] * 2^(scale[i / 32] - 127),  T = {0, 0.5, 1, 1.5, 2, 3, 4, 6};  scale 255: NaN.
#include <float.h>
#include <limits.h>
#include <math.h>
#include <string.h>

#include <algorithm>
#include <mutex>

#include "index.h"
#include "mx4_device.h"
#include "topk_keys.h"

namespace rag {

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
    long long block0;            // of the launch's first workgroup
};
constexpr int MX4_ROWS = 64;                 // most rows of one workgroup
constexpr int MX4_FEW = 256;                 // up to so many positions a workgroup looks for repeated ones itself
constexpr int MX4_UNITS = 4;
constexpr long long MX4_GRID = 1 << 20;      // most workgroups of one launch: a launch has fewer than 2^32 threads

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
    __shared__ int s_exp[MX4_ROWS];
    __shared__ int s_late[MX4_ROWS];
    const long long i0 = (a.block0 + blockIdx.x) * a.per_block;
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
        s_exp[tid] = 0;
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
            int k;
            const float inv = wave_inv_norm(x + (size_t)r * a.ldx * ESIZE, TYPE, a.dim, lane, k);
            if (lane == 0) { s_inv[r] = inv; s_exp[r] = k; }
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
            if (!AT || s_to[r] >= 0) mx4_load8<TYPE, VEC>(x + (size_t)r * a.ldx * ESIZE, c * 8, a.dim, v[j]);
        }
#pragma unroll
        for (int j = 0; j < MX4_UNITS; ++j) {
            const int u = u0 + 256 * j;
            if (u >= units) break;
            const int r = (int)__umulhi((unsigned)u, a.per), c = u - r * a.upr;
            const long long to = s_to[r];
            if (AT && to < 0) continue;                                // uniform over the four lanes of a group
            const float inv = s_inv[r];
            const int k = s_exp[r];
            unsigned most = 0;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                v[j][i] = ldexpf(v[j][i], k) * inv;              // (the power of two first, exactly: no norm leaves the range)
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
            if ((c & 3) == 0)                                            // (groups behind the row's end: zero)
                a.scales[(size_t)to * a.scale_ld + mx4_scale_at(c >> 2)] = c * 8 >= a.dim ? 0 : bad ? 255 : (uint8_t)(e + 127);
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
    long long block0;
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
    const long long i0 = (a.block0 + blockIdx.x) * a.per_block;
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

// ------------------------------------------------------------------------------------------------ products (kernels: mx4_scores.h)
constexpr long long MX4_MOST_ROWS = 8192;               // of a piece of a ragged group
constexpr long long MX4_WIDE = 100 * 1000 * 1000;        // 3 * 4 bytes * this, and a tile, stay below 2^31
constexpr long long MX4_BEYOND = 1LL << 37;              // scores, more than the memory of a card holds

// The shapes of a type, by the queries of a workgroup: those of the kernel for few queries, then those of the one for many.  32 of
// a type's queries and more go to the latter, whose fragments serve several row blocks; fp32 queries from 9 on, since the fragments of
// their three tiles, read for every block of rows, would take all that the LDS gives at the rate of HBM (16 x 4M x 768: 405 us)
struct Mx4Level {
    int qpt, mt, nb;             // nb 0: the kernel for few queries
};
struct Mx4Levels {
    int count, half;             // half: the level of one full tile, half of which is taken where the LDS does not hold it
    Mx4Level of[5];
};
static const Mx4Levels& mx4_levels(int type) {
    static const Mx4Levels f32 = {4, 0, {{4, 1, 0}, {4, 2, 0}, {16, 3, 2}, {16, 6, 3}}};                      // 4, 8, 16, 32 queries
    static const Mx4Levels f16 = {4, 1, {{4, 1, 0}, {8, 1, 0}, {8, 2, 0}, {8, 4, 4}}};                        // 4, 8, 16, 32
    static const Mx4Levels bf16 = {5, 2, {{4, 1, 0}, {8, 1, 0}, {16, 1, 0}, {16, 2, 0}, {16, 4, 4}}};         // 4, 8, 16, 32, 64
    return type == RAG_MX4_F32 ? f32 : type == RAG_MX4_F16 ? f16 : bf16;
}
static int mx4_most(int type, int level) {
    const Mx4Level& v = mx4_levels(type).of[level];
    return type == RAG_MX4_F32 && v.qpt == 16 ? v.mt / 3 * 16 : v.mt * v.qpt;
}
// lowest level whose workgroups take nq queries (or the last one)
static int mx4_level_for(int type, long long nq) {
    int level = 0;
    while (level + 1 < mx4_levels(type).count && mx4_most(type, level) < nq) ++level;
    return level;
}
// The shape of a level, or of the next lower one that there is for rows of this length.  apart: how far apart the scores of two queries may
// lie.  Beyond a lane's 32-bit offset each query needs a base of its own: the kernel for many has them, and that for up to 8 of a large
// store.  (A plan for more scores than there can be keeps the pieces of 8 queries.)
static Mx4Shape mx4_shape(int type, int dim, int level, long long apart) {
    constexpr int LDS = 160 * 1024;
    const int ks = mx4_blocks(dim);
    Mx4Shape p = {};
    for (;; --level) {
        const Mx4Level& v = mx4_levels(type).of[level];
        p.qpt = v.qpt;
        p.mt = v.mt;
        p.nb = v.nb;
        p.qb = mx4_most(type, level);
        p.many = v.nb > 0;
        p.r = 16;
        if (apart > MX4_BEYOND ? p.qb > 8 : apart > MX4_WIDE && !p.many && p.qb > 8) continue;
        if (p.many) {
            p.nw = 8;
            p.ksu = ks;
            const size_t factors = (size_t)p.qb * 8;
            p.lds = (size_t)ks * p.mt * 4096 + factors;
            p.steps = p.lds <= LDS;                          // the whole queries lie in LDS; else two blocks of them
            if (!p.steps) p.lds = (size_t)2 * p.mt * 4096 + factors;
            return p;
        }
        p.big = apart > MX4_WIDE;
        p.nb = 1;
        p.steps = ks <= 8 && ks != 5 && ks != 7;
        p.u = p.steps ? ks : (ks & 7) == 0 || (ks & 7) > 4 ? 8 : 4;      // (blocks past the row's are fetched again, from the caches)
        p.nw = p.steps ? 4 : 8;                              // eight waves share the fragments where these fill much of the LDS
        p.ksu = (ks + p.u - 1) / p.u * p.u;
        p.lds = (size_t)p.ksu * p.mt * 4096 + (size_t)p.qb * 8;      // (with a factor and a power of two for each query)
        if (p.lds <= LDS) return p;
        if (level > 0) continue;
        // the longest rows: one tile of which the LDS holds eight rows
        const Mx4Level& one = mx4_levels(type).of[mx4_levels(type).half];
        p.qpt = one.qpt;
        p.r = 8;
        p.u = 8;
        p.ksu = (ks + 7) / 8 * 8;
        p.lds = (size_t)p.ksu * 2048 + (size_t)one.qpt * 8;
        p.qb = one.qpt / 2;
        return p;
    }
}
// The shape for nq queries, where groups_of(shape) workgroups have a whole unit of rows: fewer queries to a workgroup where more would
// leave more than half of the compute units idle (32 fp32 queries x 10k x 768: 7.8 us, asked to fill a quarter of them 9.3; x 40k 14.6, 17.0;
// 64 bf16 queries x 2000 x 1024: 5.6, 7.8)
template <typename Units>
static Mx4Shape mx4_shape_for(int type, int dim, long long nq, long long apart, Units groups_of) {
    int level = mx4_level_for(type, nq);
    Mx4Shape p = mx4_shape(type, dim, level, apart);
    while (level > 0 && groups_of(p) < 128) p = mx4_shape(type, dim, --level, apart);
    return p;
}

static int mx4_launch_any(const Mx4Shape& p, int type, const Mx4ScoreArgs& a, long long grid, int device, hipStream_t s) {
    if (grid < 1 || grid * p.nw * 64 > 0xffffffffLL) return fail(RAG_ERR_INVALID, "four-bit product: grid out of range");
    return type == RAG_MX4_F32 ? mx4_launch_f32(p, a, grid, device, s) : type == RAG_MX4_F16 ? mx4_launch_f16(p, a, grid, device, s)
                                                                                          : mx4_launch_bf16(p, a, grid, device, s);
}

static bool mx4_lies_on(const void* p, size_t boundary) { return (reinterpret_cast<uintptr_t>(p) & (boundary - 1)) == 0; }
static int mx4_check_store(const rag_mx4_store_t* st) {
    if (!st) return fail(RAG_ERR_INVALID, "store is NULL");
    if (st->dim < 1 || st->dim > MX4_MAX_DIM) return fail(RAG_ERR_INVALID, "dim must be in [1, " + std::to_string(MX4_MAX_DIM) + "]");
    if (st->n < 0 || st->n > 0x7fffffffLL) return fail(RAG_ERR_INVALID, "a store holds 0 to 2^31 - 1 rows");
    if (st->n > 0 && (!st->codes || !st->scales)) return fail(RAG_ERR_INVALID, "store without buffers");
    if (!mx4_lies_on(st->codes, 16) || !mx4_lies_on(st->scales, 16))
        return fail(RAG_ERR_INVALID, "the store's buffers must lie on 16-byte boundaries");
    return RAG_OK;
}
static int mx4_check_type(int type) {
    if (type != RAG_MX4_F32 && type != RAG_MX4_BF16 && type != RAG_MX4_F16) return fail(RAG_ERR_INVALID, "unknown element type");
    return RAG_OK;
}
static size_t mx4_esize(int type) { return type == RAG_MX4_F32 ? 4 : 2; }
static int mx4_aligned(const void* p, long long ld, int type) {
    return mx4_lies_on(p, 16) && (size_t)ld * mx4_esize(type) % 16 == 0;
}
// rows of a workgroup that writes or reads rows: four units a thread, fewer where that would leave compute units without work
static int mx4_rows_per_block(long long count, int upr) {
    const long long full = std::max(1, std::min(MX4_ROWS, 256 * MX4_UNITS / upr));
    return (int)std::max<long long>(1, std::min<long long>(full, count / 512));
}
static Mx4ScoreArgs mx4_score_args(const rag_mx4_store_t* st, const Mx4Shape& p, const void* q, long long ldq, int normalize, float* out) {
    Mx4ScoreArgs a = {};
    a.codes = static_cast<const uint8_t*>(st->codes);
    a.scales = static_cast<const uint8_t*>(st->scales);
    a.q = q;
    a.ldq = ldq;
    a.dim = st->dim;
    a.ks = mx4_blocks(st->dim);
    a.per = (unsigned)((0x100000000ull + 16 * a.ks - 1) / (16 * a.ks));
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
    Mx4Shape p = mx4_shape_for(q_type, st->dim, nq, out_ld, [&](const Mx4Shape& s) {
        return (rows + 16LL * s.nb * s.nw - 1) / (16LL * s.nb * s.nw) * ((nq + s.qb - 1) / s.qb);
    });
    Mx4ScoreArgs a = mx4_score_args(st, p, q, ldq, normalize, out);
    // Past the caches once the rows exceed the 256 MB that they keep from call to call (one query x 600k x 768, 250 MB: 39 us kept, 46 past
    // them; 800k 61.6 and 59.3; 16 bf16 queries x 800k 80 and 73), and for up to 8 queries, whose waves then take 64 rows at a
    // time, once these keep the waves busy (130k x 4096: 52 us in pieces of 64 rows, 48 of 16)
    p.big = p.big || (!p.many && nq <= p.qb && rows * (a.code_ld + a.scale_ld) > 256LL << 20 && (p.qb > 8 || rows >= 64 * 4096));
    a.row0 = row0;
    a.rows = rows;
    a.out_ld = out_ld;
    a.nq = (int)nq;
    a.nqb = (int)((nq + p.qb - 1) / p.qb);
    const long long unit = 16LL * p.nb * p.nw;                  // rows of one step of a workgroup
    const long long units = (rows + unit - 1) / unit;
    // workgroups that are at work at a time
    const long long seats = 256LL * (p.many ? 1 : std::max<long long>(1, std::min<long long>(16 / p.nw, 160 * 1024 / p.lds)));
    if (!p.many && a.nqb == 1) return mx4_launch_any(p, q_type, a, std::min(units, seats), st->device, s);
    // Slabs: as many as make the workgroups come out even over the chip's compute units, each long against the staging of
    // its queries (about two units of work)
    long long best = 1, least = LLONG_MAX;
    for (long long n = 1; n <= std::min<long long>(units, std::max<long long>(64, 8 * seats / a.nqb)); ++n) {
        const long long cost = (n * a.nqb + seats - 1) / seats * ((units + n - 1) / n + (p.many ? 1 : 2));
        if (cost < least) { least = cost; best = n; }
    }
    a.slab = (units + best - 1) / best * unit;
    a.slabs = (rows + a.slab - 1) / a.slab;
    return mx4_launch_any(p, q_type, a, (a.slabs * a.nqb + 7) / 8 * 8, st->device, s);
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

// Pieces on their way to the device.  A few KB as a kernel that reads page-locked memory cost a launch; as a copy command they
// wait for its own signalling (a plan of 591 pieces with the product behind it: 47 us by copy, 30 by kernel).  The
// kernel's last store says that the block may be used again.
struct Mx4Slot {
    char* host = nullptr;
    unsigned long long* done = nullptr;     // page-locked too, behind the bytes
    unsigned long long turn = 0;            // what `done` holds once the block's last copy has been made
};
constexpr size_t MX4_SLOT_BYTES = 128 * 1024;
constexpr int MX4_SLOTS = 64;
static std::mutex g_mx4_slots_mu;
static Mx4Slot g_mx4_slots[MX4_SLOTS];
static int g_mx4_slot_next = 0;

__global__ __launch_bounds__(1024) void mx4_upload_kernel(const v4i* from, v4i* to, int n, unsigned long long* done, unsigned long long turn) {
    for (int i0 = threadIdx.x; i0 < n; i0 += 4096) {
        v4i x[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) x[j] = from[i0 + 1024 * j < n ? i0 + 1024 * j : i0];
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (i0 + 1024 * j < n) to[i0 + 1024 * j] = x[j];
    }
    __syncthreads();                        // every load has been answered
    if (threadIdx.x == 0) {
        __threadfence_system();
        *reinterpret_cast<volatile unsigned long long*>(done) = turn;
    }
}

// a block whose last copy has been made (or a new one); nullptr: all of them are on their way, or no memory
static Mx4Slot* mx4_slot() {
    for (int i = 0; i < MX4_SLOTS; ++i) {
        Mx4Slot& s = g_mx4_slots[(g_mx4_slot_next + i) % MX4_SLOTS];
        if (!s.host) {
            void* p = nullptr;
            if (hipHostMalloc(&p, MX4_SLOT_BYTES + 64, hipHostMallocPortable | hipHostMallocCoherent) != hipSuccess) {
                (void)hipGetLastError();
                return nullptr;
            }
            s.host = static_cast<char*>(p);
            s.done = reinterpret_cast<unsigned long long*>(s.host + MX4_SLOT_BYTES);
            *s.done = s.turn;
        }
        if (*reinterpret_cast<volatile unsigned long long*>(s.done) == s.turn) {
            g_mx4_slot_next = (g_mx4_slot_next + i + 1) % MX4_SLOTS;
            return &s;
        }
    }
    return nullptr;
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
    if (!mx4_lies_on(x_dev, mx4_esize(x_type))) return fail(RAG_ERR_INVALID, "x is not aligned to its elements");
    if (rows_dev) {
        if (!owner_dev) return fail(RAG_ERR_INVALID, "positions need the store's owner array");
        if (!mx4_lies_on(rows_dev, 8) || !mx4_lies_on(owner_dev, 4)) return fail(RAG_ERR_INVALID, "rows or owner is not aligned to its elements");
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
    const long long blocks = (count + a.per_block - 1) / a.per_block;
    const int vec = mx4_aligned(x_dev, x_stride, x_type);
    for (; a.block0 < blocks; a.block0 += MX4_GRID) {
        const dim3 grid((unsigned)std::min(MX4_GRID, blocks - a.block0));
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
    }
    return RAG_OK;
}

int rag_mx4_read_device(const rag_mx4_store_t* st, const int64_t* rows_dev, int64_t count, void* out_dev, int out_type, void* stream) {
    if (int rc = mx4_check_store(st)) return rc;
    if (int rc = mx4_check_type(out_type)) return rc;
    if (count < 0 || count >= 0x7fffffffLL) return fail(RAG_ERR_INVALID, "count out of range");
    if (count == 0) return RAG_OK;
    if (!rows_dev || !out_dev) return fail(RAG_ERR_INVALID, "NULL buffer");
    if (!mx4_lies_on(rows_dev, 8)) return fail(RAG_ERR_INVALID, "rows is not aligned to its elements");
    if (!mx4_lies_on(out_dev, mx4_esize(out_type))) return fail(RAG_ERR_INVALID, "out is not aligned to its elements");
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
    const long long blocks = (count + a.per_block - 1) / a.per_block;
    const int vec = st->dim % 8 == 0 && mx4_aligned(out_dev, st->dim, out_type);
    hipStream_t s = static_cast<hipStream_t>(stream);
    for (; a.block0 < blocks; a.block0 += MX4_GRID) {
        const dim3 grid((unsigned)std::min(MX4_GRID, blocks - a.block0));
#define MX4_READ(T) \
        if (out_type == T) { \
            if (vec) hipLaunchKernelGGL((mx4_read_kernel<T, true>), grid, dim3(256), 0, s, a); \
            else hipLaunchKernelGGL((mx4_read_kernel<T, false>), grid, dim3(256), 0, s, a); \
        }
        MX4_READ(RAG_MX4_F32) MX4_READ(RAG_MX4_BF16) MX4_READ(RAG_MX4_F16)
#undef MX4_READ
        RAG_HIP_CHECK(hipGetLastError());
    }
    return RAG_OK;
}

static int mx4_check_queries(const rag_mx4_store_t* st, int64_t nq, const void* q_dev, int q_type, int64_t q_stride) {
    if (int rc = mx4_check_store(st)) return rc;
    if (int rc = mx4_check_type(q_type)) return rc;
    if (nq < 0 || nq > 0x7fffffffLL) return fail(RAG_ERR_INVALID, "nq out of range");
    if (nq > 0 && !q_dev) return fail(RAG_ERR_INVALID, "NULL buffer");
    if (nq > 0 && q_stride < st->dim) return fail(RAG_ERR_INVALID, "q_stride smaller than dim");
    if (!mx4_lies_on(q_dev, mx4_esize(q_type))) return fail(RAG_ERR_INVALID, "q is not aligned to its elements");
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
    if (!mx4_lies_on(out_dev, 4)) return fail(RAG_ERR_INVALID, "out is not aligned to its elements");
    Mx4DeviceGuard g(st->device);
    if (!g.ok) return fail(RAG_ERR_HIP, "hipSetDevice failed");
    constexpr int64_t most = 1 << 22;                           // queries of one launch (see MX4_GRID)
    for (int64_t i = 0; i < nq; i += most)
        if (int rc = mx4_scores(st, row_begin, rows, std::min(most, nq - i), static_cast<const char*>(q_dev) + (size_t)i * q_stride * mx4_esize(q_type),
                                q_type, q_stride, normalize ? 1 : 0, out_dev + (size_t)i * out_stride, out_stride, static_cast<hipStream_t>(stream)))
            return rc;
    return RAG_OK;
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
    // rows of a piece: enough pieces to fill the chip several times over, each long enough to pay for staging its queries;
    // with one tile, where that costs little and more workgroups fit a compute unit, shorter ones (1000 groups of 3 fp32
    // queries x 2000 rows x 384: 96.7 us in pieces of 1024, 92.6 of 512); with many queries four units of rows at least (100 groups of 40
    // bf16 queries x 4000 x 768: 57 us, in pieces of three, two and one 71, 63 and 78)
    long long part = 0;
    auto queries = [&](long long g) { return (uint32_t)(groups[4 * g + 1] - groups[4 * g]); };
    auto rows = [&](long long g) { return (uint32_t)(groups[4 * g + 3] - groups[4 * g + 2]); };
    auto parts = [](uint32_t a, uint32_t b) { return (a + b - 1) / b; };       // (in 32 bits: a division of 64 costs several times as much)
    auto cut = [&](const Mx4Shape& s) -> long long {          // sets `part`, says how many pieces there are
        const long long unit = 16LL * s.nb * s.nw;
        long long work = 0, items = 0;
        for (long long g = 0; g < ngroups; ++g)
            work += (long long)parts(queries(g), s.qb) * rows(g);
        part = std::max<long long>(4 * unit, std::min<long long>(MX4_MOST_ROWS, (work / (!s.many && s.mt == 1 ? 4096 : 1024) + unit - 1) / unit * unit));
        for (long long g = 0; g < ngroups; ++g)
            items += (long long)parts(queries(g), s.qb) * parts(rows(g), (uint32_t)part);
        return items;
    };
    const Mx4Shape p = mx4_shape_for(q_type, dim, std::max<long long>(most_q, 1), sum, cut);       // (no group has more rows than scores)
    const long long pieces = cut(p);
    if (pieces > 0x7fffffffLL) return fail(RAG_ERR_INVALID, "too many pieces");
    *widest = (int32_t)std::min<long long>(most_q, p.qb);
    *n_items = pieces;
    if (pieces > max_items) return RAG_OK;
    // The longest pieces first, so that the last workgroups to begin are the short ones (200 groups of up to 24 fp16 queries x
    // 3000 rows x 384: 50.3 us in the groups' order, 41.6 like this; 512 lists of 400 rows x 1024: 24.3, 23.8)
    constexpr int CLASSES = MX4_MOST_ROWS / 16;
    int64_t place[CLASSES] = {};                          // pieces of each (rows - 1) / 16, then where the next one of them goes
    for (long long g = 0; g < ngroups; ++g) {
        const uint32_t gq = parts(queries(g), p.qb), full = rows(g) / (uint32_t)part, rest = rows(g) - full * (uint32_t)part;
        place[part / 16 - 1] += (int64_t)full * gq;
        if (rest) place[(rest - 1) / 16] += gq;
    }
    int64_t behind = 0;
    for (int c = CLASSES; c-- > 0;) {
        const int64_t many = place[c];
        place[c] = behind;
        behind += many;
    }
    Mx4Item* items = static_cast<Mx4Item*>(items_out);
    long long at = 0;
    for (long long g = 0; g < ngroups; ++g) {
        const int64_t* d = groups + 4 * g;
        const long long gq = d[1] - d[0], gr = d[3] - d[2];
        for (long long r = 0; r < gr && gq > 0; r += part) {
            const long long nr = std::min(part, gr - r);
            for (long long q = 0; q < gq; q += p.qb) {
                Mx4Item& it = items[place[(nr - 1) / 16]++];
                it.row0 = d[2] + r;
                it.at = at + q * gr + r;
                it.rows = (int)nr;
                it.ld = (int)gr;
                it.q0 = (int)(d[0] + q);
                it.nq = (int)std::min<long long>(p.qb, gq - q);
            }
        }
        at += gq * gr;
    }
    return RAG_OK;
}

int rag_mx4_upload_groups(const void* items, int64_t n_items, void* items_dev, int device, void* stream) {
    if (n_items < 0 || n_items > 0x7fffffffLL) return fail(RAG_ERR_INVALID, "n_items out of range");
    if (n_items == 0) return RAG_OK;
    if (!items || !items_dev) return fail(RAG_ERR_INVALID, "NULL buffer");
    if (!mx4_lies_on(items_dev, 16)) return fail(RAG_ERR_INVALID, "items must lie on a 16-byte boundary");
    Mx4DeviceGuard g(device);
    if (!g.ok) return fail(RAG_ERR_HIP, "hipSetDevice failed");
    hipStream_t s = static_cast<hipStream_t>(stream);
    hipStreamCaptureStatus capturing = hipStreamCaptureStatusNone;
    RAG_HIP_CHECK(hipStreamIsCapturing(s, &capturing));
    if (capturing != hipStreamCaptureStatusNone) return fail(RAG_ERR_INVALID, "pieces are copied outside of a graph capture");
    const size_t bytes = (size_t)n_items * sizeof(Mx4Item);
    if (bytes <= MX4_SLOT_BYTES) {
        std::lock_guard<std::mutex> lock(g_mx4_slots_mu);
        if (Mx4Slot* slot = mx4_slot()) {
            memcpy(slot->host, items, bytes);
            hipLaunchKernelGGL(mx4_upload_kernel, dim3(1), dim3(1024), 0, s, reinterpret_cast<const v4i*>(slot->host), static_cast<v4i*>(items_dev),
                               (int)(bytes / 16), slot->done, slot->turn + 1);
            RAG_HIP_CHECK(hipGetLastError());
            ++slot->turn;
            return RAG_OK;
        }
    }
    // (from pageable memory: the runtime has taken its copy when this returns)
    RAG_HIP_CHECK(hipMemcpyAsync(items_dev, items, bytes, hipMemcpyHostToDevice, s));
    RAG_HIP_CHECK(hipStreamSynchronize(s));
    return RAG_OK;
}

int rag_mx4_scores_grouped_device(const rag_mx4_store_t* st, int64_t nq, const void* q_dev, int q_type, int64_t q_stride, int normalize,
                                  const void* items_dev, int64_t n_items, int32_t widest, float* out_dev, int64_t total, void* stream) {
    if (int rc = mx4_check_queries(st, nq, q_dev, q_type, q_stride)) return rc;
    if (n_items < 0 || n_items > 0x7fffffffLL) return fail(RAG_ERR_INVALID, "n_items out of range");
    if (n_items == 0) return RAG_OK;
    if (nq == 0 || !items_dev || !out_dev) return fail(RAG_ERR_INVALID, "NULL buffer");
    if (!mx4_lies_on(items_dev, 16)) return fail(RAG_ERR_INVALID, "items must lie on a 16-byte boundary");
    if (!mx4_lies_on(out_dev, 4)) return fail(RAG_ERR_INVALID, "out is not aligned to its elements");
    if (widest < 1 || widest > nq) return fail(RAG_ERR_INVALID, "widest is not what rag_mx4_plan_groups gave for these queries");
    Mx4DeviceGuard g(st->device);
    if (!g.ok) return fail(RAG_ERR_HIP, "hipSetDevice failed");
    const Mx4Shape p = mx4_shape(q_type, st->dim, mx4_level_for(q_type, widest), total);
    Mx4ScoreArgs a = mx4_score_args(st, p, q_dev, q_stride, normalize ? 1 : 0, out_dev);
    a.nq = (int)nq;
    a.rows = st->n;
    a.total = total;
    for (int64_t i = 0; i < n_items; i += MX4_GRID) {
        a.items = static_cast<const Mx4Item*>(items_dev) + i;
        if (int rc = mx4_launch_any(p, q_type, a, std::min<int64_t>(MX4_GRID, n_items - i), st->device, static_cast<hipStream_t>(stream))) return rc;
    }
    return RAG_OK;
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
    if (!mx4_lies_on(D_dev, 4) || !mx4_lies_on(I_dev, 8)) return fail(RAG_ERR_INVALID, "D or I is not aligned to its elements");
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
    if (!workspace_dev || !mx4_lies_on(workspace_dev, 256) || workspace_bytes < (int64_t)p.total())
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
