// Products of queries with four-bit rows.  Instantiated for fp32, bf16 and fp16 queries in mx4_scores_f32.hip, _bf16.hip and
// _f16.hip.
//
// A product is that of the numbers themselves: no bit of a query or a row is left out, only the sums are rounded.  A four-bit
// value times its power of two is a bf16 number (the conversion makes it with one instruction for two of them, subnormal ones
// too).  A query's element is split into as many bf16 numbers as hold all of its bits,
//     x = h + 2^-8 m + 2^-16 l,   h = bf16(x), m = bf16(2^8 (x - h)), l = 2^8 (2^8 (x - h) - m),
// three for fp32, h and m for fp16, h alone for bf16.  Each part keeps an exponent of its own, so it does not matter what else
// the query holds; and the factors 2^8 keep the parts of the smallest numbers above the end of bf16's range, and no part is larger than x.
// The bf16 matrix instruction multiplies them exactly and adds in fp32; the parts' sums are added at the end.
//
// Every kernel here adds in the same order -- along the row in steps of the instruction, one sum per part -- so a score does not
// depend on what it is computed together with.
#pragma once
#include "mx4_device.h"

namespace rag {

// Layout of v_mfma_f32_16x16x32_bf16 (checked on the card): lane l, column c = l / 16.  Either operand: row l % 16, eight
// elements of the step of 32.  Result register r of lane l: (row 4 c + r of the queries' parts, row l % 16 of the store).  A lane
// fetches a whole group of 32 elements of its row (column c of a block of 128) with its scale, and step i of a block takes elements
// 8 i .. 8 i + 7 of every lane's group.
//
// QPT: queries of a tile of 16 rows of parts.  16 / QPT rows each (4: the three parts of an fp32 query, or those of fewer queries
// than a tile holds); 16 for fp32 (SPLIT): three tiles hold the three parts of sixteen queries.  Queries go to the columns of lanes
// in turn, so that the scores of a store lie at most three queries apart, which a lane's 32-bit offset has to reach.
template <int P, int QPT, int MT>
struct Mx4Tiles {
    static constexpr bool SPLIT = P == 3 && QPT == 16;
    static constexpr int ROWS = 16 / QPT;                        // rows of a tile per query
    static constexpr int SETS = SPLIT ? MT / 3 : MT;             // sets of tiles with QPT queries each
    static constexpr int SPL = QPT / 4;                          // queries of a set whose scores a lane of column c holds: 4 j + c
    static constexpr int QB = SETS * QPT;
    static_assert(SPLIT ? MT % 3 == 0 : ROWS >= P, "");
};

// Where part p of query s lies: (tile, row).  Of a tile of R = 8 rows two columns hold queries.
template <int P, int QPT, int MT, int R>
__device__ __forceinline__ void mx4_part_at(int s, int p, int& tile, int& m) {
    typedef Mx4Tiles<P, QPT, MT> L;
    constexpr int COLS = R / 4;
    tile = L::SPLIT ? s / 16 * 3 + p : s / QPT;
    m = s % COLS * 4 + s % QPT / COLS * L::ROWS + (L::SPLIT ? 0 : p);
}

// A block of a tile in LDS: four steps of R rows x 4 columns x 16 bytes.  A lane's place among its column's is its row number
// exclusive-or'ed with step and column, so that the lanes that write consecutive elements of a query meet different banks.
template <int R>
__device__ __forceinline__ int mx4_frag_at(int step, int col, int m) {
    return step * R * 64 + (col * R + (m ^ ((4 * step + col) & (R - 1)))) * 16;
}

// Eight elements of a query as they lie in memory; past `dim` zeros.  Rows begin anywhere on their elements' boundary.
template <int P>
struct Mx4Raw {
    int w[P == 3 ? 8 : 4];
};
template <int P>
__device__ __forceinline__ Mx4Raw<P> mx4_raw(const char* row, int at, int dim) {
    constexpr int ESIZE = P == 3 ? 4 : 2;
    Mx4Raw<P> r;
    if (at + 8 <= dim) {
        const v4i_apart* from = reinterpret_cast<const v4i_apart*>(row + (size_t)at * ESIZE);
#pragma unroll
        for (int j = 0; j < (int)sizeof(r) / 16; ++j) {
            const v4i x = from[j];
            r.w[4 * j] = x.x; r.w[4 * j + 1] = x.y; r.w[4 * j + 2] = x.z; r.w[4 * j + 3] = x.w;
        }
    } else {
        typedef typename std::conditional<P == 3, int, unsigned short>::type Elem;
        Elem e[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) e[j] = reinterpret_cast<const Elem*>(row)[at + j < dim ? at + j : dim - 1];
#pragma unroll
        for (int j = 0; j < 8; ++j) e[j] = at + j < dim ? e[j] : (Elem)0;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            if constexpr (P == 3) r.w[j] = e[j];
            else if (j % 2 == 0) r.w[j / 2] = (int)((unsigned)e[j] | (unsigned)e[j + 1] << 16);
        }
    }
    return r;
}

// The bf16 number nearest to x; of a number that would round beyond the largest one what its upper bits are (the rest fits the next
// part), and an infinity leaves a NaN for the next part
__device__ __forceinline__ unsigned mx4_head(float x) {
    const unsigned u = __float_as_uint(x), h = (u + 0x7fffu + ((u >> 16) & 1u)) & 0xffff0000u;
    return (h & 0x7f800000u) == 0x7f800000u ? u & 0xffff0000u : h;
}
// two of them, side by side, with the conversion (infinity where x is near the end of the range)
__device__ __forceinline__ unsigned mx4_head2(float x, float y) { return __builtin_bit_cast(unsigned, __builtin_convertvector((v2f){x, y}, v2bf)); }

// Eight elements of a query as parts
template <int P>
struct Mx4Split {
    int w[P][4];
    // elements 2 j and 2 j + 1; SCALED: times 2^k, exactly
    template <bool SCALED>
    __device__ __forceinline__ void pair(const Mx4Raw<P>& raw, int j, int k) {
        if constexpr (P == 1 && !SCALED) {                       // as they are; an infinity becomes a NaN
            const unsigned x = (unsigned)raw.w[j], lo = (x & 0x7f80u) == 0x7f80u ? 0x40u : 0u, hi = (x & 0x7f800000u) == 0x7f800000u ? 0x400000u : 0u;
            w[0][j] = (int)(x | lo | hi);
        } else {
            float x, y;
            if constexpr (P == 3) {
                x = __int_as_float(raw.w[2 * j]);
                y = __int_as_float(raw.w[2 * j + 1]);
            } else if constexpr (P == 2) {
                x = f16_f32((unsigned short)(unsigned)raw.w[j]);              // (an infinity's second part is NaN)
                y = f16_f32((unsigned short)((unsigned)raw.w[j] >> 16));
            } else {
                x = bf16_f32((unsigned)raw.w[j] & 0xffffu);
                y = __uint_as_float((unsigned)raw.w[j] & 0xffff0000u);
            }
            if constexpr (SCALED) {
                x = ldexpf(x, k);
                y = ldexpf(y, k);
            }
#pragma unroll
            for (int p = 0; p + 1 < P; ++p) {
                const unsigned h = mx4_head2(x, y);
                w[p][j] = (int)h;
                x = (x - __uint_as_float(h << 16)) * 256.f;
                y = (y - __uint_as_float(h & 0xffff0000u)) * 256.f;
            }
            w[P - 1][j] = (int)(__float_as_uint(x) >> 16 | (__float_as_uint(y) & 0xffff0000u));
        }
    }
    // Where an element would round beyond the range, or is beyond it, all of them again.  (Only fp32 elements can; scaled ones do not,
    // and a query that is not finite has a factor that makes its scores NaN.)
    template <bool SCALED>
    __device__ __forceinline__ void finish(const Mx4Raw<P>& raw) {
        if constexpr (P == 3 && !SCALED) {
            unsigned most = 0;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const unsigned m = (unsigned)raw.w[j] & 0x7fffffffu;
                most = m > most ? m : most;
            }
            if (most >= 0x7f7f8000u) {
                float v[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) v[j] = __int_as_float(raw.w[j]);
#pragma unroll
                for (int p = 0; p < P; ++p) {
                    unsigned h[8];
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        h[j] = mx4_head(v[j]);
                        v[j] = (v[j] - __uint_as_float(h[j])) * 256.f;
                    }
#pragma unroll
                    for (int j = 0; j < 4; ++j) w[p][j] = (int)(h[2 * j] >> 16 | h[2 * j + 1]);
                }
            }
        }
    }
    // unit `unit` of a block of query s, into the fragments of that block
    template <int QPT, int MT, int R>
    __device__ __forceinline__ void store(int s, int unit, uint8_t* frag) const {
#pragma unroll
        for (int p = 0; p < P; ++p) {
            int tile, m;
            mx4_part_at<P, QPT, MT, R>(s, p, tile, m);
            *reinterpret_cast<v4i*>(frag + tile * R * 256 + mx4_frag_at<R>(unit & 3, (unit >> 2) & 3, m)) = (v4i){w[p][0], w[p][1], w[p][2], w[p][3]};
        }
    }
};

// COSINE: the queries are multiplied with 2^k before they are split, so that neither their parts nor their sums leave the range, and
// the scores with inv
template <int P, int QB, int NT>
__device__ __forceinline__ void mx4_query_norms(const Mx4ScoreArgs& a, const char* q, int nqh, float* inv, int* k) {
    constexpr int ESIZE = P == 3 ? 4 : 2, TYPE = P == 3 ? RAG_MX4_F32 : P == 2 ? RAG_MX4_F16 : RAG_MX4_BF16;
    if (a.normalize) {
        for (int s = threadIdx.x >> 6; s < nqh; s += NT / 64) {
            int e;
            const float f = wave_inv_norm(q + (size_t)s * a.ldq * ESIZE, TYPE, a.dim, threadIdx.x & 63, e);
            if ((threadIdx.x & 63) == 0) { inv[s] = f; k[s] = e; }
        }
        __syncthreads();
    } else {
        for (int s = threadIdx.x; s < QB; s += NT) inv[s] = 1.f;
    }
}

// queries [q0, q0 + nqh) -> their parts in LDS, block after block.  Blocks past the row's are zero: they meet a real block of the
// row again.  What the fragments of absent queries hold does not matter: it stays in result rows that nobody reads.
template <int P, int QPT, int MT, int R, int NT>
__device__ __forceinline__ void mx4_stage_queries(const Mx4ScoreArgs& a, const char* q, int nqh, uint8_t* frag, float* inv, int* k) {
    typedef Mx4Tiles<P, QPT, MT> L;
    constexpr int ESIZE = P == 3 ? 4 : 2, BLOCK = MT * R * 256;
    const int tid = threadIdx.x;
    mx4_query_norms<P, L::QB, NT>(a, q, nqh, inv, k);
    if (a.ksu > a.ks) {
        const v4i zero = {0, 0, 0, 0};
        v4i* f = reinterpret_cast<v4i*>(frag + a.ks * BLOCK);
        for (int i = tid; i < (a.ksu - a.ks) * (BLOCK / 16); i += NT) f[i] = zero;
    }
    // a few units at once, so that their fetches are under way together (behind the last unit: that one again)
    const int units = nqh * a.ks * 16;
    auto stage = [&](auto together, auto scaled) {
        constexpr int N = decltype(together)::value;
        constexpr bool SCALED = decltype(scaled)::value;
        for (int u0 = tid; u0 < units; u0 += NT * N) {
            Mx4Raw<P> raw[N];
            int s[N], unit[N];
#pragma unroll
            for (int j = 0; j < N; ++j) {
                const int u = u0 + j * NT < units ? u0 + j * NT : units - 1;
                s[j] = (int)__umulhi((unsigned)u, a.per);
                unit[j] = u - s[j] * a.ks * 16;
                raw[j] = mx4_raw<P>(q + (size_t)s[j] * a.ldq * ESIZE, unit[j] * 8, a.dim);
            }
#pragma unroll
            for (int j = 0; j < N; ++j) {
                if (j > 0 && u0 + j * NT >= units) break;
                Mx4Split<P> parts;
#pragma unroll
                for (int i = 0; i < 4; ++i) parts.template pair<SCALED>(raw[j], i, SCALED ? k[s[j]] : 0);
                parts.template finish<SCALED>(raw[j]);
                parts.template store<QPT, MT, R>(s[j], unit[j] & 15, frag + (unit[j] >> 4) * BLOCK);
            }
        }
    };
    typedef std::integral_constant<int, 1> One;
    typedef std::integral_constant<int, 4> Four;
    if (a.normalize) units <= NT ? stage(One{}, std::true_type{}) : stage(Four{}, std::true_type{});
    else units <= NT ? stage(One{}, std::false_type{}) : stage(Four{}, std::false_type{});
    __syncthreads();
}

// step `i` of a block of a row: eight four-bit values of each lane as bf16 numbers.  scale: the power of two as a float
__device__ __forceinline__ v8bf mx4_unpack(int w, float scale) {
    const v2bf a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4((unsigned)w, scale, 0), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4((unsigned)w, scale, 1);
    const v2bf c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4((unsigned)w, scale, 2), d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4((unsigned)w, scale, 3);
    return (v8bf){a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}
// byte b of four scales (255: an infinity here, which the conversion takes for NaN; 0: 2^-127)
__device__ __forceinline__ float mx4_scale(int x, int b) { return __uint_as_float(__builtin_amdgcn_ubfe((unsigned)x, 8 * b, 8) << 23); }

// the sums of the parts of query j of a set in this lane -> its score
template <int P, int QPT, int MT, int NB>
__device__ __forceinline__ float mx4_sum(const v4f (&acc)[MT][NB], int set, int nb, int j) {
    constexpr float DOWN = 1.f / 256;
    if constexpr (Mx4Tiles<P, QPT, MT>::SPLIT)
        return fmaf(fmaf(acc[3 * set + 2][nb][j], DOWN, acc[3 * set + 1][nb][j]), DOWN, acc[3 * set][nb][j]);
    else {
        const v4f v = acc[set][nb];
        constexpr int ROWS = Mx4Tiles<P, QPT, MT>::ROWS;
        if constexpr (P == 1) return v[ROWS * j];
        else if constexpr (P == 2) return fmaf(v[ROWS * j + 1], DOWN, v[ROWS * j]);
        else return fmaf(fmaf(v[2], DOWN, v[1]), DOWN, v[0]);
    }
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

// What a workgroup does: rows [row0, row0 + rows) against queries [q0, q0 + nqh), score (i, r) to out[at + i * ld + r]
struct Mx4Work {
    long long row0, at, ld;
    int rows, q0, nqh;
};
__device__ __forceinline__ bool mx4_work(const Mx4ScoreArgs& a, int qb_size, Mx4Work& w) {
    if (a.items) {
        const Mx4Item it = a.items[blockIdx.x];
        w.row0 = it.row0; w.at = it.at; w.ld = it.ld; w.rows = it.rows; w.q0 = it.q0; w.nqh = it.nq;
        // a piece that was not made for this store, these queries or this result is left out
        return !(w.rows < 1 || w.row0 < 0 || w.row0 > a.rows - w.rows || w.nqh < 1 || w.nqh > qb_size || w.q0 < 0 || w.q0 > a.nq - w.nqh ||
                 w.ld < w.rows || w.at < 0 || w.at > a.total - (long long)(w.nqh - 1) * w.ld - w.rows);
    }
    // workgroups go to the eight dies in turn: each die takes a contiguous part of the (slab, query block) pairs, so the
    // query blocks of a slab stay on one die, whose L2 then holds the slab's rows for all of them
    const long long pairs = a.slabs * a.nqb, id = (blockIdx.x & 7) * ((pairs + 7) >> 3) + (blockIdx.x >> 3);
    if (id >= pairs || (blockIdx.x >> 3) >= (pairs + 7) >> 3) return false;
    const long long s = id / a.nqb;
    const int qb = (int)(id % a.nqb);
    const long long lo = s * a.slab;
    w.rows = (int)(a.rows - lo < a.slab ? a.rows - lo : a.slab);
    w.q0 = qb * qb_size;
    w.nqh = a.nq - w.q0 < qb_size ? a.nq - w.q0 : qb_size;
    w.row0 = a.row0 + lo;
    w.at = (long long)w.q0 * a.out_ld + lo;
    w.ld = a.out_ld;
    return true;
}

// Sixteen rows from r0 on are fetched through buffer descriptors that end with the store: rows past the last one of a piece are fetched
// and never stored, what would lie behind the store comes back as zeros.  (The check is lane offset >= size - uniform offset: the
// uniform part, a block or scale dword of the first row, always lies inside the store.)
struct Mx4Rows {
    __amdgpu_buffer_rsrc_t codes, scales;
    __device__ __forceinline__ Mx4Rows(const Mx4ScoreArgs& a, long long r0) {
        const size_t wat = (size_t)(r0 >> 4) * 16 * a.code_ld, sat = (size_t)r0 * a.scale_ld;
        const size_t wleft = a.code_bytes - wat, sleft = a.scale_bytes - sat;
        codes = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(a.codes) + wat, 0, (int)(wleft < 0x7fffffffu ? wleft : 0x7fffffffu), 0x00027000);
        scales = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(a.scales) + sat, 0, (int)(sleft < 0x7fffffffu ? sleft : 0x7fffffffu), 0x00027000);
    }
};
__device__ __forceinline__ void mx4_put(float v, float* base, int bytes, unsigned offset) {
    __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(v), __builtin_amdgcn_make_buffer_rsrc(base, 0, bytes, 0x00027000), offset, 0, 0);
}
constexpr unsigned MX4_NOWHERE = 0x80000000u;                    // an offset behind every descriptor's end: nothing is stored

// Few queries: MT tiles of them in LDS for the whole row, U blocks of 128 along the row fetched together, NW waves.
// STEPS 1: one fetch is a row; 0: as many as it takes.  R: rows of a tile that the LDS holds (8 where 16 of the longest rows do not
// fit: half as many queries; the lanes of the other rows read the first ones again).
//
// A wave takes 16 rows at a time and keeps the next U blocks of them in flight while the present ones go through the
// matrix unit; nothing but the query fragments goes through LDS, and there is no barrier after they are staged.  The wave's
// memory operations are the same whatever the data: the fetch ahead is made past the last rows too (of the last ones again), and
// lanes without a score to store address nothing behind a buffer descriptor's end.  Behind a branch the compiler would have to
// wait for all of them at every turn, stores too.
//
// BIG, for stores that no cache keeps: rows are fetched past them, and where up to 8 queries meet a row (LONG) a wave takes four tiles of
// sixteen rows in a row and stores their scores together, 256 contiguous bytes per query instead of 64.
//
// What bounds it: HBM.  4M x 768, one query: 265 us, 6.2 TB/s of rows, scales and scores (reading the same rows alone takes 220 us);
// 16 bf16 queries x 1M x 1024: 111 us, 5.5 TB/s.
template <int P, int QPT, int MT, int R, int U, int NW, int STEPS, bool BIG>
__global__ __launch_bounds__(NW * 64) void mx4_scores_kernel(Mx4ScoreArgs a) {
    typedef Mx4Tiles<P, QPT, MT> L;
    constexpr int QB = L::QB * R / 16, BLOCK = MT * R * 256, COLS = R / 4;
    constexpr bool LONG = BIG && QB <= 8;
    const int ks = STEPS ? U : a.ks, ksu = STEPS ? U : a.ksu;
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    uint8_t* frag = smem;
    float* inv = reinterpret_cast<float*>(frag + ksu * BLOCK);
    int* kexp = reinterpret_cast<int*>(inv + L::QB);

    // this wave takes the tiles of 16 rows first, first + stride, ... (LONG: four from each)
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    Mx4Work w;
    int first = wave, stride = NW;
    if (!a.items && a.nqb == 1) {
        w.row0 = a.row0; w.at = 0; w.ld = a.out_ld; w.rows = (int)a.rows; w.q0 = 0; w.nqh = a.nq;
        first = (int)blockIdx.x * NW + wave;
        stride = (int)gridDim.x * NW;
    } else if (!mx4_work(a, QB, w)) return;
    const int rows = w.rows, nqh = w.nqh;
    const long long ld = w.ld;
    if (LONG) first *= 4;
    const int n16 = lane & 15, col = lane >> 4;
    const int tiles = rows / 16 + (rows % 16 != 0);
    const int end = LONG ? (tiles + 3) & ~3 : tiles;
    const int sd = (ks + 3) / 4;                                // scale dwords of a lane per row
    float* out = a.out + w.at;

    constexpr int SW = (U + 3) / 4;                             // scale dwords per fetch
    struct Buf {
        v4i w[U];
        int s[SW];
    };
    const int l0 = (int)(w.row0 & 15) + n16;                    // tiles start at multiples of 16 from row0
    const int wo = (l0 >> 4) * 16 * a.code_ld + (l0 & 15) * 64 + col * 16, so = n16 * a.scale_ld + col * 4;
    constexpr int AUX = BIG ? 2 : 0;                            // 2: not to be kept in the caches
    auto load = [&](Buf& b, int tile, int ks0) {
        const Mx4Rows from(a, w.row0 + (long long)(tile < tiles ? tile : tiles - 1) * 16);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int k = STEPS || ks0 + u < ks ? ks0 + u : ks - 1;              // blocks past the row's meet zeros
            b.w[u] = __builtin_bit_cast(v4i, __builtin_amdgcn_raw_buffer_load_b128(from.codes, wo, k * 1024, AUX));
        }
#pragma unroll
        for (int d = 0; d < SW; ++d) {
            // (scales behind the row's are zero, here or in memory: those blocks' values are finite, and nothing beside zeros)
            const bool there = STEPS || (ks0 >> 2) + d < sd;
            b.s[d] = (int)__builtin_amdgcn_raw_buffer_load_b32(from.scales, there ? so : (int)MX4_NOWHERE, there ? ((ks0 >> 2) + d) * 16 : 0, 0);
        }
    };
    v4f acc[MT][1];
    auto multiply = [&](const Buf& b, int ks0, auto first_of_row) {
        constexpr bool FIRST = decltype(first_of_row)::value;   // begins the sums at zero
        const uint8_t* f = frag + ks0 * BLOCK;
        int at[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            at[i] = mx4_frag_at<R>(i, col, n16 & (R - 1));
            asm volatile("" : "+v"(at[i]));                     // fragments do not fit the registers: read from LDS each time
        }
        // query fragments AHEAD ones ahead: the LDS latency passes under the products before
        constexpr int AHEAD = 2, RING = AHEAD + 1, ALL = U * 4 * MT;
        v8bf x[RING];
        auto fetch = [&](auto ic) {
            constexpr int n = decltype(ic)::value, u = n / (4 * MT), i = n / MT % 4, mt = n % MT;
            x[n % RING] = *reinterpret_cast<const v8bf*>(f + u * BLOCK + mt * R * 256 + at[i]);
        };
        static_for<AHEAD>([&](auto ic) {
            if constexpr (decltype(ic)::value < ALL) fetch(ic);
        });
        v8bf y;
        static_for<ALL>([&](auto ic) {
            constexpr int n = decltype(ic)::value, u = n / (4 * MT), i = n / MT % 4, mt = n % MT;
            if constexpr (n + AHEAD < ALL) fetch(std::integral_constant<int, n + AHEAD>{});
            if constexpr (mt == 0) y = mx4_unpack(b.w[u][i], mx4_scale(b.s[u >> 2], u & 3));       // (a fetch begins with a scale dword)
            __builtin_amdgcn_sched_barrier(0);
            const v4f c = FIRST && u == 0 && i == 0 ? (v4f){0.f, 0.f, 0.f, 0.f} : acc[mt][0];
            acc[mt][0] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(x[n % RING], y, c, 0, 0, 0);
        });
    };
    float iv[L::SETS][L::SPL];
    unsigned place[L::SETS][L::SPL];                            // of this lane's score from the tile's first one; past the end where there is none
    float held[L::SETS][L::SPL][4];                             // LONG: the scores of the tiles since the last store
    auto total = [&](int set, int j) -> float {
        float y = mx4_sum<P, QPT, MT>(acc, set, 0, j) * iv[set][j];
        if constexpr (STEPS == 0) asm volatile("" : "+v"(y));   // here: else the products sink into the branch that asks whether a row is done
        return y;
    };
    auto store = [&](int tile) {
#pragma unroll
        for (int set = 0; set < L::SETS; ++set)
#pragma unroll
            for (int j = 0; j < L::SPL; ++j) {
                if constexpr (LONG) {
                    columns_transpose(held[set][j]);
                    const int r = (tile - 3) * 16, left = rows - r < 64 ? (rows - r) * 4 : 256;
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        const int query = set * QPT + j * COLS + c;
                        if (c < COLS) mx4_put(held[set][j][c], out + query * ld + r, query < nqh ? left : 0, lane * 4);
                    }
                } else {
                    const int r = tile * 16;
                    mx4_put(total(set, j), out + (set * QPT + j * COLS) * ld + r, 0x7fffffff, r + n16 < rows ? place[set][j] : MX4_NOWHERE);
                }
            }
    };

    Buf x, y;
    int t = first;
    load(x, t, 0);                                              // on its way while the queries are split
    mx4_stage_queries<P, QPT, MT, R, NW * 64>(a, static_cast<const char*>(a.q) + (size_t)w.q0 * a.ldq * (P == 3 ? 4 : 2), nqh, frag, inv, kexp);
    if (first >= end) return;
#pragma unroll
    for (int set = 0; set < L::SETS; ++set)
#pragma unroll
        for (int j = 0; j < L::SPL; ++j) {
            const int query = set * QPT + j * COLS + col % COLS;
            iv[set][j] = inv[query];
            place[set][j] = col < COLS && query < nqh ? (unsigned)(col * ld + n16) * 4u : MX4_NOWHERE;
        }
    auto hold = [&](auto sub) {
#pragma unroll
        for (int set = 0; set < L::SETS; ++set)
#pragma unroll
            for (int j = 0; j < L::SPL; ++j) held[set][j][decltype(sub)::value] = total(set, j);
    };
    if constexpr (STEPS == 1) {
        // pairs of tiles: x and y in turn (LONG: two pairs to a store)
        for (;;) {
            static_for<LONG ? 2 : 1>([&](auto pair) {
                constexpr int p = decltype(pair)::value * 2;
                const int t1 = LONG ? t + p + 1 : t + stride;
                const int t2 = LONG ? (p == 0 ? t + 2 : t + 4 * stride) : t + 2 * stride;
                load(y, t1, 0);
                __builtin_amdgcn_sched_barrier(0);              // the fetch goes out before the products wait for theirs
                multiply(x, 0, std::true_type{});
                if constexpr (LONG) hold(std::integral_constant<int, p>{});
                else store(t);
                if (!LONG && t1 >= end) return;
                load(x, t2, 0);
                __builtin_amdgcn_sched_barrier(0);
                multiply(y, 0, std::true_type{});
                if constexpr (LONG) hold(std::integral_constant<int, p + 1>{});
                else store(t1);
            });
            if constexpr (LONG) store(t + 3);
            t += LONG ? 4 * stride : 2 * stride;
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
                for (int set = 0; set < L::SETS; ++set)
#pragma unroll
                    for (int j = 0; j < L::SPL; ++j) {
                        held[set][j][0] = held[set][j][1];
                        held[set][j][1] = held[set][j][2];
                        held[set][j][2] = held[set][j][3];
                        held[set][j][3] = total(set, j);
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

// Many queries: MT tiles of them against NB blocks of 16 rows per wave, eight waves, block of 128 by block along the row.  A fragment
// serves NB row blocks, the four-bit values are unpacked once for MT tiles, and a query's scores of all NB blocks are stored together.
//
// WHOLE: the queries' parts of the whole row lie in LDS, and the waves go on without a barrier.  Where they do not fit, the workgroup
// makes the parts of the next block in one of two LDS buffers under the products of the present one, from elements fetched a block
// earlier: rows of any length take the same LDS, and one barrier a block stands against 4 MT NB products of every wave (256 fp32
// queries x 200k x 768: 181 us, 207 like this; fetched in the block before only: 241).
//
// What bounds it, 256 fp32 queries x 200k x 768 (2.4e14 operations on the three parts): 186 to 189 us, 1.3e15 operations a second; a large
// library product of bf16 matrices reaches as many on this card, the instruction alone 2.0e15.  With the products alone 131 us; all but the
// products 146; all but the stores 158, all but the fetch of rows 164, all but the fragments' LDS reads 179, all but the unpacking 185.  So the
// matrix unit (busy 55 % of the cycles), and stores and fetches that are not wholly hidden behind it: they share a counter, and behind the
// branch that asks whether a row is done the compiler waits for the stores.  Rows fetched two blocks ahead, fragments three to six
// ahead, and four row blocks to a fragment (184; where the parts are made on the way its registers spill) change nothing.  bf16 queries have a
// third of the products: 107 to 112 us, of which 205 MB of scores are 42.
template <int P, int QPT, int MT, int NB, bool WHOLE>
__global__ __launch_bounds__(512) void mx4_scores_many_kernel(Mx4ScoreArgs a) {
    typedef Mx4Tiles<P, QPT, MT> L;
    constexpr int QB = L::QB, NW = 8, NT = 512, R = 16, BLOCK = MT * R * 256, ESIZE = P == 3 ? 4 : 2;
    static_assert(NB <= 4, "up to four tiles' scores are stored together");
    constexpr int UNITS = QB * 16, UPT = (UNITS + NT - 1) / NT;  // units of eight elements of a block; of a thread
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    uint8_t* frag = smem;
    float* inv = reinterpret_cast<float*>(frag + (WHOLE ? a.ks : 2) * BLOCK);
    int* kexp = reinterpret_cast<int*>(inv + QB);
    Mx4Work w;
    if (!mx4_work(a, QB, w)) return;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n16 = lane & 15, col = lane >> 4, rows = w.rows, nqh = w.nqh, ks = a.ks;
    const long long ld = w.ld;
    const int tiles = rows / (16 * NB) + (rows % (16 * NB) != 0);
    float* out = a.out + w.at;
    const char* q = static_cast<const char*>(a.q) + (size_t)w.q0 * a.ldq * ESIZE;

    struct Buf {
        v4i w[NB];
        int s[NB];
    };
    const int l0 = (int)(w.row0 & 15) + n16;                    // tiles start at multiples of 16 from row0
    const int wo = (l0 >> 4) * 16 * a.code_ld + (l0 & 15) * 64 + col * 16, so = n16 * a.scale_ld + col * 4;
    auto load = [&](Buf& b, int tile, int k) __attribute__((always_inline)) {
        const Mx4Rows from(a, w.row0 + (long long)(tile < tiles ? tile : tiles - 1) * (16 * NB));
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
            b.w[nb] = __builtin_bit_cast(v4i, __builtin_amdgcn_raw_buffer_load_b128(from.codes, wo + nb * 16 * a.code_ld, k * 1024, 0));
            b.s[nb] = (int)__builtin_amdgcn_raw_buffer_load_b32(from.scales, so + nb * 16 * a.scale_ld, (k >> 2) * 16, 0);
        }
    };
    // the queries' units of block k: query u / 16 (an absent one: the last again), elements 8 (u % 16) of the block
    Mx4Raw<P> raw[UPT];
    auto fetch_queries = [&](int k) __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < UPT; ++j) {
            const int u = tid + j * NT, s = u >> 4 < nqh ? u >> 4 : nqh - 1;
            raw[j] = mx4_raw<P>(q + (size_t)s * a.ldq * ESIZE, k * 128 + (u & 15) * 8, a.dim);
        }
    };
    Mx4Split<P> parts[UPT];
    int scale[UPT];                                             // COSINE
    auto split_pair = [&](int i, auto scaled) __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < UPT; ++j) parts[j].template pair<decltype(scaled)::value>(raw[j], i, scale[j]);
    };
    auto put_queries = [&](uint8_t* to, auto scaled) __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < UPT; ++j) {
            const int u = tid + j * NT;
            parts[j].template finish<decltype(scaled)::value>(raw[j]);
            if (UNITS % NT == 0 || u < UNITS) parts[j].template store<QPT, MT, R>(u >> 4, u & 15, to);
        }
    };
    int at[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) at[i] = mx4_frag_at<R>(i, col, n16);
    v4f acc[MT][NB];
    auto clear = [&]() __attribute__((always_inline)) {
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) acc[mt][nb] = (v4f){0.f, 0.f, 0.f, 0.f};
    };
    auto multiply = [&](const Buf& b, int k, const uint8_t* f, auto meanwhile) __attribute__((always_inline)) {
        constexpr int AHEAD = 2, RING = AHEAD + 1, ALL = 4 * MT;
        v8bf x[RING], y[2][NB];
        float scale[NB];
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) scale[nb] = mx4_scale(b.s[nb], k & 3);
        auto fetch = [&](auto ic) __attribute__((always_inline)) {
            constexpr int n = decltype(ic)::value, i = n / MT, mt = n % MT;
            x[n % RING] = *reinterpret_cast<const v8bf*>(f + mt * R * 256 + at[i]);
        };
        static_for<AHEAD>([&](auto ic) { if constexpr (decltype(ic)::value < ALL) fetch(ic); });
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) y[0][nb] = mx4_unpack(b.w[nb][0], scale[nb]);
        static_for<ALL>([&](auto ic) {
            constexpr int n = decltype(ic)::value, i = n / MT, mt = n % MT;
            if constexpr (n + AHEAD < ALL) fetch(std::integral_constant<int, n + AHEAD>{});
            __builtin_amdgcn_sched_barrier(0);
            static_for<NB>([&](auto nbc) {
                constexpr int nb = decltype(nbc)::value;
                acc[mt][nb] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(x[n % RING], y[i & 1][nb], acc[mt][nb], 0, 0, 0);
                // the next step's values under these products, an even share to each tile
                if constexpr (i < 3 && nb * MT / NB == mt) y[(i + 1) & 1][nb] = mx4_unpack(b.w[nb][i + 1], scale[nb]);
            });
            meanwhile(ic);
            __builtin_amdgcn_sched_barrier(0);
        });
    };
    auto store = [&](int tile) __attribute__((always_inline)) {
        const int r = tile * (16 * NB), left = rows - r < 16 * NB ? (rows - r) * 4 : 64 * NB;
#pragma unroll
        for (int set = 0; set < L::SETS; ++set)
#pragma unroll
            for (int j = 0; j < L::SPL; ++j) {
                const float f = inv[set * QPT + j * 4 + col];
                float v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int nb = 0; nb < NB; ++nb) v[nb] = mx4_sum<P, QPT, MT>(acc, set, nb, j) * f;
                columns_transpose(v);
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    const int query = set * QPT + j * 4 + c;
                    mx4_put(v[c], out + query * ld + r, query < nqh ? left : 0, lane * 4);
                }
            }
    };

    Buf x, y;
    int t = wave, k = 0;
    load(x, t, 0);
    if constexpr (WHOLE) {
        mx4_stage_queries<P, QPT, MT, R, NT>(a, q, nqh, frag, inv, kexp);
        if (t >= tiles) return;
        clear();
        auto turn = [&](const Buf& now, Buf& next) -> bool {
            const int k2 = k + 1 < ks ? k + 1 : 0, t2 = k2 ? t : t + NW;
            load(next, t2, k2);
            __builtin_amdgcn_sched_barrier(0);
            multiply(now, k, frag + k * BLOCK, [](auto) {});
            if (!k2) {
                store(t);
                clear();
            }
            t = t2;
            k = k2;
            return t >= tiles;
        };
        for (;;) {
            if (turn(x, y)) break;
            if (turn(y, x)) break;
        }
    } else {
        // all waves of the workgroup take the same turns: those behind the last tile multiply it again and store nothing
        mx4_query_norms<P, QB, NT>(a, q, nqh, inv, kexp);
        auto run = [&](auto scaled) __attribute__((always_inline)) {
            int t0 = 0;
#pragma unroll
            for (int j = 0; j < UPT; ++j) {
                const int s = (tid + j * NT) >> 4;
                scale[j] = decltype(scaled)::value ? kexp[s < nqh ? s : nqh - 1] : 0;
            }
            fetch_queries(0);
#pragma unroll
            for (int i = 0; i < 4; ++i) split_pair(i, scaled);
            put_queries(frag, scaled);
            fetch_queries(ks > 1 ? 1 : 0);
            clear();
            __syncthreads();
            auto turn = [&](const Buf& now, Buf& next, const uint8_t* here, uint8_t* there) __attribute__((always_inline)) -> bool {
                const int k2 = k + 1 < ks ? k + 1 : 0, t2 = k2 ? t : t + NW;
                const bool last = !k2 && t0 + NW >= tiles;
                load(next, t2, k2);
                __builtin_amdgcn_sched_barrier(0);
                // the next block's queries, fetched a turn ago, are split under the second half of the products
                multiply(now, k, here, [&](auto ic) {
                    static_for<4>([&](auto pair) {
                        if constexpr (decltype(ic)::value == 2 * MT + decltype(pair)::value * MT / 2) split_pair(decltype(pair)::value, scaled);
                    });
                });
                put_queries(there, scaled);
                fetch_queries(k2 + 1 < ks ? k2 + 1 : 0);
                if (!k2) {
                    if (t < tiles) store(t);
                    clear();
                    t0 += NW;
                }
                t = t2;
                k = k2;
                __syncthreads();
                return last;
            };
            for (;;) {
                if (turn(x, y, frag, frag + BLOCK)) break;
                if (turn(y, x, frag + BLOCK, frag)) break;
            }
        };
        if (a.normalize) run(std::true_type{});
        else run(std::false_type{});
    }
}

template <typename K>
static int mx4_start(K kern, const Mx4ScoreArgs& a, long long grid, int threads, size_t lds, int device, bool (&attr_set)[64], hipStream_t s) {
    if (lds > 48 * 1024 && !attr_set[device & 63]) {            // per device: the attribute belongs to the device's code object
        RAG_HIP_CHECK(hipFuncSetAttribute(reinterpret_cast<const void*>(kern), hipFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024));
        attr_set[device & 63] = true;
    }
    hipLaunchKernelGGL(kern, dim3((unsigned)grid), dim3(threads), lds, s, a);
    RAG_HIP_CHECK(hipGetLastError());
    return RAG_OK;
}
template <int P, int QPT, int MT, int R, int U, int NW, int STEPS, bool BIG>
static int mx4_launch_few(const Mx4ScoreArgs& a, long long grid, size_t lds, int device, hipStream_t s) {
    static bool attr_set[64] = {};
    return mx4_start(mx4_scores_kernel<P, QPT, MT, R, U, NW, STEPS, BIG>, a, grid, NW * 64, lds, device, attr_set, s);
}
template <int P, int QPT, int MT, int NB, bool WHOLE>
static int mx4_launch_many(const Mx4ScoreArgs& a, long long grid, size_t lds, int device, hipStream_t s) {
    static bool attr_set[64] = {};
    return mx4_start(mx4_scores_many_kernel<P, QPT, MT, NB, WHOLE>, a, grid, 512, lds, device, attr_set, s);
}
#define MX4_CASE(P, QPT, MT, R, U, NW, STEPS) \
    if (!p.many && p.qpt == QPT && p.mt == MT && p.r == R && p.u == U && p.steps == STEPS) \
        return p.big ? mx4_launch_few<P, QPT, MT, R, U, NW, STEPS, true>(a, grid, p.lds, device, s) \
                     : mx4_launch_few<P, QPT, MT, R, U, NW, STEPS, false>(a, grid, p.lds, device, s)
#define MX4_FEW(P, QPT, MT) \
    MX4_CASE(P, QPT, MT, 16, 1, 4, 1); MX4_CASE(P, QPT, MT, 16, 2, 4, 1); MX4_CASE(P, QPT, MT, 16, 3, 4, 1); MX4_CASE(P, QPT, MT, 16, 4, 4, 1); \
    MX4_CASE(P, QPT, MT, 16, 6, 4, 1); MX4_CASE(P, QPT, MT, 16, 8, 4, 1); MX4_CASE(P, QPT, MT, 16, 4, 8, 0); MX4_CASE(P, QPT, MT, 16, 8, 8, 0)
#define MX4_MANY(P, QPT, MT, NB) \
    if (p.many && p.mt == MT && p.nb == NB) \
        return p.steps ? mx4_launch_many<P, QPT, MT, NB, true>(a, grid, p.lds, device, s) : mx4_launch_many<P, QPT, MT, NB, false>(a, grid, p.lds, device, s)

}  // namespace rag
