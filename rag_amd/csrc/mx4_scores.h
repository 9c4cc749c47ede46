// Products of queries with four-bit rows.  Instantiated for fp32 queries in mx4_scores_f32.hip, for bf16 and fp16 ones in
// mx4_scores_16.hip.
//
// Products run on the scaled matrix instruction, which reads four-bit values and their scales as they are stored: nothing
// is unpacked.  Its other operand is six bits wide (e2m3, scaled per 32 as well), so a query is split into digits first:
// with 2^E the power of two that brings the largest element of a group of 32 into [8, 16),
//     x = 2^E * (d0 + d1 / 32 + d2 / 32^2 + ...),   dj a whole number in [-16, 16],
// and a whole number up to 16 is exact in e2m3, as so many eighths (its code is the number itself, and 32 where it is
// negative).  With eight-bit digits the instruction takes twice as long and their fragments a third more of the LDS (256
// fp32 queries x 200k x 768: 154 us, 134 with six; x 2048: 613, 399).  Each digit is a row of the matrix tile of its own, with the scale
// 2^(E + 3 - 5j), so one instruction multiplies all digits; the digits' sums are added at the end.  fp32 queries take five
// digits (what is left is at most 2^-24 of the group's largest element), bf16 and fp16 four (at most 2^-19 of it: every
// element down to 2^-12 (bf16) / 2^-9 (fp16) of the largest one is exact).  Products of such digits with four-bit values
// are multiples of 1/2 up to 96, which the instruction adds without loss; it adds across groups and to the accumulator in
// fp32.  One query fills four or five of the tile's sixteen rows, so three (fp32) or four queries cost what one does.
#pragma once
#include "mx4_device.h"

namespace rag {

// Layout of the instruction (checked on the card): lane l, column c = l / 16.  Either operand: row l % 16, elements
// 32 c .. 32 c + 31 of the block of 128, and their scale.  Result register r of lane l: (row 4 c + r of the digits, row
// l % 16 of the store).
//
// Digit j < 4 of query s of a tile is row 4 s + j of the digits: the four registers of column s, added without leaving the lane.
// Fifth digits (fp32): up to three queries share their tile with them -- rows 12 + s: register s of column 3, fetched from
// there by fifth_digits().  More queries put four to a tile and have the fifth digits of each four tiles in one more tile, query s
// of tile t in row 4 s + t: register t of column s, where they are wanted.
template <int ND, int MT>
struct Mx4Digits {
    static constexpr bool INSIDE = ND == 5 && MT == 1;           // fifth digits in the tile itself
    static constexpr int EX = ND == 5 && !INSIDE ? (MT + 3) / 4 : 0;
    static constexpr int TILES = MT + EX;
    static constexpr int QPT = INSIDE ? 3 : 4;                   // queries per tile of 16 rows of digits
};

// Unit u of the queries at q, EL consecutive elements, into the fragments.  The conversions round to nearest even, so a digit is
// what a conversion makes of the rest, and the next rest is what is left of it, exactly.
template <int ND, int MT, int EL>
__device__ __forceinline__ void mx4_stage_unit(const Mx4ScoreArgs& a, const char* q, int u, uint8_t* frag, uint8_t* sc) {
    typedef Mx4Digits<ND, MT> L;
    constexpr int QPT = L::QPT, TILES = L::TILES, ESIZE = ND == 5 ? 4 : 2, SHARE = 32 / EL;
    typedef typename std::conditional<EL * ESIZE % 16 == 0, v4i_apart, v2i_apart>::type Raw;
    constexpr int PIECES = EL * ESIZE / sizeof(Raw), DW = sizeof(Raw) / 4;
    // s: the query; its group of 32 elements; the lane's part `in` of that
    const int ug = u / SHARE, in = u % SHARE, s = (int)__umulhi((unsigned)ug, a.per), group = ug - s * a.ks * 4, at0 = group * 32 + in * EL;
    const char* row = q + (size_t)s * a.ldq * ESIZE;
    float v[EL];
    if (at0 + EL <= a.dim) {
        Raw raw[PIECES];
#pragma unroll
        for (int j = 0; j < PIECES; ++j) raw[j] = reinterpret_cast<const Raw*>(row + (size_t)at0 * ESIZE)[j];
#pragma unroll
        for (int j = 0; j < EL; ++j) {
            if constexpr (ND == 5) v[j] = __int_as_float(raw[j / DW][j % DW]);
            else {
                const unsigned w = (unsigned)raw[j / 2 / DW][j / 2 % DW], h = j & 1 ? w >> 16 : w & 0xffffu;
                v[j] = a.q_type == RAG_MX4_BF16 ? bf16_f32(h) : f16_f32((unsigned short)h);
            }
        }
    } else {                                                    // the end of a row: zeros behind it
        typedef typename std::conditional<ND == 5, float, unsigned short>::type Elem;
        Elem raw[EL];
#pragma unroll
        for (int j = 0; j < EL; ++j) raw[j] = reinterpret_cast<const Elem*>(row)[at0 + j < a.dim ? at0 + j : a.dim - 1];
#pragma unroll
        for (int j = 0; j < EL; ++j) {
            if constexpr (ND == 5) v[j] = raw[j];
            else v[j] = a.q_type == RAG_MX4_BF16 ? bf16_f32(raw[j]) : f16_f32(raw[j]);
            v[j] = at0 + j < a.dim ? v[j] : 0.f;
        }
    }
    unsigned most = 0;
#pragma unroll
    for (int j = 0; j < EL; ++j) {
        const unsigned m = __float_as_uint(v[j]) & 0x7fffffffu;
        most = m > most ? m : most;
    }
    if constexpr (SHARE == 8) most = oct_max(most);
    const bool bad = most >= 0x7f800000u;
    int e = (int)(most >> 23) - 130;                            // the largest element / 2^e lies in [8, 16)
    e = e < -100 ? -100 : e;                                    // (a group below 2^-97 has its digits cut instead)
    e = bad ? 0 : e;
    const float down = mx4_pow2(-e);
    const int block = group >> 2, col = group & 3;
    const int tile = s / QPT, slot = s - tile * QPT;
    uint8_t* to = frag + block * mx4_frag_ld(TILES);
    uint8_t* ts = sc + (size_t)((block >> 2) * TILES) * 256 + col * 64 + (block & 3);
#pragma unroll
    for (int j = 0; j < EL; ++j) v[j] *= down;
#pragma unroll
    for (int d = 0; d < ND; ++d) {
        const int m = d < 4 ? 4 * slot + d : L::INSIDE ? 12 + slot : 4 * slot + (tile & 3);
        const int at = d < 4 || L::INSIDE ? tile : MT + (tile >> 2);
        const int place = col * 16 + (m ^ col);
        uint8_t* first = to + at * MX4_FRAG + place * 16;
        uint8_t* last = to + at * MX4_FRAG + 1024 + place * 8;
        if constexpr (EL == 32) {
            const float unit = mx4_pow2(3 - 5 * d);              // six-bit values are eighths
            v16f even, odd;                                     // of the pairs that the conversion interleaves
#pragma unroll
            for (int j = 0; j < 16; ++j) { even[j] = v[2 * j]; odd[j] = v[2 * j + 1]; }
            const v6u p = __builtin_amdgcn_cvt_scalef32_2xpk16_fp6_f32(even, odd, unit);
            *reinterpret_cast<v4i*>(first) = (v4i){(int)p[0], (int)p[1], (int)p[2], (int)p[3]};
            *reinterpret_cast<v2u*>(last) = (v2u){p[4], p[5]};
            if (d + 1 < ND) {
                const v32f w = __builtin_amdgcn_cvt_scalef32_pk32_f32_fp6(p, unit);
#pragma unroll
                for (int j = 0; j < 32; ++j) v[j] -= w[j];
            }
        } else {
            // by way of e4m3, whose lowest values (multiples of 2^-9, up to 16 of them) are sign and magnitude too
            const float unit = mx4_pow2(9 - 5 * d);
            v2s b = {0, 0};
            b = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(b, v[0], v[1], unit, false);
            b = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(b, v[2], v[3], unit, true);
            const unsigned x = __builtin_bit_cast(unsigned, b);
            if (d + 1 < ND) {
                const v2f lo = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(x, unit, false), hi = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(x, unit, true);
                v[0] -= lo.x; v[1] -= lo.y; v[2] -= hi.x; v[3] -= hi.y;
            }
            // four codes in 24 bits; four lanes make three dwords of them
            const unsigned y = (x & 0x1f1f1f1fu) | ((x >> 2) & 0x20202020u);
            const unsigned p = __builtin_amdgcn_udot4(y, 0x4001u, 0u, false) | __builtin_amdgcn_udot4(y, 0x40010000u, 0u, false) << 12;
            const unsigned next = (unsigned)__builtin_amdgcn_update_dpp(0, (int)p, 0xF9, 0xF, 0xF, true);      // of the lane behind this one
            const int k = in & 3, n = 3 * (in >> 2) + k;         // dword of the lane's six
            if (k < 3) *reinterpret_cast<unsigned*>(n < 4 ? first + 4 * n : last + 4 * (n - 4)) = p >> 8 * k | next << (24 - 8 * k);
        }
        // NaN: every score of the query is NaN
        if (in == 0) ts[at * 256 + m * 4] = bad && d == 0 ? 255 : (uint8_t)(130 + e - 5 * d);
    }
}

// queries [q0, q0 + nqh) -> digit fragments in LDS, 1536 bytes per block and tile: the first sixteen bytes of every lane, then the
// last eight of every lane.  Behind them the scales sc[(block / 4) * TILES + tile][lane][block % 4], then 1 / |q|.  Blocks past the
// row's are zero: they meet a real block of the row again.  A lane's place is its row number exclusive-or'ed with the column,
// and blocks lie 64 bytes more than their size apart, so that the lanes that write one digit of consecutive elements meet different
// banks.  What the fragments of absent queries hold does not matter: it stays in result rows that nobody reads.
template <int ND, int MT, int NT>
__device__ __forceinline__ void mx4_stage_queries(const Mx4ScoreArgs& a, long long q0, int nqh, uint8_t* frag, uint8_t* sc, float* inv) {
    typedef Mx4Digits<ND, MT> L;
    constexpr int QPT = L::QPT, TILES = L::TILES;
    const int tid = threadIdx.x;
    if (a.ksu > a.ks) {
        const v4i zero = {0, 0, 0, 0};
        v4i* f = reinterpret_cast<v4i*>(frag + a.ks * mx4_frag_ld(TILES));
        for (int i = tid; i < (a.ksu - a.ks) * (mx4_frag_ld(TILES) / 16); i += NT) f[i] = zero;
        v4i* s = reinterpret_cast<v4i*>(sc + (size_t)(a.ks / 4) * TILES * 256);
        for (int i = tid; i < ((a.ksu + 3) / 4 - a.ks / 4) * TILES * 16; i += NT) s[i] = zero;
        __syncthreads();
    }
    constexpr int ESIZE = ND == 5 ? 4 : 2;
    const char* q = static_cast<const char*>(a.q) + (size_t)q0 * a.ldq * ESIZE;
    for (int s = tid >> 6; s < MT * QPT; s += NT / 64) {
        float f = 1.f;
        if (a.normalize && s < nqh) f = wave_inv_norm(q + (size_t)s * a.ldq * ESIZE, a.q_type, a.dim, tid & 63);
        if ((tid & 63) == 0) inv[s] = f;
    }
    // A group of 32 elements to a lane is the least work (32 fp32 queries x 10k x 768: 7.7 us, 11.0 with four elements to a lane);
    // where there are so few that the lanes take only part of one each, it is the sum of their latencies that counts
    const int groups = nqh * a.ks * 4;
    if (MT <= 2 && groups * 8 <= NT) {
        if (tid < groups * 8) mx4_stage_unit<ND, MT, 4>(a, q, tid, frag, sc);
    } else {
        for (int u = tid; u < groups; u += NT) mx4_stage_unit<ND, MT, 32>(a, q, u, frag, sc);
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
// wait for all of them at every turn, stores too (branches around the stores cost 2.5 % of 256 fp32 queries x 200k x 768).
//
// BIG, for stores that no cache keeps: rows are fetched past them (4M x 768, one query: 303 -> 260 us), and where up to 8
// queries meet a row a wave takes four tiles of sixteen rows in a row and stores their scores together, 256 contiguous bytes
// per query instead of 64 (one query 265 -> 260, eight 320 -> 306).
//
// Where it stands.  Few queries: bound by HBM.  4M x 768, one query: 258 us, 6.4 TB/s of rows, scales and scores; reading the same
// rows alone takes 220 us (7.0 TB/s), and with one 256-byte store per 24 KB 236 to 247.  16 bf16 queries x 1M x 1024: 107 us, 5.7 TB/s.
// Many queries: 256 fp32 queries x 200k x 768: 128 us, 3.1e15 digit operations a second of the 8.6e15 that the instruction alone
// reaches; 105 without its stores and with the rows in the nearest cache.  The matrix unit is busy a third of the time and the
// LDS, whose fragments serve NB row blocks each, for three quarters by its bytes; three or four row blocks to a fragment need
// more registers than two waves to a SIMD have (four waves a workgroup with four blocks: the same time; half as many queries with
// two to four blocks: 176 to 180 us), fragments fetched three or four tiles ahead change nothing.  The longest rows
// lose most: 256 queries x 100k x 4096 546 us, since the fragments of 8 queries are all that the LDS holds.
template <int ND, int MT, int NB, int U, int NW, int STEPS, bool BIG>
__global__ __launch_bounds__(NW * 64) void mx4_scores_kernel(Mx4ScoreArgs a) {
    typedef Mx4Digits<ND, MT> L;
    constexpr int QPT = L::QPT, TILES = L::TILES, QB = MT * QPT;
    constexpr bool LONG = BIG && MT <= 2;
    static_assert(!LONG || NB == 1, "four tiles of one row block each are stored together");
    const int ks = STEPS ? STEPS * U : a.ks, ksu = STEPS ? STEPS * U : a.ksu;
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    uint8_t* frag = smem;
    uint8_t* sc = frag + ksu * mx4_frag_ld(TILES);
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
        const uint8_t* f = frag + ks0 * mx4_frag_ld(TILES);
        int fl = (col * 16 + (n16 ^ col)) * 16, fh = 1024 + fl / 2, sl = lane * 4;
        if constexpr (TILES > 1) asm volatile("" : "+v"(fl), "+v"(fh), "+v"(sl));      // more than one tile's fragments do not fit the registers: read from LDS each time
        // query fragments AHEAD tiles ahead: the LDS latency passes under the products of the tiles before
        constexpr int AHEAD = 2, RING = AHEAD + 1;
        v4i lo[RING];
        v2u hi[RING];
        // scales: a dword covers four blocks, and is kept over them where it is not replaced before its last use (256 fp32 queries x
        // 200k x 1536: 297 us, 283 like this)
        constexpr bool KEEP = TILES > AHEAD;
        int xs[KEEP ? TILES : RING];
        auto fetch = [&](auto ic) {
            constexpr int i = decltype(ic)::value, u = i / TILES, mt = i % TILES;
            lo[i % RING] = *reinterpret_cast<const v4i*>(f + u * mx4_frag_ld(TILES) + mt * MX4_FRAG + fl);
            hi[i % RING] = *reinterpret_cast<const v2u*>(f + u * mx4_frag_ld(TILES) + mt * MX4_FRAG + fh);
            if constexpr (!KEEP || u == 0 || (!SHIFT && ((K0 + u) & 3) == 0)) {
                const int x = *reinterpret_cast<const int*>(sc + (size_t)(((ks0 + (SHIFT ? 0 : u)) >> 2) * TILES + mt) * 256 + sl);
                xs[KEEP ? mt : i % RING] = SHIFT ? (int)((unsigned)x >> ((ks0 & 3) * 8)) : x;
            }
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
            const v4i l = lo[i % RING];
            const v8i x = {l.x, l.y, l.z, l.w, (int)hi[i % RING].x, (int)hi[i % RING].y, 0, 0};        // (24 bytes: the rest is not read)
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) {
                const v8i y = __builtin_shufflevector(b.w[nb][u], b.w[nb][u], 0, 1, 2, 3, -1, -1, -1, -1);
                const v4f c = FIRST && u == 0 ? (v4f){0.f, 0.f, 0.f, 0.f} : acc[mt][nb];
                acc[mt][nb] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(x, y, c, 2, 4, kk & 3, xs[KEEP ? mt : i % RING], kk & 3,
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
                const int r = (tile - 3) * 16, left = rows - r < 64 ? (rows - r) * 4 : 256;
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
    MX4_CASE(MT, 1, 1, 4, 1); MX4_CASE(MT, 1, 2, 4, 1); MX4_CASE(MT, 1, 3, 4, 1); MX4_CASE(MT, 1, 4, 4, 1); MX4_CASE(MT, 1, 6, 4, 1); \
    MX4_CASE(MT, 1, 8, 4, 1); MX4_CASE(MT, 1, 4, 8, 0); MX4_CASE(MT, 1, 8, 8, 0)
    MX4_FEW(1);
    MX4_FEW(2);
    MX4_CASE(4, 1, 3, 8, 1); MX4_CASE(4, 1, 2, 8, 2); MX4_CASE(4, 1, 3, 8, 2); MX4_CASE(4, 1, 4, 8, 2);
    MX4_CASE(4, 1, 1, 8, 0); MX4_CASE(4, 1, 2, 8, 0); MX4_CASE(4, 1, 4, 8, 0);
    MX4_CASE(8, 2, 3, 8, 1); MX4_CASE(8, 2, 2, 8, 2); MX4_CASE(8, 2, 3, 8, 2); MX4_CASE(8, 2, 1, 8, 0); MX4_CASE(8, 2, 2, 8, 0);
#undef MX4_FEW
#undef MX4_CASE
    return fail(RAG_ERR_INVALID, "internal: no four-bit product kernel for this shape");
}

}  // namespace rag
