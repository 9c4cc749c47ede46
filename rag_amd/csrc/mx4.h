// A store of rows kept at four bits: its layout in device memory and the kernels' argument blocks.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace rag {

// A row of `dim` elements is padded with zeros to ks = ceil(dim / 128) blocks of 128 (four steps of the
// matrix instruction): 64 bytes, element 2j in the low half of byte j, 2j + 1 in the high half.  codes: sixteen rows lie together,
// block by block -- [row / 16][block][row % 16][64 bytes] -- so that one load of a wave (a block of sixteen rows) is one
// contiguous KiB: 4M rows of 768 against one query 292 us with the rows one behind the other, 264 us like this.
// scales: row after row, one byte per group of 32; the bytes of four consecutive blocks lie together per group column, so that the lane
// that feeds group column g of a row fetches the scales of four blocks as one dword:
//     group G of a row (block G / 4, column G % 4)  ->  byte (G / 16) * 16 + (G % 4) * 4 + (G / 4) % 4
__host__ __device__ __forceinline__ int mx4_blocks(int dim) { return (dim + 127) / 128; }
__host__ __device__ __forceinline__ int mx4_code_bytes(int dim) { return mx4_blocks(dim) * 64; }
__host__ __device__ __forceinline__ int mx4_scale_bytes(int dim) { return (mx4_blocks(dim) + 3) / 4 * 16; }
__host__ __device__ __forceinline__ size_t mx4_code_at(long long row, int code_ld, int block) {
    return (size_t)(row >> 4) * 16 * code_ld + (size_t)block * 1024 + (row & 15) * 64;
}
__host__ __device__ __forceinline__ int mx4_scale_at(int group) { return (group >> 4) * 16 + (group & 3) * 4 + ((group >> 2) & 3); }

constexpr int MX4_MAX_DIM = 8192;          // eight rows of query parts (2 KiB per block of 128) fit the LDS

// One piece of the grouped product: `nq` queries from q0 against `rows` rows from row0; score (i, r) goes to
// out[at + i * ld + r].  Written by rag_mx4_plan_groups, read by the kernel.
struct Mx4Item {
    long long row0;
    long long at;
    int rows;
    int ld;
    int q0;
    int nq;
};
static_assert(sizeof(Mx4Item) == 32, "RAG_MX4_ITEM_BYTES");

struct Mx4ScoreArgs {
    const uint8_t* codes;        // of the store's first row
    const uint8_t* scales;
    const void* q;
    long long ldq;               // elements
    int dim, ks, ksu, code_ld, scale_ld, normalize;
    unsigned per;                        // ceil(2^32 / (16 ks)): the query of a unit of 8 elements by a multiplication
    size_t code_bytes, scale_bytes;      // of the whole store
    float* out;
    // grouped: one workgroup per item
    const Mx4Item* items;
    // dense: rows [row0, row0 + rows) cut into slabs, every slab against blocks of QB queries
    long long row0, rows, slab, slabs, out_ld;
    long long total;             // grouped: scores in out (and rows = the store's)
    int nq, nqb;
};

// Which kernel a product takes (mx4_scores.h): from the queries that meet a row, and the row's length.
struct Mx4Shape {
    bool many;                   // the kernel for many queries; else the one for few
    int qpt, mt, nb, r, u, nw, steps, ksu;
    int qb;                      // queries of a workgroup
    bool big;
    size_t lds;
};
int mx4_launch_f32(const Mx4Shape& p, const Mx4ScoreArgs& a, long long grid, int device, hipStream_t s);      // mx4_scores_f32.hip
int mx4_launch_bf16(const Mx4Shape& p, const Mx4ScoreArgs& a, long long grid, int device, hipStream_t s);     // mx4_scores_bf16.hip
int mx4_launch_f16(const Mx4Shape& p, const Mx4ScoreArgs& a, long long grid, int device, hipStream_t s);      // mx4_scores_f16.hip

}  // namespace rag
