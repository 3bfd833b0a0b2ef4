// What the two kernels of the attention of a chunk (chunk_attention.cu: many rows, chunk_attention_few.cu: few) have in common: the call, the workspace with the parts
// of blocks that are cut, and how the work is cut. The products of all blocks (rows of a sequence and a key/value head, tiles of keys) lie in one line, sequence by sequence, head by head.
#pragma once
#include <stdint.h>

#include "ptx.cuh"

namespace omc {

typedef __nv_bfloat16 bf16;

constexpr int kCaKeys = 64;   // keys of a tile: blocks are cut between tiles

struct ChunkArgs {
  const bf16* q;
  long long ldq;
  const bf16* pool;        // [n_pages][2][Hkv][page_size][D]
  const int32_t* table;    // [n_seq][max_pages]
  const int32_t* cu;       // [n_seq + 1]
  const int32_t* ctx;      // [n_seq]
  bf16* out;
  long long ldo;
  int n_seq, T, max_new, max_ctx, n_pages, max_pages, page_size, page_shift, cluster, Hq, Hkv;
  float scale_log2;
  int wide;                // out is on 32-byte boundaries, its rows too
  int4* head;              // workspace: [CTAs] (parts of the block that is cut behind this CTA or 0, first row of q, first row of the block, rows | key/value head << 16)
  float2* ml;              // [2 CTAs][part_rows] maximum (base 2, scaled) and sum
  float4* part;            // [2 CTAs][D / 4][part_rows]: the threads of a warp have neighbouring rows
  int part_rows;
  unsigned int* failed;
};

struct CaPlan {
  int grid, part_rows;
  int cluster, warps;      // of few rows: CTAs that share a block (0: the line is cut), and their warps
  bool few;                // chunk_attention_few.cu has it
  bool cut, fits;          // whether a block can be cut; whether the products can be counted in 31 bits
  long long blocks, bytes; // at most as many blocks; of the workspace
};
// Few rows: whether the call is one, with its plan, and the launches.
bool few_plan(int n_seq, int Hkv, long long rows, long long tiles, int head_dim, CaPlan& p);
int few_launch(const ChunkArgs& a, const CaPlan& plan, int head_dim, cudaStream_t st);
// Joins the parts of blocks that were cut (chunk_attention.cu).
int chunk_join(const ChunkArgs& a, const CaPlan& plan, int head_dim, cudaStream_t st);

__device__ __forceinline__ int ca_warp_scan(int v, int lane) {   // inclusive
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int up = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += up;
  }
  return v;
}
__device__ __forceinline__ float ca_ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// The maximum keeps a NaN, which then is the row's reference.
__device__ __forceinline__ float ca_max3(float a, float b, float c) {
  float d;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

}  // namespace omc
