// What the kernels over the cache of 8-bit codes have in common.
#pragma once

#include "jf_common.cuh"

namespace jf {

// Blocks that a sequence's attention goes through, where they are not those of its table from the first to the last.
struct Block8Source {
  const int32_t* chosen = nullptr;   // (B, H_kv, top): numbers of the blocks, the first min(blocks, top) entries count
  int32_t top = 0;
  const void* shared = nullptr;      // ids of the blocks that come before those of the table, the same for all sequences
  int32_t shared_blocks = 0;
  bool shared_i32 = false;
  // Partial results of the positions before, which are joined with those of the table's blocks: lengths count `behind` blocks
  // that the table does not have.  Layout and geometry: block8_shared.cu.
  int32_t behind = 0;
  const float* part_o = nullptr;
  const float4* part_ml = nullptr;
  int64_t units = 0;
  int32_t grid = 0, tiles = 0, pairs = 0, row_tiles = 0;
};
// jf_block8_attn with such blocks; its checks only where `launch` is false.
jf_status_t block8_attend(const jf_block8_attn_args* a, const Block8Source& from, jf_stream_t stream, bool launch);
uint64_t block8_attn_workspace(int B, int H_q, int H_kv, int max_S);

__device__ __forceinline__ void mma_s8_16832(int (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

}  // namespace jf
