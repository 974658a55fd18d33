// Decode attention of sequences that share their first positions, over the 8-bit cache.
#include "block8.cuh"

#include <algorithm>

extern "C" uint64_t jf_block8_shared_workspace_bytes(int32_t B, int32_t H_q, int32_t H_kv, int32_t max_S, int32_t shared_blocks) {
  if (shared_blocks < 0) return 0;
  return jf::block8_attn_workspace(B, H_q, H_kv, max_S);
}

extern "C" jf_status_t jf_block8_shared_attn(const jf_block8_shared_args* a, jf_stream_t stream) {
  using namespace jf;
  if (!a) return JF_ERR_ARG;
  const jf_block8_attn_args& at = a->attn;
  if (a->shared_blocks < 0 || at.window != 0 || at.prefix_lens || at.alibi_slopes) return JF_ERR_ARG;
  if (a->shared_blocks > INT32_MAX / JF_BLOCK_SIZE - 1) return JF_ERR_UNSUPPORTED;
  if (at.B > 0 && a->shared_blocks > 0 && !a->shared_table) return JF_ERR_ARG;
  Block8Source from;
  from.shared = a->shared_table;
  from.shared_blocks = a->shared_blocks;
  from.shared_i32 = a->shared_is_i32 != 0;
  return block8_attend(&at, from, stream, true);
}
