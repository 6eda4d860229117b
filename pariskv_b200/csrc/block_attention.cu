// Attention over listed blocks of the cache.
#include "attend.cuh"

using namespace pk;

extern "C" int64_t pk_block_attention_workspace_bytes(int64_t, int64_t, int64_t, int64_t, int64_t, int64_t) { return attend_few_workspace(); }

extern "C" int pk_block_attention(const pk_tensor* queries, const pk_tensor* keys, const pk_tensor* values, const pk_tensor* blocks,
                                  const pk_tensor* lengths, int64_t block, float scale, const pk_tensor* out, const pk_tensor* lse,
                                  void* workspace, int64_t workspace_bytes, void* stream) {
  AttendParams p = {};
  if (const int rc = fill_attend(&p, queries, keys, values, lengths, scale, out, lse)) return rc;
  PK_CHECK_TENSOR(blocks, PK_I32, 4);
  const int64_t bs = queries->shape[0];
  PK_REQUIRE(block == 16 || block == 32 || block == 64 || block == 128, "block must be 16, 32, 64 or 128");
  PK_REQUIRE(blocks->shape[0] == bs && blocks->shape[1] == p.T && blocks->shape[2] == p.H && is_contig(blocks), "blocks must be contiguous i32 [bs,T,H,n]");
  PK_REQUIRE(blocks->shape[3] >= 1 && blocks->shape[3] * block <= (1 << 24), "between one block and 2^24 keys a list");
  p.blocks = (const int32_t*)blocks->data, p.n = (int)blocks->shape[3], p.block = (int)block;
  if (bs == 0 || p.T == 0) return PK_OK;
  if (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 255) || workspace_bytes < attend_few_workspace())
    return fail(PK_ERR_WORKSPACE, "block_attention: workspace missing, misaligned or too small");
  return launch_attend_few(p, bs, workspace, "block_attention", (cudaStream_t)stream);
}
