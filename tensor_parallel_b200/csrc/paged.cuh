// Shared by the kernels of a paged cache: what a sequence of the batch comes to, and the tensor maps over the pages.
//
// A cache holds keys and values as [pages][kv_heads][page_size][head_dim]; key j of a sequence is slot j % page_size of page table[sequence][j / page_size].
// The batch is ragged: the new tokens of sequence s are the rows starts[s] .. starts[s + 1] of the queries, behind past[s] cached ones.  Lengths and
// table live in device memory and change from step to step under a captured graph, so every kernel checks what it reads of them: a sequence that
// does not fit the rows, the table or the cache is recorded as STATUS_BAD_ARG and answered with NaN (append: its tokens are not stored), and nothing is read or written through its entries.
#pragma once
#include <cuda_bf16.h>
#include <limits.h>
#include <stdint.h>

#include "attention_sm100.cuh"
#include "ptx_sm100.cuh"
#include "tpb_api.h"

namespace tpb {

struct PagedBatch {
  const int* starts;
  const int* past;
  const int* table;
  long long table_ld;
  int n, tokens, table_width, pages, page_shift;
  int most_new;  // more new tokens than this are an error
  uint32_t* status;
};

struct PagedSequence {
  int token0, fresh, past;
  bool bad;  // its rows are [token0, token0 + fresh) all the same
};

__device__ __forceinline__ PagedSequence paged_sequence(const PagedBatch& b, int s) {
  const int a = __ldg(b.starts + s), e = __ldg(b.starts + s + 1), past = __ldg(b.past + s);
  PagedSequence q;
  q.token0 = min(max(a, 0), b.tokens);
  q.fresh = min(max(e, q.token0), b.tokens) - q.token0;
  q.past = past;
  q.bad = q.token0 != a || q.token0 + q.fresh != e || past < 0 || q.fresh > b.most_new ||
          (q.fresh > 0 && (long long)past + q.fresh > ((long long)b.table_width << b.page_shift)) || (long long)past + q.fresh > INT_MAX - 256;
  return q;
}

// A cache whose slots TMA can read: head_dim contiguous, the other strides multiples of 16 bytes.  Box: 64 elements of `rows` slots of one page.
static int paged_tmap(CUtensorMap* map, const void* ptr, int head_dim, int page_size, int kv_heads, int pages, long long s_slot, long long s_head, long long s_page,
                      int rows) {
  return fa_tmap(map, ptr, head_dim, rows, page_size, kv_heads, pages, s_slot, s_head, s_page);
}

// The same, a box holding all of head_dim, 64 elements of every slot behind those of the one in front, in blocks: half as many boxes at head_dim 128 (a warp
// issues one in 70 ns, of pages of 16 slots 16 for 64 keys).
static int paged_blocks_tmap(CUtensorMap* map, const void* ptr, int head_dim, int page_size, int kv_heads, int pages, long long s_slot, long long s_head,
                             long long s_page, int rows) {
  EncodeTiledFn fn = fa_encode_fn();
  if (!fn) return TPB_ERR_DRIVER;
  const cuuint32_t blocks = cuuint32_t(head_dim / 64);
  cuuint64_t dims[5] = {64, cuuint64_t(page_size), blocks, cuuint64_t(kv_heads), cuuint64_t(pages)};
  // a dimension of extent 1 may come with any stride: give it a legal one
  cuuint64_t strides[4] = {cuuint64_t(page_size > 1 ? s_slot : head_dim) * 2, 128, cuuint64_t(kv_heads > 1 ? s_head : head_dim) * 2, cuuint64_t(pages > 1 ? s_page : head_dim) * 2};
  cuuint32_t box[5] = {64, cuuint32_t(rows), blocks, 1, 1}, estr[5] = {1, 1, 1, 1, 1};
  return fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 5, const_cast<void*>(ptr), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS
             ? TPB_OK
             : TPB_ERR_TMAP;
}

// Query rows [tokens][heads][head_dim] (strides positive where there are several); box: 64 elements, the heads of a group, `tokens_of_box` tokens.
static int paged_rows_tmap(CUtensorMap* map, const void* ptr, int head_dim, int heads, int tokens, long long s_head, long long s_token, int group, int tokens_of_box) {
  EncodeTiledFn fn = fa_encode_fn();
  if (!fn) return TPB_ERR_DRIVER;
  cuuint64_t dims[3] = {cuuint64_t(head_dim), cuuint64_t(heads), cuuint64_t(tokens)};
  cuuint64_t strides[2] = {cuuint64_t(heads > 1 ? s_head : head_dim) * 2, cuuint64_t(tokens > 1 ? s_token : head_dim) * 2};
  cuuint32_t box[3] = {64, cuuint32_t(group), cuuint32_t(tokens_of_box)}, estr[3] = {1, 1, 1};
  return fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(ptr), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS
             ? TPB_OK
             : TPB_ERR_TMAP;
}

}  // namespace tpb
