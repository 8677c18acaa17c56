// Attention kernel selection across the translation units that instantiate the kernels.
#pragma once
#include <cuda.h>

#include "attention_common.cuh"

namespace aexrt {

struct TcSplit;
struct TcKernel {
  void (*fn)(const CUtensorMap, const CUtensorMap, const CUtensorMap, const AttnParams, const TcSplit);
  void (*join)(const AttnParams, const TcSplit);
  int smem;
};
// The tensor-core kernel (attention_tc.cuh): 16-bit type, packed or paged keys, head size 8 .. 128; and the launch
// that joins split items.
TcKernel attention_tc_for(bool bf16, bool paged, bool split, int head_dim);

// The kernel of a few rows (attention_rows.cuh; rows = most query tokens x heads per kv head, at most
// 64) and the launch that joins what it left in parts.
struct RowsParams;
struct RowsKernel {
  void (*fn)(const CUtensorMap, const CUtensorMap, const RowsParams);
  void (*join)(const RowsParams);
  int smem;
};
RowsKernel attention_rows_for(bool bf16, int head_dim, int rows);

}  // namespace aexrt
