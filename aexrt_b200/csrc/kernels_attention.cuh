// Attention kernel selection across the translation units that instantiate the kernels.
#pragma once
#include <cuda.h>

#include "attention_common.cuh"

namespace aexrt {

using TcKernelFn = void (*)(const CUtensorMap, const CUtensorMap, const CUtensorMap, const AttnParams);
struct TcKernel {
  TcKernelFn fn;
  int smem;
};
// The tensor-core kernel (attention_tc.cuh): 16-bit type, packed or paged keys, head size 8 .. 128.
TcKernel attention_tc_for(bool bf16, bool paged, int head_dim);

// The kernel of a few rows (attention_rows.cuh; rows = most query tokens x heads per kv head, at most
// 64) and the launch that joins what it left in parts.
struct RowsParams;
struct RowsKernel {
  void (*fn)(const CUtensorMap, const CUtensorMap, const RowsParams);
  void (*join)(const RowsParams);
  int smem;
};
RowsKernel attention_rows_for(bool bf16, int head_dim, int rows);
constexpr int kTcBlock = 384, kTcTileRows = 128, kTcTileKeys = 128;

}  // namespace aexrt
