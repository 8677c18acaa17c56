// C ABI of attention over token sequences, its paged cache and tables (include/aexrt_b200.h):
// checks of the description, launch shapes and the launches.
#include <cuda.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdarg>
#include <cstdio>
#include <mutex>

#include "../../include/aexrt_b200.h"
#include "attention_rows.cuh"
#include "attention_tc.cuh"
#include "kernels_attention.cuh"
#include "kv_cache.cuh"
#include "launch.cuh"

namespace aexrt {
void set_last_error(const char* msg);
bool encode_tensor_map(CUtensorMap* map, CUtensorMapDataType dt, int rank, const void* base, const uint64_t* dims,
                       const uint64_t* strides_bytes, const uint32_t* box, CUtensorMapSwizzle swizzle);
}

using namespace aexrt;

namespace {

int fail(const char* fmt, ...) {
  char buf[512];
  va_list ap;
  va_start(ap, fmt);
  std::vsnprintf(buf, sizeof(buf), fmt, ap);
  va_end(ap);
  set_last_error(buf);
  return 0;
}

bool cuda_ok(cudaError_t e, const char* what) {
  if (e == cudaSuccess) return true;
  fail("%s: %s", what, cudaGetErrorString(e));
  return false;
}

bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

static __device__ uint32_t g_attention_status[2];  // the status word, and what the last read took out of it

// Reads and clears in one step: bits set meanwhile are neither lost nor seen twice.
__global__ void take_status_kernel(uint32_t* word) { word[1] = atomicExch(word, 0u); }

// This device's status word, its address resolved once per device.
uint32_t* status_word() {
  static std::mutex mu;
  static uint32_t* word[128] = {};
  int dev = 0;
  if (!cuda_ok(cudaGetDevice(&dev), "cudaGetDevice")) return nullptr;
  if (dev < 0 || dev >= 128) {
    fail("device index %d out of range", dev);
    return nullptr;
  }
  std::lock_guard<std::mutex> lock(mu);
  if (!word[dev]) {
    void* ptr = nullptr;
    if (!cuda_ok(cudaGetSymbolAddress(&ptr, g_attention_status), "cudaGetSymbolAddress")) return nullptr;
    word[dev] = static_cast<uint32_t*>(ptr);
  }
  return word[dev];
}

// Raises a kernel's dynamic shared memory limit, once per kernel and device.
bool raise_smem(const void* fn, int bytes) {
  struct Raised {
    const void* fn;
    int dev;
  };
  static std::mutex mu;
  static Raised raised[512];
  static int count = 0;
  int dev = 0;
  if (!cuda_ok(cudaGetDevice(&dev), "cudaGetDevice")) return false;
  std::lock_guard<std::mutex> lock(mu);
  for (int i = 0; i < count; ++i)
    if (raised[i].fn == fn && raised[i].dev == dev) return true;
  if (!cuda_ok(cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes), "cudaFuncSetAttribute"))
    return false;
  if (count < 512) raised[count++] = Raised{fn, dev};
  return true;
}

int log2_exact(uint32_t x) {
  int s = 0;
  while ((1u << s) < x) ++s;
  return s;
}

constexpr uint64_t kMaxStride = 1ull << 38;  // elements: byte strides stay below the tensor maps' 2^40

bool strides_ok(const char* what, uint64_t a, uint64_t b, uint64_t c = 0) {
  if ((a | b | c) % 8) return fail("%s: strides must be multiples of 8 elements", what) != 0;
  if (a >= kMaxStride || b >= kMaxStride || c >= kMaxStride) return fail("%s: stride out of range", what) != 0;
  return true;
}

// The description with the strides of dimensions of one element, which nothing is addressed by, set to a row.
AexrtB200AttentionDesc with_used_strides(const AexrtB200AttentionDesc* d, bool paged) {
  AexrtB200AttentionDesc u = *d;
  const uint64_t row = std::max(8u, d->head_dim);
  if (d->q_tokens <= 1) u.q_token_stride = u.out_token_stride = row * std::max(1u, d->q_heads);
  if (d->q_heads <= 1) u.q_head_stride = u.out_head_stride = row;
  if (d->kv_heads <= 1) u.k_head_stride = u.v_head_stride = row;
  if ((paged ? d->page_size : d->kv_tokens) <= 1) u.k_token_stride = u.v_token_stride = row;
  if (paged && d->kv_tokens <= 1) u.k_page_stride = u.v_page_stride = row;
  return u;
}

// The checks that packed and paged attention share (no pointers).
bool desc_ok(const AexrtB200AttentionDesc* d, bool paged) {
  const char* what = paged ? "attention_paged" : "attention_packed";
  if (!d) return fail("%s: null description", what) != 0;
  if (d->struct_size != sizeof(AexrtB200AttentionDesc)) return fail("%s: bad struct_size", what) != 0;
  if (d->dtype > AEXRT_B200_DTYPE_BF16) return fail("%s: unknown dtype %u", what, d->dtype) != 0;
  if (d->num_seqs > 65535u) return fail("%s: at most 65535 sequences", what) != 0;
  if (d->head_dim < 8 || d->head_dim > 128 || d->head_dim % 8)
    return fail("%s: head_dim must be a multiple of 8 from 8 to 128", what) != 0;
  if (d->q_heads == 0 || d->kv_heads == 0 || d->q_heads > 65535u || d->q_heads % d->kv_heads)
    return fail("%s: q_heads must be a multiple of kv_heads, from 1 to 65535", what) != 0;
  if (d->q_heads / d->kv_heads > 128) return fail("%s: at most 128 query heads per kv head", what) != 0;
  if (!(d->scale >= 0.f) || d->scale > 1e38f) return fail("%s: scale must be from 0 to 1e38", what) != 0;
  if (d->q_tokens > (1u << 30) || d->kv_tokens > (1u << 30)) return fail("%s: at most 2^30 rows or pages", what) != 0;
  // rows x heads index the launch grids
  if (static_cast<uint64_t>(d->q_tokens) * d->q_heads > (1ull << 32))
    return fail("%s: at most 2^32 query rows times heads", what) != 0;
  if (!strides_ok(what, d->q_token_stride, d->q_head_stride) || !strides_ok(what, d->out_token_stride, d->out_head_stride) ||
      !strides_ok(what, d->k_token_stride, d->k_head_stride, paged ? d->k_page_stride : 0) ||
      !strides_ok(what, d->v_token_stride, d->v_head_stride, paged ? d->v_page_stride : 0))
    return false;
  // rows of out that overlap would be written by several threads in no order
  const bool tokens_inside = d->out_token_stride < d->out_head_stride;
  const uint64_t lo = tokens_inside ? d->out_token_stride : d->out_head_stride;
  const uint64_t hi = tokens_inside ? d->out_head_stride : d->out_token_stride;
  const uint64_t lo_n = tokens_inside ? d->q_tokens : d->q_heads, hi_n = tokens_inside ? d->q_heads : d->q_tokens;
  if ((lo_n > 1 && lo < d->head_dim) || (hi_n > 1 && lo_n > 0 && hi < (lo_n > 1 ? lo * (lo_n - 1) : 0) + d->head_dim))
    return fail("%s: rows of out overlap", what) != 0;
  if (paged) {
    if (d->page_size < 8 || d->page_size > 1024 || (d->page_size & (d->page_size - 1)))
      return fail("%s: page_size must be a power of two from 8 to 1024", what) != 0;
    if (d->table_stride < d->table_columns) return fail("%s: table_stride below table_columns", what) != 0;
    if (static_cast<uint64_t>(d->table_columns) * d->page_size > (1ull << 30))
      return fail("%s: a table row of more than 2^30 tokens", what) != 0;
  }
  return true;
}

AttnParams make_params(const AexrtB200AttentionDesc* d, const void* q, const void* k, const void* v, void* out,
                       float* lse, const int32_t* cu_q) {
  AttnParams p = {};
  p.q = q;
  p.k = k;
  p.v = v;
  p.out = out;
  p.lse = lse;
  p.cu_q = cu_q;
  p.q_ts = static_cast<int64_t>(d->q_token_stride);
  p.q_hs = static_cast<int64_t>(d->q_head_stride);
  p.o_ts = static_cast<int64_t>(d->out_token_stride);
  p.o_hs = static_cast<int64_t>(d->out_head_stride);
  p.k_ts = static_cast<int64_t>(d->k_token_stride);
  p.k_hs = static_cast<int64_t>(d->k_head_stride);
  p.k_ps = static_cast<int64_t>(d->k_page_stride);
  p.v_ts = static_cast<int64_t>(d->v_token_stride);
  p.v_hs = static_cast<int64_t>(d->v_head_stride);
  p.v_ps = static_cast<int64_t>(d->v_page_stride);
  p.num_seqs = static_cast<int>(d->num_seqs);
  p.q_tokens = static_cast<int>(d->q_tokens);
  p.max_q = static_cast<int>(std::min(d->max_q, 1u << 30));
  p.q_heads = static_cast<int>(d->q_heads);
  p.kv_heads = static_cast<int>(d->kv_heads);
  p.group = static_cast<int>(d->q_heads / d->kv_heads);
  p.head_dim = static_cast<int>(d->head_dim);
  p.kv_tokens = static_cast<int>(d->kv_tokens);
  p.causal = d->causal ? 1 : 0;
  p.scale = std::max(d->scale, kMinScale);
  return p;
}

// Tensor maps of k and v: boxes of 64 elements of one head by `keys` rows (paged: by as many of a page).
bool kv_maps(const AexrtB200AttentionDesc* d, const AttnParams& p, bool paged, uint32_t keys, CUtensorMap* maps) {
  const CUtensorMapDataType dt =
      d->dtype == AEXRT_B200_DTYPE_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  for (int i = 0; i < 2; ++i) {
    const void* base = i ? p.v : p.k;
    const uint64_t ts = 2 * (i ? d->v_token_stride : d->k_token_stride), hs = 2 * (i ? d->v_head_stride : d->k_head_stride);
    const uint64_t rows = std::max(1u, d->kv_tokens);
    // without rows or pages the map still needs an address and an extent of 1: packed calls load no key then, paged ones
    // only no_page, which lies outside that extent
    if (d->kv_tokens == 0) base = p.q;
    const uint64_t dims[4] = {d->head_dim, d->kv_heads, paged ? d->page_size : rows, rows};
    const uint64_t strides[3] = {hs, ts, 2 * (i ? d->v_page_stride : d->k_page_stride)};
    const uint32_t box[4] = {64, 1, paged ? std::min<uint32_t>(d->page_size, keys) : keys, 1};
    if (!encode_tensor_map(&maps[i], dt, paged ? 4 : 3, base, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B)) return false;
  }
  return true;
}

// Query rows per sequence and kv head that the few-rows kernel takes; 0: the tensor-core kernel's.  The few-rows kernel
// against the tensor-core one, in us (8 kv heads of 128, bf16): 64 contexts of 4096 keys 181 against 287 with 20 rows, 187
// against 287 with 32, 305-326 against 291 with 36 and 314-345 against 292 with 64; 16 of 4096 65 against 90 with 32, 97 and
// 105 against 90 with 36 and 64; 4 of 8192 50 against 91 with 32, 69 and 80 against 91 with 36 and 64; one of 30000 69
// against 84 with 32, 91 and 114 against 84 with 36 and 64.  So up to 32 rows it is the faster one everywhere, and from 33
// to 64 over 4 contexts; over one, 16 or 64 a border of 32 would be faster.
uint32_t few_rows(const AexrtB200AttentionDesc* d) {
  const uint64_t rows = static_cast<uint64_t>(d->max_q) * (d->q_heads / d->kv_heads);
  return rows <= 64 ? static_cast<uint32_t>(rows) : 0;
}

int sm_count() {
  static int cached[128] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 128) return 148;
  if (!cached[dev]) {
    int n = 0;
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n <= 0) return 148;
    cached[dev] = n;
  }
  return cached[dev];
}

// Runs that the list of units is cut into: two blocks per SM, fewer when even full tables have no work for them.
uint32_t rows_grid(const AexrtB200AttentionDesc* d) {
  const uint64_t keys = std::min<uint64_t>(static_cast<uint64_t>(d->table_columns) * d->page_size, 1ull << 31);
  const uint64_t units = static_cast<uint64_t>(d->num_seqs) * d->kv_heads * std::max<uint64_t>(1, (keys + kRowsKeys - 1) / kRowsKeys);
  return static_cast<uint32_t>(std::min<uint64_t>(2 * sm_count(), (units + kRowsMinUnits - 1) / kRowsMinUnits));
}

uint64_t rows_workspace(uint64_t grid, uint64_t rows, uint64_t head_dim) {
  return grid * (sizeof(JoinHead) + 2 * rows * (head_dim + 2) * sizeof(float)) + 16;
}

// The joining launch may start while the launch before it ends; it waits for that before it reads anything.
template <typename... KArgs>
int launch_join(void (*fn)(KArgs...), dim3 grid, int threads, cudaStream_t st, const std::decay_t<KArgs>&... args) {
  cudaLaunchAttribute attr = {};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.stream = st;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cuda_ok(cudaLaunchKernelEx(&cfg, fn, args...), "attention join launch") ? 1 : 0;
}

int launch_rows(const AexrtB200AttentionDesc* d, const AttnParams& p, void* workspace, cudaStream_t st) {
  RowsParams rp = {};
  rp.a = p;
  rp.rows = static_cast<int>(few_rows(d));
  const uint32_t grid = rows_grid(d);
  rp.runs = static_cast<JoinHead*>(workspace);
  rp.parts = reinterpret_cast<float*>(rp.runs + grid);
  rp.stats = rp.parts + 2ull * grid * rp.rows * p.head_dim;
  const RowsKernel k = attention_rows_for(d->dtype == AEXRT_B200_DTYPE_BF16, p.head_dim, rp.rows);
  if (!raise_smem(reinterpret_cast<const void*>(k.fn), k.smem)) return 0;
  CUtensorMap maps[2];
  if (!kv_maps(d, p, true, kRowsKeys, maps)) return 0;
  if (!cuda_ok(launch_kernel(k.fn, dim3(grid), dim3(kRowsThreads), k.smem, st, maps[0], maps[1], rp), "attention launch"))
    return 0;
  if (grid == 1) return 1;
  return launch_join(k.join, dim3(grid - 1), kRowsCompute, st, rp);
}

// Items of a tensor-core call at most: every sequence ends in at most one partial pair of tiles.
uint64_t tc_items(const AexrtB200AttentionDesc* d) {
  const uint64_t tokens = kTcRows / (d->q_heads / d->kv_heads);
  uint64_t each = d->num_seqs + static_cast<uint64_t>(d->q_tokens) / (2 * tokens);
  if (d->max_q) each = std::min<uint64_t>(each, d->num_seqs * ((d->max_q + 2 * tokens - 1) / (2 * tokens)));
  return each * d->kv_heads;
}

// Whether a paged call's items are split over their keys: when there are at most 3 for every 2 SMs and a table row can hold
// keys for two parts.  Beyond, items even out by themselves, whole against split in us (32 heads over 8 of 128): two requests
// of 1024 tokens (256 items) over 16384 keys 565 against 568, over 32768 1217 against 1225; one of 2048 over 16384 572
// against 586.  Below, 64 tokens over 30000 keys take 391 whole and 66-69 split.
// Without the table's columns (the workspace's size is asked for before there is a table) as for a long row.
bool tc_splits(const AexrtB200AttentionDesc* d) {
  const uint64_t keys = static_cast<uint64_t>(d->table_columns) * d->page_size;
  return 2 * tc_items(d) <= 3 * static_cast<uint64_t>(sm_count()) && (d->table_columns == 0 || keys >= 2ull * kTcMinTiles * kTcKeys);
}

// Lays a split call's workspace out (from null: its size).
TcSplit tc_split(void* workspace, uint64_t head_dim, uint64_t* bytes) {
  const uint64_t grid = sm_count(), parts = 3 * grid;
  TcSplit split = {};
  uint8_t* at = static_cast<uint8_t*>(workspace);
  auto take = [&](uint64_t n) {
    uint8_t* here = at;
    at += (n + 15) / 16 * 16;
    return here;
  };
  split.split_items = reinterpret_cast<int*>(take(sizeof(int)));
  split.bases = reinterpret_cast<int*>(take(parts * sizeof(int)));
  split.heads = reinterpret_cast<JoinHead*>(take(2 * grid * sizeof(JoinHead)));
  split.sums = reinterpret_cast<float*>(take(parts * 256 * head_dim * sizeof(float)));
  split.stats = reinterpret_cast<float*>(take(parts * 256 * 2 * sizeof(float)));
  *bytes = static_cast<uint64_t>(at - static_cast<uint8_t*>(workspace));
  return split;
}

uint64_t tc_workspace(const AexrtB200AttentionDesc* d) {
  uint64_t bytes = 0;
  if (tc_splits(d)) tc_split(nullptr, d->head_dim, &bytes);
  return bytes;
}

int launch_tc(const AexrtB200AttentionDesc* d, const AttnParams& p, bool paged, void* workspace, cudaStream_t st) {
  const CUtensorMapDataType dt =
      d->dtype == AEXRT_B200_DTYPE_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  const uint32_t tokens = kTcRows / p.group;
  CUtensorMap maps[3];
  {
    const uint64_t dims[4] = {d->head_dim, static_cast<uint64_t>(p.group), d->kv_heads, d->q_tokens};
    const uint64_t strides[3] = {2 * d->q_head_stride, 2 * p.group * d->q_head_stride, 2 * d->q_token_stride};
    const uint32_t box[4] = {64, static_cast<uint32_t>(p.group), 1, tokens};
    if (!encode_tensor_map(&maps[0], dt, 4, p.q, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B)) return 0;
  }
  if (!kv_maps(d, p, paged, kTcKeys, maps + 1)) return 0;
  const bool splits = paged && tc_splits(d);
  uint64_t bytes = 0;
  const TcSplit split = splits ? tc_split(workspace, d->head_dim, &bytes) : TcSplit{};
  const TcKernel k = attention_tc_for(d->dtype == AEXRT_B200_DTYPE_BF16, paged, splits, p.head_dim);
  if (!raise_smem(reinterpret_cast<const void*>(k.fn), k.smem)) return 0;
  // one block per SM, fewer when there cannot be an item for each
  const unsigned sms = static_cast<unsigned>(sm_count());
  const unsigned blocks = splits ? sms : static_cast<unsigned>(std::min<uint64_t>(tc_items(d), sms));
  if (!cuda_ok(launch_kernel(k.fn, dim3(blocks), dim3(kTcThreads), k.smem, st, maps[0], maps[1], maps[2], p, split),
               "attention launch"))
    return 0;
  return splits ? launch_join(k.join, dim3((sms + 1) / 2, 256 / kTcJoinRows), kTcJoinThreads, st, p, split) : 1;
}

}  // namespace

int aexrt_b200_attention_packed(const AexrtB200AttentionDesc* d, const void* q, const void* k, const void* v,
                                const int32_t* cu_q, const int32_t* cu_k, void* out, float* lse, void* stream) {
  if (!d || d->struct_size != sizeof(AexrtB200AttentionDesc)) return desc_ok(d, false) ? 1 : 0;
  const AexrtB200AttentionDesc used = with_used_strides(d, false);
  d = &used;
  if (!desc_ok(d, false)) return 0;
  if (d->q_tokens == 0 || d->num_seqs == 0) return 1;
  if (!q || !cu_q || !cu_k || !out || (d->kv_tokens && (!k || !v))) return fail("attention_packed: null pointer");
  if (!aligned16(q) || !aligned16(k) || !aligned16(v) || !aligned16(out))
    return fail("attention_packed: q, k, v and out must be 16-byte aligned");
  AttnParams p = make_params(d, q, k, v, out, lse, cu_q);
  p.cu_k = cu_k;
  p.status = status_word();
  if (!p.status) return 0;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  return launch_tc(d, p, false, nullptr, st);
}

uint64_t aexrt_b200_attention_paged_workspace(const AexrtB200AttentionDesc* d) {
  if (!d || d->struct_size != sizeof(AexrtB200AttentionDesc)) return desc_ok(d, true), ~0ull;
  const AexrtB200AttentionDesc used = with_used_strides(d, true);
  d = &used;
  if (!desc_ok(d, true)) return ~0ull;
  if (d->q_tokens == 0 || d->num_seqs == 0 || d->max_q == 0) return 0;
  const uint32_t rows = few_rows(d);
  return rows ? rows_workspace(2ull * sm_count(), rows, d->head_dim) : tc_workspace(d);
}

int aexrt_b200_attention_paged(const AexrtB200AttentionDesc* d, const void* q, const void* k_cache, const void* v_cache,
                               const int32_t* block_table, const int32_t* cu_q, const int32_t* kv_lens, void* out,
                               float* lse, void* workspace, uint64_t workspace_bytes, void* stream) {
  if (!d || d->struct_size != sizeof(AexrtB200AttentionDesc)) return desc_ok(d, true) ? 1 : 0;
  const AexrtB200AttentionDesc used = with_used_strides(d, true);
  d = &used;
  if (!desc_ok(d, true)) return 0;
  if (d->q_tokens == 0 || d->num_seqs == 0 || d->max_q == 0) return 1;
  if (!q || !cu_q || !kv_lens || !out || (d->kv_tokens && (!k_cache || !v_cache)) || (d->table_columns && !block_table))
    return fail("attention_paged: null pointer");
  if (!aligned16(q) || !aligned16(k_cache) || !aligned16(v_cache) || !aligned16(out))
    return fail("attention_paged: q, caches and out must be 16-byte aligned");
  const uint64_t need = aexrt_b200_attention_paged_workspace(d);
  if (workspace_bytes < need || (need && (!workspace || !aligned16(workspace))))
    return fail("attention_paged: needs %llu bytes of 16-byte aligned workspace", static_cast<unsigned long long>(need));
  AttnParams p = make_params(d, q, k_cache, v_cache, out, lse, cu_q);
  p.kv_lens = kv_lens;
  p.block_table = block_table;
  p.table_columns = static_cast<int>(d->table_columns);
  p.table_stride = d->table_stride;
  p.page_shift = log2_exact(d->page_size);
  p.no_page = static_cast<int>(std::max(1u, d->kv_tokens));
  p.status = status_word();
  if (!p.status) return 0;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  return few_rows(d) ? launch_rows(d, p, workspace, st) : launch_tc(d, p, true, workspace, st);
}

int aexrt_b200_attention_status(uint32_t* status) {
  if (!status) return fail("attention_status: null pointer");
  uint32_t* word = status_word();
  if (!word) return 0;
  // the default stream does not wait for streams made without that tie, as torch's are
  if (!cuda_ok(cudaDeviceSynchronize(), "synchronize for the attention status")) return 0;
  static std::mutex mu;  // one reader at a time: the kernel and the copy of what it took
  std::lock_guard<std::mutex> lock(mu);
  take_status_kernel<<<1, 1>>>(word);
  if (!cuda_ok(cudaGetLastError(), "attention status launch")) return 0;
  return cuda_ok(cudaMemcpy(status, word + 1, sizeof(uint32_t), cudaMemcpyDeviceToHost), "read attention status") ? 1 : 0;
}

int aexrt_b200_page_tables(const int32_t* ctx_lens, const int32_t* new_lens, uint32_t num_seqs, uint32_t page_size,
                           int32_t* block_table, uint32_t table_columns, uint32_t table_stride,
                           const int32_t* free_pages, uint32_t free_capacity, const int32_t* free_state_in,
                           int32_t* free_state_out, int32_t* cu_q, int32_t* kv_lens, int32_t* slot_map,
                           uint32_t slot_capacity, void* stream) {
  if (num_seqs > static_cast<uint32_t>(kTablesMaxSeqs)) return fail("page_tables: at most %d requests", kTablesMaxSeqs);
  if (page_size == 0 || page_size > 1024 || (page_size & (page_size - 1)))
    return fail("page_tables: page_size must be a power of two up to 1024");
  if (table_columns > (1u << 30) || table_stride < table_columns) return fail("page_tables: table_stride below table_columns");
  if (free_capacity > (1u << 30) || slot_capacity > (1u << 30)) return fail("page_tables: at most 2^30 free pages or slots");
  if (!free_state_in || !free_state_out || !cu_q || (num_seqs && (!ctx_lens || !new_lens || !kv_lens)) ||
      (num_seqs && table_columns && !block_table) || (free_capacity && !free_pages) || (slot_capacity && !slot_map))
    return fail("page_tables: null pointer");
  TablesParams p = {};
  p.ctx = ctx_lens;
  p.add = new_lens;
  p.free_pages = free_pages;
  p.state_in = free_state_in;
  p.table = block_table;
  p.state_out = free_state_out;
  p.cu_q = cu_q;
  p.kv_lens = kv_lens;
  p.slots = slot_map;
  p.num_seqs = static_cast<int>(num_seqs);
  p.page_shift = log2_exact(page_size);
  p.columns = static_cast<int>(table_columns);
  p.table_stride = table_stride;
  p.free_capacity = static_cast<int>(free_capacity);
  p.slot_capacity = static_cast<int>(slot_capacity);
  const size_t smem = (3ull * num_seqs + 2) * sizeof(int32_t);
  if (!raise_smem(reinterpret_cast<const void*>(page_tables_kernel),
                  (3 * kTablesMaxSeqs + 2) * static_cast<int>(sizeof(int32_t))))
    return 0;
  // In place, every block has to have read the lengths and the state before one writes them: one cluster.  Otherwise the
  // blocks need nothing of one another.
  const bool in_place = kv_lens == ctx_lens || free_state_out == free_state_in;
  const unsigned most = in_place ? kTablesMaxCtas : static_cast<unsigned>(sm_count());
  const unsigned ctas = std::min(most, std::max(1u, (slot_capacity + kTablesThreads - 1) / kTablesThreads));
  return cuda_ok(launch_kernel_cluster(page_tables_kernel, dim3(ctas), dim3(kTablesThreads), smem,
                                       static_cast<cudaStream_t>(stream), in_place ? ctas : 1, p),
                 "page_tables launch")
             ? 1
             : 0;
}

int aexrt_b200_kv_append(const void* k, const void* v, uint32_t tokens, uint32_t kv_heads, uint32_t head_dim,
                         uint64_t k_token_stride, uint64_t k_head_stride, uint64_t v_token_stride,
                         uint64_t v_head_stride, const int32_t* slot_map, void* k_cache, void* v_cache,
                         uint32_t num_pages, uint32_t page_size, uint64_t k_cache_page_stride,
                         uint64_t k_cache_token_stride, uint64_t k_cache_head_stride, uint64_t v_cache_page_stride,
                         uint64_t v_cache_token_stride, uint64_t v_cache_head_stride, void* stream) {
  if (head_dim == 0 || head_dim % 8 || head_dim > 65536) return fail("kv_append: head_dim must be a multiple of 8");
  if (kv_heads == 0 || kv_heads > 65535u) return fail("kv_append: kv_heads must be from 1 to 65535");
  if (tokens > (1u << 30)) return fail("kv_append: at most 2^30 tokens");
  // dimensions of one element: nothing is addressed by their strides
  if (tokens <= 1) k_token_stride = v_token_stride = head_dim;
  if (kv_heads <= 1) k_head_stride = v_head_stride = k_cache_head_stride = v_cache_head_stride = head_dim;
  if (page_size <= 1) k_cache_token_stride = v_cache_token_stride = head_dim;
  if (num_pages <= 1) k_cache_page_stride = v_cache_page_stride = head_dim;
  if (page_size == 0 || page_size > 1024 || (page_size & (page_size - 1)))
    return fail("kv_append: page_size must be a power of two up to 1024");
  if (static_cast<uint64_t>(num_pages) * page_size >= (1ull << 31)) return fail("kv_append: the cache has 2^31 slots or more");
  if (!strides_ok("kv_append", k_token_stride, k_head_stride) || !strides_ok("kv_append", v_token_stride, v_head_stride) ||
      !strides_ok("kv_append", k_cache_page_stride, k_cache_token_stride, k_cache_head_stride) ||
      !strides_ok("kv_append", v_cache_page_stride, v_cache_token_stride, v_cache_head_stride))
    return 0;
  if (tokens == 0 || num_pages == 0) return 1;
  if (!k || !v || !slot_map || !k_cache || !v_cache) return fail("kv_append: null pointer");
  if (!aligned16(k) || !aligned16(v) || !aligned16(k_cache) || !aligned16(v_cache))
    return fail("kv_append: k, v and the caches must be 16-byte aligned");
  AppendParams p = {};
  p.k = static_cast<const uint4*>(k);
  p.v = static_cast<const uint4*>(v);
  p.k_cache = static_cast<uint4*>(k_cache);
  p.v_cache = static_cast<uint4*>(v_cache);
  p.slots = slot_map;
  p.tokens = static_cast<int>(tokens);
  p.kv_heads = static_cast<int>(kv_heads);
  p.row_vecs = static_cast<int>(head_dim / 8);
  p.page_shift = log2_exact(page_size);
  p.num_slots = static_cast<int>(num_pages * page_size);
  p.k_ts = static_cast<int64_t>(k_token_stride / 8);
  p.k_hs = static_cast<int64_t>(k_head_stride / 8);
  p.v_ts = static_cast<int64_t>(v_token_stride / 8);
  p.v_hs = static_cast<int64_t>(v_head_stride / 8);
  p.kc_ps = static_cast<int64_t>(k_cache_page_stride / 8);
  p.kc_ts = static_cast<int64_t>(k_cache_token_stride / 8);
  p.kc_hs = static_cast<int64_t>(k_cache_head_stride / 8);
  p.vc_ps = static_cast<int64_t>(v_cache_page_stride / 8);
  p.vc_ts = static_cast<int64_t>(v_cache_token_stride / 8);
  p.vc_hs = static_cast<int64_t>(v_cache_head_stride / 8);
  const uint64_t pieces = static_cast<uint64_t>(tokens) * kv_heads * p.row_vecs;
  if (pieces > (1ull << 38)) return fail("kv_append: too many elements");
  launch_kernel(kv_append_kernel, dim3(static_cast<unsigned>((pieces + 255) / 256)), dim3(256), 0,
                static_cast<cudaStream_t>(stream), p);
  return cuda_ok(cudaGetLastError(), "kv_append launch") ? 1 : 0;
}
