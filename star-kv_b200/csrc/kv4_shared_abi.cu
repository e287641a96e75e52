// kv4_shared_abi.cu — the starkv_kv4_shared_* entry points (declared in include/starkv.h):
// argument checks and launches.  Nothing here allocates device memory or synchronises.
#include <cuda_runtime.h>

#include <atomic>
#include <cstring>

#include "host.hpp"
#include "kv4_prefix.cuh"

using namespace starkv;

namespace {

// Rows a KV head up to which the decode kernel takes the prefix (its columns are 16).  Both ways, us in a
// graph, decode kernel and tensor cores, own 40:
//                      777 tokens   4096        16384       65536       131072
//    4 rows,  1 head    25  31     27  33      31  45      35  66      37  70
//    4 rows,  8 heads   29  36     31  37      35  47      46  92      66  158
//   16 rows,  1 head    35  35     37  35      46  47      58  68      62  74
//   16 rows,  4 heads   36  36     39  37      49  45      60  66      71  98
//   16 rows,  8 heads   37  37     39  37      49  47      70  98      98  156
//   16 rows, 32 heads   41  41     45  49      67  102
// The tensor cores gain up to 4 us in between and lose far more at both ends.
constexpr int kDecodeRows = 16;

size_t up(size_t n) { return (n + 255) & ~(size_t)255; }

// Where things lie in the workspace, behind the decode kernel's scratch.
struct Places {
  size_t rows, prefix_out, prefix_lse, own_out, own_lse, total;
  explicit Places(int64_t heads) {        // batch * num_queries * num_q_heads
    rows = up(kKv4WorkspaceBytes);
    prefix_out = rows + up(heads * 256);
    prefix_lse = prefix_out + up(heads * 512);
    own_out = prefix_lse + up(heads * 4);
    own_lse = own_out + up(heads * 512);
    total = own_lse + up(heads * 4);
  }
};

int launch_prefix(const Kv4PrefixParams& p, cudaStream_t st) {
  static std::atomic<uint64_t> ready{0};                       // one bit a device
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return host_launch_status();
  if (dev >= 64 || !(ready.load(std::memory_order_relaxed) >> dev & 1)) {
    if (cudaFuncSetAttribute(kv4_prefix_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kKvpSmemBytes) != cudaSuccess)
      return host_launch_status();
    if (dev < 64) ready.fetch_or(1ull << dev);
  }
  kv4_prefix_kernel<<<p.grid, kKvpThreads, kKvpSmemBytes, st>>>(p);
  const int rc = host_launch_status();
  // rows are cut only where there are fewer (KV head, block)s than CTAs
  const int items = p.pool.heads * p.blocks;
  if (rc || (!p.halves && items * 2 > p.grid)) return rc;
  kv4_prefix_join_kernel<<<items * (p.halves ? 1 : 2) * 16, 128, 0, st>>>(p);
  return host_launch_status();
}

}  // namespace

extern "C" {

int starkv_kv4_shared_workspace_size(int32_t batch, int32_t num_queries, int32_t num_q_heads, size_t* bytes) {
  if (!bytes || batch < 0 || num_queries < 0 || num_q_heads <= 0) return host_error(STARKV_ERR_INVALID, "bad argument");
  *bytes = Places((int64_t)batch * num_queries * num_q_heads).total;
  return STARKV_OK;
}

int starkv_kv4_shared_attention(const starkv_kv4_cache* cache, const starkv_kv4_shared_args* a, starkv_stream_t stream) {
  if (!cache || !a) return host_error(STARKV_ERR_INVALID, "null argument");
  if (cache->num_kv_heads <= 0 || a->batch < 0 || a->batch > 65535 || a->num_queries < 0 || a->num_q_heads <= 0 ||
      a->num_q_heads % cache->num_kv_heads || a->table_width <= 0 || a->prefix_width <= 0)
    return host_error(STARKV_ERR_INVALID, "bad batch (at most 65535), query count, head counts or block tables");
  const int64_t heads = (int64_t)a->batch * a->num_queries * a->num_q_heads;
  const int group = a->num_q_heads / cache->num_kv_heads;
  if ((int64_t)a->batch * a->num_queries * group > 65536) return host_error(STARKV_ERR_UNSUPPORTED, "too many queries behind one prefix");
  if (((int64_t)a->prefix_width * cache->page_size) > 0x7fffff00)
    return host_error(STARKV_ERR_UNSUPPORTED, "prefix table of 2^31 positions or more");
  const bool none = a->batch == 0 || a->num_queries == 0;
  const Places at(none ? 0 : heads);
  if (!none) {
    if (!a->prefix_table || !a->prefix_length || !a->workspace) return host_error(STARKV_ERR_INVALID, "null argument");
    if (a->workspace_bytes < at.total) return host_error(STARKV_ERR_WORKSPACE, "kv4 shared attention workspace too small");
    if ((uintptr_t)a->workspace & 15) return host_error(STARKV_ERR_WORKSPACE, "kv4 shared attention workspace must be 16-byte aligned");
  }
  uint8_t* ws = (uint8_t*)a->workspace;
  // the own tokens; the entry point checks what the two have in common
  starkv_kv4_attention_args own;
  memset(&own, 0, sizeof(own));
  own.q = a->q;
  memcpy(own.q_strides, a->q_strides, sizeof(own.q_strides));
  own.block_table = a->block_table;
  own.table_stride = a->table_stride;
  own.lengths = a->lengths;
  own.mask = a->mask, own.mask_stride = a->mask_stride, own.mask_width = a->mask_width;
  own.workspace = ws, own.workspace_bytes = kKv4WorkspaceBytes;
  own.scaling = a->scaling;
  own.q_dtype = a->q_dtype, own.out_dtype = STARKV_F32;
  own.batch = a->batch, own.num_queries = a->num_queries, own.num_q_heads = a->num_q_heads, own.table_width = a->table_width;
  own.out = none ? nullptr : ws + at.own_out;
  own.lse = none ? nullptr : (float*)(ws + at.own_lse);
  own.out_strides[0] = (int64_t)a->num_queries * a->num_q_heads * 128;
  own.out_strides[1] = (int64_t)a->num_q_heads * 128;
  own.out_strides[2] = 128;
  // what only this entry point has
  const int ob = a->out_dtype == STARKV_F32 ? 4 : a->out_dtype == STARKV_F16 || a->out_dtype == STARKV_BF16 ? 2 : 0;
  if (!ob) return host_error(STARKV_ERR_INVALID, "bad out_dtype");
  if (!none) {
    bool ok = a->out && (uintptr_t)a->out % 16 == 0;
    for (int i = 0; i < 3; ++i) ok = ok && a->out_strides[i] >= 0 && a->out_strides[i] * ob % 16 == 0;
    if (!ok) return host_error(STARKV_ERR_INVALID, "out rows must be 16-byte aligned");
    if (!(a->scaling > 0.f) || a->scaling > 1e30f) return host_error(STARKV_ERR_INVALID, "scaling must be positive and finite");
    if (((uintptr_t)a->lse | (uintptr_t)a->prefix_table | (uintptr_t)a->prefix_length) & 3)
      return host_error(STARKV_ERR_INVALID, "int32 and fp32 arguments must be 4-byte aligned");
  }
  int rc = starkv_kv4_attention(cache, &own, stream);
  if (rc || none) return rc;
  Kv4SharedParams p;
  memset(&p, 0, sizeof(p));
  p.q = a->q, p.out = a->out, p.lse = a->lse;
  memcpy(p.qs, a->q_strides, sizeof(p.qs));
  memcpy(p.os, a->out_strides, sizeof(p.os));
  p.batch = a->batch, p.queries = a->num_queries, p.q_heads = a->num_q_heads, p.kv_heads = cache->num_kv_heads, p.group = group;
  p.q_dtype = a->q_dtype, p.out_dtype = a->out_dtype;
  p.rows = ws + at.rows;
  p.prefix_out = (float*)(ws + at.prefix_out), p.prefix_lse = (float*)(ws + at.prefix_lse);
  p.own_out = (float*)(ws + at.own_out), p.own_lse = (float*)(ws + at.own_lse);
  cudaStream_t st = (cudaStream_t)stream;
  const int rows = a->batch * a->num_queries * group;
  if (rows > kDecodeRows) {
    Kv4PrefixParams k;
    memset(&k, 0, sizeof(k));
    k.s = p;
    int sms = 0;
    if ((rc = host_device(&sms))) return rc;
    const int grid = sms < kKv4MaxGrid ? sms : kKv4MaxGrid;
    k.pool.data = (uint8_t*)cache->data, k.pool.err = cache->error_word;
    k.pool.num_pages = cache->num_pages, k.pool.heads = cache->num_kv_heads, k.pool.page_tiles = cache->page_size / kKv4Tile;
    k.pool.page_shift = cache->page_size == 16 ? 4 : cache->page_size == 32 ? 5 : cache->page_size == 64 ? 6 : 7;
    k.table = a->prefix_table, k.length = a->prefix_length, k.width = a->prefix_width;
    k.rows = rows;
    k.halves = rows <= 128 && cache->num_kv_heads <= grid;
    k.blocks = (rows + 255) / 256;
    k.scale_log2 = (float)(a->scaling * 1.4426950408889634);
    k.wait_ns = host_wait_limit();
    k.skip_step = host_skip_unit();
    k.grid = grid;
    k.parts = (float*)(ws + kKv4CounterBytes);
    return launch_prefix(k, st);
  }
  const unsigned grid = (unsigned)((heads + 7) / 8);
  kv4_shared_rows_kernel<<<grid, 256, 0, st>>>(p);
  if ((rc = host_launch_status())) return rc;
  // the prefix as one sequence with one token, whose heads are all the rows
  starkv_kv4_attention_args pre = own;
  pre.q = p.rows;
  pre.q_strides[0] = pre.q_strides[1] = heads * 128, pre.q_strides[2] = 128;
  pre.out = (void*)p.prefix_out, pre.lse = (float*)p.prefix_lse;
  pre.out_strides[0] = pre.out_strides[1] = heads * 128, pre.out_strides[2] = 128;
  pre.block_table = a->prefix_table, pre.table_stride = a->prefix_width, pre.table_width = a->prefix_width;
  pre.lengths = a->prefix_length;
  pre.mask = nullptr, pre.mask_stride = pre.mask_width = 0;
  pre.batch = 1, pre.num_queries = 1, pre.num_q_heads = (int32_t)heads;
  if ((rc = starkv_kv4_attention(cache, &pre, stream))) return rc;
  kv4_shared_merge_kernel<<<grid, 256, 0, st>>>(p);
  return host_launch_status();
}

}  // extern "C"
