// kv4_abi.cu — the starkv_kv4_* entry points (declared in include/starkv.h):
// argument checks, launch geometry and launches.  Nothing here allocates device
// memory or synchronises.
#include <cuda_runtime.h>

#include <atomic>
#include <cstring>

#include "host.hpp"
#include "kv4.cuh"
#include "kv4_attn.cuh"

using namespace starkv;

namespace {

// Whether every address is a multiple of `bytes` (null is).
template <typename... P>
bool aligned(size_t bytes, P... ptrs) {
  return ((reinterpret_cast<uintptr_t>(ptrs) | ...) & (bytes - 1)) == 0;
}

int check_pool(const starkv_kv4_cache* c, Kv4Pool* pool) {
  if (!c || !c->data) return host_error(STARKV_ERR_INVALID, "null cache");
  if (c->head_dim != 128) return host_error(STARKV_ERR_UNSUPPORTED, "kv4 caches take head_dim 128");
  if (c->page_size != 16 && c->page_size != 32 && c->page_size != 64 && c->page_size != 128)
    return host_error(STARKV_ERR_UNSUPPORTED, "kv4 page_size must be 16, 32, 64 or 128");
  if (c->num_pages <= 0 || c->num_kv_heads <= 0 || c->num_kv_heads > 65535)
    return host_error(STARKV_ERR_INVALID, "kv4 cache needs pages and KV heads (at most 65535)");
  if (!aligned(16, c->data, c->bounds) || !aligned(4, c->bound_scales, c->error_word))
    return host_error(STARKV_ERR_INVALID, "kv4 data and bounds must be 16-byte aligned, scales and error word 4-byte");
  if ((c->bounds == nullptr) != (c->bound_scales == nullptr))
    return host_error(STARKV_ERR_INVALID, "kv4 bounds and bound_scales go together");
  pool->data = (uint8_t*)c->data;
  pool->bounds = (int8_t*)c->bounds;
  pool->bound_scales = c->bound_scales;
  pool->err = c->error_word;
  pool->num_pages = c->num_pages;
  pool->heads = c->num_kv_heads;
  pool->page_tiles = c->page_size / kKv4Tile;
  pool->page_shift = c->page_size == 16 ? 4 : c->page_size == 32 ? 5 : c->page_size == 64 ? 6 : 7;
  return host_device(nullptr);
}

int elem_bytes(int dtype) {
  return dtype == STARKV_F32 ? 4 : dtype == STARKV_F16 || dtype == STARKV_BF16 ? 2 : 0;
}

// Strides of a (B, tokens, heads, 128) tensor whose rows are read 16 bytes at a time.
int check_rows(const void* base, const int64_t* strides, int eb, const char* what) {
  if (!base) return host_error(STARKV_ERR_INVALID, "null tensor");
  bool ok = reinterpret_cast<uintptr_t>(base) % 16 == 0;
  for (int i = 0; i < 3; ++i) ok = ok && strides[i] >= 0 && (strides[i] * eb) % 16 == 0;
  return ok ? STARKV_OK : host_error(STARKV_ERR_INVALID, what);
}

int io_params(const starkv_kv4_cache* cache, const starkv_kv4_io_args* a, Kv4IoParams* p) {
  int rc = check_pool(cache, &p->pool);
  if (rc) return rc;
  if (!a) return host_error(STARKV_ERR_INVALID, "null argument");
  const int eb = elem_bytes(a->dtype);
  if (!eb) return host_error(STARKV_ERR_INVALID, "k / v must be fp32, fp16 or bf16");
  if (a->batch < 0 || a->batch > 65535 || a->num_tokens < 0 || a->table_width <= 0 || a->table_stride < 0)
    return host_error(STARKV_ERR_INVALID, "bad batch (at most 65535), token count or block table");
  if (a->batch == 0 || a->num_tokens == 0) return STARKV_OK;
  if (!a->block_table || !a->start) return host_error(STARKV_ERR_INVALID, "null argument");
  if (!aligned(4, a->block_table, a->start, a->count)) return host_error(STARKV_ERR_INVALID, "int32 arguments must be 4-byte aligned");
  if ((rc = check_rows(a->k, a->k_strides, eb, "k rows must be 16-byte aligned")) ||
      (rc = check_rows(a->v, a->v_strides, eb, "v rows must be 16-byte aligned")))
    return rc;
  p->k = a->k;
  p->v = a->v;
  memcpy(p->ks, a->k_strides, sizeof(p->ks));
  memcpy(p->vs, a->v_strides, sizeof(p->vs));
  p->table = a->block_table;
  p->table_stride = a->table_stride;
  p->start = a->start;
  p->count = a->count;
  p->num_tokens = a->num_tokens;
  p->width = a->table_width;
  return STARKV_OK;
}

template <int NT, int W, bool MASK>
int launch_attn(const Kv4AttnParams& p, int grid, cudaStream_t st) {
  auto kern = kv4_attn_kernel<NT, W, MASK>;
  const size_t smem = sizeof(Kv4AttnSmem<NT, W, MASK>);
  static_assert(sizeof(Kv4AttnSmem<NT, W, MASK>) <= 227 * 1024, "shared memory of one SM");
  static std::atomic<uint64_t> raised{0};                      // one bit a device
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return host_launch_status();
  if (dev >= 64 || !(raised.load(std::memory_order_relaxed) >> dev & 1)) {
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != cudaSuccess)
      return host_launch_status();
    if (dev < 64) raised.fetch_or(1ull << dev);
  }
  kern<<<grid, (W + 1) * 32, smem, st>>>(p);
  return host_launch_status();
}

}  // namespace

extern "C" {

size_t starkv_kv4_struct_size(int32_t which) {
  switch (which) {
    case 0: return sizeof(starkv_kv4_cache);
    case 1: return sizeof(starkv_kv4_io_args);
    case 2: return sizeof(starkv_kv4_attention_args);
    case 3: return sizeof(starkv_kv4_select_args);
    default: return 0;
  }
}

int starkv_kv4_write(const starkv_kv4_cache* cache, const starkv_kv4_io_args* a, starkv_stream_t stream) {
  Kv4IoParams p;
  memset(&p, 0, sizeof(p));
  const int rc = io_params(cache, a, &p);
  if (rc || a->batch == 0 || a->num_tokens == 0) return rc;
  const int ps = cache->page_size;
  p.span = (int)(((int64_t)a->num_tokens + ps - 2) / ps + 1);
  const int64_t ctas = (int64_t)p.span * p.pool.heads;
  if (ctas > 0x7fffffff) return host_error(STARKV_ERR_UNSUPPORTED, "too many pages in one write");
  const dim3 grid((unsigned)ctas, (unsigned)a->batch);
  const int threads = 32 * p.pool.page_tiles;
  cudaStream_t st = (cudaStream_t)stream;
  if (a->dtype == STARKV_F32)
    kv4_write_kernel<float><<<grid, threads, 0, st>>>(p);
  else if (a->dtype == STARKV_F16)
    kv4_write_kernel<__half><<<grid, threads, 0, st>>>(p);
  else
    kv4_write_kernel<__nv_bfloat16><<<grid, threads, 0, st>>>(p);
  return host_launch_status();
}

int starkv_kv4_read(const starkv_kv4_cache* cache, const starkv_kv4_io_args* a, starkv_stream_t stream) {
  Kv4IoParams p;
  memset(&p, 0, sizeof(p));
  const int rc = io_params(cache, a, &p);
  if (rc || a->batch == 0 || a->num_tokens == 0) return rc;
  p.span = (int)(((int64_t)a->num_tokens + kKv4Tile - 2) / kKv4Tile + 1);
  p.units = (int64_t)p.span * p.pool.heads * a->batch;
  const int64_t ctas = (p.units + kKv4ReadWarps - 1) / kKv4ReadWarps;
  if (ctas > 0x7fffffff) return host_error(STARKV_ERR_UNSUPPORTED, "too many tokens in one read");
  cudaStream_t st = (cudaStream_t)stream;
  if (a->dtype == STARKV_F32)
    kv4_read_kernel<float><<<(unsigned)ctas, kKv4ReadWarps * 32, 0, st>>>(p);
  else if (a->dtype == STARKV_F16)
    kv4_read_kernel<__half><<<(unsigned)ctas, kKv4ReadWarps * 32, 0, st>>>(p);
  else
    kv4_read_kernel<__nv_bfloat16><<<(unsigned)ctas, kKv4ReadWarps * 32, 0, st>>>(p);
  return host_launch_status();
}

int starkv_kv4_workspace_size(size_t* bytes) {
  if (!bytes) return host_error(STARKV_ERR_INVALID, "null argument");
  *bytes = kKv4WorkspaceBytes;
  return STARKV_OK;
}

int starkv_kv4_attention(const starkv_kv4_cache* cache, const starkv_kv4_attention_args* a, starkv_stream_t stream) {
  Kv4AttnParams p;
  memset(&p, 0, sizeof(p));
  int rc = check_pool(cache, &p.pool);
  if (rc) return rc;
  if (!a) return host_error(STARKV_ERR_INVALID, "null argument");
  if (a->q_dtype != STARKV_F16 && a->q_dtype != STARKV_BF16)
    return host_error(STARKV_ERR_UNSUPPORTED, "kv4 attention takes fp16 or bf16 queries");
  const int ob = elem_bytes(a->out_dtype);
  if (!ob) return host_error(STARKV_ERR_INVALID, "bad out_dtype");
  if (a->batch < 0 || a->batch > 65535 || a->num_queries < 0 || a->num_q_heads <= 0 ||
      a->num_q_heads % p.pool.heads || a->table_width <= 0 || a->table_stride < 0)
    return host_error(STARKV_ERR_INVALID, "bad batch (at most 65535), query count, head counts or block table");
  if (a->pages && a->num_selected <= 0) return host_error(STARKV_ERR_INVALID, "num_selected must be positive");
  if (a->mask && (a->mask_stride < 0 || a->mask_width < 0)) return host_error(STARKV_ERR_INVALID, "bad mask");
  if (a->batch == 0 || a->num_queries == 0) return STARKV_OK;
  if (!a->block_table || !a->lengths || !a->workspace) return host_error(STARKV_ERR_INVALID, "null argument");
  size_t need = 0;
  starkv_kv4_workspace_size(&need);
  if (a->workspace_bytes < need) return host_error(STARKV_ERR_WORKSPACE, "kv4 attention workspace too small");
  if (!aligned(16, a->workspace)) return host_error(STARKV_ERR_WORKSPACE, "kv4 attention workspace must be 16-byte aligned");
  if (!aligned(4, a->block_table, a->lengths, a->pages, a->mask, a->lse))
    return host_error(STARKV_ERR_INVALID, "int32 and fp32 arguments must be 4-byte aligned");
  if ((rc = check_rows(a->q, a->q_strides, 2, "q rows must be 16-byte aligned")) ||
      (rc = check_rows(a->out, a->out_strides, ob, "out rows must be 16-byte aligned")))
    return rc;
  p.q = a->q;
  p.out = a->out;
  p.lse = a->lse;
  memcpy(p.qs, a->q_strides, sizeof(p.qs));
  memcpy(p.os, a->out_strides, sizeof(p.os));
  p.table = a->block_table;
  p.table_stride = a->table_stride;
  p.lengths = a->lengths;
  p.mask = a->mask;
  p.mask_stride = a->mask_stride;
  p.mask_width = a->mask_width;
  p.pages = a->pages;
  p.scaling = a->scaling;
  p.num_selected = a->num_selected;
  p.out_dtype = a->out_dtype;
  p.batch = a->batch;
  p.queries = a->num_queries;
  p.q_heads = a->num_q_heads;
  p.group = a->num_q_heads / p.pool.heads;
  p.width = a->table_width;
  const int64_t cols = (int64_t)p.group * p.queries;
  if (cols > 65536) return host_error(STARKV_ERR_UNSUPPORTED, "too many query columns");
  // up to 8 columns one n-tile of the matrix instructions, more in blocks of 16
  const int nt = cols <= 8 ? 1 : 2;
  p.q_dtype = a->q_dtype;
  p.col_blocks = (int)((cols + nt * 8 - 1) / (nt * 8));
  if ((int64_t)p.pool.heads * p.col_blocks > (1 << 24))
    return host_error(STARKV_ERR_UNSUPPORTED, "too many query columns");
  if (((int64_t)a->table_width << p.pool.page_shift) > 0x7fffff00)
    return host_error(STARKV_ERR_UNSUPPORTED, "block table of 2^31 positions or more");
  const int64_t tiles = (a->pages ? (int64_t)a->num_selected : (int64_t)a->table_width) * p.pool.page_tiles + kKv4PadTiles;
  if ((double)tiles * p.pool.heads * p.col_blocks * a->batch > 2.0e9)
    return host_error(STARKV_ERR_UNSUPPORTED, "batch * KV heads * tiles of a block table row must stay below 2e9");
  p.wait_ns = host_wait_limit();
  p.skip_copy = host_skip_unit();
  p.group_m = kv4_reciprocal(p.group);
  p.col_blocks_m = kv4_reciprocal(p.col_blocks);
  int sms = 0;
  if ((rc = host_device(&sms))) return rc;
  const int grid = sms < kKv4MaxGrid ? sms : kKv4MaxGrid;
  p.counters = (int*)a->workspace;
  p.parts = (float*)((uint8_t*)a->workspace + kKv4CounterBytes);
  p.heads = p.parts + (size_t)kKv4MaxGrid * 2 * kKv4PartFloats;
  cudaStream_t st = (cudaStream_t)stream;
  if (nt == 1)
    return p.mask ? launch_attn<1, 15, true>(p, grid, st) : launch_attn<1, 15, false>(p, grid, st);
  return p.mask ? launch_attn<2, 11, true>(p, grid, st) : launch_attn<2, 11, false>(p, grid, st);
}

int starkv_kv4_select_workspace_size(const starkv_kv4_cache* cache, int32_t batch, int32_t table_width, size_t* bytes) {
  if (!cache || !bytes || batch < 0 || table_width < 0) return host_error(STARKV_ERR_INVALID, "bad argument");
  *bytes = kKv4MaxSegments * sizeof(int) + (size_t)batch * cache->num_kv_heads * table_width * sizeof(float);
  return STARKV_OK;
}

int starkv_kv4_select(const starkv_kv4_cache* cache, const starkv_kv4_select_args* a, starkv_stream_t stream) {
  Kv4SelectParams p;
  memset(&p, 0, sizeof(p));
  int rc = check_pool(cache, &p.pool);
  if (rc) return rc;
  if (!a) return host_error(STARKV_ERR_INVALID, "null argument");
  if (!p.pool.bounds) return host_error(STARKV_ERR_INVALID, "the kv4 cache was made without page bounds");
  if (a->q_dtype != STARKV_F16 && a->q_dtype != STARKV_BF16)
    return host_error(STARKV_ERR_UNSUPPORTED, "kv4 selection takes fp16 or bf16 queries");
  if (a->batch < 0 || a->batch > 65535 || a->num_queries <= 0 || a->num_q_heads <= 0 ||
      a->num_q_heads % p.pool.heads || a->table_width <= 0 || a->table_stride < 0)
    return host_error(STARKV_ERR_INVALID, "bad batch (at most 65535), query count, head counts or block table");
  if (a->num_first < 0 || a->num_last < 1 || (int64_t)a->num_first + a->num_last > a->num_selected)
    return host_error(STARKV_ERR_INVALID, "num_selected must hold num_first >= 0 and num_last >= 1 pages");
  if (a->batch == 0) return STARKV_OK;
  if (!a->block_table || !a->lengths || !a->pages_out || !a->workspace)
    return host_error(STARKV_ERR_INVALID, "null argument");
  if ((int64_t)a->batch * p.pool.heads > kKv4MaxSegments)
    return host_error(STARKV_ERR_UNSUPPORTED, "kv4 selection takes batch * KV heads up to 65536");
  size_t need = 0;
  starkv_kv4_select_workspace_size(cache, a->batch, a->table_width, &need);
  if (a->workspace_bytes < need) return host_error(STARKV_ERR_WORKSPACE, "kv4 selection workspace too small");
  if (!aligned(4, a->workspace)) return host_error(STARKV_ERR_WORKSPACE, "kv4 selection workspace must be 4-byte aligned");
  if (!aligned(4, a->block_table, a->lengths, a->pages_out))
    return host_error(STARKV_ERR_INVALID, "int32 arguments must be 4-byte aligned");
  if ((rc = check_rows(a->q, a->q_strides, 2, "q rows must be 16-byte aligned"))) return rc;
  p.q = a->q;
  memcpy(p.qs, a->q_strides, sizeof(p.qs));
  p.table = a->block_table;
  p.table_stride = a->table_stride;
  p.lengths = a->lengths;
  p.out = a->pages_out;
  p.counters = (int*)a->workspace;
  p.scores = (float*)((uint8_t*)a->workspace + kKv4MaxSegments * sizeof(int));
  p.batch = a->batch;
  p.queries = a->num_queries;
  p.q_heads = a->num_q_heads;
  p.group = a->num_q_heads / p.pool.heads;
  p.width = a->table_width;
  p.keep = a->num_selected;
  p.first = a->num_first;
  p.last = a->num_last;
  if ((int64_t)p.group * p.queries > 65536) return host_error(STARKV_ERR_UNSUPPORTED, "too many query columns");
  p.q_dtype = a->q_dtype;
  if (((int64_t)a->table_width << p.pool.page_shift) > 0x7fffff00)
    return host_error(STARKV_ERR_UNSUPPORTED, "block table of 2^31 positions or more");
  cudaStream_t st = (cudaStream_t)stream;
  const dim3 grid((unsigned)((p.width + kKv4ScoreChunk - 1) / kKv4ScoreChunk), (unsigned)p.pool.heads, (unsigned)p.batch);
  if (p.width <= 8 * kKv4SelThreads)
    kv4_select_kernel<8><<<grid, kKv4SelThreads, 0, st>>>(p);
  else if (p.width <= 32 * kKv4SelThreads)
    kv4_select_kernel<32><<<grid, kKv4SelThreads, 0, st>>>(p);
  else
    kv4_select_kernel<0><<<grid, kKv4SelThreads, 0, st>>>(p);
  return host_launch_status();
}

}  // extern "C"
