// packed_abi.cu — the starkv_packed_* entry points (declared in include/starkv.h):
// argument checks, tensor maps and the launch.  Nothing here allocates device memory
// or synchronises.
#include <cuda_runtime.h>

#include <atomic>
#include <cstring>

#include "host.hpp"
#include "packed_attn.cuh"

using namespace starkv;

namespace {

// Tensor map of (rows, heads, 128) 16-bit values: boxes of 64 channels x `heads_box` heads x `rows_box`
// rows, 128-byte swizzle, zeros past the rows.
int rows_map(CUtensorMap* map, const void* base, int dtype, int64_t rows, int heads, const int64_t* strides, int heads_box,
             int rows_box) {
  const auto encode = host_encode_tiled();
  if (!encode) return host_error(STARKV_ERR_LAUNCH, "cuTensorMapEncodeTiled is not available");
  const cuuint64_t dims[3] = {128, (cuuint64_t)heads, (cuuint64_t)rows};
  // the stride of a dimension of one is never used, but has to be valid
  const cuuint64_t st[2] = {(cuuint64_t)(heads > 1 ? strides[1] : 128) * 2, (cuuint64_t)(rows > 1 ? strides[0] : 128) * 2};
  const cuuint32_t box[3] = {64, (cuuint32_t)heads_box, (cuuint32_t)rows_box}, one[3] = {1, 1, 1};
  const CUresult rc = encode(map, dtype == STARKV_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3,
                             const_cast<void*>(base), dims, st, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
                             CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return rc == CUDA_SUCCESS ? STARKV_OK : host_error(STARKV_ERR_INVALID, "q / k / v cannot be described by a tensor map");
}

// Where calls without an error word of their own report: one word a device, looked up once with that
// device current.
__device__ int g_packed_error;
int packed_error(int** word) {
  static std::atomic<int*> known[64];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return host_launch_status();
  *word = dev < 64 ? known[dev].load(std::memory_order_relaxed) : nullptr;
  if (*word) return STARKV_OK;
  void* found = nullptr;
  if (cudaGetSymbolAddress(&found, g_packed_error) != cudaSuccess) return host_launch_status();
  *word = reinterpret_cast<int*>(found);
  if (dev < 64) known[dev].store(*word, std::memory_order_relaxed);
  return STARKV_OK;
}

template <typename T>
int launch_packed(const PackedParams& p, int grid, const CUtensorMap& q, const CUtensorMap& k, const CUtensorMap& v,
                  cudaStream_t st) {
  auto kern = packed_attn_kernel<T>;
  static std::atomic<uint64_t> ready{0};                       // one bit a device
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return host_launch_status();
  if (dev >= 64 || !(ready.load(std::memory_order_relaxed) >> dev & 1)) {
    cudaFuncAttributes attr;
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kPkSmemBytes) != cudaSuccess ||
        cudaFuncGetAttributes(&attr, kern) != cudaSuccess)
      return host_launch_status();
    // the roles' register shares come out of what the CTA is launched with
    if (attr.numRegs < kPkLaunchRegs) return host_error(STARKV_ERR_UNSUPPORTED, "packed attention was built with too few registers");
    if (dev < 64) ready.fetch_or(1ull << dev);
  }
  kern<<<grid, kPkThreads, kPkSmemBytes, st>>>(p, q, k, v);
  const int rc = host_launch_status();
  // too few keys for any to be cut
  if (rc || p.total_k <= kPkMinPiece * kPkKeys) return rc;
  packed_join_kernel<8><<<4 * grid, 128, 0, st>>>(p);
  return host_launch_status();
}

}  // namespace

extern "C" {

int starkv_packed_workspace_size(size_t* bytes) {
  if (!bytes) return host_error(STARKV_ERR_INVALID, "null argument");
  *bytes = kPkWorkspaceBytes;
  return STARKV_OK;
}

int starkv_packed_read_error(int* out_code, starkv_stream_t stream) {
  if (!out_code) return host_error(STARKV_ERR_INVALID, "null argument");
  int* word = nullptr;
  int rc = host_device(nullptr);
  if (rc || (rc = packed_error(&word))) return rc;
  return starkv_read_device_error(word, out_code, stream);
}

int starkv_packed_attention(const starkv_packed_args* a, starkv_stream_t stream) {
  if (!a) return host_error(STARKV_ERR_INVALID, "null argument");
  if (a->dtype != STARKV_F16 && a->dtype != STARKV_BF16)
    return host_error(STARKV_ERR_UNSUPPORTED, "packed attention takes fp16 or bf16 q / k / v");
  if (a->out_dtype != STARKV_F16 && a->out_dtype != STARKV_BF16 && a->out_dtype != STARKV_F32)
    return host_error(STARKV_ERR_INVALID, "bad out_dtype");
  if (a->batch < 0 || a->total_q < 0 || a->total_k < 0 || a->num_q_heads <= 0 || a->num_kv_heads <= 0 ||
      a->num_q_heads % a->num_kv_heads)
    return host_error(STARKV_ERR_INVALID, "bad batch, row or head counts");
  if (a->total_q > 0x3fffffff || a->total_k > 0x3fffffff) return host_error(STARKV_ERR_UNSUPPORTED, "2^30 rows or more");
  const int group = a->num_q_heads / a->num_kv_heads;
  if (group > 128) return host_error(STARKV_ERR_UNSUPPORTED, "packed attention takes up to 128 query heads a KV head");
  if (!(a->scaling > 0.f) || a->scaling > 1e30f) return host_error(STARKV_ERR_INVALID, "scaling must be positive and finite");
  if (a->batch == 0 || a->total_q == 0) return host_device(nullptr);
  if (!a->q || !a->out || !a->q_start || !a->q_end || !a->k_start || !a->k_end || !a->workspace || (a->total_k && (!a->k || !a->v)))
    return host_error(STARKV_ERR_INVALID, "null argument");
  const uintptr_t ints = (uintptr_t)a->q_start | (uintptr_t)a->q_end | (uintptr_t)a->k_start | (uintptr_t)a->k_end |
                         (uintptr_t)a->lse | (uintptr_t)a->error_word;
  if (ints & 3) return host_error(STARKV_ERR_INVALID, "int32 and fp32 arguments must be 4-byte aligned");
  if (a->workspace_bytes < kPkWorkspaceBytes) return host_error(STARKV_ERR_WORKSPACE, "packed attention workspace too small");
  if ((uintptr_t)a->workspace & 15) return host_error(STARKV_ERR_WORKSPACE, "packed attention workspace must be 16-byte aligned");
  const void* base[4] = {a->q, a->k, a->v, a->out};
  const int64_t* strides[4] = {a->q_strides, a->k_strides, a->v_strides, a->out_strides};
  for (int i = 0; i < 4; ++i) {
    const int eb = i == 3 && a->out_dtype == STARKV_F32 ? 4 : 2;
    bool ok = (uintptr_t)base[i] % 16 == 0;
    for (int d = 0; d < 2; ++d) ok = ok && strides[i][d] >= 0 && strides[i][d] * eb % 16 == 0;
    if (!ok) return host_error(STARKV_ERR_INVALID, "q / k / v / out rows must be 16-byte aligned");
    const int64_t rows = i == 0 || i == 3 ? a->total_q : a->total_k;
    const int heads = i == 0 || i == 3 ? a->num_q_heads : a->num_kv_heads;
    if ((rows > 1 && strides[i][0] == 0) || (heads > 1 && strides[i][1] == 0))
      return host_error(STARKV_ERR_UNSUPPORTED, "packed attention takes no repeated rows or heads (stride 0)");
  }
  PackedParams p;
  memset(&p, 0, sizeof(p));
  p.q_start = a->q_start, p.q_end = a->q_end, p.k_start = a->k_start, p.k_end = a->k_end;
  p.v = a->v;
  p.out = a->out;
  p.lse = a->lse;
  for (int d = 0; d < 2; ++d) p.vs[d] = a->v_strides[d], p.os[d] = a->out_strides[d];
  p.total_q = (int)a->total_q, p.total_k = (int)a->total_k;
  p.batch = a->batch, p.q_heads = a->num_q_heads, p.kv_heads = a->num_kv_heads, p.group = group;
  p.tokens = 128 / group;
  p.causal = a->causal, p.out_dtype = a->out_dtype;
  p.scale_log2 = (float)(a->scaling * 1.4426950408889634);
  p.err = a->error_word;
  p.wait_ns = host_wait_limit();
  p.skip_copy = host_skip_unit();
  p.counters = (int*)a->workspace;
  p.cuts = (PkCuts*)((uint8_t*)a->workspace + kPkCutsAt);
  p.parts = (float*)((uint8_t*)a->workspace + kPkPartsAt);
  // pieces are numbered in 31 bits, each cut a few times at most where there are that many
  const double pieces = ((double)a->total_q / (2 * p.tokens) + a->batch) * a->num_kv_heads;
  if (pieces > 1e8) return host_error(STARKV_ERR_UNSUPPORTED, "too many rows in one call");
  int sms = 0, rc = host_device(&sms);
  if (rc || (!p.err && (rc = packed_error(&p.err)))) return rc;
  CUtensorMap tq, tk, tv;
  memset(&tk, 0, sizeof(tk));
  memset(&tv, 0, sizeof(tv));
  if ((rc = rows_map(&tq, a->q, a->dtype, a->total_q, a->num_q_heads, a->q_strides, group, p.tokens))) return rc;
  if (a->total_k && ((rc = rows_map(&tk, a->k, a->dtype, a->total_k, a->num_kv_heads, a->k_strides, 1, 128)) ||
                     (rc = rows_map(&tv, a->v, a->dtype, a->total_k, a->num_kv_heads, a->v_strides, 1, 128))))
    return rc;
  cudaStream_t st = (cudaStream_t)stream;
  return a->dtype == STARKV_F16 ? launch_packed<__half>(p, sms, tq, tk, tv, st)
                                : launch_packed<__nv_bfloat16>(p, sms, tq, tk, tv, st);
}

}  // extern "C"
