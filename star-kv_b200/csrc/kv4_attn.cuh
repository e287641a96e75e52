// kv4_attn.cuh — attention over the paged 4-bit cache and the page selection.
#pragma once
#include "kv4.cuh"

namespace starkv {

struct Kv4AttnParams {
  Kv4Pool pool;
  const void* q;
  void* out;
  float* lse;
  int64_t qs[3], os[3];
  const int* table;
  int64_t table_stride;
  const int* lengths;
  const float* mask;
  int64_t mask_stride, mask_width;
  const int* pages;
  float scaling;
  int num_selected, out_dtype, batch, queries, q_heads, group, width;
};

// Tokens a sequence may attend to: its length, within the block table.
__device__ __forceinline__ int64_t kv4_length(const Kv4AttnParams& p, int b) {
  const int64_t cap = (int64_t)p.width << p.pool.page_shift;
  int64_t n = p.lengths[b];
  if (n > cap) {
    record_error(p.pool.err, kDevBadPosition);
    n = cap;
  }
  return n < 0 ? 0 : n;
}

__device__ __forceinline__ float kv4_key(const uint8_t* tile, int t, int d) {
  const uint32_t w = *reinterpret_cast<const uint32_t*>(tile + t * 64 + (d % 32 / 8) * 16 + (d / 32) * 4);
  const __half* par = reinterpret_cast<const __half*>(tile + kKv4KParams + t * 16) + d / 32;
  return __fmaf_rn(__half2float(par[0]), (float)((int)((w >> (4 * (d % 8))) & 15u) - 8), __half2float(par[4]));
}

__device__ __forceinline__ float kv4_value(const uint8_t* tile, int t, int d) {
  const uint16_t w = *reinterpret_cast<const uint16_t*>(tile + kKv4VCodes + (t / 2) * 128 + (d % 32 / 4) * 16 +
                                                        (d / 32) * 4 + (t % 2) * 2);
  const __half* par =
      reinterpret_cast<const __half*>(tile + kKv4VParams + (t / 2) * 32 + (d / 32) * 4 + (t % 2) * 2);
  return __fmaf_rn(__half2float(par[0]), (float)((int)((w >> (4 * (d % 4))) & 15u) - 8), __half2float(par[8]));
}

// One CTA of 128 threads per (query column, KV head, sequence): thread t scores
// token t of a block of 128, then accumulates channel t of the values.
template <typename T>
__global__ void __launch_bounds__(128) kv4_attn_kernel(const Kv4AttnParams p) {
  const int head = blockIdx.y, b = blockIdx.z, qi = blockIdx.x / p.group, qh = head * p.group + blockIdx.x % p.group;
  const int tid = threadIdx.x, ps = 1 << p.pool.page_shift;
  __shared__ float q[128], w[128], red[4];
  __shared__ const uint8_t* tiles[8];
  q[tid] = to_f32(reinterpret_cast<const T*>(p.q)[b * p.qs[0] + qi * p.qs[1] + qh * p.qs[2] + tid]);
  const int64_t len = kv4_length(p, b), end = len - p.queries + 1 + qi;
  const int* row = p.table + b * p.table_stride;
  const int* sel = p.pages ? p.pages + ((int64_t)b * p.pool.heads + head) * p.num_selected : nullptr;
  const int64_t n = sel ? (int64_t)p.num_selected * ps : len;   // positions, or slots of the selected pages
  float m = -INFINITY, l = 0.f, acc = 0.f;
  for (int64_t s0 = 0; s0 < n; s0 += 128) {
    __syncthreads();
    if (tid < 8) {
      const int64_t s = s0 + tid * 16;
      const uint8_t* tile = nullptr;
      if (s < n) {
        int64_t ord = s >> p.pool.page_shift;
        if (sel) ord = sel[ord];
        if (ord >= 0 && ord * ps < len) {
          const int page = kv4_page(p.pool, row, ord, p.width);
          if (page >= 0) tile = p.pool.tile(page, head, (int)(s & (ps - 1)) >> 4);
        }
      }
      tiles[tid] = tile;
    }
    __syncthreads();
    const uint8_t* tile = tiles[tid >> 4];
    float x = -INFINITY;
    if (tile) {
      int64_t pos = s0 + tid;
      if (sel) pos = (int64_t)sel[pos >> p.pool.page_shift] * ps + (pos & (ps - 1));
      const float add = pos < end && p.mask && pos < p.mask_width ? p.mask[b * p.mask_stride + pos] : 0.f;
      if (pos < end && add != -INFINITY) {
        float a = 0.f;
        for (int d = 0; d < 128; ++d) a += q[d] * kv4_key(tile, tid & 15, d);
        x = a * p.scaling + add;
      }
    }
    float mx = x;
    for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    if ((tid & 31) == 0) red[tid >> 5] = mx;
    __syncthreads();
    mx = fmaxf(fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3])), m);
    if (mx == -INFINITY) continue;                             // nothing attended to so far (uniform)
    const float e = expf(x - mx), r = expf(m - mx);
    w[tid] = e;
    __syncthreads();
    m = mx;
    l *= r;
    acc *= r;
    for (int t = 0; t < 128; ++t) {
      if (w[t] == 0.f) continue;
      l += w[t];
      acc += w[t] * kv4_value(tiles[t >> 4], t & 15, tid);
    }
  }
  store_from_f32(p.out, p.out_dtype, b * p.os[0] + qi * p.os[1] + qh * p.os[2] + tid, l > 0.f ? acc / l : 0.f);
  if (p.lse && tid == 0) p.lse[((int64_t)b * p.queries + qi) * p.q_heads + qh] = m == -INFINITY ? m : m + logf(l);
}

struct Kv4SelectParams {
  Kv4Pool pool;
  const void* q;
  int64_t qs[3];
  const int* table;
  int64_t table_stride;
  const int* lengths;
  int* out;
  float* scores;
  int batch, queries, q_heads, group, width, keep, first, last;
};

// Order-preserving integer of a score (larger score, larger key; -0 equals 0).
__device__ __forceinline__ uint32_t kv4_key_of(float s) {
  const uint32_t u = __float_as_uint(s + 0.f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// One CTA of 256 threads per (KV head, sequence): scores, then the keep-th largest
// key by bits, then the list in page order.
template <typename T>
__global__ void __launch_bounds__(256) kv4_select_kernel(const Kv4SelectParams p) {
  const int head = blockIdx.x, b = blockIdx.y, tid = threadIdx.x, cols = p.queries * p.group;
  __shared__ int cnt[8];
  __shared__ uint32_t qp[32], qn[32];
  __shared__ float unit;
  const int64_t cap = (int64_t)p.width << p.pool.page_shift;
  int64_t len = p.lengths[b];
  len = len < 0 ? 0 : len > cap ? cap : len;
  const int n = (int)((len + (1 << p.pool.page_shift) - 1) >> p.pool.page_shift);
  const int64_t seg = (int64_t)b * p.pool.heads + head;
  int* out = p.out + seg * p.keep;
  if (n <= p.keep) {
    for (int i = tid; i < p.keep; i += 256) out[i] = i < n ? i : -1;
    return;
  }
  float* sc = p.scores + seg * p.width;
  const int* row = p.table + b * p.table_stride;
  for (int col = 0; col < cols; ++col) {
    __syncthreads();
    if (tid < 32) {
      const T* q = reinterpret_cast<const T*>(p.q) + b * p.qs[0] + (col / p.group) * p.qs[1] +
                   (head * p.group + col % p.group) * p.qs[2] + tid * 4;
      float x[4], a = 0.f;
      for (int i = 0; i < 4; ++i) x[i] = to_f32(q[i]), a = fmaxf(a, fabsf(x[i]));
      for (int o = 16; o > 0; o >>= 1) a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, o));
      const float u = __fdiv_rn(a, 127.f);
      uint32_t wp = 0, wn = 0;
      for (int i = 0; i < 4; ++i) {
        const int c = u > 0.f ? (int)rintf(__fdiv_rn(x[i], u)) : 0;
        wp |= (uint32_t)(c > 0 ? c : 0) << (8 * i);
        wn |= (uint32_t)((c < 0 ? c : 0) & 255) << (8 * i);
      }
      qp[tid] = wp;
      qn[tid] = wn;
      if (tid == 0) unit = u;
    }
    __syncthreads();
    for (int i = tid; i < n; i += 256) {
      float s = -INFINITY;
      if (i < p.first || i >= n - p.last) {
        s = INFINITY;
      } else {
        const int page = kv4_page(p.pool, row, i, p.width);
        if (page >= 0) {
          const int* bd = reinterpret_cast<const int*>(p.pool.bounds + ((int64_t)page * p.pool.heads + head) * 256);
          int dot = 0;
          for (int j = 0; j < 32; ++j) dot = __dp4a((int)qp[j], bd[j], __dp4a((int)qn[j], bd[32 + j], dot));
          s = __fmul_rn((float)dot, unit);
          if (col > 0) s = fmaxf(s, sc[i]);
          if (col < cols - 1) {
            sc[i] = s;
            continue;
          }
          s = __fmul_rn(s, p.pool.bound_scales[(int64_t)page * p.pool.heads + head]);
        }
      }
      sc[i] = s;
    }
  }
  __syncthreads();
  // largest key with at least `keep` scores at or above it
  uint32_t key = 0;
  for (int bit = 31; bit >= 0; --bit) {
    const uint32_t trial = key | (1u << bit);
    int c = 0;
    for (int i = tid; i < n; i += 256) c += kv4_key_of(sc[i]) >= trial;
    c = __reduce_add_sync(0xffffffffu, c);
    if ((tid & 31) == 0) cnt[tid >> 5] = c;
    __syncthreads();
    c = 0;
    for (int i = 0; i < 8; ++i) c += cnt[i];
    if (c >= p.keep) key = trial;
    __syncthreads();
  }
  if (tid == 0) {
    int above = 0, at = 0;
    for (int i = 0; i < n; ++i) above += kv4_key_of(sc[i]) > key;
    int equal = p.keep - above;
    for (int i = 0; i < n && at < p.keep; ++i) {
      const uint32_t k = kv4_key_of(sc[i]);
      if (k > key || (k == key && equal-- > 0)) out[at++] = i;
    }
    for (; at < p.keep; ++at) out[at] = -1;
  }
}

}  // namespace starkv
