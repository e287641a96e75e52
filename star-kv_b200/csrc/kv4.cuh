// kv4.cuh — the paged 4-bit key / value cache: its tile layout, the quantising
// write with the page bounds, and the read-back.  Layout and quantiser are
// specified in starkv.h.
#pragma once
#include "common.cuh"
#include "sm100.cuh"

namespace starkv {

constexpr int kKv4Tile = 16;                // tokens of a tile
constexpr int kKv4TileBytes = 2560;
constexpr int kKv4VCodes = 1024;            // byte offsets within a tile
constexpr int kKv4KParams = 2048;
constexpr int kKv4VParams = 2304;
constexpr int kKv4MaxPageTiles = 8;         // page_size <= 128

constexpr int kDevBadPage = 0x201;          // page id outside the pool
constexpr int kDevBadPosition = 0x202;      // position outside the block table

struct Kv4Pool {
  uint8_t* data;
  int8_t* bounds;
  float* bound_scales;
  int* err;
  int num_pages, heads, page_tiles, page_shift;   // page_size = 16 * page_tiles = 1 << page_shift
  __device__ __forceinline__ uint8_t* tile(int page, int head, int t) const {
    return data + (((int64_t)page * heads + head) * page_tiles + t) * kKv4TileBytes;
  }
};

// Pool page of page ordinal `ord` of a sequence, or -1 (with the error word set).
__device__ __forceinline__ int kv4_page(const Kv4Pool& pool, const int* __restrict__ row, int64_t ord, int width) {
  if (ord < 0 || ord >= width) {
    record_error(pool.err, kDevBadPosition);
    return -1;
  }
  const int page = __ldg(row + ord);
  if ((unsigned)page >= (unsigned)pool.num_pages) {
    record_error(pool.err, kDevBadPage);
    return -1;
  }
  return page;
}

// Byte offsets within a tile (starkv.h): the s of a token's group in the key parameters (m: 8
// bytes on) and in the value parameters (m: 16 bytes on), and the 16-bit word of four channels
// (quad of a group) of its value codes.
__host__ __device__ constexpr int kv4_kparam(int t, int g) {
  return kKv4KParams + (t & 7) * 32 + (g >> 1) * 16 + (t >> 3) * 4 + (g & 1) * 2;
}
__host__ __device__ constexpr int kv4_vparam(int t, int g) { return kKv4VParams + (t >> 1) * 32 + g * 4 + (t & 1) * 2; }
__host__ __device__ constexpr int kv4_vcode(int t, int g, int quad) {
  return kKv4VCodes + (t >> 3) * 512 + quad * 64 + (t >> 1 & 3) * 16 + g * 4 + (t & 1) * 2;
}

struct Kv4IoParams {
  Kv4Pool pool;
  const void* k;
  const void* v;
  int64_t ks[3], vs[3];
  const int* table;
  int64_t table_stride;
  const int* start;
  const int* count;
  int num_tokens, width, span;              // span: pages (write) or tiles (read) a sequence's range can touch
  int64_t units;                            // read: warps' worth of work
};

// Eight consecutive channels of one token as fp32.
template <typename T>
struct Vec8 {
  uint4 w;
  __device__ __forceinline__ void load(const T* p) { w = __ldcs(reinterpret_cast<const uint4*>(p)); }
  __device__ __forceinline__ void zero() { w = make_uint4(0, 0, 0, 0); }
  __device__ __forceinline__ void get(float* f) const {
    const uint32_t a[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (sizeof(T) == 2) {
        const T lo = *reinterpret_cast<const T*>(&a[i]);
        const uint32_t h = a[i] >> 16;
        const unsigned short hs = (unsigned short)h;
        const T hi = *reinterpret_cast<const T*>(&hs);
        f[2 * i] = to_f32(lo);
        f[2 * i + 1] = to_f32(hi);
      }
    }
  }
};
template <>
struct Vec8<float> {
  float4 a, b;
  __device__ __forceinline__ void load(const float* p) {
    a = __ldcs(reinterpret_cast<const float4*>(p));
    b = __ldcs(reinterpret_cast<const float4*>(p) + 1);
  }
  __device__ __forceinline__ void zero() { a = b = make_float4(0.f, 0.f, 0.f, 0.f); }
  __device__ __forceinline__ void get(float* f) const {
    f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w;
    f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
  }
};

// Quantises a lane's 8 channels; the group of 32 is the lane's aligned group of
// four lanes.  Returns the 8 codes (0..15) as nibbles in channel order.
__device__ __forceinline__ uint32_t kv4_quantise8(float* f, __half& hs, __half& hm) {
  bool nan = false;
  float mn = 65504.f, mx = -65504.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    nan |= f[i] != f[i];
    f[i] = fminf(fmaxf(f[i], -65504.f), 65504.f);
    mn = fminf(mn, f[i]);
    mx = fmaxf(mx, f[i]);
  }
  const unsigned group = 0xfu << (threadIdx.x & 28);
  nan = (__ballot_sync(0xffffffffu, nan) & group) != 0;
#pragma unroll
  for (int o = 1; o <= 2; o <<= 1) {
    mn = fminf(mn, __shfl_xor_sync(0xffffffffu, mn, o));
    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
  }
  hs = __float2half_rn(__fdiv_rn(__fsub_rn(mx, mn), 15.0f));
  if (nan) hs = __float2half_rn(0.f);
  const float s = __half2float(hs);
  hm = __float2half_rn(__fadd_rn(mn, 8.0f * s));
  const float m = __half2float(hm);
  const float inv = s > 0.f ? __frcp_rn(s) : 0.f;
  uint32_t w = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float c = fminf(fmaxf(rintf(__fmul_rn(__fsub_rn(f[i], m), inv)), -8.f), 7.f);
    w |= (uint32_t)((int)c + 8) << (4 * i);
  }
  if (nan) hm = __ushort_as_half((unsigned short)0x7fff);
  return w;
}

// The lane's word of a pair of tokens' value codes: lanes 0-15 hold the even
// token's nibbles (8 channels: quads 2c and 2c + 1 of their group), lanes 16-31 the
// odd token's.  Lanes 0-15 get quad 2c of both tokens, lanes 16-31 quad 2c + 1.
__device__ __forceinline__ uint32_t kv4_pair_word(uint32_t w, int half) {
  const uint32_t o = __shfl_xor_sync(0xffffffffu, w, 16);
  return half ? __byte_perm(o, w, 0x7632) : __byte_perm(w, o, 0x5410);
}

// ---- write: one CTA per (page, KV head) of a sequence's range, one warp per tile.
// Each half-warp takes one token (16 bytes of fp16 per lane), so a group's minimum
// and maximum need two shuffles and every store of codes is a full 128-byte line.
template <typename T>
__global__ void __launch_bounds__(256) kv4_write_kernel(const Kv4IoParams p) {
  const Kv4Pool& pool = p.pool;
  const int head = blockIdx.x % pool.heads, b = blockIdx.y;
  const int64_t start = p.start[b];
  const int64_t count = p.count ? min(max(p.count[b], 0), p.num_tokens) : p.num_tokens;
  if (start < 0) {
    if (threadIdx.x == 0 && count > 0) record_error(pool.err, kDevBadPosition);
    return;
  }
  const int64_t end = start + count;
  const int64_t ord = (start >> pool.page_shift) + blockIdx.x / pool.heads;
  const int64_t base = ord << pool.page_shift;                 // position of the page's slot 0
  if (base >= end) return;
  const int page = kv4_page(pool, p.table + b * p.table_stride, ord, p.width);
  if (page < 0) return;
  const int ps = pool.page_tiles * kKv4Tile;
  const int lo = start > base ? (int)(start - base) : 0, hi = end - base < ps ? (int)(end - base) : ps;
  const bool full = hi == ps && pool.bounds != nullptr;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, half = lane >> 4, l16 = lane & 15;
  const int c = l16 & 3, g = l16 >> 2;
  const int t0 = warp * kKv4Tile;
  __shared__ float red[2][kKv4MaxPageTiles][128];
  float bmax[8], bmin[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) bmax[i] = -INFINITY, bmin[i] = INFINITY;
  if ((t0 < hi && t0 + kKv4Tile > lo) || full) {
    uint8_t* tile = pool.tile(page, head, warp);
    const T* kp = reinterpret_cast<const T*>(p.k) + b * p.ks[0] + head * p.ks[2] + l16 * 8;
    const T* vp = reinterpret_cast<const T*>(p.v) + b * p.vs[0] + head * p.vs[2] + l16 * 8;
    const int64_t first = base + t0 - start;                   // token index of the tile's slot 0
    Vec8<T> kx[8];
    Vec8<T> vx[8];
#pragma unroll
    for (int it = 0; it < 8; ++it) {
      const int t = t0 + 2 * it + half;
      kx[it].zero();
      vx[it].zero();
      if (t >= lo && t < hi) {
        kx[it].load(kp + (first + 2 * it + half) * p.ks[1]);
        vx[it].load(vp + (first + 2 * it + half) * p.vs[1]);
      }
    }
#pragma unroll
    for (int it = 0; it < 8; ++it) {
      const int tt = 2 * it + half, t = t0 + tt;
      const bool mine = t >= lo && t < hi;
      float f[8];
      __half s, m;
      kx[it].get(f);
      uint32_t w = kv4_quantise8(f, s, m);
      uint32_t* kw = reinterpret_cast<uint32_t*>(tile + tt * 64 + c * 16 + g * 4);
      __half* kpar = reinterpret_cast<__half*>(tile + kv4_kparam(tt, g));
      if (mine) {
        *kw = w;
        if (c == 0) kpar[0] = s, kpar[4] = m;
      } else if (full) {                                       // an earlier call's token of this page
        w = *kw;
        s = kpar[0];
        m = kpar[4];
      }
      if (full) {
        const float fs = __half2float(s), fm = __half2float(m);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float x = __fmaf_rn(fs, (float)((int)((w >> (4 * i)) & 15u) - 8), fm);
          bmax[i] = fmaxf(bmax[i], x);
          bmin[i] = fminf(bmin[i], x);
        }
      }
      vx[it].get(f);
      w = kv4_quantise8(f, s, m);
      const uint32_t pw = kv4_pair_word(w, half);
      const uint32_t sm = (uint32_t)__half_as_ushort(s) | ((uint32_t)__half_as_ushort(m) << 16);
      const uint32_t so = __shfl_xor_sync(0xffffffffu, sm, 16);
      const int te = t0 + 2 * it;
      if (te >= lo && te + 1 < hi) {
        *reinterpret_cast<uint32_t*>(tile + kv4_vcode(2 * it, g, 2 * c + half)) = pw;
        if (c == 0)
          *reinterpret_cast<uint32_t*>(tile + kv4_vparam(2 * it, g) + half * 16) =
              half ? __byte_perm(so, sm, 0x7632) : __byte_perm(sm, so, 0x5410);
      } else if (mine) {                                       // the pair's other token is not this call's
        *reinterpret_cast<uint16_t*>(tile + kv4_vcode(tt, g, 2 * c)) = (uint16_t)w;
        *reinterpret_cast<uint16_t*>(tile + kv4_vcode(tt, g, 2 * c + 1)) = (uint16_t)(w >> 16);
        if (c == 0) {
          *reinterpret_cast<__half*>(tile + kv4_vparam(tt, g)) = s;
          *reinterpret_cast<__half*>(tile + kv4_vparam(tt, g) + 16) = m;
        }
      }
    }
  }
  if (!full) return;                                           // uniform over the CTA
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    bmax[i] = fmaxf(bmax[i], __shfl_xor_sync(0xffffffffu, bmax[i], 16));
    bmin[i] = fminf(bmin[i], __shfl_xor_sync(0xffffffffu, bmin[i], 16));
    if (half == 0) red[0][warp][l16 * 8 + i] = bmax[i], red[1][warp][l16 * 8 + i] = bmin[i];
  }
  __syncthreads();
  if (warp != 0) return;
  float up[4], dn[4], a = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int d = lane + 32 * i;
    up[i] = red[0][0][d];
    dn[i] = red[1][0][d];
    for (int w = 1; w < pool.page_tiles; ++w) up[i] = fmaxf(up[i], red[0][w][d]), dn[i] = fminf(dn[i], red[1][w][d]);
    a = fmaxf(a, fmaxf(fabsf(up[i]), fabsf(dn[i])));
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, o));
  const float t = __fdiv_rn(a, 127.f);
  const int64_t at = (int64_t)page * pool.heads + head;
  if (lane == 0) pool.bound_scales[at] = t;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int d = lane + 32 * i;
    const float u = t > 0.f ? fminf(ceilf(__fdiv_rn(up[i], t)), 127.f) : 0.f;
    const float l = t > 0.f ? fmaxf(floorf(__fdiv_rn(dn[i], t)), -127.f) : 0.f;
    pool.bounds[at * 256 + d] = (int8_t)(int)u;
    pool.bounds[at * 256 + 128 + d] = (int8_t)(int)l;
  }
}

// A lane's 8 channels from 8 nibbles in channel order.
__device__ __forceinline__ void kv4_values8(uint32_t w, float s, float m, float* f) {
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] = __fmaf_rn(s, (float)((int)((w >> (4 * i)) & 15u) - 8), m);
}

template <typename T>
__device__ __forceinline__ void kv4_store8(T* dst, const float* f) {
  if constexpr (sizeof(T) == 4) {
    reinterpret_cast<float4*>(dst)[0] = make_float4(f[0], f[1], f[2], f[3]);
    reinterpret_cast<float4*>(dst)[1] = make_float4(f[4], f[5], f[6], f[7]);
  } else {
    T h[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) h[i] = from_f32<T>(f[i]);
    __stcs(reinterpret_cast<uint4*>(dst), *reinterpret_cast<uint4*>(h));
  }
}

// ---- read: one warp per (sequence, tile of positions, KV head), heads fastest.
// The tile comes in whole (five 16-byte loads per lane) and is unpacked from
// shared memory, a half-warp per token.
constexpr int kKv4ReadWarps = 4;

template <typename T>
__global__ void __launch_bounds__(kKv4ReadWarps * 32) kv4_read_kernel(const Kv4IoParams p) {
  __shared__ __align__(16) uint8_t buf[kKv4ReadWarps][kKv4TileBytes];
  const Kv4Pool& pool = p.pool;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, half = lane >> 4, l16 = lane & 15;
  const int64_t unit = (int64_t)blockIdx.x * kKv4ReadWarps + warp;
  if (unit >= p.units) return;
  const int head = (int)(unit % pool.heads);
  const int64_t bt = unit / pool.heads;
  const int b = (int)(bt / p.span);
  const int64_t start = p.start[b];
  const int64_t count = p.count ? min(max(p.count[b], 0), p.num_tokens) : p.num_tokens;
  const int64_t pos0 = (start >> 4 << 4) + (bt % p.span) * kKv4Tile;  // the tile's first position
  const int64_t i0 = pos0 - start;                                    // its output row
  if (i0 >= p.num_tokens) return;
  int page = -1;
  if (i0 < count) {
    if (start < 0)
      record_error(pool.err, kDevBadPosition);
    else
      page = kv4_page(pool, p.table + b * p.table_stride, pos0 >> pool.page_shift, p.width);
  }
  if (page >= 0) {
    const uint4* src = reinterpret_cast<const uint4*>(
        pool.tile(page, head, (int)(pos0 >> 4) & (pool.page_tiles - 1)));
    uint4 w[5];
#pragma unroll
    for (int i = 0; i < 5; ++i) w[i] = __ldcs(src + lane + 32 * i);
#pragma unroll
    for (int i = 0; i < 5; ++i) reinterpret_cast<uint4*>(buf[warp])[lane + 32 * i] = w[i];
    __syncwarp();
  }
  const uint8_t* tile = buf[warp];
  const int c = l16 & 3, g = l16 >> 2;
  T* kp = reinterpret_cast<T*>(const_cast<void*>(p.k)) + b * p.ks[0] + head * p.ks[2] + l16 * 8;
  T* vp = reinterpret_cast<T*>(const_cast<void*>(p.v)) + b * p.vs[0] + head * p.vs[2] + l16 * 8;
#pragma unroll
  for (int it = 0; it < 8; ++it) {
    const int tt = 2 * it + half;
    const int64_t i = i0 + tt;
    if (i < 0 || i >= p.num_tokens) continue;
    float fk[8], fv[8];
    if (page >= 0 && i < count) {
      const __half* kpar = reinterpret_cast<const __half*>(tile + kv4_kparam(tt, g));
      kv4_values8(*reinterpret_cast<const uint32_t*>(tile + tt * 64 + c * 16 + g * 4), __half2float(kpar[0]),
                  __half2float(kpar[4]), fk);
      const uint32_t w = (uint32_t)*reinterpret_cast<const uint16_t*>(tile + kv4_vcode(tt, g, 2 * c)) |
                         ((uint32_t)*reinterpret_cast<const uint16_t*>(tile + kv4_vcode(tt, g, 2 * c + 1)) << 16);
      const __half* vpar = reinterpret_cast<const __half*>(tile + kv4_vparam(tt, g));
      kv4_values8(w, __half2float(vpar[0]), __half2float(vpar[8]), fv);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) fk[j] = fv[j] = 0.f;
    }
    kv4_store8(kp + i * p.ks[1], fk);
    kv4_store8(vp + i * p.vs[1], fv);
  }
}

}  // namespace starkv
