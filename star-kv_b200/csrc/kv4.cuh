// kv4.cuh — the paged 4-bit key / value cache: its tile layout, the quantising
// write with the page bounds, and the read-back.  Layout and quantiser are
// specified in starkv.h.
#pragma once
#include <type_traits>

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

__device__ __forceinline__ float kv4_min_nan(float a, float b) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float kv4_max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// Sixteen consecutive channels of one token, as loaded.
template <typename T>
struct Kv4Row {
  static constexpr int kVecs = sizeof(T);   // 16-byte loads
  uint4 w[kVecs];
  __device__ __forceinline__ void load(const T* p) {
#pragma unroll
    for (int i = 0; i < kVecs; ++i) w[i] = __ldcs(reinterpret_cast<const uint4*>(p) + i);
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < kVecs; ++i) w[i] = make_uint4(0, 0, 0, 0);
  }
  // Values, and their minimum and maximum (NaN if one is).
  __device__ __forceinline__ void get(float* f, float& mn, float& mx) const {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        f[4 * i] = __uint_as_float(w[i].x), f[4 * i + 1] = __uint_as_float(w[i].y);
        f[4 * i + 2] = __uint_as_float(w[i].z), f[4 * i + 3] = __uint_as_float(w[i].w);
      }
      mn = mx = f[0];
#pragma unroll
      for (int i = 1; i < 16; ++i) mn = kv4_min_nan(mn, f[i]), mx = kv4_max_nan(mx, f[i]);
    } else {
      using T2 = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
      T2 v[8];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const uint32_t a[4] = {w[i].x, w[i].y, w[i].z, w[i].w};
#pragma unroll
        for (int k = 0; k < 4; ++k) v[4 * i + k] = *reinterpret_cast<const T2*>(&a[k]);
      }
      T2 lo = v[0], hi = v[0];
#pragma unroll
      for (int i = 1; i < 8; ++i) lo = __hmin2_nan(lo, v[i]), hi = __hmax2_nan(hi, v[i]);
      mn = to_f32(__hmin_nan(lo.x, lo.y));
      mx = to_f32(__hmax_nan(hi.x, hi.y));
#pragma unroll
      for (int i = 0; i < 8; ++i) f[2 * i] = to_f32(v[i].x), f[2 * i + 1] = to_f32(v[i].y);
    }
  }
};

// A lane's 16 channels quantised (its neighbour lane ^ 1 has the group's other 16).
struct Kv4Codes {
  uint32_t w[2];                            // nibbles c + 8 in channel order
  __half s, m;
  float r[16];                              // c as a float
};

// Rounding by adding 1.5 * 2^23 + 8: the low bits of the sum are c + 8.
constexpr float kKv4Magic = 12582920.f;

template <bool CLAMP>
__device__ __forceinline__ void kv4_encode16(const float* f, float m, float inv, Kv4Codes& q) {
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    uint32_t w = 0;
#pragma unroll
    for (int i = 7; i >= 0; --i) {
      float x = f[8 * h + i];
      if (CLAMP) x = fminf(fmaxf(x, -65504.f), 65504.f);
      float y = __fmul_rn(__fsub_rn(x, m), inv);
      if (CLAMP) y = fminf(fmaxf(y, -8.f), 7.f);
      y = __fadd_rn(y, kKv4Magic);
      q.r[8 * h + i] = y - kKv4Magic;
      // sum of 16^i times the bits, whose constant parts are taken off below (modulo 2^32)
      w = w * 16u + __float_as_uint(y);
    }
    q.w[h] = w - 0x11111111u * 0x4b400000u;
  }
}

// The scale, centre and codes of a row's 16 channels.  Codes can leave [-8, 7] before they are
// clamped only where fp16 holds s or m coarsely (s subnormal, |m| > 512 s) or x is beyond
// fp16; a warp without such a group skips the clamps (3 of 8 instructions a value).
template <typename T>
__device__ __forceinline__ void kv4_quantise16(const Kv4Row<T>& row, Kv4Codes& q) {
  float f[16], mn, mx;
  row.get(f, mn, mx);
  mn = kv4_min_nan(mn, __shfl_xor_sync(0xffffffffu, mn, 1));
  mx = kv4_max_nan(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
  const bool nan = mx != mx, wide = mx > 65504.f || mn < -65504.f;
  mn = fminf(fmaxf(mn, -65504.f), 65504.f);
  mx = fminf(fmaxf(mx, -65504.f), 65504.f);
  q.s = __float2half_rn(nan ? 0.f : __fdiv_rn(__fsub_rn(mx, mn), 15.0f));
  const float s = __half2float(q.s);
  q.m = __float2half_rn(__fadd_rn(mn, 8.0f * s));
  const float m = __half2float(q.m), inv = s > 0.f ? __frcp_rn(s) : 0.f;
  const bool plain = s == 0.f || (s >= 0x1p-14f && fabsf(m) <= 512.f * s);
  if (__all_sync(0xffffffffu, plain && !wide && !nan))
    kv4_encode16<false>(f, m, inv, q);
  else
    kv4_encode16<true>(f, m, inv, q);
  if (nan) q.m = __ushort_as_half((unsigned short)0x7fff);
}

// ---- write: one CTA per (page, KV head) of a sequence's range, one warp per tile, eight lanes
// per token: half a group a lane, so that a group's minimum and maximum need one shuffle and
// its scale is worked out twice, not eight times.  A full tile is put together in shared
// memory and stored 16 bytes a lane; of a part of one, each lane stores its own words.
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
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int tok = lane >> 3, g = lane >> 1 & 3, part = lane & 1;   // token of a step, group, half of it
  const int t0 = warp * kKv4Tile;
  __shared__ __align__(16) uint8_t stage[kKv4MaxPageTiles][kKv4TileBytes];
  __shared__ float red[2][kKv4MaxPageTiles][128];
  float bmax[16], bmin[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) bmax[i] = -INFINITY, bmin[i] = INFINITY;
  const bool whole = t0 >= lo && t0 + kKv4Tile <= hi;
  if ((t0 < hi && t0 + kKv4Tile > lo) || full) {
    uint8_t* tile = pool.tile(page, head, warp);
    uint8_t* to = whole ? stage[warp] : tile;
    const T* kp = reinterpret_cast<const T*>(p.k) + b * p.ks[0] + head * p.ks[2] + (lane & 7) * 16;
    const T* vp = reinterpret_cast<const T*>(p.v) + b * p.vs[0] + head * p.vs[2] + (lane & 7) * 16;
    const int64_t first = base + t0 - start;                   // token index of the tile's slot 0
    Kv4Row<T> kx[4], vx[4];
#pragma unroll
    for (int it = 0; it < 4; ++it) {
      const int t = t0 + 4 * it + tok;
      kx[it].zero();
      vx[it].zero();
      if (t >= lo && t < hi) {
        kx[it].load(kp + (first + 4 * it + tok) * p.ks[1]);
        vx[it].load(vp + (first + 4 * it + tok) * p.vs[1]);
      }
    }
#pragma unroll
    for (int it = 0; it < 4; ++it) {
      const int tt = 4 * it + tok, t = t0 + tt;
      const bool mine = t >= lo && t < hi;
      if (!full && (t0 + 4 * it >= hi || t0 + 4 * it + 4 <= lo)) continue;   // none of these four
      Kv4Codes q;
      kv4_quantise16(kx[it], q);
      uint32_t* kw = reinterpret_cast<uint32_t*>(to + tt * 64 + part * 32 + g * 4);
      __half* kpar = reinterpret_cast<__half*>(to + kv4_kparam(tt, g));
      if (mine) {
        kw[0] = q.w[0];
        kw[4] = q.w[1];
        if (part == 0) kpar[0] = q.s;
        else kpar[4] = q.m;
      } else if (full) {                                       // an earlier call's token of this page
        const uint32_t old[2] = {kw[0], kw[4]};
        q.s = kpar[0];
        q.m = kpar[4];
#pragma unroll
        for (int i = 0; i < 16; ++i) q.r[i] = (float)((int)((old[i >> 3] >> (4 * (i & 7))) & 15u) - 8);
      }
      if (full) {
        const float fs = __half2float(q.s), fm = __half2float(q.m);
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const float x = __fmaf_rn(fs, q.r[i], fm);
          bmax[i] = fmaxf(bmax[i], x);
          bmin[i] = fminf(bmin[i], x);
        }
      }
      kv4_quantise16(vx[it], q);
      // the pair's other token is eight lanes on: even tokens take quads 0 and 1 of the half group
      // for both, odd tokens quads 2 and 3
      const int odd = tok & 1;
      const uint32_t other = __shfl_xor_sync(0xffffffffu, odd ? q.w[0] : q.w[1], 8);
      const uint32_t sm = (uint32_t)__half_as_ushort(q.s) | ((uint32_t)__half_as_ushort(q.m) << 16);
      const uint32_t so = __shfl_xor_sync(0xffffffffu, sm, 8);
      const int te = t - odd;                                  // the pair's even token
      if (te >= lo && te + 1 < hi) {
        const uint32_t even = odd ? other : q.w[0], second = odd ? q.w[1] : other;
        uint32_t* vw = reinterpret_cast<uint32_t*>(to + kv4_vcode(tt & ~1, g, part * 4 + odd * 2));
        vw[0] = __byte_perm(even, second, 0x5410);
        vw[16] = __byte_perm(even, second, 0x7632);
        const uint32_t pe = odd ? so : sm, po = odd ? sm : so;
        if (part == 0)
          *reinterpret_cast<uint32_t*>(to + kv4_vparam(tt & ~1, g) + odd * 16) = __byte_perm(pe, po, odd ? 0x7632 : 0x5410);
      } else if (mine) {                                       // the pair's other token is not this call's
#pragma unroll
        for (int k = 0; k < 4; ++k)
          *reinterpret_cast<uint16_t*>(tile + kv4_vcode(tt, g, part * 4 + k)) = (uint16_t)(q.w[k >> 1] >> (16 * (k & 1)));
        __half* vpar = reinterpret_cast<__half*>(tile + kv4_vparam(tt, g));
        if (part == 0) vpar[0] = q.s;
        else vpar[8] = q.m;
      }
    }
    if (whole) {
      __syncwarp();
#pragma unroll
      for (int i = 0; i < 5; ++i)
        reinterpret_cast<uint4*>(tile)[lane + 32 * i] = reinterpret_cast<const uint4*>(stage[warp])[lane + 32 * i];
    }
  }
  if (!full) return;                                           // uniform over the CTA
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    bmax[i] = fmaxf(bmax[i], __shfl_xor_sync(0xffffffffu, bmax[i], 8));
    bmin[i] = fminf(bmin[i], __shfl_xor_sync(0xffffffffu, bmin[i], 8));
    bmax[i] = fmaxf(bmax[i], __shfl_xor_sync(0xffffffffu, bmax[i], 16));
    bmin[i] = fminf(bmin[i], __shfl_xor_sync(0xffffffffu, bmin[i], 16));
    if (tok == 0) red[0][warp][lane * 16 + i] = bmax[i], red[1][warp][lane * 16 + i] = bmin[i];
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
