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

// Both halves of a word of two fp16 numbers.
__device__ __forceinline__ float2 kv4_halves(uint32_t a) { return __half22float2(*reinterpret_cast<const __half2*>(&a)); }
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
  // The minimum and maximum (NaN if one value is).
  __device__ __forceinline__ void range(float& mn, float& mx) const {
    if constexpr (sizeof(T) == 4) {
      float f[16];
      get(f);
      mn = mx = f[0];
#pragma unroll
      for (int i = 1; i < 16; ++i) mn = kv4_min_nan(mn, f[i]), mx = kv4_max_nan(mx, f[i]);
    } else {
      using T2 = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
      T2 lo, hi;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint32_t a = word(i);
        const T2 v = *reinterpret_cast<const T2*>(&a);
        lo = i ? __hmin2_nan(lo, v) : v;
        hi = i ? __hmax2_nan(hi, v) : v;
      }
      mn = to_f32(__hmin_nan(lo.x, lo.y));
      mx = to_f32(__hmax_nan(hi.x, hi.y));
    }
  }
  __device__ __forceinline__ uint32_t word(int i) const {
    const uint4& v = w[i >> 2];
    return (i & 3) == 0 ? v.x : (i & 3) == 1 ? v.y : (i & 3) == 2 ? v.z : v.w;
  }
  __device__ __forceinline__ void get(float* f) const {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < 16; ++i) f[i] = __uint_as_float(word(i));
    } else if constexpr (std::is_same<T, __half>::value) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint32_t a = word(i);
        const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&a));
        f[2 * i] = v.x, f[2 * i + 1] = v.y;
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) f[2 * i] = __uint_as_float(word(i) << 16), f[2 * i + 1] = __uint_as_float(word(i) & 0xffff0000u);
    }
  }
};

// Rounding by adding 1.5 * 2^23 + 8: the low bits of the sum are c + 8.
constexpr float kKv4Magic = 12582920.f;

// Codes of a lane's 16 channels (nibbles c + 8 in channel order) and, where BOUNDS, the extremes
// of the values they stand for.
template <bool CLAMP, bool BOUNDS, typename T>
__device__ __forceinline__ void kv4_encode16(const Kv4Row<T>& row, float s, float m, float inv, uint32_t* w, float* bmax,
                                             float* bmin) {
  float f[16];
  row.get(f);
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    uint32_t sum = 0;
#pragma unroll
    for (int i = 7; i >= 0; --i) {
      float x = f[8 * h + i];
      if (CLAMP) x = fminf(fmaxf(x, -65504.f), 65504.f);
      float y = __fmul_rn(__fsub_rn(x, m), inv);
      if (CLAMP) y = fminf(fmaxf(y, -8.f), 7.f);
      y = __fadd_rn(y, kKv4Magic);
      if (BOUNDS) {
        x = __fmaf_rn(s, y - kKv4Magic, m);
        bmax[8 * h + i] = fmaxf(bmax[8 * h + i], x);
        bmin[8 * h + i] = fminf(bmin[8 * h + i], x);
      }
      // sum of 16^i times the bits, whose constant parts are taken off below (modulo 2^32)
      sum = sum * 16u + __float_as_uint(y);
    }
    w[h] = sum - 0x11111111u * 0x4b400000u;
  }
}

// The token that a 16-bit unit of a tile belongs to.
__device__ __forceinline__ int kv4_unit_token(int u) {
  const int o = 2 * u;
  if (o < kKv4VCodes) return o >> 6;
  if (o < kKv4KParams) return (o - kKv4VCodes) / 512 * 8 + (o >> 4 & 3) * 2 + (o >> 1 & 1);
  if (o < kKv4VParams) return (o - kKv4KParams) / 32 + (o >> 2 & 1) * 8;
  return (o - kKv4VParams) / 32 * 2 + (o >> 1 & 1);
}

// ---- write: one CTA per (page, KV head) of a sequence's range, one warp per tile, eight lanes
// per token: half a group a lane.  Of the two lanes of a group one works out the scale of
// the key's group, the other that of the value's.  The tile is put together in shared
// memory and stored 16 bytes a lane, or only its new tokens where others stay.
// Codes can leave [-8, 7] before they are clamped only where fp16 holds s or m coarsely (s
// subnormal, |m| > 512 s) or x is beyond fp16; a warp without such a group skips the clamps.
// 4 prompts of up to 32768 tokens, 8 heads, bf16 (573 MB in and out): 162 us, 3.5 TB/s; bound by
// issue (2000 warp instructions a tile, 2.35 a cycle at 16 warps an SM).  All rows of a tile are
// loaded ahead (two steps ahead: 171 us; 24 warps of 80 registers: 175-197 us).
template <typename T>
__global__ void __launch_bounds__(256, 2) kv4_write_kernel(const Kv4IoParams p) {
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
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int tok = lane >> 3, g = lane >> 1 & 3, part = lane & 1;   // token of a step, group, half of it
  const int ps = pool.page_tiles * kKv4Tile, t0 = warp * kKv4Tile;
  // new tokens: slots [lo, hi) of the page, [a, e) of the tile
  const int lo = start > base ? (int)(start - base) : 0, hi = end - base < ps ? (int)(end - base) : ps;
  const int a = max(lo - t0, 0), e = min(hi - t0, kKv4Tile);
  const bool full = hi == ps && pool.bounds != nullptr;
  __shared__ __align__(16) uint8_t stage[kKv4MaxPageTiles][kKv4TileBytes];
  __shared__ __align__(16) float red[2][kKv4MaxPageTiles][128];
  float bmax[16], bmin[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) bmax[i] = -INFINITY, bmin[i] = INFINITY;
  // the rows of the first steps, before the page is known
  const int64_t first = base + t0 - start + tok;               // token of the lane's row in step 0
  const T* kp = reinterpret_cast<const T*>(p.k) + b * p.ks[0] + first * p.ks[1] + head * p.ks[2] + (lane & 7) * 16;
  const T* vp = reinterpret_cast<const T*>(p.v) + b * p.vs[0] + first * p.vs[1] + head * p.vs[2] + (lane & 7) * 16;
  constexpr int kAhead = sizeof(T) == 2 ? 4 : 1;               // steps loaded ahead; 16 bits: the whole tile
  Kv4Row<T> kx[kAhead], vx[kAhead];
  auto load = [&](int it) {
    const int t = 4 * it + tok;
    Kv4Row<T>&k = kx[it % kAhead], &v = vx[it % kAhead];
    k.zero();
    v.zero();
    if (t >= a && t < e) {
      k.load(kp + 4 * it * p.ks[1]);
      v.load(vp + 4 * it * p.vs[1]);
    }
  };
#pragma unroll
  for (int it = 0; it < kAhead; ++it) load(it);
  const int page = kv4_page(pool, p.table + b * p.table_stride, ord, p.width);
  if (page < 0) return;
  uint8_t* tile = pool.tile(page, head, warp);
  if (a < e) {
    uint8_t* sk = stage[warp] + tok * 64 + part * 32 + g * 4;
    uint8_t* sp = stage[warp] + kKv4KParams + tok * 32 + (g >> 1) * 16 + (g & 1) * 2;
    uint8_t* sv = stage[warp] + kKv4VCodes + (part * 4 + (tok & 1) * 2) * 64 + (tok >> 1) * 16 + g * 4;
    uint8_t* sq = stage[warp] + kKv4VParams + (tok >> 1) * 32 + g * 4 + (tok & 1) * 16;
#pragma unroll
    for (int it = 0; it < 4; ++it) {
      const Kv4Row<T> k = kx[it % kAhead], v = vx[it % kAhead];
      if (it + kAhead < 4) load(it + kAhead);
      if (4 * it >= e || 4 * it + 4 <= a) continue;            // none of these four
      const bool mine = 4 * it + tok >= a && 4 * it + tok < e;
      // ranges: lane part 0 gets the key group's, part 1 the value group's
      float kmn, kmx, vmn, vmx;
      k.range(kmn, kmx);
      v.range(vmn, vmx);
      float mn = __shfl_xor_sync(0xffffffffu, part ? kmn : vmn, 1), mx = __shfl_xor_sync(0xffffffffu, part ? kmx : vmx, 1);
      mn = kv4_min_nan(mn, part ? vmn : kmn);
      mx = kv4_max_nan(mx, part ? vmx : kmx);
      const bool nan = mx != mx, wide = mx > 65504.f || mn < -65504.f;
      mn = fminf(fmaxf(mn, -65504.f), 65504.f);
      mx = fminf(fmaxf(mx, -65504.f), 65504.f);
      const __half hs = __float2half_rn(nan ? 0.f : __fdiv_rn(__fsub_rn(mx, mn), 15.0f));
      const float s = __half2float(hs);
      __half hm = __float2half_rn(__fadd_rn(mn, 8.0f * s));
      const float am = fabsf(__half2float(hm)), inv = s > 0.f ? __frcp_rn(s) : 0.f;
      const bool plain = !nan && !wide && (s == 0.f || (s >= 0x1p-14f && am <= 512.f * s));
      if (nan) hm = __ushort_as_half((unsigned short)0x7fff);
      const uint32_t sm = (uint32_t)__half_as_ushort(hs) | ((uint32_t)__half_as_ushort(hm) << 16);
      const float2 ksm = kv4_halves(__shfl_sync(0xffffffffu, sm, lane & 30)), vsm = kv4_halves(__shfl_sync(0xffffffffu, sm, lane | 1));
      const float kinv = __shfl_sync(0xffffffffu, inv, lane & 30), vinv = __shfl_sync(0xffffffffu, inv, lane | 1);
      uint32_t kw[2], vw[2];
      if (__all_sync(0xffffffffu, plain)) {
        if (full && mine) kv4_encode16<false, true>(k, ksm.x, ksm.y, kinv, kw, bmax, bmin);
        else kv4_encode16<false, false>(k, ksm.x, ksm.y, kinv, kw, bmax, bmin);
        kv4_encode16<false, false>(v, vsm.x, vsm.y, vinv, vw, bmax, bmin);
      } else {
        if (full && mine) kv4_encode16<true, true>(k, ksm.x, ksm.y, kinv, kw, bmax, bmin);
        else kv4_encode16<true, false>(k, ksm.x, ksm.y, kinv, kw, bmax, bmin);
        kv4_encode16<true, false>(v, vsm.x, vsm.y, vinv, vw, bmax, bmin);
      }
      *reinterpret_cast<uint32_t*>(sk + it * 256) = kw[0];
      *reinterpret_cast<uint32_t*>(sk + it * 256 + 16) = kw[1];
      // a pair's other token is eight lanes on: even tokens put together quads 0 and 1 of the half
      // group for both and the pair's s, odd tokens quads 2 and 3 and its m
      const int odd = tok & 1;
      const uint32_t other = __shfl_xor_sync(0xffffffffu, odd ? vw[0] : vw[1], 8);
      const uint32_t even = odd ? other : vw[0], second = odd ? vw[1] : other;
      const int at = (it >> 1) * 512 + (it & 1) * 32;
      *reinterpret_cast<uint32_t*>(sv + at) = __byte_perm(even, second, 0x5410);
      *reinterpret_cast<uint32_t*>(sv + at + 64) = __byte_perm(even, second, 0x7632);
      const uint32_t so = __shfl_xor_sync(0xffffffffu, sm, 8);
      if (part == 0) {
        *reinterpret_cast<__half*>(sp + (it & 1) * 128 + (it >> 1) * 4) = hs;
        *reinterpret_cast<__half*>(sp + (it & 1) * 128 + (it >> 1) * 4 + 8) = hm;
      } else {
        *reinterpret_cast<uint32_t*>(sq + it * 64) = __byte_perm(odd ? so : sm, odd ? sm : so, odd ? 0x7632 : 0x5410);
      }
    }
    __syncwarp();
    if (a == 0 && e == kKv4Tile) {
#pragma unroll
      for (int i = 0; i < 5; ++i)
        reinterpret_cast<uint4*>(tile)[lane + 32 * i] = reinterpret_cast<const uint4*>(stage[warp])[lane + 32 * i];
    } else {
#pragma unroll 4
      for (int u = lane; u < kKv4TileBytes / 2; u += 32) {
        const int t = kv4_unit_token(u);
        if (t >= a && t < e) reinterpret_cast<uint16_t*>(tile)[u] = reinterpret_cast<const uint16_t*>(stage[warp])[u];
      }
    }
  }
  if (!full) return;                                           // uniform over the CTA
  for (int t = tok; t < min(a, kKv4Tile); t += 4) {            // the page's tokens of earlier calls
    const uint32_t* kw = reinterpret_cast<const uint32_t*>(tile + t * 64 + part * 32 + g * 4);
    const __half* kpar = reinterpret_cast<const __half*>(tile + kv4_kparam(t, g));
    const uint32_t old[2] = {kw[0], kw[4]};
    const float s = __half2float(kpar[0]), m = __half2float(kpar[4]);
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const float x = __fmaf_rn(s, (float)((int)((old[i >> 3] >> (4 * (i & 7))) & 15u) - 8), m);
      bmax[i] = fmaxf(bmax[i], x);
      bmin[i] = fminf(bmin[i], x);
    }
  }
  // over the four tokens of a step: first half of the channels stay with lanes of bit 3 clear, and so on
  __syncwarp();
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const bool up = lane & 8;
    const float gx = __shfl_xor_sync(0xffffffffu, up ? bmax[i] : bmax[i + 8], 8);
    const float gn = __shfl_xor_sync(0xffffffffu, up ? bmin[i] : bmin[i + 8], 8);
    bmax[i] = fmaxf(gx, up ? bmax[i + 8] : bmax[i]);
    bmin[i] = fminf(gn, up ? bmin[i + 8] : bmin[i]);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const bool up = lane & 16;
    const float gx = __shfl_xor_sync(0xffffffffu, up ? bmax[i] : bmax[i + 4], 16);
    const float gn = __shfl_xor_sync(0xffffffffu, up ? bmin[i] : bmin[i + 4], 16);
    bmax[i] = fmaxf(gx, up ? bmax[i + 4] : bmax[i]);
    bmin[i] = fminf(gn, up ? bmin[i + 4] : bmin[i]);
  }
  const int ch = (lane & 7) * 16 + (lane >> 3 & 1) * 8 + (lane >> 4) * 4;
  *reinterpret_cast<float4*>(&red[0][warp][ch]) = make_float4(bmax[0], bmax[1], bmax[2], bmax[3]);
  *reinterpret_cast<float4*>(&red[1][warp][ch]) = make_float4(bmin[0], bmin[1], bmin[2], bmin[3]);
  __syncthreads();
  if (warp != 0) return;
  // a lane 4 channels
  float4 up = *reinterpret_cast<const float4*>(&red[0][0][lane * 4]), dn = *reinterpret_cast<const float4*>(&red[1][0][lane * 4]);
  for (int w = 1; w < pool.page_tiles; ++w) {
    const float4 x = *reinterpret_cast<const float4*>(&red[0][w][lane * 4]), y = *reinterpret_cast<const float4*>(&red[1][w][lane * 4]);
    up = make_float4(fmaxf(up.x, x.x), fmaxf(up.y, x.y), fmaxf(up.z, x.z), fmaxf(up.w, x.w));
    dn = make_float4(fminf(dn.x, y.x), fminf(dn.y, y.y), fminf(dn.z, y.z), fminf(dn.w, y.w));
  }
  float top = fmaxf(fmaxf(fmaxf(fabsf(up.x), fabsf(up.y)), fmaxf(fabsf(up.z), fabsf(up.w))),
                    fmaxf(fmaxf(fabsf(dn.x), fabsf(dn.y)), fmaxf(fabsf(dn.z), fabsf(dn.w))));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  const float t = __fdiv_rn(top, 127.f);
  const int64_t at = (int64_t)page * pool.heads + head;
  if (lane == 0) pool.bound_scales[at] = t;
  auto code = [&](float x, bool upper) {
    if (t <= 0.f) return 0u;
    const float y = __fdiv_rn(x, t);
    return (uint32_t)(int)(upper ? fminf(ceilf(y), 127.f) : fmaxf(floorf(y), -127.f)) & 255u;
  };
  uint32_t* bd = reinterpret_cast<uint32_t*>(pool.bounds + at * 256);
  bd[lane] = code(up.x, true) | code(up.y, true) << 8 | code(up.z, true) << 16 | code(up.w, true) << 24;
  bd[32 + lane] = code(dn.x, false) | code(dn.y, false) << 8 | code(dn.z, false) << 16 | code(dn.w, false) << 24;
}

// A lane's 8 channels from 8 nibbles in channel order.  A nibble becomes a float by standing in the
// low byte of 2^23 (one byte permute), and the offset 2^23 + 8 comes off exactly.
__device__ __forceinline__ void kv4_values8(uint32_t w, float s, float m, float* f) {
  const uint32_t even = w & 0x0f0f0f0fu, odd = w >> 4 & 0x0f0f0f0fu;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float c = __uint_as_float(__byte_perm(i & 1 ? odd : even, 0x4b000000u, 0x7440 + (i >> 1)));
    f[i] = __fmaf_rn(s, c - 8388616.f, m);
  }
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
// shared memory, a half-warp per token.  4 x 32768 tokens, 32 heads, fp16 (2.8 GB): 461 us,
// 6.1 TB/s, 95 % of a copy (with integer conversions in place of the byte permutes the ALU
// pipe bound it at 501 us).
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
  T* kp = reinterpret_cast<T*>(const_cast<void*>(p.k)) + b * p.ks[0] + head * p.ks[2] + l16 * 8 + (i0 + half) * p.ks[1];
  T* vp = reinterpret_cast<T*>(const_cast<void*>(p.v)) + b * p.vs[0] + head * p.vs[2] + l16 * 8 + (i0 + half) * p.vs[1];
  // rows of the tile that are written, and those that hold tokens
  const int first = i0 < 0 ? (int)-i0 : 0, rows = (int)min((int64_t)kKv4Tile, p.num_tokens - i0);
  const int live = page >= 0 ? (int)min((int64_t)kKv4Tile, count - i0) : 0;
#pragma unroll
  for (int it = 0; it < 8; ++it) {
    const int tt = 2 * it + half;
    if (tt >= first && tt < rows) {
      float fk[8], fv[8];
      if (tt < live) {
        // the lane's part of an offset is the same in every step, the step's part a constant
        const __half* kpar = reinterpret_cast<const __half*>(tile + kv4_kparam(half, g) + kv4_kparam(2 * it, 0) - kKv4KParams);
        kv4_values8(*reinterpret_cast<const uint32_t*>(tile + half * 64 + c * 16 + g * 4 + it * 128), __half2float(kpar[0]),
                    __half2float(kpar[4]), fk);
        const uint8_t* quads = tile + kv4_vcode(half, g, 2 * c) + kv4_vcode(2 * it, 0, 0) - kKv4VCodes;
        const uint32_t w = (uint32_t)*reinterpret_cast<const uint16_t*>(quads) |
                           ((uint32_t)*reinterpret_cast<const uint16_t*>(quads + 64) << 16);
        const __half* vpar = reinterpret_cast<const __half*>(tile + kv4_vparam(half, g) + it * 32);
        kv4_values8(w, __half2float(vpar[0]), __half2float(vpar[8]), fv);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) fk[j] = fv[j] = 0.f;
      }
      kv4_store8(kp, fk);
      kv4_store8(vp, fv);
    }
    kp += 2 * p.ks[1];
    vp += 2 * p.vs[1];
  }
}

}  // namespace starkv
