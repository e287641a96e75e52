// kv4_attn.cuh — attention over the paged 4-bit cache and the page selection.
//
// Attention.  x_t = q.k_t in the log2 domain, out = sum_t 2^(x_t - m) v_t / sum_t
// 2^(x_t - m) in one pass with a running maximum m per query column (a query token
// of a query head).  A warp takes tiles of 16 tokens of one KV head against all the
// columns that share it, so the cache is read once for up to 16 of them.
//
// Both products run on mma.sync m16n8k16 straight from the packed codes: a word's
// nibbles masked to 0x000f000f / 0x00f000f0 are two fp16 subnormals c * 2^-24 /
// c * 2^-20, exact operands, so unpacking costs 5 integer instructions per 8 values
// and no conversion.  (tcgen05 would need the codes widened into shared or tensor
// memory first; with one to 16 columns the work is bound by the cache's bytes, at
// 25-100 flop a byte, and the legacy instructions keep up.)
//   Scores: tokens are rows, columns are columns.  Per group of 32 channels
//     d_g = sum c' q - 8 sum q   (c' = c + 8 stored; the second term is the
//                                 accumulator's start value)
//     x = sum_g s_g d_g + sum_g m_g sum q_g   (the last by one more mma, with
//                                 sum q_g split into two fp16 parts)
//   Values: channels are rows, tokens are summed.  w' = fp16(w) times s_g rounds once
//     more to fp16 (two roundings of at most 2^-11 on a softmax weight), then
//     o = sum (w' s_g) c' - 8 sum (w' s_g) + sum w' m_g,
//     where the second and third sums share one accumulator tile (rows 8 + g and g).
//     The -8 uses the same rounded w' s_g, so the rounding acts on s c, not on
//     s (c + 8).  w' is scaled by 2^(15 - e), e >= 0 the exponent that keeps every
//     s_g seen so far <= 2^e, so that neither small weights nor large s leave fp16.
//
// Work split.  All (sequence, KV head, column block) segments form one line of
// tiles; CTA i of a grid of one CTA per SM takes an equal stretch of it, its warps
// equal parts of that, whatever the lengths are (they are read on the GPU).  A warp
// that holds a whole segment writes its output; other pieces merge in shared memory,
// and what a CTA does not hold whole goes to the workspace, where the CTA that
// arrives last merges it in CTA order (the same result every time).
#pragma once
#include "kv4.cuh"

namespace starkv {

constexpr int kKv4Warps = 8;
constexpr int kKv4StageTiles = 4;
constexpr int kKv4Stages = 2;
constexpr int kKv4StageBytes = kKv4StageTiles * kKv4TileBytes;
constexpr int kKv4MaxGrid = 1024;           // CTAs the workspace has room for
constexpr int kKv4MinTiles = kKv4Warps;     // smallest stretch of a CTA
constexpr int kKv4MaxCols = 16;
constexpr size_t kKv4PartFloats = kKv4MaxCols * 130;   // one piece: o (cols, 128), meff (cols), l (cols)
constexpr size_t kKv4CounterBytes = kKv4MaxGrid * sizeof(int);

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
  int* counters;                            // (kKv4MaxGrid) zero between calls
  float* parts;                             // (grid, 2, kKv4PartFloats)
  float scaling;
  int num_selected, q_dtype, out_dtype, batch, queries, q_heads, group, width, col_blocks;
};

__device__ __forceinline__ void kv4_mma(float* d, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void kv4_mma8(float* d, uint32_t a0, uint32_t a1, uint32_t b0) {
  asm volatile("mma.sync.aligned.m16n8k8.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5}, {%6}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a0), "r"(a1), "r"(b0));
}
__device__ __forceinline__ uint32_t kv4_transpose(uint32_t a) {
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}
__device__ __forceinline__ float kv4_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t kv4_half2(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t kv4_hmul2(uint32_t a, uint32_t b) {
  const __half2 h = __hmul2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float2 kv4_float2(uint32_t a) {
  return __half22float2(*reinterpret_cast<const __half2*>(&a));
}

// Tokens of a sequence, within the block table.
__device__ __forceinline__ int64_t kv4_length(const Kv4AttnParams& p, int b) {
  const int64_t cap = (int64_t)p.width << p.pool.page_shift;
  int64_t n = __ldg(p.lengths + b);
  if (n > cap) {
    record_error(p.pool.err, kDevBadPosition);
    n = cap;
  }
  return n < 0 ? 0 : n;
}
// Tiles of one of its segments.
__device__ __forceinline__ int kv4_tiles(const Kv4AttnParams& p, int64_t len) {
  if (p.pages) return len > 0 ? p.num_selected * p.pool.page_tiles : 0;
  return (int)((len + kKv4Tile - 1) >> 4);
}

// Position on the line of tiles.
struct Kv4Cursor {
  int b, hc, t, tiles;                      // sequence, KV head * col_blocks + column block, tile, tiles of the segment
  int64_t len, left;                        // the sequence's length; tiles left of the warp's stretch
  __device__ __forceinline__ int take() const {
    int n = tiles - t < kKv4StageTiles ? tiles - t : kKv4StageTiles;
    return left < n ? (int)left : n;
  }
  __device__ __forceinline__ void advance(const Kv4AttnParams& p, int n) {
    t += n;
    left -= n;
    if (t < tiles || left <= 0) return;
    t = 0;
    if (++hc < p.pool.heads * p.col_blocks) return;
    hc = 0;
    tiles = 0;
    while (tiles == 0 && b + 1 < p.batch) {
      len = kv4_length(p, ++b);
      tiles = kv4_tiles(p, len);
    }
  }
};

// Writes 4 channels of one column's output, and its log-sum-exp once.
__device__ __forceinline__ void kv4_store_out(const Kv4AttnParams& p, int b, int hc, int col, int cols, int d, float4 o,
                                              float meff, float l) {
  const int head = hc / p.col_blocks, gcol = (hc % p.col_blocks) * cols + col;
  if (gcol >= p.group * p.queries) return;
  const int qi = gcol / p.group, qh = head * p.group + gcol % p.group;
  const float inv = l > 0.f ? 1.f / l : l == 0.f ? 0.f : l;    // a NaN stays one
  o.x *= inv, o.y *= inv, o.z *= inv, o.w *= inv;
  const int64_t at = b * p.os[0] + qi * p.os[1] + qh * p.os[2] + d;
  if (p.out_dtype == STARKV_F32) {
    *reinterpret_cast<float4*>(reinterpret_cast<float*>(p.out) + at) = o;
  } else if (p.out_dtype == STARKV_F16) {
    *reinterpret_cast<uint2*>(reinterpret_cast<__half*>(p.out) + at) = make_uint2(kv4_half2(o.x, o.y), kv4_half2(o.z, o.w));
  } else {
    __nv_bfloat162 h[2] = {__floats2bfloat162_rn(o.x, o.y), __floats2bfloat162_rn(o.z, o.w)};
    *reinterpret_cast<uint2*>(reinterpret_cast<__nv_bfloat16*>(p.out) + at) = *reinterpret_cast<uint2*>(h);
  }
  if (p.lse && d == 0)
    p.lse[((int64_t)b * p.queries + qi) * p.q_heads + qh] =
        l == 0.f ? -INFINITY : (meff + log2f(l)) * 0.69314718055994531f;
}

// Weight of a piece with exponent base m against the joint base.
__device__ __forceinline__ float kv4_weight(float m, float joint) {
  return m == -INFINITY ? 0.f : exp2f(m - joint);
}

struct Kv4Piece {
  int64_t start;                            // first tile of its segment on the line
  int b, hc, tiles, used;
};

template <int NT>
struct Kv4AttnSmem {
  static constexpr int kCols = NT * 8;
  alignas(128) uint8_t stage[kKv4Warps][kKv4Stages][kKv4StageBytes];
  alignas(16) float head_o[kKv4Warps][kCols * 128];
  float meff[2 * kKv4Warps][kCols], l[2 * kKv4Warps][kCols];
  alignas(8) uint64_t bar[kKv4Warps][kKv4Stages];
  int pos[kKv4Warps][kKv4Stages][kKv4StageTiles];   // position of a staged tile's first token, -1: not staged
  Kv4Piece piece[2 * kKv4Warps];
  int64_t scan[kKv4Warps];
  int64_t base[kKv4Warps];                  // first tile of the warp's first sequence
  int first[kKv4Warps];                     // that sequence
  int last;
  // o of piece i: the first piece of a warp has its own space, the second lies over the warp's stages
  __device__ __forceinline__ float* o(int i) {
    return i & 1 ? reinterpret_cast<float*>(stage[i >> 1][0]) : head_o[i >> 1];
  }
};

template <int NT, bool MASK>
__global__ void __launch_bounds__(kKv4Warps * 32, 1) kv4_attn_kernel(const Kv4AttnParams p) {
  extern __shared__ __align__(128) uint8_t smem_raw[];
  using Smem = Kv4AttnSmem<NT>;
  constexpr int kCols = Smem::kCols;
  Smem& sm = *reinterpret_cast<Smem*>(smem_raw);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, r = lane >> 2, c = lane & 3;
  const int HC = p.pool.heads * p.col_blocks, ps = 1 << p.pool.page_shift;

  // ---- the line of tiles: total, this CTA's stretch, the warps' first sequences
  const int per_thread = (p.batch + kKv4Warps * 32 - 1) / (kKv4Warps * 32);
  const int b_lo = tid * per_thread;
  int64_t mine = 0;
  for (int b = b_lo; b < b_lo + per_thread && b < p.batch; ++b) mine += (int64_t)kv4_tiles(p, kv4_length(p, b)) * HC;
  int64_t upto = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t y = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += y;
  }
  if (lane == 31) sm.scan[warp] = upto;
  if (lane < kKv4Stages) mbar_init(&sm.bar[warp][lane], 1);
  if (lane < 2) sm.piece[2 * warp + lane].used = 0;
  fence_mbar_init();
  __syncthreads();
  int64_t total = 0;
#pragma unroll
  for (int w = 0; w < kKv4Warps; ++w) {
    if (w < warp) upto += sm.scan[w];
    total += sm.scan[w];
  }
  int64_t per = (total + gridDim.x - 1) / gridDim.x;
  if (per < kKv4MinTiles) per = kKv4MinTiles;
  const int64_t c0 = blockIdx.x * per < total ? blockIdx.x * per : total;
  const int64_t c1 = c0 + per < total ? c0 + per : total;
#pragma unroll
  for (int w = 0; w < kKv4Warps; ++w) {
    const int64_t g = c0 + (c1 - c0) * w / kKv4Warps;
    if (g >= upto - mine && g < upto) {
      int64_t base = upto - mine;
      int b = b_lo;
      for (; b + 1 < p.batch; ++b) {
        const int64_t n = (int64_t)kv4_tiles(p, kv4_length(p, b)) * HC;
        if (g < base + n) break;
        base += n;
      }
      sm.first[w] = b;
      sm.base[w] = base;
    }
  }
  // sequences without a tile: nothing to attend to
  for (int b = blockIdx.x; b < p.batch; b += gridDim.x)
    if (kv4_length(p, b) == 0)
      for (int i = tid; i < HC * kCols * 32; i += kKv4Warps * 32)
        kv4_store_out(p, b, i / (kCols * 32), i / 32 % kCols, kCols, i % 32 * 4, make_float4(0.f, 0.f, 0.f, 0.f), 0.f, 0.f);
  __syncthreads();
  if (c0 >= c1) return;

  const int64_t g0 = c0 + (c1 - c0) * warp / kKv4Warps, g1 = c0 + (c1 - c0) * (warp + 1) / kKv4Warps;
  if (g0 < g1) {
    Kv4Cursor use, get;
    use.b = sm.first[warp];
    use.len = kv4_length(p, use.b);
    use.tiles = kv4_tiles(p, use.len);
    const int64_t off = g0 - sm.base[warp];
    use.hc = use.tiles ? (int)(off / use.tiles) : 0;
    use.t = use.tiles ? (int)(off % use.tiles) : 0;
    use.left = g1 - g0;
    get = use;
    int64_t seg_start = g0 - use.t;         // the segment's first tile on the line

    // Issues the copies of the next tiles into a stage.
    auto fetch = [&](int slot) {
      if (get.left <= 0) return;
      const int n = get.take();
      if (n <= 0) return;
      const uint8_t* src = nullptr;
      int pos = -1;
      if (lane < n) {
        const int t = get.t + lane;
        int64_t ord = t >> (p.pool.page_shift - 4);
        if (p.pages)
          ord = __ldg(p.pages + ((int64_t)get.b * p.pool.heads + get.hc / p.col_blocks) * p.num_selected + ord);
        if (ord >= 0 && ord * ps < get.len) {
          const int in_page = t & (p.pool.page_tiles - 1);
          const int page = kv4_page(p.pool, p.table + get.b * p.table_stride, ord, p.width);
          if (page >= 0 && ord * ps + in_page * kKv4Tile < get.len) {
            pos = (int)(ord * ps) + in_page * kKv4Tile;
            src = p.pool.tile(page, get.hc / p.col_blocks, in_page);
          }
        }
      }
      const unsigned have = __ballot_sync(0xffffffffu, src != nullptr);
      if (lane < kKv4StageTiles) sm.pos[warp][slot][lane] = pos;
      if (lane == 0) mbar_arrive_expect_tx(&sm.bar[warp][slot], __popc(have) * kKv4TileBytes);
      __syncwarp();
      if (src) bulk_g2s(sm.stage[warp][slot] + lane * kKv4TileBytes, src, kKv4TileBytes, &sm.bar[warp][slot]);
      get.advance(p, n);
    };
#pragma unroll
    for (int s = 0; s < kKv4Stages; ++s) fetch(s);

    uint32_t qb[NT][4][4], qm[NT];          // B operands of the scores: 16 * q or q by nibble; sums of q
    float cq[NT][4][2], cs[NT][2];          // -8 sum q; scale of a column's scores (log2 domain)
    int end[NT][2];                         // first position a column does not attend to
    float o[8][NT][4], z[NT][4], m[NT][2], l[NT][2];
    int e_run = 0, npieces = 0;
    bool ok = true;
    int64_t done = 0;
    bool fresh = true;

    for (int k = 0; done < g1 - g0; ++k) {
      const int slot = k % kKv4Stages;
      if (fresh) {                          // a new segment: its queries
        fresh = false;
        const int head = use.hc / p.col_blocks, cb = use.hc % p.col_blocks;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          const int gcol = cb * kCols + nt * 8 + r;
          float f[32];
          if (gcol < p.group * p.queries) {
            const int64_t at = use.b * p.qs[0] + (gcol / p.group) * p.qs[1] + (head * p.group + gcol % p.group) * p.qs[2] + c * 8;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const uint4 w = __ldg(reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(p.q) + at + j * 32));
              const uint32_t a[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                if (p.q_dtype == STARKV_F16) {
                  const float2 h = kv4_float2(a[i]);
                  f[j * 8 + 2 * i] = h.x;
                  f[j * 8 + 2 * i + 1] = h.y;
                } else {
                  f[j * 8 + 2 * i] = __uint_as_float(a[i] << 16);
                  f[j * 8 + 2 * i + 1] = __uint_as_float(a[i] & 0xffff0000u);
                }
              }
            }
          } else {
#pragma unroll
            for (int i = 0; i < 32; ++i) f[i] = 0.f;
          }
          float a = 0.f;
#pragma unroll
          for (int i = 0; i < 32; ++i) a = fmaxf(a, fabsf(f[i]));
          a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, 1));
          a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, 2));
          // q scaled by a power of two to [512, 1024) in magnitude, the scaling's sign with it; a
          // column whose scores vanish (q or scaling below 2^-100) becomes zero
          float up = 0.f, scale = 1.f;
          if (a >= 0x1p-100f && fabsf(p.scaling) >= 0x1p-100f) {
            const int ex = (__float_as_int(a) >> 23) - 127;
            up = __int_as_float((127 + 9 - ex) << 23);
            scale = fabsf(p.scaling) * 1.4426950408889634f * __int_as_float((127 - 9 + ex > 0 ? 127 - 9 + ex : 1) << 23);
            if (p.scaling < 0.f) up = -up;
          } else if (a != a) {
            up = a;
          }
          float sum[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            sum[j] = 0.f;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              f[j * 8 + i] *= up;
              sum[j] += f[j * 8 + i];
            }
            qb[nt][j][0] = kv4_half2(f[j * 8] * 16.f, f[j * 8 + 4] * 16.f);
            qb[nt][j][1] = kv4_half2(f[j * 8 + 1], f[j * 8 + 5]);
            qb[nt][j][2] = kv4_half2(f[j * 8 + 2] * 16.f, f[j * 8 + 6] * 16.f);
            qb[nt][j][3] = kv4_half2(f[j * 8 + 3], f[j * 8 + 7]);
            sum[j] += __shfl_xor_sync(0xffffffffu, sum[j], 1);
            sum[j] += __shfl_xor_sync(0xffffffffu, sum[j], 2);
          }
          const float s0 = c & 1 ? sum[2] : sum[0], s1 = c & 1 ? sum[3] : sum[1];
          const float h0 = __half2float(__float2half_rn(s0)), h1 = __half2float(__float2half_rn(s1));
          qm[nt] = c & 2 ? kv4_half2(s0 - h0, s1 - h1) : kv4_half2(h0, h1);
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const int from = (2 * c + u) * 4;
#pragma unroll
            for (int j = 0; j < 4; ++j) cq[nt][j][u] = -8.f * 0x1p-20f * __shfl_sync(0xffffffffu, sum[j], from);
            cs[nt][u] = __shfl_sync(0xffffffffu, scale, from);
            const int gc = cb * kCols + nt * 8 + 2 * c + u;
            end[nt][u] = (int)use.len - p.queries + 1 + gc / p.group;
            m[nt][u] = -INFINITY;
            l[nt][u] = 0.f;
          }
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            z[nt][i] = 0.f;
#pragma unroll
            for (int mt = 0; mt < 8; ++mt) o[mt][nt][i] = 0.f;
          }
        }
        e_run = 0;
      }
      const int n = use.take();
      if (n <= 0) break;                    // lengths that changed under the kernel
      // a wait that runs out is recorded; what follows waits briefly and computes on what is there
      if (!mbar_wait(&sm.bar[warp][slot], (k / kKv4Stages) & 1, ok ? kWaitLimitNs : 1000000ull)) {
        ok = false;
        if (lane == 0) record_error(p.pool.err, kDevWaitCopy);
      }
      const uint8_t* stage = sm.stage[warp][slot];
      int pos[kKv4StageTiles];
#pragma unroll
      for (int i = 0; i < kKv4StageTiles; ++i) pos[i] = i < n ? sm.pos[warp][slot][i] : -1;
      const int len = (int)use.len, all_end = len - p.queries + 1;

      // ---- scores
      float x[kKv4StageTiles][NT][4];
      unsigned keep[kKv4StageTiles];        // MASK: positions of the tile that are not masked out
#pragma unroll
      for (int i = 0; i < kKv4StageTiles; ++i) {
        keep[i] = 0xffffu;
        if (pos[i] < 0) {
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int u = 0; u < 4; ++u) x[i][nt][u] = -INFINITY;
          continue;
        }
        const uint8_t* tl = stage + i * kKv4TileBytes;
        const uint4 ka = *reinterpret_cast<const uint4*>(tl + r * 64 + c * 16);
        const uint4 kb = *reinterpret_cast<const uint4*>(tl + (r + 8) * 64 + c * 16);
        const uint4 pa = *reinterpret_cast<const uint4*>(tl + kKv4KParams + r * 16);
        const uint4 pb = *reinterpret_cast<const uint4*>(tl + kKv4KParams + (r + 8) * 16);
        const uint32_t wa[4] = {ka.x, ka.y, ka.z, ka.w}, wb[4] = {kb.x, kb.y, kb.z, kb.w};
        const float2 sa01 = kv4_float2(pa.x), sa23 = kv4_float2(pa.y), sb01 = kv4_float2(pb.x), sb23 = kv4_float2(pb.y);
        const float sa[4] = {sa01.x, sa01.y, sa23.x, sa23.y}, sb[4] = {sb01.x, sb01.y, sb23.x, sb23.y};
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int u = 0; u < 4; ++u) x[i][nt][u] = 0.f;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t a0 = wa[j] & 0x000f000fu, a1 = wb[j] & 0x000f000fu, a2 = wa[j] & 0x00f000f0u,
                         a3 = wb[j] & 0x00f000f0u;
          const uint32_t ua = wa[j] >> 8, ub = wb[j] >> 8;
          const uint32_t b0 = ua & 0x000f000fu, b1 = ub & 0x000f000fu, b2 = ua & 0x00f000f0u, b3 = ub & 0x00f000f0u;
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            float d[4] = {cq[nt][j][0], cq[nt][j][1], cq[nt][j][0], cq[nt][j][1]};
            kv4_mma(d, a0, a1, a2, a3, qb[nt][j][0], qb[nt][j][1]);
            kv4_mma(d, b0, b1, b2, b3, qb[nt][j][2], qb[nt][j][3]);
            x[i][nt][0] = fmaf(sa[j], d[0], x[i][nt][0]);
            x[i][nt][1] = fmaf(sa[j], d[1], x[i][nt][1]);
            x[i][nt][2] = fmaf(sb[j], d[2], x[i][nt][2]);
            x[i][nt][3] = fmaf(sb[j], d[3], x[i][nt][3]);
          }
        }
        float add0 = 0.f, add1 = 0.f;
        if (MASK) {
          const float* row = p.mask + use.b * p.mask_stride;
          const int t0 = pos[i] + r, t1 = t0 + 8;
          if (t0 < len && t0 < p.mask_width) add0 = __ldg(row + t0);
          if (t1 < len && t1 < p.mask_width) add1 = __ldg(row + t1);
          // one bit a token (the four lanes of a row agree)
          const unsigned k0 = __ballot_sync(0xffffffffu, add0 != -INFINITY && c == 0);
          const unsigned k1 = __ballot_sync(0xffffffffu, add1 != -INFINITY && c == 0);
          unsigned bits = 0;
#pragma unroll
          for (int rr = 0; rr < 8; ++rr) bits |= ((k0 >> (4 * rr)) & 1u) << rr | ((k1 >> (4 * rr)) & 1u) << (8 + rr);
          keep[i] = bits;
          // beyond -2.3e38 the sum would leave fp32 in the log2 domain
          add0 = add0 == -INFINITY ? add0 : fmaxf(add0, -2.3e38f) * 1.4426950408889634f;
          add1 = add1 == -INFINITY ? add1 : fmaxf(add1, -2.3e38f) * 1.4426950408889634f;
        }
        const bool inside = pos[i] + kKv4Tile <= all_end;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          float d[4];
#pragma unroll
          for (int u = 0; u < 4; ++u) d[u] = x[i][nt][u] * 0x1p20f;
          kv4_mma8(d, c & 1 ? pa.w : pa.z, c & 1 ? pb.w : pb.z, qm[nt]);
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            float y = d[u] * cs[nt][u & 1];
            if (MASK) {
              const float add = u & 2 ? add1 : add0;
              y = add == -INFINITY ? -INFINITY : y + add;
            }
            if (!inside && pos[i] + r + (u & 2 ? 8 : 0) >= end[nt][u & 1]) y = -INFINITY;
            x[i][nt][u] = y;
          }
        }
      }

      // ---- largest s of the stage's values (one pair of tokens per lane), running maxima
      {
        const int i = lane >> 3, pr = lane & 7;
        const int pi = i < n ? sm.pos[warp][slot][i] : -1;
        uint32_t big = 0;
        if (pi >= 0) {
          const uint4 s = *reinterpret_cast<const uint4*>(stage + i * kKv4TileBytes + kKv4VParams + pr * 32);
          const uint32_t live = (pi + 2 * pr < len ? 0xffffu : 0u) | (pi + 2 * pr + 1 < len ? 0xffff0000u : 0u);
          const uint32_t w = __vmaxu2(__vmaxu2(s.x, s.y), __vmaxu2(s.z, s.w)) & live;
          big = max(w & 0xffffu, w >> 16);
        }
        big = __reduce_max_sync(0xffffffffu, big);
        const int e_new = big > 0x3c00u ? max(e_run, (int)((big + 0x3ffu) >> 10) - 15) : e_run;
        bool moved = e_new != e_run;
        float f[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            float t = -INFINITY;
#pragma unroll
            for (int i2 = 0; i2 < kKv4StageTiles; ++i2) t = fmaxf(t, fmaxf(x[i2][nt][u], x[i2][nt][u + 2]));
            t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 4));
            t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 8));
            t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 16));
            t = fmaxf(t, m[nt][u]);
            moved |= t != m[nt][u];
            f[nt][u] = m[nt][u] == -INFINITY ? 0.f : kv4_exp2((m[nt][u] - t) + (float)(e_run - e_new));
            m[nt][u] = t;
          }
        e_run = e_new;
        if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int u = 0; u < 4; ++u) {
              z[nt][u] *= f[nt][u & 1];
#pragma unroll
              for (int mt = 0; mt < 8; ++mt) o[mt][nt][u] *= f[nt][u & 1];
            }
            l[nt][0] *= f[nt][0];
            l[nt][1] *= f[nt][1];
          }
        }
      }

      // ---- weights and values
#pragma unroll
      for (int i = 0; i < kKv4StageTiles; ++i) {
        if (pos[i] < 0) continue;
        const uint8_t* tl = stage + i * kKv4TileBytes;
        uint32_t p0[NT], p1[NT];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          float w[4];
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            const float base = m[nt][u & 1] == -INFINITY ? 0.f : m[nt][u & 1] + (float)(e_run - 15);
            w[u] = kv4_exp2(x[i][nt][u] - base);
          }
          l[nt][0] += w[0] + w[2];
          l[nt][1] += w[1] + w[3];
          p0[nt] = kv4_transpose(kv4_half2(w[0], w[1]));
          p1[nt] = kv4_transpose(kv4_half2(w[2], w[3]));
        }
        const uint4 va = *reinterpret_cast<const uint4*>(tl + kKv4VCodes + c * 128 + r * 16);
        const uint4 vb = *reinterpret_cast<const uint4*>(tl + kKv4VCodes + (c + 4) * 128 + r * 16);
        uint4 ta = *reinterpret_cast<const uint4*>(tl + kKv4VParams + c * 32);
        uint4 tb = *reinterpret_cast<const uint4*>(tl + kKv4VParams + (c + 4) * 32);
        uint32_t ma = 0, mb = 0;
        if (r < 4) {
          ma = *reinterpret_cast<const uint32_t*>(tl + kKv4VParams + c * 32 + 16 + r * 4);
          mb = *reinterpret_cast<const uint32_t*>(tl + kKv4VParams + (c + 4) * 32 + 16 + r * 4);
        }
        if (MASK || pos[i] + kKv4Tile > len) {   // tokens that do not count may hold anything
          const int t = pos[i] + 2 * c;
          uint32_t la = (t < len ? 0xffffu : 0u) | (t + 1 < len ? 0xffff0000u : 0u);
          uint32_t lb = (t + 8 < len ? 0xffffu : 0u) | (t + 9 < len ? 0xffff0000u : 0u);
          if (MASK) {
            const unsigned ba = keep[i] >> (2 * c), bb = keep[i] >> (2 * c + 8);
            la &= (ba & 1 ? 0xffffu : 0u) | (ba & 2 ? 0xffff0000u : 0u);
            lb &= (bb & 1 ? 0xffffu : 0u) | (bb & 2 ? 0xffff0000u : 0u);
          }
          ta.x &= la, ta.y &= la, ta.z &= la, ta.w &= la, ma &= la;
          tb.x &= lb, tb.y &= lb, tb.z &= lb, tb.w &= lb, mb &= lb;
        }
        const uint32_t wa[4] = {va.x, va.y, va.z, va.w}, wb[4] = {vb.x, vb.y, vb.z, vb.w};
        const uint32_t sa[4] = {ta.x, ta.y, ta.z, ta.w}, sb[4] = {tb.x, tb.y, tb.z, tb.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t ua = wa[j] >> 8, ub = wb[j] >> 8, eight = r == j ? 0xc800c800u : 0u;
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            const uint32_t b0 = kv4_hmul2(p0[nt], sa[j]), b1 = kv4_hmul2(p1[nt], sb[j]);
            kv4_mma(o[2 * j][nt], wa[j] & 0x000f000fu, wa[j] & 0x00f000f0u, wb[j] & 0x000f000fu, wb[j] & 0x00f000f0u, b0, b1);
            kv4_mma(o[2 * j + 1][nt], ua & 0x000f000fu, ua & 0x00f000f0u, ub & 0x000f000fu, ub & 0x00f000f0u, b0, b1);
            kv4_mma(z[nt], 0u, eight, 0u, eight, b0, b1);
          }
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) kv4_mma(z[nt], ma, 0u, mb, 0u, p0[nt], p1[nt]);
      }
      __syncwarp();                         // the stage is read: its next copies may land
      fetch(slot);

      // ---- end of the segment, or of the stretch
      done += n;
      const bool seg_end = use.t + n == use.tiles;
      if (seg_end || done == g1 - g0) {
        const bool whole = seg_end && seg_start >= g0;
        const int pi = 2 * warp + npieces;
        float* po = sm.o(pi);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            l[nt][u] += __shfl_xor_sync(0xffffffffu, l[nt][u], 4);
            l[nt][u] += __shfl_xor_sync(0xffffffffu, l[nt][u], 8);
            l[nt][u] += __shfl_xor_sync(0xffffffffu, l[nt][u], 16);
          }
          const float z0 = z[nt][0] + z[nt][2], z1 = z[nt][1] + z[nt][3];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float y0 = __shfl_sync(0xffffffffu, z0, j * 4 + c), y1 = __shfl_sync(0xffffffffu, z1, j * 4 + c);
#pragma unroll
            for (int u = 0; u < 2; ++u) {
              const float y = u ? y1 : y0;
              const float4 v = make_float4(fmaf(o[2 * j][nt][u], 0x1p24f, y), fmaf(o[2 * j][nt][u + 2], 0x1p20f, y),
                                           fmaf(o[2 * j + 1][nt][u], 0x1p24f, y), fmaf(o[2 * j + 1][nt][u + 2], 0x1p20f, y));
              const int col = nt * 8 + 2 * c + u, d = j * 32 + 4 * r;
              if (whole)
                kv4_store_out(p, use.b, use.hc, col, kCols, d, v, m[nt][u] + (float)(e_run - 15), l[nt][u]);
              else
                *reinterpret_cast<float4*>(po + col * 128 + d) = v;
            }
          }
          if (!whole && r == 0)
#pragma unroll
            for (int u = 0; u < 2; ++u) {
              sm.meff[pi][nt * 8 + 2 * c + u] = m[nt][u] == -INFINITY ? -INFINITY : m[nt][u] + (float)(e_run - 15);
              sm.l[pi][nt * 8 + 2 * c + u] = l[nt][u];
            }
        }
        if (!whole) {
          if (lane == 0) {
            Kv4Piece& q = sm.piece[pi];
            q.start = seg_start;
            q.b = use.b;
            q.hc = use.hc;
            q.tiles = use.tiles;
            q.used = 1;
          }
          ++npieces;
        }
        seg_start = g0 + done;
        fresh = true;
      }
      use.advance(p, n);
    }
  }
  __syncthreads();

  // ---- merge the pieces of each segment, in line order
  for (int i = 0; i < 2 * kKv4Warps;) {
    if (!sm.piece[i].used) {
      ++i;
      continue;
    }
    const Kv4Piece pc = sm.piece[i];
    int i1 = i + 1;
    for (int k = i + 1; k < 2 * kKv4Warps; ++k) {
      if (!sm.piece[k].used) continue;
      if (sm.piece[k].start != pc.start) break;
      i1 = k + 1;
    }
    const bool whole = pc.start >= c0 && pc.start + pc.tiles <= c1;
    const int slot = pc.start <= c0 ? 0 : 1;
    float* part = p.parts + (blockIdx.x * 2 + slot) * kKv4PartFloats;
    for (int e = tid; e < kCols * 32; e += kKv4Warps * 32) {
      const int col = e >> 5, d = (e & 31) * 4;
      float mx = -INFINITY;
      for (int k = i; k < i1; ++k)
        if (sm.piece[k].used) mx = fmaxf(mx, sm.meff[k][col]);
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
      float sum = 0.f;
      for (int k = i; k < i1; ++k) {
        if (!sm.piece[k].used) continue;
        const float w = kv4_weight(sm.meff[k][col], mx);
        const float4 v = *reinterpret_cast<const float4*>(sm.o(k) + col * 128 + d);
        acc.x = fmaf(w, v.x, acc.x), acc.y = fmaf(w, v.y, acc.y), acc.z = fmaf(w, v.z, acc.z), acc.w = fmaf(w, v.w, acc.w);
        sum = fmaf(w, sm.l[k][col], sum);
      }
      if (whole) {
        kv4_store_out(p, pc.b, pc.hc, col, kCols, d, acc, mx, sum);
      } else {
        __stcg(reinterpret_cast<float4*>(part + col * 128 + d), acc);
        if (d == 0) {
          __stcg(part + kCols * 128 + col, mx);
          __stcg(part + kCols * 129 + col, sum);
        }
      }
    }
    if (!whole) {
      const int first = (int)(pc.start / per), last = (int)((pc.start + pc.tiles - 1) / per), n = last - first + 1;
      __threadfence();
      __syncthreads();
      if (tid == 0) sm.last = atomicAdd(p.counters + first, 1) == n - 1;
      __syncthreads();
      if (sm.last) {
        __threadfence();
        if (tid == 0) p.counters[first] = 0;
        for (int e = tid; e < kCols * 32; e += kKv4Warps * 32) {
          const int col = e >> 5, d = (e & 31) * 4;
          // the segment's piece of CTA k: its first one, but for the CTA in whose middle it starts
          const float* at = p.parts + ((int64_t)first * 2 + (pc.start > first * per ? 1 : 0)) * kKv4PartFloats;
          float mx = -INFINITY, sum = 0.f;
          float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
          for (int k = 0; k < n; ++k) {
            const float* pk = k == 0 ? at : p.parts + (int64_t)(first + k) * 2 * kKv4PartFloats;
            const float4 v = __ldcg(reinterpret_cast<const float4*>(pk + col * 128 + d));
            const float mk = __ldcg(pk + kCols * 128 + col), lk = __ldcg(pk + kCols * 129 + col);
            const float joint = fmaxf(mx, mk);
            const float wa = kv4_weight(mx, joint), wb = kv4_weight(mk, joint);
            acc.x = acc.x * wa + v.x * wb, acc.y = acc.y * wa + v.y * wb;
            acc.z = acc.z * wa + v.z * wb, acc.w = acc.w * wa + v.w * wb;
            sum = sum * wa + lk * wb;
            mx = joint;
          }
          kv4_store_out(p, pc.b, pc.hc, col, kCols, d, acc, mx, sum);
        }
      }
      __syncthreads();
    }
    i = i1;
  }
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
