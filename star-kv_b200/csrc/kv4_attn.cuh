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
//   Scores: tokens are rows, columns are columns.  With c' = c + 8 as stored, per
//     group g of 32 channels d_g = sum c' q, and
//     x = sum_g s_g d_g + sum_g (m_g - 8 s_g) sum q_g,
//     the second sum by one more mma over (m_g, s_g), sum q_g as two fp16 parts.
//   Values: channels are rows, tokens are summed.  The weight w, rounded to fp16, times
//     s_g rounds once more to fp16 (two roundings of at most 2^-11 of a softmax
//     weight), then o += sum (w s_g) c' and at once o += sum (w s_g) (-8) with a constant
//     operand: the running sums stay centred, so that the truncating fp32 additions
//     of the tensor cores do not act on sums 8 s times as large (measured at 32K
//     tokens: relative error 1.5e-3 when the -8 is taken at the end instead).
//     Where one channel of a group is many times the others, s c and m nearly cancel for
//     those and the rounding of w s_g shows: relative error of an fp16 output 2.1e-4 to
//     4.1e-4, against 2.0e-4 of the exact one rounded (bf16: a few percent more than
//     that).  The rest of w s_g as a second operand would cost an estimated eighth more.
//     The centres add sum w m_g, and a row of ones sums the rounded weights: dividing by
//     that sum takes their rounding out of what they have in common (one key that
//     outweighs the rest has no error from it).  The log-sum-exp has the sum in fp32.
//     w is 2^(x - m + 11 - max(e, 0)): m a running maximum that may trail by 2^4, 2^e the
//     least of 2^-14, 2^-7 and 2^0, 2^1 .. that no s_g so far is above; with e < 0 the
//     factors are w (s_g 2^-e).  So no factor passes 2^15, and a weight 2^-20 of the
//     largest still has 8 bits or more where all s are alike, for any s from 2^-21 up.
//
// Work split.  All (sequence, KV head, column block) segments form one line of
// tiles; CTA i of a grid of one CTA per SM takes an equal stretch of it, its warps
// equal parts of that, whatever the lengths are (they are read on the GPU).  A warp
// that holds a whole segment writes its output; other pieces merge in shared memory,
// and what a CTA does not hold whole goes to the workspace, where the CTA that
// arrives last merges it in CTA order (the same result every time).
//
// Measured on a B200 (copy: 6.45 TB/s), device time with the L2 flushed: 16 sequences of 32768
// tokens, 32 KV heads, one query head each (2.7 GB): 510 us, 5.3 TB/s (call after call at the power
// cap 532-561 us); 64 sequences of up to 8192, 8 KV heads of 4, pages of 16: 88 us; one sequence of
// 32769, 8 of 4: 28 us (23 with the L2 warm); 8 sequences of up to 16384, 8 of 4, 4 query tokens,
// masked: 53 us.  Long contexts are bound by issue and dependent latencies: 274 warp instructions a
// tile (80 of them the nibbles' masks and shifts, 26 matrix instructions of 8 cycles), about 140
// cycles a tile and SM where HBM takes 115 for its 2560 bytes.  Short ones by the chain of start
// (lengths, queries, block table, first tile: 5 us) and merge (6 us).
#pragma once
#include "kv4.cuh"

namespace starkv {

constexpr int kKv4PadTiles = 4;             // see kv4_tiles; 64 mixed sequences, when chosen: 115 us with 0, 85 with 2, 82 with 4 or 7
constexpr int kKv4MaxGrid = 160;            // CTAs the workspace has room for
constexpr int kKv4MaxCols = 16;
// One piece of a segment: o (cols, 128), then per column the base, the sum of the weights and the
// sum of the weights as rounded to fp16.
constexpr int kKv4PieceRows = 131;
constexpr int kKv4PartFloats = kKv4MaxCols * kKv4PieceRows;
// Two pieces a warp: up to 15 warps of 8 columns or 11 of 16.
constexpr int kKv4HeadFloats = 2 * 11 * 16 * kKv4PieceRows;
constexpr size_t kKv4CounterBytes = 1024;
static_assert(kKv4MaxGrid * sizeof(int) <= kKv4CounterBytes, "a counter a CTA");
// counters, two pieces a CTA for other CTAs, two a warp
constexpr size_t kKv4WorkspaceBytes =
    kKv4CounterBytes + (size_t)kKv4MaxGrid * (2 * kKv4PartFloats + kKv4HeadFloats) * sizeof(float);

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
  float* heads;                             // (grid, kKv4HeadFloats)
  float scaling;
  int num_selected, q_dtype, out_dtype, batch, queries, q_heads, group, width, col_blocks;
  uint64_t group_m, col_blocks_m;           // kv4_reciprocal of the two
  unsigned long long wait_ns;               // limit of one wait
  int skip_copy;                            // tests: tile of the first warp whose copy is withheld, or -1
};

// n / d for n * d < 2^38, from floor(2^38 / d) + 1 (a division of run-time integers takes some 40
// dependent instructions, and what runs once a segment is made of such chains).
__host__ __device__ constexpr uint64_t kv4_reciprocal(int d) { return ((uint64_t)1 << 38) / (unsigned)d + 1; }
__device__ __forceinline__ int kv4_divide(int n, uint64_t reciprocal) { return (int)(((uint64_t)(unsigned)n * reciprocal) >> 38); }

__device__ __forceinline__ void kv4_mma(float* d, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// The same with a zero start value.
__device__ __forceinline__ void kv4_mma0(float* d, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ uint32_t kv4_transpose(uint32_t a) {
  uint32_t d;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
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

// 0xffff for each of a word's two fp16 numbers that is a NaN.
__device__ __forceinline__ uint32_t kv4_nans(uint32_t a) {
  const __half2 h = *reinterpret_cast<const __half2*>(&a);
  return __hneu2_mask(h, h);
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
// Tiles of one of its segments, with four that hold nothing: about what a warp's change of segment
// costs, so that stretches with many short segments are not longer than others.
__device__ __forceinline__ int kv4_tiles(const Kv4AttnParams& p, int64_t len) {
  if (len <= 0) return 0;
  return (p.pages ? p.num_selected * p.pool.page_tiles : (int)((len + kKv4Tile - 1) >> 4)) + kKv4PadTiles;
}

// An additive mask's value for the log2 domain: times log2 e.  Beyond 1e38 in magnitude, where the
// product would soon leave fp32, the slope is 3/4: numbers stay apart and in order (so far out any
// two weigh as 0 and 1), the type's lowest becomes -3.24e38, infinities and NaN stay.  kv4_lse is the way back.
constexpr float kKv4MaskKnee = 1e38f, kKv4Log2e = 1.4426950408889634f;
__device__ __forceinline__ float kv4_mask_log2(float a) {
  const float t = fminf(fmaxf(a, -kKv4MaskKnee), kKv4MaskKnee);
  return fmaf(a - t, 0.75f, t * kKv4Log2e);
}
__device__ __forceinline__ float kv4_lse(float x) {
  const float t = fminf(fmaxf(x, -kKv4MaskKnee * kKv4Log2e), kKv4MaskKnee * kKv4Log2e);
  const float y = fmaf(x - t, 1.f / 0.75f, t * 0.69314718055994531f);
  return fabsf(y) == INFINITY && fabsf(x) != INFINITY ? copysignf(3.402823466e38f, y) : y;   // a rounding past the end
}

// Writes one column of a segment, a lane 4 channels: o over the rounded weights' sum, log(l) above the base.
__device__ __forceinline__ void kv4_store_column(const Kv4AttnParams& p, int b, int hc, int col, int cols, float4 o, float base,
                                              float l, float rounded) {
  const int lane = threadIdx.x & 31, head = kv4_divide(hc, p.col_blocks_m), gcol = (hc - head * p.col_blocks) * cols + col;
  const int qi = kv4_divide(gcol, p.group_m), qh = head * p.group + gcol - qi * p.group;
  const float inv = l == 0.f ? 0.f : 1.f / rounded;   // a NaN stays one
  o.x *= inv, o.y *= inv, o.z *= inv, o.w *= inv;
  const int64_t at = b * p.os[0] + qi * p.os[1] + qh * p.os[2] + lane * 4;
  if (p.out_dtype == STARKV_F32) {
    *reinterpret_cast<float4*>(reinterpret_cast<float*>(p.out) + at) = o;
  } else if (p.out_dtype == STARKV_F16) {
    *reinterpret_cast<uint2*>(reinterpret_cast<__half*>(p.out) + at) = make_uint2(kv4_half2(o.x, o.y), kv4_half2(o.z, o.w));
  } else {
    __nv_bfloat162 h[2] = {__floats2bfloat162_rn(o.x, o.y), __floats2bfloat162_rn(o.z, o.w)};
    *reinterpret_cast<uint2*>(reinterpret_cast<__nv_bfloat16*>(p.out) + at) = *reinterpret_cast<uint2*>(h);
  }
  if (p.lse && lane == 0)
    p.lse[((int64_t)b * p.queries + qi) * p.q_heads + qh] =
        l == 0.f ? -INFINITY : kv4_lse(base + log2f(l));
}

// Weight of a piece against the joint base.
__device__ __forceinline__ float kv4_weight(float base, float joint) {
  return base == -INFINITY ? 0.f : kv4_exp2(base - joint);
}

// mask[i] to shared memory, 0 where i is past its width (grouped with the thread's other copies).
__device__ __forceinline__ void kv4_cp_async4(void* dst, const float* mask, int i, int64_t width) {
  const int bytes = i < width ? 4 : 0;
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(smem_u32(dst)), "l"(mask + (bytes ? i : 0)), "r"(bytes)
               : "memory");
}

// The largest of a warp's values, by its order-preserving integers.
__device__ __forceinline__ float kv4_warp_max(float x) {
  const int u = __float_as_int(x), k = __reduce_max_sync(0xffffffffu, u ^ ((u >> 31) & 0x7fffffff));
  return __int_as_float(k ^ ((k >> 31) & 0x7fffffff));
}

__device__ __forceinline__ uint4 kv4_lds128(uint32_t at) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at));
  return v;
}
__device__ __forceinline__ uint32_t kv4_lds32(uint32_t at) {
  uint32_t v;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(at));
  return v;
}

// Position on the line of tiles.
struct Kv4Cursor {
  int b, hc, t, tiles, len;                 // sequence, KV head * col_blocks + column block, tile, tiles of the segment, length
  int left;                                 // tiles left of the warp's stretch
  // The tiles of the segment from t on that belong to the stretch.
  __device__ __forceinline__ int here() const { return min(tiles - t, left); }
  // Moves on by n <= here() tiles, into the next segment where this one ends.
  __device__ __forceinline__ void advance(const Kv4AttnParams& p, int n) {
    t += n;
    left -= n;
    if (t < tiles || left <= 0) return;
    t = 0;
    if (++hc < p.pool.heads * p.col_blocks) return;
    hc = 0;
    tiles = 0;
    while (tiles == 0 && b + 1 < p.batch) {
      len = (int)kv4_length(p, ++b);
      tiles = kv4_tiles(p, len);
    }
    if (tiles == 0) left = 0;               // lengths that changed under the kernel
  }
};

constexpr int kKv4QueryVecs = 5 * 32;       // vectors of the prepared queries of 8 columns

struct Kv4Piece {
  int start, b, hc, tiles;                  // first tile of its segment on the line (-1: unused)
};

template <int NT, int W, bool MASK>
struct Kv4AttnSmem {
  static constexpr int kCols = NT * 8;
  static constexpr int kRing = W > 11 ? 4 : 5;   // tile slots of a warp
  alignas(128) uint8_t ring[W][kRing][kKv4TileBytes];
  static constexpr int kShared = 4;         // segments whose queries are prepared once for the CTA
  alignas(16) uint4 shared[kShared][NT * kKv4QueryVecs];
  alignas(16) uint4 queries[W][NT * kKv4QueryVecs];   // a warp's own, for segments beyond those
  alignas(16) float mask[MASK ? W : 1][MASK ? kRing : 1][kKv4Tile];
  alignas(8) uint64_t full[W][kRing], empty[W][kRing];
  int pos[W][kRing];                        // position of a tile's first token, -1: nothing to attend to
  Kv4Piece piece[2 * W];
  int shared_start[kShared];                // first tiles of the shared segments
  int scan[W + 1];
  int upto[(W + 1) * 32];                   // tiles of the sequences up to and with a thread's
  int last[2];
  int empties;                              // there are sequences of no tokens
  int stop, done;                           // a wait ran out; no more copies will be started
  int issued[32];                           // tiles that a lane of the copying warp started, once it is done
};

__device__ __forceinline__ uint2 kv4_lds64(uint32_t at) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(at));
  return v;
}

// A lane's byte offsets within a tile, kept in registers (opaque to the compiler, which would
// otherwise compute them anew for every load).
struct Kv4Lane {
  uint32_t code, kpar, kown, vpar, vmid, row, pair;
  __device__ __forceinline__ explicit Kv4Lane(int lane) {
    const int r = lane >> 2, c = lane & 3;
    code = lane * 16;
    kpar = kKv4KParams + r * 32;
    kown = kKv4KParams + r * 32 + (c & 1) * 16;
    vpar = kKv4VParams + c * 32;
    vmid = kKv4VParams + c * 32 + 16 + (r & 1) * 8;
    row = r * 4;                            // of the mask: the lane's rows, and its pairs of tokens
    pair = c * 8;
    asm volatile("" : "+r"(code), "+r"(kpar), "+r"(kown), "+r"(vpar), "+r"(vmid));
  }
};

// A flag in shared memory from one warp to the others, with what its lane wrote before.
__device__ __forceinline__ void kv4_raise(int* flag) {
  __threadfence_block();
  *(volatile int*)flag = 1;
}
__device__ __forceinline__ bool kv4_raised(const int* flag) {
  const bool up = *(const volatile int*)flag != 0;
  __threadfence_block();
  return up;
}

// Waits for a tile, the same answer for the whole warp: false when limit_ns pass first or `stop` is raised.
// (The vote costs 1-2 % of a long call; what comes after a wait has to be one path for all lanes.)
__device__ __forceinline__ bool kv4_wait_tile(uint64_t* bar, uint32_t parity, unsigned long long limit_ns, const int* stop) {
  bool there = mbar_try_wait_plain(bar, parity);
  if (!there) {
    const unsigned long long t0 = global_timer_ns();
#pragma unroll 1
    while (!(there = mbar_try_wait_plain(bar, parity)))
      if (kv4_raised(stop) || global_timer_ns() - t0 > limit_ns) break;
  }
  return __all_sync(0xffffffffu, there);
}

// The columns of one segment in a warp's registers.
template <int NT>
struct Kv4Columns {
  uint32_t qb[1][4][4];                     // B operands of the scores, 16 q or q by nibble (NT > 1: in shared memory)
  uint32_t qc[NT][2];                       // sums of q for s and m
  float cs[NT][2];                          // a column's scores, as computed (an eighth), to the log2 domain
  int end[NT][2];                           // first position a column does not attend to
  float o[8][NT][4], l[NT][2];
  float z[NT][4];                           // sum w m: group j in rows j / 2 and j / 2 + 8; sum w in row 2
  float base[NT][2], thr[NT][2];            // w = 2^(x - base); x beyond thr moves the base
  int e;                                    // no s so far is above 2^e: -14, -7 or >= 0; o is in units of 2^min(e, 0)
};

// The queries of 8 columns of a segment as the scores' operands: five vectors a lane in `buf` (32
// vectors apart), the four groups' B operands and { sums of q for s, for m, scale, - }.
__device__ __forceinline__ void kv4_prepare(const Kv4AttnParams& p, uint4* buf, int b, int hc, int nt, int cols, int lane) {
  const int r = lane >> 2, c = lane & 3, head = kv4_divide(hc, p.col_blocks_m);
  const int gcol = (hc - head * p.col_blocks) * cols + nt * 8 + r, qi = kv4_divide(gcol, p.group_m);
  const bool f16 = p.q_dtype == STARKV_F16;
  const int64_t at = b * p.qs[0] + qi * p.qs[1] + (head * p.group + gcol - qi * p.group) * p.qs[2] + c * 8;
  const uint4* src = reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(p.q) + at);
  uint32_t raw[16];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint4 w = gcol < p.group * p.queries ? __ldg(src + j * 4) : make_uint4(0, 0, 0, 0);
    raw[4 * j] = w.x, raw[4 * j + 1] = w.y, raw[4 * j + 2] = w.z, raw[4 * j + 3] = w.w;
  }
  uint32_t big = 0;                         // the largest magnitude's bits (they order like integers)
#pragma unroll
  for (int i = 0; i < 16; i += 2) big = __vimax3_u16x2(big, raw[i] & 0x7fff7fffu, raw[i + 1] & 0x7fff7fffu);
  big = max(big & 0xffffu, big >> 16);
  big = max(big, __shfl_xor_sync(0xffffffffu, big, 1));
  big = max(big, __shfl_xor_sync(0xffffffffu, big, 2));
  const float a = f16 ? kv4_halves(big).x : __uint_as_float(big << 16);
  // q scaled by a power of two to [512, 1024) in magnitude, the scaling's sign with it; a column
  // whose scores vanish (q below 2^-117, or q times scaling below 2^-110: `up` or `scale` would leave
  // fp32) becomes zero; one with a NaN for a scaling becomes NaN
  float up = 0.f, scale = 1.f;
  const float size = fabsf(p.scaling);
  if (size != size) {
    up = size;
  } else if (!(a < 0x1p-117f) && !(a * size < 0x1p-110f)) {
    const int ex = (__float_as_int(a) >> 23) - 127;
    up = __int_as_float((127 + 9 - ex) << 23);
    scale = size * kKv4Log2e * __int_as_float((127 - 9 + 3 + ex) << 23);
    if (p.scaling < 0.f) up = -up;
  }
  float sum[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    float f[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t w = raw[4 * j + i];
      const float2 h = kv4_halves(w);
      f[2 * i] = (f16 ? h.x : __uint_as_float(w << 16)) * up;
      f[2 * i + 1] = (f16 ? h.y : __uint_as_float(w & 0xffff0000u)) * up;
    }
    buf[j * 32 + lane] = make_uint4(kv4_half2(f[0] * 16.f, f[4] * 16.f), kv4_half2(f[1], f[5]),
                                    kv4_half2(f[2] * 16.f, f[6] * 16.f), kv4_half2(f[3], f[7]));
    sum[j] = ((f[0] + f[1]) + (f[2] + f[3])) + ((f[4] + f[5]) + (f[6] + f[7]));
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) sum[j] += __shfl_xor_sync(0xffffffffu, sum[j], 1);
#pragma unroll
  for (int j = 0; j < 4; ++j) sum[j] += __shfl_xor_sync(0xffffffffu, sum[j], 2);
  // lanes c = 0, 1: the upper parts of sums 0, 1 and 2, 3; c = 2, 3: what is left of them.
  // An eighth of the sums (exact) for m, so that -8 times it, for s, fits fp16 too.
  const float s0 = c & 1 ? sum[2] : sum[0], s1 = c & 1 ? sum[3] : sum[1];
  const float h0 = __half2float(__float2half_rn(s0)), h1 = __half2float(__float2half_rn(s1));
  const float t0 = c & 2 ? s0 - h0 : h0, t1 = c & 2 ? s1 - h1 : h1;
  buf[128 + lane] = make_uint4(kv4_half2(-t0, -t1), kv4_half2(0.125f * t0, 0.125f * t1), __float_as_uint(scale), 0);
}

// Takes a segment's prepared queries and clears its sums.
template <int NT>
__device__ __forceinline__ void kv4_begin(const Kv4AttnParams& p, Kv4Columns<NT>& s, const uint4* buf, int hc, int len, int lane) {
  const int first = (hc - kv4_divide(hc, p.col_blocks_m) * p.col_blocks) * (NT * 8), c = lane & 3;
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    if (NT == 1) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint4 v = buf[j * 32 + lane];
        s.qb[0][j][0] = v.x, s.qb[0][j][1] = v.y, s.qb[0][j][2] = v.z, s.qb[0][j][3] = v.w;
      }
    }
    const uint4 v = buf[nt * kKv4QueryVecs + 128 + lane];
    s.qc[nt][0] = v.x;
    s.qc[nt][1] = v.y;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      s.cs[nt][u] = __uint_as_float(__shfl_sync(0xffffffffu, v.z, (2 * c + u) * 4));
      s.end[nt][u] = len - p.queries + 1 + kv4_divide(first + nt * 8 + 2 * c + u, p.group_m);
      s.l[nt][u] = 0.f;
      s.base[nt][u] = 0.f;
      s.thr[nt][u] = -INFINITY;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      s.z[nt][i] = 0.f;
#pragma unroll
      for (int mt = 0; mt < 8; ++mt) s.o[mt][nt][i] = 0.f;
    }
  }
  s.e = -14;
}

// One tile at shared address tl.  MASK: its additive mask at shared address mk.  EDGE: some of its
// positions are beyond what a column attends to, or beyond the length.
template <int NT, bool MASK, bool EDGE>
__device__ __forceinline__ void kv4_tile(Kv4Columns<NT>& s, const uint4* queries, uint32_t tl, int pos, int len, uint32_t mk,
                                         const Kv4Lane& at, int lane) {
  float x[NT][4];
  // ---- scores
  const uint4 ka = kv4_lds128(tl + at.code), kb = kv4_lds128(tl + at.code + 512);
  // rows r and r + 8 of s, then of m: groups 0 and 1, groups 2 and 3, and those the lane's columns of A take
  const uint4 pa = kv4_lds128(tl + at.kpar), pb = kv4_lds128(tl + at.kpar + 16), own = kv4_lds128(tl + at.kown);
  uint4 ta = kv4_lds128(tl + at.vpar), tb = kv4_lds128(tl + at.vpar + 128);
  {
    const uint32_t wa[4] = {ka.x, ka.y, ka.z, ka.w}, wb[4] = {kb.x, kb.y, kb.z, kb.w};
    const float2 sa01 = kv4_halves(pa.x), sb01 = kv4_halves(pa.y), sa23 = kv4_halves(pb.x), sb23 = kv4_halves(pb.y);
    const float sa[4] = {sa01.x, sa01.y, sa23.x, sa23.y}, sb[4] = {sb01.x, sb01.y, sb23.x, sb23.y};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t ua = wa[j] >> 8, ub = wb[j] >> 8;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const uint4 q = NT == 1 ? make_uint4(s.qb[0][j][0], s.qb[0][j][1], s.qb[0][j][2], s.qb[0][j][3])
                                : queries[nt * kKv4QueryVecs + j * 32 + lane];
        float d[4];
        kv4_mma0(d, wa[j] & 0x000f000fu, wb[j] & 0x000f000fu, wa[j] & 0x00f000f0u, wb[j] & 0x00f000f0u, q.x, q.y);
        kv4_mma(d, ua & 0x000f000fu, ub & 0x000f000fu, ua & 0x00f000f0u, ub & 0x00f000f0u, q.z, q.w);
        x[nt][0] = j ? fmaf(sa[j], d[0], x[nt][0]) : sa[j] * d[0];
        x[nt][1] = j ? fmaf(sa[j], d[1], x[nt][1]) : sa[j] * d[1];
        x[nt][2] = j ? fmaf(sb[j], d[2], x[nt][2]) : sb[j] * d[2];
        x[nt][3] = j ? fmaf(sb[j], d[3], x[nt][3]) : sb[j] * d[3];
      }
    }
  }
  float add0 = 0.f, add1 = 0.f;
  if (MASK) {
    add0 = __uint_as_float(kv4_lds32(mk + at.row));
    add1 = __uint_as_float(kv4_lds32(mk + at.row + 32));
    add0 = kv4_mask_log2(add0);
    add1 = kv4_mask_log2(add1);
  }
  bool over = false;
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    float d[4];
    kv4_mma0(d, own.x, own.y, own.z, own.w, s.qc[nt][0], s.qc[nt][1]);
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      float y = fmaf(x[nt][u], 0x1p17f, d[u]);    // an eighth of the column's score
      if (MASK) {
        const float add = u & 2 ? add1 : add0;
        y = add == -INFINITY ? -INFINITY : fmaf(y, s.cs[nt][u & 1], add);
      }
      if (EDGE && pos + (lane >> 2) + (u & 2 ? 8 : 0) >= s.end[nt][u & 1]) y = -INFINITY;
      x[nt][u] = y;
    }
    over |= fmaxf(x[nt][0], x[nt][2]) > s.thr[nt][0];
    over |= fmaxf(x[nt][1], x[nt][3]) > s.thr[nt][1];
  }
  uint32_t la = 0xffffffffu, lb = 0xffffffffu;
  if (MASK || EDGE) {                       // tokens that do not count may hold anything
    if (EDGE) {
      const int t = pos + 2 * (lane & 3);
      la = (t < len ? 0xffffu : 0u) | (t + 1 < len ? 0xffff0000u : 0u);
      lb = (t + 8 < len ? 0xffffu : 0u) | (t + 9 < len ? 0xffff0000u : 0u);
    }
    if (MASK) {                             // 0xff800000: -inf
      const uint2 m0 = kv4_lds64(mk + at.pair), m1 = kv4_lds64(mk + at.pair + 32);
      la &= (m0.x != 0xff800000u ? 0xffffu : 0u) | (m0.y != 0xff800000u ? 0xffff0000u : 0u);
      lb &= (m1.x != 0xff800000u ? 0xffffu : 0u) | (m1.y != 0xff800000u ? 0xffff0000u : 0u);
    }
    ta.x &= la, ta.y &= la, ta.z &= la, ta.w &= la;
    tb.x &= lb, tb.y &= lb, tb.z &= lb, tb.w &= lb;
  }
  // an s above 2^e (the bits of positive fp16 numbers order like integers)
  const uint32_t lim = (uint32_t)(15 + s.e) * 0x04000400u;
  const uint32_t big = __vimax3_u16x2(__vimax3_u16x2(ta.x, ta.y, ta.z), __vimax3_u16x2(ta.w, tb.x, tb.y),
                                      __vimax3_u16x2(tb.z, tb.w, lim));
  over |= big != lim;
  // With 16 columns the value codes come in before the vote (53 -> 50 us for 4 drafts; there are fewer
  // warps to hide the loads), with 8 after it (their registers are needed for it: 2 % slower before).
  uint4 va, vb;
  uint2 ma, mb;
  auto load_values = [&]() {
    va = kv4_lds128(tl + at.code + kKv4VCodes), vb = kv4_lds128(tl + at.code + kKv4VCodes + 512);
    ma = kv4_lds64(tl + at.vmid), mb = kv4_lds64(tl + at.vmid + 128);
  };
  if (NT > 1) load_values();
  // ---- a score or an s that the base does not cover
  if (__any_sync(0xffffffffu, over)) {
    const uint32_t top = __reduce_max_sync(0xffffffffu, max(big & 0xffffu, big >> 16));
    int e_new = (int)((top + 0x3ffu) >> 10) - 15;
    if (e_new < 0) e_new = e_new <= -14 ? -14 : e_new <= -7 ? -7 : 0;
    const float unit_o = __int_as_float((127 + min(s.e, 0) - min(e_new, 0)) << 23);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        float t = fmaxf(x[nt][u], x[nt][u + 2]);
        t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 4));
        t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 8));
        t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 16));
        const float unit = MASK ? 1.f : s.cs[nt][u];
        t *= unit;
        const bool before = s.thr[nt][u] != -INFINITY;
        const float m = before ? fmaxf(t, s.base[nt][u] + (float)(11 - max(s.e, 0))) : t;
        if (m == -INFINITY) continue;
        const float moved = m + (float)(max(e_new, 0) - 11);
        const float f = before ? kv4_exp2(s.base[nt][u] - moved) : 0.f;
        s.base[nt][u] = moved;
        s.thr[nt][u] = (m + 4.f) / unit;
        s.l[nt][u] *= f;
        s.z[nt][u] *= f;
        s.z[nt][u + 2] *= f;
#pragma unroll
        for (int mt = 0; mt < 8; ++mt) s.o[mt][nt][u] *= f * unit_o, s.o[mt][nt][u + 2] *= f * unit_o;
      }
    s.e = e_new;
  }
  if (s.e < 0) {                            // values far below one
    const uint32_t up = (uint32_t)(15 - s.e) * 0x04000400u;
    ta.x = kv4_hmul2(ta.x, up), ta.y = kv4_hmul2(ta.y, up), ta.z = kv4_hmul2(ta.z, up), ta.w = kv4_hmul2(ta.w, up);
    tb.x = kv4_hmul2(tb.x, up), tb.y = kv4_hmul2(tb.y, up), tb.z = kv4_hmul2(tb.z, up), tb.w = kv4_hmul2(tb.w, up);
  }
  // ---- weights and values
  if (NT == 1) load_values();
  if (MASK || EDGE) ma.x &= la, ma.y &= la, mb.x &= lb, mb.y &= lb;
  if (EDGE) {
    // A group that holds a NaN has one for m.  Here not every column attends to its token, and 0 times
    // it must not reach those that do not: the centres go on without it, and one more product says
    // which columns' sums it belongs to.
    const uint32_t na = kv4_nans(ma.x), nb = kv4_nans(ma.y), nc = kv4_nans(mb.x), nd = kv4_nans(mb.y);
    if (__any_sync(0xffffffffu, na | nb | nc | nd)) {
      ma.x &= ~na, ma.y &= ~nb, mb.x &= ~nc, mb.y &= ~nd;
      const uint32_t one = lane >> 2 == 2 ? 0u : 0x3c003c00u;   // row 2 is the weights' sum
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        auto seen = [&](int u) { return x[nt][u] == -INFINITY ? 0.f : 1.f; };
        float d[4];
        kv4_mma0(d, na & one, nb & 0x3c003c00u, nc & one, nd & 0x3c003c00u, kv4_transpose(kv4_half2(seen(0), seen(1))),
                 kv4_transpose(kv4_half2(seen(2), seen(3))));
#pragma unroll
        for (int u = 0; u < 4; ++u)
          if (d[u] > 0.f) s.z[nt][u] = __int_as_float(0x7fffffff);
      }
    }
  }
  if (lane >> 2 == 2) ma.x = mb.x = 0x3c003c00u;   // row 2: ones
  uint32_t p0[NT], p1[NT];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    float w[4];
#pragma unroll
    for (int u = 0; u < 4; ++u)
      w[u] = kv4_exp2(MASK ? x[nt][u] - s.base[nt][u & 1] : fmaf(x[nt][u], s.cs[nt][u & 1], -s.base[nt][u & 1]));
    s.l[nt][0] += w[0] + w[2];
    s.l[nt][1] += w[1] + w[3];
    p0[nt] = kv4_transpose(kv4_half2(w[0], w[1]));
    p1[nt] = kv4_transpose(kv4_half2(w[2], w[3]));
  }
  const uint32_t wa[4] = {va.x, va.y, va.z, va.w}, wb[4] = {vb.x, vb.y, vb.z, vb.w};
  const uint32_t sa[4] = {ta.x, ta.y, ta.z, ta.w}, sb[4] = {tb.x, tb.y, tb.z, tb.w};
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint32_t ua = wa[j] >> 8, ub = wb[j] >> 8;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const uint32_t b0 = kv4_hmul2(p0[nt], sa[j]), b1 = kv4_hmul2(p1[nt], sb[j]);
      kv4_mma(s.o[2 * j][nt], wa[j] & 0x000f000fu, wa[j] & 0x00f000f0u, wb[j] & 0x000f000fu, wb[j] & 0x00f000f0u, b0, b1);
      kv4_mma(s.o[2 * j + 1][nt], ua & 0x000f000fu, ua & 0x00f000f0u, ub & 0x000f000fu, ub & 0x00f000f0u, b0, b1);
      // -8 * 2^-24 in rows r, -8 * 2^-20 in rows r + 8
      kv4_mma(s.o[2 * j][nt], 0x80088008u, 0x80808080u, 0x80088008u, 0x80808080u, b0, b1);
      kv4_mma(s.o[2 * j + 1][nt], 0x80088008u, 0x80808080u, 0x80088008u, 0x80808080u, b0, b1);
    }
  }
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) kv4_mma(s.z[nt], ma.x, ma.y, mb.x, mb.y, p0[nt], p1[nt]);
}

// NT: n-tiles of 8 columns.  W: warps that compute; one more starts the copies, its lanes 2 w
// and 2 w + 1 taking turns at the tiles of warp w.  Up to 8 columns 15 warps of 128 registers
// (about 4 a scheduler: enough to hide the latencies of a tile's dependent steps; 8
// warps that took 4 tiles a step ran at 37 % of the issue slots, 2.5 TB/s); 16 columns need
// twice the accumulators and take 11 warps of 168, with the queries' operands in shared memory.
template <int NT, int W, bool MASK>
__global__ void __launch_bounds__((W + 1) * 32, 1) kv4_attn_kernel(const Kv4AttnParams p) {
  extern __shared__ __align__(128) uint8_t smem_raw[];
  using Smem = Kv4AttnSmem<NT, W, MASK>;
  constexpr int kCols = Smem::kCols, kRing = Smem::kRing;
  Smem& sm = *reinterpret_cast<Smem*>(smem_raw);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int HC = p.pool.heads * p.col_blocks;
  // piece i of the CTA (see kKv4PieceRows): 2 w is the last of warp w and lies over its ring, 2 w + 1 is
  // the end of a segment that an earlier warp began and lies in the workspace
  constexpr int kPiece = kCols * kKv4PieceRows;
  static_assert(2 * W * kPiece <= kKv4HeadFloats && kPiece <= kKv4PartFloats, "room in the workspace");
  static_assert(kPiece * sizeof(float) <= sizeof(sm.ring[0]), "room over the ring");
  float* const heads = p.heads + (int64_t)blockIdx.x * kKv4HeadFloats;
  auto piece_at = [&](int i) {
    return i & 1 ? heads + (i >> 1) * kPiece : reinterpret_cast<float*>(sm.ring[i >> 1][0]);
  };

  // ---- the line of tiles: total, this CTA's stretch, the warps' first sequences
  constexpr int kThreads = (W + 1) * 32;
  const int per_thread = (p.batch + kThreads - 1) / kThreads;
  const int b_lo = tid * per_thread, b_hi = min(b_lo + per_thread, p.batch);
  int mine = 0;
  bool empty = false;                       // a sequence of no tokens
  for (int b = b_lo; b < b_hi; ++b) {
    const int t = kv4_tiles(p, kv4_length(p, b));
    mine += t * HC;
    empty |= t == 0;
  }
  int upto = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += y;
  }
  if (lane == 31) sm.scan[warp] = upto;
  if (warp < W) {
    if (lane < kRing) mbar_init(&sm.full[warp][lane], MASK ? 2 : 1), mbar_init(&sm.empty[warp][lane], 1);
    if (lane < 2) sm.piece[2 * warp + lane].start = -1;
  }
  if (tid < Smem::kShared) sm.shared_start[tid] = -1;
  fence_mbar_init();
  const int empties = __syncthreads_or(empty);
  if (tid == 0) sm.empties = empties, sm.stop = sm.done = 0;   // kept there: it would take a register all along
  int warps = lane <= W ? sm.scan[lane] : 0;  // tiles up to and with a warp's
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, warps, o);
    if (lane >= o) warps += y;
  }
  const int total = __shfl_sync(0xffffffffu, warps, W);
  if (warp > 0) upto += __shfl_sync(0xffffffffu, warps, warp - 1);
  sm.upto[tid] = upto;
  // equal stretches, a tile a warp at least
  const int per = max((int)((unsigned)(total + gridDim.x - 1) / gridDim.x), W);
  const int c0 = (int)min((int64_t)blockIdx.x * per, (int64_t)total), c1 = min(c0 + per, total), width = c1 - c0;
  __syncthreads();

  // the cursor at tile g of the line
  auto seek = [&](int g, int left) {
    Kv4Cursor k;
    int lo = 0;                             // the first thread whose sequences reach beyond g
    if (warp < W) {                         // one g for the warp
      const unsigned beyond = __ballot_sync(0xffffffffu, lane <= W && warps > g);
      lo = beyond ? (__ffs(beyond) - 1) * 32 : 0;
      const unsigned in = __ballot_sync(0xffffffffu, sm.upto[lo + lane] > g);
      lo += in ? __ffs(in) - 1 : 0;
    } else {
      int hi = kThreads - 1;
      while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (sm.upto[mid] > g) hi = mid;
        else lo = mid + 1;
      }
    }
    unsigned off = g - (lo ? sm.upto[lo - 1] : 0);
    k.b = min(lo * per_thread, p.batch - 1);
    k.len = (int)kv4_length(p, k.b);
    k.tiles = kv4_tiles(p, k.len);
    while (off >= (unsigned)(k.tiles * HC) && k.b + 1 < p.batch) {
      off -= k.tiles * HC;
      k.len = (int)kv4_length(p, ++k.b);
      k.tiles = kv4_tiles(p, k.len);
    }
    k.hc = k.tiles ? (int)(off / (unsigned)k.tiles) : 0;
    k.t = (int)(off - (unsigned)(k.hc * k.tiles));
    k.left = k.tiles ? left : 0;
    return k;
  };
  // a warp's stretch; the last warp's lanes have the stretches of the warps they serve
  const int who = min(warp < W ? warp : lane >> 1, W - 1);
  const int g0 = c0 + width / W * who + width % W * who / W;
  const int stretch = c0 + width / W * (who + 1) + width % W * (who + 1) / W - g0;
  if (warp < W) {
    // the queries of the CTA's first segments, a warp 8 columns of one
    if (warp < Smem::kShared * NT && width > 0) {
      Kv4Cursor k = seek(c0, width);
      int start = c0 - k.t;
      for (int i = 0; i < warp / NT && k.left > 0; ++i) {
        start += k.tiles;
        k.advance(p, k.here());
      }
      if (k.left > 0) {
        kv4_prepare(p, sm.shared[warp / NT] + warp % NT * kKv4QueryVecs, k.b, k.hc, warp % NT, kCols, lane);
        if (lane == 0 && warp % NT == 0) sm.shared_start[warp / NT] = start;
      }
    }
    named_bar_sync(1, W * 32);
  }
  Kv4Cursor use{};
  if (stretch > 0 && (warp < W || lane < 2 * W)) use = seek(g0, stretch);
  int seg_start = g0 - use.t;               // first tile of the segment at hand
  if (warp == W) {
    // ---- copies.  The page of a lane's next tile is looked up a turn ahead, so that the block
    // table's latency is not waited for.
    static_assert(2 * W <= 32, "two lanes a warp");
    int slot = lane & 1, parity = 1, at = 0, page = 0, tile = 0, head = 0, seq = 0;
    bool more = false, there = false;       // a tile to issue; it has tokens
    auto look = [&]() {
      more = use.left > 0;
      there = false;
      if (!more) return;
      head = kv4_divide(use.hc, p.col_blocks_m);
      seq = use.b;
      tile = use.t & (p.pool.page_tiles - 1);
      int ord = use.t >> (p.pool.page_shift - 4);
      if (p.pages) ord = ord < p.num_selected ? __ldg(p.pages + ((int64_t)use.b * p.pool.heads + head) * p.num_selected + ord) : -1;
      const int64_t pos = ((int64_t)ord << p.pool.page_shift) + tile * kKv4Tile;
      if (ord >= 0 && pos < use.len) {      // a selected page may lie past the length, or end before it
        at = (int)pos;
        page = __ldg(p.table + use.b * p.table_stride + ord);
        there = true;
      }
      use.advance(p, 1);
      if (use.left > 0) use.advance(p, 1);  // the other lane's
    };
    if ((lane & 1) && use.left > 0) use.advance(p, 1);
    look();
    unsigned long long idle_since = 0;
    int issued = 0;
    while (__any_sync(0xffffffffu, more)) {
      const bool go = more && mbar_test_wait(&sm.empty[who][slot], parity);
      if (!__any_sync(0xffffffffu, go)) {
        const unsigned long long now = global_timer_ns();
        if (idle_since == 0) idle_since = now;
        const bool late = __any_sync(0xffffffffu, now - idle_since > p.wait_ns);
        if (late && lane == 0) {
          record_error(p.pool.err, kDevWaitCopy);
          kv4_raise(&sm.stop);
        }
        if (late || __any_sync(0xffffffffu, kv4_raised(&sm.stop))) break;
        __nanosleep(40);
        continue;
      }
      idle_since = 0;
      if (go) {
        if (there && (unsigned)page >= (unsigned)p.pool.num_pages) {
          record_error(p.pool.err, kDevBadPage);
          there = false;
        }
        sm.pos[who][slot] = there ? at : -1;
        uint64_t* bar = &sm.full[who][slot];
        if (there) {
          mbar_arrive_expect_tx(bar, kKv4TileBytes);
          if (blockIdx.x || who || 2 * issued + (lane & 1) != p.skip_copy)
            bulk_g2s(sm.ring[who][slot], p.pool.tile(page, head, tile), kKv4TileBytes, bar);
        } else {
          mbar_arrive(bar);
        }
        if (MASK) {
          if (there) {
            const float* row = p.mask + seq * p.mask_stride;
            if (at + kKv4Tile <= p.mask_width && (reinterpret_cast<uintptr_t>(row + at) & 15) == 0) {
#pragma unroll
              for (int i = 0; i < 4; ++i) cp_async16(&sm.mask[who][slot][4 * i], row + at + 4 * i);
            } else {
#pragma unroll 1
              for (int i = 0; i < kKv4Tile; ++i) kv4_cp_async4(&sm.mask[who][slot][i], row, at + i, p.mask_width);
            }
            cp_async_arrive(bar);
          } else {
            mbar_arrive(bar);
          }
        }
        ++issued;
        slot += 2;
        if (slot >= kRing) slot -= kRing, parity ^= 1;
        look();
      }
    }
    sm.issued[lane] = issued;
    __syncwarp();
    if (lane == 0) kv4_raise(&sm.done);
  } else if (use.left > 0) {
    const Kv4Lane offsets(lane);
    Kv4Columns<NT> s;
    int slot = 0, parity = 0;
    bool failed = false;
    while (use.left > 0) {
      const int n = use.here();
      const uint4* queries = nullptr;
#pragma unroll
      for (int i = 0; i < Smem::kShared; ++i)
        if (sm.shared_start[i] == seg_start) queries = sm.shared[i];
      if (!queries) {
        __syncwarp();                       // the segment before is done with them
        for (int nt = 0; nt < NT; ++nt)
          kv4_prepare(p, sm.queries[warp] + nt * kKv4QueryVecs, use.b, use.hc, nt, kCols, lane);
        __syncwarp();
        queries = sm.queries[warp];
      }
      kv4_begin<NT>(p, s, queries, use.hc, use.len, lane);
#pragma unroll 1
      for (int i = 0; i < n && !failed; ++i) {
        if (!kv4_wait_tile(&sm.full[warp][slot], parity, p.wait_ns, &sm.stop)) {
          // A wait ran out: reported, and no result of this call counts.  No slot is given back, the copying
          // warp stops, and this one waits for its own copies in flight before its pieces go over the
          // ring; they are merged and counted as ever, so that the workspace is left clear.
          failed = true;
          if (lane == 0) {
            record_error(p.pool.err, kDevWaitCopy);
            kv4_raise(&sm.stop);
          }
          const unsigned long long since = global_timer_ns();
          while (!kv4_raised(&sm.done) && global_timer_ns() - since < p.wait_ns) __nanosleep(200);
          __syncwarp();
          for (int j = stretch - use.left + i, k = 0; k < kRing; ++j, ++k) {
            if ((j >> 1) < *(volatile int*)&sm.issued[2 * warp + (j & 1)])
              mbar_wait(&sm.full[warp][slot], parity, p.wait_ns);
            if (++slot == kRing) slot = 0, parity ^= 1;
          }
          __syncwarp();
          break;
        }
        const int pos = sm.pos[warp][slot];
        if (pos >= 0) {
          const uint32_t tl = smem_u32(sm.ring[warp][slot]), mk = MASK ? smem_u32(sm.mask[warp][slot]) : 0;
          if (pos + kKv4Tile > use.len - p.queries + 1)
            kv4_tile<NT, MASK, true>(s, queries, tl, pos, use.len, mk, offsets, lane);
          else
            kv4_tile<NT, MASK, false>(s, queries, tl, pos, use.len, mk, offsets, lane);
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm.empty[warp][slot]);   // the slot is read: its next copy may land
        if (++slot == kRing) slot = 0, parity ^= 1;
      }

      // ---- end of the segment, or of the stretch
      const int r = lane >> 2, c = lane & 3;
      const int real = min(kCols, p.group * p.queries - (use.hc - kv4_divide(use.hc, p.col_blocks_m) * p.col_blocks) * kCols);
      // a whole segment that is not the stretch's last goes through a place of its own: the ring is
      // in use, and the piece before it waits for the merge
      const bool whole = n == use.tiles;
      const int pi = 2 * warp + (use.left > n);
      float* part = whole && use.left > n ? heads + (W + warp) * kPiece : piece_at(pi);
      const float u24 = __int_as_float((127 + 24 + min(s.e, 0)) << 23), u20 = u24 * 0x1p-4f;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const int col = nt * 8 + 2 * c + u;
          float l = s.l[nt][u];
          l += __shfl_xor_sync(0xffffffffu, l, 4);
          l += __shfl_xor_sync(0xffffffffu, l, 8);
          l += __shfl_xor_sync(0xffffffffu, l, 16);
          if (r == 0) {
            part[kCols * 128 + col] = s.thr[nt][u] == -INFINITY ? -INFINITY : s.base[nt][u];
            part[kCols * 129 + col] = l;
          }
          if (r == 2) part[kCols * 130 + col] = s.z[nt][u];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float y = __shfl_sync(0xffffffffu, s.z[nt][u + 2 * (j & 1)], (j >> 1) * 4 + c);
            if (col < real)
              *reinterpret_cast<float4*>(part + col * 128 + j * 32 + 4 * r) =
                  make_float4(fmaf(s.o[2 * j][nt][u], u24, y), fmaf(s.o[2 * j][nt][u + 2], u20, y),
                              fmaf(s.o[2 * j + 1][nt][u], u24, y), fmaf(s.o[2 * j + 1][nt][u + 2], u20, y));
          }
        }
      if (whole) {
        __syncwarp();
#pragma unroll 1
        for (int col = 0; col < real; ++col)
          kv4_store_column(p, use.b, use.hc, col, kCols, *reinterpret_cast<const float4*>(part + col * 128 + lane * 4),
                           part[kCols * 128 + col], part[kCols * 129 + col], part[kCols * 130 + col]);
        __syncwarp();
      } else if (lane == 0) {
        Kv4Piece& q = sm.piece[pi];
        q.start = seg_start;
        q.b = use.b;
        q.hc = use.hc;
        q.tiles = use.tiles;
      }
      seg_start += use.tiles;
      use.advance(p, n);
    }
  }
  // sequences of no tokens: zeros, the columns of each spread over the grid's warps
  if (sm.empties) {
#pragma unroll 1
    for (int b0 = 0; b0 < p.batch; b0 += 32) {
      unsigned none = __ballot_sync(0xffffffffu, b0 + lane < p.batch && kv4_length(p, min(b0 + lane, p.batch - 1)) == 0);
      for (; none; none &= none - 1) {
        const int b = b0 + __ffs(none) - 1;
        for (int i = ((blockIdx.x + b) % gridDim.x) * (W + 1) + warp; i < HC * kCols; i += gridDim.x * (W + 1))
          if ((i / kCols) % p.col_blocks * kCols + i % kCols < p.group * p.queries)
            kv4_store_column(p, b, i / kCols, i % kCols, kCols, make_float4(0.f, 0.f, 0.f, 0.f), 0.f, 0.f, 0.f);
      }
    }
  }
  if (c0 >= c1) return;
  __syncthreads();

  // ---- merge the pieces of each segment, in line order.  A lane has a piece, the lowest of a
  // segment's pieces leads; a warp takes a (segment, column): a lane a piece for the weights,
  // then a lane 4 channels.  What is not whole here goes to the workspace: at most the CTA's
  // first and last segment.
  static_assert(2 * W <= 32, "a lane a piece");
  const Kv4Piece pc = sm.piece[min(lane, 2 * W - 1)];
  const int my_start = lane < 2 * W ? pc.start : -1;
  const unsigned same = __match_any_sync(0xffffffffu, my_start);
  const bool leads = my_start >= 0 && __ffs(same) - 1 == lane;
  const bool whole = pc.start >= c0 && pc.start + pc.tiles <= c1;
  const int side = pc.start <= c0 ? 0 : 1;
  const int cols = leads ? min(kCols, p.group * p.queries - (pc.hc - kv4_divide(pc.hc, p.col_blocks_m) * p.col_blocks) * kCols) : 0;
  int units = cols;                         // up to and with a leader's
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, units, o);
    if (lane >= o) units += y;
  }
  const int all_units = __shfl_sync(0xffffffffu, units, 31);
  int cross[2];                             // leaders of the segments that other CTAs share, or -1
  cross[0] = __ffs(__ballot_sync(0xffffffffu, leads && !whole && side == 0)) - 1;
  cross[1] = __ffs(__ballot_sync(0xffffffffu, leads && !whole && side == 1)) - 1;
#pragma unroll 1
  for (int u = warp; u < all_units; u += W + 1) {
    const int lead = __ffs(__ballot_sync(0xffffffffu, units > u)) - 1;
    const unsigned members = __shfl_sync(0xffffffffu, same, lead);
    const int col = u - __shfl_sync(0xffffffffu, units - cols, lead);
    const bool in = members >> lane & 1;
    const float* at = piece_at(in ? lane : lead);
    const float base = in ? at[kCols * 128 + col] : -INFINITY;
    const float mx = kv4_warp_max(base), w = kv4_weight(base, mx);
    const float wl = in ? w * at[kCols * 129 + col] : 0.f, wr = in ? w * at[kCols * 130 + col] : 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    float l = 0.f, rounded = 0.f;
#pragma unroll 1
    for (unsigned m = members; m;) {        // four pieces a turn, their loads in flight together
      float4 v[4];
      float wk[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int k = m ? __ffs(m) - 1 : lead;
        const float lk = __shfl_sync(0xffffffffu, wl, k), rk = __shfl_sync(0xffffffffu, wr, k);
        wk[i] = __shfl_sync(0xffffffffu, w, k);
        l += m ? lk : 0.f;
        rounded += m ? rk : 0.f;
        wk[i] = m ? wk[i] : 0.f;
        v[i] = *reinterpret_cast<const float4*>(piece_at(k) + col * 128 + lane * 4);
        m &= m - 1;
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
        acc.x = fmaf(wk[i], v[i].x, acc.x), acc.y = fmaf(wk[i], v[i].y, acc.y), acc.z = fmaf(wk[i], v[i].z, acc.z),
        acc.w = fmaf(wk[i], v[i].w, acc.w);
    }
    if (__shfl_sync(0xffffffffu, whole, lead)) {
      kv4_store_column(p, __shfl_sync(0xffffffffu, pc.b, lead), __shfl_sync(0xffffffffu, pc.hc, lead), col, kCols, acc, mx, l,
                       rounded);
    } else {
      float* part = p.parts + ((int64_t)blockIdx.x * 2 + __shfl_sync(0xffffffffu, side, lead)) * kKv4PartFloats;
      __stcg(reinterpret_cast<float4*>(part + col * 128 + lane * 4), acc);
      if (lane == 0) {
        __stcg(part + kCols * 128 + col, mx);
        __stcg(part + kCols * 129 + col, l);
        __stcg(part + kCols * 130 + col, rounded);
      }
    }
  }
  if (cross[0] < 0 && cross[1] < 0) return; // the same for every warp
  __syncthreads();
  if (tid < 2 && cross[tid] >= 0) {
    const Kv4Piece pc = sm.piece[cross[tid]];
    const int first = pc.start / per, n = (pc.start + pc.tiles - 1) / per - first + 1;
    // releases what the CTA wrote before the barrier, acquires what the others did
    int before;
    asm volatile("atom.add.acq_rel.gpu.global.s32 %0, [%1], 1;" : "=r"(before) : "l"(p.counters + first) : "memory");
    sm.last[tid] = before == n - 1;
    if (before == n - 1) p.counters[first] = 0;
  }
  __syncthreads();
  int unit = 0;
#pragma unroll 1
  for (int s = 0; s < 2; ++s) {
    if (cross[s] < 0 || !sm.last[s]) continue;
    // every CTA's piece is there.  The segment's piece of a CTA is its first one, but for the CTA
    // in whose middle it starts
    const Kv4Piece pc = sm.piece[cross[s]];
    const int first = pc.start / per, n = (pc.start + pc.tiles - 1) / per - first + 1;
    const int skip = pc.start > first * per ? 1 : 0;
    const int cols = min(kCols, p.group * p.queries - (pc.hc - kv4_divide(pc.hc, p.col_blocks_m) * p.col_blocks) * kCols);
    for (int col = 0; col < cols; ++col) {
      if (unit++ % (W + 1) != warp) continue;
      float mx = -INFINITY, l = 0.f, rounded = 0.f;
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
      for (int k0 = 0; k0 < n; k0 += 16) {  // 16 pieces a turn, their loads in flight together
        const int k = k0 + (lane & 15);
        const float* pk = p.parts + ((int64_t)(first + k) * 2 + (k == 0 ? skip : 0)) * kKv4PartFloats;
        const float base = k < n ? __ldcg(pk + kCols * 128 + col) : -INFINITY;
        const float lk = k < n ? __ldcg(pk + kCols * 129 + col) : 0.f, rk = k < n ? __ldcg(pk + kCols * 130 + col) : 0.f;
        float4 v[16];
#pragma unroll
        for (int i = 0; i < 16; ++i)
          v[i] = __ldcg(reinterpret_cast<const float4*>(
              p.parts + ((int64_t)(first + min(k0 + i, n - 1)) * 2 + (min(k0 + i, n - 1) == 0 ? skip : 0)) * kKv4PartFloats +
              col * 128 + lane * 4));       // past the last piece: that one again, times 0
        const float joint = fmaxf(mx, kv4_warp_max(base)), old = kv4_weight(mx, joint);
        const float w = kv4_weight(base, joint), wl = w * lk, wr = w * rk;
        l *= old;
        rounded *= old;
        acc.x *= old, acc.y *= old, acc.z *= old, acc.w *= old;
        mx = joint;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const float wi = __shfl_sync(0xffffffffu, w, i);
          l += __shfl_sync(0xffffffffu, wl, i);
          rounded += __shfl_sync(0xffffffffu, wr, i);
          acc.x = fmaf(wi, v[i].x, acc.x), acc.y = fmaf(wi, v[i].y, acc.y), acc.z = fmaf(wi, v[i].z, acc.z),
          acc.w = fmaf(wi, v[i].w, acc.w);
        }
      }
      kv4_store_column(p, pc.b, pc.hc, col, kCols, acc, mx, l, rounded);
    }
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
  int* counters;                            // (batch, KV heads) zero between calls
  float* scores;                            // (batch, KV heads, width)
  int q_dtype, batch, queries, q_heads, group, width, keep, first, last;
};

// Pages of a sequence, within the block table.
__device__ __forceinline__ int kv4_pages(const Kv4SelectParams& p, int b) {
  const int64_t cap = (int64_t)p.width << p.pool.page_shift;
  int64_t len = __ldg(p.lengths + b);
  if (len > cap) {
    record_error(p.pool.err, kDevBadPosition);
    len = cap;
  }
  return len <= 0 ? 0 : (int)((len + (1 << p.pool.page_shift) - 1) >> p.pool.page_shift);
}

// Order-preserving integer of a score (larger score, larger key; -0 equals 0).
__device__ __forceinline__ uint32_t kv4_key_of(float s) {
  const uint32_t u = __float_as_uint(s + 0.f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

constexpr int kKv4SelWarps = 8, kKv4SelThreads = kKv4SelWarps * 32;
constexpr int kKv4ScorePages = 8;           // pages of a warp
constexpr int kKv4ScoreChunk = kKv4SelWarps * kKv4ScorePages, kKv4ScoreCols = 16;
constexpr int kKv4MaxSegments = 65536;      // (sequence, KV head) pairs the counters have room for

struct Kv4SelectSmem {
  int pos[kKv4ScoreCols][32], neg[kKv4ScoreCols][32];   // positive and negative query codes, four a word
  float unit[kKv4ScoreCols];
  uint32_t lane[2][kKv4SelWarps];           // a value a warp, two sets in turn
  int last;
};

// The pages to keep of one (KV head, sequence), by its last CTA: thread t has the keys of the pages
// [t * per, (t + 1) * per) (REGS > 0: in registers), the smallest key to keep is found bit by bit
// below the bits that all keys share, and scans put the kept pages in order.
template <int REGS>
__device__ __forceinline__ void kv4_choose(const Kv4SelectParams& p, Kv4SelectSmem& sm, const float* sc, int* out, int n) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int per = (n + kKv4SelThreads - 1) / kKv4SelThreads, i0 = min(tid * per, n), mine = min(per, n - i0);
  auto forced = [&](int i) { return i < p.first || i >= n - p.last; };
  uint32_t held[REGS ? REGS : 1];
  if (REGS) {
#pragma unroll
    for (int i = 0; i < REGS; ++i) held[i] = i < mine && !forced(i0 + i) ? kv4_key_of(__ldcg(sc + i0 + i)) : 0;
  }
  // f(page, key) over this thread's scored pages
  auto each = [&](auto f) {
    if (REGS) {
#pragma unroll
      for (int i = 0; i < REGS; ++i)
        if (i < mine && !forced(i0 + i)) f(i0 + i, held[i]);
    } else {
      for (int i = i0; i < i0 + mine; ++i)
        if (!forced(i)) f(i, kv4_key_of(__ldcg(sc + i)));
    }
  };
  int turn = 0;
  // one value a warp, exchanged: lane w < 8 gets warp w's
  auto exchange = [&](uint32_t x) {
    if (lane == 0) sm.lane[turn][warp] = x;
    __syncthreads();
    const uint32_t y = sm.lane[turn][lane & (kKv4SelWarps - 1)];
    turn ^= 1;
    return y;
  };
  // what all threads before this one hold, and what all hold
  auto scan = [&](int x, int* all) {
    int y = x;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int z = __shfl_up_sync(0xffffffffu, y, o);
      if (lane >= o) y += z;
    }
    const int w = (int)exchange((uint32_t)__shfl_sync(0xffffffffu, y, 31));
    *all = __reduce_add_sync(0xffffffffu, lane < kKv4SelWarps ? w : 0);
    return y - x + __reduce_add_sync(0xffffffffu, lane < warp ? w : 0);
  };
  const int need = p.keep - p.first - p.last;   // of the scored pages; there are more
  uint32_t ones = 0xffffffffu, any = 0;
  each([&](int, uint32_t k) { ones &= k, any |= k; });
  ones = __reduce_and_sync(0xffffffffu, exchange(__reduce_and_sync(0xffffffffu, ones)));
  any = __reduce_or_sync(0xffffffffu, exchange(__reduce_or_sync(0xffffffffu, any)));
  // the largest key with at least `need` keys at or above it
  const int top = 31 - __clz(ones ^ any);
  uint32_t key = top < 0 ? ones : ones >> top >> 1 << top << 1;
  bool exact = false;                       // exactly `need`
  for (int bit = top; bit >= 0 && !exact; --bit) {
    const uint32_t trial = key | (1u << bit);
    int c = 0;
    each([&](int, uint32_t k) { c += k >= trial; });
    c = (int)exchange((uint32_t)__reduce_add_sync(0xffffffffu, c));
    c = __reduce_add_sync(0xffffffffu, lane < kKv4SelWarps ? c : 0);
    if (c >= need) key = trial;
    exact = c == need;
  }
  int above = 0, equal = 0, total = 0, take = 0x7fffffff;
  each([&](int, uint32_t k) { above += k > key, equal += k == key; });
  if (!exact) {                             // of the keys equal to it only the first
    const int before = scan(equal, &total);
    int all_above;
    scan(above, &all_above);
    take = max(0, need - all_above - before);
  }
  take = min(equal, take);
  int pinned = 0;
  for (int i = i0; i < i0 + mine; ++i) pinned += forced(i);
  int at = scan(above + take + pinned, &total);
  if (REGS) {
#pragma unroll
    for (int i = 0; i < REGS; ++i)
      if (i < mine && (forced(i0 + i) || held[i] > key || (held[i] == key && take-- > 0))) out[at++] = i0 + i;
  } else {
    for (int i = i0; i < i0 + mine; ++i) {
      const uint32_t k = kv4_key_of(__ldcg(sc + i));
      if (forced(i) || k > key || (k == key && take-- > 0)) out[at++] = i;
    }
  }
}

// ---- selection.  A CTA scores 64 pages of one (KV head, sequence): a warp takes 8, a lane 4
// channels of their bounds; per page and column two dp4a (the positive codes against the
// upper bounds, the negative ones against the lower) and one warp sum.  The CTA that is done
// last keeps the best pages.  4 sequences of 131072 tokens in pages of 64, 8 heads of 4 (17 MB of
// bounds, 2.6 us of HBM time): 12 us, the latency of four dependent loads, an atomic and some
// fifteen exchanges; as two launches 23 us.
template <int REGS>
__global__ void __launch_bounds__(kKv4SelThreads) kv4_select_kernel(const Kv4SelectParams p) {
  __shared__ Kv4SelectSmem sm;
  const int head = blockIdx.y, b = blockIdx.z, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int n = kv4_pages(p, b), lo = p.first, hi = n - p.last;   // the pages to score
  const int64_t seg = (int64_t)b * p.pool.heads + head;
  int* out = p.out + seg * p.keep;
  if (n <= p.keep) {
    if (blockIdx.x == 0)
      for (int i = threadIdx.x; i < p.keep; i += kKv4SelThreads) out[i] = i < n ? i : -1;
    return;
  }
  if (lo + (int)blockIdx.x * kKv4ScoreChunk >= hi) return;
  const int p0 = lo + (blockIdx.x * kKv4SelWarps + warp) * kKv4ScorePages;
  // the pages' bounds, all in flight together
  int page = -1;
  if (lane < kKv4ScorePages && p0 + lane < hi) page = kv4_page(p.pool, p.table + b * p.table_stride, p0 + lane, p.width);
  int up[kKv4ScorePages], dn[kKv4ScorePages];
#pragma unroll
  for (int i = 0; i < kKv4ScorePages; ++i) {
    const int pg = __shfl_sync(0xffffffffu, page, i);
    up[i] = dn[i] = 0;
    if (pg >= 0) {
      const int* bd = reinterpret_cast<const int*>(p.pool.bounds + ((int64_t)pg * p.pool.heads + head) * 256);
      up[i] = __ldg(bd + lane);
      dn[i] = __ldg(bd + 32 + lane);
    }
  }
  const float scale = page >= 0 ? __ldg(p.pool.bound_scales + (int64_t)page * p.pool.heads + head) : 0.f;
  float best[kKv4ScorePages];
#pragma unroll
  for (int i = 0; i < kKv4ScorePages; ++i) best[i] = -INFINITY;
  const int cols = p.queries * p.group;
  for (int c0 = 0; c0 < cols; c0 += kKv4ScoreCols) {
    const int nc = min(kKv4ScoreCols, cols - c0);
    if (c0) __syncthreads();
    for (int col = warp; col < nc; col += kKv4SelWarps) {
      const int gc = c0 + col;
      const int64_t at = b * p.qs[0] + (gc / p.group) * p.qs[1] + (head * p.group + gc % p.group) * p.qs[2] + lane * 4;
      const uint2 raw = __ldg(reinterpret_cast<const uint2*>(reinterpret_cast<const uint16_t*>(p.q) + at));
      float x[4];
      if (p.q_dtype == STARKV_F16) {
        const float2 f0 = kv4_halves(raw.x), f1 = kv4_halves(raw.y);
        x[0] = f0.x, x[1] = f0.y, x[2] = f1.x, x[3] = f1.y;
      } else {
        x[0] = __uint_as_float(raw.x << 16), x[1] = __uint_as_float(raw.x & 0xffff0000u);
        x[2] = __uint_as_float(raw.y << 16), x[3] = __uint_as_float(raw.y & 0xffff0000u);
      }
      float a = fmaxf(fmaxf(fabsf(x[0]), fabsf(x[1])), fmaxf(fabsf(x[2]), fabsf(x[3])));
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, o));
      const float u = __fdiv_rn(a, 127.f);
      uint32_t wp = 0, wn = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int c = u > 0.f ? (int)rintf(__fdiv_rn(x[i], u)) : 0;
        wp |= (uint32_t)max(c, 0) << (8 * i);
        wn |= (uint32_t)(min(c, 0) & 255) << (8 * i);
      }
      sm.pos[col][lane] = (int)wp;
      sm.neg[col][lane] = (int)wn;
      if (lane == 0) sm.unit[col] = u;
    }
    __syncthreads();
    for (int col = 0; col < nc; ++col) {
      const int wp = sm.pos[col][lane], wn = sm.neg[col][lane];
      const float u = sm.unit[col];
#pragma unroll
      for (int i = 0; i < kKv4ScorePages; ++i) {
        const int dot = __reduce_add_sync(0xffffffffu, __dp4a(wp, up[i], __dp4a(wn, dn[i], 0)));
        best[i] = fmaxf(best[i], __fmul_rn((float)dot, u));
      }
    }
  }
  float mine = 0.f;
#pragma unroll
  for (int i = 0; i < kKv4ScorePages; ++i)
    if (lane == i) mine = best[i];
  float* sc = p.scores + seg * p.width;
  if (lane < kKv4ScorePages && p0 + lane < hi) __stcg(sc + p0 + lane, page >= 0 ? __fmul_rn(mine, scale) : -INFINITY);
  const int ctas = (hi - lo + kKv4ScoreChunk - 1) / kKv4ScoreChunk;
  __syncthreads();
  if (threadIdx.x == 0) {
    // releases the scores that the CTA wrote before the barrier, acquires the others'
    int before;
    asm volatile("atom.add.acq_rel.gpu.global.s32 %0, [%1], 1;" : "=r"(before) : "l"(p.counters + seg) : "memory");
    sm.last = before == ctas - 1;
    if (before == ctas - 1) p.counters[seg] = 0;
  }
  __syncthreads();
  if (sm.last) kv4_choose<REGS>(p, sm, sc, out, n);
}

}  // namespace starkv
