// kv4_prefix.cuh — many queries over one prefix in the paged 4-bit cache, on the tensor cores, and the
// joining with the queries' own tokens.
//
// All queries of a KV head, of whatever sequence, are rows of S = Q K^T and O += P V with the prefix's
// keys and values; the softmax and the products are those of packed_attn.cuh, without masks.  The
// operands come from 4-bit codes, value = s c + m for each group of 32 channels.
//   Values are rounded once to fp16 (2^-11, as the weights are).
//   Keys are exact: a score errs by the sum over all channels, and a rounded key put the outputs of
//   fp16 off by 1.0e-3 where one channel in a hundred is eight times as large (2.7e-4 now).  With
//   s = s' + s'', s' the upper 7 bits, s' c and s'' c are fp16 numbers, and so is m:
//     q.k = sum_d q_d (s' c_d) + sum_d q_d (s'' c_d) + sum_g m_g sum_{d in g} q_d,
//   three products into one accumulator, the last with the sums of q as two fp16 parts (nine matrix
//   instructions more for each tile and step).  A group whose parts leave fp16 is rounded and held
//   at 65504 instead.
//   Queries go to fp16 with a power of two a row (exact for bf16 down to 2^-24 of the row's largest).
// Within eight channels operands hold channels 0 4 1 5 2 6 3 7, as the masked nibbles of a word come:
// the same for Q and K, undone where O is written.
//
// CTA, one an SM, 25 warps:
//   warps 0-7   a thread a row of tile 0 (0-3) and tile 1 (4-7): lays out Q, softmax, output;
//   warp 8      issues the matrix products;
//   warps 9-24  turn codes into operands, straight from global memory: keys or values of a tile of 16
//               tokens each.
// Rows.  Up to 128 rows a KV head: both tiles hold them, and take the even and the odd steps of 128
// tokens.  More: tiles of 128 rows each, 256 a CTA, each block of 256 reads the prefix.
// Bound: a step of 256 rows takes about 6100 cycles, of which the products need 3200.  Of a tile's turn
// the rows' softmax is 3600 (S read twice in short loops, as registers are few: the 25 warps are allotted
// as 28, which leaves 72 a thread, and 204 bytes are spilled), the wait for its products behind the other
// tile's 1700; the codes are turned in less.  Beside the steps a CTA takes about 46000 cycles: 3000 to
// start, 27000 to lay out the queries (a thread reads a row of its own, twice), 9000 to the first
// weights (instructions come in), 7000 for the parts and the end.  256 rows of 8 KV heads, 32769
// tokens, 15 steps at most: 143000 cycles, 82 us, 404 TFLOP/s of products over 128 channels, 630 with the
// parts of the exact keys.  The warps share one instruction cache, so
// code is kept short rather than unrolled.  Measured and slower: seven warps for the codes and 192
// registers for a row's softmax, bulk copies of the codes into shared memory, the next tile's codes in
// registers ahead, a row's S in 64 registers (28 warps), loads of S ahead (spills: 127 us).
// Work.  A KV head and block of rows is cut into equal ranges of the prefix so that there is a piece
// for every SM; a second kernel adds the parts in order, the own tokens' part last.
#pragma once
#include "kv4_shared.cuh"
#include "packed_attn.cuh"

namespace starkv {

constexpr int kKvpThreads = 25 * 32;                         // of 72 registers
constexpr int kKvpMaxParts = 2 * kKv4MaxGrid;                // tile parts in the workspace
constexpr int kKvpMinPiece = 2;                              // steps of 128 tokens a piece has at least
constexpr size_t kKvpPartBytes = (size_t)kKvpMaxParts * kPkTilePart * sizeof(float);
static_assert(kKvpPartBytes <= kKv4WorkspaceBytes - kKv4CounterBytes, "parts lie where the own tokens' attention had its scratch");

struct Kv4PrefixParams {
  Kv4Pool pool;
  Kv4SharedParams s;           // queries, outputs, the own tokens' part
  const int* table;
  const int* length;
  int width;
  int rows, blocks, halves;    // rows a KV head, blocks of 256, whether both tiles hold the same rows
  float scale_log2;
  unsigned long long wait_ns;
  int skip_step;               // tests: the first CTA's step whose values one warp keeps, or -1
  int grid;                    // CTAs of the first kernel
  float* parts;
};

// One step of a row, as pk_softmax, with S read from tensor memory 32 columns at a time and twice (for
// the maximum, for the weights): few registers and short loops.  `seen` tokens of the step are there,
// less those 16 whose byte of skip is not zero.
__device__ __forceinline__ void kvp_softmax(uint32_t sa, float sl2, int seen, bool held, PkRow& row, uint64_t* most, uint64_t skip) {
  const bool border = seen < kPkKeys || skip;
  auto hide = [&](int c, float* s) {
    const uint32_t gone = (uint32_t)(skip >> (c * 16));
#pragma unroll
    for (int i = 0; i < 32; ++i) s[i] = i < seen - c * 32 && !(gone >> (i >> 4 << 3) & 255) ? s[i] : -INFINITY;
  };
  float mt = -INFINITY;
#pragma unroll 1
  for (int c = 0; c < 4; ++c) {
    float s[32];
    tmem_ld32(sa + c * 32, s);
    if (border) hide(c, s);
    float mq[4] = {mt, s[0], s[1], s[2]};
#pragma unroll
    for (int i = 3; i < 31; i += 2) mq[i / 2 & 3] = pk_max3_nan(mq[i / 2 & 3], s[i], s[i + 1]);
    mt = pk_max3_nan(pk_max3_nan(mq[0], mq[1], mq[2]), mq[3], s[31]);
  }
  mt *= sl2;
  if (!(mt < INFINITY)) row.bad = true;
  const bool need = !row.bad && mt - kPkBias > row.m + kPkLazy;
  if (__any_sync(0xffffffffu, need)) {
    float alpha = 1.f;
    if (need) {
      alpha = row.m == -INFINITY ? 0.f : fast_exp2(row.m - (mt - kPkBias));
      row.l *= alpha;
      row.m = mt - kPkBias;
    }
    if (held) {
#pragma unroll 1
      for (int c = 0; c < 8; ++c) {
        float v[16];
        tmem_ld16(sa + 128 + c * 16, v);
        uint32_t w[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) w[i] = __float_as_uint(v[i] * alpha);
        tmem_st16(sa + 128 + c * 16, w);
      }
    }
  }
  // beyond 2^16 the exact product in the fma and m, which was rounded, would be far apart
  const bool far = __any_sync(0xffffffffu, fabsf(mt) > 65536.f && fabsf(mt) < INFINITY);
  const float base = row.m == -INFINITY ? 0.f : -row.m;
  float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll 1
  for (int c = 0; c < 4; ++c) {
    float s[32];
    tmem_ld32(sa + c * 32, s);
    if (border) hide(c, s);
    float f = sl2;
    if (far) {
#pragma unroll
      for (int i = 0; i < 32; ++i) s[i] *= sl2;
      f = 1.f;
    }
    uint32_t pk[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const float2 x = __ffma2_rn(make_float2(s[2 * i], s[2 * i + 1]), make_float2(f, f), make_float2(base, base));
      const float2 e = make_float2(fast_exp2(x.x), fast_exp2(x.y));
      sum[i & 1] = __fadd2_rn(sum[i & 1], e);
      pk[i] = pack2<__half>(e.x, e.y);
    }
    if (c * 32 == kPkMost) {
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if ((threadIdx.x & 31) == 0) mbar_arrive(most);
    }
    tmem_st16(sa + c * 16, pk);
  }
  row.l += (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
  tmem_st_wait();
}

struct KvpSmem {
  uint64_t q_full[2], k_full, k_empty, v_full[2], v_empty[2], s_full[2], p_most[2], p_full[2], o_full[2], mma_done;
  uint64_t skip[4];            // a byte a tile of 16 tokens: its page is bad
  uint32_t tmem;
  int abort;
};
constexpr int kKvpHeader = 1024;
static_assert(sizeof(KvpSmem) <= kKvpHeader, "header");
constexpr int kKvpSumBytes = 128 * 32;                      // 128 rows of 16 values: sums of a query, centres of a token
constexpr size_t kKvpSmemBytes = kKvpHeader + 1024 + 6 * (size_t)kPkTileBytes + 3 * kKvpSumBytes;
static_assert(kKvpSmemBytes <= 227 * 1024, "shared memory of one SM");

// The codes of a word as fp16 numbers -8 .. 7: channels (k, k + 4) in word k.  A nibble masked into the
// mantissa of 1024 is 1024 + c' (or 1024 + 16 c'), c = c' - 8.
__device__ __forceinline__ void kvp_codes(uint32_t codes, __half2* c) {
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const uint32_t a = ((k < 2 ? codes : codes >> 8) & (k & 1 ? 0x00f000f0u : 0x000f000fu)) | 0x64006400u;
    const __half2 h = *reinterpret_cast<const __half2*>(&a);
    c[k] = k & 1 ? __hfma2(h, __float2half2_rn(0.0625f), __float2half2_rn(-72.f)) : __hsub2(h, __float2half2_rn(1032.f));
  }
}
__device__ __forceinline__ uint4 kvp_words(const __half2* v) {
  const uint32_t* w = reinterpret_cast<const uint32_t*>(v);
  return make_uint4(w[0], w[1], w[2], w[3]);
}
// Values beyond 65504 are held there (they would become infinite); NaN stays.
__device__ __forceinline__ __half2 kvp_held(__half2 v) {
  return __hmin2_nan(__hmax2_nan(v, __float2half2_rn(-65504.f)), __float2half2_rn(65504.f));
}
// Eight values s c + m, rounded once.  CAREFUL, one branch a tile: where some may be beyond 65504, and
// tokens that are not there are zeros.
template <bool CAREFUL>
__device__ __forceinline__ uint4 kvp_values(uint32_t codes, __half2 s, __half2 m, bool here) {
  __half2 c[4];
  kvp_codes(codes, c);
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    c[k] = __hfma2(c[k], s, m);
    if (CAREFUL) c[k] = here ? kvp_held(c[k]) : __float2half2_rn(0.f);
  }
  return kvp_words(c);
}

// Whether 8 |s| + |m| of two groups leaves fp16 (values beyond 65504 would become infinite).
__device__ __forceinline__ bool kvp_large(uint32_t s, uint32_t m) {
  const __half2 t = __hfma2(__habs2(*reinterpret_cast<const __half2*>(&s)), __float2half2_rn(8.f), __habs2(*reinterpret_cast<const __half2*>(&m)));
  const uint32_t a = *reinterpret_cast<const uint32_t*>(&t);
  return ((a & 0x7c007c00u) + 0x04000400u) & 0x80008000u;
}

// Byte offset of the 16 bytes of channels 8 c16 .. 8 c16 + 7 of a row in a tile of two swizzled halves.
__device__ __forceinline__ uint32_t kvp_place(int row, int c16) {
  return (c16 >> 3) * (kPkTileBytes / 2) + row * 128 + (((c16 & 7) ^ (row & 7)) << 4);
}

// Byte offset of the 16 bytes of values 8 h .. 8 h + 7 of a row of 16, in core matrices of 8 rows (no
// swizzle): 128 bytes to the next along the row, 256 to the next rows.
__device__ __forceinline__ uint32_t kvp_sum_place(int row, int h) { return (row >> 3) * 256 + h * 128 + (row & 7) * 16; }

__device__ __forceinline__ __half2 kvp_both(uint32_t pair, int high) {
  const __half2 h = *reinterpret_cast<const __half2*>(&pair);
  return high ? __high2half2(h) : __low2half2(h);
}

// What a lane takes of 16 tokens' keys or values: codes and parameters.  Keys: lane = (half of the
// codes' 16-byte words, token).  Values: lane = (pair of quads of a group, pair of tokens).
struct KvpRaw {
  uint4 c[2], p[2];
  __device__ __forceinline__ void load(const uint8_t* tile, bool keys, int lane) {
    const uint8_t* code = tile + (keys ? (lane & 15) * 64 + (lane >> 4) * 32
                                       : kKv4VCodes + (lane >> 2 & 1) * 512 + (lane >> 3) * 128 + (lane & 3) * 16);
    const uint8_t* par = tile + (keys ? kKv4KParams : kKv4VParams) + (lane & 7) * 32;
    c[0] = __ldg(reinterpret_cast<const uint4*>(code)), c[1] = __ldg(reinterpret_cast<const uint4*>(code + (keys ? 16 : 64)));
    p[0] = __ldg(reinterpret_cast<const uint4*>(par)), p[1] = __ldg(reinterpret_cast<const uint4*>(par + 16));
  }
};

// Keys into rows row0 .. row0 + 15 of the operand tiles (s' c at dst, s'' c behind it) and of the
// centres; the eight lanes of a store go to eight banks.  Tokens from `left` on, for which raw may
// hold anything, are zeros.
__device__ __forceinline__ void kvp_keys(const KvpRaw& raw, uint8_t* dst, uint8_t* centres, int row0, int left, int lane) {
  const int t = lane & 15, q = (lane >> 4) * 2;
  const bool up = t >> 3;                                     // s of groups 2 i, 2 i + 1 in one word, m two on
  const uint32_t s[2] = {up ? raw.p[0].y : raw.p[0].x, up ? raw.p[1].y : raw.p[1].x};
  const uint32_t m[2] = {up ? raw.p[0].w : raw.p[0].z, up ? raw.p[1].w : raw.p[1].z};
  const bool here = t < left;
  const bool careful = __any_sync(0xffffffffu, !here || kvp_large(s[0], m[0]) || kvp_large(s[1], m[1]));
  // channels 8 (4 g + q + i): 64 bytes on where g is odd, in the other half from g = 2 on
  uint8_t* row = dst + (row0 + t) * 128;
  uint32_t sh[2], sl[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    sh[i] = s[i] & 0xfff0fff0u;
    const __half2 l = __hsub2(*reinterpret_cast<const __half2*>(&s[i]), *reinterpret_cast<const __half2*>(&sh[i]));
    sl[i] = *reinterpret_cast<const uint32_t*>(&l);
  }
  uint32_t centre[2] = {m[0], m[1]};
  if (careful) {
    // a group whose parts may leave fp16: the value itself, rounded, for the first product alone
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int h = 0; h < 2; ++h)
        if (!here || kvp_large(__byte_perm(s[i], 0, h ? 0x3232 : 0x1010), __byte_perm(m[i], 0, h ? 0x3232 : 0x1010)))
          centre[i] &= h ? 0x0000ffffu : 0xffff0000u;
  }
  auto put = [&](auto mode) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const uint32_t w[4] = {raw.c[i].x, raw.c[i].y, raw.c[i].z, raw.c[i].w};
      const int o = ((q + i) ^ (t & 7)) << 4;
      uint8_t* to[2] = {row + o, row + (o ^ 64)};
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        uint8_t* at = to[g & 1] + (g >> 1) * (kPkTileBytes / 2);
        __half2 c[4], hi[4], lo[4];
        kvp_codes(w[g], c);
        const __half2 h = kvp_both(sh[g >> 1], g & 1), l = kvp_both(sl[g >> 1], g & 1);
#pragma unroll
        for (int k = 0; k < 4; ++k) hi[k] = __hmul2(c[k], h), lo[k] = __hmul2(c[k], l);
        if constexpr (decltype(mode)::value) {
          const uint32_t pick = g & 1 ? 0x3232 : 0x1010;
          if (!here || kvp_large(__byte_perm(s[g >> 1], 0, pick), __byte_perm(m[g >> 1], 0, pick))) {
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              hi[k] = here ? kvp_held(__hfma2(c[k], kvp_both(s[g >> 1], g & 1), kvp_both(m[g >> 1], g & 1))) : __float2half2_rn(0.f);
              lo[k] = __float2half2_rn(0.f);
            }
          }
        }
        *reinterpret_cast<uint4*>(at) = kvp_words(hi);
        *reinterpret_cast<uint4*>(at + kPkTileBytes) = kvp_words(lo);
      }
    }
  };
  if (careful) put(std::true_type());
  else put(std::false_type());
  // (m_0, m_0, m_1, m_1, ...), then zeros
  uint4 c = make_uint4(0, 0, 0, 0);
  if (q == 0)
    c = make_uint4(__byte_perm(centre[0], 0, 0x1010), __byte_perm(centre[0], 0, 0x3232), __byte_perm(centre[1], 0, 0x1010),
                   __byte_perm(centre[1], 0, 0x3232));
  *reinterpret_cast<uint4*>(centres + kvp_sum_place(row0 + t, q >> 1)) = c;
}

// Values; the later four pairs take their odd token first, so that the eight lanes of a store go to
// eight banks.
__device__ __forceinline__ void kvp_vals(const KvpRaw& raw, uint8_t* dst, int row0, int left, int lane) {
  const int pair = lane & 7, e = lane >> 3;                   // tokens 2 pair, 2 pair + 1; channels 8 e .. 8 e + 7 of each group
  const uint32_t aw[4] = {raw.c[0].x, raw.c[0].y, raw.c[0].z, raw.c[0].w}, bw[4] = {raw.c[1].x, raw.c[1].y, raw.c[1].z, raw.c[1].w};
  const uint32_t sw[4] = {raw.p[0].x, raw.p[0].y, raw.p[0].z, raw.p[0].w}, mw[4] = {raw.p[1].x, raw.p[1].y, raw.p[1].z, raw.p[1].w};
  bool large = false;
#pragma unroll
  for (int g = 0; g < 4; ++g) large = large || kvp_large(sw[g], mw[g]);
  const bool careful = __any_sync(0xffffffffu, 2 * pair + 2 > left || large);
  auto put = [&](auto mode) {
#pragma unroll
    for (int turn = 0; turn < 2; ++turn) {
      const int odd = turn ^ (pair >> 2), t = 2 * pair + odd;
      const uint32_t both = odd ? 0x3232 : 0x1010, join = odd ? 0x7632 : 0x5410;
      const int o = (e ^ (t & 7)) << 4;
      uint8_t* row = dst + (row0 + t) * 128;
      uint8_t* to[2] = {row + o, row + (o ^ 64)};
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const uint32_t sg = __byte_perm(sw[g], 0, both), mg = __byte_perm(mw[g], 0, both);
        *reinterpret_cast<uint4*>(to[g & 1] + (g >> 1) * (kPkTileBytes / 2)) =
            kvp_values<decltype(mode)::value>(__byte_perm(aw[g], bw[g], join), *reinterpret_cast<const __half2*>(&sg),
                                              *reinterpret_cast<const __half2*>(&mg), t < left);
      }
    }
  };
  if (careful) put(std::true_type());
  else put(std::false_type());
}

// A row of queries as an operand, times 2^-k, and its sums over the groups of 32 channels, as two fp16
// parts each; returns k.
__device__ __forceinline__ int kvp_query(const void* q, int dtype, int64_t at, bool live, uint8_t* dst, uint8_t* sums, int row) {
  const uint4* src = reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(q) + at);
  const bool bf = dtype == STARKV_BF16;
  const uint32_t limit = bf ? 0x7f80u : 0x7c00u;              // bits of infinity
  uint32_t top = 0;                                           // bits of the largest finite magnitude
  if (live) {
#pragma unroll 8
    for (int i = 0; i < 16; ++i) {
      const uint4 w = __ldg(src + i);
      const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t lo = u[j] & 0x7fffu, hi = u[j] >> 16 & 0x7fffu;
        top = max(top, max(lo < limit ? lo : 0u, hi < limit ? hi : 0u));
      }
    }
  }
  // the largest value below 2^10, so that 32 of them stay in fp16: bf16 to [2^9, 2^10), fp16 only down
  const int k = bf ? (top >= 0x80u ? (int)(top >> 7) - 127 - 9 : 0) : max((int)(top >> 10) - 15 - 9, 0);
  // 2^-k in two factors: k reaches from -135 to 118
  const float f0 = __uint_as_float((127 - k / 2) << 23), f1 = __uint_as_float((127 - (k - k / 2)) << 23);
  uint32_t parts[4];
#pragma unroll
  for (int g = 0; g < 4; ++g) {
    float sum = 0.f;
#pragma unroll 4
    for (int i = 4 * g; i < 4 * g + 4; ++i) {
      const uint4 w = live ? __ldg(src + i) : make_uint4(0, 0, 0, 0);
      uint32_t h[4] = {w.x, w.y, w.z, w.w};                   // pairs (0, 1) (2, 3) (4, 5) (6, 7)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float2 x = kv4_halves(h[j]);
        if (bf) x = make_float2(__uint_as_float(h[j] << 16), __uint_as_float(h[j] & 0xffff0000u));
        h[j] = pack2<__half>(x.x * f0 * f1, x.y * f0 * f1);
        x = kv4_halves(h[j]);
        sum += x.x + x.y;
      }
      *reinterpret_cast<uint4*>(dst + kvp_place(row, i)) =
          make_uint4(__byte_perm(h[0], h[2], 0x5410), __byte_perm(h[0], h[2], 0x7632), __byte_perm(h[1], h[3], 0x5410), __byte_perm(h[1], h[3], 0x7632));
    }
    const float hi = __half2float(__float2half_rn(sum));
    parts[g] = pack2<__half>(hi, fabsf(hi) < INFINITY ? sum - hi : 0.f);
  }
  *reinterpret_cast<uint4*>(sums + kvp_sum_place(row, 0)) = make_uint4(parts[0], parts[1], parts[2], parts[3]);
  *reinterpret_cast<uint4*>(sums + kvp_sum_place(row, 1)) = make_uint4(0, 0, 0, 0);
  return k;
}

// Where a row's query is, and its own part.
struct KvpRow {
  int64_t q, out, own;         // elements; row of own_out, own_lse and lse
  bool live;
};
__device__ __forceinline__ KvpRow kvp_row(const Kv4PrefixParams& p, int kvh, int r) {
  KvpRow a;
  a.live = r < p.rows;
  const int token = r / p.s.group, head = kvh * p.s.group + r - token * p.s.group;
  const int b = token / p.s.queries, t = token - b * p.s.queries;
  a.q = b * p.s.qs[0] + t * p.s.qs[1] + head * p.s.qs[2];
  a.out = b * p.s.os[0] + t * p.s.os[1] + head * p.s.os[2];
  a.own = (int64_t)token * p.s.q_heads + head;
  return a;
}

// How the two parts of a row go together: out = x O + y own, with O the prefix's sums (m, l in the log2
// domain) and own the own tokens' output.
struct KvpJoin {
  float x, y, lse;
};
__device__ __forceinline__ KvpJoin kvp_join(float m, float l, float own_lse) {
  const float own = own_lse * 1.4426950408889634f, top = kv4_max_nan(m, own);
  KvpJoin j = {0.f, 0.f, -INFINITY};
  if (top == -INFINITY) return j;
  const float wp = m == -INFINITY ? 0.f : fast_exp2(m - top), ws = own == -INFINITY ? 0.f : fast_exp2(own - top);
  const float total = fmaf(wp, l, ws);
  j.x = wp / total, j.y = ws / total, j.lse = (top + log2f(total)) * 0.6931471805599453f;
  return j;
}

// Adds eight channels of the own part to eight of the prefix's (operand order) and writes them in the
// channels' order.
__device__ __forceinline__ void kvp_write8(const Kv4PrefixParams& p, const KvpRow& at, int block, const float* v, float y) {
  const float4* mine = reinterpret_cast<const float4*>(p.s.own_out + at.own * 128 + block * 8);
  const float4 a = mine[0], b = mine[1];
  const float u[8] = {fmaf(a.x, y, v[0]), fmaf(a.y, y, v[2]), fmaf(a.z, y, v[4]), fmaf(a.w, y, v[6]),
                      fmaf(b.x, y, v[1]), fmaf(b.y, y, v[3]), fmaf(b.z, y, v[5]), fmaf(b.w, y, v[7])};
  const int64_t to = at.out + block * 8;
  if (p.s.out_dtype == STARKV_F32) {
    float4* d = reinterpret_cast<float4*>(reinterpret_cast<float*>(p.s.out) + to);
    d[0] = make_float4(u[0], u[1], u[2], u[3]), d[1] = make_float4(u[4], u[5], u[6], u[7]);
    return;
  }
  uint32_t w[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) w[k] = p.s.out_dtype == STARKV_BF16 ? pack2<__nv_bfloat16>(u[2 * k], u[2 * k + 1]) : pack2<__half>(u[2 * k], u[2 * k + 1]);
  *reinterpret_cast<uint4*>(reinterpret_cast<__half*>(p.s.out) + to) = make_uint4(w[0], w[1], w[2], w[3]);
}

// A row whose whole prefix is in tensor memory.
static __device__ __noinline__ void kvp_finish(const Kv4PrefixParams& p, KvpRow at, uint32_t o_col, float m, float l) {
  KvpJoin j = {0.f, 0.f, 0.f};
  if (at.live) j = kvp_join(m, l, p.s.own_lse[at.own]);
#pragma unroll 1
  for (int c = 0; c < 4; ++c) {
    float v[32];
    __syncwarp();
    tmem_ld32(o_col + c * 32, v);
    if (!at.live) continue;
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] = m == -INFINITY ? 0.f : v[i] * j.x;
#pragma unroll
    for (int i = 0; i < 4; ++i) kvp_write8(p, at, c * 4 + i, v + 8 * i, j.y);
  }
  if (at.live && p.s.lse) p.s.lse[at.own] = j.lse;
}

// How the prefix is cut: the same in both kernels.
struct KvpCut {
  int length, steps, splits, parts;        // tokens, steps of 128 of them, ranges, parts of a row
};
__device__ __forceinline__ KvpCut kvp_cut(const Kv4PrefixParams& p) {
  KvpCut c;
  c.length = min(max(*p.length, 0), p.width << p.pool.page_shift);
  c.steps = (c.length + kPkKeys - 1) / kPkKeys;
  c.splits = max(1, min(c.steps / kKvpMinPiece, p.grid / (p.pool.heads * p.blocks)));
  c.parts = p.halves ? 2 * c.splits : c.splits;
  return c;
}

// The parts of cut rows, in order, then the own tokens': a thread eight channels of a row, a CTA those
// of a tile's 128 rows (so that a part is read in lines).
__global__ void __launch_bounds__(128) kv4_prefix_join_kernel(const __grid_constant__ Kv4PrefixParams p) {
  const KvpCut cut = kvp_cut(p);
  if (cut.parts == 1) return;
  const int tiles = p.halves ? 1 : 2, tile = blockIdx.x >> 4, block = blockIdx.x & 15, r = threadIdx.x;
  const int item = tile / tiles, x = tile % tiles;
  const KvpRow at = kvp_row(p, item / p.blocks, item % p.blocks * 256 + x * 128 + r);
  if (!at.live) return;
  const float* parts = p.parts + (int64_t)tile * cut.parts * kPkTilePart;
  float m = -INFINITY, l = 0.f, v[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = 0.f;
  constexpr int kAhead = 9;
#pragma unroll 1
  for (int k0 = 0; k0 < cut.parts; k0 += kAhead) {
    float2 a[kAhead];
    float4 o[kAhead][2];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const float* one = parts + (int64_t)min(k0 + i, cut.parts - 1) * kPkTilePart;
      a[i] = __ldcg(reinterpret_cast<const float2*>(one) + r);
      if (k0 + i >= cut.parts) a[i].x = -INFINITY;
#pragma unroll
      for (int h = 0; h < 2; ++h) o[i][h] = __ldcg(reinterpret_cast<const float4*>(one + 256) + (block * 2 + h) * 128 + r);
    }
    float top = m;
#pragma unroll
    for (int i = 0; i < kAhead; ++i) top = fmaxf(top, a[i].x);
    if (top == -INFINITY) continue;
    const float down = m == -INFINITY ? 0.f : fast_exp2(m - top);
    m = top;
    l *= down;
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] *= down;
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      if (a[i].x == -INFINITY) continue;                               // what such a part holds of O is not set
      const float w = fast_exp2(a[i].x - m);
      l = fmaf(w, a[i].y, l);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        v[4 * h] = fmaf(o[i][h].x, w, v[4 * h]), v[4 * h + 1] = fmaf(o[i][h].y, w, v[4 * h + 1]);
        v[4 * h + 2] = fmaf(o[i][h].z, w, v[4 * h + 2]), v[4 * h + 3] = fmaf(o[i][h].w, w, v[4 * h + 3]);
      }
    }
  }
  const KvpJoin j = kvp_join(m, l, p.s.own_lse[at.own]);
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] *= j.x;
  kvp_write8(p, at, block, v, j.y);
  if (block == 0 && p.s.lse) p.s.lse[at.own] = j.lse;
}

static __device__ __noinline__ void kvp_put_part(uint32_t o_col, bool live, float m, float l, float* part, int r) {
  __stcg(reinterpret_cast<float2*>(part) + r, make_float2(m, l));
#pragma unroll 1
  for (int c = 0; c < 4; ++c) {
    float v[32];
    __syncwarp();
    tmem_ld32(o_col + c * 32, v);
    if (!live) continue;
#pragma unroll
    for (int i = 0; i < 8; ++i)
      __stcg(reinterpret_cast<float4*>(part + 256) + (c * 8 + i) * 128 + r, make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]));
  }
}

__global__ void __launch_bounds__(kKvpThreads, 1) kv4_prefix_kernel(const __grid_constant__ Kv4PrefixParams p) {
  extern __shared__ uint8_t raw[];
  uint8_t* smem = raw + ((1024 - (smem_u32(raw) & 1023)) & 1023);
  KvpSmem& sm = *reinterpret_cast<KvpSmem*>(smem);
  uint8_t* Qs = smem + kKvpHeader;
  uint8_t* Ks = Qs + 2 * kPkTileBytes;                       // s' c, then s'' c
  uint8_t* Vs = Ks + 2 * kPkTileBytes;                       // two stages
  uint8_t* Qm = Vs + 2 * kPkTileBytes;                       // sums of the queries, two tiles
  uint8_t* Km = Qm + 2 * kKvpSumBytes;                       // m
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  volatile int* abort = &sm.abort;
  if (tid == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&sm.q_full[i], 4);
      mbar_init(&sm.v_full[i], 8);
      mbar_init(&sm.v_empty[i], 1);
      mbar_init(&sm.s_full[i], 1);
      mbar_init(&sm.p_most[i], 4);
      mbar_init(&sm.p_full[i], 4);
      mbar_init(&sm.o_full[i], 1);
    }
    mbar_init(&sm.k_full, 8);
    mbar_init(&sm.k_empty, 1);
    mbar_init(&sm.mma_done, 1);
    sm.abort = 0;
    fence_mbar_init();
  }
  if (warp == 8) {
    tmem_alloc(&sm.tmem, 512);
    tmem_relinquish();
  }
  const KvpCut cut = kvp_cut(p);
  const int length = cut.length, steps = cut.steps, splits = cut.splits;
  if (tid == 0 && *p.length > p.width << p.pool.page_shift) record_error(p.pool.err, kDevBadPosition);
  const int pieces = p.pool.heads * p.blocks * splits;
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sm.tmem;
  const unsigned long long lim = p.wait_ns;
  const int halves = p.halves;
  bool ok = true;
  auto wait = [&](uint64_t* bar, uint32_t parity, int code) {
    ok = pk_wait_warp(bar, parity, abort, p.pool.err, code, lim);
    return ok;
  };
  // piece -> (KV head, range of steps, block of rows), blocks side by side: they read the same codes
  auto first_step = [&](int split) { return (int)((int64_t)steps * split / splits); };

  if (warp >= 8) {
    if (warp == 8) {
      // -------------------------------------------------------- matrix products
      auto uniform = [](uint32_t v) { return __shfl_sync(0xffffffffu, v, 0); };
      constexpr uint32_t IS = idesc_pf<__half>(false), IO = idesc_pf<__half>(true);
      const uint32_t q_lo = uniform(smem_u32(Qs)), k_lo = uniform(smem_u32(Ks)), v_lo = uniform(smem_u32(Vs)), tm = uniform(tmem);
      uint32_t g = 0, round = 0, ps[2] = {0, 0};            // steps and pieces so far
      const uint32_t qm_lo = uniform(smem_u32(Qm)), km_lo = uniform(smem_u32(Km));
      auto scores = [&](uint32_t x) {
        const uint64_t a = smem_desc_sw128(q_lo + x * kPkTileBytes, 16, 1024), b = smem_desc_sw128(k_lo, 16, 1024);
#pragma unroll
        for (int part = 0; part < 2; ++part)
#pragma unroll
          for (int kk = 0; kk < 8; ++kk) {
            const uint64_t off = ((kk >> 2) * (kPkTileBytes / 2) + (kk & 3) * 32) >> 4;
            mma_f16_ss(tm + x * 256, a + off, b + off + part * (kPkTileBytes >> 4), IS, part + kk > 0);
          }
        mma_f16_ss(tm + x * 256, smem_desc(qm_lo + x * kKvpSumBytes, 128, 256), smem_desc(km_lo, 128, 256), IS, 1);
        mma_commit(&sm.s_full[x]);
      };
      auto values = [&](uint32_t x, auto rest, uint32_t stage, bool held) {
        const uint64_t b = smem_desc_sw128(v_lo + stage * kPkTileBytes, kPkTileBytes / 2, 1024);
#pragma unroll
        for (int kk = rest ? kPkMost / 16 : 0; kk < (rest ? 8 : kPkMost / 16); ++kk)
          mma_f16_ts(tm + x * 256 + 128, tm + x * 256 + kk * 8, b + ((kk * 2048) >> 4), IO, held || kk > 0);
      };
      for (int piece = blockIdx.x; ok && piece < pieces; piece += gridDim.x, ++round) {
        const int split = piece / p.blocks % splits, n = first_step(split + 1) - first_step(split);
        const int ahead = halves ? 2 : 1;                   // a tile's next step
        if (n == 0) continue;                               // an empty prefix: no piece has a step
        for (int x = 0; ok && x < 2; ++x) wait(&sm.q_full[x], round & 1, kDevWaitCopy);
        if (!ok) break;
        // step u of the piece is step g + u of all; with halves tile u & 1 takes it, else both do
        for (int u = 0; ok && u < min(ahead, n); ++u) {
          if (!wait(&sm.k_full, (g + u) & 1, kDevWaitCopy)) break;
          tc_fence_after();
          if (elect_one()) {
            if (!halves || u == 0) scores(0);
            if (!halves || u == 1) scores(1);
            mma_commit(&sm.k_empty);
          }
          __syncwarp();
        }
        for (int u = 0; ok && u < n; ++u) {
          const uint32_t st = (g + u) & 1;
          if (!wait(&sm.v_full[st], (g + u) >> 1 & 1, kDevWaitCopy)) break;
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            if (halves && (u & 1) != x) continue;
            if (!wait(&sm.p_most[x], ps[x] & 1, kDevWaitMma)) break;
            tc_fence_after();
            if (elect_one()) values(x, std::false_type(), st, u >= ahead);
            __syncwarp();
            if (!wait(&sm.p_full[x], ps[x] & 1, kDevWaitMma)) break;
            ++ps[x];
            tc_fence_after();
            if (elect_one()) {
              values(x, std::true_type(), st, true);
              if (u + ahead >= n) mma_commit(&sm.o_full[x]);
              if (halves || x == 1) mma_commit(&sm.v_empty[st]);
            }
            __syncwarp();
            if (u + ahead < n) {
              if ((halves || x == 0) && !wait(&sm.k_full, (g + u + ahead) & 1, kDevWaitCopy)) break;
              tc_fence_after();
              if (elect_one()) {
                scores(x);
                if (halves || x == 1) mma_commit(&sm.k_empty);
              }
              __syncwarp();
            }
          }
        }
        g += n;
      }
      if (elect_one()) mma_commit(&sm.mma_done);
      __syncwarp();
      mbar_wait(&sm.mma_done, 0, lim);
    } else if (warp < 25) {
      // -------------------------------------------------------- codes to operands
      // the keys (warps 9-16) or the values (17-24) of one tile of 16 tokens in eight, every step.  While
      // one is turned the next one's codes are on their way, and the page of the one after.
      const int i = (warp - 9) & 7;
      const bool keys = warp < 17;
      uint32_t g = 0;                                       // steps of the pieces before
      for (int piece = blockIdx.x; ok && piece < pieces; piece += gridDim.x) {
        const int split = piece / p.blocks % splits, kvh = piece / p.blocks / splits;
        const int u0 = first_step(split), n = first_step(split + 1) - u0;
        const int order = p.pool.page_shift - 4;
        const uint8_t* const codes = p.pool.data + (int64_t)kvh * p.pool.page_tiles * kKv4TileBytes;
        const int64_t page_bytes = (int64_t)p.pool.heads * p.pool.page_tiles * kKv4TileBytes;
        // step u's page as the table has it, read a step ahead
        auto there = [&](int u) { return u < n && ((u0 + u) * 8 + i) * 16 < length; };
        auto entry = [&](int u) { return there(u) ? __ldg(p.table + (((u0 + u) * 8 + i) >> order)) : 0; };
        int later = entry(0);
#pragma unroll 1
        for (int u = 0; u < n; ++u) {
          const int page = later;
          const bool good = there(u) && (unsigned)page < (unsigned)p.pool.num_pages, skip = there(u) && !good;
          KvpRaw raw;
          if (good) raw.load(codes + page * page_bytes + (((u0 + u) * 8 + i) & (p.pool.page_tiles - 1)) * kKv4TileBytes, keys, lane);
          later = entry(u + 1);
          const int left = good ? length - ((u0 + u) * 8 + i) * 16 : 0;
          if (skip && lane == 0) record_error(p.pool.err, kDevBadPage);
          // one place for keys (they are turned while the rows work on the step before), two for values
          const uint32_t step = g + u, st = step & 1;
          if (keys) {
            if (step >= 1 && !wait(&sm.k_empty, (step + 1) & 1, kDevWaitMma)) break;
            if (lane == 0) reinterpret_cast<volatile uint8_t*>(&sm.skip[step & 3])[i] = skip;
            kvp_keys(raw, Ks, Km, i * 16, left, lane);
          } else {
            if (step >= 2 && !wait(&sm.v_empty[st], (step >> 1) + 1 & 1, kDevWaitMma)) break;
            kvp_vals(raw, Vs + st * kPkTileBytes, i * 16, left, lane);
          }
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0 && (keys || i || blockIdx.x || (int)step != p.skip_step)) mbar_arrive(keys ? &sm.k_full : &sm.v_full[st]);
        }
        g += n;
      }
    }
  } else {
    // ------------------------------------------------------------ a thread a row
    const int x = warp >> 2, r = tid & 127;
    const uint32_t sa = tmem + x * 256 + ((uint32_t)((warp & 3) * 32) << 16);
    uint32_t g = 0, ss = 0, os = 0;
    auto arrive = [&](uint64_t* bar) {
      __syncwarp();
      if (lane == 0) mbar_arrive(bar);
    };
    for (int piece = blockIdx.x; ok && piece < pieces; piece += gridDim.x) {
      const int split = piece / p.blocks % splits, kvh = piece / p.blocks / splits, block = piece % p.blocks;
      const int u0 = first_step(split), n = first_step(split + 1) - u0;
      const int row_id = block * 256 + (halves ? 0 : x * 128) + r;
      PkRow row = {-INFINITY, 0.f, false};
      // Queries are laid out for products only: without a step nothing holds the rows back, and a tile's
      // would arrive for their next piece while the issuer still waits for the other tile's first.
      if (n > 0) {
        const KvpRow at = kvp_row(p, kvh, row_id);
        const int k = kvp_query(p.s.q, p.s.q_dtype, at.q, at.live, Qs + x * kPkTileBytes, Qm + x * kKvpSumBytes, r);
        fence_proxy_async_smem();
        arrive(&sm.q_full[x]);
        const float sl2 = fmaxf(ldexpf(p.scale_log2, k), 1.17549435e-38f);   // not 0: hidden scores are -inf times it
        bool held = false;
        for (int u = halves ? x : 0; u < n; u += halves ? 2 : 1) {
          if (!wait(&sm.s_full[x], ss & 1, kDevWaitMma)) break;
          ++ss;
          tc_fence_after();
          const int seen = length - (u0 + u) * kPkKeys;
          uint64_t skip = *reinterpret_cast<const volatile uint64_t*>(&sm.skip[(g + u) & 3]);
          kvp_softmax(sa, sl2, seen, held, row, &sm.p_most[x], skip);
          held = true;
          tc_fence_before();
          arrive(&sm.p_full[x]);
        }
        if (!ok) break;
        if (held) {
          if (!wait(&sm.o_full[x], os & 1, kDevWaitMma)) break;
          ++os;
          tc_fence_after();
        }
      }
      g += n;
      if (row.bad) row.m = 0.f, row.l = NAN;
      const KvpRow at = kvp_row(p, kvh, row_id);
      const int item = kvh * p.blocks + block;
      if (cut.parts == 1) {
        kvp_finish(p, at, sa + 128, row.m, row.l);
        continue;
      }
      // parts of a row lie one after another: of an item's tile, or of both
      const int64_t first = (int64_t)(halves ? item : item * 2 + x) * cut.parts;
      kvp_put_part(sa + 128, at.live, row.m, row.l, p.parts + (first + (halves ? 2 * split + x : split)) * kPkTilePart, r);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 8) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

}  // namespace starkv
