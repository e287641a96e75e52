// packed_attn.cuh — attention of packed sequences of different lengths on the tensor cores.
//
// Sequence b: queries q_start[b] .. q_end[b] - 1 (rows of q), keys and values k_start[b] ..
// k_end[b] - 1 (rows of k and v), the newest query on the newest key.  One pass with a running
// reference m per row: with s = scaling * log2(e) * q.k, p = 2^(s - m), out = sum p v / sum p,
// lse = ln 2 (m + log2 sum p).
//
// Rows.  A KV head's query heads share its keys, so a row is (token, head of the group): a tile
// has 128 / group tokens, and the masked part of a causal tile shrinks with it.  Keys and values
// cross from the L2 once for 256 rows (two tiles a CTA).
//
// CTA, one an SM, 12 warps:
//   warp 9     takes pieces of work from a counter, loads Q, K and V tiles by TMA (128-byte
//              swizzle; K-major for Q and K, MN-major for V) into a ring of four;
//   warp 8     issues the matrix products: S_x = Q_x K^T, O_x += P_x V for tiles x = 0, 1 in turn, so
//              that one tile's softmax runs under the other's products; S_x(j + 1) is issued right
//              behind P_x(j) V(j), in the columns that P_x(j) held;
//   warps 0-3 and 4-7, a thread a row of tile 0 and 1: maximum, weights, sum in fp32 registers;
//              P goes back over S as 16-bit operands.  m moves only when a row's maximum has
//              grown by 2^kPkLazy, then O is scaled in tensor memory;
//   warps 10-11 look over the value tiles at the border of what is visible: rows of other
//              sequences become 0, and values that are not finite become 0 and are added again
//              at the end, by the rows that see them (0 * NaN would reach all the others).
// Work.  A piece is a pair of tiles of one (sequence, KV head), and where there are too few for
// the SMs a range of its keys; a second kernel joins such parts in order (the same result every
// time).  Lengths are read on the GPU: each CTA works out the same table.
#pragma once
#include <cuda.h>

#include "kv4.cuh"
#include "prefill.cuh"

namespace starkv {

constexpr int kPkKeys = 128;                     // keys of a step
constexpr int kPkTileBytes = 128 * 128 * 2;
constexpr int kPkStages = 4;                     // K, V, K, V
constexpr int kPkItems = 4;                      // pieces ahead
constexpr int kPkRowWarps = 8;                   // four a tile
constexpr int kPkThreads = (kPkRowWarps + 4) * 32;
// Registers of a thread of the row warps and of the other four; the sum of the three warpgroups' is at
// most the CTA's at launch, three times 168.
constexpr int kPkRowRegs = 208, kPkRoleRegs = 88, kPkLaunchRegs = 168;
static_assert(2 * kPkRowRegs + kPkRoleRegs <= 3 * kPkLaunchRegs, "register shares");
constexpr int kPkEntries = 1024;                 // entries of the table of sequences
constexpr int kPkSorted = 256;                   // up to so many sequences the longest go first
constexpr int kPkMaxSlots = 320;                 // partial sums that the workspace holds
constexpr int kPkCounters = 1024;                // ints that are zero between calls: work, done
// per tile: m and l of each row, then its 128 values of O, four at a time
constexpr int kPkTilePart = 128 * (2 + 128);
constexpr int kPkPartFloats = 2 * kPkTilePart;
constexpr int kPkMaxCut = kPkMaxSlots / 2;       // cut pairs: each has two slots at least
constexpr int kPkMinPiece = 4;                   // key tiles
constexpr int kPkMost = 64;                     // keys whose weights go to the products ahead of the rest
constexpr float kPkMaxThreadPieces = 5e6f;       // that a thread counts for the table of sequences
static_assert(kPkMaxThreadPieces * kPkThreads < 2147483648.f, "the sum over threads");
constexpr int kPkTooMany = 0x7fffffff;           // more: in the place of the longest sequence, which is below 2^30
constexpr float kPkLazy = 5.f;
// p is up to 2^(kPkBias + kPkLazy): the least fp16 weight is 2^-34 of the largest then.
constexpr float kPkBias = 10.f;
constexpr int kDevBadRange = 0x203;              // a range of rows outside the tensors

// A pair of tiles whose keys were cut, for the kernel that joins the parts.
struct PkCut {
  int q_row, tok0, q_len, kvh, slot, splits, unused[2];
};
struct PkCuts {
  int count, unused[7];
  PkCut cut[kPkMaxCut];
};
constexpr size_t kPkCutsAt = kPkCounters * sizeof(int), kPkPartsAt = kPkCutsAt + (sizeof(PkCuts) + 255) / 256 * 256;
constexpr size_t kPkWorkspaceBytes = kPkPartsAt + (size_t)kPkMaxSlots * kPkPartFloats * sizeof(float);

struct PackedParams {
  const int *q_start, *q_end, *k_start, *k_end;
  const void* v;
  void* out;
  float* lse;
  int64_t vs[2], os[2];                          // elements: row, head
  int total_q, total_k;
  int batch, q_heads, kv_heads, group, tokens;   // tokens of a tile
  int causal, out_dtype;
  float scale_log2;
  int* err;
  unsigned long long wait_ns;
  int skip_copy;                                 // tests: the first CTA's K or V tile that is withheld, or -1
  int* counters;
  PkCuts* cuts;
  float* parts;
};

struct PkItem {
  int kvh, q_row, tok0, q_len, k_row, k_len, first, n[2], splits, split, slot, valid;
  int poison;
};

struct PkSeq {
  int q0, qn, k0, kn;
};

struct PkSmem {
  uint64_t q_full, q_empty, kv_full[kPkStages], kv_empty[kPkStages], v_ok[2], s_full[2], p_most[2], p_full[2], o_full[2],
      item_full[kPkItems], item_empty[kPkItems], mma_done;
  uint32_t tmem;
  int abort;
  int last;
  int pieces, limit;                             // totals; key tiles of a piece at most
  int scan[kPkThreads / 32][5];
  PkItem item[kPkItems];
  int pre[kPkEntries], slot_pre[kPkEntries], counter_pre[kPkEntries];
  PkSeq seq[kPkSorted];
};
constexpr int kPkHeader = 18432;
static_assert(sizeof(PkSmem) <= kPkHeader, "header");
constexpr size_t kPkSmemBytes = kPkHeader + 1024 + (2 + kPkStages) * (size_t)kPkTileBytes;
static_assert(kPkSmemBytes <= 227 * 1024, "shared memory of one SM");

__device__ __forceinline__ PkSeq pk_seq(const PackedParams& p, int b) {
  const int q0 = p.q_start[b], q1 = p.q_end[b], k0 = p.k_start[b], k1 = p.k_end[b];
  // ends are held within the tensors before any difference is taken: one far below zero would wrap around
  PkSeq s;
  s.q0 = min(max(q0, 0), p.total_q);
  s.k0 = min(max(k0, 0), p.total_k);
  const int qe = min(max(q1, s.q0), p.total_q), ke = min(max(k1, s.k0), p.total_k);
  s.qn = qe - s.q0;
  s.kn = ke - s.k0;
  if (s.q0 != q0 || s.k0 != k0 || qe != q1 || ke != k1) record_error(p.err, kDevBadRange);
  return s;
}

// Keys that the first `upto` queries of a sequence see, together.
__device__ __forceinline__ int pk_visible(const PackedParams& p, const PkSeq& s, int upto) {
  return p.causal ? max(min(s.kn, s.kn - s.qn + upto), 0) : s.kn;
}

struct PkShape {
  int tiles, live, splits;                       // pairs of tiles; those with a key to see; pieces of each
  float units;                                   // key tiles, about
};
__device__ __forceinline__ PkShape pk_shape(const PackedParams& p, const PkSeq& s, int limit) {
  const int w = 2 * p.tokens;
  PkShape r;
  r.tiles = (s.qn + w - 1) / w;
  const int idle = s.kn == 0 ? r.tiles : p.causal && s.qn > s.kn ? (s.qn - s.kn) / w : 0;
  r.live = r.tiles - idle;
  const int most = (s.kn + kPkKeys - 1) / kPkKeys;
  r.splits = r.live && limit ? (most + limit - 1) / limit : 1;
  if (r.splits < 1) r.splits = 1;
  const int least = r.live ? (pk_visible(p, s, min((idle + 1) * w, s.qn)) + kPkKeys - 1) / kPkKeys : 0;
  r.units = 0.5f * r.live * (least + most);
  return r;
}

__device__ __forceinline__ float pk_max3_nan(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

__device__ __forceinline__ void tma_load_3d(void* dst, const CUtensorMap* map, int c0, int c1, int c2, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(
          smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(c2), "r"(smem_u32(bar))
      : "memory");
}

__device__ __forceinline__ bool elect_one() {
  uint32_t pred;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(pred));
  return pred != 0;
}

// Bounded wait that ends early when another role has given up.
__device__ __forceinline__ bool pk_wait(uint64_t* bar, uint32_t parity, volatile int* abort, int* err, int code,
                                        unsigned long long limit) {
  if (__builtin_expect(mbar_try_wait_plain(bar, parity), 1)) return true;
  const unsigned long long t0 = global_timer_ns();
#pragma unroll 1
  while (!mbar_try_wait_plain(bar, parity)) {
    if (*abort) return false;
    if (global_timer_ns() - t0 > limit) {
      record_error(err, code);
      *abort = 1;
      return false;
    }
  }
  return true;
}
// The same for a whole warp: all lanes go on, or none.
__device__ __forceinline__ bool pk_wait_warp(uint64_t* bar, uint32_t parity, volatile int* abort, int* err, int code,
                                             unsigned long long limit) {
  return __all_sync(0xffffffffu, pk_wait(bar, parity, abort, err, code, limit));
}

// All 128 columns of a row and the wait for them.
__device__ __forceinline__ void pk_load128(uint32_t taddr, float* v) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x128.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,"
      "%32,%33,%34,%35,%36,%37,%38,%39,%40,%41,%42,%43,%44,%45,%46,%47,"
      "%48,%49,%50,%51,%52,%53,%54,%55,%56,%57,%58,%59,%60,%61,%62,%63,"
      "%64,%65,%66,%67,%68,%69,%70,%71,%72,%73,%74,%75,%76,%77,%78,%79,"
      "%80,%81,%82,%83,%84,%85,%86,%87,%88,%89,%90,%91,%92,%93,%94,%95,"
      "%96,%97,%98,%99,%100,%101,%102,%103,%104,%105,%106,%107,%108,%109,%110,%111,"
      "%112,%113,%114,%115,%116,%117,%118,%119,%120,%121,%122,%123,%124,%125,%126,%127}, [%128];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]),
        "=f"(v[8]), "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15]),
        "=f"(v[16]), "=f"(v[17]), "=f"(v[18]), "=f"(v[19]), "=f"(v[20]), "=f"(v[21]), "=f"(v[22]), "=f"(v[23]),
        "=f"(v[24]), "=f"(v[25]), "=f"(v[26]), "=f"(v[27]), "=f"(v[28]), "=f"(v[29]), "=f"(v[30]), "=f"(v[31]),
        "=f"(v[32]), "=f"(v[33]), "=f"(v[34]), "=f"(v[35]), "=f"(v[36]), "=f"(v[37]), "=f"(v[38]), "=f"(v[39]),
        "=f"(v[40]), "=f"(v[41]), "=f"(v[42]), "=f"(v[43]), "=f"(v[44]), "=f"(v[45]), "=f"(v[46]), "=f"(v[47]),
        "=f"(v[48]), "=f"(v[49]), "=f"(v[50]), "=f"(v[51]), "=f"(v[52]), "=f"(v[53]), "=f"(v[54]), "=f"(v[55]),
        "=f"(v[56]), "=f"(v[57]), "=f"(v[58]), "=f"(v[59]), "=f"(v[60]), "=f"(v[61]), "=f"(v[62]), "=f"(v[63]),
        "=f"(v[64]), "=f"(v[65]), "=f"(v[66]), "=f"(v[67]), "=f"(v[68]), "=f"(v[69]), "=f"(v[70]), "=f"(v[71]),
        "=f"(v[72]), "=f"(v[73]), "=f"(v[74]), "=f"(v[75]), "=f"(v[76]), "=f"(v[77]), "=f"(v[78]), "=f"(v[79]),
        "=f"(v[80]), "=f"(v[81]), "=f"(v[82]), "=f"(v[83]), "=f"(v[84]), "=f"(v[85]), "=f"(v[86]), "=f"(v[87]),
        "=f"(v[88]), "=f"(v[89]), "=f"(v[90]), "=f"(v[91]), "=f"(v[92]), "=f"(v[93]), "=f"(v[94]), "=f"(v[95]),
        "=f"(v[96]), "=f"(v[97]), "=f"(v[98]), "=f"(v[99]), "=f"(v[100]), "=f"(v[101]), "=f"(v[102]), "=f"(v[103]),
        "=f"(v[104]), "=f"(v[105]), "=f"(v[106]), "=f"(v[107]), "=f"(v[108]), "=f"(v[109]), "=f"(v[110]), "=f"(v[111]),
        "=f"(v[112]), "=f"(v[113]), "=f"(v[114]), "=f"(v[115]), "=f"(v[116]), "=f"(v[117]), "=f"(v[118]), "=f"(v[119]),
        "=f"(v[120]), "=f"(v[121]), "=f"(v[122]), "=f"(v[123]), "=f"(v[124]), "=f"(v[125]), "=f"(v[126]), "=f"(v[127])
      : "r"(taddr)
      : "memory");
}

// 64 columns of sixteen rows (the low or the high half of the warp's 32), four lanes a row.
__device__ __forceinline__ void pk_load16x64(uint32_t taddr, float* v) {
  asm volatile(
      "tcgen05.ld.sync.aligned.16x256b.x8.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]),
        "=f"(v[8]), "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15]),
        "=f"(v[16]), "=f"(v[17]), "=f"(v[18]), "=f"(v[19]), "=f"(v[20]), "=f"(v[21]), "=f"(v[22]), "=f"(v[23]),
        "=f"(v[24]), "=f"(v[25]), "=f"(v[26]), "=f"(v[27]), "=f"(v[28]), "=f"(v[29]), "=f"(v[30]), "=f"(v[31])
      : "r"(taddr)
      : "memory");
}

// A row's state: reference m (log2 domain, -inf before the first visible key), sum of weights,
// and whether a score was NaN or +inf.
struct PkRow {
  float m, l;
  bool bad;
};

// One key tile of a row: S (128 columns of tensor memory at sa) to weights P over it; in a border tile
// `seen` keys are visible.  The row's O columns are scaled where m moves (held: O has sums already).
// The weights of the first kPkMost keys are announced on `most`, while those of the others are on
// their way (a store into tensor memory takes some 450 cycles to settle).
template <typename T>
__device__ __forceinline__ void pk_softmax(uint32_t sa, float sl2, bool border, int seen, bool held, PkRow& row, uint64_t* most) {
  float s[128];
  pk_load128(sa, s);
  if (border) {
#pragma unroll
    for (int i = 0; i < 128; ++i) s[i] = i < seen ? s[i] : -INFINITY;
  }
  float mq[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) mq[i] = kv4_max_nan(s[2 * i], s[2 * i + 1]);
#pragma unroll
  for (int i = 16; i < 128; i += 2) mq[i / 2 & 7] = pk_max3_nan(mq[i / 2 & 7], s[i], s[i + 1]);
  const float mt = pk_max3_nan(pk_max3_nan(mq[0], mq[1], mq[2]), pk_max3_nan(mq[3], mq[4], mq[5]), kv4_max_nan(mq[6], mq[7])) * sl2;
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
#pragma unroll
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
  if (__any_sync(0xffffffffu, fabsf(mt) > 65536.f && fabsf(mt) < INFINITY)) {
#pragma unroll
    for (int i = 0; i < 128; ++i) s[i] *= sl2;
    sl2 = 1.f;
  }
  const float base = row.m == -INFINITY ? 0.f : -row.m;
  float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    uint32_t pk[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int at = c * 32 + 2 * i;
      const float2 x = __ffma2_rn(make_float2(s[at], s[at + 1]), make_float2(sl2, sl2), make_float2(base, base));
      const float2 e = make_float2(fast_exp2(x.x), fast_exp2(x.y));
      sum[i & 1] = __fadd2_rn(sum[i & 1], e);
      pk[i] = pack2<T>(e.x, e.y);
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

// Where a thread's row of a tile goes.
struct PkPlace {
  int64_t q_row;
  int head;
  bool live;
};

__device__ __forceinline__ void pk_write_lse(const PackedParams& p, const PkPlace& at, float m, float l) {
  if (at.live && p.lse) p.lse[at.q_row * p.q_heads + at.head] = m == -INFINITY ? -INFINITY : (m + log2f(l)) * 0.6931471805599453f;
}

// 32 channels of a row's sums in tensor memory, with the values that are not finite: those of the
// visible keys from border0 on.
template <typename T>
__device__ __forceinline__ void pk_sums(const PackedParams& p, const PkItem& it, const PkPlace& at, uint32_t o_col, int c, int border0,
                                        int upto, float* v) {
  __syncwarp();
  tmem_ld32(o_col + c * 32, v);
  if (!at.live) return;
#pragma unroll 1
  for (int key = border0; key < upto; ++key) {
    const T* src = reinterpret_cast<const T*>(p.v) + ((int64_t)it.k_row + key) * p.vs[0] + it.kvh * p.vs[1] + c * 32;
#pragma unroll
    for (int i = 0; i < 32; ++i) {
      const float y = to_f32(src[i]);
      if (!(fabsf(y) < INFINITY)) v[i] += y;
    }
  }
}

// What pk_load16x64 gave, rounded and written to rows dst[0] and dst[1] (where not negative).  Of every
// eight columns a lane holds two; an exchange among the row's four lanes gives each eight that follow
// one another: lane k has pair k of four blocks and takes all of block k.
template <typename U>
__device__ __forceinline__ void pk_store16x64(void* base, const int64_t* dst, int c, const float* v) {
  const int lane = threadIdx.x & 31;
  uint32_t w[4][4];                                    // [row, 32 channels][block]
#pragma unroll
  for (int j = 0; j < 4; ++j)
#pragma unroll
    for (int i = 0; i < 4; ++i) w[j][i] = pack2<U>(v[16 * (j >> 1) + 4 * i + 2 * (j & 1)], v[16 * (j >> 1) + 4 * i + 2 * (j & 1) + 1]);
#pragma unroll
  for (int o = 1; o < 4; o <<= 1) {
    const bool up = lane & o;
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (i & o) continue;
        const uint32_t got = __shfl_xor_sync(0xffffffffu, up ? w[j][i] : w[j][i | o], o);
        w[j][i] = up ? got : w[j][i];
        w[j][i | o] = up ? w[j][i | o] : got;
      }
  }
#pragma unroll
  for (int j = 0; j < 4; ++j)
    if (dst[j & 1] >= 0)
      *reinterpret_cast<uint4*>(reinterpret_cast<U*>(base) + dst[j & 1] + c + 32 * (j >> 1) + 8 * (lane & 3)) =
          make_uint4(w[j][0], w[j][1], w[j][2], w[j][3]);
}

// Whole rows of a warp: out = O / l.  Sixteen rows at a time, four lanes a row: lane l holds rows l / 4
// (the first two values of four) and l / 4 + 8, so that a store writes 64 bytes in eight places (16 in
// 32 with a lane a row).  About 5600 cycles for a pair of tiles, in which no products run: what most
// of the gap to the floor is where a piece has few key tiles (24 mixed prompts, in a graph: 246 us; 262
// with a lane's conversions to both types and exchanges of one row after the other).  Values that are not
// finite are added first, a lane a row, into tensor memory (the 0 that stands for them made them 0).
template <typename T>
__device__ __noinline__ void pk_finish(const PackedParams& p, const PkItem& it, PkPlace at, uint32_t o_col, int nx, int border0, int upto,
                                       float m, float l) {
  const int lane = threadIdx.x & 31;
  const bool none = m == -INFINITY;
  const float f = none ? 0.f : 1.f / l;
  pk_write_lse(p, at, m, l);
  if (nx > 0 && __any_sync(0xffffffffu, upto > 0)) {
#pragma unroll 1
    for (int c = 0; c < 4; ++c) {
      float v[32];
      pk_sums<T>(p, it, at, o_col, c, border0, upto, v);
      __syncwarp();
      uint32_t w[32];
#pragma unroll
      for (int i = 0; i < 32; ++i) w[i] = __float_as_uint(v[i]);
      tmem_st32(o_col + c * 32, w);
    }
    tmem_st_wait();
  }
  const int64_t to = at.live ? at.q_row * p.os[0] + at.head * p.os[1] : -1;
  // read once: the loads below are ordered with everything else that touches memory
  const int type = p.out_dtype;
  void* const base = p.out;
  const bool clear = __any_sync(0xffffffffu, at.live && none);                     // rows that saw nothing
#pragma unroll 1
  for (int h = 0; h < 2; ++h) {
    float g[2];
    int64_t dst[2];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const int row = h * 16 + (lane >> 2) + 8 * r;
      g[r] = __shfl_sync(0xffffffffu, none ? -1.f : f, row);
      dst[r] = __shfl_sync(0xffffffffu, to, row);
    }
#pragma unroll 1
    for (int c = 0; c < 128; c += 64) {
      float v[32];
      __syncwarp();
      if (nx > 0) pk_load16x64(o_col + ((uint32_t)h << 20) + c, v);
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const float2 x = __fmul2_rn(make_float2(v[2 * i], v[2 * i + 1]), make_float2(g[i & 1], g[i & 1]));
        v[2 * i] = x.x, v[2 * i + 1] = x.y;
      }
      if (clear) {
#pragma unroll
        for (int i = 0; i < 32; ++i) v[i] = g[i >> 1 & 1] == -1.f ? 0.f : v[i];
      }
      if (type == STARKV_F32) {
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          if (dst[r] < 0) continue;
          float* d = reinterpret_cast<float*>(base) + dst[r] + c + 2 * (lane & 3);
#pragma unroll
          for (int i = 0; i < 8; ++i) *reinterpret_cast<float2*>(d + 8 * i) = make_float2(v[4 * i + 2 * r], v[4 * i + 2 * r + 1]);
        }
        continue;
      }
      if (type == STARKV_BF16) pk_store16x64<__nv_bfloat16>(base, dst, c, v);
      else pk_store16x64<__half>(base, dst, c, v);
    }
  }
}

// A row's sums over a part of its keys, to the workspace: m and l, then O, four channels of all
// rows after another.
template <typename T>
__device__ __noinline__ void pk_put_part(const PackedParams& p, const PkItem& it, PkPlace at, uint32_t o_col, int nx, int border0, int upto,
                                         float m, float l, float* part, int r) {
  __stcg(reinterpret_cast<float2*>(part) + r, make_float2(m, l));
#pragma unroll 1
  for (int c = 0; nx > 0 && c < 4; ++c) {
    float v[32];
    pk_sums<T>(p, it, at, o_col, c, border0, upto, v);
    if (!at.live) continue;
#pragma unroll
    for (int i = 0; i < 8; ++i)
      __stcg(reinterpret_cast<float4*>(part + 256) + (c * 8 + i) * 128 + r, make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]));
  }
}

// The parts of rows whose keys were cut, in order: out = sum 2^(m_k - m) O_k / sum 2^(m_k - m) l_k.  A
// CTA takes eight channels of a tile's 128 rows at a time, a thread a row, so that parts are read in
// lines and by all SMs (the last arriver of a pair alone, 1.8 MB: 18 us).
// kAhead parts are read before the first is used.
template <int kAhead>
__global__ void __launch_bounds__(128) packed_join_kernel(const __grid_constant__ PackedParams p) {
  const int count = min(p.cuts->count, kPkMaxCut), r = threadIdx.x, tok_in = r / p.group;
  if (tok_in >= p.tokens) return;
  for (int unit = blockIdx.x; unit < count * 32; unit += gridDim.x) {
    const PkCut cut = p.cuts->cut[unit >> 5];
    const int x = unit >> 4 & 1, block = unit & 15, tok = cut.tok0 + x * p.tokens + tok_in;
    // a piece that was given up (a wait ran out) leaves an earlier call's entry here: nothing of it may
    // reach outside this call's tensors
    if (cut.splits < 2 || tok >= cut.q_len || (unsigned)(cut.q_row + tok) >= (unsigned)p.total_q ||
        (unsigned)cut.kvh >= (unsigned)p.kv_heads || (unsigned)cut.slot >= kPkMaxSlots || cut.splits > kPkMaxSlots - cut.slot)
      continue;
    const float* parts = p.parts + (int64_t)cut.slot * kPkPartFloats + x * kPkTilePart;
    float m = -INFINITY, l = 0.f, v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = 0.f;
#pragma unroll 1
    for (int k0 = 0; k0 < cut.splits; k0 += kAhead) {
      float2 a[kAhead];
      float4 o[kAhead][2];
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        const float* one = parts + (int64_t)min(k0 + i, cut.splits - 1) * kPkPartFloats;
        a[i] = __ldcg(reinterpret_cast<const float2*>(one) + r);
        if (k0 + i >= cut.splits) a[i].x = -INFINITY;
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
        if (a[i].x == -INFINITY) continue;                             // what such a part holds of O is not set
        const float w = fast_exp2(a[i].x - m);
        l = fmaf(w, a[i].y, l);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          v[4 * h] = fmaf(o[i][h].x, w, v[4 * h]), v[4 * h + 1] = fmaf(o[i][h].y, w, v[4 * h + 1]);
          v[4 * h + 2] = fmaf(o[i][h].z, w, v[4 * h + 2]), v[4 * h + 3] = fmaf(o[i][h].w, w, v[4 * h + 3]);
        }
      }
    }
    const float f = m == -INFINITY ? 0.f : 1.f / l;
    const PkPlace at = {(int64_t)cut.q_row + tok, cut.kvh * p.group + r - tok_in * p.group, true};
    if (block == 0) pk_write_lse(p, at, m, l);
    const int64_t to = at.q_row * p.os[0] + at.head * p.os[1] + block * 8;
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] *= f;
    if (p.out_dtype == STARKV_F32) {
      float4* d = reinterpret_cast<float4*>(reinterpret_cast<float*>(p.out) + to);
      d[0] = make_float4(v[0], v[1], v[2], v[3]), d[1] = make_float4(v[4], v[5], v[6], v[7]);
    } else {
      uint32_t w[4];
#pragma unroll
      for (int k = 0; k < 4; ++k)
        w[k] = p.out_dtype == STARKV_BF16 ? pack2<__nv_bfloat16>(v[2 * k], v[2 * k + 1]) : pack2<__half>(v[2 * k], v[2 * k + 1]);
      *reinterpret_cast<uint4*>(reinterpret_cast<__half*>(p.out) + to) = make_uint4(w[0], w[1], w[2], w[3]);
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(kPkThreads, 1)
    packed_attn_kernel(const __grid_constant__ PackedParams p, const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                       const __grid_constant__ CUtensorMap tm_v) {
  extern __shared__ uint8_t raw[];
  // the swizzled tiles start on 1024 bytes
  uint8_t* smem = raw + ((1024 - (smem_u32(raw) & 1023)) & 1023);
  PkSmem& sm = *reinterpret_cast<PkSmem*>(smem);
  uint8_t* Qs = smem + kPkHeader;
  uint8_t* KVs = Qs + 2 * kPkTileBytes;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  volatile int* abort = &sm.abort;

  if (tid == 0) {
    mbar_init(&sm.q_full, 1);
    mbar_init(&sm.q_empty, 1);
    // a value tile is also released by the warps that look them over
    for (int i = 0; i < kPkStages; ++i) mbar_init(&sm.kv_full[i], 1), mbar_init(&sm.kv_empty[i], i & 1 ? 3 : 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&sm.v_ok[i], 2);
      mbar_init(&sm.s_full[i], 1);
      mbar_init(&sm.p_most[i], 4);
      mbar_init(&sm.p_full[i], 4);
      mbar_init(&sm.o_full[i], 1);
    }
    for (int i = 0; i < kPkItems; ++i) mbar_init(&sm.item_full[i], 1), mbar_init(&sm.item_empty[i], kPkRowWarps + 3);
    mbar_init(&sm.mma_done, 1);
    sm.abort = 0;
    fence_mbar_init();
  }
  if (warp == kPkRowWarps) {
    tmem_alloc(&sm.tmem, 512);
    tmem_relinquish();
  }

  // ------------------------------------------------ the table of sequences
  const int per_entry = (p.batch + kPkEntries - 1) / kPkEntries;
  const int entries = (p.batch + per_entry - 1) / per_entry;
  const bool sorted = p.batch <= kPkSorted;          // an entry a sequence, the longest first, with its ranges
  if (sorted) {
    PkSeq mine;
    if (tid < p.batch) {
      mine = pk_seq(p, tid);
      sm.pre[tid] = mine.qn ? mine.kn : -1;
    }
    __syncthreads();
    if (tid < p.batch) {
      const int length = sm.pre[tid];
      int rank = 0;
      for (int b = 0; b < p.batch; ++b) rank += sm.pre[b] > length || (sm.pre[b] == length && b < tid);
      sm.seq[rank] = mine;
    }
    __syncthreads();
  }
  // sequence i of an entry
  auto sequence = [&](int e, int i) { return sorted ? sm.seq[e] : pk_seq(p, e * per_entry + i); };
  auto in_entry = [&](int e) { return min(per_entry, p.batch - e * per_entry); };
  {
    const int per_thread = (entries + kPkThreads - 1) / kPkThreads;
    const int e0 = min(tid * per_thread, entries), e1 = min(e0 + per_thread, entries);
    // pieces, slots and counters of a thread's entries, with pieces of `limit` key tiles at most; key
    // tiles, about; then all threads' sums, and those before this one
    int s[3], before[3], most = 0;
    float units = 0.f;
    auto sums = [&](int limit) {
      s[0] = s[1] = s[2] = most = 0;
      units = 0.f;
      float all = 0.f;
      for (int e = e0; e < e1; ++e)
        for (int i = 0; i < in_entry(e); ++i) {
          const PkSeq q = sequence(e, i);
          const PkShape h = pk_shape(p, q, limit);
          s[0] += h.tiles * h.splits * p.kv_heads;
          all += (float)h.tiles * h.splits;
          if (h.splits > 1) s[1] += h.live * h.splits * p.kv_heads, s[2] += h.live * p.kv_heads;
          units += h.units * p.kv_heads;
          most = max(most, h.live ? q.kn : 0);
        }
      // A thread has this many pieces only where the same rows were given to many sequences (rows of
      // one sequence each would not fit a GPU's memory); up to there the sum of 384 threads has 31 bits.
      if (all * p.kv_heads > kPkMaxThreadPieces) most = kPkTooMany;
    };
    auto scan = [&]() {
#pragma unroll
      for (int k = 0; k < 3; ++k) {
        int x = s[k];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int y = __shfl_up_sync(0xffffffffu, x, o);
          if (lane >= o) x += y;
        }
        before[k] = x - s[k];
        if (lane == 31) sm.scan[warp][k] = x;
      }
#pragma unroll
      for (int o = 16; o; o >>= 1) units += __shfl_xor_sync(0xffffffffu, units, o);
      const int longest = __reduce_max_sync(0xffffffffu, most);
      if (lane == 0) sm.scan[warp][3] = __float_as_int(units), sm.scan[warp][4] = longest;
      __syncthreads();
      s[0] = s[1] = s[2] = 0;
      units = 0.f;
#pragma unroll
      for (int w = 0; w < kPkThreads / 32; ++w) {
#pragma unroll
        for (int k = 0; k < 3; ++k) {
          const int x = sm.scan[w][k];
          if (w < warp) before[k] += x;
          s[k] += x;
        }
        units += __int_as_float(sm.scan[w][3]);
        most = max(most, sm.scan[w][4]);
      }
      __syncthreads();
    };
    sums(0);
    scan();
    // pieces of half a CTA's share at most (four new pieces behind up to 16 K tokens and two single
    // tokens: 102 us with whole shares, 88 with two thirds, 84 with halves and thirds)
    int limit = max((int)fminf(units / (2.f * gridDim.x), 1e9f) + 1, kPkMinPiece);
    const bool crowded = most == kPkTooMany;
    if (!crowded && (most + kPkKeys - 1) / kPkKeys > limit)
      for (;;) {
        sums(limit);
        scan();
        if (s[1] <= kPkMaxSlots && most != kPkTooMany) break;
        // one piece each from 2^24 key tiles on, so this ends; at once where cuts of idle tiles are too many
        limit = most == kPkTooMany ? 1 << 28 : limit < (1 << 28) ? limit + limit / 4 + 1 : limit;
      }
    if (crowded) {                                     // nothing is done
      if (tid == 0) record_error(p.err, kDevBadRange);
      s[0] = s[2] = 0;
    }
    for (int e = crowded ? e1 : e0; e < e1; ++e) {
      sm.pre[e] = before[0], sm.slot_pre[e] = before[1], sm.counter_pre[e] = before[2];
      for (int i = 0; i < in_entry(e); ++i) {
        const PkShape h = pk_shape(p, sequence(e, i), limit);
        before[0] += h.tiles * h.splits * p.kv_heads;
        if (h.splits > 1) before[1] += h.live * h.splits * p.kv_heads, before[2] += h.live * p.kv_heads;
      }
    }
    if (tid == 0) sm.pieces = s[0], sm.limit = limit;
    if (tid == 0 && blockIdx.x == 0) p.cuts->count = s[2];
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sm.tmem;
  const unsigned long long lim = p.wait_ns;

  // Keys that queries up to `upto` of an item's sequence see.
  auto visible = [&](const PkItem& it, int upto) {
    return p.causal ? max(min(it.k_len, it.k_len - it.q_len + upto), 0) : it.k_len;
  };
  // Whether key tile j of the item holds keys that some row of the pair does not see.
  auto border = [&](const PkItem& it, int j) { return (it.first + j + 1) * kPkKeys > visible(it, it.tok0 + 1); };

  if (warp >= kPkRowWarps) {
    regs_dec<kPkRoleRegs>();
    if (warp == kPkRowWarps + 1) {
      // -------------------------------------------------------- pieces of work and loads
      if (lane == 0) {
        uint32_t items = 0, kv = 0, qs = 0;            // items, K / V tiles and Q pairs so far
        uint32_t piece = blockIdx.x;
        bool ok = true;
        while (ok) {
          const int slot = items % kPkItems;
          if (items >= kPkItems && !pk_wait(&sm.item_empty[slot], (items / kPkItems - 1) & 1, abort, p.err, kDevWaitMma, lim)) break;
          PkItem& it = sm.item[slot];
          it.valid = piece < (uint32_t)sm.pieces;
          it.poison = 0;
          int n = 0;
          if (it.valid) {
            int lo = 0, hi = entries - 1;              // the last entry that begins at or before the piece
            while (lo < hi) {
              const int mid = (lo + hi + 1) >> 1;
              if (sm.pre[mid] <= (int)piece) lo = mid;
              else hi = mid - 1;
            }
            int off = (int)piece - sm.pre[lo], part = sm.slot_pre[lo], counter = sm.counter_pre[lo];
            PkSeq s = sequence(lo, 0);
            PkShape h = pk_shape(p, s, sm.limit);
            for (int i = 1; off >= h.tiles * h.splits * p.kv_heads; ++i) {
              off -= h.tiles * h.splits * p.kv_heads;
              if (h.splits > 1) part += h.live * h.splits * p.kv_heads, counter += h.live * p.kv_heads;
              s = sequence(lo, i);
              h = pk_shape(p, s, sm.limit);
            }
            // as many KV heads together as the L2 holds with ease, the longest tiles of them all first
            const int held = min(max((48 << 11) / max(s.kn, 1), 1), p.kv_heads);       // 48 MB of 512 bytes a key
            const int each = h.tiles * h.splits, head0 = off / (each * held) * held, heads = min(held, p.kv_heads - head0);
            const int rest = off - head0 * each, row = rest / (heads * h.splits), in = rest % (heads * h.splits);
            const int tile = h.tiles - 1 - row, kvh = head0 + in / h.splits, split = in % h.splits;
            it.kvh = kvh;
            it.q_row = s.q0, it.q_len = s.qn, it.k_row = s.k0, it.k_len = s.kn;
            it.tok0 = tile * 2 * p.tokens;
            int c[2];
            for (int x = 0; x < 2; ++x) {
              const int t0 = it.tok0 + x * p.tokens;
              c[x] = t0 < s.qn ? (visible(it, min(t0 + p.tokens, s.qn)) + kPkKeys - 1) / kPkKeys : 0;
            }
            const int cost = max(c[0], c[1]);
            const int parts = cost > sm.limit ? (cost + sm.limit - 1) / sm.limit : 1;
            // 2^23 key tiles at most, and some 300 parts: below 2^32
            const int p0 = (int)((unsigned)cost * min(split, parts) / parts), p1 = (int)((unsigned)cost * min(split + 1, parts) / parts);
            it.first = p0;
            for (int x = 0; x < 2; ++x) it.n[x] = max(min(c[x], p1) - p0, 0);
            n = max(it.n[0], it.n[1]);
            it.splits = parts;
            const int at = kvh * h.live + tile - (h.tiles - h.live);
            it.slot = part + at * h.splits, it.split = split;
            if (h.splits > 1 && split == 0 && at >= kvh * h.live) p.cuts->cut[counter + at] = {it.q_row, it.tok0, it.q_len, kvh, it.slot, parts};
            if (split >= parts) it.valid = 2;          // nothing in this piece
          }
          const bool more = it.valid != 0;
          mbar_arrive(&sm.item_full[slot]);
          ++items;
          if (!more) break;
          piece = sm.pieces > gridDim.x ? gridDim.x + atomicAdd((unsigned*)p.counters, 1u) : (uint32_t)sm.pieces;
          if (it.valid == 2 || n == 0) continue;
          const int krow = it.k_row + it.first * kPkKeys;
          for (int j = 0; ok && j < 2 * n; ++j, ++kv) {
            const int st = kv % kPkStages;
            if (kv >= kPkStages && !pk_wait(&sm.kv_empty[st], (kv / kPkStages - 1) & 1, abort, p.err, kDevWaitMma, lim)) {
              ok = false;
              break;
            }
            if (blockIdx.x == 0 && (int)kv == p.skip_copy) continue;
            uint8_t* dst = KVs + (size_t)st * kPkTileBytes;
            const CUtensorMap* map = j & 1 ? &tm_v : &tm_k;
            mbar_arrive_expect_tx(&sm.kv_full[st], kPkTileBytes);
            tma_load_3d(dst, map, 0, it.kvh, krow + (j >> 1) * kPkKeys, &sm.kv_full[st]);
            tma_load_3d(dst + kPkTileBytes / 2, map, 64, it.kvh, krow + (j >> 1) * kPkKeys, &sm.kv_full[st]);
            if (j == 0) {
              if (qs && !pk_wait(&sm.q_empty, (qs - 1) & 1, abort, p.err, kDevWaitMma, lim)) {
                ++kv;
                ok = false;
                break;
              }
              const uint32_t half = 128u * p.group * p.tokens;
              mbar_arrive_expect_tx(&sm.q_full, 2 * half * ((it.n[0] > 0) + (it.n[1] > 0)));
              for (int x = 0; x < 2; ++x) {
                if (!it.n[x]) continue;
                uint8_t* q = Qs + (size_t)x * kPkTileBytes;
                const int row = it.q_row + it.tok0 + x * p.tokens;
                tma_load_3d(q, &tm_q, 0, it.kvh * p.group, row, &sm.q_full);
                tma_load_3d(q + kPkTileBytes / 2, &tm_q, 64, it.kvh * p.group, row, &sm.q_full);
              }
              ++qs;
            }
          }
        }
        if (*abort) {                                  // what was asked for lands before the CTA ends
          for (uint32_t i = kv > kPkStages ? kv - kPkStages : 0; i < kv; ++i) mbar_wait(&sm.kv_full[i % kPkStages], (i / kPkStages) & 1, lim);
          if (qs) mbar_wait(&sm.q_full, (qs - 1) & 1, lim);
        }
      }
      __syncwarp();
    } else if (warp == kPkRowWarps) {
      // -------------------------------------------------------- matrix products
      // What the instructions' descriptors and the loops depend on is taken from lane 0, so that it
      // is kept in uniform registers: an instruction costs the issuing warp 54 cycles otherwise.
      auto uniform = [](uint32_t v) { return __shfl_sync(0xffffffffu, v, 0); };
      constexpr uint32_t IS = idesc_pf<T>(false), IO = idesc_pf<T>(true);
      const uint32_t q_lo = uniform(smem_u32(Qs)), kv_lo = uniform(smem_u32(KVs)), tm = uniform(tmem);
      uint32_t items = 0, kv = 0, qs = 0, ps0 = 0, ps1 = 0, vb0 = 0, vb1 = 0;
      bool ok = true;
      auto wait = [&](uint64_t* bar, uint32_t parity, int code) {
        ok = pk_wait_warp(bar, parity, abort, p.err, code, lim);
        return ok;
      };
      // S_x = Q_x K^T with the K tile of a stage
      auto scores = [&](auto tile, uint32_t stage) {
        constexpr int x = decltype(tile)::value;
        const uint64_t a = smem_desc_sw128(q_lo + x * kPkTileBytes, 16, 1024);
        const uint64_t b = smem_desc_sw128(kv_lo + stage * kPkTileBytes, 16, 1024);
#pragma unroll
        for (int kk = 0; kk < 8; ++kk) {
          const uint64_t off = ((kk >> 2) * (kPkTileBytes / 2) + (kk & 3) * 32) >> 4;
          mma_f16_ss(tm + x * 256, a + off, b + off, IS, kk > 0);
        }
        mma_commit(&sm.s_full[x]);
      };
      // O_x += P_x V with the V tile of a stage: the first kPkMost keys, or the others
      auto values = [&](auto tile, auto rest, uint32_t stage, bool held) {
        constexpr int x = decltype(tile)::value;
        const uint64_t b = smem_desc_sw128(kv_lo + stage * kPkTileBytes, kPkTileBytes / 2, 1024);
#pragma unroll
        for (int kk = rest ? kPkMost / 16 : 0; kk < (rest ? 8 : kPkMost / 16); ++kk)
          mma_f16_ts(tm + x * 256 + 128, tm + x * 256 + kk * 8, b + ((kk * 2048) >> 4), IO, held || kk > 0);
      };
      using X0 = std::integral_constant<int, 0>;
      using X1 = std::integral_constant<int, 1>;
      while (ok) {
        const uint32_t slot = items % kPkItems;
        if (!wait(&sm.item_full[slot], (items / kPkItems) & 1, kDevWaitCopy)) break;
        ++items;
        const PkItem& it = sm.item[slot];
        const int valid = uniform(it.valid);
        if (!valid) break;
        const int n0 = uniform(it.n[0]), n1 = uniform(it.n[1]), n = valid == 1 ? max(n0, n1) : 0;
        if (n > 0) {
          const int clear = uniform(visible(it, it.tok0 + 1) / kPkKeys - it.first);   // key tiles ahead of the border
          const uint32_t k0 = kv % kPkStages;
          if (!wait(&sm.kv_full[k0], (kv / kPkStages) & 1, kDevWaitCopy)) break;
          if (!wait(&sm.q_full, qs & 1, kDevWaitCopy)) break;
          ++qs;
          if (elect_one()) {
            if (n0 > 0) scores(X0(), k0);
            if (n1 > 0) scores(X1(), k0);
            mma_commit(&sm.kv_empty[k0]);
            if (n == 1) mma_commit(&sm.q_empty);
          }
          __syncwarp();
          for (int j = 0; j < n; ++j, kv += 2) {
            const uint32_t v = (kv + 1) % kPkStages, next = (kv + 2) % kPkStages;
            if (j >= clear) {
              if (!wait(&sm.v_ok[v >> 1], (v >> 1 ? vb1 : vb0) & 1, kDevWaitCopy)) break;
              if (v >> 1) ++vb1;
              else ++vb0;
            } else if (!wait(&sm.kv_full[v], ((kv + 1) / kPkStages) & 1, kDevWaitCopy)) {
              break;
            }
            if (j + 1 < n && !wait(&sm.kv_full[next], ((kv + 2) / kPkStages) & 1, kDevWaitCopy)) break;
            if (j < n0) {
              if (!wait(&sm.p_most[0], ps0 & 1, kDevWaitMma)) break;
              tc_fence_after();
              if (elect_one()) values(X0(), std::false_type(), v, j > 0);
              __syncwarp();
              if (!wait(&sm.p_full[0], ps0 & 1, kDevWaitMma)) break;
              ++ps0;
              tc_fence_after();
              if (elect_one()) {
                values(X0(), std::true_type(), v, true);
                if (j + 1 < n0) scores(X0(), next);
                else mma_commit(&sm.o_full[0]);
                if (j >= n1) {
                  mma_commit(&sm.kv_empty[v]);
                  if (j + 1 < n) mma_commit(&sm.kv_empty[next]);
                }
                if (j >= n1 && j + 2 == n) mma_commit(&sm.q_empty);
              }
              __syncwarp();
            }
            if (j < n1) {
              if (!wait(&sm.p_most[1], ps1 & 1, kDevWaitMma)) break;
              tc_fence_after();
              if (elect_one()) values(X1(), std::false_type(), v, j > 0);
              __syncwarp();
              if (!wait(&sm.p_full[1], ps1 & 1, kDevWaitMma)) break;
              ++ps1;
              tc_fence_after();
              if (elect_one()) {
                values(X1(), std::true_type(), v, true);
                if (j + 1 < n1) scores(X1(), next);
                else mma_commit(&sm.o_full[1]);
                mma_commit(&sm.kv_empty[v]);
                if (j + 1 < n) mma_commit(&sm.kv_empty[next]);
                if (j + 2 == n) mma_commit(&sm.q_empty);
              }
              __syncwarp();
            }
          }
          if (!ok) break;
        }
        if (lane == 0) mbar_arrive(&sm.item_empty[slot]);
        __syncwarp();
      }
      if (elect_one()) mma_commit(&sm.mma_done);
      __syncwarp();
      mbar_wait(&sm.mma_done, 0, lim);
    } else {
      // -------------------------------------------------------- value tiles at the border
      constexpr uint32_t kExp = std::is_same<T, __half>::value ? 0x7c007c00u : 0x7f807f80u;
      constexpr uint32_t kOne = std::is_same<T, __half>::value ? 0x04000400u : 0x00800080u;
      uint32_t items = 0, kv = 0;
      bool ok = true;
      while (ok) {
        const int slot = items % kPkItems;
        ok = pk_wait_warp(&sm.item_full[slot], (items / kPkItems) & 1, abort, p.err, kDevWaitCopy, lim);
        if (!ok) break;
        ++items;
        PkItem& it = sm.item[slot];
        if (!it.valid) break;
        const int n = it.valid == 1 ? max(it.n[0], it.n[1]) : 0;
        for (int j = 0; j < n; ++j, kv += 2) {
          const uint32_t v = (kv + 1) % kPkStages;
          ok = pk_wait_warp(&sm.kv_full[v], ((kv + 1) / kPkStages) & 1, abort, p.err, kDevWaitCopy, lim);
          if (!ok) break;
          if (!border(it, j)) {
            if (lane == 0) mbar_arrive(&sm.kv_empty[v]);
            __syncwarp();
            continue;
          }
          uint4* tile = reinterpret_cast<uint4*>(KVs + (size_t)v * kPkTileBytes);
          const int keys = it.k_len - (it.first + j) * kPkKeys;   // rows that are the sequence's
          bool found = false;
#pragma unroll 8
          for (int i = tid - (kPkRowWarps + 2) * 32; i < kPkTileBytes / 16; i += 64) {
            uint4 w = tile[i];
            const int key = (i >> 3) & 127;                       // a row of 128 bytes in either half
            const uint32_t odd = ((((w.x & kExp) + kOne) | ((w.y & kExp) + kOne) | ((w.z & kExp) + kOne) | ((w.w & kExp) + kOne))) & 0x80008000u;
            if (key >= keys) {
              tile[i] = make_uint4(0, 0, 0, 0);
            } else if (odd) {
              found = true;
              auto clean = [&](uint32_t a) {
                const uint32_t o = ((a & kExp) + kOne) & 0x80008000u;
                return a & ~((o >> 15) * 0xffffu);
              };
              tile[i] = make_uint4(clean(w.x), clean(w.y), clean(w.z), clean(w.w));
            }
          }
          if (found) *reinterpret_cast<volatile int*>(&it.poison) = 1;
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) mbar_arrive(&sm.v_ok[v >> 1]), mbar_arrive(&sm.kv_empty[v]);
        }
        if (ok && lane == 0) mbar_arrive(&sm.item_empty[slot]);
        __syncwarp();
      }
    }
  } else {
    // ------------------------------------------------------------ a thread a row
    regs_inc<kPkRowRegs>();
    const int x = warp >> 2;
    const uint32_t sa = tmem + x * 256 + ((uint32_t)((warp & 3) * 32) << 16);
    uint32_t items = 0, ss = 0, os = 0;
    bool ok = true;
    auto wait = [&](uint64_t* bar, uint32_t parity, int code) {
      ok = pk_wait_warp(bar, parity, abort, p.err, code, lim);
      return ok;
    };
    auto arrive = [&](uint64_t* bar) {
      __syncwarp();
      if (lane == 0) mbar_arrive(bar);
    };
    while (ok) {
      const int slot = items % kPkItems;
      if (!wait(&sm.item_full[slot], (items / kPkItems) & 1, kDevWaitCopy)) break;
      ++items;
      const PkItem& it = sm.item[slot];
      if (!it.valid) break;
      if (it.valid == 1) {
        PkRow row = {-INFINITY, 0.f, false};
        {
          const int nx = it.n[x], first_tok = it.tok0 + x * p.tokens;
          // keys from the piece's first on that every row of the tile sees, and that this row does
          const int key0 = it.first * kPkKeys, all = visible(it, first_tok + 1) - key0;
          const int see = visible(it, min(first_tok + (tid & 127) / p.group, it.q_len) + 1) - key0;
          for (int j = 0; j < nx; ++j) {
            if (!wait(&sm.s_full[x], ss & 1, kDevWaitMma)) break;
            ++ss;
            tc_fence_after();
            pk_softmax<T>(sa, p.scale_log2, (j + 1) * kPkKeys > all, see - j * kPkKeys, j > 0, row, &sm.p_most[x]);
            tc_fence_before();
            arrive(&sm.p_full[x]);
          }
        }
        if (!ok) break;
        const int nx = it.n[x], r = tid & 127, tok_in = r / p.group, tok = it.tok0 + x * p.tokens + tok_in;
        if (nx > 0) {
          if (!wait(&sm.o_full[x], os & 1, kDevWaitMma)) break;
          ++os;
          tc_fence_after();
        }
        const PkPlace at = {(int64_t)it.q_row + tok, it.kvh * p.group + r - tok_in * p.group, tok_in < p.tokens && tok < it.q_len};
        const int border0 = max(it.first, visible(it, it.tok0 + 1) / kPkKeys) * kPkKeys;
        const int upto = *reinterpret_cast<const volatile int*>(&it.poison) ? min(visible(it, tok + 1), (it.first + nx) * kPkKeys) : 0;
        if (row.bad) row.m = 0.f, row.l = NAN;
        if (it.splits == 1) {
          pk_finish<T>(p, it, at, sa + 128, nx, border0, upto, row.m, row.l);
        } else {
          float* part = p.parts + (int64_t)(it.slot + it.split) * kPkPartFloats + x * kPkTilePart;
          pk_put_part<T>(p, it, at, sa + 128, nx, border0, upto, row.m, row.l, part, r);
        }
      }
      arrive(&sm.item_empty[slot]);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == kPkRowWarps) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
  // the last CTA leaves the counters clear for the next call, where any were used
  if (sm.pieces <= gridDim.x || tid != 0) return;
  if (atomicAdd(p.counters + 1, 1) == (int)gridDim.x - 1) p.counters[0] = p.counters[1] = 0;
}

}  // namespace starkv
