// attention_cached.cu - attention of each sequence's newest tokens over a paged
// cache held in 8 bits (kv_cache.cu), on the sm_100a fp8 tensor cores.
//
// o[t, h] = sum_j p_j v_j / sum_j p_j, p_j = 2^(x_j), x_j = scale log2(e) *
// q[t, h] . k_j, over the tokens j of t's sequence that t sees; k_j and v_j are
// e4m3 codes times their page's scale. Groups of heads / kv_heads query heads
// share a K/V head; a K/V head's `rows` are its query heads times the new
// tokens.
//
// HBM bound: 2 * len * kv_heads * head_dim bytes of codes are read once. So the
// codes go from global to shared memory by TMA and from there into tcgen05.mma
// (kind::f8f6f4) as they are: no thread touches them.
//   S^T[line, column] = K[line, 128 bytes] . Q[column, 128 bytes]
//   O^T[byte, column] += V[line, byte] . P[line, column]
// A line is 128 bytes of codes: one token of head_dim 128 or two of 64. The
// large operand is the M = 128 side, the few rows are columns of the N side.
// A row of Q takes three columns, the terms of an exact split of an 11-bit
// number into e4m3 numbers: y = t0 + t1/16 + t2/256, each term the rounding
// (4 bits, to nearest) of what is left. fp16 and bf16 queries (scaled by a
// power of two, the largest to [128, 256)) are represented exactly down to 2^-6,
// smaller elements to within 2^-18, 2^-25 of the row's largest.
// A row's weights p are rounded to fp16 (half a step of 2^-11) and take four
// columns, e5m2 numbers: p = t0 + t1/8 + t2/64 + t3/512, each term the three
// leading bits of what is left. e5m2 is fp16's upper byte, so the split is exact
// for every fp16 number, the subnormal ones too, and a weight that is far below
// its row's largest keeps its bits: all 11 down to 2^-26 of it, and what lies
// below to within 2^-37. (Three e4m3 terms end 2^-23 below the largest: of a
// row with one heavy key and 130,000 light ones that hold a fifth of the sum,
// 5 % of the light ones' share went. The fourth term costs 4 % at 16 rows of
// head_dim 64, 2 % at 16 of 128 and nothing with fewer.) Products are exact and
// sums fp32. For head_dim 64 a column serves one of the line's two tokens: Q's
// other half is zero, and of O^T only the half of the column's token is used (the
// tensor cores have room: an MMA is bound by its 128-row operand up to 64
// columns).
// 0 * NaN is NaN, so a line's other token must not be a NaN code that the row
// does not see: warp 3 looks through the K lines where that can be, the odd
// token behind a sequence's end and the newest tokens, before the MMA.
//
// A CTA, two per SM: warp 0 streams tiles of 128 lines (16 KB of K, 16 KB of V)
// page by page through the table; warp 1 issues the MMAs; warp 2 loads and
// splits the next item's queries; warps 4-7, one thread per line, turn scores
// into weights: a handful of exponentials per thread and tile. The running
// maximum moves only when a score exceeds it by 2.8, found by one barrier with
// a vote; only then are maxima exchanged and O^T rescaled in tensor memory.
//
// Split: the context is cut into units of tiles, the units of all items
// (sequence, K/V head, row block) are counted through, an item's begin and end
// as two more, and each of the 2 * num_sms CTAs takes an equal run of them,
// whatever the sequences' lengths. Where a run
// begins or ends inside an item, the CTA leaves its unnormalised sum, maximum
// and row sum in the workspace, and cached_join_kernel adds the pieces in the
// order of the CTAs (no atomics: the result does not depend on timing).
//
// V's scale joins the exponent: P = 2^(x + log2(vs) - M + 12) with M the running
// maximum of x + log2(vs), at most 2^14.8 < 57344, e5m2's largest; "largest"
// above is that of p times vs. The row sum adds P / vs in fp32.
//
// Measured (32 heads on 8 of 128): two contexts of 131,072 and 100,003 tokens,
// pages of 128, 474 MB: 79 us, 6.0 TB/s, 92 % of a copy's rate, and 2 to 3 for
// the join; 64 contexts of 33 to 4096 tokens, one new token each, pages of 64: 30
// us for 114 MB, where plan, first loads, and the end and join of items that
// are cut cost about 10. 8 contexts of 5200 to 5500 tokens, 1 to 8 new tokens, 16
// heads on 4 of 64, pages of 32: 24.2 us, bound by the 32 rows' terms, which read
// the cache twice. One context of 77 tokens: 6.8 us, latency from the lengths to
// the result. (With the codes unpacked by the threads and fed to mma.sync the
// four took 115, 57, 25 and 7.8 us.) Pages of 16 tokens with head_dim 64 cost
// a long context 28 % more than larger ones: a TMA box of 1 KB each.
#include <algorithm>

#include "common.cuh"
#include "internal.h"

#include <cuda_bf16.h>

namespace sam3 {
namespace {

constexpr int THREADS = 256;
constexpr int MAX_SEQS = SAM3_CACHED_MAX_SEQS;
constexpr int LINES = 128;             // lines per tile
constexpr int TILE = LINES * 128;      // bytes of K or V per tile
constexpr int UNIT_TILES = 4;          // tiles per unit of small jobs
constexpr int ITEM_COST = 2;           // what an item costs besides its tiles, in tiles
constexpr float P_EXP = 12.f;          // the weight at the running maximum is 2^12
constexpr float NO_MAX = 1e30f;        // P_EXP - M of a row that has seen nothing
constexpr float P_TOP = 14.8f;         // and may grow to 2^14.8 before M moves
enum : int { kFirst = 1, kLast = 2, kFinal = 4, kCheck = 8 };
constexpr int kNever = 0x7FFFFFFF;

template <int D, int RB>
struct Cfg {
  static constexpr int TPL = 128 / D;             // tokens per line
  static constexpr int TT = LINES * TPL;          // tokens per tile
  static constexpr int NS = (3 * RB * TPL + 15) / 16 * 16;  // columns of S^T
  static constexpr int N = 4 * RB * TPL;          // columns of O^T
  static constexpr int PW = N <= 32 ? 32 : N;     // bytes of a line of P
  static constexpr int ST = N <= 32 ? 3 : 2;      // ring stages (K and V tile each)
  static constexpr uint32_t COLS = N <= 16 ? 32 : N <= 32 ? 64 : N <= 64 ? 128 : 256;
  static constexpr int GRAN = TT / 16;            // scale entries per tile (16 tokens)
  static constexpr int OFF_Q = ST * 2 * TILE;               // [2][NS][128]
  static constexpr int OFF_P = OFF_Q + 2 * NS * 128;        // [LINES][PW]
  static constexpr int OFF_SCALE = OFF_P + LINES * PW;      // [ST][GRAN] float4
  static constexpr int OFF_INFO = OFF_SCALE + ST * GRAN * 16;     // [ST] int4
  static constexpr int OFF_ITEM = OFF_INFO + ST * 16;       // [2] ItemInfo
  static constexpr int ITEM = 16 + RB * 16;
  static constexpr int OFF_MAX = OFF_ITEM + 2 * ITEM;       // [RB] float4
  static constexpr int OFF_POISON = OFF_MAX + RB * 16;      // [128] u32
  static constexpr int OFF_BAR = OFF_POISON + 512;
  static constexpr int BARS = 3 * ST + 4 + 7;
  static constexpr int OFF_MISC = OFF_BAR + BARS * 8;
  static constexpr int SMEM = OFF_MISC + 128 + 1024;
  // column of term t of row r for token p of a line: a pair of rows takes six
  // neighbours of S^T, as split3 gives them, or eight of O^T
  static constexpr __host__ __device__ int col_s(int p, int r, int t) {
    return (p * RB + r) / 2 * 6 + 2 * t + (r & 1);
  }
  static constexpr __host__ __device__ int col_o(int p, int r, int t) {
    return (p * RB + r) / 2 * 8 + 2 * t + (r & 1);
  }
  // row of a column of O^T
  static constexpr __host__ __device__ int row_of(int n) { return (n / 8 * 2 + (n & 1)) % RB; }
};
static_assert(2 * (Cfg<128, 8>::SMEM + 1024) <= 228 * 1024, "two CTAs per SM");
static_assert(2 * (Cfg<128, 16>::SMEM + 1024) <= 228 * 1024, "two CTAs per SM");
static_assert(2 * (Cfg<64, 4>::SMEM + 1024) <= 228 * 1024, "two CTAs per SM");
static_assert(2 * (Cfg<64, 16>::SMEM + 1024) <= 228 * 1024, "two CTAs per SM");

struct CachedArgs {
  const uint16_t* q;
  uint16_t* o;
  int64_t q_stride, o_stride;
  const int32_t* cu;
  const int32_t* lens;
  const int32_t* table;
  const float* k_scale;
  const float* v_scale;
  float* part;
  int32_t* meta;
  int* err;
  int table_stride, num_pages, page_shift, kv_heads, group, n_seqs, rows, max_new;
  int causal;
  int whole;  // no sequence has more than one unit of UNIT_TILES tiles
  float scale_log2;
};

// What the query warp tells the others of an item (smem).
struct ItemInfo {
  int n_rows, starts, ends, pad;
};

__device__ __forceinline__ bool vote_any(bool p) {  // over warps 4-7
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %1, 0;\n\t"
      "barrier.cta.red.or.pred q, 2, 128, p;\n\tselp.b32 %0, 1, 0, q;\n\t}"
      : "=r"(r)
      : "r"((uint32_t)p)
      : "memory");
  return r != 0;
}
__device__ __forceinline__ void compute_barrier() {
  asm volatile("barrier.cta.sync 2, 128;" ::: "memory");
}
// Largest of the warp, by the integer order of floats (its own inverse).
__device__ __forceinline__ int float_order(int b) { return b ^ ((b >> 31) & 0x7FFFFFFF); }
__device__ __forceinline__ float warp_max(float v) {
  return __int_as_float(
      float_order(__reduce_max_sync(0xffffffffu, float_order(__float_as_int(v)))));
}
// Sums of RB values over the warp: lane i returns that of value i * RB / 32.
template <int RB>
__device__ __forceinline__ float warp_add(float (&v)[RB]) {
  const int lane = threadIdx.x & 31;
  int o = 16;
#pragma unroll
  for (int n = RB / 2; n > 0; n /= 2, o /= 2)
#pragma unroll
    for (int k = 0; k < n; ++k) {
      const bool up = lane & o;
      const float keep = up ? v[k + n] : v[k], send = up ? v[k] : v[k + n];
      v[k] = keep + __shfl_xor_sync(0xffffffffu, send, o);
    }
#pragma unroll
  for (int k = 16 / RB; k > 0; k /= 2) v[0] += __shfl_xor_sync(0xffffffffu, v[0], k);
  return v[0];
}

// The three terms of a pair of fp16 numbers of at most 448, as code pairs:
// every subtraction and product below is exact.
__device__ __forceinline__ void split3(__half2 h, uint16_t (&t)[3]) {
#pragma unroll
  for (int i = 0; i < 3; ++i) {
    const uint32_t w = *reinterpret_cast<const uint32_t*>(&h);
    asm("cvt.rn.satfinite.e4m3x2.f16x2 %0, %1;" : "=h"(t[i]) : "r"(w));
    if (i == 2) break;
    uint32_t b;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(b) : "h"(t[i]));
    h = __hmul2(__hsub2(h, *reinterpret_cast<const __half2*>(&b)), __float2half2_rn(16.f));
  }
}

// The four terms of two pairs of fp16 numbers below 57344, as e5m2 code pairs in
// the order of the columns: every subtraction and product below is exact.
__device__ __forceinline__ uint4 split4(__half2 a, __half2 b) {
  auto pair = [](__half2 h, uint32_t& t01, uint32_t& t23) {
    uint32_t t[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      t[i] = *reinterpret_cast<const uint32_t*>(&h) & 0xFF00FF00u;
      if (i < 3)
        h = __hmul2(__hsub2(h, *reinterpret_cast<const __half2*>(&t[i])), __float2half2_rn(8.f));
    }
    t01 = __byte_perm(t[0], t[1], 0x7531);
    t23 = __byte_perm(t[2], t[3], 0x7531);
  };
  uint4 w;
  pair(a, w.x, w.y);
  pair(b, w.z, w.w);
  return w;
}

// Bytes of w whose code is NaN (0x7F or 0xFF), as 0xFF.
__device__ __forceinline__ uint32_t nan_codes(uint32_t w) {
  return __vcmpeq4(w & 0x7F7F7F7Fu, 0x7F7F7F7Fu);
}

// A sequence as the kernels see it; one that does not fit its buffers counts
// as having no new tokens.
struct Seq {
  int len, row0, fresh;
};
struct RawSeq {
  int len, row0, row1;
};
__device__ __forceinline__ RawSeq fetch_seq(const CachedArgs& a, int i) {
  return {a.lens[i], a.cu ? a.cu[i] : i, a.cu ? a.cu[i + 1] : i + 1};
}
__device__ __forceinline__ Seq checked_seq(const CachedArgs& a, const RawSeq& r, bool report) {
  const bool ok =
      tokens_fit(r.row0, r.row1, a.rows, a.max_new, r.len, a.table_stride, a.page_shift);
  if (!ok && report) report_bad_index(a.err, kDevErrBadLengths);
  return {r.len, r.row0, ok ? r.row1 - r.row0 : 0};
}
__device__ __forceinline__ Seq load_seq(const CachedArgs& a, int i) {
  return checked_seq(a, fetch_seq(a, i), false);
}

// A run of cost over the items (sequence; K/V head and row block): an item costs
// `extra` and then one for each of its units. A run that ends inside the extra
// part leaves the item to the next CTA, one that begins there takes it from its
// first unit.
template <int D, int RB>
struct Run {
  int seq, sub, unit;        // where it is
  int left;                  // cost to go, with the extra part of this item behind it
  int unit_tiles, extra;
  Seq s;
  int units, blocks, tiles;  // of the sequence

  __device__ __forceinline__ void enter(const Seq& seq_, int group) {
    s = seq_;
    blocks = (s.fresh * group + RB - 1) / RB;
    tiles = s.fresh ? (s.len + Cfg<D, RB>::TT - 1) / Cfg<D, RB>::TT : 0;
    units = (tiles + unit_tiles - 1) / unit_tiles;
  }
  // `at`: cost of the sequence before the run's begin
  __device__ __forceinline__ void start(int seq_, const Seq& first, int at, int cost, int ut, int ex,
                                        int group) {
    seq = seq_;
    unit_tiles = ut;
    extra = ex;
    enter(first, group);
    sub = at / (units + extra);
    const int f = at - sub * (units + extra);
    unit = max(0, f - extra);
    left = cost - max(0, extra - f);
  }
  // tiles [tile0(), tile1()) of the item are next
  __device__ __forceinline__ int n_units() const { return min(left, units - unit); }
  __device__ __forceinline__ int tile0() const { return unit * unit_tiles; }
  __device__ __forceinline__ int tile1() const { return min((unit + n_units()) * unit_tiles, tiles); }
  __device__ __forceinline__ int head() const { return sub / blocks; }
  __device__ __forceinline__ void next(const CachedArgs& a) {
    left -= n_units() + extra;
    unit = 0;
    if (left <= 0 || ++sub < a.kv_heads * blocks) return;
    sub = 0;
    do {
      if (++seq >= a.n_seqs) {
        left = 0;
        return;
      }
      enter(load_seq(a, seq), a.group);
    } while (units == 0);
  }
};

template <bool BF>
__device__ __forceinline__ uint16_t to_out(float v) {
  if (BF) return __bfloat16_as_ushort(__float2bfloat16_rn(v));
  return __half_as_ushort(__float2half_rn(v));
}

template <int D, int RB, bool BF>
__global__ void __launch_bounds__(THREADS, 2)
    cached_attn_kernel(const __grid_constant__ CUtensorMap map_k,
                       const __grid_constant__ CUtensorMap map_v, const CachedArgs a) {
  using C = Cfg<D, RB>;
  constexpr int TPL = C::TPL, NS = C::NS, N = C::N, ST = C::ST;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  const uint32_t sbase = smem_u32(smem);
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;

  const uint32_t bar_k = sbase + C::OFF_BAR;    // [ST] K tile, scales and info are there
  const uint32_t bar_v = bar_k + 8 * ST;        // [ST] V tile is there
  const uint32_t bar_empty = bar_v + 8 * ST;    // [ST] the tile's P V is done
  const uint32_t bar_q = bar_empty + 8 * ST;    // [2] an item's queries are split
  const uint32_t bar_q_empty = bar_q + 16;      // [2] the item is finished
  const uint32_t bar_s = bar_q_empty + 16;      // scores are in tensor memory
  const uint32_t bar_s_free = bar_s + 8;        // and have been read
  const uint32_t bar_p = bar_s_free + 8;        // weights are in shared memory
  const uint32_t bar_o = bar_p + 8;             // P V done: weights read, O^T current
  const uint32_t bar_drain = bar_o + 8;
  const uint32_t bar_raw = bar_drain + 8;       // a K tile for warp 3 is there (head_dim 64)
  const uint32_t bar_raw_free = bar_raw + 8;    // and looked through
  uint8_t* misc = smem + C::OFF_MISC;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(misc);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(misc + 4);
  volatile int* softmax_failed = reinterpret_cast<volatile int*>(misc + 8);
  volatile int* progress = reinterpret_cast<volatile int*>(misc + 12);  // tiles passed on
  volatile int* raw_stage = reinterpret_cast<volatile int*>(misc + 64);
  volatile int* k_nan = reinterpret_cast<volatile int*>(misc + 68);       // [ST]
  float4* scales = reinterpret_cast<float4*>(smem + C::OFF_SCALE);
  int4* infos = reinterpret_cast<int4*>(smem + C::OFF_INFO);
  uint32_t* poison = reinterpret_cast<uint32_t*>(smem + C::OFF_POISON);
  auto item_info = [&](int b) { return reinterpret_cast<ItemInfo*>(smem + C::OFF_ITEM + b * C::ITEM); };
  // of each row: where its output goes, the power of two its queries were
  // divided by, how many tokens it sees
  auto item_out = [&](int b) { return reinterpret_cast<int64_t*>(smem + C::OFF_ITEM + b * C::ITEM + 16); };
  auto item_rs = [&](int b) { return reinterpret_cast<float*>(item_out(b) + RB); };
  auto item_lim = [&](int b) { return reinterpret_cast<int*>(item_rs(b) + RB); };

  if (threadIdx.x == 0) {
    for (int s = 0; s < ST; ++s) {
      mbar_init(bar_k + 8 * s, 1);
      mbar_init(bar_v + 8 * s, 1);
      mbar_init(bar_empty + 8 * s, 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(bar_q + 8 * b, 1);
      mbar_init(bar_q_empty + 8 * b, 128);
    }
    mbar_init(bar_s, 1);
    mbar_init(bar_s_free, 128);
    mbar_init(bar_p, 128);
    mbar_init(bar_o, 1);
    mbar_init(bar_drain, 1);
    mbar_init(bar_raw, 1);
    mbar_init(bar_raw_free, 1);
    for (int s = 0; s < ST; ++s) k_nan[s] = kNever;
    *abort_flag = 0;
    *softmax_failed = 0;
    *progress = 0;
    fence_mbar_init();
    prefetch_tmap(&map_k);
    prefetch_tmap(&map_v);
  }
  if (threadIdx.x < 128) poison[threadIdx.x] = 0;
  if (warp == 1) {
    tmem_alloc(smem_u32(tmem_slot), C::COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  griddep_launch_dependents();  // behind the allocation: the next kernel allocates too
  griddep_wait();  // lengths, pages, codes and queries may be earlier kernels' outputs

  // ------------------------------------------------- this CTA's run
  // Each warp plans for itself (no barrier): lane l gets the costs of the 32
  // sequences from 32 l on, as single tiles and as units of UNIT_TILES.
  // (Whole lines of lengths at a time: with 32 sequences in a row to each lane the
  // plan of 1000 took 25 us, and a single sequence's call 0.3 us less.)
  const int m = (a.n_seqs + 31) / 32;
  auto cost_of = [&](const Seq& s, bool units) {
    if (s.fresh == 0) return 0;
    const int tiles = (s.len + C::TT - 1) / C::TT;
    const int items = (s.fresh * a.group + RB - 1) / RB * a.kv_heads;
    return (units ? (tiles + UNIT_TILES - 1) / UNIT_TILES : tiles + ITEM_COST) * items;
  };
  int sum_tiles = 0, sum_units = 0;
  for (int j0 = 0; j0 < m; j0 += 8) {  // loads of 256 sequences in flight
    RawSeq r[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int i = 32 * (j0 + j) + lane;
      r[j] = i < a.n_seqs ? fetch_seq(a, i) : RawSeq{0, 0, 0};
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if (j0 + j >= m) break;
      const Seq s = checked_seq(a, r[j], blockIdx.x == 0 && warp == 0);
      const int n_tiles = __reduce_add_sync(0xffffffffu, cost_of(s, false));
      const int n_units = __reduce_add_sync(0xffffffffu, cost_of(s, true));
      if (lane == j0 + j) {
        sum_tiles = n_tiles;
        sum_units = n_units;
      }
    }
  }
  // Few tiles: runs of whole units of UNIT_TILES, so that short items are not cut
  // (a piece costs a join, about as much as four tiles), as long as no CTA gets
  // more than one. Else single tiles, for balance.
  const bool few = a.whole || __reduce_add_sync(0xffffffffu, sum_units) <= (int)gridDim.x;
  const int ut = few ? UNIT_TILES : 1, extra = few ? 0 : ITEM_COST;
  const int own = few ? sum_units : sum_tiles;
  auto sums_to_here = [&](int v) {
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, v, o);
      if (lane >= o) v += u;
    }
    return v;
  };
  const int upto = sums_to_here(own);
  const int total = __shfl_sync(0xffffffffu, upto, 31);
  // equal runs, without a gap between the CTAs that have one (the join's order)
  const int ctas = min((int)gridDim.x, total), cta = min((int)blockIdx.x, ctas);
  const int each = total / max(1, ctas), more = total - each * ctas;
  const int x0 = cta * each + min(cta, more);
  const int cost = cta < ctas ? each + (cta < more) : 0;
  Run<D, RB> run;
  bool busy = cost > 0;
  if (busy) {
    // the 32 sequences, and the one of them, that x0 is in
    const int l = __ffs(__ballot_sync(0xffffffffu, upto > x0)) - 1;
    const int at = x0 - __shfl_sync(0xffffffffu, upto - own, l);
    Seq s{0, 0, 0};
    if (32 * l + lane < a.n_seqs) s = load_seq(a, 32 * l + lane);
    const int its = cost_of(s, few), end = sums_to_here(its);
    const int w = __ffs(__ballot_sync(0xffffffffu, end > at)) - 1;
    s.len = __shfl_sync(0xffffffffu, s.len, w);
    s.row0 = __shfl_sync(0xffffffffu, s.row0, w);
    s.fresh = __shfl_sync(0xffffffffu, s.fresh, w);
    run.start(32 * l + w, s, at - __shfl_sync(0xffffffffu, end - its, w), cost, ut, extra, a.group);
    busy = run.left > 0;  // a run may lie inside one item's extra part
  }
  if (threadIdx.x == 64) a.meta[blockIdx.x * 4] = 0;  // warp 2 knows better later

  if (busy && warp == 0) {
    // ------------------------------------------------------------- producer
    const int page = 1 << a.page_shift;
    const int per = C::TT >> a.page_shift;  // pages per tile: 1 ... 16
    const uint32_t copy_bytes = (uint32_t)page * D;
    int stage = 0;
    uint32_t phase = 0, used = 0, raws = 0;
    int passed = 0;  // tiles
    bool ok = true;
    Run<D, RB>& r = run;
    // Pages come in windows of 32, one per lane, with their scales. Loads run
    // ahead of their use: page numbers two windows, scales one; and where a
    // sequence fits one window, the next head's scales while this one's tiles
    // are streamed.
    struct Scales {
      float k = 0.f, v = 1.f;
    };
    auto load_slot = [&](const int32_t* row, int window, int pages) {
      const int p = window + lane;
      int s = p < pages ? row[p] : -1;
      if (p < pages && !page_fits(s, a.num_pages)) {
        report_bad_index(a.err, kDevErrBadPage);
        s = -1;
      }
      return s;
    };
    auto load_scales = [&](int s, int head) {
      Scales v;
      if (s >= 0) {
        v.k = a.k_scale[(size_t)s * a.kv_heads + head];
        v.v = a.v_scale[(size_t)s * a.kv_heads + head];
      }
      return v;
    };
    int seq = -1, slot = -1, slot1 = -1, slot2 = -1, window = 0;
    Scales sc0, sc1;  // of slot, and of slot1 or the next head
    bool one_window = false;
    while (r.left > 0 && ok) {
      const int len = r.s.len, head = r.head();
      const int tile0 = r.tile0(), tile1 = r.tile1();
      const int lim_min = a.causal ? len - r.s.fresh + 1 : len;
      const int pages = (len + page - 1) >> a.page_shift;
      const int32_t* row = a.table + (size_t)r.seq * a.table_stride;
      const bool final_item = r.left <= r.n_units() + r.extra;
      if (one_window && seq == r.seq) {
        sc0 = sc1;
      } else {
        seq = r.seq;
        one_window = pages <= 32 && r.blocks == 1;
        window = (tile0 * per) & ~31;
        slot = load_slot(row, window, pages);
        slot1 = load_slot(row, window + 32, pages);
        slot2 = load_slot(row, window + 64, pages);
        sc0 = load_scales(slot, head);
        if (!one_window) sc1 = load_scales(slot1, head);
      }
      if (one_window && head + 1 < a.kv_heads) sc1 = load_scales(slot, head + 1);
      for (int tile = tile0; tile < tile1 && ok; ++tile) {
        const int first = tile * per;
        if (first >= window + 32) {
          window += 32;
          slot = slot1;
          slot1 = slot2;
          slot2 = load_slot(row, window + 64, pages);
          sc0 = sc1;
          sc1 = load_scales(slot1, head);
        }
        ok = mbar_wait(bar_empty + 8 * stage, phase ^ 1, abort_flag, a.err, kDevErrTimeoutCached);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        // lane l copies K (l < 16) or V of page l % 16 of the tile
        const int my_page = first + (lane & 15);
        const int my_slot = __shfl_sync(0xffffffffu, slot, my_page & 31);
        const bool copies = (lane & 15) < per && my_page < pages && my_slot >= 0;
        const uint32_t n_copies = __popc(__ballot_sync(0xffffffffu, copies) & 0xFFFFu);
        const bool hole = __any_sync(0xffffffffu, (lane & 15) < per && my_page < pages && my_slot < 0);
        // a line of this tile may hold a K code that not all rows see of it
        const int tile_end = (tile + 1) * C::TT;
        const bool raw = TPL == 2 && ((len & 1 && len < tile_end && len >= tile * C::TT) ||
                                      (lim_min < len && tile_end > lim_min));
        if (raw) {
          ok = __all_sync(0xffffffffu, mbar_wait(bar_raw_free, (raws & 1u) ^ 1, abort_flag, a.err,
                                                 kDevErrTimeoutCached));
          if (!ok) break;
          ++raws;
        }
        const uint32_t bar_k_tile = raw ? bar_raw : bar_k + 8 * stage;
        if (lane == 0) {
          mbar_expect_tx(bar_k_tile, n_copies * copy_bytes);
          mbar_arrive_expect_tx(bar_v + 8 * stage, n_copies * copy_bytes);
        }
        __syncwarp();
        if (copies) {
          const int which = lane >> 4;
          const uint32_t dst =
              sbase + (stage * 2 + which) * TILE + (uint32_t)(lane & 15) * copy_bytes;
          const long long at = ((long long)my_slot * a.kv_heads + head) << a.page_shift;
          tma_load_2d(dst, which ? &map_v : &map_k, which ? bar_v + 8 * stage : bar_k_tile, 0,
                      (int)(at / TPL));
        }
        // the scales may still be on their way
        const int sp = (first + (((lane & 15) * 16) >> a.page_shift)) & 31;
        const float ks = __shfl_sync(0xffffffffu, sc0.k, sp), vs = __shfl_sync(0xffffffffu, sc0.v, sp);
        const bool there = __shfl_sync(0xffffffffu, slot, sp) >= 0;
        // .w: the page is there; the tokens of one that is not count as masked
        if (lane < C::GRAN)
          scales[stage * C::GRAN + lane] =
              make_float4(ks * a.scale_log2, __log2f(vs), 1.f / vs, there ? 1.f : 0.f);
        if (lane == 0) {
          int flags = 0;
          if (tile == tile0) flags |= kFirst;
          if (tile == tile1 - 1) flags |= final_item ? kLast | kFinal : kLast;
          if ((tile + 1) * C::TT > lim_min || hole) flags |= kCheck;
          infos[stage] = make_int4(tile * C::TT, len, flags, lim_min);
          *progress = ++passed;
          if (raw)
            *raw_stage = stage;
          else if (TPL == 2)
            k_nan[stage] = kNever;
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(bar_k_tile);
        used = min(used + 1, (uint32_t)ST);
        if (++stage == ST) {
          stage = 0;
          phase ^= 1;
        }
      }
      if (ok) r.next(a);
    }
    if (TPL == 2) {  // warp 3 may go
      if (ok)
        ok = __all_sync(0xffffffffu, mbar_wait(bar_raw_free, (raws & 1u) ^ 1, abort_flag, a.err,
                                               kDevErrTimeoutCached));
      if (ok && lane == 0) {
        *raw_stage = -1;
        mbar_arrive(bar_raw);
      }
    }
    if (*abort_flag) {
      if (raws) mbar_wait_drain(bar_raw, (raws - 1) & 1u);
      // nothing may still be in flight into this CTA's shared memory
      for (uint32_t i = 0; i < used; ++i) {
        if (--stage < 0) {
          stage = ST - 1;
          phase ^= 1;
        }
        mbar_wait_drain(bar_k + 8 * stage, phase);
        mbar_wait_drain(bar_v + 8 * stage, phase);
      }
    }
  } else if (busy && warp == 1) {
    // ------------------------------------------------------------- MMA issuer
    constexpr uint32_t IDESC_S = umma_idesc_f8(128, NS, 0, kE4M3);
    constexpr uint32_t IDESC_O = umma_idesc_f8(128, N, 1, kE5M2);
    const uint32_t s_col = tmem, o_col = tmem + C::COLS / 2;
    struct Slot {
      int st = 0;
      uint32_t ph = 0;
      __device__ void step() {
        if (++st == ST) {
          st = 0;
          ph ^= 1;
        }
      }
    } qk, pv;                     // stages of the next Q K^T and P V
    uint32_t n_qk = 0, n_pv = 0;  // issued
    uint32_t items = 0;           // begun by Q K^T
    bool all_qk = false, ok = true;
    // what the next of each waits for, as far as it has been seen to be there
    bool have_k = false, have_s = true, have_p = false;
    uint64_t since = global_timer_ns();
    // The whole warp runs this and one elected thread issues, so that what the MMAs
    // take is uniform to the compiler.
    auto here = [](uint32_t bar, uint32_t par) {
      return __all_sync(0xffffffffu, mbar_test(bar, par)) != 0;
    };
    const uint64_t desc_q = umma_desc_sw128(sbase + C::OFF_Q), desc_k = umma_desc_sw128(sbase);
    const uint64_t desc_v = umma_desc_mn<128>(sbase + TILE);
    const uint64_t desc_p = umma_desc_mn<C::PW>(sbase + C::OFF_P);
    // Whichever is ready goes first: the next tile's scores (its K may be late,
    // its item's queries too) or this tile's P V.
    while (ok) {
      bool did = false;
      if (n_pv < n_qk) {
        have_p = have_p || here(bar_p, n_pv & 1u);
        if (have_p && here(bar_v + 8 * pv.st, pv.ph)) {
          const int flags = __shfl_sync(0xffffffffu, infos[pv.st].z, 0);
          tc_fence_after();
          const uint64_t dv = desc_advance(desc_v, pv.st * 2 * TILE);
          if (elect_one()) {
#pragma unroll
            for (int k = 0; k < 4; ++k)
              umma_f8_ss(o_col, desc_advance(dv, k * 4096), desc_advance(desc_p, k * 32 * C::PW),
                         IDESC_O, !(flags & kFirst) || k != 0);
            umma_commit(bar_o);
            umma_commit(bar_empty + 8 * pv.st);
          }
          pv.step();
          ++n_pv;
          have_p = false;
          did = true;
          if (flags & kFinal) break;
        }
      }
      if (!all_qk) {
        have_s = have_s || here(bar_s_free, (n_qk - 1) & 1u);
        have_k = have_k || here(bar_k + 8 * qk.st, qk.ph);
        if (have_s && have_k) {
          const int flags = __shfl_sync(0xffffffffu, infos[qk.st].z, 0);
          if (!(flags & kFirst) || here(bar_q + 8 * (items & 1), (items >> 1) & 1u)) {
            if (flags & kFirst) ++items;
            const uint64_t dk = desc_advance(desc_k, qk.st * 2 * TILE);
            const uint64_t dq = desc_advance(desc_q, ((items - 1) & 1) * NS * 128);
            tc_fence_after();
            if (elect_one()) {
#pragma unroll
              for (int k = 0; k < 4; ++k)
                umma_f8_ss(s_col, desc_advance(dk, k * 32), desc_advance(dq, k * 32), IDESC_S,
                           k != 0);
              umma_commit(bar_s);
            }
            all_qk = flags & kFinal;
            qk.step();
            ++n_qk;
            have_s = have_k = false;
            did = true;
          }
        }
      }
      if (did) {
        since = global_timer_ns();
      } else if (__any_sync(0xffffffffu, *abort_flag)) {
        ok = false;
      } else if (__any_sync(0xffffffffu, global_timer_ns() - since > kWaitTimeoutNs)) {
        *abort_flag = 1;
        atomicExch(a.err, kDevErrTimeoutCached);
        ok = false;
      }
    }
    if (__any_sync(0xffffffffu, *abort_flag)) {
      if (elect_one()) umma_commit(bar_drain);
      mbar_wait_drain(bar_drain, 0);
    }
  } else if (busy && warp == 2) {
    // ------------------------------------------------------------- queries
    constexpr int EPL = D / 32;  // elements per lane
    Run<D, RB>& r = run;
    uint32_t w[RB][EPL / 2];  // this lane's elements of an item's rows
    int n_rows = 0, lim = 0;  // lane i: of row i
    int64_t out = 0;
    auto load_rows = [&]() {
      const int head = r.head(), block = r.sub - head * r.blocks;
      n_rows = min(RB, r.s.fresh * a.group - block * RB);
      const int gr = block * RB + lane;
      const int tok = gr / a.group, col = (head * a.group + gr - tok * a.group) * D;
      out = (int64_t)(r.s.row0 + tok) * a.o_stride + col;
      lim = a.causal && lane < n_rows ? r.s.len - r.s.fresh + tok + 1 : r.s.len;
      const int64_t from = (int64_t)(r.s.row0 + tok) * a.q_stride + col;
#pragma unroll
      for (int i = 0; i < RB; ++i) {
        const uint32_t* src =
            reinterpret_cast<const uint32_t*>(a.q + __shfl_sync(0xffffffffu, from, i)) +
            lane * (EPL / 2);
#pragma unroll
        for (int e = 0; e < EPL / 2; ++e) w[i][e] = i < n_rows ? src[e] : 0u;
      }
    };
    load_rows();
    for (uint32_t item = 0;; ++item) {
      const int b = item & 1;
      if (!__all_sync(0xffffffffu, mbar_wait_idle(bar_q_empty + 8 * b, (item >> 1 & 1) ^ 1,
                                                  abort_flag, progress, a.err,
                                                  kDevErrTimeoutCached)))
        break;
      uint8_t* qb = smem + C::OFF_Q + b * NS * 128;
      float rs = 0.f;
#pragma unroll
      for (int i = 0; i < RB; ++i) {
        float x[EPL];
        float top = 0.f;
#pragma unroll
        for (int e = 0; e < EPL / 2; ++e) {
          const float2 f = BF ? make_float2(__uint_as_float(w[i][e] << 16),
                                            __uint_as_float(w[i][e] & 0xFFFF0000u))
                              : unpack_half2(w[i][e]);
          x[2 * e] = f.x;
          x[2 * e + 1] = f.y;
          top = fmaxf(top, fmaxf(fabsf(f.x), fabsf(f.y)));
        }
        top = warp_max(top);
        // the power of two that brings the largest to [128, 256); a row with an
        // infinity becomes NaN, like its softmax (the codes would saturate)
        const int e2 = min(max(((__float_as_int(top) >> 23) & 255) - 127 - 7, -120), 120);
        const float down = top == INFINITY ? NAN : __int_as_float((127 - e2) << 23);
        if (lane == (i & 31)) rs = __int_as_float((127 + e2) << 23);
        uint16_t t[EPL / 2][3];
#pragma unroll
        for (int e = 0; e < EPL / 2; ++e)
          split3(__floats2half2_rn(x[2 * e] * down, x[2 * e + 1] * down), t[e]);
#pragma unroll
        for (int p = 0; p < TPL; ++p)
#pragma unroll
          for (int k = 0; k < 3; ++k) {
            const int n = C::col_s(p, i, k);
            if (D == 128) {
              const uint32_t at = (uint32_t)(lane * 4) ^ ((n & 7) << 4);
              *reinterpret_cast<uint32_t*>(qb + n * 128 + at) =
                  t[0][k] | (uint32_t)t[EPL / 2 - 1][k] << 16;
            } else {
              const uint32_t at = (uint32_t)(p * 64 + lane * 2) ^ ((n & 7) << 4);
              const uint32_t not_at = (uint32_t)((p ^ 1) * 64 + lane * 2) ^ ((n & 7) << 4);
              *reinterpret_cast<uint16_t*>(qb + n * 128 + at) = t[0][k];
              *reinterpret_cast<uint16_t*>(qb + n * 128 + not_at) = 0;
            }
          }
      }
      if (lane < RB) {
        item_out(b)[lane] = out;
        item_rs(b)[lane] = rs;
        item_lim(b)[lane] = lim;
      }
      const bool starts = r.unit == 0, ends = r.unit + r.n_units() == r.units;
      if (lane == 0) {
        *item_info(b) = {n_rows, starts, ends, 0};
        if (r.left <= r.n_units() + r.extra && !ends) {
          // for the join: 2: an item that begins here ends in a later CTA, 4:
          // the run lies inside one item
          a.meta[blockIdx.x * 4 + 1] = r.seq;
          a.meta[blockIdx.x * 4 + 2] = r.sub;
          a.meta[blockIdx.x * 4] = starts ? 2 : 4;
        }
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar_q + 8 * b);
      r.next(a);
      if (r.left <= 0) break;
      load_rows();  // on their way while the item before is worked on
    }
  } else if (TPL == 2 && busy && warp == 3) {
    // ------------------------------------------- K lines shared by two tokens
    // (there may be none in the whole run)
    for (uint32_t i = 0;; ++i) {
      if (!__all_sync(0xffffffffu, mbar_wait_idle(bar_raw, i & 1u, abort_flag, progress, a.err,
                                                  kDevErrTimeoutCached)))
        break;
      const int st = *raw_stage;
      if (st < 0) break;
      const int4 info = infos[st];
      uint8_t* kt = smem + st * 2 * TILE;
      auto group = [&](int tok, int c) {  // 16 bytes of a token's row
        const int line = (tok - info.x) / TPL, p = (tok - info.x) % TPL;
        return reinterpret_cast<uint4*>(kt + line * 128 + (((p * (D / 16) + c) ^ (line & 7)) << 4));
      };
      // the token behind the end, if its line has the last one
      if ((info.y & 1) && info.y < info.x + C::TT && lane < D / 16)
        *group(info.y, lane) = make_uint4(0, 0, 0, 0);
      // the newest tokens: NaN codes become 0, and the first token with one is told
      const int from = max(info.x, info.w), to = min(info.y, info.x + C::TT);
      int bad_tok = kNever;
      for (int j = lane; j < (to - from) * (D / 16); j += 32) {
        const int tok = from + j / (D / 16);
        uint4* at = group(tok, j % (D / 16));
        const uint4 v = *at;
        const uint4 n = make_uint4(nan_codes(v.x), nan_codes(v.y), nan_codes(v.z), nan_codes(v.w));
        if (n.x | n.y | n.z | n.w) {
          *at = make_uint4(v.x & ~n.x, v.y & ~n.y, v.z & ~n.z, v.w & ~n.w);
          bad_tok = min(bad_tok, tok);
        }
      }
      bad_tok = __reduce_min_sync(0xffffffffu, bad_tok);
      if (lane == 0) k_nan[st] = bad_tok;
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(bar_k + 8 * st);
        mbar_arrive(bar_raw_free);
      }
    }
  } else if (busy && warp >= 4) {
    // ------------------------------------------------------------- weights
    const int line = (warp - 4) * 32 + lane;
    const uint32_t lane_base = tmem + ((uint32_t)((warp - 4) * 32) << 16);
    const uint32_t s_col = lane_base, o_col = lane_base + C::COLS / 2;
    // columns of S^T from col on: the scores of all rows, their three terms added
    auto read_scores = [&](uint32_t col, float (&v)[RB]) {
      constexpr int W = RB;  // a load
      uint32_t s[3][W];
#pragma unroll
      for (int i = 0; i < 3; ++i) tmem_ld_32x32b(col + W * i, s[i]);
      tmem_wait_ld();
      auto at = [&](int n) { return __uint_as_float(s[n / W][n % W]); };
#pragma unroll
      for (int r = 0; r < RB; ++r)
        v[r] = fmaf(at(C::col_s(0, r, 2)), 1.f / 256,
                    fmaf(at(C::col_s(0, r, 1)), 1.f / 16, at(C::col_s(0, r, 0))));
    };
    // 16 columns of O^T from col on: the outputs of 4 rows, their four terms added
    auto read_outputs = [&](uint32_t col, float* v) {
      uint32_t s[16];
      tmem_ld_32x32b(col, s);
      tmem_wait_ld();
      auto at = [&](int r, int t) { return __uint_as_float(s[C::col_o(0, r, t)]); };
#pragma unroll
      for (int r = 0; r < 4; ++r)
        v[r] = fmaf(fmaf(fmaf(at(r, 3), 1.f / 8, at(r, 2)), 1.f / 8, at(r, 1)), 1.f / 8, at(r, 0));
    };
    float4* wmax = reinterpret_cast<float4*>(smem + C::OFF_MAX);
    uint8_t* pb = smem + C::OFF_P;
    float off[RB], l[RB];
    int stage = 0;
    uint32_t phase = 0, items = 0;
    bool ok = true;
    for (uint32_t i = 0;; ++i) {
      // an expired wait is remembered, and all threads leave together below
      ok = ok && mbar_wait(bar_k + 8 * stage, phase, abort_flag, a.err, kDevErrTimeoutCached);
      ok = ok && mbar_wait(bar_s, i & 1u, abort_flag, a.err, kDevErrTimeoutCached);
      ok = __all_sync(0xffffffffu, ok);
      const int4 info = infos[stage];
      const int b = items & 1;
      if (ok && (info.z & kFirst))
        ok = __all_sync(0xffffffffu, mbar_wait(bar_q + 8 * b, (items >> 1) & 1u, abort_flag, a.err,
                                               kDevErrTimeoutCached));
      tc_fence_after();
      float x[TPL][RB];
#pragma unroll
      for (int p = 0; p < TPL; ++p) read_scores(s_col + C::col_s(p, 0, 0), x[p]);
      tc_fence_before();
      mbar_arrive(bar_s_free);
      const float4 sc = scales[stage * C::GRAN + line * TPL / 16];
      const float* rs = item_rs(b);
#pragma unroll
      for (int r = 0; r < RB; ++r) {
        const float f = sc.x * rs[r];
#pragma unroll
        for (int p = 0; p < TPL; ++p) x[p][r] = fmaf(x[p][r], f, sc.y);
      }
      const int tok0 = info.x + line * TPL;
      const bool check = info.z & kCheck;
      if (check) {
        const int* lim = item_lim(b);
        const int bad_tok = k_nan[stage];
#pragma unroll
        for (int r = 0; r < RB; ++r)
#pragma unroll
          for (int p = 0; p < TPL; ++p)
            if (tok0 + p >= lim[r] || sc.w == 0.f)
              x[p][r] = -INFINITY;
            else if (TPL == 2 && tok0 + p == bad_tok)
              x[p][r] = NAN;
      }
      bool grow = !ok || (info.z & kFirst);
      if (!grow) {
        float top = -INFINITY;
#pragma unroll
        for (int r = 0; r < RB; ++r)
#pragma unroll
          for (int p = 0; p < TPL; ++p) top = fmaxf(top, x[p][r] + off[r]);
        grow = top > P_TOP;
      }
      bool o_waited = false;
      if (vote_any(grow)) {
        // the rows' maxima over the tile; M moves where they exceed it by 2.8
        if (!ok) *softmax_failed = 1;
#pragma unroll
        for (int r = 0; r < RB; ++r) {
          float m = x[0][r];
          if (TPL == 2) m = fmaxf(m, x[TPL - 1][r]);
          m = warp_max(m);
          if (lane == (r & 31)) reinterpret_cast<float*>(wmax + r)[warp - 4] = m;
        }
        compute_barrier();
        const bool failed = *softmax_failed;
        float alpha[RB];
        const bool first = info.z & kFirst;
#pragma unroll
        for (int r = 0; r < RB; ++r) {
          const float4 w = wmax[r];
          const float m = fmaxf(fmaxf(w.x, w.y), fmaxf(w.z, w.w));
          if (first) {
            // a row that sees nothing yet (its page may not exist): anything that
            // it sees later exceeds M
            off[r] = m == -INFINITY ? NO_MAX : P_EXP - m;
            l[r] = 0.f;
            alpha[r] = 1.f;
          } else {
            const float to = m + off[r] > P_TOP ? P_EXP - m : off[r];
            alpha[r] = ex2_approx(to - off[r]);
            off[r] = to;
            l[r] *= alpha[r];
          }
        }
        compute_barrier();  // wmax and the flag may be written again
        if (failed) break;
        if (!first) {
          ok = __all_sync(0xffffffffu, mbar_wait(bar_o, (i - 1) & 1u, abort_flag, a.err,
                                                 kDevErrTimeoutCached));
          o_waited = true;
          tc_fence_after();
#pragma unroll
          for (int c = 0; c < N / 16; ++c) {
            bool any = false;  // the same for all threads
#pragma unroll
            for (int e = 0; e < 16; ++e) any |= alpha[C::row_of(16 * c + e)] != 1.f;
            if (!any) continue;
            uint32_t o[16];
            tmem_ld_32x32b(o_col + 16 * c, o);
            tmem_wait_ld();
#pragma unroll
            for (int e = 0; e < 16; ++e)
              o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha[C::row_of(16 * c + e)]);
            tmem_st_32x32b_x16(o_col + 16 * c, o);
          }
          tmem_wait_st();
        }
      }
      if (i > 0 && !o_waited) {  // P V of the tile before has read the weights
        const bool w = mbar_wait(bar_o, (i - 1) & 1u, abort_flag, a.err, kDevErrTimeoutCached);
        ok = __all_sync(0xffffffffu, w) && ok;
      }
      // the weights' terms: a line of P in the order of the columns, its 16-byte
      // groups (4 rows each) swizzled like the tensor cores' PW-byte pattern
      {
        constexpr int G = C::PW / 16;
        const int sw = (line * C::PW >> 7) & (G - 1);
#pragma unroll
        for (int p = 0; p < TPL; ++p)
#pragma unroll
          for (int r = 0; r < RB; r += 4) {
            float w[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              w[e] = ex2_approx(x[p][r + e] + off[r + e]);
              l[r + e] = fmaf(w[e], sc.z, l[r + e]);
            }
            *reinterpret_cast<uint4*>(pb + line * C::PW + (((p * RB + r) / 4 ^ sw) << 4)) =
                split4(__floats2half2_rn(w[0], w[1]), __floats2half2_rn(w[2], w[3]));
          }
      }
      if (check) {
        // Codes of tokens that no row sees become 0 (their weight is 0, but 0 *
        // NaN is not); NaN codes of new tokens that only later rows see become 0
        // and are put into those rows' results at the end.
        const bool w = mbar_wait(bar_v + 8 * stage, phase, abort_flag, a.err, kDevErrTimeoutCached);
        ok = __all_sync(0xffffffffu, w) && ok;
        uint8_t* vl = smem + (stage * 2 + 1) * TILE + line * 128;
#pragma unroll
        for (int p = 0; p < TPL; ++p) {
          const int tok = tok0 + p;
          const bool gone = tok >= info.y || sc.w == 0.f;
          const bool look = a.causal && tok >= info.w;
          if (!gone && !look) continue;
#pragma unroll
          for (int c = 0; c < D / 16; ++c) {
            uint4* at = reinterpret_cast<uint4*>(vl + (((p * (D / 16) + c) ^ (line & 7)) << 4));
            if (gone) {
              *at = make_uint4(0, 0, 0, 0);
              continue;
            }
            const uint4 v = *at;
            const uint32_t bad[4] = {nan_codes(v.x), nan_codes(v.y), nan_codes(v.z), nan_codes(v.w)};
            if (bad[0] | bad[1] | bad[2] | bad[3]) {
              *at = make_uint4(v.x & ~bad[0], v.y & ~bad[1], v.z & ~bad[2], v.w & ~bad[3]);
              uint32_t rows = 0;
#pragma unroll
              for (int r = 0; r < RB; ++r)
                if (tok < item_lim(b)[r]) rows |= 1u << r;
              for (int e = 0; e < 16; ++e)
                if (bad[e >> 2] >> (8 * (e & 3)) & 1u)
                  atomicOr(&poison[p * D + c * 16 + e], rows);
            }
          }
        }
      }
      fence_proxy_async_smem();
      tc_fence_before();
      mbar_arrive(bar_p);

      if (info.z & kLast) {
        // ---------------------------------------------------- the item's end
        const bool w = mbar_wait(bar_o, i & 1u, abort_flag, a.err, kDevErrTimeoutCached);
        ok = __all_sync(0xffffffffu, w) && ok;
        compute_barrier();  // all of `poison` is there
        tc_fence_after();
        // O^T: this thread's byte is column d of token half `half` of the lines
        const int half = TPL == 2 ? line >> 6 : 0, d = TPL == 2 ? line & 63 : line;
        float v[RB];
#pragma unroll
        for (int r = 0; r < RB; r += 4) read_outputs(o_col + C::col_o(half, r, 0), v + r);
        const uint32_t bits = poison[line];
        if (bits) {
#pragma unroll
          for (int r = 0; r < RB; ++r)
            if (bits >> r & 1u) v[r] = NAN;
        }
        const float sums = warp_add<RB>(l);
        if (lane % (32 / RB) == 0)
          reinterpret_cast<float*>(wmax + lane / (32 / RB))[warp - 4] = sums;
        // rows of [token half][column] in the weights' buffer, which has been read
        float* rows = reinterpret_cast<float*>(pb);
#pragma unroll
        for (int r = 0; r < RB; ++r) rows[r * 128 + line] = v[r];
        compute_barrier();
        poison[line] = 0;
        const ItemInfo it = *item_info(b);
        const bool whole = it.starts && it.ends;
        // a piece that continues an earlier CTA's item goes to slot 0, one that
        // begins here and ends elsewhere to slot 1
        float* part = a.part + ((size_t)blockIdx.x * 2 + (it.starts ? 1 : 0)) * kCachedPartFloats;
#pragma unroll
        for (int k = 0; k < (RB * D / 4 + 127) / 128; ++k) {
          const int r = (k * 128 + line) / (D / 4), c = line % (D / 4);
          if (r >= it.n_rows) break;
          float4 y = reinterpret_cast<const float4*>(rows + r * 128)[c];
          if (TPL == 2) {
            const float4 z = reinterpret_cast<const float4*>(rows + r * 128 + 64)[c];
            y = make_float4(y.x + z.x, y.y + z.y, y.z + z.z, y.w + z.w);
          }
          if (!whole) {
            reinterpret_cast<float4*>(part + r * D)[c] = y;
            continue;
          }
          const float4 w4 = wmax[r];
          const float sum = (w4.x + w4.y) + (w4.z + w4.w);
          const float inv = sum == 0.f ? 0.f : __fdividef(1.f, sum);
          *reinterpret_cast<uint2*>(a.o + item_out(b)[r] + 4 * c) =
              make_uint2(to_out<BF>(y.x * inv) | (uint32_t)to_out<BF>(y.y * inv) << 16,
                         to_out<BF>(y.z * inv) | (uint32_t)to_out<BF>(y.w * inv) << 16);
        }
        if (!whole && line < it.n_rows) {
          const float4 w4 = wmax[line];
          const float sum = (w4.x + w4.y) + (w4.z + w4.w);
          float top = 0.f;
#pragma unroll
          for (int r = 0; r < RB; ++r) top = line == r ? P_EXP - off[r] : top;
          // a row that saw nothing has no maximum
          part[kCachedPartRows * 128 + line] = sum == 0.f ? -INFINITY : top;
          part[kCachedPartRows * 129 + line] = sum;
        }
        tc_fence_before();
        mbar_arrive(bar_q_empty + 8 * b);
        compute_barrier();  // `rows`, wmax and poison may be written again
        ++items;
        if (info.z & kFinal) break;
      }
      if (++stage == ST) {
        stage = 0;
        phase ^= 1;
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, C::COLS);
  }
}

// Adds the pieces of the items that attention left in parts. Blocks (c, *) look
// after the item that CTA c began and did not end: its slot 1, then slot 0 of
// the CTAs that follow, in order. Block (c, y) has RB / 4 of its rows: first
// the pieces' weights 2^(M_k - M) and the row sum, one warp per row, then the
// weighted sums, the warps of a row taking every G-th piece.
template <int D, int RB, bool BF>
__global__ void __launch_bounds__(256) cached_join_kernel(const CachedArgs a, int ctas) {
  constexpr int NR = RB / 4;              // rows per block
  constexpr int L = D / 4;                // lanes for a row's float4
  constexpr int G = 8 / NR * (32 / L);    // piece groups
  constexpr int CHUNK = 64;               // pieces at a time
  __shared__ float weight[NR][CHUNK];
  __shared__ float4 sums[G][NR][L];
  __shared__ float inv_sum[NR];
  griddep_launch_dependents();
  griddep_wait();  // the pieces are the previous kernel's output
  const int c0 = blockIdx.x;
  if (a.meta[c0 * 4] != 2) return;
  const int seq = a.meta[c0 * 4 + 1], sub = a.meta[c0 * 4 + 2];
  const int row0 = a.cu ? a.cu[seq] : seq;
  const int fresh = a.cu ? a.cu[seq + 1] - row0 : 1;
  const int blocks = (fresh * a.group + RB - 1) / RB;
  const int head = sub / blocks, block = sub - head * blocks;
  const int n_rows = min(RB, fresh * a.group - block * RB);
  const int first_row = blockIdx.y * NR;
  if (first_row >= n_rows) return;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // the CTA that ends the item: the first behind c0 that does not pass it on
  int pieces = 2;
  for (int c = c0 + 1;; c += 32) {
    const uint32_t pass = __ballot_sync(0xffffffffu, c + lane < ctas && a.meta[(c + lane) * 4] == 4);
    if (pass != 0xffffffffu) {
      pieces = c - c0 + __ffs(~pass);
      break;
    }
  }
  pieces = min(pieces, ctas - c0);
  auto piece = [&](int k) {
    return a.part + ((size_t)(c0 + k) * 2 + (k == 0 ? 1 : 0)) * kCachedPartFloats;
  };
  // this warp's row (of the block) for the weights, the largest maximum
  const int wr = warp % NR;
  float top = -INFINITY;
  for (int k = lane; k < pieces; k += 32)
    top = fmaxf(top, piece(k)[kCachedPartRows * 128 + first_row + wr]);
  top = warp_max(top);
  const float mu = top == -INFINITY ? 0.f : top;
  const int sr = warp % NR;  // and for the sums
  const int grp = warp / NR * (32 / L) + lane / L, col = lane % L;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  float sum = 0.f;
  for (int k0 = 0; k0 < pieces; k0 += CHUNK) {
    if (warp < NR) {
      for (int k = lane; k < CHUNK; k += 32) {
        float w = 0.f;
        if (k0 + k < pieces) {
          const float* p = piece(k0 + k) + kCachedPartRows * 128 + first_row + wr;
          w = ex2_approx(p[0] - mu);
          sum = fmaf(p[kCachedPartRows], w, sum);
        }
        weight[wr][k] = w;
      }
    }
    __syncthreads();
    const int n = min(CHUNK, pieces - k0);
#pragma unroll 8
    for (int k = grp; k < n; k += G) {
      const float w = weight[sr][k];
      const float4 y = reinterpret_cast<const float4*>(piece(k0 + k) + (first_row + sr) * D)[col];
      acc.x = fmaf(y.x, w, acc.x);
      acc.y = fmaf(y.y, w, acc.y);
      acc.z = fmaf(y.z, w, acc.z);
      acc.w = fmaf(y.w, w, acc.w);
    }
    __syncthreads();
  }
  if (warp < NR) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) inv_sum[wr] = sum == 0.f ? 0.f : 1.f / sum;
  }
  sums[grp][sr][col] = acc;
  __syncthreads();
  for (int i = threadIdx.x; i < NR * L; i += 256) {
    const int rr = i / L, c = i % L, r = first_row + rr;
    if (r >= n_rows) break;
    float4 v = sums[0][rr][c];
#pragma unroll
    for (int g = 1; g < G; ++g) {
      const float4 y = sums[g][rr][c];
      v.x += y.x;
      v.y += y.y;
      v.z += y.z;
      v.w += y.w;
    }
    const float inv = inv_sum[rr];
    const int gr = block * RB + r;
    const int tok = gr / a.group, gq = gr - tok * a.group;
    uint16_t* o = a.o + (int64_t)(row0 + tok) * a.o_stride + (head * a.group + gq) * D + 4 * c;
    *reinterpret_cast<uint2*>(o) =
        make_uint2(to_out<BF>(v.x * inv) | (uint32_t)to_out<BF>(v.y * inv) << 16,
                   to_out<BF>(v.z * inv) | (uint32_t)to_out<BF>(v.w * inv) << 16);
  }
}

bool pool_map(CUtensorMap* map, const uint8_t* codes, long long lines, int box_lines) {
  cuuint64_t dims[2] = {128, (cuuint64_t)lines};
  cuuint64_t strides[1] = {128};
  cuuint32_t box[2] = {128, (cuuint32_t)box_lines};
  cuuint32_t es[2] = {1, 1};
  return encode_tiled()(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<uint8_t*>(codes), dims,
                        strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
                        CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int D, int RB, bool BF>
sam3_status_t launch_cached(sam3_ctx_t* ctx, const CUtensorMap& mk, const CUtensorMap& mv,
                            CachedArgs& a, long long capacity) {
  using C = Cfg<D, RB>;
  constexpr int variant = (RB == 4 ? 0 : RB == 8 ? 1 : 2) * 4 + (D == 128) * 2 + BF;
  sam3_status_t st = ensure_smem_attr(ctx, (uint32_t)kSmemCached << variant,
                                      cached_attn_kernel<D, RB, BF>, C::SMEM,
                                      "attention_cached smem attribute");
  if (st != SAM3_OK) return st;
  const long long blocks = ((long long)a.max_new * a.group + RB - 1) / RB;
  const long long tiles = (capacity + C::TT - 1) / C::TT;
  if ((double)blocks * a.kv_heads * a.n_seqs * (double)(tiles + ITEM_COST) > 2147483647.0)
    return set_error(ctx, SAM3_ERR_SHAPE, "attention_cached: too much work for one call");
  a.whole = tiles <= UNIT_TILES;
  const int ctas = 2 * ctx->num_sms;
  cudaError_t e = launch_pdl(cached_attn_kernel<D, RB, BF>, dim3(ctas), dim3(THREADS), C::SMEM,
                             ctx->stream, mk, mv, a);
  st = check_launch_ret(ctx, e, "cached_attn_kernel");
  if (st != SAM3_OK || a.whole) return st;  // whole items: nothing to join
  e = launch_pdl(cached_join_kernel<D, RB, BF>, dim3(ctas, 4), dim3(256), 0, ctx->stream, a, ctas);
  return check_launch_ret(ctx, e, "cached_join_kernel");
}

template <int D, bool BF>
sam3_status_t pick_rows(sam3_ctx_t* ctx, const CUtensorMap& mk, const CUtensorMap& mv,
                        CachedArgs& a, long long capacity, long long rows) {
  if (rows <= 4) return launch_cached<D, 4, BF>(ctx, mk, mv, a, capacity);
  if (rows <= 8) return launch_cached<D, 8, BF>(ctx, mk, mv, a, capacity);
  // More rows read the cache again for each 16. (32 at a time for head_dim 128: a
  // thread holds 32 scores and spills, 77 against 39 us at 16 contexts of 4000 and
  // 32 rows. 8 at a time: 46 us, and 29.6 against 27.4 at 16 rows. At head_dim 64 a
  // thread holds 32 scores with 16 rows, of two tokens, and spills 68 bytes.)
  return launch_cached<D, 16, BF>(ctx, mk, mv, a, capacity);
}

}  // namespace

sam3_status_t attention_cached(sam3_ctx_t* ctx, const sam3_kv_cache_t* c, int dtype,
                               const uint16_t* q, int64_t q_stride, const int32_t* cu_new,
                               int n_seqs, int rows, int max_new, const int32_t* table,
                               int table_stride, const int32_t* lens, int heads, float scale,
                               int causal, uint16_t* o, int64_t o_stride) {
  sam3_status_t st = check_kv_cache(ctx, c, "attention_cached");
  if (st != SAM3_OK) return st;
  if (!q || !o || !table || !lens)
    return set_error(ctx, SAM3_ERR_INVALID_ARG, "attention_cached: null pointer");
  if (dtype != SAM3_F16 && dtype != SAM3_BF16)
    return set_error(ctx, SAM3_ERR_INVALID_ARG, "attention_cached: unknown dtype %d", dtype);
  if (!aligned16(q) || !aligned16(o))
    return set_error(ctx, SAM3_ERR_INVALID_ARG, "attention_cached: rows must be 16-byte aligned");
  if (!scale_ok(scale))
    return set_error(ctx, SAM3_ERR_INVALID_ARG, "attention_cached: scale must be positive and finite");
  if (heads <= 0 || heads > 1024 || heads % c->kv_heads)
    return set_error(ctx, SAM3_ERR_SHAPE, "attention_cached: %d heads over %d K/V heads", heads,
                     c->kv_heads);
  const int64_t width = (int64_t)heads * c->head_dim;
  if (!stride_ok(q_stride, width) || !stride_ok(o_stride, width))
    return set_error(ctx, SAM3_ERR_SHAPE,
                     "attention_cached: row strides must be multiples of 8 of at least heads * "
                     "head_dim");
  const long long capacity = (long long)table_stride * c->page_size;
  const long long most = (long long)max_new * (heads / c->kv_heads);  // rows per K/V head
  if (n_seqs <= 0 || n_seqs > MAX_SEQS || rows <= 0 || max_new <= 0 || max_new > rows ||
      table_stride <= 0 || capacity > kMaxContext || most > kMaxContext ||
      (!cu_new && (max_new != 1 || rows < n_seqs)))
    return set_error(ctx, SAM3_ERR_SHAPE, "attention_cached: bad shape (at most %d sequences)",
                     MAX_SEQS);
  CachedArgs a{};
  a.group = heads / c->kv_heads;
  a.q = q;
  a.o = o;
  a.q_stride = q_stride;
  a.o_stride = o_stride;
  a.cu = cu_new;
  a.lens = lens;
  a.table = table;
  a.k_scale = c->k_scale;
  a.v_scale = c->v_scale;
  a.part = ctx->cached_part;
  a.meta = ctx->cached_meta;
  a.err = ctx->dev_err;
  a.table_stride = table_stride;
  a.num_pages = c->num_pages;
  a.page_shift = __builtin_ctz((unsigned)c->page_size);
  a.kv_heads = c->kv_heads;
  a.n_seqs = n_seqs;
  a.rows = rows;
  a.max_new = max_new;
  a.causal = causal != 0;
  a.scale_log2 = scale * kLog2E;
  const long long lines =
      (long long)c->num_pages * c->kv_heads * c->page_size * c->head_dim / 128;
  const int box = c->page_size * c->head_dim / 128;
  CUtensorMap mk, mv;
  if (!pool_map(&mk, c->k, lines, box) || !pool_map(&mv, c->v, lines, box))
    return set_error(ctx, SAM3_ERR_CUDA, "attention_cached: cuTensorMapEncodeTiled failed");
  // lengths stay on the device: the work counted here is q and o alone
  ProfScope prof(ctx, SAM3_PROF_ATTENTION, 0.0, 4.0 * rows * width);
  const bool bf = dtype == SAM3_BF16;
  if (c->head_dim == 128)
    return bf ? pick_rows<128, true>(ctx, mk, mv, a, capacity, most)
              : pick_rows<128, false>(ctx, mk, mv, a, capacity, most);
  return bf ? pick_rows<64, true>(ctx, mk, mv, a, capacity, most)
            : pick_rows<64, false>(ctx, mk, mv, a, capacity, most);
}

}  // namespace sam3

using namespace sam3;

extern "C" sam3_status_t sam3_attention_cached(
    sam3_ctx_t* ctx, const sam3_kv_cache_t* cache, int32_t dtype, const uint16_t* q,
    int64_t q_stride, const int32_t* cu_new, int32_t n_seqs, int32_t rows, int32_t max_new,
    const int32_t* page_table, int32_t table_stride, const int32_t* seq_lens, int32_t heads,
    float scale, int32_t causal, uint16_t* o, int64_t o_stride) {
  SAM3_CHECK_CTX(ctx);
  cudaSetDevice(ctx->device);
  return attention_cached(ctx, cache, dtype, q, q_stride, cu_new, n_seqs, rows, max_new, page_table,
                          table_stride, seq_lens, heads, scale, causal, o, o_stride);
}
