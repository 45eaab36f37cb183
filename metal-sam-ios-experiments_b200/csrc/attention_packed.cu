// attention_packed.cu - softmax attention over packed sequences of different
// lengths, causal or not, with grouped K/V heads, on the sm_100a tensor cores.
//
// o[i, h] = sum_j p_ij v_j / sum_j p_ij, p_ij = 2^(c q_i . k_j - m_i), c =
// scale log2(e), over the rows j of i's sequence (j <= i if causal); m_i is a
// running maximum, so one pass over the keys suffices.
//
// A query tile is 128 rows of one sequence and head; keys come in tiles of 128.
//   head_dim 64: one query tile per CTA, two CTAs per SM; S (fp32 scores, 128
//     TMEM columns), P (64) and O (64) apart, so that the next S = Q K^T runs
//     while this tile's exponentials are computed.
//   head_dim 128: two query tiles per CTA sharing K and V, one CTA per SM. Two
//     CTAs would each stream K and V: 64 KB per key tile and query tile, near
//     what L2 delivers. The two tiles are two heads of one K/V head where the
//     group is even (the same keys, the same causal length), else 256 rows of
//     one head. P takes the first half of its S's columns (TMEM is full: two S,
//     two O of 128); the next Q K^T of a tile is issued right behind the P V
//     that reads P: the tensor pipe runs one thread's MMAs in order. While one
//     tile's MMAs run, the other's softmax does.
// Warps: four of softmax per query tile, one thread per row (the row's 128
// scores to registers, maximum, exponentials, P back to TMEM), then the TMA
// producer, the MMA issuer, and two that look through V tiles (below). O is
// rescaled in place, and only when a row's maximum grew by more than 2^8. The
// issuing warp stays converged and one elected thread issues: with a lone lane
// an MMA took 87 clocks to issue, more than the 64 that one of 128 x 128 x 16
// runs (8192 causal rows, 32 heads on 8: 487 -> 440 us). Registers go to the
// softmax warps (setmaxnreg), so that nothing spills: 448 -> 435 us.
//
// Work: a tile of every sequence and head, longest first, so that the last to
// finish are short (Finder). The grid has a CTA for each, but a running CTA takes
// over the items of CTAs that are not launched yet (clusterlaunchcontrol), so
// that the next item's loads and first MMAs run under this one's last tiles: 16
// causal sequences of 17 to 2048 rows (7,445 in all, 32 heads on 8 of 128) took
// 108 us with it when the same order dealt out beforehand took 114, and four
// images' tokens with head_dim 64 took 210 when a CTA per item took 218. Results
// leave through shared memory and TMA stores, for which nobody waits.
//
// Masked places: scores become -inf in tensor memory before the tile is read,
// whatever they are. V needs more, because 0 * inf is NaN: in a sequence's last
// key tile and in the causal diagonal ones the V rows behind the sequence's end
// become 0 and, on the diagonal, so do the infinities and NaN of rows that only
// some queries see, before the MMA reads the tile; those are added to the rows
// that see them at the end (rare; read again from global memory), whatever their
// weight; in other tiles the MMA multiplies, and 0 times an infinity is NaN.
//
// P is rounded to the inputs' type (kind::f16 takes both operands in one): half
// a step (fp16 2^-11, bf16 2^-8) of each weight. fp16 ends at 2^-24, so its
// weights are 2^7 at the running maximum, and at most 2^15 before O is rescaled:
// a weight keeps its 11 bits down to 2^-21 of its row's largest and is held to
// within 2^-32 of that below (at 1 it would be 2^-14 and 2^-25, and thousands of
// light keys beside a heavy one come out 17 % off).
//
// Bounds, measured. head_dim 64: the exponentials (16 per clock and SM; packed
// FMAs and additions beside them leave them 90 % of it). Four images' tokens
// (2592, 1733, 5184 and 901 rows, 16 heads): 210 us, 731 TFLOP/s, where the
// exponentials alone need 133 us and the MMAs 94. head_dim 128: exponentials
// and MMAs need about the same time (1024 clocks each for a 128 x 128 tile), and
// the chain from a tile's scores through its softmax to its next scores has only
// one other tile beside it: 8192 causal rows, 32 heads on 8, 435 us, 1265
// TFLOP/s, 77 % of cuBLAS's burst rate; under load for seconds the power limit
// holds it to 1070. Tried and no faster at head_dim 128: P told in two parts
// (96 + 32 keys 446, 64 + 64 449 against 444 us), K and V looked at between P V
// and Q K^T (453), an issuer that polls for whatever is ready, a part of the
// exponentials as polynomials (the last two while a lone lane still issued).
#include <algorithm>

#include "common.cuh"
#include "internal.h"

#include <cuda_bf16.h>

namespace sam3 {
namespace {

constexpr int BQ = 128, BKV = 128;
constexpr int KST = 2, VST = 2;  // K and V tiles in shared memory

template <int D>
struct PK {
  static constexpr int T = D == 128 ? 2 : 1;     // query tiles per CTA
  static constexpr bool OVERLAY = D == 128;      // P in its S's columns
  static constexpr int HALVES = D / 64;          // 128-byte wide parts of a tile
  // Warps: four of softmax per tile, then a warpgroup of others. The registers of
  // the launch (2 x 256 x 128 or 384 x 168 per SM) are split among them.
  static constexpr int PRODUCER = 4 * T, ISSUER = 4 * T + 1, CHECKER = 4 * T + 2;
  static constexpr int THREADS = 128 * (T + 1);
  static constexpr int REGS = D == 128 ? 208 : 192, REGS_OTHERS = D == 128 ? 88 : 64;
  static constexpr int TILE = BKV * D * 2;       // bytes of a Q, K or V tile
  static constexpr int HALF = BKV * 128;
  static constexpr int OFF_K = T * TILE;
  static constexpr int OFF_V = OFF_K + KST * TILE;
  static constexpr int OFF_OUT = OFF_V + VST * TILE;  // [T] 128 rows of 64 outputs
  static constexpr int OFF_BAR = OFF_OUT + T * HALF;
  static constexpr int BARS = 4 * T + 2 * KST + 2 * VST + 11;
  static constexpr int OFF_MISC = (OFF_BAR + BARS * 8 + 15) / 16 * 16;
  static constexpr int EMPTY = 8;  // CTAs without work that are taken over at a time
  static constexpr int MISC = 176 + 16 * EMPTY;
  static constexpr int SMEM = OFF_MISC + MISC + 1024;
  static constexpr uint32_t COLS = D == 128 ? 512 : 256;
  static constexpr uint32_t S(int t) { return 128u * t; }
  static constexpr uint32_t P(int t) { return OVERLAY ? 128u * t : 128u; }
  static constexpr uint32_t O(int t) { return OVERLAY ? 256u + 128u * t : 192u; }
};
static_assert(2 * (PK<64>::SMEM + 1024) <= 228 * 1024 && 3 * PK<64>::SMEM > 228 * 1024,
              "exactly two CTAs per SM: 256 TMEM columns each");
static_assert(PK<128>::SMEM <= 227 * 1024 && 2 * PK<128>::SMEM > 228 * 1024, "one CTA per SM");

struct PackedArgs {
  uint16_t* o;
  const uint16_t* v;
  const int32_t* cu;
  int* err;
  int64_t o_stride, v_stride;
  int n_seqs, rows, group;
  int pair_heads;  // the CTA's two tiles are two heads (else 256 rows of one)
  int units;       // heads, or pairs of heads
  unsigned resident;  // CTAs that run at once
  int causal;
  float c;         // scale * log2(e)
};

struct Item {
  int row0, len, tile, unit;  // tile < 0: no more
};

__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
template <bool BF>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  if (BF) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  return pack_half2(lo, hi);
}
// 0xFFFF in each half of w that is an infinity or NaN.
template <bool BF>
__device__ __forceinline__ uint32_t not_finite(uint32_t w) {
  constexpr uint32_t E = BF ? 0x7F807F80u : 0x7C007C00u;
  return __vcmpeq2(w & E, E);
}

// The tiles of `span` rows of all sequences, in the order they are worked on:
// those with the most keys first, so that the last ones to finish are short (a
// causal tile's keys grow with its place in the sequence, another's with its
// sequence). Up to 4 sequences per lane of the warp are kept in registers and a
// tile is found by bisection over its key count; with more sequences the tiles
// come sequence by sequence, from the last backwards, 32 sequences at a time. A
// CTA's numbers grow, so the search goes on where it was: searched for from the
// end each time, 1000 sequences cost some 15 us per item.
struct Finder {
  static constexpr int KEEP = 4;
  int row0[KEEP], len[KEEP], tiles[KEEP];
  int span, most;
  int total;     // tiles, known once find has found none
  int at, seen;  // the 32 sequences that are looked at (the first; -1: none), tiles before

  __device__ __forceinline__ int load(const PackedArgs& a, int i, int& r0, int& n) const {
    r0 = n = 0;
    if (i < 0 || i >= a.n_seqs) return 0;
    r0 = a.cu[i];
    const int r1 = a.cu[i + 1];
    if (!rows_fit(r0, r1, a.rows)) {
      report_bad_index(a.err, kDevErrBadLengths);
      r0 = 0;
      return 0;
    }
    n = r1 - r0;
    return (n + span - 1) / span;
  }
  __device__ __forceinline__ void init(const PackedArgs& a, int span_) {
    span = span_;
    most = 0;
    at = -1;
    if (a.n_seqs > 32 * KEEP) return;
#pragma unroll
    for (int k = 0; k < KEEP; ++k) {
      tiles[k] = 32 * k < a.n_seqs ? load(a, 32 * k + (threadIdx.x & 31), row0[k], len[k]) : 0;
      most = max(most, tiles[k]);
    }
    most = __reduce_max_sync(0xffffffffu, most);
  }
  // tiles with at least `keys` key tiles
  __device__ __forceinline__ int at_least(bool causal, int keys) const {
    int n = 0;
#pragma unroll
    for (int k = 0; k < KEEP; ++k)
      n += causal ? max(0, tiles[k] - keys + 1) : tiles[k] >= keys ? tiles[k] : 0;
    return __reduce_add_sync(0xffffffffu, n);
  }
  __device__ __forceinline__ Item find(const PackedArgs& a, int number) {
    const int lane = threadIdx.x & 31;
    if (a.n_seqs <= 32 * KEEP) {
      int lo = 0, hi = most;  // the largest count with more than `number` tiles at or above it
      while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (at_least(a.causal, mid) > number)
          lo = mid;
        else
          hi = mid - 1;
      }
      if (lo == 0) {
        total = at_least(a.causal, 1);
        return {0, 0, -1, 0};
      }
      int rank = number - at_least(a.causal, lo + 1), tile = lo - 1;
      if (!a.causal) {
        tile = rank % lo;
        rank /= lo;
      }
#pragma unroll
      for (int k = 0; k < KEEP; ++k) {
        const bool in = a.causal ? tiles[k] >= lo : tiles[k] == lo;
        const uint32_t set = __ballot_sync(0xffffffffu, in);
        const int n = __popc(set);
        if (rank < n) {
          const uint32_t hit =
              __ballot_sync(0xffffffffu, in && __popc(set & ((1u << lane) - 1)) == rank);
          const int l = __ffs(hit) - 1;
          return {__shfl_sync(0xffffffffu, row0[k], l), __shfl_sync(0xffffffffu, len[k], l), tile, 0};
        }
        rank -= n;
      }
      return {0, 0, -1, 0};
    }
    auto look = [&]() {  // tiles[0]: of the lanes up to this one; lane 0 has the last sequence
      tiles[0] = load(a, at + 31 - lane, row0[0], len[0]);
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, tiles[0], o);
        if (lane >= o) tiles[0] += u;
      }
    };
    if (at < 0 || number < seen) {
      at = (a.n_seqs - 1) / 32 * 32;
      seen = 0;
      look();
    }
    for (;;) {
      const uint32_t hit = __ballot_sync(0xffffffffu, seen + tiles[0] > number);
      if (hit) {
        const int l = __ffs(hit) - 1;
        return {__shfl_sync(0xffffffffu, row0[0], l), __shfl_sync(0xffffffffu, len[0], l),
                seen + __shfl_sync(0xffffffffu, tiles[0], l) - 1 - number, 0};
      }
      seen += __shfl_sync(0xffffffffu, tiles[0], 31);
      at -= 32;
      if (at < 0) break;
      look();
    }
    total = seen;
    return {0, 0, -1, 0};
  }
};

// What an item means to a CTA: per query tile its head, first row in the
// sequence and key tiles.
struct Work {
  int row0, len, head0, kv_head, qt[2], n[2], nmax;
  bool ph;
};
template <int T>
__device__ __forceinline__ Work work_of(const PackedArgs& a, const Item& it) {
  Work w;
  w.row0 = it.row0;
  w.len = it.len;
  w.ph = T == 2 && a.pair_heads;
  w.head0 = w.ph ? 2 * it.unit : it.unit;
  w.kv_head = w.head0 / a.group;
  w.qt[0] = T == 2 && !w.ph ? it.tile * 256 : it.tile * 128;
  w.qt[1] = w.ph ? w.qt[0] : w.qt[0] + 128;
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    const int keys = a.causal ? min(w.len, w.qt[t] + BQ) : w.len;
    w.n[t] = t < T && w.qt[t] < w.len ? (keys + BKV - 1) / BKV : 0;
  }
  w.nmax = max(w.n[0], w.n[1]);
  return w;
}
// Tile c of a stream through a ring of N stages.
template <int N>
struct Ring {
  int st = 0;
  uint32_t ph = 0;
  __device__ __forceinline__ void step() {
    if (++st == N) {
      st = 0;
      ph ^= 1;
    }
  }
};

template <int D, bool BF>
__global__ void __launch_bounds__(PK<D>::THREADS, D == 128 ? 1 : 2)
    packed_attn_kernel(const __grid_constant__ CUtensorMap map_q,
                       const __grid_constant__ CUtensorMap map_k,
                       const __grid_constant__ CUtensorMap map_v,
                       const __grid_constant__ CUtensorMap map_o, const PackedArgs a) {
  using C = PK<D>;
  constexpr int T = C::T;
  constexpr uint32_t FMT = BF ? (1u << 7) | (1u << 10) : 0u;  // bf16 operands
  constexpr uint32_t IDESC_S = umma_idesc_f16(128, BKV, 0) | FMT;
  constexpr uint32_t IDESC_O = umma_idesc_f16(128, D, 1) | FMT;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  const uint32_t sbase = smem_u32(smem);
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;

  const uint32_t bar_item = sbase + C::OFF_BAR;  // [2] an item is told
  const uint32_t bar_item_free = bar_item + 16;     // [2] and done with
  const uint32_t bar_q = bar_item_free + 16;        // [T] queries are there
  const uint32_t bar_q_free = bar_q + 8 * T;        // the item's last Q K^T is done
  const uint32_t bar_k_full = bar_q_free + 8;
  const uint32_t bar_k_empty = bar_k_full + 8 * KST;
  const uint32_t bar_v_full = bar_k_empty + 8 * KST;
  const uint32_t bar_v_empty = bar_v_full + 8 * VST;
  const uint32_t bar_v_raw = bar_v_empty + 8 * VST;  // a V tile to look through before its use
  const uint32_t bar_s_full = bar_v_raw + 8;         // [T] Q K^T done (and the P V before it)
  const uint32_t bar_s_free = bar_s_full + 8 * T;    // scores are in registers (P apart)
  const uint32_t bar_p_full = bar_s_free + 8;        // [T] P written
  const uint32_t bar_o_full = bar_p_full + 8 * T;    // P V done (P apart)
  const uint32_t bar_o_done = bar_o_full + 8;        // [T] after an item's last P V
  const uint32_t bar_drain = bar_o_done + 8 * T;
  const uint32_t bar_raw_free = bar_drain + 8;       // the checkers may take the next
  const uint32_t bar_next = bar_raw_free + 8;        // which CTA's item comes next
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + C::OFF_MISC);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + C::OFF_MISC + 4);
  // [2] items; of each the V tiles looked through and the rows with infinities
  Item* items = reinterpret_cast<Item*>(smem + C::OFF_MISC + 16);
  int* fix_tile = reinterpret_cast<int*>(smem + C::OFF_MISC + 48);            // [2][2]
  uint32_t* fix_rows = reinterpret_cast<uint32_t*>(smem + C::OFF_MISC + 64);  // [2][2][4]
  // the V tile to look through: stage (-1: no more), rows of the sequence in it,
  // whether some query sees a part of it only, its place in fix_tile, its number
  volatile int* raw = reinterpret_cast<volatile int*>(smem + C::OFF_MISC + 128);
  volatile int* progress = raw + 5;  // key tiles that the producer has passed on
  const uint32_t next_slot = sbase + C::OFF_MISC + 160;  // the answer of cta_try_cancel
  const uint32_t empty_slots = next_slot + 16;           // [EMPTY] such

  if (warp == C::PRODUCER && lane == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(bar_item + 8 * i, 1);
      mbar_init(bar_item_free + 8 * i, 1 + 4 * T);  // the issuer and the softmax warps
    }
    mbar_init(bar_q_free, 1);
    for (int t = 0; t < T; ++t) {
      mbar_init(bar_q + 8 * t, 1);
      mbar_init(bar_s_full + 8 * t, 1);
      mbar_init(bar_p_full + 8 * t, 128);
      mbar_init(bar_o_done + 8 * t, 1);
    }
    for (int s = 0; s < KST; ++s) {
      mbar_init(bar_k_full + 8 * s, 1);
      mbar_init(bar_k_empty + 8 * s, 1);
    }
    for (int s = 0; s < VST; ++s) {
      mbar_init(bar_v_full + 8 * s, 1);
      mbar_init(bar_v_empty + 8 * s, 1);
    }
    mbar_init(bar_v_raw, 1);
    mbar_init(bar_s_free, 128);
    mbar_init(bar_o_full, 1);
    mbar_init(bar_drain, 1);
    mbar_init(bar_raw_free, 1);
    mbar_init(bar_next, 1);
    *abort_flag = 0;
    *progress = 0;
    fence_mbar_init();
    prefetch_tmap(&map_q);
    prefetch_tmap(&map_k);
    prefetch_tmap(&map_v);
    prefetch_tmap(&map_o);
  }
  // The producer does not wait for the allocation: it finds its first item and
  // starts its loads meanwhile.
  uint32_t tmem = 0;
  if (warp == C::PRODUCER) {
    __syncwarp();
    asm volatile("barrier.cta.arrive 1, %0;" ::"n"(C::THREADS) : "memory");
  } else {
    if (warp == C::ISSUER) {
      tmem_alloc(smem_u32(tmem_slot), C::COLS);
      tmem_relinquish();
    }
    tc_fence_before();
    asm volatile("barrier.cta.sync 1, %0;" ::"n"(C::THREADS) : "memory");
    tc_fence_after();
    tmem = *tmem_slot;
    // Behind the allocation, as the next kernel allocates too; so not by the
    // producer, which does not wait for it (one thread speaks for its CTA).
    griddep_launch_dependents();
  }
  griddep_wait();  // offsets and rows may be earlier kernels' outputs

  // Looks through a V tile before the MMA reads it (by 64 threads, `id` among
  // them): rows behind the sequence's end become 0, and so do infinities and NaN
  // on the diagonal, whose rows are noted.
  auto carry = [](uint32_t w) {
    return BF ? (w & 0x7F807F80u) + 0x00800080u : (w & 0x7C007C00u) + 0x04000400u;
  };
  auto look_through = [&](int st, int held, bool diag, int nth, int id) {
    constexpr int threads = 64;
    uint4* vt = reinterpret_cast<uint4*>(smem + C::OFF_V + st * C::TILE);
    for (int h = 0; h < C::HALVES; ++h)
      for (int e = held * 8 + id; e < BKV * 8; e += threads)
        vt[h * BKV * 8 + e] = make_uint4(0, 0, 0, 0);
    if (diag) {
      uint32_t found = 0;  // an exponent of ones and 1 carry into the sign bit
#pragma unroll 8
      for (int e = id; e < C::TILE / 16; e += threads) {
        const uint4 x = vt[e];
        found |= carry(x.x) | carry(x.y) | carry(x.z) | carry(x.w);
      }
      if (found & 0x80008000u)
        for (int e = id; e < C::TILE / 16; e += threads) {
          const int r = (e >> 3) & (BKV - 1);
          const uint4 x = vt[e];
          const uint4 b = make_uint4(not_finite<BF>(x.x), not_finite<BF>(x.y), not_finite<BF>(x.z),
                                     not_finite<BF>(x.w));
          if (b.x | b.y | b.z | b.w) {
            vt[e] = make_uint4(x.x & ~b.x, x.y & ~b.y, x.z & ~b.z, x.w & ~b.w);
            atomicOr(&fix_rows[nth * 4 + (r >> 5)], 1u << (r & 31));
          }
        }
    }
    fence_proxy_async_smem();
  };

  if (warp >= 4 * T) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(C::REGS_OTHERS));
    if (warp == C::PRODUCER) {
      // ----------------------------------------------------------- producer
      Finder finder;
      finder.init(a, T == 2 && !a.pair_heads ? 256 : 128);
      uint32_t k_bits = 0, k_par = 0, v_bits = 0, v_par = 0;  // loads to drain on abort
      uint32_t raw_uses = 0, q_par = 0, asked = 0;
      int passed = 0;  // key tiles
      Ring<KST> rk;
      Ring<VST> rv;
      bool ok = true;
      // The first item is the CTA's own, the next ones those of CTAs that are then
      // never launched: where all run at once there is nothing to take over.
      bool others = gridDim.x > a.resident, outstanding = false;
      int held = -1;  // numbers taken over and not yet worked on, one per lane
      auto ask = [&](int n, uint32_t slots) {
        if (lane == 0) mbar_arrive_expect_tx(bar_next, 16 * n);
        __syncwarp();
        if (lane < n) cta_try_cancel(slots + 16 * lane, bar_next);
        ++asked;
      };
      auto answered = [&](int n, uint32_t slots) {  // numbers in `held`
        ok = __all_sync(0xffffffffu, mbar_wait(bar_next, (asked - 1) & 1u, abort_flag, a.err,
                                               kDevErrTimeoutPacked));
        if (!ok) return;
        held = lane < n ? cta_cancelled(slots + 16 * lane) : -1;
        __syncwarp();
        // nothing may be asked for once a refusal has been seen
        others = !__any_sync(0xffffffffu, lane < n && held < 0);
      };
      auto held_set = [&]() { return __ballot_sync(0xffffffffu, held >= 0); };
      for (uint32_t i = 0; ok; ++i) {
        Item it{0, 0, -1, 0};
        int number = -1;
        for (bool own = i == 0;; own = false) {
          if (outstanding) {
            outstanding = false;
            answered(1, next_slot);
            if (!ok) break;
          }
          number = blockIdx.x;
          if (!own) {
            const uint32_t set = held_set();
            if (!set) break;
            const int l = __ffs(set) - 1;
            number = __shfl_sync(0xffffffffu, held, l);
            if (lane == l) held = -1;
          }
          it = finder.find(a, number / a.units);
          if (it.tile >= 0) break;
          // A number behind the last tile (the grid is an upper bound), as a rule like
          // all that are not launched yet. They are done away with several at a time
          // (one by one: 334 against 184 us for 1000 sequences of 1 to 80 rows).
          while (ok && others && !held_set()) {
            ask(C::EMPTY, empty_slots);
            answered(C::EMPTY, empty_slots);
            if (held >= 0 && held / a.units >= finder.total) held = -1;
          }
          if (!ok) break;
        }
        if (!ok) break;
        it.unit = number % a.units;
        const int slot = i & 1;
        ok = __all_sync(0xffffffffu, mbar_wait(bar_item_free + 8 * slot, (i >> 1 & 1) ^ 1,
                                               abort_flag, a.err, kDevErrTimeoutPacked));
        if (!ok) break;
        if (lane == 0) items[slot] = it;
        if (lane < 2) fix_tile[slot * 2 + lane] = 0;
        if (lane < 8) fix_rows[slot * 8 + lane] = 0;
        __syncwarp();
        if (lane == 0) mbar_arrive(bar_item + 8 * slot);
        if (it.tile < 0) break;
        const Work w = work_of<T>(a, it);
        if (lane == 0) {
          ok = mbar_wait(bar_q_free, (i & 1) ^ 1, abort_flag, a.err, kDevErrTimeoutPacked);
          for (int t = 0; t < T && ok; ++t) {
            if (!w.n[t]) {  // nothing to load, but a phase like every item's
              mbar_arrive(bar_q + 8 * t);
              continue;
            }
            mbar_arrive_expect_tx(bar_q + 8 * t, C::TILE);
            tma_load_3d(sbase + t * C::TILE, &map_q, bar_q + 8 * t, 0, w.row0 + w.qt[t],
                        (w.ph ? w.head0 + t : w.head0) * C::HALVES);
          }
          if (ok) q_par = i + 1;
        }
        int fixes = 0;
        ok = __shfl_sync(0xffffffffu, (int)ok, 0) != 0;
        for (int j = 0; j < w.nmax && ok; ++j) {
          // no earlier than the answer is needed, two tiles before the item's last MMA:
          // until then it may fall to a CTA that is done before
          if (j == w.nmax - 1 && others && !held_set()) {
            ask(1, next_slot);
            outstanding = true;
          }
          // does some query of the CTA see a part of this tile only?
          const bool diag = a.causal && (j == w.n[0] - 1 || j == w.n[1] - 1);
          const bool fix = diag || (j + 1) * BKV > w.len;
          if (lane == 0) {
            ok = mbar_wait(bar_k_empty + 8 * rk.st, rk.ph ^ 1, abort_flag, a.err,
                           kDevErrTimeoutPacked);
            if (ok) {
              mbar_arrive_expect_tx(bar_k_full + 8 * rk.st, C::TILE);
              tma_load_3d(sbase + C::OFF_K + rk.st * C::TILE, &map_k, bar_k_full + 8 * rk.st, 0,
                          w.row0 + j * BKV, w.kv_head * C::HALVES);
              k_bits |= 1u << rk.st;
              k_par = (k_par & ~(1u << rk.st)) | (rk.ph << rk.st);
              ok = mbar_wait(bar_v_empty + 8 * rv.st, rv.ph ^ 1, abort_flag, a.err,
                             kDevErrTimeoutPacked);
            }
            if (ok && fix) {
              ok = mbar_wait(bar_raw_free, (raw_uses & 1u) ^ 1, abort_flag, a.err,
                             kDevErrTimeoutPacked);
              raw[0] = rv.st;
              raw[1] = w.len - j * BKV;
              raw[2] = diag | (slot * 2 + fixes) << 1;  // at most two such tiles per item
              raw[3] = j;
            }
            if (ok) {
              const uint32_t bar = fix ? bar_v_raw : bar_v_full + 8 * rv.st;
              mbar_arrive_expect_tx(bar, C::TILE);
              tma_load_3d(sbase + C::OFF_V + rv.st * C::TILE, &map_v, bar, 0, w.row0 + j * BKV,
                          w.kv_head * C::HALVES);
              if (!fix) {
                v_bits |= 1u << rv.st;
                v_par = (v_par & ~(1u << rv.st)) | (rv.ph << rv.st);
              } else {
                v_bits &= ~(1u << rv.st);
              }
            }
          }
          ok = __shfl_sync(0xffffffffu, (int)ok, 0) != 0;
          if (ok && fix) {
            ++raw_uses;
            ++fixes;
          }
          if (lane == 0) *progress = ++passed;
          rk.step();
          rv.step();
        }
      }
      if (ok && lane == 0 &&
          mbar_wait(bar_raw_free, (raw_uses & 1u) ^ 1, abort_flag, a.err, kDevErrTimeoutPacked)) {
        raw[0] = -1;  // the checkers may go
        mbar_arrive(bar_v_raw);
      }
      if (lane == 0 && *abort_flag) {
        if (asked) mbar_wait_drain(bar_next, (asked - 1) & 1u);
        if (raw_uses) mbar_wait_drain(bar_v_raw, (raw_uses - 1) & 1u);
        for (int t = 0; t < T; ++t)
          if (q_par) mbar_wait_drain(bar_q + 8 * t, (q_par - 1) & 1u);
        for (int s = 0; s < KST; ++s)
          if (k_bits & (1u << s)) mbar_wait_drain(bar_k_full + 8 * s, (k_par >> s) & 1u);
        for (int s = 0; s < VST; ++s)
          if (v_bits & (1u << s)) mbar_wait_drain(bar_v_full + 8 * s, (v_par >> s) & 1u);
      }
    } else if (warp == C::ISSUER) {
      // ----------------------------------------------------------- MMA issuer
      // The whole warp runs this and one elected thread issues, so that what the MMAs
      // take (descriptors, columns) is uniform to the compiler.
      bool ok = true, issued = false;
      auto wait = [&](uint32_t bar, uint32_t par) {
        return __all_sync(0xffffffffu,
                          mbar_wait(bar, par, abort_flag, a.err, kDevErrTimeoutPacked)) != 0;
      };
      Ring<KST> rk;   // of the next Q K^T
      Ring<VST> rv;   // of the next P V
      uint32_t n_p[2] = {0, 0};  // P tiles waited for
      uint32_t n_s = 0;          // S tiles issued (P apart)
      const uint64_t desc_q = umma_desc_sw128(sbase), desc_k = umma_desc_sw128(sbase + C::OFF_K);
      // V tile: keys along K, head_dim along N in 64-wide groups HALF apart
      const uint64_t desc_v = (umma_desc_sw128_mn(sbase + C::OFF_V) & ~(0x3FFFull << 16)) |
                              ((uint64_t)(C::HALF >> 4) << 16);
      for (uint32_t i = 0; ok; ++i) {
        ok = wait(bar_item + 8 * (i & 1), i >> 1 & 1);
        if (!ok) break;
        const Item it = items[i & 1];
        const Work w = work_of<T>(a, it);
        const bool none = __shfl_sync(0xffffffffu, it.tile, 0) < 0;
        const int n0 = __shfl_sync(0xffffffffu, w.n[0], 0);
        const int n1 = __shfl_sync(0xffffffffu, w.n[1], 0);
        const int nmax = max(n0, n1);
        if (lane == 0) mbar_arrive(bar_item_free + 8 * (i & 1));
        if (none) break;
        auto last_of = [&](int j) { return T == 2 && j < n1 ? 1 : 0; };
        auto issue_qk = [&](int t, int j) {
          const uint64_t dq = desc_advance(desc_q, t * C::TILE);
          const uint64_t dk = desc_advance(desc_k, rk.st * C::TILE);
          const bool last = t == last_of(j);
          if (elect_one()) {
#pragma unroll
            for (int kk = 0; kk < D / 16; ++kk) {
              const uint32_t off = (kk / 4) * C::HALF + (kk % 4) * 32;
              umma_f16_ss(tmem + C::S(t), desc_advance(dq, off), desc_advance(dk, off), IDESC_S,
                          kk != 0);
            }
            umma_commit(bar_s_full + 8 * t);
            if (last) umma_commit(bar_k_empty + 8 * rk.st);
            if (last && j == nmax - 1) umma_commit(bar_q_free);
          }
          issued = true;
          if (last) rk.step();
        };
        auto issue_pv = [&](int t, int j) {
          const uint64_t dv = desc_advance(desc_v, rv.st * C::TILE);
          const bool last = t == last_of(j);
          if (elect_one()) {
#pragma unroll
            for (int kk = 0; kk < BKV / 16; ++kk)
              umma_f16_ts(tmem + C::O(t), tmem + C::P(t) + kk * 8, desc_advance(dv, kk * 2048),
                          IDESC_O, (j | kk) != 0);
            if (!C::OVERLAY) umma_commit(bar_o_full);
            if (last) umma_commit(bar_v_empty + 8 * rv.st);
            if (j == (t ? n1 : n0) - 1) umma_commit(bar_o_done + 8 * t);
          }
          if (last) rv.step();
        };
        ok = wait(bar_q, i & 1) && wait(bar_k_full + 8 * rk.st, rk.ph);
        if (C::OVERLAY) {
          if (ok) {
            tc_fence_after();
            issue_qk(0, 0);
            if (n1) {
              ok = wait(bar_q + 8 * (T - 1), i & 1);
              if (ok) issue_qk(1, 0);
            }
          }
          for (int j = 0; j < nmax && ok; ++j) {
            bool v_here = false, k_here = false;
#pragma unroll
            for (int t = 0; t < T; ++t) {
              const int n = t ? n1 : n0;
              if (j >= n || !ok) continue;
              // V and the next K are early as a rule: their waits come first, so that
              // nothing stands between P and its MMAs
              const bool more = j + 1 < n;
              ok = (v_here || wait(bar_v_full + 8 * rv.st, rv.ph)) &&
                   (!more || k_here || wait(bar_k_full + 8 * rk.st, rk.ph));
              v_here = true;
              k_here |= more;
              ok = ok && wait(bar_p_full + 8 * t, n_p[t]++ & 1u);
              if (!ok) continue;
              tc_fence_after();
              issue_pv(t, j);
              if (more) issue_qk(t, j + 1);
            }
          }
        } else {
          // S is free once the softmax has read the tile before
          auto next_s = [&](int j) {
            ok = wait(bar_k_full + 8 * rk.st, rk.ph) &&
                 (n_s == 0 || wait(bar_s_free, (n_s - 1) & 1u));
            if (!ok) return;
            tc_fence_after();
            issue_qk(0, j);
            ++n_s;
          };
          if (ok) next_s(0);
          if (ok && nmax > 1) next_s(1);
          for (int j = 0; j < nmax && ok; ++j) {
            ok = wait(bar_p_full, n_p[0]++ & 1u) && wait(bar_v_full + 8 * rv.st, rv.ph);
            if (!ok) break;
            tc_fence_after();
            issue_pv(0, j);
            if (j + 2 < nmax) next_s(j + 2);
          }
        }
      }
      if (__any_sync(0xffffffffu, *abort_flag) && issued) {
        if (elect_one()) umma_commit(bar_drain);
        mbar_wait_drain(bar_drain, 0);
      }
    } else {
      // ----------------------------------------------------------- V tiles
      const int id = threadIdx.x - 32 * C::CHECKER;
      // Such a tile may never come: without a mask, and with whole tiles, the two
      // warps wait until the CTA's last item.
      for (uint32_t u = 0;; ++u) {
        const bool there =
            __all_sync(0xffffffffu, mbar_wait_idle(bar_v_raw, u & 1u, abort_flag, progress, a.err,
                                                   kDevErrTimeoutPacked));
        if (id == 0) raw[4] = there;  // one decision for both warps
        asm volatile("barrier.cta.sync 3, 64;" ::: "memory");
        const int st = raw[0], held = raw[1], flags = raw[2], j = raw[3];
        const bool go = raw[4] && st >= 0;
        asm volatile("barrier.cta.sync 3, 64;" ::: "memory");
        if (!go) break;
        if (id == 0) fix_tile[flags >> 1] = j;
        look_through(st, held, flags & 1, flags >> 1, id);
        asm volatile("barrier.cta.sync 3, 64;" ::: "memory");
        if (id == 0) {
          mbar_arrive(bar_v_full + 8 * st);
          mbar_arrive(bar_raw_free);
        }
      }
    }
  } else {
    // ----------------------------------------------------------- softmax rows
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(C::REGS));
    constexpr float kRescaleLog2 = 8.0f;
    constexpr float kTopLog2 = BF ? 0.f : 7.f;  // the weight at the running maximum
    const int t = T == 2 ? warp >> 2 : 0;
    const int quad = warp & 3;  // this warp's TMEM lane quadrant
    const int r = quad * 32 + lane;
    const uint32_t lane_base = tmem + ((uint32_t)(quad * 32) << 16);
    const uint32_t s_col = lane_base + C::S(t), p_col = lane_base + C::P(t),
                   o_col = lane_base + C::O(t);
    const float c = a.c;
    auto wait = [&](uint32_t bar, uint32_t par) {
      return __all_sync(0xffffffffu, mbar_wait(bar, par, abort_flag, a.err, kDevErrTimeoutPacked));
    };
    uint8_t* out = smem + C::OFF_OUT + t * C::HALF + quad * 4096;  // this warp's rows of 64 outputs
    uint32_t tiles = 0, outs = 0;  // key tiles and items of this query tile so far
    for (uint32_t i = 0;; ++i) {
      if (!wait(bar_item + 8 * (i & 1), i >> 1 & 1)) break;
      // What the key loop needs of the item and no more: its registers are scarce.
      // The item is read again for its end.
      auto item = [&]() {
        const volatile Item& s = items[i & 1];
        return Item{s.row0, s.len, s.tile, s.unit};
      };
      int n, lim, lim_min;
      {
        const Item it = item();
        if (it.tile < 0) break;
        const Work w = work_of<T>(a, it);
        const int q0 = T == 2 && t ? w.qt[1] : w.qt[0];
        n = T == 2 && t ? w.n[1] : w.n[0];
        lim = a.causal ? min(w.len, q0 + r + 1) : w.len;    // keys that the row sees
        lim_min = a.causal ? min(w.len, q0 + 1) : w.len;    // that all rows of the tile see
      }
      // Not -inf: while a row's scores are all -inf (keys that hold infinities) its
      // weights are 0, not 2^(-inf + inf).
      float m_run = -3.402823466e38f, l_run = 0.f;
      bool ok = true;
      for (int j = 0; j < n; ++j, ++tiles) {
        ok = wait(bar_s_full + 8 * t, tiles & 1u);
        if (!ok) break;
        tc_fence_after();
        // Masked scores become -inf in tensor memory, so that the code below is the
        // same for all tiles.
        if ((j + 1) * BKV > lim_min) {
          const int valid = lim - j * BKV;
#pragma unroll 1
          for (int g = __reduce_min_sync(0xffffffffu, valid) >> 5; g < BKV / 32; ++g) {
            uint32_t s[32];
            tmem_ld_32x32b_x32(s_col + 32 * g, s);
            tmem_wait_ld();
#pragma unroll
            for (int e = 0; e < 32; ++e)
              if (32 * g + e >= valid) s[e] = __float_as_uint(-INFINITY);
#pragma unroll
            for (int q = 0; q < 2; ++q)
              tmem_st_32x32b_x16(s_col + 32 * g + 16 * q,
                                 *reinterpret_cast<uint32_t(*)[16]>(s + 16 * q));
          }
          tmem_wait_st();
        }
        uint32_t v[BKV];
        float mx[4];
        auto half_max = [&](int h0) {
#pragma unroll
          for (int q = h0; q < h0 + 2; ++q) {
            float m = fmaxf(__uint_as_float(v[32 * q]), __uint_as_float(v[32 * q + 31]));
#pragma unroll
            for (int e = 1; e < 31; e += 2)
              m = max3(m, __uint_as_float(v[32 * q + e]), __uint_as_float(v[32 * q + e + 1]));
            mx[q] = m;
          }
        };
        tmem_ld_32x32b_x32(s_col, *reinterpret_cast<uint32_t(*)[32]>(v));
        tmem_ld_32x32b_x32(s_col + 32, *reinterpret_cast<uint32_t(*)[32]>(v + 32));
        tmem_wait_ld();
        tmem_ld_32x32b_x32(s_col + 64, *reinterpret_cast<uint32_t(*)[32]>(v + 64));
        tmem_ld_32x32b_x32(s_col + 96, *reinterpret_cast<uint32_t(*)[32]>(v + 96));
        half_max(0);
        tmem_wait_ld();
        if (!C::OVERLAY) {
          tc_fence_before();
          mbar_arrive(bar_s_free);  // the next Q K^T may overwrite S now
        }
        half_max(2);
        const float m_tile = max3(fmaxf(mx[0], mx[1]), mx[2], mx[3]) * c;
        const bool grow = m_tile > m_run + kRescaleLog2;
        const float m_use = grow ? m_tile : m_run;
        const float alpha = grow ? ex2_approx(m_run - m_use) : 1.0f;  // 0 on the first tile
        const float to = kTopLog2 - m_use;
        float2 ls[2] = {{0.f, 0.f}, {0.f, 0.f}};
        uint32_t pk[BKV / 2];
#pragma unroll
        for (int e = 0; e < BKV / 2; ++e) {
          // pairs: a warp alone does 128 exponentials with them in 1141 clocks, with
          // single FMAs and additions in some 1300 (the exponentials' own time: 1024)
          const float2 x = __ffma2_rn(
              make_float2(__uint_as_float(v[2 * e]), __uint_as_float(v[2 * e + 1])),
              make_float2(c, c), make_float2(to, to));
          const float2 p = make_float2(ex2_approx(x.x), ex2_approx(x.y));
          ls[e & 1] = __fadd2_rn(ls[e & 1], p);
          pk[e] = pack2<BF>(p.x, p.y);
        }
        // tcgen05.ld/st are warp-wide: the whole warp takes the branch when any
        // of its rows grew (alpha is 1 for the others)
        auto rescale = [&]() {
          if (j > 0 && __any_sync(0xffffffffu, grow)) {
#pragma unroll
            for (int h = 0; h < D / 32; ++h) {
              uint32_t o[32];
              tmem_ld_32x32b_x32(o_col + 32 * h, o);
              tmem_wait_ld();
#pragma unroll
              for (int d = 0; d < 32; ++d) o[d] = __float_as_uint(__uint_as_float(o[d]) * alpha);
#pragma unroll
              for (int q = 0; q < 2; ++q)
                tmem_st_32x32b_x16(o_col + 32 * h + q * 16,
                                   *reinterpret_cast<uint32_t(*)[16]>(o + 16 * q));
            }
          }
        };
        if (!C::OVERLAY && tiles > 0) {  // P V of the tile before still reads P
          ok = wait(bar_o_full, (tiles - 1) & 1u);
          if (!ok) break;
          tc_fence_after();
        }
#pragma unroll
        for (int q = 0; q < 4; ++q)
          tmem_st_32x32b_x16(p_col + q * 16, *reinterpret_cast<uint32_t(*)[16]>(pk + 16 * q));
        rescale();
        tmem_wait_st();
        tc_fence_before();
        mbar_arrive(bar_p_full + 8 * t);
        l_run = fmaf(l_run, alpha, (ls[0].x + ls[0].y) + (ls[1].x + ls[1].y));
        m_run = m_use;
      }
      if (!ok) break;
      if (n) {
        if (!wait(bar_o_done + 8 * t, outs++ & 1u)) break;
        tc_fence_after();
        const float inv = 1.f / l_run;
        const Work w = work_of<T>(a, item());
        const int q0 = T == 2 && t ? w.qt[1] : w.qt[0], len = w.len;
        const int head = w.ph ? w.head0 + t : w.head0;
        uint32_t fixes = 0;
#pragma unroll
        for (int f = 0; f < 8; ++f) fixes |= fix_rows[(i & 1) * 8 + f];
        // (Not unrolled: this runs once per item, and fetching its code is what it
        // costs.)
#pragma unroll 1
        for (int h = 0; h < C::HALVES; ++h) {
          uint32_t o[64];
          tmem_ld_32x32b_x32(o_col + 64 * h, *reinterpret_cast<uint32_t(*)[32]>(o));
          tmem_ld_32x32b_x32(o_col + 64 * h + 32, *reinterpret_cast<uint32_t(*)[32]>(o + 32));
          tmem_wait_ld();
#pragma unroll
          for (int d = 0; d < 64; ++d) o[d] = __float_as_uint(__uint_as_float(o[d]) * inv);
          // infinities and NaN taken out of the diagonal V tiles
          for (int f = 0; f < 8 && __builtin_expect(fixes != 0, 0); ++f) {
            uint32_t bits = fix_rows[(i & 1) * 8 + f];
            while (bits) {
              const int key =
                  fix_tile[(i & 1) * 2 + (f >> 2)] * BKV + (f & 3) * 32 + __ffs(bits) - 1;
              bits &= bits - 1;
              if (key >= lim) continue;
              const uint16_t* vr =
                  a.v + (int64_t)(w.row0 + key) * a.v_stride + w.kv_head * D + 64 * h;
#pragma unroll
              for (int d = 0; d < 64; ++d) {
                const uint32_t x16 = vr[d];
                const float x = BF ? __uint_as_float(x16 << 16) : unpack_half2(x16).x;
                if (not_finite<BF>(x16) & 0xFFFFu)
                  o[d] = __float_as_uint(__uint_as_float(o[d]) + x);
              }
            }
          }
          uint32_t x[32];
#pragma unroll
          for (int e = 0; e < 32; ++e)
            x[e] = pack2<BF>(__uint_as_float(o[2 * e]), __uint_as_float(o[2 * e + 1]));
          // Through shared memory (the warp's own 32 rows, 128-byte swizzle): one
          // TMA store takes them, and nobody waits for it. Where the sequence ends
          // among the rows, lanes store what is there, four whole lines at a time.
          if (lane == 0) bulk_wait_read();  // the store before has read the buffer
          __syncwarp();
#pragma unroll
          for (int c8 = 0; c8 < 8; ++c8)
            *reinterpret_cast<uint4*>(out + lane * 128 + ((c8 ^ (lane & 7)) << 4)) =
                make_uint4(x[4 * c8], x[4 * c8 + 1], x[4 * c8 + 2], x[4 * c8 + 3]);
          if (q0 + quad * 32 + 32 <= len) {
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) {
              tma_store_3d(&map_o, smem_u32(out), 0, w.row0 + q0 + quad * 32,
                           head * C::HALVES + h);
              bulk_commit();
            }
          } else {
            __syncwarp();
#pragma unroll 1
            for (int rr = lane / 8; rr < 32 && q0 + quad * 32 + rr < len; rr += 4)
              *reinterpret_cast<uint4*>(a.o + (int64_t)(w.row0 + q0 + quad * 32 + rr) * a.o_stride +
                                        head * D + 64 * h + 8 * (lane & 7)) =
                  *reinterpret_cast<const uint4*>(out + rr * 128 + (((lane & 7) ^ (rr & 7)) << 4));
            __syncwarp();
          }
        }
        tc_fence_before();  // O has been read before the next item's P is told
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(bar_item_free + 8 * (i & 1));
    }
    if (lane == 0) bulk_wait();
  }

  tc_fence_before();
  __syncthreads();
  if (warp == C::ISSUER) {
    tc_fence_after();
    tmem_dealloc(tmem, C::COLS);
  }
}

// Rows [rows, heads * D] as (64, rows, heads * D / 64): one box holds some rows of
// one head, its 64-wide parts one after another.
template <int D>
bool rows_map(CUtensorMap* map, const uint16_t* x, int rows, int heads, int64_t stride, bool bf,
              int box_rows, int box_parts) {
  cuuint64_t dims[3] = {64, (cuuint64_t)rows, (cuuint64_t)heads * (D / 64)};
  cuuint64_t strides[2] = {(cuuint64_t)stride * 2, 128};
  cuuint32_t box[3] = {64, (cuuint32_t)box_rows, (cuuint32_t)box_parts};
  cuuint32_t es[3] = {1, 1, 1};
  return encode_tiled()(map,
                        bf ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3,
                        const_cast<uint16_t*>(x), dims, strides, box, es,
                        CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                        CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int D, bool BF>
sam3_status_t launch_packed(sam3_ctx_t* ctx, const uint16_t* q, int64_t q_stride,
                            const uint16_t* k, int64_t k_stride, PackedArgs& a, int heads,
                            int kv_heads) {
  using C = PK<D>;
  CUtensorMap mq, mk, mv, mo;
  if (!rows_map<D>(&mq, q, a.rows, heads, q_stride, BF, BQ, C::HALVES) ||
      !rows_map<D>(&mk, k, a.rows, kv_heads, k_stride, BF, BKV, C::HALVES) ||
      !rows_map<D>(&mv, a.v, a.rows, kv_heads, a.v_stride, BF, BKV, C::HALVES) ||
      !rows_map<D>(&mo, a.o, a.rows, heads, a.o_stride, BF, 32, 1))
    return set_error(ctx, SAM3_ERR_CUDA, "attention_packed: cuTensorMapEncodeTiled failed");
  const uint32_t bit = (uint32_t)kSmemPacked << ((D == 128) * 2 + BF);
  const sam3_status_t st = ensure_smem_attr(ctx, bit, packed_attn_kernel<D, BF>, C::SMEM,
                                            "attention_packed smem attribute");
  if (st != SAM3_OK) return st;
  a.pair_heads = C::T == 2 && a.group % 2 == 0;
  a.units = a.pair_heads ? heads / 2 : heads;
  const int span = C::T == 2 && !a.pair_heads ? 256 : 128;
  // at most rows / span full tiles, and one more for each sequence with rows
  const long long tiles = a.rows / span + std::min(a.n_seqs, a.rows);
  if (tiles * a.units > 0x7FFFFFFFll)
    return set_error(ctx, SAM3_ERR_SHAPE, "attention_packed: too many rows for one call");
  const unsigned grid = (unsigned)(tiles * a.units);
  a.resident = ctx->num_sms * (D == 128 ? 1 : 2);
  const cudaError_t e = launch_pdl(packed_attn_kernel<D, BF>, dim3(grid), dim3(C::THREADS), C::SMEM,
                                   ctx->stream, mq, mk, mv, mo, a);
  return check_launch_ret(ctx, e, "packed_attn_kernel");
}

}  // namespace

sam3_status_t attention_packed(sam3_ctx_t* ctx, int dtype, const uint16_t* q, int64_t q_stride,
                               const uint16_t* k, int64_t k_stride, const uint16_t* v,
                               int64_t v_stride, const int32_t* cu, int n_seqs, int rows, int heads,
                               int kv_heads, int head_dim, float scale, int causal, uint16_t* o,
                               int64_t o_stride) {
  if (!q || !k || !v || !cu || !o)
    return set_error(ctx, SAM3_ERR_INVALID_ARG, "attention_packed: null pointer");
  if (dtype != SAM3_F16 && dtype != SAM3_BF16)
    return set_error(ctx, SAM3_ERR_INVALID_ARG, "attention_packed: unknown dtype %d", dtype);
  if (!aligned16(q) || !aligned16(k) || !aligned16(v) || !aligned16(o))
    return set_error(ctx, SAM3_ERR_INVALID_ARG, "attention_packed: rows must be 16-byte aligned");
  if (!scale_ok(scale))
    return set_error(ctx, SAM3_ERR_INVALID_ARG,
                     "attention_packed: scale must be positive and finite");
  if (head_dim != 64 && head_dim != 128)
    return set_error(ctx, SAM3_ERR_SHAPE, "attention_packed: head_dim must be 64 or 128 (got %d)",
                     head_dim);
  if (heads <= 0 || kv_heads <= 0 || heads > 1024 || heads % kv_heads)
    return set_error(ctx, SAM3_ERR_SHAPE, "attention_packed: %d heads over %d K/V heads", heads,
                     kv_heads);
  const int64_t wide = (int64_t)heads * head_dim, narrow = (int64_t)kv_heads * head_dim;
  if (!stride_ok(q_stride, wide) || !stride_ok(o_stride, wide) || !stride_ok(k_stride, narrow) ||
      !stride_ok(v_stride, narrow))
    return set_error(ctx, SAM3_ERR_SHAPE,
                     "attention_packed: row strides must be multiples of 8 that hold a row's heads");
  if (n_seqs <= 0 || n_seqs > 65535 || rows <= 0 || rows > kMaxContext)
    return set_error(ctx, SAM3_ERR_SHAPE, "attention_packed: bad shape");
  PackedArgs a{};
  a.o = o;
  a.v = v;
  a.cu = cu;
  a.err = ctx->dev_err;
  a.o_stride = o_stride;
  a.v_stride = v_stride;
  a.n_seqs = n_seqs;
  a.rows = rows;
  a.group = heads / kv_heads;
  a.causal = causal != 0;
  a.c = scale * kLog2E;
  // lengths stay on the device: the work counted here is the rows read and written
  ProfScope prof(ctx, SAM3_PROF_ATTENTION, 0.0, 4.0 * rows * (wide + narrow));
  const bool bf = dtype == SAM3_BF16;
  if (head_dim == 128)
    return bf ? launch_packed<128, true>(ctx, q, q_stride, k, k_stride, a, heads, kv_heads)
              : launch_packed<128, false>(ctx, q, q_stride, k, k_stride, a, heads, kv_heads);
  return bf ? launch_packed<64, true>(ctx, q, q_stride, k, k_stride, a, heads, kv_heads)
            : launch_packed<64, false>(ctx, q, q_stride, k, k_stride, a, heads, kv_heads);
}

}  // namespace sam3

using namespace sam3;

extern "C" sam3_status_t sam3_attention_packed(
    sam3_ctx_t* ctx, int32_t dtype, const uint16_t* q, int64_t q_stride, const uint16_t* k,
    int64_t k_stride, const uint16_t* v, int64_t v_stride, const int32_t* cu, int32_t n_seqs,
    int32_t rows, int32_t heads, int32_t kv_heads, int32_t head_dim, float scale, int32_t causal,
    uint16_t* o, int64_t o_stride) {
  SAM3_CHECK_CTX(ctx);
  cudaSetDevice(ctx->device);
  return attention_packed(ctx, dtype, q, q_stride, k, k_stride, v, v_stride, cu, n_seqs, rows,
                          heads, kv_heads, head_dim, scale, causal, o, o_stride);
}
