// attention_cached.cu - attention of each sequence's newest tokens over a paged
// cache held in 8 bits (kv_cache.cu).
//
// o[t, h] = sum_j p_j v_j / sum_j p_j, p_j = 2^(x_j), x_j = scale log2(e) *
// q[t, h] . k_j, over the tokens j of t's sequence that t sees; k_j and v_j are
// e4m3 codes times their page's scale. The K/V heads are shared by groups of
// heads / kv_heads query heads.
//
// HBM bound: every code is read once (2 * len * kv_heads * head_dim bytes) and
// serves the `group * new` query rows of its K/V head, a handful, so the matrix
// work is small: warp-level fp16 matrix instructions on 16-row tiles, not
// tcgen05, whose smallest tile has 64 rows. Every e4m3 code is exact in fp16.
//
// Split: the context is cut into units of a few 64-token tiles (one for each
// warp group of a CTA, below), the units of all (sequence, K/V head, row block)
// are counted through, and each of the num_sms CTAs takes an equal run of them,
// whatever the sequences' lengths. Where a run begins or ends inside an item,
// the CTA leaves its unnormalised sum, maximum and row sum in the workspace, and
// cached_join_kernel adds the pieces in the order of the CTAs (no atomics: the
// result does not depend on timing).
//
// A CTA: warp 8 streams tiles (64 tokens of K and V) through a shared-memory
// ring by TMA, page by page through the table, 128-byte swizzled lines; warps
// 0-7 are `rt` row tiles times 8 / rt groups, group g takes every (8 / rt)-th
// tile of an item and keeps its own running maximum, sums and output in
// registers. At the end of an item the groups meet in shared memory.
//
// V's scale joins the exponent: P = 2^(x + log2(vs) - M) with M the running
// maximum of x + log2(vs), so that P * code needs no second scale; the row sum
// adds P / vs in fp32. P is rounded to fp16 at 2^12 times its value (its
// largest entry is 2^12), which keeps weights down to 2^-26 of the largest in
// fp16's normal range: half a step of 2^-11 of each weight.
#include <algorithm>

#include "common.cuh"
#include "internal.h"

#include <cuda_bf16.h>

namespace sam3 {
namespace {

constexpr int KT = 64;                 // tokens per tile
constexpr int CWARPS = 8;              // computing warps
constexpr int THREADS = 32 * (CWARPS + 1);
constexpr int MAX_SEQS = SAM3_CACHED_MAX_SEQS;
constexpr int RING_BYTES = 128 * 1024;
constexpr float P_SHIFT = 12.f;

template <int D>
struct Cfg {
  static constexpr int TILE = KT * D;               // bytes of K or V in a tile
  static constexpr int ST = RING_BYTES / (2 * TILE);
  static constexpr int OFF_COMB = RING_BYTES;       // [CWARPS][16][D] f32
  static constexpr int OFF_ML = OFF_COMB + CWARPS * 16 * D * 4;    // [CWARPS][16] (max, sum)
  static constexpr int OFF_SCALE = OFF_ML + CWARPS * 16 * 8;       // [ST][4] float4
  static constexpr int OFF_SEQ = OFF_SCALE + ST * 4 * 16;          // prefix, len, row, new
  static constexpr int OFF_BAR = OFF_SEQ + (4 * MAX_SEQS + 4) * 4;
  static constexpr int OFF_MISC = OFF_BAR + 2 * ST * 8;
  static constexpr int SMEM = OFF_MISC + 16 + 1024;
};
static_assert(Cfg<128>::SMEM <= 227 * 1024 && Cfg<64>::SMEM <= 227 * 1024, "shared memory");
static_assert(Cfg<128>::ST >= CWARPS, "a unit's tiles fit the ring");

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
  int rt;  // row tiles of 16 in a row block: 1, 2 or 4
  int causal;
  float scale_log2;
};

__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0,
                                         uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// Four codes to two fp16 pairs.
__device__ __forceinline__ void codes_to_half(uint32_t w, uint32_t& lo, uint32_t& hi) {
  asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\t"
      "cvt.rn.f16x2.e4m3x2 %0, l;\n\tcvt.rn.f16x2.e4m3x2 %1, h;\n\t}"
      : "=r"(lo), "=r"(hi)
      : "r"(w));
}
__device__ __forceinline__ float quad_max(float v) {
  v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 1));
  return fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 2));
}
__device__ __forceinline__ float quad_sum(float v) {
  v += __shfl_xor_sync(0xffffffffu, v, 1);
  return v + __shfl_xor_sync(0xffffffffu, v, 2);
}
// Whether any of the four codes is NaN (0x7F or 0xFF).
__device__ __forceinline__ uint32_t nan_codes(uint32_t w) {
  return __vcmpeq4(w & 0x7F7F7F7Fu, 0x7F7F7F7Fu);
}
__device__ __forceinline__ void compute_barrier() {
  asm volatile("bar.sync 1, %0;" ::"n"(32 * CWARPS) : "memory");
}

// Byte offset of 16-byte group `c` of a token's row in a tile. Lines of 128
// bytes (one token of head_dim 128, two of 64) with TMA's 128-byte swizzle:
// group index XOR line mod 8. The fragment loads below then hit every bank
// once (V at head_dim 64: twice).
template <int D>
__device__ __forceinline__ uint32_t tile_off(int row, int c) {
  const int line = D == 128 ? row : row >> 1;
  const int grp = D == 128 ? c : (row & 1) * 4 + c;
  return line * 128 + ((grp ^ (line & 7)) << 4);
}

// Row blocks of 16 * rt query rows per K/V head of a sequence.
__device__ __forceinline__ int row_blocks(const CachedArgs& a, int fresh) {
  return (fresh * a.group + 16 * a.rt - 1) / (16 * a.rt);
}
// The sequences' units times row blocks (prefix sums), lengths, first rows and
// new tokens in shared memory. A sequence that does not fit its buffers counts
// none.
struct SeqTable {
  int *prefix, *len, *row, *fresh;
};
__device__ __forceinline__ SeqTable seq_table(uint8_t* base) {
  int* p = reinterpret_cast<int*>(base);
  return {p, p + MAX_SEQS + 1, p + 2 * MAX_SEQS + 1, p + 3 * MAX_SEQS + 1};
}
__device__ void load_seqs(const CachedArgs& a, const SeqTable& s, int kg, bool report) {
  for (int i = threadIdx.x; i < a.n_seqs; i += blockDim.x) {
    const int len = a.lens[i];
    const int r0 = a.cu ? a.cu[i] : i;
    const int r1 = a.cu ? a.cu[i + 1] : i + 1;
    const bool ok = tokens_fit(r0, r1, a.rows, a.max_new, len, a.table_stride, a.page_shift);
    if (!ok && report) atomicExch(a.err, kDevErrBadLengths);
    const int fresh = ok ? r1 - r0 : 0;
    s.prefix[i + 1] = fresh ? (len + KT * kg - 1) / (KT * kg) * row_blocks(a, fresh) : 0;
    s.len[i] = len;
    s.row[i] = r0;
    s.fresh[i] = fresh;
  }
  if (threadIdx.x == 0) s.prefix[0] = 0;
  __syncthreads();
  if (threadIdx.x < 32) {
    int sum = 0;
    for (int i0 = 0; i0 < a.n_seqs; i0 += 32) {
      const int i = i0 + threadIdx.x;
      int v = i < a.n_seqs ? s.prefix[i + 1] : 0;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, v, o);
        if ((int)threadIdx.x >= o) v += u;
      }
      if (i < a.n_seqs) s.prefix[i + 1] = sum + v;
      sum += __shfl_sync(0xffffffffu, v, 31);
    }
  }
  __syncthreads();
}

// A run of units over the items (sequence, K/V head and row block).
struct Run {
  int seq, sub, unit;
  int left;           // units to go
  int units, blocks;  // of the sequence
};
__device__ __forceinline__ void run_enter(const CachedArgs& a, const SeqTable& s, Run& r) {
  r.blocks = row_blocks(a, s.fresh[r.seq]);
  r.units = max(1, (s.prefix[r.seq + 1] - s.prefix[r.seq]) / max(1, r.blocks));
}
__device__ __forceinline__ Run run_start(const CachedArgs& a, const SeqTable& s, int x0, int x1) {
  Run r;
  r.left = x1 - x0;
  int lo = 0, hi = a.n_seqs - 1;  // the first sequence that ends behind x0
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (s.prefix[mid + 1] * a.kv_heads > x0)
      hi = mid;
    else
      lo = mid + 1;
  }
  r.seq = lo;
  const int at = x0 - s.prefix[lo] * a.kv_heads;
  run_enter(a, s, r);
  r.sub = at / r.units;
  r.unit = at - r.sub * r.units;
  return r;
}
__device__ __forceinline__ void run_next(const CachedArgs& a, const SeqTable& s, Run& r, int taken) {
  r.left -= taken;
  r.unit = 0;
  if (++r.sub < a.kv_heads * r.blocks) return;
  r.sub = 0;
  do {
    ++r.seq;
  } while (r.seq < a.n_seqs - 1 && s.prefix[r.seq + 1] == s.prefix[r.seq]);
  if (r.seq < a.n_seqs) run_enter(a, s, r);
}

template <bool BF>
__device__ __forceinline__ uint32_t pack_out(float lo, float hi) {
  if (BF) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  return pack_half2(lo, hi);
}
// Four outputs of one (row, head): 8 bytes.
template <bool BF>
__device__ __forceinline__ void store_out4(uint16_t* p, float4 v) {
  *reinterpret_cast<uint2*>(p) = make_uint2(pack_out<BF>(v.x, v.y), pack_out<BF>(v.z, v.w));
}

// Query fragments of one row in the K permutation (thread t of a quad holds
// elements t*D/4 ... of the row), in fp16. A bf16 row is first multiplied by a
// power of two that brings its largest element to [2^14, 2^15): exact for all
// elements down to 2^-28 of the largest, and below that off by at most 2^-40
// of it. Returns the power that undoes it.
template <int D, bool BF>
__device__ __forceinline__ float load_q_row(const uint16_t* row, int t, uint32_t (&f)[D / 8]) {
  const uint4* src = reinterpret_cast<const uint4*>(row + t * (D / 4));
#pragma unroll
  for (int i = 0; i < D / 32; ++i) {
    const uint4 u = row ? src[i] : make_uint4(0, 0, 0, 0);
    f[4 * i] = u.x;
    f[4 * i + 1] = u.y;
    f[4 * i + 2] = u.z;
    f[4 * i + 3] = u.w;
  }
  if (!BF) return 1.f;
  float top = 0.f;
#pragma unroll
  for (int i = 0; i < D / 8; ++i)
    top = fmaxf(top, fmaxf(fabsf(__uint_as_float(f[i] << 16)),
                           fabsf(__uint_as_float(f[i] & 0xFFFF0000u))));
  top = quad_max(top);
  // exponent of the largest, kept where both powers below are normal numbers
  const int e = min(max(((__float_as_int(top) >> 23) & 255) - 127 - 14, -126), 113);
  const float down = __int_as_float((127 - e) << 23);
#pragma unroll
  for (int i = 0; i < D / 8; ++i)
    f[i] = pack_half2(__uint_as_float(f[i] << 16) * down,
                      __uint_as_float(f[i] & 0xFFFF0000u) * down);
  return __int_as_float((127 + e) << 23);
}

template <int D, bool BF>
__global__ void __launch_bounds__(THREADS, 1)
    cached_attn_kernel(const __grid_constant__ CUtensorMap map_k,
                       const __grid_constant__ CUtensorMap map_v, const CachedArgs a) {
  using C = Cfg<D>;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  const uint32_t sbase = smem_u32(smem);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rt = a.rt, kg = CWARPS / rt;
  const uint32_t bar_full = sbase + C::OFF_BAR, bar_empty = bar_full + 8 * C::ST;
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + C::OFF_MISC);
  const SeqTable seqs = seq_table(smem + C::OFF_SEQ);
  float4* scales = reinterpret_cast<float4*>(smem + C::OFF_SCALE);

  if (threadIdx.x == 0) {
    for (int s = 0; s < C::ST; ++s) {
      mbar_init(bar_full + 8 * s, 1);
      mbar_init(bar_empty + 8 * s, rt);
    }
    *abort_flag = 0;
    fence_mbar_init();
    prefetch_tmap(&map_k);
    prefetch_tmap(&map_v);
  }
  griddep_launch_dependents();
  griddep_wait();  // lengths, pages, codes and queries may be earlier kernels' outputs
  load_seqs(a, seqs, kg, blockIdx.x == 0);

  const int total = seqs.prefix[a.n_seqs] * a.kv_heads;
  const int chunk = (total + gridDim.x - 1) / gridDim.x;
  const int x0 = min(total, (int)blockIdx.x * chunk), x1 = min(total, x0 + chunk);
  if (threadIdx.x == 0) {
    // bit 0: the run begins inside an item, 1: it ends inside an item that
    // begins in it, 2: it lies inside one item and does not end it
    int flags = 0, item_seq = 0, item_sub = 0;
    if (x1 > x0) {
      const Run f = run_start(a, seqs, x0, x1), l = run_start(a, seqs, x1 - 1, x1);
      const bool open = l.unit + 1 < l.units;
      const bool same = f.seq == l.seq && f.sub == l.sub;
      if (f.unit > 0) flags |= 1;
      if (open && (!same || f.unit == 0)) flags |= 2;
      if (open && same && f.unit > 0) flags |= 4;
      item_seq = l.seq;
      item_sub = l.sub;
    }
    a.meta[blockIdx.x * 4] = flags;
    a.meta[blockIdx.x * 4 + 1] = item_seq;
    a.meta[blockIdx.x * 4 + 2] = item_sub;
  }
  if (x1 <= x0) return;

  if (warp == CWARPS) {
    // ------------------------------------------------------------- producer
    const int page = 1 << a.page_shift;
    const int per = KT >> min(a.page_shift, 6);  // pages per tile
    const int box = min(page, KT);               // tokens per copy
    const uint32_t copy_bytes = box * D;
    int stage = 0;
    uint32_t phase = 0, used = 0;
    Run r = run_start(a, seqs, x0, x1);
    while (r.left > 0) {
      const int n_units = min(r.left, r.units - r.unit);
      const int len = seqs.len[r.seq];
      const int head = r.sub / r.blocks;
      const int tile1 = min((r.unit + n_units) * kg, (len + KT - 1) / KT);
      const int pages = (len + page - 1) >> a.page_shift;
      const int32_t* row = a.table + (size_t)r.seq * a.table_stride;
      int window = -32;
      int slot = 0;
      float ks = 0.f, lvs = 0.f, ivs = 0.f;
      for (int tile = r.unit * kg; tile < tile1; ++tile) {
        const int first = (tile * KT) >> a.page_shift;
        if (first >= window + 32) {
          // the next 32 pages of the sequence, one per lane, with their scales
          window = first & ~31;
          const int p = window + lane;
          slot = p < pages ? row[p] : -1;
          if (p < pages && !page_fits(slot, a.num_pages)) {
            atomicExch(a.err, kDevErrBadPage);
            slot = -1;
          }
          ks = 0.f;
          float vs = 1.f;
          if (slot >= 0) {
            ks = a.k_scale[(size_t)slot * a.kv_heads + head] * a.scale_log2;
            vs = a.v_scale[(size_t)slot * a.kv_heads + head];
          }
          lvs = __log2f(vs);
          ivs = 1.f / vs;
        }
        mbar_wait(bar_empty + 8 * stage, phase ^ 1, abort_flag, a.err, kDevErrTimeoutCached);
        if (*abort_flag) break;
        // lane l copies K (even) or V (odd) of page l / 2 of the tile
        const int mine = first + (lane >> 1);
        const int my_slot = __shfl_sync(0xffffffffu, slot, mine & 31);
        const bool copies = lane < 2 * per && mine < pages && my_slot >= 0;
        const uint32_t n_copies = __popc(__ballot_sync(0xffffffffu, copies));
        // a missing page's codes are never used: its tokens count as masked
        const int sp = first + ((lane & 3) * 16 >> min(a.page_shift, 6));
        const float4 sc = make_float4(__shfl_sync(0xffffffffu, ks, sp & 31),
                                      __shfl_sync(0xffffffffu, lvs, sp & 31),
                                      __shfl_sync(0xffffffffu, ivs, sp & 31),
                                      __shfl_sync(0xffffffffu, slot, sp & 31) >= 0 ? 1.f : 0.f);
        if (lane < 4) scales[stage * 4 + lane] = sc;
        __syncwarp();
        if (lane == 0) mbar_arrive_expect_tx(bar_full + 8 * stage, n_copies * copy_bytes);
        __syncwarp();
        if (copies) {
          const int which = lane & 1;
          const uint32_t dst = sbase + (stage * 2 + which) * C::TILE + (lane >> 1) * copy_bytes;
          const int tok = page > KT ? (tile * KT) & (page - 1) : 0;
          const long long at = ((long long)my_slot * a.kv_heads + head) << a.page_shift;
          const int line = (int)((at + tok) / (128 / D));
          tma_load_2d(dst, which ? &map_v : &map_k, bar_full + 8 * stage, 0, line);
        }
        used = min(used + 1, (uint32_t)C::ST);
        if (++stage == C::ST) {
          stage = 0;
          phase ^= 1;
        }
      }
      if (*abort_flag) break;
      run_next(a, seqs, r, n_units);
    }
    if (*abort_flag) {
      // nothing may still be in flight into this CTA's shared memory
      for (uint32_t i = 0; i < used; ++i) {
        if (--stage < 0) {
          stage = C::ST - 1;
          phase ^= 1;
        }
        mbar_wait_drain(bar_full + 8 * stage, phase);
      }
    }
    return;
  }

  // --------------------------------------------------------------- computing
  const int g = lane >> 2, t = lane & 3;
  const int my_rt = warp % rt, my_kg = warp / rt;
  float* comb = reinterpret_cast<float*>(smem + C::OFF_COMB);
  float2* ml = reinterpret_cast<float2*>(smem + C::OFF_ML);
  int stage = 0;
  uint32_t phase = 0;
  Run r = run_start(a, seqs, x0, x1);
  while (r.left > 0) {
    const int n_units = min(r.left, r.units - r.unit);
    const int len = seqs.len[r.seq], row0 = seqs.row[r.seq], fresh = seqs.fresh[r.seq];
    const int head = r.sub / r.blocks, block = r.sub - head * r.blocks;
    const int n_rows = min(16 * rt, fresh * a.group - block * 16 * rt);
    const int tile0 = r.unit * kg;
    const int tile1 = min((r.unit + n_units) * kg, (len + KT - 1) / KT);
    // this thread's two rows: query token and head, tokens it sees
    uint32_t qf[D / 16][4];
    float rs[2];
    int lim[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int lr = my_rt * 16 + g + 8 * h;
      const int gr = block * 16 * rt + lr;
      const int tok = gr / a.group, gq = gr - tok * a.group;
      const uint16_t* src =
          lr < n_rows ? a.q + (int64_t)(row0 + tok) * a.q_stride + (head * a.group + gq) * D
                      : nullptr;
      uint32_t f[D / 8];
      rs[h] = load_q_row<D, BF>(src, t, f);
#pragma unroll
      for (int s = 0; s < D / 16; ++s) {
        qf[s][h] = f[2 * s];
        qf[s][2 + h] = f[2 * s + 1];
      }
      lim[h] = a.causal && lr < n_rows ? len - fresh + tok + 1 : len;
    }
    const int lim_min = a.causal ? len - fresh + 1 : len;
    float o[D / 8][4];
#pragma unroll
    for (int i = 0; i < D / 8; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[i][e] = 0.f;
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};

    for (int tile = tile0; tile < tile1; ++tile) {
      const int st = stage;
      const uint32_t ph = phase;
      if (++stage == C::ST) {
        stage = 0;
        phase ^= 1;
      }
      if ((tile & (kg - 1)) != my_kg) continue;
      // on an expired wait the loop runs on over stale data: the barriers below
      // are met by every warp, and the host learns of the error
      mbar_wait(bar_full + 8 * st, ph, abort_flag, a.err, kDevErrTimeoutCached);
      __syncwarp();
      const uint8_t *sk = smem + st * 2 * C::TILE, *sv = sk + C::TILE;
      const int kbase = tile * KT;
      float s[KT / 8][4];
#pragma unroll
      for (int j = 0; j < KT / 8; ++j) {
        s[j][0] = s[j][1] = s[j][2] = s[j][3] = 0.f;
        const int row = 8 * j + g;
        uint4 w[D / 64];
#pragma unroll
        for (int i = 0; i < D / 64; ++i) 
          w[i] = *reinterpret_cast<const uint4*>(sk + tile_off<D>(row, t * (D / 64) + i));
#pragma unroll
        for (int i = 0; i < D / 64; ++i) {
          const uint32_t ww[4] = {w[i].x, w[i].y, w[i].z, w[i].w};
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            uint32_t b0, b1;
            codes_to_half(ww[q], b0, b1);
            mma16816(s[j], qf[4 * i + q], b0, b1);
          }
        }
      }
      float ivs[4];
      const bool edge = kbase + KT > lim_min;
      float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
      for (int kk = 0; kk < 4; ++kk) {
        const float4 sc = scales[st * 4 + kk];
        ivs[kk] = sc.z;
        const float c0 = sc.x * rs[0], c1 = sc.x * rs[1];
#pragma unroll
        for (int j = 2 * kk; j < 2 * kk + 2; ++j) {
          s[j][0] = fmaf(s[j][0], c0, sc.y);
          s[j][1] = fmaf(s[j][1], c0, sc.y);
          s[j][2] = fmaf(s[j][2], c1, sc.y);
          s[j][3] = fmaf(s[j][3], c1, sc.y);
          if (edge || sc.w == 0.f) {
            const int key = kbase + 8 * j + 2 * t;
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (key + (e & 1) >= lim[e >> 1] || sc.w == 0.f) s[j][e] = -INFINITY;
          }
          top[0] = fmaxf(top[0], fmaxf(s[j][0], s[j][1]));
          top[1] = fmaxf(top[1], fmaxf(s[j][2], s[j][3]));
        }
      }
      float off[2], alpha[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const float mn = fmaxf(m[h], quad_max(top[h]));
        const float mu = mn == -INFINITY ? 0.f : mn;  // nothing seen yet: weights of 0
        alpha[h] = ex2_approx(m[h] - mu);
        off[h] = P_SHIFT - mu;
        m[h] = mn;
        l[h] *= alpha[h];
      }
      uint32_t p[4][4];
#pragma unroll
      for (int kk = 0; kk < 4; ++kk) {
        float sum[2] = {0.f, 0.f};
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          float* x = s[2 * kk + j];
          x[0] = ex2_approx(x[0] + off[0]);
          x[1] = ex2_approx(x[1] + off[0]);
          x[2] = ex2_approx(x[2] + off[1]);
          x[3] = ex2_approx(x[3] + off[1]);
          sum[0] += x[0] + x[1];
          sum[1] += x[2] + x[3];
          p[kk][2 * j] = pack_half2(x[0], x[1]);
          p[kk][2 * j + 1] = pack_half2(x[2], x[3]);
        }
        l[0] = fmaf(sum[0], ivs[kk], l[0]);
        l[1] = fmaf(sum[1], ivs[kk], l[1]);
      }
      if (__any_sync(0xffffffffu, alpha[0] != 1.f || alpha[1] != 1.f)) {
#pragma unroll
        for (int i = 0; i < D / 8; ++i) {
          o[i][0] *= alpha[0];
          o[i][1] *= alpha[0];
          o[i][2] *= alpha[1];
          o[i][3] *= alpha[1];
        }
      }
      // Codes of tokens that no row sees are taken as 0 (their weight is 0, but
      // 0 * NaN is not); a NaN code of a new token that only later rows see is
      // taken as 0 here and set in those rows below.
      const bool tail = kbase + KT > len;
      const bool look = a.causal && fresh > 1 && edge;
      uint32_t found = 0;
#pragma unroll
      for (int kk = 0; kk < 4; ++kk) {
        uint32_t v[4][D / 32];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int row = 16 * kk + 2 * t + (i & 1) + (i >> 1) * 8;
          if (D == 128) {
            const uint4 w = *reinterpret_cast<const uint4*>(sv + tile_off<D>(row, g));
            v[i][0] = w.x;
            v[i][1] = w.y;
            v[i][D / 32 - 2] = w.z;
            v[i][D / 32 - 1] = w.w;
          } else {
            const uint2 w =
                *reinterpret_cast<const uint2*>(sv + tile_off<D>(row, g >> 1) + (g & 1) * 8);
            v[i][0] = w.x;
            v[i][1] = w.y;
          }
          if (tail && kbase + row >= len)
#pragma unroll
            for (int q = 0; q < D / 32; ++q) v[i][q] = 0;
          if (look && kbase + row >= lim_min)
#pragma unroll
            for (int q = 0; q < D / 32; ++q) {
              const uint32_t bad = nan_codes(v[i][q]);
              found |= bad;
              v[i][q] &= ~bad;
            }
        }
        if (scales[st * 4 + kk].w == 0.f)
#pragma unroll
          for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int q = 0; q < D / 32; ++q) v[i][q] = 0;
#pragma unroll
        for (int q = 0; q < D / 32; ++q) {
          uint32_t b0[4], b1[4];
          codes_to_half(__byte_perm(v[0][q], v[1][q], 0x5140), b0[0], b0[1]);
          codes_to_half(__byte_perm(v[0][q], v[1][q], 0x7362), b0[2], b0[3]);
          codes_to_half(__byte_perm(v[2][q], v[3][q], 0x5140), b1[0], b1[1]);
          codes_to_half(__byte_perm(v[2][q], v[3][q], 0x7362), b1[2], b1[3]);
#pragma unroll
          for (int n = 0; n < 4; ++n) mma16816(o[4 * q + n], p[kk], b0[n], b1[n]);
        }
      }
      if (look && __any_sync(0xffffffffu, found != 0)) {
        for (int key = max(kbase, lim_min); key < min(len, kbase + KT); ++key)
#pragma unroll
          for (int i = 0; i < D / 8; ++i)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const int d = (2 * t + e) * (D / 8) + i;  // the output's column
              const uint32_t code = sv[tile_off<D>(key - kbase, d >> 4) + (d & 15)];
              if ((code & 0x7F) == 0x7F) {
                if (key < lim[0]) o[i][e] = NAN;
                if (key < lim[1]) o[i][2 + e] = NAN;
              }
            }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(bar_empty + 8 * st);
    }

    // The groups' sums meet: outputs [row][D] (16-byte groups permuted so that
    // the stores hit every bank once), maxima and row sums.
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const float ls = quad_sum(l[h]);
      if (t == 0) ml[warp * 16 + g + 8 * h] = make_float2(m[h], ls);
      float4* dst = reinterpret_cast<float4*>(comb + (warp * 16 + g + 8 * h) * D);
      // thread t holds columns [2t * D/8, (2t + 2) * D/8): first o[.][0], then o[.][1]
#pragma unroll
      for (int u = 0; u < D / 16; ++u) {
        const int e = u / (D / 32), i = 4 * (u % (D / 32));
        const int perm = D == 128 ? (2 * t + g) & 7 : (g & 1) | (t >> 1) << 1;
        dst[t * (D / 16) + (u ^ perm)] = make_float4(o[i][2 * h + e], o[i + 1][2 * h + e],
                                                     o[i + 2][2 * h + e], o[i + 3][2 * h + e]);
      }
    }
    compute_barrier();
    const bool starts = r.unit == 0, ends = r.unit + n_units == r.units;
    // a piece that continues an earlier CTA's item goes to slot 0, one that
    // this CTA begins and does not end to slot 1
    float* part = a.part + ((size_t)blockIdx.x * 2 + (starts ? 1 : 0)) * kCachedPartFloats;
    for (int i = threadIdx.x; i < n_rows * (D / 4); i += 32 * CWARPS) {
      const int lr = i / (D / 4), c = i % (D / 4);
      const int rr = lr & 15, w0 = lr >> 4;
      const int tt = c / (D / 16), u = c % (D / 16);
      const int perm = D == 128 ? (2 * tt + rr) & 7 : (rr & 1) | (tt >> 1) << 1;
      const int pos = tt * (D / 16) + (u ^ perm);
      float top = -INFINITY;
      for (int k = 0; k < kg; ++k) top = fmaxf(top, ml[(w0 + rt * k) * 16 + rr].x);
      const float mu = top == -INFINITY ? 0.f : top;
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
      float sum = 0.f;
      for (int k = 0; k < kg; ++k) {
        const float2 x = ml[(w0 + rt * k) * 16 + rr];
        const float f = ex2_approx(x.x - mu);
        const float4 y =
            reinterpret_cast<const float4*>(comb + ((w0 + rt * k) * 16 + rr) * D)[pos];
        sum = fmaf(x.y, f, sum);
        acc.x = fmaf(y.x, f, acc.x);
        acc.y = fmaf(y.y, f, acc.y);
        acc.z = fmaf(y.z, f, acc.z);
        acc.w = fmaf(y.w, f, acc.w);
      }
      if (starts && ends) {
        const float inv = sum == 0.f ? 0.f : 1.f / sum;
        const int gr = block * 16 * rt + lr;
        const int tok = gr / a.group, gq = gr - tok * a.group;
        store_out4<BF>(a.o + (int64_t)(row0 + tok) * a.o_stride + (head * a.group + gq) * D + 4 * c,
                       make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv));
      } else {
        reinterpret_cast<float4*>(part + lr * D)[c] = acc;
        if (c == 0) {
          part[kCachedPartRows * 128 + lr] = top;
          part[kCachedPartRows * 129 + lr] = sum;
        }
      }
    }
    compute_barrier();
    run_next(a, seqs, r, n_units);
  }
}

// Adds the pieces of the items that attention left in parts. Block c looks
// after the item that CTA c began and did not end: its slot 1, then slot 0 of
// the CTAs that follow, in order.
template <int D, bool BF>
__global__ void __launch_bounds__(256) cached_join_kernel(const CachedArgs a, int ctas) {
  griddep_launch_dependents();
  griddep_wait();  // the pieces are the previous kernel's output
  const int c0 = blockIdx.x;
  if (!(a.meta[c0 * 4] & 2)) return;
  const int seq = a.meta[c0 * 4 + 1], sub = a.meta[c0 * 4 + 2];
  const int row0 = a.cu ? a.cu[seq] : seq;
  const int fresh = a.cu ? a.cu[seq + 1] - row0 : 1;
  const int blocks = row_blocks(a, fresh);
  const int head = sub / blocks, block = sub - head * blocks;
  const int n_rows = min(16 * a.rt, fresh * a.group - block * 16 * a.rt);
  int last = c0 + 1;  // the CTA that ends the item
  while (last < ctas - 1 && (a.meta[last * 4] & 4)) ++last;
  for (int i = blockIdx.y * 256 + threadIdx.x; i < n_rows * (D / 4); i += 256 * gridDim.y) {
    const int lr = i / (D / 4), c = i % (D / 4);
    float top = -INFINITY, sum = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int k = c0; k <= last; ++k) {
      const float* part = a.part + ((size_t)k * 2 + (k == c0 ? 1 : 0)) * kCachedPartFloats;
      const float pm = part[kCachedPartRows * 128 + lr], pl = part[kCachedPartRows * 129 + lr];
      const float4 y = reinterpret_cast<const float4*>(part + lr * D)[c];
      const float mn = fmaxf(top, pm);
      const float mu = mn == -INFINITY ? 0.f : mn;
      const float f0 = ex2_approx(top - mu), f1 = ex2_approx(pm - mu);
      top = mn;
      sum = fmaf(sum, f0, pl * f1);
      acc.x = fmaf(acc.x, f0, y.x * f1);
      acc.y = fmaf(acc.y, f0, y.y * f1);
      acc.z = fmaf(acc.z, f0, y.z * f1);
      acc.w = fmaf(acc.w, f0, y.w * f1);
    }
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    const int gr = block * 16 * a.rt + lr;
    const int tok = gr / a.group, gq = gr - tok * a.group;
    store_out4<BF>(a.o + (int64_t)(row0 + tok) * a.o_stride + (head * a.group + gq) * D + 4 * c,
                   make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv));
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

template <int D, bool BF>
sam3_status_t launch_cached(sam3_ctx_t* ctx, const CUtensorMap& mk, const CUtensorMap& mv,
                            const CachedArgs& a) {
  const uint32_t bit = (uint32_t)kSmemCached << ((D == 128) * 2 + BF);
  sam3_status_t st = ensure_smem_attr(ctx, bit, cached_attn_kernel<D, BF>, Cfg<D>::SMEM,
                                      "attention_cached smem attribute");
  if (st != SAM3_OK) return st;
  const int ctas = ctx->num_sms;
  cudaError_t e = launch_pdl(cached_attn_kernel<D, BF>, dim3(ctas), dim3(THREADS), Cfg<D>::SMEM,
                             ctx->stream, mk, mv, a);
  if ((st = check_launch_ret(ctx, e, "cached_attn_kernel")) != SAM3_OK) return st;
  e = launch_pdl(cached_join_kernel<D, BF>, dim3(ctas), dim3(256), 0, ctx->stream, a, ctas);
  return check_launch_ret(ctx, e, "cached_join_kernel");
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
  if (!(scale > 0.f) || scale > 3.402823466e38f)
    return set_error(ctx, SAM3_ERR_INVALID_ARG, "attention_cached: scale must be positive");
  if (heads <= 0 || heads > 1024 || heads % c->kv_heads)
    return set_error(ctx, SAM3_ERR_SHAPE, "attention_cached: %d heads over %d K/V heads", heads,
                     c->kv_heads);
  const int64_t width = (int64_t)heads * c->head_dim;
  if (!stride_ok(q_stride, width) || !stride_ok(o_stride, width))
    return set_error(ctx, SAM3_ERR_SHAPE,
                     "attention_cached: row strides must be multiples of 8 of at least heads * "
                     "head_dim");
  if (n_seqs <= 0 || n_seqs > MAX_SEQS || rows <= 0 || max_new <= 0 || max_new > rows ||
      table_stride <= 0 || (long long)table_stride * c->page_size > kMaxContext ||
      (!cu_new && (max_new != 1 || rows < n_seqs)))
    return set_error(ctx, SAM3_ERR_SHAPE, "attention_cached: bad shape (at most %d sequences)",
                     MAX_SEQS);
  CachedArgs a;
  a.group = heads / c->kv_heads;
  const long long most = (long long)max_new * a.group;  // query rows per K/V head
  a.rt = most <= 16 ? 1 : most <= 32 ? 2 : 4;
  const long long blocks = (most + 16 * a.rt - 1) / (16 * a.rt);
  const long long tiles = ((long long)table_stride * c->page_size + KT - 1) / KT;
  if (most > 0x7FFFFF00ll || blocks * c->kv_heads * n_seqs * tiles > 0x7FFFFFFFll)
    return set_error(ctx, SAM3_ERR_SHAPE, "attention_cached: too much work for one call");
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
  a.scale_log2 = scale * 1.4426950408889634f;
  const long long lines =
      (long long)c->num_pages * c->kv_heads * c->page_size * c->head_dim / 128;
  const int box = std::min(c->page_size, KT) * c->head_dim / 128;
  CUtensorMap mk, mv;
  if (!pool_map(&mk, c->k, lines, box) || !pool_map(&mv, c->v, lines, box))
    return set_error(ctx, SAM3_ERR_CUDA, "attention_cached: cuTensorMapEncodeTiled failed");
  // lengths stay on the device: the work counted here is q and o alone
  ProfScope prof(ctx, SAM3_PROF_ATTENTION, 0.0, 4.0 * rows * width);
  const bool bf = dtype == SAM3_BF16;
  if (c->head_dim == 128)
    return bf ? launch_cached<128, true>(ctx, mk, mv, a) : launch_cached<128, false>(ctx, mk, mv, a);
  return bf ? launch_cached<64, true>(ctx, mk, mv, a) : launch_cached<64, false>(ctx, mk, mv, a);
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
