// kv_cache.cu - writing keys and values into a paged cache held in 8 bits.
//
// A page holds `page` tokens of one sequence: [kv_heads, page, head_dim] e4m3
// codes for K and the same for V, with one fp32 scale for each page and head.
// A code c stands for c * scale. The scale is a power of two, 2^e with the
// least e that brings the page's largest finite |value| to 448 = 1.75 * 2^8 or
// below, so
//  - value / scale is exact and the code is one rounding (to nearest, ties to
//    even) away from the value: at most 2^-4 of it, or 2^-10 scales near zero;
//  - when a later token is larger than the page's scale allows, the codes that
//    are there move to the new scale by an exact division by a power of two:
//    only those that fall below 2^-6 scales (e4m3's subnormals) are rounded a
//    second time. A scale never shrinks while its page fills.
// A scale that is not a power of two would use up to 0.8 bits more of the
// code's range (it changes no rounding step relative to the value) and would
// round every held code again whenever it grew.
//
// HBM bound: 2 bytes in and 1 byte out per element. One unit of work is one
// (page, head, K or V); its elements stay in registers between the maximum and
// the rounding, so each is read once. Measured: 8 prompts of 8192 tokens (8
// heads of 128, pages of 128) 65 us, 6.2 TB/s, 94 % of a copy's rate (89 us with
// two CTAs per SM and pages before heads in the grid); four images' tokens
// (10,410 rows, 16 heads of 64, pages of 16) 13.6 us, 4.7 TB/s: the
// same chain of loads at the begin and the end is a larger part of it. One token
// each of 64 sequences: 4.9 us, a launch, three dependent loads (length, page,
// scale) and a store. Four CTAs per SM leave 64 registers a thread, and 12 to 84
// bytes spill; three do without (4 bytes at most) and take 69.3, 14.4 and 4.9 us.
#include <algorithm>

#include "common.cuh"
#include "internal.h"

#include <cuda_bf16.h>

namespace sam3 {
namespace {

constexpr int kScaleExpMin = -60, kScaleExpMax = 60;
constexpr int THREADS = 256;

struct AppendArgs {
  uint8_t *k_codes, *v_codes;
  float *k_scale, *v_scale;
  const uint16_t *k, *v;
  int64_t k_stride, v_stride;  // elements between rows
  const int32_t* cu;   // [n + 1] or null: one row per sequence
  const int32_t* lens; // [n] tokens of each sequence with the new ones
  const int32_t* table;
  int table_stride, num_pages, kv_heads, page_shift, rows, max_new;
  int groups;  // CTAs per page: its units over the units per CTA
  int* err;
};

// The least e with a <= 448 * 2^e, for a >= 0 finite; the smallest for 0.
__device__ __forceinline__ int scale_exp(float a) {
  const int b = __float_as_int(a);
  const int e = (b >> 23) - 127 - ((b & 0x7FFFFF) <= 0x600000 ? 8 : 7);
  return a > 0.f ? min(max(e, kScaleExpMin), kScaleExpMax) : kScaleExpMin;
}
__device__ __forceinline__ float exp2_int(int e) { return __int_as_float((127 + e) << 23); }

// Two values to two codes; beyond 448 they saturate, NaN stays NaN.
__device__ __forceinline__ uint32_t to_e4m3x2(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ float2 from_e4m3x2(uint16_t v) {
  uint32_t h;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(v));
  return unpack_half2(h);
}
template <bool BF>
__device__ __forceinline__ float2 unpack2(uint32_t v) {
  if (BF) return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xFFFF0000u));
  return unpack_half2(v);
}
__device__ __forceinline__ float finite_abs(float x) {
  const float a = fabsf(x);
  return a <= 3.402823466e38f ? a : 0.f;  // infinities and NaN set no scale
}

// UNIT_WARPS warps hold one unit, VEC vectors of 8 elements per lane; or one warp
// UNITS of them one after another. The CTA's 8 warps take the units of
// consecutive (head, K or V) of one page, whose rows are neighbours in the source.
template <int D, int UNIT_WARPS, int UNITS, int VEC, bool BF>
__global__ void __launch_bounds__(THREADS, 4) kv_append_kernel(const AppendArgs a) {
  constexpr int VPR = D / 8;                     // vectors per token
  constexpr int STEP = 32 * UNIT_WARPS / VPR;    // tokens between a lane's vectors
  __shared__ float warp_max[THREADS / 32];
  griddep_launch_dependents();
  griddep_wait();  // rows, lengths and pages may be earlier kernels' outputs
  const int seq = blockIdx.y;
  const int page_no = blockIdx.x / a.groups, group = blockIdx.x - page_no * a.groups;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int page = 1 << a.page_shift;
  const int len = a.lens[seq];
  const int row0 = a.cu ? a.cu[seq] : seq;
  const int row1 = a.cu ? a.cu[seq + 1] : seq + 1;
  if (!tokens_fit(row0, row1, a.rows, a.max_new, len, a.table_stride, a.page_shift)) {
    if (threadIdx.x == 0) report_bad_index(a.err, kDevErrBadLengths);
    return;
  }
  const int fresh = row1 - row0;
  const int start = len - fresh;  // position of the first new token
  const int page_at = (start >> a.page_shift) + page_no;
  if (fresh == 0 || page_at > (len - 1) >> a.page_shift) return;
  const int pos0 = page_at << a.page_shift;
  const int slot = a.table[(size_t)seq * a.table_stride + page_at];
  const int held = max(0, start - pos0);   // tokens of the page that were there
  const int last = min(page, len - pos0);  // tokens of the page now
  // vector i of this lane: token tok0 + i * STEP of the page, the same part of it
  const int v0 = (warp % UNIT_WARPS) * 32 + lane;
  const int tok0 = v0 / VPR;
  const int lo = held - tok0, hi = last - tok0;  // i * STEP of new tokens
  const int unit0 = (group * (THREADS / 32 / UNIT_WARPS) + warp / UNIT_WARPS) * UNITS;
  uint4 x[UNITS][VEC];
#pragma unroll
  for (int u = 0; u < UNITS; ++u) {
    const int unit = unit0 + u;
    const bool on = unit < 2 * a.kv_heads, is_v = unit >= a.kv_heads;
    const int64_t stride = is_v ? a.v_stride : a.k_stride;
    const uint16_t* src = (is_v ? a.v : a.k) + (unit - (is_v ? a.kv_heads : 0)) * D +
                          (v0 % VPR) * 8 + ((int64_t)row0 + pos0 + tok0 - start) * stride;
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      x[u][i] = make_uint4(0, 0, 0, 0);
      if (on && i * STEP >= lo && i * STEP < hi) x[u][i] = *reinterpret_cast<const uint4*>(src);
      src += STEP * stride;
    }
  }
  // the page's number is first needed here: it travels with the rows
  if (!page_fits(slot, a.num_pages)) {
    if (threadIdx.x == 0) report_bad_index(a.err, kDevErrBadPage);
    return;
  }
#pragma unroll
  for (int u = 0; u < UNITS; ++u) {
    const int unit = unit0 + u;
    const bool on = unit < 2 * a.kv_heads, is_v = unit >= a.kv_heads;
    const size_t at = (size_t)slot * a.kv_heads + (on ? unit - (is_v ? a.kv_heads : 0) : 0);
    float* scale = (is_v ? a.v_scale : a.k_scale) + at;
    const int was = held > 0 && on ? __float_as_int(*scale) : 0;
    float top = 0.f;
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      const uint32_t w[4] = {x[u][i].x, x[u][i].y, x[u][i].z, x[u][i].w};
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const float2 p = unpack2<BF>(w[q]);
        top = fmaxf(top, fmaxf(finite_abs(p.x), finite_abs(p.y)));
      }
    }
    // floats that are not negative compare like their bits
    top = __int_as_float(__reduce_max_sync(0xffffffffu, __float_as_int(top)));
    if (UNIT_WARPS > 1) {
      if (lane == 0) warp_max[warp] = top;
      __syncthreads();  // also: every thread has read the old scale
      const int first = warp / UNIT_WARPS * UNIT_WARPS;
#pragma unroll
      for (int i = 0; i < UNIT_WARPS; ++i) top = fmaxf(top, warp_max[first + i]);
    }
    if (!on) return;
    int e = scale_exp(top);
    const int e_was = min(max(((was >> 23) & 255) - 127, kScaleExpMin), kScaleExpMax);
    if (held > 0) e = max(e, e_was);
    const float inv = exp2_int(-e);
    uint8_t* dst = (is_v ? a.v_codes : a.k_codes) + (at << a.page_shift) * D + (size_t)v0 * 8;
    const bool grow = held > 0 && e > e_was;
    const float shrink = exp2_int(max(e_was - e, -126));
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      uint2* p = reinterpret_cast<uint2*>(dst + i * 32 * UNIT_WARPS * 8);
      if (i * STEP >= lo && i * STEP < hi) {
        const uint32_t w[4] = {x[u][i].x, x[u][i].y, x[u][i].z, x[u][i].w};
        uint32_t c[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const float2 f = unpack2<BF>(w[q]);
          c[q] = to_e4m3x2(f.x * inv, f.y * inv);
        }
        *p = make_uint2(c[0] | c[1] << 16, c[2] | c[3] << 16);
      } else if (grow && i * STEP < lo) {
        const uint2 old = *p;
        const uint32_t w[2] = {old.x, old.y};
        uint32_t c[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const float2 f = from_e4m3x2((uint16_t)(w[q >> 1] >> (16 * (q & 1))));
          c[q] = to_e4m3x2(f.x * shrink, f.y * shrink);
        }
        *p = make_uint2(c[0] | c[1] << 16, c[2] | c[3] << 16);
      }
    }
    __syncwarp();  // every lane has read the old scale
    if (warp % UNIT_WARPS == 0 && lane == 0) *scale = exp2_int(e);
  }
}

template <int D, int UNIT_WARPS, int UNITS, int VEC>
cudaError_t launch_append(sam3_ctx_t* ctx, bool bf, AppendArgs& a, int n_seqs) {
  const int per_cta = THREADS / 32 / UNIT_WARPS * UNITS;
  // the most pages that max_new tokens can touch
  const long long pages = ((long long)a.max_new - 1 + (1 << a.page_shift) - 1 >> a.page_shift) + 1;
  // heads before pages: CTAs that run together read whole rows
  a.groups = (2 * a.kv_heads + per_cta - 1) / per_cta;
  if (pages * a.groups > 0x7FFFFFFFll) return cudaErrorInvalidConfiguration;
  const dim3 grid((unsigned)(pages * a.groups), n_seqs);
  if (bf)
    return launch_pdl(kv_append_kernel<D, UNIT_WARPS, UNITS, VEC, true>, grid, dim3(THREADS), 0,
                      ctx->stream, a);
  return launch_pdl(kv_append_kernel<D, UNIT_WARPS, UNITS, VEC, false>, grid, dim3(THREADS), 0,
                    ctx->stream, a);
}

}  // namespace

sam3_status_t check_kv_cache(sam3_ctx_t* ctx, const sam3_kv_cache_t* c, const char* what) {
  if (!c || !c->k || !c->v || !c->k_scale || !c->v_scale)
    return set_error(ctx, SAM3_ERR_INVALID_ARG, "%s: null cache", what);
  if (!aligned16(c->k) || !aligned16(c->v) ||
      ((reinterpret_cast<uintptr_t>(c->k_scale) | reinterpret_cast<uintptr_t>(c->v_scale)) & 3))
    return set_error(ctx, SAM3_ERR_INVALID_ARG,
                     "%s: cache codes must be 16-byte aligned, scales 4-byte aligned", what);
  if (c->page_size != 16 && c->page_size != 32 && c->page_size != 64 && c->page_size != 128)
    return set_error(ctx, SAM3_ERR_SHAPE, "%s: page_size must be 16, 32, 64 or 128 (got %d)", what,
                     c->page_size);
  if (c->head_dim != 64 && c->head_dim != 128)
    return set_error(ctx, SAM3_ERR_SHAPE, "%s: head_dim must be 64 or 128 (got %d)", what,
                     c->head_dim);
  // 128-byte lines of the pool are addressed with 32 bits
  if (c->num_pages <= 0 || c->kv_heads <= 0 || c->kv_heads > 1024 ||
      (long long)c->num_pages * c->kv_heads * c->page_size * c->head_dim / 128 > 0x7FFFFFFFll)
    return set_error(ctx, SAM3_ERR_SHAPE, "%s: bad cache shape", what);
  return SAM3_OK;
}

sam3_status_t kv_append(sam3_ctx_t* ctx, const sam3_kv_cache_t* c, int dtype, const uint16_t* k,
                        int64_t k_stride, const uint16_t* v, int64_t v_stride,
                        const int32_t* cu_new, int n_seqs, int rows, int max_new,
                        const int32_t* table, int table_stride, const int32_t* lens) {
  sam3_status_t st = check_kv_cache(ctx, c, "kv_append");
  if (st != SAM3_OK) return st;
  if (!k || !v || !table || !lens)
    return set_error(ctx, SAM3_ERR_INVALID_ARG, "kv_append: null pointer");
  if (dtype != SAM3_F16 && dtype != SAM3_BF16)
    return set_error(ctx, SAM3_ERR_INVALID_ARG, "kv_append: unknown dtype %d", dtype);
  if (!aligned16(k) || !aligned16(v))
    return set_error(ctx, SAM3_ERR_INVALID_ARG, "kv_append: rows must be 16-byte aligned");
  const int64_t width = (int64_t)c->kv_heads * c->head_dim;
  if (!stride_ok(k_stride, width) || !stride_ok(v_stride, width))
    return set_error(ctx, SAM3_ERR_SHAPE,
                     "kv_append: row strides must be multiples of 8 of at least kv_heads * head_dim");
  if (n_seqs <= 0 || n_seqs > 65535 || rows <= 0 || max_new <= 0 || max_new > rows ||
      table_stride <= 0 || (long long)table_stride * c->page_size > kMaxContext ||
      (!cu_new && (max_new != 1 || rows < n_seqs)))
    return set_error(ctx, SAM3_ERR_SHAPE, "kv_append: bad shape");
  AppendArgs a;
  a.k_codes = c->k;
  a.v_codes = c->v;
  a.k_scale = c->k_scale;
  a.v_scale = c->v_scale;
  a.k = k;
  a.v = v;
  a.k_stride = k_stride;
  a.v_stride = v_stride;
  a.cu = cu_new;
  a.lens = lens;
  a.table = table;
  a.table_stride = table_stride;
  a.num_pages = c->num_pages;
  a.kv_heads = c->kv_heads;
  a.page_shift = __builtin_ctz((unsigned)c->page_size);
  a.rows = rows;
  a.max_new = max_new;
  a.err = ctx->dev_err;
  ProfScope prof(ctx, SAM3_PROF_OTHER, 0.0, 6.0 * rows * width);
  const bool bf = dtype == SAM3_BF16;
  cudaError_t e;
  // A lane holds 64 elements (8 vectors): a unit takes as many warps as that
  // makes, or a warp two of the smallest units.
  switch (c->page_size * c->head_dim) {
    case 16 * 64: e = launch_append<64, 1, 2, 4>(ctx, bf, a, n_seqs); break;
    case 32 * 64:
      e = c->head_dim == 64 ? launch_append<64, 1, 1, 8>(ctx, bf, a, n_seqs)
                            : launch_append<128, 1, 1, 8>(ctx, bf, a, n_seqs);
      break;
    case 64 * 64:
      e = c->head_dim == 64 ? launch_append<64, 2, 1, 8>(ctx, bf, a, n_seqs)
                            : launch_append<128, 2, 1, 8>(ctx, bf, a, n_seqs);
      break;
    case 128 * 64:
      e = c->head_dim == 64 ? launch_append<64, 4, 1, 8>(ctx, bf, a, n_seqs)
                            : launch_append<128, 4, 1, 8>(ctx, bf, a, n_seqs);
      break;
    default: e = launch_append<128, 8, 1, 8>(ctx, bf, a, n_seqs); break;
  }
  return check_launch_ret(ctx, e, "kv_append_kernel");
}

}  // namespace sam3

using namespace sam3;

extern "C" sam3_status_t sam3_kv_append(sam3_ctx_t* ctx, const sam3_kv_cache_t* cache,
                                        int32_t dtype, const uint16_t* k, int64_t k_stride,
                                        const uint16_t* v, int64_t v_stride, const int32_t* cu_new,
                                        int32_t n_seqs, int32_t rows, int32_t max_new,
                                        const int32_t* page_table, int32_t table_stride,
                                        const int32_t* seq_lens) {
  SAM3_CHECK_CTX(ctx);
  cudaSetDevice(ctx->device);
  return kv_append(ctx, cache, dtype, k, k_stride, v, v_stride, cu_new, n_seqs, rows, max_new,
                   page_table, table_stride, seq_lens);
}
