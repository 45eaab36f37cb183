// Host-side refusals of the packed-prompt and cache entry points, and the
// checks that their kernels make of lengths, offsets and page numbers, without
// a GPU: the context here is a plain object, and every call below is refused
// before it touches a device.
#include <stdio.h>

#include "../metal-sam-ios-experiments_b200/csrc/internal.h"

static int failed = 0;
#define EXPECT(cond)                                       \
  do {                                                     \
    if (!(cond)) {                                         \
      printf("line %d: %s\n", __LINE__, #cond);            \
      ++failed;                                            \
    }                                                      \
  } while (0)

struct Packed {
  int dtype = SAM3_F16;
  uintptr_t q = 4096, k = 4096, v = 4096, cu = 4096, o = 4096;
  int64_t qs = 512, ks = 256, vs = 256, os = 512;
  int n = 1, rows = 8, heads = 8, kv = 4, dim = 64;
  float scale = 0.125f;
  sam3_status_t call(sam3_ctx_t* c) const {
    return sam3_attention_packed(c, dtype, (uint16_t*)q, qs, (uint16_t*)k, ks, (uint16_t*)v, vs,
                                 (int32_t*)cu, n, rows, heads, kv, dim, scale, 1, (uint16_t*)o, os);
  }
};
struct Cached {
  sam3_kv_cache_t cache{(uint8_t*)4096, (uint8_t*)4096, (float*)4096, (float*)4096, 8, 16, 4, 64};
  int dtype = SAM3_F16;
  uintptr_t q = 4096, k = 4096, v = 4096, cu = 4096, table = 4096, lens = 4096, o = 4096;
  int64_t qs = 512, ks = 256, vs = 256, os = 512;
  int n = 1, rows = 8, max_new = 8, stride = 4, heads = 8;
  float scale = 0.125f;
  sam3_status_t append(sam3_ctx_t* c) const {
    return sam3_kv_append(c, &cache, dtype, (uint16_t*)k, ks, (uint16_t*)v, vs, (int32_t*)cu, n,
                          rows, max_new, (int32_t*)table, stride, (int32_t*)lens);
  }
  sam3_status_t attend(sam3_ctx_t* c) const {
    return sam3_attention_cached(c, &cache, dtype, (uint16_t*)q, qs, (int32_t*)cu, n, rows,
                                 max_new, (int32_t*)table, stride, (int32_t*)lens, heads, scale, 1,
                                 (uint16_t*)o, os);
  }
};

int main() {
  sam3_ctx ctx;
  const sam3_status_t ARG = SAM3_ERR_INVALID_ARG, SHAPE = SAM3_ERR_SHAPE;
#define PACKED(set, want)              \
  do {                                 \
    Packed p;                          \
    set;                               \
    ctx.last_error.clear();            \
    EXPECT(p.call(&ctx) == want);      \
    EXPECT(!ctx.last_error.empty());   \
  } while (0)
#define APPEND(set, want)              \
  do {                                 \
    Cached p;                          \
    set;                               \
    ctx.last_error.clear();            \
    EXPECT(p.append(&ctx) == want);    \
    EXPECT(!ctx.last_error.empty());   \
  } while (0)
#define ATTEND(set, want)              \
  do {                                 \
    Cached p;                          \
    set;                               \
    ctx.last_error.clear();            \
    EXPECT(p.attend(&ctx) == want);    \
    EXPECT(!ctx.last_error.empty());   \
  } while (0)
#define BOTH(set, want) \
  do {                  \
    APPEND(set, want);  \
    ATTEND(set, want);  \
  } while (0)

  EXPECT(Packed().call(nullptr) == ARG);
  EXPECT(Cached().append(nullptr) == ARG);
  EXPECT(Cached().attend(nullptr) == ARG);

  PACKED(p.q = 0, ARG);
  PACKED(p.k = 0, ARG);
  PACKED(p.v = 0, ARG);
  PACKED(p.cu = 0, ARG);
  PACKED(p.o = 0, ARG);
  PACKED(p.q += 8, ARG);
  PACKED(p.k += 2, ARG);
  PACKED(p.v += 8, ARG);
  PACKED(p.o += 4, ARG);
  PACKED(p.dtype = 2, ARG);
  PACKED(p.dtype = -1, ARG);
  PACKED(p.scale = 0.f, ARG);
  PACKED(p.scale = -1.f, ARG);
  PACKED(p.scale = __builtin_nanf(""), ARG);
  PACKED(p.scale = __builtin_inff(), ARG);
  PACKED(p.scale = 3e38f, ARG);  // infinite in base 2
  PACKED(p.dim = 96, SHAPE);
  PACKED(p.dim = 0, SHAPE);
  PACKED(p.kv = 3, SHAPE);
  PACKED(p.kv = 0, SHAPE);
  PACKED(p.heads = 0, SHAPE);
  PACKED(p.heads = 2, SHAPE);
  PACKED(p.qs = 504, SHAPE);   // narrower than the heads
  PACKED(p.qs = 516, SHAPE);   // not whole 16-byte groups
  PACKED(p.ks = 248, SHAPE);
  PACKED(p.vs = -256, SHAPE);
  PACKED(p.os = 0, SHAPE);
  PACKED(p.n = 0, SHAPE);
  PACKED(p.n = -1, SHAPE);
  PACKED(p.n = 65536, SHAPE);
  PACKED(p.rows = 0, SHAPE);
  PACKED(p.rows = -4, SHAPE);
  PACKED(p.rows = 0x7FFFFFFF, SHAPE);

  BOTH(p.cache.k = nullptr, ARG);
  BOTH(p.cache.v = nullptr, ARG);
  BOTH(p.cache.k_scale = nullptr, ARG);
  BOTH(p.cache.v_scale = nullptr, ARG);
  BOTH(p.cache.k += 8, ARG);
  BOTH(p.cache.v_scale = (float*)4098, ARG);
  BOTH(p.cache.page_size = 24, SHAPE);
  BOTH(p.cache.page_size = 256, SHAPE);
  BOTH(p.cache.page_size = 0, SHAPE);
  BOTH(p.cache.head_dim = 32, SHAPE);
  BOTH(p.cache.kv_heads = 0, SHAPE);
  BOTH(p.cache.num_pages = 0, SHAPE);
  BOTH(p.cache.num_pages = 0x7FFFFFFF, SHAPE);
  BOTH(p.table = 0, ARG);
  BOTH(p.lens = 0, ARG);
  BOTH(p.dtype = 7, ARG);
  BOTH(p.n = 0, SHAPE);
  BOTH(p.rows = 0, SHAPE);
  BOTH(p.max_new = 0, SHAPE);
  BOTH(p.max_new = 9, SHAPE);                         // more than rows
  BOTH(p.stride = 0, SHAPE);
  BOTH(p.stride = 0x7FFFFFFF, SHAPE);                 // positions beyond 32 bits
  BOTH((p.cu = 0, p.max_new = 2), SHAPE);             // one row per sequence only
  BOTH((p.cu = 0, p.max_new = 1, p.n = 9), SHAPE);    // fewer rows than sequences
  APPEND(p.k = 0, ARG);
  APPEND(p.v = 0, ARG);
  APPEND(p.k += 8, ARG);
  APPEND(p.ks = 128, SHAPE);
  APPEND(p.vs = 260, SHAPE);
  APPEND(p.n = 65536, SHAPE);
  ATTEND(p.q = 0, ARG);
  ATTEND(p.o = 0, ARG);
  ATTEND(p.q += 2, ARG);
  ATTEND(p.scale = 0.f, ARG);
  ATTEND(p.scale = 3e38f, ARG);
  ATTEND(p.heads = 6, SHAPE);
  ATTEND(p.heads = 0, SHAPE);
  ATTEND(p.qs = 256, SHAPE);
  ATTEND(p.os = 513, SHAPE);
  ATTEND(p.n = SAM3_CACHED_MAX_SEQS + 1, SHAPE);
  ATTEND((p.rows = p.max_new = 1 << 30, p.n = 1000, p.stride = 1 << 20), SHAPE);  // work beyond 32 bits

  using namespace sam3;
  const int big = 0x7FFFFFFF;
  EXPECT(rows_fit(0, 0, 5) && rows_fit(0, 5, 5) && rows_fit(5, 5, 5));
  EXPECT(!rows_fit(-1, 3, 5) && !rows_fit(3, 2, 5) && !rows_fit(3, 6, 5) && !rows_fit(6, 6, 5));
  EXPECT(!rows_fit(-big, big, 5) && !rows_fit(big, -big, 5) && !rows_fit(0, big, 5));
  EXPECT(tokens_fit(0, 3, 8, 3, 3, 1, 4) && tokens_fit(5, 8, 8, 3, 64, 4, 4));
  EXPECT(tokens_fit(2, 2, 8, 3, 0, 1, 4));             // no new tokens
  EXPECT(!tokens_fit(0, 4, 8, 3, 9, 4, 4));            // more new than max_new
  EXPECT(!tokens_fit(0, 3, 8, 3, 2, 4, 4));            // longer than its sequence
  EXPECT(!tokens_fit(0, 3, 8, 3, -1, 4, 4));
  EXPECT(!tokens_fit(0, 3, 8, 3, 65, 4, 4));           // more tokens than the table's pages
  EXPECT(!tokens_fit(0, 3, 8, 3, big, 4, 4) && !tokens_fit(0, 1, 8, 3, -big, 4, 4));
  EXPECT(tokens_fit(0, 1, 8, 3, 1 << 30, 1 << 23, 7));
  EXPECT(page_fits(0, 1) && page_fits(7, 8) && !page_fits(8, 8) && !page_fits(-1, 8));
  EXPECT(!page_fits(big, 8) && !page_fits(-big - 1, 8));

  if (!failed) printf("all checks passed\n");
  return failed != 0;
}
