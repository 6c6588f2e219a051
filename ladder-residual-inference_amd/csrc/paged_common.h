// What the kernels of the paged key-value cache share (lr_paged_write, lr_paged_read, lr_paged_attention): where a row of the call
// belongs, where a token lies, and the 8-bit rows.
#pragma once
#include "lr_common.h"

typedef uint8_t u8;

struct PagedCache {
  u8 *k, *v, *scales;   // bytes; scales [n_pages][Hkv][2][page]
  int n_pages, shift, Hkv;   // page == 1 << shift
};
struct PagedBatch {
  const int32_t *table, *lengths, *starts;
  int64_t ld_table;
  int B, pages;
  int32_t* err;
};

// A sequence's keys: none for a negative length, no more than its pages hold.
__device__ __forceinline__ int paged_length(const PagedBatch& t, int shift, int b) {
  const int n = t.lengths[b], most = t.pages << shift;
  if (n > most && t.err) *t.err = LR_DEV_POS_RANGE;
  return n < 0 ? 0 : n > most ? most : n;
}

// Inclusive sums over a wave's lanes, on the vector unit.
template <int CTRL, int ROWS>
__device__ __forceinline__ int paged_dpp0(int v) { return __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xf, false); }
__device__ __forceinline__ int paged_sums(int v) {
  v += paged_dpp0<0x111, 0xf>(v);   // row_shr:1, 2, 4, 8: within 16 lanes
  v += paged_dpp0<0x112, 0xf>(v);
  v += paged_dpp0<0x114, 0xf>(v);
  v += paged_dpp0<0x118, 0xf>(v);
  v += paged_dpp0<0x142, 0xa>(v);   // row_bcast:15: lane 15 to row 1, 47 to row 3
  v += paged_dpp0<0x143, 0xc>(v);   // row_bcast:31: to rows 2 and 3
  return v;
}

// (page, kv head) as one number of 32 bits, and the bytes from the start of k, v to its slot 0
__device__ __forceinline__ int paged_index(const PagedCache& c, int page, int head) { return page * c.Hkv + head; }
template <int ROW>
__device__ __forceinline__ int64_t paged_offset(const PagedCache& c, int index) { return ((int64_t)index << c.shift) * ROW; }
template <int ROW>
__device__ __forceinline__ int64_t paged_offset(const PagedCache& c, int page, int head) { return paged_offset<ROW>(c, paged_index(c, page, head)); }
// and of the scales, to those of the page's keys; its values' follow
__device__ __forceinline__ int64_t paged_scales(const PagedCache& c, int index) { return (int64_t)index << (c.shift + 1); }
__device__ __forceinline__ int64_t paged_scales(const PagedCache& c, int page, int head) { return paged_scales(c, paged_index(c, page, head)); }

// An 8-bit row holds x / 2^e as e4m3, e the smallest exponent with max|x| <= 448 * 2^e, kept as the byte e + 127.  A power of two: dividing
// and multiplying by it rounds nothing, so a value is rounded once, and what is read back is exact in bf16.  (amax: the largest finite
// magnitude; 448 = 1.75 * 2^8.  Bytes from 1 on, so that 2^e and 2^-e are normal numbers.)
__device__ __forceinline__ u32 paged_exponent(float amax) {
  const u32 u = __float_as_uint(amax);
  const int e = (int)(u >> 23) - 8 + ((u & 0x7fffffu) > 0x600000u);
  return e < 1 ? 1u : (u32)e;
}
__device__ __forceinline__ float paged_scale(u32 byte) { return __uint_as_float(byte << 23); }
__device__ __forceinline__ float paged_inverse(u32 byte) { return __uint_as_float((254u - byte) << 23); }

// Whether two matrices of `rows` rows of bf16, a of `wa` and b of `wb` elements each, have memory in common.  Columns of one matrix have not.
static inline bool paged_overlap(const void* a, int64_t lda, const void* b, int64_t ldb, int rows, int64_t wa, int64_t wb) {
  typedef __int128 wide;
  if (rows == 1) lda = ldb = wa > wb ? wa : wb;
  const wide a0 = (uintptr_t)a, b0 = (uintptr_t)b, a1 = a0 + ((wide)(rows - 1) * lda + wa) * 2, b1 = b0 + ((wide)(rows - 1) * ldb + wb) * 2;
  if (a1 <= b0 || b1 <= a0) return false;
  if (lda != ldb) return true;
  const wide ld = (wide)lda * 2, off = ((b0 - a0) % ld + ld) % ld;   // where b's rows begin in a's
  return off < wa * 2 || off + wb * 2 > ld;
}

// Checks of the descriptors that the entry points share; fills the kernels' forms of them.
static inline int paged_arguments(const lr_paged_cache_t* cache, const lr_paged_batch_t* batch, PagedCache& c, PagedBatch& t) {
  if (cache == nullptr || batch == nullptr) return LR_E_NULL;
  LR_REQUIRE_PTR(cache->k);
  LR_REQUIRE_PTR(cache->v);
  if (batch->table == nullptr || batch->lengths == nullptr) return LR_E_NULL;
  if (((uintptr_t)batch->table | (uintptr_t)batch->lengths | (uintptr_t)batch->starts | (uintptr_t)batch->err) & 3) return LR_E_ALIGN;
  if (cache->n_pages <= 0 || cache->n_kv_head <= 0 || cache->page <= 0 || cache->head_dim <= 0) return LR_E_SHAPE;
  if (batch->B <= 0 || batch->pages <= 0 || batch->ld_table < batch->pages) return LR_E_SHAPE;
  if (cache->format != LR_CACHE_BF16 && cache->format != LR_CACHE_E4M3) return LR_E_UNSUPPORTED;
  if (cache->format == LR_CACHE_E4M3) LR_REQUIRE_PTR(cache->scales);
  if (cache->head_dim != 64 && cache->head_dim != 128) return LR_E_UNSUPPORTED;
  if (cache->page < 16 || cache->page > 256 || (cache->page & (cache->page - 1))) return LR_E_UNSUPPORTED;
  // (positions, tiles of 32 keys of all sequences, and pages times heads are 32-bit numbers)
  if ((int64_t)cache->n_pages * cache->n_kv_head > 0x7fffffff) return LR_E_UNSUPPORTED;
  const int64_t most = (int64_t)batch->pages * cache->page;
  if (batch->B > 65535 || most > (1 << 30) || batch->B * (most / 32 + 8) >= 0x7fffffff) return LR_E_UNSUPPORTED;
  c.k = (u8*)cache->k;
  c.v = (u8*)cache->v;
  c.scales = (u8*)cache->scales;
  c.n_pages = cache->n_pages;
  c.shift = __builtin_ctz((unsigned)cache->page);
  c.Hkv = cache->n_kv_head;
  t.table = batch->table;
  t.lengths = batch->lengths;
  t.starts = batch->starts;
  t.ld_table = batch->ld_table;
  t.B = batch->B;
  t.pages = batch->pages;
  t.err = batch->err;
  return LR_OK;
}
