// lr_paged_attention: softmax attention of a call's rows on the pages of a key-value cache.
#include "paged_common.h"

struct PagedQuery {
  const u16* q;
  int64_t ldq;
  u16* y;
  int64_t ldy;
  int rows, Hq;
  float scale;
};

// One wave per (row, q head): 64 keys at a time, a lane one key's score, then 64 values weighted, a lane HD / 64 dimensions.
template <int HD, bool E4M3>
__global__ __launch_bounds__(64) void k_paged_attention(const PagedCache c, const PagedBatch t, const PagedQuery a) {
  constexpr int ROW = HD * (E4M3 ? 1 : 2), D = HD / 64;
  const int row = blockIdx.x, h = blockIdx.y, kvh = h / (a.Hq / c.Hkv), lane = threadIdx.x;
  int b = row, back = 1;
  if (t.starts) {
    b = paged_sequence(t, row);
    if (b >= t.B) return;
    back = t.starts[b + 1] - row;
  }
  const int seen = paged_length(t, c.shift, b) - back + 1;   // keys
  const u16* const q = a.q + row * a.ldq + h * HD;
  float m = -INFINITY, l = 0.0f, o[D] = {};
  for (int k0 = 0; k0 < seen; k0 += 64) {
    const int key = k0 + lane;
    int page = -1;
    if (key < seen) {
      page = t.table[b * t.ld_table + (key >> c.shift)];
      if (page < 0 || page >= c.n_pages) {
        page = -1;
        if (t.err) *t.err = LR_DEV_PAGE_RANGE;
      }
    }
    const int slot = key & ((1 << c.shift) - 1);
    float s = -INFINITY, vs = 1.0f;
    if (page >= 0) {
      const u8* const k = c.k + paged_offset<ROW>(c, page, kvh) + slot * ROW;
      float sum = 0.0f;
      for (int d = 0; d < HD; ++d) {
        float x;
        if constexpr (E4M3) x = __builtin_amdgcn_cvt_f32_fp8(k[d], 0);
        else x = bf_to_f(reinterpret_cast<const u16*>(k)[d]);
        sum = fmaf(x, bf_to_f(q[d]), sum);
      }
      s = sum * a.scale;
      if constexpr (E4M3) {
        const u8* const e = c.scales + paged_scales(c, page, kvh) + slot;
        s *= paged_scale(e[0]);
        vs = paged_scale(e[1 << c.shift]);
      }
    }
    const float mn = fmaxf(m, wave_max(s));
    if (mn == -INFINITY) continue;
    const float corr = expf(m - mn), p = expf(s - mn);
    m = mn;
    l = l * corr + wave_sum(p);
#pragma unroll
    for (int i = 0; i < D; ++i) o[i] *= corr;
    for (int j = 0; j < 64; ++j) {
      const int pj = __builtin_amdgcn_readlane(page, j);
      if (pj < 0) continue;
      const float w = lr_lane(p, j) * lr_lane(vs, j);
      const u8* const v = c.v + paged_offset<ROW>(c, pj, kvh) + ((k0 + j) & ((1 << c.shift) - 1)) * ROW;
#pragma unroll
      for (int i = 0; i < D; ++i) {
        float x;
        if constexpr (E4M3) x = __builtin_amdgcn_cvt_f32_fp8(v[i * 64 + lane], 0);
        else x = bf_to_f(reinterpret_cast<const u16*>(v)[i * 64 + lane]);
        o[i] = fmaf(w, x, o[i]);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < D; ++i) a.y[row * a.ldy + h * HD + i * 64 + lane] = f_to_bf(l != 0.0f ? o[i] / l : 0.0f);
}

extern "C" size_t lr_paged_attention_scratch_bytes(const lr_paged_cache_t* cache, const lr_paged_batch_t* batch, int rows, int Hq) {
  PagedCache c;
  PagedBatch t;
  if (paged_arguments(cache, batch, c, t) || rows <= 0 || Hq <= 0 || Hq % c.Hkv) return 0;
  return 256;
}

extern "C" int lr_paged_attention(const lr_paged_cache_t* cache, const lr_paged_batch_t* batch, const void* q, int64_t ldq, void* y, int64_t ldy,
                                  int rows, int Hq, float scale, void* scratch, size_t scratch_bytes, lr_stream_t stream) {
  PagedCache c;
  PagedBatch t;
  if (const int rc = paged_arguments(cache, batch, c, t)) return rc;
  LR_REQUIRE_PTR(q);
  LR_REQUIRE_PTR(y);
  LR_REQUIRE_PTR(scratch);
  const int hd = cache->head_dim;
  if (rows <= 0 || Hq <= 0 || Hq % c.Hkv || (t.starts == nullptr && rows != t.B)) return LR_E_SHAPE;
  if (Hq > 65535 || ldq < (int64_t)Hq * hd || ldy < (int64_t)Hq * hd || !(scale > 0.0f && scale < INFINITY)) return LR_E_SHAPE;
  if (ldq % 8 || ldy % 8) return LR_E_ALIGN;
  if (scratch_bytes < lr_paged_attention_scratch_bytes(cache, batch, rows, Hq)) return LR_E_SHAPE;
  const PagedQuery a = {(const u16*)q, ldq, (u16*)y, ldy, rows, Hq, scale};
  const dim3 grid((unsigned)rows, (unsigned)Hq);
  hipStream_t s = (hipStream_t)stream;
  const bool e4m3 = cache->format == LR_CACHE_E4M3;
  if (hd == 128 && e4m3) k_paged_attention<128, true><<<grid, dim3(64), 0, s>>>(c, t, a);
  else if (hd == 128) k_paged_attention<128, false><<<grid, dim3(64), 0, s>>>(c, t, a);
  else if (e4m3) k_paged_attention<64, true><<<grid, dim3(64), 0, s>>>(c, t, a);
  else k_paged_attention<64, false><<<grid, dim3(64), 0, s>>>(c, t, a);
  return lr_launch_status();
}
