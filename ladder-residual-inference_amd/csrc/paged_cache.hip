// lr_paged_write and lr_paged_read: rows of a call into the pages of a key-value cache, and back.
//
// Both move every byte once and compute next to nothing: memory-bound, and in a decode step bound by the launch and two dependent
// reads (where the row belongs, then its page).  A lane has 8 elements of a head's row (16 bytes of bf16), HD / 8 lanes a row.
// Six prompts of the 8B model into e4m3, 110 MB: 23.3 us, 4.7 TB/s (a large copy 5.05); 16 sequences of it read back, 116 MB: 20.0 us, 5.8 TB/s; a row of
// one sequence, or of 64: 6.0 us from Python, most of it the call (in a captured graph 2.4 and 4.0).
#include "paged_common.h"

constexpr int PAGED_TOKENS = 16;   // of a workgroup, at most
constexpr int PAGED_AHEAD = 4;     // rows that a lane of a write asks for before it works on the first (two: four prompts of the 70B model's shard 8.4 -> 9.3 us)
constexpr int PAGED_AHEAD_READ = 2;   // of a read (four: 333 tokens of 8 heads of 64 2.7 -> 3.2 us)

// Where a workgroup's tokens belong.  page -1: the token is left alone.
struct PagedPlace {
  int pos[PAGED_TOKENS], page[PAGED_TOKENS];
};
// `limit`: positions from there on have no angle.  A token ahead of the first sequence or behind the last, or an empty place of a batch, has no place and is no
// error; a position or a page that is out of range is one.  A wave looks after every fourth token, and lane j of it after its j-th.
__device__ __forceinline__ void paged_places(const PagedCache& c, const PagedBatch& t, int row0, int rows, int tokens, int limit, PagedPlace& at) {
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int i = wave + 4 * lane, row = row0 + i;
  int b = row, begin = 0;
  if (t.starts) {
    b = 0;
    begin = t.starts[0];   // (asked for with the first ends; where starts[b] was asked for behind the search, 16 sequences read back took 20.5 us instead of 20.0)
    for (int i0 = 0; i0 < t.B; i0 += 64) {   // as many sequences as have ended by then: 64 of them at a time
      const int end = i0 + lane < t.B ? t.starts[i0 + lane + 1] : 0x7fffffff;
      int most = 0;
      for (int j = 0; wave + 4 * j < tokens; ++j) {
        const int n = __popcll(__ballot(end <= row0 + wave + 4 * j));
        if (lane == j) b += n;
        most = n > most ? n : most;
      }
      if (most < 64) break;
    }
  }
  if (i < tokens) {
    int page = -1, pos = 0;
    if (row >= begin && row < rows && b < t.B) {
      const int length = t.lengths[b];
      pos = length - ((t.starts ? t.starts[b + 1] : row + 1) - row);
      int code = 0;
      if (pos < 0 || pos >> c.shift >= t.pages || pos >= limit) {
        code = t.starts || length != 0 ? LR_DEV_POS_RANGE : 0;
      } else {
        page = t.table[(int64_t)b * t.ld_table + (pos >> c.shift)];
        if (page < 0 || page >= c.n_pages) code = LR_DEV_PAGE_RANGE, page = -1;
      }
      if (code && t.err) *t.err = code;
    }
    at.pos[i] = pos;
    at.page[i] = page;
  }
  __syncthreads();
}

// The largest of a row's HD / 8 lanes, in all of them: exchanges within 16 lanes on the vector unit.
template <int HD>
__device__ __forceinline__ float row_max(float v) {
  v = fmaxf(v, lr_dpp<0xb1>(v));    // quad_perm [1,0,3,2]
  v = fmaxf(v, lr_dpp<0x4e>(v));    // quad_perm [2,3,0,1]
  v = fmaxf(v, lr_dpp<0x141>(v));   // row_half_mirror: 8 lanes
  if (HD == 128) v = fmaxf(v, lr_dpp<0x140>(v));   // row_mirror: 16 lanes
  return v;
}

struct PagedWrite {
  const u16* x;
  int64_t ldx;
  u16* q;
  int64_t ldq;
  const void* rope;
  int rope_len, rot, rows, Hq, tokens;
};

// The angles that a lane's 8 elements from d on take, (cos, sin) pairs as they lie: 4 of them where a pair is two neighbours (PAIRS), else 8, of
// element i and i + rot / 2.
template <bool PAIRS, typename T>
struct PagedAngles {
  static constexpr int N = PAIRS ? 8 : 16, LOADS = N * (int)sizeof(T) / 16;
  uint4 raw[LOADS];
  __device__ __forceinline__ void load(const void* rope, int pos, int rot, int d) {
    const T* const from = (const T*)rope + (int64_t)pos * rot + (PAIRS ? d : 2 * (d >= rot >> 1 ? d - (rot >> 1) : d));
#pragma unroll
    for (int i = 0; i < LOADS; ++i) raw[i] = ld16(reinterpret_cast<const unsigned char*>(from) + 16 * i);
  }
  __device__ __forceinline__ void values(float* t) const {
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      if constexpr (sizeof(T) == 2) {
        unpack8(raw[i], t + 8 * i);
      } else {
        t[4 * i] = __uint_as_float(raw[i].x);
        t[4 * i + 1] = __uint_as_float(raw[i].y);
        t[4 * i + 2] = __uint_as_float(raw[i].z);
        t[4 * i + 3] = __uint_as_float(raw[i].w);
      }
    }
  }
};

// x[lo] c - x[hi] s and x[hi] c + x[lo] s for the 8 elements x from d on, each product rounded by itself (as lr_rope_kv_write does it).  The other
// halves are rot / 16 lanes away.
template <bool PAIRS, typename T>
__device__ __forceinline__ void paged_turn(float* f, const uint4& x, int d, const PagedAngles<PAIRS, T>& angles, int rot) {
#pragma clang fp contract(off)
  float t[PagedAngles<PAIRS, T>::N];
  angles.values(t);
  if constexpr (PAIRS) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float a = f[2 * i], b = f[2 * i + 1], c = t[2 * i], s = t[2 * i + 1];
      f[2 * i] = a * c - b * s;
      f[2 * i + 1] = b * c + a * s;
    }
  } else {
    const bool second = d >= rot >> 1;
    const int from = (int)(threadIdx.x & 63) + (second ? -(rot >> 4) : rot >> 4);
    float o[8];
    unpack8(make_uint4(__shfl(x.x, from, 64), __shfl(x.y, from, 64), __shfl(x.z, from, 64), __shfl(x.w, from, 64)), o);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float p = f[j] * t[2 * j], r = o[j] * t[2 * j + 1];
      f[j] = second ? p + r : p - r;
    }
  }
}

template <int HD, bool E4M3, bool PAIRS, typename T>
__global__ __launch_bounds__(256) void k_paged_write(const PagedCache c, const PagedBatch t, const PagedWrite w) {
  __shared__ PagedPlace at;
  const int row0 = blockIdx.x * w.tokens;
  paged_places(c, t, row0, w.rows, w.tokens, w.rope ? w.rope_len : 0x7fffffff, at);
  constexpr int LANES = HD / 8, ROWS = 256 / LANES;
  const int heads = w.Hq + 2 * c.Hkv, d = threadIdx.x % LANES * 8, n = w.tokens * heads;
  PagedAngles<PAIRS, T> angles;   // of token `turned`, asked for behind its first rows: once for all heads (six prompts, by halves in fp32: 33.1 -> 25.5 us)
  int turned = -1;
  for (int i0 = threadIdx.x / LANES; i0 < n; i0 += ROWS * PAGED_AHEAD) {   // (all lanes of a row go round together)
    uint4 x[PAGED_AHEAD];
#pragma unroll
    for (int u = 0; u < PAGED_AHEAD; ++u) {
      const int i = i0 + u * ROWS < n ? i0 + u * ROWS : i0, token = i / heads, head = i - token * heads;
      x[u] = ld16_once(w.x + (at.page[token] >= 0 ? row0 + token : 0) * w.ldx + head * HD + d);
    }
    const int token0 = i0 / heads;
    if (w.rope && d < w.rot && turned != token0 && at.page[token0] >= 0) {
      angles.load(w.rope, at.pos[token0], w.rot, d);
      turned = token0;
    }
#pragma unroll
    for (int u = 0; u < PAGED_AHEAD; ++u) {
      const int i = i0 + u * ROWS;
      if (i >= n) break;
      const int token = i / heads, head = i - token * heads, page = at.page[token];
      if (page < 0) continue;
      const int pos = at.pos[token];
      float f[8];
      unpack8(x[u], f);
      if (w.rope && head < w.Hq + c.Hkv && d < w.rot) {
        if (turned != token) {
          angles.load(w.rope, pos, w.rot, d);
          turned = token;
        }
        paged_turn(f, x[u], d, angles, w.rot);
      }
      if (head < w.Hq) {
        // (qkv and q non-temporal: 26.7 -> 24.4 us of those prompts.  k and v are not: 23.2, but the attention behind it 16 us longer)
        const uint4 o = pack8(f);
        __builtin_nontemporal_store(u32x4_t{o.x, o.y, o.z, o.w}, reinterpret_cast<u32x4_t*>(w.q + (row0 + token) * w.ldq + head * HD + d));
        continue;
      }
      const int value = head >= w.Hq + c.Hkv, kvh = head - w.Hq - value * c.Hkv, slot = pos & ((1 << c.shift) - 1);
      u8* const to = (value ? c.v : c.k) + paged_offset<HD * (E4M3 ? 1 : 2)>(c, page, kvh);
      if constexpr (!E4M3) {
        st16(to + (slot * HD + d) * 2, pack8(f));
      } else {
        float amax = 0.0f;
#pragma unroll
        for (int j = 0; j < 8; ++j) amax = fmaxf(amax, fabsf(f[j]) < INFINITY ? fabsf(f[j]) : 0.0f);
        amax = row_max<HD>(amax);
        const u32 byte = paged_exponent(amax);
        const float inv = paged_inverse(byte);
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j] = fabsf(f[j]) < INFINITY ? f[j] * inv : NAN;   // (e4m3 has no infinities)
        u32x2_t o;
        o.x = __builtin_amdgcn_cvt_pk_fp8_f32(f[2], f[3], __builtin_amdgcn_cvt_pk_fp8_f32(f[0], f[1], 0, false), true);
        o.y = __builtin_amdgcn_cvt_pk_fp8_f32(f[6], f[7], __builtin_amdgcn_cvt_pk_fp8_f32(f[4], f[5], 0, false), true);
        *reinterpret_cast<u32x2_t*>(to + slot * HD + d) = o;
        if (d == 0) c.scales[paged_scales(c, page, kvh) + (value << c.shift) + slot] = (u8)byte;
      }
    }
  }
}

struct PagedRead {
  u16 *k, *v;
  int64_t ldk, ldv;
  int rows, tokens;
};

template <int HD, bool E4M3>
__global__ __launch_bounds__(256) void k_paged_read(const PagedCache c, const PagedBatch t, const PagedRead r) {
  __shared__ PagedPlace at;
  const int row0 = blockIdx.x * r.tokens;
  paged_places(c, t, row0, r.rows, r.tokens, 0x7fffffff, at);
  constexpr int LANES = HD / 8, ROWS = 256 / LANES;
  const int d = threadIdx.x % LANES * 8, n = r.tokens * 2 * c.Hkv;
  for (int i0 = threadIdx.x / LANES; i0 < n; i0 += ROWS * PAGED_AHEAD_READ) {
    uint4 x[PAGED_AHEAD_READ];   // (e4m3: eight bytes)
    u32 byte[PAGED_AHEAD_READ];
#pragma unroll
    for (int u = 0; u < PAGED_AHEAD_READ; ++u) {
      const int i = i0 + u * ROWS < n ? i0 + u * ROWS : i0, token = i / (2 * c.Hkv), j = i - token * 2 * c.Hkv, value = j >= c.Hkv, kvh = j - value * c.Hkv;
      const int page = at.page[token] < 0 ? 0 : at.page[token], slot = at.page[token] < 0 ? 0 : at.pos[token] & ((1 << c.shift) - 1);
      const u8* const from = (value ? c.v : c.k) + paged_offset<HD * (E4M3 ? 1 : 2)>(c, page, kvh);
      if constexpr (!E4M3) {
        x[u] = ld16(from + (slot * HD + d) * 2);
      } else {
        const u32x2_t raw = *reinterpret_cast<const u32x2_t*>(from + slot * HD + d);
        x[u].x = raw.x;
        x[u].y = raw.y;
        byte[u] = c.scales[paged_scales(c, page, kvh) + (value << c.shift) + slot];
      }
    }
#pragma unroll
    for (int u = 0; u < PAGED_AHEAD_READ; ++u) {
      const int i = i0 + u * ROWS;
      if (i >= n) break;
      const int token = i / (2 * c.Hkv), j = i - token * 2 * c.Hkv, value = j >= c.Hkv, kvh = j - value * c.Hkv;
      if (at.page[token] < 0) continue;
      uint4 o = x[u];
      if constexpr (E4M3) {
        const float s = paged_scale(byte[u]);
        o.x = __builtin_bit_cast(u32, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x[u].x, s, false));
        o.y = __builtin_bit_cast(u32, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x[u].x, s, true));
        o.z = __builtin_bit_cast(u32, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x[u].y, s, false));
        o.w = __builtin_bit_cast(u32, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x[u].y, s, true));
      }
      // (non-temporal: those 16 sequences 27.5 -> 21.2 us)
      u16* const to = (value ? r.v + (row0 + token) * r.ldv : r.k + (row0 + token) * r.ldk) + kvh * HD + d;
      __builtin_nontemporal_store(u32x4_t{o.x, o.y, o.z, o.w}, reinterpret_cast<u32x4_t*>(to));
    }
  }
}

// Tokens of a workgroup, which share the search for their places: as many as its lanes ask for at once (`heads` rows of a token), where that leaves each of
// 256 CUs two workgroups.  us, 6 prompts of the 8B model (48 rows of q, k and v per token) written with 1, 2 and 4 tokens: 23.5, 26.1, 27.3; 4 of
// the 70B model's rank shard (10 rows) with 1, 4, 6 and 12: 14.6, 11.2, 8.4, 11.8; 16 sequences of the 8B model read back (16 rows) with 2, 4 and 8: 20.1, 20.1, 22.1.
template <int AHEAD>
static inline int paged_tokens(int rows, int heads, int hd) {
  const int n = rows / (2 * 256), fit = 256 / (hd / 8) * AHEAD / heads, most = fit < PAGED_TOKENS ? fit : PAGED_TOKENS;
  return n < 1 || most < 1 ? 1 : n > most ? most : n;
}

// (0: a grid of 2^32 threads or more, which a launch has not)
static inline unsigned paged_workgroups(int rows, int tokens) {
  const int64_t n = ((int64_t)rows + tokens - 1) / tokens;
  return n > 0xffffffff / 256 ? 0 : (unsigned)n;
}

template <int HD, bool E4M3, bool PAIRS>
static void launch_write(bool f32, unsigned grid, const PagedCache& c, const PagedBatch& t, const PagedWrite& w, hipStream_t s) {
  if (f32) k_paged_write<HD, E4M3, PAIRS, float><<<dim3(grid), dim3(256), 0, s>>>(c, t, w);
  else k_paged_write<HD, E4M3, PAIRS, u16><<<dim3(grid), dim3(256), 0, s>>>(c, t, w);
}

extern "C" int lr_paged_write(const lr_paged_write_t* desc, lr_stream_t stream) {
  if (desc == nullptr) return LR_E_NULL;
  const auto& [cache, batch, qkv, ldqkv, q, ldq, rope, rows, Hq, rope_len, rot, interleaved, rope_dtype] = *desc;
  PagedCache c;
  PagedBatch t;
  if (const int rc = paged_arguments(cache, batch, c, t)) return rc;
  LR_REQUIRE_PTR(qkv);
  LR_REQUIRE_PTR(q);
  LR_OPTIONAL_PTR(rope);
  const int hd = cache->head_dim;
  if (rows <= 0 || Hq <= 0 || Hq % c.Hkv || (t.starts == nullptr && rows != t.B)) return LR_E_SHAPE;
  if (Hq > 65535 / 3 || ldqkv < (int64_t)(Hq + 2 * c.Hkv) * hd || ldq < (int64_t)Hq * hd) return LR_E_SHAPE;
  if (ldqkv % 8 || ldq % 8) return LR_E_ALIGN;
  const int tokens = paged_tokens<PAGED_AHEAD>(rows, Hq + 2 * c.Hkv, hd);
  const unsigned grid = paged_workgroups(rows, tokens);
  if (grid == 0) return LR_E_UNSUPPORTED;
  const bool in_place = q == qkv && (ldq == ldqkv || rows == 1);
  if (!in_place && paged_overlap(qkv, ldqkv, q, ldq, rows, (int64_t)(Hq + 2 * c.Hkv) * hd, (int64_t)Hq * hd)) return LR_E_SHAPE;
  if (rope && (rope_len <= 0 || rot <= 0 || rot > hd)) return LR_E_SHAPE;
  if (rope && (rot % 16 || (rope_dtype != LR_BF16 && rope_dtype != LR_F32))) return LR_E_UNSUPPORTED;
  const PagedWrite w = {(const u16*)qkv, ldqkv, (u16*)q, ldq, rope, rope_len, rot, rows, Hq, tokens};
  const bool f32 = rope_dtype == LR_F32;
  hipStream_t s = (hipStream_t)stream;
  const bool e4m3 = cache->format == LR_CACHE_E4M3;
#define LR_WRITE(HDV, E, P) \
  if (hd == HDV && e4m3 == E && (interleaved != 0) == P) launch_write<HDV, E, P>(f32, grid, c, t, w, s);
  LR_WRITE(64, false, false) LR_WRITE(64, false, true) LR_WRITE(64, true, false) LR_WRITE(64, true, true)
  LR_WRITE(128, false, false) LR_WRITE(128, false, true) LR_WRITE(128, true, false) LR_WRITE(128, true, true)
#undef LR_WRITE
  return lr_launch_status();
}

extern "C" int lr_paged_read(const lr_paged_read_t* desc, lr_stream_t stream) {
  if (desc == nullptr) return LR_E_NULL;
  const auto& [cache, batch, k, ldk, v, ldv, rows] = *desc;
  PagedCache c;
  PagedBatch t;
  if (const int rc = paged_arguments(cache, batch, c, t)) return rc;
  LR_REQUIRE_PTR(k);
  LR_REQUIRE_PTR(v);
  const int hd = cache->head_dim;
  if (rows <= 0 || (t.starts == nullptr && rows != t.B) || c.Hkv > 65535) return LR_E_SHAPE;
  if (ldk < (int64_t)c.Hkv * hd || ldv < (int64_t)c.Hkv * hd) return LR_E_SHAPE;
  if (ldk % 8 || ldv % 8) return LR_E_ALIGN;
  const int tokens = paged_tokens<PAGED_AHEAD_READ>(rows, 2 * c.Hkv, hd);
  const unsigned grid = paged_workgroups(rows, tokens);
  if (grid == 0) return LR_E_UNSUPPORTED;
  if (paged_overlap(k, ldk, v, ldv, rows, (int64_t)c.Hkv * hd, (int64_t)c.Hkv * hd)) return LR_E_SHAPE;
  const PagedRead r = {(u16*)k, (u16*)v, ldk, ldv, rows, tokens};
  hipStream_t s = (hipStream_t)stream;
  const bool e4m3 = cache->format == LR_CACHE_E4M3;
  if (hd == 128 && e4m3) k_paged_read<128, true><<<dim3(grid), dim3(256), 0, s>>>(c, t, r);
  else if (hd == 128) k_paged_read<128, false><<<dim3(grid), dim3(256), 0, s>>>(c, t, r);
  else if (e4m3) k_paged_read<64, true><<<dim3(grid), dim3(256), 0, s>>>(c, t, r);
  else k_paged_read<64, false><<<dim3(grid), dim3(256), 0, s>>>(c, t, r);
  return lr_launch_status();
}
