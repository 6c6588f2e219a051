// lr_paged_attention: softmax attention of a call's rows on the pages of a key-value cache.
#include "paged_common.h"

#include <atomic>

typedef short i16x4_t __attribute__((ext_vector_type(4)));

struct PagedQuery {
  const u16* q;
  int64_t ldq;
  u16* y;
  int64_t ldy;
  int rows, Hq;
  float scale;
};

// ------------------------------------------------------------------------------------ one row per sequence
// All sequences' keys lie on one line of tiles of 32, sequence after sequence, and the workers of a kv head (workgroups of four waves) take
// equal parts of it, wherever sequences begin and end: batches of any lengths keep the chip evenly busy, and the host, which knows no
// length, launches the same grid always.  A part of a sequence leaves its maximum, sum and weighted values in the scratch, and whoever ends
// last puts a sequence's parts together (in their order: the same bits every time); a sequence inside one part is written directly.
//
// A wave streams tiles of its own through its own LDS (no barrier in the loop): rows come by loads straight into LDS, K's of the next tile
// as soon as K's of this one are in registers, V's likewise.  S[key][head] = K q^T and O^T[dim][head] += V^T P on the matrix cores
// (16x16x32, up to 16 q heads of the kv head are the columns): a lane holds eight scores of one head and, since the order of keys in a product
// is free, hands them on as the second product's operand without moving them.  Weights enter as two bf16 numbers (2^-16 of the
// weight).  e4m3: K is expanded with its row's power of two on the way to the product, V without, its power goes into the weight.
// Bound: memory.
typedef int i32x4_t __attribute__((ext_vector_type(4)));
typedef int i32x2_t __attribute__((ext_vector_type(2)));
__device__ __forceinline__ float exp2_hw(float x) { return __builtin_amdgcn_exp2f(x); }
constexpr float PAGED_TAU2 = 8.0f;   // log2 of the largest weight before the reference point of the exponentials moves
constexpr int PAGED_OUT = (int)0x80000000;   // an offset outside every resource: comes as zeros
constexpr int PAGED_COHERENT = 17;   // sc0 sc1: past this XCD's L2

__device__ __forceinline__ i32x4_t paged_resource(const u8* at) {
  return i32x4_t{(int)(u32)(unsigned long long)at, (int)(u32)((unsigned long long)at >> 32) & 0xffff, 0x7fffffff, 0x00020000};
}
// 16 (4) bytes per lane from resource + voff + soff to LDS address `lds` + 16 (4) * lane; counted by vmcnt, not by the compiler
__device__ __forceinline__ void paged_load16(const i32x4_t& res, int voff, int soff, u32 lds) {
  asm volatile("s_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds" ::"{m0}"(lds), "v"(voff), "s"(res), "s"(soff) : "memory");
}
__device__ __forceinline__ void paged_load4(const i32x4_t& res, int voff, int soff, u32 lds) {
  asm volatile("s_nop 0\n\tbuffer_load_dword %1, %2, %3 offen lds" ::"{m0}"(lds), "v"(voff), "s"(res), "s"(soff) : "memory");
}
template <int N>
__device__ __forceinline__ void paged_wait_loads() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"i"(N) : "memory");
}
__device__ __forceinline__ void paged_wait_lds() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

// Over the four rows of 16 lanes (lanes l, l + 16, l + 32, l + 48)
__device__ __forceinline__ float rows_max(float v) {
  const u32 u = __float_as_uint(v);
  auto a = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  const u32 w = __float_as_uint(v);
  a = __builtin_amdgcn_permlane16_swap(w, w, false, false);
  return fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
}
__device__ __forceinline__ float rows_sum(float v) {
  const u32 u = __float_as_uint(v);
  auto a = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
  const u32 w = __float_as_uint(v);
  a = __builtin_amdgcn_permlane16_swap(w, w, false, false);
  return __uint_as_float(a[0]) + __uint_as_float(a[1]);
}

template <int HD, bool E4M3>
struct DecodeTile {
  static constexpr int ROW = HD * (E4M3 ? 1 : 2), PIECES = ROW / 16;   // bytes of a row; its 16-byte pieces
  static constexpr int RPL = 64 / PIECES, LOADS = 32 / RPL;            // rows per load instruction; loads of a tile's K or V
  static constexpr int TILE = 32 * ROW, SCALES = E4M3 ? 512 : 0;       // (256 bytes for the 16-key halves' scales each)
  static constexpr int LDO = HD + 4;                                   // row length of the waves' results when they are put together
  static constexpr int WAVE = 2 * TILE + SCALES;
  static_assert(16 * LDO * 4 <= WAVE, "");
  static constexpr int PER_CU = HD == 64 ? 4 : E4M3 ? 3 : 2;            // workgroups that a CU holds, by LDS or registers
  static constexpr int LDS = 4 * WAVE + 512 + 16;   // (the waves' maxima and sums; a ticket)
  // which place among its row's pieces a piece has: its number XOR this.  16 lanes reading a piece of 16 consecutive keys, and 32 lanes
  // reading across the keys that V's products take (0..7 or 8..15 and, e4m3, 16 more), meet no bank of the 64 twice
  static __device__ __forceinline__ int k_place(int row) { return (row * PIECES / 16) & (PIECES - 1); }
  static __device__ __forceinline__ int v_place(int row) {
    if constexpr (!E4M3) return HD == 128 ? (row & 7) << 1 : ((row >> 1) & 3) << 1;
    else return HD == 128 ? ((row >> 1) & 3) | ((row >> 4) & 1) << 2 : ((row >> 2) & 1) | ((row >> 4) & 1) << 1;
  }
};

struct PagedDecode {
  const u16* q;
  int64_t ldq;
  u16* y;
  int64_t ldy;
  int Hq, groups_per_kv;   // of 16 q heads
  float scale;
  // results [16][HD] and their (maximum, sum) [16][2]: [group][worker][2] of a worker's first sequence, that began before it, and its last; then
  // [group][block][2] of blocks' likewise
  float *o_part, *ml_part;
  u32* tickets;   // [group][B], then [group][block][2]; zero between calls
};

// A sequence's parts are put together by the last of its workers, of no more than so many at a time: more go through their blocks' last ones.
constexpr int PAGED_BLOCK = 16;

template <int HD, bool E4M3>
__global__ __launch_bounds__(256, (DecodeTile<HD, E4M3>::PER_CU)) void k_paged_decode(const PagedCache c, const PagedBatch t, const PagedDecode a) {
  using T = DecodeTile<HD, E4M3>;
  constexpr int KS = HD / 32, DT = HD / 16;   // k-steps of a score product; 16-dimension tiles of O^T
  extern __shared__ __attribute__((aligned(1024))) unsigned char paged_lds[];
  float (*const s_ml)[16][2] = reinterpret_cast<float (*)[16][2]>(paged_lds + 4 * T::WAVE);   // [4]
  u32* const s_ticket = reinterpret_cast<u32*>(paged_lds + 4 * T::WAVE + 512);
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l16 = lane & 15, l4 = lane >> 4;
  const int group = blockIdx.y, kvh = group / a.groups_per_kv, G = a.Hq / c.Hkv;
  const int h0 = kvh * G + group % a.groups_per_kv * 16, left = (kvh + 1) * G - h0, nh = left < 16 ? left : 16;   // this group's q heads

  // ---- which tiles are this worker's
  int b0 = 0;   // lane i looks after sequence b0 + i
  int len, tiles;
  auto look = [&](int from) {
    b0 = from;
    len = b0 + lane < t.B ? paged_length(t, c.shift, b0 + lane) : 0;
    tiles = (len + 31) >> 5;
  };
  auto sum_to = [&](int v) {   // inclusive sums over the lanes
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int u = __shfl_up(v, o, 64);
      v += lane >= o ? u : 0;
    }
    return v;
  };
  int total = 0, upto = 0;
  for (int i = 0; i < t.B; i += 64) {
    look(i);
    upto = sum_to(tiles);
    total += __builtin_amdgcn_readlane(upto, 63);
    if (wave == 0) {   // empty places: zeros, one worker each
      unsigned long long empty = __ballot(i + lane < t.B && tiles == 0 && (i + lane) % gridDim.x == blockIdx.x);
      for (; empty; empty &= empty - 1) {
        u16* const y = a.y + (int64_t)(i + __builtin_ctzll(empty)) * a.ldy + h0 * HD;
        for (int d = lane * 8; d < nh * HD; d += 512) st16(y + d, make_uint4(0, 0, 0, 0));
      }
    }
  }
  const int workers = min((int)gridDim.x, (total + 3) >> 2), w = blockIdx.x;   // (four tiles at least: one for each wave)
  if (w >= workers) return;
  int at = (int)((int64_t)w * total / workers);
  const int end = (int)((int64_t)(w + 1) * total / workers);
  // the sequence that tile `at` belongs to: b0 + s, whose first tile is `first`
  int s, first;
  {
    int before = 0;
    if (t.B > 64) {
      for (int i = 0;; i += 64) {
        look(i);
        upto = sum_to(tiles);
        const int n = __builtin_amdgcn_readlane(upto, 63);
        if (at < before + n) break;
        before += n;
      }
    }
    s = __popcll(__ballot(before + upto <= at));
    first = before + __builtin_amdgcn_readlane(upto - tiles, s);
  }

  const u32 lds0 = __builtin_amdgcn_readfirstlane((u32)(uintptr_t)(__attribute__((address_space(3))) unsigned char*)paged_lds) + wave * T::WAVE;
  unsigned char* const mine = paged_lds + wave * T::WAVE;
  const int lrow = lane / T::PIECES, place = lane % T::PIECES;
  const float c2 = a.scale * 1.4426950408889634f;   // e^(x scale) = 2^(x c2)
  const float tau = PAGED_TAU2 / c2;

  while (at < end) {
    const int b = b0 + s, length = __builtin_amdgcn_readlane(len, s), n_tiles = __builtin_amdgcn_readlane(tiles, s);
    const int from = at - first, to = min(n_tiles, end - first);   // this worker's tiles of the sequence
    const int32_t* const row = t.table + (int64_t)b * t.ld_table;

    // q as the products' second operand: column = head lane % 16; e4m3: in the order in which K's 16-byte pieces hold the elements
    bf16x8_t qf[KS];
    {
      const u16* const q = a.q + b * a.ldq + (h0 + (l16 < nh ? l16 : 0)) * HD;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks)
        qf[ks] = __builtin_bit_cast(bf16x8_t, ld16(q + (E4M3 ? (ks >> 1) * 64 + l4 * 16 + (ks & 1) * 8 : ks * 32 + l4 * 8)));
    }
    // the pages of this wave's next 32 tiles: lane i has that of tile i / 2, its 16-key half i % 2
    auto pages_of = [&](int tile) {
      const int key = (tile + 4 * (lane >> 1)) * 32 + (lane & 1) * 16;
      int p = -1;
      if (tile + 4 * (lane >> 1) < to && key < length) {
        p = row[key >> c.shift];
        if ((u32)p >= (u32)c.n_pages) {
          p = -1;
          if (t.err) *t.err = LR_DEV_PAGE_RANGE;
        }
      }
      return p;
    };
    int tile = from + wave, j = 0;
    int pages = pages_of(tile), pages_next = pages_of(tile + 128);
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) asm volatile("" : "+v"(qf[ks]));   // (waited for here, not behind the loads below)

    auto load_rows = [&](const u8* base, bool value, int tile, int p0, int p1, u32 lds) {
#pragma unroll
      for (int i = 0; i < T::LOADS; ++i) {
        const int r0 = i * T::RPL, half = r0 >> 4, p = half ? p1 : p0;
        const i32x4_t res = paged_resource(base + paged_offset<T::ROW>(c, p < 0 ? 0 : p, kvh));
        const int slot = (tile * 32 + half * 16) & ((1 << c.shift) - 1), r = r0 + lrow;
        const int piece = place ^ (value ? T::v_place(r) : T::k_place(r));
        const bool ok = p >= 0 && tile * 32 + r < length;
        paged_load16(res, ok ? lrow * T::ROW + piece * 16 : PAGED_OUT, (slot + (r0 & 15)) * T::ROW, lds + i * 1024);
      }
    };
    // lanes 0..3: the scales of a half's keys, 4..7 of its values
    auto load_scales = [&](int tile, int p0, int p1) {
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int p = half ? p1 : p0, slot = (tile * 32 + half * 16) & ((1 << c.shift) - 1);
        const i32x4_t res = paged_resource(c.scales + paged_scales(c, p < 0 ? 0 : p, kvh));
        paged_load4(res, p >= 0 && lane < 8 ? (lane >> 2 << c.shift) + (lane & 3) * 4 : PAGED_OUT, slot, lds0 + 2 * T::TILE + half * 256);
      }
    };

    f32x4_t o[DT], o_low[E4M3 ? 1 : DT];   // o_low: what the weights' second parts give, apart, since an infinite value times zero is none
#pragma unroll
    for (int d = 0; d < DT; ++d) o[d] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
    if constexpr (!E4M3)
#pragma unroll
      for (int d = 0; d < DT; ++d) o_low[d] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
    float m = -INFINITY, l = 0.0f;   // m: reference point in raw scores; l: this lane's part of the sum

    int p0 = 0, p1 = 0;
    if (tile < to) {
      p0 = __builtin_amdgcn_readlane(pages, 0);
      p1 = __builtin_amdgcn_readlane(pages, 1);
      load_rows(c.k, false, tile, p0, p1, lds0);
      if constexpr (E4M3) load_scales(tile, p0, p1);
      load_rows(c.v, true, tile, p0, p1, lds0 + T::TILE);
    }
    while (tile < to) {
      const int next = tile + 4;
      const bool more = next < to;
      int q0 = 0, q1 = 0;
      if (more) {
        if (++j == 32) {
          j = 0;
          pages = pages_next;
          pages_next = pages_of(next + 128);
        }
        q0 = __builtin_amdgcn_readlane(pages, 2 * j);
        q1 = __builtin_amdgcn_readlane(pages, 2 * j + 1);
      }
      // ---- scores of 2 x 16 keys
      paged_wait_loads<T::LOADS>();
      f32x4_t sc[2];
      u32 vs[2] = {};   // e4m3: the bytes of this lane's four keys' values' scales, per half
      {
        u32x4_t raw[2][E4M3 ? KS / 2 : KS];
        float ks_scale[2] = {};
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int r = h * 16 + l16;
          const unsigned char* const krow = mine + r * T::ROW;
#pragma unroll
          for (int i = 0; i < (E4M3 ? KS / 2 : KS); ++i) raw[h][i] = *reinterpret_cast<const u32x4_t*>(krow + ((i * 4 + l4) ^ T::k_place(r)) * 16);
          if constexpr (E4M3) {
            const unsigned char* const e = mine + 2 * T::TILE + h * 256;
            ks_scale[h] = paged_scale(e[l16]);
            vs[h] = *reinterpret_cast<const u32*>(e + 16 + l4 * 4);
          }
        }
        if (more) {
          paged_wait_lds();
          load_rows(c.k, false, next, q0, q1, lds0);
          if constexpr (E4M3) load_scales(next, q0, q1);
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          sc[h] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
          for (int ks = 0; ks < KS; ++ks) {
            bf16x8_t kf;
            if constexpr (E4M3) {
              u32x4_t x;
              const u32 lo = raw[h][ks >> 1][(ks & 1) * 2], hi = raw[h][ks >> 1][(ks & 1) * 2 + 1];
              x[0] = __builtin_bit_cast(u32, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, ks_scale[h], false));
              x[1] = __builtin_bit_cast(u32, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, ks_scale[h], true));
              x[2] = __builtin_bit_cast(u32, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, ks_scale[h], false));
              x[3] = __builtin_bit_cast(u32, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, ks_scale[h], true));
              kf = __builtin_bit_cast(bf16x8_t, x);
            } else {
              kf = __builtin_bit_cast(bf16x8_t, raw[h][ks]);
            }
            sc[h] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf, qf[ks], sc[h], 0, 0, 0);
          }
        }
      }
      // element e of half h: key 16 h + 4 l4 + e of the tile, head l16
      const int there = length - tile * 32;
      if (there < 32 || (p0 | p1) < 0) {   // uniform
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            sc[h][e] = (h ? p1 : p0) >= 0 && 16 * h + 4 * l4 + e < there ? sc[h][e] : -INFINITY;
      }
      float top = sc[0][0];
#pragma unroll
      for (int e = 1; e < 8; ++e) top = fmaxf(top, sc[e >> 2][e & 3]);
      top = rows_max(top);
      // (the reference point moves only when a tile's maximum exceeds it by more than tau: weights stay below 2^PAGED_TAU2)
      const bool grow = top > m + tau;   // m = -inf: any finite maximum
      const float mn = grow ? top : m, nmc = mn == -INFINITY ? 0.0f : -mn * c2;
      if (__any(grow)) {
        const float corr = grow ? exp2_hw((m - mn) * c2) : 1.0f;   // m = -inf: 0
        l *= corr;
#pragma unroll
        for (int d = 0; d < DT; ++d) o[d] *= corr;
        if constexpr (!E4M3)
#pragma unroll
          for (int d = 0; d < DT; ++d) o_low[d] *= corr;
      }
      m = mn;
      u32x4_t ph, pl;
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int e = 0; e < 4; e += 2) {
          float x0 = exp2_hw(fmaf(sc[h][e], c2, nmc)), x1 = exp2_hw(fmaf(sc[h][e + 1], c2, nmc));   // masked: 0
          l += x0 + x1;
          if constexpr (E4M3) {
            x0 *= paged_scale((vs[h] >> 8 * e) & 255);
            x1 *= paged_scale((vs[h] >> (8 * e + 8)) & 255);
          }
          const u32 hi = pack_bf2(x0, x1);
          ph[h * 2 + (e >> 1)] = hi;
          pl[h * 2 + (e >> 1)] = pack_bf2(x0 - bf_lo(hi), x1 - bf_hi(hi));
        }
      // ---- values, read across the keys: place i < 4 of a lane's eight is key 4 l4 + i, else 16 + 4 l4 + i - 4
      if (more) paged_wait_loads<T::LOADS + (E4M3 ? 2 : 0)>();
      else paged_wait_loads<0>();
      const unsigned char* const vt = mine + T::TILE;
      bf16x8_t vf[DT];
      i32x2_t raw[E4M3 ? DT : 1];
#pragma unroll
      for (int d = 0; d < DT; ++d) {
        if constexpr (E4M3) {
          const int r = 4 * l4 + ((l16 >> 1) & 3) + (l16 >> 3) * 16;   // 16 lanes read 8 keys of 16 dimensions
          raw[d] = __builtin_amdgcn_ds_read_tr8_b64_v2i32(
              (__attribute__((address_space(3))) i32x2_t*)(vt + r * T::ROW + (d ^ T::v_place(r)) * 16 + (l16 & 1) * 8));
        } else {
          const int r = 4 * l4 + (l16 >> 2);   // 16 lanes read 4 keys of 16 dimensions
          const unsigned char* const v0 = vt + r * T::ROW + ((2 * d + ((l16 & 3) >> 1)) ^ T::v_place(r)) * 16 + (l16 & 1) * 8;
          const i16x4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) i16x4_t*)(v0));
          const i16x4_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) i16x4_t*)(v0 + 16 * T::ROW));
          vf[d] = __builtin_bit_cast(bf16x8_t, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
        }
      }
      if (more) {
        paged_wait_lds();
        load_rows(c.v, true, next, q0, q1, lds0 + T::TILE);
      }
#pragma unroll
      for (int d = 0; d < DT; ++d) {
        if constexpr (E4M3) {
          u32x4_t x;
          x[0] = __builtin_bit_cast(u32, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(raw[d][0], 1.0f, false));
          x[1] = __builtin_bit_cast(u32, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(raw[d][0], 1.0f, true));
          x[2] = __builtin_bit_cast(u32, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(raw[d][1], 1.0f, false));
          x[3] = __builtin_bit_cast(u32, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(raw[d][1], 1.0f, true));
          vf[d] = __builtin_bit_cast(bf16x8_t, x);
        }
        o[d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf[d], __builtin_bit_cast(bf16x8_t, ph), o[d], 0, 0, 0);
      }
#pragma unroll
      for (int d = 0; d < DT; ++d) {
        f32x4_t& to_low = E4M3 ? o[d] : o_low[E4M3 ? 0 : d];
        to_low = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf[d], __builtin_bit_cast(bf16x8_t, pl), to_low, 0, 0, 0);
      }
      tile = next;
      p0 = q0;
      p1 = q1;
    }

    // ---- the four waves' results together (each in its own LDS, where nothing is on its way any more)
    l = rows_sum(l);
    float* const my_o = reinterpret_cast<float*>(mine);
#pragma unroll
    for (int d = 0; d < DT; ++d) {
      f32x4_t v = o[d];
      if constexpr (!E4M3)
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = fabsf(v[e]) < INFINITY ? v[e] + o_low[d][e] : v[e];
      *reinterpret_cast<f32x4_t*>(my_o + l16 * T::LDO + d * 16 + l4 * 4) = v;
    }
    if (l4 == 0) s_ml[wave][l16][0] = m * c2, s_ml[wave][l16][1] = l;   // (from here on in powers of two)
    __syncthreads();
    const bool whole = from == 0 && to == n_tiles;
    const int slot = (group * (int)gridDim.x + w) * 2 + (from == 0 ? 1 : 0);
    const __amdgpu_buffer_rsrc_t ores = __builtin_amdgcn_make_buffer_rsrc(a.o_part, 0, 0x7fffffff, 0x00020000);
    const __amdgpu_buffer_rsrc_t mres = __builtin_amdgcn_make_buffer_rsrc(a.ml_part, 0, 0x7fffffff, 0x00020000);
    u16* const y = a.y + b * a.ldy + h0 * HD;
    auto store_y = [&](int h, int d, const f32x4_t& v, float L) {
      const float inv = L != 0.0f ? 1.0f / L : 0.0f;
      u32x2_t out;
      out.x = pack_bf2(v[0] * inv, v[1] * inv);
      out.y = pack_bf2(v[2] * inv, v[3] * inv);
      *reinterpret_cast<u32x2_t*>(y + h * HD + d) = out;
    };
    auto store_part = [&](int part, int h, int d, const f32x4_t& v, float M, float L) {
      __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4_t, v), ores, ((part * 16 + h) * HD + d) * 4, 0, PAGED_COHERENT);
      if (d == 0) __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(u32x2_t, f32x2_t{M, L}), mres, (part * 16 + h) * 8, 0, PAGED_COHERENT);
    };
    for (int i = tid; i < nh * (HD / 4); i += 256) {
      const int h = i / (HD / 4), d = i % (HD / 4) * 4;
      float M = s_ml[0][h][0], L = 0.0f;
#pragma unroll
      for (int k = 1; k < 4; ++k) M = fmaxf(M, s_ml[k][h][0]);
      // (a wave that has seen no key has -inf, 0, 0; one that has seen only NaN -inf, NaN, NaN)
      const float ref = M == -INFINITY ? 0.0f : M;
      f32x4_t v = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float f = exp2_hw(s_ml[k][h][0] - ref);
        L += f * s_ml[k][h][1];
        v += f * *reinterpret_cast<const f32x4_t*>(reinterpret_cast<const float*>(paged_lds + k * T::WAVE) + h * T::LDO + d);
      }
      if (whole) store_y(h, d, v, L);
      else store_part(slot, h, d, v, M, L);
    }
    if (!whole) {
      // Workers w0 .. w1 have parts of this sequence.  Those of one block of PAGED_BLOCK workers are put together by the block's last, the
      // blocks' results by the last block's.
      const auto worker = [&](int tile) { return (int)((((int64_t)tile + 1) * workers - 1) / total); };
      const int w0 = worker(first), w1 = worker(first + n_tiles - 1), k0 = w0 / PAGED_BLOCK, k1 = w1 / PAGED_BLOCK, kw = w / PAGED_BLOCK;
      const int n_blocks = (gridDim.x + PAGED_BLOCK - 1) / PAGED_BLOCK;
      const auto part_of = [&](int x) { return (group * (int)gridDim.x + x) * 2 + (x == w0 ? 1 : 0); };
      const auto block_of = [&](int k) { return (group * n_blocks + k) * 2 + (k == k0 ? 1 : 0); };
      const int block_parts = gridDim.y * gridDim.x * 2;
      // true in the last of n workers: then all others' results can be read
      auto last_of = [&](u32* ticket, int n) {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        if (tid == 0) {
          const u32 was = __hip_atomic_fetch_add(ticket, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
          if (was + 1 == (u32)n) __hip_atomic_store(ticket, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
          *s_ticket = was + 1;
        }
        __syncthreads();
        const bool last = *s_ticket == (u32)n;
        asm volatile("" ::: "memory");
        return last;
      };
      // parts u0 .. u1, at places(u), into y or the place `out`
      auto together = [&](int u0, int u1, auto places, int out) {
        for (int i = tid; i < nh * (HD / 4); i += 256) {
          const int h = i / (HD / 4), d = i % (HD / 4) * 4;
          float M = -INFINITY, L = 0.0f;
          f32x4_t v = {0.0f, 0.0f, 0.0f, 0.0f};
          for (int u = u0; u <= u1; u += 8) {
            f32x4_t ov[8];
            f32x2_t ml[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) {   // (all of them on their way before the first is used)
              const int from_ = u + k <= u1 ? places(u + k) * 16 + h : -1;
              ov[k] = __builtin_bit_cast(f32x4_t, __builtin_amdgcn_raw_buffer_load_b128(ores, from_ < 0 ? PAGED_OUT : (from_ * HD + d) * 4, 0, PAGED_COHERENT));
              ml[k] = __builtin_bit_cast(f32x2_t, __builtin_amdgcn_raw_buffer_load_b64(mres, from_ < 0 ? PAGED_OUT : from_ * 8, 0, PAGED_COHERENT));
            }
#pragma unroll
            for (int k = 0; k < 8; ++k)
              if (u + k <= u1) {
                const float Mn = fmaxf(M, ml[k][0]), ref = Mn == -INFINITY ? 0.0f : Mn;
                const float f0 = exp2_hw(M - ref), f1 = exp2_hw(ml[k][0] - ref);
                L = L * f0 + ml[k][1] * f1;
                v = v * f0 + ov[k] * f1;
                M = Mn;
              }
          }
          if (out < 0) store_y(h, d, v, L);
          else store_part(out, h, d, v, M, L);
        }
      };
      u32* const own = a.tickets + (int64_t)group * t.B + b;
      if (k0 == k1) {
        if (last_of(own, w1 - w0 + 1)) together(w0, w1, part_of, -1);
      } else {
        u32* const blocks = a.tickets + (int64_t)gridDim.y * t.B + block_of(kw);
        const int u0 = max(w0, kw * PAGED_BLOCK), u1 = min(w1, kw * PAGED_BLOCK + PAGED_BLOCK - 1);
        if (last_of(blocks, u1 - u0 + 1)) {
          together(u0, u1, part_of, block_parts + block_of(kw));
          if (last_of(own, k1 - k0 + 1)) together(k0, k1, [&](int k) { return block_parts + block_of(k); }, -1);
        }
      }
    }
    __syncthreads();
    // ---- on to the next sequence that has tiles
    at = first + to;
    if (at >= end) return;
    first += n_tiles;
    unsigned long long others = __ballot(tiles > 0) & (s == 63 ? 0ull : ~0ull << (s + 1));
    while (!others) {
      if (b0 + 64 >= t.B) return;   // (never: there are tiles left)
      look(b0 + 64);
      others = __ballot(tiles > 0);
    }
    s = __builtin_ctzll(others);
  }
}

struct DecodePlan {
  int groups_per_kv, groups, workers, blocks;
  size_t o_bytes, ml_bytes, ticket_bytes;
};
// Workers of a kv head (a group of up to 16 of its q heads): as many as the chip holds at once, no more than the table's pages could give
// four tiles each.
template <int HD, bool E4M3>
static DecodePlan decode_plan(const PagedCache& c, const PagedBatch& t, int Hq) {
  DecodePlan p;
  p.groups_per_kv = (Hq / c.Hkv + 15) / 16;
  p.groups = c.Hkv * p.groups_per_kv;
  const int per_cu = DecodeTile<HD, E4M3>::PER_CU, cus = lr_num_cus();
  const int64_t tiles = (int64_t)t.B * (((int64_t)t.pages << c.shift) / 32 + 1);
  int64_t n = (int64_t)(cus ? cus : 256) * per_cu / p.groups;
  if (n > (tiles + 3) / 4) n = (tiles + 3) / 4;
  p.workers = n < 1 ? 1 : (int)n;
  p.blocks = (p.workers + PAGED_BLOCK - 1) / PAGED_BLOCK;
  const size_t parts = (size_t)p.groups * (p.workers + p.blocks) * 2;
  p.o_bytes = parts * 16 * HD * 4;
  p.ml_bytes = parts * 16 * 2 * 4;
  p.ticket_bytes = ((size_t)p.groups * (t.B + p.blocks * 2) * 4 + 255) & ~(size_t)255;
  return p;
}

template <int HD, bool E4M3>
static int launch_paged_decode(const PagedCache& c, const PagedBatch& t, const PagedQuery& q, void* scratch, hipStream_t s) {
  const DecodePlan p = decode_plan<HD, E4M3>(c, t, q.Hq);
  PagedDecode a = {q.q, q.ldq, q.y, q.ldy, q.Hq, p.groups_per_kv, q.scale, nullptr, nullptr, nullptr};
  a.tickets = (u32*)scratch;
  a.o_part = (float*)((u8*)scratch + p.ticket_bytes);
  a.ml_part = (float*)((u8*)a.o_part + p.o_bytes);
  constexpr size_t lds = DecodeTile<HD, E4M3>::LDS;
  static std::atomic<unsigned long long> raised{0};
  if (!lr_raise_lds_limit(reinterpret_cast<const void*>(&k_paged_decode<HD, E4M3>), lds, raised)) return LR_E_LAUNCH;
  k_paged_decode<HD, E4M3><<<dim3(p.workers, p.groups), dim3(256), lds, s>>>(c, t, a);
  return lr_launch_status();
}

// ------------------------------------------------------------------------------------ prompts
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

static size_t paged_scratch(const PagedCache& c, const PagedBatch& t, int hd, bool e4m3, int rows, int Hq) {
  if (t.starts) return 256;
  const DecodePlan p = hd == 128 ? (e4m3 ? decode_plan<128, true>(c, t, Hq) : decode_plan<128, false>(c, t, Hq))
                                 : (e4m3 ? decode_plan<64, true>(c, t, Hq) : decode_plan<64, false>(c, t, Hq));
  if (p.groups > 65535) return 0;   // (a grid's second dimension)
  return p.ticket_bytes + p.o_bytes + p.ml_bytes;
}

extern "C" size_t lr_paged_attention_scratch_bytes(const lr_paged_cache_t* cache, const lr_paged_batch_t* batch, int rows, int Hq) {
  PagedCache c;
  PagedBatch t;
  if (paged_arguments(cache, batch, c, t) || rows <= 0 || Hq <= 0 || Hq % c.Hkv) return 0;
  return paged_scratch(c, t, cache->head_dim, cache->format == LR_CACHE_E4M3, rows, Hq);
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
  const bool e4m3 = cache->format == LR_CACHE_E4M3;
  if (rows <= 0 || Hq <= 0 || Hq % c.Hkv || (t.starts == nullptr && rows != t.B)) return LR_E_SHAPE;
  if (Hq > 65535 || ldq < (int64_t)Hq * hd || ldy < (int64_t)Hq * hd || !(scale > 0.0f && scale < INFINITY)) return LR_E_SHAPE;
  if (ldq % 8 || ldy % 8) return LR_E_ALIGN;
  const size_t need = paged_scratch(c, t, hd, e4m3, rows, Hq);
  if (need == 0) return LR_E_UNSUPPORTED;
  if (scratch_bytes < need) return LR_E_SHAPE;
  const PagedQuery a = {(const u16*)q, ldq, (u16*)y, ldy, rows, Hq, scale};
  hipStream_t s = (hipStream_t)stream;
  if (t.starts == nullptr)
    return hd == 128 ? (e4m3 ? launch_paged_decode<128, true>(c, t, a, scratch, s) : launch_paged_decode<128, false>(c, t, a, scratch, s))
                     : (e4m3 ? launch_paged_decode<64, true>(c, t, a, scratch, s) : launch_paged_decode<64, false>(c, t, a, scratch, s));
  const dim3 grid((unsigned)rows, (unsigned)Hq);
  if (hd == 128 && e4m3) k_paged_attention<128, true><<<grid, dim3(64), 0, s>>>(c, t, a);
  else if (hd == 128) k_paged_attention<128, false><<<grid, dim3(64), 0, s>>>(c, t, a);
  else if (e4m3) k_paged_attention<64, true><<<grid, dim3(64), 0, s>>>(c, t, a);
  else k_paged_attention<64, false><<<grid, dim3(64), 0, s>>>(c, t, a);
  return lr_launch_status();
}
