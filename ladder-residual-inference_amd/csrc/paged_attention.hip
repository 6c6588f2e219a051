// lr_paged_attention: softmax attention of a call's rows on the pages of a key-value cache.
#include "attention_common.h"
#include "paged_common.h"

#include <atomic>
#include <cfloat>
#include <type_traits>

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
// equal parts of it, wherever sequences begin and end (or of each sequence, where these are few): batches of any lengths keep the chip evenly busy,
// and the host, which knows no length, launches the same grid always.  A part of a sequence leaves its maximum, sum and weighted values in the scratch, and whoever ends
// last puts a sequence's parts together (in their order: the same bits every time); a sequence inside one part is written directly.
//
// A wave streams tiles of its own through its own LDS (no barrier in the loop): rows come by loads straight into LDS, K's of the next tile
// as soon as K's of this one are in registers, V's likewise.  S[key][head] = K q^T and O^T[dim][head] += V^T P on the matrix cores
// (16x16x32, up to 16 q heads of the kv head are the columns): a lane holds eight scores of one head and, since the order of keys in a product
// is free, hands them on as the second product's operand without moving them.  Weights enter as two bf16 numbers (2^-16 of the
// weight).  e4m3: K is expanded with its row's power of two on the way to the product, V without, its power goes into the weight.
//
// Bound: memory.  64 sequences of 2048 keys, 8 kv heads of 128, e4m3: 43.4 us, 6.3 TB/s (a plain read 7.0); one of 131072 in bf16 84.0 us, 6.4 TB/s;
// 24 of 1 to 4096 26.4 us.  One workgroup per CU with four waves whose tiles are all in flight reads faster than two or three smaller ones (the first
// of these 43.6, 50, 58), rows that nobody else reads come non-temporally (10 %).  Few keys: a chain of waits, 8.4 us at first for one sequence of 2048
// and one kv head, 7.3 now: the lengths 0.7, page numbers and q 1.1, keys, values and products 1.5, four waves' results 0.9, what a worker leaves
// and its ticket 1.0, the parts together 1.8, the rest start and end.
typedef int i32x2_t __attribute__((ext_vector_type(2)));
constexpr float PAGED_TAU2 = 8.0f;   // log2 of the largest weight before the reference point of the exponentials moves
// Exponents are score * c2 - m * c2 with one rounding, m * c2 rounded once for all: a factor that all weights of a row share.  Where it could leave fp32
// (it is 2 to the power of 2^-25 of m * c2) scores are taken less m first: from this |m * c2| on, at which a score of fp32 is itself off by more.
constexpr float PAGED_FAR = 0x1p20f;
constexpr int PAGED_OUT = (int)0x80000000;   // an offset outside every resource: comes as zeros
constexpr int PAGED_COHERENT = 17;   // sc0 sc1: past this XCD's L2

__device__ __forceinline__ i32x4_t paged_resource(const u8* at) {
  return i32x4_t{(int)(u32)(unsigned long long)at, (int)(u32)((unsigned long long)at >> 32), 0x7fffffff, 0x00020000};   // (addresses have 47 bits: no stride)
}
// 16 (4) bytes per lane from resource + voff + soff to LDS address `lds` + 16 (4) * lane; counted by vmcnt, not by the compiler
// (ONCE: rows that nobody else reads, non-temporal)
template <bool ONCE = false>
__device__ __forceinline__ void paged_load16(const i32x4_t& res, int voff, int soff, u32 lds) {
  if constexpr (ONCE)
    asm volatile("s_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen nt lds" ::"{m0}"(lds), "v"(voff), "s"(res), "s"(soff) : "memory");
  else
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
  static constexpr int NW = 4, PER_CU = HD == 64 ? 2 : 1;              // waves of a workgroup; workgroups of a CU
  static constexpr int RESULT = 16 * LDO * 4;                          // a wave's results
  static constexpr int LDS = NW * (WAVE + RESULT + 128) + 16;          // (with the waves' maxima and sums, and two tickets)
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

// What a sequence costs a worker besides its tiles, in tiles (7 us in a row of short sequences for two of them; a tile 0.45 us): as much more room
// it has on the line.
constexpr int PAGED_SEQUENCE = 6;
// A sequence's parts are read that many at a time by the last of its workers; where there are more than PAGED_ONE, blocks of so many workers go first.  (us,
// 24 sequences of up to 4096 keys with 32 workers per kv head: 26.4, all through blocks 27.8.)
constexpr int PAGED_BLOCK = 16, PAGED_ONE = 32;
// Parts of a sequence, where they would have fewer than PAGED_FEW tiles: 62 parts of 4 tiles take 15.0 us, 16 of 16 13.8 (16 q heads on one kv head of 128, 7888
// keys); at 30000 235 parts of 4 17.0, 59 of 16 19.1.
constexpr int PAGED_PARTS = 16, PAGED_FEW = 16;
// Tiles of a worker that sequences cut on their own may cost.  us, the line / sequences: 7 of 7888 keys, 16 q heads on one kv head 26.6 / 15.9; 14 of up to 843,
// 8 kv heads 17.1 / 10.4; 24 of up to 4096 with 16 instead of 8 27.4 / 27.9.
constexpr int PAGED_MORE = 8;
// Tiles of sequences that are not cut at all where there are many.  us, cut / whole: 40 of up to 270 keys, 8 kv heads of 64 10.9 / 7.6; 46 of up to 478, of 128
// 15.4 / 11.2; of 34 of up to 300, 24 kv heads 21.0 / 15.5.
constexpr int PAGED_WHOLE = 16;

// MANY: more than one place in the batch.  (A kernel of its own for one: less to look up, and no scalar registers kept in lanes of vector ones;
// 8.4 -> 7.3 us for 2048 keys of one kv head.)
template <int HD, bool E4M3, bool MANY>
__global__ __launch_bounds__((DecodeTile<HD, E4M3>::NW * 64), (DecodeTile<HD, E4M3>::PER_CU * DecodeTile<HD, E4M3>::NW / 4)) void k_paged_decode(const PagedCache c, const PagedBatch t, const PagedDecode a) {
  using T = DecodeTile<HD, E4M3>;
  constexpr int KS = HD / 32, DT = HD / 16, NW = T::NW;   // k-steps of a score product; 16-dimension tiles of O^T
  const int B = MANY ? t.B : 1;
  extern __shared__ __attribute__((aligned(1024))) unsigned char paged_lds[];
  float (*const s_ml)[16][2] = reinterpret_cast<float (*)[16][2]>(paged_lds + NW * (T::WAVE + T::RESULT));   // [NW]
  u32* const s_ticket = reinterpret_cast<u32*>(paged_lds + NW * (T::WAVE + T::RESULT + 128));
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l16 = lane & 15, l4 = lane >> 4;
  const int group = blockIdx.y, kvh = group / a.groups_per_kv, G = a.Hq / c.Hkv;
  const int h0 = kvh * G + group % a.groups_per_kv * 16, left = (kvh + 1) * G - h0, nh = left < 16 ? left : 16;   // this group's q heads

  // ---- which tiles are this worker's
  int b0 = 0;   // lane i looks after sequence b0 + i
  int len, tiles, upto;   // its keys, its tiles, and the tiles up to it of the 64 sequences
  unsigned long long some;   // which of them have tiles
  auto look = [&](int from) {
    b0 = from;
    len = b0 + lane < B ? paged_length(t, c.shift, b0 + lane) : 0;
    tiles = (len + 31) >> 5;
    upto = paged_sums(tiles);
    some = __ballot(tiles > 0);
  };
  int total = 0, sequences = 0;
  for (int i = 0; i < B; i += 64) {
    look(i);
    total += __builtin_amdgcn_readlane(upto, 63);
    sequences += __popcll(some);
    if (wave == 0) {   // empty places: zeros, one worker each
      unsigned long long empty = __ballot(i + lane < B && tiles == 0 && (i + lane) % gridDim.x == blockIdx.x);
      for (; empty; empty &= empty - 1) {
        u16* const y = a.y + (int64_t)(i + __builtin_ctzll(empty)) * a.ldy + h0 * HD;
        for (int d = lane * 8; d < nh * HD; d += 512) st16(y + d, make_uint4(0, 0, 0, 0));
      }
    }
  }
  // a worker's tiles at least: one for each of its waves, and where that leaves a sequence no more than PAGED_PARTS parts up to PAGED_FEW
  const auto few = [&](int tiles) { return tiles <= PAGED_PARTS * PAGED_FEW ? max(NW, (tiles + PAGED_PARTS - 1) / PAGED_PARTS) : NW; };
  const int w = blockIdx.x;
  int workers = min((int)gridDim.x, max((total + NW - 1) / NW, sequences));
  if (sequences == 1 && few(total) > NW) workers = min(workers, PAGED_PARTS);
  // Workers from0 on take equal parts of the line from `line0` on, `each` places and the first `larger` of them one more; this one's begins in sequence
  // b0 + s, which begins at `first`
  int from0 = 0, line0 = 0, each = 0, larger, s, first, extra = 0;
  // Sequences cut on their own, into equal parts of no more than `most` tiles, where that takes few tiles more than the line in equal parts: a worker has
  // one sequence only, and its results to join with others' once.
  const int longest = MANY && B <= 64 && sequences > 1 ? wave_max(tiles) : 0;   // (0: not known or not wanted)
  if (longest && sequences < workers) {
    const int even = max((total + workers - 1) / workers, few(longest)), last = even + PAGED_MORE;
    // (half a part per sequence is lost: hopeless where even the last does not have that much room)
    for (int most = (long long)last * ((int)gridDim.x - sequences / 2) < total ? last + 1 : even; most <= last; most += 1 + most / 8) {
      const int parts = (u32)(tiles + most - 1) / (u32)most, sum = paged_sums(parts), all = __builtin_amdgcn_readlane(sum, 63);
      if (all > (int)gridDim.x) continue;
      if (w >= all) return;
      s = __popcll(__ballot(sum <= w)) & 63;
      const int n = __builtin_amdgcn_readlane(parts, s), mine = __builtin_amdgcn_readlane(tiles, s);
      from0 = __builtin_amdgcn_readlane(sum, s) - n;
      line0 = first = __builtin_amdgcn_readlane(upto, s) - mine;
      each = (u32)mine / (u32)n;
      larger = mine - each * n;
      break;
    }
  }
  const bool alone = each > 0;
  if (!alone) {
    if (w >= workers) return;
    // what a sequence costs besides its tiles, as more room on the line: where workers have one sequence or several; where a sequence has
    // many workers, it is the same for all of them
    extra = MANY && 2 * sequences >= workers ? PAGED_SEQUENCE : 0;
    total += extra * sequences;
    each = (u32)total / (u32)workers;
    larger = total - each * workers;
  }
  int at = line0 + (w - from0) * each + min(w - from0, larger);
  int end = at + each + (w - from0 < larger);
  if (!alone) {
    int before = 0;
    auto places_upto = [&]() { return upto + extra * __popcll(some & (~0ull >> (63 - lane))); };   // of the 64 sequences, in all lanes
    if (B > 64) {
      for (int i = 0;; i += 64) {
        look(i);
        const int n = __builtin_amdgcn_readlane(upto, 63) + extra * __popcll(some);
        if (at < before + n || i + 64 >= B) break;
        before += n;
      }
    }
    const int places = places_upto();
    if (longest && longest <= PAGED_WHOLE) {   // short sequences go whole to the worker that has their middle: nothing to join
      const int middle = places - (tiles + extra) / 2;
      const unsigned long long from = __ballot(tiles > 0 && middle >= at), behind = __ballot(tiles > 0 && middle >= end);
      if (from == behind) return;
      const auto begin = [&](int i) { return __builtin_amdgcn_readlane(places, i) - __builtin_amdgcn_readlane(tiles, i) - extra; };
      at = begin(__builtin_ctzll(from));
      end = behind ? begin(__builtin_ctzll(behind)) : total;
    }
    s = __popcll(__ballot(before + places <= at)) & 63;
    first = before + __builtin_amdgcn_readlane(places, s) - __builtin_amdgcn_readlane(tiles, s) - extra;
  }

  const u32 lds0 = __builtin_amdgcn_readfirstlane((u32)(uintptr_t)(__attribute__((address_space(3))) unsigned char*)paged_lds) + wave * T::WAVE;
  unsigned char* const mine = paged_lds + wave * T::WAVE;
  const int lrow = lane / T::PIECES, place = lane % T::PIECES;
  const float c2 = a.scale * 1.4426950408889634f;   // e^(x scale) = 2^(x c2)
  const float tau = fminf(PAGED_TAU2 / c2, FLT_MAX);   // (-inf + tau stays -inf)

  // this worker's tiles from .. to of the n_tiles of a sequence, the first of which is at `first` of the line, behind the sequence's own cost
  struct Segment {
    int b, length, n_tiles, first, from, to;
  };
  auto segment = [&]() {
    Segment g;
    g.b = b0 + s;
    g.length = __builtin_amdgcn_readlane(len, s);
    g.n_tiles = __builtin_amdgcn_readlane(tiles, s);
    g.first = first + extra;
    g.from = max(0, at - g.first);
    g.to = min(g.n_tiles, end - g.first);
    return g;
  };
  // on to the next sequence that has tiles; false: this worker's part of the line ends before its first one
  auto next_segment = [&](Segment& g) {
    if constexpr (!MANY) return false;
    first += __builtin_amdgcn_readlane(tiles, s) + extra;
    if (first + extra >= end) return false;
    unsigned long long others = some & (s == 63 ? 0ull : ~0ull << (s + 1));
    while (!others) {
      if (b0 + 64 >= B) return false;
      look(b0 + 64);
      others = some;
    }
    s = __builtin_ctzll(others);
    g = segment();
    return true;
  };
  // q as the products' second operand: column = head lane % 16; e4m3: in the order in which K's 16-byte pieces hold the elements
  auto load_q = [&](const Segment& g, bf16x8_t* qf) {
    const u16* const q = a.q + g.b * a.ldq + (h0 + (l16 < nh ? l16 : 0)) * HD;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)
      qf[ks] = __builtin_bit_cast(bf16x8_t, ld16(q + (E4M3 ? (ks >> 1) * 64 + l4 * 16 + (ks & 1) * 8 : ks * 32 + l4 * 8)));
  };
  // the pages of this wave's next 32 tiles from `tile` on: lane i has that of tile i / 2, its 16-key half i % 2
  auto pages_of = [&](const Segment& g, int tile) {
    const int key = (tile + NW * (lane >> 1)) * 32 + (lane & 1) * 16;
    int p = -1;
    if (tile + NW * (lane >> 1) < g.to && key < g.length) {
      p = t.table[(int64_t)g.b * t.ld_table + (key >> c.shift)];
      if ((u32)p >= (u32)c.n_pages) {
        p = -1;
        if (t.err) *t.err = LR_DEV_PAGE_RANGE;
      }
    }
    return p;
  };
  auto load_rows = [&](const u8* base, bool value, int length, int tile, int p0, int p1, u32 lds) {
#pragma unroll
    for (int i = 0; i < T::LOADS; ++i) {
      const int r0 = i * T::RPL, half = r0 >> 4, p = half ? p1 : p0;
      const i32x4_t res = paged_resource(base + paged_offset<T::ROW>(c, p < 0 ? 0 : p, kvh));
      const int slot = (tile * 32 + half * 16) & ((1 << c.shift) - 1), r = r0 + lrow;
      const int piece = place ^ (value ? T::v_place(r) : T::k_place(r));
      const bool ok = p >= 0 && tile * 32 + r < length;
      paged_load16<true>(res, ok ? lrow * T::ROW + piece * 16 : PAGED_OUT, (slot + (r0 & 15)) * T::ROW, lds + i * 1024);
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
  auto load_k = [&](int length, int tile, int p0, int p1) {
    load_rows(c.k, false, length, tile, p0, p1, lds0);
    if constexpr (E4M3) load_scales(tile, p0, p1);
  };
  auto load_v = [&](int length, int tile, int p0, int p1) { load_rows(c.v, true, length, tile, p0, p1, lds0 + T::TILE); };
  // (for LDS only: __syncthreads() would wait for the next tiles, too)
  auto barrier = [] { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); };

  const __amdgpu_buffer_rsrc_t ores = __builtin_amdgcn_make_buffer_rsrc(a.o_part, 0, 0x7fffffff, 0x00020000);
  const __amdgpu_buffer_rsrc_t mres = __builtin_amdgcn_make_buffer_rsrc(a.ml_part, 0, 0x7fffffff, 0x00020000);
  auto store_y = [&](int b, int h, int d, const f32x4_t& v, float L) {
    const float inv = L != 0.0f ? 1.0f / L : 0.0f;
    u32x2_t out;
    out.x = pack_bf2(v[0] * inv, v[1] * inv);
    out.y = pack_bf2(v[2] * inv, v[3] * inv);
    *reinterpret_cast<u32x2_t*>(a.y + b * a.ldy + (h0 + h) * HD + d) = out;
  };
  auto store_part = [&](int part, int h, int d, const f32x4_t& v, float M, float L) {
    __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4_t, v), ores, ((part * 16 + h) * HD + d) * 4, 0, PAGED_COHERENT);
    if (d == 0) __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(u32x2_t, f32x2_t{M, L}), mres, (part * 16 + h) * 8, 0, PAGED_COHERENT);
  };
  // the sequences of which others have parts, too: one that began before this worker, one that goes on behind it
  constexpr int OPEN = MANY ? 2 : 1;
  int open_b[OPEN], open_first[OPEN] = {}, open_tiles[OPEN] = {};
#pragma unroll
  for (int i = 0; i < OPEN; ++i) open_b[i] = -1;
  Segment g = segment();
  if (g.to <= g.from && !next_segment(g)) return;   // (the sequence's cost alone)
  bf16x8_t qf[KS];
  load_q(g, qf);
  int pages = pages_of(g, g.from + wave), p0 = __builtin_amdgcn_readlane(pages, 0), p1 = __builtin_amdgcn_readlane(pages, 1);   // (all of it here by now)
  if (g.from + wave < g.to) {
    load_k(g.length, g.from + wave, p0, p1);
    load_v(g.length, g.from + wave, p0, p1);
  }
  for (;;) {
    // ---- the sequence after this one: its pages and q are asked for now, its first tile when this wave's last one is in registers
    Segment gn = {};
    const bool more_sequences = next_segment(gn);
    int pages_n = -1, pages_next = pages_of(g, g.from + wave + 32 * NW);
    bf16x8_t qn[KS];
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) qn[ks] = qf[ks];
    if (more_sequences) {
      load_q(gn, qn);
      pages_n = pages_of(gn, gn.from + wave);
    }
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) asm volatile("" : "+v"(qn[ks]));   // (waited for here, together with this sequence's first tile)
    asm volatile("" : "+v"(pages_n), "+v"(pages_next));
    const bool next_here = more_sequences && gn.from + wave < gn.to;   // this wave has a tile of it
    int tile = g.from + wave, j = 0;
    if (next_here && tile >= g.to) {   // and none of this one
      p0 = __builtin_amdgcn_readlane(pages_n, 0);
      p1 = __builtin_amdgcn_readlane(pages_n, 1);
      load_k(gn.length, gn.from + wave, p0, p1);
      load_v(gn.length, gn.from + wave, p0, p1);
    }

    f32x4_t o[DT], o_low[E4M3 ? 1 : DT];   // o_low: what the weights' second parts give, apart, since an infinite value times zero is none
#pragma unroll
    for (int d = 0; d < DT; ++d) o[d] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
    if constexpr (!E4M3)
#pragma unroll
      for (int d = 0; d < DT; ++d) o_low[d] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
    float m = -INFINITY, l = 0.0f;   // m: reference point in raw scores; l: this lane's part of the sum

    while (tile < g.to) {
      const bool same = tile + NW < g.to, more = same || next_here;
      const int next = same ? tile + NW : gn.from + wave, next_length = same ? g.length : gn.length;
      int q0 = 0, q1 = 0;
      if (same) {
        if (++j == 32) {
          j = 0;
          pages = pages_next;
          pages_next = pages_of(g, next + 32 * NW);
        }
        q0 = __builtin_amdgcn_readlane(pages, 2 * j);
        q1 = __builtin_amdgcn_readlane(pages, 2 * j + 1);
      } else if (next_here) {
        q0 = __builtin_amdgcn_readlane(pages_n, 0);
        q1 = __builtin_amdgcn_readlane(pages_n, 1);
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
          load_k(next_length, next, q0, q1);
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
      const int there = g.length - tile * 32;
      if (there < 32 || (p0 | p1) < 0) {   // uniform
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            sc[h][e] = (h ? p1 : p0) >= 0 && 16 * h + 4 * l4 + e < there ? sc[h][e] : -INFINITY;
        if constexpr (E4M3)   // (a slot that nobody has written holds any byte: 255 is infinity, and their weights are 0)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int n = there - 16 * h - 4 * l4;   // of this lane's four keys, those that there are
            vs[h] &= n >= 4 ? ~0u : n <= 0 ? 0u : ~0u >> (32 - 8 * n);
          }
      }
      float top = sc[0][0];
#pragma unroll
      for (int e = 1; e < 8; ++e) top = fmaxf(top, sc[e >> 2][e & 3]);
      top = rows_max(top);
      // (the reference point moves only when a tile's maximum exceeds it by more than tau: weights stay below 2^PAGED_TAU2)
      const bool grow = top > m + tau;   // m = -inf: any finite maximum
      const float mn = grow ? top : m;
      float nmc = mn == -INFINITY ? 0.0f : -mn * c2;
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
      const bool far = fabsf(nmc) >= PAGED_FAR;
      if (__any(far)) {
        nmc = far ? 0.0f : nmc;
#pragma unroll
        for (int e = 0; e < 8; ++e) sc[e >> 2][e & 3] = far ? sc[e >> 2][e & 3] - m : sc[e >> 2][e & 3];
      }
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
        load_v(next_length, next, q0, q1);
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
      tile = same ? next : g.to;
      p0 = q0;
      p1 = q1;
    }

    // ---- the waves' results together
    l = rows_sum(l);
    float* const results = reinterpret_cast<float*>(paged_lds + NW * T::WAVE);
    float* const my_o = results + wave * (T::RESULT / 4);
    barrier();   // (nobody reads the sequence's before any more)
#pragma unroll
    for (int d = 0; d < DT; ++d) {
      f32x4_t v = o[d];
      if constexpr (!E4M3)
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = fabsf(v[e]) < INFINITY ? v[e] + o_low[d][e] : v[e];
      *reinterpret_cast<f32x4_t*>(my_o + l16 * T::LDO + d * 16 + l4 * 4) = v;
    }
    if (l4 == 0) s_ml[wave][l16][0] = m * c2, s_ml[wave][l16][1] = l;   // (from here on in powers of two)
    barrier();
    const bool whole = g.from == 0 && g.to == g.n_tiles;
    const int slot = (group * (int)gridDim.x + w) * 2 + (g.from == 0 ? 1 : 0);
    for (int i = tid; i < nh * (HD / 4); i += 64 * NW) {
      const int h = i / (HD / 4), d = i % (HD / 4) * 4;
      float M = s_ml[0][h][0], L = 0.0f;
#pragma unroll
      for (int k = 1; k < NW; ++k) M = fmaxf(M, s_ml[k][h][0]);
      // (a wave that has seen no key has -inf, 0, 0; one that has seen only NaN -inf, NaN, NaN)
      const float ref = M == -INFINITY ? 0.0f : M;
      f32x4_t v = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int k = 0; k < NW; ++k) {
        const float f = exp2_hw(s_ml[k][h][0] - ref);
        L += f * s_ml[k][h][1];
        v += f * *reinterpret_cast<const f32x4_t*>(results + k * (T::RESULT / 4) + h * T::LDO + d);
      }
      if (whole) store_y(g.b, h, d, v, L);
      else store_part(slot, h, d, v, M, L);
    }
    if (!whole) {
      const int i = MANY && g.from == 0;
      open_b[i] = g.b;
      open_first[i] = g.first;
      open_tiles[i] = g.n_tiles;
    }
    if (!more_sequences) break;
    g = gn;
    pages = pages_n;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) qf[ks] = qn[ks];
  }

  // ---- parts put together (at the end: the stream above waits for nobody).  Workers w0 .. w1 have parts of a sequence, which the last of them puts
  // together; where they are more than PAGED_ONE, those of a block of PAGED_BLOCK workers by the block's last, and the blocks' results by the last block's.
  const int n_blocks = (gridDim.x + PAGED_BLOCK - 1) / PAGED_BLOCK, kw = w / PAGED_BLOCK, block_parts = 2 * (int)(gridDim.y * gridDim.x);
  const auto worker = [&](int at) {
    const int place = at - line0, n = larger * (each + 1);
    return from0 + (int)(place < n ? (u32)place / (u32)(each + 1) : larger + (u32)(place - n) / (u32)each);
  };
  // workers' parts first (of a block, or all of them), then blocks'; part u lies at places + 2 u, + 1 for the one
  // with the sequence's first tile
  struct Open {
    u32* ticket;
    int u0, u1, places, began, n_parts;
  };
  int k0[OPEN] = {}, k1[OPEN] = {};
  auto workers_of = [&](int i) {
    Open p = {};
    if (open_b[i] < 0) return p;
    const int w0 = MANY ? worker(open_first[i]) : 0, w1 = MANY ? worker(open_first[i] + open_tiles[i] - 1) : workers - 1;
    k0[i] = w0 / PAGED_BLOCK;
    k1[i] = w1 / PAGED_BLOCK;
    const bool one = k0[i] == k1[i] || w1 - w0 < PAGED_ONE;
    if (one) k1[i] = k0[i];
    p.u0 = one ? w0 : max(w0, kw * PAGED_BLOCK);
    p.u1 = one ? w1 : min(w1, kw * PAGED_BLOCK + PAGED_BLOCK - 1);
    p.places = group * (int)gridDim.x * 2;
    p.began = w0;
    p.ticket = a.tickets + (one ? (int64_t)group * B + open_b[i] : (int64_t)gridDim.y * B + (group * n_blocks + kw) * 2 + (kw == k0[i]));
    p.n_parts = p.u1 - p.u0 + 1;
    return p;
  };
  // s_ticket[i] = how many of p's parts there are with this one; then, in the last worker, all others' results can be read
  auto count = [&](const Open& p, int i) {
    if (tid == 64 * i && p.n_parts) {
      const u32 was = __hip_atomic_fetch_add(p.ticket, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      if (was + 1 == (u32)p.n_parts) __hip_atomic_store(p.ticket, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      s_ticket[i] = was + 1;
    }
  };
  if (open_b[0] < 0 && open_b[OPEN - 1] < 0) return;
  Open both[OPEN];
#pragma unroll
  for (int i = 0; i < OPEN; ++i) both[i] = workers_of(i);
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  barrier();
#pragma unroll
  for (int i = 0; i < OPEN; ++i) count(both[i], i);
  barrier();
  const bool last0 = both[0].n_parts && s_ticket[0] == (u32)both[0].n_parts, last1 = MANY && both[OPEN - 1].n_parts && s_ticket[1] == (u32)both[OPEN - 1].n_parts;
  asm volatile("" ::: "memory");
#pragma unroll 1
  for (int i = 0; i < OPEN; ++i) {
    bool last = i ? last1 : last0;
    Open p = i ? both[OPEN - 1] : both[0];
    const int b = i ? open_b[OPEN - 1] : open_b[0], first_block = i ? k0[OPEN - 1] : k0[0], last_block = i ? k1[OPEN - 1] : k1[0];
    bool final = first_block == last_block;
    const int block = (group * n_blocks + kw) * 2 + (kw == first_block ? 1 : 0);
#pragma unroll 1
    while (last) {
#pragma unroll 1
      for (int x = tid; x < nh * (HD / 4); x += 64 * NW) {
        const int h = x / (HD / 4), d = x % (HD / 4) * 4;
        float M = -INFINITY, L = 0.0f;
        f32x4_t v = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 1
        for (int u = p.u0; u <= p.u1; u += PAGED_BLOCK) {
          f32x4_t ov[PAGED_BLOCK];
          f32x2_t ml[PAGED_BLOCK];
#pragma unroll
          for (int k = 0; k < PAGED_BLOCK; ++k) {   // (all of them on their way before the first is used)
            const int from = (p.places + 2 * (u + k) + (u + k == p.began ? 1 : 0)) * 16 + h;
            ml[k] = __builtin_bit_cast(f32x2_t, __builtin_amdgcn_raw_buffer_load_b64(mres, u + k <= p.u1 ? from * 8 : PAGED_OUT, 0, PAGED_COHERENT));
            ov[k] = __builtin_bit_cast(f32x4_t, __builtin_amdgcn_raw_buffer_load_b128(ores, u + k <= p.u1 ? (from * HD + d) * 4 : PAGED_OUT, 0, PAGED_COHERENT));
          }
          float top = M;
#pragma unroll
          for (int k = 0; k < PAGED_BLOCK; ++k) {
            ml[k][0] = u + k <= p.u1 ? ml[k][0] : -INFINITY;   // (what is not there: weight, sum and values zero)
            top = fmaxf(top, ml[k][0]);
          }
          const float ref = top == -INFINITY ? 0.0f : top, f0 = exp2_hw(M - ref);
          L *= f0;
          v *= f0;
          M = top;
#pragma unroll
          for (int k = 0; k < PAGED_BLOCK; ++k) {
            const float f = exp2_hw(ml[k][0] - ref);
            L = fmaf(f, ml[k][1], L);
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = fmaf(f, ov[k][e], v[e]);
          }
        }
        if (final) store_y(b, h, d, v, L);
        else store_part(block_parts + block, h, d, v, M, L);
      }
      if (final) break;
      final = true;
      p = {a.tickets + (int64_t)group * B + b, first_block, last_block, block_parts + group * n_blocks * 2, first_block, last_block - first_block + 1};
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      barrier();
      count(p, 0);
      barrier();
      last = s_ticket[0] == (u32)p.n_parts;
      asm volatile("" ::: "memory");
    }
  }
}

struct DecodePlan {
  int groups_per_kv, groups, workers, blocks;
  size_t o_bytes, ml_bytes, ticket_bytes;
};
// Workers of a kv head (a group of up to 16 of its q heads): as many as the chip holds at once, no more than the table's pages could give
// four tiles each, one for each of their waves.
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
  static std::atomic<unsigned long long> raised[2] = {};
  const auto as = [&](auto MANY) -> int {
    if (!lr_raise_lds_limit(reinterpret_cast<const void*>(&k_paged_decode<HD, E4M3, MANY>), lds, raised[MANY])) return LR_E_LAUNCH;
    k_paged_decode<HD, E4M3, MANY><<<dim3(p.workers, p.groups), dim3(64 * DecodeTile<HD, E4M3>::NW), lds, s>>>(c, t, a);
    return lr_launch_status();
  };
  return t.B > 1 ? as(std::true_type{}) : as(std::false_type{});
}

// ------------------------------------------------------------------------------------ rows of prompts
// A kv head's rows of a sequence are its tokens' q heads, token after token: row r is token r / G, head r % G.  A workgroup has 128 of them,
// a wave 32, whatever G is: the columns of the products
//   S^T[key][row] = K q^T,   O^T[dim][row] += V^T P^T
// on the matrix cores (32x32x16).  A column is a lane, so maxima, sums and factors are a lane's own, and the 16 scores that it holds of 32 keys are, in
// their order, the second product's operand.  Weights enter as two bf16 numbers (2^-16 of the weight), as in a step of single tokens and in the prompts
// of the contiguous cache: a third of the products, 173 us instead of 136 for the prompts below.  (One number loses up to 2^-8 of each weight, about as
// much of y as its own rounding.)  Keys come 64 at a time into one of
// two buffers, one barrier per 64; bf16 by loads straight into LDS, e4m3 through registers, expanded on the way with its row's power of two:
// from there on the two are the same.
// Few rows: a workgroup's keys are cut among several, whose results a second launch puts together.
//
// Bound: the waves' instructions, one after another: 48 products of 32 cycles, 32 exponentials of 16 and 275 others of 4 per wave and 64 keys
// (counted) are 3150 cycles, of which a SIMD takes 2860: matrix instructions 54 % of its cycles, vector instructions 49 %, so that they run at the
// same time hardly more than neither does, though it has two waves (222 registers).  e4m3 46 % and 54 %.  Five prompts of up to 2048 tokens, 32 q and 8 kv heads of
// 128: 174 us (e4m3 186), 0.65 PFLOP/s of the 1.35 of a large library product, 0.98 with the weights' second numbers counted.  Slower, measured with
// weights of one number: products and exponentials of two tiles interleaved (137 -> 140), two groups of waves in turn (26.8 -> 28.4 for 256 tokens behind
// 8000), workgroups that take several blocks (the registers spill: 138 -> 146).
constexpr int PROMPT_ROWS = 128, PROMPT_KEYS = 64;
// Into how many parts a row's keys are cut at most: of 128 up to 16 parts, which are joined at once, else of 256.  (us, all of 256 / this: 4 sequences of 420 and 4
// tokens of the 8B model 14.1 / 10.6, 23 behind 1057 15.7 / 13.5; all of 128 / this: 8 tokens of 8 q heads on one kv head behind 7000 17.5 / 15.9.)
__host__ __device__ constexpr int prompt_parts_of(int keys) {
  const int half = (keys + 127) / 128, whole = (keys + 255) / 256;
  return half <= 16 ? half : whole > 16 ? whole : 16;
}

struct PagedPrompt {
  const u16* q;
  int64_t ldq;
  u16* y;
  int64_t ldy;
  int rows, Hq, n_split, bound;   // bound: blocks of a kv head at most
  float scale;
  float *o_part, *ml_part;        // [block][part][128][HD], [..][128][2]
};

// Which rows a block has.
struct PromptBlock {
  int b, row0, n, ahead, r0;     // sequence, its first row of the call and their number, its tokens ahead of them; the block's first row of the kv head's
  int held;                      // keys that the table has room for
};
// Blocks of a kv head, last ones first (they see the most keys).  false: there are fewer.
__device__ __forceinline__ bool prompt_block(const PagedCache& c, const PagedBatch& t, int rows, int G, int index, PromptBlock& at) {
  const int lane = threadIdx.x & 63;
  int start = 0, n = 0, ahead = 0, blocks = 0, upto = 0, total = 0;
  at.held = t.pages << c.shift;
  auto look = [&](int from) {
    const int i = from + lane;
    start = i < t.B ? t.starts[i] : 0;
    n = i < t.B ? t.starts[i + 1] - start : 0;
    n = start < 0 || start > rows || n < 0 ? 0 : n;
    const int length = i < t.B ? max(t.lengths[i], 0) : 0;   // (positions are the length's, also where the table has not all of its keys)
    if (n && length > at.held && t.err) *t.err = LR_DEV_POS_RANGE;
    ahead = length - n;
    n = min(n, rows - start);   // (a call may have fewer rows than starts says)
    blocks = (int)(((int64_t)n * G + PROMPT_ROWS - 1) / PROMPT_ROWS);
    upto = paged_sums(blocks);
    return __builtin_amdgcn_readlane(upto, 63);
  };
  for (int i = 0; i < t.B; i += 64) total += look(i);
  if (index >= total) return false;
  index = total - 1 - index;
  int b0 = 0, before = 0;
  if (t.B > 64)
    for (;; b0 += 64) {
      const int k = look(b0);
      if (index < before + k || b0 + 64 >= t.B) break;
      before += k;
    }
  int s = __popcll(__ballot(before + upto <= index));
  s = s > 63 ? 63 : s;
  at.b = b0 + s;
  at.row0 = __builtin_amdgcn_readlane(start, s);
  at.n = __builtin_amdgcn_readlane(n, s);
  at.r0 = (index - before - __builtin_amdgcn_readlane(upto - blocks, s)) * PROMPT_ROWS;
  at.ahead = __builtin_amdgcn_readlane(ahead, s);
  return at.r0 >= 0 && at.r0 < at.n * G;   // (starts that do not ascend name more blocks than 32 bits count)
}
// keys that the block's last row sees
__device__ __forceinline__ int prompt_keys(const PromptBlock& at, int G) {
  const int last = min(at.r0 + PROMPT_ROWS, at.n * G) - 1;
  return max(0, min(at.ahead + last / G + 1, at.held));
}
// and into how many parts they are cut
__device__ __forceinline__ int prompt_parts(int keys, int n_split) { return max(1, min(n_split, prompt_parts_of(keys))); }

template <int HD, int KSP>
struct PromptLds {
  static constexpr int ROW = HD * 2, TILE = PROMPT_KEYS * ROW, STAGE = 2 * TILE;   // a portion's keys or values; both
  static constexpr int MERGE = KSP == 2 ? 4 * (HD / 2 + 2) * 64 * 4 : 0;
  static constexpr int BYTES = 2 * STAGE > MERGE ? 2 * STAGE : MERGE;
};
// KSP 2: eight waves, the second four the second 32 keys of every portion for the same rows; their results meet in LDS.
template <int HD, bool E4M3, int KSP, bool SPLIT>
__global__ __launch_bounds__(256 * KSP, 2) void k_paged_prompt(const PagedCache c, const PagedBatch t, const PagedPrompt a) {
  using L = PromptLds<HD, KSP>;
  constexpr int KS = HD / 16, DT = HD / 32;   // k-steps of the score product; 32-row tiles of O^T
  constexpr int NW = 4 * KSP, RB = L::ROW, PIECES = RB / 16;
  extern __shared__ __attribute__((aligned(1024))) unsigned char prompt_lds[];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int part = KSP == 2 ? wave >> 2 : 0, w4 = wave & 3, col = lane & 31, half = lane >> 5;
  const int G = a.Hq / c.Hkv;
  // (workgroup i runs on XCD i % 8: the blocks of a kv head meet in few L2s)
  const int kvh = blockIdx.x % c.Hkv, item = blockIdx.x / c.Hkv, split = SPLIT ? item % a.n_split : 0, index = SPLIT ? item / a.n_split : item;
  PromptBlock at;
  if (!prompt_block(c, t, a.rows, G, index, at)) return;
  const int nkeys = prompt_keys(at, G), portions = (nkeys + PROMPT_KEYS - 1) / PROMPT_KEYS;
  int t_first = 0, t_end = nkeys;
  if constexpr (SPLIT) {
    const int parts = prompt_parts(nkeys, a.n_split);
    if (split >= parts) return;
    t_first = (int)((int64_t)portions * split / parts) * PROMPT_KEYS;
    t_end = min(nkeys, (int)((int64_t)portions * (split + 1) / parts) * PROMPT_KEYS);
  }
  // this lane's row, the last key that it sees, and the smallest and largest of the wave's
  const int n_rows = at.n * G, r = at.r0 + w4 * 32 + col, token = r / G;
  const bool valid = r < n_rows;
  const int p = valid ? min(at.ahead + token, at.held - 1) : -1;
  const int wr0 = at.r0 + w4 * 32;
  const int pmin = __builtin_amdgcn_readfirstlane(min(at.ahead + wr0 / G, at.held - 1));
  const int pmax = __builtin_amdgcn_readfirstlane(wr0 < n_rows ? min(at.ahead + (min(wr0 + 32, n_rows) - 1) / G, at.held - 1) : -1);
  const int64_t my_row = at.row0 + (valid ? token : 0);
  const int head = kvh * G + (valid ? r - token * G : 0);

  // the pages of 16 keys each, 64 of these at a time; which are not there
  const int32_t* const row = t.table + (int64_t)at.b * t.ld_table;
  int pages, groups0;
  u32 page_lo, page_hi;   // bf16: where the page's rows of this kv head begin (e4m3 has the page's number times the kv heads and its own in `pages`)
  unsigned long long gone;
  auto ask_pages = [&](int key0) {
    groups0 = key0;
    const int key = key0 + 16 * lane;
    pages = key < t_end ? row[key >> c.shift] : 0;
  };
  auto check_pages = [&]() {
    const bool bad = (u32)pages >= (u32)c.n_pages;
    if (bad && t.err) *t.err = LR_DEV_PAGE_RANGE;
    pages = bad || groups0 + 16 * lane >= t_end ? -1 : pages;
    gone = __ballot(bad);
    const int64_t off = paged_offset<RB>(c, pages < 0 ? 0 : pages, kvh);
    page_lo = (u32)off;
    page_hi = (u32)(off >> 32);
    pages = pages < 0 ? -1 : paged_index(c, pages, kvh);
  };
  auto pages_from = [&](int key0) {
    ask_pages(key0);
    check_pages();
  };
  ask_pages(t_first);
  // q as the products' second operand: k-step i holds elements 16 i + 8 half .. + 8 of this lane's row
  u32x4_t qb[KS];
  {
    const u16* const qrow = a.q + my_row * a.ldq + head * HD;
#pragma unroll
    for (int i = 0; i < KS; ++i) {
      const uint4 x = ld16(qrow + 16 * i + 8 * half);
      qb[i] = u32x4_t{x.x, x.y, x.z, x.w};
    }
  }
  check_pages();   // (asked for ahead of q: what is asked for comes in its order)
  f32x16_t o[DT];
#pragma unroll
  for (int d = 0; d < DT; ++d)
#pragma unroll
    for (int v = 0; v < 16; ++v) o[d][v] = 0.0f;
  float m = -INFINITY, l = 0.0f;   // m: reference point in raw scores; l: this lane's half of the row's sum
  const float c2 = a.scale * 1.4426950408889634f, tau = fminf(PAGED_TAU2 / c2, FLT_MAX);

  // ---- loads of a portion
  constexpr int RPL = 1024 / RB, LOADS = PROMPT_KEYS / RPL / NW;   // bf16: rows per load instruction; a wave's loads of K or V
  const u32 lds0 = __builtin_amdgcn_readfirstlane((u32)(uintptr_t)(__attribute__((address_space(3))) unsigned char*)prompt_lds);
  const int lrow = lane / PIECES, place = lane % PIECES;
  static_assert(NW * RPL % 16 == 0 && RPL % 4 == 0, "a lane's piece is the same for all of a wave's loads");
  const int kvoff = lrow * RB + (place ^ key_swizzle<HD>(wave * RPL + lrow)) * 16;
  const int vvoff = lrow * RB + (place ^ value_swizzle<HD>(lrow)) * 16;
  // (with few scalar instructions per load, which a wave issues one by one beside everything else: 150 for the eight of a portion, now 70; 143.5 -> 141 us)
  auto stage_as = [&](auto WHOLE, int t0, int buf) {
    const int group0 = (t0 - groups0 + wave * RPL) >> 4;
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      const int first = (i * NW + wave) * RPL, group = group0 + i * NW * RPL / 16;
      const int64_t off = (int64_t)((unsigned long long)__builtin_amdgcn_readlane(page_hi, group) << 32 | (u32)__builtin_amdgcn_readlane(page_lo, group));
      const bool ok = WHOLE || (t0 + first + lrow < t_end && !(gone >> group & 1));
      const int soff = ((t0 + first) & ((1 << c.shift) - 1)) * RB;
      const u32 to = lds0 + buf * L::STAGE + (i * NW + wave) * 1024;
      paged_load16(paged_resource(c.k + off), ok ? kvoff : PAGED_OUT, soff, to);
      paged_load16(paged_resource(c.v + off), ok ? vvoff : PAGED_OUT, soff, to + L::TILE);
    }
  };
  auto stage = [&](int t0, int buf) {
    if (t0 + PROMPT_KEYS <= t_end && gone == 0) stage_as(std::true_type{}, t0, buf);
    else stage_as(std::false_type{}, t0, buf);
  };
  // e4m3: 16 elements of K's or V's rows per piece
  constexpr int NP = 8 * HD / (256 * KSP), HP = HD / 16;
  uint4 raw[E4M3 ? NP : 1];
  u32 byte[E4M3 ? NP : 1];
  auto fetch = [&](int t0) {
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      const int x = i * 256 * KSP + tid, value = x >= 4 * HD, key = x % (4 * HD) / HP, pc = x % HP;
      const int index = __shfl(pages, (t0 - groups0 + key) >> 4, 64);
      const bool ok = index >= 0 && t0 + key < t_end;
      const int slot = (t0 + key) & ((1 << c.shift) - 1), safe = ok ? index : 0;
      raw[i] = ld16((value ? c.v : c.k) + paged_offset<HD>(c, safe) + slot * HD + pc * 16);
      byte[i] = c.scales[paged_scales(c, safe) + (value << c.shift) + slot];
      if (!ok) raw[i] = make_uint4(0, 0, 0, 0), byte[i] = 127;
    }
  };
  auto expand = [&](int buf) {
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      const int x = i * 256 * KSP + tid, value = x >= 4 * HD, key = x % (4 * HD) / HP, pc = x % HP;
      const float s = paged_scale(byte[i]);
      auto two = [&](u32 lo, u32 hi) {
        return make_uint4(__builtin_bit_cast(u32, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, s, false)),
                          __builtin_bit_cast(u32, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, s, true)),
                          __builtin_bit_cast(u32, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, s, false)),
                          __builtin_bit_cast(u32, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, s, true)));
      };
      unsigned char* const to = prompt_lds + buf * L::STAGE + value * L::TILE + key * RB;
      const int swap = value ? value_swizzle<HD>(key) : key_swizzle<HD>(key);
      *reinterpret_cast<uint4*>(to + ((2 * pc) ^ swap) * 16) = two(raw[i].x, raw[i].y);
      *reinterpret_cast<uint4*>(to + ((2 * pc + 1) ^ swap) * 16) = two(raw[i].z, raw[i].w);
    }
  };

  // where this lane reads: the K fragments of key `col` of a tile (k-step i: XOR 32 i), and 4 dimensions of key (lane % 16) / 4 of the
  // four keys whose values 16 lanes exchange (32-row tile d of O^T)
  const int kat = (part * 32 + col) * RB + ((half ^ key_swizzle<HD>(col)) * 16);
  const int vkey = (lane & 15) >> 2;
  int vat[DT];
#pragma unroll
  for (int d = 0; d < DT; ++d) {
    const int piece = 4 * d + ((lane >> 4) & 1) * 2 + ((lane & 3) >> 1);
    vat[d] = L::TILE + (part * 32 + 4 * half + vkey) * RB + (piece ^ value_swizzle<HD>(vkey)) * 16 + (lane & 1) * 8;
  }
  // this wave's tiles of 32 keys of the portion at t0
  auto tiles = [&](int t0, int buf) {
    constexpr int N = KSP == 2 ? 1 : 2;
    const int tk = t0 + part * 32;
    const unsigned char* const from = prompt_lds + buf * L::STAGE;
    f32x16_t sacc[N];
#pragma unroll
    for (int n = 0; n < N; ++n)
#pragma unroll
      for (int v = 0; v < 16; ++v) sacc[n][v] = 0.0f;
    u32x4_t ka[KS][N];
#pragma unroll
    for (int i = 0; i < KS; ++i)
#pragma unroll
      for (int n = 0; n < N; ++n) ka[i][n] = *reinterpret_cast<const u32x4_t*>(from + (kat ^ (32 * i)) + n * 32 * RB);
    // (all of them on their way before the first product: 136 -> 134.5 us; e4m3 has no registers for that)
    if constexpr (!E4M3) __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < KS; ++i)
#pragma unroll
      for (int n = 0; n < N; ++n)
        sacc[n] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, ka[i][n]), __builtin_bit_cast(bf16x8_t, qb[i]), sacc[n], 0, 0, 0);
    __builtin_amdgcn_s_setprio(1);   // (softmax and second product ahead of the other workgroup's first one: 140 -> 136.6 us, e4m3 159 -> 151)
    // element v of tile n: key tk + 32 n + (v / 4) * 8 + half * 4 + v % 4
    const u32 lost = (u32)(gone >> ((tk - groups0) >> 4)) & (N == 2 ? 15 : 3);
    if (tk + 32 * N - 1 > pmin || lost) {   // uniform
#pragma unroll
      for (int n = 0; n < N; ++n)
#pragma unroll
        for (int v = 0; v < 16; ++v) {
          const int key = tk + 32 * n + (v / 4) * 8 + half * 4 + (v % 4);
          sacc[n][v] = key <= p && !(lost >> (2 * n + v / 8) & 1) ? sacc[n][v] : -INFINITY;
        }
    }
    float top = sacc[0][0];
#pragma unroll
    for (int v = 1; v < 16 * N; ++v) top = max_med3(top, sacc[v / 16][v % 16]);   // (a row that sees NaN is NaN, whatever this is)
    {
      const u32 u = __float_as_uint(top);
      const auto x = __builtin_amdgcn_permlane32_swap(u, u, false, false);
      top = fmaxf(__uint_as_float(x[0]), __uint_as_float(x[1]));
    }
    const bool grow = top > m + tau;   // m = -inf: any finite maximum
    const float mn = grow ? top : m;
    float nmc = mn == -INFINITY ? 0.0f : -mn * c2;
    if (__any(grow)) {
      const float corr = grow ? exp2_hw((m - mn) * c2) : 1.0f;   // m = -inf: 0
      l *= corr;
#pragma unroll
      for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int v = 0; v < 16; ++v) o[d][v] *= corr;
    }
    m = mn;
    const bool far = fabsf(nmc) >= PAGED_FAR;
    if (__any(far)) {
      nmc = far ? 0.0f : nmc;
#pragma unroll
      for (int n = 0; n < N; ++n)
#pragma unroll
        for (int v = 0; v < 16; ++v) sacc[n][v] = far ? sacc[n][v] - m : sacc[n][v];
    }
#pragma unroll
    for (int n = 0; n < N; ++n) {
      u32x4_t ph[2], pl[2];
#pragma unroll
      for (int h2 = 0; h2 < 2; ++h2)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float x0 = exp2_hw(fmaf(sacc[n][8 * h2 + 2 * j], c2, nmc)), x1 = exp2_hw(fmaf(sacc[n][8 * h2 + 2 * j + 1], c2, nmc));   // masked: 0
          l += x0 + x1;
          const u32 hi = pack_bf2(x0, x1);
          ph[h2][j] = hi;
          pl[h2][j] = pack_bf2(x0 - bf_lo(hi), x1 - bf_hi(hi));
        }
      // k-step h2 covers keys 16 h2 + {0..3, 8..11} + 4 half of the tile, in the order of sacc
#pragma unroll
      for (int h2 = 0; h2 < 2; ++h2) {
        bf16x8_t va[DT];
#pragma unroll
        for (int d = 0; d < DT; ++d) {
          const unsigned char* const v0 = from + vat[d] + (n * 32 + 16 * h2) * RB;
          const i16x4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) i16x4_t*)(v0));
          const i16x4_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) i16x4_t*)(v0 + 8 * RB));
          va[d] = __builtin_bit_cast(bf16x8_t, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
        }
#pragma unroll
        for (int d = 0; d < DT; ++d)
          o[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(va[d], __builtin_bit_cast(bf16x8_t, ph[h2]), o[d], 0, 0, 0);
#pragma unroll
        for (int d = 0; d < DT; ++d)
          o[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(va[d], __builtin_bit_cast(bf16x8_t, pl[h2]), o[d], 0, 0, 0);
      }
    }
  };

  int buf = 0;
  if (t_first < t_end) {
    if constexpr (E4M3) {
      fetch(t_first);
      expand(0);
    } else {
      stage(t_first, 0);
    }
  }
  paged_wait_loads<0>();
#pragma unroll
  for (int i = 0; i < KS; ++i) asm volatile("" : "+v"(qb[i]));   // (q is here with the first portion; inside the loop its wait would be one for the next portion)
  for (int t0 = t_first; t0 < t_end; t0 += PROMPT_KEYS, buf ^= 1) {
    // the portion has arrived, for all waves, and nobody reads the one before any more
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    const bool more = t0 + PROMPT_KEYS < t_end;
    const unsigned long long gone_now = gone;
    const int groups_now = groups0;
    if (more) {
      if (t0 + PROMPT_KEYS - groups0 == 1024) pages_from(t0 + PROMPT_KEYS);
      if constexpr (E4M3) fetch(t0 + PROMPT_KEYS);
      else stage(t0 + PROMPT_KEYS, buf ^ 1);
    }
    {
      const unsigned long long gone_next = gone;
      const int groups_next = groups0;
      gone = gone_now;
      groups0 = groups_now;
      const int tk = t0 + part * 32;
      if (tk <= pmax) tiles(t0, buf);
      gone = gone_next;
      groups0 = groups_next;
    }
    __builtin_amdgcn_s_setprio(0);
    if constexpr (E4M3)
      if (more) expand(buf ^ 1);
  }
  // The products take a tile's values for all rows: one that is not finite reached also those that do not see its key, as 0 * v.  And an infinite
  // one that all see met the weights' second numbers, of which some are zero or negative.  Rare, and not worth a look at every value: a wave that ends with
  // something that is not finite, and has such a value among its keys, does its rows again, key by key.  (NaN that all rows see is right as it is.)
  {
    float none = 0.0f;
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int v = 0; v < 16; ++v) none = fmaf(o[d][v], 0.0f, none);
    if (__any(none != none)) {
      auto my_key = [&](int key) { return key >= t_first && key < t_end && (KSP == 1 || ((key - t_first) >> 5 & 1) == part); };
      auto page_of = [&](int key) {
        const int page = row[key >> c.shift];
        return (u32)page < (u32)c.n_pages ? page : -1;
      };
      // elements d .. d + 3 of a key's row
      auto four = [&](bool value, int page, int key, int d) {
        const int slot = key & ((1 << c.shift) - 1);
        const u8* const from = (value ? c.v : c.k) + paged_offset<HD * (E4M3 ? 1 : 2)>(c, page, kvh) + (slot * HD + d) * (E4M3 ? 1 : 2);
        u32x2_t x;
        if constexpr (E4M3) {
          const u32 u = *reinterpret_cast<const u32*>(from);
          const float s = paged_scale(c.scales[paged_scales(c, page, kvh) + ((int)value << c.shift) + slot]);
          x.x = __builtin_bit_cast(u32, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(u, s, false));
          x.y = __builtin_bit_cast(u32, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(u, s, true));
        } else {
          x = *reinterpret_cast<const u32x2_t*>(from);
        }
        return f32x4_t{bf_lo(x.x), bf_hi(x.x), bf_lo(x.y), bf_hi(x.y)};
      };
      bool some = false;
      const auto finite = [](float x) { return fabsf(x) < INFINITY; };
      constexpr int AT_ONCE = 64 / (HD / 8);   // keys: a lane looks at eight elements
#pragma unroll 1
      for (int k0 = t_first; k0 < t_end && k0 < pmax + PROMPT_KEYS; k0 += AT_ONCE) {   // (those of its last portion that none of them sees, too)
        const int key = k0 + lane / (HD / 8), page = my_key(key) ? page_of(key) : -1;
        if (page < 0) continue;
#pragma unroll
        for (int j = 0; j < 8; j += 4) {
          const f32x4_t v = four(true, page, key, lane % (HD / 8) * 8 + j);
#pragma unroll
          for (int e = 0; e < 4; ++e) some |= key > pmin ? !finite(v[e]) : fabsf(v[e]) == INFINITY;
        }
      }
      if (__any(some)) {
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
          for (int v = 0; v < 16; ++v) o[d][v] = 0.0f;
        const float ref = m == -INFINITY ? 0.0f : m;
#pragma unroll 1
        for (int key = t_first; key < t_end && key <= pmax; ++key) {
          const int page = my_key(key) ? page_of(key) : -1;
          if (page < 0) continue;
          float s = 0.0f;
#pragma unroll
          for (int i = 0; i < KS; ++i)
#pragma unroll
            for (int j = 0; j < 8; j += 4) {
              const f32x4_t k4 = four(false, page, key, 16 * i + 8 * half + j);
              const u32 q0 = qb[i][j / 2], q1 = qb[i][j / 2 + 1];
              s = fmaf(bf_lo(q0), k4[0], s);
              s = fmaf(bf_hi(q0), k4[1], s);
              s = fmaf(bf_lo(q1), k4[2], s);
              s = fmaf(bf_hi(q1), k4[3], s);
            }
          s += __shfl_xor(s, 32, LR_WAVE);
          const float weight = exp2_hw(fminf(s - ref, tau) * c2);   // (no larger than the products' ones, however this sum is rounded)
#pragma unroll
          for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int g4 = 0; g4 < 4; ++g4) {
              const f32x4_t v4 = four(true, page, key, d * 32 + g4 * 8 + half * 4);
#pragma unroll
              for (int e = 0; e < 4; ++e) o[d][4 * g4 + e] = key <= p ? fmaf(weight, v4[e], o[d][4 * g4 + e]) : o[d][4 * g4 + e];
            }
        }
      }
    }
  }
  if constexpr (KSP == 2) {
    // the second four waves' results to the first four
    __syncthreads();
    float* const mine = reinterpret_cast<float*>(prompt_lds) + w4 * (HD / 2 + 2) * 64 + lane;
    if (part) {
#pragma unroll
      for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int v = 0; v < 16; ++v) mine[(d * 16 + v) * 64] = o[d][v];
      mine[(HD / 2) * 64] = m;
      mine[(HD / 2 + 1) * 64] = l;
    }
    __syncthreads();
    if (!part) {
      // (-inf, 0, 0: no key seen; -inf, NaN, NaN: only NaN)
      const float m1 = mine[(HD / 2) * 64], mn = fmaxf(m, m1), ref = mn == -INFINITY ? 0.0f : mn;
      const float f0 = exp2_hw((m - ref) * c2), f1 = exp2_hw((m1 - ref) * c2);
      l = l * f0 + mine[(HD / 2 + 1) * 64] * f1;
#pragma unroll
      for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int v = 0; v < 16; ++v) o[d][v] = fmaf(o[d][v], f0, mine[(d * 16 + v) * 64] * f1);
      m = mn;
    }
  }
  l += __shfl_xor(l, 32, LR_WAVE);
  // element v of tile d: dimension d * 32 + (v / 4) * 8 + half * 4 + v % 4
  if (!SPLIT || prompt_parts(nkeys, a.n_split) == 1) {
    // through the wave's part of LDS, so that whole rows are stored: 16 bytes a lane, as they lie
    const float inv = l != 0.0f ? 1.0f / l : 0.0f;
    unsigned char* const mine = prompt_lds + w4 * 32 * RB;
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");   // (nobody reads keys and values, or the other four waves' results, any more)
    if (part) return;
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int g4 = 0; g4 < 4; ++g4) {
        uint2 w2;
        w2.x = pack_bf2(o[d][4 * g4] * inv, o[d][4 * g4 + 1] * inv);
        w2.y = pack_bf2(o[d][4 * g4 + 2] * inv, o[d][4 * g4 + 3] * inv);
        *reinterpret_cast<uint2*>(mine + col * RB + ((d * 4 + g4) ^ (col & (PIECES - 1))) * 16 + half * 8) = w2;
      }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
    for (int i = 0; i < 32 / RPL; ++i) {
      const int k = i * RPL + lrow, rk = wr0 + k, tk = rk / G;
      const uint4 x = *reinterpret_cast<const uint4*>(mine + k * RB + (place ^ (k & (PIECES - 1))) * 16);
      if (rk < n_rows) st16(a.y + (at.row0 + tk) * a.ldy + (kvh * G + rk - tk * G) * HD + place * 8, x);
    }
  } else if (valid && !part) {
    const int64_t place_ = ((int64_t)(kvh * a.bound + index) * a.n_split + split) * PROMPT_ROWS + w4 * 32 + col;
    float* const to = a.o_part + place_ * HD;
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int g4 = 0; g4 < 4; ++g4)
        *reinterpret_cast<f32x4_t*>(to + d * 32 + g4 * 8 + half * 4) = f32x4_t{o[d][4 * g4], o[d][4 * g4 + 1], o[d][4 * g4 + 2], o[d][4 * g4 + 3]};
    if (half == 0) *reinterpret_cast<f32x2_t*>(a.ml_part + place_ * 2) = f32x2_t{m * c2, l};
  }
}

// The parts of a block's rows together: a workgroup takes 1024 / HD of its 128 rows at a time, a lane four dimensions of one.
template <int HD>
__global__ __launch_bounds__(256) void k_paged_prompt_join(const PagedCache c, const PagedBatch t, const PagedPrompt a) {
  const int G = a.Hq / c.Hkv, kvh = blockIdx.x % c.Hkv, index = blockIdx.x / c.Hkv;
  PromptBlock at;
  if (!prompt_block(c, t, a.rows, G, index, at)) return;
  const int parts = prompt_parts(prompt_keys(at, G), a.n_split);
  if (parts == 1) return;
  const int d = threadIdx.x % (HD / 4) * 4;
  auto rows = [&](auto N_) __attribute__((always_inline)) {
    constexpr int AT_ONCE = decltype(N_)::value;
    for (int k = blockIdx.y * (1024 / HD) + threadIdx.x / (HD / 4); k < PROMPT_ROWS && at.r0 + k < at.n * G; k += gridDim.y * (1024 / HD)) {
      const int r = at.r0 + k;
      const int64_t place = (int64_t)(kvh * a.bound + index) * a.n_split * PROMPT_ROWS + k;
      float M = -INFINITY, L = 0.0f;
      f32x4_t v = {0.0f, 0.0f, 0.0f, 0.0f};
      for (int u = 0; u < parts; u += AT_ONCE) {
        f32x4_t ov[AT_ONCE];
        f32x2_t ml[AT_ONCE];
#pragma unroll
        for (int j = 0; j < AT_ONCE; ++j) {   // (all of them on their way before the first is used; behind the last part, that one again)
          const int64_t x = place + (int64_t)min(u + j, parts - 1) * PROMPT_ROWS;
          ml[j] = *reinterpret_cast<const f32x2_t*>(a.ml_part + x * 2);
          ov[j] = *reinterpret_cast<const f32x4_t*>(a.o_part + x * HD + d);
        }
        float top = M;
#pragma unroll
        for (int j = 0; j < AT_ONCE; ++j) top = fmaxf(top, ml[j][0]);
        const float ref = top == -INFINITY ? 0.0f : top, f0 = exp2_hw(M - ref);
        L *= f0;
        v *= f0;
        M = top;
#pragma unroll
        for (int j = 0; j < AT_ONCE; ++j) {
          if (u + j < parts) {
            const float f = exp2_hw(ml[j][0] - ref);
            L = fmaf(f, ml[j][1], L);
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = fmaf(f, ov[j][e], v[e]);
          }
        }
      }
      const float inv = L != 0.0f ? 1.0f / L : 0.0f;
      u32x2_t out;
      out.x = pack_bf2(v[0] * inv, v[1] * inv);
      out.y = pack_bf2(v[2] * inv, v[3] * inv);
      *reinterpret_cast<u32x2_t*>(a.y + (at.row0 + r / G) * a.ldy + (kvh * G + r % G) * HD + d) = out;
    }
  };
  if (parts <= 4) rows(std::integral_constant<int, 4>{});
  else rows(std::integral_constant<int, 16>{});
}

struct PromptPlan {
  int bound, n_split, waves;   // waves: four or eight of a workgroup
  int64_t items;
  size_t bytes;   // of parts that any number of rows could need
};
static PromptPlan prompt_plan(const PagedCache& c, const PagedBatch& t, int hd, int rows, int Hq) {
  PromptPlan p;
  const int G = Hq / c.Hkv, cus = lr_num_cus() ? lr_num_cus() : 256;
  const int64_t some = t.B < rows ? t.B : rows;   // sequences with rows, at most: the last block of each may be short
  p.items = ((int64_t)rows * G + (PROMPT_ROWS - 1) * some) / PROMPT_ROWS;
  p.bound = p.items > 0x3fffffff ? 0x3fffffff : (int)p.items;
  p.items *= c.Hkv;
  const int most = prompt_parts_of(t.pages << c.shift);
  int64_t n = p.items ? cus / p.items : 1;
  if (n > most) n = most;
  // Parts save a row's last block (1 - 1 / n) of its portions, about 1.3 us each, and cost a second launch, 4 to 6 us.  us, one part / several:
  // 300 tokens of the 8B model (6 portions, 2 parts) 12.0 / 15.9, 700 of 12 heads of 64 (12, 3) 12.6 / 14.1, 8 tokens behind 1000 (17, 5) 23.7 / 12.8.
  const int64_t portions = (((int64_t)t.pages << c.shift) + PROMPT_KEYS - 1) / PROMPT_KEYS;
  if (n < 1 || portions * (n - 1) <= 8 * n) n = 1;
  p.n_split = (int)n;
  // eight waves where they would be the CU's only ones and have something to share (us, four / eight: 700 tokens of 12 heads of 64 14.5 / 12.7,
  // 300 of the 8B model 12.0 / 12.2, 100 of 32 heads of 64 6.8 / 7.3)
  p.waves = n > 1 || (p.items <= cus && portions >= 8) ? 8 : 4;
  p.bytes = most > 1 ? (size_t)cus * PROMPT_ROWS * (hd + 2) * 4 : 0;
  return p;
}

template <int HD, bool E4M3, int KSP, bool SPLIT>
static int launch_prompt_as(const PagedCache& c, const PagedBatch& t, const PagedPrompt& a, unsigned grid, hipStream_t s) {
  constexpr size_t lds = PromptLds<HD, KSP>::BYTES;
  static std::atomic<unsigned long long> raised{0};
  if (!lr_raise_lds_limit(reinterpret_cast<const void*>(&k_paged_prompt<HD, E4M3, KSP, SPLIT>), lds, raised)) return LR_E_LAUNCH;
  k_paged_prompt<HD, E4M3, KSP, SPLIT><<<dim3(grid), dim3(256 * KSP), lds, s>>>(c, t, a);
  return lr_launch_status();
}
template <int HD, bool E4M3>
static int launch_prompt(const PagedCache& c, const PagedBatch& t, const PagedQuery& q, void* scratch, hipStream_t s) {
  const PromptPlan p = prompt_plan(c, t, HD, q.rows, q.Hq);
  PagedPrompt a = {q.q, q.ldq, q.y, q.ldy, q.rows, q.Hq, p.n_split, p.bound, q.scale, (float*)scratch, nullptr};
  a.ml_part = a.o_part + (size_t)p.items * p.n_split * PROMPT_ROWS * HD;
  if (p.n_split == 1)
    return p.waves == 8 ? launch_prompt_as<HD, E4M3, 2, false>(c, t, a, (unsigned)p.items, s) : launch_prompt_as<HD, E4M3, 1, false>(c, t, a, (unsigned)p.items, s);
  if (const int rc = launch_prompt_as<HD, E4M3, 2, true>(c, t, a, (unsigned)(p.items * p.n_split), s)) return rc;
  // (us, 16 blocks in 16 parts with 8 and 16 workgroups a block 8.2, 5.6; 128 blocks in 2 parts 7.6, 12.3)
  const int64_t join = p.items < 64 ? PROMPT_ROWS * HD / 1024 : 1024 / p.items;
  k_paged_prompt_join<HD><<<dim3((unsigned)p.items, (unsigned)(join < 1 ? 1 : join)), dim3(256), 0, s>>>(c, t, a);
  return lr_launch_status();
}

// (0: refused)
static size_t paged_scratch(const PagedCache& c, const PagedBatch& t, int hd, bool e4m3, int rows, int Hq) {
  // (rows times heads and 128 more are 32-bit numbers)
  if (rows <= 0 || Hq <= 0 || Hq > 65535 || Hq % c.Hkv || (int64_t)rows * Hq > 1 << 30 || (t.starts == nullptr && rows != t.B)) return 0;
  if (t.starts) {
    const PromptPlan p = prompt_plan(c, t, hd, rows, Hq);
    return p.items * p.n_split * p.waves > 0xffffffff / 64 ? 0 : 256 + p.bytes;   // (a grid has fewer than 2^32 threads)
  }
  const DecodePlan p = hd == 128 ? (e4m3 ? decode_plan<128, true>(c, t, Hq) : decode_plan<128, false>(c, t, Hq))
                                 : (e4m3 ? decode_plan<64, true>(c, t, Hq) : decode_plan<64, false>(c, t, Hq));
  if (p.groups > 65535) return 0;   // (a grid's second dimension)
  return p.ticket_bytes + p.o_bytes + p.ml_bytes;
}

extern "C" size_t lr_paged_attention_scratch_bytes(const lr_paged_cache_t* cache, const lr_paged_batch_t* batch, int rows, int Hq) {
  PagedCache c;
  PagedBatch t;
  if (paged_arguments(cache, batch, c, t)) return 0;
  return paged_scratch(c, t, cache->head_dim, cache->format == LR_CACHE_E4M3, rows, Hq);
}

extern "C" int lr_paged_attention(const lr_paged_attention_t* desc, lr_stream_t stream) {
  if (desc == nullptr) return LR_E_NULL;
  const auto& [cache, batch, q, ldq, y, ldy, scratch, scratch_bytes, rows, Hq, scale] = *desc;
  PagedCache c;
  PagedBatch t;
  if (const int rc = paged_arguments(cache, batch, c, t)) return rc;
  LR_REQUIRE_PTR(q);
  LR_REQUIRE_PTR(y);
  LR_REQUIRE_PTR(scratch);
  const int hd = cache->head_dim;
  const bool e4m3 = cache->format == LR_CACHE_E4M3;
  if (rows <= 0 || Hq <= 0 || Hq > 65535 || Hq % c.Hkv || (t.starts == nullptr && rows != t.B)) return LR_E_SHAPE;
  if (ldq < (int64_t)Hq * hd || ldy < (int64_t)Hq * hd) return LR_E_SHAPE;
  // (the matrix cores give 0 for sums of some 2^-120: a scale that would lift those to numbers that matter is not served)
  if (!(scale > 0.0f && scale <= 0x1p64f)) return LR_E_SHAPE;
  if (ldq % 8 || ldy % 8) return LR_E_ALIGN;
  if (paged_overlap(q, ldq, y, ldy, rows, (int64_t)Hq * hd, (int64_t)Hq * hd)) return LR_E_SHAPE;
  const size_t need = paged_scratch(c, t, hd, e4m3, rows, Hq);
  if (need == 0) return LR_E_UNSUPPORTED;
  if (scratch_bytes < need) return LR_E_SHAPE;
  const PagedQuery a = {(const u16*)q, ldq, (u16*)y, ldy, rows, Hq, scale};
  hipStream_t s = (hipStream_t)stream;
  if (t.starts == nullptr)
    return hd == 128 ? (e4m3 ? launch_paged_decode<128, true>(c, t, a, scratch, s) : launch_paged_decode<128, false>(c, t, a, scratch, s))
                     : (e4m3 ? launch_paged_decode<64, true>(c, t, a, scratch, s) : launch_paged_decode<64, false>(c, t, a, scratch, s));
  return hd == 128 ? (e4m3 ? launch_prompt<128, true>(c, t, a, scratch, s) : launch_prompt<128, false>(c, t, a, scratch, s))
                   : (e4m3 ? launch_prompt<64, true>(c, t, a, scratch, s) : launch_prompt<64, false>(c, t, a, scratch, s));
}
