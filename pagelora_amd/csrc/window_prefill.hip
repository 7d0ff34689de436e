// Prefill attention over a paged KV cache of 16 or of 4 bits per value, under a
// sliding window with sinks (gfx950).
//
// Request r's queries are the last qo_len of its kv_len positions; the one at
// position p sees t <= p with t > p - window (window 0: every one) or t < sinks:
//   o = sum_t p_t v_t / sum_t p_t,  p_t = exp(s q . k_t).
//
// An item is 128 rows (query, head of the GQA group) of a request over a range of
// the kv tiles, 64 tokens each, that some of its rows see; the host plan cuts the
// ranges where the rows alone would leave the chip idle, and merge_kernel joins them
// in order.  Four waves of 32 rows, two columns of 16 each.
//
// A tile lies in LDS in 16 bits, two buffers, its 16-byte chunks permuted by the row
// so that the operand reads are free of bank conflicts.  16-bit pages are loaded
// straight into it; 4-bit ones are loaded into registers two tiles ahead and become
// bf16 (exact) on the way in, while the waves work on the tile before.  S^T = K Q^T
// keeps a query per lane, whose probabilities are the B operand of O^T += V^T P^T as
// they lie; V^T comes out of LDS transposed.
//
// For queries of fp16, K and V of 4 bits are multiplied in fp16, which takes fewer
// planes than bf16: one of q, two of the probabilities.  The values are exact there
// while their groups' scales are in a range; an item that met others is worked on again
// in bf16, which holds all of them.  For bf16 queries they are multiplied in bf16: a
// weight that fp16 cannot hold, under 2^-36 of the row's largest, counts in an output
// of bf16 where the larger ones meet zeros.
//
// Where an output is NaN (0 times an infinity, or the difference of two planes'
// infinities, is not what a row sees), the item is worked on again: V's infinities and
// NaN become ones in LDS, kind by kind, to find who sees them, then zeros.
//
// Long items run at the rate of a large library product (1.24 PFLOP/s in bf16, 1.19 in
// fp16), P's planes counted: a CU with two workgroups takes 1.65 us per 128 rows by 64
// tokens in bf16, 1.30 PFLOP/s (three planes: half of the products), and 1.33 in fp16,
// 1.21, over 16 bits and over 4 alike.  Shorter ones are bound by their starts (~6 us)
// and by the last items, which have a CU for themselves.
// Measured (head_dim 128; us of a pass, with the merge's 8 where ranges are cut):
//   2048 tokens, 4 bits, GQA 4, bf16       86 (94 .. 97 after pauses, at lower clocks; 55
//                                          with one plane of P in fp16, 11 bits)
//   512 behind 16384, 4 bits, GQA 7, fp16  171 (both in bf16, with two planes of q and P
//                                          and cut at one length for 512 slots 377)
//   8192 under 1024, 16 bits, GQA 4, bf16  249, 1.15 PFLOP/s with the masked products
//                                          and the planes (205 with two of them)
//   5 ragged prompts under 512, MHA, fp16  44.5
// Those after this with two planes of P in bf16.  A half's weights are formed between
// the products of the other half: 236 -> 225 us at 8192.  Tried, and not faster:
// products of 32 x 32 (half as many instructions: 226 us, spills over 4 bits), eight
// waves of 16 rows (twice the waves per SIMD: 270), the conversions of the next tile
// between the scores' products (spills: 2.3 times as long), a wave priority in the
// products or by the wave's slot.
#include <algorithm>
#include <functional>
#include <vector>

#include "window_common.h"

namespace pl {
namespace window {
namespace pre {

constexpr int kWaves = 4;
constexpr int kThreads = kWave * kWaves;
constexpr int kCols = 2;                    // 16-query columns per wave
constexpr int kWaveRows = 16 * kCols;
constexpr int kRows = kWaveRows * kWaves;   // rows per item
constexpr int kTile = 64;                   // kv tokens per tile

typedef short i16x4 __attribute__((ext_vector_type(4)));

// One work item, or (in the merge list) one row item split into parts: with all that
// its workgroup needs of its request, so that the page ids are its next load.  Tiles
// are counted by what the item's first row sees on.
struct alignas(64) Item {
  int32_t request, row0, rows;            // rows: all of the request's
  int32_t qo_begin, kv_len, page_begin;
  int32_t tile_begin, tile_end;
  int32_t slot;  // first part of the row item; -1: writes the output itself
  int32_t part, parts;
  int32_t pad[5];
};
static_assert(sizeof(Item) == 64, "the plan's record: 16 words");

// Scales that fp16 holds, V's after 2^kShift: down to the smallest normal number for
// the smallest code (0.5), up to 6 times a power.
constexpr uint32_t kShift = 10;
constexpr uint32_t kKLeast = 127 - 13, kKMost = 127 + 13;
constexpr uint32_t kVLeast = kKLeast - kShift, kVMost = kKMost - kShift;

constexpr int part_floats(int d) { return kRows * (d + 2); }  // outputs [row][dim], then (m, sum) per row

__device__ __forceinline__ void load_lds16(const char* g, char* l) {
  __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)g,
                                   (__attribute__((address_space(3))) void*)l, 16, 0, 0);
}
__device__ __forceinline__ u32x2 read_tr(const char* p) {
  return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) i16x4*)p));
}

struct Args {
  const char *q, *k, *v;
  char* o;
  float* part;
  const int32_t* kv_indices;
  const Item* items;
  int64_t q_st, q_sh, o_st, o_sh, page_stride, token_stride, head_stride;  // bytes
  int64_t num_pages;
  int hq, hkv, page_size, page_shift, window, sinks;
  float scale_log2;  // > 0; a negative scale negates q instead
  uint32_t q_flip;
};

// Which of V's values a walk over the tiles takes: all, or each kind of those that
// are not finite by itself (as ones, to find who sees them), or the finite ones.
enum Walk { kAll, kInf, kMinusInf, kNan, kFinite };

// Two halves of a word of V as `walk` takes them.
template <typename MT> __device__ __forceinline__ uint32_t taken(uint32_t w, int walk) {
  constexpr bool kBf16 = std::is_same<MT, bf16_t>::value;
  constexpr uint32_t kOne = kBf16 ? 0x3f80u : 0x3c00u, kTop = kBf16 ? 0x7f80u : 0x7c00u;
  uint32_t out = 0;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint32_t x = (w >> (16 * i)) & 0xffffu;
    const uint32_t y = walk == kFinite     ? (finite16(x, kBf16) ? x : 0u)
                       : walk == kInf      ? (x == kTop ? kOne : 0u)
                       : walk == kMinusInf ? (x == (kTop | 0x8000u) ? kOne : 0u)
                                           : ((x & 0x7fffu) > kTop ? kOne : 0u);
    out |= y << (16 * i);
  }
  return out;
}

constexpr int buffer_bytes(int d) { return kTile * d * 2; }

// One item's work.  N (narrow, fp16 over 4 bits): in fp16; false where a scale was out of
// its range, and nothing is written then.  s_k0 .. s_v1: a K and a V buffer each, one
// object per buffer, so that writes into one never alias reads of another.
template <typename T, bool FOUR, int D, bool PAGE16, bool N>
__device__ __forceinline__ bool work(const Args& A, char* __restrict__ s_k0, char* __restrict__ s_v0,
                                     char* __restrict__ s_k1, char* __restrict__ s_v1) {
  constexpr bool kHalf = std::is_same<T, f16_t>::value;
  static_assert(!N || (FOUR && kHalf), "narrow: fp16 over 4 bits");
  using MT = typename std::conditional<FOUR && !N, bf16_t, T>::type;  // what is multiplied
  using P = Planes<MT>;
  constexpr int QP = FOUR && !N && kHalf ? 2 : 1;  // planes of q
  constexpr int NP = P::kPlanes;                   // planes of p
  constexpr int NS = D / 32, NA = D / 16;
  constexpr int RB = D * 2;              // bytes of a row
  constexpr int CH = D / 8;              // its 16-byte chunks
  constexpr int TPL = kWave / CH;        // tokens of a load instruction
  constexpr int NL = 16 / TPL;           // load instructions of a wave's 16 tokens
  const int h = blockIdx.x % A.hkv;
  const Item it = A.items[blockIdx.x / A.hkv];
  const int row0 = uniform(it.row0), n_rows = uniform(it.rows);
  const int g = A.hq / A.hkv, qo_begin = uniform(it.qo_begin), kv_len = uniform(it.kv_len);
  const int32_t* ind = A.kv_indices + uniform(it.page_begin);
  const int ps = A.page_size;

  // (not known to be the thread's index, so that nothing is kept in registers from the
  // narrow work to the other)
  int tid = threadIdx.x;
  asm volatile("" : "+v"(tid));
  const int lane = tid % kWave, wave = uniform(tid / kWave);
  const int lr = lane % 16, grp = lane / 16;

  // what rows see: t <= lim and (t >= lo or t < sinks)
  const int base = kv_len - n_rows / g;
  const Seen seen = seen_from(base + row0 / g, A.window, A.sinks, kTile);
  auto low = [&](int p) { return A.window > 0 ? max(p - A.window + 1, 0) : 0; };
  // 4 bits: what no row of the item sees becomes zeros, so that it neither takes the item
  // out of fp16 nor through the tiles again for its NaN.
  const int last = base + (min(row0 + kRows, n_rows) - 1) / g;
  auto unseen = [&](int t) { return t > last || (t >= seen.se && t < seen.lo); };
  const int wrow = row0 + wave * kWaveRows;
  const bool wave_on = wrow < n_rows;
  const int lim_lo = wave_on ? base + wrow / g : -1;
  const int lim_hi = wave_on ? base + (min(wrow + kWaveRows, n_rows) - 1) / g : -1;
  const int lo_lo = low(lim_lo), lo_hi = low(lim_hi);
  int lim[kCols];
#pragma unroll
  for (int c = 0; c < kCols; ++c)  // rows past the end repeat the last one; not stored
    lim[c] = base + min(wrow + c * 16 + lr, n_rows - 1) / g;

  // q as the B operand, in the planes of what is multiplied
  u32x4 qb[QP][kCols][NS];
#pragma unroll
  for (int c = 0; c < kCols; ++c) {
    const int row = min(wrow + c * 16 + lr, n_rows - 1), pos = row / g;
    const char* qp = A.q + (int64_t)(qo_begin + pos) * A.q_st + (int64_t)(h * g + row - pos * g) * A.q_sh + grp * 16;
#pragma unroll
    for (int ks = 0; ks < NS; ++ks) {
      u32x4 w = *reinterpret_cast<const u32x4*>(qp + ks * 64);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        w[e] ^= A.q_flip;
        if constexpr (QP == 2) {
          float a, b;
          unpack2<f16_t>(w[e], a, b);
          w[e] = f32x2_to_bf16x2_bits(a, b);
          const float ra = a - bf16_lo(w[e]), rb = b - bf16_hi(w[e]);  // (the rest of an infinity is none)
          qb[QP - 1][c][ks][e] = f32x2_to_bf16x2_bits(ra == ra ? ra : 0.f, rb == rb ? rb : 0.f);
        }
      }
      qb[0][c][ks] = w;
    }
  }

  auto page_of = [&](int t) { return A.page_shift >= 0 ? t >> A.page_shift : t / ps; };
  auto clamp_page = [&](int id) -> int64_t {
    return (id < 0 ? 0 : ((int64_t)id >= A.num_pages ? A.num_pages - 1 : (int64_t)id)) * A.page_stride;
  };
  const int t_begin = uniform(it.tile_begin), t_end = uniform(it.tile_end);
  const char* kh = A.k + (int64_t)h * A.head_stride;
  const char* vh = A.v + (int64_t)h * A.head_stride;
  // Pages of 16 and more: lane l holds where the wave's 16 tokens of tile l of the
  // next 64 begin, so that no tile's loads wait for its page id.
  int64_t places = 0;
  auto load_places = [&](int tile) __attribute__((always_inline)) {
    const int t = min(seen_tile(seen, min(tile + lane, t_end - 1)) * kTile + wave * 16, (kv_len - 1) & ~15);
    const int page = page_of(t);
    places = clamp_page(ind[page]) + (int64_t)(t - page * ps) * (FOUR ? (int64_t)(D / 2) : A.token_stride);
  };
  auto place = [&](int tile) -> int64_t {
    const int l = (tile - t_begin) % 64;
    return (int64_t)((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(places >> 32), l) << 32 |
                     (uint32_t)__builtin_amdgcn_readlane((int)places, l));
  };
  // 16 bits: a wave fetches its 16 tokens of a tile, TPL per instruction; lane l of
  // one token l / CH, chunk (l % CH) permuted by the row
  uint32_t k_own[NL], v_own[NL];
#pragma unroll
  for (int j = 0; j < NL; ++j) {
    const int row = j * TPL + lane / CH;
    const uint32_t at = PAGE16 ? (uint32_t)(row * A.token_stride) : 0u;
    k_own[j] = at + ((lane % CH) ^ (row % CH)) * 16;
    v_own[j] = at + ((lane % CH) ^ (2 * (row % (CH / 2)))) * 16;
  }
  auto load_wide = [&](int tile, char* kd, char* vd) __attribute__((always_inline)) {
    kd += wave * 16 * RB;
    vd += wave * 16 * RB;
    if constexpr (PAGE16) {
      const int64_t at = place(tile);
#pragma unroll
      for (int j = 0; j < NL; ++j) {
        load_lds16((kh + at) + k_own[j], kd + j * TPL * RB);
        load_lds16((vh + at) + v_own[j], vd + j * TPL * RB);
      }
    } else {
      const int t0 = seen_tile(seen, tile) * kTile + wave * 16;
#pragma unroll
      for (int j = 0; j < NL; ++j) {
        const int t = min(t0 + j * TPL + lane / CH, kv_len - 1), pg = page_of(t);
        const int64_t at = clamp_page(ind[pg]) + (int64_t)(t - pg * ps) * A.token_stride;
        load_lds16(kh + at + k_own[j], kd + j * TPL * RB);
        load_lds16(vh + at + v_own[j], vd + j * TPL * RB);
      }
    }
  };
  // 4 bits: thread tid holds a quarter of K token tid / 4, and eight dims of V's
  // tokens 4 q .., q = tid / CH (at head_dim 64 the first half of the threads)
  constexpr int KQ = D / 32;             // words of a quarter
  struct Raw {
    uint32_t k[KQ], ks, vs;
    u32x4 v;
  } raw;
  const int k_tok = tid / 4, v_quad = CH == 16 ? tid / 16 : tid % (16 * CH) / CH, v_chunk = tid % CH;
  auto load_four = [&](int tile) __attribute__((always_inline)) {
    const int t0 = seen_tile(seen, tile) * kTile;
    const char *kp, *sp, *vp, *wp;  // K's codes and scale, V's
    if constexpr (PAGE16) {
      const int64_t at = place(tile);
      const int t = min(t0 + wave * 16, (kv_len - 1) & ~15), slot = A.page_shift >= 0 ? t & (ps - 1) : t % ps;
      const int64_t sat = at + ps * (D / 2) - slot * (D / 2 - D / 32);  // scales: D / 32 bytes a token, codes D / 2
      kp = (kh + at) + (uint32_t)(k_tok % 16 * (D / 2) + tid % 4 * (D / 8));
      sp = (kh + sat) + (uint32_t)(k_tok % 16 * (D / kGroup) + tid % 4 * (D / 4) / kGroup);
      vp = (vh + at) + (uint32_t)(v_quad % 4 * (2 * D) + v_chunk * 16);
      wp = (vh + sat) + (uint32_t)(v_quad % 4 * (D / 8) + v_chunk / 4 * 4);
    } else {
      const int t = min(t0 + k_tok, kv_len - 1), pg = page_of(t), ok = t - pg * ps;
      const char* page = kh + clamp_page(ind[pg]);
      kp = page + ok * (D / 2) + tid % 4 * (D / 8);
      sp = page + ps * (D / 2) + ok * (D / kGroup) + tid % 4 * (D / 4) / kGroup;
    }
    if constexpr (!PAGE16 || D != 128) {  // (at head_dim 64 V's tokens are not the wave's)
      const int t = min(t0 + v_quad * 4, (kv_len - 1) & ~3), pg = page_of(t), ov = t - pg * ps;
      const char* page = vh + clamp_page(ind[pg]);
      vp = page + ov / 4 * (2 * D) + v_chunk * 16;
      wp = page + ps * (D / 2) + ov / 4 * (D / 8) + v_chunk / 4 * 4;
    }
    if constexpr (KQ == 4) {
      const u32x4 x = *reinterpret_cast<const u32x4*>(kp);
#pragma unroll
      for (int e = 0; e < 4; ++e) raw.k[e % KQ] = x[e];
    } else {
      const u32x2 x = *reinterpret_cast<const u32x2*>(kp);
      raw.k[0] = x[0];
      raw.k[1] = x[1];
    }
    raw.ks = *reinterpret_cast<const uint8_t*>(sp);
    raw.v = *reinterpret_cast<const u32x4*>(vp);
    raw.vs = *reinterpret_cast<const uint32_t*>(wp);
  };
  // Narrow: K in fp16, and V times 2^kShift, exact where the scales are in range
  uint32_t v_least = ~0u, v_most = 0u, k_least = ~0u, k_most = 0u;
  auto store_four = [&](int tile, char* kd, char* vd) __attribute__((always_inline)) {
    const int t0 = seen_tile(seen, min(tile, t_end - 1)) * kTile;
    if (N && unseen(t0 + k_tok)) raw.ks = kScaleZero;
    const float ks = scale_of(raw.ks);
    if constexpr (N) {
      k_least = min(k_least, raw.ks);
      k_most = max(k_most, raw.ks);
    }
#pragma unroll
    for (int c = 0; c < KQ; ++c)
      *reinterpret_cast<u32x4*>(kd + k_tok * RB + (((tid % 4) * KQ + c) ^ (k_tok % CH)) * 16) =
          N ? halves8(raw.k[c], ks) : codes8(raw.k[c], ks);
    if (CH == 16 || tid < 16 * CH) {
      if (t0 + kTile > last + 1 || (t0 < seen.lo && t0 + kTile > seen.se)) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (unseen(t0 + v_quad * 4 + j)) {
            raw.v[j] = 0u;
            raw.vs = (raw.vs & ~(255u << (8 * j))) | (uint32_t)kScaleZero << (8 * j);
          }
      }
      if constexpr (N) {
        // the four bytes as two pairs of halves
        const uint32_t even = raw.vs & 0x00ff00ffu, odd = (raw.vs >> 8) & 0x00ff00ffu;
        v_least = pk_min(v_least, pk_min(even, odd));
        v_most = pk_max(v_most, pk_max(even, odd));
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int row = v_quad * 4 + j;
        const uint32_t byte = (raw.vs >> (8 * j)) & 255u;
        *reinterpret_cast<u32x4*>(vd + row * RB + (v_chunk ^ (2 * (row % (CH / 2)))) * 16) =
            N ? halves8(raw.v[j], scale_of(byte + kShift)) : codes8(raw.v[j], scale_of(byte));
      }
    }
  };

  auto load_next = [&](int tile) __attribute__((always_inline)) {
    tile = min(tile, t_end - 1);
    if (PAGE16 && (tile - t_begin) % 64 == 0) load_places(tile);
    load_four(tile);
  };

  // operand reads: K row blk*16 + lr, chunk 4 ks + grp; V tokens 4 grp + lr/4
  // (+16 per half, +32 per kc), dims 16 a + 4 (lr % 4)
  int kaddr[NS], vaddr[NA];
#pragma unroll
  for (int ks = 0; ks < NS; ++ks) kaddr[ks] = lr * RB + ((ks * 4 + grp) ^ (lr % CH)) * 16;
#pragma unroll
  for (int a = 0; a < NA; ++a) {
    const int row = grp * 4 + lr / 4;
    vaddr[a] = row * RB + (((2 * a + (lr % 4) / 2) ^ (2 * (row % (CH / 2)))) * 16) + (lr % 2) * 8;
  }

  f32x4 acc[kCols][NA];
  float m[kCols], l[kCols];
  const float sc = A.scale_log2, lag = P::kLag / sc;

  auto body = [&](int tile, const char* kb, char* vb, char* kn, char* vn, int walk) __attribute__((always_inline)) {
    if constexpr (!FOUR) {
      // this wave's loads of the tile are done, and past the barrier everyone's
      // are, and every wave is done with the other buffers
      __builtin_amdgcn_sched_barrier(0);
      __builtin_amdgcn_s_waitcnt(0xF70);
      __builtin_amdgcn_s_barrier();
      __builtin_amdgcn_sched_barrier(0);
      if (tile + 1 < t_end) {
        if (PAGE16 && (tile + 1 - t_begin) % 64 == 0) load_places(tile + 1);
        load_wide(tile + 1, kn, vn);
      }
    } else {
      __syncthreads();
      // (without branches past the end, where loads in flight would be waited for: the
      // last tile is loaded and stored again, into the buffer that is free)
      store_four(tile + 1, kn, vn);
      load_next(tile + 2);
    }
    const int t0 = seen_tile(seen, tile) * kTile;
    if (!FOUR && t0 + kTile > kv_len) {
      // past the last token the pages hold anything: zero V there (0 * NaN; before the
      // window it is left to the walks, since a barrier per item cost 2 to 4 %)
      for (int c = tid; c < kTile * CH; c += kThreads)
        if (t0 + c / CH >= kv_len) *reinterpret_cast<u32x4*>(vb + c * 16) = u32x4{0u, 0u, 0u, 0u};
      __syncthreads();
    }
    if (!N && walk != kAll) {
      for (int c = tid; c < kTile * CH; c += kThreads) {
        u32x4 x = *reinterpret_cast<const u32x4*>(vb + c * 16);
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = taken<MT>(x[e], walk);
        *reinterpret_cast<u32x4*>(vb + c * 16) = x;
      }
      __syncthreads();
    }
    // (uniform) no row of the wave sees the tile
    if (t0 > lim_hi || (t0 + kTile <= lo_lo && t0 >= A.sinks)) return;

    f32x4 s[kCols][4], from[kCols];  // scores begin at -m, so that they come out as the differences
#pragma unroll
    for (int c = 0; c < kCols; ++c) {
      const float f = m[c] == -INFINITY ? 0.f : -m[c];
      from[c] = f32x4{f, f, f, f};
    }
    // four independent accumulations in turn, here and below: an MFMA waits
    // for the one before it on the same accumulator
#pragma unroll
    for (int b0 = 0; b0 < 4; b0 += 2) {
#pragma unroll
      for (int c = 0; c < kCols; ++c)
#pragma unroll
        for (int b = 0; b < 2; ++b) s[c][b0 + b] = from[c];
#pragma unroll
      for (int ks = 0; ks < NS; ++ks) {
        u32x4 ka[2];
#pragma unroll
        for (int b = 0; b < 2; ++b) ka[b] = *reinterpret_cast<const u32x4*>(kb + kaddr[ks] + (b0 + b) * 16 * RB);
#pragma unroll
        for (int pl = 0; pl < QP; ++pl)
#pragma unroll
          for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int c = 0; c < kCols; ++c) s[c][b0 + b] = mfma32<MT>(ka[b], qb[pl][c][ks], s[c][b0 + b]);
      }
    }
    const bool odd = !N && walk != kAll && walk != kFinite;
    if (odd) {  // ones for what is seen
#pragma unroll
      for (int c = 0; c < kCols; ++c)
#pragma unroll
        for (int blk = 0; blk < 4; ++blk) s[c][blk] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    if (t0 + kTile - 1 > lim_lo || (t0 < lo_hi && t0 + kTile > A.sinks)) {
      const int t1 = t0 + 4 * grp;
#pragma unroll
      for (int c = 0; c < kCols; ++c) {
        const int lo = low(lim[c]);
#pragma unroll
        for (int blk = 0; blk < 4; ++blk)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int t = t1 + blk * 16 + i;
            s[c][blk][i] = t <= lim[c] && (t >= lo || t < A.sinks) ? s[c][blk][i] : -INFINITY;
          }
      }
    }
    float mx[kCols];
    bool rose = false;
#pragma unroll
    for (int c = 0; c < kCols; ++c) {
      float v = -INFINITY;
#pragma unroll
      for (int blk = 0; blk < 4; ++blk)
#pragma unroll
        for (int i = 0; i < 4; ++i) v = fmaxf(v, s[c][blk][i]);
      mx[c] = v;
      rose |= v > (m[c] == -INFINITY ? -INFINITY : lag);
    }
    // the columns' maxima are reduced over their lanes, and the sums and
    // accumulators rescaled, only where some lane saw a score kLag past its
    // maximum
    if (__builtin_amdgcn_ballot_w64(rose) != 0) {
#pragma unroll
      for (int c = 0; c < kCols; ++c) {
        const Rise rise = rise_to(column_max(mx[c]), m[c], sc);
        const float alpha = rise.alpha;
#pragma unroll
        for (int blk = 0; blk < 4; ++blk)
#pragma unroll
          for (int i = 0; i < 4; ++i) s[c][blk][i] -= rise.up;
        l[c] *= alpha;
#pragma unroll
        for (int a = 0; a < NA; ++a)
#pragma unroll
          for (int i = 0; i < 4; ++i) acc[c][a][i] *= alpha;
      }
    }
    u32x4 pb[kCols][2][NP];
    // P^T as the B operand: k = 8*grp + e <-> tokens of blocks 2kc (e < 4) and 2kc+1 (e >= 4)
    auto weights = [&](int c, int blk) __attribute__((always_inline)) {
      float p[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        p[i] = P::weight(s[c][blk][i], sc);
        l[c] += p[i];  // per lane; the column's lanes meet after the last tile
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        uint32_t w[NP];
        P::split(p[2 * i], p[2 * i + 1], w);
#pragma unroll
        for (int pl = 0; pl < NP; ++pl) pb[c][blk / 2][pl][blk % 2 * 2 + i] = w[pl];
      }
    };
    // Two 16-dim blocks of V^T for tokens 32 kc ..
    auto read_v = [&](int step, u32x4 (&va)[2]) __attribute__((always_inline)) {
      const int kc = step / (NA / 2), a0 = step % (NA / 2) * 2;
#pragma unroll
      for (int a = 0; a < 2; ++a) {
        const u32x2 v0 = read_tr(vb + vaddr[a0 + a] + kc * 32 * RB);
        const u32x2 v1 = read_tr(vb + vaddr[a0 + a] + (kc * 32 + 16) * RB);
        va[a] = u32x4{v0[0], v0[1], v1[0], v1[1]};
      }
    };
#pragma unroll
    for (int c = 0; c < kCols; ++c)
#pragma unroll
      for (int blk = 0; blk < 2; ++blk) weights(c, blk);
    u32x4 va[2][2];
    read_v(0, va[0]);
#pragma unroll
    for (int step = 0; step < NA; ++step) {
      const int kc = step / (NA / 2), a0 = step % (NA / 2) * 2;
      if (step + 1 < NA) read_v(step + 1, va[(step + 1) % 2]);
#pragma unroll
      for (int pl = 0; pl < NP; ++pl)
#pragma unroll
        for (int a = 0; a < 2; ++a)
#pragma unroll
          for (int c = 0; c < kCols; ++c) acc[c][a0 + a] = mfma32<MT>(va[step % 2][a], pb[c][kc][pl], acc[c][a0 + a]);
      if (kc == 0) {  // the other half's weights go between the first half's products
#pragma unroll
        for (int i = 0; i < 8 / NA; ++i) weights((step * (8 / NA) + i) / 2, 2 + (step * (8 / NA) + i) % 2);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
  };

  uint32_t who[3][kCols] = {};  // outputs that see each kind of what is not finite
  for (int walk = kAll;; ++walk) {
#pragma unroll
    for (int c = 0; c < kCols; ++c) {
      m[c] = -INFINITY;
      l[c] = 0.f;
#pragma unroll
      for (int a = 0; a < NA; ++a) acc[c][a] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    if (t_begin < t_end) {
      if (PAGE16) load_places(t_begin);
      if constexpr (FOUR) {
        load_four(t_begin);
        store_four(t_begin, s_k0, s_v0);
        load_next(t_begin + 1);
      } else {
        load_wide(t_begin, s_k0, s_v0);
      }
    }
    int tile = t_begin;
    for (; tile + 2 <= t_end; tile += 2) {
      body(tile, s_k0, s_v0, s_k1, s_v1, walk);
      body(tile + 1, s_k1, s_v1, s_k0, s_v0, walk);
    }
    if (tile < t_end) body(tile, s_k0, s_v0, s_k1, s_v1, walk);
    if constexpr (N) {
      const uint32_t least = min(v_least & 0xffffu, v_least >> 16), most = max(v_most & 0xffffu, v_most >> 16);
      if (__syncthreads_or(least < kVLeast || most > kVMost || k_least < kKLeast || k_most > kKMost))
        return false;
      // as the sums of bf16 are held, since a row's other parts may be worked on in it
      constexpr float kDown = Planes<bf16_t>::kScale / P::kScale;
      const float down = __uint_as_float((127u - kShift) << 23) * kDown;
#pragma unroll
      for (int c = 0; c < kCols; ++c) {
        l[c] *= kDown;
#pragma unroll
        for (int a = 0; a < NA; ++a)
#pragma unroll
          for (int i = 0; i < 4; ++i) acc[c][a][i] *= down;
      }
      break;
    }
    if (walk == kAll) {
      bool odd = false;
#pragma unroll
      for (int c = 0; c < kCols; ++c)
#pragma unroll
        for (int a = 0; a < NA; ++a)
#pragma unroll
          for (int i = 0; i < 4; ++i) odd |= acc[c][a][i] != acc[c][a][i];
      if (!__syncthreads_or(odd)) break;
    } else if (walk != kFinite) {
      __syncthreads();
#pragma unroll
      for (int c = 0; c < kCols; ++c) {
        uint32_t bits = 0;
#pragma unroll
        for (int a = 0; a < NA; ++a)
#pragma unroll
          for (int i = 0; i < 4; ++i) bits |= (acc[c][a][i] > 0.f ? 1u : 0u) << (4 * a + i);
        if (walk == kInf) who[0][c] = bits;
        if (walk == kMinusInf) who[1][c] = bits;
        if (walk == kNan) who[2][c] = bits;
      }
    } else {
#pragma unroll
      for (int c = 0; c < kCols; ++c)
#pragma unroll
        for (int a = 0; a < NA; ++a)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint32_t bit = 1u << (4 * a + i);
            if ((who[2][c] | (who[0][c] & who[1][c])) & bit) acc[c][a][i] = NAN;
            else if (who[0][c] & bit) acc[c][a][i] = INFINITY;
            else if (who[1][c] & bit) acc[c][a][i] = -INFINITY;
          }
      break;
    }
  }

  const int slot = uniform(it.slot);
#pragma unroll
  for (int c = 0; c < kCols; ++c) {
    float sum = l[c];
    sum += __shfl_xor(sum, 16);
    sum += __shfl_xor(sum, 32);
    const int row = wrow + c * 16 + lr;
    if (row >= n_rows) continue;
    if (slot >= 0) {
      float* p = A.part + ((int64_t)(slot + it.part) * A.hkv + h) * part_floats(D);
      const int pr = wave * kWaveRows + c * 16 + lr;
#pragma unroll
      for (int a = 0; a < NA; ++a) *reinterpret_cast<f32x4*>(p + pr * D + a * 16 + grp * 4) = acc[c][a];
      if (grp == 0)
        *reinterpret_cast<f32x2*>(p + kRows * D + pr * 2) = f32x2{m[c], sum};
      continue;
    }
    const float inv = sum > 0.f ? 1.f / sum : (sum == 0.f ? 0.f : sum);
    const int pos = row / g;
    T* op = reinterpret_cast<T*>(A.o + (int64_t)(qo_begin + pos) * A.o_st + (int64_t)(h * g + row - pos * g) * A.o_sh) +
            grp * 4;
#pragma unroll
    for (int a = 0; a < NA; ++a)
      *reinterpret_cast<u32x2*>(op + a * 16) = u32x2{pack2<T>(acc[c][a][0] * inv, acc[c][a][1] * inv),
                                                     pack2<T>(acc[c][a][2] * inv, acc[c][a][3] * inv)};
  }
  return true;
}

// The other work over 4 bits for an item that fp16 does not hold.  A function of its own,
// so that its registers are none of the narrow work's: a load of one that was put aside
// waits for the tiles' loads in flight (512 behind 16384, fp16: 226 us with both in one
// body, 180 so; 2048 tokens whose V it takes twice 198, 77 without).
typedef __attribute__((address_space(3))) char* Lds;
template <typename T, int D, bool PAGE16>
__device__ __attribute__((noinline)) void wide_work(const __attribute__((address_space(4))) Args* A, Lds s_k0, Lds s_v0,
                                                    Lds s_k1, Lds s_v1) {
  work<T, true, D, PAGE16, false>(*(const Args*)A, (char*)s_k0, (char*)s_v0, (char*)s_k1, (char*)s_v1);
}

template <typename T, bool FOUR, int D, bool PAGE16>
__global__ __launch_bounds__(kThreads, 2) void prefill_kernel(Args A) {
  __shared__ __align__(16) char s_k0[buffer_bytes(D)];
  __shared__ __align__(16) char s_v0[buffer_bytes(D)];
  __shared__ __align__(16) char s_k1[buffer_bytes(D)];
  __shared__ __align__(16) char s_v1[buffer_bytes(D)];
  constexpr bool kNarrow = FOUR && std::is_same<T, f16_t>::value;
  if (!work<T, FOUR, D, PAGE16, kNarrow>(A, s_k0, s_v0, s_k1, s_v1)) {
    if constexpr (kNarrow)
      wide_work<T, D, PAGE16>((const __attribute__((address_space(4))) Args*)__builtin_amdgcn_kernarg_segment_ptr(), (Lds)s_k0,
                              (Lds)s_v0, (Lds)s_k1, (Lds)s_v1);
  }
}

// D / 4 lanes per row of a split row item, four dims each, its parts in order.
template <typename T, int D>
__global__ __launch_bounds__(kThreads) void merge_kernel(Args A, const Item* merges) {
  constexpr int kLanes = D / 4, kAhead = 4;
  const int h = blockIdx.x % A.hkv;
  const Item it = merges[blockIdx.x / A.hkv];
  const int g = A.hq / A.hkv, qo_begin = uniform(it.qo_begin), n_rows = uniform(it.rows);
  const int pr = blockIdx.y * (kThreads / kLanes) + threadIdx.x / kLanes, d = threadIdx.x % kLanes * 4;
  const int row = uniform(it.row0) + pr;
  if (row >= n_rows) return;
  const int parts = uniform(it.parts);
  const float* p = A.part + ((int64_t)uniform(it.slot) * A.hkv + h) * part_floats(D);
  const int64_t step = (int64_t)A.hkv * part_floats(D);
  float m = -INFINITY, sum = 0.f;
  f32x4 o = f32x4{0.f, 0.f, 0.f, 0.f};
  for (int i0 = 0; i0 < parts; i0 += kAhead) {
    f32x4 v[kAhead];
    f32x2 ml[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const float* q = p + min(i0 + i, parts - 1) * step;
      v[i] = *reinterpret_cast<const f32x4*>(q + pr * D + d);
      ml[i] = *reinterpret_cast<const f32x2*>(q + kRows * D + pr * 2);
    }
    float top = m;
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      if (i0 + i >= parts) ml[i] = f32x2{-INFINITY, 0.f}, v[i] = f32x4{0.f, 0.f, 0.f, 0.f};
      top = fmaxf(top, ml[i][0]);
    }
    const float w = weight(m, top, A.scale_log2);
    sum *= w;
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = weighted(o[e], w);
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const float wi = weight(ml[i][0], top, A.scale_log2);
      sum += ml[i][1] * wi;
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] += weighted(v[i][e], wi);
    }
    m = top;
  }
  const float inv = sum > 0.f ? 1.f / sum : (sum == 0.f ? 0.f : sum);
  const int pos = row / g;
  char* op = A.o + (int64_t)(qo_begin + pos) * A.o_st + (int64_t)(h * g + row - pos * g) * A.o_sh + d * 2;
  *reinterpret_cast<u32x2*>(op) = u32x2{pack2<T>(o[0] * inv, o[1] * inv), pack2<T>(o[2] * inv, o[3] * inv)};
}

// ------------------------------------------------------------ host plan ---
constexpr int kCus = 256;     // two workgroups run on each at a time: the first ones i and i + kCus
constexpr int kMinTiles = 4;  // fewest tiles of a part

template <typename T, bool FOUR, int D> int launch(const Args& a, int num_items, int num_merges, hipStream_t s) {
  const dim3 grid((unsigned)a.hkv * num_items);
  // (16 tokens of a page within 32 bits of each other)
  if (a.page_size % 16 == 0 && a.token_stride < (1 << 27))
    hipLaunchKernelGGL((prefill_kernel<T, FOUR, D, true>), grid, dim3(kThreads), 0, s, a);
  else
    hipLaunchKernelGGL((prefill_kernel<T, FOUR, D, false>), grid, dim3(kThreads), 0, s, a);
  PL_LAUNCH_CHECK("window prefill_kernel");
  if (num_merges > 0) {
    hipLaunchKernelGGL((merge_kernel<T, D>), dim3((unsigned)a.hkv * num_merges, kRows * D / 4 / kThreads), dim3(kThreads), 0, s,
                       a, a.items + num_items);
    PL_LAUNCH_CHECK("window prefill merge_kernel");
  }
  return ok();
}
template <typename T, bool FOUR> int launch_d(const Args& a, int d, int items, int merges, hipStream_t s) {
  return d == 64 ? launch<T, FOUR, 64>(a, items, merges, s) : launch<T, FOUR, 128>(a, items, merges, s);
}

// The first workgroups go round the CUs twice: so that the longest meets the shortest
// of them, the second the second shortest, the second round is turned about.
template <typename I> static void pair_up(std::vector<I>& items, size_t cus) {
  std::reverse(items.begin() + std::min(items.size(), cus), items.begin() + std::min(items.size(), 2 * cus));
}

// When the last of these items ends, in tiles of a workgroup that has a CU for itself
// (1.7 us in fp16, 2.0 .. 2.3 in bf16): two on one are kShared times as fast each (2.7
// and 3.3 us a tile).  (fp16, and bf16 with one plane of P:)
// 512 behind 16384 all in parts of 132, 88, 66, 53, 44 and 33 tiles: 287, 261, 213, 248,
// 224 and 215 us, in 53 and 66, two parts per CU, 194; 2048 whole 62, in parts of up to
// 28 and 16 tiles 58 + 5 and 61 + 10 with the merge.
static double end_of(const std::vector<int>& items, size_t cus) {
  constexpr double kShared = 0.6;
  struct Cu {
    double at;         // when its items' remaining tiles were counted
    double left[2];    // < 0: none
  };
  std::vector<Cu> cu(cus, Cu{0, {-1, -1}});
  auto next = [&](const Cu& c) {  // when its first item ends
    const bool both = c.left[0] >= 0 && c.left[1] >= 0;
    const double first = both ? std::min(c.left[0], c.left[1]) / kShared : std::max(c.left[0], c.left[1]);
    return c.at + first;
  };
  size_t i = 0;
  for (int round = 0; round < 2; ++round)
    for (size_t c = 0; c < cus && i < items.size(); ++c) cu[c].left[round] = items[i++];
  using Event = std::pair<double, size_t>;
  std::vector<Event> heap;
  const auto later = std::greater<Event>();
  for (size_t c = 0; c < cus; ++c)
    if (cu[c].left[0] >= 0) heap.push_back(Event{next(cu[c]), c});
  std::make_heap(heap.begin(), heap.end(), later);
  double end = 0;
  while (!heap.empty()) {
    std::pop_heap(heap.begin(), heap.end(), later);
    const Event e = heap.back();
    heap.pop_back();
    Cu& c = cu[e.second];
    end = e.first;
    const bool both = c.left[0] >= 0 && c.left[1] >= 0;
    const int done = both ? c.left[1] < c.left[0] : c.left[1] >= 0;
    if (both) c.left[1 - done] -= (e.first - c.at) * kShared;
    if (both && c.left[1 - done] < 0) c.left[1 - done] = 0;
    c.at = e.first;
    c.left[done] = i < items.size() ? items[i++] : -1;
    if (c.left[0] >= 0 || c.left[1] >= 0) {
      heap.push_back(Event{next(c), e.second});
      std::push_heap(heap.begin(), heap.end(), later);
    }
  }
  return end;
}

// Into how many parts each row item is cut: of the numbers of parts in all that are
// tried, dealt out so that the longest part is as short as can be, the one whose last
// part of a head ends first.  An item costs kStart tiles beside its own, a part one
// more, and the merge kMerge and what the parts' 66 KiB each take.  (In tiles of ~2 us.)
static std::vector<int> parts_of(const std::vector<int>& lengths, int hkv) {
  constexpr int kStart = 2, kMerge = 2, kPartsPerTile = 200;
  constexpr size_t kMost = 4096;  // items past which no cut is needed to fill the chip
  std::vector<int> parts(lengths.size(), 1), best = parts;
  if (lengths.empty() || lengths.size() * hkv > kMost) return best;
  const size_t cus = std::max(1, kCus / hkv);
  double least = -1;
  std::vector<int> items;
  // the longest part first
  using Part = std::pair<int, size_t>;
  std::vector<Part> heap;
  for (size_t i = 0; i < lengths.size(); ++i) heap.push_back(Part{lengths[i], i});
  std::make_heap(heap.begin(), heap.end());
  size_t all = lengths.size();
  for (size_t half = 0; half <= 16; ++half) {  // no cut, then half a part per CU and on
    const size_t want = half * cus / 2;
    if (half > 0 && (want <= all || want * hkv > kMost)) continue;
    while (all < want) {
      const Part top = heap.front();
      if (lengths[top.second] < (parts[top.second] + 1) * kMinTiles) break;
      std::pop_heap(heap.begin(), heap.end());
      ++parts[top.second];
      heap.back().first = (lengths[top.second] + parts[top.second] - 1) / parts[top.second];
      std::push_heap(heap.begin(), heap.end());
      ++all;
    }
    items.clear();
    int64_t cut = 0;
    for (size_t i = 0; i < lengths.size(); ++i) {
      const int t = lengths[i], n = parts[i];
      if (n > 1) cut += n;
      for (int j = 0; j < n; ++j)
        items.push_back((int)((int64_t)t * (j + 1) / n - (int64_t)t * j / n) + kStart + (n > 1 ? 1 : 0));
    }
    std::sort(items.begin(), items.end(), std::greater<int>());
    pair_up(items, cus);
    const double end = end_of(items, cus) + (cut > 0 ? kMerge + (double)cut * hkv / kPartsPerTile : 0.0);
    if (least < 0 || end < least) {
      least = end;
      best = parts;
    }
  }
  return best;
}

// The records of a plan; entry points catch what vectors throw.
static int make_plan(const int32_t* qo, const int32_t* kv, const int32_t* kv_last, int batch, int hq, int hkv,
                     int page_size, int window, int sinks, std::vector<Item>& items, std::vector<Item>& merges,
                     int& slots) {
  const int g = hq / hkv;
  std::vector<Item> list;  // row items, whole
  std::vector<int> lengths;
  for (int r = 0; r < batch; ++r) {
    const int64_t qo_len = (int64_t)qo[r + 1] - qo[r], pages = (int64_t)kv[r + 1] - kv[r];
    if (qo_len < 0) return fail(PL_ERR_INVALID, "qo_indptr_h must be non-decreasing (row %d)", r);
    if (pages < 0) return fail(PL_ERR_INVALID, "kv_indptr_h must be non-decreasing (row %d)", r);
    if (pages > 0 && (kv_last[r] < 1 || kv_last[r] > page_size))
      return fail(PL_ERR_INVALID, "last_page_len[%d] = %d outside [1, %d]", r, kv_last[r], page_size);
    const int64_t kv_len = pages > 0 ? (pages - 1) * page_size + kv_last[r] : 0;
    if (kv_len > kMaxLen) return fail(PL_ERR_INVALID, "row %d: kv_len %lld too large", r, (long long)kv_len);
    if (qo_len > kv_len)
      return fail(PL_ERR_INVALID, "row %d: %lld queries exceed its %lld tokens", r, (long long)qo_len,
                  (long long)kv_len);
    const int64_t rows = qo_len * g;
    if (rows > INT32_MAX / 2) return fail(PL_ERR_INVALID, "row %d: %lld query rows too many", r, (long long)rows);
    for (int64_t r0 = 0; r0 < rows; r0 += kRows) {
      const int64_t last_row = std::min<int64_t>(r0 + kRows, rows) - 1;
      const Seen s = seen_from((int)(kv_len - qo_len + r0 / g), window, sinks, kTile);
      const int tiles = s.ns + (int)((kv_len - qo_len + last_row / g) / kTile) + 1 - s.fw;
      Item it{};
      it.request = r;
      it.row0 = (int32_t)r0;
      it.rows = (int32_t)rows;
      it.qo_begin = qo[r];
      it.kv_len = (int32_t)kv_len;
      it.page_begin = kv[r];
      it.tile_end = tiles;
      it.slot = -1;
      it.parts = 1;
      list.push_back(it);
      lengths.push_back(tiles);
    }
  }
  if (list.size() > (size_t)INT32_MAX / 64) return fail(PL_ERR_INVALID, "too many prefill work items");
  const std::vector<int> cuts = parts_of(lengths, hkv);
  for (size_t i = 0; i < list.size(); ++i) {
    const int tiles = list[i].tile_end, parts = cuts[i];
    Item it = list[i];
    it.parts = parts;
    it.slot = parts > 1 ? slots : -1;
    for (it.part = 0; it.part < parts; ++it.part) {
      it.tile_begin = (int32_t)((int64_t)tiles * it.part / parts);
      it.tile_end = (int32_t)((int64_t)tiles * (it.part + 1) / parts);
      items.push_back(it);
    }
    if (parts > 1) {
      it.part = it.tile_begin = it.tile_end = 0;
      merges.push_back(it);
      slots += parts;
    }
  }
  // longest first; items of one length by request and kv range, so that the row
  // items sharing a range run side by side
  std::stable_sort(items.begin(), items.end(), [](const Item& a, const Item& b) {
    const int la = a.tile_end - a.tile_begin, lb = b.tile_end - b.tile_begin;
    if (la != lb) return la > lb;
    if (a.request != b.request) return a.request < b.request;
    return a.tile_begin < b.tile_begin;
  });
  pair_up(items, std::max(1, kCus / hkv));
  return PL_OK;
}

}  // namespace pre
}  // namespace window
}  // namespace pl

using namespace pl;
using namespace pl::window;
using namespace pl::window::pre;

extern "C" int pl_window_prefill_plan(const int32_t* qo_indptr_h, const int32_t* kv_indptr_h,
                                      const int32_t* kv_last_page_len_h, int batch, int num_qo_heads,
                                      int num_kv_heads, int head_dim, int page_size, int window, int sinks,
                                      int32_t* items_h, int max_records, int* num_items_h, int* num_merges_h,
                                      size_t* workspace_bytes_h) {
  if (!num_items_h || !num_merges_h || !workspace_bytes_h)
    return fail(PL_ERR_INVALID, "num_items_h, num_merges_h and workspace_bytes_h must not be null");
  *num_items_h = *num_merges_h = 0;
  *workspace_bytes_h = 0;
  if (batch < 0) return fail(PL_ERR_INVALID, "batch must be >= 0");
  if (batch > 0 && (!qo_indptr_h || !kv_indptr_h || !kv_last_page_len_h))
    return fail(PL_ERR_INVALID, "null table pointer");
  if (num_kv_heads <= 0 || num_qo_heads <= 0 || num_qo_heads % num_kv_heads)
    return fail(PL_ERR_INVALID, "num_qo_heads (%d) must be a multiple of num_kv_heads (%d)", num_qo_heads,
                num_kv_heads);
  if (head_dim != 64 && head_dim != 128)
    return fail(PL_ERR_UNSUPPORTED, "head_dim must be 64 or 128 (got %d)", head_dim);
  if (page_size <= 0) return fail(PL_ERR_INVALID, "page_size must be positive (got %d)", page_size);
  if (window < 0 || sinks < 0) return fail(PL_ERR_INVALID, "window and sinks must be >= 0");
  if (batch > 0 && (qo_indptr_h[0] != 0 || kv_indptr_h[0] != 0))
    return fail(PL_ERR_INVALID, "qo_indptr_h[0] and kv_indptr_h[0] must be 0");
  try {
    std::vector<Item> items, merges;
    int slots = 0;
    if (int e = make_plan(qo_indptr_h, kv_indptr_h, kv_last_page_len_h, batch, num_qo_heads, num_kv_heads, page_size,
                          window, sinks, items, merges, slots))
      return e;
    *num_items_h = (int)items.size();
    *num_merges_h = (int)merges.size();
    *workspace_bytes_h = (size_t)slots * num_kv_heads * part_floats(head_dim) * sizeof(float);
    if (items_h == nullptr) return ok();
    if (items.size() + merges.size() > (size_t)std::max(max_records, 0))
      return fail(PL_ERR_WORKSPACE, "%zu prefill plan records exceed the %d provided", items.size() + merges.size(),
                  max_records);
    std::copy(items.begin(), items.end(), reinterpret_cast<Item*>(items_h));
    std::copy(merges.begin(), merges.end(), reinterpret_cast<Item*>(items_h) + items.size());
    return ok();
  } catch (const std::exception&) {
    return fail(PL_ERR_INVALID, "no host memory for the prefill plan");
  }
}

extern "C" int pl_window_prefill_run(const void* q, int64_t q_stride_t, int64_t q_stride_h, const void* k_cache,
                                     const void* v_cache, int64_t page_stride, int64_t token_stride,
                                     int64_t head_stride, int64_t num_pages, int kv_bits, const int32_t* kv_indices,
                                     const int32_t* items, int num_items, int num_merges, void* o, int64_t o_stride_t,
                                     int64_t o_stride_h, int num_qo_heads, int num_kv_heads, int head_dim,
                                     int page_size, int window, int sinks, float sm_scale, int dtype, void* workspace,
                                     size_t workspace_bytes, size_t plan_workspace_bytes, void* stream) {
  if (num_items < 0 || num_merges < 0) return fail(PL_ERR_INVALID, "num_items and num_merges must be >= 0");
  if (num_kv_heads <= 0 || num_qo_heads <= 0 || num_qo_heads % num_kv_heads)
    return fail(PL_ERR_INVALID, "num_qo_heads (%d) must be a multiple of num_kv_heads (%d)", num_qo_heads,
                num_kv_heads);
  if (head_dim != 64 && head_dim != 128)
    return fail(PL_ERR_UNSUPPORTED, "head_dim must be 64 or 128 (got %d)", head_dim);
  if (dtype != PL_DTYPE_BF16 && dtype != PL_DTYPE_F16)
    return fail(PL_ERR_UNSUPPORTED, "dtype must be F16 or BF16 (got %d)", dtype);
  if (kv_bits != 16 && kv_bits != 4) return fail(PL_ERR_UNSUPPORTED, "kv_bits must be 16 or 4 (got %d)", kv_bits);
  if (page_size <= 0 || num_pages <= 0) return fail(PL_ERR_INVALID, "page_size and num_pages must be positive");
  if (kv_bits == 4 && (page_size % 8 || page_size > (1 << 20)))
    return fail(PL_ERR_INVALID, "pages of a 4-bit cache hold a multiple of 8 tokens, up to 2^20 (got %d)", page_size);
  if (window < 0 || sinks < 0) return fail(PL_ERR_INVALID, "window and sinks must be >= 0");
  if (num_items == 0) return ok();
  if (!q || !k_cache || !v_cache || !kv_indices || !items || !o)
    return fail(PL_ERR_INVALID, "null pointer argument");
  const int eb = kv_bits == 4 ? 1 : 2;  // a 4-bit cache's strides are bytes
  const int64_t strides[] = {q_stride_t * 2, q_stride_h * 2, o_stride_t * 2, o_stride_h * 2, page_stride * eb,
                             kv_bits == 4 ? 0 : token_stride * eb, head_stride * eb};
  for (int64_t st : strides)
    if (st % 16) return fail(PL_ERR_INVALID, "strides must be multiples of 16 bytes");
  const void* ptrs[] = {q, k_cache, v_cache, o, workspace};
  for (const void* p : ptrs)
    if ((uintptr_t)p % 16) return fail(PL_ERR_INVALID, "q, o, the caches and workspace must be 16-byte aligned");
  if ((uintptr_t)items % 64) return fail(PL_ERR_INVALID, "the plan's records must be 64-byte aligned");
  if ((int64_t)std::max(num_items, num_merges) * num_kv_heads >= kMaxGroups)
    return fail(PL_ERR_INVALID, "grid of %d items x %d heads too large", num_items, num_kv_heads);
  if (num_merges > 0 && (!workspace || workspace_bytes < plan_workspace_bytes))
    return fail(PL_ERR_WORKSPACE, "prefill workspace of %zu bytes < %zu needed", workspace_bytes,
                plan_workspace_bytes);
  Args a{};
  a.q = (const char*)q;
  a.k = (const char*)k_cache;
  a.v = (const char*)v_cache;
  a.o = (char*)o;
  a.part = (float*)workspace;
  a.kv_indices = kv_indices;
  a.items = reinterpret_cast<const Item*>(items);
  a.q_st = strides[0];
  a.q_sh = strides[1];
  a.o_st = strides[2];
  a.o_sh = strides[3];
  a.page_stride = strides[4];
  a.token_stride = strides[5];
  a.head_stride = strides[6];
  a.num_pages = num_pages;
  a.hq = num_qo_heads;
  a.hkv = num_kv_heads;
  a.page_size = page_size;
  a.page_shift = (page_size & (page_size - 1)) == 0 ? __builtin_ctz(page_size) : -1;
  a.window = window;
  a.sinks = sinks;
  // maxima are taken before scaling: a positive scale (a zero one as one far below
  // any score's rounding), the sign moved into q
  const float s2 = sm_scale * 1.44269504088896340736f;
  a.scale_log2 = std::max(s2 < 0 ? -s2 : s2, 1e-30f);
  a.q_flip = s2 < 0 ? 0x80008000u : 0u;
  const hipStream_t st = (hipStream_t)stream;
  if (dtype == PL_DTYPE_BF16)
    return kv_bits == 4 ? launch_d<bf16_t, true>(a, head_dim, num_items, num_merges, st)
                        : launch_d<bf16_t, false>(a, head_dim, num_items, num_merges, st);
  return kv_bits == 4 ? launch_d<f16_t, true>(a, head_dim, num_items, num_merges, st)
                      : launch_d<f16_t, false>(a, head_dim, num_items, num_merges, st);
}
