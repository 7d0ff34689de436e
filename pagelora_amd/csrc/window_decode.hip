// Decode attention of one query per request over a paged KV cache of 16 or of 4
// bits per value, under a sliding window with sinks (gfx950).
//
// The query of a request of n tokens is at position p = n - 1 and sees
// t > p - window (window 0: every t) and t < sinks:
//   o = sum_t p_t v_t / sum_t p_t,  p_t = exp(s q . k_t).
// A request of no tokens gets o = 0 and lse = -inf.
//
// plan_kernel (once per step, for all layers) cuts what the requests see, tiles of
// 32 tokens, into items of about equal length.  A workgroup takes an item of one kv
// head for up to 16 heads of its group; its four waves take a quarter of the tiles
// each, and their states meet in LDS.  merge_kernel joins the items of a request
// in order.
//
// A wave holds its operands in registers: S^T = K Q^T has a query per lane column
// and four tokens per lane, which are the B operand of O^T += V^T P^T as they lie; of
// V^T, whose lanes hold eight tokens of one dim, a lane loads D / 16 dims of those
// tokens and pairs tokens by byte permutes.  Values of 4 bits become bf16 on the way
// (exact, two per instruction), so that a 4-bit cache is always multiplied in bf16;
// queries of fp16 go in as two planes (exact).
//
// An output that is NaN is looked at again: 0 times an infinity, or the difference of
// two planes' infinities, is not what the row sees.  The wave's tiles are walked once
// more with infinities and NaN taken out of V, and once with nothing but them, each
// with weight 1, added to the sums.
//
// Measured (head_dim 128; us of a pass, decode_kernel and merge_kernel, of which the
// second 3.8 .. 8):
//   64 x 4096 .. 16384, 4 bits, GQA 4   137, 5.2 TB/s, issue in 98 % of the cycles; the
//                                       same loads with next to no arithmetic 118 + 7.
//                                       131 with two planes of P for three; with two,
//                                       the kernel 289 where a tile's loads waited for
//                                       its page ids (128), and three tiles in flight
//                                       no faster than two
//   1 x 131072, 4 bits, GQA 4           35, 4.1 TB/s: ~6 us of start (record, page ids,
//                                       first tiles), 24 of stream, 5 of the merge
//   64 x 1028 of 8192, 16 bits, GQA 4   53.4, 5.1 TB/s; pages of one token 56
//   1 x 4112 of 32768, 16 bits, MHA     22.2: two tiles per wave, start and end
//   23 ragged under 1000, 4 bits, GQA 7  14.1, 1 x 2048, 4 bits  12.1 (6 + 4 in the
//                                       kernels): dependent round trips, two launches
// Heads fastest in the grid, so that a page's heads are read together, lost as much
// (16 bits 52 -> 56 us) as it won (head_dim 64, 16 bits 44 -> 36).
#include <algorithm>

#include "window_common.h"

namespace pl {
namespace window {
namespace dec {

constexpr int kWaves = 4;
constexpr int kThreads = kWave * kWaves;
constexpr int kTile = 32;          // tokens of a step of a wave
constexpr int kPlanThreads = 1024;
constexpr int kMagic = 0x57444543;
constexpr int kMinTiles = 4;       // fewest tiles of an item that is cut: one per wave

// What a plan was made for, then what it holds.
struct alignas(64) Header {
  int32_t magic, batch, page_size, window, sinks, indices_capacity, max_items, num_items;
  int32_t pad[8];
};
static_assert(sizeof(Header) == 64, "the plan's header");
struct Item {
  int32_t row, kv_len, page_begin, tile_begin, tile_end, slot, parts, pad;
};
static_assert(sizeof(Item) == 32, "the plan's record");
struct Row {
  int32_t first, parts, slot;  // its items, and where their parts lie if it is cut
};

struct Layout {
  size_t items, rows, indices, bytes;
};
inline Layout layout(int batch, int indices_capacity, int max_items) {
  Layout l;
  l.items = sizeof(Header);
  l.rows = l.items + sizeof(Item) * (size_t)max_items;
  l.indices = align_up(l.rows + sizeof(Row) * (size_t)batch, 64);
  l.bytes = align_up(l.indices + sizeof(int32_t) * (size_t)indices_capacity, 64);
  return l;
}

// Heads of a workgroup: a kv head's group in blocks of 16.
inline int head_blocks(int hq, int hkv) { return (hq / hkv + 15) / 16; }
// Items per kv head and head block that the work is cut into: as many as fill the
// chip with workgroups twice per CU, more where an item then still has kItemTiles, up
// to four times as many.  us (two planes of P), at 512 / 768 / 1024 / 1536 / 2048 workgroups: 64 x 4096
// .. 16384 tokens of 4 bits 156 / 151 / 141 / 135 / 133, 1 x 131072 39 / 35 / 38 / 41 /
// 46, 64 x 1028 of 16 bits (whole rows at 512) 55 / 62 / 62 / 59 / 74.
constexpr int kItemTiles = 42;
__host__ __device__ inline int target_items(int64_t tiles, int heads) {
  const int64_t least = 512 / heads > 1 ? 512 / heads : 1, most = 2048 / heads > 1 ? 2048 / heads : 1;
  const int64_t n = tiles / kItemTiles;
  return (int)(n < least ? least : n > most ? most : n);
}
// At most so many items: every request's last may be short.
inline int max_items_of(int batch, int hq, int hkv, int page_size, int window, int sinks, int indices_capacity) {
  int64_t tiles = (int64_t)indices_capacity * page_size / kTile + batch;
  if (window > 0) tiles = std::min(tiles, batch * (((int64_t)window + sinks) / kTile + 4));
  const int64_t cut = std::min((int64_t)target_items(tiles, hkv * head_blocks(hq, hkv)), tiles / kMinTiles + 1);
  return batch + (int)cut;
}

// Parts of the rows that are cut: a row of n > 1 parts has more than n - 1 chunks of
// tiles, n / 2 or more, and all rows together no more chunks than the work is cut into.
// (A part for every row's item took 1.1 GB for 4096 rows of 32 kv heads, so 34 MB.)
__host__ __device__ inline int max_slots_of(int batch, int max_items) {
  const int cut = max_items - batch;
  return 2 * cut < max_items ? 2 * cut : max_items;
}

// ------------------------------------------------------------------- plan ---
struct PlanArgs {
  const int32_t *indptr, *indices, *last;
  Header want;
  Header* header;
  Item* items;
  Row* rows;
  int32_t* ids;
  int heads;  // kv heads times head blocks
};

struct Request {
  int page_begin, len, tiles;
};
// Request r, its tables brought into their ranges.
__device__ __forceinline__ Request read_request(const PlanArgs& A, int r) {
  Request q;
  const int cap = A.want.indices_capacity;
  q.page_begin = min(max(A.indptr[r], 0), cap);
  const int pages = min(max(A.indptr[r + 1], q.page_begin), cap) - q.page_begin;
  const int last = min(max(A.last[r], 1), A.want.page_size);
  const int64_t len = pages > 0 ? (int64_t)(pages - 1) * A.want.page_size + last : 0;
  q.len = (int)min(len, (int64_t)kMaxLen);
  const Seen s = seen_from(q.len - 1, A.want.window, A.want.sinks, kTile);
  q.tiles = s.ns + (q.len + kTile - 1) / kTile - s.fw;
  return q;
}

// Workgroup 0 cuts the work; the others copy the page ids.
__global__ __launch_bounds__(kPlanThreads) void plan_kernel(PlanArgs A) {
  const int tid = threadIdx.x, batch = A.want.batch;
  if (blockIdx.x > 0) {
    const int64_t step = (int64_t)(gridDim.x - 1) * kPlanThreads;
    for (int64_t i = (int64_t)(blockIdx.x - 1) * kPlanThreads + tid; i < A.want.indices_capacity; i += step)
      A.ids[i] = A.indices[i];
    return;
  }
  __shared__ int64_t s_sum[kPlanThreads / kWave];
  __shared__ int64_t s_scan[kPlanThreads / kWave];
  const int lane = tid % kWave, wave = tid / kWave;
  int64_t sum = 0;
  for (int r = tid; r < batch; r += kPlanThreads) sum += read_request(A, r).tiles;
  for (int d = 1; d < kWave; d <<= 1) sum += __shfl_xor(sum, d);
  if (lane == 0) s_sum[wave] = sum;
  __syncthreads();
  int64_t total = 0;
  for (int w = 0; w < kPlanThreads / kWave; ++w) total += s_sum[w];
  // (tables that overlap hold more than any that do not: no more items than there is room for)
  const int target = min(target_items(total, A.heads), A.want.max_items - batch);
  const int chunk = (int)max((total + target - 1) / target, (int64_t)kMinTiles);
  int64_t base = 0;  // items before, and the parts among them in the upper half
  for (int r0 = 0; r0 < batch; r0 += kPlanThreads) {
    const int r = r0 + tid;
    const int n = r < batch ? max(1, (read_request(A, r).tiles + chunk - 1) / chunk) : 0;
    const int64_t own = n | (int64_t)(n > 1 ? n : 0) << 32;
    int64_t incl = own;
    for (int d = 1; d < kWave; d <<= 1) {
      const int64_t up = __shfl_up(incl, d);
      incl += lane >= d ? up : 0;
    }
    __syncthreads();
    if (lane == kWave - 1) s_scan[wave] = incl;
    __syncthreads();
    int64_t before = base;
    for (int w = 0; w < kPlanThreads / kWave; ++w) {
      before += w < wave ? s_scan[w] : 0;
      base += s_scan[w];
    }
    if (r < batch) A.rows[r] = Row{(int)(before + incl - own), n, (int)((before + incl - own) >> 32)};
  }
  __syncthreads();
  const int num = min((int)base, A.want.max_items);
  for (int i = tid; i < num; i += kPlanThreads) {
    int lo = 0, hi = batch;  // the row that holds item i: the last whose first item is <= i
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (A.rows[mid].first <= i) lo = mid; else hi = mid;
    }
    const Row row = A.rows[lo];
    const Request q = read_request(A, lo);
    const int part = i - row.first;
    A.items[i] = Item{lo, q.len, q.page_begin, (int)((int64_t)q.tiles * part / row.parts),
                      (int)((int64_t)q.tiles * (part + 1) / row.parts), row.slot + part, row.parts, 0};
  }
  if (tid == 0) {
    Header h = A.want;
    h.num_items = num;
    *A.header = h;
  }
}

// ----------------------------------------------------------------- decode ---
struct Args {
  const char *q, *k, *v;
  char* o;
  float *lse, *part;
  const Header* header;
  const Item* items;
  const Row* rows;
  const int32_t* ids;
  Header want;
  int64_t q_sb, q_sh, o_sb, o_sh;                        // bytes
  int64_t page_stride, token_stride, head_stride, num_pages;  // bytes, bytes, bytes (a 4-bit cache has no token stride)
  int hq, hkv, blocks, page_shift;                       // page_shift: -1 where page_size is no power of two
  float scale_log2;  // > 0; a negative scale negates q instead
  uint32_t q_flip;
};

// Floats of a part: outputs [16][D], then (m, sum) per head.
template <int D> constexpr int part_floats() { return 16 * (D + 2); }

__device__ __forceinline__ bool stale(const Header& h, const Header& want) {
  return h.magic != want.magic || h.batch != want.batch || h.page_size != want.page_size || h.window != want.window ||
         h.sinks != want.sinks || h.indices_capacity != want.indices_capacity || h.max_items != want.max_items;
}

// ln of sum 2^(m sc - shift); -inf where nothing was seen.
__device__ __forceinline__ float log_sum(float m, float sc, float sum, float shift) {
  return sum > 0.f ? __builtin_fmaf(m, sc, log2f(sum) - shift) * 0.69314718055994531f : (sum == 0.f ? -INFINITY : sum);
}

template <typename T, bool FOUR, int D, bool PAGE16>
__global__ __launch_bounds__(kThreads, FOUR ? 3 : 2) void decode_kernel(Args A) {
  using MT = typename std::conditional<FOUR, bf16_t, T>::type;  // what is multiplied
  using P = Planes<MT>;
  constexpr bool kBf16 = std::is_same<MT, bf16_t>::value;
  constexpr int NS = D / 32;                                    // products of a score
  constexpr int NA = D / 16;                                    // dims of a lane in V
  constexpr int ND = D / 32;                                    // words of them
  constexpr int QP = FOUR && std::is_same<T, f16_t>::value ? 2 : 1;  // planes of q
  constexpr int KW = FOUR ? D / 32 : D / 8;                     // words of a lane's K per block of 16 tokens
  constexpr int VW = FOUR ? 4 : 4 * ND;                         // words of a lane's V per block
  __shared__ __align__(16) float s_o[kWaves][16][D];
  __shared__ float s_m[kWaves][16], s_l[kWaves][16];

  const Header head = *A.header;
  const Item it = A.items[blockIdx.x];
  if (stale(head, A.want) || blockIdx.x >= (unsigned)head.num_items) return;
  const int row = uniform(it.row), len = uniform(it.kv_len), pb = uniform(it.page_begin);
  if (row < 0 || row >= A.want.batch) return;
  const int h = blockIdx.y / A.blocks, hb = blockIdx.y % A.blocks;
  const int g = A.hq / A.hkv, rows = min(g - hb * 16, 16);
  const int lane = threadIdx.x % kWave, wave = uniform(threadIdx.x / kWave);
  const int lr = lane % 16, grp = lane / 16;
  const Seen seen = seen_from(len - 1, A.want.window, A.want.sinks, kTile);
  const int ps = A.want.page_size;
  const int32_t* ids = A.ids + pb;
  const int cap = A.want.indices_capacity - pb;

  // q as the B operand: 4-bit K's lanes hold D / 4 dims in a row, 16-bit K's
  // eight of every 32
  u32x4 qb[QP][NS];
  {
    const int head_q = h * g + hb * 16 + min(lr, rows - 1);  // columns past the heads repeat the last one
    const char* qp = A.q + (int64_t)row * A.q_sb + (int64_t)head_q * A.q_sh + (FOUR ? grp * (D / 2) : grp * 16);
#pragma unroll
    for (int ks = 0; ks < NS; ++ks) {
      u32x4 w = *reinterpret_cast<const u32x4*>(qp + ks * (FOUR ? 16 : 64));
#pragma unroll
      for (int e = 0; e < 4; ++e) w[e] ^= A.q_flip;
      if constexpr (QP == 2) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float a, b;
          unpack2<f16_t>(w[e], a, b);
          const uint32_t hi = f32x2_to_bf16x2_bits(a, b);
          // (the rest of an infinity is none)
          const float ra = a - bf16_lo(hi), rb = b - bf16_hi(hi);
          qb[0][ks][e] = hi;
          qb[QP - 1][ks][e] = f32x2_to_bf16x2_bits(ra == ra ? ra : 0.f, rb == rb ? rb : 0.f);
        }
      } else {
        qb[0][ks] = w;
      }
    }
  }

  auto page_of = [&](int t) { return A.page_shift >= 0 ? t >> A.page_shift : t / ps; };
  auto id_of = [&](int page) { return ids[min(page, cap - 1)]; };
  auto page_at = [&](int id) -> int64_t {
    return (id < 0 ? 0 : ((int64_t)id >= A.num_pages ? A.num_pages - 1 : (int64_t)id)) * A.page_stride;
  };
  const int top = len - 1;  // addresses past the sequence repeat its end's
  const int n_tiles = it.tile_end - it.tile_begin;
  const int begin = uniform(it.tile_begin + (int)((int64_t)n_tiles * wave / kWaves));
  const int end = uniform(it.tile_begin + (int)((int64_t)n_tiles * (wave + 1) / kWaves));
  const int64_t unit = FOUR ? (int64_t)(D / 2) : A.token_stride;
  // Pages of 16 tokens and more: lane l holds where block l % 2 of tile l / 2 of the
  // next 32 begins, so that no tile's loads wait for its page ids.
  int64_t places = 0;
  auto load_places = [&](int i) {
    const int tb = min(seen_tile(seen, min(i + lane / 2, end - 1)) * kTile + lane % 2 * 16, top & ~15);
    const int page = page_of(tb);
    places = page_at(id_of(page)) + (int64_t)(tb - page * ps) * unit;
  };
  auto place = [&](int i, int b) -> int64_t {
    const int l = (i - begin) % 32 * 2 + b;
    return (int64_t)((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(places >> 32), l) << 32 |
                     (uint32_t)__builtin_amdgcn_readlane((int)places, l));
  };

  // Other pages: lane l holds where token l % 32 of the next tile lies; its page id is
  // loaded a tile ahead.
  int id_next = 0, slot_next = 0;
  auto ask = [&](int i) {
    const int t = min(seen_tile(seen, i) * kTile + lane % 32, top), page = page_of(t);
    slot_next = t - page * ps;
    id_next = id_of(page);
  };
  auto from_lane = [&](int64_t x, int l) -> int64_t {
    return (int64_t)((uint64_t)(uint32_t)__shfl((int)(x >> 32), l) << 32 | (uint32_t)__shfl((int)x, l));
  };

  struct Raw {
    uint32_t k[2][KW], v[2][VW], ks[2], vs[2];
  };
  const char* kh = A.k + (int64_t)h * A.head_stride;
  const char* vh = A.v + (int64_t)h * A.head_stride;
  // the dims' place of a lane in a 4-bit V's codes, and its scale group
  const int vchunk = D == 64 ? (lr / 2) * 16 : lr * (D / 8), vgroup = lr * NA / kGroup;

  auto load_words = [](const char* p, uint32_t* w, auto count) {
    constexpr int N = decltype(count)::value;
    if constexpr (N == 2) {
      const u32x2 x = __builtin_nontemporal_load(reinterpret_cast<const u32x2*>(p));
      w[0] = x[0];
      w[1] = x[1];
    } else {
#pragma unroll
      for (int i = 0; i < N; i += 4) {
        const u32x4 x = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(p) + i / 4);
#pragma unroll
        for (int j = 0; j < 4; ++j) w[i + j] = x[j];
      }
    }
  };
  // the lane's own part of the addresses in a block: K, V, their scales
  const uint32_t k_own = FOUR ? lr * (D / 2) + grp * (D / 8) : grp * 16, v_own = FOUR ? grp * (2 * D) + vchunk : lr * (2 * NA);
  const uint32_t ks_own = lr * (D / 32) + grp * (D / 4) / kGroup, vs_own = grp * (D / 8) + vgroup * 4;
  auto fetch = [&](int i, Raw& raw) {
    const int t0 = seen_tile(seen, i) * kTile;
    int codes = 0;  // of the lane's token: its codes' bytes in the page
    if constexpr (PAGE16) {
      if ((i - begin) % 32 == 0) load_places(i);
    } else {
      places = page_at(id_next) + slot_next * unit;
      codes = slot_next * (D / 2);
      ask(min(i + 1, end - 1));
    }
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      // a block's first token, or where it is past the end the last block's
      const int tb = min(t0 + 16 * b, top & ~15);
      if constexpr (PAGE16) {
        const int64_t at = place(i, b);
        if constexpr (FOUR) {
          const int slot = A.page_shift >= 0 ? tb & (ps - 1) : tb % ps;
          // scales: from the codes' end, D / 32 bytes a token (codes D / 2)
          const int64_t sat = at + ps * (D / 2) - slot * (D / 2 - D / 32);
          load_words((kh + at) + k_own, raw.k[b], std::integral_constant<int, KW>{});
          raw.ks[b] = *reinterpret_cast<const uint8_t*>((kh + sat) + ks_own);
          load_words((vh + at) + v_own, raw.v[b], std::integral_constant<int, VW>{});
          raw.vs[b] = *reinterpret_cast<const uint32_t*>((vh + sat) + vs_own);
        } else {
          const char* kp = kh + at + ((int64_t)lr * A.token_stride + k_own);
#pragma unroll
          for (int ks = 0; ks < NS; ++ks) load_words(kp + ks * 64, raw.k[b] + 4 * ks, std::integral_constant<int, 4>{});
          const char* vp = vh + at + ((int64_t)(4 * grp) * A.token_stride + v_own);
#pragma unroll
          for (int j = 0; j < 4; ++j)
            load_words(vp + j * A.token_stride, raw.v[b] + j * ND, std::integral_constant<int, ND>{});
        }
      } else {
        // (tokens past the end are its last one)
        if constexpr (FOUR) {
          const int kl = 16 * b + lr, vl = 16 * b + 4 * grp;
          const char* kp = kh + from_lane(places, kl);
          load_words(kp + grp * (D / 8), raw.k[b], std::integral_constant<int, KW>{});
          // scales: from the codes' end, D / 32 bytes a token (codes D / 2)
          raw.ks[b] = *reinterpret_cast<const uint8_t*>(kp + ps * (D / 2) - __shfl(codes, kl) / 16 * 15 + grp * (D / 4) / kGroup);
          // V's codes go by four tokens: the last one may be within them
          const int rest = __shfl(codes, vl) % (2 * D);
          const char* vp = vh + from_lane(places, vl) - rest;
          load_words(vp + vchunk, raw.v[b], std::integral_constant<int, VW>{});
          raw.vs[b] = *reinterpret_cast<const uint32_t*>(vp + ps * (D / 2) - (__shfl(codes, vl) - rest) / 16 * 15 + vgroup * 4);
        } else {
          const char* kp = kh + from_lane(places, 16 * b + lr) + k_own;
#pragma unroll
          for (int ks = 0; ks < NS; ++ks) load_words(kp + ks * 64, raw.k[b] + 4 * ks, std::integral_constant<int, 4>{});
#pragma unroll
          for (int j = 0; j < 4; ++j)
            load_words(vh + from_lane(places, 16 * b + 4 * grp + j) + v_own, raw.v[b] + j * ND,
                       std::integral_constant<int, ND>{});
        }
      }
    }
  };

  f32x4 acc[NA];
  float m, l;
  const float sc = A.scale_log2, lag = P::kLag / sc;

  enum { kAll, kFinite, kOdd };  // what of V a walk takes
  auto consume = [&](int i, const Raw& raw, int walk) {
    const int t0 = seen_tile(seen, i) * kTile;
    f32x4 s[2];
    const float from = m == -INFINITY ? 0.f : -m;  // scores begin at -m, so that they come out as the differences
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      s[b] = f32x4{from, from, from, from};
#pragma unroll
      for (int ks = 0; ks < NS; ++ks) {
        u32x4 ka;
        if constexpr (FOUR) {
          ka = codes8(raw.k[b][ks], scale_of(raw.ks[b]));
        } else {
          ka = u32x4{raw.k[b][4 * ks], raw.k[b][4 * ks + 1], raw.k[b][4 * ks + 2], raw.k[b][4 * ks + 3]};
        }
#pragma unroll
        for (int pl = 0; pl < QP; ++pl) s[b] = mfma32<MT>(ka, qb[pl][ks], s[b]);
      }
    }
    // V: words [token 4 grp + j of block b][pairs of dims]
    uint32_t vt[8][ND];
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        uint32_t* w = vt[4 * b + j];
        if constexpr (FOUR) {
          const float scale = scale_of((raw.vs[b] >> (8 * j)) & 255u);
          if constexpr (D == 64) {
            const uint32_t x = raw.v[b][j] >> (lr % 2 * 16);
            w[0] = codes2<0>(x, scale);
            w[1] = codes2<1>(x, scale);
          } else {
            const u32x4 x = codes8(raw.v[b][j], scale);
#pragma unroll
            for (int e = 0; e < 4; ++e) w[e] = x[e];
          }
        } else {
#pragma unroll
          for (int e = 0; e < ND; ++e) w[e] = raw.v[b][j * ND + e];
        }
      }
    if (t0 + kTile > len || (t0 < seen.lo && t0 + kTile > seen.se)) {
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int t = t0 + 16 * b + 4 * grp + j;
          const bool on = t < len && (t >= seen.lo || t < seen.se);
          s[b][j] = on ? s[b][j] : -INFINITY;
#pragma unroll
          for (int e = 0; e < ND; ++e) vt[4 * b + j][e] = on ? vt[4 * b + j][e] : 0u;  // (0 times what lies there)
        }
    }
    if (walk != kAll) {
#pragma unroll
      for (int j = 0; j < 8; ++j)
#pragma unroll
        for (int e = 0; e < ND; ++e) {
          const uint32_t held = (finite16(vt[j][e] & 0xffffu, kBf16) ? 0xffffu : 0u) |
                                (finite16(vt[j][e] >> 16, kBf16) ? 0xffff0000u : 0u);
          vt[j][e] &= walk == kFinite ? held : ~held;
        }
    }
    u32x4 pb[P::kPlanes];
    if (walk == kOdd) {
      const uint32_t one = pack2<MT>(1.f, 1.f);
#pragma unroll
      for (int pl = 0; pl < P::kPlanes; ++pl) pb[pl] = u32x4{one, one, one, one};
    } else {
      float mx = -INFINITY;
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int j = 0; j < 4; ++j) mx = fmaxf(mx, s[b][j]);
      if (__builtin_amdgcn_ballot_w64(mx > (m == -INFINITY ? -INFINITY : lag)) != 0) {
        const Rise rise = rise_to(column_max(mx), m, sc);
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
          for (int j = 0; j < 4; ++j) s[b][j] -= rise.up;
        const float alpha = rise.alpha;
        l *= alpha;
#pragma unroll
        for (int a = 0; a < NA; ++a)
#pragma unroll
          for (int j = 0; j < 4; ++j) acc[a][j] *= alpha;
      }
      float ps_ = 0.f;
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        float p[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          p[j] = P::weight(s[b][j], sc);
          ps_ += p[j];
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          uint32_t w[P::kPlanes];
          P::split(p[2 * i], p[2 * i + 1], w);
#pragma unroll
          for (int pl = 0; pl < P::kPlanes; ++pl) pb[pl][2 * b + i] = w[pl];
        }
      }
      l += ps_;  // per lane; the column's lanes meet after the last tile
    }
#pragma unroll
    for (int e = 0; e < ND; ++e) {
      u32x4 v0, v1;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        v0[j] = __builtin_amdgcn_perm(vt[2 * j + 1][e], vt[2 * j][e], 0x05040100u);
        v1[j] = __builtin_amdgcn_perm(vt[2 * j + 1][e], vt[2 * j][e], 0x07060302u);
      }
#pragma unroll
      for (int pl = 0; pl < P::kPlanes; ++pl) {
        acc[2 * e] = mfma32<MT>(v0, pb[pl], acc[2 * e]);
        acc[2 * e + 1] = mfma32<MT>(v1, pb[pl], acc[2 * e + 1]);
      }
    }
  };

  for (int walk = kAll;; ++walk) {
    if (walk != kOdd) {
      m = -INFINITY;
      l = 0.f;
#pragma unroll
      for (int a = 0; a < NA; ++a) acc[a] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    if (begin < end) {
      Raw r0, r1;
      if (!PAGE16) ask(begin);
      fetch(begin, r0);
      int i = begin;
      for (; i + 2 <= end; i += 2) {
        fetch(i + 1, r1);
        consume(i, r0, walk);
        fetch(min(i + 2, end - 1), r0);
        consume(i + 1, r1, walk);
      }
      if (i < end) consume(i, r0, walk);
    }
    if (walk == kOdd) break;
    bool odd = false;
#pragma unroll
    for (int a = 0; a < NA; ++a)
#pragma unroll
      for (int j = 0; j < 4; ++j) odd |= acc[a][j] != acc[a][j];
    if (walk == kAll && __builtin_amdgcn_ballot_w64(odd) == 0) break;
  }
  l += __shfl_xor(l, 16);
  l += __shfl_xor(l, 32);
  if (lr < rows) {
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int a = 0; a < NA; a += 4)
        *reinterpret_cast<f32x4*>(&s_o[wave][lr][(4 * grp + j) * NA + a]) =
            f32x4{acc[a][j], acc[a + 1][j], acc[a + 2][j], acc[a + 3][j]};
    if (grp == 0) {
      s_m[wave][lr] = m;
      s_l[wave][lr] = l;
    }
  }
  __syncthreads();
  const int parts = uniform(it.parts);
  if (parts > 1 && (unsigned)it.slot >= (unsigned)max_slots_of(A.want.batch, A.want.max_items)) return;
  float* part = A.part + ((int64_t)uniform(it.slot) * A.hkv * A.blocks + blockIdx.y) * part_floats<D>();
  for (int c = threadIdx.x; c < rows * (D / 4); c += kThreads) {
    const int r = c / (D / 4), d = c % (D / 4) * 4;
    float mx = -INFINITY;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) mx = fmaxf(mx, s_m[w][r]);
    float sum = 0.f;
    f32x4 o = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      const float f = weight(s_m[w][r], mx, A.scale_log2);
      const f32x4 x = *reinterpret_cast<const f32x4*>(&s_o[w][r][d]);
      sum += s_l[w][r] * f;
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] += weighted(x[e], f);
    }
    if (parts > 1) {
      *reinterpret_cast<f32x4*>(part + r * D + d) = o;
      if (d == 0) *reinterpret_cast<f32x2*>(part + 16 * D + 2 * r) = f32x2{mx, sum};
      continue;
    }
    const float inv = sum > 0.f ? 1.f / sum : (sum == 0.f ? 0.f : sum);
    const int hq = h * g + hb * 16 + r;
    *reinterpret_cast<u32x2*>(A.o + (int64_t)row * A.o_sb + (int64_t)hq * A.o_sh + d * 2) =
        u32x2{pack2<T>(o[0] * inv, o[1] * inv), pack2<T>(o[2] * inv, o[3] * inv)};
    if (d == 0 && A.lse) A.lse[(int64_t)row * A.hq + hq] = log_sum(mx, A.scale_log2, sum, P::kShift);
  }
}

// A workgroup per (request, head) of several items: D / 4 lanes take a part, four dims
// each, and so many parts at a time; what they saw meets in LDS.
template <typename T, bool FOUR, int D>
__global__ __launch_bounds__(kThreads) void merge_kernel(Args A) {
  using P = Planes<typename std::conditional<FOUR, bf16_t, T>::type>;
  constexpr int kLanes = D / 4, kGroups = kThreads / kLanes, kAhead = 4;
  __shared__ __align__(16) float s_o[kGroups][D];
  __shared__ float s_m[kGroups], s_l[kGroups];
  const int row = blockIdx.x / A.hq, hq = blockIdx.x % A.hq;
  const Header head = *A.header;
  const Row rec = A.rows[row];
  const int parts = uniform(rec.parts), first = uniform(rec.slot);
  if (stale(head, A.want) || parts <= 1 || first < 0 || first + parts > max_slots_of(A.want.batch, A.want.max_items)) return;
  const int g = A.hq / A.hkv, h = hq / g, r = hq % g;
  const float* p = A.part + ((int64_t)first * A.hkv * A.blocks + h * A.blocks + r / 16) * part_floats<D>();
  const int64_t step = (int64_t)A.hkv * A.blocks * part_floats<D>();
  const int group = threadIdx.x / kLanes, d = threadIdx.x % kLanes * 4;
  float m = -INFINITY, l = 0.f;
  f32x4 o = f32x4{0.f, 0.f, 0.f, 0.f};
  for (int i0 = group; i0 < parts; i0 += kAhead * kGroups) {
    f32x4 v[kAhead];
    f32x2 ml[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const float* q = p + min(i0 + i * kGroups, parts - 1) * step;
      v[i] = *reinterpret_cast<const f32x4*>(q + (r % 16) * D + d);
      ml[i] = *reinterpret_cast<const f32x2*>(q + 16 * D + 2 * (r % 16));
    }
    float top = m;
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      if (i0 + i * kGroups >= parts) ml[i] = f32x2{-INFINITY, 0.f}, v[i] = f32x4{0.f, 0.f, 0.f, 0.f};
      top = fmaxf(top, ml[i][0]);
    }
    const float w = weight(m, top, A.scale_log2);
    l *= w;
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = weighted(o[e], w);
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const float wi = weight(ml[i][0], top, A.scale_log2);
      l += ml[i][1] * wi;
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] += weighted(v[i][e], wi);
    }
    m = top;
  }
  *reinterpret_cast<f32x4*>(&s_o[group][d]) = o;
  if (d == 0) {
    s_m[group] = m;
    s_l[group] = l;
  }
  __syncthreads();
  if (group > 0) return;
  float top = -INFINITY, sum = 0.f;
#pragma unroll
  for (int i = 0; i < kGroups; ++i) top = fmaxf(top, s_m[i]);
  o = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < kGroups; ++i) {
    const float w = weight(s_m[i], top, A.scale_log2);
    const f32x4 x = *reinterpret_cast<const f32x4*>(&s_o[i][d]);
    sum += s_l[i] * w;
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] += weighted(x[e], w);
  }
  const float inv = sum > 0.f ? 1.f / sum : (sum == 0.f ? 0.f : sum);
  *reinterpret_cast<u32x2*>(A.o + (int64_t)row * A.o_sb + (int64_t)hq * A.o_sh + d * 2) =
      u32x2{pack2<T>(o[0] * inv, o[1] * inv), pack2<T>(o[2] * inv, o[3] * inv)};
  if (d == 0 && A.lse) A.lse[(int64_t)row * A.hq + hq] = log_sum(top, A.scale_log2, sum, P::kShift);
}

template <typename T, bool FOUR, int D>
int launch(const Args& a, hipStream_t s) {
  const dim3 grid((unsigned)a.want.max_items, (unsigned)(a.hkv * a.blocks));
  if (a.want.page_size % 16 == 0)
    hipLaunchKernelGGL((decode_kernel<T, FOUR, D, true>), grid, dim3(kThreads), 0, s, a);
  else
    hipLaunchKernelGGL((decode_kernel<T, FOUR, D, false>), grid, dim3(kThreads), 0, s, a);
  PL_LAUNCH_CHECK("window decode_kernel");
  hipLaunchKernelGGL((merge_kernel<T, FOUR, D>), dim3((unsigned)(a.want.batch * a.hq)), dim3(kThreads), 0, s, a);
  PL_LAUNCH_CHECK("window merge_kernel");
  return ok();
}

template <typename T, bool FOUR>
int launch_d(const Args& a, int d, hipStream_t s) {
  return d == 64 ? launch<T, FOUR, 64>(a, s) : launch<T, FOUR, 128>(a, s);
}

}  // namespace dec
}  // namespace window
}  // namespace pl

using namespace pl;
using namespace pl::window;
using namespace pl::window::dec;

static int check_shape(int batch, int hq, int hkv, int page_size, int window, int sinks) {
  if (batch < 0) return fail(PL_ERR_INVALID, "batch must be >= 0 (got %d)", batch);
  if (hkv <= 0 || hq <= 0 || hq % hkv)
    return fail(PL_ERR_INVALID, "num_qo_heads (%d) must be a multiple of num_kv_heads (%d)", hq, hkv);
  if ((int64_t)batch * hq >= kMaxGroups || batch + 2048 >= kMaxGroups) return fail(PL_ERR_INVALID, "%d rows of %d heads are too many", batch, hq);
  if ((int64_t)hkv * head_blocks(hq, hkv) > 65535) return fail(PL_ERR_INVALID, "%d kv heads are too many", hkv);
  if (page_size <= 0 || page_size > kMaxLen) return fail(PL_ERR_INVALID, "page_size must be positive (got %d)", page_size);
  if (window < 0 || sinks < 0) return fail(PL_ERR_INVALID, "window and sinks must be >= 0");
  return PL_OK;
}

extern "C" size_t pl_window_decode_plan_size(int batch, int indices_capacity, int num_qo_heads, int num_kv_heads,
                                             int page_size, int window, int sinks) {
  if (check_shape(batch, num_qo_heads, num_kv_heads, page_size, window, sinks) != PL_OK) return 0;
  if (indices_capacity < 0) return fail(PL_ERR_INVALID, "indices_capacity must be >= 0"), 0;
  return layout(batch, indices_capacity, max_items_of(batch, num_qo_heads, num_kv_heads, page_size, window, sinks,
                                                      indices_capacity)).bytes;
}

extern "C" size_t pl_window_decode_workspace_size(int batch, int indices_capacity, int num_qo_heads, int num_kv_heads,
                                                  int head_dim, int page_size, int window, int sinks) {
  if (check_shape(batch, num_qo_heads, num_kv_heads, page_size, window, sinks) != PL_OK) return 0;
  if (indices_capacity < 0 || head_dim < 0) return fail(PL_ERR_INVALID, "sizes must be >= 0"), 0;
  const int items = max_items_of(batch, num_qo_heads, num_kv_heads, page_size, window, sinks, indices_capacity);
  return (size_t)max_slots_of(batch, items) * num_kv_heads * head_blocks(num_qo_heads, num_kv_heads) * 16 *
         (head_dim + 2) * sizeof(float);
}

static Header wanted(int batch, int page_size, int window, int sinks, int capacity, int hq, int hkv) {
  Header h{};
  h.magic = kMagic ^ (hq << 8) ^ hkv;
  h.batch = batch;
  h.page_size = page_size;
  h.window = window;
  h.sinks = sinks;
  h.indices_capacity = capacity;
  h.max_items = max_items_of(batch, hq, hkv, page_size, window, sinks, capacity);
  return h;
}

extern "C" int pl_window_decode_plan(const int32_t* indptr, const int32_t* indices, int indices_capacity,
                                     const int32_t* last_page_len, int batch, int num_qo_heads, int num_kv_heads,
                                     int page_size, int window, int sinks, void* plan, size_t plan_bytes,
                                     void* stream) {
  if (int e = check_shape(batch, num_qo_heads, num_kv_heads, page_size, window, sinks)) return e;
  if (indices_capacity < 0) return fail(PL_ERR_INVALID, "indices_capacity must be >= 0");
  if (batch == 0) return ok();
  if (!indptr || !last_page_len || !plan || (indices_capacity > 0 && !indices))
    return fail(PL_ERR_INVALID, "null pointer argument");
  if ((uintptr_t)plan % 64) return fail(PL_ERR_INVALID, "the plan must be 64-byte aligned");
  const Header want = wanted(batch, page_size, window, sinks, indices_capacity, num_qo_heads, num_kv_heads);
  const Layout l = layout(batch, indices_capacity, want.max_items);
  if (plan_bytes < l.bytes) return fail(PL_ERR_WORKSPACE, "plan of %zu bytes < %zu needed", plan_bytes, l.bytes);
  PlanArgs a{};
  char* p = (char*)plan;
  a.indptr = indptr;
  a.indices = indices;
  a.last = last_page_len;
  a.want = want;
  a.header = (Header*)p;
  a.items = (Item*)(p + l.items);
  a.rows = (Row*)(p + l.rows);
  a.ids = (int32_t*)(p + l.indices);
  a.heads = num_kv_heads * head_blocks(num_qo_heads, num_kv_heads);
  const int copies = (indices_capacity + 4 * kPlanThreads - 1) / (4 * kPlanThreads);
  hipLaunchKernelGGL(plan_kernel, dim3(1 + (copies < 64 ? copies : 64)), dim3(kPlanThreads), 0, (hipStream_t)stream, a);
  PL_LAUNCH_CHECK("window plan_kernel");
  return ok();
}

extern "C" int pl_window_decode_run(const void* q, int64_t q_stride_b, int64_t q_stride_h, const void* k_cache,
                                    const void* v_cache, int64_t page_stride, int64_t token_stride,
                                    int64_t head_stride, int64_t num_pages, int kv_bits, void* o, int64_t o_stride_b,
                                    int64_t o_stride_h, float* lse, int batch, int num_qo_heads, int num_kv_heads,
                                    int head_dim, int page_size, int window, int sinks, float sm_scale, int dtype,
                                    const void* plan, size_t plan_bytes, int indices_capacity, void* workspace,
                                    size_t workspace_bytes, void* stream) {
  if (int e = check_shape(batch, num_qo_heads, num_kv_heads, page_size, window, sinks)) return e;
  if (head_dim != 64 && head_dim != 128)
    return fail(PL_ERR_UNSUPPORTED, "head_dim must be 64 or 128 (got %d)", head_dim);
  if (dtype != PL_DTYPE_BF16 && dtype != PL_DTYPE_F16)
    return fail(PL_ERR_UNSUPPORTED, "dtype must be F16 or BF16 (got %d)", dtype);
  if (kv_bits != 16 && kv_bits != 4) return fail(PL_ERR_UNSUPPORTED, "kv_bits must be 16 or 4 (got %d)", kv_bits);
  if (kv_bits == 4 && (page_size % 8 || page_size > (1 << 20)))
    return fail(PL_ERR_INVALID, "pages of a 4-bit cache hold a multiple of 8 tokens, up to 2^20 (got %d)", page_size);
  if (num_pages <= 0 || indices_capacity < 0) return fail(PL_ERR_INVALID, "num_pages must be positive");
  if (batch == 0) return ok();
  if (!q || !k_cache || !v_cache || !o || !plan || !workspace) return fail(PL_ERR_INVALID, "null pointer argument");
  const int eb = kv_bits == 4 ? 1 : 2;  // a 4-bit cache's strides are bytes
  const int64_t strides[] = {q_stride_b * 2, q_stride_h * 2, o_stride_b * 2, o_stride_h * 2, page_stride * eb,
                             kv_bits == 4 ? 0 : token_stride * eb, head_stride * eb};
  for (int64_t st : strides)
    if (st % 16) return fail(PL_ERR_INVALID, "strides must be multiples of 16 bytes");
  const void* ptrs[] = {q, k_cache, v_cache, o, workspace};
  for (const void* p : ptrs)
    if ((uintptr_t)p % 16) return fail(PL_ERR_INVALID, "q, o, the caches and workspace must be 16-byte aligned");
  if ((uintptr_t)plan % 64) return fail(PL_ERR_INVALID, "the plan must be 64-byte aligned");
  const Header want = wanted(batch, page_size, window, sinks, indices_capacity, num_qo_heads, num_kv_heads);
  const Layout lay = layout(batch, indices_capacity, want.max_items);
  if (plan_bytes < lay.bytes) return fail(PL_ERR_WORKSPACE, "plan of %zu bytes < %zu needed", plan_bytes, lay.bytes);
  const size_t need = pl_window_decode_workspace_size(batch, indices_capacity, num_qo_heads, num_kv_heads,
                                                      head_dim, page_size, window, sinks);
  if (workspace_bytes < need)
    return fail(PL_ERR_WORKSPACE, "workspace of %zu bytes < %zu needed", workspace_bytes, need);
  Args a{};
  const char* p = (const char*)plan;
  a.q = (const char*)q;
  a.k = (const char*)k_cache;
  a.v = (const char*)v_cache;
  a.o = (char*)o;
  a.lse = lse;
  a.part = (float*)workspace;
  a.header = (const Header*)p;
  a.items = (const Item*)(p + lay.items);
  a.rows = (const Row*)(p + lay.rows);
  a.ids = (const int32_t*)(p + lay.indices);
  a.want = want;
  a.q_sb = strides[0];
  a.q_sh = strides[1];
  a.o_sb = strides[2];
  a.o_sh = strides[3];
  a.page_stride = strides[4];
  a.token_stride = strides[5];
  a.head_stride = strides[6];
  a.num_pages = num_pages;
  a.hq = num_qo_heads;
  a.hkv = num_kv_heads;
  a.blocks = head_blocks(num_qo_heads, num_kv_heads);
  a.page_shift = (page_size & (page_size - 1)) == 0 ? __builtin_ctz(page_size) : -1;
  // maxima are taken before scaling: a positive scale (a zero one as one far below
  // any score's rounding), the sign moved into q
  const float s2 = sm_scale * 1.44269504088896340736f;
  a.scale_log2 = fmaxf(fabsf(s2), 1e-30f);
  a.q_flip = s2 < 0 ? 0x80008000u : 0u;
  const hipStream_t st = (hipStream_t)stream;
  if (dtype == PL_DTYPE_BF16)
    return kv_bits == 4 ? launch_d<bf16_t, true>(a, head_dim, st) : launch_d<bf16_t, false>(a, head_dim, st);
  return kv_bits == 4 ? launch_d<f16_t, true>(a, head_dim, st) : launch_d<f16_t, false>(a, head_dim, st);
}
