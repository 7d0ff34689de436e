// Attention of trees of drafted tokens over a paged KV cache (gfx950).
//
// Request r has T_r tree tokens, the last T_r of its kv_len_r positions; the
// P_r = kv_len_r - T_r before them are its committed tokens.  Tree token i
// attends the committed tokens and those tree tokens j that its mask names
// (itself and its ancestors where the tree is given by parents):
//   o_i = sum_t p_it v_t / sum_t p_it,  p_it = exp(s q_i . k_t)
// over t < P_r and t = P_r + j with sees(i, j).  A row that sees nothing gets
// o = 0 and lse = -inf.
//
// plan_kernel (once per step, for all layers) checks the tables, cuts the work
// and packs the masks into 64-bit words.  A work item is R rows (tree token,
// head of the GQA group) of a request over a range of kv tiles; one workgroup
// takes one item for one kv head.  Its waves share the rows and take 32 tokens
// of a tile each, in LDS buffers of their own that are filled straight from the
// pages while the block before is worked on: no wave waits for another until
// the item ends.  Few rows then cost few instructions per byte, and one pass
// over the cache serves all rows.  S^T = K Q^T keeps a query per lane; the
// probabilities are the B operand of O^T += V^T P^T as they lie, and V comes
// out of LDS transposed.  The waves' states meet in LDS at the item's end, and
// the parts of rows whose range was cut in merge_kernel, in order.
#include <algorithm>
#include <type_traits>

#include "pl_common.h"

namespace pl {
namespace tree {

constexpr int kWave = 64;
constexpr int kBlock = 32;        // kv tokens of a wave per tile
constexpr int kMaxRequests = 4096;
constexpr int kMagic = 0x54524545;
constexpr int kPlanThreads = 1024;
constexpr int kCandidates = 128;  // split counts of the longest range that the plan weighs

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef short i16x4 __attribute__((ext_vector_type(4)));
typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned int u32x2 __attribute__((ext_vector_type(2)));

// What a plan was made for, then what it holds.
struct Header {
  int32_t magic, batch, tokens, max_tree, indices_capacity, hq, hkv, head_dim, page_size;
  int32_t num_items, num_blocks, pad[5];
};
static_assert(sizeof(Header) == 64, "the plan's header");
struct Request {
  int32_t q_begin, tree, page_begin, kv_len;
};
// R rows of a request: its parts are the items slot, slot + step, ...
struct RowBlock {
  int32_t request, row0, slot, step, parts, pad[3];
};
struct Item {
  int32_t request, row0, tile_begin, tile_end, parts, pad[3];
};

// ------------------------------------------------------- sizes and layout ---
inline int waves_of(int head_dim) { return head_dim == 256 ? 2 : 4; }
inline int tile_of(int head_dim) { return kBlock * waves_of(head_dim); }

// 16-row columns a wave holds: as few as the widest tree needs, at most 4 (2 at
// head_dim 256, by its accumulators).
inline int cols_of(int64_t max_tree, int g, int head_dim) {
  const int64_t rows = max_tree * g;
  const int most = head_dim == 256 ? 2 : 4;
  return std::min(most, rows <= 16 ? 1 : (rows <= 32 ? 2 : 4));
}

// Workgroups per kv head that run at once: one per CU by their LDS, two at head_dim 64.
inline int slots_of(int hkv, int head_dim) { return std::max(1, (head_dim == 64 ? 512 : 256) / hkv); }

struct Layout {
  int rows, slots, max_blocks, max_items, mask_words;
  size_t requests, blocks, items, masks, indices, bytes;  // offsets, then the size
};

inline Layout layout(int batch, int tokens, int max_tree, int indices_capacity, int hq, int hkv, int head_dim) {
  Layout l{};
  const int g = hq / hkv;
  l.rows = 16 * cols_of(max_tree, g, head_dim);
  l.slots = slots_of(hkv, head_dim);
  l.max_blocks = (int)((int64_t)tokens * g / l.rows) + batch;
  l.max_items = l.max_blocks + 3 * l.slots;
  l.mask_words = (max_tree + 63) / 64;
  size_t at = sizeof(Header);
  l.requests = at;
  at += align_up(sizeof(Request) * (size_t)batch, 64);
  l.blocks = at;
  at += sizeof(RowBlock) * (size_t)l.max_blocks;
  l.items = at;
  at += sizeof(Item) * (size_t)l.max_items;
  l.masks = at;
  at += align_up(sizeof(uint64_t) * (size_t)tokens * l.mask_words, 64);
  l.indices = at;
  at += align_up(sizeof(int32_t) * (size_t)indices_capacity, 64);
  l.bytes = at;
  return l;
}

// ------------------------------------------------------------------- plan ---
struct PlanArgs {
  const int32_t *qo_indptr, *kv_indptr, *kv_indices, *kv_last, *parents;
  const uint8_t* mask;
  int64_t mask_ld;
  Header* header;
  Request* requests;
  RowBlock* blocks;
  Item* items;
  uint64_t* masks;
  int32_t* indices;
  int batch, tokens, max_tree, indices_count, indices_capacity, hq, hkv, head_dim, page_size;
  int rows, tile, slots, max_items, max_blocks, mask_words;
  int parts_fixed;  // > 0: cuts of the longest range (0: weighed)
};

__device__ __forceinline__ Request read_request(const PlanArgs& A, int r) {
  Request q;
  q.q_begin = min(max(A.qo_indptr[r], 0), A.tokens);
  q.tree = min(min(max(A.qo_indptr[r + 1], q.q_begin), A.tokens) - q.q_begin, A.max_tree);
  q.page_begin = min(max(A.kv_indptr[r], 0), A.indices_count);
  const int pages = min(max(A.kv_indptr[r + 1], q.page_begin), A.indices_count) - q.page_begin;
  const int last = min(max(A.kv_last[r], 1), A.page_size);
  const int64_t len = pages > 0 ? (int64_t)(pages - 1) * A.page_size + last : 0;
  q.kv_len = (int)min(len, (int64_t)(INT32_MAX / 2));
  return q;
}

// Workgroup 0 cuts the work; the others copy the page ids and pack the masks.
__global__ __launch_bounds__(kPlanThreads) void plan_kernel(PlanArgs A) {
  const int tid = threadIdx.x, lane = tid % kWave, wave = tid / kWave;
  if (blockIdx.x > 0) {
    const int64_t step = (int64_t)(gridDim.x - 1) * kPlanThreads;
    const int64_t first = (int64_t)(blockIdx.x - 1) * kPlanThreads + tid;
    for (int64_t i = first; i < A.indices_count; i += step) A.indices[i] = A.kv_indices[i];
    for (int64_t i = first; i < (int64_t)A.tokens * A.mask_words; i += step) {
      const int t = (int)(i / A.mask_words), w = (int)(i % A.mask_words);
      int lo = 0, hi = A.batch;  // the request that holds token t: the last whose first token is <= t
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (A.qo_indptr[mid] <= t) lo = mid; else hi = mid;
      }
      const Request q = read_request(A, lo);
      const int node = t - q.q_begin;
      uint64_t bits = 0;
      if (node >= 0 && node < q.tree) {
        if (A.parents) {
          // a parent is an earlier node: the walk ends
          for (int at = node; at >= 0;) {
            if (at / 64 == w) bits |= 1ull << (at % 64);
            const int up = A.parents[q.q_begin + at];
            at = up < at ? up : -1;
          }
        } else {
          const uint8_t* m = A.mask + (int64_t)t * A.mask_ld + w * 64;
          const int n = min(q.tree - w * 64, 64);
          for (int j = 0; j < n; ++j) bits |= (uint64_t)(m[j] != 0) << j;
        }
      }
      A.masks[i] = bits;
    }
    return;
  }

  __shared__ int s_tiles[kMaxRequests];       // tiles of a request's kv
  __shared__ int s_nblocks[kMaxRequests];     // row blocks of its tree
  __shared__ int s_item[kMaxRequests];        // items before it
  __shared__ int s_block[kMaxRequests];       // row blocks before it
  __shared__ int s_scan[2][kPlanThreads];
  __shared__ int s_longest, s_chunk;
  __shared__ float s_cost[kCandidates];
  const int g = A.hq / A.hkv;
  if (tid == 0) s_longest = 1;
  __syncthreads();
  for (int r = tid; r < A.batch; r += kPlanThreads) {
    const Request q = read_request(A, r);
    A.requests[r] = q;
    s_tiles[r] = max(1, (q.kv_len + A.tile - 1) / A.tile);
    s_nblocks[r] = (int)(((int64_t)q.tree * g + A.rows - 1) / A.rows);
    if (q.tree > 0) atomicMax(&s_longest, s_tiles[r]);
  }
  __syncthreads();
  const int longest = s_longest;

  // The length of a part: of the longest range cut 1 .. 128 times, the one with
  // the least estimated time in tiles.  An item costs its tiles and kOver more
  // (its first loads, its partial results and the merge's reading of them);
  // items in excess of the slots share them evenly but for half a part.
  constexpr float kOver = 2.f;
  for (int k = wave; k < kCandidates; k += kPlanThreads / kWave) {
    const int chunk = (longest + k) / (k + 1);
    long long items = 0, work = 0;
    for (int r = lane; r < A.batch; r += kWave) {
      items += (long long)((s_tiles[r] + chunk - 1) / chunk) * s_nblocks[r];
      work += (long long)s_tiles[r] * s_nblocks[r];
    }
#pragma unroll
    for (int d = 1; d < kWave; d <<= 1) {
      items += __shfl_xor(items, d);
      work += __shfl_xor(work, d);
    }
    float cost = ((float)work + kOver * (float)items) / A.slots + (items > A.slots ? 0.5f * chunk : 0.f);
    cost = fmaxf(cost, chunk + kOver);
    if (k > 0 && items > A.max_items) cost = INFINITY;
    if (A.parts_fixed > 0 && k > 0 && k + 1 != A.parts_fixed) cost = INFINITY;
    if (A.parts_fixed > 1 && k == 0) cost = 1e37f;
    if (lane == 0) s_cost[k] = cost;
  }
  __syncthreads();
  if (tid == 0) {
    int best = 0;
    for (int k = 1; k < kCandidates; ++k)
      if (s_cost[k] < s_cost[best]) best = k;
    s_chunk = (longest + best) / (best + 1);
  }
  __syncthreads();
  const int chunk = s_chunk;

  // items and row blocks before each request: each thread owns a run of requests
  const int per = (A.batch + kPlanThreads - 1) / kPlanThreads;
  const int r0 = min(A.batch, tid * per), r1 = min(A.batch, r0 + per);
  int items = 0, blocks = 0;
  for (int r = r0; r < r1; ++r) {
    items += (s_tiles[r] + chunk - 1) / chunk * s_nblocks[r];
    blocks += s_nblocks[r];
  }
  s_scan[0][tid] = items;
  s_scan[1][tid] = blocks;
  __syncthreads();
  for (int off = 1; off < kPlanThreads; off <<= 1) {
    const int a = tid >= off ? s_scan[0][tid - off] : 0, b = tid >= off ? s_scan[1][tid - off] : 0;
    __syncthreads();
    s_scan[0][tid] += a;
    s_scan[1][tid] += b;
    __syncthreads();
  }
  items = s_scan[0][tid] - items;
  blocks = s_scan[1][tid] - blocks;
  for (int r = r0; r < r1; ++r) {
    s_item[r] = items;
    s_block[r] = blocks;
    items += (s_tiles[r] + chunk - 1) / chunk * s_nblocks[r];
    blocks += s_nblocks[r];
  }
  // (a decreasing qo_indptr can ask for more than there is room for: it loses the rest)
  const int n_items = min(s_scan[0][kPlanThreads - 1], A.max_items);
  const int n_blocks = min(s_scan[1][kPlanThreads - 1], A.max_blocks);
  __syncthreads();
  auto owner = [&](const int* before, int i) {  // the last request r with before[r] <= i
    int lo = 0, hi = A.batch;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (before[mid] <= i) lo = mid; else hi = mid;
    }
    return lo;
  };
  // the row blocks of one kv range side by side: they find its pages in the L2
  for (int i = tid; i < n_items; i += kPlanThreads) {
    const int r = owner(s_item, i), at = i - s_item[r], nb = s_nblocks[r];
    const int parts = (s_tiles[r] + chunk - 1) / chunk, part = at / nb;
    Item it{};
    it.request = r;
    it.row0 = (at % nb) * A.rows;
    it.tile_begin = (int)((int64_t)s_tiles[r] * part / parts);
    it.tile_end = (int)((int64_t)s_tiles[r] * (part + 1) / parts);
    it.parts = parts;
    A.items[i] = it;
  }
  for (int i = tid; i < n_blocks; i += kPlanThreads) {
    const int r = owner(s_block, i), at = i - s_block[r];
    RowBlock b{};
    b.request = r;
    b.row0 = at * A.rows;
    b.slot = s_item[r] + at;
    b.step = s_nblocks[r];
    b.parts = (s_tiles[r] + chunk - 1) / chunk;
    if (b.slot + (int64_t)(b.parts - 1) * b.step >= n_items) b.parts = 0;
    A.blocks[i] = b;
  }
  if (tid == 0) {
    Header h{};
    h.magic = kMagic;
    h.batch = A.batch;
    h.tokens = A.tokens;
    h.max_tree = A.max_tree;
    h.indices_capacity = A.indices_capacity;
    h.hq = A.hq;
    h.hkv = A.hkv;
    h.head_dim = A.head_dim;
    h.page_size = A.page_size;
    h.num_items = n_items;
    h.num_blocks = n_blocks;
    *A.header = h;
  }
}

// -------------------------------------------------------------- attention ---
template <typename T> __device__ __forceinline__ f32x4 mfma32(u32x4 a, u32x4 b, f32x4 c);
template <> __device__ __forceinline__ f32x4 mfma32<bf16_t>(u32x4 a, u32x4 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0,
                                                 0, 0);
}
template <> __device__ __forceinline__ f32x4 mfma32<f16_t>(u32x4 a, u32x4 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0,
                                                0);
}

// The largest of the four lanes l, l ^ 16, l ^ 32, l ^ 48.
__device__ __forceinline__ float column_max(float v) {
  auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}

__device__ __forceinline__ void load_lds16(const char* g, char* l) {
  __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)g,
                                   (__attribute__((address_space(3))) void*)l, 16, 0, 0);
}

__device__ __forceinline__ u32x2 read_tr(const char* p) {
  return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) i16x4*)p));
}

// Infinities and NaN of two packed 16-bit values: the exponent is all ones.
template <typename T> __device__ __forceinline__ bool nonfinite16(uint32_t v) {
  constexpr uint32_t e = std::is_same<T, bf16_t>::value ? 0x7f80u : 0x7c00u;
  return (v & e) == e;
}

struct Args {
  const char *q, *k, *v;
  char* o;
  float *lse, *part;
  const Header* header;
  const Request* requests;
  const RowBlock* blocks;
  const Item* items;
  const uint64_t* masks;
  const int32_t* indices;
  int64_t q_st, q_sh, o_st, o_sh, page_stride, token_stride, head_stride, num_pages;  // elements
  Header want;
  int max_items, max_blocks, mask_words;
  float scale_log2;  // > 0; a negative scale negates q instead
  uint32_t q_flip;
};

// A run on a plan made for other arguments does nothing rather than read astray.
__device__ __forceinline__ bool plan_fits(const Args& A) {
  const Header& h = *A.header;
  const Header& w = A.want;
  return h.magic == kMagic && h.batch == w.batch && h.tokens == w.tokens && h.max_tree == w.max_tree &&
         h.indices_capacity == w.indices_capacity && h.hq == w.hq && h.hkv == w.hkv && h.head_dim == w.head_dim &&
         h.page_size == w.page_size && h.num_items <= A.max_items && h.num_blocks <= A.max_blocks;
}

template <typename T> struct Softmax {
  static constexpr bool kTwo = std::is_same<T, bf16_t>::value;
  // bf16 probabilities enter the product as two planes, hi + lo, so they carry
  // 16 bits; fp16's one plane carries its 11.
  static constexpr int kPlanes = kTwo ? 2 : 1;
  // A column's running maximum follows only scores more than kLag above it,
  // which takes the rescale out of the steady state.  One fp16 plane is exact
  // for the largest probability only where that is a power of two: no lag.
  static constexpr float kLag = kTwo ? 8.f : 0.f;
  // Probabilities are held 2^kShift times as large: fp16 ends at 2^-24, and
  // 32768 tokens of 2^-25 are no small part of a row.  2^14 keeps them to 2^-38.
  static constexpr float kShift = kTwo ? 0.f : 14.f;
};

// Finishes a row: its four dims by one lane, and the row's lse by lane `first`.
template <typename T>
__device__ __forceinline__ void store_row(const Args& A, const Request& q, int h, int row, int dim, f32x4 o, float top,
                                          float sum, bool first) {
  const int g = A.want.hq / A.want.hkv, node = row / g;
  const int64_t token = q.q_begin + node;
  const int head = h * g + row - node * g;
  const float inv = sum > 0.f ? 1.f / sum : (sum == 0.f ? 0.f : sum);
  T* op = (T*)A.o + token * A.o_st + (int64_t)head * A.o_sh + dim;
  *reinterpret_cast<u32x2*>(op) = u32x2{pack2<T>(o[0] * inv, o[1] * inv), pack2<T>(o[2] * inv, o[3] * inv)};
  if (A.lse && first)
    A.lse[token * A.want.hq + head] =
        sum == 0.f ? -INFINITY : (top + log2f(sum) - Softmax<T>::kShift) * 0.693147180559945309f;
}

template <typename T, int D, int C, bool PAGE16>
__global__ __launch_bounds__(D == 256 ? 128 : 256, 1) void tree_kernel(Args A) {
  using S = Softmax<T>;
  constexpr int NPP = S::kPlanes;
  constexpr int W = D == 256 ? 2 : 4;          // waves
  constexpr int NT = W * kWave;
  constexpr int R = 16 * C;
  constexpr int RB = D * 2;                    // bytes of a token's row
  constexpr int CPR = D / 8;                   // 16-byte chunks of a row
  constexpr int TPI = kWave / CPR;             // tokens per load
  constexpr int NL = kBlock / TPI;             // loads of a block's K
  constexpr int KS = D / 32, NA = D / 16;
  constexpr int kBuf = W * kBlock * RB;
  constexpr int kTile = W * kBlock;
  constexpr int kPartFloats = R * (D + 2);     // outputs [row][dim], then (max, sum) per row
  constexpr int kSwz = CPR < 16 ? CPR - 1 : 15;
  static_assert(kBuf >= R * D * 4, "a wave's outputs fit one buffer");
  // one object per buffer: loads into one never alias reads of another
  __shared__ __align__(16) char s_k0[kBuf];
  __shared__ __align__(16) char s_v0[kBuf];
  __shared__ __align__(16) char s_k1[kBuf];
  __shared__ __align__(16) char s_v1[kBuf];
  __shared__ float s_ml[W][R][2];

  if (!plan_fits(A)) return;
  const int n_items = A.header->num_items, hkv = A.want.hkv;
  // Workgroups go round the 8 XCDs.  Where the kv heads divide 8, each XCD keeps
  // one head and one run of the items, so row blocks of one range share an L2.
  int h, index;
  if (8 % hkv == 0) {
    const int rep = 8 / hkv, x = blockIdx.x % 8, per = (n_items + rep - 1) / rep, at = blockIdx.x / 8;
    h = x % hkv;
    index = at < per ? x / hkv * per + at : n_items;
  } else {
    h = blockIdx.x % hkv;
    index = blockIdx.x / hkv;
  }
  if (index >= n_items) return;
  const Item it = A.items[index];
  const Request rq = A.requests[it.request];
  const int g = A.want.hq / hkv, n_rows = rq.tree * g;
  const int kv_len = rq.kv_len, prefix = max(0, kv_len - rq.tree);
  const int page_size = A.want.page_size, n_pages = (kv_len + page_size - 1) / page_size;
  const int32_t* ind = A.indices + rq.page_begin;
  const int lane = threadIdx.x % kWave, wave = uniform(threadIdx.x / kWave);
  const int lr = lane % 16, grp = lane / 16;

  u32x4 qb[C][KS];
  const uint64_t* masks[C];
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const int row = min(it.row0 + c * 16 + lr, n_rows - 1);  // rows past the end repeat the last one, unstored
    const int node = row / g;
    masks[c] = A.masks + (int64_t)(rq.q_begin + node) * A.mask_words;
    const char* qp = A.q + ((int64_t)(rq.q_begin + node) * A.q_st + (int64_t)(h * g + row - node * g) * A.q_sh) * 2 + grp * 16;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      u32x4 v = *reinterpret_cast<const u32x4*>(qp + ks * 64);
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] ^= A.q_flip;
      qb[c][ks] = v;
    }
  }

  auto swz_k = [](int n) { return n & kSwz; };
  auto swz_v = [](int n) { return CPR < 16 ? (n & kSwz) : 2 * (n & 7); };
  auto clamp_page = [&](int page) -> int64_t {
    return page < 0 ? 0 : ((int64_t)page >= A.num_pages ? A.num_pages - 1 : (int64_t)page);
  };
  // byte offset of token t of the sequence (or of the page's rest behind the last one)
  auto token_offset = [&](int t) -> int64_t {
    const int page = t / page_size;
    return (clamp_page(ind[min(page, n_pages - 1)]) * A.page_stride + (int64_t)(t - page * page_size) * A.token_stride) * 2;
  };
  // Offsets of the wave's tokens, one per lane.  Pages of a multiple of 16
  // tokens: of the 16-token groups of 32 tiles; others: of a block's 32 tokens.
  auto load_offsets = [&](int tile) -> int64_t {
    if constexpr (PAGE16) return token_offset((tile + lane / 2) * kTile + wave * kBlock + (lane % 2) * 16);
    return token_offset(min(tile * kTile + wave * kBlock + lane % kBlock, kv_len - 1));
  };
  // loads: instruction j fetches tokens j TPI .. of the block, lane l chunk
  // l % CPR of token l / CPR, permuted by the token
  constexpr int JG = PAGE16 ? 16 / TPI : 1;
  int64_t koff[NL], voff[NL];
#pragma unroll
  for (int j = 0; j < NL; ++j) {
    const int n = j * TPI + lane / CPR;
    const int64_t base = ((PAGE16 ? (int64_t)(n % 16) * A.token_stride : 0) + (int64_t)h * A.head_stride) * 2;
    koff[j] = base + ((lane % CPR) ^ swz_k(n)) * 16;
    voff[j] = base + ((lane % CPR) ^ swz_v(n)) * 16;
  }
  auto load_block = [&](int64_t offs, int at, char* kd, char* vd) {
    kd += wave * kBlock * RB;
    vd += wave * kBlock * RB;
#pragma unroll
    for (int j = 0; j < NL; ++j) {
      int64_t off;
      if constexpr (PAGE16) {
        const int from = at * 2 + j / JG;
        off = (int64_t)((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)offs, from) |
                        (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(offs >> 32), from) << 32);
      } else {
        off = __shfl(offs, j * TPI + lane / CPR);
      }
      load_lds16(A.k + off + koff[j], kd + j * kWave * 16);
      load_lds16(A.v + off + voff[j], vd + j * kWave * 16);
    }
  };

  // operand reads: K row blk*16 + lr, chunk 4 ks + grp; V tokens 4 grp + lr/4
  // (+16), dims 16 a + 4 (lr % 4)
  int kaddr[KS], vaddr[NA];
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) kaddr[ks] = wave * kBlock * RB + lr * RB + ((ks * 4 + grp) ^ swz_k(lr)) * 16;
#pragma unroll
  for (int a = 0; a < NA; ++a) {
    const int n = grp * 4 + lr / 4;
    vaddr[a] = wave * kBlock * RB + n * RB + ((2 * a + (lr % 4) / 2) ^ swz_v(n)) * 16 + (lr % 2) * 8;
  }

  f32x4 acc[C][NA];
  float m[C], l[C];
#pragma unroll
  for (int c = 0; c < C; ++c) {
    m[c] = -INFINITY;
    l[c] = 0.f;
#pragma unroll
    for (int a = 0; a < NA; ++a) acc[c][a] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  const float sc = A.scale_log2;

  // the wave's blocks: only the last tile can lie behind its tokens
  const int t_begin = it.tile_begin;
  const int t_end = (it.tile_end - 1) * kTile + wave * kBlock < kv_len ? it.tile_end : it.tile_end - 1;
  int64_t offs = 0, offs_next = 0;

  auto body = [&](int tile, const char* kb, char* vb, char* kn, char* vn) {
    __builtin_amdgcn_sched_barrier(0);
    if (tile + 1 < t_end) {
      if constexpr (PAGE16) {
        const int at = (tile + 1 - t_begin) % 32;
        if (at == 0) {
          offs = offs_next;
          offs_next = load_offsets(tile + 33);
        }
        load_block(offs, at, kn, vn);
      } else {
        offs = offs_next;
        offs_next = load_offsets(tile + 2);
        load_block(offs, 0, kn, vn);
      }
      __builtin_amdgcn_sched_barrier(0);
      // all but the 2 NL loads of the next block are done
      __builtin_amdgcn_s_waitcnt(0xF70 | ((2 * NL) & 15) | ((2 * NL) >> 4) << 14);
    } else {
      __builtin_amdgcn_s_waitcnt(0xF70);
    }
    __builtin_amdgcn_sched_barrier(0);
    const int tb = tile * kTile + wave * kBlock;
    uint32_t vis[C];
    const bool tail = tb + kBlock > prefix;
    if (tail) {
      // bit n: the column's row sees token tb + n
      const int j0 = tb - prefix, w = j0 >> 6, sh = j0 & 63, n = min(kv_len - tb, kBlock);
      const uint32_t inside = n == kBlock ? ~0u : (1u << n) - 1;
#pragma unroll
      for (int c = 0; c < C; ++c) {
        const uint64_t lo = w < 0 ? ~0ull : (w < A.mask_words ? masks[c][w] : 0);
        const uint64_t hi = w + 1 < 0 ? ~0ull : (w + 1 < A.mask_words ? masks[c][w + 1] : 0);
        vis[c] = (uint32_t)(sh ? lo >> sh | hi << (64 - sh) : lo) & inside;
      }
      // 0 * V is NaN where V is not finite: V behind the last token is set to
      // zero, and so are infinities and NaN of tree tokens, which go to the
      // outputs of the rows that see them by themselves
      char* v0 = vb + wave * kBlock * RB;
      bool found = false;
#pragma unroll
      for (int j = 0; j < NL; ++j) {
        const int nn = j * TPI + lane / CPR;
        u32x4* p = reinterpret_cast<u32x4*>(v0 + (j * kWave + lane) * 16);
        if (nn >= n) {
          *p = u32x4{0u, 0u, 0u, 0u};
        } else if (nn + tb >= prefix) {
          const u32x4 x = *p;
#pragma unroll
          for (int e = 0; e < 4; ++e) found = found || nonfinite16<T>(x[e]) || nonfinite16<T>(x[e] >> 16);
        }
      }
      if (__builtin_amdgcn_ballot_w64(found) != 0) {
        for (int nn = max(0, prefix - tb); nn < n; ++nn) {
#pragma unroll
          for (int a = 0; a < NA; ++a) {
            u32x2* p = reinterpret_cast<u32x2*>(v0 + nn * RB + ((2 * a + grp / 2) ^ swz_v(nn)) * 16 + (grp % 2) * 8);
            u32x2 x = *p;
            u32x2 keep = x;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const uint32_t b = i % 2 ? x[i / 2] >> 16 : x[i / 2] & 0xffffu;
              if (nonfinite16<T>(b)) {
                float f, unused;
                unpack2<T>(b, f, unused);
#pragma unroll
                for (int c = 0; c < C; ++c)
                  if (vis[c] >> nn & 1) acc[c][a][i] += f;
                keep[i / 2] &= i % 2 ? 0x0000ffffu : 0xffff0000u;
              }
            }
            // (the 16 lanes of a group write the same values)
            *p = keep;
          }
        }
      }
    }

    f32x4 s[C][2];
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
      for (int b = 0; b < 2; ++b) s[c][b] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      u32x4 ka[2];
#pragma unroll
      for (int b = 0; b < 2; ++b) ka[b] = *reinterpret_cast<const u32x4*>(kb + kaddr[ks] + b * 16 * RB);
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int c = 0; c < C; ++c) s[c][b] = mfma32<T>(ka[b], qb[c][ks], s[c][b]);
    }
    if (tail) {
#pragma unroll
      for (int c = 0; c < C; ++c)
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            s[c][b][i] = vis[c] >> (b * 16 + 4 * grp + i) & 1 ? s[c][b][i] : -INFINITY;
    }
    float mx[C];
    bool rose = false;
#pragma unroll
    for (int c = 0; c < C; ++c) {
      float v = -INFINITY;
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int i = 0; i < 4; ++i) v = fmaxf(v, s[c][b][i]);
      mx[c] = v * sc;
      rose |= mx[c] > m[c] + S::kLag;
    }
    if (__builtin_amdgcn_ballot_w64(rose) != 0) {
#pragma unroll
      for (int c = 0; c < C; ++c) {
        const float mn = fmaxf(m[c], column_max(mx[c]));
        const float alpha = fast_exp2(m[c] - (mn == -INFINITY ? 0.f : mn));
        m[c] = mn;
        l[c] *= alpha;
#pragma unroll
        for (int a = 0; a < NA; ++a)
#pragma unroll
          for (int i = 0; i < 4; ++i) acc[c][a][i] *= alpha;
      }
    }
    u32x4 pb[C][NPP];
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const float mu = (m[c] == -INFINITY ? 0.f : m[c]) - S::kShift;
      float ps = 0.f;
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float e = fast_exp2(__builtin_fmaf(s[c][b][i], sc, -mu));
          s[c][b][i] = e;
          ps += e;
        }
      l[c] += ps;  // per lane; the column's lanes meet after the last block
      // P^T as the B operand: k = 8 grp + e is token 4 grp + e % 4 of block e / 4
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const f32x4 src = s[c][e / 2];
        const float p0 = src[(e % 2) * 2], p1 = src[(e % 2) * 2 + 1];
        const uint32_t hw = pack2_hw<T>(p0, p1);
        pb[c][0][e] = hw;
        if constexpr (NPP == 2) {
          float h0, h1;
          unpack2<T>(hw, h0, h1);
          pb[c][NPP - 1][e] = pack2_hw<T>(p0 - h0, p1 - h1);
        }
      }
    }
#pragma unroll
    for (int a = 0; a < NA; ++a) {
      const u32x2 v0 = read_tr(vb + vaddr[a]), v1 = read_tr(vb + vaddr[a] + 16 * RB);
      const u32x4 va = u32x4{v0[0], v0[1], v1[0], v1[1]};
#pragma unroll
      for (int pl = 0; pl < NPP; ++pl)
#pragma unroll
        for (int c = 0; c < C; ++c) acc[c][a] = mfma32<T>(va, pb[c][pl], acc[c][a]);
    }
  };

  if (t_begin < t_end && kv_len > 0) {
    offs = load_offsets(t_begin);
    offs_next = load_offsets(t_begin + (PAGE16 ? 32 : 1));
    load_block(offs, 0, s_k0, s_v0);
    int tile = t_begin;
    for (; tile + 2 <= t_end; tile += 2) {
      body(tile, s_k0, s_v0, s_k1, s_v1);
      body(tile + 1, s_k1, s_v1, s_k0, s_v0);
    }
    if (tile < t_end) body(tile, s_k0, s_v0, s_k1, s_v1);
  }

  // the waves' states meet: outputs in one buffer per wave, rows' 16-byte chunks permuted
  __syncthreads();
  float* mine = reinterpret_cast<float*>(wave == 0 ? s_k0 : wave == 1 ? s_v0 : wave == 2 ? s_k1 : s_v1);
#pragma unroll
  for (int c = 0; c < C; ++c) {
    float sum = l[c];
    sum += __shfl_xor(sum, 16);
    sum += __shfl_xor(sum, 32);
    const int pr = c * 16 + lr;
#pragma unroll
    for (int a = 0; a < NA; ++a) *reinterpret_cast<f32x4*>(mine + pr * D + ((a * 4 + grp) ^ lr) * 4) = acc[c][a];
    if (grp == 0) {
      s_ml[wave][pr][0] = m[c];
      s_ml[wave][pr][1] = sum;
    }
  }
  __syncthreads();
  constexpr int LPR = D / 4;  // lanes of a row, four dims each
  const int ch = threadIdx.x % LPR;
  float* part = A.part + ((int64_t)index * hkv + h) * kPartFloats;
  for (int pr = threadIdx.x / LPR; pr < R; pr += NT / LPR) {
    const int row = it.row0 + pr;
    if (row >= n_rows) break;
    float top = -INFINITY;
#pragma unroll
    for (int w = 0; w < W; ++w) top = fmaxf(top, s_ml[w][pr][0]);
    const float ref = top == -INFINITY ? 0.f : top;
    float sum = 0.f;
    f32x4 o = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < W; ++w) {
      const float wt = fast_exp2(s_ml[w][pr][0] - ref);
      const char* buf = w == 0 ? s_k0 : w == 1 ? s_v0 : w == 2 ? s_k1 : s_v1;
      const f32x4 x = *reinterpret_cast<const f32x4*>(buf + (pr * D + (ch ^ (pr & 15)) * 4) * 4);
      sum = __builtin_fmaf(s_ml[w][pr][1], wt, sum);
#pragma unroll
      for (int i = 0; i < 4; ++i) o[i] = __builtin_fmaf(x[i], wt, o[i]);
    }
    if (it.parts > 1) {
      *reinterpret_cast<f32x4*>(part + pr * D + ch * 4) = o;
      if (ch == 0) *reinterpret_cast<f32x2*>(part + R * D + pr * 2) = f32x2{top, sum};
    } else {
      store_row<T>(A, rq, h, row, ch * 4, o, top, sum, ch == 0);
    }
  }
}

// The parts of a row, in order: D / 4 lanes per row, four dims each.
template <typename T, int D>
__global__ __launch_bounds__(256) void merge_kernel(Args A, int rows) {
  if (!plan_fits(A)) return;
  const int hkv = A.want.hkv, h = blockIdx.x % hkv, index = blockIdx.x / hkv;
  if (index >= A.header->num_blocks) return;
  const RowBlock b = A.blocks[index];
  if (b.parts <= 1) return;
  const Request rq = A.requests[b.request];
  constexpr int LPR = D / 4;
  const int pr = blockIdx.y * (256 / LPR) + threadIdx.x / LPR, ch = threadIdx.x % LPR;
  const int row = b.row0 + pr, g = A.want.hq / hkv;
  if (pr >= rows || row >= rq.tree * g) return;
  const int64_t size = (int64_t)rows * (D + 2);
  const float* p = A.part + ((int64_t)b.slot * hkv + h) * size;
  const int64_t step = (int64_t)b.step * hkv * size;
  const float* ml = p + rows * D + pr * 2;
  float top = -INFINITY;
  for (int i = 0; i < b.parts; ++i) top = fmaxf(top, ml[i * step]);
  const float ref = top == -INFINITY ? 0.f : top;
  float sum = 0.f;
  f32x4 o = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll 8
  for (int i = 0; i < b.parts; ++i) {
    const f32x2 own = *reinterpret_cast<const f32x2*>(ml + i * step);
    const f32x4 x = *reinterpret_cast<const f32x4*>(p + i * step + pr * D + ch * 4);
    const float wt = fast_exp2(own[0] - ref);
    sum = __builtin_fmaf(own[1], wt, sum);
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = __builtin_fmaf(x[e], wt, o[e]);
  }
  store_row<T>(A, rq, h, row, ch * 4, o, top, sum, ch == 0);
}

template <typename T, int D, int C>
int launch(const Args& a, const Layout& l, hipStream_t s) {
  const int hkv = a.want.hkv;
  const int64_t grid = 8 % hkv == 0 ? 8ll * ((l.max_items + 8 / hkv - 1) / (8 / hkv)) : (int64_t)l.max_items * hkv;
  constexpr int threads = D == 256 ? 128 : 256;
  if (a.want.page_size % 16 == 0)
    hipLaunchKernelGGL((tree_kernel<T, D, C, true>), dim3((unsigned)grid), dim3(threads), 0, s, a);
  else
    hipLaunchKernelGGL((tree_kernel<T, D, C, false>), dim3((unsigned)grid), dim3(threads), 0, s, a);
  PL_LAUNCH_CHECK("tree_kernel");
  const int per = 256 / (D / 4);
  hipLaunchKernelGGL((merge_kernel<T, D>), dim3((unsigned)(l.max_blocks * hkv), (l.rows + per - 1) / per), dim3(256), 0,
                     s, a, l.rows);
  PL_LAUNCH_CHECK("tree merge_kernel");
  return ok();
}

template <typename T, int D>
int launch_cols(const Args& a, const Layout& l, hipStream_t s) {
  if (l.rows == 16) return launch<T, D, 1>(a, l, s);
  if (l.rows == 32) return launch<T, D, 2>(a, l, s);
  if constexpr (D != 256) return launch<T, D, 4>(a, l, s);
  return fail(PL_ERR_UNSUPPORTED, "tree rows %d", l.rows);
}

template <typename T>
int launch_dim(const Args& a, const Layout& l, hipStream_t s) {
  switch (a.want.head_dim) {
    case 64: return launch_cols<T, 64>(a, l, s);
    case 128: return launch_cols<T, 128>(a, l, s);
    default: return launch_cols<T, 256>(a, l, s);
  }
}

// What both calls need of their sizes; PL_OK or the failure.
inline int check_sizes(int batch, int tokens, int max_tree, int indices_capacity, int hq, int hkv, int head_dim,
                       int page_size) {
  if (batch < 0 || tokens < 0 || max_tree < 0 || indices_capacity < 0)
    return fail(PL_ERR_INVALID, "batch, tokens, max_tree and indices_capacity must be >= 0");
  if (hkv <= 0 || hq <= 0 || hq % hkv)
    return fail(PL_ERR_INVALID, "num_qo_heads (%d) must be a multiple of num_kv_heads (%d)", hq, hkv);
  if (head_dim != 64 && head_dim != 128 && head_dim != 256)
    return fail(PL_ERR_UNSUPPORTED, "tree head_dim %d not built (64, 128, 256)", head_dim);
  if (page_size <= 0 || page_size > 65536)
    return fail(PL_ERR_INVALID, "page_size must be in [1, 65536] (got %d)", page_size);
  if (batch > kMaxRequests) return fail(PL_ERR_UNSUPPORTED, "batch %d exceeds %d requests", batch, kMaxRequests);
  if (max_tree > tokens) return fail(PL_ERR_INVALID, "max_tree %d exceeds the %d tokens", max_tree, tokens);
  // row numbers, grids and mask words stay below 2^31
  if ((int64_t)tokens * hq > (1 << 28) || (int64_t)tokens * ((max_tree + 63) / 64) > INT32_MAX)
    return fail(PL_ERR_UNSUPPORTED, "%d tree tokens of %d heads are too many", tokens, hq);
  if (hkv > 65536) return fail(PL_ERR_UNSUPPORTED, "%d kv heads are too many", hkv);
  return PL_OK;
}

}  // namespace tree
}  // namespace pl

using namespace pl;
using namespace pl::tree;

extern "C" size_t pl_tree_plan_size(int batch, int tokens, int max_tree, int indices_capacity, int num_qo_heads,
                                    int num_kv_heads, int head_dim) {
  if (check_sizes(batch, tokens, max_tree, indices_capacity, num_qo_heads, num_kv_heads, head_dim, 1) != PL_OK) return 0;
  return layout(batch, tokens, max_tree, indices_capacity, num_qo_heads, num_kv_heads, head_dim).bytes;
}

extern "C" size_t pl_tree_workspace_size(int batch, int tokens, int max_tree, int num_qo_heads, int num_kv_heads,
                                         int head_dim) {
  if (check_sizes(batch, tokens, max_tree, 0, num_qo_heads, num_kv_heads, head_dim, 1) != PL_OK) return 0;
  const Layout l = layout(batch, tokens, max_tree, 0, num_qo_heads, num_kv_heads, head_dim);
  return (size_t)l.max_items * num_kv_heads * l.rows * (head_dim + 2) * sizeof(float);
}

extern "C" int pl_tree_plan(const int32_t* qo_indptr, const int32_t* kv_indptr, const int32_t* kv_indices,
                            int num_indices, const int32_t* kv_last_page_len, int batch, int tokens, int max_tree,
                            const int32_t* tree_parents, const uint8_t* tree_mask, int64_t mask_ld, int num_qo_heads,
                            int num_kv_heads, int head_dim, int page_size, int parts, int indices_capacity, void* plan,
                            size_t plan_bytes, void* stream) {
  if (int st = check_sizes(batch, tokens, max_tree, indices_capacity, num_qo_heads, num_kv_heads, head_dim, page_size))
    return st;
  if (batch == 0 || tokens == 0) return ok();
  if (num_indices < 0 || num_indices > indices_capacity)
    return fail(PL_ERR_INVALID, "num_indices (%d) must be in [0, indices_capacity = %d]", num_indices,
                indices_capacity);
  if (!qo_indptr || !kv_indptr || !kv_last_page_len || !plan || (num_indices > 0 && !kv_indices))
    return fail(PL_ERR_INVALID, "null pointer argument");
  if (!tree_parents == !tree_mask) return fail(PL_ERR_INVALID, "give tree_parents or tree_mask, and not both");
  if (tree_mask && mask_ld < max_tree)
    return fail(PL_ERR_INVALID, "mask_ld (%lld) must be at least max_tree (%d)", (long long)mask_ld, max_tree);
  if (parts < 0 || parts > kCandidates)
    return fail(PL_ERR_INVALID, "parts must be in [0, %d] (got %d)", kCandidates, parts);
  if ((uintptr_t)plan % 16) return fail(PL_ERR_INVALID, "plan must be 16-byte aligned");
  const Layout l = layout(batch, tokens, max_tree, indices_capacity, num_qo_heads, num_kv_heads, head_dim);
  if (plan_bytes < l.bytes) return fail(PL_ERR_WORKSPACE, "tree plan of %zu bytes < %zu needed", plan_bytes, l.bytes);
  char* base = (char*)plan;
  PlanArgs a{};
  a.qo_indptr = qo_indptr;
  a.kv_indptr = kv_indptr;
  a.kv_indices = kv_indices;
  a.kv_last = kv_last_page_len;
  a.parents = tree_parents;
  a.mask = tree_mask;
  a.mask_ld = mask_ld;
  a.header = (Header*)base;
  a.requests = (Request*)(base + l.requests);
  a.blocks = (RowBlock*)(base + l.blocks);
  a.items = (Item*)(base + l.items);
  a.masks = (uint64_t*)(base + l.masks);
  a.indices = (int32_t*)(base + l.indices);
  a.batch = batch;
  a.tokens = tokens;
  a.max_tree = max_tree;
  a.indices_count = num_indices;
  a.indices_capacity = indices_capacity;
  a.hq = num_qo_heads;
  a.hkv = num_kv_heads;
  a.head_dim = head_dim;
  a.page_size = page_size;
  a.rows = l.rows;
  a.tile = tile_of(head_dim);
  a.slots = l.slots;
  a.max_items = l.max_items;
  a.max_blocks = l.max_blocks;
  a.mask_words = l.mask_words;
  a.parts_fixed = parts;
  const int64_t side = std::max<int64_t>(num_indices, (int64_t)tokens * l.mask_words);
  const int grid = 1 + (int)std::min<int64_t>(255, (side + kPlanThreads - 1) / kPlanThreads);
  hipLaunchKernelGGL(plan_kernel, dim3(grid), dim3(kPlanThreads), 0, (hipStream_t)stream, a);
  PL_LAUNCH_CHECK("tree plan_kernel");
  return ok();
}

extern "C" int pl_tree_run(const void* q, int64_t q_stride_t, int64_t q_stride_h, const void* k_cache,
                           const void* v_cache, int64_t page_stride, int64_t token_stride, int64_t head_stride,
                           int64_t num_pages, void* o, int64_t o_stride_t, int64_t o_stride_h, float* lse, int batch,
                           int tokens, int max_tree, int num_qo_heads, int num_kv_heads, int head_dim, int page_size,
                           float sm_scale, int dtype, const void* plan, size_t plan_bytes, int indices_capacity,
                           void* workspace, size_t workspace_bytes, void* stream) {
  if (int st = check_sizes(batch, tokens, max_tree, indices_capacity, num_qo_heads, num_kv_heads, head_dim, page_size))
    return st;
  if (dtype != PL_DTYPE_BF16 && dtype != PL_DTYPE_F16)
    return fail(PL_ERR_UNSUPPORTED, "tree attention dtype must be F16 or BF16 (got %d)", dtype);
  if (batch == 0 || tokens == 0 || max_tree == 0) return ok();
  if (!q || !k_cache || !v_cache || !o || !plan || !workspace) return fail(PL_ERR_INVALID, "null pointer argument");
  if (num_pages <= 0) return fail(PL_ERR_INVALID, "num_pages must be > 0");
  const int64_t strides[] = {q_stride_t, q_stride_h, page_stride, token_stride, head_stride};
  for (int64_t st : strides)
    if (st % 8) return fail(PL_ERR_INVALID, "q and cache strides must be multiples of 8 elements");
  if (o_stride_t % 4 || o_stride_h % 4) return fail(PL_ERR_INVALID, "o strides must be multiples of 4 elements");
  const void* ptrs[] = {q, k_cache, v_cache, plan, workspace};
  for (const void* p : ptrs)
    if ((uintptr_t)p % 16)
      return fail(PL_ERR_INVALID, "q, the caches, the plan and the workspace must be 16-byte aligned");
  if ((uintptr_t)o % 8) return fail(PL_ERR_INVALID, "o must be 8-byte aligned");
  const Layout l = layout(batch, tokens, max_tree, indices_capacity, num_qo_heads, num_kv_heads, head_dim);
  if (plan_bytes < l.bytes) return fail(PL_ERR_WORKSPACE, "tree plan of %zu bytes < %zu needed", plan_bytes, l.bytes);
  const size_t need = (size_t)l.max_items * num_kv_heads * l.rows * (head_dim + 2) * sizeof(float);
  if (workspace_bytes < need)
    return fail(PL_ERR_WORKSPACE, "tree workspace of %zu bytes < %zu needed", workspace_bytes, need);
  const char* base = (const char*)plan;
  Args a{};
  a.q = (const char*)q;
  a.k = (const char*)k_cache;
  a.v = (const char*)v_cache;
  a.o = (char*)o;
  a.lse = lse;
  a.part = (float*)workspace;
  a.header = (const Header*)base;
  a.requests = (const Request*)(base + l.requests);
  a.blocks = (const RowBlock*)(base + l.blocks);
  a.items = (const Item*)(base + l.items);
  a.masks = (const uint64_t*)(base + l.masks);
  a.indices = (const int32_t*)(base + l.indices);
  a.q_st = q_stride_t;
  a.q_sh = q_stride_h;
  a.o_st = o_stride_t;
  a.o_sh = o_stride_h;
  a.page_stride = page_stride;
  a.token_stride = token_stride;
  a.head_stride = head_stride;
  a.num_pages = num_pages;
  a.want.batch = batch;
  a.want.tokens = tokens;
  a.want.max_tree = max_tree;
  a.want.indices_capacity = indices_capacity;
  a.want.hq = num_qo_heads;
  a.want.hkv = num_kv_heads;
  a.want.head_dim = head_dim;
  a.want.page_size = page_size;
  a.max_items = l.max_items;
  a.max_blocks = l.max_blocks;
  a.mask_words = l.mask_words;
  // the kernel takes maxima before scaling: a positive scale (a zero one as
  // one far below any score's rounding), the sign moved into q
  const float s2 = sm_scale * 1.44269504088896340736f;
  a.scale_log2 = std::max(s2 < 0 ? -s2 : s2, 1e-30f);
  a.q_flip = s2 < 0 ? 0x80008000u : 0u;
  return dtype == PL_DTYPE_BF16 ? launch_dim<bf16_t>(a, l, (hipStream_t)stream)
                                : launch_dim<f16_t>(a, l, (hipStream_t)stream);
}
