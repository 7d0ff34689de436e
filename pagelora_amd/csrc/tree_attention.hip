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
// and packs the masks into 64-bit words.  A row block is up to 64 rows (tree
// token, head of the GQA group) of a request.  The kv tiles of all row blocks,
// one after another, are dealt out in equal shares to as many slots as the chip
// holds workgroups (per kv head), so that all of them end together however
// ragged the batch is; a workgroup takes what its share holds in turn.  Where a
// request has several row blocks, its kv range is cut into chunks of a share and
// a chunk's row blocks follow one another: neighbouring slots read the same
// pages at the same time, and find them in the L2.
//
// A tile is four blocks (two at head_dim 256) of 32 tokens.  A wave, or two of 32
// rows each, works on a block of every tile, in LDS buffers of its own that are
// filled straight from the pages while the block before is worked on, and waits
// for no other block's waves until the row block ends.  Few rows then cost few
// instructions per byte, and one pass over the cache serves all rows of a block.
// S^T = K Q^T keeps a query per lane; the probabilities are the B operand of
// O^T += V^T P^T as they lie, and V comes out of LDS transposed.  The blocks'
// states meet in LDS at the row block's end, and the parts of row blocks that
// several slots share in merge_kernel, in order.
//
// Infinities and NaN in V would spoil the products of rows that do not see them, and
// 0 times an infinity those of rows that do.  Nodes' are taken out of V in LDS; where
// they are found, or an output is NaN, the row block's V is looked through once more
// at its end, and what a row sees of them is its output (see_nonfinite).
//
// Measured (head_dim 128, GQA 4, bf16 unless said otherwise; tree_kernel + merge_kernel):
//   1 x 8 nodes behind 2048     9 + 4 us: dependent round trips (the place, the
//                               page ids, the pages) and two launches
//   1 x 64 behind 32768         81 .. 87 + 6 us, 34 GFLOP, 0.4 PFLOP/s: four row blocks of
//                               the same pages, matrix and vector issue; 2 x as many
//                               matrix operations with the planes of P
//   23 ragged, up to 4099, GQA 7  45 + 7 us: 12 tiles and the starts and
//                               ends of ~3 row blocks per slot
//   8 x 32 behind 4096, no GQA, fp16  92 + 5 us, 5.9 TB/s: HBM (6.4 without any arithmetic)
//   64 x 16 behind 2048 .. 8192  253 .. 270 + 8 us, 5.2 TB/s: HBM, row blocks' starts;
//                               279 in all with pages of 8 tokens, 285 with pages of 1
//   640 x 16 behind 112         177 us in all: ~8 us per row block of one tile
// Tried with two planes of P, and slower: 128 and 256 rows per row block, which read a
// page once for all (80 - 91 us instead of 78 at 1 x 64); the next block's scores beside
// this one's softmax in one wave (no faster at 1 x 64, 59 - 70 us instead of 55 at 23
// requests: registers spill and every row block computes one block of scores more); the
// next row block's first loads while this one's states meet in half of the LDS (no faster).
#include <algorithm>
#include <type_traits>

#include "pl_common.h"

namespace pl {
namespace tree {

constexpr int kWave = 64;
constexpr int kBlock = 32;        // kv tokens of a wave per tile
constexpr int kMaxRequests = 4096;
constexpr int kMaxLen = 1 << 30;
constexpr int kMagic = 0x54524545;
constexpr int kPlanThreads = 256;
// What a row block costs a slot beside its tiles, in tiles: its first loads, its
// blocks' states that meet.  Dealt out with them, 23 ragged requests take 50 us
// instead of 57 (1: 55, 3 and 4: 51).
constexpr int kSetup = 2;

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef short i16x4 __attribute__((ext_vector_type(4)));
typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned int u32x2 __attribute__((ext_vector_type(2)));
typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));

// What a plan was made for, then what it holds.
struct alignas(64) Header {
  int32_t magic, batch, tokens, max_tree, indices_capacity, hq, hkv, head_dim, page_size;
  int32_t num_requests, num_slots, num_shared, chunk_per_slot, setup;
  int64_t share;     // tiles of a slot
  uint64_t indices;  // the address of the page ids: in the plan or apart from it
};
static_assert(sizeof(Header) == 128, "the plan's header");
// A request with nodes: `prefix` tokens before them, `tree` of them worked on.  Its
// work is tiles x blocks (row blocks), from `base` of all work on: chunk after chunk
// of its tiles, of a chunk row block after row block.  The first `setup` tiles are
// none and stand for what a row block costs beside its tiles.  The first `longer`
// chunks have chunk_len + 1 tiles, the others chunk_len.
// Either every chunk of a row block is a slot's (`base` and all work then count
// those), or only requests of several row blocks have several chunks, none less
// than a share.
struct Request {
  int32_t q_begin, tree, prefix, page_begin, kv_len, blocks, chunks, chunk_len, longer, index;
  int64_t base;
};
// A place in the work: of a row block (`block`) in a chunk, after `tile` tiles of
// it.  Of a row block that slots share: in `tile` the slot of its first part, in
// `parts` the slots of its one chunk, times two, and whether the first one's
// second partial result is of it.
struct Place {
  Request rq;
  int32_t chunk, block, tile, parts;
};
static_assert(sizeof(Place) == 64, "one load");

// ------------------------------------------------------- sizes and layout ---
// Rows of a row block: as few as the widest tree needs.
constexpr int rows_of(int64_t rows) { return rows <= 16 ? 16 : rows <= 32 ? 32 : 64; }
// Waves of a block: their rows' outputs and queries stay in registers.
constexpr int ranks_of(int rows) { return rows == 64 ? 2 : 1; }
// Blocks of a tile: two buffers of their K and V fill 128 KiB of LDS (64 at head_dim 64).
constexpr int blocks_of(int head_dim) { return head_dim == 256 ? 2 : 4; }
constexpr int tile_of(int head_dim) { return kBlock * blocks_of(head_dim); }
constexpr int threads_of(int rows, int head_dim) { return kWave * ranks_of(rows) * blocks_of(head_dim); }

// Workgroups per kv head that run at once: one per CU by their LDS (two at
// head_dim 64, where 64 rows' registers allow one again).
inline int slots_of(int rows, int hkv, int head_dim) {
  return std::max(1, (head_dim == 64 && rows < 64 ? 512 : 256) / hkv);
}

struct Layout {
  int rows, slots, mask_words;
  size_t requests, first, shared, masks, indices, bytes;  // offsets, then the size
};

inline Layout layout(int batch, int tokens, int max_tree, int indices_capacity, int hq, int hkv, int head_dim) {
  Layout l{};
  l.rows = rows_of((int64_t)max_tree * (hq / hkv));
  l.slots = slots_of(l.rows, hkv, head_dim);
  l.mask_words = (max_tree + 63) / 64;
  size_t at = sizeof(Header);
  l.first = at;  // where each slot begins
  at += sizeof(Place) * (size_t)l.slots;
  l.shared = at;  // the row blocks that slots share, by the slot in which they begin
  at += sizeof(Place) * (size_t)l.slots;
  l.requests = at;
  at += align_up(sizeof(Request) * (size_t)batch, 64);
  l.masks = at;
  at += align_up(sizeof(uint64_t) * (size_t)tokens * l.mask_words, 64);
  l.indices = at;
  at += align_up(sizeof(int32_t) * (size_t)indices_capacity, 64);
  l.bytes = at;
  return l;
}

// A slot leaves at most two partial results: of the row block it takes over and
// of the one it hands on.
inline size_t workspace_bytes(const Layout& l, int hkv, int head_dim) {
  return (size_t)l.slots * 2 * hkv * l.rows * (head_dim + 2) * sizeof(float);
}

// ------------------------------------------------------------------- plan ---
struct PlanArgs {
  const int32_t *qo_indptr, *kv_indptr, *kv_indices, *kv_last, *parents;
  const uint8_t* mask;
  int64_t mask_ld;
  Header* header;
  Request* requests;
  Place *first, *shared;
  uint64_t* masks;
  int32_t* indices;
  Header want;
  int indices_count;
  int rows, tile, slots, mask_words;
  int min_share;
};

// Request r, every entry of the tables brought into its range.
__device__ __forceinline__ Request read_request(const PlanArgs& A, int r) {
  Request q{};
  q.q_begin = min(max(A.qo_indptr[r], 0), A.want.tokens);
  const int nodes = min(max(A.qo_indptr[r + 1], q.q_begin), A.want.tokens) - q.q_begin;
  q.tree = min(nodes, A.want.max_tree);  // the first of them
  q.page_begin = min(max(A.kv_indptr[r], 0), A.indices_count);
  const int pages = min(max(A.kv_indptr[r + 1], q.page_begin), A.indices_count) - q.page_begin;
  const int last = min(max(A.kv_last[r], 1), A.want.page_size);
  const int64_t len = pages > 0 ? (int64_t)(pages - 1) * A.want.page_size + last : 0;
  q.kv_len = (int)min(len, (int64_t)kMaxLen);
  q.prefix = max(0, q.kv_len - nodes);
  q.chunks = 1;
  q.chunk_len = max(1, (q.kv_len + A.tile - 1) / A.tile);
  q.blocks = (int)(((int64_t)q.tree * (A.want.hq / A.want.hkv) + A.rows - 1) / A.rows);
  return q;
}

// The chunk's first tile, and its tiles.
__device__ __forceinline__ int chunk_tile(const Request& q, int chunk) {
  return chunk * q.chunk_len + min(chunk, q.longer);
}
__device__ __forceinline__ int chunk_tiles(const Request& q, int chunk) { return q.chunk_len + (chunk < q.longer); }

// The place at x of the request's own work; `single`: the x-th chunk of a row block.
__device__ __forceinline__ Place place_at(const Request& q, int64_t x, bool single) {
  Place p{};
  p.rq = q;
  if (single) {
    p.chunk = (int)(x / q.blocks);
    p.block = (int)(x % q.blocks);
    return p;
  }
  const int64_t longer = (int64_t)q.longer * (q.chunk_len + 1) * q.blocks;
  p.chunk = q.chunks == 1 ? 0
            : x < longer  ? (int)(x / ((int64_t)(q.chunk_len + 1) * q.blocks))
                          : q.longer + (int)((x - longer) / ((int64_t)q.chunk_len * q.blocks));
  const int64_t y = x - (int64_t)chunk_tile(q, p.chunk) * q.blocks;
  const int n = chunk_tiles(q, p.chunk);
  p.block = (int)(y / n);
  p.tile = (int)(y % n);
  return p;
}

// Workgroup 0 cuts the work; the others copy the page ids and pack the masks.
// Bound by workgroup 0's dependent loads and scans: 6 us at one request, 12 at 64,
// once per step.
__global__ __launch_bounds__(kPlanThreads) void plan_kernel(PlanArgs A) {
  const int tid = threadIdx.x, batch = A.want.batch;
  if (blockIdx.x > 0) {
    const int64_t step = (int64_t)(gridDim.x - 1) * kPlanThreads;
    const int64_t first = (int64_t)(blockIdx.x - 1) * kPlanThreads + tid;
    for (int64_t i = first; i < A.indices_count; i += step) A.indices[i] = A.kv_indices[i];
    // Given by parents, a thread packs a token's words from the last to the first on
    // one walk to the root; given by a mask, a thread packs a word.
    const int words = A.mask_words;
    const int64_t items = words == 0 ? 0 : (int64_t)A.want.tokens * (A.parents ? 1 : words);
    for (int64_t i = first; i < items; i += step) {
      const int t = (int)(A.parents ? i : i / words);
      int lo = 0, hi = batch;  // the request that holds token t: the last whose first token is <= t
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (A.qo_indptr[mid] <= t) lo = mid; else hi = mid;
      }
      const Request q = read_request(A, lo);
      const int node = t - q.q_begin;
      const bool on = node >= 0 && node < q.tree;
      if (A.parents) {
        int at = on ? node : -1;
        for (int w = words - 1; w >= 0; --w) {
          uint64_t bits = 0;
          while (at >= w * 64) {  // a parent is an earlier node: the walk ends
            bits |= 1ull << (at % 64);
            const int up = A.parents[q.q_begin + at];
            at = up < at ? up : -1;
          }
          A.masks[i * words + w] = bits;
        }
      } else {
        const int w = (int)(i % words), n = on ? min(q.tree - w * 64, 64) : 0;
        const uint8_t* m = A.mask + (int64_t)t * A.mask_ld + w * 64;
        uint64_t bits = 0;
        for (int j = 0; j < n; ++j) bits |= (uint64_t)(m[j] != 0) << j;
        A.masks[i] = bits;
      }
    }
    return;
  }

  // The work before each request: a thread owns a run of requests, and the
  // threads' sums are added up over the wave, then over the waves.
  __shared__ long long s_base[kMaxRequests];  // of the n-th request with nodes
  __shared__ long long s_wave[kPlanThreads / kWave];
  const int lane = tid % kWave, wave = tid / kWave;
  const int per = (batch + kPlanThreads - 1) / kPlanThreads;
  const int r0 = min(batch, tid * per), r1 = min(batch, r0 + per);
  // sums over all threads, and those before this one
  auto scan = [&](long long& before, long long& total, long long v) {
    long long upto = v;
#pragma unroll
    for (int d = 1; d < kWave; d <<= 1) {
      const long long t = __shfl_up(upto, d);
      if (lane >= d) upto += t;
    }
    if (lane == kWave - 1) s_wave[wave] = upto;
    __syncthreads();
    before = upto - v;
    total = 0;
    for (int w = 0; w < kPlanThreads / kWave; ++w) {
      if (w < wave) before += s_wave[w];
      total += s_wave[w];
    }
    __syncthreads();
  };
  long long work = 0, live = 0, blocks = 0;
  for (int r = r0; r < r1; ++r) {
    const Request q = read_request(A, r);
    work += (long long)q.chunk_len * q.blocks;
    live += q.blocks > 0;
    blocks += q.blocks;
  }
  long long base, index, total, n_live, before_blocks, n_blocks;
  scan(base, total, work);
  scan(index, n_live, live);
  scan(before_blocks, n_blocks, blocks);
  long long share = max((long long)max(A.min_share, 1), (total + A.slots - 1) / A.slots);
  // A slot for every chunk of a row block saves the slots that would work on two:
  // taken where the chunks so need no more than an eighth longer.
  bool single = false;
  for (int i = 0; i < 4 && !single; ++i) {
    const long long at = share + share * i / 24;
    long long chunks = 0, before, all;
    for (int r = r0; r < r1; ++r) {
      const Request q = read_request(A, r);
      chunks += (q.chunk_len + at - 1) / at * q.blocks;
    }
    scan(before, all, chunks);
    if (all <= A.slots) {
      single = true;
      share = at;
      base = before;
      total = all;
    }
  }
  const int setup = single ? 0 : kSetup;
  if (!single) {
    base += before_blocks * setup;
    total += n_blocks * setup;
    share = max((long long)max(A.min_share, 1), (total + A.slots - 1) / A.slots);
  }
  const int n_slots = (int)(single ? total : (total + share - 1) / share);
  for (int r = r0; r < r1; ++r) {
    Request q = read_request(A, r);
    if (q.blocks <= 0) continue;
    const long long tiles = q.chunk_len + setup;
    const long long chunks = single ? (tiles + share - 1) / share : q.blocks > 1 ? max(1ll, tiles / share) : 1;
    q.index = (int)index;
    q.base = base;
    q.chunks = (int)chunks;
    q.chunk_len = (int)(tiles / chunks);
    q.longer = (int)(tiles % chunks);
    A.requests[index] = q;
    s_base[index] = base;
    base += (single ? chunks : tiles) * q.blocks;
    ++index;
  }
  __syncthreads();
  auto locate = [&](long long x) {
    int lo = 0, hi = (int)n_live;  // the last request with base <= x
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (s_base[mid] <= x) lo = mid; else hi = mid;
    }
    return place_at(A.requests[lo], x - s_base[lo], single);
  };
  long long n_shared = 0;
  for (int s0 = 0; s0 < n_slots; s0 += kPlanThreads) {
    const int s = s0 + tid;
    Place p{};
    if (s < n_slots) {
      p = locate(single ? s : s * share);
      A.first[s] = p;
      if (single) {
        if (p.chunk > 0 || p.rq.chunks == 1) p.rq.blocks = 0;
      } else {
        // The row block at the slot's end is shared if it begins in the slot and does
        // not end there, or is one of several chunks (a chunk is no less than a share)
        const long long end = min((s + 1) * share, total);
        p = locate(end - 1);
        const long long start = end - 1 - p.tile;
        const int parts = (int)((start + chunk_tiles(p.rq, 0) - 1) / share - s) + 1;
        if (p.chunk > 0 || start < s * share || (p.rq.chunks == 1 && parts == 1)) p.rq.blocks = 0;
        p.parts = 2 * parts + (start > s * share);
      }
      p.tile = s;
    }
    long long before, all;
    scan(before, all, p.rq.blocks > 0);
    const long long at = n_shared + before;
    n_shared += all;
    if (p.rq.blocks > 0) A.shared[at] = p;
  }
  if (tid == 0) {
    Header h = A.want;
    h.num_requests = (int)n_live;
    h.num_slots = n_slots;
    h.num_shared = (int)n_shared;
    h.chunk_per_slot = single;
    h.setup = setup;
    h.share = share;
    h.indices = (uint64_t)A.indices;
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

// 16 bytes per lane from base + offset (bytes, per lane) into LDS at l + 16 lane.
// Written as asm because the compiler, which cannot tell which buffer a
// transposed LDS read is from, waits for every such load in flight before one:
// the loads of the next block would be waited for in the middle of this one.
// They have no register outputs; wait_loads() waits for them.
__device__ __forceinline__ uint32_t lds_address(char* l) {
  return uniform((int)(uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)l);
}
// ONCE: the lines go first from the caches.  Bytes that one workgroup reads alone
// stream 11 % faster so (5.8 and 6.4 TB/s); a request's row blocks that share them do
// not.  Requests that share pages (forks) lose nothing by it: 16 x 8 nodes behind 8192
// shared tokens 58 us with and without, behind 8192 of their own 94 and 106;
// 64 x 16 behind 4096 shared 149 and 148, of their own 202 and 214.
template <bool ONCE>
__device__ __forceinline__ void load_lds16(const char* base, uint32_t offset, uint32_t l) {
  if constexpr (ONCE)
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2 nt" ::"s"(l), "v"(offset), "s"(base)
                 : "memory", "m0");
  else
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(l), "v"(offset), "s"(base)
                 : "memory", "m0");
}
__device__ __forceinline__ void load_lds16(const char* address, uint32_t l) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(l), "v"(address) : "memory", "m0");
}
// All but the N newest loads are done.
template <int N> __device__ __forceinline__ void wait_loads() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

__device__ __forceinline__ u32x2 read_tr(const char* p) {
  return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) i16x4*)p));
}

// Infinities and NaN of two packed 16-bit values: the exponent is all ones.
template <typename T> __device__ __forceinline__ bool nonfinite16(uint32_t v) {
  constexpr uint32_t e = std::is_same<T, bf16_t>::value ? 0x7f80u : 0x7c00u;
  return (v & e) == e;
}

// A plane of two floats, bf16 cut towards zero, fp16 rounded to nearest; what it
// leaves stays in them.
template <typename T> __device__ __forceinline__ uint32_t plane(float& a, float& b);
template <> __device__ __forceinline__ uint32_t plane<bf16_t>(float& a, float& b) {
  const uint32_t x = __float_as_uint(a), y = __float_as_uint(b);
  a -= __uint_as_float(x & 0xffff0000u);
  b -= __uint_as_float(y & 0xffff0000u);
  return __builtin_amdgcn_perm(y, x, 0x07060302u);
}
template <> __device__ __forceinline__ uint32_t plane<f16_t>(float& a, float& b) {
  const uint32_t w = pack2_hw<f16_t>(a, b);
  a -= h_lo(w);
  b -= h_hi(w);
  return w;
}

struct Args {
  const char *q, *k, *v;
  char* o;
  float *lse, *part;
  const Header* header;
  const Request* requests;
  const Place *first, *shared;
  const uint64_t* masks;
  int64_t q_st, q_sh, o_st, o_sh, page_stride, token_stride, head_stride, num_pages;  // elements
  Header want;
  int slots, mask_words;
  int once;  // no two row blocks of a request read the same tokens
  float scale_log2;  // > 0; a negative scale negates q instead
  uint32_t q_flip;
};

// A run on a plan made for other arguments does nothing rather than read astray.
__device__ __forceinline__ bool plan_fits(const Args& A) {
  const Header& h = *A.header;
  const Header& w = A.want;
  return h.magic == w.magic && h.batch == w.batch && h.tokens == w.tokens && h.max_tree == w.max_tree &&
         h.indices_capacity == w.indices_capacity && h.hq == w.hq && h.hkv == w.hkv && h.head_dim == w.head_dim &&
         h.page_size == w.page_size && h.num_requests <= w.batch && h.num_slots <= A.slots && h.num_shared <= A.slots;
}

template <typename T> struct Softmax {
  static constexpr bool kBf16 = std::is_same<T, bf16_t>::value;
  // Probabilities enter the product as planes of the cache's type, each what the
  // one before left: three of bf16 hold the value's 24 bits, two of fp16, the first
  // rounded to nearest, all but the last of them.  So drafts are verified with the
  // precision of a decode step.  Two planes of bf16 leave 2^-17, 2.3e-2 of terms that
  // cancel to 2^-12 of themselves (three: 2.5e-3, the output's rounding).  bf16, two
  // planes -> three: 1 x 64 nodes behind 32768 81 -> 91 us, 23 ragged requests
  // 49 -> 54, 64 x 16 behind 8192 261 -> 269.
  static constexpr int kPlanes = kBf16 ? 3 : 2;
  // A column's running maximum, rounded up to a whole number, follows only scores more
  // than kLag above it, which takes the rescale out of the steady state and makes it
  // exact.
  static constexpr float kLag = kBf16 ? 8.f : 1.f;
  // Probabilities are held 2^kShift times as large.  bf16: with the lag none is above 1,
  // so that V of any size stays finite.  fp16 ends at 2^-24, and 32768 tokens of 2^-25
  // are no small part of a row: 2^14 keeps them to 2^-38, and the largest, 2^15 with
  // the lag, below fp16's 65504.
  static constexpr float kShift = kBf16 ? -8.f : 14.f;
};

// x / g: the product with 2^32 / g rounded up is the quotient or one more.
struct Group {
  uint32_t g, inverse;
  __device__ __forceinline__ explicit Group(int g_) : g(g_), inverse(0xffffffffu / g + 1) {}
  __device__ __forceinline__ int of(int x) const {
    if (g == 1) return x;
    const uint32_t n = __umulhi((uint32_t)x, inverse);
    return (int)(n - (n * g > (uint32_t)x));
  }
};

// Finishes a row: its four dims by one lane, and the row's lse by lane `first`.
template <typename T>
__device__ __forceinline__ void store_row(const Args& A, const Group& group, int q_begin, int h, int row, int dim,
                                          f32x4 o, float top, float sum, bool first) {
  const int g = group.g, node = group.of(row);
  const int64_t token = q_begin + node;
  const int head = h * g + row - node * g;
  const float inv = sum > 0.f ? 1.f / sum : (sum == 0.f ? 0.f : sum);
  T* op = (T*)A.o + token * A.o_st + (int64_t)head * A.o_sh + dim;
  *reinterpret_cast<u32x2*>(op) = u32x2{pack2<T>(o[0] * inv, o[1] * inv), pack2<T>(o[2] * inv, o[3] * inv)};
  if (A.lse && first)
    A.lse[token * A.want.hq + head] =
        sum == 0.f ? -INFINITY : (top + log2f(sum) - Softmax<T>::kShift) * 0.693147180559945309f;
}

__device__ __forceinline__ bool nonfinite(float x) { return (__float_as_uint(x) & 0x7f800000u) == 0x7f800000u; }

// A weighted sum of parts with its maximum: joins N more, those past n left out.
template <int N>
__device__ __forceinline__ void join(float& top, float& sum, f32x4& o, const f32x4 (&x)[N], const f32x2 (&own)[N], int n) {
  float here = top;
#pragma unroll
  for (int i = 0; i < N; ++i)
    if (i < n) here = fmaxf(here, own[i][0]);
  const float ref = here == -INFINITY ? 0.f : here, old = fast_exp2(top - ref);
  top = here;
  sum *= old;
#pragma unroll
  for (int e = 0; e < 4; ++e) o[e] *= old;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    if (i >= n) break;
    const float wt = fast_exp2(own[i][0] - ref);
    sum = __builtin_fmaf(own[i][1], wt, sum);
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = __builtin_fmaf(x[i][e], wt, o[e]);
  }
}
__device__ __forceinline__ bool has_nan(f32x4 o) {  // (or infinities of both signs)
  const float all = (o[0] + o[1]) + (o[2] + o[3]);
  return all != all;
}
// The same for parts that may hold infinities: a weight is above 0, also where fp32
// has it as 0, and 0 times a part's infinity is put right.
template <int N>
__device__ __forceinline__ void join_kept(float& top, float& sum, f32x4& o, const f32x4 (&x)[N], const f32x2 (&own)[N],
                                          int n) {
  const f32x4 before = o;
  join(top, sum, o, x, own, n);
  if (__builtin_expect(__builtin_amdgcn_ballot_w64(has_nan(o)) != 0, 0)) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      float f = nonfinite(before[e]) ? before[e] : 0.f;
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (i < n && nonfinite(x[i][e])) f += x[i][e];
      if (f != 0.f) o[e] = f;
    }
  }
}

template <typename T, int D, int R, bool PAGE16>
__global__ __launch_bounds__(threads_of(R, D), D == 64 || threads_of(R, D) > 256 ? 2 : 1) void tree_kernel(Args A) {
  using S = Softmax<T>;
  constexpr int NPP = S::kPlanes;
  constexpr int W = blocks_of(D);              // blocks of a tile
  constexpr int WR = ranks_of(R);              // waves of a block
  constexpr int NT = threads_of(R, D);
  constexpr int C = R / WR / 16;               // 16-row columns of a wave
  constexpr int RB = D * 2;                    // bytes of a token's row
  constexpr int CPR = D / 8;                   // 16-byte chunks of a row
  constexpr int TPI = kWave / CPR;             // tokens per load
  constexpr int NL = kBlock / TPI;             // loads of a block's K
  constexpr int JG = 16 / TPI;                 // loads of 16 tokens
  constexpr int KS = D / 32, NA = D / 16;
  constexpr int kTile = W * kBlock;
  constexpr int kK = kBlock * RB;              // bytes of a block's K, then its V
  constexpr int kStage = W * 2 * kK;
  constexpr int kMine = 2 * NL / WR;           // a wave's loads of a block: K and V, or one of them
  constexpr int kPartFloats = R * (D + 2);     // outputs [row][dim], then (max, sum) per row
  constexpr int kSwz = CPR < 16 ? CPR - 1 : 15;
  static_assert(W * R * D * 4 <= 2 * kStage, "the blocks' outputs fit the buffers");
  __shared__ __align__(16) char s_ring[2 * kStage];
  __shared__ float s_ml[W][R][2];
  __shared__ int s_turn[W * WR];
  __shared__ int s_bad[W * WR];

  const int hkv = A.want.hkv, h = blockIdx.x % hkv;
  // Workgroups go round the 8 XCDs.  Where the heads divide 8 and row blocks share
  // their pages, an XCD has one head and a run of the slots, so that the row blocks
  // of a chunk share an L2.
  int slot = blockIdx.x / hkv;
  if (!A.once && 8 % hkv == 0) {
    const int runs = 8 / hkv, per = (A.header->num_slots + runs - 1) / runs, at = slot / runs;
    slot = at < per ? slot % runs * per + at : A.slots;
  }
  // (asked for before the checks: one latency for both)
  Place pl = A.first[min(slot, A.slots - 1)];
  if (!plan_fits(A)) return;
  const int64_t share = A.header->share;
  if (slot >= A.header->num_slots) return;
  const bool single = A.header->chunk_per_slot;
  const int setup = A.header->setup;
  const int32_t* indices = gptr<const int32_t*>(A.header->indices);
  const int n_requests = A.header->num_requests;
  int64_t left = share;  // tiles of the share to come

  const int g = A.want.hq / hkv, page_size = A.want.page_size;
  const Group group(g);
  const int lane = threadIdx.x % kWave, wave = uniform(threadIdx.x / kWave);
  // The wave's block of a tile, its rows of the row block.  Two waves of a block
  // are on two SIMDs, each beside one of another block: one's softmax then runs
  // beside the other's matrix instructions.
  const int blk = wave / WR, rank = wave % WR;
  const int lr = lane % 16, grp = lane / 16;
  const float sc = A.scale_log2;

  auto swz_k = [](int n) { return n & kSwz; };
  auto swz_v = [](int n) { return CPR < 16 ? (n & kSwz) : 2 * (n & 7); };
  auto clamp_page = [&](int page) -> int64_t {
    return page < 0 ? 0 : ((int64_t)page >= A.num_pages ? A.num_pages - 1 : (int64_t)page);
  };
  // Loads: instruction j fetches tokens j TPI .. of the block, lane l chunk
  // l % CPR of token l / CPR, permuted by the token.  A wave alone fetches K (0)
  // and V (1), of two the first K and the second V.
  const bool second = rank > 0;
  uint32_t off0[JG], off1[JG];  // within 16 tokens of a page (others: within the token's row)
#pragma unroll
  for (int j = 0; j < JG; ++j) {
    const int n = j * TPI + lane / CPR;
    const uint32_t base = PAGE16 ? n * (uint32_t)A.token_stride * 2 : 0;
    off0[j] = base + ((lane % CPR) ^ (second ? swz_v(n) : swz_k(n))) * 16;
    off1[j] = base + ((lane % CPR) ^ swz_v(n)) * 16;
  }
  const char* src0 = (second ? A.v : A.k) + (int64_t)h * A.head_stride * 2;
  const char* src1 = A.v + (int64_t)h * A.head_stride * 2;
  const uint32_t ring = lds_address(s_ring + blk * 2 * kK + (second ? kK : 0));
  auto load_group = [&](auto ONCE, int64_t off, uint32_t to) {  // 16 tokens of a page
#pragma unroll
    for (int j = 0; j < JG; ++j) {
      load_lds16<decltype(ONCE)::value>(src0 + off, off0[j], to + j * kWave * 16);
      if constexpr (WR == 1) load_lds16<decltype(ONCE)::value>(src1 + off, off1[j], to + kK + j * kWave * 16);
    }
  };
  auto load_block = [&](int64_t offs, int at, int stage) {
    const uint32_t to = ring + stage * kStage;
    if constexpr (PAGE16) {
      int64_t off[2];
#pragma unroll
      for (int half = 0; half < 2; ++half)
        off[half] = (int64_t)((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)offs, at * 2 + half) |
                              (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(offs >> 32), at * 2 + half) << 32);
      // (fewer than 64 rows are one row block)
      if (R < 64 || A.once) {
        load_group(std::true_type{}, off[0], to);
        load_group(std::true_type{}, off[1], to + JG * kWave * 16);
      } else {
        load_group(std::false_type{}, off[0], to);
        load_group(std::false_type{}, off[1], to + JG * kWave * 16);
      }
    } else {
#pragma unroll
      for (int j = 0; j < NL; ++j) {
        const int64_t off = __shfl(offs, j * TPI + lane / CPR);
        load_lds16(src0 + off + off0[j % JG], to + j * kWave * 16);
        if constexpr (WR == 1) load_lds16(src1 + off + off1[j % JG], to + kK + j * kWave * 16);
      }
    }
  };

  // operand reads: K row b*16 + lr, chunk 4 ks + grp; V tokens 4 grp + lr/4
  // (+16), dims 16 a + 4 (lr % 4)
  int kaddr[KS], vaddr[NA];
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) kaddr[ks] = blk * 2 * kK + lr * RB + ((ks * 4 + grp) ^ swz_k(lr)) * 16;
#pragma unroll
  for (int a = 0; a < NA; ++a) {
    const int n = grp * 4 + lr / 4;
    vaddr[a] = blk * 2 * kK + kK + n * RB + ((2 * a + (lr % 4) / 2) ^ swz_v(n)) * 16 + (lr % 2) * 8;
  }

  // The two waves of a block meet: each leaves the number of its meetings and
  // waits for the other's.  Both work on the same blocks in the same order, so
  // they come as often, and the wait ends.
  int turn = 0;
  auto meet = [&]() {
    if constexpr (WR > 1) {
      __builtin_amdgcn_sched_barrier(0);
      ++turn;
      asm volatile("" ::: "memory");
      if (lane == 0) __hip_atomic_store(&s_turn[wave], turn, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
      const int* other = &s_turn[wave ^ 1];
      while (uniform(__hip_atomic_load(other, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP)) < turn) {
      }
      asm volatile("" ::: "memory");
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  if constexpr (WR > 1) {
    if (lane == 0) s_turn[wave] = 0;
    __syncthreads();
  }

  // What the share holds of a row block.
  struct Segment {
    int q_begin, page_begin, row0, n_rows, kv_len, prefix, n_pages, t_first, t_last, t_end, units;
    bool whole, second;
  };
  auto segment_at = [&](const Place& p) {
    const Request& rq = p.rq;
    Segment g_;
    const int c_first = chunk_tile(rq, p.chunk), c_tiles = chunk_tiles(rq, p.chunk);
    g_.q_begin = rq.q_begin;
    g_.page_begin = rq.page_begin;
    g_.row0 = p.block * R;
    g_.n_rows = rq.tree * g;
    g_.kv_len = rq.kv_len;
    g_.prefix = rq.prefix;
    g_.n_pages = (rq.kv_len + page_size - 1) / page_size;
    const int upto = single ? c_tiles : (int)min((int64_t)c_tiles, p.tile + left);
    g_.units = upto - p.tile;
    g_.t_first = max(0, c_first + p.tile - setup);
    g_.t_last = max(0, c_first + upto - setup);
    // the block's tokens: only the last tile can lie behind them
    g_.t_end = rq.kv_len <= 0 || g_.t_first == g_.t_last ? g_.t_first
               : (int64_t)(g_.t_last - 1) * kTile + blk * kBlock < rq.kv_len ? g_.t_last : g_.t_last - 1;
    g_.whole = rq.chunks == 1 && g_.units == c_tiles;
    // a slot's first partial result is of what it takes over, its second of what it hands on
    g_.second = left < share;
    return g_;
  };

  // Page ids are asked for long before their use: `id` is in flight, `rest` the
  // byte offset within the page.
  struct Offset {
    int id;
    int64_t rest;
  };
  // Of the block's tokens, one per lane.  Pages of a multiple of 16 tokens: of the
  // 16-token groups of 32 tiles; others: of a block's 32 tokens.  Behind the last
  // token it is the rest of the last page.
  auto ask_offsets = [&](const Segment& e, int tile) {
    const int t = PAGE16 ? (tile + lane / 2) * kTile + blk * kBlock + (lane % 2) * 16
                         : min(tile * kTile + blk * kBlock + lane % kBlock, e.kv_len - 1);
    const int page = t / page_size;
    return Offset{indices[e.page_begin + min(page, e.n_pages - 1)], (int64_t)(t - page * page_size) * A.token_stride};
  };
  auto offsets = [&](const Offset& o) -> int64_t { return (clamp_page(o.id) * A.page_stride + o.rest) * 2; };

  u32x4 qb[C][KS];
  Offset ask0{}, ask1{};
  uint64_t mask0[C];  // the rows' masks where they are one word
  auto ask = [&](const Segment& e) {  // queries, masks and page ids
    if (e.t_first < e.t_end) {
      ask0 = ask_offsets(e, e.t_first);
      ask1 = ask_offsets(e, e.t_first + (PAGE16 ? 32 : 1));
    }
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const int row = min(e.row0 + (rank * C + c) * 16 + lr, e.n_rows - 1);  // rows past the end repeat the last one, unstored
      const int node = group.of(row);
      mask0[c] = A.masks[(int64_t)(e.q_begin + node) * A.mask_words];
      const char* qp = A.q + ((int64_t)(e.q_begin + node) * A.q_st + (int64_t)(h * g + row - node * g) * A.q_sh) * 2 + grp * 16;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) qb[c][ks] = *reinterpret_cast<const u32x4*>(qp + ks * 64);
    }
  };

  // What the thread's rows (four dims each, by passes over the row block) see of the
  // infinities and NaN in V, from token `from` of the segment on: their outputs, since
  // a weight is above 0, however small, unless K is infinite too.  Slow, since rare:
  // 64 x 16 nodes behind 2048 .. 8192 take 1.9 ms with an infinity among each request's
  // committed tokens, and 4 % more than without with one among its nodes.
  constexpr int LPR = D / 4;  // lanes of a row, four dims each
  constexpr int P = R * LPR / NT;
  auto see_nonfinite = [&](const Segment& e, int from, f32x4 (&seen)[P]) {
    auto row_of = [&](const char* cache, int t) {
      const int page = t / page_size;
      return cache + (clamp_page(indices[e.page_begin + page]) * A.page_stride +
                      (int64_t)(t - page * page_size) * A.token_stride + (int64_t)h * A.head_stride) * 2;
    };
    auto any_nonfinite = [&](const char* p) {
      const u32x4 x = *reinterpret_cast<const u32x4*>(p);
      bool is = false;
#pragma unroll
      for (int i = 0; i < 4; ++i) is |= nonfinite16<T>(x[i]) || nonfinite16<T>(x[i] >> 16);
      return is;
    };
    const int end = min(e.t_last * kTile, e.kv_len);
#pragma unroll 1
    for (int t0 = from; t0 < end; t0 += TPI) {  // tokens of a load
      const int mine = min(t0 + lane / CPR, end - 1);
      uint64_t found = __builtin_amdgcn_ballot_w64(t0 + lane / CPR < end && any_nonfinite(row_of(A.v, mine) + lane % CPR * 16));
#pragma unroll 1
      while (found) {
        const int i = __builtin_ctzll(found) / CPR, t = t0 + i, node = t - e.prefix;
        found &= CPR * (i + 1) < 64 ? ~0ull << (CPR * (i + 1)) : 0;
        const bool no_weight = __builtin_amdgcn_ballot_w64(any_nonfinite(row_of(A.k, t) + lane % CPR * 16)) != 0;
        const u32x2 x = *reinterpret_cast<const u32x2*>(row_of(A.v, t) + threadIdx.x % LPR * 8);
#pragma unroll
        for (int k = 0; k < P; ++k) {
          const int row = min(e.row0 + k * (NT / LPR) + (int)threadIdx.x / LPR, e.n_rows - 1);
          const uint64_t* mask = A.masks + (int64_t)(e.q_begin + group.of(row)) * A.mask_words;
          if (node >= 0 && !(node / 64 < A.mask_words && (mask[node / 64] >> (node % 64) & 1))) continue;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const uint32_t b = j % 2 ? x[j / 2] >> 16 : x[j / 2] & 0xffffu;
            float f, unused;
            unpack2<T>(b, f, unused);
            if (nonfinite16<T>(b)) seen[k][j] += no_weight ? __builtin_nanf("") : f;
          }
        }
      }
    }
  };

  Segment e = segment_at(pl);
  ask(e);
  for (;;) {
    // the place behind this row block
    left -= e.units;
    bool more = !single && left > 0;
    pl.tile = 0;
    if (more && ++pl.block == pl.rq.blocks) {
      pl.block = 0;
      if (++pl.chunk == pl.rq.chunks) {
        pl.chunk = 0;
        more = pl.rq.index + 1 < n_requests;
        if (more) pl.rq = A.requests[pl.rq.index + 1];
      }
    }
    const int kv_len = e.kv_len, prefix = e.prefix, t_first = e.t_first, t_end = e.t_end;
    int64_t offs = offsets(ask0);
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
      for (int ks = 0; ks < KS; ++ks)
#pragma unroll
        for (int i = 0; i < 4; ++i) qb[c][ks][i] ^= A.q_flip;
    f32x4 acc[C][NA];
    float m[C], l[C];
#pragma unroll
    for (int c = 0; c < C; ++c) {
      m[c] = -INFINITY;
      l[c] = 0.f;
#pragma unroll
      for (int a = 0; a < NA; ++a) acc[c][a] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    bool bad = false;  // infinities and NaN were taken out of V
    if (t_first < t_end) load_block(offs, 0, 0);

    for (int tile = t_first; tile < t_end; ++tile) {
      __builtin_amdgcn_sched_barrier(0);
      const int stage = (tile - t_first) % 2;
      meet();  // both are done with the other stage
      if (tile + 1 < t_end) {
        const int at = PAGE16 ? (tile + 1 - t_first) % 32 : 0;
        if (at == 0) {
          offs = offsets(ask1);
          ask1 = ask_offsets(e, tile + (PAGE16 ? 33 : 2));
        }
        load_block(offs, at, stage ^ 1);
        __builtin_amdgcn_sched_barrier(0);
        wait_loads<kMine>();  // all but those of the next block
      } else {
        wait_loads<0>();
      }
      meet();  // the other's are done too
      __builtin_amdgcn_sched_barrier(0);
      char* kb = s_ring + stage * kStage;
      const int tb = tile * kTile + blk * kBlock;
      uint32_t vis[C];
      const bool tail = tb + kBlock > prefix;
      if (tail) {
        // bit n: the column's row sees token tb + n
        const int j0 = tb - prefix, w = j0 >> 6, sh = j0 & 63, n = min(kv_len - tb, kBlock);
        const uint32_t inside = n == kBlock ? ~0u : (1u << n) - 1;
#pragma unroll
        for (int c = 0; c < C; ++c) {
          uint64_t lo = w < 0 ? ~0ull : (w == 0 ? mask0[c] : 0), hi = w + 1 < 0 ? ~0ull : (w + 1 == 0 ? mask0[c] : 0);
          if (A.mask_words > 1) {
            const int row = min(e.row0 + (rank * C + c) * 16 + lr, e.n_rows - 1);
            const uint64_t* mask = A.masks + (int64_t)(e.q_begin + group.of(row)) * A.mask_words;
            if (w > 0 && w < A.mask_words) lo = mask[w];
            if (w >= 0 && w + 1 < A.mask_words) hi = mask[w + 1];
          }
          vis[c] = (uint32_t)(sh ? lo >> sh | hi << (64 - sh) : lo) & inside;
        }
        // 0 * V is NaN where V is not finite: V behind the last token is set to
        // zero, and so are infinities and NaN of nodes, which rows may not see
        // (see_nonfinite gives them to the rows that do).  (Looked for in two
        // halves of V: all of it at once spills registers.)
        char* v0 = kb + blk * 2 * kK + kK;
        u16x2 top2 = {0, 0};  // the largest magnitudes: not finite from infinity on
#pragma unroll
        for (int j0 = 0; j0 < NL; j0 += 4) {
          u32x4 x[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) x[j] = *reinterpret_cast<const u32x4*>(v0 + ((j0 + j) * kWave + lane) * 16);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int nn = (j0 + j) * TPI + lane / CPR;
            const uint32_t tree = nn < n && nn + tb >= prefix ? 0x7fff7fffu : 0u;
#pragma unroll
            for (int i = 0; i < 4; ++i) top2 = __builtin_elementwise_max(top2, __builtin_bit_cast(u16x2, x[j][i] & tree));
          }
        }
        constexpr int kInf = std::is_same<T, bf16_t>::value ? 0x7f80 : 0x7c00;
        const bool found = top2[0] >= kInf || top2[1] >= kInf;
        const bool any = __builtin_amdgcn_ballot_w64(found) != 0;
        bad |= any;
        if (any || n < kBlock) {
          meet();  // both have read the block's V
#pragma unroll
          for (int j = 0; j < NL; ++j) {
            const int nn = j * TPI + lane / CPR;
            u32x4* p = reinterpret_cast<u32x4*>(v0 + (j * kWave + lane) * 16);
            if (nn >= n) {
              *p = u32x4{0u, 0u, 0u, 0u};
            } else if (any && nn + tb >= prefix) {
              u32x4 x = *p;
#pragma unroll
              for (int e = 0; e < 4; ++e)
                x[e] &= (nonfinite16<T>(x[e]) ? 0u : 0xffffu) | (nonfinite16<T>(x[e] >> 16) ? 0u : 0xffff0000u);
              *p = x;
            }
          }
          meet();  // (both have written the same)
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
          const float mn = fmaxf(m[c], __builtin_ceilf(column_max(mx[c])));
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
          float p0 = src[(e % 2) * 2], p1 = src[(e % 2) * 2 + 1];
#pragma unroll
          for (int n = 0; n < NPP; ++n) pb[c][n][e] = plane<T>(p0, p1);
        }
      }
      // four independent accumulations in turn: an MFMA waits for the one before
      // it on the same accumulator
#pragma unroll
      for (int a0 = 0; a0 < NA; a0 += 2) {
        u32x4 va[2];
#pragma unroll
        for (int a = 0; a < 2; ++a) {
          const u32x2 v0 = read_tr(kb + vaddr[a0 + a]), v1 = read_tr(kb + vaddr[a0 + a] + 16 * RB);
          va[a] = u32x4{v0[0], v0[1], v1[0], v1[1]};
        }
#pragma unroll
        for (int i = 0; i < NPP; ++i)
#pragma unroll
          for (int a = 0; a < 2; ++a)
#pragma unroll
            for (int c = 0; c < C; ++c) acc[c][a0 + a] = mfma32<T>(va[a], pb[c][i], acc[c][a0 + a]);
      }
    }

    if (lane == 0) s_bad[wave] = bad;
    // the next row block's queries and page ids come while this one's states meet
    const Segment was = e;
    if (more) {
      e = segment_at(pl);
      ask(e);
    }
    // the blocks' states meet in the buffers, rows' 16-byte chunks permuted
    __syncthreads();
    float* outs = reinterpret_cast<float*>(s_ring);
#pragma unroll
    for (int c = 0; c < C; ++c) {
      float sum = l[c];
      sum += __shfl_xor(sum, 16);
      sum += __shfl_xor(sum, 32);
      const int pr = (rank * C + c) * 16 + lr;
#pragma unroll
      for (int a = 0; a < NA; ++a)
        *reinterpret_cast<f32x4*>(outs + (blk * R + pr) * D + ((a * 4 + grp) ^ lr) * 4) = acc[c][a];
      if (grp == 0) {
        s_ml[blk][pr][0] = m[c];
        s_ml[blk][pr][1] = sum;
      }
    }
    __syncthreads();
    const int ch = threadIdx.x % LPR;
    float* part = A.part + ((2 * (int64_t)slot + was.second) * hkv + h) * kPartFloats;
    // A pass over the row block; `seen` where it is not 0.  Whether there is a NaN:
    // 0 times an infinity, of a plane of a probability, a rescale or a block's weight.
    auto finish = [&](int k, const f32x4& seen) {
      const int pr = k * (NT / LPR) + threadIdx.x / LPR, row = was.row0 + pr;
      f32x4 x[W];
      f32x2 own[W];
#pragma unroll
      for (int w = 0; w < W; ++w) {
        own[w] = f32x2{s_ml[w][pr][0], s_ml[w][pr][1]};
        x[w] = *reinterpret_cast<const f32x4*>(outs + (w * R + pr) * D + (ch ^ (pr % 16)) * 4);
      }
      float top = -INFINITY, sum = 0.f;
      f32x4 o = f32x4{0.f, 0.f, 0.f, 0.f};
      join(top, sum, o, x, own, W);
      const bool nan = has_nan(o);
#pragma unroll
      for (int i = 0; i < 4; ++i) o[i] = seen[i] != 0.f ? seen[i] : o[i];
      if (row >= was.n_rows) return nan;
      if (was.whole) {
        store_row<T>(A, group, was.q_begin, h, row, ch * 4, o, top, sum, ch == 0);
      } else {
        *reinterpret_cast<f32x4*>(part + pr * D + ch * 4) = o;
        if (ch == 0) *reinterpret_cast<f32x2*>(part + R * D + pr * 2) = f32x2{top, sum};
      }
      return nan;
    };
    bool nan = false;
#pragma unroll
    for (int k = 0; k < P; ++k) nan |= finish(k, f32x4{0.f, 0.f, 0.f, 0.f});
    nan = __builtin_amdgcn_ballot_w64(nan) != 0;
    if (__builtin_expect(nan || __builtin_amdgcn_ballot_w64(s_bad[lane % (W * WR)] != 0) != 0, 0)) {
      f32x4 seen[P];
#pragma unroll
      for (int k = 0; k < P; ++k) seen[k] = f32x4{0.f, 0.f, 0.f, 0.f};
      see_nonfinite(was, max(was.t_first * kTile, nan ? 0 : was.prefix / TPI * TPI), seen);
#pragma unroll
      for (int k = 0; k < P; ++k) finish(k, seen[k]);
    }
    if (!more) return;
    __syncthreads();  // the outputs are read: the buffers may be filled again
  }
}

// The parts of a row block that slots share, in order: D / 4 lanes per row, four
// dims each.  A wave takes all parts of its rows where they are up to 8, and as
// many rows as keep 8 loads in flight; of more parts each of the workgroup's four
// waves takes every fourth of the same rows.  Bound by latency: 4 - 8 us.
template <typename T, int D>
__global__ __launch_bounds__(256) void merge_kernel(Args A, int rows) {
  constexpr int LPR = D / 4, RPW = kWave / LPR, W = 4;  // lanes of a row, rows of a wave, waves
  __shared__ f32x4 s_o[W][kWave];
  __shared__ f32x2 s_ml[W][kWave];
  const int hkv = A.want.hkv, h = blockIdx.x % hkv, index = blockIdx.x / hkv;
  const Place pl = A.shared[index];
  if (!plan_fits(A) || index >= A.header->num_shared) return;
  const int64_t share = A.header->share;
  const Request& rq = pl.rq;
  const int lane = threadIdx.x % kWave, wave = uniform(threadIdx.x / kWave), ch = lane % LPR;
  const int row0 = pl.block * rows, n_rows = min(rows, rq.tree * (A.want.hq / hkv) - row0);
  const int64_t size = (int64_t)rows * (D + 2);
  const Group group(A.want.hq / A.want.hkv);
  // One of several chunks lies in up to three slots: candidate i is slot i % 3 of
  // chunk i / 3's.
  const bool single = A.header->chunk_per_slot;
  const int candidates = single ? rq.chunks : rq.chunks > 1 ? rq.chunks * 3 : pl.parts / 2;
  auto part_at = [&](int i) -> int {  // the candidate's partial result, or -1
    if (i >= candidates) return -1;
    if (single) return 2 * (pl.tile + i * rq.blocks);
    if (rq.chunks == 1) return 2 * (pl.tile + i) + (i == 0 ? pl.parts % 2 : 0);
    const int chunk = i / 3, t0 = chunk_tile(rq, chunk), n = chunk_tiles(rq, chunk);
    const int64_t start = rq.base + (int64_t)t0 * rq.blocks + (int64_t)pl.block * n;
    const int64_t s = start / share + i % 3;
    return s * share < start + n ? (int)(2 * s + (start > s * share)) : -1;
  };
  // the next N live parts' results
  auto take = [&](auto& p, int part, uint64_t& live) {
    constexpr int N = sizeof(p) / sizeof(p[0]);
    int n = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int from = live ? __builtin_ctzll(live) : 0;
      if (live) n = i + 1;
      p[i] = live ? A.part + ((int64_t)__builtin_amdgcn_readlane(part, from) * hkv + h) * size : p[0];
      live &= live - 1;
    }
    return n;
  };

  const int all = part_at(lane);
  uint64_t live = __builtin_amdgcn_ballot_w64(all >= 0);
  if (candidates <= kWave && __builtin_popcountll(live) <= 8) {
    auto rows_at_once = [&](auto P_) {
      constexpr int P = decltype(P_)::value, G = 8 / P;
      const float* p[P];
      const int n = take(p, all, live);
      for (int r0 = (blockIdx.y * W + wave) * RPW * G; r0 < n_rows; r0 += gridDim.y * W * RPW * G) {
        f32x4 x[G][P];
        f32x2 own[G][P];
#pragma unroll
        for (int k = 0; k < G; ++k) {
          const int pr = min(r0 + k * RPW + lane / LPR, n_rows - 1);
#pragma unroll
          for (int i = 0; i < P; ++i) {
            x[k][i] = *reinterpret_cast<const f32x4*>(p[i] + pr * D + ch * 4);
            own[k][i] = *reinterpret_cast<const f32x2*>(p[i] + rows * D + pr * 2);
          }
        }
#pragma unroll
        for (int k = 0; k < G; ++k) {
          const int pr = r0 + k * RPW + lane / LPR;
          float top = -INFINITY, sum = 0.f;
          f32x4 o = f32x4{0.f, 0.f, 0.f, 0.f};
          join_kept(top, sum, o, x[k], own[k], n);
          if (pr < n_rows) store_row<T>(A, group, rq.q_begin, h, row0 + pr, ch * 4, o, top, sum, ch == 0);
        }
      }
    };
    const int n = __builtin_popcountll(live);
    if (n == 0) return;
    if (n <= 2) rows_at_once(std::integral_constant<int, 2>{});
    else if (n <= 4) rows_at_once(std::integral_constant<int, 4>{});
    else rows_at_once(std::integral_constant<int, 8>{});
    return;
  }
  for (int r0 = blockIdx.y * RPW; r0 < n_rows; r0 += gridDim.y * RPW) {
    const int pr = min(r0 + lane / LPR, n_rows - 1);
    float top = -INFINITY, sum = 0.f;
    f32x4 o = f32x4{0.f, 0.f, 0.f, 0.f};
    for (int i0 = 0; i0 < candidates; i0 += kWave * W) {
      const int mine = part_at(i0 + lane * W + wave);
      live = __builtin_amdgcn_ballot_w64(mine >= 0);
      while (live) {
        const float* p[8];
        const int n = take(p, mine, live);
        f32x4 x[8];
        f32x2 own[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          if (i >= n) break;
          x[i] = *reinterpret_cast<const f32x4*>(p[i] + pr * D + ch * 4);
          own[i] = *reinterpret_cast<const f32x2*>(p[i] + rows * D + pr * 2);
        }
        join_kept(top, sum, o, x, own, n);
      }
    }
    s_o[wave][lane] = o;
    s_ml[wave][lane] = f32x2{top, sum};
    __syncthreads();
    if (wave == 0) {
      f32x4 x[W];
      f32x2 own[W];
#pragma unroll
      for (int w = 0; w < W; ++w) {
        x[w] = s_o[w][lane];
        own[w] = s_ml[w][lane];
      }
      top = -INFINITY;
      sum = 0.f;
      o = f32x4{0.f, 0.f, 0.f, 0.f};
      join_kept(top, sum, o, x, own, W);
      if (r0 + lane / LPR < n_rows) store_row<T>(A, group, rq.q_begin, h, row0 + pr, ch * 4, o, top, sum, ch == 0);
    }
    __syncthreads();
  }
}

template <typename T, int D, int R>
int launch(const Args& a, const Layout& l, hipStream_t s) {
  const int hkv = a.want.hkv;
  const int64_t grid = ((int64_t)l.slots * hkv + 7) / 8 * 8;
  // (32-bit offsets within 16 tokens)
  if (a.want.page_size % 16 == 0 && a.token_stride >= 0 && a.token_stride < (1 << 26))
    hipLaunchKernelGGL((tree_kernel<T, D, R, true>), dim3((unsigned)grid), dim3(threads_of(R, D)), 0, s, a);
  else
    hipLaunchKernelGGL((tree_kernel<T, D, R, false>), dim3((unsigned)grid), dim3(threads_of(R, D)), 0, s, a);
  PL_LAUNCH_CHECK("tree_kernel");
  // A slot's end falls into one row block.  A workgroup for every few rows, and
  // fewer where row blocks are many: 2,048 empty ones take 5 us.
  const int g = a.want.hq / hkv, blocks = (int)(((int64_t)a.want.max_tree * g + R - 1) / R);
  const int shared = (int)std::min<int64_t>(l.slots, (int64_t)a.want.batch * blocks);
  const int rows = kWave / (D / 4), across = std::max(1, std::min(R / rows, 512 / (shared * hkv)));
  hipLaunchKernelGGL((merge_kernel<T, D>), dim3((unsigned)(shared * hkv), across), dim3(256), 0, s, a, R);
  PL_LAUNCH_CHECK("tree merge_kernel");
  return ok();
}

template <typename T, int D>
int launch_rows(const Args& a, const Layout& l, hipStream_t s) {
  if (l.rows == 16) return launch<T, D, 16>(a, l, s);
  if (l.rows == 32) return launch<T, D, 32>(a, l, s);
  return launch<T, D, 64>(a, l, s);
}

template <typename T>
int launch_dim(const Args& a, const Layout& l, hipStream_t s) {
  switch (a.want.head_dim) {
    case 64: return launch_rows<T, 64>(a, l, s);
    case 128: return launch_rows<T, 128>(a, l, s);
    default: return launch_rows<T, 256>(a, l, s);
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

inline Header wanted(int batch, int tokens, int max_tree, int indices_capacity, int hq, int hkv, int head_dim,
                     int page_size) {
  Header h{};
  h.magic = kMagic;
  h.batch = batch;
  h.tokens = tokens;
  h.max_tree = max_tree;
  h.indices_capacity = indices_capacity;
  h.hq = hq;
  h.hkv = hkv;
  h.head_dim = head_dim;
  h.page_size = page_size;
  return h;
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
  return workspace_bytes(l, num_kv_heads, head_dim);
}

namespace {
// `ids`: where the page ids go, or null: behind the rest of the plan, room for indices_capacity.
int make_plan(const int32_t* qo_indptr, const int32_t* kv_indptr, const int32_t* kv_indices, int num_indices,
              const int32_t* kv_last_page_len, int batch, int tokens, int max_tree, const int32_t* tree_parents,
              const uint8_t* tree_mask, int64_t mask_ld, int num_qo_heads, int num_kv_heads, int head_dim, int page_size,
              int min_share, int32_t* ids, int ids_capacity, int indices_capacity, void* plan, size_t plan_bytes,
              void* stream) {
  if (int st = check_sizes(batch, tokens, max_tree, indices_capacity, num_qo_heads, num_kv_heads, head_dim, page_size))
    return st;
  if (batch == 0 || tokens == 0) return ok();
  if (num_indices < 0 || num_indices > ids_capacity)
    return fail(PL_ERR_INVALID, "num_indices (%d) must be in [0, %s = %d]", num_indices,
                ids ? "ids_capacity" : "indices_capacity", ids_capacity);
  if (!qo_indptr || !kv_indptr || !kv_last_page_len || !plan || (num_indices > 0 && !kv_indices))
    return fail(PL_ERR_INVALID, "null pointer argument");
  if (!tree_parents == !tree_mask) return fail(PL_ERR_INVALID, "give tree_parents or tree_mask, and not both");
  if (tree_mask && mask_ld < max_tree)
    return fail(PL_ERR_INVALID, "mask_ld (%lld) must be at least max_tree (%d)", (long long)mask_ld, max_tree);
  if (min_share < 0) return fail(PL_ERR_INVALID, "min_share must be >= 0 (got %d)", min_share);
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
  a.first = (Place*)(base + l.first);
  a.shared = (Place*)(base + l.shared);
  a.masks = (uint64_t*)(base + l.masks);
  a.indices = ids ? ids : (int32_t*)(base + l.indices);
  a.want = wanted(batch, tokens, max_tree, indices_capacity, num_qo_heads, num_kv_heads, head_dim, page_size);
  a.indices_count = num_indices;
  a.rows = l.rows;
  a.tile = tile_of(head_dim);
  a.slots = l.slots;
  a.mask_words = l.mask_words;
  a.min_share = min_share;
  const int64_t side = std::max<int64_t>(num_indices, (int64_t)tokens * (tree_parents ? 1 : l.mask_words));
  const int grid = 1 + (int)std::min<int64_t>(255, (side + kPlanThreads - 1) / kPlanThreads);
  hipLaunchKernelGGL(plan_kernel, dim3(grid), dim3(kPlanThreads), 0, (hipStream_t)stream, a);
  PL_LAUNCH_CHECK("tree plan_kernel");
  return ok();
}
}  // namespace

extern "C" int pl_tree_plan(const int32_t* qo_indptr, const int32_t* kv_indptr, const int32_t* kv_indices,
                            int num_indices, const int32_t* kv_last_page_len, int batch, int tokens, int max_tree,
                            const int32_t* tree_parents, const uint8_t* tree_mask, int64_t mask_ld, int num_qo_heads,
                            int num_kv_heads, int head_dim, int page_size, int min_share, int indices_capacity, void* plan,
                            size_t plan_bytes, void* stream) {
  return make_plan(qo_indptr, kv_indptr, kv_indices, num_indices, kv_last_page_len, batch, tokens, max_tree, tree_parents,
                   tree_mask, mask_ld, num_qo_heads, num_kv_heads, head_dim, page_size, min_share, nullptr,
                   indices_capacity, indices_capacity, plan, plan_bytes, stream);
}

extern "C" int pl_tree_plan_ids(const int32_t* qo_indptr, const int32_t* kv_indptr, const int32_t* kv_indices,
                                int num_indices, const int32_t* kv_last_page_len, int batch, int tokens, int max_tree,
                                const int32_t* tree_parents, const uint8_t* tree_mask, int64_t mask_ld, int num_qo_heads,
                                int num_kv_heads, int head_dim, int page_size, int min_share, int32_t* ids,
                                int ids_capacity, void* plan, size_t plan_bytes, void* stream) {
  if (num_indices > 0 && !ids) return fail(PL_ERR_INVALID, "null pointer argument");
  if ((uintptr_t)ids % 4) return fail(PL_ERR_INVALID, "ids must be 4-byte aligned");
  return make_plan(qo_indptr, kv_indptr, kv_indices, num_indices, kv_last_page_len, batch, tokens, max_tree, tree_parents,
                   tree_mask, mask_ld, num_qo_heads, num_kv_heads, head_dim, page_size, min_share, ids, ids_capacity, 0,
                   plan, plan_bytes, stream);
}

extern "C" int pl_tree_run(const void* q, int64_t q_stride_t, int64_t q_stride_h, const void* k_cache,
                           const void* v_cache, int64_t page_stride, int64_t token_stride, int64_t head_stride,
                           int64_t num_pages, void* o, int64_t o_stride_t, int64_t o_stride_h, float* lse, int batch,
                           int tokens, int max_tree, int num_qo_heads, int num_kv_heads, int head_dim, int page_size,
                           float sm_scale, int dtype, const void* plan, size_t plan_bytes, int indices_capacity,
                           void* workspace, size_t workspace_size, void* stream) {
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
  const size_t need = workspace_bytes(l, num_kv_heads, head_dim);
  if (workspace_size < need)
    return fail(PL_ERR_WORKSPACE, "tree workspace of %zu bytes < %zu needed", workspace_size, need);
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
  a.first = (const Place*)(base + l.first);
  a.shared = (const Place*)(base + l.shared);
  a.masks = (const uint64_t*)(base + l.masks);
  a.q_st = q_stride_t;
  a.q_sh = q_stride_h;
  a.o_st = o_stride_t;
  a.o_sh = o_stride_h;
  a.page_stride = page_stride;
  a.token_stride = token_stride;
  a.head_stride = head_stride;
  a.num_pages = num_pages;
  a.want = wanted(batch, tokens, max_tree, indices_capacity, num_qo_heads, num_kv_heads, head_dim, page_size);
  a.slots = l.slots;
  a.mask_words = l.mask_words;
  a.once = (int64_t)max_tree * (num_qo_heads / num_kv_heads) <= l.rows;
  // the kernel takes maxima before scaling: a positive scale (a zero one as
  // one far below any score's rounding), the sign moved into q
  const float s2 = sm_scale * 1.44269504088896340736f;
  a.scale_log2 = std::max(s2 < 0 ? -s2 : s2, 1e-30f);
  a.q_flip = s2 < 0 ? 0x80008000u : 0u;
  return dtype == PL_DTYPE_BF16 ? launch_dim<bf16_t>(a, l, (hipStream_t)stream)
                                : launch_dim<f16_t>(a, l, (hipStream_t)stream);
}
