// What follows a tree's attention (gfx950): the path of the tree that the target's
// picks follow, and that path's K/V moved together in the cache.
//
// accept_kernel: node 0 is the root, whose token is already decided.  From node
// i the walk goes on to its first child whose drafted token is the target's
// pick after i (of equal drafts beside each other the first, though another may
// lead further).  The kept tokens are the picks along the path: the children's
// own tokens, then the pick after the last node.  One wave per request; a tree
// of up to 64 nodes lies one node per lane, and a step is two lane reads and a
// ballot; of more nodes a step is a round trip to the caches.  Bound by latency,
// the loads and a launch: 1.7 us for one tree of 8 nodes, 3.3 for 256 of up to 64;
// in a graph 3.9 for one of 64 random nodes and 8.9 for a chain of 64 that is kept
// whole, 4.9 and 83 for 256 nodes.
//
// commit_kernel: slot(P + k) <- slot(P + path[k]) for the tokens of an accepted
// path, in every layer, P the committed tokens before the tree.  path[k] >= k,
// so no token is overwritten before it is read if a thread takes its bytes of
// all tokens in order.  Bound by latency at few requests (4.8 us for one with 4
// tokens in 36 layers): a chain of look-ups, then a burst of loads and one of
// stores, which all workgroups do at once.  64 requests' 1 .. 8 tokens in 36
// layers, 58 MB, 18 us, 3.2 TB/s; 3 tokens of each, 57 MB, 14 us; 8 of each,
// 151 MB, 30 us, 5.0 TB/s, and 256 requests' 128 us, 4.7 TB/s.  Whether pages and
// tokens lie in order makes no difference (30.2 and 30.7 us).
#include "pl_common.h"

namespace pl {
namespace commit {

constexpr int kWave = 64;
constexpr int kThreads = 256;

typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));

__global__ __launch_bounds__(kWave) void accept_kernel(const int64_t* __restrict__ tokens,
                                                       const int32_t* __restrict__ parents,
                                                       const int64_t* __restrict__ picks,
                                                       const int32_t* __restrict__ qo_indptr, int n_tokens,
                                                       int max_path, int32_t* __restrict__ path,
                                                       int32_t* __restrict__ count, int64_t* __restrict__ kept) {
  const int r = blockIdx.x, lane = threadIdx.x;
  const int begin = min(max(uniform(qo_indptr[r]), 0), n_tokens);
  const int n = min(max(uniform(qo_indptr[r + 1]), begin), n_tokens) - begin;
  tokens += begin;
  parents += begin;
  picks += begin;
  path += (int64_t)r * max_path;
  kept += (int64_t)r * max_path;
  int steps = 0;
  if (n > 0 && n <= kWave) {
    const bool on = lane < n;
    const int up = on ? parents[lane] : -1;
    const int64_t token = on ? tokens[lane] : 0, pick = on ? picks[lane] : 0;
    for (int at = 0; steps < max_path;) {
      const uint32_t lo = __builtin_amdgcn_readlane((int)pick, at), hi = __builtin_amdgcn_readlane((int)(pick >> 32), at);
      const int64_t want = (int64_t)((uint64_t)hi << 32 | lo);
      if (lane == 0) {
        path[steps] = at;
        kept[steps] = want;
      }
      ++steps;
      const uint64_t next = __builtin_amdgcn_ballot_w64(on && up == at && lane > at && token == want);
      if (next == 0) break;
      at = __builtin_ctzll(next);
    }
  } else if (n > 0) {
    for (int at = 0; steps < max_path;) {
      const int64_t want = picks[at];
      if (lane == 0) {
        path[steps] = at;
        kept[steps] = want;
      }
      ++steps;
      int child = -1;
      for (int base = at + 1; base < n && child < 0; base += kWave) {
        const int i = base + lane;
        const uint64_t next = __builtin_amdgcn_ballot_w64(i < n && parents[i] == at && tokens[i] == want);
        if (next) child = base + __builtin_ctzll(next);
      }
      if (child < 0) break;
      at = child;
    }
  }
  for (int k = steps + lane; k < max_path; k += kWave) {
    path[k] = -1;
    kept[k] = -1;
  }
  if (lane == 0) count[r] = steps;
}

struct Args {
  char* k;
  char* v;
  int64_t layer_stride, page_stride, token_stride, head_stride, num_pages;  // bytes; pages
  const int32_t *qo_indptr, *kv_indptr, *kv_indices, *kv_last, *path, *count;
  int layers, layers_each, num_indices, max_path, page_size;
  int row_chunks, head_chunks;  // 16-byte chunks of a token's K row, of one head
};

// A workgroup: 256 chunks of one request's token rows (K, then V) in some layers.
__global__ __launch_bounds__(kThreads) void commit_kernel(Args A) {
  __shared__ int64_t s_src[kWave], s_dst[kWave];
  __shared__ int s_live;
  const int r = blockIdx.y, layer0 = blockIdx.z * A.layers_each;
  const int layers = min(A.layers - layer0, A.layers_each);
  const int begin = uniform(A.kv_indptr[r]), pages = min(uniform(A.kv_indptr[r + 1]), A.num_indices) - begin;
  const int count = min(uniform(A.count[r]), A.max_path);
  if (begin < 0 || pages <= 0 || count <= 0) return;
  const int tree = uniform(A.qo_indptr[r + 1]) - uniform(A.qo_indptr[r]);
  const int last = min(max(uniform(A.kv_last[r]), 1), A.page_size);
  const int64_t len = (int64_t)(pages - 1) * A.page_size + last, base = len - tree;
  if (tree <= 0 || base < 0) return;
  const int chunk = blockIdx.x * kThreads + threadIdx.x;
  const bool on = chunk < 2 * A.row_chunks;
  const int c = chunk % A.row_chunks;
  char* row = (chunk < A.row_chunks ? A.k : A.v) + (int64_t)layer0 * A.layer_stride +
              (int64_t)(c / A.head_chunks) * A.head_stride + (int64_t)(c % A.head_chunks) * 16;
  auto slot = [&](int64_t pos) -> int64_t {  // byte offset, -1 outside the pool
    const int64_t page = pos / A.page_size;
    const int64_t id = A.kv_indices[begin + page];
    return id < 0 || id >= A.num_pages ? -1 : id * A.page_stride + (pos - page * A.page_size) * A.token_stride;
  };
  for (int k0 = 0; k0 < count; k0 += kWave) {
    // the slots of 64 tokens; the path ends before an entry outside [k, tree)
    if (threadIdx.x < kWave) {
      const int k = k0 + threadIdx.x;
      const int from = k < count ? A.path[(int64_t)r * A.max_path + k] : -1;
      const bool good = from >= k && from < tree;
      const uint64_t bad = __builtin_amdgcn_ballot_w64(!good);
      if (threadIdx.x == 0) s_live = bad ? __builtin_ctzll(bad) : kWave;
      s_src[threadIdx.x] = good && from != k ? slot(base + from) : -1;
      s_dst[threadIdx.x] = good && from != k ? slot(base + k) : -1;
    }
    __syncthreads();
    const int live = s_live;
    if (on) {
      // The loads of eight tokens in two layers, then their stores: a token's slot
      // is no source of a later one.
      for (int i0 = 0; i0 < live; i0 += 8) {
        for (int l0 = 0; l0 < layers; l0 += 2) {
          u32x4 x[2][8];
#pragma unroll
          for (int l = 0; l < 2; ++l)
#pragma unroll
            for (int i = 0; i < 8; ++i)
              if (l0 + l < layers && i0 + i < live && s_src[i0 + i] >= 0 && s_dst[i0 + i] >= 0)
                x[l][i] = __builtin_nontemporal_load(
                    reinterpret_cast<const u32x4*>(row + (l0 + l) * A.layer_stride + s_src[i0 + i]));
#pragma unroll
          for (int l = 0; l < 2; ++l)
#pragma unroll
            for (int i = 0; i < 8; ++i)
              if (l0 + l < layers && i0 + i < live && s_src[i0 + i] >= 0 && s_dst[i0 + i] >= 0)
                __builtin_nontemporal_store(
                    x[l][i], reinterpret_cast<u32x4*>(row + (l0 + l) * A.layer_stride + s_dst[i0 + i]));
        }
      }
    }
    if (live < kWave) return;
    __syncthreads();
  }
}

}  // namespace commit
}  // namespace pl

using namespace pl;

extern "C" int pl_tree_accept(const int64_t* tokens, const int32_t* parents, const int64_t* picks,
                              const int32_t* qo_indptr, int batch, int num_tokens, int max_path, int32_t* path,
                              int32_t* count, int64_t* kept, void* stream) {
  if (batch < 0 || num_tokens < 0) return fail(PL_ERR_INVALID, "batch and num_tokens must be >= 0");
  if (max_path <= 0) return fail(PL_ERR_INVALID, "max_path must be > 0");
  if (batch == 0) return ok();
  if (!qo_indptr || !path || !count || !kept || (num_tokens > 0 && (!tokens || !parents || !picks)))
    return fail(PL_ERR_INVALID, "null pointer argument");
  hipLaunchKernelGGL(commit::accept_kernel, dim3((unsigned)batch), dim3(commit::kWave), 0, (hipStream_t)stream, tokens,
                     parents, picks, qo_indptr, num_tokens, max_path, path, count, kept);
  PL_LAUNCH_CHECK("tree accept_kernel");
  return ok();
}

extern "C" int pl_tree_commit(void* k_cache, void* v_cache, int64_t layer_stride, int64_t page_stride,
                              int64_t token_stride, int64_t head_stride, int num_layers, int64_t num_pages,
                              const int32_t* qo_indptr, const int32_t* kv_indptr, const int32_t* kv_indices,
                              int num_indices, const int32_t* kv_last_page_len, const int32_t* path,
                              const int32_t* count, int batch, int max_path, int num_kv_heads, int head_dim,
                              int page_size, int dtype, void* stream) {
  if (batch < 0 || num_layers < 0 || num_indices < 0 || num_kv_heads <= 0 || head_dim <= 0)
    return fail(PL_ERR_INVALID, "bad shape");
  if (max_path <= 0) return fail(PL_ERR_INVALID, "max_path must be > 0");
  if (num_pages <= 0 || page_size <= 0) return fail(PL_ERR_INVALID, "num_pages and page_size must be > 0");
  if (dtype != PL_DTYPE_F32 && dtype != PL_DTYPE_F16 && dtype != PL_DTYPE_BF16)
    return fail(PL_ERR_UNSUPPORTED, "dtype %d", dtype);
  if (batch == 0 || num_layers == 0 || num_indices == 0) return ok();
  if (!k_cache || !v_cache || !qo_indptr || !kv_indptr || !kv_indices || !kv_last_page_len || !path || !count)
    return fail(PL_ERR_INVALID, "null pointer argument");
  const int eb = dtype_bytes(dtype), per = 16 / eb;
  if (head_dim % per) return fail(PL_ERR_INVALID, "head_dim must be a multiple of %d", per);
  const int64_t strides[] = {layer_stride, page_stride, token_stride, head_stride};
  for (int64_t s : strides)
    if (s % per) return fail(PL_ERR_INVALID, "strides must be multiples of %d elements", per);
  if ((uintptr_t)k_cache % 16 || (uintptr_t)v_cache % 16)
    return fail(PL_ERR_INVALID, "caches must be 16-byte aligned");
  if (batch > 65535 || num_layers > 65535 || (int64_t)num_kv_heads * head_dim > (1 << 24))
    return fail(PL_ERR_UNSUPPORTED, "batch %d, %d layers or %d heads of %d are too many", batch, num_layers,
                num_kv_heads, head_dim);
  commit::Args a{};
  a.k = (char*)k_cache;
  a.v = (char*)v_cache;
  a.layer_stride = layer_stride * eb;
  a.page_stride = page_stride * eb;
  a.token_stride = token_stride * eb;
  a.head_stride = head_stride * eb;
  a.num_pages = num_pages;
  a.qo_indptr = qo_indptr;
  a.kv_indptr = kv_indptr;
  a.kv_indices = kv_indices;
  a.kv_last = kv_last_page_len;
  a.path = path;
  a.count = count;
  a.layers = num_layers;
  a.num_indices = num_indices;
  a.max_path = max_path;
  a.page_size = page_size;
  a.head_chunks = head_dim / per;
  a.row_chunks = num_kv_heads * a.head_chunks;
  // Enough workgroups to fill the chip, and no more: each first looks up its request's slots.
  const int across = (2 * a.row_chunks + commit::kThreads - 1) / commit::kThreads;
  const int64_t each = ((int64_t)across * batch * num_layers + 2047) / 2048;
  a.layers_each = (int)(each < num_layers ? each : num_layers);
  const dim3 grid(across, batch, (num_layers + a.layers_each - 1) / a.layers_each);
  hipLaunchKernelGGL(commit::commit_kernel, grid, dim3(commit::kThreads), 0, (hipStream_t)stream, a);
  PL_LAUNCH_CHECK("tree commit_kernel");
  return ok();
}
