// Tokens into a paged 4-bit KV cache and back (gfx950).
//
// Each 32 values x of a token and kv head become codes c of 4 bits (e2m1: sign, two
// bits of exponent, one of mantissa) and a power of two: x ~ c 2^e, e the least with
// max |x| <= 6 2^e, c the nearest code of x 2^-e, halfway to the even one.  The
// values c 2^e are exact in bf16, which the attention over this cache multiplies.
// e is kept in -125 .. 125: below, values fall to 0; above, they end at 6 2^125.  A
// group that holds a NaN or an infinity reads back as NaN.  In a group of zeros e is 0
// (head dims that only pad, say): the least one is past fp16's range, in which prompts of
// fp16 are multiplied (2048 tokens of 32 heads: 77 us, 198 where V is out of it).
//
// A lane works on eight values: one 16-byte load, the hardware's conversions, four
// bytes of codes.  A group is four lanes, which share its largest magnitude by two
// lane exchanges.  A wave takes four tokens of one head (head_dim 128), so that a
// prompt's V codes, laid out by four tokens, fill whole lines.
//
// Bound by memory: 8192 tokens of 32 heads, in no order, 170 MB each way: append 42.5
// us (4.0 TB/s; its V codes are pieces of 4 bytes, whose lines meet in the L2; 51 where
// the sources passed through it too), read 27.2 us (6.2 TB/s; 34 without the hint).
// Four heads per wave, for more loads in flight, were slower: 53 and 42.5 us.  64
// tokens of 8 heads: 3.2 and 3.1 us, a launch and two round trips.
#include "window_common.h"

namespace pl {
namespace window {
namespace kv4 {

constexpr int kThreads = 256;

struct Args {
  const char *k, *v;      // append: sources; read: where the values go
  char *kc, *vc;          // the cache's K and V
  const int64_t *page_id, *offset;
  int64_t k_st, k_sh, v_st, v_sh, page_stride, head_stride;  // bytes
  int64_t num_pages;
  int tokens, hkv, page_size;
};

// The place of eight values of a token: lanes go through them, then tokens, then
// heads, then blocks of tokens.
template <int D> struct Place {
  static constexpr int kLanes = D / 8;                 // of a token
  static constexpr int kTokens = kWave / kLanes;       // of a wave
  int64_t token;
  int head, chunk;
  __device__ Place(const Args& A, int64_t wave) {
    const int lane = threadIdx.x % kWave;
    head = (int)(wave % A.hkv);
    token = wave / A.hkv * kTokens + lane / kLanes;
    chunk = lane % kLanes;
  }
};
template <int D> int64_t waves_of(int tokens, int hkv) {
  return ((int64_t)tokens + Place<D>::kTokens - 1) / Place<D>::kTokens * hkv;
}

// Bytes of a lane's codes and of its group's scale, from a (page, kv head) on.
template <int D> __device__ __forceinline__ int codes_at(bool v, int slot, int chunk) {
  return v ? slot / 4 * (2 * D) + chunk * 16 + slot % 4 * 4 : slot * (D / 2) + chunk * 4;
}
template <int D> __device__ __forceinline__ int scale_at(bool v, int page_size, int slot, int chunk) {
  return page_size * (D / 2) + (v ? slot / 4 * (D / 8) + chunk / 4 * 4 + slot % 4 : slot * (D / kGroup) + chunk / 4);
}

// Eight values as codes; `byte` is their group's scale.
template <typename T> __device__ __forceinline__ uint32_t quantize8(u32x4 w, uint32_t& byte) {
  float x[8];
#pragma unroll
  for (int e = 0; e < 4; ++e) unpack2<T>(w[e], x[2 * e], x[2 * e + 1]);
  uint32_t bits = 0;  // of the largest magnitude: they order as numbers do, NaN above all
#pragma unroll
  for (int e = 0; e < 8; ++e) bits = max(bits, __float_as_uint(x[e]) & 0x7fffffffu);
  bits = max(bits, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)bits, 0xb1, 0xf, 0xf, false));  // lane ^ 1
  bits = max(bits, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)bits, 0x4e, 0xf, 0xf, false));  // lane ^ 2
  if (bits >= 0x7f800000u) {
    byte = kScaleNan;
    return 0u;
  }
  // the largest is 1.f 2^(E - 127) <= 6 2^(s - 127): s = E - 2, and one more where 1.f > 1.5
  const int s = (int)(bits >> 23) - 2 + ((bits & 0x7fffffu) > 0x400000u ? 1 : 0);
  byte = (uint32_t)(bits == 0 ? kScaleZero : min(max(s, kScaleMin), kScaleMax));
  const float scale = scale_of(byte);
  uint32_t c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0u, x[0], x[1], scale, 0);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, x[2], x[3], scale, 1);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, x[4], x[5], scale, 2);
  return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, x[6], x[7], scale, 3);
}

template <typename T, int D>
__global__ __launch_bounds__(kThreads) void append_kernel(Args A) {
  const int64_t wave = (int64_t)blockIdx.x * (kThreads / kWave) + threadIdx.x / kWave;
  const Place<D> at(A, wave);
  if (at.token >= A.tokens) return;
  const int64_t p = A.page_id[at.token], off = A.offset[at.token];
  // (read once: kept out of the L2, where pieces of a line from several tokens meet)
  const u32x4 k = __builtin_nontemporal_load(
      reinterpret_cast<const u32x4*>(A.k + at.token * A.k_st + at.head * A.k_sh + at.chunk * 16));
  const u32x4 v = __builtin_nontemporal_load(
      reinterpret_cast<const u32x4*>(A.v + at.token * A.v_st + at.head * A.v_sh + at.chunk * 16));
  if (p < 0 || p >= A.num_pages || off < 0 || off >= A.page_size) return;  // outside the pool
  const int slot = (int)off;
  const int64_t page = p * A.page_stride + at.head * A.head_stride;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    uint32_t byte;
    const uint32_t codes = quantize8<T>(i ? v : k, byte);
    char* to = (i ? A.vc : A.kc) + page;
    *reinterpret_cast<uint32_t*>(to + codes_at<D>(i, slot, at.chunk)) = codes;
    if (at.chunk % 4 == 0) *reinterpret_cast<uint8_t*>(to + scale_at<D>(i, A.page_size, slot, at.chunk)) = (uint8_t)byte;
  }
}

template <typename T> __device__ __forceinline__ u32x4 from_bf16(u32x4 w);
template <> __device__ __forceinline__ u32x4 from_bf16<bf16_t>(u32x4 w) { return w; }
template <> __device__ __forceinline__ u32x4 from_bf16<f16_t>(u32x4 w) {
#pragma unroll
  for (int e = 0; e < 4; ++e) w[e] = pack2<f16_t>(bf16_lo(w[e]), bf16_hi(w[e]));
  return w;
}

template <typename T, int D>
__global__ __launch_bounds__(kThreads) void read_kernel(Args A) {
  const int64_t wave = (int64_t)blockIdx.x * (kThreads / kWave) + threadIdx.x / kWave;
  const Place<D> at(A, wave);
  if (at.token >= A.tokens) return;
  const int64_t p = A.page_id[at.token], off = A.offset[at.token];
  const bool held = p >= 0 && p < A.num_pages && off >= 0 && off < A.page_size;
  const int slot = held ? (int)off : 0;
  const int64_t page = (held ? p : 0) * A.page_stride + at.head * A.head_stride;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const char* from = (i ? A.vc : A.kc) + page;
    const uint32_t codes = *reinterpret_cast<const uint32_t*>(from + codes_at<D>(i, slot, at.chunk));
    const uint32_t byte = *reinterpret_cast<const uint8_t*>(from + scale_at<D>(i, A.page_size, slot, at.chunk));
    char* to = const_cast<char*>(i ? A.v + at.token * A.v_st + at.head * A.v_sh : A.k + at.token * A.k_st + at.head * A.k_sh);
    __builtin_nontemporal_store(from_bf16<T>(codes8(codes, scale_of(held ? byte : (uint32_t)kScaleNan))),
                                reinterpret_cast<u32x4*>(to + at.chunk * 16));
  }
}

template <typename T, int D> int launch(const Args& a, bool read, hipStream_t s) {
  const dim3 grid((unsigned)((waves_of<D>(a.tokens, a.hkv) + kThreads / kWave - 1) / (kThreads / kWave)));
  if (read)
    hipLaunchKernelGGL((read_kernel<T, D>), grid, dim3(kThreads), 0, s, a);
  else
    hipLaunchKernelGGL((append_kernel<T, D>), grid, dim3(kThreads), 0, s, a);
  PL_LAUNCH_CHECK("kv4 kernel");
  return ok();
}

int run(const void* k, const void* v, int64_t k_st, int64_t k_sh, int64_t v_st, int64_t v_sh, const void* k_cache,
        const void* v_cache, int64_t page_stride, int64_t head_stride, int64_t num_pages, int page_size,
        const int64_t* page_id, const int64_t* offset, int tokens, int hkv, int head_dim, int dtype, bool read,
        void* stream) {
  if (tokens < 0 || hkv <= 0) return fail(PL_ERR_INVALID, "tokens must be >= 0 and num_kv_heads > 0");
  if (head_dim != 64 && head_dim != 128)
    return fail(PL_ERR_UNSUPPORTED, "head_dim must be 64 or 128 (got %d)", head_dim);
  if (dtype != PL_DTYPE_BF16 && dtype != PL_DTYPE_F16)
    return fail(PL_ERR_UNSUPPORTED, "dtype must be F16 or BF16 (got %d)", dtype);
  if (page_size <= 0 || page_size % 8 || page_size > (1 << 20) || num_pages <= 0)
    return fail(PL_ERR_INVALID, "pages of a 4-bit cache hold a multiple of 8 tokens, up to 2^20 (got %d)", page_size);
  if (tokens == 0) return ok();
  if (!k || !v || !k_cache || !v_cache || !page_id || !offset) return fail(PL_ERR_INVALID, "null pointer argument");
  const int64_t strides[] = {k_st * 2, k_sh * 2, v_st * 2, v_sh * 2, page_stride, head_stride};
  for (int64_t s : strides)
    if (s % 16) return fail(PL_ERR_INVALID, "strides must be multiples of 16 bytes");
  const void* ptrs[] = {k, v, k_cache, v_cache};
  for (const void* p : ptrs)
    if ((uintptr_t)p % 16) return fail(PL_ERR_INVALID, "k, v and the cache must be 16-byte aligned");
  if ((head_dim == 64 ? waves_of<64>(tokens, hkv) : waves_of<128>(tokens, hkv)) >= kMaxGroups * (kThreads / kWave))
    return fail(PL_ERR_INVALID, "%d tokens of %d kv heads exceed a launch", tokens, hkv);
  Args a{};
  a.k = (const char*)k;
  a.v = (const char*)v;
  a.kc = (char*)k_cache;
  a.vc = (char*)v_cache;
  a.page_id = page_id;
  a.offset = offset;
  a.k_st = strides[0];
  a.k_sh = strides[1];
  a.v_st = strides[2];
  a.v_sh = strides[3];
  a.page_stride = page_stride;
  a.head_stride = head_stride;
  a.num_pages = num_pages;
  a.tokens = tokens;
  a.hkv = hkv;
  a.page_size = page_size;
  const hipStream_t s = (hipStream_t)stream;
  if (dtype == PL_DTYPE_BF16) return head_dim == 64 ? launch<bf16_t, 64>(a, read, s) : launch<bf16_t, 128>(a, read, s);
  return head_dim == 64 ? launch<f16_t, 64>(a, read, s) : launch<f16_t, 128>(a, read, s);
}

}  // namespace kv4
}  // namespace window
}  // namespace pl

extern "C" int pl_kv4_append(const void* k, const void* v, int64_t k_stride_t, int64_t k_stride_h, int64_t v_stride_t,
                             int64_t v_stride_h, void* k_cache, void* v_cache, int64_t page_stride,
                             int64_t head_stride, int64_t num_pages, int page_size, const int64_t* page_id,
                             const int64_t* offset, int tokens, int num_kv_heads, int head_dim, int dtype,
                             void* stream) {
  return pl::window::kv4::run(k, v, k_stride_t, k_stride_h, v_stride_t, v_stride_h, k_cache, v_cache, page_stride,
                              head_stride, num_pages, page_size, page_id, offset, tokens, num_kv_heads, head_dim,
                              dtype, false, stream);
}

extern "C" int pl_kv4_read(const void* k_cache, const void* v_cache, int64_t page_stride, int64_t head_stride,
                           int64_t num_pages, int page_size, const int64_t* page_id, const int64_t* offset,
                           int tokens, int num_kv_heads, int head_dim, void* k, void* v, int64_t k_stride_t,
                           int64_t k_stride_h, int64_t v_stride_t, int64_t v_stride_h, int dtype, void* stream) {
  return pl::window::kv4::run(k, v, k_stride_t, k_stride_h, v_stride_t, v_stride_h, k_cache, v_cache, page_stride,
                              head_stride, num_pages, page_size, page_id, offset, tokens, num_kv_heads, head_dim,
                              dtype, true, stream);
}
