// Device helpers shared by the attention kernels over the 8-bit KV cache.
#pragma once

#include "common.cuh"
#include "kv8.h"
#include "launch.h"

namespace atlas {

namespace {
constexpr int kHd = 128;
}  // namespace

// Weights are rounded to fp16, 2^(u - ref).  The reference is set 7 below a row's largest u and moves when a weight
// would pass 2^15, so that the largest weight is at least 2^7 and what fp16 loses at its lower end (2^-25) is below
// 2^-32 of it: a million such keys hold less than a quarter of a thousandth of the row.  (Set to the largest u itself,
// keys below 2^-25 of it vanished from O and stayed in the sum.)
constexpr float kTopWeight = 7.f;
constexpr float kMaxWeight = 15.f;
__device__ __forceinline__ bool ref_moves(float top, float ref) { return top - ref > kMaxWeight; }

struct Attn8Shape {
  int shared_len, n_shared, mask_base, shared_end;
};

__device__ __forceinline__ Attn8Shape attn8_shape(const Attn8Params& p) {
  Attn8Shape s;
  const bool dev = p.dparams != nullptr;
  s.shared_len = dev ? p.dparams[0] : p.shared_len;
  s.n_shared = dev ? p.dparams[1] : p.n_shared_pages;
  s.mask_base = dev ? p.dparams[2] : p.mask_base;
  s.shared_end = max(s.n_shared << p.page_shift, s.shared_len);
  return s;
}

// End of the shared keys that rows of length up to len_max read, held to the pages that are listed.
__device__ __forceinline__ int attn8_end(const Attn8Params& p, const Attn8Shape& s, int len_max) {
  const int end = min(s.shared_end, len_max), listed = p.n_prefix << p.page_shift;
  if (end > listed) set_error(p.err, kErrBadIndex);
  return min(end, listed);
}

// Scales of a page and head (k and v) as the kernels use them: k scale, log2(v scale), 1 / v scale.  An empty
// page (scale 0) holds zero codes: any positive scale reads it right.
__device__ __forceinline__ float4 attn8_scales(float k, float v) {
  const int e = v > 0.f ? static_cast<int>(__float_as_uint(v) >> 23) - 127 : 0;
  return make_float4(k > 0.f ? k : 1.f, static_cast<float>(e), __int_as_float((127 - e) << 23), 0.f);
}

// A row's factor (softmax scale, log2(e) and the power of two taken out of Q) times a page's k scale, kept positive
// and finite: a factor that left fp32 would turn a hidden key's -inf (times 0) or an exact zero (times inf) into NaN.
// The added 2^-126 is lost in any product above 2^-102, and Q K is at most 2^17 and at least 2^-33 where it is not
// zero: only scores below 2^-84 or above 2^94 change.  (2048 rows behind 6001 keys: 1.4 us of 260.)
__device__ __forceinline__ float attn8_factor(float fac, float k_scale) {
  return fminf(fmaf(fac, k_scale, 0x1p-126f), 0x1.fffffep127f);
}

__device__ __forceinline__ bool attn8_visible(const Attn8Params& p, int m, int x, int full, int len, int mask_base) {
  if (x >= len) return false;
  if (x < full) return true;
  const int b = x - mask_base;
  if (b < 0 || b >= 64 * p.mask_words) return false;
  return (static_cast<uint64_t>(p.row_mask[static_cast<int64_t>(m) * p.mask_words + (b >> 6)]) >> (b & 63)) & 1ull;
}

// Visibility of keys x0 .. x0 + 63 to row m, one bit each: those below `full`, and the marked ones
// below `len`.
__device__ __forceinline__ uint64_t visible64(const Attn8Params& p, int m, int x0, int full, int len, int mask_base) {
  auto first = [](int n) { return n <= 0 ? 0ull : n >= 64 ? ~0ull : (1ull << n) - 1ull; };
  const uint64_t sure = first(full - x0), in = first(len - x0);
  if (!(in & ~sure)) return sure & in;
  const int off = x0 - mask_base;  // mask bit of key x0; words outside the mask are zero
  const int w = off >> 6, b = off & 63;
  const int64_t* words = p.row_mask + static_cast<int64_t>(m) * p.mask_words;
  const uint64_t lo = w >= 0 && w < p.mask_words ? static_cast<uint64_t>(words[w]) : 0ull;
  const uint64_t hi = w + 1 >= 0 && w + 1 < p.mask_words ? static_cast<uint64_t>(words[w + 1]) : 0ull;
  const uint64_t marked = b ? (lo >> b) | (hi << (64 - b)) : lo;
  return (sure | marked) & in;
}

// Power of two that brings a row's largest magnitude (given as bits) into [1, 2); 0 for rows of zeros
// and rows that are not finite.
__device__ __forceinline__ int row_exponent(uint32_t amax_bits) {
  if (amax_bits == 0 || amax_bits >= 0x7f800000u) return 0;
  return min(max(static_cast<int>(amax_bits >> 23) - 127, -126), 126);
}

// The two codes in the low (high) half of w as fp16 values.
__device__ __forceinline__ uint32_t half_pair_lo(uint32_t w) {
  uint32_t r;
  asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\t}" : "=r"(r) : "r"(w));
  return r;
}
__device__ __forceinline__ uint32_t half_pair_hi(uint32_t w) {
  uint32_t r;
  asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, h;\n\t}" : "=r"(r) : "r"(w));
  return r;
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ uint32_t pack_half2(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// mbar_wait as a short loop: the passes here run several roles side by side and are sensitive to the size
// of their code.
__device__ __forceinline__ bool wait8(uint64_t* bar, uint32_t parity, int* err) {
#pragma unroll 1
  for (uint32_t i = 0; i < kSpinLimit; ++i)
    if (mbar_try_wait(bar, parity)) return true;
  set_error(err, kErrWaitTimeout);
  return false;
}

}  // namespace atlas
