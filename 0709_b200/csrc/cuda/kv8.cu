// 8-bit paged KV cache: append (rotary + rounding), page copies, slot moves, read back.
//
// An element stands for code * scale with e4m3 codes and one power-of-two scale per page, side
// (k, v) and head.  Powers of two make every step exact but the one rounding to e4m3: x / scale is
// exact, re-rounding a page after its scale grew changes only codes that fall below e4m3's smallest
// normal number, and a page whose scale did not change is never touched.  The scale a row needs is
// 2^e with the smallest e in [-40, 56] for which max |x| <= 448 * 2^e.
//
// Writing slots of a page (append and moves alike): the page's scale becomes the largest its new
// rows need, or keeps its old value if that is larger, and the codes of its other slots are rounded
// again when it grew.  Writing slot 0 starts the page anew: the scale is that of its new rows alone
// and its other slots read zero, so a recycled page carries nothing of its last use.  Rows that cannot be
// stored are reported and write no slot.

#include <cuda_fp8.h>

#include "common.cuh"
#include "kv8.h"
#include "launch.h"

namespace atlas {

namespace {
constexpr int kHd = 128;
constexpr int kMaxPage = 64;
constexpr int kExpMin = -40, kExpMax = 56;
constexpr float kF16Max = 65504.f;
}  // namespace

__device__ __forceinline__ float kv8_pow2(int e) { return __int_as_float((e + 127) << 23); }

// Exponent of the scale for max |x| given as its bits (448 = 1.75 * 2^8).
__device__ __forceinline__ int kv8_exponent(uint32_t amax_bits) {
  const int ex = static_cast<int>(amax_bits >> 23) - 127;
  return max(kExpMin, ex - ((amax_bits & 0x7fffffu) <= 0x600000u ? 8 : 7));
}
__device__ __forceinline__ bool kv8_storable(uint32_t amax_bits) {
  return amax_bits < 0x7f800000u && kv8_exponent(amax_bits) <= kExpMax;
}

__device__ __forceinline__ uint32_t kv8_encode4(const float* x, float inv) {
  const uint32_t lo =
      __nv_cvt_float2_to_fp8x2(make_float2(x[0] * inv, x[1] * inv), __NV_SATFINITE, __NV_E4M3);
  const uint32_t hi =
      __nv_cvt_float2_to_fp8x2(make_float2(x[2] * inv, x[3] * inv), __NV_SATFINITE, __NV_E4M3);
  return lo | (hi << 16);
}
__device__ __forceinline__ void kv8_decode4(uint32_t w, float* x) {
  const __half2_raw a = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(w & 0xffff), __NV_E4M3);
  const __half2_raw b = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(w >> 16), __NV_E4M3);
  const float2 fa = __half22float2(__half2(a)), fb = __half22float2(__half2(b));
  x[0] = fa.x;
  x[1] = fa.y;
  x[2] = fb.x;
  x[3] = fb.y;
}
// The codes of w rounded again for a scale larger by 1 / ratio (ratio <= 1, a power of two).
__device__ __forceinline__ uint32_t kv8_rescale4(uint32_t w, float ratio) {
  float x[4];
  kv8_decode4(w, x);
  return kv8_encode4(x, ratio);
}

template <typename T>
__device__ __forceinline__ void load4(const T* p, float* x) {
  const uint2 r = *reinterpret_cast<const uint2*>(p);
  const T* e = reinterpret_cast<const T*>(&r);
#pragma unroll
  for (int i = 0; i < 4; ++i) x[i] = to_f32(e[i]);
}
template <>
__device__ __forceinline__ void load4<float>(const float* p, float* x) {
  *reinterpret_cast<float4*>(x) = *reinterpret_cast<const float4*>(p);
}

// a * b - c * d with the error of the second product put back (two roundings in all): near a
// rounding border of e4m3 a plain fp32 difference would more often fall on the wrong side.
__device__ __forceinline__ float diff_of_products(float a, float b, float c, float d) {
  const float cd = c * d;
  const float err = fmaf(-c, d, cd);
  return fmaf(a, b, -cd) + err;
}

// Dimensions i .. i + 3 and 64 + i .. 64 + i + 3 of the head at x, rotated (rotate-half pairing:
// dimension i < 64 pairs with i + 64).  kExact: the rounding that follows is the coarse one of e4m3.
template <typename T, bool kExact>
__device__ __forceinline__ void rotate8(const T* x, const float* cs, int i, float* y) {
  float a[4], b[4], c[4], s[4];
  load4<T>(x + i, a);
  load4<T>(x + 64 + i, b);
  load4<float>(cs + i, c);
  load4<float>(cs + 64 + i, s);
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    y[e] = kExact ? diff_of_products(a[e], c[e], b[e], s[e]) : a[e] * c[e] - b[e] * s[e];
    y[4 + e] = kExact ? diff_of_products(b[e], c[e], -a[e], s[e]) : b[e] * c[e] + a[e] * s[e];
  }
}

__device__ __forceinline__ uint32_t abs_bits_max8(const float* x) {
  uint32_t m = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) m = max(m, __float_as_uint(x[e]) & 0x7fffffffu);
  return m;
}

template <typename O>
__device__ __forceinline__ void store4(O* p, const float* x) {
  O v[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) v[e] = from_f32<O>(x[e]);
  *reinterpret_cast<uint2*>(p) = *reinterpret_cast<const uint2*>(v);
}

// Row r's k (rotated) and v of kv head h: this lane of 16 holds k dimensions i .. i + 3, 64 + i .. 64 + i + 3
// and v dimensions 2 i .. 2 i + 7, i = 4 * (lane & 15).
template <typename T>
__device__ __forceinline__ void load_kv8(const Kv8AppendParams& p, int r, int pos, int h, int i, float* k, float* v) {
  const T* row = static_cast<const T*>(p.qkv) + r * p.ld;
  rotate8<T, true>(row + (p.Hq + h) * kHd, p.table + static_cast<int64_t>(pos) * kHd, i, k);
  load4<T>(row + (p.Hq + p.Hkv + h) * kHd + 2 * i, v);
  load4<T>(row + (p.Hq + p.Hkv + h) * kHd + 2 * i + 4, v + 4);
}

// One kv head of `page`, which row m writes, if m is the first row of the batch to write it: all of the
// page's rows.  So each page and head has one writer and no order of blocks matters.  The price is that
// every such block looks through all slots: about a fifth of the time at 16384 rows (138 us with the pages
// read back, 3.5 times that of 5001 rows), growing with the square of the rows.
template <typename T, bool kDense>
__device__ __forceinline__ void append_page(const Kv8AppendParams& p, int m, int page, int h) {
  __shared__ int owner[kMaxPage];  // row that writes slot o, -1: none
  __shared__ uint32_t amax_s[2];
  __shared__ int follower;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int ps = 1 << p.page_shift;
  __syncthreads();  // a page before this one may still be in use
  if (tid < kMaxPage) owner[tid] = -1;
  if (tid < 2) amax_s[tid] = 0;
  if (tid == 0) follower = 0;
  __syncthreads();
  auto note = [&](int j, int s) {
    if (s >= 0 && (s >> p.page_shift) == page) {
      if (j < m) follower = 1;
      atomicMax(&owner[s & (ps - 1)], j);
    }
  };
  const int vec = (reinterpret_cast<uintptr_t>(p.slots) & 15) == 0 ? p.M >> 2 : 0;
#pragma unroll 4
  for (int j = tid; j < vec; j += 128) {
    const int4 s = reinterpret_cast<const int4*>(p.slots)[j];
    note(4 * j, s.x);
    note(4 * j + 1, s.y);
    note(4 * j + 2, s.z);
    note(4 * j + 3, s.w);
  }
  for (int j = 4 * vec + tid; j < p.M; j += 128) note(j, p.slots[j]);
  float* scale = p.scale + (static_cast<int64_t>(page) * 2) * p.Hkv + h;
  const float old_k = scale[0], old_v = scale[p.Hkv];
  __syncthreads();
  if (follower) return;
  // Largest magnitudes of the new rows, 16 lanes to a row; a row that cannot be stored is reported and
  // left out.
  const int i = (lane & 15) * 4, sub = lane >> 4;
  uint32_t ak = 0, av = 0;
#pragma unroll (kDense ? 1 : 2)
  for (int o2 = warp * 2; o2 < ps; o2 += 8) {
    const int o = o2 + sub, r = owner[o];
    const int pos = r >= 0 ? p.pos[r] : -1;
    const bool in = pos >= 0 && pos < p.max_pos;
    uint32_t lk = 0, lv = 0;
    if (in) {
      float k[8], v[8];
      load_kv8<T>(p, r, pos, h, i, k, v);
      lk = abs_bits_max8(k);
      lv = abs_bits_max8(v);
    }
    const uint32_t fine = __ballot_sync(0xffffffffu, kv8_storable(lk) && kv8_storable(lv)) >> (16 * sub);
    const bool ok = in && (fine & 0xffffu) == 0xffffu;
    if (ok) {
      ak = max(ak, lk);
      av = max(av, lv);
    } else if (r >= 0 && (lane & 15) == 0) {
      set_error(p.err, in ? kErrNonFinite : kErrBadIndex);
      owner[o] = -1;
    }
  }
  ak = __reduce_max_sync(0xffffffffu, ak);
  av = __reduce_max_sync(0xffffffffu, av);
  if (lane == 0) {
    atomicMax(&amax_s[0], ak);
    atomicMax(&amax_s[1], av);
  }
  __syncthreads();
  const bool anew = owner[0] >= 0;
  bool any = false;
  for (int o = 0; o < ps; ++o) any |= owner[o] >= 0;
  if (!any) return;
  const float need_k = kv8_pow2(kv8_exponent(amax_s[0])), need_v = kv8_pow2(kv8_exponent(amax_s[1]));
  const float new_k = anew ? need_k : fmaxf(old_k, need_k);
  const float new_v = anew ? need_v : fmaxf(old_v, need_v);
  const float inv_k = 1.f / new_k, inv_v = 1.f / new_v;
  uint32_t* kd = reinterpret_cast<uint32_t*>(p.data) + ((static_cast<int64_t>(page) * 2) * p.Hkv + h) * ps * (kHd / 4);
  uint32_t* vd = kd + static_cast<int64_t>(p.Hkv) * ps * (kHd / 4);
#pragma unroll (kDense ? 1 : 2)
  for (int o2 = warp * 2; o2 < ps; o2 += 8) {
    const int o = o2 + sub, r = owner[o];
    uint32_t* ko = kd + o * (kHd / 4) + i / 4;  // words of dimensions i and 64 + i: 16 apart
    uint2* vo = reinterpret_cast<uint2*>(vd + o * (kHd / 4) + i / 2);
    if (r >= 0) {
      float k[8], v[8];
      load_kv8<T>(p, r, p.pos[r], h, i, k, v);
      ko[0] = kv8_encode4(k, inv_k);
      ko[16] = kv8_encode4(k + 4, inv_k);
      *vo = make_uint2(kv8_encode4(v, inv_v), kv8_encode4(v + 4, inv_v));
    } else if (anew) {
      ko[0] = 0;
      ko[16] = 0;
      *vo = make_uint2(0, 0);
    } else {
      if (new_k > old_k && old_k > 0.f) {
        ko[0] = kv8_rescale4(ko[0], old_k * inv_k);
        ko[16] = kv8_rescale4(ko[16], old_k * inv_k);
      }
      if (new_v > old_v && old_v > 0.f)
        *vo = make_uint2(kv8_rescale4(vo->x, old_v * inv_v), kv8_rescale4(vo->y, old_v * inv_v));
    }
  }
  if (tid == 0) {
    scale[0] = new_k;
    scale[p.Hkv] = new_v;
  }
}

// 128 threads.  The first q_blocks blocks rotate Q, q_per_warp (row, head) pairs per warp; the others
// take kv_rows consecutive rows of one kv head each and write the pages that these rows start.
// Few rows are bound by latency: launch, slots, then the rows and the page they meet (one row 4.4 us, 13
// rows 4.9 us with the pages read back, 32 / 8 heads).  A prompt is bound by bytes and by the two reads of each row, for the maximum
// and for the codes (the second one hits the L1 or L2): 5001 rows of bf16 30 us for 113 MB.
template <typename T, typename O, bool kDense>
__device__ __forceinline__ void append_body(const Kv8AppendParams& p) {
  pdl_wait();
  pdl_trigger();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (static_cast<int>(blockIdx.x) < p.q_blocks) {
    const uint32_t pairs = static_cast<uint32_t>(p.M) * p.Hq;  // below 2^31
    uint32_t pair = (blockIdx.x * 4 + warp) * p.q_per_warp + (lane >> 4);  // 16 lanes each
    const uint32_t stop = min(pairs, (blockIdx.x * 4 + warp + 1) * p.q_per_warp);
    const int i = (lane & 15) * 4;
#pragma unroll (kDense ? 2 : 4)
    for (; pair < stop; pair += 2) {
      const int m = pair / static_cast<uint32_t>(p.Hq), head = pair - m * p.Hq;
      const int pos = p.pos[m];
      float y[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
      if (pos >= 0 && pos < p.max_pos)
        rotate8<T, false>(static_cast<const T*>(p.qkv) + m * p.ld + head * kHd,
                          p.table + static_cast<int64_t>(pos) * kHd, i, y);
      else if ((lane & 15) == 0)
        set_error(p.err, kErrBadIndex);
      O* out = static_cast<O*>(p.q_out) + static_cast<int64_t>(pair) * kHd + i;
      store4<O>(out, y);
      store4<O>(out + 64, y + 4);
    }
    return;
  }
  const int b = blockIdx.x - p.q_blocks;
  const int h = b % p.Hkv, m0 = b / p.Hkv * p.kv_rows;
  // The rows whose predecessor writes another page (one of 16 in a prompt) may be the first of theirs.
  const int m = m0 + lane;
  const bool mine = lane < p.kv_rows && m < p.M;
  const int slot = mine ? p.slots[m] : 0, before = mine && m > 0 ? p.slots[m - 1] : -1;
  const int page = slot >> p.page_shift;
  const bool good = slot >= 0 && page < p.num_pages;
  if (!good) set_error(p.err, kErrBadIndex);
  uint32_t todo =
      __ballot_sync(0xffffffffu, mine && good && !(before >= 0 && (before >> p.page_shift) == page));
  while (todo) {
    const int i = __ffs(todo) - 1;
    todo &= todo - 1;
    append_page<T, kDense>(p, m0 + i, __shfl_sync(0xffffffffu, page, i), h);
  }
}

template <typename T, typename O>
__global__ void __launch_bounds__(128) kv8_append_kernel(Kv8AppendParams p) {
  append_body<T, O, false>(p);
}
template <typename T, typename O>
__global__ void __launch_bounds__(128, 12) kv8_append_dense_kernel(Kv8AppendParams p) {
  append_body<T, O, true>(p);
}

// grid (min(n, 64), layers, 2 * Hkv): one page and head per block and step, 2 KB for 16 slots, so that a
// fork of a few pages spreads over the device (9 pages in 16 layers, 8 kv heads: 6.5 us with the read-back of
// the copies, 24 MB in all).  With a count on the device the grid cannot follow it and is (1, layers, 2 * Hkv):
// 9 copies in 16 layers take 5.8 us for 2.8, one 1.8 for 1.7.
// Copies of one call are independent: a destination that is also a source, or twice a destination, is
// reported and skipped.  The slots behind the copied ones are zeroed; a copy of no token leaves an empty page
// (scale 0), which is how a page is freed.
__global__ void __launch_bounds__(128)
    kv8_copy_pages_kernel(uint4* __restrict__ data, float* __restrict__ scale, const int* __restrict__ plan,
                          const int* __restrict__ count, int max_n, int num_pages, int Hkv, int page_shift, int* err) {
  pdl_wait();
  pdl_trigger();
  const int n = count != nullptr ? min(*count, max_n) : max_n;
  const int ps = 1 << page_shift;
  const int64_t layer = blockIdx.y;
  const int kvh = blockIdx.z;
  const int vec = ps * (kHd / 16);
  for (int ci = blockIdx.x; ci < n; ci += gridDim.x) {
    const int src = plan[ci * 3 + 0], dst = plan[ci * 3 + 1], ntok = plan[ci * 3 + 2];
    bool bad = src < 0 || src >= num_pages || dst < 0 || dst >= num_pages || ntok < 0 || ntok > ps || src == dst;
    for (int j = threadIdx.x; j < n; j += blockDim.x)
      if (j != ci && (plan[j * 3] == dst || plan[j * 3 + 1] == dst)) bad = true;
    if (__syncthreads_or(bad)) {
      if (threadIdx.x == 0) set_error(err, kErrBadIndex);
      continue;
    }
    const int64_t s = (layer * num_pages + src) * 2 * Hkv + kvh, d = (layer * num_pages + dst) * 2 * Hkv + kvh;
    const int keep = ntok * (kHd / 16);
    for (int i = threadIdx.x; i < vec; i += blockDim.x)
      data[d * vec + i] = i < keep ? data[s * vec + i] : make_uint4(0, 0, 0, 0);
    if (threadIdx.x == 0) scale[d] = ntok > 0 ? scale[s] : 0.f;
  }
}

// grid (layers, 2 * Hkv), 256 threads; shared memory: n codes rows, scales, slots, page tables.
// Every source is read before any slot is written; then one warp per destination page, which may have to
// round its other slots again.  Bound by latency, three dependent trips to memory (4 moves in 32 layers 7.3 us with the pages
// read back).
__global__ void __launch_bounds__(256)
    kv8_move_slots_kernel(uint8_t* __restrict__ data, float* __restrict__ scale, const int* __restrict__ src,
                          const int* __restrict__ dst, int n, int num_pages, int Hkv, int page_shift, int* err) {
  extern __shared__ uint4 buf[];
  uint32_t* rows = reinterpret_cast<uint32_t*>(buf);  // [n][32]
  float* from = reinterpret_cast<float*>(rows + n * 32);
  int* to = reinterpret_cast<int*>(from + n);
  __shared__ int owners[8][kMaxPage];
  pdl_wait();
  pdl_trigger();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int ps = 1 << page_shift;
  const int64_t layer = blockIdx.x;
  const int64_t head = layer * num_pages * 2 * Hkv + blockIdx.y;  // + page * 2 Hkv: page-head index
  for (int j = warp; j < n; j += 8) {
    const int s = src[j], d = dst[j];
    const bool ok = s >= 0 && (s >> page_shift) < num_pages && d >= 0 && (d >> page_shift) < num_pages;
    if (ok) {
      const int64_t ph = head + static_cast<int64_t>(s >> page_shift) * 2 * Hkv;
      rows[j * 32 + lane] = *reinterpret_cast<const uint32_t*>(data + (ph * ps + (s & (ps - 1))) * kHd + lane * 4);
      if (lane == 0) from[j] = scale[ph];
    } else if (lane == 0) {
      set_error(err, kErrBadIndex);
    }
    if (lane == 0) to[j] = ok ? d : -1;
  }
  __syncthreads();
  int* owner = owners[warp];
  for (int j = warp; j < n; j += 8) {
    const int d = to[j];
    if (d < 0) continue;
    const int page = d >> page_shift;
    bool seen = false;  // an earlier move of this page handles it
    for (int i = lane; i < j; i += 32) seen |= to[i] >= 0 && (to[i] >> page_shift) == page;
    if (__any_sync(0xffffffffu, seen)) continue;
    owner[lane] = -1;
    owner[lane + 32] = -1;
    __syncwarp();
    for (int i = j + lane; i < n; i += 32)
      if (to[i] >= 0 && (to[i] >> page_shift) == page) atomicMax(&owner[to[i] & (ps - 1)], i);  // the later move wins
    __syncwarp();
    float need = 0.f;
    for (int o = lane; o < ps; o += 32)
      if (owner[o] >= 0) need = fmaxf(need, from[owner[o]]);
    need = warp_max(need);
    const bool anew = owner[0] >= 0;
    const int64_t ph = head + static_cast<int64_t>(page) * 2 * Hkv;
    const float old = scale[ph];
    const float now = anew ? need : fmaxf(old, need);
    const float inv = now > 0.f ? 1.f / now : 0.f;
    uint32_t* out = reinterpret_cast<uint32_t*>(data + ph * ps * kHd) + lane;
    for (int o = 0; o < ps; ++o) {
      const int i = owner[o];
      if (i >= 0)
        out[o * 32] = from[i] == now ? rows[i * 32 + lane] : kv8_rescale4(rows[i * 32 + lane], from[i] * inv);
      else if (anew)
        out[o * 32] = 0;
      else if (now > old && old > 0.f)
        out[o * 32] = kv8_rescale4(out[o * 32], old * inv);
    }
    __syncwarp();  // every lane has read `old` and the owners
    if (lane == 0) scale[ph] = now;
  }
}

template <typename O>
__device__ __forceinline__ O kv8_value(float x);
template <>
__device__ __forceinline__ __half kv8_value<__half>(float x) {
  return __float2half_rn(fminf(fmaxf(x, -kF16Max), kF16Max));
}
template <>
__device__ __forceinline__ __nv_bfloat16 kv8_value<__nv_bfloat16>(float x) {
  return __float2bfloat16_rn(x);
}

// grid (n, layers, 2 * Hkv): one page and head, 16 codes per thread and step; bound by the bytes written (313
// pages of 16 x 8 heads: 9.1 us for 31 MB, L2 cold).  fp16 values are held
// to its largest finite number (rounding up to e4m3 can pass it).
template <typename O>
__global__ void __launch_bounds__(128)
    kv8_read_pages_kernel(const uint4* __restrict__ data, const float* __restrict__ scale,
                          const int* __restrict__ pages, O* __restrict__ out, int num_pages, int Hkv, int page_shift,
                          int* err) {
  pdl_wait();
  pdl_trigger();
  const int64_t layer = blockIdx.y;
  const int kvh = blockIdx.z;
  const int vec = (1 << page_shift) * (kHd / 16);
  const int page = pages[blockIdx.x];
  const bool ok = page >= 0 && page < num_pages;
  if (!ok && threadIdx.x == 0) set_error(err, kErrBadIndex);
  const int64_t s = (layer * num_pages + (ok ? page : 0)) * 2 * Hkv + kvh;
  const float sc = ok ? scale[s] : 0.f;
  uint4* o = reinterpret_cast<uint4*>(out) +
             ((layer * gridDim.x + blockIdx.x) * 2 * Hkv + kvh) * static_cast<int64_t>(vec) * 2;
  for (int i = threadIdx.x; i < vec; i += blockDim.x) {
    const uint4 w = ok ? data[s * vec + i] : make_uint4(0, 0, 0, 0);
    const uint32_t c[4] = {w.x, w.y, w.z, w.w};
    O v[16];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      float x[4];
      kv8_decode4(c[e], x);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        v[e * 4 + k] = kv8_value<O>(x[k] * sc);
      }
    }
    o[2 * i] = reinterpret_cast<const uint4*>(v)[0];
    o[2 * i + 1] = reinterpret_cast<const uint4*>(v)[1];
  }
}

template <typename T, typename O>
static cudaError_t launch_append(const Kv8AppendParams& p, bool dense, dim3 grid, cudaStream_t st) {
  return launch_k(dense ? kv8_append_dense_kernel<T, O> : kv8_append_kernel<T, O>, grid, dim3(128), 0, st, p);
}

cudaError_t launch_kv8_append(const Kv8AppendParams& params, cudaStream_t st) {
  if (params.M == 0) return cudaSuccess;
  // Few rows: every (row, head) on a warp of its own, for latency.  Many: blocks of one such piece each
  // spend their time starting (98 us for 5001 rows); 8 pairs per warp and 16 rows per page block.  From 64 K
  // (row, head) pairs on, 32 pairs per warp and 40 registers for 12 blocks per SM (39 us where the form with
  // 64 registers took 48; 1200 rows 16.3 us in both, 300 rows 7.5 in this one and 8.1 in that).
  Kv8AppendParams p = params;
  const bool dense = static_cast<int64_t>(p.M) * p.Hq >= 65536;
  p.q_per_warp = dense ? 32 : p.M > 64 ? 8 : 2;
  p.kv_rows = p.M > 64 ? 16 : 1;
  const int64_t pairs = static_cast<int64_t>(p.M) * p.Hq;
  const int64_t per_block = 4 * p.q_per_warp;
  p.q_blocks = static_cast<int>((pairs + per_block - 1) / per_block);
  const dim3 grid(p.q_blocks + (p.M + p.kv_rows - 1) / p.kv_rows * p.Hkv);
  using B = __nv_bfloat16;
  if (p.in_type == kKv8Bf16) return launch_append<B, B>(p, dense, grid, st);
  if (p.in_type == kKv8F16) return launch_append<__half, __half>(p, dense, grid, st);
  return p.out_bf16 ? launch_append<float, B>(p, dense, grid, st) : launch_append<float, __half>(p, dense, grid, st);
}

cudaError_t launch_kv8_copy_pages(uint8_t* data, float* scale, const int* plan, const int* count, int n, int layers,
                                  int num_pages, int Hkv, int page_shift, int* err, cudaStream_t st) {
  if (n == 0) return cudaSuccess;
  const dim3 grid(count != nullptr ? 1 : (n < 64 ? n : 64), layers, 2 * Hkv);
  return launch_k(kv8_copy_pages_kernel, grid, dim3(128), 0, st, reinterpret_cast<uint4*>(data), scale, plan, count, n,
                  num_pages, Hkv, page_shift, err);
}

cudaError_t launch_kv8_move_slots(uint8_t* data, float* scale, const int* src, const int* dst, int n, int layers,
                                  int num_pages, int Hkv, int page_shift, int* err, cudaStream_t st) {
  if (n == 0) return cudaSuccess;
  const size_t smem = static_cast<size_t>(n) * (kHd + 8);
  if (smem > 40 * 1024) {
    static std::atomic<uint64_t> done{0};
    const cudaError_t e = allow_smem(kv8_move_slots_kernel, kKv8MaxMoves * (kHd + 8), done);
    if (e != cudaSuccess) return e;
  }
  return launch_k(kv8_move_slots_kernel, dim3(layers, 2 * Hkv), dim3(256), smem, st, data, scale, src, dst, n,
                  num_pages, Hkv, page_shift, err);
}

cudaError_t launch_kv8_read_pages(const uint8_t* data, const float* scale, const int* pages, void* out, int n,
                                  int layers, int num_pages, int Hkv, int page_shift, bool bf16, int* err,
                                  cudaStream_t st) {
  if (n == 0) return cudaSuccess;
  const dim3 grid(n, layers, 2 * Hkv);
  const uint4* d = reinterpret_cast<const uint4*>(data);
  if (bf16)
    return launch_k(kv8_read_pages_kernel<__nv_bfloat16>, grid, dim3(128), 0, st, d, scale, pages,
                    static_cast<__nv_bfloat16*>(out), num_pages, Hkv, page_shift, err);
  return launch_k(kv8_read_pages_kernel<__half>, grid, dim3(128), 0, st, d, scale, pages, static_cast<__half*>(out),
                  num_pages, Hkv, page_shift, err);
}

}  // namespace atlas
