// Paged attention over the 8-bit KV cache (e4m3 codes, one power-of-two scale per page, side, head).
//
// Keys in the shared pages -- positions below E = max(n_shared_pages * page_size, shared_len) -- are
// read by the split pass, private tail pages (drafter routes) by the merge, which also joins the
// splits.  Position x of row r is visible when x < row_len[r] and (x < row_full[r] or bit
// x - mask_base of row_mask[r] is set).
//
// The weights carry V's scale: with u = score * log2(e) + log2(v_scale) a key adds 2^(u - ref) * code_v
// to O and 2^(u - ref) / v_scale to the sum, ref following the largest u, so pages of very different
// size meet in one accumulator without overflow.

#include <cuda_fp8.h>

#include "common.cuh"
#include "kv8.h"
#include "launch.h"

namespace atlas {

namespace {
constexpr int kHd = 128;
}  // namespace

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

__device__ __forceinline__ bool attn8_visible(const Attn8Params& p, int m, int x, int full, int len, int mask_base) {
  if (x >= len) return false;
  if (x < full) return true;
  const int b = x - mask_base;
  if (b < 0 || b >= 64 * p.mask_words) return false;
  return (static_cast<uint64_t>(p.row_mask[static_cast<int64_t>(m) * p.mask_words + (b >> 6)]) >> (b & 63)) & 1ull;
}

__device__ __forceinline__ void decode4(uint32_t w, float* x) {
  const __half2_raw a = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(w & 0xffff), __NV_E4M3);
  const __half2_raw b = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(w >> 16), __NV_E4M3);
  const float2 fa = __half22float2(__half2(a)), fb = __half22float2(__half2(b));
  x[0] = fa.x;
  x[1] = fa.y;
  x[2] = fb.x;
  x[3] = fb.y;
}

// One warp folds keys [x0, x1) of row m (kv head h) into its running (ref, l, o); lane t holds
// dimensions 4 t .. 4 t + 3.  `tail`: the keys' pages are the row's private ones.
template <bool kTail>
__device__ __forceinline__ void fold_keys8(const Attn8Params& p, const Attn8Shape& s, int m, int h, int lane,
                                           const float* q, int x0, int x1, int full, int len, float& ref, float& l,
                                           float* o) {
  const int ps = 1 << p.page_shift;
  for (int t0 = x0; t0 < x1; t0 += 32) {
    // Lane i resolves key t0 + i: its page-head index and scales.
    const int x = t0 + lane;
    int64_t ph = -1;
    float ks = 0.f, vs = 0.f;
    if (x < x1 && attn8_visible(p, m, x, full, len, s.mask_base)) {
      const int j = kTail ? (x >> p.page_shift) - s.n_shared : x >> p.page_shift;
      const bool in = j >= 0 && j < (kTail ? p.tail_stride : p.n_prefix);
      const int page = !in ? -1 : kTail ? p.tail_pages[static_cast<int64_t>(m) * p.tail_stride + j] : p.prefix_pages[j];
      if (page < 0 || page >= p.num_pages) {
        set_error(p.err, kErrBadIndex);
      } else {
        ph = static_cast<int64_t>(page) * 2 * p.Hkv + h;
        ks = p.scale[ph];
        vs = p.scale[ph + p.Hkv];
        if (!(vs > 0.f)) vs = 1.f;  // an empty page: its codes are zero
      }
    }
    const int cnt = min(32, x1 - t0);
    for (int j0 = 0; j0 < cnt; j0 += 8) {
      uint32_t kw[8], vw[8];
      int64_t pj[8];
      float kj[8], vj[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const int jj = (j0 + u) & 31;
        pj[u] = __shfl_sync(0xffffffffu, ph, jj);
        kj[u] = __shfl_sync(0xffffffffu, ks, jj);
        vj[u] = __shfl_sync(0xffffffffu, vs, jj);
        if (j0 + u >= cnt) pj[u] = -1;
        if (pj[u] >= 0) {
          const uint8_t* kp = p.data + (pj[u] * ps + ((t0 + j0 + u) & (ps - 1))) * kHd + lane * 4;
          kw[u] = __ldcg(reinterpret_cast<const uint32_t*>(kp));
          vw[u] = __ldcg(reinterpret_cast<const uint32_t*>(kp + static_cast<int64_t>(p.Hkv) * ps * kHd));
        }
      }
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        if (pj[u] < 0) continue;  // warp-uniform
        float k[4], v[4];
        decode4(kw[u], k);
        decode4(vw[u], v);
        const float dot = warp_sum(q[0] * k[0] + q[1] * k[1] + q[2] * k[2] + q[3] * k[3]);
        const float sc = dot * kj[u] * p.scale_log2 + log2f(vj[u]);
        const float nm = fmaxf(ref, sc);
        const float a = ref > -INFINITY ? exp2f(ref - nm) : 0.f, w = exp2f(sc - nm);
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = o[e] * a + w * v[e];
        l = l * a + w / vj[u];
        ref = nm;
      }
    }
  }
}

template <typename T>
__device__ __forceinline__ void load_q4(const Attn8Params& p, int64_t pair, int lane, float* q) {
  const uint2 raw = *reinterpret_cast<const uint2*>(static_cast<const T*>(p.q) + pair * kHd + lane * 4);
  const T* e = reinterpret_cast<const T*>(&raw);
#pragma unroll
  for (int i = 0; i < 4; ++i) q[i] = to_f32(e[i]);
}

// One warp per (row, q head) and split over the shared keys.
template <typename T>
__global__ void __launch_bounds__(128) attn8_split_kernel(Attn8Params p) {
  pdl_wait();
  pdl_trigger();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t pairs = static_cast<int64_t>(p.M) * p.Hq;
  const int64_t pair = static_cast<int64_t>(blockIdx.x) * 4 + warp;
  if (pair >= pairs) return;
  const int m = static_cast<int>(pair / p.Hq), hq = static_cast<int>(pair % p.Hq);
  const Attn8Shape s = attn8_shape(p);
  const int len = p.row_len[m], full = min(p.row_full[m], len);
  const int end = min(s.shared_end, len);
  const int per = (((s.shared_end + p.splits - 1) / p.splits) + 31) & ~31;
  const int x0 = blockIdx.y * per;
  float q[4], o[4] = {0.f, 0.f, 0.f, 0.f}, ref = -INFINITY, l = 0.f;
  load_q4<T>(p, pair, lane, q);
  fold_keys8<false>(p, s, m, hq / (p.Hq / p.Hkv), lane, q, x0, min(end, x0 + per), full, len, ref, l, o);
  const int64_t rec = blockIdx.y * pairs + pair;
  if (lane == 0) p.part_ml[rec] = make_float2(ref, l);
  *reinterpret_cast<float4*>(p.part_o + rec * kHd + lane * 4) = make_float4(o[0], o[1], o[2], o[3]);
}

// One warp per (row, q head): the row's private tail keys, then the splits' records in split order
// (a fixed order: the result does not depend on timing).
template <typename T>
__global__ void __launch_bounds__(128) attn8_merge_kernel(Attn8Params p) {
  pdl_wait();
  pdl_trigger();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t pairs = static_cast<int64_t>(p.M) * p.Hq;
  const int64_t pair = static_cast<int64_t>(blockIdx.x) * 4 + warp;
  if (pair >= pairs) return;
  const int m = static_cast<int>(pair / p.Hq), hq = static_cast<int>(pair % p.Hq);
  const Attn8Shape s = attn8_shape(p);
  const int len = p.row_len[m], full = min(p.row_full[m], len);
  float o[4] = {0.f, 0.f, 0.f, 0.f}, ref = -INFINITY, l = 0.f;
  if (s.shared_end < len) {
    float q[4];
    load_q4<T>(p, pair, lane, q);
    fold_keys8<true>(p, s, m, hq / (p.Hq / p.Hkv), lane, q, s.shared_end, len, full, len, ref, l, o);
  }
  for (int i = 0; i < p.splits; ++i) {
    const int64_t rec = i * pairs + pair;
    const float2 ml = __ldcg(p.part_ml + rec);
    if (ml.y == 0.f) continue;  // no key of this row in the split (a NaN sum goes on)
    const float4 v = __ldcg(reinterpret_cast<const float4*>(p.part_o + rec * kHd + lane * 4));
    const float nm = fmaxf(ref, ml.x);
    const float a = ref > -INFINITY ? exp2f(ref - nm) : 0.f, b = exp2f(ml.x - nm);
    o[0] = o[0] * a + v.x * b;
    o[1] = o[1] * a + v.y * b;
    o[2] = o[2] * a + v.z * b;
    o[3] = o[3] * a + v.w * b;
    l = l * a + ml.y * b;
    ref = nm;
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;  // a row without a key answers zero
  T v[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) v[e] = from_f32<T>(o[e] * inv);
  *reinterpret_cast<uint2*>(static_cast<T*>(p.out) + pair * kHd + lane * 4) = *reinterpret_cast<const uint2*>(v);
}

template <typename T>
static cudaError_t launch_typed8(const Attn8Params& p, cudaStream_t st) {
  const unsigned blocks = static_cast<unsigned>((static_cast<int64_t>(p.M) * p.Hq + 3) / 4);
  if (p.splits > 0) {
    const cudaError_t e = launch_k(attn8_split_kernel<T>, dim3(blocks, p.splits), dim3(128), 0, st, p);
    if (e != cudaSuccess) return e;
  }
  return launch_k(attn8_merge_kernel<T>, dim3(blocks), dim3(128), 0, st, p);
}

cudaError_t launch_attention8(const CUtensorMap&, const Attn8Params& p, cudaStream_t st) {
  if (p.M == 0) return cudaSuccess;
  return p.bf16 ? launch_typed8<__nv_bfloat16>(p, st) : launch_typed8<__half>(p, st);
}

}  // namespace atlas
