// Paged attention over the 8-bit KV cache (e4m3 codes, one power-of-two scale per page, side, head).
//
// Keys in the shared pages -- positions below E = max(n_shared_pages * page_size, shared_len) -- are
// read by the split pass, private tail pages (drafter routes) by the merge, which also joins the
// splits.  Position x of row r is visible when x < row_len[r] and (x < row_full[r] or bit
// x - mask_base of row_mask[r] is set).
//
// The weights carry V's scale: with u = score * log2(e) + log2(v_scale) a key adds 2^(u - ref) * code_v
// to O and 2^(u - ref) / v_scale to the sum, ref following the largest u, so pages of very different
// size meet in one accumulator without overflow.  The split passes round the weights of O to fp16 (11 bits
// for codes of 4) and sum them in fp32.

#include <cuda_fp8.h>

#include "attention8.cuh"

namespace atlas {

__device__ __forceinline__ void decode4(uint32_t w, float* x) {
  const __half2_raw a = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(w & 0xffff), __NV_E4M3);
  const __half2_raw b = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(w >> 16), __NV_E4M3);
  const float2 fa = __half22float2(__half2(a)), fb = __half22float2(__half2(b));
  x[0] = fa.x;
  x[1] = fa.y;
  x[2] = fb.x;
  x[3] = fb.y;
}

// One warp folds keys [x0, x1) of row m (kv head h), in the row's private pages, into its running
// (ref, l, o); lane t holds dimensions 4 t .. 4 t + 3.
__device__ __forceinline__ void fold_tail8(const Attn8Params& p, const Attn8Shape& s, int m, int h, int lane,
                                           const float* q, int x0, int x1, int full, int len, float& ref, float& l,
                                           float* o) {
  const int ps = 1 << p.page_shift;
  for (int t0 = x0; t0 < x1; t0 += 32) {
    // Lane i resolves key t0 + i: its page-head index and scales.
    const int x = t0 + lane;
    int64_t ph = -1;
    float4 sc = make_float4(1.f, 0.f, 1.f, 0.f);
    if (x < x1 && attn8_visible(p, m, x, full, len, s.mask_base)) {
      const int page = p.tail_pages[static_cast<int64_t>(m) * p.tail_stride + ((x >> p.page_shift) - s.n_shared)];
      if (page < 0 || page >= p.num_pages) {
        set_error(p.err, kErrBadIndex);
      } else {
        ph = static_cast<int64_t>(page) * 2 * p.Hkv + h;
        sc = attn8_scales(p.scale[ph], p.scale[ph + p.Hkv]);
      }
    }
    const int cnt = min(32, x1 - t0);
    constexpr int kBatch = 4;
#pragma unroll 1
    for (int j0 = 0; j0 < cnt; j0 += kBatch) {
      uint32_t kw[kBatch], vw[kBatch];
      int64_t pj[kBatch];
#pragma unroll
      for (int u = 0; u < kBatch; ++u) {
        pj[u] = __shfl_sync(0xffffffffu, ph, j0 + u);
        if (j0 + u >= cnt) pj[u] = -1;
        if (pj[u] >= 0) {
          const uint8_t* kp = p.data + (pj[u] * ps + ((t0 + j0 + u) & (ps - 1))) * kHd + lane * 4;
          kw[u] = __ldcg(reinterpret_cast<const uint32_t*>(kp));
          vw[u] = __ldcg(reinterpret_cast<const uint32_t*>(kp + static_cast<int64_t>(p.Hkv) * ps * kHd));
        }
      }
#pragma unroll
      for (int u = 0; u < kBatch; ++u) {
        const float4 c = make_float4(__shfl_sync(0xffffffffu, sc.x, j0 + u), __shfl_sync(0xffffffffu, sc.y, j0 + u),
                                     __shfl_sync(0xffffffffu, sc.z, j0 + u), 0.f);
        if (pj[u] < 0) continue;  // warp-uniform
        float k[4], v[4];
        decode4(kw[u], k);
        decode4(vw[u], v);
        const float dot = warp_sum(q[0] * k[0] + q[1] * k[1] + q[2] * k[2] + q[3] * k[3]);
        const float s2 = fmaf(dot, attn8_factor(p.scale_log2, c.x), c.y);
        const float nm = fmaxf(ref, s2);
        const float a = ref > -INFINITY ? ex2(ref - nm) : 0.f, w = ex2(s2 - nm);
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = o[e] * a + w * v[e];
        l = fmaf(w, c.z, l * a);
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

// ------------------------------------------------------------ split pass
__device__ __forceinline__ void mma16816(float* c, const uint4& a, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, "
      "%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1));
}

template <int MT>
struct SplitCfg {
  static constexpr int kWarps = 8;
  static constexpr int kRows = 16 * MT;
  static constexpr int kStages = MT == 1 ? 3 : 6;
  static constexpr int kUnitBytes = 4096;  // 16 keys: K 2 KB, V 2 KB
  static constexpr int kRingBytes = kWarps * kStages * kUnitBytes;
  static constexpr int kQBytes = MT * 8 * 512;
  static constexpr int kMergeBytes = kWarps * kRows * kHd * 4;
  static_assert(kMergeBytes <= kRingBytes, "the warps' partial rows reuse the ring");
  static constexpr int kSmem = 1024 + kRingBytes + kQBytes + kRows * 4 + kWarps * kRows * 8 + kWarps * kStages * 8;
};

// One CTA per (kv head, split of the shared keys, tile of 16 MT query rows); query rows are
// (row, head of the group) pairs.  Each warp streams its own units of 16 keys (K and V of one head:
// 4 KB by TMA, 128B-swizzled) through a private ring, so no warp waits for another before the final
// merge; a warp holds all the tile's rows: S = Q K^T and O += P V on m16n8k16 tensor-core
// instructions whose operands are converted from the codes in registers.  With few rows the pass is
// bound by the cache's bytes; going through registers costs the shared memory one write and one read
// of the codes and nothing else, where a TMEM pipeline would have to write both operands back in fp16.
// Measured: one row (4 query rows a kv head) behind 131077 keys, 8 kv heads, 55 us with the merge for 270 MB:
// 4.9 TB/s, 0.75 of the measured copy rate; issue slots 51 % busy, ALU 44 % (conversion), tensor pipe 32 %, so
// that what is left is the start and the merge (5 us) and loads that stop while a warp converts.  Separate
// accumulators for the two 64-dimension halves of S, to shorten its chain of products, spilled (56 us).
// Short calls: 36 rows a kv head on 2051 keys take 4100 cycles to the first products, 5500 for two units per
// warp and 4200 to join the warps, then 3.6 us of merge (13.3 us in all).
template <typename T, int MT>
__global__ void __launch_bounds__(256, MT == 1 ? 2 : 1)
    attn8_split_kernel(const __grid_constant__ CUtensorMap map, Attn8Params p) {
  using C = SplitCfg<MT>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* ring = smem;
  uint8_t* q_s = ring + C::kRingBytes;                       // A fragments [MT][8 k-steps][32 lanes] x 16 B
  float* rowfac = reinterpret_cast<float*>(q_s + C::kQBytes);  // [rows]: scores per unit of Q K (log2 units)
  float2* ml_s = reinterpret_cast<float2*>(rowfac + C::kRows);  // [warps][rows]
  uint64_t* bars = reinterpret_cast<uint64_t*>(ml_s + C::kWarps * C::kRows);

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int g = lane >> 2, t = lane & 3;
  const int h = blockIdx.x, split = blockIdx.y;
  const int G = p.Hq / p.Hkv;
  const int rows_total = p.M * G;
  const int tile0 = blockIdx.z * C::kRows;
  uint64_t* bar = bars + warp * C::kStages;
  if (lane == 0) {
    for (int s = 0; s < C::kStages; ++s) mbar_init(&bar[s], 1);
    fence_barrier_init();
  }
  if (tid == 0) tma_prefetch_desc(&map);
  __syncwarp();
  pdl_wait();
  pdl_trigger();
  // The tile's Q rows, a row per load of a warp, on their way before anything waits for memory.
  constexpr int kQRows = C::kRows / C::kWarps;
  uint2 qraw[kQRows];
#pragma unroll
  for (int i = 0; i < kQRows; ++i) {
    const int grow = tile0 + warp + i * C::kWarps;
    const int m = grow / G;
    qraw[i] = make_uint2(0, 0);
    if (grow < rows_total)
      qraw[i] = *reinterpret_cast<const uint2*>(static_cast<const T*>(p.q) +
                                                (static_cast<int64_t>(m) * p.Hq + h * G + grow - m * G) * kHd + lane * 4);
  }
  const Attn8Shape sh = attn8_shape(p);

  // The tile's limits: last visible key of any row, first key that some row may not see.
  int len_max = 0, full_min = 0x7fffffff;
  if (lane < C::kRows && tile0 + lane < rows_total) {
    const int m = (tile0 + lane) / G;
    len_max = p.row_len[m];
    full_min = min(p.row_full[m], len_max);
  }
  len_max = __reduce_max_sync(0xffffffffu, len_max);
  full_min = __reduce_min_sync(0xffffffffu, full_min);
  const int end = attn8_end(p, sh, len_max);
  const int units = (end + 15) >> 4;
  const int per = max((units + p.splits - 1) / p.splits, C::kWarps);
  const int u0 = split * per;
  const int mine = max(0, (min(units, u0 + per) - u0 - warp + C::kWarps - 1) / C::kWarps);  // units of this warp

  // Lane i: page and scales of this warp's unit base + i (two pages when a page has 8 slots).
  const int ps = 1 << p.page_shift;
  const bool two = p.page_shift == 3;
  struct Window {
    int page[2];
    float ks[2], vs[2];
  };
  auto load_window = [&](int base) {
    Window w;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      w.page[e] = 0;
      w.ks[e] = w.vs[e] = 1.f;
      const int x = ((u0 + warp + (base + lane) * C::kWarps) << 4) + e * 8;
      if (base + lane < mine && x < end && (e == 0 || two)) {
        const int page = p.prefix_pages[x >> p.page_shift];
        if (page < 0 || page >= p.num_pages) {
          set_error(p.err, kErrBadIndex);
        } else {
          w.page[e] = page;
          const int64_t ph = static_cast<int64_t>(page) * 2 * p.Hkv + h;
          const float k = p.scale[ph], v = p.scale[ph + p.Hkv];
          if (k > 0.f) w.ks[e] = k;
          if (v > 0.f) w.vs[e] = v;
        }
      }
    }
    if (!two) {
      w.ks[1] = w.ks[0];
      w.vs[1] = w.vs[0];
    }
    return w;
  };
  Window cur = load_window(0), nxt = load_window(32);
  int window = 0;  // first unit of cur

  uint8_t* my_ring = ring + warp * C::kStages * C::kUnitBytes;
  auto issue = [&](int i) {  // whole warp: unit i of this warp into its stage
    const int w = i - window;
    const int pa = __shfl_sync(0xffffffffu, w < 32 ? cur.page[0] : nxt.page[0], w & 31);
    const int pb = two ? __shfl_sync(0xffffffffu, w < 32 ? cur.page[1] : nxt.page[1], w & 31) : 0;
    if (lane == 0) {
      const int s = i % C::kStages;
      uint8_t* dst = my_ring + s * C::kUnitBytes;
      const int off = ((u0 + warp + i * C::kWarps) << 4) & (ps - 1);
      mbar_arrive_expect_tx(&bar[s], C::kUnitBytes);
      const int yk = ((pa * 2) * p.Hkv + h) * ps + off, yv = yk + p.Hkv * ps;
      tma_load_2d(dst, &map, &bar[s], 0, yk);
      tma_load_2d(dst + 2048, &map, &bar[s], 0, yv);
      if (two) {
        const int zk = ((pb * 2) * p.Hkv + h) * ps;
        tma_load_2d(dst + 1024, &map, &bar[s], 0, zk);
        tma_load_2d(dst + 2048 + 1024, &map, &bar[s], 0, zk + p.Hkv * ps);
      }
    }
  };
  const int ahead = min(mine, C::kStages);
  for (int i = 0; i < ahead; ++i) issue(i);

  // Q rows as fp16 A fragments, each row scaled by a power of two so that its largest element is in
  // [1, 2): bf16 rows of any size fit.  Dimensions 16 (2 t + s) + 4 i .. + 3 of a row belong to k-step
  // 4 s + i of the lanes t: the bytes of the K word that these lanes convert.
#pragma unroll
  for (int i = 0; i < kQRows; ++i) {
    const int r = warp + i * C::kWarps;
    const T* e = reinterpret_cast<const T*>(&qraw[i]);
    const float q[4] = {to_f32(e[0]), to_f32(e[1]), to_f32(e[2]), to_f32(e[3])};
    uint32_t ab = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) ab = max(ab, __float_as_uint(q[k]) & 0x7fffffffu);
    ab = __reduce_max_sync(0xffffffffu, ab);
    const int e2 = row_exponent(ab);
    const float down = __int_as_float((127 - e2) << 23);
    const int c = lane >> 2, ks = (c & 1) * 4 + (lane & 3);
    const int hi = (r >> 3) & 1;
    uint32_t* dst = reinterpret_cast<uint32_t*>(q_s) + (((r >> 4) * 8 + ks) * 32 + (r & 7) * 4 + (c >> 1)) * 4;
    dst[hi] = pack_half2(q[0] * down, q[1] * down);
    dst[2 + hi] = pack_half2(q[2] * down, q[3] * down);
    if (lane == 0) rowfac[r] = p.scale_log2 * __int_as_float((127 + e2) << 23);
  }
  __syncthreads();

  float o[MT][16][4];
  float ref[MT][2], sum[MT][2], fac[MT][2];
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
    for (int j = 0; j < 16; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[mt][j][e] = 0.f;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      ref[mt][e] = -INFINITY;
      sum[mt][e] = 0.f;
      fac[mt][e] = rowfac[mt * 16 + e * 8 + g];
    }
  }

  bool ok = true;
  for (int i = 0; i < mine && __all_sync(0xffffffffu, ok); ++i) {
    if (i - window == 32) {
      window += 32;
      cur = nxt;
      nxt = load_window(window + 32);
    }
    const int stage = i % C::kStages;
    ok = wait8(&bar[stage], (i / C::kStages) & 1, p.err);
    __syncwarp();  // the matrix instructions need the whole warp together
    const uint8_t* kb = my_ring + stage * C::kUnitBytes;
    const uint8_t* vb = kb + 2048;
    // S: lanes 4 g + t hold keys 8 nt + 2 t, + 1 of rows g and g + 8.
    float s[MT][2][4];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int nt = 0; nt < 2; ++nt)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[mt][nt][e] = 0.f;
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      uint4 kw[2];
#pragma unroll
      for (int nt = 0; nt < 2; ++nt)
        kw[nt] = *reinterpret_cast<const uint4*>(kb + sw128_offset(nt * 8 + g, 2 * t + half));
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        uint4 a[MT];
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
          a[mt] = *reinterpret_cast<const uint4*>(q_s + ((mt * 8 + half * 4 + w) * 32 + lane) * 16);
#pragma unroll
        for (int nt = 0; nt < 2; ++nt) {
          const uint32_t x = w == 0 ? kw[nt].x : w == 1 ? kw[nt].y : w == 2 ? kw[nt].z : kw[nt].w;
          const uint32_t b0 = half_pair_lo(x), b1 = half_pair_hi(x);
#pragma unroll
          for (int mt = 0; mt < MT; ++mt) mma16816(s[mt][nt], a[mt], b0, b1);
        }
      }
    }
    // u = score * log2(e) + log2(v scale); P = 2^(u - ref).
    const int wl = (i - window) & 31;
    float kf[2], lv[2], iv[2];
#pragma unroll
    for (int nt = 0; nt < 2; ++nt) {
      kf[nt] = __shfl_sync(0xffffffffu, cur.ks[nt], wl);
      const float v = __shfl_sync(0xffffffffu, cur.vs[nt], wl);
      const int ev = static_cast<int>(__float_as_uint(v) >> 23) - 127;
      lv[nt] = static_cast<float>(ev);
      iv[nt] = __int_as_float((127 - ev) << 23);
    }
    const int x0 = (u0 + warp + i * C::kWarps) << 4;
    const bool masked = x0 + 16 > min(full_min, end);
    uint4 pa[MT];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
      for (int e = 0; e < 2; ++e) {
#pragma unroll
        for (int nt = 0; nt < 2; ++nt) {
          const float f = attn8_factor(fac[mt][e], kf[nt]);
#pragma unroll
          for (int k = 0; k < 2; ++k) s[mt][nt][e * 2 + k] = fmaf(s[mt][nt][e * 2 + k], f, lv[nt]);
        }
        if (masked) {
          const int grow = tile0 + mt * 16 + e * 8 + g;
          uint32_t vis = 0;
          if (grow < rows_total) {
            const int m = grow / G;
            const int len = min(p.row_len[m], end);
            vis = static_cast<uint32_t>(visible64(p, m, x0, min(p.row_full[m], len), len, sh.mask_base));
          }
#pragma unroll
          for (int nt = 0; nt < 2; ++nt)
#pragma unroll
            for (int k = 0; k < 2; ++k)
              if (!((vis >> (nt * 8 + 2 * t + k)) & 1u)) s[mt][nt][e * 2 + k] = -INFINITY;
        }
        top[e] = fmaxf(fmaxf(s[mt][0][e * 2], s[mt][0][e * 2 + 1]), fmaxf(s[mt][1][e * 2], s[mt][1][e * 2 + 1]));
      }
      // ref follows the row's largest u only when that grew by more than 8 (a factor of 256): O is rarely
      // rescaled.
      if (__any_sync(0xffffffffu, ref_moves(top[0], ref[mt][0]) || ref_moves(top[1], ref[mt][1]))) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float mx = fmaxf(top[e], __shfl_xor_sync(0xffffffffu, top[e], 1));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
          if (ref_moves(mx, ref[mt][e])) {
            const float to = mx - kTopWeight;
            const float a = ref[mt][e] > -INFINITY ? ex2(ref[mt][e] - to) : 0.f;
            ref[mt][e] = to;
            sum[mt][e] *= a;
#pragma unroll
            for (int j = 0; j < 16; ++j) {
              o[mt][j][e * 2] *= a;
              o[mt][j][e * 2 + 1] *= a;
            }
          }
        }
      }
      uint32_t packed[2][2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float neg = ref[mt][e] > -INFINITY ? -ref[mt][e] : 0.f;
#pragma unroll
        for (int nt = 0; nt < 2; ++nt) {
          const float p0 = ex2(s[mt][nt][e * 2] + neg), p1 = ex2(s[mt][nt][e * 2 + 1] + neg);
          sum[mt][e] = fmaf(p0 + p1, iv[nt], sum[mt][e]);
          packed[nt][e] = pack_half2(p0, p1);
        }
      }
      pa[mt] = make_uint4(packed[0][0], packed[0][1], packed[1][0], packed[1][1]);
    }
    __syncwarp();
    // O += P V: lane (g, t) converts dimensions 16 g .. 16 g + 15 of keys 2 t, 2 t + 1, 2 t + 8, 2 t + 9.
    uint4 v4[4];
#pragma unroll
    for (int k = 0; k < 4; ++k)
      v4[k] = *reinterpret_cast<const uint4*>(vb + sw128_offset(2 * t + (k & 1) + (k >> 1) * 8, g));
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      uint32_t x[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) x[k] = w == 0 ? v4[k].x : w == 1 ? v4[k].y : w == 2 ? v4[k].z : v4[k].w;
#pragma unroll
      for (int b = 0; b < 4; b += 2) {  // codes b, b + 1 of both keys, one pair per dimension
        const uint32_t sel = b == 0 ? 0x5140u : 0x7362u;
        const uint32_t y0 = __byte_perm(x[0], x[1], sel), y1 = __byte_perm(x[2], x[3], sel);
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) mma16816(o[mt][w * 4 + b], pa[mt], half_pair_lo(y0), half_pair_lo(y1));
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) mma16816(o[mt][w * 4 + b + 1], pa[mt], half_pair_hi(y0), half_pair_hi(y1));
      }
    }
    __syncwarp();  // the stage is read: it may be filled again
    if (i + C::kStages < mine) issue(i + C::kStages);
  }

  // Merge the warps: (ref, sum) per row, then O over the drained rings.  Lane (g, t) holds
  // dimensions 32 t .. 32 t + 31 of rows g and g + 8; float4 f of a row lands at f ^ (2 t + (g & 1)).
#pragma unroll
  for (int mt = 0; mt < MT; ++mt)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      float l = sum[mt][e];
      l += __shfl_xor_sync(0xffffffffu, l, 1);
      l += __shfl_xor_sync(0xffffffffu, l, 2);
      if (t == 0) ml_s[warp * C::kRows + mt * 16 + e * 8 + g] = make_float2(ref[mt][e], l);
    }
  __syncthreads();  // every warp is done with its ring
  float* o_s = reinterpret_cast<float*>(ring);
#pragma unroll
  for (int mt = 0; mt < MT; ++mt)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      float* row = o_s + (warp * C::kRows + mt * 16 + e * 8 + g) * kHd;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        // c registers 2 e + k of n-tile j: dimension 32 t + 16 k + j
        const int k = i >> 2, j = (i & 3) * 4;
        *reinterpret_cast<float4*>(row + (t * 8 + (i ^ (2 * t + (g & 1)))) * 4) =
            make_float4(o[mt][j][e * 2 + k], o[mt][j + 1][e * 2 + k], o[mt][j + 2][e * 2 + k], o[mt][j + 3][e * 2 + k]);
      }
    }
  __syncthreads();
#pragma unroll
  for (int it = tid; it < C::kRows * 32; it += 256) {
    const int r = it >> 5, f = it & 31;  // one warp per row
    const int grow = tile0 + r;
    if (grow >= rows_total) break;  // whole warps, rows in order
    float2 ml = make_float2(-INFINITY, 0.f);
    if (lane < C::kWarps) ml = ml_s[lane * C::kRows + r];
    if (ml.y == 0.f) ml.x = -INFINITY;
    const float mx = warp_max(ml.x);
    // A NaN sum keeps its weight so that it shows in the result.
    const float w = ml.y == 0.f ? 0.f : mx > -INFINITY ? ex2(ml.x - mx) : 1.f;
    const float l = warp_sum(ml.y == 0.f ? 0.f : w * ml.y);
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    const int at = (f & ~7) + ((f & 7) ^ (2 * (f >> 3) + (r & 1)));
#pragma unroll
    for (int k = 0; k < C::kWarps; ++k) {
      const float wk = __shfl_sync(0xffffffffu, w, k);
      const float4 v = *reinterpret_cast<const float4*>(o_s + (k * C::kRows + r) * kHd + at * 4);
      if (wk != 0.f) {
        acc.x = fmaf(wk, v.x, acc.x);
        acc.y = fmaf(wk, v.y, acc.y);
        acc.z = fmaf(wk, v.z, acc.z);
        acc.w = fmaf(wk, v.w, acc.w);
      }
    }
    const int64_t rec = (static_cast<int64_t>(split) * p.M + grow / G) * p.Hq + h * G + grow % G;
    if (f == 0) p.part_ml[rec] = make_float2(mx, l);
    if (l != 0.f) *reinterpret_cast<float4*>(p.part_o + rec * kHd + f * 4) = acc;
  }
}

// One warp per (row, q head): the splits' records, joined in split order, and the row's private tail
// keys (a fixed order: the result does not depend on timing).  Bound by latency: the records are read
// in one trip and the partial rows in batches of 16 (one record after the other took 24 us for 37
// splits), while the tail's keys are on their way.
template <typename T>
__global__ void __launch_bounds__(128) attn8_merge_kernel(Attn8Params p) {
  constexpr int kBatch = 16;
  pdl_wait();
  pdl_trigger();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t pairs = static_cast<int64_t>(p.M) * p.Hq;
  const int64_t pair = static_cast<int64_t>(blockIdx.x) * 4 + warp;
  if (pair >= pairs) return;
  const int m = static_cast<int>(pair / p.Hq), hq = static_cast<int>(pair % p.Hq);
  const int S = p.splits;
  // Lane i holds records i and i + 32 (at most 64).
  float2 ml0 = make_float2(-INFINITY, 0.f), ml1 = ml0;
  if (lane < S) ml0 = __ldcg(p.part_ml + lane * pairs + pair);
  if (lane + 32 < S) ml1 = __ldcg(p.part_ml + (lane + 32) * pairs + pair);
  const float* po = p.part_o + pair * kHd + lane * 4;
  float4 ov[kBatch];
#pragma unroll
  for (int j = 0; j < kBatch; ++j)
    if (j < S) ov[j] = __ldcg(reinterpret_cast<const float4*>(po + j * pairs * kHd));

  const Attn8Shape s = attn8_shape(p);
  float o[4] = {0.f, 0.f, 0.f, 0.f}, ref = -INFINITY, l = 0.f;
  const int len = p.causal_start >= 0 ? 0 : p.row_len[m];  // a causal chunk has no private pages
  if (s.shared_end < len) {
    const int full = min(p.row_full[m], len);
    const int listed = (s.n_shared + p.tail_stride) << p.page_shift;  // the row's private pages end here
    if (len > listed && lane == 0) set_error(p.err, kErrBadIndex);
    float q[4];
    load_q4<T>(p, pair, lane, q);
    fold_tail8(p, s, m, hq / (p.Hq / p.Hkv), lane, q, s.shared_end, min(len, listed), full, len, ref, l, o);
  }

  // A record without keys has sum 0 and no partial row; a NaN sum keeps its weight, so that it shows.
  const bool has0 = ml0.y != 0.f, has1 = ml1.y != 0.f;
  const float top = warp_max(fmaxf(has0 ? ml0.x : -INFINITY, has1 ? ml1.x : -INFINITY));
  const float mx = fmaxf(top, ref);
  const float w0 = !has0 ? 0.f : mx > -INFINITY ? ex2(ml0.x - mx) : 1.f;
  const float w1 = !has1 ? 0.f : mx > -INFINITY ? ex2(ml1.x - mx) : 1.f;
  const float own = ref > -INFINITY ? ex2(ref - mx) : (l != 0.f ? 1.f : 0.f);
  l = l * own + warp_sum((has0 ? w0 * ml0.y : 0.f) + (has1 ? w1 * ml1.y : 0.f));
#pragma unroll
  for (int e = 0; e < 4; ++e) o[e] *= own;
  const uint32_t some0 = __ballot_sync(0xffffffffu, has0), some1 = __ballot_sync(0xffffffffu, has1);
  for (int s0 = 0; s0 < S; s0 += kBatch) {
    if (s0 > 0) {
#pragma unroll
      for (int j = 0; j < kBatch; ++j)
        if (s0 + j < S) ov[j] = __ldcg(reinterpret_cast<const float4*>(po + (s0 + j) * pairs * kHd));
    }
#pragma unroll
    for (int j = 0; j < kBatch; ++j) {
      const int i = s0 + j;
      const float w = __shfl_sync(0xffffffffu, i < 32 ? w0 : w1, i & 31);
      if (i < S && (((i < 32 ? some0 : some1) >> (i & 31)) & 1u)) {  // warp-uniform
        o[0] = fmaf(w, ov[j].x, o[0]);
        o[1] = fmaf(w, ov[j].y, o[1]);
        o[2] = fmaf(w, ov[j].z, o[2]);
        o[3] = fmaf(w, ov[j].w, o[3]);
      }
    }
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;  // a row without a key answers zero
  T v[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) v[e] = from_f32<T>(o[e] * inv);
  *reinterpret_cast<uint2*>(static_cast<T*>(p.out) + pair * kHd + lane * 4) = *reinterpret_cast<const uint2*>(v);
}

template <typename T, int MT>
static cudaError_t launch_split8(const CUtensorMap& map, const Attn8Params& p, cudaStream_t st) {
  constexpr int smem = SplitCfg<MT>::kSmem;
  static std::atomic<uint64_t> done{0};
  const cudaError_t e = allow_smem(attn8_split_kernel<T, MT>, smem, done);
  if (e != cudaSuccess) return e;
  const int rows = p.M * (p.Hq / p.Hkv);
  const dim3 grid(p.Hkv, p.splits, (rows + 16 * MT - 1) / (16 * MT));
  return launch_k(attn8_split_kernel<T, MT>, grid, dim3(256), smem, st, map, p);
}

template <typename T>
static cudaError_t launch_typed8(const CUtensorMap& map, const Attn8Params& p, cudaStream_t st) {
  if (p.splits > 0) {
    const cudaError_t e = p.row_tile == 0    ? launch_attention8_tc(map, p, st)
                          : p.row_tile == 16 ? launch_split8<T, 1>(map, p, st)
                                             : launch_split8<T, 2>(map, p, st);
    if (e != cudaSuccess) return e;
  }
  const unsigned blocks = static_cast<unsigned>((static_cast<int64_t>(p.M) * p.Hq + 3) / 4);
  return launch_k(attn8_merge_kernel<T>, dim3(blocks), dim3(128), 0, st, p);
}

cudaError_t launch_attention8(const CUtensorMap& map, const Attn8Params& p, cudaStream_t st) {
  if (p.M == 0) return cudaSuccess;
  if (p.direct) return launch_attention8_tc(map, p, st);
  return p.bf16 ? launch_typed8<__nv_bfloat16>(map, p, st) : launch_typed8<__half>(map, p, st);
}

}  // namespace atlas
