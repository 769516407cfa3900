// Paged attention over the 8-bit KV cache for many query rows: tcgen05 tiles of 128 rows.
//
// One CTA holds two tiles ("slots") of 128 query rows of one kv head: two different row tiles over
// the same keys, or -- when one tile holds all rows -- the same rows over alternate 64-key chunks,
// each slot then being a split of its own.  Warps:
//   0-7   softmax, one thread per query row (0-3 slot 0, 4-7 slot 1);
//   8-    converters: e4m3 codes of a chunk -> fp16 operand tiles in the 128B-swizzled layout (four
//         warps, or two groups of four on alternate chunks);
//   then  the TMA producer (the chunk's pages, K and V codes, and their scales) and two MMA issuers, one
//         per slot (one for both spent its time in turn on waits and issue: 2450 cycles per pair of S and
//         P V tiles whose products take 1280).
// S is double-buffered in TMEM, so that a slot's next scores are ready when its softmax is; P (fp16)
// replaces its S in place and is the A operand of O += P V.  Q is read from shared memory (TMEM has no
// room left; a form with Q and P in TMEM and a single S took 362 us where this one took 306).
//
// TMEM columns: S/P of slot s, buffer b at 128 s + 64 b; O of slot s at 256 + 128 s.
//
// Measured: 2048 rows x 32 heads behind 6001 keys (8 kv heads) 267 us, 0.54 of the measured bf16 matrix rate;
// 192 rows a head on 16384 keys 35.8 us and 104 rows on 33001 keys 42.2 us with the merge.  What bounds it,
// from cycle stamps of the first: a chunk takes 2150 cycles; the tensor pipe works for 1580 of them (an S
// product of 64 keys reads 6 KB of shared memory and runs at half rate: 65 cycles for 32), a softmax warp for
// 1700 (two share a scheduler), the converters for 880.  The short calls are bound by their ends (stamps in a
// replayed graph): with 256 rows a CTA's first scores come 11000 cycles (five chunks of keys in all) to 14400
// cycles (16K keys) after its launch, most of it Q, whose 24 rows per warp are loaded in three trips; with 128
// rows 11400, 6200 of them Q.  O takes 4400 to 8000 cycles from the last chunk to the last byte.

#include <type_traits>

#include "attention8.cuh"

namespace atlas {

namespace {
constexpr int kChunk = 64;
constexpr int kBytes8 = kChunk * kHd * 2;      // K | V codes
constexpr int kHalf16 = kChunk * 128;          // 64 keys x 64 dimensions of fp16
constexpr int kBytes16 = 4 * kHalf16;          // K halves | V halves
constexpr int kBytesQ = 128 * kHd * 2;         // two halves of 128 rows x 128 B
constexpr int kStages16 = 4;  // converted chunks
static_assert(256 * (kHd * 4 + 16) <= 2 * kBytes8 + kStages16 * kBytes16, "the output rows reuse the chunks' space");
static_assert(kBytesQ == 2 * kBytes8, "slot 1's own Q takes the place of two chunks of codes");
// Converter groups of four warps: with split keys a chunk feeds one slot only and two groups keep up.  Where
// both slots share the chunks, a fourth converted one is worth more than two more chunks of codes (the slots
// need not keep step: 265 -> 259 us); with split keys six chunks of codes and three converted took 45.7 us
// for 42.3.
template <bool kSplitKeys>
struct Roles {
  static constexpr int kStages8 = kSplitKeys ? 4 : 2;  // chunks of codes in flight
  static constexpr int kConvGroups = kSplitKeys ? 2 : 1;
  static constexpr int kProducer = 8 + 4 * kConvGroups;
  static constexpr int kThreads = (kProducer + 3) * 32;
};
constexpr int kSmem = 1024 + 4 * kBytes8 + kStages16 * kBytes16 + kBytesQ + (4 + kStages16) * 128 + 256 + 256;
constexpr uint32_t kColO = 256;
}  // namespace

// D (+)= A(tmem) * B(smem); B's descriptor as two words, so that the tiles of one operand differ by
// an addition to the low word.
__device__ __forceinline__ void umma_f16_ts(uint32_t tmem_d, uint32_t tmem_a, uint32_t desc_lo, uint32_t desc_hi,
                                            uint32_t idesc, bool accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 d;\n\t"
      "setp.ne.b32 p, %5, 0;\n\t"
      "mov.b64 d, {%2, %3};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], d, %4, {%6, %6, %6, %6}, p;\n\t}" ::"r"(tmem_d),
      "r"(tmem_a), "r"(desc_lo), "r"(desc_hi), "r"(idesc), "r"(static_cast<uint32_t>(accumulate)), "r"(0)
      : "memory");
}

__device__ __forceinline__ void umma_f16_ss2(uint32_t tmem_d, uint32_t a_lo, uint32_t b_lo, uint32_t desc_hi,
                                             uint32_t idesc, bool accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 a, b;\n\t"
      "setp.ne.b32 p, %5, 0;\n\t"
      "mov.b64 a, {%1, %3};\n\t"
      "mov.b64 b, {%2, %3};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %4, {%6, %6, %6, %6}, p;\n\t}" ::"r"(tmem_d),
      "r"(a_lo), "r"(b_lo), "r"(desc_hi), "r"(idesc), "r"(static_cast<uint32_t>(accumulate)), "r"(0)
      : "memory");
}

// Two fp32 values as one 64-bit operand of the packed fp32 instructions.
__device__ __forceinline__ uint64_t pair2(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void unpair2(uint64_t v, float& a, float& b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// Keys whose bit is 0 get no weight.
__device__ __forceinline__ void hide(float* s, uint64_t vis) {
  const uint32_t v = static_cast<uint32_t>(vis);
#pragma unroll
  for (int j = 0; j < 32; ++j)
    if (!((v >> j) & 1u)) s[j] = -INFINITY;
}

// Store 16 consecutive 32-bit columns of this thread's TMEM lane (warp-collective).
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const float* v) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16};" ::"r"(taddr),
      "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]), "f"(v[8]), "f"(v[9]),
      "f"(v[10]), "f"(v[11]), "f"(v[12]), "f"(v[13]), "f"(v[14]), "f"(v[15])
      : "memory");
  asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}

// Copy `bytes` (a multiple of 16) from shared to global memory, both 16-byte aligned; the wait returns
// when the copies of this thread are written (not only read: the merge kernel follows on their heels).
__device__ __forceinline__ void bulk_store(void* dst, const void* src, uint32_t bytes) {
  asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(dst), "r"(smem_u32(src)), "r"(bytes)
               : "memory");
}
__device__ __forceinline__ void bulk_store_wait() {
  asm volatile("cp.async.bulk.commit_group;\n\tcp.async.bulk.wait_group 0;" ::: "memory");
}

// One lane of a converged warp, the same one every time.
__device__ __forceinline__ bool elect_one() {
  uint32_t r;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(r));
  return r != 0;
}

// kGroup: keys that share their scales, 8 or 16 (pages of 8 slots, or more).  Groups of 16 halve the scale
// reads and their arithmetic: 279 -> 265 us.
template <typename T, bool kSplitKeys, int kGroup>
__global__ void __launch_bounds__(Roles<kSplitKeys>::kThreads, 1)
    attn8_tc_kernel(const __grid_constant__ CUtensorMap map, Attn8Params p) {
  constexpr bool ksplit = kSplitKeys;
  using R = Roles<kSplitKeys>;
  constexpr int kStages8 = R::kStages8;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* ring8 = smem;
  uint8_t* ring16 = ring8 + kStages8 * kBytes8;
  uint8_t* q_s = ring16 + kStages16 * kBytes16;  // slot 0 (and both slots with split keys)
  uint8_t* q1_s = q_s + kBytesQ;
  // Per 8 keys of a chunk: k scale, log2(v scale), 1 / v scale.
  float4* sc8 = reinterpret_cast<float4*>(q_s + (ksplit ? 1 : 2) * kBytesQ);  // [kStages8][8]
  float4* sc16 = sc8 + kStages8 * 8;                                       // [kStages16][8]
  uint64_t* full8 = reinterpret_cast<uint64_t*>(sc16 + 4 * 8);
  uint64_t* empty8 = full8 + kStages8;
  uint64_t* full16 = empty8 + kStages8;
  uint64_t* empty16 = full16 + kStages16;
  uint64_t* s_full = empty16 + kStages16;  // [slot][buffer]
  // [slot][buffer], 128 arrivals: a warp may write P(k + 1) while another still works on P(k)
  uint64_t* p_full = s_full + 4;
  uint64_t* pv_done = p_full + 4;          // [2], a phase per P V product but the last
  // [2], one phase: the slot's last product.  A warp may leave the loop while the product before the last is
  // still to run (its last S proves only the third from last), and a parity of pv_done could not tell the two.
  uint64_t* fin = pv_done + 2;
  uint64_t* q_full = fin + 2;              // every staging thread
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(q_full + 1);
  int8_t* q_exp = reinterpret_cast<int8_t*>(full8) + 256;  // [256] exponent that scaled each row of Q

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int h = blockIdx.x;
  const int G = p.Hq / p.Hkv;
  const int rows_total = p.M * G;
  // The longest causal tiles are launched first, so that the short ones fill the last wave.
  const int z = p.causal_start >= 0 ? static_cast<int>(gridDim.z - 1 - blockIdx.z) : static_cast<int>(blockIdx.z);
  const int row0 = z * (ksplit ? 128 : 256);
  const int rows_cta = min(rows_total - row0, ksplit ? 128 : 256);

  if (tid == 0) {
    for (int s = 0; s < kStages8; ++s) {
      mbar_init(&full8[s], 1);
      mbar_init(&empty8[s], 128);
    }
    for (int s = 0; s < kStages16; ++s) {
      mbar_init(&full16[s], 128);
      mbar_init(&empty16[s], ksplit ? 1 : 2);
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(&s_full[2 * s], 2);
      mbar_init(&s_full[2 * s + 1], 2);
      mbar_init(&p_full[2 * s], 128);
      mbar_init(&p_full[2 * s + 1], 128);
      mbar_init(&pv_done[s], 1);
      mbar_init(&fin[s], 1);
    }
    mbar_init(q_full, R::kProducer * 32);
    fence_barrier_init();
    tma_prefetch_desc(&map);
  }
  if (warp == 0) tmem_alloc(tmem_slot, 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  pdl_wait();
  pdl_trigger();  // after this CTA's TMEM allocation

  // Q: an equal share of the rows per warp, a row per load of the whole warp (a thread per row would touch
  // 32 lines with every load), eight rows at a time; the first eight are on their way before anything
  // waits for memory.
  constexpr int kQRows = ksplit ? 8 : 24;  // rows past the tile are not kept
  int row = warp * kQRows, qm = (row0 + row) / G, qg = (row0 + row) - qm * G;
  uint2 qraw[8];
  auto load_q8 = [&]() {
    const uint2* src = reinterpret_cast<const uint2*>(static_cast<const T*>(p.q) + h * G * kHd + lane * 4);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      qraw[i] = make_uint2(0, 0);
      if (row + i < rows_cta) qraw[i] = src[(static_cast<int64_t>(qm) * p.Hq + qg) * (kHd / 4)];
      if (++qg == G) {
        qg = 0;
        ++qm;
      }
    }
  };
  if (warp < R::kProducer) load_q8();

  // This split's chunks: up to the last key that any row of the CTA may see.
  const Attn8Shape sh = attn8_shape(p);
  int len_max = 0;
  if (p.causal_start >= 0) {
    len_max = p.causal_start + (row0 + rows_cta - 1) / G + 1;
  } else {
    for (int m = row0 / G + lane; m <= (row0 + rows_cta - 1) / G; m += 32) len_max = max(len_max, p.row_len[m]);
    len_max = __reduce_max_sync(0xffffffffu, len_max);
  }
  const int end = attn8_end(p, sh, len_max);
  const int chunks_all = (end + kChunk - 1) / kChunk;
  const int per = (chunks_all + p.tc_splits - 1) / p.tc_splits;
  const int c0 = static_cast<int>(blockIdx.y) * per;
  const int chunks = max(0, min(chunks_all, c0 + per) - c0);
  const int ps = 1 << p.page_shift;

  if (warp < R::kProducer) {
    // Each row of Q scaled by a power of two so that its largest element is in [1, 2), as fp16, swizzled.
#pragma unroll 1
    for (int i0 = 0; i0 < kQRows; i0 += 8) {
      if (i0 > 0) load_q8();
#pragma unroll
      for (int i = 0; i < 8; ++i, ++row) {
        const T* e = reinterpret_cast<const T*>(&qraw[i]);
        const float q[4] = {to_f32(e[0]), to_f32(e[1]), to_f32(e[2]), to_f32(e[3])};
        const float am = fmaxf(max3(fabsf(q[0]), fabsf(q[1]), fabsf(q[2])), fabsf(q[3]));
        const int e2 = row_exponent(__reduce_max_sync(0xffffffffu, __float_as_uint(am)));
        const float down = __int_as_float((127 - e2) << 23);
        uint8_t* qs = row < 128 ? q_s : q1_s;
        if (row < 256) {
          *reinterpret_cast<uint2*>(qs + (lane >> 4) * (kBytesQ / 2) + (lane & 1) * 8 +
                                    sw128_offset(row & 127, (lane & 15) >> 1)) =
              make_uint2(pack_half2(q[0] * down, q[1] * down), pack_half2(q[2] * down, q[3] * down));
          if (lane == 0) q_exp[row] = static_cast<int8_t>(e2);
        }
      }
    }
    fence_proxy_async_smem();
    mbar_arrive(q_full);
  }

  if (warp == R::kProducer) {
    // ---- producer.  Lane l holds page and scales of 8 keys, l & 7, of chunk l >> 3 of a window of four.
    // A chunk's copies need its pages, which are read two windows ahead; the scales, another dependent trip to
    // memory, are read one window ahead and handed over after the copies are issued.
    const int box = min(ps, 16);
    constexpr int kNone = -1;  // no key of this split
    auto load_page = [&](int first) {
      const int c = first + (lane >> 3), x = (c0 + c) * kChunk + (lane & 7) * 8;
      return c < chunks && x < end ? p.prefix_pages[x >> p.page_shift] : kNone;
    };
    struct Scales {
      float k, v;
    };
    // Sets a page that is not of the cache to kNone after reporting it; its keys read as page 0 does.
    auto load_scales = [&](int& page, int first) {
      if (page < 0 || page >= p.num_pages) {
        const int c = first + (lane >> 3), x = (c0 + c) * kChunk + (lane & 7) * 8;
        if (c < chunks && x < end) set_error(p.err, kErrBadIndex);
        page = kNone;
      }
      Scales r{0.f, 0.f};
      if (page != kNone) {
        const float* f = p.scale + static_cast<int64_t>(page) * 2 * p.Hkv + h;
        r.k = f[0];
        r.v = f[p.Hkv];
      }
      return r;
    };
    // Lane g < 8 issues the box that starts at its 8 keys (every other lane when a box holds 16).
    auto issue = [&](int c, int window_page) {
      const int page = max(0, __shfl_sync(0xffffffffu, window_page, (c & 3) * 8 + (lane & 7)));
      const int s = c % kStages8;
      if (lane < 8 && (box == 8 || (lane & 1) == 0)) {
        const int y = (page * 2 * p.Hkv + h) * ps + (((c0 + c) * kChunk + lane * 8) & (ps - 1));
        uint8_t* dst = ring8 + s * kBytes8 + lane * 8 * kHd;
        tma_load_2d(dst, &map, &full8[s], 0, y);
        tma_load_2d(dst + kBytes8 / 2, &map, &full8[s], 0, y + p.Hkv * ps);
      }
    };
    int page = load_page(0), next_page = load_page(4), far_page = load_page(8);
    Scales cur = load_scales(page, 0);
    for (int c = 0; c < min(chunks, kStages8); ++c) issue(c, page);
    Scales next = load_scales(next_page, 4);
    for (int c = 0; c < chunks; ++c) {
      if (c > 0 && (c & 3) == 0) {
        page = next_page;
        cur = next;
        next_page = far_page;
        next = load_scales(next_page, c + 4);
        far_page = load_page(c + 8);
      }
      const int s = c % kStages8;
      if (c >= kStages8) {
        const bool ok = wait8(&empty8[s], ((c / kStages8) - 1) & 1, p.err);
        if (!__all_sync(0xffffffffu, ok)) break;
        issue(c, page);
      }
      const float k = __shfl_sync(0xffffffffu, cur.k, (c & 3) * 8 + (lane & 7));
      const float v = __shfl_sync(0xffffffffu, cur.v, (c & 3) * 8 + (lane & 7));
      if (lane < 8) sc8[s * 8 + lane] = attn8_scales(k, v);
      __syncwarp();
      if (lane == 0) mbar_arrive_expect_tx(&full8[s], kBytes8);
      __syncwarp();
    }
  } else if (warp >= 8 && warp < R::kProducer) {
    // ---- converters: one 16-byte piece of codes (16 dimensions of a key) per thread and step
    // Pieces p and p + 4 of a row would meet the same banks (its two 64-dimension halves): the upper
    // pieces take the neighbouring row.
    const int piece = tid & 7, upper = piece >> 2;
    const int row = ((tid & 127) >> 3) ^ upper;  // rows row, row + 16, ..
    bool ok = true;
    for (int c = (warp - 8) >> 2; c < chunks && ok; c += R::kConvGroups) {
      const int s = c % kStages8, d = c % kStages16;
      ok = wait8(&full8[s], (c / kStages8) & 1, p.err);
      if (ok && c >= kStages16) ok = wait8(&empty16[d], ((c / kStages16) - 1) & 1, p.err);
      if (!ok) break;
      if ((tid & 127) < 8) sc16[d * 8 + (tid & 127)] = sc8[s * 8 + (tid & 127)];
      const uint8_t* src = ring8 + s * kBytes8;
      uint8_t* dst = ring16 + d * kBytes16;
      uint4 w[8];
#pragma unroll
      for (int i = 0; i < 8; ++i)  // K rows, then V rows
        w[i] = *reinterpret_cast<const uint4*>(src + (i >> 2) * (kBytes8 / 2) + sw128_offset(row + (i & 3) * 16, piece));
      mbar_arrive(&empty8[s]);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        uint4 lo, hi;
        lo.x = half_pair_lo(w[i].x);
        lo.y = half_pair_hi(w[i].x);
        lo.z = half_pair_lo(w[i].y);
        lo.w = half_pair_hi(w[i].y);
        hi.x = half_pair_lo(w[i].z);
        hi.y = half_pair_hi(w[i].z);
        hi.z = half_pair_lo(w[i].w);
        hi.w = half_pair_hi(w[i].w);
        uint8_t* half = dst + ((i >> 2) * 2 + upper) * kHalf16;
        const int r = row + (i & 3) * 16, at = 2 * (piece & 3);
        *reinterpret_cast<uint4*>(half + sw128_offset(r, at)) = lo;
        *reinterpret_cast<uint4*>(half + sw128_offset(r, at + 1)) = hi;
      }
      fence_proxy_async_smem();
      mbar_arrive(&full16[d]);
    }
  } else if (warp > R::kProducer) {
    // ---- MMA issuer of a slot.  The whole warp walks the loop and one elected lane issues: addresses
    // and descriptors then live in uniform registers (a single thread that builds each descriptor took
    // about 700 cycles for the eight instructions of an S tile, more than the products themselves).
    const int slot = warp - R::kProducer - 1;
    const int n = ksplit ? (chunks + 1 - slot) / 2 : chunks;
    if (n > 0) {
      constexpr uint32_t idesc_s = umma_idesc_f16(128, kChunk, false, false, false);
      constexpr uint32_t idesc_o = umma_idesc_f16(128, kHd, false, false, true);
      constexpr uint32_t kDescHi = (1024 >> 4) | (1u << 14) | (2u << 29);  // 8-row step, version, 128B swizzle
      const uint32_t q_lo = (smem_u32(ksplit || slot == 0 ? q_s : q1_s) >> 4) | (16 >> 4) << 16;
      const uint32_t k_lo = (smem_u32(ring16) >> 4) | (16 >> 4) << 16;
      const uint32_t v_lo = ((smem_u32(ring16) + 2 * kHalf16) >> 4) | (kHalf16 >> 4) << 16;
      const uint32_t tS0 = tmem + slot * 128, tO = tmem + kColO + slot * 128;
      const bool leader = elect_one();
      bool ok = wait8(q_full, 0, p.err);
      for (int k = 0; k <= n && ok; ++k) {
        if (k < n) {  // S(k); its buffer holds P(k - 2) until that P V is done
          const int c = ksplit ? 2 * k + slot : k, d = c % kStages16;
          if (k >= 2) ok = wait8(&pv_done[slot], k & 1, p.err);
          ok = ok && wait8(&full16[d], (c / kStages16) & 1, p.err);
          tc_fence_after();
          const uint32_t lo = k_lo + d * (kBytes16 >> 4);
          if (leader && ok) {
#pragma unroll
            for (int kk = 0; kk < 8; ++kk)
              umma_f16_ss2(tS0 + (k & 1) * 64, q_lo + (((kk >> 2) * (kBytesQ / 2) + (kk & 3) * 32) >> 4),
                           lo + (((kk >> 2) * kHalf16 + (kk & 3) * 32) >> 4), kDescHi, idesc_s, kk > 0);
            umma_commit(&s_full[slot * 2 + (k & 1)]);
            mbar_arrive(&s_full[slot * 2 + (k & 1)]);  // passes on what full16 covers: the chunk's scales
          }
          __syncwarp();
        }
        if (k > 0) {  // P(k - 1) V
          const int j = k - 1, c = ksplit ? 2 * j + slot : j, d = c % kStages16;
          ok = ok && wait8(&p_full[slot * 2 + (j & 1)], (j >> 1) & 1, p.err);
          tc_fence_after();
          const uint32_t lo = v_lo + d * (kBytes16 >> 4);
          if (leader && ok) {
#pragma unroll
            for (int kk = 0; kk < 4; ++kk)
              umma_f16_ts(tO, tS0 + (j & 1) * 64 + kk * 8, lo + kk * (2048 >> 4), kDescHi, idesc_o, j > 0 || kk > 0);
            umma_commit(k < n ? &pv_done[slot] : &fin[slot]);
            umma_commit(&empty16[d]);
          }
          __syncwarp();
        }
      }
    }
  } else if (warp < 8) {
    // ---- softmax: one thread per query row
    const int slot = warp >> 2;
    const int r = (ksplit ? 0 : slot * 128) + (tid & 127);
    const bool live = r < rows_cta;
    const int grow = row0 + (live ? r : 0);
    const int m = grow / G;
    const int hq = h * G + grow % G;
    const int64_t pair = static_cast<int64_t>(m) * p.Hq + hq;
    const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t tS0 = tmem + slot * 128 + lanes, tO = tmem + kColO + slot * 128 + lanes;
    int len = 0, full = 0;
    if (live) {
      len = p.causal_start >= 0 ? p.causal_start + m + 1 : p.row_len[m];
      full = p.causal_start >= 0 ? len : min(p.row_full[m], len);
    }
    const int lim = min(len, end), sure = min(full, end);  // keys below `sure` are visible
    wait8(q_full, 0, p.err);
    const int e2 = q_exp[r];
    const float fac = p.scale_log2 * __int_as_float((127 + e2) << 23);

    const int n = ksplit ? (chunks + 1 - slot) / 2 : chunks;
    float ref = -INFINITY, sum = 0.f;
    bool ok = true;
    // One chunk.  Once a row's reference is beyond 2^20, u - ref has to be taken from the rounded u, as the maximum
    // was (in one step the two can differ by more than fp16 holds): the plain form returns false and leaves the chunk
    // to the far one, which is kept small (4 us of the 2048-row chunk; as a branch within one form 10 us).
    auto fold_chunk = [&](auto far_form, int k) {
      constexpr bool kFar = decltype(far_form)::value;
      const int c = ksplit ? 2 * k + slot : k;
      const int d = c % kStages16;
      ok = wait8(&s_full[slot * 2 + (k & 1)], (k >> 1) & 1, p.err);
      __syncwarp();  // TMEM accesses need the whole warp together: after every wait and divergent step
      tc_fence_after();
      const uint32_t tS = tS0 + (k & 1) * 64;
      const int x0 = (c0 + c) * kChunk;
      // The warp masks as one: rows that see the whole chunk get a mask of ones.
      const bool partial = __any_sync(0xffffffffu, x0 + kChunk > sure);
      const uint64_t vis = partial ? visible64(p, m, x0, sure, lim, sh.mask_base) : ~0ull;
      __syncwarp();
      const float4* sc = sc16 + d * 8;
      // S 32 keys at a time.  With eight converter warps a row of S does not fit the registers and is read
      // twice, for the maximum and for the weights; with four it stays.
      constexpr bool kTwice = ksplit || kFar;
      constexpr int kKept = kTwice ? 1 : 2;
      float s[kKept][32];
      float top = -INFINITY;
      auto load_half = [&](int half, float* v) {
        tmem_ld32(tS + half * 32, v);
        if (partial) hide(v, vis >> (half * 32));
      };
      auto half_top = [&](int half, const float* v) {
#pragma unroll
        for (int gk = 0; gk < 4; gk += kGroup / 8, v += kGroup) {
          const float4 w = sc[half * 4 + gk];
          float mx = max3(max3(v[0], v[1], v[2]), max3(v[3], v[4], v[5]), fmaxf(v[6], v[7]));
          if constexpr (kGroup == 16)
            mx = max3(mx, max3(max3(v[8], v[9], v[10]), v[11], v[12]), max3(v[13], v[14], v[15]));
          top = fmaxf(top, fmaf(mx, attn8_factor(fac, w.x), w.y));
        }
      };
      if constexpr (kTwice) {
#pragma unroll 1
        for (int half = 0; half < 2; ++half) {
          load_half(half, s[0]);
          half_top(half, s[0]);
        }
      } else {
#pragma unroll
        for (int half = 0; half < 2; ++half) load_half(half, s[half % kKept]);
#pragma unroll
        for (int half = 0; half < 2; ++half) half_top(half, s[half % kKept]);
      }
      const bool moves = ref_moves(top, ref);
      bool far = false;
      if (__any_sync(0xffffffffu, moves)) {
        float a = 1.f;
        if (moves) {
          const float to = top - kTopWeight;
          a = ref > -INFINITY ? ex2(ref - to) : 0.f;
          ref = to;
          sum *= a;
        }
        if constexpr (!kFar) far = __any_sync(0xffffffffu, ref > -INFINITY && fabsf(ref) > 0x1p20f);
        // O has to hold P V of every chunk before; S(k) was started after product k - 2, so the phase of
        // product k - 1 is the one that its parity names.
        if (k > 0) {
          ok = wait8(&pv_done[slot], (k - 1) & 1, p.err) && ok;
          __syncwarp();
          tc_fence_after();
#pragma unroll 1
          for (int q4 = 0; q4 < 4; ++q4) {
            float ov[32];
            tmem_ld32(tO + q4 * 32, ov);
#pragma unroll
            for (int i = 0; i < 32; ++i) ov[i] *= a;
            tmem_st32(tO + q4 * 32, ov);
          }
        }
      }
      if (far) return false;
      const float neg = ref > -INFINITY ? -ref : 0.f;
      __syncwarp();
      auto weigh_half = [&](int half, const float* v) {
        float pk[16];
#pragma unroll
        for (int gk = 0; gk < 4; gk += kGroup / 8) {
          const float4 w = sc[half * 4 + gk];
          const float f1 = attn8_factor(fac, w.x), b1 = kFar ? w.y : w.y + neg;
          const uint64_t f = pair2(f1, f1), b = pair2(b1, b1);
          uint64_t acc = 0;
#pragma unroll
          for (int j = 0; j < kGroup; j += 2) {
            float p0, p1;
            unpair2(fma2(pair2(v[gk * 8 + j], v[gk * 8 + j + 1]), f, b), p0, p1);
            p0 = ex2(kFar ? p0 + neg : p0);
            p1 = ex2(kFar ? p1 + neg : p1);
            acc = add2(acc, pair2(p0, p1));
            pk[gk * 4 + j / 2] = __uint_as_float(pack_half2(p0, p1));
          }
          float a0, a1;
          unpair2(acc, a0, a1);
          sum = fmaf(a0 + a1, w.z, sum);
        }
        tmem_st16(tS + half * 16, pk);  // over keys of the first half, which are read
      };
      if constexpr (kTwice) {
#pragma unroll 1
        for (int half = 0; half < 2; ++half) {
          load_half(half, s[0]);
          weigh_half(half, s[0]);
        }
      } else {
#pragma unroll
        for (int half = 0; half < 2; ++half) weigh_half(half, s[half % kKept]);
      }
      tc_fence_before();
      mbar_arrive(&p_full[slot * 2 + (k & 1)]);
      return true;
    };
    int k = 0;
    while (k < n && __all_sync(0xffffffffu, ok) && fold_chunk(std::false_type{}, k)) ++k;
    for (; k < n && __all_sync(0xffffffffu, ok); ++k) fold_chunk(std::true_type{}, k);
    // ---- epilogue
    if (n > 0) ok = wait8(&fin[slot], 0, p.err) && ok;
    __syncwarp();
    const int64_t pairs = static_cast<int64_t>(p.M) * p.Hq;
    const int64_t record = (ksplit ? 2 * blockIdx.y + slot : blockIdx.y) * pairs;
    const bool direct = p.direct != 0;
    if (live && !direct) p.part_ml[record + pair] = make_float2(ref, sum);
    // O by way of shared memory (the chunks' space, once both slots are done with it): a thread lays its
    // row down and copies it out as one bulk transfer.  Rows are padded by 16 bytes against bank conflicts.
    asm volatile("bar.sync 1, 256;" ::: "memory");
    tc_fence_after();  // the loads of O stay behind the wait above, and the rows behind both slots' products
    constexpr int kRowOut = kHd * 4 + 16;
    uint8_t* row_s = ring8 + tid * kRowOut;
    const bool any = n > 0 && sum != 0.f;
    const float inv = !any ? 0.f : direct ? 1.f / sum : 1.f;
#pragma unroll 1
    for (int q4 = 0; q4 < 4; ++q4) {
      float ov[32];
      if (n > 0) tmem_ld32(tO + q4 * 32, ov);
      if (direct) {
#pragma unroll
        for (int i = 0; i < 32; i += 8) {
          T t[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) t[e] = from_f32<T>(any ? ov[i + e] * inv : 0.f);
          *reinterpret_cast<uint4*>(row_s + (q4 * 32 + i) * 2) = *reinterpret_cast<const uint4*>(t);
        }
      } else {
#pragma unroll
        for (int i = 0; i < 32; i += 4)
          *reinterpret_cast<float4*>(row_s + (q4 * 32 + i) * 4) = make_float4(ov[i], ov[i + 1], ov[i + 2], ov[i + 3]);
      }
    }
    fence_proxy_async_smem();
    if (live && (direct || any)) {
      void* to = direct ? static_cast<void*>(static_cast<T*>(p.out) + pair * kHd)
                        : static_cast<void*>(p.part_o + (record + pair) * kHd);
      bulk_store(to, row_s, direct ? kHd * 2 : kHd * 4);
    }
    bulk_store_wait();
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 0) tmem_dealloc(tmem, 512);
}

template <typename T, bool kSplitKeys, int kGroup>
static cudaError_t launch_tc_grouped(const CUtensorMap& map, const Attn8Params& p, cudaStream_t st) {
  static std::atomic<uint64_t> done{0};
  const cudaError_t e = allow_smem(attn8_tc_kernel<T, kSplitKeys, kGroup>, kSmem, done);
  if (e != cudaSuccess) return e;
  const int rows = p.M * (p.Hq / p.Hkv), tile = kSplitKeys ? 128 : 256;
  return launch_k(attn8_tc_kernel<T, kSplitKeys, kGroup>, dim3(p.Hkv, p.tc_splits, (rows + tile - 1) / tile),
                  dim3(Roles<kSplitKeys>::kThreads), kSmem, st, map, p);
}

template <typename T, bool kSplitKeys>
static cudaError_t launch_tc_typed(const CUtensorMap& map, const Attn8Params& p, cudaStream_t st) {
  return p.page_shift == 3 ? launch_tc_grouped<T, kSplitKeys, 8>(map, p, st)
                           : launch_tc_grouped<T, kSplitKeys, 16>(map, p, st);
}

cudaError_t launch_attention8_tc(const CUtensorMap& map, const Attn8Params& p, cudaStream_t st) {
  if (p.tc_ksplit)
    return p.bf16 ? launch_tc_typed<__nv_bfloat16, true>(map, p, st) : launch_tc_typed<__half, true>(map, p, st);
  return p.bf16 ? launch_tc_typed<__nv_bfloat16, false>(map, p, st) : launch_tc_typed<__half, false>(map, p, st);
}

}  // namespace atlas
