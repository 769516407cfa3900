// Python bindings of the 8-bit KV cache kernels.  Outputs and split records are allocated here, on
// the current stream (no workspace outlives a call, so calls on several streams and captured graphs
// share nothing), and every launch status becomes an exception.

#include "bindings_kv8.h"

#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>

#include <algorithm>
#include <cmath>
#include <string>

#include "kv8.h"

namespace {

constexpr double kLog2e = 1.4426950408889634;
constexpr int64_t kPositions = int64_t{1} << 30;  // positions and their differences fit 32 bits

// Numbers in messages: streaming one into TORCH_CHECK from this extension ends the process (its copy of
// the number formatting and torch's do not share their locale).
std::string str(int64_t n) { return std::to_string(n); }

// A cache data [L, pages, 2, Hkv, ps, 128] e4m3 with scale [L, pages, 2, Hkv], or one of its layers.
struct Cache8 {
  uint8_t* data;
  float* scale;
  int64_t layers, pages, Hkv, ps;
  int shift;  // log2(ps)
};

Cache8 check_cache(const torch::Tensor& data, const torch::Tensor& scale, int64_t layer = -1) {
  TORCH_CHECK(data.is_cuda() && data.dim() == 6 && data.is_contiguous() &&
                  data.scalar_type() == torch::kFloat8_e4m3fn,
              "the 8-bit cache must be a contiguous float8_e4m3fn CUDA tensor [L, pages, 2, Hkv, page, 128]");
  TORCH_CHECK(data.size(5) == 128 && data.size(2) == 2, "the 8-bit cache kernels need [L, pages, 2, Hkv, page, 128]");
  const int64_t L = data.size(0), pages = data.size(1), Hkv = data.size(3), ps = data.size(4);
  TORCH_CHECK(ps == 8 || ps == 16 || ps == 32 || ps == 64, "the 8-bit cache kernels need pages of 8, 16, 32 or 64 slots");
  TORCH_CHECK(scale.scalar_type() == torch::kFloat32 && scale.is_contiguous() && scale.device() == data.device() &&
                  scale.sizes() == data.sizes().slice(0, 4),
              "the 8-bit cache needs one float32 scale per page, side and head on its device");
  TORCH_CHECK(L > 0 && pages > 0 && Hkv > 0 && L <= 65535 && 2 * Hkv <= 65535 &&
                  pages * 2 * Hkv * ps < (int64_t{1} << 31),
              "a layer of the 8-bit cache holds fewer than 2^31 rows of 128 codes");
  TORCH_CHECK(reinterpret_cast<uintptr_t>(data.data_ptr()) % 16 == 0, "the 8-bit cache must be 16-byte aligned");
  TORCH_CHECK(layer >= -1 && layer < L, "layer ", str(layer), " of a cache of ", str(L));
  Cache8 c{static_cast<uint8_t*>(data.data_ptr()), scale.data_ptr<float>(), L, pages, Hkv, ps,
           ps == 8 ? 3 : ps == 16 ? 4 : ps == 32 ? 5 : 6};
  if (layer >= 0) {
    c.data += layer * pages * 2 * Hkv * ps * 128;
    c.scale += layer * pages * 2 * Hkv;
    c.layers = 1;
  }
  return c;
}

void check_int(const torch::Tensor& t, const torch::Tensor& like, const char* name, int64_t n = -1) {
  TORCH_CHECK(t.device() == like.device() && t.scalar_type() == torch::kInt32 && t.is_contiguous(), name,
              " must be a contiguous int32 tensor on the cache's device");
  TORCH_CHECK(n < 0 || t.numel() == n, name, " must hold ", str(n), " values, not ", str(t.numel()));
}

void check_err(const torch::Tensor& err, const torch::Tensor& like) {
  TORCH_CHECK(err.device() == like.device() && err.scalar_type() == torch::kInt32 && err.numel() >= 1,
              "the op table belongs to ", err.device().str(), ", the cache to ", like.device().str());
}

// An uninitialized tensor on `like`'s device, without the dispatcher's round (small calls are host-bound).
torch::Tensor fresh(at::IntArrayRef size, torch::ScalarType type, const torch::Tensor& like) {
  return at::detail::empty_cuda(size, type, like.device(), c10::nullopt);
}

void check_launch(cudaError_t e, const char* what) {
  TORCH_CHECK(e == cudaSuccess, what, ": ", cudaGetErrorString(e));
}

torch::Tensor kv8_append(torch::Tensor qkv, torch::Tensor table, torch::Tensor pos, torch::Tensor slots,
                         torch::Tensor data, torch::Tensor scale, int64_t layer, int64_t Hq, bool out_bf16,
                         torch::Tensor err) {
  TORCH_CHECK(layer >= 0, "layer ", str(layer));
  const Cache8 c = check_cache(data, scale, layer);
  check_err(err, data);
  const int64_t Hkv = c.Hkv, M = qkv.size(0);
  const auto t = qkv.scalar_type();
  TORCH_CHECK(t == torch::kHalf || t == torch::kBFloat16 || t == torch::kFloat32, "qkv must be fp16, bf16 or fp32");
  TORCH_CHECK(qkv.device() == data.device() && qkv.dim() == 2 && Hq >= 1 && qkv.size(1) == (Hq + 2 * Hkv) * 128,
              "qkv must be [M, (Hq + 2 Hkv) * 128] on the cache's device");
  if (qkv.stride(1) != 1 || (M > 1 && qkv.stride(0) % 4 != 0) || reinterpret_cast<uintptr_t>(qkv.data_ptr()) % 16 != 0)
    qkv = qkv.clone(at::MemoryFormat::Contiguous);
  TORCH_CHECK(table.device() == data.device() && table.scalar_type() == torch::kFloat32 && table.is_contiguous() &&
                  table.dim() == 2 && table.size(1) == 128 && table.size(0) < (int64_t{1} << 31) &&
                  reinterpret_cast<uintptr_t>(table.data_ptr()) % 16 == 0,
              "the rotary table must be contiguous fp32 [positions, 128] on the cache's device");
  check_int(pos, data, "positions", M);
  check_int(slots, data, "slots", M);
  TORCH_CHECK(M * (Hq + Hkv) < (int64_t{1} << 31), "kv8 append size");
  const bool bf16 = t == torch::kFloat32 ? out_bf16 : t == torch::kBFloat16;
  const c10::cuda::CUDAGuard guard(data.device());
  auto q = fresh({M, Hq, 128}, bf16 ? torch::kBFloat16 : torch::kHalf, data);
  atlas::Kv8AppendParams p{};
  p.qkv = qkv.data_ptr();
  p.table = table.data_ptr<float>();
  p.pos = pos.data_ptr<int>();
  p.slots = slots.data_ptr<int>();
  p.data = c.data;
  p.scale = c.scale;
  p.q_out = q.data_ptr();
  p.err = err.data_ptr<int>();
  p.ld = qkv.stride(0);
  p.M = static_cast<int>(M);
  p.Hq = static_cast<int>(Hq);
  p.Hkv = static_cast<int>(Hkv);
  p.page_shift = c.shift;
  p.num_pages = static_cast<int>(c.pages);
  p.max_pos = static_cast<int>(table.size(0));
  p.in_type = t == torch::kFloat32 ? atlas::kKv8F32 : t == torch::kBFloat16 ? atlas::kKv8Bf16 : atlas::kKv8F16;
  p.out_bf16 = bf16 ? 1 : 0;
  check_launch(atlas::launch_kv8_append(p, at::cuda::getCurrentCUDAStream()), "kv8_append");
  return q;
}

void kv8_copy_pages(torch::Tensor data, torch::Tensor scale, torch::Tensor plan, c10::optional<torch::Tensor> count,
                    torch::Tensor err) {
  const Cache8 c = check_cache(data, scale);
  check_err(err, data);
  check_int(plan, data, "the copy plan");
  TORCH_CHECK(plan.dim() == 2 && plan.size(1) == 3, "the copy plan must be [n, 3]");
  if (count.has_value()) {
    check_int(*count, data, "the copy count");
    TORCH_CHECK(count->numel() >= 1, "the copy count must hold one value");
  }
  const c10::cuda::CUDAGuard guard(data.device());
  check_launch(atlas::launch_kv8_copy_pages(c.data, c.scale, plan.data_ptr<int>(),
                                            count.has_value() ? count->data_ptr<int>() : nullptr,
                                            static_cast<int>(plan.size(0)), static_cast<int>(c.layers),
                                            static_cast<int>(c.pages), static_cast<int>(c.Hkv), c.shift,
                                            err.data_ptr<int>(), at::cuda::getCurrentCUDAStream()),
               "kv8_copy_pages");
}

void kv8_move_slots(torch::Tensor data, torch::Tensor scale, torch::Tensor src, torch::Tensor dst, torch::Tensor err) {
  const Cache8 c = check_cache(data, scale);
  check_err(err, data);
  check_int(src, data, "source slots");
  check_int(dst, data, "destination slots", src.numel());
  TORCH_CHECK(src.numel() <= atlas::kKv8MaxMoves, "at most ", str(atlas::kKv8MaxMoves), " slot moves per call, not ",
              str(src.numel()));
  const c10::cuda::CUDAGuard guard(data.device());
  check_launch(atlas::launch_kv8_move_slots(c.data, c.scale, src.data_ptr<int>(), dst.data_ptr<int>(),
                                            static_cast<int>(src.numel()), static_cast<int>(c.layers),
                                            static_cast<int>(c.pages), static_cast<int>(c.Hkv), c.shift,
                                            err.data_ptr<int>(), at::cuda::getCurrentCUDAStream()),
               "kv8_move_slots");
}

// One layer -> [n, 2, Hkv, ps, 128]; the whole cache (layer -1) -> [L, n, 2, Hkv, ps, 128].
torch::Tensor kv8_read_pages(torch::Tensor data, torch::Tensor scale, int64_t layer, torch::Tensor pages, bool bf16,
                             torch::Tensor err) {
  const Cache8 c = check_cache(data, scale, layer);
  check_err(err, data);
  check_int(pages, data, "pages");
  const int64_t n = pages.numel();
  const c10::cuda::CUDAGuard guard(data.device());
  const auto type = bf16 ? torch::kBFloat16 : torch::kHalf;
  auto out = layer < 0 ? fresh({c.layers, n, 2, c.Hkv, c.ps, 128}, type, data)
                       : fresh({n, 2, c.Hkv, c.ps, 128}, type, data);
  check_launch(atlas::launch_kv8_read_pages(c.data, c.scale, pages.data_ptr<int>(), out.data_ptr(),
                                            static_cast<int>(n), static_cast<int>(c.layers),
                                            static_cast<int>(c.pages), static_cast<int>(c.Hkv), c.shift, bf16,
                                            err.data_ptr<int>(), at::cuda::getCurrentCUDAStream()),
               "kv8_read_pages");
  return out;
}

// The split pass's launch shape for `rows` query rows of a kv head (query rows times group).
//
// The register tensor-core pass takes tiles of 16 rows (two CTAs per SM) or 32; its work is a term per tile
// and key.  The tcgen05 pass holds 128 rows over alternate chunks of keys, or 256 rows, in a CTA: it starts
// about 5 us later and then spends on all of its rows what the other spends on 2.5 tiles of 16.  Hence the
// border: Hkv * keys * (tiles - 2.5) = 120 K (us, tiles of 16 against tcgen05; 8 kv heads: 48 rows on 4096
// keys 13.9 / 17.4, on 16K 26.4 / 29.8, on 64K 75.9 / 66.6; 96 rows on 4096 18.0 / 18.0, on 8192 25.9 / 23.6;
// 160 rows on 1024 13.6 / 15.9, on 4096 25.8 / 19.8; 16 kv heads, 320 rows on 300: 23.2 / 18.9, more CTAs
// than fit at once).  Up to 32 rows it never pays, and one tile of 32 beats two of 16 from Hkv * keys = 128 K
// on (8 kv heads, 20 rows: 4096 keys 12.8 / 11.9, 64K 50.1 / 54.9).
//
// The splits fill the CTA slots with at least 128 keys each up to eight splits and 256 beyond (36 rows on
// 2051 keys: 17 splits 16.8 us, 9 splits 15.1 us; 48 rows on 1000 keys: 8 splits 10.9 us, 4 splits 12.4 us).
void pick_shape8(atlas::Attn8Params& p, int64_t rows, int64_t keys, int sms) {
  const int64_t tiles = (rows + 15) / 16, work = p.Hkv * keys;
  const bool registers = tiles <= 2 || (work * (2 * tiles - 5) < 240 * 1024 && tiles * p.Hkv <= 2 * sms);
  p.row_tile = p.causal_start >= 0 || !registers ? 0 : tiles == 2 && work >= 128 * 1024 ? 32 : 16;
  p.tc_ksplit = rows <= 128 ? 1 : 0;
  const int64_t tile = p.row_tile ? p.row_tile : p.tc_ksplit ? 128 : 256;
  const int64_t slots = static_cast<int64_t>(sms) * (p.row_tile == 16 ? 2 : 1);
  const int64_t ctas = p.Hkv * ((rows + tile - 1) / tile);
  const int64_t most = p.row_tile == 0 && p.tc_ksplit ? 32 : 64;  // records
  // A causal chunk writes its output directly unless splits of 512 keys help (301 rows of a fresh prompt:
  // direct 15.4 us, three splits and their merge 21.0 us; 100 rows behind 4000 keys: 26.3 us with splits).
  const int64_t useful = p.causal_start >= 0
                             ? keys / 512
                             : std::max<int64_t>((keys + 255) / 256, std::min<int64_t>(8, (keys + 127) / 128));
  const int64_t n = std::max<int64_t>(1, std::min<int64_t>({most, slots / ctas, useful}));
  p.tc_splits = static_cast<int>(n);
  p.splits = static_cast<int>(most == 32 ? 2 * n : n);
  if (p.causal_start >= 0 && n == 1) {  // no split of the keys: rows of 256 write their output directly
    p.tc_ksplit = 0;
    p.direct = 1;
    p.splits = 0;
  }
}

// The splits' records: a partial row (unnormalized, fp32) and its (reference, sum) per split and query head.
torch::Tensor split_records(atlas::Attn8Params& p, const torch::Tensor& data) {
  if (p.splits == 0) return {};
  const int64_t rows = static_cast<int64_t>(p.splits) * p.M * p.Hq;
  torch::Tensor parts = fresh({rows * 130}, torch::kFloat32, data);
  p.part_o = parts.data_ptr<float>();
  p.part_ml = reinterpret_cast<float2*>(p.part_o + rows * 128);
  return parts;
}

void check_q8(torch::Tensor& q, const torch::Tensor& data, const Cache8& c, double softmax_scale) {
  TORCH_CHECK(q.device() == data.device() && q.dim() == 3 && q.size(2) == 128 &&
                  (q.scalar_type() == torch::kHalf || q.scalar_type() == torch::kBFloat16),
              "q must be fp16 or bf16 [M, Hq, 128] on the cache's device");
  TORCH_CHECK(q.size(1) >= 1 && q.size(1) % c.Hkv == 0, "Hq must be a multiple of Hkv");
  TORCH_CHECK(q.size(0) * (q.size(1) / c.Hkv) <= 65535 * 128,
              "attention8 takes at most 65535 * 128 query rows per kv head");
  TORCH_CHECK(softmax_scale > 0 && std::isfinite(softmax_scale), "the softmax scale must be positive and finite");
  if (!q.is_contiguous() || reinterpret_cast<uintptr_t>(q.data_ptr()) % 16 != 0)
    q = q.clone(at::MemoryFormat::Contiguous);
}

atlas::Attn8Params params8(const torch::Tensor& q, const Cache8& c, const torch::Tensor& out,
                            const torch::Tensor& prefix_pages, double softmax_scale, const torch::Tensor& err) {
  atlas::Attn8Params p{};
  p.q = q.data_ptr();
  p.data = c.data;
  p.scale = c.scale;
  p.out = out.data_ptr();
  p.prefix_pages = prefix_pages.data_ptr<int>();
  p.err = err.data_ptr<int>();
  p.M = static_cast<int>(q.size(0));
  p.Hq = static_cast<int>(q.size(1));
  p.Hkv = static_cast<int>(c.Hkv);
  p.page_shift = c.shift;
  p.num_pages = static_cast<int>(c.pages);
  p.n_prefix = static_cast<int>(prefix_pages.numel());
  p.bf16 = q.scalar_type() == torch::kBFloat16;
  p.scale_log2 = static_cast<float>(softmax_scale * kLog2e);
  p.causal_start = -1;
  return p;
}

// Returns the output and the number of kernels launched.
std::pair<torch::Tensor, int64_t> attention8(torch::Tensor q, torch::Tensor data, torch::Tensor scale, int64_t layer,
                                             c10::optional<torch::Tensor> dparams, int64_t shared_len,
                                             int64_t n_shared_pages, int64_t mask_base, torch::Tensor prefix_pages,
                                             torch::Tensor row_full, torch::Tensor row_len, torch::Tensor row_mask,
                                             torch::Tensor tail_pages, double softmax_scale, int64_t max_keys,
                                             torch::Tensor err) {
  TORCH_CHECK(layer >= 0, "layer ", str(layer));
  const Cache8 c = check_cache(data, scale, layer);
  check_err(err, data);
  check_q8(q, data, c, softmax_scale);
  const int64_t M = q.size(0), Hq = q.size(1), Hkv = c.Hkv;
  check_int(prefix_pages, data, "prefix_pages");
  check_int(row_full, data, "row_full", M);
  check_int(row_len, data, "row_len", M);
  TORCH_CHECK(row_mask.device() == data.device() && row_mask.scalar_type() == torch::kInt64 &&
                  row_mask.is_contiguous() && row_mask.dim() == 2 && row_mask.size(0) == M,
              "row_mask must be contiguous int64 [M, words] on the cache's device");
  check_int(tail_pages, data, "tail_pages");
  TORCH_CHECK(tail_pages.dim() == 2 && tail_pages.size(0) == M, "tail_pages must be [M, T]");
  TORCH_CHECK(shared_len >= 0 && shared_len < kPositions && n_shared_pages >= 0 &&
                  n_shared_pages < (kPositions >> c.shift),
              "shared_len and n_shared_pages must be positions below 2^30");
  TORCH_CHECK((prefix_pages.numel() << c.shift) < kPositions &&
                  ((n_shared_pages + tail_pages.size(1)) << c.shift) < kPositions,
              "the descriptor's page lists must end below position 2^30");
  TORCH_CHECK(mask_base > -kPositions && mask_base < kPositions, "mask_base must be a position below 2^30");
  if (dparams.has_value()) {
    check_int(*dparams, data, "the descriptor's device scalars");
    TORCH_CHECK(dparams->numel() >= 3, "the descriptor's device scalars are shared_len, n_shared_pages, mask_base");
  }
  const c10::cuda::CUDAGuard guard(data.device());
  auto out = fresh({M, Hq * 128}, q.scalar_type(), data);
  if (M == 0) return {out, 0};
  atlas::Attn8Params p = params8(q, c, out, prefix_pages, softmax_scale, err);
  p.dparams = dparams.has_value() ? dparams->data_ptr<int>() : nullptr;
  p.shared_len = static_cast<int>(shared_len);
  p.n_shared_pages = static_cast<int>(n_shared_pages);
  p.mask_base = static_cast<int>(mask_base);
  p.row_full = row_full.data_ptr<int>();
  p.row_len = row_len.data_ptr<int>();
  p.row_mask = row_mask.data_ptr<int64_t>();
  p.tail_pages = tail_pages.data_ptr<int>();
  p.mask_words = static_cast<int>(row_mask.size(1));
  p.tail_stride = static_cast<int>(tail_pages.size(1));
  // A captured call is sized for the longest context its graph may see (max_keys), an eager one for its own.
  const int64_t keys = std::max<int64_t>({shared_len, n_shared_pages << c.shift, max_keys});
  CUtensorMap map{};
  if (keys > 0 || dparams.has_value()) {
    pick_shape8(p, M * (Hq / Hkv), keys, at::cuda::getCurrentDeviceProperties()->multiProcessorCount);
    map = map_kv8(c.data, c.pages * 2 * Hkv * c.ps, c.ps);
  }
  const torch::Tensor parts = split_records(p, data);
  check_launch(atlas::launch_attention8(map, p, at::cuda::getCurrentCUDAStream()), "attention8");
  return {out, p.splits > 0 ? 2 : 1};
}

// Row m is at position start + m and sees the keys up to itself, all in prefix_pages.
std::pair<torch::Tensor, int64_t> attention8_causal(torch::Tensor q, torch::Tensor data, torch::Tensor scale,
                                                    int64_t layer, torch::Tensor prefix_pages, int64_t start,
                                                    double softmax_scale, torch::Tensor err) {
  TORCH_CHECK(layer >= 0, "layer ", str(layer));
  const Cache8 c = check_cache(data, scale, layer);
  check_err(err, data);
  check_q8(q, data, c, softmax_scale);
  check_int(prefix_pages, data, "prefix_pages");
  const int64_t M = q.size(0), ps = c.ps;
  TORCH_CHECK(start >= 0 && start < kPositions && start + M < kPositions, "positions must be in [0, 2^30)");
  const int64_t n = (start + M + ps - 1) / ps;
  TORCH_CHECK(n <= prefix_pages.numel(), str(start + M), " positions need ", str(n), " pages of ", str(ps),
              " slots; the descriptor lists ", str(prefix_pages.numel()));
  const c10::cuda::CUDAGuard guard(data.device());
  auto out = fresh({M, q.size(1) * 128}, q.scalar_type(), data);
  if (M == 0) return {out, 0};
  atlas::Attn8Params p = params8(q, c, out, prefix_pages, softmax_scale, err);
  p.causal_start = static_cast<int>(start);
  p.shared_len = static_cast<int>(start + M);
  // A short chunk behind a long prefix has too few row tiles to fill the device: its keys are split.
  pick_shape8(p, M * (q.size(1) / c.Hkv), start + M, at::cuda::getCurrentDeviceProperties()->multiProcessorCount);
  const torch::Tensor parts = split_records(p, data);
  check_launch(atlas::launch_attention8(map_kv8(c.data, c.pages * 2 * c.Hkv * ps, ps), p,
                                        at::cuda::getCurrentCUDAStream()),
               "attention8_causal");
  return {out, p.direct ? 1 : 2};
}

}  // namespace

void register_kv8(pybind11::module& m) {
  m.def("kv8_append", &kv8_append, "rotary embedding and rounding of k and v into the 8-bit cache; returns rotated q");
  m.def("kv8_copy_pages", &kv8_copy_pages, "copies of partial pages in every layer of the 8-bit cache");
  m.def("kv8_move_slots", &kv8_move_slots, "slot moves in every layer of the 8-bit cache (sources read first)");
  m.def("kv8_read_pages", &kv8_read_pages, "pages of the 8-bit cache as fp16 or bf16 values");
  m.def("attention8_causal", &attention8_causal, "causal attention of a prefill chunk over one layer of the 8-bit cache");
  m.def("attention8", &attention8, "paged attention over one layer of the 8-bit cache");
}
