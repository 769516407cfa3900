// Host/device interface of the 8-bit paged KV cache kernels (head_dim 128).
//
// One layer of the cache is data [pages, 2 (k, v), Hkv, page_size, 128] of e4m3 codes and scale
// [pages, 2, Hkv] of fp32 powers of two; an element stands for code * scale, scale 0 marks a page
// that holds nothing.  Page sizes are 8, 16, 32 or 64 slots.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace atlas {

enum Kv8In : int { kKv8F16 = 0, kKv8Bf16 = 1, kKv8F32 = 2 };

struct Kv8AppendParams {
  const void* qkv;     // [M, (Hq + 2 Hkv) * 128], row stride `ld`
  const float* table;  // [max_pos, 128] cos | sin
  const int* pos;      // [M]
  const int* slots;    // [M]
  uint8_t* data;       // one layer
  float* scale;
  void* q_out;         // [M, Hq, 128]
  int* err;
  int64_t ld;
  int M, Hq, Hkv, page_shift, num_pages, max_pos;
  int in_type, out_bf16;
  int q_blocks, q_per_warp, kv_rows;  // launch shape, filled in by the launch
};
cudaError_t launch_kv8_append(const Kv8AppendParams& p, cudaStream_t st);

// plan [n, 3] (source page, destination page, tokens); count: device int bounding the rows used, or null.
cudaError_t launch_kv8_copy_pages(uint8_t* data, float* scale, const int* plan, const int* count, int n, int layers,
                                  int num_pages, int Hkv, int page_shift, int* err, cudaStream_t st);

constexpr int kKv8MaxMoves = 1024;
cudaError_t launch_kv8_move_slots(uint8_t* data, float* scale, const int* src, const int* dst, int n, int layers,
                                  int num_pages, int Hkv, int page_shift, int* err, cudaStream_t st);

// out [layers, n, 2, Hkv, page_size, 128] in fp16 or bf16.
cudaError_t launch_kv8_read_pages(const uint8_t* data, const float* scale, const int* pages, void* out, int n,
                                  int layers, int num_pages, int Hkv, int page_shift, bool bf16, int* err,
                                  cudaStream_t st);

struct Attn8Params {
  const void* q;         // [M, Hq, 128]
  const uint8_t* data;   // one layer
  const float* scale;
  void* out;             // [M, Hq, 128]
  const int* dparams;    // device scalars shared_len, n_shared_pages, mask_base; null: the fields below
  int shared_len, n_shared_pages, mask_base;
  const int* prefix_pages;
  const int* row_full;
  const int* row_len;
  const int64_t* row_mask;  // [M, mask_words]
  const int* tail_pages;    // [M, tail_stride]
  float* part_o;            // [splits, M, Hq, 128]
  float2* part_ml;          // [splits, M, Hq] (reference maximum in log2 units, sum of weights)
  int* err;
  int M, Hq, Hkv, page_shift, num_pages, n_prefix;
  int mask_words, tail_stride, splits, bf16;
  int row_tile;      // query rows of a kv head per CTA of the split pass: 16, 32, or 0 for the tcgen05 pass
  int tc_splits;     // tcgen05 pass: key splits (grid), each two records when tc_ksplit
  int tc_ksplit;     // both slots of a CTA hold the same 128 rows and take alternate chunks
  int causal_start;  // >= 0: row m is at position causal_start + m and sees the keys up to itself
  int direct;        // tcgen05 pass: one split, writes `out` itself
  float scale_log2;  // softmax scale * log2(e)
};
// map: the layer as rows of 128 bytes, box (128, min(page size, 16)), 128B swizzle.
cudaError_t launch_attention8(const CUtensorMap& map, const Attn8Params& p, cudaStream_t st);

// The tcgen05 pass alone: all there is to a direct call.
cudaError_t launch_attention8_tc(const CUtensorMap& map, const Attn8Params& p, cudaStream_t st);

}  // namespace atlas
