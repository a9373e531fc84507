// Internal interface between the runtime and the kernels of a decoder layer
// held in 8 and 4 bits: block quantization to e4m3 and products of such
// operands (block_fp8.hip), rotary positions (rotary.hip), the 4-bit cache of
// keys and values (cache4.hip).  Everything here works on GPU pointers only.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace om {

// Element types of activations; everything is computed in f32.
enum FloatKind : int { kF32 = 0, kF16 = 1, kBF16 = 2 };

// HIP counts a launch's threads in 32 bits along each axis, and takes more than that
// for what is left of them: a launch has at most this many blocks (of up to 256
// threads), and what needs more takes several.
constexpr int64_t kMostGrid = (int64_t)1 << 23;

// ---- e4m3 with a scale for each block --------------------------------------
constexpr int kBlock = 128; // elements of a row under one scale

// y e4m3 [M, K], scale f32 [ceil(M / rows), ceil(K / 128)]; rows 1 or 128.
hipError_t launch_quantize_blocks(hipStream_t s, const void *x, FloatKind kind,
    int64_t M, int64_t K, int rows, uint8_t *y, float *scale);

// y [M, N] = act(sum over blocks of a_scale b_scale (a . b) + bias)
struct BlockGemm {
  const uint8_t *a;      // e4m3 [M, K]
  const float *a_scale;  // [M, ceil(K / 128)]
  const uint8_t *b;      // e4m3 [N, K]
  const float *b_scale;  // [ceil(N / 128), ceil(K / 128)]
  const float *bias;     // null, [1] or [N]
  void *y;
  int64_t M, N, K;
  int64_t bias_len;
  FloatKind kind; // of y
  int activation; // OM_MI355X_ACTIVATION_*
  // Scratch, aligned to 16 bytes, without which the product is slower:
  uint8_t *rows; // block_gemm_row_bytes(): aligned copies of rows
  float *parts;  // block_gemm_part_bytes(): sums of parts of K
};
// 0: none is of use.  `parts` is asked for once `rows` is known.
size_t block_gemm_row_bytes(const BlockGemm &g);
size_t block_gemm_part_bytes(const BlockGemm &g);
hipError_t launch_block_gemm(hipStream_t s, const BlockGemm &g);

// ---- rotary positions ------------------------------------------------------
struct Rotary {
  const void *x;
  void *y;
  const float *cos, *sin;     // [positions, rot / 2], or [B, S, rot / 2]
  const int64_t *positions;   // [B, S], or null: row b * S + s of the tables
  int64_t B, S, H, table_rows;
  int D, rot;
  bool interleaved;
  bool heads_first; // [B, H, S, D], otherwise [B, S, H, D]
  FloatKind kind;
};
hipError_t launch_rotary(hipStream_t s, const Rotary &r);

// ---- 4-bit cache -----------------------------------------------------------
constexpr int kCacheGroup = 32; // elements under one scale and lowest value

// codes u8 [pages, H, page_size, D / 2], scales f16 [pages, H, page_size,
// D / 32, 2].  Token t of sequence b lies in page table[b * table_pages +
// t / page_size], or in page b where there is no table.
struct Cache4 {
  uint8_t *k_codes, *v_codes;
  uint16_t *k_scales, *v_scales;
  const int32_t *table; // [B, table_pages] or null
  const int32_t *past;  // [B]: tokens in front of the new ones
  const int32_t *counts; // [B]: new tokens, or null: S of each
  int64_t pages, page_size, table_pages;
  int H, D;
};
struct Append4 {
  Cache4 c;
  const void *k, *v;
  int64_t B, S;
  bool heads_first; // of k and v
  FloatKind kind;
};
hipError_t launch_cache_append(hipStream_t s, const Append4 &a);

struct Attention4 {
  Cache4 c;
  const void *q;
  void *y;
  const int32_t *starts; // [B]: first key of each sequence, or null
  const float *scale;    // [1], or null: 1 / sqrt(D)
  int64_t B, S, heads;
  int64_t window;        // keys a query sees at most, 0: all
  bool causal, heads_first;
  FloatKind kind;
  int splits;            // parts of the keys, attention_splits()
  float *parts;          // attention_parts_bytes(), if splits > 1
};
bool attention_head_ok(int D);
int attention_splits(const Attention4 &a);
size_t attention_parts_bytes(const Attention4 &a);
hipError_t launch_cache_attention(hipStream_t s, const Attention4 &a);

} // namespace om
