// 8-bit floating point (e4m3) with one f32 scale for each block of 128:
// quantization, and products of such operands.
//
//   quantize   s = max(max |x| / 448, 2^-126) over the block,  y = e4m3(x / s)
//   product    y[m,n] = act(sum_kb sa[m,kb] sb[n/128,kb] sum_{k in kb} a[m,k] b[n,k] + bias[n])
//
// b is [N, K], as weights lie in memory (Gemm with transB = 1): both operands
// of a matrix instruction are then 16 or 32 neighbouring bytes of a row.

#include "gemm_common.h"
#include "llm_common.h"
#include "om_mi355x.h"

namespace om {
namespace llm {
namespace {

// ---------------------------------------------------------------------------
// quantization
// ---------------------------------------------------------------------------
constexpr float kE4M3Max = 448.0f;
constexpr float kTiny = 0x1p-126f; // scales below are subnormal

__device__ __forceinline__ float block_scale(float top) {
  return __builtin_fmaxf(top / kE4M3Max, kTiny);
}

// x / s, correctly rounded, in four instructions instead of the divide's
// eleven where r = RN(1 / s) (Markstein's correction of a quotient, "Computation of
// elementary functions on the IBM RISC System/6000", 1990): q0 = RN(x r), e = x - q0 s
// (exact), q = RN(q0 + e r).  Nothing under- or overflows for scales from 2^-80 to 2^96 and
// quotients of 2^-11 .. 1024; smaller ones become 0 either way, larger ones do
// not occur or are infinite, and clamped they give 448, as they would divided.
// Other scales, an infinite block's among them, take the divide.
template <bool TAME>
__device__ __forceinline__ float block_quotient(float x, float s, float r) {
  float q;
  if (TAME) {
    const float q0 = x * r;
    q = __builtin_fmaf(__builtin_fmaf(-q0, s, x), r, q0);
  } else {
    q = x / s;
  }
  // (NaN stays NaN: med3 would return a bound)
  return q > kE4M3Max ? kE4M3Max : q < -kE4M3Max ? -kE4M3Max : q;
}

template <bool TAME, int N>
__device__ __forceinline__ void quantize_n(
    const float (&x)[N], float s, unsigned (&out)[N / 4]) {
  const float r = TAME ? 1.0f / s : 0.0f;
#pragma unroll
  for (int i = 0; i < N / 4; ++i) {
    float q[4];
#pragma unroll
    for (int j = 0; j < 4; ++j)
      q[j] = block_quotient<TAME>(x[4 * i + j], s, r);
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(q[0], q[1], 0, false);
    w = __builtin_amdgcn_cvt_pk_fp8_f32(q[2], q[3], w, true);
    out[i] = (unsigned)w;
  }
}
template <int N>
__device__ __forceinline__ void quantize_any(
    const float (&x)[N], float s, unsigned (&out)[N / 4]) {
  if (__all(s >= 0x1p-80f && s <= 0x1p96f))
    quantize_n<true>(x, s, out);
  else
    quantize_n<false>(x, s, out);
}

// Elements k .. k + 7 of a row; what lies past its end is 0.
template <typename T, bool WIDE>
__device__ __forceinline__ void load8(
    const T *row, int k, int K, float (&v)[8]) {
  if (WIDE) { // (K is a multiple of 8)
    if (k < K) {
      Pack<T, 8> p; // two 16-byte loads of f32, one of 16-bit types
#pragma unroll
      for (int i = 0; i < 8; i += 16 / (int)sizeof(T))
        *(Pack<T, 16 / sizeof(T)> *)(p.v + i) =
            *(const Pack<T, 16 / sizeof(T)> *)(row + k + i);
#pragma unroll
      for (int i = 0; i < 8; ++i)
        v[i] = to_f32(p.v[i]);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        v[i] = 0.0f;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      v[i] = k + i < K ? to_f32(row[k + i]) : 0.0f;
  }
}
template <bool WIDE>
__device__ __forceinline__ void store8(
    uint8_t *row, int k, int K, const unsigned (&w)[2]) {
  if (WIDE) {
    if (k < K)
      *(v2u *)(row + k) = v2u{w[0], w[1]};
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (k + i < K)
        row[k + i] = (uint8_t)(w[i / 4] >> (8 * (i % 4)));
  }
}

// One row's blocks.  16 lanes hold a block, 8 elements each, and find its
// largest by rotating within their 16; nothing passes through LDS.  Bound by
// memory: every element is read once, every code written once.
template <typename T, bool WIDE, int UNROLL>
__global__ __launch_bounds__(256) void k_quantize_rows(
    const T *x, uint8_t *y, float *scale, int64_t blocks, int K, int per_row) {
  const int lane16 = threadIdx.x & 15;
  int64_t at = ((int64_t)blockIdx.x * 256 + threadIdx.x) / 16 * UNROLL;
  float v[UNROLL][8];
  int64_t row[UNROLL];
  int kb[UNROLL];
#pragma unroll
  for (int u = 0; u < UNROLL; ++u) {
    const int64_t b = at + u < blocks ? at + u : blocks - 1;
    row[u] = (uint64_t)b >> 32 ? b / per_row : (unsigned)b / (unsigned)per_row;
    kb[u] = (int)(b - row[u] * per_row);
    load8<T, WIDE>(x + row[u] * K, kb[u] * kBlock + lane16 * 8, K, v[u]);
  }
#pragma unroll
  for (int u = 0; u < UNROLL; ++u) {
    float top = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i)
      top = __builtin_fmaxf(top, __builtin_fabsf(v[u][i]));
    const float s = block_scale(row_max(top));
    unsigned w[2];
    quantize_any(v[u], s, w);
    if (at + u < blocks) {
      store8<WIDE>(y + row[u] * K, kb[u] * kBlock + lane16 * 8, K, w);
      if (lane16 == 0)
        scale[at + u] = s;
    }
  }
}

// Blocks of 128 rows: a workgroup holds one, thread (r, c) elements 8 c .. of
// rows r, r + 16, ...
template <typename T, bool WIDE>
__global__ __launch_bounds__(256) void k_quantize_tiles(
    const T *x, uint8_t *y, float *scale, int64_t M, int K, int per_row) {
  __shared__ float tops[16];
  const int lane16 = threadIdx.x & 15, r0 = threadIdx.x >> 4;
  const int64_t tile = (unsigned)blockIdx.x / (unsigned)per_row;
  const int k = (int)(blockIdx.x - tile * per_row) * kBlock + lane16 * 8;
  float v[8][8];
  float top = 0.0f;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int64_t row = tile * 128 + j * 16 + r0;
    if (row < M) {
      load8<T, WIDE>(x + row * K, k, K, v[j]);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        v[j][i] = 0.0f;
    }
  }
#pragma unroll
  for (int j = 0; j < 8; ++j)
#pragma unroll
    for (int i = 0; i < 8; ++i)
      top = __builtin_fmaxf(top, __builtin_fabsf(v[j][i]));
  top = row_max(top);
  if (lane16 == 0)
    tops[r0] = top;
  __syncthreads();
  const float s = block_scale(row_max(tops[lane16]));
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int64_t row = tile * 128 + j * 16 + r0;
    unsigned w[2];
    quantize_any(v[j], s, w);
    if (row < M)
      store8<WIDE>(y + row * K, k, K, w);
  }
  if (threadIdx.x == 0)
    scale[blockIdx.x] = s;
}

// (A launch's rows, or tiles of 128: those of the most blocks that it may have.)
template <typename T>
hipError_t quantize(hipStream_t st, const T *x, int64_t M, int64_t K, int rows,
    uint8_t *y, float *scale) {
  const int per_row = (int)((K + kBlock - 1) / kBlock);
  const bool wide = K % 8 == 0 && ((uintptr_t)x & 15) == 0 && ((uintptr_t)y & 7) == 0;
  constexpr int U = 2;
  const int64_t most = rows == 1 ? kMostGrid * 16 * U / per_row : kMostGrid / per_row * 128;
  for (; M > 0; M -= most) {
    const int64_t m = M < most ? M : most;
    if (rows == 1) {
      const int64_t blocks = m * per_row;
      const dim3 grid((unsigned)((blocks + 16 * U - 1) / (16 * U)));
      if (wide)
        k_quantize_rows<T, true, U><<<grid, 256, 0, st>>>(x, y, scale, blocks, (int)K, per_row);
      else
        k_quantize_rows<T, false, U><<<grid, 256, 0, st>>>(x, y, scale, blocks, (int)K, per_row);
    } else {
      const dim3 grid((unsigned)((m + 127) / 128 * per_row));
      if (wide)
        k_quantize_tiles<T, true><<<grid, 256, 0, st>>>(x, y, scale, m, (int)K, per_row);
      else
        k_quantize_tiles<T, false><<<grid, 256, 0, st>>>(x, y, scale, m, (int)K, per_row);
    }
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess)
      return e;
    x += m * K;
    y += m * K;
    scale += (m + rows - 1) / rows * per_row;
  }
  return hipSuccess;
}

// ---------------------------------------------------------------------------
// products
// ---------------------------------------------------------------------------
// The matrix instructions for 8-bit operands take eight neighbouring products at a
// time and drop, toward zero, what lies below 2^-13 of 2^E, E the largest sum of two
// operands' exponents among them (at least -6 each); the eights are joined, and the
// blocks added, in f32.  (Found by single products beside large ones that cancel, and
// held by a test.)  A result is off by less than 2^-10 times the sum of all 2^E: by
// 1.1e-5 of the results' root mean square in the mean on normally distributed operands,
// 2.2e-5 where 1 % of the channels are 16 times as large (K = 4096).  That is far below
// the rounding of results in bf16 (1.7e-3) and below that of f16 (2.1e-4), and they run
// twice as fast as those for bf16, so results in 16 bits take them.  Where large
// products cancel it is not below: f32 results are there for that, summed by the bf16
// instructions (6e-8 to 1.4e-7 on the same operands), which hold every e4m3 value
// exactly; so are those of few rows, which are bound by reading weights.

// Four e4m3 values of a word, two to each result.
__device__ __forceinline__ void widen4(unsigned w, v2bf &lo, v2bf &hi) {
  lo = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, false);
  hi = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, true);
}
// Eight of two words: an operand of a 16x16x32 instruction.
__device__ __forceinline__ v8bf widen8(unsigned w0, unsigned w1) {
  v2bf a, b, c, d;
  widen4(w0, a, b);
  widen4(w1, c, d);
  return v8bf{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// The operands of the four instructions of a block of 128, from a lane's bytes of
// either half of it.
__device__ __forceinline__ void widen16(v4u l, v4u u, v8bf (&w)[4]) {
  w[0] = widen8(l[0], l[1]);
  w[1] = widen8(l[2], l[3]);
  w[2] = widen8(u[0], u[1]);
  w[3] = widen8(u[2], u[3]);
}
__device__ __forceinline__ v8i operand(v4u l, v4u u) {
  return v8i{(int)l[0], (int)l[1], (int)l[2], (int)l[3], (int)u[0], (int)u[1],
      (int)u[2], (int)u[3]};
}
__device__ __forceinline__ void add_scaled(float (&total)[4], v4f acc, float s) {
#pragma unroll
  for (int r = 0; r < 4; ++r)
    total[r] = __builtin_fmaf(acc[r], s, total[r]);
}

struct GemmParams {
  const uint8_t *a, *b;
  const float *a_scale, *b_scale, *bias;
  void *y;
  int M, N, K;
  int lda, ldb;      // bytes from row to row
  int kblocks;       // scales of a row: ceil(K / 128) of the caller's K
  int bias_step;     // 0: one bias for all columns
  int activation;
  int parts;         // of the blocks of K, part_blocks each
  int part_blocks;
  int part_pitch;    // N, rounded up to whole pieces of four
  float *part_sums;  // [parts, M, part_pitch] if parts > 1
};

__device__ __forceinline__ float finish(float v, const GemmParams &p, float bias) {
  v += bias;
  if (p.activation == OM_MI355X_ACTIVATION_RELU)
    v = __builtin_fmaxf(v, 0.0f);
  else if (p.activation == OM_MI355X_ACTIVATION_GELU)
    v = gemm::gelu_f32(v);
  return v;
}

// 16 bytes at any element of type T.
template <typename T> struct Loose {
  typedef unsigned v4 __attribute__((ext_vector_type(4), aligned(2)));
};
template <> struct Loose<float> {
  typedef unsigned v4 __attribute__((ext_vector_type(4), aligned(4)));
};

// Four neighbouring columns n .. n + 3 of row m; those past N are left out.
template <typename T>
__device__ __forceinline__ void store4(
    const GemmParams &p, int m, int n, const float (&v)[4]) {
  T *const y = (T *)p.y + (int64_t)m * p.N + n;
  T t[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int c = n + i < p.N ? n + i : p.N - 1;
    const float bias = p.bias ? p.bias[c * p.bias_step] : 0.0f;
    t[i] = from_f32<T>(finish(v[i], p, bias));
  }
  if (n + 4 <= p.N) { // (rows may start at any element)
    struct __attribute__((packed, aligned(alignof(T)))) Four {
      T v[4];
    };
    *(Four *)y = Four{{t[0], t[1], t[2], t[3]}};
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (n + i < p.N)
        y[i] = t[i];
  }
}

// 16 bytes a lane from `from` + at + k (k the same in all lanes) into LDS, the wave's
// from `to` on, one after the other.  Nothing comes from `bytes` on where k is 0: only
// a lane's own offset takes part in the range check.
__device__ __forceinline__ void copy16(
    const void *from, void *to, int at, int k, unsigned bytes = 0x7FFFFFFF) {
  typedef __attribute__((address_space(3))) void *lds_ptr;
  __builtin_amdgcn_raw_ptr_buffer_load_lds(
      __builtin_amdgcn_make_buffer_rsrc((void *)from, 0, bytes, 0x00020000),
      (lds_ptr)to, 16, at, k, 0, 0);
}

// --- few rows ---------------------------------------------------------------
// Up to 16 MT rows: a block owns 16 columns, its WAVES waves take every
// WAVES-th block of 128 of K.  Bound by reading the weights once: a wave has the
// weights of DEPTH blocks on their way, lanes (c, h) the bytes 16 h .. of each half
// of column c's 128, whole lines together; rows of a that are not there are not
// asked for.  Scales come by way of LDS, once a block: asked for by every wave,
// the few lines that hold them are what L2 is busiest with.  Products by bf16
// instructions; sums of the waves meet in LDS in a fixed order.
// One row, 4096 x 11008: 11.1 us (12.4 with scales asked for by every wave, 11.9
// with the weights copied into LDS, 9.8 with neither rows of a nor scales); 16 rows 14.7.
// TAIL: any K and any alignment, what lies past a row's end 0; and any number of
// rows, 16 MT a blockIdx.y, for products that have no room for aligned copies.
template <typename T, int MT, int WAVES, int DEPTH, bool TAIL, bool STAGED>
__global__ __launch_bounds__(WAVES * 64) void k_block_skinny(GemmParams p) {
  if (TAIL) {
    const int m0 = blockIdx.y * (16 * MT);
    p.a += (int64_t)m0 * p.lda;
    p.a_scale += (int64_t)m0 * p.kblocks;
    p.y = (T *)p.y + (int64_t)m0 * p.N;
    p.M = p.M - m0 < 16 * MT ? p.M - m0 : 16 * MT;
  }
  extern __shared__ float staged[]; // scales of b's columns, then of a's rows
  __shared__ v4f sums[WAVES][MT][64];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c = lane & 15, h = lane >> 4;
  const int n0 = blockIdx.x * 16;
  const int col = n0 + c < p.N ? n0 + c : p.N - 1;
  const uint8_t *const b = p.b + (int64_t)col * p.ldb + 16 * h;
  const uint8_t *a[MT];
  int a_row[MT];
#pragma unroll
  for (int i = 0; i < MT; ++i) {
    a_row[i] = 16 * i + c < p.M ? 16 * i + c : p.M - 1;
    a[i] = p.a + (int64_t)a_row[i] * p.lda + 16 * h;
  }
  const float *const bs = p.b_scale + (int64_t)(n0 / kBlock) * p.kblocks;

  float total[MT][4];
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int r = 0; r < 4; ++r)
      total[i][r] = 0.0f;

  v4u wb[DEPTH][2], wa[DEPTH][MT][2];
  // 16 bytes of a row from k on; past its end they are 0.
  auto load16 = [&](const uint8_t *row, int k) -> v4u {
    if (!TAIL)
      return *(const v4u *)(row + k);
    v4u w = {0, 0, 0, 0};
    const int left = p.K - k - 16 * h;
    if (left >= 16) {
      typedef unsigned v4u_any __attribute__((ext_vector_type(4), aligned(1)));
      return *(const v4u_any *)(row + k);
    }
#pragma unroll
    for (int i = 0; i < 16; ++i)
      if (i < left)
        w[i / 4] |= (unsigned)row[k + i] << (8 * (i % 4));
    return w;
  };
  auto fetch = [&](int d, int kb) {
    const int k = kb * kBlock;
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      wb[d][half] = load16(b, k + 64 * half);
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        wa[d][i][half] = v4u{0, 0, 0, 0};
        if (16 * i + c < p.M)
          wa[d][i][half] = load16(a[i], k + 64 * half);
      }
    }
  };
  // (the scales are asked for first: loads come back in order)
  const int scales = (p.M + 1) * p.kblocks;
  auto scale = [&](int i) {
    i = i < scales ? i : scales - 1;
    return i < p.kblocks ? bs + i : p.a_scale + (i - p.kblocks);
  };
  float mine = 0.0f;
  if (STAGED && scales > 0)
    mine = *scale(threadIdx.x);
  __builtin_amdgcn_sched_barrier(0);
#pragma unroll
  for (int d = 0; d < DEPTH; ++d)
    if (wave + d * WAVES < p.kblocks)
      fetch(d, wave + d * WAVES);
  if (STAGED) {
    __builtin_amdgcn_sched_barrier(0);
    if ((int)threadIdx.x < scales)
      staged[threadIdx.x] = mine;
    for (int i = threadIdx.x + WAVES * 64; i < scales; i += WAVES * 64)
      staged[i] = *scale(i);
    gemm::lds_barrier();
  }
  auto b_scale = [&](int kb) { return STAGED ? staged[kb] : bs[kb]; };
  auto a_scale = [&](int i, int kb) {
    return STAGED ? staged[p.kblocks + a_row[i] * p.kblocks + kb]
                  : p.a_scale[(int64_t)a_row[i] * p.kblocks + kb];
  };
  for (int kb = wave; kb < p.kblocks; kb += DEPTH * WAVES) {
#pragma unroll
    for (int d = 0; d < DEPTH; ++d) {
      const int at = kb + d * WAVES;
      if (at >= p.kblocks)
        break;
      const float sb = b_scale(at);
      v4f acc[MT];
#pragma unroll
      for (int i = 0; i < MT; ++i)
        acc[i] = v4f{0, 0, 0, 0};
#pragma unroll
      for (int half = 0; half < 2; ++half)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const v8bf fb = widen8(wb[d][half][2 * j], wb[d][half][2 * j + 1]);
#pragma unroll
          for (int i = 0; i < MT; ++i)
            acc[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fb,
                widen8(wa[d][i][half][2 * j], wa[d][i][half][2 * j + 1]), acc[i], 0,
                0, 0);
        }
#pragma unroll
      for (int i = 0; i < MT; ++i)
        add_scaled(total[i], acc[i], a_scale(i, at) * sb);
      if (at + DEPTH * WAVES < p.kblocks)
        fetch(d, at + DEPTH * WAVES);
    }
  }
#pragma unroll
  for (int i = 0; i < MT; ++i)
    sums[wave][i][lane] = v4f{total[i][0], total[i][1], total[i][2], total[i][3]};
  __syncthreads();
  // lane (c, h) of wave i: row 16 i + c, columns n0 + 4 h ..
  for (int i = wave; i < MT; i += WAVES) {
    v4f t = {0, 0, 0, 0};
#pragma unroll
    for (int w = 0; w < WAVES; ++w)
      t += sums[w][i][lane];
    const float v[4] = {t[0], t[1], t[2], t[3]};
    if (16 * i + c < p.M)
      store4<T>(p, 16 * i + c, n0 + 4 * h, v);
  }
}

// --- tiles ------------------------------------------------------------------
// BM x BN tiles, WM x WN waves.  A step is one block of 128 of K: the rows'
// 128 bytes go straight into LDS (two or three stages), 16-byte chunk q of row r at
// place q ^ (r % 8), so that neither the copies nor the operand reads meet a
// bank twice.  Columns are the first operand of the matrix instruction, so a
// lane holds one row of the result and four neighbouring columns: one scale
// for all it gets from an instruction, and whole pieces to store.  A part of
// the blocks of K (parts > 1) leaves f32 sums for k_join_parts.
template <typename T, int BM, int BN, int WM, int WN, int STAGES, bool EXACT>
__global__ __launch_bounds__(WM * WN * 64, 2) void k_block_tile(const GemmParams p) {
  constexpr int THREADS = WM * WN * 64, STAGE = (BM + BN) * kBlock;
  constexpr int TM = BM / WM / 16, TN = BN / WN / 16;
  constexpr int COPIES = STAGE / (THREADS * 16); // of 16 bytes a thread
  static_assert(STAGE % (THREADS * 16) == 0 && BM * 8 % THREADS == 0, "copies");
  extern __shared__ __attribute__((aligned(16))) uint8_t sm[];

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c = lane & 15, h = lane >> 4;
  const int wm = wave / WN, wn = wave % WN;
  const int tiles_m = (p.M + BM - 1) / BM, tiles_n = (p.N + BN - 1) / BN;
  // Neighbouring blocks of an XCD share rows of a and of b in its L2.
  int id = xcd_contiguous(blockIdx.x, tiles_m * tiles_n * p.parts);
  const int part = id / (tiles_m * tiles_n);
  id -= part * (tiles_m * tiles_n);
  constexpr int GROUP = 8;
  const int first = id / (GROUP * tiles_n) * GROUP;
  const int span = tiles_m - first < GROUP ? tiles_m - first : GROUP;
  const int m0 = (first + id % (GROUP * tiles_n) % span) * BM;
  const int n0 = id % (GROUP * tiles_n) / span * BN;
  const int kb0 = part * p.part_blocks;
  const int kb1 = kb0 + p.part_blocks < p.kblocks ? kb0 + p.part_blocks : p.kblocks;

  // Copies: thread t's piece j is chunk t % 8 of row (t + j THREADS) / 8 of the
  // stage, rows of a first, by descriptors that begin at the tile's rows.  Rows
  // past the matrix repeat its last one.
  const int chunk = (threadIdx.x & 7) ^ ((threadIdx.x >> 3) & 7);
  static_assert(THREADS / 8 % 8 == 0, "a thread's pieces have one place in their rows");
  const uint8_t *const a0 = p.a + (int64_t)m0 * p.lda;
  const uint8_t *const b0 = p.b + (int64_t)n0 * p.ldb;
  int from[COPIES];
#pragma unroll
  for (int j = 0; j < COPIES; ++j) {
    const int r = ((int)threadIdx.x + j * THREADS) / 8;
    if (j * THREADS / 8 < BM)
      from[j] = (m0 + r < p.M ? r : p.M - 1 - m0) * p.lda + 16 * chunk;
    else
      from[j] = (n0 + r - BM < p.N ? r - BM : p.N - 1 - n0) * p.ldb + 16 * chunk;
  }
  // Pieces j0 .. j1 - 1 of a step's copies.
  auto copy = [&](int kb, int stage, int j0, int j1) {
    const int k = kb * kBlock;
    // (in the last block: chunks past the row's end come from its last one and
    // are cleared below)
    const int left = p.K - k;
    const int back = 16 * (chunk + 1) > left ? 16 * (chunk + 1) - left : 0;
    uint8_t *const to = sm + stage * STAGE + wave * 1024;
#pragma unroll
    for (int j = j0; j < j1; ++j)
      copy16(j * THREADS / 8 < BM ? a0 : b0, to + j * THREADS * 16, from[j] - back, k);
  };

  // Scales, one for each row and one for 128 columns, come four steps at a time, 16
  // bytes a row, 64 rows a wave: waves 0 .. BM / 64 - 1 those of the rows, the next
  // the columns'.  A CU has some 64 requests to
  // L2 on their way, each a line at most, and a scale by itself is one: a step's
  // 256 + 256 rows are 512, their scales one by one were 260 more (256 x 256 tiles,
  // 8192x8192x8192 530 us; every wave fetching its own 16 rows' 1170).
  constexpr int WAVES = WM * WN, NB = (BN + 2 * kBlock - 2) / kBlock; // columns' blocks
  constexpr int SET = (BM / 64 + 1) * 256; // floats of four steps' scales
  // (of the waves that fetch some, so that a CU holds three blocks of 64 x 128: 520 of
  // them, 4099 x 777 x 1001 in f32, 24.4 us, with two 27.4)
  static_assert(BM % 64 == 0 && WAVES > BM / 64 && NB <= 64, "a wave for the columns' scales");
  float *const scales = (float *)(sm + STAGES * STAGE); // [2][BM / 64 + 1][64][4]
  const float *scale0 = p.a_scale + (int64_t)m0 * p.kblocks;
  int scale_at;
  unsigned scale_bytes; // from scale0 on
  {
    const int m = wave * 64 + lane, last = (p.N - 1) / kBlock;
    const int n = n0 / kBlock + (lane < NB ? lane : 0);
    int64_t rows_left = (int64_t)p.M - m0;
    if (wave < BM / 64) {
      scale_at = (m0 + m < p.M ? m : p.M - 1 - m0) * p.kblocks * 4;
    } else {
      scale0 = p.b_scale + (int64_t)(n0 / kBlock) * p.kblocks;
      scale_at = ((n < last ? n : last) - n0 / kBlock) * p.kblocks * 4;
      rows_left = last + 1 - n0 / kBlock;
    }
    const int64_t bytes = rows_left * p.kblocks * 4;
    scale_bytes = bytes < 0x7FFFFFFF ? (unsigned)bytes : 0x7FFFFFFFu;
  }
  scale_bytes = __builtin_amdgcn_readfirstlane(scale_bytes);
  // Of blocks kb .. kb + 3; those behind a row's last are the next row's, and behind
  // the last row's nothing is read.
  auto scales_of = [&](int kb, int set) {
    if (wave <= BM / 64)
      copy16(scale0, scales + set * SET + wave * 256, scale_at + kb * 4, 0, scale_bytes);
  };

  float total[TM][TN][4];
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j)
#pragma unroll
      for (int r = 0; r < 4; ++r)
        total[i][j][r] = 0.0f;

  // A step's memory operations of a wave: the scales of four, in every fourth step,
  // then COPIES copies.  All but the COPIES (STAGES - 2) last having landed, the
  // step's rows have, and its scales, which are fetched four steps before.
  const int steps = kb1 - kb0;
  auto step_at = [&](int i) { return kb0 + (i < steps ? i : steps - 1); };
  if (steps > 0) { // (no elements in a row: the sums are 0)
    scales_of(kb0, 0);
#pragma unroll
    for (int i = 0; i < STAGES - 1; ++i)
      copy(step_at(i), i, 0, COPIES);
  }
  int stage = 0;
  for (int step = 0; step < steps; ++step) {
    // this step's rows are in LDS; those of the step before have been read by all,
    // and the last of the steps ahead goes where they were
    // (not __syncthreads, which waits for every copy on its way)
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"((STAGES - 2) * COPIES)
                 : "memory");
    const int kb = kb0 + step;
    uint8_t *const st = sm + stage * STAGE;
    const float *const sc = scales + (step >> 2 & 1) * SET + (step & 3);
    if (kb * kBlock + kBlock > p.K) { // chunks past the row's end
      const int left = (p.K - kb * kBlock) / 16;
      for (int i = threadIdx.x; i < (BM + BN) * 8; i += THREADS)
        if (((i & 7) ^ ((i >> 3) & 7)) >= left)
          *(v4u *)(st + i * 16) = v4u{0, 0, 0, 0};
      __syncthreads();
    }
    // The copies are dealt out over the wave's rows: a wave is held at each until
    // the path to memory has taken the one before.
    const int ahead = step_at(step + STAGES - 1);
    const int to_stage = stage == 0 ? STAGES - 1 : stage - 1;
    auto copies_of = [&](int i) {
      if (i == 0 && (step & 3) == 0)
        scales_of(kb + 4, (step >> 2 & 1) ^ 1);
      copy(ahead, to_stage, COPIES * i / TM, COPIES * (i + 1) / TM);
      __builtin_amdgcn_sched_barrier(0x38F); // (only memory operations stay in place)
    };
    stage = stage + 1 < STAGES ? stage + 1 : 0;
    float sa_now[TM], sb_now[TN];
#pragma unroll
    for (int i = 0; i < TM; ++i)
      sa_now[i] = sc[((wm * TM + i) * 16 + c) * 4];
#pragma unroll
    for (int j = 0; j < TN; ++j)
      sb_now[j] = sc[(BM + (n0 % kBlock + (wn * TN + j) * 16) / kBlock) * 4];
    // lane (c, h): chunks h and h + 4 of row c of each 16
    auto read = [&](int row, int half) -> v4u {
      const int r = row + c;
      return *(const v4u *)(st + r * kBlock + (((h + 4 * half) ^ (r & 7)) << 4));
    };
    // The wave's columns stay in registers, its rows pass through them.
    auto columns = [&](int j, int half) { return read(BM + (wn * TN + j) * 16, half); };
    auto rows = [&](int i, int half) { return read((wm * TM + i) * 16, half); };
    if constexpr (EXACT) {
      v8bf wb[TN][4];
#pragma unroll
      for (int j = 0; j < TN; ++j)
        widen16(columns(j, 0), columns(j, 1), wb[j]);
#pragma unroll
      for (int i = 0; i < TM; ++i) {
        copies_of(i);
        v8bf wa[4];
        widen16(rows(i, 0), rows(i, 1), wa);
#pragma unroll
        for (int j = 0; j < TN; ++j) {
          v4f acc = {0, 0, 0, 0};
#pragma unroll
          for (int e = 0; e < 4; ++e)
            acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wb[j][e], wa[e], acc, 0, 0, 0);
          add_scaled(total[i][j], acc, sa_now[i] * sb_now[j]);
        }
      }
    } else {
      v8i fb[TN];
#pragma unroll
      for (int j = 0; j < TN; ++j)
        fb[j] = operand(columns(j, 0), columns(j, 1));
      v8i next = operand(rows(0, 0), rows(0, 1));
#pragma unroll
      for (int i = 0; i < TM; ++i) {
        copies_of(i);
        const v8i fa = next;
        if (i + 1 < TM)
          next = operand(rows(i + 1, 0), rows(i + 1, 1));
        v4f acc[TN];
#pragma unroll
        for (int j = 0; j < TN; ++j)
          acc[j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(
              fb[j], fa, v4f{0, 0, 0, 0}, 0, 0, 0, 0, 0, 0);
#pragma unroll
        for (int j = 0; j < TN; ++j)
          add_scaled(total[i][j], acc[j], sa_now[i] * sb_now[j]);
      }
    }
  }
  // (the last steps have copied the last one once more)
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  if (p.parts > 1) {
#pragma unroll
    for (int i = 0; i < TM; ++i) {
      const int m = m0 + (wm * TM + i) * 16 + c;
#pragma unroll
      for (int j = 0; j < TN; ++j) {
        const int n = n0 + (wn * TN + j) * 16 + 4 * h;
        const float *const t = total[i][j];
        if (m < p.M && n < p.N)
          *(v4f *)(p.part_sums + ((int64_t)part * p.M + m) * p.part_pitch + n) =
              v4f{t[0], t[1], t[2], t[3]};
      }
    }
    return;
  }
  // Results leave by way of LDS, so that a store takes whole lines of rows: each
  // wave's 16 TM x 16 TN, 16-byte chunk q of row r at place q ^ (r % 8).
  constexpr int ROW = TN * 16 * (int)sizeof(T), CHUNKS = ROW / 16;
  static_assert(WM * WN * TM * 16 * ROW <= STAGES * STAGE && CHUNKS <= 64, "LDS");
  __syncthreads();
  uint8_t *const mine = sm + wave * (TM * 16 * ROW);
  auto place = [&](int row, int chunk) {
    return row * ROW + ((CHUNKS % 8 == 0 ? chunk ^ (row & 7) : chunk) << 4);
  };
  float bias[TN][4];
#pragma unroll
  for (int j = 0; j < TN; ++j)
#pragma unroll
    for (int r = 0; r < 4; ++r)
      bias[j][r] = 0.0f;
  if (p.bias) {
#pragma unroll
    for (int j = 0; j < TN; ++j)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int n = n0 + (wn * TN + j) * 16 + 4 * h + r;
        bias[j][r] = p.bias[(n < p.N ? n : p.N - 1) * p.bias_step];
      }
  }
#pragma unroll
  for (int j = 0; j < TN; ++j) {
#pragma unroll
    for (int i = 0; i < TM; ++i) {
      Pack<T, 4> out;
#pragma unroll
      for (int r = 0; r < 4; ++r)
        total[i][j][r] += bias[j][r];
      if (p.activation)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          total[i][j][r] = p.activation == OM_MI355X_ACTIVATION_RELU
                               ? __builtin_fmaxf(total[i][j][r], 0.0f)
                               : gemm::gelu_f32(total[i][j][r]);
#pragma unroll
      for (int r = 0; r < 4; ++r)
        out.v[r] = from_f32<T>(total[i][j][r]);
      const int at = (j * 16 + 4 * h) * (int)sizeof(T);
      *(Pack<T, 4> *)(mine + place(i * 16 + c, at / 16) + at % 16) = out;
    }
  }
  // (a wave reads what it wrote itself)
  const int per_store = 64 / CHUNKS; // rows
  // (rows may start at any element: stores of 16 bytes need no more than theirs)
  typedef typename Loose<T>::v4 v4u_any;
#pragma unroll 4
  for (int r0 = 0; r0 < TM * 16; r0 += per_store) {
    const int row = r0 + lane / CHUNKS, q = lane % CHUNKS;
    const int m = m0 + wm * (TM * 16) + row;
    const int n = n0 + wn * (TN * 16) + q * (16 / (int)sizeof(T));
    if (lane >= per_store * CHUNKS || row >= TM * 16 || m >= p.M || n >= p.N)
      continue;
    const v4u w = *(const v4u *)(mine + place(row, q));
    T *const y = (T *)p.y + (int64_t)m * p.N + n;
    if (n + 16 / (int)sizeof(T) <= p.N) {
      *(v4u_any *)y = w;
    } else {
      const Pack<T, 16 / sizeof(T)> e = __builtin_bit_cast(Pack<T, 16 / sizeof(T)>, w);
#pragma unroll
      for (int i = 0; i < 16 / (int)sizeof(T); ++i)
        if (n + i < p.N)
          y[i] = e.v[i];
    }
  }
}

// The parts' sums added in their order, four columns a thread.
template <typename T>
__global__ __launch_bounds__(256) void k_join_parts(const GemmParams p) {
  const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const unsigned quads = (unsigned)p.part_pitch / 4;
  const int64_t m = id / quads;
  const int n = (int)(id - m * quads) * 4;
  if (m >= p.M)
    return;
  v4f t = {0, 0, 0, 0};
#pragma unroll 4
  for (int i = 0; i < p.parts; ++i)
    t += *(const v4f *)(p.part_sums + ((int64_t)i * p.M + m) * p.part_pitch + n);
  const float v[4] = {t[0], t[1], t[2], t[3]};
  store4<T>(p, (int)m, n, v);
}

// Rows of up to two matrices copied to a pitch of whole 16-byte chunks, zeros
// behind them, a wave a row.
struct AlignRows {
  const uint8_t *from[2];
  uint8_t *to[2];
  int64_t rows[2];
  int64_t first; // of a launch
  int K, pitch;
};
__global__ __launch_bounds__(256) void k_align_rows(const AlignRows p) {
  int64_t row = p.first + (int64_t)blockIdx.x * 4 + threadIdx.x / 64;
  const int which = row >= p.rows[0];
  row -= which ? p.rows[0] : 0;
  if (row >= p.rows[which])
    return;
  const uint8_t *const x = p.from[which] + row * p.K;
  uint8_t *const y = p.to[which] + row * p.pitch;
#pragma unroll 2
  for (int k = threadIdx.x % 64 * 16; k < p.pitch; k += 64 * 16) {
    v4u w = {0, 0, 0, 0};
    if (k + 16 <= p.K) {
      typedef unsigned v4u_any __attribute__((ext_vector_type(4), aligned(1)));
      w = *(const v4u_any *)(x + k);
    } else {
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if (k + i < p.K)
          w[i / 4] |= (unsigned)x[k + i] << (8 * (i % 4));
    }
    *(v4u *)(y + k) = w;
  }
}

// Rows that the kernel for few of them takes: 16, and 32 of small products, where a
// tile's steps cost more than fetching a's rows in every block (32 rows, skinny /
// tiles: 768x768 4.5 / 5.5, 2048x2048 7.5 / 7.5, 4096x1024 9.2 / 8.3, 4096x11008
// 26 / 13.5 us).
bool few_rows(int64_t M, int64_t K, int64_t N) {
  return M <= 16 || (M <= 32 && K * N < (int64_t)1 << 21);
}

bool rows_aligned(const void *p, int64_t K) {
  return K % 16 == 0 && ((uintptr_t)p & 15) == 0;
}

template <typename T, int MT, int WAVES, int DEPTH, bool TAIL>
hipError_t skinny_in(hipStream_t st, const GemmParams &p) {
  const int rows = p.M < 16 * MT ? p.M : 16 * MT; // of a block
  const dim3 grid((unsigned)((p.N + 15) / 16), (unsigned)((p.M + rows - 1) / rows)), block(WAVES * 64);
  // (32 KB of scales: 16 rows of 61000 elements)
  const int64_t floats = (int64_t)(rows + 1) * p.kblocks;
  if (floats <= 8192)
    k_block_skinny<T, MT, WAVES, DEPTH, TAIL, true><<<grid, block, (size_t)floats * 4, st>>>(p);
  else
    k_block_skinny<T, MT, WAVES, DEPTH, TAIL, false><<<grid, block, 0, st>>>(p);
  return hipGetLastError();
}

template <typename T, int MT>
hipError_t skinny(hipStream_t st, const GemmParams &p) {
  note_gemm_kernel("k_block_skinny");
  if (p.K % kBlock != 0 || !rows_aligned(p.a, p.lda) || !rows_aligned(p.b, p.ldb))
    return skinny_in<T, MT, 8, 2, true>(st, p);
  return skinny_in<T, MT, (MT > 1 ? 4 : 8), 4, false>(st, p);
}

// Tiles that a product can be dealt in.
enum TileForm { k256x256, k256x128, k128x128, k64x128, kTileForms };
constexpr int kUnaligned = kTileForms; // no tiles: rows that they cannot copy

// Which tile, and in how many parts of K: what takes the least time by
//   base + steps (full rounds * full + the rest of the fullest CU * lone) + rounds * round
//   [+ 3.7 + 1.43 us per million sums of all parts, to write, read and add them]
// microseconds, where a CU holds per_cu tiles at once and takes its share of them
// one round after the other.  Fitted to 84 products of 80 .. 4096 rows timed in every
// form (872 times), when a CU held two tiles of 64 x 128; it holds three now.  Of the
// same products on the kernels as they are, its times are off by 8 - 11 % (root mean
// square), and the forms that it takes are 2.1 % slower than the fastest in the
// geometric mean, 17 % at most (128 rows, where 64 x 128 in more parts is faster).
struct TileCost {
  int bm, bn, per_cu;
  float base, full, lone, round;
};
constexpr TileCost kTileCosts16[kTileForms] = {
    {256, 256, 1, 3.2f, 0.0f, 1.54f, 1.83f},
    {256, 128, 1, 4.7f, 0.0f, 0.91f, 0.0f},
    {128, 128, 2, 3.7f, 1.08f, 0.74f, 0.0f},
    {64, 128, 2, 2.7f, 0.77f, 0.59f, 0.0f},
};
constexpr TileCost kTileCosts32[kTileForms] = { // (the first two are not there)
    {0, 0, 0, 0, 0, 0, 0},
    {0, 0, 0, 0, 0, 0, 0},
    {128, 128, 2, 5.1f, 1.76f, 1.04f, 0.0f},
    {64, 128, 2, 3.4f, 1.12f, 0.76f, 0.0f},
};
struct TilePlan {
  int form, parts;
};
constexpr int kMostParts = 16;
constexpr int64_t kMostSums = (int64_t)64 << 20; // of all parts
TilePlan plan_tiles(const BlockGemm &g, int most_parts = kMostParts) {
  const int64_t kblocks = (g.K + kBlock - 1) / kBlock;
  TilePlan best = {k128x128, 1};
  float least = 0.0f;
  for (int form = 0; form < kTileForms; ++form) {
    const TileCost &c = g.kind == kF32 ? kTileCosts32[form] : kTileCosts16[form];
    if (!c.bm)
      continue;
    const int64_t tiles = ((g.M + c.bm - 1) / c.bm) * ((g.N + c.bn - 1) / c.bn);
    for (int parts = 1; parts <= most_parts; parts *= 2) {
      if (parts > 1 && (parts > kblocks || g.M * g.N > kMostSums / parts))
        break;
      const int64_t steps = (kblocks + parts - 1) / parts;
      const int64_t n = (tiles * parts + 255) / 256; // on the fullest CU
      const int64_t full = n / c.per_cu, rest = n % c.per_cu;
      // (one tile at a time: every round is a lone one)
      float us = c.base + c.round * (float)(full + (rest > 0));
      us += (float)steps * (c.per_cu > 1 ? full * c.full + rest * c.lone : full * c.lone);
      if (parts > 1)
        us += 3.7f + 1.43e-6f * (float)(parts * g.M * g.N);
      if (least == 0.0f || us < least) {
        least = us;
        best = {form, parts};
      }
    }
  }
  return best;
}

const char *tile_name(int bm, int bn, bool parts) {
  if (bm == 256)
    return bn == 256 ? (parts ? "k_block_tile (256x256, K in parts)" : "k_block_tile (256x256)")
                     : (parts ? "k_block_tile (256x128, K in parts)" : "k_block_tile (256x128)");
  return bm == 128 ? (parts ? "k_block_tile (128x128, K in parts)" : "k_block_tile (128x128)")
                   : (parts ? "k_block_tile (64x128, K in parts)" : "k_block_tile (64x128)");
}

template <typename T, int BM, int BN, int WM, int WN, int STAGES>
hipError_t tile(hipStream_t st, const GemmParams &p) {
  constexpr bool kExact = sizeof(T) == 4;
  constexpr int kLds = STAGES * (BM + BN) * kBlock + 2 * (BM / 64 + 1) * 1024;
  static_assert(kLds <= 160 * 1024, "LDS");
  auto *const kernel = k_block_tile<T, BM, BN, WM, WN, STAGES, kExact>;
  if (kLds > 65536) {
    const hipError_t e = hipFuncSetAttribute((const void *)kernel,
        hipFuncAttributeMaxDynamicSharedMemorySize, kLds);
    if (e != hipSuccess)
      return e;
  }
  note_gemm_kernel(tile_name(BM, BN, p.parts > 1));
  const unsigned tiles = (unsigned)((p.M + BM - 1) / BM) * (unsigned)((p.N + BN - 1) / BN);
  kernel<<<dim3(tiles * p.parts), WM * WN * 64, kLds, st>>>(p);
  hipError_t e = hipGetLastError();
  if (e == hipSuccess && p.parts > 1) {
    const int64_t n = (int64_t)p.M * (p.part_pitch / 4);
    k_join_parts<T><<<dim3((unsigned)((n + 255) / 256)), 256, 0, st>>>(p);
    e = hipGetLastError();
  }
  return e;
}

// Rows where they lie, any number of them, in launches of as many as a grid has.
template <typename T> hipError_t unaligned(hipStream_t st, GemmParams p) {
  note_gemm_kernel("k_block_skinny (many rows)");
  constexpr int kRows = 32 * 65535;
  for (int left = p.M; left > 0; left -= kRows) {
    p.M = left < kRows ? left : kRows;
    const hipError_t e = skinny_in<T, 2, 8, 2, true>(st, p);
    if (e != hipSuccess)
      return e;
    p.a += (int64_t)kRows * p.lda;
    p.a_scale += (int64_t)kRows * p.kblocks;
    p.y = (T *)p.y + (int64_t)kRows * p.N;
  }
  return hipSuccess;
}

template <typename T>
hipError_t product(hipStream_t st, const GemmParams &p, int form) {
  if (few_rows(p.M, p.K, p.N))
    return p.M <= 16 ? skinny<T, 1>(st, p) : skinny<T, 2>(st, p);
  if (form == kUnaligned)
    return unaligned<T>(st, p);
  // (f32 results of larger tiles do not fit in LDS)
  if constexpr (sizeof(T) == 2) {
    switch (form) {
    case k256x256:
      return tile<T, 256, 256, 2, 4, 2>(st, p);
    case k256x128:
      return tile<T, 256, 128, 4, 2, 3>(st, p);
    }
  }
  return form == k64x128 ? tile<T, 64, 128, 1, 4, 2>(st, p) : tile<T, 128, 128, 2, 2, 2>(st, p);
}

} // namespace
} // namespace llm

using namespace llm;

hipError_t launch_quantize_blocks(hipStream_t s, const void *x, FloatKind kind,
    int64_t M, int64_t K, int rows, uint8_t *y, float *scale) {
  switch (kind) {
  case kF32:
    return quantize(s, (const float *)x, M, K, rows, y, scale);
  case kF16:
    return quantize(s, (const _Float16 *)x, M, K, rows, y, scale);
  default:
    return quantize(s, (const __bf16 *)x, M, K, rows, y, scale);
  }
}

// The tile kernel copies 16-byte chunks of rows that start on such: others are
// copied first, or, without room for that, multiplied where they lie.
static size_t aligned_bytes(const void *p, int64_t rows, int64_t K) {
  return rows_aligned(p, K) ? 0 : (size_t)rows * (size_t)((K + 15) / 16 * 16);
}
static int64_t part_pitch(const BlockGemm &g) { return (g.N + 3) / 4 * 4; }
static size_t parts_bytes(const BlockGemm &g, const TilePlan &plan) {
  return plan.parts > 1 ? (size_t)plan.parts * g.M * part_pitch(g) * sizeof(float) : 0;
}
size_t block_gemm_row_bytes(const BlockGemm &g) {
  if (few_rows(g.M, g.K, g.N))
    return 0;
  return aligned_bytes(g.a, g.M, g.K) + aligned_bytes(g.b, g.N, g.K);
}
size_t block_gemm_part_bytes(const BlockGemm &g) {
  if (few_rows(g.M, g.K, g.N) || (!g.rows && block_gemm_row_bytes(g)))
    return 0;
  return parts_bytes(g, plan_tiles(g));
}

hipError_t launch_block_gemm(hipStream_t s, const BlockGemm &g) {
  GemmParams p = {};
  p.a = g.a;
  p.b = g.b;
  p.a_scale = g.a_scale;
  p.b_scale = g.b_scale;
  p.bias = g.bias;
  p.y = g.y;
  p.M = (int)g.M;
  p.N = (int)g.N;
  p.K = p.lda = p.ldb = (int)g.K;
  p.kblocks = (int)((g.K + kBlock - 1) / kBlock);
  p.bias_step = g.bias_len > 1;
  p.activation = g.activation;
  p.parts = 1;
  p.part_blocks = p.kblocks;
  TilePlan plan = {};
  if (!g.rows && block_gemm_row_bytes(g)) {
    plan.form = kUnaligned;
  } else if (!few_rows(g.M, g.K, g.N)) {
    plan = plan_tiles(g, g.parts ? kMostParts : 1);
    p.parts = plan.parts;
    p.part_blocks = (p.kblocks + plan.parts - 1) / plan.parts;
    p.part_pitch = (int)part_pitch(g);
    p.part_sums = g.parts;
    uint8_t *at = g.rows;
    const int pitch = (int)((g.K + 15) / 16 * 16);
    AlignRows copies = {};
    int n = 0;
    auto align = [&](const uint8_t *&rows_of, int64_t rows, int &ld) {
      if (rows_aligned(rows_of, g.K))
        return;
      copies.from[n] = rows_of;
      copies.to[n] = at;
      copies.rows[n++] = rows;
      rows_of = at;
      ld = pitch;
      at += (size_t)rows * pitch;
    };
    align(p.a, g.M, p.lda);
    align(p.b, g.N, p.ldb);
    if (n) {
      copies.K = (int)g.K;
      copies.pitch = pitch;
      int64_t blocks = (copies.rows[0] + copies.rows[1] + 3) / 4;
      for (copies.first = 0; blocks > 0; blocks -= kMostGrid, copies.first += 4 * kMostGrid) {
        k_align_rows<<<dim3((unsigned)(blocks < kMostGrid ? blocks : kMostGrid)), 256, 0, s>>>(copies);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess)
          return e;
      }
    }
    if (p.lda == pitch && p.ldb == pitch)
      p.K = pitch; // (zeros behind the last element of both)
  }
  switch (g.kind) {
  case kF32:
    return product<float>(s, p, plan.form);
  case kF16:
    return product<_Float16>(s, p, plan.form);
  default:
    return product<__bf16>(s, p, plan.form);
  }
}

} // namespace om
