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
// eleven where r = RN(1 / s): q0 = RN(x r), e = x - q0 s (exact), q = RN(q0 +
// e r).  Nothing under- or overflows for scales from 2^-80 to 2^96 and
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

template <typename T>
hipError_t quantize(hipStream_t st, const T *x, int64_t M, int64_t K, int rows,
    uint8_t *y, float *scale) {
  const int per_row = (int)((K + kBlock - 1) / kBlock);
  const bool wide = K % 8 == 0 && ((uintptr_t)x & 15) == 0 && ((uintptr_t)y & 7) == 0;
  if (rows == 1) {
    const int64_t blocks = M * per_row;
    constexpr int U = 2;
    const dim3 grid((unsigned)((blocks + 16 * U - 1) / (16 * U)));
    if (wide)
      k_quantize_rows<T, true, U><<<grid, 256, 0, st>>>(x, y, scale, blocks, (int)K, per_row);
    else
      k_quantize_rows<T, false, U><<<grid, 256, 0, st>>>(x, y, scale, blocks, (int)K, per_row);
  } else {
    const dim3 grid((unsigned)((M + 127) / 128 * per_row));
    if (wide)
      k_quantize_tiles<T, true><<<grid, 256, 0, st>>>(x, y, scale, M, (int)K, per_row);
    else
      k_quantize_tiles<T, false><<<grid, 256, 0, st>>>(x, y, scale, M, (int)K, per_row);
  }
  return hipGetLastError();
}

// ---------------------------------------------------------------------------
// products
// ---------------------------------------------------------------------------
// The matrix instructions for 8-bit operands align the products of one
// instruction to the largest before they add them: against 64 bits their sums
// are off by 1.5e-5 relative to the result on normally distributed operands
// and up to 9e-5 where few channels are much larger than the others (measured,
// K = 4096).  That is far below the rounding of results in bf16 (1.7e-3) and
// below that of f16 (2.1e-4), and they run twice as fast as those for bf16, so
// results in 16 bits take them.  Results in f32 are summed by the bf16
// instructions (6e-8 to 1.4e-7 on the same operands), which hold every e4m3
// value exactly; so does everything that is bound by reading its weights.

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

struct GemmParams {
  const uint8_t *a, *b;
  const float *a_scale, *b_scale, *bias;
  void *y;
  int M, N, K;
  int lda, ldb;      // bytes from row to row
  int kblocks;       // scales of a row: ceil(K / 128) of the caller's K
  int bias_step;     // 0: one bias for all columns
  int activation;
};

__device__ __forceinline__ float finish(float v, const GemmParams &p, float bias) {
  v += bias;
  if (p.activation == OM_MI355X_ACTIVATION_RELU)
    v = __builtin_fmaxf(v, 0.0f);
  else if (p.activation == OM_MI355X_ACTIVATION_GELU)
    v = gemm::gelu_f32(v);
  return v;
}

// Four neighbouring columns n .. n + 3 of row m; those past N are left out.
template <typename T>
__device__ __forceinline__ void store4(
    const GemmParams &p, int m, int n, const float (&v)[4], bool whole) {
  T *const y = (T *)p.y + (int64_t)m * p.N + n;
  T t[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int c = n + i < p.N ? n + i : p.N - 1;
    const float bias = p.bias ? p.bias[c * p.bias_step] : 0.0f;
    t[i] = from_f32<T>(finish(v[i], p, bias));
  }
  if (whole && n + 4 <= p.N) {
    *(Pack<T, 4> *)y = *(const Pack<T, 4> *)t;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (n + i < p.N)
        y[i] = t[i];
  }
}

// --- few rows ---------------------------------------------------------------
// Up to 16 MT rows: a block owns 16 columns, its WAVES waves take every
// WAVES-th block of 128 of K.  Bound by reading the weights once: a wave has
// the weights of DEPTH blocks on their way, lanes (c, h) the bytes 16 h .. of
// each half of column c's 128, whole lines together.  Products by bf16
// instructions; sums of the waves meet in LDS in a fixed order.
template <typename T, int MT, int WAVES, int DEPTH, bool TAIL>
__global__ __launch_bounds__(WAVES * 64) void k_block_skinny(const GemmParams p) {
  __shared__ float sums[WAVES][MT][64][4];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c = lane & 15, h = lane >> 4;
  const int n0 = blockIdx.x * 16;
  const int col = n0 + c < p.N ? n0 + c : p.N - 1;
  const uint8_t *const b = p.b + (int64_t)col * p.ldb + 16 * h;
  const uint8_t *a[MT];
  const float *as[MT];
#pragma unroll
  for (int i = 0; i < MT; ++i) {
    const int row = 16 * i + c < p.M ? 16 * i + c : p.M - 1;
    a[i] = p.a + (int64_t)row * p.lda + 16 * h;
    as[i] = p.a_scale + (int64_t)row * p.kblocks;
  }
  const float *const bs = p.b_scale + (int64_t)(n0 / kBlock) * p.kblocks;

  float total[MT][4];
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int r = 0; r < 4; ++r)
      total[i][r] = 0.0f;

  v4u wb[DEPTH][2], wa[DEPTH][MT][2];
  float sa[DEPTH][MT], sb[DEPTH];
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
      for (int i = 0; i < MT; ++i)
        wa[d][i][half] = load16(a[i], k + 64 * half);
    }
    sb[d] = bs[kb];
#pragma unroll
    for (int i = 0; i < MT; ++i)
      sa[d][i] = as[i][kb];
  };
#pragma unroll
  for (int d = 0; d < DEPTH; ++d)
    if (wave + d * WAVES < p.kblocks)
      fetch(d, wave + d * WAVES);
  for (int kb = wave; kb < p.kblocks; kb += DEPTH * WAVES) {
#pragma unroll
    for (int d = 0; d < DEPTH; ++d) {
      const int at = kb + d * WAVES;
      if (at >= p.kblocks)
        break;
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
      for (int i = 0; i < MT; ++i) {
        const float s = sa[d][i] * sb[d];
#pragma unroll
        for (int r = 0; r < 4; ++r)
          total[i][r] = __builtin_fmaf(acc[i][r], s, total[i][r]);
      }
      if (at + DEPTH * WAVES < p.kblocks)
        fetch(d, at + DEPTH * WAVES);
    }
  }
#pragma unroll
  for (int i = 0; i < MT; ++i)
    *(v4f *)sums[wave][i][lane] = v4f{total[i][0], total[i][1], total[i][2], total[i][3]};
  __syncthreads();
  // lane (c, h) of wave i: row 16 i + c, columns n0 + 4 h ..
  for (int i = wave; i < MT; i += WAVES) {
    v4f t = {0, 0, 0, 0};
#pragma unroll
    for (int w = 0; w < WAVES; ++w)
      t += *(const v4f *)sums[w][i][lane];
    const float v[4] = {t[0], t[1], t[2], t[3]};
    if (16 * i + c < p.M)
      store4<T>(p, 16 * i + c, n0 + 4 * h, v, p.N % 4 == 0);
  }
}

// --- tiles ------------------------------------------------------------------
// BM x BN tiles, WM x WN waves.  A step is one block of 128 of K: the rows'
// 128 bytes go straight into LDS (two stages), 16-byte chunk q of row r at
// place q ^ (r % 8), so that neither the copies nor the operand reads meet a
// bank twice.  Columns are the first operand of the matrix instruction, so a
// lane holds one row of the result and four neighbouring columns: one scale
// for all it gets from an instruction, and whole pieces to store.
template <typename T, int BM, int BN, int WM, int WN, bool EXACT>
__global__ __launch_bounds__(WM * WN * 64) void k_block_tile(const GemmParams p) {
  constexpr int THREADS = WM * WN * 64, STAGE = (BM + BN) * kBlock;
  constexpr int TM = BM / WM / 16, TN = BN / WN / 16;
  constexpr int COPIES = STAGE / (THREADS * 16); // of 16 bytes a thread
  static_assert(BN % kBlock == 0 || kBlock % BN == 0, "one scale a tile's columns");
  static_assert(STAGE % (THREADS * 16) == 0, "copies");
  extern __shared__ __attribute__((aligned(16))) uint8_t sm[];

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c = lane & 15, h = lane >> 4;
  const int wm = wave / WN, wn = wave % WN;
  const int tiles_m = (p.M + BM - 1) / BM, tiles_n = (p.N + BN - 1) / BN;
  // Neighbouring blocks of an XCD share rows of a and of b in its L2.
  const int id = xcd_contiguous(blockIdx.x, tiles_m * tiles_n);
  constexpr int GROUP = 8;
  const int first = id / (GROUP * tiles_n) * GROUP;
  const int span = tiles_m - first < GROUP ? tiles_m - first : GROUP;
  const int m0 = (first + id % (GROUP * tiles_n) % span) * BM;
  const int n0 = id % (GROUP * tiles_n) / span * BN;

  // Copies: thread t's piece j is chunk t % 8 of row (t + j THREADS) / 8 of the
  // stage, rows of a first.  Rows past the matrix repeat its last one.
  typedef __attribute__((address_space(3))) void *lds_ptr;
  typedef const __attribute__((address_space(1))) void *glb_ptr;
  const uint8_t *from[COPIES];
#pragma unroll
  for (int j = 0; j < COPIES; ++j) {
    const int r = ((int)threadIdx.x + j * THREADS) / 8;
    const int q = (threadIdx.x & 7) ^ (r & 7);
    if (j * THREADS / 8 < BM) {
      const int m = m0 + r < p.M ? m0 + r : p.M - 1;
      from[j] = p.a + (int64_t)m * p.lda + 16 * q;
    } else {
      const int n = n0 + r - BM < p.N ? n0 + r - BM : p.N - 1;
      from[j] = p.b + (int64_t)n * p.ldb + 16 * q;
    }
  }
  static_assert(BM * 8 % THREADS == 0, "a copy is of one operand");
  auto copy = [&](int kb, int stage) {
    const int k = kb * kBlock;
#pragma unroll
    for (int j = 0; j < COPIES; ++j) {
      uint8_t *const to = sm + stage * STAGE + j * THREADS * 16 + wave * 1024;
      // (in the last block: chunks past the row's end come from its last one
      // and are cleared below)
      const int over = k + kBlock > p.K ? k + kBlock - p.K : 0;
      const int q = ((threadIdx.x & 7) ^ ((((int)threadIdx.x + j * THREADS) / 8) & 7));
      const int back = over && 16 * (q + 1) > kBlock - over ? 16 * (q + 1) - (kBlock - over) : 0;
      __builtin_amdgcn_global_load_lds((glb_ptr)(from[j] + k - back), (lds_ptr)to, 16, 0, 0);
    }
  };

  // Scales: one a row of the result and step, and one for all columns.
  const float *as[TM];
#pragma unroll
  for (int i = 0; i < TM; ++i) {
    const int m = m0 + (wm * TM + i) * 16 + c;
    as[i] = p.a_scale + (int64_t)(m < p.M ? m : p.M - 1) * p.kblocks;
  }
  constexpr int NB = BN / WN > kBlock ? BN / WN / kBlock : 1; // scales of a wave's columns
  const float *bs[NB];
#pragma unroll
  for (int j = 0; j < NB; ++j) {
    const int n = n0 + wn * (BN / WN) + j * kBlock;
    bs[j] = p.b_scale + (int64_t)((n < p.N ? n : p.N - 1) / kBlock) * p.kblocks;
  }

  float total[TM][TN][4];
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j)
#pragma unroll
      for (int r = 0; r < 4; ++r)
        total[i][j][r] = 0.0f;

  float sa[TM], sb[NB];
  if (p.kblocks > 0) { // (no elements in a row: the sums are 0)
    copy(0, 0);
#pragma unroll
    for (int i = 0; i < TM; ++i)
      sa[i] = as[i][0];
#pragma unroll
    for (int j = 0; j < NB; ++j)
      sb[j] = bs[j][0];
  }
  for (int kb = 0; kb < p.kblocks; ++kb) {
    // this step's rows are in LDS, the last step's have been read by all
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    uint8_t *const st = sm + (kb & 1) * STAGE;
    float s[TM][NB];
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
      for (int j = 0; j < NB; ++j)
        s[i][j] = sa[i] * sb[j];
    if (kb * kBlock + kBlock > p.K) { // chunks past the row's end
      const int left = (p.K - kb * kBlock) / 16;
      for (int i = threadIdx.x; i < (BM + BN) * 8; i += THREADS)
        if (((i & 7) ^ ((i >> 3) & 7)) >= left)
          *(v4u *)(st + i * 16) = v4u{0, 0, 0, 0};
      __syncthreads();
    }
    if (kb + 1 < p.kblocks) {
      copy(kb + 1, (kb + 1) & 1);
#pragma unroll
      for (int i = 0; i < TM; ++i)
        sa[i] = as[i][kb + 1];
#pragma unroll
      for (int j = 0; j < NB; ++j)
        sb[j] = bs[j][kb + 1];
    }
    // lane (c, h): chunks h and h + 4 of row c of each 16
    auto read = [&](int row, int half) -> v4u {
      const int r = row + c;
      return *(const v4u *)(st + r * kBlock + (((h + 4 * half) ^ (r & 7)) << 4));
    };
    v4u fa[TM][2];
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
      for (int half = 0; half < 2; ++half)
        fa[i][half] = read((wm * TM + i) * 16, half);
    if (EXACT) {
#pragma unroll
      for (int j = 0; j < TN; ++j) {
        v4f acc[TM];
#pragma unroll
        for (int i = 0; i < TM; ++i)
          acc[i] = v4f{0, 0, 0, 0};
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const v4u w = read(BM + (wn * TN + j) * 16, half);
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const v8bf fb = widen8(w[2 * e], w[2 * e + 1]);
#pragma unroll
            for (int i = 0; i < TM; ++i)
              acc[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fb,
                  widen8(fa[i][half][2 * e], fa[i][half][2 * e + 1]), acc[i], 0, 0, 0);
          }
        }
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            total[i][j][r] = __builtin_fmaf(
                acc[i][r], s[i][NB > 1 ? j * 16 / kBlock : 0], total[i][j][r]);
      }
    } else {
#pragma unroll
      for (int j = 0; j < TN; ++j) {
        const v4u lo = read(BM + (wn * TN + j) * 16, 0);
        const v4u hi = read(BM + (wn * TN + j) * 16, 1);
        const v8i fb = {(int)lo[0], (int)lo[1], (int)lo[2], (int)lo[3], (int)hi[0],
            (int)hi[1], (int)hi[2], (int)hi[3]};
        v4f acc[TM];
#pragma unroll
        for (int i = 0; i < TM; ++i) {
          const v8i f = {(int)fa[i][0][0], (int)fa[i][0][1], (int)fa[i][0][2],
              (int)fa[i][0][3], (int)fa[i][1][0], (int)fa[i][1][1],
              (int)fa[i][1][2], (int)fa[i][1][3]};
          acc[i] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(
              fb, f, v4f{0, 0, 0, 0}, 0, 0, 0, 0, 0, 0);
        }
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            total[i][j][r] = __builtin_fmaf(
                acc[i][r], s[i][NB > 1 ? j * 16 / kBlock : 0], total[i][j][r]);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < TM; ++i) {
    const int m = m0 + (wm * TM + i) * 16 + c;
    if (m < p.M)
#pragma unroll
      for (int j = 0; j < TN; ++j) {
        const int n = n0 + (wn * TN + j) * 16 + 4 * h;
        if (n < p.N)
          store4<T>(p, m, n, total[i][j], p.N % 4 == 0);
      }
  }
}

// Rows copied to a pitch of whole 16-byte chunks, zeros behind them.
__global__ __launch_bounds__(256) void k_align_rows(
    const uint8_t *from, uint8_t *to, int64_t rows, int K, int pitch) {
  const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int chunks = pitch / 16;
  const int64_t row = id / chunks;
  const int k = (int)(id - row * chunks) * 16;
  if (row >= rows)
    return;
  const uint8_t *const x = from + row * K + k;
  v4u w = {0, 0, 0, 0};
  if (k + 16 <= K) {
    typedef unsigned v4u_any __attribute__((ext_vector_type(4), aligned(1)));
    w = *(const v4u_any *)x;
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i)
      if (k + i < K)
        w[i / 4] |= (unsigned)x[i] << (8 * (i % 4));
  }
  *(v4u *)(to + row * pitch + k) = w;
}

constexpr int kSkinnyRows = 64;

bool rows_aligned(const void *p, int64_t K) {
  return K % 16 == 0 && ((uintptr_t)p & 15) == 0;
}

template <typename T, int MT>
hipError_t skinny(hipStream_t st, const GemmParams &p) {
  const dim3 grid((unsigned)((p.N + 15) / 16));
  const bool tail = p.K % kBlock != 0 || !rows_aligned(p.a, p.lda) || !rows_aligned(p.b, p.ldb);
  constexpr int D = MT > 2 ? 2 : 4;
  if (tail)
    k_block_skinny<T, MT, 4, 2, true><<<grid, 256, 0, st>>>(p);
  else if (grid.x <= 512 && p.kblocks >= 16)
    k_block_skinny<T, MT, 8, D, false><<<grid, 512, 0, st>>>(p);
  else
    k_block_skinny<T, MT, 4, D, false><<<grid, 256, 0, st>>>(p);
  return hipGetLastError();
}

template <typename T, int BM, int BN, int WM, int WN>
hipError_t tile(hipStream_t st, const GemmParams &p) {
  constexpr bool kExact = sizeof(T) == 4;
  constexpr int kLds = 2 * (BM + BN) * kBlock;
  auto *const kernel = k_block_tile<T, BM, BN, WM, WN, kExact>;
  if (kLds > 65536) {
    const hipError_t e = hipFuncSetAttribute((const void *)kernel,
        hipFuncAttributeMaxDynamicSharedMemorySize, kLds);
    if (e != hipSuccess)
      return e;
  }
  const unsigned tiles = (unsigned)((p.M + BM - 1) / BM) * (unsigned)((p.N + BN - 1) / BN);
  kernel<<<dim3(tiles), WM * WN * 64, kLds, st>>>(p);
  return hipGetLastError();
}

template <typename T>
hipError_t product(hipStream_t st, const GemmParams &p) {
  if (p.M <= 16)
    return skinny<T, 1>(st, p);
  if (p.M <= 32)
    return skinny<T, 2>(st, p);
  if (p.M <= kSkinnyRows)
    return skinny<T, 4>(st, p);
  return tile<T, 128, 128, 2, 2>(st, p);
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
// copied first.
static size_t aligned_bytes(const void *p, int64_t rows, int64_t K) {
  return rows_aligned(p, K) ? 0 : (size_t)rows * (size_t)((K + 15) / 16 * 16);
}
size_t block_gemm_scratch(const BlockGemm &g) {
  if (g.M <= kSkinnyRows)
    return 0;
  return aligned_bytes(g.a, g.M, g.K) + aligned_bytes(g.b, g.N, g.K);
}

hipError_t launch_block_gemm(hipStream_t s, const BlockGemm &g, void *scratch) {
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
  if (g.M > kSkinnyRows) {
    const int pitch = (int)((g.K + 15) / 16 * 16);
    uint8_t *at = (uint8_t *)scratch;
    auto align = [&](const uint8_t *&rows_of, int64_t rows, int &ld) {
      if (rows_aligned(rows_of, g.K))
        return hipSuccess;
      const int64_t n = rows * (pitch / 16);
      k_align_rows<<<dim3((unsigned)((n + 255) / 256)), 256, 0, s>>>(
          rows_of, at, rows, (int)g.K, pitch);
      rows_of = at;
      ld = pitch;
      at += (size_t)rows * pitch;
      return hipGetLastError();
    };
    hipError_t e = align(p.a, g.M, p.lda);
    if (e == hipSuccess)
      e = align(p.b, g.N, p.ldb);
    if (e != hipSuccess)
      return e;
    if (p.lda == pitch && p.ldb == pitch)
      p.K = pitch; // (zeros behind the last element of both)
  }
  switch (g.kind) {
  case kF32:
    return product<float>(s, p);
  case kF16:
    return product<_Float16>(s, p);
  default:
    return product<__bf16>(s, p);
  }
}

} // namespace om
