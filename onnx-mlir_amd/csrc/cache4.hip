// Keys and values in 4 bits: appending to the cache, and attention over it.
//
// A row of D elements (one token in one head) is held in groups of 32: codes
// 0 .. 15, and for each group a scale s and a lowest value m in f16,
//     x ~ s * code + m.
// With G = D / 32, byte n G + g of the row's 16 G holds elements 32 g + 2 n
// (low half) and 32 g + 2 n + 1 (high half).  In that order both products of
// attention read what a lane needs in one piece: a quarter of a key's row is
// 8 elements of every group, and G neighbouring bytes of a value's row are the
// elements (2 n, 2 n + 1) of every group.

#include "llm_common.h"

namespace om {
namespace llm {
namespace {

typedef _Float16 v2h __attribute__((ext_vector_type(2)));

// Where the 16 keys from key0 on lie: rows of one page (pages hold a multiple
// of 16 tokens, or the sequence has one).
struct Place {
  int64_t row; // of the page's slot, in rows of the cache
  int last;    // key row + min(i, last) stays within the page
  bool known;  // the page is one of the cache's
};
__device__ __forceinline__ Place place_of(const Cache4 &c, int64_t b, int h, int64_t key) {
  int64_t page = b, slot = key;
  bool known = key >= 0;
  if (c.table) {
    const int64_t at = key / c.page_size;
    known = known && at < c.table_pages;
    page = known ? c.table[b * c.table_pages + at] : -1;
    slot = key - at * c.page_size;
  }
  known = known && page >= 0 && page < c.pages && slot < c.page_size;
  if (!known)
    page = slot = 0;
  return {(page * c.H + h) * c.page_size + slot, (int)(c.page_size - 1 - slot), known};
}

// ---------------------------------------------------------------------------
// append
// ---------------------------------------------------------------------------
// 16 lanes quantize a row, lane n elements 2 n and 2 n + 1 of every group.
// Bound by the launch for the few rows of a decode step, by memory for a
// prompt's: each element is read once, each code written once.
template <typename T, int G>
__global__ __launch_bounds__(256) void k_cache_append(const Append4 p) {
  const int n = threadIdx.x & 15;
  int64_t id = ((int64_t)blockIdx.x * 256 + threadIdx.x) >> 4;
  const int64_t rows = p.B * p.S * p.c.H;
  if (id >= 2 * rows)
    return;
  const bool value = id >= rows;
  if (value)
    id -= rows;
  // rows in the order of k and v
  int64_t b, i;
  int h;
  if (p.heads_first) {
    const int64_t bh = id / p.S;
    i = id - bh * p.S;
    b = bh / p.c.H;
    h = (int)(bh - b * p.c.H);
  } else {
    const int64_t t = id / p.c.H;
    h = (int)(id - t * p.c.H);
    b = t / p.S;
    i = t - b * p.S;
  }
  if (p.c.counts && i >= p.c.counts[b])
    return;
  const Place at = place_of(p.c, b, h, (int64_t)p.c.past[b] + i);
  if (!at.known)
    return;
  const T *const x = (const T *)(value ? p.v : p.k) + id * (32 * G) + 2 * n;
  Pack<T, 2> in[G];
#pragma unroll
  for (int g = 0; g < G; ++g)
    in[g] = *(const Pack<T, 2> *)(x + 32 * g);
  uint8_t *const codes = (value ? p.c.v_codes : p.c.k_codes) + at.row * (16 * G) + n * G;
  unsigned *const pairs =
      (unsigned *)(value ? p.c.v_scales : p.c.k_scales) + at.row * G;
  Pack<uint8_t, G> out;
  unsigned mine = 0;
#pragma unroll
  for (int g = 0; g < G; ++g) {
    float e[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      e[j] = to_f32(in[g].v[j]);
      e[j] = e[j] > 65504.0f ? 65504.0f : e[j] < -65504.0f ? -65504.0f : e[j];
    }
    const float top = row_max(__builtin_fmaxf(e[0], e[1]));
    const float low = -row_max(__builtin_fmaxf(-e[0], -e[1]));
    const bool none = row_max(e[0] != e[0] || e[1] != e[1] ? 1.0f : 0.0f) > 0.0f;
    const _Float16 m = none ? (_Float16)__builtin_nanf("") : (_Float16)low;
    // (lowest may have been rounded up, past the largest)
    const _Float16 s = none ? m : (_Float16)__builtin_fmaxf((top - (float)m) * (1.0f / 15.0f), 0.0f);
    unsigned code = 0;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      float q = __builtin_rintf((e[j] - (float)m) / (float)s);
      q = __builtin_fminf(__builtin_fmaxf(q, 0.0f), 15.0f);
      code |= (float)s > 0.0f ? (unsigned)q << (4 * j) : 0u;
    }
    out.v[g] = (uint8_t)code;
    if (n == g)
      mine = __builtin_bit_cast(unsigned, v2h{s, m});
  }
  *(Pack<uint8_t, G> *)codes = out;
  if (n < G)
    pairs[n] = mine;
}

// ---------------------------------------------------------------------------
// attention
// ---------------------------------------------------------------------------
// With khat = s c + m, a query's score for key t is
//     sum_g s_tg (q_g . c_tg) + m_tg sum(q_g)
// and the output's element d of group g
//     sum_t (p_t s_tg) c_td + sum_t p_t m_tg,
// so the matrix instructions multiply codes, which bf16 holds exactly, by q and
// by p s, which are split into bf16 terms: as many as q's type has bits (1, 2, 3
// for bf16, f16, f32), and 2 (16-bit results) or 3 for p s.  Sums, scores and
// softmax statistics are f32.
//
// A wave takes 16 RT rows (queries of the heads that share one of keys) and 32
// keys at a time.  Keys are the first operand of the first product and elements
// of a value that of the second, so that lane (c, h) holds row c throughout:
// scores of keys 4 h .. of either 16, which are also its places of the second
// product's operand, and output elements 32 g + 8 h ...  Nothing is moved
// between lanes but the rows' maxima, and those only when one grows by more
// than 8 (powers of two) over what p is relative to.
struct Arguments {
  Cache4 c;
  const void *q;
  void *y;
  const int32_t *starts;
  const float *scale;
  float *parts;  // [units, splits, rows, D], then (max, sum) of each row
  int64_t window;
  int B, S, heads, per_head, groups; // query heads a head of keys; groups of rows
  int splits;
  bool causal, heads_first;
};

// Bytes a.g and b.g of words a and b, then those of g + 1.
__device__ __forceinline__ unsigned two_of(unsigned a, unsigned b, int byte) {
  const unsigned s = (unsigned)byte;
  return __builtin_amdgcn_perm(b, a, s | (4 + s) << 8 | (s + 1) << 16 | (5 + s) << 24);
}
__device__ __forceinline__ unsigned one_of(
    unsigned a, int ia, unsigned b, int ib) {
  return __builtin_amdgcn_perm(b, a, (unsigned)ia | (unsigned)(4 + ib) << 8);
}

// Byte at[i] + g of word string i, for i = 0 .. 3 and every g: codes[g].
template <int G, int STEP, int WORDS>
__device__ __forceinline__ void bytes_of(
    const unsigned (&w)[4][WORDS], unsigned (&codes)[G]) {
#pragma unroll
  for (int g = 0; g < G; g += G % 2 ? 1 : 2) {
    auto word = [&](int i) { return w[i][(i * STEP + g) / 4]; };
    auto byte = [&](int i) { return (i * STEP + g) % 4; };
    if (G % 2) {
      const unsigned x = one_of(word(0), byte(0), word(1), byte(1));
      const unsigned y = one_of(word(2), byte(2), word(3), byte(3));
      codes[g] = __builtin_amdgcn_perm(y, x, 0x05040100);
    } else {
      const unsigned s0 = byte(0), s1 = byte(1), s2 = byte(2), s3 = byte(3);
      const unsigned x = __builtin_amdgcn_perm(
          word(1), word(0), s0 | (4 + s1) << 8 | (s0 + 1) << 16 | (5 + s1) << 24);
      const unsigned y = __builtin_amdgcn_perm(
          word(3), word(2), s2 | (4 + s3) << 8 | (s2 + 1) << 16 | (5 + s3) << 24);
      codes[g] = __builtin_amdgcn_perm(y, x, 0x05040100);
      codes[g + 1] = __builtin_amdgcn_perm(y, x, 0x07060302);
    }
  }
}

// Four bytes of 0 .. 15 as bf16: such a byte taken for an e4m3 value is 2^-9 of
// its number, below and above its subnormals alike.
__device__ __forceinline__ void numbers(unsigned w, v2bf &a, v2bf &b) {
  a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 512.0f, false);
  b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 512.0f, true);
}
__device__ __forceinline__ v8bf join(v2bf a, v2bf b, v2bf c, v2bf d) {
  return v8bf{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// x as a sum of N bf16 values, each the nearest to what the ones before leave.
template <int N>
__device__ __forceinline__ void terms_of(const float (&x)[8], v8bf (&t)[N]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    float rest = x[i];
#pragma unroll
    for (int k = 0; k < N; ++k) {
      t[k][i] = (__bf16)rest;
      if (k + 1 < N)
        rest -= to_f32(t[k][i]);
    }
  }
}

// N bytes from an address aligned to `ALIGN`.
template <int N, int ALIGN>
__device__ __forceinline__ void load_bytes(
    const uint8_t *p, unsigned (&w)[(N + 3) / 4]) {
  struct alignas(ALIGN) Bytes {
    uint8_t b[N];
  };
  const Bytes v = *(const Bytes *)p;
#pragma unroll
  for (int i = 0; i < (N + 3) / 4; ++i) {
    w[i] = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (4 * i + j < N)
        w[i] |= (unsigned)v.b[4 * i + j] << (8 * j);
  }
}

constexpr int kWaves = 4;
constexpr float kLog2E = 0x1.715476p+0f;

template <typename T> struct Terms;
template <> struct Terms<float> { static constexpr int q = 3, p = 3; };
template <> struct Terms<_Float16> { static constexpr int q = 2, p = 2; };
template <> struct Terms<__bf16> { static constexpr int q = 1, p = 2; };

template <typename T, int G, int RT>
__global__ __launch_bounds__(kWaves * 64) void k_cache_attention(const Arguments p) {
  constexpr int D = 32 * G, TQ = Terms<T>::q, TP = Terms<T>::p;
  extern __shared__ __attribute__((aligned(16))) float shared[];
  const int lane = threadIdx.x & 63, c = lane & 15, h = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const float inf = __builtin_inff();

  // Blocks of one head of keys are neighbours: an XCD's L2 holds it once.
  int id = xcd_contiguous(blockIdx.x, (int)gridDim.x);
  const int split = id % p.splits;
  const int unit = id / p.splits;
  const int group = unit % p.groups;
  const int bh = unit / p.groups;
  const int b = bh / p.c.H, head = bh % p.c.H;

  const int past = p.c.past[b];
  int count = p.S;
  if (p.c.counts) {
    const int n = p.c.counts[b];
    count = n < 0 ? 0 : n < p.S ? n : p.S;
  }
  const int rows = count * p.per_head, row0 = group * RT * 16;
  if (row0 >= rows)
    return;
  const int last_row = (row0 + RT * 16 < rows ? row0 + RT * 16 : rows) - 1;
  const int64_t capacity =
      p.c.table ? p.c.table_pages * p.c.page_size : p.c.page_size;
  // Keys [first, end) of the query of token i.
  const int64_t start = p.starts ? p.starts[b] : 0;
  auto first_of = [&](int i) -> int {
    int64_t f = start > 0 ? start : 0;
    if (p.window > 0 && past + (int64_t)i - p.window + 1 > f)
      f = past + (int64_t)i - p.window + 1;
    return (int)(f < capacity ? f : capacity);
  };
  auto end_of = [&](int i) -> int {
    const int64_t e = past + (int64_t)(p.causal ? i : count - 1) + 1;
    return (int)(e < 0 ? 0 : e < capacity ? e : capacity);
  };
  const int i0 = row0 / p.per_head, i1 = last_row / p.per_head;
  const int lo = first_of(i0), hi = end_of(i1);
  const int all_lo = first_of(i1), all_hi = end_of(i0); // seen by all rows
  int tile = lo / 32, tiles = hi > lo ? (hi + 31) / 32 - tile : 0;
  {
    const int each = (tiles + p.splits - 1) / p.splits;
    tile += split * each;
    tiles = tiles - split * each < each ? tiles - split * each : each;
  }

  // This lane's rows.
  v8bf q[RT][G][TQ];
  float qsum[RT][G];
  int row_lo[RT], row_hi[RT];
#pragma unroll
  for (int r = 0; r < RT; ++r) {
    int row = row0 + 16 * r + c;
    row = row < rows ? row : rows - 1;
    const int i = row / p.per_head, qh = head * p.per_head + row % p.per_head;
    row_lo[r] = first_of(i);
    row_hi[r] = end_of(i);
    const int64_t at = p.heads_first ? ((int64_t)b * p.heads + qh) * p.S + i
                                     : ((int64_t)b * p.S + i) * p.heads + qh;
    const T *const x = (const T *)p.q + at * D + 8 * h;
#pragma unroll
    for (int g = 0; g < G; ++g) {
      float v[8];
#pragma unroll
      for (int j = 0; j < 8; ++j)
        v[j] = to_f32(x[32 * g + j]);
      float sum = ((v[0] + v[1]) + (v[2] + v[3])) + ((v[4] + v[5]) + (v[6] + v[7]));
      sum += __shfl_xor(sum, 16);
      qsum[r][g] = sum + __shfl_xor(sum, 32);
      const float order[8] = {v[0], v[2], v[4], v[6], v[1], v[3], v[5], v[7]};
      terms_of<TQ>(order, q[r][g]);
    }
  }
  const float scale =
      (p.scale ? p.scale[0] : 1.0f / __builtin_sqrtf((float)D)) * kLog2E;

  v4f o[RT][2 * G];
  float top[RT], sum[RT], low[RT][G]; // low: sum of p m
#pragma unroll
  for (int r = 0; r < RT; ++r) {
    top[r] = -inf;
    sum[r] = 0.0f;
#pragma unroll
    for (int g = 0; g < G; ++g) {
      low[r][g] = 0.0f;
      o[r][2 * g] = o[r][2 * g + 1] = v4f{0, 0, 0, 0};
    }
  }

  for (int t = tile + wave; t < tile + tiles; t += kWaves) {
    const int key0 = t * 32;
    bool whole = key0 >= all_lo && key0 + 32 <= all_hi;
    bool known[2];
    unsigned kw[2][4][G], vw[2][4][(G + 3) / 4];
    v2h ks[2][4][G], vs[2][4][G];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const Place at = place_of(p.c, b, head, key0 + 16 * u < capacity ? key0 + 16 * u : 0);
      known[u] = at.known;
      whole = whole && at.known;
      const int mine = c < at.last ? c : at.last;
      unsigned w[G];
      load_bytes<4 * G, 4 * (G & -G) < 16 ? 4 * (G & -G) : 16>(
          p.c.k_codes + at.row * (16 * G) + mine * (16 * G) + h * (4 * G), w);
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < G; ++j)
          kw[u][i][j] = w[j];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int key = 4 * h + i < at.last ? 4 * h + i : at.last;
        load_bytes<G, (G & -G)>(p.c.v_codes + at.row * (16 * G) + key * (16 * G) + c * G, vw[u][i]);
        const unsigned *const ka = (const unsigned *)p.c.k_scales + at.row * G + key * G;
        const unsigned *const va = (const unsigned *)p.c.v_scales + at.row * G + key * G;
        const Pack<unsigned, G & -G> *const kp = (const Pack<unsigned, G & -G> *)ka;
        const Pack<unsigned, G & -G> *const vp = (const Pack<unsigned, G & -G> *)va;
#pragma unroll
        for (int g = 0; g < G; g += G & -G) {
          const Pack<unsigned, G & -G> a = kp[g / (G & -G)], bb = vp[g / (G & -G)];
#pragma unroll
          for (int j = 0; j < (G & -G); ++j) {
            ks[u][i][g + j] = __builtin_bit_cast(v2h, a.v[j]);
            vs[u][i][g + j] = __builtin_bit_cast(v2h, bb.v[j]);
          }
        }
      }
    }

    // scores, in powers of two
    float s[RT][8];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      unsigned codes[G];
      bytes_of<G, G>(kw[u], codes);
      float part[RT][4];
#pragma unroll
      for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          part[r][i] = 0.0f;
#pragma unroll
      for (int g = 0; g < G; ++g) {
        v2bf n0, n1, n2, n3;
        numbers(codes[g] & 0x0F0F0F0Fu, n0, n1);
        numbers(codes[g] >> 4 & 0x0F0F0F0Fu, n2, n3);
        const v8bf k = join(n0, n1, n2, n3);
#pragma unroll
        for (int r = 0; r < RT; ++r) {
          v4f acc = {0, 0, 0, 0};
#pragma unroll
          for (int e = TQ - 1; e >= 0; --e)
            acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k, q[r][g][e], acc, 0, 0, 0);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            part[r][i] = __builtin_fmaf((float)ks[u][i][g][0], acc[i], part[r][i]);
            part[r][i] = __builtin_fmaf((float)ks[u][i][g][1], qsum[r][g], part[r][i]);
          }
        }
      }
#pragma unroll
      for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          s[r][4 * u + i] = part[r][i] * scale;
    }
    if (!whole) {
#pragma unroll
      for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int key = key0 + 16 * (j / 4) + 4 * h + j % 4;
          if (!(known[j / 4] && key >= row_lo[r] && key < row_hi[r]))
            s[r][j] = -inf;
        }
    }

    // maxima: what p is relative to stays unless a row's grows by more than 8
    float most[RT];
    bool grown = false;
#pragma unroll
    for (int r = 0; r < RT; ++r) {
      most[r] = s[r][0];
#pragma unroll
      for (int j = 1; j < 8; ++j)
        most[r] = __builtin_fmaxf(most[r], s[r][j]);
      grown = grown || most[r] > top[r] + 8.0f;
    }
    if (__any(grown)) {
#pragma unroll
      for (int r = 0; r < RT; ++r) {
        float m = __builtin_fmaxf(most[r], __shfl_xor(most[r], 16));
        m = __builtin_fmaxf(m, __shfl_xor(m, 32));
        m = __builtin_fmaxf(m, top[r]);
        const float less = m == top[r] ? 1.0f : __builtin_amdgcn_exp2f(top[r] - m);
        top[r] = m;
        sum[r] *= less;
#pragma unroll
        for (int g = 0; g < G; ++g) {
          low[r][g] *= less;
          o[r][2 * g] *= less;
          o[r][2 * g + 1] *= less;
        }
      }
    }
#pragma unroll
    for (int r = 0; r < RT; ++r) {
      const float base = top[r] == -inf ? 0.0f : top[r]; // no key seen so far
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        s[r][j] = __builtin_amdgcn_exp2f(s[r][j] - base);
        sum[r] += s[r][j];
      }
    }

    // output
    unsigned codes[2][G];
    bytes_of<G, 0>(vw[0], codes[0]);
    bytes_of<G, 0>(vw[1], codes[1]);
#pragma unroll
    for (int g = 0; g < G; ++g) {
      v2bf n0, n1, n2, n3, n4, n5, n6, n7;
      numbers(codes[0][g] & 0x0F0F0F0Fu, n0, n1);
      numbers(codes[1][g] & 0x0F0F0F0Fu, n2, n3);
      numbers(codes[0][g] >> 4 & 0x0F0F0F0Fu, n4, n5);
      numbers(codes[1][g] >> 4 & 0x0F0F0F0Fu, n6, n7);
      const v8bf even = join(n0, n1, n2, n3), odd = join(n4, n5, n6, n7);
#pragma unroll
      for (int r = 0; r < RT; ++r) {
        float ps[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const v2h pair = vs[j / 4][j % 4][g];
          float vscale = (float)pair[0], vlow = (float)pair[1];
          if (!whole && s[r][j] == 0.0f) // nothing of a key that is not seen
            vscale = vlow = 0.0f;
          ps[j] = s[r][j] * vscale;
          low[r][g] = __builtin_fmaf(s[r][j], vlow, low[r][g]);
        }
        v8bf t[TP];
        terms_of<TP>(ps, t);
#pragma unroll
        for (int e = TP - 1; e >= 0; --e) {
          o[r][2 * g] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(even, t[e], o[r][2 * g], 0, 0, 0);
          o[r][2 * g + 1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(odd, t[e], o[r][2 * g + 1], 0, 0, 0);
        }
      }
    }
  }

  // The waves' results meet in LDS: [wave][g][lane][8] output, then (max, sum).
  float *const stats = shared + kWaves * G * 64 * 8;
#pragma unroll 1
  for (int r = 0; r < RT; ++r) {
    float my_top = 0, my_sum = 0;
#pragma unroll
    for (int k = 0; k < RT; ++k) {
      if (k != r)
        continue;
      my_top = top[k];
      my_sum = sum[k];
      my_sum += __shfl_xor(my_sum, 16);
      my_sum += __shfl_xor(my_sum, 32);
#pragma unroll
      for (int g = 0; g < G; ++g) {
        float l = low[k][g];
        l += __shfl_xor(l, 16);
        l += __shfl_xor(l, 32);
        float *const to = shared + ((wave * G + g) * 64 + lane) * 8;
        const v4f e = o[k][2 * g] + l, f = o[k][2 * g + 1] + l;
        *(v4f *)to = v4f{e[0], f[0], e[1], f[1]};
        *(v4f *)(to + 4) = v4f{e[2], f[2], e[3], f[3]};
      }
    }
    if (h == 0) {
      stats[(wave * 16 + c) * 2] = my_top;
      stats[(wave * 16 + c) * 2 + 1] = my_sum;
    }
    __syncthreads();
    const int row = row0 + 16 * r + c;
    float m = -inf, total = 0.0f, factor[kWaves];
#pragma unroll
    for (int w = 0; w < kWaves; ++w)
      m = __builtin_fmaxf(m, stats[(w * 16 + c) * 2]);
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      const float mw = stats[(w * 16 + c) * 2];
      factor[w] = mw == -inf ? 0.0f : __builtin_amdgcn_exp2f(mw - m);
      total += stats[(w * 16 + c) * 2 + 1] * factor[w];
    }
    if (row < rows) {
      const int64_t part = ((int64_t)unit * p.splits + split) * (RT * 16) + 16 * r + c;
      const int i = row / p.per_head, qh = head * p.per_head + row % p.per_head;
      const int64_t at = p.heads_first ? ((int64_t)b * p.heads + qh) * p.S + i
                                       : ((int64_t)b * p.S + i) * p.heads + qh;
      for (int g = wave; g < G; g += kWaves) {
        float v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j)
          v[j] = 0.0f;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
          const float *const from = shared + ((w * G + g) * 64 + lane) * 8;
          // (a wave without keys holds zeros)
#pragma unroll
          for (int j = 0; j < 8; ++j)
            v[j] = __builtin_fmaf(from[j], factor[w], v[j]);
        }
        if (p.splits == 1) {
          const float over = total == 0.0f ? 0.0f : 1.0f / total;
          T *const y = (T *)p.y + at * D + 32 * g + 8 * h;
          Pack<T, 8> out;
#pragma unroll
          for (int j = 0; j < 8; ++j)
            out.v[j] = from_f32<T>(v[j] * over);
          *(Pack<T, 8> *)y = out;
        } else {
          float *const y = p.parts + part * D + 32 * g + 8 * h;
          *(v4f *)y = v4f{v[0], v[1], v[2], v[3]};
          *(v4f *)(y + 4) = v4f{v[4], v[5], v[6], v[7]};
        }
      }
      if (p.splits > 1 && wave == 0 && h == 0) {
        float *const st = p.parts + (int64_t)p.B * p.c.H * p.groups * p.splits * (RT * 16) * D + part * 2;
        st[0] = m;
        st[1] = total;
      }
    }
    __syncthreads();
  }
}

// The parts of a row's keys joined: thread (s, d) sums every 8th part's
// elements 4 d .., and the eight sums meet in LDS.
template <typename T>
__global__ __launch_bounds__(256) void k_cache_join(const Arguments p, int D, int tile_rows) {
  extern __shared__ __attribute__((aligned(16))) float shared[];
  const int lanes = D / 4, across = 256 / lanes; // threads of a row, parts at once
  const int unit = blockIdx.x / tile_rows, r = blockIdx.x % tile_rows;
  const int group = unit % p.groups, bh = unit / p.groups;
  const int b = bh / p.c.H, head = bh % p.c.H;
  int count = p.S;
  if (p.c.counts) {
    const int n = p.c.counts[b];
    count = n < 0 ? 0 : n < p.S ? n : p.S;
  }
  const int row = group * tile_rows + r;
  if (row >= count * p.per_head)
    return;
  const float inf = __builtin_inff();
  const float *const stats = p.parts + (int64_t)p.B * p.c.H * p.groups * p.splits * tile_rows * D;
  const int64_t part0 = (int64_t)unit * p.splits * tile_rows + r;
  const int s0 = threadIdx.x / lanes, d = threadIdx.x % lanes;
  float m = -inf;
  for (int s = 0; s < p.splits; ++s)
    m = __builtin_fmaxf(m, stats[(part0 + (int64_t)s * tile_rows) * 2]);
  v4f v = {0, 0, 0, 0};
  float total = 0.0f;
  if (s0 < across)
    for (int s = s0; s < p.splits; s += across) {
      const int64_t part = part0 + (int64_t)s * tile_rows;
      const float ms = stats[part * 2];
      const float f = ms == -inf ? 0.0f : __builtin_amdgcn_exp2f(ms - m);
      total += stats[part * 2 + 1] * f;
      v += *(const v4f *)(p.parts + part * D + 4 * d) * f;
    }
  float *const mine = shared + threadIdx.x * 8;
  *(v4f *)mine = v;
  mine[4] = total;
  __syncthreads();
  if (s0 > 0)
    return;
  for (int s = 1; s < across; ++s) {
    const float *const other = shared + (s * lanes + d) * 8;
    v += *(const v4f *)other;
    total += other[4];
  }
  const float over = total == 0.0f ? 0.0f : 1.0f / total;
  const int i = row / p.per_head, qh = head * p.per_head + row % p.per_head;
  const int64_t at = p.heads_first ? ((int64_t)b * p.heads + qh) * p.S + i
                                   : ((int64_t)b * p.S + i) * p.heads + qh;
  Pack<T, 4> out;
#pragma unroll
  for (int j = 0; j < 4; ++j)
    out.v[j] = from_f32<T>(v[j] * over);
  *(Pack<T, 4> *)((T *)p.y + at * D + 4 * d) = out;
}

int row_tiles(const Attention4 &a) {
  return a.S * (a.heads / a.c.H) > 16 && a.c.D <= 128 ? 2 : 1;
}
int64_t row_groups(const Attention4 &a) {
  const int rows = 16 * row_tiles(a);
  return (a.S * (a.heads / a.c.H) + rows - 1) / rows;
}

template <typename T, int G, int RT>
hipError_t attend(hipStream_t st, const Arguments &p) {
  constexpr int kLds = (kWaves * G * 64 * 8 + kWaves * 16 * 2) * 4;
  auto *const kernel = k_cache_attention<T, G, RT>;
  if (kLds > 65536) {
    const hipError_t e = hipFuncSetAttribute((const void *)kernel,
        hipFuncAttributeMaxDynamicSharedMemorySize, kLds);
    if (e != hipSuccess)
      return e;
  }
  const int64_t units = (int64_t)p.B * p.c.H * p.groups;
  kernel<<<dim3((unsigned)(units * p.splits)), kWaves * 64, kLds, st>>>(p);
  hipError_t e = hipGetLastError();
  if (e == hipSuccess && p.splits > 1) {
    k_cache_join<T><<<dim3((unsigned)(units * RT * 16)), 256, 256 * 8 * 4, st>>>(p, 32 * G, RT * 16);
    e = hipGetLastError();
  }
  return e;
}

template <typename T>
hipError_t attend_any(hipStream_t st, const Arguments &p, int tiles) {
  switch (p.c.D / kCacheGroup) {
  case 2:
    return tiles > 1 ? attend<T, 2, 2>(st, p) : attend<T, 2, 1>(st, p);
  case 3:
    return tiles > 1 ? attend<T, 3, 2>(st, p) : attend<T, 3, 1>(st, p);
  case 4:
    return tiles > 1 ? attend<T, 4, 2>(st, p) : attend<T, 4, 1>(st, p);
  case 6:
    return attend<T, 6, 1>(st, p);
  default:
    return attend<T, 8, 1>(st, p);
  }
}

template <typename T>
hipError_t append_any(hipStream_t st, const Append4 &a) {
  const int64_t threads = 2 * a.B * a.S * a.c.H * 16;
  const dim3 grid((unsigned)((threads + 255) / 256));
  switch (a.c.D / kCacheGroup) {
  case 2:
    k_cache_append<T, 2><<<grid, 256, 0, st>>>(a);
    break;
  case 3:
    k_cache_append<T, 3><<<grid, 256, 0, st>>>(a);
    break;
  case 4:
    k_cache_append<T, 4><<<grid, 256, 0, st>>>(a);
    break;
  case 6:
    k_cache_append<T, 6><<<grid, 256, 0, st>>>(a);
    break;
  default:
    k_cache_append<T, 8><<<grid, 256, 0, st>>>(a);
  }
  return hipGetLastError();
}

} // namespace
} // namespace llm

using namespace llm;

bool attention_head_ok(int D) {
  return D == 64 || D == 96 || D == 128 || D == 192 || D == 256;
}

hipError_t launch_cache_append(hipStream_t s, const Append4 &a) {
  switch (a.kind) {
  case kF32:
    return append_any<float>(s, a);
  case kF16:
    return append_any<_Float16>(s, a);
  default:
    return append_any<__bf16>(s, a);
  }
}

// Parts of the keys, so that a few rows fill the GPU: about four blocks a CU,
// of 128 keys at least.  (How many keys there are, only the GPU knows: a block
// takes its share of what its rows see.)
int attention_splits(const Attention4 &a) {
  const int64_t units = a.B * a.c.H * row_groups(a);
  const int64_t capacity = a.c.table ? a.c.table_pages * a.c.page_size : a.c.page_size;
  int64_t n = 1024 / (units > 0 ? units : 1);
  if (n > (capacity + 127) / 128)
    n = (capacity + 127) / 128;
  return (int)(n < 1 ? 1 : n < 256 ? n : 256);
}
size_t attention_parts_bytes(const Attention4 &a) {
  const int64_t rows = a.B * a.c.H * row_groups(a) * 16 * row_tiles(a);
  return (size_t)rows * a.splits * (a.c.D + 2) * sizeof(float);
}

hipError_t launch_cache_attention(hipStream_t s, const Attention4 &a) {
  Arguments p = {a.c, a.q, a.y, a.starts, a.scale, a.parts, a.window, (int)a.B,
      (int)a.S, (int)a.heads, (int)(a.heads / a.c.H), (int)row_groups(a), a.splits,
      a.causal, a.heads_first};
  switch (a.kind) {
  case kF32:
    return attend_any<float>(s, p, row_tiles(a));
  case kF16:
    return attend_any<_Float16>(s, p, row_tiles(a));
  default:
    return attend_any<__bf16>(s, p, row_tiles(a));
  }
}

} // namespace om
