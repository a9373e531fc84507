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

#include <type_traits>

#include "gemm_common.h"
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
  // (a sequence's pages hold 2^30 tokens at most)
  bool known = key >= 0 && key < (c.table ? c.table_pages * c.page_size : c.page_size);
  if (c.table && known) {
    const unsigned at = (unsigned)key / (unsigned)c.page_size;
    page = c.table[b * c.table_pages + at];
    slot = (unsigned)key - at * (unsigned)c.page_size;
  }
  known = known && page >= 0 && page < c.pages;
  if (!known)
    page = slot = 0;
  return {(page * c.H + h) * c.page_size + slot, (int)(c.page_size - 1 - slot), known};
}

// ---------------------------------------------------------------------------
// append
// ---------------------------------------------------------------------------
// 16 lanes quantize a row, lane n elements 2 n and 2 n + 1 of every group.
// Bound by the launch for the few rows of a decode step, by vector instructions for
// a prompt's: some 90 for each group and 64 lanes, of them 34 for extremes and 24 for
// exact quotients (4 x 512 tokens of 8 heads of 128, f16: 7.6 us; 8.5 with branches
// around the quotients, which worked on one group after the other).
template <typename T, int G>
__global__ __launch_bounds__(256) void k_cache_append(const Append4 p, int64_t first) {
  const int n = threadIdx.x & 15;
  int64_t id = first + (((int64_t)blockIdx.x * 256 + threadIdx.x) >> 4);
  const int64_t rows = p.B * p.S * p.c.H;
  if (id >= 2 * rows)
    return;
  const bool value = id >= rows;
  if (value)
    id -= rows;
  // rows in the order of k and v (there are fewer than 2^31: each has 64 elements)
  const unsigned row = (unsigned)id, S = (unsigned)p.S, H = (unsigned)p.c.H;
  const unsigned outer = row / (p.heads_first ? S : H), inner = row - outer * (p.heads_first ? S : H);
  const unsigned b = outer / (p.heads_first ? H : S), mid = outer - b * (p.heads_first ? H : S);
  const int64_t i = p.heads_first ? inner : mid;
  const int h = (int)(p.heads_first ? mid : inner);
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
    bool bad = false;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      e[j] = to_f32(in[g].v[j]);
      bad = bad || e[j] != e[j];
      e[j] = __builtin_fminf(__builtin_fmaxf(e[j], -65504.0f), 65504.0f);
    }
    const bool none = (__ballot(bad) >> (threadIdx.x & 48) & 0xFFFF) != 0;
    const float top = row_max(__builtin_fmaxf(e[0], e[1]));
    const float low = -row_max(__builtin_fmaxf(-e[0], -e[1]));
    const _Float16 m = none ? (_Float16)__builtin_nanf("") : (_Float16)low;
    // (lowest may have been rounded up, past the largest)
    const _Float16 s = none ? m : (_Float16)__builtin_fmaxf((top - (float)m) * (1.0f / 15.0f), 0.0f);
    // (0 where s is 0 or NaN, without a branch: groups are worked on side by side)
    const float most = (float)s > 0.0f ? 15.0f : 0.0f;
    unsigned code = 0;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const float q = __builtin_rintf((e[j] - (float)m) / (float)s);
      code |= (unsigned)__builtin_fminf(__builtin_fmaxf(q, 0.0f), most) << (4 * j);
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
// A wave takes RT tiles of rows (queries of the heads that share one of keys)
// and 32 keys at a time.  Keys are the first operand of the first product and
// elements of a value that of the second, so that lane (c, h) holds column c of
// either throughout: scores of keys 4 h .. of each 16, which are also its places
// of the second product's operand.  No score moves between lanes but the rows'
// maxima, and those only when one grows by more than 8 (powers of two) over
// what p is relative to.
//
// A tile's 16 columns are 16 rows; or, where there are few, PACKED: 16 / G rows
// times G groups.  Column (g, r) of q then holds group g of row r and zeros, its
// products that group's part of the score, to be scaled by the one scale the
// lane has and summed over the columns of the row; and its weights are scaled
// for group g, of whose elements alone the results are kept.  The matrix
// instructions are as many, the vector ones, which bound the kernel, less than
// half: a lane scales and splits 8 weights for 32 keys, not 8 G.
//
// An infinity in a query, or as the scale, makes every score infinite or NaN, and so
// each row that sees a key NaN: it is taken as NaN, for scores of -inf alone would
// look like a row that sees none.
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

__device__ __forceinline__ float finite_or_nan(float x) { return __builtin_fmaf(x, 0.0f, x); }

// Bytes at[i] + g of the four strings w[i], for i = 0 .. 3 and every g.
template <int G, int STEP, int WORDS>
__device__ __forceinline__ void bytes_of(
    const unsigned *const (&w)[4], unsigned (&codes)[G]) {
#pragma unroll
  for (int g = 0; g < G; g += G % 2 ? 1 : 2) {
    const unsigned w0 = w[0][g / 4], w1 = w[1][(STEP + g) / 4],
                   w2 = w[2][(2 * STEP + g) / 4], w3 = w[3][(3 * STEP + g) / 4];
    const unsigned s0 = g % 4, s1 = (STEP + g) % 4, s2 = (2 * STEP + g) % 4,
                   s3 = (3 * STEP + g) % 4;
    if (G % 2) {
      const unsigned x = __builtin_amdgcn_perm(w1, w0, s0 | (4 + s1) << 8);
      const unsigned y = __builtin_amdgcn_perm(w3, w2, s2 | (4 + s3) << 8);
      codes[g] = __builtin_amdgcn_perm(y, x, 0x05040100);
    } else {
      const unsigned x = __builtin_amdgcn_perm(
          w1, w0, s0 | (4 + s1) << 8 | (s0 + 1) << 16 | (5 + s1) << 24);
      const unsigned y = __builtin_amdgcn_perm(
          w3, w2, s2 | (4 + s3) << 8 | (s2 + 1) << 16 | (5 + s3) << 24);
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
  typedef float v2f __attribute__((ext_vector_type(2)));
  v2bf part[N][4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float a = x[2 * i], b = x[2 * i + 1];
#pragma unroll
    for (int k = 0; k < N; ++k) {
      part[k][i] = __builtin_convertvector(v2f{a, b}, v2bf);
      if (k + 1 < N) {
        const unsigned w = __builtin_bit_cast(unsigned, part[k][i]);
        a -= __builtin_bit_cast(float, w << 16);
        b -= __builtin_bit_cast(float, w & 0xFFFF0000u);
      }
    }
  }
#pragma unroll
  for (int k = 0; k < N; ++k)
    t[k] = join(part[k][0], part[k][1], part[k][2], part[k][3]);
}

// N words (or, with B, bytes) at a lane's offset from what a descriptor covers;
// behind its end lie zeros.
template <int N>
__device__ __forceinline__ void load_words(
    __amdgpu_buffer_rsrc_t from, int at, unsigned (&w)[N]) {
  constexpr int W = N % 4 == 0 ? 4 : N % 3 == 0 ? 3 : N;
  static_assert(W <= 4, "words of a load");
#pragma unroll
  for (int i = 0; i < N; i += W) {
    if constexpr (W == 4) {
      const v4u v = __builtin_amdgcn_raw_buffer_load_b128(from, at + 4 * i, 0, 0);
      w[i] = v[0], w[i + 1] = v[1], w[i + 2] = v[2], w[i + 3] = v[3];
    } else if constexpr (W == 3) {
      const auto v = __builtin_amdgcn_raw_buffer_load_b96(from, at + 4 * i, 0, 0);
      w[i] = v[0], w[i + 1] = v[1], w[i + 2] = v[2];
    } else if constexpr (W == 2) {
      const v2u v = __builtin_amdgcn_raw_buffer_load_b64(from, at + 4 * i, 0, 0);
      w[i] = v[0], w[i + 1] = v[1];
    } else {
      w[i] = __builtin_amdgcn_raw_buffer_load_b32(from, at + 4 * i, 0, 0);
    }
  }
}
template <int B>
__device__ __forceinline__ void load_bytes(
    __amdgpu_buffer_rsrc_t from, int at, unsigned (&w)[(B + 3) / 4]) {
  if constexpr (B % 4 == 0) {
    load_words<B / 4>(from, at, w);
  } else {
    constexpr int P = B % 2 ? 1 : 2; // bytes of a load
#pragma unroll
    for (int i = 0; i < (B + 3) / 4; ++i)
      w[i] = 0;
#pragma unroll
    for (int i = 0; i < B; i += P)
      w[i / 4] |= (unsigned)(P == 2 ? (unsigned)__builtin_amdgcn_raw_buffer_load_b16(from, at + i, 0, 0)
                                    : (unsigned)__builtin_amdgcn_raw_buffer_load_b8(from, at + i, 0, 0))
                  << (8 * (i % 4));
  }
}

// The sum over the G columns of a row (lanes c, c + 16 / G, ..), in all of them:
// each step adds what the other half of a rotation holds, so every lane adds the
// same numbers in the same order.
template <int G> __device__ __forceinline__ float columns_sum(float v) {
#define OM_ROW_ADD(ctrl)                                                       \
  v += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(                    \
                                     0, __builtin_bit_cast(int, v), ctrl, 0xF,   \
                                     0xF, true))
  OM_ROW_ADD(0x128); // row_ror:8
  if (G > 2)
    OM_ROW_ADD(0x124);
  if (G > 4)
    OM_ROW_ADD(0x122);
#undef OM_ROW_ADD
  return v;
}

constexpr int kWaves = 4;
constexpr float kLog2E = 0x1.715476p+0f;

template <typename T> struct Terms;
template <> struct Terms<float> { static constexpr int q = 3, p = 3; };
template <> struct Terms<_Float16> { static constexpr int q = 2, p = 2; };
template <> struct Terms<__bf16> { static constexpr int q = 1, p = 2; };

template <typename T, int G, int RT, bool PACKED>
__global__ __launch_bounds__(kWaves * 64, PACKED && G * RT <= 4 ? 2 : 1) void k_cache_attention(const Arguments p) {
  constexpr int D = 32 * G, TQ = Terms<T>::q, TP = Terms<T>::p;
  constexpr int ROWS = PACKED ? 16 / G : 16; // of a tile
  constexpr int SG = PACKED ? 1 : G;         // groups whose scales a lane holds
  static_assert(!PACKED || 16 % G == 0, "columns");
  extern __shared__ __attribute__((aligned(16))) float shared[];
  const int lane = threadIdx.x & 63, c = lane & 15, h = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int my_row = PACKED ? c % ROWS : c, my_group = PACKED ? c / ROWS : 0;
  const float inf = __builtin_inff();

  // Blocks of one head of keys are neighbours: an XCD's L2 holds it once.
  const int id = xcd_contiguous(blockIdx.x, (int)gridDim.x);
  const int split = (unsigned)id % (unsigned)p.splits;
  const int unit = (unsigned)id / (unsigned)p.splits;
  const int group = (unsigned)unit % (unsigned)p.groups;
  const int bh = (unsigned)unit / (unsigned)p.groups;
  const int b = (unsigned)bh / (unsigned)p.c.H, head = (unsigned)bh % (unsigned)p.c.H;

  const int past = p.c.past[b];
  int count = p.S;
  if (p.c.counts) {
    const int n = p.c.counts[b];
    count = n < 0 ? 0 : n < p.S ? n : p.S;
  }
  const int rows = count * p.per_head, row0 = group * RT * ROWS;
  if (row0 >= rows)
    return;
  const int last_row = (row0 + RT * ROWS < rows ? row0 + RT * ROWS : rows) - 1;
  const unsigned page_size = (unsigned)p.c.page_size;
  const int capacity = (int)(p.c.table ? p.c.table_pages * p.c.page_size : p.c.page_size);
  // Keys [first, end) of the query of token i.
  const int start = p.starts ? p.starts[b] : 0;
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
  // Tiles of 32 keys: this part's, of which the wave takes every kWaves-th.
  int tile = lo / 32, tiles = hi > lo ? (hi + 31) / 32 - tile : 0;
  {
    const int each = (tiles + p.splits - 1) / p.splits;
    tile += split * each;
    tiles = tiles - split * each < each ? tiles - split * each : each;
    tile += wave;
    tiles = tiles > wave ? (tiles - wave + kWaves - 1) / kWaves : 0;
  }

  // This lane's rows.
  v8bf q[RT][G][TQ];
  float qsum[RT][SG];
  int row_lo[RT], row_hi[RT];
#pragma unroll
  for (int r = 0; r < RT; ++r) {
    int row = row0 + ROWS * r + my_row;
    row = row < rows ? row : rows - 1;
    const int i = row / p.per_head, qh = head * p.per_head + row % p.per_head;
    row_lo[r] = first_of(i);
    row_hi[r] = end_of(i);
    const int64_t at = p.heads_first ? ((int64_t)b * p.heads + qh) * p.S + i
                                     : ((int64_t)b * p.S + i) * p.heads + qh;
    const T *const x = (const T *)p.q + at * D + 8 * h;
    if (PACKED)
      qsum[r][0] = 0.0f;
#pragma unroll
    for (int g = 0; g < G; ++g) {
      const bool held = !PACKED || g == my_group;
      float v[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        v[j] = held ? to_f32(x[32 * g + j]) : 0.0f;
        if (TQ == 1) // (an infinity's second term is NaN by itself)
          v[j] = finite_or_nan(v[j]);
      }
      float sum = ((v[0] + v[1]) + (v[2] + v[3])) + ((v[4] + v[5]) + (v[6] + v[7]));
      sum += __shfl_xor(sum, 16);
      sum += __shfl_xor(sum, 32);
      if (PACKED)
        qsum[r][0] = held ? sum : qsum[r][0];
      else
        qsum[r][g] = sum;
      const float order[8] = {v[0], v[2], v[4], v[6], v[1], v[3], v[5], v[7]};
      terms_of<TQ>(order, q[r][g]);
    }
  }
  const float scale =
      (p.scale ? finite_or_nan(p.scale[0]) : 1.0f / __builtin_sqrtf((float)D)) * kLog2E;

  v4f o[RT][2 * G];
  float top[RT], sum[RT], low[RT][SG]; // low: sum of p m
#pragma unroll
  for (int r = 0; r < RT; ++r) {
    top[r] = -inf;
    sum[r] = 0.0f;
#pragma unroll
    for (int g = 0; g < SG; ++g)
      low[r][g] = 0.0f;
#pragma unroll
    for (int g = 0; g < 2 * G; ++g)
      o[r][g] = v4f{0, 0, 0, 0};
  }

  // Where the wave's keys lie: lane l knows the cache's row of the first of 16
  // keys, half l % 2 of the wave's tile l / 2 from `known_from` on.  (There are
  // fewer than 2^32 rows: the smallest take 40 bytes twice.)
  constexpr unsigned kNowhere = ~0u;
  unsigned place = kNowhere;
  int known_from = 0;
  auto find_places = [&](int from) {
    known_from = from;
    const int key = (tile + kWaves * (from + (lane >> 1))) * 32 + 16 * (lane & 1);
    place = kNowhere;
    if (key < capacity) {
      unsigned page = (unsigned)b, slot = (unsigned)key;
      if (p.c.table) {
        const unsigned at = (unsigned)key / page_size;
        page = (unsigned)p.c.table[b * p.c.table_pages + at];
        slot = (unsigned)key - at * page_size;
      }
      if (page < (uint64_t)p.c.pages)
        place = (page * (unsigned)p.c.H + (unsigned)head) * page_size + slot;
    }
  };

  // Codes and scales of 32 keys, as they lie: of keys c of each 16, the quarter h
  // of the row; of keys 4 h + i, bytes c G .. of the values' rows.  Descriptors
  // cover what the page holds of the 16 keys, nothing of a page that is none.
  struct Tile {
    unsigned k[2][G], v[2][4][(G + 3) / 4], ks[2][4][SG], vs[2][4][SG];
    bool known[2];
  };
  const int k_at = c * (16 * G) + h * (4 * G);
  const int v_at = 4 * h * (16 * G) + c * G, s_at = 4 * h * (4 * G) + 4 * my_group;
  auto load = [&](Tile &t, int j) {
    if (j - known_from >= 32)
      find_places(j);
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const unsigned found = __builtin_amdgcn_readlane(place, 2 * (j - known_from) + u);
      const bool known = found != kNowhere;
      t.known[u] = known;
      const int64_t row = known ? found : 0;
      int room = capacity - ((tile + kWaves * j) * 32 + 16 * u);
      room = !known ? 0 : room < 16 ? room : 16; // (whole pages hold all 16)
      auto part = [&](const void *base, int row_bytes) {
        return __builtin_amdgcn_make_buffer_rsrc(
            (void *)((const char *)base + row * row_bytes), 0, room * row_bytes, 0x00020000);
      };
      const auto kc = part(p.c.k_codes, 16 * G), vc = part(p.c.v_codes, 16 * G);
      const auto kp = part(p.c.k_scales, 4 * G), vp = part(p.c.v_scales, 4 * G);
      load_words<G>(kc, k_at, t.k[u]);
#pragma unroll
      for (int i = 0; i < 4; ++i)
        load_words<SG>(kp, s_at + i * (4 * G), t.ks[u][i]);
#pragma unroll
      for (int i = 0; i < 4; ++i)
        load_bytes<G>(vc, v_at + i * (16 * G), t.v[u][i]);
#pragma unroll
      for (int i = 0; i < 4; ++i)
        load_words<SG>(vp, s_at + i * (4 * G), t.vs[u][i]);
    }
  };
  auto halves = [](unsigned w) { return __builtin_bit_cast(v2h, w); };

  // masked: some rows do not see some of the keys.
  auto step_on = [&](const Tile &t, int key0, auto masked) {
    // scores, in powers of two
    float s[RT][8];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      unsigned codes[G];
      const unsigned *const w[4] = {t.k[u], t.k[u], t.k[u], t.k[u]};
      bytes_of<G, G, G>(w, codes);
      v4f acc[RT][SG];
#pragma unroll
      for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int g = 0; g < SG; ++g)
          acc[r][g] = v4f{0, 0, 0, 0};
#pragma unroll
      for (int g = 0; g < G; ++g) {
        v2bf n0, n1, n2, n3;
        numbers(codes[g] & 0x0F0F0F0Fu, n0, n1);
        numbers(codes[g] >> 4 & 0x0F0F0F0Fu, n2, n3);
        const v8bf k = join(n0, n1, n2, n3);
#pragma unroll
        for (int r = 0; r < RT; ++r)
#pragma unroll
          for (int e = TQ - 1; e >= 0; --e)
            acc[r][PACKED ? 0 : g] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                k, q[r][g][e], acc[r][PACKED ? 0 : g], 0, 0, 0);
      }
#pragma unroll
      for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float part = 0.0f;
#pragma unroll
          for (int g = 0; g < SG; ++g) {
            const v2h pair = halves(t.ks[u][i][g]);
            part = __builtin_fmaf((float)pair[0], acc[r][g][i], part);
            part = __builtin_fmaf((float)pair[1], qsum[r][g], part);
          }
          s[r][4 * u + i] = (PACKED ? columns_sum<G>(part) : part) * scale;
        }
    }
    bool seen[RT][8];
    if (masked.value) {
#pragma unroll
      for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int key = key0 + 16 * (j / 4) + 4 * h + j % 4;
          seen[r][j] = t.known[j / 4] && key >= row_lo[r] && key < row_hi[r];
          s[r][j] = seen[r][j] ? s[r][j] : -inf;
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
        for (int g = 0; g < SG; ++g)
          low[r][g] *= less;
#pragma unroll
        for (int g = 0; g < 2 * G; ++g)
          o[r][g] *= less;
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

    // output: scaled weights, then their products
    v8bf ps[RT][SG][TP];
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
      for (int g = 0; g < SG; ++g) {
        float x[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const v2h pair = halves(t.vs[j / 4][j % 4][g]);
          float vscale = (float)pair[0], vlow = (float)pair[1];
          if (masked.value) { // nothing of a key that is not seen
            vscale = seen[r][j] ? vscale : 0.0f;
            vlow = seen[r][j] ? vlow : 0.0f;
          }
          x[j] = s[r][j] * vscale;
          low[r][g] = __builtin_fmaf(s[r][j], vlow, low[r][g]);
        }
        terms_of<TP>(x, ps[r][g]);
      }
    unsigned codes[2][G];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const unsigned *const w[4] = {t.v[u][0], t.v[u][1], t.v[u][2], t.v[u][3]};
      bytes_of<G, 0, (G + 3) / 4>(w, codes[u]);
    }
#pragma unroll
    for (int g = 0; g < G; ++g) {
      v2bf n0, n1, n2, n3, n4, n5, n6, n7;
      numbers(codes[0][g] & 0x0F0F0F0Fu, n0, n1);
      numbers(codes[1][g] & 0x0F0F0F0Fu, n2, n3);
      numbers(codes[0][g] >> 4 & 0x0F0F0F0Fu, n4, n5);
      numbers(codes[1][g] >> 4 & 0x0F0F0F0Fu, n6, n7);
      const v8bf even = join(n0, n1, n2, n3), odd = join(n4, n5, n6, n7);
#pragma unroll
      for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int e = TP - 1; e >= 0; --e) {
          const v8bf w = ps[r][PACKED ? 0 : g][e];
          o[r][2 * g] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(even, w, o[r][2 * g], 0, 0, 0);
          o[r][2 * g + 1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(odd, w, o[r][2 * g + 1], 0, 0, 0);
        }
    }
  };

  auto step = [&](const Tile &t, int j) {
    const int key0 = (tile + kWaves * j) * 32;
    if (key0 >= all_lo && key0 + 32 <= all_hi && t.known[0] && t.known[1])
      step_on(t, key0, std::false_type{});
    else
      step_on(t, key0, std::true_type{});
  };

  // The next tile is on its way while one is worked on; 16 rows a tile leave no
  // registers for that (their scales alone are 16 G of them).
  if (tiles > 0)
    find_places(0);
  if constexpr (PACKED) {
    Tile one, other;
    if (tiles > 0)
      load(one, 0);
    for (int j = 0; j < tiles; j += 2) {
      load(other, j + 1 < tiles ? j + 1 : j);
      step(one, j);
      if (j + 1 < tiles) {
        load(one, j + 2 < tiles ? j + 2 : j + 1);
        step(other, j + 1);
      }
    }
  } else {
    for (int j = 0; j < tiles; ++j) {
      Tile one;
      load(one, j);
      step(one, j);
    }
  }

  // The waves' results meet in LDS: [wave][g][h][row][8] output, then (max, sum).
  constexpr int kPiece = 4 * ROWS * 8;
  float *const stats = shared + kWaves * G * kPiece;
#pragma unroll
  for (int r = 0; r < RT; ++r) {
    float all = sum[r];
    all += __shfl_xor(all, 16);
    all += __shfl_xor(all, 32);
#pragma unroll
    for (int g = 0; g < G; ++g) {
      float l = low[r][PACKED ? 0 : g];
      l += __shfl_xor(l, 16);
      l += __shfl_xor(l, 32);
      if (!PACKED || g == my_group) {
        float *const to = shared + (wave * G + g) * kPiece + (h * ROWS + my_row) * 8;
        const v4f e = o[r][2 * g] + l, f = o[r][2 * g + 1] + l;
        *(v4f *)to = v4f{e[0], f[0], e[1], f[1]};
        *(v4f *)(to + 4) = v4f{e[2], f[2], e[3], f[3]};
      }
    }
    if (lane < ROWS) {
      stats[(wave * ROWS + lane) * 2] = top[r];
      stats[(wave * ROWS + lane) * 2 + 1] = all;
    }
    __syncthreads();
    // Pieces of 8 elements: (g, quarter, row).
    for (int at = threadIdx.x; at < G * 4 * ROWS; at += kWaves * 64) {
      const int mr = at % ROWS, g = at / (4 * ROWS), quarter = at / ROWS % 4;
      const int row = row0 + ROWS * r + mr;
      if (row >= rows)
        continue;
      float m = -inf, total = 0.0f, v[8];
#pragma unroll
      for (int j = 0; j < 8; ++j)
        v[j] = 0.0f;
#pragma unroll
      for (int w = 0; w < kWaves; ++w)
        m = __builtin_fmaxf(m, stats[(w * ROWS + mr) * 2]);
#pragma unroll
      for (int w = 0; w < kWaves; ++w) {
        const float mw = stats[(w * ROWS + mr) * 2];
        const float f = mw == -inf ? 0.0f : __builtin_amdgcn_exp2f(mw - m);
        total += stats[(w * ROWS + mr) * 2 + 1] * f;
        const float *const from = shared + w * G * kPiece + at * 8;
#pragma unroll
        for (int j = 0; j < 8; ++j)
          v[j] = __builtin_fmaf(from[j], f, v[j]);
      }
      if (p.splits == 1) {
        const int i = row / p.per_head, qh = head * p.per_head + row % p.per_head;
        const int64_t to = p.heads_first ? ((int64_t)b * p.heads + qh) * p.S + i
                                         : ((int64_t)b * p.S + i) * p.heads + qh;
        const float over = total == 0.0f ? 0.0f : 1.0f / total;
        Pack<T, 8> out;
#pragma unroll
        for (int j = 0; j < 8; ++j)
          out.v[j] = from_f32<T>(v[j] * over);
        *(Pack<T, 8> *)((T *)p.y + to * D + 32 * g + 8 * quarter) = out;
      } else {
        const int64_t part = ((int64_t)unit * p.splits + split) * (RT * ROWS) + ROWS * r + mr;
        float *const y = p.parts + part * D + 32 * g + 8 * quarter;
        *(v4f *)y = v4f{v[0], v[1], v[2], v[3]};
        *(v4f *)(y + 4) = v4f{v[4], v[5], v[6], v[7]};
        if (g == 0 && quarter == 0) {
          float *const st = p.parts +
              (int64_t)p.B * p.c.H * p.groups * p.splits * (RT * ROWS) * D + part * 2;
          st[0] = m;
          st[1] = total;
        }
      }
    }
    __syncthreads();
  }
}

// ---------------------------------------------------------------------------
// attention of many rows
// ---------------------------------------------------------------------------
// Where a head of keys has many rows, what bounds the kernel above is scaling and
// splitting weights anew in every wave.  Here a block of 128 rows makes 64 keys and
// values at a time into f16 in LDS, s c + m with one rounding (2^-11; what lies
// beyond 65504, up to which rows are stored, becomes that), and its waves multiply
// those by q, which f16 holds with each row's largest at 2^14 (what it drops of
// others is 2^-38 of it), and by p in f16 (2^-11 again), 2^7 times what it is
// relative to a maximum that is at most 8 powers of two behind: what f16 loses of p
// is below 2^-32 of the largest.  Sums, scores and statistics are f32.  Results in
// bf16, whose own rounding is 2^-8, are as near to the exact ones as the tiles'
// (0.0018 and 0.0017 of their magnitude); f16's, 2^-11, would be off by up to three
// times as much (0.0006 and 0.0002), so those and f32's stay with the tiles.
//
// A wave has 32 rows in two tiles: both operands that it reads from LDS, 1 KB each,
// feed two instructions, which is as fast as LDS can feed four waves.  Scores'
// layout is that of the second product's operand, as above.
//
// LDS: keys' fragments (u, f), u of four 16s, f of G: lane (c, h) has word f of the
// quarter h of key c's codes, 8 elements; values' (half, t): lane (c, h) has, of the
// keys 4 h .. of either 16, element 16 t + c in the order z (4 G) + j: byte z / 2 of
// word j, z % 2 its half.  All are read as they lie, 1024 bytes after one another.
//
// 2048 rows on 4096 keys, 32 heads on 8 of 128, causal: 140 us, 735 TFLOP/s (534 us in
// tiles); heads of 256, 16 on 4, 251 us: they spill 21 registers.  Bound by instructions: vector ones take 48 % of the clocks (of some 300 for 64
// keys a wave, 130 make its share of them and 32 are exponentials at a quarter of the
// rate), matrix ones 28 %, and the two blocks that a CU has registers for overlap little;
// blocks of unequal length leave it with one for the rest.
//
// A group of a value whose scale or lowest value is not finite must give NaN to rows
// that see its key and nothing to others: it is made into zeros, and marked.
typedef _Float16 v8h __attribute__((ext_vector_type(8)));
constexpr unsigned kUnknown = 1u << 31; // a key without a place in the cache
constexpr int kPromptRows = 128;

__device__ __forceinline__ v2h halves_of(unsigned w) { return __builtin_bit_cast(v2h, w); }
__device__ __forceinline__ unsigned low_halves(unsigned a, unsigned b) {
  return __builtin_amdgcn_perm(b, a, 0x05040100);
}
__device__ __forceinline__ unsigned high_halves(unsigned a, unsigned b) {
  return __builtin_amdgcn_perm(b, a, 0x07060302);
}
// Codes in bits 0 .. 3 (LOW) or 4 .. 7 of the halves of w, as f16: 1024 + code
// and 1024 + 16 code have the bits `ones` (0x6400) | code.  It comes in a register:
// an instruction takes one constant, and so `and` and `or` are one.
template <bool LOW> __device__ __forceinline__ v2h codes_of(unsigned w, unsigned ones) {
  if (LOW)
    return halves_of((w & 0x000F000Fu) | ones) - v2h{1024, 1024};
  return __builtin_elementwise_fma(halves_of((w & 0x00F000F0u) | ones),
      v2h{0.0625f16, 0.0625f16}, v2h{-64, -64});
}
__device__ __forceinline__ v2h within(v2h x) { // NaN stays
  const _Float16 top = 65504;
#pragma unroll
  for (int i = 0; i < 2; ++i)
    x[i] = x[i] > top ? top : x[i] < -top ? -top : x[i];
  return x;
}
__device__ __forceinline__ bool is_finite(_Float16 x) {
  return (__builtin_bit_cast(unsigned short, x) & 0x7C00) != 0x7C00;
}

template <int G>
__global__ __launch_bounds__(256, G <= 4 ? 2 : 1) void k_cache_prompt(const Arguments p) {
  typedef __bf16 T;
  constexpr int D = 32 * G, WORDS = 4 * G, ITEMS = (WORDS + 15) / 16;
  constexpr int SG = G < 4 ? G : 4; // groups of a word's bytes
  constexpr int PITCH = D + 4; // of a row of results in LDS
  extern __shared__ __attribute__((aligned(16))) float shared[];
  uint8_t *const keys = (uint8_t *)shared, *const values = keys + G * 4096;
  // [parity][key]: groups of its value that are not finite, and whether it is known
  unsigned *const marks = (unsigned *)(values + G * 4096);
  const int lane = threadIdx.x & 63, c = lane & 15, h = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const float inf = __builtin_inff();

  const int id = xcd_contiguous(blockIdx.x, (int)gridDim.x);
  const int split = (unsigned)id % (unsigned)p.splits;
  const int unit = (unsigned)id / (unsigned)p.splits;
  const int bh = (unsigned)unit / (unsigned)p.groups;
  int group = unit - bh * p.groups;
  const int b = (unsigned)bh / (unsigned)p.c.H, head = (unsigned)bh % (unsigned)p.c.H;
  // Those with the most keys first (2048 / 4096 / 4 x 2048 rows: 156 / 196 / 510 us, in
  // order of the keys 175 / 236 / 579).
  if (p.causal)
    group = p.groups - 1 - group;

  const int past = p.c.past[b];
  int count = p.S;
  if (p.c.counts) {
    const int n = p.c.counts[b];
    count = n < 0 ? 0 : n < p.S ? n : p.S;
  }
  const int rows = count * p.per_head, row0 = group * kPromptRows;
  if (row0 >= rows)
    return;
  const int last_row = (row0 + kPromptRows < rows ? row0 + kPromptRows : rows) - 1;
  const unsigned page_size = (unsigned)p.c.page_size;
  const int capacity = (int)(p.c.table ? p.c.table_pages * p.c.page_size : p.c.page_size);
  // Keys [first, end) of the query of token i.
  const int start = p.starts ? p.starts[b] : 0;
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
  int tile, tiles; // of 64 keys: this part's
  {
    const int lo = first_of(row0 / p.per_head), hi = end_of(last_row / p.per_head);
    tile = lo / 64;
    tiles = hi > lo ? (hi + 63) / 64 - tile : 0;
    const int each = (tiles + p.splits - 1) / p.splits;
    tile += split * each;
    tiles = tiles - split * each < each ? tiles - split * each : each;
  }
  // Keys that some, and that all of the wave's rows see.
  int lo = 0, hi = 0, all_lo = 0, all_hi = 0;
  if (row0 + 32 * wave < rows) {
    const int r1 = row0 + 32 * wave + 31;
    const int i0 = (row0 + 32 * wave) / p.per_head, i1 = (r1 < rows ? r1 : rows - 1) / p.per_head;
    lo = first_of(i0), hi = end_of(i1);
    all_lo = first_of(i1), all_hi = end_of(i0);
  }

  // This lane's rows: q in the order of a word's codes as they come out of it.
  const float scale =
      (p.scale ? finite_or_nan(p.scale[0]) : 1.0f / __builtin_sqrtf((float)D)) * kLog2E;
  v8h q[2][G];
  float by[2]; // a score's factor
  int row_lo[2], row_hi[2];
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    int row = row0 + 32 * wave + 16 * r + c;
    row = row < rows ? row : rows - 1;
    const int i = row / p.per_head, qh = head * p.per_head + row % p.per_head;
    row_lo[r] = first_of(i);
    row_hi[r] = end_of(i);
    const int64_t at = p.heads_first ? ((int64_t)b * p.heads + qh) * p.S + i
                                     : ((int64_t)b * p.S + i) * p.heads + qh;
    const T *const x = (const T *)p.q + at * D;
    Pack<T, 2> pairs[G][4];
    float most = 0.0f;
#pragma unroll
    for (int f = 0; f < G; ++f)
#pragma unroll
      for (int y = 0; y < 4; ++y) {
        const int byte = WORDS * h + 4 * f + y;
        pairs[f][y] = *(const Pack<T, 2> *)(x + 32 * (byte % G) + 2 * (byte / G));
        most = __builtin_fmaxf(most, __builtin_fmaxf(__builtin_fabsf(to_f32(pairs[f][y].v[0])),
                                         __builtin_fabsf(to_f32(pairs[f][y].v[1]))));
      }
    most = __builtin_fmaxf(most, __shfl_xor(most, 16));
    most = __builtin_fmaxf(most, __shfl_xor(most, 32));
    const int up = 14 + 127 - (int)(__builtin_bit_cast(unsigned, most) >> 23);
    // (not 0: what is not seen has the score -inf)
    by[r] = __builtin_fmaxf(__builtin_ldexpf(__builtin_fabsf(scale), -up), 0x1p-126f);
    const float sign = most == inf ? __builtin_nanf("") : scale < 0.0f ? -1.0f : 1.0f;
#pragma unroll
    for (int f = 0; f < G; ++f) {
      constexpr int order[4] = {0, 2, 1, 3};
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float v = to_f32(pairs[f][order[e % 4]].v[e / 4]);
        q[r][f][e] = (_Float16)__builtin_ldexpf(v * sign, up);
      }
    }
  }

  v4f o[2][2 * G];
  float top[2], sum[2];
  unsigned nan[2] = {0, 0}; // groups of the result that are NaN
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    top[r] = -inf;
    sum[r] = 0.0f;
#pragma unroll
    for (int t = 0; t < 2 * G; ++t)
      o[r][t] = v4f{0, 0, 0, 0};
  }

  // The wave makes 16 of a tile's keys, those from 16 wave on; lane l knows where
  // those of the tile `known_from` + l lie, as the cache's row of the first.
  constexpr unsigned kNowhere = ~0u;
  unsigned place = kNowhere;
  int known_from = 0;
  auto find_places = [&](int from) {
    known_from = from;
    const unsigned key = (unsigned)(tile + from + lane) * 64 + 16 * wave;
    place = kNowhere;
    if (key < (unsigned)capacity) {
      unsigned page = (unsigned)b, slot = key;
      if (p.c.table) {
        const unsigned at = key / page_size;
        page = (unsigned)p.c.table[b * p.c.table_pages + at];
        slot = key - at * page_size;
      }
      if (page < (uint64_t)p.c.pages)
        place = (page * (unsigned)p.c.H + (unsigned)head) * page_size + slot;
    }
  };
  // What a lane makes: the quarter h of key c, and of the keys 4 h + i the words
  // c + 16 e.
  struct Raw {
    unsigned k[G], kp[G], v[4][ITEMS], vp[4][SG];
    bool known;
  } raw;
  auto load = [&](int j) {
    if (j - known_from >= 64)
      find_places(j);
    const unsigned found = __builtin_amdgcn_readlane(place, j - known_from);
    raw.known = found != kNowhere;
    const int64_t row = raw.known ? found : 0;
    int room = capacity - ((tile + j) * 64 + 16 * wave);
    room = !raw.known ? 0 : room < 16 ? room : 16; // (whole pages hold all 16)
    auto part = [&](const void *base, int row_bytes) {
      return __builtin_amdgcn_make_buffer_rsrc(
          (void *)((const char *)base + row * row_bytes), 0, room * row_bytes, 0x00020000);
    };
    const auto kc = part(p.c.k_codes, 16 * G), vc = part(p.c.v_codes, 16 * G);
    const auto kp = part(p.c.k_scales, 4 * G), vp = part(p.c.v_scales, 4 * G);
    load_words<G>(kc, c * (16 * G) + h * (4 * G), raw.k);
    load_words<G>(kp, c * (4 * G), raw.kp);
    const int word = WORDS < 16 ? c % WORDS : c;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
#pragma unroll
      for (int e = 0; e < ITEMS; ++e)
        load_words<1>(vc, (4 * h + i) * (16 * G) + 4 * (word + 16 * e), *(unsigned(*)[1])&raw.v[i][e]);
      load_words<SG>(vp, (4 * h + i) * (4 * G) + (4 * word) % G * 4, raw.vp[i]);
    }
  };

  unsigned ones = 0x64006400u;
  asm("" : "+v"(ones));
  // careful: some scale or lowest value is not finite, or what they give too large.
  auto make_keys = [&](auto careful) {
    v2h s[G], m[G]; // of the groups of bytes x, x + 2
#pragma unroll
    for (int x = 0; x < G; ++x) {
      const unsigned one = raw.kp[x], other = raw.kp[(x + 2) % G];
      s[x] = halves_of(low_halves(one, other)), m[x] = halves_of(high_halves(one, other));
    }
#pragma unroll
    for (int f = 0; f < G; ++f) {
      const unsigned w = raw.k[f];
      const int x = 4 * f % G, x1 = (4 * f + 1) % G;
      v2h v[4] = {__builtin_elementwise_fma(codes_of<true>(w, ones), s[x], m[x]),
          __builtin_elementwise_fma(codes_of<true>(w >> 8, ones), s[x1], m[x1]),
          __builtin_elementwise_fma(codes_of<false>(w, ones), s[x], m[x]),
          __builtin_elementwise_fma(codes_of<false>(w >> 8, ones), s[x1], m[x1])};
      if (careful.value) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          v[i] = within(v[i]);
          const int g = i % 2 ? x1 : x;
#pragma unroll
          for (int e = 0; e < 2; ++e)
            if (!is_finite(s[g][e]) || !is_finite(m[g][e]))
              v[i][e] = (_Float16)__builtin_nanf("");
        }
      }
      *(v8h *)(keys + ((wave * G + f) * 64 + lane) * 16) =
          v8h{v[0][0], v[0][1], v[1][0], v[1][1], v[2][0], v[2][1], v[3][0], v[3][1]};
    }
  };
  auto make_values = [&](auto careful, unsigned *marked) {
    v2h s[2][SG], m[2][SG]; // of keys 4 h + 2 i and the next
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int g = 0; g < SG; ++g) {
        const unsigned one = raw.vp[2 * i][g], other = raw.vp[2 * i + 1][g];
        s[i][g] = halves_of(low_halves(one, other)), m[i][g] = halves_of(high_halves(one, other));
        if (careful.value) {
#pragma unroll
          for (int e = 0; e < 2; ++e)
            if (!is_finite(s[i][g][e]) || !is_finite(m[i][g][e])) {
              s[i][g][e] = m[i][g][e] = 0;
              const int all = G > 4 ? 4 * c % G + g : g;
              atomicOr(marked + 16 * wave + 4 * h + 2 * i + e, 1u << all);
            }
        }
      }
#pragma unroll
    for (int e = 0; e < ITEMS; ++e) {
      v2h v[8][2]; // [z][keys]
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const unsigned one = raw.v[2 * i][e], other = raw.v[2 * i + 1][e];
        const unsigned w[2] = {low_halves(one, other), high_halves(one, other)};
#pragma unroll
        for (int y = 0; y < 4; ++y) {
          const unsigned at = w[y / 2] >> (8 * (y % 2));
          v[2 * y][i] = __builtin_elementwise_fma(codes_of<true>(at, ones), s[i][y % SG], m[i][y % SG]);
          v[2 * y + 1][i] = __builtin_elementwise_fma(codes_of<false>(at, ones), s[i][y % SG], m[i][y % SG]);
          if (careful.value)
            v[2 * y][i] = within(v[2 * y][i]), v[2 * y + 1][i] = within(v[2 * y + 1][i]);
        }
      }
      if (WORDS < 16 && c >= WORDS)
        continue;
#pragma unroll
      for (int z = 0; z < 8; ++z) {
        const int element = z * WORDS + c + 16 * e;
        uint8_t *const to = values +
            (((wave / 2) * (2 * G) + element / 16) * 64 + h * 16 + element % 16) * 16 + wave % 2 * 8;
        typedef _Float16 v4h __attribute__((ext_vector_type(4)));
        *(v4h *)to = v4h{v[z][0][0], v[z][0][1], v[z][1][0], v[z][1][1]};
      }
    }
  };
  auto make = [&](int parity) {
    // (a code is at most 15: if 15 s + m is finite, so is what lies between)
    v2h worst = {0, 0};
    auto look = [&](unsigned one, unsigned other) {
      const v2h s = halves_of(low_halves(one, other)), m = halves_of(high_halves(one, other));
      worst = __builtin_elementwise_fma(
          __builtin_elementwise_fma(s, v2h{15, 15}, m), v2h{0, 0}, worst);
    };
#pragma unroll
    for (int g = 0; g < G; g += 2)
      look(raw.kp[g], raw.kp[g + 1]);
    const bool k_careful = !(worst[0] == 0) || !(worst[1] == 0);
    worst = v2h{0, 0};
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int g = 0; g < SG; ++g)
        look(raw.vp[2 * i][g], raw.vp[2 * i + 1][g]);
    const bool v_careful = !(worst[0] == 0) || !(worst[1] == 0);
    unsigned *const marked = marks + 64 * parity;
    if (!raw.known && lane < 16)
      atomicOr(marked + 16 * wave + lane, kUnknown);
    if (__any(k_careful))
      make_keys(std::true_type{});
    else
      make_keys(std::false_type{});
    if (__any(v_careful))
      make_values(std::true_type{}, marked);
    else
      make_values(std::false_type{}, marked);
  };

  // masked: some rows do not see some of the keys, or some are marked.
  auto work = [&](int key0, int parity, bool masked) {
    v4f s[2][4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
#pragma unroll
      for (int r = 0; r < 2; ++r)
        s[r][u] = v4f{0, 0, 0, 0};
#pragma unroll
      for (int f = 0; f < G; ++f) {
        const v8h k = *(const v8h *)(keys + ((u * G + f) * 64 + lane) * 16);
#pragma unroll
        for (int r = 0; r < 2; ++r)
          s[r][u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k, q[r][f], s[r][u], 0, 0, 0);
      }
    }
    // Four fragments on their way (512 rows of 4 heads 50 us, 256 elements 141; with two,
    // as they would be, 53 and 153).
    __builtin_amdgcn_sched_group_barrier(0x100, 4, 0); // LDS reads
#pragma unroll
    for (int i = 0; i < 4 * G; ++i) {
      __builtin_amdgcn_sched_group_barrier(0x008, 2, 0); // matrix instructions
      __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
    }
    if (masked) {
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const v4u mark = *(const v4u *)(marks + 64 * parity + 16 * u + 4 * h);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int key = key0 + 16 * u + 4 * h + i;
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            const bool sees = !(mark[i] & kUnknown) && key >= row_lo[r] && key < row_hi[r];
            nan[r] |= sees ? mark[i] : 0u;
            s[r][u][i] = sees ? s[r][u][i] : -inf;
          }
        }
      }
    }
    // maxima, as above
    float most[2];
    bool grown = false;
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      float m = s[r][0][0];
#pragma unroll
      for (int j = 1; j < 16; ++j)
        m = __builtin_fmaxf(m, s[r][j / 4][j % 4]);
      most[r] = m * by[r];
      grown = grown || most[r] > top[r] + 8.0f;
    }
    if (__any(grown)) {
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        float m = __builtin_fmaxf(most[r], __shfl_xor(most[r], 16));
        m = __builtin_fmaxf(m, __shfl_xor(m, 32));
        m = __builtin_fmaxf(m, top[r]);
        const float less = m == top[r] ? 1.0f : __builtin_amdgcn_exp2f(top[r] - m);
        top[r] = m;
        sum[r] *= less;
#pragma unroll
        for (int t = 0; t < 2 * G; ++t)
          o[r][t] *= less;
      }
    }
    v8h weights[2][2];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const float base = top[r] == -inf ? 0.0f : 7.0f - top[r]; // -inf: no key seen so far
#pragma unroll
      for (int j = 0; j < 16; j += 2) {
        float e[2];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const int at = j + k;
          e[k] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[r][at / 4][at % 4], by[r], base));
          sum[r] += e[k];
        }
        typedef float v2f __attribute__((ext_vector_type(2)));
        const v2h w = __builtin_convertvector(v2f{e[0], e[1]}, v2h);
        weights[r][j / 8][j % 8] = w[0], weights[r][j / 8][j % 8 + 1] = w[1];
      }
    }
#pragma unroll
    for (int half = 0; half < 2; ++half)
#pragma unroll
      for (int t = 0; t < 2 * G; ++t) {
        const v8h v = *(const v8h *)(values + ((half * (2 * G) + t) * 64 + lane) * 16);
#pragma unroll
        for (int r = 0; r < 2; ++r)
          o[r][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, weights[r][half], o[r][t], 0, 0, 0);
      }
  };

  if (threadIdx.x < 128)
    marks[threadIdx.x] = 0;
  if (tiles > 0) {
    find_places(0);
    load(0);
  }
  for (int j = 0; j < tiles; ++j) {
    const int parity = j & 1, key0 = (tile + j) * 64;
    gemm::lds_barrier(); // the last tile has been read
    make(parity);
    if (j + 1 < tiles)
      load(j + 1);
    gemm::lds_barrier();
    // (the other marks were read before the last barrier but one)
    if (threadIdx.x < 64)
      marks[64 * (1 - parity) + threadIdx.x] = 0;
    if (key0 >= hi || key0 + 64 <= lo)
      continue;
    work(key0, parity, key0 < all_lo || key0 + 64 > all_hi ||
                           __any(marks[64 * parity + lane] != 0));
  }

#pragma unroll
  for (int r = 0; r < 2; ++r) {
    sum[r] += __shfl_xor(sum[r], 16);
    sum[r] += __shfl_xor(sum[r], 32);
    nan[r] |= __shfl_xor(nan[r], 16);
    nan[r] |= __shfl_xor(nan[r], 32);
    if (scale != scale && sum[r] > 0.0f) // (rows that see nothing stay 0)
      nan[r] = ~0u;
  }
  // Element 4 h + i of tile t is z (4 G) + j.
  auto element_of = [&](int t, int i, int &g) {
    const int element = 16 * t + 4 * h + i, z = element / WORDS, j = element % WORDS;
    const int byte = 4 * j + z / 2;
    g = byte % G;
    return 32 * g + 2 * (byte / G) + z % 2;
  };
  // Results leave by way of LDS, so that a store takes whole pieces of rows.
  float *const mine = shared + wave * (16 * PITCH);
  const int64_t part0 = (((int64_t)bh * p.groups + group) * p.splits + split) * kPromptRows;
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const float over = p.splits > 1 ? 1.0f : sum[r] == 0.0f ? 0.0f : 1.0f / sum[r];
    gemm::lds_barrier();
#pragma unroll
    for (int t = 0; t < 2 * G; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        int g;
        const int d = element_of(t, i, g);
        mine[c * PITCH + d] = nan[r] >> g & 1 ? __builtin_nanf("") : o[r][t][i] * over;
      }
    gemm::lds_barrier();
    const int first = 32 * wave + 16 * r;
#pragma unroll 2
    for (int at = lane; at < 16 * (D / 8); at += 64) {
      const int mr = at / (D / 8), d = at % (D / 8) * 8, row = row0 + first + mr;
      if (row >= rows)
        break;
      const v4f x = *(const v4f *)(mine + mr * PITCH + d),
                y = *(const v4f *)(mine + mr * PITCH + d + 4);
      if (p.splits > 1) {
        float *const to = p.parts + (part0 + first + mr) * D + d;
        *(v4f *)to = x;
        *(v4f *)(to + 4) = y;
        continue;
      }
      const int i = row / p.per_head, qh = head * p.per_head + row % p.per_head;
      const int64_t to = p.heads_first ? ((int64_t)b * p.heads + qh) * p.S + i
                                       : ((int64_t)b * p.S + i) * p.heads + qh;
      Pack<T, 8> out;
#pragma unroll
      for (int j = 0; j < 4; ++j)
        out.v[j] = from_f32<T>(x[j]), out.v[4 + j] = from_f32<T>(y[j]);
      *(Pack<T, 8> *)((T *)p.y + to * D + d) = out;
    }
    if (p.splits > 1 && h == 0 && row0 + first + c < rows) {
      float *const st = p.parts +
          (int64_t)p.B * p.c.H * p.groups * p.splits * kPromptRows * D +
          (part0 + first + c) * 2;
      st[0] = top[r];
      st[1] = sum[r];
    }
  }
}

// The parts of a row's keys joined, a block a row: thread t weighs part t (there
// are at most 256), then thread (s, d) sums elements 4 d .. of every part s, s +
// across, .., and those sums meet in LDS.
template <typename T>
__global__ __launch_bounds__(256) void k_cache_join(const Arguments p, int D, int tile_rows) {
  __shared__ float weight[256], tops[4], sums[4];
  __shared__ __attribute__((aligned(16))) float pieces[256 * 4];
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
  const int t = threadIdx.x;
  const int lanes = D / 4, across = 256 / lanes; // threads of a row, parts at once
  const float inf = __builtin_inff();
  const float *const stats = p.parts + (int64_t)p.B * p.c.H * p.groups * p.splits * tile_rows * D;
  const int64_t part0 = (int64_t)unit * p.splits * tile_rows + r;
  float m = -inf, total = 0.0f;
  if (t < p.splits) {
    m = stats[(part0 + (int64_t)t * tile_rows) * 2];
    total = stats[(part0 + (int64_t)t * tile_rows) * 2 + 1];
  }
  auto over_block = [&](float v, float (&of)[4], auto fold) {
#pragma unroll
    for (int i = 1; i < 64; i *= 2)
      v = fold(v, __shfl_xor(v, i));
    if (t % 64 == 0)
      of[t / 64] = v;
    __syncthreads();
    return fold(fold(of[0], of[1]), fold(of[2], of[3]));
  };
  const float top = over_block(m, tops, [](float x, float y) { return __builtin_fmaxf(x, y); });
  const float f = m == -inf ? 0.0f : __builtin_amdgcn_exp2f(m - top);
  weight[t] = f;
  total = over_block(total * f, sums, [](float x, float y) { return x + y; });
  const int s0 = t / lanes, d = t % lanes;
  v4f v = {0, 0, 0, 0};
  if (s0 < across) {
#pragma unroll 4
    for (int s = s0; s < p.splits; s += across)
      v += *(const v4f *)(p.parts + (part0 + (int64_t)s * tile_rows) * D + 4 * d) * weight[s];
  }
  *(v4f *)(pieces + 4 * t) = v;
  __syncthreads();
  if (s0 > 0)
    return;
  for (int s = 1; s < across; ++s)
    v += *(const v4f *)(pieces + 4 * (s * lanes + d));
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

// The same where parts are few and rows many: 256 / (D / 4) rows a block, a thread
// weighs all parts of its row and sums four elements of them.
template <typename T>
__global__ __launch_bounds__(256) void k_cache_join_rows(const Arguments p, int D, int tile_rows) {
  const int lanes = D / 4;
  const int64_t units = (int64_t)p.B * p.c.H * p.groups;
  const int64_t id = (int64_t)blockIdx.x * (256 / lanes) + threadIdx.x / lanes;
  const int unit = (int)(id / tile_rows), r = (int)(id % tile_rows), d = threadIdx.x % lanes;
  if ((int)threadIdx.x >= 256 / lanes * lanes || unit >= units)
    return;
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
  const float *const stats = p.parts + units * p.splits * tile_rows * D;
  const int64_t part0 = (int64_t)unit * p.splits * tile_rows + r;
  const float inf = __builtin_inff();
  float top = -inf, total = 0.0f;
  v4f v = {0, 0, 0, 0};
#pragma unroll 4
  for (int s = 0; s < p.splits; ++s)
    top = __builtin_fmaxf(top, stats[(part0 + (int64_t)s * tile_rows) * 2]);
#pragma unroll 4
  for (int s = 0; s < p.splits; ++s) {
    const int64_t part = part0 + (int64_t)s * tile_rows;
    const float m = stats[part * 2];
    const float f = m == -inf ? 0.0f : __builtin_amdgcn_exp2f(m - top);
    total += stats[part * 2 + 1] * f;
    v += *(const v4f *)(p.parts + part * D + 4 * d) * f;
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

// A block a row / threads a row: 16384 rows of 128 in 8 parts 70 / 53 us with the
// attention itself, 32768 of 64 in 2 parts 87 / 49; 128 rows in 16 parts 21 / 23, 32
// in 64 parts 41 / 51.
template <typename T>
hipError_t join_parts(hipStream_t st, const Arguments &p, int D, int tile_rows) {
  const int64_t rows = (int64_t)p.B * p.c.H * p.groups * tile_rows;
  if (p.splits <= 8) {
    const int each = 256 / (D / 4);
    k_cache_join_rows<T><<<dim3((unsigned)((rows + each - 1) / each)), 256, 0, st>>>(p, D, tile_rows);
  } else {
    k_cache_join<T><<<dim3((unsigned)rows), 256, 0, st>>>(p, D, tile_rows);
  }
  return hipGetLastError();
}

// How rows are dealt: tiles of 16 a wave, or of 16 / G where that takes one tile
// (D = 64, 128, 256) or two (64, 128); or bf16's 128 rows a block, once there are
// as many (128 rows a head, tiles / blocks: 4096 keys 31 / 27 us, 1100 keys 39 / 33;
// 2048 rows a head and 2500 keys 104 / 74).
struct Shape {
  enum { kTiles, kPacked, kPrompt } form;
  int tiles, rows; // tiles of a unit of blocks; rows of a tile
};
Shape shape_of(const Attention4 &a) {
  const int64_t n = a.S * (a.heads / a.c.H);
  const int G = a.c.D / kCacheGroup;
  if (16 % G == 0 && n <= (G <= 4 ? 2 : 1) * (16 / G))
    return {Shape::kPacked, n > 16 / G ? 2 : 1, 16 / G};
  if (a.kind == kBF16 && 16 % G == 0 && n >= kPromptRows)
    return {Shape::kPrompt, kPromptRows / 16, 16};
  return {Shape::kTiles, n > 16 && G <= 4 ? 2 : 1, 16};
}
int64_t row_groups(const Attention4 &a) {
  const Shape s = shape_of(a);
  const int rows = s.rows * s.tiles;
  return (a.S * (a.heads / a.c.H) + rows - 1) / rows;
}

template <typename T, int G, int RT, bool PACKED>
hipError_t attend(hipStream_t st, const Arguments &p) {
  constexpr int kRows = PACKED ? 16 / G : 16;
  constexpr int kLds = (kWaves * G * 4 * kRows * 8 + kWaves * kRows * 2) * 4;
  auto *const kernel = k_cache_attention<T, G, RT, PACKED>;
  if (kLds > 65536) {
    const hipError_t e = hipFuncSetAttribute((const void *)kernel,
        hipFuncAttributeMaxDynamicSharedMemorySize, kLds);
    if (e != hipSuccess)
      return e;
  }
  const int64_t units = (int64_t)p.B * p.c.H * p.groups;
  kernel<<<dim3((unsigned)(units * p.splits)), kWaves * 64, kLds, st>>>(p);
  hipError_t e = hipGetLastError();
  if (e == hipSuccess && p.splits > 1)
    e = join_parts<T>(st, p, 32 * G, RT * kRows);
  return e;
}

template <int G> hipError_t attend_prompt(hipStream_t st, const Arguments &p) {
  // (keys, values and marks; then 16 rows a wave of 128 G + 16 bytes)
  constexpr int kLds = 8192 * G + 1024;
  auto *const kernel = k_cache_prompt<G>;
  if (kLds > 65536) {
    const hipError_t e = hipFuncSetAttribute((const void *)kernel,
        hipFuncAttributeMaxDynamicSharedMemorySize, kLds);
    if (e != hipSuccess)
      return e;
  }
  const int64_t units = (int64_t)p.B * p.c.H * p.groups;
  kernel<<<dim3((unsigned)(units * p.splits)), 256, kLds, st>>>(p);
  hipError_t e = hipGetLastError();
  if (e == hipSuccess && p.splits > 1)
    e = join_parts<__bf16>(st, p, 32 * G, kPromptRows);
  return e;
}

template <typename T, int G>
hipError_t attend_group(hipStream_t st, const Arguments &p, const Shape &s) {
  if constexpr (16 % G == 0 && std::is_same<T, __bf16>::value) {
    if (s.form == Shape::kPrompt)
      return attend_prompt<G>(st, p);
  }
  if constexpr (16 % G == 0) {
    if (s.form == Shape::kPacked && s.tiles == 1)
      return attend<T, G, 1, true>(st, p);
  }
  if constexpr (G <= 4) {
    if constexpr (16 % G == 0) {
      if (s.form == Shape::kPacked)
        return attend<T, G, 2, true>(st, p);
    }
    if (s.tiles > 1)
      return attend<T, G, 2, false>(st, p);
  }
  return attend<T, G, 1, false>(st, p);
}

template <typename T>
hipError_t attend_any(hipStream_t st, const Arguments &p, const Shape &s) {
  switch (p.c.D / kCacheGroup) {
  case 2:
    return attend_group<T, 2>(st, p, s);
  case 3:
    return attend_group<T, 3>(st, p, s);
  case 4:
    return attend_group<T, 4>(st, p, s);
  case 6:
    return attend_group<T, 6>(st, p, s);
  default:
    return attend_group<T, 8>(st, p, s);
  }
}

template <typename T, int G>
hipError_t append_group(hipStream_t st, const Append4 &a) {
  const int64_t rows = 2 * a.B * a.S * a.c.H;
  for (int64_t first = 0; first < rows; first += kMostGrid * 16) {
    const int64_t blocks = (rows - first + 15) / 16;
    const dim3 grid((unsigned)(blocks < kMostGrid ? blocks : kMostGrid));
    k_cache_append<T, G><<<grid, 256, 0, st>>>(a, first);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess)
      return e;
  }
  return hipSuccess;
}

template <typename T>
hipError_t append_any(hipStream_t st, const Append4 &a) {
  switch (a.c.D / kCacheGroup) {
  case 2:
    return append_group<T, 2>(st, a);
  case 3:
    return append_group<T, 3>(st, a);
  case 4:
    return append_group<T, 4>(st, a);
  case 6:
    return append_group<T, 6>(st, a);
  default:
    return append_group<T, 8>(st, a);
  }
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

// Parts of the keys, so that a few rows fill the GPU: two blocks a CU, which is
// what its registers hold (one of many rows of 256), of 128 keys at least, or 256 for
// many rows (4 x 8 heads of 128 rows, 1100 keys, 128 / 256: 33 / 26 us).  (How many keys there are, only
// the GPU knows: a block takes its share of what its rows see.)  131072 keys, 8
// heads of 128, in parts for 256 / 512 / 768 / 1024 / 2048 blocks: 42 / 44 / 48 /
// 53 / 64 us; 32 sequences of 2000 - 4000 keys 38 / 37 / 43 / 44 / 58.
int attention_splits(const Attention4 &a) {
  const int64_t units = a.B * a.c.H * row_groups(a);
  const int64_t capacity = a.c.table ? a.c.table_pages * a.c.page_size : a.c.page_size;
  const bool prompt = shape_of(a).form == Shape::kPrompt;
  const int64_t least = prompt ? 256 : 128; // keys of a part
  int64_t n = (prompt && a.c.D > 128 ? 256 : 512) / (units > 0 ? units : 1);
  if (n > (capacity + least - 1) / least)
    n = (capacity + least - 1) / least;
  return (int)(n < 1 ? 1 : n < 256 ? n : 256);
}
size_t attention_parts_bytes(const Attention4 &a) {
  const Shape shape = shape_of(a);
  const int64_t rows = a.B * a.c.H * row_groups(a) * shape.rows * shape.tiles;
  return (size_t)rows * a.splits * (a.c.D + 2) * sizeof(float);
}

hipError_t launch_cache_attention(hipStream_t s, const Attention4 &a) {
  Arguments p = {a.c, a.q, a.y, a.starts, a.scale, a.parts, a.window, (int)a.B,
      (int)a.S, (int)a.heads, (int)(a.heads / a.c.H), (int)row_groups(a), a.splits,
      a.causal, a.heads_first};
  switch (a.kind) {
  case kF32:
    return attend_any<float>(s, p, shape_of(a));
  case kF16:
    return attend_any<_Float16>(s, p, shape_of(a));
  default:
    return attend_any<__bf16>(s, p, shape_of(a));
  }
}

} // namespace om
