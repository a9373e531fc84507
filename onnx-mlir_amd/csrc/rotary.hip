// Rotary positions (onnx.RotaryEmbedding).  Pair i of a head, elements (a, b),
// turns by the angle whose cosine and sine the tables hold for the token's
// position:
//     a' = a cos - b sin,   b' = b cos + a sin
// with (a, b) = elements (i, i + rot / 2), or (2 i, 2 i + 1) interleaved;
// elements from `rot` on pass through.
//
// Bound by memory: every element is read and written once, in 16-byte pieces,
// and the tables of a token, read by all its heads, come from the caches.  A
// thread owns both elements of its pairs, so y may be x.

#include "llm_common.h"

namespace om {
namespace llm {
namespace {

struct RotaryArgs {
  const void *x;
  void *y;
  const float *cos, *sin;
  const int64_t *positions;
  int64_t S, table_rows, rows; // rows: B * S * H
  int64_t first;               // row of a launch
  int H, D, half;              // half: rot / 2
  int units;                   // threads a row takes
  bool heads_first;
};

// A thread takes V pairs (V = 1 where rows or halves do not divide into
// aligned pieces), or 2 V elements that pass through.
template <typename T, int V, bool INTERLEAVED>
__global__ __launch_bounds__(256) void k_rotary(const RotaryArgs p) {
  const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
  int64_t row = id / p.units;
  const int u = (int)(id - row * p.units);
  row += p.first;
  if (row >= p.rows)
    return;
  int64_t token; // b * S + s
  if (p.heads_first) {
    const int64_t bh = row / p.S;
    token = bh / p.H * p.S + (row - bh * p.S);
  } else {
    token = row / p.H;
  }
  const T *const x = (const T *)p.x + row * p.D;
  T *const y = (T *)p.y + row * p.D;
  const int pair = u * V;
  if (pair >= p.half) { // behind the rotated part
    const int at = 2 * p.half + (pair - p.half) * 2;
    if (V > 1 || at + 2 <= p.D) {
      *(Pack<T, V> *)(y + at) = *(const Pack<T, V> *)(x + at);
      *(Pack<T, V> *)(y + at + V) = *(const Pack<T, V> *)(x + at + V);
    } else {
      y[at] = x[at]; // (an odd head: its last element)
    }
    return;
  }
  const int64_t at = p.positions ? p.positions[token] : token;
  const bool known = at >= 0 && at < p.table_rows;
  Pack<float, V> c, s;
  if (known) {
    c = *(const Pack<float, V> *)(p.cos + at * p.half + pair);
    s = *(const Pack<float, V> *)(p.sin + at * p.half + pair);
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i)
      c.v[i] = s.v[i] = __builtin_nanf("");
  }
  Pack<T, V> a, b;
  if (INTERLEAVED) {
    const Pack<T, V> lo = *(const Pack<T, V> *)(x + 2 * pair);
    const Pack<T, V> hi = *(const Pack<T, V> *)(x + 2 * pair + V);
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int e = 2 * i;
      a.v[i] = e < V ? lo.v[e % V] : hi.v[e % V];
      b.v[i] = e + 1 < V ? lo.v[(e + 1) % V] : hi.v[(e + 1) % V];
    }
  } else {
    a = *(const Pack<T, V> *)(x + pair);
    b = *(const Pack<T, V> *)(x + p.half + pair);
  }
  Pack<T, V> ta, tb;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const float fa = to_f32(a.v[i]), fb = to_f32(b.v[i]);
    ta.v[i] = from_f32<T>(fa * c.v[i] - fb * s.v[i]);
    tb.v[i] = from_f32<T>(fb * c.v[i] + fa * s.v[i]);
  }
  if (INTERLEAVED) {
    Pack<T, V> lo, hi;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int e = 2 * i;
      (e < V ? lo : hi).v[e % V] = ta.v[i];
      (e + 1 < V ? lo : hi).v[(e + 1) % V] = tb.v[i];
    }
    *(Pack<T, V> *)(y + 2 * pair) = lo;
    *(Pack<T, V> *)(y + 2 * pair + V) = hi;
  } else {
    *(Pack<T, V> *)(y + pair) = ta;
    *(Pack<T, V> *)(y + p.half + pair) = tb;
  }
}

template <typename T>
hipError_t launch(hipStream_t st, const Rotary &r) {
  constexpr int V = 16 / (int)sizeof(T);
  RotaryArgs p = {r.x, r.y, r.cos, r.sin, r.positions, r.S, r.table_rows,
      r.B * r.S * r.H, 0, (int)r.H, r.D, r.rot / 2, 0, r.heads_first};
  // 16-byte pieces: the halves of a head, what passes through, and every row.
  const auto aligned = [](const void *q) { return ((uintptr_t)q & 15) == 0; };
  const bool wide = p.half % V == 0 && (r.D - r.rot) % (2 * V) == 0 &&
                    aligned(r.x) && aligned(r.y) && aligned(r.cos) && aligned(r.sin);
  p.units = wide ? r.D / 2 / V : (r.D + 1) / 2;
  const int64_t most = kMostGrid * 256 / p.units; // rows of a launch
  for (; p.first < p.rows; p.first += most) {
    const int64_t rows = p.rows - p.first < most ? p.rows - p.first : most;
    const dim3 grid((unsigned)((rows * p.units + 255) / 256)), block(256);
    if (wide && r.interleaved)
      k_rotary<T, V, true><<<grid, block, 0, st>>>(p);
    else if (wide)
      k_rotary<T, V, false><<<grid, block, 0, st>>>(p);
    else if (r.interleaved)
      k_rotary<T, 1, true><<<grid, block, 0, st>>>(p);
    else
      k_rotary<T, 1, false><<<grid, block, 0, st>>>(p);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess)
      return e;
  }
  return hipSuccess;
}

} // namespace
} // namespace llm

hipError_t launch_rotary(hipStream_t s, const Rotary &r) {
  switch (r.kind) {
  case kF32:
    return llm::launch<float>(s, r);
  case kF16:
    return llm::launch<_Float16>(s, r);
  default:
    return llm::launch<__bf16>(s, r);
  }
}

} // namespace om
