// mluOpExtGatedScanForward / Backward (no counterpart in the reference): a linear recurrence with gates along the rows of every
// sample, and its gradients.
//
//   h_t = a_t h_(t-1) + b_t       a = sigmoid(gate), b = (1 - a) x      or  a = exp(gate), b = x
//
// A row's step is the map h -> a h + b; maps are composed, (A, B) then (a, b) giving (a A, a B + b), and that is associative: a
// sample is cut into tiles, every tile into the rows of its threads, and only compositions wait for one another.  The
// gradients are a recurrence the other way: r = a_(t+1) l_(t+1) flows into row t, l_t = dh_t + r, and a_t l_t = a_t r + a_t dh_t
// flows on.  Sums and states are fp32.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>

#include "core/core.h"
#include "core/elements.h"
#include "core/ragged.h"
#include "mlu_op_ext.h"

namespace {

using namespace mluop;

constexpr int kThreads = 256;
// Rows of a tile.  The states at the tiles' beginnings are what the backward pass takes: the same for all types and
// alignments.
constexpr int kTileRows = 256;
constexpr int kOutsideBlocks = 16;  // workgroups for the rows of no sample

// How a workgroup lies over a tile of a slab of channels: ACROSS threads of V channels each, side by side (128 bytes of a row, 64
// of 2-byte types one or two at a time), and kTeams of them one after the other along the rows, kRows each.
template <typename T, int V>
struct Slab {
  static constexpr int kAcross = V >= 4 ? 8 : 32 / V;
  static constexpr int kTeams = kThreads / kAcross;
  static constexpr int kRows = kTileRows / kTeams;
  static constexpr int kChannels = kAcross * V;
  static constexpr int kParts = kThreads / kChannels;  // threads that compose a channel's teams
  static constexpr int kPartTeams = kTeams / kParts;
  static_assert(kParts * kChannels == kThreads && kParts * kPartTeams == kTeams, "no thread is left over");
};

struct Shape {
  int rows, channels, samples;
  int64_t x_stride, g_stride, dh_stride;  // elements from row to row; results lie row by row
  int most_tiles;
  const int32_t *starts;
  bool reverse;
  bool streamed;  // results go past the caches
};

// A tile's rows in the order in which they are taken: row i of it is at `first + i * step`.
struct Way {
  int64_t first;
  int step, rows, sample;
  bool begins, ends;  // it is its sample's first, its last
  __device__ Way(const RaggedTile &t, bool reverse)
      : first(reverse ? (int64_t)t.segment_first + t.segment_rows - 1 - t.in_segment * (int64_t)kTileRows : t.first),
        step(reverse ? -1 : 1), rows(t.rows), sample(t.segment), begins(t.in_segment == 0),
        ends(t.in_segment * (int64_t)kTileRows + t.rows == t.segment_rows) {}
};

// Sigmoids of a gate and of its negative, both to some 2^-22 of themselves: the exponential's argument is taken to log2 in two
// parts, and the reciprocal is put right once.
__device__ __forceinline__ float exponential(float v) {
  const float hi = v * 1.44269504f, lo = fmaf(v, 1.44269504f, -hi) + v * 1.92596299e-8f;
  const float e = __builtin_amdgcn_exp2f(hi);
  // (out of range: no correction, which would make a NaN of an infinity)
  return fabsf(hi) < 126.f ? fmaf(e, lo * 0.693147181f, e) : e;
}
__device__ __forceinline__ float reciprocal(float v) {  // of one or more
  const float r = __builtin_amdgcn_rcpf(v);
  return v < 1e38f ? fmaf(r, fmaf(-v, r, 1.f), r) : r;
}

// a and u of a gate: a row's step is h -> a h + u x.
template <int KIND>
__device__ __forceinline__ void gate(float g, float *a, float *u) {
  if (KIND == MLUOP_EXT_GATE_SIGMOID) {
    const float e = exponential(-fabsf(g)), big = reciprocal(1.f + e), small = e * big;
    *a = g < 0.f ? small : big;
    *u = g < 0.f ? big : small;
  } else {
    *a = exponential(g);
    *u = 1.f;
  }
}

// Composes what the teams of a workgroup have (a, b: of this thread's channels, over its rows in their order; teams in their
// order, or with FROM_LAST from the last), and leaves in `a` and `b` the composition of all teams in front of this thread's.
// Thread c of [0, kChannels) returns that of all in (*all_a, *all_b).  By the whole workgroup.
template <typename T, int V, bool FROM_LAST>
__device__ __forceinline__ void composeTeams(int team, int lane, float (&a)[V], float (&b)[V], float *all_a, float *all_b) {
  typedef Slab<T, V> S;
  __shared__ float s_a[S::kTeams][S::kChannels], s_b[S::kTeams][S::kChannels];
  __shared__ float s_part_a[S::kParts][S::kChannels], s_part_b[S::kParts][S::kChannels];
  __syncthreads();
  const int mine = FROM_LAST ? S::kTeams - 1 - team : team;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    s_a[mine][lane * V + i] = a[i];
    s_b[mine][lane * V + i] = b[i];
  }
  __syncthreads();
  const int c = (int)threadIdx.x % S::kChannels, part = (int)threadIdx.x / S::kChannels;
  float ta[S::kPartTeams], tb[S::kPartTeams], pa = 1.f, pb = 0.f;
#pragma unroll
  for (int t = 0; t < S::kPartTeams; ++t) {
    ta[t] = s_a[part * S::kPartTeams + t][c];
    tb[t] = s_b[part * S::kPartTeams + t][c];
  }
#pragma unroll
  for (int t = 0; t < S::kPartTeams; ++t) {
    pb = fmaf(ta[t], pb, tb[t]);
    pa *= ta[t];
  }
  s_part_a[part][c] = pa;
  s_part_b[part][c] = pb;
  __syncthreads();
  pa = 1.f;
  pb = 0.f;
  float fa = 1.f, fb = 0.f;
#pragma unroll
  for (int q = 0; q < S::kParts; ++q) {
    const float qa = s_part_a[q][c], qb = s_part_b[q][c];
    if (q < part) {
      pb = fmaf(qa, pb, qb);
      pa *= qa;
    }
    fb = fmaf(qa, fb, qb);
    fa *= qa;
  }
  *all_a = fa;
  *all_b = fb;
#pragma unroll
  for (int t = 0; t < S::kPartTeams; ++t) {
    s_a[part * S::kPartTeams + t][c] = pa;
    s_b[part * S::kPartTeams + t][c] = pb;
    pb = fmaf(ta[t], pb, tb[t]);
    pa *= ta[t];
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < V; ++i) {
    a[i] = s_a[mine][lane * V + i];
    b[i] = s_b[mine][lane * V + i];
  }
}

// This thread's rows of a tensor; zero behind the tile.
template <typename T, int V>
__device__ __forceinline__ void loadRows(const T *from, int64_t stride, const Way &way, int first, bool there,
                                         Vector<T, V> (&to)[Slab<T, V>::kRows]) {
#pragma unroll
  for (int i = 0; i < Slab<T, V>::kRows; ++i) {
    to[i] = {};
    if (there && first + i < way.rows)
      to[i] = *reinterpret_cast<const Vector<T, V> *>(from + (way.first + (int64_t)(first + i) * way.step) * stride);
  }
}

// ---- forward -------------------------------------------------------------------------------

// What a tile does to the state that comes into it, to tiles[tile][channel].  GRAD: to the gradient that comes into it from behind.
template <typename T, int V, int KIND, bool GRAD>
__global__ __launch_bounds__(kThreads) void gatedScanTiles(const T *__restrict__ x, const T *__restrict__ g, Shape s,
                                                           float2 *__restrict__ tiles) {
  typedef Slab<T, V> S;
  const RaggedTile t = findRaggedTile<false>(s.starts, s.rows, s.samples, kTileRows, blockIdx.x);
  if (t.segment < 0) return;
  const Way way(t, s.reverse);
  const int lane = (int)threadIdx.x % S::kAcross, team = (int)threadIdx.x / S::kAcross;
  const int channel = (int)blockIdx.y * S::kChannels + lane * V, first = team * S::kRows;
  const bool there = channel < s.channels;
  Vector<T, V> xs[S::kRows], gs[S::kRows];
  loadRows<T, V>(g + channel, s.g_stride, way, first, there, gs);
  loadRows<T, V>(x + channel, GRAD ? s.dh_stride : s.x_stride, way, first, there, xs);
  float a[V], b[V];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    a[i] = 1.f;
    b[i] = 0.f;
  }
#pragma unroll
  for (int k = 0; k < S::kRows; ++k) {
    const int r = GRAD ? S::kRows - 1 - k : k;
    if (first + r >= way.rows) continue;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      float ga, u;
      gate<KIND>((float)gs[r].v[i], &ga, &u);
      b[i] = GRAD ? ga * (b[i] + (float)xs[r].v[i]) : fmaf(ga, b[i], u * (float)xs[r].v[i]);
      a[i] *= ga;
    }
  }
  float all_a, all_b;
  composeTeams<T, V, GRAD>(team, lane, a, b, &all_a, &all_b);
  const int c = (int)blockIdx.y * S::kChannels + (int)threadIdx.x;
  if ((int)threadIdx.x < S::kChannels && c < s.channels) tiles[(int64_t)blockIdx.x * s.channels + c] = make_float2(all_a, all_b);
}

// The state at every tile's beginning (from that of its sample, zero where there is none), to carries[tile][channel], and behind
// the last tile.  FROM_LAST: tiles from a sample's last to its first.  kJoinChannels channels of a sample a workgroup; its
// tiles are cut into runs, one for each of the threads that share a channel.
constexpr int kJoinChannels = 16, kJoinRuns = kThreads / kJoinChannels, kJoinAhead = 8;
template <bool FROM_LAST>
__global__ __launch_bounds__(kThreads) void gatedScanJoin(const float2 *__restrict__ tiles, Shape s, int first_sample,
                                                          const float *__restrict__ initial, float *__restrict__ carries,
                                                          float *__restrict__ final) {
  __shared__ float s_a[kJoinRuns][kJoinChannels], s_b[kJoinRuns][kJoinChannels];
  const int sample = first_sample + (int)blockIdx.y;
  int first, rows;
  const int count = raggedTilesOf(s.starts, s.rows, sample, kTileRows, s.most_tiles, &first, &rows);
  const int lane = threadIdx.x % kJoinChannels, run = threadIdx.x / kJoinChannels;
  const int channel = (int)blockIdx.x * kJoinChannels + lane;
  const bool there = channel < s.channels;
  const int per = (count + kJoinRuns - 1) / kJoinRuns, lo = min(run * per, count), hi = min(lo + per, count);
  auto at = [&](int tile) { return (int64_t)(first + (FROM_LAST ? count - 1 - tile : tile)) * s.channels + channel; };
  float a = 1.f, b = 0.f;
  if (there) {
    for (int t0 = lo; t0 < hi; t0 += kJoinAhead) {
      float2 v[kJoinAhead];
#pragma unroll
      for (int j = 0; j < kJoinAhead; ++j) v[j] = tiles[at(min(t0 + j, hi - 1))];
#pragma unroll
      for (int j = 0; j < kJoinAhead; ++j) {
        if (t0 + j >= hi) break;
        b = fmaf(v[j].x, b, v[j].y);
        a *= v[j].x;
      }
    }
  }
  s_a[run][lane] = a;
  s_b[run][lane] = b;
  __syncthreads();
  if (!there) return;
  float h = initial == nullptr ? 0.f : initial[(int64_t)sample * s.channels + channel];
  for (int q = 0; q < run; ++q) h = fmaf(s_a[q][lane], h, s_b[q][lane]);
  for (int t0 = lo; t0 < hi; t0 += kJoinAhead) {
    float2 v[kJoinAhead];
#pragma unroll
    for (int j = 0; j < kJoinAhead; ++j) v[j] = tiles[at(min(t0 + j, hi - 1))];
#pragma unroll
    for (int j = 0; j < kJoinAhead; ++j) {
      if (t0 + j >= hi) break;
      carries[at(t0 + j)] = h;
      h = fmaf(v[j].x, h, v[j].y);
    }
  }
  if (run == kJoinRuns - 1 && final != nullptr) final[(int64_t)sample * s.channels + channel] = h;
}

// The rows of no sample, which are zero in every result, and with STATES what a sample without rows hands on.  By the workgroups
// behind those of the tiles.
template <typename T, int V>
__device__ void gatedScanOutside(const Shape &s, int block, const float *initial, float *final, T *out, T *out2) {
  typedef Slab<T, V> S;
  const int lane = (int)threadIdx.x % S::kAcross, team = (int)threadIdx.x / S::kAcross;
  const int channel = (int)blockIdx.y * S::kChannels + lane * V;
  if (channel >= s.channels) return;
  const float zero[V] = {};
  for (int side = 0; side < 2; ++side) {
    int first, rows;
    segmentOrOutside(s.starts, s.rows, s.samples, side == 0 ? 0 : s.samples + 1, &first, &rows);
    for (int64_t r = block * S::kTeams + team; r < rows; r += kOutsideBlocks * S::kTeams) {
      storeFloats<T, V>(out + (first + r) * s.channels + channel, zero);
      if (out2 != nullptr) storeFloats<T, V>(out2 + (first + r) * s.channels + channel, zero);
    }
  }
  if (final == nullptr) return;
  for (int sample = block * S::kTeams + team; sample < s.samples; sample += kOutsideBlocks * S::kTeams) {
    int first, rows;
    segmentRows(s.starts, s.rows, sample, &first, &rows);
    if (rows > 0) continue;
    const int64_t at = (int64_t)sample * s.channels + channel;
#pragma unroll
    for (int i = 0; i < V; ++i) final[at + i] = initial == nullptr ? 0.f : initial[at + i];
  }
}

// The states of a tile's rows from the one at its beginning.  SINGLE: no sample has more than one tile, whose beginning is the
// sample's, and nothing has run in front.
template <typename T, int V, int KIND, bool SINGLE>
__global__ __launch_bounds__(kThreads) void gatedScanApply(const T *__restrict__ x, const T *__restrict__ g, Shape s,
                                                           const float *__restrict__ initial, float *__restrict__ carries,
                                                           float *__restrict__ final, T *__restrict__ out) {
  typedef Slab<T, V> S;
  if ((int)blockIdx.x >= s.most_tiles) {
    gatedScanOutside<T, V>(s, (int)blockIdx.x - s.most_tiles, initial, SINGLE ? final : nullptr, out, nullptr);
    return;
  }
  // (from the last tile to the first: what has been read last is still in the caches)
  const int tile = SINGLE ? (int)blockIdx.x : s.most_tiles - 1 - (int)blockIdx.x;
  const RaggedTile t = findRaggedTile<false>(s.starts, s.rows, s.samples, kTileRows, tile);
  if (t.segment < 0) return;
  const Way way(t, s.reverse);
  const int lane = (int)threadIdx.x % S::kAcross, team = (int)threadIdx.x / S::kAcross;
  const int channel = (int)blockIdx.y * S::kChannels + lane * V, first = team * S::kRows;
  const bool there = channel < s.channels;
  Vector<T, V> xs[S::kRows], gs[S::kRows];
  loadRows<T, V>(g + channel, s.g_stride, way, first, there, gs);
  loadRows<T, V>(x + channel, s.x_stride, way, first, there, xs);
  float h[V] = {};
  if (there) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      if (SINGLE)
        h[i] = initial == nullptr ? 0.f : initial[(int64_t)way.sample * s.channels + channel + i];
      else
        h[i] = carries[(int64_t)tile * s.channels + channel + i];
    }
    if (SINGLE && team == 0) {
#pragma unroll
      for (int i = 0; i < V; ++i) carries[(int64_t)tile * s.channels + channel + i] = h[i];
    }
  }
  float ra[S::kRows][V], rb[S::kRows][V], a[V], b[V];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    a[i] = 1.f;
    b[i] = 0.f;
  }
#pragma unroll
  for (int r = 0; r < S::kRows; ++r)
#pragma unroll
    for (int i = 0; i < V; ++i) {
      float u;
      gate<KIND>((float)gs[r].v[i], &ra[r][i], &u);
      rb[r][i] = u * (float)xs[r].v[i];
      // (rows behind the tile are behind its last in every thread: what they do goes nowhere)
      b[i] = fmaf(ra[r][i], b[i], rb[r][i]);
      a[i] *= ra[r][i];
    }
  float all_a, all_b;
  composeTeams<T, V, false>(team, lane, a, b, &all_a, &all_b);
  if (!there) return;
#pragma unroll
  for (int i = 0; i < V; ++i) h[i] = fmaf(a[i], h[i], b[i]);
#pragma unroll
  for (int r = 0; r < S::kRows; ++r) {
    if (first + r >= way.rows) break;
#pragma unroll
    for (int i = 0; i < V; ++i) h[i] = fmaf(ra[r][i], h[i], rb[r][i]);
    storeFloats<T, V>(out + (way.first + (int64_t)(first + r) * way.step) * s.channels + channel, h, s.streamed);
    if (SINGLE && way.ends && first + r == way.rows - 1) {
#pragma unroll
      for (int i = 0; i < V; ++i) final[(int64_t)way.sample * s.channels + channel + i] = h[i];
    }
  }
}

// ---- backward ------------------------------------------------------------------------------

// The gradients of a tile's rows: their states again from the one at the tile's beginning, and the gradient that comes in from
// behind.  SINGLE: as above.
template <typename T, int V, int KIND, bool SINGLE>
__global__ __launch_bounds__(kThreads) void gatedScanGrad(const T *__restrict__ dh, const T *__restrict__ x,
                                                          const T *__restrict__ g, Shape s, const float *__restrict__ carries,
                                                          const float *__restrict__ final_grad,
                                                          const float *__restrict__ grad_carries,
                                                          float *__restrict__ initial_grad, T *__restrict__ dx,
                                                          T *__restrict__ dg) {
  typedef Slab<T, V> S;
  if ((int)blockIdx.x >= s.most_tiles) {
    gatedScanOutside<T, V>(s, (int)blockIdx.x - s.most_tiles, final_grad, SINGLE ? initial_grad : nullptr, dx, dg);
    return;
  }
  const int tile = blockIdx.x;
  const RaggedTile t = findRaggedTile<false>(s.starts, s.rows, s.samples, kTileRows, tile);
  if (t.segment < 0) return;
  const Way way(t, s.reverse);
  const int lane = (int)threadIdx.x % S::kAcross, team = (int)threadIdx.x / S::kAcross;
  const int channel = (int)blockIdx.y * S::kChannels + lane * V, first = team * S::kRows;
  const bool there = channel < s.channels;
  Vector<T, V> xs[S::kRows], gs[S::kRows], ds[S::kRows];
  loadRows<T, V>(g + channel, s.g_stride, way, first, there, gs);
  loadRows<T, V>(x + channel, s.x_stride, way, first, there, xs);
  loadRows<T, V>(dh + channel, s.dh_stride, way, first, there, ds);
  float h[V] = {}, l[V] = {};
  if (there) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      h[i] = carries[(int64_t)tile * s.channels + channel + i];
      if (SINGLE)
        l[i] = final_grad == nullptr ? 0.f : final_grad[(int64_t)way.sample * s.channels + channel + i];
      else
        l[i] = grad_carries[(int64_t)tile * s.channels + channel + i];
    }
  }
  float a[V], b[V], c[V];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    a[i] = 1.f;
    b[i] = c[i] = 0.f;
  }
#pragma unroll
  for (int r = 0; r < S::kRows; ++r) {
    if (first + r >= way.rows) continue;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      float ga, u;
      gate<KIND>((float)gs[r].v[i], &ga, &u);
      // (the gradient comes from behind: through this row first, then through those in front of it, composed so far)
      c[i] = fmaf(a[i] * ga, (float)ds[r].v[i], c[i]);
      b[i] = fmaf(ga, b[i], u * (float)xs[r].v[i]);
      a[i] *= ga;
    }
  }
  float behind_a[V], all_a, all_b;
#pragma unroll
  for (int i = 0; i < V; ++i) behind_a[i] = a[i];
  composeTeams<T, V, false>(team, lane, a, b, &all_a, &all_b);
  composeTeams<T, V, true>(team, lane, behind_a, c, &all_a, &all_b);
  if (!there) return;
  // states in front of every row
  float before[S::kRows][V];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    h[i] = fmaf(a[i], h[i], b[i]);
    l[i] = fmaf(behind_a[i], l[i], c[i]);
  }
#pragma unroll
  for (int r = 0; r < S::kRows; ++r)
#pragma unroll
    for (int i = 0; i < V; ++i) {
      float ga, u;
      gate<KIND>((float)gs[r].v[i], &ga, &u);
      before[r][i] = h[i];
      h[i] = fmaf(ga, h[i], u * (float)xs[r].v[i]);
    }
#pragma unroll
  for (int k = 0; k < S::kRows; ++k) {
    const int r = S::kRows - 1 - k;
    if (first + r >= way.rows) continue;
    float gx[V], gg[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
      float ga, u;
      gate<KIND>((float)gs[r].v[i], &ga, &u);
      const float all = (float)ds[r].v[i] + l[i];
      gx[i] = u * all;
      gg[i] = KIND == MLUOP_EXT_GATE_SIGMOID ? gx[i] * ga * (before[r][i] - (float)xs[r].v[i]) : all * before[r][i] * ga;
      l[i] = ga * all;
    }
    const int64_t at = (way.first + (int64_t)(first + r) * way.step) * s.channels + channel;
    storeFloats<T, V>(dx + at, gx, s.streamed);
    storeFloats<T, V>(dg + at, gg, s.streamed);
  }
  if (SINGLE && team == 0 && way.begins && initial_grad != nullptr) {
#pragma unroll
    for (int i = 0; i < V; ++i) initial_grad[(int64_t)way.sample * s.channels + channel + i] = l[i];
  }
}

// ---- host side -----------------------------------------------------------------------------

// Calls f(element type, V): vectors that divide a row and lie at multiples of their length.
template <typename F>
void byType(mluOpDataType_t type, int64_t channels, int64_t strides, uintptr_t addresses, F f) {
  auto fits = [&](int v) {
    return channels % v == 0 && strides % v == 0 && addresses % (v * (size_t)elementBytes(type)) == 0;
  };
  auto sixteen = [&](auto zero) {
    if (fits(8))
      f(zero, std::integral_constant<int, 8>());
    else if (fits(2))
      f(zero, std::integral_constant<int, 2>());
    else
      f(zero, std::integral_constant<int, 1>());
  };
  if (type == MLUOP_DTYPE_HALF) {
    sixteen((_Float16)0);
  } else if (type == MLUOP_DTYPE_BFLOAT16) {
    sixteen((__bf16)0.f);
  } else if (fits(4)) {
    f(0.f, std::integral_constant<int, 4>());
  } else {
    f(0.f, std::integral_constant<int, 1>());
  }
}

template <typename F>
void byKind(mluOpExtGate_t kind, F f) {
  if (kind == MLUOP_EXT_GATE_SIGMOID)
    f(std::integral_constant<int, MLUOP_EXT_GATE_SIGMOID>());
  else
    f(std::integral_constant<int, MLUOP_EXT_GATE_EXP>());
}

mluOpStatus_t checkShape(const char *api, int64_t rows, int64_t channels, int64_t samples) {
  PARAM_CHECK(api, rows >= 0);
  PARAM_CHECK(api, channels > 0);
  PARAM_CHECK(api, samples > 0);
  // (slabs of at least 32 channels along y)
  if (rows > INT32_MAX - 4096 || channels > (1 << 20) || samples > (1 << 20) || rows * channels > ((int64_t)1 << 46)) {
    MLUOP_LOG(ERROR) << api << " At most 2^31 - 4097 rows, 2^20 channels, 2^20 samples and 2^46 values are supported.";
    return MLUOP_STATUS_NOT_SUPPORTED;
  }
  return MLUOP_STATUS_SUCCESS;
}

bool strideFits(int64_t rows, int64_t channels, int64_t stride) {
  return stride >= channels && (rows == 0 || stride <= ((int64_t)1 << 46) / rows);
}

int64_t mostTiles(int64_t rows, int64_t samples) { return mostRaggedTiles(rows, samples, kTileRows); }

// (the caller's memory need not be aligned)
size_t workspaceBytes(int64_t rows, int64_t channels, int64_t samples) {
  return 16 + (size_t)mostTiles(rows, samples) * channels * (sizeof(float2) + sizeof(float));
}

constexpr int64_t kMostAlongY = 65535;  // workgroups of a grid

template <bool FROM_LAST>
void join(const mluop::LaunchCtx &lc, const float2 *tiles, const Shape &s, const float *initial, float *carries, float *final) {
  for (int64_t first = 0; first < s.samples; first += kMostAlongY) {
    lc.begin("gatedScanJoin");
    gatedScanJoin<FROM_LAST><<<dim3((unsigned)((s.channels + kJoinChannels - 1) / kJoinChannels),
                                    (unsigned)std::min<int64_t>(s.samples - first, kMostAlongY)),
                               kThreads, 0, lc.stream>>>(tiles, s, (int)first, initial, carries, final);
    lc.end();
  }
}

}  // namespace

mluOpStatus_t MLUOP_WIN_API mluOpExtGetGatedScanSizes(int64_t rows, int64_t channels, int64_t samples, size_t *carries,
                                                      size_t *workspace_size) {
  const char *api = "[mluOpExtGetGatedScanSizes]";
  PARAM_CHECK(api, carries != NULL);
  PARAM_CHECK(api, workspace_size != NULL);
  const mluOpStatus_t status = checkShape(api, rows, channels, samples);
  if (status != MLUOP_STATUS_SUCCESS) return status;
  *carries = (size_t)mostTiles(rows, samples);
  *workspace_size = workspaceBytes(rows, channels, samples);
  return MLUOP_STATUS_SUCCESS;
}

mluOpStatus_t MLUOP_WIN_API mluOpExtGatedScanForward(mluOpHandle_t handle, mluOpDataType_t type, const void *features,
                                                     int64_t features_stride, const void *gates, int64_t gates_stride,
                                                     int64_t rows, int64_t channels, const int32_t *row_starts,
                                                     int64_t samples, const float *initial, mluOpExtGate_t kind,
                                                     int reverse, void *workspace, size_t workspace_size, void *out,
                                                     float *final, float *carries) {
  const char *api = "[mluOpExtGatedScanForward]";
  PARAM_CHECK(api, handle != NULL);
  PARAM_CHECK(api, isFloating(type));
  const mluOpStatus_t status = checkShape(api, rows, channels, samples);
  if (status != MLUOP_STATUS_SUCCESS) return status;
  PARAM_CHECK(api, strideFits(rows, channels, features_stride) && strideFits(rows, channels, gates_stride));
  PARAM_CHECK(api, row_starts != NULL || samples == 1);
  PARAM_CHECK(api, kind == MLUOP_EXT_GATE_SIGMOID || kind == MLUOP_EXT_GATE_EXP);
  PARAM_CHECK(api, rows == 0 || (features != NULL && gates != NULL && out != NULL && carries != NULL));
  PARAM_CHECK(api, final != NULL);
  PARAM_CHECK(api, workspace != NULL);
  PARAM_CHECK(api, workspace_size >= workspaceBytes(rows, channels, samples));
  DEVICE_HANDLE_CHECK(api, handle);
  HIP_CHECK_RETURN(api, hipSetDevice(handle->device));
  const size_t bytes = (size_t)rows * channels * elementBytes(type);
  const int64_t most = mostTiles(rows, samples);
  if (handle->hasNotes()) {
    handle->forgetNotesIn(out, bytes);
    handle->forgetNotesIn(final, (size_t)samples * channels * sizeof(float));
    handle->forgetNotesIn(carries, (size_t)most * channels * sizeof(float));
    handle->forgetNotesIn(workspace, workspace_size);
  }
  const Shape s = {(int)rows,  (int)channels, (int)samples, features_stride, gates_stride, 0, (int)most,
                   row_starts, reverse != 0,  bytes >= kStreamedBytes};
  float2 *tiles = reinterpret_cast<float2 *>((reinterpret_cast<uintptr_t>(workspace) + 15) & ~(uintptr_t)15);
  const mluop::LaunchCtx lc = handle->launchCtx();
  const uintptr_t addresses = reinterpret_cast<uintptr_t>(features) | reinterpret_cast<uintptr_t>(gates) |
                              reinterpret_cast<uintptr_t>(out);
  byType(type, channels, features_stride | gates_stride, addresses, [&](auto zero, auto v) {
    byKind(kind, [&](auto of_kind) {
      typedef decltype(zero) T;
      constexpr int V = decltype(v)::value, KIND = decltype(of_kind)::value;
      const T *x = static_cast<const T *>(features), *g = static_cast<const T *>(gates);
      const unsigned slabs = (unsigned)((channels + Slab<T, V>::kChannels - 1) / Slab<T, V>::kChannels);
      const bool single = rows <= kTileRows;
      if (!single) {
        lc.begin("gatedScanTiles");
        gatedScanTiles<T, V, KIND, false><<<dim3((unsigned)most, slabs), kThreads, 0, lc.stream>>>(x, g, s, tiles);
        lc.end();
        join<false>(lc, tiles, s, initial, carries, final);
      }
      lc.begin("gatedScanApply");
      auto kernel = single ? gatedScanApply<T, V, KIND, true> : gatedScanApply<T, V, KIND, false>;
      kernel<<<dim3((unsigned)most + kOutsideBlocks, slabs), kThreads, 0, lc.stream>>>(x, g, s, initial, carries, final,
                                                                                       static_cast<T *>(out));
      lc.end();
    });
  });
  HIP_CHECK_RETURN(api, hipGetLastError());
  return MLUOP_STATUS_SUCCESS;
}

mluOpStatus_t MLUOP_WIN_API mluOpExtGatedScanBackward(mluOpHandle_t handle, mluOpDataType_t type, const void *output_grad,
                                                      int64_t output_grad_stride, const float *final_grad,
                                                      const void *features, int64_t features_stride, const void *gates,
                                                      int64_t gates_stride, int64_t rows, int64_t channels,
                                                      const int32_t *row_starts, int64_t samples, const float *carries,
                                                      mluOpExtGate_t kind, int reverse, void *workspace,
                                                      size_t workspace_size, void *features_grad, void *gates_grad,
                                                      float *initial_grad) {
  const char *api = "[mluOpExtGatedScanBackward]";
  PARAM_CHECK(api, handle != NULL);
  PARAM_CHECK(api, isFloating(type));
  const mluOpStatus_t status = checkShape(api, rows, channels, samples);
  if (status != MLUOP_STATUS_SUCCESS) return status;
  PARAM_CHECK(api, strideFits(rows, channels, features_stride) && strideFits(rows, channels, gates_stride) &&
                       strideFits(rows, channels, output_grad_stride));
  PARAM_CHECK(api, row_starts != NULL || samples == 1);
  PARAM_CHECK(api, kind == MLUOP_EXT_GATE_SIGMOID || kind == MLUOP_EXT_GATE_EXP);
  PARAM_CHECK(api, rows == 0 || (output_grad != NULL && features != NULL && gates != NULL && carries != NULL));
  PARAM_CHECK(api, rows == 0 || (features_grad != NULL && gates_grad != NULL));
  PARAM_CHECK(api, workspace != NULL);
  PARAM_CHECK(api, workspace_size >= workspaceBytes(rows, channels, samples));
  DEVICE_HANDLE_CHECK(api, handle);
  HIP_CHECK_RETURN(api, hipSetDevice(handle->device));
  const size_t bytes = (size_t)rows * channels * elementBytes(type);
  const int64_t most = mostTiles(rows, samples);
  if (handle->hasNotes()) {
    handle->forgetNotesIn(features_grad, bytes);
    handle->forgetNotesIn(gates_grad, bytes);
    if (initial_grad) handle->forgetNotesIn(initial_grad, (size_t)samples * channels * sizeof(float));
    handle->forgetNotesIn(workspace, workspace_size);
  }
  const Shape s = {(int)rows,  (int)channels, (int)samples, features_stride, gates_stride, output_grad_stride, (int)most,
                   row_starts, reverse != 0,  bytes >= kStreamedBytes};
  float2 *tiles = reinterpret_cast<float2 *>((reinterpret_cast<uintptr_t>(workspace) + 15) & ~(uintptr_t)15);
  float *grad_carries = reinterpret_cast<float *>(tiles + most * channels);
  const mluop::LaunchCtx lc = handle->launchCtx();
  const uintptr_t addresses = reinterpret_cast<uintptr_t>(features) | reinterpret_cast<uintptr_t>(gates) |
                              reinterpret_cast<uintptr_t>(output_grad) | reinterpret_cast<uintptr_t>(features_grad) |
                              reinterpret_cast<uintptr_t>(gates_grad);
  byType(type, channels, features_stride | gates_stride | output_grad_stride, addresses, [&](auto zero, auto v) {
    byKind(kind, [&](auto of_kind) {
      typedef decltype(zero) T;
      constexpr int V = decltype(v)::value, KIND = decltype(of_kind)::value;
      const T *dh = static_cast<const T *>(output_grad), *x = static_cast<const T *>(features);
      const T *g = static_cast<const T *>(gates);
      const unsigned slabs = (unsigned)((channels + Slab<T, V>::kChannels - 1) / Slab<T, V>::kChannels);
      const bool single = rows <= kTileRows;
      if (!single) {
        lc.begin("gatedScanTiles");
        gatedScanTiles<T, V, KIND, true><<<dim3((unsigned)most, slabs), kThreads, 0, lc.stream>>>(dh, g, s, tiles);
        lc.end();
        join<true>(lc, tiles, s, final_grad, grad_carries, initial_grad);
      }
      lc.begin("gatedScanGrad");
      auto kernel = single ? gatedScanGrad<T, V, KIND, true> : gatedScanGrad<T, V, KIND, false>;
      kernel<<<dim3((unsigned)most + kOutsideBlocks, slabs), kThreads, 0, lc.stream>>>(
          dh, x, g, s, carries, final_grad, grad_carries, initial_grad, static_cast<T *>(features_grad),
          static_cast<T *>(gates_grad));
      lc.end();
    });
  });
  HIP_CHECK_RETURN(api, hipGetLastError());
  return MLUOP_STATUS_SUCCESS;
}
