// mluOpExtGatedScanForward / Backward (no counterpart in the reference): a linear recurrence with gates along the rows of every
// sample, and its gradients.
//
//   h_t = a_t h_(t-1) + b_t       a = sigmoid(gate), b = (1 - a) x      or  a = exp(gate), b = x
//
// A row's step is the map h -> a h + b; maps are composed, (A, B) then (a, b) giving (a A, a B + b), and that is associative: a
// sample is cut into tiles, a tile into the rows of its threads, and only compositions wait for one another.  The gradients are
// a recurrence the other way: r = a_(t+1) l_(t+1) flows into row t, l_t = dh_t + r, and a_t l_t = a_t r + a_t dh_t flows on.
// Maps, states and sums are fp32.
//
// Everything is done by single waves, which wait for no other: 16 lanes hold 8 bytes of a row each, a line of 128, and four
// teams of 16 lanes have 8 rows each, one behind the other.  (Workgroups that composed 256 rows through LDS had 152 to 256
// registers a thread and three waves or fewer a SIMD, which all waited together: 248 636 x 128 fp16, 48 us to read and 54 to
// apply.)
#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>

#include "core/core.h"
#include "core/elements.h"
#include "core/ragged.h"
#include "mlu_op_ext.h"

namespace {

using namespace mluop;

constexpr int kThreads = 256, kWaves = kThreads / 64;
constexpr int kAcross = 16, kTeams = 64 / kAcross;  // lanes side by side, and teams of them behind one another
constexpr int kRows = 8;                            // of a thread in a step
// Rows that a wave takes at a time.  The states in front of every step are what the backward pass takes: the same for all types
// and alignments.
constexpr int kStepRows = kTeams * kRows;
constexpr int kTileSteps = 4, kTileRows = kTileSteps * kStepRows;  // of a wave
constexpr int kOutsideBlocks = 16;  // workgroups for the rows of no sample

struct Shape {
  int rows, channels, samples;
  int64_t x_stride, g_stride, dh_stride;  // elements from row to row; results lie row by row
  int most_tiles, slabs;
  const int32_t *starts;
  bool reverse;
  bool streamed;  // results go past the caches
};

// Where what is kept of a sample's tiles or steps begins: every sample's are behind those of the one in front, whatever their
// lengths, and all are inside mostSlots.
template <int ROWS>
__device__ __forceinline__ int64_t firstSlot(int sample, int first_row) { return (int64_t)first_row / ROWS + sample; }
template <int ROWS>
int64_t mostSlots(int64_t rows, int64_t samples) { return rows / ROWS + samples; }

// What a wave has: a tile's rows in the order in which they are taken (row i of it is at `first + i * step`), or with WHOLE those of
// a sample, and a slab of channels.
template <int V, bool WHOLE>
struct Work {
  static constexpr int kChannels = kAcross * V;
  int64_t first, tile_slot, step_slot;
  int step, rows, sample;  // sample -1: nothing
  int team, channel;
  bool there;              // this lane has channels; one that has none reads what the slab's first has

  __device__ Work(int64_t unit, const Shape &s) : sample(-1) {
    const int lane = (int)threadIdx.x % kAcross;
    team = (int)threadIdx.x / kAcross % kTeams;
    const int64_t of = unit / s.slabs;
    channel = (int)(unit - of * s.slabs) * kChannels + lane * V;
    there = channel < s.channels;
    if (!there) channel -= lane * V;
    int segment_first, segment_rows, in_segment = 0;
    if (WHOLE) {
      if (of >= s.samples) return;
      sample = (int)of;
      segmentRows(s.starts, s.rows, sample, &segment_first, &segment_rows);
      rows = segment_rows;
    } else {
      if (of >= s.most_tiles) return;
      const RaggedTile t = findRaggedTile<false>(s.starts, s.rows, s.samples, kTileRows, (int)of);
      if (t.segment < 0) return;
      sample = t.segment;
      segment_first = t.segment_first;
      segment_rows = t.segment_rows;
      in_segment = t.in_segment;
      rows = t.rows;
    }
    step = s.reverse ? -1 : 1;
    first = s.reverse ? (int64_t)segment_first + segment_rows - 1 - (int64_t)in_segment * kTileRows
                      : (int64_t)segment_first + (int64_t)in_segment * kTileRows;
    tile_slot = firstSlot<kTileRows>(sample, segment_first) + in_segment;
    step_slot = firstSlot<kStepRows>(sample, segment_first) + (int64_t)in_segment * kTileSteps;
  }
  __device__ __forceinline__ int steps() const { return (rows + kStepRows - 1) / kStepRows; }
};

// Where the threads of a wave have TEAM_ROWS rows each of a tensor, row `at` and the following of the first team: a scalar address
// for every row and one 32-bit offset for every thread (addresses of their own took most of the registers).
template <typename T, int TEAM_ROWS>
struct Lines {
  uintptr_t base;
  int64_t row_bytes;
  uint32_t offset;
  template <typename WORK>
  __device__ __forceinline__ Lines(const T *from, int64_t stride, const WORK &w, int at) {
    // (backwards the last team's rows lie first)
    const int64_t row = w.first + (int64_t)w.step * at - (w.step < 0 ? (kTeams - 1) * TEAM_ROWS : 0);
    base = reinterpret_cast<uintptr_t>(from) + (uintptr_t)(row * stride * (int64_t)sizeof(T));
    row_bytes = w.step * stride * (int64_t)sizeof(T);
    offset = (uint32_t)(w.step < 0 ? kTeams - 1 - w.team : w.team) * (uint32_t)(TEAM_ROWS * stride * (int64_t)sizeof(T)) +
             (uint32_t)w.channel * (uint32_t)sizeof(T);
  }
  __device__ __forceinline__ T *row(int r) const {
    return reinterpret_cast<T *>(base + (uintptr_t)(r * row_bytes) + (uintptr_t)offset);
  }
};
constexpr int64_t kMostStride = (int64_t)1 << 23;  // elements from row to row: offsets stay within 32 bits

// The wave's unit of work.  Workgroups go round the 8 XCDs one by one.  FROM_LAST: what the launch before had last comes first, on
// the XCDs whose caches have it.
constexpr int kXcds = 8;
__device__ __forceinline__ int64_t unitOf(int64_t block, int64_t blocks, bool from_last) {
  if (from_last) block = (blocks / kXcds - 1 - block / kXcds) * kXcds + block % kXcds;
  return block * kWaves + __builtin_amdgcn_readfirstlane((int)threadIdx.x / 64);
}
int64_t blocksOf(int64_t units, int slabs) {
  const int64_t blocks = (units * slabs + kWaves - 1) / kWaves;
  return (blocks + kXcds - 1) / kXcds * kXcds;
}

// a and u of a gate: a row's step is h -> a h + u x.  Half of what these kernels compute is here.  What has to be exact is an a
// close to one, whose error all steps of a long memory repeat: it is what a small u leaves of one.  An exponential beyond the
// range is infinite, its reciprocal zero.
template <int KIND>
__device__ __forceinline__ void gate(float g, float *a, float *u) {
  const float e = __builtin_amdgcn_exp2f(g * 1.44269504f);
  if (KIND == MLUOP_EXT_GATE_SIGMOID) {
    *u = __builtin_amdgcn_rcpf(1.f + e);
    *a = g < 0.f ? e * *u : 1.f - *u;
  } else {
    *a = e;
    *u = 1.f;
  }
}

// A thread's rows of a step of a tensor, as they lie in memory (whole words: elements of their own would take a register each).
// Rows behind the last are `none`, which makes a gate's step change nothing.
template <int BYTES>
struct Word;
template <>
struct Word<8> { typedef uint64_t type; };
template <>
struct Word<4> { typedef uint32_t type; };
template <>
struct Word<2> { typedef uint16_t type; };

template <typename T, int V>
struct Rows {
  typedef typename Word<sizeof(T) * V>::type W;
  W at[kRows];
  template <int TEAM_ROWS, typename WORK>
  __device__ __forceinline__ void load(const T *from, int64_t stride, const WORK &w, int first, float none) {
    const Lines<T, TEAM_ROWS> lines(from, stride, w, first);
    if (first + (kTeams - 1) * TEAM_ROWS + kRows <= w.rows) {
#pragma unroll
      for (int r = 0; r < kRows; ++r) at[r] = *reinterpret_cast<const W *>(lines.row(r));
      return;
    }
    Vector<T, V> empty;
#pragma unroll
    for (int i = 0; i < V; ++i) empty.v[i] = (T)none;
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      at[r] = __builtin_bit_cast(W, empty);
      if (first + w.team * TEAM_ROWS + r < w.rows) at[r] = *reinterpret_cast<const W *>(lines.row(r));
    }
  }
  __device__ __forceinline__ float value(int r, int i) const { return (float)__builtin_bit_cast(Vector<T, V>, at[r]).v[i]; }
};
template <int KIND>
__device__ __forceinline__ float idle() {
  return KIND == MLUOP_EXT_GATE_SIGMOID ? __builtin_inff() : 0.f;
}

// 8 bytes past the caches.
template <typename T, int V>
__device__ __forceinline__ void storeRow(T *to, const float (&v)[V], bool streamed) {
  if constexpr (sizeof(T) * V == 8) {
    if (streamed) {
      Vector<T, V> packed;
#pragma unroll
      for (int i = 0; i < V; ++i) packed.v[i] = (T)v[i];
      __builtin_nontemporal_store(__builtin_bit_cast(uint64_t, packed), reinterpret_cast<uint64_t *>(to));
      return;
    }
  }
  storeFloats<T, V>(to, v);
}

// Rows 0 and 2 of a wave's four rows of 16 lanes, in rows 0, 1 and 2, 3; and rows 1 and 3.
__device__ __forceinline__ void rowsOfPairs(float v, float *even, float *odd) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  *even = __uint_as_float(r[0]);
  *odd = __uint_as_float(r[1]);
}
// The lower and the upper half of a wave, in both.
__device__ __forceinline__ void halves(float v, float *low, float *high) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  *low = __uint_as_float(r[0]);
  *high = __uint_as_float(r[1]);
}

// The four teams' maps (a, b) composed, the first team's first, or with FROM_LAST the last's.  `a` and `b` become the composition
// of the teams in front of this one; all_a, all_b that of all four.  By whole waves.
template <bool FROM_LAST>
__device__ __forceinline__ void composeTeams(int team, float &a, float &b, float *all_a, float *all_b) {
  float a_even, a_odd, b_even, b_odd;
  rowsOfPairs(a, &a_even, &a_odd);
  rowsOfPairs(b, &b_even, &b_odd);
  // (first and second as they are taken)
  const float a1 = FROM_LAST ? a_odd : a_even, b1 = FROM_LAST ? b_odd : b_even;
  const float a2 = FROM_LAST ? a_even : a_odd, b2 = FROM_LAST ? b_even : b_odd;
  float pa_low, pa_high, pb_low, pb_high;
  halves(a1 * a2, &pa_low, &pa_high);
  halves(fmaf(a2, b1, b2), &pb_low, &pb_high);
  const float pa1 = FROM_LAST ? pa_high : pa_low, pb1 = FROM_LAST ? pb_high : pb_low;
  const float pa2 = FROM_LAST ? pa_low : pa_high, pb2 = FROM_LAST ? pb_low : pb_high;
  *all_a = pa1 * pa2;
  *all_b = fmaf(pa2, pb1, pb2);
  const bool second = ((team & 1) != 0) != FROM_LAST, behind = (team >= 2) != FROM_LAST;
  a = second ? a1 : 1.f;
  b = second ? b1 : 0.f;
  b = fmaf(a, behind ? pb1 : 0.f, b);
  a *= behind ? pa1 : 1.f;
}

// ---- forward -------------------------------------------------------------------------------

// What a tile does to the state that comes into it, to tiles[slot][channel].  GRAD: to the gradient that comes into it from behind.
// A team has 32 rows of the tile here, and the teams are composed once.
template <typename T, int V, int KIND, bool GRAD>
__global__ __launch_bounds__(kThreads) void gatedScanTiles(const T *__restrict__ x, const T *__restrict__ g, Shape s,
                                                           int64_t first_block, int64_t blocks, float2 *__restrict__ tiles) {
  const Work<V, false> w(unitOf(first_block + blockIdx.x, blocks, false), s);
  if (w.sample < 0) return;
  const int64_t x_stride = GRAD ? s.dh_stride : s.x_stride;
  float a[V], b[V];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    a[i] = 1.f;
    b[i] = 0.f;
  }
  // (8 rows of it are on their way while 8 others are composed)
  struct Piece {
    Rows<T, V> x, g;
  } one, other;
  auto load = [&](Piece &p, int k) {
    const int first = (GRAD ? kTileSteps - 1 - k : k) * kRows;
    p.g.template load<kTileSteps * kRows>(g, s.g_stride, w, first, idle<KIND>());
    p.x.template load<kTileSteps * kRows>(x, x_stride, w, first, 0.f);
  };
  auto compose = [&](const Piece &p) {
#pragma unroll
    for (int q = 0; q < kRows; ++q) {
      const int r = GRAD ? kRows - 1 - q : q;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        float ga, u;
        gate<KIND>(p.g.value(r, i), &ga, &u);
        const float v = p.x.value(r, i);
        b[i] = GRAD ? ga * (b[i] + v) : fmaf(ga, b[i], u * v);
        a[i] *= ga;
      }
    }
  };
  load(one, 0);
#pragma unroll 1
  for (int k = 0; k < kTileSteps; k += 2) {
    load(other, k + 1);
    compose(one);
    if (k + 2 < kTileSteps) load(one, k + 2);
    compose(other);
  }
#pragma unroll
  for (int i = 0; i < V; ++i) {
    float all_a, all_b;
    composeTeams<GRAD>(w.team, a[i], b[i], &all_a, &all_b);
    if (w.there && w.team == 0) tiles[w.tile_slot * s.channels + w.channel + i] = make_float2(all_a, all_b);
  }
}

// The state at every tile's beginning (from that of its sample, zero where there is none), to carries[slot][channel], and behind
// the last tile.  FROM_LAST: tiles from a sample's last to its first.  kJoinChannels channels of a sample a workgroup; its tiles
// are cut into runs, one for each of the threads that share a channel.  A run of up to kJoinAhead is read once.
constexpr int kJoinThreads = 512, kJoinChannels = 8, kJoinRuns = kJoinThreads / kJoinChannels, kJoinAhead = 8;
template <bool FROM_LAST>
__global__ __launch_bounds__(kJoinThreads) void gatedScanJoin(const float2 *__restrict__ tiles, Shape s, int first_sample,
                                                              const float *__restrict__ initial,
                                                              float *__restrict__ carries, float *__restrict__ final) {
  __shared__ float s_a[kJoinRuns][kJoinChannels], s_b[kJoinRuns][kJoinChannels];
  const int sample = first_sample + (int)blockIdx.y;
  int first, rows;
  segmentRows(s.starts, s.rows, sample, &first, &rows);
  const int count = (rows + kTileRows - 1) / kTileRows;
  const int lane = threadIdx.x % kJoinChannels, run = threadIdx.x / kJoinChannels;
  const int channel = (int)blockIdx.x * kJoinChannels + lane;
  const bool there = channel < s.channels;
  const int per = (count + kJoinRuns - 1) / kJoinRuns, lo = min(run * per, count), hi = there ? min(lo + per, count) : lo;
  const int64_t slot = firstSlot<kTileRows>(sample, first);
  auto at = [&](int tile) { return (slot + (FROM_LAST ? count - 1 - tile : tile)) * s.channels + channel; };
  float h = initial == nullptr || !there ? 0.f : initial[(int64_t)sample * s.channels + channel];
  float a = 1.f, b = 0.f;
  float2 v[kJoinAhead];
  for (int t0 = lo; t0 < hi; t0 += kJoinAhead) {
#pragma unroll
    for (int j = 0; j < kJoinAhead; ++j) v[j] = tiles[at(min(t0 + j, hi - 1))];
#pragma unroll
    for (int j = 0; j < kJoinAhead; ++j) {
      if (t0 + j >= hi) break;
      b = fmaf(v[j].x, b, v[j].y);
      a *= v[j].x;
    }
  }
  s_a[run][lane] = a;
  s_b[run][lane] = b;
  __syncthreads();
  if (!there) return;
  for (int q = 0; q < run; ++q) h = fmaf(s_a[q][lane], h, s_b[q][lane]);
  for (int t0 = lo; t0 < hi; t0 += kJoinAhead) {
    if (per > kJoinAhead) {
#pragma unroll
      for (int j = 0; j < kJoinAhead; ++j) v[j] = tiles[at(min(t0 + j, hi - 1))];
    }
#pragma unroll
    for (int j = 0; j < kJoinAhead; ++j) {
      if (t0 + j >= hi) break;
      carries[at(t0 + j)] = h;
      h = fmaf(v[j].x, h, v[j].y);
    }
  }
  if (run == kJoinRuns - 1 && final != nullptr) final[(int64_t)sample * s.channels + channel] = h;
}

// The rows of no sample, which are zero in every result: by workgroup `block` of kOutsideBlocks.
template <typename T, int V>
__device__ void zeroOutside(const Shape &s, int block, T *out, T *out2) {
  const float zero[V] = {};
  const int vectors = s.channels / V;
  for (int side = 0; side < 2; ++side) {
    int first, rows;
    segmentOrOutside(s.starts, s.rows, s.samples, side == 0 ? 0 : s.samples + 1, &first, &rows);
    const int64_t end = (int64_t)rows * vectors;
    for (int64_t at = (int64_t)block * kThreads + threadIdx.x; at < end; at += kOutsideBlocks * kThreads) {
      storeFloats<T, V>(out + (int64_t)first * s.channels + at * V, zero);
      if (out2 != nullptr) storeFloats<T, V>(out2 + (int64_t)first * s.channels + at * V, zero);
    }
  }
}

// The states of a tile's rows, step by step, from the one at its beginning; the states in front of every step to step_states.
// WHOLE: a wave has a sample, and nothing has run in front: `carries` are the samples' initial states, and it writes `final`.
template <typename T, int V, int KIND, bool WHOLE>
__global__ __launch_bounds__(kThreads) void gatedScanApply(const T *__restrict__ x, const T *__restrict__ g, Shape s,
                                                           int64_t first_block, int64_t blocks,
                                                           const float *__restrict__ carries,
                                                           float *__restrict__ step_states, float *__restrict__ final,
                                                           T *__restrict__ out) {
  const int64_t block = first_block + blockIdx.x;
  if (block >= blocks) {
    zeroOutside<T, V>(s, (int)(block - blocks), out, static_cast<T *>(nullptr));
    return;
  }
  const Work<V, WHOLE> w(unitOf(block, blocks, !WHOLE), s);
  if (w.sample < 0) return;
  const int64_t from = (WHOLE ? w.sample : w.tile_slot) * s.channels + w.channel;
  float h0[V];
#pragma unroll
  for (int i = 0; i < V; ++i) h0[i] = carries == nullptr || !w.there ? 0.f : carries[from + i];
  const int steps = w.steps();
  Rows<T, V> xs, gs;
  auto load = [&](int k) {
    gs.template load<kRows>(g, s.g_stride, w, k * kStepRows, idle<KIND>());
    xs.template load<kRows>(x, s.x_stride, w, k * kStepRows, 0.f);
  };
  load(0);
  for (int k = 0; k < steps; ++k) {
    float ra[kRows][V], rb[kRows][V], a[V], b[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
      a[i] = 1.f;
      b[i] = 0.f;
    }
#pragma unroll
    for (int r = 0; r < kRows; ++r)
#pragma unroll
      for (int i = 0; i < V; ++i) {
        float u;
        gate<KIND>(gs.value(r, i), &ra[r][i], &u);
        rb[r][i] = u * xs.value(r, i);
        b[i] = fmaf(ra[r][i], b[i], rb[r][i]);
        a[i] *= ra[r][i];
      }
    if (k + 1 < steps) load(k + 1);
    if (w.there && w.team == 0)
#pragma unroll
      for (int i = 0; i < V; ++i) step_states[(w.step_slot + k) * s.channels + w.channel + i] = h0[i];
    float h[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
      float all_a, all_b;
      composeTeams<false>(w.team, a[i], b[i], &all_a, &all_b);
      h[i] = fmaf(a[i], h0[i], b[i]);
      h0[i] = fmaf(all_a, h0[i], all_b);
    }
    const Lines<T, kRows> lines(out, s.channels, w, k * kStepRows);
    const int mine = w.there ? w.rows - k * kStepRows - w.team * kRows : 0;
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
#pragma unroll
      for (int i = 0; i < V; ++i) h[i] = fmaf(ra[r][i], h[i], rb[r][i]);
      if (r < mine) storeRow<T, V>(lines.row(r), h, s.streamed);
    }
  }
  if (WHOLE && w.there && w.team == 0) {
#pragma unroll
    for (int i = 0; i < V; ++i) final[from + i] = h0[i];
  }
}

// ---- backward ------------------------------------------------------------------------------

// The gradients of a tile's rows, from the last step to the first: a step's states again from the one in front of it, and the
// gradient that comes in from behind.  WHOLE: as above, `grad_carries` are the gradients of the final states.
template <typename T, int V, int KIND, bool WHOLE>
__global__ __launch_bounds__(kThreads, 3) void gatedScanGrad(const T *__restrict__ dh, const T *__restrict__ x,
                                                          const T *__restrict__ g, Shape s, int64_t first_block,
                                                          int64_t blocks, const float *__restrict__ step_states,
                                                          const float *__restrict__ grad_carries,
                                                          float *__restrict__ initial_grad, T *__restrict__ dx,
                                                          T *__restrict__ dg) {
  const int64_t block = first_block + blockIdx.x;
  if (block >= blocks) {
    zeroOutside<T, V>(s, (int)(block - blocks), dx, dg);
    return;
  }
  const Work<V, WHOLE> w(unitOf(block, blocks, !WHOLE), s);
  if (w.sample < 0) return;
  const int64_t from = (WHOLE ? w.sample : w.tile_slot) * s.channels + w.channel;
  float l0[V];
#pragma unroll
  for (int i = 0; i < V; ++i) l0[i] = grad_carries == nullptr || !w.there ? 0.f : grad_carries[from + i];
  for (int k = w.steps() - 1; k >= 0; --k) {
    Rows<T, V> xs, gs, ds;
    gs.template load<kRows>(g, s.g_stride, w, k * kStepRows, idle<KIND>());
    xs.template load<kRows>(x, s.x_stride, w, k * kStepRows, 0.f);
    ds.template load<kRows>(dh, s.dh_stride, w, k * kStepRows, 0.f);
    float h[V];
#pragma unroll
    for (int i = 0; i < V; ++i) h[i] = w.there ? step_states[(w.step_slot + k) * s.channels + w.channel + i] : 0.f;
    float ra[kRows][V], ru[kRows][V], a[V], b[V], c[V], l[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
      a[i] = 1.f;
      b[i] = c[i] = 0.f;
    }
#pragma unroll
    for (int r = 0; r < kRows; ++r)
#pragma unroll
      for (int i = 0; i < V; ++i) {
        gate<KIND>(gs.value(r, i), &ra[r][i], &ru[r][i]);
        b[i] = fmaf(ra[r][i], b[i], ru[r][i] * xs.value(r, i));
        // (the gradient comes from behind: through this row first, then through those in front of it, composed so far)
        a[i] *= ra[r][i];
        c[i] = fmaf(a[i], ds.value(r, i), c[i]);
      }
#pragma unroll
    for (int i = 0; i < V; ++i) {
      float all_a, all_b, behind = a[i];
      composeTeams<false>(w.team, a[i], b[i], &all_a, &all_b);
      h[i] = fmaf(a[i], h[i], b[i]);
      composeTeams<true>(w.team, behind, c[i], &all_a, &all_b);
      l[i] = fmaf(behind, l0[i], c[i]);
      l0[i] = fmaf(all_a, l0[i], all_b);
    }
    // states in front of every row
    float before[kRows][V];
#pragma unroll
    for (int r = 0; r < kRows; ++r)
#pragma unroll
      for (int i = 0; i < V; ++i) {
        before[r][i] = h[i];
        h[i] = fmaf(ra[r][i], h[i], ru[r][i] * xs.value(r, i));
      }
    const Lines<T, kRows> to_x(dx, s.channels, w, k * kStepRows), to_g(dg, s.channels, w, k * kStepRows);
    const int mine = w.there ? w.rows - k * kStepRows - w.team * kRows : 0;
#pragma unroll
    for (int r = kRows - 1; r >= 0; --r) {
      float gx[V], gg[V];
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float all = ds.value(r, i) + l[i];
        l[i] = ra[r][i] * all;
        gx[i] = ru[r][i] * all;
        gg[i] = KIND == MLUOP_EXT_GATE_SIGMOID ? ru[r][i] * l[i] * (before[r][i] - xs.value(r, i)) : l[i] * before[r][i];
      }
      if (r >= mine) continue;
      storeRow<T, V>(to_x.row(r), gx, s.streamed);
      storeRow<T, V>(to_g.row(r), gg, s.streamed);
    }
  }
  if (WHOLE && w.there && w.team == 0 && initial_grad != nullptr) {
#pragma unroll
    for (int i = 0; i < V; ++i) initial_grad[from + i] = l0[i];
  }
}

// ---- host side -----------------------------------------------------------------------------

// Calls f(element type, V): up to 8 bytes a lane, which divide a row and lie at multiples of their length.
template <typename F>
void byType(mluOpDataType_t type, int64_t channels, int64_t strides, uintptr_t addresses, F f) {
  auto fits = [&](int v) {
    return channels % v == 0 && strides % v == 0 && addresses % (v * (size_t)elementBytes(type)) == 0;
  };
  auto sixteen = [&](auto zero) {
    if (fits(4))
      f(zero, std::integral_constant<int, 4>());
    else if (fits(2))
      f(zero, std::integral_constant<int, 2>());
    else
      f(zero, std::integral_constant<int, 1>());
  };
  if (type == MLUOP_DTYPE_HALF) {
    sixteen((_Float16)0);
  } else if (type == MLUOP_DTYPE_BFLOAT16) {
    sixteen((__bf16)0.f);
  } else if (fits(2)) {
    f(0.f, std::integral_constant<int, 2>());
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

bool strideFits(int64_t channels, int64_t stride) { return stride >= channels && stride <= kMostStride; }

// Maps of the tiles and states in front of them.  (The caller's memory need not be aligned.)
size_t workspaceBytes(int64_t rows, int64_t channels, int64_t samples) {
  return 16 + (size_t)mostSlots<kTileRows>(rows, samples) * channels * (sizeof(float2) + sizeof(float));
}
struct Workspace {
  float2 *tiles;
  float *carries;
  Workspace(void *workspace, int64_t rows, int64_t channels, int64_t samples) {
    tiles = reinterpret_cast<float2 *>((reinterpret_cast<uintptr_t>(workspace) + 15) & ~(uintptr_t)15);
    carries = reinterpret_cast<float *>(tiles + mostSlots<kTileRows>(rows, samples) * channels);
  }
};

// A wave for a whole sample, and one launch in place of three: where there are few rows, or about one a sample, as in a step of many
// sequences.  (At worst one sample has them all, in 128 steps of a microsecond.)
bool wholeSamples(int64_t rows, int64_t samples) { return rows <= std::max<int64_t>(512, std::min<int64_t>(2 * samples, 4096)); }

constexpr int64_t kMostAlongY = 65535;  // workgroups of a grid

template <bool FROM_LAST>
void join(const mluop::LaunchCtx &lc, const float2 *tiles, const Shape &s, const float *initial, float *carries, float *final) {
  for (int64_t first = 0; first < s.samples; first += kMostAlongY) {
    lc.begin("gatedScanJoin");
    gatedScanJoin<FROM_LAST><<<dim3((unsigned)((s.channels + kJoinChannels - 1) / kJoinChannels),
                                    (unsigned)std::min<int64_t>(s.samples - first, kMostAlongY)),
                               kJoinThreads, 0, lc.stream>>>(tiles, s, (int)first, initial, carries, final);
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
  *carries = (size_t)mostSlots<kStepRows>(rows, samples);
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
  PARAM_CHECK(api, strideFits(channels, features_stride) && strideFits(channels, gates_stride));
  PARAM_CHECK(api, row_starts != NULL || samples == 1);
  PARAM_CHECK(api, kind == MLUOP_EXT_GATE_SIGMOID || kind == MLUOP_EXT_GATE_EXP);
  PARAM_CHECK(api, rows == 0 || (features != NULL && gates != NULL && out != NULL && carries != NULL));
  PARAM_CHECK(api, final != NULL);
  PARAM_CHECK(api, workspace != NULL);
  PARAM_CHECK(api, workspace_size >= workspaceBytes(rows, channels, samples));
  DEVICE_HANDLE_CHECK(api, handle);
  HIP_CHECK_RETURN(api, hipSetDevice(handle->device));
  const size_t bytes = (size_t)rows * channels * elementBytes(type);
  const int64_t most = mostRaggedTiles(rows, samples, kTileRows);
  if (handle->hasNotes()) {
    handle->forgetNotesIn(out, bytes);
    handle->forgetNotesIn(final, (size_t)samples * channels * sizeof(float));
    handle->forgetNotesIn(carries, (size_t)mostSlots<kStepRows>(rows, samples) * channels * sizeof(float));
    handle->forgetNotesIn(workspace, workspace_size);
  }
  Shape s = {(int)rows,  (int)channels, (int)samples, features_stride, gates_stride, 0, (int)most, 0,
             row_starts, reverse != 0,  bytes >= kStreamedBytes};
  const Workspace w(workspace, rows, channels, samples);
  const mluop::LaunchCtx lc = handle->launchCtx();
  const uintptr_t addresses = reinterpret_cast<uintptr_t>(features) | reinterpret_cast<uintptr_t>(gates) |
                              reinterpret_cast<uintptr_t>(out);
  byType(type, channels, features_stride | gates_stride, addresses, [&](auto zero, auto v) {
    byKind(kind, [&](auto of_kind) {
      typedef decltype(zero) T;
      constexpr int V = decltype(v)::value, KIND = decltype(of_kind)::value;
      const T *x = static_cast<const T *>(features), *g = static_cast<const T *>(gates);
      s.slabs = (int)((channels + kAcross * V - 1) / (kAcross * V));
      const bool whole = wholeSamples(rows, samples);
      const int64_t blocks = blocksOf(whole ? samples : most, s.slabs);
      if (!whole) {
        inLaunches(blocks, kThreads, [&](int64_t first, unsigned count) {
          lc.begin("gatedScanTiles");
          gatedScanTiles<T, V, KIND, false><<<count, kThreads, 0, lc.stream>>>(x, g, s, first, blocks, w.tiles);
          lc.end();
        });
        join<false>(lc, w.tiles, s, initial, w.carries, final);
      }
      auto kernel = whole ? gatedScanApply<T, V, KIND, true> : gatedScanApply<T, V, KIND, false>;
      inLaunches(blocks + kOutsideBlocks, kThreads, [&](int64_t first, unsigned count) {
        lc.begin("gatedScanApply");
        kernel<<<count, kThreads, 0, lc.stream>>>(x, g, s, first, blocks, whole ? initial : w.carries, carries, final,
                                                  static_cast<T *>(out));
        lc.end();
      });
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
  PARAM_CHECK(api, strideFits(channels, features_stride) && strideFits(channels, gates_stride) &&
                       strideFits(channels, output_grad_stride));
  PARAM_CHECK(api, row_starts != NULL || samples == 1);
  PARAM_CHECK(api, kind == MLUOP_EXT_GATE_SIGMOID || kind == MLUOP_EXT_GATE_EXP);
  PARAM_CHECK(api, rows == 0 || (output_grad != NULL && features != NULL && gates != NULL && carries != NULL));
  PARAM_CHECK(api, rows == 0 || (features_grad != NULL && gates_grad != NULL));
  PARAM_CHECK(api, workspace != NULL);
  PARAM_CHECK(api, workspace_size >= workspaceBytes(rows, channels, samples));
  DEVICE_HANDLE_CHECK(api, handle);
  HIP_CHECK_RETURN(api, hipSetDevice(handle->device));
  const size_t bytes = (size_t)rows * channels * elementBytes(type);
  const int64_t most = mostRaggedTiles(rows, samples, kTileRows);
  if (handle->hasNotes()) {
    handle->forgetNotesIn(features_grad, bytes);
    handle->forgetNotesIn(gates_grad, bytes);
    if (initial_grad) handle->forgetNotesIn(initial_grad, (size_t)samples * channels * sizeof(float));
    handle->forgetNotesIn(workspace, workspace_size);
  }
  Shape s = {(int)rows,  (int)channels, (int)samples, features_stride, gates_stride, output_grad_stride, (int)most, 0,
             row_starts, reverse != 0,  bytes >= kStreamedBytes};
  const Workspace w(workspace, rows, channels, samples);
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
      s.slabs = (int)((channels + kAcross * V - 1) / (kAcross * V));
      const bool whole = wholeSamples(rows, samples);
      const int64_t blocks = blocksOf(whole ? samples : most, s.slabs);
      if (!whole) {
        inLaunches(blocks, kThreads, [&](int64_t first, unsigned count) {
          lc.begin("gatedScanTiles");
          gatedScanTiles<T, V, KIND, true><<<count, kThreads, 0, lc.stream>>>(dh, g, s, first, blocks, w.tiles);
          lc.end();
        });
        join<true>(lc, w.tiles, s, final_grad, w.carries, initial_grad);
      }
      auto kernel = whole ? gatedScanGrad<T, V, KIND, true> : gatedScanGrad<T, V, KIND, false>;
      inLaunches(blocks + kOutsideBlocks, kThreads, [&](int64_t first, unsigned count) {
        lc.begin("gatedScanGrad");
        kernel<<<count, kThreads, 0, lc.stream>>>(dh, x, g, s, first, blocks, carries, whole ? final_grad : w.carries,
                                                  initial_grad, static_cast<T *>(features_grad), static_cast<T *>(gates_grad));
        lc.end();
      });
    });
  });
  HIP_CHECK_RETURN(api, hipGetLastError());
  return MLUOP_STATUS_SUCCESS;
}
