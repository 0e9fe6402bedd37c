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
// teams of 16 lanes have rows one behind the other, 16 each where a tile is read, 4 each of a step.  Narrow rows are held by 4 or
// 8 lanes, and there are 16 or 8 teams.  (Workgroups that composed
// 256 rows through LDS had 152 to 256 registers a thread and three waves or fewer a SIMD, which all waited together: 248 636 x
// 128 fp16, 48 us to read and 54 to apply.)
#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>

#include "core/core.h"
#include "core/elements.h"
#include "core/lane_sum.h"
#include "core/ragged.h"
#include "mlu_op_ext.h"

namespace {

using namespace mluop;

constexpr int kThreads = 256, kWaves = kThreads / 64;
constexpr int kPiece = 8;       // rows of a thread that are read together
// Rows that a thread applies at a time.  (Eight rows have an a and a u each in registers, and leave two or three waves a SIMD:
// 248 636 x 128 fp16 44 us to apply, four rows 39; gradients of 65 536 x 1024 bf16 135 and 120.)
constexpr int kRows = 4;
constexpr int kStateRows = 16;  // from one of the states that the backward pass takes to the next, whatever lies how
constexpr int kLeastTile = 64, kMostTile = 256;

// ACROSS lanes side by side, and teams of them behind one another.  (1 875 000 x 16 bf16: by 16 lanes, of which four have
// channels, 76 us to read and 94 to apply, by 4 31 and 43; its gradients 142 and 88.  937 500 x 32, by 16 and 8: 43 and 49, 30
// and 38; 82 and 73.)
template <int ACROSS>
struct Layout {
  static constexpr int kTeams = 64 / ACROSS;
  static constexpr int kTileRows = 2 * kPiece * kTeams, kStepRows = kRows * kTeams;  // of a wave
  static_assert(kTileRows >= kLeastTile && kTileRows <= kMostTile && kStepRows % kStateRows == 0, "");
};

// Who works out the states in front of the tiles: nobody (a wave has a whole sample), every wave for itself, a launch of its own.
enum Joining { kWhole, kFolded, kJoined };

struct Shape {
  int rows, channels, samples;
  int64_t x_stride, g_stride, dh_stride;  // elements from row to row; results lie row by row
  int slots;         // for tiles
  int side_by_side;  // waves of a workgroup that have slabs of the same rows
  int outside;       // workgroups along y for the rows of no sample
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

// The last sample whose first slot is not behind `slot` (0 where there is none), in scalar registers: of 64 pieces of the samples
// at a time, by whole waves.  (Slots rise with the samples.  One tile after the other, 64 samples at a time, 2001 rows in 1000
// samples took 48 us to read, so 38.)
template <int ROWS>
__device__ __forceinline__ int sampleOfSlot(const Shape &s, int slot) {
  const int lane = (int)threadIdx.x % 64;
  int from = 0, count = s.samples;
  while (count > 1) {
    const int step = (count + 63) / 64, at = from + min(lane * step, count - 1);
    int first, rows;
    segmentRows(s.starts, s.rows, at, &first, &rows);
    const uint64_t reached = __ballot(lane * step < count && firstSlot<ROWS>(at, first) <= slot);
    const int piece = reached == 0 ? 0 : 63 - __builtin_clzll(reached);
    from += piece * step;
    count = min(step, count - piece * step);
  }
  return __builtin_amdgcn_readfirstlane(from);
}

// What a wave has: a tile's rows in the order in which they are taken (row i of it is at `first + i * step`), or with WHOLE those
// of a sample, and a slab of channels.
template <int V, int ACROSS, bool WHOLE>
struct Work : Layout<ACROSS> {
  using Layout<ACROSS>::kTeams, Layout<ACROSS>::kTileRows, Layout<ACROSS>::kStepRows;
  static constexpr int kChannels = ACROSS * V;
  int64_t first, tile_slot, state_slot;
  int step, rows, sample;  // sample -1: nothing
  int in_sample, tiles;    // the tile's number in its sample, and how many that has
  int team, channel;
  bool there;              // this lane has channels; one that has none reads what the slab's first has

  // Slabs lie along x, and as many of a workgroup's waves as can be have slabs side by side, so that it reads what lies together
  // (four tiles of one slab: 35 us to read 248 636 x 128 fp16 in place of 31); tiles, or samples, along y.  FROM_LAST: the launch
  // before had them in order, and what it had last comes first.
  __device__ Work(const Shape &s, int64_t block, int64_t blocks, bool from_last) : sample(-1) {
    const int lane = (int)threadIdx.x % ACROSS, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x / 64);
    team = (int)threadIdx.x / ACROSS % kTeams;
    channel = ((int)blockIdx.x * s.side_by_side + wave % s.side_by_side) * kChannels;
    if (channel >= s.channels) return;
    there = channel + lane * V < s.channels;
    if (there) channel += lane * V;
    const int of = (int)(from_last ? blocks - 1 - block : block) * (kWaves / s.side_by_side) + wave / s.side_by_side;
    int segment_first, segment_rows;
    in_sample = 0;
    if (WHOLE) {
      if (of >= s.samples) return;
      sample = of;
      segmentRows(s.starts, s.rows, sample, &segment_first, &segment_rows);
      rows = segment_rows;
    } else {
      if (of >= s.slots) return;
      const int found = sampleOfSlot<kTileRows>(s, of);
      segmentRows(s.starts, s.rows, found, &segment_first, &segment_rows);
      in_sample = (int)(of - firstSlot<kTileRows>(found, segment_first));
      // (a sample without rows has a slot, too)
      if (in_sample < 0 || (in_sample > 0 && in_sample * kTileRows >= segment_rows)) return;
      sample = found;
      rows = min(kTileRows, segment_rows - in_sample * kTileRows);
    }
    const int from = in_sample * kTileRows;
    tiles = (segment_rows + kTileRows - 1) / kTileRows;
    step = s.reverse ? -1 : 1;
    first = s.reverse ? (int64_t)segment_first + segment_rows - 1 - from : (int64_t)segment_first + from;
    tile_slot = firstSlot<kTileRows>(sample, segment_first) + in_sample;
    state_slot = firstSlot<kStateRows>(sample, segment_first) + from / kStateRows;
  }
  __device__ __forceinline__ bool begins() const { return in_sample == 0; }
  __device__ __forceinline__ bool ends() const { return WHOLE || in_sample == tiles - 1; }
  __device__ __forceinline__ int steps() const { return (rows + kStepRows - 1) / kStepRows; }
};

// Where the threads of a wave have TEAM_ROWS rows each of a tensor, row `at` and the following of the first team: a scalar
// address for every row and one 32-bit offset for every thread (addresses of their own took most of the registers).
template <typename T, int TEAM_ROWS>
struct Lines {
  uintptr_t base;
  int64_t row_bytes;
  uint32_t offset;
  template <typename WORK>
  __device__ __forceinline__ Lines(const T *from, int64_t stride, const WORK &w, int at) {
    // (backwards the last team's rows lie first)
    const int64_t row = w.first + (int64_t)w.step * at - (w.step < 0 ? (WORK::kTeams - 1) * TEAM_ROWS : 0);
    base = reinterpret_cast<uintptr_t>(from) + (uintptr_t)(row * stride * (int64_t)sizeof(T));
    row_bytes = w.step * stride * (int64_t)sizeof(T);
    offset = (uint32_t)(w.step < 0 ? WORK::kTeams - 1 - w.team : w.team) * (uint32_t)(TEAM_ROWS * stride * (int64_t)sizeof(T)) +
             (uint32_t)w.channel * (uint32_t)sizeof(T);
  }
  __device__ __forceinline__ T *row(int r) const {
    return reinterpret_cast<T *>(base + (uintptr_t)(r * row_bytes) + (uintptr_t)offset);
  }
};
// (a tile's rows of fp32 that far apart: offsets stay within 32 bits; longer tiles are for rows less far apart)
constexpr int64_t kMostStride = MLUOP_EXT_GATED_SCAN_MOST_STRIDE, kNarrowStride = kMostStride * kLeastTile / kMostTile;
static_assert((uint64_t)(kLeastTile + 1) * kMostStride * sizeof(float) < (uint64_t)1 << 32, "32-bit offsets");
static_assert((uint64_t)(kMostTile + 1) * kNarrowStride * sizeof(float) < (uint64_t)1 << 32, "32-bit offsets");

// e^g of a gate of type T.  Its product with log2(e) is rounded, by which 2^p is off by up to 1.23 |g| units of 2^-24 of itself.
// With fp32 rows that is put right: c = g - p ln(2) is what was lost, and e + e c has it again; where 2^p is infinite, zero or
// no number it stays that (248 636 x 128 fp32 127 us in either way).  Rows of 16 bits, whose results are rounded to 2^13 such
// units and more, do without (us without and with it: 248 636 x 128 fp16 75 and 80, 65 536 x 1024 bf16 forward and backward 328
// and 336).
template <typename T>
__device__ __forceinline__ float exponential(float g) {
  const float p = g * 1.44269504f, e = __builtin_amdgcn_exp2f(p);
  if constexpr (!std::is_same_v<T, float>) return e;
  const float c = fmaf(p, 1.9046542e-9f, fmaf(p, -0.693147182f, g));  // (ln(2) is 0.693147182 - 1.9046542e-9)
  return fabsf(p) < 128.f ? fmaf(e, c, e) : e;
}

// a and u of a gate: a row's step is h -> a h + u x.  Half of what these kernels compute is here.  What has to be exact is an a
// close to one, whose error all steps of a long memory repeat: it is what a small u leaves of one.  An exponential beyond the
// range is infinite, its reciprocal zero.  In units of 2^-24 of the result: the power is off by 2 and the step that puts it right
// by 1, a sum or a product by 1, a reciprocal by 2; with fp32 rows together at most 7 for a and 6 for u, whatever the gate is.
template <typename T, int KIND>
__device__ __forceinline__ void gate(float g, float *a, float *u) {
  const float e = exponential<T>(g);
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

template <typename T, int V, int R>
struct Rows {
  typedef typename Word<sizeof(T) * V>::type W;
  W at[R];
  template <int TEAM_ROWS, typename WORK>
  __device__ __forceinline__ void load(const T *from, int64_t stride, const WORK &w, int first, float none) {
    const Lines<T, TEAM_ROWS> lines(from, stride, w, first);
    if (first + (WORK::kTeams - 1) * TEAM_ROWS + R <= w.rows) {
#pragma unroll
      for (int r = 0; r < R; ++r) at[r] = *reinterpret_cast<const W *>(lines.row(r));
      return;
    }
    Vector<T, V> empty;
#pragma unroll
    for (int i = 0; i < V; ++i) empty.v[i] = (T)none;
#pragma unroll
    for (int r = 0; r < R; ++r) {
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

// What the lane 4 or 8 away has, inside of a row of 16.
template <int AWAY>
__device__ __forceinline__ float exchanged(float v) {
  static_assert(AWAY == 4 || AWAY == 8, "");
  if constexpr (AWAY == 8) return lanesMoved<0x128>(v);  // turned by eight
  return lanesMoved<0x1B>(lanesMoved<0x141>(v));         // eight mirrored, then every four
}

// The teams' maps (a, b) composed, the first team's first, or with FROM_LAST the last's.  `a` and `b` become the composition
// of the teams in front of this one; all_a, all_b that of all.  By whole waves.
template <int ACROSS, bool FROM_LAST>
__device__ __forceinline__ void composeTeams(int team, float &a, float &b, float *all_a, float *all_b) {
  // teams inside of a row of 16 lanes: what is in front of this one (pa, pb) there, and all of the row's in a and b
  float pa = 1.f, pb = 0.f;
  auto pairs = [&](auto away) {
    constexpr int AWAY = decltype(away)::value;
    const bool second = ((team & (AWAY / ACROSS)) != 0) != FROM_LAST;
    const float oa = exchanged<AWAY>(a), ob = exchanged<AWAY>(b);
    // (in front of what is in front so far: the other's)
    pb = second ? fmaf(pa, ob, pb) : pb;
    pa = second ? pa * oa : pa;
    b = second ? fmaf(a, ob, b) : fmaf(oa, b, ob);
    a *= oa;
  };
  if constexpr (ACROSS <= 4) pairs(std::integral_constant<int, 4>());
  if constexpr (ACROSS <= 8) pairs(std::integral_constant<int, 8>());
  // rows of 16 lanes
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
  const int row = team / (16 / ACROSS);
  const bool second = ((row & 1) != 0) != FROM_LAST, behind = (row >= 2) != FROM_LAST;
  // (selected, not multiplied with zero: `a` may be infinite)
  a = second ? a1 : 1.f;
  b = second ? b1 : 0.f;
  b = behind ? fmaf(a, pb1, b) : b;
  a = behind ? a * pa1 : a;
  if constexpr (ACROSS < 16) {
    b = fmaf(pa, b, pb);
    a *= pa;
  }
}

// ---- forward -------------------------------------------------------------------------------

// What a tile does to the state that comes into it, to tiles[slot][channel].  GRAD: to the gradient that comes into it from
// behind.  A team has 16 rows of a tile here, and the teams are composed once.
template <typename T, int V, int ACROSS, int KIND, bool GRAD>
__global__ __launch_bounds__(kThreads) void gatedScanTiles(const T *__restrict__ x, const T *__restrict__ g, Shape s,
                                                           int64_t first_block, float2 *__restrict__ tiles) {
  typedef Work<V, ACROSS, false> Waves;
  const Waves w(s, first_block + blockIdx.y, 0, false);
  // (the tile that comes last makes no state that is kept, and samples of one tile are not read here at all: 2001 rows in 1000
  // samples 38 us else, so 14)
  if (w.sample < 0 || w.rows == 0 || (GRAD ? w.begins() : w.ends())) return;
  const int64_t x_stride = GRAD ? s.dh_stride : s.x_stride;
  constexpr int kTeamRows = Waves::kTileRows / Waves::kTeams, kPieces = kTeamRows / kPiece;
  float a[V], b[V];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    a[i] = 1.f;
    b[i] = 0.f;
  }
  struct Piece {
    Rows<T, V, kPiece> x, g;
  } one, other;
  auto load = [&](Piece &p, int k) {
    const int first = (GRAD ? kPieces - 1 - k : k) * kPiece;
    p.g.template load<kTeamRows>(g, s.g_stride, w, first, idle<KIND>());
    p.x.template load<kTeamRows>(x, x_stride, w, first, 0.f);
  };
  auto compose = [&](const Piece &p) {
#pragma unroll
    for (int q = 0; q < kPiece; ++q) {
      const int r = GRAD ? kPiece - 1 - q : q;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        float ga, u;
        gate<T, KIND>(p.g.value(r, i), &ga, &u);
        const float v = p.x.value(r, i);
        b[i] = GRAD ? ga * (b[i] + v) : fmaf(ga, b[i], u * v);
        a[i] *= ga;
      }
    }
  };
  // (a loop whatever the number of pieces: in a straight line the compiler mixes what it computes of two, and their loads are
  // waited for together: 38 us in place of 31)
  load(one, 0);
#pragma unroll 1
  for (int k = 0; k < kPieces; k += 2) {
    load(other, k + 1);
    compose(one);
    if (k + 2 < kPieces) load(one, k + 2);
    compose(other);
  }
#pragma unroll
  for (int i = 0; i < V; ++i) {
    float all_a, all_b;
    composeTeams<ACROSS, GRAD>(w.team, a[i], b[i], &all_a, &all_b);
    if (w.there && w.team == 0) tiles[w.tile_slot * s.channels + w.channel + i] = make_float2(all_a, all_b);
  }
}

// The state in front of every tile of TILE rows but a sample's first (from that in front of the sample, zero where there is
// none), to states[slot][channel].  FROM_LAST: tiles from a sample's last to its first.  kJoinChannels channels of a sample a
// workgroup; its tiles are cut into runs of kJoinRun, one for each of the threads that share a channel, and are read once:
// kJoinTiles at a time.  (One sample of 7325 tiles of 64 channels 25 us, 3 for each turn.  The next turn's tiles on their way
// meanwhile: no less.  Four channels a workgroup, and turns twice as long: 22, but four samples of some 970 tiles of 128 channels
// 10 in place of 9.)  Samples of few tiles go by 64 at a time.  (A workgroup for each: 10 000 samples of 10 rows of 256 channels
// 702 us, 1000 of 100 rows 72; so 13 and 14.)
constexpr int kJoinThreads = 512, kJoinChannels = 8, kJoinRun = 16;
constexpr int kJoinTiles = kJoinThreads / kJoinChannels * kJoinRun;
constexpr int kJoinBlocks = 4096;  // most workgroups; each takes every so many samples
template <int TILE, bool FROM_LAST>
__device__ __forceinline__ void joinSample(const float2 *tiles, const Shape &s, int sample, const float *initial, float *states) {
  constexpr int kJoinWaves = kJoinThreads / 64;
  __shared__ float2 s_wave[kJoinWaves][kJoinChannels];
  int first, rows;
  segmentRows(s.starts, s.rows, sample, &first, &rows);
  const int count = (rows + TILE - 1) / TILE, maps = count - 1;
  const int lane = threadIdx.x % kJoinChannels, run = threadIdx.x / kJoinChannels, wave = threadIdx.x / 64;
  const int channel = (int)blockIdx.x * kJoinChannels + lane;
  const bool there = channel < s.channels;
  const int64_t slot = firstSlot<TILE>(sample, first);
  auto at = [&](int tile) { return (slot + (FROM_LAST ? count - 1 - tile : tile)) * s.channels + (there ? channel : 0); };
  float h0 = initial == nullptr || !there ? 0.f : initial[(int64_t)sample * s.channels + channel];
  for (int t0 = 0; t0 < maps; t0 += kJoinTiles) {
    // (runs of one length as short as they can be)
    const int here = min(maps - t0, kJoinTiles), per = (here + kJoinTiles / kJoinRun - 1) / (kJoinTiles / kJoinRun);
    const int lo = t0 + run * per, left = min(per, t0 + here - lo);
    float2 v[kJoinRun];
#pragma unroll
    for (int j = 0; j < kJoinRun; ++j) {
      v[j] = make_float2(1.f, 0.f);
      if (j < left) v[j] = tiles[at(lo + j)];
    }
    float a = 1.f, b = 0.f;
#pragma unroll
    for (int j = 0; j < kJoinRun; ++j) {
      b = fmaf(v[j].x, b, v[j].y);
      a *= v[j].x;
    }
    // the runs in front: of this wave, then of those before
#pragma unroll
    for (int d = kJoinChannels; d < 64; d <<= 1) {
      const float fa = __shfl_up(a, d, 64), fb = __shfl_up(b, d, 64);
      const bool has = (int)(threadIdx.x & 63) >= d;
      b = has ? fmaf(a, fb, b) : b;
      a = has ? a * fa : a;
    }
    __syncthreads();
    if ((threadIdx.x & 63) >= 64 - kJoinChannels) s_wave[wave][lane] = make_float2(a, b);
    float ea = __shfl_up(a, kJoinChannels, 64), eb = __shfl_up(b, kJoinChannels, 64);
    if ((threadIdx.x & 63) < kJoinChannels) {
      ea = 1.f;
      eb = 0.f;
    }
    __syncthreads();
    float h = h0;
#pragma unroll
    for (int q = 0; q < kJoinWaves; ++q) {
      const float2 m = s_wave[q][lane];
      h0 = fmaf(m.x, h0, m.y);
      h = q + 1 == wave ? h0 : h;
    }
    h = fmaf(ea, h, eb);
#pragma unroll
    for (int j = 0; j < kJoinRun; ++j) {
      h = fmaf(v[j].x, h, v[j].y);
      if (j < left && there) states[at(lo + j + 1)] = h;
    }
  }
}
template <int TILE, bool FROM_LAST>
__global__ __launch_bounds__(kJoinThreads) void gatedScanJoin(const float2 *__restrict__ tiles, Shape s,
                                                              const float *__restrict__ initial,
                                                              float *__restrict__ states) {
  constexpr int kAtOnce = kJoinThreads / kJoinChannels;
  static_assert(kAtOnce == 64, "a ballot names the samples");
  const int by = (int)gridDim.y, channel = (int)blockIdx.x * kJoinChannels + (int)threadIdx.x % kJoinChannels;
  for (int64_t first = blockIdx.y; first < s.samples; first += (int64_t)kAtOnce * by) {
    // 64 samples together: those of few tiles by a thread for every channel
    const int64_t mine = first + (int64_t)(threadIdx.x / kJoinChannels) * by;
    int begin = 0, rows = 0;
    if (mine < s.samples) segmentRows(s.starts, s.rows, (int)mine, &begin, &rows);
    const int maps = (rows + TILE - 1) / TILE - 1;
    if (maps > 0 && maps <= kJoinRun && channel < s.channels) {
      const int64_t slot = firstSlot<TILE>((int)mine, begin);
      auto at = [&](int tile) { return (slot + (FROM_LAST ? maps - tile : tile)) * s.channels + channel; };
      float h = initial == nullptr ? 0.f : initial[mine * s.channels + channel];
      float2 v[kJoinRun];
#pragma unroll
      for (int j = 0; j < kJoinRun; ++j) v[j] = tiles[at(min(j, maps - 1))];
      // (stores behind the last of the loads, which are waited for in one order with them: 100 samples of 16 tiles 33 us, so 13)
#pragma unroll
      for (int j = 0; j < kJoinRun; ++j) v[j].y = h = fmaf(v[j].x, h, v[j].y);
#pragma unroll
      for (int j = 0; j < kJoinRun; ++j)
        if (j < maps) states[at(j + 1)] = v[j].y;
    }
    // then those of many, one after the other: the same ones for every wave
    const int64_t looked_at = first + (int64_t)(threadIdx.x & 63) * by;
    rows = 0;
    if (looked_at < s.samples) segmentRows(s.starts, s.rows, (int)looked_at, &begin, &rows);
    for (uint64_t some = __ballot(rows > TILE * (kJoinRun + 1)); some != 0; some &= some - 1)
      joinSample<TILE, FROM_LAST>(tiles, s, (int)(first + (int64_t)__builtin_ctzll(some) * by), initial, states);
  }
}

// The state that comes into a wave's rows: from the one in front of its tile (JOINED), or of its sample through the tiles in
// front.  FROM_LAST: the gradient that comes in from behind.  `initial` are those of the samples (null: zero).
template <int V, int ACROSS, Joining JOINING, bool FROM_LAST, typename WORK>
__device__ __forceinline__ void incoming(const WORK &w, const Shape &s, const float *initial, const float2 *tiles,
                                         const float *states, float (&h)[V]) {
  const bool joined = JOINING == kJoined && !(FROM_LAST ? w.ends() : w.begins());
  const float *from = joined ? states + w.tile_slot * s.channels
                             : (initial == nullptr ? nullptr : initial + (int64_t)w.sample * s.channels);
#pragma unroll
  for (int i = 0; i < V; ++i) h[i] = from == nullptr ? 0.f : from[w.channel + i];
  if (JOINING != kFolded) return;
  // as many of the tiles by each team
  const int count = FROM_LAST ? w.tiles - 1 - w.in_sample : w.in_sample;
  const int per = (count + WORK::kTeams - 1) / WORK::kTeams, lo = min(w.team * per, count), hi = min(lo + per, count);
  const int64_t slot = w.tile_slot - w.in_sample;
  float a[V], b[V];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    a[i] = 1.f;
    b[i] = 0.f;
  }
  constexpr int kFoldAhead = 4;
  for (int t0 = lo; t0 < hi; t0 += kFoldAhead) {
    float2 v[kFoldAhead][V];
#pragma unroll
    for (int j = 0; j < kFoldAhead; ++j) {
      const int t = min(t0 + j, hi - 1);
      const float2 *at = tiles + (slot + (FROM_LAST ? w.tiles - 1 - t : t)) * s.channels + w.channel;
#pragma unroll
      for (int i = 0; i < V; ++i) v[j][i] = at[i];
    }
#pragma unroll
    for (int j = 0; j < kFoldAhead; ++j) {
      if (t0 + j >= hi) break;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        b[i] = fmaf(v[j][i].x, b[i], v[j][i].y);
        a[i] *= v[j][i].x;
      }
    }
  }
#pragma unroll
  for (int i = 0; i < V; ++i) {
    float all_a, all_b;
    composeTeams<ACROSS, false>(w.team, a[i], b[i], &all_a, &all_b);
    h[i] = fmaf(all_a, h[i], all_b);
  }
}

// The rows of no sample, which are zero in every result: by workgroup `block` of those of every slab.
template <typename T, int V>
__device__ void outside(const Shape &s, int block, T *out, T *out2) {
  const float zero[V] = {};
  const int vectors = s.channels / V;
  block = block * (int)gridDim.x + (int)blockIdx.x;
  const int blocks = s.outside * (int)gridDim.x;
  for (int side = 0; side < 2; ++side) {
    int first, rows;
    segmentOrOutside(s.starts, s.rows, s.samples, side == 0 ? 0 : s.samples + 1, &first, &rows);
    const int64_t end = (int64_t)rows * vectors;
    for (int64_t at = (int64_t)block * kThreads + threadIdx.x; at < end; at += (int64_t)blocks * kThreads) {
      storeFloats<T, V>(out + (int64_t)first * s.channels + at * V, zero);
      if (out2 != nullptr) storeFloats<T, V>(out2 + (int64_t)first * s.channels + at * V, zero);
    }
  }
}

// What a sample without rows hands on, by the wave that has its slot.
template <typename WORK, int V>
__device__ __forceinline__ void handOn(const WORK &w, const Shape &s, const float *from, float *to) {
  if (!w.there || w.team != 0) return;
  const int64_t at = (int64_t)w.sample * s.channels + w.channel;
#pragma unroll
  for (int i = 0; i < V; ++i) to[at + i] = from == nullptr ? 0.f : from[at + i];
}

// The states of a tile's rows, step by step, and the state in front of every kStateRows rows to kept.
template <typename T, int V, int ACROSS, int KIND, Joining JOINING>
__global__ __launch_bounds__(kThreads, 5) void gatedScanApply(const T *__restrict__ x, const T *__restrict__ g, Shape s,
                                                           int64_t first_block, int64_t blocks,
                                                           const float *__restrict__ initial,
                                                           const float2 *__restrict__ tiles,
                                                           const float *__restrict__ states, float *__restrict__ kept,
                                                           float *__restrict__ final, T *__restrict__ out) {
  const int64_t block = first_block + blockIdx.y;
  if (block >= blocks) {
    outside<T, V>(s, (int)(block - blocks), out, static_cast<T *>(nullptr));
    return;
  }
  typedef Work<V, ACROSS, JOINING == kWhole> Waves;
  constexpr int kStepRows = Waves::kStepRows, kStates = kStepRows / kStateRows;
  const Waves w(s, block, blocks, JOINING != kWhole);
  if (w.sample < 0) return;
  if (w.rows == 0) {
    handOn<Waves, V>(w, s, initial, final);
    return;
  }
  float h0[V];
  const int steps = w.steps();
  Rows<T, V, kRows> xs, gs;
  auto load = [&](int k) {
    gs.template load<kRows>(g, s.g_stride, w, k * kStepRows, idle<KIND>());
    xs.template load<kRows>(x, s.x_stride, w, k * kStepRows, 0.f);
  };
  load(0);
  incoming<V, ACROSS, JOINING, false>(w, s, initial, tiles, states, h0);
  for (int k = 0; k < steps; ++k) {
    float ra[kRows][V], rb[kRows][V], a[V], b[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
      a[i] = 1.f;
      b[i] = 0.f;
    }
    auto row = [&](int r) {
#pragma unroll
      for (int i = 0; i < V; ++i) {
        float u;
        gate<T, KIND>(gs.value(r, i), &ra[r][i], &u);
        rb[r][i] = u * xs.value(r, i);
        b[i] = fmaf(ra[r][i], b[i], rb[r][i]);
        a[i] *= ra[r][i];
      }
    };
    row(0);
    // (the one row of a sample, as in a step of many sequences, is the first team's first: of 2048 x 1024 bf16 38 us without this)
    if (JOINING != kWhole || w.rows > 1) {
#pragma unroll
      for (int r = 1; r < kRows; ++r) row(r);
    } else {
#pragma unroll
      for (int r = 1; r < kRows; ++r)
#pragma unroll
        for (int i = 0; i < V; ++i) ra[r][i] = rb[r][i] = 0.f;
    }
    if (k + 1 < steps) load(k + 1);
    if (kStates == 1 && w.there && w.team == 0)
#pragma unroll
      for (int i = 0; i < V; ++i) kept[(w.state_slot + k) * s.channels + w.channel + i] = h0[i];
    float h[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
      float all_a, all_b;
      composeTeams<ACROSS, false>(w.team, a[i], b[i], &all_a, &all_b);
      h[i] = fmaf(a[i], h0[i], b[i]);
      h0[i] = fmaf(all_a, h0[i], all_b);
    }
    const Lines<T, kRows> lines(out, s.channels, w, k * kStepRows);
    const int mine = w.there ? w.rows - k * kStepRows - w.team * kRows : 0;
    if (kStates > 1 && mine > 0 && w.team * kRows % kStateRows == 0)
#pragma unroll
      for (int i = 0; i < V; ++i)
        kept[(w.state_slot + k * kStates + w.team * kRows / kStateRows) * s.channels + w.channel + i] = h[i];
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
#pragma unroll
      for (int i = 0; i < V; ++i) h[i] = fmaf(ra[r][i], h[i], rb[r][i]);
      if (r < mine) storeRow<T, V>(lines.row(r), h, s.streamed);
    }
  }
  if (w.ends() && w.there && w.team == 0) {
#pragma unroll
    for (int i = 0; i < V; ++i) final[(int64_t)w.sample * s.channels + w.channel + i] = h0[i];
  }
}

// ---- backward ------------------------------------------------------------------------------

// The gradients of a tile's rows, from the last step to the first: a step's states again from the one in front of it, and the
// gradient that comes in from behind.
template <typename T, int V, int ACROSS, int KIND, Joining JOINING>
__global__ __launch_bounds__(kThreads, 4) void gatedScanGrad(const T *__restrict__ dh, const T *__restrict__ x,
                                                          const T *__restrict__ g, Shape s, int64_t first_block,
                                                          int64_t blocks, const float *__restrict__ kept,
                                                          const float *__restrict__ final_grad,
                                                          const float2 *__restrict__ tiles,
                                                          const float *__restrict__ grads,
                                                          float *__restrict__ initial_grad, T *__restrict__ dx,
                                                          T *__restrict__ dg) {
  const int64_t block = first_block + blockIdx.y;
  if (block >= blocks) {
    outside<T, V>(s, (int)(block - blocks), dx, dg);
    return;
  }
  typedef Work<V, ACROSS, JOINING == kWhole> Waves;
  constexpr int kStepRows = Waves::kStepRows, kStates = kStepRows / kStateRows;
  const Waves w(s, block, blocks, JOINING != kWhole);
  if (w.sample < 0) return;
  if (w.rows == 0) {
    if (initial_grad != nullptr) handOn<Waves, V>(w, s, final_grad, initial_grad);
    return;
  }
  float l0[V];
  incoming<V, ACROSS, JOINING, true>(w, s, final_grad, tiles, grads, l0);
  for (int k = w.steps() - 1; k >= 0; --k) {
    Rows<T, V, kRows> xs, gs, ds;
    gs.template load<kRows>(g, s.g_stride, w, k * kStepRows, idle<KIND>());
    xs.template load<kRows>(x, s.x_stride, w, k * kStepRows, 0.f);
    ds.template load<kRows>(dh, s.dh_stride, w, k * kStepRows, 0.f);
    float h[V];
#pragma unroll
    for (int i = 0; i < V; ++i) h[i] = w.there ? kept[(w.state_slot + k * kStates) * s.channels + w.channel + i] : 0.f;
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
        gate<T, KIND>(gs.value(r, i), &ra[r][i], &ru[r][i]);
        b[i] = fmaf(ra[r][i], b[i], ru[r][i] * xs.value(r, i));
        // (the gradient comes from behind: through this row first, then through those in front of it, composed so far)
        a[i] *= ra[r][i];
        c[i] = fmaf(a[i], ds.value(r, i), c[i]);
      }
#pragma unroll
    for (int i = 0; i < V; ++i) {
      float all_a, all_b, behind = a[i];
      composeTeams<ACROSS, false>(w.team, a[i], b[i], &all_a, &all_b);
      h[i] = fmaf(a[i], h[i], b[i]);
      composeTeams<ACROSS, true>(w.team, behind, c[i], &all_a, &all_b);
      l[i] = fmaf(behind, l0[i], c[i]);
      l0[i] = fmaf(all_a, l0[i], all_b);
    }
    // the states again, and what a row's gradient is multiplied with for its gate's
    float slope[kRows][V];
#pragma unroll
    for (int r = 0; r < kRows; ++r)
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float v = xs.value(r, i);
        slope[r][i] = KIND == MLUOP_EXT_GATE_SIGMOID ? ru[r][i] * (h[i] - v) : h[i];
        h[i] = fmaf(ra[r][i], h[i], ru[r][i] * v);
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
        gg[i] = l[i] * slope[r][i];
      }
      if (r >= mine) continue;
      storeRow<T, V>(to_x.row(r), gx, s.streamed);
      storeRow<T, V>(to_g.row(r), gg, s.streamed);
    }
  }
  if (w.begins() && w.there && w.team == 0 && initial_grad != nullptr) {
#pragma unroll
    for (int i = 0; i < V; ++i) initial_grad[(int64_t)w.sample * s.channels + w.channel + i] = l0[i];
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

// Calls f(ACROSS): the lanes that hold a row, at least 4 and at most 16.
template <typename F>
void byAcross(int64_t vectors, int64_t most_stride, F f) {
  if (vectors > 8 || most_stride > kNarrowStride)
    f(std::integral_constant<int, 16>());
  else if (vectors > 4)
    f(std::integral_constant<int, 8>());
  else
    f(std::integral_constant<int, 4>());
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
  return 16 + (size_t)mostSlots<kLeastTile>(rows, samples) * channels * (sizeof(float2) + sizeof(float));
}
struct Workspace {
  float2 *tiles;
  float *states;
  Workspace(void *workspace, int64_t rows, int64_t channels, int64_t samples) {
    tiles = reinterpret_cast<float2 *>((reinterpret_cast<uintptr_t>(workspace) + 15) & ~(uintptr_t)15);
    states = reinterpret_cast<float *>(tiles + mostSlots<kLeastTile>(rows, samples) * channels);
  }
};

// A wave for a whole sample, and one launch in place of two or three, where there are few rows more than samples, as in a step of
// many sequences: it takes a microsecond for every 16 rows of the longest.  (us with a launch more / whole: one sample of 129
// rows of 1024 12 / 9, of 257 12 / 18, of 501 13 / 33; 400 sequences of which one has 113 rows 24 / 14.  At worst one of as many
// samples has all 4096 rows, in 256 such steps.)  Every wave folds the tiles in front of its own where these are few, at most 16
// for a team.
constexpr int64_t kFoldedRows = 4096, kWholeRows = 128;
Joining joiningOf(int64_t rows, int64_t samples) {
  if (rows > kFoldedRows) return kJoined;
  return rows <= samples + kWholeRows ? kWhole : kFolded;
}
template <typename F>
void byJoining(Joining joining, F f) {
  if (joining == kWhole)
    f(std::integral_constant<Joining, kWhole>());
  else if (joining == kFolded)
    f(std::integral_constant<Joining, kFolded>());
  else
    f(std::integral_constant<Joining, kJoined>());
}

// Workgroups for the rows of no sample: as many as would have so many values each, if all rows were such.  (8 of a slab: 60 us to
// apply 248 636 x 128 fp16 where the last 98 636 rows are no sample's, 110 where all but 100 are; so 27 and 13, and 38 as before
// where none are.)
constexpr int64_t kOutsideValues = 16384, kMostOutside = 1024;

// Slabs of CHANNELS channels along x, as many of a workgroup's waves as can be with slabs side by side; tiles, or samples, along
// y.
struct Grid {
  unsigned slabs;
  int64_t blocks;
};
template <int CHANNELS>
Grid gridOf(Shape *s, Joining joining, int tile) {
  const int64_t all = (s->channels + CHANNELS - 1) / CHANNELS;
  s->side_by_side = all >= 3 ? 4 : (int)all;
  s->slots = s->rows / tile + s->samples;
  const int64_t in_block = kWaves / s->side_by_side, items = joining == kWhole ? s->samples : s->slots;
  const unsigned slabs = (unsigned)((all + s->side_by_side - 1) / s->side_by_side);
  const int64_t pieces = (int64_t)s->rows * s->channels / kOutsideValues;
  s->outside = (int)std::max<int64_t>(std::min<int64_t>(pieces, kMostOutside) / slabs, 8);
  return {slabs, (items + in_block - 1) / in_block};
}

// Workgroups along y in as many launches as they need.
constexpr int64_t kMostAlongY = 65535;
template <typename F>
void alongY(int64_t blocks, F f) {
  for (int64_t first = 0; first < blocks; first += kMostAlongY) f(first, (unsigned)std::min(blocks - first, kMostAlongY));
}

template <int TILE, bool FROM_LAST>
void join(const mluop::LaunchCtx &lc, const float2 *tiles, const Shape &s, const float *initial, float *states) {
  lc.begin("gatedScanJoin");
  const int slabs = (s.channels + kJoinChannels - 1) / kJoinChannels;
  const int along_y = std::min(s.samples, std::max(kJoinBlocks / slabs, 1));
  gatedScanJoin<TILE, FROM_LAST><<<dim3((unsigned)slabs, (unsigned)along_y), kJoinThreads, 0, lc.stream>>>(tiles, s, initial,
                                                                                                         states);
  lc.end();
}

}  // namespace

mluOpStatus_t MLUOP_WIN_API mluOpExtGetGatedScanSizes(int64_t rows, int64_t channels, int64_t samples, size_t *carries,
                                                      size_t *workspace_size) {
  const char *api = "[mluOpExtGetGatedScanSizes]";
  PARAM_CHECK(api, carries != NULL);
  PARAM_CHECK(api, workspace_size != NULL);
  const mluOpStatus_t status = checkShape(api, rows, channels, samples);
  if (status != MLUOP_STATUS_SUCCESS) return status;
  *carries = (size_t)mostSlots<kStateRows>(rows, samples);
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
  const Joining joining = joiningOf(rows, samples);
  if (handle->hasNotes()) {
    handle->forgetNotesIn(out, bytes);
    handle->forgetNotesIn(final, (size_t)samples * channels * sizeof(float));
    handle->forgetNotesIn(carries, (size_t)mostSlots<kStateRows>(rows, samples) * channels * sizeof(float));
    handle->forgetNotesIn(workspace, workspace_size);
  }
  Shape s = {(int)rows,  (int)channels, (int)samples, features_stride, gates_stride, 0, 0, 1, 0,
             row_starts, reverse != 0,  bytes >= kStreamedBytes};
  const Workspace w(workspace, rows, channels, samples);
  const mluop::LaunchCtx lc = handle->launchCtx();
  const uintptr_t addresses = reinterpret_cast<uintptr_t>(features) | reinterpret_cast<uintptr_t>(gates) |
                              reinterpret_cast<uintptr_t>(out);
  byType(type, channels, features_stride | gates_stride, addresses, [&](auto zero, auto v) {
    typedef decltype(zero) T;
    constexpr int V = decltype(v)::value;
    const T *x = static_cast<const T *>(features), *g = static_cast<const T *>(gates);
    byAcross(channels / V, std::max(features_stride, gates_stride), [&](auto across) {
      byKind(kind, [&](auto of_kind) {
        constexpr int ACROSS = decltype(across)::value, KIND = decltype(of_kind)::value, TILE = Layout<ACROSS>::kTileRows;
        const Grid grid = gridOf<ACROSS * V>(&s, joining, TILE);
        if (joining != kWhole) {
          alongY(grid.blocks, [&](int64_t first, unsigned count) {
            lc.begin("gatedScanTiles");
            gatedScanTiles<T, V, ACROSS, KIND, false><<<dim3(grid.slabs, count), kThreads, 0, lc.stream>>>(x, g, s, first,
                                                                                                        w.tiles);
            lc.end();
          });
        }
        if (joining == kJoined) join<TILE, false>(lc, w.tiles, s, initial, w.states);
        byJoining(joining, [&](auto how) {
          constexpr Joining JOINING = decltype(how)::value;
          alongY(grid.blocks + s.outside, [&](int64_t first, unsigned count) {
            lc.begin("gatedScanApply");
            gatedScanApply<T, V, ACROSS, KIND, JOINING><<<dim3(grid.slabs, count), kThreads, 0, lc.stream>>>(
                x, g, s, first, grid.blocks, initial, w.tiles, w.states, carries, final,
                static_cast<T *>(out));
            lc.end();
          });
        });
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
  const Joining joining = joiningOf(rows, samples);
  if (handle->hasNotes()) {
    handle->forgetNotesIn(features_grad, bytes);
    handle->forgetNotesIn(gates_grad, bytes);
    if (initial_grad) handle->forgetNotesIn(initial_grad, (size_t)samples * channels * sizeof(float));
    handle->forgetNotesIn(workspace, workspace_size);
  }
  Shape s = {(int)rows,  (int)channels, (int)samples, features_stride, gates_stride, output_grad_stride, 0, 1, 0,
             row_starts, reverse != 0,  bytes >= kStreamedBytes};
  const Workspace w(workspace, rows, channels, samples);
  const mluop::LaunchCtx lc = handle->launchCtx();
  const uintptr_t addresses = reinterpret_cast<uintptr_t>(features) | reinterpret_cast<uintptr_t>(gates) |
                              reinterpret_cast<uintptr_t>(output_grad) | reinterpret_cast<uintptr_t>(features_grad) |
                              reinterpret_cast<uintptr_t>(gates_grad);
  byType(type, channels, features_stride | gates_stride | output_grad_stride, addresses, [&](auto zero, auto v) {
    typedef decltype(zero) T;
    constexpr int V = decltype(v)::value;
    const T *dh = static_cast<const T *>(output_grad), *x = static_cast<const T *>(features);
    const T *g = static_cast<const T *>(gates);
    byAcross(channels / V, std::max({features_stride, gates_stride, output_grad_stride}), [&](auto across) {
      byKind(kind, [&](auto of_kind) {
        constexpr int ACROSS = decltype(across)::value, KIND = decltype(of_kind)::value, TILE = Layout<ACROSS>::kTileRows;
        const Grid grid = gridOf<ACROSS * V>(&s, joining, TILE);
        if (joining != kWhole) {
          alongY(grid.blocks, [&](int64_t first, unsigned count) {
            lc.begin("gatedScanTiles");
            gatedScanTiles<T, V, ACROSS, KIND, true><<<dim3(grid.slabs, count), kThreads, 0, lc.stream>>>(dh, g, s, first,
                                                                                                       w.tiles);
            lc.end();
          });
        }
        if (joining == kJoined) join<TILE, true>(lc, w.tiles, s, final_grad, w.states);
        byJoining(joining, [&](auto how) {
          constexpr Joining JOINING = decltype(how)::value;
          alongY(grid.blocks + s.outside, [&](int64_t first, unsigned count) {
            lc.begin("gatedScanGrad");
            gatedScanGrad<T, V, ACROSS, KIND, JOINING><<<dim3(grid.slabs, count), kThreads, 0, lc.stream>>>(
                dh, x, g, s, first, grid.blocks, carries, final_grad, w.tiles, w.states, initial_grad,
                static_cast<T *>(features_grad), static_cast<T *>(gates_grad));
            lc.end();
          });
        });
      });
    });
  });
  HIP_CHECK_RETURN(api, hipGetLastError());
  return MLUOP_STATUS_SUCCESS;
}
