// Gated linear recurrence over packed sequences, and its gradients.
//
// h = a h + b is a scan of affine maps, one scan a channel.  A tile is 64 channels of some
// hundred rows: a thread folds its rows' maps into one, (A, B) with h -> A h + B, the maps of
// the row groups are scanned through LDS, and the state in front of the tile comes by a look-back over the
// tiles before it.  Rows are read once, stay in registers, and are written once.
//
// The look-back applies maps to a state, one after the other, and never joins two of them: whether
// it begins at the state that the tile before it has published or at one some tiles further back, it goes
// through the same operations on the same numbers, so every run gives the same bits.
//
// Bound by latency in front of the memory: of a tile's 11 us, loads, the fold, the look-back and
// the stores follow one another, and two (backwards three) tiles share a compute unit.  65536 x 2048
// bfloat16 210 us, 3.8 TB/s; 161 without the look-back's wait, which is all that is known to be left.
// Gradients of 31744 x 4096 390 us, 4.0 TB/s.  (Rows of a thread, us, 16 / 8 / 4 / 2: forwards 392 / 229 / 269 / 384 of the first
// form, backwards 8 / 4 / 2: 614 / 465 / 524: shorter tiles walk back more often than they fill the
// waits.  Blocks that go on from tile to tile, the next one's loads in front of the stores: 280 and 440.
// Polls as seldom as every 2048 cycles: no difference.)
//
// A sequence's first row is a reset: its map forgets what comes in, whatever that is (a NaN
// times 0 would still be one).  A reset is marked by A = -0, which no product of
// decays gives.  Backwards, with P[t] = a[t] G[t] for the state, G[t] = grad_out[t] + P[t+1] is the same scan
// from the last row to the first; what is said of first rows holds of last ones.
#include "gates.hpp"
#include "operators.hpp"

namespace ilgpu_hip {

namespace {

constexpr int kBlock = 256;
constexpr int kWaves = kBlock / kWaveSize;
constexpr int kTileChannels = kWaveSize;  // a wave's lanes walk back, a channel each
constexpr int kWindow = 4;                // tiles that a look-back asks at a time
constexpr int kWideWindow = 16;           // and of few columns of tiles
constexpr uint32_t kMostPolls = 1 << 24;  // of a look-back: many seconds
constexpr int64_t kMostBlocks = 1 << 22;  // of a launch

// Rows of a thread; row groups of a tile; rows of a tile.
template <int W> constexpr int groups_of() { return kBlock * W / kTileChannels; }
constexpr int kRows = 8, kBackRows = 4, kLongBackRows = 8;
constexpr int kFewestRows = kRows < kBackRows ? kRows : kBackRows;

constexpr float kSmallestNormal = 0x1p-126f;

constexpr int64_t kTicketBytes = 128;  // of a column of tiles: a line of its own
constexpr int64_t kStateBytes = kTileChannels * 16;

// h -> 2^e a h + b, 1 <= a < 2 (or 0, infinity, a NaN; -0: a reset).  The decays of some rows
// leave float32 together where each of them and the state do not: infinity times a state of 0, or 0 times an
// infinite one, would be a NaN.  2^e goes to the state, which rounds nothing but results below the
// normal numbers.
struct Map {
  float a, b;
  int32_t e;
};
__device__ __forceinline__ bool is_reset(float a) {
  return __builtin_bit_cast(uint32_t, a) == 0x80000000u;
}
// 2^e a is multiplied by `factor`, 1/2 <= a < 1 behind it.
__device__ __forceinline__ void multiply(float& a, int32_t& e, float factor) {
  const float product = a * factor;
  a = __builtin_amdgcn_frexp_mantf(product);
  e += __builtin_amdgcn_frexp_expf(product);
}
__device__ __forceinline__ float apply(Map m, float h) {
  return is_reset(m.a) ? m.b : fmaf(m.a, __builtin_ldexpf(h, m.e), m.b);
}
// The map that does `first`, then `then`.
__device__ __forceinline__ Map behind(Map then, Map first) {
  Map m{then.a, apply(then, first.b), then.e + first.e};
  multiply(m.a, m.e, first.a);
  m.a = is_reset(then.a) || is_reset(first.a) ? -0.0f : 2.0f * m.a;
  --m.e;
  return m;
}

// a and 1 - a of a gate, each to some units in its last place.
template <typename T, bool SIGMOID>
__device__ __forceinline__ void decay_of(float gate, float& a, float& left) {
  if constexpr (SIGMOID) {
    logistic<T>(gate, a, left);
  } else {
    a = exp_of<T>(gate);
    // Near 0, where the difference has lost its bits, 1 - exp by its series (off by 2e-8 at most).
    const float series =
        -gate * fmaf(gate * (1.0f / 2), fmaf(gate * (1.0f / 3), fmaf(gate * (1.0f / 4), fmaf(gate * (1.0f / 5), fmaf(
        gate * (1.0f / 6), fmaf(gate, 1.0f / 7, 1.0f), 1.0f), 1.0f), 1.0f), 1.0f), 1.0f);
    left = fabsf(gate) < 0.35f ? series : 1.0f - a;
  }
}

// Hides where a vector comes from, so that what is made of it is made anew.
template <typename V> __device__ __forceinline__ void keep(V& v) {
  if constexpr (sizeof(V) == 16) {
    typedef uint32_t Words __attribute__((ext_vector_type(4)));
    Words w = __builtin_bit_cast(Words, v);
    asm volatile("" : "+v"(w));
    v = __builtin_bit_cast(V, w);
  } else if constexpr (sizeof(V) == 4) {
    uint32_t w = __builtin_bit_cast(uint32_t, v);
    asm volatile("" : "+v"(w));
    v = __builtin_bit_cast(V, w);
  } else {
    static_assert(sizeof(V) == 2, "a vector of 16 bytes or one element");
    uint32_t w = __builtin_bit_cast(uint16_t, v);
    asm volatile("" : "+v"(w));
    v = __builtin_bit_cast(V, (uint16_t)w);
  }
}

struct Sequences {
  const void* offsets;   // nullptr: `count` of `length` rows each
  int32_t wide;          // offsets are int64
  int64_t count;
  uint32_t length;
  __device__ __forceinline__ int64_t offset(int64_t i) const {
    return wide ? static_cast<const int64_t*>(offsets)[i]
                : (int64_t) static_cast<const int32_t*>(offsets)[i];
  }
};

// Where sequences begin and end in a tile: a bit for each row of a row group, in the order of the
// scan, and the sequence for each row that has one.
template <int GROUPS, int ROWS> struct Marks {
  uint32_t begin_bits[GROUPS], end_bits[GROUPS];
  int32_t begins[GROUPS * ROWS], ends[GROUPS * ROWS];
};

// Marks the rows of the tile from `first` on; called by the whole block.  Rows [*from, *to) belong to
// sequences.  (Offsets that are none put marks in wrong rows of the tile, but in none outside.)
template <bool BACK, int GROUPS, int ROWS>
__device__ __forceinline__ void mark_rows(const Sequences& s, int64_t first, int64_t rows,
                                          Marks<GROUPS, ROWS>& marks, int64_t* from, int64_t* to) {
  constexpr int kTileRows = GROUPS * ROWS;
  if (threadIdx.x < GROUPS) marks.begin_bits[threadIdx.x] = marks.end_bits[threadIdx.x] = 0;
  const auto mark = [&](uint32_t* bits, int32_t* sequences, int row, int64_t sequence) {
    const int i = BACK ? kTileRows - 1 - row : row;
    sequences[row] = (int32_t)sequence;
    atomicOr(&bits[i / ROWS], 1u << (i % ROWS));
  };
  if (s.offsets == nullptr) {
    __syncthreads();
    const uint32_t before = (uint32_t)first / s.length;
    for (int64_t j = before + threadIdx.x; j <= s.count; j += kBlock) {
      const int64_t row = j * s.length - first;
      if (row > kTileRows) break;
      if (row >= 0 && row < kTileRows && j < s.count) mark(marks.begin_bits, marks.begins, (int)row, j);
      if (row > 0) mark(marks.end_bits, marks.ends, (int)row - 1, j - 1);
    }
    *from = 0;
    *to = rows;
    __syncthreads();
    return;
  }
  // The first offset that is not below `first` lies in [at, at + left].
  int64_t at = 0, left = s.count + 1;
  while (left > kBlock) {
    const int64_t step = (left + kBlock - 1) / kBlock, i = at + threadIdx.x * step;
    const int below = __syncthreads_count(i < at + left && s.offset(i) < first);
    const int64_t end = at + left;
    if (below > 0) at += (below - 1) * step;
    left = step < end - at ? step : end - at;
  }
  const int64_t low = s.offset(0), high = s.offset(s.count);
  *from = low > 0 ? low : 0;
  *to = high < rows ? high : rows;
  __syncthreads();
  for (int64_t j = at + threadIdx.x; j <= s.count; j += kBlock) {
    const int64_t o = s.offset(j), row = o - first;
    if (row > kTileRows) break;
    if (row >= 0 && row < kTileRows && j < s.count && s.offset(j + 1) > o)
      mark(marks.begin_bits, marks.begins, (int)row, j);
    if (row > 0 && j > 0 && s.offset(j - 1) < o) mark(marks.end_bits, marks.ends, (int)row - 1, j - 1);
  }
  __syncthreads();
}

struct Scan {
  const void *gate, *in, *grad_out, *states;  // grad_out and states: backwards
  int64_t gate_stride, in_stride, grad_out_stride, states_stride;
  int64_t rows, channels;
  int32_t complement;
  Sequences sequences;
  const float* initial;     // nullptr: zeros
  const float* grad_final;  // backwards
  int64_t initial_stride, grad_final_stride;
  void *out, *grad_in;      // backwards: out is the gate's gradient; each may be nullptr
  int64_t out_stride, grad_in_stride;
  float* last;              // the state that a sequence leaves; may be nullptr
  int64_t last_stride;
  uint32_t* tickets;        // nullptr: one tile of rows
  uint64_t* words;
  int64_t tiles;            // of rows
  uint32_t columns_of_tiles;
  bool wide;                // what a look-back asks at a time
  int64_t first_block;      // of this launch
};

// What a tile leaves for those behind it, two words a channel: {B, 1} and {A, 1 and its exponent} of
// its map, then {state behind it, 2} in the first, at once if it is a reset.
__device__ __forceinline__ uint64_t* words_of(const Scan& s, int64_t tile, uint32_t column) {
  return s.words + (tile * s.columns_of_tiles + column) * (kStateBytes / 8) +
         2 * (threadIdx.x & (kWaveSize - 1));
}
__device__ __forceinline__ void put_word(uint64_t* w, uint32_t flag, float v) {
  __hip_atomic_store(w, (uint64_t)flag << 32 | __builtin_bit_cast(uint32_t, v), __ATOMIC_RELAXED,
                     __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ uint64_t get_word(const uint64_t* w) {
  return __hip_atomic_load(w, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ float value_of(uint64_t w) {
  return __builtin_bit_cast(float, (uint32_t)w);
}
// (Of a tile's rows together less than 2^20, either way.)
__device__ __forceinline__ int32_t exponent_of(uint64_t w) { return (int32_t)(w >> 32) >> 1; }

// The state in front of a tile that is not the first, from up to WINDOW tiles in front.  (A wait ends
// all the same, with a NaN, if the words are another call's, to which the temp was given at the same time.)
template <int WINDOW>
__device__ __forceinline__ float walk_back(const Scan& s, int64_t tile, uint32_t column) {
  float h = __builtin_nanf("");
  for (uint32_t polls = 0; polls < kMostPolls; ++polls) {
    uint64_t low[WINDOW], high[WINDOW];
#pragma unroll
    for (int d = 0; d < WINDOW; ++d) {
      const int64_t front = tile - 1 - d;
      const uint64_t* w = words_of(s, front > 0 ? front : 0, column);
      low[d] = get_word(w);
      high[d] = get_word(w + 1);
    }
    int found = -1;  // the nearest tile whose state is known, all maps behind it being there
    bool whole = true;
#pragma unroll
    for (int d = 0; d < WINDOW; ++d) {
      if (whole && found < 0 && low[d] >> 32 == 2) found = d;
      whole = whole && low[d] >> 32 == 1 && high[d] >> 32 != 0;
    }
    if (__all(found >= 0)) {
#pragma unroll
      for (int d = WINDOW - 1; d >= 0; --d) {
        // (Tiles that end in a reset publish no map; what d > found makes is not used.)
        h = d == found ? value_of(low[d])
                       : fmaf(value_of(high[d]), __builtin_ldexpf(h, exponent_of(high[d])), value_of(low[d]));
      }
      break;
    }
    __builtin_amdgcn_s_sleep(1);
  }
  return h;
}

// The state in front of a tile, a channel a lane, by one wave.  The tiles in front have drawn
// their tickets before this one, so they run and publish, and no wait is long.
template <int WIDE>
__device__ __forceinline__ float look_back(const Scan& s, int64_t tile, uint32_t column, Map own) {
  uint64_t* mine = words_of(s, tile, column);
  float h = 0.0f;
  if (tile > 0) {
    if (is_reset(own.a)) {
      put_word(mine, 2, own.b);
    } else {
      put_word(mine + 1, (uint32_t)own.e << 1 | 1, own.a);
      put_word(mine, 1, own.b);
    }
    h = s.wide ? walk_back<WIDE>(s, tile, column) : walk_back<kWindow>(s, tile, column);
  }
  put_word(mine, 2, apply(own, h));
  return h;
}

template <typename T, int W, int R, bool BACK, bool SIGMOID, bool COMPLEMENT>
__global__ __launch_bounds__(kBlock, 2) void recurrence_kernel(Scan s) {
  constexpr int kGroups = groups_of<W>(), kTileRows = kGroups * R, kLanes = kTileChannels / W;
  constexpr int kWaveGroups = kGroups / kWaves;
  // (Backwards there are no registers for 16.)
  constexpr int kWide = BACK ? kWideWindow / 2 : kWideWindow;
  using V = typename Pack<T, W>::vec;
  using P = typename Pack<T, W>::type;
  // In LDS the k-th channels of all lanes lie side by side, and a row group begins a group's lanes further:
  // 64 lanes that read or write a word each meet 64 banks.  The scan goes by these places.  (Channels in their
  // order, us: gradients of 31744 x 4096 397 instead of 390.)
  __shared__ Map maps[kGroups][kTileChannels + kLanes];
  __shared__ Map wave_maps[kWaves][kTileChannels];
  __shared__ float wave_states[kWaves][kTileChannels];
  __shared__ Marks<kGroups, R> marks;
  __shared__ uint32_t ticket;

  const uint32_t column = (uint32_t)((s.first_block + blockIdx.x) % s.columns_of_tiles);
  int64_t tile = 0;
  if (s.tickets != nullptr) {
    if (threadIdx.x == 0)
      ticket = __hip_atomic_fetch_add(s.tickets + column * (kTicketBytes / 4), 1u,
                                      __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __syncthreads();
    tile = __builtin_amdgcn_readfirstlane(ticket);
    if (tile >= s.tiles) return;
  }
  const int64_t first = (BACK ? s.tiles - 1 - tile : tile) * kTileRows;
  const int lane = threadIdx.x % kLanes, group = threadIdx.x / kLanes;
  // This thread's channels: the last W of the row where it ends inside them, `skip` of which
  // are another thread's.
  const int64_t c = (int64_t)column * kTileChannels + lane * W;
  const int64_t at = c + W <= s.channels ? c : s.channels - W;
  const int skip = (int)(c - at < W ? c - at : W);
  // Its rows, in the order of the scan: the r-th is `origin` + r steps.
  constexpr int kStep = BACK ? -1 : 1;
  const int place = BACK ? kTileRows - 1 - group * R : group * R;  // of the first in the tile
  const int64_t origin = first + place;
  V gate[R], in[R], grad[BACK ? R : 1], before[BACK ? R : 1];
  if (first + kTileRows <= s.rows && (!BACK || first > 0)) {
    const T* gates = static_cast<const T*>(s.gate) + origin * s.gate_stride + at;
    const T* ins = static_cast<const T*>(s.in) + origin * s.in_stride + at;
    const T* grads = static_cast<const T*>(s.grad_out) + origin * s.grad_out_stride + at;
    const T* states = static_cast<const T*>(s.states) + (origin - 1) * s.states_stride + at;
#pragma unroll
    for (int r = 0; r < R; ++r) {
      gate[r] = *reinterpret_cast<const P*>(gates + kStep * r * s.gate_stride);
      in[r] = *reinterpret_cast<const P*>(ins + kStep * r * s.in_stride);
      if constexpr (BACK) {
        grad[r] = *reinterpret_cast<const P*>(grads + kStep * r * s.grad_out_stride);
        before[r] = *reinterpret_cast<const P*>(states + kStep * r * s.states_stride);
      }
    }
  } else {
#pragma unroll
    for (int r = 0; r < R; ++r) {
      int64_t row = origin + kStep * r;
      row = row < s.rows ? row : s.rows - 1;
      gate[r] = *reinterpret_cast<const P*>(static_cast<const T*>(s.gate) + row * s.gate_stride + at);
      in[r] = *reinterpret_cast<const P*>(static_cast<const T*>(s.in) + row * s.in_stride + at);
      if constexpr (BACK) {
        grad[r] = *reinterpret_cast<const P*>(static_cast<const T*>(s.grad_out) +
                                              row * s.grad_out_stride + at);
        before[r] = *reinterpret_cast<const P*>(static_cast<const T*>(s.states) +
                                                (row > 0 ? row - 1 : 0) * s.states_stride + at);
      }
    }
  }
  int64_t from, to;
  mark_rows<BACK>(s.sequences, first, s.rows, marks, &from, &to);
  // A bit a row: rows of sequences, rows that forget what comes in, and rows whose state is left.
  constexpr uint32_t kAll = R == 32 ? ~0u : (1u << R) - 1u;
  uint32_t there = kAll;
  if (first < from || first + kTileRows > to) {
    there = 0;
#pragma unroll
    for (int r = 0; r < R; ++r)
      if (origin + kStep * r >= from && origin + kStep * r < to) there |= 1u << r;
  }
  const uint32_t resets = (BACK ? marks.end_bits : marks.begin_bits)[group] & there;
  const uint32_t lasts = (BACK ? marks.begin_bits : marks.end_bits)[group] & there;
  const int32_t* reset_of = (BACK ? marks.ends : marks.begins) + place;
  const int32_t* last_of = (BACK ? marks.begins : marks.ends) + place;
  // Most waves have none of these, and go without what they ask for.
  const bool special = __any((resets | lasts | (there ^ kAll)) != 0);

  // What sequences begin with, in the order of the scan.
  const float* begin_state = BACK ? s.grad_final : s.initial;
  const int64_t begin_stride = BACK ? s.grad_final_stride : s.initial_stride;
  // Decays of the r-th row and what is left of them; its b (backwards: grad_out), of which what a sequence
  // begins with is a part.
  const auto decays = [&](int r, float (&a)[W], float (&left)[W]) {
#pragma unroll
    for (int k = 0; k < W; ++k) decay_of<T, SIGMOID>((float)gate[r][k], a[k], left[k]);
    if (!special) return;
    asm volatile("");  // (a branch: as selects, all rows would pay for it)
    if (!(there >> r & 1u)) {
#pragma unroll
      for (int k = 0; k < W; ++k) a[k] = 1.0f;
    }
  };
  const auto addends = [&](int r, const float (&a)[W], const float (&left)[W], float (&b)[W]) {
#pragma unroll
    for (int k = 0; k < W; ++k) {
      if (BACK) b[k] = (float)grad[BACK ? r : 0][k];
      else b[k] = COMPLEMENT ? left[k] * (float)in[r][k] : (float)in[r][k];
    }
    if (!special) return;
    asm volatile("");
    if ((resets >> r & 1u) != 0 && begin_state != nullptr) {
      float state[W];
      load_floats<float, W>(state, begin_state + reset_of[kStep * r] * begin_stride + at, W);
#pragma unroll
      for (int k = 0; k < W; ++k) b[k] = BACK ? b[k] + state[k] : fmaf(a[k], state[k], b[k]);
    }
    if (!(there >> r & 1u)) {
#pragma unroll
      for (int k = 0; k < W; ++k) b[k] = 0.0f;
    }
  };
  // What comes in to the r-th row is forgotten where a sequence begins.
  const auto forget = [&](int r, float (&h)[W]) {
    if (!special) return;
    asm volatile("");
    if (resets >> r & 1u) {
#pragma unroll
      for (int k = 0; k < W; ++k) h[k] = 0.0f;
    }
  };
  // What is made of a row stays in registers until the state in front of the tile is known; backwards,
  // where there is more of it, the decays are made again.  (b is not: what a sequence begins with may be
  // written over by what it leaves, once this tile's map is known.)
  constexpr int kHeld = BACK ? 1 : R;
  float held_a[kHeld][W], b[R][W];
  float own_a[W], h[W], largest = 0.0f;
#pragma unroll
  for (int k = 0; k < W; ++k) {
    own_a[k] = 1.0f;
    h[k] = 0.0f;
  }
#pragma unroll
  for (int r = 0; r < R; ++r) {
    float a[W], left[W];
    decays(r, a, left);
    addends(r, a, left, b[r]);
    forget(r, h);
#pragma unroll
    for (int k = 0; k < W; ++k) {
      h[k] = BACK ? a[k] * (b[r][k] + h[k]) : fmaf(a[k], h[k], b[r][k]);
      own_a[k] *= a[k];
      if (!SIGMOID) largest = fmaxf(largest, a[k]);
      if constexpr (!BACK) held_a[r][k] = a[k];
    }
    if (BACK) __builtin_amdgcn_sched_barrier(0);  // (rows side by side take more registers)
  }
  // Decays of up to 1 whose product is a normal number have not left float32 on the way.  (With the exponent
  // apart in every row, us: 65536 x 2048 211.1 instead of 209.8, gradients of 8192 x 1024 27.0 instead of 26.6.)
  bool left_range = largest > 1.0f;
#pragma unroll
  for (int k = 0; k < W; ++k) {
    left_range = left_range || !(own_a[k] >= kSmallestNormal);
    maps[group][k * kLanes + lane].b = h[k];
  }
  const auto put_decay = [&](int k, float a, int32_t e) {  // 2^e a, 1/2 <= a < 1
    Map& m = maps[group][k * kLanes + lane];
    m.a = resets != 0 ? -0.0f : 2.0f * a;
    m.e = e - 1;
  };
  if (__any(left_range && resets == 0)) {
    int32_t own_e[W];
#pragma unroll
    for (int k = 0; k < W; ++k) {
      own_a[k] = 0.5f;
      own_e[k] = 1;
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
      float a[W], left[W];
      if constexpr (BACK) keep(gate[r]);
      decays(r, a, left);
#pragma unroll
      for (int k = 0; k < W; ++k) multiply(own_a[k], own_e[k], a[k]);
      __builtin_amdgcn_sched_barrier(0);
    }
#pragma unroll
    for (int k = 0; k < W; ++k) put_decay(k, own_a[k], own_e[k]);
  } else {
#pragma unroll
    for (int k = 0; k < W; ++k)
      put_decay(k, __builtin_amdgcn_frexp_mantf(own_a[k]), __builtin_amdgcn_frexp_expf(own_a[k]));
  }
  if constexpr (BACK) {
#pragma unroll
    for (int r = 0; r < R; ++r) keep(gate[r]);
  }
  __syncthreads();
  // The maps in front of each group of a wave, then those in front of each wave.
  const int wave = threadIdx.x / kWaveSize, channel = threadIdx.x % kWaveSize;
  Map front{1.0f, 0.0f, 0};
#pragma unroll
  for (int g = 0; g < kWaveGroups; ++g) {
    const Map here = maps[wave * kWaveGroups + g][channel];
    maps[wave * kWaveGroups + g][channel] = front;
    front = behind(here, front);
  }
  wave_maps[wave][channel] = front;
  __syncthreads();
  if (wave == 0) {
    Map all = wave_maps[0][channel];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) all = behind(wave_maps[w][channel], all);
    float state = s.tickets != nullptr ? look_back<kWide>(s, tile, column, all) : 0.0f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      wave_states[w][channel] = state;
      state = apply(wave_maps[w][channel], state);
    }
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < W; ++k)
    h[k] = apply(maps[group][k * kLanes + lane], wave_states[wave][k * kLanes + lane]);

  const bool whole = s.channels % W == 0;
  const auto store = [&](void* to_, int64_t stride, int r, const float (&v)[W]) {
    T* p = static_cast<T*>(to_) + origin * stride + at + kStep * r * stride;
    if (whole || skip == 0) {
      V packed;
#pragma unroll
      for (int k = 0; k < W; ++k) packed[k] = (T)v[k];
      __builtin_nontemporal_store(packed, reinterpret_cast<P*>(p));
    } else {
#pragma unroll
      for (int k = 0; k < W; ++k)
        if (k >= skip) p[k] = (T)v[k];
    }
  };
  if (skip < W) {
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const bool mine = !special || (there >> r & 1u) != 0;
      forget(r, h);
      if constexpr (!BACK) {
#pragma unroll
        for (int k = 0; k < W; ++k) h[k] = fmaf(held_a[r][k], h[k], b[r][k]);
        if (mine) store(s.out, s.out_stride, r, h);
      } else {
        float a[W], left[W];
        decays(r, a, left);
        float of_gate[W], of_in[W], state[W];
#pragma unroll
        for (int k = 0; k < W; ++k) state[k] = (float)before[r][k];
        if (special) {
          asm volatile("");
          if (lasts >> r & 1u) {
#pragma unroll
            for (int k = 0; k < W; ++k)
              state[k] = s.initial != nullptr
                             ? s.initial[last_of[kStep * r] * s.initial_stride + at + k] : 0.0f;
          }
        }
#pragma unroll
        for (int k = 0; k < W; ++k) {
          const float reaches = b[r][k] + h[k];
          h[k] = a[k] * reaches;
          of_in[k] = COMPLEMENT ? reaches * left[k] : reaches;
          // (a G is the state that goes on; its slope has 1 - a for the other factor.)
          const float of_decay = COMPLEMENT ? state[k] - (float)in[r][k] : state[k];
          of_gate[k] = SIGMOID ? h[k] * left[k] * of_decay : h[k] * of_decay;
        }
        if (mine && s.out != nullptr) store(s.out, s.out_stride, r, of_gate);
        if (mine && s.grad_in != nullptr) store(s.grad_in, s.grad_in_stride, r, of_in);
      }
      if (BACK) __builtin_amdgcn_sched_barrier(0);
      if (special) {
        asm volatile("");
        if ((lasts >> r & 1u) != 0 && s.last != nullptr) {
          float* p = s.last + last_of[kStep * r] * s.last_stride + at;
#pragma unroll
          for (int k = 0; k < W; ++k)
            if (k >= skip) p[k] = h[k];
        }
      }
    }
  }
  // Sequences without rows leave what they begin with.
  if (s.last == nullptr || s.sequences.offsets == nullptr) return;
  for (int64_t i = tile * kBlock + threadIdx.x; i < s.sequences.count; i += s.tiles * kBlock) {
    if (s.sequences.offset(i + 1) > s.sequences.offset(i)) continue;
    for (int64_t k = (int64_t)column * kTileChannels;
         k < s.channels && k < (int64_t)(column + 1) * kTileChannels; ++k)
      s.last[i * s.last_stride + k] = begin_state != nullptr ? begin_state[i * begin_stride + k] : 0.0f;
  }
}

// One row for each sequence.
template <typename T, int W, bool SIGMOID>
__global__ __launch_bounds__(kBlock) void recurrence_step_kernel(Scan s) {
  const int64_t vectors = (s.channels + W - 1) / W, step = (int64_t)gridDim.x * kBlock;
  for (int64_t i = (int64_t)blockIdx.x * kBlock + threadIdx.x; i < s.rows * vectors; i += step) {
    const int64_t row = i / vectors, c = i % vectors * W, count = s.channels - c;
    float gate[W], in[W], h[W];
    load_floats<T, W>(gate, static_cast<const T*>(s.gate) + row * s.gate_stride + c, count);
    load_floats<T, W>(in, static_cast<const T*>(s.in) + row * s.in_stride + c, count);
    if (s.initial != nullptr) {
      load_floats<float, W>(h, s.initial + row * s.initial_stride + c, count);
    } else {
#pragma unroll
      for (int k = 0; k < W; ++k) h[k] = 0.0f;
    }
#pragma unroll
    for (int k = 0; k < W; ++k) {
      float a, left;
      decay_of<T, SIGMOID>(gate[k], a, left);
      h[k] = fmaf(a, h[k], s.complement ? left * in[k] : in[k]);
    }
    store_floats<T, W>(static_cast<T*>(s.out) + row * s.out_stride + c, h, count);
    if (s.last != nullptr) store_floats<float, W>(s.last + row * s.last_stride + c, h, count);
  }
}

// No rows at all: every sequence leaves what it begins with.
__global__ __launch_bounds__(kBlock) void recurrence_states_kernel(
    const float* from, int64_t from_stride, float* to, int64_t to_stride, int64_t sequences,
    int64_t channels) {
  const int64_t step = (int64_t)gridDim.x * kBlock;
  for (int64_t i = (int64_t)blockIdx.x * kBlock + threadIdx.x; i < sequences * channels; i += step) {
    const int64_t row = i / channels, c = i % channels;
    to[row * to_stride + c] = from != nullptr ? from[row * from_stride + c] : 0.0f;
  }
}

inline unsigned blocks_for_elements(int64_t threads) {
  const int64_t blocks = div_up(threads, kBlock);
  return (unsigned)(blocks < kMostBlocks ? blocks : kMostBlocks);
}

// Few columns of tiles that all run at once wait for the state to come through them: a look-back that
// asks more tiles at a time takes fewer turns.  (Window 4 and 16, us: 131072 x 64 101 and 59, 32768 x 512 36 and 31;
// but 65536 x 2048 208 and 213, 2000 x 512 11.2 and 11.9; backwards 4 and 8: 65536 x 64 101 and 75; all bfloat16.)
constexpr int kFewColumns = 8;
// Backwards, three tiles of four rows a thread or two of eight share a compute unit.  Eight rows are taken
// where they make one turn of a grid that four would not, and where the chain of tiles is long but one turn still holds
// it (us, 4 and 8: 8192 x 1024 28.6 and 26.7, 16384 x 512 32.7 and 27.7, 65536 x 64 75 and 43; but
// 4096 x 1024 18.3 and 20.7, 16384 x 768 41 and 45; all bfloat16).
constexpr int64_t kManyTiles = 128;

inline int64_t columns_of_tiles(int64_t channels) { return div_up(channels, kTileChannels); }

template <typename T, int W, int R, bool BACK, bool SIGMOID, bool COMPLEMENT>
int32_t launch_scan_tiles(hipStream_t stream, Scan s, void* temp) {
  s.tiles = div_up(s.rows, (int64_t)groups_of<W>() * R);
  s.columns_of_tiles = (uint32_t)columns_of_tiles(s.channels);
  if (s.tiles > 1) {
    char* base = reinterpret_cast<char*>(align_up((int64_t)(uintptr_t)temp, 128));
    const int64_t tickets = s.columns_of_tiles * kTicketBytes;
    s.tickets = reinterpret_cast<uint32_t*>(base);
    s.words = reinterpret_cast<uint64_t*>(base + tickets);
    const int32_t rc = launch_zero_words(
        stream, s.tickets, (tickets + s.tiles * s.columns_of_tiles * kStateBytes) / 4);
    if (rc != ILGPU_HIP_SUCCESS) return rc;
  }
  const int64_t blocks = s.tiles * s.columns_of_tiles;
  s.wide = s.columns_of_tiles <= kFewColumns && s.tiles > kWideWindow;
  for (s.first_block = 0; s.first_block < blocks; s.first_block += kMostBlocks) {
    const int64_t left = blocks - s.first_block;
    {
      ProfileScope scope(stream, BACK ? "recurrence_gradient" : "recurrence");
      hipLaunchKernelGGL((recurrence_kernel<T, W, R, BACK, SIGMOID, COMPLEMENT>),
                         dim3((unsigned)(left < kMostBlocks ? left : kMostBlocks)), dim3(kBlock), 0,
                         stream, s);
    }
    ILGPU_HIP_CHECK(hipGetLastError());
  }
  return ILGPU_HIP_SUCCESS;
}

template <bool BACK, bool SIGMOID, bool COMPLEMENT>
int32_t launch_scan_of(hipStream_t stream, int32_t type, const Scan& s, void* temp) {
  return with_type(type, [&](auto t) -> int32_t {
    using T = decltype(t);
    constexpr int W = 16 / sizeof(T), R = BACK ? kBackRows : kRows;
    if (!BACK && s.sequences.offsets == nullptr && s.sequences.length == 1) {
      {
        ProfileScope scope(stream, "recurrence_step");
        hipLaunchKernelGGL((recurrence_step_kernel<T, W, SIGMOID>),
                           dim3(blocks_for_elements(s.rows * div_up(s.channels, W))), dim3(kBlock),
                           0, stream, s);
      }
      ILGPU_HIP_CHECK(hipGetLastError());
      return ILGPU_HIP_SUCCESS;
    }
    // (A row shorter than a vector: an element a thread.)
    if (s.channels < W) return launch_scan_tiles<T, 1, R, BACK, SIGMOID, COMPLEMENT>(stream, s, temp);
    if constexpr (BACK) {
      const int64_t tiles = div_up(s.rows, (int64_t)groups_of<W>() * R);
      const int64_t blocks = tiles * columns_of_tiles(s.channels);
      if (blocks <= 4 * device_cu_count() &&
          (blocks > 3 * device_cu_count() || tiles >= kManyTiles))
        return launch_scan_tiles<T, W, kLongBackRows, BACK, SIGMOID, COMPLEMENT>(stream, s, temp);
    }
    return launch_scan_tiles<T, W, R, BACK, SIGMOID, COMPLEMENT>(stream, s, temp);
  });
}

template <bool BACK>
int32_t launch_scan(hipStream_t stream, int32_t type, int32_t decay, const Scan& s, void* temp) {
  if (s.rows == 0) {
    if (s.last == nullptr || s.sequences.count == 0) return ILGPU_HIP_SUCCESS;
    {
      ProfileScope scope(stream, "recurrence_states");
      hipLaunchKernelGGL(recurrence_states_kernel,
                         dim3(blocks_for_elements(s.sequences.count * s.channels)), dim3(kBlock), 0,
                         stream, BACK ? s.grad_final : s.initial,
                         BACK ? s.grad_final_stride : s.initial_stride, s.last, s.last_stride,
                         s.sequences.count, s.channels);
    }
    ILGPU_HIP_CHECK(hipGetLastError());
    return ILGPU_HIP_SUCCESS;
  }
  if (decay == ILGPU_HIP_DECAY_SIGMOID)
    return s.complement ? launch_scan_of<BACK, true, true>(stream, type, s, temp)
                        : launch_scan_of<BACK, true, false>(stream, type, s, temp);
  return s.complement ? launch_scan_of<BACK, false, true>(stream, type, s, temp)
                      : launch_scan_of<BACK, false, false>(stream, type, s, temp);
}

}  // namespace

// Tickets and words of the shortest tiles that such a call may take.
int64_t gated_recurrence_temp_bytes(int64_t rows, int64_t channels) {
  const int64_t tile_rows = (channels < 8 ? groups_of<1>() : groups_of<4>()) * kFewestRows;
  const int64_t tiles = div_up(rows, tile_rows);
  if (tiles <= 1) return 0;
  return 128 + columns_of_tiles(channels) * (kTicketBytes + tiles * kStateBytes);
}

int32_t launch_gated_recurrence(hipStream_t stream, const GatedRecurrenceArgs& a) {
  Scan s{};
  s.gate = a.gate;
  s.gate_stride = a.gate_stride;
  s.in = a.in;
  s.in_stride = a.in_stride;
  s.rows = a.rows;
  s.channels = a.channels;
  s.complement = a.complement;
  s.sequences = Sequences{a.offsets, a.offset_type == ILGPU_HIP_I64, a.sequences,
                          (uint32_t)(a.sequences > 0 ? a.rows / a.sequences : 0)};
  s.initial = a.initial;
  s.initial_stride = a.initial_stride;
  if (!a.backwards) {
    s.out = a.out;
    s.out_stride = a.out_stride;
    s.last = a.final_state;
    s.last_stride = a.final_stride;
    return launch_scan<false>(stream, a.type, a.decay, s, a.temp);
  }
  s.states = a.out;
  s.states_stride = a.out_stride;
  s.grad_out = a.grad_out;
  s.grad_out_stride = a.grad_out_stride;
  s.grad_final = a.grad_final;
  s.grad_final_stride = a.grad_final_stride;
  s.out = a.grad_gate;
  s.out_stride = a.grad_gate_stride;
  s.grad_in = a.grad_in;
  s.grad_in_stride = a.grad_in_stride;
  s.last = a.grad_initial;
  s.last_stride = a.grad_initial_stride;
  return launch_scan<true>(stream, a.type, a.decay, s, a.temp);
}

}  // namespace ilgpu_hip
