// Embedding lookup, out[i] = scale * table[tokens[i]], and its gradient,
// grad_table[v] = scale * sum of grad_out[i] over the positions of token v.
#include "elements.hpp"
#include "operators.hpp"

namespace ilgpu_hip {

namespace {

constexpr int kBlock = 256;
constexpr int64_t kMaxBlocks = 1 << 22;  // blocks go on to further rows beyond

// Lanes that share a row: a power of two, at most a block.
inline int lanes_log2(int64_t dimension, int width) {
  int log2 = 0;
  while ((1 << log2) < kBlock && ((int64_t)width << log2) < dimension) ++log2;
  return log2;
}
inline unsigned row_blocks(int64_t rows, int log2) {
  const int64_t blocks = div_up(rows, kBlock >> log2);
  return (unsigned)(blocks < kMaxBlocks ? blocks : kMaxBlocks);
}

template <typename TI, typename TO> struct Width {
  static constexpr int value = 16 / (sizeof(TI) > sizeof(TO) ? sizeof(TI) : sizeof(TO));
};

// U rows at a time for every group of lanes: their tokens, then all of their loads, are on
// their way together; rows go out past the caches, which the table's rows want.  A token
// outside the table reads its first row and stores zeros.
//
// 65536 x 4096 bfloat16 from 131072 rows, us: 143 (one row at a time 152, plain stores 151).
// 512 MiB are written and as much is asked for, a row of the table 3.4 times on average.  304 MiB
// of it pass the eight L2s, each of which fetches the frequent rows for itself; 151 are distinct
// and fit the last-level cache, so how much comes from HBM is not known.
constexpr int kRowsAtOnce = 4;
template <typename TI, typename TO, typename TT, int W, int U>
__global__ __launch_bounds__(kBlock) void embedding_kernel(
    const TI* __restrict__ table, int64_t vocabulary, int64_t dimension, int64_t table_stride,
    const TT* __restrict__ tokens, int64_t count, float scale, TO* __restrict__ out,
    int64_t out_stride, int log2) {
  using P = typename Pack<TI, W>::type;
  const int64_t rows = (int64_t)(kBlock >> log2) * U;
  const int64_t lane = threadIdx.x & ((1u << log2) - 1);
  for (int64_t i = blockIdx.x * rows + (threadIdx.x >> log2) * U; i < count;
       i += gridDim.x * rows) {
    const TI* from[U];
    bool there[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t token = (int64_t)tokens[i + u < count ? i + u : i];
      there[u] = (uint64_t)token < (uint64_t)vocabulary;
      from[u] = table + (there[u] ? token : 0) * table_stride;
    }
    for (int64_t c = lane * W; c < dimension; c += (int64_t)W << log2) {
      // The last thread of a row reads its last W columns and stores its own of them.
      const int64_t at = c + W <= dimension ? c : dimension - W;
      typename Pack<TI, W>::vec v[U] = {};
      if (vocabulary > 0) {
#pragma unroll
        for (int u = 0; u < U; ++u) v[u] = *reinterpret_cast<const P*>(from[u] + at);
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        typename Pack<TO, W>::vec r;
#pragma unroll
        for (int k = 0; k < W; ++k) r[k] = (TO)(there[u] ? product_for<TO>((float)v[u][k], scale) : 0.0f);
        TO* to = out + (i + u) * out_stride + at;
        if (i + u >= count) continue;
        if (at == c) {
          __builtin_nontemporal_store(r, reinterpret_cast<typename Pack<TO, W>::type*>(to));
        } else {
#pragma unroll
          for (int k = 0; k < W; ++k)
            if (at + k >= c) to[k] = r[k];
        }
      }
    }
  }
}

// ---- gradient -----------------------------------------------------------------
// Positions are brought into an order in which those of one token lie side by side
// (keys: their tokens, order: the positions; positions that count nowhere come last
// under the key `vocabulary`).  Chunks of kChunk positions of that order are added up
// by a wave each, whatever tokens they hold, so a token that fills half of the input
// takes no longer than the rest: a run of one token goes straight into the table where
// it ends before the next chunk does, parts of longer ones go into `parts` and are joined
// by a second kernel.  Rows of no token are cleared by further blocks of both and of the
// grouping.
constexpr int kChunk = 32, kShortChunk = 8;
// Few and narrow rows fill the chip only in short chunks: where long ones of 256 columns are
// fewer than this.
constexpr int64_t kFewChunks = 1024;
inline int64_t most_in_short_chunks(int64_t dimension) {
  return (kFewChunks - 1) / div_up(dimension, 256) * kChunk;
}
inline int chunk_length(int64_t count, int64_t dimension) {
  return count <= most_in_short_chunks(dimension) ? kShortChunk : kChunk;
}

// Sort keys of the positions: their tokens, `vocabulary` for those that count nowhere.
template <typename TT>
__global__ __launch_bounds__(kBlock) void token_keys_kernel(
    const TT* __restrict__ tokens, int64_t count, int64_t padded, int64_t vocabulary,
    int64_t padding_token, uint32_t* __restrict__ keys, uint32_t* __restrict__ crossings) {
  if (blockIdx.x == 0 && threadIdx.x == 0) crossings[0] = 0;
  for (int64_t i = (int64_t)blockIdx.x * kBlock + threadIdx.x; i < padded;
       i += (int64_t)gridDim.x * kBlock) {
    const int64_t token = i < count ? (int64_t)tokens[i] : -1;
    const bool counts = (uint64_t)token < (uint64_t)vocabulary && token != padding_token;
    keys[i] = (uint32_t)(counts ? token : vocabulary);
  }
}

// The same order for a moderate number of tokens in one launch instead of a sort's
// several: block g of `1 << log2` gathers the positions of the tokens that are g modulo
// the number of blocks.  Every block reads all tokens (from its XCD's L2) and counts
// those of the blocks before it, so it knows where its own begin without a word from
// them.  Sixteen waves take a stretch of the input each, keep the positions of their tokens
// and count them by (wave, token); the counts' prefix sums are the places.  Lanes of one LDS
// atomic are served in lane order (check_sort_device), so the order is the same in every
// call; it is not that of the positions, which no sum needs.  Bound by the vector units
// (some ten operations a token in every block): 65536 tokens 10 us, 16 where one token is 6 %
// of them and its block counts and places 3800.
constexpr int kGroupBlock = 1024;
constexpr int kGroupWaves = kGroupBlock / kWaveSize;
constexpr int kGroupMinLog2 = 8;          // blocks: one per compute unit
constexpr int kGroupMaxLog2 = 10;
constexpr int kGroupRows = 1024;          // most tokens a block gathers
// Places a wave remembers; beyond them it reads its tokens again.  (Two blocks of up to 2^17
// table rows fit a compute unit with 512.)
inline int group_list(int64_t count) { return count <= (1 << 16) ? 512 : 1024; }
constexpr int kGroupCountLog2 = 17;       // most tokens in all: place and row share a word
static_assert(((uint64_t)kGroupRows << kGroupCountLog2) <= (1ull << 32), "a word");

inline int group_log2(int64_t vocabulary) {
  int log2 = kGroupMinLog2;
  while (log2 < kGroupMaxLog2 && ((int64_t)kGroupRows << log2) < vocabulary) ++log2;
  return log2;
}
// Each block reads all tokens: with 256 blocks (up to 2^18 table rows) ahead of the sort up
// to 2^17 tokens, with more blocks up to as much fewer.  (Whole gradient into 131072 x 64, us,
// groups / sort: 8192 tokens 23 / 53, 32768 39 / 88, 131072 65 / 102, of 1000 rows 67 / 70; 2^18
// tokens, which overflow the waves' lists, 162 / 116.)
inline int64_t most_in_groups(int64_t vocabulary) {  // -1: not even none
  const int log2 = group_log2(vocabulary);
  if (vocabulary > ((int64_t)kGroupRows << log2)) return -1;
  return (int64_t)1 << (kGroupCountLog2 + kGroupMinLog2 - log2);
}
inline bool takes_groups(int64_t count, int64_t vocabulary) {
  return count <= most_in_groups(vocabulary);
}

// The table's last rows from `first` on, which further blocks of the grouping clear, met or
// not: the sums of those that are met come later.  In units of 16 bits, whatever the type.  As
// many bytes as are written while the grouping computes, whose blocks leave room for a second
// one on a compute unit (64 registers, of which tokens of 64 bits keep 28 bytes a lane in scratch,
// outside of loops; with more registers nothing is gained): 8192 tokens into 50021 x 1024 42.4 to
// 39.4 us, 65536 into 131072 x 2048 260 to 255.
constexpr int64_t kGroupClearBytes = 24 << 20, kGroupClearPerToken = 900;
struct Clearing {
  uint16_t* table;
  int64_t first, rows, columns, stride;
  int lanes_log2;
};

__device__ __forceinline__ void clear_all(const Clearing& t, uint32_t block, uint32_t blocks) {
  constexpr int W = 8;
  const typename Pack<uint16_t, W>::vec zeros = {};
  const int64_t at_once = kGroupBlock >> t.lanes_log2;
  for (int64_t r = t.first + block * at_once + (threadIdx.x >> t.lanes_log2); r < t.rows;
       r += blocks * at_once) {
    uint16_t* row = t.table + r * t.stride;
    for (int64_t c = (int64_t)(threadIdx.x & ((1u << t.lanes_log2) - 1)) * W; c < t.columns;
         c += (int64_t)W << t.lanes_log2) {
      if (c + W <= t.columns) {
        __builtin_nontemporal_store(zeros, reinterpret_cast<typename Pack<uint16_t, W>::type*>(row + c));
      } else {
        for (int64_t k = c; k < t.columns; ++k) row[k] = 0;
      }
    }
  }
}

// What a wave's lanes have written to LDS, its other lanes read from here on.  (The hardware
// runs a wave's LDS instructions in order; this keeps the compiler to it.)
__device__ __forceinline__ void wave_lds_fence() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

template <typename TT>
__global__ __launch_bounds__(kGroupBlock, 8) void group_tokens_kernel(
    const TT* __restrict__ tokens, int64_t count, int64_t padded, int64_t vocabulary,
    int64_t padding_token, int log2, int rows, uint32_t list_length, uint32_t* __restrict__ keys,
    uint32_t* __restrict__ order, uint64_t* __restrict__ met, uint32_t* __restrict__ crossings,
    Clearing clearing) {
  extern __shared__ uint32_t group_lds[];
  __shared__ uint32_t wave_rows[kGroupWaves], wave_below[kGroupWaves];
  const uint32_t group = blockIdx.x, groups = 1u << log2;
  if (group >= groups) {
    clear_all(clearing, group - groups, gridDim.x - groups);
    return;
  }
  const int wave = threadIdx.x / kWaveSize, lane = threadIdx.x & (kWaveSize - 1);
  uint32_t* const counters = group_lds + wave * rows;
  uint32_t* const list = group_lds + kGroupWaves * rows + wave * list_length;
  if (group == 0 && threadIdx.x == 0) crossings[0] = 0;
  for (int i = threadIdx.x; i < kGroupWaves * rows; i += kGroupBlock) group_lds[i] = 0;
  __syncthreads();

  constexpr int V = 4, U = 4;  // tokens a load, loads in flight
  constexpr int64_t kStep = (int64_t)kWaveSize * V * U;
  const int64_t stretch = (count + kGroupWaves * kStep - 1) / (kGroupWaves * kStep) * kStep;
  const int64_t begin = wave * stretch;
  const int64_t end = begin + stretch < count ? begin + stretch : count;
  const uint32_t limit = (uint32_t)vocabulary, mask = groups - 1;
  // (A padding token outside the table is none.)
  const uint32_t padding = (uint64_t)padding_token < (uint64_t)vocabulary ? (uint32_t)padding_token
                                                                          : 0xffffffffu;
  uint32_t below = 0, listed = 0;

  // Calls f(position, token, its block or none) for every position of the stretch, 64 lanes
  // at a time.
  const auto scan = [&](auto f) {
    for (int64_t base = begin; base < end; base += kStep) {
      TT t[U][V];
      const TT* from = tokens + base + lane * V;
      if (base + kStep <= end) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const auto r = *reinterpret_cast<const typename Pack<TT, V>::type*>(from + u * kWaveSize * V);
#pragma unroll
          for (int k = 0; k < V; ++k) t[u][k] = r[k];
        }
      } else {
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
          for (int k = 0; k < V; ++k)
            t[u][k] = base + (u * kWaveSize + lane) * V + k < end ? from[u * kWaveSize * V + k] : (TT)-1;
      }
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int k = 0; k < V; ++k) {
          const uint32_t token = (uint32_t)t[u][k];
          bool counts = token < limit && token != padding;
          if constexpr (sizeof(TT) == 8) counts = counts && (uint64_t)t[u][k] >> 32 == 0;
          f((uint32_t)base + (u * kWaveSize + lane) * V + k, token, counts ? token & mask : ~0u);
        }
    }
  };

  // One add for all lanes whose row is that of the first lane (a frequent token's, mostly:
  // 64 adds to one counter take as many cycles), one for each other lane; the counter
  // before the add and the lanes in front, or nothing.
  const auto count_row = [&](uint32_t row) {
    const uint64_t same = __builtin_amdgcn_ballot_w64(row == __builtin_amdgcn_readfirstlane(row));
    const bool mine = (same >> lane) & 1;
    const uint32_t before = mine ? mbcnt(same) : 0;
    uint32_t at = 0;
    if (before == 0) at = atomicAdd(&counters[row], mine ? (uint32_t)__popcll(same) : 1u);
    const uint32_t first = __builtin_amdgcn_readfirstlane(at);
    return mine ? first + before : at;
  };

  scan([&](uint32_t at, uint32_t token, uint32_t of) {
    below += __popcll(__builtin_amdgcn_ballot_w64(of < group));
    const uint64_t owns = __builtin_amdgcn_ballot_w64(of == group);
    if (owns != 0) {
      const uint32_t place = listed + mbcnt(owns);
      if (of == group && place < list_length) list[place] = (token >> log2) << kGroupCountLog2 | at;
      listed += __popcll(owns);
    }
  });
  wave_lds_fence();  // the list's entries go to other lanes
  if (listed <= list_length) {
    for (uint32_t j = lane; j < listed; j += kWaveSize) count_row(list[j] >> kGroupCountLog2);
  } else {
    scan([&](uint32_t, uint32_t token, uint32_t of) {
      if (of == group) count_row(token >> log2);
    });
  }
  if (lane == 0) wave_below[wave] = below;
  __syncthreads();

  // Places: by token, then by wave.
  uint32_t total = 0;
  if ((int)threadIdx.x < rows) {
    for (int w = 0; w < kGroupWaves; ++w) total += group_lds[w * rows + threadIdx.x];
  }
  const uint64_t any = __ballot(total > 0);
  if (lane == 0 && wave * kWaveSize < rows) met[(int64_t)wave * groups + group] = any;
  uint32_t before = total;
  for (int off = 1; off < kWaveSize; off <<= 1) {
    const uint32_t other = __shfl_up(before, off, kWaveSize);
    if (lane >= off) before += other;
  }
  if (lane == kWaveSize - 1) wave_rows[wave] = before;
  __syncthreads();
  uint32_t place = before - total, all_own = 0, all_below = 0;
  for (int w = 0; w < kGroupWaves; ++w) {
    if (w < wave) place += wave_rows[w];
    all_own += wave_rows[w];
    all_below += wave_below[w];
  }
  place += all_below;
  if ((int)threadIdx.x < rows) {
    for (int w = 0; w < kGroupWaves; ++w) {
      const uint32_t here = group_lds[w * rows + threadIdx.x];
      group_lds[w * rows + threadIdx.x] = place;
      place += here;
    }
  }
  __syncthreads();

  if (listed <= list_length) {
    for (uint32_t j = lane; j < listed; j += kWaveSize) {
      const uint32_t row = list[j] >> kGroupCountLog2;
      const uint32_t to = count_row(row);
      keys[to] = row << log2 | group;
      order[to] = list[j] & ((1u << kGroupCountLog2) - 1);
    }
  } else {
    scan([&](uint32_t at, uint32_t token, uint32_t of) {
      if (of == group) {
        const uint32_t to = count_row(token >> log2);
        keys[to] = token;
        order[to] = at;
      }
    });
  }
  if (group == groups - 1)
    for (int64_t i = (int64_t)all_below + all_own + threadIdx.x; i < padded; i += kGroupBlock)
      keys[i] = (uint32_t)vocabulary;
}

struct Sums {
  const uint64_t* met;   // bit (v >> group_log2) & 63 of word (v >> group_log2 >> 6, v modulo the
  int group_log2;        // groups): row v has a token; nullptr where the keys are sorted
  uint32_t* crossings;   // [0]: their number; then the chunks in which a run begins that
                         // goes on into the next
  float* parts;          // per chunk the part of a run from before it, then as many of
                         // runs that go on behind it
  int64_t count, chunks, part_stride;
  int64_t chunk;         // positions in one
  int64_t vocabulary, dimension;
  int64_t grad_stride, table_stride;
  float scale;
  int32_t accumulate;
  uint32_t slices;       // column slices of a row, in the sums and in the join
  uint32_t join_slices;
  uint32_t sum_blocks;   // blocks of the sums and of the join; further ones clear rows,
  uint32_t join_blocks;  // those from early_rows on beside the join
  int64_t early_rows, late_end;
  int32_t clear_rows;    // rows a block clears, lanes that share one
  int32_t clear_lanes_log2;
  int lanes_log2;        // lanes that share a row
  int join_lanes_log2;
};

// A thread's columns of a row, which begin at its `own`-th of W sums (0, or what the last
// columns of a row leave over), into the table.
template <typename TW, int W>
__device__ __forceinline__ void finish_row(TW* to, const float (&sum)[W], int own, float scale,
                                           int32_t accumulate) {
  float v[W];
  if (own == 0) {
    if (accumulate) {
      load_floats<TW, W>(v, to, W);
#pragma unroll
      for (int k = 0; k < W; ++k) v[k] = sum[k] * scale + v[k];
    } else {
#pragma unroll
      for (int k = 0; k < W; ++k) v[k] = product_for<TW>(sum[k], scale);
    }
    store_floats<TW, W>(to, v, W);
  } else {
#pragma unroll
    for (int k = 0; k < W; ++k)
      if (k >= own)
        to[k] = (TW)(accumulate ? sum[k] * scale + (float)to[k] : product_for<TW>(sum[k], scale));
  }
}

// Whether a row has a token: by its bit, or its key is among the sorted ones.
__device__ __forceinline__ bool is_met(const Sums& s, const uint32_t* __restrict__ keys,
                                       int64_t row) {
  if (s.met != nullptr) {
    const uint32_t of = (uint32_t)row & ((1u << s.group_log2) - 1), local = (uint32_t)(row >> s.group_log2);
    return (s.met[((uint64_t)(local >> 6) << s.group_log2) + of] >> (local & 63)) & 1;
  }
  int64_t low = 0, high = s.count;
  while (low < high) {
    const int64_t middle = (low + high) >> 1;
    if ((int64_t)keys[middle] < row) low = middle + 1;
    else high = middle;
  }
  return low < s.count && (int64_t)keys[low] == row;
}

// Clears the rows of no token in [begin, end): zeros, past the caches that the rows in use
// are in (8192 tokens into 50021 x 1024: 47.5 us, 54.7 with plain stores).  A block clears
// 8 KB, as many rows at a time as its threads cover; with longer stretches a block, more
// places are written at once (65536 tokens into 131072 x 2048: 259 us, 271 with 16 KB, 275
// with 32 KB), shorter ones are too many blocks (8192 into 50021 x 1024: 42.0, 44.5 with
// 4 KB).
constexpr int64_t kClearBytes = 8192;
template <typename TW>
__device__ __forceinline__ void clear_rows(const Sums& s, const uint32_t* __restrict__ keys,
                                           TW* __restrict__ table, int64_t begin, int64_t end,
                                           uint32_t block, uint32_t blocks) {
  constexpr int W = 16 / sizeof(TW);
  const int log2 = s.clear_lanes_log2;
  const typename Pack<TW, W>::vec zeros = {};
  for (int64_t first = begin + (int64_t)block * s.clear_rows; first < end;
       first += (int64_t)blocks * s.clear_rows) {
    for (int64_t r = first + (threadIdx.x >> log2); r < first + s.clear_rows && r < end;
         r += kBlock >> log2) {
      if (is_met(s, keys, r)) continue;
      TW* row = table + r * s.table_stride;
      for (int64_t c = (int64_t)(threadIdx.x & ((1u << log2) - 1)) * W; c < s.dimension;
           c += (int64_t)W << log2) {
        if (c + W <= s.dimension) {
          __builtin_nontemporal_store(zeros, reinterpret_cast<typename Pack<TW, W>::type*>(row + c));
        } else {
          for (int64_t k = c; k < s.dimension; ++k) row[k] = (TW)0.0f;
        }
      }
    }
  }
}

constexpr int64_t kLateBytes = 32 << 20;

// What becomes of a run's sum: a part of it is left for the join, it is the row, or it is
// the business of the chunk before, which reads on to the end of a run that begins in it and
// ends in the next.  Both know by the same two keys: a run over a chunk's border is short if
// it began in the chunk before the border and the key a chunk behind the border is another.
enum class Run { kPart, kOwn, kOther };

template <typename TG, typename TW, int W, int CHUNK, bool WHOLE_WAVE>
__device__ __forceinline__ void sum_chunk(const Sums& s, const uint32_t* __restrict__ keys,
                                          const uint32_t* __restrict__ order, uint32_t group,
                                          const TG* __restrict__ grad_out,
                                          TW* __restrict__ table) {
  using P = typename Pack<TG, W>::type;
  constexpr int U = WHOLE_WAVE && CHUNK > 8 ? 16 : 8;  // rows in flight
  const int log2 = WHOLE_WAVE ? 6 : s.lanes_log2;
  uint32_t chunk = group / s.slices;
  uint32_t slice = group - chunk * s.slices;
  if (WHOLE_WAVE) {
    chunk = __builtin_amdgcn_readfirstlane(chunk);
    slice = __builtin_amdgcn_readfirstlane(slice);
  }
  if (chunk >= s.chunks) return;
  const uint32_t lane = threadIdx.x & ((1u << log2) - 1);
  // The last thread of a row begins early enough for whole loads and leaves the columns of
  // the one before it alone; a thread beyond does the same for none (W >= dimension: see
  // the launch).
  const int64_t first = (((int64_t)slice << log2) + lane) * W;
  const int64_t c = first + W <= s.dimension ? first : s.dimension - W;
  const int own = (int)(first - c < W ? first - c : W);
  const uint32_t none = (uint32_t)s.vocabulary;
  const int64_t p0 = (int64_t)chunk * CHUNK;
  float* const head = s.parts + (int64_t)chunk * s.part_stride + first;
  float* const tail = head + s.chunks * s.part_stride;
  const auto store_part = [&](float* to, const float (&v)[W]) {
    if (own == 0) {
      store_floats<float, W>(to, v, W);
    } else {
#pragma unroll
      for (int k = 0; k < W; ++k)
        if (k >= own) to[k - own] = v[k];
    }
  };

  // The keys and positions of this chunk and of the next one, which a short run may reach: one
  // per lane where a whole wave shares a row, otherwise the batch that comes next, on its way
  // while one is added up (60696 tokens into 1024 x 64 half: these sums 17 us, 33 with loads when wanted).
  // keys and order go on for a chunk behind those.
  uint32_t lane_key = 0, lane_order = 0, next_key[U], next_order[U];
  const auto fetch = [&](int u0) {
    using Q = typename Pack<uint32_t, 4>::type;
#pragma unroll
    for (int u = 0; u < U; u += 4) {
      const Q k = *reinterpret_cast<const Q*>(keys + p0 + u0 + u);
      const Q o = *reinterpret_cast<const Q*>(order + p0 + u0 + u);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        next_key[u + i] = k[i];
        next_order[u + i] = o[i];
      }
    }
  };
  if (WHOLE_WAVE) {
    static_assert(2 * CHUNK <= kWaveSize, "a chunk and the next in a wave's lanes");
    lane_key = lane < 2 * CHUNK ? keys[p0 + lane] : none;
    lane_order = lane < 2 * CHUNK ? order[p0 + lane] : 0;
  } else {
    fetch(0);
  }
  // The keys around the chunk's borders.
  const uint32_t before = keys[p0 > 0 ? p0 - 1 : 0], far_before = keys[p0 > CHUNK ? p0 - CHUNK - 1 : 0];
  const uint32_t behind = keys[p0 + CHUNK], far_behind = keys[p0 + 2 * CHUNK];
  uint32_t run = WHOLE_WAVE ? __builtin_amdgcn_readlane(lane_key, 0) : next_key[0];
  if (run == none) return;
  const uint32_t some = WHOLE_WAVE ? __builtin_amdgcn_readlane(lane_order, 0) : next_order[0];
  Run what = Run::kOwn;
  if (p0 > 0 && run == before)
    what = (p0 > CHUNK && run == far_before) || run == behind ? Run::kPart : Run::kOther;
  const uint32_t other = what == Run::kOther ? run : none;
  float sum[W];
#pragma unroll
  for (int k = 0; k < W; ++k) sum[k] = 0.0f;
  bool extended = false;
  for (int u0 = 0;; u0 += U) {
    if (u0 == CHUNK) {
      const bool goes_on = behind == run;
      if (what == Run::kOwn && goes_on && far_behind != run) {
        extended = true;
      } else {
        if (what == Run::kOwn && !goes_on)
          finish_row<TW, W>(table + run * s.table_stride + c, sum, own, s.scale, s.accumulate);
        else if (what != Run::kOther)
          store_part(what == Run::kOwn ? tail : head, sum);
        if (what == Run::kOwn && goes_on && slice == 0 && lane == 0)
          s.crossings[1 + atomicAdd(s.crossings, 1u)] = chunk;
        return;
      }
    }
    if (u0 == 2 * CHUNK) {
      finish_row<TW, W>(table + run * s.table_stride + c, sum, own, s.scale, s.accumulate);
      return;
    }
    // Loads first, without a branch: positions that are not wanted read one that is.
    uint32_t key[U];
    typename Pack<TG, W>::vec v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      key[u] = WHOLE_WAVE ? __builtin_amdgcn_readlane(lane_key, u0 + u) : next_key[u];
      if (extended && key[u] != run) key[u] = none;
      const bool wanted = key[u] != none && key[u] != other;
      const uint32_t position = WHOLE_WAVE ? __builtin_amdgcn_readlane(lane_order, u0 + u) : next_order[u];
      const uint32_t at = wanted ? position : some;
      v[u] = *reinterpret_cast<const P*>(grad_out + at * s.grad_stride + c);
    }
    if (!WHOLE_WAVE) fetch(u0 + U);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (key[u] != run) {
        // The run ends here.
        if (what == Run::kOwn)
          finish_row<TW, W>(table + run * s.table_stride + c, sum, own, s.scale, s.accumulate);
        else if (what == Run::kPart)
          store_part(head, sum);
        if (key[u] == none) return;
#pragma unroll
        for (int k = 0; k < W; ++k) sum[k] = 0.0f;
        run = key[u];
        what = Run::kOwn;
      }
      // (Of a run that is another chunk's the sum is never used.)
#pragma unroll
      for (int k = 0; k < W; ++k) sum[k] += (float)v[u][k];
    }
  }
}

template <typename TG, typename TW, int W, int CHUNK, bool WHOLE_WAVE>
__global__ __launch_bounds__(kBlock) void embedding_gradient_kernel(
    Sums s, const uint32_t* __restrict__ keys, const uint32_t* __restrict__ order,
    const TG* __restrict__ grad_out, TW* __restrict__ table) {
  if (blockIdx.x >= s.sum_blocks) {
    clear_rows(s, keys, table, 0, s.early_rows, blockIdx.x - s.sum_blocks,
               gridDim.x - s.sum_blocks);
    return;
  }
  const int log2 = WHOLE_WAVE ? 6 : s.lanes_log2;
  const uint32_t group = (blockIdx.x << (8 - log2)) + (threadIdx.x >> log2);
  sum_chunk<TG, TW, W, CHUNK, WHOLE_WAVE>(s, keys, order, group, grad_out, table);
}

// The lanes of `inside` whose key is `row`, which differs between the groups of a wave. Any lane's
// key is read, so all lanes of the wave take part, also those whose row lies beyond the table.
__device__ __forceinline__ uint64_t positions_of(uint64_t inside, uint32_t key, uint32_t row) {
  uint64_t mine = 0;
  for (; inside != 0; inside &= inside - 1) {
    const int i = __builtin_ctzll(inside);
    if ((uint32_t)__builtin_amdgcn_readlane(key, i) == row) mine |= 1ull << i;
  }
  return mine;
}

// Up to 64 tokens, in one launch: every wave holds them all, one a lane, and each row of the
// table looks for its own among them.  So few tokens are bound by launches and by the clearing
// of the table (64 tokens, us, this / three launches: into 1000 x 64 5.9 / 13.0, into 30000 x
// 512 11.1 / 19.0, into 131072 x 1024 91 / 97; the worst, 64 times one token of 4096 columns,
// 19.7 / 14.7).
//
// Accumulated, only the tokens' rows are written, but the launch still has blocks for all rows
// (64 tokens, us, this / three launches: into 32768 x 1024 8.6 / 13.8, 49152 x 1024 11.3 / 13.7, 65536 x
// 1024 14.1 / 13.9, 131072 x 4096 52 / 13.7; 2^19 x 128 14.0 / 18.7, 2^19 x 256 26.1 / 18.3, 2^21 x 64 26.3 /
// 17.3): up to kFewBytes of table, more where the grouping takes more blocks or is a sort.
constexpr int64_t kFewTokens = kWaveSize;
constexpr int64_t kFewBytes = 192 << 20, kFewBytesOfManyRows = 320 << 20;
template <typename TG, typename TW, typename TT, int W>
__global__ __launch_bounds__(kBlock) void embedding_gradient_of_few_kernel(
    Sums s, const TT* __restrict__ tokens, int64_t padding_token, const TG* __restrict__ grad_out,
    TW* __restrict__ table) {
  constexpr int U = 8;  // rows in flight
  using P = typename Pack<TG, W>::type;
  const int lane = threadIdx.x & (kWaveSize - 1), log2 = s.clear_lanes_log2;
  const int64_t token = lane < s.count ? (int64_t)tokens[lane] : -1;
  const bool counts = (uint64_t)token < (uint64_t)s.vocabulary && token != padding_token;
  const uint32_t key = counts ? (uint32_t)token : 0xffffffffu;
  for (int64_t first = (int64_t)blockIdx.x * s.clear_rows; first < s.vocabulary;
       first += (int64_t)gridDim.x * s.clear_rows) {
    // The positions whose rows are among the block's.
    const uint64_t inside = __ballot(counts && key - (uint32_t)first < (uint32_t)s.clear_rows);
    if (inside == 0 && s.accumulate) continue;
    for (int64_t r0 = first; r0 < first + s.clear_rows && r0 < s.vocabulary; r0 += kBlock >> log2) {
      const int64_t r = r0 + (threadIdx.x >> log2);
      const uint64_t mine = inside == 0 ? 0 : positions_of(inside, key, (uint32_t)r);
      if (r >= s.vocabulary) continue;
      TW* const row = table + r * s.table_stride;
      for (int64_t c = (int64_t)(threadIdx.x & ((1u << log2) - 1)) * W; c < s.dimension;
           c += (int64_t)W << log2) {
        // (The last thread of a row: as in sum_chunk.)
        const int64_t at = c + W <= s.dimension ? c : s.dimension - W;
        float sum[W];
#pragma unroll
        for (int k = 0; k < W; ++k) sum[k] = 0.0f;
        for (uint64_t left = mine; left != 0;) {
          typename Pack<TG, W>::vec v[U];
          bool there[U];
#pragma unroll
          for (int u = 0; u < U; ++u) {
            there[u] = left != 0;
            const int i = __builtin_ctzll(there[u] ? left : mine);
            left &= left - 1;
            v[u] = *reinterpret_cast<const P*>(grad_out + i * s.grad_stride + at);
          }
#pragma unroll
          for (int u = 0; u < U; ++u)
#pragma unroll
            for (int k = 0; k < W; ++k) sum[k] += there[u] ? (float)v[u][k] : 0.0f;
        }
        if (mine != 0) {
          finish_row<TW, W>(row + at, sum, (int)(c - at), s.scale, s.accumulate);
        } else if (!s.accumulate) {
          if (at == c) {
            const typename Pack<TW, W>::vec zeros = {};
            __builtin_nontemporal_store(zeros, reinterpret_cast<typename Pack<TW, W>::type*>(row + c));
          } else {
            for (int64_t k = c; k < s.dimension; ++k) row[k] = (TW)0.0f;
          }
        }
      }
    }
  }
}

// Joins the parts of the long runs: the waves of a block take the parts in turn, of narrow rows
// several at a time, and their sums are added in the order of the waves.  The blocks behind clear
// rows.  (10^6 tokens into 1000 x 32 float, where one token has 3000 parts: 14 us; 29 with
// the run's end looked for 64 chunks at a time, 60 with one part a wave at a time too.)
constexpr int kJoinBlock = kBlock;
constexpr int kJoinBlocks = 2048;
constexpr int kJoinWaves = kJoinBlock / kWaveSize;

template <typename TW>
__global__ __launch_bounds__(kJoinBlock) void join_runs_kernel(
    Sums s, const uint32_t* __restrict__ keys, TW* __restrict__ table) {
  constexpr int W = 4;
  if (blockIdx.x >= s.join_blocks) {
    clear_rows(s, keys, table, s.early_rows, s.late_end, blockIdx.x - s.join_blocks,
               gridDim.x - s.join_blocks);
    return;
  }
  __shared__ float lds[kJoinWaves][kWaveSize * W];
  const uint32_t slices = s.join_slices;
  const int wave = threadIdx.x / kWaveSize, lane = threadIdx.x & (kWaveSize - 1);
  const int log2 = s.join_lanes_log2, at_once = kJoinBlock >> log2;  // parts
  const int part = threadIdx.x >> log2, column = lane & ((1 << log2) - 1);
  const uint32_t items = s.crossings[0] * slices;
  for (uint32_t item = blockIdx.x; item < items; item += s.join_blocks) {
    const int64_t chunk = s.crossings[1 + item / slices];
    const int64_t c = (((int64_t)(item % slices) << log2) + column) * W;
    const int64_t columns = s.dimension - c;  // a part's row is padded to whole loads
    const uint32_t run = keys[chunk * s.chunk + s.chunk - 1];
    // Chunks behind it that begin inside the run, as all do up to its end: 64 at a time, of long
    // runs then by 64 places among those that are left, 64 in the stretch between two of them...
    int64_t more = 0, left = s.chunks - chunk - 1, stretch = 1;
    while (left > 0) {
      const int64_t at = (lane + 1) * stretch - 1;
      const uint64_t inside = __ballot(at < left && keys[(chunk + 1 + more + (at < left ? at : 0)) * s.chunk] == run);
      const int found = inside == ~0ull ? kWaveSize : __builtin_ctzll(~inside);
      more += found * stretch;
      left -= found * stretch;
      if (found < kWaveSize && left > stretch - 1) left = stretch - 1;
      stretch = more < 4 * kWaveSize ? 1 : (left + kWaveSize - 1) / kWaveSize;
    }
    float sum[W];
#pragma unroll
    for (int k = 0; k < W; ++k) sum[k] = 0.0f;
    if (columns > 0) {
      const float* from = s.parts + (chunk + 1) * s.part_stride + c;
      if (part == 0) load_floats<float, W>(sum, s.parts + (s.chunks + chunk) * s.part_stride + c, W);
      constexpr int U = 8;  // in flight
      for (int64_t first = part; first < more; first += (int64_t)U * at_once) {
        float v[U][W];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int64_t j = first + u * at_once;
          load_floats<float, W>(v[u], from + (j < more ? j : first) * s.part_stride, W);
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
          for (int k = 0; k < W; ++k) sum[k] += first + u * at_once < more ? v[u][k] : 0.0f;
      }
    }
    for (int off = 1 << log2; off < kWaveSize; off <<= 1)
#pragma unroll
      for (int k = 0; k < W; ++k) sum[k] += __shfl_xor(sum[k], off, kWaveSize);
#pragma unroll
    for (int k = 0; k < W; ++k) lds[wave][lane * W + k] = sum[k];
    __syncthreads();
    if (part == 0) {
      for (int w = 1; w < kJoinWaves; ++w)
#pragma unroll
        for (int k = 0; k < W; ++k) sum[k] += lds[w][lane * W + k];
      TW* to = table + run * s.table_stride + c;
      if (columns >= W) {
        finish_row<TW, W>(to, sum, 0, s.scale, s.accumulate);
      } else {
#pragma unroll
        for (int k = 0; k < W; ++k)
          if (k < columns) {
            const float one[1] = {sum[k]};
            finish_row<TW, 1>(to + k, one, 0, s.scale, s.accumulate);
          }
      }
    }
    __syncthreads();
  }
}

struct GradientTemp {
  int64_t keys, order, met, crossings, parts, sort, bytes;  // offsets
  int64_t chunk, chunks, part_stride;
  int64_t padded;  // length of keys and order: whole chunks and the reach of the last one
};
GradientTemp gradient_temp(int64_t count, int64_t vocabulary, int64_t dimension) {
  GradientTemp t;
  const bool groups = takes_groups(count, vocabulary);
  t.chunk = chunk_length(count, dimension);
  t.chunks = div_up(count, t.chunk);
  t.part_stride = align_up(dimension, 8);
  t.keys = 0;
  t.padded = (t.chunks + 2) * t.chunk;
  t.order = align_up(t.padded * 4, 256);
  t.met = t.order + align_up(t.padded * 4, 256);
  t.crossings =
      t.met + (groups ? (div_up(vocabulary, (int64_t)64 << group_log2(vocabulary)) * 8)
                            << group_log2(vocabulary)
                      : 0);
  t.parts = t.crossings + align_up((t.chunks + 1) * 4, 256);
  t.sort = t.parts + align_up(2 * t.chunks * t.part_stride * 4, 256);
  t.bytes = t.sort + (count > 0 && !groups ? radix_sort_temp_bytes(count, 4, 4) : 0) + 256;
  return t;
}

}  // namespace

int32_t launch_embedding(hipStream_t stream, const EmbeddingArgs& a) {
  if (a.count == 0) return ILGPU_HIP_SUCCESS;
  return with_type(a.table_type, [&](auto ti) {
    return with_type(a.out_type, [&](auto to) {
      return with_token_type(a.token_type, [&](auto tt) -> int32_t {
        using TI = decltype(ti);
        using TO = decltype(to);
        using TT = decltype(tt);
        constexpr int kWide = Width<TI, TO>::value;
        const int W = a.dimension >= kWide ? kWide : 1;
        const int log2 = lanes_log2(a.dimension, W);
        // Four rows at a time where that still leaves every compute unit its blocks.
        const bool four = div_up(a.count, kBlock >> log2) >= (int64_t)device_cu_count() * 32;
        const auto kernel_of = [&](auto u) {
          constexpr int U = decltype(u)::value;
          return W == 1 ? embedding_kernel<TI, TO, TT, 1, U>
                        : embedding_kernel<TI, TO, TT, kWide, U>;
        };
        auto kernel = four ? kernel_of(std::integral_constant<int, kRowsAtOnce>())
                           : kernel_of(std::integral_constant<int, 1>());
        const int64_t rows = four ? div_up(a.count, kRowsAtOnce) : a.count;
        {
          ProfileScope scope(stream, "embedding");
          hipLaunchKernelGGL(kernel, dim3(row_blocks(rows, log2)), dim3(kBlock), 0, stream,
                             static_cast<const TI*>(a.table), a.vocabulary, a.dimension,
                             a.table_stride, static_cast<const TT*>(a.tokens), a.count, a.scale,
                             static_cast<TO*>(a.out), a.out_stride, log2);
        }
        ILGPU_HIP_CHECK(hipGetLastError());
        return ILGPU_HIP_SUCCESS;
      });
    });
  });
}

static Sums sums_of(const EmbeddingGradientArgs& a) {
  Sums s{};
  s.count = a.count;
  s.vocabulary = a.vocabulary;
  s.dimension = a.dimension;
  s.grad_stride = a.grad_out_stride;
  s.table_stride = a.table_stride;
  s.scale = a.scale;
  s.accumulate = a.accumulate;
  return s;
}
// A block's rows of about kClearBytes, and the lanes that share one.
template <typename TW> static void set_clear_shape(Sums& s, int width) {
  s.clear_lanes_log2 = lanes_log2(s.dimension, width);
  s.clear_rows = kBlock >> s.clear_lanes_log2;
  while (2 * s.clear_rows * s.dimension * (int64_t)sizeof(TW) <= kClearBytes) s.clear_rows *= 2;
}
// Blocks that clear `rows` rows.
static int64_t clear_blocks(const Sums& s, int64_t rows) {
  const int64_t blocks = div_up(rows, s.clear_rows);
  return blocks < kMaxBlocks ? blocks : kMaxBlocks;
}

static int32_t launch_gradient_of_few(hipStream_t stream, const EmbeddingGradientArgs& a) {
  return with_type(a.grad_out_type, [&](auto tg) {
    return with_type(a.table_type, [&](auto tw) {
      return with_token_type(a.token_type, [&](auto tt) -> int32_t {
        using TG = decltype(tg);
        using TW = decltype(tw);
        using TT = decltype(tt);
        constexpr int kWide = Width<TG, TW>::value;
        const int W = a.dimension >= kWide ? kWide : 1;
        Sums s = sums_of(a);
        set_clear_shape<TW>(s, W);
        {
          ProfileScope scope(stream, "embedding_gradient_of_few");
          hipLaunchKernelGGL((W == 1 ? embedding_gradient_of_few_kernel<TG, TW, TT, 1>
                                     : embedding_gradient_of_few_kernel<TG, TW, TT, kWide>),
                             dim3((unsigned)clear_blocks(s, a.vocabulary)), dim3(kBlock), 0, stream,
                             s, static_cast<const TT*>(a.tokens), a.padding_token,
                             static_cast<const TG*>(a.grad_out), static_cast<TW*>(a.grad_table));
        }
        ILGPU_HIP_CHECK(hipGetLastError());
        return ILGPU_HIP_SUCCESS;
      });
    });
  });
}

static bool takes_one_launch(const EmbeddingGradientArgs& a) {
  if (a.count > kFewTokens || !a.accumulate) return a.count <= kFewTokens;
  const int64_t most = group_log2(a.vocabulary) > kGroupMinLog2 ? kFewBytesOfManyRows : kFewBytes;
  return a.vocabulary <= most / (a.dimension * operator_elem_size(a.table_type));
}

// Whether the sums' launch, with the blocks that clear rows, has fewer threads than a grid can
// hold (2^32) and its items fit their 32 bits: not so only where there are more than 12.5 million
// blocks of sums, whose parts take more than 50 GB.
static bool grid_holds(const GradientTemp& t, const EmbeddingGradientArgs& a) {
  const int gb = operator_elem_size(a.grad_out_type), wb = operator_elem_size(a.table_type);
  const int wide = 16 / (gb > wb ? gb : wb), W = a.dimension >= wide ? wide : 1;
  const int all_log2 = lanes_log2(a.dimension, W), log2 = all_log2 < 6 ? all_log2 : 6;
  const int64_t blocks = div_up(t.chunks * div_up(a.dimension, (int64_t)W << log2), kBlock >> log2);
  return blocks + kMaxBlocks < (INT64_C(1) << 32) / kBlock &&
         t.chunks * div_up(a.dimension, kWaveSize * 4) <= INT32_MAX;
}

// What `count` tokens need, or fewer: a program keeps one temp for batches of any length up to a
// largest.  The layout grows with the tokens but for two steps back: long chunks leave a quarter
// of the parts, and sorted tokens no bits of met rows.
int64_t embedding_gradient_temp_bytes(int64_t count, int64_t vocabulary, int64_t dimension) {
  int64_t bytes = gradient_temp(count, vocabulary, dimension).bytes;
  for (const int64_t last : {most_in_short_chunks(dimension), most_in_groups(vocabulary)}) {
    if (last < 0 || last >= count) continue;
    const int64_t there = gradient_temp(last, vocabulary, dimension).bytes;
    if (there > bytes) bytes = there;
  }
  return bytes;
}

int32_t launch_embedding_gradient(hipStream_t stream, const EmbeddingGradientArgs& a) {
  if (a.vocabulary == 0) return ILGPU_HIP_SUCCESS;
  const GradientTemp t = gradient_temp(a.count, a.vocabulary, a.dimension);
  if (!grid_holds(t, a)) return ILGPU_HIP_ERROR_NOT_SUPPORTED;
  if (a.count > 0) {
    const int32_t rc = check_sort_device(stream);  // before anything is launched
    if (rc != ILGPU_HIP_SUCCESS) return rc;
  }
  if (takes_one_launch(a)) return launch_gradient_of_few(stream, a);
  char* base = reinterpret_cast<char*>(align_up((int64_t)(uintptr_t)a.temp, 256));
  uint32_t* keys = reinterpret_cast<uint32_t*>(base + t.keys);
  uint32_t* order = reinterpret_cast<uint32_t*>(base + t.order);
  uint32_t* crossings = reinterpret_cast<uint32_t*>(base + t.crossings);
  const bool groups = a.count > 0 && takes_groups(a.count, a.vocabulary);
  int64_t rows_left = a.vocabulary;  // in front of those that are cleared beside the grouping
  unsigned clearing_blocks = 0;
  Clearing clearing{};
  if (groups && !a.accumulate) {
    const int64_t units = operator_elem_size(a.table_type) / 2;
    clearing = {static_cast<uint16_t*>(a.grad_table), 0, a.vocabulary, a.dimension * units,
                a.table_stride * units, 0};
    while ((1 << clearing.lanes_log2) < kGroupBlock && (8 << clearing.lanes_log2) < clearing.columns)
      ++clearing.lanes_log2;
    const int64_t some = (kGroupClearBytes + a.count * kGroupClearPerToken) / (clearing.columns * 2);
    rows_left = a.vocabulary > some ? a.vocabulary - some : 0;
    clearing.first = rows_left;
    const int64_t blocks =
        div_up(a.vocabulary - rows_left, kGroupBlock >> clearing.lanes_log2);
    clearing_blocks = (unsigned)(blocks < kMaxBlocks / 8 ? blocks : kMaxBlocks / 8);
  }
  if (groups) {
    const int32_t rc = with_token_type(a.token_type, [&](auto tt) -> int32_t {
      using TT = decltype(tt);
      const int log2 = group_log2(a.vocabulary);
      const int rows = (int)div_up(a.vocabulary, (int64_t)1 << log2), list = group_list(a.count);
      {
        ProfileScope scope(stream, "embedding_group_tokens");
        hipLaunchKernelGGL((group_tokens_kernel<TT>), dim3((1u << log2) + clearing_blocks),
                           dim3(kGroupBlock), (unsigned)(kGroupWaves * (rows + list) * 4), stream,
                           static_cast<const TT*>(a.tokens), a.count, t.padded, a.vocabulary,
                           a.padding_token, log2, rows, (uint32_t)list, keys, order,
                           reinterpret_cast<uint64_t*>(base + t.met), crossings, clearing);
      }
      ILGPU_HIP_CHECK(hipGetLastError());
      return ILGPU_HIP_SUCCESS;
    });
    if (rc != ILGPU_HIP_SUCCESS) return rc;
  } else if (a.count > 0) {
    const int32_t rc = with_token_type(a.token_type, [&](auto tt) -> int32_t {
      using TT = decltype(tt);
      const int64_t blocks = div_up(t.padded, kBlock);
      {
        ProfileScope scope(stream, "embedding_token_keys");
        hipLaunchKernelGGL((token_keys_kernel<TT>),
                           dim3((unsigned)(blocks < kMaxBlocks ? blocks : kMaxBlocks)),
                           dim3(kBlock), 0, stream, static_cast<const TT*>(a.tokens), a.count,
                           t.padded, a.vocabulary, a.padding_token, keys, crossings);
      }
      ILGPU_HIP_CHECK(hipGetLastError());
      return ILGPU_HIP_SUCCESS;
    });
    if (rc != ILGPU_HIP_SUCCESS) return rc;
    const SortArgs sort{keys, order, 1, 1, a.count, ILGPU_HIP_U32, 4, 0,
                        ILGPU_HIP_VALUES_FROM_INDEX, base + t.sort};
    const int32_t sorted = launch_radix_sort(stream, sort);
    if (sorted != ILGPU_HIP_SUCCESS) return sorted;
  }
  return with_type(a.grad_out_type, [&](auto tg) {
    return with_type(a.table_type, [&](auto tw) -> int32_t {
      using TG = decltype(tg);
      using TW = decltype(tw);
      constexpr int kWide = Width<TG, TW>::value;
      const int W = a.dimension >= kWide ? kWide : 1;  // a thread's columns
      TW* table = static_cast<TW*>(a.grad_table);
      const int all_log2 = lanes_log2(a.dimension, W);
      const int log2 = all_log2 < 6 ? all_log2 : 6;
      const int64_t slices = div_up(a.dimension, (int64_t)W << log2);
      const int join_log2 = lanes_log2(a.dimension, 4) < 6 ? lanes_log2(a.dimension, 4) : 6;
      const int64_t join_slices = div_up(a.dimension, kWaveSize * 4);
      const int64_t sum_blocks = div_up(t.chunks * slices, kBlock >> log2);
      const int64_t items = t.chunks > 2 ? (t.chunks - 2) * join_slices : 0;
      const int64_t join_blocks = items < kJoinBlocks ? items : kJoinBlocks;
      Sums s = sums_of(a);
      s.met = groups ? reinterpret_cast<const uint64_t*>(base + t.met) : nullptr;
      s.group_log2 = group_log2(a.vocabulary);
      s.crossings = crossings;
      s.parts = reinterpret_cast<float*>(base + t.parts);
      s.chunks = t.chunks;
      s.part_stride = t.part_stride;
      s.chunk = t.chunk;
      s.slices = (uint32_t)slices;
      s.join_slices = (uint32_t)join_slices;
      s.sum_blocks = (uint32_t)sum_blocks;
      s.join_blocks = (uint32_t)join_blocks;
      s.lanes_log2 = log2;
      s.join_lanes_log2 = join_log2;
      set_clear_shape<TW>(s, 16 / sizeof(TW));
      // Rows cleared beside the join are as many as it has time for while it waits for its
      // own reads; those before them keep the memory busy while the sums wait for theirs
      // (8192 tokens into 50021 x 1024: 43.6 us, 46.9 with all of them beside the sums, 56.9
      // with all beside the join).
      const int64_t late = kLateBytes / ((int64_t)sizeof(TW) * a.dimension);
      s.late_end = rows_left;
      if (!a.accumulate && s.late_end > late)
        s.early_rows = (s.late_end - late) / s.clear_rows * s.clear_rows;
      const int64_t early_blocks = clear_blocks(s, s.early_rows);
      const int64_t late_blocks = a.accumulate ? 0 : clear_blocks(s, s.late_end - s.early_rows);
      if (sum_blocks + early_blocks > 0) {
        ProfileScope scope(stream, "embedding_gradient");
        const auto kernel_of = [&](auto chunk) {
          constexpr int C = decltype(chunk)::value;
          return W == 1      ? embedding_gradient_kernel<TG, TW, 1, C, false>
                 : log2 == 6 ? embedding_gradient_kernel<TG, TW, kWide, C, true>
                             : embedding_gradient_kernel<TG, TW, kWide, C, false>;
        };
        auto kernel = t.chunk == kChunk ? kernel_of(std::integral_constant<int, kChunk>())
                                        : kernel_of(std::integral_constant<int, kShortChunk>());
        hipLaunchKernelGGL(kernel, dim3((unsigned)(sum_blocks + early_blocks)), dim3(kBlock), 0,
                           stream, s, keys, order, static_cast<const TG*>(a.grad_out), table);
      }
      ILGPU_HIP_CHECK(hipGetLastError());
      if (join_blocks + late_blocks > 0) {
        ProfileScope scope(stream, "embedding_gradient_rest");
        hipLaunchKernelGGL((join_runs_kernel<TW>), dim3((unsigned)(join_blocks + late_blocks)),
                           dim3(kJoinBlock), 0, stream, s, keys, table);
      }
      ILGPU_HIP_CHECK(hipGetLastError());
      return ILGPU_HIP_SUCCESS;
    });
  });
}

}  // namespace ilgpu_hip
