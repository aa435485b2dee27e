// Embedding lookup, out[i] = scale * table[tokens[i]], and its gradient,
// grad_table[v] = scale * sum of grad_out[i] over the positions of token v.
#include "elements.hpp"
#include "kernels.hpp"

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

template <typename TI, typename TO, typename TT>
__global__ __launch_bounds__(kBlock) void embedding_kernel(
    const TI* __restrict__ table, int64_t vocabulary, int64_t dimension, int64_t table_stride,
    const TT* __restrict__ tokens, int64_t count, float scale, TO* __restrict__ out,
    int64_t out_stride, int log2) {
  constexpr int W = Width<TI, TO>::value;
  const int64_t rows_per_block = kBlock >> log2;
  const int64_t first = (int64_t)(threadIdx.x & ((1u << log2) - 1)) * W;
  for (int64_t i = blockIdx.x * rows_per_block + (threadIdx.x >> log2); i < count;
       i += gridDim.x * rows_per_block) {
    const int64_t token = (int64_t)tokens[i];
    const bool there = (uint64_t)token < (uint64_t)vocabulary;
    const TI* from = table + (there ? token : 0) * table_stride;
    TO* to = out + i * out_stride;
    for (int64_t c = first; c < dimension; c += (int64_t)W << log2) {
      float v[W];
      load_floats<TI, W>(v, from + c, there ? dimension - c : 0);
#pragma unroll
      for (int k = 0; k < W; ++k) v[k] = there ? v[k] * scale : 0.0f;
      store_floats<TO, W>(to + c, v, dimension - c);
    }
  }
}

// ---- gradient -----------------------------------------------------------------
// Positions are brought into an order in which those of one token lie side by side
// (keys: their tokens, order: the positions; positions that count nowhere come last
// under the key `vocabulary`).  Chunks of kChunk positions of that order are added up
// by a wave each, whatever tokens they hold, so a token that fills half of the input
// takes no longer than the rest: a run of one token inside a chunk goes straight into
// the table, the parts of a run that crosses chunks go into `parts` and are joined by
// a second kernel.  Rows of no token are cleared by further blocks of the first.
constexpr int kChunk = 32;

// Sort keys of the positions: their tokens, `vocabulary` for those that count nowhere.
template <typename TT>
__global__ __launch_bounds__(kBlock) void token_keys_kernel(
    const TT* __restrict__ tokens, int64_t count, int64_t vocabulary, int64_t padding_token,
    uint32_t* __restrict__ keys, uint32_t* __restrict__ crossings) {
  if (blockIdx.x == 0 && threadIdx.x == 0) crossings[0] = 0;
  for (int64_t i = (int64_t)blockIdx.x * kBlock + threadIdx.x; i < count;
       i += (int64_t)gridDim.x * kBlock) {
    const int64_t token = (int64_t)tokens[i];
    const bool counts = (uint64_t)token < (uint64_t)vocabulary && token != padding_token;
    keys[i] = (uint32_t)(counts ? token : vocabulary);
  }
}

// The same order for a moderate number of tokens in one launch instead of a sort's
// several: block g of `1 << log2` gathers the positions of the tokens that are g modulo
// the number of blocks.  Every block reads all tokens (from its XCD's L2) and counts
// those of the blocks before it, so it knows where its own begin without a word from
// them.  Sixteen waves take a stretch of the input each, and count their tokens by
// (wave, token); the counts' prefix sums are the places.  Lanes of one LDS atomic are
// served in lane order (check_sort_device), so the order is the same in every call; it is
// not that of the positions, which no sum needs.
constexpr int kGroupBlock = 1024;
constexpr int kGroupWaves = kGroupBlock / kWaveSize;
constexpr int kGroupMinLog2 = 8;          // blocks: one per compute unit
constexpr int kGroupMaxLog2 = 10;
constexpr int kGroupRows = 1024;          // most tokens a block gathers
constexpr int kGroupList = 512;           // positions a wave remembers; beyond it reads again
constexpr int64_t kGroupMaxCount = 1 << 18;

inline int group_log2(int64_t vocabulary) {
  int log2 = kGroupMinLog2;
  while (log2 < kGroupMaxLog2 && ((int64_t)kGroupRows << log2) < vocabulary) ++log2;
  return log2;
}
inline bool takes_groups(int64_t count, int64_t vocabulary) {
  return count <= kGroupMaxCount && vocabulary <= ((int64_t)kGroupRows << kGroupMaxLog2);
}

template <typename TT>
__global__ __launch_bounds__(kGroupBlock) void group_tokens_kernel(
    const TT* __restrict__ tokens, int64_t count, int64_t vocabulary, int64_t padding_token,
    int log2, int rows, uint32_t* __restrict__ keys, uint32_t* __restrict__ order,
    uint64_t* __restrict__ met, uint32_t* __restrict__ crossings) {
  extern __shared__ uint32_t group_lds[];
  __shared__ uint32_t wave_rows[kGroupWaves], wave_below[kGroupWaves];
  const uint32_t group = blockIdx.x, groups = gridDim.x;
  const int wave = threadIdx.x / kWaveSize, lane = threadIdx.x & (kWaveSize - 1);
  uint32_t* const counters = group_lds + wave * rows;
  uint32_t* const list = group_lds + kGroupWaves * rows + wave * kGroupList;
  if (group == 0 && threadIdx.x == 0) crossings[0] = 0;
  for (int i = threadIdx.x; i < kGroupWaves * rows; i += kGroupBlock) group_lds[i] = 0;
  __syncthreads();

  constexpr int V = 4, U = 4;  // tokens a load, loads in flight
  constexpr int64_t kStep = (int64_t)kWaveSize * V * U;
  const int64_t stretch = (count + kGroupWaves * kStep - 1) / (kGroupWaves * kStep) * kStep;
  const int64_t begin = wave * stretch;
  const int64_t end = begin + stretch < count ? begin + stretch : count;
  uint32_t below = 0, listed = 0;

  // Calls f(position, token, own) for every position of the stretch, 64 lanes at a time.
  auto scan = [&](auto f) {
    for (int64_t base = begin; base < end; base += kStep) {
      TT t[U][V];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int64_t at = base + (u * kWaveSize + lane) * V;
        if (at + V <= end) {
          const auto r = *reinterpret_cast<const typename Pack<TT, V>::type*>(tokens + at);
#pragma unroll
          for (int k = 0; k < V; ++k) t[u][k] = r[k];
        } else {
#pragma unroll
          for (int k = 0; k < V; ++k) t[u][k] = at + k < end ? tokens[at + k] : (TT)-1;
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int k = 0; k < V; ++k) {
          const int64_t token = (int64_t)t[u][k];
          f((uint32_t)(base + (u * kWaveSize + lane) * V + k), (uint32_t)token,
            (uint64_t)token < (uint64_t)vocabulary && token != padding_token);
        }
    }
  };

  scan([&](uint32_t at, uint32_t token, bool counts) {
    const uint32_t of = token & (groups - 1);
    below += counts && of < group ? 1 : 0;
    const bool own = counts && of == group;
    const uint64_t owns = __ballot(own);
    if (owns != 0) {
      if (own) {
        atomicAdd(&counters[token >> log2], 1u);
        const uint32_t place = listed + mbcnt(owns);
        if (place < kGroupList) list[place] = at;
      }
      listed += __popcll(owns);
    }
  });
  for (int off = kWaveSize / 2; off > 0; off >>= 1) below += __shfl_xor(below, off, kWaveSize);
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

  if (listed <= kGroupList) {
    for (uint32_t j = lane; j < listed; j += kWaveSize) {
      const uint32_t at = list[j], token = (uint32_t)tokens[at];
      const uint32_t to = atomicAdd(&counters[token >> log2], 1u);
      keys[to] = token;
      order[to] = at;
    }
  } else {
    scan([&](uint32_t at, uint32_t token, bool counts) {
      if (counts && (token & (groups - 1)) == group) {
        const uint32_t to = atomicAdd(&counters[token >> log2], 1u);
        keys[to] = token;
        order[to] = at;
      }
    });
  }
  if (group == groups - 1)
    for (int64_t i = (int64_t)all_below + all_own + threadIdx.x; i < count; i += kGroupBlock)
      keys[i] = (uint32_t)vocabulary;
}

struct Sums {
  const uint32_t* keys;
  const uint32_t* order;
  const uint64_t* met;   // bit (v >> group_log2) & 63 of word (v >> group_log2 >> 6, v modulo the
  int group_log2;        // groups): row v has a token; nullptr where the keys are sorted
  uint32_t* crossings;   // [0]: their number; then the chunks in which a run begins that
                         // goes on into the next
  float* parts;          // per chunk the part of a run from before it, then as many of
                         // runs that go on behind it
  int64_t count, chunks, part_stride;
  int64_t vocabulary, dimension;
  int64_t grad_stride, table_stride;
  float scale;
  int32_t accumulate;
  uint32_t sum_blocks;   // further blocks clear rows
  uint32_t clear_blocks;
  uint32_t slices;       // column slices of a row
  uint32_t join_slices;
  int lanes_log2;        // lanes that share a row
};

template <typename TW, int W>
__device__ __forceinline__ void finish_row(TW* to, float (&sum)[W], int64_t columns, float scale,
                                           int32_t accumulate) {
  if (columns <= 0) return;
  float old[W];
  load_floats<TW, W>(old, to, accumulate ? columns : 0);
#pragma unroll
  for (int k = 0; k < W; ++k) sum[k] = sum[k] * scale + old[k];
  store_floats<TW, W>(to, sum, columns);
}

constexpr int kClearRows = 16;  // per block

// Whether a row has a token: by its bit, or its key is among the sorted ones.
__device__ __forceinline__ bool is_met(const Sums& s, int64_t row) {
  if (s.met != nullptr) {
    const uint32_t of = (uint32_t)row & ((1u << s.group_log2) - 1), local = (uint32_t)(row >> s.group_log2);
    return (s.met[((uint64_t)(local >> 6) << s.group_log2) + of] >> (local & 63)) & 1;
  }
  int64_t low = 0, high = s.count;
  while (low < high) {
    const int64_t middle = (low + high) >> 1;
    if ((int64_t)s.keys[middle] < row) low = middle + 1;
    else high = middle;
  }
  return low < s.count && (int64_t)s.keys[low] == row;
}

template <typename TW>
__device__ __forceinline__ void clear_rows(const Sums& s, TW* __restrict__ table, int64_t first) {
  constexpr int W = 16 / sizeof(TW);
  const int64_t mine = first + (threadIdx.x & (kClearRows - 1));
  const bool met = mine >= s.vocabulary || is_met(s, mine);
  uint32_t unmet = ~(uint32_t)__ballot(met) & ((1u << kClearRows) - 1);
  float zeros[W];
#pragma unroll
  for (int k = 0; k < W; ++k) zeros[k] = 0.0f;
  for (; unmet != 0; unmet &= unmet - 1) {
    TW* row = table + (first + __builtin_ctz(unmet)) * s.table_stride;
    for (int64_t c = (int64_t)threadIdx.x * W; c < s.dimension; c += kBlock * W)
      store_floats<TW, W>(row + c, zeros, s.dimension - c);
  }
}

template <typename TG, typename TW, bool WHOLE_WAVE>
__global__ __launch_bounds__(kBlock) void embedding_gradient_kernel(
    Sums s, const TG* __restrict__ grad_out, TW* __restrict__ table) {
  constexpr int W = Width<TG, TW>::value;
  constexpr int U = 8;  // rows in flight
  if (blockIdx.x >= s.sum_blocks) {
    for (int64_t first = (int64_t)(blockIdx.x - s.sum_blocks) * kClearRows; first < s.vocabulary;
         first += (int64_t)s.clear_blocks * kClearRows)
      clear_rows(s, table, first);
    return;
  }
  const int log2 = WHOLE_WAVE ? 6 : s.lanes_log2;
  const uint32_t group = (blockIdx.x << (8 - log2)) + (threadIdx.x >> log2);
  uint32_t chunk = group / s.slices;
  uint32_t slice = group - chunk * s.slices;
  if (WHOLE_WAVE) {
    chunk = __builtin_amdgcn_readfirstlane(chunk);
    slice = __builtin_amdgcn_readfirstlane(slice);
  }
  if (chunk >= s.chunks) return;
  const uint32_t lane = threadIdx.x & ((1u << log2) - 1);
  const int64_t c = (((int64_t)slice << log2) + lane) * W;
  const int64_t columns = s.dimension - c;
  const uint32_t none = (uint32_t)s.vocabulary;
  const int64_t p0 = (int64_t)chunk * kChunk;
  const uint32_t before = p0 > 0 ? s.keys[p0 - 1] : none;
  float* const head = s.parts + (int64_t)chunk * s.part_stride + c;
  float* const tail = head + s.chunks * s.part_stride;

  uint32_t run = s.keys[p0];
  bool began = run != before;  // the run began in this chunk
  float sum[W];
#pragma unroll
  for (int k = 0; k < W; ++k) sum[k] = 0.0f;
  for (int u0 = 0; u0 < kChunk && run != none; u0 += U) {
    uint32_t key[U];
    float v[U][W];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t p = p0 + u0 + u;
      key[u] = p < s.count ? s.keys[p] : none;
      load_floats<TG, W>(v[u], grad_out + (key[u] != none ? s.order[p] * s.grad_stride : 0) + c,
                         key[u] != none ? columns : 0);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (key[u] != run) {
        // The run ends here.
        if (began) finish_row<TW, W>(table + run * s.table_stride + c, sum, columns, s.scale,
                                     s.accumulate);
        else if (columns > 0) store_floats<float, W>(head, sum, W);
#pragma unroll
        for (int k = 0; k < W; ++k) sum[k] = 0.0f;
        run = key[u];
        began = true;
      }
#pragma unroll
      for (int k = 0; k < W; ++k) sum[k] += v[u][k];
    }
  }
  if (run == none) return;
  const int64_t next = p0 + kChunk;
  const bool goes_on = next < s.count && s.keys[next] == run;
  if (began && !goes_on) {
    finish_row<TW, W>(table + run * s.table_stride + c, sum, columns, s.scale, s.accumulate);
    return;
  }
  if (columns > 0) store_floats<float, W>(began ? tail : head, sum, W);
  if (began && slice == 0 && lane == 0) s.crossings[1 + atomicAdd(s.crossings, 1u)] = chunk;
}

// Joins the parts of the runs that cross chunks: the waves of a block take every 16th
// part, and their sums are added in the order of the waves.
constexpr int kJoinBlock = 1024;
constexpr int kJoinWaves = kJoinBlock / kWaveSize;
template <typename TW>
__global__ __launch_bounds__(kJoinBlock) void join_runs_kernel(Sums s, TW* __restrict__ table) {
  constexpr int W = 4;
  __shared__ float lds[kJoinWaves][kWaveSize * W];
  const uint32_t slices = s.join_slices;
  const int wave = threadIdx.x / kWaveSize, lane = threadIdx.x & (kWaveSize - 1);
  const uint32_t items = s.crossings[0] * slices;
  for (uint32_t item = blockIdx.x; item < items; item += gridDim.x) {
    const int64_t chunk = s.crossings[1 + item / slices];
    const int64_t c = ((int64_t)(item % slices) * kWaveSize + lane) * W;
    const int64_t columns = s.dimension - c;
    const uint32_t run = s.keys[chunk * kChunk + kChunk - 1];
    // Chunks behind it that begin inside the run.
    int64_t more = 0;
    for (;;) {
      const int64_t p = (chunk + 1 + more + lane) * kChunk;
      const uint64_t inside = __ballot(p < s.count && s.keys[p < s.count ? p : 0] == run);
      if (inside == ~0ull) {
        more += kWaveSize;
        continue;
      }
      more += __builtin_ctzll(~inside);
      break;
    }
    float sum[W];
#pragma unroll
    for (int k = 0; k < W; ++k) sum[k] = 0.0f;
    if (columns > 0) {
      const float* from = s.parts + (chunk + 1) * s.part_stride + c;
      if (wave == 0) load_floats<float, W>(sum, s.parts + (s.chunks + chunk) * s.part_stride + c, W);
#pragma unroll 8
      for (int64_t j = wave; j < more; j += kJoinWaves) {
        float v[W];
        load_floats<float, W>(v, from + j * s.part_stride, W);
#pragma unroll
        for (int k = 0; k < W; ++k) sum[k] += v[k];
      }
    }
#pragma unroll
    for (int k = 0; k < W; ++k) lds[wave][lane * W + k] = sum[k];
    __syncthreads();
    if (wave == 0) {
      for (int w = 1; w < kJoinWaves; ++w)
#pragma unroll
        for (int k = 0; k < W; ++k) sum[k] += lds[w][lane * W + k];
      finish_row<TW, W>(table + run * s.table_stride + c, sum, columns, s.scale, s.accumulate);
    }
    __syncthreads();
  }
}

struct GradientTemp {
  int64_t keys, order, met, crossings, parts, sort, bytes;  // offsets
  int64_t chunks, part_stride;
};
GradientTemp gradient_temp(int64_t count, int64_t vocabulary, int64_t dimension) {
  GradientTemp t;
  const bool groups = takes_groups(count, vocabulary);
  t.chunks = div_up(count, kChunk);
  t.part_stride = align_up(dimension, 8);
  t.keys = 0;
  t.order = align_up(count * 4, 256);
  t.met = t.order + align_up(count * 4, 256);
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
        const int log2 = lanes_log2(a.dimension, Width<TI, TO>::value);
        {
          ProfileScope scope(stream, "embedding");
          hipLaunchKernelGGL((embedding_kernel<TI, TO, TT>), dim3(row_blocks(a.count, log2)),
                             dim3(kBlock), 0, stream, static_cast<const TI*>(a.table),
                             a.vocabulary, a.dimension, a.table_stride,
                             static_cast<const TT*>(a.tokens), a.count, a.scale,
                             static_cast<TO*>(a.out), a.out_stride, log2);
        }
        ILGPU_HIP_CHECK(hipGetLastError());
        return ILGPU_HIP_SUCCESS;
      });
    });
  });
}

int64_t embedding_gradient_temp_bytes(int64_t count, int64_t vocabulary, int64_t dimension) {
  return gradient_temp(count, vocabulary, dimension).bytes;
}

int32_t launch_embedding_gradient(hipStream_t stream, const EmbeddingGradientArgs& a) {
  if (a.vocabulary == 0) return ILGPU_HIP_SUCCESS;
  if (a.count > 0) {
    const int32_t rc = check_sort_device(stream);  // before anything is launched
    if (rc != ILGPU_HIP_SUCCESS) return rc;
  }
  const GradientTemp t = gradient_temp(a.count, a.vocabulary, a.dimension);
  char* base = reinterpret_cast<char*>(align_up((int64_t)(uintptr_t)a.temp, 256));
  uint32_t* keys = reinterpret_cast<uint32_t*>(base + t.keys);
  uint32_t* order = reinterpret_cast<uint32_t*>(base + t.order);
  uint32_t* crossings = reinterpret_cast<uint32_t*>(base + t.crossings);
  const bool groups = a.count > 0 && takes_groups(a.count, a.vocabulary);
  if (groups) {
    const int32_t rc = with_token_type(a.token_type, [&](auto tt) -> int32_t {
      using TT = decltype(tt);
      const int log2 = group_log2(a.vocabulary);
      const int rows = (int)div_up(a.vocabulary, (int64_t)1 << log2);
      {
        ProfileScope scope(stream, "embedding_group_tokens");
        hipLaunchKernelGGL((group_tokens_kernel<TT>), dim3(1u << log2), dim3(kGroupBlock),
                           (unsigned)(kGroupWaves * (rows + kGroupList) * 4), stream,
                           static_cast<const TT*>(a.tokens), a.count, a.vocabulary,
                           a.padding_token, log2, rows, keys, order,
                           reinterpret_cast<uint64_t*>(base + t.met), crossings);
      }
      ILGPU_HIP_CHECK(hipGetLastError());
      return ILGPU_HIP_SUCCESS;
    });
    if (rc != ILGPU_HIP_SUCCESS) return rc;
  } else if (a.count > 0) {
    const int32_t rc = with_token_type(a.token_type, [&](auto tt) -> int32_t {
      using TT = decltype(tt);
      const int64_t blocks = div_up(a.count, kBlock);
      {
        ProfileScope scope(stream, "embedding_token_keys");
        hipLaunchKernelGGL((token_keys_kernel<TT>),
                           dim3((unsigned)(blocks < kMaxBlocks ? blocks : kMaxBlocks)),
                           dim3(kBlock), 0, stream, static_cast<const TT*>(a.tokens), a.count,
                           a.vocabulary, a.padding_token, keys, crossings);
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
      constexpr int W = Width<TG, TW>::value;
      TW* table = static_cast<TW*>(a.grad_table);
      const int all_log2 = lanes_log2(a.dimension, W);
      const int log2 = all_log2 < 6 ? all_log2 : 6;
      const int64_t slices = div_up(a.dimension, (int64_t)W << log2);
      const int64_t join_slices = div_up(a.dimension, kWaveSize * 4);
      // (That many chunks and slices have parts of 2^42 bytes: no device holds such a temp.)
      if (t.chunks * join_slices > INT32_MAX) return ILGPU_HIP_ERROR_NOT_SUPPORTED;
      const int64_t sum_blocks = div_up(t.chunks * slices, kBlock >> log2);
      int64_t clear_blocks = a.accumulate ? 0 : div_up(a.vocabulary, kClearRows);
      if (clear_blocks > kMaxBlocks) clear_blocks = kMaxBlocks;
      const Sums s{keys, order,
                   groups ? reinterpret_cast<const uint64_t*>(base + t.met) : nullptr,
                   group_log2(a.vocabulary), crossings, reinterpret_cast<float*>(base + t.parts), a.count,
                   t.chunks, t.part_stride, a.vocabulary, a.dimension, a.grad_out_stride,
                   a.table_stride, a.scale, a.accumulate, (uint32_t)sum_blocks,
                   (uint32_t)clear_blocks, (uint32_t)slices, (uint32_t)join_slices, log2};
      if (sum_blocks + clear_blocks > 0) {
        ProfileScope scope(stream, "embedding_gradient");
        auto kernel = log2 == 6 ? embedding_gradient_kernel<TG, TW, true>
                                : embedding_gradient_kernel<TG, TW, false>;
        hipLaunchKernelGGL(kernel, dim3((unsigned)(sum_blocks + clear_blocks)), dim3(kBlock), 0,
                           stream, s, static_cast<const TG*>(a.grad_out), table);
      }
      ILGPU_HIP_CHECK(hipGetLastError());
      if (t.chunks > 1) {
        const int64_t items = (t.chunks - 1) * join_slices;
        ProfileScope scope(stream, "embedding_join_runs");
        hipLaunchKernelGGL((join_runs_kernel<TW>), dim3((unsigned)(items < 512 ? items : 512)),
                           dim3(kJoinBlock), 0, stream, s, table);
      }
      ILGPU_HIP_CHECK(hipGetLastError());
      return ILGPU_HIP_SUCCESS;
    });
  });
}

}  // namespace ilgpu_hip
