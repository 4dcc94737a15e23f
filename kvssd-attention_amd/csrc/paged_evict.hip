// Eviction from a paged cache by accumulated attention weight.
//
// Per sequence of n > budget slots: keep the `budget` slots of largest key,
// of equal keys the lower slots, where a held slot (position below `sink` or
// among the last `recent`) has the largest key of all and any other its weight's
// bits in their numeric order.  The threshold key comes from three counting
// passes over its digits (11, 11 and 10 bits), the ties' cut and the places
// from prefix counts over the slots.  A kept slot at or past the budget moves to
// the freed slot of its rank before it: sources lie past the budget,
// destinations before it, so that rows move in place with nothing to order.
// Attention does not depend on the slots' order (keys are rotated already),
// and what is recent is read from the stored positions.
//
// Where the page table has at most kOneSlots slots a sequence, used or not, a
// sequence is one workgroup's, its weights and positions in registers from one
// read: 64 sequences of 4,160 slots cut to 4,096 take
// 17 us, moves included -- 0.9 until all is read, 0.5 for the latest position,
// 2.1 + 1.3 + 1.3 for the digits (the first has few bins, and their counts meet),
// 4.2 for ranks and lists, 3.7 for the moves' round trips, and the launch.  Longer
// ones take a workgroup a chunk and a launch a step, each step's result found
// again by every workgroup from the sequence's counts (8 KB): four sequences of
// 65,545 to 131,072 slots cut to 16,384 take 40 us in six launches (425 us by one
// workgroup each) and 27 for the moves, 122 MB at 4.6 TB/s.  The 64 sequences of
// 4,160 slots take that way too where their table is wider: a call 17.0 us in a table
// of 4,160 slots, 24.7 of 8,192, 48.6 of 8,256 and 79.6 of 131,072, over all of which
// weights and positions are written.  Counts are integers,
// so that the order in which atomics add them has no part in the result.
#include "paged.hpp"

#include <string>

namespace kvssd {
namespace {

constexpr int kBins = 2048;
constexpr int kPasses = 3;
// A sequence of one workgroup: what its registers hold (64 of 4,160 slots: 16.9 us, by chunks 38.8; 64 of 8,192 with
// 4,096 moves each: 113 and 140).
constexpr int kOneThreads = 1024, kOneSlots = 8 * kOneThreads;
constexpr int kChunkThreads = 256, kKeys = 8;                    // a chunk of one: kKeys slots a thread at a time
constexpr int kChunkSlots = kKeys * kChunkThreads, kMostChunks = 1024;
// So few rows move within the selecting workgroup: 64 rows of each of 64 sequences cost 0.8 us more of the GPU's time
// than a second launch (16.9 and 16.1 us) and 3 less of the host's; 192 rows of 4 sequences would cost 9.6 more.
constexpr int kInnerMoves = 64;
constexpr uint32_t kHeld = 0xFFFFFFFFu;

struct EvictParams {
  kvssd_paged_cache c;
  int32_t* lengths_out;
  float* weights_out;
  int32_t* positions_out;
  int32_t* counts;    // [sequences]: rows to move
  int32_t* to;        // [sequences][most]
  int32_t* from;
  int32_t* state;     // [sequences][kState]
  int32_t* hist;      // [sequences][kPasses][kBins]
  int32_t* chunk;     // [sequences][chunks][4]: latest position; then slots above and equal to the threshold, by side
  int budget, sink, recent, capacity, most, chunks, chunk_slots;
};
constexpr int kState = 2 * kPasses + 1;  // (key, need) after every pass, then the latest position

__device__ __forceinline__ uint32_t weight_key(float w, int position, int sink, int64_t latest, int recent) {
  if (position < sink || position > latest - recent) return kHeld;
  if (!(w == w)) w = -INFINITY;
  const uint32_t u = __builtin_bit_cast(uint32_t, w + 0.0f);  // -0 counts as 0
  return u >> 31 ? ~u : u | 0x80000000u;
}

__device__ __forceinline__ int pass_shift(int pass) { return pass == 0 ? 21 : pass == 1 ? 10 : 0; }
__device__ __forceinline__ uint32_t pass_above(int pass) { return pass == 0 ? 0u : pass == 1 ? 0xFFE00000u : 0xFFFFFC00u; }

__device__ __forceinline__ int scalar_wave() { return __builtin_amdgcn_readfirstlane(threadIdx.x / kWave); }

// Counts a key's digit; held keys, many and alike, once a wave.
__device__ __forceinline__ void count_key(int* hist, uint32_t k, bool live, int pass, uint32_t key) {
  const bool of = live && (k & pass_above(pass)) == key;
  const uint64_t held = __ballot(of && k == kHeld);
  const uint32_t digit = (k >> pass_shift(pass)) & (pass == 2 ? 1023u : 2047u);
  if (of && k != kHeld) atomicAdd(&hist[digit], 1);
  if (held != 0 && threadIdx.x % kWave == __builtin_ctzll(held)) atomicAdd(&hist[digit], __popcll(held));
}

// The latest of the workgroup's threads' positions.
template <int THREADS>
__device__ __forceinline__ int latest_of(int x, int* scratch) {
  const uint32_t most = wave_most(static_cast<uint32_t>(x) ^ 0x80000000u);
  if (threadIdx.x % kWave == 0) scratch[threadIdx.x / kWave] = static_cast<int>(most ^ 0x80000000u);
  __syncthreads();
  int latest = scratch[0];
#pragma unroll
  for (int v = 1; v < THREADS / kWave; ++v) latest = max(latest, scratch[v]);
  return latest;
}

// The bin, counted from the top, in which the need-th key lies, and the keys above it; -> key and need.
template <int THREADS>
__device__ __forceinline__ void find_digit(const int* hist, int pass, uint32_t& key, int& need, int* scratch) {
  constexpr int kEach = kBins / THREADS;
  const int tid = threadIdx.x, lane = tid % kWave, wave = tid / kWave;
  int c[kEach], sum = 0;
#pragma unroll
  for (int i = 0; i < kEach; ++i) sum += c[i] = hist[kBins - 1 - kEach * tid - i];
  const int incl = wave_prefix(sum);
  if (lane == kWave - 1) scratch[wave] = incl;
  __syncthreads();
  int before = incl - sum;
#pragma unroll
  for (int w = 0; w < THREADS / kWave; ++w) before += w < wave ? scratch[w] : 0;
  int* found = scratch + THREADS / kWave;
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    if (before < need && need <= before + c[i]) {
      found[0] = kBins - 1 - kEach * tid - i;
      found[1] = before;
    }
    before += c[i];
  }
  __syncthreads();
  key |= static_cast<uint32_t>(found[0]) << pass_shift(pass);
  need -= found[1];
}

// Exclusive prefix counts, in slot order, of flags over the slots j THREADS + thread, j < KEYS; total: of all.  The
// counts of two kinds of flags go in a word's halves (at most 2^14 slots).  Past `slots` there are none.
template <int THREADS, int KEYS>
__device__ __forceinline__ void prefix_counts(const uint32_t (&flag)[KEYS], uint32_t (&before)[KEYS], uint32_t& total,
                                              uint32_t* scratch, int slots) {
  constexpr int kWaves = THREADS / kWave, kEntries = KEYS * kWaves, kEach = (kEntries + kWave - 1) / kWave;
  const int lane = threadIdx.x % kWave, wave = scalar_wave();
  const uint64_t lower = (1ull << lane) - 1;
  __syncthreads();  // (scratch is free)
#pragma unroll
  for (int j = 0; j < KEYS; ++j) {
    if (j * THREADS >= slots) break;
    const uint64_t a = __ballot(flag[j] & 0xFFFFu), b = __ballot(flag[j] >> 16);
    before[j] = __popcll(a & lower) | __popcll(b & lower) << 16;
    if (lane == 0) scratch[j * kWaves + wave] = __popcll(a) | __popcll(b) << 16;
  }
  __syncthreads();
  uint32_t e[kEach], sum = 0;
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    const int at = lane * kEach + i;
    e[i] = sum;
    sum += at / kWaves * THREADS < slots && at < kEntries ? scratch[at] : 0;
  }
  const uint32_t incl = wave_prefix(sum);
  total = __builtin_amdgcn_readlane(incl, kWave - 1);
#pragma unroll
  for (int j = 0; j < KEYS; ++j) {
    if (j * THREADS >= slots) break;
    const int at = j * kWaves + wave;
    uint32_t x = __builtin_amdgcn_readlane(incl - sum, at / kEach);
#pragma unroll
    for (int i = 1; i < kEach; ++i) {
      const uint32_t y = __builtin_amdgcn_readlane(incl - sum + e[i], at / kEach);
      x = at % kEach == i ? y : x;
    }
    before[j] += x;
  }
}

// A wave moves slots from[i] to slots to[i], first <= i < count, kRows at a time with every load before the first
// store: codes of K and V, scales of every kv head, weights and positions.
constexpr int kRows = 4;
__device__ __forceinline__ void move_slots(const EvictParams& p, int b, const int32_t* to, const int32_t* from, int first,
                                           int count) {
  const int lane = threadIdx.x % kWave;
  const kvssd_paged_cache& c = p.c;
  const int64_t row = static_cast<int64_t>(b) * p.capacity;
  const int32_t* pages = c.page_table + static_cast<int64_t>(b) * c.max_pages;
  const int code_bytes = c.kv_heads * (c.head_dim * c.bits / 8);  // a multiple of 8; (below 2^31: the row's elements are)
  const int scale_count = c.kv_heads * (c.head_dim / c.group_size);
  int64_t dst[kRows], src[kRows];
  bool has[kRows];
#pragma unroll
  for (int r = 0; r < kRows; ++r) {
    const int i = min(first + r, count - 1);
    const int t = __builtin_amdgcn_readfirstlane(to[i]), f = __builtin_amdgcn_readfirstlane(from[i]);
    const int tp = uniform_load(pages + t / c.page_tokens), fp = uniform_load(pages + f / c.page_tokens);
    has[r] = first + r < count && tp >= 0 && tp < c.num_pages && fp >= 0 && fp < c.num_pages;
    dst[r] = static_cast<int64_t>(tp) * c.page_tokens + t % c.page_tokens;
    src[r] = static_cast<int64_t>(fp) * c.page_tokens + f % c.page_tokens;
  }
  for (int at = 0; at * 8 < code_bytes || at < scale_count; at += kWave) {
    const int piece = at + lane, byte = 8 * piece;
    uint64_t k[kRows], v[kRows];
    uint16_t sk[kRows], sv[kRows];
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      if (has[r] && byte < code_bytes) {
        k[r] = *reinterpret_cast<const uint64_t*>(c.packed_k + src[r] * code_bytes + byte);
        v[r] = *reinterpret_cast<const uint64_t*>(c.packed_v + src[r] * code_bytes + byte);
      }
      if (has[r] && piece < scale_count) {
        sk[r] = c.scales_k[src[r] * scale_count + piece];
        sv[r] = c.scales_v[src[r] * scale_count + piece];
      }
    }
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      if (has[r] && byte < code_bytes) {
        *reinterpret_cast<uint64_t*>(c.packed_k + dst[r] * code_bytes + byte) = k[r];
        *reinterpret_cast<uint64_t*>(c.packed_v + dst[r] * code_bytes + byte) = v[r];
      }
      if (has[r] && piece < scale_count) {
        c.scales_k[dst[r] * scale_count + piece] = sk[r];
        c.scales_v[dst[r] * scale_count + piece] = sv[r];
      }
    }
  }
  if (lane < kRows && first + lane < count) {
    const int t = to[first + lane], f = from[first + lane];
    p.weights_out[row + t] = c.weights[row + f];
    p.positions_out[row + t] = c.positions[row + f];
  }
}

__device__ __forceinline__ void clear_tail(const EvictParams& p, int64_t row, int begin, int end, int step) {
  for (int s = begin + threadIdx.x; s < end; s += step) {
    p.weights_out[row + s] = 0.0f;
    p.positions_out[row + s] = -1;
  }
}

// A sequence of at most kOneSlots slots in one workgroup: weights and positions are read once and stay in registers.
template <bool INNER>
__global__ __launch_bounds__(kOneThreads) void evict_one_kernel(EvictParams p) {
  constexpr int T = kOneThreads, K = kOneSlots / T;
  __shared__ int hist[kPasses][kBins];
  __shared__ uint32_t scratch[kOneSlots / kWave];
  __shared__ int small[T / kWave + 2];
  __shared__ int moves[2][INNER ? kInnerMoves : 1];
  const int b = blockIdx.x, tid = threadIdx.x;
  const int64_t row = static_cast<int64_t>(b) * p.capacity;
  float w[K];
  int pos[K];
#pragma unroll
  for (int j = 0; j < K; ++j) {
    const int s = j * T + tid;
    w[j] = 0.0f;
    pos[j] = INT32_MIN;
    if (s < p.capacity) {  // (not waiting for the length)
      w[j] = p.c.weights[row + s];
      pos[j] = p.c.positions[row + s];
    }
  }
  for (int i = tid; i < kPasses * kBins; i += T) hist[0][i] = 0;
  const int n = paged_length(p.c.lengths, b, p.capacity);
  const int m = n < p.budget ? n : p.budget;
  if (tid == 0) p.lengths_out[b] = m;
  if (n <= p.budget) {
    clear_tail(p, row, m, p.capacity, T);
#pragma unroll
    for (int j = 0; j < K; ++j) {
      const int s = j * T + tid;
      if (s < n) {
        p.weights_out[row + s] = w[j];
        p.positions_out[row + s] = pos[j];
      }
    }
    if (!INNER && tid == 0) p.counts[b] = 0;
    return;
  }
  int latest = INT32_MIN;
#pragma unroll
  for (int j = 0; j < K; ++j) latest = max(latest, j * T + tid < n ? pos[j] : INT32_MIN);
  latest = latest_of<T>(latest, small);
  uint32_t k[K];
#pragma unroll
  for (int j = 0; j < K; ++j) k[j] = weight_key(w[j], pos[j], p.sink, latest, p.recent);
  uint32_t key = 0;  // digits found so far
  int need = m;      // kept keys among those that share them
#pragma unroll
  for (int pass = 0; pass < kPasses; ++pass) {
#pragma unroll
    for (int j = 0; j < K; ++j)
      if (j * T < n) count_key(hist[pass], k[j], j * T + tid < n, pass, key);
    __syncthreads();
    find_digit<T>(hist[pass], pass, key, need, small);
  }
  // keys above the threshold stay, and the first `need` of those equal to it
  uint32_t flag[K], before[K], total;
#pragma unroll
  for (int j = 0; j < K; ++j) flag[j] = j * T + tid < n && k[j] == key;
  prefix_counts<T>(flag, before, total, scratch, n);
  bool kept[K];
#pragma unroll
  for (int j = 0; j < K; ++j) {
    if (j * T >= n) break;
    const int s = j * T + tid;
    kept[j] = s < n && (k[j] > key || (k[j] == key && static_cast<int>(before[j]) < need));
    flag[j] = s >= n ? 0 : s < m ? !kept[j] : kept[j] ? 0x10000u : 0;
  }
  prefix_counts<T>(flag, before, total, scratch, n);
  int32_t* to = INNER ? moves[0] : p.to + static_cast<int64_t>(b) * p.most;
  int32_t* from = INNER ? moves[INNER ? 1 : 0] : p.from + static_cast<int64_t>(b) * p.most;
#pragma unroll
  for (int j = 0; j < K; ++j) {
    if (j * T >= n) break;
    const int s = j * T + tid;
    if (flag[j] & 0xFFFFu) to[before[j] & 0xFFFFu] = s;
    if (flag[j] >> 16) from[before[j] >> 16] = s;
  }
  const int count = total >> 16;
  if constexpr (INNER) {
    __syncthreads();
    for (int i = kRows * scalar_wave(); i < count; i += kRows * (T / kWave)) move_slots(p, b, moves[0], moves[1], i, count);
  } else if (tid == 0) {
    p.counts[b] = count;
  }
  // (last: a barrier waits for the stores before it)
#pragma unroll
  for (int j = 0; j < K; ++j) {
    if (j * T >= m) break;
    const int s = j * T + tid;
    if (s < m && kept[j]) {
      p.weights_out[row + s] = w[j];
      p.positions_out[row + s] = pos[j];
    }
  }
  clear_tail(p, row, m, p.capacity, T);
}

__global__ __launch_bounds__(256) void evict_move_kernel(EvictParams p) {
  const int b = blockIdx.y;
  const int count = p.counts[b];
  const int64_t at = static_cast<int64_t>(b) * p.most;
  for (int i = kRows * (blockIdx.x * 4 + scalar_wave()); i < count; i += kRows * 4 * gridDim.x)
    move_slots(p, b, p.to + at, p.from + at, i, count);
}

// ---- longer sequences: a workgroup a chunk, a launch a step -------------------------------------------------------

struct Chunk {
  int b, nth, n, m, begin, end;  // slots [begin, end) of sequence b's n
  int64_t row;
};
__device__ __forceinline__ Chunk chunk_of(const EvictParams& p) {
  Chunk c;
  c.b = blockIdx.x / p.chunks;
  c.nth = blockIdx.x % p.chunks;
  c.n = paged_length(p.c.lengths, c.b, p.capacity);
  c.m = c.n < p.budget ? c.n : p.budget;
  c.row = static_cast<int64_t>(c.b) * p.capacity;
  c.begin = min(c.nth * p.chunk_slots, c.n);  // (below 2^31: at most 2^30 slots, and a chunk)
  c.end = min(c.begin + p.chunk_slots, c.n);
  return c;
}

// Step 1: a chunk's latest position; empty counts.
__global__ __launch_bounds__(kChunkThreads) void evict_latest_kernel(EvictParams p) {
  __shared__ int small[kChunkThreads / kWave];
  const Chunk c = chunk_of(p);
  const int tid = threadIdx.x;
  int32_t* hist = p.hist + static_cast<int64_t>(c.b) * kPasses * kBins;
  for (int i = c.nth * kChunkThreads + tid; i < kPasses * kBins; i += p.chunks * kChunkThreads) hist[i] = 0;
  int latest = INT32_MIN;
  for (int s = c.begin + tid; s < c.end; s += kChunkThreads) latest = max(latest, p.c.positions[c.row + s]);
  latest = latest_of<kChunkThreads>(latest, small);
  if (tid == 0) p.chunk[4 * static_cast<int64_t>(blockIdx.x)] = latest;
}

__device__ __forceinline__ uint32_t slot_key(const EvictParams& p, const Chunk& c, int s, int latest) {
  return weight_key(p.c.weights[c.row + s], p.c.positions[c.row + s], p.sink, latest, p.recent);
}

// Steps 2 to 4: the sequence's counts of a digit; the digit before it is found first, by every workgroup.
template <int PASS>
__global__ __launch_bounds__(kChunkThreads) void evict_count_kernel(EvictParams p) {
  constexpr int T = kChunkThreads;
  __shared__ int counts[kBins];
  __shared__ int small[T / kWave + 2];
  const Chunk c = chunk_of(p);
  if (c.n <= p.budget || c.begin >= c.end) return;
  const int tid = threadIdx.x;
  int32_t* hist = p.hist + static_cast<int64_t>(c.b) * kPasses * kBins;
  int32_t* state = p.state + static_cast<int64_t>(c.b) * kState;
  for (int i = tid; i < kBins; i += T) counts[i] = 0;
  uint32_t key = 0;
  int need = c.m, latest;
  if constexpr (PASS == 0) {
    latest = INT32_MIN;
    for (int i = tid; i < p.chunks && i * p.chunk_slots < c.n; i += T)
      latest = max(latest, p.chunk[4 * (static_cast<int64_t>(c.b) * p.chunks + i)]);
    latest = latest_of<T>(latest, small);
    if (c.nth == 0 && tid == 0) state[2 * kPasses] = latest;
  } else {
    latest = state[2 * kPasses];
    if constexpr (PASS > 1) {
      key = state[2 * (PASS - 2)];
      need = state[2 * (PASS - 2) + 1];
    }
    find_digit<T>(hist + (PASS - 1) * kBins, PASS - 1, key, need, small);
    if (c.nth == 0 && tid == 0) {
      state[2 * (PASS - 1)] = key;
      state[2 * (PASS - 1) + 1] = need;
    }
  }
  __syncthreads();
  for (int base = c.begin; base < c.end; base += kChunkSlots) {
    uint32_t k[kKeys];
#pragma unroll
    for (int j = 0; j < kKeys; ++j) {
      const int s = base + j * T + tid;
      k[j] = s < c.end ? slot_key(p, c, s, latest) : 0;
    }
#pragma unroll
    for (int j = 0; j < kKeys; ++j) count_key(counts, k[j], base + j * T + tid < c.end, PASS, key);
  }
  __syncthreads();
  for (int i = tid; i < kBins; i += T)
    if (counts[i] != 0) atomicAdd(&hist[PASS * kBins + i], counts[i]);  // (integers: any order)
}

// Step 5: a chunk's slots above and equal to the threshold, before the budget and from it on.
__global__ __launch_bounds__(kChunkThreads) void evict_tally_kernel(EvictParams p) {
  constexpr int T = kChunkThreads;
  __shared__ int small[T / kWave + 2];
  __shared__ int tally[4];
  const Chunk c = chunk_of(p);
  if (c.n <= p.budget || c.begin >= c.end) return;
  const int tid = threadIdx.x;
  int32_t* state = p.state + static_cast<int64_t>(c.b) * kState;
  uint32_t key = state[2 * (kPasses - 2)];
  int need = state[2 * (kPasses - 2) + 1];
  const int latest = state[2 * kPasses];
  if (tid < 4) tally[tid] = 0;
  find_digit<T>(p.hist + (static_cast<int64_t>(c.b) * kPasses + kPasses - 1) * kBins, kPasses - 1, key, need, small);
  if (c.nth == 0 && tid == 0) {
    state[2 * (kPasses - 1)] = key;
    state[2 * (kPasses - 1) + 1] = need;
  }
  int mine[4] = {0, 0, 0, 0};
  for (int base = c.begin; base < c.end; base += kChunkSlots) {
#pragma unroll
    for (int j = 0; j < kKeys; ++j) {
      const int s = base + j * T + tid;
      const uint32_t k = s < c.end ? slot_key(p, c, s, latest) : 0;
      const bool far = s >= c.m, above = s < c.end && k > key, equal = s < c.end && k == key;
      mine[0] += __popcll(__ballot(above && !far));
      mine[1] += __popcll(__ballot(above && far));
      mine[2] += __popcll(__ballot(equal && !far));
      mine[3] += __popcll(__ballot(equal && far));
    }
  }
  if (tid % kWave == 0) {
#pragma unroll
    for (int i = 0; i < 4; ++i) atomicAdd(&tally[i], mine[i]);
  }
  __syncthreads();
  if (tid < 4) p.chunk[4 * static_cast<int64_t>(blockIdx.x) + tid] = tally[tid];
}

// Step 6: the kept slots' weights and positions, and the lists of the moves.
__global__ __launch_bounds__(kChunkThreads) void evict_place_kernel(EvictParams p) {
  constexpr int T = kChunkThreads;
  __shared__ uint32_t scratch[kChunkSlots / kWave];
  __shared__ int sums[3][T / kWave];
  const Chunk c = chunk_of(p);
  const int tid = threadIdx.x, lane = tid % kWave, wave = tid / kWave;
  if (c.nth == 0 && tid == 0) p.lengths_out[c.b] = c.m;
  const int64_t tail = static_cast<int64_t>(c.nth) * p.chunk_slots;
  clear_tail(p, c.row, static_cast<int>(tail > c.m ? tail : c.m),
             static_cast<int>(tail + p.chunk_slots < p.capacity ? tail + p.chunk_slots : p.capacity), T);
  if (c.n <= p.budget) {
    for (int s = c.begin + tid; s < c.end; s += T) {
      p.weights_out[c.row + s] = p.c.weights[c.row + s];
      p.positions_out[c.row + s] = p.c.positions[c.row + s];
    }
    if (c.nth == 0 && tid == 0) p.counts[c.b] = 0;
    return;
  }
  const int32_t* state = p.state + static_cast<int64_t>(c.b) * kState;
  const uint32_t key = state[2 * (kPasses - 1)];
  const int need = state[2 * (kPasses - 1) + 1], latest = state[2 * kPasses];
  // of the chunks before: slots equal to the threshold; then, from those, holes before the budget and kept slots past it
  const int32_t* tallies = p.chunk + 4 * static_cast<int64_t>(c.b) * p.chunks;
  int equal_before = 0, holes = 0, fars = 0;
  for (int i0 = 0; i0 < c.nth && i0 * p.chunk_slots < c.n; i0 += T) {  // (the same number of times in every thread)
    const int i = i0 + tid;
    int above[2] = {0, 0}, equal[2] = {0, 0};
    const bool of = i < c.nth && static_cast<int64_t>(i) * p.chunk_slots < c.n;
    if (of) {
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        above[x] = tallies[4 * i + x];
        equal[x] = tallies[4 * i + 2 + x];
      }
    }
    const int incl = wave_prefix(equal[0] + equal[1]);
    __syncthreads();
    if (lane == kWave - 1) sums[0][wave] = incl;
    __syncthreads();
    int at = equal_before + incl - equal[0] - equal[1];
    for (int v = 0; v < T / kWave; ++v) {
      at += v < wave ? sums[0][v] : 0;
      equal_before += sums[0][v];
    }
    if (of) {
      const int64_t first = static_cast<int64_t>(i) * p.chunk_slots;
      const int64_t stop = first + p.chunk_slots < c.n ? first + p.chunk_slots : c.n;
      const int near = static_cast<int>(first >= c.m ? 0 : (stop < c.m ? stop : c.m) - first);
      const int kept_near = max(0, min(need - at, equal[0]));
      holes += near - above[0] - kept_near;
      fars += above[1] + max(0, min(need - at - equal[0], equal[1]));
    }
  }
  for (int k = 1; k < kWave; k <<= 1) {
    holes += __shfl_xor(holes, k, kWave);
    fars += __shfl_xor(fars, k, kWave);
  }
  if (lane == 0) {
    sums[1][wave] = holes;
    sums[2][wave] = fars;
  }
  __syncthreads();
  holes = fars = 0;
  for (int v = 0; v < T / kWave; ++v) {
    holes += sums[1][v];
    fars += sums[2][v];
  }
  int32_t* to = p.to + static_cast<int64_t>(c.b) * p.most;
  int32_t* from = p.from + static_cast<int64_t>(c.b) * p.most;
  for (int base = c.begin; base < c.end; base += kChunkSlots) {
    float w[kKeys];
    int pos[kKeys];
    uint32_t k[kKeys], flag[kKeys], before[kKeys], total;
#pragma unroll
    for (int j = 0; j < kKeys; ++j) {
      const int s = base + j * T + tid;
      w[j] = 0.0f;
      pos[j] = 0;
      if (s < c.end) {
        w[j] = p.c.weights[c.row + s];
        pos[j] = p.c.positions[c.row + s];
      }
      k[j] = weight_key(w[j], pos[j], p.sink, latest, p.recent);
      flag[j] = s < c.end && k[j] == key;
    }
    prefix_counts<T>(flag, before, total, scratch, kChunkSlots);
#pragma unroll
    for (int j = 0; j < kKeys; ++j) {
      const int s = base + j * T + tid;
      const bool kept =
          s < c.end && (k[j] > key || (k[j] == key && equal_before + static_cast<int>(before[j]) < need));
      if (s < c.m && kept) {
        p.weights_out[c.row + s] = w[j];
        p.positions_out[c.row + s] = pos[j];
      }
      flag[j] = s >= c.end ? 0 : s < c.m ? !kept : kept ? 0x10000u : 0;
    }
    equal_before += total;
    prefix_counts<T>(flag, before, total, scratch, kChunkSlots);
#pragma unroll
    for (int j = 0; j < kKeys; ++j) {
      const int s = base + j * T + tid;
      if (flag[j] & 0xFFFFu) to[holes + (before[j] & 0xFFFFu)] = s;
      if (flag[j] >> 16) from[fars + (before[j] >> 16)] = s;
    }
    holes += total & 0xFFFFu;
    fars += total >> 16;
  }
  if (c.end == c.n && c.begin < c.end && tid == 0) p.counts[c.b] = fars;
}

int most_moves(const kvssd_paged_cache& c, int budget) {
  const int64_t rest = paged_capacity(c) - budget;
  return static_cast<int>(rest < 0 ? 0 : rest < budget ? rest : budget);
}

// Workspace: chunked sequences' counts, then lengths and lists of the moves.
struct EvictPlan {
  bool one, inner;
  int most, chunks, chunk_slots;
  size_t words;
};
EvictPlan plan_evict(const kvssd_paged_cache& c, int budget) {
  EvictPlan e{};
  const int64_t capacity = paged_capacity(c);
  e.most = most_moves(c, budget);
  e.one = capacity <= kOneSlots;
  e.inner = e.one && e.most <= kInnerMoves;
  const size_t n = c.sequences;
  e.words = n * (1 + 2 * static_cast<size_t>(e.most));  // (also where no move's list leaves LDS: one size a budget)
  if (e.one) return e;
  const int64_t most_chunks = capacity / kChunkSlots / kMostChunks + 1;  // units of kChunkSlots a chunk
  e.chunk_slots = static_cast<int>(most_chunks) * kChunkSlots;
  e.chunks = static_cast<int>((capacity + e.chunk_slots - 1) / e.chunk_slots);
  e.words += n * (kState + kPasses * kBins + 4 * static_cast<size_t>(e.chunks));
  return e;
}

}  // namespace

int launch_paged_evict(const kvssd_paged_cache& c, const kvssd_paged_evict_args& a, hipStream_t stream) {
  EvictParams p{};
  p.c = c;
  p.lengths_out = a.lengths_out;
  p.weights_out = a.weights_out;
  p.positions_out = a.positions_out;
  p.budget = a.budget;
  p.sink = a.sink;
  p.recent = a.recent;
  p.capacity = static_cast<int>(paged_capacity(c));
  const EvictPlan plan = plan_evict(c, a.budget);
  p.most = plan.most;
  if (plan.inner) {
    hipLaunchKernelGGL(evict_one_kernel<true>, dim3(c.sequences), dim3(kOneThreads), 0, stream, p);
    return hip_status(hipGetLastError(), "evict launch");
  }
  const size_t n = c.sequences;
  p.counts = static_cast<int32_t*>(a.workspace);
  p.to = p.counts + n;
  p.from = p.to + n * p.most;
  if (plan.one) {
    hipLaunchKernelGGL(evict_one_kernel<false>, dim3(c.sequences), dim3(kOneThreads), 0, stream, p);
  } else {
    p.chunks = plan.chunks;
    p.chunk_slots = plan.chunk_slots;
    p.state = p.from + n * p.most;
    p.hist = p.state + n * kState;
    p.chunk = p.hist + n * kPasses * kBins;
    const dim3 grid(static_cast<unsigned>(n * plan.chunks)), block(kChunkThreads);
    hipLaunchKernelGGL(evict_latest_kernel, grid, block, 0, stream, p);
    hipLaunchKernelGGL(evict_count_kernel<0>, grid, block, 0, stream, p);
    hipLaunchKernelGGL(evict_count_kernel<1>, grid, block, 0, stream, p);
    hipLaunchKernelGGL(evict_count_kernel<2>, grid, block, 0, stream, p);
    hipLaunchKernelGGL(evict_tally_kernel, grid, block, 0, stream, p);
    hipLaunchKernelGGL(evict_place_kernel, grid, block, 0, stream, p);
  }
  if (int rc = hip_status(hipGetLastError(), "evict launch")) return rc;
  if (p.most == 0) return 0;
  for (int b0 = 0; b0 < c.sequences; b0 += 65535) {  // (a grid's second dimension)
    EvictParams q = p;
    const int nb = c.sequences - b0 < 65535 ? c.sequences - b0 : 65535;
    q.counts += b0;
    q.to += static_cast<int64_t>(b0) * p.most;
    q.from += static_cast<int64_t>(b0) * p.most;
    q.c.page_table += static_cast<int64_t>(b0) * c.max_pages;
    q.c.weights += b0 * static_cast<int64_t>(p.capacity);
    q.c.positions += b0 * static_cast<int64_t>(p.capacity);
    q.weights_out += b0 * static_cast<int64_t>(p.capacity);
    q.positions_out += b0 * static_cast<int64_t>(p.capacity);
    int blocks = (p.most + 4 * kRows - 1) / (4 * kRows);
    const int cap = 4096 / nb < 1 ? 1 : 4096 / nb;
    blocks = blocks < cap ? blocks : cap;
    hipLaunchKernelGGL(evict_move_kernel, dim3(blocks, nb), dim3(256), 0, stream, q);
  }
  return hip_status(hipGetLastError(), "evict_move launch");
}

}  // namespace kvssd

using namespace kvssd;

namespace {
int check_evict(const kvssd_paged_cache* cache, const kvssd_paged_evict_args* args) {
  if (int rc = check_paged_cache(cache)) return rc;
  if (args == nullptr) return arg_error("arguments are NULL");
  if (args->budget < 1) return arg_error("budget must be positive");
  if (args->sink < 0 || args->recent < 0) return arg_error("sink and recent counts must be non-negative");
  if (static_cast<int64_t>(args->sink) + args->recent > args->budget)
    return arg_error("sink and recent must fit the budget");
  return 0;
}
size_t evict_bytes(const kvssd_paged_cache& c, int budget) { return plan_evict(c, budget).words * sizeof(int32_t); }
}  // namespace

extern "C" {

__attribute__((visibility("default"))) int kvssd_hip_paged_evict_workspace_bytes(const kvssd_paged_cache* cache,
                                                                                 const kvssd_paged_evict_args* args,
                                                                                 size_t* bytes) {
  if (int rc = check_evict(cache, args)) return rc;
  if (bytes == nullptr) return arg_error("bytes output pointer is NULL");
  *bytes = evict_bytes(*cache, args->budget);
  return 0;
}

__attribute__((visibility("default"))) int kvssd_hip_paged_evict(const kvssd_paged_cache* cache,
                                                                 const kvssd_paged_evict_args* args, void* stream) {
  if (int rc = check_evict(cache, args)) return rc;
  if (!cache->weights || !cache->positions) return arg_error("eviction needs a cache with weights and positions");
  if (!args->lengths_out || !args->weights_out || !args->positions_out)
    return arg_error("a required buffer pointer is NULL");
  if (args->weights_out == cache->weights || args->positions_out == cache->positions ||
      args->lengths_out == cache->lengths)
    return arg_error("eviction writes arrays of their own, not the cache's");
  const size_t need = evict_bytes(*cache, args->budget);
  if (args->workspace == nullptr || args->workspace_bytes < need)
    return arg_error("workspace too small: need " + std::to_string(need) + " bytes");
  return launch_paged_evict(*cache, *args, static_cast<hipStream_t>(stream));
}

}  // extern "C"
