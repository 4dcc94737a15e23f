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
#include "paged.hpp"

#include <string>

namespace kvssd {
namespace {

constexpr int kThreads = 1024;
constexpr int kWaves = kThreads / kWave;
constexpr int kBins = 2048;

struct EvictParams {
  kvssd_paged_cache c;
  int32_t* lengths_out;
  float* weights_out;
  int32_t* positions_out;
  int32_t* counts;  // [sequences]: rows to move
  int32_t* to;      // [sequences][most]
  int32_t* from;
  int budget, sink, recent, capacity, most;
};

__device__ __forceinline__ uint32_t weight_key(float w, int position, int sink, int64_t latest, int recent) {
  if (position < sink || position > latest - recent) return 0xFFFFFFFFu;
  if (!(w == w)) w = -INFINITY;
  const uint32_t u = __builtin_bit_cast(uint32_t, w + 0.0f);  // -0 counts as 0
  return u >> 31 ? ~u : u | 0x80000000u;
}

// Exclusive prefix count of `flag` over the workgroup's threads; *total: of all.
__device__ __forceinline__ int prefix_count(bool flag, int* scratch, int* total) {
  const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
  const uint64_t mask = __ballot(flag);
  if (lane == 0) scratch[wave] = __popcll(mask);
  __syncthreads();
  int before = 0, all = 0;
  for (int w = 0; w < kWaves; ++w) {
    const int x = scratch[w];
    before += w < wave ? x : 0;
    all += x;
  }
  __syncthreads();
  *total = all;
  return before + __popcll(mask & ((1ull << lane) - 1));
}

__global__ __launch_bounds__(kThreads) void evict_select_kernel(EvictParams p) {
  __shared__ int hist[kBins];
  __shared__ int scratch[kWaves];
  __shared__ int found[2];  // digit, keys above it
  const int b = blockIdx.x, tid = threadIdx.x;
  const int n = paged_length(p.c.lengths, b, p.capacity);
  const int m = n < p.budget ? n : p.budget;
  const int64_t row = static_cast<int64_t>(b) * p.capacity;
  const float* weights = p.c.weights + row;
  const int32_t* positions = p.c.positions + row;
  float* weights_out = p.weights_out + row;
  int32_t* positions_out = p.positions_out + row;
  if (tid == 0) p.lengths_out[b] = m;
  for (int s = m + tid; s < p.capacity; s += kThreads) {
    weights_out[s] = 0.0f;
    positions_out[s] = -1;
  }
  if (n <= p.budget) {
    for (int s = tid; s < n; s += kThreads) {
      weights_out[s] = weights[s];
      positions_out[s] = positions[s];
    }
    if (tid == 0) p.counts[b] = 0;
    return;
  }
  // ---- the latest position
  int latest = INT32_MIN;
  for (int s = tid; s < n; s += kThreads) latest = max(latest, positions[s]);
  for (int k = 1; k < kWave; k <<= 1) latest = max(latest, __shfl_xor(latest, k, kWave));
  if (tid % kWave == 0) scratch[tid / kWave] = latest;
  __syncthreads();
  for (int w = 0; w < kWaves; ++w) latest = max(latest, scratch[w]);
  __syncthreads();
  // ---- the threshold key, digit by digit from the top
  uint32_t key = 0;  // digits found so far
  int need = m;      // kept keys among those that share them
  for (int pass = 0; pass < 3; ++pass) {
    const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0;
    const uint32_t digits = pass == 2 ? 1023u : 2047u;
    const uint32_t above = pass == 0 ? 0u : pass == 1 ? 0xFFE00000u : 0xFFFFFC00u;
    for (int i = tid; i < kBins; i += kThreads) hist[i] = 0;
    __syncthreads();
    for (int s = tid; s < n; s += kThreads) {
      const uint32_t k = weight_key(weights[s], positions[s], p.sink, latest, p.recent);
      if ((k & above) == key) atomicAdd(&hist[(k >> shift) & digits], 1);
    }
    __syncthreads();
    // bins in falling order, two a thread: the one in which the need-th key lies
    const int i0 = kBins - 1 - 2 * tid;
    const int c0 = hist[i0], c1 = hist[i0 - 1];
    int sum = c0 + c1;
    const int lane = tid % kWave, wave = tid / kWave;
    int incl = sum;
    for (int k = 1; k < kWave; k <<= 1) {
      const int x = __shfl_up(incl, k, kWave);
      if (lane >= k) incl += x;
    }
    if (lane == kWave - 1) scratch[wave] = incl;
    __syncthreads();
    int before = incl - sum;
    for (int w = 0; w < wave; ++w) before += scratch[w];
    if (before < need && need <= before + c0) {
      found[0] = i0;
      found[1] = before;
    } else if (before + c0 < need && need <= before + sum) {
      found[0] = i0 - 1;
      found[1] = before + c0;
    }
    __syncthreads();
    key |= static_cast<uint32_t>(found[0]) << shift;
    need -= found[1];
    __syncthreads();
  }
  // ---- keys above the threshold stay, and the first `need` of those equal to it
  int32_t* to = p.to + static_cast<int64_t>(b) * p.most;
  int32_t* from = p.from + static_cast<int64_t>(b) * p.most;
  int equal_before = 0, moved_to = 0, moved_from = 0;
  for (int base = 0; base < n; base += kThreads) {
    const int s = base + tid;
    float w = 0.0f;
    int pos = 0;
    uint32_t k = 0;
    if (s < n) {
      w = weights[s];
      pos = positions[s];
      k = weight_key(w, pos, p.sink, latest, p.recent);
    }
    int total;
    const bool equal = s < n && k == key;
    const int rank = equal_before + prefix_count(equal, scratch, &total);
    equal_before += total;
    const bool kept = s < n && (k > key || (equal && rank < need));
    const bool hole = s < m && !kept, far = s >= m && kept;
    const int hole_rank = moved_to + prefix_count(hole, scratch, &total);
    moved_to += total;
    const int far_rank = moved_from + prefix_count(far, scratch, &total);
    moved_from += total;
    if (hole) to[hole_rank] = s;
    if (far) from[far_rank] = s;
    if (s < m && kept) {
      weights_out[s] = w;
      positions_out[s] = pos;
    }
  }
  __syncthreads();  // (the lists, read below, were written by this workgroup)
  for (int i = tid; i < moved_to; i += kThreads) {
    const int t = to[i], f = from[i];
    weights_out[t] = weights[f];
    positions_out[t] = positions[f];
  }
  if (tid == 0) p.counts[b] = moved_to;
}

// A wave moves a row: codes of K and V, then scales, of every kv head.
__global__ __launch_bounds__(256) void evict_move_kernel(EvictParams p) {
  const int b = blockIdx.y;
  const int lane = threadIdx.x % kWave;
  const kvssd_paged_cache& c = p.c;
  const int count = p.counts[b];
  const int32_t* pages = c.page_table + static_cast<int64_t>(b) * c.max_pages;
  const int64_t code_bytes = static_cast<int64_t>(c.kv_heads) * c.head_dim * c.bits / 8;
  const int64_t scale_count = static_cast<int64_t>(c.kv_heads) * (c.head_dim / c.group_size);
  for (int i = blockIdx.x * 4 + threadIdx.x / kWave; i < count; i += gridDim.x * 4) {
    const int t = p.to[static_cast<int64_t>(b) * p.most + i], f = p.from[static_cast<int64_t>(b) * p.most + i];
    const int tp = pages[t / c.page_tokens], fp = pages[f / c.page_tokens];
    if (tp < 0 || tp >= c.num_pages || fp < 0 || fp >= c.num_pages) continue;
    const int64_t dst = static_cast<int64_t>(tp) * c.page_tokens + t % c.page_tokens;
    const int64_t src = static_cast<int64_t>(fp) * c.page_tokens + f % c.page_tokens;
    for (int64_t at = lane * 8; at < code_bytes; at += kWave * 8) {  // rows are multiples of 8 bytes
      *reinterpret_cast<uint64_t*>(c.packed_k + dst * code_bytes + at) =
          *reinterpret_cast<const uint64_t*>(c.packed_k + src * code_bytes + at);
      *reinterpret_cast<uint64_t*>(c.packed_v + dst * code_bytes + at) =
          *reinterpret_cast<const uint64_t*>(c.packed_v + src * code_bytes + at);
    }
    for (int64_t at = lane; at < scale_count; at += kWave) {
      c.scales_k[dst * scale_count + at] = c.scales_k[src * scale_count + at];
      c.scales_v[dst * scale_count + at] = c.scales_v[src * scale_count + at];
    }
  }
}

int most_moves(const kvssd_paged_cache& c, int budget) {
  const int64_t rest = paged_capacity(c) - budget;
  return static_cast<int>(rest < 0 ? 0 : rest < budget ? rest : budget);
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
  p.most = most_moves(c, a.budget);
  p.counts = static_cast<int32_t*>(a.workspace);
  p.to = p.counts + c.sequences;
  p.from = p.to + static_cast<int64_t>(c.sequences) * p.most;
  hipLaunchKernelGGL(evict_select_kernel, dim3(c.sequences), dim3(kThreads), 0, stream, p);
  if (int rc = hip_status(hipGetLastError(), "evict_select launch")) return rc;
  if (p.most == 0) return 0;
  for (int b0 = 0; b0 < c.sequences; b0 += 65535) {  // (a grid's second dimension)
    EvictParams q = p;
    const int nb = c.sequences - b0 < 65535 ? c.sequences - b0 : 65535;
    q.counts += b0;
    q.to += static_cast<int64_t>(b0) * p.most;
    q.from += static_cast<int64_t>(b0) * p.most;
    q.c.page_table += static_cast<int64_t>(b0) * c.max_pages;
    int blocks = (p.most + 3) / 4;
    const int cap = 8192 / nb < 1 ? 1 : 8192 / nb;
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
size_t evict_bytes(const kvssd_paged_cache& c, int budget) {
  return (static_cast<size_t>(c.sequences) + 2 * static_cast<size_t>(c.sequences) * most_moves(c, budget)) * sizeof(int32_t);
}
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
