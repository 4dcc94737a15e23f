// Keeping some of a sequence's last (drafted) slots: slot base + j takes the row
// of slot base + kept[j], for an ascending list, in place.
//
// A workgroup takes a sequence.  It checks the list and finds the rows' places
// once (LDS), then a thread takes one column of the rows, up to 16 bytes of one
// of the four arrays, through the whole list: as the list ascends, kept[j] >= j,
// a row's source is never the place of an earlier one, so that a thread that
// reads ahead of its writes needs to wait for no other.  Bound by round trips (list,
// page table, rows): 4.4 us for 64 sequences that keep up to 8 of 32 tokens, 10.3 for
// 256 that keep up to 32 of 64 and move weights and positions; a pass from Python,
// 12 and 13 us, is the host's.
#include "paged.hpp"

namespace kvssd {
namespace {

constexpr int kThreads = 256;
constexpr int kList = 512;  // entries of the list at a time
constexpr int kAhead = 8;   // rows on the way in a thread

struct KeepParams {
  kvssd_paged_cache c;
  const int32_t* drafted;
  const int32_t* kept;
  int32_t* lengths_out;
  int width, capacity;
  int64_t code_row, scale_row;       // bytes of a slot
  int code_columns, scale_columns;   // of code_unit and scale_unit bytes
  int code_unit, scale_unit;
};

template <typename T>
__device__ __forceinline__ void move_column(uint8_t* at, int64_t row_bytes, const int* from, const int* to, int n) {
  for (int j0 = 0; j0 < n; j0 += kAhead) {
    T v[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i)
      if (j0 + i < n && from[j0 + i] >= 0) v[i] = *reinterpret_cast<const T*>(at + from[j0 + i] * row_bytes);
#pragma unroll
    for (int i = 0; i < kAhead; ++i)
      if (j0 + i < n && from[j0 + i] >= 0) *reinterpret_cast<T*>(at + to[j0 + i] * row_bytes) = v[i];
  }
}

__device__ __forceinline__ void move_unit(int unit, uint8_t* at, int64_t row_bytes, const int* from, const int* to, int n) {
  typedef uint32_t words4 __attribute__((ext_vector_type(4)));
  if (unit == 16) move_column<words4>(at, row_bytes, from, to, n);
  else if (unit == 8) move_column<uint64_t>(at, row_bytes, from, to, n);
  else if (unit == 4) move_column<uint32_t>(at, row_bytes, from, to, n);
  else move_column<uint16_t>(at, row_bytes, from, to, n);
}

__global__ __launch_bounds__(kThreads) void paged_keep_kernel(KeepParams p) {
  __shared__ int from[kList], to[kList];          // rows of the pool; from -1: does not move
  __shared__ int slot_from[kList], slot_to[kList];  // the same as slots; of rows that cannot move too
  __shared__ int end;
  const kvssd_paged_cache& c = p.c;
  const int b = blockIdx.x, tid = threadIdx.x;
  const int length = paged_length(c.lengths, b, p.capacity);
  const int count = p.drafted[b];
  const int drafted = count < 0 ? 0 : (count > length ? length : count);
  const int base = length - drafted;
  const int32_t* kept = p.kept + static_cast<int64_t>(b) * p.width;
  const int32_t* pages = c.page_table + static_cast<int64_t>(b) * c.max_pages;
  auto row_of = [&](int slot) {
    const int page = pages[slot / c.page_tokens];
    return page >= 0 && page < c.num_pages ? page * c.page_tokens + slot % c.page_tokens : -1;
  };
  int total = 0;
  for (int first = 0;; first += kList) {
    const int most = p.width - first < kList ? p.width - first : kList;
    if (tid == 0) end = most;
    __syncthreads();
    for (int j = tid; j < most; j += kThreads) {
      const int node = kept[first + j], before = first + j > 0 ? kept[first + j - 1] : -1;
      // An entry of an ascending list is not below its place.  One that is lies behind the list's end, where anything may
      // stand; so do all that are negative, which would name slots before the sequence's.
      if (node < first + j || node <= before || node >= drafted) {
        atomicMin(&end, j);
        continue;
      }
      const int target = base + first + j, source = base + node;  // base <= target <= source < length
      slot_from[j] = source;
      slot_to[j] = target;
      int r = -1, s = -1;
      if (node != first + j) {
        r = row_of(source);
        s = row_of(target);
      }
      from[j] = s < 0 ? -1 : r;
      to[j] = s;
    }
    __syncthreads();
    const int n = end;
    const int columns = 2 * (p.code_columns + p.scale_columns) + 2;
    for (int i = tid; i < columns; i += kThreads) {
      int k = i;
      if (k < 2 * p.code_columns) {
        uint8_t* pool = k < p.code_columns ? c.packed_k : c.packed_v;
        k -= k < p.code_columns ? 0 : p.code_columns;
        move_unit(p.code_unit, pool + static_cast<int64_t>(k) * p.code_unit, p.code_row, from, to, n);
        continue;
      }
      k -= 2 * p.code_columns;
      if (k < 2 * p.scale_columns) {
        uint8_t* pool = reinterpret_cast<uint8_t*>(k < p.scale_columns ? c.scales_k : c.scales_v);
        k -= k < p.scale_columns ? 0 : p.scale_columns;
        move_unit(p.scale_unit, pool + static_cast<int64_t>(k) * p.scale_unit, p.scale_row, from, to, n);
        continue;
      }
      uint8_t* per_slot = k == 2 * p.scale_columns ? reinterpret_cast<uint8_t*>(c.weights) : reinterpret_cast<uint8_t*>(c.positions);
      if (per_slot != nullptr) move_column<uint32_t>(per_slot + static_cast<int64_t>(b) * p.capacity * 4, 4, slot_from, slot_to, n);
    }
    total += n;
    if (n < kList || first + kList >= p.width) break;  // (n is the same for all)
    __syncthreads();
  }
  if (tid == 0) p.lengths_out[b] = base + total;
}

int unit_of(int64_t row_bytes) { return row_bytes % 16 == 0 ? 16 : row_bytes % 8 == 0 ? 8 : row_bytes % 4 == 0 ? 4 : 2; }

int launch_paged_keep(const kvssd_paged_cache& c, const kvssd_paged_keep_args& a, hipStream_t stream) {
  KeepParams p{};
  p.c = c;
  p.drafted = a.drafted;
  p.kept = a.kept;
  p.lengths_out = a.lengths_out;
  p.width = a.width;
  p.capacity = static_cast<int>(paged_capacity(c));
  p.code_row = static_cast<int64_t>(c.kv_heads) * c.head_dim * c.bits / 8;
  p.scale_row = static_cast<int64_t>(c.kv_heads) * (c.head_dim / c.group_size) * 2;
  p.code_unit = unit_of(p.code_row);
  p.scale_unit = unit_of(p.scale_row);
  p.code_columns = static_cast<int>(p.code_row / p.code_unit);
  p.scale_columns = static_cast<int>(p.scale_row / p.scale_unit);
  hipLaunchKernelGGL(paged_keep_kernel, dim3(c.sequences), dim3(kThreads), 0, stream, p);
  return hip_status(hipGetLastError(), "paged_keep launch");
}

}  // namespace
}  // namespace kvssd

using namespace kvssd;

extern "C" __attribute__((visibility("default"))) int kvssd_hip_paged_keep(const kvssd_paged_cache* cache,
                                                                           const kvssd_paged_keep_args* args,
                                                                           void* stream) {
  if (int rc = check_paged_cache(cache)) return rc;
  if (args == nullptr) return arg_error("arguments are NULL");
  if (args->width < 0) return arg_error("width must be >= 0");
  if (!args->drafted || !args->lengths_out || (args->width > 0 && !args->kept))
    return arg_error("a required buffer pointer is NULL");
  return launch_paged_keep(*cache, *args, static_cast<hipStream_t>(stream));
}
