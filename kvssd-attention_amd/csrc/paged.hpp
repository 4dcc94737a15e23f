// Shared by the generation operators: rotary positions and the paged packed
// cache (rotary.hip, paged_append.hip, paged_decode*.hip, paged_evict.hip).
#pragma once

#include "common.hpp"

namespace kvssd {

inline int64_t paged_capacity(const kvssd_paged_cache& c) { return static_cast<int64_t>(c.max_pages) * c.page_tokens; }

// the checks every paged entry point makes of a cache
int check_paged_cache(const kvssd_paged_cache* c);
int check_rotary(const kvssd_rotary_spec* r);

inline size_t dtype_bytes(int dtype) { return dtype == KVSSD_DTYPE_F32 ? 4 : 2; }
inline bool paged_dtype(int dtype) {
  return dtype == KVSSD_DTYPE_F16 || dtype == KVSSD_DTYPE_BF16 || dtype == KVSSD_DTYPE_F32;
}

int launch_rotary(const kvssd_rotary_spec& r, const void* positions, int positions_64, int64_t tokens, int dtype,
                  const kvssd_heads* tensors, int count, hipStream_t stream);
int launch_paged_append(const kvssd_paged_cache& c, const kvssd_paged_append_args& a, hipStream_t stream);
int paged_decode_bytes(const kvssd_paged_cache& c, const kvssd_paged_decode_args& a, size_t* bytes);
int launch_paged_decode(const kvssd_paged_cache& c, const kvssd_paged_decode_args& a, hipStream_t stream);
int launch_paged_evict(const kvssd_paged_cache& c, const kvssd_paged_evict_args& a, hipStream_t stream);

// ------------------------------------------------------------ device side ---

// *p for a wave-uniform p of memory that the launch does not write: a scalar load
__device__ __forceinline__ int32_t uniform_load(const int32_t* p) {
  typedef const __attribute__((address_space(4))) int32_t* constant_ptr;
  return __builtin_amdgcn_readfirstlane(*(constant_ptr)(uintptr_t)p);
}

// Length of sequence b as every kernel takes it.
__device__ __forceinline__ int clamp_length(int n, int capacity) { return n < 0 ? 0 : (n > capacity ? capacity : n); }
__device__ __forceinline__ int paged_length(const int32_t* lengths, int b, int capacity) {
  return clamp_length(lengths[b], capacity);
}

// Parent of token i of a sequence's tree (whose entries begin at `parents`), -1 if it has none there: any entry that is
// not an earlier token's.
__device__ __forceinline__ int parent_of(const int32_t* parents, int i) {
  const int up = parents[i];
  return up < i ? max(up, -1) : -1;
}

// x of a lane before this one (0 where there is none): CTRL 0x110 + n, n lanes
// before in the row of 16; 0x142 / 0x143, lane 15 of the row before / lane 31
template <int CTRL, int ROWS>
__device__ __forceinline__ int lane_before(int x) {
  return __builtin_amdgcn_update_dpp(0, x, CTRL, ROWS, 0xF, false);
}
__device__ __forceinline__ int wave_prefix(int x) {  // inclusive sum over the lanes
  x += lane_before<0x111, 0xF>(x);
  x += lane_before<0x112, 0xF>(x);
  x += lane_before<0x114, 0xF>(x);
  x += lane_before<0x118, 0xF>(x);
  x += lane_before<0x142, 0xA>(x);
  return x + lane_before<0x143, 0xC>(x);
}
__device__ __forceinline__ uint32_t wave_most(uint32_t x) {
  x = max(x, static_cast<uint32_t>(lane_before<0x111, 0xF>(x)));
  x = max(x, static_cast<uint32_t>(lane_before<0x112, 0xF>(x)));
  x = max(x, static_cast<uint32_t>(lane_before<0x114, 0xF>(x)));
  x = max(x, static_cast<uint32_t>(lane_before<0x118, 0xF>(x)));
  x = max(x, static_cast<uint32_t>(lane_before<0x142, 0xA>(x)));
  return __builtin_amdgcn_readlane(max(x, static_cast<uint32_t>(lane_before<0x143, 0xC>(x))), kWave - 1);
}

}  // namespace kvssd
