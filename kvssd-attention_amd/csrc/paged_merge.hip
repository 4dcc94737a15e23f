// Paged decode: the split plan, the join of a sequence's runs, the sum of its
// attention weights, and the C entry points.
//
// Join, per (sequence, query head): with partials (O_r unnormalised, m_r in
// log2 units, l_r) of the sequence's runs r,
//   M = max m_r, L = sum l_r 2^(m_r - M), out = sum O_r 2^(m_r - M) / L,
//   lse = ln 2 (M + log2 L);
// runs with l = 0 (no slot took part) add nothing.  The number of runs follows
// from the sequence's length on the device, as in the decode kernel.
//
// Weights: slot t of sequence b gains sum over heads of 2^(s_bht - lse2_bh) from
// the scores that the decode left (4 bytes a slot and head): a second pass
// over the keys would read head_dim * bits / 8 + scales per kv head instead.
// Scores lie by stage, one sequence's behind the other's, in as many places as
// the caller's hints make out (a page table has far more slots than its pool
// where every sequence may grow into all of it); a stage past them, of lengths
// past the hints, has its scores formed again here, a slot a lane.
// 16 sequences of 64 heads and up to 16,384 slots: 9.8 us (43 with a thread's heads
// one after the other), 1 of them the search for the sequence's place.
#include "paged_decode.hpp"

#include <string>

namespace kvssd {
namespace {

constexpr int kThreads = 256;
constexpr int kFewRows = 1024;

// LANES: lanes of a run, 4 dims each; kThreads / LANES runs side by side.  Bound by its round trips: lengths, then
// sums and partials together, then the joined row.  Many rows take all their dims in one workgroup (64 sequences of 32
// heads, 128 dims: 6.9 us; 2.4 more in two of 64 dims), few are spread over slices of 64 (one sequence of 32 heads:
// 4.1 us; 0.9 more in one).
template <int LANES>
__global__ __launch_bounds__(kThreads) void paged_merge_kernel(PagedDecodeParams p) {
  __shared__ float w_s[kMaxSplits];
  __shared__ float red[2][kThreads / kWave];
  __shared__ f32x4 sum_s[kThreads / kWave][LANES];
  const int seq = blockIdx.x / p.query_heads, h = blockIdx.x % p.query_heads;
  const int tid = threadIdx.x, lane = tid % kWave, wave = tid / kWave;
  int first_run, n;
  runs_of(p, seq, &first_run, &n);
  const int64_t row0 = static_cast<int64_t>(first_run) * p.query_heads + h;  // run r: row0 + r * query_heads
  const int d0 = 4 * (blockIdx.y * LANES + tid % LANES);
  const int d = p.c.head_dim;
  // the thread's first partials set out together, the sums behind them waiting for none
  constexpr int kAhead = 4, kSide = kThreads / LANES;
  typedef float f32x2 __attribute__((ext_vector_type(2)));
  const f32x2* ml = reinterpret_cast<const f32x2*>(p.part_ml) + row0;
  const float* o = p.part_o + row0 * d + d0;
  const int64_t step = static_cast<int64_t>(p.query_heads) * d;
  f32x2 own = {-INFINITY, 0.0f};
  if (tid < n) own = ml[static_cast<int64_t>(tid) * p.query_heads];
  f32x4 ahead[kAhead];
#pragma unroll
  for (int i = 0; i < kAhead; ++i) {
    const int r = tid / LANES + i * kSide;
    ahead[i] = r < n && d0 < d ? *reinterpret_cast<const f32x4*>(o + r * step) : f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  }
  float big = own[1] != 0.0f ? own[0] : -INFINITY;  // (a NaN sum keeps its run)
  for (int r = tid + kThreads; r < n; r += kThreads) {
    const f32x2 x = ml[static_cast<int64_t>(r) * p.query_heads];
    if (x[1] != 0.0f) big = fmaxf(big, x[0]);
  }
  big = wave_max(big);
  if (lane == 0) red[0][wave] = big;
  __syncthreads();
  big = fmaxf(fmaxf(red[0][0], red[0][1]), fmaxf(red[0][2], red[0][3]));
  float total = 0.0f;
  for (int r = tid; r < n; r += kThreads) {
    const f32x2 x = r == tid ? own : ml[static_cast<int64_t>(r) * p.query_heads];
    const float w = x[1] != 0.0f ? exp2f(x[0] - big) : 0.0f;
    w_s[r] = w;
    total += w * x[1];
  }
  total = wave_sum(total);
  if (lane == 0) red[1][wave] = total;
  __syncthreads();
  total = (red[1][0] + red[1][1]) + (red[1][2] + red[1][3]);
  f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
  for (int i = 0; i < kAhead; ++i) {
    const int r = tid / LANES + i * kSide;
    const float w = r < n ? w_s[r] : 0.0f;
    if (w != 0.0f) acc += w * ahead[i];  // (NaN weights take part)
  }
  if (d0 < d) {
#pragma unroll 4
    for (int r = tid / LANES + kAhead * kSide; r < n; r += kSide) {
      const float w = w_s[r];
      const f32x4 v = *reinterpret_cast<const f32x4*>(o + r * step);
      if (w != 0.0f) acc += w * v;
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (LANES <= 16) acc[i] += __shfl_xor(acc[i], 16, kWave);
    if constexpr (LANES <= 32) acc[i] += __shfl_xor(acc[i], 32, kWave);
  }
  if (lane < LANES) sum_s[wave][lane] = acc;
  __syncthreads();
  const int64_t row = static_cast<int64_t>(seq) * p.query_heads + h;
  if (tid < LANES && d0 < d) {
    const f32x4 v = (sum_s[0][tid] + sum_s[1][tid]) + (sum_s[2][tid] + sum_s[3][tid]);
#pragma unroll
    for (int i = 0; i < 4; ++i) store_out(p.out, p.out_dtype, row * d + d0 + i, total == 0.0f ? 0.0f : v[i] / total);
  }
  if (tid == 0 && blockIdx.y == 0) p.lse[row] = total == 0.0f ? -INFINITY : kLn2 * (big + log2f(total));
}

__device__ __forceinline__ float query_value(const void* row, int dtype, int dim) {
  if (dtype == KVSSD_DTYPE_F32) return load_query<float>(row, dim);
  return dtype == KVSSD_DTYPE_F16 ? load_query<_Float16>(row, dim) : load_query<uint16_t>(row, dim);
}

// The score of a row of the pool for query head h of a sequence, log2 units.
__device__ float row_score(const PagedDecodeParams& p, int seq, int h, int64_t row) {
  const kvssd_paged_cache& c = p.c;
  const int64_t at = row * c.kv_heads + h / p.gq;
  const uint32_t* codes = reinterpret_cast<const uint32_t*>(c.packed_k + at * (c.head_dim * c.bits / 8));
  const void* query = static_cast<const char*>(p.query) + (static_cast<int64_t>(seq) * p.query_heads + h) * c.head_dim *
                                                              (p.query_dtype == KVSSD_DTYPE_F32 ? 4 : 2);
  const int words = c.group_size * c.bits / 32, mask = (1 << c.bits) - 1, mid = 1 << (c.bits - 1);
  float score = 0.0f;
  for (int g = 0, dim = 0; g < p.groups; ++g) {
    float sum = 0.0f;
    for (int w = 0; w < words; ++w) {
      uint32_t x = *codes++;
      for (int i = 0; i < 32; i += c.bits, x >>= c.bits)
        sum = __builtin_fmaf(query_value(query, p.query_dtype, dim++), static_cast<float>(static_cast<int>(x & mask) - mid), sum);
    }
    score = __builtin_fmaf(sum, half_bits_to_float(c.scales_k[at * p.groups + g]), score);
  }
  return score * p.scale_log2;
}

// A slot's weight: 2^(score - the head's sum) over its heads.  A workgroup takes 4 kWave slots; its waves take a
// quarter of the heads each, kDeep rows of scores on the way at a time, and are joined in LDS in a fixed order.
__global__ __launch_bounds__(kThreads) void paged_weights_kernel(PagedDecodeParams p, int blocks) {
  constexpr int kDeep = 8, kWaves = kThreads / kWave;
  __shared__ f32x4 sums[kWaves][kWave];
  const int seq = blockIdx.x / blocks, nth = blockIdx.x % blocks;
  const int lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int length = paged_length(p.c.lengths, seq, p.capacity);
  if (static_cast<int64_t>(nth) * 4 * kWave >= length) return;
  const int before = stages_before(p, seq, length_of(p, lane));
  const float* lse = p.lse + static_cast<int64_t>(seq) * p.query_heads;
  for (int64_t t0 = static_cast<int64_t>(nth) * 4 * kWave; t0 < length; t0 += static_cast<int64_t>(blocks) * 4 * kWave) {
    const int64_t t = t0 + 4 * lane;
    const int64_t stage = before + t / kTile;
    f32x4 sum = {0.0f, 0.0f, 0.0f, 0.0f};
    if (t < length && stage < p.score_stages) {  // (rows are of whole 64 slots)
      const float* scores = p.scores + stage * p.query_heads * kTile + t % kTile;
      for (int h0 = wave; h0 < p.query_heads; h0 += kDeep * kWaves) {
        f32x4 v[kDeep];
        float e[kDeep];
#pragma unroll
        for (int i = 0; i < kDeep; ++i) {
          const int h = h0 + i * kWaves;
          e[i] = h < p.query_heads ? lse[h] * kLog2e : -INFINITY;
          if (h < p.query_heads) v[i] = *reinterpret_cast<const f32x4*>(scores + h * kTile);
        }
#pragma unroll
        for (int i = 0; i < kDeep; ++i) {
          if (e[i] == -INFINITY) continue;  // no such head, or none of its slots took part
#pragma unroll
          for (int x = 0; x < 4; ++x) sum[x] += __builtin_amdgcn_exp2f(v[i][x] - e[i]);
        }
      }
    } else if (t < length) {
      for (int x = 0; x < 4 && t + x < length; ++x) {
        const int slot = static_cast<int>(t) + x;
        const int page = p.c.page_table[static_cast<int64_t>(seq) * p.c.max_pages + slot / p.c.page_tokens];
        if (page < 0 || page >= p.c.num_pages) continue;
        const int64_t row = static_cast<int64_t>(page) * p.c.page_tokens + slot % p.c.page_tokens;
        float w = 0.0f;
        for (int h = wave; h < p.query_heads; h += kWaves) {
          const float e = lse[h] * kLog2e;
          if (e != -INFINITY) w += __builtin_amdgcn_exp2f(row_score(p, seq, h, row) - e);
        }
#pragma unroll
        for (int y = 0; y < 4; ++y) sum[y] = y == x ? w : sum[y];
      }
    }
    sums[wave][lane] = sum;
    __syncthreads();
    // thread n: slot n of the workgroup's
    float w = 0.0f;
#pragma unroll
    for (int v = 0; v < kWaves; ++v) w += reinterpret_cast<const float*>(sums[v])[threadIdx.x];
    if (t0 + threadIdx.x < length) p.c.weights[static_cast<int64_t>(seq) * p.capacity + t0 + threadIdx.x] += w;
    __syncthreads();
  }
}
static_assert(kThreads == 4 * kWave, "a thread a slot");

// Runs and shapes of a decode; the workspace's arrays as offsets from its start.
struct Plan {
  PagedDecodeParams p;
  int dp, gp = 1;
  size_t o_bytes, ml_bytes, score_bytes;
};

size_t aligned(size_t n) { return (n + 255) & ~static_cast<size_t>(255); }

int plan_of(const kvssd_paged_cache& c, const kvssd_paged_decode_args& a, Plan* out) {
  if (a.query_heads <= 0 || a.query_heads % c.kv_heads) return arg_error("query heads must be divisible by KV heads");
  if (!paged_dtype(a.query_dtype)) return arg_error("unsupported query dtype");
  if (a.out_query_dtype != 0 && a.out_query_dtype != 1) return arg_error("out_query_dtype must be 0 or 1");
  if (a.max_length < 0 || a.total_tokens < 0) return arg_error("max_length and total_tokens must be >= 0");
  if (a.accumulate && !c.weights) return arg_error("accumulate needs a cache with weights");
  PagedDecodeParams& p = out->p;
  p = PagedDecodeParams{};
  p.c = c;
  p.query = a.query;
  p.out = a.out;
  p.lse = a.lse;
  p.capacity = static_cast<int>(paged_capacity(c));
  p.query_heads = a.query_heads;
  p.gq = a.query_heads / c.kv_heads;
  p.query_dtype = a.query_dtype;
  p.out_dtype = a.out_query_dtype ? a.query_dtype : KVSSD_DTYPE_F32;
  p.scale_log2 = static_cast<float>(a.sm_scale) * kLog2e;
  p.groups = c.head_dim / c.group_size;
  while (out->gp < p.groups) out->gp *= 2;
  const int heads = 16 / out->gp;
  p.tiles = (p.gq + heads - 1) / heads;
  out->dp = c.head_dim <= 64 ? 64 : c.head_dim <= 128 ? 128 : 256;
  const int waves = decode_waves(out->dp);
  const int64_t units = static_cast<int64_t>(c.kv_heads) * p.tiles;
  if (units > (1 << 18)) return arg_error("too many heads");
  p.groups_of_units = static_cast<int>((units + waves - 1) / waves);
  p.group_units = static_cast<int>((units + p.groups_of_units - 1) / p.groups_of_units);

  while ((1 << p.group_log2) < c.group_size) ++p.group_log2;

  auto tiles_of = [](int64_t n) { return (n + kTile - 1) / kTile; };
  const int64_t longest = a.max_length > 0 && a.max_length < p.capacity ? a.max_length : p.capacity;
  if (tiles_of(p.capacity) * c.sequences >= int64_t{1} << 31) return arg_error("sequences * capacity is past 2^37 slots");
  int64_t all = tiles_of(longest) * c.sequences;  // stages to be worked on
  if (a.total_tokens > 0 && a.total_tokens / kTile + c.sequences < all) all = a.total_tokens / kTile + c.sequences;
  // one round of workgroups: every CU holds one (its LDS)
  const int64_t room = 256 * waves / units;  // runs
  const int64_t cut = room - c.sequences > room / 2 ? room - c.sequences : (room + 1) / 2;
  int64_t per = (all + cut - 1) / (cut > 0 ? cut : 1);
  const int64_t least = (tiles_of(longest) + kMaxSplits - 1) / kMaxSplits;
  if (per < least) per = least;
  p.run_tiles = static_cast<int>(per);
  p.runs = per >= tiles_of(longest) ? c.sequences : static_cast<int>(all / per + c.sequences);
  p.group_runs = waves / p.group_units;
  if (p.group_runs > p.runs) p.group_runs = p.runs;

  const bool whole = p.runs <= c.sequences;
  const size_t rows = static_cast<size_t>(p.runs) * p.query_heads;
  out->o_bytes = whole ? 0 : aligned(rows * c.head_dim * sizeof(float));
  out->ml_bytes = whole ? 0 : aligned(rows * 2 * sizeof(float));
  p.score_stages = static_cast<int>(all);
  out->score_bytes = a.accumulate ? static_cast<size_t>(all) * p.query_heads * kTile * sizeof(float) : 0;
  if (static_cast<int64_t>(p.runs) * waves * kWave > 0xFFFFFFFFll ||
      static_cast<int64_t>(c.sequences) * p.query_heads * kThreads > 0xFFFFFFFFll)
    return arg_error("too many sequences for one call");
  return 0;
}

}  // namespace

int launch_paged_merge(const PagedDecodeParams& p, hipStream_t stream) {
  const int rows = p.c.sequences * p.query_heads, d = p.c.head_dim;
  if (rows < kFewRows || d <= 64) hipLaunchKernelGGL(paged_merge_kernel<16>, dim3(rows, (d + 63) / 64), dim3(kThreads), 0, stream, p);
  else if (d <= 128) hipLaunchKernelGGL(paged_merge_kernel<32>, dim3(rows), dim3(kThreads), 0, stream, p);
  else hipLaunchKernelGGL(paged_merge_kernel<64>, dim3(rows), dim3(kThreads), 0, stream, p);
  return hip_status(hipGetLastError(), "paged_merge launch");
}

int paged_decode_bytes(const kvssd_paged_cache& c, const kvssd_paged_decode_args& a, size_t* bytes) {
  Plan plan{};
  if (int rc = plan_of(c, a, &plan)) return rc;
  *bytes = plan.o_bytes + plan.ml_bytes + plan.score_bytes;
  return 0;
}

int launch_paged_decode(const kvssd_paged_cache& c, const kvssd_paged_decode_args& a, hipStream_t stream) {
  Plan plan{};
  if (int rc = plan_of(c, a, &plan)) return rc;
  PagedDecodeParams& p = plan.p;
  const size_t need = plan.o_bytes + plan.ml_bytes + plan.score_bytes;
  if (need > 0 && (a.workspace == nullptr || a.workspace_bytes < need))
    return arg_error("workspace too small: need " + std::to_string(need) + " bytes");
  if (reinterpret_cast<uintptr_t>(a.workspace) % 256) return arg_error("workspace must be 256-byte aligned");
  char* ws = static_cast<char*>(a.workspace);
  p.part_o = reinterpret_cast<float*>(ws);
  p.part_ml = reinterpret_cast<float*>(ws + plan.o_bytes);
  if (a.accumulate) p.scores = reinterpret_cast<float*>(ws + plan.o_bytes + plan.ml_bytes);
  const bool precise = p.out_dtype == KVSSD_DTYPE_F32 || p.query_dtype == KVSSD_DTYPE_F32;
  if (reinterpret_cast<uintptr_t>(a.query) % 16) return arg_error("query must be 16-byte aligned");
  const auto launch = c.bits == 4 ? (plan.dp == 64    ? launch_paged_dims<4, 64>
                                     : plan.dp == 128 ? launch_paged_dims<4, 128>
                                                      : launch_paged_dims<4, 256>)
                                  : (plan.dp == 64    ? launch_paged_dims<2, 64>
                                     : plan.dp == 128 ? launch_paged_dims<2, 128>
                                                      : launch_paged_dims<2, 256>);
  if (int rc = launch(p, plan.gp, precise, stream)) return rc;
  if (p.runs > c.sequences)
    if (int rc = launch_paged_merge(p, stream)) return rc;
  if (a.accumulate) {
    const int64_t longest = a.max_length > 0 && a.max_length < p.capacity ? a.max_length : p.capacity;
    // of a sequence; together fewer than 2^32 threads (a grid's second dimension would end at 65535 sequences)
    const int64_t most = ((int64_t{1} << 24) - 1) / c.sequences;
    int64_t blocks = (longest + 4 * kWave - 1) / (4 * kWave);
    blocks = blocks < most ? blocks : most;
    hipLaunchKernelGGL(paged_weights_kernel, dim3(static_cast<unsigned>(blocks * c.sequences)), dim3(kThreads), 0, stream,
                       p, static_cast<int>(blocks));
    return hip_status(hipGetLastError(), "paged_weights launch");
  }
  return 0;
}

}  // namespace kvssd

using namespace kvssd;

extern "C" {

__attribute__((visibility("default"))) int kvssd_hip_paged_decode_workspace_bytes(const kvssd_paged_cache* cache,
                                                                                  const kvssd_paged_decode_args* args,
                                                                                  size_t* bytes) {
  if (int rc = check_paged_cache(cache)) return rc;
  if (args == nullptr || bytes == nullptr) return arg_error("arguments are NULL");
  return paged_decode_bytes(*cache, *args, bytes);
}

__attribute__((visibility("default"))) int kvssd_hip_paged_decode(const kvssd_paged_cache* cache,
                                                                  const kvssd_paged_decode_args* args, void* stream) {
  if (int rc = check_paged_cache(cache)) return rc;
  if (args == nullptr) return arg_error("arguments are NULL");
  if (!args->query || !args->out || !args->lse) return arg_error("a required buffer pointer is NULL");
  return launch_paged_decode(*cache, *args, static_cast<hipStream_t>(stream));
}

}  // extern "C"
