// Attention of many tokens a sequence: the plan, the join of a block's runs and
// the C entry points.
//
// Join, per (token, query head): with partials (O_r unnormalised, m_r in log2
// units, l_r) of the runs r of its block,
//   M = max m_r, L = sum l_r 2^(m_r - M), out = sum O_r 2^(m_r - M) / L,
//   lse = ln 2 (M + log2 L);
// runs with l = 0 (nothing was seen) add nothing.
#include "paged_tokens.hpp"

#include <string>

namespace kvssd {
namespace {

constexpr int kThreads = 256;
constexpr int kLeastStages = 2;  // of a run

// A workgroup takes kThreads / (d / 4) rows at a time, of `rows` of a block: their runs' sums by a lane a run first, whose
// weights go to LDS, then 4 dims a thread.
template <int STAGE>
__global__ __launch_bounds__(kThreads) void paged_tokens_merge_kernel(PagedTokensParams p, int rows, int chunks) {
  constexpr int kRuns = 1024, kSide = 32;  // weights at a time, of all rows at once; lanes of a row's sums
  __shared__ float weights[kRuns];
  __shared__ float most_s[kThreads / 8], sum_s[kThreads / 8];
  const int chunk = blockIdx.x % chunks, kvh = blockIdx.x / chunks % p.c.kv_heads;
  int first;
  const TokenItem work = find_item<STAGE>(p, blockIdx.x / chunks / p.c.kv_heads, true, &first);
  if (work.seq < 0 || work.runs == 1) return;
  const int d = p.c.head_dim, lanes = d / 4, side = kThreads / lanes;  // rows side by side: 4 to 32
  const int end = min(min(work.span.count * p.gq - work.block * p.block_rows, p.block_rows), (chunk + 1) * rows);
  typedef float f32x2 __attribute__((ext_vector_type(2)));
  const int64_t step = static_cast<int64_t>(p.c.kv_heads) * p.block_rows;  // rows between runs
  const int64_t at0 = (static_cast<int64_t>(first) * p.c.kv_heads + kvh) * p.block_rows;
  const f32x2* ml = reinterpret_cast<const f32x2*>(p.part_ml);
  const int tid = threadIdx.x, own = tid / lanes, dim = tid % lanes * 4;
  for (int row0 = chunk * rows; row0 < end; row0 += side) {
    // largest reference of each row, then its sum: 32 lanes a row, 8 rows at a time, the first 64 runs kept in registers
    for (int r0 = tid / kSide; r0 < side; r0 += kThreads / kSide) {
      const f32x2* of = ml + at0 + row0 + r0;
      const int runs = row0 + r0 < end ? work.runs : 0, n = tid % kSide;
      f32x2 x[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) x[i] = n + i * kSide < runs ? of[(n + i * kSide) * step] : f32x2{-INFINITY, 0.0f};
      float most = fmaxf(x[0][1] != 0.0f ? x[0][0] : -INFINITY, x[1][1] != 0.0f ? x[1][0] : -INFINITY);  // (a NaN sum takes part)
      for (int i = n + 2 * kSide; i < runs; i += kSide) {
        const f32x2 y = of[i * step];
        if (y[1] != 0.0f) most = fmaxf(most, y[0]);
      }
#pragma unroll
      for (int k = 1; k < kSide; k *= 2) most = fmaxf(most, __shfl_xor(most, k, kWave));
      float sum = 0.0f;
#pragma unroll
      for (int i = 0; i < 2; ++i)
        if (x[i][1] != 0.0f) sum += exp2f(x[i][0] - most) * x[i][1];
      for (int i = n + 2 * kSide; i < runs; i += kSide) {
        const f32x2 y = of[i * step];
        if (y[1] != 0.0f) sum += exp2f(y[0] - most) * y[1];
      }
#pragma unroll
      for (int k = 1; k < kSide; k *= 2) sum += __shfl_xor(sum, k, kWave);
      if (n == 0) {
        most_s[r0] = most;
        sum_s[r0] = sum;
      }
    }
    const int together = kRuns / side;  // runs
    f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int n0 = 0; n0 < work.runs; n0 += together) {
      const int here = min(together, work.runs - n0);
      __syncthreads();
      for (int i = tid; i < side * here; i += kThreads) {
        const int r = i / here, n = i - r * here;
        float w = 0.0f;
        if (row0 + r < end) {
          const f32x2 x = ml[at0 + row0 + r + (n0 + n) * step];
          if (x[1] != 0.0f) w = exp2f(x[0] - most_s[r]);
        }
        weights[r * together + n] = w;
      }
      __syncthreads();
      if (own < side && row0 + own < end) {
        const float* o = p.part_o + (at0 + row0 + own + n0 * step) * d + dim;
#pragma unroll 8
        for (int n = 0; n < here; ++n) {
          const f32x4 v = *reinterpret_cast<const f32x4*>(o + n * step * d);
          const float w = weights[own * together + n];
          if (w != 0.0f) acc += w * v;  // (NaN weights take part)
        }
      }
    }
    if (own < side && row0 + own < end) {
      const float sum = sum_s[own];
      const int in_seq = work.block * p.block_rows + row0 + own, token = in_seq / p.gq;
      const int64_t to = (work.span.begin + token) * p.query_heads + kvh * p.gq + in_seq - token * p.gq;
#pragma unroll
      for (int i = 0; i < 4; ++i) store_out(p.out, p.out_dtype, to * d + dim + i, sum == 0.0f ? 0.0f : acc[i] / sum);
      if (dim == 0) p.lse[to] = sum == 0.0f ? -INFINITY : kLn2 * (most_s[own] + log2f(sum));
    }
    __syncthreads();
  }
}

size_t aligned(size_t n) { return (n + 255) & ~static_cast<size_t>(255); }

struct Plan {
  PagedTokensParams p;
  int dp, waves, stage;
  bool precise;
  int64_t blocks;  // at most
  size_t o_bytes, ml_bytes;
};

int plan_of(const kvssd_paged_cache& c, const kvssd_paged_tokens_args& a, Plan* plan) {
  if (a.query.heads <= 0 || a.query.heads % c.kv_heads) return arg_error("query heads must be divisible by KV heads");
  if (!paged_dtype(a.query_dtype)) return arg_error("unsupported query dtype");
  if (a.out_query_dtype != 0 && a.out_query_dtype != 1) return arg_error("out_query_dtype must be 0 or 1");
  if (a.max_length < 0 || a.total_tokens < 0) return arg_error("max_length and total_tokens must be >= 0");
  if (a.window < 0 || a.sink < 0) return arg_error("window and sink must be >= 0");
  if (a.tokens < 0 || a.tokens > (int64_t{1} << 30) || a.tokens * a.query.heads > (int64_t{1} << 30))
    return arg_error("tokens * query heads must be at most 2^30");
  *plan = Plan{};
  PagedTokensParams& p = plan->p;
  p.c = c;
  p.query = a.query;
  p.out = a.out;
  p.lse = a.lse;
  p.offsets = a.offsets;
  p.parents = a.parents;
  p.tokens = a.tokens;
  p.capacity = static_cast<int>(paged_capacity(c));
  const int far = 1 << 30;  // as good as any larger one
  p.window = a.window < far ? a.window : far;
  p.sink = a.sink < far ? a.sink : far;
  p.query_heads = a.query.heads;
  p.gq = a.query.heads / c.kv_heads;
  p.query_dtype = a.query_dtype;
  p.out_dtype = a.out_query_dtype ? a.query_dtype : KVSSD_DTYPE_F32;
  p.groups = c.head_dim / c.group_size;
  p.of_page = divisor(c.page_tokens);
  while ((32 << p.slices_log2) < c.group_size) ++p.slices_log2;
  p.scale_log2 = static_cast<float>(a.sm_scale) * kLog2e;
  plan->precise = p.out_dtype == KVSSD_DTYPE_F32 || p.query_dtype == KVSSD_DTYPE_F32;
  plan->dp = c.head_dim <= 64 ? 64 : c.head_dim <= 128 ? 128 : 256;

  // rows of a workgroup, after a sequence's rows on average
  const int64_t each = (a.tokens * p.gq + c.sequences - 1) / c.sequences;
  plan->waves = each > 128 && !plan->precise && plan->dp <= 128 ? 8 : 4;
  const int stage = plan->stage = tokens_stage(plan->dp, plan->waves);
  p.row_tiles = each > 128 ? plan->waves : each > 64 ? 4 : each > 32 ? 2 : 1;
  p.parts = plan->waves / p.row_tiles < stage / 64 ? plan->waves / p.row_tiles : stage / 64;
  p.block_rows = 32 * p.row_tiles;
  plan->blocks = a.tokens * p.gq / p.block_rows + c.sequences + 2;

  // runs, where blocks alone would leave compute units idle
  auto stages = [&](int64_t n) { return (n + stage - 1) / stage; };
  int64_t longest = a.max_length > 0 && a.max_length < p.capacity ? a.max_length : p.capacity;
  int64_t total = a.total_tokens > 0 && a.total_tokens < longest * c.sequences ? a.total_tokens : longest * c.sequences;
  if (p.window > 0) {
    const int64_t seen = p.window + p.block_rows / p.gq + p.sink + 3 * stage;
    longest = longest < seen ? longest : seen;
    total = total < longest * c.sequences ? total : longest * c.sequences;
  }
  const int64_t likely = (each + p.block_rows - 1) / p.block_rows * c.sequences;  // blocks
  const int64_t work = (total / stage + c.sequences) * (likely / c.sequences);    // stages of all blocks
  // workgroups that run at a time (LDS and registers); two rounds of them where blocks are few, four of more, whose
  // lengths differ
  const int64_t at_once = plan->waves == 4 && !plan->precise && plan->dp <= 128 ? 512 : 256;
  const int64_t wanted = (likely * c.kv_heads < at_once ? 2 : 4) * at_once / c.kv_heads;
  const int64_t cut = wanted - likely > wanted / 2 ? wanted - likely : (wanted + 1) / 2;
  int64_t size = (work + cut - 1) / (cut > 0 ? cut : 1);
  if (size < kLeastStages) size = kLeastStages;
  p.items = static_cast<int>(plan->blocks);
  p.least_stages = 1 << 30;
  if (size < stages(longest)) {
    p.least_stages = static_cast<int>(size);
    p.items = static_cast<int>(plan->blocks + work / size + 1);
  }
  if (static_cast<int64_t>(p.items) * c.kv_heads > (int64_t{1} << 22)) return arg_error("too many sequences or tokens for one call");
  const bool split = p.least_stages < (1 << 30);
  const size_t rows = split ? static_cast<size_t>(p.items) * c.kv_heads * p.block_rows : 0;
  plan->o_bytes = aligned(rows * c.head_dim * sizeof(float));
  plan->ml_bytes = aligned(rows * 2 * sizeof(float));
  return 0;
}

int launch_paged_tokens(const kvssd_paged_cache& c, const kvssd_paged_tokens_args& a, hipStream_t stream) {
  Plan plan;
  if (int rc = plan_of(c, a, &plan)) return rc;
  PagedTokensParams& p = plan.p;
  const size_t need = plan.o_bytes + plan.ml_bytes;
  if (need > 0 && (a.workspace == nullptr || a.workspace_bytes < need))
    return arg_error("workspace too small: need " + std::to_string(need) + " bytes");
  if (reinterpret_cast<uintptr_t>(a.workspace) % 256) return arg_error("workspace must be 256-byte aligned");
  if (!heads_vector(a.query, dtype_bytes(a.query_dtype), false))
    return arg_error("query must be 16-byte aligned, as must its tokens and heads be");
  if (reinterpret_cast<uintptr_t>(a.out) % 16) return arg_error("out must be 16-byte aligned");
  p.part_o = static_cast<float*>(a.workspace);
  p.part_ml = reinterpret_cast<float*>(static_cast<char*>(a.workspace) + plan.o_bytes);
  const int64_t work = static_cast<int64_t>(p.items) * c.kv_heads;
  const unsigned groups = static_cast<unsigned>(c.kv_heads % 2 ? work : (work + 15) / 16 * 16);
  const auto launch = plan.dp == 64    ? launch_paged_tokens_dims<64>
                      : plan.dp == 128 ? launch_paged_tokens_dims<128>
                                       : launch_paged_tokens_dims<256>;
  if (int rc = launch(p, plan.waves, plan.precise, groups, stream)) return rc;
  if (need == 0) return 0;
  // few blocks are spread over more workgroups
  const int rows = plan.blocks * c.kv_heads * p.block_rows > 16384 ? 32 : kThreads / (c.head_dim / 4);
  const int chunks = (p.block_rows + rows - 1) / rows;
  const dim3 grid(static_cast<unsigned>(plan.blocks * c.kv_heads * chunks));
  if (plan.stage == 256) hipLaunchKernelGGL(paged_tokens_merge_kernel<256>, grid, dim3(kThreads), 0, stream, p, rows, chunks);
  else if (plan.stage == 128) hipLaunchKernelGGL(paged_tokens_merge_kernel<128>, grid, dim3(kThreads), 0, stream, p, rows, chunks);
  else hipLaunchKernelGGL(paged_tokens_merge_kernel<64>, grid, dim3(kThreads), 0, stream, p, rows, chunks);
  return hip_status(hipGetLastError(), "paged_tokens_merge launch");
}

}  // namespace
}  // namespace kvssd

using namespace kvssd;

extern "C" {

__attribute__((visibility("default"))) int kvssd_hip_paged_tokens_workspace_bytes(const kvssd_paged_cache* cache,
                                                                                  const kvssd_paged_tokens_args* args,
                                                                                  size_t* bytes) {
  if (int rc = check_paged_cache(cache)) return rc;
  if (args == nullptr || bytes == nullptr) return arg_error("arguments are NULL");
  Plan plan;
  if (int rc = plan_of(*cache, *args, &plan)) return rc;
  *bytes = plan.o_bytes + plan.ml_bytes;
  return 0;
}

__attribute__((visibility("default"))) int kvssd_hip_paged_tokens(const kvssd_paged_cache* cache,
                                                                  const kvssd_paged_tokens_args* args, void* stream) {
  if (int rc = check_paged_cache(cache)) return rc;
  if (args == nullptr) return arg_error("arguments are NULL");
  if (args->tokens == 0) return 0;
  if (!args->query.data || !args->out || !args->lse || !args->offsets) return arg_error("a required buffer pointer is NULL");
  return launch_paged_tokens(*cache, *args, static_cast<hipStream_t>(stream));
}

}  // extern "C"
