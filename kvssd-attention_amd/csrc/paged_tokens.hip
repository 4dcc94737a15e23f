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

constexpr int kLocate = 1024;  // threads
constexpr int kCounted = kWave - 2;  // sequences that a workgroup counts by itself, at one look

// The items' and blocks' first numbers of every sequence, where they are so many that a workgroup should not count them by
// itself, at about a microsecond for every 64 of them (256 sequences of 8 tokens: 425 us without this launch, 341 with it;
// 64: no difference).  One workgroup, bound by the round trips of offsets and lengths.
template <int STAGE>
__global__ __launch_bounds__(kLocate) void paged_tokens_locate_kernel(PagedTokensParams p) {
  constexpr int kWaves = kLocate / kWave, kMost = 1 << 30;
  __shared__ float work_s[kWaves], blocks_s[kWaves];
  __shared__ int items_s[kWaves], sums_s[kWaves];
  const int tid = threadIdx.x, lane = tid % kWave, wave = tid / kWave, sequences = p.c.sequences + 2;
  float work = 0.0f, blocks = 0.0f;
  for (int s = tid; s < sequences; s += kLocate) {
    const TokenSpan span = token_span(p, s);
    const int n = blocks_of(p, span);
    if (n == 0) continue;
    blocks += static_cast<float>(n);
    work += static_cast<float>(n) * static_cast<float>(stages_of(p, span, n - 1, STAGE).count());
  }
  work = wave_sum(work);
  blocks = wave_sum(blocks);
  if (lane == 0) {
    work_s[wave] = work;
    blocks_s[wave] = blocks;
  }
  __syncthreads();
  work = blocks = 0.0f;
  for (int w = 0; w < kWaves; ++w) {
    work += work_s[w];
    blocks += blocks_s[w];
  }
  const int size = size_of_runs(p, work, blocks);
  int32_t* const item_starts = p.starts;
  int32_t* const block_starts = p.starts + sequences + 1;
  if (tid == 0) p.starts[2 * sequences + 2] = size;
  int items = 0, sums = 0;  // of the sequences before; more than a call takes count as 2^30
  for (int s0 = 0; s0 < sequences; s0 += kLocate) {
    const TokenSpan span = token_span(p, s0 + tid);  // (none behind the last)
    const int n = blocks_of(p, span);
    const int64_t all = static_cast<int64_t>(n) * runs_of_sequence<STAGE>(p, span, n, size);
    const int own = all < (1 << 24) ? static_cast<int>(all) : 1 << 24;
    const int item_end = wave_prefix(own), block_end = wave_prefix(n);
    __syncthreads();
    if (lane == kWave - 1) {
      items_s[wave] = item_end;
      sums_s[wave] = block_end;
    }
    __syncthreads();
    int before = items, blocks_before = sums;
    for (int w = 0; w < kWaves; ++w) {
      if (w == wave) {
        before = items;
        blocks_before = sums;
      }
      items = min(items + items_s[w], kMost);
      sums = min(sums + sums_s[w], kMost);
    }
    if (s0 + tid < sequences) {
      item_starts[s0 + tid] = min(before + item_end - own, kMost);
      block_starts[s0 + tid] = min(blocks_before + block_end - n, kMost);
    }
  }
  if (tid == 0) {
    item_starts[sequences] = items;
    block_starts[sequences] = sums;
  }
}

// A row is `unit` threads' (d / 4, up to a power of two), 4 dims each, of every `splits`-th run, kAhead runs' sums read before
// the first one's weight is known; a lane a run forms the weights.  With few rows, whose time is the latency of these reads,
// a row's runs are split between the units of a workgroup (8 tokens of 4 heads at 4,096 tokens of context, 17 runs: 6.5 us;
// 33 runs one after the other took 16).  With many it is bound by the partials' way through memory: 16 trees of up to 32
// tokens 20 us.
template <int STAGE>
__global__ __launch_bounds__(kThreads) void paged_tokens_merge_kernel(PagedTokensParams p, int rows, int chunks, int unit_log2,
                                                                      int splits_log2) {
  constexpr int kAhead = 8;
  __shared__ f32x4 acc_s[kThreads];
  __shared__ float most_s[kThreads / 8], sum_s[kThreads / 8];
  const int chunk = blockIdx.x % chunks, kvh = blockIdx.x / chunks % p.c.kv_heads;
  int first;
  const TokenItem work = find_item<STAGE>(p, blockIdx.x / chunks / p.c.kv_heads, true, &first);
  if (work.seq < 0 || work.runs == 1) return;
  const int d = p.c.head_dim, tid = threadIdx.x;
  const int unit = tid >> unit_log2, i = tid - (unit << unit_log2), dim = i * 4, size = 1 << unit_log2;
  const int side_log2 = 8 - unit_log2 - splits_log2;  // rows side by side (of 256 threads)
  const int own = unit & ((1 << side_log2) - 1), split = unit >> side_log2;
  const int end = min(min(work.span.count * p.gq - work.block * p.block_rows, p.block_rows), (chunk + 1) * rows);
  const int64_t step = static_cast<int64_t>(p.c.kv_heads) * p.block_rows << splits_log2;  // rows to the unit's next run
  const int64_t at0 = (static_cast<int64_t>(first + split) * p.c.kv_heads + kvh) * p.block_rows;
  const int runs = work.runs > split ? ((work.runs - 1 - split) >> splits_log2) + 1 : 0;  // of the unit
  for (int row0 = chunk * rows; row0 < end; row0 += 1 << side_log2) {
    const int row = row0 + own;
    f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
    float most = -INFINITY, sum = 0.0f;
    if (row < end) {
      const f32x2* ml = reinterpret_cast<const f32x2*>(p.part_ml) + at0 + row;
      const float* o = p.part_o + (at0 + row) * d + dim;
      float w = 0.0f;  // of the unit's run n0 / size * size + i
      for (int n0 = 0; n0 < runs; n0 += kAhead) {
        f32x4 v[kAhead];
#pragma unroll
        for (int k = 0; k < kAhead; ++k)
          if (n0 + k < runs && dim < d) v[k] = *reinterpret_cast<const f32x4*>(o + (n0 + k) * step * d);
        if (n0 % size == 0) {
          const f32x2 x = n0 + i < runs ? ml[(n0 + i) * step] : f32x2{-INFINITY, 0.0f};
          float here = x[1] != 0.0f ? x[0] : -INFINITY;  // (a NaN sum takes part)
          for (int k = 1; k < size; k *= 2) here = fmaxf(here, __shfl_xor(here, k, kWave));
          here = fmaxf(here, most);
          w = x[1] != 0.0f ? exp2f(x[0] - here) : 0.0f;
          if (sum != 0.0f) {
            const float scale = exp2f(most - here);
            acc *= scale;
            sum *= scale;
          }
          most = here;
          float more = x[1] != 0.0f ? w * x[1] : 0.0f;
          for (int k = 1; k < size; k *= 2) more += __shfl_xor(more, k, kWave);
          sum += more;
        }
#pragma unroll
        for (int k = 0; k < kAhead; ++k) {
          const float of = __shfl(w, n0 % size + k, size);
          if (n0 + k < runs) acc += of * v[k];  // (sums that are not finite take part whatever their weight, as slots' values do)
        }
      }
    }
    if (splits_log2 > 0) {
      acc_s[tid] = acc;
      if (i == 0) {
        most_s[unit] = most;
        sum_s[unit] = sum;
      }
      __syncthreads();
      if (split == 0) {
        float all = -INFINITY;
        for (int u = own; u < kThreads >> unit_log2; u += 1 << side_log2)
          if (sum_s[u] != 0.0f) all = fmaxf(all, most_s[u]);
        acc = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        sum = 0.0f;
        for (int u = own; u < kThreads >> unit_log2; u += 1 << side_log2) {
          if (sum_s[u] == 0.0f) continue;
          const float of = exp2f(most_s[u] - all);
          acc += of * acc_s[(u << unit_log2) + i];
          sum += of * sum_s[u];
        }
        most = all;
      }
      __syncthreads();
    }
    if (split == 0 && row < end && dim < d) {
      const int in_seq = work.block * p.block_rows + row, token = in_seq / p.gq;
      const int64_t to = (work.span.begin + token) * p.query_heads + kvh * p.gq + in_seq - token * p.gq;
#pragma unroll
      for (int x = 0; x < 4; ++x) store_out(p.out, p.out_dtype, to * d + dim + x, sum == 0.0f ? 0.0f : acc[x] / sum);
      if (dim == 0) p.lse[to] = sum == 0.0f ? -INFINITY : kLn2 * (most + log2f(sum));
    }
  }
}

size_t aligned(size_t n) { return (n + 255) & ~static_cast<size_t>(255); }

struct Plan {
  PagedTokensParams p;
  int dp, waves, stage;
  bool precise, own;  // `own`: every wave unpacks slots of its own
  int64_t blocks;  // at most
  size_t o_bytes, ml_bytes, starts_bytes;
  size_t bytes() const { return o_bytes + ml_bytes + starts_bytes; }
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

  // rows of a workgroup, after a sequence's rows on average: 256 where they fill half of them, 128 where they fill a quarter
  // (16 trees of up to 32 tokens and 4 heads 126 us, in blocks of 32 151; 256 trees of 16 tokens 170 and 199, though 16 of
  // them 97 and 85), else 32
  const int64_t each = (a.tokens * p.gq + c.sequences - 1) / c.sequences;
  plan->own = each <= 32 && !plan->precise && plan->dp <= 128;
  plan->waves = each > 128 && !plan->precise && plan->dp <= 128 ? 8 : 4;
  const int stage = plan->stage = plan->own ? plan->waves * 32 : tokens_stage(plan->dp, plan->waves);
  p.row_tiles = each > 128 ? plan->waves : each > 32 ? 4 : 1;
  p.parts = plan->own || plan->waves / p.row_tiles < stage / 64 ? plan->waves / p.row_tiles : stage / 64;
  p.block_rows = 32 * p.row_tiles;
  p.block_log2 = 31 - __builtin_clz(p.block_rows);
  plan->blocks = a.tokens * p.gq / p.block_rows + c.sequences + 2;

  // runs, where blocks alone would leave compute units idle
  auto stages = [&](int64_t n) { return (n + stage - 1) / stage; };
  int64_t longest = a.max_length > 0 && a.max_length < p.capacity ? a.max_length : p.capacity;
  int64_t total = a.total_tokens > 0 && a.total_tokens < longest * c.sequences ? a.total_tokens : longest * c.sequences;
  if (p.window > 0) {
    const int64_t seen = int64_t{p.window} + p.block_rows / p.gq + p.sink + 3 * stage;
    longest = longest < seen ? longest : seen;
    total = total < longest * c.sequences ? total : longest * c.sequences;
  }
  const int64_t likely = (each + p.block_rows - 1) / p.block_rows * c.sequences;  // blocks
  const int64_t work = (total / stage + c.sequences) * (likely / c.sequences);    // stages of all blocks
  // workgroups that run at a time (LDS and registers); one or two rounds of them where blocks are few, four of more, whose
  // lengths differ (8 tokens over 4,096 in runs of one stage, which are more than compute units, 25 us, of two 23, of three
  // 25; 16 such trees over 1,000 to 2,000 in a round 45, in two 53, 64 in four 91, in two 89; 16 trees of up to 32 in runs
  // of 8, 15 and 28 stages 176, 152 and 151)
  const int64_t at_once = plan->waves == 4 && !plan->precise && plan->dp <= 128 ? 512 : 256;
  const int64_t wanted = (likely * c.kv_heads >= at_once ? 4 : plan->own ? 1 : 2) * at_once / c.kv_heads;
  const int64_t cut = wanted - likely > wanted / 2 ? wanted - likely : (wanted + 1) / 2;
  int64_t size = (work + cut - 1) / (cut > 0 ? cut : 1);
  if (size < 1) size = 1;
  if (size < 2 && work * c.kv_heads > 256) size = 2;  // (a run's start takes as long as two stages)
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
  if (c.sequences > kCounted) plan->starts_bytes = aligned((2 * (static_cast<size_t>(c.sequences) + 3) + 1) * sizeof(int32_t));
  return 0;
}

int launch_paged_tokens(const kvssd_paged_cache& c, const kvssd_paged_tokens_args& a, hipStream_t stream) {
  Plan plan;
  if (int rc = plan_of(c, a, &plan)) return rc;
  PagedTokensParams& p = plan.p;
  const size_t need = plan.bytes();
  if (need > 0 && (a.workspace == nullptr || a.workspace_bytes < need))
    return arg_error("workspace too small: need " + std::to_string(need) + " bytes");
  if (reinterpret_cast<uintptr_t>(a.workspace) % 256) return arg_error("workspace must be 256-byte aligned");
  if (!heads_vector(a.query, dtype_bytes(a.query_dtype), false))
    return arg_error("query must be 16-byte aligned, as must its tokens and heads be");
  if (reinterpret_cast<uintptr_t>(a.out) % 16) return arg_error("out must be 16-byte aligned");
  p.part_o = static_cast<float*>(a.workspace);
  p.part_ml = reinterpret_cast<float*>(static_cast<char*>(a.workspace) + plan.o_bytes);
  const auto of_stage = [&](auto of256, auto of128, auto of64) { return plan.stage == 256 ? of256 : plan.stage == 128 ? of128 : of64; };
  if (plan.starts_bytes > 0) {
    p.starts = reinterpret_cast<int32_t*>(static_cast<char*>(a.workspace) + plan.o_bytes + plan.ml_bytes);
    const auto locate = of_stage(paged_tokens_locate_kernel<256>, paged_tokens_locate_kernel<128>, paged_tokens_locate_kernel<64>);
    hipLaunchKernelGGL(locate, dim3(1), dim3(kLocate), 0, stream, p);
    if (int rc = hip_status(hipGetLastError(), "paged_tokens_locate launch")) return rc;
  }
  const int64_t work = static_cast<int64_t>(p.items) * c.kv_heads;
  const unsigned groups = static_cast<unsigned>(c.kv_heads % 2 ? work : (work + 15) / 16 * 16);
  const auto launch = plan.dp == 64    ? launch_paged_tokens_dims<64>
                      : plan.dp == 128 ? launch_paged_tokens_dims<128>
                                       : launch_paged_tokens_dims<256>;
  if (int rc = launch(p, plan.waves, plan.precise, plan.own, groups, stream)) return rc;
  if (plan.o_bytes == 0) return 0;
  int unit_log2 = 3;  // 8 to 64 threads a row
  while ((4 << unit_log2) < c.head_dim) ++unit_log2;
  // few rows' runs are split between units, and their rows spread over more workgroups
  const bool few = plan.blocks * c.kv_heads * p.block_rows <= 16384;
  const int splits_log2 = few ? 2 : 0, rows = few ? kThreads >> unit_log2 >> splits_log2 : 32;
  const int chunks = (p.block_rows + rows - 1) / rows;
  const dim3 grid(static_cast<unsigned>(plan.blocks * c.kv_heads * chunks));
  const auto merge = of_stage(paged_tokens_merge_kernel<256>, paged_tokens_merge_kernel<128>, paged_tokens_merge_kernel<64>);
  hipLaunchKernelGGL(merge, grid, dim3(kThreads), 0, stream, p, rows, chunks, unit_log2, splits_log2);
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
  *bytes = plan.bytes();
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
