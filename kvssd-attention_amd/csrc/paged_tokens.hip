// Attention of many new tokens a sequence over its packed pages, their own
// among them: prompts and chunks of prompts (causal) and trees of drafted tokens,
// with or without a sliding window and sinks.
//
//   s_it = sm_scale q_i.k_t over the slots t that token i sees,
//   out_i = sum_t softmax(s_i)_t v_t,  lse_i = log sum_t e^s_it
//
// The plain form: a wave a (token, query head); a lane a slot for the scores, a
// lane a few dims for the values.
#include "paged_decode.hpp"

namespace kvssd {
namespace {

struct TokensParams {
  kvssd_paged_cache c;
  kvssd_heads query;
  void* out;
  float* lse;
  const int32_t* offsets;
  const int32_t* parents;
  int64_t tokens;
  int capacity, window, sink;
  int query_heads, gq, query_dtype, out_dtype;
  int groups, group_log2;
  float scale_log2;
};

__device__ __forceinline__ float query_at(const void* q, int dtype, int64_t at) {
  if (dtype == KVSSD_DTYPE_F32) return static_cast<const float*>(q)[at];
  if (dtype == KVSSD_DTYPE_F16) return static_cast<float>(static_cast<const _Float16*>(q)[at]);
  return __builtin_bit_cast(float, static_cast<uint32_t>(static_cast<const uint16_t*>(q)[at]) << 16);
}

__global__ __launch_bounds__(kWave) void paged_tokens_kernel(TokensParams p) {
  const kvssd_paged_cache& c = p.c;
  const int lane = threadIdx.x;
  const int64_t t = blockIdx.x / p.query_heads;
  const int h = blockIdx.x % p.query_heads, kvh = h / p.gq;
  const int d = c.head_dim, mid = 1 << (c.bits - 1), mask = (1 << c.bits) - 1;
  int seq = -1;
  if (t >= p.offsets[0] && t < p.offsets[c.sequences]) {
    int lo = 0, hi = c.sequences;
    while (hi - lo > 1) {
      const int at = (lo + hi) / 2;
      if (p.offsets[at] <= t) lo = at;
      else hi = at;
    }
    seq = lo;
  }
  float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f}, m = -INFINITY, l = 0.0f;
  if (seq >= 0) {
    const int begin = p.offsets[seq], n = p.offsets[seq + 1] - begin;
    const int i = static_cast<int>(t - begin);
    const int length = paged_length(c.lengths, seq, p.capacity);
    const int base = length - n;
    const int32_t* parents = p.parents ? p.parents + begin : nullptr;
    int position = base + i;
    if (parents != nullptr) {
      position = base;
      for (int up = parent_of(parents, i); up >= 0; up = parent_of(parents, up)) ++position;
    }
    const int32_t* pages = c.page_table + static_cast<int64_t>(seq) * c.max_pages;
    const int64_t q0 = t * p.query.token_stride + h * p.query.head_stride;
    for (int s0 = 0; s0 <= base + i; s0 += kWave) {
      const int slot = s0 + lane;
      bool seen = slot <= base + i && slot < length;
      int where = slot;
      if (seen && parents != nullptr && slot >= base) {
        int x = i;
        where = position;
        while (x > slot - base) {
          x = parent_of(parents, x);
          --where;
        }
        seen = x == slot - base;
      }
      if (p.window > 0) seen = seen && (where > position - p.window || where < p.sink);
      int64_t row = -1;
      if (seen) {
        const int page = pages[slot / c.page_tokens];
        if (page >= 0 && page < c.num_pages) row = static_cast<int64_t>(page) * c.page_tokens + slot % c.page_tokens;
      }
      float score = -INFINITY;
      if (row >= 0) {
        const uint8_t* codes = c.packed_k + (row * c.kv_heads + kvh) * (d * c.bits / 8);
        const uint16_t* scales = c.scales_k + (row * c.kv_heads + kvh) * p.groups;
        score = 0.0f;
        for (int g = 0; g < p.groups; ++g) {
          float sum = 0.0f;
          for (int x = 0; x < c.group_size; ++x) {
            const int dim = g * c.group_size + x;
            const int code = codes[dim * c.bits / 8] >> (dim * c.bits % 8) & mask;
            sum = __builtin_fmaf(query_at(p.query.data, p.query_dtype, q0 + dim), static_cast<float>(code - mid), sum);
          }
          score = __builtin_fmaf(sum, half_bits_to_float(scales[g]), score);
        }
        score *= p.scale_log2;
      }
      const float m_new = fmaxf(m, wave_max(score));
      const uint64_t live = __ballot(row >= 0);
      if (live == 0) continue;
      const float alpha = m == -INFINITY ? 0.0f : exp2f(m - m_new);
      const float e = row >= 0 ? exp2f(score - (m_new == -INFINITY ? 0.0f : m_new)) : 0.0f;
      m = m_new;
      l = l * alpha + wave_sum(e);
      for (int x = 0; x < 4; ++x) acc[x] *= alpha;
      for (int k = 0; k < kWave; ++k) {
        if (!(live >> k & 1)) continue;
        const float w = __shfl(e, k, kWave);
        const int64_t r = __shfl(row, k, kWave);
        for (int x = 0; x < 4; ++x) {
          const int dim = lane + x * kWave;
          if (dim >= d) break;
          const int code = c.packed_v[(r * c.kv_heads + kvh) * (d * c.bits / 8) + dim * c.bits / 8] >> (dim * c.bits % 8) & mask;
          const float scale = half_bits_to_float(c.scales_v[(r * c.kv_heads + kvh) * p.groups + (dim >> p.group_log2)]);
          acc[x] = __builtin_fmaf(w, static_cast<float>(code - mid) * scale, acc[x]);
        }
      }
    }
  }
  const int64_t row = t * p.query_heads + h;
  for (int x = 0; x < 4; ++x) {
    const int dim = lane + x * kWave;
    if (dim < d) store_out(p.out, p.out_dtype, row * d + dim, l == 0.0f ? 0.0f : acc[x] / l);
  }
  if (lane == 0) p.lse[row] = l == 0.0f ? -INFINITY : kLn2 * (m + log2f(l));
}

int plan_of(const kvssd_paged_cache& c, const kvssd_paged_tokens_args& a, TokensParams* p) {
  if (a.query.heads <= 0 || a.query.heads % c.kv_heads) return arg_error("query heads must be divisible by KV heads");
  if (!paged_dtype(a.query_dtype)) return arg_error("unsupported query dtype");
  if (a.out_query_dtype != 0 && a.out_query_dtype != 1) return arg_error("out_query_dtype must be 0 or 1");
  if (a.max_length < 0 || a.total_tokens < 0) return arg_error("max_length and total_tokens must be >= 0");
  if (a.window < 0 || a.sink < 0) return arg_error("window and sink must be >= 0");
  if (a.tokens < 0 || a.tokens * a.query.heads > (int64_t{1} << 30)) return arg_error("too many tokens for one call");
  *p = TokensParams{};
  p->c = c;
  p->query = a.query;
  p->out = a.out;
  p->lse = a.lse;
  p->offsets = a.offsets;
  p->parents = a.parents;
  p->tokens = a.tokens;
  p->capacity = static_cast<int>(paged_capacity(c));
  p->window = a.window;
  p->sink = a.sink;
  p->query_heads = a.query.heads;
  p->gq = a.query.heads / c.kv_heads;
  p->query_dtype = a.query_dtype;
  p->out_dtype = a.out_query_dtype ? a.query_dtype : KVSSD_DTYPE_F32;
  p->groups = c.head_dim / c.group_size;
  while ((1 << p->group_log2) < c.group_size) ++p->group_log2;
  p->scale_log2 = static_cast<float>(a.sm_scale) * kLog2e;
  return 0;
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
  TokensParams p;
  if (int rc = plan_of(*cache, *args, &p)) return rc;
  *bytes = 0;
  return 0;
}

__attribute__((visibility("default"))) int kvssd_hip_paged_tokens(const kvssd_paged_cache* cache,
                                                                  const kvssd_paged_tokens_args* args, void* stream) {
  if (int rc = check_paged_cache(cache)) return rc;
  if (args == nullptr) return arg_error("arguments are NULL");
  TokensParams p;
  if (int rc = plan_of(*cache, *args, &p)) return rc;
  if (p.tokens == 0) return 0;
  if (!args->query.data || !args->out || !args->lse || !args->offsets) return arg_error("a required buffer pointer is NULL");
  if (reinterpret_cast<uintptr_t>(args->workspace) % 256) return arg_error("workspace must be 256-byte aligned");
  hipLaunchKernelGGL(paged_tokens_kernel, dim3(static_cast<unsigned>(p.tokens * p.query_heads)), dim3(kWave), 0,
                     static_cast<hipStream_t>(stream), p);
  return hip_status(hipGetLastError(), "paged_tokens launch");
}

}  // extern "C"
