// New tokens into a paged packed cache: keys rotated, keys and values
// quantised into their sequences' pages, queries rotated, in one launch.
//
// A workgroup takes one token (or a few of a prompt): where the token goes and
// its sines are formed once, then each thread takes words of codes (8 values
// in INT4, 16 in INT2), those of a group side by side in the wave so that the
// group's maximum is a few lane exchanges (quant_ops.hpp).  A key's word needs
// the other half of its pairs: half layouts load it too (the lines are in the
// cache, their neighbours' threads read them), so that no value passes between
// threads between rotation and coding.  The rotated key is rounded to its type
// first: the codes are those of a key rotated by kvssd_hip_rotary and quantised
// by kvssd_hip_quantize, bit for bit.
#include "paged.hpp"
#include "rotary_ops.hpp"

namespace kvssd {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxTurns = 512;
constexpr int kMaxTokens = 4;  // of a workgroup

struct AppendParams {
  kvssd_paged_cache c;
  kvssd_heads keys, values, query;
  const double* frequencies;  // nullptr: no rotation
  double magnitude;
  const int32_t* offsets;
  const int32_t* first_positions;
  int32_t* lengths_out;
  RotaryShape shape;  // of the query's items
  int64_t tokens;
  int inverse, per_group, capacity;
  int words, lanes, groups;  // code words of a head's row, words of a group, groups of a row
  int query_heads;
};

// Sequence of token t: the b with offsets[b] <= t < offsets[b + 1], -1 if none.
__device__ __forceinline__ int sequence_of(const int32_t* offsets, int sequences, int64_t t) {
  int lo = 0, hi = sequences;  // offsets[lo] <= t < offsets[hi], if anywhere
  if (t < offsets[0] || t >= offsets[sequences]) return -1;
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (offsets[mid] <= t) lo = mid;
    else hi = mid;
  }
  return lo;
}

// A word's values: loaded, and rotated if `turns`.
template <typename T, int N, bool VEC>
__device__ __forceinline__ void word_values(const T* x, int d0, const RotaryShape& s, const Turn* turns, float (&out)[N]) {
  if constexpr (VEC) {  // no word mixes low, high and unturned values, and all loads are 16-byte aligned
    T a[N];
    load_values(x + d0, a);
    if (turns == nullptr || d0 >= 2 * s.pairs) {
#pragma unroll
      for (int i = 0; i < N; ++i) out[i] = to_f32(a[i]);
    } else if (s.interleaved) {
#pragma unroll
      for (int i = 0; i < N; i += 2) {
        const Turn t = turns[d0 / 2 + i / 2];
        out[i] = to_f32(store_cast<T>(turn_low(to_f32(a[i]), to_f32(a[i + 1]), t)));
        out[i + 1] = to_f32(store_cast<T>(turn_high(to_f32(a[i]), to_f32(a[i + 1]), t)));
      }
    } else {
      const bool high = d0 >= s.pairs;
      const int p0 = high ? d0 - s.pairs : d0;
      T b[N];
      load_values(x + (high ? p0 : d0 + s.pairs), b);
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const Turn t = turns[p0 + i];
        const float own = to_f32(a[i]), other = to_f32(b[i]);
        out[i] = to_f32(store_cast<T>(high ? turn_high(other, own, t) : turn_low(own, other, t)));
      }
    }
  } else {
    for (int i = 0; i < N; ++i) {
      const int d = d0 + i;
      const float own = to_f32(x[d]);
      if (turns == nullptr || d >= 2 * s.pairs) {
        out[i] = own;
        continue;
      }
      const bool high = s.interleaved ? d % 2 : d >= s.pairs;
      const int p = s.interleaved ? d / 2 : (high ? d - s.pairs : d);
      const float other = to_f32(x[s.interleaved ? d ^ 1 : (high ? p : d + s.pairs)]);
      out[i] = to_f32(store_cast<T>(high ? turn_high(other, own, turns[p]) : turn_low(own, other, turns[p])));
    }
  }
}

template <typename T, int BITS, bool VEC>
__global__ __launch_bounds__(kThreads) void paged_append_kernel(AppendParams p) {
  constexpr int kVals = 32 / BITS;
  constexpr int kItem = VEC ? 16 / sizeof(T) : 1;
  __shared__ Turn turns[kMaxTurns];
  __shared__ int64_t row_s[kMaxTokens];  // row of the pool, -1: dropped
  __shared__ double position_s[kMaxTokens];
  const kvssd_paged_cache& c = p.c;
  const int64_t t0 = static_cast<int64_t>(blockIdx.x) * p.per_group;
  const int n = static_cast<int>(p.tokens - t0 < p.per_group ? p.tokens - t0 : p.per_group);
  if (static_cast<int>(threadIdx.x) < n) {
    const int64_t t = t0 + threadIdx.x;
    const int b = p.offsets ? sequence_of(p.offsets, c.sequences, t) : static_cast<int>(t);
    int64_t row = -1;
    double position = 0.0;
    if (b >= 0) {
      const int64_t nth = p.offsets ? t - p.offsets[b] : 0;
      const int length = paged_length(c.lengths, b, p.capacity);
      const int64_t slot = length + nth;
      const int64_t where = p.first_positions ? p.first_positions[b] + nth : slot;
      position = static_cast<double>(where);
      if (slot < p.capacity) {
        const int page = c.page_table[static_cast<int64_t>(b) * c.max_pages + slot / c.page_tokens];
        if (page >= 0 && page < c.num_pages) row = static_cast<int64_t>(page) * c.page_tokens + slot % c.page_tokens;
        const int64_t at = static_cast<int64_t>(b) * p.capacity + slot;
        if (c.weights) c.weights[at] = 0.0f;
        if (c.positions) c.positions[at] = static_cast<int32_t>(where);
      }
      // one token a sequence: this thread is the only one that reads lengths[b]
      if (p.lengths_out && !p.offsets) p.lengths_out[b] = length < p.capacity ? length + 1 : length;
    }
    row_s[threadIdx.x] = row;
    position_s[threadIdx.x] = position;
  }
  if (p.offsets && p.lengths_out) {
    for (int64_t b = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x; b < c.sequences;
         b += static_cast<int64_t>(gridDim.x) * kThreads) {
      const int64_t count = static_cast<int64_t>(p.offsets[b + 1]) - p.offsets[b];
      const int64_t after = paged_length(c.lengths, static_cast<int>(b), p.capacity) + (count > 0 ? count : 0);
      p.lengths_out[b] = static_cast<int32_t>(after < p.capacity ? after : p.capacity);
    }
  }
  __syncthreads();
  if (p.frequencies) {
    for (int i = threadIdx.x; i < n * p.shape.pairs; i += kThreads)
      turns[i] = make_turn(position_s[i / p.shape.pairs], p.frequencies[i % p.shape.pairs], p.magnitude, p.inverse);
    __syncthreads();
  }
  const int coded = c.kv_heads * p.words;  // words of a token's keys, and of its values
  const int per_token = 2 * coded + p.query_heads * p.shape.items;
  for (int i = threadIdx.x; i < n * per_token; i += kThreads) {
    const int tok = i / per_token;
    int rest = i % per_token;
    const Turn* turn = p.frequencies ? turns + tok * p.shape.pairs : nullptr;
    if (rest < 2 * coded) {
      const int64_t row = row_s[tok];
      if (row < 0) continue;  // the same for every lane of a group
      const bool is_v = rest >= coded;
      if (is_v) rest -= coded;
      const int head = rest / p.words, word = rest % p.words;
      const kvssd_heads& h = is_v ? p.values : p.keys;
      const T* x = static_cast<const T*>(h.data) + (t0 + tok) * h.token_stride + head * h.head_stride;
      float v[kVals];
      word_values<T, kVals, VEC>(x, word * kVals, p.shape, is_v ? nullptr : turn, v);
      float amax = 0.0f;
#pragma unroll
      for (int k = 0; k < kVals; ++k) amax = fmaxf(amax, fabsf(v[k]));
      const float s32 = group_scale<BITS>(lanes_max(amax, p.lanes));
      const uint32_t code = code_word<T, BITS>(v, s32);
      const int64_t at = row * c.kv_heads + head;
      uint8_t* packed = (is_v ? c.packed_v : c.packed_k) + (at * p.words + word) * 4;
      __builtin_memcpy(__builtin_assume_aligned(packed, 4), &code, 4);
      if ((word & (p.lanes - 1)) == 0)
        (is_v ? c.scales_v : c.scales_k)[at * p.groups + word / p.lanes] =
            __builtin_bit_cast(uint16_t, static_cast<_Float16>(s32));
    } else {
      rest -= 2 * coded;
      const int head = rest / p.shape.items, item = rest % p.shape.items;
      rotary_item<T, kItem>(p.shape, item,
                            static_cast<const T*>(p.query.data) + (t0 + tok) * p.query.token_stride +
                                head * p.query.head_stride,
                            static_cast<T*>(p.query.out) + (t0 + tok) * p.query.out_token_stride +
                                head * p.query.out_head_stride,
                            turn);
    }
  }
}

template <typename T>
void launch_typed(AppendParams& p, const kvssd_paged_append_args& a, hipStream_t stream) {
  const int item = 16 / sizeof(T), vals = 32 / p.c.bits;
  bool vec = heads_vector(p.keys, sizeof(T), false) && heads_vector(p.values, sizeof(T), false) &&
             (p.query_heads == 0 || heads_vector(p.query, sizeof(T), true));
  if (a.rotary) {
    const int pairs = a.rotary->rotary_dim / 2;
    vec = vec && pairs % item == 0 && (a.rotary->head_dim - a.rotary->rotary_dim) % item == 0;
    vec = vec && (a.rotary->interleaved ? a.rotary->rotary_dim % vals == 0 : pairs % vals == 0);
    p.shape = rotary_shape(*a.rotary, vec ? item : 1);
  }
  int per = p.shape.pairs ? kMaxTurns / p.shape.pairs : kMaxTokens;
  per = per < kMaxTokens ? per : kMaxTokens;
  p.per_group = p.tokens >= 2048 ? per : 1;  // as the rotary kernel's
  const int64_t blocks = (p.tokens + p.per_group - 1) / p.per_group;
  const dim3 grid(static_cast<unsigned>(blocks > 0 ? blocks : 1));  // no token: lengths_out alone
  if (p.c.bits == 4) {
    if (vec) hipLaunchKernelGGL((paged_append_kernel<T, 4, true>), grid, dim3(kThreads), 0, stream, p);
    else hipLaunchKernelGGL((paged_append_kernel<T, 4, false>), grid, dim3(kThreads), 0, stream, p);
  } else {
    if (vec) hipLaunchKernelGGL((paged_append_kernel<T, 2, true>), grid, dim3(kThreads), 0, stream, p);
    else hipLaunchKernelGGL((paged_append_kernel<T, 2, false>), grid, dim3(kThreads), 0, stream, p);
  }
}

}  // namespace

int check_paged_cache(const kvssd_paged_cache* c) {
  if (c == nullptr) return arg_error("cache is NULL");
  if (c->bits != 2 && c->bits != 4) return arg_error("bits must be 2 or 4");
  if (c->kv_heads <= 0 || c->kv_heads > 65536 || c->num_pages <= 0 || c->page_tokens <= 0)
    return arg_error("packed pages must match [pages,tokens,kv_heads,packed_dim]");
  if (c->head_dim < 32 || c->head_dim > 256 || c->head_dim % 32)
    return arg_error("head_dim must be a multiple of 32 up to 256");
  if (c->group_size < 32 || (c->group_size & (c->group_size - 1)) || c->head_dim % c->group_size)
    return arg_error("group_size must be a power of two, 32 or more, that divides head_dim");
  if (c->sequences <= 0 || c->sequences > (1 << 20) || c->max_pages <= 0)
    return arg_error("page_table must be [sequences, max_pages] with at most 2^20 sequences");
  if (paged_capacity(*c) > (int64_t{1} << 30)) return arg_error("a sequence may hold at most 2^30 slots");
  if (static_cast<int64_t>(c->num_pages) * c->page_tokens > (int64_t{1} << 30))
    return arg_error("a pool may hold at most 2^30 slots");
  if (static_cast<int64_t>(c->num_pages) * c->page_tokens * c->kv_heads == 1 && (c->head_dim / c->group_size) % 2)
    return arg_error("a pool of one row needs an even number of scale groups");  // (they are read 4 bytes at a time)
  if (!c->packed_k || !c->packed_v || !c->scales_k || !c->scales_v || !c->page_table || !c->lengths)
    return arg_error("a required buffer pointer is NULL");
  for (const void* ptr : {static_cast<const void*>(c->packed_k), static_cast<const void*>(c->packed_v),
                          static_cast<const void*>(c->scales_k), static_cast<const void*>(c->scales_v)})
    if (reinterpret_cast<uintptr_t>(ptr) % 16) return arg_error("pages must be 16-byte aligned");
  return 0;
}

int launch_paged_append(const kvssd_paged_cache& c, const kvssd_paged_append_args& a, hipStream_t stream) {
  AppendParams p{};
  p.c = c;
  p.keys = a.keys;
  p.values = a.values;
  p.query = a.query;
  p.query_heads = a.query.data ? a.query.heads : 0;
  p.offsets = a.offsets;
  p.first_positions = a.first_positions;
  p.lengths_out = a.lengths_out;
  p.tokens = a.tokens;
  p.capacity = static_cast<int>(paged_capacity(c));
  p.words = c.head_dim * c.bits / 32;
  p.lanes = c.group_size * c.bits / 32;
  p.groups = c.head_dim / c.group_size;
  if (a.rotary) {
    p.frequencies = a.rotary->frequencies;
    p.magnitude = a.rotary->magnitude;
    p.inverse = a.rotary->inverse;
  }
  switch (a.dtype) {
    case KVSSD_DTYPE_F16:
      launch_typed<_Float16>(p, a, stream);
      break;
    case KVSSD_DTYPE_BF16:
      launch_typed<uint16_t>(p, a, stream);
      break;
    default:
      launch_typed<float>(p, a, stream);
  }
  return hip_status(hipGetLastError(), "paged_append launch");
}

}  // namespace kvssd

using namespace kvssd;

extern "C" __attribute__((visibility("default"))) int kvssd_hip_paged_append(const kvssd_paged_cache* cache,
                                                                             const kvssd_paged_append_args* args,
                                                                             void* stream) {
  if (int rc = check_paged_cache(cache)) return rc;
  if (args == nullptr) return arg_error("arguments are NULL");
  const kvssd_paged_append_args& a = *args;
  if (!paged_dtype(a.dtype)) return arg_error("unsupported dtype");
  if (a.tokens < 0 || a.tokens > (int64_t{1} << 23)) return arg_error("append takes at most 2^23 tokens a call");
  if (!a.offsets && a.tokens != cache->sequences) return arg_error("without offsets there is one token a sequence");
  if (a.offsets && a.lengths_out == cache->lengths)
    return arg_error("lengths_out must not be the cache's lengths where offsets are given");
  if (a.tokens == 0 && !a.lengths_out) return 0;
  if (a.tokens > 0 && (!a.keys.data || !a.values.data)) return arg_error("a required buffer pointer is NULL");
  if (a.keys.heads != cache->kv_heads || a.values.heads != cache->kv_heads)
    return arg_error("keys and values must be [tokens, kv_heads, head_dim]");
  if (a.rotary) {
    if (int rc = check_rotary(a.rotary)) return rc;
    if (a.rotary->head_dim != cache->head_dim) return arg_error("rotary head_dim differs from the cache's");
  }
  if (a.query.data) {
    if (!a.rotary) return arg_error("a query is only taken to be rotated");
    if (!a.query.out) return arg_error("a required buffer pointer is NULL");
    if (a.query.heads <= 0 || a.query.heads > 65536) return arg_error("query takes at most 65536 heads");
  }
  return launch_paged_append(*cache, a, static_cast<hipStream_t>(stream));
}
