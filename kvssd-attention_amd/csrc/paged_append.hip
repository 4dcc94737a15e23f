// New tokens into a paged packed cache: keys rotated, keys and values
// quantised into their sequences' pages, queries rotated, in one launch.
//
// A workgroup takes one token (or up to 8 of a prompt): where the token goes and
// its sines are formed once, then each thread takes words of codes (8 values
// in INT4, 16 in INT2) at one place of every token, so that its addresses are
// formed once; those of a group lie side by side in the wave, and the group's
// maximum is a few lane exchanges (quant_ops.hpp).  A key's word needs
// the other half of its pairs: half layouts load it too (the lines are in the
// cache, their neighbours' threads read them), so that no value passes between
// threads between rotation and coding.
//
// Bound by its instructions on a prompt: 16,381 tokens of 8 kv heads of 128 in
// bfloat16 into INT4 (86 MB in and out, 18 us at a copy's rate) take 31.5 us, of
// which the vector units are busy 26 (a key's word ~200 instructions, 60 of them
// 64-bit; a value's ~100); four tokens a workgroup take 2 us more.  A word loaded ahead of
// the one that is coded changed nothing but the registers (35.3 and 35.9 us).
// 4,097 tokens of 4 kv and 16 query heads of 64 in 32 bits into INT2: 13.9-15.2 us.
// One token of each of 64 sequences: 6.2 us, four dependent reads.
//  The rotated key is rounded to its type
// first: the codes are those of a key rotated by kvssd_hip_rotary and quantised
// by kvssd_hip_quantize, bit for bit.
#include "paged.hpp"
#include "rotary_ops.hpp"

namespace kvssd {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxTurns = 512;
constexpr int kMaxTokens = 8;  // of a workgroup

struct AppendParams {
  kvssd_paged_cache c;
  kvssd_heads keys, values, query;
  const double* frequencies;  // nullptr: no rotation
  double magnitude;
  const int32_t* offsets;
  const int32_t* first_positions;
  const int32_t* parents;
  int32_t* lengths_out;
  RotaryShape shape;  // of the query's items
  int64_t tokens;
  int inverse, per_group, capacity;
  int words, lanes, groups;  // code words of a head's row, words of a group, groups of a row
  int query_heads, lanes_log2;
  uint32_t of_token;  // code words of a token's keys and values
  Divisor of_head;    // of a head
  int width;          // threads side by side on a token's, log2
  int row_bytes, row_scales;
  Divisor of_query, items;    // items of a token's queries, of a head
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

// A word's values: loaded, then rotated if `turns`.  Either half of a pair is own cos -+ other sin, so that a thread
// forms its own half alone, with the sign on the other.
template <typename T, int N, bool VEC>
struct Word {
  T a[N], b[N];  // the values; their partners, in a half layout

  __device__ __forceinline__ void load(const T* x, int d0, const RotaryShape& s, bool turned) {
    if constexpr (VEC) {  // no word mixes low, high and unturned values, and all loads are 16-byte aligned
      load_values(x + d0, a);
      if (turned && d0 < 2 * s.pairs && !s.interleaved) load_values(x + (d0 >= s.pairs ? d0 - s.pairs : d0 + s.pairs), b);
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int d = d0 + i;
        a[i] = b[i] = x[d];
        if (turned && d < 2 * s.pairs) b[i] = x[s.interleaved ? d ^ 1 : (d >= s.pairs ? d - s.pairs : d + s.pairs)];
      }
    }
  }
  static __device__ __forceinline__ float turn(float own, float other, bool high, Turn t) {
    return to_f32(round_to<T>(turn_high(high ? other : -other, own, t)));
  }
  __device__ __forceinline__ void values(int d0, const RotaryShape& s, const Turn* turns, float (&out)[N]) const {
    if (turns == nullptr || (VEC && d0 >= 2 * s.pairs)) {
#pragma unroll
      for (int i = 0; i < N; ++i) out[i] = to_f32(a[i]);
    } else if constexpr (VEC) {
      if (s.interleaved) {
#pragma unroll
        for (int i = 0; i < N; ++i) out[i] = turn(to_f32(a[i]), to_f32(a[i ^ 1]), i % 2, turns[turn_place(d0 / 2 + i / 2)]);
      } else {
        const bool high = d0 >= s.pairs;
        const Turn* t = turns + turn_place(high ? d0 - s.pairs : d0);
#pragma unroll
        for (int i = 0; i < N; ++i) out[i] = turn(to_f32(a[i]), to_f32(b[i]), high, t[turn_place(i)]);  // (d0: a multiple of 8)
      }
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int d = d0 + i;
        const bool high = s.interleaved ? d % 2 : d >= s.pairs;
        const int p = s.interleaved ? d / 2 : (high ? d - s.pairs : d);
        out[i] = d < 2 * s.pairs ? turn(to_f32(a[i]), to_f32(b[i]), high, turns[turn_place(p)]) : to_f32(a[i]);
      }
    }
  }
};

template <typename T, int BITS, bool VEC>
__global__ __launch_bounds__(kThreads, VEC ? 4 : 1) void paged_append_kernel(AppendParams p) {
  constexpr int kVals = 32 / BITS;
  constexpr int kItem = VEC ? 16 / sizeof(T) : 1;
  __shared__ Turn turns[turn_place(kMaxTurns) + kMaxTokens];
  __shared__ int64_t row_s[kMaxTokens];  // row of the pool, -1: dropped
  __shared__ double position_s[kMaxTokens];
  const kvssd_paged_cache& c = p.c;
  const int64_t t0 = static_cast<int64_t>(blockIdx.x) * p.per_group;
  const int n = static_cast<int>(p.tokens - t0 < p.per_group ? p.tokens - t0 : p.per_group);
  // a thread's words lie at one place of every token that it takes
  const uint32_t per_token = p.of_token, coded = per_token / 2;
  const int first = threadIdx.x >> p.width, step = kThreads >> p.width;  // tokens
  // its first item of the queries sets out now, the others one ahead
  const bool in_place = p.query.data == p.query.out;
  const uint32_t queries = static_cast<uint32_t>(n) * p.of_query.d;
  struct Query {
    RotaryItem<T, kItem> v;
    int tok, head, item;
  } next_query;
  auto fetch_query = [&](uint32_t i) {
    next_query.tok = p.of_query.quotient(i);
    const uint32_t rest = i - next_query.tok * p.of_query.d;
    next_query.head = p.items.quotient(rest);
    next_query.item = rest - next_query.head * p.items.d;
    next_query.v.load(p.shape, next_query.item,
                      static_cast<const T*>(p.query.data) + (t0 + next_query.tok) * p.query.token_stride +
                          next_query.head * p.query.head_stride, in_place);
  };
  if (threadIdx.x < queries) fetch_query(threadIdx.x);
  if (static_cast<int>(threadIdx.x) < n) {
    const int64_t t = t0 + threadIdx.x;
    const int b = p.offsets ? sequence_of(p.offsets, c.sequences, t) : static_cast<int>(t);
    int64_t row = -1;
    double position = 0.0;
    if (b >= 0) {
      const int64_t nth = p.offsets ? t - p.offsets[b] : 0;
      const int length = paged_length(c.lengths, b, p.capacity);
      const int64_t slot = length + nth;
      int64_t where = (p.first_positions ? p.first_positions[b] : length) + nth;
      if (p.parents && t >= nth) {  // the depth instead of nth: a read a level, 0.08 us each (a path of 64 5 us)
        const int32_t* parents = p.parents + (t - nth);
        where -= nth;
        for (int up = parent_of(parents, static_cast<int>(nth)); up >= 0; up = parent_of(parents, up)) ++where;
      }
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
  const int token_turns = turn_place(p.shape.pairs) + 1;
  if (p.frequencies) {
    for (int i = threadIdx.x; i < n * p.shape.pairs; i += kThreads)
      turns[i / p.shape.pairs * token_turns + turn_place(i % p.shape.pairs)] =
          make_turn(position_s[i / p.shape.pairs], p.frequencies[i % p.shape.pairs], p.magnitude, p.inverse);
    __syncthreads();
  }
  for (uint32_t r = threadIdx.x & ((1u << p.width) - 1); r < per_token; r += 1u << p.width) {
    const bool is_v = r >= coded, turned = p.frequencies != nullptr && !is_v;
    const uint32_t rest = is_v ? r - coded : r;
    const int head = p.of_head.quotient(rest), word = rest - head * p.of_head.d;
    const int64_t stride = is_v ? p.values.token_stride : p.keys.token_stride;
    const T* x = static_cast<const T*>(is_v ? p.values.data : p.keys.data) + t0 * stride +
                 head * (is_v ? p.values.head_stride : p.keys.head_stride);
    uint8_t* packed = (is_v ? c.packed_v : c.packed_k) + (head * p.words + word) * 4;
    uint16_t* scales = (is_v ? c.scales_v : c.scales_k) + head * p.groups + (word >> p.lanes_log2);
    const bool scaler = (word & (p.lanes - 1)) == 0;
#pragma unroll 1
    for (int tok = first; tok < n; tok += step) {
      const int64_t row = row_s[tok];
      if (row < 0) continue;  // the same for every lane of a group
      Word<T, kVals, VEC> w;
      w.load(x + tok * stride, word * kVals, p.shape, turned);
      float v[kVals];
      w.values(word * kVals, p.shape, turned ? turns + tok * token_turns : nullptr, v);
      float amax = 0.0f;
#pragma unroll
      for (int k = 0; k < kVals; ++k) amax = fmaxf(amax, fabsf(v[k]));
      const float s32 = group_scale<BITS>(lanes_max(amax, p.lanes));
      const uint32_t code = code_word<T, BITS>(v, s32);
      __builtin_memcpy(__builtin_assume_aligned(packed + row * p.row_bytes, 4), &code, 4);
      if (scaler) scales[row * p.row_scales] = __builtin_bit_cast(uint16_t, static_cast<_Float16>(s32));
    }
  }
  for (uint32_t i = threadIdx.x; i < queries; i += kThreads) {
    Query now = next_query;
    if (i + kThreads < queries) fetch_query(i + kThreads);
    now.v.store(p.shape, now.item,
                static_cast<T*>(p.query.out) + (t0 + now.tok) * p.query.out_token_stride +
                    now.head * p.query.out_head_stride,
                turns + now.tok * token_turns, in_place);
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
  const int64_t share = p.tokens / 1024;  // four workgroups a CU
  p.per_group = share < 1 ? 1 : share < per ? static_cast<int>(share) : per;
  p.of_token = 2u * p.c.kv_heads * p.words;
  while ((1u << p.width) < p.of_token && (1 << p.width) < kThreads) ++p.width;
  p.row_bytes = p.c.kv_heads * p.words * 4;
  p.row_scales = p.c.kv_heads * p.groups;
  p.of_head = divisor(p.words);
  p.items = divisor(p.shape.items);
  p.of_query = divisor(int64_t{p.query_heads} * p.shape.items);
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
  p.parents = a.parents;
  p.lengths_out = a.lengths_out;
  p.tokens = a.tokens;
  p.capacity = static_cast<int>(paged_capacity(c));
  p.words = c.head_dim * c.bits / 32;
  p.lanes = c.group_size * c.bits / 32;
  p.groups = c.head_dim / c.group_size;
  while ((1 << p.lanes_log2) < p.lanes) ++p.lanes_log2;
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
