// Rotary positions of queries and keys (rotary_ops.hpp has the arithmetic).
//
// A workgroup takes one token, or a few of a long prompt: its threads form the
// tokens' sines once (LDS), then take items of 2 x 16 bytes -- the two
// partners of 8 (16-bit types) or 4 pairs -- over all heads of both tensors,
// the next on its way while one is turned.
//
// Bound by memory: 8,187 tokens of 40 heads of 128 (168 MB in and out) take
// 28.0 us where they lie in the last-level cache and 35.4 from HBM (4.7 TB/s,
// a large copy's rate); with 32-bit products and sines the same.  4,099 tokens
// of 28 heads of 256, a quarter of them turned (117 MB): 37 us from HBM.  All
// heads' pairs before the values passed through, so that fewer waves form
// products: no faster there, and 38.0 for the first shape.  One token's 64 sequences are
// the launch and three round trips: 5.2 us.
#include "paged.hpp"
#include "rotary_ops.hpp"

namespace kvssd {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxTurns = 512, kMostTokens = 4;  // of a workgroup: 9 KB of LDS

struct RotaryParams {
  const double* frequencies;
  const void* positions;
  double magnitude;
  kvssd_heads t[2];
  RotaryShape shape;
  int64_t tokens;
  int count, inverse, positions_64, per_group;  // tokens of a workgroup
  Divisor items, per_token[2];  // of a head, of a tensor's token
};

template <typename T, int PV>
__global__ __launch_bounds__(kThreads) void rotary_kernel(RotaryParams p) {
  __shared__ Turn turns[turn_place(kMaxTurns) + kMostTokens];
  const int token_turns = turn_place(p.shape.pairs) + 1;
  const int64_t t0 = static_cast<int64_t>(blockIdx.x) * p.per_group;
  const int n = static_cast<int>(p.tokens - t0 < p.per_group ? p.tokens - t0 : p.per_group);
  for (int i = threadIdx.x; i < n * p.shape.pairs; i += kThreads) {
    const int64_t t = t0 + i / p.shape.pairs;
    const double pos = p.positions_64 ? static_cast<double>(static_cast<const int64_t*>(p.positions)[t])
                                      : static_cast<double>(static_cast<const int32_t*>(p.positions)[t]);
    turns[i / p.shape.pairs * token_turns + turn_place(i % p.shape.pairs)] =
        make_turn(pos, p.frequencies[i % p.shape.pairs], p.magnitude, p.inverse);
  }
  __syncthreads();
  for (int k = 0; k < p.count; ++k) {
    const kvssd_heads& h = p.t[k];
    const bool in_place = h.data == h.out;
    const uint32_t count = static_cast<uint32_t>(n) * p.per_token[k].d;
    struct Next {
      RotaryItem<T, PV> v;
      int tok, head, item;
    } next;
    auto fetch = [&](uint32_t i) {
      next.tok = p.per_token[k].quotient(i);
      const uint32_t rest = i - next.tok * p.per_token[k].d;
      next.head = p.items.quotient(rest);
      next.item = rest - next.head * p.items.d;
      next.v.load(p.shape, next.item,
                  static_cast<const T*>(h.data) + (t0 + next.tok) * h.token_stride + next.head * h.head_stride, in_place);
    };
    if (threadIdx.x < count) fetch(threadIdx.x);
    for (uint32_t i = threadIdx.x; i < count; i += kThreads) {
      Next now = next;
      if (i + kThreads < count) fetch(i + kThreads);
      now.v.store(p.shape, now.item,
                  static_cast<T*>(h.out) + (t0 + now.tok) * h.out_token_stride + now.head * h.out_head_stride,
                  turns + now.tok * token_turns, in_place);
    }
  }
}

template <typename T>
void launch_typed(RotaryParams& p, const kvssd_rotary_spec& r, hipStream_t stream) {
  constexpr int kVec = 16 / sizeof(T);
  bool vec = (r.rotary_dim / 2) % kVec == 0 && (r.head_dim - r.rotary_dim) % kVec == 0;
  for (int k = 0; k < p.count; ++k) vec = vec && heads_vector(p.t[k], sizeof(T), true);
  p.shape = rotary_shape(r, vec ? kVec : 1);
  // long prompts: as many tokens as give a thread about four items, whose sines
  // then take few threads' time (8,187 tokens of 320 items: three a workgroup 35.4
  // us, one 40.2; 4,099 of 784: one 37.0, four 40.4); short ones: a workgroup a
  // token, so that more CUs take part
  int64_t all = 0;
  for (int k = 0; k < p.count; ++k) all += static_cast<int64_t>(p.t[k].heads) * p.shape.items;
  int64_t per = p.tokens < 2048 ? 1 : all > 0 ? 4 * kThreads / all : kMostTokens;
  per = per < 1 ? 1 : per > kMostTokens ? kMostTokens : per;
  if (per > kMaxTurns / p.shape.pairs) per = kMaxTurns / p.shape.pairs;  // >= 1: at most 512 pairs
  p.per_group = static_cast<int>(per);
  p.items = divisor(p.shape.items);
  for (int k = 0; k < p.count; ++k) p.per_token[k] = divisor(static_cast<int64_t>(p.t[k].heads) * p.shape.items);
  const dim3 grid(static_cast<unsigned>((p.tokens + per - 1) / per));
  if (vec) hipLaunchKernelGGL((rotary_kernel<T, kVec>), grid, dim3(kThreads), 0, stream, p);
  else hipLaunchKernelGGL((rotary_kernel<T, 1>), grid, dim3(kThreads), 0, stream, p);
}

}  // namespace

int check_rotary(const kvssd_rotary_spec* r) {
  if (r == nullptr || r->frequencies == nullptr) return arg_error("a required buffer pointer is NULL");
  if (r->rotary_dim < 2 || r->rotary_dim % 2 || r->rotary_dim > r->head_dim)
    return arg_error("rotary_dim must be even and between 2 and head_dim");
  if (r->head_dim > 1024) return arg_error("rotary head_dim must be <= 1024");
  return 0;
}

int launch_rotary(const kvssd_rotary_spec& r, const void* positions, int positions_64, int64_t tokens, int dtype,
                  const kvssd_heads* tensors, int count, hipStream_t stream) {
  RotaryParams p{};
  p.frequencies = r.frequencies;
  p.positions = positions;
  p.magnitude = r.magnitude;
  for (int k = 0; k < count; ++k) p.t[k] = tensors[k];
  p.tokens = tokens;
  p.count = count;
  p.inverse = r.inverse;
  p.positions_64 = positions_64;
  switch (dtype) {
    case KVSSD_DTYPE_F16:
      launch_typed<_Float16>(p, r, stream);
      break;
    case KVSSD_DTYPE_BF16:
      launch_typed<uint16_t>(p, r, stream);
      break;
    default:
      launch_typed<float>(p, r, stream);
  }
  return hip_status(hipGetLastError(), "rotary launch");
}

}  // namespace kvssd

using namespace kvssd;

extern "C" __attribute__((visibility("default"))) int kvssd_hip_rotary(const kvssd_rotary_spec* spec,
                                                                       const void* positions, int positions_64,
                                                                       int64_t tokens, int dtype,
                                                                       const kvssd_heads* tensors, int count,
                                                                       void* stream) {
  if (int rc = check_rotary(spec)) return rc;
  if (!paged_dtype(dtype)) return arg_error("unsupported dtype");
  if (count < 1 || count > 2 || tensors == nullptr) return arg_error("rotary takes one or two tensors");
  if (tokens < 0 || tokens > (int64_t{1} << 23)) return arg_error("rotary takes at most 2^23 tokens a call");
  for (int k = 0; k < count; ++k) {
    if (tensors[k].heads < 0 || tensors[k].heads > 65536) return arg_error("rotary takes at most 65536 heads");
    if (tokens > 0 && tensors[k].heads > 0 && (!tensors[k].data || !tensors[k].out))
      return arg_error("a required buffer pointer is NULL");
  }
  if (tokens == 0) return 0;
  if (positions == nullptr) return arg_error("a required buffer pointer is NULL");
  return launch_rotary(*spec, positions, positions_64, tokens, dtype, tensors, count,
                       static_cast<hipStream_t>(stream));
}
