// Attention of many new tokens a sequence over its packed pages, their own
// among them: prompts and chunks of prompts (causal) and trees of drafted tokens,
// with or without a sliding window and sinks.
//
//   s_it = sm_scale q_i.k_t over the slots t that token i sees,
//   out_i = sum_t softmax(s_i)_t v_t,  lse_i = log sum_t e^s_it
//
// with k and v held as INT2/INT4 codes c and group scales, k = (c - mid) sk.
//
// Work split.  The rows of a kv head are its sequence's (token, query head) pairs,
// a token's heads side by side.  A workgroup takes a block of them, 32 a wave, and a
// run of the slots that they see, a stage at a time.  Three forms, after the rows that
// a sequence has on average:
//   8 waves, 256 rows, stages of 16,384 numbers of K and of V (128 slots of heads of
//     128), two of them in LDS: while one is worked on, the next, which each thread
//     loaded a stage earlier (32 dims of a slot), is unpacked into the other;
//   4 waves, 128 rows, stages of half that: two workgroups a CU.  Long heads take no
//     more (registers), 32-bit results neither, with one stage in LDS;
//   4 waves, 32 rows, every wave with a tile of 32 slots of its own (OWN), without a
//     barrier, two workgroups a CU, joined at the end: with few rows a stage that all
//     unpack feeds one or two waves (64 sequences of 8 tokens and 4 heads a kv head
//     89 us; 116 with 64 slots a wave, for which one workgroup has room; 129 with
//     stages that eight waves unpack).
//
// QK (v_mfma_f32_32x32x16_f16): rows = slots, columns = query rows, so that a lane
//   holds 16 scores of one query row and softmax needs no exchange but between the
//   wave's halves.  Codes enter exactly, as (c - mid) / 2^6 (INT4) or / 2^2; the
//   products of 32 dims are taken apart and a group's scale multiplies in 32 bits.
//   The query is scaled by a power of two per row into fp16's range, its largest element to
//   2^10 or more (exact for fp16 and bf16 but for elements below 2^-24 of that one, which
//   are off by 2^-35 of it); a 32-bit one is a sum of two fp16 parts.
// Softmax.  The reference is lazy: it is moved (and sums rescaled) only where a score
//   exceeds the range that fp16 weights have above it.  A weight is one fp16 number (32-bit
//   results: two) whose smallest step is 2^-24, and 2^8 (2^14) or more at the row's maximum: it
//   is off by 2^-11 (2^-22) of itself or by 2^-33 (2^-39) of the row's largest, which is more
//   where it is below 2^-22 (2^-17) of that.
// PV: rows = dims, columns = query rows, K = slots: the scores' lanes are the weights'
//   lanes.  Values are codes times scale, rounded to fp16 once (32-bit results: a sum of two
//   fp16 parts, which holds them exactly), whatever other scales the cache has.  Scales below
//   2^8 are multiplied by 2^7 first: the smallest normal one, 2^-14, times the smallest code
//   (in units of 2^-6 or 2^-2) is then 2^-13, in fp16's normal range, and the last place of
//   any product, 2^-23, is in fp16's.  A run of stages with a larger one is gone through
//   again for those alone, which are multiplied by 2^-1, so that it takes twice as long.
//
// Nearest bound: a SIMD's vector instructions.  Two tiles of 32 slots of heads of 128 take a
//   wave 32 products (1,024 cycles) and, with its part of unpacking, some 410 vector
//   instructions (4 cycles each), of which 128 multiply scales in, 32 are exponentials (of
//   two), 96 scale, sum and bound the scores.  Counted over chunks behind contexts of up to
//   32,768 tokens: products 36 % of the time, other vector instructions 58 %, LDS conflicts
//   5 %.  The two kinds may run side by side, of a SIMD's two waves, so that their sum is no
//   bound: each wave waits 29 % of its time, and the vector instructions alone would take 58 %
//   of it all.  8,187 tokens of 32 heads of 128 with a window of 1,024 take 262 to 282 us,
//   some 475 TFLOP/s (a large fp16 product reaches 1,540 on this card); trees of 64 tokens
//   over 65,536 to 131,072 slots 570 us, some 720 TFLOP/s.  32-bit results, in four waves of
//   512 registers each and one stage in LDS, take 2.3 to 2.7 times as long.  16x16x32 products, which
//   leave registers for more waves, scale twice as many results' lanes: 310 us for the former
//   where these took 292.
//
// A value scale that is not finite is left out of the products, where a masked row's
// weight of 0 times it would be NaN, and makes its group of the rows that see it NaN.
#pragma once

#include "paged_decode.hpp"
#include "rotary_ops.hpp"

namespace kvssd {

// slots of a stage that waves unpack together, a multiple of 64: a thread has a piece of 32 dims of one (of two, of long heads)
constexpr int tokens_stage(int dp, int waves) { return waves * 2048 / dp < 64 ? 64 : waves * 2048 / dp; }

struct PagedTokensParams {
  kvssd_paged_cache c;
  kvssd_heads query;
  void* out;
  float* lse;
  const int32_t* offsets;
  const int32_t* parents;
  float* part_o;   // [item][kv head][row][head_dim]
  float* part_ml;  // [item][kv head][row][2]
  int32_t* starts;  // of many sequences: first items [sequences + 3], first blocks [sequences + 3], the runs' size
  int64_t tokens;
  int capacity, window, sink;
  int query_heads, gq, query_dtype, out_dtype;
  int groups, slices_log2;  // scale groups of a head; 32-dim slices of a group
  Divisor of_page;          // slots of a page
  int row_tiles, parts;     // of a workgroup: waves side by side on rows, on slots
  int block_rows;           // rows of a workgroup, 2^block_log2
  int block_log2;
  int items;                // (row block, run) pairs that the grid and the workspace hold
  int least_stages;         // of a run, unless the lengths call for more
  float scale_log2;
};

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

__device__ __forceinline__ f32x16 mfma32(u32x4 a, u32x4 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(half8_t, a), __builtin_bit_cast(half8_t, b), c, 0, 0, 0);
}

// ds_read_b64_tr_b16: within each group of 16 lanes, lane j receives half j % 4 of lanes j / 4, j / 4 + 4, + 8 and + 12
__device__ __forceinline__ u32x2 lds_read_tr16(const uint8_t* lds) {
  typedef short i16x4 __attribute__((ext_vector_type(4)));
  typedef __attribute__((address_space(3))) i16x4 lds_i16x4;
  return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4*)lds));
}

__device__ __forceinline__ uint32_t low_halves(uint32_t a, uint32_t b) { return __builtin_amdgcn_perm(b, a, 0x05040100u); }
__device__ __forceinline__ uint32_t high_halves(uint32_t a, uint32_t b) { return __builtin_amdgcn_perm(b, a, 0x07060302u); }

// two bf16, rounded to nearest, ties to even
__device__ __forceinline__ uint32_t bf16_pair(float lo, float hi) {
  typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{lo, hi}, bf16x2));
}

// ---------------------------------------------------------------- the work ---

// A sequence's tokens in the call; numbers `sequences` and one on are the tokens before and behind all of them, which
// see nothing.
struct TokenSpan {
  int64_t begin;
  int count;
  int length;  // of the sequence, its new tokens included
};

__device__ __forceinline__ TokenSpan token_span(const PagedTokensParams& p, int s) {
  const int last = p.c.sequences;
  auto place = [&](int i) {
    const int64_t at = p.offsets[i];
    return at < 0 ? 0 : (at > p.tokens ? p.tokens : at);
  };
  if (s > last + 1) return {0, 0, 0};
  const int64_t begin = s <= last ? (s == last ? 0 : place(s)) : place(last);
  const int64_t end = s < last ? place(s + 1) : (s == last ? place(0) : p.tokens);
  return {begin, end > begin ? static_cast<int>(end - begin) : 0, s < last ? paged_length(p.c.lengths, s, p.capacity) : 0};
}

__device__ __forceinline__ int blocks_of(const PagedTokensParams& p, const TokenSpan& s) {
  // (2^24 of them are more than a call takes; so do their sums over a wave stay below 2^31, whatever the offsets)
  const int64_t n = (static_cast<int64_t>(s.count) * p.gq + p.block_rows - 1) >> p.block_log2;
  return static_cast<int>(n < (1 << 24) ? n : 1 << 24);
}

// Stages that a block's tokens see something of: those of the sinks, then from `second` to `end`.
struct StageList {
  int sinks, second, end;
  __device__ __forceinline__ int count() const { return sinks + end - second; }
  __device__ __forceinline__ int stage(int n) const { return n < sinks ? n : n - sinks + second; }
};

__device__ __forceinline__ StageList stages_of(const PagedTokensParams& p, const TokenSpan& s, int block, int stage_slots) {
  const int base = s.length - s.count;
  const int first = block * p.block_rows / p.gq;  // (fewer than 2^30 rows)
  const int last = min((block * p.block_rows + p.block_rows - 1) / p.gq, s.count - 1);
  const int hi = max(min(base + last + 1, s.length), 0);  // the first slot that none sees
  StageList list{0, 0, (hi + stage_slots - 1) / stage_slots};
  if (p.window > 0) {
    const int at = (p.parents ? base : base + first) - p.window + 1;  // the first that one sees, but for sinks
    list.second = min(max(at, 0) / stage_slots, list.end);
    list.sinks = min((min(p.sink, hi) + stage_slots - 1) / stage_slots, list.second);
  }
  return list;
}

// Which work a workgroup does: its item, of the batch's, is run `run` of `runs` of a block of rows.
struct TokenItem {
  int seq, block, run, runs;
  TokenSpan span;
};

// Every sequence's blocks are cut into the same number of runs, after the stages of its last one (which sees most, but
// for borders).  p.least_stages comes from the caller's hints, and grows here where the lengths would need more items
// than there are: sum of blocks * runs <= sum of blocks * stages / size + sum of blocks.
template <int STAGE>
__device__ __forceinline__ int runs_of_sequence(const PagedTokensParams& p, const TokenSpan& s, int blocks, int size) {
  if (blocks == 0) return 0;
  const int stages = stages_of(p, s, blocks - 1, STAGE).count();
  return stages <= size ? 1 : (stages + size - 1) / size;
}

__device__ __forceinline__ int size_of_runs(const PagedTokensParams& p, float work, float blocks) {
  const float room = static_cast<float>(p.items) - blocks;
  if (room < 1.0f) return 1 << 30;
  const float least = work / room * 1.0001f + 1.0f;  // (sums of 24 bits)
  return max(p.least_stages, least < 1e9f ? static_cast<int>(least) : 1 << 30);
}

template <int STAGE>
__device__ __forceinline__ int run_size(const PagedTokensParams& p) {
  const int lane = threadIdx.x % kWave;
  float work = 0.0f, blocks = 0.0f;
  for (int s0 = 0; s0 < p.c.sequences + 2; s0 += kWave) {
    const TokenSpan s = token_span(p, s0 + lane);
    const int n = blocks_of(p, s);
    if (n > 0) {
      blocks += static_cast<float>(n);
      work += static_cast<float>(n) * static_cast<float>(stages_of(p, s, n - 1, STAGE).count());
    }
  }
  work = wave_sum(work);
  blocks = wave_sum(blocks);
  return size_of_runs(p, work, blocks);
}

// What item `own` of a sequence is; `blocks_alone`: items are blocks.
__device__ __forceinline__ TokenItem item_of(int seq, const TokenSpan& span, int blocks, int runs, int own, bool blocks_alone) {
  const int place = blocks_alone || runs <= 1 ? own : own / runs;
  return {seq, blocks - 1 - place, blocks_alone ? 0 : own - place * runs, runs, span};  // the longest first
}

// Item `item`; seq -1 where there are fewer.  first: of the item's first run.
template <int STAGE>
__device__ __forceinline__ TokenItem find_item(const PagedTokensParams& p, int item, bool blocks_alone, int* first) {
  const int lane = threadIdx.x % kWave;
  const int sequences = p.c.sequences + 2;  // with the two of no sequence
  if (p.starts) {
    // the last one that starts at or before the item: 64 of them compared at a time
    const int32_t* starts = p.starts + (blocks_alone ? sequences + 1 : 0);
    if (item >= starts[sequences]) return TokenItem{-1, 0, 0, 1, {0, 0, 0}};
    int at = 0;
    for (int n = sequences; n > 1;) {
      const int step = (n + kWave - 1) / kWave;
      const bool upto = lane * step < n && starts[at + lane * step] <= item;
      const int last = 63 - __builtin_clzll(__ballot(upto));  // (the first one does)
      at += last * step;
      n = min(step, n - last * step);
    }
    const TokenSpan span = token_span(p, at);
    const int blocks = blocks_of(p, span), runs = runs_of_sequence<STAGE>(p, span, blocks, p.starts[2 * sequences + 2]);
    const TokenItem t = item_of(at, span, blocks, runs, item - starts[at], blocks_alone);
    if (first != nullptr) *first = p.starts[at] + (blocks - 1 - t.block) * runs;
    return t;
  }
  const int size = run_size<STAGE>(p);
  int before = 0;  // items of the sequences before
  for (int s0 = 0; s0 < sequences; s0 += kWave) {
    const TokenSpan s = token_span(p, s0 + lane);
    const int blocks = blocks_of(p, s);
    const int runs = runs_of_sequence<STAGE>(p, s, blocks, size);
    const int n = blocks_alone ? blocks : blocks * runs;
    const int upto = wave_prefix(n);
    const uint64_t past = __ballot(item < upto);
    if (past) {
      const int at = __builtin_ctzll(past);
      const int own = item - (__builtin_amdgcn_readlane(upto, at) - __builtin_amdgcn_readlane(n, at));
      const TokenSpan span = {static_cast<int64_t>(__builtin_amdgcn_readlane(static_cast<int>(s.begin), at)),  // (below 2^30)
                              __builtin_amdgcn_readlane(s.count, at), __builtin_amdgcn_readlane(s.length, at)};
      const int count = __builtin_amdgcn_readlane(blocks, at);
      const TokenItem t = item_of(s0 + at, span, count, __builtin_amdgcn_readlane(runs, at), own, blocks_alone);
      if (first != nullptr) {
        const int all = wave_prefix(blocks * runs);
        *first = before + __builtin_amdgcn_readlane(all, at) - (t.block + 1) * t.runs;
      }
      return t;
    }
    item -= __builtin_amdgcn_readlane(upto, kWave - 1);
    before += __builtin_amdgcn_readlane(wave_prefix(blocks * runs), kWave - 1);
  }
  return TokenItem{-1, 0, 0, 1, {0, 0, 0}};
}

// Workgroup -> (item, kv head).  Workgroups go to the eight dies in turn, each with an L2 of its own; a line of codes
// holds two neighbouring heads' rows (of 64 bytes), whose workgroups should so be of one die and near in time.
__device__ __forceinline__ void place_of(const PagedTokensParams& p, int id, int* item, int* head) {
  const int heads = p.c.kv_heads;
  if (heads % 2) {
    *item = id / heads;
    *head = id - *item * heads;
    return;
  }
  const int pair = id / 16 * 8 + id % 8;
  *item = pair / (heads / 2);
  *head = (pair - *item * (heads / 2)) * 2 + id / 8 % 2;
}

template <int DP>
int launch_paged_tokens_dims(const PagedTokensParams& p, int waves, bool precise, bool own, unsigned groups, hipStream_t stream);
template <>
int launch_paged_tokens_dims<64>(const PagedTokensParams& p, int waves, bool precise, bool own, unsigned groups, hipStream_t stream);
template <>
int launch_paged_tokens_dims<128>(const PagedTokensParams& p, int waves, bool precise, bool own, unsigned groups, hipStream_t stream);
template <>
int launch_paged_tokens_dims<256>(const PagedTokensParams& p, int waves, bool precise, bool own, unsigned groups, hipStream_t stream);

// ------------------------------------------------------------------ kernel ---

// 32 INT2 codes as fp16 pairs (c - 2) / 4 in the dims' order
__device__ __forceinline__ void unpack_int2(const uint32_t* x, const Masks& k, uint32_t m01, uint32_t m23, u32x4 (&out)[4]) {
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    const u32x4 a = code_operand<2>(x[w], 0, k, m01, m23), b = code_operand<2>(x[w], 1, k, m01, m23);
#pragma unroll
    for (int i = 0; i < 4; ++i) {  // dims (2 i, 2 i + 8) and (2 i + 1, 2 i + 9)
      out[2 * w][i] = low_halves(a[i], b[i]);
      out[2 * w + 1][i] = high_halves(a[i], b[i]);
    }
  }
}

// s[r] = dot[r] * (scale of lane r of the lane's row of 16), r from R to END - 1
template <int R, int END>
__device__ __forceinline__ void scale_rows(float (&s)[16], const f32x16& dot, float scale) {
  const float by = __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, scale), 0x150 + R, 0xF, 0xF, true));
  s[R] = by * dot[R];
  if constexpr (R + 1 < END) scale_rows<R + 1, END>(s, dot, scale);
}
// The same added to what s holds, in rows 0 to 7 or 8 to 15.  The compiler makes two instructions of each (a broadcast, a
// multiply-add); here the broadcast is the multiply-add's operand.  What such assembly needs of its surroundings: the
// results of a matrix instruction may be read some time after it only, which the compiler sees to at the half's first
// product, that it forms itself and that the others take as an operand, so that they follow it; and a broadcast register
// must not have been written just before, hence the s_nop.
template <int HALF>
__device__ __forceinline__ void add_scaled_rows(float (&s)[16], const f32x16& dot, float scale) {
  const float by =
      __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, scale), 0x150 + 8 * HALF, 0xF, 0xF, true));
  float* v = s + 8 * HALF;
  constexpr int o = 8 * HALF;
  v[0] = __builtin_fmaf(by, dot[o], v[0]);
#define KVSSD_ROW(n, lo, hi) "v_fmac_f32_dpp %[s" #n "], %[scale], %[d" #n "] row_newbcast:%c[r" #n "] row_mask:0xf bank_mask:0xf bound_ctrl:1\n\t"
  asm volatile("s_nop 1\n\t" KVSSD_ROW(1, 1, 9) KVSSD_ROW(2, 2, 10) KVSSD_ROW(3, 3, 11) KVSSD_ROW(4, 4, 12) KVSSD_ROW(5, 5, 13)
                   KVSSD_ROW(6, 6, 14) KVSSD_ROW(7, 7, 15)
               : [s1] "+v"(v[1]), [s2] "+v"(v[2]), [s3] "+v"(v[3]), [s4] "+v"(v[4]), [s5] "+v"(v[5]), [s6] "+v"(v[6]), [s7] "+v"(v[7])
               : [scale] "v"(scale), [after] "v"(v[0]), [d1] "v"(dot[o + 1]), [d2] "v"(dot[o + 2]), [d3] "v"(dot[o + 3]),
                 [d4] "v"(dot[o + 4]), [d5] "v"(dot[o + 5]), [d6] "v"(dot[o + 6]), [d7] "v"(dot[o + 7]), [r1] "n"(o + 1),
                 [r2] "n"(o + 2), [r3] "n"(o + 3), [r4] "n"(o + 4), [r5] "n"(o + 5), [r6] "n"(o + 6), [r7] "n"(o + 7));
#undef KVSSD_ROW
}

// W: waves; PREC: 32-bit queries or results; OWN: waves with slots of their own.
template <int DP, int W, bool PREC, bool OWN>
__global__ __launch_bounds__(W * kWave, DP < 256 && !(PREC && DP > 64) ? 2 : 1) void paged_tokens_kernel(PagedTokensParams p) {
  constexpr int kPair = OWN ? 1 : 2;              // tiles of 32 slots that a wave works on at a time
  constexpr int kStage = OWN ? 32 * W : tokens_stage(DP, W);
  constexpr int kSlots = OWN ? 32 : kStage;       // of a buffer in LDS
  constexpr int kSlices = DP / 32;
  constexpr int kParts = PREC ? 2 : 1;
  // in LDS: stages, one of which is unpacked while another is worked on, or the waves' parts of one
  constexpr int kBuffers = OWN ? W : PREC ? 1 : 2;
  constexpr int kTiles = kSlots / 32;             // of a buffer
  constexpr int kOwn = kWave / kSlices;           // slots of a wave's pieces at a time
  constexpr int kGroups = kSlots / kOwn;          // of so many slots
  constexpr int kPieces = OWN ? kGroups : kGroups / W;  // of a thread
  constexpr int kValueRow = DP * 2 + (DP == 64 ? 32 : 64);  // bytes; so (but for short heads) do transposed reads meet in no bank
  constexpr int kKeyBytes = DP * kSlots * 2, kValueBytes = kValueRow * kSlots;
  constexpr int kBytes = kKeyBytes + kParts * kValueBytes;
  // log2 of a weight at the reference's maximum, and at most.  (The smallest step is 2^-24: with 32-bit results 2^-38 of
  // the former, at the price of references that move more often.)
  constexpr float kBias = PREC ? 14.0f : 8.0f, kRoom = PREC ? 15.9f : 14.0f;
  // value scales below kLarge, 2^8, times 2^7 and those from there on times 2^-1 have all their bits in fp16, times codes too
  constexpr uint32_t kLarge = 23 << 10, kInfinite = 31 << 10;
  // keys: [chunk of 8 dims][slot] 16 bytes each, slots turned by their slice; values: [part][slot][dim], the chunks of
  // 8 dims of a slice turned by their slot's number: so do writes of 16 lanes meet in no bank either
  constexpr int kTurn = 16 / kSlices;
  auto value_turn = [](int slot, int slice) {
    return DP == 128 ? slot & 3 : DP == 64 ? (slot & 1) + 2 * (slot >> 2 & 1) : (slot & 1) + 2 * (slice >> 2 & 1);
  };
  __shared__ __attribute__((aligned(1024))) uint8_t lds[kBuffers][kBytes];
  __shared__ float scale_lds[kBuffers][kSlices][kTiles][2][16];  // keys': of slots 8 (i / 4) + 4 half + i % 4 of a tile
  __shared__ uint64_t live_lds[kBuffers][kGroups], bad_lds[kBuffers][kGroups];  // a bit a lane of a group's pieces
  // of a group: whether slots take no part, or value scales are not finite, or kLarge or more
  constexpr uint32_t kGaps = 1, kBad = 2, kOver = 4;
  __shared__ __attribute__((aligned(16))) uint32_t flags_lds[kBuffers][(kGroups + 3) / 4 * 4];

  constexpr int kTree = 1024;  // tokens of a tree whose parents are kept in LDS
  __shared__ int16_t parent_lds[kTree];

  const kvssd_paged_cache& c = p.c;
  const int tid = threadIdx.x, lane = tid % kWave, wave = scalar(tid / kWave);
  const int col = lane & 31, half = lane >> 5;
  int item, kvh;
  place_of(p, blockIdx.x, &item, &kvh);
  item = scalar(item);
  kvh = scalar(kvh);
  if (item >= p.items) return;
  const TokenItem work = find_item<kStage>(p, item, false, nullptr);
  if (work.seq < 0) return;
  const int seq = scalar(work.seq), block = scalar(work.block), runs = scalar(work.runs);
  const int count = scalar(work.span.count), length = scalar(work.span.length);
  const int64_t token0 = scalar(static_cast<int>(work.span.begin));
  const int base = length - count;
  const int rows = count * p.gq;
  StageList list{0, 0, 0};
  int n_begin = 0, n_end = 0;
  if (seq < c.sequences) {
    list = stages_of(p, {token0, count, length}, block, kStage);
    const int n = list.count();
    const int run = scalar(work.run);
    n_begin = static_cast<int>(static_cast<int64_t>(n) * run / runs);
    n_end = static_cast<int>(static_cast<int64_t>(n) * (run + 1) / runs);
  }

  // a tree's token above `i`, -1 if none
  const bool tree = p.parents != nullptr && seq < c.sequences;
  auto above = [&](int i) -> int { return i < kTree ? parent_lds[i] : parent_of(p.parents + token0, i); };
  if (tree) {
    for (int i = tid; i < min(count, kTree); i += W * kWave) parent_lds[i] = static_cast<int16_t>(parent_of(p.parents + token0, i));
  }

  // ---- a thread's pieces: 32 dims of a slot
  const int slice = tid % kSlices;
  int first_slot = (OWN ? lane : tid) / kSlices;  // in a buffer
  constexpr int kNext = OWN ? kOwn : W * kOwn;  // slots to the thread's next piece
  const int d = c.head_dim, row_bytes = d * c.bits / 8;
  const bool has_dims = slice * 32 < d;
  const int piece_bytes = 4 * c.bits;
  const int32_t* pages = c.page_table + static_cast<int64_t>(seq < c.sequences ? seq : 0) * c.max_pages;
  // of the pool's row 0
  const uint32_t slot_bytes = c.kv_heads * row_bytes, slot_scales = c.kv_heads * p.groups;
  const uint32_t piece_at = kvh * row_bytes + slice * piece_bytes, scale_at = kvh * p.groups + (slice >> p.slices_log2);
  struct Piece {
    uint32_t k[4], v[4];
    uint16_t sk, sv;
    bool live;
  } next[kPieces];
  int page_next[kPieces], row_next[kPieces];  // of the stage after it: the page, and the row in it
#pragma unroll
  for (int i = 0; i < kPieces; ++i) next[i] = Piece{};
  auto find = [&](int n, int piece) {  // of the piece's slot in the list's stage n; page -1: none
    const int slot = list.stage(n) * kStage + (OWN ? wave * kSlots : 0) + first_slot + piece * kNext;
    page_next[piece] = -1;
    if (n < n_end && slot < length) {
      const int nth = p.of_page.quotient(slot);
      row_next[piece] = slot - nth * c.page_tokens;
      page_next[piece] = pages[nth];
    }
  };
  auto load = [&](int piece) {
    Piece& x = next[piece];
    const int page = page_next[piece];
    x.live = page >= 0 && page < c.num_pages;
    x.sk = x.sv = 0;
    if (x.live && has_dims) {  // (other codes stay: any are finite, and their scales are 0)
      const uint32_t row = page * c.page_tokens + row_next[piece];
      const uint64_t byte = static_cast<uint64_t>(row) * slot_bytes + piece_at;
      const uint64_t scale = static_cast<uint64_t>(row) * slot_scales + scale_at;
      if (c.bits == 4) {
        __builtin_memcpy(x.k, __builtin_assume_aligned(c.packed_k + byte, 16), 16);
        __builtin_memcpy(x.v, __builtin_assume_aligned(c.packed_v + byte, 16), 16);
      } else {
        __builtin_memcpy(x.k, __builtin_assume_aligned(c.packed_k + byte, 8), 8);
        __builtin_memcpy(x.v, __builtin_assume_aligned(c.packed_v + byte, 8), 8);
      }
      x.sk = c.scales_k[scale];
      x.sv = c.scales_v[scale];
    }
  };
  auto begin = [&] {
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      row_next[i] = 0;
      find(n_begin, i);
    }
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      load(i);
      find(n_begin + 1, i);
    }
  };
  begin();

  // ---- the wave's rows
  const int part = wave / p.row_tiles;
  const int wave_row0 = block * p.block_rows + (wave % p.row_tiles) * 32;
  const bool active = part < p.parts && wave_row0 < rows;  // (the others unpack alone)
  const int row = min(wave_row0 + col, rows - 1);
  const int own = row / p.gq;  // the lane's token among the sequence's, and its position
  int place = base + own;
  if (tree) {
    __syncthreads();
    place = base;
    for (int up = above(own); up >= 0; up = above(up)) ++place;
  }
  const int head = kvh * p.gq + row - own * p.gq;
  u32x4 q[kParts][DP / 16];
  float factor;
  const bool wide = PREC && p.query_dtype == KVSSD_DTYPE_F32;
  {
    const int64_t from = (token0 + own) * p.query.token_stride + head * p.query.head_stride;
    const bool bf16 = p.query_dtype == KVSSD_DTYPE_BF16;
    u32x4 raw[DP / 16][kParts];  // dims 16 j + 8 half ..
    float big = 0.0f;
    auto value = [&](int j, int i) {
      const uint32_t word = raw[j][0][i / 2];
      if constexpr (PREC) {
        if (wide) {
          const uint32_t whole = raw[j][i / 4][i % 4];
          return __builtin_bit_cast(float, whole);
        }
      }
      const float as_half = i % 2 ? half_hi(word) : half_lo(word);
      return bf16 ? __builtin_bit_cast(float, i % 2 ? word & 0xFFFF0000u : word << 16) : as_half;
    };
#pragma unroll
    for (int j = 0; j < DP / 16; ++j) {
      const int dim = 16 * j + 8 * half;
      raw[j][0] = raw[j][kParts - 1] = u32x4{0, 0, 0, 0};
      if (active && dim < d) {
        const uint8_t* src = static_cast<const uint8_t*>(p.query.data) + (from + dim) * (wide ? 4 : 2);
        raw[j][0] = *reinterpret_cast<const u32x4*>(src);
        if (wide) raw[j][kParts - 1] = *reinterpret_cast<const u32x4*>(src + 16);
      }
    }
#pragma unroll
    for (int j = 0; j < DP / 16; ++j)
#pragma unroll
      for (int i = 0; i < 8; ++i) big = fmaxf(big, fabsf(value(j, i)));
    big = fmaxf(big, __shfl_xor(big, 32, kWave));
    int ex = static_cast<int>((__builtin_bit_cast(uint32_t, big) >> 23) & 255u);
    ex = ex < 12 ? 12 : (ex > 253 ? 253 : ex);
    const int up = 10 + 127 - ex;  // 2^up big in [2^10, 2^11)
    const float scale_up = __builtin_bit_cast(float, static_cast<uint32_t>(127 + up) << 23);
    const float scale_down = __builtin_bit_cast(float, static_cast<uint32_t>(127 - up) << 23);
    factor = scale_down * ((c.bits == 4 ? kUnpackScale<4> : kUnpackScale<2>) * p.scale_log2);
    // the keys' order of a chunk's dims: INT4 (0, 4) (1, 5) (2, 6) (3, 7), INT2 as they are
    auto ordered = [&](u32x4 x) {
      const u32x4 y = {low_halves(x[0], x[2]), high_halves(x[0], x[2]), low_halves(x[1], x[3]), high_halves(x[1], x[3])};
      return c.bits == 4 ? y : x;
    };
#pragma unroll
    for (int j = 0; j < DP / 16; ++j) {
      u32x4 hi, lo = {};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float a = value(j, 2 * i) * scale_up, b = value(j, 2 * i + 1) * scale_up;
        const _Float16 ah = static_cast<_Float16>(a), bh = static_cast<_Float16>(b);
        hi[i] = pack_half2(ah, bh);
        if constexpr (PREC)
          lo[i] = pack_half2(static_cast<_Float16>(a - static_cast<float>(ah)), static_cast<_Float16>(b - static_cast<float>(bh)));
      }
      q[0][j] = ordered(hi);
      if constexpr (PREC) q[kParts - 1][j] = ordered(lo);
    }
  }
  // of the wave's rows: first and last token, as slots
  const int own_lo = base + scalar(min(wave_row0, rows - 1) / p.gq);
  const int own_hi = base + scalar((min(wave_row0 + 32, rows) - 1) / p.gq);

  bool again = false;  // whether large value scales alone enter

  auto unpack_piece_into = [&](const Piece& x, int buf, int piece) {
    const int piece_slot = first_slot + piece * kNext;
    uint32_t zero = 0;
    asm volatile("" : "+v"(zero));  // (masks live here only)
    const Masks masks = make_masks(zero);
    const uint32_t m01 = 0x00030003u | zero, m23 = 0x000C000Cu | zero;
    u32x4 codes[4];
    // dims of a chunk: INT4 (0, 4) (1, 5) (2, 6) (3, 7), INT2 in their order
    auto unpack = [&](const uint32_t* from, u32x4 (&to)[4]) {
      if (c.bits == 4) {
#pragma unroll
        for (int w = 0; w < 4; ++w) to[w] = code_operand<4>(from[w], 0, masks, m01, m23);
      } else {
        unpack_int2(from, masks, m01, m23, to);
      }
    };
    unpack(x.k, codes);
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const int chunk = 4 * slice + w;
      *reinterpret_cast<u32x4*>(&lds[buf][(chunk * kSlots + (piece_slot ^ slice * kTurn)) * 16]) = codes[w];
    }
    const int in_tile = piece_slot % 32;
    scale_lds[buf][slice][piece_slot / 32][in_tile >> 2 & 1][(in_tile >> 3) * 4 + in_tile % 4] = half_bits_to_float(x.sk);
    const uint32_t size = x.sv & 0x7FFFu;
    const uint64_t live = __ballot(x.live), bads = __ballot(size >= kInfinite), overs = __ballot(size >= kLarge);
    if (lane == 0) {
      const int group = OWN ? piece : piece * W + wave;
      live_lds[buf][group] = live;
      bad_lds[buf][group] = bads;
      flags_lds[buf][group] = (live == ~0ull ? 0u : kGaps) | (bads != 0 ? kBad : 0u) | (overs != bads ? kOver : 0u);
    }
    unpack(x.v, codes);
    const bool enters = again ? size - kLarge < kInfinite - kLarge : size < kLarge;
    const _Float16 up = again ? static_cast<_Float16>(0.5f) : static_cast<_Float16>(128.0f);
    const _Float16 s = __builtin_bit_cast(_Float16, static_cast<uint16_t>(enters ? x.sv : 0)) * up;
    const half2v ss = {s, s};
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      u32x4 hi, lo;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t pair = codes[w][i];  // (a bit cast of a vector's element takes the first one)
        const half2v n = __builtin_bit_cast(half2v, pair);
        const half2v v = n * ss;
        hi[i] = __builtin_bit_cast(uint32_t, v);
        if constexpr (PREC) lo[i] = __builtin_bit_cast(uint32_t, __builtin_elementwise_fma(n, ss, -v));
      }
      uint8_t* dst = &lds[buf][kKeyBytes + piece_slot * kValueRow + slice * 64 + (w ^ value_turn(piece_slot, slice)) * 16];
      *reinterpret_cast<u32x4*>(dst) = hi;
      if constexpr (PREC) *reinterpret_cast<u32x4*>(dst + kValueBytes) = lo;
    }
  };

  f32x16 acc[kSlices];
#pragma unroll
  for (int i = 0; i < kSlices; ++i) acc[i] = f32x16{};
  float m = 0.0f, l = 0.0f;  // the reference, and the sum of the half's weights
  uint32_t poison = 0;  // slices of a row that see a value scale that is not finite

  // where the lane reads values: slots 16 step + 4 half + (lane / 4) % 4 (and 8 on), dims 16 (lane / 16 % 2) + 4 (lane % 4)
  const int value_slot = 4 * half + (lane >> 2 & 3), value_chunk = (lane >> 4 & 1) * 2 + (lane >> 1 & 1);
  const int value_at = kKeyBytes + value_slot * kValueRow + (value_chunk ^ value_turn(value_slot, 0)) * 16 + (lane & 1) * 8;

  // A wave that forms products goes first, scores before values: so do the two waves of a SIMD come to different parts of
  // a pair, and one's products are formed beside the other's exponentials (chunks behind long contexts 1,585 -> 1,481 us,
  // about half of it where all of a pair goes first).
  // A pair of tiles of 32 slots (or one).  `plain`: every row sees all of them, and their values' scales are finite.
  auto work_pair = [&](int buf, int tile, int t0, bool plain, bool all_live, bool any_bad) {
    const uint8_t* const stage = lds[buf];
    // ---- scores.  Steps: (slice, tile), the tiles in turn, so that a step's products are formed while those of the one
    // before, of the other tile, are scaled
    constexpr int kSteps = kPair * kSlices, kRing = 3;
    float s[kPair][16], sk[kRing];
    u32x4 key[kRing][2];
    int at_col = 32 * tile + col;
    asm volatile("" : "+v"(at_col));  // (a register for every turn of it would be kept otherwise)
    auto read_keys = [&](int n) {
      sk[n % kRing] = scale_lds[buf][n / kPair][tile + n % kPair][half][lane & 15];  // a slot's a lane, alike in the half's two rows
      const uint8_t* at = stage + ((4 * (n / kPair) + half) * kSlots + (at_col ^ n / kPair * kTurn) + 32 * (n % kPair)) * 16;
#pragma unroll
      for (int j = 0; j < 2; ++j) __builtin_memcpy(&key[n % kRing][j], __builtin_assume_aligned(at + 2 * j * kSlots * 16, 16), 16);
    };
    auto product = [&](int n, int j, f32x16 to) {
      to = mfma32(key[n % kRing][j], q[0][n / kPair * 2 + j], to);
      if constexpr (PREC) {
        if (wide) to = mfma32(key[n % kRing][j], q[kParts - 1][n / kPair * 2 + j], to);
      }
      return to;
    };
#pragma unroll
    for (int n = 0; n < kRing && n < kSteps; ++n) read_keys(n);
    f32x16 dot[2];
    dot[0] = product(0, 0, f32x16{});
    dot[0] = product(0, 1, dot[0]);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int n = 0; n < kSteps; ++n) {
      const bool more = n + 1 < kSteps;
      const float by = sk[n % kRing];
      if (n > 0 && n + kRing - 1 < kSteps) read_keys(n + kRing - 1);
      if (more) dot[(n + 1) % 2] = product(n + 1, 0, f32x16{});
      __builtin_amdgcn_sched_barrier(0);
      if (n < kPair) scale_rows<0, 8>(s[n % kPair], dot[n % 2], by);
      else add_scaled_rows<0>(s[n % kPair], dot[n % 2], by);
      __builtin_amdgcn_sched_barrier(0);
      if (more) dot[(n + 1) % 2] = product(n + 1, 1, dot[(n + 1) % 2]);
      __builtin_amdgcn_sched_barrier(0);
      if (n < kPair) scale_rows<8, 16>(s[n % kPair], dot[n % 2], by);
      else add_scaled_rows<1>(s[n % kPair], dot[n % 2], by);
      __builtin_amdgcn_sched_barrier(0);
    }
    __builtin_amdgcn_s_setprio(0);
    // ---- the first tile's values set out
    constexpr int kValues = 2 * kSlices;  // steps of a tile
    constexpr int kAhead = PREC ? 2 : kValues;
    u32x4 value[kAhead];
    auto fetch = [&](int of, int n, int from) {  // of a tile, step n % 2 of slice n / 2
      const int start = value_turn(0, n / 2) ? value_at ^ value_turn(0, n / 2) * 16 : value_at;
      const uint8_t* at = stage + start + (32 * (tile + of) + 16 * (n % 2)) * kValueRow + 64 * (n / 2) + from;
      const u32x2 lo = lds_read_tr16(at), hi = lds_read_tr16(at + 8 * kValueRow);
      return u32x4{lo[0], lo[1], hi[0], hi[1]};
    };
#pragma unroll
    for (int i = 0; i < kAhead; ++i) value[i] = fetch(0, i, 0);
    __builtin_amdgcn_sched_barrier(0);
    // ---- weights: s is turned into log2 units above the reference, then into its powers
#pragma unroll
    for (int x = 0; x < kPair; ++x)
#pragma unroll
      for (int r = 0; r < 16; ++r) s[x][r] = __builtin_fmaf(s[x][r], factor, -m);
    uint32_t seen[kPair];  // of the lane's slots: bit r, slot 8 (r / 4) + 4 half + r % 4
    if (!plain) {
#pragma unroll
      for (int x = 0; x < kPair; ++x) {
        const int s0 = t0 + 32 * x;
        uint32_t bits = 0xFFFFFFFFu;  // of the tile's slots
        const int before = tree ? base : base + own + 1;  // slots below it are seen, but for the window
        bits = before >= s0 + 32 ? bits : before <= s0 ? 0u : (1u << (before - s0)) - 1;
        if (p.window > 0) {
          const int low = place - p.window + 1;  // slots from here on, or below the sinks' end
          const uint32_t from = low <= s0 ? ~0u : low >= s0 + 32 ? 0u : ~0u << (low - s0);
          const uint32_t sinks = p.sink >= s0 + 32 ? ~0u : p.sink <= s0 ? 0u : (1u << (p.sink - s0)) - 1;
          bits &= from | sinks;
        }
        if (tree && s0 + 31 >= base) {
          int at = place;
          for (int up = own; up >= 0 && base + up >= s0; up = above(up), --at)
            if (base + up < s0 + 32 && (p.window == 0 || at > place - p.window || at < p.sink)) bits |= 1u << (base + up - s0);
        }
        const int in_buffer = 32 * (tile + x) + col, group = in_buffer / kOwn, piece_lane = in_buffer % kOwn * kSlices;  // col's slot
        if (!all_live) bits &= static_cast<uint32_t>(__ballot(live_lds[buf][group] >> piece_lane & 1));
        bits >>= 4 * half;
        seen[x] = (bits & 0xFu) | (bits >> 4 & 0xF0u) | (bits >> 8 & 0xF00u) | (bits >> 12 & 0xF000u);
#pragma unroll
        for (int r = 0; r < 16; ++r) s[x][r] = seen[x] >> r & 1u ? s[x][r] : -INFINITY;
        if (any_bad) {
          const uint32_t bad_slices = static_cast<uint32_t>(bad_lds[buf][group] >> piece_lane) & ((1u << kSlices) - 1);
#pragma unroll 1
          for (uint32_t slots = static_cast<uint32_t>(__ballot(bad_slices != 0)); slots != 0; slots &= slots - 1) {
            const int y = __builtin_ctz(slots);  // a slot of the tile with a value scale that is not finite
            const int r = (y >> 3) * 4 + y % 4;
            const int here = half == (y >> 2 & 1) && (seen[x] >> r & 1u);
            if (here | __shfl_xor(here, 32, kWave)) poison |= __builtin_amdgcn_readlane(bad_slices, y);
          }
        }
      }
    }
    float of[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
    for (int r = 0; r < 16 * kPair; ++r) of[r % 4] = fmaxf(of[r % 4], s[r / 16][r % 16]);
    float most = fmaxf(fmaxf(of[0], of[1]), fmaxf(of[2], of[3]));
    // a new reference where a weight would be too large, or where these are the first that the row sees
    if (__any(most > kRoom || (l == 0.0f && most > -INFINITY))) {
      most = fmaxf(most, __shfl_xor(most, 32, kWave));
      const bool none = l + __shfl_xor(l, 32, kWave) == 0.0f;
      const bool moves = most > kRoom || (none && most > -INFINITY);
      const float up = moves ? most - kBias : 0.0f;
      const float alpha = none ? 0.0f : exp2f(-up);
      m += up;
      l *= alpha;
#pragma unroll
      for (int i = 0; i < kSlices; ++i) acc[i] *= alpha;
#pragma unroll
      for (int x = 0; x < kPair; ++x)
#pragma unroll
        for (int r = 0; r < 16; ++r) s[x][r] -= up;
    }
    u32x4 w[kParts][2];
    auto power = [&](int x, int r) {
      s[x][r] = __builtin_amdgcn_exp2f(s[x][r]);
      l += s[x][r];
    };
    auto operands = [&](int x) {
      float (&t)[16] = s[x];
#pragma unroll
      for (int step = 0; step < 2; ++step)
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const f32x2 v = {t[8 * step + 2 * k], t[8 * step + 2 * k + 1]};
          const half2v h = __builtin_convertvector(v, half2v);
          w[0][step][k] = __builtin_bit_cast(uint32_t, h);
          if constexpr (PREC) {
            const half2v rest = __builtin_convertvector(v - __builtin_convertvector(h, f32x2), half2v);
            w[kParts - 1][step][k] = __builtin_bit_cast(uint32_t, rest);
          }
        }
    };
    // weights times values, step n of both tiles'; the later ones are read as these are used
    auto weigh = [&](int n) {
      const int i = n % kValues / 2, step = n % 2, later = n + kAhead;
      const u32x4 v = value[n % kAhead];
      acc[i] = mfma32(v, w[0][step], acc[i]);
      if (later < kPair * kValues) value[n % kAhead] = fetch(later / kValues, later % kValues, 0);
      if constexpr (PREC) {
        acc[i] = mfma32(v, w[kParts - 1][step], acc[i]);
        acc[i] = mfma32(fetch(n / kValues, n % kValues, kValueBytes), w[0][step], acc[i]);
      }
    };
#pragma unroll
    for (int r = 0; r < 16; ++r) power(0, r);
    operands(0);
    __builtin_amdgcn_s_setprio(1);
    __builtin_amdgcn_sched_barrier(0);
    if constexpr (kPair == 2) {
#pragma unroll
      for (int r = 0; r < 16; ++r) {  // beside the second tile's powers
#pragma unroll
        for (int n = r * kValues / 16; n < (r + 1) * kValues / 16; ++n) weigh(n);
        power(kPair - 1, r);
        if (r % 2) __builtin_amdgcn_sched_barrier(0);
      }
      operands(kPair - 1);
    }
#pragma unroll
    for (int n = (kPair - 1) * kValues; n < kPair * kValues; ++n) weigh(n);
  };

  // What some lanes have written to LDS others may read from here on, and write over what they have read.  Waves with slots
  // of their own exchange within the wave, whose LDS operations the hardware does in their order; the fence and the barrier
  // (no instructions) hold the compiler to it.
  auto meet = [&] {
    if constexpr (OWN) {
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
    } else {
      __syncthreads();
    }
  };
  // the stage after `n` into LDS, and the one after that on its way
  auto advance = [&](int n) {
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      if (n + 1 < n_end) unpack_piece_into(next[i], OWN ? wave : kBuffers > 1 ? (n + 1 - n_begin) & 1 : 0, i);
      load(i);
      find(n + 3, i);
    }
  };
  for (;;) {
    bool over = false;  // whether there are large value scales
    advance(n_begin - 1);
    meet();
    for (int n = n_begin; n < n_end; ++n) {
      const int buf = OWN ? wave : kBuffers > 1 ? (n - n_begin) & 1 : 0;
      const int slot0 = list.stage(n) * kStage + (OWN ? wave * kSlots : 0);
      uint32_t flags = 0;
      {
        uint32_t of[kGroups];
        __builtin_memcpy(of, __builtin_assume_aligned(flags_lds[buf], 16), sizeof(of));
#pragma unroll
        for (int w = 0; w < kGroups; ++w) flags |= of[w];
      }
      flags = scalar(flags);
      const bool all_live = !(flags & kGaps), any_bad = flags & kBad;
      over = over || (flags & kOver);
      if (active) {
        for (int tile = OWN ? 0 : 2 * part; tile < kTiles; tile += 2 * (OWN ? 1 : p.parts)) {
          const int t0 = slot0 + 32 * tile, t1 = t0 + 32 * kPair - 1;
          // whether every row of the wave sees all of the tiles' slots, or none
          const int reach_lo = tree ? base : own_lo;  // the lowest position; slots up to it are seen, but for the window
          bool all = all_live && !any_bad && (tree ? t1 < base : t1 <= own_lo);
          if (p.window > 0) {
            all = all && (t0 > own_hi - p.window || t1 < p.sink);
            if (t1 <= reach_lo - p.window && t0 >= p.sink) continue;
          }
          if (t0 > own_hi) continue;
          __builtin_amdgcn_s_setprio(2);
          work_pair(buf, tile, t0, all, all_live, any_bad);
          __builtin_amdgcn_s_setprio(0);
        }
      }
      if (OWN || kBuffers == 1) meet();
      advance(n);
      meet();
    }
    // The large scales' turn, after the same stages: references stay, which hold for all of the scores, and so every weight
    // is added to `l` a second time.  (A run of the workgroup's, or of a wave with slots of its own, without a scale of 2^8
    // or more is through.)
    if (__builtin_expect(again || !over, 1)) break;
    again = true;
    asm volatile("" : "+v"(first_slot));  // (what the start formed of it is not kept for this)
#pragma unroll
    for (int i = 0; i < kSlices; ++i) acc[i] *= 1.0f / 256.0f;
    begin();
  }
  if (again) {
    l *= 0.5f;
#pragma unroll
    for (int i = 0; i < kSlices; ++i) acc[i] *= 256.0f;
  }

  // ---- waves of the same rows are joined (their parts of the slots in LDS, one after the other)
  if constexpr (OWN) __syncthreads();
  l += __shfl_xor(l, 32, kWave);
#pragma unroll
  for (int i = 0; i < kSlices; ++i) acc[i] *= poison >> i & 1u ? __builtin_nanf("") : 1.0f;
  if (!OWN && p.parts > 1) {
    constexpr int kRow = kSlices * 16 + 2;
    static_assert(OWN || kTiles == 2 || W / 2 * kRow * kWave * 4 <= kBuffers * kBytes, "a part's accumulators");
    float* mine = reinterpret_cast<float*>(lds[0]) + (wave % p.row_tiles) * kRow * kWave + lane;  // [row tile][kRow][lane]
    for (int other = 1; other < p.parts; ++other) {
      __syncthreads();
      if (part == other) {
#pragma unroll
        for (int i = 0; i < kSlices; ++i)
#pragma unroll
          for (int r = 0; r < 16; ++r) mine[(16 * i + r) * kWave] = acc[i][r];
        mine[(kRow - 2) * kWave] = m;
        mine[(kRow - 1) * kWave] = l;
      }
      __syncthreads();
      if (part == 0) {
        const float m2 = mine[(kRow - 2) * kWave], l2 = mine[(kRow - 1) * kWave];
        // (a part that saw nothing has l = 0, and its reference counts for nothing)
        const float ref = l2 == 0.0f ? m : l == 0.0f ? m2 : fmaxf(m, m2);
        const float a = l == 0.0f ? 0.0f : exp2f(m - ref), b = l2 == 0.0f ? 0.0f : exp2f(m2 - ref);
        m = ref;
        l = l * a + l2 * b;
#pragma unroll
        for (int i = 0; i < kSlices; ++i)
#pragma unroll
          for (int r = 0; r < 16; ++r) acc[i][r] = acc[i][r] * a + mine[(16 * i + r) * kWave] * b;
      }
    }
  }
  constexpr int kQuads = 4 * kSlices;  // of four dims of a row: the accumulators of a lane
  constexpr int kFinish = OWN ? kQuads / W : kQuads;  // of a wave
  f32x4 quads[kFinish];
  if constexpr (OWN) {  // every wave joins some of the dims
    f32x4* all = reinterpret_cast<f32x4*>(lds[0]);  // [quad][part][lane]
    f32x2* sums = reinterpret_cast<f32x2*>(all + kQuads * W * kWave);  // [part][lane]
    static_assert((kQuads * 16 + 8) * W * kWave <= kBuffers * kBytes, "the parts' accumulators");
    // (no wave reads what it has unpacked any more: they have met above)
#pragma unroll
    for (int q = 0; q < kQuads; ++q) {
      const f32x16& of = acc[q / 4];
      all[(q * W + wave) * kWave + lane] = f32x4{of[q % 4 * 4], of[q % 4 * 4 + 1], of[q % 4 * 4 + 2], of[q % 4 * 4 + 3]};
    }
    sums[wave * kWave + lane] = f32x2{m, l};
    __syncthreads();
    f32x2 of[W];
    float ref = -INFINITY;  // (a part that saw nothing has l = 0, and its reference counts for nothing)
#pragma unroll
    for (int w = 0; w < W; ++w) {
      of[w] = sums[w * kWave + lane];
      if (of[w][1] != 0.0f) ref = fmaxf(ref, of[w][0]);
    }
    m = ref;
    l = 0.0f;
#pragma unroll
    for (int i = 0; i < kFinish; ++i) quads[i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int w = 0; w < W; ++w) {
      const float by = of[w][1] != 0.0f ? exp2f(of[w][0] - ref) : 0.0f;
      l += of[w][1] != 0.0f ? of[w][1] * by : 0.0f;
#pragma unroll
      for (int i = 0; i < kFinish; ++i) quads[i] += by * all[((wave * kFinish + i) * W + w) * kWave + lane];
    }
  } else {
    if (part != 0) return;
#pragma unroll
    for (int i = 0; i < kFinish; ++i) quads[i] = f32x4{acc[i / 4][i % 4 * 4], acc[i / 4][i % 4 * 4 + 1], acc[i / 4][i % 4 * 4 + 2], acc[i / 4][i % 4 * 4 + 3]};
  }
  if (c.bits == 4) {  // a chunk's dims lie 0, 4, 1, 5 in the lower half's lanes, 2, 6, 3, 7 in the upper one's
#pragma unroll
    for (int i = 0; i < kFinish; ++i) {
      const float v[4] = {quads[i][0], quads[i][1], quads[i][2], quads[i][3]};
      const auto even = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, v[0]), __builtin_bit_cast(uint32_t, v[1]), false, false);
      const auto odd = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, v[2]), __builtin_bit_cast(uint32_t, v[3]), false, false);
      const uint32_t lanes[4] = {even[0], odd[0], even[1], odd[1]};
#pragma unroll
      for (int y = 0; y < 4; ++y) quads[i][y] = __builtin_bit_cast(float, lanes[y]);
    }
  }

  // ---- the result, or the run's partial
  const bool whole = runs == 1, none = l == 0.0f;
  const float unit = (c.bits == 4 ? kUnpackScale<4> : kUnpackScale<2>) / 128.0f;  // (of the values' scales)
  // (formed anew, the lane's number too: a register for each was kept since the query otherwise, and some in memory)
  uint32_t none_before = 0;
  asm volatile("" : "+v"(none_before));
  const int own_row = wave_row0 + static_cast<int>(__builtin_amdgcn_mbcnt_hi(~0u, __builtin_amdgcn_mbcnt_lo(~0u, none_before))) % 32;
  if (own_row >= rows) return;
  const int own_token = OWN ? own : own_row / p.gq;
  const int64_t at = (token0 + own_token) * p.query_heads + kvh * p.gq + own_row - own_token * p.gq;
  const int64_t part_at = (static_cast<int64_t>(item) * c.kv_heads + kvh) * p.block_rows + own_row - block * p.block_rows;
  const float by = !whole ? unit : none ? 0.0f : unit / l;
#pragma unroll
  for (int i = 0; i < kFinish; ++i) {
    const int dim = 8 * ((OWN ? wave * kFinish : 0) + i) + 4 * half;
    if (dim >= d) continue;
    f32x4 v;
#pragma unroll
    for (int y = 0; y < 4; ++y) v[y] = whole && none ? 0.0f : quads[i][y] * by;
    if (!whole) {
      *reinterpret_cast<f32x4*>(p.part_o + part_at * d + dim) = v;
    } else if (p.out_dtype == KVSSD_DTYPE_F32) {
      *reinterpret_cast<f32x4*>(static_cast<float*>(p.out) + at * d + dim) = v;
    } else {
      u32x2 o;
      if (p.out_dtype == KVSSD_DTYPE_F16) {
        o = u32x2{pack_half2(static_cast<_Float16>(v[0]), static_cast<_Float16>(v[1])),
                  pack_half2(static_cast<_Float16>(v[2]), static_cast<_Float16>(v[3]))};
      } else {
        o = u32x2{bf16_pair(v[0], v[1]), bf16_pair(v[2], v[3])};
      }
      *reinterpret_cast<u32x2*>(static_cast<uint16_t*>(p.out) + at * d + dim) = o;
    }
  }
  if (half == 0 && (!OWN || wave == 0)) {
    if (whole) {
      p.lse[at] = none ? -INFINITY : kLn2 * (m + log2f(l));
    } else {
      p.part_ml[2 * part_at] = m;
      p.part_ml[2 * part_at + 1] = l;
    }
  }
}

template <int DP, int W, bool PREC, bool OWN>
int launch_paged_tokens_kernel(const PagedTokensParams& p, unsigned groups, hipStream_t stream) {
  hipLaunchKernelGGL((paged_tokens_kernel<DP, W, PREC, OWN>), dim3(groups), dim3(W * kWave), 0, stream, p);
  return hip_status(hipGetLastError(), "paged_tokens launch");
}

}  // namespace kvssd
