// Paged decode attention: one query per sequence over its packed pages.
//
//   s_t = sm_scale q.k_t,  out = sum_t softmax(s)_t v_t,  lse = log sum_t e^s_t
//
// with k and v held as INT2/INT4 codes c and group scales, k = (c - mid) sk.
// Bound by the read of codes and scales (144 bytes a token and kv head in INT4
// at head_dim 128); the arithmetic below is arranged to take fewer VALU cycles
// than those bytes take to arrive.
// Measured (one MI355X; 8 kv and 32 query heads of 128 unless said, with the join,
// from memory): INT4, 4 sequences of 131,000 to 262,144 tokens (795 MB) 162 us,
// 4.9 TB/s of a plain read's 7.0; 64 ragged sequences up to 16,384 tokens (126 MB)
// 48 us; one of 4,096 tokens 12.2 us, round trips and one stage; INT2, 16 sequences up
// to 16,384, 64 query heads, this kernel alone 45 us, bound by its instructions (two
// head tiles unpack every code twice).  With 32-bit results, twice the products: 198,
// 52 and 13.9 us.
// A slot's codes of one head are half a line and its scales a sixteenth: waves that
// drift apart fetch the same lines again, some from memory (the 795 MB: 197 us, and
// a third more fetched; 524,288 tokens 132 us, 105 without the scales).  They meet
// before every stage's copies, which costs the arithmetic (524,288 tokens with every
// page in L2: 89 us, 103 in step) less than it saves.  Meeting every second stage,
// from the eighth on: 166 us, and 51.7 the 64 sequences.  Two kv heads a wave, with
// whole lines, need more registers than there are (300 bytes a lane spilled).
//
// Work split.  A wave owns one kv head, up to 16 / GP of its query heads (GP:
// scale groups per head, rounded up to a power of two) and one run of a
// sequence's slots, 64 slots (a stage) at a time.  The waves of a workgroup take
// neighbouring kv heads of the same run, whose rows lie side by side in a page, so
// that whole cache lines are used.  Waves pass each other nothing: each leaves an
// unnormalised partial (O, m, l), which paged_merge.hip joins.
//
// Copies.  Codes, scales and the query go from memory straight to LDS (16 or 4
// bytes a lane), into the wave's own two buffers and without a register or a
// barrier.  A stage's codes and scales are taken into registers when it begins,
// and the copies of two stages on go to their place at once: between one and two
// stages are always on the way, each awaited by the count of later copies
// (vmcnt).  With the waves' copies joined into rows of all kv heads, awaited by all
// at a barrier a stage, 524,288 slots took 142 us.  A row's 16-byte chunks are
// stored in an order turned by the row's number, so that neither the key rows' nor
// the value columns' reads meet in a bank.  Scales are laid out by group in LDS when
// their stage begins.
//
// QK (v_mfma_f32_16x16x32_f16): one side is 16 slots' codes, the other (query
//   head, group): the query masked to one group, so that a result is one group's
//   share of a score and its scale multiplies in 32 bits afterwards.  A code
//   enters as the exact number (c - mid) / 2^6 (INT4) or / 2^2, as in PV.  (As
//   1 + c / 2^6, with the offset's share taken out of the sum, it costs two
//   instructions fewer a word, 161 for 163 us of the 795 MB, and the scores what
//   the offset outweighs them by: the lse of up to 7 slots of 256 dims was off
//   1.3e-6 of itself, 1.5e-7 now.)  The query is scaled by a power of two per
//   head into fp16's range (exact for fp16 and bf16) and, with 32-bit results,
//   taken as a sum of two fp16 parts.
// Four groups and more (GP >= 4): rows = (head, group), columns = slots.  A lane
//   holds a slot's shares of four groups and adds them itself; the softmax's 2^x
//   go through LDS to the lanes that form the weights.  One or two groups: rows =
//   slots, columns = (head, group), whose lanes are the weights' lanes; with two,
//   the lanes of a head form the same scores twice.  (For four groups that form
//   took 543 vector instructions a stage, this one 418: 524,288 slots in L2 111 and
//   89 us; 25 more in both since keys are centred.)
// Softmax.  The running maximum is lazy: scores up to 2^6 above the reference are
//   summed as they are (no wave-wide maximum per stage); where one exceeds that,
//   all lanes take the new maximum and rescale.  The reference also holds the
//   exponent of the largest value scale met, so that W = 2^(s - m) sv lies in
//   fp16's normal range (at most 2^15) whatever the scales' size.
// PV: rows = (head, group) weights W, columns = 16 dims, K = 32 slots: lane
//   (row, lane / 16) forms those of the 16 slots 16 (lane / 16) + e.  V's codes
//   come transposed from LDS (ds_read_b64_tr_b4: a dim's codes of 16 slots a
//   lane) and enter as the exact numbers (c - mid) / 2^6: an offset taken out of
//   the sums afterwards would cost a share of their precision that grows with
//   the number of slots.  Of a column's 16 rows those of its own group count.
//   Where 32-bit grade is asked for, W is a sum of two fp16 parts.
#pragma once

#include <type_traits>

#include "paged.hpp"
#include "staged_ops.hpp"

namespace kvssd {

constexpr int kTile = 64;        // slots of a stage
constexpr int kMaxSplits = 1024;

// waves of a workgroup: two stages of codes each fit the CU's LDS
constexpr int decode_waves(int dp) { return dp == 256 ? 4 : 8; }

struct PagedDecodeParams {
  kvssd_paged_cache c;
  const void* query;
  void* out;
  float* lse;
  float* part_o;
  float* part_ml;
  float* scores;  // nullptr unless weights are summed: [score_stages][query_heads][kTile], log2 units
  int score_stages;  // of all sequences, one after the other; later ones have no place, and their scores are not kept
  int capacity;
  int run_tiles;    // stages of a run, unless the lengths call for more
  int runs;         // runs of all sequences that the grid and the workspace hold; == sequences: one run each
  int group_runs;   // runs of a workgroup (waves beyond one per unit)
  int group_units, groups_of_units;  // units (kv head, head tile) of a workgroup, workgroups over them
  int query_heads, gq, query_dtype, out_dtype;
  int tiles;             // head tiles of a kv head
  int groups;            // scale groups per head
  int group_log2;        // log2 of the group size
  float scale_log2;
};

// Where the runs of a ragged batch lie.  Every sequence is cut into runs of the
// same number of stages (its last may be shorter); run r of the batch is the
// r-th in the order of the sequences.  Worked out from the lengths on the
// device, by every wave for itself (64 lengths a step), so that a grid of about
// as many runs as there are serves any lengths: p.run_tiles comes from the
// caller's hints, and grows here where the lengths would need more runs than
// the grid has (sum of runs <= stages / run_tiles + sequences) or a sequence
// more than its join takes.
struct RunMap {
  int tiles;  // stages of a run
  int seq;    // of run r; -1: there is no such run
  int nth;    // its place among the sequence's
  int length;  // of the sequence (found with the run; in `runs_of`, not)
  int before;  // stages of the sequences before it, where scores are kept (as `length`)
};

__device__ __forceinline__ int length_of(const PagedDecodeParams& p, int seq) {
  return seq < p.c.sequences ? paged_length(p.c.lengths, seq, p.capacity) : 0;
}
// (`first`: the length of sequence `lane`, read once for all steps)
__device__ __forceinline__ int tiles_of_runs(const PagedDecodeParams& p, int first) {
  const int lane = threadIdx.x % kWave;
  int sum = (first + kTile - 1) / kTile, most = sum;
  for (int s = lane + kWave; s - lane < p.c.sequences; s += kWave) {
    const int n = (length_of(p, s) + kTile - 1) / kTile;
    sum += n;
    most = max(most, n);
  }
  sum = __builtin_amdgcn_readlane(wave_prefix(sum), kWave - 1);
  most = wave_most(most);
  if (p.runs <= p.c.sequences) return max(most, 1);  // one run a sequence
  const int room = p.runs - p.c.sequences;
  return max(p.run_tiles, max((sum + room - 1) / room, (most + kMaxSplits - 1) / kMaxSplits));
}

// Stages of the sequences before `seq` (fewer than 2^31 in all); `first` as there.
__device__ __forceinline__ int stages_before(const PagedDecodeParams& p, int seq, int first) {
  const int lane = threadIdx.x % kWave;
  int sum = lane < seq ? (first + kTile - 1) / kTile : 0;
  for (int s = lane + kWave; s - lane < seq; s += kWave) sum += s < seq ? (length_of(p, s) + kTile - 1) / kTile : 0;
  return __builtin_amdgcn_readlane(wave_prefix(sum), kWave - 1);
}

__device__ __forceinline__ RunMap find_run(const PagedDecodeParams& p, int r) {
  const int lane = threadIdx.x % kWave;
  const int first = length_of(p, lane);
  RunMap m{tiles_of_runs(p, first), -1, 0, 0, 0};
  if (p.runs <= p.c.sequences) {
    if (r < p.c.sequences) {
      m.seq = r;
      m.length = clamp_length(uniform_load(p.c.lengths + r), p.capacity);
      if (p.scores != nullptr) m.before = stages_before(p, r, first);
    }
    return m;
  }
  for (int s0 = 0; s0 < p.c.sequences; s0 += kWave) {
    const int length = s0 == 0 ? first : length_of(p, s0 + lane);
    const int n = ((length + kTile - 1) / kTile + m.tiles - 1) / m.tiles;
    const int upto = wave_prefix(n);
    const uint64_t past = __ballot(r < upto);
    if (past) {
      const int at = __builtin_ctzll(past);
      m.seq = s0 + at;
      m.nth = r - (__builtin_amdgcn_readlane(upto, at) - __builtin_amdgcn_readlane(n, at));
      m.length = __builtin_amdgcn_readlane(length, at);
      if (p.scores != nullptr) m.before = stages_before(p, m.seq, first);
      return m;
    }
    r -= __builtin_amdgcn_readlane(upto, kWave - 1);
  }
  return m;
}

// first run of a sequence, and its number of runs
__device__ __forceinline__ RunMap runs_of(const PagedDecodeParams& p, int seq, int* first, int* count) {
  const int lane = threadIdx.x % kWave;
  const int mine = length_of(p, lane);
  const RunMap m{tiles_of_runs(p, mine), seq, 0, 0, 0};
  int before = 0;
  for (int s0 = 0; s0 <= seq; s0 += kWave) {
    const int length = s0 == 0 ? mine : length_of(p, s0 + lane);
    const int n = ((length + kTile - 1) / kTile + m.tiles - 1) / m.tiles;
    const int upto = wave_prefix(n);
    if (seq < s0 + kWave) {
      *count = __builtin_amdgcn_readlane(n, seq - s0);
      *first = before + __builtin_amdgcn_readlane(upto, seq - s0) - *count;
    }
    before += __builtin_amdgcn_readlane(upto, kWave - 1);
  }
  return m;
}

template <typename T>
__device__ __forceinline__ void store_as(void* out, int64_t at, float v) {
  static_cast<T*>(out)[at] = store_cast<T>(v);
}
__device__ __forceinline__ void store_out(void* out, int dtype, int64_t at, float v) {
  if (dtype == KVSSD_DTYPE_F32) store_as<float>(out, at, v);
  else if (dtype == KVSSD_DTYPE_F16) store_as<_Float16>(out, at, v);
  else store_as<uint16_t>(out, at, v);
}

int launch_paged_merge(const PagedDecodeParams& p, hipStream_t stream);
// dp: head_dim padded to 64, 128 or 256; gp: groups padded to a power of two
template <int BITS, int DP>
int launch_paged_dims(const PagedDecodeParams& p, int gp, bool precise, hipStream_t stream);
template <>
int launch_paged_dims<4, 64>(const PagedDecodeParams& p, int gp, bool precise, hipStream_t stream);
template <>
int launch_paged_dims<4, 128>(const PagedDecodeParams& p, int gp, bool precise, hipStream_t stream);
template <>
int launch_paged_dims<4, 256>(const PagedDecodeParams& p, int gp, bool precise, hipStream_t stream);
template <>
int launch_paged_dims<2, 64>(const PagedDecodeParams& p, int gp, bool precise, hipStream_t stream);
template <>
int launch_paged_dims<2, 128>(const PagedDecodeParams& p, int gp, bool precise, hipStream_t stream);
template <>
int launch_paged_dims<2, 256>(const PagedDecodeParams& p, int gp, bool precise, hipStream_t stream);

// ------------------------------------------------------------------ kernel ---

typedef _Float16 half2v __attribute__((ext_vector_type(2)));

// v * a + b for an fp16 pair
__device__ __forceinline__ uint32_t fma_pair(uint32_t v, _Float16 a, _Float16 b) {
  const half2v r = __builtin_elementwise_fma(__builtin_bit_cast(half2v, v), half2v{a, a}, half2v{b, b});
  return __builtin_bit_cast(uint32_t, r);
}

// A word's codes as operand pairs.  Values: 8 slots' transposed codes (nibble e:
// slot e) as pairs (e, e + 4); INT4, the dim's (c - 8) / 64; INT2, (c - 2) / 4 of
// the nibble's even (odd = 0) or odd dim.  Keys, the same bits: a row's codes
// i and i + 4 of 8 (INT4), 2 i + odd and 2 i + odd + 8 of 16.  Codes stay where
// they are in their half, at 1 + c / F for the F of that place; one fused
// multiply-add takes out the 1 and the offset and brings all to one F, exactly.
template <int BITS>
__device__ __forceinline__ u32x4 code_operand(uint32_t x, int odd, const Masks& k, uint32_t m01, uint32_t m23) {
  const uint32_t y = x >> 8;
  if constexpr (BITS == 4) {
    const _Float16 f = 16.0f, fo = -16.125f, o = -1.125f;
    return u32x4{fma_pair(ao(x, k.m03), f, fo), fma_pair(ao(x, k.m47), 1.0f, o), fma_pair(ao(y, k.m03), f, fo),
                 fma_pair(ao(y, k.m47), 1.0f, o)};
  } else if (odd == 0) {
    const _Float16 f0 = 256.0f, o0 = -256.5f, f1 = 16.0f, o1 = -16.5f;
    return u32x4{fma_pair(ao(x, m01), f0, o0), fma_pair(ao(x, k.m45), f1, o1), fma_pair(ao(y, m01), f0, o0),
                 fma_pair(ao(y, k.m45), f1, o1)};
  } else {
    const _Float16 f0 = 64.0f, o0 = -64.5f, f1 = 4.0f, o1 = -4.5f;
    return u32x4{fma_pair(ao(x, m23), f0, o0), fma_pair(ao(x, k.m67), f1, o1), fma_pair(ao(y, m23), f0, o0),
                 fma_pair(ao(y, k.m67), f1, o1)};
  }
}

// fp16 number e of packed pairs
__device__ __forceinline__ float half_of(const uint32_t* w, int e) { return e % 2 ? half_hi(w[e / 2]) : half_lo(w[e / 2]); }

template <int CTRL>
__device__ __forceinline__ float dpp_add(float v) {
  return v + __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xF, 0xF, false));
}

// As dma16 / dma4 with a 64-bit address per lane.
__device__ __forceinline__ void dma16_at(const uint8_t* src, uint32_t lds_dst) {
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(src), "s"(lds_dst) : "memory");
}
__device__ __forceinline__ void dma4_at(const uint8_t* src, uint32_t lds_dst) {
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dword %0, off" ::"v"(src), "s"(lds_dst) : "memory");
}

// N consecutive query values (16-byte aligned) in 32 bits
template <int N>
__device__ __forceinline__ void query_span(const uint8_t* q, int dtype, int at, float* v) {
  if (dtype == KVSSD_DTYPE_F32) {
    __builtin_memcpy(v, __builtin_assume_aligned(q + 4 * at, 16), 4 * N);
    return;
  }
  uint32_t w[N / 2];
  __builtin_memcpy(w, __builtin_assume_aligned(q + 2 * at, 16), 2 * N);
  if (dtype == KVSSD_DTYPE_F16) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = i % 2 ? half_hi(w[i / 2]) : half_lo(w[i / 2]);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = __builtin_bit_cast(float, i % 2 ? w[i / 2] & 0xFFFF0000u : w[i / 2] << 16);
  }
}

__device__ __forceinline__ int scalar(int x) { return __builtin_amdgcn_readfirstlane(x); }

// UNI: pages hold whole halves (32 slots) of a stage, rows whole 16-byte chunks
// and a head's scales begin in a word alike in every row, so that a copy's rows
// have one uniform base; else every lane finds its own row's address (whole passes
// of the 64 ragged sequences 43.9 and 47.6 us, of the 795 MB 159 and 179).
template <int BITS, int DP, int GP, bool PREC, bool UNI>
__global__ __launch_bounds__(decode_waves(DP) * kWave) void paged_decode_kernel(PagedDecodeParams p) {
  constexpr int kWaves = decode_waves(DP);
  constexpr int kRow = DP * BITS / 8;      // bytes of a (padded) row in LDS
  constexpr int kChunks = kRow / 16;       // 16-byte chunks of a row; also the copies of a stage's keys or values
  constexpr int kArray = kTile * kRow;
  constexpr int kRowsOfCopy = kTile / kChunks;
  constexpr int kSlices = DP / 32;         // QK products of 16 slots
  constexpr int kSpan = DP / 4;            // dims of a lane in QK
  constexpr int kCols = DP / 16;           // PV column tiles
  constexpr int kParts = PREC ? 2 : 1;
  constexpr int kHeads = 16 / GP;          // query heads of a head tile
  constexpr float kF = kUnpackScale<BITS>;
  constexpr float kLazy = 6.0f;            // log2 units a score may exceed the reference by
  // 4-byte words copied of a slot's scales of one head (two for one: a copy's slots are then of one half)
  constexpr int kScaleWords = GP <= 4 ? 2 : 4, kScaleCopies = kScaleWords;
  constexpr int kStageCopies = 2 * (kChunks + kScaleCopies);
  __shared__ __attribute__((aligned(1024))) uint8_t codes_lds[kWaves][2][2 * kArray];
  __shared__ __attribute__((aligned(16))) uint32_t raw_lds[kWaves][2][2][kTile][kScaleWords];
  constexpr bool kSlotColumns = GP >= 4;   // QK with slots in the columns
  // [keys (where they are rows), values][group][slot], and the softmax's powers [head][slot] (rows 16 bytes apart in
  // the banks)
  __shared__ __attribute__((aligned(16))) uint16_t scale_lds[kWaves][kSlotColumns ? 1 : 2][GP][kTile];
  constexpr int kPowerRow = kTile + 4;
  __shared__ __attribute__((aligned(16))) float power_lds[kWaves][kSlotColumns ? kHeads * kPowerRow : 1];

  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int lane = threadIdx.x % kWave;
  const int col = lane & 15, lg = lane >> 4;
  // (quotients are formed in vector registers: back to scalars, as the copies' bases have to be)
  const int run = scalar(blockIdx.x * p.group_runs + wave / p.group_units);
  const int unit = scalar(blockIdx.y * p.group_units + wave % p.group_units);
  const int kvh = scalar(unit / p.tiles);
  const kvssd_paged_cache& c = p.c;
  if (kvh >= c.kv_heads) return;
  const RunMap map = find_run(p, run);
  if (map.seq < 0) return;
  const int seq = scalar(map.seq);
  const int length = scalar(map.length);
  const int begin = scalar(map.nth * map.tiles) * kTile;
  const int end = min(length, begin + scalar(map.tiles) * kTile);  // (at most 2^30 + 64 each)
  const int score_stage = scalar(map.before) + begin / kTile;  // where the run's scores lie, if they are kept

  const int d = c.head_dim;
  const int row_bytes = d * BITS / 8;
  const int64_t slot_bytes = static_cast<int64_t>(c.kv_heads) * row_bytes;
  const int64_t slot_scales = static_cast<int64_t>(c.kv_heads) * p.groups;
  const int own_g = col & (GP - 1);

  // ---- copies of a stage
  const uint8_t* pk = c.packed_k + static_cast<int64_t>(kvh) * row_bytes;
  const uint8_t* pv = c.packed_v + static_cast<int64_t>(kvh) * row_bytes;
  const uint16_t* sk = c.scales_k + static_cast<int64_t>(kvh) * p.groups;
  const uint16_t* sv = c.scales_v + static_cast<int64_t>(kvh) * p.groups;
  const int32_t* pages = c.page_table + static_cast<int64_t>(seq) * c.max_pages;
  const int bt = c.page_tokens;
  // a row's chunk i lies at place i ^ turned(row)
  auto turned = [](int row) { return ((row / (256 / kRow)) ^ (row >> 4)) & (kChunks - 1); };
  uint32_t copy_at[kChunks];  // of copy n: the lane's chunk, from its row's start (not UNI) or the copy's first row's
#pragma unroll
  for (int n = 0; n < kChunks; ++n) {
    const int lr = lane / kChunks;
    const int chunk = (lane % kChunks) ^ turned(n * kRowsOfCopy + lr);
    const int byte = chunk * 16 < row_bytes ? chunk * 16 : 0;  // (padding: the row's start again)
    copy_at[n] = UNI ? static_cast<uint32_t>((n * kRowsOfCopy % 32 + lr) * slot_bytes) + byte : byte;
  }
  // the lane's scale word of a copy of 64 / kScaleWords slots (the last word there is, where there are fewer)
  const int scale_slot = lane / kScaleWords;
  const int scale_byte = 4 * min(lane % kScaleWords, (p.groups - 1) / 2);
  const uint32_t codes0 = lds_addr(codes_lds[wave][0]);
  const uint32_t raw0 = lds_addr(reinterpret_cast<const uint8_t*>(raw_lds[wave]));
  const bool chunked = row_bytes % 16 == 0;
  // The pages of the next stage's halves, fetched one stage before they are used
  int half_page = 0, half_off = 0;  // index into `pages`, slot within the page
  if constexpr (UNI) {
    half_page = scalar(begin / bt);
    half_off = begin - half_page * bt;
  }
  int next_page[2] = {-1, -1}, next_off[2] = {0, 0};
  auto fetch_pages = [&](int base) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      next_page[h] = base + 32 * h < end ? uniform_load(pages + half_page) : -1;
      next_off[h] = half_off;
      half_off += 32;
      if (half_off == bt) {
        half_off = 0;
        ++half_page;
      }
    }
  };
  // Whether a slot's scales begin in a word's upper half, for an odd number of groups: they are copied from the word's
  // start, so that every address is a multiple of four (the arrays are).  The last scale of a pool that holds an odd
  // number of them is copied with the two bytes behind the array, of the same aligned word; they are cut off below.
  auto upper = [&](int row) { return p.groups % 2 && ((static_cast<uint32_t>(row) * c.kv_heads + kvh) & 1u); };
  // A stage to be copied: rows of the pool (of its halves; of the lane's slot where not UNI), slots that take part,
  // slots whose scales begin in a word's upper half
  struct Stage {
    int row[2];
    uint64_t live, odd;
  };
  auto locate = [&](int base) {
    Stage s;
    if constexpr (UNI) {  // (an odd number of groups: of an even number of kv heads)
      const int left = end - base;
      s.live = left >= kTile ? ~0ull : (1ull << left) - 1;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const bool ok = static_cast<uint32_t>(next_page[h]) < static_cast<uint32_t>(c.num_pages);
        s.row[h] = ok ? next_page[h] * bt + next_off[h] : 0;
        if (!ok) s.live &= h ? 0xFFFFFFFFull : 0xFFFFFFFF00000000ull;
      }
      fetch_pages(base + kTile);
      s.odd = p.groups & kvh & 1 ? ~0ull : 0;
    } else {
      const int slot = base + lane;
      int mine = -1;
      if (slot < end) {
        const int page = pages[slot / bt];
        if (page >= 0 && page < c.num_pages) mine = page * bt + slot % bt;
      }
      s.live = __ballot(mine >= 0);
      s.row[0] = s.row[1] = max(mine, 0);
      s.odd = __ballot(upper(s.row[0]));
    }
    return s;
  };
  auto copy_codes = [&](const uint8_t* src, const Stage& s, uint32_t dst) {
    if constexpr (UNI) {
      const uint8_t* half[2] = {src + s.row[0] * slot_bytes, src + s.row[1] * slot_bytes};
#pragma unroll
      for (int n = 0; n < kChunks; ++n) dma16<false>(half[n * kRowsOfCopy / 32], copy_at[n], dst + n * 1024);
    } else if (chunked) {
#pragma unroll
      for (int n = 0; n < kChunks; ++n) {
        const int64_t row = __shfl(s.row[0], n * kRowsOfCopy + lane / kChunks, kWave);
        dma16_at(src + row * slot_bytes + copy_at[n], dst + n * 1024);
      }
    } else {  // INT2 rows of an odd number of 8-byte pieces: 4 bytes a lane
      constexpr int kUnits = kRow / 4;
      for (int n = 0; n < kUnits; ++n) {
        const int r = n * (kWave / kUnits) + lane / kUnits, part = lane % kUnits;
        int byte = ((part / 4) ^ turned(r)) * 16 + part % 4 * 4;
        byte = byte < row_bytes ? byte : 0;
        const int64_t row = __shfl(s.row[0], r, kWave);
        dma4_at(src + row * slot_bytes + byte, dst + n * 256);
      }
    }
  };
  const uint32_t scale_at = static_cast<uint32_t>(scale_slot * slot_scales * 2) + scale_byte;
  auto copy_scales = [&](const uint16_t* scales, const Stage& s, uint32_t dst) {
    const uint8_t* src = reinterpret_cast<const uint8_t*>(scales);
    constexpr int kSlots = kTile / kScaleCopies;  // of a copy: 32 or 16
#pragma unroll
    for (int n = 0; n < kScaleCopies; ++n) {
      if constexpr (UNI) {
        const int64_t row = s.row[n * kSlots / 32] + n * kSlots % 32;
        dma4(src + row * slot_scales * 2 - (p.groups & kvh & 1) * 2, scale_at, dst + n * 256);
      } else {
        const int row = __shfl(s.row[0], n * kSlots + scale_slot, kWave);
        dma4_at(src + row * slot_scales * 2 - (upper(row) ? 2 : 0) + scale_byte, dst + n * 256);
      }
    }
  };
  auto copy_stage = [&](const Stage& s, int buf) {
    copy_scales(sk, s, raw0 + buf * 2 * (kScaleCopies * 256));
    copy_codes(pk, s, codes0 + buf * (2 * kArray));
    copy_scales(sv, s, raw0 + (buf * 2 + 1) * (kScaleCopies * 256));
    copy_codes(pv, s, codes0 + buf * (2 * kArray) + kArray);
  };

  // ---- the query's rows first, into the second buffer (into both, before any stage, where they need them)
  const int head_first = (unit - kvh * p.tiles) * kHeads;  // first query head of this wave within its kv head
  const int64_t head0 = static_cast<int64_t>(seq) * p.query_heads + kvh * p.gq;
  const int query_item = p.query_dtype == KVSSD_DTYPE_F32 ? 4 : 2;
  const int query_bytes = min(kHeads, p.gq - head_first) * d * query_item;
  const bool crowded = query_bytes > 2 * kArray;
  const int query_lds = crowded ? 0 : 2 * kArray;  // within the wave's buffers
  {
    const uint8_t* src = static_cast<const uint8_t*>(p.query) + (head0 + head_first) * d * query_item;
    for (int n = 0; n * 1024 < query_bytes; ++n) {
      const int at = n * 1024 + lane * 16;
      dma16_at(src + (at < query_bytes ? at : 0), codes0 + query_lds + n * 1024);
    }
  }
  const int stages = (end - begin + kTile - 1) / kTile;
  Stage now{}, next{};
  if (stages > 0) {
    if constexpr (UNI) fetch_pages(begin);
    now = locate(begin);
    if (!crowded) copy_stage(now, 0);
  }
  if (!crowded && stages > 0 && chunked) __builtin_amdgcn_s_waitcnt(vmcnt_wait(kStageCopies));
  else __builtin_amdgcn_s_waitcnt(vmcnt_wait(0));
  asm volatile("" ::: "memory");

  // ---- query operand and its scale (while the first stage arrives)
  u32x4 q[kParts][kSlices];
  const int head = head_first + col / GP;  // of the lane's column, within its kv head
  float s_factor;
  {
    float x[kSpan];
    float big = 0.0f;
    constexpr int kPieces = DP == 256 ? 2 : 1, kPiece = kSpan / kPieces;
#pragma unroll
    for (int g = 0; g < kPieces; ++g) {
      const int dim = g * 128 + lg * kPiece;
      float* v = x + g * kPiece;
      query_span<kPiece>(codes_lds[wave][0] + query_lds, p.query_dtype, (head < p.gq ? col / GP : 0) * d + (dim < d ? dim : 0), v);
#pragma unroll
      for (int i = 0; i < kPiece; ++i) big = fmaxf(big, fabsf(v[i]));
      const bool mine = head < p.gq && dim < d && dim >> p.group_log2 == own_g;
#pragma unroll
      for (int i = 0; i < kPiece; ++i) v[i] = mine ? v[i] : 0.0f;
    }
    big = fmaxf(big, __shfl_xor(big, 16, kWave));
    big = fmaxf(big, __shfl_xor(big, 32, kWave));
    int ex = static_cast<int>((__builtin_bit_cast(uint32_t, big) >> 23) & 255u);
    ex = ex < 12 ? 12 : (ex > 253 ? 253 : ex);
    const int up = 10 + 127 - ex;  // 2^up big in [2^10, 2^11)
    const float scale_up = __builtin_bit_cast(float, static_cast<uint32_t>(127 + up) << 23);
    const float scale_down = __builtin_bit_cast(float, static_cast<uint32_t>(127 - up) << 23);
    s_factor = scale_down * (kF * p.scale_log2);
#pragma unroll
    for (int j = 0; j < kSlices; ++j)
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const int lo = BITS == 4 ? j * 8 + w : j / 2 * 16 + j % 2 + 2 * w;  // the codes' order in code_operand
        const float a = x[lo] * scale_up, b = x[lo + (BITS == 4 ? 4 : 8)] * scale_up;
        const _Float16 ah = static_cast<_Float16>(a), bh = static_cast<_Float16>(b);
        q[0][j][w] = pack_half2(ah, bh);
        if constexpr (PREC) {
          const _Float16 al = static_cast<_Float16>(a - static_cast<float>(ah));
          const _Float16 bl = static_cast<_Float16>(b - static_cast<float>(bh));
          q[kParts - 1][j][w] = pack_half2(al, bl);
        }
      }
  }
  int head_own = head;  // of the lane's own results: rows 4 lg + i, all of one head, or its column
  if constexpr (kSlotColumns) {
    s_factor = __shfl(s_factor, 4 * lg, kWave);
    head_own = head_first + 4 * lg / GP;
  }
  // the query is read: the second stage may follow
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  if (crowded && stages > 0) copy_stage(now, 0);
  if (stages > 1) {
    next = locate(begin + kTile);
    copy_stage(next, 1);
  }

  // ---- where the lane reads a stage's codes
  // QK tile u's slots: 16 u + column, or row r: 16 (r / 4) + 4 u + r % 4 (and, in DP 256, chunks kChunks / 2 on)
  int key_at[4];
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    const int slot = kSlotColumns ? 16 * u + col : 16 * (col / 4) + 4 * u + col % 4;
    constexpr int kLaneBytes = (DP == 256 ? 128 : DP) * BITS / 32;  // of a lane's piece: 16, 8 or 4
    key_at[u] = slot * kRow + ((lg * kLaneBytes / 16) ^ turned(slot)) * 16 + lg * kLaneBytes % 16;
  }
  const int value_turn = turned(lane);  // slot 16 lg + col
  const int value_at = kArray + lane * kRow;
  uint32_t zero = 0;
  asm("" : "+v"(zero));
  const Masks masks = make_masks(zero);
  const uint32_t m01 = 0x00030003u | zero, m23 = 0x000C000Cu | zero;

  f32x4 acc[kCols];
#pragma unroll
  for (int i = 0; i < kCols; ++i) acc[i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  float m_ref = -INFINITY, l = 0.0f;
  int w_exp = -32;  // W = 2^(s - m_ref) sv, m_ref = maximum + w_exp: sv < 2^(w_exp + 9)
  bool first = true;

  constexpr int kLaneBytes = (DP == 256 ? 128 : DP) * BITS / 32;  // of a lane's piece of a key row: 16, 8 or 4
  // weights of a lane's 16 slots: pairs (e, e + 4) of each step's 8, the order of the values' pairs
  auto form_weights = [&](const float (&tv)[16], const uint32_t (&svw)[8], u32x4 (&w)[kParts][2]) {
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int e0 = 8 * s + k, e1 = e0 + 4;
        if constexpr (PREC) {
          // one product in 32 bits for both parts: a first part rounded straight from the factors (v_fma_mixlo_f16)
          // may be the other of its two neighbours, and the parts' sum then a step of it off
          float a = tv[e0] * half_of(svw, e0), b = tv[e1] * half_of(svw, e1);
          asm("" : "+v"(a), "+v"(b));
          const _Float16 ah = static_cast<_Float16>(a), bh = static_cast<_Float16>(b);
          w[0][s][k] = pack_half2(ah, bh);
          w[kParts - 1][s][k] = pack_half2(static_cast<_Float16>(a - static_cast<float>(ah)),
                                           static_cast<_Float16>(b - static_cast<float>(bh)));
        } else {
          w[0][s][k] = wpair(tv[e0], half_of(svw, e0), tv[e1], half_of(svw, e1));
        }
      }
  };
  // slots in the rows: the lane's column's weights of its slots 16 lg + e; some may take no part (kRagged)
  auto weigh_rows = [&](float* rows, uint64_t live, f32x4 (&s_acc)[4], const uint32_t (&skw)[8], uint32_t (&svw)[8],
                   u32x4 (&w)[kParts][2], auto ragged_tag) {
    constexpr bool kRagged = decltype(ragged_tag)::value;
    const uint32_t mask16 = static_cast<uint32_t>(live >> (16 * lg)) & 0xFFFFu;  // slots 16 lg + e
    if constexpr (kRagged) {  // value scales of slots that take no part may be anything: 0 (codes are always finite)
#pragma unroll
      for (int e = 0; e < 16; ++e)
        if (!(mask16 >> e & 1u)) svw[e / 2] &= e % 2 ? 0x0000FFFFu : 0xFFFF0000u;
    }
    uint32_t sv_top;
    {
      typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
      u16x2 m = __builtin_bit_cast(u16x2, svw[0] & 0x7FFF7FFFu);
#pragma unroll
      for (int i = 1; i < 8; ++i) m = __builtin_elementwise_max(m, __builtin_bit_cast(u16x2, svw[i] & 0x7FFF7FFFu));
      sv_top = m[0] > m[1] ? m[0] : m[1];
    }
    float tv[16];  // log2 units above the reference
    bool over = static_cast<int>(sv_top >> 10) - 23 > w_exp;
    float top = -INFINITY;
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      // products with an fp16 scale as fused multiply-adds of 0: one v_fma_mix each.  Opaque, so that the sums below
      // take the rounded product (fused into one lane's sum, it would leave a head's lanes with different scores)
      float x = __builtin_fmaf(s_acc[e / 4][e % 4], half_of(skw, e), 0.0f);
      asm("" : "+v"(x));
      if constexpr (GP > 1) x = dpp_add<0xB1>(x);
      s_acc[e / 4][e % 4] = x;
      tv[e] = kRagged && !(mask16 >> e & 1u) ? -INFINITY : __builtin_fmaf(x, s_factor, -m_ref);
      top = fmaxf(top, tv[e]);
    }
    over = over || top > kLazy - static_cast<float>(w_exp);
    if (first || __any(over)) {
      // new reference points: the largest score so far and the largest value scale so far
      const int e_new = max(static_cast<int>(wave_most((sv_top >> 10) + 9)) - 32, w_exp);
      top = -INFINITY;
#pragma unroll
      for (int e = 0; e < 16; ++e)
        if (!kRagged || (mask16 >> e & 1u)) top = fmaxf(top, s_acc[e / 4][e % 4] * s_factor);
      top = fmaxf(top, __shfl_xor(top, 16, kWave));
      top = fmaxf(top, __shfl_xor(top, 32, kWave));
      const float m_old = m_ref - static_cast<float>(w_exp);
      const float ref = fmaxf(first ? -INFINITY : m_old, top) + static_cast<float>(e_new);
      const float alpha = first ? 0.0f : (ref == m_ref ? 1.0f : exp2f(m_ref - ref));
      m_ref = ref;
      if (!first) {
        l *= alpha;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float a = __shfl(alpha, 4 * lg + i, kWave);
#pragma unroll
          for (int k = 0; k < kCols; ++k) acc[k][i] *= a;
        }
      }
#pragma unroll
      for (int e = 0; e < 16; ++e)
        tv[e] = kRagged && !(mask16 >> e & 1u) ? -INFINITY : __builtin_fmaf(s_acc[e / 4][e % 4], s_factor, -m_ref);
      w_exp = e_new;
      first = false;
    }
    if (rows != nullptr && own_g == 0 && head < p.gq) {
      float* dst = rows + head * kTile + 16 * lg;
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        f32x4 v;
#pragma unroll
        for (int i = 0; i < 4; ++i)
          v[i] = kRagged && !(mask16 >> (4 * u + i) & 1u) ? -INFINITY : s_acc[u][i] * s_factor;
        *reinterpret_cast<f32x4*>(dst + 4 * u) = v;
      }
    }
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      tv[e] = __builtin_amdgcn_exp2f(tv[e]);
      l += tv[e];
    }
    form_weights(tv, svw, w);
  };

  // slots in the columns: the powers of the lane's slots 16 u + col, of one head, left in LDS
  auto weigh_columns = [&](float* rows, uint64_t live, int e_stage, const f32x4 (&s_acc)[4], const uint32_t (&skw)[4][2],
                           auto ragged_tag) {
    constexpr bool kRagged = decltype(ragged_tag)::value;
    float s[4], tv[4];
    float top = -INFINITY;
    bool out[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      float x = 0.0f;
#pragma unroll
      for (int i = 0; i < 4; ++i) x = __builtin_fmaf(s_acc[u][i], half_of(skw[u], i), x);
      if constexpr (GP == 8) x += __shfl_xor(x, 16, kWave);
      out[u] = kRagged && !(live >> (16 * u + col) & 1);
      s[u] = x;
      tv[u] = out[u] ? -INFINITY : __builtin_fmaf(x, s_factor, -m_ref);
      top = fmaxf(top, tv[u]);
    }
    if (first || __any(e_stage > w_exp || top > kLazy - static_cast<float>(w_exp))) {
      // new reference points: the largest score so far and the largest value scale so far
      const int e_new = max(static_cast<int>(wave_most(e_stage + 32)) - 32, w_exp);
      top = -INFINITY;
#pragma unroll
      for (int u = 0; u < 4; ++u) top = out[u] ? top : fmaxf(top, s[u] * s_factor);
      top = row_max16(top);
      if constexpr (GP == 8) top = fmaxf(top, __shfl_xor(top, 16, kWave));
      const float m_old = m_ref - static_cast<float>(w_exp);
      const float ref = fmaxf(first ? -INFINITY : m_old, top) + static_cast<float>(e_new);
      const float alpha = first ? 0.0f : (ref == m_ref ? 1.0f : exp2f(m_ref - ref));
      m_ref = ref;
      if (!first) {
        l *= alpha;
#pragma unroll
        for (int k = 0; k < kCols; ++k) acc[k] *= alpha;  // (rows of the lane's own head)
      }
#pragma unroll
      for (int u = 0; u < 4; ++u) tv[u] = out[u] ? -INFINITY : __builtin_fmaf(s[u], s_factor, -m_ref);
      w_exp = e_new;
      first = false;
    }
    if (rows != nullptr && (GP < 8 || lg % 2 == 0) && head_own < p.gq) {
      float* dst = rows + head_own * kTile + col;
#pragma unroll
      for (int u = 0; u < 4; ++u) dst[16 * u] = out[u] ? -INFINITY : s[u] * s_factor;
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const float e = __builtin_amdgcn_exp2f(tv[u]);
      l += e;
      power_lds[wave][4 * lg / GP * kPowerRow + 16 * u + col] = e;
    }
  };

  // Waves of neighbouring kv heads, which share lines, meet before every stage's copies, so that a line is still in L1
  // when its other readers come.  (All waves that are left have one run, and so as many meetings.)  Not in INT2 with
  // several head tiles, which its instructions bind (16 sequences of 64 query heads: 42.5 us, 45 in step).
  const bool in_step = p.group_units > 1 && p.group_runs == 1 && (BITS == 4 || p.tiles == 1);
  for (int i = 0, base = begin; i < stages; ++i, base += kTile) {
    // the stage has landed
    if (chunked && i + 1 < stages) __builtin_amdgcn_s_waitcnt(vmcnt_wait(kStageCopies));
    else __builtin_amdgcn_s_waitcnt(vmcnt_wait(0));
    asm volatile("" ::: "memory");
    const int buf = i & 1;
    const uint8_t* stage = codes_lds[wave][buf];
    // Scales of slot `lane` as they were copied.  Groups that are fewer than GP, or begin in a word's upper half, are
    // put in order first, the missing ones as zeros (nothing else may meet a sum of zero products).
    const bool uneven = p.groups != GP;
    uint32_t raw[2][kScaleWords + 1];
#pragma unroll
    for (int a = kSlotColumns ? 1 : 0; a < 2; ++a)
      __builtin_memcpy(raw[a], __builtin_assume_aligned(raw_lds[wave][buf][a][lane], 4 * kScaleWords), 4 * kScaleWords);
    if (kSlotColumns && uneven)
      __builtin_memcpy(raw[0], __builtin_assume_aligned(raw_lds[wave][buf][0][lane], 4 * kScaleWords), 4 * kScaleWords);
    if (uneven || GP == 1) {
#pragma unroll
      for (int a = 0; a < 2; ++a) {
        raw[a][kScaleWords] = 0;
        if (now.odd >> lane & 1) {
#pragma unroll
          for (int n = 0; n < kScaleWords; ++n) raw[a][n] = raw[a][n] >> 16 | raw[a][n + 1] << 16;
        }
#pragma unroll
        for (int n = 0; n < kScaleWords; ++n)
          raw[a][n] = 2 * n + 1 < p.groups ? raw[a][n] : 2 * n < p.groups ? raw[a][n] & 0xFFFFu : 0u;
      }
      if constexpr (kSlotColumns)
        __builtin_memcpy(__builtin_assume_aligned(raw_lds[wave][buf][0][lane], 4 * kScaleWords), raw[0], 4 * kScaleWords);
    }
    uint32_t kw[4][kSpan * BITS / 32];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      __builtin_memcpy(kw[u], __builtin_assume_aligned(stage + key_at[u], kLaneBytes), kLaneBytes);
      if constexpr (DP == 256)
        __builtin_memcpy(kw[u] + kLaneBytes / 4, __builtin_assume_aligned(stage + (key_at[u] ^ (kRow / 2)), kLaneBytes), kLaneBytes);
    }
    i32x2 vw[kRow / 8];
#pragma unroll
    for (int r = 0; r < kRow / 8; ++r) vw[r] = lds_read_tr4(stage, value_at + (((r / 2) ^ value_turn) * 16) + r % 2 * 8);
#pragma unroll
    for (int a = kSlotColumns ? 1 : 0; a < 2; ++a)
#pragma unroll
      for (int g = 0; g < GP; ++g)
        scale_lds[wave][kSlotColumns ? 0 : a][g][lane] = static_cast<uint16_t>(raw[a][g / 2] >> (16 * (g % 2)));
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    uint32_t skw[8], svw[8], sk_slot[4][2];
    if constexpr (kSlotColumns) {
#pragma unroll
      for (int u = 0; u < 4; ++u)
        __builtin_memcpy(sk_slot[u], __builtin_assume_aligned(&raw_lds[wave][buf][0][16 * u + col][GP == 8 ? lg % 2 * 2 : 0], 8), 8);
    } else {
      __builtin_memcpy(skw, __builtin_assume_aligned(&scale_lds[wave][0][own_g][16 * lg], 16), 32);
    }
    __builtin_memcpy(svw, __builtin_assume_aligned(&scale_lds[wave][kSlotColumns ? 0 : 1][own_g][16 * lg], 16), 32);
    // it is read: the stage after the next may take its place
    Stage later{};
    if (i + 2 < stages) {
      later = locate(base + 2 * kTile);
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      if (in_step) __builtin_amdgcn_s_barrier();
      copy_stage(later, buf);
    }
    // ---- scores; where the kv head's are kept
    float* rows = nullptr;
    if (p.scores != nullptr && score_stage + i < p.score_stages)
      rows = p.scores + (static_cast<int64_t>(score_stage + i) * p.query_heads + kvh * p.gq) * kTile;
    f32x4 s_acc[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      f32x4 s = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int j = 0; j < kSlices; ++j) {
        const u32x4 a = BITS == 4 ? code_operand<BITS>(kw[u][j], 0, masks, m01, m23)
                                  : code_operand<BITS>(kw[u][j / 2], j % 2, masks, m01, m23);
#pragma unroll
        for (int n = 0; n < kParts; ++n) s = kSlotColumns ? mfma16(q[n][j], a, s) : mfma16(a, q[n][j], s);
      }
      s_acc[u] = s;
    }
    u32x4 w[kParts][2];
    if constexpr (kSlotColumns) {
      // exponent of the slot's largest value scale; none of a slot that takes no part, whose scales may be anything
      // (its weights are 0, and so have its scales to be; codes are always finite)
      typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
      u16x2 m = __builtin_bit_cast(u16x2, raw[1][0] & 0x7FFF7FFFu);
#pragma unroll
      for (int n = 1; n < GP / 2; ++n) m = __builtin_elementwise_max(m, __builtin_bit_cast(u16x2, raw[1][n] & 0x7FFF7FFFu));
      const int e_stage = (m[0] > m[1] ? m[0] >> 10 : m[1] >> 10) - 23;
      if (now.live == ~0ull) {
        weigh_columns(rows, now.live, e_stage, s_acc, sk_slot, std::false_type{});
      } else {
        weigh_columns(rows, now.live, now.live >> lane & 1 ? e_stage : -32, s_acc, sk_slot, std::true_type{});
        const uint32_t mask16 = static_cast<uint32_t>(now.live >> (16 * lg)) & 0xFFFFu;
#pragma unroll
        for (int e = 0; e < 16; ++e)
          if (!(mask16 >> e & 1u)) svw[e / 2] &= e % 2 ? 0x0000FFFFu : 0xFFFF0000u;
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
      float powers[16];
      __builtin_memcpy(powers, __builtin_assume_aligned(&power_lds[wave][col / GP * kPowerRow + 16 * lg], 16), 64);
      form_weights(powers, svw, w);
    } else {
      if (now.live == ~0ull) weigh_rows(rows, now.live, s_acc, skw, svw, w, std::false_type{});
      else weigh_rows(rows, now.live, s_acc, skw, svw, w, std::true_type{});
    }
    // ---- weights times values: 8 bytes of a row a read, 16 (INT4) or 32 (INT2) dims
#pragma unroll
    for (int r = 0; r < kRow / 8; ++r) {
      const i32x2 x = vw[r];
#pragma unroll
      for (int s = 0; s < 2; ++s)
#pragma unroll
        for (int odd = 0; odd < (BITS == 4 ? 1 : 2); ++odd) {
          const u32x4 b = code_operand<BITS>(static_cast<uint32_t>(x[s]), odd, masks, m01, m23);
          const int tile = BITS == 4 ? r : 2 * r + odd;
          acc[tile] = mfma16(w[0][s], b, acc[tile]);
          if constexpr (PREC) acc[tile] = mfma16(w[kParts - 1][s], b, acc[tile]);
        }
    }
    now = next;
    next = later;
  }

  // ---- this run's partial, or the result where a sequence has one run
  const bool whole = p.runs <= c.sequences;
  const int64_t part0 = static_cast<int64_t>(run) * p.query_heads + kvh * p.gq;
  if constexpr (kSlotColumns) {
    l = row_sum16(l);
  } else {
    l += __shfl_xor(l, 16, kWave);
    l += __shfl_xor(l, 32, kWave);
  }
  // a column tile's dims are of one group gk; of the lane's rows 4 lg + i = (head, group) the kRows with that group
  // hold them
  constexpr int kRows = 4 / (GP < 4 ? GP : 4);
#pragma unroll
  for (int n = 0; n < kRows; ++n) {
    const int h = GP >= 4 ? 4 * lg / GP : kRows * lg + n;  // within the head tile
    const float l_head = kSlotColumns ? l : __shfl(l, h * GP, kWave);
    const float factor = !whole ? kF : l_head == 0.0f ? 0.0f : kF / l_head;
    const bool has = head_first + h < p.gq;
#pragma unroll
    for (int k = 0; k < kCols; ++k) {
      const int dim = BITS == 4 ? 16 * k + col : 32 * (k / 2) + 2 * col + k % 2;
      const int gk = scalar((BITS == 4 ? 16 * k : 32 * (k / 2)) >> p.group_log2);
      const int i = GP >= 4 ? gk & 3 : GP == 2 ? gk % 2 + 2 * n : n;
      const float v01 = i & 1 ? acc[k][1] : acc[k][0], v23 = i & 1 ? acc[k][3] : acc[k][2];
      const float v = (i & 2 ? v23 : v01) * factor;
      if (!has || dim >= d || (GP == 8 && (lg & 1) != gk >> 2)) continue;
      if (whole) store_out(p.out, p.out_dtype, (head0 + head_first + h) * d + dim, l_head == 0.0f ? 0.0f : v);
      else p.part_o[(part0 + head_first + h) * d + dim] = v;
    }
  }
  if (kSlotColumns ? col == 0 && (GP < 8 || lg % 2 == 0) && head_own < p.gq : lg == 0 && own_g == 0 && head < p.gq) {
    if (whole) {
      p.lse[head0 + head_own] = l == 0.0f ? -INFINITY : kLn2 * (m_ref + log2f(l));
    } else {
      p.part_ml[2 * (part0 + head_own)] = m_ref;
      p.part_ml[2 * (part0 + head_own) + 1] = l;
    }
  }
}

template <int BITS, int DP, int GP, bool PREC>
int launch_paged_kernel(const PagedDecodeParams& p, hipStream_t stream) {
  const dim3 grid((p.runs + p.group_runs - 1) / p.group_runs, p.groups_of_units);
  const dim3 block(p.group_units * p.group_runs * kWave);
  if constexpr (DP * BITS >= 256) {
    if (p.c.page_tokens % 32 == 0 && p.c.head_dim * BITS % 128 == 0 && !(p.groups % 2 && p.c.kv_heads % 2)) {
      hipLaunchKernelGGL((paged_decode_kernel<BITS, DP, GP, PREC, true>), grid, block, 0, stream, p);
      return hip_status(hipGetLastError(), "paged_decode launch");
    }
  }
  hipLaunchKernelGGL((paged_decode_kernel<BITS, DP, GP, PREC, false>), grid, block, 0, stream, p);
  return hip_status(hipGetLastError(), "paged_decode launch");
}

template <int BITS, int DP, int GP>
int launch_paged_shape(const PagedDecodeParams& p, bool precise, hipStream_t stream) {
  return precise ? launch_paged_kernel<BITS, DP, GP, true>(p, stream) : launch_paged_kernel<BITS, DP, GP, false>(p, stream);
}

}  // namespace kvssd
