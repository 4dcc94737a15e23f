// Paged decode attention: one query per sequence over its packed pages.
//
//   s_t = sm_scale q.k_t,  out = sum_t softmax(s)_t v_t,  lse = log sum_t e^s_t
//
// with k and v held as INT2/INT4 codes c and group scales, k = (c - mid) sk.
// Bound by the read of codes and scales (144 bytes a token and kv head in INT4
// at head_dim 128); the arithmetic below is arranged to take fewer VALU cycles
// than those bytes take to arrive.
//
// Work split.  A wave owns one kv head, up to 16 / GP of its query heads (GP:
// scale groups per head, rounded up to a power of two; NT such head tiles) and
// one run of a sequence's slots, 32 slots (a tile) at a time.  The waves of a
// workgroup take neighbouring kv heads of the same run, whose rows lie side by
// side in a page, so that whole cache lines are used.  Waves do not meet: each
// leaves an unnormalised partial (O, m, l), which paged_merge.hip joins.
//
// QK (v_mfma_f32_16x16x32_f16, two per 32 dims and tile): rows = 16 tokens'
//   codes, columns = (query head, group): the query masked to one group, so
//   that a column's sum is one group's and its scale multiplies in 32 bits
//   afterwards.  A code enters as the fp16 number 1 + c / 2^6 (INT4) or
//   1 + c / 2^2 (two bit operations for a pair); the offset's share,
//   -(1 + mid/2^6) sum q, is the accumulator's initial value.  The query is
//   scaled by a power of two per head into fp16's range (exact for fp16 and
//   bf16) and, with 32-bit queries, taken as a sum of two fp16 parts.
// Softmax in the columns' lanes: a lane holds its (head, group)'s scores of 8
//   slots; the groups' shares meet by lane exchanges within 8 lanes.  The
//   running maximum is lazy: scores up to 2^6 above the reference are summed as
//   they are (no wave-wide maximum per tile); where one exceeds that, all lanes
//   take the new maximum and rescale.  The reference also holds the exponent of
//   the largest value scale met, so that W = 2^(s - m) sv lies in fp16's normal
//   range (at most 2^15) whatever the scales' size.
// PV: rows = (head, group) weights W, columns = 16 column units of a V row, K =
//   the tile's 32 slots.  The QK result's layout (lane: column (head, group),
//   rows 4 (lane / 16) + i of both halves) is the A operand's layout if slots are
//   taken in that order, so W needs no exchange; V's codes of two slots form an
//   operand pair.  V codes enter as the exact numbers (c - mid) / 2^6: an offset
//   taken out of the sums afterwards would cost a share of their precision that
//   grows with the number of slots.  Of a unit's 16 rows those of its own group
//   count.  Where 32-bit grade is asked for, W is a sum of two fp16 parts.
#pragma once

#include "paged.hpp"

namespace kvssd {

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef _Float16 half2v __attribute__((ext_vector_type(2)));
typedef float float4v __attribute__((ext_vector_type(4)));

constexpr int kTile = 32;        // slots of a tile
constexpr int kDecodeWaves = 8;  // most waves of a workgroup
constexpr int kMaxSplits = 1024;

struct PagedDecodeParams {
  kvssd_paged_cache c;
  const void* query;
  void* out;
  float* lse;
  float* part_o;
  float* part_ml;
  float* scores;  // nullptr unless weights are summed: [sequences][query_heads][score_stride], log2 units
  int64_t score_stride;
  int capacity, chunk, splits;  // slots of a run at least, runs of a sequence at most
  int group_splits;             // runs of a workgroup (waves beyond one per kv head)
  int heads_of_group, head_groups;  // kv heads of a workgroup, workgroups over the kv heads
  int query_heads, gq, query_dtype, out_dtype;
  int tiles, tile_sets;  // head tiles of a kv head, sets of NT
  int gp_log2, groups;   // log2 of GP, groups per head
  float scale_log2;
};

// a sequence's slots per run, and its runs
__device__ __forceinline__ int run_of(int length, int chunk, int splits) {
  const int per = (length + splits - 1) / splits;
  const int up = (per + kTile - 1) / kTile * kTile;
  return up > chunk ? up : chunk;
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
int launch_paged_int2(const PagedDecodeParams& p, int dp, int nt, bool precise, hipStream_t stream);
int launch_paged_int4(const PagedDecodeParams& p, int dp, int nt, bool precise, hipStream_t stream);

// ------------------------------------------------------------------ kernel ---

__device__ __forceinline__ uint32_t sub_pair(uint32_t w, half2v off) {
  return __builtin_bit_cast(uint32_t, __builtin_bit_cast(half2v, w) - off);
}

template <int CTRL>
__device__ __forceinline__ float dpp_add(float v) {
  return v + __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xF, 0xF, false));
}

__device__ __forceinline__ float query_value(const void* q, int dtype, int64_t at) {
  if (dtype == KVSSD_DTYPE_F32) return static_cast<const float*>(q)[at];
  if (dtype == KVSSD_DTYPE_F16) return static_cast<float>(static_cast<const _Float16*>(q)[at]);
  return __builtin_bit_cast(float, static_cast<uint32_t>(static_cast<const uint16_t*>(q)[at]) << 16);
}

// Codes, scales and slot validity of one tile in a lane's registers.
template <int BITS, int DP>
struct PagedTile {
  static constexpr int kKeyWords = DP * BITS / 128;                       // a lane's quarter of a key row
  static constexpr int kUnit = DP / 16;                                   // codes of a V column unit
  static constexpr int kValueWords = kUnit * BITS > 32 ? kUnit * BITS / 32 : 1;  // (a unit below 32 bits: in one register)
  uint32_t k[2][kKeyWords];
  uint32_t v[8][kValueWords];
  uint32_t s[4];  // lanes 0-31: the slot's key scales, 32-63: its value scales (8 fp16)
  uint32_t live;  // bit e: slot tau(lane / 16, e) takes part
};

template <int BITS, int DP, int NT, bool PREC, bool UNI>
__global__ __launch_bounds__(kDecodeWaves * kWave) void paged_decode_kernel(PagedDecodeParams p) {
  using Tile = PagedTile<BITS, DP>;
  constexpr int kSlices = DP / 32;  // QK products of a half tile
  constexpr int kUnit = Tile::kUnit;
  constexpr int kParts = PREC ? 2 : 1;
  constexpr float kF = kUnpackScale<BITS>;
  constexpr float kOff = kUnpackOffset<BITS>;
  constexpr float kLazy = 6.0f;  // log2 units a score may exceed the reference by
  __shared__ uint16_t scale_lds[kDecodeWaves][2][8][kTile];  // [keys, values][group][slot order]

  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int lane = threadIdx.x % kWave;
  const int col = lane & 15, lg = lane >> 4;
  const int group_splits = p.group_splits;
  const int wg_splits = (p.splits + group_splits - 1) / group_splits;
  const int seq = blockIdx.x / wg_splits;
  const int split = (blockIdx.x % wg_splits) * group_splits + wave / p.heads_of_group;
  const int kvh = (blockIdx.y / p.tile_sets) * p.heads_of_group + wave % p.heads_of_group;
  const int set = blockIdx.y % p.tile_sets;
  const kvssd_paged_cache& c = p.c;
  if (split >= p.splits || kvh >= c.kv_heads) return;
  const int length = paged_length(c.lengths, seq, p.capacity);
  const int run = run_of(length, p.chunk, p.splits);
  const int begin = split * run;  // < 2^31: splits * run < length + splits * (chunk + 32)
  if (begin >= length && (split > 0 || p.splits > 1)) return;  // the merge knows which runs exist
  const int end = min(length, begin + run);

  const int d = c.head_dim, gs = c.group_size, gp_log2 = p.gp_log2;
  const int gp = 1 << gp_log2, hpt = 16 >> gp_log2;  // heads of a tile
  const int row_bytes = d * BITS / 8;
  const int64_t slot_bytes = static_cast<int64_t>(c.kv_heads) * row_bytes;
  const int own_g = col & (gp - 1);
  const int gq0 = set * NT * hpt;  // first query head of this wave within its kv head

  // ---- query operand, its scale and the accumulator's initial value
  // dims of the lane in slice j: granule A (j < kSlices / pieces) and, in DP 256, granule B
  half8 q[kParts][NT][kSlices];
  float c_init[NT], s_factor[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const int hh = gq0 + t * hpt + (col >> gp_log2);
    const bool has = hh < p.gq && own_g < p.groups;
    const int64_t q0 = (static_cast<int64_t>(seq) * p.query_heads + kvh * p.gq + (hh < p.gq ? hh : 0)) * d;
    float qv[kSlices][8];
    float big = 0.0f;
#pragma unroll
    for (int j = 0; j < kSlices; ++j)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        // dim of operand element (j, e): the codes' order in unpack_int4_f16 / unpack_int2_f16
        int dim;
        if constexpr (BITS == 4) {
          const int in = (e >> 1) + (e & 1) * 4;
          dim = DP == 64 ? lg * 16 + j * 8 + in : (j / 4) * 128 + lg * 32 + (j % 4) * 8 + in;
        } else {
          const int in = (j & 1) * 4 + (e >> 1) + (e & 1) * 8;
          dim = DP == 64 ? lg * 16 + in : (j / 4) * 128 + lg * 32 + ((j % 4) / 2) * 16 + in;
        }
        const float x = dim < d ? query_value(p.query, p.query_dtype, q0 + dim) : 0.0f;
        big = fmaxf(big, fabsf(x));
        qv[j][e] = has && dim < d && dim / gs == own_g ? x : 0.0f;
      }
    big = fmaxf(big, __shfl_xor(big, 16, kWave));
    big = fmaxf(big, __shfl_xor(big, 32, kWave));
    int ex = static_cast<int>((__builtin_bit_cast(uint32_t, big) >> 23) & 255u);
    ex = ex < 12 ? 12 : (ex > 253 ? 253 : ex);
    const int up = 10 + 127 - ex;  // 2^up big in [2^10, 2^11)
    const float scale_up = __builtin_bit_cast(float, static_cast<uint32_t>(127 + up) << 23);
    const float scale_down = __builtin_bit_cast(float, static_cast<uint32_t>(127 - up) << 23);
    s_factor[t] = scale_down * (kF * p.scale_log2);
    float sum = 0.0f;
#pragma unroll
    for (int j = 0; j < kSlices; ++j)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float x = qv[j][e] * scale_up;
        const _Float16 hi = static_cast<_Float16>(x);
        q[0][t][j][e] = hi;
        sum += static_cast<float>(hi);
        if constexpr (PREC) {
          const _Float16 lo = static_cast<_Float16>(x - static_cast<float>(hi));
          q[kParts - 1][t][j][e] = lo;
          sum += static_cast<float>(lo);
        }
      }
    sum += __shfl_xor(sum, 16, kWave);
    sum += __shfl_xor(sum, 32, kWave);
    c_init[t] = -kOff * sum;
  }

  // ---- where the lane's loads lie within a slot's rows (units past head_dim read from the row's start)
  const uint8_t* pk = c.packed_k + static_cast<int64_t>(kvh) * row_bytes;
  const uint8_t* pv = c.packed_v + static_cast<int64_t>(kvh) * row_bytes;
  int k_at[DP == 256 ? 2 : 1];
  if constexpr (DP == 64) {
    k_at[0] = lg * 16 < d ? lg * 2 * BITS : 0;
  } else {
#pragma unroll
    for (int g = 0; g < DP / 128; ++g) k_at[g] = g * 128 + lg * 32 < d ? (g * 128 + lg * 32) * BITS / 8 : 0;
  }
  const int v_at = col * kUnit < d ? col * kUnit * BITS / 8 : 0;
  const uint16_t* scales = (lane < 32 ? c.scales_k : c.scales_v) + static_cast<int64_t>(kvh) * p.groups;
  const int64_t slot_scales = static_cast<int64_t>(c.kv_heads) * p.groups;
  const int32_t* pages = c.page_table + static_cast<int64_t>(seq) * c.max_pages;
  const int bt = c.page_tokens;

  auto load_key = [&](const uint8_t* row, uint32_t* k) {
    if constexpr (DP == 64) {
      __builtin_memcpy(k, __builtin_assume_aligned(row + k_at[0], 4 * Tile::kKeyWords), 4 * Tile::kKeyWords);
    } else {
#pragma unroll
      for (int g = 0; g < DP / 128; ++g)
        __builtin_memcpy(k + g * BITS, __builtin_assume_aligned(row + k_at[g], 4 * BITS), 4 * BITS);
    }
  };
  auto load_value = [&](const uint8_t* row, uint32_t* v) {
    constexpr int kBytes = kUnit * BITS / 8;
    if constexpr (kBytes >= 4) {
      __builtin_memcpy(v, __builtin_assume_aligned(row + v_at, kBytes), kBytes);
    } else if constexpr (kBytes == 2) {
      v[0] = *reinterpret_cast<const uint16_t*>(row + v_at);
    } else {
      v[0] = row[v_at];
    }
  };
  auto load_scales = [&](const uint16_t* row, uint32_t* s) {
    if (p.groups == 4) {
      __builtin_memcpy(s, __builtin_assume_aligned(row, 8), 8);
    } else if (p.groups == 2) {
      __builtin_memcpy(s, __builtin_assume_aligned(row, 4), 4);
    } else if (p.groups == 8) {
      __builtin_memcpy(s, __builtin_assume_aligned(row, 16), 16);
    } else {
#pragma unroll
      for (int g = 0; g < 8; ++g)
        if (g < p.groups) {
          const uint32_t x = row[g];
          s[g / 2] = g % 2 ? s[g / 2] | x << 16 : x;
        }
    }
  };

  // slot of the tile that operand element e of this lane stands for
  auto tau = [&](int e) { return (e < 4 ? 0 : 12) + 4 * lg + e; };

  // Every load of a tile.  UNI: pages of whole tiles, so that a tile lies in one page.
  auto load_tile = [&](int base, Tile& tile) {
    uint32_t live = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) live |= (base + tau(e) < end ? 1u : 0u) << e;
    if constexpr (UNI) {
      int page = pages[base / bt];
      if (page < 0 || page >= c.num_pages) {
        page = 0;
        live = 0;
      }
      const int64_t row0 = static_cast<int64_t>(page) * bt + base % bt;
      const uint8_t* kb = pk + row0 * slot_bytes;
      const uint8_t* vb = pv + row0 * slot_bytes;
#pragma unroll
      for (int u = 0; u < 2; ++u) load_key(kb + (16 * u + col) * static_cast<int>(slot_bytes), tile.k[u]);
      load_scales(scales + (row0 + (lane & 31)) * slot_scales, tile.s);
#pragma unroll
      for (int e = 0; e < 8; ++e) load_value(vb + tau(e) * static_cast<int>(slot_bytes), tile.v[e]);
    } else {
      const int slot = base + (lane & 31);
      int row = -1;
      if (slot < end) {
        const int page = pages[slot / bt];
        if (page >= 0 && page < c.num_pages) row = page * bt + slot % bt;
      }
#pragma unroll
      for (int u = 0; u < 2; ++u)
        load_key(pk + static_cast<int64_t>(max(__shfl(row, 16 * u + col, kWave), 0)) * slot_bytes, tile.k[u]);
      load_scales(scales + static_cast<int64_t>(max(row, 0)) * slot_scales, tile.s);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int r = __shfl(row, tau(e), kWave);
        if (r < 0) live &= ~(1u << e);
        load_value(pv + static_cast<int64_t>(max(r, 0)) * slot_bytes, tile.v[e]);
      }
    }
    tile.live = live;
  };

  float4v acc[NT][kUnit];
  float m_ref[NT], l[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    m_ref[t] = -INFINITY;
    l[t] = 0.0f;
#pragma unroll
    for (int i = 0; i < kUnit; ++i) acc[t][i] = float4v{0.0f, 0.0f, 0.0f, 0.0f};
  }
  int w_exp = -32;  // W = 2^(s - m_ref) sv, m_ref = maximum + w_exp: sv < 2^(w_exp + 9)
  bool first = true;

  auto compute = [&](int base, const Tile& tile) {
    // scales into the lanes that use them: [group][lg][e]
    {
      const int x = lane & 31;
      const int at = (x & 12) * 2 + (x & 3) + (x & 16) / 4;  // 8 (x % 16 / 4) + x % 4 + 4 (x / 16)
      uint16_t(*dst)[kTile] = scale_lds[wave][lane >> 5];
      __builtin_amdgcn_wave_barrier();
#pragma unroll
      for (int g = 0; g < 8; ++g)
        if (g < p.groups) dst[g][at] = static_cast<uint16_t>(tile.s[g / 2] >> (16 * (g % 2)));
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
    }
    const int g_read = own_g < p.groups ? own_g : 0;
    uint32_t skw[4], svw[4];
    __builtin_memcpy(skw, __builtin_assume_aligned(&scale_lds[wave][0][g_read][8 * lg], 16), 16);
    __builtin_memcpy(svw, __builtin_assume_aligned(&scale_lds[wave][1][g_read][8 * lg], 16), 16);
    const bool ragged = !__all(tile.live == 255u);
    if (ragged) {  // value scales of slots that take no part may be anything: 0 (codes are always finite)
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (!(tile.live >> e & 1u)) svw[e / 2] &= e % 2 ? 0x0000FFFFu : 0xFFFF0000u;
    }
    // ---- scores
    float4v s_acc[NT][2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      half8 a[kSlices];
#pragma unroll
      for (int j = 0; j < kSlices; ++j) {
        uint32_t w[8];
        if constexpr (BITS == 4) {
          unpack_int4_f16(tile.k[u][j], w);
          __builtin_memcpy(&a[j], w, 16);
        } else if (j % 2 == 0) {
          unpack_int2_f16(tile.k[u][j / 2], w);
          __builtin_memcpy(&a[j], w, 16);
          __builtin_memcpy(&a[j + 1], w + 4, 16);
        }
      }
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        float4v s = {c_init[t], c_init[t], c_init[t], c_init[t]};
#pragma unroll
        for (int j = 0; j < kSlices; ++j) {
          s = __builtin_amdgcn_mfma_f32_16x16x32_f16(a[j], q[0][t][j], s, 0, 0, 0);
          if constexpr (PREC) s = __builtin_amdgcn_mfma_f32_16x16x32_f16(a[j], q[kParts - 1][t][j], s, 0, 0, 0);
        }
        s_acc[t][u] = s;
      }
    }
    // ---- V operands are formed per column unit below; weights first
    uint32_t sv_top;
    {
      typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
      u16x2 m = __builtin_elementwise_max(__builtin_bit_cast(u16x2, svw[0] & 0x7FFF7FFFu), __builtin_bit_cast(u16x2, svw[1] & 0x7FFF7FFFu));
      m = __builtin_elementwise_max(m, __builtin_bit_cast(u16x2, svw[2] & 0x7FFF7FFFu));
      m = __builtin_elementwise_max(m, __builtin_bit_cast(u16x2, svw[3] & 0x7FFF7FFFu));
      sv_top = m[0] > m[1] ? m[0] : m[1];
    }
    float s2[NT][8];  // scores over s_factor, summed over the groups
    float tv[NT][8];
    bool over = static_cast<int>(sv_top >> 10) - 23 > w_exp;
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      float top = -INFINITY;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const _Float16 sk = __builtin_bit_cast(half2v, skw[e / 2])[e % 2];
        float x = s_acc[t][e / 4][e % 4] * static_cast<float>(sk);
        if (own_g >= p.groups) x = 0.0f;
        if (gp_log2 > 0) x = dpp_add<0xB1>(x);
        if (gp_log2 > 1) x = dpp_add<0x4E>(x);
        if (gp_log2 > 2) x = dpp_add<0x141>(x);
        if (ragged && !(tile.live >> e & 1u)) x = -INFINITY;
        s2[t][e] = x;
        tv[t][e] = __builtin_fmaf(x, s_factor[t], -m_ref[t]);
        if (ragged && !(tile.live >> e & 1u)) tv[t][e] = -INFINITY;
        top = fmaxf(top, tv[t][e]);
      }
      over = over || top > kLazy - static_cast<float>(w_exp);
    }
    if (first || __any(over)) {
      // new reference points: the largest score so far and the largest value scale so far
      int e_new = static_cast<int>(sv_top >> 10) - 23;
#pragma unroll
      for (int k = 1; k < kWave; k <<= 1) e_new = max(e_new, __shfl_xor(e_new, k, kWave));
      e_new = max(e_new, w_exp);
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        float top = -INFINITY;
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (!ragged || (tile.live >> e & 1u)) top = fmaxf(top, s2[t][e] * s_factor[t]);
        top = fmaxf(top, __shfl_xor(top, 16, kWave));
        top = fmaxf(top, __shfl_xor(top, 32, kWave));
        const float m_old = m_ref[t] - static_cast<float>(w_exp);
        const float m_new = fmaxf(first ? -INFINITY : m_old, top);
        const float ref = m_new + static_cast<float>(e_new);
        const float alpha = first ? 0.0f : (ref == m_ref[t] ? 1.0f : exp2f(m_ref[t] - ref));
        m_ref[t] = ref;
        if (!first) {
          l[t] *= alpha;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float a = __shfl(alpha, 4 * lg + i, kWave);
#pragma unroll
            for (int k = 0; k < kUnit; ++k) acc[t][k][i] *= a;
          }
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          tv[t][e] = __builtin_fmaf(s2[t][e], s_factor[t], -ref);
          if (ragged && !(tile.live >> e & 1u)) tv[t][e] = -INFINITY;
        }
      }
      w_exp = e_new;
      first = false;
    }
    if (p.scores != nullptr) {
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const int hh = gq0 + t * hpt + (col >> gp_log2);
        if (own_g == 0 && hh < p.gq) {
          float* dst = p.scores + (static_cast<int64_t>(seq) * p.query_heads + kvh * p.gq + hh) * p.score_stride + base + 4 * lg;
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            float4v v;
#pragma unroll
            for (int i = 0; i < 4; ++i)
              v[i] = ragged && !(tile.live >> (4 * u + i) & 1u) ? -INFINITY : s2[t][4 * u + i] * s_factor[t];
            *reinterpret_cast<float4v*>(dst + 16 * u) = v;
          }
        }
      }
    }
    half8 w[kParts][NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      float sum = 0.0f;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float pe = __builtin_amdgcn_exp2f(tv[t][e]);
        sum += pe;
        const float x = pe * static_cast<float>(__builtin_bit_cast(half2v, svw[e / 2])[e % 2]);
        const _Float16 hi = static_cast<_Float16>(x);
        w[0][t][e] = hi;
        if constexpr (PREC) w[kParts - 1][t][e] = static_cast<_Float16>(x - static_cast<float>(hi));
      }
      l[t] += sum;
    }
    // ---- weights times values
    const half2v off = {static_cast<_Float16>(kOff), static_cast<_Float16>(kOff)};
    constexpr int kCodes = kUnit < 16 / BITS ? kUnit : 16 / BITS;  // codes of a 16-bit piece of a unit
#pragma unroll
    for (int piece = 0; piece < kUnit / kCodes; ++piece) {
      uint32_t b[kCodes][4];
#pragma unroll
      for (int m = 0; m < 4; ++m) {
        const uint32_t x0 = tile.v[2 * m][piece / 2], x1 = tile.v[2 * m + 1][piece / 2];
        uint32_t y;
        if constexpr (kUnit * BITS >= 32) {
          y = __builtin_amdgcn_perm(x1, x0, piece % 2 ? 0x07060302u : 0x05040100u);
        } else {
          y = x0 | (x1 << 16);
        }
        uint32_t u[8];
        if constexpr (BITS == 4) unpack_int4_f16(y, u);
        else unpack_int2_f16(y, u);
#pragma unroll
        for (int k = 0; k < kCodes; ++k) b[k][m] = sub_pair(u[k], off);
      }
#pragma unroll
      for (int k = 0; k < kCodes; ++k) {
        half8 bv;
        __builtin_memcpy(&bv, b[k], 16);
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          float4v& o = acc[t][piece * kCodes + k];
          o = __builtin_amdgcn_mfma_f32_16x16x32_f16(w[0][t], bv, o, 0, 0, 0);
          if constexpr (PREC) o = __builtin_amdgcn_mfma_f32_16x16x32_f16(w[kParts - 1][t], bv, o, 0, 0, 0);
        }
      }
    }
  };

  if (begin < end) {
    // two tiles' registers: one is loaded while the other is worked on
    const int last = begin + (end - begin - 1) / kTile * kTile;
    Tile a, b;
    load_tile(begin, a);
    for (int base = begin; base <= last; base += 2 * kTile) {
      load_tile(min(base + kTile, last), b);
      compute(base, a);
      if (base + kTile > last) break;
      load_tile(min(base + 2 * kTile, last), a);
      compute(base + kTile, b);
    }
  }

  // ---- this run's partial, or the result where a sequence has one run
  const bool whole = p.splits == 1;
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    float lt = l[t] + __shfl_xor(l[t], 16, kWave);
    lt += __shfl_xor(lt, 32, kWave);
    const int unit_g = col * kUnit / gs;  // group of this lane's column unit
    const int64_t head0 = static_cast<int64_t>(seq) * p.query_heads + kvh * p.gq;
    const int64_t part0 = (static_cast<int64_t>(seq) * p.splits + split) * p.query_heads + kvh * p.gq;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = 4 * lg + i;
      const int hh = gq0 + t * hpt + (r >> gp_log2);
      const float l_row = __shfl(lt, r, kWave);
      if ((r & (gp - 1)) != unit_g || hh >= p.gq || col * kUnit >= d) continue;
      if (whole) {
        const float inv = l_row == 0.0f ? 0.0f : kF / l_row;
#pragma unroll
        for (int k = 0; k < kUnit; ++k)
          store_out(p.out, p.out_dtype, (head0 + hh) * d + col * kUnit + k, l_row == 0.0f ? 0.0f : acc[t][k][i] * inv);
      } else {
        float* o = p.part_o + (part0 + hh) * d + col * kUnit;
#pragma unroll
        for (int k = 0; k < kUnit; k += 4)
          *reinterpret_cast<float4v*>(o + k) =
              float4v{kF * acc[t][k][i], kF * acc[t][k + 1][i], kF * acc[t][k + 2][i], kF * acc[t][k + 3][i]};
      }
    }
    const int hh = gq0 + t * hpt + (col >> gp_log2);
    if (lg == 0 && own_g == 0 && hh < p.gq) {
      if (whole) {
        p.lse[head0 + hh] = lt == 0.0f ? -INFINITY : kLn2 * (m_ref[t] + log2f(lt));
      } else {
        p.part_ml[2 * (part0 + hh)] = m_ref[t];
        p.part_ml[2 * (part0 + hh) + 1] = lt;
      }
    }
  }
}

template <int BITS, int DP, int NT, bool PREC>
int launch_paged_kernel(const PagedDecodeParams& p, hipStream_t stream) {
  const int wg_splits = (p.splits + p.group_splits - 1) / p.group_splits;
  const dim3 grid(static_cast<unsigned>(p.c.sequences) * wg_splits, p.head_groups * p.tile_sets);
  const dim3 block(p.heads_of_group * p.group_splits * kWave);
  if (p.c.page_tokens % kTile == 0)
    hipLaunchKernelGGL((paged_decode_kernel<BITS, DP, NT, PREC, true>), grid, block, 0, stream, p);
  else
    hipLaunchKernelGGL((paged_decode_kernel<BITS, DP, NT, PREC, false>), grid, block, 0, stream, p);
  return hip_status(hipGetLastError(), "paged_decode launch");
}

template <int BITS>
int launch_paged_bits(const PagedDecodeParams& p, int dp, int nt, bool precise, hipStream_t stream) {
  if (dp == 64) {
    if (nt == 1) return precise ? launch_paged_kernel<BITS, 64, 1, true>(p, stream) : launch_paged_kernel<BITS, 64, 1, false>(p, stream);
    return precise ? launch_paged_kernel<BITS, 64, 2, true>(p, stream) : launch_paged_kernel<BITS, 64, 2, false>(p, stream);
  }
  if (dp == 128) {
    if (nt == 1) return precise ? launch_paged_kernel<BITS, 128, 1, true>(p, stream) : launch_paged_kernel<BITS, 128, 1, false>(p, stream);
    return precise ? launch_paged_kernel<BITS, 128, 2, true>(p, stream) : launch_paged_kernel<BITS, 128, 2, false>(p, stream);
  }
  if (nt == 1) return precise ? launch_paged_kernel<BITS, 256, 1, true>(p, stream) : launch_paged_kernel<BITS, 256, 1, false>(p, stream);
  return precise ? launch_paged_kernel<BITS, 256, 2, true>(p, stream) : launch_paged_kernel<BITS, 256, 2, false>(p, stream);
}

}  // namespace kvssd
