// Attention of one new token per sequence over a paged key-value cache, split
// over the caches' lengths and joined.
//
//   out[b][h] = sum_t p_t v_t / sum_t p_t,  p_t = exp(scale q[b][h].k_t - max)
//
// Bound by reading K and V once.  The visible keys of all (sequence, KV head)
// items are cut into tiles of 32 keys, laid end to end, and dealt to the
// workgroups in equal runs, so that ragged batches, single long sequences and
// many short ones fill the chip alike.  A run that covers an item's tiles only in
// part leaves a partial (O, max, sum), and a second kernel joins these in order.
//
// A wave takes 32 keys at a time on MFMA, with no LDS in the loop:
//   S^T [keys x heads] = K Q^T: a lane's A operand is 16 bytes of a key's row,
//     loaded as they lie; the 16 columns are the KV head's query heads.
//   O^T [dims x heads] += V^T P^T: the lane's S^T values are its B operand as
//     they are (the order of the contraction's keys is free), and the A operand
//     is a transposition of 8 keys x D / 16 dims within the lane's registers.
// Row maximum and sum belong to a column, so each lane holds its own head's.
//
// Measured (32 / 8 heads, D = 128): one sequence of 131072 keys 92 .. 98 us, 5.5 .. 5.8 TB/s,
// what plain reads reach; 24 sequences of 61 to 16001 keys in pages of 64 rows 62 us,
// 4.9 TB/s; 1000 keys 6.6 us. 16 / 4 heads of D = 256, windows of 4096 keys, 8 sequences: 34 us,
// 4.1 TB/s. The join takes 5 to 6 us, most of it a launch and three dependent loads.
// Without gain: tiles of 64 keys, a tile's loads a step ahead (the registers cost a
// workgroup a CU), more than two workgroups a CU.
#pragma once

#include "fpv2_common.h"
#include "fpv2_decode.h"

namespace fpv2 {
namespace {

constexpr int kTileKeys = 32;   // keys of a wave's tile
constexpr int kWaves = 4;
constexpr int kStepKeys = kWaves * kTileKeys;
// What an item costs a workgroup beside its tiles (its queries, its first rows'
// addresses, the join of the waves), in tiles.  24 sequences of 61 to 16001 keys:
// counted as none 69 us, as 4 62.5, 8 62.4, 16 63.6 us.
constexpr int kItemUnits = 8;
constexpr int kMaxGrid = 4096;   // workgroups of a call
constexpr int kMaxHeads = 16;  // query heads of an item (columns of an MFMA tile)

struct DecodeArgs {
  const uint16_t* q;
  const uint16_t* k;
  const uint16_t* v;
  uint16_t* out;
  const int32_t* table;
  const int32_t* lengths;
  float* part_o;   // [2 * grid][item_heads][D]
  float* part_ml;  // [2 * grid][item_heads][2]
  int64_t q_bs, q_hs, k_ps, k_hs, k_rs, v_ps, v_hs, v_rs, o_bs, o_hs, table_stride;
  int batch, kv_heads, group, item_heads, head_items;  // head_items * item_heads >= group
  int pages, page_size, capacity, length, window, sinks, grid;
  int join_runs;  // the join's workgroups go by runs, not by items
  uint32_t page_mul, page_shift;  // t / page_size = (umulhi(t, mul) + t) >> shift
  float scale_log2;
};

struct Sequence {
  int n;      // visible keys
  int sinks;  // of which at the start
  int skip;   // key of visible index u >= sinks: u + skip
  int tiles;
  __device__ __forceinline__ int units() const { return kItemUnits + tiles; }
};

__device__ __forceinline__ Sequence sequence_of(const DecodeArgs& a, int b) {
  int len = a.lengths != nullptr ? a.lengths[b] : a.length;
  len = min(max(len, 0), a.capacity);
  Sequence s;
  s.sinks = min(a.sinks, len);
  const int start = max(s.sinks, len - a.window);
  s.skip = start - s.sinks;
  s.n = len - s.skip;
  s.tiles = max(1, (s.n + kTileKeys - 1) / kTileKeys);  // (an empty one writes its zeros)
  return s;
}

// Units of one item of a lane's sequences [lane per, ..) and the lanes' before it.
struct Prefix {
  int per, upto, total;
};
__device__ __forceinline__ int scan_add(int x, int lane) {
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const int up = __shfl_up(x, off, 64);
    x += lane >= off ? up : 0;
  }
  return x;
}
__device__ __forceinline__ Prefix prefix_of(const DecodeArgs& a, int lane) {
  Prefix p;
  p.per = (a.batch + 63) / 64;
  int sum = 0;
#pragma unroll 4
  for (int i = 0; i < p.per; ++i) {
    const int b = lane * p.per + i;
    sum += b < a.batch ? sequence_of(a, b).units() : 0;
  }
  p.upto = scan_add(sum, lane);
  p.total = __builtin_amdgcn_readlane(p.upto, 63);
  return p;
}
// Units of one item of the sequences before b.
__device__ __forceinline__ int units_before(const DecodeArgs& a, const Prefix& p, int lane, int b) {
  const int at = b / p.per;
  const int base = at > 0 ? __shfl(p.upto, at - 1, 64) : 0;
  if (p.per == 1) return base;
  int some = 0;
  for (int i = at * p.per + lane; i < b; i += 64) some += sequence_of(a, i).units();
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) some += __shfl_xor(some, off, 64);
  return base + some;
}
// The sequence that holds a unit of all items, and its first unit.
__device__ __forceinline__ int sequence_at(const DecodeArgs& a, const Prefix& p, int lane, int unit, int* first) {
  const int items = a.kv_heads * a.head_items;
  const int at = __ffsll(static_cast<unsigned long long>(__ballot(p.upto * items > unit))) - 1;
  int b = at * p.per, base = at > 0 ? __shfl(p.upto, at - 1, 64) * items : 0;
  if (p.per > 1) {
    for (int b0 = b; b0 < a.batch; b0 += 64) {
      const int sum = scan_add(b0 + lane < a.batch ? sequence_of(a, b0 + lane).units() * items : 0, lane);
      const uint64_t past = __ballot(base + sum > unit);
      if (past != 0) {
        const int l = __ffsll(static_cast<unsigned long long>(past)) - 1;
        b = b0 + l;
        base += l > 0 ? __shfl(sum, l - 1, 64) : 0;
        break;
      }
      base += __shfl(sum, 63, 64);
    }
  }
  *first = __builtin_amdgcn_readfirstlane(base);
  return __builtin_amdgcn_readfirstlane(b);
}

// The workgroups that have a run: of a tile for each wave at least.
__device__ __forceinline__ uint32_t runs_of(const DecodeArgs& a, int total) {
  return min(a.grid, (total + kWaves - 1) / kWaves);
}
// The first unit of a workgroup's run (runs differ by a unit at most), and the
// workgroup that has a unit.
__device__ __forceinline__ int first_of(const DecodeArgs& a, uint32_t w, int total) {
  const uint32_t runs = runs_of(a, total), per = static_cast<uint32_t>(total) / runs, i = min(w, runs);
  return static_cast<int>(i * per + i * (static_cast<uint32_t>(total) - per * runs) / runs);  // i total / runs
}
__device__ __forceinline__ int workgroup_of(const DecodeArgs& a, int unit, int total) {
  const uint32_t runs = runs_of(a, total);
  return static_cast<int>((static_cast<uint64_t>(unit + 1) * runs - 1) / static_cast<uint32_t>(total));
}

// What a tile's float16 weights are relative to: `headroom` below their greatest exponent, so that this
// one's weight is 2^headroom.  From 2^24 on not every whole number is a float32 one, and 16 below would be a
// weight of infinity: there 7 below it, which no rounding makes more than 8.
__device__ __forceinline__ float below(float greatest, float headroom) {
  const float to = greatest - headroom;
  return greatest - to > 15.f ? greatest - 7.f : to;
}

// The maximum of a column's four lanes, in each of them.
__device__ __forceinline__ float column_max(float x) {
  const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}

template <int NW>
struct Words { uint32_t w[NW]; };

template <int NW>
__device__ __forceinline__ Words<NW> load_words(const uint16_t* p) {
  Words<NW> r;
  if constexpr (NW % 4 == 0) {
#pragma unroll
    for (int i = 0; i < NW / 4; ++i) {
      const u32x4 x = load16(p + 8 * i);
#pragma unroll
      for (int j = 0; j < 4; ++j) r.w[4 * i + j] = x[j];
    }
  } else if constexpr (NW == 2) {
    const u32x2 x = *reinterpret_cast<const u32x2*>(p);
    r.w[0] = x[0];
    r.w[1] = x[1];
  } else {
#pragma unroll
    for (int i = 0; i < NW; ++i) r.w[i] = reinterpret_cast<const uint32_t*>(p)[i];
  }
  return r;
}

template <int D>
struct DecodeShared {
  // (at head dim 256 the queries would not fit the registers beside K, V and O)
  static constexpr bool kLdsQ = D > 128;
  float o[4][kMaxHeads][D + 4];
  float ml[4][kMaxHeads][2];
  u32x4 q[kLdsQ ? 2 * D : 1];
};

// A workgroup of 256 threads.
template <typename T, int D>
__device__ __forceinline__ void decode_attn(const DecodeArgs& a, int block, DecodeShared<D>& sh) {
  constexpr int KK = D / 32;  // MFMA steps of a key's dot product
  constexpr int DV = D / 16;  // dims of a lane
  // Weights are rounded to the storage type for their product with V, as MFMA takes them; the
  // sum is of the unrounded ones.  float16 has only 2^-14 to 1 at full precision, so there
  // they are relative to 2^-15 of the tile's own greatest instead of the greatest so far
  // (a tile 2^-40 and more below it: of 2^-40 of it, so that no float32 sum overflows).
  // Relative to the greatest, the rest of a sequence 12 to 17 nats below one key lost up to
  // a quarter of its weight.
  constexpr bool kByTile = std::is_same<T, f16_t>::value;
  constexpr float kHeadroom = 15.f, kBelow = 40.f;
  constexpr bool kLdsQ = DecodeShared<D>::kLdsQ;
  auto& sh_o = sh.o;
  auto& sh_ml = sh.ml;
  auto& sh_q = sh.q;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 15, quad = lane >> 4;
  const int items = a.kv_heads * a.head_items;

  const Prefix prefix = prefix_of(a, lane);
  const int total = prefix.total * items;
  const int lo = first_of(a, block, total), hi = first_of(a, block + 1, total);
  if (lo >= hi) return;

  int base;
  int b = sequence_at(a, prefix, lane, lo, &base);
  Sequence s = sequence_of(a, b);
  for (int cur = lo, end; cur < hi; cur = end) {
    const int units = s.units();
    const int item = (cur - base) / units;
    const int item_start = base + item * units;
    end = min(hi, item_start + units);
    // tiles [first, last) of the item; the run may start or end among the other units
    const int first = max(0, cur - item_start - kItemUnits), last = end - item_start - kItemUnits;
    const int b_now = b;
    const Sequence s_now = s;
    if (end < hi && end == base + items * units) {
      base = end;
      s = sequence_of(a, ++b);
    }
    if (last <= first) continue;
    const int kvh = item / a.head_items;
    const int h0 = (item - kvh * a.head_items) * a.item_heads;
    const int heads = min(a.item_heads, a.group - h0);
    const int head = kvh * a.group + h0 + col;

    u32x4 qf[kLdsQ ? 1 : KK];
    const auto load_q = [&](int kk) {
      return col < heads ? load16(a.q + b_now * a.q_bs + head * a.q_hs + 32 * kk + 8 * quad) : u32x4{0, 0, 0, 0};
    };
    if constexpr (kLdsQ) {
      for (int kk = wave; kk < KK; kk += 4) sh_q[64 * kk + lane] = load_q(kk);
      __syncthreads();
    } else {
#pragma unroll
      for (int kk = 0; kk < KK; ++kk) qf[kk] = load_q(kk);
    }
    f32x4 o[DV];
#pragma unroll
    for (int d = 0; d < DV; ++d) o[d] = f32x4{0.f, 0.f, 0.f, 0.f};
    float m = neg_inf(), l = 0.f;  // the exponent that O and l are relative to
    float greatest = neg_inf();

    const uint16_t* kb = a.k + kvh * a.k_hs;
    const uint16_t* vb = a.v + kvh * a.v_hs;
    const int32_t* table = a.table != nullptr ? a.table + b_now * a.table_stride : nullptr;
    // lane i (and i + 32) looks up the row of the tile's key i
    auto lookup = [&](int u0, int* row) {
      const int u = min(u0 + (lane & 31), s_now.n - 1);
      const uint32_t t = u < s_now.sinks ? u : u + s_now.skip;
      const uint32_t page = (__umulhi(t, a.page_mul) + t) >> a.page_shift;
      *row = t - page * a.page_size;
      const int id = table != nullptr ? table[page] : b_now;
      return min(max(id, 0), a.pages - 1);
    };
    int u0 = first * kTileKeys + wave * kTileKeys;
    const int u_end = min(s_now.n, last * kTileKeys);
    int row = 0, page = 0;
    if (u0 < u_end) page = lookup(u0, &row);
    for (; u0 < u_end; u0 += kStepKeys) {
      const int64_t koff = page * a.k_ps + row * a.k_rs;
      const int64_t voff = page * a.v_ps + row * a.v_rs;
      u32x4 kf[2][KK];
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const uint16_t* p = kb + __shfl(koff, 16 * t + col, 64) + 8 * quad;
#pragma unroll
        for (int kk = 0; kk < KK; ++kk) kf[t][kk] = load16(p + 32 * kk);
      }
      // (at head dim 256 half of V waits for K's registers)
      constexpr int kEarly = D > 128 ? 4 : 8;
      Words<DV / 2> vf[8];
      const auto load_v = [&](int j) {
        return load_words<DV / 2>(vb + __shfl(voff, 16 * (j / 4) + 4 * quad + j % 4, 64) + DV * col);
      };
#pragma unroll
      for (int j = 0; j < kEarly; ++j) vf[j] = load_v(j);
      if (u0 + kStepKeys < u_end) page = lookup(u0 + kStepKeys, &row);

      int q_at = lane;
      if constexpr (kLdsQ) asm volatile("" : "+v"(q_at));  // (read again for each tile)
      f32x4 sc[2];
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        sc[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int kk = 0; kk < KK; ++kk)
          sc[t] = Elem<T>::mfma16(as_vec8<T>(kf[t][kk]), as_vec8<T>(kLdsQ ? sh_q[64 * kk + q_at] : qf[kLdsQ ? 0 : kk]), sc[t]);
      }
#pragma unroll
      for (int j = kEarly; j < 8; ++j) vf[j] = load_v(j);
      const bool cut = u0 + kTileKeys > s_now.n;
      float x[8], top = neg_inf();
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        x[j] = sc[j / 4][j % 4] * a.scale_log2;
        if (cut && u0 + 16 * (j / 4) + 4 * quad + j % 4 >= s_now.n) {
          x[j] = neg_inf();
          // (a zero weight would make NaN of what an unused row may hold)
#pragma unroll
          for (int w = 0; w < DV / 2; ++w) vf[j].w[w] = 0;
        }
        top = fmaxf(top, x[j]);
      }
      top = fmaxf(top, __shfl_xor(top, 16, 64));
      top = fmaxf(top, __shfl_xor(top, 32, 64));
      float m_new = fmaxf(m, top);
      if constexpr (kByTile) {
        greatest = fmaxf(greatest, top);
        m_new = below(fmaxf(top, greatest - kBelow), kHeadroom);
      }
      // (nothing but -inf so far: weights of zero instead of NaN)
      const float ref = m_new == neg_inf() ? 0.f : m_new;
      const float fix = __builtin_amdgcn_exp2f(m - ref);
      m = m_new;
      l *= fix;
      u32x4 pf;
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = __builtin_amdgcn_exp2f(x[j] - ref);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        pf[j] = pack2<T>(x[2 * j], x[2 * j + 1]);
        l += x[2 * j] + x[2 * j + 1];
      }
#pragma unroll
      for (int d = 0; d < DV; ++d) {
        o[d] *= fix;
        u32x4 vt;  // dim d of the lane's 8 keys
#pragma unroll
        for (int j = 0; j < 4; ++j)
          vt[j] = __builtin_amdgcn_perm(vf[2 * j + 1].w[d / 2], vf[2 * j].w[d / 2],
                                        d % 2 ? 0x07060302u : 0x05040100u);
        o[d] = Elem<T>::mfma16(as_vec8<T>(vt), as_vec8<T>(pf), o[d]);
      }
    }
    l += __shfl_xor(l, 16, 64);
    l += __shfl_xor(l, 32, 64);

    // join the four waves
    if (quad == 0) {
      sh_ml[wave][col][0] = m;
      sh_ml[wave][col][1] = l;
    }
    if (col < heads) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int d = 0; d < DV; ++d) sh_o[wave][col][(4 * quad + i) * DV + d] = o[d][i];
    }
    __syncthreads();
    const bool whole = first == 0 && last == s_now.tiles;
    const int64_t slot = 2 * static_cast<int64_t>(block) + (cur == lo ? 0 : 1);
    for (int e = tid; e < heads * D; e += 256) {
      const int h = e / D, d = e % D;
      float top = neg_inf();
#pragma unroll
      for (int w = 0; w < 4; ++w) top = fmaxf(top, sh_ml[w][h][0]);
      const float ref = top == neg_inf() ? 0.f : top;
      float sum = 0.f, den = 0.f;
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        // (a wave without keys has max -inf, sum 0 and O 0)
        const float f = __builtin_amdgcn_exp2f(sh_ml[w][h][0] - ref);
        sum += f * sh_o[w][h][d];
        den += f * sh_ml[w][h][1];
      }
      if (whole) {
        const float r = s_now.n == 0 ? 0.f : sum / den;
        a.out[b_now * a.o_bs + (kvh * a.group + h0 + h) * a.o_hs + d] = Elem<T>::from_float(r);
      } else {
        a.part_o[(slot * a.item_heads + h) * D + d] = sum;
        if (d == 0) {
          a.part_ml[(slot * a.item_heads + h) * 2] = top;
          a.part_ml[(slot * a.item_heads + h) * 2 + 1] = den;
        }
      }
    }
    __syncthreads();
  }
}

template <typename T, int D>
__global__ __launch_bounds__(256, 2) void decode_attn_kernel(DecodeArgs a) {
  __shared__ DecodeShared<D> sh;
  decode_attn<T, D>(a, blockIdx.x, sh);
}

// Joins the partials of an item that several workgroups shared: one workgroup
// per (item, query head, DS of the dims), or where there are more items than runs,
// per (run, ..) for the item that goes on in the next one.  First the weights of
// all partials, then their sum, 16 bytes of a partial a thread.
template <typename T, int D, int DS>
__global__ __launch_bounds__(256) void decode_join_kernel(DecodeArgs a) {
  constexpr int kLanes = DS / 4, kSlots = 256 / kLanes;  // partials at a time
  constexpr int kParts = D / DS;
  __shared__ float sh_f[kMaxGrid];
  __shared__ float sh_r[4];
  __shared__ f32x4 sh_o[kSlots][kLanes];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int items = a.kv_heads * a.head_items;
  const int d0 = blockIdx.x % kParts * DS, h = blockIdx.x / kParts % a.item_heads;
  const int at = blockIdx.x / kParts / a.item_heads;
  const Prefix prefix = prefix_of(a, lane);
  const int total = prefix.total * items;
  int b, item, base;
  if (a.join_runs) {
    if (at + 1 >= static_cast<int>(runs_of(a, total))) return;
    const int unit = first_of(a, at + 1, total);
    b = sequence_at(a, prefix, lane, unit, &base);
    item = (unit - base) / sequence_of(a, b).units();
  } else {
    b = at / items;
    item = at - b * items;
    base = units_before(a, prefix, lane, b) * items;
  }
  const int kvh = item / a.head_items, h0 = (item - kvh * a.head_items) * a.item_heads;
  if (h0 + h >= a.group) return;
  const Sequence s = sequence_of(a, b);
  const int start = base + item * s.units();
  const int w0 = workgroup_of(a, start + kItemUnits, total);
  if (a.join_runs && w0 != at) return;  // not in the run, or another run's item
  const int n = workgroup_of(a, start + s.units() - 1, total) - w0 + 1;
  if (n == 1) return;  // written by its workgroup
  // a workgroup's first item is in its slot 0, its last in slot 1
  const int in_last = start > first_of(a, w0, total) ? 1 : 0;
  const auto slot_of = [&](int i) { return 2 * static_cast<int64_t>(w0 + i) + (i == 0 ? in_last : 0); };
  float top = neg_inf();
  for (int i = tid; i < n; i += 256) {
    const float m = a.part_ml[(slot_of(i) * a.item_heads + h) * 2];
    sh_f[i] = m;
    top = fmaxf(top, m);
  }
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) top = fmaxf(top, __shfl_xor(top, off, 64));
  if (lane == 0) sh_r[wave] = top;
  __syncthreads();
  top = fmaxf(fmaxf(sh_r[0], sh_r[1]), fmaxf(sh_r[2], sh_r[3]));
  const float ref = top == neg_inf() ? 0.f : top;
  __syncthreads();
  float den = 0.f;
  for (int i = tid; i < n; i += 256) {
    const float f = __builtin_amdgcn_exp2f(sh_f[i] - ref);
    sh_f[i] = f;
    den += f * a.part_ml[(slot_of(i) * a.item_heads + h) * 2 + 1];
  }
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) den += __shfl_xor(den, off, 64);
  if (lane == 0) sh_r[wave] = den;
  __syncthreads();
  den = (sh_r[0] + sh_r[1]) + (sh_r[2] + sh_r[3]);
  f32x4 o = {0.f, 0.f, 0.f, 0.f};
  const int g = tid / kLanes, e = tid % kLanes;
  if (g < kSlots) {
#pragma unroll 8
    for (int i = g; i < n; i += kSlots)
      o += sh_f[i] * *reinterpret_cast<const f32x4*>(a.part_o + (slot_of(i) * a.item_heads + h) * D + d0 + 4 * e);
    sh_o[g][e] = o;
  }
  __syncthreads();
  if (tid < kLanes) {
#pragma unroll
    for (int i = 1; i < kSlots; ++i) o += sh_o[i][tid];
    uint16_t* out = a.out + b * a.o_bs + (kvh * a.group + h0 + h) * a.o_hs + d0 + 4 * tid;
#pragma unroll
    for (int j = 0; j < 4; ++j) out[j] = Elem<T>::from_float(o[j] / den);
  }
}

template <typename T, int D>
void launch_join(const DecodeArgs& a, hipStream_t s) {
  // An item of many partials is joined by several workgroups.  One item of 512
  // partials, 8 heads: the call 27.4 us by whole heads / 24.8 by 32 dims at D =
  // 128, 41.8 / 35.1 at D = 256; 8 items of 64 partials: the join 5.7 / 6.1.
  // With more items than runs most have one workgroup, and there is a join for a run at
  // most: 512 sequences of 64 keys, 32 / 8 heads of D = 64: the join 36 us by items, 12.7
  // by runs; 64 sequences of 8 items 3.9 by items.
  const unsigned items = a.join_runs ? a.grid - 1 : static_cast<unsigned>(a.batch) * a.kv_heads * a.head_items;
  if (a.grid >= 128u * items)
    hipLaunchKernelGGL((decode_join_kernel<T, D, 32>), dim3(items * a.item_heads * (D / 32)), dim3(256), 0, s, a);
  else
    hipLaunchKernelGGL((decode_join_kernel<T, D, D>), dim3(items * a.item_heads), dim3(256), 0, s, a);
}

struct DecodePlan {
  int head_items, item_heads, grid;
  int64_t most_tiles;  // of an item
};

// The launch of a call; its workspace goes by the same numbers.
inline DecodePlan decode_plan(const fpv2_decode_params& p) {
  DecodePlan plan;
  const int64_t group = p.query_heads / p.kv_heads;
  plan.head_items = static_cast<int>((group + kMaxHeads - 1) / kMaxHeads);
  plan.item_heads = static_cast<int>((group + plan.head_items - 1) / plan.head_items);
  int64_t keys = p.table_width * p.page_size;
  if (p.window_tokens > 0 && p.window_tokens < keys && p.sink_tokens < keys - p.window_tokens)
    keys = p.window_tokens + p.sink_tokens;
  plan.most_tiles = (keys + kTileKeys - 1) / kTileKeys;
  if (plan.most_tiles < 1) plan.most_tiles = 1;
  const int64_t units = p.batch * p.kv_heads * plan.head_items * (plan.most_tiles + kItemUnits);
  const int64_t runs = (units + kWaves - 1) / kWaves, most = 2 * static_cast<int64_t>(cu_count());
  plan.grid = static_cast<int>(runs < most ? runs : most < kMaxGrid ? most : kMaxGrid);
  return plan;
}

inline int check_params(const char* name, const fpv2_decode_params* p) {
  if (p == nullptr) return fail(FPV2_ERR_ARGUMENT, "%s: null params", name);
  if (p->batch < 0 || p->query_heads <= 0 || p->kv_heads <= 0 || p->query_heads % p->kv_heads)
    return fail(FPV2_ERR_ARGUMENT, "%s: query heads must be divisible by KV heads", name);
  if (p->head_dim != 64 && p->head_dim != 96 && p->head_dim != 128 && p->head_dim != 256)
    return fail(FPV2_ERR_UNSUPPORTED, "%s: head_dim must be 64, 96, 128 or 256", name);
  if (p->batch > 0xffff || p->query_heads > 0xffff)
    return fail(FPV2_ERR_UNSUPPORTED, "%s: more than 65535 sequences or query heads", name);
  if (p->pages <= 0 || p->page_size <= 0 || p->table_width <= 0 || p->pages > 0x7fffffff ||
      p->page_size > 0x3fffffff || p->table_width > 0x3fffffff ||
      p->table_width * p->page_size > 0x3fffffff)
    return fail(FPV2_ERR_ARGUMENT, "%s: pages, page_size and table_width must be positive and a "
                "sequence's pages hold fewer than 2^30 tokens", name);
  if (p->window_tokens < 0 || p->sink_tokens < 0 || p->length < 0)
    return fail(FPV2_ERR_ARGUMENT, "%s: length, window_tokens and sink_tokens must not be negative", name);
  const int64_t group = p->query_heads / p->kv_heads;
  const int64_t items = p->batch * p->kv_heads * ((group + kMaxHeads - 1) / kMaxHeads);
  if (items * kMaxHeads > 0x7fffffff ||
      items * ((p->table_width * p->page_size + kTileKeys - 1) / kTileKeys + kItemUnits) > 0x3fffffff)
    return fail(FPV2_ERR_UNSUPPORTED, "%s: the call has too many tiles of keys", name);
  return FPV2_OK;
}

inline int64_t partial_bytes(const fpv2_decode_params& p, const DecodePlan& plan) {
  if (p.batch == 0 || plan.most_tiles <= 1) return 0;  // every item has one workgroup
  return 2LL * plan.grid * plan.item_heads * (p.head_dim + 2) * 4;
}

// The launch's arguments but for the pointers.
inline DecodeArgs decode_args(const fpv2_decode_params& p, const DecodePlan& plan) {
  DecodeArgs a{};
  a.q_bs = p.q_batch_stride;
  a.q_hs = p.q_head_stride;
  a.k_ps = p.k_page_stride;
  a.k_hs = p.k_head_stride;
  a.k_rs = p.k_row_stride;
  a.v_ps = p.v_page_stride;
  a.v_hs = p.v_head_stride;
  a.v_rs = p.v_row_stride;
  a.o_bs = p.o_batch_stride;
  a.o_hs = p.o_head_stride;
  a.table_stride = p.table_stride;
  a.batch = static_cast<int>(p.batch);
  a.kv_heads = static_cast<int>(p.kv_heads);
  a.group = static_cast<int>(p.query_heads / p.kv_heads);
  a.head_items = plan.head_items;
  a.item_heads = plan.item_heads;
  a.pages = static_cast<int>(p.pages);
  a.page_size = static_cast<int>(p.page_size);
  a.capacity = static_cast<int>(p.table_width * p.page_size);
  a.length = static_cast<int>(p.length < a.capacity ? p.length : a.capacity);
  a.window = static_cast<int>(p.window_tokens > 0 && p.window_tokens < a.capacity ? p.window_tokens
                                                                                  : a.capacity);
  a.sinks = static_cast<int>(p.sink_tokens < a.capacity ? p.sink_tokens : a.capacity);
  a.grid = plan.grid;
  a.join_runs = p.batch * p.kv_heads * plan.head_items > plan.grid;
  page_division(p.page_size, &a.page_mul, &a.page_shift);
  a.scale_log2 = static_cast<float>(p.scale * 1.4426950408889634);
  return a;
}

}  // namespace
}  // namespace fpv2
