// Attention of one new token per sequence of a batch that shares a prefix: the
// prefix's keys once for all sequences, each sequence's own keys, and the join.
//
//   out[b][h] = sum_t p_t v_t / sum_t p_t,  p_t = exp(scale q[b][h].k_t - max),
//   t over the prefix and over b's own keys
//
// The sums split over t: partials (O, max, sum) of parts of the keys are joined as
//   O = sum_i exp(m_i - m) O_i, l = sum_i exp(m_i - m) l_i, m = max_i m_i.
// Two launches: workgroups of the own keys and of the prefix, then the join.
//
// Prefix: the rows of a KV head are the batch's query heads of it, packed; a workgroup
// takes a tile of them and a part of the prefix's keys, on MFMA: S^T = K Q^T and O^T += V^T P^T,
// so that a lane's scores are its operand of the second product as they are.  Up to 16 rows
// are one tile of MFMA and the reads of the keys bound it: its waves take 32 keys each straight
// from memory, as the decode attention does.  Of more rows each key serves several waves, which
// share it through LDS; MFMA, the exponentials beside it and the partials bound that.
//
// Measured (32 / 8 heads, D = 128; caches that change from call to call): 40 sequences of 20 to 700 own
// keys after 32768 in pages of 64, bfloat16, 58 us + the join's 8; 128 of 5 to 300 after 8191, float16,
// 44 + 10; 64 of up to 32 after 32768 61 + 10.5; 16 / 4 heads of D = 256, 21 of 9 to 1500 after 20011, 40 + 8.
// Up to 16 rows 4 sequences after 32768 keys 34 + 8, one after 131072 93 + 7.5 (5.7 TB/s); 16 / 4 heads of
// D = 256, 4 of 30 after 32768 43 for both.  A launch takes
// some 5 us of these, and each MB of partials (10 to 33 of them) half a microsecond.
// Without gain: workgroups of 8 waves in two groups of keys that join in LDS (half the partials,
// but a barrier of 8 waves in each step), partials past the caches (1.5 us less here, 1.5 more in
// the join).
#include "fpv2_batch.h"
#include "fpv2_decode_split.h"

namespace fpv2 {
namespace {

// What a tile of own keys costs a wave beside what one of the prefix, of more than 16 rows, costs
// each wave of its workgroup: measured best of 1 to 8, at head dim 256 (kOwnWide) of 1 to 20 by one batch, 21
// sequences of 9 to 1500 after 20011 keys.
constexpr float kOwnTile = 2.f, kOwnWide = 8.f;
constexpr int kLong = 24, kCoarse = 8;

struct PrefixArgs {
  const uint16_t* q;
  const uint16_t* k;
  const uint16_t* v;
  const int32_t* table;
  const int32_t* lengths;  // of one
  float* part_o;           // [splits][kv_heads][rows][D]
  float* part_ml;          // [splits][kv_heads][rows][2]
  int32_t* units;          // [64]: the own keys' Prefix, for the join
  int64_t q_bs, q_hs, k_ps, k_hs, k_rs, v_ps, v_hs, v_rs;
  int kv_heads, group, rows, row_tiles, tile_rows;  // rows: batch * group
  int cus, roomy, most_splits, most_own;  // most_own: workgroups of the own keys
  int pages, page_size, capacity, length;
  uint32_t page_mul, page_shift;
  float scale_log2;
};

// The launch's first argument, read again: what the workgroups' two kinds of work, and their starts
// and ends, hold of their arguments would not fit the scalar registers together, and the loop over the keys
// would fetch the rest of it from lanes of vector registers.
typedef const __attribute__((address_space(4))) PrefixArgs ScalarArgs;
__device__ __forceinline__ ScalarArgs& again() {
  uintptr_t p = reinterpret_cast<uintptr_t>(__builtin_amdgcn_kernarg_segment_ptr());
  asm volatile("" : "+s"(p));
  return *reinterpret_cast<ScalarArgs*>(p);
}

__device__ __forceinline__ int prefix_length(const PrefixArgs& a) {
  const int n = a.lengths != nullptr ? *a.lengths : a.length;
  return min(max(n, 0), a.capacity);
}

// What the launch's workgroups do: the first own_blocks the own keys, by waves; then the parts
// of the prefix.
struct Division {
  int own_blocks, splits;
};
// The waves of a workgroup.
template <int D>
__host__ __device__ __forceinline__ int waves_of(int64_t rows) { return D > 128 && rows > 16 ? 8 : 4; }

// The workgroups that run at once are shared out by the work, which the lengths on the device say,
// so that both kinds take equally long, side by side: the own keys wait for memory, the prefix for
// MFMA, and no workgroup waits for another's place.  Against the own keys first, in as many waves as
// they have tiles for, and then the prefix: 40 sequences after 32768 keys 66 to 58 us, 128 after 8191
// 50 to 44, 8 after 16384 31 to 23, 64 of up to 2000 after 4096 37 to 33.
// - A few own keys (a 32nd of the work and less) before many of the prefix (kLong tiles a workgroup)
//   come first all the same: to round the parts down to what they leave costs more (64 sequences after
//   32768 keys 65 us beside, 61 before; 8 after 16384, 8 tiles a workgroup, 23 and 31).  So they do where
//   a part has an 8th of the workgroups and more (kCoarse) and that takes longer by the tiles of a
//   workgroup (512 sequences after 4096 keys 75 beside, 66 before).
// - The prefix has a second workgroup on a CU where each of one has more than 8 tiles of more than 16
//   rows (31 sequences after 8192 keys, 8 tiles: 20 us by one, 21 by two and the join 7 and 10;
//   64 after 8192, 16 tiles: 31 and 26).
// - Where all that the caches can hold has room at once (roomy), the prefix's workgroups need not
//   know the own keys' lengths: 4 sequences after 1000 keys 1 us less.
// n: the prefix's length; units: of all own items, 8 of each item's beside its tiles (counted as 2
// here).  (Nothing to contract in it: both launches divide alike.)
template <int D>
__device__ __forceinline__ Division divide(const PrefixArgs& p, const DecodeArgs& a, int n, int units) {
#pragma clang fp contract(off)
  const bool few = p.rows <= 16;
  const int tiles = (n + kTileKeys - 1) / kTileKeys, waves = waves_of<D>(p.rows);
  const int each = p.kv_heads * p.row_tiles;  // workgroups of a part
  const int most = max(min((tiles + kWaves - 1) / kWaves, p.most_splits), 1);
  if (p.roomy) return {p.most_own, most};
  const float all = static_cast<float>(tiles) * static_cast<float>(each);
  const int slots = D <= 128 ? 2 * p.cus : p.cus;
  const int mine = units - (kItemUnits - 2) * a.batch * a.kv_heads * a.head_items;
  const float own = static_cast<float>(mine) * (few ? 1.f : D > 128 ? kOwnWide : kOwnTile);
  const float pre = few ? all : all * static_cast<float>(waves);
  // (the parts that then follow on them take all workgroups)
  const int share = min(static_cast<int>(static_cast<float>(slots) * pre * __builtin_amdgcn_rcpf(own + pre)),
                        few || all <= static_cast<float>(8 * p.cus) ? min(p.cus, slots - 8) : slots - 8);
  // (half a workgroup off a whole number: the quotient's floor)
  const int quotient = static_cast<int>((static_cast<float>(share) + 0.5f) *
                                        __builtin_amdgcn_rcpf(static_cast<float>(each)));
  const int splits = min(max(quotient, 1), most);
  const int need = ((units / kWaves + waves) / waves + 7) / 8 * 8;
  const int blocks = min(max(slots - splits * each, slots - share) / 8 * 8, need);
  bool before = !few && D <= 128 && all >= static_cast<float>(kLong * slots) && 32.f * mine < pre;
  if (!few && kCoarse * each >= slots) {
    const float beside = fmaxf(static_cast<float>(tiles) * __builtin_amdgcn_rcpf(static_cast<float>(splits)),
                               own * __builtin_amdgcn_rcpf(static_cast<float>(blocks * waves)));
    const float turns = static_cast<float>(tiles) * __builtin_amdgcn_rcpf(static_cast<float>(most));
    before = before || turns + own * __builtin_amdgcn_rcpf(static_cast<float>(slots * waves)) + 2.f < beside;
  }
  if (before) return {__builtin_amdgcn_readfirstlane(min(need, p.most_own)), __builtin_amdgcn_readfirstlane(most)};
  // (known to be the wave's, and all that follows from them)
  return {__builtin_amdgcn_readfirstlane(min(blocks, p.most_own)), __builtin_amdgcn_readfirstlane(splits)};
}

// A column's weights are 2^(x - m), x = scale log2(e) q.k, with a reference m that moves when
// it has to, so that most tiles rescale nothing.
//   bfloat16: where a weight exceeds 1, to 2^-kLag of the greatest score (not above 1: sums of values
// next to the type's greatest would leave float32).
//   float16, which has only 2^-14 to 2^16: where a weight would exceed 2^kMost or the
// tile's greatest is below 2^kLeast, to 2^-12 of the tile's greatest score (or 2^-40 of the
// greatest so far, so that no float32 sum overflows).  So weights down to 2^-19 of their
// tile's greatest keep their bits, whatever lies above that tile, and smaller ones are off by
// 2^-30 of it.  (2^-15 instead of 2^-12: most tiles have a column that exceeds it, 128
// sequences of an 8191-key prefix 41 us instead of 38.)
constexpr float kLag = 8.f, kMost = 15.9f, kLeast = 5.f, kHeadroom = 12.f, kBelow = 40.f;
constexpr float kNone = -3.4028234663852886e38f;  // the reference before any score: no finite one is below

// A tile's exponents of 16 rows from its scores (of 32 keys the ones before `live`, counted
// from the lane's first); O, l and m of the rows are moved where they have to be.
struct Exponents {
  float y[8];
};
template <typename T, int DT>
__device__ __forceinline__ Exponents relate(const f32x4 (&sc)[2], float scale, int live, float& m, float& l,
                                            float& greatest, f32x4 (&o)[DT]) {
  constexpr bool kHalf = std::is_same<T, f16_t>::value;
  const bool cut = live < 32;
  Exponents e;
  float top = neg_inf();
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    e.y[j] = __builtin_fmaf(sc[j / 4][j % 4], scale, -m);
    if (cut && 16 * (j / 4) + j % 4 >= live) e.y[j] = neg_inf();
    top = fmaxf(top, e.y[j]);
  }
  bool move;
  if constexpr (kHalf) {
    const uint64_t some = __ballot(top >= kLeast);
    const uint32_t any = static_cast<uint32_t>(some) | static_cast<uint32_t>(some >> 32);
    move = ((any | any >> 16) & 0xffffu) != 0xffffu || __any(top > kMost);
  } else {
    move = __any(top > 0.f);
  }
  if (move) {
    top = neg_inf();
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      e.y[j] = sc[j / 4][j % 4] * scale;
      if (cut && 16 * (j / 4) + j % 4 >= live) e.y[j] = neg_inf();
      top = fmaxf(top, e.y[j]);
    }
    top = column_max(top);
    float to = m;
    if constexpr (kHalf) {
      greatest = fmaxf(greatest, top);
      // (by their difference, which is what the weight will be: a sum of m may round to 2^16's)
      if ((top - m > kMost || top - m < kLeast) && greatest > neg_inf())
        to = below(fmaxf(top, greatest - kBelow), kHeadroom);
    } else {
      to = top > m ? top + kLag : m;
    }
    const float fix = __builtin_amdgcn_exp2f(m - to);
    m = to;
    l *= fix;
#pragma unroll
    for (int d = 0; d < DT; ++d) o[d] *= fix;
#pragma unroll
    for (int j = 0; j < 8; ++j) e.y[j] -= to;
  }
  return e;
}
// Their weights, as the B operand of the product with V, and l's share.  MFMA takes both of one type, so they are
// rounded to V's: half a step of each, which together is about as much as the result's own rounding (against
// float64 0.0023 of the result in bfloat16, 0.0017 of it the result's); l is the sum of the unrounded ones.
template <typename T>
__device__ __forceinline__ u32x4 weigh(const Exponents& e, float& l) {
  u32x4 pf;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float a = __builtin_amdgcn_exp2f(e.y[2 * j]), b = __builtin_amdgcn_exp2f(e.y[2 * j + 1]);
    pf[j] = pack2<T>(a, b);
    l += a + b;
  }
  return pf;
}

// A page of the prefix (as the table has it) and a row in it.  In scalar registers where t
// is: a vector load would have to wait for all that were issued before it.
struct At {
  int id, row;
};
__device__ const int32_t kPageZero = 0;
__device__ __forceinline__ At prefix_at(ScalarArgs& a, int t) {
  typedef const __attribute__((address_space(4))) int32_t* scalar_ptr;
  const uint32_t page = (__umulhi(static_cast<uint32_t>(t), a.page_mul) + t) >> a.page_shift;
  const int32_t* p = a.table != nullptr ? a.table + page : &kPageZero;
  return {*reinterpret_cast<scalar_ptr>(reinterpret_cast<uintptr_t>(p)), t - static_cast<int>(page) * a.page_size};
}
__device__ __forceinline__ int64_t page_of(ScalarArgs& a, int id) { return min(max(id, 0), a.pages - 1); }
// Loads stay in the order that they are written in.
__device__ __forceinline__ void in_order() { asm volatile("" ::: "memory"); }

// A row's queries as the B operand of the scores, negated where the scale is negative.
template <int KK>
__device__ __forceinline__ void load_queries(ScalarArgs& a, int kvh, int row, bool live, int quad, u32x4 (&qf)[KK]) {
  const int b = row / a.group, g = row - b * a.group;
  const uint16_t* p = a.q + b * a.q_bs + (kvh * a.group + g) * a.q_hs + 8 * quad;
  const uint32_t sign = a.scale_log2 < 0.f ? 0x80008000u : 0u;
#pragma unroll
  for (int kk = 0; kk < KK; ++kk) qf[kk] = live ? load16(p + 32 * kk) ^ sign : u32x4{0, 0, 0, 0};
}

// A wave's 32 keys: K as the A operands of the scores, V as 8 rows' dims of a lane.
template <int D>
struct Tile {
  u32x4 k[2][D / 32];
  Words<D / 32> v[8];
};

// A KV head's keys of one table, tile after tile.
struct Keys {
  const uint16_t* k;
  const uint16_t* v;
  const int32_t* table;
  int64_t k_ps, k_rs, v_ps, v_rs;
  int page, pages, page_size, n;  // page: of all keys where there is no table
  uint32_t page_mul, page_shift;
};
// 16 rows' sums over a wave's keys: the tiles at u0, u0 + STEP .. before u_end.  AHEAD: with a tile's
// loads on their way beside another's products (own keys, of a few tiles each, take as long
// without, whose K and V share registers).
template <int D>
struct Rows {
  u32x4 q[D / 32];
  f32x4 o[D / 16];
  float scale, m, l, greatest;
};
template <int D>
__device__ __forceinline__ void start_rows(Rows<D>& r, float scale_log2) {
  r.scale = __builtin_fabsf(scale_log2);
  r.m = kNone;
  r.l = 0.f;
  r.greatest = neg_inf();
#pragma unroll
  for (int d = 0; d < D / 16; ++d) r.o[d] = f32x4{0.f, 0.f, 0.f, 0.f};
}
template <typename T, int D, int STEP, bool AHEAD>
__device__ __forceinline__ void walk(const Keys& a, int u0, int u_end, int lane, Rows<D>& r) {
  constexpr int KK = D / 32, DV = D / 16;
  const int col = lane & 15, quad = lane >> 4;
  int row = 0, page = 0;  // lane i's (and i + 32's) of the next tile's key i
  const auto look_up = [&](int u) {
    const uint32_t t = min(u + (lane & 31), a.n - 1);
    const uint32_t at = (__umulhi(t, a.page_mul) + t) >> a.page_shift;
    row = t - at * a.page_size;
    const int id = a.table != nullptr ? a.table[at] : a.page;
    page = min(max(id, 0), a.pages - 1);
  };
  const auto load_k = [&](Tile<D>& x) {
    const int64_t koff = page * a.k_ps + row * a.k_rs;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const uint16_t* p = a.k + __shfl(koff, 16 * t + col, 64) + 8 * quad;
#pragma unroll
      for (int kk = 0; kk < KK; ++kk) x.k[t][kk] = load16(p + 32 * kk);
    }
  };
  const auto load_v = [&](Tile<D>& x, int64_t voff) {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      x.v[j] = load_words<DV / 2>(a.v + __shfl(voff, 16 * (j / 4) + 4 * quad + j % 4, 64) + DV * col);
  };
  const auto score = [&](const Tile<D>& y, f32x4 (&sc)[2]) {
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      sc[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int kk = 0; kk < KK; ++kk) sc[t] = Elem<T>::mfma16(as_vec8<T>(y.k[t][kk]), as_vec8<T>(r.q[kk]), sc[t]);
    }
  };
  const auto multiply = [&](Tile<D>& y, const f32x4 (&sc)[2], int u) {
    const int left = a.n - u;
    const u32x4 pf = weigh<T>(
        relate<T>(sc, r.scale, left < kTileKeys ? left - 4 * quad : kTileKeys, r.m, r.l, r.greatest, r.o), r.l);
    if (left < kTileKeys) {
      // (a zero weight would make NaN of what an unused row may hold)
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (16 * (j / 4) + 4 * quad + j % 4 >= left) {
#pragma unroll
          for (int w = 0; w < DV / 2; ++w) y.v[j].w[w] = 0;
        }
    }
#pragma unroll
    for (int d = 0; d < DV; ++d) {
      u32x4 vt;  // dim d of the lane's 8 keys
#pragma unroll
      for (int j = 0; j < 4; ++j)
        vt[j] = __builtin_amdgcn_perm(y.v[2 * j + 1].w[d / 2], y.v[2 * j].w[d / 2],
                                      d % 2 ? 0x07060302u : 0x05040100u);
      r.o[d] = Elem<T>::mfma16(as_vec8<T>(vt), as_vec8<T>(pf), r.o[d]);
    }
  };
  if (u0 >= u_end) return;
  look_up(u0);
  if constexpr (AHEAD) {
    // A tile's loads are a tile ahead of its products, and its pages one more.  (Tiles behind
    // the last one are loaded too, as the last key again, so that it is known at each product
    // how many loads were issued since its own.)
    Tile<D> even, odd;
    const auto load = [&](Tile<D>& x, int next) {
      load_k(x);
      load_v(x, page * a.v_ps + row * a.v_rs);
      look_up(next);
    };
    const auto both = [&](Tile<D>& x, int u) {
      f32x4 sc[2];
      score(x, sc);
      multiply(x, sc, u);
    };
    load(even, u0 + STEP);
    for (; u0 < u_end; u0 += 2 * STEP) {
      load(odd, u0 + 2 * STEP);
      both(even, u0);
      load(even, u0 + 3 * STEP);
      if (u0 + STEP < u_end) both(odd, u0 + STEP);
    }
  } else {
    for (; u0 < u_end; u0 += STEP) {
      Tile<D> x;
      load_k(x);
      const int64_t voff = page * a.v_ps + row * a.v_rs;
      look_up(u0 + STEP);
      f32x4 sc[2];
      score(x, sc);
      load_v(x, voff);
      multiply(x, sc, u0);
    }
  }
}

// Own keys: the decode attention's schedule (fpv2_decode_split.h) with runs of waves instead of
// workgroups, as they are short: a wave takes its items' tiles one after the other and
// leaves a partial of each, a whole item's behind the runs' slots.
template <typename T, int D>
__device__ __forceinline__ void own_attn(const DecodeArgs& a, const Prefix& prefix, int run, int whole_slots) {
  constexpr int DV = D / 16;
  const int lane = threadIdx.x & 63, col = lane & 15, quad = lane >> 4;
  const int items = a.kv_heads * a.head_items;
  const int total = prefix.total * items;
  const int lo = first_of(a, run, total), hi = first_of(a, run + 1, total);
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
    Rows<D> r;
    const uint32_t sign = a.scale_log2 < 0.f ? 0x80008000u : 0u;
#pragma unroll
    for (int kk = 0; kk < D / 32; ++kk)
      r.q[kk] = col < heads ? load16(a.q + b_now * a.q_bs + head * a.q_hs + 32 * kk + 8 * quad) ^ sign
                            : u32x4{0, 0, 0, 0};
    start_rows(r, a.scale_log2);
    walk<T, D, kTileKeys, false>(
        {a.k + kvh * a.k_hs, a.v + kvh * a.v_hs, a.table != nullptr ? a.table + b_now * a.table_stride : nullptr,
         a.k_ps, a.k_rs, a.v_ps, a.v_rs, b_now, a.pages, a.page_size, s_now.n, a.page_mul, a.page_shift},
        first * kTileKeys, min(s_now.n, last * kTileKeys), lane, r);
    r.l += __shfl_xor(r.l, 16, 64);
    r.l += __shfl_xor(r.l, 32, 64);
    const bool whole = first == 0 && last == s_now.tiles;
    const int64_t slot = whole ? whole_slots + static_cast<int64_t>(b_now) * items + item
                               : 2 * static_cast<int64_t>(run) + (cur == lo ? 0 : 1);
    if (col < heads) {
      const int64_t at = slot * a.item_heads + col;
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int d = 0; d < DV; ++d) a.part_o[at * D + (4 * quad + i) * DV + d] = r.o[d][i];
      if (quad == 0) {
        a.part_ml[at * 2] = r.m;
        a.part_ml[at * 2 + 1] = r.l;
      }
    }
  }
}

// At most 16 rows: one tile of MFMA; the workgroup's waves take 32 keys each, as they lie.
template <int D>
struct FewShared {
  float o[4][16][D + 4];
  float ml[4][16][2];
};
template <typename T, int D>
__device__ __forceinline__ void prefix_few(ScalarArgs& a, int n, int splits, int unit, FewShared<D>& sh) {
  constexpr int DV = D / 16;
  auto& sh_o = sh.o;
  auto& sh_ml = sh.ml;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 15, quad = lane >> 4;
  if (unit >= a.kv_heads * splits) return;
  const int split = unit / a.kv_heads, kvh = unit - split * a.kv_heads;
  const int tiles = (n + kTileKeys - 1) / kTileKeys;
  const int per = tiles / splits, more = tiles - per * splits;
  const int first = split * per + min(split, more), last = first + per + (split < more ? 1 : 0);
  Rows<D> r;
  load_queries<D / 32>(a, kvh, col, col < a.rows, quad, r.q);
  start_rows(r, a.scale_log2);
  walk<T, D, kStepKeys, true>({a.k + kvh * a.k_hs, a.v + kvh * a.v_hs, a.table, a.k_ps, a.k_rs, a.v_ps, a.v_rs, 0,
                               a.pages, a.page_size, n, a.page_mul, a.page_shift},
                              (first + wave) * kTileKeys, min(n, last * kTileKeys), lane, r);

  // join the four waves
  r.l += __shfl_xor(r.l, 16, 64);
  r.l += __shfl_xor(r.l, 32, 64);
  if (quad == 0) {
    sh_ml[wave][col][0] = r.m;
    sh_ml[wave][col][1] = r.l;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int d = 0; d < DV; ++d) sh_o[wave][col][(4 * quad + i) * DV + d] = r.o[d][i];
  __syncthreads();
  for (int e = tid; e < a.rows * D; e += 256) {
    const int h = e / D, d = e % D;
    float top = neg_inf();
#pragma unroll
    for (int w = 0; w < 4; ++w) top = fmaxf(top, sh_ml[w][h][0]);
    float sum = 0.f, den = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      // (a wave without keys has sum 0 and O 0)
      const float f = __builtin_amdgcn_exp2f(sh_ml[w][h][0] - top);
      sum += f * sh_o[w][h][d];
      den += f * sh_ml[w][h][1];
    }
    const int64_t at = static_cast<int64_t>(unit) * a.rows + h;
    a.part_o[at * D + d] = sum;
    if (d == 0) {
      a.part_ml[at * 2] = top;
      a.part_ml[at * 2 + 1] = den;
    }
  }
}

template <typename T, int D>
__global__ __launch_bounds__(256, D > 128 ? 1 : 2) void prefix_few_kernel(PrefixArgs p, DecodeArgs a) {
  __shared__ FewShared<D> sh;
  const int n = __builtin_amdgcn_readfirstlane(prefix_length(p));
  Prefix prefix = {};
  if (!p.roomy || static_cast<int>(blockIdx.x) < p.most_own) prefix = prefix_of(a, threadIdx.x & 63);
  const Division by = divide<D>(p, a, n, prefix.total * a.kv_heads * a.head_items);
  a.grid = 4 * by.own_blocks;
  if (blockIdx.x == 0 && threadIdx.x < 64) p.units[threadIdx.x] = prefix.upto;
  const int block = static_cast<int>(blockIdx.x) - by.own_blocks;
  if (block < 0)
    own_attn<T, D>(a, prefix, blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), 8 * p.most_own);
  else
    prefix_few<T, D>(again(), n, by.splits, block, sh);
}

// More rows than a tile of MFMA: the workgroup's waves, 32 rows each (at head dim 256, whose
// rows are twice as long, 8 waves of 16 rows), share the keys through LDS.  A stage is 32
// keys' K and V, rows of a power of two of bytes whose 16-byte chunks are permuted so that
// neither the reads of K (16 keys' chunks) nor the transposing reads of V (8 keys, 32 bytes
// each) meet in a bank.  Three stages in LDS, three more on their way in registers.  Each wave
// loads some keys' K or V: one page, one descriptor a stage.
template <int D>
struct Stage {
  static constexpr int kRow = D <= 64 ? 128 : D <= 128 ? 256 : 512;  // bytes of a row in LDS
  static constexpr int kMatrix = kTileKeys * kRow;
  static constexpr int kChunks = D / 8;             // 16-byte chunks of a row
  static constexpr int kWaves = D > 128 ? 8 : 4;
  static constexpr int kTiles = D > 128 ? 1 : 2;    // 16-row tiles of a wave
  static constexpr int kKeys = 2 * kTileKeys / kWaves;    // of a wave's loads
  static constexpr int kLoads = kKeys * kChunks / 64;     // of a lane
  static __device__ __forceinline__ int k_mask(int row) { return kRow >= 256 ? row & 15 : row >> 1 & 7; }
  static __device__ __forceinline__ int v_mask(int row) { return (kRow >= 256 ? row & 7 : row >> 1 & 3) << 1; }
};
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

// A barrier for what ds_write wrote: it waits for this wave's LDS operations only, not for
// its loads from memory (as __syncthreads() does).
__device__ __forceinline__ void barrier_lds() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// HALVES: 16 keys from a multiple of 16 on lie in one page (or there is no table): their
// addresses are the wave's, a lane's offsets do not change, and a descriptor of the rows
// up to the prefix's end reads zeros behind it.  128 sequences of 16 own keys, 8192 of the prefix:
// 37.3 us, with each lane's own page and row 42.6; 40 sequences, 32768 in pages of 64: 52 and 77.  (Up to
// 16 rows the same either way, so that form has the lanes' own alone.)
template <typename T, int D, bool HALVES>
__device__ __forceinline__ void prefix_many(ScalarArgs& a, int n, int splits, int block, uint8_t (&sh)[3][2 * Stage<D>::kMatrix]) {
  using S = Stage<D>;
  constexpr int KK = D / 32, DT = D / 16, CT = S::kTiles, L = S::kLoads, R = 3;  // stages
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 15, quad = lane >> 4;
  // A unit is a part of a KV head's keys; its row tiles' workgroups are 8 apart, so
  // that they share an XCD's L2.
  const int unit = block % 8 + 8 * (block / (8 * a.row_tiles));
  const int rt = block / 8 % a.row_tiles;
  if (unit >= a.kv_heads * splits) return;
  const int split = unit / a.kv_heads, kvh = unit - split * a.kv_heads;
  const int tiles = (n + kTileKeys - 1) / kTileKeys;
  const int per = tiles / splits, more = tiles - per * splits;
  const int first = split * per + min(split, more), last = first + per + (split < more ? 1 : 0);
  const int steps = last - first;
  const auto tile_of = [&](int step) { return first + step; };
  const int r0 = rt * a.tile_rows + 16 * CT * wave;  // this wave's rows
  const int r_end = min(a.rows, (rt + 1) * a.tile_rows);

  // this wave's loads: some keys' K or V of a stage, chunk lane + 64 i of their rows
  const bool is_v = wave >= S::kWaves / 2;
  const int key0 = S::kKeys * (wave % (S::kWaves / 2));
  const uint16_t* const base = is_v ? a.v + kvh * a.v_hs : a.k + kvh * a.k_hs;
  const int64_t ps = is_v ? a.v_ps : a.k_ps, rs = is_v ? a.v_rs : a.k_rs;
  int key[L], part[L];
  uint32_t from[L], to[L];
#pragma unroll
  for (int i = 0; i < L; ++i) {
    const int c = lane + 64 * i;
    key[i] = c / S::kChunks;
    part[i] = c - key[i] * S::kChunks;
    from[i] = (key[i] * static_cast<uint32_t>(rs) + 8 * part[i]) * 2;
    const int row = key0 + key[i];
    to[i] = (is_v ? S::kMatrix : 0) + row * S::kRow + (part[i] ^ (is_v ? S::v_mask(row) : S::k_mask(row))) * 16;
  }
  At here;           // HALVES: of a coming stage's keys
  At there[L];       // else: of the lane's loads
  const auto look_up = [&](int tile) __attribute__((always_inline)) {
    const int u0 = tile * kTileKeys + key0;
    if constexpr (HALVES) {
      here = prefix_at(a, u0 < n ? u0 : 0);
    } else {
#pragma unroll
      for (int i = 0; i < L; ++i) {
        const uint32_t t = min(u0 + key[i], n - 1);
        const uint32_t page = (__umulhi(t, a.page_mul) + t) >> a.page_shift;
        there[i] = {a.table != nullptr ? a.table[page] : 0, static_cast<int>(t - page * a.page_size)};
      }
    }
  };
  struct Regs {
    u32x4 x[L];
  };
  const auto load = [&](Regs& r, int tile) __attribute__((always_inline)) {
    if constexpr (HALVES) {
      const int live = min(n - tile * kTileKeys - key0, S::kKeys);  // (0 and less: zeros)
      const rsrc_t src = make_rsrc(base + page_of(a, here.id) * ps + here.row * rs,
                                   live > 0 ? ((live - 1) * static_cast<int>(rs) + D) * 2 : 0);
#pragma unroll
      for (int i = 0; i < L; ++i) r.x[i] = buf_load16(src, from[i]);
    } else {
#pragma unroll
      for (int i = 0; i < L; ++i)
        r.x[i] = load16(base + page_of(a, there[i].id) * ps + there[i].row * rs + 8 * part[i]);
    }
    in_order();
  };
  const auto store = [&](const Regs& r, int tile, auto buffer) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < L; ++i) {
      // (a zero weight would make NaN of what an unused row may hold)
      const bool live = HALVES || tile * kTileKeys + key0 + key[i] < n;
      store16(&sh[decltype(buffer)::value][to[i]], live ? r.x[i] : u32x4{0, 0, 0, 0});
    }
  };

  const float scale = __builtin_fabsf(a.scale_log2);
  u32x4 qf[CT][KK];
  f32x4 o[CT][DT];
  float m[CT], l[CT], greatest[CT];
#pragma unroll
  for (int c = 0; c < CT; ++c) {
    load_queries<KK>(a, kvh, r0 + 16 * c + col, r0 + 16 * c + col < r_end, quad, qf[c]);
    m[c] = kNone;
    greatest[c] = neg_inf();
    l[c] = 0.f;
#pragma unroll
    for (int d = 0; d < DT; ++d) o[c][d] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  // this lane's reads: of K row col's chunks, of V 8 bytes of row 4 quad + col / 4 (16 rows on
  // the masks are the same)
  const int v_row = 4 * quad + col / 4;
  uint32_t k_at[KK], v_at[DT];
#pragma unroll
  for (int kk = 0; kk < KK; ++kk) k_at[kk] = col * S::kRow + ((4 * kk + quad) ^ S::k_mask(col)) * 16;
#pragma unroll
  for (int d = 0; d < DT; ++d)
    v_at[d] = lds_addr(&sh[0][0]) + S::kMatrix + v_row * S::kRow + ((2 * d + (col % 4) / 2) ^ S::v_mask(v_row)) * 16 + col % 2 * 8;

  f32x4 sc[CT][2];  // a tile's scores
  const auto score = [&](auto buffer) __attribute__((always_inline)) {
#pragma unroll
    for (int t = 0; t < 2; ++t) {
#pragma unroll
      for (int c = 0; c < CT; ++c) sc[c][t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int kk = 0; kk < KK; ++kk) {
        const u32x4 kf = load16(&sh[decltype(buffer)::value][16 * t * S::kRow + k_at[kk]]);
#pragma unroll
        for (int c = 0; c < CT; ++c) sc[c][t] = Elem<T>::mfma16(as_vec8<T>(kf), as_vec8<T>(qf[c][kk]), sc[c][t]);
      }
    }
  };
  // A tile's weights and their product with V beside the scores of the next one: matrix
  // instructions of the one while the other's exponentials are computed.
  const auto multiply = [&](int tile, auto buffer, auto next) __attribute__((always_inline)) {
    const int left = n - tile * kTileKeys;
    Exponents e[CT];
#pragma unroll
    for (int c = 0; c < CT; ++c)
      e[c] = relate<T>(sc[c], scale, left < kTileKeys ? left - 4 * quad : kTileKeys, m[c], l[c], greatest[c], o[c]);
    score(next);
    u32x4 pf[CT];
#pragma unroll
    for (int c = 0; c < CT; ++c) pf[c] = weigh<T>(e[c], l[c]);
#pragma unroll
    for (int d = 0; d < DT; ++d) {
      u32x4 vt;  // dim d of the lane's 8 keys
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const s16x4 w = __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<lds_s16x4*>(
            static_cast<uintptr_t>(v_at[d] + decltype(buffer)::value * 2 * S::kMatrix + 16 * t * S::kRow)));
        const u32x2 words = __builtin_bit_cast(u32x2, w);
        vt[2 * t] = words[0];
        vt[2 * t + 1] = words[1];
      }
#pragma unroll
      for (int c = 0; c < CT; ++c) o[c][d] = Elem<T>::mfma16(as_vec8<T>(vt), as_vec8<T>(pf[c]), o[c][d]);
    }
  };

  // (Stages behind the last one are loaded too, HALVES: as zeros, else the last key again; so
  // that it is known at each store how many loads were issued since its own.)
  if (first < last) {
    const bool rows_here = r0 < r_end;
    Regs regs[R];  // stage i, i + R .. in regs[i % R]
    look_up(tile_of(0));
    StaticFor<0, R>::run([&](auto i) {
      load(regs[i], tile_of(i));
      look_up(tile_of(i + 1));
    });
    StaticFor<0, 2>::run([&](auto i) {
      store(regs[i], tile_of(i), i);
      load(regs[i], tile_of(i + R));
      look_up(tile_of(i + 1 + R));
    });
    barrier_lds();
    if (rows_here) score(std::integral_constant<int, 0>{});
    for (int at = 0; at < steps; at += R)
      StaticFor<0, R>::run([&](auto i) __attribute__((always_inline)) {
        // (R = 3: the next stage is written, and the one before this one read)
        constexpr std::integral_constant<int, i> kThis{};
        constexpr std::integral_constant<int, (i + 1) % R> kNext{};
        constexpr std::integral_constant<int, (i + 2) % R> kAfter{};
        barrier_lds();
        store(regs[kAfter], tile_of(at + i + 2), kAfter);
        load(regs[kAfter], tile_of(at + i + 2 + R));
        look_up(tile_of(at + i + 3 + R));
        if (rows_here && tile_of(at + i) < last) multiply(tile_of(at + i), kThis, kNext);
      });
  }

  // The sums, each row one wave's: through its part of the ring, so that a store is of whole
  // rows.
  constexpr int kWide = D < 128 ? D : 128, kPad = kWide + 4;  // dims at a time
  static_assert(sizeof(sh) >= S::kWaves * 16 * kPad * 4, "16 rows of every wave fit the ring");
  float* const mine = reinterpret_cast<float*>(&sh[0][0]) + wave * 16 * kPad;
  barrier_lds();
  ScalarArgs& z = again();
#pragma unroll
  for (int c = 0; c < CT; ++c) {
    l[c] += __shfl_xor(l[c], 16, 64);
    l[c] += __shfl_xor(l[c], 32, 64);
    const int row0 = r0 + 16 * c;
    const int64_t at = static_cast<int64_t>(unit) * z.rows + row0;
#pragma unroll
    for (int d0 = 0; d0 < D; d0 += kWide) {
#pragma unroll
      for (int d = 0; d < kWide / 16; ++d)
        *reinterpret_cast<f32x4*>(mine + col * kPad + 16 * d + 4 * quad) = o[c][d0 / 16 + d];
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
#pragma unroll
      for (int i = 0; i < 16 * kWide / 4 / 64; ++i) {
        const int e = lane + 64 * i, row = e / (kWide / 4), part = e - row * (kWide / 4);
        if (row0 + row < r_end)
          *reinterpret_cast<f32x4*>(z.part_o + (at + row) * D + d0 + 4 * part) =
              *reinterpret_cast<const f32x4*>(mine + row * kPad + 4 * part);
      }
      __builtin_amdgcn_wave_barrier();
    }
    if (quad == 0 && row0 + col < r_end) {
      z.part_ml[(at + col) * 2] = m[c];
      z.part_ml[(at + col) * 2 + 1] = l[c];
    }
  }
}

template <typename T, int D, bool HALVES>
__global__ __launch_bounds__(64 * Stage<D>::kWaves, D > 128 ? 1 : 2) void prefix_many_kernel(PrefixArgs p, DecodeArgs a) {
  __shared__ alignas(1024) uint8_t ring[3][2 * Stage<D>::kMatrix];
  constexpr int kGroup = Stage<D>::kWaves;
  const int n = __builtin_amdgcn_readfirstlane(prefix_length(p));
  Prefix prefix = {};
  if (!p.roomy || static_cast<int>(blockIdx.x) < p.most_own) prefix = prefix_of(a, threadIdx.x & 63);
  const Division by = divide<D>(p, a, n, prefix.total * a.kv_heads * a.head_items);
  a.grid = kGroup * by.own_blocks;
  if (blockIdx.x == 0 && threadIdx.x < 64) p.units[threadIdx.x] = prefix.upto;
  const int block = static_cast<int>(blockIdx.x) - by.own_blocks;
  if (block < 0)
    own_attn<T, D>(a, prefix, blockIdx.x * kGroup + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6),
                             2 * kGroup * p.most_own);
  else
    prefix_many<T, D, HALVES>(again(), n, by.splits, block, ring);
}

// Joins a query head's partials of the prefix and of its sequence's own keys: WAVES waves
// a head, each of which finds the maximum and the sum of all partials; then their share of
// the partials' O, 16 bytes a lane.
template <typename T, int D, int WAVES>
__global__ __launch_bounds__(256) void shared_join_kernel(PrefixArgs p, DecodeArgs a) {
  constexpr int kLanes = D / 4, kAtOnce = 64 / kLanes, kHeads = 4 / WAVES;
  __shared__ f32x4 sh_o[4][kAtOnce][kLanes];
  constexpr int kFactors = 512;  // partials whose weights are in LDS at a time
  __shared__ float sh_f[4][kFactors];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int items = a.kv_heads * a.head_items, heads = a.kv_heads * a.group;
  const int at = min(static_cast<int>(blockIdx.x) * kHeads + wave / WAVES, a.batch * heads - 1);
  const int b = at / heads, head = at - b * heads;
  const int kvh = head / a.group, g = head - kvh * a.group;
  const int item = kvh * a.head_items + g / a.item_heads, h = g % a.item_heads;
  const int of_prefix = prefix_length(p);
  // (as the first launch had it)
  const int upto = p.units[lane];
  const Prefix prefix = {(a.batch + 63) / 64, upto, __builtin_amdgcn_readlane(upto, 63)};
  const int total = prefix.total * items;
  const Division by = divide<D>(p, a, of_prefix, total);
  a.grid = waves_of<D>(p.rows) * by.own_blocks;
  const int whole_slots = 2 * waves_of<D>(p.rows) * p.most_own;
  const int base = units_before(a, prefix, lane, b) * items;
  const Sequence s = sequence_of(a, b);
  const int start = base + item * s.units();
  const int w0 = workgroup_of(a, start + kItemUnits, total);
  const int own = workgroup_of(a, start + s.units() - 1, total) - w0 + 1;
  const int in_last = start > first_of(a, w0, total) ? 1 : 0;
  const int n = by.splits + own;
  // the partials' rows: the prefix's parts, then the own keys' (one workgroup's whole item
  // lies behind the runs' slots)
  const auto row_of = [&](int i) __attribute__((always_inline)) -> int64_t {
    if (i < by.splits) return (static_cast<int64_t>(i) * p.kv_heads + kvh) * p.rows + b * p.group + g;
    i -= by.splits;
    const int64_t slot = own == 1 ? whole_slots + static_cast<int64_t>(b) * items + item
                                  : 2 * static_cast<int64_t>(w0 + i) + (i == 0 ? in_last : 0);
    return slot * a.item_heads + h;
  };
  typedef float f32x2 __attribute__((ext_vector_type(2)));
  const auto ml_of = [&](int i) __attribute__((always_inline)) {
    return *reinterpret_cast<const f32x2*>((i < by.splits ? p.part_ml : a.part_ml) + row_of(i) * 2);
  };
  float top = neg_inf();
  for (int i = lane; i < n; i += 64) top = fmaxf(top, ml_of(i)[0]);
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) top = fmaxf(top, __shfl_xor(top, off, 64));
  const float ref = top == neg_inf() ? 0.f : top;
  float den = 0.f;
  f32x4 o = {0.f, 0.f, 0.f, 0.f};
  const int slot = lane / kLanes, e = lane % kLanes;
  for (int i0 = 0; i0 < n; i0 += kFactors) {
    const int upto = min(n, i0 + kFactors);
    for (int i = i0 + lane; i < upto; i += 64) {
      const f32x2 ml = ml_of(i);
      const float f = __builtin_amdgcn_exp2f(ml[0] - ref);
      sh_f[wave][i - i0] = f;
      den += f * ml[1];
    }
    // (its own wave's LDS)
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    if (slot < kAtOnce) {
      // (8 loads on their way, behind the last partial of this one again)
      constexpr int kStep = WAVES * kAtOnce;
      for (int i = i0 + wave % WAVES * kAtOnce + slot; i < upto; i += 8 * kStep) {
        f32x4 x[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int at_j = i + j * kStep < upto ? i + j * kStep : i;
          x[j] = *reinterpret_cast<const f32x4*>((at_j < by.splits ? p.part_o : a.part_o) + row_of(at_j) * D + 4 * e);
        }
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (i + j * kStep < upto) o += sh_f[wave][i + j * kStep - i0] * x[j];
      }
    }
    __builtin_amdgcn_wave_barrier();
  }
  if (slot < kAtOnce) sh_o[wave][slot][e] = o;
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) den += __shfl_xor(den, off, 64);
  __syncthreads();
  if (wave % WAVES == 0 && lane < kLanes) {
    o = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < WAVES; ++w)
#pragma unroll
      for (int i = 0; i < kAtOnce; ++i) o += sh_o[wave + w][i][lane];
    const bool none = s.n == 0 && of_prefix == 0;
    uint16_t* out = a.out + b * a.o_bs + head * a.o_hs + 4 * lane;
#pragma unroll
    for (int j = 0; j < 4; ++j) out[j] = Elem<T>::from_float(none ? 0.f : o[j] / den);
  }
}

// (Own keys have 8 workgroups at least, and multiples of 8.)
int cus_of() {
  const int n = cu_count() / 8 * 8;
  return n > 16 ? n : 16;
}

struct SharedPlan {
  DecodePlan own;
  int row_tiles, tile_rows, most_splits, most_own;
  int64_t blocks;
  bool roomy;
  int64_t own_rows, prefix_rows;  // of partials
};

SharedPlan shared_plan(const fpv2_shared_prefix_params& p) {
  SharedPlan plan;
  plan.own = decode_plan(p.own);
  const int64_t cus = cus_of(), rows = p.own.batch * (p.own.query_heads / p.own.kv_heads);
  const int64_t items = p.own.kv_heads * plan.own.head_items;
  // tiles of at most 128 rows, all alike, of whole waves
  const int64_t most_tiles = (rows + 127) / 128;
  plan.tile_rows = rows <= 16 ? 16 : static_cast<int>((rows + 32 * most_tiles - 1) / (32 * most_tiles) * 32);
  plan.row_tiles = rows > 0 ? static_cast<int>((rows + plan.tile_rows - 1) / plan.tile_rows) : 1;
  // What the division on the device can come to at most.
  const int64_t slots = (p.own.head_dim > 128 ? 1 : 2) * cus, waves = p.own.head_dim > 128 ? waves_of<256>(rows) : waves_of<128>(rows);
  const int64_t units = p.own.batch * items * (plan.own.most_tiles + kItemUnits);
  const int64_t need = ((units / kWaves + waves) / waves + 7) / 8 * 8;
  plan.most_own = static_cast<int>(need < slots ? need : slots);
  const int64_t tiles = (p.prefix_table_width * p.prefix_page_size + kTileKeys - 1) / kTileKeys;
  const int64_t most = (tiles + kWaves - 1) / kWaves;
  int64_t splits = (rows <= 16 ? cus : slots) / (p.own.kv_heads * plan.row_tiles);
  splits = splits < most ? splits : most;
  plan.most_splits = static_cast<int>(splits > 1 ? splits : 1);
  // (the parts' workgroups begin at multiples of 8, and so do their ends)
  const int64_t each = p.own.kv_heads * plan.row_tiles, rest = p.own.kv_heads % 8 ? 7 * plan.row_tiles : 0;
  const int64_t all = plan.most_own + plan.most_splits * each + rest, one = plan.most_own + each + rest;
  const bool before =
      rows > 16 && (p.own.head_dim <= 128 && tiles * each >= kLong * slots || kCoarse * each >= slots);
  const int64_t full = slots + rest + (before ? plan.most_own : 0);
  plan.blocks = all < full ? all : one < full ? full : one;
  plan.roomy = plan.most_splits * each <= cus && plan.most_own + plan.most_splits * each <= slots;
  plan.own_rows = (2LL * plan.most_own * waves + p.own.batch * items) * plan.own.item_heads;
  plan.prefix_rows = static_cast<int64_t>(plan.most_splits) * p.own.kv_heads * rows;
  return plan;
}

int check_shared(const char* name, const fpv2_shared_prefix_params* p) {
  if (p == nullptr) return fail(FPV2_ERR_ARGUMENT, "%s: null params", name);
  if (const int rc = check_params(name, &p->own)) return rc;
  if (p->own.window_tokens != 0 || p->own.sink_tokens != 0)
    return fail(FPV2_ERR_ARGUMENT, "%s: no window and no sinks", name);
  if (p->prefix_pages <= 0 || p->prefix_page_size <= 0 || p->prefix_table_width <= 0 ||
      p->prefix_pages > 0x7fffffff || p->prefix_page_size > 0x3fffffff || p->prefix_table_width > 0x3fffffff ||
      p->prefix_table_width * p->prefix_page_size > 0x3fffffff)
    return fail(FPV2_ERR_ARGUMENT, "%s: the prefix's pages, page_size and table_width must be positive and "
                "hold fewer than 2^30 tokens", name);
  if (p->prefix_length < 0) return fail(FPV2_ERR_ARGUMENT, "%s: prefix_length must not be negative", name);
  if (p->own.batch * p->own.query_heads > 0xffffff)
    return fail(FPV2_ERR_UNSUPPORTED, "%s: more than 2^24 - 1 query heads of the batch", name);
  return FPV2_OK;
}

int64_t shared_bytes(const fpv2_shared_prefix_params& p, const SharedPlan& plan) {
  return p.own.batch == 0 ? 0 : (plan.own_rows + plan.prefix_rows) * (p.own.head_dim + 2) * 4 + 64 * 4;
}

template <typename T, int D>
int launch(const PrefixArgs& p, const DecodeArgs& a, unsigned blocks, hipStream_t s) {
  // (offsets within 16 rows are 32 bits)
  const bool halves = (p.table == nullptr || p.page_size % 16 == 0) && p.k_rs < (1 << 25) && p.v_rs < (1 << 25);
  // (16 rows: 32768 keys 29 us by few, 35 by many; 131072 keys, one sequence 96 and 105; 1000 keys 7.6
  // and 9.4)
  if (p.rows <= 16)
    hipLaunchKernelGGL((prefix_few_kernel<T, D>), dim3(blocks), dim3(256), 0, s, p, a);
  else if (halves)
    hipLaunchKernelGGL((prefix_many_kernel<T, D, true>), dim3(blocks), dim3(64 * Stage<D>::kWaves), 0, s, p, a);
  else
    hipLaunchKernelGGL((prefix_many_kernel<T, D, false>), dim3(blocks), dim3(64 * Stage<D>::kWaves), 0, s, p, a);
  if (const int rc = check_launch("prefix_kernel")) return rc;
  const unsigned heads = static_cast<unsigned>(a.batch) * a.kv_heads * a.group;
  // Few heads have four waves each.  128 heads of 32 partials 5.6 us by four waves, 7.4 by one; 512 heads
  // of 62 7.6 and 9.2; 896 heads 9.7 and 9.6; 1536 heads 10.2 and 8.6 (D = 256: 128 heads 6.3 and
  // 10.1, 640 8.8 and 9.8; D = 64: 5.7 and 7.0, 7.2 and 6.9).
  if (heads <= 768)
    hipLaunchKernelGGL((shared_join_kernel<T, D, 4>), dim3(heads), dim3(256), 0, s, p, a);
  else
    hipLaunchKernelGGL((shared_join_kernel<T, D, 1>), dim3((heads + 3) / 4), dim3(256), 0, s, p, a);
  return check_launch("shared_join_kernel");
}

template <typename T>
int launch_dim(const PrefixArgs& p, const DecodeArgs& a, int64_t dim, unsigned blocks, hipStream_t s) {
  switch (dim) {
    case 64: return launch<T, 64>(p, a, blocks, s);
    case 96: return launch<T, 96>(p, a, blocks, s);
    case 128: return launch<T, 128>(p, a, blocks, s);
    default: return launch<T, 256>(p, a, blocks, s);
  }
}

}  // namespace
}  // namespace fpv2

extern "C" int64_t fpv2_shared_prefix_attention_workspace_bytes(const fpv2_shared_prefix_params* params) {
  using namespace fpv2;
  if (const int rc = check_shared("fpv2_shared_prefix_attention", params)) return rc;
  return shared_bytes(*params, shared_plan(*params));
}

extern "C" int fpv2_shared_prefix_attention(const void* q, const void* prefix_k, const void* prefix_v,
                                            const int32_t* prefix_table, const int32_t* prefix_length,
                                            const void* k_pages, const void* v_pages,
                                            const int32_t* page_table, const int32_t* lengths, void* out,
                                            int dtype, const fpv2_shared_prefix_params* params,
                                            void* workspace, int64_t workspace_bytes, void* stream) {
  using namespace fpv2;
  const char* name = "fpv2_shared_prefix_attention";
  const auto a16 = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; };
  if (const int rc = check_shared(name, params)) return rc;
  const fpv2_shared_prefix_params& p = *params;
  if (dtype != FPV2_BF16 && dtype != FPV2_F16)
    return fail(FPV2_ERR_UNSUPPORTED, "%s: dtype must be bf16 or f16", name);
  if (p.own.batch == 0) return FPV2_OK;
  if (!q || !prefix_k || !prefix_v || !k_pages || !v_pages || !out)
    return fail(FPV2_ERR_ARGUMENT, "%s: null pointer", name);
  if (page_table == nullptr && (p.own.table_width != 1 || p.own.pages < p.own.batch))
    return fail(FPV2_ERR_ARGUMENT, "%s: without a page table every sequence has one page", name);
  if (prefix_table == nullptr && p.prefix_table_width != 1)
    return fail(FPV2_ERR_ARGUMENT, "%s: without a prefix table the prefix has one page", name);
  if (page_table != nullptr && p.own.table_stride < 0)
    return fail(FPV2_ERR_ARGUMENT, "%s: table_stride must not be negative", name);
  const int64_t strides[] = {
      p.own.q_batch_stride, p.own.q_head_stride, p.own.k_page_stride, p.own.k_head_stride, p.own.k_row_stride,
      p.own.v_page_stride,  p.own.v_head_stride, p.own.v_row_stride,  p.pk_page_stride,    p.pk_head_stride,
      p.pk_row_stride,      p.pv_page_stride,    p.pv_head_stride,    p.pv_row_stride};
  for (const int64_t x : strides)
    if (x < 0 || x % 8)
      return fail(FPV2_ERR_ARGUMENT, "%s: strides of q, k and v must be multiples of 8", name);
  if (p.own.o_batch_stride < 0 || p.own.o_head_stride < 0)
    return fail(FPV2_ERR_ARGUMENT, "%s: output strides must not be negative", name);
  if (!a16(q) || !a16(k_pages) || !a16(v_pages) || !a16(prefix_k) || !a16(prefix_v))
    return fail(FPV2_ERR_ARGUMENT, "%s: q, k and v must be 16-byte aligned", name);
  const SharedPlan plan = shared_plan(p);
  const int64_t need = shared_bytes(p, plan);
  if (workspace == nullptr || workspace_bytes < need || !a16(workspace))
    return fail(FPV2_ERR_ARGUMENT, "%s: needs a 16-byte aligned workspace of %lld bytes", name,
                static_cast<long long>(need));
  DecodeArgs a = decode_args(p.own, plan.own);
  a.q = static_cast<const uint16_t*>(q);
  a.k = static_cast<const uint16_t*>(k_pages);
  a.v = static_cast<const uint16_t*>(v_pages);
  a.out = static_cast<uint16_t*>(out);
  a.table = page_table;
  a.lengths = lengths;
  // all partials' O first, so that each is 16-byte aligned
  a.part_o = static_cast<float*>(workspace);
  PrefixArgs x{};
  x.part_o = a.part_o + plan.own_rows * p.own.head_dim;
  a.part_ml = x.part_o + plan.prefix_rows * p.own.head_dim;
  x.part_ml = a.part_ml + plan.own_rows * 2;
  x.units = reinterpret_cast<int32_t*>(x.part_ml + plan.prefix_rows * 2);
  x.q = a.q;
  x.k = static_cast<const uint16_t*>(prefix_k);
  x.v = static_cast<const uint16_t*>(prefix_v);
  x.table = prefix_table;
  x.lengths = prefix_length;
  x.q_bs = a.q_bs;
  x.q_hs = a.q_hs;
  x.k_ps = p.pk_page_stride;
  x.k_hs = p.pk_head_stride;
  x.k_rs = p.pk_row_stride;
  x.v_ps = p.pv_page_stride;
  x.v_hs = p.pv_head_stride;
  x.v_rs = p.pv_row_stride;
  x.kv_heads = a.kv_heads;
  x.group = a.group;
  x.rows = a.batch * a.group;
  x.row_tiles = plan.row_tiles;
  x.tile_rows = plan.tile_rows;
  x.roomy = plan.roomy;
  x.most_splits = plan.most_splits;
  x.most_own = plan.most_own;
  x.cus = cus_of();
  x.pages = static_cast<int>(p.prefix_pages);
  x.page_size = static_cast<int>(p.prefix_page_size);
  x.capacity = static_cast<int>(p.prefix_table_width * p.prefix_page_size);
  x.length = static_cast<int>(p.prefix_length < x.capacity ? p.prefix_length : x.capacity);
  page_division(p.prefix_page_size, &x.page_mul, &x.page_shift);
  x.scale_log2 = a.scale_log2;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  const unsigned blocks = static_cast<unsigned>(plan.blocks);
  return dtype == FPV2_BF16 ? launch_dim<bf16_t>(x, a, p.own.head_dim, blocks, s)
                            : launch_dim<f16_t>(x, a, p.own.head_dim, blocks, s);
}
