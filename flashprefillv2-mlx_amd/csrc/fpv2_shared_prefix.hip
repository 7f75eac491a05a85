// Attention of one new token per sequence of a batch that shares a prefix: the
// prefix's keys once for all sequences, each sequence's own keys, and the join.
//
//   out[b][h] = sum_t p_t v_t / sum_t p_t,  p_t = exp(scale q[b][h].k_t - max),
//   t over the prefix and over b's own keys
//
// The sums split over t: partials (O, max, sum) of parts of the keys are joined as
//   O = sum_i exp(m_i - m) O_i, l = sum_i exp(m_i - m) l_i, m = max_i m_i.
// Three launches: the prefix (here), the own keys (decode_attn_kernel, all items left
// as partials), and the join.
//
// Prefix: the rows of a KV head are the batch's query heads of it, packed; a workgroup
// takes a tile of them and a part of the prefix's keys.  Its waves take 32 keys each on
// MFMA, as the decode attention does, for all rows of the tile.
#include "fpv2_batch.h"
#include "fpv2_decode_split.h"

namespace fpv2 {
namespace {

constexpr int kMaxSplits = 512;

struct PrefixArgs {
  const uint16_t* q;
  const uint16_t* k;
  const uint16_t* v;
  const int32_t* table;
  const int32_t* lengths;  // of one
  float* part_o;           // [splits][kv_heads][rows][D]
  float* part_ml;          // [splits][kv_heads][rows][2]
  int64_t q_bs, q_hs, k_ps, k_hs, k_rs, v_ps, v_hs, v_rs;
  int kv_heads, group, rows, row_tiles, tile_rows, splits;  // rows: batch * group
  int pages, page_size, capacity, length;
  uint32_t page_mul, page_shift;
  float scale_log2;
};

__device__ __forceinline__ int prefix_length(const PrefixArgs& a) {
  const int n = a.lengths != nullptr ? *a.lengths : a.length;
  return min(max(n, 0), a.capacity);
}

// A column's weights are relative to a reference.  bfloat16: one that moves only when a
// score exceeds it by 2^kLag, so that most tiles rescale nothing (weights reach 2^kLag).
// float16, which has only 2^-14 to 1 at full precision: by tile, as in the decode attention.
constexpr float kLag = 8.f, kHeadroom = 15.f, kBelow = 40.f;

// A page of the prefix (as the table has it) and a row in it.  In scalar registers where t
// is: a vector load would have to wait for all that were issued before it.
struct At {
  int id, row;
};
__device__ const int32_t kPageZero = 0;
__device__ __forceinline__ At prefix_at(const PrefixArgs& a, int t) {
  typedef const __attribute__((address_space(4))) int32_t* scalar_ptr;
  const uint32_t page = (__umulhi(static_cast<uint32_t>(t), a.page_mul) + t) >> a.page_shift;
  const int32_t* p = a.table != nullptr ? a.table + page : &kPageZero;
  return {*reinterpret_cast<scalar_ptr>(reinterpret_cast<uintptr_t>(p)), t - static_cast<int>(page) * a.page_size};
}
__device__ __forceinline__ int64_t page_of(const PrefixArgs& a, int id) { return min(max(id, 0), a.pages - 1); }
// Loads stay in the order that they are written in.
__device__ __forceinline__ void in_order() { asm volatile("" ::: "memory"); }

// A wave's 32 keys: K as the A operands of the scores, V as 8 rows' dims of a lane.
template <int D>
struct Tile {
  u32x4 k[2][D / 32];
  Words<D / 32> v[8];
};

template <int NW>
__device__ __forceinline__ Words<NW> buf_load_words(rsrc_t r, uint32_t off, uint32_t base) {
  Words<NW> x;
  if constexpr (NW % 4 == 0) {
#pragma unroll
    for (int i = 0; i < NW / 4; ++i) {
      const u32x4 w = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(r, off + 16 * i, base, 0));
#pragma unroll
      for (int j = 0; j < 4; ++j) x.w[4 * i + j] = w[j];
    }
  } else if constexpr (NW == 2) {
    const u32x2 w = __builtin_bit_cast(u32x2, __builtin_amdgcn_raw_buffer_load_b64(r, off, base, 0));
    x.w[0] = w[0];
    x.w[1] = w[1];
  } else {
#pragma unroll
    for (int i = 0; i < NW; ++i) x.w[i] = __builtin_amdgcn_raw_buffer_load_b32(r, off + 4 * i, base, 0);
  }
  return x;
}

// HALVES: 16 keys from a multiple of 16 on lie in one page (or there is no table): their
// addresses are the wave's, a lane's offsets do not change, and a descriptor of the rows
// up to the prefix's end reads zeros behind it.
template <typename T, int D, bool HALVES>
__global__ __launch_bounds__(256, D > 128 ? 1 : 2) void prefix_few_kernel(PrefixArgs a) {
  constexpr int KK = D / 32, DV = D / 16, CT = 1, ROWS = 16 * CT;
  constexpr bool kByTile = std::is_same<T, f16_t>::value;
  __shared__ float sh_o[4][16][D + 4];
  __shared__ float sh_ml[4][16][2];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 15, quad = lane >> 4;
  // A unit is a part of a KV head's keys; its row tiles' workgroups are 8 apart, so
  // that they share an XCD's L2.
  const int unit = blockIdx.x % 8 + 8 * (blockIdx.x / (8 * a.row_tiles));
  const int rt = blockIdx.x / 8 % a.row_tiles;
  if (unit >= a.kv_heads * a.splits) return;
  const int split = unit / a.kv_heads, kvh = unit - split * a.kv_heads;
  const int n = __builtin_amdgcn_readfirstlane(prefix_length(a));
  const int tiles = (n + kTileKeys - 1) / kTileKeys;
  const int first = static_cast<int>(static_cast<int64_t>(tiles) * split / a.splits);
  const int last = static_cast<int>(static_cast<int64_t>(tiles) * (split + 1) / a.splits);

  const uint16_t* kb = a.k + kvh * a.k_hs;
  const uint16_t* vb = a.v + kvh * a.v_hs;
  const uint32_t k_lane = (col * static_cast<uint32_t>(a.k_rs) + 8 * quad) * 2;
  const uint32_t v_lane = (4 * quad * static_cast<uint32_t>(a.v_rs) + DV * col) * 2;
  At half[2];  // HALVES: of the next tile's first and 17th key
  int row = 0, page = 0;  // else: lane i's (and i + 32's) of its key i
  const auto look_up = [&](int u0) {
    if constexpr (HALVES) {
#pragma unroll
      for (int t = 0; t < 2; ++t) half[t] = prefix_at(a, u0 + 16 * t < n ? u0 + 16 * t : 0);
    } else {
      const uint32_t t = min(u0 + (lane & 31), n - 1);
      const uint32_t at = (__umulhi(t, a.page_mul) + t) >> a.page_shift;
      row = t - at * a.page_size;
      const int id = a.table != nullptr ? a.table[at] : 0;
      page = min(max(id, 0), a.pages - 1);
    }
  };
  const auto load = [&](Tile<D>& x, int u0) {
    if constexpr (HALVES) {
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const int live = min(n - u0 - 16 * t, 16);  // (0 and less: zeros)
        const rsrc_t kr = make_rsrc(kb + page_of(a, half[t].id) * a.k_ps + half[t].row * a.k_rs,
                                    live > 0 ? ((live - 1) * a.k_rs + D) * 2 : 0);
        const rsrc_t vr = make_rsrc(vb + page_of(a, half[t].id) * a.v_ps + half[t].row * a.v_rs,
                                    live > 0 ? ((live - 1) * a.v_rs + D) * 2 : 0);
#pragma unroll
        for (int kk = 0; kk < KK; ++kk) x.k[t][kk] = buf_load16(kr, k_lane + 64 * kk);
#pragma unroll
        for (int j = 0; j < 4; ++j)
          x.v[4 * t + j] = buf_load_words<DV / 2>(vr, v_lane, j * static_cast<uint32_t>(a.v_rs) * 2);
      }
    } else {
      const int64_t koff = page * a.k_ps + row * a.k_rs;
      const int64_t voff = page * a.v_ps + row * a.v_rs;
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const uint16_t* p = kb + __shfl(koff, 16 * t + col, 64) + 8 * quad;
#pragma unroll
        for (int kk = 0; kk < KK; ++kk) x.k[t][kk] = load16(p + 32 * kk);
      }
#pragma unroll
      for (int j = 0; j < 8; ++j)
        x.v[j] = load_words<DV / 2>(vb + __shfl(voff, 16 * (j / 4) + 4 * quad + j % 4, 64) + DV * col);
    }
  };

  u32x4 qf[CT][KK];
#pragma unroll
  for (int c = 0; c < CT; ++c) {
    const int at = rt * ROWS + 16 * c + col;
    const int b = at / a.group, g = at - b * a.group;
    const uint16_t* p = a.q + b * a.q_bs + (kvh * a.group + g) * a.q_hs + 8 * quad;
#pragma unroll
    for (int kk = 0; kk < KK; ++kk) qf[c][kk] = at < a.rows ? load16(p + 32 * kk) : u32x4{0, 0, 0, 0};
  }
  f32x4 o[CT][DV];
  float m[CT], l[CT], greatest[CT];
#pragma unroll
  for (int c = 0; c < CT; ++c) {
    m[c] = greatest[c] = neg_inf();
    l[c] = 0.f;
#pragma unroll
    for (int d = 0; d < DV; ++d) o[c][d] = f32x4{0.f, 0.f, 0.f, 0.f};
  }

  const auto multiply = [&](Tile<D>& y, int u0) {
    const bool cut = u0 + kTileKeys > n;
    u32x4 pf[CT];
#pragma unroll
    for (int c = 0; c < CT; ++c) {
      f32x4 sc[2];
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        sc[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int kk = 0; kk < KK; ++kk)
          sc[t] = Elem<T>::mfma16(as_vec8<T>(y.k[t][kk]), as_vec8<T>(qf[c][kk]), sc[t]);
      }
      float x[8], top = neg_inf();
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        x[j] = sc[j / 4][j % 4] * a.scale_log2;
        if (cut && u0 + 16 * (j / 4) + 4 * quad + j % 4 >= n) x[j] = neg_inf();
        top = fmaxf(top, x[j]);
      }
      if (kByTile || __any(top > m[c] + kLag)) {
        top = fmaxf(top, __shfl_xor(top, 16, 64));
        top = fmaxf(top, __shfl_xor(top, 32, 64));
        float to = top > m[c] + kLag ? top : m[c];
        if constexpr (kByTile) {
          greatest[c] = fmaxf(greatest[c], top);
          to = fmaxf(top, greatest[c] - kBelow) - kHeadroom;
        }
        const float fix = __builtin_amdgcn_exp2f(m[c] - (to == neg_inf() ? 0.f : to));
        m[c] = to;
        l[c] *= fix;
#pragma unroll
        for (int d = 0; d < DV; ++d) o[c][d] *= fix;
      }
      // (nothing but -inf so far: weights of zero instead of NaN)
      const float ref = m[c] == neg_inf() ? 0.f : m[c];
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = __builtin_amdgcn_exp2f(x[j] - ref);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        pf[c][j] = pack2<T>(x[2 * j], x[2 * j + 1]);
        l[c] += x[2 * j] + x[2 * j + 1];
      }
    }
    if (!HALVES && cut) {
      // (a zero weight would make NaN of what an unused row may hold)
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (u0 + 16 * (j / 4) + 4 * quad + j % 4 >= n) {
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
#pragma unroll
      for (int c = 0; c < CT; ++c) o[c][d] = Elem<T>::mfma16(as_vec8<T>(vt), as_vec8<T>(pf[c]), o[c][d]);
    }
  };

  // A tile's loads are a tile ahead of its products, and its pages one more.  (Tiles behind
  // the last one are loaded too, HALVES: as zeros, else the last key again; so that it is
  // known at each product how many loads were issued since its own.)
  int u0 = (first + wave) * kTileKeys;
  const int u_end = min(n, last * kTileKeys);
  if (u0 < u_end) {
    Tile<D> even, odd;
    look_up(u0);
    load(even, u0);
    look_up(u0 + kStepKeys);
    for (; u0 < u_end; u0 += 2 * kStepKeys) {
      load(odd, u0 + kStepKeys);
      look_up(u0 + 2 * kStepKeys);
      multiply(even, u0);
      load(even, u0 + 2 * kStepKeys);
      look_up(u0 + 3 * kStepKeys);
      if (u0 + kStepKeys < u_end) multiply(odd, u0 + kStepKeys);
    }
  }

  // join the four waves, 16 rows at a time
#pragma unroll
  for (int c = 0; c < CT; ++c) {
    l[c] += __shfl_xor(l[c], 16, 64);
    l[c] += __shfl_xor(l[c], 32, 64);
    if (c > 0) __syncthreads();
    if (quad == 0) {
      sh_ml[wave][col][0] = m[c];
      sh_ml[wave][col][1] = l[c];
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int d = 0; d < DV; ++d) sh_o[wave][col][(4 * quad + i) * DV + d] = o[c][d][i];
    __syncthreads();
    const int r0 = rt * ROWS + 16 * c;
    for (int e = tid; e < 16 * D; e += 256) {
      const int r = e / D, d = e % D;
      if (r0 + r >= a.rows) break;
      float top = neg_inf();
#pragma unroll
      for (int w = 0; w < 4; ++w) top = fmaxf(top, sh_ml[w][r][0]);
      const float ref = top == neg_inf() ? 0.f : top;
      float sum = 0.f, den = 0.f;
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        // (a wave without keys has max -inf, sum 0 and O 0)
        const float f = __builtin_amdgcn_exp2f(sh_ml[w][r][0] - ref);
        sum += f * sh_o[w][r][d];
        den += f * sh_ml[w][r][1];
      }
      const int64_t at = static_cast<int64_t>(unit) * a.rows + r0 + r;
      a.part_o[at * D + d] = sum;
      if (d == 0) {
        a.part_ml[at * 2] = top;
        a.part_ml[at * 2 + 1] = den;
      }
    }
  }
}


// More rows than a tile of MFMA: the workgroup's waves, 32 rows each, share the keys
// through LDS.  A stage is 32 keys' K and V, rows of a power of two of bytes whose 16-byte
// chunks are permuted so that neither the reads of K (16 keys' chunks) nor the transposing
// reads of V (8 keys, 32 bytes each) meet in a bank.  Two stages in LDS, kAhead more on
// their way in registers: 16 bytes a load, a few loads a thread and stage.
template <int D>
struct Stage {
  static constexpr int kRow = D <= 64 ? 128 : D <= 128 ? 256 : 512;  // bytes of a row in LDS
  static constexpr int kMatrix = kTileKeys * kRow;
  static constexpr int kChunks = D / 8;                              // 16-byte chunks of a row
  static constexpr int kLoads = (kTileKeys * kChunks + 255) / 256;   // a thread's, of K and of V each
  static constexpr int kSpan = D <= 96 ? 32 : 16;                    // keys of a load, in one page
  static __device__ __forceinline__ int k_mask(int row) { return kRow >= 256 ? row & 15 : row >> 1 & 7; }
  static __device__ __forceinline__ int v_mask(int row) { return (kRow >= 256 ? row & 7 : row >> 1 & 3) << 1; }
};
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

// A barrier for what ds_write wrote: it waits for this wave's LDS operations only, not for
// its loads from memory (as __syncthreads() does).
__device__ __forceinline__ void barrier_lds() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// SPANS: the keys of a load lie in one page (or there is no table): their addresses are the
// wave's, and a descriptor of the rows up to the prefix's end reads zeros behind it.
template <typename T, int D, bool SPANS>
__global__ __launch_bounds__(256, D > 128 ? 1 : 2) void prefix_many_kernel(PrefixArgs a) {
  using S = Stage<D>;
  constexpr int KK = D / 32, DT = D / 16, CT = 2, L = S::kLoads, kAhead = 2;
  constexpr bool kByTile = std::is_same<T, f16_t>::value;
  __shared__ alignas(1024) uint8_t sh[2][2][S::kMatrix];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 15, quad = lane >> 4;
  // A unit is a part of a KV head's keys; its row tiles' workgroups are 8 apart, so
  // that they share an XCD's L2.
  const int unit = blockIdx.x % 8 + 8 * (blockIdx.x / (8 * a.row_tiles));
  const int rt = blockIdx.x / 8 % a.row_tiles;
  if (unit >= a.kv_heads * a.splits) return;
  const int split = unit / a.kv_heads, kvh = unit - split * a.kv_heads;
  const int n = __builtin_amdgcn_readfirstlane(prefix_length(a));
  const int tiles = (n + kTileKeys - 1) / kTileKeys;
  const int first = static_cast<int>(static_cast<int64_t>(tiles) * split / a.splits);
  const int last = static_cast<int>(static_cast<int64_t>(tiles) * (split + 1) / a.splits);
  const int r0 = rt * a.tile_rows + 32 * wave;                    // this wave's rows
  const int r_end = min(a.rows, (rt + 1) * a.tile_rows);

  const uint16_t* kb = a.k + kvh * a.k_hs;
  const uint16_t* vb = a.v + kvh * a.v_hs;
  // a thread's loads: chunk at[i] of the stage, row at[i] / kChunks of it
  int key[L], part[L], k_to[L], v_to[L];
#pragma unroll
  for (int i = 0; i < L; ++i) {
    const int c = tid + 256 * i;
    key[i] = c / S::kChunks;
    part[i] = c - key[i] * S::kChunks;
    k_to[i] = key[i] * S::kRow + (part[i] ^ S::k_mask(key[i])) * 16;
    v_to[i] = key[i] * S::kRow + (part[i] ^ S::v_mask(key[i])) * 16;
  }
  const auto in_stage = [&](int i) { return kTileKeys * S::kChunks % 256 == 0 || key[i] < kTileKeys; };
  constexpr int kSpans = SPANS && S::kSpan == 16 ? 2 : 1;
  constexpr int kPer = 256 / S::kChunks;  // keys of a thread's load and the next
  At from[SPANS ? kSpans : L];  // of a coming stage's spans, or the thread's loads
  const auto look_up = [&](int tile) {
    const int u0 = tile * kTileKeys;
    if constexpr (SPANS) {
#pragma unroll
      for (int i = 0; i < kSpans; ++i) from[i] = prefix_at(a, u0 + 16 * i < n ? u0 + 16 * i : 0);
    } else {
#pragma unroll
      for (int i = 0; i < L; ++i) {
        const uint32_t t = min(u0 + min(key[i], kTileKeys - 1), n - 1);
        const uint32_t page = (__umulhi(t, a.page_mul) + t) >> a.page_shift;
        from[i] = {a.table != nullptr ? a.table[page] : 0, static_cast<int>(t - page * a.page_size)};
      }
    }
  };
  struct Regs {
    u32x4 k[L], v[L];
  };
  const auto load = [&](Regs& x, int tile) {
#pragma unroll
    for (int i = 0; i < L; ++i) {
      if constexpr (SPANS) {
        constexpr bool kBoth = kSpans == 2;
        const int s = kBoth ? i * kPer / 16 : 0;  // the load's span
        const int live = min(n - tile * kTileKeys - 16 * s, kTileKeys);  // (0 and less: zeros)
        const rsrc_t kr = make_rsrc(kb + page_of(a, from[s].id) * a.k_ps + from[s].row * a.k_rs,
                                    live > 0 ? ((live - 1) * a.k_rs + D) * 2 : 0);
        const rsrc_t vr = make_rsrc(vb + page_of(a, from[s].id) * a.v_ps + from[s].row * a.v_rs,
                                    live > 0 ? ((live - 1) * a.v_rs + D) * 2 : 0);
        const uint32_t in = key[i] - 16 * s;
        x.k[i] = buf_load16(kr, in_stage(i) ? (in * static_cast<uint32_t>(a.k_rs) + 8 * part[i]) * 2 : kOOB);
        in_order();
        x.v[i] = buf_load16(vr, in_stage(i) ? (in * static_cast<uint32_t>(a.v_rs) + 8 * part[i]) * 2 : kOOB);
        in_order();
      } else {
        x.k[i] = load16(kb + page_of(a, from[i].id) * a.k_ps + from[i].row * a.k_rs + 8 * part[i]);
        in_order();
        x.v[i] = load16(vb + page_of(a, from[i].id) * a.v_ps + from[i].row * a.v_rs + 8 * part[i]);
        in_order();
      }
    }
  };
  const auto store = [&](const Regs& x, int tile) {
    uint8_t* const at = &sh[tile & 1][0][0];
#pragma unroll
    for (int i = 0; i < L; ++i)
      if (in_stage(i)) {
        store16(at + k_to[i], x.k[i]);
        // (a zero weight would make NaN of what an unused row may hold)
        const bool live = SPANS || tile * kTileKeys + key[i] < n;
        store16(at + S::kMatrix + v_to[i], live ? x.v[i] : u32x4{0, 0, 0, 0});
      }
  };

  u32x4 qf[CT][KK];
#pragma unroll
  for (int c = 0; c < CT; ++c) {
    const int at = r0 + 16 * c + col;
    const int b = at / a.group, g = at - b * a.group;
    const uint16_t* p = a.q + b * a.q_bs + (kvh * a.group + g) * a.q_hs + 8 * quad;
#pragma unroll
    for (int kk = 0; kk < KK; ++kk) qf[c][kk] = at < r_end ? load16(p + 32 * kk) : u32x4{0, 0, 0, 0};
  }
  f32x4 o[CT][DT];
  float m[CT], l[CT], greatest[CT];
#pragma unroll
  for (int c = 0; c < CT; ++c) {
    m[c] = greatest[c] = neg_inf();
    l[c] = 0.f;
#pragma unroll
    for (int d = 0; d < DT; ++d) o[c][d] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  // this lane's reads: K row col's chunk, V rows 4 quad + col / 4's 8 bytes
  const int v_row = 4 * quad + col / 4;

  const auto multiply = [&](int tile) {
    const uint8_t* const ks = &sh[tile & 1][0][0];
    const uint8_t* const vs = ks + S::kMatrix;
    f32x4 sc[CT][2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
#pragma unroll
      for (int c = 0; c < CT; ++c) sc[c][t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int kk = 0; kk < KK; ++kk) {
        const u32x4 kf = load16(ks + (16 * t + col) * S::kRow + ((4 * kk + quad) ^ S::k_mask(16 * t + col)) * 16);
#pragma unroll
        for (int c = 0; c < CT; ++c) sc[c][t] = Elem<T>::mfma16(as_vec8<T>(kf), as_vec8<T>(qf[c][kk]), sc[c][t]);
      }
    }
    const int u0 = tile * kTileKeys;
    const bool cut = u0 + kTileKeys > n;
    u32x4 pf[CT];
#pragma unroll
    for (int c = 0; c < CT; ++c) {
      float x[8], top = neg_inf();
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        x[j] = sc[c][j / 4][j % 4] * a.scale_log2;
        if (cut && u0 + 16 * (j / 4) + 4 * quad + j % 4 >= n) x[j] = neg_inf();
        top = fmaxf(top, x[j]);
      }
      if (kByTile || __any(top > m[c] + kLag)) {
        top = fmaxf(top, __shfl_xor(top, 16, 64));
        top = fmaxf(top, __shfl_xor(top, 32, 64));
        float to = top > m[c] + kLag ? top : m[c];
        if constexpr (kByTile) {
          greatest[c] = fmaxf(greatest[c], top);
          to = fmaxf(top, greatest[c] - kBelow) - kHeadroom;
        }
        const float fix = __builtin_amdgcn_exp2f(m[c] - (to == neg_inf() ? 0.f : to));
        m[c] = to;
        l[c] *= fix;
#pragma unroll
        for (int d = 0; d < DT; ++d) o[c][d] *= fix;
      }
      // (nothing but -inf so far: weights of zero instead of NaN)
      const float ref = m[c] == neg_inf() ? 0.f : m[c];
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = __builtin_amdgcn_exp2f(x[j] - ref);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        pf[c][j] = pack2<T>(x[2 * j], x[2 * j + 1]);
        l[c] += x[2 * j] + x[2 * j + 1];
      }
    }
#pragma unroll
    for (int d = 0; d < DT; ++d) {
      u32x4 vt;  // dim d of the lane's 8 keys
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const int row = 16 * t + v_row;
        const uint8_t* p = vs + row * S::kRow + ((2 * d + (col % 4) / 2) ^ S::v_mask(row)) * 16 + col % 2 * 8;
        const s16x4 w = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
            reinterpret_cast<lds_s16x4*>(static_cast<uintptr_t>(lds_addr(p))));
        const u32x2 words = __builtin_bit_cast(u32x2, w);
        vt[2 * t] = words[0];
        vt[2 * t + 1] = words[1];
      }
#pragma unroll
      for (int c = 0; c < CT; ++c) o[c][d] = Elem<T>::mfma16(as_vec8<T>(vt), as_vec8<T>(pf[c]), o[c][d]);
    }
  };

  const bool rows_here = r0 < r_end;
  // (Stages behind the last one are loaded too, SPANS: as zeros, else the last key again; so
  // that it is known at each store how many loads were issued since its own.)
  if (first < last) {
    Regs even, odd;  // stages first + 1, + 3 .. and + 2, + 4 ..
    look_up(first);
    load(even, first);
    look_up(first + 1);
    store(even, first);
    load(even, first + 1);
    look_up(first + 2);
    load(odd, first + 2);
    look_up(first + 3);
    for (int at = first; at < last; at += 2) {
      const auto step = [&](Regs& next, int tile) {
        barrier_lds();  // the stage is written, and the other one read
        store(next, tile + 1);
        load(next, tile + 1 + kAhead);
        look_up(tile + 2 + kAhead);
        if (rows_here && tile < last) multiply(tile);
      };
      step(even, at);
      step(odd, at + 1);
    }
  }

  // (each row is one wave's)
#pragma unroll
  for (int c = 0; c < CT; ++c) {
    l[c] += __shfl_xor(l[c], 16, 64);
    l[c] += __shfl_xor(l[c], 32, 64);
    const int row = r0 + 16 * c + col;
    if (row >= r_end) continue;
    const int64_t at = static_cast<int64_t>(unit) * a.rows + row;
#pragma unroll
    for (int d = 0; d < DT; ++d) *reinterpret_cast<f32x4*>(a.part_o + at * D + 16 * d + 4 * quad) = o[c][d];
    if (quad == 0) {
      a.part_ml[at * 2] = m[c];
      a.part_ml[at * 2 + 1] = l[c];
    }
  }
}

// Joins a query head's partials of the prefix and of its sequence's own keys: first
// the weights of all partials, then their sum, 16 bytes of a partial a thread.
template <typename T, int D>
__global__ __launch_bounds__(256) void shared_join_kernel(PrefixArgs p, DecodeArgs a) {
  constexpr int kLanes = D / 4, kSlots = 256 / kLanes;  // partials at a time
  __shared__ float sh_f[kMaxSplits + kMaxGrid];
  __shared__ float sh_r[4];
  __shared__ f32x4 sh_o[kSlots][kLanes];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int items = a.kv_heads * a.head_items, heads = a.kv_heads * a.group;
  const int b = blockIdx.x / heads, head = blockIdx.x - b * heads;
  const int kvh = head / a.group, g = head - kvh * a.group;
  const int item = kvh * a.head_items + g / a.item_heads, h = g % a.item_heads;
  const Prefix prefix = prefix_of(a, lane);
  const int total = prefix.total * items;
  const int base = units_before(a, prefix, lane, b) * items;
  const Sequence s = sequence_of(a, b);
  const int start = base + item * s.units();
  const int w0 = workgroup_of(a, start + kItemUnits, total);
  const int own = workgroup_of(a, start + s.units() - 1, total) - w0 + 1;
  const int in_last = start > first_of(a, w0, total) ? 1 : 0;
  const int n = p.splits + own;
  // the partials' rows: the prefix's parts, then the own keys' (one workgroup's whole item
  // lies behind the runs' slots)
  const auto row_of = [&](int i) -> int64_t {
    if (i < p.splits) return (static_cast<int64_t>(i) * p.kv_heads + kvh) * p.rows + b * p.group + g;
    i -= p.splits;
    const int64_t slot = own == 1 ? 2 * static_cast<int64_t>(a.grid) + static_cast<int64_t>(b) * items + item
                                  : 2 * static_cast<int64_t>(w0 + i) + (i == 0 ? in_last : 0);
    return slot * a.item_heads + h;
  };
  float top = neg_inf();
  for (int i = tid; i < n; i += 256) {
    const float m = (i < p.splits ? p.part_ml : a.part_ml)[row_of(i) * 2];
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
    den += f * (i < p.splits ? p.part_ml : a.part_ml)[row_of(i) * 2 + 1];
  }
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) den += __shfl_xor(den, off, 64);
  if (lane == 0) sh_r[wave] = den;
  __syncthreads();
  den = (sh_r[0] + sh_r[1]) + (sh_r[2] + sh_r[3]);
  f32x4 o = {0.f, 0.f, 0.f, 0.f};
  const int slot = tid / kLanes, e = tid % kLanes;
  if (slot < kSlots) {
#pragma unroll 4
    for (int i = slot; i < n; i += kSlots)
      o += sh_f[i] * *reinterpret_cast<const f32x4*>((i < p.splits ? p.part_o : a.part_o) + row_of(i) * D + 4 * e);
    sh_o[slot][e] = o;
  }
  __syncthreads();
  if (tid < kLanes) {
#pragma unroll
    for (int i = 1; i < kSlots; ++i) o += sh_o[i][tid];
    const bool none = s.n == 0 && prefix_length(p) == 0;
    uint16_t* out = a.out + b * a.o_bs + head * a.o_hs + 4 * tid;
#pragma unroll
    for (int j = 0; j < 4; ++j) out[j] = Elem<T>::from_float(none ? 0.f : o[j] / den);
  }
}

struct SharedPlan {
  DecodePlan own;
  int row_tiles, tile_rows, splits;
  int64_t own_rows, prefix_rows;  // of partials
};

SharedPlan shared_plan(const fpv2_shared_prefix_params& p) {
  SharedPlan plan;
  plan.own = decode_plan(p.own);
  const int64_t rows = p.own.batch * (p.own.query_heads / p.own.kv_heads);
  // tiles of at most 128 rows, all alike, of whole waves
  plan.row_tiles = static_cast<int>((rows + 127) / 128);
  plan.tile_rows = rows <= 16 ? 16 : static_cast<int>((rows + 32 * plan.row_tiles - 1) / (32 * plan.row_tiles) * 32);
  if (plan.row_tiles > 0) plan.row_tiles = static_cast<int>((rows + plan.tile_rows - 1) / plan.tile_rows);
  const int64_t tiles = (p.prefix_table_width * p.prefix_page_size + kTileKeys - 1) / kTileKeys;
  const int64_t per = p.own.head_dim > 128 ? 1 : 2;
  int64_t splits = per * cu_count() / (p.own.kv_heads * (plan.row_tiles > 0 ? plan.row_tiles : 1));
  const int64_t most = (tiles + 2 * kWaves - 1) / (2 * kWaves);
  splits = splits < most ? splits : most;
  splits = splits < kMaxSplits ? splits : kMaxSplits;
  plan.splits = static_cast<int>(splits > 1 ? splits : 1);
  const int64_t items = p.own.kv_heads * plan.own.head_items;
  plan.own_rows = (2LL * plan.own.grid + p.own.batch * items) * plan.own.item_heads;
  plan.prefix_rows = static_cast<int64_t>(plan.splits) * p.own.kv_heads * rows;
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
  return p.own.batch == 0 ? 0 : (plan.own_rows + plan.prefix_rows) * (p.own.head_dim + 2) * 4;
}

template <typename T, int D>
int launch(const PrefixArgs& p, const DecodeArgs& a, hipStream_t s) {
  const unsigned units = (static_cast<unsigned>(p.kv_heads) * p.splits + 7) / 8 * 8;
  const dim3 grid(units * p.row_tiles);
  const bool few = p.rows <= 16;
  // (offsets within a stage are 32 bits)
  const bool spans = (p.table == nullptr || p.page_size % (few ? 16 : Stage<D>::kSpan) == 0) &&
                     p.k_rs < (1 << 24) && p.v_rs < (1 << 24);
  if (few && spans)
    hipLaunchKernelGGL((prefix_few_kernel<T, D, true>), grid, dim3(256), 0, s, p);
  else if (few)
    hipLaunchKernelGGL((prefix_few_kernel<T, D, false>), grid, dim3(256), 0, s, p);
  else if (spans)
    hipLaunchKernelGGL((prefix_many_kernel<T, D, true>), grid, dim3(256), 0, s, p);
  else
    hipLaunchKernelGGL((prefix_many_kernel<T, D, false>), grid, dim3(256), 0, s, p);
  if (const int rc = check_launch("prefix_many_kernel")) return rc;
  hipLaunchKernelGGL((decode_attn_kernel<T, D, true>), dim3(a.grid), dim3(256), 0, s, a);
  hipLaunchKernelGGL((shared_join_kernel<T, D>), dim3(static_cast<unsigned>(a.batch) * a.kv_heads * a.group),
                     dim3(256), 0, s, p, a);
  return check_launch("shared_join_kernel");
}

template <typename T>
int launch_dim(const PrefixArgs& p, const DecodeArgs& a, int64_t dim, hipStream_t s) {
  switch (dim) {
    case 64: return launch<T, 64>(p, a, s);
    case 96: return launch<T, 96>(p, a, s);
    case 128: return launch<T, 128>(p, a, s);
    default: return launch<T, 256>(p, a, s);
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
  x.splits = plan.splits;
  x.pages = static_cast<int>(p.prefix_pages);
  x.page_size = static_cast<int>(p.prefix_page_size);
  x.capacity = static_cast<int>(p.prefix_table_width * p.prefix_page_size);
  x.length = static_cast<int>(p.prefix_length < x.capacity ? p.prefix_length : x.capacity);
  page_division(p.prefix_page_size, &x.page_mul, &x.page_shift);
  x.scale_log2 = a.scale_log2;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  return dtype == FPV2_BF16 ? launch_dim<bf16_t>(x, a, p.own.head_dim, s)
                            : launch_dim<f16_t>(x, a, p.own.head_dim, s);
}
