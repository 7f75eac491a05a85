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
  int kv_heads, group, rows, row_tiles, splits;  // rows: batch * group
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

template <typename T, int D, int CT>
__global__ __launch_bounds__(256, (CT > 2 || D > 128) ? 1 : 2) void prefix_attn_kernel(PrefixArgs a) {
  constexpr int KK = D / 32, DV = D / 16, ROWS = 16 * CT;
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
  const int n = prefix_length(a);
  const int tiles = (n + kTileKeys - 1) / kTileKeys;
  const int first = static_cast<int>(static_cast<int64_t>(tiles) * split / a.splits);
  const int last = static_cast<int>(static_cast<int64_t>(tiles) * (split + 1) / a.splits);

  u32x4 qf[CT][KK];
#pragma unroll
  for (int c = 0; c < CT; ++c) {
    const int row = rt * ROWS + 16 * c + col;
    const int b = row / a.group, g = row - b * a.group;
    const uint16_t* p = a.q + b * a.q_bs + (kvh * a.group + g) * a.q_hs + 8 * quad;
#pragma unroll
    for (int kk = 0; kk < KK; ++kk) qf[c][kk] = row < a.rows ? load16(p + 32 * kk) : u32x4{0, 0, 0, 0};
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

  const uint16_t* kb = a.k + kvh * a.k_hs;
  const uint16_t* vb = a.v + kvh * a.v_hs;
  // lane i (and i + 32) looks up the row of the tile's key i
  auto lookup = [&](int u0, int* row) {
    const uint32_t t = min(u0 + (lane & 31), n - 1);
    const uint32_t page = (__umulhi(t, a.page_mul) + t) >> a.page_shift;
    *row = t - page * a.page_size;
    const int id = a.table != nullptr ? a.table[page] : 0;
    return min(max(id, 0), a.pages - 1);
  };
  int u0 = (first + wave) * kTileKeys;
  const int u_end = min(n, last * kTileKeys);
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
    Words<DV / 2> vf[8];
#pragma unroll
    for (int j = 0; j < 8; ++j)
      vf[j] = load_words<DV / 2>(vb + __shfl(voff, 16 * (j / 4) + 4 * quad + j % 4, 64) + DV * col);
    if (u0 + kStepKeys < u_end) page = lookup(u0 + kStepKeys, &row);

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
          sc[t] = Elem<T>::mfma16(as_vec8<T>(kf[t][kk]), as_vec8<T>(qf[c][kk]), sc[t]);
      }
      float x[8], top = neg_inf();
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        x[j] = sc[j / 4][j % 4] * a.scale_log2;
        if (cut && u0 + 16 * (j / 4) + 4 * quad + j % 4 >= n) x[j] = neg_inf();
        top = fmaxf(top, x[j]);
      }
      top = fmaxf(top, __shfl_xor(top, 16, 64));
      top = fmaxf(top, __shfl_xor(top, 32, 64));
      if (kByTile || __any(top > m[c] + kLag)) {
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
    if (cut) {
      // (a zero weight would make NaN of what an unused row may hold)
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (u0 + 16 * (j / 4) + 4 * quad + j % 4 >= n) {
#pragma unroll
          for (int w = 0; w < DV / 2; ++w) vf[j].w[w] = 0;
        }
    }
#pragma unroll
    for (int d = 0; d < DV; ++d) {
      u32x4 vt;  // dim d of the lane's 8 keys
#pragma unroll
      for (int j = 0; j < 4; ++j)
        vt[j] = __builtin_amdgcn_perm(vf[2 * j + 1].w[d / 2], vf[2 * j].w[d / 2],
                                      d % 2 ? 0x07060302u : 0x05040100u);
#pragma unroll
      for (int c = 0; c < CT; ++c) o[c][d] = Elem<T>::mfma16(as_vec8<T>(vt), as_vec8<T>(pf[c]), o[c][d]);
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
  int col_tiles, row_tiles, splits;
  int64_t own_rows, prefix_rows;  // of partials
};

SharedPlan shared_plan(const fpv2_shared_prefix_params& p) {
  SharedPlan plan;
  plan.own = decode_plan(p.own);
  const int64_t rows = p.own.batch * (p.own.query_heads / p.own.kv_heads);
  plan.col_tiles = rows <= 16 ? 1 : rows <= 32 || p.own.head_dim > 128 ? 2 : 4;
  plan.row_tiles = static_cast<int>((rows + 16 * plan.col_tiles - 1) / (16 * plan.col_tiles));
  const int64_t tiles = (p.prefix_table_width * p.prefix_page_size + kTileKeys - 1) / kTileKeys;
  const int64_t per = plan.col_tiles > 2 || p.own.head_dim > 128 ? 1 : 2;
  int64_t splits = per * cu_count() / (p.own.kv_heads * plan.row_tiles);
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
int launch(const PrefixArgs& p, const DecodeArgs& a, const SharedPlan& plan, hipStream_t s) {
  const unsigned units = (static_cast<unsigned>(p.kv_heads) * p.splits + 7) / 8 * 8;
  const dim3 grid(units * p.row_tiles);
  if (plan.col_tiles == 1)
    hipLaunchKernelGGL((prefix_attn_kernel<T, D, 1>), grid, dim3(256), 0, s, p);
  else if (D > 128 || plan.col_tiles == 2)
    hipLaunchKernelGGL((prefix_attn_kernel<T, D, 2>), grid, dim3(256), 0, s, p);
  else
    hipLaunchKernelGGL((prefix_attn_kernel<T, D, (D > 128 ? 2 : 4)>), grid, dim3(256), 0, s, p);
  if (const int rc = check_launch("prefix_attn_kernel")) return rc;
  hipLaunchKernelGGL((decode_attn_kernel<T, D, true>), dim3(a.grid), dim3(256), 0, s, a);
  hipLaunchKernelGGL((shared_join_kernel<T, D>), dim3(static_cast<unsigned>(a.batch) * a.kv_heads * a.group),
                     dim3(256), 0, s, p, a);
  return check_launch("shared_join_kernel");
}

template <typename T>
int launch_dim(const PrefixArgs& p, const DecodeArgs& a, const SharedPlan& plan, int64_t dim, hipStream_t s) {
  switch (dim) {
    case 64: return launch<T, 64>(p, a, plan, s);
    case 96: return launch<T, 96>(p, a, plan, s);
    case 128: return launch<T, 128>(p, a, plan, s);
    default: return launch<T, 256>(p, a, plan, s);
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
  x.splits = plan.splits;
  x.pages = static_cast<int>(p.prefix_pages);
  x.page_size = static_cast<int>(p.prefix_page_size);
  x.capacity = static_cast<int>(p.prefix_table_width * p.prefix_page_size);
  x.length = static_cast<int>(p.prefix_length < x.capacity ? p.prefix_length : x.capacity);
  page_division(p.prefix_page_size, &x.page_mul, &x.page_shift);
  x.scale_log2 = a.scale_log2;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  return dtype == FPV2_BF16 ? launch_dim<bf16_t>(x, a, plan, p.own.head_dim, s)
                            : launch_dim<f16_t>(x, a, plan, p.own.head_dim, s);
}
