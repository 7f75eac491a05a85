// Attention of one new token per sequence over pages of 8-bit codes.
//
//   out[b][h] = sum_t p_t vs_t v_t / sum_t p_t,  p_t = exp(scale ks_t q[b][h].k_t - max)
//
// with the codes k, v and a scale ks, vs of each key's row.  Bound by reading codes and
// scales once; schedule, waves and join are the decode attention's (fpv2_decode_split.h).
//
// The codes are whole numbers of 8 bits, exact in float16: byte b + 128 under the
// exponent of 1024 is 1152 + b.  So both products are float16 MFMA with operands made
// in registers:
//   the queries relative to the power of two of their greatest (bf16's 8 and f16's 11
//   bits stay whole down to 2^-14 of it, below that they are off by 2^-25 of it);
//   a key's scale on its score, in float32;
//   a value's scale on its weight: w_t = p_t vs_t = exp2((x_t - m) + log2 vs_t), m the greatest
//   x so far, rounded to float16 relative to 2^-15 of the tile's greatest such weight (a tile
//   2^-40 and more below the greatest so far: of 2^-40 of that one), so that neither the scores' range nor
//   the values' sizes cost bits: the logarithm is added to a difference of exponents, beside whose sizes
//   (2^17 and more) it would be rounded away.  The sum of the p_t is of unrounded ones.
//
// Measured (32 / 8 heads, D = 128): one sequence of 131072 keys 56 us, 4.9 TB/s of codes and scales,
// where 16-bit keys take 95; 32 sequences of 61 to 16001 keys 47; 1000 keys 7.5 us.  A byte costs
// four times the instructions of the 16-bit attention's, which fill what the reads leave.
// Without gain: loads a tile ahead (58.6 us), three and four workgroups a CU (58, 65); codes with
// their offset of 128 taken off the sums afterwards (55 us, but sums that cancel lose bits).
#include "fpv2_batch.h"
#include "fpv2_decode_split.h"

namespace fpv2 {
namespace {

struct Q8Args {
  DecodeArgs a;  // k and v: codes, their strides in bytes
  const float* ks;
  const float* vs;
  int64_t ks_ps, ks_hs, ks_rs, vs_ps, vs_hs, vs_rs;
};

constexpr float kHeadroom = 15.f, kBelow = 40.f;
constexpr float kLeast = -150.f;  // weights below are zeros, so that all exponents are small and exact

// Two bytes with the byte of float16's 1024 above each (from words with their top bits
// turned), less 1152: the codes.
__device__ __forceinline__ uint32_t less_offset(uint32_t pair) {
  const f16x2 offset = {static_cast<_Float16>(-1152.f), static_cast<_Float16>(-1152.f)};
  return __builtin_bit_cast(uint32_t, __builtin_bit_cast(f16x2, pair) + offset);
}
__device__ __forceinline__ u32x4 widen8(uint32_t a, uint32_t b) {
  a ^= 0x80808080u;
  b ^= 0x80808080u;
  return u32x4{less_offset(__builtin_amdgcn_perm(a, 0x64646464u, 0x00050004u)),
               less_offset(__builtin_amdgcn_perm(a, 0x64646464u, 0x00070006u)),
               less_offset(__builtin_amdgcn_perm(b, 0x64646464u, 0x00050004u)),
               less_offset(__builtin_amdgcn_perm(b, 0x64646464u, 0x00070006u))};
}

template <typename T, int D>
__global__ __launch_bounds__(256, 2) void decode_q8_kernel(Q8Args args) {
  const DecodeArgs& a = args.a;
  constexpr int KK = D / 32;         // MFMA steps of a key's dot product
  constexpr int KC = D / 64;         // 16-byte chunks of a lane's key (and 8 bytes more at D = 96)
  constexpr int DV = D / 16;         // dims of a lane
  constexpr int VW = (DV + 3) / 4;   // words of a lane's value
  __shared__ float sh_o[4][kMaxHeads][D + 4];
  __shared__ float sh_ml[4][kMaxHeads][2];
  __shared__ alignas(16) float sh_s[4][2][kTileKeys];  // a wave's tile: scales of k, log2 of v's
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 15, quad = lane >> 4;
  const int items = a.kv_heads * a.head_items;
  const int8_t* const k_codes = reinterpret_cast<const int8_t*>(a.k);
  const int8_t* const v_codes = reinterpret_cast<const int8_t*>(a.v);
  // the first dimension of a step's 8 for this lane; dimension d of lane c's values
  const auto step_dim = [&](int s) { return s < 2 * KC ? 64 * (s / 2) + 16 * quad + 8 * (s % 2) : 64 * KC + 8 * quad; };
  const auto value_dim = [](int c, int d) { return D != 96 ? DV * c + d : d < 4 ? 4 * c + d : 64 + 2 * c + d - 4; };

  const Prefix prefix = prefix_of(a, lane);
  const int total = prefix.total * items;
  const int lo = first_of(a, blockIdx.x, total), hi = first_of(a, blockIdx.x + 1, total);
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

    // queries as float16, relative to a power of two
    u32x4 qf[KK];
    float score_scale;
    {
      u32x4 w[KK];
      float size = 0.f;
#pragma unroll
      for (int i = 0; i < KK; ++i) {
        w[i] = col < heads ? load16(a.q + b_now * a.q_bs + head * a.q_hs + step_dim(i)) : u32x4{0, 0, 0, 0};
#pragma unroll
        for (int j = 0; j < 8; ++j)
          size = fmaxf(size, __builtin_fabsf(Elem<T>::to_float(static_cast<uint16_t>(w[i][j / 2] >> (16 * (j % 2))))));
      }
      size = fmaxf(size, __shfl_xor(size, 16, 64));
      size = fmaxf(size, __shfl_xor(size, 32, 64));
      const uint32_t exponent = min(max(__float_as_uint(size) >> 23, 1u), 253u);
      const float down = __uint_as_float((254u - exponent) << 23);
      score_scale = __uint_as_float(exponent << 23) * a.scale_log2;
#pragma unroll
      for (int i = 0; i < KK; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          qf[i][j] = pack2<f16_t>(Elem<T>::to_float(static_cast<uint16_t>(w[i][j])) * down,
                                  Elem<T>::to_float(static_cast<uint16_t>(w[i][j] >> 16)) * down);
    }
    f32x4 o[DV];
#pragma unroll
    for (int d = 0; d < DV; ++d) o[d] = f32x4{0.f, 0.f, 0.f, 0.f};
    float m = neg_inf(), l = 0.f;  // the exponent that l is relative to
    float off = 0.f, greatest = neg_inf();  // and, relative to m, the one that O is, and the greatest so far

    const int8_t* kb = k_codes + kvh * a.k_hs;
    const int8_t* vb = v_codes + kvh * a.v_hs;
    const int32_t* table = a.table != nullptr ? a.table + b_now * a.table_stride : nullptr;
    const float* sb = lane < 32 ? args.ks + kvh * args.ks_hs : args.vs + kvh * args.vs_hs;
    const int64_t s_ps = lane < 32 ? args.ks_ps : args.vs_ps, s_rs = lane < 32 ? args.ks_rs : args.vs_rs;
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
      float scale = sb[page * s_ps + row * s_rs];
      u32x4 kf[2][KC];
      u32x2 kr[2];
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const int8_t* p = kb + __shfl(koff, 16 * t + col, 64);
#pragma unroll
        for (int i = 0; i < KC; ++i) kf[t][i] = load16(p + 64 * i + 16 * quad);
        if constexpr (KK % 2) kr[t] = *reinterpret_cast<const u32x2*>(p + 64 * KC + 8 * quad);
      }
      Words<VW> vf[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int8_t* p = vb + __shfl(voff, 16 * (j / 4) + 4 * quad + j % 4, 64);
        if constexpr (D == 96) {
          vf[j].w[0] = *reinterpret_cast<const uint32_t*>(p + 4 * col);
          vf[j].w[1] = *reinterpret_cast<const uint16_t*>(p + 64 + 2 * col);
        } else {
          vf[j] = load_words<VW>(reinterpret_cast<const uint16_t*>(p + DV * col));
        }
      }
      if (u0 + kStepKeys < u_end) page = lookup(u0 + kStepKeys, &row);

      // the tile's scales to the lanes that hold their keys (by the wave's own LDS)
      sh_s[wave][lane / 32][lane % 32] = lane < 32 ? scale : __builtin_amdgcn_logf(scale);
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
      f32x4 sc[2];
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        sc[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < KK; ++i) {
          const u32x4 wide = i < 2 * KC ? widen8(kf[t][i / 2][i % 2 * 2], kf[t][i / 2][i % 2 * 2 + 1])
                                        : widen8(kr[t][0], kr[t][1]);
          sc[t] = Elem<f16_t>::mfma16(as_vec8<f16_t>(wide), as_vec8<f16_t>(qf[i]), sc[t]);
        }
      }
      const bool cut = u0 + kTileKeys > s_now.n;
      float x[8], y[8], top = neg_inf(), top_o = neg_inf();
      f32x4 vs[2];
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const f32x4 ks = *reinterpret_cast<const f32x4*>(&sh_s[wave][0][16 * t + 4 * quad]);
        vs[t] = *reinterpret_cast<const f32x4*>(&sh_s[wave][1][16 * t + 4 * quad]);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int j = 4 * t + i;
          x[j] = sc[t][i] * score_scale * ks[i];
          if (cut && u0 + 16 * t + 4 * quad + i >= s_now.n) x[j] = neg_inf();
          top = fmaxf(top, x[j]);
        }
      }
      __builtin_amdgcn_wave_barrier();
      top = fmaxf(m, column_max(top));
      // (nothing but -inf so far: weights of zero instead of NaN)
      const float ref = top == neg_inf() ? 0.f : top, down = m - ref;
      m = top;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        x[j] -= ref;
        y[j] = x[j] + vs[j / 4][j % 4];
        top_o = fmaxf(top_o, y[j]);
      }
      top_o = column_max(top_o);
      greatest = fmaxf(greatest + down, top_o);
      const float to = fmaxf(fmaxf(top_o, greatest - kBelow), kLeast) - kHeadroom;
      l *= __builtin_amdgcn_exp2f(down);
      const float fix = __builtin_amdgcn_exp2f(down + (off - to));
      off = to;
      u32x4 pf;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        l += __builtin_amdgcn_exp2f(x[2 * j]) + __builtin_amdgcn_exp2f(x[2 * j + 1]);
        pf[j] = pack2<f16_t>(__builtin_amdgcn_exp2f(y[2 * j] - to), __builtin_amdgcn_exp2f(y[2 * j + 1] - to));
      }
#pragma unroll
      for (int d = 0; d < DV; ++d) {
        u32x4 vt;  // dim d of the lane's 8 keys
#pragma unroll
        for (int j = 0; j < 4; ++j)
          vt[j] = less_offset(__builtin_amdgcn_perm(vf[2 * j + 1].w[d / 4], vf[2 * j].w[d / 4],
                                                    0x0c040c00u + 0x00010001u * (d % 4)) ^ 0x64806480u);
        o[d] *= fix;
        o[d] = Elem<f16_t>::mfma16(as_vec8<f16_t>(vt), as_vec8<f16_t>(pf), o[d]);
      }
    }
    l += __shfl_xor(l, 16, 64);
    l += __shfl_xor(l, 32, 64);
    // O relative to what l is
    const float fix = __builtin_amdgcn_exp2f(off);

    // join the four waves
    if (quad == 0) {
      sh_ml[wave][col][0] = m;
      sh_ml[wave][col][1] = l;
    }
    if (col < heads) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int d = 0; d < DV; ++d) sh_o[wave][col][value_dim(4 * quad + i, d)] = o[d][i] * fix;
    }
    __syncthreads();
    const bool whole = first == 0 && last == s_now.tiles;
    const int64_t slot = 2 * static_cast<int64_t>(blockIdx.x) + (cur == lo ? 0 : 1);
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
int launch(const Q8Args& x, bool join, hipStream_t s) {
  const DecodeArgs& a = x.a;
  hipLaunchKernelGGL((decode_q8_kernel<T, D>), dim3(a.grid), dim3(256), 0, s, x);
  if (join) launch_join<T, D>(a, s);
  return check_launch("decode_q8_kernel");
}

template <typename T>
int launch_dim(const Q8Args& a, int64_t dim, bool join, hipStream_t s) {
  switch (dim) {
    case 64: return launch<T, 64>(a, join, s);
    case 96: return launch<T, 96>(a, join, s);
    case 128: return launch<T, 128>(a, join, s);
    default: return launch<T, 256>(a, join, s);
  }
}

int check_q8(const char* name, const fpv2_quantized_decode_params* p) {
  if (p == nullptr) return fail(FPV2_ERR_ARGUMENT, "%s: null params", name);
  return check_params(name, &p->attention);
}

}  // namespace
}  // namespace fpv2

extern "C" int64_t fpv2_quantized_decode_attention_workspace_bytes(const fpv2_quantized_decode_params* params) {
  using namespace fpv2;
  if (const int rc = check_q8("fpv2_quantized_decode_attention", params)) return rc;
  return partial_bytes(params->attention, decode_plan(params->attention));
}

extern "C" int fpv2_quantized_decode_attention(const void* q, const void* k_codes, const float* k_scales,
                                               const void* v_codes, const float* v_scales,
                                               const int32_t* page_table, const int32_t* lengths, void* out,
                                               int dtype, const fpv2_quantized_decode_params* params,
                                               void* workspace, int64_t workspace_bytes, void* stream) {
  using namespace fpv2;
  const char* name = "fpv2_quantized_decode_attention";
  const auto a16 = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; };
  if (const int rc = check_q8(name, params)) return rc;
  const fpv2_decode_params& p = params->attention;
  if (dtype != FPV2_BF16 && dtype != FPV2_F16)
    return fail(FPV2_ERR_UNSUPPORTED, "%s: dtype must be bf16 or f16", name);
  if (p.batch == 0) return FPV2_OK;
  if (!q || !k_codes || !v_codes || !k_scales || !v_scales || !out)
    return fail(FPV2_ERR_ARGUMENT, "%s: null pointer", name);
  if (page_table == nullptr && (p.table_width != 1 || p.pages < p.batch))
    return fail(FPV2_ERR_ARGUMENT, "%s: without a page table every sequence has one page", name);
  if (page_table != nullptr && p.table_stride < 0)
    return fail(FPV2_ERR_ARGUMENT, "%s: table_stride must not be negative", name);
  if (p.q_batch_stride < 0 || p.q_batch_stride % 8 || p.q_head_stride < 0 || p.q_head_stride % 8)
    return fail(FPV2_ERR_ARGUMENT, "%s: strides of q must be multiples of 8", name);
  const int64_t strides[] = {p.k_page_stride, p.k_head_stride, p.k_row_stride,
                             p.v_page_stride, p.v_head_stride, p.v_row_stride};
  for (const int64_t x : strides)
    if (x < 0 || x % 16) return fail(FPV2_ERR_ARGUMENT, "%s: strides of codes must be multiples of 16", name);
  const int64_t rest[] = {params->ks_page_stride, params->ks_head_stride, params->ks_row_stride,
                          params->vs_page_stride, params->vs_head_stride, params->vs_row_stride,
                          p.o_batch_stride,       p.o_head_stride};
  for (const int64_t x : rest)
    if (x < 0) return fail(FPV2_ERR_ARGUMENT, "%s: strides of scales and output must not be negative", name);
  if (!a16(q) || !a16(k_codes) || !a16(v_codes))
    return fail(FPV2_ERR_ARGUMENT, "%s: q and the codes must be 16-byte aligned", name);
  const DecodePlan plan = decode_plan(p);
  const int64_t need = partial_bytes(p, plan);
  if (need > 0 && (workspace == nullptr || workspace_bytes < need || !a16(workspace)))
    return fail(FPV2_ERR_ARGUMENT, "%s: needs a 16-byte aligned workspace of %lld bytes", name,
                static_cast<long long>(need));
  Q8Args x{};
  DecodeArgs& a = x.a;
  a = decode_args(p, plan);
  a.q = static_cast<const uint16_t*>(q);
  a.k = static_cast<const uint16_t*>(k_codes);
  a.v = static_cast<const uint16_t*>(v_codes);
  a.out = static_cast<uint16_t*>(out);
  a.table = page_table;
  a.lengths = lengths;
  a.part_o = static_cast<float*>(workspace);
  a.part_ml = a.part_o + 2LL * plan.grid * plan.item_heads * p.head_dim;
  x.ks = k_scales;
  x.vs = v_scales;
  x.ks_ps = params->ks_page_stride;
  x.ks_hs = params->ks_head_stride;
  x.ks_rs = params->ks_row_stride;
  x.vs_ps = params->vs_page_stride;
  x.vs_hs = params->vs_head_stride;
  x.vs_rs = params->vs_row_stride;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  const bool join = plan.most_tiles > 1;
  return dtype == FPV2_BF16 ? launch_dim<bf16_t>(x, p.head_dim, join, s) : launch_dim<f16_t>(x, p.head_dim, join, s);
}
