// Products of a few rows with 4-bit weights (group scales and biases).
//
//   out[m][n] = sum_g ( s[n][g] sum_k q[n][k] x[m][k] + b[n][g] sum_k x[m][k] )
//
// Bound by reading the weights.  On MFMA, a tile of 16 weight rows as the B
// operand: a lane loads 16 bytes of a row (32 weights) as they lie, and two
// operations make two operands of a word's nibbles: (16 + q) in the storage
// type is a constant exponent with q in the top of the mantissa, exact in both
// types.  So
//   out = sum_g s P + (b - 16 s) X,  P = sum (16 + q) x,  X = sum x,
// with X from MFMA against ones.  (An offset of 16 instead of the smallest that
// bits allow keeps the cancellation of P against 16 X small: float32 outputs
// are good to 2^-22 or so.)
//
// A step is 128 weights of a row, 32 on each quad of lanes, which is at most a
// group's.  A product over all lanes would mix the quads' groups, so the quads first
// exchange words (four swaps of half waves and rows): then word j of a quad is its
// quarter of group j's 32 weights, and each product has one group.
//
// Waves of a workgroup take the steps of the same weight rows in turn and add
// their sums in LDS at the end; the next step's loads are in flight while one is
// computed.
#include "fpv2_common.h"
#include "fpv2_decode.h"

namespace fpv2 {
namespace {

struct Q4Args {
  const uint16_t* x;
  const uint32_t* packed;
  const uint16_t* scales;
  const uint16_t* biases;
  void* out;
  int rows, n, k, groups;
  int64_t x_rs, p_rs, s_rs, o_rs;
  int out_f32;
};

template <typename T> struct Nibbles;
template <> struct Nibbles<bf16_t> {
  static constexpr int kBit = 3;  // of the nibble in the operand: 16 (1 + q / 16)
  static constexpr uint32_t kMask = 0x00780078u, kBase = 0x41804180u, kOnes = 0x3f803f80u;
};
template <> struct Nibbles<f16_t> {
  static constexpr int kBit = 6;
  static constexpr uint32_t kMask = 0x03c003c0u, kBase = 0x4c004c00u, kOnes = 0x3c003c00u;
};

// (16 + q) of a word's nibbles, in the order 0 4 1 5 2 6 3 7.
template <typename T>
__device__ __forceinline__ u32x4 widen(uint32_t w) {
  u32x4 r;
#pragma unroll
  for (int p = 0; p < 4; ++p) {
    const int shift = 4 * p - Nibbles<T>::kBit;
    const uint32_t v = shift < 0 ? w << -shift : w >> shift;
    r[p] = (v & Nibbles<T>::kMask) | Nibbles<T>::kBase;
  }
  return r;
}
// 8 elements of x in the same order.
__device__ __forceinline__ u32x4 reorder(u32x4 d) {
  u32x4 r;
  r[0] = __builtin_amdgcn_perm(d[2], d[0], 0x05040100u);
  r[1] = __builtin_amdgcn_perm(d[2], d[0], 0x07060302u);
  r[2] = __builtin_amdgcn_perm(d[3], d[1], 0x05040100u);
  r[3] = __builtin_amdgcn_perm(d[3], d[1], 0x07060302u);
  return r;
}

// out[j] of quad q = in[q] of quad j.
__device__ __forceinline__ u32x4 exchange(u32x4 v) {
  const auto a = __builtin_amdgcn_permlane32_swap(v[0], v[2], false, false);
  const auto b = __builtin_amdgcn_permlane32_swap(v[1], v[3], false, false);
  const auto c = __builtin_amdgcn_permlane16_swap(a[0], b[0], false, false);
  const auto d = __builtin_amdgcn_permlane16_swap(a[1], b[1], false, false);
  return u32x4{c[0], c[1], d[0], d[1]};
}

// Scales (or biases) of a step's S groups: one load where they are all there and
// aligned.
template <int S, bool EVEN>
__device__ __forceinline__ void load_scales(const uint16_t* p, int g, int groups, uint16_t* out) {
  if constexpr (EVEN && S == 4) {
    const u32x2 v = *reinterpret_cast<const u32x2*>(p + g);
    out[0] = v[0] & 0xffffu, out[1] = v[0] >> 16, out[2] = v[1] & 0xffffu, out[3] = v[1] >> 16;
  } else if constexpr (EVEN && S == 2) {
    const uint32_t v = *reinterpret_cast<const uint32_t*>(p + g);
    out[0] = v & 0xffffu, out[1] = v >> 16;
  } else {
#pragma unroll
    for (int j = 0; j < S; ++j) out[j] = EVEN || g + j < groups ? p[g + j] : 0;
  }
}

// S: groups of a step of 128 weights; R: tiles of 16 weight rows, MT: tiles of 16
// rows of x of a workgroup, of whose rows 4 quad .. + Y - 1 are used; W: its waves.
// EVEN: the columns are whole steps, the scales aligned.
template <typename T, int S, int R, int MT, int Y, int W, bool EVEN>
__global__ __launch_bounds__(64 * W) void q4_linear_kernel(Q4Args a) {
  __shared__ float sh[W][R * MT * Y][64];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 15, quad = lane >> 4;
  const int n0 = blockIdx.x * (16 * R);
  const int m0 = blockIdx.y * (16 * MT);

  const uint32_t* wp[R];
  const uint16_t* sp[R];
  const uint16_t* bp[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int64_t n = min(n0 + 16 * r + col, a.n - 1);
    wp[r] = a.packed + n * a.p_rs;
    sp[r] = a.scales + n * a.s_rs;
    bp[r] = a.biases + n * a.s_rs;
  }
  const uint16_t* xp[MT];  // (rows past the last give results that are not used)
#pragma unroll
  for (int t = 0; t < MT; ++t)
    xp[t] = a.x + static_cast<int64_t>(min(m0 + 16 * t + col, a.rows - 1)) * a.x_rs + 8 * quad;

  float y[R][MT][Y];
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
      for (int i = 0; i < Y; ++i) y[r][t][i] = 0.f;
  const u32x4 ones = {Nibbles<T>::kOnes, Nibbles<T>::kOnes, Nibbles<T>::kOnes, Nibbles<T>::kOnes};
  const f32x4 zero = {0.f, 0.f, 0.f, 0.f};

  struct Stage {
    u32x4 w[R], x[MT][4];
    uint16_t s[R][S], b[R][S];
  };
  const auto load = [&](Stage& st, int step) {
    const int k0 = 128 * step + 32 * quad;
    const int kc = EVEN || k0 < a.k ? k0 : a.k - 32;
#pragma unroll
    for (int r = 0; r < R; ++r) {
      st.w[r] = load16(wp[r] + kc / 8);
      load_scales<S, EVEN>(sp[r], step * S, a.groups, st.s[r]);
      load_scales<S, EVEN>(bp[r], step * S, a.groups, st.b[r]);
    }
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int k = 128 * step + 32 * j;
        st.x[t][j] = EVEN || k < a.k ? load16(xp[t] + k) : u32x4{0, 0, 0, 0};
      }
  };
  const auto compute = [&](const Stage& st) {
    u32x4 xv[MT][4];
    f32x4 xs[MT][S];
#pragma unroll
    for (int t = 0; t < MT; ++t) {
#pragma unroll
      for (int g = 0; g < S; ++g) xs[t][g] = zero;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        xv[t][j] = reorder(st.x[t][j]);
        xs[t][j * S / 4] = Elem<T>::mfma16(as_vec8<T>(xv[t][j]), as_vec8<T>(ones), xs[t][j * S / 4]);
      }
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const u32x4 w = exchange(st.w[r]);
      u32x4 wide[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) wide[j] = widen<T>(w[j]);
      float s[S], c[S];
#pragma unroll
      for (int g = 0; g < S; ++g) {
        s[g] = Elem<T>::to_float(st.s[r][g]);
        c[g] = Elem<T>::to_float(st.b[r][g]) - 16.f * s[g];
      }
#pragma unroll
      for (int t = 0; t < MT; ++t) {
        f32x4 p[S];
#pragma unroll
        for (int g = 0; g < S; ++g) p[g] = zero;
#pragma unroll
        for (int j = 0; j < 4; ++j)
          p[j * S / 4] = Elem<T>::mfma16(as_vec8<T>(xv[t][j]), as_vec8<T>(wide[j]), p[j * S / 4]);
#pragma unroll
        for (int g = 0; g < S; ++g)
#pragma unroll
          for (int i = 0; i < Y; ++i)
            y[r][t][i] = fmaf(s[g], p[g][i], fmaf(c[g], xs[t][g][i], y[r][t][i]));
      }
    }
  };
  const int steps = (a.k + 127) / 128;
  if (wave < steps) {
    Stage st[2];
    load(st[0], wave);
    for (int step = wave; step < steps; step += 2 * W) {
      if (step + W < steps) load(st[1], step + W);
      compute(st[0]);
      if (step + W >= steps) break;
      if (step + 2 * W < steps) load(st[0], step + 2 * W);
      compute(st[1]);
    }
  }
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
      for (int i = 0; i < Y; ++i) sh[wave][(r * MT + t) * Y + i][lane] = y[r][t][i];
  __syncthreads();
  for (int e = wave; e < R * MT * Y; e += W) {
    float sum = 0.f;
#pragma unroll
    for (int w = 0; w < W; ++w) sum += sh[w][e][lane];
    const int i = e % Y, t = e / Y % MT, r = e / (Y * MT);
    const int n = n0 + 16 * r + col;
    const int m = m0 + 16 * t + 4 * quad + i;
    if (n < a.n && m < a.rows) {
      if (a.out_f32)
        static_cast<float*>(a.out)[m * a.o_rs + n] = sum;
      else
        static_cast<uint16_t*>(a.out)[m * a.o_rs + n] = Elem<T>::from_float(sum);
    }
  }
}

template <typename T, int S, int R, int MT, int Y, int W>
void launch(const Q4Args& a, hipStream_t s) {
  const dim3 grid((a.n + 16 * R - 1) / (16 * R), (a.rows + 16 * MT - 1) / (16 * MT));
  const auto aligned = [](const void* p) { return reinterpret_cast<uintptr_t>(p) % (2 * S) == 0; };
  if (a.k % 128 == 0 && a.s_rs % S == 0 && aligned(a.scales) && aligned(a.biases))
    hipLaunchKernelGGL((q4_linear_kernel<T, S, R, MT, Y, W, true>), grid, dim3(64 * W), 0, s, a);
  else
    hipLaunchKernelGGL((q4_linear_kernel<T, S, R, MT, Y, W, false>), grid, dim3(64 * W), 0, s, a);
}

template <typename T, int S>
void launch_rows(const Q4Args& a, hipStream_t s) {
  const bool wide = a.n >= 256 * cu_count();
  const bool few = a.n <= 16 * cu_count();
  if (a.rows == 1)
    wide ? launch<T, S, 2, 1, 1, 4>(a, s) : few ? launch<T, S, 1, 1, 1, 16>(a, s) : launch<T, S, 1, 1, 1, 8>(a, s);
  else if (a.rows <= 16)
    wide ? launch<T, S, 2, 1, 4, 4>(a, s) : few ? launch<T, S, 1, 1, 4, 16>(a, s) : launch<T, S, 1, 1, 4, 8>(a, s);
  else
    wide ? launch<T, S, 2, 2, 4, 4>(a, s) : launch<T, S, 1, 2, 4, 8>(a, s);
}

template <typename T>
void launch_group(const Q4Args& a, int64_t group, hipStream_t s) {
  if (group == 32)
    launch_rows<T, 4>(a, s);
  else if (group == 64)
    launch_rows<T, 2>(a, s);
  else
    launch_rows<T, 1>(a, s);
}

}  // namespace
}  // namespace fpv2

extern "C" int fpv2_quantized_linear(const void* x, const void* packed, const void* scales,
                                     const void* biases, void* out, int dtype, int out_dtype,
                                     int64_t rows, int64_t out_cols, int64_t cols, int64_t group,
                                     int64_t x_row_stride, int64_t packed_row_stride,
                                     int64_t scale_row_stride, int64_t out_row_stride,
                                     void* stream) {
  using namespace fpv2;
  const char* name = "fpv2_quantized_linear";
  const auto a16 = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; };
  if (dtype != FPV2_BF16 && dtype != FPV2_F16)
    return fail(FPV2_ERR_UNSUPPORTED, "%s: dtype must be bf16 or f16", name);
  if (out_dtype != dtype && out_dtype != FPV2_F32)
    return fail(FPV2_ERR_UNSUPPORTED, "%s: out_dtype must be dtype or float32", name);
  if (group != 32 && group != 64 && group != 128)
    return fail(FPV2_ERR_UNSUPPORTED, "%s: group must be 32, 64 or 128", name);
  if (rows < 0 || out_cols < 0 || cols <= 0 || cols % group || cols > (1 << 28) ||
      out_cols > (1 << 28) || rows > (1 << 18))
    return fail(FPV2_ERR_ARGUMENT, "%s: cols must be a positive multiple of group; at most 2^28 "
                "columns and 2^18 rows", name);
  if (rows == 0 || out_cols == 0) return FPV2_OK;
  if (!x || !packed || !scales || !biases || !out)
    return fail(FPV2_ERR_ARGUMENT, "%s: null pointer", name);
  if (x_row_stride % 8 || packed_row_stride % 4 || x_row_stride < 0 || packed_row_stride < 0 ||
      scale_row_stride < 0 || out_row_stride < 0 || (rows > 1 && x_row_stride < cols) ||
      (rows > 1 && out_row_stride < out_cols) ||
      (out_cols > 1 && (packed_row_stride < cols / 8 || scale_row_stride < cols / group)))
    return fail(FPV2_ERR_ARGUMENT, "%s: rows must not overlap, x_row_stride be a multiple of 8 and "
                "packed_row_stride of 4", name);
  if (!a16(x) || !a16(packed))
    return fail(FPV2_ERR_ARGUMENT, "%s: x and packed must be 16-byte aligned", name);
  Q4Args a{static_cast<const uint16_t*>(x), static_cast<const uint32_t*>(packed),
           static_cast<const uint16_t*>(scales), static_cast<const uint16_t*>(biases), out,
           static_cast<int>(rows), static_cast<int>(out_cols), static_cast<int>(cols),
           static_cast<int>(cols / group), x_row_stride, packed_row_stride, scale_row_stride,
           out_row_stride, out_dtype == FPV2_F32};
  const hipStream_t s = static_cast<hipStream_t>(stream);
  if (dtype == FPV2_BF16)
    launch_group<bf16_t>(a, group, s);
  else
    launch_group<f16_t>(a, group, s);
  return check_launch("q4_linear_kernel");
}
