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
// A step is 128 weights of a row, 32 on each quad of lanes, so a dot product over
// all lanes would mix 128 / group groups.  The A operand keeps them apart: its
// row m S + j (S = 128 / group) is x[m] with zeros outside the step's group j, so
// that P comes out per group.  16 / S rows of x make a tile.
//
// Waves of a workgroup take the steps of the same weight rows in turn and add
// their sums in LDS at the end.
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

// S: groups of a step of 128 weights; R: tiles of 16 weight rows and MT: tiles of
// 16 / S rows of x of a workgroup; W: its waves.
template <typename T, int S, int R, int MT, int W>
__global__ __launch_bounds__(64 * W) void q4_linear_kernel(Q4Args a) {
  constexpr int MP = 16 / S;  // rows of x of a tile
  constexpr int Y = 4 / S;    // of which in a lane
  __shared__ float sh[W][R * MT * Y][64];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 15, quad = lane >> 4;
  const int n0 = blockIdx.x * (16 * R);
  const int m0 = blockIdx.y * (MP * MT);
  const bool mine = col % S == quad * S / 4;  // the lane's weights are in its row's group

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
  const uint16_t* xp[MT];
#pragma unroll
  for (int t = 0; t < MT; ++t)
    xp[t] = a.x + static_cast<int64_t>(min(m0 + t * MP + col / S, a.rows - 1)) * a.x_rs;

  float y[R][MT][Y];
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
      for (int i = 0; i < Y; ++i) y[r][t][i] = 0.f;
  const u32x4 ones = {Nibbles<T>::kOnes, Nibbles<T>::kOnes, Nibbles<T>::kOnes, Nibbles<T>::kOnes};
  const f32x4 zero = {0.f, 0.f, 0.f, 0.f};

  const int steps = (a.k + 127) / 128;
  for (int step = wave; step < steps; step += W) {
    const int k0 = 128 * step + 32 * quad;  // the lane's 32 weights
    const bool in = k0 < a.k;
    const int kc = in ? k0 : a.k - 32;
    u32x4 w[R];
    float s[R][S], c[R][S];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      w[r] = load16(wp[r] + kc / 8);
#pragma unroll
      for (int j = 0; j < S; ++j) {
        const int g = step * S + j;
        s[r][j] = c[r][j] = 0.f;
        if (g < a.groups) {
          s[r][j] = Elem<T>::to_float(sp[r][g]);
          c[r][j] = Elem<T>::to_float(bp[r][g]) - 16.f * s[r][j];
        }
      }
    }
    u32x4 xv[MT][4];
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        xv[t][j] = u32x4{0, 0, 0, 0};
        if (mine && in) xv[t][j] = reorder(load16(xp[t] + k0 + 8 * j));
      }
    f32x4 xs[MT];
#pragma unroll
    for (int t = 0; t < MT; ++t) {
      xs[t] = zero;
#pragma unroll
      for (int j = 0; j < 4; ++j)
        xs[t] = Elem<T>::mfma16(as_vec8<T>(xv[t][j]), as_vec8<T>(ones), xs[t]);
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
      u32x4 wide[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) wide[j] = widen<T>(w[r][j]);
#pragma unroll
      for (int t = 0; t < MT; ++t) {
        f32x4 p = zero;
#pragma unroll
        for (int j = 0; j < 4; ++j)
          p = Elem<T>::mfma16(as_vec8<T>(xv[t][j]), as_vec8<T>(wide[j]), p);
        // row 4 quad + i of the tile: group i % S of x's row (4 quad + i) / S
#pragma unroll
        for (int i = 0; i < 4; ++i)
          y[r][t][i / S] = fmaf(s[r][i % S], p[i], fmaf(c[r][i % S], xs[t][i], y[r][t][i / S]));
      }
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
    const int m = m0 + t * MP + quad * Y + i;
    if (n < a.n && m < a.rows) {
      if (a.out_f32)
        static_cast<float*>(a.out)[m * a.o_rs + n] = sum;
      else
        static_cast<uint16_t*>(a.out)[m * a.o_rs + n] = Elem<T>::from_float(sum);
    }
  }
}

template <typename T, int S, int R, int MT>
void launch(const Q4Args& a, hipStream_t s) {
  constexpr int W = 8;
  const dim3 grid((a.n + 16 * R - 1) / (16 * R), (a.rows + 16 / S * MT - 1) / (16 / S * MT));
  hipLaunchKernelGGL((q4_linear_kernel<T, S, R, MT, W>), grid, dim3(64 * W), 0, s, a);
}

template <typename T, int S>
void launch_rows(const Q4Args& a, hipStream_t s) {
  const int tiles = (a.rows + 16 / S - 1) / (16 / S);
  const bool wide = a.n >= 32 * 2 * cu_count();
  if (tiles <= 1)
    wide ? launch<T, S, 2, 1>(a, s) : launch<T, S, 1, 1>(a, s);
  else if (tiles == 2)
    wide ? launch<T, S, 2, 2>(a, s) : launch<T, S, 1, 2>(a, s);
  else
    wide ? launch<T, S, 2, 4>(a, s) : launch<T, S, 1, 4>(a, s);
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
