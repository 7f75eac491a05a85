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
// Waves of a workgroup take pairs of steps of the same weight rows in turn and add
// their sums in LDS at the end; the next pair's weights are in flight while one is
// computed.  x lies in LDS, in the order of the operands: loaded from memory by
// every wave, it kept the address units busier than the weights did.
//
// Measured: 151936 x 2560, groups of 128, 3 rows 50 us (4.2 TB/s); 19456 x 2560, groups of
// 32, 12 rows of float16 15 us (2.1 TB/s); 2560 x 9728, groups of 64, one row 8.1 us (1.7
// TB/s: a launch, x, two turns of loads and the sum), 16 rows 14, 64 rows 31 us.  Without
// gain: two or three pairs in flight (8.8 and 9.6 us for one row), 16 waves, two rows'
// tiles a wave; weights loaded 128 bytes of a row at a time would give 5 %.
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
  int wn;     // tiles of weight rows of a workgroup, each its own waves'
  int panel;  // pairs of steps whose x lies in LDS at a time
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

// (16 + q) of a word's nibbles, in the order 0 4 1 5 2 6 3 7; base: kBase, in a vector
// register, so that masking and joining are one instruction.
template <typename T>
__device__ __forceinline__ u32x4 widen(uint32_t w, uint32_t base) {
  u32x4 r;
#pragma unroll
  for (int p = 0; p < 4; ++p) {
    const int shift = 4 * p - Nibbles<T>::kBit;
    const uint32_t v = shift < 0 ? w << -shift : w >> shift;
    r[p] = (v & Nibbles<T>::kMask) | base;
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

// N scales (or biases) from group g on: one load where they are all there and aligned.
template <int N, bool EVEN>
__device__ __forceinline__ void load_scales(const uint16_t* p, int g, int groups, uint16_t* out) {
  if constexpr (EVEN) {
    uint32_t v[N / 2];
    if constexpr (N == 8) {
      const u32x4 x = load16(p + g);
      v[0] = x[0], v[1] = x[1], v[2] = x[2], v[3] = x[3];
    } else if constexpr (N == 4) {
      const u32x2 x = *reinterpret_cast<const u32x2*>(p + g);
      v[0] = x[0], v[1] = x[1];
    } else {
      v[0] = *reinterpret_cast<const uint32_t*>(p + g);
    }
#pragma unroll
    for (int j = 0; j < N; ++j) out[j] = j % 2 ? v[j / 2] >> 16 : v[j / 2] & 0xffffu;
  } else {
#pragma unroll
    for (int j = 0; j < N; ++j) out[j] = g + j < groups ? p[g + j] : 0;
  }
}

constexpr int W = 8;  // waves of a workgroup

// S: groups of a step of 128 weights; M: rows of x of a workgroup (1, 4 or a number of
// tiles of 16).  EVEN: the columns are whole pairs of steps, the scales aligned.
template <typename T, int S, int M, bool EVEN>
__global__ __launch_bounds__(64 * W) void q4_linear_kernel(Q4Args a) {
  constexpr int MT = (M + 15) / 16;  // tiles of rows of x,
  constexpr int MR = M < 16 ? M : 16;  // of so many rows,
  // of x in flight in a thread (19456 x 2560, 12 rows: 1 17.7, 5 16.5, 10, whose registers leave
  // three waves a SIMD, 19.1 us)
  constexpr int LOADS = M < 16 ? 1 : 5;
  constexpr int Y = M < 4 ? M : 4;   // of which rows 4 quad .. + Y - 1 in a lane
  extern __shared__ __attribute__((aligned(16))) char sh[];
  // [panel * 8][MT][4 quads][MR] of 8 columns.  Lanes that write a row's next 8 columns would
  // meet in a bank: 16 rows lie turned by the columns' number.
  u32x4* sh_x = reinterpret_cast<u32x4*>(sh);
  const auto place = [](int m, int at) { return MR == 16 ? (m + at) % 8 + (m & 8) : m; };
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 15, quad = lane >> 4;
  const int wk = W / a.wn, wave_n = wave / wk, wave_k = wave - wave_n * wk;
  const int n = (blockIdx.x * a.wn + wave_n) * 16 + col;  // the lane's weight row
  const int m0 = blockIdx.y * M;

  const int64_t row = min(n, a.n - 1);
  const uint32_t* wp = a.packed + row * a.p_rs;
  const uint16_t* sp = a.scales + row * a.s_rs;
  const uint16_t* bp = a.biases + row * a.s_rs;
  float y[MT][Y];
#pragma unroll
  for (int t = 0; t < MT; ++t)
#pragma unroll
    for (int i = 0; i < Y; ++i) y[t][i] = 0.f;
  const int x_at[2] = {place(min(col, MR - 1), quad), place(min(col, MR - 1), 4 + quad)};
  const u32x4 ones = {Nibbles<T>::kOnes, Nibbles<T>::kOnes, Nibbles<T>::kOnes, Nibbles<T>::kOnes};
  const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
  uint32_t base = Nibbles<T>::kBase;
  asm("" : "+v"(base));

  struct Stage {
    u32x4 w[2];
    uint16_t s[2 * S], b[2 * S];
  };
  const auto load = [&](Stage& st, int pair) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int k0 = 256 * pair + 128 * h + 32 * quad;
      st.w[h] = load16(wp + (EVEN || k0 < a.k ? k0 : a.k - 32) / 8);
    }
    load_scales<2 * S, EVEN>(sp, pair * 2 * S, a.groups, st.s);
    load_scales<2 * S, EVEN>(bp, pair * 2 * S, a.groups, st.b);
  };
  // (rows of x past the last are copies of it, columns past the last zeros)
  const auto compute = [&](const Stage& st, int at) {  // at: the pair's place in the panel
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const u32x4 w = exchange(st.w[h]);
      u32x4 wide[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) wide[j] = widen<T>(w[j], base);
#pragma unroll
      for (int t = 0; t < MT; ++t) {
        f32x4 xs[S], p[S];
#pragma unroll
        for (int g = 0; g < S; ++g) xs[g] = p[g] = zero;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const u32x4 x = sh_x[(((8 * at + 4 * h + j) * MT + t) * 4 + quad) * MR + x_at[j % 2]];
          xs[j * S / 4] = Elem<T>::mfma16(as_vec8<T>(x), as_vec8<T>(ones), xs[j * S / 4]);
          p[j * S / 4] = Elem<T>::mfma16(as_vec8<T>(x), as_vec8<T>(wide[j]), p[j * S / 4]);
        }
#pragma unroll
        for (int g = 0; g < S; ++g) {
          const float s = Elem<T>::to_float(st.s[S * h + g]);
          const float c = fmaf(-16.f, s, Elem<T>::to_float(st.b[S * h + g]));
#pragma unroll
          for (int i = 0; i < Y; ++i) y[t][i] = fmaf(s, p[g][i], fmaf(c, xs[g][i], y[t][i]));
        }
      }
    }
  };
  const int pairs = (a.k + 255) / 256;
  Stage st[2];
  if (wave_k < pairs) load(st[0], wave_k);
  for (int p0 = 0; p0 < pairs; p0 += a.panel) {
    const int p1 = min(pairs, p0 + a.panel);
    if (p0 > 0) __syncthreads();
    for (int e0 = tid; e0 < (p1 - p0) * (32 * M); e0 += 64 * W * LOADS) {
      u32x4 v[LOADS];
#pragma unroll
      for (int i = 0; i < LOADS; ++i) {
        // (8 lanes read 128 bytes of a row)
        const int e = e0 + i * 64 * W;
        const int m = e / 8 % MR, t = e / (8 * MR) % MT, at = e / (8 * MR * MT) * 8 + e % 8;
        const int k = 256 * p0 + 8 * at;
        v[i] = u32x4{0, 0, 0, 0};
        if (e < (p1 - p0) * (32 * M) && (EVEN || k < a.k))
          v[i] = load16(a.x + static_cast<int64_t>(min(m0 + 16 * t + m, a.rows - 1)) * a.x_rs + k);
      }
#pragma unroll
      for (int i = 0; i < LOADS; ++i) {
        const int e = e0 + i * 64 * W;
        const int m = e / 8 % MR, t = e / (8 * MR) % MT, at = e / (8 * MR * MT) * 8 + e % 8;
        if (e < (p1 - p0) * (32 * M)) sh_x[((at / 4 * MT + t) * 4 + at % 4) * MR + place(m, at)] = reorder(v[i]);
      }
    }
    __syncthreads();
    // the wave's first pair of the panel is in st[0] already
    for (int pair = p0 + (wave_k - p0 % wk + wk) % wk; pair < p1; pair += 2 * wk) {
      if (pair + wk < pairs) load(st[1], pair + wk);
      compute(st[0], pair - p0);
      if (pair + wk >= p1) {
        st[0] = st[1];
        break;
      }
      if (pair + 2 * wk < pairs) load(st[0], pair + 2 * wk);
      compute(st[1], pair + wk - p0);
    }
  }
  __syncthreads();
  float(*sum)[MT * Y][64] = reinterpret_cast<float(*)[MT * Y][64]>(sh);
#pragma unroll
  for (int t = 0; t < MT; ++t)
#pragma unroll
    for (int i = 0; i < Y; ++i) sum[wave][t * Y + i][lane] = y[t][i];
  __syncthreads();
  for (int e = wave_k; e < MT * Y; e += wk) {
    float v = 0.f;
    for (int w = 0; w < wk; ++w) v += sum[wave_n * wk + w][e][lane];
    const int i = e % Y, t = e / Y, x_row = 4 * quad + i, m = m0 + 16 * t + x_row;
    if (n < a.n && x_row < MR && m < a.rows) {
      if (a.out_f32)
        static_cast<float*>(a.out)[m * a.o_rs + n] = v;
      else
        static_cast<uint16_t*>(a.out)[m * a.o_rs + n] = Elem<T>::from_float(v);
    }
  }
}

constexpr int kPanelBytes = 81920;  // of x in LDS at most where two workgroups share a CU

template <typename T, int S, int M>
void launch(Q4Args a, hipStream_t s) {
  constexpr int kSum = W * ((M + 15) / 16) * (M < 4 ? M : 4) * 256;
  const int tiles = (a.n + 15) / 16, many = (a.rows + M - 1) / M;
  // A workgroup reads M rows of x and 16 wn rows of weights, so wn pays in x's reads
  // and costs in workgroups.  Microseconds for wn = 1 / 2 / 4 / 8, one row: 19456 x 2560 10.4 /
  // 10.3 / 11.5 / 12.9, 151936 x 2560 61.5 / 48.5 / 46.1 / 51.0, 6144 x 2560 5.9 / 6.6 / 8.1 / 12.4; 3
  // rows: 151936 x 2560 86 / 65 / 56 / 49.5; 4 rows: 9728 x 2560 10.7 / 9.9 / 9.1 / 14.0.
  // From 5 rows on x fills the LDS, and a workgroup alone on its CU has twice as much of it:
  // the fewest that make the workgroups no more than the CUs, but two a CU rather than
  // all waves with rows of their own.  wn = 1 / 2, 16 rows: 6144 x 2560 8.6 / 7.8, 4096 x 4096
  // 8.5 / 10.1; 2 / 4: 10240 x 5120 19.2 / 16.7; 4 / 8: 19456 x 2560, 12 rows 16.4 / 17.4.
  const auto grid_of = [&](int wn) { return (tiles + wn - 1) / wn * many; };
  a.wn = 1;
  if (M < 16) {
    const int least = M == 1 ? 8 * cu_count() : cu_count() / 2;
    while (a.wn < W && tiles / (2 * a.wn) * many >= least) a.wn *= 2;
  } else {
    while (a.wn < W && grid_of(a.wn) > (a.wn == 4 ? 2 : 1) * cu_count()) a.wn *= 2;
  }
  const int pairs = (a.k + 255) / 256;
  const bool alone = grid_of(a.wn) <= cu_count();
  const int most = (alone ? 2 : 1) * kPanelBytes / (512 * M);
  a.panel = pairs < most ? pairs : most;
  const int bytes = a.panel * 512 * M > kSum ? a.panel * 512 * M : kSum;
  const dim3 grid((tiles + a.wn - 1) / a.wn, many);
  // Whole pairs of steps with aligned scales load these as vectors, others one by one and
  // with a condition each.  The same products with aligned scales / with scales moved by an
  // element, 8192 x 2816, groups of 32: one row 6.8 / 11.1, 4 rows 11.0 / 19.1, 32 rows 15.1 / 18.1
  // us, groups of 128: 6.2 / 6.5, 9.7 / 10.9, 13.2 / 13.9; 19456 x 2560 in float16, 12 rows,
  // groups of 32 17.2 / 49.8 (143 registers against 127: a workgroup a CU instead of two),
  // of 64 15.7 / 20.5.  Columns that are no multiple of 256 pay the same: 8192 x 2880, groups
  // of 32, one row 10.5.
  const auto aligned = [](const void* p) { return reinterpret_cast<uintptr_t>(p) % (4 * S) == 0; };
  if (a.k % 256 == 0 && a.s_rs % (2 * S) == 0 && aligned(a.scales) && aligned(a.biases))
    hipLaunchKernelGGL((q4_linear_kernel<T, S, M, true>), grid, dim3(64 * W), bytes, s, a);
  else
    hipLaunchKernelGGL((q4_linear_kernel<T, S, M, false>), grid, dim3(64 * W), bytes, s, a);
}

template <typename T, int S>
void launch_rows(const Q4Args& a, hipStream_t s) {
  if (a.rows == 1)
    launch<T, S, 1>(a, s);
  else if (a.rows <= 4)
    launch<T, S, 4>(a, s);
  else if (a.rows <= 16)
    launch<T, S, 16>(a, s);
  else
    launch<T, S, 32>(a, s);
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
