// Keys and values as 8-bit codes in pages: writing tokens and reading them back.
//
//   a = max_j |x_j|,  code_j = rint(127 x_j / a),  scale = a / 127;  x_j ~ code_j scale
//
// for each row of a head.  Equal steps of a / 127 are off by at most a / 254, 0.23 % of a
// in the mean square; an 8-bit float of 3 fraction bits rounds each value by up to a 16th of it.
//
// 127 x is exact in float32 (bf16 and f16 have 8 and 11 bits), and half way between two
// codes (x = a / 2 is) means 127 x / a is so exactly, so the quotients have to be rounded
// correctly: with y = 1 / a rounded, q = n y, q + (n - q a) y is (a is not all ones).
//
// Both are bound by memory: 3 bytes a value.
#include "fpv2_batch.h"
#include "fpv2_common.h"

namespace fpv2 {
namespace {

typedef int i32x2 __attribute__((ext_vector_type(2)));

struct QuantArgs {
  const uint16_t* x[2];   // k, v
  int8_t* codes[2];
  float* scales[2];
  const void* slots;
  int64_t x_ts[2], x_hs[2];
  int64_t c_ps[2], c_hs[2], c_rs[2];
  int64_t s_ps[2], s_hs[2], s_rs[2];
  int64_t first_slot, pages, page_size, rows;  // rows: tokens * kv_heads
  int slot_bytes, kv_heads;
};

// One group of lanes a row, 8 values a lane.
template <typename T, int D>
__global__ __launch_bounds__(256) void quantize_kernel(QuantArgs a) {
  constexpr int kLanes = D / 8 <= 8 ? 8 : D / 8 <= 16 ? 16 : 32;
  const int tid = threadIdx.x, at = tid % kLanes;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * (256 / kLanes) + tid / kLanes;
  const int side = blockIdx.y;
  const bool live = row < a.rows && 8 * at < D;
  const int64_t t = row / a.kv_heads;
  const int h = static_cast<int>(row - t * a.kv_heads);
  u32x4 w = {0, 0, 0, 0};
  int64_t slot = -1;
  if (live) {
    w = load16(a.x[side] + t * a.x_ts[side] + h * a.x_hs[side] + 8 * at);
    slot = a.slot_bytes == 8   ? static_cast<const int64_t*>(a.slots)[t]
           : a.slot_bytes == 4 ? static_cast<const int32_t*>(a.slots)[t]
                               : a.first_slot + t;
  }
  float x[8], top = 0.f;
  uint32_t bad = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    x[j] = Elem<T>::to_float(static_cast<uint16_t>(w[j / 2] >> (16 * (j % 2))));
    const float size = __builtin_fabsf(x[j]);
    bad |= !(size <= 3.402823466e38f);
    top = fmaxf(top, size);
  }
#pragma unroll
  for (int off = kLanes / 2; off >= 1; off >>= 1) {
    top = fmaxf(top, __shfl_xor(top, off, 64));
    bad |= __shfl_xor(bad, off, 64);
  }
  if (!live || slot < 0 || slot >= a.pages * a.page_size) return;
  // (the quotients are the same for rows of tiny or huge values times a power of two)
  const float up = top < 0x1p-64f ? 0x1p64f : top > 0x1p64f ? 0x1p-64f : 1.f;
  const float most = top * up;
  const float y = 1.f / most;
  uint32_t code[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float n = 127.f * (x[j] * up);
    float q = n * y;
    q = __builtin_fmaf(__builtin_fmaf(-q, most, n), y, q);
    code[j] = top == 0.f || bad ? 0 : static_cast<uint32_t>(static_cast<int>(__builtin_rintf(q)));
  }
  i32x2 out;
#pragma unroll
  for (int i = 0; i < 2; ++i)
    out[i] = static_cast<int>((code[4 * i] & 255) | (code[4 * i + 1] & 255) << 8 | (code[4 * i + 2] & 255) << 16 |
                              code[4 * i + 3] << 24);
  const int64_t page = slot / a.page_size, r = slot - page * a.page_size;
  *reinterpret_cast<i32x2*>(a.codes[side] + page * a.c_ps[side] + h * a.c_hs[side] + r * a.c_rs[side] + 8 * at) = out;
  if (at == 0)
    a.scales[side][page * a.s_ps[side] + h * a.s_hs[side] + r * a.s_rs[side]] =
        bad ? __builtin_nanf("") : top / 127.f;
}

struct ReadArgs {
  const int8_t* codes[2];
  const float* scales[2];
  uint16_t* out[2];
  const int32_t* table;
  const int32_t* lengths;
  int64_t c_ps[2], c_hs[2], c_rs[2];
  int64_t s_ps[2], s_hs[2], s_rs[2];
  int64_t o_bs[2], o_hs[2], o_rs[2];
  int64_t table_stride;
  int kv_heads, pages, page_size, capacity, length, tokens, zero_rest;
};

// 16 values a lane, a row's chunks next to one another; blocks: (tokens, sequence * head, side).
template <typename T, int D>
__global__ __launch_bounds__(256) void dequantize_kernel(ReadArgs a) {
  constexpr int kChunks = D / 16;
  const int64_t e = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  const int64_t t = e / kChunks;
  const int c = static_cast<int>(e - t * kChunks), side = blockIdx.z;
  const int b = blockIdx.y / a.kv_heads, h = blockIdx.y - b * a.kv_heads;
  if (t >= a.tokens) return;
  int len = a.lengths != nullptr ? a.lengths[b] : a.length;
  len = min(max(len, 0), a.capacity);
  uint16_t* out = a.out[side] + b * a.o_bs[side] + h * a.o_hs[side] + t * a.o_rs[side] + 16 * c;
  if (t >= len) {
    if (a.zero_rest) {
      store16(out, u32x4{0, 0, 0, 0});
      store16(out + 8, u32x4{0, 0, 0, 0});
    }
    return;
  }
  const int at = static_cast<int>(t) / a.page_size, r = static_cast<int>(t) - at * a.page_size;
  const int id = a.table != nullptr ? a.table[b * a.table_stride + at] : b;
  const int64_t page = min(max(id, 0), a.pages - 1);
  const u32x4 w = load16(a.codes[side] + page * a.c_ps[side] + h * a.c_hs[side] + r * a.c_rs[side] + 16 * c);
  const float scale = a.scales[side][page * a.s_ps[side] + h * a.s_hs[side] + r * a.s_rs[side]];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    u32x4 v;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int word = static_cast<int>(w[2 * i + j / 2]) >> (16 * (j % 2));
      v[j] = pack2<T>(static_cast<float>(static_cast<int8_t>(word)) * scale,
                      static_cast<float>(static_cast<int8_t>(word >> 8)) * scale);
    }
    store16(out + 8 * i, v);
  }
}

int check_cache(const char* name, const fpv2_code_pages& c) {
  if (c.kv_heads <= 0 || c.kv_heads > 0xffff)
    return fail(FPV2_ERR_ARGUMENT, "%s: kv_heads must be 1 to 65535", name);
  if (c.head_dim != 64 && c.head_dim != 96 && c.head_dim != 128 && c.head_dim != 256)
    return fail(FPV2_ERR_UNSUPPORTED, "%s: head_dim must be 64, 96, 128 or 256", name);
  if (c.pages <= 0 || c.page_size <= 0 || c.pages > 0x7fffffff || c.page_size > 0x3fffffff)
    return fail(FPV2_ERR_ARGUMENT, "%s: pages and page_size must be positive", name);
  const int64_t bytes[] = {c.k_page_stride, c.k_head_stride, c.k_row_stride,
                           c.v_page_stride, c.v_head_stride, c.v_row_stride};
  for (const int64_t x : bytes)
    if (x < 0 || x % 16) return fail(FPV2_ERR_ARGUMENT, "%s: strides of codes must be multiples of 16", name);
  const int64_t scales[] = {c.ks_page_stride, c.ks_head_stride, c.ks_row_stride,
                            c.vs_page_stride, c.vs_head_stride, c.vs_row_stride};
  for (const int64_t x : scales)
    if (x < 0) return fail(FPV2_ERR_ARGUMENT, "%s: strides of scales must not be negative", name);
  return FPV2_OK;
}

bool a16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

template <typename A>
void set_cache(A* a, const fpv2_code_pages& c) {
  a->c_ps[0] = c.k_page_stride, a->c_hs[0] = c.k_head_stride, a->c_rs[0] = c.k_row_stride;
  a->c_ps[1] = c.v_page_stride, a->c_hs[1] = c.v_head_stride, a->c_rs[1] = c.v_row_stride;
  a->s_ps[0] = c.ks_page_stride, a->s_hs[0] = c.ks_head_stride, a->s_rs[0] = c.ks_row_stride;
  a->s_ps[1] = c.vs_page_stride, a->s_hs[1] = c.vs_head_stride, a->s_rs[1] = c.vs_row_stride;
}

template <typename T, int D>
int launch_quantize(const QuantArgs& a, hipStream_t s) {
  constexpr int kRows = 256 / (D / 8 <= 8 ? 8 : D / 8 <= 16 ? 16 : 32);
  hipLaunchKernelGGL((quantize_kernel<T, D>), dim3(static_cast<unsigned>((a.rows + kRows - 1) / kRows), 2), dim3(256),
                     0, s, a);
  return check_launch("quantize_kernel");
}

template <typename T, int D>
int launch_dequantize(const ReadArgs& a, int batch, hipStream_t s) {
  const int64_t blocks = (static_cast<int64_t>(a.tokens) * (D / 16) + 255) / 256;
  hipLaunchKernelGGL((dequantize_kernel<T, D>),
                     dim3(static_cast<unsigned>(blocks), static_cast<unsigned>(batch) * a.kv_heads, 2), dim3(256), 0, s, a);
  return check_launch("dequantize_kernel");
}

template <typename T>
int quantize_dim(const QuantArgs& a, int64_t dim, hipStream_t s) {
  switch (dim) {
    case 64: return launch_quantize<T, 64>(a, s);
    case 96: return launch_quantize<T, 96>(a, s);
    case 128: return launch_quantize<T, 128>(a, s);
    default: return launch_quantize<T, 256>(a, s);
  }
}

template <typename T>
int dequantize_dim(const ReadArgs& a, int batch, int64_t dim, hipStream_t s) {
  switch (dim) {
    case 64: return launch_dequantize<T, 64>(a, batch, s);
    case 96: return launch_dequantize<T, 96>(a, batch, s);
    case 128: return launch_dequantize<T, 128>(a, batch, s);
    default: return launch_dequantize<T, 256>(a, batch, s);
  }
}

}  // namespace
}  // namespace fpv2

extern "C" int fpv2_quantize_to_pages(const void* k, const void* v, const void* slots, void* k_codes,
                                      float* k_scales, void* v_codes, float* v_scales, int dtype,
                                      const fpv2_quantize_params* params, void* stream) {
  using namespace fpv2;
  const char* name = "fpv2_quantize_to_pages";
  if (params == nullptr) return fail(FPV2_ERR_ARGUMENT, "%s: null params", name);
  const fpv2_quantize_params& p = *params;
  if (const int rc = check_cache(name, p.cache)) return rc;
  if (dtype != FPV2_BF16 && dtype != FPV2_F16)
    return fail(FPV2_ERR_UNSUPPORTED, "%s: dtype must be bf16 or f16", name);
  if (p.tokens < 0 || p.tokens > 0x7fffffff / p.cache.kv_heads)
    return fail(FPV2_ERR_ARGUMENT, "%s: tokens * kv_heads must be 0 to 2^31 - 1", name);
  if (p.slot_bytes != 0 && p.slot_bytes != 4 && p.slot_bytes != 8)
    return fail(FPV2_ERR_ARGUMENT, "%s: slot_bytes must be 0, 4 or 8", name);
  const int64_t strides[] = {p.k_token_stride, p.k_head_stride, p.v_token_stride, p.v_head_stride};
  for (const int64_t x : strides)
    if (x < 0 || x % 8) return fail(FPV2_ERR_ARGUMENT, "%s: strides of k and v must be multiples of 8", name);
  if (p.slot_bytes == 0 && (p.first_slot < 0 || p.first_slot > (1LL << 62)))
    return fail(FPV2_ERR_ARGUMENT, "%s: first_slot must be 0 to 2^62", name);
  if (p.tokens == 0) return FPV2_OK;
  if (!k || !v || !k_codes || !v_codes || !k_scales || !v_scales || (p.slot_bytes != 0 && !slots))
    return fail(FPV2_ERR_ARGUMENT, "%s: null pointer", name);
  if (!a16(k) || !a16(v) || !a16(k_codes) || !a16(v_codes))
    return fail(FPV2_ERR_ARGUMENT, "%s: k, v and the codes must be 16-byte aligned", name);
  QuantArgs a{};
  set_cache(&a, p.cache);
  a.x[0] = static_cast<const uint16_t*>(k), a.x[1] = static_cast<const uint16_t*>(v);
  a.codes[0] = static_cast<int8_t*>(k_codes), a.codes[1] = static_cast<int8_t*>(v_codes);
  a.scales[0] = k_scales, a.scales[1] = v_scales;
  a.slots = slots;
  a.x_ts[0] = p.k_token_stride, a.x_hs[0] = p.k_head_stride;
  a.x_ts[1] = p.v_token_stride, a.x_hs[1] = p.v_head_stride;
  a.first_slot = p.first_slot;
  a.pages = p.cache.pages;
  a.page_size = p.cache.page_size;
  a.rows = p.tokens * p.cache.kv_heads;
  a.slot_bytes = static_cast<int>(p.slot_bytes);
  a.kv_heads = static_cast<int>(p.cache.kv_heads);
  const hipStream_t s = static_cast<hipStream_t>(stream);
  return dtype == FPV2_BF16 ? quantize_dim<bf16_t>(a, p.cache.head_dim, s) : quantize_dim<f16_t>(a, p.cache.head_dim, s);
}

extern "C" int fpv2_dequantize_pages(const void* k_codes, const float* k_scales, const void* v_codes,
                                     const float* v_scales, const int32_t* page_table,
                                     const int32_t* lengths, void* k_out, void* v_out, int dtype,
                                     const fpv2_dequantize_params* params, void* stream) {
  using namespace fpv2;
  const char* name = "fpv2_dequantize_pages";
  if (params == nullptr) return fail(FPV2_ERR_ARGUMENT, "%s: null params", name);
  const fpv2_dequantize_params& p = *params;
  if (const int rc = check_cache(name, p.cache)) return rc;
  if (dtype != FPV2_BF16 && dtype != FPV2_F16)
    return fail(FPV2_ERR_UNSUPPORTED, "%s: dtype must be bf16 or f16", name);
  if (p.batch < 0 || p.batch * p.cache.kv_heads > 0xffff)
    return fail(FPV2_ERR_UNSUPPORTED, "%s: batch * kv_heads must be 0 to 65535", name);
  if (p.table_width <= 0 || p.table_width > 0x3fffffff || p.table_width * p.cache.page_size > 0x3fffffff)
    return fail(FPV2_ERR_ARGUMENT, "%s: table_width must be positive and a sequence's pages hold fewer than "
                "2^30 tokens", name);
  if (p.length < 0 || p.tokens < 0 || p.tokens > 0x3fffffff || p.table_stride < 0)
    return fail(FPV2_ERR_ARGUMENT, "%s: length, tokens and table_stride must not be negative, tokens below 2^30", name);
  const int64_t strides[] = {p.k_batch_stride, p.k_head_stride, p.k_row_stride,
                             p.v_batch_stride, p.v_head_stride, p.v_row_stride};
  for (const int64_t x : strides)
    if (x < 0 || x % 8) return fail(FPV2_ERR_ARGUMENT, "%s: strides of the results must be multiples of 8", name);
  if (p.batch == 0 || p.tokens == 0) return FPV2_OK;
  if (!k_out || !v_out || !k_codes || !v_codes || !k_scales || !v_scales)
    return fail(FPV2_ERR_ARGUMENT, "%s: null pointer", name);
  if (page_table == nullptr && (p.table_width != 1 || p.cache.pages < p.batch))
    return fail(FPV2_ERR_ARGUMENT, "%s: without a page table every sequence has one page", name);
  if (!a16(k_out) || !a16(v_out) || !a16(k_codes) || !a16(v_codes))
    return fail(FPV2_ERR_ARGUMENT, "%s: the results and the codes must be 16-byte aligned", name);
  ReadArgs a{};
  set_cache(&a, p.cache);
  a.codes[0] = static_cast<const int8_t*>(k_codes), a.codes[1] = static_cast<const int8_t*>(v_codes);
  a.scales[0] = k_scales, a.scales[1] = v_scales;
  a.out[0] = static_cast<uint16_t*>(k_out), a.out[1] = static_cast<uint16_t*>(v_out);
  a.table = page_table;
  a.lengths = lengths;
  a.o_bs[0] = p.k_batch_stride, a.o_hs[0] = p.k_head_stride, a.o_rs[0] = p.k_row_stride;
  a.o_bs[1] = p.v_batch_stride, a.o_hs[1] = p.v_head_stride, a.o_rs[1] = p.v_row_stride;
  a.table_stride = p.table_stride;
  a.kv_heads = static_cast<int>(p.cache.kv_heads);
  a.pages = static_cast<int>(p.cache.pages);
  a.page_size = static_cast<int>(p.cache.page_size);
  a.capacity = static_cast<int>(p.table_width * p.cache.page_size);
  a.length = static_cast<int>(p.length < a.capacity ? p.length : a.capacity);
  a.tokens = static_cast<int>(p.tokens);
  a.zero_rest = p.zero_rest != 0;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  const int batch = static_cast<int>(p.batch);
  return dtype == FPV2_BF16 ? dequantize_dim<bf16_t>(a, batch, p.cache.head_dim, s)
                            : dequantize_dim<f16_t>(a, batch, p.cache.head_dim, s);
}
