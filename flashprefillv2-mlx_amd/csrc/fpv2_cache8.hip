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
// Both are bound by memory, 3 bytes a value.  8 heads of D = 128: 32768 tokens written in 35 us, read
// in 31 (201 MB, 5.8 and 6.6 TB/s, where the caches hold some of it), 131072 tokens 165 and 164 (4.9 TB/s);
// a few tokens 3.1 and 3.3, a launch.  The greatest magnitude by pairs of bits instead of
// floats, and the codes by one sum: 97 us to 71 where 24 sequences' prompts are written.
#include "fpv2_batch.h"
#include "fpv2_common.h"

namespace fpv2 {
namespace {

typedef int i32x2 __attribute__((ext_vector_type(2)));
typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));

struct QuantArgs {
  const uint16_t* x[2];   // k, v
  int8_t* codes[2];
  float* scales[2];
  const void* slots;
  int64_t x_ts[2], x_hs[2];
  int64_t c_ps[2], c_hs[2], c_rs[2];
  int64_t s_ps[2], s_hs[2], s_rs[2];
  int64_t first_slot, slot_count, page_size;
  int slot_bytes, kv_heads, tokens;
  uint32_t page_mul, page_shift;  // slot / page_size = (umulhi(slot, mul) + slot) >> shift
};

constexpr int kMaxBlocks = 1 << 18;  // of a launch; more work is done in turns

// A group of lanes a row, 8 values a lane; HEADS rows of a token, with as many loads in flight.
template <typename T, int D, int HEADS>
__global__ __launch_bounds__(256) void quantize_kernel(QuantArgs a) {
  constexpr int kLanes = D / 8 <= 8 ? 8 : D / 8 <= 16 ? 16 : 32;
  constexpr uint32_t kInf = std::is_same<T, bf16_t>::value ? 0x7f80u : 0x7c00u;
  const int tid = threadIdx.x, at = tid % kLanes;
  const int side = blockIdx.y, chunks = (a.kv_heads + HEADS - 1) / HEADS;
  const uint32_t groups = static_cast<uint32_t>(a.tokens) * chunks;
  for (uint32_t g = blockIdx.x * (256 / kLanes) + tid / kLanes; g < groups; g += gridDim.x * (256 / kLanes)) {
    const int64_t t = g / chunks;
    const int h0 = static_cast<int>(g - static_cast<uint32_t>(t) * chunks) * HEADS;
    u32x4 w[HEADS];
#pragma unroll
    for (int i = 0; i < HEADS; ++i)
      w[i] = 8 * at < D && h0 + i < a.kv_heads
                 ? load16(a.x[side] + t * a.x_ts[side] + (h0 + i) * a.x_hs[side] + 8 * at)
                 : u32x4{0, 0, 0, 0};
    const int64_t slot = a.slot_bytes == 8   ? static_cast<const int64_t*>(a.slots)[t]
                         : a.slot_bytes == 4 ? static_cast<const int32_t*>(a.slots)[t]
                                             : a.first_slot + t;
    const bool live = slot >= 0 && slot < a.slot_count && 8 * at < D;
    int64_t page, r;
    if (a.slot_count <= 0x7fffffff) {
      const uint32_t s = live ? static_cast<uint32_t>(slot) : 0;
      page = (__umulhi(s, a.page_mul) + s) >> a.page_shift;
      r = s - static_cast<uint32_t>(page) * static_cast<uint32_t>(a.page_size);
    } else {
      page = live ? slot / a.page_size : 0;
      r = live ? slot - page * a.page_size : 0;
    }
    int8_t* const codes = a.codes[side] + page * a.c_ps[side] + r * a.c_rs[side] + 8 * at;
    float* const scales = a.scales[side] + page * a.s_ps[side] + r * a.s_rs[side];
#pragma unroll
    for (int i = 0; i < HEADS; ++i) {
      // the greatest magnitude, as the bits of the type: two at a time
      u16x2 two = {0, 0};
#pragma unroll
      for (int j = 0; j < 4; ++j)
        two = __builtin_elementwise_max(two, __builtin_bit_cast(u16x2, w[i][j] & 0x7fff7fffu));
      uint32_t bits = max(static_cast<uint32_t>(two[0]), static_cast<uint32_t>(two[1]));
#pragma unroll
      for (int off = kLanes / 2; off >= 1; off >>= 1) bits = max(bits, static_cast<uint32_t>(__shfl_xor(bits, off, 64)));
      const bool bad = bits >= kInf;
      const float top = Elem<T>::to_float(static_cast<uint16_t>(bits));
      // (the quotients are the same for rows of tiny or huge values times a power of two)
      const float up = top < 0x1p-64f ? 0x1p64f : top > 0x1p64f ? 0x1p-64f : 1.f;
      const float most = top * up, factor = 127.f * up;
      const float y = top > 0.f ? 1.f / most : 0.f;
      uint32_t code[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float n = Elem<T>::to_float(static_cast<uint16_t>(w[i][j / 2] >> (16 * (j % 2)))) * factor;
        float q = n * y;
        q = __builtin_fmaf(__builtin_fmaf(-q, most, n), y, q);
        // (the sum is rounded to a whole number, whose two's complement is in its low bits)
        code[j] = __float_as_uint(q + 0x1.8p23f);
      }
      i32x2 out;
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const uint32_t low = __builtin_amdgcn_perm(code[4 * k + 1], code[4 * k], 0x0c0c0400u);
        const uint32_t high = __builtin_amdgcn_perm(code[4 * k + 3], code[4 * k + 2], 0x04000c0cu);
        out[k] = bad ? 0 : static_cast<int>(low | high);
      }
      if (live && h0 + i < a.kv_heads) {
        *reinterpret_cast<i32x2*>(codes + (h0 + i) * a.c_hs[side]) = out;
        if (at == 0) scales[(h0 + i) * a.s_hs[side]] = bad ? __builtin_nanf("") : top / 127.f;
      }
    }
  }
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
  uint32_t page_mul, page_shift;  // t / page_size = (umulhi(t, mul) + t) >> shift
};

// 8 values a lane, a row's chunks next to one another, TURNS of them in flight; blocks:
// (tokens, sequence * head, side).  More than one: the stores go past the caches.
template <typename T, int D, int TURNS>
__global__ __launch_bounds__(256) void dequantize_kernel(ReadArgs a) {
  constexpr int kChunks = D / 8;
  const int side = blockIdx.z;
  const int b = blockIdx.y / a.kv_heads, h = blockIdx.y - b * a.kv_heads;
  int len = a.lengths != nullptr ? a.lengths[b] : a.length;
  len = min(max(len, 0), a.capacity);
  const uint32_t end = static_cast<uint32_t>(a.zero_rest ? a.tokens : min(a.tokens, len));
  uint16_t* const base = a.out[side] + b * a.o_bs[side] + h * a.o_hs[side];
  const int8_t* const codes = a.codes[side] + h * a.c_hs[side];
  const float* const scales = a.scales[side] + h * a.s_hs[side];
  const int64_t count = static_cast<int64_t>(end) * kChunks;
  for (int64_t e0 = static_cast<int64_t>(blockIdx.x) * (256 * TURNS) + threadIdx.x; e0 < count;
       e0 += static_cast<int64_t>(gridDim.x) * (256 * TURNS)) {
    u32x2 w[TURNS];
    float scale[TURNS];
#pragma unroll
    for (int i = 0; i < TURNS; ++i) {
      const uint32_t t = static_cast<uint32_t>((e0 + 256 * i) / kChunks);
      const int c = static_cast<int>(e0 + 256 * i - static_cast<int64_t>(t) * kChunks);
      w[i] = u32x2{0, 0};
      scale[i] = 0.f;
      if (t < end && t < static_cast<uint32_t>(len)) {
        const uint32_t at = (__umulhi(t, a.page_mul) + t) >> a.page_shift;
        const int64_t r = t - at * static_cast<uint32_t>(a.page_size);
        const int id = a.table != nullptr ? a.table[b * a.table_stride + at] : b;
        const int64_t page = min(max(id, 0), a.pages - 1);
        w[i] = *reinterpret_cast<const u32x2*>(codes + page * a.c_ps[side] + r * a.c_rs[side] + 8 * c);
        scale[i] = scales[page * a.s_ps[side] + r * a.s_rs[side]];
      }
    }
#pragma unroll
    for (int i = 0; i < TURNS; ++i) {
      const uint32_t t = static_cast<uint32_t>((e0 + 256 * i) / kChunks);
      const int c = static_cast<int>(e0 + 256 * i - static_cast<int64_t>(t) * kChunks);
      u32x4 v;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int word = static_cast<int>(w[i][j / 2]) >> (16 * (j % 2));
        v[j] = pack2<T>(static_cast<float>(static_cast<int8_t>(word)) * scale[i],
                        static_cast<float>(static_cast<int8_t>(word >> 8)) * scale[i]);
      }
      u32x4* const out = reinterpret_cast<u32x4*>(base + t * a.o_rs[side] + 8 * c);
      if (t < end) {
        if constexpr (TURNS > 1)
          __builtin_nontemporal_store(v, out);
        else
          *out = v;
      }
    }
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

template <typename T, int D, int HEADS>
int launch_quantize(const QuantArgs& a, hipStream_t s) {
  constexpr int kRows = 256 / (D / 8 <= 8 ? 8 : D / 8 <= 16 ? 16 : 32);
  const int64_t blocks = (static_cast<int64_t>(a.tokens) * ((a.kv_heads + HEADS - 1) / HEADS) + kRows - 1) / kRows;
  hipLaunchKernelGGL((quantize_kernel<T, D, HEADS>),
                     dim3(static_cast<unsigned>(blocks < kMaxBlocks ? blocks : kMaxBlocks), 2), dim3(256), 0, s, a);
  return check_launch("quantize_kernel");
}

// Many rows: several of a token in turn.  8 heads of D = 128, four rows in turn / one: 512 tokens 4.7 / 3.7
// us, 2048 (2^14 rows) 5.6 / 5.8, 32768 35 / 41, 131072 165 / 185.
template <typename T, int D>
int launch_rows(const QuantArgs& a, hipStream_t s) {
  return a.kv_heads > 1 && static_cast<int64_t>(a.tokens) * a.kv_heads >= 1 << 14 ? launch_quantize<T, D, 4>(a, s)
                                                                                   : launch_quantize<T, D, 1>(a, s);
}

template <typename T, int D, int TURNS>
int launch_turns(const ReadArgs& a, int batch, hipStream_t s) {
  const int64_t blocks = (static_cast<int64_t>(a.tokens) * (D / 8) + 256 * TURNS - 1) / (256 * TURNS);
  hipLaunchKernelGGL((dequantize_kernel<T, D, TURNS>),
                     dim3(static_cast<unsigned>(blocks < kMaxBlocks ? blocks : kMaxBlocks),
                          static_cast<unsigned>(batch) * a.kv_heads, 2),
                     dim3(256), 0, s, a);
  return check_launch("dequantize_kernel");
}

// Results of which few stay in the L2s (2^23 bytes and more of K and of V each).  8 heads of
// D = 128, four turns / one: 512 tokens 4.4 / 3.6 us, 2048 5.3 / 5.5, 4096 (2^22 values) 5.9 / 7.8,
// 32768 31 / 38, 131072 164 / 229.
template <typename T, int D>
int launch_dequantize(const ReadArgs& a, int batch, hipStream_t s) {
  return static_cast<int64_t>(a.tokens) * batch * a.kv_heads * D >= 1 << 22 ? launch_turns<T, D, 4>(a, batch, s)
                                                                            : launch_turns<T, D, 1>(a, batch, s);
}

template <typename T>
int quantize_dim(const QuantArgs& a, int64_t dim, hipStream_t s) {
  switch (dim) {
    case 64: return launch_rows<T, 64>(a, s);
    case 96: return launch_rows<T, 96>(a, s);
    case 128: return launch_rows<T, 128>(a, s);
    default: return launch_rows<T, 256>(a, s);
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
  if (p.tokens < 0 || p.tokens > 0x3fffffff / p.cache.kv_heads)
    return fail(FPV2_ERR_ARGUMENT, "%s: tokens * kv_heads must be 0 to 2^30 - 1", name);
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
  a.slot_count = p.cache.pages * p.cache.page_size;
  a.page_size = p.cache.page_size;
  page_division(p.cache.page_size, &a.page_mul, &a.page_shift);
  a.tokens = static_cast<int>(p.tokens);
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
  page_division(p.cache.page_size, &a.page_mul, &a.page_shift);
  a.capacity = static_cast<int>(p.table_width * p.cache.page_size);
  a.length = static_cast<int>(p.length < a.capacity ? p.length : a.capacity);
  a.tokens = static_cast<int>(p.tokens);
  a.zero_rest = p.zero_rest != 0;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  const int batch = static_cast<int>(p.batch);
  return dtype == FPV2_BF16 ? dequantize_dim<bf16_t>(a, batch, p.cache.head_dim, s)
                            : dequantize_dim<f16_t>(a, batch, p.cache.head_dim, s);
}
