// Norms of query and key heads, rotary embedding and the K/V write into a
// paged cache, in one pass over the fused projection rows.
//
// Bound by the bytes: each element is read once and written once.  A wave
// works on one token: 16-byte loads, a head on 4 to 32 lanes that hold two
// vectors of 8 elements each, the rotation's partners.  The angles of the
// token stay in registers over the wave's heads.  8192 tokens of 32 / 8 heads, D = 128,
// run at 5.2 TB/s (a copy of 2 GiB: 4.8); 5 tokens take the kernel 4 us.
#include "fpv2_common.h"
#include "fpv2_decode.h"

namespace fpv2 {
namespace {

struct RopePagesArgs {
  const uint16_t* qkv;
  const uint16_t* qw;
  const uint16_t* kw;
  const float* cos;
  const float* sin;
  const void* positions;
  const void* slots;
  uint16_t* q;
  uint16_t* k;
  uint16_t* v;
  int64_t tokens, table_rows, first_position, first_slot, slot_count;
  int64_t qkv_rs, q_ts, q_hs, k_ps, k_hs, k_rs, v_ps, v_hs, v_rs;
  int position_bytes, slot_bytes, interleaved, page_size;
  int qh, kh, d, half;
  int lanes;       // of a head: a power of two >= d / 16
  int chunk;       // heads of a wave
  int chunks;      // waves of a token
  float eps;
};

__device__ __forceinline__ int64_t index_of(const void* p, int bytes, int64_t first, int64_t t) {
  if (bytes == 8) return static_cast<const int64_t*>(p)[t];
  if (bytes == 4) return static_cast<const int32_t*>(p)[t];
  return first + t;
}

template <typename T>
__device__ __forceinline__ void unpack8(u32x4 w, float* x) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    x[2 * j] = Elem<T>::to_float(w[j] & 0xffffu);
    x[2 * j + 1] = Elem<T>::to_float(w[j] >> 16);
  }
}
template <typename T>
__device__ __forceinline__ u32x4 pack8(const float* x) {
  u32x4 w;
#pragma unroll
  for (int j = 0; j < 4; ++j) w[j] = pack2<T>(x[2 * j], x[2 * j + 1]);
  return w;
}

// STREAM: the stores go past the caches.
template <typename T, bool STREAM>
__global__ __launch_bounds__(256) void rope_pages_kernel(RopePagesArgs a) {
  const int lane = threadIdx.x & 63;
  const int64_t work = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6);
  const int64_t t = work / a.chunks;
  if (t >= a.tokens) return;
  const int heads = a.qh + 2 * a.kh;
  const int h_begin = static_cast<int>(work - t * a.chunks) * a.chunk;
  const int h_end = min(heads, h_begin + a.chunk);
  const int s = lane & (a.lanes - 1);
  const int per_wave = 64 / a.lanes;
  const int units = a.d / 8, rot = a.half / 8;
  const bool valid = s < units / 2;
  // the lane's two vectors: rotation partners (halves), or any two
  int ua = s, ub = s + units / 2;
  if (!a.interleaved) {
    const int rest = (units - 2 * rot) / 2;
    ub = s < rot ? s + rot : s + rot + rest;
    ua = s < rot ? s : s + rot;
  }
  int64_t pos = index_of(a.positions, a.position_bytes, a.first_position, t);
  pos = min(max(pos, static_cast<int64_t>(0)), a.table_rows - 1);
  const int64_t slot = index_of(a.slots, a.slot_bytes, a.first_slot, t);
  const bool stored = slot >= 0 && slot < a.slot_count;
  const int64_t page = stored ? static_cast<uint32_t>(slot) / static_cast<uint32_t>(a.page_size) : 0;
  const int64_t row = stored ? slot - page * a.page_size : 0;
  // angles: of the pair's 8 elements, or of 4 pairs in each vector
  float c[8], sn[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) c[j] = 1.f, sn[j] = 0.f;
  const float* ct = a.cos + pos * a.half;
  const float* st = a.sin + pos * a.half;
  if (valid) {
    const int at0 = a.interleaved ? 4 * ua : 8 * s, at1 = a.interleaved ? 4 * ub : 8 * s + 4;
    if (at0 < a.half) {
      const f32x4 x = *reinterpret_cast<const f32x4*>(ct + at0);
      const f32x4 y = *reinterpret_cast<const f32x4*>(st + at0);
#pragma unroll
      for (int j = 0; j < 4; ++j) c[j] = x[j], sn[j] = y[j];
    }
    if (at1 < a.half) {
      const f32x4 x = *reinterpret_cast<const f32x4*>(ct + at1);
      const f32x4 y = *reinterpret_cast<const f32x4*>(st + at1);
#pragma unroll
      for (int j = 0; j < 4; ++j) c[4 + j] = x[j], sn[4 + j] = y[j];
    }
  }
  const uint16_t* src = a.qkv + t * a.qkv_rs;
  for (int h0 = h_begin; h0 < h_end; h0 += per_wave) {
    const int h = h0 + lane / a.lanes;
    const bool on = valid && h < h_end;
    u32x4 xa = {0, 0, 0, 0}, xb = {0, 0, 0, 0};
    if (on) {
      xa = load16(src + static_cast<int64_t>(h) * a.d + 8 * ua);
      xb = load16(src + static_cast<int64_t>(h) * a.d + 8 * ub);
    }
    const int kind = h < a.qh ? 0 : (h < a.qh + a.kh ? 1 : 2);
    const uint16_t* w = kind == 0 ? a.qw : a.kw;
    float na[8], nb[8];
    unpack8<T>(xa, na);
    unpack8<T>(xb, nb);
    float ss = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) ss += na[j] * na[j] + nb[j] * nb[j];
    for (int off = a.lanes / 2; off >= 1; off >>= 1) ss += __shfl_xor(ss, off, 64);
    if (!on) continue;
    if (kind < 2) {
      if (w != nullptr) {
        const float r = rsqrtf(ss / static_cast<float>(a.d) + a.eps);
        float wa[8], wb[8];
        unpack8<T>(load16(w + 8 * ua), wa);
        unpack8<T>(load16(w + 8 * ub), wb);
#pragma unroll
        for (int j = 0; j < 8; ++j) na[j] *= r * wa[j], nb[j] *= r * wb[j];
      }
      // (a vector behind the rotated ones stays as it is: a product with (1, 0) would make NaN
      // of what lies beside an infinity)
      if (a.interleaved) {
        if (ua < 2 * rot) {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float a0 = na[2 * j], a1 = na[2 * j + 1];
            na[2 * j] = a0 * c[j] - a1 * sn[j];
            na[2 * j + 1] = a1 * c[j] + a0 * sn[j];
          }
        }
        if (ub < 2 * rot) {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float b0 = nb[2 * j], b1 = nb[2 * j + 1];
            nb[2 * j] = b0 * c[4 + j] - b1 * sn[4 + j];
            nb[2 * j + 1] = b1 * c[4 + j] + b0 * sn[4 + j];
          }
        }
      } else if (s < rot) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float x = na[j], y = nb[j];
          na[j] = x * c[j] - y * sn[j];
          nb[j] = y * c[j] + x * sn[j];
        }
      }
      xa = pack8<T>(na);
      xb = pack8<T>(nb);
    }
    uint16_t* dst;
    if (kind == 0)
      dst = a.q + t * a.q_ts + h * a.q_hs;
    else if (kind == 1)
      dst = a.k + page * a.k_ps + (h - a.qh) * a.k_hs + row * a.k_rs;
    else
      dst = a.v + page * a.v_ps + (h - a.qh - a.kh) * a.v_hs + row * a.v_rs;
    if (kind == 0 || stored) {
      if constexpr (STREAM) {
        __builtin_nontemporal_store(xa, reinterpret_cast<u32x4*>(dst + 8 * ua));
        __builtin_nontemporal_store(xb, reinterpret_cast<u32x4*>(dst + 8 * ub));
      } else {
        store16(dst + 8 * ua, xa);
        store16(dst + 8 * ub, xb);
      }
    }
  }
}

}  // namespace
}  // namespace fpv2

extern "C" int fpv2_rope_to_pages(const void* qkv, const void* q_weight, const void* k_weight,
                                  const float* cos, const float* sin, const void* positions,
                                  const void* slots, void* q_out, void* k_pages, void* v_pages,
                                  int dtype, const fpv2_rope_pages_params* params, void* stream) {
  using namespace fpv2;
  const char* name = "fpv2_rope_to_pages";
  const auto aligned = [](const void* p, int n) { return reinterpret_cast<uintptr_t>(p) % n == 0; };
  if (params == nullptr) return fail(FPV2_ERR_ARGUMENT, "%s: null params", name);
  const fpv2_rope_pages_params& p = *params;
  if (dtype != FPV2_BF16 && dtype != FPV2_F16)
    return fail(FPV2_ERR_UNSUPPORTED, "%s: dtype must be bf16 or f16", name);
  if (p.tokens < 0 || p.query_heads <= 0 || p.kv_heads <= 0 || p.query_heads + 2 * p.kv_heads > 65535)
    return fail(FPV2_ERR_ARGUMENT, "%s: bad tokens or head counts", name);
  if (p.head_dim <= 0 || p.head_dim % 16 || p.head_dim > 512)
    return fail(FPV2_ERR_UNSUPPORTED, "%s: head_dim must be a multiple of 16 and at most 512", name);
  if (p.rotary_half <= 0 || p.rotary_half % 8 || 2 * p.rotary_half > p.head_dim)
    return fail(FPV2_ERR_UNSUPPORTED, "%s: cos and sin must have a multiple of 8 columns, at most "
                "head_dim / 2", name);
  if (p.table_rows <= 0 || p.pages <= 0 || p.page_size <= 0 || p.pages > 0x7fffffff ||
      p.page_size > 0x7fffffff || p.pages * p.page_size > 0x7fffffff)
    return fail(FPV2_ERR_ARGUMENT, "%s: table_rows, pages and page_size must be positive and the "
                "pages hold fewer than 2^31 tokens", name);
  if ((p.position_bytes != 0 && p.position_bytes != 4 && p.position_bytes != 8) ||
      (p.slot_bytes != 0 && p.slot_bytes != 4 && p.slot_bytes != 8))
    return fail(FPV2_ERR_ARGUMENT, "%s: positions and slots are int32 or int64", name);
  if (p.tokens == 0) return FPV2_OK;
  if (!qkv || !cos || !sin || !q_out || !k_pages || !v_pages || (p.position_bytes && !positions) ||
      (p.slot_bytes && !slots))
    return fail(FPV2_ERR_ARGUMENT, "%s: null pointer", name);
  if (p.qkv_row_stride < (p.query_heads + 2 * p.kv_heads) * p.head_dim && p.tokens > 1)
    return fail(FPV2_ERR_ARGUMENT, "%s: qkv rows are shorter than the heads read", name);
  const int64_t strides[] = {p.qkv_row_stride, p.q_token_stride, p.q_head_stride, p.k_page_stride,
                             p.k_head_stride,  p.k_row_stride,   p.v_page_stride, p.v_head_stride,
                             p.v_row_stride};
  for (const int64_t x : strides)
    if (x < 0 || x % 8) return fail(FPV2_ERR_ARGUMENT, "%s: strides must be multiples of 8", name);
  if (!aligned(qkv, 16) || !aligned(q_weight, 16) || !aligned(k_weight, 16) || !aligned(cos, 16) ||
      !aligned(sin, 16) || !aligned(q_out, 16) || !aligned(k_pages, 16) || !aligned(v_pages, 16) ||
      (p.position_bytes && !aligned(positions, static_cast<int>(p.position_bytes))) ||
      (p.slot_bytes && !aligned(slots, static_cast<int>(p.slot_bytes))))
    return fail(FPV2_ERR_ARGUMENT, "%s: pointers must be 16-byte aligned", name);
  RopePagesArgs a{};
  a.qkv = static_cast<const uint16_t*>(qkv);
  a.qw = static_cast<const uint16_t*>(q_weight);
  a.kw = static_cast<const uint16_t*>(k_weight);
  a.cos = cos;
  a.sin = sin;
  a.positions = positions;
  a.slots = slots;
  a.q = static_cast<uint16_t*>(q_out);
  a.k = static_cast<uint16_t*>(k_pages);
  a.v = static_cast<uint16_t*>(v_pages);
  a.tokens = p.tokens;
  a.table_rows = p.table_rows;
  a.first_position = p.first_position;
  a.first_slot = p.first_slot;
  a.slot_count = p.pages * p.page_size;
  a.qkv_rs = p.qkv_row_stride;
  a.q_ts = p.q_token_stride;
  a.q_hs = p.q_head_stride;
  a.k_ps = p.k_page_stride;
  a.k_hs = p.k_head_stride;
  a.k_rs = p.k_row_stride;
  a.v_ps = p.v_page_stride;
  a.v_hs = p.v_head_stride;
  a.v_rs = p.v_row_stride;
  a.position_bytes = static_cast<int>(p.position_bytes);
  a.slot_bytes = static_cast<int>(p.slot_bytes);
  a.interleaved = p.interleaved != 0;
  a.page_size = static_cast<int>(p.page_size);
  a.qh = static_cast<int>(p.query_heads);
  a.kh = static_cast<int>(p.kv_heads);
  a.d = static_cast<int>(p.head_dim);
  a.half = static_cast<int>(p.rotary_half);
  a.lanes = 1;
  while (a.lanes < a.d / 16) a.lanes *= 2;
  a.eps = static_cast<float>(p.eps);
  // Where the tokens fill the chip, a wave takes two rounds of heads (the angles are
  // loaded once for both) and stores past the caches, which the outputs of so
  // many tokens overflow.  8192 tokens of 32 / 8 heads, D = 128: one round 44.5 us, two
  // 42.6, all six 49.4; with such stores 42.5, 39.7 (5.2 TB/s) and 42.4 us.
  const int heads = a.qh + 2 * a.kh, per_wave = 64 / a.lanes;
  const bool many = p.tokens >= 8 * static_cast<int64_t>(cu_count());
  a.chunk = many ? 2 * per_wave : per_wave;
  a.chunks = (heads + a.chunk - 1) / a.chunk;
  const int64_t grid = (p.tokens * a.chunks + 3) / 4;
  if (grid > 0x7fffffff) return fail(FPV2_ERR_ARGUMENT, "%s: too many tokens", name);
  const hipStream_t s = static_cast<hipStream_t>(stream);
  const dim3 blocks(static_cast<unsigned>(grid)), threads(256);
  if (dtype == FPV2_BF16) {
    if (many)
      hipLaunchKernelGGL((rope_pages_kernel<bf16_t, true>), blocks, threads, 0, s, a);
    else
      hipLaunchKernelGGL((rope_pages_kernel<bf16_t, false>), blocks, threads, 0, s, a);
  } else {
    if (many)
      hipLaunchKernelGGL((rope_pages_kernel<f16_t, true>), blocks, threads, 0, s, a);
    else
      hipLaunchKernelGGL((rope_pages_kernel<f16_t, false>), blocks, threads, 0, s, a);
  }
  return check_launch("rope_pages_kernel");
}
