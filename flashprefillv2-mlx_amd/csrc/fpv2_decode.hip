// Attention of one new token per sequence over a paged key-value cache: the C entry
// (kernels, schedule and plan: fpv2_decode_split.h).
#include "fpv2_decode_split.h"

namespace fpv2 {
namespace {

template <typename T, int D>
int launch(const DecodeArgs& a, bool join, hipStream_t s) {
  hipLaunchKernelGGL((decode_attn_kernel<T, D>), dim3(a.grid), dim3(256), 0, s, a);
  if (join) launch_join<T, D>(a, s);
  return check_launch("decode_attn_kernel");
}

template <typename T>
int launch_dim(const DecodeArgs& a, int64_t dim, bool join, hipStream_t s) {
  switch (dim) {
    case 64: return launch<T, 64>(a, join, s);
    case 96: return launch<T, 96>(a, join, s);
    case 128: return launch<T, 128>(a, join, s);
    default: return launch<T, 256>(a, join, s);
  }
}

}  // namespace
}  // namespace fpv2

extern "C" int64_t fpv2_decode_attention_workspace_bytes(const fpv2_decode_params* params) {
  using namespace fpv2;
  if (const int rc = check_params("fpv2_decode_attention", params)) return rc;
  return partial_bytes(*params, decode_plan(*params));
}

extern "C" int fpv2_decode_attention(const void* q, const void* k_pages, const void* v_pages,
                                     const int32_t* page_table, const int32_t* lengths, void* out,
                                     int dtype, const fpv2_decode_params* params, void* workspace,
                                     int64_t workspace_bytes, void* stream) {
  using namespace fpv2;
  const char* name = "fpv2_decode_attention";
  const auto a16 = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; };
  if (const int rc = check_params(name, params)) return rc;
  const fpv2_decode_params& p = *params;
  if (dtype != FPV2_BF16 && dtype != FPV2_F16)
    return fail(FPV2_ERR_UNSUPPORTED, "%s: dtype must be bf16 or f16", name);
  if (p.batch == 0) return FPV2_OK;
  if (!q || !k_pages || !v_pages || !out) return fail(FPV2_ERR_ARGUMENT, "%s: null pointer", name);
  if (page_table == nullptr && (p.table_width != 1 || p.pages < p.batch))
    return fail(FPV2_ERR_ARGUMENT, "%s: without a page table every sequence has one page", name);
  if (page_table != nullptr && p.table_stride < 0)
    return fail(FPV2_ERR_ARGUMENT, "%s: table_stride must not be negative", name);
  const int64_t strides[] = {p.q_batch_stride, p.q_head_stride, p.k_page_stride, p.k_head_stride,
                             p.k_row_stride,   p.v_page_stride, p.v_head_stride, p.v_row_stride};
  for (const int64_t x : strides)
    if (x < 0 || x % 8)
      return fail(FPV2_ERR_ARGUMENT, "%s: strides of q, k and v must be multiples of 8", name);
  if (p.o_batch_stride < 0 || p.o_head_stride < 0)
    return fail(FPV2_ERR_ARGUMENT, "%s: output strides must not be negative", name);
  if (!a16(q) || !a16(k_pages) || !a16(v_pages))
    return fail(FPV2_ERR_ARGUMENT, "%s: q, k and v must be 16-byte aligned", name);
  const DecodePlan plan = decode_plan(p);
  const int64_t need = partial_bytes(p, plan);
  if (need > 0 && (workspace == nullptr || workspace_bytes < need || !a16(workspace)))
    return fail(FPV2_ERR_ARGUMENT, "%s: needs a 16-byte aligned workspace of %lld bytes", name,
                static_cast<long long>(need));
  DecodeArgs a = decode_args(p, plan);
  a.q = static_cast<const uint16_t*>(q);
  a.k = static_cast<const uint16_t*>(k_pages);
  a.v = static_cast<const uint16_t*>(v_pages);
  a.out = static_cast<uint16_t*>(out);
  a.table = page_table;
  a.lengths = lengths;
  a.part_o = static_cast<float*>(workspace);
  a.part_ml = a.part_o + 2LL * plan.grid * plan.item_heads * p.head_dim;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  const bool join = plan.most_tiles > 1;
  return dtype == FPV2_BF16 ? launch_dim<bf16_t>(a, p.head_dim, join, s)
                            : launch_dim<f16_t>(a, p.head_dim, join, s);
}
