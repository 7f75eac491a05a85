// Log probabilities of given tokens, entropies and the most likely alternatives.
//
// With e_i = x_i log2(e) - R for any reference R, p_i = 2^e_i / s, s = sum 2^e_i:
//   log p_i = (e_i - log2 s) ln 2,  -sum p log p = (log2 s - t / s) ln 2,  t = sum 2^e_i e_i
// so one pass over the logits is enough: each thread holds (R, s, t) of what it has
// seen, R the greatest x log2(e), and moves to a greater reference R' by
//   t' = f (t + (R - R') s), s' = f s, f = 2^(R - R').
// e is one fused multiply-add, so neither large logits nor R's own rounding cost bits.
//
// The alternatives: each wave keeps its greatest logits in order, one a lane, and
// inserts the ones above its last.  Bound by reading the logits.
#include "fpv2_batch.h"
#include "fpv2_common.h"

namespace fpv2 {
namespace {

constexpr float kLog2e = 1.44269504088896341f, kLn2 = 0.693147180559945309f;
constexpr float kHuge = 0x1p126f;  // logits beyond it count as it: differences of x log2(e) are finite
constexpr float kTiny = -300.f;    // weights of 2^-300 and less are zeros
constexpr int kVecs = 4;           // 16-byte loads in flight of a thread

struct LogArgs {
  const void* logits;
  const void* tokens;
  float* logprobs;
  float* entropy;
  int64_t* top_tokens;
  float* top_logprobs;
  f32x4* parts;  // [rows][chunks] {R, s, t, -}
  u32x2* lists;  // [rows][chunks][top] {bits of the logit, index}
  int64_t stride;
  int rows, vocab, top, chunks, token_bytes;
};

template <typename T> struct Logit {
  static constexpr int kPer = 8;  // of 16 bytes
  typedef uint16_t raw;
  static __device__ __forceinline__ float get(u32x4 w, int j) {
    return Elem<T>::to_float(static_cast<uint16_t>(w[j / 2] >> (16 * (j % 2))));
  }
  static __device__ __forceinline__ float one(uint16_t r) { return Elem<T>::to_float(r); }
};
template <> struct Logit<float> {
  static constexpr int kPer = 4;
  typedef float raw;
  static __device__ __forceinline__ float get(u32x4 w, int j) { return __uint_as_float(w[j]); }
  static __device__ __forceinline__ float one(float r) { return r; }
};

__device__ __forceinline__ float clamped(float x) {
  return x == neg_inf() ? x : fminf(fmaxf(x, -kHuge), kHuge);
}

struct Sums {
  float r, s, t;
};
__device__ __forceinline__ void move_to(Sums& a, float r) {
  const float d = fmaxf(a.r - r, kTiny);  // (NaN, of nothing seen so far, too)
  const float f = __builtin_amdgcn_exp2f(d);
  a.t = f * __builtin_fmaf(d, a.s, a.t);
  a.s *= f;
  a.r = r;
}
__device__ __forceinline__ Sums join(Sums a, Sums b) {
  const float r = fmaxf(a.r, b.r);
  move_to(a, r);
  move_to(b, r);
  return {r, a.s + b.s, a.t + b.t};
}

// A wave's greatest logits so far, in order, equal ones by index: one a lane.
struct List {
  float x;
  int at;
  float last_x;  // of the last lane: what is not above it does not enter
  int last_at;
  __device__ __forceinline__ void clear() {
    x = last_x = neg_inf();
    at = last_at = 0x7fffffff;
  }
  __device__ __forceinline__ bool enters(float cx, int c) const {
    return cx > last_x || (cx == last_x && c < last_at);
  }
  // all lanes with (cx, c) that enter, one after the other
  __device__ __forceinline__ void insert(float cx, int c, bool live, int lane, int top) {
    uint64_t mask = __ballot(live && cx > neg_inf() && enters(cx, c));
    while (mask != 0) {
      const int from = __builtin_ctzll(mask);
      const float nx = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(cx), from));
      const int n = __builtin_amdgcn_readlane(c, from);
      const int before = __popcll(__ballot(lane < top && (x > nx || (x == nx && at < n))));
      const float up_x = __shfl_up(x, 1, 64);
      const int up = __shfl_up(at, 1, 64);
      x = lane == before ? nx : lane > before ? up_x : x;
      at = lane == before ? n : lane > before ? up : at;
      last_x = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(x), top - 1));
      last_at = __builtin_amdgcn_readlane(at, top - 1);
      mask &= mask - 1;
      mask &= __ballot(enters(cx, c));
    }
  }
};

// The sums of a workgroup's threads, in every thread (sh: 4 of them).
__device__ __forceinline__ Sums join_all(Sums a, Sums* sh, int tid) {
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1)
    a = join(a, Sums{__shfl_xor(a.r, off, 64), __shfl_xor(a.s, off, 64), __shfl_xor(a.t, off, 64)});
  if ((tid & 63) == 0) sh[tid >> 6] = a;
  __syncthreads();
  return join(join(sh[0], sh[1]), join(sh[2], sh[3]));
}

// The lists of a workgroup's waves in its first one's (sh: [4][FPV2_MAX_TOP]).
__device__ __forceinline__ void join_lists(List& list, u32x2 (*sh)[FPV2_MAX_TOP], int tid, int top) {
  const int lane = tid & 63, wave = tid >> 6;
  if (lane < top) sh[wave][lane] = u32x2{__float_as_uint(list.x), static_cast<uint32_t>(list.at)};
  __syncthreads();
  if (wave != 0) return;
  for (int w = 1; w < 4; ++w) {
    const u32x2 c = sh[w][lane % FPV2_MAX_TOP];
    list.insert(__uint_as_float(c[0]), static_cast<int>(c[1]), lane < top, lane, top);
  }
}

// (rounding could leave a sure token 2^-24 above 0)
__device__ __forceinline__ float log_share(float x, float r, float norm) {
  return fminf((__builtin_fmaf(x, kLog2e, -r) - norm) * kLn2, 0.f);
}

template <typename T>
__device__ __forceinline__ void write_row(const LogArgs& a, int row, Sums s, const List& list, int tid) {
  const float norm = log2f(s.s);
  const bool none = s.r == neg_inf();
  if (tid == 0) {
    const int64_t token = a.token_bytes == 8 ? static_cast<const int64_t*>(a.tokens)[row]
                                             : static_cast<const int32_t*>(a.tokens)[row];
    float x = neg_inf();
    if (token >= 0 && token < a.vocab)
      x = Logit<T>::one(static_cast<const typename Logit<T>::raw*>(a.logits)[row * a.stride + token]);
    x = x != x ? neg_inf() : clamped(x);
    a.logprobs[row] = none ? neg_inf() : log_share(x, s.r, norm);
    a.entropy[row] = none ? 0.f : fmaxf((norm - s.t / s.s) * kLn2, 0.f);
  }
  if (tid < a.top) {
    const bool some = list.x > neg_inf();
    a.top_tokens[static_cast<int64_t>(row) * a.top + tid] = some ? list.at : -1;
    a.top_logprobs[static_cast<int64_t>(row) * a.top + tid] =
        some ? log_share(clamped(list.x), s.r, norm) : neg_inf();
  }
}

// One workgroup a chunk of a row.
template <typename T, bool TOP>
__global__ __launch_bounds__(256) void logprobs_kernel(LogArgs a) {
  typedef typename Logit<T>::raw raw;
  constexpr int kPer = Logit<T>::kPer, kEach = kVecs * kPer;
  __shared__ Sums sh_s[4];
  __shared__ u32x2 sh_l[4][FPV2_MAX_TOP];
  const int tid = threadIdx.x, lane = tid & 63;
  const int row = blockIdx.x / a.chunks, chunk = blockIdx.x - row * a.chunks;
  const raw* const p = static_cast<const raw*>(a.logits) + row * a.stride;
  // the row in 16-byte vectors of memory; its first and last ones may be partly others'
  const int skew = static_cast<int>((reinterpret_cast<uintptr_t>(p) & 15u) / sizeof(raw));
  const int vecs = (skew + a.vocab + kPer - 1) / kPer;
  const int first = static_cast<int>(static_cast<int64_t>(vecs) * chunk / a.chunks);
  const int last = static_cast<int>(static_cast<int64_t>(vecs) * (chunk + 1) / a.chunks);
  Sums s = {neg_inf(), 0.f, 0.f};
  List list;
  list.clear();
  for (int v0 = first; v0 < last; v0 += 256 * kVecs) {
    float x[kEach];
#pragma unroll
    for (int i = 0; i < kVecs; ++i) {
      const int v = v0 + 256 * i + tid, e = v * kPer - skew;
      if (v < last && e >= 0 && e + kPer <= a.vocab) {
        const u32x4 w = load16(p + e);
#pragma unroll
        for (int j = 0; j < kPer; ++j) x[i * kPer + j] = Logit<T>::get(w, j);
      } else {
#pragma unroll
        for (int j = 0; j < kPer; ++j)
          x[i * kPer + j] = v < last && e + j >= 0 && e + j < a.vocab ? Logit<T>::one(p[e + j]) : neg_inf();
      }
    }
    float most = neg_inf();
#pragma unroll
    for (int j = 0; j < kEach; ++j) most = fmaxf(most, x[j]);
    if constexpr (TOP) {
      if (__any(most >= list.last_x)) {
#pragma unroll
        for (int j = 0; j < kEach; ++j)
          list.insert(x[j], (v0 + 256 * (j / kPer) + tid) * kPer - skew + j % kPer, true, lane, a.top);
      }
    }
    if (__builtin_fabsf(most) > kHuge && most != neg_inf()) {
      most = clamped(most);
#pragma unroll
      for (int j = 0; j < kEach; ++j) x[j] = x[j] != x[j] ? x[j] : clamped(x[j]);
    }
    if (most * kLog2e > s.r) move_to(s, most * kLog2e);
#pragma unroll
    for (int j = 0; j < kEach; ++j) {
      const float e = fmaxf(__builtin_fmaf(x[j], kLog2e, -s.r), kTiny);  // (a NaN's too)
      const float w = __builtin_amdgcn_exp2f(e);
      s.s += w;
      s.t = __builtin_fmaf(w, e, s.t);
    }
  }
  s = join_all(s, sh_s, tid);
  if constexpr (TOP) join_lists(list, sh_l, tid, a.top);
  if (a.chunks == 1) {
    write_row<T>(a, row, s, list, tid);
    return;
  }
  const int64_t at = static_cast<int64_t>(row) * a.chunks + chunk;
  if (tid == 0) a.parts[at] = f32x4{s.r, s.s, s.t, 0.f};
  if (TOP && tid < a.top) a.lists[at * a.top + tid] = u32x2{__float_as_uint(list.x), static_cast<uint32_t>(list.at)};
}

// Joins a row's chunks: one workgroup a row.
template <typename T, bool TOP>
__global__ __launch_bounds__(256) void logprobs_join_kernel(LogArgs a) {
  __shared__ Sums sh_s[4];
  __shared__ u32x2 sh_l[4][FPV2_MAX_TOP];
  const int tid = threadIdx.x, lane = tid & 63, row = blockIdx.x;
  const int64_t base = static_cast<int64_t>(row) * a.chunks;
  Sums s = {neg_inf(), 0.f, 0.f};
  for (int i = tid; i < a.chunks; i += 256) {
    const f32x4 part = a.parts[base + i];
    s = join(s, Sums{part[0], part[1], part[2]});
  }
  s = join_all(s, sh_s, tid);
  List list;
  list.clear();
  if constexpr (TOP) {
    const int n = a.chunks * a.top;
    for (int i0 = 0; i0 < n; i0 += 256) {
      const int i = i0 + tid;
      const u32x2 c = i < n ? a.lists[base * a.top + i] : u32x2{0xff800000u, 0u};
      list.insert(__uint_as_float(c[0]), static_cast<int>(c[1]), i < n, lane, a.top);
    }
    join_lists(list, sh_l, tid, a.top);
  }
  write_row<T>(a, row, s, list, tid);
}

// Workgroups of a row: as many as fill the chip, of 1024 16-byte vectors at least.
int chunks_of(const fpv2_logprobs_params& p, int dtype) {
  const int64_t vecs = (p.vocab * (dtype == FPV2_F32 ? 4 : 2) + 15) / 16;
  const int64_t most = (vecs + 256 * kVecs - 1) / (256 * kVecs);
  const int64_t want = (4LL * cu_count() + p.rows - 1) / (p.rows > 0 ? p.rows : 1);
  const int64_t n = most < want ? most : want;
  return n > 1 ? static_cast<int>(n) : 1;
}

int check_logprobs(const char* name, const fpv2_logprobs_params* p) {
  if (p == nullptr) return fail(FPV2_ERR_ARGUMENT, "%s: null params", name);
  if (p->rows < 0 || p->rows > 0xffffff) return fail(FPV2_ERR_ARGUMENT, "%s: rows must be 0 to 2^24 - 1", name);
  if (p->vocab <= 0 || p->vocab > FPV2_MAX_VOCAB)
    return fail(FPV2_ERR_UNSUPPORTED, "%s: the vocabulary must have 1 to %d tokens", name, FPV2_MAX_VOCAB);
  if (p->logits_stride < 0) return fail(FPV2_ERR_ARGUMENT, "%s: logits_stride must not be negative", name);
  if (p->token_bytes != 4 && p->token_bytes != 8)
    return fail(FPV2_ERR_ARGUMENT, "%s: token_bytes must be 4 or 8", name);
  if (p->top < 0 || p->top > FPV2_MAX_TOP)
    return fail(FPV2_ERR_ARGUMENT, "%s: top must be 0 to %d", name, FPV2_MAX_TOP);
  return FPV2_OK;
}

// (of the most chunks of any type)
int64_t logprobs_bytes(const fpv2_logprobs_params& p) {
  const int chunks = chunks_of(p, FPV2_F32);
  return chunks == 1 ? 0 : p.rows * chunks * (16 + 8 * p.top);
}

template <typename T, bool TOP>
int launch(const LogArgs& a, hipStream_t s) {
  hipLaunchKernelGGL((logprobs_kernel<T, TOP>), dim3(static_cast<unsigned>(a.rows) * a.chunks), dim3(256), 0, s, a);
  if (a.chunks > 1) {
    if (const int rc = check_launch("logprobs_kernel")) return rc;
    hipLaunchKernelGGL((logprobs_join_kernel<T, TOP>), dim3(a.rows), dim3(256), 0, s, a);
  }
  return check_launch("logprobs_kernel");
}

template <typename T>
int launch_top(const LogArgs& a, hipStream_t s) {
  return a.top > 0 ? launch<T, true>(a, s) : launch<T, false>(a, s);
}

}  // namespace
}  // namespace fpv2

extern "C" int64_t fpv2_token_logprobs_workspace_bytes(const fpv2_logprobs_params* params) {
  using namespace fpv2;
  if (const int rc = check_logprobs("fpv2_token_logprobs", params)) return rc;
  return logprobs_bytes(*params);
}

extern "C" int fpv2_token_logprobs(const void* logits, const void* tokens, int dtype,
                                   const fpv2_logprobs_params* params, float* logprobs, float* entropy,
                                   int64_t* top_tokens, float* top_logprobs, void* workspace,
                                   int64_t workspace_bytes, void* stream) {
  using namespace fpv2;
  const char* name = "fpv2_token_logprobs";
  if (const int rc = check_logprobs(name, params)) return rc;
  const fpv2_logprobs_params& p = *params;
  if (dtype != FPV2_F32 && dtype != FPV2_BF16 && dtype != FPV2_F16)
    return fail(FPV2_ERR_UNSUPPORTED, "%s: dtype must be f32, bf16 or f16", name);
  if (p.rows == 0) return FPV2_OK;
  if (!logits || !tokens || !logprobs || !entropy || (p.top > 0 && (!top_tokens || !top_logprobs)))
    return fail(FPV2_ERR_ARGUMENT, "%s: null pointer", name);
  if (reinterpret_cast<uintptr_t>(logits) % (dtype == FPV2_F32 ? 4 : 2))
    return fail(FPV2_ERR_ARGUMENT, "%s: logits must be aligned to their type", name);
  const int64_t need = logprobs_bytes(p);
  if (need > 0 && (workspace == nullptr || workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 15u)))
    return fail(FPV2_ERR_ARGUMENT, "%s: needs a 16-byte aligned workspace of %lld bytes", name,
                static_cast<long long>(need));
  LogArgs a{};
  a.logits = logits;
  a.tokens = tokens;
  a.logprobs = logprobs;
  a.entropy = entropy;
  a.top_tokens = top_tokens;
  a.top_logprobs = top_logprobs;
  a.stride = p.logits_stride;
  a.rows = static_cast<int>(p.rows);
  a.vocab = static_cast<int>(p.vocab);
  a.top = static_cast<int>(p.top);
  a.token_bytes = static_cast<int>(p.token_bytes);
  a.chunks = chunks_of(p, dtype);
  a.parts = static_cast<f32x4*>(workspace);
  a.lists = reinterpret_cast<u32x2*>(a.parts + p.rows * a.chunks);
  const hipStream_t s = static_cast<hipStream_t>(stream);
  return dtype == FPV2_F32    ? launch_top<float>(a, s)
         : dtype == FPV2_BF16 ? launch_top<bf16_t>(a, s)
                              : launch_top<f16_t>(a, s);
}
