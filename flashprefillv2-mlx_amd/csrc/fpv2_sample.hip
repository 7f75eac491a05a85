// Sampling with temperature, top-k, top-p and min-p from given random numbers.
//
// The weight of a token is exp((logit - max) / temperature) in float64, rounded to
// an integer of 2^-44: sums of up to 2^19 of them are exact in 64 bits, so that
// histograms can be added in any order and a token next to a border is the same
// in every call.  Kept tokens are a prefix of the order (logit descending, index
// ascending): all tokens with a greater key than the border's, and the first few of
// the border's own (a key is the logit's bits, ordered as unsigned integers).
//
// One workgroup per row.  The border of top-k is found by counts over the key's
// four bytes, the one of top-p by weights in the same way.
#include "fpv2_common.h"
#include "fpv2_decode.h"

namespace fpv2 {
namespace {

constexpr int kThreads = 1024;
constexpr int kWaves = kThreads / 64;
constexpr int kWeightBits = 44;
typedef unsigned long long u64;

struct SampleArgs {
  const void* logits;
  const float* uniforms;
  const float* temperatures;
  const int32_t* top_ks;
  const float* top_ps;
  const float* min_ps;
  int64_t* tokens;
  float* logprobs;
  double temperature, top_p, min_p;
  int64_t top_k, stride;
  int vocab;
};

struct f32_t { float v; };
template <typename T>
__device__ __forceinline__ float logit_at(const void* row, int i) {
  return Elem<T>::to_float(static_cast<const uint16_t*>(row)[i]);
}
template <>
__device__ __forceinline__ float logit_at<f32_t>(const void* row, int i) {
  return static_cast<const float*>(row)[i];
}

// Order-preserving key: -inf and NaN least, both zeros alike.
constexpr uint32_t kLeastKey = 0x007fffffu;  // of -inf
__device__ __forceinline__ uint32_t key_of(float x) {
  if (x != x) return kLeastKey;
  const uint32_t b = __float_as_uint(x + 0.f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float logit_of(uint32_t key) {
  return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key);
}

struct Row {
  const void* logits;
  uint32_t top;     // greatest key
  double max, inv;  // its logit, 1 / temperature
  u64 least;        // least weight that min_p keeps
};

// log of a weight, and the weight (0 below 2^-45)
__device__ __forceinline__ double exponent_of(const Row& r, uint32_t key) {
  if (key == r.top) return 0.0;
  if (key <= kLeastKey) return -__builtin_inf();
  return (static_cast<double>(logit_of(key)) - r.max) * r.inv;
}
__device__ __forceinline__ u64 weight_of(const Row& r, uint32_t key) {
  const double z = exponent_of(r, key);
  if (!(z > -31.2)) return 0;
  return static_cast<u64>(exp(z) * (1ull << kWeightBits) + 0.5);
}

__device__ __forceinline__ u64 shfl_xor64(u64 v, int off) {
  return static_cast<u64>(__shfl_xor(static_cast<long long>(v), off, 64));
}

// Sum (or greatest) of a value of each thread, in every thread.
template <bool MAX>
__device__ u64 across(u64 v, u64* sh) {
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) {
    const u64 o = shfl_xor64(v, off);
    v = MAX ? (o > v ? o : v) : v + o;
  }
  __syncthreads();
  if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = v;
  __syncthreads();
  v = sh[0];
#pragma unroll
  for (int w = 1; w < kWaves; ++w) v = MAX ? (sh[w] > v ? sh[w] : v) : v + sh[w];
  return v;
}

// The first index i in [0, n) for which past(sum of value(0..i)) holds, or n: sums of a
// wave's share, then of its shares, until one wave is left with a piece.
template <typename Value, typename Past>
__device__ int find_first(int n, Value value, Past past, u64* sh, int* sh_at) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int lo = 0, hi = n;
  u64 before = 0;
  while (hi - lo > 512) {
    const int share = (hi - lo + kWaves - 1) / kWaves;
    const int a = min(hi, lo + wave * share), b = min(hi, a + share);
    u64 sum = 0;
    for (int i = a + lane; i < b; i += 64) sum += value(i);
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) sum += shfl_xor64(sum, off);
    __syncthreads();
    if (lane == 0) sh[wave] = sum;
    __syncthreads();
    int w = 0;
    while (w < kWaves && !past(before + sh[w])) before += sh[w++];
    if (w == kWaves) return n;
    const int next = min(hi, lo + w * share);
    hi = min(hi, next + share);
    lo = next;
  }
  __syncthreads();
  if (threadIdx.x == 0) *sh_at = n;
  __syncthreads();
  if (wave == 0) {
    for (int i0 = lo; i0 < hi; i0 += 64) {
      u64 sum = i0 + lane < hi ? value(i0 + lane) : 0;
#pragma unroll
      for (int off = 1; off < 64; off <<= 1) {
        const u64 up = static_cast<u64>(__shfl_up(static_cast<long long>(sum), off, 64));
        sum += lane >= off ? up : 0;
      }
      const uint64_t hit = __ballot(i0 + lane < hi && past(before + sum));
      if (hit != 0) {
        if (lane == 0) *sh_at = i0 + __ffsll(static_cast<unsigned long long>(hit)) - 1;
        break;
      }
      before += static_cast<u64>(__shfl(static_cast<long long>(sum), 63, 64));
    }
  }
  __syncthreads();
  return *sh_at;
}

struct Border {
  uint32_t key;  // tokens of a greater key are kept,
  uint32_t ties; // and the first so many of this key
  u64 above;     // weight of the tokens of a greater key
};

struct Shared {
  u64 sums[kWaves];
  u64 weights[256];
  uint32_t counts[256];
  int at;
};

// The key at which `past(count, weight)` of all tokens down to it first holds, from
// histograms over its bytes; all tokens' least key where it never does.
template <typename T, typename Past>
__device__ Border border_of(const Row& r, int vocab, Shared& sh, bool weigh, Past past) {
  uint32_t prefix = 0;
  u64 above = 0;
  uint32_t count = 0, in_key = 0;
  for (int shift = 24; shift >= 0; shift -= 8) {
    __syncthreads();
    for (int i = threadIdx.x; i < 256; i += kThreads) sh.weights[i] = 0, sh.counts[i] = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < vocab; i += kThreads) {
      const uint32_t key = key_of(logit_at<T>(r.logits, i));
      if (shift < 24 && (key >> (shift + 8)) != prefix) continue;
      const int bin = (key >> shift) & 255;
      atomicAdd(&sh.counts[bin], 1u);
      if (weigh) atomicAdd(&sh.weights[bin], weight_of(r, key));
    }
    __syncthreads();
    int bin = 255, least = 0;
    for (; bin >= 0; --bin) {
      if (sh.counts[bin] == 0) continue;
      least = bin;
      if (past(count + sh.counts[bin], above + sh.weights[bin])) break;
      count += sh.counts[bin];
      above += sh.weights[bin];
    }
    if (bin < 0) {  // never: the border is the least key there is
      bin = least;
      count -= sh.counts[bin];
      above -= sh.weights[bin];
    }
    prefix = (prefix << 8) | bin;
    in_key = sh.counts[bin];
  }
  // the fewest tokens of the key for which it holds
  const u64 w = weigh ? weight_of(r, prefix) : 0;
  uint32_t lo = 1, hi = in_key;
  while (lo < hi) {
    const uint32_t mid = lo + (hi - lo) / 2;
    if (past(count + mid, above + mid * w))
      hi = mid;
    else
      lo = mid + 1;
  }
  return {prefix, lo, above};
}

template <typename T>
__global__ __launch_bounds__(kThreads) void sample_kernel(SampleArgs a) {
  __shared__ Shared sh;
  const int b = blockIdx.x, tid = threadIdx.x, vocab = a.vocab;
  Row r;
  r.logits = static_cast<const char*>(a.logits) +
             b * a.stride * static_cast<int64_t>(std::is_same<T, f32_t>::value ? 4 : 2);
  u64 best = 0;  // key, then the lowest index
  for (int i = tid; i < vocab; i += kThreads) {
    const u64 k = (static_cast<u64>(key_of(logit_at<T>(r.logits, i))) << 32) | ~static_cast<uint32_t>(i);
    best = k > best ? k : best;
  }
  best = across<true>(best, sh.sums);
  r.top = static_cast<uint32_t>(best >> 32);
  const int first = static_cast<int>(~static_cast<uint32_t>(best));
  const double temperature = a.temperatures ? a.temperatures[b] : a.temperature;
  if (r.top <= kLeastKey || !(temperature > 0)) {
    if (tid == 0) {
      a.tokens[b] = r.top <= kLeastKey ? -1 : first;
      if (a.logprobs) a.logprobs[b] = r.top <= kLeastKey ? -__builtin_inff() : 0.f;
    }
    return;
  }
  r.max = logit_of(r.top);
  r.inv = 1.0 / temperature;
  const int64_t top_k = a.top_ks ? a.top_ks[b] : a.top_k;
  const double top_p = a.top_ps ? a.top_ps[b] : a.top_p;
  const double min_p = fmin(a.min_ps ? a.min_ps[b] : a.min_p, 1.0);

  Border border = {0, 0, 0};  // every key is greater
  if (top_k > 0 && top_k < vocab)
    border = border_of<T>(r, vocab, sh, top_p < 1, [&](uint32_t n, u64) { return n >= top_k; });
  if (top_p < 1) {
    u64 all;
    if (border.key != 0) {
      all = border.above + border.ties * weight_of(r, border.key);
    } else {
      all = 0;
      for (int i = tid; i < vocab; i += kThreads) all += weight_of(r, key_of(logit_at<T>(r.logits, i)));
      all = across<false>(all, sh.sums);
    }
    // (the first token's weight before it is 0: it is kept whatever top_p)
    const double share = top_p * static_cast<double>(all);
    const Border p = border_of<T>(r, vocab, sh, true,
                                  [&](uint32_t, u64 w) { return static_cast<double>(w) >= share; });
    if (p.key > border.key || (p.key == border.key && p.ties < border.ties)) border = p;
  }
  int last_tie = -1;  // the border key's tokens up to this one are kept
  if (border.key != 0)
    last_tie = find_first(vocab, [&](int i) -> u64 { return key_of(logit_at<T>(r.logits, i)) == border.key; },
                          [&](u64 n) { return n >= border.ties; }, sh.sums, &sh.at);
  const auto kept = [&](int i) -> u64 {
    const uint32_t key = key_of(logit_at<T>(r.logits, i));
    if (key < border.key || (key == border.key && i > last_tie)) return 0;
    if (key != r.top && !(exp(exponent_of(r, key)) >= min_p)) return 0;
    return weight_of(r, key);
  };
  u64 all = 0;
  for (int i = tid; i < vocab; i += kThreads) all += kept(i);
  all = across<false>(all, sh.sums);
  const double target = fmin(fmax(static_cast<double>(a.uniforms[b]), 0.0), 1.0) * static_cast<double>(all);
  int token = find_first(vocab, kept, [&](u64 w) { return static_cast<double>(w) > target; }, sh.sums, &sh.at);
  if (token >= vocab)  // (a number of 1): the last one
    token = find_first(vocab, kept, [&](u64 w) { return w >= all; }, sh.sums, &sh.at);
  if (tid == 0) {
    a.tokens[b] = token;
    if (a.logprobs)
      a.logprobs[b] = static_cast<float>(exponent_of(r, key_of(logit_at<T>(r.logits, token))) -
                                         log(static_cast<double>(all) / (1ull << kWeightBits)));
  }
}

}  // namespace
}  // namespace fpv2

extern "C" int fpv2_sample_tokens(const void* logits, const float* uniforms, int dtype,
                                  const fpv2_sample_params* params, int64_t* tokens,
                                  float* logprobs, void* stream) {
  using namespace fpv2;
  const char* name = "fpv2_sample_tokens";
  if (params == nullptr) return fail(FPV2_ERR_ARGUMENT, "%s: null params", name);
  const fpv2_sample_params& p = *params;
  if (dtype != FPV2_F32 && dtype != FPV2_BF16 && dtype != FPV2_F16)
    return fail(FPV2_ERR_UNSUPPORTED, "%s: dtype must be float32, bf16 or f16", name);
  if (p.batch < 0 || p.batch > 0x7fffffff || p.vocab <= 0 || p.logits_stride < 0)
    return fail(FPV2_ERR_ARGUMENT, "%s: bad batch, vocab or stride", name);
  if (p.vocab > FPV2_MAX_VOCAB)
    return fail(FPV2_ERR_UNSUPPORTED, "%s: more than %d tokens", name, FPV2_MAX_VOCAB);
  if (p.batch == 0) return FPV2_OK;
  if (!logits || !uniforms || !tokens) return fail(FPV2_ERR_ARGUMENT, "%s: null pointer", name);
  SampleArgs a{logits,    uniforms,      p.temperatures, p.top_ks, p.top_ps,  p.min_ps,
               tokens,    logprobs,      p.temperature,  p.top_p,  p.min_p,   p.top_k,
               p.logits_stride, static_cast<int>(p.vocab)};
  const hipStream_t s = static_cast<hipStream_t>(stream);
  const dim3 grid(static_cast<unsigned>(p.batch)), block(kThreads);
  if (dtype == FPV2_F32)
    hipLaunchKernelGGL(sample_kernel<f32_t>, grid, block, 0, s, a);
  else if (dtype == FPV2_BF16)
    hipLaunchKernelGGL(sample_kernel<bf16_t>, grid, block, 0, s, a);
  else
    hipLaunchKernelGGL(sample_kernel<f16_t>, grid, block, 0, s, a);
  return check_launch("sample_kernel");
}
