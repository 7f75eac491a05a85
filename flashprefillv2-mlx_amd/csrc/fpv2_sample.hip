// Sampling with temperature, top-k, top-p and min-p from given random numbers.
//
// The weight of a token is exp((logit - max) / temperature) in float64, rounded to
// an integer of 2^-44: sums of up to 2^19 of them are exact in 64 bits, so that
// histograms can be added in any order and a token next to a border is the same
// in every call.  A token's rank is a number of 52 bits: its logit's bits, ordered as
// unsigned integers, above the complement of its index.  Ranks are distinct, and the
// kept tokens are the ones from some least rank on: no sort is needed, only
// the ranks at which the count (top-k) and the weight (top-p) of all tokens from
// there on reach their limits.
//
// A short row is one workgroup's.  A long one takes passes over chunks of it, bound by
// reading the logits (the second and third time from the caches):
//   1. the greatest logit;
//   2. a histogram over (max - logit) / temperature, of the count and with top-p alone of
//      the weight, or the chunks' sums where the row has neither top-k nor top-p;
//   3. the tokens of the histogram's bin that holds the border go to a list, the ones
//      above it into the chunks' sums, or where they are few to the list too;
//   4. one workgroup finds the borders in the list and the token in it, or in its chunk.
// What bounds it: for one row the four launches, each a chain of loads and barriers (151936
// float32 logits with top-k and top-p: 3.0 + 5.2 + 6.0 + 7.6 us); for many the
// second pass's float64 (48 bf16 rows of 151936 with settings of their own: 6 + 22 + 14 +
// 13 us; 160 float32 rows of 50001 with min-p: 9 + 8 + 7 us, 3.5 TB/s in the first).
// A border in a bin of more tokens than a list holds is left to the row's one workgroup,
// some passes over the whole row: 0.4 to 0.6 ms for 151936 equal logits, for top-k of 5000
// with top-p, for 2^18 ordinary logits at a temperature of 2 with a top-p of 0.7 (at 1: 31 us);
// 0.8 ms where fewer tokens than top-k are not masked (the border is among the -inf ones),
// 1.7 ms with top-p as well; 1.1 ms for 2^19 ordinary logits with top-p.
#include "fpv2_common.h"
#include "fpv2_decode.h"

namespace fpv2 {
namespace {

typedef unsigned long long u64;
constexpr int kRowThreads = 1024;   // of a workgroup that has a row alone
// of one that finishes a row of chunks (one row with top-k 100: 256 threads 8.9, 512 7.6, 1024 9.6 us)
constexpr int kFinishThreads = 512;
constexpr int kChunkThreads = 256;  // of one that has a chunk
constexpr int kWeightBits = 44;
constexpr int kIndexBits = 20;
constexpr int kRankBits = 32 + kIndexBits;
constexpr int kBins = 1024;     // of the histogram,
constexpr float kPerUnit = 32;  // so many to a unit of the exponent
// and so many to a unit of the logits at least: high temperatures draw the logits together
// (one row of 151936, top-p 0.9 at a temperature of 30: all of it one workgroup's, 338 us,
// against 29)
constexpr double kPerLogit = 16;
constexpr int kList = 4096;     // tokens of a row's list
constexpr int kChunkList = 512; // of which a chunk's workgroup collects in LDS
constexpr int kMaxChunks = 256;
constexpr int kEach = 8;        // tokens of a thread where one is searched for
constexpr int kFew = kFinishThreads / 2;  // tokens that are compared with one another
constexpr int kMostChunk = kFinishThreads * kEach;
constexpr int kRoots = 64;      // powers 2^(k / kRoots) of which a weight is made

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
  // chunks of a long row, and its workspace
  int chunks, chunk, group;  // (in the passes after the first, `group` of them a workgroup)
  u64* best;         // [batch][chunks] greatest rank of a chunk
  u64* sums;         // [batch][chunks] weight of a chunk's tokens that are kept for sure
  u64* weights;      // [batch][kBins]
  u64* list;         // [batch][kList]
  uint32_t* counts;  // [batch][kBins]
  uint32_t* listed;  // [batch]
};

struct f32_t { float v; };
template <typename T> constexpr int kLogitBytes = 2;
template <> constexpr int kLogitBytes<f32_t> = 4;
template <typename T>
__device__ __forceinline__ float logit_at(const void* row, int i) {
  return Elem<T>::to_float(static_cast<const uint16_t*>(row)[i]);
}
template <>
__device__ __forceinline__ float logit_at<f32_t>(const void* row, int i) {
  return static_cast<const float*>(row)[i];
}
// Logit j of a 16-byte vector.
template <typename T>
__device__ __forceinline__ float logit_in(u32x4 v, int j) {
  return Elem<T>::to_float(j % 2 ? v[j / 2] >> 16 : v[j / 2] & 0xffffu);
}
template <>
__device__ __forceinline__ float logit_in<f32_t>(u32x4 v, int j) {
  return __uint_as_float(v[j]);
}

// Order-preserving key: -inf and NaN least, both zeros alike.
constexpr uint32_t kLeastKey = 0x007fffffu;  // of -inf
__device__ __forceinline__ float without_nan(float x) { return fmaxf(x, neg_inf()); }
__device__ __forceinline__ uint32_t key_of(float x) {
  const uint32_t b = __float_as_uint(without_nan(x) + 0.f);
  return b ^ (static_cast<uint32_t>(static_cast<int32_t>(b) >> 31) | 0x80000000u);
}
__device__ __forceinline__ float logit_of(uint32_t key) {
  return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key);
}
__device__ __forceinline__ u64 rank_of(uint32_t key, int i) {
  return (static_cast<u64>(key) << kIndexBits) | ((1u << kIndexBits) - 1 - i);
}
__device__ __forceinline__ uint32_t key_in(u64 rank) { return static_cast<uint32_t>(rank >> kIndexBits); }
__device__ __forceinline__ int index_in(u64 rank) {
  return (1 << kIndexBits) - 1 - static_cast<int>(rank & ((1u << kIndexBits) - 1));
}

// A row's settings and greatest logit.
struct Row {
  const void* logits;
  uint32_t top;     // greatest key
  float top_logit;
  double max, inv;  // the same, 1 / temperature
  double scale;     // kRoots log2 e / temperature
  const double* roots;
  float bins;       // of the histogram to a unit of the logits
  u64 least;        // weight from which on min_p keeps
  float reached;    // temperature, rounded up
  float from;       // a logit below all that min_p keeps with any weight
  double top_p;
  int64_t top_k;    // 0: no limit
  bool greedy, limited;

  // A logit below all whose weight's log is -units or more (float arithmetic, and
  // units good to 2^-19, are off by less than what is taken off).
  __device__ __forceinline__ float reach(float units) const {
    if (top_logit == __builtin_inff()) return top_logit;  // (no other has weight)
    const float down = units * reached * 1.00001f;
    return (top_logit - down) - (fabsf(top_logit) + down) * 0x1p-20f;
  }
};

template <typename T>
__device__ __forceinline__ const void* row_of(const SampleArgs& a, int b) {
  return static_cast<const char*>(a.logits) + b * a.stride * kLogitBytes<T>;
}
// (the loads of a pass come first, so that it waits for memory once)
struct Settings {
  double temperature, top_p, min_p;
  int64_t top_k;
};
__device__ __forceinline__ Settings load_settings(const SampleArgs& a, int b) {
  return {a.temperatures ? a.temperatures[b] : a.temperature, a.top_ps ? a.top_ps[b] : a.top_p,
          a.min_ps ? a.min_ps[b] : a.min_p, a.top_ks ? a.top_ks[b] : a.top_k};
}
template <typename T>
__device__ __forceinline__ Row row_with(const SampleArgs& a, int b, const Settings& set, u64 best,
                                        const double* roots) {
  Row r;
  r.roots = roots;
  r.logits = row_of<T>(a, b);
  r.top = key_in(best);
  r.max = r.top_logit = logit_of(r.top);
  const double temperature = fmin(set.temperature, 1e30);
  r.greedy = r.top <= kLeastKey || !(set.temperature > 0);
  r.inv = fmin(1.0 / temperature, 1e300);
  r.scale = r.inv * (1.4426950408889634 * kRoots);
  r.bins = static_cast<float>(fmin(fmax(kPerUnit * r.inv, kPerLogit), 1e38));
  r.top_p = set.top_p;
  r.top_k = set.top_k;
  if (r.top_k < 0 || r.top_k >= a.vocab) r.top_k = 0;
  const double min_p = fmin(fmax(set.min_p, 0.0), 1.0);
  r.least = static_cast<u64>(min_p * (1ull << kWeightBits));
  r.reached = static_cast<float>(temperature) * 1.000001f;
  r.limited = !r.greedy && (r.top_k > 0 || r.top_p < 1);
  r.from = r.reach(fminf(-__logf(static_cast<float>(min_p)) + 1e-5f, 32.f));
  return r;
}

// log of a logit's weight.
__device__ __forceinline__ double exponent_of(const Row& r, float x) {
  return x == r.top_logit ? 0.0 : (static_cast<double>(without_nan(x)) - r.max) * r.inv;
}
// (by the workgroup's first threads, before a barrier: the series leaves 2^-62)
__device__ __forceinline__ void fill_roots(double* roots) {
  if (threadIdx.x < kRoots) {
    const double f = threadIdx.x * (0.6931471805599453 / kRoots);
    double p = 1;
#pragma unroll
    for (int i = 17; i > 0; --i) p = __builtin_fma(p, f * (1.0 / i), 1.0);
    roots[threadIdx.x] = p;
  }
}
// Weight of a logit, without branches, as a pass's threads do this for every logit:
// e^z = 2^((n + f) / kRoots), |f| <= 1/2, is root n mod kRoots with n / kRoots added to its
// exponent, times the series in f to the fifth power, which leaves 2^-54.  n and the
// rounding to an integer come of sums with a large number, whose low bits they are.
// (Half as many instructions in float64 as the series on |z| <= ln 2 / 2: the second pass
// over 48 rows of 151936 without limits took 17.6 us, and takes 14.3.)
__device__ __forceinline__ u64 weight_of(const Row& r, float x) {
  const double d = static_cast<double>(without_nan(x)) - r.max;
  const double t = fmax((x == r.top_logit ? 0.0 : d) * r.scale, -64.0 * kRoots);  // (no weight there)
  constexpr double kWhole = 6755399441055744.0;  // 1.5 * 2^52
  const double whole = t + kWhole;
  const int n = static_cast<int>(__double_as_longlong(whole));
  const double f = t - (whole - kWhole);
  constexpr double l = 0.6931471805599453 / kRoots;
  double p = l * l * l * l * l / 120;
  p = __builtin_fma(p, f, l * l * l * l / 24);
  p = __builtin_fma(p, f, l * l * l / 6);
  p = __builtin_fma(p, f, l * l / 2);
  p = __builtin_fma(p, f, l);
  p = __builtin_fma(p, f, 1.0);
  const u64 root = static_cast<u64>(__double_as_longlong(r.roots[n & (kRoots - 1)]));
  const u64 power = static_cast<u64>(static_cast<uint32_t>((n >> 6) + kWeightBits) << 20) << 32;
  const double w = __builtin_fma(__longlong_as_double(static_cast<long long>(root + power)), p, 4503599627370496.0);
  return static_cast<u64>(__double_as_longlong(w)) & 0xfffffffffffffull;
}
static_assert(kRoots == 1 << 6, "a weight's power");
// Bin of a logit: any number that doesn't fall where the logit rises will do, for what
// lies in a bin is decided by ranks.
__device__ __forceinline__ int bin_of(const Row& r, float x) {
  const float down = (r.top_logit - without_nan(x)) * r.bins;
  return x == r.top_logit ? 0 : static_cast<int>(fminf(down, static_cast<float>(kBins - 1)));
}
// Weight of a token if min_p keeps it.
__device__ __forceinline__ u64 likely_weight(const Row& r, float x) {
  const u64 w = weight_of(r, x);
  return w >= r.least ? w : 0;
}

// Sum (or greatest) of a value over a wave's lanes up to this one, by DPP: shifts
// within rows of 16 lanes, then the rows' last lanes to the rows after them.
// (Through shuffles the six dependent steps take three times as long.)
template <int CTRL, int ROWS>
__device__ __forceinline__ u64 from_lanes(u64 v) {  // 0 where there is no such lane
  const uint32_t lo = __builtin_amdgcn_update_dpp(0, static_cast<int>(v), CTRL, ROWS, 0xf, false);
  const uint32_t hi = __builtin_amdgcn_update_dpp(0, static_cast<int>(v >> 32), CTRL, ROWS, 0xf, false);
  return (static_cast<u64>(hi) << 32) | lo;
}
template <bool MAX = false>
__device__ __forceinline__ u64 wave_scan(u64 v) {
  const auto with = [&](u64 o) { v = MAX ? (o > v ? o : v) : v + o; };
  with(from_lanes<0x111, 0xf>(v));  // row_shr 1, 2, 4, 8
  with(from_lanes<0x112, 0xf>(v));
  with(from_lanes<0x114, 0xf>(v));
  with(from_lanes<0x118, 0xf>(v));
  with(from_lanes<0x142, 0xa>(v));  // row_bcast 15, to the odd rows
  with(from_lanes<0x143, 0xc>(v));  // row_bcast 31, to the upper half
  return v;
}
__device__ __forceinline__ u64 last_lane(u64 v) {
  const uint32_t lo = __builtin_amdgcn_readlane(static_cast<int>(v), 63);
  const uint32_t hi = __builtin_amdgcn_readlane(static_cast<int>(v >> 32), 63);
  return (static_cast<u64>(hi) << 32) | lo;
}
// Sum (or greatest) of a value of each of the workgroup's threads, in every thread.
template <int THREADS, bool MAX>
__device__ __forceinline__ u64 across(u64 v, u64* sh) {
  v = wave_scan<MAX>(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 63) sh[threadIdx.x >> 6] = v;
  __syncthreads();
  v = sh[0];
#pragma unroll
  for (int w = 1; w < THREADS / 64; ++w) v = MAX ? (sh[w] > v ? sh[w] : v) : v + sh[w];
  return v;
}

// f(i, logits) is called for logits of token i and the next ones: the 16 bytes of a
// load, or one.
template <int N>
struct Logits {
  float x[N];
  __device__ __forceinline__ float greatest() const {  // (NaN if all are)
    float m = x[0];
#pragma unroll
    for (int j = 1; j < N; ++j) m = fmaxf(m, x[j]);
    return m;
  }
};
template <typename T, typename F>
__device__ __forceinline__ void with_vector(int i, u32x4 v, F f) {
  constexpr int N = 16 / kLogitBytes<T>;
  Logits<N> logits;
#pragma unroll
  for (int j = 0; j < N; ++j) logits.x[j] = logit_in<T>(v, j);
  f(i, logits);
}
// The tokens [lo, hi) of a row: whole vectors from the first aligned logit on, and a
// thread's token before or after them.
template <typename T, int THREADS>
struct Span {
  static constexpr int N = 16 / kLogitBytes<T>;
  int first, vectors, edge;  // edge: -1 for none
  const char* at;
  __device__ __forceinline__ Span(const void* row, int lo, int hi) {
    const uintptr_t from = reinterpret_cast<uintptr_t>(row) + static_cast<uintptr_t>(lo) * kLogitBytes<T>;
    const int head = min(hi - lo, static_cast<int>((16 - from % 16) % 16) / kLogitBytes<T>);
    const int tid = threadIdx.x;
    first = lo + head;
    vectors = (hi - first) / N;
    const int last = first + N * vectors;
    edge = tid < head ? lo + tid : last + tid - head;
    if (edge >= hi || tid >= 2 * N) edge = -1;
    at = static_cast<const char*>(row) + static_cast<int64_t>(first) * kLogitBytes<T>;
  }
  __device__ __forceinline__ u32x4 load(int v) const { return load16(at + 16 * static_cast<int64_t>(v)); }
};
// A workgroup's chunk, loaded at once: before the pass has its row's settings.
template <typename T>
struct Chunk {
  using Vectors = Span<T, kChunkThreads>;
  static constexpr int kEachThread = kMostChunk / (Vectors::N * kChunkThreads);
  Vectors span;
  u32x4 v[kEachThread];
  float edge;
  __device__ __forceinline__ Chunk(const SampleArgs& a, const void* row, int c)
      : span(row, c * a.chunk, min(a.vocab, (c + 1) * a.chunk)) {
#pragma unroll
    for (int k = 0; k < kEachThread; ++k) {
      const int i = threadIdx.x + k * kChunkThreads;
      v[k] = u32x4{};
      if (i < span.vectors) v[k] = span.load(i);
    }
    edge = span.edge >= 0 ? logit_at<T>(row, span.edge) : 0.f;
  }
  template <typename F>
  __device__ __forceinline__ void for_vectors(F f) const {
    if (span.edge >= 0) f(span.edge, Logits<1>{{edge}});
#pragma unroll
    for (int k = 0; k < kEachThread; ++k) {
      const int i = threadIdx.x + k * kChunkThreads;
      if (i < span.vectors) with_vector<T>(span.first + Vectors::N * i, v[k], f);
    }
  }
};
// f(i, logit) for the tokens [lo, hi) of a row, in any order, by THREADS threads.
template <typename T, int THREADS, typename F>
__device__ __forceinline__ void for_each(const void* row, int lo, int hi, F f) {
  const Span<T, THREADS> span(row, lo, hi);
  if (span.edge >= 0) f(span.edge, logit_at<T>(row, span.edge));
#pragma unroll 1
  for (int v = threadIdx.x; v < span.vectors; v += THREADS)
    with_vector<T>(span.first + span.N * v, span.load(v), [&](int i, const Logits<span.N>& logits) {
#pragma unroll
      for (int j = 0; j < span.N; ++j) f(i + j, logits.x[j]);
    });
}

// The greatest rank of tokens, one after the other.
struct Best {
  float logit = neg_inf();
  int at = 1 << kIndexBits;
  __device__ __forceinline__ void add(int i, float x) {
    at = x > logit || (x == logit && i < at) ? i : at;
    logit = fmaxf(x, logit);
  }
  __device__ __forceinline__ u64 rank() const { return at < 1 << kIndexBits ? rank_of(key_of(logit), at) : 0; }
};

struct Shared {
  u64 sums[kRowThreads / 64];
  u64 weights[256];
  uint32_t counts[256];
  u64 found[4];
  int at;
};

// The first i in [lo, hi), at most kEach a thread, for which past(before + value(lo) +
// .. + value(i)) holds, or hi.
template <int THREADS, typename Value, typename Past>
__device__ int find_first(int lo, int hi, u64 before, Value value, Past past, Shared& sh) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int each = (hi - lo + THREADS - 1) / THREADS;
  const int from = min(hi, lo + tid * each), to = min(hi, from + each);
  u64 v[kEach], sum = 0;
#pragma unroll
  for (int j = 0; j < kEach; ++j) {
    v[j] = from + j < to ? value(from + j) : 0;
    sum += v[j];
  }
  const u64 upto = wave_scan(sum);
  __syncthreads();
  if (lane == 63) sh.sums[wave] = upto;
  if (tid == 0) sh.at = hi;
  __syncthreads();
  u64 run = before + upto - sum;
  for (int w = 0; w < wave; ++w) run += sh.sums[w];
  if (sum > 0 && past(run + sum) && (run == before || !past(run))) {
    int at = -1;
#pragma unroll
    for (int j = 0; j < kEach; ++j) {
      run += v[j];
      if (at < 0 && v[j] > 0 && past(run)) at = from + j;
    }
    sh.at = at;
  }
  __syncthreads();
  return sh.at;
}

// Of a group of tokens (each(f) calls f(rank, weight()) for all of them) the greatest rank from
// which on past(count, weight) holds, given the count and weight of the tokens
// above the group; 0 where it never does.  *weight: weight of the tokens from there on.
// Histograms over the rank's bits, 8 at a time from the first that differ, until one
// token is left in the border's bin.
template <int THREADS, typename Each, typename Past>
__device__ u64 least_rank(const Row& r, Each each, u64 count, u64 weight, Past past, bool weigh,
                          u64* weight_from, Shared& sh) {
  const int tid = threadIdx.x, lane = tid & 63;
  u64 low = ~0ull, high = 0;
  each([&](u64 rank, auto) {
    low = rank < low ? rank : low;
    high = rank > high ? rank : high;
  });
  high = across<THREADS, true>(high, sh.sums);
  low = ~across<THREADS, true>(~low, sh.sums);
  int shift = low < high ? 64 - __clzll(static_cast<long long>(low ^ high)) - 8 : 0;
  int width = 8;  // the bits shift .. shift + width - 1 are the bin
  if (shift < 0) shift = 0;
  u64 prefix = high >> (shift + width);
  for (;;) {
    __syncthreads();
    if (tid < 256) sh.weights[tid] = 0, sh.counts[tid] = 0;
    __syncthreads();
    each([&](u64 rank, auto of) {
      if ((rank >> (shift + width)) != prefix) return;
      const int bin = static_cast<int>(rank >> shift) & ((1 << width) - 1);
      atomicAdd(&sh.counts[bin], 1u);
      if (weigh) atomicAdd(&sh.weights[bin], of());
    });
    __syncthreads();
    if (tid < 64) {
      // the lane's bins 255 - 4 lane and the three below
      u64 c[4], w[4], cs = 0, ws = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int bin = 255 - 4 * lane - j;
        c[j] = cs += sh.counts[bin];
        w[j] = ws += sh.weights[bin];
      }
      const u64 c0 = count + wave_scan(cs) - cs, w0 = weight + wave_scan(ws) - ws;
      int mine = -1;
#pragma unroll
      for (int j = 3; j >= 0; --j) {
        const u64 own = c[j] - (j > 0 ? c[j > 0 ? j - 1 : 0] : 0);
        if (own > 0 && past(c0 + c[j], w0 + w[j])) mine = j;
      }
      const uint64_t hit = __ballot(mine >= 0);
      if (lane == 0) sh.found[0] = hit;
      if (hit != 0 && lane == __ffsll(static_cast<unsigned long long>(hit)) - 1) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (j == mine) {
            const u64 before_c = j > 0 ? c[j > 0 ? j - 1 : 0] : 0, before_w = j > 0 ? w[j > 0 ? j - 1 : 0] : 0;
            sh.found[1] = (static_cast<u64>(255 - 4 * lane - j) << 32) | (c[j] - before_c);
            sh.found[2] = c0 + before_c;
            sh.found[3] = w0 + before_w;
          }
      }
    }
    __syncthreads();
    if (sh.found[0] == 0) {  // never (the first time round: later the bin has it)
      *weight_from = weight;
      return 0;
    }
    const int bin = static_cast<int>(sh.found[1] >> 32);
    const uint32_t in_bin = static_cast<uint32_t>(sh.found[1]);
    prefix = (prefix << width) | bin;
    count = sh.found[2];
    weight = sh.found[3];
    if (in_bin == 1 || shift == 0) {
      *weight_from = weight + sh.weights[bin];
      return prefix << shift;
    }
    width = shift < 8 ? shift : 8;
    shift -= width;
  }
}

// The least kept rank of a row whose borders lie in a group of tokens.
template <int THREADS, typename Each>
__device__ u64 border_of(const Row& r, Each each, u64 count, u64 weight, u64 all, Shared& sh) {
  u64 least = 0, from = all;
  if (r.top_k > 0)
    least = least_rank<THREADS>(r, each, count, weight, [&](u64 n, u64) { return n >= static_cast<u64>(r.top_k); },
                       r.top_p < 1, &from, sh);
  if (r.top_p < 1) {
    // (a token is kept while the weight before it is less than the share)
    const double share = r.top_p * static_cast<double>(from);
    const u64 p = least_rank<THREADS>(r, each, count, weight,
                             [&](u64, u64 w) { return static_cast<double>(w) >= share; }, true, &from, sh);
    least = p > least ? p : least;
  }
  return least;
}

__device__ __forceinline__ void write_greedy(const SampleArgs& a, int b, u64 best) {
  const bool none = key_in(best) <= kLeastKey;
  a.tokens[b] = none ? -1 : index_in(best);
  if (a.logprobs) a.logprobs[b] = none ? -__builtin_inff() : 0.f;
}

__device__ __forceinline__ double target_of(const SampleArgs& a, int b, u64 all) {
  return fmin(fmax(static_cast<double>(a.uniforms[b]), 0.0), 1.0) * static_cast<double>(all);
}
__device__ __forceinline__ void write_token(const SampleArgs& a, const Row& r, int b, int token, float logit, u64 all) {
  a.tokens[b] = token;
  if (a.logprobs)
    a.logprobs[b] = static_cast<float>(exponent_of(r, logit) - log(static_cast<double>(all) / (1ull << kWeightBits)));
}

// The token: kept weight `all`, of which `before` lies before the tokens [lo, hi), where
// the one searched for is.
template <typename T, int THREADS>
__device__ void pick(const SampleArgs& a, const Row& r, int b, u64 least, u64 all, u64 before, double target,
                     int lo, int hi, Shared& sh) {
  const auto kept = [&](int i) -> u64 {
    const float x = logit_at<T>(r.logits, i);
    return x >= r.from && rank_of(key_of(x), i) >= least ? likely_weight(r, x) : 0;
  };
  const int token = min(hi - 1, find_first<THREADS>(
      lo, hi, before, kept, [&](u64 w) { return static_cast<double>(w) > target || w == all; }, sh));
  if (threadIdx.x == 0) write_token(a, r, b, token, logit_at<T>(r.logits, token), all);
}

// Kept weight of each chunk into LDS and of the row, then the token.
template <typename T>
__device__ void pick_in_chunks(const SampleArgs& a, const Row& r, int b, u64 least, u64* chunk_sums, Shared& sh) {
  const int tid = threadIdx.x, lane = tid & 63;
  __syncthreads();
  u64 mine = tid < a.chunks ? chunk_sums[tid] : 0;
  const u64 all = across<kFinishThreads, false>(mine, sh.sums);
  const double target = target_of(a, b, all);
  if (tid < 64) {  // kMaxChunks: four a lane
    u64 c[4], sum = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) c[j] = sum += 4 * lane + j < a.chunks ? chunk_sums[4 * lane + j] : 0;
    const u64 before = wave_scan(sum) - sum;
    int at = -1;
#pragma unroll
    for (int j = 3; j >= 0; --j)
      if (static_cast<double>(before + c[j]) > target || before + c[j] == all) at = j;
    const uint64_t hit = __ballot(at >= 0);
    if (lane == __ffsll(static_cast<unsigned long long>(hit)) - 1) {
      u64 up = before;
#pragma unroll
      for (int j = 1; j < 4; ++j)
        if (j == at) up = before + c[j - 1];
      sh.at = 4 * lane + at;
      sh.found[0] = up;
    }
  }
  __syncthreads();
  const int chunk = sh.at;
  const u64 before = sh.found[0];
  __syncthreads();
  pick<T, kFinishThreads>(a, r, b, least, all, before, target, chunk * a.chunk, min(a.vocab, (chunk + 1) * a.chunk), sh);
}

// A whole row by one workgroup.
template <typename T>
__global__ __launch_bounds__(kRowThreads) void sample_row_kernel(SampleArgs a) {
  __shared__ Shared sh;
  const int b = blockIdx.x;
  __shared__ double roots[kRoots];
  fill_roots(roots);
  Best mine;
  for_each<T, kRowThreads>(row_of<T>(a, b), 0, a.vocab, [&](int i, float x) { mine.add(i, x); });
  const u64 best = across<kRowThreads, true>(mine.rank(), sh.sums);
  const Row r = row_with<T>(a, b, load_settings(a, b), best, roots);
  if (r.greedy) {
    if (threadIdx.x == 0) write_greedy(a, b, best);
    return;
  }
  u64 least = 0;
  if (r.limited) {
    u64 all = 0;
    if (r.top_k == 0) {
      for_each<T, kRowThreads>(r.logits, 0, a.vocab, [&](int, float x) { all += weight_of(r, x); });
      all = across<kRowThreads, false>(all, sh.sums);
    }
    least = border_of<kRowThreads>(r, [&](auto f) {
      for_each<T, kRowThreads>(r.logits, 0, a.vocab, [&](int i, float x) {
        f(rank_of(key_of(x), i), [&] { return weight_of(r, x); });
      });
    }, 0, 0, all, sh);
  }
  u64 all = 0;
  for_each<T, kRowThreads>(r.logits, 0, a.vocab, [&](int i, float x) {
    if (rank_of(key_of(x), i) >= least) all += likely_weight(r, x);
  });
  all = across<kRowThreads, false>(all, sh.sums);
  pick<T, kRowThreads>(a, r, b, least, all, 0, target_of(a, b, all), 0, a.vocab, sh);
}

// ---- long rows -------------------------------------------------------------

template <typename T>
__global__ __launch_bounds__(kChunkThreads) void chunk_max_kernel(SampleArgs a) {
  __shared__ u64 sh[kChunkThreads / 64];
  const int c = blockIdx.x, b = blockIdx.y, tid = threadIdx.x;
  const Chunk<T> chunk(a, row_of<T>(a, b), c);
  // (the row's histogram and list for the next passes)
  if (a.counts != nullptr) {
    for (int i = c * kChunkThreads + tid; i < kBins; i += a.chunks * kChunkThreads) {
      a.counts[static_cast<int64_t>(b) * kBins + i] = 0;
      a.weights[static_cast<int64_t>(b) * kBins + i] = 0;
    }
    if (c == 0 && tid == 0) a.listed[b] = 0;
  }
  Best mine;
  chunk.for_vectors([&](int i, const auto& logits) {
    constexpr int N = sizeof(logits) / sizeof(float);
#pragma unroll
    for (int j = 0; j < N; ++j) mine.add(i + j, logits.x[j]);
  });
  const u64 best = across<kChunkThreads, true>(mine.rank(), sh);
  if (tid == 0) a.best[static_cast<int64_t>(b) * a.chunks + c] = best;
}

template <int THREADS>
__device__ __forceinline__ u64 row_best(const SampleArgs& a, int b, u64* sh) {
  u64 best = 0;
  for (int i = threadIdx.x; i < a.chunks; i += THREADS) {
    const u64 x = a.best[static_cast<int64_t>(b) * a.chunks + i];
    best = x > best ? x : best;
  }
  return across<THREADS, true>(best, sh);
}

// The row of a workgroup in a grid of [chunks][batch].  Rows differ in what they need: one
// after the other, and shifted by one from chunk to chunk, they spread over the CUs
// in whatever order kinds of rows come.  (The second pass over 48 rows of 151936 in an
// order of six kinds: 26.1 us with a row's chunks one after the other, when a CU had
// eight of a kind, against 23.8.)
__device__ __forceinline__ int spread_row() { return (blockIdx.x + blockIdx.y) % gridDim.x; }

// a.group chunks by a workgroup: one histogram of them in LDS, so that fewer are
// added to the row's (each line of it that an atomic goes to is one in memory).
template <typename T>
__global__ __launch_bounds__(kChunkThreads) void chunk_weigh_kernel(SampleArgs a) {
  __shared__ u64 sh[kChunkThreads / 64];
  __shared__ u64 weights[kBins];
  __shared__ uint32_t counts[kBins];
  const int b = spread_row(), tid = threadIdx.x;
  const int c0 = blockIdx.y * a.group, c1 = min(a.chunks, c0 + a.group);
  Chunk<T> chunk(a, row_of<T>(a, b), c0);
  const Settings set = load_settings(a, b);
  __shared__ double roots[kRoots];
  fill_roots(roots);
  const Row r = row_with<T>(a, b, set, row_best<kChunkThreads>(a, b, sh), roots);
  if (r.greedy) return;
  if (!r.limited) {
    for (int c = c0; c < c1; ++c) {
      if (c > c0) chunk = Chunk<T>(a, r.logits, c);
      u64 sum = 0;
      chunk.for_vectors([&](int, const auto& logits) {
        if (!(logits.greatest() >= r.from)) return;
        constexpr int N = sizeof(logits) / sizeof(float);
#pragma unroll
        for (int j = 0; j < N; ++j) sum += likely_weight(r, logits.x[j]);
      });
      sum = across<kChunkThreads, false>(sum, sh);
      if (tid == 0) a.sums[static_cast<int64_t>(b) * a.chunks + c] = sum;
    }
    return;
  }
  for (int i = tid; i < kBins; i += kChunkThreads) weights[i] = 0, counts[i] = 0;
  __syncthreads();
  const bool weigh = r.top_k == 0;  // (with top_k the borders' list is weighed)
  uint32_t far = 0;  // of the last bin, where masked tokens are
  u64 far_weight = 0;
  // (a load's weights before its atomics: the roots that are read in LDS come back in order)
  const auto add = [&](int, const auto& logits) {
    constexpr int N = sizeof(logits) / sizeof(float);
    int bin[N];
    u64 w[N];
#pragma unroll
    for (int j = 0; j < N; ++j) {
      bin[j] = bin_of(r, logits.x[j]);
      w[j] = 0;
    }
    if (weigh) {
#pragma unroll
      for (int j = 0; j < N; ++j) w[j] = weight_of(r, logits.x[j]);
    }
#pragma unroll
    for (int j = 0; j < N; ++j) {
      if (bin[j] == kBins - 1) {
        ++far;
        far_weight += w[j];
      } else {
        atomicAdd(&counts[bin[j]], 1u);
        if (weigh) atomicAdd(&weights[bin[j]], w[j]);
      }
    }
  };
  for (int c = c0; c < c1; ++c) {
    if (c > c0) chunk = Chunk<T>(a, r.logits, c);
    chunk.for_vectors(add);
  }
  if (far > 0) {
    atomicAdd(&counts[kBins - 1], far);
    atomicAdd(&weights[kBins - 1], far_weight);
  }
  __syncthreads();
  for (int i = tid; i < kBins; i += kChunkThreads)
    if (counts[i] > 0) {
      atomicAdd(&a.counts[static_cast<int64_t>(b) * kBins + i], counts[i]);
      if (weights[i] > 0) atomicAdd(&a.weights[static_cast<int64_t>(b) * kBins + i], weights[i]);
    }
}

// The bins [lo, hi] that hold a row's borders, and what lies above and in them.
struct Bins {
  int lo, hi;
  uint32_t above, in;
  u64 above_weight, all;
};

// A thread's share of the histogram, in order; the first 256 threads have it.
constexpr int kShare = kBins / 256;
struct HistShare {
  uint32_t c[kShare];
  u64 w[kShare];
};
__device__ __forceinline__ HistShare load_hist(const SampleArgs& a, int b) {
  HistShare h{};
  const int64_t at = static_cast<int64_t>(b) * kBins + threadIdx.x * kShare;
  if (threadIdx.x < 256 && a.counts != nullptr) {
    __builtin_memcpy(h.c, __builtin_assume_aligned(a.counts + at, 16), sizeof(h.c));
    __builtin_memcpy(h.w, __builtin_assume_aligned(a.weights + at, 16), sizeof(h.w));
  }
  return h;
}

__device__ Bins bins_of(const HistShare& h, const Row& r) {
  __shared__ u64 found[4];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const uint32_t(&c)[kShare] = h.c;
  const u64(&w)[kShare] = h.w;
  u64 cs = 0, ws = 0;
#pragma unroll
  for (int j = 0; j < kShare; ++j) cs += c[j], ws += w[j];
  u64 c_run = wave_scan(cs), w_run = wave_scan(ws);
  __shared__ u64 waves[2][4];
  if (lane == 63 && wave < 4) waves[0][wave] = c_run, waves[1][wave] = w_run;
  if (tid < 4) found[tid] = 0;
  __syncthreads();
  u64 all = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    c_run += i < wave ? waves[0][i] : 0;
    w_run += i < wave ? waves[1][i] : 0;
    all += waves[1][i];
  }
  c_run -= cs;
  w_run -= ws;
  // top_k alone or with top_p: the bin of token top_k; top_p alone: the share's
  const double share = r.top_p * static_cast<double>(all);
  const auto past = [&](u64 n, u64 weight) {
    return r.top_k > 0 ? n >= static_cast<u64>(r.top_k) : static_cast<double>(weight) >= share;
  };
  if (tid < 256) {
#pragma unroll
    for (int j = 0; j < kShare; ++j) {
      // (an empty bin is passed over: the border is a token's)
      if (c[j] > 0 && past(c_run + c[j], w_run + w[j]) && (c_run == 0 || !past(c_run, w_run))) {
        found[0] = tid * kShare + j;
        found[1] = c_run;
        found[2] = w_run;
        found[3] = c[j];
      }
      c_run += c[j];
      w_run += w[j];
    }
  }
  __syncthreads();
  Bins s;
  s.hi = static_cast<int>(found[0]);
  s.all = all;
  // all down to the bin for both limits, as top_p's border may lie anywhere above, and for
  // few tokens, among which the token is found without its chunk
  if ((r.top_k > 0 && r.top_p < 1) || found[1] + found[3] <= kFew) {
    s.lo = 0;
    s.above = 0;
    s.above_weight = 0;
    s.in = static_cast<uint32_t>(found[1] + found[3]);
  } else {
    s.lo = s.hi;
    s.above = static_cast<uint32_t>(found[1]);
    s.above_weight = found[2];
    s.in = static_cast<uint32_t>(found[3]);
  }
  return s;
}

template <typename T>
__global__ __launch_bounds__(kChunkThreads) void chunk_list_kernel(SampleArgs a) {
  __shared__ u64 sh[kChunkThreads / 64];
  __shared__ u64 list[kChunkList];
  __shared__ uint32_t listed, at;
  const int b = spread_row(), tid = threadIdx.x;
  const int c0 = blockIdx.y * a.group, c1 = min(a.chunks, c0 + a.group);
  Chunk<T> chunk(a, row_of<T>(a, b), c0);
  const Settings set = load_settings(a, b);
  const HistShare hist = load_hist(a, b);
  __shared__ double roots[kRoots];
  fill_roots(roots);
  const Row r = row_with<T>(a, b, set, row_best<kChunkThreads>(a, b, sh), roots);
  if (!r.limited) return;
  const Bins bins = bins_of(hist, r);
  if (bins.in > kList) return;  // the row's workgroup does it all
  // (the list holds as many as the histogram counted, if nobody writes the logits)
  const auto put = [&](uint32_t i, u64 rank) {
    if (i < kList) a.list[static_cast<int64_t>(b) * kList + i] = rank;
  };
  if (tid == 0) listed = 0;
  __syncthreads();
  for (int c = c0; c < c1; ++c) {
    u64 sum = 0;
    if (c > c0) chunk = Chunk<T>(a, r.logits, c);
    chunk.for_vectors([&](int i, const auto& logits) {
      if (bin_of(r, logits.greatest()) > bins.hi) return;
      constexpr int N = sizeof(logits) / sizeof(float);
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const float x = logits.x[j];
        const int bin = bin_of(r, x);
        if (bin > bins.hi) continue;
        if (bin < bins.lo) {
          sum += likely_weight(r, x);
          continue;
        }
        const u64 rank = rank_of(key_of(x), i + j);
        const uint32_t slot = atomicAdd(&listed, 1u);
        if (slot < kChunkList)
          list[slot] = rank;
        else
          put(atomicAdd(&a.listed[b], 1u), rank);
      }
    });
    sum = across<kChunkThreads, false>(sum, sh);
    if (tid == 0) a.sums[static_cast<int64_t>(b) * a.chunks + c] = sum;
  }
  __syncthreads();
  const uint32_t n = listed < kChunkList ? listed : kChunkList;
  if (tid == 0) at = n > 0 ? atomicAdd(&a.listed[b], n) : 0;
  __syncthreads();
  for (uint32_t i = tid; i < n; i += kChunkThreads) put(at + i, list[i]);
}

// At most kFew tokens of a list, compared all with all: each token by `parts` lanes next to
// one another, which have a part of the others each.
typedef u64 u64x2 __attribute__((ext_vector_type(2)));
struct Few {
  u64x2 tokens[kFew];  // rank and weight, 0 for none
};
struct Place {
  int n, parts, token, part;
  __device__ __forceinline__ explicit Place(int n)
      : n(n), parts(n <= kFew / 8 ? 16 : n <= kFew / 4 ? 8 : n <= kFew / 2 ? 4 : 2),
        token(static_cast<int>(threadIdx.x) / parts), part(static_cast<int>(threadIdx.x) % parts) {}
};
// Count and weight of the tokens that come before the lane's one.
template <typename Before>
__device__ __forceinline__ void sum_before(const Few& few, const Place& at, Before before, u64* count, u64* weight) {
  const u64 own = few.tokens[at.token][0];
  uint32_t c = 0;
  u64 w = 0;
#pragma unroll 1
  for (int j = at.part; j < at.n; j += 4 * at.parts) {  // (kFew / parts is a multiple of 4)
    u64x2 other[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) other[i] = few.tokens[j + i * at.parts];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const bool is = before(other[i][0], own);
      c += is;
      w += is ? other[i][1] : 0;
    }
  }
  u64 n = c;
  n += from_lanes<0xb1, 0xf>(n), w += from_lanes<0xb1, 0xf>(w);  // of pairs of lanes,
  if (at.parts > 2) n += from_lanes<0x4e, 0xf>(n), w += from_lanes<0x4e, 0xf>(w);    // fours,
  if (at.parts > 4) n += from_lanes<0x141, 0xf>(n), w += from_lanes<0x141, 0xf>(w);  // eights
  if (at.parts > 8) n += from_lanes<0x140, 0xf>(n), w += from_lanes<0x140, 0xf>(w);  // and sixteens
  *count = n;
  *weight = w;
}
// border_of for them (the first kFew threads bring one each).
__device__ u64 border_of_few(const Row& r, u64 rank, u64 weight, const Bins& bins, const Place& at, Few& few,
                             Shared& sh) {
  if (threadIdx.x < kFew) {
    few.tokens[threadIdx.x][0] = rank;
    few.tokens[threadIdx.x][1] = weight;
  }
  __syncthreads();
  u64 above, above_weight;
  sum_before(few, at, [](u64 other, u64 own) { return other > own; }, &above, &above_weight);
  above += bins.above;
  above_weight += bins.above_weight;
  bool kept = at.token < at.n && (r.top_k == 0 || above < static_cast<u64>(r.top_k));
  if (r.top_p < 1) {
    const u64 all = r.top_k == 0 ? bins.all
                                 : across<kFinishThreads, true>(kept ? above_weight + few.tokens[at.token][1] : 0, sh.sums);
    // (the first token has nothing before it: it is kept whatever the share)
    kept = kept && (above == 0 || static_cast<double>(above_weight) < r.top_p * static_cast<double>(all));
  }
  return ~across<kFinishThreads, true>(kept ? ~few.tokens[at.token][0] : 0, sh.sums);
}

// The token where all that may be kept are among them.
__device__ void pick_of_few(const SampleArgs& a, const Row& r, int b, u64 least, const Place& at, Few& few, Shared& sh) {
  const u64 rank = few.tokens[at.token][0], weight = few.tokens[at.token][1];
  const u64 w = at.part == 0 && at.token < at.n && rank >= least && weight >= r.least ? weight : 0;
  if (at.part == 0) few.tokens[at.token][1] = w;
  const u64 all = across<kFinishThreads, false>(w, sh.sums);
  u64 count, before;
  sum_before(few, at, [](u64 other, u64 own) { return index_in(other) < index_in(own); }, &count, &before);
  const double target = target_of(a, b, all);
  const auto past = [&](u64 v) { return static_cast<double>(v) > target || v == all; };
  if (w > 0 && past(before + w) && (before == 0 || !past(before)))
    write_token(a, r, b, index_in(rank), logit_of(key_in(rank)), all);
}

template <typename T>
__global__ __launch_bounds__(kFinishThreads) void sample_finish_kernel(SampleArgs a) {
  __shared__ Shared sh;
  __shared__ Few few;
  __shared__ u64 chunk_sums[kMaxChunks];
  const int b = blockIdx.x, tid = threadIdx.x;
  const Settings set = load_settings(a, b);
  const HistShare hist = load_hist(a, b);
  const u64 sum = tid < a.chunks ? a.sums[static_cast<int64_t>(b) * a.chunks + tid] : 0;
  u64 mine[kList / kFinishThreads];  // tokens of the list: how many count is known later
  const u64* list = a.list + static_cast<int64_t>(b) * kList;
#pragma unroll
  for (int j = 0; j < kList / kFinishThreads; ++j)
    mine[j] = a.counts != nullptr ? list[tid + j * kFinishThreads] : 0;
  __shared__ double roots[kRoots];
  fill_roots(roots);
  const u64 best = row_best<kFinishThreads>(a, b, sh.sums);
  const Row r = row_with<T>(a, b, set, best, roots);
  if (r.greedy) {
    if (tid == 0) write_greedy(a, b, best);
    return;
  }
  u64 least = 0;
  if (r.limited) {
    const Bins bins = bins_of(hist, r);
    if (bins.in <= kList) {
#pragma unroll
      for (int j = 0; j < kList / kFinishThreads; ++j)
        if (tid + j * kFinishThreads >= bins.in) mine[j] = 0;  // (no token's rank is 0)
      u64 weight[kList / kFinishThreads];
#pragma unroll
      for (int j = 0; j < kList / kFinishThreads; ++j)
        weight[j] = j * kFinishThreads < bins.in && mine[j] != 0 ? weight_of(r, logit_of(key_in(mine[j]))) : 0;
      const auto each = [&](auto f) {
#pragma unroll
        for (int j = 0; j < kList / kFinishThreads; ++j)
          if (mine[j] != 0) f(mine[j], [&] { return weight[j]; });
      };
      const bool is_few = bins.in <= kFew;
      const Place place(static_cast<int>(bins.in));
      least = is_few ? border_of_few(r, mine[0], weight[0], bins, place, few, sh)
                     : border_of<kFinishThreads>(r, each, bins.above, bins.above_weight, bins.all, sh);
      if (is_few && bins.lo == 0) {
        pick_of_few(a, r, b, least, place, few, sh);
        return;
      }
      __syncthreads();
      if (tid < a.chunks) chunk_sums[tid] = sum;
      __syncthreads();
      each([&](u64 rank, auto of) {
        const u64 w = of();
        if (rank >= least && w >= r.least) atomicAdd(&chunk_sums[index_in(rank) / a.chunk], w);
      });
    } else {  // more tokens than a list holds: by the row itself
      least = border_of<kFinishThreads>(r, [&](auto f) {
        for_each<T, kFinishThreads>(r.logits, 0, a.vocab, [&](int i, float x) {
        f(rank_of(key_of(x), i), [&] { return weight_of(r, x); });
      });
      }, 0, 0, bins.all, sh);
      for (int c = 0; c < a.chunks; ++c) {
        u64 sum = 0;
        for_each<T, kFinishThreads>(r.logits, c * a.chunk, min(a.vocab, (c + 1) * a.chunk), [&](int i, float x) {
          if (rank_of(key_of(x), i) >= least) sum += likely_weight(r, x);
        });
        sum = across<kFinishThreads, false>(sum, sh.sums);
        if (tid == 0) chunk_sums[c] = sum;
      }
    }
  } else if (tid < a.chunks) {
    chunk_sums[tid] = sum;
  }
  pick_in_chunks<T>(a, r, b, least, chunk_sums, sh);
}

// Chunks of a row in a call (0: a workgroup has a whole row).
constexpr int kShortRow = 4096;
constexpr int kLeastChunk = 2048;
int chunks_of(int64_t batch, int64_t vocab) {
  if (vocab <= kShortRow) return 0;
  const int64_t least = (vocab + kMostChunk - 1) / kMostChunk;
  const int64_t most = (vocab + kLeastChunk - 1) / kLeastChunk;
  const int64_t want = 8LL * cu_count() / batch;
  return static_cast<int>(want < least ? least : want > most ? most : want);
}
static_assert(kShortRow <= kRowThreads * kEach, "a row's workgroup has kEach tokens a thread");
static_assert(FPV2_MAX_VOCAB <= kMaxChunks * kLeastChunk, "chunks of the longest row");

int64_t align16(int64_t n) { return (n + 15) / 16 * 16; }

// (a greedy call is the first and the last pass: 5.3 us for a row of 151936)
bool all_greedy(const fpv2_sample_params& p) { return p.temperatures == nullptr && !(p.temperature > 0); }
// Workspace: best, sums, and with a limit weights, list, counts, listed.
bool may_limit(const fpv2_sample_params& p) {
  if (all_greedy(p)) return false;
  return p.top_ks != nullptr || p.top_ps != nullptr || (p.top_k > 0 && p.top_k < p.vocab) || p.top_p < 1;
}
int64_t workspace_of(const fpv2_sample_params& p, SampleArgs* a, char* base) {
  const int64_t chunks = chunks_of(p.batch, p.vocab);
  if (chunks == 0) return 0;
  int64_t at = 0;
  const auto take = [&](int64_t bytes) {
    const int64_t here = at;
    at += align16(bytes);
    return base + here;
  };
  a->chunks = static_cast<int>(chunks);
  a->chunk = static_cast<int>((p.vocab + chunks - 1) / chunks);
  // (a workgroup's start costs the passes as much as half a chunk: four waves a SIMD)
  const int64_t group = p.batch * chunks / (4 * cu_count());
  a->group = static_cast<int>(group < 1 ? 1 : group > chunks ? chunks : group);
  a->best = reinterpret_cast<u64*>(take(8 * p.batch * chunks));
  a->sums = reinterpret_cast<u64*>(take(8 * p.batch * chunks));
  if (may_limit(p)) {
    a->weights = reinterpret_cast<u64*>(take(8 * p.batch * kBins));
    a->list = reinterpret_cast<u64*>(take(8 * p.batch * kList));
    a->counts = reinterpret_cast<uint32_t*>(take(4 * p.batch * kBins));
    a->listed = reinterpret_cast<uint32_t*>(take(4 * p.batch));
  }
  return at;
}

template <typename T>
int launch_sample(const SampleArgs& a, int64_t batch, bool greedy, hipStream_t s) {
  const dim3 rows(static_cast<unsigned>(batch)), row_threads(kRowThreads), threads(kChunkThreads);
  if (a.chunks == 0) {
    hipLaunchKernelGGL(sample_row_kernel<T>, rows, row_threads, 0, s, a);
    return check_launch("sample_row_kernel");
  }
  const dim3 chunks(static_cast<unsigned>(a.chunks), static_cast<unsigned>(batch));
  hipLaunchKernelGGL(chunk_max_kernel<T>, chunks, threads, 0, s, a);
  const dim3 groups(static_cast<unsigned>(batch), static_cast<unsigned>((a.chunks + a.group - 1) / a.group));
  if (!greedy) hipLaunchKernelGGL(chunk_weigh_kernel<T>, groups, threads, 0, s, a);
  if (a.counts != nullptr) hipLaunchKernelGGL(chunk_list_kernel<T>, groups, threads, 0, s, a);
  hipLaunchKernelGGL(sample_finish_kernel<T>, rows, dim3(kFinishThreads), 0, s, a);
  return check_launch("sample_finish_kernel");
}

int check_sample(const char* name, const fpv2_sample_params* p) {
  if (p == nullptr) return fail(FPV2_ERR_ARGUMENT, "%s: null params", name);
  if (p->batch < 0 || p->batch > 0xffff || p->vocab <= 0 || p->logits_stride < 0)
    return fail(FPV2_ERR_ARGUMENT, "%s: bad batch (at most 65535), vocab or stride", name);
  if (p->vocab > FPV2_MAX_VOCAB)
    return fail(FPV2_ERR_UNSUPPORTED, "%s: more than %d tokens", name, FPV2_MAX_VOCAB);
  return FPV2_OK;
}

}  // namespace
}  // namespace fpv2

extern "C" int64_t fpv2_sample_tokens_workspace_bytes(const fpv2_sample_params* params) {
  using namespace fpv2;
  if (const int rc = check_sample("fpv2_sample_tokens", params)) return rc;
  SampleArgs a{};
  return params->batch == 0 ? 0 : workspace_of(*params, &a, nullptr);
}

extern "C" int fpv2_sample_tokens(const void* logits, const float* uniforms, int dtype,
                                  const fpv2_sample_params* params, int64_t* tokens,
                                  float* logprobs, void* workspace, int64_t workspace_bytes,
                                  void* stream) {
  using namespace fpv2;
  const char* name = "fpv2_sample_tokens";
  if (const int rc = check_sample(name, params)) return rc;
  const fpv2_sample_params& p = *params;
  if (dtype != FPV2_F32 && dtype != FPV2_BF16 && dtype != FPV2_F16)
    return fail(FPV2_ERR_UNSUPPORTED, "%s: dtype must be float32, bf16 or f16", name);
  if (p.batch == 0) return FPV2_OK;
  if (!logits || !uniforms || !tokens) return fail(FPV2_ERR_ARGUMENT, "%s: null pointer", name);
  SampleArgs a{};
  const int64_t need = workspace_of(p, &a, static_cast<char*>(workspace));
  if (need > 0 && (workspace == nullptr || workspace_bytes < need ||
                   (reinterpret_cast<uintptr_t>(workspace) & 15u) != 0))
    return fail(FPV2_ERR_ARGUMENT, "%s: needs a 16-byte aligned workspace of %lld bytes", name,
                static_cast<long long>(need));
  a.logits = logits;
  a.uniforms = uniforms;
  a.temperatures = p.temperatures;
  a.top_ks = p.top_ks;
  a.top_ps = p.top_ps;
  a.min_ps = p.min_ps;
  a.tokens = tokens;
  a.logprobs = logprobs;
  a.temperature = p.temperature;
  a.top_p = p.top_p;
  a.min_p = p.min_p;
  a.top_k = p.top_k;
  a.stride = p.logits_stride;
  a.vocab = static_cast<int>(p.vocab);
  const hipStream_t s = static_cast<hipStream_t>(stream);
  if (dtype == FPV2_F32) return launch_sample<f32_t>(a, p.batch, all_greedy(p), s);
  if (dtype == FPV2_BF16) return launch_sample<bf16_t>(a, p.batch, all_greedy(p), s);
  return launch_sample<f16_t>(a, p.batch, all_greedy(p), s);
}
