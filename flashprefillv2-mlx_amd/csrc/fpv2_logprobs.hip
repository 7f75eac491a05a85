// Log probabilities of given tokens, entropies and the most likely alternatives.
//
// With e_i = x_i log2(e) - R for any reference R, p_i = 2^e_i / s, s = sum 2^e_i:
//   log p_i = (e_i - log2 s) ln 2,  -sum p log p = (log2 s - t / s) ln 2,  t = sum 2^e_i e_i
// so one pass over the logits is enough: each thread holds (R, s, t) of what it has
// seen, R the greatest x log2(e), and moves to a greater reference R' by
//   t' = f (t + (R - R') s), s' = f s, f = 2^(R - R').
// e is one fused multiply-add, so neither large logits nor R's own rounding cost bits.
//
// The alternatives: a logit and its token are one 64-bit key, whose order is theirs.  A
// wave collects the keys above a floor in 64 slots and, when these are full, sorts them
// and keeps the first.  The floor of its first logits is the greatest number that enough
// lanes' maxima reach, so that few more than the wanted ones are collected at all.
// Bound by reading the logits: 1536 bfloat16 rows of 151936 84 us, 5.5 TB/s; few rows by two launches
// and their chains: one float32 row of 151936 with 20 alternatives 8.8 + 5.4 us (34.7 + 21 with the
// keys collected from none on), 160 float16 rows of 50001 with 5 15.0 + 5.7.
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
  f32x4* parts;     // [rows][chunks] {R, s, t, -}
  uint64_t* lists;  // [rows][chunks][top] keys
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

// Keys: greater logits first, equal ones (0 and -0 too) by token; 0: none.
__device__ __forceinline__ uint32_t ordered(float x) {
  const uint32_t b = __float_as_uint(x + 0.f);
  return b ^ (static_cast<int32_t>(b) < 0 ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float logit_of(uint64_t key) {
  const uint32_t s = static_cast<uint32_t>(key >> 32);
  return __uint_as_float(s ^ (s & 0x80000000u ? 0x80000000u : 0xffffffffu));
}
__device__ __forceinline__ int token_of(uint64_t key) { return static_cast<int>(~static_cast<uint32_t>(key)); }
__device__ __forceinline__ uint64_t key_of(float x, uint32_t token) {
  return x > neg_inf() ? static_cast<uint64_t>(ordered(x)) << 32 | static_cast<uint32_t>(~token) : 0;
}

// The wave's keys from the greatest on, one a lane.  HALVES: where the first 32 fall and
// the rest rise, the last steps alone.
template <bool HALVES>
__device__ __forceinline__ uint64_t sorted(uint64_t key, int lane) {
#pragma unroll
  for (int size = HALVES ? 64 : 2; size <= 64; size *= 2)
#pragma unroll
    for (int step = size / 2; step >= 1; step /= 2) {
      const uint64_t other = __shfl_xor(key, step, 64);
      const bool first = (lane & step) == 0, falling = (lane & size) == 0 || size == 64;
      key = (key > other) == (first == falling) ? key : other;
    }
  return key;
}

// A wave's greatest keys.
struct Best {
  uint64_t* slots;  // 64 of the wave's LDS
  int top, count;
  uint64_t floor;   // keys above it enter
  float floor_x;    // which are of this logit or greater ones
  __device__ __forceinline__ void start(uint64_t* lds, int wanted) {
    slots = lds;
    top = wanted;
    count = 0;
    floor = 0;
    floor_x = neg_inf();
  }
  __device__ __forceinline__ void raise(uint64_t to) {
    floor = to;
    floor_x = logit_of(to + 1);  // (to is of the same logit, or just below all keys of the next)
  }
  // The floor under a wave's first keys, from each lane's greatest (its high word, 0: none).
  __device__ __forceinline__ void first_floor(uint32_t most) {
    uint32_t at = 0;
#pragma unroll
    for (int bit = 31; bit >= 8; --bit) {
      const uint32_t to = at | 1u << bit;
      if (__popcll(__ballot(most >= to)) >= top) at = to;
    }
    if (at != 0) raise((static_cast<uint64_t>(at) << 32) - 1);
  }
  // All slots in order, the first ones kept; returns the lane's.
  __device__ __forceinline__ uint64_t settle(int lane) {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    uint64_t key = sorted<false>(lane < count ? slots[lane] : 0, lane);
    key = lane < top ? key : 0;
    slots[lane] = key;
    count = __popcll(__ballot(key != 0));
    if (count == top) {
      const uint32_t high = __builtin_amdgcn_readlane(static_cast<uint32_t>(key >> 32), top - 1);
      const uint32_t low = __builtin_amdgcn_readlane(static_cast<uint32_t>(key), top - 1);
      floor = static_cast<uint64_t>(high) << 32 | low;
      floor_x = logit_of(floor);
    }
    return key;
  }
  __device__ __forceinline__ void add(uint64_t key, int lane) {
    uint64_t mask = __ballot(key > floor);
    while (mask != 0) {
      const int room = 64 - count;
      const int before = __builtin_amdgcn_mbcnt_hi(mask >> 32, __builtin_amdgcn_mbcnt_lo(mask, 0));
      const bool mine = mask >> lane & 1;
      if (mine && before < room) slots[count + before] = key;
      const int n = __popcll(mask);
      if (n <= room) {
        count += n;
        return;
      }
      count = 64;
      settle(lane);
      mask = __ballot(mine && before >= room && key > floor);
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

// The greatest keys of a workgroup's waves, in the first one's lanes.
__device__ __forceinline__ uint64_t join_best(Best& best, uint64_t (*sh)[64], int tid) {
  const int lane = tid & 63, wave = tid >> 6;
  uint64_t key = best.settle(lane);
#pragma unroll
  for (int with = 1; with <= 2; with *= 2) {
    __syncthreads();
    if (wave % (2 * with) == 0) {
      // (32 keys of each at most, the other's from its last on)
      key = lane < 32 ? key : sh[wave + with][63 - lane];
      key = sorted<true>(key, lane);
      key = lane < best.top ? key : 0;
      sh[wave][lane] = key;
    }
  }
  return key;
}

// (rounding could leave a sure token 2^-24 above 0)
__device__ __forceinline__ float log_share(float x, float r, float norm) {
  return fminf((__builtin_fmaf(x, kLog2e, -r) - norm) * kLn2, 0.f);
}

template <typename T>
__device__ __forceinline__ void write_row(const LogArgs& a, int row, Sums s, uint64_t key, int tid) {
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
    a.top_tokens[static_cast<int64_t>(row) * a.top + tid] = key != 0 ? token_of(key) : -1;
    a.top_logprobs[static_cast<int64_t>(row) * a.top + tid] =
        key != 0 ? log_share(clamped(logit_of(key)), s.r, norm) : neg_inf();
  }
}

// One workgroup a chunk of a row.
template <typename T, bool TOP>
__global__ __launch_bounds__(256) void logprobs_kernel(LogArgs a) {
  typedef typename Logit<T>::raw raw;
  constexpr int kPer = Logit<T>::kPer, kEach = kVecs * kPer;
  __shared__ Sums sh_s[4];
  __shared__ uint64_t sh_l[TOP ? 4 : 1][64];
  const int tid = threadIdx.x, lane = tid & 63;
  const int row = blockIdx.x / a.chunks, chunk = blockIdx.x - row * a.chunks;
  const raw* const p = static_cast<const raw*>(a.logits) + row * a.stride;
  // the row in 16-byte vectors of memory; its first and last ones may be partly others'
  const int skew = static_cast<int>((reinterpret_cast<uintptr_t>(p) & 15u) / sizeof(raw));
  const int vecs = (skew + a.vocab + kPer - 1) / kPer;
  const int first = static_cast<int>(static_cast<int64_t>(vecs) * chunk / a.chunks);
  const int last = static_cast<int>(static_cast<int64_t>(vecs) * (chunk + 1) / a.chunks);
  Sums s = {neg_inf(), 0.f, 0.f};
  Best best;
  if constexpr (TOP) best.start(sh_l[tid >> 6], a.top);
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
      if (v0 == first) best.first_floor(most > neg_inf() ? ordered(most) : 0);
      if (__any(most >= best.floor_x)) {
#pragma unroll
        for (int j = 0; j < kEach; ++j)
          if (__any(x[j] >= best.floor_x))
            best.add(key_of(x[j], (v0 + 256 * (j / kPer) + tid) * kPer - skew + j % kPer), lane);
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
  uint64_t key = 0;
  if constexpr (TOP) key = join_best(best, sh_l, tid);
  if (a.chunks == 1) {
    write_row<T>(a, row, s, key, tid);
    return;
  }
  const int64_t at = static_cast<int64_t>(row) * a.chunks + chunk;
  if (tid == 0) a.parts[at] = f32x4{s.r, s.s, s.t, 0.f};
  if (TOP && tid < a.top) a.lists[at * a.top + tid] = key;
}

// Joins a row's chunks: one workgroup a row.
template <typename T, bool TOP>
__global__ __launch_bounds__(256) void logprobs_join_kernel(LogArgs a) {
  __shared__ Sums sh_s[4];
  __shared__ uint64_t sh_l[TOP ? 4 : 1][64];
  const int tid = threadIdx.x, lane = tid & 63, row = blockIdx.x;
  const int64_t base = static_cast<int64_t>(row) * a.chunks;
  uint64_t key = 0;
  if constexpr (TOP) {
    Best best;
    best.start(sh_l[tid >> 6], a.top);
    const int n = a.chunks * a.top;
    for (int i0 = 0; i0 < n; i0 += 256 * kVecs) {
      uint64_t keys[kVecs], most = 0;
#pragma unroll
      for (int i = 0; i < kVecs; ++i) {
        const int at = i0 + 256 * i + tid;
        keys[i] = at < n ? a.lists[base * a.top + at] : 0;
        most = keys[i] > most ? keys[i] : most;
      }
      if (i0 == 0) best.first_floor(static_cast<uint32_t>(most >> 32));
#pragma unroll
      for (int i = 0; i < kVecs; ++i) best.add(keys[i], lane);
    }
    key = join_best(best, sh_l, tid);
  }
  Sums s = {neg_inf(), 0.f, 0.f};
  for (int i = tid; i < a.chunks; i += 256) {
    const f32x4 part = a.parts[base + i];
    s = join(s, Sums{part[0], part[1], part[2]});
  }
  s = join_all(s, sh_s, tid);
  write_row<T>(a, row, s, key, tid);
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
  a.lists = reinterpret_cast<uint64_t*>(a.parts + p.rows * a.chunks);
  const hipStream_t s = static_cast<hipStream_t>(stream);
  return dtype == FPV2_F32    ? launch_top<float>(a, s)
         : dtype == FPV2_BF16 ? launch_top<bf16_t>(a, s)
                              : launch_top<f16_t>(a, s);
}
