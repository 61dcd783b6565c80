// Next-token sampling and top logits over rows of fp16 logits.
//
// The reference draws its tokens on the host from the logits that generate_torch.next_token_logits
// returns (Midstream-LLM src/jishui/generate_torch.py:278-345); here the draw stays on the device, from
// uniform numbers that the caller supplies, so a generation loop never waits for a copy of the logits.
//
// fp16 values are compared through 16-bit keys in their order (order_key): -0 and +0 share one, a NaN
// sorts below everything. Rank means: larger value first, among equal values the lower index first.
// A filter of the sampler (top-k, top-p, min-p) keeps a prefix of the ranking, so the three together keep
// every value above one threshold key and the first few (by index) of the values at it.
#include <cuda_fp16.h>

#include <algorithm>
#include <atomic>

#include "jx_common.cuh"
#include "jx_host.h"

namespace jx {
namespace sel {

typedef unsigned long long u64;

constexpr uint32_t kKeyNegInf = 0x03ffu;  // key of -inf; NaN has key 0

__device__ __forceinline__ uint32_t order_key(uint32_t h) {
  if ((h & 0x7fffu) > 0x7c00u) return 0u;
  if (h == 0x8000u) h = 0u;
  return (h & 0x8000u) ? (~h & 0xffffu) : (h | 0x8000u);
}

// The same of anything but a NaN.
__device__ __forceinline__ uint32_t order_key_num(uint32_t h) {
  h = h == 0x8000u ? 0u : h;
  return (h ^ ((uint32_t)((int)(h << 16) >> 31) | 0x8000u)) & 0xffffu;
}

__device__ __forceinline__ uint32_t key_bits(uint32_t key) { return (key & 0x8000u) ? key ^ 0x8000u : ~key & 0xffffu; }

__device__ __forceinline__ __half key_half(uint32_t key) { return __ushort_as_half((unsigned short)key_bits(key)); }

// Eight consecutive logits; elements at and past `vocab` read as `fill` (twice the same half: a NaN, which no
// comparison selects, or -inf). A row starts on a 16-byte boundary; only whole vectors are read as one.
constexpr uint32_t kFillNan = 0xffffu, kFillNegInf = 0xfc00u;

struct Vec {
  uint32_t w[4];
  __device__ __forceinline__ uint32_t bits(int j) const { return (w[j >> 1] >> ((j & 1) * 16)) & 0xffffu; }
};

template <uint32_t kFill>
__device__ __noinline__ Vec load_part(const __half* row, int64_t first, int vocab) {
  const unsigned short* p = reinterpret_cast<const unsigned short*>(row);
  Vec v;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint32_t lo = first + 2 * j < vocab ? p[first + 2 * j] : kFill;
    const uint32_t hi = first + 2 * j + 1 < vocab ? p[first + 2 * j + 1] : kFill;
    v.w[j] = lo | (hi << 16);
  }
  return v;
}

template <uint32_t kFill>
__device__ __forceinline__ Vec load_vec(const __half* row, int i, int vocab) {  // vector i
  Vec v;
  v.w[0] = v.w[1] = v.w[2] = v.w[3] = kFill * 0x10001u;
  if (i < vocab >> 3) {
    const uint4 u = __ldg(reinterpret_cast<const uint4*>(row) + i);
    v.w[0] = u.x, v.w[1] = u.y, v.w[2] = u.z, v.w[3] = u.w;
  } else if (i * 8 < vocab) {
    v = load_part<kFill>(row, 8 * i, vocab);
  }
  return v;
}

__device__ __forceinline__ __half2 as_half2(uint32_t w) { return *reinterpret_cast<__half2*>(&w); }

// Largest of the vector's values (NaN only if all are).
__device__ __forceinline__ __half2 vec_max2(const Vec& v) {
  return __hmax2(__hmax2(as_half2(v.w[0]), as_half2(v.w[1])), __hmax2(as_half2(v.w[2]), as_half2(v.w[3])));
}

__device__ __forceinline__ __half max_of(__half2 m) { return __hmax(__low2half(m), __high2half(m)); }

// Bit j set where element j >= limit (never for a NaN).
__device__ __forceinline__ uint32_t vec_ge(const Vec& v, __half2 limit) {
  uint32_t m = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) m |= __hge2_mask(as_half2(v.w[j]), limit) & (0x10001u << j);
  // bits 0..3: elements 0, 2, 4, 6; bits 16..19: elements 1, 3, 5, 7
  return m;
}
__device__ __forceinline__ uint32_t ge_bit(int j) { return (j & 1) ? 0x10000u << (j >> 1) : 1u << (j >> 1); }

// ---------------------------------------------------------------------------------------------------------
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Block helpers. Every thread of the block calls them.
// ---------------------------------------------------------------------------------------------------------
template <int NT>
__device__ __forceinline__ uint32_t block_max(uint32_t v, uint32_t* red) {
  v = __reduce_max_sync(0xffffffffu, v);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  v = (threadIdx.x & 31) < NT / 32 ? red[threadIdx.x & 31] : 0u;
  v = __reduce_max_sync(0xffffffffu, v);
  __syncthreads();
  return v;
}

__device__ __forceinline__ u64 warp_sum64(u64 v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

__device__ __forceinline__ double warp_sum_d(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Inclusive prefix sums over the lanes of a warp.
template <typename T>
__device__ __forceinline__ T warp_scan(T v) {
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const T n = __shfl_up_sync(0xffffffffu, v, o);
    if ((threadIdx.x & 31) >= o) v += n;
  }
  return v;
}

// Exclusive prefix sum of one value a thread over the block; *total gets the sum.
template <int NT, typename T>
__device__ __forceinline__ T block_scan(T v, T* red, T* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const T inc = warp_scan(v);
  if (lane == 31) red[warp] = inc;
  __syncthreads();
  const T w = lane < NT / 32 ? red[lane] : T(0);
  const T winc = warp_scan(w);
  *total = __shfl_sync(0xffffffffu, winc, NT / 32 - 1);
  const T before = __shfl_sync(0xffffffffu, winc - w, warp);
  __syncthreads();
  return before + inc - v;
}

// ---------------------------------------------------------------------------------------------------------
// Top logits: the k largest of a row in rank order.
//
// One block per row with the row in registers (rows longer than NT * 8 * VPT elements are read again for the
// later passes). The k-th largest of the threads' maxima is a limit that at least k elements pass, and in general few
// more: a histogram of the maxima, in bins of 16 keys down from the largest, gives it to within a bin. Where k is large
// against the threads the maxima of the 8-element vectors take their place. The few vectors that
// hold such elements go to shared memory, their elements above the limit are collected, ranked among themselves by
// counting and written. A row where too many pass (many equal values) or k is large against the vectors takes
// the exact way: two histograms of all keys find the threshold, values at it are taken in index order.
// 16384 rows of 32000, top 64: 235 us, 4.5 TB/s; what follows the loads costs with k (4096 rows, top 16 51.7 us, 64 63.6,
// 256 143), since the ranking's compares grow with its square.
// ---------------------------------------------------------------------------------------------------------
constexpr int kBins = 2048;     // upper 11 bits of a key
constexpr int kCand = 2048;     // candidates a block can hold
constexpr int kMaxTop = 1024;

// With hist[bin] counting keys, finds the bin (from the top) in which the k-th key falls and how many keys lie
// in higher bins; found[0] = -1 if there are fewer than k keys in all.
template <int NT, int kBins = sel::kBins>
__device__ __forceinline__ void find_bin(const uint32_t* hist, uint32_t k, uint32_t* red, int* found) {
  constexpr int PER = kBins / NT;
  uint32_t c[PER], sum = 0;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    c[i] = hist[kBins - 1 - (threadIdx.x * PER + i)];
    sum += c[i];
  }
  if (threadIdx.x == 0) found[0] = -1;
  uint32_t total;
  uint32_t above = block_scan<NT>(sum, red, &total);
  if (above < k && above + sum >= k) {
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      if (above < k && above + c[i] >= k) {
        found[0] = kBins - 1 - (threadIdx.x * PER + i);
        found[1] = (int)above;
      }
      above += c[i];
    }
  }
  __syncthreads();
}

// A candidate: key and complemented index, so that larger means earlier in rank. 32 bits where the index fits 16.
template <typename C>
struct CandidateOf {
  static constexpr int kShift = sizeof(C) * 4;
  static constexpr C kMask = (C(1) << kShift) - 1;
  static __device__ __forceinline__ C make(uint32_t key, uint32_t index) { return (C)key << kShift | (kMask - (C)index); }
  static __device__ __forceinline__ uint32_t key(C c) { return (uint32_t)(c >> kShift); }
  static __device__ __forceinline__ uint32_t index(C c) { return (uint32_t)(kMask - (c & kMask)); }
};

// The exact way: k candidates in any order. Rare, so plain.
template <int NT, typename C>
__device__ __noinline__ void exact_candidates(const unsigned short* row, int vocab, uint32_t k, uint32_t* hist, uint32_t* red,
                                              int* found, C* cand, uint32_t* ncand) {
  const int tid = threadIdx.x;
  __syncthreads();
  for (int i = tid; i < kBins; i += NT) hist[i] = 0;
  if (tid == 0) *ncand = 0;
  __syncthreads();
  for (int i = tid; i < vocab; i += NT) atomicAdd(&hist[order_key(row[i]) >> 5], 1u);
  __syncthreads();
  find_bin<NT>(hist, k, red, found);
  const uint32_t bin = (uint32_t)found[0];
  uint32_t left = k - (uint32_t)found[1];
  __syncthreads();
  for (int i = tid; i < kBins; i += NT) hist[i] = 0;
  __syncthreads();
  for (int i = tid; i < vocab; i += NT) {
    const uint32_t key = order_key(row[i]);
    if (key >> 5 == bin) atomicAdd(&hist[key & 31u], 1u);
  }
  __syncthreads();
  uint32_t sub = 31;
  while (hist[sub] < left) left -= hist[sub--];
  const uint32_t tau = (bin << 5) | sub;
  uint32_t taken = 0;
  for (int base = 0; base < vocab; base += NT) {
    const int i = base + tid;
    const uint32_t key = i < vocab ? order_key(row[i]) : 0u;
    const uint32_t tie = i < vocab && key == tau ? 1u : 0u;
    uint32_t total = 0, before = 0;
    if (taken < left) before = taken + block_scan<NT>(tie, red, &total);
    if (i < vocab && (key > tau || (tie && taken < left && before < left)))
      cand[atomicAdd(ncand, 1u)] = CandidateOf<C>::make(key, (uint32_t)i);
    taken += total;
  }
  __syncthreads();
}

template <int NT, typename C, bool kLarge>
struct TopShared {
  static constexpr int kOwn = kLarge ? 128 : 32;  // vectors with candidates that a warp can hold
  union {
    struct {
      uint4 v[NT / 32 * kOwn];
      int index[NT / 32 * kOwn];
    } vec;
    uint32_t hist[kBins];
  };
  __align__(16) C cand[kCand];
  uint32_t red[32];
  int found[2];
  uint32_t ncand;
};

template <int NT, int VPT, typename C, bool kLarge>
__global__ void __launch_bounds__(NT, 1024 / NT)
    top_logits_kernel(const __half* __restrict__ logits, int64_t ld, int vocab, int k, __half* __restrict__ values,
                      int64_t* __restrict__ ids) {
  typedef CandidateOf<C> Cand;
  constexpr int kOwn = TopShared<NT, C, kLarge>::kOwn;
  extern __shared__ __align__(16) uint8_t smem_raw[];
  TopShared<NT, C, kLarge>& s = *reinterpret_cast<TopShared<NT, C, kLarge>*>(smem_raw);
  C* cand = s.cand;
  uint32_t* red = s.red;
  int* found = s.found;
  uint32_t& ncand = s.ncand;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const __half* row = logits + (int64_t)blockIdx.x * ld;
  const int nvec = (vocab + 7) / 8;
  const int nchunk = (nvec + NT * VPT - 1) / (NT * VPT);

  Vec v[VPT];
  __half2 tmax = __half2half2(__ushort_as_half(0xffffu));
  auto load = [&](int c) {
#pragma unroll
    for (int i = 0; i < VPT; ++i) v[i] = load_vec<kFillNan>(row, (c * VPT + i) * NT + tid, vocab);
  };
  for (int c = 0; c < nchunk; ++c) {
    load(c);
#pragma unroll
    for (int i = 0; i < VPT; ++i) tmax = __hmax2(tmax, vec_max2(v[i]));
  }
  // The limit.
  constexpr int kTopBins = 1024;
  const bool by_vector = kLarge && k <= nvec / 2;
  for (int i = tid; i < (by_vector ? kBins : kTopBins); i += NT) s.hist[i] = 0;
  if (tid == 0) ncand = 0;
  const uint32_t tkey = order_key(__half_as_ushort(max_of(tmax)));
  const uint32_t mkey = block_max<NT>(tkey, red);
  uint32_t lkey = 0;
  if (by_vector) {
    for (int c = 0; c < nchunk; ++c) {
      if (nchunk > 1) load(c);
#pragma unroll
      for (int i = 0; i < VPT; ++i)
        if ((c * VPT + i) * NT + tid < nvec) atomicAdd(&s.hist[order_key(__half_as_ushort(max_of(vec_max2(v[i])))) >> 5], 1u);
    }
    __syncthreads();
    find_bin<NT>(s.hist, (uint32_t)k, red, found);
    if (found[0] > 0) lkey = (uint32_t)found[0] << 5;
  } else if (k <= min(nvec, NT)) {
    const uint32_t d = (mkey - tkey) >> 4;
    if (tkey && d < kTopBins) atomicAdd(&s.hist[kTopBins - 1 - d], 1u);
    __syncthreads();
    find_bin<NT, kTopBins>(s.hist, (uint32_t)k, red, found);
    if (found[0] >= 0) {
      const uint32_t down = (uint32_t)(kTopBins - found[0]) * 16 - 1;  // to the bin's lowest key
      lkey = mkey > down ? mkey - down : 0u;
    }
  }
  // Without a limit every element of a short row is a candidate (NaN too).
  const bool all = lkey <= kKeyNegInf;
  const __half limit = key_half(max(lkey, kKeyNegInf));
  uint32_t n = kCand + 1;
  if (!all || nvec * 8 <= kCand) {
    // Each warp gathers its vectors and looks through them by itself.
    const uint32_t below = (1u << lane) - 1u;
    uint32_t nv = 0;
    for (int c = 0; c < nchunk; ++c) {
      if (nchunk > 1) load(c);
#pragma unroll
      for (int i = 0; i < VPT; ++i) {
        const int at = (c * VPT + i) * NT + tid;
        const bool hit = all ? at < nvec : __hge(max_of(vec_max2(v[i])), limit);
        const uint32_t hits = __ballot_sync(0xffffffffu, hit);
        if (hits) {
          const uint32_t p = nv + __popc(hits & below);
          if (hit && p < kOwn) {
            s.vec.v[warp * kOwn + p] = make_uint4(v[i].w[0], v[i].w[1], v[i].w[2], v[i].w[3]);
            s.vec.index[warp * kOwn + p] = at;
          }
          nv += __popc(hits);
        }
      }
    }
    __syncwarp();
    if (nv > kOwn) {
      if (lane == 0) atomicAdd(&ncand, kCand + 1u);  // too many: the exact way
    } else {
      const unsigned short* h = reinterpret_cast<const unsigned short*>(&s.vec.v[warp * kOwn]);
#pragma unroll 1
      for (uint32_t e = lane; e < (nv * 8 + 31 & ~31u); e += 32) {
        uint32_t key = 0, index = 0xffffffffu;
        if (e < nv * 8) {
          key = order_key(h[e]);
          index = (uint32_t)s.vec.index[warp * kOwn + (e >> 3)] * 8 + (e & 7);
        }
        const bool in = (all || key >= lkey) && index < (uint32_t)vocab;
        const uint32_t ins = __ballot_sync(0xffffffffu, in);
        uint32_t p = 0;
        if (lane == 0 && ins) p = atomicAdd(&ncand, (uint32_t)__popc(ins));
        p = __shfl_sync(0xffffffffu, p, 0) + __popc(ins & below);
        if (in && p < kCand) cand[p] = Cand::make(key, index);
      }
    }
    __syncthreads();
    n = ncand;
  }
  if (n > kCand) {
    exact_candidates<NT, C>(reinterpret_cast<const unsigned short*>(row), vocab, (uint32_t)k, s.hist, red, found, cand, &ncand);
    n = (uint32_t)k;
  }
  __half* vout = values + (int64_t)blockIdx.x * k;
  int64_t* iout = ids + (int64_t)blockIdx.x * k;
  auto write = [&](uint32_t rank, C c) {
    vout[rank] = key_half(Cand::key(c));
    iout[rank] = (int64_t)Cand::index(c);
  };
  // Padded with zeros (which no candidate is), to the vectors of the count or the power of two of the sort.
  constexpr uint32_t kCount = 1024;
  uint32_t size = (n + 3) & ~3u;
  if (n > kCount)
    for (size = 2 * kCount; size < n;) size <<= 1;
  if (n + tid < size) cand[n + tid] = 0;
  for (uint32_t i = n + tid + NT; i < size; i += NT) cand[i] = 0;
  __syncthreads();
  if (n <= kCount) {
    // The rank of each is the number of larger ones (no two are equal: the index is part of them).
#pragma unroll 1
    for (uint32_t i = tid; i < n; i += NT) {
      const C mine = cand[i];
      uint32_t rank = 0;
      constexpr int kPer = 16 / sizeof(C);
      for (uint32_t j = 0; j < size; j += kPer) {
        const uint4 u = *reinterpret_cast<const uint4*>(&cand[j]);
        const C* o = reinterpret_cast<const C*>(&u);
#pragma unroll
        for (int e = 0; e < kPer; ++e) rank += o[e] > mine;
      }
      if (rank < (uint32_t)k) write(rank, mine);
    }
  } else {
    // Bitonic sort, largest first.
    for (uint32_t len = 2; len <= size; len <<= 1) {
      for (uint32_t half = len >> 1; half > 0; half >>= 1) {
        for (uint32_t t = tid; t < size / 2; t += NT) {
          const uint32_t i = 2 * half * (t / half) + t % half, j = i + half;
          const bool down = (i & len) == 0;
          const C a = cand[i], b = cand[j];
          if ((a < b) == down) {
            cand[i] = b;
            cand[j] = a;
          }
        }
        __syncthreads();
      }
    }
    for (uint32_t i = tid; i < (uint32_t)k; i += NT) write(i, cand[i]);
  }
}

// ---------------------------------------------------------------------------------------------------------
// Sampling. With M the row's maximum and e_i = exp((x_i - M) / T): top-k keeps the first k of the ranking,
// top-p the fewest of those whose e reach top_p of their sum, min-p those with e_i >= min_p (= probability
// >= min_p times the largest); the token is the first index at which the running sum of the kept e, in index
// order, exceeds u times their whole sum.
//
// Which token comes out hangs on where running sums lie against u, so e has to be good to far more digits
// than fp32 holds (an error of 1e-8 in the sums draws another token for one row in a few thousand): the
// weights are 64-bit integers round(e * 2^42), from exponentials in double precision. Integer sums do not
// depend on their order, so results repeat bit for bit.
//
// One block per row, which reads it twice (from memory, then from the caches): for the maximum, and to copy what
// can matter, in index order, to lists in shared memory (one for each warp's stretch of the row), so that the
// exponentials run on full warps. Below a limit an element cannot be kept, or only its part of a sum counts:
//   - e < 2^-43: its weight rounds to 0;
//   - top-k: below a limit that a histogram of the threads' maxima gives, or of the maxima of the 8-element vectors
//     where k is large;
//   - top-p without top-k: e < (1 - top_p) / V, since all such elements together weigh less than what top-p
//     drops (the maximum alone weighs 1). That limit is low, so a higher one is tried first, which a part of the row
//     says leaves three quarters of 1 - top_p below; whether it does is seen from the sums, and if not, the
//     safe one is taken. What lies below the limit is summed from fp32 exponentials, which only moves the place of the
//     cut; where the cut is nearer to a border between two ranks than that sum's error (kTailError of it), it is
//     taken again with that sum in the weights' own units.
// Lists of up to 256 entries together are ranked by counting, and the cuts are running sums over the ranks. Else a histogram
// of the list's keys gives the threshold: counts alone where a bin is one key (its weight is the
// count times one exponential), else counts and weights, the latter in four 11-bit limbs, since shared memory adds 32
// bits at a time. Then the kept weights are summed per 256 list places, and the group where the running sum passes
// its target is walked by one warp. Lists that do not fit are replaced by the whole row. All of this runs
// once a row, mostly as cold code, so it is written in loops rather than unrolled.
constexpr int kGroups = 4096;    // groups of 256 elements of a whole row: vocabularies up to 2^20
constexpr int kShort = 8192;     // rows up to here get small blocks, whose lists always hold them
constexpr double kUnit = 4398046511104.0;  // 2^42: weights of a row of 2^20 elements sum to at most 2^62
constexpr int kExpTab = 256;
// Bound of the error of the weight below a limit, relative: ex2.approx 2^-22; its argument, up to 2^5 octaves under the
// maximum, rounded to fp32, 2^-20 ln 2; the rounded factor c, made up for at one place, at most 2^5 octaves from there, 2^-24
// 2^5 ln 2; three additions of fp32 numbers, 3 2^-24; all that follows is added in 64 bits: together below 2.4e-6.
// Further down than 2^5 octaves lies at most 2^20 2^-32 in all, good to 4e-6, which is below 2^-30 (4096 units).
constexpr double kTailError = 2.4e-6, kTailFar = 4300.0;
constexpr int kGuess = 8;        // limits tried, 2.5 octaves of weight apart

struct SampleParams {
  const __half* logits;
  int64_t ld;
  int vocab;
  const float* u;
  const float* temperature;  // per row, or NULL: the scalar
  const int* top_k;
  const float* top_p;
  const float* min_p;
  float temperature_s, top_p_s, min_p_s;
  int top_k_s;
  int64_t* tokens;
  float* logp;
};

// e * 2^42: 2^(j/256) from the table, the rest of the exponent by the Taylor series of 2^(r/256), |r| <= 1/2, to the
// third power (relative error below 2e-13). At the maximum the result is 2^42 exactly.
struct Exp {
  double m;        // the row's maximum
  double c;        // 256 log2(e) / T
  const double* tab;

  // kAny: also for values whose weight rounds to 0, down to -inf.
  template <bool kAny>
  __device__ __forceinline__ double value(uint32_t h) const {
    // A half's bits moved to a double's places are the value times 2^-1008, subnormals too.
    const double x = __hiloint2double((int)((h & 0x8000u) << 16 | (h & 0x7fffu) << 10), 0);
    double y = fma(x, 0x1p1008, -m) * c;  // 256 log2(e_i), exact difference
    if (kAny) y = fmax(y, -256.0 * 60.0);  // (2^-18 units, which round to 0)
    const double t = y + 0x1.8p52;  // rounds to an integer, which sits in the low word
    const int n = __double2loint(t);
    const double r = y - (t - 0x1.8p52);
    constexpr double b = 0.6931471805599453 / 256.0;
    const double p = fma(r, fma(r, fma(r, b * b * b / 6.0, b * b / 2.0), b), 1.0);
    const double w = tab[n & (kExpTab - 1)];
    return __hiloint2double(__double2hiint(w) + ((n >> 8) << 20), __double2loint(w)) * p;
  }
};

// round(v) of 0 <= v < 2^51 as an integer: one weight (at most 2^42), not a sum of them.
__device__ __forceinline__ u64 to_units(double v) {
  return (u64)__double_as_longlong(v + 0x1p52) & 0xfffffffffffffull;
}

template <int NT>
struct SampleShared {
  static constexpr int kList = NT == 128 ? kShort : 32768;  // list places, over all warps
  static constexpr int kFine = NT == 128 ? 4096 : 8192;     // bins of one key
  static constexpr int kCoarse = NT == 128 ? 1024 : 2048;   // bins of several
  static constexpr int kGroups = NT == 128 ? kShort / 256 : sel::kGroups;
  union {
    unsigned short list[kList];
    struct {
      u64 mass[kGroups];
      uint32_t ties[kGroups];
    } row;  // groups of the whole row, where there is no list
  };
  union {
    uint32_t fine[kFine];
    struct {
      uint32_t count[kCoarse];
      uint32_t limb[4][kCoarse];
    } coarse;
    struct {
      u64 mass[kList / 256];
      uint32_t ties[kList / 256];
    } group;
  };
  uint32_t listed[32];            // entries of each warp's list
  unsigned short upto[32][32];    // of those, how many stand before each 32nd part of the warp's stretch
  uint32_t sub[64];
  double tab[kExpTab];
  u64 red64[32];
  uint32_t red[32];
  float redf[32][kGuess + 1];
  uint32_t key, left, bin, again;
  u64 before;
};
static_assert(2 * (sizeof(SampleShared<512>) + 1024) <= 233472, "two blocks an SM");
static_assert(5 * (sizeof(SampleShared<128>) + 1024) <= 233472, "five blocks an SM");

// Weight of a logit in units of 2^-42, as an integer.
struct Weights {
  Exp ex;
  uint32_t mkey;
  __device__ __forceinline__ u64 of(uint32_t bits) const { return to_units(ex.value<false>(bits)); }  // not below the least lkey
};

// The same as a call, for any key: an infinite maximum leaves every finite logit without weight.
__device__ __noinline__ u64 weight_of_key(const Weights& w, uint32_t key) {
  return key == w.mkey ? (u64)kUnit : w.mkey == 0xfc00u ? 0ull : to_units(w.ex.value<true>(key_bits(key)));
}

// The first place whose running weight exceeds this has the token.
__device__ __forceinline__ u64 draw_at(float u, u64 total) {
  const double ut = (double)u * (double)total;
  const u64 target = ut > 0.0 ? (u64)ut : 0ull;
  return target >= total ? total - 1 : target;
}

// What weighs below `lkey` in the row, exactly. Every thread of the block calls it.
template <int NT>
__device__ __noinline__ u64 exact_tail(const __half* row, int vocab, Weights wt, uint32_t lkey, u64* red) {
  u64 sum = 0, total;
  const int nvec = (vocab + 7) / 8;
#pragma unroll 1
  for (int i = threadIdx.x; i < nvec; i += NT) {
    const Vec v = load_vec<kFillNegInf>(row, i, vocab);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const uint32_t key = order_key_num(v.bits(j));
      const u64 w = to_units(wt.ex.value<true>(v.bits(j)));
      sum += key > kKeyNegInf && key < lkey ? w : 0ull;
    }
  }
  block_scan<NT>(sum, red, &total);
  return total;
}

constexpr int kFew = 256;

// The draw from lists of at most 256 entries together: ranked by counting, then every cut is a running sum over that many
// places. Leaves the list place, its key and the kept weight in s.bin, s.key and s.before.
template <int NT>
__device__ __noinline__ void draw_of_few(SampleShared<NT>& s, Weights wt, uint32_t top_k, float top_p, uint32_t mpkey,
                                         float u) {
  constexpr int NW = NT / 32, kOwn = SampleShared<NT>::kList / NW;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const uint32_t listed = lane < NW ? s.listed[lane] : 0u, listed_to = warp_scan(listed);
  const uint32_t n = __shfl_sync(0xffffffffu, listed_to, 31);
  const uint32_t before = __shfl_sync(0xffffffffu, listed_to - listed, warp);
  uint32_t* ck = s.fine;       // key, and the complement of the position in index order
  uint32_t* cp = s.fine + 256;  // list place
  u64* rw = reinterpret_cast<u64*>(s.fine + 512);   // weights in rank order
  u64* kw = reinterpret_cast<u64*>(s.fine + 1024);  // kept weights in index order
#pragma unroll 1
  for (uint32_t i = lane; i < s.listed[warp]; i += 32) {
    ck[before + i] = order_key_num(s.list[warp * kOwn + i]) << 16 | (0xffffu - (before + i));
    cp[before + i] = warp * kOwn + i;
  }
  if (tid < 4 && n + tid < kFew) ck[n + tid] = 0;
  __syncthreads();
  u64 w = 0;
  uint32_t rank = 0, key = 0;
  if (tid < n) {
    const uint32_t mine = ck[tid];
    for (uint32_t j = 0; j < n; j += 4) {
      const uint4 o = *reinterpret_cast<const uint4*>(&ck[j]);
      rank += (o.x > mine) + (o.y > mine) + (o.z > mine) + (o.w > mine);
    }
    key = mine >> 16;
    w = wt.of(key_bits(key));
    rw[rank] = w;
  }
  __syncthreads();
  const int c8 = lane * 8;
  u64 w8[8], sum = 0;
  if (warp == 0) {
    const uint32_t kk = min(top_k, n);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      w8[j] = c8 + j < kk ? rw[c8 + j] : 0ull;
      sum += w8[j];
    }
    const u64 inc = warp_scan(sum);
    uint32_t keep = kk;
    if (top_p < 1.f) {  // the ranks with less than the target before them
      const double target = fmax((double)top_p * (double)__shfl_sync(0xffffffffu, inc, 31), 1.0);
      u64 b = inc - sum;
      uint32_t cnt = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        cnt += c8 + j < kk && (double)b < target;
        b += w8[j];
      }
      keep = __reduce_add_sync(0xffffffffu, cnt);
    }
    if (lane == 0) s.left = keep;
  }
  __syncthreads();
  if (tid < n) kw[tid] = rank < s.left && key >= mpkey ? w : 0ull;
  __syncthreads();
  if (warp != 0) return;
  sum = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    w8[j] = c8 + j < n ? kw[c8 + j] : 0ull;
    sum += w8[j];
  }
  const u64 inc = warp_scan(sum);
  const u64 total = __shfl_sync(0xffffffffu, inc, 31);
  const u64 target = draw_at(u, total);
  u64 b = inc - sum;
  uint32_t found = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    if (b <= target && target < b + w8[j]) found = c8 + j + 1;
    b += w8[j];
  }
  found = __reduce_max_sync(0xffffffffu, found) - 1;
  if (lane == 0) {
    s.bin = cp[found];
    s.key = ck[found] >> 16;
    s.before = total;
  }
  __syncwarp();
}

template <int NT, bool kTryFew>
__global__ void __launch_bounds__(NT, 1024 / NT) sample_kernel(const SampleParams a) {
  extern __shared__ __align__(16) uint8_t smem_raw[];
  typedef SampleShared<NT> Shared;
  Shared& s = *reinterpret_cast<Shared*>(smem_raw);
  constexpr int NW = NT / 32;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int64_t r = blockIdx.x;
  const __half* row = a.logits + r * a.ld;
  const int vocab = a.vocab;
  const int nvec = (vocab + 7) / 8;
  constexpr int kOwn = Shared::kList / NW;       // places of a warp's list
  constexpr int kPer = kOwn / 256;               // groups of it
  const int stretch = (nvec + NW - 1) / NW;      // vectors of a warp's part of the row
  const int part = (stretch + 1023) / 1024 * 32;  // vectors of a 32nd of it, whole steps
  const int v0 = warp * stretch, v1 = min(v0 + stretch, nvec);
  auto vec = [&](int i) { return load_vec<kFillNegInf>(row, i, vocab); };
  const float Tr = a.temperature ? a.temperature[r] : a.temperature_s;
  // Past these bounds the weights no longer change: fp16 logits differ by 6e-8 to 131008, or not at all.
  const float T = Tr > 1e30f ? 1e30f : Tr > 0.f && Tr < 1e-9f ? 1e-9f : Tr;
  const int top_k = a.top_k ? a.top_k[r] : a.top_k_s;
  const float top_p = a.top_p ? a.top_p[r] : a.top_p_s;
  const float min_p = a.min_p ? a.min_p[r] : a.min_p_s;
  for (int i = tid; i < kExpTab; i += NT) s.tab[i] = exp2((double)i / kExpTab) * kUnit;

  const bool use_k = top_k > 0 && top_k < vocab;
  const bool use_p = top_p < 1.f;
  // A limit for top-k comes from a histogram of maxima: of the threads, or of the vectors if those are few against k.
  const bool by_thread = use_k && top_k <= min(nvec, NT) / 4, by_vector = use_k && !by_thread && top_k <= nvec / 4;
  if (by_thread || by_vector) {
    for (int i = tid; i < kBins; i += NT) s.fine[i] = 0;
    if (by_vector) __syncthreads();  // else block_max has one before the first use
  }

  // The maximum, NaN if one stands in the row.
  __half2 tmax = __half2half2(__ushort_as_half((unsigned short)kFillNegInf));
#pragma unroll 8
  for (int i = tid; i < nvec; i += NT) {
    const Vec v = vec(i);
    const __half2 m = __hmax2_nan(__hmax2_nan(as_half2(v.w[0]), as_half2(v.w[1])),
                                  __hmax2_nan(as_half2(v.w[2]), as_half2(v.w[3])));
    tmax = __hmax2_nan(tmax, m);
    if (by_vector) atomicAdd(&s.fine[order_key(__half_as_ushort(max_of(m))) >> 5], 1u);
  }
  const uint32_t tkey = order_key(__half_as_ushort(__hmax_nan(__low2half(tmax), __high2half(tmax))));
  const uint32_t mkey = block_max<NT>(tkey == 0 ? 0xffffu : tkey, s.red);
  if (mkey == 0xffffu || mkey <= kKeyNegInf) {  // a NaN, or nothing to draw from
    if (tid == 0) {
      a.tokens[r] = -1;
      if (a.logp) a.logp[r] = __int_as_float(0x7fc00000);
    }
    return;
  }
  const float m32 = __half2float(key_half(mkey));

  if (!(T > 0.f) || (use_k && top_k == 1) || min_p > 1.f) {  // the lowest index of the maximum
    const __half2 limit = __half2half2(key_half(mkey));
    uint32_t best = 0;  // ~index, so that the largest is the lowest index
#pragma unroll 1
    for (int i = tid; i < nvec; i += NT) {
      const uint32_t ge = vec_ge(vec(i), limit);
      if (ge) {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (ge & ge_bit(j)) best = max(best, ~(uint32_t)(8 * i + j));
        break;
      }
    }
    best = block_max<NT>(best, s.red);
    if (tid == 0) {
      a.tokens[r] = (int64_t)(~best);
      if (a.logp) a.logp[r] = 0.f;
    }
    return;
  }

  const bool minf = mkey == 0xfc00u;  // (Exp sees the bits of an infinity as 65536)
  const Weights wt{{minf ? 65536.0 : (double)m32, 256.0 * 1.4426950408889634 / (double)T, s.tab}, mkey};

  // Elements below `lkey` stay out of the list. First: weights that round to 0.
  auto key_below = [&](float x) {  // key of the largest half <= x, and never that of -inf
    return max(order_key(__half_as_ushort(__float2half_rd(x))), kKeyNegInf + 1);
  };
  // (30.2 nats are 2^-43.57; the bound itself is rounded up, so that no exponent is below that.)
  uint32_t lkey = mkey;
  if (!minf) lkey = min(mkey, max(order_key(__half_as_ushort(__float2half_ru(m32 - 30.2f * T))), kKeyNegInf + 1));

  // min-p as a key: the smallest key whose weight reaches it (32 probes a step, every warp for itself).
  uint32_t mpkey = 0;
  if (min_p > 0.f) {
    uint32_t lo = kKeyNegInf, hi = mkey;  // the weight of hi reaches min_p, that of lo does not
    const double want = (double)min_p * kUnit;
    while (hi - lo > 1) {
      const uint32_t step = (hi - lo + 31) / 32;
      const uint32_t key = min(lo + (lane + 1) * step, hi);
      const bool ok = key == mkey || (!minf && wt.ex.value<true>(key_bits(key)) >= want);
      const uint32_t first = __ffs(__ballot_sync(0xffffffffu, ok)) - 1;
      hi = min(lo + (first + 1) * step, hi);
      lo += first * step;
    }
    mpkey = hi;
    if (!use_p) lkey = max(lkey, mpkey);  // with top-p, what min-p drops still counts toward the sum
  }

  const bool tail = use_p && !use_k && !minf;  // what is below the limit is part of the sum
  uint32_t safe = lkey;                        // of a tried limit: the one that is always low enough
  const float c = (float)(1.4426950408889634 / (double)T);  // exponents are fma(x, c, c0)
  const float c0 = (float)(-(double)m32 * (double)c);
  if (by_thread || by_vector) {
    if (by_thread) atomicAdd(&s.fine[tkey >> 5], 1u);
    __syncthreads();
    int* found = reinterpret_cast<int*>(&s.key);  // key, left
    find_bin<NT>(s.fine, (uint32_t)top_k, s.red, found);
    if (found[0] >= 0) lkey = max(lkey, (uint32_t)found[0] << 5);
  } else if (tail) {
    safe = lkey = max(lkey, min(mkey, key_below(m32 + T * logf((1.f - fmaxf(top_p, 0.f)) * 0.999f / (float)vocab))));
    // From the row's first part: the weight below 2^-2.5, 2^-5, ... of the maximum.
    float below[kGuess + 1] = {};
    const Vec v = vec(tid);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 f = __half22float2(as_half2(v.w[j]));
      const float y0 = fmaf(f.x, c, c0), y1 = fmaf(f.y, c, c0);
      const float e0 = ex2(y0), e1 = ex2(y1);
      below[kGuess] += e0 + e1;
#pragma unroll
      for (int g = 0; g < kGuess; ++g) {
        if (y0 < -2.5f * (g + 1)) below[g] += e0;
        if (y1 < -2.5f * (g + 1)) below[g] += e1;
      }
    }
#pragma unroll
    for (int g = 0; g <= kGuess; ++g) {
      below[g] = warp_sum(below[g]);
      if (lane == 0) s.redf[warp][g] = below[g];
    }
    __syncthreads();
    float sum = 0.f;
    if (lane <= kGuess)
      for (int w = 0; w < NW; ++w) sum += s.redf[w][lane];
    // The whole row's weight: the light part scaled up, of the heavy one what was seen, or the maximum's.
    const float share = (float)vocab / (float)min(vocab, NT * 8);
    const float light = __shfl_sync(0xffffffffu, sum, 1);
    const float all = fmaxf(__shfl_sync(0xffffffffu, sum, kGuess) - light, 1.f) + light * share;
    // The first level that leaves three quarters of 1 - top_p below it, and a place between it and the one before.
    const float want = 0.75f * (1.f - top_p) * all;
    const uint32_t fits = __ballot_sync(0xffffffffu, lane < kGuess && sum * share <= want);
    if (fits) {
      const int g = __ffs(fits) - 1;
      const float upper = __shfl_sync(0xffffffffu, sum, max(g - 1, 0)) * share, lower = __shfl_sync(0xffffffffu, sum, g) * share;
      float at = (float)(g + 1);
      if (g > 0) at = (float)g + log2f(upper / want) / fmaxf(log2f(upper / fmaxf(lower, 1e-30f)), 1e-3f);
      lkey = max(lkey, min(mkey, key_below(m32 - 2.5f * fminf(at, (float)(g + 1)) / c)));
    }
    __syncthreads();
  }

  uint32_t tau, left;      // the lowest key kept; how many of the elements at it (0xffffffff: all)
  bool few = false;            // all lists together are short
  bool lists;              // or the whole row
  int ngroup, rounds;
  __half2 limit;
  // Group g: up to 256 entries that follow each other in the row.
  auto group = [&](int g, int& count) -> const unsigned short* {
    if (!lists) {
      count = min(256, vocab - g * 256);
      return reinterpret_cast<const unsigned short*>(row) + g * 256;
    }
    count = min(256, (int)s.listed[g / kPer] - g % kPer * 256);
    return s.list + g * 256;
  };
  // The groups of a warp: with lists, the k-th group of another list for every k, since the last ones are empty.
  auto group_of = [&](int k) -> int { return lists ? (warp + k) % NW * kPer + k : k * NW + warp; };
  auto key_of = [&](uint32_t bits) -> uint32_t {  // 0 below the limit (a whole row has such entries)
    const uint32_t key = order_key_num(bits);
    return key >= lkey ? key : 0u;
  };
  for (;;) {  // at most twice
    // The lists, and the weight of what stays out of them.
    limit = __half2half2(key_half(lkey));
    const float limit32 = __half2float(key_half(lkey));
    double rest = 0.0;
    uint32_t mine = 0;
    int parts = 0, mark = lane == 0 ? v0 : 0x7fffffff;
    auto own_vec = [&](int i) {
      Vec v;
      v.w[0] = v.w[1] = v.w[2] = v.w[3] = kFillNegInf * 0x10001u;
      if (i < v1) v = vec(i);
      return v;
    };
    // The next two steps' vectors are on their way while one is looked at.
    Vec v = own_vec(v0 + lane), ahead = own_vec(v0 + lane + 32), after;
#pragma unroll 1
    for (int i = v0 + lane; i < v0 + (v1 - v0 + 31 & ~31); i += 32, v = ahead, ahead = after) {
      after = own_vec(i + 64);
      const uint32_t ge = vec_ge(v, limit);
      if (i >= mark) {  // lane 0, at the first vector of a part
        s.upto[warp][parts++] = (unsigned short)min(mine, 0xffffu);
        mark += part;
      }
      if (__any_sync(0xffffffffu, ge)) {
        const uint32_t cnt = __popc(ge);
        const uint32_t upto = warp_scan(cnt);
        uint32_t at = mine + upto - cnt;
        mine += __shfl_sync(0xffffffffu, upto, 31);
        if (mine <= kOwn) {
#pragma unroll
          for (int j = 0; j < 8; ++j)
            if (ge & ge_bit(j)) s.list[warp * kOwn + at++] = (unsigned short)v.bits(j);
        }
      }
      if (tail) {
        float pair[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float2 f = __half22float2(as_half2(v.w[j]));
          const float e0 = ex2(fmaf(f.x, c, c0)), e1 = ex2(fmaf(f.y, c, c0));
          pair[j] = (f.x < limit32 ? e0 : 0.f) + (f.y < limit32 ? e1 : 0.f);
        }
        rest += (double)((pair[0] + pair[1]) + (pair[2] + pair[3]));
      }
    }
    if (lane == 0) s.listed[warp] = mine;
    if (tail) {
      rest = warp_sum_d(rest);
      if (lane == 0) s.red64[warp] = (u64)__double_as_longlong(rest);
    }
    __syncthreads();
    u64 tail_mass = 0;
    if (tail) {
      // What c and c0 lost to rounding, for the difference to the maximum that the weight below the limit has about: a
      // nat under it.
      const double lost = ((double)limit32 - (double)m32 - (double)T) * (1.4426950408889634 / (double)T - (double)c) +
                          (-(double)m32 * (double)c - (double)c0);
      const double below = warp_sum_d(lane < NW ? __longlong_as_double((long long)s.red64[lane]) : 0.0);
      // (Up to 2^62: below a tried limit may lie most of a smooth row's weight, many times the maximum's.)
      tail_mass = __double2ull_rn(below * (1.0 + 0.6931471805599453 * lost) * kUnit);
    }
    lists = __reduce_max_sync(0xffffffffu, lane < NW ? s.listed[lane] : 0u) <= kOwn;
    if (kTryFew && !tail) {
      few = __reduce_add_sync(0xffffffffu, lane < NW ? s.listed[lane] : 0u) <= min(NT, kFew);
      if (few) break;
    }
    ngroup = lists ? Shared::kList / 256 : (vocab + 255) / 256;
    rounds = (ngroup + NW - 1) / NW;

    tau = lkey, left = 0xffffffffu;
    if (!use_k && !use_p) break;
    // Bins in descending order of the keys; more than one key to a bin only where the range is wide.
    const uint32_t range = mkey - lkey;
    int shift = 0;
    if (range >= Shared::kFine)
      for (shift = 1; (range >> shift) >= Shared::kCoarse;) ++shift;
    const int bins = (int)(range >> shift) + 1;
    for (int i = tid; i < bins; i += NT) s.fine[i] = 0;
    if (shift)
      for (int i = tid; i < bins; i += NT)
        s.coarse.limb[0][i] = s.coarse.limb[1][i] = s.coarse.limb[2][i] = s.coarse.limb[3][i] = 0;
    __syncthreads();
#pragma unroll 1
    for (int k = 0; k < rounds; ++k) {
      const int g = group_of(k);
      if (g >= ngroup) break;
      int count;
      const unsigned short* p = group(g, count);
#pragma unroll 1
      for (int i = lane; i < count; i += 32) {
        const uint32_t bits = p[i], key = key_of(bits);
        if (!key) continue;
        const uint32_t b = (mkey - key) >> shift;
        atomicAdd(&s.fine[b], 1u);
        if (shift && use_p) {
          const u64 w = wt.of(bits);
#pragma unroll
          for (int l = 0; l < 4; ++l) atomicAdd(&s.coarse.limb[l][b], (uint32_t)(w >> (11 * l)) & 0x7ffu);
        }
      }
    }
    __syncthreads();
    auto bin_mass = [&](int b) -> u64 {
      if (shift)
        return s.coarse.limb[0][b] + ((u64)s.coarse.limb[1][b] << 11) + ((u64)s.coarse.limb[2][b] << 22) +
               ((u64)s.coarse.limb[3][b] << 33);
      const uint32_t cnt = s.fine[b];
      return cnt ? cnt * weight_of_key(wt, mkey - b) : 0ull;
    };
    const int per = (bins + NT - 1) / NT;
    const int b0 = min(tid * per, bins), b1 = min(b0 + per, bins);
    uint32_t csum = 0, ctotal;
    u64 msum = 0, mtotal = 0, mabove = 0;
#pragma unroll 1
    for (int i = b0; i < b1; ++i) {
      csum += s.fine[i];
      if (use_p) {
        if (shift)
          msum += bin_mass(i);
        else if (s.fine[i])
          msum += s.fine[i] * wt.of(key_bits(mkey - i));
      }
    }
    const uint32_t cabove = block_scan<NT>(csum, s.red, &ctotal);
    if (use_p) mabove = block_scan<NT>(msum, s.red64, &mtotal);
    if (lkey > safe && (double)mtotal < (double)fmaxf(top_p, 0.f) * (double)(mtotal + tail_mass) * (1.0 + kTailError) + kTailFar) {
      lkey = safe;  // the cut lies below the limit after all
      continue;
    }
    mtotal += tail_mass;

    // Counts of a bin's keys (up to 64), in descending order of the keys.
    auto fill_sub = [&](uint32_t bin) {
      if (tid < 64) s.sub[tid] = 0;
      __syncthreads();
#pragma unroll 1
      for (int k = 0; k < rounds; ++k) {
      const int g = group_of(k);
      if (g >= ngroup) break;
        int count;
        const unsigned short* p = group(g, count);
#pragma unroll 1
        for (int i = lane; i < count; i += 32) {
          const uint32_t key = key_of(p[i]), d = mkey - key;
          if (key && d >> shift == bin) atomicAdd(&s.sub[d & ((1u << shift) - 1u)], 1u);
        }
      }
      __syncthreads();
    };

    if (use_k && (uint32_t)top_k < ctotal) {
      if (cabove < (uint32_t)top_k && cabove + csum >= (uint32_t)top_k) {  // one thread
        uint32_t ab = cabove;
        u64 mb = mabove;
        int i = b0;
        while (ab + s.fine[i] < (uint32_t)top_k) {
          ab += s.fine[i];
          if (use_p) mb += bin_mass(i);
          ++i;
        }
        s.bin = i;
        s.left = (uint32_t)top_k - ab;
        s.before = mb;
      }
      __syncthreads();
      const uint32_t bin = s.bin;
      if (shift) fill_sub(bin);
      if (tid == 0) {
        uint32_t want = s.left, key = mkey - (bin << shift);
        if (shift)
          for (int i = 0; s.sub[i] < want; ++i, --key) {
            want -= s.sub[i];
            if (use_p && s.sub[i]) s.before += s.sub[i] * weight_of_key(wt, key);
          }
        if (use_p) s.before += want * weight_of_key(wt, key);  // the weight of the first top_k
        s.key = key;
        s.left = want;
      }
      __syncthreads();
      tau = s.key;
      left = s.left;
      mtotal = s.before;
      __syncthreads();
    }
    if (use_p) {
      // Kept are the ranks with less than `target` before them, and the first.
      for (bool exact = !tail;; exact = true) {  // at most twice
        const double target = fmax((double)top_p * (double)mtotal, 1.0);  // in units: the first has 2^42
        if (tid == 0) s.bin = 0xffffffffu;
        __syncthreads();
        if ((double)mabove < target && (double)(mabove + msum) >= target) {  // one thread, if the target is within
          u64 mb = mabove;
          int i = b0;
          for (; i < b1 - 1; ++i) {
            const u64 m = bin_mass(i);
            if ((double)(mb + m) >= target) break;
            mb += m;
          }
          s.bin = i;
          s.before = mb;
        }
        __syncthreads();
        const uint32_t bin = s.bin;
        if (bin == 0xffffffffu) break;
        if (shift) fill_sub(bin);
        if (tid == 0) {
          uint32_t key = mkey - (bin << shift), cnt = shift ? s.sub[0] : s.fine[bin];
          u64 mb = s.before, w = weight_of_key(wt, key);
          if (shift) {
            const int last = (1 << shift) - 1;
            for (int i = 0; i < last && (double)(mb + cnt * w) < target;) {
              mb += cnt * w;
              cnt = s.sub[++i];
              --key;
              w = cnt ? weight_of_key(wt, key) : 0ull;
            }
          }
          const double q = w ? (target - (double)mb) / (double)w : 0.0;
          s.key = key;
          s.left = w ? (uint32_t)fmin(fmax(ceil(q), 1.0), (double)cnt) : cnt;
          // Too near to a border for the error of the weight below the limit: once more with the exact one.
          s.again = !exact && fabs(q - rint(q)) * (double)w <= kTailError * (double)tail_mass + kTailFar ? 1u : 0u;
        }
        __syncthreads();
        if (s.again) {
          mtotal += exact_tail<NT>(row, vocab, wt, lkey, s.red64) - tail_mass;
          continue;
        }
        // Never past the top-k threshold.
        if (s.key > tau || (s.key == tau && s.left < left)) {
          tau = s.key;
          left = s.left;
        }
        break;
      }
    }
    if (mpkey > tau) {
      tau = mpkey;
      left = 0xffffffffu;
    }
    __syncthreads();  // the histogram's memory becomes the groups'
    break;
  }

  uint32_t place = 0, tkeyf = 0;  // of the token, and the sum of all that is kept
  u64 total = 0;
  if (kTryFew && few) {
    draw_of_few<NT>(s, wt, use_k ? (uint32_t)top_k : 0xffffffffu, use_p ? top_p : 1.f, mpkey, a.u[r]);
    if (warp != 0) return;
    place = s.bin, tkeyf = s.key, total = s.before;
  } else {
    // Weights and ties at tau per group.
    const bool ties = left != 0xffffffffu;
    u64* gmass = lists ? s.group.mass : s.row.mass;
    uint32_t* gties = lists ? s.group.ties : s.row.ties;
#pragma unroll 1
    for (int k = 0; k < rounds; ++k) {
      const int g = group_of(k);
      if (g >= ngroup) break;
      int count;
      const unsigned short* p = group(g, count);
      u64 w = 0;
      uint32_t tie = 0;
#pragma unroll 1
      for (int i = lane; i < count; i += 32) {
        const uint32_t bits = p[i], key = key_of(bits);
        if (ties && key == tau)
          ++tie;
        else if (key >= tau)
          w += wt.of(bits);
      }
      __syncwarp();
      if (count > 0) {
        w = warp_sum64(w);
        tie = __reduce_add_sync(0xffffffffu, tie);
      }
      if (lane == 0) {
        gmass[g] = w;
        gties[g] = tie;
      }
    }
    __syncthreads();
    if (warp != 0) return;

    // One warp: a run of groups per lane. Ties are kept while fewer than `left` stand before them.
    const u64 wtie = ties ? weight_of_key(wt, tau) : 0ull;
    const int per = (ngroup + 31) / 32;
    const int g0 = min(lane * per, ngroup), g1 = min(g0 + per, ngroup);
    uint32_t tsum = 0;
    u64 wsum = 0;
#pragma unroll 1
    for (int g = g0; g < g1; ++g) tsum += gties[g], wsum += gmass[g];
    uint32_t tb = warp_scan(tsum) - tsum;
    auto kept = [&](uint32_t before, uint32_t n) -> uint32_t { return before >= left ? 0u : min(n, left - before); };
    wsum += (u64)kept(tb, tsum) * wtie;
    const u64 winc = warp_scan(wsum);
    total = __shfl_sync(0xffffffffu, winc, 31);
    const u64 target = draw_at(a.u[r], total);
    u64 wb = winc - wsum;
    int g = 0;
    const bool mine = wb <= target && target < winc;
    if (mine) {
#pragma unroll 1
      for (g = g0; g < g1; ++g) {
        const u64 w = gmass[g] + (u64)kept(tb, gties[g]) * wtie;
        if (target < wb + w) break;
        wb += w;
        tb += gties[g];
      }
    }
    const int src = __ffs(__ballot_sync(0xffffffffu, mine)) - 1;
    g = __shfl_sync(0xffffffffu, g, src);
    wb = __shfl_sync(0xffffffffu, wb, src);
    tb = __shfl_sync(0xffffffffu, tb, src);
    // Within the group, eight entries a lane.
    int count;
    const unsigned short* p = group(g, count);
    u64 w8[8];
    uint32_t tie8 = 0, bits8[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const bool in = lane * 8 + j < count;
      bits8[j] = in ? p[lane * 8 + j] : 0u;
      const uint32_t key = in ? key_of(bits8[j]) : 0u;
      const bool tie = ties && key == tau;
      tie8 |= tie ? 1u << j : 0u;
      w8[j] = !tie && key >= tau ? wt.of(bits8[j]) : 0ull;
    }
    tb += warp_scan((uint32_t)__popc(tie8)) - __popc(tie8);
    wsum = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if (tie8 >> j & 1) {
        w8[j] = tb < left ? wtie : 0ull;
        ++tb;
      }
      wsum += w8[j];
    }
    wb += warp_scan(wsum) - wsum;
    uint32_t bitsf = 0;  // (place and bitsf: of the lane that has it)
    if (wb <= target && target < wb + wsum) {
      bool open = true;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        wb += w8[j];
        if (open && target < wb) {
          open = false;
          place = g * 256 + lane * 8 + j + 1;
          bitsf = bits8[j];
        }
      }
    }
    place = __reduce_max_sync(0xffffffffu, place) - 1;
    tkeyf = order_key_num(__reduce_max_sync(0xffffffffu, bitsf));

  }

  // The element of that place: in a list, the so-manieth above the limit of its warp's stretch.
  int64_t token = place;
  if (lists) {
    const int w = place / kOwn;
    uint32_t want = place - w * kOwn;
    const int e0 = w * stretch, e1 = min(e0 + stretch, nvec);
    const uint32_t here = e0 + lane * part < e1 ? s.upto[w][lane] : 0xffffffffu;
    const int at = __popc(__ballot_sync(0xffffffffu, here <= want)) - 1;  // the part that holds it
    want -= __shfl_sync(0xffffffffu, here, at);
#pragma unroll 1
    for (int i = e0 + at * part + lane; i - lane < e1; i += 32) {
      const uint32_t ge = i < e1 ? vec_ge(vec(i), limit) : 0u;
      const uint32_t cnt = __popc(ge), sum = __reduce_add_sync(0xffffffffu, cnt);
      if (want >= sum) {
        want -= sum;
        continue;
      }
      uint32_t before = warp_scan(cnt) - cnt, found = 0;  // index + 1
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (ge & ge_bit(j)) {
          if (before == want) found = (uint32_t)(i * 8 + j) + 1;
          ++before;
        }
      token = (int64_t)__reduce_max_sync(0xffffffffu, found) - 1;
      break;
    }
  }
  if (lane == 0) {
    a.tokens[r] = token;
    if (a.logp) {
      const double d = tkeyf == mkey ? 0.0 : ((double)__half2float(key_half(tkeyf)) - (double)m32) / (double)T;
      a.logp[r] = (float)(d - log((double)total / kUnit));
    }
  }
}

template <int NT, typename C, bool kLarge>
int launch_top_as(const __half* x, int64_t rows, int64_t ld, int vocab, int k, __half* values, int64_t* ids, cudaStream_t s) {
  static std::atomic<uint64_t> done{0};
  JX_CUDA_TRY(once_per_device(done,
                              [] {
                                return cudaFuncSetAttribute(top_logits_kernel<NT, 8, C, kLarge>,
                                                            cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                            (int)sizeof(TopShared<NT, C, kLarge>));
                              }),
              "jx_top_logits: shared memory");
  top_logits_kernel<NT, 8, C, kLarge><<<(unsigned)rows, NT, sizeof(TopShared<NT, C, kLarge>), s>>>(x, ld, vocab, k, values, ids);
  JX_CHECK_LAUNCH("jx_top_logits");
  return JX_OK;
}

// A limit from the threads' maxima lets few elements more than k pass while k is small against the threads; from there
// on the vectors' maxima give it (4096 rows of 32000: top 160 95 us by threads, 105 by vectors; top 256 330 and 138).
template <int NT, typename C>
int launch_top(const __half* x, int64_t rows, int64_t ld, int vocab, int k, __half* values, int64_t* ids, cudaStream_t s) {
  return k > std::min((vocab + 7) / 8, NT) * 3 / 8 ? launch_top_as<NT, C, true>(x, rows, ld, vocab, k, values, ids, s)
                                                   : launch_top_as<NT, C, false>(x, rows, ld, vocab, k, values, ids, s);
}

template <int NT, bool kTryFew>
int launch_sample_as(const SampleParams& p, int64_t rows, cudaStream_t s) {
  static std::atomic<uint64_t> done{0};
  JX_CUDA_TRY(once_per_device(done,
                              [] {
                                return cudaFuncSetAttribute(sample_kernel<NT, kTryFew>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                            (int)sizeof(SampleShared<NT>));
                              }),
              "jx_sample: shared memory");
  sample_kernel<NT, kTryFew><<<(unsigned)rows, NT, sizeof(SampleShared<NT>), s>>>(p);
  JX_CHECK_LAUNCH("jx_sample");
  return JX_OK;
}

// Short lists are worth the look where top-k or min-p may make them (one row of 32000 with all filters 15.7 -> 10.6 us, 20000
// rows of 2000 with top-k 680 -> 204). Where neither can, the code for them would only cost the long lists' loops registers
// (1024 rows of 50257 with top-p 170 -> 171 us).
template <int NT>
int launch_sample(const SampleParams& p, int64_t rows, cudaStream_t s) {
  return p.top_k || p.top_k_s > 0 || p.min_p || p.min_p_s > 0.f ? launch_sample_as<NT, true>(p, rows, s)
                                                                : launch_sample_as<NT, false>(p, rows, s);
}

}  // namespace sel
}  // namespace jx

using namespace jx;

extern "C" int jx_top_logits(const void* logits16, int64_t rows, int vocab, int64_t ld, int k, void* values16,
                             int64_t* ids, jx_stream_t stream) {
  JX_CHECK_ARG(rows > 0 && rows <= 0x7fffffff && vocab > 0 && vocab <= 1 << 30 && ld >= vocab, "jx_top_logits: bad shape");
  JX_CHECK_ARG(k > 0 && k <= vocab && k <= sel::kMaxTop, "jx_top_logits: k must be in [1, min(vocab, %d)] (got %d)",
               sel::kMaxTop, k);
  JX_CHECK_ARG(logits16 && values16 && ids, "jx_top_logits: NULL argument");
  JX_CHECK_ARG(ld % 8 == 0 && aligned16(logits16), "jx_top_logits: ld%%8 and 16B alignment required");
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const __half* x = static_cast<const __half*>(logits16);
  __half* v = static_cast<__half*>(values16);
  // Threads by the row's length, so that their registers hold it and short rows do not leave most of them idle (4096
  // rows of 8000 with 512 threads each 60.8 us for the top 100, with 128 35.5 us).
  if (vocab <= 128 * 64) return sel::launch_top<128, uint32_t>(x, rows, ld, vocab, k, v, ids, s);
  if (vocab <= 256 * 64) return sel::launch_top<256, uint32_t>(x, rows, ld, vocab, k, v, ids, s);
  if (vocab <= 65536) return sel::launch_top<512, uint32_t>(x, rows, ld, vocab, k, v, ids, s);
  return sel::launch_top<512, sel::u64>(x, rows, ld, vocab, k, v, ids, s);
}

extern "C" int jx_sample(const void* logits16, int64_t rows, int vocab, int64_t ld, const float* uniforms,
                         const float* temperatures, float temperature, const int32_t* top_ks, int top_k,
                         const float* top_ps, float top_p, const float* min_ps, float min_p, int64_t* tokens,
                         float* logprobs, jx_stream_t stream) {
  JX_CHECK_ARG(logits16 && uniforms && tokens, "jx_sample: NULL argument");
  JX_CHECK_ARG(rows > 0 && rows <= 0x7fffffff && vocab > 0 && vocab <= sel::kGroups * 256 && ld >= vocab,
               "jx_sample: bad shape (rows %lld, vocab %d, at most %d)", (long long)rows, vocab, sel::kGroups * 256);
  JX_CHECK_ARG(ld % 8 == 0 && aligned16(logits16), "jx_sample: ld%%8 and 16B alignment required");
  sel::SampleParams p{static_cast<const __half*>(logits16), ld, vocab, uniforms, temperatures, top_ks, top_ps, min_ps,
                      temperature, top_p, min_p, top_k, tokens, logprobs};
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  // Two blocks of 512 threads share an SM where there are rows for them, else a row gets 1024 (one row of 32000 with top-k
  // and top-p: 10.7 us, 1024 rows of 50257 with top-p 170 us). Five small blocks where rows are short and
  // many waves of them come (20000 rows of 2000 with top-p 1070 -> 527 us; 600 rows of 4000 with settings row by row 38 -> 46).
  if (rows > 8 * num_sms() && vocab <= sel::kShort) return sel::launch_sample<128>(p, rows, s);
  return rows > num_sms() ? sel::launch_sample<512>(p, rows, s) : sel::launch_sample<1024>(p, rows, s);
}
