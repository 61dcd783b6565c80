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

__device__ __forceinline__ uint32_t key_bits(uint32_t key) { return (key & 0x8000u) ? key ^ 0x8000u : ~key & 0xffffu; }

__device__ __forceinline__ __half key_half(uint32_t key) { return __ushort_as_half((unsigned short)key_bits(key)); }

// Eight consecutive logits; elements at and past `vocab` read as NaN, which no comparison selects. A row
// starts on a 16-byte boundary; only whole vectors are read as one.
struct Vec {
  uint32_t w[4];
  __device__ __forceinline__ uint32_t bits(int j) const { return (w[j >> 1] >> ((j & 1) * 16)) & 0xffffu; }
};

__device__ __forceinline__ Vec load_vec(const __half* row, int64_t first, int vocab) {
  Vec v;
  if (first + 8 <= vocab) {
    const uint4 u = __ldg(reinterpret_cast<const uint4*>(row + first));
    v.w[0] = u.x, v.w[1] = u.y, v.w[2] = u.z, v.w[3] = u.w;
  } else {
    const unsigned short* p = reinterpret_cast<const unsigned short*>(row);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t lo = first + 2 * j < vocab ? p[first + 2 * j] : 0xffffu;
      const uint32_t hi = first + 2 * j + 1 < vocab ? p[first + 2 * j + 1] : 0xffffu;
      v.w[j] = lo | (hi << 16);
    }
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
  for (int j = 0; j < 4; ++j) m |= (__hge2_mask(as_half2(v.w[j]), limit) & 0x10001u) << j;
  // bits 0..3: elements 0, 2, 4, 6; bits 16..19: elements 1, 3, 5, 7
  return m;
}
__device__ __forceinline__ uint32_t ge_bit(int j) { return (j & 1) ? 0x10000u << (j >> 1) : 1u << (j >> 1); }

// ---------------------------------------------------------------------------------------------------------
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
// second pass). The k-th largest of any part of the row is a lower bound of the k-th largest of all of it, so
// the maxima of the threads (or of the 8-element vectors where k is large) go into a histogram of their
// keys' upper 11 bits and the bin that holds the k-th of them gives a limit that little more than k elements
// pass. Those are collected, ranked among themselves and written. A row where more than kCand elements pass
// (many equal values) takes the exact way: two histograms find the threshold key, values at it are taken
// in index order.
// ---------------------------------------------------------------------------------------------------------
constexpr int kBins = 2048;     // upper 11 bits of a key
constexpr int kCand = 2048;     // candidates a block can hold
constexpr int kMaxTop = 1024;

// With hist[bin] counting keys, finds the bin (from the top) in which the k-th key falls and how many keys lie
// in higher bins; found[0] = -1 if there are fewer than k keys in all.
template <int NT>
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

template <int NT, int VPT>
__global__ void __launch_bounds__(NT, 1024 / NT)
    top_logits_kernel(const __half* __restrict__ logits, int64_t ld, int vocab, int k, __half* __restrict__ values,
                      int64_t* __restrict__ ids) {
  __shared__ uint32_t hist[kBins];
  __shared__ u64 cand[kCand];
  __shared__ uint32_t red[32];
  __shared__ int found[2];
  __shared__ uint32_t ncand;
  const int tid = threadIdx.x;
  const __half* row = logits + (int64_t)blockIdx.x * ld;
  const int nvec = (vocab + 7) / 8;
  const int nchunk = (nvec + NT * VPT - 1) / (NT * VPT);

  for (int i = tid; i < kBins; i += NT) hist[i] = 0;
  if (tid == 0) ncand = 0;
  __syncthreads();

  // Maxima into the histogram: one a thread, or one a vector where k is large against their number.
  const bool fine = (int64_t)k * 4 > min(nvec, NT);
  Vec v[VPT];
  __half2 tmax = __half2half2(__ushort_as_half(0xffffu));
  for (int c = 0; c < nchunk; ++c) {
#pragma unroll
    for (int i = 0; i < VPT; ++i) v[i] = load_vec(row, 8 * (int64_t)((c * VPT + i) * NT + tid), vocab);
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const __half2 m = vec_max2(v[i]);
      if (fine) {
        const uint32_t key = order_key(__half_as_ushort(max_of(m)));
        if (key) atomicAdd(&hist[key >> 5], 1u);
      }
      tmax = __hmax2(tmax, m);
    }
  }
  if (!fine) {
    const uint32_t key = order_key(__half_as_ushort(max_of(tmax)));
    if (key) atomicAdd(&hist[key >> 5], 1u);
  }
  __syncthreads();
  find_bin<NT>(hist, (uint32_t)k, red, found);
  // Fewer maxima than k: every element is a candidate (NaN too), if they fit.
  const bool all = found[0] < 0;
  const __half2 limit = __half2half2(key_half(all ? kKeyNegInf : max((uint32_t)found[0] << 5, kKeyNegInf)));
  uint32_t n = kCand + 1;
  if (!all || vocab <= kCand) {
    for (int c = 0; c < nchunk; ++c) {
      if (nchunk > 1) {
#pragma unroll
        for (int i = 0; i < VPT; ++i) v[i] = load_vec(row, 8 * (int64_t)((c * VPT + i) * NT + tid), vocab);
      }
#pragma unroll
      for (int i = 0; i < VPT; ++i) {
        const int64_t first = 8 * (int64_t)((c * VPT + i) * NT + tid);
        const uint32_t m = all ? 0xf000fu : vec_ge(v[i], limit);
        if (m) {
#pragma unroll
          for (int j = 0; j < 8; ++j)
            if ((m & ge_bit(j)) && first + j < vocab) {
              const uint32_t p = atomicAdd(&ncand, 1u);
              if (p < kCand) cand[p] = ((u64)order_key(v[i].bits(j)) << 32) | (0xffffffffu - (uint32_t)(first + j));
            }
        }
      }
    }
    __syncthreads();
    n = ncand;
  }
  if (n > kCand) {
    // The exact way: threshold key from histograms over the whole row, then the keys above it and, in index
    // order, as many at it as are left to take.
    __syncthreads();
    for (int i = tid; i < kBins; i += NT) hist[i] = 0;
    if (tid == 0) ncand = 0;
    __syncthreads();
    const unsigned short* p = reinterpret_cast<const unsigned short*>(row);
    for (int i = tid; i < vocab; i += NT) atomicAdd(&hist[order_key(p[i]) >> 5], 1u);
    __syncthreads();
    find_bin<NT>(hist, (uint32_t)k, red, found);
    const uint32_t bin = (uint32_t)found[0];
    uint32_t left = (uint32_t)k - (uint32_t)found[1];
    __syncthreads();
    for (int i = tid; i < kBins; i += NT) hist[i] = 0;
    __syncthreads();
    for (int i = tid; i < vocab; i += NT) {
      const uint32_t key = order_key(p[i]);
      if (key >> 5 == bin) atomicAdd(&hist[key & 31u], 1u);
    }
    __syncthreads();
    uint32_t sub = 31;
    while (hist[sub] < left) left -= hist[sub--];
    const uint32_t tau = (bin << 5) | sub;
    uint32_t taken = 0;
    for (int base = 0; base < vocab; base += NT) {
      const int i = base + tid;
      const uint32_t key = i < vocab ? order_key(p[i]) : 0u;
      const uint32_t tie = i < vocab && key == tau ? 1u : 0u;
      uint32_t total = 0, before = 0;
      if (taken < left) before = taken + block_scan<NT>(tie, red, &total);
      if (i < vocab && (key > tau || (tie && taken < left && before < left)))
        cand[atomicAdd(&ncand, 1u)] = ((u64)key << 32) | (0xffffffffu - (uint32_t)i);
      taken += total;
    }
    __syncthreads();
    n = ncand;  // k
  }
  __half* vout = values + (int64_t)blockIdx.x * k;
  int64_t* iout = ids + (int64_t)blockIdx.x * k;
  auto write = [&](uint32_t rank, u64 c) {
    vout[rank] = key_half((uint32_t)(c >> 32));
    iout[rank] = (int64_t)(0xffffffffu - (uint32_t)c);
  };
  if (n <= 256) {
    // Few: the rank of each is the number of larger ones (no two are equal: the index is part of them).
    for (uint32_t i = tid; i < n; i += NT) {
      const u64 mine = cand[i];
      uint32_t rank = 0;
      for (uint32_t j = 0; j < n; ++j) rank += cand[j] > mine;
      if (rank < (uint32_t)k) write(rank, mine);
    }
  } else {
    // Bitonic sort, largest first, padded with zeros to a power of two (no candidate is 0).
    uint32_t size = 512;
    while (size < n) size <<= 1;
    for (uint32_t i = n + tid; i < size; i += NT) cand[i] = 0;
    __syncthreads();
    for (uint32_t len = 2; len <= size; len <<= 1) {
      for (uint32_t half = len >> 1; half > 0; half >>= 1) {
        for (uint32_t t = tid; t < size / 2; t += NT) {
          const uint32_t i = 2 * half * (t / half) + t % half, j = i + half;
          const bool down = (i & len) == 0;
          const u64 a = cand[i], b = cand[j];
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
// One block per row. The maximum first; it gives a limit below which an element cannot be kept, or only as part
// of a sum:
//   - e < 2^-43: its weight rounds to 0;
//   - top-k: below a limit from the threads' maxima, as in top_logits_kernel;
//   - top-p without top-k: e < (1 - top_p) / V, since all such elements together weigh less than what top-p
//     drops (the maximum alone weighs 1). Their sum, a part of the total of at most 1 - top_p, is taken in fp32;
//     its error (about 1e-9 of the total, from arguments with an exact difference and a two-part 1 / T) only
//     moves the place of the cut, by less than a thousandth of the tokens' weight there.
// The elements above the limit are copied, in index order, to a list in shared memory, so that the exponentials
// run on full warps. A histogram of the list's keys (counts and weights) gives the threshold key; then the kept
// weights are summed per 256 list places, and the group where the running sum passes its target is walked
// by one warp. A list that does not fit is replaced by the whole row, read again from memory (L2) by each step.
constexpr int kSegs = 4096;                // segments of 256 elements: vocabularies up to 2^20
constexpr int kList = 32768;               // list places
constexpr double kUnit = 4398046511104.0;  // 2^42: weights of a row of 2^20 elements sum to at most 2^62
constexpr int kExpTab = 64;

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

// e * 2^42 for x = M + d (see weight()): 2^(j/64) from the table, the rest of the exponent by the Taylor
// series of 2^(r/64), |r| <= 1/2, to the fourth power (relative error below 4e-14).
struct Exp {
  double m;        // the row's maximum
  double c;        // 64 log2(e) / T
  const double* tab;

  __device__ __forceinline__ double value(uint32_t h) const {
    // A half's bits moved to a double's places are the value times 2^-1008, subnormals too.
    const double x = __hiloint2double((int)((h & 0x8000u) << 16 | (h & 0x7fffu) << 10), 0);
    const double y = fma(x, 0x1p1008, -m) * c;  // 64 log2(e_i), exact difference
    if (!(y > -64.0 * 60.0)) return 0.0;
    const double t = y + 0x1.8p52;  // rounds to an integer, which sits in the low word
    const int n = __double2loint(t);
    const double r = y - (t - 0x1.8p52);
    const double b = 0.010830424696249145;  // ln 2 / 64
    const double z = r * b;
    const double p = fma(z, fma(z, fma(z, fma(z, 1.0 / 24.0, 1.0 / 6.0), 0.5), 1.0), 1.0);
    const double w = tab[n & (kExpTab - 1)];
    return __hiloint2double(__double2hiint(w) + ((n >> 6) << 20), __double2loint(w)) * p;
  }
};

// round(v) of 0 <= v < 2^51 as an integer.
__device__ __forceinline__ u64 to_units(double v) {
  return (u64)__double_as_longlong(v + 0x1p52) & 0xfffffffffffffull;
}

struct SampleShared {
  union {
    unsigned short list[kList];
    struct {
      u64 mass[kSegs];
      uint32_t ties[kSegs];
    } row;  // groups of the whole row, where there is no list
  };
  union {
    struct {
      u64 mass[kBins];
      uint32_t count[kBins];
    } hist;
    struct {
      u64 mass[kList / 256];
      uint32_t ties[kList / 256];
    } group;
  };
  uint32_t seg[kSegs];  // list place of each segment's first entry
  uint32_t sub[32];
  double tab[kExpTab];
  u64 red64[32];
  uint32_t red[32];
  float redf[32];
  uint32_t key, left, bin;
  u64 before;
};

template <int NT, int VPT, bool kRegs>
__global__ void __launch_bounds__(NT, 1024 / NT) sample_kernel(const SampleParams a) {
  extern __shared__ __align__(16) uint8_t smem_raw[];
  SampleShared& s = *reinterpret_cast<SampleShared*>(smem_raw);
  constexpr int NW = NT / 32;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int64_t r = blockIdx.x;
  const __half* row = a.logits + r * a.ld;
  const int vocab = a.vocab;
  const int nvec = (vocab + 7) / 8;
  const int nchunk = kRegs ? 1 : (nvec + NT * VPT - 1) / (NT * VPT);
  Vec v[VPT];
  auto load = [&](int c) {
#pragma unroll
    for (int i = 0; i < VPT; ++i) v[i] = load_vec(row, 8 * (int64_t)((c * VPT + i) * NT + tid), vocab);
  };
  load(0);
  const float T = a.temperature ? a.temperature[r] : a.temperature_s;
  const int top_k = a.top_k ? a.top_k[r] : a.top_k_s;
  const float top_p = a.top_p ? a.top_p[r] : a.top_p_s;
  const float min_p = a.min_p ? a.min_p[r] : a.min_p_s;
  if (tid < kExpTab) s.tab[tid] = exp2((double)tid / kExpTab) * kUnit;

  // Maximum, and whether a NaN stands in the row (a position past the end reads as one, and is not asked).
  __half2 tmax = __half2half2(__ushort_as_half(0xffffu));
  bool nan = false;
  for (int c = 0; c < nchunk; ++c) {
    if (c) load(c);
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int64_t first = 8 * (int64_t)((c * VPT + i) * NT + tid);
      tmax = __hmax2(tmax, vec_max2(v[i]));
      uint32_t bad = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) bad |= __hneu2_mask(as_half2(v[i].w[j]), as_half2(v[i].w[j]));
      if (bad) {
#pragma unroll
        for (int j = 0; j < 8; ++j) nan |= first + j < vocab && (v[i].bits(j) & 0x7fffu) > 0x7c00u;
      }
    }
  }
  const uint32_t tkey = order_key(__half_as_ushort(max_of(tmax)));
  const uint32_t mkey = block_max<NT>(nan ? 0xffffu : tkey, s.red);
  if (mkey == 0xffffu || mkey <= kKeyNegInf) {  // a NaN, or nothing to draw from
    if (tid == 0) {
      a.tokens[r] = -1;
      if (a.logp) a.logp[r] = __int_as_float(0x7fc00000);
    }
    return;
  }
  const __half mhalf = key_half(mkey);
  const float m32 = __half2float(mhalf);
  const bool greedy = !(T > 0.f);
  const bool use_k = top_k > 0 && top_k < vocab;
  const bool use_p = top_p < 1.f;

  if (greedy || (use_k && top_k == 1) || min_p > 1.f) {  // the lowest index of the maximum
    const __half2 limit = __half2half2(mhalf);
    uint32_t best = 0;  // ~index, so that the largest is the lowest index
    for (int c = 0; c < nchunk; ++c) {
      if (nchunk > 1) load(c);
#pragma unroll
      for (int i = 0; i < VPT; ++i) {
        const uint32_t ge = vec_ge(v[i], limit);
        if (ge) {
#pragma unroll
          for (int j = 7; j >= 0; --j)
            if (ge & ge_bit(j)) best = max(best, ~(uint32_t)(8 * ((c * VPT + i) * NT + tid) + j));
        }
      }
    }
    best = block_max<NT>(best, s.red);
    if (tid == 0) {
      a.tokens[r] = (int64_t)(~best);
      if (a.logp) a.logp[r] = 0.f;
    }
    return;
  }

  const Exp ex{(double)m32, 64.0 * 1.4426950408889634 / (double)T, s.tab};
  // An infinite maximum leaves every finite logit without weight.
  const bool minf = mkey == 0xfc00u;
  auto units = [&](uint32_t bits, uint32_t key) -> u64 {
    return key == mkey ? (u64)kUnit : minf ? 0ull : to_units(ex.value(bits));
  };

  // Elements below `lkey` stay out of the list. First: weights that round to 0.
  auto key_below = [&](float x) {  // key of the largest half <= x, and never that of -inf
    return max(order_key(__half_as_ushort(__float2half_rd(x))), kKeyNegInf + 1);
  };
  uint32_t lkey = minf ? mkey : min(mkey, key_below(m32 - 30.2f * T));

  // min-p as a key: the smallest key whose weight reaches it (32 probes a step, every warp for itself).
  uint32_t mpkey = 0;
  if (min_p > 0.f) {
    uint32_t lo = kKeyNegInf, hi = mkey;  // the weight of hi reaches min_p, that of lo does not
    const double want = (double)min_p * kUnit;
    while (hi - lo > 1) {
      const uint32_t step = (hi - lo + 31) / 32;
      const uint32_t key = min(lo + (lane + 1) * step, hi);
      const bool ok = key == mkey || (!minf && ex.value(key_bits(key)) >= want);
      const uint32_t first = __ffs(__ballot_sync(0xffffffffu, ok)) - 1;
      hi = min(lo + (first + 1) * step, hi);
      lo += first * step;
    }
    mpkey = hi;
    if (!use_p) lkey = max(lkey, mpkey);  // with top-p, what min-p drops still counts toward the sum
  }

  const bool tail = use_p && !use_k && !minf;  // what is below the limit is part of the sum
  if (use_k && top_k * 4 <= min(nvec, NT)) {
    for (int i = tid; i < kBins; i += NT) s.hist.count[i] = 0;
    __syncthreads();
    if (tkey) atomicAdd(&s.hist.count[tkey >> 5], 1u);
    __syncthreads();
    int* found = reinterpret_cast<int*>(&s.key);  // key, left
    find_bin<NT>(s.hist.count, (uint32_t)top_k, s.red, found);
    if (found[0] >= 0) lkey = max(lkey, (uint32_t)found[0] << 5);
  } else if (tail) {
    lkey = max(lkey, min(mkey, key_below(m32 + T * logf((1.f - fmaxf(top_p, 0.f)) * 0.999f / (float)vocab))));
  }

  // The list: entries per segment of 256 elements (one warp's vectors of one step), their places, the copy.
  const __half2 limit = __half2half2(key_half(lkey));
  const int nseg = (vocab + 255) / 256;
  float rest = 0.f;
  const float c_hi = (float)(1.4426950408889634 / (double)T);
  const float c_lo = (float)(1.4426950408889634 / (double)T - (double)c_hi);
  for (int c = 0; c < nchunk; ++c) {
    if (nchunk > 1) load(c);
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const uint32_t ge = vec_ge(v[i], limit);
      const uint32_t n = __reduce_add_sync(0xffffffffu, __popc(ge));
      const int seg = (c * VPT + i) * NW + warp;
      if (lane == 0 && seg < nseg) s.seg[seg] = n;
      if (tail) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float2 f = __half22float2(as_half2(v[i].w[j]));
          const float d0 = f.x - m32, d1 = f.y - m32;
          const float e0 = exp2f(fmaf(d0, c_hi, d0 * c_lo)), e1 = exp2f(fmaf(d1, c_hi, d1 * c_lo));
          // a position past the end is a NaN, for which e < 2 is false too
          rest += (!(ge & ge_bit(2 * j)) && e0 < 2.f ? e0 : 0.f) + (!(ge & ge_bit(2 * j + 1)) && e1 < 2.f ? e1 : 0.f);
        }
      }
    }
  }
  u64 tail_mass = 0;
  if (tail) {
    rest = warp_sum(rest);
    if (lane == 0) s.redf[warp] = rest;
    __syncthreads();
    tail_mass = to_units((double)warp_sum(lane < NW ? s.redf[lane] : 0.f) * kUnit);
  }
  __syncthreads();
  uint32_t nlist;
  {
    constexpr int PER = kSegs / NT;
    uint32_t n[PER], sum = 0;
    const int per = (nseg + NT - 1) / NT;  // segments a thread
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      n[i] = i < per && tid * per + i < nseg ? s.seg[tid * per + i] : 0u;
      sum += n[i];
    }
    uint32_t at = block_scan<NT>(sum, s.red, &nlist);
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      if (i < per && tid * per + i < nseg) s.seg[tid * per + i] = at;
      at += n[i];
    }
  }
  __syncthreads();
  const bool listed = nlist <= kList;
  if (listed) {
    for (int c = 0; c < nchunk; ++c) {
      if (nchunk > 1) load(c);
#pragma unroll
      for (int i = 0; i < VPT; ++i) {
        const uint32_t ge = vec_ge(v[i], limit);
        if (__any_sync(0xffffffffu, ge)) {
          const int seg = (c * VPT + i) * NW + warp;
          const uint32_t n = __popc(ge);
          uint32_t at = s.seg[min(seg, nseg - 1)] + warp_scan(n) - n;
#pragma unroll
          for (int j = 0; j < 8; ++j)
            if (ge & ge_bit(j)) s.list[at++] = (unsigned short)v[i].bits(j);
        }
      }
    }
  }
  const uint32_t n = listed ? nlist : (uint32_t)vocab;  // places
  const unsigned short* source = listed ? s.list : reinterpret_cast<const unsigned short*>(row);
  auto entry = [&](uint32_t place, uint32_t& bits) -> uint32_t {  // key, or 0 where nothing is
    bits = source[place];
    const uint32_t key = order_key(bits);
    return key >= lkey ? key : 0u;
  };
  __syncthreads();

  // tau: the lowest key kept; left: how many of the elements at it (0xffffffff: all).
  uint32_t tau = lkey, left = 0xffffffffu;
  if (use_k || use_p) {
    int shift = 0;
    while (((mkey - lkey) >> shift) >= kBins) ++shift;
    for (int i = tid; i < kBins; i += NT) {
      s.hist.count[i] = 0;
      s.hist.mass[i] = 0;
    }
    __syncthreads();
    for (uint32_t p = tid; p < n; p += NT) {
      uint32_t bits;
      const uint32_t key = entry(p, bits);
      if (key) {
        const uint32_t b = (mkey - key) >> shift;
        atomicAdd(&s.hist.count[b], 1u);
        if (use_p) atomicAdd(&s.hist.mass[b], units(bits, key));
      }
    }
    __syncthreads();
    constexpr int PER = kBins / NT;
    uint32_t cnt[PER], csum = 0, ctotal;
    u64 mass[PER], msum = 0, mtotal = 0, mabove = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      cnt[i] = s.hist.count[tid * PER + i];
      csum += cnt[i];
      mass[i] = s.hist.mass[tid * PER + i];
      msum += mass[i];
    }
    const uint32_t cabove = block_scan<NT>(csum, s.red, &ctotal);
    if (use_p) mabove = block_scan<NT>(msum, s.red64, &mtotal);
    mtotal += tail_mass;

    // Counts of a bin's keys, in descending order of the keys.
    auto fill_sub = [&](uint32_t bin) {
      if (tid < 32) s.sub[tid] = 0;
      __syncthreads();
      for (uint32_t p = tid; p < n; p += NT) {
        uint32_t bits;
        const uint32_t key = entry(p, bits), d = mkey - key;
        if (key && d >> shift == bin) atomicAdd(&s.sub[d & ((1u << shift) - 1u)], 1u);
      }
      __syncthreads();
    };

    if (use_k && (uint32_t)top_k < ctotal) {
      uint32_t ab = cabove;
      u64 mb = mabove;
      if (ab < (uint32_t)top_k && ab + csum >= (uint32_t)top_k) {
#pragma unroll
        for (int i = 0; i < PER; ++i) {
          if (ab < (uint32_t)top_k && ab + cnt[i] >= (uint32_t)top_k) {
            s.bin = tid * PER + i;
            s.left = (uint32_t)top_k - ab;
            s.before = mb;
          }
          ab += cnt[i];
          mb += mass[i];
        }
      }
      __syncthreads();
      const uint32_t bin = s.bin;
      if (shift) fill_sub(bin);
      if (tid < 32) {
        const uint32_t key = mkey - ((bin << shift) + (shift ? lane : 0));
        const uint32_t want = s.left;
        const uint32_t c = shift ? s.sub[lane] : lane == 0 ? want : 0u;
        const uint32_t inc = warp_scan(c);
        const bool here = inc - c < want && inc >= want;
        const uint32_t take = here ? want - (inc - c) : inc < want ? c : 0u;
        const u64 w = warp_sum64(take ? (u64)take * units(key_bits(key), key) : 0ull);
        if (here) {
          s.key = key;
          s.left = take;
          s.before += w;  // the weight of the first top_k
        }
      }
      __syncthreads();
      tau = s.key;
      left = s.left;
      mtotal = s.before;
      __syncthreads();
    }
    if (use_p) {
      // Kept are the ranks with less than `target` before them, and the first.
      const double target = (double)fmaxf(top_p, 0.f) * (double)mtotal;
      u64 mb = mabove;
      if (tid == 0) s.bin = 0xffffffffu;
      __syncthreads();
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        // Of one bin at most: the weight before it is below the target (or it is the maximum's), that with it not.
        if (mass[i] && (mb == 0 || (double)mb < target) && (double)(mb + mass[i]) >= target) {
          s.bin = tid * PER + i;
          s.before = mb;
        }
        mb += mass[i];
      }
      __syncthreads();
      const uint32_t bin = s.bin;
      if (bin != 0xffffffffu) {
        if (shift) fill_sub(bin);
        if (tid < 32) {
          const uint32_t key = mkey - ((bin << shift) + (shift ? lane : 0));
          const uint32_t c = shift ? s.sub[lane] : lane == 0 ? s.hist.count[bin] : 0u;
          const u64 w = c ? units(key_bits(key), key) : 0ull;
          const u64 inc = s.before + warp_scan((u64)c * w), exc = inc - (u64)c * w;
          if (w && (exc == 0 || (double)exc < target) && (double)inc >= target) {
            s.key = key;
            s.left = (uint32_t)fmin(fmax(ceil((target - (double)exc) / (double)w), 1.0), (double)c);
          }
        }
        __syncthreads();
        // Never past the top-k threshold.
        if (s.key > tau || (s.key == tau && s.left < left)) {
          tau = s.key;
          left = s.left;
        }
      }
    }
    if (mpkey > tau) {
      tau = mpkey;
      left = 0xffffffffu;
    }
    __syncthreads();  // the histogram's memory becomes the groups'
  }

  // Weights and ties at tau per group of 256 places, which lie in the order (step, lane).
  const bool ties = left != 0xffffffffu;
  u64* gmass = listed ? s.group.mass : s.row.mass;
  uint32_t* gties = listed ? s.group.ties : s.row.ties;
  const int ngroup = (int)((n + 255) / 256);
  for (int g = warp; g < ngroup; g += NW) {
    u64 w = 0;
    uint32_t tie = 0;
#pragma unroll 2
    for (int j = 0; j < 8; ++j) {
      const uint32_t p = g * 256 + j * 32 + lane;
      if (p < n) {
        uint32_t bits;
        const uint32_t key = entry(p, bits);
        if (ties && key == tau)
          ++tie;
        else if (key >= tau)
          w += units(bits, key);
      }
    }
    w = warp_sum64(w);
    tie = __reduce_add_sync(0xffffffffu, tie);
    if (lane == 0) {
      gmass[g] = w;
      gties[g] = tie;
    }
  }
  __syncthreads();
  if (warp != 0) return;

  // One warp: a run of groups per lane. Ties are kept while fewer than `left` stand before them.
  const u64 wtie = ties ? units(key_bits(tau), tau) : 0ull;
  const int per = (ngroup + 31) / 32;
  const int g0 = min(lane * per, ngroup), g1 = min(g0 + per, ngroup);
  uint32_t tsum = 0;
  for (int g = g0; g < g1; ++g) tsum += gties[g];
  uint32_t tb = warp_scan(tsum) - tsum;
  auto kept = [&](uint32_t before, uint32_t c) -> uint32_t { return before >= left ? 0u : min(c, left - before); };
  u64 wsum = (u64)kept(tb, tsum) * wtie;
  for (int g = g0; g < g1; ++g) wsum += gmass[g];
  const u64 winc = warp_scan(wsum);
  const u64 total = __shfl_sync(0xffffffffu, winc, 31);
  // The first place whose running weight exceeds u * total.
  const double ut = (double)a.u[r] * (double)total;
  u64 target = ut > 0.0 ? (u64)ut : 0ull;
  if (target >= total) target = total - 1;
  u64 wb = winc - wsum;
  int g = 0;
  const bool mine = wb <= target && target < winc;
  if (mine) {
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
  uint32_t place = 0, tkeyf = mkey;
  for (int j = 0; j < 8; ++j) {
    const uint32_t p = g * 256 + j * 32 + lane;
    uint32_t bits = 0;
    const uint32_t key = p < n ? entry(p, bits) : 0u;
    const uint32_t tie = __ballot_sync(0xffffffffu, ties && key == tau);
    const uint32_t t_here = tb + __popc(tie & ((1u << lane) - 1u));
    const u64 w = ties && key == tau ? (t_here < left ? wtie : 0ull) : key >= tau ? units(bits, key) : 0ull;
    const u64 inc = wb + warp_scan(w);
    const uint32_t hit = __ballot_sync(0xffffffffu, target < inc);
    if (hit) {
      const int l = __ffs(hit) - 1;
      place = g * 256 + j * 32 + l;
      tkeyf = __shfl_sync(0xffffffffu, key, l);
      break;
    }
    wb = __shfl_sync(0xffffffffu, inc, 31);
    tb += __popc(tie);
  }

  // The element at that place: its segment, then the entry's rank within it.
  int64_t token = place;
  if (listed) {
    int lo = 0, hi = nseg;  // the last segment that begins at or before the place
    while (hi - lo > 1) {
      const int mid = (lo + hi) / 2;
      if (s.seg[mid] <= place)
        lo = mid;
      else
        hi = mid;
    }
    const int64_t first = (int64_t)lo * 256 + lane * 8;
    const uint32_t ge = vec_ge(load_vec(row, first, vocab), limit);
    const uint32_t c = __popc(ge), want = place - s.seg[lo];
    uint32_t before = warp_scan(c) - c;
    uint32_t found = 0;  // index + 1
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (ge & ge_bit(j)) {
        if (before == want) found = (uint32_t)(first + j) + 1;
        ++before;
      }
    token = (int64_t)__reduce_max_sync(0xffffffffu, found) - 1;
  }
  if (lane == 0) {
    a.tokens[r] = token;
    if (a.logp) {
      const double d = tkeyf == mkey ? 0.0 : ((double)__half2float(key_half(tkeyf)) - (double)m32) / (double)T;
      a.logp[r] = (float)(d - log((double)total / kUnit));
    }
  }
}

template <int NT, int VPT, bool kRegs>
int launch_sample(const SampleParams& p, int64_t rows, cudaStream_t s) {
  static std::atomic<uint64_t> done{0};
  JX_CUDA_TRY(once_per_device(done,
                              [] {
                                return cudaFuncSetAttribute(sample_kernel<NT, VPT, kRegs>,
                                                            cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                            (int)sizeof(SampleShared));
                              }),
              "jx_sample: shared memory");
  sample_kernel<NT, VPT, kRegs><<<(unsigned)rows, NT, sizeof(SampleShared), s>>>(p);
  JX_CHECK_LAUNCH("jx_sample");
  return JX_OK;
}

}  // namespace sel
}  // namespace jx

using namespace jx;

extern "C" int jx_top_logits(const void* logits16, int64_t rows, int vocab, int64_t ld, int k, void* values16,
                             int64_t* ids, jx_stream_t stream) {
  JX_CHECK_ARG(rows > 0 && rows <= 0x7fffffff && vocab > 0 && ld >= vocab, "jx_top_logits: bad shape");
  JX_CHECK_ARG(k > 0 && k <= vocab && k <= sel::kMaxTop, "jx_top_logits: k must be in [1, min(vocab, %d)] (got %d)",
               sel::kMaxTop, k);
  JX_CHECK_ARG(logits16 && values16 && ids, "jx_top_logits: NULL argument");
  JX_CHECK_ARG(ld % 8 == 0 && aligned16(logits16), "jx_top_logits: ld%%8 and 16B alignment required");
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  sel::top_logits_kernel<512, 8><<<(unsigned)rows, 512, 0, s>>>(static_cast<const __half*>(logits16), ld, vocab, k,
                                                               static_cast<__half*>(values16), ids);
  JX_CHECK_LAUNCH("jx_top_logits");
  return JX_OK;
}

extern "C" int jx_sample(const void* logits16, int64_t rows, int vocab, int64_t ld, const float* uniforms,
                         const float* temperatures, float temperature, const int32_t* top_ks, int top_k,
                         const float* top_ps, float top_p, const float* min_ps, float min_p, int64_t* tokens,
                         float* logprobs, jx_stream_t stream) {
  JX_CHECK_ARG(logits16 && uniforms && tokens, "jx_sample: NULL argument");
  JX_CHECK_ARG(rows > 0 && rows <= 0x7fffffff && vocab > 0 && vocab <= sel::kSegs * 256 && ld >= vocab,
               "jx_sample: bad shape (rows %lld, vocab %d, at most %d)", (long long)rows, vocab, sel::kSegs * 256);
  JX_CHECK_ARG(ld % 8 == 0 && aligned16(logits16), "jx_sample: ld%%8 and 16B alignment required");
  sel::SampleParams p{static_cast<const __half*>(logits16), ld, vocab, uniforms, temperatures, top_ks, top_ps, min_ps,
                      temperature, top_p, min_p, top_k, tokens, logprobs};
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  // Rows that a block's registers hold are read once, longer ones again by each step.
  if (vocab <= 1024 * 8 * 4) return sel::launch_sample<1024, 4, true>(p, rows, s);
  return sel::launch_sample<1024, 4, false>(p, rows, s);
}
