// Distillation from a teacher's top logits: a row's loss and its logit gradient.
//
// Stands beside the cross-entropy of embed_ce.cu (Midstream-LLM src/jishui/model_torch.py:102-104). A row has
// the student's logits z [vocab], K teacher slots (token id, teacher logit t; id < 0: unused) and a target y:
//   p = softmax(t / tau) over the used slots,  q = softmax(z / tau),  q1 = softmax(z)
//   loss = alpha tau^2 sum_k p_k (log p_k - log q[id_k]) + (1 - alpha) (-log q1[y])
//   d loss / d z_j = alpha tau (q_j - sum_{k: id_k = j} p_k) + (1 - alpha) (q1_j - [j = y])
// A row without a used slot (or with only -inf teacher logits) has no first term; a row whose target is
// ignore_index has neither loss nor gradient.
#include "jx_common.cuh"
#include "jx_host.h"

namespace jx {
namespace kd {

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kMaxSlots = 1024;
constexpr int kSeen = 1024;

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// What a row's softmax at temperature 1 costs the forward next to the one at tau: nothing (kOne: tau = 1, alpha = 1 or given block
// statistics), multiplications or a second exponential (kBoth). Multiplications do at temperatures a / b with a of 2 to 4 and b
// of 1 or 2, where exp(z / tau) and exp(z) are the b-th and the a-th power of exp(z / a), two products each at most: tau = 2, 3,
// 4, and 3 / 2. The exponential unit takes 2000 cycles of an SM for 32000 logits where memory takes 2700,
// so a second one would set the time (loss of 16384 x 32000: kBoth 270 us, kPow2 187 us, kPow1h 194 us, kOne 175 us; the
// logits' read alone is 160 us at the copy rate).
enum Mode : int { kOne = 0, kBoth = 1, kPow2 = 2, kPow3 = 3, kPow4 = 4, kPow1h = 5 };

inline Mode mode_of(float tau, bool two) {
  if (!two) return kOne;
  return tau == 2.f ? kPow2 : tau == 3.f ? kPow3 : tau == 4.f ? kPow4 : tau == 1.5f ? kPow1h : kBoth;
}

template <int MODE>
__device__ __forceinline__ float power(float w) {
  const float w2 = w * w;
  return MODE == kPow2 ? w2 : MODE == kPow3 || MODE == kPow1h ? w2 * w : w2 * w2;
}

struct Params {
  const __half* logits;
  int64_t ld;
  int vocab;
  const int64_t* ids;    // [rows, K]
  const void* teacher;   // [rows, K], f16 or f32
  int teacher_f16;
  int K;
  const int64_t* targets;
  int64_t ignore_index;
  float tau, alpha;
  const float2* parts;   // [rows, nblk] (max, sum exp(z - max)) of 128-column blocks, or NULL
  int nblk;
  float* stats;          // [3, rows]: log-sum-exp of z / tau, of z, of the used t / tau
  int64_t rows;
};

__device__ __forceinline__ float teacher_logit(const Params& p, int64_t i) {
  return p.teacher_f16 ? __half2float(static_cast<const __half*>(p.teacher)[i]) : static_cast<const float*>(p.teacher)[i];
}

// Eight logits from `first` on; past the end of the row they read as `fill`.
__device__ __forceinline__ uint4 load8(const __half* row, int64_t first, int vocab, uint32_t fill) {
  if (first + 8 <= vocab) return *reinterpret_cast<const uint4*>(row + first);
  const unsigned short* s = reinterpret_cast<const unsigned short*>(row);
  uint32_t w[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint32_t lo = first + 2 * j < vocab ? s[first + 2 * j] : fill;
    const uint32_t hi = first + 2 * j + 1 < vocab ? s[first + 2 * j + 1] : fill;
    w[j] = lo | (hi << 16);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// ln(s) with the exponent split off, so that the fp32 logarithm's error is that of a number below 0.35.
__device__ __forceinline__ double log_wide(float s) {
  if (!(s > 1e-30f && s < 1e30f)) return (double)logf(s);
  int e = (__float_as_int(s) >> 23) - 127;
  float m = __int_as_float((__float_as_int(s) & 0x7fffff) | 0x3f800000);
  if (m > 1.41421356f) m *= 0.5f, ++e;
  return e * 0.69314718055994530942 + (double)logf(m);
}

__device__ __forceinline__ double warp_sum_d(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// The row's loss from the log-sum-exp of z / tau and of z, by one warp: slot_t / slot_z hold the teacher's and the
// student's logits of the slots, t = -inf for an unused one.
// The few terms of a row are put together in 64 bits, since the two logarithms of sums nearly cancel where
// student and teacher agree.
__device__ __forceinline__ void finish_row(const Params& p, int64_t row, double lse, double lse1,
                                           const float* slot_t, const float* slot_z, bool bad_id, float zy,
                                           float* row_loss, int* status) {
  const int lane = threadIdx.x & 31;
  float tm = -INFINITY;
  bool nan = false;
  for (int k = lane; k < p.K; k += 32) {
    tm = fmaxf(tm, slot_t[k]);
    nan |= slot_t[k] != slot_t[k];
  }
  tm = warp_max(tm);
  const float c = kLog2e / p.tau;
  float s = 0.f;
  double d = 0.0;
  for (int k = lane; k < p.K; k += 32) {
    const float t = slot_t[k];
    if (t == -INFINITY) continue;  // no weight, whatever the student's logit is
    const float e = t == tm ? 1.f : exp2f((t - tm) * c);
    s += e;
    d += (double)e * ((double)t - (double)slot_z[k]);
  }
  s = warp_sum(s);
  d = warp_sum_d(d);
  nan = __any_sync(0xffffffffu, nan || bad_id);
  if (lane != 0) return;
  const bool used = tm != -INFINITY || nan;
  const double lse_t = used ? (double)tm / p.tau + log_wide(s) : -INFINITY;
  double kl = 0.0;
  if (used) kl = d / s / p.tau + lse - lse_t;
  const int64_t y = p.targets[row];
  float loss;
  if (y < 0 || y >= p.vocab) {
    if (status) atomicExch(status, kStatusCeBadTarget);
    loss = __int_as_float(0x7fc00000);
  } else {
    loss = p.alpha > 0.f ? (float)(p.alpha * ((double)p.tau * p.tau) * kl) : 0.f;
    if (p.alpha < 1.f) loss = (float)((double)loss + (1.0 - p.alpha) * (lse1 - (double)zy));
    if (nan) loss = __int_as_float(0x7fc00000);
  }
  row_loss[row] = loss;
  p.stats[row] = (float)lse;
  p.stats[p.rows + row] = (float)lse1;
  p.stats[2 * p.rows + row] = nan ? __int_as_float(0x7fc00000) : (float)lse_t;
}

// A row's slots into shared memory; true if an id is past the vocabulary.
template <int NT>
__device__ __forceinline__ bool load_slots(const Params& p, int64_t row, const __half* z, float* slot_t, float* slot_z,
                                           int* slot_id, int tid, int* status) {
  bool bad = false;
  for (int k = tid; k < p.K; k += NT) {
    const int64_t i = row * p.K + k, id = p.ids[i];
    const bool ok = id >= 0 && id < p.vocab;
    if (id >= p.vocab) {
      bad = true;
      if (status) atomicExch(status, kStatusDistillBadId);
    }
    const float t = ok ? teacher_logit(p, i) : -INFINITY;
    slot_t[k] = t;
    slot_z[k] = ok ? __half2float(z[id]) : 0.f;
    if (slot_id) slot_id[k] = ok ? (int)id : -1;
  }
  return bad;
}

// A row that counts for nothing: nothing else of it is read. One thread.
__device__ __forceinline__ void skip_row(const Params& p, int64_t row, float* row_loss) {
  row_loss[row] = 0.f;
  p.stats[row] = p.stats[p.rows + row] = p.stats[2 * p.rows + row] = 0.f;
}

// Merges a row's block statistics (max, sum) by one warp; every lane gets log sum exp(z).
__device__ __forceinline__ double parts_lse(const float2* parts, int nblk, float* gmax) {
  float m = -INFINITY, s = 0.f;
  for (int b = threadIdx.x & 31; b < nblk; b += 32) {
    const float2 q = parts[b];
    if (q.y == 0.f) continue;
    const float nm = fmaxf(m, q.x);
    s = (m == -INFINITY ? 0.f : s * ex2((m - nm) * kLog2e)) + q.y * ex2((q.x - nm) * kLog2e);
    m = nm;
  }
  const float gm = warp_max(m);
  if (m != -INFINITY) s *= ex2((m - gm) * kLog2e);
  *gmax = gm;
  return (double)gm + log_wide(warp_sum(s));
}

// Temperature 1 with the head's block statistics: the logits are read at the slots and the target only. One
// warp per row. (16384 x 32000, K 64: 44 us; its 77 MB of statistics, ids, logits and gathered sectors are 12 us at the copy
// rate, so latency sets it: a warp's loads of a row follow one another, logits at the slots after their ids.)
constexpr int kPartWarps = 4;

__global__ void __launch_bounds__(kPartWarps * 32) distill_parts_kernel(const Params p, float* __restrict__ row_loss,
                                                                        int* status) {
  extern __shared__ float slots[];  // [warps][2][K]
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t row = (int64_t)blockIdx.x * kPartWarps + warp;
  if (row >= p.rows) return;
  const int64_t y = p.targets[row];
  if (y == p.ignore_index) {
    if (lane == 0) skip_row(p, row, row_loss);
    return;
  }
  float* st = slots + warp * 2 * p.K;
  const __half* z = p.logits + row * p.ld;
  const bool bad = load_slots<32>(p, row, z, st, st + p.K, nullptr, lane, status);
  const float zy = y >= 0 && y < p.vocab ? __half2float(z[y]) : 0.f;
  float gm;
  const double lse = parts_lse(p.parts + row * p.nblk, p.nblk, &gm);
  __syncwarp();
  finish_row(p, row, lse, lse, st, st + p.K, bad, zy, row_loss, status);
}

// One block per row, one pass over the logits: each thread keeps a running maximum of what it has read and the
// sums against it. Small blocks, so that the few warps of a row's end (a chain of about a thousand cycles over the
// slots) are covered by the other rows on the SM; rows of few-row calls are spread over more threads.
template <int NT, int VPT, int MODE>
__global__ void __launch_bounds__(NT, 1024 / NT) distill_fwd_kernel(const Params p, float* __restrict__ row_loss,
                                                                    int* status) {
  constexpr bool kTwo = MODE != kOne;
  extern __shared__ float slots[];  // [2][K]
  __shared__ float rm[NT / 32], rs[NT / 32], rs1[NT / 32];
  __shared__ double rlse1;
  __shared__ int rbad;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int64_t row = blockIdx.x;
  const __half* z = p.logits + row * p.ld;
  const int nvec = (p.vocab + 7) / 8;
  const float c = kLog2e / p.tau;
  const int64_t y = p.targets[row];
  if (y == p.ignore_index) {
    if (tid == 0) skip_row(p, row, row_loss);
    return;
  }
  if (tid == 0) rbad = 0;
  // Exponents are x ce - m ce in one rounding, but m ce has been rounded before: fix and fix1 make up for that in the sums (at
  // m ce = 1e4 it is 5e-4 of them).
  float m = -INFINITY, s = 0.f, s1 = 0.f, fix = 1.f, fix1 = 1.f;
  const float ce = MODE == kPow1h ? kLog2e / 3.f : c;  // of the exponential that is taken
  for (int base = 0; base < nvec; base += NT * VPT) {
    uint4 v[VPT];
#pragma unroll
    for (int i = 0; i < VPT; ++i) v[i] = load8(z, 8 * (int64_t)(base + i * NT + tid), p.vocab, 0xfc00u);
    __half2 hm = __half2half2(__ushort_as_half(0xfc00u));
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const __half2* h = reinterpret_cast<const __half2*>(&v[i]);
      hm = __hmax2(hm, __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3])));
    }
    const float nm = fmaxf(m, fmaxf(__low2float(hm), __high2float(hm)));
    if (nm == -INFINITY) {  // nothing but -inf, or NaN
#pragma unroll
      for (int i = 0; i < VPT; ++i) {
        const __half2* h = reinterpret_cast<const __half2*>(&v[i]);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float2 f = __half22float2(h[j]);
          if (f.x != f.x || f.y != f.y) s = s1 = __int_as_float(0x7fc00000);
        }
      }
      continue;
    }
    if (nm > m) {
      if (m != -INFINITY) {
        s *= ex2((m - nm) * c);
        s1 *= ex2((m - nm) * kLog2e);
      }
      m = nm;
      const float w = ex2(-fmaf(m, ce, -m * ce));
      fix = MODE == kPow1h ? w * w : w;
      if constexpr (MODE == kBoth)
        fix1 = ex2(-fmaf(m, kLog2e, -m * kLog2e));
      else if constexpr (kTwo)
        fix1 = power<MODE>(w);
    }
    const float mc = -m * ce, mc1 = -m * kLog2e;
    float a[4] = {0.f, 0.f, 0.f, 0.f}, b[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const __half2* h = reinterpret_cast<const __half2*>(&v[i]);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 f = __half22float2(h[j]);
        const float w0 = ex2(fmaf(f.x, ce, mc)), w1 = ex2(fmaf(f.y, ce, mc));
        a[j] += MODE == kPow1h ? fmaf(w0, w0, w1 * w1) : w0 + w1;
        if constexpr (MODE == kBoth)
          b[j] += ex2(fmaf(f.x, kLog2e, mc1)) + ex2(fmaf(f.y, kLog2e, mc1));
        else if constexpr (kTwo)
          b[j] += power<MODE>(w0) + power<MODE>(w1);
      }
    }
    s = fmaf((a[0] + a[1]) + (a[2] + a[3]), fix, s);
    if constexpr (kTwo) s1 = fmaf((b[0] + b[1]) + (b[2] + b[3]), fix1, s1);
  }
  const float wm = warp_max(m);
  if (m != -INFINITY) {
    s *= ex2((m - wm) * c);
    s1 *= ex2((m - wm) * kLog2e);
  }
  s = warp_sum(s);
  if constexpr (kTwo) s1 = warp_sum(s1);
  if (lane == 0) {
    rm[warp] = wm;
    rs[warp] = s;
    rs1[warp] = s1;
  }
  const bool bad = load_slots<NT>(p, row, z, slots, slots + p.K, nullptr, tid, status);
  if (p.parts && warp == NT / 32 - 1) {
    float pm;
    const double l = parts_lse(p.parts + row * p.nblk, p.nblk, &pm);
    if (lane == 0) rlse1 = l;
  }
  __syncthreads();
  if (bad) rbad = 1;
  __syncthreads();
  if (warp != 0) return;
  m = lane < NT / 32 ? rm[lane] : -INFINITY;
  s = lane < NT / 32 ? rs[lane] : 0.f;
  s1 = lane < NT / 32 ? rs1[lane] : 0.f;
  const float gm = warp_max(m);
  if (m != -INFINITY) {
    s *= ex2((m - gm) * c);
    s1 *= ex2((m - gm) * kLog2e);
  }
  s = warp_sum(s);
  s1 = warp_sum(s1);
  const double lse = (double)gm / p.tau + log_wide(s);
  const double lse1 = kTwo ? (double)gm + log_wide(s1) : p.parts ? rlse1 : lse;
  const float zy = y >= 0 && y < p.vocab ? __half2float(z[y]) : 0.f;
  finish_row(p, row, lse, lse1, slots, slots + p.K, rbad != 0, zy, row_loss, status);
}

// The maximum and the logarithms (base 2) of the sums of 2^((z - max) c) and (kTwo) 2^((z - max) log2 e) of a row, by a block.
struct RowSums {
  float m, l, l1;
};

template <int NT, bool kTwo>
__device__ __noinline__ RowSums row_sums(const __half* z, int vocab, float c) {
  __shared__ float red[3][NT / 32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nvec = (vocab + 7) / 8;
  float m = -INFINITY;
#pragma unroll 4
  for (int i = threadIdx.x; i < nvec; i += NT) {
    const uint4 v = load8(z, 8 * (int64_t)i, vocab, 0xfc00u);
    const __half2* h = reinterpret_cast<const __half2*>(&v);
    const __half2 hm = __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
    m = fmaxf(m, fmaxf(__low2float(hm), __high2float(hm)));
  }
  m = warp_max(m);
  if (lane == 0) red[0][warp] = m;
  __syncthreads();
  m = warp_max(lane < NT / 32 ? red[0][lane] : -INFINITY);
  float s = 0.f, s1 = 0.f;
#pragma unroll 4
  for (int i = threadIdx.x; i < nvec; i += NT) {
    const uint4 v = load8(z, 8 * (int64_t)i, vocab, 0xfc00u);
    const __half2* h = reinterpret_cast<const __half2*>(&v);
    float a = 0.f, b = 0.f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 f = __half22float2(h[j]);
      a += ex2((f.x - m) * c) + ex2((f.y - m) * c);
      if constexpr (kTwo) b += ex2((f.x - m) * kLog2e) + ex2((f.y - m) * kLog2e);
    }
    s += a, s1 += b;
  }
  s = warp_sum(s), s1 = warp_sum(s1);
  if (lane == 0) red[1][warp] = s, red[2][warp] = s1;
  __syncthreads();
  s = warp_sum(lane < NT / 32 ? red[1][lane] : 0.f);
  s1 = warp_sum(lane < NT / 32 ? red[2][lane] : 0.f);
  return {m, log2f(s), log2f(s1)};
}

// The same of a row's K teacher logits at 2^((t - max) c), by every warp for itself.
__device__ __noinline__ float2 slot_sums(const float* t, int K, float c) {
  const int lane = threadIdx.x & 31;
  float m = -INFINITY, s = 0.f;
  for (int k = lane; k < K; k += 32) m = fmaxf(m, t[k]);
  m = warp_max(m);
  for (int k = lane; k < K; k += 32) s += ex2((t[k] - m) * c);
  return make_float2(m, log2f(warp_sum(s)));
}

// Whether a log-sum-exp is so large that its rounding to fp32 shows in a weight: at 64 half a step is 2e-6 of the weight.
__device__ __forceinline__ bool far_off(float lse) { return fabsf(lse) > 64.f && fabsf(lse) < INFINITY; }

// The gradient. One block per row; the slots' logits are read before anything is stored (out may be the logits).
// Every element gets the dense part, then the slots' elements and the target's are stored once more with
// their own terms, each by the first slot that names it, so that each is rounded once.
// (Its time is that of its reads and writes, 343 us for 16384 x 32000, with one exponential or two.)
// A row whose logits are large (against the temperature) has its sums taken again from its logits, relative to their
// maximum, which its statistics in fp32 cannot hold to enough places (a weight would be off by 1.5e-5 at temperature 0.1,
// by 3e-3 at 0.001). That reads the row twice more: loss and gradient of 16384 x 32000 at temperature 0.1 600 -> 970 us.
template <int NT, int VPT, bool kTwo>
__global__ void __launch_bounds__(NT, 1024 / NT) distill_bwd_kernel(const Params p, const float* __restrict__ grad_loss,
                                                                    const float* __restrict__ count, __half* out,
                                                                    int64_t ld_out) {
  extern __shared__ float slots[];  // t, z, then ids: [3][K + 1]
  __shared__ uint32_t seen[kSeen];  // a bit per id (modulo 32 kSeen): tells whether two slots may name the same
  __shared__ int repeated;
  const int tid = threadIdx.x;
  const int64_t row = blockIdx.x;
  const __half* z = p.logits + row * p.ld;
  __half* o = out + row * ld_out;
  const int nvec = (p.vocab + 7) / 8;
  const int64_t y = p.targets[row];
  const float cnt = *count;
  const bool live = y != p.ignore_index && y >= 0 && y < p.vocab && cnt > 0.f;
  if (!live) {
    for (int i = tid; i < nvec; i += NT) {
      if (8 * i + 8 <= p.vocab)
        *reinterpret_cast<uint4*>(o + 8 * (int64_t)i) = make_uint4(0, 0, 0, 0);
      else
        for (int j = 8 * i; j < p.vocab; ++j) o[j] = __ushort_as_half(0);
    }
    return;
  }
  const float g = *grad_loss / cnt;
  const float lse = p.stats[row], lse1 = p.stats[p.rows + row], lse_t = p.stats[2 * p.rows + row];
  const float ga = lse_t == -INFINITY ? 0.f : g * p.alpha * p.tau, gb = g * (1.f - p.alpha);
  const int K = p.K;
  float* delta = slots;            // what a slot adds to its element's gradient
  float* slot_z = slots + K + 1;
  int* slot_id = reinterpret_cast<int*>(slots + 2 * (K + 1));
  for (int i = tid; i < kSeen; i += NT) seen[i] = 0;
  load_slots<NT>(p, row, z, delta, slot_z, slot_id, tid, nullptr);
  // Slot K: the target.
  if (tid == 0) {
    repeated = 0;
    slot_id[K] = (int)y;
    slot_z[K] = __half2float(z[y]);
    delta[K] = -gb;
  }
  const float c = kLog2e / p.tau;
  const bool far = far_off(lse) || far_off(lse1) || far_off(lse_t);
  float m = 0.f, b = -lse * kLog2e, b1 = -lse1 * kLog2e;  // exponents (x - m) c + b and (x - m) log2 e + b1
  if (far) {
    const RowSums r = row_sums<NT, kTwo>(z, p.vocab, c);
    m = r.m, b = -r.l, b1 = -r.l1;
  }
  auto both = [](float x) { return make_float2(x, x); };
  auto dense = [&](float2 x) {
    x = __fadd2_rn(x, both(-m));
    const float2 e = __ffma2_rn(x, both(c), both(b));
    const float2 w = make_float2(ex2(e.x), ex2(e.y));
    if constexpr (kTwo) {
      const float2 e1 = __ffma2_rn(x, both(kLog2e), both(b1));
      return __ffma2_rn(both(gb), make_float2(ex2(e1.x), ex2(e1.y)), __fmul2_rn(both(ga), w));
    }
    return __fmul2_rn(both(ga + gb), w);  // tau = 1, or gb = 0
  };
  for (int base = 0; base < nvec; base += NT * VPT) {
    uint4 v[VPT];
#pragma unroll
    for (int i = 0; i < VPT; ++i) v[i] = load8(z, 8 * (int64_t)(base + i * NT + tid), p.vocab, 0xfc00u);
    if (base == 0) {
      __syncthreads();  // every slot's logit has been read
      float2 ts = make_float2(0.f, 0.f);
      if (far) {
        ts = slot_sums(delta, K, c);
        __syncthreads();
      }
      for (int k = tid; k < K; k += NT) {
        const float t = delta[k];
        const float e = far && fabsf(lse_t) < INFINITY ? fmaf(t - ts.x, c, -ts.y) : (t / p.tau - lse_t) * kLog2e;
        delta[k] = t == -INFINITY ? 0.f : -ga * exp2f(e);
      }
      for (int k = tid; k <= K; k += NT) {
        const int id = slot_id[k];
        if (id >= 0 && (atomicOr(&seen[(id >> 5) % kSeen], 1u << (id & 31)) >> (id & 31) & 1u)) repeated = 1;
      }
    }
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int64_t first = 8 * (int64_t)(base + i * NT + tid);
      if (first >= p.vocab) continue;
      __half2* h = reinterpret_cast<__half2*>(&v[i]);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        h[j] = __float22half2_rn(dense(__half22float2(h[j])));
      }
      if (first + 8 <= p.vocab) {
        *reinterpret_cast<uint4*>(o + first) = v[i];
      } else {
        const __half* e = reinterpret_cast<const __half*>(&v[i]);
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (first + j < p.vocab) o[first + j] = e[j];
      }
    }
  }
  __syncthreads();
  for (int k = tid; k <= K; k += NT) {
    const int id = slot_id[k];
    if (id < 0) continue;
    float d = delta[k];
    bool mine = true;
    if (repeated) {
      d = 0.f;
      for (int j = 0; j <= K; ++j) {
        if (slot_id[j] != id) continue;
        if (j < k) {
          mine = false;
          break;
        }
        d += delta[j];
      }
    }
    if (mine) o[id] = __float2half_rn(dense(both(slot_z[k])).x + d);
  }
}

}  // namespace kd
}  // namespace jx

using namespace jx;

namespace {

int check(const kd::Params& p, const char* name) {
  JX_CHECK_ARG(p.rows > 0 && p.rows <= 0x7fffffff && p.vocab > 0 && p.ld >= p.vocab, "%s: bad shape", name);
  JX_CHECK_ARG(p.ld % 8 == 0 && aligned16(p.logits), "%s: ld%%8 and 16B alignment required", name);
  JX_CHECK_ARG(p.K > 0 && p.K <= kd::kMaxSlots, "%s: 1 to %d teacher slots (got %d)", name, kd::kMaxSlots, p.K);
  JX_CHECK_ARG(p.logits && p.ids && p.teacher && p.targets && p.stats, "%s: NULL argument", name);
  JX_CHECK_ARG(p.tau >= 1e-3f && p.tau <= 1e3f, "%s: temperature must be in [0.001, 1000]", name);
  JX_CHECK_ARG(p.alpha >= 0.f && p.alpha <= 1.f, "%s: alpha must be in [0, 1]", name);
  return JX_OK;
}

// Threads of a row's block: 128, or 512 where rows are few and long enough for them. Loss and gradient of rows of 32000
// with 128 / 512 threads: 64 rows 17.1 / 12.4 us, 300 rows 20.0 / 19.6, 600 rows 29.7 / 33.7, 4000 rows 146 / 191.
bool wide_block(int64_t rows, int vocab) { return rows < 2 * num_sms() && vocab > 8192; }

template <int NT>
void launch_fwd(const kd::Params& p, kd::Mode mode, float* row_loss, cudaStream_t s) {
  const unsigned grid = (unsigned)p.rows;
  const size_t smem = 2 * p.K * sizeof(float);
  int* status = status_ptr();
  switch (mode) {
    case kd::kOne: kd::distill_fwd_kernel<NT, 8, kd::kOne><<<grid, NT, smem, s>>>(p, row_loss, status); break;
    case kd::kBoth: kd::distill_fwd_kernel<NT, 8, kd::kBoth><<<grid, NT, smem, s>>>(p, row_loss, status); break;
    case kd::kPow2: kd::distill_fwd_kernel<NT, 8, kd::kPow2><<<grid, NT, smem, s>>>(p, row_loss, status); break;
    case kd::kPow3: kd::distill_fwd_kernel<NT, 8, kd::kPow3><<<grid, NT, smem, s>>>(p, row_loss, status); break;
    case kd::kPow4: kd::distill_fwd_kernel<NT, 8, kd::kPow4><<<grid, NT, smem, s>>>(p, row_loss, status); break;
    case kd::kPow1h: kd::distill_fwd_kernel<NT, 8, kd::kPow1h><<<grid, NT, smem, s>>>(p, row_loss, status); break;
  }
}

template <int NT>
void launch_bwd(const kd::Params& p, bool two, const float* grad_loss, const float* count, __half* out, int64_t ld_out,
                cudaStream_t s) {
  const unsigned grid = (unsigned)p.rows;
  const size_t smem = 3 * (p.K + 1) * sizeof(float);
  if (two)
    kd::distill_bwd_kernel<NT, 8, true><<<grid, NT, smem, s>>>(p, grad_loss, count, out, ld_out);
  else
    kd::distill_bwd_kernel<NT, 8, false><<<grid, NT, smem, s>>>(p, grad_loss, count, out, ld_out);
}

}  // namespace

extern "C" int jx_distill_fwd(const void* logits16, int64_t rows, int vocab, int64_t ld, const int64_t* teacher_ids,
                              const void* teacher_logits, int teacher_is_f16, int K, const int64_t* targets,
                              int64_t ignore_index, float temperature, float alpha, const void* parts, float* stats,
                              float* row_loss, jx_stream_t stream) {
  kd::Params p{static_cast<const __half*>(logits16), ld, vocab, teacher_ids, teacher_logits, teacher_is_f16, K, targets,
               ignore_index, temperature, alpha, static_cast<const float2*>(parts), (vocab + 127) / 128, stats, rows};
  const int rc = check(p, "jx_distill_fwd");
  if (rc != JX_OK) return rc;
  JX_CHECK_ARG(row_loss && ((uintptr_t)parts & 7) == 0, "jx_distill_fwd: bad argument");
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (parts && temperature == 1.f) {
    kd::distill_parts_kernel<<<(unsigned)((rows + kd::kPartWarps - 1) / kd::kPartWarps), kd::kPartWarps * 32,
                               kd::kPartWarps * 2 * K * sizeof(float), s>>>(p, row_loss, status_ptr());
    JX_CHECK_LAUNCH("jx_distill_fwd");
    return JX_OK;
  }
  const bool two = alpha < 1.f && temperature != 1.f && !parts;
  if (wide_block(rows, vocab))
    launch_fwd<512>(p, kd::mode_of(temperature, two), row_loss, s);
  else
    launch_fwd<128>(p, kd::mode_of(temperature, two), row_loss, s);
  JX_CHECK_LAUNCH("jx_distill_fwd");
  return JX_OK;
}

extern "C" int jx_distill_bwd(const void* logits16, int64_t rows, int vocab, int64_t ld, const int64_t* teacher_ids,
                              const void* teacher_logits, int teacher_is_f16, int K, const int64_t* targets,
                              int64_t ignore_index, float temperature, float alpha, const float* stats,
                              const float* grad_loss, const float* count, void* out16, int64_t ld_out,
                              jx_stream_t stream) {
  kd::Params p{static_cast<const __half*>(logits16), ld, vocab, teacher_ids, teacher_logits, teacher_is_f16, K, targets,
               ignore_index, temperature, alpha, nullptr, 0, const_cast<float*>(stats), rows};
  const int rc = check(p, "jx_distill_bwd");
  if (rc != JX_OK) return rc;
  JX_CHECK_ARG(grad_loss && count && out16, "jx_distill_bwd: NULL argument");
  JX_CHECK_ARG(ld_out % 8 == 0 && ld_out >= vocab && aligned16(out16), "jx_distill_bwd: ld_out%%8 and 16B alignment required");
  JX_CHECK_ARG(out16 != logits16 || ld_out == ld, "jx_distill_bwd: in place, the row strides must be the same");
  const bool two = alpha < 1.f && temperature != 1.f;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  __half* out = static_cast<__half*>(out16);
  if (wide_block(rows, vocab))
    launch_bwd<512>(p, two, grad_loss, count, out, ld_out, s);
  else
    launch_bwd<128>(p, two, grad_loss, count, out, ld_out, s);
  JX_CHECK_LAUNCH("jx_distill_bwd");
  return JX_OK;
}
