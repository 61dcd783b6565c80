// Single-token attention of a batch whose sequences share a long prefix (head_dim 64).
//
// Every sequence's new query attends to the P keys of one shared prefix and to its own keys (of which the last
// is the new token's, appended here). The reference has no counterpart: it re-runs each whole context
// (Midstream-LLM src/jishui/generate_torch.py:279-285); decode_attn.cu is the form for caches that share nothing.
//
// With G query heads per key / value head, the queries of all sequences at one key / value head are rows of one
// matrix, so the prefix is read once for up to 64 rows and its scores are matrix products. They are formed
// transposed, with the keys along the matrix unit's 128 rows: then a thread owns one key, and the softmax's work is
// in proportion to the query rows and spread over all four warps however few they are. For every 128 keys
//   S^T = K Q^T        (tcgen05, M 128 keys, N 16-64 rows, K 64, both from shared memory)          -> TMEM
//   P   = exp2(S scale - m) as two fp16 numbers, against a reference m per row                     -> shared memory
//   [O^T; l] += [V^T; 1] P  (tcgen05, M 128 = 64 head columns and the sum's row, N twice the rows, K 128 keys) -> TMEM
// m lies 7 (log2 units) below the row's maximum over the first tile and is raised only when a later P passes 2^15 (a rare
// step that rescales O^T), so no other tile needs a maximum across threads. The sum l comes out of the same product
// from the same P, by a block of ones behind V^T.
//
// A probability is held in 22 bits at least, as what fp16 leaves of it is an fp16 number of its own: the rest's columns stand
// behind P's, so the same product takes both, and their results are added where a part is written. P in fp16 alone
// would leave 2^-12 of each: 2.9e-4 of the output's norm from the exact one, instead of 2.1e-4, which its own rounding to fp16
// makes. It costs conversions and stores in the softmax warps: 59.1 -> 62.8 us for 64 sequences behind 32749 keys,
// 42.9 -> 47.6 us for 96 of 32 heads on 8 key heads, less than 2 % for 16 rows and fewer.
//
// A sequence's own keys belong to no other, so a product has only its G heads as rows, and an item as short as a few
// keys still pays the whole chain from TMA to the output (about 3 us). With up to four heads a key head they are
// therefore scored by the second kernel, which joins the parts anyway, in plain fp32 arithmetic (one block per
// sequence and key / value head, many blocks an SM; 64 sequences of 16 heads with a prefix of 128 and one token of their
// own: 21.5 -> 14.3 us when this came in). Larger groups, and few sequences with long own parts, which have to be
// split, take the matrix way.
//
// Work of the first kernel: the prefix tiles of all (row tile, key / value head) units stand in one line that is cut
// into equal runs, one a block, so that each unit is split over a few blocks; the (sequence, head, chunk) items of
// own keys, where it has them, follow, dealt round robin. Each part leaves (m, l, o[64]) of its rows in the
// workspace, the second kernel joins them. The schedule is fixed by the sizes, so results repeat bit for bit.
//
// 224 threads, two blocks an SM (256 TMEM columns each):
//   warp 0    TMA producer: Q of the item, K and V tiles (2 slots of 16 KB each),
//   warp 1    issues the first products; into the tile that holds a sequence's end it first puts the new key (and into the
//             cache),
//   warps 2-5 softmax, one key per thread, and the parts' output,
//   warp 6    issues the second products, and puts the new value into such a tile and clears what is behind it, since
//             0 * garbage may be NaN. It alone touches V's slots: it waits for every fill of theirs in turn, so no wait
//             can take an earlier fill for its own (with one warp for both products, its twelve products a tile, their waits and
//             commits follow each other: 36.4 against 35.4 us at 64 rows of 32749 keys, 29.4 against 27.6 at one, with P in
//             one fp16 number).
// 64 sequences of 16 heads on a prefix of 32749, 1 to 1000 own tokens: 63 us, 4.2 TB/s. The prefix's tiles are bound by
// the chain scores - exponents - exponentials - product of a tile, not by memory: with one own token each 43.8 us, of which
// about 4 are the join, for 4096 tiles in 296 blocks: 2.9 us a tile in a block, 1.4 us a tile and SM, as two blocks share one.
#include <algorithm>
#include <atomic>
#include <type_traits>

#include "jx_common.cuh"
#include "jx_host.h"

namespace jx {
namespace pfx {

constexpr int D = 64;
constexpr int BKV = 128;
constexpr int kRows = 64;  // query rows of a tile at most
constexpr int kThreads = 224;
constexpr uint32_t kTile = BKV * D * 2;   // 16 KiB
constexpr uint32_t kQTile = kRows * D * 2;  // 8 KiB
constexpr uint32_t kOnes = 2048;          // 16 keys x 64 ones
constexpr int kKSlots = 2, kVSlots = 2;
constexpr int kLens = 512;  // lengths kept in shared memory
constexpr uint32_t kTmemCols = 256;  // S^T [0,64) and [64,128), [O^T; l] and that of P's rest [128,256)

// A row's reference is its maximum less kLift (log2 units) and may be passed by kLift + 8, so P is 2^7 at the maximum and at
// most 2^15, and what fp16 has below 1 goes to the keys far under the maximum. The rest of P, at most 2^-11 of it, is
// held kRest times as large.
constexpr float kLift = 7.f;
constexpr float kRest = 2048.f;
// Where the rest's columns stand behind P's, by the rows of an item.
__host__ __device__ constexpr int rest_at(int rows) { return rows <= 16 ? 16 : rows <= 32 ? 32 : 64; }
constexpr float kNoKey = -1e30f;  // the running maximum before the first key: below every product of fp16 numbers, and
                                 // a score of -infinity less it is no NaN

enum Status : int { kProducer = 601, kMma = 602, kSoftmax = 603 };

struct Sched {
  int B, G, Hkv, H;
  int nb;              // sequences per row tile
  int P, NT;           // prefix keys and tiles of one unit
  int T, gp;           // prefix tiles in all, and blocks that share them:
  int per, more;       // `per` each, one more for the first `more` blocks
  int max_len, OC;     // own keys: upper bound, tiles per item
  int chunks;          // items of one (sequence, key / value head)
  int step_b, step_h;  // (sequence, head) distance of a block's consecutive items: grid = step_b Hkv + step_h
  bool plain;          // own keys are left to the second kernel (chunks is 0)
  int nparts;          // parts a row has room for
  int nsp;             // of those, for the prefix

  // Block that has prefix tile x.
  __device__ int block_of(int x) const {
    const int big = more * (per + 1);
    return x < big ? x / (per + 1) : more + (x - big) / per;
  }
};

__device__ __forceinline__ int own_length(const Sched& s, int raw) { return raw > 0 && raw <= s.max_len ? raw : 0; }

// The tiles of one block in order. Every role walks its own copy.
struct Cursor {
  int t, t1;    // prefix tiles left
  int ob, oh, oc;  // sequence, head and chunk of the next item of own keys
  int b, h;     // first sequence of the row tile, or the sequence; key / value head
  int key0, n, j, limit;  // first key, tiles, current tile, end of the keys
  int part, ipre, iown;   // part index; prefix / own items begun before
  bool is_own;

  __device__ __forceinline__ void init(const Sched& s) {
    const int c = blockIdx.x;
    t = t1 = 0;
    if (c < s.gp) {
      t = c * s.per + min(c, s.more);
      t1 = t + s.per + (c < s.more ? 1 : 0);
    }
    const int own = gridDim.x - 1 - c;  // dealt from the last block on: those may have no prefix tiles
    ob = own / s.Hkv;
    oh = own - ob * s.Hkv;
    oc = ob / s.B;
    ob -= oc * s.B;
    ipre = iown = -1;
    n = j = 0;
  }
  // The next tile; false at the end.
  __device__ __forceinline__ bool advance(const Sched& s, const int* lens) {
    if (++j < n) return true;
    j = 0;
    if (t < t1) {
      const int unit = t / s.NT, first = t - unit * s.NT;
      h = unit % s.Hkv;
      b = unit / s.Hkv * s.nb;
      n = min(s.NT - first, t1 - t);
      key0 = first * BKV;
      limit = s.P;
      part = (int)blockIdx.x - s.block_of(unit * s.NT);
      is_own = false;
      ++ipre;
      t += n;
      return true;
    }
    while (oc < s.chunks) {
      b = ob, h = oh;
      const int chunk = oc;
      oh += s.step_h;
      ob += s.step_b;
      if (oh >= s.Hkv) oh -= s.Hkv, ++ob;
      while (ob >= s.B) ob -= s.B, ++oc;
      limit = own_length(s, lens[b]);
      key0 = chunk * s.OC * BKV;
      if (key0 >= limit) continue;
      n = min(s.OC, (limit - key0 + BKV - 1) / BKV);
      part = s.nsp + chunk;
      is_own = true;
      ++iown;
      return true;
    }
    return false;
  }
  __device__ __forceinline__ int rows(const Sched& s) const { return is_own ? s.G : min(s.nb, s.B - b) * s.G; }
  __device__ __forceinline__ int key() const { return key0 + j * BKV; }
  __device__ __forceinline__ bool ends() const { return is_own && key() + BKV >= limit; }
};

struct Bars {
  uint64_t k_full[kKSlots], k_empty[kKSlots], v_full[kVSlots], v_empty[kVSlots];
  uint64_t q_full[3], q_empty[3];  // own items alternate between 0 and 1, prefix items use 2
  uint64_t s_full[2], s_free[2], p_full, p_empty;
  uint32_t tmem_base;
  int abort;
  alignas(16) float m[kRows];        // minus each row's reference, log2 units; -inf for columns without a row
  alignas(16) float alpha[kRows];    // factor of a raised reference
  alignas(16) float wmax[4][kRows];  // each warp's maxima
  alignas(16) int at[kRows];         // place of each row's part in the workspace
  int lens[kLens];
};

__device__ __forceinline__ bool wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag, int* status, int code) {
  if (mbar_try_wait(bar, parity)) return true;
  const long long start = clock64();
  for (uint32_t i = 0;; ++i) {
    if (mbar_try_wait(bar, parity)) return true;
    if ((i & 255u) == 255u) {
      if (*abort_flag) return false;
      if (clock64() - start > (1ll << 32)) {
        *abort_flag = 1;
        if (status) atomicExch(status, code);
        return false;
      }
    }
  }
}

// Every lane polls.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag, int* status,
                                          int code) {
  return __all_sync(0xffffffffu, wait(bar, parity, abort_flag, status, code));
}

// Barrier of the four softmax warps; true if any thread's flag is set.
__device__ __forceinline__ bool softmax_any(bool flag) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.u32 p, %1, 0;\n\t"
      "barrier.cta.red.or.pred q, 1, 128, p;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(r)
      : "r"((uint32_t)flag)
      : "memory");
  return r != 0;
}

// max(a, b, c) in one instruction (sm_100).
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

__device__ __forceinline__ float redux_max(float v) {
  float r;
  asm("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
  return r;
}

__device__ __forceinline__ void tma_load_3d(void* dst, const CUtensorMap* map, uint64_t* bar, int x, int y, int z) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], "
      "[%2];" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z)
      : "memory");
}

// Until the kernel before this one is done and what it wrote is visible.
__device__ __forceinline__ void prior_kernel_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// 16 bytes to shared memory, of which the first `bytes` are read and the others zero.
__device__ __forceinline__ void cp_async_16(void* dst, const void* src, uint32_t bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

struct Params {
  Sched s;
  const __half* qkv;
  int64_t ld_qkv;
  __half* kcache;
  __half* vcache;
  int64_t ld_cache, batch_stride;
  const int* lens;
  float scale_log2;
  float2* ml;  // [B * H][nparts]
  float* o;    // [B * H][nparts][64]
  __half* out;
  int64_t ld_out;
  uint32_t q_own_bytes, q_own_stride, q_pre_bytes;
};

template <int N>
__device__ __forceinline__ void load_cols(uint32_t addr, uint32_t (&r)[N]) {
  if constexpr (N == 8) {
    tmem_ld8(addr, r);
  } else if constexpr (N == 16) {
    tmem_ld16(addr, r);
  } else {
#pragma unroll
    for (int q = 0; q < N / 32; ++q) tmem_ld32(addr + q * 32, *reinterpret_cast<uint32_t(*)[32]>(&r[q * 32]));
  }
  tmem_ld_wait();
}

// The tiles of one item, by the four softmax warps: thread = key, W columns of which the first `rows` are rows.
// `g` counts tiles over all items. Columns behind the rows hold garbage on all ways and are never looked at; their
// reference is +inf, so that they pass no bound.
template <int W>
__device__ __forceinline__ bool softmax_item(const Params& p, Cursor& c, const int rows, uint32_t& g, Bars* bars, uint8_t* sP,
                                             uint32_t tmem, int* status) {
  volatile int* abort_flag = &bars->abort;
  const Sched& s = p.s;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int quarter = warp & 3;  // TMEM lanes this warp may access
  const int key = quarter * 32 + lane;
  const uint32_t base = tmem + (static_cast<uint32_t>(quarter * 32) << 16);
  uint8_t* prow = sP + key * 128;
  constexpr int R = rest_at(W);
  const float scale = p.scale_log2;
  for (c.j = 0; c.j < c.n; ++c.j, ++g) {
    const int x = g & 1;
    if (!warp_wait(&bars->s_full[x], (g >> 1) & 1, abort_flag, status, kSoftmax)) return false;
    tc_fence_after();
    uint32_t sr[W];
    load_cols(base + x * 64, sr);
    const bool past = c.key() + key >= c.limit;  // a key past the end
    // The scores become exponents against the references; true if one passes the bound.
    auto exponents = [&]() -> bool {
      float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
      constexpr int B = W < 16 ? W : 16;  // columns whose references are read ahead of their use
      const float2 sc = make_float2(scale, scale);
#pragma unroll
      for (int i0 = 0; i0 < W; i0 += B) {
        float4 m[B / 4];
#pragma unroll
        for (int i = 0; i < B / 4; ++i) m[i] = *reinterpret_cast<const float4*>(&bars->m[i0 + 4 * i]);
#pragma unroll
        for (int i = 0; i < B / 4; ++i) {
          uint32_t* r = &sr[i0 + 4 * i];
          const float2 y0 = __ffma2_rn(make_float2(__uint_as_float(r[0]), __uint_as_float(r[1])), sc, make_float2(m[i].x, m[i].y));
          const float2 y1 = __ffma2_rn(make_float2(__uint_as_float(r[2]), __uint_as_float(r[3])), sc, make_float2(m[i].z, m[i].w));
          top[i & 3] = max3(max3(top[i & 3], y0.x, y0.y), y1.x, y1.y);
          r[0] = __float_as_uint(y0.x), r[1] = __float_as_uint(y0.y);
          r[2] = __float_as_uint(y1.x), r[3] = __float_as_uint(y1.y);
        }
      }
      return !past && fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])) > kLift + 8.f;
    };
    bool raise = c.j == 0;
    if (!raise) raise = softmax_any(exponents());
    if (raise) {
      // Maxima over the tile's keys, per warp, then over the warps. A loop, like every part that runs once an item: cold
      // straight code costs more in instruction fetches than it saves.
#pragma unroll 1
      for (int i = 0; i < W; i += 8) {
        uint32_t u[8];
        load_cols(base + x * 64 + i, u);
        float w[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) w[k] = redux_max(past ? -INFINITY : __uint_as_float(u[k]));
        if (lane == 0) {
          *reinterpret_cast<float4*>(&bars->wmax[quarter][i]) = make_float4(w[0], w[1], w[2], w[3]);
          *reinterpret_cast<float4*>(&bars->wmax[quarter][i + 4]) = make_float4(w[4], w[5], w[6], w[7]);
        }
      }
      softmax_any(false);
      const int i = threadIdx.x - 64;
      if (i < W) {
        float mx = INFINITY;
        if (i < rows) {
          mx = fmaxf(fmaxf(bars->wmax[0][i], bars->wmax[1][i]), fmaxf(bars->wmax[2][i], bars->wmax[3][i])) * scale;
          mx = fmaxf(mx - kLift, kNoKey);  // (scores of -infinity alone)
          if (c.j > 0) {
            const float old = -bars->m[i];
            mx = fmaxf(mx, old);
            bars->alpha[i] = ex2(old - mx);
          } else {
            const int sq = i / s.G;
            bars->at[i] = ((c.b + sq) * s.H + c.h * s.G + i - sq * s.G) * s.nparts + c.part;
          }
        }
        bars->m[i] = -mx;
      }
      softmax_any(false);
      load_cols(base + x * 64, sr);
      exponents();
    }
    tc_fence_before();
    __syncwarp();
    if (lane == 0) mbar_arrive(&bars->s_free[x]);  // the scores have been read
    // The product of the tile before must be done before P is overwritten or [O^T; l] rescaled.
    if (g > 0 && !warp_wait(&bars->p_empty, (g - 1) & 1, abort_flag, status, kSoftmax)) return false;
    if (raise && c.j > 0) {
      tc_fence_after();
#pragma unroll 1
      for (int q = 0; q < W; q += 8) {
#pragma unroll
        for (int at = 128; at <= 128 + R; at += R) {
          uint32_t orr[8];
          load_cols(base + at + q, orr);
#pragma unroll
          for (int i = 0; i < 8; ++i) orr[i] = __float_as_uint(__uint_as_float(orr[i]) * bars->alpha[q + i]);
          tmem_st8(base + at + q, orr);
        }
      }
      tmem_st_wait();
      tc_fence_before();
    }
#pragma unroll
    for (int q = 0; q < W / 8; ++q) {
      uint32_t pw[4], pr[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float p0 = ex2(__uint_as_float(sr[q * 8 + 2 * e])), p1 = ex2(__uint_as_float(sr[q * 8 + 2 * e + 1]));
        const __half2 hp = __floats2half2_rn(p0, p1);
        const float2 b = __half22float2(hp);
        const float2 d = __ffma2_rn(b, make_float2(-kRest, -kRest), __fmul2_rn(make_float2(p0, p1), make_float2(kRest, kRest)));
        const __half2 hr = __floats2half2_rn(d.x, d.y);
        pw[e] = past ? 0u : *reinterpret_cast<const uint32_t*>(&hp);
        pr[e] = past ? 0u : *reinterpret_cast<const uint32_t*>(&hr);
      }
      *reinterpret_cast<uint4*>(prow + ((q ^ (key & 7)) << 4)) = make_uint4(pw[0], pw[1], pw[2], pw[3]);
      *reinterpret_cast<uint4*>(prow + R / 64 * kTile + (((R % 64 / 8 + q) ^ (key & 7)) << 4)) =
          make_uint4(pr[0], pr[1], pr[2], pr[3]);
    }
    fence_proxy_async_smem();
    __syncwarp();
    if (lane == 0) mbar_arrive(&bars->p_full);
  }
  // The item's part: columns of [O^T; l] and of the rest's, 64 values from two warps, the sum from the third.
  if (!warp_wait(&bars->p_empty, (g - 1) & 1, abort_flag, status, kSoftmax)) return false;
  tc_fence_after();
  if (quarter < 3) {
#pragma unroll 1
    for (int q = 0; q < rows; q += 8) {
      uint32_t orr[8], rest[8];
      load_cols(base + 128 + q, orr);
      load_cols(base + 128 + R + q, rest);
#pragma unroll
      for (int i = 0; i < 8; ++i)
        orr[i] = __float_as_uint(fmaf(__uint_as_float(rest[i]), 1.f / kRest, __uint_as_float(orr[i])));
      int at[8];
      *reinterpret_cast<int4*>(&at[0]) = *reinterpret_cast<const int4*>(&bars->at[q]);
      *reinterpret_cast<int4*>(&at[4]) = *reinterpret_cast<const int4*>(&bars->at[q + 4]);
      if (quarter < 2) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (q + i < rows) p.o[(int64_t)at[i] * D + key] = __uint_as_float(orr[i]);
      } else {  // every lane has every sum: lane i takes row q + i
        uint32_t l = orr[0];
#pragma unroll
        for (int i = 1; i < 8; ++i) l = lane == i ? orr[i] : l;
        if (lane < 8 && q + lane < rows) p.ml[bars->at[q + lane]] = make_float2(-bars->m[q + lane], __uint_as_float(l));
      }
    }
  }
  // The next item's first product with V waits for this warp's next arrival at p_full, after these reads.
  tc_fence_before();
  c.j = c.n - 1;
  return true;
}

__global__ void __launch_bounds__(kThreads, 2)
    attn_prefix_part_kernel(const __grid_constant__ CUtensorMap tm_qp, const __grid_constant__ CUtensorMap tm_qo,
                            const __grid_constant__ CUtensorMap tm_kp, const __grid_constant__ CUtensorMap tm_vp,
                            const __grid_constant__ CUtensorMap tm_kc, const __grid_constant__ CUtensorMap tm_vc,
                            const Params p, int* status) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  // Queries of own items (two, G rows each), of a prefix item, K and V slots, P and its rest, ones. The matrix unit reads the
  // rows of a query tile in sixteens; behind an own item's G rows it finds other data, which only reaches columns
  // of S^T and O^T that nobody reads.
  uint8_t* sQ = smem;
  uint8_t* sQp = smem + 2 * p.q_own_stride;
  uint8_t* sK = sQp + kQTile;
  uint8_t* sV = sK + kKSlots * kTile;
  uint8_t* sP = sV + kVSlots * kTile;
  uint8_t* s1 = sP + 2 * kTile;
  Bars* bars = reinterpret_cast<Bars*>(s1 + kOnes);
  volatile int* abort_flag = &bars->abort;
  const Sched& s = p.s;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 32) {
    if (s.T > 0) tma_prefetch_desc(&tm_qp), tma_prefetch_desc(&tm_kp), tma_prefetch_desc(&tm_vp);
    if (s.chunks > 0) tma_prefetch_desc(&tm_qo), tma_prefetch_desc(&tm_kc), tma_prefetch_desc(&tm_vc);
  }
  if (threadIdx.x == 0) {
    for (int i = 0; i < kKSlots; ++i) mbar_init(&bars->k_full[i], 1), mbar_init(&bars->k_empty[i], 1);
    for (int i = 0; i < kVSlots; ++i) mbar_init(&bars->v_full[i], 1), mbar_init(&bars->v_empty[i], 1);
    for (int i = 0; i < 3; ++i) mbar_init(&bars->q_full[i], 1), mbar_init(&bars->q_empty[i], 1);
    for (int i = 0; i < 2; ++i) mbar_init(&bars->s_full[i], 1), mbar_init(&bars->s_free[i], 4);
    mbar_init(&bars->p_full, 4);
    mbar_init(&bars->p_empty, 1);
    bars->abort = 0;
    fence_barrier_init();
  }
  if (warp == 1) {
    tmem_alloc(&bars->tmem_base, kTmemCols);
    tmem_relinquish();
  }
  for (int i = threadIdx.x; i < (int)kOnes / 4; i += kThreads) reinterpret_cast<uint32_t*>(s1)[i] = 0x3c003c00u;
  fence_proxy_async_smem();
  prior_kernel_wait();  // what is above may run while the kernel before finishes
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");  // the second kernel's blocks may use what is free
  const bool staged = s.B <= kLens;
  if (staged)
    for (int i = threadIdx.x; i < s.B; i += kThreads) bars->lens[i] = p.lens[i];
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = bars->tmem_base;
  const int* lens = staged ? bars->lens : p.lens;
  Cursor c;
  c.init(s);

  if (warp == 0) {
    if (lane == 0) {
      // K and V take turns as their slots come free: V's are held longer, and K must not wait behind them.
      bool more_k = c.advance(s, lens), more_v = more_k;
      Cursor v = c;
      uint32_t nk = 0, nv = 0, filled = 0;  // filled: bit q, Q slot q was; bit 8 + q, an odd number of times
      long long since = clock64();
      while (more_k || more_v) {
        bool idle = true;
        const uint32_t ks = nk % kKSlots, vs = nv % kVSlots;
        if (more_k && mbar_test_wait(&bars->k_empty[ks], ((nk / kKSlots) & 1) ^ 1)) {
          const int q = c.is_own ? (c.iown & 1) : 2;
          const uint32_t use = c.is_own ? (uint32_t)(c.iown >> 1) : (uint32_t)c.ipre;
          if (c.j > 0 || mbar_test_wait(&bars->q_empty[q], (use & 1) ^ 1)) {
            if (c.j == 0) {
              filled = (filled | 1u << q) ^ 256u << q;
              mbar_expect_tx(&bars->q_full[q], c.is_own ? p.q_own_bytes : p.q_pre_bytes);
              tma_load_3d(q == 2 ? sQp : sQ + q * p.q_own_stride, c.is_own ? &tm_qo : &tm_qp, &bars->q_full[q], 0, c.h * s.G,
                          c.b);
            }
            mbar_expect_tx(&bars->k_full[ks], kTile);
            if (c.is_own)
              tma_load_3d(sK + ks * kTile, &tm_kc, &bars->k_full[ks], c.h * D, c.key(), c.b);
            else
              tma_load_2d(sK + ks * kTile, &tm_kp, &bars->k_full[ks], c.h * D, c.key());
            more_k = c.advance(s, lens);
            ++nk;
            idle = false;
          }
        }
        if (more_v && mbar_test_wait(&bars->v_empty[vs], ((nv / kVSlots) & 1) ^ 1)) {
          mbar_expect_tx(&bars->v_full[vs], kTile);
          if (v.is_own)
            tma_load_3d(sV + vs * kTile, &tm_vc, &bars->v_full[vs], v.h * D, v.key(), v.b);
          else
            tma_load_2d(sV + vs * kTile, &tm_vp, &bars->v_full[vs], v.h * D, v.key());
          more_v = v.advance(s, lens);
          ++nv;
          idle = false;
        }
        if (!idle) {
          since = clock64();
        } else if (*abort_flag) {
          break;
        } else if (clock64() - since > (1ll << 32)) {
          *abort_flag = 1;
          if (status) atomicExch(status, kProducer);
          break;
        }
      }
      if (*abort_flag) {  // a wait somewhere ran out: the copies under way come in before the block ends
        auto drain = [&](uint64_t* bar, uint32_t fills) {
          for (int i = 0; fills > 0 && i < (1 << 16) && !mbar_test_wait(bar, (fills - 1) & 1); ++i) __nanosleep(100);
        };
        for (int i = 0; i < 3; ++i) drain(&bars->q_full[i], filled >> i & 1 ? 2 - (filled >> (8 + i) & 1) : 0);
        for (uint32_t i = 0; i < kKSlots; ++i) drain(&bars->k_full[i], (nk + kKSlots - 1 - i) / kKSlots);
        for (uint32_t i = 0; i < kVSlots; ++i) drain(&bars->v_full[i], (nv + kVSlots - 1 - i) / kVSlots);
        __nanosleep(1 << 19);  // and the products
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    const uint64_t dK0 = smem_desc_sw128(smem_u32(sK), 16, 1024);
    const uint64_t dQ0 = smem_desc_sw128(smem_u32(sQ), 16, 1024), dQp = smem_desc_sw128(smem_u32(sQp), 16, 1024);
    for (uint32_t ts = 0; c.advance(s, lens); ++ts) {
      const int x = ts & 1;
      const uint32_t ks = ts % kKSlots;
      const int q = c.is_own ? (c.iown & 1) : 2;
      if (c.j == 0) {
        const uint32_t use = c.is_own ? (uint32_t)(c.iown >> 1) : (uint32_t)c.ipre;
        if (!warp_wait(&bars->q_full[q], use & 1, abort_flag, status, kMma)) break;
      }
      const bool ends = c.ends();
      uint4 fresh = make_uint4(0, 0, 0, 0);  // lanes 0-7: the new key
      if (ends && lane < 8)
        fresh = *reinterpret_cast<const uint4*>(p.qkv + (int64_t)c.b * p.ld_qkv + (s.H + c.h) * D + lane * 8);
      if (!warp_wait(&bars->k_full[ks], (ts / kKSlots) & 1, abort_flag, status, kMma)) break;
      if (ends) {  // the sequence ends in this tile: row `last` is the new token's
        const int last = c.limit - 1 - c.key();
        if (lane < 8) {
          *reinterpret_cast<uint4*>(sK + ks * kTile + last * 128 + ((lane ^ (last & 7)) << 4)) = fresh;
          *reinterpret_cast<uint4*>(p.kcache + (int64_t)c.b * p.batch_stride + (int64_t)(c.limit - 1) * p.ld_cache + c.h * D +
                                    lane * 8) = fresh;
        }
        fence_proxy_async_smem();
        __syncwarp();
      }
      if (!warp_wait(&bars->s_free[x], ((ts >> 1) & 1) ^ 1, abort_flag, status, kMma)) break;
      tc_fence_after();
      if (lane == 0) {
        const uint32_t idesc = idesc_f16_f32(BKV, 0, false, false) | ((uint32_t)(c.rows(s) + 15) >> 4) << 18;
        const uint64_t a = desc_adv(dK0, ks * kTile);
        const uint64_t b = q == 2 ? dQp : desc_adv(dQ0, q * p.q_own_stride);
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk)
          umma_f16(tmem + x * 64, desc_adv(a, kk * 32), desc_adv(b, kk * 32), idesc, kk > 0 ? 1u : 0u);
        umma_commit(&bars->s_full[x]);
        umma_commit(&bars->k_empty[ks]);
        if (c.j == c.n - 1) umma_commit(&bars->q_empty[q]);
      }
      __syncwarp();
    }
  } else if (warp == 6) {
    const uint64_t dP0 = smem_desc_sw128(smem_u32(sP), kTile, 1024);
    // A of the second product for slot 0 and keys 0-15: rows 0-63 are V^T, rows 64-127, one leading offset on, ones.
    // 16 keys (2 KB) or a slot further, the start moves up and the leading offset down by as much, both in units of 16.
    const uint64_t dV0 = smem_desc_sw128(smem_u32(sV), smem_u32(s1) - smem_u32(sV), 1024);
    constexpr uint64_t kStep = 2048 / 16, kSlot = kTile / 16;
    for (uint32_t tp = 0; c.advance(s, lens); ++tp) {
      const uint32_t vs = tp % kVSlots;
      const bool ends = c.ends();
      uint4 fresh = make_uint4(0, 0, 0, 0);  // lanes 0-7: the new value
      if (ends && lane < 8)
        fresh = *reinterpret_cast<const uint4*>(p.qkv + (int64_t)c.b * p.ld_qkv + (s.H + s.Hkv + c.h) * D + lane * 8);
      if (!warp_wait(&bars->v_full[vs], (tp / kVSlots) & 1, abort_flag, status, kMma)) break;
      if (ends) {
        const int last = c.limit - 1 - c.key();
        uint8_t* tile = sV + vs * kTile;
        if (lane < 8) {
          *reinterpret_cast<uint4*>(tile + last * 128 + ((lane ^ (last & 7)) << 4)) = fresh;
          *reinterpret_cast<uint4*>(p.vcache + (int64_t)c.b * p.batch_stride + (int64_t)(c.limit - 1) * p.ld_cache + c.h * D +
                                    lane * 8) = fresh;
        }
        for (int i = (last + 1) * 8 + lane; i < BKV * 8; i += 32)
          *reinterpret_cast<uint4*>(tile + i * 16) = make_uint4(0, 0, 0, 0);
        fence_proxy_async_smem();
        __syncwarp();
      }
      if (!warp_wait(&bars->p_full, tp & 1, abort_flag, status, kMma)) break;
      tc_fence_after();
      if (lane == 0) {
        const uint32_t idesc = idesc_f16_f32(128, 0, true, true) | (uint32_t)rest_at(c.rows(s)) >> 3 << 18;  // both parts
        const uint64_t dv = dV0 + vs * (kSlot - (kSlot << 16));
#pragma unroll
        for (int kk = 0; kk < BKV / 16; ++kk)
          umma_f16(tmem + 128, dv + kk * (kStep - (kStep << 16)), desc_adv(dP0, kk * 2048), idesc,
                   (c.j > 0 || kk > 0) ? 1u : 0u);
        umma_commit(&bars->v_empty[vs]);
        umma_commit(&bars->p_empty);
      }
      __syncwarp();
    }
  } else {
    bool ok = true;
    for (uint32_t g = 0; ok && c.advance(s, lens);) {
      const int rows = c.rows(s);
      // Straight code for a few widths: branches per row cost more than the columns they save.
      if (rows <= 8)
        ok = softmax_item<8>(p, c, rows, g, bars, sP, tmem, status);
      else if (rows <= 16)
        ok = softmax_item<16>(p, c, rows, g, bars, sP, tmem, status);
      else if (rows <= 32)
        ok = softmax_item<32>(p, c, rows, g, bars, sP, tmem, status);
      else
        ok = softmax_item<64>(p, c, rows, g, bars, sP, tmem, status);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, kTmemCols);
  }
}

// out[b][h*64 + c] = f16(sum_s o_s[c] 2^(m_s - M) / sum_s l_s 2^(m_s - M)) over the row's parts; zeros for an idle
// sequence. One block of 128 threads per row: warp w takes parts w, w + 4, ..., a lane two columns.
__global__ void __launch_bounds__(128) attn_prefix_join_kernel(const Params p, int* status) {
  __shared__ float2 wacc[4][32];
  __shared__ float wm[4], wl[4];
  const Sched& s = p.s;
  const int row = blockIdx.x, b = row / s.H, hq = row - b * s.H;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int raw = p.lens[b], len = own_length(s, raw);
  prior_kernel_wait();
  __half2* dst = reinterpret_cast<__half2*>(p.out + (int64_t)b * p.ld_out + hq * D);
  if (len == 0) {
    if (raw > s.max_len && threadIdx.x == 0 && hq == 0 && status) atomicExch(status, kStatusDecodeBadLength);
    if (warp == 0) dst[lane] = __floats2half2_rn(0.f, 0.f);
    return;
  }
  int npre = 0;
  if (s.T > 0) {
    const int unit = b / s.nb * s.Hkv + hq / s.G;
    npre = s.block_of(unit * s.NT + s.NT - 1) - s.block_of(unit * s.NT) + 1;
  }
  const int nown = ((len + BKV - 1) / BKV + s.OC - 1) / s.OC, n = npre + nown;
  const float2* ml = p.ml + (int64_t)row * s.nparts;
  const float* o = p.o + (int64_t)row * s.nparts * D;
  float M = -INFINITY, L = 0.f;
  float2 acc = make_float2(0.f, 0.f);
#pragma unroll 4
  for (int i = warp; i < n; i += 4) {
    const int part = i < npre ? i : s.nsp + i - npre;
    const float2 q = ml[part];
    const float2 v = *reinterpret_cast<const float2*>(o + (int64_t)part * D + 2 * lane);
    const float nm = fmaxf(M, q.x);
    const float a = M == -INFINITY ? 0.f : ex2(M - nm), w = ex2(q.x - nm);
    L = L * a + q.y * w;
    acc.x = acc.x * a + v.x * w;
    acc.y = acc.y * a + v.y * w;
    M = nm;
  }
  if (lane == 0) wm[warp] = M, wl[warp] = L;
  wacc[warp][lane] = acc;
  __syncthreads();
  if (warp != 0) return;
  float gm = fmaxf(fmaxf(wm[0], wm[1]), fmaxf(wm[2], wm[3]));
  L = 0.f, acc = make_float2(0.f, 0.f);
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    if (wl[w] == 0.f) continue;  // no part
    const float a = ex2(wm[w] - gm);
    L += wl[w] * a;
    acc.x += wacc[w][lane].x * a;
    acc.y += wacc[w][lane].y * a;
  }
  dst[lane] = __floats2half2_rn(acc.x / L, acc.y / L);
}

// The same with the own keys: a block per (sequence, key / value head), NT threads. A warp takes 16 keys at a time, eight
// lanes to a key (16 bytes each), four keys side by side, and every lane group keeps its own running (m, l, o) of the
// keys it has seen for each of the G heads. The prefix's parts are then added by warps (a head each, a lane two
// columns), and all partial results meet in shared memory. Only the parts wait for the first kernel, so a block begins
// while that still runs. Products go two columns at a time (packed fp32), and only a row's last step looks at the
// length.
//
// What bounds it is how many bytes are on their way: copies go to a ring of two 16-key steps a warp in shared memory
// (loads straight to registers, a step at a time: 72.2 us for 64 sequences of 16 heads, up to 1000 own keys behind 32749;
// rings of two, three and four steps 59.0, 59.8 and 73.8, since four leave too few blocks an SM; all with the prefix's P in
// one fp16 number). Without a prefix the same sequences take 25.5 us, 5.2 TB/s. With four heads a key head it is bound by
// their instructions: 96 sequences of 32 heads, up to 500 keys, add 18.9 us.
constexpr int kOwnStages = 2, kOwnStage = 4096;  // bytes of 16 keys and values

template <int G, int NT>
__global__ void __launch_bounds__(NT, (G <= 2 ? 640 : G == 3 ? 512 : 384) / NT) attn_prefix_own_kernel(const Params p, int* status) {
  constexpr int U = 4, KW = NT / 32;  // warps that share the keys
  constexpr int JW = KW / G;          // warps that share a head's parts
  static_assert(JW >= 1, "");
  extern __shared__ __align__(16) uint8_t own_smem[];  // a ring a warp; in the end the partial results
  __shared__ float sm[KW + JW][G], sl[KW + JW][G];
  const Sched& s = p.s;
  const int b = blockIdx.x / s.Hkv, h = blockIdx.x - b * s.Hkv;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int raw = p.lens[b], len = own_length(s, raw);
  __half* dst = p.out + (int64_t)b * p.ld_out + h * G * D;
  if (len == 0) {
    if (raw > s.max_len && threadIdx.x == 0 && h == 0 && status) atomicExch(status, kStatusDecodeBadLength);
    for (int i = threadIdx.x; i < G * D; i += NT) dst[i] = __ushort_as_half(0);
    prior_kernel_wait();
    return;
  }
  const __half* row = p.qkv + (int64_t)b * p.ld_qkv;
  __half* kc = p.kcache + (int64_t)b * p.batch_stride + h * D;
  __half* vc = p.vcache + (int64_t)b * p.batch_stride + h * D;
  const __half* nk = row + (s.H + h) * D;
  const __half* nv = nk + s.Hkv * D;
  const int part = (lane & 7) * 8;
  // Steps of the warp: keys k0 + 4 i + lane / 8, fetched kOwnStages ahead. Every lane copies what it reads itself, so nobody
  // waits for another lane; the new token's row comes from qkv.
  constexpr int kStep = KW * 4 * U;
  static_assert(kOwnStage == 2 * U * 512, "");
  uint8_t* region = own_smem + warp * (kOwnStages * kOwnStage);
  uint8_t* ring = region + lane * 16;
  int k0 = warp * 4 * U, kf = k0;
  const int64_t row4 = 4 * p.ld_cache;
  const __half* kp = kc + (int64_t)(k0 + (lane >> 3)) * p.ld_cache + part;
  const __half* vp = vc + (int64_t)(k0 + (lane >> 3)) * p.ld_cache + part;
  auto fetch = [&](uint8_t* slot) {
    if (kf + 4 * U < len) {
#pragma unroll
      for (int i = 0; i < U; ++i) {
        cp_async_16(slot + i * 512, kp + i * row4, 16);
        cp_async_16(slot + (U + i) * 512, vp + i * row4, 16);
      }
    } else if (kf < len) {
#pragma unroll
      for (int i = 0; i < U; ++i) {
        const int key = kf + 4 * i + (lane >> 3);
        const uint32_t bytes = key < len ? 16 : 0;  // zeros behind the end
        cp_async_16(slot + i * 512, key < len - 1 ? kp + i * row4 : nk + part, bytes);
        cp_async_16(slot + (U + i) * 512, key < len - 1 ? vp + i * row4 : nv + part, bytes);
      }
    }
    cp_async_commit();
    kf += kStep, kp += kStep * p.ld_cache, vp += kStep * p.ld_cache;
  };
#pragma unroll
  for (int i = 0; i < kOwnStages; ++i) fetch(ring + i * kOwnStage);
  float2 q[G][4], o[G][4];
  float m[G], l[G];
#pragma unroll
  for (int g = 0; g < G; ++g) {
    const uint4 u = *reinterpret_cast<const uint4*>(row + (h * G + g) * D + part);
    const __half2* hq = reinterpret_cast<const __half2*>(&u);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      q[g][j] = __fmul2_rn(__half22float2(hq[j]), make_float2(p.scale_log2, p.scale_log2));
      o[g][j] = make_float2(0.f, 0.f);
    }
    m[g] = kNoKey, l[g] = 0.f;
  }
  if (threadIdx.x < 16) {  // the new key and value are appended
    const int ch = (threadIdx.x & 7) * 8;
    const bool is_v = threadIdx.x >= 8;
    *reinterpret_cast<uint4*>((is_v ? vc : kc) + (int64_t)(len - 1) * p.ld_cache + ch) =
        *reinterpret_cast<const uint4*>((is_v ? nv : nk) + ch);
  }
  auto step = [&](auto full, const uint8_t* slot) {
    uint4 ku[U], vu[U];
#pragma unroll
    for (int i = 0; i < U; ++i) {
      ku[i] = *reinterpret_cast<const uint4*>(slot + i * 512);
      vu[i] = *reinterpret_cast<const uint4*>(slot + (U + i) * 512);
    }
    float sc[G][U];
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const __half2* hk = reinterpret_cast<const __half2*>(&ku[i]);
      float2 f[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) f[j] = __half22float2(hk[j]);
#pragma unroll
      for (int g = 0; g < G; ++g) {
        float2 a = __fmul2_rn(q[g][0], f[0]);
#pragma unroll
        for (int j = 1; j < 4; ++j) a = __ffma2_rn(q[g][j], f[j], a);
        sc[g][i] = a.x + a.y;
      }
    }
#pragma unroll
    for (int x = 1; x < 8; x <<= 1)
#pragma unroll
      for (int g = 0; g < G; ++g)
#pragma unroll
        for (int i = 0; i < U; ++i) sc[g][i] += __shfl_xor_sync(0xffffffffu, sc[g][i], x);
#pragma unroll
    for (int g = 0; g < G; ++g) {
      float nm = m[g];
#pragma unroll
      for (int i = 0; i < U; ++i) {
        if (!full.value && k0 + i * 4 + (lane >> 3) >= len) sc[g][i] = -INFINITY;
        nm = fmaxf(nm, sc[g][i]);
      }
      if (__any_sync(0xffffffffu, nm > m[g])) {  // (a step in which no maximum grows rescales nothing)
        const float a = ex2(m[g] - nm);
        l[g] *= a;
#pragma unroll
        for (int j = 0; j < 4; ++j) o[g][j] = __fmul2_rn(o[g][j], make_float2(a, a));
        m[g] = nm;
      }
#pragma unroll
      for (int i = 0; i < U; ++i) {
        sc[g][i] = ex2(sc[g][i] - m[g]);
        l[g] += sc[g][i];
      }
    }
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const __half2* hv = reinterpret_cast<const __half2*>(&vu[i]);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 x = __half22float2(hv[j]);
#pragma unroll
        for (int g = 0; g < G; ++g) o[g][j] = __ffma2_rn(make_float2(sc[g][i], sc[g][i]), x, o[g][j]);
      }
    }
  };
  uint32_t at_slot = 0;
  while (k0 < len) {
    cp_async_wait<kOwnStages - 1>();
    const uint8_t* slot = ring + at_slot;
    if (k0 + 4 * U <= len)
      step(std::true_type{}, slot);
    else
      step(std::false_type{}, slot);
    fetch(ring + at_slot);  // every lane has used what it overwrites
    at_slot = at_slot == (kOwnStages - 1) * kOwnStage ? 0 : at_slot + kOwnStage;
    k0 += kStep;
  }
  // The prefix's parts: warp j G + g takes parts j, j + JW, .. of head g. The first four are under way while the own keys'
  // results are brought together.
  prior_kernel_wait();
  int npre = 0;
  if (s.T > 0) {
    const int unit = b / s.nb * s.Hkv + h;
    npre = s.block_of(unit * s.NT + s.NT - 1) - s.block_of(unit * s.NT) + 1;
  }
  const int part0 = warp < JW * G ? warp / G : npre;
  const int64_t at = ((int64_t)b * s.H + h * G + warp % G) * s.nparts;
  float2 ml[4], po[4];
  auto read_parts = [&](int i0) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const bool is = i0 + i * JW < npre;
      ml[i] = is ? p.ml[at + i0 + i * JW] : make_float2(-INFINITY, 0.f);
      po[i] = is ? *reinterpret_cast<const float2*>(p.o + (at + i0 + i * JW) * D + 2 * lane) : make_float2(0.f, 0.f);
    }
  };
  read_parts(part0);
  // The four lane groups of the warp, then the warp's result to its ring, which nothing is on its way to any more.
  __syncwarp();
#pragma unroll
  for (int g = 0; g < G; ++g) {
    float wm = fmaxf(m[g], __shfl_xor_sync(0xffffffffu, m[g], 8));
    wm = fmaxf(wm, __shfl_xor_sync(0xffffffffu, wm, 16));
    const float a = ex2(m[g] - wm);
    l[g] *= a;
    l[g] += __shfl_xor_sync(0xffffffffu, l[g], 8);
    l[g] += __shfl_xor_sync(0xffffffffu, l[g], 16);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float2 v = __fmul2_rn(o[g][j], make_float2(a, a));
      v.x += __shfl_xor_sync(0xffffffffu, v.x, 8);
      v.y += __shfl_xor_sync(0xffffffffu, v.y, 8);
      v.x += __shfl_xor_sync(0xffffffffu, v.x, 16);
      v.y += __shfl_xor_sync(0xffffffffu, v.y, 16);
      if (lane < 8) *reinterpret_cast<float2*>(region + (g * D + part + 2 * j) * 4) = v;
    }
    if (lane == 0) sm[warp][g] = wm, sl[warp][g] = l[g];
  }
  if (warp < JW * G) {
    const int g = warp % G, j = warp / G;
    float M = kNoKey, L = 0.f;
    float2 acc = make_float2(0.f, 0.f);
    for (int i0 = part0;;) {
      float nm = M;
#pragma unroll
      for (int i = 0; i < 4; ++i) nm = fmaxf(nm, ml[i].x);
      const float a = ex2(M - nm);
      L *= a, acc = __fmul2_rn(acc, make_float2(a, a));
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float w = ex2(ml[i].x - nm);
        L = fmaf(ml[i].y, w, L);
        acc = __ffma2_rn(make_float2(w, w), po[i], acc);
      }
      M = nm;
      if ((i0 += 4 * JW) >= npre) break;
      read_parts(i0);
    }
    *reinterpret_cast<float2*>(region + (G * D + 2 * lane) * 4) = acc;
    if (lane == 0) sm[KW + j][g] = M, sl[KW + j][g] = L;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < G * D; i += NT) {
    const int g = i / D, d = i % D;
    float M = -INFINITY;
#pragma unroll
    for (int w = 0; w < KW + JW; ++w) M = fmaxf(M, sm[w][g]);
    float L = 0.f, a = 0.f;
#pragma unroll
    for (int w = 0; w < KW + JW; ++w) {
      const float e = sm[w][g] == -INFINITY ? 0.f : ex2(sm[w][g] - M);
      L = fmaf(sl[w][g], e, L);
      const int from = w < KW ? w : (w - KW) * G + g, at = w < KW ? i : G * D + d;
      a = fmaf(reinterpret_cast<const float*>(own_smem + from * (kOwnStages * kOwnStage))[at], e, a);
    }
    dst[i] = __float2half_rn(a / L);
  }
}

// The schedule, from sizes and the SM count alone.
bool plan(int B, int H, int Hkv, int64_t prefix_len, int64_t max_len, Sched* s, int* grid) {
  if (B <= 0 || Hkv <= 0 || H <= 0 || H % Hkv || H / Hkv > kRows || prefix_len < 0 || max_len <= 0) return false;
  // (Columns of a row of qkv are counted in 32 bits.)
  if (prefix_len > (1 << 28) || max_len > (1 << 28) || (int64_t)B * H > (1 << 24) || H > (1 << 22)) return false;
  const int blocks = 2 * num_sms();
  s->B = B, s->H = H, s->Hkv = Hkv, s->G = H / Hkv;
  s->nb = std::min(kRows / s->G, B);
  s->P = (int)prefix_len;
  s->NT = (s->P + BKV - 1) / BKV;
  const int64_t T = (int64_t)((B + s->nb - 1) / s->nb) * Hkv * s->NT;
  const int own_tiles = (int)((max_len + BKV - 1) / BKV);
  const int64_t own_all = (int64_t)B * Hkv * own_tiles;
  if (T >= (1ll << 31) || own_all >= (1ll << 31)) return false;
  s->T = (int)T;
  s->gp = (int)std::min<int64_t>(T, blocks);
  s->per = s->gp > 0 ? s->T / s->gp : 0;
  s->more = s->gp > 0 ? s->T % s->gp : 0;
  s->max_len = (int)max_len;
  // One block per pair reads few keys, or there are pairs enough to fill the GPU; up to four heads' state in registers.
  // Four sequences of 16 heads, up to 1000 own keys behind 2000: 11.9 us plain, 14.0 as products; up to 2000 own keys
  // 15.3 and 15.3. With 64 heads on the 16, 16 sequences, up to 512 keys 21.0 and 20.3, up to 1000 keys 25.5 and 22.9.
  s->plain = s->G <= 4 && (max_len <= (s->G == 1 ? 1024 : 512) || (int64_t)B * Hkv >= blocks);
  // Enough items to even out ragged lengths, few parts to join.
  s->OC = (int)std::max<int64_t>(1, (own_all + 3 * blocks - 1) / (3 * blocks));
  s->OC = std::min(s->OC, own_tiles);
  s->chunks = s->plain ? 0 : (own_tiles + s->OC - 1) / s->OC;
  s->nsp = T > 0 ? std::min(s->NT, (s->NT - 1 + s->per - 1) / s->per + 1) : 0;  // blocks that a unit may be split over
  s->nparts = s->nsp + s->chunks;
  if ((int64_t)B * H * s->nparts >= (1ll << 31)) return false;
  *grid = (int)std::min<int64_t>(blocks, std::max<int64_t>(s->gp, T + (int64_t)B * Hkv * s->chunks));
  s->step_b = *grid / Hkv;
  s->step_h = *grid % Hkv;
  if (s->nparts == 0) s->nparts = 1;
  return true;
}

int64_t ml_bytes(const Sched& s) { return ((int64_t)s.B * s.H * s.nparts * 8 + 255) / 256 * 256; }

}  // namespace pfx
}  // namespace jx

using namespace jx;

extern "C" int64_t jx_attn_decode_prefix_workspace_bytes(int B, int H, int Hkv, int64_t prefix_len, int64_t max_len) {
  pfx::Sched s;
  int grid;
  if (!pfx::plan(B, H, Hkv, prefix_len, max_len, &s, &grid)) return -1;
  return pfx::ml_bytes(s) + (int64_t)B * H * s.nparts * pfx::D * 4;
}

extern "C" int jx_attn_decode_prefix(const void* qkv, int64_t ld_qkv, const void* kprefix, const void* vprefix,
                                     int64_t ld_prefix, int64_t prefix_len, void* kcache, void* vcache, int64_t ld_cache,
                                     int64_t cache_batch_stride, const int32_t* lens, int64_t max_len, int B, int H,
                                     int Hkv, int Dh, float scale, void* workspace, void* out, int64_t ld_out,
                                     jx_stream_t stream) {
  const char* name = "jx_attn_decode_prefix";
  JX_CHECK_ARG(Dh == 64, "%s: head_dim must be 64 (got %d)", name, Dh);
  // (The row maximum is taken before the scale.)
  JX_CHECK_ARG(scale >= 0.f && scale <= 1e30f, "%s: scale must be a number of at least 0 (got %g)", name, scale);
  JX_CHECK_ARG(qkv && kcache && vcache && lens && workspace && out && (prefix_len == 0 || (kprefix && vprefix)),
               "%s: NULL argument", name);
  pfx::Params p{};
  int grid;
  JX_CHECK_ARG(pfx::plan(B, H, Hkv, prefix_len, max_len, &p.s, &grid),
               "%s: bad shape B %d, H %d, Hkv %d (at most %d query heads per key head), prefix %lld, max_len %lld", name, B, H,
               Hkv, pfx::kRows, (long long)prefix_len, (long long)max_len);
  const int G = p.s.G;
  const int64_t width = (H + 2 * (int64_t)Hkv) * 64, own_width = (int64_t)Hkv * 64;
  JX_CHECK_ARG(aligned16(qkv) && aligned16(kcache) && aligned16(vcache) && aligned16(workspace) &&
                   aligned16(kprefix) && aligned16(vprefix) && ((uintptr_t)out & 3) == 0,
               "%s: operands must be 16-byte aligned", name);
  JX_CHECK_ARG(ld_qkv % 8 == 0 && ld_qkv >= width && ld_out % 2 == 0 && ld_out >= (int64_t)H * 64 && ld_cache % 8 == 0 &&
                   ld_cache >= own_width && cache_batch_stride % 8 == 0 && cache_batch_stride >= 0 &&
                   (prefix_len == 0 || (ld_prefix % 8 == 0 && ld_prefix >= own_width)),
               "%s: row strides must be multiples of 8 and hold a row", name);
  // Sequence by sequence or position by position; each appends to its own.
  JX_CHECK_ARG(B == 1 || (cache_batch_stride >= own_width && (cache_batch_stride >= (max_len - 1) * ld_cache + own_width ||
                                                              ld_cache >= (B - 1) * cache_batch_stride + own_width)),
               "%s: the sequences' caches overlap", name);
  // Queries as [sequence][head][64]: one box holds G heads of one sequence, or of a row tile's sequences.
  CUtensorMap qp{}, qo{}, kp{}, vp{}, kc{}, vc{};  // those of what there is
  const uint64_t qdims[3] = {64, (uint64_t)H, (uint64_t)B}, qstr[2] = {128, (uint64_t)ld_qkv * 2};
  const uint32_t qob[3] = {64, (uint32_t)G, 1}, qpb[3] = {64, (uint32_t)G, (uint32_t)p.s.nb};
  const uint64_t cdims[3] = {(uint64_t)Hkv * 64, (uint64_t)max_len, (uint64_t)B};
  const uint64_t cstr[2] = {(uint64_t)ld_cache * 2, (uint64_t)(B > 1 ? cache_batch_stride : ld_cache) * 2};
  const uint32_t cbox[3] = {64, 128, 1};
  bool ok = true;
  if (p.s.chunks > 0)
    ok = make_tmap_f16_3d(&qo, qkv, qdims, qstr, qob) && make_tmap_f16_3d(&kc, kcache, cdims, cstr, cbox) &&
         make_tmap_f16_3d(&vc, vcache, cdims, cstr, cbox);
  if (ok && p.s.T > 0)
    ok = make_tmap_f16_3d(&qp, qkv, qdims, qstr, qpb) &&
         make_tmap_f16(&kp, kprefix, (uint64_t)Hkv * 64, prefix_len, ld_prefix, 64, 128) &&
         make_tmap_f16(&vp, vprefix, (uint64_t)Hkv * 64, prefix_len, ld_prefix, 64, 128);
  JX_CHECK_ARG(ok, "%s: cannot encode a TMA descriptor", name);
  p.qkv = static_cast<const __half*>(qkv);
  p.ld_qkv = ld_qkv;
  p.kcache = static_cast<__half*>(kcache);
  p.vcache = static_cast<__half*>(vcache);
  p.ld_cache = ld_cache;
  p.batch_stride = cache_batch_stride;
  p.lens = lens;
  p.scale_log2 = scale * 1.4426950408889634f;
  p.ml = static_cast<float2*>(workspace);
  p.o = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + pfx::ml_bytes(p.s));
  p.out = static_cast<__half*>(out);
  p.ld_out = ld_out;
  p.q_own_bytes = G * 128;
  p.q_own_stride = (G + 7) / 8 * 1024;
  p.q_pre_bytes = p.s.nb * G * 128;
  constexpr size_t kFixed = 1024 + pfx::kQTile + (pfx::kKSlots + pfx::kVSlots + 2) * pfx::kTile + pfx::kOnes + sizeof(pfx::Bars);
  static_assert(kFixed + 2 * 1024 + 1024 <= 233472 / 2, "two blocks an SM with up to eight heads a key / value head");
  const size_t smem = kFixed + 2 * p.q_own_stride;
  static std::atomic<uint64_t> done{0};
  static void (*const own[2][4])(const pfx::Params, int*) = {
      {pfx::attn_prefix_own_kernel<1, 128>, pfx::attn_prefix_own_kernel<2, 128>, pfx::attn_prefix_own_kernel<3, 128>,
       pfx::attn_prefix_own_kernel<4, 128>},
      {pfx::attn_prefix_own_kernel<1, 256>, pfx::attn_prefix_own_kernel<2, 256>, pfx::attn_prefix_own_kernel<3, 256>,
       pfx::attn_prefix_own_kernel<4, 256>}};
  auto set_up = [] {
    cudaError_t e = cudaFuncSetAttribute(pfx::attn_prefix_part_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         (int)(kFixed + 2 * pfx::kQTile));
    for (int i = 0; e == cudaSuccess && i < 8; ++i)
      e = cudaFuncSetAttribute(own[i / 4][i % 4], cudaFuncAttributeMaxDynamicSharedMemorySize,
                               (i < 4 ? 4 : 8) * pfx::kOwnStages * pfx::kOwnStage);
    return e;
  };
  JX_CUDA_TRY(once_per_device(done, set_up), name);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  int* status = status_ptr();
  // Both kernels may be set up while the one before them finishes; they wait before they read what it wrote.
  cudaLaunchConfig_t cfg{};
  cfg.stream = st;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  if (grid > 0) {
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(pfx::kThreads);
    cfg.dynamicSmemBytes = smem;
    JX_CUDA_TRY(cudaLaunchKernelEx(&cfg, pfx::attn_prefix_part_kernel, qp, qo, kp, vp, kc, vc, p, status), name);
    JX_CHECK_LAUNCH(name);
  } else {
    cfg.numAttrs = 0;  // no prefix: the second kernel alone, which reads before it waits
  }
  cfg.dynamicSmemBytes = 0;
  if (p.s.plain) {
    // Eight warps share the keys of a pair where four would leave SMs empty (256 pairs of up to 257 keys behind 1791:
    // 12.0 -> 11.2 us; 1024 pairs of up to 1000 62.6 either way).
    const int NT = max_len > 128 && B * Hkv < 2 * num_sms() ? 256 : 128;
    cfg.gridDim = dim3(B * Hkv);
    cfg.blockDim = dim3(NT);
    cfg.dynamicSmemBytes = NT / 32 * pfx::kOwnStages * pfx::kOwnStage;
    JX_CUDA_TRY(cudaLaunchKernelEx(&cfg, own[NT == 256][G - 1], p, status), name);
  } else {
    cfg.gridDim = dim3(B * H);
    cfg.blockDim = dim3(128);
    JX_CUDA_TRY(cudaLaunchKernelEx(&cfg, pfx::attn_prefix_join_kernel, p, status), name);
  }
  JX_CHECK_LAUNCH(name);
  return JX_OK;
}
