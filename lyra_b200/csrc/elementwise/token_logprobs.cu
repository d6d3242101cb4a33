// Scores of given tokens from logits: log probability, entropy and the k most likely alternatives of every row, and the
// gradient of the first two.
//
//   lse = log sum_v e^{x_v}      logprob = x_t - lse      H = lse - sum_v p_v x_v
//   dx_v = g_l ([v = t] - p_v) - g_H p_v (log p_v + H)
//
// Forward: one pass over a row with the running maximum m, s = sum e^{x-m} and u = sum e^{x-m} (x-m), from
// which lse = m + log s and H = log s - u / s: no cancellation between two large numbers. The pass also leaves the maximum of
// every run of loads in shared memory. The alternatives then need no second pass: the k-th largest of 64 disjoint subset maxima
// is a bound that at least k elements reach and few exceed, and only the runs that reach it are read again (a few hundred
// bytes, still in L2). The candidates are ranked by (value, lowest id), so the order in which they were found does not matter.
//
// Two CTAs per SM walk the rows. A producer warp streams them through a ring of bulk copies in shared memory (64 KB), eight warps add up
// and note run maxima, and a ninth finishes a row - joins the sums, picks the alternatives, writes - while the eight are in the next
// one: with the same warps doing both, finishing took as long as a third of a row (2048 rows of 201088 bf16 logits with 4 alternatives:
// 223 us, now 171 = 4.8 TB/s). What bounds it is the issue of about five instructions per logit (bf16: widen, multiply-add, exponential,
// two sums) beside the finishing warp. The gradient is bound by memory (1024 such rows, both directions: 211 us = 5.8 TB/s).
//
// Few rows are split over a cluster of up to eight CTAs (each SM streams a slice; partial results meet in the first CTA through
// distributed shared memory): one row of 201088 fp32 logits would otherwise be read by one SM. Such a row takes 22 us, most of them
// for steps that wait for one another.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include "../common/sm100.cuh"
#include "../common/tmap.h"

namespace lyra {
namespace tlp {

namespace cg = cooperative_groups;

constexpr int THREADS = 256, ALL = THREADS + 64;            // warps 0..7 add up, warp 8 finishes rows, warp 9 copies
constexpr int UNROLL = 4;            // 16-byte vectors per thread and chunk
constexpr int CHUNK = THREADS * UNROLL * 16, STAGES = 4;   // bytes of a chunk; chunks in flight or in use
constexpr int MAX_TOP = 32;
constexpr int CAP = 1024;            // candidates kept; more (long runs of equal logits) take the slower selection
constexpr int MAX_HITS = 256;        // runs looked at again
constexpr int MAX_VOCAB = 1 << 22;   // one warp sweeps a row of ties up to 33 times (a vector of 16 bytes per lane in about 800 cycles): 0.9e9
                                     // cycles, while the other warps' waits run out after 4e9
constexpr int MAX_RUNS = 3584;       // run maxima kept per row (14 KB, twice: two CTAs fit an SM)
constexpr float L2E = 1.4426950408889634f;
// Distances below a maximum (in log2 units) are cut off here: 2^-1000 is 0 in fp32 as well, and 0 * y stays 0.
constexpr float FLOOR = -1000.f;
// Logits are read as at least -BIG (a mask of -inf or of the type's lowest value is a token of probability 0 either way, and stays clear
// of inf * 0). Slices whose own maximum lies outside of -BIG .. BIG - nothing but such masks, as a rule - are scanned once more with
// distances formed in the logits' own unit: a row of the type's lowest value is a uniform distribution.
constexpr float BIG = 1e30f;

struct Fwd {
  const void* x;
  const long long* target;           // [N], negative: the row has no target (logprob 0)
  float* logprob;                    // [N]
  float* entropy;                    // [N]
  float* norm;                       // [2, N]: m and log s, for the gradient; or null
  float* top_lp;                     // [N, k]
  long long* top_id;                 // [N, k]
  long long stride;                  // elements between rows
  int* status;
  int N, V, k, chunks_per_run, runs;
};

// Order of the alternatives: larger value first (NaN above +inf, as a sort in torch has it; -0 equals 0), then lower id.
__device__ __forceinline__ uint32_t order_key(float x) {
  if (x != x) return 0xffffffffu;
  const uint32_t b = __float_as_uint(x + 0.0f);
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float key_value(uint32_t k) {
  if (k == 0xffffffffu) return __uint_as_float(0x7fc00000u);
  return __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k);
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// Two fp32 operations per instruction.
__device__ __forceinline__ uint64_t pair2(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void split2(uint64_t v, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

template <typename T>
struct Vec;
template <>
struct Vec<float> {
  static constexpr int N = 4;
  __device__ static void unpack(const uint4& v, float (&f)[4]) {
    f[0] = __uint_as_float(v.x); f[1] = __uint_as_float(v.y); f[2] = __uint_as_float(v.z); f[3] = __uint_as_float(v.w);
  }
  __device__ static uint4 pack(const float (&f)[4]) {
    return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
  }
  // the four logits as two pairs, at least -BIG
  __device__ static void pairs(const uint4& v, uint64_t (&x)[2]) {
    x[0] = pair2(fmaxf(__uint_as_float(v.x), -BIG), fmaxf(__uint_as_float(v.y), -BIG));
    x[1] = pair2(fmaxf(__uint_as_float(v.z), -BIG), fmaxf(__uint_as_float(v.w), -BIG));
  }
  __device__ static float load(const float* p) { return *p; }
  __device__ static float largest(const uint4& v) {
    return max_nan(max_nan(__uint_as_float(v.x), __uint_as_float(v.y)), max_nan(__uint_as_float(v.z), __uint_as_float(v.w)));
  }
  static constexpr uint32_t MINUS_INF = 0xff800000u;
};
template <>
struct Vec<__nv_bfloat16> {
  static constexpr int N = 8;
  __device__ static void unpack(const uint4& v, float (&f)[8]) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[2 * i] = __uint_as_float(w[i] << 16);
      f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
  __device__ static uint4 pack(const float (&f)[8]) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      __nv_bfloat162 t = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
      w[i] = *reinterpret_cast<uint32_t*>(&t);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
  __device__ static void pairs(const uint4& v, uint64_t (&x)[4]) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint32_t c;
      asm("max.bf16x2 %0, %1, %2;" : "=r"(c) : "r"(w[i]), "r"(0xf149f149u));          // -1e30 in bf16, twice
      x[i] = pair2(__uint_as_float(c << 16), __uint_as_float(c & 0xffff0000u));
    }
  }
  __device__ static float load(const __nv_bfloat16* p) { return __bfloat162float(*p); }
  __device__ static uint32_t max2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
  }
  __device__ static float largest(const uint4& v) {          // two values per instruction, unpacked once per 16 bytes
    const uint32_t m = max2(max2(v.x, v.y), max2(v.z, v.w));
    return max_nan(__uint_as_float(m << 16), __uint_as_float(m & 0xffff0000u));
  }
  static constexpr uint32_t MINUS_INF = 0xff80ff80u;
};

// A row is a list of 16-byte vectors on 16-byte boundaries: vector i holds elements i * VE - lead .. + VE - 1, where lead is the
// row's distance from the boundary below it. The first and the last vector may reach over the row's ends: those are gathered
// element by element and filled with -inf.
template <typename T>
struct Row {
  static constexpr int VE = Vec<T>::N;
  const T* p;
  int V, lead, n_vec;
  __device__ Row(const T* row, int v) : p(row), V(v) {
    lead = int((reinterpret_cast<uintptr_t>(row) & 15) / sizeof(T));
    n_vec = int(((long long)v + lead + VE - 1) / VE);
  }
  __device__ uint4 vec(int i) const {
    const int e0 = i * VE - lead;
    if (e0 >= 0 && e0 + VE <= V) return __ldg(reinterpret_cast<const uint4*>(p + e0));
    uint32_t w[4];
    if (sizeof(T) == 4) {
#pragma unroll
      for (int j = 0; j < 4; ++j) w[j] = (e0 + j >= 0 && e0 + j < V) ? reinterpret_cast<const uint32_t*>(p)[e0 + j] : 0xff800000u;
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int a = e0 + 2 * j, b = a + 1;
        const uint32_t lo = (a >= 0 && a < V) ? reinterpret_cast<const uint16_t*>(p)[a] : 0xff80u;
        const uint32_t hi = (b >= 0 && b < V) ? reinterpret_cast<const uint16_t*>(p)[b] : 0xff80u;
        w[j] = lo | (hi << 16);
      }
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
};

struct Stat {      // maximum m (NaN once a NaN was seen), s = sum 2^y, u = sum 2^y y with y = (x - m) log2 e
  float m, s, u;
};
__device__ __forceinline__ Stat merge(const Stat& a, const Stat& b) {
  Stat r;
  r.m = max_nan(a.m, b.m);
  // an empty side has m = -inf, s = u = 0: its distance must not become inf * 0
  const float da = a.m == -INFINITY ? 0.f : fmaxf((a.m - r.m) * L2E, FLOOR), db = b.m == -INFINITY ? 0.f : fmaxf((b.m - r.m) * L2E, FLOOR);
  const float ea = exp2f(da), eb = exp2f(db);
  r.s = a.s * ea + b.s * eb;
  r.u = ea * (a.u + da * a.s) + eb * (b.u + db * b.s);
  return r;
}
__device__ __forceinline__ Stat shfl_stat(const Stat& a, int o) {
  return Stat{__shfl_xor_sync(0xffffffffu, a.m, o), __shfl_xor_sync(0xffffffffu, a.s, o), __shfl_xor_sync(0xffffffffu, a.u, o)};
}

struct Shared {
  uint64_t full[STAGES], empty[STAGES];             // the ring
  uint64_t ready[2], finished[2];                   // sums and run maxima of a row (by parity): complete; no longer needed
  int abort;
  Stat part[2][THREADS / 32];
  uint32_t tmax[2][THREADS];
  int n_hits, n_cand;
  int hits[MAX_HITS];
  Stat total;                                       // clusters: read by the first CTA
  unsigned long long cand[CAP];                     // (key << 32) | ~id : one unsigned comparison is the whole order
  unsigned long long best[MAX_TOP];
};

__device__ __forceinline__ unsigned long long entry(uint32_t key, int id) { return ((unsigned long long)key << 32) | (uint32_t)(~id); }

// k best of list[0..n) into out[0..k), by one warp: entries are distinct (their ids are), so an entry's rank is the number of larger ones.
__device__ __forceinline__ void rank_select(const unsigned long long* list, int n, int k, unsigned long long* out) {
  for (int i = threadIdx.x & 31; i < n; i += 32) {
    const unsigned long long mine = list[i];
    int rank = 0;
#pragma unroll 8
    for (int j = 0; j < n; ++j) rank += list[j] > mine;
    if (rank < k) out[rank] = mine;
  }
  __syncwarp();
}

// A CTA's slice of a row: vectors [v0, v1), of which [w0, w1) lie wholly inside the row.
template <typename T>
struct Slice {
  Row<T> row;
  int v0, v1, w0, w1, n_chunks;
  __device__ Slice(const Fwd& p, int row_id, int cr, int lg)
      : row(reinterpret_cast<const T*>(p.x) + (long long)row_id * p.stride, p.V) {
    v0 = int((long long)row.n_vec * cr >> lg);
    v1 = int((long long)row.n_vec * (cr + 1) >> lg);
    w0 = row.lead > 0 ? 1 : 0;
    w1 = int(((long long)p.V + row.lead) / Vec<T>::N);
    n_chunks = (v1 - v0 + THREADS * UNROLL - 1) / (THREADS * UNROLL);
  }
};

// The k largest entries of a slice into sh.best (unfilled places 0), by one warp, from its run maxima. Returns nothing on purpose: a
// slice with fewer than k logits leaves places at 0.
template <typename T>
__device__ void pick(const Fwd& p, const Slice<T>& slice, Shared& sh, const uint32_t* run_key, const uint32_t* tmax) {
  constexpr int VE = Vec<T>::N, STEP = THREADS * UNROLL;
  const int lane = threadIdx.x & 31, k = p.k;
  const Row<T>& row = slice.row;
  auto elements = [&](int i, auto&& use) {            // (key, id) of the elements of vector i
    const int e0 = i * VE - row.lead;
    float f[VE];
    Vec<T>::unpack(row.vec(i), f);
#pragma unroll
    for (int x = 0; x < VE; ++x)
      if (e0 + x >= 0 && e0 + x < p.V) use(order_key(f[x]), e0 + x);
  };
  auto push = [&](uint32_t key, int id) {
    const int at = atomicAdd(&sh.n_cand, 1);
    if (at < CAP) sh.cand[at] = entry(key, id);
  };
  // a bound that at least k elements reach: the k-th largest of 64 disjoint subset maxima (a subset without elements has key 0)
  uint32_t a = 0, b = 0;
#pragma unroll
  for (int j = 0; j < THREADS / 64; ++j) {
    a = max(a, tmax[j * 64 + lane]);
    b = max(b, tmax[j * 64 + 32 + lane]);
  }
  int ra = 0, rb = 0;
#pragma unroll 4
  for (int s = 0; s < 32; ++s) {
    const uint32_t oa = __shfl_sync(0xffffffffu, a, s), ob = __shfl_sync(0xffffffffu, b, s);
    ra += (oa > a || (oa == a && s < lane)) + (ob > a);
    rb += (oa >= b) + (ob > b || (ob == b && s < lane));
  }
  const uint32_t hit_a = __ballot_sync(0xffffffffu, ra == k - 1), hit_b = __ballot_sync(0xffffffffu, rb == k - 1);    // ranks 0..63 are all taken once
  uint32_t bound = hit_a ? __shfl_sync(0xffffffffu, a, __ffs(hit_a) - 1) : __shfl_sync(0xffffffffu, b, __ffs(hit_b) - 1);
  bound = max(bound, 1u);                           // every real key is larger than 0 (-inf has 0x007fffff)
  if (lane < k) sh.best[lane] = 0;
  if (lane == 0) sh.n_hits = sh.n_cand = 0;
  __syncwarp();
  // runs that reach it
  const int n_runs = (slice.n_chunks + p.chunks_per_run - 1) / p.chunks_per_run * THREADS;
#pragma unroll 8
  for (int e = lane; e < n_runs; e += 32)
    if (run_key[e] >= bound) {
      const int at = atomicAdd(&sh.n_hits, 1);
      if (at < MAX_HITS) sh.hits[at] = e;
    }
  __syncwarp();
  const int n_hits = *reinterpret_cast<volatile int*>(&sh.n_hits);
  if (n_hits <= MAX_HITS) {
    const int per = UNROLL * p.chunks_per_run;      // vectors of a run
    for (int w = lane; w < n_hits * per; w += 32) {
      const int e = sh.hits[w / per], x = w % per, c = e / THREADS * p.chunks_per_run + x / UNROLL;
      const int i = slice.v0 + c * STEP + (x % UNROLL) * THREADS + e % THREADS;
      if (c < slice.n_chunks && i < slice.v1) elements(i, [&](uint32_t key, int id) { if (key >= bound) push(key, id); });
    }
    __syncwarp();
    const int n = *reinterpret_cast<volatile int*>(&sh.n_cand);
    if (n <= CAP) {
      rank_select(sh.cand, n, k, sh.best);
      return;
    }
    __syncwarp();
    if (lane == 0) sh.n_cand = 0;
    __syncwarp();
  }
  // Long runs of equal logits: what exceeds the bound, and of what equals it the k lowest ids, in one sweep in the order of the ids.
  int equal = 0;
  for (int i0 = slice.v0; i0 < slice.v1; i0 += 32) {
    int mine = 0;
    if (i0 + lane < slice.v1) elements(i0 + lane, [&](uint32_t key, int id) { mine += key == bound; if (key > bound) push(key, id); });
    if (equal < k) {
      int before = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, before, o);
        if (lane >= o) before += v;
      }
      const int all = __shfl_sync(0xffffffffu, before, 31);
      int at = equal + before - mine;
      if (mine && at < k) elements(i0 + lane, [&](uint32_t key, int id) { if (key == bound && at++ < k) push(key, id); });
      equal += all;
    }
  }
  __syncwarp();
  const int n = *reinterpret_cast<volatile int*>(&sh.n_cand);
  if (n <= CAP) {
    rank_select(sh.cand, n, k, sh.best);
    return;
  }
  // One of the 64 subsets holds more than CAP logits above all others' maxima: k sweeps, each takes the largest entry below the last.
  unsigned long long last = ~0ull;
  for (int q = 0; q < k; ++q) {
    unsigned long long mine = 0;
    for (int i = slice.v0 + lane; i < slice.v1; i += 32)
      elements(i, [&](uint32_t key, int id) {
        const unsigned long long en = entry(key, id);
        if (en < last && en > mine) mine = en;
      });
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) mine = max(mine, __shfl_xor_sync(0xffffffffu, mine, o));
    if (lane == 0) sh.best[q] = mine;
    last = mine;
  }
  __syncwarp();
}

// Results of a row from its sums and (lane i of the warp) its i-th best entry.
template <typename T>
__device__ void finish_row(const Fwd& p, const Slice<T>& slice, int row_id, const Stat& t, unsigned long long b) {
  const int lane = threadIdx.x & 31;
  const bool bad = !(fabsf(t.m) < INFINITY);        // a NaN, a +inf, or nothing but -inf: no distribution
  const float nan = __uint_as_float(0x7fc00000u);
  const double log_s = log(double(t.s));
  // (x - m) - log s, never x - lse: in a row of the type's lowest value m + log s would swallow log s
  auto logp = [&](float x) { return float((double(x) - double(t.m)) - log_s); };
  if (lane == 0) {
    const long long tg = p.target[row_id];
    float lp = nan;
    if (tg < 0) lp = 0.f;
    else if (tg < p.V && !bad) lp = logp(Vec<T>::load(slice.row.p + tg));
    p.logprob[row_id] = lp;
    p.entropy[row_id] = bad ? nan : float(log_s - double(t.u) / double(t.s) * 0.69314718055994530942);
    if (p.norm) {
      p.norm[row_id] = bad ? nan : t.m;
      p.norm[p.N + row_id] = bad ? nan : float(log_s);
    }
  }
  if (lane < p.k) {
    p.top_id[(long long)row_id * p.k + lane] = (long long)(uint32_t)~(uint32_t)b;
    p.top_lp[(long long)row_id * p.k + lane] = bad ? nan : logp(key_value(uint32_t(b >> 32)));
  }
}

template <typename T>
__global__ void __launch_bounds__(ALL, 2) token_logprobs_kernel(const Fwd p) {
  constexpr int VE = Vec<T>::N, STEP = THREADS * UNROLL;
  extern __shared__ __align__(128) uint8_t dyn[];
  uint8_t* ring = dyn;
  Shared& sh = *reinterpret_cast<Shared*>(dyn + STAGES * CHUNK);
  uint32_t* run_keys = reinterpret_cast<uint32_t*>(dyn + STAGES * CHUNK + sizeof(Shared));      // [2][p.runs][THREADS]
  cg::cluster_group cluster = cg::this_cluster();
  const int cs = int(cluster.num_blocks()), cr = int(cluster.block_rank()), lg = 31 - __clz(cs);
  const int row0 = int(blockIdx.x) >> lg, row_step = int(gridDim.x) >> lg;      // in a cluster of several CTAs: one row each
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;

  if (tid == 0) {
    for (int i = 0; i < STAGES; ++i) {
      mbar_init(smem_u32(&sh.full[i]), 1);
      mbar_init(smem_u32(&sh.empty[i]), THREADS / 32);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(smem_u32(&sh.ready[i]), THREADS / 32);
      mbar_init(smem_u32(&sh.finished[i]), 1);
    }
    sh.abort = 0;
    fence_mbar_init();
  }
  __syncthreads();
  volatile int* abortp = &sh.abort;
  auto wait = [&](uint64_t& bar, uint32_t parity) {
    if (!mbar_wait(smem_u32(&bar), parity & 1, abortp)) {
      *abortp = 1;                                  // every later wait gives up at once; the results are void, the status word says so
      atomicCAS(p.status, 0, STATUS_TIMEOUT_FULL);
    }
  };

  if (warp == 9) {
    if (lane == 0) {
      uint32_t q = 0;
      for (int row_id = row0; row_id < p.N; row_id += row_step) {
        const Slice<T> slice(p, row_id, cr, lg);
        for (int c = 0; c < slice.n_chunks; ++c, ++q) {
          const uint32_t s = q % STAGES, bar = smem_u32(&sh.full[s]);
          wait(sh.empty[s], q / STAGES + 1);
          if (*abortp) continue;
          // the chunk's whole vectors; the one or two that reach over the row's ends are gathered by the threads that own them
          const int at = slice.v0 + c * STEP, a = max(at, slice.w0), b = min(min(at + STEP, slice.v1), slice.w1), n = max(b - a, 0) * 16;
          mbar_expect_tx(bar, n);
          if (n)
            asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(smem_u32(ring + s * CHUNK + (a - at) * 16)),
                         "l"(slice.row.p + (long long)a * VE - slice.row.lead), "r"(n), "r"(bar)
                         : "memory");
        }
      }
    }
    __syncwarp();
  } else if (warp < 8) {
    uint32_t q = 0, it = 0;                         // chunks, rows so far
    const uint64_t l2e2 = pair2(L2E, L2E);
    for (int row_id = row0; row_id < p.N; row_id += row_step, ++it) {
      const Slice<T> slice(p, row_id, cr, lg);
      const int v0 = slice.v0, v1 = slice.v1;
      uint32_t* run_key = run_keys + (it & 1) * p.runs * THREADS;
      wait(sh.finished[it & 1], (it >> 1) + 1);     // the row before the last has been finished: its places are free
      // y' = x log2e - ml with ml = m log2e as it is rounded
      float m = -INFINITY, ml = 0.f;
      uint64_t s2 = pair2(0.f, 0.f), u2 = s2;
      uint32_t best_key = 0, this_run = 0;
      int in_run = 0, run = 0;
      for (int c = 0; c < slice.n_chunks; ++c, ++q) {
        const uint32_t s = q % STAGES;
        wait(sh.full[s], q / STAGES);
        uint4 v[UNROLL];
        const int first = v0 + c * STEP + tid;
        const uint8_t* stage = ring + s * CHUNK;
        if (v0 + c * STEP >= slice.w0 && v0 + (c + 1) * STEP <= min(v1, slice.w1)) {
#pragma unroll
          for (int j = 0; j < UNROLL; ++j) v[j] = *reinterpret_cast<const uint4*>(stage + (j * THREADS + tid) * 16);
        } else {
#pragma unroll
          for (int j = 0; j < UNROLL; ++j) {
            const int i = first + j * THREADS;
            if (i >= v1) v[j] = make_uint4(Vec<T>::MINUS_INF, Vec<T>::MINUS_INF, Vec<T>::MINUS_INF, Vec<T>::MINUS_INF);
            else if (i >= slice.w0 && i < slice.w1) v[j] = *reinterpret_cast<const uint4*>(stage + (j * THREADS + tid) * 16);
            else v[j] = slice.row.vec(i);
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&sh.empty[s]));
        float g = Vec<T>::largest(v[0]);
#pragma unroll
        for (int j = 1; j < UNROLL; ++j) g = max_nan(g, Vec<T>::largest(v[j]));
        if (p.k) {
          if (first < v1) this_run = max(this_run, order_key(g));
          if (++in_run == p.chunks_per_run) {
            run_key[run++ * THREADS + tid] = this_run;
            best_key = max(best_key, this_run);
            this_run = 0;
            in_run = 0;
          }
        }
        g = max_nan(m, g);
        if (!(g <= m)) {                            // moved up (or NaN)
          const float to = fabsf(g) <= BIG ? g * L2E : 0.f;      // out of range: nothing is added up (masks), or scanned once more
          if (fabsf(m) <= BIG) {
            const float d = fmaxf(ml - to, FLOOR), e = exp2f(d);
            const uint64_t e2 = pair2(e, e), d2 = pair2(d, d), zero = pair2(0.f, 0.f);
            u2 = fma2(fma2(d2, s2, u2), e2, zero);
            s2 = fma2(s2, e2, zero);
          }
          m = g;
          ml = to;
        }
        const uint64_t off = pair2(-ml, -ml);
#pragma unroll
        for (int j = 0; j < UNROLL; ++j) {
          uint64_t x[VE / 2];
          Vec<T>::pairs(v[j], x);
#pragma unroll
          for (int i = 0; i < VE / 2; ++i) {
            const uint64_t y = fma2(x[i], l2e2, off);
            float a, b;
            split2(y, a, b);
            const uint64_t e = pair2(exp2f(a), exp2f(b));
            s2 = add2(s2, e);
            u2 = fma2(e, y, u2);
          }
        }
      }
      if (p.k) {
        if (in_run) {
          run_key[run++ * THREADS + tid] = this_run;
          best_key = max(best_key, this_run);
        }
        sh.tmax[it & 1][tid] = best_key;
      }
      float sa, sb, ua, ub;
      split2(s2, sa, sb);
      split2(u2, ua, ub);
      // from ml to m log2e: the rounding of ml, exactly (a product's error in one fma)
      const float d = fabsf(m) <= BIG ? -fmaf(m, L2E, -ml) : 0.f, e = exp2f(d);
      Stat st{m, m == -INFINITY ? 0.f : (sa + sb) * e, m == -INFINITY ? 0.f : ((ua + ub) + d * (sa + sb)) * e};
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) st = merge(st, shfl_stat(st, o));
      if (lane == 0) sh.part[it & 1][warp] = st;
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&sh.ready[it & 1]));
    }
  } else {
    // ---- the finishing warp
    uint32_t it = 0;
    for (int row_id = row0; row_id < p.N; row_id += row_step, ++it) {
      const Slice<T> slice(p, row_id, cr, lg);
      wait(sh.ready[it & 1], it >> 1);
      Stat t = lane < THREADS / 32 ? sh.part[it & 1][lane] : Stat{-INFINITY, 0.f, 0.f};
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) t = merge(t, shfl_stat(t, o));
      if (const float top = t.m; fabsf(top) > BIG && fabsf(top) < INFINITY) {      // masks only (or logits beyond any use): see BIG
        t = Stat{top, 0.f, 0.f};
        for (int i = slice.v0 + lane; i < slice.v1; i += 32) {
          float f[VE];
          Vec<T>::unpack(slice.row.vec(i), f);
#pragma unroll
          for (int x = 0; x < VE; ++x) {
            const float y = fmaxf((f[x] - top) * L2E, FLOOR), e = exp2f(y);
            t.s += e;
            t.u = fmaf(e, y, t.u);
          }
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) t = merge(t, shfl_stat(t, o));
      }
      if (p.k) pick(p, slice, sh, run_keys + (it & 1) * p.runs * THREADS, sh.tmax[it & 1]);
      if (lane == 0) mbar_arrive(smem_u32(&sh.finished[it & 1]));
      if (cs > 1) {
        if (lane == 0) sh.total = t;
      } else {
        finish_row<T>(p, slice, row_id, t, lane < p.k ? sh.best[lane] : 0ull);
        __syncwarp();
      }
    }
  }
  if (cs > 1) {                                     // one row per cluster: its first CTA joins the slices
    cluster.sync();
    if (cr == 0) {
      // unfilled places of small slices are 0: below every entry, but equal to one another, so they are dropped
      const int n = cs * p.k;                       // at most 256
      unsigned long long* out = sh.cand + 8 * MAX_TOP;
      if (tid < n) sh.cand[tid] = cluster.map_shared_rank(&sh, tid / p.k)->best[tid % p.k];
      __syncthreads();
      if (tid < n && sh.cand[tid]) {
        const unsigned long long mine = sh.cand[tid];
        int rank = 0;
#pragma unroll 8
        for (int j = 0; j < n; ++j) rank += sh.cand[j] > mine;
        if (rank < p.k) out[rank] = mine;
      }
      __syncthreads();
      if (warp == 8) {
        Stat t = lane < cs ? cluster.map_shared_rank(&sh, lane)->total : Stat{-INFINITY, 0.f, 0.f};
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) t = merge(t, shfl_stat(t, o));
        finish_row<T>(p, Slice<T>(p, row0, cr, lg), row0, t, lane < p.k ? out[lane] : 0ull);
      }
    }
    cluster.sync();                                 // no CTA leaves while its shared memory is read
  }
  if (*abortp)
    for (int i = 0; i < 64; ++i) __nanosleep(1000);  // copies still in flight land before the shared memory is given back
}

// ------------------------------------------------------------------------------------------------ gradient
struct Bwd {
  const void* x;
  void* dx;                          // [N, W] contiguous
  const long long* target;
  const float *norm, *entropy, *g_lp, *g_h;     // g_lp / g_h may be null (no gradient from that output)
  long long stride;
  int N, V, W, blocks_per_row;       // columns V .. W - 1 (vocabulary padding) get zeros
};

constexpr int B_THREADS = 256, B_UNROLL = 4;

// Bound by memory: every logit is read once and every gradient written once, in 16-byte pieces aligned to the gradient's row
// (which a row of logits with the same distance from a 16-byte boundary shares; otherwise its elements are loaded one by one).
// With d = x - m:  p = 2^{d log2e - log2 s},  g = -p (g_H d + c),  c = g_l + g_H (H - log s): 5.5 operations a logit, the target's
// term is added to the one vector that holds it. A row without a distribution has NaN for m, d is cut off and p is 0, but c is NaN.
template <typename T>
__global__ void __launch_bounds__(B_THREADS) token_logprobs_bwd_kernel(const Bwd p) {
  constexpr int VE = Vec<T>::N;
  const long long r = blockIdx.x / p.blocks_per_row;
  const int blk = int(blockIdx.x - r * p.blocks_per_row);
  const T* x = reinterpret_cast<const T*>(p.x) + r * p.stride;
  T* dx = reinterpret_cast<T*>(p.dx) + r * (long long)p.W;
  const int lead = int((reinterpret_cast<uintptr_t>(dx) & 15) / sizeof(T));
  const bool same = ((reinterpret_cast<uintptr_t>(x) ^ reinterpret_cast<uintptr_t>(dx)) & 15) == 0;
  const int n_vec = int(((long long)p.W + lead + VE - 1) / VE);
  const int first = blk * B_THREADS * B_UNROLL + threadIdx.x;
  uint4 v[B_UNROLL];
#pragma unroll
  for (int j = 0; j < B_UNROLL; ++j) {
    const int i = first + j * B_THREADS, e0 = i * VE - lead;
    if (i < n_vec && same && e0 >= 0 && e0 + VE <= p.V) v[j] = __ldg(reinterpret_cast<const uint4*>(x + e0));
  }
  const long long tg = p.target[r];
  float gl = p.g_lp && tg >= 0 ? p.g_lp[r] : 0.f;
  if (tg >= p.V) gl = __uint_as_float(0x7fc00000u);
  const float gh = p.g_h ? p.g_h[r] : 0.f, m = p.norm[r], log_s = p.norm[p.N + r], H = p.entropy[r];
  const float c = m != m ? m : fmaf(gh, H - log_s, gl), shift = -log_s * L2E;
  // whatever the target's place, as a vector index; -1 for none
  const int hot = tg >= 0 && tg < p.V ? int((tg + lead) / VE) : -1;
#pragma unroll
  for (int j = 0; j < B_UNROLL; ++j) {
    const int i = first + j * B_THREADS, e0 = i * VE - lead;
    if (i >= n_vec) continue;
    const bool inside = e0 >= 0 && e0 + VE <= p.V;
    float f[VE];
    if (same && inside) {
      Vec<T>::unpack(v[j], f);
    } else {
#pragma unroll
      for (int q = 0; q < VE; ++q) f[q] = (e0 + q >= 0 && e0 + q < p.V) ? Vec<T>::load(x + e0 + q) : -INFINITY;
    }
#pragma unroll
    for (int q = 0; q < VE; q += 2) {
      const float d0 = fmaxf(f[q] - m, FLOOR), d1 = fmaxf(f[q + 1] - m, FLOOR);      // a probability of 0 contributes 0, not 0 * inf
      const uint64_t d = pair2(d0, d1);
      float y0, y1, w0, w1;
      split2(fma2(d, pair2(L2E, L2E), pair2(shift, shift)), y0, y1);
      split2(fma2(d, pair2(gh, gh), pair2(c, c)), w0, w1);
      f[q] = -exp2f(y0) * w0;
      f[q + 1] = -exp2f(y1) * w1;
    }
    if (i == hot) {
#pragma unroll
      for (int q = 0; q < VE; ++q)
        if (e0 + q == tg) f[q] += gl;
    }
    if (inside) {
      *reinterpret_cast<uint4*>(dx + e0) = Vec<T>::pack(f);
    } else {
#pragma unroll
      for (int q = 0; q < VE; ++q)
        if (e0 + q >= 0 && e0 + q < p.W) dx[e0 + q] = T(e0 + q < p.V ? f[q] : 0.f);
    }
  }
}

template <typename T>
int launch_fwd(Fwd p, cudaStream_t stream) {
  // Slices: as many CTAs per row (1, 2, 4, 8) as keep two CTAs on each of the 148 SMs, but at least 32 KB of logits each.
  int cs = 1;
  while (cs < 8 && (long long)p.N * cs * 2 <= 2 * sm_count() && (long long)p.V * int(sizeof(T)) >= (long long)cs * 2 * 32768) cs *= 2;
  const long long n_vec = ((long long)p.V + 2 * Vec<T>::N) / Vec<T>::N + 1;
  const long long chunks = (n_vec / cs + 1 + THREADS * UNROLL - 1) / (THREADS * UNROLL) + 1;
  p.chunks_per_run = int((chunks * THREADS + MAX_RUNS - 1) / MAX_RUNS);
  p.runs = int((chunks + p.chunks_per_run - 1) / p.chunks_per_run);
  const size_t smem = STAGES * CHUNK + sizeof(Shared) + (p.k ? size_t(2) * p.runs * THREADS * 4 : 0);
  static std::mutex lock;
  static size_t configured[64] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev >= 64) return -91;
  {
    std::lock_guard<std::mutex> guard(lock);
    if (smem > configured[dev]) {
      if (cudaFuncSetAttribute(token_logprobs_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, int(smem)) != cudaSuccess) return -92;
      configured[dev] = smem;
    }
  }
  cudaLaunchConfig_t cfg = {};
  const long long groups = 2LL * sm_count() / cs;               // two CTAs per SM, each walks rows
  cfg.gridDim = dim3(unsigned(p.N < groups ? p.N : groups) * cs);
  cfg.blockDim = dim3(ALL);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = cs;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (cudaLaunchKernelEx(&cfg, token_logprobs_kernel<T>, p) != cudaSuccess) {
    LYRA_CHECK_LAUNCH();
    return -93;
  }
  return 0;
}

template <typename T>
int launch_bwd(Bwd p, cudaStream_t stream) {
  const long long n_vec = ((long long)p.W + 2 * Vec<T>::N - 2) / Vec<T>::N;        // the most any alignment of the row needs
  p.blocks_per_row = int((n_vec + B_THREADS * B_UNROLL - 1) / (B_THREADS * B_UNROLL));
  const long long blocks = (long long)p.N * p.blocks_per_row;
  if (blocks > 0x7fffffffLL) return -94;
  token_logprobs_bwd_kernel<T><<<unsigned(blocks), B_THREADS, 0, stream>>>(p);
  LYRA_CHECK_LAUNCH();
  return 0;
}

}  // namespace tlp
}  // namespace lyra

// x [N, *] (rows `stride` elements apart, columns 0 .. V - 1 are used), bf16 or fp32; target int64 [N].
extern "C" int lyra_token_logprobs(const void* x, int is_bf16, const long long* target, float* logprob, float* entropy, float* norm, float* top_lp,
                                   long long* top_id, int N, int V, int k, long long stride, int* status, cudaStream_t stream) {
  using namespace lyra::tlp;
  if (N < 1 || N > (1 << 28) || V < 1 || V > MAX_VOCAB || k < 0 || k > MAX_TOP || k > V || stride < V) return -90;
  if (reinterpret_cast<uintptr_t>(x) % (is_bf16 ? 2 : 4)) return -90;
  Fwd p{x, target, logprob, entropy, norm, top_lp, top_id, stride, status, N, V, k, 1, 1};
  return is_bf16 ? launch_fwd<__nv_bfloat16>(p, stream) : launch_fwd<float>(p, stream);
}

// dx [N, W] contiguous (W >= V): gradient of the logits from the gradients of logprob and entropy (either may be null).
extern "C" int lyra_token_logprobs_bwd(const void* x, int is_bf16, void* dx, const long long* target, const float* norm, const float* entropy,
                                       const float* g_lp, const float* g_h, int N, int V, int W, long long stride, cudaStream_t stream) {
  using namespace lyra::tlp;
  if (N < 1 || V < 1 || W < V || W > (1 << 30) || stride < V) return -90;
  if (reinterpret_cast<uintptr_t>(x) % (is_bf16 ? 2 : 4) || reinterpret_cast<uintptr_t>(dx) % (is_bf16 ? 2 : 4)) return -90;
  Bwd p{x, dx, target, norm, entropy, g_lp, g_h, stride, N, V, W, 1};
  return is_bf16 ? launch_bwd<__nv_bfloat16>(p, stream) : launch_bwd<float>(p, stream);
}
