// A whole pre-norm mixture-of-experts block for the few tokens (1..64) of a decode step, in one persistent cooperative launch:
//
//   xn = rms_norm(x) * norm;  logits = xn R + r;  e_1..e_k = top-k of logits, s = softmax over the chosen logits
//   out = x + rs * sum_j s_j (W_down[e_j]^T a_j + b_down),  a_j = swiglu(W_up[e_j]^T xn + b_up)     (shared experts: s = 1)
//
// The work is reading the chosen experts' weights once; every expert is a product with a handful of columns. So the design is
// about bytes in flight and about the order in which memory sees them. Each SM holds one CTA; the weights of a phase are cut into
// equal units (64 x 256 bf16 or 128 x 256 e4m3 values: 32 KB), the units are numbered through all chosen experts and dealt to the CTAs
// in contiguous runs of equal length (experts x column panels rarely divide by 148); teams of up to four neighbouring CTAs walk
// neighbouring panels side by side, so that memory sees longer pieces of each row (a CTA's own piece of a W_up row is 2 x 128 bytes). Two producer warps stream a run through a ring
// of stages (weights by TMA, the matching piece of the activations by cp.async; 100-190 KB in flight); eight consumer warps multiply
// with m16n8k16 MMAs in which the weight columns are the 16 rows and the tokens the 8 columns, two tiles of 16 columns per warp - in
// the up-projection the gate and the linear column of the same hidden units, so SwiGLU happens in registers. A tcgen05 tile has 128
// rows of one operand and its accumulator in TMEM: with one to eight tokens per expert it would wait for the same bytes.
// Panels that a run boundary cuts are summed through small fp32 slots: in the up-projection by whichever CTA arrives last, in the
// down-projection by all CTAs after a last barrier; always in team order, so the result does not depend on timing.
//
// What bounds it: memory, at 4 to 5 TB/s while a phase runs (pieces of 128 to 512 bytes of a row instead of long runs), and what lies
// between the phases. One token of 4 of 32 experts of 2880 x 2880 (200 MB), 69 us on the device: router and choice 8, up 38 (the
// slowest CTA 10 after the fastest), down 14, barrier and join 4, launch 5. 64 tokens of e4m3 (2.8 GB): 640 us, 4.3 TB/s.
//
//   phase 1  router: logits and row norms from the unrounded input in fp32, split over experts, tokens and input columns
//   grid barrier; every CTA derives the same choice and row lists on its own
//   phase 2  up-projection + SwiGLU -> act (bf16);   grid barrier (the first stages of phase 3 are already loading)
//   phase 3  down-projection; a panel of output columns passes through all experts, scaled by their scores in an fp32 tile
//
// Roundings: x * norm is rounded to the MMA's operand type (its 1/rms factor is applied to the fp32 sum), so is the SwiGLU result;
// the output is rounded once at the end. The router sees neither rounding. The operand type is bf16 for bf16 weights. For e4m3
// weights it is fp16, into which e4m3 converts in one instruction per pair (by way of bf16 it is four, and the conversions then set
// the pace: 3.8 instead of 4.9 TB/s while units run); fp16 has three more bits of mantissa and a smaller range, so each token's x * norm is scaled by
// a power of two that puts its largest value below 2^10, and the SwiGLU result by one that makes its bound fit: g sigmoid(beta g) lies in
// [-0.2785 / beta, limit] for beta > 0, |l + 1| in 0 .. limit + 1.
#include <cooperative_groups.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "../common/sm100.cuh"
#include "../common/tmap.h"

namespace lyra {
namespace moeblk {

namespace cg = cooperative_groups;

constexpr int CONSUMERS = 256, THREADS = CONSUMERS + 64;   // + a warp that copies weights and one that copies activations
constexpr int MAX_F = 64, MAX_N = 256, MAX_ROWS = 512;   // tokens, experts (shared ones included), assignments
constexpr int W_STAGE = 32768, PANEL = 256;              // bytes of weights per stage, columns per panel
constexpr int MAX_STAGES = 6;
constexpr int SCALE_STAGE = 1024;                        // end of an e4m3 stage: 16 column groups x 8 k-16 steps of fp32 (512 bytes used)
constexpr int MAX_CSPLIT = 8;                            // pieces of the input width in the router
constexpr float L2E = 1.4426950408889634f;

// Rows a slot has room for: the accumulators of an expert hold 8, 16, 32 or 64 rows.
__host__ __device__ inline int slot_rows(int F) { return F <= 8 ? 8 : F <= 16 ? 16 : F <= 32 ? 32 : 64; }

// fp32 tile of a CTA: [F][256] sums in phase 3; before that the router's logits [F][E <= 256] and the reductions of its tasks
__host__ __device__ inline int buf_bytes(int F) { return (F < 4 ? 4 : F) * PANEL * 4; }

struct Params {
  const __nv_bfloat16* x;      // [F, C]
  const float* norm;           // [C]
  const float* router;         // [C, E]
  const float* router_bias;    // [E] or null
  const float* up_scale;       // e4m3: [n, C / up_bk, 2H / up_bn]
  const float* down_scale;     // e4m3: [n, H / dn_bk, C / dn_bn]
  const float* up_bias;        // [n, 2H] or null
  const float* down_bias;      // [n, C] or null
  __nv_bfloat16* out;          // [F, C]
  float* scores;               // [F, k]
  long long* idx;              // [F, k]
  // workspace
  float* part_logits;          // [csplit, F, E]
  float* part_sq;              // [csplit, F]
  float* gain;                 // [F]  e4m3: what a token's x * norm was divided by
  uint16_t* xs;                // [F, C]  x * norm in the operand type
  uint16_t* act;               // [rows, H]
  float* slots;                // [grid, 2, slot_rows(F), 256]
  int* counters;               // [n, up panels]
  int* status;
  int F, C, H, E, shared, k, csplit, stages, x_stage, up_team, dn_team, up_bk, up_bn, dn_bk, dn_bn;
  float eps, beta, limit, residual_scale, act_scale, act_gain;     // act_scale: power of two, act_gain its inverse
};

struct Lists {                                    // derived by every CTA from the logits; the same everywhere
  unsigned long long mask[MAX_N];                 // tokens of each expert
  float rstd[MAX_F];
  float gain[MAX_F];                              // of the tokens' sums in the up-projection: rstd and the operand's own factor
  float bias[MAX_N];                              // of the router, fetched before the barrier that the logits wait for
  float score[MAX_ROWS];                          // by row
  short chosen[MAX_F * 8];
  float chosen_score[MAX_F * 8];
  unsigned char tok[MAX_ROWS];                    // token of each row; rows are grouped by expert
  short expert[MAX_N];                            // active experts in ascending order
  short base[MAX_N + 1];                          // first row of each active expert
  int n_active;
  int last;
  int abort;
};

__device__ __forceinline__ void consumer_sync() { asm volatile("bar.sync 1, 256;" ::: "memory"); }
__device__ __forceinline__ void cp16(uint32_t dst, const void* src, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp4(uint32_t dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void lds128(uint32_t addr, float& a, float& b, float& c, float& d) {
  asm volatile("ld.shared.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(a), "=f"(b), "=f"(c), "=f"(d) : "r"(addr));
}
__device__ __forceinline__ void cp_arrive(uint32_t bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
__device__ __forceinline__ void ldsm4t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// the same with fp16 operands, into a fresh accumulator
__device__ __forceinline__ void mma16816_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ uint32_t e4m3x2_to_f16x2(uint16_t two) {       // exact, NaN included
  const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(two, __NV_E4M3);
  return *reinterpret_cast<const uint32_t*>(&h);
}
// Order of the logits: larger first, NaN above +inf (as torch.topk has it), -0 equal to 0; 0 is below every logit.
__device__ __forceinline__ uint32_t order_key(float v) {
  if (v != v) return 0xffffffffu;
  const uint32_t b = __float_as_uint(v + 0.0f);
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float key_value(uint32_t k) {
  if (k == 0xffffffffu) return __uint_as_float(0x7fc00000u);
  return __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k);
}

// ------------------------------------------------------------------------------------------------ unit runs
// U units over G CTAs in contiguous runs: the first U % G CTAs take one unit more (with U < G the first U CTAs take one each).
struct Runs {
  int per, rem;
  __device__ Runs(int U, int G) : per(U / G), rem(U % G) {}
  __device__ int begin(int c) const { return c * per + min(c, rem); }
  __device__ int owner(int u) const {
    const int wide = rem * (per + 1);
    return u < wide ? u / (per + 1) : rem + (u - wide) / per;
  }
};

// ------------------------------------------------------------------------------------------------ phase 1
constexpr int RT = 8, RE = 8;      // tokens and experts of one router task
constexpr int NV = RT * (RE + 1);  // sums of a task: logits and squares

template <int T, bool WHOLE>
__device__ __forceinline__ void router_dots(const Params& p, int e0, int t0, int c0, int c1, float (&acc)[RT][RE], float (&sq)[RT]) {
  const __nv_bfloat16* __restrict__ x = p.x + (long long)t0 * p.C;
  const float* __restrict__ router = p.router + e0;
  const float* __restrict__ norm = p.norm;
#pragma unroll 2
  for (int c = c0 + threadIdx.x; c < c1; c += CONSUMERS) {
    float r[RE], v[T];
    const float* rp = router + (long long)c * p.E;
    if (WHOLE) {
      const float4 a = __ldg(reinterpret_cast<const float4*>(rp)), b = __ldg(reinterpret_cast<const float4*>(rp) + 1);
      r[0] = a.x; r[1] = a.y; r[2] = a.z; r[3] = a.w; r[4] = b.x; r[5] = b.y; r[6] = b.z; r[7] = b.w;
    } else {
#pragma unroll
      for (int e = 0; e < RE; ++e) r[e] = e0 + e < p.E ? __ldg(rp + e) : 0.f;
    }
#pragma unroll
    for (int t = 0; t < T; ++t) v[t] = t0 + t < p.F ? __bfloat162float(__ldg(x + (long long)t * p.C + c)) : 0.f;
    const float w = __ldg(norm + c);
#pragma unroll
    for (int t = 0; t < T; ++t) {
      sq[t] = fmaf(v[t], v[t], sq[t]);
      const float s = v[t] * w;
#pragma unroll
      for (int e = 0; e < RE; ++e) acc[t][e] = fmaf(s, r[e], acc[t][e]);
    }
  }
}

__device__ void router_task(const Params& p, int task, float* red) {
  const int n_es = (p.E + RE - 1) / RE, n_tg = (p.F + RT - 1) / RT;
  const int es = task % n_es, tg = (task / n_es) % n_tg, cs = task / (n_es * n_tg);
  const int e0 = es * RE, t0 = tg * RT, n_t = min(RT, p.F - t0);
  const int c0 = int((long long)p.C * cs / p.csplit), c1 = int((long long)p.C * (cs + 1) / p.csplit);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const bool whole = e0 + RE <= p.E && p.E % 4 == 0 && (reinterpret_cast<uintptr_t>(p.router) & 15) == 0;
  float acc[RT][RE], sq[RT];
#pragma unroll
  for (int t = 0; t < RT; ++t) {
    sq[t] = 0.f;
#pragma unroll
    for (int e = 0; e < RE; ++e) acc[t][e] = 0.f;
  }
  if (n_t == 1) {                                  // one token: four rows of the router in flight per thread instead of eight tokens
    whole ? router_dots<1, true>(p, e0, t0, c0, c1, acc, sq) : router_dots<1, false>(p, e0, t0, c0, c1, acc, sq);
  } else {
    whole ? router_dots<RT, true>(p, e0, t0, c0, c1, acc, sq) : router_dots<RT, false>(p, e0, t0, c0, c1, acc, sq);
  }
#pragma unroll
  for (int t = 0; t < RT; ++t) {
    if (t < n_t) {
#pragma unroll
      for (int e = 0; e <= RE; ++e) {
        float v = e < RE ? acc[t][e < RE ? e : 0] : sq[t];
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
        if (lane == 0) red[warp * NV + t * (RE + 1) + e] = v;
      }
    }
  }
  consumer_sync();
  if (threadIdx.x < n_t * (RE + 1)) {
    float v = 0.f;
#pragma unroll
    for (int w = 0; w < CONSUMERS / 32; ++w) v += red[w * NV + threadIdx.x];
    const int t = threadIdx.x / (RE + 1), e = threadIdx.x % (RE + 1);
    if (e < RE) {
      if (e0 + e < p.E) p.part_logits[((long long)cs * p.F + t0 + t) * p.E + e0 + e] = v;
    } else if (es == 0) {
      p.part_sq[cs * p.F + t0 + t] = v;
    }
  }
  consumer_sync();
}

// x * norm of token t in fp16, scaled by a power of two so that its largest value lies in [2^9, 2^10).
__device__ void operand_row_f16(const Params& p, int t, float* red) {
  const __nv_bfloat16* x = p.x + (long long)t * p.C;
  float m = 0.f;
  for (int c = threadIdx.x; c < p.C; c += CONSUMERS) m = fmaxf(m, fabsf(__bfloat162float(__ldg(x + c)) * __ldg(p.norm + c)));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = m;
  consumer_sync();
  m = red[0];
#pragma unroll
  for (int w = 1; w < CONSUMERS / 32; ++w) m = fmaxf(m, red[w]);
  // exponent arithmetic: 2^(9 - floor(log2 m)); zeros, subnormal sizes and infinities are left as they are
  const int e = int(__float_as_uint(m) >> 23);
  const bool usual = e > 30 && e < 254;
  const float to = usual ? __uint_as_float(uint32_t(254 + 9 - e) << 23) : 1.f, back = usual ? __uint_as_float(uint32_t(e - 9) << 23) : 1.f;
  for (int c = threadIdx.x; c < p.C; c += CONSUMERS)
    p.xs[(long long)t * p.C + c] = __half_as_ushort(__float2half_rn(__bfloat162float(__ldg(x + c)) * __ldg(p.norm + c) * to));
  if (threadIdx.x == 0) p.gain[t] = back;
  consumer_sync();
}

// The k experts of every token, a token per warp; NE * 32 >= E.
template <int NE>
__device__ __forceinline__ void choose(const Params& p, Lists& L, const float* logits) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int f = warp; f < p.F; f += CONSUMERS / 32) {
    const float rstd = L.rstd[f];
    uint32_t key[NE];
#pragma unroll
    for (int i = 0; i < NE; ++i) {
      const int e = i * 32 + lane;
      key[i] = e < p.E ? order_key(fmaf(logits[f * p.E + e], rstd, L.bias[e])) : 0u;
    }
    float top = 0.f, den = 0.f, mine = 0.f;
    int my_e = 0;
    for (int j = 0; j < p.k; ++j) {
      uint32_t bk = key[0];
      int be = lane;
#pragma unroll
      for (int i = 1; i < NE; ++i)
        if (key[i] > bk) { bk = key[i]; be = i * 32 + lane; }       // ascending e: the first of equals stays
      const uint32_t best = __reduce_max_sync(0xffffffffu, bk);
      be = int(__reduce_min_sync(0xffffffffu, bk == best ? uint32_t(be) : 0xffffffffu));
#pragma unroll
      for (int i = 0; i < NE; ++i)
        if (i * 32 + lane == be) key[i] = 0;
      const float v = key_value(best);
      if (j == 0) top = v;
      const float w = exp2f((v - top) * L2E);
      den += w;
      if (lane == j) { mine = w; my_e = be; }
    }
    if (lane < p.k) {
      const float s = mine / den;
      L.chosen[f * 8 + lane] = short(my_e);
      L.chosen_score[f * 8 + lane] = s;
      atomicOr(&L.mask[my_e], 1ull << f);
      if (blockIdx.x == 0) {
        p.scores[(long long)f * p.k + lane] = s;
        p.idx[(long long)f * p.k + lane] = my_e;
      }
    }
  }
}

// Choice of every token and the experts' row lists, in shared memory.
__device__ void route(const Params& p, Lists& L, float* logits) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int n = p.E + p.shared;
  for (int e = threadIdx.x; e < n; e += CONSUMERS)
    L.mask[e] = e < p.E ? 0ull : (p.F == 64 ? ~0ull : (1ull << p.F) - 1ull);
  // all partial sums of the router are fetched at once (eight independent loads per thread and round), summed in a fixed order
  const int cells = p.F * p.E;
  if (p.csplit == 1) {
    for (int i0 = threadIdx.x; i0 < cells; i0 += 8 * CONSUMERS) {
      float v[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = i0 + j * CONSUMERS < cells ? __ldcg(p.part_logits + i0 + j * CONSUMERS) : 0.f;
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (i0 + j * CONSUMERS < cells) logits[i0 + j * CONSUMERS] = v[j];
    }
  }
  for (int i = threadIdx.x + (p.csplit == 1 ? cells : 0); i < cells + p.F; i += CONSUMERS) {
    const float* from = i < cells ? p.part_logits + i : p.part_sq + (i - cells);
    const int step = i < cells ? cells : p.F;
    float part[MAX_CSPLIT];
#pragma unroll
    for (int s = 0; s < MAX_CSPLIT; ++s) part[s] = s < p.csplit ? __ldcg(from + (long long)s * step) : 0.f;
    float v = 0.f;
#pragma unroll
    for (int s = 0; s < MAX_CSPLIT; ++s) v += part[s];
    if (i < cells) logits[i] = v;
    else {
      const float rstd = rsqrtf(v / float(p.C) + p.eps);
      L.rstd[i - cells] = rstd;
      L.gain[i - cells] = p.up_scale ? rstd * __ldcg(p.gain + i - cells) : rstd;
    }
  }
  consumer_sync();
  if (p.E <= 32) choose<1>(p, L, logits);
  else if (p.E <= 64) choose<2>(p, L, logits);
  else if (p.E <= 128) choose<4>(p, L, logits);
  else choose<8>(p, L, logits);
  consumer_sync();
  if (warp == 0) {
    int active = 0, rows = 0;
    for (int e0 = 0; e0 < n; e0 += 32) {
      const int e = e0 + lane;
      const int c = e < n ? __popcll(L.mask[e]) : 0;
      const uint32_t have = __ballot_sync(0xffffffffu, c > 0);
      int incl = c;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += v;
      }
      if (c > 0) {
        const int a = active + __popc(have & ((1u << lane) - 1u));
        L.expert[a] = short(e);
        L.base[a] = short(rows + incl - c);
      }
      active += __popc(have);
      rows += __shfl_sync(0xffffffffu, incl, 31);
    }
    if (lane == 0) {
      L.n_active = active;
      L.base[active] = short(rows);
    }
  }
  consumer_sync();
  for (int a = threadIdx.x; a < L.n_active; a += CONSUMERS) {
    const int e = L.expert[a];
    unsigned long long m = L.mask[e];
    for (int r = L.base[a]; m; ++r, m &= m - 1) {
      const int f = __ffsll(m) - 1;
      float s = 1.f;
      if (e < p.E)
        for (int j = 0; j < p.k; ++j)
          if (L.chosen[f * 8 + j] == e) s = L.chosen_score[f * 8 + j];
      L.tok[r] = (unsigned char)f;
      L.score[r] = s;
    }
  }
}

// ------------------------------------------------------------------------------------------------ the ring
struct Ring {
  uint32_t stages_addr;            // shared address of stage 0: [weights 32 KB | activations | e4m3: scales]
  uint32_t full, empty;            // barrier arrays
  int stage_bytes, n;
  int s = 0;
  uint32_t ph = 0;
  __device__ void next() {
    if (++s == n) { s = 0; ph ^= 1; }
  }
};

// A bounded wait ran out: record it and go on. Every later wait of the CTA then returns at once, no copy is started any more, and
// all warps keep walking the same sequence of barriers to the end of the kernel (its outputs are void, the status word says so).
struct Giveup {
  volatile int* flag;
  int* status;
  __device__ void operator()(int code) const {
    if ((threadIdx.x & 31) == 0) {
      *flag = 1;
      atomicCAS(status, 0, code);
    }
  }
};

// A unit of weights in shared memory: boxes of 128-byte rows (128B swizzle), 64 bf16 or 128 e4m3 columns wide and KT rows high.
// Tile j of warp w (16 columns): bf16 box 2j + w / 4, columns 16 (w % 4); e4m3 box j, columns 16 w.
template <bool FP8>
struct Geo {
  static constexpr int KT = FP8 ? 128 : 64;        // input rows per unit
  static constexpr int BOX = KT * 128;             // bytes of a box
};

// Rows [0, rows) of the activation piece of a unit: KT values each, in KT / 64 tiles of 128-byte rows with the 128B swizzle.
template <bool FP8, class RowPtr>
__device__ __forceinline__ void load_acts(uint32_t dst, int lane, int rows, int rows_pad, int k0, int K, RowPtr row_ptr) {
  constexpr int CH = Geo<FP8>::KT / 8;             // 16-byte chunks per row
  for (int i = lane; i < rows * CH; i += 32) {
    const int r = i / CH, c = i % CH;
    const uint16_t* src = row_ptr(r);
    const int kk = k0 + c * 8;
    const bool in = kk < K;                        // K is a multiple of 8; the rest of the last unit is zero, like the weights there
    cp16(dst + (c >> 3) * rows_pad * 128 + swz128(r, c & 7), src + (in ? kk : 0), in ? 16 : 0);
  }
}

// n_units units of one expert through the ring: two tiles of 16 weight columns times NT * 8 tokens, in fp32. e4m3: every k-16 product
// gets a fresh accumulator and joins the total with the scale of its block (a table in the stage, [column group of 16][k-16 step]), so
// the loop has no branches at the block borders; such a branch after every MMA kept the conversions of neighbouring steps apart.
template <bool FP8, int NT>
__device__ __forceinline__ void multiply(Ring& ring, int n_units, int rows_pad, const Giveup& give, float (&tot)[2][NT][4]) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int t = 0; t < 2; ++t)
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) tot[t][i][j] = 0.f;
  const uint32_t w_off = FP8 ? 0u : uint32_t(warp >> 2) * Geo<FP8>::BOX;
  constexpr int TILE1 = (FP8 ? 1 : 2) * Geo<FP8>::BOX;
  constexpr int STEPS = Geo<FP8>::KT / 32;         // two k-16 MMAs per step and tile
  for (int u = 0; u < n_units; ++u) {
    if (!mbar_wait(ring.full + ring.s * 8, ring.ph, give.flag)) give(STATUS_TIMEOUT_FULL);
    const uint32_t stage = ring.stages_addr + ring.s * ring.stage_bytes, w = stage + w_off, xa = stage + W_STAGE;
    float sc[2][8];
    if (FP8) {
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const uint32_t at = stage + ring.stage_bytes - SCALE_STAGE + (t * 8 + warp) * 32;
        lds128(at, sc[t][0], sc[t][1], sc[t][2], sc[t][3]);
        lds128(at + 16, sc[t][4], sc[t][5], sc[t][6], sc[t][7]);
      }
    }
    auto fetch = [&](int st, uint32_t (&raw)[2][2][4]) {           // [tile][k-16 step (bf16)]
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        if (FP8) {
          ldsm4t(raw[t][0], w + t * TILE1 + swz128(st * 32 + lane, warp));
        } else {
#pragma unroll
          for (int h = 0; h < 2; ++h)
            ldsm4t(raw[t][h], w + t * TILE1 + swz128(st * 32 + h * 16 + ((lane >> 4) << 3) + (lane & 7), (warp & 3) * 2 + ((lane >> 3) & 1)));
        }
      }
    };
    auto fetch_rows = [&](int st, uint32_t (&b)[NT][4]) {
#pragma unroll
      for (int i = 0; i < NT; ++i) ldsm4(b[i], xa + (st >> 1) * rows_pad * 128 + i * 1024 + swz128(lane & 7, (st & 1) * 4 + (lane >> 3)));
    };
    auto operand = [&](const uint32_t (&raw)[2][2][4], uint32_t (&a)[2][2][4]) {       // [tile][k-16 step]
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        if (FP8) {
          // raw[j]: k = 8j + 2 (lane % 4) in the low half, k + 1 in the high half; columns 2 (lane / 4) and + 1 as the two bytes
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const uint32_t v = __byte_perm(raw[t][0][j], 0, 0x3120);
            a[t][j >> 1][(j & 1) * 2] = e4m3x2_to_f16x2(uint16_t(v & 0xffffu));
            a[t][j >> 1][(j & 1) * 2 + 1] = e4m3x2_to_f16x2(uint16_t(v >> 16));
          }
        } else {
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int j = 0; j < 4; ++j) a[t][h][j] = raw[t][h][j];
        }
      }
    };
    auto products = [&](int st, const uint32_t (&a)[2][2][4], const uint32_t (&b)[NT][4]) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int i = 0; i < NT; ++i) {
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            if (FP8) {
              float d[4];
              mma16816_f16(d, a[t][h], b[i][2 * h], b[i][2 * h + 1]);
#pragma unroll
              for (int j = 0; j < 4; ++j) tot[t][i][j] = fmaf(d[j], sc[t][(st * 2 + h) & 7], tot[t][i][j]);
            } else {
              mma16816(tot[t][i], a[t][h], b[i][2 * h], b[i][2 * h + 1]);
            }
          }
        }
      }
    };
    if (FP8 && NT <= 2) {
      // Few rows: all of the unit goes through the conversion into registers, the stage is given back, then come the products. With
      // 64 tokens the ring has three stages; held for the whole of a unit, one of them was missing in flight.
      uint32_t a[STEPS][2][2][4], b[STEPS][NT][4];
#pragma unroll
      for (int st = 0; st < STEPS; ++st) {
        uint32_t raw[2][2][4];
        fetch(st, raw);
        fetch_rows(st, b[st]);
        operand(raw, a[st]);
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(ring.empty + ring.s * 8);         // a release: the loads above come before it
      ring.next();
#pragma unroll
      for (int st = 0; st < STEPS; ++st) products(st, a[st], b[st]);
      continue;
    }
    uint32_t raw[2][2][2][4];                      // the weights one step ahead of the products
    fetch(0, raw[0]);
#pragma unroll
    for (int st = 0; st < STEPS; ++st) {
      uint32_t a[2][2][4], b[NT][4];
      fetch_rows(st, b);
      if (st + 1 < STEPS) fetch(st + 1, raw[(st + 1) & 1]);
      operand(raw[st & 1], a);
      products(st, a, b);
    }
    __syncwarp();
    if (lane == 0) mbar_arrive(ring.empty + ring.s * 8);
    ring.next();
  }
}

// ------------------------------------------------------------------------------------------------ the kernel
template <bool FP8>
struct Block {
  static constexpr int KT = Geo<FP8>::KT;
  const Params& p;
  Lists& L;
  Ring ring;
  float* buf;                       // [F][256] fp32: the tokens' sums of one panel of output columns (phase 3)
  Giveup give;
  int c, rows_pad;
  // A team of up_team (dn_team) CTAs has one run; its members take neighbouring panels of the same units. up_groups (dn_groups):
  // panels per matrix in teams; up_units (dn_units): units along the input.
  int G, up_team, up_groups, up_units, dn_team, dn_groups, dn_units;
  __device__ Runs up_runs() const { return Runs(L.n_active * up_groups * up_units, G / up_team); }
  __device__ Runs down_runs() const { return Runs(dn_groups * L.n_active * dn_units, G / dn_team); }

  // column of accumulator pair `second` of tile `t` inside the panel (the e4m3 path pairs neighbouring columns, see multiply())
  __device__ static int col(int t, int second) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    return t * 128 + warp * 16 + (FP8 ? 2 * (lane >> 2) + second : (lane >> 2) + 8 * second);
  }
  // A cut panel (units [q0, q0 + per)) is the first or the last of a team's run: slot 0 or 1 of the team's member.
  __device__ float* slot_of(const Runs& runs, int q0, int team, int size, int member) const {
    return p.slots + ((long long)(team * size + member) * 2 + (runs.begin(team) >= q0 ? 0 : 1)) * slot_rows(p.F) * PANEL;
  }
  // After this CTA's part is in its slot: true in the CTA that arrives last of the n that share the panel.
  __device__ bool arrive(int* counter, int n) {
    __threadfence();
    consumer_sync();
    if (threadIdx.x == 0) L.last = atomicAdd(counter, 1) == n - 1;
    consumer_sync();
    if (!L.last) return false;
    __threadfence();
    return true;
  }

  // Units [u, u + n) of the up-projection, all of expert slot `a` and panel `panel`.
  template <int NT>
  __device__ void up_segment(const Runs& runs, int a, int panel, int q0, int u, int n) {
    const int lane = threadIdx.x & 31;
    const int e = L.expert[a], base = L.base[a], cnt = L.base[a + 1] - base;
    float tot[2][NT][4];
    multiply<FP8, NT>(ring, n, rows_pad, give, tot);
    if (n < up_units) {                            // cut: every thread leaves its registers in the slot and picks up the same ones
      const int first = runs.owner(q0), last = runs.owner(q0 + up_units - 1), member = c % up_team;
      float* slot = slot_of(runs, q0, c / up_team, up_team, member) + threadIdx.x;
#pragma unroll
      for (int i = 0; i < 2 * NT * 4; ++i) __stcg(slot + i * CONSUMERS, tot[i / (NT * 4)][i / 4 % NT][i % 4]);
      if (!arrive(p.counters + e * up_groups * up_team + panel, last - first + 1)) return;
#pragma unroll
      for (int i = 0; i < 2 * NT * 4; ++i) tot[i / (NT * 4)][i / 4 % NT][i % 4] = 0.f;
      for (int k = first; k <= last; ++k) {
        const float* from = slot_of(runs, q0, k, up_team, member) + threadIdx.x;
#pragma unroll
        for (int i = 0; i < 2 * NT * 4; ++i) tot[i / (NT * 4)][i / 4 % NT][i % 4] += __ldcg(from + i * CONSUMERS);
      }
    }
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const int h = panel * 128 + col(0, s);
      if (h < p.H) {
        float bg = 0.f, bl = 0.f;
        if (p.up_bias) {
          bg = __ldg(p.up_bias + (long long)e * 2 * p.H + h);
          bl = __ldg(p.up_bias + (long long)e * 2 * p.H + p.H + h);
        }
#pragma unroll
        for (int i = 0; i < NT; ++i) {
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const int r = i * 8 + (lane & 3) * 2 + j;
            if (r < cnt) {
              const float gain = L.gain[L.tok[base + r]];
              float g = fmaf(gain, tot[0][i][2 * s + j], bg), l = fmaf(gain, tot[1][i][2 * s + j], bl);
              // comparisons keep a NaN where fminf / fmaxf would drop it
              g = g > p.limit ? p.limit : g;
              l = l > p.limit ? p.limit : (l < -p.limit ? -p.limit : l);
              const float act = (l + 1.f) * g / (1.f + exp2f(-p.beta * L2E * g));
              p.act[(long long)(base + r) * p.H + h] = FP8 ? __half_as_ushort(__float2half_rn(act * p.act_scale)) : __bfloat16_as_ushort(__float2bfloat16(act));
            }
          }
        }
      }
    }
  }
  // Units of expert slot `a` of the down-projection, weighted by the scores into the tokens' sums.
  template <int NT>
  __device__ void down_segment(int a, int panel, int k_unit, int n) {
    const int lane = threadIdx.x & 31;
    const int e = L.expert[a], base = L.base[a], cnt = L.base[a + 1] - base;
    float tot[2][NT][4];
    multiply<FP8, NT>(ring, n, rows_pad, give, tot);
#pragma unroll
    for (int t = 0; t < 2; ++t) {
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const int cc = col(t, s), g = panel * PANEL + cc;
        // the run that holds the expert's first unit of this panel adds its bias
        const float bias = k_unit == 0 && p.down_bias && g < p.C ? __ldg(p.down_bias + (long long)e * p.C + g) : 0.f;
#pragma unroll
        for (int i = 0; i < NT; ++i) {
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const int r = i * 8 + (lane & 3) * 2 + j;
            if (r < cnt) buf[L.tok[base + r] * PANEL + cc] += L.score[base + r] * fmaf(tot[t][i][2 * s + j], FP8 ? p.act_gain : 1.f, bias);
          }
        }
      }
    }
    __syncwarp();                                  // another lane adds to the same token for the next expert
  }

  __device__ void consume_up() {
    const Runs runs = up_runs();
    int u = runs.begin(c / up_team);
    const int end = runs.begin(c / up_team + 1);
    while (u < end) {
      const int q = u / up_units, q0 = q * up_units, n = min(end, q0 + up_units) - u, a = q / up_groups;
      const int panel = (q - a * up_groups) * up_team + c % up_team;
      const int cnt = L.base[a + 1] - L.base[a];
      if (cnt <= 8) up_segment<1>(runs, a, panel, q0, u, n);
      else if (cnt <= 16) up_segment<2>(runs, a, panel, q0, u, n);
      else if (cnt <= 32) up_segment<4>(runs, a, panel, q0, u, n);
      else up_segment<8>(runs, a, panel, q0, u, n);
      u += n;
    }
  }

  __device__ void consume_down() {
    const int per = L.n_active * dn_units, team = c / dn_team, member = c % dn_team;
    const Runs runs = down_runs();
    int u = runs.begin(team);
    const int end = runs.begin(team + 1);
    while (u < end) {
      const int group = u / per, q0 = group * per, stop = min(end, q0 + per), q = group * dn_team + member;
      const bool whole = stop - u == per;
      for (int i = threadIdx.x; i < p.F * PANEL; i += CONSUMERS) buf[i] = 0.f;
      consumer_sync();
      while (u < stop) {
        const int v = u - q0, a = v / dn_units, k_unit = v - a * dn_units, n = min(stop - u, dn_units - k_unit);
        const int cnt = L.base[a + 1] - L.base[a];
        if (cnt <= 8) down_segment<1>(a, q, k_unit, n);
        else if (cnt <= 16) down_segment<2>(a, q, k_unit, n);
        else if (cnt <= 32) down_segment<4>(a, q, k_unit, n);
        else down_segment<8>(a, q, k_unit, n);
        u += n;
      }
      consumer_sync();
      const int g = q * PANEL + int(threadIdx.x);                // 256 threads, 256 columns: thread and column go together
      if (g < p.C) {
        float* slot = slot_of(runs, q0, team, dn_team, member) + threadIdx.x;
        for (int t = 0; t < p.F; ++t) {
          if (whole) store_out((long long)t * p.C + g, buf[t * PANEL + threadIdx.x]);
          else __stcg(slot + t * PANEL, buf[t * PANEL + threadIdx.x]);
        }
      }
      consumer_sync();
    }
  }
  __device__ void store_out(long long at, float v) const {
    p.out[at] = __float2bfloat16(fmaf(p.residual_scale, v, __bfloat162float(p.x[at])));
  }
  struct Join {                                    // four neighbouring outputs of one token and the teams first .. last that share their panel
    const float* at[2];                            // in the slot of the first team; of a team for which the panel is the first of its run
    long long out;
    int first, last;
    uint2 x;
  };
  __device__ bool find(int i, Join& w) const {
    const int quads = p.C / 4, per = L.n_active * dn_units;      // C is a multiple of 8: four columns at a time stay inside a panel
    if (i >= p.F * quads) return false;
    const Runs runs = down_runs();
    const int t = i / quads, g = (i - t * quads) * 4, q = g / PANEL, group = q / dn_team, q0 = group * per;
    w.first = runs.owner(q0);
    w.last = runs.owner(q0 + per - 1);
    w.out = (long long)t * p.C + g;
    const int in_slot = t * PANEL + g % PANEL, member = q % dn_team;
    w.at[0] = slot_of(runs, q0, w.first, dn_team, member) + in_slot;
    w.at[1] = slot_of(runs, q0, w.first + 1, dn_team, member) + in_slot;       // the following teams begin inside the panel: slot 0 each
    w.x = *reinterpret_cast<const uint2*>(p.x + w.out);
    return true;
  }
  __device__ void join(const Join& w) const {
    if (w.first == w.last) return;
    float4 v = __ldcg(reinterpret_cast<const float4*>(w.at[0]));
    const long long step = (long long)dn_team * 2 * slot_rows(p.F) * PANEL;
#pragma unroll 8
    for (int k = 0; k < w.last - w.first; ++k) {
      const float4 part = __ldcg(reinterpret_cast<const float4*>(w.at[1] + k * step));
      v.x += part.x;
      v.y += part.y;
      v.z += part.z;
      v.w += part.w;
    }
    const uint32_t in[2] = {w.x.x, w.x.y};
    uint2 o;
    o.x = pack_bf16(fmaf(p.residual_scale, v.x, __uint_as_float(in[0] << 16)), fmaf(p.residual_scale, v.y, __uint_as_float(in[0] & 0xffff0000u)));
    o.y = pack_bf16(fmaf(p.residual_scale, v.z, __uint_as_float(in[1] << 16)), fmaf(p.residual_scale, v.w, __uint_as_float(in[1] & 0xffff0000u)));
    *reinterpret_cast<uint2*>(p.out + w.out) = o;
  }

  // ---- producer side. A cursor walks a run without divisions: a warp that issues a unit every few hundred cycles has no time for
  // them (with the divisions the producer, not the memory, set the pace: 98 us instead of 85 us for one token).
  struct Cursor {
    int a, group, k;
  };
  __device__ Cursor at_up(int u) const { return Cursor{u / up_units / up_groups, u / up_units % up_groups, u % up_units}; }
  __device__ Cursor at_down(int u) const {
    const int per = L.n_active * dn_units;
    return Cursor{u % per / dn_units, u / per, u % dn_units};
  }
  __device__ void advance(Cursor& w, bool down) const {
    if (down) {
      if (++w.k == dn_units) {
        w.k = 0;
        if (++w.a == L.n_active) { w.a = 0; ++w.group; }
      }
    } else if (++w.k == up_units) {
      w.k = 0;
      if (++w.group == up_groups) { w.group = 0; ++w.a; }
    }
  }
  // `n` units from `w` on: the weights (one lane) or the activations (a warp) of each into the next stage
  template <bool DOWN>
  __device__ void feed_weights(Ring& r, const CUtensorMap* map, Cursor& w, int n) const {
    const int up_cols = (2 * p.H + 15) / 16 * 16;  // a first column past the matrix, on a 16-byte boundary
    for (int i = 0; i < n; ++i) {
      if (!mbar_wait(r.empty + r.s * 8, r.ph ^ 1, give.flag)) give(STATUS_TIMEOUT_EMPTY);
      if (!*give.flag) {
        const uint32_t bar = r.full + r.s * 8, dst = r.stages_addr + r.s * r.stage_bytes;
        // columns past the matrix (the last panel, a team's surplus member) are out of bounds for the map: zeros without traffic
        const int e = L.expert[w.a], member = c % (DOWN ? dn_team : up_team), panel = w.group * (DOWN ? dn_team : up_team) + member;
        const int at = panel * (DOWN ? PANEL : 128), x0 = !DOWN && at >= p.H ? up_cols : at, x1 = DOWN ? x0 + 128 : p.H + at;
        mbar_expect_tx(bar, W_STAGE);
        tma_load_3d(dst, map, bar, x0, w.k * KT, e);
        if (!FP8) tma_load_3d(dst + Geo<FP8>::BOX, map, bar, x0 + 64, w.k * KT, e);
        tma_load_3d(dst + W_STAGE / 2, map, bar, x1, w.k * KT, e);
        if (!FP8) tma_load_3d(dst + W_STAGE / 2 + Geo<FP8>::BOX, map, bar, x1 + 64, w.k * KT, e);
      }
      advance(w, DOWN);
      r.next();
    }
  }
  template <bool DOWN>
  __device__ void feed_rows(Ring& r, Cursor& w, int n) const {
    const int lane = threadIdx.x & 31;
    // e4m3: this lane's column group (of 16; tile lane / 8 % 2, warp lane % 8) of the scale table and its first k-16 step
    const int K = DOWN ? p.H : p.C, N = DOWN ? p.C : 2 * p.H, bk = DOWN ? p.dn_bk : p.up_bk, bn = DOWN ? p.dn_bn : p.up_bn;
    const int n_kb = FP8 ? K / bk : 0, n_nb = FP8 ? N / bn : 0;
    const float per_bk = 1.f / float(bk);
    const float* scales = nullptr;
    int scales_a = -1, scales_group = -1;
    for (int i = 0; i < n; ++i) {
      if (!mbar_wait(r.empty + r.s * 8, r.ph ^ 1, give.flag)) give(STATUS_TIMEOUT_EMPTY);
      __syncwarp();
      if (!*give.flag) {
        const uint32_t dst = r.stages_addr + r.s * r.stage_bytes + W_STAGE;
        const int base = L.base[w.a], cnt = L.base[w.a + 1] - base;
        if (FP8) {
          if (w.a != scales_a || w.group != scales_group) {
            scales_a = w.a;
            scales_group = w.group;
            const int tile = (lane >> 3) & 1, wc = (lane & 7) * 16, panel = w.group * (DOWN ? dn_team : up_team) + c % (DOWN ? dn_team : up_team);
            const int col = DOWN ? panel * PANEL + tile * 128 + wc : tile * p.H + panel * 128 + wc;
            scales = (DOWN ? p.down_scale : p.up_scale) + (long long)L.expert[w.a] * n_kb * n_nb + min(col, N - 16) / bn;
          }
          const uint32_t table = r.stages_addr + (r.s + 1) * r.stage_bytes - SCALE_STAGE + (lane & 15) * 32;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int step = (lane >> 4) * 4 + j;
            // block of the step's first input: exact for inputs below 2^21 (the half keeps the product off the integers)
            const int kb = int((float(min(w.k * KT + step * 16, K - 16)) + 0.5f) * per_bk);
            cp4(table + step * 4, scales + (long long)min(kb, n_kb - 1) * n_nb);
          }
        }
        if (DOWN)
          load_acts<FP8>(dst, lane, cnt, rows_pad, w.k * KT, p.H, [&](int j) { return p.act + (long long)(base + j) * p.H; });
        else
          load_acts<FP8>(dst, lane, cnt, rows_pad, w.k * KT, p.C, [&](int j) { return p.xs + (long long)L.tok[base + j] * p.C; });
        cp_arrive(r.full + r.s * 8);
      }
      advance(w, DOWN);
      r.next();
    }
  }
};

template <bool FP8>
__global__ void __launch_bounds__(THREADS, 1)
moe_block_kernel(const __grid_constant__ CUtensorMap up_map, const __grid_constant__ CUtensorMap down_map, const Params p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int stage_bytes = W_STAGE + p.x_stage;
  uint8_t* after = smem + p.stages * stage_bytes;
  float* buf = reinterpret_cast<float*>(after);
  Lists& L = *reinterpret_cast<Lists*>(after + buf_bytes(p.F));
  __shared__ uint64_t full[MAX_STAGES], empty[MAX_STAGES];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int G = int(gridDim.x), c = int(blockIdx.x);
  constexpr int KT = Geo<FP8>::KT;
  cg::grid_group grid = cg::this_grid();

  Block<FP8> blk{p, L, Ring{smem_u32(smem), smem_u32(full), smem_u32(empty), stage_bytes, p.stages}, buf, Giveup{&L.abort, p.status}, c, (p.F + 7) / 8 * 8,
                 G, p.up_team, ((p.H + 127) / 128 + p.up_team - 1) / p.up_team, (p.C + KT - 1) / KT,
                 p.dn_team, ((p.C + PANEL - 1) / PANEL + p.dn_team - 1) / p.dn_team, (p.H + KT - 1) / KT};
  if (threadIdx.x == 0) {
    for (int s = 0; s < p.stages; ++s) {
      mbar_init(smem_u32(&full[s]), 1 + 32);       // the weights' expect_tx and one arrival per lane for its copies of activations
      mbar_init(smem_u32(&empty[s]), CONSUMERS / 32);
    }
    L.abort = 0;
    fence_mbar_init();
  }
  __syncthreads();

  // ---- phase 1
  if (warp < CONSUMERS / 32) {
    for (int e = threadIdx.x; e < p.E; e += CONSUMERS) L.bias[e] = p.router_bias ? __ldg(p.router_bias + e) : 0.f;
    const int n_counters = (p.E + p.shared) * blk.up_groups * blk.up_team;
    for (int i = c * CONSUMERS + threadIdx.x; i < n_counters; i += G * CONSUMERS) p.counters[i] = 0;
    if (FP8) {
      for (int t = G - 1 - c; t < p.F; t += G) operand_row_f16(p, t, buf);     // the CTAs with the fewest router tasks
    } else {
      for (int i = (G - 1 - c) * CONSUMERS + int(threadIdx.x); i < p.F * p.C; i += G * CONSUMERS)      // from the far end: the first CTAs have the router's tasks
        p.xs[i] = __bfloat16_as_ushort(__float2bfloat16(__bfloat162float(__ldg(p.x + i)) * __ldg(p.norm + i % p.C)));
    }
    const int tasks = (p.E + RE - 1) / RE * ((p.F + RT - 1) / RT) * p.csplit;
    for (int t = c; t < tasks; t += G) router_task(p, t, buf);
  } else if (lane == 0) {
    tma_prefetch_desc(&up_map);
    tma_prefetch_desc(&down_map);
  }
  grid.sync();
  if (warp < CONSUMERS / 32) route(p, L, buf);
  __syncthreads();

  // ---- phases 2 and 3
  const Runs up_runs = blk.up_runs(), down_runs = blk.down_runs();
  const int b2 = up_runs.begin(c / p.up_team), n2 = up_runs.begin(c / p.up_team + 1) - b2;
  const int b3 = down_runs.begin(c / p.dn_team), n3 = down_runs.begin(c / p.dn_team + 1) - b3;
  if (warp == CONSUMERS / 32) {
    // weights: those of the first units of phase 3 need no barrier, they cross it in flight
    Ring r = blk.ring;
    const int early = min(p.stages, n3);
    auto w2 = blk.at_up(b2), w3 = blk.at_down(b3);
    if (lane == 0) {
      blk.template feed_weights<false>(r, &up_map, w2, n2);
      blk.template feed_weights<true>(r, &down_map, w3, early);
    }
    __syncwarp();
    grid.sync();
    if (lane == 0) blk.template feed_weights<true>(r, &down_map, w3, n3 - early);
    __syncwarp();
  } else if (warp == CONSUMERS / 32 + 1) {
    Ring r = blk.ring;
    auto w2 = blk.at_up(b2), w3 = blk.at_down(b3);
    blk.template feed_rows<false>(r, w2, n2);
    grid.sync();
    blk.template feed_rows<true>(r, w3, n3);
  } else {
    blk.consume_up();
    grid.sync();
    blk.consume_down();
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
  // the outputs of panels that run borders cut, summed in team order by all CTAs together (the CTA that happened to come last took
  // 75 us for it at 64 tokens); where they lie is found out before the barrier
  typename Block<FP8>::Join w;
  int i = c * THREADS + int(threadIdx.x);
  bool some = blk.find(i, w);
  grid.sync();
  while (some) {
    blk.join(w);
    some = blk.find(i += G * THREADS, w);
  }
  if (L.abort)
    for (int i = 0; i < 64; ++i) __nanosleep(1000);   // copies still in flight land before the shared memory is given back
}

template <bool FP8>
int launch(const CUtensorMap& up, const CUtensorMap& down, const Params& p, int grid, int smem, cudaStream_t stream) {
  static std::mutex lock;
  static int configured[64] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev >= 64) return -101;
  {
    std::lock_guard<std::mutex> guard(lock);
    if (smem > configured[dev]) {
      if (cudaFuncSetAttribute(moe_block_kernel<FP8>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess) return -102;
      configured[dev] = smem;
    }
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(THREADS);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeCooperative;
  attr[0].val.cooperative = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (cudaLaunchKernelEx(&cfg, moe_block_kernel<FP8>, up, down, p) != cudaSuccess) {
    LYRA_CHECK_LAUNCH();
    return -103;
  }
  return 0;
}

struct Plan {
  int grid, csplit, stages, x_stage, smem, up_team, dn_team;
  long long logits, sq, gain, xs, act, slots, counters, total;      // byte offsets into the workspace
};

// Grid, ring depth and workspace of a call: functions of the sizes alone.
inline Plan make_plan(int F, int C, int H, int E, int shared, int k, bool fp8) {
  Plan q;
  const int KT = fp8 ? 128 : 64, sms = sm_count();
  const long long chosen = (long long)(E < F * k ? E : F * k) + shared;
  const long long up_panels = (H + 127) / 128, dn_panels = (C + PANEL - 1) / PANEL;
  const long long u2 = chosen * up_panels * ((C + KT - 1) / KT), u3 = chosen * dn_panels * ((H + KT - 1) / KT);
  const long long want = ((u2 > u3 ? u2 : u3) + 1) / 2;        // two units per CTA at least: below that a barrier of more CTAs costs more
  q.grid = int(want < sms ? (want > 1 ? want : 1) : sms);
  if (q.grid > 4) q.grid = q.grid / 4 * 4;
  // Members per team: as many of 4, 2, 1 as divide the grid and leave at most a tenth of the members without a panel.
  auto team = [&](long long panels) {
    for (int t = 4; t > 1; t /= 2)
      if (q.grid % t == 0 && (panels + t - 1) / t * t * 10 <= panels * 11) return t;
    return 1;
  };
  q.up_team = team(up_panels);
  q.dn_team = team(dn_panels);
  const int tasks = (E + RE - 1) / RE * ((F + RT - 1) / RT);
  q.csplit = q.grid / tasks;
  if (q.csplit > MAX_CSPLIT) q.csplit = MAX_CSPLIT;
  if (q.csplit > C / 128) q.csplit = C / 128;
  if (q.csplit < 1) q.csplit = 1;
  q.x_stage = (F + 7) / 8 * 8 * 128 * (KT / 64) + (fp8 ? SCALE_STAGE : 0);
  const int fixed = 1024 + buf_bytes(F) + int(sizeof(Lists));
  q.stages = (232448 - 1024 - fixed) / (W_STAGE + q.x_stage);  // 227 KB per CTA; the barriers are static
  if (q.stages > MAX_STAGES) q.stages = MAX_STAGES;
  q.smem = fixed + q.stages * (W_STAGE + q.x_stage);
  long long at = 0;
  auto take = [&](long long bytes) { const long long here = at; at += (bytes + 255) / 256 * 256; return here; };
  q.logits = take(4LL * q.csplit * F * E);
  q.sq = take(4LL * q.csplit * F);
  q.gain = take(4LL * F);
  q.xs = take(2LL * F * C);
  q.act = take(2LL * F * (k + shared) * H);
  q.slots = take(4LL * q.grid * 2 * slot_rows(F) * PANEL);
  q.counters = take(4LL * (E + shared) * ((up_panels + q.up_team - 1) / q.up_team * q.up_team));
  q.total = at;
  return q;
}

}  // namespace moeblk
}  // namespace lyra

// Bytes of workspace a call needs (its contents need no initialisation), or a negative code for sizes the kernel does not take.
extern "C" long long lyra_moe_block_workspace(int F, int C, int H, int E, int shared, int k, int fp8) {
  using namespace lyra::moeblk;
  if (F < 1 || F > MAX_F || E < 1 || shared < 0 || E + shared > MAX_N || k < 1 || k > E || k + shared > 8) return -100;
  const int unit = fp8 ? 16 : 8;
  if (C < unit || H < unit || C % unit || H % unit || C > (1 << 20) || H > (1 << 20)) return -100;
  const long long chosen = (long long)(E < F * k ? E : F * k) + shared;
  if (chosen * ((H + 511) / 128) * ((C + 63) / 64) > (1LL << 30) || chosen * ((C + 1023) / 256) * ((H + 63) / 64) > (1LL << 30)) return -100;
  return make_plan(F, C, H, E, shared, k, fp8 != 0).total;
}

// x, out [F, C] bf16; up [n, C, 2H], down [n, H, C] bf16 or e4m3 with fp32 scales per (bk x bn) block; n = E + shared.
extern "C" int lyra_moe_block(const void* x, const float* norm, float eps, const float* router, const float* router_bias, const void* up, const float* up_scale,
                              int up_bk, int up_bn, const float* up_bias, const void* down, const float* down_scale, int dn_bk, int dn_bn,
                              const float* down_bias, void* out, float* scores, long long* idx, void* workspace, long long workspace_bytes, int F, int C, int H, int E,
                              int shared, int k, int fp8, float beta, float limit, float residual_scale, int* status, cudaStream_t stream) {
  using namespace lyra;
  using namespace lyra::moeblk;
  const long long need = lyra_moe_block_workspace(F, C, H, E, shared, k, fp8);
  if (need < 0 || workspace_bytes < need) return -100;
  if (fp8 && !(limit >= 0.f && limit <= 1e4f && beta >= 2.8e-5f)) return -100;      // the fp16 operand's range is fitted to them
  if (fp8 && (!up_scale || !down_scale || up_bk % 16 || up_bn % 16 || dn_bk % 16 || dn_bn % 16 || up_bk < 16 || up_bn < 16 || dn_bk < 16 || dn_bn < 16 ||
              C % up_bk || (2 * H) % up_bn || H % dn_bk || C % dn_bn))
    return -100;
  const uintptr_t aligned = reinterpret_cast<uintptr_t>(up) | reinterpret_cast<uintptr_t>(down) | reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(out) |
                            reinterpret_cast<uintptr_t>(workspace);
  if (aligned & 15) return -100;
  const Plan q = make_plan(F, C, H, E, shared, k, fp8 != 0);
  const uint64_t n = uint64_t(E + shared), esz = fp8 ? 1 : 2;
  const CUtensorMapDataType dt = fp8 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  const CUtensorMapSwizzle swz = CU_TENSOR_MAP_SWIZZLE_128B;
  const uint32_t box[3] = {uint32_t(fp8 ? 128 : 64), uint32_t(fp8 ? 128 : 64), 1};
  // 256 bytes of a bf16 row are asked for together; of an e4m3 row of W_up it is 128, and fetching the other half of a 256-byte
  // block early pushes as much out of L2 before it is used (2.9 instead of 3.7 TB/s with narrower boxes)
  const CUtensorMapL2promotion promo = fp8 ? CU_TENSOR_MAP_L2_PROMOTION_L2_128B : CU_TENSOR_MAP_L2_PROMOTION_L2_256B;
  CUtensorMap um, dm;
  const uint64_t ud[3] = {uint64_t(2 * H), uint64_t(C), n}, us[2] = {uint64_t(2 * H) * esz, uint64_t(2 * H) * C * esz};
  const uint64_t dd[3] = {uint64_t(C), uint64_t(H), n}, ds[2] = {uint64_t(C) * esz, uint64_t(C) * H * esz};
  if (make_tmap_cached(&um, up, dt, 3, ud, us, box, swz, promo)) return -104;
  if (make_tmap_cached(&dm, down, dt, 3, dd, ds, box, swz, promo)) return -104;
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  Params p;
  p.x = static_cast<const __nv_bfloat16*>(x);
  p.norm = norm;
  p.router = router;
  p.router_bias = router_bias;
  p.up_scale = up_scale;
  p.down_scale = down_scale;
  p.up_bias = up_bias;
  p.down_bias = down_bias;
  p.out = static_cast<__nv_bfloat16*>(out);
  p.scores = scores;
  p.idx = idx;
  p.part_logits = reinterpret_cast<float*>(ws + q.logits);
  p.part_sq = reinterpret_cast<float*>(ws + q.sq);
  p.gain = reinterpret_cast<float*>(ws + q.gain);
  p.xs = reinterpret_cast<uint16_t*>(ws + q.xs);
  p.act = reinterpret_cast<uint16_t*>(ws + q.act);
  p.slots = reinterpret_cast<float*>(ws + q.slots);
  p.counters = reinterpret_cast<int*>(ws + q.counters);
  p.status = status;
  p.F = F; p.C = C; p.H = H; p.E = E; p.shared = shared; p.k = k;
  p.csplit = q.csplit; p.stages = q.stages; p.x_stage = q.x_stage; p.up_team = q.up_team; p.dn_team = q.dn_team;
  p.up_bk = up_bk; p.up_bn = up_bn; p.dn_bk = dn_bk; p.dn_bn = dn_bn;
  p.eps = eps; p.beta = beta; p.limit = limit; p.residual_scale = residual_scale;
  int halvings = 0;                                            // that bring the SwiGLU result's bound below fp16's 65504
  const double gate = limit * double(beta) > 0.279 ? limit : 0.279 / double(beta);
  while (fp8 && double(limit + 1.f) * gate > 60000.0 * exp2(halvings)) ++halvings;
  p.act_scale = float(exp2(-halvings));
  p.act_gain = float(exp2(halvings));
  return fp8 ? launch<true>(um, dm, p, q.grid, q.smem, stream) : launch<false>(um, dm, p, q.grid, q.smem, stream);
}
