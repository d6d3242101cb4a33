// Attention of a batch whose sequences share a prefix: every sequence's queries see the prefix's keys (stored once) and its own.
//
//   out = (sum_j e^{s_j} v_j) / (sum_j e^{s_j} + e^{sink}),  j over the visible prefix positions and the visible own positions
//
// A softmax over two sets of keys is the merge of two partial softmaxes (maximum, sum, unnormalised output), so the work is split
// where the reuse changes:
//
//   prefix_kernel  the rows of all sequences (and of the query heads that share a kv head) against the prefix. Per kv head this is a
//                  dense product of M = B * T * rep rows with P keys: 128-row tiles on tcgen05 with accumulators in TMEM, keys read once
//                  per row tile. Few row tiles: the key axis is split so that every SM has work.
//   own_kernel     each sequence against its own cache: no reuse beyond the rep heads, bound by reading the cache, so warp MMAs with
//                  many bytes in flight. Its last step merges the prefix partials, its own and the sink, and rounds once.
//
// 64 query heads of 64 over 8 kv heads, bf16: 256 sequences behind 32768 shared positions with up to 1024 own ones 272 us, of which the
// prefix kernel has 218: the softmax (its exponentials and their issue, about 1450 clk per 128 x 128 tile and SM) bounds it, the tensor
// cores need 600 of them; the rest is the own caches at 4 TB/s. 64 sequences behind 8192 positions with up to 512: 40 us.
//
// Prefix kernel, per item (row tile, kv head, key split), one persistent CTA per SM:
//   warp 0        TMA producer: K and V tiles of 128 keys (bf16: straight into the operand tiles; e4m3: into a raw ring)
//   warp 1        tcgen05 issuer:  S = Q K_j^T  and, e4m3, O_g += P V_j   (g = j mod 2)
//   warp 10       bf16: issuer of O_g += P V_j, so that neither product's barriers hold up the other's instructions
//   warps 2..9    two softmax groups of four warps, alternate key tiles, one row per thread; each has its own scores, maximum, sum and
//                 accumulator, merged once per item. P replaces S in TMEM as packed bf16 and is the MMA's TMEM operand.
//   warp 11, e4m3: 10 and 11   gather the query rows (any strides) into the operand tile; e4m3: also turn raw K / V tiles into bf16
//                 operand tiles.
//                 That conversion is exact; a key's scale multiplies its score, a value's scale its probability, both in fp32.
#include <cooperative_groups.h>
#include <cuda_fp8.h>

#include "../common/sm100.cuh"
#include "../common/tmap.h"

namespace lyra {
namespace prefix {

namespace cg = cooperative_groups;

constexpr float L2E = 1.4426950408889634f;
constexpr int THREADS = 384;                    // warps 0, 1 | 2..9 | 10, 11
constexpr int BM = 128, BN = 128;               // rows and keys of a tile
constexpr int MAX_SPLITS = 32;
constexpr int POLY_AT = 6;                      // place in a run of eight scores of the pair that is exponentiated by polynomial
constexpr int SLOTS = 8;                        // scales of so many key tiles

struct Params {
  const __nv_bfloat16* q;                       // [B, Nq, T, D] by strides (in elements)
  long long q_sb, q_sn, q_st;
  const int* pos;                               // own positions before the new tokens, one per sequence (pos_n = B) or one for all
  int pos_n, pos_host;                          // pos == null: pos_host
  const float *pk_scale, *pv_scale;             // e4m3 prefix: [Nkv, P] with head strides
  long long pks_sh, pvs_sh;
  float* part_o;                                // [Nkv, row tiles, splits, D, 128] unnormalised: a column's rows side by side
  float2* part_ml;                              // [Nkv, row tiles, splits, 128] (maximum in log2 units, sum)
  int B, T, P, Nq, Nkv, rep, window, splits, key0;   // key0: first prefix position any row can see
  float scale_log2;
  int* status;
};

__device__ __forceinline__ int position(const int* pos, int n, int host, int b) { return pos ? __ldg(pos + (n == 1 ? 0 : b)) : host; }

struct Item {
  int m0, h, split, key, tiles;                 // first row, kv head, first key and number of key tiles
};

__device__ __forceinline__ void cp16(uint32_t dst, const void* src, int nbytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(nbytes) : "memory");
}
// Barrier of the loader warps that also tells all whether all are well: they leave together or not at all.
template <int LOADERS>
__device__ __forceinline__ bool loaders_agree(bool ok) {
  if (LOADERS == 32) return __all_sync(0xffffffffu, ok);
  uint32_t all;
  asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbar.red.and.pred q, 2, 64, p;\n\tselp.u32 %0, 1, 0, q;\n\t}" : "=r"(all) : "r"(uint32_t(ok)) : "memory");
  return all != 0;
}
// Two fp32 operations per instruction.
__device__ __forceinline__ uint64_t pair(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void unpair(uint64_t v, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
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
// 2^x of both halves without the special-function unit (16 results per clock and SM, 1024 clk for a 128 x 128 tile): x = n + f with n the
// nearest integer (adding 1.5 * 2^23 leaves it in the low bits), 2^f by the polynomial of degree 4 with the smallest largest relative
// error on [-1/2, 1/2] (2.7e-6, fitted by reweighted least squares), n added to the exponent. Inputs below -126 give 2^-126.
__device__ __forceinline__ uint64_t exp2_poly(uint64_t x) {
  float a, b;
  unpair(x, a, b);
  x = pair(fmaxf(a, -126.f), fmaxf(b, -126.f));
  const uint64_t magic = pair(12582912.f, 12582912.f), minus = pair(-12582912.f, -12582912.f), one = pair(-1.f, -1.f);
  const uint64_t t = add2(x, magic), f = fma2(add2(t, minus), one, x);
  uint64_t y = fma2(f, pair(0.009570079855620861f, 0.009570079855620861f), pair(0.05591783672571182f, 0.05591783672571182f));
  y = fma2(y, f, pair(0.240247443318367f, 0.240247443318367f));
  y = fma2(y, f, pair(0.6931217908859253f, 0.6931217908859253f));
  y = fma2(y, f, pair(0.9999992847442627f, 0.9999992847442627f));
  float ta, tb, ya, yb;
  unpair(t, ta, tb);
  unpair(y, ya, yb);
  return pair(__uint_as_float(__float_as_uint(ya) + (__float_as_uint(ta) << 23)), __uint_as_float(__float_as_uint(yb) + (__float_as_uint(tb) << 23)));
}
__device__ __forceinline__ bool elect_one() {
  uint32_t one;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(one));
  return one != 0;
}

template <int D, bool FP8>
struct Smem {
  static constexpr int TILE = 128 * D * 2, RAW_TILE = 128 * D;
  static constexpr int RAW = D == 64 ? 4 : 3;   // raw e4m3 tiles in flight (what 227 KB leave room for)
  // Score buffers in TMEM and stages of the K and V rings. Head dim 64: two accumulators leave room for a third score buffer, so the
  // scores of a group's next tile are ready when it finishes one; with two it waits for P V and Q K^T in between.
  static constexpr int NS = D == 64 ? 3 : 2;
  static constexpr int LOADERS = FP8 ? 64 : 32;
  static constexpr int BYTES = (1 + 2 * NS) * TILE + (FP8 ? RAW * RAW_TILE : 0) + 1024;
};

__device__ __forceinline__ uint32_t e4m3x2_to_bf16x2(uint16_t two) {      // exact
  const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(two, __NV_E4M3);
  const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h));
  return pack_bf16(f.x, f.y);
}

template <int D, bool FP8>
__global__ void __launch_bounds__(THREADS, 1)
prefix_kernel(const __grid_constant__ CUtensorMap tk, const __grid_constant__ CUtensorMap tv, const Params p) {
  constexpr int TILE = Smem<D, FP8>::TILE, RAW_TILE = Smem<D, FP8>::RAW_TILE, RAW = Smem<D, FP8>::RAW, NS = Smem<D, FP8>::NS, LOADERS = Smem<D, FP8>::LOADERS;
  constexpr int HALF = 128 * 128;               // bytes of one 64-column block of an operand tile
  constexpr uint32_t TMEM_COLS = 512, S_COL = 0, O_COL = NS * 128, O_COLS = NS == 3 ? 64 : 128;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");         // own_kernel may start wherever there is room
  constexpr uint32_t IDESC_S = make_idesc(BM, BN, 1, 1, 0, 0), IDESC_O = make_idesc(BM, D, 1, 1, 0, 1);

  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t *sQ = smem, *sK = sQ + TILE, *sV = sK + NS * TILE, *sR = sV + NS * TILE;
  __shared__ uint64_t q_full, q_empty, k_full[NS], v_empty[NS], s_full[NS], p_full[NS], o_full, o_empty, l_full;   // p_full: P and V are there
  __shared__ uint64_t raw_full[RAW], raw_empty[RAW], sc_full[SLOTS];
  __shared__ float xm[2][2][BM], xl[2][2][BM];  // [item parity][group][row]
  __shared__ __align__(16) float ksc[FP8 ? SLOTS : 1][BN], vsc[FP8 ? SLOTS : 1][BN];   // scales of the key tiles in flight
  __shared__ long long q_row[BM];
  __shared__ uint32_t tmem_holder;
  __shared__ int abort_flag;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int M = p.B * p.T * p.rep, n_mt = (M + BM - 1) / BM;
  const int n_tiles = (p.P - p.key0 + BN - 1) / BN;
  const int n_items = n_mt * p.Nkv * p.splits;

  // Items of a CTA: row tiles fastest, so that the CTAs running at the same time read the same keys.
  auto item_at = [&](int round, Item& it) -> bool {
    const int idx = round * int(gridDim.x) + int(blockIdx.x);
    if (idx >= n_items) return false;
    const int mt = idx % n_mt, rest = idx / n_mt;
    it.m0 = mt * BM;
    it.h = rest % p.Nkv;
    it.split = rest / p.Nkv;
    const int t0 = int((long long)n_tiles * it.split / p.splits), t1 = int((long long)n_tiles * (it.split + 1) / p.splits);
    it.key = p.key0 + t0 * BN;
    it.tiles = t1 - t0;
    return true;
  };

  if (threadIdx.x == 0) {
    mbar_init(smem_u32(&q_full), LOADERS);
    mbar_init(smem_u32(&q_empty), 1);
    for (int s = 0; s < NS; ++s) {
      mbar_init(smem_u32(&k_full[s]), FP8 ? LOADERS : 1);
      mbar_init(smem_u32(&v_empty[s]), 1);
      mbar_init(smem_u32(&s_full[s]), 1);
      mbar_init(smem_u32(&p_full[s]), 128 + (FP8 ? LOADERS : 1));
    }
    for (int s = 0; s < RAW; ++s) {
      mbar_init(smem_u32(&raw_full[s]), 1);
      mbar_init(smem_u32(&raw_empty[s]), LOADERS);
    }
    for (int s = 0; s < SLOTS; ++s) mbar_init(smem_u32(&sc_full[s]), LOADERS);
    mbar_init(smem_u32(&l_full), 256);
    mbar_init(smem_u32(&o_full), 1);
    mbar_init(smem_u32(&o_empty), 256);
    abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(&tmem_holder), TMEM_COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = __shfl_sync(0xffffffffu, tmem_holder, 0);
  volatile int* abortp = &abort_flag;
  Item w;

  // Counters that run across the items (every role advances its own copies the same way; every item has at least one key tile):
  //   t   key tiles so far: stage t % NS of the K and V operand tiles, score buffer t % NS (s_full, p_full), slot t % 8 of the scales
  //   n   items so far: parity of q_full / q_empty / o_full / o_empty / l_full
  // s_full of a tile (its scores are done) also means that its K stage is free, v_empty (its P V is done) that O holds it.
  if (warp == 0) {
    if (lane == 0) {
      tma_prefetch_desc(&tk);
      tma_prefetch_desc(&tv);
      uint32_t t = 0;
      bool ok = true;
      for (int round = 0; ok && item_at(round, w); ++round) {
        for (int j = 0; ok && j < w.tiles; ++j, ++t) {
          const int k0 = w.key + j * BN;
          if (FP8) {
            for (int which = 0; ok && which < 2; ++which) {
              const uint32_t i = 2 * t + which, s = i % RAW;
              if (!mbar_wait(smem_u32(&raw_empty[s]), ((i / RAW) & 1) ^ 1, abortp)) { ok = false; break; }
              mbar_expect_tx(smem_u32(&raw_full[s]), RAW_TILE);
              tma_load_3d(smem_u32(sR + s * RAW_TILE), which ? &tv : &tk, smem_u32(&raw_full[s]), 0, k0, w.h);
            }
          } else {
            const uint32_t s = t % NS, ph = (t / NS) & 1;
            if (!mbar_wait(smem_u32(&s_full[s]), ph ^ 1, abortp)) { ok = false; break; }      // scores done = K stage free
            mbar_expect_tx(smem_u32(&k_full[s]), TILE);
            for (int c = 0; c < D / 64; ++c) tma_load_3d(smem_u32(sK + s * TILE + c * HALF), &tk, smem_u32(&k_full[s]), c * 64, k0, w.h);
            if (!mbar_wait(smem_u32(&v_empty[s]), ph ^ 1, abortp)) { ok = false; break; }
            mbar_expect_tx(smem_u32(&p_full[s]), TILE);
            for (int c = 0; c < D / 64; ++c) tma_load_3d(smem_u32(sV + s * TILE + c * HALF), &tv, smem_u32(&p_full[s]), c * 64, k0, w.h);
          }
        }
      }
      if (!ok) {
        atomicCAS(p.status, 0, STATUS_TIMEOUT_EMPTY);
        abort_flag = 1;
      }
    }
  } else if (warp == 1 || (!FP8 && warp == 10)) {
    // A whole warp walks the tiles and one elected lane issues: the loop's values are then the same in all lanes for the compiler
    // too and live in uniform registers, from which the MMA takes its descriptors. (With the loop itself inside `lane == 0`, moving
    // them there took most of 2000 clk per tile; the tensor core needs about 600 for it.)
    const bool scores = warp == 1, outputs = FP8 || warp == 10;
    uint32_t n = 0, ks = 0, kph = 0, vs = 0, vph = 0;       // stage and parity of the next K tile (scores) and of the next V tile
    bool ok = true;
    const uint64_t dq0 = make_smem_desc(smem_u32(sQ), 16, 1024), dk0 = make_smem_desc(smem_u32(sK), 16, 1024);
    const uint64_t dv0 = make_smem_desc(smem_u32(sV), HALF, 1024);
    auto issue_s = [&](bool last) -> bool {
      if (!mbar_wait(smem_u32(&k_full[ks]), kph, abortp)) return false;
      if (!outputs && !mbar_wait(smem_u32(&v_empty[ks]), kph ^ 1, abortp)) return false;   // the buffer's P has been read (own MMAs retire in order)
      tc_fence_after();
      if (elect_one()) {
        const uint64_t dk = desc_advance(dk0, ks * TILE);
#pragma unroll
        for (int k = 0; k < D / 16; ++k)
          tc_mma_ss(tmem + S_COL + ks * 128, desc_advance(dq0, (k / 4) * HALF + (k % 4) * 32), desc_advance(dk, (k / 4) * HALF + (k % 4) * 32), IDESC_S, k > 0);
        tc_commit(smem_u32(&s_full[ks]));
        if (last) tc_commit(smem_u32(&q_empty));
      }
      __syncwarp();
      if (++ks == NS) { ks = 0; kph ^= 1; }
      return true;
    };
    auto issue_o = [&](int j, bool last) -> bool {
      if (!mbar_wait(smem_u32(&p_full[vs]), vph, abortp)) return false;
      tc_fence_after();
      if (elect_one()) {
        const uint64_t dv = desc_advance(dv0, vs * TILE);
#pragma unroll
        for (int k = 0; k < BN / 16; ++k)
          tc_mma_ts(tmem + O_COL + (j & 1) * O_COLS, tmem + S_COL + vs * 128 + k * 8, desc_advance(dv, k * 2048), IDESC_O, (j >= 2 || k > 0) ? 1u : 0u);
        tc_commit(smem_u32(&v_empty[vs]));
        if (last) tc_commit(smem_u32(&o_full));
      }
      __syncwarp();
      if (++vs == NS) { vs = 0; vph ^= 1; }
      return true;
    };
    for (int round = 0; ok && item_at(round, w); ++round, ++n) {
      if (scores) ok = mbar_wait(smem_u32(&q_full), n & 1, abortp);
      if (scores && !outputs) {
        for (int j = 0; j < w.tiles && ok; ++j) ok = issue_s(j == w.tiles - 1);
        continue;
      }
      if (scores)
        for (int j = 0; ok && j < NS && j < w.tiles; ++j) ok = issue_s(j == w.tiles - 1);
      if (ok) ok = mbar_wait(smem_u32(&o_empty), (n & 1) ^ 1, abortp);       // the previous item's output has been read
      for (int j = 0; j < w.tiles && ok; ++j) {
        ok = issue_o(j, j == w.tiles - 1);
        if (scores && ok && j + NS < w.tiles) ok = issue_s(j + NS == w.tiles - 1);
      }
    }
    if (!ok) {
      if (lane == 0) atomicCAS(p.status, 0, STATUS_TIMEOUT_FULL);
      abort_flag = 1;
    }
  } else if (warp >= 10) {
    // ------------------------------------------------------------ query rows; e4m3 tiles to bf16
    const int tid = threadIdx.x - (THREADS - LOADERS);
    constexpr int CPR = D / 8;                  // 16-byte chunks per query row
    uint32_t t = 0, n = 0;
    bool ok = true;
    for (int round = 0; item_at(round, w); ++round, ++n) {
#pragma unroll
      for (int r = tid; r < BM; r += LOADERS) {              // where each row of the item starts, in elements; -1: past the last row
        const int m = w.m0 + r, bt = m / p.rep, b = bt / p.T;
        q_row[r] = m < M ? b * p.q_sb + (long long)(w.h * p.rep + m - bt * p.rep) * p.q_sn + (long long)(bt - b * p.T) * p.q_st : -1;
      }
      if (!(ok = loaders_agree<LOADERS>(ok))) break;
      if (!mbar_wait(smem_u32(&q_empty), (n & 1) ^ 1, abortp)) ok = false;
      if (ok) {
#pragma unroll 4
        for (int i = tid; i < BM * CPR; i += LOADERS) {
          const int r = i / CPR, c = i % CPR;
          const long long at = q_row[r];
          cp16(smem_u32(sQ + (c >> 3) * HALF + swz128(r, c & 7)), p.q + (at < 0 ? 0 : at + c * 8), at < 0 ? 0 : 16);
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
      }
      if (!(ok = loaders_agree<LOADERS>(ok))) break;                  // the table is rewritten for the next item after this
      fence_proxy_async_smem();
      mbar_arrive(smem_u32(&q_full));
      if (FP8) {
        for (int j = 0; ok && j < w.tiles; ++j, ++t) {
          const uint32_t s = t % NS, ph = (t / NS) & 1;
          const int k0 = w.key + j * BN;
          // slot t % 8 is free: the stage of tile t is, so the scores of tile t - NS are done; they were asked for after the
          // probabilities of tile t - 2 NS, and those came after the group was through with tile t - 8
#pragma unroll 1
          for (int which = 0; which < 2; ++which) {
            const uint32_t i = 2 * t + which, rs = i % RAW;
            if (!mbar_wait(smem_u32(which ? &v_empty[s] : &s_full[s]), ph ^ 1, abortp) || !mbar_wait(smem_u32(&raw_full[rs]), (i / RAW) & 1, abortp)) {
              ok = false;
              break;
            }
            const uint8_t* from = sR + rs * RAW_TILE;
            uint8_t* to = (which ? sV : sK) + s * TILE;
            constexpr int RC = D / 16;          // 16-byte chunks per raw row
#pragma unroll 2
            for (int x = tid; x < BN * RC; x += LOADERS) {
              const int r = x / RC, c = x % RC;
              const uint4 v = *reinterpret_cast<const uint4*>(from + x * 16);
              const uint32_t in[4] = {v.x, v.y, v.z, v.w};
              uint32_t o[8];
#pragma unroll
              for (int y = 0; y < 4; ++y) {
                o[2 * y] = e4m3x2_to_bf16x2(uint16_t(in[y] & 0xffffu));
                o[2 * y + 1] = e4m3x2_to_bf16x2(uint16_t(in[y] >> 16));
              }
              uint8_t* dst = to + (c >> 2) * HALF;
              *reinterpret_cast<uint4*>(dst + swz128(r, (c & 3) * 2)) = make_uint4(o[0], o[1], o[2], o[3]);
              *reinterpret_cast<uint4*>(dst + swz128(r, (c & 3) * 2 + 1)) = make_uint4(o[4], o[5], o[6], o[7]);
            }
            if (which == 0) {
#pragma unroll
              for (int y = 0; y < BN / LOADERS; ++y) {
                const int key = k0 + tid + y * LOADERS;
                const bool in = key < p.P;      // 1 past the end: those scores are masked, -inf * 0 would not be -inf
                ksc[t % SLOTS][tid + y * LOADERS] = in ? __ldg(p.pk_scale + w.h * p.pks_sh + key) * p.scale_log2 : 1.f;
                vsc[t % SLOTS][tid + y * LOADERS] = in ? __ldg(p.pv_scale + w.h * p.pvs_sh + key) : 1.f;
              }
              mbar_arrive(smem_u32(&sc_full[t % SLOTS]));
            }
            fence_proxy_async_smem();
            mbar_arrive(smem_u32(&raw_empty[rs]));
            mbar_arrive(smem_u32(which ? &p_full[s] : &k_full[s]));
          }
        }
      }
    }
    if (!ok) {
      if (lane == 0) atomicCAS(p.status, 0, STATUS_TIMEOUT_EMPTY);
      abort_flag = 1;
    }
  } else {
    // ------------------------------------------------------------ softmax and epilogue
    const int quarter = warp & 3;
    const int row = quarter * 32 + lane;        // row of the tile == TMEM lane
    const uint32_t lane_addr = uint32_t(quarter * 32) << 16;
    const int g = (warp - 2) >> 2;              // group 0: key tiles 0, 2, ...; group 1: 1, 3, ...
    const uint32_t o_addr = tmem + lane_addr + O_COL + g * O_COLS;
    const float sc = p.scale_log2;
    uint32_t t = 0, n = 0;
    bool failed = false;

    for (int round = 0; !failed && item_at(round, w); ++round) {
      const int m_row = w.m0 + row;
      const bool row_valid = m_row < M, warp_idle = w.m0 + quarter * 32 >= M;
      const int bt = m_row / p.rep, b = bt / p.T;
      const int lo = p.window > 0 && row_valid ? p.P + position(p.pos, p.pos_n, p.pos_host, b) + (bt - b * p.T) - p.window + 1 : 0;   // first visible key
      float m = -INFINITY, l = 0.f;

      for (int j = g; j < w.tiles; j += 2) {
        const int k0 = w.key + j * BN;
        const uint32_t slot = (t + j) % SLOTS, sb = (t + j) % NS;
        const uint32_t s_addr = tmem + lane_addr + S_COL + sb * 128;
        if (FP8 && !mbar_wait(smem_u32(&sc_full[slot]), ((t + j) / SLOTS) & 1, abortp)) { failed = true; break; }
        if (!mbar_wait(smem_u32(&s_full[sb]), ((t + j) / NS) & 1, abortp)) { failed = true; break; }
        tc_fence_after();
        if (!warp_idle) {                       // rows past the last one keep whatever their lanes hold: no other row sees it
          const bool need_mask = k0 + BN > p.P || (p.window > 0);
          // scores as they enter the softmax: times the key's scale (e4m3), -inf where the row must not look
          auto prepare = [&](int c, uint32_t (&r)[32]) {
            if (FP8) {
#pragma unroll
              for (int i = 0; i < 32; i += 4) {
                const float4 f = *reinterpret_cast<const float4*>(&ksc[slot][c * 32 + i]);
                r[i] = __float_as_uint(__uint_as_float(r[i]) * f.x);
                r[i + 1] = __float_as_uint(__uint_as_float(r[i + 1]) * f.y);
                r[i + 2] = __float_as_uint(__uint_as_float(r[i + 2]) * f.z);
                r[i + 3] = __float_as_uint(__uint_as_float(r[i + 3]) * f.w);
              }
            }
            if (need_mask) {
              const int from = lo - (k0 + c * 32), to = p.P - (k0 + c * 32);        // places [from, to) of the 32 are visible
              const uint32_t seen = (to >= 32 ? ~0u : to > 0 ? (1u << to) - 1u : 0u) & (from <= 0 ? ~0u : from < 32 ? ~0u << from : 0u);
#pragma unroll
              for (int i = 0; i < 32; ++i)
                if (!(seen >> i & 1u)) r[i] = 0xff800000u;
            }
          };
          const float s2 = FP8 ? 1.f : sc;      // e4m3: the softmax scale came in with the key's
          // A row without a reference yet (its first tile, or nothing visible so far) takes the tile's maximum first.
          if (__any_sync(0xffffffffu, m == -INFINITY)) {
            float mx = -INFINITY;
#pragma unroll 1
            for (int c = 0; c < 4; ++c) {
              uint32_t r[32];
              tmem_ld32(s_addr + c * 32, r);
              tmem_ld_wait();
              prepare(c, r);
#pragma unroll
              for (int i = 0; i < 32; ++i) mx = fmaxf(mx, __uint_as_float(r[i]));
            }
            if (m == -INFINITY) m = mx * s2;
          }
          // One pass in the common case: probabilities against the current reference while the tile's maximum is tracked; redone
          // (the scores are still in TMEM) when a row has to move its reference by more than 2^8. The next quarter of the scores is
          // on its way while one is exponentiated.
          float mx4[4];
          uint64_t sum2[2];
          uint32_t pk[2][32];
          float ref = m == -INFINITY ? 0.f : m;
          auto pass = [&]() {
            uint32_t r[2][32];
            const uint64_t scale2 = pair(s2, s2), ref2 = pair(-ref, -ref);
            sum2[0] = sum2[1] = pair(0.f, 0.f);
            tmem_ld32(s_addr, r[0]);
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              tmem_ld_wait();
              if (c < 3) tmem_ld32(s_addr + (c + 1) * 32, r[(c + 1) & 1]);
              prepare(c, r[c & 1]);
              mx4[c] = -INFINITY;
#pragma unroll
              for (int i = 0; i < 32; i += 2) {
                const float a = __uint_as_float(r[c & 1][i]), d = __uint_as_float(r[c & 1][i + 1]);
                mx4[c] = fmaxf(mx4[c], fmaxf(a, d));
                uint64_t x = fma2(pair(a, d), scale2, ref2);
                float p0, p1;
                if (i % 8 == POLY_AT) {         // a quarter of the exponentials: the special-function unit is what they queue for
                  x = exp2_poly(x);
                  unpair(x, p0, p1);
                } else {
                  unpair(x, p0, p1);
                  p0 = exp2f(p0);
                  p1 = exp2f(p1);
                  x = pair(p0, p1);
                }
                sum2[(i >> 1) & 1] = add2(sum2[(i >> 1) & 1], x);
                if (FP8) {
                  const float2 f = *reinterpret_cast<const float2*>(&vsc[slot][c * 32 + i]);
                  p0 *= f.x;
                  p1 *= f.y;
                }
                pk[c >> 1][(c & 1) * 16 + (i >> 1)] = pack_bf16(p0, p1);
              }
            }
          };
#pragma unroll 1                                 // one copy of the pass in the program (see the merge in own_kernel)
          for (int again = 0;; ++again) {
            pass();
            const float mx = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3])) * s2;
            if (again || !__any_sync(0xffffffffu, mx > ref + 8.f)) break;
            float factor = 1.f;
            if (mx > ref + 8.f) {
              factor = exp2f(ref - mx);
              m = ref = mx;
            }
            l *= factor;
            if (j >= 2) {                       // O_g holds tiles j - 2, j - 4, ...: wait until the last of them has been added
              if (!mbar_wait(smem_u32(&v_empty[(t + j - 2) % NS]), ((t + j - 2) / NS) & 1, abortp)) abort_flag = 1;
              tc_fence_after();
#pragma unroll 1
              for (int c = 0; c < D / 32; ++c) {
                uint32_t o[32];
                tmem_ld32(o_addr + c * 32, o);
                tmem_ld_wait();
#pragma unroll
                for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * factor);
                tmem_st32(o_addr + c * 32, o);
              }
            }
          }
          tmem_st32(s_addr, pk[0]);
          tmem_st32(s_addr + 32, pk[1]);
          tmem_st_wait();
          float sum_a, sum_b;
          unpair(add2(sum2[0], sum2[1]), sum_a, sum_b);
          l += sum_a + sum_b;
        }
        tc_fence_before();
        mbar_arrive(smem_u32(&p_full[sb]));
      }
      if (failed) break;
      t += w.tiles;

      // merge of the two groups -> the split's partial result
      const int par = n & 1;
      xm[par][g][row] = m;
      xl[par][g][row] = l;
      mbar_arrive(smem_u32(&l_full));
      if (!mbar_wait(smem_u32(&o_full), par, abortp)) { failed = true; break; }
      if (!mbar_wait(smem_u32(&l_full), par, abortp)) { failed = true; break; }
      tc_fence_after();
      const bool two = w.tiles > 1;
      const float m0 = xm[par][0][row], m1 = two ? xm[par][1][row] : -INFINITY;
      const float mt = fmaxf(m0, m1);
      const float a0 = m0 == -INFINITY ? 0.f : exp2f(m0 - mt), a1 = m1 == -INFINITY ? 0.f : exp2f(m1 - mt);
      const float lt = a0 * xl[par][0][row] + (two ? a1 * xl[par][1][row] : 0.f);
      const long long part = ((long long)w.h * n_mt + w.m0 / BM) * p.splits + w.split;
      if (!warp_idle) {
        float* dst = p.part_o + part * D * BM + row;         // the warp's 32 rows of one column make one 128-byte store
#pragma unroll 1
        for (int c = g; c < D / 32; c += 2) {                // each group writes half of the columns
          uint32_t r0[32], r1[32];
          tmem_ld32(tmem + lane_addr + O_COL + c * 32, r0);
          if (two) tmem_ld32(tmem + lane_addr + O_COL + O_COLS + c * 32, r1);
          tmem_ld_wait();
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            float v = __uint_as_float(r0[i]) * a0;
            if (two) v = fmaf(__uint_as_float(r1[i]), a1, v);
            dst[(c * 32 + i) * BM] = v;
          }
        }
        if (g == 0) p.part_ml[part * BM + row] = make_float2(mt, lt);
      }
      tc_fence_before();
      mbar_arrive(smem_u32(&o_empty));
      ++n;
    }
    if (failed) {
      if (lane == 0) atomicCAS(p.status, 0, STATUS_TIMEOUT_TMEM);
      abort_flag = 1;
    }
  }

  tc_fence_before();
  __syncthreads();
  if (abort_flag) {
    for (int i = 0; i < 64; ++i) __nanosleep(1000);
    __syncthreads();
  }
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, TMEM_COLS);
  }
}

// ------------------------------------------------------------------------------------------------ own keys and merge
constexpr int OWARPS = 4, OTHREADS = OWARPS * 32, OSTAGES = 2;

struct OwnParams {
  const __nv_bfloat16* q;
  long long q_sb, q_sn, q_st;
  const uint8_t *k, *v;                         // [B, Nkv, S, D] contiguous, bf16 or e4m3
  const float *k_scale, *v_scale;               // e4m3: [B, Nkv, S]
  const int* pos;
  int pos_n, pos_host;
  const float* sinks;                           // [Nq] or null
  const float* part_o;                          // prefix partials (splits > 0)
  const float2* part_ml;
  __nv_bfloat16* out;                           // [B, T, Nq, D]
  int B, T, S, Nq, Nkv, rep, window, splits, row_tiles, cluster, prefix_tiles;
  float scale_log2;
};

__device__ __forceinline__ void cp4(uint32_t dst, const void* src, int nbytes) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(nbytes) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
__device__ __forceinline__ void ldsm4t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// ROWS: 64 query rows per CTA, 16 per warp, all warps walk the same key tiles (several tokens per sequence: the tiles are shared).
// Otherwise at most 16 rows, and the warps (and the CTAs of a cluster) split the keys (one token: all bytes in flight at once).
template <int D, bool FP8, bool ROWS>
struct OwnGeo {
  static constexpr int TK = ROWS ? 2048 / D : 16;                // keys per tile; split keys: small rings, so that 12 to 16 warps fit an SM
  static constexpr int ROWB = D * 2 + 16;                        // padded operand row: ldmatrix rows fall in distinct banks
  static constexpr int TILE_B = TK * ROWB;
  static constexpr int RAW_B = FP8 ? TK * D : TILE_B;            // one K or V tile as it arrives
  static constexpr int STAGE_B = 2 * RAW_B + 2 * TK * 4;         // + scales
  static constexpr int RING_B = OSTAGES * STAGE_B + (FP8 ? 2 * TILE_B : 0);
  static constexpr int ROWS_CTA = ROWS ? 64 : 16;
  static constexpr int PITCH = D + 4;                            // floats per row of the partial results: rows start in different banks
  static constexpr int COMB_B = ROWS_CTA * PITCH * 4, WARP_O_B = ROWS ? 0 : OWARPS * 16 * PITCH * 4;
  static constexpr int RINGS_B = (ROWS ? 1 : OWARPS) * RING_B;
  static constexpr int SMEM_B = RINGS_B > COMB_B + WARP_O_B ? RINGS_B : COMB_B + WARP_O_B;
};

template <int D, bool FP8, bool ROWS>
__global__ void __launch_bounds__(OTHREADS, D == 64 ? 4 : 3) own_kernel(const OwnParams p) {
  using G_ = OwnGeo<D, FP8, ROWS>;
  constexpr int TK = G_::TK, ROWB = G_::ROWB, TILE_B = G_::TILE_B, RAW_B = G_::RAW_B, STAGE_B = G_::STAGE_B, RC = G_::ROWS_CTA, PITCH = G_::PITCH;
  constexpr int ESZ = FP8 ? 1 : 2, LT = ROWS ? OTHREADS : 32;    // threads that fill one ring
  constexpr int MAXW = 8 + MAX_SPLITS;
  static_assert(TK * D * ESZ / 16 % LT == 0 && 2 * TK * (D / 16) % LT == 0 && TK <= LT && TK % 16 == 0, "every thread of a ring copies and converts whole pieces");
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ float red_m[OWARPS * 16], red_l[OWARPS * 16];       // per warp and row
  __shared__ float comb_m[RC], comb_l[RC], weight[RC][MAXW + 1];
  float* comb = reinterpret_cast<float*>(smem);                  // [RC][PITCH], after the key loop
  float* warp_o = comb + RC * PITCH;                             // [OWARPS][16][PITCH]

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, lt = ROWS ? tid : lane;
  const int rank = int(blockIdx.x) % p.cluster;
  int rest = int(blockIdx.x) / p.cluster;
  const int rt = rest % p.row_tiles;
  rest /= p.row_tiles;
  const int h = rest % p.Nkv, b = rest / p.Nkv;
  const int R = p.T * p.rep, row0 = rt * RC, n_rows = min(RC, R - row0);
  const int pos = position(p.pos, p.pos_n, p.pos_host, b);
  auto out_row = [&](int r) {
    const int rr = row0 + r, t = rr / p.rep;
    return ((long long)b * p.T + t) * p.Nq + h * p.rep + (rr - t * p.rep);
  };
  const bool idle = pos < 0;                                     // an unused place of the batch: zeros
  // keys any row of this CTA can see
  const int t_lo = row0 / p.rep, t_hi = (row0 + n_rows - 1) / p.rep;
  const int lo = p.window > 0 ? max(0, pos + t_lo - p.window + 1) : 0, hi = idle ? -1 : min(pos + t_hi, p.S - 1);
  const int n_keys = max(hi - lo + 1, 0);
  const int chunk = ((n_keys + p.cluster - 1) / p.cluster + TK - 1) / TK * TK;
  const int kbeg = lo + rank * chunk, kend = min(kbeg + chunk, hi + 1);
  const int n_tiles = kend > kbeg ? (kend - kbeg + TK - 1) / TK : 0;
  const int first = ROWS ? 0 : warp, step = ROWS ? 1 : OWARPS;
  const int nt = n_tiles > first ? (n_tiles - first + step - 1) / step : 0;

  uint8_t* ring = smem + (ROWS ? 0 : warp * G_::RING_B);
  const size_t head = (size_t(b) * p.Nkv + h) * p.S;
  const uint8_t *kbase = p.k + head * D * ESZ, *vbase = p.v + head * D * ESZ;

  auto issue = [&](int i) {                                      // i-th tile of this ring -> stage i % OSTAGES
    const int key0 = kbeg + (first + i * step) * TK;
    uint8_t* st = ring + (i % OSTAGES) * STAGE_B;
    constexpr int CPR = D * ESZ / 16, DROW = FP8 ? D : ROWB;
#pragma unroll
    for (int j = 0; j < TK * CPR / LT; ++j) {
      const int c = lt + LT * j, row = c / CPR, col = c % CPR, key = key0 + row;
      const bool ok = key < kend;
      const size_t off = size_t(ok ? key : kbeg) * D * ESZ + col * 16;
      cp16(smem_u32(st + row * DROW + col * 16), kbase + off, ok ? 16 : 0);
      cp16(smem_u32(st + RAW_B + row * DROW + col * 16), vbase + off, ok ? 16 : 0);
    }
    if (FP8 && lt < TK) {
      const int key = key0 + lt;
      const bool ok = key < kend;
      const size_t off = head + (ok ? key : kbeg);
      cp4(smem_u32(st + 2 * RAW_B + lt * 4), p.k_scale + off, ok ? 4 : 0);
      cp4(smem_u32(st + 2 * RAW_B + TK * 4 + lt * 4), p.v_scale + off, ok ? 4 : 0);
    }
  };
#pragma unroll
  for (int s = 0; s < OSTAGES - 1; ++s) {
    if (s < nt) issue(s);
    cp_commit();
  }

  // ---- query fragments (rows past the last one are zero) and each row's visible keys
  const int wr = (ROWS ? warp * 16 : 0) + (lane >> 2);           // this thread's first row; the second is 8 further on
  uint32_t qa[D / 16][4];
  int row_hi[2], row_lo[2];
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const int r = wr + 8 * e, rr = row0 + r, t = rr / p.rep;
    const bool ok = r < n_rows;
    row_hi[e] = ok ? pos + t : -1;
    row_lo[e] = p.window > 0 ? pos + t - p.window + 1 : 0;
    const __nv_bfloat16* src = p.q + b * p.q_sb + (long long)(h * p.rep + (rr - t * p.rep)) * p.q_sn + t * p.q_st + (lane & 3) * 2;
#pragma unroll
    for (int ks = 0; ks < D / 16; ++ks) {
      qa[ks][e] = ok ? __ldg(reinterpret_cast<const uint32_t*>(src + ks * 16)) : 0u;
      qa[ks][e + 2] = ok ? __ldg(reinterpret_cast<const uint32_t*>(src + ks * 16 + 8)) : 0u;
    }
  }
  float o[D / 8][4];
#pragma unroll
  for (int i = 0; i < D / 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};

  for (int i = 0; i < nt; ++i) {
    if (i + OSTAGES - 1 < nt) issue(i + OSTAGES - 1);
    cp_commit();
    cp_wait<OSTAGES - 1>();
    if (ROWS) __syncthreads(); else __syncwarp();
    uint8_t* st = ring + (i % OSTAGES) * STAGE_B;
    uint8_t *kt = st, *vt = st + RAW_B;
    const float *ksc = reinterpret_cast<const float*>(st + 2 * RAW_B), *vsc = ksc + TK;
    if (FP8) {                                                   // e4m3 rows -> bf16 operand rows, exactly; the scales come later
      kt = ring + OSTAGES * STAGE_B;
      vt = kt + TILE_B;
      constexpr int CPR = D / 16;
#pragma unroll
      for (int j = 0; j < 2 * TK * CPR / LT; ++j) {
        const int c = lt + LT * j, which = c / (TK * CPR), row = c % (TK * CPR) / CPR, col = c % CPR;
        const uint4 raw = *reinterpret_cast<const uint4*>(st + which * RAW_B + row * D + col * 16);
        const uint32_t in[4] = {raw.x, raw.y, raw.z, raw.w};
        uint32_t ow[8];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          ow[2 * u] = e4m3x2_to_bf16x2(uint16_t(in[u] & 0xffffu));
          ow[2 * u + 1] = e4m3x2_to_bf16x2(uint16_t(in[u] >> 16));
        }
        uint8_t* dst = (which ? vt : kt) + row * ROWB + col * 32;
        *reinterpret_cast<uint4*>(dst) = make_uint4(ow[0], ow[1], ow[2], ow[3]);
        *reinterpret_cast<uint4*>(dst + 16) = make_uint4(ow[4], ow[5], ow[6], ow[7]);
      }
      if (ROWS) __syncthreads(); else __syncwarp();
    }
    const int key0 = kbeg + (first + i * step) * TK;

    float s[TK / 8][4];
#pragma unroll
    for (int j = 0; j < TK / 8; ++j) s[j][0] = s[j][1] = s[j][2] = s[j][3] = 0.f;
    const uint32_t kaddr = smem_u32(kt) + ((lane >> 4) * 8 + (lane & 7)) * ROWB + ((lane >> 3) & 1) * 16;
#pragma unroll
    for (int ks = 0; ks < D / 16; ++ks) {
#pragma unroll
      for (int jp = 0; jp < TK / 16; ++jp) {
        uint32_t r[4];
        ldsm4(r, kaddr + jp * 16 * ROWB + ks * 32);
        mma16816(s[jp * 2], qa[ks], r[0], r[1]);
        mma16816(s[jp * 2 + 1], qa[ks], r[2], r[3]);
      }
    }
    float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (int j = 0; j < TK / 8; ++j) {
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const int e = x >> 1, at = j * 8 + (lane & 3) * 2 + (x & 1), key = key0 + at;
        const float f = FP8 ? p.scale_log2 * ksc[at] : p.scale_log2;
        s[j][x] = key < kend && key <= row_hi[e] && key >= row_lo[e] ? s[j][x] * f : -INFINITY;
        mx[e] = fmaxf(mx[e], s[j][x]);
      }
    }
    float alpha[2], ref[2], sum[2] = {0.f, 0.f};
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      mx[e] = fmaxf(mx[e], __shfl_xor_sync(0xffffffffu, mx[e], 1));
      mx[e] = fmaxf(mx[e], __shfl_xor_sync(0xffffffffu, mx[e], 2));
      const float mn = fmaxf(m[e], mx[e]);
      alpha[e] = mn == -INFINITY ? 1.f : exp2f(m[e] - mn);
      ref[e] = mn == -INFINITY ? 0.f : mn;
      m[e] = mn;
    }
#pragma unroll
    for (int j = 0; j < TK / 8; ++j)
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        s[j][x] = exp2f(s[j][x] - ref[x >> 1]);
        sum[x >> 1] += s[j][x];
        if (FP8) s[j][x] *= vsc[j * 8 + (lane & 3) * 2 + (x & 1)];
      }
    l[0] = l[0] * alpha[0] + sum[0];
    l[1] = l[1] * alpha[1] + sum[1];
#pragma unroll
    for (int d = 0; d < D / 8; ++d) {
      o[d][0] *= alpha[0];
      o[d][1] *= alpha[0];
      o[d][2] *= alpha[1];
      o[d][3] *= alpha[1];
    }
    const uint32_t vaddr = smem_u32(vt) + (((lane >> 3) & 1) * 8 + (lane & 7)) * ROWB + (lane >> 4) * 16;
#pragma unroll
    for (int kk = 0; kk < TK / 16; ++kk) {                       // P's accumulator layout is the A-operand layout of the next product
      const uint32_t pa[4] = {pack_bf16(s[2 * kk][0], s[2 * kk][1]), pack_bf16(s[2 * kk][2], s[2 * kk][3]),
                              pack_bf16(s[2 * kk + 1][0], s[2 * kk + 1][1]), pack_bf16(s[2 * kk + 1][2], s[2 * kk + 1][3])};
#pragma unroll
      for (int dp = 0; dp < D / 16; ++dp) {
        uint32_t r[4];
        ldsm4t(r, vaddr + kk * 16 * ROWB + dp * 32);
        mma16816(o[dp * 2], pa, r[0], r[1]);
        mma16816(o[dp * 2 + 1], pa, r[2], r[3]);
      }
    }
    if (ROWS) __syncthreads(); else __syncwarp();
  }
  cp_wait<0>();
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    l[e] += __shfl_xor_sync(0xffffffffu, l[e], 1);
    l[e] += __shfl_xor_sync(0xffffffffu, l[e], 2);
  }
  __syncthreads();                                               // every ring is drained: its space is reused

  // ---- the CTA's partial result in comb / comb_m / comb_l
  {
    float* dst = (ROWS ? comb : warp_o) + warp * 16 * PITCH;
    const int r0 = lane >> 2, c = (lane & 3) * 2;
#pragma unroll
    for (int d = 0; d < D / 8; ++d) {
      *reinterpret_cast<float2*>(dst + r0 * PITCH + d * 8 + c) = make_float2(o[d][0], o[d][1]);
      *reinterpret_cast<float2*>(dst + (r0 + 8) * PITCH + d * 8 + c) = make_float2(o[d][2], o[d][3]);
    }
    if ((lane & 3) == 0) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int at = warp * 16 + r0 + 8 * e;
        if (ROWS) {
          comb_m[at % RC] = m[e];
          comb_l[at % RC] = l[e];
        } else {
          red_m[at] = m[e];
          red_l[at] = l[e];
        }
      }
    }
  }
  if (!ROWS) {
    __syncthreads();
    for (int i = tid; i < n_rows * D; i += OTHREADS) {
      const int r = i / D, d = i % D;
      float M = -INFINITY;
#pragma unroll
      for (int x = 0; x < OWARPS; ++x) M = fmaxf(M, red_m[x * 16 + r]);
      float L = 0.f, O = 0.f;
#pragma unroll
      for (int x = 0; x < OWARPS; ++x) {
        const float mw = red_m[x * 16 + r], f = mw == -INFINITY ? 0.f : exp2f(mw - M);
        L += red_l[x * 16 + r] * f;
        O += warp_o[(x * 16 + r) * PITCH + d] * f;
      }
      comb[r * PITCH + d] = O;
      if (d == 0) {
        comb_m[r] = M;
        comb_l[r] = L;
      }
    }
  }
  __syncthreads();
  cg::cluster_group cluster = cg::this_cluster();
  if (!ROWS && p.cluster > 1) cluster.sync();

  if (p.splits > 0) asm volatile("griddepcontrol.wait;" ::: "memory");     // the prefix kernel is through
  // ---- weights of all partial results of a row: the cluster's CTAs, then the prefix splits; the last place holds 1 / (their sum)
  constexpr int TPR = OTHREADS / RC;                             // threads per row
  {
    const int r = tid / TPR, x = tid % TPR, n_own = ROWS ? 1 : p.cluster, n = n_own + p.splits;
    const int mrow = b * R + row0 + (r < n_rows ? r : 0);      // row of the prefix product
    const float2* prefix_ml = p.part_ml + ((long long)h * p.prefix_tiles + mrow / BM) * p.splits * BM + mrow % BM;
    auto ml = [&](int j) -> float2 {
      if (j >= n_own) return __ldcg(prefix_ml + (j - n_own) * BM);
      if (ROWS || p.cluster == 1) return make_float2(comb_m[r], comb_l[r]);
      return make_float2(*cluster.map_shared_rank(&comb_m[r], j), *cluster.map_shared_rank(&comb_l[r], j));
    };
    const float sink = p.sinks && r < n_rows ? __ldg(p.sinks + h * p.rep + (row0 + r) % p.rep) * L2E : -INFINITY;
    constexpr int PER = (MAXW + TPR - 1) / TPR;                  // a thread's share, all fetched at once
    float2 part[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) part[i] = r < n_rows && x + i * TPR < n ? ml(x + i * TPR) : make_float2(-INFINITY, 0.f);
    float M = -INFINITY, L = 0.f;
#pragma unroll
    for (int i = 0; i < PER; ++i) M = fmaxf(M, part[i].x);
#pragma unroll
    for (int of = TPR / 2; of > 0; of >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, of));
    M = fmaxf(M, sink);
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      if (r < n_rows && x + i * TPR < n) {
        const float f = part[i].x == -INFINITY ? 0.f : exp2f(part[i].x - M);
        weight[r][x + i * TPR] = f;
        L += part[i].y * f;
      }
    }
#pragma unroll
    for (int of = TPR / 2; of > 0; of >>= 1) L += __shfl_xor_sync(0xffffffffu, L, of);
    if (sink != -INFINITY) L += exp2f(sink - M);
    if (r < n_rows && x == 0) weight[r][MAXW] = idle || L == 0.f ? 0.f : 1.f / L;      // nothing visible and no sink: zeros
  }
  __syncthreads();

  // ---- sums, a row's columns dealt to the CTAs of a cluster. Neighbouring threads take neighbouring rows, which lie side by side in
  // the prefix partials (four at a time where they start on such a border); the results go through shared memory and leave row by row.
  // A thread fetches the splits of several places before it adds them up: one place at a time this took up to 15 us, most of it waiting.
  // The program is kept short on purpose, here and in the softmax: in a decode step a kernel's instructions come from memory as often as
  // not, and with twice the unrolling a call of 4 x 16 heads took 24 us instead of 18, one of 32 x 32 heads over e4m3 49 instead of 39.
  const int dn = D / p.cluster, d0 = rank * dn;                  // this CTA's columns
  const int m0 = b * R + row0, n_own = ROWS ? 1 : p.cluster;
  float* result = ROWS || p.cluster == 1 ? comb : warp_o;        // in place, unless the cluster's other CTAs still read it
  const float* part = p.part_o + ((long long)h * p.prefix_tiles + m0 / BM) * p.splits * D * BM + m0 % BM;
  auto own_part = [&](int r, int d) -> float {
    if (ROWS || p.cluster == 1) return comb[r * PITCH + d] * weight[r][0];
    float v = 0.f;
    for (int j = 0; j < p.cluster; ++j) v += *cluster.map_shared_rank(comb + r * PITCH + d, j) * weight[r][j];
    return v;
  };
  // a tile's rows end at a multiple of 128: row r of this CTA in tile (m0 + r) / 128
  auto place = [&](int r, int d) { return part + (long long)((m0 % BM + r) / BM) * p.splits * D * BM + d * BM + r - (m0 % BM + r) / BM * BM; };
  if (n_rows % 4 == 0 && m0 % 4 == 0) {
    const int nq = n_rows / 4, total = dn * nq;
    constexpr int E = ROWS ? 2 : 1, J = ROWS ? 4 : 8;            // places and splits in flight per thread (few rows: 128 places or fewer)
    for (int i0 = tid; i0 < total; i0 += E * OTHREADS) {
      float4 v[E];
#pragma unroll
      for (int e = 0; e < E; ++e) v[e] = make_float4(0.f, 0.f, 0.f, 0.f);
      for (int j0 = 0; j0 < p.splits; j0 += J) {
        float4 x[E][J];
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const int i = min(i0 + e * OTHREADS, total - 1), d = d0 + i / nq, r = i % nq * 4;
          const float* at = place(r, d);
#pragma unroll
          for (int j = 0; j < J; ++j) x[e][j] = __ldcg(reinterpret_cast<const float4*>(at + (long long)min(j0 + j, p.splits - 1) * D * BM));
        }
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const int r = min(i0 + e * OTHREADS, total - 1) % nq * 4;
#pragma unroll
          for (int j = 0; j < J; ++j) {
            if (j0 + j < p.splits) {
              v[e].x = fmaf(x[e][j].x, weight[r][n_own + j0 + j], v[e].x);
              v[e].y = fmaf(x[e][j].y, weight[r + 1][n_own + j0 + j], v[e].y);
              v[e].z = fmaf(x[e][j].z, weight[r + 2][n_own + j0 + j], v[e].z);
              v[e].w = fmaf(x[e][j].w, weight[r + 3][n_own + j0 + j], v[e].w);
            }
          }
        }
      }
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const int i = i0 + e * OTHREADS, d = d0 + i / nq, r = i % nq * 4;
        if (i < total) {
#pragma unroll 1
          for (int y = 0; y < 4; ++y) {
            const float add = y == 0 ? v[e].x : y == 1 ? v[e].y : y == 2 ? v[e].z : v[e].w;
            const float inv = weight[r + y][MAXW];               // 0: nothing visible, or an unused place - whatever the sums hold
            result[(r + y) * PITCH + d] = inv == 0.f ? 0.f : (own_part(r + y, d) + add) * inv;
          }
        }
      }
    }
  } else {
    for (int i = tid; i < n_rows * dn; i += OTHREADS) {
      const int d = d0 + i / n_rows, r = i % n_rows;
      const float inv = weight[r][MAXW];
      const float* at = place(r, d);
      float v = 0.f;
#pragma unroll 2
      for (int j = 0; j < p.splits; ++j) v = fmaf(__ldcg(at + (long long)j * D * BM), weight[r][n_own + j], v);
      result[r * PITCH + d] = inv == 0.f ? 0.f : (own_part(r, d) + v) * inv;
    }
  }
  __syncthreads();
  const float* done = result;
  for (int i = tid; i < n_rows * (dn / 8); i += OTHREADS) {
    const int r = i / (dn / 8), d = d0 + i % (dn / 8) * 8;
    const float4 x = *reinterpret_cast<const float4*>(done + r * PITCH + d), y = *reinterpret_cast<const float4*>(done + r * PITCH + d + 4);
    *reinterpret_cast<uint4*>(p.out + out_row(r) * D + d) = make_uint4(pack_bf16(x.x, x.y), pack_bf16(x.z, x.w), pack_bf16(y.x, y.y), pack_bf16(y.z, y.w));
  }
  if (!ROWS && p.cluster > 1) cluster.sync();                    // no CTA leaves while its shared memory is read
}

// ------------------------------------------------------------------------------------------------ host
template <class K>
int allow_smem(K kernel, int smem, int (&configured)[64]) {
  static std::mutex lock;
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev >= 64) return -111;
  std::lock_guard<std::mutex> guard(lock);
  if (!configured[dev]) {
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess) return -112;
    configured[dev] = 1;
  }
  return 0;
}

// Key splits of the prefix: the smallest estimated time of `waves of items on the SMs` x (key tiles of an item + two tiles' worth
// of fixed cost per item).
inline int prefix_splits(long long row_tiles, int Nkv, int n_tiles) {
  const long long sms = sm_count();
  long long best = 1LL << 60;
  int best_s = 1;
  for (int s = 1; s <= MAX_SPLITS && s <= n_tiles; ++s) {
    const long long items = row_tiles * Nkv * s, cost = (items + sms - 1) / sms * ((n_tiles + s - 1) / s + 2);
    if (cost < best) {
      best = cost;
      best_s = s;
    }
  }
  return best_s;
}

struct Shape {
  int key0, n_tiles, splits;
};
inline Shape prefix_shape(int B, int T, int P, int Nq, int Nkv, int window) {
  Shape s;
  s.key0 = window > 0 && P > window - 1 ? P - window + 1 : 0;      // the first new token of a sequence sees the most of the prefix
  s.n_tiles = (P - s.key0 + BN - 1) / BN;
  const long long rows = (long long)B * T * (Nq / Nkv);
  s.splits = s.n_tiles > 0 ? prefix_splits((rows + BM - 1) / BM, Nkv, s.n_tiles) : 0;
  return s;
}

template <int D, bool FP8>
int launch_prefix(const CUtensorMap& tk, const CUtensorMap& tv, const Params& p, cudaStream_t stream) {
  static int configured[64] = {};
  constexpr int smem = Smem<D, FP8>::BYTES;
  if (int rc = allow_smem(prefix_kernel<D, FP8>, smem, configured)) return rc;
  const long long items = ((long long)p.B * p.T * p.rep + BM - 1) / BM * p.Nkv * p.splits;
  const int sms = sm_count();
  prefix_kernel<D, FP8><<<unsigned(items < sms ? items : sms), THREADS, smem, stream>>>(tk, tv, p);
  LYRA_CHECK_LAUNCH();
  return 0;
}

template <int D, bool FP8, bool ROWS>
int launch_own(const OwnParams& p, cudaStream_t stream) {
  static int configured[64] = {};
  constexpr int smem = OwnGeo<D, FP8, ROWS>::SMEM_B;
  if (int rc = allow_smem(own_kernel<D, FP8, ROWS>, smem, configured)) return rc;
  const long long ctas = (long long)p.B * p.Nkv * p.row_tiles * p.cluster;
  if (ctas > 0x7fffffffLL) return -113;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(unsigned(ctas));
  cfg.blockDim = dim3(OTHREADS);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  // After the prefix kernel: launched beside it, waits for it just before the merge. All it reads until then (queries, caches,
  // positions) was there before the prefix kernel started.
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = p.cluster;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = p.splits > 0 ? 2 : 1;
  if (cudaLaunchKernelEx(&cfg, own_kernel<D, FP8, ROWS>, p) != cudaSuccess) {
    LYRA_CHECK_LAUNCH();
    return -114;
  }
  return 0;
}

template <int D>
int launch_own_d(const OwnParams& p, bool fp8, bool rows, cudaStream_t s) {
  if (fp8) return rows ? launch_own<D, true, true>(p, s) : launch_own<D, true, false>(p, s);
  return rows ? launch_own<D, false, true>(p, s) : launch_own<D, false, false>(p, s);
}

}  // namespace prefix
}  // namespace lyra

// Bytes of workspace of a call (no initialisation needed).
extern "C" long long lyra_prefix_attention_workspace(int B, int T, int P, int Nq, int Nkv, int D, int window) {
  using namespace lyra::prefix;
  if (B < 1 || T < 1 || P < 0 || Nkv < 1 || Nq < 1 || Nq % Nkv || (D != 64 && D != 128)) return -110;
  const long long rows = (long long)B * T * Nq;
  if (rows > (1LL << 30)) return -110;
  const Shape s = prefix_shape(B, T, P, Nq, Nkv, window);
  const long long tiles = (rows / Nkv + BM - 1) / BM * Nkv;
  return tiles * BM * s.splits * (D * 4 + 8);
}

// q [B, Nq, T, D] bf16 by element strides (unit inner stride, 16-byte aligned rows); prefix K / V [Nkv, P, D] by (head, position) element
// strides, bf16 or e4m3 with fp32 scales [Nkv, P] by head stride; own caches [B, Nkv, S, D] contiguous, bf16 or e4m3 with scales
// [B, Nkv, S]; pos int32 on the device, pos_n (1 or B) values, or null and pos_host; out [B, T, Nq, D] bf16.
extern "C" int lyra_prefix_attention(const void* q, long long q_sb, long long q_sn, long long q_st, const void* pk, long long pk_sh, long long pk_sp,
                                     const void* pv, long long pv_sh, long long pv_sp, const float* pk_scale, long long pks_sh, const float* pv_scale,
                                     long long pvs_sh, int prefix_fp8, const void* k, const void* v, const float* k_scale, const float* v_scale, int own_fp8,
                                     const float* sinks, const int* pos, int pos_n, int pos_host, void* out, void* workspace, long long workspace_bytes,
                                     int B, int T, int P, int S, int Nq, int Nkv, int D, float scale, int window, int* status, cudaStream_t stream) {
  using namespace lyra;
  using namespace lyra::prefix;
  const long long need = lyra_prefix_attention_workspace(B, T, P, Nq, Nkv, D, window);
  if (need < 0 || workspace_bytes < need || S < 0 || window < 0 || !(scale > 0.f)) return -110;
  if (pos && pos_n != 1 && pos_n != B) return -110;
  if ((prefix_fp8 && P > 0 && (!pk_scale || !pv_scale)) || (own_fp8 && S > 0 && (!k_scale || !v_scale))) return -110;
  const Shape shape = prefix_shape(B, T, P, Nq, Nkv, window);
  const int rep = Nq / Nkv, prefix_tiles = int(((long long)B * T * rep + BM - 1) / BM);
  float* part_o = static_cast<float*>(workspace);
  float2* part_ml = reinterpret_cast<float2*>(part_o + (long long)prefix_tiles * Nkv * BM * shape.splits * D);
  if (shape.splits > 0) {
    CUtensorMap tk, tv;
    const uint64_t esz = prefix_fp8 ? 1 : 2;
    const CUtensorMapDataType dt = prefix_fp8 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
    const CUtensorMapSwizzle swz = prefix_fp8 ? CU_TENSOR_MAP_SWIZZLE_NONE : CU_TENSOR_MAP_SWIZZLE_128B;
    const uint64_t dims[3] = {uint64_t(D), uint64_t(P), uint64_t(Nkv)};
    const uint32_t box[3] = {uint32_t(prefix_fp8 ? D : 64), uint32_t(BN), 1};
    const uint64_t ks[2] = {uint64_t(pk_sp) * esz, uint64_t(pk_sh) * esz}, vs[2] = {uint64_t(pv_sp) * esz, uint64_t(pv_sh) * esz};
    if (make_tmap_cached(&tk, pk, dt, 3, dims, ks, box, swz) || make_tmap_cached(&tv, pv, dt, 3, dims, vs, box, swz)) return -115;
    Params p;
    p.q = static_cast<const __nv_bfloat16*>(q);
    p.q_sb = q_sb; p.q_sn = q_sn; p.q_st = q_st;
    p.pos = pos; p.pos_n = pos_n; p.pos_host = pos_host;
    p.pk_scale = pk_scale; p.pv_scale = pv_scale; p.pks_sh = pks_sh; p.pvs_sh = pvs_sh;
    p.part_o = part_o; p.part_ml = part_ml;
    p.B = B; p.T = T; p.P = P; p.Nq = Nq; p.Nkv = Nkv; p.rep = rep; p.window = window; p.splits = shape.splits; p.key0 = shape.key0;
    p.scale_log2 = scale * L2E;
    p.status = status;
    int rc;
    if (D == 64) rc = prefix_fp8 ? launch_prefix<64, true>(tk, tv, p, stream) : launch_prefix<64, false>(tk, tv, p, stream);
    else rc = prefix_fp8 ? launch_prefix<128, true>(tk, tv, p, stream) : launch_prefix<128, false>(tk, tv, p, stream);
    if (rc) return rc;
  }
  OwnParams o;
  o.q = static_cast<const __nv_bfloat16*>(q);
  o.q_sb = q_sb; o.q_sn = q_sn; o.q_st = q_st;
  o.k = static_cast<const uint8_t*>(k); o.v = static_cast<const uint8_t*>(v);
  o.k_scale = k_scale; o.v_scale = v_scale;
  o.pos = pos; o.pos_n = pos_n; o.pos_host = pos_host;
  o.sinks = sinks; o.part_o = part_o; o.part_ml = part_ml;
  o.out = static_cast<__nv_bfloat16*>(out);
  o.B = B; o.T = T; o.S = S; o.Nq = Nq; o.Nkv = Nkv; o.rep = rep; o.window = window; o.splits = shape.splits; o.prefix_tiles = prefix_tiles;
  o.scale_log2 = scale * L2E;
  const bool by_rows = T * rep > 16;
  o.row_tiles = by_rows ? (T * rep + 63) / 64 : 1;
  // One token per sequence, few sequences, long caches: up to eight CTAs share a cache (128 keys each at least) until there are three
  // for every SM.
  o.cluster = 1;
  const int seen = window > 0 && window + T < S ? window + T : S;
  while (!by_rows && o.cluster < 8 && (long long)B * Nkv * o.cluster * 2 <= 3LL * sm_count() && seen >= o.cluster * 256) o.cluster *= 2;
  return D == 64 ? launch_own_d<64>(o, own_fp8, by_rows, stream) : launch_own_d<128>(o, own_fp8, by_rows, stream);
}
