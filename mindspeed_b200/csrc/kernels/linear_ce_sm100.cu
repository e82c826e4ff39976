// Output projection with its loss, without the [tokens, vocab] matrix of logits (bf16 / fp16, sm_100a).
//
//   z = hidden W^T,   lse_t = log sum_v exp(z_tv / tau),   loss_t = tau^2 sum_k q_tk (log q_tk - z_t,i(t,k) / tau + lse_t)
//   dz_tv = g_t tau (exp(z_tv / tau - lse_t) - sum_{k: i(t,k) = v} q_tk),   d hidden = dz W,   dW = dz^T hidden
//
// i(t, .) are K listed words of token t with weights q that add up to one.  Cross entropy is K = 1, q = 1, tau = 1 (the label); distillation
// lists a teacher's top logits, q being their softmax at temperature tau.
//
// Rows without a listed word (ignored labels) leave the products: a scan numbers the rows that stay, and every product runs over their
// count, which only the device knows.  When all rows stay, the products read the caller's hidden states directly, else a packed copy.
//
// Forward:  scan -> rows (packed copy, the K listed logits as dot products, q) -> GEMM whose epilogue keeps a (max, sum of exponentials)
//           pair per row and 256 columns -> join of the pairs.
// Backward: per piece of the vocabulary: the GEMM again, its epilogue now writing the 16-bit dz of the piece -> the listed words' entries
//           -> d hidden += dz W -> dW rows of the piece = dz^T hidden.  dz is rounded to the 16-bit type of the operands (the tensor cores
//           take nothing wider next to them): half a step on each term, as much as the rounding of the result itself.
//           With fp16, dz is scaled by a power of two that puts the largest |g| at 2^14 or above, so that probabilities down to 2^-28 keep
//           all their bits; the products' epilogues take the power out again in fp32.
//
// The products are the CTA-pair pipeline of gemm2_sm100.cu (same roles, barriers and bounded waits) with other work lists and epilogues.
#include "msb_common.cuh"
#include "msb_sm100.cuh"
#include <algorithm>

using namespace msb;
using namespace msb::sm100;

namespace {

constexpr int BM = 128;          // rows per CTA; the pair covers 256
constexpr int BN = 256;
constexpr int BK = 64;           // 64 16-bit values = one 128-byte swizzle row
constexpr int UMMA_K = 16;
constexpr float LOG2E = 1.4426950408889634f;

enum Epi : int { EPI_STATS = 0, EPI_DLOGITS = 1, EPI_OUT16 = 2, EPI_OUT32 = 3 };

struct LceGemm {
  CUtensorMap tmA, tmB, tmD;
  CUtensorMap tmPacked;        // the packed copy of the hidden states, read in place of A (forward) / B (weight gradient) when rows left
  int M, N, K;                 // upper bounds; the dimension that counts rows is cut to *rows
  const int* rows;             // rows that stay
  int all_rows;                // rows there are: the packed copy is unused when *rows equals it
  int group_m;
  int splits, slab_rows;       // K splits; rows between the slabs of their fp32 results
  int accumulate;              // OUT32: add to what is there
  int half;                    // operands are fp16 (else bf16)
  float2* part;                // STATS: [column tile][part_ld] (max, sum)
  long long part_ld;
  const float* lse;            // DLOGITS: per packed row, in units of z / tau
  const int* rowmap;           // DLOGITS: packed row -> token
  const float* g;              // DLOGITS: gradient of the token's loss
  int g_stride;
  float g_factor;              // DLOGITS: tau
  float inv_tau;
  const float* scale;          // fp16: scale[0] multiplies dz, scale[1] takes it out of the products
  unsigned int* status;
};

template <int EPI>
struct Cfg {
  static constexpr int NSTAGE = EPI == EPI_STATS ? 7 : EPI == EPI_OUT32 ? 5 : 6;
  static constexpr int A_BYTES = BM * BK * 2;
  static constexpr int STAGE_BYTES = A_BYTES + (BN / 2) * BK * 2;
  static constexpr int EPI_BUF = EPI == EPI_STATS ? 0 : EPI == EPI_OUT32 ? 8192 : 4096;   // 32 rows x 64 columns of the output type
  static constexpr int EPI_OFFSET = NSTAGE * STAGE_BYTES;
  static constexpr int BAR_OFFSET = EPI_OFFSET + 4 * 2 * EPI_BUF;
  static constexpr int TOTAL = BAR_OFFSET + 256 + 1024;
  static_assert(TOTAL <= 232448, "exceeds the 227 KB of shared memory a CTA may use");
};

// Work items of a pair: (tile, split of K).  Every role walks its own copy.  Tiles in groups of `group_m` tile rows share panels in L2.
struct Work {
  int num_m, num_n, num_kb, group_m, splits, item, items, stride;
  int m, n, split, kb0, kb1;
  __device__ Work(int M, int N, int K, int group_m_, int splits_, int pair, int npairs)
      : num_m((M + 2 * BM - 1) / (2 * BM)), num_n((N + BN - 1) / BN), num_kb((K + BK - 1) / BK), splits(splits_), item(pair),
        stride(npairs), m(0), n(0), split(0), kb0(0), kb1(0) {
    group_m = min(group_m_, max(num_m, 1));
    items = num_m * num_n * splits;
  }
  __device__ bool next() {
    if (item >= items) return false;
    const int tiles = num_m * num_n;
    split = item / tiles;
    const int t = item - split * tiles;
    const int per_group = group_m * num_n, grp = t / per_group, first_m = grp * group_m;
    const int gsz = min(num_m - first_m, group_m), r = t - grp * per_group;
    m = first_m + r % gsz;
    n = r / gsz;
    kb0 = (int)((long long)num_kb * split / splits);
    kb1 = (int)((long long)num_kb * (split + 1) / splits);
    item += stride;
    return true;
  }
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t pack16(float lo, float hi, int half) {
  if (half) {
    __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&h);
  }
  return pack_bf16(lo, hi);
}

// EPI_STATS / EPI_DLOGITS: A = hidden [M, K], B = W [N, K], rows on M.     EPI_OUT32, A_MN = false: A = dz [M, K], B = W [K, N], rows on M.
// A_MN = true: A = dz [K, M], B = hidden [K, N], rows on K.
template <int EPI, bool A_MN, bool B_MN>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(192, 1) lce_gemm_kernel(const __grid_constant__ LceGemm p) {
  using L = Cfg<EPI>;
  constexpr int NSTAGE = L::NSTAGE;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;   // identical in both CTAs of the pair
  const uint32_t bar_base = smem_base + L::BAR_OFFSET;
  auto full_bar = [&](int s) { return bar_base + 8u * s; };
  auto empty_bar = [&](int s) { return bar_base + 8u * (NSTAGE + s); };
  auto tfull_bar = [&](int a) { return bar_base + 8u * (2 * NSTAGE + a); };
  auto tempty_bar = [&](int a) { return bar_base + 8u * (2 * NSTAGE + 2 + a); };
  const uint32_t tmem_slot = bar_base + 8u * (2 * NSTAGE + 4);
  uint32_t* tmem_slot_ptr = reinterpret_cast<uint32_t*>(smem_raw + (tmem_slot - smem_u32(smem_raw)));

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t cta = cluster_ctarank();                 // 0 = leader
  const int pair = blockIdx.x >> 1, npairs = gridDim.x >> 1;
  const int rows = *p.rows;
  const int M = A_MN ? p.M : rows, K = A_MN ? rows : p.K;
  const bool packed = rows != p.all_rows;
  constexpr uint32_t TMEM_COLS = 512u;                    // two accumulators of 256 columns

  if (threadIdx.x == 0) {
    for (int s = 0; s < NSTAGE; ++s) { mbar_init(full_bar(s), 1); mbar_init(empty_bar(s), 1); }
    for (int a = 0; a < 2; ++a) { mbar_init(tfull_bar(a), 1); mbar_init(tempty_bar(a), 8); }
    mbar_fence_init();
  }
  if (warp == 1) { tmem_alloc_pair(tmem_slot, TMEM_COLS); tmem_relinquish_pair(); }
  tc_fence_before();
  __syncwarp();
  cluster_sync_all();          // barriers of both CTAs are initialised before anyone signals across the pair
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot_ptr;

  bool alive = true;
  if (warp == 0) {
    // ===================== TMA producer (both CTAs) =====================
    if (lane == 0) {
      const CUtensorMap* mapA = (EPI <= EPI_DLOGITS && packed) ? &p.tmPacked : &p.tmA;
      const CUtensorMap* mapB = (A_MN && packed) ? &p.tmPacked : &p.tmB;
      tma_prefetch_desc(mapA);
      tma_prefetch_desc(mapB);
      int stage = 0; uint32_t phase = 0;
      Work w(M, p.N, K, p.group_m, p.splits, pair, npairs);
      while (alive && w.next()) {
        const int m0 = w.m * (2 * BM) + (int)cta * BM;
        const int n0 = w.n * BN + (int)cta * (BN / 2);
        for (int kb = w.kb0; kb < w.kb1; ++kb) {
          if (!mbar_wait(empty_bar(stage), phase ^ 1u, p.status, 0x10u)) { alive = false; break; }
          const uint32_t sa = smem_base + stage * L::STAGE_BYTES;
          const uint32_t sb = sa + L::A_BYTES;
          if (cta == 0) mbar_arrive_expect_tx(full_bar(stage), 2 * L::STAGE_BYTES);
          const uint32_t lead_full = mapa_u32(full_bar(stage), 0);
          const int k0 = kb * BK;
          if (!A_MN) {
            tma_load_2d_pair(sa, mapA, lead_full, k0, m0);                             // box [128 rows x 64 k]
          } else {
#pragma unroll
            for (int j = 0; j < BM / 64; ++j)                                          // boxes [64 k x 64 m]
              tma_load_2d_pair(sa + j * (BK * 128), mapA, lead_full, m0 + j * 64, k0);
          }
          if (!B_MN) {
            tma_load_2d_pair(sb, mapB, lead_full, k0, n0);                             // box [128 rows x 64 k]
          } else {
#pragma unroll
            for (int j = 0; j < BN / 128; ++j)                                         // boxes [64 k x 64 n]
              tma_load_2d_pair(sb + j * (BK * 128), mapB, lead_full, n0 + j * 64, k0);
          }
          if (++stage == NSTAGE) { stage = 0; phase ^= 1u; }
        }
      }
      // tail: every commit aimed at this CTA's empty barriers must have landed before the CTA may exit
      for (int i = 0; i < NSTAGE && alive; ++i) {
        if (!mbar_wait(empty_bar(stage), phase ^ 1u, p.status, 0x11u)) { alive = false; break; }
        if (++stage == NSTAGE) { stage = 0; phase ^= 1u; }
      }
    }
  } else if (warp == 1) {
    // ===================== MMA issuer (leader CTA, one thread) =====================
    if (lane == 0 && cta == 0) {
      const uint32_t idesc = make_idesc_f16(2 * BM, BN, p.half ? 0 : 1, A_MN ? 1 : 0, B_MN ? 1 : 0);
      int stage = 0; uint32_t phase = 0;
      int acc = 0; uint32_t acc_phase = 0;
      Work w(M, p.N, K, p.group_m, p.splits, pair, npairs);
      while (alive && w.next()) {
        if (!mbar_wait(tempty_bar(acc), acc_phase ^ 1u, p.status, 0x20u)) { alive = false; break; }
        tc_fence_after();
        const uint32_t d_tmem = tmem_base + (uint32_t)(acc * BN);
        for (int kb = w.kb0; kb < w.kb1; ++kb) {
          if (!mbar_wait(full_bar(stage), phase, p.status, 0x21u)) { alive = false; break; }
          tc_fence_after();
          const uint32_t sa = smem_base + stage * L::STAGE_BYTES;
          const uint32_t sb = sa + L::A_BYTES;
#pragma unroll
          for (int k = 0; k < BK / UMMA_K; ++k) {
            // K-major: advance 16 elements = 32 bytes inside the swizzled row; MN-major: 16 k-rows = 2048 bytes
            const uint64_t adesc = A_MN ? make_smem_desc(sa + k * (UMMA_K * 128), BK * 128, 1024)
                                        : make_smem_desc(sa + k * (UMMA_K * 2), 0, 1024);
            const uint64_t bdesc = B_MN ? make_smem_desc(sb + k * (UMMA_K * 128), BK * 128, 1024)
                                        : make_smem_desc(sb + k * (UMMA_K * 2), 0, 1024);
            umma_f16_pair(d_tmem, adesc, bdesc, idesc, (kb != w.kb0 || k != 0) ? 1u : 0u);
          }
          umma_commit_pair(empty_bar(stage), 3);      // both CTAs may refill this stage once these MMAs have read it
          if (++stage == NSTAGE) { stage = 0; phase ^= 1u; }
        }
        if (!alive) break;
        umma_commit_pair(tfull_bar(acc), 3);          // accumulator complete in both CTAs
        if (++acc == 2) { acc = 0; acc_phase ^= 1u; }
      }
    }
  } else {
    // ===================== epilogue (warps 2..5, both CTAs) =====================
    const int q = warp & 3;                          // TMEM lane quarter this warp may access
    const uint32_t buf_base = smem_base + L::EPI_OFFSET + (uint32_t)q * 2u * L::EPI_BUF;
    const uint32_t lead_tempty[2] = {mapa_u32(tempty_bar(0), 0), mapa_u32(tempty_bar(1), 0)};
    const float unscale = (EPI >= EPI_OUT16 && p.scale) ? p.scale[1] : 1.f;
    const float ctau = p.inv_tau * LOG2E;
    int acc = 0; uint32_t acc_phase = 0;
    uint32_t chunk = 0;
    Work w(M, p.N, K, p.group_m, p.splits, pair, npairs);
    while (alive && w.next()) {
      const int row0 = w.m * (2 * BM) + (int)cta * BM + q * 32, row = row0 + lane;
      float coef = 0.f, lse = 0.f;
      if (EPI == EPI_DLOGITS && row < rows) {
        coef = p.g[(long long)p.rowmap[row] * p.g_stride] * p.g_factor;
        if (p.scale) coef *= p.scale[0];
        lse = p.lse[row];
      }
      if (!mbar_wait_warp(tfull_bar(acc), acc_phase, p.status, 0x30u)) { alive = false; break; }
      tc_fence_after();
      const uint32_t t_row = tmem_base + ((uint32_t)(q * 32) << 16) + (uint32_t)(acc * BN);
      if (EPI == EPI_STATS) {
        // online softmax over the 256 columns of this row; differences are taken before the scaling so that the terms that weigh
        // most (z near the maximum) keep their bits
        float m = -INFINITY, s = 0.f;
#pragma unroll 1
        for (int c2 = 0; c2 < BN; c2 += 64) {
          const int left = p.N - (w.n * BN + c2);
          if (left <= 0) break;
          uint32_t rr[64];
          tmem_ld_32x32(t_row + (uint32_t)c2, rr);
          tmem_ld_32x32(t_row + (uint32_t)(c2 + 32), rr + 32);
          tmem_ld_wait();
          if (left < 64) {
#pragma unroll
            for (int j = 0; j < 64; ++j)
              if (j >= left) rr[j] = 0xff800000u;          // -inf: columns past the vocabulary
          }
          float mx[4];
#pragma unroll
          for (int u = 0; u < 4; ++u) mx[u] = __uint_as_float(rr[u]);
#pragma unroll
          for (int j = 4; j < 64; ++j) mx[j & 3] = fmaxf(mx[j & 3], __uint_as_float(rr[j]));
          const float mn = fmaxf(m, fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])));
          const float base = mn == -INFINITY ? 0.f : mn;
          float sm[4] = {s * ex2((m - base) * ctau), 0.f, 0.f, 0.f};
#pragma unroll
          for (int j = 0; j < 64; ++j) sm[j & 3] += ex2((__uint_as_float(rr[j]) - base) * ctau);
          s = (sm[0] + sm[1]) + (sm[2] + sm[3]);
          m = mn;
        }
        if (row < rows) p.part[(long long)w.n * p.part_ld + row] = make_float2(m, s);
      } else {
        const uint32_t sw = (uint32_t)(lane & 7);
        const bool empty = A_MN && w.kb1 == w.kb0;          // no row at all: the weight gradient is zero
#pragma unroll 1
        for (int c2 = 0; c2 < BN; c2 += 64, ++chunk) {
          const int col0 = w.n * BN + c2;
          if (col0 >= p.N) break;                       // the rest of this tile is beyond the last column
          uint32_t rr[64];
          tmem_ld_32x32(t_row + (uint32_t)c2, rr);
          tmem_ld_32x32(t_row + (uint32_t)(c2 + 32), rr + 32);
          tmem_ld_wait();
          if (EPI == EPI_DLOGITS) {
            // a row with no gradient writes zeros even where its logits are not finite
#pragma unroll
            for (int j = 0; j < 64; ++j) {
              const float e = ex2(fmaf(__uint_as_float(rr[j]), p.inv_tau, -lse) * LOG2E) * coef;
              rr[j] = __float_as_uint(coef == 0.f ? 0.f : e);
            }
          } else {
#pragma unroll
            for (int j = 0; j < 64; ++j) rr[j] = empty ? 0u : __float_as_uint(__uint_as_float(rr[j]) * unscale);
          }
          const uint32_t buf = buf_base + (chunk & 1u) * L::EPI_BUF;
          if (lane == 0) tma_store_wait_read<1>();      // the store that last read this buffer (two chunks ago) is done with it
          __syncwarp();
          const uint32_t row_addr = buf + (uint32_t)lane * 128u;
          if (EPI != EPI_OUT32) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {                 // 16-byte chunk j = columns 8j .. 8j+7
              uint32_t pk[4];
#pragma unroll
              for (int e = 0; e < 4; ++e) pk[e] = pack16(__uint_as_float(rr[8 * j + 2 * e]), __uint_as_float(rr[8 * j + 2 * e + 1]), p.half);
              asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(row_addr + ((((uint32_t)j) ^ sw) << 4)), "r"(pk[0]), "r"(pk[1]),
                           "r"(pk[2]), "r"(pk[3])
                           : "memory");
            }
          } else {
#pragma unroll
            for (int h = 0; h < 2; ++h)                   // two [32 x 32] fp32 boxes per 64 columns
#pragma unroll
              for (int j = 0; j < 8; ++j)
                asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(row_addr + (uint32_t)h * 4096u + ((((uint32_t)j) ^ sw) << 4)),
                             "r"(rr[32 * h + 4 * j]), "r"(rr[32 * h + 4 * j + 1]), "r"(rr[32 * h + 4 * j + 2]), "r"(rr[32 * h + 4 * j + 3])
                             : "memory");
          }
          fence_proxy_async_smem();                       // generic-proxy writes -> visible to the TMA store
          __syncwarp();
          if (lane == 0) {
            // OUT32 of the hidden gradient: slabs of `slab_rows` rows, a multiple of the 32 rows of a box
            const int y = (EPI == EPI_OUT32 && !A_MN) ? w.split * p.slab_rows + row0 : row0;
            const bool inside = (EPI == EPI_OUT32 && !A_MN) ? row0 < p.slab_rows : row0 < p.M;
            if (inside) {
              if (EPI != EPI_OUT32) {
                tma_store_2d(&p.tmD, buf, col0, y);
              } else if (!p.accumulate) {
                tma_store_2d(&p.tmD, buf, col0, y);
                if (col0 + 32 < p.N) tma_store_2d(&p.tmD, buf + 4096u, col0 + 32, y);
              } else {
                tma_reduce_add_2d(&p.tmD, buf, col0, y);
                if (col0 + 32 < p.N) tma_reduce_add_2d(&p.tmD, buf + 4096u, col0 + 32, y);
              }
            }
            tma_store_commit();                           // one group per chunk, empty or not: the wait above counts groups
          }
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_remote(lead_tempty[acc]);   // this warp has read its lanes of the accumulator
      if (++acc == 2) { acc = 0; acc_phase ^= 1u; }
    }
    if (lane == 0) tma_store_wait<0>();                 // staging buffers are read and the stores are complete before exit
  }

  // ---- teardown: both CTAs meet, TMEM is returned ----
  tc_fence_before();
  __syncwarp();
  cluster_sync_all();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem_base, TMEM_COLS);
  }
}

// ---------------------------------------------------------------------------------------------------------
// rows
// ---------------------------------------------------------------------------------------------------------
// What a token's list says: 0 nothing (no listed word: the token is ignored), 1 at least one word, 2 a word outside the vocabulary.
// Cross entropy: the label.  Distillation: negative indices and teacher logits of -inf are unused places.
__device__ __forceinline__ int label_kind(long long y, long long vocab, long long ignore_index) {
  return y == ignore_index ? 0 : (y >= 0 && y < vocab) ? 1 : 2;
}
__device__ __forceinline__ bool place_used(long long i, float a, long long vocab) { return i >= 0 && i < vocab && !(a == -INFINITY); }

// One warp a token.
__global__ void __launch_bounds__(256) lce_kind_kernel(const long long* __restrict__ idx, const float* __restrict__ teacher, int T, int K,
                                                       long long vocab, unsigned char* __restrict__ kind) {
  const int t = blockIdx.x * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (t >= T) return;
  bool used = false, bad = false;
  for (int k = lane; k < K; k += 32) {
    const long long i = idx[(long long)t * K + k];
    used |= place_used(i, teacher[(long long)t * K + k], vocab);
    bad |= i >= vocab;
  }
  used = __any_sync(0xffffffffu, used);
  bad = __any_sync(0xffffffffu, bad);
  if (lane == 0) kind[t] = bad ? 2 : used ? 1 : 0;
}

// Numbers the rows that stay, in the order of the tokens: pos[t] = packed row, -1 ignored, -2 a word outside the vocabulary (also noted
// in `error`); rowmap is the inverse.  One block: 8 tokens a thread and round, so up to 8192 tokens take one round.
__global__ void __launch_bounds__(1024) lce_scan_kernel(const long long* __restrict__ labels, const unsigned char* __restrict__ kind, int T,
                                                        long long vocab, long long ignore_index, int* __restrict__ pos,
                                                        int* __restrict__ rowmap, int* __restrict__ count, unsigned int* error) {
  __shared__ int warp_sum_s[32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int base = 0;
  for (long long t0 = 0; t0 < T; t0 += 8192) {
    int kd[8], mine = 0;
    const long long first = t0 + (long long)threadIdx.x * 8;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const long long t = first + j;
      kd[j] = t >= T ? 0 : labels ? label_kind(labels[t], vocab, ignore_index) : kind[t];
      mine += kd[j] == 1;
    }
    int incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += v;
    }
    __syncthreads();                      // the sums of the last round have been read
    if (lane == 31) warp_sum_s[warp] = incl;
    __syncthreads();
    int before = 0, total = 0;
    for (int w = 0; w < 32; ++w) {
      const int v = warp_sum_s[w];
      before += w < warp ? v : 0;
      total += v;
    }
    int at = base + before + incl - mine;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const long long t = first + j;
      if (t >= T) break;
      if (kd[j] == 1) {
        pos[t] = at;
        rowmap[at++] = (int)t;
      } else {
        pos[t] = kd[j] == 2 ? -2 : -1;
        if (kd[j] == 2) atomicCAS(error, 0u, 0x703u);
      }
    }
    base += total;
  }
  if (threadIdx.x == 0) *count = base;
}

// Dot product of two rows of H 16-bit values by one warp (H a multiple of 8, rows 16-byte aligned): fp32 sums, same value in all lanes.
template <typename T>
__device__ __forceinline__ float warp_dot(const T* __restrict__ a, const T* __restrict__ b, int H, int lane) {
  float s0 = 0.f, s1 = 0.f;
#pragma unroll 4
  for (int c = lane * 8; c < H; c += 256) {
    Vec8<T> x, y;
    x.load(a + c);
    y.load(b + c);
    float fx[8], fy[8];
    x.to_float(fx);
    y.to_float(fy);
#pragma unroll
    for (int j = 0; j < 8; j += 2) { s0 = fmaf(fx[j], fy[j], s0); s1 = fmaf(fx[j + 1], fy[j + 1], s1); }
  }
  return warp_sum(s0 + s1);
}

// Per token: the packed copy of its hidden state (when rows left), the listed logits z (raw; 0 where the word is another rank's), their
// weights q, and  dot = sum q z / tau,  ent = sum q log q.  Tokens that left get loss 0 (NaN where a word is outside the vocabulary).
// WPT warps a token: one for a single listed word, eight for lists.  Blocks past the tokens zero the packed rows up to the next
// multiple of 64: the weight gradient reads whole blocks of 64 rows.
template <typename T, int WPT>
__global__ void __launch_bounds__(256) lce_rows_kernel(const T* __restrict__ hidden, long long ldh, const T* __restrict__ weight, long long ldw,
                                                       const long long* __restrict__ idx, const float* __restrict__ teacher, int Tn, int H,
                                                       int K, int vocab_local, long long vocab_start, long long vocab, float inv_tau,
                                                       const int* __restrict__ pos, const int* __restrict__ count, T* __restrict__ packed,
                                                       float* __restrict__ z, float* __restrict__ qout, float* __restrict__ dot,
                                                       float* __restrict__ ent, float* __restrict__ loss) {
  constexpr int PER_BLOCK = 8 / WPT;
  extern __shared__ float zs[];            // WPT = 8: the token's K logits
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int n = *count;
  const int token_blocks = (Tn + PER_BLOCK - 1) / PER_BLOCK;
  if ((int)blockIdx.x >= token_blocks) {
    const int r = n + ((int)blockIdx.x - token_blocks);
    if (n == Tn || r >= min(Tn, (n + 63) / 64 * 64)) return;
    const uint4 zero = make_uint4(0, 0, 0, 0);
    for (int c = threadIdx.x * 8; c < H; c += 2048) *reinterpret_cast<uint4*>(packed + (long long)r * H + c) = zero;
    return;
  }
  const int t = (int)blockIdx.x * PER_BLOCK + (WPT == 1 ? warp : 0);
  if (t >= Tn) return;
  const int at = pos[t];
  if (at < 0) {
    if (lane == 0 && (WPT == 1 || warp == 0)) loss[t] = at == -2 ? NAN : 0.f;
    return;
  }
  const T* h = hidden + (long long)t * ldh;
  if (n != Tn) {
    const int step = WPT == 1 ? 256 : 2048;
    for (int c = (WPT == 1 ? lane : (int)threadIdx.x) * 8; c < H; c += step)
      *reinterpret_cast<uint4*>(packed + (long long)at * H + c) = *reinterpret_cast<const uint4*>(h + c);
  }
  if (WPT == 1) {
    const long long v = idx[t] - vocab_start;
    const bool here = v >= 0 && v < vocab_local;
    const float d = here ? warp_dot(h, weight + v * ldw, H, lane) : 0.f;
    if (lane == 0) { z[at] = d; qout[at] = 1.f; dot[at] = d * inv_tau; ent[at] = 0.f; }
    return;
  }
  const long long first = (long long)t * K;
  for (int k = warp; k < K; k += 8) {
    const long long v = idx[first + k] - vocab_start;
    const bool here = v >= 0 && v < vocab_local && place_used(idx[first + k], teacher[first + k], vocab);
    const float d = here ? warp_dot(h, weight + v * ldw, H, lane) : 0.f;
    if (lane == 0) { zs[k] = d; z[(long long)at * K + k] = d; }
  }
  __syncthreads();
  if (warp != 0) return;
  float mx = -INFINITY;
  for (int k = lane; k < K; k += 32)
    if (place_used(idx[first + k], teacher[first + k], vocab)) mx = fmaxf(mx, teacher[first + k]);
  mx = warp_max(mx);
  float s = 0.f;
  for (int k = lane; k < K; k += 32)
    if (place_used(idx[first + k], teacher[first + k], vocab)) s += ex2((teacher[first + k] - mx) * (inv_tau * LOG2E));
  s = warp_sum(s);
  const float ls = (float)log((double)s);
  float d = 0.f, e = 0.f;
  for (int k = lane; k < K; k += 32) {
    float q = 0.f;
    if (place_used(idx[first + k], teacher[first + k], vocab)) {
      const float a = (teacher[first + k] - mx) * inv_tau;
      q = ex2(a * LOG2E) / s;
      d = fmaf(q, zs[k] * inv_tau, d);
      if (!(q == 0.f)) e = fmaf(q, a - ls, e);
    }
    qout[(long long)at * K + k] = q;
  }
  d = warp_sum(d);
  e = warp_sum(e);
  if (lane == 0) { dot[at] = d; ent[at] = e; }
}

// ---------------------------------------------------------------------------------------------------------
// join of the (max, sum) pairs, loss
// ---------------------------------------------------------------------------------------------------------
__device__ __forceinline__ void lce_finish(float m, float s, float dot, float ent, float inv_tau, float tau2, float* lse, float* loss) {
  const float ls = (float)log((double)s);
  *lse = m * inv_tau + ls;
  *loss = tau2 * (ent + (m * inv_tau - dot) + ls);       // the two large numbers are subtracted first
}

// 32 rows a block (coalesced over the rows), 32 threads a row over the column tiles; the order of the sums is fixed.
__global__ void __launch_bounds__(1024) lce_join_kernel(const float2* __restrict__ part, long long part_ld, int tiles, float inv_tau, float tau2,
                                                        const int* __restrict__ count, const int* __restrict__ rowmap,
                                                        const float* __restrict__ dot, const float* __restrict__ ent, float* __restrict__ mo,
                                                        float* __restrict__ so, float* __restrict__ lse, float* __restrict__ loss) {
  __shared__ float ms[32][33], ss[32][33];
  const int r = threadIdx.x & 31, y = threadIdx.x >> 5;
  const int n = *count, row = blockIdx.x * 32 + r;
  if ((int)blockIdx.x * 32 >= n) return;
  const float c = inv_tau * LOG2E;
  float m = -INFINITY, s = 0.f;
  if (row < n)
    for (int i = y; i < tiles; i += 32) {
      const float2 v = part[(long long)i * part_ld + row];
      const float mn = fmaxf(m, v.x), base = mn == -INFINITY ? 0.f : mn;
      s = s * ex2((m - base) * c) + v.y * ex2((v.x - base) * c);
      m = mn;
    }
  ms[y][r] = m;
  ss[y][r] = s;
  __syncthreads();
  if (y == 0 && row < n) {
    float mm = -INFINITY;
    for (int i = 0; i < 32; ++i) mm = fmaxf(mm, ms[i][r]);
    float t = 0.f;
    for (int i = 0; i < 32; ++i) t += ss[i][r] * ex2((ms[i][r] - (ms[i][r] == -INFINITY && mm != -INFINITY ? 0.f : mm)) * c);
    if (mo) {
      mo[row] = mm;
      so[row] = t;
    } else {
      float l, o;
      lce_finish(mm, t, dot[row], ent[row], inv_tau, tau2, &l, &o);
      lse[row] = l;
      loss[rowmap[row]] = o;
    }
  }
}

// Vocabulary-parallel form, around the reductions over the group.
__global__ void lce_rescale_kernel(float* s, const float* m, const float* gm, float inv_tau, const int* count) {
  const int i = blockIdx.x * blockDim.x + threadIdx.x;
  if (i < *count) s[i] *= ex2((m[i] - gm[i]) * (inv_tau * LOG2E));
}
__global__ void lce_loss_kernel(const float* gm, const float* gs, const float* dot, const float* ent, const int* rowmap, const int* count,
                                float inv_tau, float tau2, float* lse, float* loss) {
  const int i = blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= *count) return;
  float l, o;
  lce_finish(gm[i], gs[i], dot[i], ent[i], inv_tau, tau2, &l, &o);
  lse[i] = l;
  loss[rowmap[i]] = o;
}

// ---------------------------------------------------------------------------------------------------------
// backward helpers
// ---------------------------------------------------------------------------------------------------------
// scale[0] = 2^e with max |g| * factor * 2^e in [2^14, 2^15), scale[1] = 2^-e (one block; 1 where there is no finite gradient but 0)
__global__ void __launch_bounds__(1024) lce_scale_kernel(const float* __restrict__ g, int g_stride, const int* __restrict__ rowmap,
                                                         const int* __restrict__ count, float factor, float* __restrict__ scale) {
  __shared__ float red[32];
  const int n = *count;
  float m = 0.f;
  for (int i = threadIdx.x; i < n; i += 1024) {
    const float v = fabsf(g[(long long)rowmap[i] * g_stride] * factor);
    if (v < INFINITY) m = fmaxf(m, v);
  }
  m = block_max(m, red);
  if (threadIdx.x == 0) {
    int e = 0;
    if (m > 0.f) e = max(-100, min(100, 14 - (int)floorf(log2f(m))));
    scale[0] = ldexpf(1.f, e);
    scale[1] = ldexpf(1.f, -e);
  }
}

// The listed words' entries of the piece: dz[i, v] = (exp(z / tau - lse) - sum of the q of all places that list v) * coefficient.  Places
// that list a word twice write the same value.
template <typename T>
__global__ void __launch_bounds__(256) lce_listed_kernel(T* __restrict__ dz, long long ldz, const long long* __restrict__ idx,
                                                         const float* __restrict__ z, const float* __restrict__ q, const float* __restrict__ lse,
                                                         const int* __restrict__ rowmap, const int* __restrict__ count, int K,
                                                         long long piece_start, int piece_cols, const float* __restrict__ g, int g_stride,
                                                         float g_factor, float inv_tau, const float* __restrict__ scale) {
  const long long f = (long long)blockIdx.x * 256 + threadIdx.x;
  const int i = (int)(f / K), k = (int)(f - (long long)i * K);
  if (i >= *count) return;
  const int t = rowmap[i];
  const long long* list = idx + (long long)t * K;
  const long long v = list[k] - piece_start;
  if (v < 0 || v >= piece_cols) return;
  const float* qi = q + (long long)i * K;
  if (qi[k] == 0.f && K > 1) {
    // an unused place (or one of no weight): another place may list the same word, and what it writes is right; where none
    // does, the entry is the plain probability that is there already
    return;
  }
  float sum = 0.f;
  for (int j = 0; j < K; ++j) sum += list[j] == list[k] ? qi[j] : 0.f;
  float coef = g[(long long)t * g_stride] * g_factor;
  if (scale) coef *= scale[0];
  const float p = ex2((z[(long long)i * K + k] * inv_tau - lse[i]) * LOG2E);
  dz[(long long)i * ldz + v] = from_f<T>(coef == 0.f ? 0.f : (p - sum) * coef);
}

// d hidden: the fp32 slabs of the K splits, added in order, back in the order of the tokens; zero rows for tokens that left.
template <typename T>
__global__ void __launch_bounds__(256) lce_dhidden_kernel(const float* __restrict__ acc, int splits, long long slab, const int* __restrict__ pos,
                                                          T* __restrict__ out, int Tn, int H) {
  const int per_row = H / 8;
  const long long total = (long long)Tn * per_row;
  for (long long f = (long long)blockIdx.x * 256 + threadIdx.x; f < total; f += (long long)gridDim.x * 256) {
    const int t = (int)(f / per_row), c = (int)(f - (long long)t * per_row) * 8;
    const int at = pos[t];
    float o[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (at >= 0) {
      const float* a = acc + (long long)at * H + c;
      for (int s = 0; s < splits; ++s, a += slab) {
        const float4 u = __ldcs(reinterpret_cast<const float4*>(a)), v = __ldcs(reinterpret_cast<const float4*>(a + 4));
        o[0] += u.x; o[1] += u.y; o[2] += u.z; o[3] += u.w;
        o[4] += v.x; o[5] += v.y; o[6] += v.z; o[7] += v.w;
      }
    }
    Vec8<T> w;
    w.from_float(o);
    w.store(out + (long long)t * H + c);
  }
}

// ---------------------------------------------------------------------------------------------------------
// launchers
// ---------------------------------------------------------------------------------------------------------
template <int EPI, bool A_MN, bool B_MN>
int launch_gemm(const LceGemm& p, cudaStream_t s) {
  using L = Cfg<EPI>;
  auto kern = lce_gemm_kernel<EPI, A_MN, B_MN>;
  static std::atomic<unsigned long long> stated{0};
  if (int bad = msb::allow_smem((const void*)kern, L::TOTAL, "lce_gemm", stated)) return bad;
  const long long items = (long long)((p.M + 2 * BM - 1) / (2 * BM)) * ((p.N + BN - 1) / BN) * p.splits;
  const int pairs = (int)std::min<long long>(items, msb::num_sms() / 2);
  kern<<<2 * pairs, 192, L::TOTAL, s>>>(p);
  MSB_CHECK_LAUNCH("lce_gemm");
  return 0;
}

CUtensorMapDataType map_type(int dtype) { return dtype == MSB_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16; }

}  // namespace

// What both directions are given.  Pointers are device memory; the caller owns every buffer.
struct MsbLceArgs {
  const void* hidden;          // [T, H], row pitch ldh
  const void* weight;          // [V, H] (this rank's words), row pitch ldw
  const long long* idx;        // [T, K] listed words (labels: K = 1)
  const float* teacher;        // [T, K] teacher logits, or null: cross entropy
  long long ldh, ldw;
  long long vocab_start, vocab, ignore_index;
  int T, H, V, K;
  int dtype;
  float tau;
  int* pos;                    // [T]
  int* rowmap;                 // [T]
  int* count;                  // [1]
  unsigned char* kind;         // [T] scratch (lists)
  void* packed;                // [T, H]
  float* z;                    // [T, K]
  float* q;                    // [T, K]
  float* dot;                  // [T]
  float* ent;                  // [T]
  float* lse;                  // [T]
  float* loss;                 // [T]
  float* part;                 // [column tiles, T] pairs, scratch
  float* mx;                   // [T], [T]: local statistics for the vocabulary-parallel form, else null
  float* sum;
  // backward
  const float* g;
  long long g_stride;          // 0: one value for all tokens
  void* dz;                    // [T, piece] scratch, row pitch ldz
  long long ldz;
  int piece;                   // columns of a piece (a multiple of 256)
  float* acc;                  // [splits, slab_rows, H] fp32 scratch, or null: no hidden gradient
  int splits, slab_rows;
  void* dhidden;               // [T, H]
  void* dweight;               // [V, H], 16-bit or fp32; null: no weight gradient
  int dweight_fp32_add;        // dweight is fp32 and added to
  float* scale;                // [2] scratch (fp16), else null
  unsigned int* status;        // [0] expired waits, [1] words outside the vocabulary
};

static int lce_check(const MsbLceArgs* a) {
  MSB_REQUIRE(a->T > 0 && a->H > 0 && a->V > 0 && a->K > 0, "linear_ce: empty problem T=%d H=%d V=%d K=%d", a->T, a->H, a->V, a->K);
  MSB_REQUIRE(a->dtype == MSB_BF16 || a->dtype == MSB_F16, "linear_ce: dtype code %d is not bf16 or fp16", a->dtype);
  MSB_REQUIRE(a->H % 8 == 0 && a->ldh % 8 == 0 && a->ldw % 8 == 0, "linear_ce: H=%d and the row pitches must be multiples of 8", a->H);
  MSB_REQUIRE(a->status != nullptr, "linear_ce: status words are required");
  MSB_REQUIRE(a->tau > 0.f, "linear_ce: the temperature must be positive");
  MSB_REQUIRE(a->K == 1 || a->teacher, "linear_ce: lists need teacher logits");
  return 0;
}

// Scan, rows, GEMM with row statistics, join.  With `mx` the join stops at the local (max, sum).
MSB_API int msb_lce_forward(const MsbLceArgs* a, cudaStream_t s) {
  if (int rc = lce_check(a)) return rc;
  const float inv_tau = 1.f / a->tau, tau2 = a->tau * a->tau;
  if (a->teacher) {
    lce_kind_kernel<<<(a->T + 7) / 8, 256, 0, s>>>(a->idx, a->teacher, a->T, a->K, a->vocab, a->kind);
    MSB_CHECK_LAUNCH("lce_kind");
  }
  lce_scan_kernel<<<1, 1024, 0, s>>>(a->teacher ? nullptr : a->idx, a->kind, a->T, a->vocab, a->ignore_index, a->pos, a->rowmap, a->count,
                                     a->status + 1);
  MSB_CHECK_LAUNCH("lce_scan");
  const int per_block = a->teacher ? 1 : 8;
  const unsigned grid = (unsigned)((a->T + per_block - 1) / per_block + 63);
#define LCE_ROWS(DT, WPT)                                                                                                                    \
  lce_rows_kernel<DT, WPT><<<grid, 256, WPT == 8 ? a->K * 4 : 0, s>>>((const DT*)a->hidden, a->ldh, (const DT*)a->weight, a->ldw, a->idx,      \
                                                                     a->teacher, a->T, a->H, a->K, a->V, a->vocab_start, a->vocab, inv_tau,   \
                                                                     a->pos, a->count, (DT*)a->packed, a->z, a->q, a->dot, a->ent, a->loss)
  if (a->dtype == MSB_F16) { if (a->teacher) LCE_ROWS(__half, 8); else LCE_ROWS(__half, 1); }
  else { if (a->teacher) LCE_ROWS(__nv_bfloat16, 8); else LCE_ROWS(__nv_bfloat16, 1); }
#undef LCE_ROWS
  MSB_CHECK_LAUNCH("lce_rows");
  LceGemm p;
  memset(&p, 0, sizeof(p));
  const CUtensorMapDataType dt = map_type(a->dtype);
  int rc;
  if ((rc = make_tmap_2d(&p.tmA, a->hidden, dt, 2, a->T, a->H, a->ldh, BM, BK))) return rc;
  if ((rc = make_tmap_2d(&p.tmPacked, a->packed, dt, 2, a->T, a->H, a->H, BM, BK))) return rc;
  if ((rc = make_tmap_2d(&p.tmB, a->weight, dt, 2, a->V, a->H, a->ldw, BN / 2, BK))) return rc;
  p.M = a->T; p.N = a->V; p.K = a->H;
  p.rows = a->count; p.all_rows = a->T;
  p.group_m = 8; p.splits = 1;
  p.half = a->dtype == MSB_F16;
  p.part = reinterpret_cast<float2*>(a->part); p.part_ld = a->T;
  p.inv_tau = inv_tau;
  p.status = a->status;
  if ((rc = launch_gemm<EPI_STATS, false, false>(p, s))) return rc;
  lce_join_kernel<<<(a->T + 31) / 32, 1024, 0, s>>>(p.part, p.part_ld, (a->V + BN - 1) / BN, inv_tau, tau2, a->count, a->rowmap, a->dot, a->ent,
                                                    a->mx, a->sum, a->lse, a->loss);
  MSB_CHECK_LAUNCH("lce_join");
  return 0;
}

// Vocabulary-parallel form: sum *= exp((local max - global max) / tau), then (after the sums over the group) the loss.
MSB_API int msb_lce_rescale(float* sum, const float* mx, const float* gmx, float tau, const int* count, int T, cudaStream_t s) {
  lce_rescale_kernel<<<(T + 255) / 256, 256, 0, s>>>(sum, mx, gmx, 1.f / tau, count);
  MSB_CHECK_LAUNCH("lce_rescale");
  return 0;
}
MSB_API int msb_lce_loss(const float* gmx, const float* gsum, const float* dot, const float* ent, const int* rowmap, const int* count, float tau,
                         int T, float* lse, float* loss, cudaStream_t s) {
  lce_loss_kernel<<<(T + 255) / 256, 256, 0, s>>>(gmx, gsum, dot, ent, rowmap, count, 1.f / tau, tau * tau, lse, loss);
  MSB_CHECK_LAUNCH("lce_loss");
  return 0;
}

// Hidden and weight gradients, a piece of the vocabulary at a time.
MSB_API int msb_lce_backward(const MsbLceArgs* a, cudaStream_t s) {
  if (int rc = lce_check(a)) return rc;
  MSB_REQUIRE(a->piece > 0 && a->piece % BN == 0 && a->ldz % 8 == 0 && a->ldz >= std::min(a->piece, a->V), "linear_ce: piece of %d columns, pitch %lld", a->piece, a->ldz);
  MSB_REQUIRE(!a->acc || (a->splits >= 1 && a->slab_rows >= a->T && a->slab_rows % 32 == 0 && (long long)a->splits * a->slab_rows < 0x7fffffffll),
              "linear_ce: %d slabs of %d rows", a->splits, a->slab_rows);
  MSB_REQUIRE(!a->acc || a->splits <= (a->V + BK - 1) / BK, "linear_ce: more K splits than blocks of %d words", BK);
  MSB_REQUIRE(!a->acc || a->splits == 1 || a->piece >= a->V, "linear_ce: K splits need the vocabulary in one piece");
  const float inv_tau = 1.f / a->tau;
  const CUtensorMapDataType dt = map_type(a->dtype);
  if (a->scale) {
    lce_scale_kernel<<<1, 1024, 0, s>>>(a->g, (int)a->g_stride, a->rowmap, a->count, a->tau, a->scale);
    MSB_CHECK_LAUNCH("lce_scale");
  }
  LceGemm p;
  memset(&p, 0, sizeof(p));
  p.rows = a->count; p.all_rows = a->T;
  p.half = a->dtype == MSB_F16;
  p.rowmap = a->rowmap; p.lse = a->lse;
  p.g = a->g; p.g_stride = (int)a->g_stride; p.g_factor = a->tau;
  p.inv_tau = inv_tau;
  p.scale = a->scale;
  p.status = a->status;
  int rc;
  for (long long v0 = 0; v0 < a->V; v0 += a->piece) {
    const int cols = (int)std::min<long long>(a->piece, a->V - v0);
    const char* w = (const char*)a->weight + v0 * a->ldw * 2;
    // dz of the piece
    if ((rc = make_tmap_2d(&p.tmA, a->hidden, dt, 2, a->T, a->H, a->ldh, BM, BK))) return rc;
    if ((rc = make_tmap_2d(&p.tmPacked, a->packed, dt, 2, a->T, a->H, a->H, BM, BK))) return rc;
    if ((rc = make_tmap_2d(&p.tmB, w, dt, 2, cols, a->H, a->ldw, BN / 2, BK))) return rc;
    if ((rc = make_tmap_2d(&p.tmD, a->dz, dt, 2, a->T, cols, a->ldz, 32, 64))) return rc;
    p.M = a->T; p.N = cols; p.K = a->H; p.group_m = 8; p.splits = 1; p.accumulate = 0;
    if ((rc = launch_gemm<EPI_DLOGITS, false, false>(p, s))) return rc;
    const long long places = (long long)a->T * a->K;
    const unsigned grid = (unsigned)((places + 255) / 256);
    if (a->dtype == MSB_F16)
      lce_listed_kernel<__half><<<grid, 256, 0, s>>>((__half*)a->dz, a->ldz, a->idx, a->z, a->q, a->lse, a->rowmap, a->count, a->K,
                                                     a->vocab_start + v0, cols, a->g, (int)a->g_stride, a->tau, inv_tau, a->scale);
    else
      lce_listed_kernel<__nv_bfloat16><<<grid, 256, 0, s>>>((__nv_bfloat16*)a->dz, a->ldz, a->idx, a->z, a->q, a->lse, a->rowmap, a->count, a->K,
                                                            a->vocab_start + v0, cols, a->g, (int)a->g_stride, a->tau, inv_tau, a->scale);
    MSB_CHECK_LAUNCH("lce_listed");
    if (a->acc) {
      if ((rc = make_tmap_2d(&p.tmA, a->dz, dt, 2, a->T, cols, a->ldz, BM, BK))) return rc;
      if ((rc = make_tmap_2d(&p.tmB, w, dt, 2, cols, a->H, a->ldw, BK, 64))) return rc;
      if ((rc = make_tmap_2d(&p.tmD, a->acc, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 4, (uint64_t)a->splits * a->slab_rows, a->H, a->H, 32, 32))) return rc;
      p.M = a->T; p.N = a->H; p.K = cols; p.splits = a->splits; p.slab_rows = a->slab_rows; p.accumulate = v0 > 0;
      if ((rc = launch_gemm<EPI_OUT32, false, true>(p, s))) return rc;
    }
    if (a->dweight) {
      if ((rc = make_tmap_2d(&p.tmA, a->dz, dt, 2, a->T, cols, a->ldz, BK, 64))) return rc;
      if ((rc = make_tmap_2d(&p.tmB, a->hidden, dt, 2, a->T, a->H, a->ldh, BK, 64))) return rc;
      if ((rc = make_tmap_2d(&p.tmPacked, a->packed, dt, 2, a->T, a->H, a->H, BK, 64))) return rc;
      p.M = cols; p.N = a->H; p.K = a->T; p.splits = 1; p.slab_rows = 0;
      if (a->dweight_fp32_add) {
        float* d = (float*)a->dweight + v0 * a->H;
        if ((rc = make_tmap_2d(&p.tmD, d, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 4, cols, a->H, a->H, 32, 32))) return rc;
        p.accumulate = 1;
        if ((rc = launch_gemm<EPI_OUT32, true, true>(p, s))) return rc;
      } else {
        if ((rc = make_tmap_2d(&p.tmD, (char*)a->dweight + v0 * a->H * 2, dt, 2, cols, a->H, a->H, 32, 64))) return rc;
        p.accumulate = 0;
        if ((rc = launch_gemm<EPI_OUT16, true, true>(p, s))) return rc;
      }
    }
  }
  if (a->acc) {
    const long long vecs = (long long)a->T * (a->H / 8);
    const unsigned grid = (unsigned)std::min<long long>((vecs + 255) / 256, (long long)msb::num_sms() * 16);
    const long long slab = (long long)a->slab_rows * a->H;
    if (a->dtype == MSB_F16) lce_dhidden_kernel<__half><<<grid, 256, 0, s>>>(a->acc, a->splits, slab, a->pos, (__half*)a->dhidden, a->T, a->H);
    else lce_dhidden_kernel<__nv_bfloat16><<<grid, 256, 0, s>>>(a->acc, a->splits, slab, a->pos, (__nv_bfloat16*)a->dhidden, a->T, a->H);
    MSB_CHECK_LAUNCH("lce_dhidden");
  }
  return 0;
}
