// Output projection with its loss, with a bounded part of the [tokens, vocab] matrix of logits in memory (bf16 / fp16, sm_100a).
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
// Forward:  scan (part of the rows kernel for short inputs) -> rows (packed copy) -> GEMM whose epilogue keeps (max, where, sum of
//           exponentials) per row and half a tile, and takes listed logits from the accumulators where the lists are sorted; else four
//           warps a CTA make them as dot products beside it -> join.  (4096 rows, 64 words each, W of 129280 x 4096: the products' rows of
//           W are 2.1 GB, 0.3 ms as a kernel of its own and as much beside the GEMM.)
//           The tensor cores cut every addition to their fp32 sums off: a logit comes out 0.26 (H / 16) 2^-24 of itself too small (0.258
//           to 0.273 measured at H 1024 to 5120; half a unit in the last place for each of the H / 16 additions, of a sum that grows).
//           The scale 1 / tau of such logits takes that up on average: it was fitted to sums that grow steadily on this chip, and a logit
//           whose partial sums exceed it is corrected by too little (of the order of the error itself, 4e-6 at H 4096, which is what the
//           bounds allow without it).  The join computes the largest logit of a row again as a dot product.
// Backward: per piece of the vocabulary: the GEMM again, its epilogue now writing the 16-bit dz of the piece (with the label's -1; a
//           list's q are subtracted by a kernel of its own) -> d hidden += dz W -> dW rows of the piece = dz^T hidden.  dz is rounded to
//           the 16-bit type of the operands (the tensor cores take nothing wider next to them): half a step on each term, as much as the
//           rounding of the result itself.  With fp16, dz is scaled by a power of two that puts the largest |g| at 2^14 or above, so that
//           probabilities down to 2^-28 keep all their bits; the products' epilogues take the power out again in fp32.
// Kept logits: the forward can keep the fp32 logits of the first words (transposed, [words, rows]: rows are the lanes of the epilogue),
//           and an elementwise pass makes dz of them instead of the GEMM.  Few rows (at most 64, or the logits take at most an eighth of
//           the weight's bytes, but for rows rounded up to 8) keep all: one reading of W less, a quarter of all
//           traffic (96 x 128256 x 4096, both directions, with the kernels of that step: 1043 -> 755 us; 714 now).  More rows keep what the
//           caller's limit holds, where H is wide enough (KEEP_BYTES and KEEP_WIDTH in ops/linear_cross_entropy.py, with the figures of
//           both sides).
//           Up to 64 rows dz goes in two 16-bit terms, as 128 rows: the products take no longer, and so few roundings do not average out.
//
// The products are the CTA-pair pipeline of gemm2_sm100.cu (same roles, barriers and bounded waits) with other work lists and epilogues.
// Up to 128 rows they run on single CTAs with tiles of 128 rows: half of a pair's 256 rows would be padding, and although W's bytes bound
// such calls, products of padding draw the power that the clocks then lack (96 x 128256 x 4096 forward: 215 us at first, 255 at the power
// limit with pairs).
#include "msb_common.cuh"
#include "msb_sm100.cuh"
#include <algorithm>

using namespace msb;
using namespace msb::sm100;

extern "C" int msb_gemm_get_cta_limit();   // gemm_sm100.cu

namespace {

constexpr int BM = 128;          // rows per CTA; the pair covers 256
constexpr int BK = 64;           // 64 16-bit values = one 128-byte swizzle row
constexpr int UMMA_K = 16;
// tile rows that share the other operand's panels in L2.  Logits: 16 keep W's bytes from DRAM at three times its size (forward of 8192 x
// 128256 x 4096 in 6.7 ms, 7.5 with 8, 6.7 with 32).  Gradients: sums over thousands of words or tokens, whose panels do not outlive a
// round of tiles in L2; 8 make the rounds square (8192 tokens: dz and weight gradient 13.4 ms, 13.8 with 16, 14.3 with 32).
constexpr int GROUP_LOGITS = 16, GROUP_GRADS = 8;
constexpr float LOG2E = 1.4426950408889634f;

constexpr int EPI_WARPS = 8;       // two a quarter of the 128 accumulator lanes, each half of the columns
constexpr int GATHER_WARPS = 4;    // of the forward: listed logits
constexpr int TWO_ROWS = 64;       // up to so many rows dz has a second term (one block of K, half of a tile's rows)

enum Epi : int { EPI_STATS = 0, EPI_DLOGITS = 1, EPI_OUT16 = 2, EPI_OUT32 = 3 };

struct LceGemm {
  CUtensorMap tmA, tmB, tmD;
  CUtensorMap tmPacked;        // the packed copy of the hidden states, read in place of A (forward) / B (weight gradient) when rows left
  int M, N, K;                 // upper bounds; the dimension that counts rows is cut to *rows
  const int* rows;             // [0] rows that stay, [1] K splits of the hidden gradient
  int all_rows;                // rows there are: the packed copy is unused when *rows equals it
  int group_m;
  int rows_on_k;               // the rows are summed over (weight gradient), else they are output rows
  int two;                     // dz in two terms, TWO_ROWS rows each: 2 TWO_ROWS rows whatever *rows says
  int split;                   // take rows[1] K splits, their fp32 results in slabs of slab_rows rows
  int slab_rows;
  int accumulate;              // OUT32: add to what is there
  int half;                    // operands are fp16 (else bf16)
  float2* part;                // STATS: [half a tile's columns][part_ld] (max, sum)
  unsigned char* part_at;      // STATS: column of the max
  long long part_ld;
  const unsigned long long* sorted;   // STATS: (word << 16 | place) ascending, [T, list], or null: the gathering warps read idx
  const long long* idx;        // STATS: listed words [T, list], their logits go to listed [rows, list]
  const float* teacher;
  float* listed;
  int list;
  const void* hidden;
  const void* weight;
  long long ldh, ldw, vocab_start, vocab;
  int width, words;            // H, words of this rank
  float* zt;                   // STATS: keep the logits of the first `kept` columns, [kept][ldt], or null
  int ldt, kept;
  const float* lse;            // DLOGITS: per packed row, in units of z / tau
  const int* rowmap;           // DLOGITS: packed row -> token
  const float* g;              // DLOGITS: gradient of the token's loss
  int g_stride;
  float g_factor;              // DLOGITS: tau
  float inv_tau, tc_inv_tau;   // 1 / tau for exact logits and for those of the tensor cores
  const long long* label;      // DLOGITS: the token's word (cross entropy), or null
  const float* z;              // DLOGITS: its logit, per packed row
  long long piece_start;       // DLOGITS: word of column 0
  const float* scale;          // fp16: scale[0] multiplies dz, scale[1] takes it out of the products
  unsigned int* status;
};

// HOW a product is tiled: on single CTAs (128 x 256), on pairs (256 x 256, two accumulators that take turns), or on pairs with both
// accumulators side by side (256 x 512).
enum How : int { SINGLE = 0, PAIRED = 1, WIDE = 2 };
constexpr int BN = 256;            // columns of an accumulator

template <int EPI, int HOW>
struct Cfg {
  static constexpr int CTAS = HOW == SINGLE ? 1 : 2, SUBS = HOW == WIDE ? 2 : 1;
  static constexpr int THREADS = 64 + 32 * (EPI_WARPS + (EPI == EPI_STATS ? GATHER_WARPS : 0));
  // what the staging leaves of 227 KB
  static constexpr int NSTAGE = HOW != PAIRED ? 4 : EPI == EPI_STATS ? 7 : EPI == EPI_DLOGITS ? 6 : 5;
  static constexpr int A_BYTES = BM * BK * 2, B_BYTES = BN / CTAS * BK * 2;
  static constexpr int STAGE_BYTES = A_BYTES + SUBS * B_BYTES;
  // 32 rows x 64 columns of the output type; twice that for OUT16 where there is room (two buffers), half for OUT32 where there is not
  static constexpr int EPI_BUF = EPI == EPI_STATS ? 0 : EPI == EPI_DLOGITS || HOW != PAIRED ? 4096 : 8192;
  static constexpr int EPI_OFFSET = NSTAGE * STAGE_BYTES;
  static constexpr int BAR_OFFSET = EPI_OFFSET + EPI_WARPS * EPI_BUF;
  static constexpr int TOTAL = BAR_OFFSET + 256 + 1024;
  static_assert(TOTAL <= 232448, "exceeds the 227 KB of shared memory a CTA may use");
};

// Work items of a pair (or single CTA): (tile, split of K).  Every role walks its own copy.  Tiles in groups of `group_m` tile rows share panels in L2.
template <int TILE_M, int TILE_N>
struct Work {
  int num_m, num_n, num_kb, group_m, splits, item, items, stride;
  int m, n, split, kb0, kb1;
  __device__ Work(int M, int N, int K, int group_m_, int splits_, int pair, int npairs)
      : num_m((M + TILE_M - 1) / TILE_M), num_n((N + TILE_N - 1) / TILE_N), num_kb((K + BK - 1) / BK), splits(splits_), item(pair),
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
// One column of the warp's 32 accumulator lanes.
__device__ __forceinline__ uint32_t tmem_ld_column(uint32_t taddr) {
  uint32_t v;
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x1.b32 {%0}, [%1];" : "=r"(v) : "r"(taddr) : "memory");
  tmem_ld_wait();
  return v;
}
__device__ __forceinline__ uint32_t pack16(float lo, float hi, int half) {
  if (half) {
    __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&h);
  }
  return pack_bf16(lo, hi);
}

// What a token's list says: 0 nothing (no listed word: the token is ignored), 1 at least one word, 2 a word outside the vocabulary.
// Cross entropy: the label.  Distillation: negative indices and teacher logits of -inf are unused places.
__device__ __forceinline__ int label_kind(long long y, long long vocab, long long ignore_index) {
  return y == ignore_index ? 0 : (y >= 0 && y < vocab) ? 1 : 2;
}
__device__ __forceinline__ bool place_used(long long i, float a, long long vocab) { return i >= 0 && i < vocab && !(a == -INFINITY); }

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

// Logits of row i (token t) for up to four words: their rows of W are in flight together.
template <typename T>
__device__ __forceinline__ void dots_of_row(const LceGemm& p, int i, int k0, int t, long long mine, int lane) {
  const T* h = (const T*)p.hidden + t * p.ldh;
  const T* w[4];
  bool here[4];
  float s[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const long long v = __shfl_sync(0xffffffffu, mine, j);
    here[j] = v >= 0;
    w[j] = (const T*)p.weight + (here[j] ? v : 0) * p.ldw;
  }
#pragma unroll 2
  for (int c = lane * 8; c < p.width; c += 256) {
    Vec8<T> x, y[4];
    x.load(h + c);
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (here[j]) y[j].load(w[j] + c);
    float fx[8], fy[8];
    x.to_float(fx);
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (here[j]) {
        y[j].to_float(fy);
#pragma unroll
        for (int e = 0; e < 8; ++e) s[j] = fmaf(fx[e], fy[e], s[j]);
      }
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    s[j] = warp_sum(s[j]);
    if (lane == 0 && k0 + j < p.list) p.listed[(long long)i * p.list + k0 + j] = here[j] ? s[j] : 0.f;
  }
}

// EPI_STATS / EPI_DLOGITS: A = hidden [M, K], B = W [N, K].      Hidden gradient: A = dz [M, K], B = W [K, N].
// Weight gradient: A = dz [K, M], B = hidden [K, N], rows on K.  A_MN tells how dz lies in memory ([tokens, words] or transposed).
template <int EPI, bool A_MN, bool B_MN, int HOW>
__global__ void __cluster_dims__(HOW == SINGLE ? 1 : 2, 1, 1) __launch_bounds__(Cfg<EPI, HOW>::THREADS, 1)
    lce_gemm_kernel(const __grid_constant__ LceGemm p) {
  using L = Cfg<EPI, HOW>;
  constexpr bool PAIR = HOW != SINGLE;
  constexpr int CTAS = L::CTAS, SUBS = L::SUBS, NSTAGE = L::NSTAGE;
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
  const uint32_t cta = PAIR ? cluster_ctarank() : 0;      // 0 = leader
  const int pair = blockIdx.x / CTAS, npairs = gridDim.x / CTAS;
  constexpr uint32_t TMEM_COLS = 2u * BN;                 // two accumulators

  if (threadIdx.x == 0) {
    for (int s = 0; s < NSTAGE; ++s) { mbar_init(full_bar(s), 1); mbar_init(empty_bar(s), 1); }
    for (int a = 0; a < 2; ++a) { mbar_init(tfull_bar(a), 1); mbar_init(tempty_bar(a), CTAS * EPI_WARPS); }
    mbar_fence_init();
    tma_prefetch_desc(&p.tmA);
    tma_prefetch_desc(&p.tmB);
  }
  if (warp == 1) {
    if (PAIR) { tmem_alloc_pair(tmem_slot, TMEM_COLS); tmem_relinquish_pair(); }
    else { tmem_alloc(tmem_slot, TMEM_COLS); tmem_relinquish(); }
  }
  tc_fence_before();
  __syncwarp();
  if (PAIR) cluster_sync_all();   // barriers of both CTAs are initialised before anyone signals across the pair
  else __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot_ptr;
  after_previous();

  const int rows = p.rows[0], splits = p.split ? p.rows[1] : 1;
  const int padded = p.two && rows > 0 ? 2 * TWO_ROWS : rows;
  const int M = p.rows_on_k ? p.M : padded, K = p.rows_on_k ? padded : p.K;
  const bool packed = rows != p.all_rows;

  bool alive = true;
  if (warp == 0) {
    // ===================== TMA producer (both CTAs) =====================
    if (lane == 0) {
      const CUtensorMap* mapA = (EPI <= EPI_DLOGITS && packed) ? &p.tmPacked : &p.tmA;
      const CUtensorMap* mapB = (p.rows_on_k && packed) ? &p.tmPacked : &p.tmB;
      int stage = 0; uint32_t phase = 0;
      Work<CTAS * BM, SUBS * BN> w(M, p.N, K, p.group_m, splits, pair, npairs);
      while (alive && w.next()) {
        const int m0 = (w.m * CTAS + (int)cta) * BM;
        const int n0 = w.n * (SUBS * BN) + (int)cta * (BN / 2);
        const int subs = SUBS == 2 && n0 - (int)cta * (BN / 2) + BN >= p.N ? 1 : SUBS;      // the second half may lie past the last column
        for (int kb = w.kb0; kb < w.kb1; ++kb) {
          if (!mbar_wait(empty_bar(stage), phase ^ 1u, p.status, 0x10u)) { alive = false; break; }
          const uint32_t sa = smem_base + stage * L::STAGE_BYTES;
          const uint32_t sb = sa + L::A_BYTES;
          if (cta == 0) mbar_arrive_expect_tx(full_bar(stage), CTAS * (L::A_BYTES + subs * L::B_BYTES));
          const uint32_t lead_full = PAIR ? mapa_u32(full_bar(stage), 0) : full_bar(stage);
          auto load = [&](uint32_t dst, const CUtensorMap* map, int x, int y) {
            if (PAIR) tma_load_2d_pair(dst, map, lead_full, x, y);
            else tma_load_2d(dst, map, lead_full, x, y);
          };
          const int k0 = kb * BK;
          if (!A_MN) {
            load(sa, mapA, k0, m0);                                                    // box [128 rows x 64 k]
          } else {
#pragma unroll
            for (int j = 0; j < BM / 64; ++j) load(sa + j * (BK * 128), mapA, m0 + j * 64, k0);   // boxes [64 k x 64 m]
          }
#pragma unroll
          for (int h = 0; h < SUBS; ++h) {
            if (h >= subs) break;
            const uint32_t sh = sb + h * L::B_BYTES;
            const int nh = n0 + h * BN;
            if (!B_MN) {
              load(sh, mapB, k0, nh);                                                  // box [128 rows x 64 k] (256 on a single CTA)
            } else {
#pragma unroll
              for (int j = 0; j < BN / CTAS / 64; ++j)                                 // boxes [64 k x 64 n]; both terms times the same rows
                load(sh + j * (BK * 128), mapB, nh + j * 64, p.rows_on_k && p.two ? 0 : k0);
            }
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
      const uint32_t idesc = make_idesc_f16(CTAS * BM, BN, p.half ? 0 : 1, A_MN ? 1 : 0, B_MN ? 1 : 0);
      int stage = 0; uint32_t phase = 0;
      Work<CTAS * BM, SUBS * BN> w(M, p.N, K, p.group_m, splits, pair, npairs);
      if constexpr (SUBS == 1) {
        int acc = 0; uint32_t acc_phase = 0;
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
              if (PAIR) umma_f16_pair(d_tmem, adesc, bdesc, idesc, (kb != w.kb0 || k != 0) ? 1u : 0u);
              else umma_f16(d_tmem, adesc, bdesc, idesc, (kb != w.kb0 || k != 0) ? 1u : 0u);
            }
            // both CTAs may refill this stage once these MMAs have read it
            if (PAIR) umma_commit_pair(empty_bar(stage), 3);
            else umma_commit(empty_bar(stage));
            if (++stage == NSTAGE) { stage = 0; phase ^= 1u; }
          }
          if (!alive) break;
          if (PAIR) umma_commit_pair(tfull_bar(acc), 3);          // accumulator complete in both CTAs
          else umma_commit(tfull_bar(acc));
          if (++acc == 2) { acc = 0; acc_phase ^= 1u; }
        }
      } else {
        uint32_t turn0 = 0, turn1 = 0;                            // phases of the two accumulators' barriers
        auto into = [&](int st, int h, uint32_t add) {            // the products of one stage for accumulator h
          const uint32_t sa = smem_base + st * L::STAGE_BYTES, sb = sa + L::A_BYTES + h * L::B_BYTES;
#pragma unroll
          for (int k = 0; k < BK / UMMA_K; ++k) {
            const uint64_t adesc = A_MN ? make_smem_desc(sa + k * (UMMA_K * 128), BK * 128, 1024)
                                        : make_smem_desc(sa + k * (UMMA_K * 2), 0, 1024);
            const uint64_t bdesc = B_MN ? make_smem_desc(sb + k * (UMMA_K * 128), BK * 128, 1024)
                                        : make_smem_desc(sb + k * (UMMA_K * 2), 0, 1024);
            umma_f16_pair(tmem_base + h * BN, adesc, bdesc, idesc, k != 0 ? 1u : add);
          }
        };
        while (alive && w.next()) {
          const bool both = (w.n * SUBS + 1) * BN < p.N;          // else the second half lies past the last column
          if (!mbar_wait(tempty_bar(0), turn0 ^ 1u, p.status, 0x20u)) { alive = false; break; }
          tc_fence_after();
          int kb = w.kb0;
          if (both) {
            // the first blocks go into the first accumulator while the epilogue still reads the second; their stages wait for it
            const int lead = min(NSTAGE - 1, w.kb1 - w.kb0);
            const int from = stage;
            for (int i = 0; i < lead; ++i, ++kb) {
              if (!mbar_wait(full_bar(stage), phase, p.status, 0x21u)) { alive = false; break; }
              tc_fence_after();
              into(stage, 0, i != 0 ? 1u : 0u);
              if (++stage == NSTAGE) { stage = 0; phase ^= 1u; }
            }
            if (!alive || !mbar_wait(tempty_bar(1), turn1 ^ 1u, p.status, 0x22u)) { alive = false; break; }
            tc_fence_after();
            for (int i = 0; i < lead; ++i) {
              const int st = from + i < NSTAGE ? from + i : from + i - NSTAGE;
              into(st, 1, i != 0 ? 1u : 0u);
              umma_commit_pair(empty_bar(st), 3);
            }
          }
          for (; kb < w.kb1; ++kb) {
            if (!mbar_wait(full_bar(stage), phase, p.status, 0x21u)) { alive = false; break; }
            tc_fence_after();
            into(stage, 0, kb != w.kb0 ? 1u : 0u);
            if (both) into(stage, 1, 1u);
            umma_commit_pair(empty_bar(stage), 3);
            if (++stage == NSTAGE) { stage = 0; phase ^= 1u; }
          }
          if (!alive) break;
          umma_commit_pair(tfull_bar(0), 3);                      // (with nothing to sum at once: the epilogue writes zeros)
          turn0 ^= 1u;
          if (both) { umma_commit_pair(tfull_bar(1), 3); turn1 ^= 1u; }
        }
      }
    }
  } else if (EPI == EPI_STATS && warp >= 2 + EPI_WARPS) {
    // ===================== listed logits (warps 10..13): four words of a row at a time =====================
    const int groups = (p.list + 3) / 4;
    const long long total = p.sorted ? 0 : (long long)rows * groups, workers = (long long)gridDim.x * GATHER_WARPS;
    for (long long f = (long long)blockIdx.x * GATHER_WARPS + warp - 2 - EPI_WARPS; f < total; f += workers) {
      const int i = (int)(f / groups), k0 = (int)(f - (long long)i * groups) * 4, t = p.rowmap[i];
      long long mine = -1;                              // lane j: place of word k0 + j among this rank's, or -1
      if (lane < 4 && k0 + lane < p.list) {
        const long long word = p.idx[(long long)t * p.list + k0 + lane], v = word - p.vocab_start;
        if (v >= 0 && v < p.words && (!p.teacher || place_used(word, p.teacher[(long long)t * p.list + k0 + lane], p.vocab))) mine = v;
      }
      if (p.half) dots_of_row<__half>(p, i, k0, t, mine, lane);
      else dots_of_row<__nv_bfloat16>(p, i, k0, t, mine, lane);
    }
  } else {
    // ===================== epilogue (warps 2..9, both CTAs) =====================
    const int q = warp & 3, half = (warp - 2) >> 2;   // TMEM lane quarter this warp may access; which half of the columns it takes
    const uint32_t buf_base = smem_base + L::EPI_OFFSET + (uint32_t)(warp - 2) * L::EPI_BUF;
    const uint32_t lead_tempty[2] = {PAIR ? mapa_u32(tempty_bar(0), 0) : tempty_bar(0), PAIR ? mapa_u32(tempty_bar(1), 0) : tempty_bar(1)};
    const float unscale = (EPI >= EPI_OUT16 && p.scale) ? p.scale[1] : 1.f;
    const float ctau = p.tc_inv_tau * LOG2E;
    uint32_t chunk = 0;
    int acc = 0; uint32_t turn[2] = {0, 0};
    Work<CTAS * BM, SUBS * BN> w(M, p.N, K, p.group_m, splits, pair, npairs);
    while (alive && w.next()) {
      const int row0 = (w.m * CTAS + (int)cta) * BM + q * 32, row = row0 + lane;
      float coef = 0.f, lse = 0.f, at_label = 0.f;
      long long label = -1;
      if (EPI == EPI_DLOGITS && row < rows) {
        const int t = p.rowmap[row];
        coef = p.g[(long long)t * p.g_stride] * p.g_factor;
        if (p.scale) coef *= p.scale[0];
        lse = p.lse[row];
        if (p.label) {
          label = p.label[t] - p.piece_start;
          at_label = coef == 0.f ? 0.f : (ex2((p.z[row] * p.inv_tau - lse) * LOG2E) - 1.f) * coef;
        }
      }
      // the first listed word of this row at or behind the warp's first column, for each accumulator
      const unsigned long long* list = nullptr;
      int first_listed[SUBS];
      if (EPI == EPI_STATS && p.sorted) {
        list = row < rows ? p.sorted + (long long)p.rowmap[row] * p.list : nullptr;
#pragma unroll
        for (int h = 0; h < SUBS; ++h) {
          int lo = 0, hi = list ? p.list : 0;
          while (lo < hi) {
            const int mid = (lo + hi) >> 1;
            if ((long long)(list[mid] >> 16) < (long long)(w.n * SUBS + h) * BN + half * (BN / 2)) lo = mid + 1;
            else hi = mid;
          }
          first_listed[h] = list ? lo : p.list;
        }
      }
#pragma unroll 1
      for (int sub = 0; sub < SUBS; ++sub) {
        const int tn = w.n * SUBS + sub;
        if (SUBS == 2) {
          if (tn * BN >= p.N) break;                      // the second half lies past the last column
          acc = sub;
        }
        const long long c1 = min((long long)p.N, (long long)tn * BN + (half + 1) * (BN / 2));
        int at_list = 0;
        unsigned long long next = ~0ull;
        if (EPI == EPI_STATS && p.sorted) {
          at_list = SUBS == 2 && sub ? first_listed[SUBS - 1] : first_listed[0];
          if (at_list < p.list) next = list[at_list];
        }
        if (!mbar_wait_warp(tfull_bar(acc), turn[acc], p.status, 0x30u)) { alive = false; break; }
        tc_fence_after();
        const uint32_t t_row = tmem_base + ((uint32_t)(q * 32) << 16) + (uint32_t)(acc * BN);
        // gives this warp's part of the accumulator back: as soon as the last of it is in registers
        bool held = true;
        auto hand_back = [&] {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) {
            if (PAIR) mbar_arrive_remote(lead_tempty[acc]);
            else mbar_arrive(lead_tempty[acc]);
          }
          held = false;
        };
        if (EPI == EPI_STATS) {
          // online softmax over this warp's columns of the row; differences are taken before the scaling so that the terms that weigh
          // most (z near the maximum) keep their bits
          float m = -INFINITY, s = 0.f;
          int at = 0;
#pragma unroll 1
          for (int c2 = half * (BN / 2); c2 < (half + 1) * (BN / 2); c2 += 64) {
            const int col0 = tn * BN + c2, left = p.N - col0;
            if (left <= 0) break;
            uint32_t rr[64];
            tmem_ld_32x32(t_row + (uint32_t)c2, rr);
            tmem_ld_32x32(t_row + (uint32_t)(c2 + 32), rr + 32);
            tmem_ld_wait();
            if (!p.sorted && (c2 & 64)) hand_back();
            if (left < 64) {
#pragma unroll
              for (int j = 0; j < 64; ++j)
                if (j >= left) rr[j] = 0xff800000u;          // -inf: columns past the vocabulary
            }
            if (col0 < p.kept && row < rows) {
              float* z = p.zt + (long long)col0 * p.ldt + row;
#pragma unroll
              for (int j = 0; j < 64; ++j)
                if (j < left) z[(long long)j * p.ldt] = __uint_as_float(rr[j]);      // (`kept` is N or a multiple of 64)
            }
            float mx[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) mx[u] = __uint_as_float(rr[u]);
#pragma unroll
            for (int j = 4; j < 64; ++j) mx[j & 3] = fmaxf(mx[j & 3], __uint_as_float(rr[j]));
            const float cm = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
            if (cm > m) {
#pragma unroll
              for (int j = 63; j >= 0; --j) at = __uint_as_float(rr[j]) == cm ? c2 - half * (BN / 2) + j : at;
            }
            const float mn = fmaxf(m, cm);
            const float base = mn == -INFINITY ? 0.f : mn;
            float sm[4] = {s * ex2((m - base) * ctau), 0.f, 0.f, 0.f};
#pragma unroll
            for (int j = 0; j < 64; ++j) sm[j & 3] += ex2((__uint_as_float(rr[j]) - base) * ctau);
            s = (sm[0] + sm[1]) + (sm[2] + sm[3]);
            m = mn;
          }
          if (p.sorted) {
            for (;;) {
              const unsigned int hits = __ballot_sync(0xffffffffu, (long long)(next >> 16) < c1);
              if (!hits) break;
              const int who = __ffs(hits) - 1;
              const int col = __shfl_sync(0xffffffffu, (int)((long long)(next >> 16) - (long long)tn * BN), who);
              const float z = __uint_as_float(tmem_ld_column(t_row + (uint32_t)col));
              if (lane == who) {
                p.listed[(long long)row * p.list + (int)(next & 0xffffu)] = z * (p.tc_inv_tau / p.inv_tau);
                next = ++at_list < p.list ? list[at_list] : ~0ull;
              }
            }
          }
          if (row < rows) {
            const long long o = (long long)(2 * tn + half) * p.part_ld + row;
            p.part[o] = make_float2(m, s);
            p.part_at[o] = (unsigned char)at;
          }
        } else {
          const uint32_t sw = (uint32_t)(lane & 7);
          const bool empty = w.kb1 == w.kb0;                // nothing to sum: no rows, or more splits than blocks of a short last piece
#pragma unroll 1
          for (int c2 = half * (BN / 2); c2 < (half + 1) * (BN / 2); c2 += 64) {
            const int col0 = tn * BN + c2;
            if (col0 >= p.N) break;                       // the rest of this tile is beyond the last column
            uint32_t rr[64];
            tmem_ld_32x32(t_row + (uint32_t)c2, rr);
            tmem_ld_32x32(t_row + (uint32_t)(c2 + 32), rr + 32);
            tmem_ld_wait();
            if (c2 & 64) hand_back();
            if (EPI == EPI_DLOGITS) {
              // a row with no gradient writes zeros even where its logits are not finite
#pragma unroll
              for (int j = 0; j < 64; ++j) {
                const float e = ex2(fmaf(__uint_as_float(rr[j]), p.tc_inv_tau, -lse) * LOG2E) * coef;
                rr[j] = __float_as_uint(coef == 0.f ? 0.f : e);
              }
              const long long j0 = label - col0;
              if (__any_sync(0xffffffffu, j0 >= 0 && j0 < 64)) {
#pragma unroll
                for (int j = 0; j < 64; ++j) rr[j] = j0 == j ? __float_as_uint(at_label) : rr[j];
              }
            } else {
#pragma unroll
              for (int j = 0; j < 64; ++j) rr[j] = empty ? 0u : __float_as_uint(__uint_as_float(rr[j]) * unscale);
            }
            const uint32_t sw_row = (uint32_t)lane * 128u;
            // hidden gradient: slabs of `slab_rows` rows, a multiple of the 32 rows of a box; rows past the last are never read
            const int y = p.split ? w.split * p.slab_rows + row0 : row0;
            const bool inside = p.split ? (p.two ? row0 < p.slab_rows && (row0 & (TWO_ROWS - 1)) < rows : row0 < rows) : row0 < p.M;
            constexpr int BOXES = EPI == EPI_OUT32 ? 2 : 1, TOGETHER = EPI == EPI_OUT32 && L::EPI_BUF == 8192 ? 2 : 1;   // boxes of 128-byte rows; in one go
#pragma unroll
            for (int b0 = 0; b0 < BOXES; b0 += TOGETHER) {
              constexpr bool TURNS = EPI == EPI_OUT16 && L::EPI_BUF == 8192;
              const uint32_t buf = buf_base + (TURNS ? (chunk++ & 1u) * 4096u : 0u);
              if (lane == 0) tma_store_wait_read<TURNS ? 1 : 0>();   // the store that last read this buffer is done with it
              __syncwarp();
#pragma unroll
              for (int b = b0; b < b0 + TOGETHER; ++b) {
                const uint32_t row_addr = buf + (uint32_t)(b - b0) * 4096u + sw_row;
#pragma unroll
                for (int j = 0; j < 8; ++j) {                 // 16-byte chunk j of the row: eight 16-bit or four 32-bit columns
                  uint32_t v[4];
                  if (EPI == EPI_OUT32) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[e] = rr[32 * b + 4 * j + e];
                  } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[e] = pack16(__uint_as_float(rr[8 * j + 2 * e]), __uint_as_float(rr[8 * j + 2 * e + 1]), p.half);
                  }
                  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(row_addr + ((((uint32_t)j) ^ sw) << 4)), "r"(v[0]), "r"(v[1]), "r"(v[2]),
                               "r"(v[3])
                               : "memory");
                }
              }
              fence_proxy_async_smem();                       // generic-proxy writes -> visible to the TMA store
              __syncwarp();
              if (lane == 0) {
#pragma unroll
                for (int b = b0; b < b0 + TOGETHER; ++b) {
                  const int x = col0 + 32 * b;
                  const uint32_t src = buf + (uint32_t)(b - b0) * 4096u;
                  if (inside && x < p.N) {
                    if (EPI == EPI_OUT32 && p.accumulate) tma_reduce_add_2d(&p.tmD, src, x, y);
                    else tma_store_2d(&p.tmD, src, x, y);
                  }
                }
                tma_store_commit();
              }
            }
          }
        }
        if (held) hand_back();
        turn[acc] ^= 1u;
        if (SUBS == 1) acc ^= 1;
      }
    }
    if (lane == 0) tma_store_wait<0>();                 // staging buffers are read and the stores are complete before exit
  }

  // ---- teardown: both CTAs meet, TMEM is returned ----
  tc_fence_before();
  __syncwarp();
  if (PAIR) cluster_sync_all();
  else __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    if (PAIR) tmem_dealloc_pair(tmem_base, TMEM_COLS);
    else tmem_dealloc(tmem_base, TMEM_COLS);
  }
}

// ---------------------------------------------------------------------------------------------------------
// rows
// ---------------------------------------------------------------------------------------------------------
__device__ __forceinline__ int list_kind(const long long* idx, const float* teacher, int K, long long vocab, long long ignore_index) {
  if (!teacher) return label_kind(*idx, vocab, ignore_index);
  bool used = false, bad = false;
  for (int k = 0; k < K; ++k) {
    used |= place_used(idx[k], teacher[k], vocab);
    bad |= idx[k] >= vocab;
  }
  return bad ? 2 : used ? 1 : 0;
}

// K splits of the hidden gradient, for `n` rows.  Its tiles (256 rows x 256 of H) are few where there are few rows, or fill the last round of
// the SM pairs badly; split along the vocabulary every pair gets a part, at the price of writing and adding more results.  Times in us: a
// block of 64 words takes a tile 0.40 (0.72 a wide one, subs = 2), its read-out 2; the slabs move at 6 TB/s.  One warp; all lanes get the result.
__device__ __forceinline__ int choose_splits(int n, int H, int blocks, int pairs, int most, int subs, int lane) {
  const int tiles = max(1, (n + 255) / 256 * ((H + 256 * subs - 1) / (256 * subs)));
  float best_t = INFINITY;
  int best = 1;
  for (int s = lane + 1; s <= most; s += 32) {
    const float tile = (float)((blocks + s - 1) / s) * (subs == 2 ? 0.72f : 0.40f) + 2.f;
    const float t = (float)((tiles * s + pairs - 1) / pairs) * tile + (float)s * n * H * (8.f / 6e6f);
    if (t < best_t) { best_t = t; best = s; }
  }
  for (int o = 16; o > 0; o >>= 1) {
    const float t = __shfl_xor_sync(0xffffffffu, best_t, o);
    const int s = __shfl_xor_sync(0xffffffffu, best, o);
    if (t < best_t || (t == best_t && s < best)) { best_t = t; best = s; }
  }
  return best;
}

struct Splits { int blocks, pairs, most, subs; };        // blocks of 64 words, SM pairs (or SMs) that take the tiles, most splits

// One warp a token: what its list says, and the words of this rank sorted with their places (bitonic, `padded` = K up to a power of two);
// the rest of the places behind them as all ones.
__global__ void __launch_bounds__(128) lce_kind_kernel(const long long* __restrict__ idx, const float* __restrict__ teacher, int T, int K, int padded,
                                                       long long vocab, long long vocab_start, int words, unsigned char* kind,
                                                       unsigned long long* sorted) {
  after_previous();
  extern __shared__ unsigned long long keys_s[];
  const int t = blockIdx.x * 4 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  unsigned long long* key = keys_s + (threadIdx.x >> 5) * padded;
  if (t >= T) return;
  bool used = false, bad = false;
  for (int k = lane; k < padded; k += 32) {
    unsigned long long mine = ~0ull;
    if (k < K) {
      const long long i = idx[(long long)t * K + k], v = i - vocab_start;
      const bool u = place_used(i, teacher[(long long)t * K + k], vocab);
      used |= u;
      bad |= i >= vocab;
      if (u && v >= 0 && v < words) mine = (unsigned long long)v << 16 | (unsigned)k;
    }
    key[k] = mine;
  }
  used = __any_sync(0xffffffffu, used);
  bad = __any_sync(0xffffffffu, bad);
  if (lane == 0) kind[t] = bad ? 2 : used ? 1 : 0;
  for (int size = 2; size <= padded; size <<= 1)
    for (int gap = size >> 1; gap > 0; gap >>= 1) {
      __syncwarp();
      for (int i = lane; i < padded / 2; i += 32) {
        const int lo = (i / gap) * 2 * gap + i % gap, hi = lo + gap;
        const unsigned long long x = key[lo], y = key[hi];
        if ((x > y) == ((lo & size) == 0)) { key[lo] = y; key[hi] = x; }
      }
    }
  __syncwarp();
  for (int k = lane; k < K; k += 32) sorted[(long long)t * K + k] = key[k];
}

// Numbers the rows that stay, in the order of the tokens: pos[t] = packed row, -1 ignored, -2 a word outside the vocabulary (also noted
// in `error`); rowmap is the inverse.  One block; a warp takes 256 neighbouring tokens a round (8192 tokens a round of the block), their
// kinds as eight ballots.
__global__ void __launch_bounds__(1024) lce_scan_kernel(const long long* __restrict__ labels, const unsigned char* kind, int T, int H,
                                                        long long vocab, long long ignore_index, Splits sp, int* pos,
                                                        int* rowmap, int* count, unsigned int* error) {
  after_previous();
  __shared__ int warp_n[32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int base = 0;
  for (long long t0 = 0; t0 < T; t0 += 8192) {
    const long long first = t0 + warp * 256 + lane;
    int kd[8];
    unsigned int keep[8];
    int mine = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const long long t = first + 32 * j;
      kd[j] = t >= T ? 0 : labels ? label_kind(labels[t], vocab, ignore_index) : kind[t];
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      keep[j] = __ballot_sync(0xffffffffu, kd[j] == 1);
      mine += __popc(keep[j]);
    }
    __syncthreads();                      // the numbers of the last round have been read
    if (lane == 0) warp_n[warp] = mine;
    __syncthreads();
    const int v = warp_n[lane];
    int at = base + __reduce_add_sync(0xffffffffu, lane < warp ? v : 0);
    base += __reduce_add_sync(0xffffffffu, v);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const long long t = first + 32 * j;
      if (t < T) {
        if (kd[j] == 1) {
          const int i = at + __popc(keep[j] & ((1u << lane) - 1u));
          pos[t] = i;
          rowmap[i] = (int)t;
        } else {
          pos[t] = kd[j] == 2 ? -2 : -1;
          if (kd[j] == 2) atomicCAS(error, 0u, 0x703u);
        }
      }
      at += __popc(keep[j]);
    }
  }
  if (warp == 0) {
    const int s = choose_splits(base, H, sp.blocks, sp.pairs, sp.most, sp.subs, lane);
    if (lane == 0) { count[0] = base; count[1] = s; }
  }
}

// The packed copy of the hidden states (when rows left), a warp a token.  Tokens that left get loss 0 (NaN where a word is outside the
// vocabulary).  Blocks past the tokens zero the packed rows up to the next multiple of 64: the weight gradient reads whole blocks of 64.
// SCAN (up to SCAN_MOST tokens with short lists): every block numbers the rows itself, which saves the launches of the scan; the first
// block writes the numbers out.
constexpr int SCAN_MOST = 2048, SCAN_LIST = 16;
template <bool SCAN>
__global__ void __launch_bounds__(256) lce_rows_kernel(const uint4* __restrict__ hidden, long long ldh, const long long* __restrict__ idx,
                                                       const float* __restrict__ teacher, int Tn, int H, int K, long long vocab,
                                                       long long ignore_index, Splits sp, int* pos, int* rowmap,
                                                       int* count, unsigned int* error, uint4* packed,
                                                       float* loss) {
  after_previous();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int token_blocks = (Tn + 7) / 8, t = (int)blockIdx.x * 8 + warp, vecs = H / 8;
  int n, at = -1;
  if (SCAN) {
    __shared__ unsigned int keep[SCAN_MOST / 32], wrong[SCAN_MOST / 32];
    const int words = (Tn + 31) / 32;
    for (int w = warp; w < words; w += 8) {
      const int u = w * 32 + lane;
      const int kd = u < Tn ? list_kind(idx + (long long)u * K, teacher ? teacher + (long long)u * K : nullptr, K, vocab, ignore_index) : 0;
      const unsigned int k = __ballot_sync(0xffffffffu, kd == 1), b = __ballot_sync(0xffffffffu, kd == 2);
      if (lane == 0) { keep[w] = k; wrong[w] = b; }
    }
    __syncthreads();
    // rows kept in words below `w`, over all of them for the last
    auto below = [&](int w) {
      int c = 0;
      for (int i = lane; i < w; i += 32) c += __popc(keep[i]);
      return __reduce_add_sync(0xffffffffu, c);
    };
    n = below(words);
    if (t < Tn) {
      const unsigned int bit = 1u << (t & 31);
      const int b = below(t >> 5);
      at = keep[t >> 5] & bit ? b + __popc(keep[t >> 5] & (bit - 1u)) : wrong[t >> 5] & bit ? -2 : -1;
    }
    if (blockIdx.x == 0) {
      for (int w = warp; w < words; w += 8) {
        const int u = w * 32 + lane, b = below(w);
        const unsigned int bit = 1u << lane;
        if (u < Tn) {
          if (keep[w] & bit) {
            const int i = b + __popc(keep[w] & (bit - 1u));
            pos[u] = i;
            rowmap[i] = u;
          } else {
            pos[u] = wrong[w] & bit ? -2 : -1;
            if (wrong[w] & bit) atomicCAS(error, 0u, 0x703u);
          }
        }
      }
      if (warp == 0) {
        const int s = choose_splits(n, H, sp.blocks, sp.pairs, sp.most, sp.subs, lane);
        if (lane == 0) { count[0] = n; count[1] = s; }
      }
    }
  } else {
    n = *count;
    if (t < Tn) at = pos[t];
  }
  if ((int)blockIdx.x >= token_blocks) {
    const int r = n + ((int)blockIdx.x - token_blocks) * 8 + warp;
    if (n == Tn || r >= min(Tn, (n + 63) / 64 * 64)) return;
    for (int c = lane; c < vecs; c += 32) packed[(long long)r * vecs + c] = make_uint4(0, 0, 0, 0);
    return;
  }
  if (t >= Tn) return;
  if (at < 0) {
    if (lane == 0) loss[t] = at == -2 ? NAN : 0.f;
    return;
  }
  if (n == Tn) return;
  const uint4* h = hidden + t * (ldh / 8);
#pragma unroll 4
  for (int c = lane; c < vecs; c += 32) packed[(long long)at * vecs + c] = h[c];
}

// ---------------------------------------------------------------------------------------------------------
// join of the (max, sum) pairs, loss
// ---------------------------------------------------------------------------------------------------------
__device__ __forceinline__ void lce_finish(float m, float s, float dot, float ent, float inv_tau, float tau2, float* lse, float* loss) {
  const float ls = (float)log((double)s);
  *lse = m * inv_tau + ls;
  *loss = tau2 * (ent + (m * inv_tau - dot) + ls);       // the two large numbers are subtracted first
}

// R rows a block, S threads a row over the parts of `width` columns (neighbouring threads take neighbouring rows); the order of the sums is fixed.
// Then one warp a row computes the largest logit again in fp32 and rebases the sum on it: s = 1 + (s - 1) exp((m - m') / tau), m' the new
// value; for a list it makes the weights q, dot = sum q z / tau and ent = sum q log q.
// 256 threads and 8 rows keep five blocks on an SM (8192 rows, 128256 words: 52 us with 32 rows a block); few rows take 128 threads each.
template <typename T, int R, int S>
__global__ void __launch_bounds__(R * S) lce_join_kernel(const float2* part, const unsigned char* part_at,
                                                        long long part_ld, int parts, int width, const T* __restrict__ hidden, long long ldh,
                                                        const T* __restrict__ weight, long long ldw, int H, float inv_tau, float tc_inv_tau,
                                                        float tau2, const int* count, const int* rowmap,
                                                        const long long* __restrict__ idx, const float* __restrict__ teacher, int K,
                                                        long long vocab, long long vocab_start, int words, const float* z, float* qout,
                                                        float* dot, float* ent, float* mo,
                                                        float* so, float* lse, float* loss) {
  after_previous();
  __shared__ float ms[S][R + 1], ss[S][R + 1];
  __shared__ int as[S][R + 1];
  const int n = *count;
  if ((int)blockIdx.x * R >= n) return;
  const float c = tc_inv_tau * LOG2E;
  {
    const int r = threadIdx.x % R, y = threadIdx.x / R, row = blockIdx.x * R + r;
    float m = -INFINITY, s = 0.f;
    int at = 0;
    if (row < n) {
#pragma unroll 4
      for (int i = y; i < parts; i += S) {
        const float2 v = part[(long long)i * part_ld + row];
        const float mn = fmaxf(m, v.x), base = mn == -INFINITY ? 0.f : mn;
        s = s * ex2((m - base) * c) + v.y * ex2((v.x - base) * c);
        if (v.x > m) at = i;
        m = mn;
      }
      at = at * width + part_at[(long long)at * part_ld + row];
    }
    ms[y][r] = m;
    ss[y][r] = s;
    as[y][r] = at;
  }
  __syncthreads();
  const int r = threadIdx.x >> 5, lane = threadIdx.x & 31, row = blockIdx.x * R + r;
  if (r >= R || row >= n) return;
  float mm = -INFINITY;
  int word = 0;
#pragma unroll
  for (int i = lane; i < S; i += 32)
    if (ms[i][r] > mm) { mm = ms[i][r]; word = as[i][r]; }
  const float mine = mm;
  mm = warp_max(mm);
  const unsigned int who = __ballot_sync(0xffffffffu, mine == mm);
  word = __shfl_sync(0xffffffffu, word, who ? __ffs(who) - 1 : 0);
  float s = 0.f;
#pragma unroll
  for (int i = lane; i < S; i += 32) s += ss[i][r] * ex2((ms[i][r] - (ms[i][r] == -INFINITY && mm != -INFINITY ? 0.f : mm)) * c);
  s = warp_sum(s);
  const int t = rowmap[row];
  const float again = warp_dot(hidden + t * ldh, weight + word * ldw, H, lane);
  float d, e = 0.f;
  if (teacher) {
    const long long* list = idx + (long long)t * K;
    const float* a = teacher + (long long)t * K;
    const float* zi = z + (long long)row * K;
    float mx = -INFINITY, sum = 0.f;
    for (int k = lane; k < K; k += 32)
      if (place_used(list[k], a[k], vocab)) mx = fmaxf(mx, a[k]);
    mx = warp_max(mx);
    for (int k = lane; k < K; k += 32)
      if (place_used(list[k], a[k], vocab)) sum += ex2((a[k] - mx) * (inv_tau * LOG2E));
    sum = warp_sum(sum);
    const float ls = (float)log((double)sum);
    d = 0.f;
    for (int k = lane; k < K; k += 32) {
      float q = 0.f;
      if (place_used(list[k], a[k], vocab)) {
        const float b = (a[k] - mx) * inv_tau;
        q = ex2(b * LOG2E) / sum;
        const long long v = list[k] - vocab_start;
        if (v >= 0 && v < words) d = fmaf(q, zi[k] * inv_tau, d);
        if (!(q == 0.f)) e = fmaf(q, b - ls, e);
      }
      qout[(long long)row * K + k] = q;
    }
    d = warp_sum(d);
    e = warp_sum(e);
  } else {
    const long long v = idx[t] - vocab_start;
    d = v >= 0 && v < words ? z[row] * inv_tau : 0.f;
  }
  if (lane == 0) {
    const float m2 = mm == -INFINITY ? mm : again;         // nothing but -inf: NaN, as the formula
    const float s2 = 1.f + (s - 1.f) * ex2(fmaf(mm, tc_inv_tau, -(m2 * inv_tau)) * LOG2E);
    if (mo) {
      mo[row] = m2;
      so[row] = s2;
      dot[row] = d;
      ent[row] = e;
    } else {
      float l, o;
      lce_finish(m2, s2, d, e, inv_tau, tau2, &l, &o);
      lse[row] = l;
      loss[t] = o;
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
__global__ void __launch_bounds__(1024) lce_scale_kernel(const float* __restrict__ g, int g_stride, const int* rowmap,
                                                         const int* count, float factor, float* scale) {
  after_previous();
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
__global__ void __launch_bounds__(256) lce_listed_kernel(T* dz, long long ld_row, long long ld_word, int two, const long long* __restrict__ idx,
                                                         const float* z, const float* q, const float* lse,
                                                         const int* rowmap, const int* count, int K,
                                                         long long piece_start, int piece_cols, const float* __restrict__ g, int g_stride,
                                                         float g_factor, float inv_tau, const float* scale) {
  after_previous();
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
  const float d = coef == 0.f ? 0.f : (p - sum) * coef;
  const T hi = from_f<T>(d);
  dz[i * ld_row + v * ld_word] = hi;
  if (two) dz[(i + TWO_ROWS) * ld_row + v * ld_word] = from_f<T>(d - to_f(hi));
}

// dz of kept logits, both [words, ldt] with the rows innermost: eight rows of one word a thread, 256 rows a block.  Rows past the last
// are zero up to the next multiple of 64, which is what the products read.  TWO: dz is [words, 2 ldt], the second half what the rounding of
// the first left.  Bound by the memory rate: one wave of blocks, with the logits of DZ_AHEAD words of each thread in flight (4096 rows x
// 32000 words 120 us, 6.5 TB/s: two words at four blocks an SM spill, 129; four waves of blocks of three words 138).
constexpr int DZ_AHEAD = 4, DZ_RESIDENT = 2;
template <typename T, bool TWO>
__global__ void __launch_bounds__(256, DZ_RESIDENT) lce_dz_kernel(const float* __restrict__ zt, T* __restrict__ dz, int ldt, int words, const float* lse,
                                                        const long long* __restrict__ label, const float* z,
                                                        const int* rowmap, const int* count, long long word_start,
                                                        const float* __restrict__ g, int g_stride, float g_factor, float inv_tau,
                                                        float tc_inv_tau, const float* scale) {
  after_previous();
  const int n = *count, groups = min(ldt, (n + 63) / 64 * 64) / 8, chunks = (groups + 31) / 32;
  if (n == 0) return;
  // block b takes rows of chunk b mod chunks; its threads take `per` words a round, always the same rows
  const int chunk = (int)blockIdx.x % chunks, wide = min(groups - chunk * 32, 32), per = 256 / wide, sub = threadIdx.x / wide;
  if (sub >= per) return;
  const int r0 = (chunk * 32 + (int)threadIdx.x % wide) * 8;
  float coef[8], ls[8];
  int lab[8];                                   // word of the piece that is the row's label, or -1
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int i = r0 + j;
    coef[j] = ls[j] = 0.f;
    lab[j] = -1;
    if (i < n) {
      const int t = rowmap[i];
      coef[j] = g[(long long)t * g_stride] * g_factor;
      if (scale) coef[j] *= scale[0];
      ls[j] = lse[i];
      if (label) {
        const long long l = label[t] - word_start;
        if (l >= 0 && l < words) lab[j] = (int)l;
      }
    }
  }
  const unsigned step = ((gridDim.x - chunk + chunks - 1) / chunks) * per;
  unsigned v = (blockIdx.x / chunks) * per + sub;
  const long long hop = (long long)step * ldt;
  const float* from = zt + (long long)v * ldt + r0;
  T* to = dz + (long long)v * (TWO ? 2 : 1) * ldt + r0;
  while (v < (unsigned)words) {
    Vec8<float> x[DZ_AHEAD];
#pragma unroll
    for (int u = 0; u < DZ_AHEAD; ++u)
      if (v + u * step < (unsigned)words) x[u].load(from + u * hop);
    from += DZ_AHEAD * hop;
#pragma unroll
    for (int u = 0; u < DZ_AHEAD; ++u) {
      if (v >= (unsigned)words) return;
      float f[8];
      x[u].to_float(f);
      bool listed = false;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float e = ex2(fmaf(f[j], tc_inv_tau, -ls[j]) * LOG2E) * coef[j];
        f[j] = coef[j] == 0.f ? 0.f : e;
        listed |= lab[j] == (int)v;
      }
      if (listed) {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (lab[j] == (int)v && coef[j] != 0.f) f[j] = (ex2((z[r0 + j] * inv_tau - ls[j]) * LOG2E) - 1.f) * coef[j];
      }
      Vec8<T> w;
      w.from_float(f);
      w.store(to);
      if (TWO) {
        float hi[8];
        w.to_float(hi);
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j] -= hi[j];
        w.from_float(f);
        w.store(to + ldt);
      }
      v += step;
      to += TWO ? 2 * hop : hop;
    }
  }
}

// d hidden: the fp32 slabs of the K splits, added in a fixed order, back in the order of the tokens; zero rows for tokens that left.
// Y threads share the slabs of eight columns: one where there are few slabs, eight where there are many (few rows), which would
// otherwise be a chain of loads (one token, 37 slabs: 13 us with one thread).
template <typename T, int Y>
__global__ void __launch_bounds__(256) lce_dhidden_kernel(const float* acc, const int* count, long long slab, int two, const int* pos,
                                                          T* __restrict__ out, int Tn, int H) {
  after_previous();
  constexpr int X = 256 / Y;
  __shared__ float part[Y == 1 ? 1 : Y][X][9];
  const int x = threadIdx.x % X, y = threadIdx.x / X;
  const int per_row = H / 8, terms = count[1] * (two ? 2 : 1);
  const long long total = (long long)Tn * per_row;
  for (long long f0 = (long long)blockIdx.x * X; f0 < total; f0 += (long long)gridDim.x * X) {
    const long long f = f0 + x;
    const bool in = f < total;
    const int t = in ? (int)(f / per_row) : 0, c = in ? (int)(f - (long long)t * per_row) * 8 : 0;
    const int at = in ? pos[t] : -1;
    float o[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (at >= 0) {
      const float* a = acc + (long long)at * H + c;
#pragma unroll 4
      for (int s = y; s < terms; s += Y) {
        const float* b = a + (two ? (s >> 1) * slab + (s & 1) * (TWO_ROWS * (long long)H) : s * slab);
        const float4 u = __ldcs(reinterpret_cast<const float4*>(b)), v = __ldcs(reinterpret_cast<const float4*>(b + 4));
        o[0] += u.x; o[1] += u.y; o[2] += u.z; o[3] += u.w;
        o[4] += v.x; o[5] += v.y; o[6] += v.z; o[7] += v.w;
      }
    }
    if (Y > 1) {
      __syncthreads();                      // the sums of the last round have been read
#pragma unroll
      for (int j = 0; j < 8; ++j) part[y][x][j] = o[j];
      __syncthreads();
      if (y == 0)
#pragma unroll
        for (int j = 0; j < 8; ++j)
#pragma unroll
          for (int i = 1; i < Y; ++i) o[j] += part[i][x][j];
    }
    if (in && y == 0) {
      Vec8<T> w;
      w.from_float(o);
      w.store(out + (long long)t * H + c);
    }
  }
}

// ---------------------------------------------------------------------------------------------------------
// launchers
// ---------------------------------------------------------------------------------------------------------
#define LCE_FIRST(name, kern, grid, block, smem, ...)          \
  do {                                                         \
    auto k__ = kern;                                           \
    k__<<<grid, block, smem, s>>>(__VA_ARGS__);                \
    MSB_CHECK_LAUNCH(name);                                    \
  } while (0)
#define LCE_AFTER(name, kern, grid, block, smem, ...)          \
  do {                                                         \
    auto k__ = kern;                                           \
    msb::launch_after(k__, dim3(grid), block, smem, s, __VA_ARGS__); \
    MSB_CHECK_LAUNCH(name);                                    \
  } while (0)

// SMs that the products may take: all, or as many as the caller has left to GEMM-class kernels.
int product_sms() {
  const int cap = msb_gemm_get_cta_limit(), sms = msb::num_sms();
  return cap > 0 && cap < sms ? std::max(cap, 2) : sms;
}

template <int EPI, bool A_MN, bool B_MN, int HOW>
int launch_gemm_on(const LceGemm& p, int most_splits, bool first, cudaStream_t s) {
  using L = Cfg<EPI, HOW>;
  auto kern = lce_gemm_kernel<EPI, A_MN, B_MN, HOW>;
  static std::atomic<unsigned long long> stated{0};
  if (int bad = msb::allow_smem((const void*)kern, L::TOTAL, "lce_gemm", stated)) return bad;
  const long long items = (long long)((p.M + L::CTAS * BM - 1) / (L::CTAS * BM)) * ((p.N + L::SUBS * BN - 1) / (L::SUBS * BN)) * most_splits;
  const unsigned grid = L::CTAS * (unsigned)std::min<long long>(items, product_sms() / L::CTAS);
  if (first) kern<<<grid, L::THREADS, L::TOTAL, s>>>(p);
  else msb::launch_after(kern, dim3(grid), L::THREADS, L::TOTAL, s, p);
  MSB_CHECK_LAUNCH("lce_gemm");
  return 0;
}
template <int EPI, bool A_MN, bool B_MN>
int launch_gemm(const LceGemm& p, How how, int most_splits, bool first, cudaStream_t s) {
  if constexpr (EPI != EPI_OUT16)
    if (how == SINGLE) return launch_gemm_on<EPI, A_MN, B_MN, SINGLE>(p, most_splits, first, s);
  if (how == WIDE) return launch_gemm_on<EPI, A_MN, B_MN, WIDE>(p, most_splits, first, s);
  return launch_gemm_on<EPI, A_MN, B_MN, PAIRED>(p, most_splits, first, s);
}

// How a product of M x N with sums over K is tiled: by its modelled time in us, rounds of tiles over the SM pairs.  A block of 64 of the
// sum takes a pair 0.40 on 256 x 256 and 0.72 on 256 x 512 (A is staged once for both halves: shared memory, whose bandwidth bounds the
// former, moves a quarter less, and so do L2 and the power it takes), but nothing hides the read-out of the wide tile, 2.  `rows` of at
// most 128 take single CTAs.  (In turn on one GPU at its power limit, 8192 x 128256 x 4096: forward 6.63 -> 6.45 ms, backward 20.3 -> 19.4;
// 1500 x 60000 x 1024, where the rule keeps pairs: forward 190, 193 wide.)  The rule counts all tokens: how many stay is not known here.
float modelled_us(long long M, long long N, long long K, int splits, How how) {
  const int pairs = std::max(1, product_sms() / 2), width = how == WIDE ? 512 : 256;
  const long long tiles = ((M + 255) / 256) * ((N + width - 1) / width) * splits, blocks = ((K + BK - 1) / BK + splits - 1) / splits;
  return (float)((tiles + pairs - 1) / pairs) * (how == WIDE ? 0.72f * blocks + 2.f : 0.40f * blocks);
}
How choose_how(long long M, long long N, long long K, int most_splits = 1) {
  float best[2] = {INFINITY, INFINITY};
  for (int s = 1; s <= most_splits; ++s) {
    best[0] = std::min(best[0], modelled_us(M, N, K, s, PAIRED));
    best[1] = std::min(best[1], modelled_us(M, N, K, s, WIDE));
  }
  return best[1] < best[0] ? WIDE : PAIRED;
}
How rows_how(int rows, long long N, long long K, int most_splits = 1) { return rows <= BM ? SINGLE : choose_how(rows, N, K, most_splits); }

// Rows of the boxes that load W as [words, H], for T tokens.
uint32_t words_box(int T) { return T <= BM ? 256 : 128; }

// 1 / tau for logits that the tensor cores summed over H products (see the top of the file).
float tc_scale(float inv_tau, int H) { return (float)((double)inv_tau * (1.0 + 0.26 * (H / 16) / 16777216.0)); }

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
  int* count;                  // [2]: rows that stay, K splits
  unsigned char* kind;         // [T] scratch (lists)
  unsigned long long* sorted;  // [T, K] scratch (lists)
  void* packed;                // [T, H]
  float* z;                    // [T, K]
  float* q;                    // [T, K]
  float* dot;                  // [T]
  float* ent;                  // [T]
  float* lse;                  // [T]
  float* loss;                 // [T]
  float* part;                 // [ceil(V / 256) * 2, T] pairs, scratch
  unsigned char* part_at;      // [ceil(V / 256) * 2, T] scratch
  float* zt;                   // [kept, ldt] logits of the first `kept` words, for the backward, or null
  int ldt;                     // T rounded up to a multiple of 8; TWO_ROWS for up to so many tokens
  int kept;                    // V, or a multiple of 64
  float* mx;                   // [T], [T]: local statistics for the vocabulary-parallel form, else null
  float* sum;
  // backward
  const float* g;
  long long g_stride;          // 0: one value for all tokens
  void* dz;                    // scratch of a piece: [T, piece], row pitch ldz; of kept words [piece, ldt], or [piece, 2 TWO_ROWS]
  long long ldz;
  int piece;                   // columns of a piece (a multiple of 256)
  float* acc;                  // [splits, slab_rows, H] fp32 scratch, or null: no hidden gradient
  int splits, slab_rows;       // most K splits (both directions are given the same, and the same piece)
  void* dhidden;               // [T, H]
  void* dweight;               // [V, H], 16-bit or fp32; null: no weight gradient
  int dweight_fp32_add;        // dweight is fp32 and added to
  float* scale;                // [2] scratch (fp16), else null
  unsigned int* status;        // [0] expired waits, [1] words outside the vocabulary
};

// Tiles of the hidden gradient (both directions ask: the forward counts its splits).
static How dhidden_how(const MsbLceArgs* a) { return rows_how(a->T, a->H, std::min(a->piece, a->V), a->splits); }

static int lce_check(const MsbLceArgs* a) {
  MSB_REQUIRE(a->T > 0 && a->H > 0 && a->V > 0 && a->K > 0, "linear_ce: empty problem T=%d H=%d V=%d K=%d", a->T, a->H, a->V, a->K);
  MSB_REQUIRE(a->dtype == MSB_BF16 || a->dtype == MSB_F16, "linear_ce: dtype code %d is not bf16 or fp16", a->dtype);
  MSB_REQUIRE(a->H % 8 == 0 && a->ldh % 8 == 0 && a->ldw % 8 == 0, "linear_ce: H=%d and the row pitches must be multiples of 8", a->H);
  MSB_REQUIRE(a->status != nullptr, "linear_ce: status words are required");
  MSB_REQUIRE(a->tau > 0.f, "linear_ce: the temperature must be positive");
  MSB_REQUIRE(a->K == 1 || a->teacher, "linear_ce: lists need teacher logits");
  MSB_REQUIRE(a->K <= 1024, "linear_ce: %d listed words", a->K);
  MSB_REQUIRE(!a->zt || (a->ldt % 8 == 0 && a->ldt >= a->T && (a->T > TWO_ROWS || a->ldt == TWO_ROWS)), "linear_ce: pitch %d of the kept logits", a->ldt);
  MSB_REQUIRE(a->zt ? a->kept == a->V || (a->kept > 0 && a->kept < a->V && a->kept % 64 == 0 && a->T > TWO_ROWS) : a->kept == 0,
              "linear_ce: logits of %d words kept", a->kept);
  MSB_REQUIRE(a->piece > 0 && a->piece % 256 == 0 && a->splits >= 1, "linear_ce: piece of %d columns, %d splits", a->piece, a->splits);
  return 0;
}

template <typename DT>
static int lce_forward(const MsbLceArgs* a, cudaStream_t s) {
  const float inv_tau = 1.f / a->tau, tau2 = a->tau * a->tau;
  const DT* hidden = (const DT*)a->hidden;
  const DT* weight = (const DT*)a->weight;
  const Splits sp = {(std::min(a->piece, a->V) + BK - 1) / BK, a->T <= BM ? product_sms() : product_sms() / 2, a->splits,
                     dhidden_how(a) == WIDE ? 2 : 1};
  const bool scan = a->T <= SCAN_MOST && a->K <= SCAN_LIST;
  if (!scan) {
    if (a->teacher) {
      int padded = 1;
      while (padded < a->K) padded *= 2;
      LCE_FIRST("lce_kind", lce_kind_kernel, (a->T + 3) / 4, 128, 4 * padded * 8, a->idx, a->teacher, a->T, a->K, padded, a->vocab, a->vocab_start,
                a->V, a->kind, a->sorted);
    }
    const long long* labels = a->teacher ? nullptr : a->idx;
    if (a->teacher)
      LCE_AFTER("lce_scan", lce_scan_kernel, 1, 1024, 0, labels, a->kind, a->T, a->H, a->vocab, a->ignore_index, sp, a->pos, a->rowmap, a->count,
                a->status + 1);
    else
      LCE_FIRST("lce_scan", lce_scan_kernel, 1, 1024, 0, labels, a->kind, a->T, a->H, a->vocab, a->ignore_index, sp, a->pos, a->rowmap, a->count,
                a->status + 1);
  }
  const unsigned grid = (unsigned)((a->T + 7) / 8 + 8);
#define LCE_ROWS(HOW, SCAN)                                                                                                                  \
  HOW("lce_rows", lce_rows_kernel<SCAN>, grid, 256, 0, (const uint4*)hidden, a->ldh, a->idx, a->teacher, a->T, a->H, a->K, a->vocab,           \
      a->ignore_index, sp, a->pos, a->rowmap, a->count, a->status + 1, (uint4*)a->packed, a->loss)
  if (scan) LCE_ROWS(LCE_FIRST, true);
  else LCE_ROWS(LCE_AFTER, false);
#undef LCE_ROWS
  LceGemm p;
  memset(&p, 0, sizeof(p));
  const CUtensorMapDataType dt = map_type(a->dtype);
  int rc;
  if ((rc = make_tmap_2d(&p.tmA, hidden, dt, 2, a->T, a->H, a->ldh, BM, BK))) return rc;
  if ((rc = make_tmap_2d(&p.tmPacked, a->packed, dt, 2, a->T, a->H, a->H, BM, BK))) return rc;
  if ((rc = make_tmap_2d(&p.tmB, weight, dt, 2, a->V, a->H, a->ldw, words_box(a->T), BK))) return rc;
  p.M = a->T; p.N = a->V; p.K = a->H;
  p.rows = a->count; p.all_rows = a->T;
  p.group_m = GROUP_LOGITS;
  p.half = a->dtype == MSB_F16;
  p.part = reinterpret_cast<float2*>(a->part); p.part_at = a->part_at; p.part_ld = a->T;
  p.zt = a->zt; p.ldt = a->ldt; p.kept = a->kept;
  p.sorted = a->teacher && !scan ? a->sorted : nullptr;
  p.idx = a->idx; p.teacher = a->teacher; p.listed = a->z; p.list = a->K;
  p.hidden = hidden; p.weight = weight; p.ldh = a->ldh; p.ldw = a->ldw; p.vocab_start = a->vocab_start; p.vocab = a->vocab;
  p.width = a->H; p.words = a->V;
  p.rowmap = a->rowmap;
  p.inv_tau = inv_tau; p.tc_inv_tau = tc_scale(inv_tau, a->H);
  p.status = a->status;
  if ((rc = launch_gemm<EPI_STATS, false, false>(p, rows_how(a->T, a->V, a->H), 1, false, s))) return rc;
  constexpr int width = 128;
#define LCE_JOIN(R, S)                                                                                                                       \
  LCE_AFTER("lce_join", (lce_join_kernel<DT, R, S>), (a->T + R - 1) / R, R * S, 0, p.part, p.part_at, p.part_ld, (a->V + width - 1) / width, width, hidden, \
            a->ldh, weight, a->ldw, a->H, inv_tau, p.tc_inv_tau, tau2, a->count, a->rowmap, a->idx, a->teacher, a->K, a->vocab, a->vocab_start, \
            a->V, a->z, a->q, a->dot, a->ent, a->mx, a->sum, a->lse, a->loss)
  if (a->T <= 1024) LCE_JOIN(4, 128);
  else LCE_JOIN(8, 32);
#undef LCE_JOIN
  return 0;
}

// Scan, rows, GEMM with row statistics, join.  With `mx` the join stops at the local (max, sum).
MSB_API int msb_lce_forward(const MsbLceArgs* a, cudaStream_t s) {
  if (int rc = lce_check(a)) return rc;
  return a->dtype == MSB_F16 ? lce_forward<__half>(a, s) : lce_forward<__nv_bfloat16>(a, s);
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

template <typename DT>
static int lce_backward(const MsbLceArgs* a, cudaStream_t s) {
  const float inv_tau = 1.f / a->tau;
  const CUtensorMapDataType dt = map_type(a->dtype);
  const long long* label = a->teacher ? nullptr : a->idx;
  DT* dz = (DT*)a->dz;
  if (a->scale) {
    LCE_FIRST("lce_scale", lce_scale_kernel, 1, 1024, 0, a->g, (int)a->g_stride, a->rowmap, a->count, a->tau, a->scale);
  }
  LceGemm p;
  memset(&p, 0, sizeof(p));
  p.rows = a->count; p.all_rows = a->T;
  p.half = a->dtype == MSB_F16;
  p.rowmap = a->rowmap; p.lse = a->lse;
  p.g = a->g; p.g_stride = (int)a->g_stride; p.g_factor = a->tau;
  p.inv_tau = inv_tau; p.tc_inv_tau = tc_scale(inv_tau, a->H);
  p.label = label; p.z = a->z;
  p.scale = a->scale;
  p.status = a->status;
  const int two = a->zt && a->T <= TWO_ROWS, dz_rows = two ? 2 * TWO_ROWS : a->T, dz_ld = two ? 2 * TWO_ROWS : a->ldt;
  int rc, cols;
  for (long long v0 = 0; v0 < a->V; v0 += cols) {
    const bool kept = v0 < a->kept;
    cols = (int)std::min<long long>(a->piece, (kept ? a->kept : a->V) - v0);
    const DT* w = (const DT*)a->weight + v0 * a->ldw;
    // dz of the piece
    if (kept) {
      const int chunks = (a->ldt + 255) / 256, per = 256 / std::min(32, a->ldt / 8);
      const long long most = (long long)((cols + per - 1) / per) * chunks;
      const unsigned grid = (unsigned)std::max<long long>(chunks, std::min<long long>(most, (long long)msb::num_sms() * DZ_RESIDENT));
#define LCE_DZ(HOW, TWO)                                                                                                                     \
  HOW("lce_dz", (lce_dz_kernel<DT, TWO>), grid, 256, 0, a->zt + v0 * a->ldt, dz, a->ldt, cols, a->lse, label, a->z, a->rowmap, a->count,        \
      a->vocab_start + v0, a->g, (int)a->g_stride, a->tau, inv_tau, p.tc_inv_tau, a->scale)
      if (a->scale || v0 > 0) {
        if (two) LCE_DZ(LCE_AFTER, true);
        else LCE_DZ(LCE_AFTER, false);
      } else {
        if (two) LCE_DZ(LCE_FIRST, true);
        else LCE_DZ(LCE_FIRST, false);
      }
#undef LCE_DZ
    } else {
      if ((rc = make_tmap_2d(&p.tmA, a->hidden, dt, 2, a->T, a->H, a->ldh, BM, BK))) return rc;
      if ((rc = make_tmap_2d(&p.tmPacked, a->packed, dt, 2, a->T, a->H, a->H, BM, BK))) return rc;
      if ((rc = make_tmap_2d(&p.tmB, w, dt, 2, cols, a->H, a->ldw, words_box(a->T), BK))) return rc;
      if ((rc = make_tmap_2d(&p.tmD, dz, dt, 2, a->T, cols, a->ldz, 32, 64))) return rc;
      p.M = a->T; p.N = cols; p.K = a->H; p.group_m = GROUP_LOGITS; p.rows_on_k = 0; p.split = 0; p.two = 0; p.piece_start = a->vocab_start + v0;
      if ((rc = launch_gemm<EPI_DLOGITS, false, false>(p, rows_how(a->T, cols, a->H), 1, v0 == 0 && !a->scale, s))) return rc;
    }
    if (a->teacher) {
      const long long places = (long long)a->T * a->K;
      LCE_AFTER("lce_listed", lce_listed_kernel<DT>, (unsigned)((places + 255) / 256), 256, 0, dz, kept ? 1 : a->ldz, kept ? dz_ld : 1, two,
                a->idx, a->z, a->q, a->lse, a->rowmap, a->count, a->K, a->vocab_start + v0, cols, a->g, (int)a->g_stride, a->tau, inv_tau,
                a->scale);
    }
    if (a->acc) {
      if (kept) rc = make_tmap_2d(&p.tmA, dz, dt, 2, cols, dz_rows, dz_ld, BK, 64);
      else rc = make_tmap_2d(&p.tmA, dz, dt, 2, a->T, cols, a->ldz, BM, BK);
      if (rc) return rc;
      if ((rc = make_tmap_2d(&p.tmB, w, dt, 2, cols, a->H, a->ldw, BK, 64))) return rc;
      if ((rc = make_tmap_2d(&p.tmD, a->acc, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 4, (uint64_t)a->splits * a->slab_rows, a->H, a->H, 32, 32))) return rc;
      p.M = dz_rows; p.N = a->H; p.K = cols; p.group_m = GROUP_GRADS; p.rows_on_k = 0; p.two = two;
      p.split = 1; p.slab_rows = a->slab_rows; p.accumulate = v0 > 0;
      rc = kept ? launch_gemm<EPI_OUT32, true, true>(p, dhidden_how(a), a->splits, false, s)
                 : launch_gemm<EPI_OUT32, false, true>(p, dhidden_how(a), a->splits, false, s);
      if (rc) return rc;
    }
    if (a->dweight) {
      if (kept) rc = make_tmap_2d(&p.tmA, dz, dt, 2, cols, dz_rows, dz_ld, BM, BK);
      else rc = make_tmap_2d(&p.tmA, dz, dt, 2, a->T, cols, a->ldz, BK, 64);
      if (rc) return rc;
      if ((rc = make_tmap_2d(&p.tmB, a->hidden, dt, 2, a->T, a->H, a->ldh, BK, 64))) return rc;
      if ((rc = make_tmap_2d(&p.tmPacked, a->packed, dt, 2, a->T, a->H, a->H, BK, 64))) return rc;
      p.M = cols; p.N = a->H; p.K = a->T; p.group_m = GROUP_GRADS; p.rows_on_k = 1; p.split = 0; p.two = two;
      const How how = choose_how(cols, a->H, a->T);
      if (a->dweight_fp32_add) {
        if ((rc = make_tmap_2d(&p.tmD, (float*)a->dweight + v0 * a->H, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 4, cols, a->H, a->H, 32, 32))) return rc;
        p.accumulate = 1;
        rc = kept ? launch_gemm<EPI_OUT32, false, true>(p, how, 1, false, s) : launch_gemm<EPI_OUT32, true, true>(p, how, 1, false, s);
      } else {
        if ((rc = make_tmap_2d(&p.tmD, (DT*)a->dweight + v0 * a->H, dt, 2, cols, a->H, a->H, 32, 64))) return rc;
        p.accumulate = 0;
        rc = kept ? launch_gemm<EPI_OUT16, false, true>(p, how, 1, false, s) : launch_gemm<EPI_OUT16, true, true>(p, how, 1, false, s);
      }
      if (rc) return rc;
    }
  }
  if (a->acc) {
    const long long vecs = (long long)a->T * (a->H / 8);
#define LCE_DHIDDEN(Y)                                                                                                                       \
  LCE_AFTER("lce_dhidden", (lce_dhidden_kernel<DT, Y>),                                                                                       \
            (unsigned)std::min<long long>((vecs + 256 / Y - 1) / (256 / Y), (long long)msb::num_sms() * 16), 256, 0, a->acc, a->count,         \
            (long long)a->slab_rows * a->H, two, a->pos, (DT*)a->dhidden, a->T, a->H)
    if (a->splits >= 16) LCE_DHIDDEN(8);
    else LCE_DHIDDEN(1);
#undef LCE_DHIDDEN
  }
  return 0;
}

// Hidden and weight gradients, a piece of the vocabulary at a time.
MSB_API int msb_lce_backward(const MsbLceArgs* a, cudaStream_t s) {
  if (int rc = lce_check(a)) return rc;
  MSB_REQUIRE(a->kept == a->V || (a->ldz % 8 == 0 && a->ldz >= std::min(a->piece, a->V)), "linear_ce: pitch %lld of a piece of %d columns", a->ldz, a->piece);
  const int dz_rows = a->zt && a->T <= TWO_ROWS ? 2 * TWO_ROWS : a->T;
  MSB_REQUIRE(!a->acc || (a->slab_rows >= dz_rows && a->slab_rows % 32 == 0 && (long long)a->splits * a->slab_rows < 0x7fffffffll),
              "linear_ce: %d slabs of %d rows", a->splits, a->slab_rows);
  return a->dtype == MSB_F16 ? lce_backward<__half>(a, s) : lce_backward<__nv_bfloat16>(a, s);
}
