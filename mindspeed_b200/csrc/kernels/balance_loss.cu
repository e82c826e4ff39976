// Balance loss of a mixture-of-experts router with its per-expert counts, and its gradient.
//
//   p = softmax(x) or sigmoid(x) / (sum_e sigmoid(x_e) + 1e-20)      per token over the E experts
//   P_be = sum of p over the tokens of sequence b,   f_be = entries of the routing map there
//   loss = C sum_be P_be f_be                        (C = coeff E / (S^2 topk B), from the caller)
//   dx_e = g C p_e (f_e - sum p f)                   softmax
//   dx_e = g C s_e (1 - s_e) / n (f_e - sum p f)     sigmoid, n the normaliser
// Token t belongs to sequence t mod B ([s, b] order); the loss over the whole batch is B = 1.
//
// Bound by the memory rate (logits and map read once, gradient written once) or, for short batches, by the launches: one each way, two
// forward for long ones.  A row lives in the registers of 1 to 32 lanes (VEC experts a load, NJ loads), so a warp takes up to 32 rows at once; the
// sums over tokens stay in registers until the block ends and are joined in a fixed order: the same bits on every run.
#include "msb_common.cuh"
#include "msb_sm100.cuh"
#include <algorithm>
using namespace msb;
using namespace msb::sm100;

namespace {

constexpr float LOG2E = 1.4426950408889634f;
constexpr int WARPS = 8;

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

template <int VEC> __device__ __forceinline__ void load_row(const float* p, float* f) {
  if (VEC == 4) { const float4 v = *reinterpret_cast<const float4*>(p); f[0] = v.x; f[1] = v.y; f[2] = v.z; f[3] = v.w; }
  else f[0] = *p;
}
template <int VEC, typename T> __device__ __forceinline__ void load_row(const T* p, float* f) {
  if (VEC == 4) {
    const uint2 v = *reinterpret_cast<const uint2*>(p);
    const T* h = reinterpret_cast<const T*>(&v);
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = to_f(h[i]);
  } else f[0] = to_f(*p);
}
template <int VEC> __device__ __forceinline__ void store_row(float* p, const float* f) {
  if (VEC == 4) *reinterpret_cast<float4*>(p) = make_float4(f[0], f[1], f[2], f[3]);
  else *p = f[0];
}
template <int VEC, typename T> __device__ __forceinline__ void store_row(T* p, const float* f) {
  if (VEC == 4) {
    T h[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = from_f<T>(f[i]);
    *reinterpret_cast<uint2*>(p) = *reinterpret_cast<const uint2*>(h);
  } else *p = from_f<T>(f[0]);
}

__device__ __forceinline__ float lanes_sum(float v, int lanes) {
  for (int o = lanes >> 1; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ float lanes_max(float v, int lanes) {
  for (int o = lanes >> 1; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

// Scores of one row, in place of its logits: p, and for the sigmoid also d p_e / d x_e without the shared term (slope).  Places past
// the row hold -inf and come out as 0.  Returns what the row's scores lack of 1 (the 1e-20 of the sigmoid's normaliser).
template <int N, bool SIGMOID>
__device__ __forceinline__ float scores(float* x, float* slope, int lanes) {
  if (SIGMOID) {
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float t = ex2(-fabsf(x[i]) * LOG2E), r = 1.f / (1.f + t);
      const float big = r, small = t * r;              // sigmoid of |x| and of -|x|: neither is found by subtraction
      const bool pos = x[i] >= 0.f;
      const float sg = x[i] != x[i] ? x[i] : pos ? big : small;
      slope[i] = sg * (pos ? small : big);
      x[i] = sg;
      s += sg;
    }
    const float inv = 1.f / (lanes_sum(s, lanes) + 1e-20f);
#pragma unroll
    for (int i = 0; i < N; ++i) { x[i] *= inv; slope[i] *= inv; }
    return 1e-20f * inv;
  } else {
    float m = -INFINITY;
#pragma unroll
    for (int i = 0; i < N; ++i) m = fmaxf(m, x[i]);
    m = lanes_max(m, lanes);
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) { x[i] = ex2((x[i] - m) * LOG2E); s += x[i]; }
    const float inv = 1.f / lanes_sum(s, lanes);
#pragma unroll
    for (int i = 0; i < N; ++i) { x[i] *= inv; slope[i] = x[i]; }
    return 0.f;
  }
}

// Sums of p and counts of one sequence over the rows of warp `wid` of `warps`; every lane has its experts' of the whole warp.  `lanes` lanes
// a row; expert of (lane l, load j, element v) is (l + lanes j) VEC + v.
template <typename T, int VEC, int NJ, bool SIGMOID>
__device__ __forceinline__ void sum_rows(const T* __restrict__ logits, const unsigned char* __restrict__ map, int S, int B, int E, int lanes,
                                         int seq, int wid, int warps, float* P, int* c) {
  constexpr int N = NJ * VEC;
  const int lane = threadIdx.x & 31, l = lane & (lanes - 1), sub = lane / lanes, rows_per_warp = 32 / lanes;
#pragma unroll
  for (int i = 0; i < N; ++i) { P[i] = 0.f; c[i] = 0; }
  const long long stride = (long long)warps * rows_per_warp;
  // the next rows are loaded while these are summed (not for wide rows: two rows of more than 16 experts a lane do not fit the registers)
  constexpr int AHEAD = N <= 16 ? 2 : 1;
  float x[AHEAD][N];
  uint32_t m[AHEAD][NJ];
  auto fetch = [&](long long r0, float* xr, uint32_t* mr) {
    const long long at = ((r0 + sub) * B + seq) * E;
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
      const int e = (l + lanes * j) * VEC;
      mr[j] = 0;
#pragma unroll
      for (int v = 0; v < VEC; ++v) xr[j * VEC + v] = -INFINITY;
      if (r0 + sub < S && e < E) {
        load_row<VEC>(logits + at + e, xr + j * VEC);
        mr[j] = VEC == 4 ? *reinterpret_cast<const uint32_t*>(map + at + e) : (uint32_t)map[at + e];
      }
    }
  };
  long long r0 = (long long)wid * rows_per_warp;
  if (AHEAD == 2 && r0 < S) fetch(r0, x[0], m[0]);
  for (; r0 < S; r0 += stride) {
    if (AHEAD == 2) fetch(r0 + stride, x[AHEAD - 1], m[AHEAD - 1]);
    else fetch(r0, x[0], m[0]);
    float slope[N];
    scores<N, SIGMOID>(x[0], slope, lanes);
    if (r0 + sub < S) {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        if (!((l + lanes * (i / VEC)) * VEC >= E)) P[i] += x[0][i];
        c[i] += (m[0][i / VEC] >> (8 * (i % VEC))) & 0xffu ? 1 : 0;
      }
    }
    if (AHEAD == 2) {
#pragma unroll
      for (int i = 0; i < N; ++i) x[0][i] = x[AHEAD - 1][i];
#pragma unroll
      for (int j = 0; j < NJ; ++j) m[0][j] = m[AHEAD - 1][j];
    }
  }
  for (int o = lanes; o < 32; o <<= 1)
#pragma unroll
    for (int i = 0; i < N; ++i) {
      P[i] += __shfl_xor_sync(0xffffffffu, P[i], o);
      c[i] += __shfl_xor_sync(0xffffffffu, c[i], o);
    }
}

// Joins the warps of a block in a fixed order: `take(e, P, c)` for each expert.  sh: [warps][E] floats.
template <int VEC, int NJ, typename Take>
__device__ __forceinline__ void join_warps(float* sh, const float* P, const int* c, int warps, int E, int lanes, Take take) {
  constexpr int N = NJ * VEC;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, l = lane & (lanes - 1), sub = lane / lanes;
#pragma unroll
  for (int pass = 0; pass < 2; ++pass) {
    __syncthreads();                              // what was in `sh` has been read
    if (sub == 0)
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int e = (l + lanes * (i / VEC)) * VEC + i % VEC;
        if (e < E) sh[warp * E + e] = pass ? __int_as_float(c[i]) : P[i];
      }
    __syncthreads();
    for (int e = threadIdx.x; e < E; e += blockDim.x) {
      float p = 0.f;
      int n = 0;
      for (int w = 0; w < warps; ++w) {
        if (pass) n += __float_as_int(sh[w * E + e]);
        else p += sh[w * E + e];
      }
      take(e, pass, p, n);
    }
  }
}

// grid (blocks, B): partial sums of p and counts of the block's tokens.
template <typename T, int VEC, int NJ, bool SIGMOID>
__global__ void __launch_bounds__(WARPS * 32) balance_sums_kernel(const T* __restrict__ logits, const unsigned char* __restrict__ map, int S,
                                                                 int B, int E, int lanes, float* psum, int* csum, unsigned int* ticket) {
  after_previous();
  extern __shared__ float sh[];                 // [WARPS][E]
  const int seq = blockIdx.y;
  if (blockIdx.x == 0 && seq == 0 && threadIdx.x == 0) *ticket = 0;
  float P[NJ * VEC];
  int c[NJ * VEC];
  sum_rows<T, VEC, NJ, SIGMOID>(logits, map, S, B, E, lanes, seq, blockIdx.x * WARPS + (threadIdx.x >> 5), gridDim.x * WARPS, P, c);
  const long long out = ((long long)seq * gridDim.x + blockIdx.x) * E;
  join_warps<VEC, NJ>(sh, P, c, WARPS, E, lanes, [&](int e, int pass, float p, int n) {
    if (pass) csum[out + e] = n;
    else psum[out + e] = p;
  });
}

// The whole forward of a short batch in one launch: one cluster of eight CTAs, whose sums meet in distributed shared memory.  Such calls are
// bound by the host, for which a launch is 5 us: at the limit, 8192 tokens of 64 experts, both directions take 97 us with this kernel and 103
// with two, although the GPU's own time is longer (19 us, the two 10; 4096 tokens: 11).
constexpr int CLUSTER = 8, SMALL_WARPS = 16, SMALL_EXPERTS = 512, SMALL_CELLS = 1024;   // cells: sequences x experts
constexpr long long SMALL_ELEMENTS = 1 << 19;
__device__ __forceinline__ uint32_t ld_cluster(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}
template <typename T, int VEC, int NJ, bool SIGMOID>
__global__ void __cluster_dims__(CLUSTER, 1, 1) __launch_bounds__(SMALL_WARPS * 32)
    balance_small_kernel(const T* __restrict__ logits, const unsigned char* __restrict__ map, int S, int B, int E, int lanes, float scale,
                         float* load, float* loss, long long* counts) {
  extern __shared__ float sh[];                 // [SMALL_WARPS][E]
  __shared__ float ps[SMALL_CELLS];
  __shared__ int cs[SMALL_CELLS];
  __shared__ float red[32], mine;
  const uint32_t rank = cluster_ctarank();
  for (int seq = 0; seq < B; ++seq) {
    float P[NJ * VEC];
    int c[NJ * VEC];
    sum_rows<T, VEC, NJ, SIGMOID>(logits, map, S, B, E, lanes, seq, (int)rank * SMALL_WARPS + (threadIdx.x >> 5), CLUSTER * SMALL_WARPS, P, c);
    join_warps<VEC, NJ>(sh, P, c, SMALL_WARPS, E, lanes, [&](int e, int pass, float p, int n) {
      if (pass) cs[seq * E + e] = n;
      else ps[seq * E + e] = p;
    });
  }
  __syncwarp();
  cluster_sync_all();
  // each CTA joins a share of the experts
  const int each = (E + CLUSTER - 1) / CLUSTER, mine_e = (int)rank * each + (int)threadIdx.x;
  const bool owner = (int)threadIdx.x < each && mine_e < E;
  float products = 0.f;
  long long tokens = 0;
  if (owner)
    for (int seq = 0; seq < B; ++seq) {
      const int cell = seq * E + mine_e;
      float p = 0.f;
      int n = 0;
#pragma unroll
      for (uint32_t r = 0; r < CLUSTER; ++r) {
        p += __uint_as_float(ld_cluster(mapa_u32(smem_u32(ps + cell), r)));
        n += (int)ld_cluster(mapa_u32(smem_u32(cs + cell), r));
      }
      load[cell] = (float)n;
      products += p * (float)n;
      tokens += n;
    }
  if (owner) counts[mine_e] = tokens;
  products = block_sum(products, red);
  if (threadIdx.x == 0) mine = products;
  __syncwarp();
  cluster_sync_all();
  if (rank == 0 && threadIdx.x == 0) {
    float s = 0.f;
    for (uint32_t r = 0; r < CLUSTER; ++r) s += __uint_as_float(ld_cluster(mapa_u32(smem_u32(&mine), r)));
    *loss = s * scale;
  }
  __syncwarp();
  cluster_sync_all();                           // no CTA leaves while its shared memory is read
}

// grid (ceil(E / 32), B), 32 experts x 32 slices of the blocks: loads f, the products' sum; the last block to end adds those in order and
// the counts over the sequences.
__global__ void __launch_bounds__(1024) balance_join_kernel(const float* psum, const int* csum, int blocks, int B, int E,
                                                            float scale, float* __restrict__ load, float* __restrict__ lpart,
                                                            unsigned int* ticket, float* __restrict__ loss, long long* __restrict__ counts) {
  after_previous();
  __shared__ float ps[32][33];
  __shared__ int cs[32][33];
  __shared__ bool last;
  const int x = threadIdx.x & 31, y = threadIdx.x >> 5, seq = blockIdx.y, e = blockIdx.x * 32 + x;
  float P = 0.f;
  int c = 0;
  if (e < E)
#pragma unroll 4
    for (int b = y; b < blocks; b += 32) {
      const long long at = ((long long)seq * blocks + b) * E + e;
      P += psum[at];
      c += csum[at];
    }
  ps[y][x] = P;
  cs[y][x] = c;
  __syncthreads();
  if (y == 0) {
    P = 0.f; c = 0;
#pragma unroll
    for (int i = 0; i < 32; ++i) { P += ps[i][x]; c += cs[i][x]; }
    if (e < E) load[(long long)seq * E + e] = (float)c;
    const float s = warp_sum(e < E ? P * (float)c : 0.f);
    if (x == 0) lpart[seq * gridDim.x + blockIdx.x] = s;
    __threadfence();
    __syncwarp();
    if (x == 0) last = atomicAdd(ticket, 1u) == gridDim.x * gridDim.y - 1;
  }
  __syncthreads();
  if (!last) return;
  __threadfence();
  for (int i = threadIdx.x; i < E; i += 1024) {
    long long t = 0;
    for (int b = 0; b < B; ++b) t += (long long)__ldcg(load + (long long)b * E + i);
    counts[i] = t;
  }
  if (y == 0) {
    float s = 0.f;
    for (int i = x; i < (int)(gridDim.x * gridDim.y); i += 32) s += __ldcg(lpart + i);
    s = warp_sum(s);
    if (x == 0) *loss = s * scale;
  }
}

// grid (blocks, B).  f_e - sum p f is taken as (f_e - f_0) - sum p (f - f_0) + f_0 (1 - sum p): loads that are nearly or exactly balanced
// then cancel before any rounding.
template <typename T, int VEC, int NJ, bool SIGMOID>
__global__ void __launch_bounds__(WARPS * 32) balance_grad_kernel(const T* __restrict__ logits, const float* __restrict__ load, int S, int B,
                                                                 int E, int lanes, float scale, const float* __restrict__ g,
                                                                 T* __restrict__ grad) {
  constexpr int N = NJ * VEC;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, l = lane & (lanes - 1), sub = lane / lanes, rows_per_warp = 32 / lanes;
  const int seq = blockIdx.y;
  const float gs = scale * *g;
  const float f0 = load[(long long)seq * E];
  float f[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int e = (l + lanes * (i / VEC)) * VEC + i % VEC;
    f[i] = e < E ? load[(long long)seq * E + e] - f0 : 0.f;
  }
  const long long stride = (long long)gridDim.x * WARPS * rows_per_warp;
  constexpr int AHEAD = N <= 16 ? 2 : 1;        // as above
  float x[AHEAD][N];
  auto fetch = [&](long long r0, float* xr) {
    const long long at = ((r0 + sub) * B + seq) * E;
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
      const int e = (l + lanes * j) * VEC;
#pragma unroll
      for (int v = 0; v < VEC; ++v) xr[j * VEC + v] = -INFINITY;
      if (r0 + sub < S && e < E) load_row<VEC>(logits + at + e, xr + j * VEC);
    }
  };
  long long r0 = ((long long)blockIdx.x * WARPS + warp) * rows_per_warp;
  if (AHEAD == 2 && r0 < S) fetch(r0, x[0]);
  for (; r0 < S; r0 += stride) {
    if (AHEAD == 2) fetch(r0 + stride, x[AHEAD - 1]);
    else fetch(r0, x[0]);
    float slope[N];
    const float lack = scores<N, SIGMOID>(x[0], slope, lanes);
    float d = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) d = fmaf(x[0][i], f[i], d);
    d = lanes_sum(d, lanes) - f0 * lack;
#pragma unroll
    for (int i = 0; i < N; ++i) slope[i] *= (f[i] - d) * gs;
    if (r0 + sub < S) {
      const long long at = ((r0 + sub) * B + seq) * E;
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        const int e = (l + lanes * j) * VEC;
        if (e < E) store_row<VEC>(grad + at + e, slope + j * VEC);
      }
    }
    if (AHEAD == 2)
#pragma unroll
      for (int i = 0; i < N; ++i) x[0][i] = x[AHEAD - 1][i];
  }
}

struct Shape { int vec, nj, lanes; };

// VEC = 4 where every row of logits, gradient and map starts on a boundary of four elements (E a multiple of 4, bases aligned).
Shape shape_of(int E, bool aligned) {
  Shape s;
  s.vec = aligned && E % 4 == 0 ? 4 : 1;
  const int units = E / s.vec;
  s.lanes = 32;
  while (s.lanes > 1 && s.lanes / 2 >= units) s.lanes /= 2;
  s.nj = (units + s.lanes - 1) / s.lanes;
  return s;
}

#define BAL_NJ(T, SIG, CALL)                                                                         \
  if (sh.vec == 4) {                                                                                 \
    if (sh.nj <= 1) { CALL(T, 4, 1, SIG); } else if (sh.nj <= 2) { CALL(T, 4, 2, SIG); }             \
    else if (sh.nj <= 4) { CALL(T, 4, 4, SIG); } else { CALL(T, 4, 8, SIG); }                        \
  } else {                                                                                           \
    if (sh.nj <= 1) { CALL(T, 1, 1, SIG); } else if (sh.nj <= 4) { CALL(T, 1, 4, SIG); }             \
    else if (sh.nj <= 16) { CALL(T, 1, 16, SIG); } else { CALL(T, 1, 32, SIG); }                     \
  }
#define BAL_DISPATCH(CALL)                                                                           \
  MSB_DISPATCH_FLOAT(dtype, T, if (sigmoid) { BAL_NJ(T, true, CALL) } else { BAL_NJ(T, false, CALL) })

int bal_check(int S, int B, int E) {
  MSB_REQUIRE(S > 0 && B > 0 && E > 0 && E <= 1024, "balance_loss: %d x %d tokens, %d experts (at most 1024)", S, B, E);
  MSB_REQUIRE(B <= 65535 && (long long)S * B <= (1 << 24), "balance_loss: %d sequences of %d tokens (at most 2^24 tokens, counted in fp32)", B, S);
  return 0;
}

// blocks a sequence
int balance_grid(int S, int B, int E) {
  const int units = E % 4 == 0 ? E / 4 : E;
  int lanes = 32;
  while (lanes > 1 && lanes / 2 >= units) lanes /= 2;
  const long long rows_per_block = WARPS * (32 / lanes);
  const long long want = (S + rows_per_block - 1) / rows_per_block;
  const long long cap = std::max<long long>(1, (long long)msb::num_sms() * 4 / B);
  return (int)std::min(want, cap);
}

}  // namespace

// Blocks a sequence that the forward launches, by which its scratch is sized ([B, blocks, E] floats and ints).
// 0: a short batch, whose forward is one launch and needs none.
MSB_API int msb_balance_blocks(int S, int B, int E) {
  if ((long long)S * B * E <= SMALL_ELEMENTS && E <= SMALL_EXPERTS && (long long)B * E <= SMALL_CELLS) return 0;
  return balance_grid(S, B, E);
}
MSB_API int msb_balance_forward(const void* logits, const unsigned char* map, int S, int B, int E, int sigmoid, float scale, int dtype,
                                float* psum, int* csum, int blocks, float* load, float* lpart, unsigned int* ticket, float* loss,
                                long long* counts, cudaStream_t s) {
  if (int rc = bal_check(S, B, E)) return rc;
  const Shape sh = shape_of(E, ((uintptr_t)logits & 15) == 0 && ((uintptr_t)map & 3) == 0);
  const dim3 grid(blocks, B);
  if (blocks == 0) {
#define BAL_CALL(T, V, NJ, SIG)                                                                                                         \
  if constexpr ((V) * (NJ) <= 16)                                                                                                       \
    balance_small_kernel<T, V, NJ, SIG><<<CLUSTER, SMALL_WARPS * 32, SMALL_WARPS * E * 4, s>>>((const T*)logits, map, S, B, E, sh.lanes, \
                                                                                              scale, load, loss, counts)
    BAL_DISPATCH(BAL_CALL)
#undef BAL_CALL
    MSB_CHECK_LAUNCH("balance_small");
    return 0;
  }
#define BAL_CALL(T, V, NJ, SIG)                                                                                                        \
  balance_sums_kernel<T, V, NJ, SIG><<<grid, WARPS * 32, WARPS * E * 4, s>>>((const T*)logits, map, S, B, E, sh.lanes, psum, csum, ticket)
  BAL_DISPATCH(BAL_CALL)
#undef BAL_CALL
  MSB_CHECK_LAUNCH("balance_sums");
  msb::launch_after(balance_join_kernel, dim3((E + 31) / 32, B), 1024, 0, s, psum, csum, blocks, B, E, scale, load, lpart, ticket, loss, counts);
  MSB_CHECK_LAUNCH("balance_join");
  return 0;
}

MSB_API int msb_balance_backward(const void* logits, const float* load, int S, int B, int E, int sigmoid, float scale, const float* g, int dtype,
                                 void* grad, cudaStream_t s) {
  if (int rc = bal_check(S, B, E)) return rc;
  const Shape sh = shape_of(E, (((uintptr_t)logits | (uintptr_t)grad) & 15) == 0);
  const dim3 grid(balance_grid(S, B, E), B);
#define BAL_CALL(T, V, NJ, SIG) \
  balance_grad_kernel<T, V, NJ, SIG><<<grid, WARPS * 32, 0, s>>>((const T*)logits, load, S, B, E, sh.lanes, scale, g, (T*)grad)
  BAL_DISPATCH(BAL_CALL)
#undef BAL_CALL
  MSB_CHECK_LAUNCH("balance_grad");
  return 0;
}
