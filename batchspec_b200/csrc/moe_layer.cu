// A whole routed feed-forward for a few tokens (at most 64) in two kernels:
//   z = Wr h,  (ids, w) = choice(z)                      the rules of moe_choose.cuh
//   u[t, k] = act(Wup[ids[t, k]] h[t])                   act: GELU, or silu(gate) * up with Wup = [gate; up]
//   out[t]  = add[t] * sigmoid(gate logit) + sum over k of w[t, k] * (Wdown[ids[t, k]] u[t, k], or h[t] for an identity expert)
// Experts in bfloat16, or in 8-bit floating point (e4m3) with a scale per 128 x 128 block; sums are float32.
//
// Bound by the read of the chosen experts' weights, each of which is used once per step.  So the weights take the 128 rows of
// tcgen05 products, streamed at full tile efficiency by TMA into a ring of 16 KB stages, and the tokens their 16 to 64 columns:
// a stage costs two copies of weights and a few instructions, and what the sums cost does not grow with the weights.
//   up     all tokens of the step are columns of every expert (no gather: the columns that did not choose it are dropped)
//   down   an expert's tokens are its columns: u lies sorted by expert, 16 rows to a copy
// Activations take two columns of the same product.  bfloat16 weights: every number of u is the sum of two bfloat16 numbers, 16 bits.
// 8-bit weights: every activation is the sum of two e4m3 numbers, x = s (a + b / 16): a is x / s rounded to 4 bits, b what is left, times 16; s
// is a power of two, one for a token's h and one for 64 numbers of u.  That is 8 bits, as many as bfloat16 has, for numbers of h down to 2^-14.8 of
// the token's largest; below that they lose bits one by one (steps of 2^-22 of the largest).  The result's error goes from 1.66e-3 to 1.8e-3 by it.
// A block of 128 k (of 64 in the down products, for the scales of u) gets an accumulator of its own, which the epilogue warps read back and add to
// float32 sums.
//
//   route    one cluster of 8 CTAs per 8 tokens: 64 warps share the router's rows and k, partial sums meet in the first CTA's
//            shared memory, whose warps choose for a token each.  It also clears the counters of the second kernel.
//   experts  one CTA per SM: a TMA warp that draws pieces of work, an MMA warp, two groups of epilogue warps that take the pieces in
//            turn.  First the pieces of the up products (128 rows of one expert) are drawn from one counter, then those of the down
//            products (128 output columns of one expert, perhaps a slice of its k).  A piece of the second kind waits until every piece of the first kind is done; those
//            have all been drawn by CTAs that run and wait for nothing, so it ends however many CTAs the device can hold.
//            When the last down piece is done, all CTAs add the experts' results in the order of the choices: no atomic adds numbers.
//
// With few tokens what bounds a step are the phases that wait for each other: router 7 to 8 us, start and lists 3, first weights 4, then the
// weights, then u through the L2 4, the last pieces and the sum over choices 3.  A good part of each is the fetch of its code, which the
// weights have pushed out of the L2 since the last step: loops are kept as loops, and the polls of a wait are a call (1 token 38.4 -> 35.9 us,
// 8 tokens of 8-bit experts 59.7 -> 53.0; running the epilogue over made-up pieces while the router runs made it slower, 24 us of code),
// and pieces are numbered without divisions by numbers of the step (61 tokens 133.8 -> 130.5).
// Measured on B200, 64 experts of 2,048 x 1,408, 6 per token: 1 token, gated, 36 us; 8 tokens of which 12 experts are taken, gated, 8-bit, 55; 61 tokens,
// GELU, 129.5 (5.7 TB/s); 23 tokens, 20 experts of 1,040 x 720, 8-bit with float32 scales, 36.  Gated, evenly chosen, bfloat16 / 8-bit: 8 tokens (34
// experts) 110 / 90, 32 tokens 173 / 142, 61 tokens 184 / 201: there the epilogue's steps for 8-bit experts, an accumulator per 64 or 128 k, take longer
// than the weights.
#include "moe_choose.cuh"
#include "e4m3.cuh"
#include "umma.cuh"
#include <math.h>

using namespace bspec;

namespace {

constexpr int LAYER_TOKENS = 64;             // most tokens of a step
constexpr int ROUTE_CLUSTER = 8, ROUTE_WARPS = 8, ROUTE_TOKENS = 8;
constexpr int LAYER_THREADS = 320;           // TMA warp, MMA warp, two groups of 4 epilogue warps
constexpr int SMEM_BUDGET = 225 * 1024;

// ------------------------------------------------------------------------------------------------ the router
// z partials: [unit = (16 rows of the router, slice of k)][8 tokens][16 rows] in the first CTA of the cluster.
__global__ void __cluster_dims__(ROUTE_CLUSTER, 1, 1) __launch_bounds__(32 * ROUTE_WARPS)
moe_layer_route_kernel(const __nv_bfloat16* __restrict__ h, int n, int d, const __nv_bfloat16* __restrict__ wr, int rows, int slices,
                       const void* __restrict__ corr, int corr_dtype, int C, int G, int keep, int top, float scale, int rule,
                       int* __restrict__ ids, float* __restrict__ wts, float* __restrict__ gate, int* __restrict__ counters,
                       uint8_t* __restrict__ hq, float* __restrict__ hs) {
  const int tiles = (rows + 15) / 16, units = tiles * slices;
  const int rank = blockIdx.x % ROUTE_CLUSTER, t0 = blockIdx.x / ROUTE_CLUSTER * ROUTE_TOKENS;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, q = lane & 3;
  const int steps = (d + 31) / 32, per = (steps + slices - 1) / slices;
  bspec::pdl_prologue(84);
  const int chooses = ROUTE_CLUSTER * ((n + ROUTE_TOKENS - 1) / ROUTE_TOKENS);      // CTAs
  if ((int)blockIdx.x >= chooses) {
    // 8-bit experts: the clusters behind those that choose bring a token per CTA into two 8-bit numbers for each of its own, with one scale
    const int row = blockIdx.x - chooses;
    if (row >= n) return;
    __shared__ uint32_t warp_max[ROUTE_WARPS];
    uint32_t m = 0u;
#pragma unroll 1
    for (int k = 8 * threadIdx.x; k < d; k += 8 * 32 * ROUTE_WARPS) {
      const uint4 raw = *reinterpret_cast<const uint4*>(h + (size_t)row * d + k);
      const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) m = max(m, max((w[i] << 16) & 0x7fffffffu, w[i] & 0x7fff0000u));
    }
    m = __reduce_max_sync(0xffffffffu, m);
    if (lane == 0) warp_max[warp] = m;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < ROUTE_WARPS; ++i) m = max(m, warp_max[i]);
    const int code = scale_code(m);
    const float inv = inverse_scale(code);
#pragma unroll 1
    for (int k = 8 * threadIdx.x; k < d; k += 8 * 32 * ROUTE_WARPS) {
      const uint4 raw = *reinterpret_cast<const uint4*>(h + (size_t)row * d + k);
      const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
      uint32_t hi[2], lo[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float v[4] = {__uint_as_float(w[2 * i] << 16), __uint_as_float(w[2 * i] & 0xffff0000u),
                            __uint_as_float(w[2 * i + 1] << 16), __uint_as_float(w[2 * i + 1] & 0xffff0000u)};
        two_e4m3x4(v, inv, hi[i], lo[i]);
      }
      *reinterpret_cast<uint2*>(hq + (size_t)row * d + k) = make_uint2(hi[0], hi[1]);
      *reinterpret_cast<uint2*>(hq + (size_t)(n + row) * d + k) = make_uint2(lo[0], lo[1]);
    }
    if (threadIdx.x == 0) hs[row] = scale_value(code);
    return;
  }
  extern __shared__ float sm[];
  float* part = sm;                                            // [units][8][16]
  if (blockIdx.x == 0 && threadIdx.x < 4) counters[threadIdx.x] = 0;
  // every CTA of the cluster runs before another one writes to its memory
  asm volatile("barrier.cluster.arrive.relaxed.aligned;\n\tbarrier.cluster.wait.aligned;" ::: "memory");
  uint32_t first;                                              // the first CTA's partials
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(first) : "r"(s32(part)), "r"(0));
  const uint4 zero = make_uint4(0u, 0u, 0u, 0u);
  const bool token = t0 + g < n;
#pragma unroll 1
  for (int unit = rank * ROUTE_WARPS + warp; unit < units; unit += ROUTE_CLUSTER * ROUTE_WARPS) {
    const int r0 = unit / slices * 16, s0 = unit % slices * per, s1 = min(steps, s0 + per);
    const __nv_bfloat16* lo = wr + (size_t)min(r0 + g, rows - 1) * d + 8 * q;
    const __nv_bfloat16* hi = wr + (size_t)min(r0 + g + 8, rows - 1) * d + 8 * q;
    const __nv_bfloat16* x = h + (size_t)min(t0 + g, n - 1) * d + 8 * q;
    float acc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
    for (int s = s0; s < s1; s += 4) {
      uint4 a[4], b[4], c[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int k = 32 * (s + j);
        const bool live = s + j < s1 && k + 8 * q < d;
        a[j] = live ? __ldg(reinterpret_cast<const uint4*>(lo + k)) : zero;
        b[j] = live ? __ldg(reinterpret_cast<const uint4*>(hi + k)) : zero;
        c[j] = live && token ? *reinterpret_cast<const uint4*>(x + k) : zero;
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        mma_bf16_16816(acc, a[j].x, b[j].x, a[j].y, b[j].y, c[j].x, c[j].y);
        mma_bf16_16816(acc, a[j].z, b[j].z, a[j].w, b[j].w, c[j].z, c[j].w);
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int at = (unit * ROUTE_TOKENS + 2 * q + (i & 1)) * 16 + g + 8 * (i >> 1);
      asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(first + 4u * (uint32_t)at), "f"(acc[i]) : "memory");
    }
  }
  float* bias = part + (size_t)units * 16 * ROUTE_TOKENS;      // [C]
  if (rank == 0)
#pragma unroll 1
    for (int e = threadIdx.x; e < C; e += 32 * ROUTE_WARPS) bias[e] = corr != nullptr ? load_as_f32(corr, corr_dtype, e) : 0.f;
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  __syncwarp();
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  const int t = t0 + warp;
  if (rank != 0 || t >= n) return;
  float* sc = bias + C + (size_t)warp * 3 * C;
  float* ch = sc + C;
#pragma unroll 1
  for (int e = lane; e < rows; e += 32) {
    const float* from = part + ((size_t)(e / 16 * slices) * ROUTE_TOKENS + warp) * 16 + e % 16;
    float z = 0.f;
#pragma unroll 4
    for (int s = 0; s < slices; ++s) z += from[s * ROUTE_TOKENS * 16];
    if (e < C) route_score(rule, z, bias[e], sc + e, ch + e);
    else gate[t] = z;                                          // the row behind the experts' rows
  }
  __syncwarp();
  choose_experts<true>(sc, ch, ch + C, corr != nullptr ? bias : nullptr, BSPEC_F32, C, G, keep, top, scale, rule, ids + (size_t)t * top, wts + (size_t)t * top);
}

// ------------------------------------------------------------------------------------------------ the experts
constexpr int TILE = 128;                    // weight rows of a piece
constexpr int A_BYTES = TILE * 128;          // of a stage: 128 bytes of every row
constexpr int QUEUE = 4;                     // pieces on their way through the roles
constexpr int MAX_STAGES = 10;
constexpr int WINDOW = 64;                   // blocks of u whose scales wait in shared memory at a time
constexpr int MAX_SPLITS = 4;                // slices of k of the down products: 1, 2 or 4

// Division by a number that the host knows: the product with its reciprocal is at most one too small.
struct Divide {
  uint32_t by, inverse;
  __host__ __device__ static Divide of(int n) { return {(uint32_t)n, 0xffffffffu / (uint32_t)n}; }
  __device__ __forceinline__ int operator()(int n, int& rest) const {
    uint32_t q = __umulhi((uint32_t)n, inverse), left = (uint32_t)n - q * by;
    if (left >= by) { ++q; left -= by; }
    rest = (int)left;
    return (int)q;
  }
};

struct LayerParams {
  const float* su;                           // scales of 128 x 128 blocks: float32, or 8-bit exponents (e8m0)
  const float* sd;
  int e8m0;
  const int* ids;                            // [n, top]; E and above: the token's own h
  const float* wts;
  const float* gate;                         // [n] or null
  const __nv_bfloat16* h;                    // [n, d]
  const __nv_bfloat16* add;                  // [n, d] or null
  const float* hs;                           // [n] scales of the tokens' 8-bit numbers
  unsigned char* u;                          // entries sorted by expert, two numbers for each: [2][n top, ff] bfloat16 or e4m3
  float* us;                                 // [n top, blocks of 64] their scales
  float* y;                                  // [splits][n top, d] the experts' results
  __nv_bfloat16* out;                        // [n, d]
  int* counters;                             // zero: {up pieces drawn, up pieces done, down pieces drawn, down pieces done}
  int* status;
  int n, d, ff, E, top;
  int stages;
  Divide up_tiles, down_tiles, quads;         // tiles of an expert's products, groups of four numbers of a token
};

struct Piece {
  int down;                                  // 0: up, 1: down, -1: no more
  int a, tile, s0, s1, split;                // place in the list of chosen experts, 128 rows, stages of k
};

__device__ __forceinline__ void fence_async_all() { asm volatile("fence.proxy.async;" ::: "memory"); }
__device__ __forceinline__ float block_scale(const float* p, int e8m0, size_t i) {
  return e8m0 ? scale_value(reinterpret_cast<const uint8_t*>(p)[i]) : p[i];
}

// Waits until *counter reaches `target` (a bounded wait, as every other one).
__device__ __forceinline__ bool wait_for(const int* counter, int target, int* status, volatile int* abort_flag) {
  unsigned long long t_from = 0ull;
#pragma unroll 1
  for (uint32_t i = 0;; ++i) {
    int v;
    asm volatile("ld.acquire.gpu.global.s32 %0, [%1];" : "=r"(v) : "l"(counter) : "memory");
    if (v >= target) return true;
    if (*abort_flag) return false;
    if ((i & 255u) == 255u) {
      const unsigned long long now = bspec::global_timer();
      if (t_from == 0ull) t_from = now;
      if (now - t_from > WAIT_NS || i >= WAIT_LIMIT || *reinterpret_cast<volatile int*>(status) != 0) {
        atomicCAS(status, 0, 111);
        *abort_flag = 1;
        return false;
      }
    }
  }
}
__device__ __forceinline__ float4 four_bf16(const __nv_bfloat16* from) {
  const uint2 raw = *reinterpret_cast<const uint2*>(from);
  return make_float4(__uint_as_float(raw.x << 16), __uint_as_float(raw.x & 0xffff0000u), __uint_as_float(raw.y << 16),
                     __uint_as_float(raw.y & 0xffff0000u));
}
__device__ __forceinline__ float4 scaled(const float4& v, float f) { return make_float4(f * v.x, f * v.y, f * v.z, f * v.w); }

// Shared memory behind the stages.  NB: columns, 16, 32 or 64.
template <bool FP8, int NB>
struct Layout {
  // room for two numbers per column; 64 columns of bfloat16: for one, as few experts have more than 32 tokens and
  // stages are worth more (61 tokens: 4 stages 138 us, 6 stages 128.5)
  static constexpr int B_BYTES = (!FP8 && NB == 64 ? 1 : 2) * NB * 128, STAGE = A_BYTES + B_BYTES;
  // where an expert's tokens do not fit in twice, its stages come twice (the second time out of the L2)
  __device__ static int twice(int boxes) { return boxes * 4096 > B_BYTES ? 1 : 0; }
  // rows of scales: blocks of 64 in whole stages, a window of them at most
  __host__ __device__ static int rows(int ff) { return (ff + 127) / 128 * 2 < WINDOW ? (ff + 127) / 128 * 2 : WINDOW; }
  // of each epilogue group: tile [NB][128], scales of a piece's u [rows][NB]; then the lists
  __host__ __device__ static size_t fixed(int ff, int slots, int E) {
    return (size_t)2 * NB * TILE * 4 + (FP8 ? (size_t)2 * rows(ff) * NB * 4 : 0) + ((size_t)2 * slots + 3 * (size_t)E + 1) * 4 + 1024;
  }
  // stages that fit beside them, three at least or none
  static int stages(int ff, int slots, int E) {
    const size_t taken = 1024 + fixed(ff, slots, E);
    if (taken + 3 * (size_t)STAGE > SMEM_BUDGET) return 0;
    const size_t room = (SMEM_BUDGET - taken) / STAGE;
    return room > MAX_STAGES ? MAX_STAGES : (int)room;
  }
};

template <bool FP8, bool GLU, int NB>
__global__ void __launch_bounds__(LAYER_THREADS, 1)
moe_layer_experts_kernel(const __grid_constant__ CUtensorMap map_up, const __grid_constant__ CUtensorMap map_down,
                         const __grid_constant__ CUtensorMap map_h, const __grid_constant__ CUtensorMap map_u, LayerParams p) {
  using Lay = Layout<FP8, NB>;
  constexpr int STAGE_K = FP8 ? 128 : 64;                      // k of a stage
  constexpr int WIDTH = 2 * NB;                                // columns of an accumulator
  constexpr int SLOTS = NB == 64 ? 2 : 4;                      // accumulators of each epilogue group
  constexpr uint32_t TMEM_COLS = 2 * SLOTS * WIDTH;            // 256 or 512
  constexpr int OUT = GLU ? 64 : 128;                          // numbers of u per up piece
  extern __shared__ unsigned char smem_dyn[];
  unsigned char* smem = reinterpret_cast<unsigned char*>(((uintptr_t)smem_dyn + 1023) & ~(uintptr_t)1023);
  __shared__ uint64_t full[MAX_STAGES], empty[MAX_STAGES], acc_full[2 * SLOTS], acc_empty[2 * SLOTS], q_full[QUEUE], q_empty[QUEUE], meet[2], up_done;
  __shared__ Piece queue[QUEUE];
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_word, n_active;
  volatile int* abort_flag = &abort_word;
  const int slots = p.n * p.top, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  float* tile = reinterpret_cast<float*>(smem + (size_t)p.stages * Lay::STAGE);          // [2][NB][128]
  float* ys = tile + 2 * NB * TILE;
  int* pos = reinterpret_cast<int*>(ys + (FP8 ? 2 * Lay::rows(p.ff) * NB : 0));            // [slots] where a (token, choice) lies by expert, or -1
  int* tok = pos + slots;                                                                // [slots] tokens by expert
  int* active = tok + slots;                                                             // [E] chosen experts
  int* first = active + p.E;                                                             // [E + 1] where their entries begin
  int* count = first + p.E + 1;                                                          // [E]

  if (threadIdx.x >= 64 && threadIdx.x < 68) {
    const CUtensorMap* map = threadIdx.x == 64 ? &map_up : (threadIdx.x == 65 ? &map_down : (threadIdx.x == 66 ? &map_h : &map_u));
    asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory");
  }
  if (threadIdx.x == 0) {
#pragma unroll 1
    for (int i = 0; i < MAX_STAGES; ++i) {
      mbar_init(full + i, 1);
      mbar_init(empty + i, 1);
    }
    for (int i = 0; i < 2 * SLOTS; ++i) {
      mbar_init(acc_full + i, 1);
      mbar_init(acc_empty + i, 4);
    }
    for (int i = 0; i < QUEUE; ++i) {
      mbar_init(q_full + i, 1);
      mbar_init(q_empty + i, 9);
    }
    mbar_init(meet, 4);
    mbar_init(meet + 1, 4);
    mbar_init(&up_done, 1);
    abort_word = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(s32(&tmem_slot)), "r"(TMEM_COLS) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
#pragma unroll 1
  for (int e = threadIdx.x; e < p.E; e += LAYER_THREADS) count[e] = 0;
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = tmem_slot;
  // Where a step chooses so often that nearly every expert is taken (of evenly chosen ones 1 in 20 is not), and weights enough follow, the first pieces'
  // weights are asked into the L2 while the router runs.  Measured: 61 tokens of 64 experts, 4.8 rounds of pieces, 137.2 -> 133.8 us; with 1.6
  // rounds, 23 tokens of 20 small experts, 35.1 -> 36.1.
  if (warp == 0 && slots >= 3 * p.E && p.E * (int)p.up_tiles.by >= 3 * (int)gridDim.x) {
    const uint32_t one = elect_one();
    int i0;
    const int e = p.up_tiles((int)blockIdx.x, i0);
    if (e < p.E && one) {
      const int y0 = e * (GLU ? 2 * p.ff : p.ff) + i0 * OUT, y1 = y0 + (GLU ? p.ff : 64), stages = (p.d + STAGE_K - 1) / STAGE_K;
#pragma unroll 1
      for (int s = 0; s < stages; ++s) {
        tma_prefetch_2d(&map_up, s * STAGE_K, y0);
        tma_prefetch_2d(&map_up, s * STAGE_K, y1);
      }
    }
  }
  bspec::pdl_prologue(85);

  // this CTA's first up piece, drawn while the lists are made
  int first_piece = 0;
  if (threadIdx.x == 0) first_piece = atomicAdd(p.counters, 1);
  // ---- the entries by expert, in an order that every CTA finds alike
  if (slots > 32) {
#pragma unroll 1
    for (int s = threadIdx.x; s < slots; s += LAYER_THREADS) {
      const int e = p.ids[s];
      if (e < p.E) atomicAdd(count + e, 1);
    }
    __syncthreads();
  }
  if (slots <= 32 && warp == 0) {
    // one entry per lane: experts in the order of their first entries
    const int e = lane < slots ? p.ids[lane] : p.E;
    const unsigned same = __match_any_sync(0xffffffffu, e), before = (1u << lane) - 1u;
    const int leader = __ffs(same) - 1;
    const bool leads = lane == leader && e < p.E;
    int upto = leads ? __popc(same) : 0;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += v;
    }
    const int start = __shfl_sync(0xffffffffu, upto, leader) - __popc(same);
    const unsigned leaders = __ballot_sync(0xffffffffu, leads);
    if (leads) {
      active[__popc(leaders & before)] = e;
      first[__popc(leaders & before)] = start;
    }
    if (e < p.E) {
      pos[lane] = start + __popc(same & before);
      tok[start + __popc(same & before)] = lane / p.top;
    } else if (lane < slots) {
      pos[lane] = -1;
    }
    if (lane == 31) {
      first[__popc(leaders)] = upto;
      n_active = __popc(leaders);
    }
  } else if (warp == 0) {
    // counted; they take their places below
    int found = 0, run = 0;
#pragma unroll 1
    for (int e0 = 0; e0 < p.E; e0 += 32) {
      const int e = e0 + lane, c = e < p.E ? count[e] : 0;
      int upto = c;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += v;
      }
      const unsigned mask = __ballot_sync(0xffffffffu, c > 0);
      if (c > 0) {
        const int at = found + __popc(mask & ((1u << lane) - 1u));
        active[at] = e;
        first[at] = count[e] = run + upto - c;
      }
      found += __popc(mask);
      run += __shfl_sync(0xffffffffu, upto, 31);
    }
    if (lane == 0) {
      first[found] = run;
      n_active = found;
    }
  }
  __syncthreads();

  const int A = n_active, ffu = GLU ? 2 * p.ff : p.ff;
  const int up_pieces = A * (int)p.up_tiles.by, up_stages = (p.d + STAGE_K - 1) / STAGE_K;
  const int down_tiles = (int)p.down_tiles.by, down_stages = (p.ff + STAGE_K - 1) / STAGE_K;
  // slices of the down products' k, four stages each at least: more of them only where that fills the CTAs' rounds by a seventh better
  int shift = 0;
  {
    const float whole = (float)(A * down_tiles) / (float)gridDim.x;
    float best = ceilf(whole);                                 // rounds of whole pieces
    for (int i = 1; (1 << i) <= MAX_SPLITS && down_stages >= (4 << i); ++i) {
      const float rounds = ceilf(whole * (1 << i)) / (1 << i);
      if (rounds * 7.f <= best * 6.f) { best = rounds; shift = i; }
    }
  }
  const int splits = 1 << shift, down_per = (down_stages + splits - 1) >> shift, down_pieces = (A * down_tiles) << shift;
  const int entries = first[A];

  if (warp == 0) {
    const uint32_t one = elect_one();
    int st = 0, np = 0;                                        // stage of the ring, pieces so far
    uint32_t phase = 0u;
    bool ok = true;
    auto push = [&](const Piece& piece) {
      const int q = np % QUEUE;
      if (ok) ok = warp_wait_short(q_empty + q, ((uint32_t)(np / QUEUE) & 1u) ^ 1u, abort_flag, p.status, 113);
      if (lane == 0 && ok) {
        queue[q] = piece;
        mbar_arrive(q_full + q);
      }
      ++np;
      __syncwarp();
    };
    auto draw = [&](int counter) {
      int t = 0;
      if (lane == 0) t = atomicAdd(p.counters + counter, 1);
      return __shfl_sync(0xffffffffu, t, 0);
    };
    // stage s of a piece: the weights' two halves, and its tokens; the first copies also say how many bytes will come
    auto weights = [&](const CUtensorMap* map, int y0, int y1, int boxes, int s) {
      if (ok) ok = warp_wait_short(empty + st, phase ^ 1u, abort_flag, p.status, 114);
      if (!ok) return;
      unsigned char* at = smem + (size_t)st * Lay::STAGE;
      mbar_expect_tx_by(one, full + st, A_BYTES + (uint32_t)boxes * 2048u);
      tma_load_2d_by(one, at, map, full + st, s * STAGE_K, y0);
      tma_load_2d_by(one, at + A_BYTES / 2, map, full + st, s * STAGE_K, y1);
    };
    auto tokens = [&](const CUtensorMap* map, int y, int mid, int boxes, bool two, int s) {
      if (!ok) return;
      unsigned char* at = smem + (size_t)st * Lay::STAGE + A_BYTES;
#pragma unroll
      for (int b = 0; b < NB / 16; ++b) {
        if (b >= boxes) break;
        tma_load_2d_by(one, at + b * 2048, map, full + st, s * STAGE_K, y + 16 * b);
        if (two) tma_load_2d_by(one, at + (boxes + b) * 2048, map, full + st, s * STAGE_K, mid + y + 16 * b);
      }
    };
    auto step = [&]() {
      if (++st == p.stages) { st = 0; phase ^= 1u; }
    };
    // the up products
    int t = __shfl_sync(0xffffffffu, first_piece, 0);
    while (ok && t < up_pieces) {
      int tile_at;
      const int a = p.up_tiles(t, tile_at), i0 = tile_at * OUT, e = active[a];
      push({0, a, tile_at, 0, up_stages, 0});
      const int y0 = e * ffu + i0, y1 = y0 + (GLU ? p.ff : 64);
#pragma unroll 1
      for (int s = 0; s < up_stages && ok; ++s, step()) {
        weights(&map_up, y0, y1, NB / 16 * (FP8 ? 2 : 1), s);
        tokens(&map_h, 0, p.n, NB / 16, FP8, s);
      }
      t = draw(0);                                             // not earlier: a CTA that starts first would take the others' first pieces
    }
    // the down products
    t = draw(2);
    bool waited = false;
    while (ok && t < down_pieces) {
      int dt;
      const int split = t & (splits - 1), a = p.down_tiles(t >> shift, dt), e = active[a];
      const int s0 = split * down_per, s1 = min(down_stages, s0 + down_per), c0 = first[a];
      push({1, a, dt, s0, s1, split});
      const int y0 = e * p.d + dt * TILE, boxes = (first[a + 1] - c0 + 15) / 16;
      const int twice = Lay::twice(boxes), end = s1 << twice, at_once = twice ? boxes : 2 * boxes;
      auto down_tokens = [&](int s) { tokens(&map_u, c0 + (s & twice) * slots, slots, boxes, !twice, s >> twice); };
      int s = s0 << twice;
      if (!waited) {
        // the first weights are asked for before the wait for the up products
        waited = true;
        const int ahead = min(end - s, p.stages), st_from = st;
        const uint32_t phase_from = phase;
#pragma unroll 1
        for (int i = 0; i < ahead && ok; ++i, step()) weights(&map_down, y0, y0 + 64, at_once, (s + i) >> twice);
        if (lane == 0 && ok) ok = wait_for(p.counters + 1, up_pieces, p.status, abort_flag);
        if (lane == 0 && ok) mbar_arrive(&up_done);            // the epilogue may read the scales of u
        ok = __shfl_sync(0xffffffffu, (int)ok, 0) != 0;
        __syncwarp();
        fence_async_all();                                     // u was written through the generic proxy
        st = st_from;
        phase = phase_from;
#pragma unroll 1
        for (int i = 0; i < ahead; ++i, step()) down_tokens(s + i);
        s += ahead;
      }
#pragma unroll 1
      for (; s < end && ok; ++s, step()) {
        weights(&map_down, y0, y0 + 64, at_once, s >> twice);
        down_tokens(s);
      }
      t = draw(2);
    }
    push({-1, 0, 0, 0, 0, 0});
    if (*abort_flag)                                           // copies in flight land (they take microseconds) before the CTA ends
      for (int i = 0; i < 1000; ++i) __nanosleep(1000);
  } else if (warp == 1) {
    const uint32_t one = elect_one();
    int st = 0, ring[2] = {0, 0};                              // the groups' running accumulators
    uint32_t phase = 0u, ring_phase[2] = {0u, 0u};
    bool ok = true;
    const uint64_t desc0 = smem_desc(smem);
#pragma unroll 1
    for (int np = 0; ok; ++np) {
      const int q = np % QUEUE;
      if (!(ok = warp_wait_short(q_full + q, (uint32_t)(np / QUEUE) & 1u, abort_flag, p.status, 115))) break;
      const Piece piece = queue[q];
      __syncwarp();
      if (lane == 0) mbar_arrive(q_empty + q);
      if (piece.down < 0) break;
      const int boxes = piece.down ? (first[piece.a + 1] - first[piece.a] + 15) / 16 : NB / 16;
      const int twice = piece.down ? Lay::twice(boxes) : 0;
      const int cols = boxes * 16 * ((FP8 || piece.down) && !twice ? 2 : 1);
      const uint32_t idesc = FP8 ? instr_desc_e4m3(cols) : instr_desc(cols);
      const int group = np & 1;
      int slot = group ? SLOTS + ring[1] : ring[0];
      uint32_t slot_phase = group ? ring_phase[1] : ring_phase[0];
      auto next_slot = [&]() {
        ok = ok && warp_wait_short(acc_empty + slot, slot_phase ^ 1u, abort_flag, p.status, 116);
        tc_fence_after();
      };
      auto commit_slot = [&]() {
        tc_commit_by(one, acc_full + slot);
        if (++slot == SLOTS * (group + 1)) { slot = SLOTS * group; slot_phase ^= 1u; }
      };
      if (!FP8) next_slot();
#pragma unroll 1
      for (int s = piece.s0 << twice; s < piece.s1 << twice && ok; ++s) {
        if (!(ok = warp_wait_short(full + st, phase, abort_flag, p.status, 117))) break;
        tc_fence_after();
        const uint64_t wd = desc0 + (uint64_t)(st * (Lay::STAGE / 16)), xd = wd + A_BYTES / 16;      // addresses count 16 bytes
        if (FP8) {
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const bool fresh = k == 0 || (k == 2 && piece.down);      // a stage has one accumulator, in the down products two
            if (fresh) {
              if (k > 0) commit_slot();
              next_slot();
              if (!ok) break;
            }
            tc_mma_8bit_by(one, tmem_base + slot * WIDTH, wd + 2 * k, xd + 2 * k, idesc, fresh ? 0u : 1u);
          }
          if (!ok) break;
          tc_commit_by(one, empty + st);
          commit_slot();
        } else {
#pragma unroll
          for (int k = 0; k < 4; ++k)
            tc_mma_by(one, tmem_base + slot * WIDTH + (s & twice) * cols, wd + 2 * k, xd + 2 * k, idesc, ((s >> twice) > piece.s0 || k > 0) ? 1u : 0u);
          tc_commit_by(one, empty + st);
        }
        if (++st == p.stages) { st = 0; phase ^= 1u; }
      }
      if (!FP8 && ok) commit_slot();
      if (group) ring[1] = slot - SLOTS, ring_phase[1] = slot_phase;
      else ring[0] = slot, ring_phase[0] = slot_phase;
    }
  } else {
    const int group = (warp - 2) >> 2, et = (threadIdx.x - 64) & 127, ew = (warp - 2) & 3;
    tile += group * NB * TILE;
    ys += FP8 ? group * Lay::rows(p.ff) * NB : 0;
    const uint32_t quad = warp & 3;
    const int row = (int)quad * 32 + lane;
    const uint32_t lane_base = tmem_base + ((quad * 32u) << 16);
    int slot = group * SLOTS;
    uint32_t slot_phase = 0u, meet_phase = 0u;
    bool ok = true, up_known = false;
    if (slots > 32) {
      // the entries take their places while the first copies are on their way
      if (warp == 2) {
#pragma unroll 1
        for (int s0 = 0; s0 < slots; s0 += 32) {
          const int s = s0 + lane, e = s < slots ? p.ids[s] : p.E;
          const unsigned same = __match_any_sync(0xffffffffu, e);
          if (e < p.E) {
            const int from = count[e], at = from + __popc(same & ((1u << lane) - 1u));
            pos[s] = at;
            tok[at] = s / p.top;
            __syncwarp(same);
            if (lane == __ffs(same) - 1) count[e] = from + __popc(same);
          } else if (s < slots) {
            pos[s] = -1;
          }
          __syncwarp();
        }
      }
      asm volatile("bar.sync 1, 256;" ::: "memory");
    }
    // one arrival per warp: those of 32 lanes on one barrier would come one after the other
    auto arrive = [&](uint64_t* bar) {
      __syncwarp();
      if (lane == 0) mbar_arrive(bar);
    };
    // the threads of a group meet (a bounded wait, so that none is left behind when another one gives up).  Here as in every wait of a warp its lanes
    // learn one answer: what follows is for whole warps.
    auto meet_all = [&]() {
      arrive(meet + group);
      ok = ok && warp_wait_short(meet + group, meet_phase, abort_flag, p.status, 118);
      meet_phase ^= 1u;
    };
#pragma unroll 1
    for (int np = 0; ok; ++np) {
      const int q = np % QUEUE;
      if (!(ok = warp_wait_short(q_full + q, (uint32_t)(np / QUEUE) & 1u, abort_flag, p.status, 119))) break;
      const Piece piece = queue[q];
      arrive(q_empty + q);
      if (piece.down < 0) break;
      if ((np & 1) != group) continue;                         // the other group's
      const int c0 = first[piece.a], cnt = first[piece.a + 1] - c0, e = active[piece.a];
      const int cols = piece.down ? (cnt + 15) / 16 * 16 : NB;
      float acc[FP8 ? NB : 1];
      if (FP8) {
#pragma unroll
        for (int c = 0; c < NB; ++c) acc[c] = 0.f;
        // the weights' scale of this thread's row
        const int rows_all = piece.down ? p.d : ffu, KB = ((piece.down ? p.ff : p.d) + 127) / 128;
        const int w_row = piece.down ? piece.tile * TILE + row : (GLU && row >= 64 ? p.ff + piece.tile * 64 + row - 64 : piece.tile * OUT + row);
        // lane l holds those of stage l of the next 32, for the two row blocks that the warp's rows can lie in
        const int w_block = min(w_row, rows_all - 1) / 128, block_a = __shfl_sync(0xffffffffu, w_block, 0), block_b = __shfl_sync(0xffffffffu, w_block, 31);
        const size_t ws_at = (size_t)e * ((rows_all + 127) / 128);
        const float* ws = piece.down ? p.sd : p.su;
        const int steps = (piece.s1 - piece.s0) << piece.down;          // accumulators: a stage has one, in the down products two
        const float* f = ys;
        // the columns' scales: of the tokens, or of a window of this expert's u (whose first copies are on their way)
        auto column_scales = [&](int i) {
          if (piece.down && !up_known) ok = ok && warp_wait_short(&up_done, 0u, abort_flag, p.status, 120);
          up_known = piece.down;
          meet_all();                                        // nobody reads the last ones any more
          const int blocks = (p.ff + 63) / 64, b0 = 2 * piece.s0 + i, rows = piece.down ? min(steps - i, WINDOW) : 1, some = piece.down ? cnt : p.n;
          const float* scales = piece.down ? p.us + (size_t)c0 * blocks + b0 : p.hs;
#pragma unroll 2
          for (int j = et; j < rows * cols; j += 128) {
            const int c = j / rows, b = j - c * rows;        // neighbours read neighbouring blocks of an entry
            ys[b * NB + c] = c < some && (!piece.down || b0 + b < blocks) ? __ldcg(scales + (piece.down ? c * blocks + b : c)) : 0.f;
          }
          meet_all();
          f = ys;
        };
        column_scales(0);
        float wa = 0.f, wb = 0.f;
#pragma unroll 1
        for (int i = 0; i < steps; ++i) {
          const int s = i >> piece.down;
          if ((i & (32 << piece.down) - 1) == 0 && piece.s0 + s + lane < piece.s1) {
            wa = block_scale(ws, p.e8m0, (ws_at + block_a) * KB + piece.s0 + s + lane);
            wb = block_scale(ws, p.e8m0, (ws_at + block_b) * KB + piece.s0 + s + lane);
          }
          if (piece.down && i > 0 && i % WINDOW == 0) column_scales(i);
          __syncwarp();
          const float w_a = __shfl_sync(0xffffffffu, wa, s & 31), w_b = __shfl_sync(0xffffffffu, wb, s & 31);
          // the weights' scale first: what it makes of a sum (up to 2^25) stays in float32's range for scales up to 2^100, and tokens may be of any size
          const float w = w_block == block_a ? w_a : w_b;
          if (ok) ok = warp_wait_short(acc_full + slot, slot_phase, abort_flag, p.status, 120);
          const uint32_t from = lane_base + (uint32_t)(slot * WIDTH);
          tc_fence_after();
#pragma unroll
          for (int cc = 0; cc < NB; cc += 16)
            if (cc < cols) {
              uint32_t hi[16], lo[16];
              tc_ld16(from + cc, hi);
              tc_ld16(from + cols + cc, lo);
              tc_wait_ld();
#pragma unroll
              for (int j = 0; j < 16; j += 4) {
                const float4 x = *reinterpret_cast<const float4*>(f + cc + j);
                const float fx[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
                for (int k = 0; k < 4; ++k)
                  acc[cc + j + k] = fmaf(fmaf(__uint_as_float(lo[j + k]), 0.0625f, __uint_as_float(hi[j + k])) * w, fx[k], acc[cc + j + k]);
              }
            }
          tc_fence_before();
          arrive(acc_empty + slot);
          if (++slot == SLOTS * (group + 1)) { slot = SLOTS * group; slot_phase ^= 1u; }
          f += piece.down ? NB : 0;
        }
      } else {
        ok = warp_wait_short(acc_full + slot, slot_phase, abort_flag, p.status, 120);
        tc_fence_after();
      }
      // to shared memory, from where a few instructions per entry take them on: what is executed once per piece costs the fetch of its
      // code (most of it from DRAM, as a step's weights pass through the L2) more than its work
      meet_all();                                              // the last piece's tile has been read
      if (FP8) {
#pragma unroll
        for (int c = 0; c < NB; ++c) tile[c * TILE + row] = acc[FP8 ? c : 0];
      } else if (ok) {
#pragma unroll 1
        for (int cc = 0; cc < cols; cc += 16) {
          uint32_t v[16], lo[16];
          tc_ld16(lane_base + (uint32_t)(slot * WIDTH + cc), v);
          tc_ld16(lane_base + (uint32_t)(slot * WIDTH + (piece.down ? cols + cc : cc)), lo);
          tc_wait_ld();
#pragma unroll
          for (int c = 0; c < 16; ++c) tile[(cc + c) * TILE + row] = __uint_as_float(v[c]) + (piece.down ? __uint_as_float(lo[c]) : 0.f);
        }
      }
      if (!piece.down) {
        meet_all();
        const int blocks = (p.ff + 63) / 64;
#pragma unroll 1
        for (int i = ew; i < cnt; i += 4) {
          const float* from = tile + tok[c0 + i] * TILE;
#pragma unroll 1
          for (int b = 0; b < OUT / 64; ++b) {
            const int f0 = piece.tile * OUT + 64 * b;          // 64 numbers of u: two per lane
            float v[2];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              const float z = from[64 * b + 32 * j + lane];
              v[j] = GLU ? z / (1.f + expf(-z)) * from[64 + 32 * j + lane] : gelu_erf(z);
            }
            if (FP8) {
              uint32_t m = 0u;
#pragma unroll
              for (int j = 0; j < 2; ++j)
                if (f0 + 32 * j + lane < p.ff) m = max(m, __float_as_uint(v[j]) & 0x7fffffffu);
              m = __reduce_max_sync(0xffffffffu, m);
              const int code = scale_code(m);
              const float inv = inverse_scale(code);
              uint32_t hi, lo;
              two_e4m3x2(v[0], v[1], inv, hi, lo);
#pragma unroll
              for (int j = 0; j < 2; ++j)
                if (f0 + 32 * j + lane < p.ff) {
                  unsigned char* to = p.u + (size_t)(c0 + i) * p.ff + f0 + 32 * j + lane;
                  to[0] = (unsigned char)(hi >> (8 * j));
                  to[(size_t)slots * p.ff] = (unsigned char)(lo >> (8 * j));
                }
              if (lane == 0 && f0 < p.ff) p.us[(size_t)(c0 + i) * blocks + f0 / 64] = scale_value(code);
            } else {
#pragma unroll
              for (int j = 0; j < 2; ++j)
                if (f0 + 32 * j + lane < p.ff) {
                  __nv_bfloat16* to = reinterpret_cast<__nv_bfloat16*>(p.u) + (size_t)(c0 + i) * p.ff + f0 + 32 * j + lane;
                  const __nv_bfloat16 hi = __float2bfloat16_rn(v[j]);
                  to[0] = hi;
                  to[(size_t)slots * p.ff] = __float2bfloat16_rn(isinf(__bfloat162float(hi)) ? 0.f : v[j] - __bfloat162float(hi));
                }
            }
          }
        }
        fence_async_all();                                     // u is read through the async proxy
        __threadfence();
        meet_all();
        if (et == 0 && ok) atomicAdd(p.counters + 1, 1);
      } else {
        const int col = piece.tile * TILE + row;
        float* y = p.y + ((size_t)piece.split * entries + c0) * p.d + col;
        if (col < p.d) {
#pragma unroll 4
          for (int c = 0; c < cnt; ++c) y[(size_t)c * p.d] = tile[c * TILE + row];
        }
        __threadfence();
        meet_all();
        if (et == 0 && ok) atomicAdd(p.counters + 3, 1);
      }
      if (!FP8) {
        tc_fence_before();
        arrive(acc_empty + slot);
        if (++slot == SLOTS * (group + 1)) { slot = SLOTS * group; slot_phase ^= 1u; }
      }
    }
    // ---- when every down piece of every CTA is done: the sums over the choices, four columns of a token per thread
    if (et == 0 && ok && !wait_for(p.counters + 3, down_pieces, p.status, abort_flag)) ok = false;
    ok = __all_sync(0xffffffffu, ok);
    __threadfence();
    meet_all();
    // few of them: eight lanes share a thread's results
    const int quads = (int)p.quads.by, parts = p.top * splits, threads = (int)gridDim.x * 256, share = p.n * quads * 8 <= threads ? 8 : 1;
    const int sub = (threadIdx.x - 64) % share;
#pragma unroll 1
    for (int i = ((int)blockIdx.x * 256 + (int)threadIdx.x - 64) / share; ok && i < p.n * quads; i += threads / share) {
      int rest;
      const int t = p.quads(i, rest), c4 = 4 * rest;
      float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
      if (p.add != nullptr && sub == 0)
        sum = scaled(four_bf16(p.add + (size_t)t * p.d + c4), p.gate != nullptr ? 1.f / (1.f + expf(-p.gate[t])) : 1.f);
#pragma unroll 1
      for (int i0 = sub; i0 < parts; i0 += 4 * share) {        // four (choice, slice) results in flight
        float4 x[4];
        float w[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int part = i0 + j * share, k = part >> shift, split = part & (splits - 1);
          w[j] = 0.f;
          x[j] = make_float4(0.f, 0.f, 0.f, 0.f);
          if (part < parts) {
            const int at = pos[t * p.top + k];
            w[j] = p.wts[t * p.top + k];
            if (at >= 0) x[j] = __ldcg(reinterpret_cast<const float4*>(p.y + ((size_t)split * entries + at) * p.d + c4));
            else if (split == 0) x[j] = four_bf16(p.h + (size_t)t * p.d + c4);
          }
        }
#pragma unroll
        for (int j = 0; j < 4; ++j)
          sum = make_float4(fmaf(w[j], x[j].x, sum.x), fmaf(w[j], x[j].y, sum.y), fmaf(w[j], x[j].z, sum.z), fmaf(w[j], x[j].w, sum.w));
      }
      if (share == 8) {
        const unsigned eight = 0xffu << (lane & 24);
#pragma unroll
        for (int o = 4; o > 0; o >>= 1)
          sum = make_float4(sum.x + __shfl_xor_sync(eight, sum.x, o), sum.y + __shfl_xor_sync(eight, sum.y, o),
                            sum.z + __shfl_xor_sync(eight, sum.z, o), sum.w + __shfl_xor_sync(eight, sum.w, o));
        if (sub != 0) continue;
      }
      const __nv_bfloat162 lo = __floats2bfloat162_rn(sum.x, sum.y), hi = __floats2bfloat162_rn(sum.z, sum.w);
      *reinterpret_cast<uint2*>(p.out + (size_t)t * p.d + c4) =
          make_uint2(*reinterpret_cast<const uint32_t*>(&lo), *reinterpret_cast<const uint32_t*>(&hi));
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(TMEM_COLS) : "memory");
  }
}

// rows x K numbers of one or two bytes; box = box_rows x 128 bytes, 128-byte swizzle; what lies outside reads as 0
bool make_map(CUtensorMap* map, const void* base, long long rows, int K, int bytes, int box_rows) {
  auto fn = encode_fn();
  if (fn == nullptr) return false;
  cuuint64_t dims[2] = {(cuuint64_t)K, (cuuint64_t)rows};
  cuuint64_t strides[1] = {(cuuint64_t)K * bytes};
  cuuint32_t box[2] = {(cuuint32_t)(128 / bytes), (cuuint32_t)box_rows};
  cuuint32_t elem[2] = {1, 1};
  return fn(map, bytes == 1 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(base), dims, strides,
            box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <bool FP8, bool GLU, int NB>
int launch_experts(const CUtensorMap* maps, LayerParams p, cudaStream_t stream) {
  using Lay = Layout<FP8, NB>;
  p.stages = Lay::stages(p.ff, p.n * p.top, p.E);
  if (p.stages == 0) return (int)cudaErrorInvalidValue;
  p.up_tiles = Divide::of((p.ff + (GLU ? 63 : 127)) / (GLU ? 64 : 128));
  p.down_tiles = Divide::of((p.d + TILE - 1) / TILE);
  p.quads = Divide::of(p.d / 4);
  static bool set_dev[bspec::kMaxDevices] = {};
  bool& set = set_dev[bspec::current_device()];
  if (!set) {
    const cudaError_t e = cudaFuncSetAttribute(moe_layer_experts_kernel<FP8, GLU, NB>, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_BUDGET);
    if (e != cudaSuccess) return (int)e;
    set = true;
  }
  BSPEC_LAUNCH((moe_layer_experts_kernel<FP8, GLU, NB>), bspec::sm_count(), LAYER_THREADS,
               1024 + Lay::fixed(p.ff, p.n * p.top, p.E) + (size_t)p.stages * Lay::STAGE, stream,
               maps[0], maps[1], maps[2], maps[3], p);
  return BSPEC_LAUNCH_CHECK();
}

}  // namespace

namespace {
// Places of a call's intermediate results in its scratch (counters at 0): expert numbers, weights, gate logits, the tokens' 8-bit numbers and their
// scales, u and its scales, the experts' results.  Returns the size.
enum { AT_IDS, AT_WTS, AT_GATE, AT_HQ, AT_HS, AT_U, AT_US, AT_Y, AT_PARTS };
long long places(int n, int d, int ff, int top, bool fp8, long long (&at)[AT_PARTS]) {
  const long long slots = (long long)n * top, blocks_ff = (ff + 63) / 64;
  const long long bytes[AT_PARTS] = {4 * slots, 4 * slots, 4ll * n, fp8 ? 2ll * n * d : 0, fp8 ? 4ll * n : 0,
                                     (fp8 ? 2 : 4) * slots * ff, fp8 ? 4 * slots * blocks_ff : 0, 4 * MAX_SPLITS * slots * d};
  long long size = 16;
  for (int i = 0; i < AT_PARTS; ++i) {
    at[i] = (size + 127) / 128 * 128;
    size = at[i] + bytes[i];
  }
  return size;
}
}  // namespace

// Bytes of scratch of a call; 0 where its lists (two words per choice, three per expert) do not fit into shared memory beside three stages: 64
// tokens with 8-bit experts of inner sizes of 4,096 and more take 60 of 64 experts each, 55 of 256, 37 of 1,024; with bfloat16 ones all of 64, 167 of 256,
// 149 of 1,024.
BSPEC_API long long bspec_moe_layer_scratch(int n, int d, int ff, int top, int fp8, int E) {
  long long at[AT_PARTS];
  const int slots = n * top;
  const int stages = fp8 ? (n <= 16 ? Layout<true, 16>::stages(ff, slots, E) : n <= 32 ? Layout<true, 32>::stages(ff, slots, E) : Layout<true, 64>::stages(ff, slots, E))
                         : (n <= 16 ? Layout<false, 16>::stages(ff, slots, E) : n <= 32 ? Layout<false, 32>::stages(ff, slots, E) : Layout<false, 64>::stages(ff, slots, E));
  return stages == 0 ? 0 : places(n, d, ff, top, fp8 != 0, at);
}

// h, add (may be null), out: bfloat16 [n, d].  router: `rows` rows, C = experts and identity experts, then perhaps one (rows = C + 1) whose
// logit's sigmoid multiplies add.  corr (may be null): C numbers.  wu [E, ff, d] (glu: [E, 2 ff, d]), wd [E, d, ff]: bfloat16, or e4m3 with
// su, sd, the scales of their 128 x 128 blocks (float32, or 8-bit exponents with e8m0).  status: one int on the device, 0 unless a
// bounded wait ran out.
BSPEC_API int bspec_moe_layer(const void* h, int n, int d, const void* router, int rows, const void* corr, int corr_dtype, int C, int G,
                              int keep, int top, float scale, int rule, const void* wu, const void* wd, const void* su, const void* sd,
                              int e8m0, int E, int ff, int glu, const void* add, void* out, void* scratch, int* status, cudaStream_t stream) {
  if (n <= 0) return 0;
  const bool fp8 = su != nullptr;
  const int unit = fp8 ? 16 : 8, bytes = fp8 ? 1 : 2, ffu = glu ? 2 * ff : ff;
  if (n > LAYER_TOKENS || d <= 0 || ff <= 0 || d % unit || ff % unit || E <= 0 || C < E || C > MAX_EXPERTS || rows < C || rows > C + 1 || top <= 0 ||
      top > C || G <= 0 || C % G || keep <= 0 || keep > G || (long long)keep * (C / G) < top || (fp8 && sd == nullptr) || (rows > C && add == nullptr) ||
      ((reinterpret_cast<uintptr_t>(h) | reinterpret_cast<uintptr_t>(router) | reinterpret_cast<uintptr_t>(wu) | reinterpret_cast<uintptr_t>(wd) |
        reinterpret_cast<uintptr_t>(scratch) | reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(add)) & 15) ||
      (long long)E * ffu > 0x7fffffff - 256 || (long long)E * d > 0x7fffffff - 256)
    return (int)cudaErrorInvalidValue;
  if (bspec_moe_layer_scratch(n, d, ff, top, fp8, E) == 0) return (int)cudaErrorInvalidValue;       // before the first kernel
  long long at[AT_PARTS];
  places(n, d, ff, top, fp8, at);
  char* base = (char*)scratch;
  int* counters = (int*)base;
  LayerParams p = {};
  p.su = (const float*)su; p.sd = (const float*)sd; p.e8m0 = e8m0;
  p.ids = (const int*)(base + at[AT_IDS]); p.wts = (const float*)(base + at[AT_WTS]);
  p.gate = rows > C ? (const float*)(base + at[AT_GATE]) : nullptr;
  p.h = (const __nv_bfloat16*)h; p.add = (const __nv_bfloat16*)add;
  p.hs = (const float*)(base + at[AT_HS]); p.u = (unsigned char*)(base + at[AT_U]); p.us = (float*)(base + at[AT_US]);
  p.y = (float*)(base + at[AT_Y]);
  p.out = (__nv_bfloat16*)out; p.counters = counters; p.status = status;
  p.n = n; p.d = d; p.ff = ff; p.E = E; p.top = top;
  CUtensorMap maps[4];
  if (!make_map(maps, wu, (long long)E * ffu, d, bytes, 64) || !make_map(maps + 1, wd, (long long)E * d, ff, bytes, 64) ||
      !make_map(maps + 2, fp8 ? (const void*)(base + at[AT_HQ]) : h, fp8 ? 2 * n : n, d, bytes, 16) ||
      !make_map(maps + 3, p.u, 2ll * n * top, ff, bytes, 16))
    return (int)cudaErrorInvalidValue;

  const int tiles = (rows + 15) / 16, steps = (d + 31) / 32;
  int slices = ROUTE_CLUSTER * ROUTE_WARPS / tiles;              // of the router's k: as many as there are warps left
  if (slices > (steps + 3) / 4) slices = (steps + 3) / 4;        // at least one batch of loads each
  if (slices < 1) slices = 1;
  const size_t smem = ((size_t)tiles * slices * 16 * ROUTE_TOKENS + (size_t)(ROUTE_WARPS * 3 + 1) * C) * 4;
  if (smem > 48 * 1024) {
    const cudaError_t e = cudaFuncSetAttribute(moe_layer_route_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 200 * 1024);
    if (e != cudaSuccess) return (int)e;
  }
  // started when the kernel before has ended: launched early, its clusters go wherever that one's CTAs happen to end first (measured, 61 tokens:
  // 151 us instead of 142)
  BSPEC_LAUNCH_SERIALIZED((moe_layer_route_kernel), ROUTE_CLUSTER * ((n + ROUTE_TOKENS - 1) / ROUTE_TOKENS) * (fp8 ? 2 : 1), 32 * ROUTE_WARPS, smem, stream,
               (const __nv_bfloat16*)h, n, d, (const __nv_bfloat16*)router, rows, slices, corr, corr_dtype, C, G, keep, top, scale, rule,
               (int*)(base + at[AT_IDS]), (float*)(base + at[AT_WTS]), (float*)(base + at[AT_GATE]), counters,
               fp8 ? (uint8_t*)(base + at[AT_HQ]) : (uint8_t*)nullptr, (float*)(base + at[AT_HS]));
  const int e = BSPEC_LAUNCH_CHECK();
  if (e != 0) return e;
#define LN(F, G) (n <= 16 ? launch_experts<F, G, 16>(maps, p, stream) : n <= 32 ? launch_experts<F, G, 32>(maps, p, stream) \
                                                                              : launch_experts<F, G, 64>(maps, p, stream))
  if (fp8) return glu ? LN(true, true) : LN(true, false);
  return glu ? LN(false, true) : LN(false, false);
#undef LN
}

BSPEC_DEFINE_TRACE_SETTER(bspec_trace_set_moe_layer)
