// A whole routed feed-forward for a few tokens (at most 64) in two kernels:
//   z = Wr h,  (ids, w) = choice(z)                      the rules of moe_choose.cuh
//   u[t, k] = act(Wup[ids[t, k]] h[t])                   act: GELU, or silu(gate) * up with Wup = [gate; up]
//   out[t]  = add[t] * sigmoid(gate logit) + sum over k of w[t, k] * (Wdown[ids[t, k]] u[t, k], or h[t] for an identity expert)
// Experts in bfloat16, or in 8-bit floating point (e4m3) with a scale per 128 x 128 block; activations stay bfloat16 either
// way (u is rounded to bfloat16 between the products: it is the operand of a bfloat16 product), sums are float32.
//
// Bound by the read of the chosen experts' weights, each of which is used once per step: a weight is fetched once, by
// cp.async into a ring of its warp's own (a lane reads back the 16 bytes it fetched itself, so the ring needs no barriers, and
// several KB per warp are in flight whatever the registers hold), and meets up to 64 token columns on mma.sync m16n8k16.  The
// WEIGHT rows take the 16 rows of the product, the expert's tokens its columns, 8 at a time; both operands number the k of a
// step in the same permuted order (lane l % 4 holds neighbouring k), which a sum over k does not notice.
//
//   route    one cluster of 8 CTAs per 8 tokens: 64 warps share the router's rows and k, partial sums meet in the first CTA's
//            shared memory, whose warps choose for a token each.  It also clears the counters of the second kernel.
//   experts  one CTA per SM.  First all pieces of the up products are drawn from one counter, then pieces of 16 output columns
//            over all chosen experts.  A piece of the second kind waits until every piece of the first kind is done; those have
//            all been drawn by CTAs that run and wait for nothing, so it ends however many CTAs the device can hold.  A column's
//            sum runs over the experts in a fixed order: no atomic adds numbers.
#include "moe_choose.cuh"
#include <math.h>

using namespace bspec;

namespace {

constexpr int LAYER_TOKENS = 64;             // most tokens of a step
constexpr int ROUTE_CLUSTER = 8, ROUTE_WARPS = 8, ROUTE_TOKENS = 8;
constexpr int WARPS = 16, LAYER_THREADS = 32 * WARPS;
constexpr int SMEM_BUDGET = 220 * 1024;

__device__ __forceinline__ uint32_t smem_addr(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }

// ------------------------------------------------------------------------------------------------ the router
// z partials: [unit = (16 rows of the router, slice of k)][16 rows][8 tokens] in the first CTA of the cluster.
__global__ void __cluster_dims__(ROUTE_CLUSTER, 1, 1) __launch_bounds__(32 * ROUTE_WARPS)
moe_layer_route_kernel(const __nv_bfloat16* __restrict__ h, int n, int d, const __nv_bfloat16* __restrict__ wr, int rows, int slices,
                       const void* __restrict__ corr, int corr_dtype, int C, int G, int keep, int top, float scale, int rule,
                       int* __restrict__ ids, float* __restrict__ wts, float* __restrict__ gate, int* __restrict__ counters) {
  bspec::pdl_prologue(84);
  extern __shared__ float sm[];
  const int tiles = (rows + 15) / 16, units = tiles * slices;
  float* part = sm;                                            // [units][16][8]
  const int rank = blockIdx.x % ROUTE_CLUSTER, t0 = blockIdx.x / ROUTE_CLUSTER * ROUTE_TOKENS;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, q = lane & 3;
  if (blockIdx.x == 0 && threadIdx.x < 4) counters[threadIdx.x] = 0;
  // every CTA of the cluster runs before another one writes to its memory
  asm volatile("barrier.cluster.arrive.relaxed.aligned;\n\tbarrier.cluster.wait.aligned;" ::: "memory");
  uint32_t first;                                              // the first CTA's partials
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(first) : "r"(smem_addr(part)), "r"(0));
  const int steps = (d + 31) / 32, per = (steps + slices - 1) / slices;
  const uint4 zero = make_uint4(0u, 0u, 0u, 0u);
  const bool token = t0 + g < n;
  for (int unit = rank * ROUTE_WARPS + warp; unit < units; unit += ROUTE_CLUSTER * ROUTE_WARPS) {
    const int r0 = unit / slices * 16, s0 = unit % slices * per, s1 = min(steps, s0 + per);
    const __nv_bfloat16* lo = wr + (size_t)min(r0 + g, rows - 1) * d + 8 * q;
    const __nv_bfloat16* hi = wr + (size_t)min(r0 + g + 8, rows - 1) * d + 8 * q;
    const __nv_bfloat16* x = h + (size_t)min(t0 + g, n - 1) * d + 8 * q;
    float acc[4] = {0.f, 0.f, 0.f, 0.f};
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
      const int at = (unit * 16 + g + 8 * (i >> 1)) * ROUTE_TOKENS + 2 * q + (i & 1);
      asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(first + 4u * (uint32_t)at), "f"(acc[i]) : "memory");
    }
  }
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
  const int t = t0 + warp;
  if (rank != 0 || t >= n) return;
  float* sc = part + (size_t)units * 16 * ROUTE_TOKENS + (size_t)warp * 3 * C;
  float* ch = sc + C;
  for (int e = lane; e < rows; e += 32) {
    float z = 0.f;
    for (int s = 0; s < slices; ++s) z += part[((e / 16 * slices + s) * 16 + e % 16) * ROUTE_TOKENS + warp];
    if (e < C) route_score(rule, z, corr != nullptr ? load_as_f32(corr, corr_dtype, e) : 0.f, sc + e, ch + e);
    else gate[t] = z;                                          // the row behind the experts' rows
  }
  __syncwarp();
  choose_experts<true>(sc, ch, ch + C, corr, corr_dtype, C, G, keep, top, scale, rule, ids + (size_t)t * top, wts + (size_t)t * top);
}

// ------------------------------------------------------------------------------------------------ the experts
struct LayerParams {
  const __nv_bfloat16* h;                    // [n, d]
  const unsigned char* wu;                   // [E, ffu, d]
  const unsigned char* wd;                   // [E, d, ff]
  const void* su;                            // scales of 128 x 128 blocks, or null
  const void* sd;
  int e8m0;
  const int* ids;                            // [n, top]; E and above: the token's own h
  const float* wts;
  const float* gate;                         // [n] or null
  const __nv_bfloat16* add;                  // [n, d] or null
  __nv_bfloat16* u;                          // [n top, ff]
  __nv_bfloat16* out;                        // [n, d]
  int* counters;                             // {pieces drawn, up pieces done, output pieces drawn}, zero
  int* status;
  int n, d, ff, E, top;
  int stages, ring_tiles;                    // of a warp's ring: stages, and column tiles whose tokens are fetched through it
};

__device__ __forceinline__ void cp16(uint32_t dst, const void* src, bool live) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(live ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp16_l1(uint32_t dst, const void* src, bool live) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(live ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
// all but the newest `left` groups have landed
__device__ __forceinline__ void cp_wait(int left) {
  if (left <= 0) asm volatile("cp.async.wait_group 0;" ::: "memory");
  else if (left == 1) asm volatile("cp.async.wait_group 1;" ::: "memory");
  else if (left == 2) asm volatile("cp.async.wait_group 2;" ::: "memory");
  else asm volatile("cp.async.wait_group 3;" ::: "memory");
}
__device__ __forceinline__ uint4 lds16(uint32_t at) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at) : "memory");
  return v;
}
// Four e4m3 numbers -> bfloat16, two to a register.  Sign, exponent and fraction move to their places, which leaves a number 2^120 times
// too small (the exponents' biases differ by 120; numbers below e4m3's normal ones become bfloat16 numbers below its normal ones); the
// product with 2^120 is exact.
__device__ __forceinline__ uint32_t widen(uint32_t halves) {       // each half: the number in its high byte, 0 in its low one
  const uint32_t r = (halves & 0x80008000u) | ((halves >> 4) & 0x07f007f0u);
  const __nv_bfloat162 big = __halves2bfloat162(__ushort_as_bfloat16(0x7b80), __ushort_as_bfloat16(0x7b80));      // 2^120
  const __nv_bfloat162 v = __hmul2(*reinterpret_cast<const __nv_bfloat162*>(&r), big);
  return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ void widen4(uint32_t w, uint32_t& lo, uint32_t& hi) {
  lo = widen(__byte_perm(w, 0u, 0x1404));
  hi = widen(__byte_perm(w, 0u, 0x3424));
}
__device__ __forceinline__ float block_scale(const void* p, int e8m0, size_t i) {
  if (!e8m0) return reinterpret_cast<const float*>(p)[i];
  const uint32_t code = reinterpret_cast<const uint8_t*>(p)[i];
  return __uint_as_float(code == 0u ? 0x00400000u : (code == 255u ? 0x7fc00000u : code << 23));
}

// A stage of a warp's ring: 16 weight rows of DEPTH k (2 KB), then for each column tile 8 tokens' numbers.
template <bool FP8> struct Ring;
template <> struct Ring<false> { static constexpr int DEPTH = 64, ESZ = 2, STEP = 32, B_PIECES = 2; };
template <> struct Ring<true> { static constexpr int DEPTH = 128, ESZ = 1, STEP = 64, B_PIECES = 4; };
constexpr int A_BYTES = 2048;

// the weights of a stage: rows `lo` and `hi` of this lane (null: zeros), k from k0
template <bool FP8>
__device__ __forceinline__ void fetch_weights(uint32_t at, const unsigned char* lo, const unsigned char* hi, const unsigned char* any,
                                              int k0, int K) {
  using R = Ring<FP8>;
  const int q = threadIdx.x & 3;
#pragma unroll
  for (int s = 0; s < 2; ++s) {
    const int k = k0 + R::STEP * s + (16 / R::ESZ) * q;
    const bool in = k < K;
    cp16(at + (2 * s) * 512, in && lo ? lo + (size_t)k * R::ESZ : any, in && lo);
    cp16(at + (2 * s + 1) * 512, in && hi ? hi + (size_t)k * R::ESZ : any, in && hi);
  }
}
// the k of piece p of a token's numbers in a stage
template <bool FP8>
__device__ __forceinline__ int token_k(int k0, int p) {
  const int q = threadIdx.x & 3;
  return FP8 ? k0 + 64 * (p >> 1) + 16 * q + 8 * (p & 1) : k0 + 32 * p + 8 * q;
}
template <bool FP8, bool L1>
__device__ __forceinline__ void fetch_tokens(uint32_t at, const __nv_bfloat16* row, const void* any, int k0, int K) {
#pragma unroll
  for (int p = 0; p < Ring<FP8>::B_PIECES; ++p) {
    const int k = token_k<FP8>(k0, p);
    const bool live = row != nullptr && k < K;
    if (L1) cp16_l1(at + p * 512, live ? (const void*)(row + k) : any, live);
    else cp16(at + p * 512, live ? (const void*)(row + k) : any, live);
  }
}

// The products of one stage: acc[t] += the 16 rows x column tile t, for the first `nt` tiles.  `b_at`: the tokens' numbers in the
// ring (T column tiles of them), or 0: they are read from `rows`.  8-bit weights: s_lo, s_hi are the scales of this lane's two rows.
template <bool FP8, int T>
__device__ __forceinline__ void multiply(uint32_t a_at, uint32_t b_at, const __nv_bfloat16* const* rows, int k0, int K, int nt,
                                         float s_lo, float s_hi, float (&acc)[T][4]) {
  using R = Ring<FP8>;
  const uint4 zero = make_uint4(0u, 0u, 0u, 0u);
  auto token = [&](int t, int p) -> uint4 {
    if (b_at != 0u) return lds16(b_at + (uint32_t)(t * R::B_PIECES + p) * 512u);
    const int k = token_k<FP8>(k0, p);
    return rows[t] != nullptr && k < K ? __ldcg(reinterpret_cast<const uint4*>(rows[t] + k)) : zero;
  };
  if (FP8) {
    float sum[T][4];
#pragma unroll
    for (int t = 0; t < T; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) sum[t][i] = 0.f;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const uint4 lo = lds16(a_at + (2 * s) * 512), hi = lds16(a_at + (2 * s + 1) * 512);
      const uint32_t l[4] = {lo.x, lo.y, lo.z, lo.w}, h[4] = {hi.x, hi.y, hi.z, hi.w};
      uint32_t wl[8], wh[8];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        widen4(l[j], wl[2 * j], wl[2 * j + 1]);
        widen4(h[j], wh[2 * j], wh[2 * j + 1]);
      }
#pragma unroll
      for (int t = 0; t < T; ++t)
        if (t < nt) {
          const uint4 x = token(t, 2 * s), y = token(t, 2 * s + 1);
          mma_bf16_16816(sum[t], wl[0], wh[0], wl[1], wh[1], x.x, x.y);
          mma_bf16_16816(sum[t], wl[2], wh[2], wl[3], wh[3], x.z, x.w);
          mma_bf16_16816(sum[t], wl[4], wh[4], wl[5], wh[5], y.x, y.y);
          mma_bf16_16816(sum[t], wl[6], wh[6], wl[7], wh[7], y.z, y.w);
        }
    }
#pragma unroll
    for (int t = 0; t < T; ++t) {
      acc[t][0] = fmaf(sum[t][0], s_lo, acc[t][0]);
      acc[t][1] = fmaf(sum[t][1], s_lo, acc[t][1]);
      acc[t][2] = fmaf(sum[t][2], s_hi, acc[t][2]);
      acc[t][3] = fmaf(sum[t][3], s_hi, acc[t][3]);
    }
  } else {
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const uint4 lo = lds16(a_at + (2 * s) * 512), hi = lds16(a_at + (2 * s + 1) * 512);
#pragma unroll
      for (int t = 0; t < T; ++t)
        if (t < nt) {
          const uint4 x = token(t, s);
          mma_bf16_16816(acc[t], lo.x, hi.x, lo.y, hi.y, x.x, x.y);
          mma_bf16_16816(acc[t], lo.z, hi.z, lo.w, hi.w, x.z, x.w);
        }
    }
  }
}

// What all pieces of a CTA know of the step, in shared memory.
struct Lists {
  int* active;                               // chosen experts, ascending
  int* first;                                // [active + 1] where an expert's entries begin
  int* slot;                                 // entries: (token, choice) numbers by expert
  int* count;                                // [E] scratch
  float* total;                              // [WARPS][8 tiles][16 rows] sums of a warp; before that its partial tiles
  uint32_t ring;                             // this warp's
};
struct Block {
  int drawn[WARPS];                          // a team's next piece
  int base, n_active, most, done, piece, stop;
};

template <bool FP8, bool GLU, int T>
__device__ __forceinline__ void run_layer(const LayerParams& p, const Lists& L, Block& B) {
  using R = Ring<FP8>;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, q = lane & 3;
  const bool ringed = T <= p.ring_tiles;
  const uint32_t stage_bytes = A_BYTES + (uint32_t)p.ring_tiles * R::B_PIECES * 512u;
  const uint32_t my_ring = L.ring + 16u * lane;
  const int A = B.n_active, ffu = GLU ? 2 * p.ff : p.ff;
  const int stages = p.stages;
  const __nv_bfloat16* rows[T];

  // ---- up products: a piece is 16 rows of one expert (GLU: 8 gate rows and their 8 up rows), shared by the warps of a team
  {
    constexpr int OUT = GLU ? 8 : 16;
    const int tiles = (p.ff + OUT - 1) / OUT, pieces = A * tiles, depth = (p.d + R::DEPTH - 1) / R::DEPTH;
    // fewer pieces than warps: a team of 2, 4 or 8 warps cuts a piece's k, as long as each has four stages
    int team_size = 1;
    while (team_size < 8 && (long long)pieces * team_size * 2 <= (long long)gridDim.x * WARPS && depth >= 8 * team_size) team_size *= 2;
    const int team = warp / team_size, member = warp % team_size;
    const int per = (depth + team_size - 1) / team_size, from = min(depth, member * per), to = min(depth, from + per);
    if (threadIdx.x == 0) B.base = atomicAdd(p.counters, WARPS / team_size);
    __syncthreads();
    int piece = B.base + team, mine = 0;
    while (piece < pieces) {
      int next = 0;
      if (member == 0 && lane == 0) next = atomicAdd(p.counters, 1);
      const int a = piece / tiles, i0 = (piece - a * tiles) * OUT, e = L.active[a];
      const int c0 = L.first[a], cnt = L.first[a + 1] - c0, nt = (cnt + 7) / 8;
      const int r_lo = i0 + g, r_hi = GLU ? p.ff + i0 + g : i0 + 8 + g;
      const unsigned char* we = p.wu + (size_t)e * ffu * p.d * R::ESZ;
      const unsigned char* lo = i0 + g < p.ff ? we + (size_t)r_lo * p.d * R::ESZ : nullptr;
      const unsigned char* hi = (GLU ? i0 + g : i0 + 8 + g) < p.ff ? we + (size_t)r_hi * p.d * R::ESZ : nullptr;
#pragma unroll
      for (int t = 0; t < T; ++t) rows[t] = 8 * t + g < cnt ? p.h + (size_t)(L.slot[c0 + 8 * t + g] / p.top) * p.d : nullptr;
      float acc[T][4];
#pragma unroll
      for (int t = 0; t < T; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[t][i] = 0.f;
      const int KB = (p.d + 127) / 128, RB = (ffu + 127) / 128;
      const size_t s_lo_at = ((size_t)e * RB + min(r_lo, ffu - 1) / 128) * KB, s_hi_at = ((size_t)e * RB + min(r_hi, ffu - 1) / 128) * KB;
      auto fetch = [&](int j) {
        if (j < to) {
          const uint32_t at = my_ring + (uint32_t)((j - from) % stages) * stage_bytes;
          fetch_weights<FP8>(at, lo, hi, we, j * R::DEPTH, p.d);
          if (ringed) {
#pragma unroll
            for (int t = 0; t < T; ++t)
              if (t < nt) fetch_tokens<FP8, true>(at + A_BYTES + t * R::B_PIECES * 512, rows[t], we, j * R::DEPTH, p.d);
          }
        }
        cp_commit();
      };
      float s_lo = 1.f, s_hi = 1.f;
      if (FP8 && from < to) {
        s_lo = block_scale(p.su, p.e8m0, s_lo_at + from);
        s_hi = block_scale(p.su, p.e8m0, s_hi_at + from);
      }
      for (int j = 0; j < stages - 1; ++j) fetch(from + j);
      for (int j = from; j < to; ++j) {
        fetch(j + stages - 1);
        cp_wait(stages - 1);
        float n_lo = 1.f, n_hi = 1.f;
        if (FP8 && j + 1 < to) {
          n_lo = block_scale(p.su, p.e8m0, s_lo_at + j + 1);
          n_hi = block_scale(p.su, p.e8m0, s_hi_at + j + 1);
        }
        const uint32_t at = my_ring + (uint32_t)((j - from) % stages) * stage_bytes;
        multiply<FP8, T>(at, ringed ? at + A_BYTES : 0u, rows, j * R::DEPTH, p.d, nt, s_lo, s_hi, acc);
        s_lo = n_lo;
        s_hi = n_hi;
      }
      cp_wait(0);
      if (team_size > 1) {
        float* red = L.total + (size_t)warp * T * 128;
        if (member != 0) {
#pragma unroll
          for (int t = 0; t < T; ++t)
            if (t < nt) {
#pragma unroll
              for (int i = 0; i < 4; ++i) red[(t * 4 + i) * 32 + lane] = acc[t][i];
            }
        }
        if (member == 0 && lane == 0) B.drawn[team] = next;
        asm volatile("bar.sync %0, %1;" ::"r"(team + 1), "r"(team_size * 32) : "memory");
        if (member == 0) {
          for (int m = 1; m < team_size; ++m)
#pragma unroll
            for (int t = 0; t < T; ++t)
              if (t < nt) {
#pragma unroll
                for (int i = 0; i < 4; ++i) acc[t][i] += red[(size_t)m * T * 128 + (t * 4 + i) * 32 + lane];
              }
        }
        next = B.drawn[team];
        asm volatile("bar.sync %0, %1;" ::"r"(team + 1), "r"(team_size * 32) : "memory");
      } else {
        next = __shfl_sync(0xffffffffu, next, 0);
      }
      if (member == 0) {
#pragma unroll
        for (int t = 0; t < T; ++t)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const int c = 8 * t + 2 * q + i;
            if (c >= cnt) continue;
            __nv_bfloat16* u = p.u + (size_t)L.slot[c0 + c] * p.ff + i0 + g;
            if (GLU) {
              const float gv = acc[t][i];
              if (i0 + g < p.ff) *u = __float2bfloat16_rn(gv / (1.f + expf(-gv)) * acc[t][2 + i]);
            } else {
              if (i0 + g < p.ff) u[0] = __float2bfloat16_rn(gelu_erf(acc[t][i]));
              if (i0 + 8 + g < p.ff) u[8] = __float2bfloat16_rn(gelu_erf(acc[t][2 + i]));
            }
          }
        ++mine;
      }
      piece = next;
    }
    if (member == 0 && lane == 0 && mine) atomicAdd(&B.done, mine);
    __syncthreads();
    if (threadIdx.x == 0) {
      if (B.done) {
        __threadfence();
        atomicAdd(p.counters + 1, B.done);
      }
      B.piece = atomicAdd(p.counters + 2, 1);
    }
    __syncthreads();
    // ---- down products: a piece is 16 output columns over all chosen experts; the warps take equal shares of the (expert, k) stages
    const int out_pieces = (p.d + 15) / 16, per_expert = (p.ff + R::DEPTH - 1) / R::DEPTH;
    const int all = A * per_expert, w0 = (int)((long long)all * warp / WARPS), w1 = (int)((long long)all * (warp + 1) / WARPS);
    const int KB = (p.ff + 127) / 128, RB = (p.d + 127) / 128;
    float* total = L.total + (size_t)warp * 8 * T * 16;          // [tokens][16]
    bool first = true;
    while (B.piece < out_pieces) {
      const int n0 = B.piece * 16;
      for (int i = lane; i < p.n * 16; i += 32) total[i] = 0.f;
      __syncwarp();
      const bool live_lo = n0 + g < p.d, live_hi = n0 + 8 + g < p.d;
      auto fetch_w = [&](int j) {
        const int a = j / per_expert, k0 = (j - a * per_expert) * R::DEPTH;
        const unsigned char* we = p.wd + (size_t)L.active[a] * p.d * p.ff * R::ESZ;
        const unsigned char* lo = live_lo ? we + (size_t)(n0 + g) * p.ff * R::ESZ : nullptr;
        const unsigned char* hi = live_hi ? we + (size_t)(n0 + 8 + g) * p.ff * R::ESZ : nullptr;
        fetch_weights<FP8>(my_ring + (uint32_t)((j - w0) % stages) * stage_bytes, lo, hi, we, k0, p.ff);
      };
      auto fetch_u = [&](int j) {
        if (!ringed) return;
        const int a = j / per_expert, k0 = (j - a * per_expert) * R::DEPTH;
        const int c0 = L.first[a], cnt = L.first[a + 1] - c0;
        const uint32_t at = my_ring + (uint32_t)((j - w0) % stages) * stage_bytes + A_BYTES;
#pragma unroll
        for (int t = 0; t < T; ++t)
          if (8 * t < cnt)
            fetch_tokens<FP8, false>(at + t * R::B_PIECES * 512, 8 * t + g < cnt ? p.u + (size_t)L.slot[c0 + 8 * t + g] * p.ff : nullptr,
                                     p.u, k0, p.ff);
      };
      // the first weights are asked for before the wait for the up products
      for (int j = w0; j < min(w1, w0 + stages - 1); ++j) fetch_w(j);
      if (first) {
        first = false;
        if (threadIdx.x == 0) {
          unsigned long long t_from = 0ull;
          for (uint32_t i = 0;; ++i) {
            int v;
            asm volatile("ld.acquire.gpu.global.s32 %0, [%1];" : "=r"(v) : "l"(p.counters + 1) : "memory");
            if (v >= pieces) break;
            if ((i & 255u) == 255u) {
              const unsigned long long now = bspec::global_timer();
              if (t_from == 0ull) t_from = now;
              if (now - t_from > 2000000000ull || i >= (1u << 24) || *reinterpret_cast<volatile int*>(p.status) != 0) {
                atomicCAS(p.status, 0, 111);
                B.stop = 1;
                break;
              }
            }
          }
          __threadfence();
        }
        __syncthreads();
        if (B.stop) break;
      }
      for (int j = w0; j < w0 + stages - 1; ++j) {
        if (j < w1) fetch_u(j);
        cp_commit();
      }
      float acc[T][4];
#pragma unroll
      for (int t = 0; t < T; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[t][i] = 0.f;
      int a = w0 < w1 ? w0 / per_expert : 0, kb = w0 - a * per_expert;
      int c0 = 0, cnt = 0;
      const __nv_bfloat16* at_rows[T];
      auto enter = [&]() {
        c0 = L.first[a];
        cnt = L.first[a + 1] - c0;
#pragma unroll
        for (int t = 0; t < T; ++t) at_rows[t] = 8 * t + g < cnt ? p.u + (size_t)L.slot[c0 + 8 * t + g] * p.ff : nullptr;
      };
      auto scale_of = [&](int aa, int k, int row) {
        return block_scale(p.sd, p.e8m0, ((size_t)L.active[aa] * RB + min(row, p.d - 1) / 128) * KB + k);
      };
      float s_lo = 1.f, s_hi = 1.f;
      if (w0 < w1) {
        enter();
        if (FP8) s_lo = scale_of(a, kb, n0 + g), s_hi = scale_of(a, kb, n0 + 8 + g);
      }
      for (int j = w0; j < w1; ++j) {
        if (j + stages - 1 < w1) {
          fetch_w(j + stages - 1);
          fetch_u(j + stages - 1);
        }
        cp_commit();
        cp_wait(stages - 1);
        float n_lo = 1.f, n_hi = 1.f;
        const bool last = kb + 1 == per_expert;
        if (FP8 && j + 1 < w1) {
          n_lo = scale_of(last ? a + 1 : a, last ? 0 : kb + 1, n0 + g);
          n_hi = scale_of(last ? a + 1 : a, last ? 0 : kb + 1, n0 + 8 + g);
        }
        const uint32_t at = my_ring + (uint32_t)((j - w0) % stages) * stage_bytes;
        multiply<FP8, T>(at, ringed ? at + A_BYTES : 0u, at_rows, kb * R::DEPTH, p.ff, (cnt + 7) / 8, s_lo, s_hi, acc);
        s_lo = n_lo;
        s_hi = n_hi;
        ++kb;
        if (last || j + 1 == w1) {
          // this expert's share is complete: into the warp's sums, weighted
#pragma unroll
          for (int t = 0; t < T; ++t)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const int c = 8 * t + 2 * q + i;
              if (c < cnt) {
                const int slot = L.slot[c0 + c];
                const float w = p.wts[slot];
                float* to = total + slot / p.top * 16 + g;
                to[0] = fmaf(w, acc[t][i], to[0]);
                to[8] = fmaf(w, acc[t][2 + i], to[8]);
              }
              acc[t][i] = acc[t][2 + i] = 0.f;
            }
          __syncwarp();
          if (last && j + 1 < w1) {
            ++a;
            kb = 0;
            enter();
          }
        }
      }
      cp_wait(0);
      __syncthreads();
      if (threadIdx.x == 0) B.base = atomicAdd(p.counters + 2, 1);
      for (int i = threadIdx.x; i < p.n * 16; i += LAYER_THREADS) {
        const int t = i >> 4, col = n0 + (i & 15);
        if (col >= p.d) continue;
        float v = 0.f;
        if (p.add != nullptr) {
          v = to_f32(p.add[(size_t)t * p.d + col]);
          if (p.gate != nullptr) v *= 1.f / (1.f + expf(-p.gate[t]));
        }
#pragma unroll
        for (int w = 0; w < WARPS; ++w) v += L.total[(size_t)w * 8 * T * 16 + i];
        for (int k = 0; k < p.top; ++k)
          if (p.ids[(size_t)t * p.top + k] >= p.E) v = fmaf(p.wts[(size_t)t * p.top + k], to_f32(p.h[(size_t)t * p.d + col]), v);
        p.out[(size_t)t * p.d + col] = __float2bfloat16_rn(v);
      }
      __syncthreads();
      if (threadIdx.x == 0) B.piece = B.base;
      __syncthreads();
    }
    cp_wait(0);
  }
}

template <bool FP8, bool GLU>
__global__ void __launch_bounds__(LAYER_THREADS, 1) moe_layer_experts_kernel(LayerParams p) {
  bspec::pdl_prologue(85);
  extern __shared__ __align__(16) unsigned char smem[];
  __shared__ Block B;
  const int slots = p.n * p.top, tiles = (p.n + 7) / 8, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int T = tiles <= 1 ? 1 : (tiles <= 2 ? 2 : 8);           // sizes of the sums: as many column tiles as the tokens can fill
  Lists L;
  L.total = reinterpret_cast<float*>(smem);
  unsigned char* at = smem + (size_t)WARPS * 8 * T * 16 * 4;
  const uint32_t warp_ring = (uint32_t)p.stages * (A_BYTES + (uint32_t)p.ring_tiles * Ring<FP8>::B_PIECES * 512u);
  L.ring = smem_addr(at) + warp * warp_ring;
  at += (size_t)WARPS * warp_ring;
  L.slot = reinterpret_cast<int*>(at);
  L.active = L.slot + slots;
  L.first = L.active + p.E;
  L.count = L.first + p.E + 1;
  // the entries by expert: counted, placed (in any order within an expert: a column's sums do not depend on its place)
  for (int e = threadIdx.x; e < p.E; e += LAYER_THREADS) L.count[e] = 0;
  if (threadIdx.x == 0) B.done = B.stop = 0;
  __syncthreads();
  for (int s = threadIdx.x; s < slots; s += LAYER_THREADS) {
    const int e = p.ids[s];
    if (e < p.E) atomicAdd(L.count + e, 1);
  }
  __syncthreads();
  if (warp == 0) {
    int n_active = 0, run = 0, most = 0;
    for (int e0 = 0; e0 < p.E; e0 += 32) {
      const int e = e0 + lane, c = e < p.E ? L.count[e] : 0;
      int upto = c;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += v;
      }
      const unsigned mask = __ballot_sync(0xffffffffu, c > 0);
      const int at_a = n_active + __popc(mask & ((1u << lane) - 1u));
      if (c > 0) {
        L.active[at_a] = e;
        L.first[at_a] = run + upto - c;
        L.count[e] = run + upto - c;                              // where the next entry of this expert goes
      }
      most = max(most, c);
      n_active += __popc(mask);
      run += __shfl_sync(0xffffffffu, upto, 31);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) most = max(most, __shfl_xor_sync(0xffffffffu, most, o));
    if (lane == 0) {
      L.first[n_active] = run;
      B.n_active = n_active;
      B.most = most;
    }
  }
  __syncthreads();
  for (int s = threadIdx.x; s < slots; s += LAYER_THREADS) {
    const int e = p.ids[s];
    if (e < p.E) L.slot[atomicAdd(L.count + e, 1)] = s;
  }
  __syncthreads();
  if (T == 1) run_layer<FP8, GLU, 1>(p, L, B);
  else if (T == 2) run_layer<FP8, GLU, 2>(p, L, B);
  else run_layer<FP8, GLU, 8>(p, L, B);
}

template <bool FP8>
size_t layer_smem(int n, int E, int top, int* stages, int* ring_tiles) {
  const int tiles = (n + 7) / 8, T = tiles <= 1 ? 1 : (tiles <= 2 ? 2 : 8);
  const size_t fixed = (size_t)WARPS * 8 * T * 16 * 4 + ((size_t)n * top + 3 * (size_t)E + 1) * 4;
  // the tokens' numbers ride in the ring while two stages of it fit
  for (int rt = T < 8 ? T : 0;; rt = 0) {
    const size_t stage = (size_t)WARPS * (A_BYTES + rt * Ring<FP8>::B_PIECES * 512);
    const long long st = ((long long)SMEM_BUDGET - (long long)fixed) / (long long)stage;
    if (st >= 2 || rt == 0) {
      *ring_tiles = rt;
      *stages = st > 4 ? 4 : (int)st;
      return st < 2 ? 0 : fixed + (size_t)*stages * stage;
    }
  }
}

}  // namespace

// counters: 4 ints, ids [n top], wts [n top] and gate [n] floats: the results of the router and of its choice, and zeroed counters.
// rows: of the router, C = experts and identity experts, then perhaps one for the gate.
BSPEC_API int bspec_moe_layer_route(const void* h, int n, int d, const void* router, int rows, const void* corr, int corr_dtype, int C,
                                    int G, int keep, int top, float scale, int rule, int* ids, float* wts, float* gate, int* counters,
                                    cudaStream_t stream) {
  if (n <= 0) return 0;
  if (n > LAYER_TOKENS || d <= 0 || d % 8 != 0 || C <= 0 || C > MAX_EXPERTS || rows < C || rows > C + 1 || top <= 0 || top > C || G <= 0 || C % G ||
      keep <= 0 || keep > G || (long long)keep * (C / G) < top || (reinterpret_cast<uintptr_t>(h) & 15) ||
      (reinterpret_cast<uintptr_t>(router) & 15))
    return (int)cudaErrorInvalidValue;
  const int tiles = (rows + 15) / 16, steps = (d + 31) / 32;
  int slices = ROUTE_CLUSTER * ROUTE_WARPS / tiles;              // of k: as many as there are warps left
  if (slices > (steps + 3) / 4) slices = (steps + 3) / 4;        // at least one batch of loads each
  if (slices < 1) slices = 1;
  const size_t smem = ((size_t)tiles * slices * 16 * ROUTE_TOKENS + (size_t)ROUTE_WARPS * 3 * C) * 4;
  if (smem > 48 * 1024) {
    const cudaError_t e = cudaFuncSetAttribute(moe_layer_route_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 200 * 1024);
    if (e != cudaSuccess) return (int)e;
  }
  BSPEC_LAUNCH((moe_layer_route_kernel), ROUTE_CLUSTER * ((n + ROUTE_TOKENS - 1) / ROUTE_TOKENS), 32 * ROUTE_WARPS, smem, stream,
               (const __nv_bfloat16*)h, n, d, (const __nv_bfloat16*)router, rows, slices, corr, corr_dtype, C, G, keep, top, scale, rule,
               ids, wts, gate, counters);
  return BSPEC_LAUNCH_CHECK();
}

// The experts' products and the weighted sum, after bspec_moe_layer_route on the same stream.  su, sd: scales of the 128 x 128 blocks of
// e4m3 weights (float32, or 8-bit exponents with e8m0), null for bfloat16 weights.  u: [n top, ff] bfloat16 scratch.
BSPEC_API int bspec_moe_layer_experts(const void* h, int n, int d, const void* wu, const void* wd, const void* su, const void* sd, int e8m0,
                                      int E, int ff, int glu, const int* ids, const float* wts, int top, const float* gate, const void* add,
                                      void* u, void* out, int* counters, int* status, cudaStream_t stream) {
  if (n <= 0) return 0;
  const bool fp8 = su != nullptr;
  const int unit = fp8 ? 16 : 8;
  if (n > LAYER_TOKENS || d <= 0 || ff <= 0 || d % unit || ff % unit || E <= 0 || E > MAX_EXPERTS || top <= 0 || (fp8 && sd == nullptr) ||
      ((reinterpret_cast<uintptr_t>(h) | reinterpret_cast<uintptr_t>(wu) | reinterpret_cast<uintptr_t>(wd) | reinterpret_cast<uintptr_t>(u)) & 15))
    return (int)cudaErrorInvalidValue;
  LayerParams p = {};
  p.h = (const __nv_bfloat16*)h; p.wu = (const unsigned char*)wu; p.wd = (const unsigned char*)wd;
  p.su = su; p.sd = sd; p.e8m0 = e8m0; p.ids = ids; p.wts = wts; p.gate = gate; p.add = (const __nv_bfloat16*)add;
  p.u = (__nv_bfloat16*)u; p.out = (__nv_bfloat16*)out; p.counters = counters; p.status = status;
  p.n = n; p.d = d; p.ff = ff; p.E = E; p.top = top;
  const size_t smem = fp8 ? layer_smem<true>(n, E, top, &p.stages, &p.ring_tiles) : layer_smem<false>(n, E, top, &p.stages, &p.ring_tiles);
  if (smem == 0) return (int)cudaErrorInvalidValue;
#define LE(F, G)                                                                                                          \
  do {                                                                                                                    \
    static bool set_dev[bspec::kMaxDevices] = {};                                                                         \
    bool& set = set_dev[bspec::current_device()];                                                                         \
    if (!set) {                                                                                                           \
      const cudaError_t e = cudaFuncSetAttribute(moe_layer_experts_kernel<F, G>, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_BUDGET); \
      if (e != cudaSuccess) return (int)e;                                                                                \
      set = true;                                                                                                         \
    }                                                                                                                     \
    BSPEC_LAUNCH((moe_layer_experts_kernel<F, G>), bspec::sm_count(), LAYER_THREADS, smem, stream, p);                    \
  } while (0)
  if (fp8) { if (glu) LE(true, true); else LE(true, false); }
  else { if (glu) LE(false, true); else LE(false, false); }
#undef LE
  return BSPEC_LAUNCH_CHECK();
}

BSPEC_DEFINE_TRACE_SETTER(bspec_trace_set_moe_layer)
