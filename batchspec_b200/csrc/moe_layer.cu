// A whole routed feed-forward for a few tokens (at most 64) in two kernels:
//   z = Wr h,  (ids, w) = choice(z)                      the rules of moe_choose.cuh
//   u[t, k] = act(Wup[ids[t, k]] h[t])                   act: GELU, or silu(gate) * up with Wup = [gate; up]
//   out[t]  = add[t] * sigmoid(gate logit) + sum over k of w[t, k] * (Wdown[ids[t, k]] u[t, k], or h[t] for an identity expert)
// Experts in bfloat16, or in 8-bit floating point (e4m3) with a scale per 128 x 128 block; activations stay bfloat16 either
// way (u is rounded to bfloat16 between the products: it is the operand of a bfloat16 product), sums are float32.
//
// Bound by the read of the chosen experts' weights.  A weight is fetched once per 16 tokens of its expert, by bulk copies into a ring
// of its warp's own (several KB per warp are in flight, whatever the registers hold), and meets its tokens on mma.sync m16n8k16: the
// WEIGHT rows take the 16 rows of the product, the expert's tokens its columns, 8 at a time.  Both operands number the k of a step in
// the same permuted order (lane l % 4 holds neighbouring k), which a sum over k does not notice.
//
//   route    one cluster of 8 CTAs per 8 tokens: 64 warps share the router's rows and k, partial sums meet in the first CTA's
//            shared memory, whose warps choose for a token each.  It also clears the counters of the second kernel.
//   experts  one CTA per SM.  First all pieces of the up products are drawn from one counter, then pieces of 16 output columns
//            over all chosen experts.  A piece of the second kind waits until every piece of the first kind is done; those have
//            all been drawn by CTAs that run and wait for nothing, so it ends however many CTAs the device can hold.  A column's
//            sum runs over the experts in a fixed order: no atomic adds numbers.
#include "moe_choose.cuh"
#include "tma.cuh"
#include <math.h>

using namespace bspec;

namespace {

constexpr int LAYER_TOKENS = 64;             // most tokens of a step
constexpr int ROUTE_CLUSTER = 8, ROUTE_WARPS = 8, ROUTE_TOKENS = 8;
constexpr int WARPS = 16, LAYER_THREADS = 32 * WARPS;
constexpr int SMEM_BUDGET = 225 * 1024;

// ------------------------------------------------------------------------------------------------ the router
// z partials: [unit = (16 rows of the router, slice of k)][8 tokens][16 rows] in the first CTA of the cluster.
__global__ void __cluster_dims__(ROUTE_CLUSTER, 1, 1) __launch_bounds__(32 * ROUTE_WARPS)
moe_layer_route_kernel(const __nv_bfloat16* __restrict__ h, int n, int d, const __nv_bfloat16* __restrict__ wr, int rows, int slices,
                       const void* __restrict__ corr, int corr_dtype, int C, int G, int keep, int top, float scale, int rule,
                       int* __restrict__ ids, float* __restrict__ wts, float* __restrict__ gate, int* __restrict__ counters) {
  bspec::pdl_prologue(84);
  extern __shared__ float sm[];
  const int tiles = (rows + 15) / 16, units = tiles * slices;
  float* part = sm;                                            // [units][8][16]
  const int rank = blockIdx.x % ROUTE_CLUSTER, t0 = blockIdx.x / ROUTE_CLUSTER * ROUTE_TOKENS;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, q = lane & 3;
  if (blockIdx.x == 0 && threadIdx.x < 4) counters[threadIdx.x] = 0;
  // every CTA of the cluster runs before another one writes to its memory
  asm volatile("barrier.cluster.arrive.relaxed.aligned;\n\tbarrier.cluster.wait.aligned;" ::: "memory");
  uint32_t first;                                              // the first CTA's partials
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(first) : "r"(s32(part)), "r"(0));
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
      const int at = (unit * ROUTE_TOKENS + 2 * q + (i & 1)) * 16 + g + 8 * (i >> 1);
      asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(first + 4u * (uint32_t)at), "f"(acc[i]) : "memory");
    }
  }
  float* bias = part + (size_t)units * 16 * ROUTE_TOKENS;      // [C]
  if (rank == 0)
    for (int e = threadIdx.x; e < C; e += 32 * ROUTE_WARPS) bias[e] = corr != nullptr ? load_as_f32(corr, corr_dtype, e) : 0.f;
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
  const int t = t0 + warp;
  if (rank != 0 || t >= n) return;
  float* sc = bias + C + (size_t)warp * 3 * C;
  float* ch = sc + C;
  for (int e = lane; e < rows; e += 32) {
    const float* from = part + ((size_t)(e / 16 * slices) * ROUTE_TOKENS + warp) * 16 + e % 16;
    float z = 0.f;
#pragma unroll 8
    for (int s = 0; s < slices; ++s) z += from[s * ROUTE_TOKENS * 16];
    if (e < C) route_score(rule, z, bias[e], sc + e, ch + e);
    else gate[t] = z;                                          // the row behind the experts' rows
  }
  __syncwarp();
  choose_experts<true>(sc, ch, ch + C, corr != nullptr ? bias : nullptr, BSPEC_F32, C, G, keep, top, scale, rule, ids + (size_t)t * top, wts + (size_t)t * top);
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
  int stages;                                // of a warp's ring
};

__device__ __forceinline__ uint4 lds16(uint32_t at) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at) : "memory");
  return v;
}
__device__ __forceinline__ void copy_bulk(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
               ::"r"(dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
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

// A stage of a warp's ring: 256 bytes of each of 16 weight rows, fetched row by row by bulk copies.  Lanes 8 i .. 8 i + 7 read the rows
// 2 i and 2 i + 1 together, 64 bytes of each: an odd row begins 64 bytes further round the 128 bytes that the banks span.
constexpr int ROW_BYTES = 256, STAGE_BYTES = 8 * 576;
__device__ __forceinline__ uint32_t row_at(int r) { return (uint32_t)((r >> 1) * 576 + (r & 1) * 320); }
// k of a stage, and of a step of the products; tokens' numbers are read 128 k (a scale's block) at a time
template <bool FP8> struct Depth { static constexpr int ESZ = FP8 ? 1 : 2, STAGE = ROW_BYTES / ESZ, STEP = FP8 ? 64 : 32, STEPS = 128 / STEP; };

// What all pieces of a CTA know of the step, in shared memory.
struct Lists {
  int* active;                               // chosen experts, ascending; one with more than 16 tokens stands here once for every 16
  int* first;                                // [active + 1] where their entries begin
  int* slot;                                 // entries: (token, choice) numbers by expert
  int* count;                                // [E] scratch
  float* total;                              // this warp's sums [tokens][16 rows]; before that its partial tiles
};
struct Block {
  int drawn[WARPS];                          // a team's next piece
  int base, n_active, most, done, piece;
  int stop;                                  // a wait ran out
};
constexpr int MOST_COLUMNS = 16;             // tokens that meet a weight at a time
__host__ __device__ inline int most_active(int n, int E, int top) { return E + n * top / MOST_COLUMNS; }
// A warp's ring: `stages` slots; running slot and phase of the next stage to fill and to use.
struct Ring {
  uint32_t at, bars;
  uint64_t* bar;
  int stages, fill, use;
  uint32_t phase;
};

// Streams the stages [begin, begin + count) of the weight rows row_lo + 0 .. 7, row_hi + 0 .. 7 of the chosen experts, one expert's
// after the other's (`per` stages each), through this warp's ring, and multiplies them with the experts' tokens.  `done(a, acc)` is called
// when the last stage of expert a's share has been added to acc[column tile][4]; acc is cleared afterwards.  `ready()` is called when the
// first stages have been asked for and before any token is read, `ending()` before the last stage is waited for.
template <bool FP8, int T, bool DOWN, typename Ready, typename Ending, typename Done>
__device__ __forceinline__ void stream(const LayerParams& p, const Lists& L, Block& B, Ring& R, int begin, int count, int per, int row_lo,
                                       int row_hi, int rows_all, int K, Ready ready, Ending ending, Done done) {
  using D = Depth<FP8>;
  const int lane = threadIdx.x & 31, g = lane >> 2, q = lane & 3;
  const __nv_bfloat16* const tokens = DOWN ? p.u : p.h;
  const int KB = (K + 127) / 128, RB = (rows_all + 127) / 128;
  const uint32_t row_bytes = (uint32_t)K * D::ESZ;

  // filling: lane r copies row r; a running source, set anew where the next expert begins
  const int my_row = lane < 8 ? row_lo + lane : row_hi + (lane & 7);
  const bool copies = lane < 16 && my_row < rows_all;
  const uint32_t n_copies = __popc(__ballot_sync(0xffffffffu, copies));
  const uint32_t last_bytes = row_bytes - (uint32_t)(per - 1) * ROW_BYTES, my_slot = R.at + row_at(lane);
  int a = begin / per, s = begin - a * per, fa = a, f_left = per - s, to_fill = count;
  const unsigned char* src = nullptr;
  auto open = [&](int from) { src = (DOWN ? p.wd : p.wu) + ((size_t)L.active[fa] * rows_all + my_row) * row_bytes + (size_t)from * ROW_BYTES; };
  auto fill = [&]() {
    if (to_fill == 0) return;
    const uint32_t bytes = f_left == 1 ? last_bytes : (uint32_t)ROW_BYTES, bar = R.bars + 8u * R.fill;
    if (lane == 0) asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes * n_copies) : "memory");
    if (copies) copy_bulk(my_slot + (uint32_t)R.fill * STAGE_BYTES, src, bytes, bar);
    if (++R.fill == R.stages) R.fill = 0;
    src += ROW_BYTES;
    --to_fill;
    if (--f_left == 0 && to_fill > 0) {
      ++fa;
      f_left = per;
      open(0);
    }
  };
  // the tokens' numbers: a cursor of its own, one block of 128 k ahead of the products; a column without a token reads its neighbour's
  constexpr int Q_STEP = FP8 ? 16 : 8;
  uint4 b[T][4];
  const __nv_bfloat16* from[T];
  int tiles = 0;                              // column tiles of the expert that the cursor is in
  auto enter = [&](int at, int k) {
    const int c0 = L.first[at], cnt = L.first[at + 1] - c0;
    tiles = (cnt + 7) >> 3;
#pragma unroll
    for (int t = 0; t < T; ++t) {
      const int slot = L.slot[c0 + min(8 * t + g, cnt - 1)];
      from[t] = tokens + (size_t)(DOWN ? slot : slot / p.top) * K + k + Q_STEP * q;
    }
  };
  // piece i of a block: bfloat16 weights meet k 32 i + 8 q, 8-bit ones 64 (i / 2) + 16 q + 8 (i % 2); `left` k to the rows' ends
  auto fetch = [&](int i, int left) {
    const int off = FP8 ? 64 * (i >> 1) + 8 * (i & 1) : 32 * i;
    const bool in = off + Q_STEP * q < left;
#pragma unroll
    for (int t = 0; t < T; ++t)
      if (t < tiles) {
        const uint4* at = reinterpret_cast<const uint4*>(from[t] + off);
        b[t][i] = !in ? make_uint4(0u, 0u, 0u, 0u) : (DOWN ? __ldcg(at) : __ldg(at));
      }
  };
  float acc[T][4];
#pragma unroll
  for (int t = 0; t < T; ++t)
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[t][i] = 0.f;

  if (count > 0) open(s);
  for (int i = 0; i < R.stages; ++i) fill();
  ready();
  if (count > 0) {
    enter(a, s * D::STAGE);
#pragma unroll
    for (int i = 0; i < 4; ++i) fetch(i, K - s * D::STAGE);
  }
  int nt = tiles;                             // ... and of the expert of the products
  size_t scale_lo = 0, scale_hi = 0;
  auto scales_of = [&](int at) {
    scale_lo = ((size_t)L.active[at] * RB + min(row_lo + g, rows_all - 1) / 128) * KB;
    scale_hi = ((size_t)L.active[at] * RB + min(row_hi + g, rows_all - 1) / 128) * KB;
  };
  if (FP8 && count > 0) scales_of(a);
  bool ok = B.stop == 0;
#pragma unroll 1
  for (int j = 0; j < count; ++j) {
    const bool last_stage = s + 1 == per, more = j + 1 < count;
    if (!more) ending();
    if (ok) ok = mbar_wait(R.bar + R.use, R.phase, &B.stop, p.status, 112);
    if (!ok) to_fill = 0;
    const uint32_t at = R.at + (uint32_t)R.use * STAGE_BYTES + row_at(g) + 16u * q;
    if (++R.use == R.stages) { R.use = 0; R.phase ^= 1u; }
#pragma unroll
    for (int blk = 0; blk < D::STAGE / 128; ++blk) {
      const int left = K - s * D::STAGE - 128 * blk;      // k from this block to the rows' ends
      if (blk > 0 && left <= 0) break;
      float s_lo = 1.f, s_hi = 1.f;
      if (FP8) {
        const int kb = s * (D::STAGE / 128) + blk;
        s_lo = block_scale(DOWN ? p.sd : p.su, p.e8m0, scale_lo + kb);
        s_hi = block_scale(DOWN ? p.sd : p.su, p.e8m0, scale_hi + kb);
      }
      // the next block's tokens; each piece is asked for when the one before it in its registers has been used
      int next_left = 0;
      if (left > 128 && (blk + 1 < D::STAGE / 128 || more)) {
        next_left = left - 128;
#pragma unroll
        for (int t = 0; t < T; ++t) from[t] += 128;
      } else if (left <= 128 && more) {
        next_left = K;
        enter(a + 1, 0);
      }
      float sum[FP8 ? T : 1][4];
      if (FP8) {
#pragma unroll
        for (int t = 0; t < T; ++t)
#pragma unroll
          for (int i = 0; i < 4; ++i) sum[t][i] = 0.f;
      }
#pragma unroll
      for (int st = 0; st < D::STEPS; ++st) {
        const uint32_t off = (uint32_t)(blk * D::STEPS + st) * 64u;
        uint4 lo = lds16(at + off), hi = lds16(at + off + 4 * 576);
        if (left < 128 && st * D::STEP + (16 / D::ESZ) * q >= left) lo = hi = make_uint4(0u, 0u, 0u, 0u);   // what an earlier stage left
        if (FP8) {
          const uint32_t l[4] = {lo.x, lo.y, lo.z, lo.w}, h[4] = {hi.x, hi.y, hi.z, hi.w};
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            uint32_t wl[4], wh[4];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              widen4(l[2 * half + i], wl[2 * i], wl[2 * i + 1]);
              widen4(h[2 * half + i], wh[2 * i], wh[2 * i + 1]);
            }
#pragma unroll
            for (int t = 0; t < T; ++t)
              if (t < nt) {
                const uint4 x = b[t][2 * st + half];
                mma_bf16_16816(sum[t], wl[0], wh[0], wl[1], wh[1], x.x, x.y);
                mma_bf16_16816(sum[t], wl[2], wh[2], wl[3], wh[3], x.z, x.w);
              }
          }
        } else {
#pragma unroll
          for (int t = 0; t < T; ++t)
            if (t < nt) {
              const uint4 x = b[t][st];
              mma_bf16_16816(acc[t], lo.x, hi.x, lo.y, hi.y, x.x, x.y);
              mma_bf16_16816(acc[t], lo.z, hi.z, lo.w, hi.w, x.z, x.w);
            }
        }
        if (next_left > 0) {
#pragma unroll
          for (int i = 0; i < 4 / D::STEPS; ++i) fetch(4 / D::STEPS * st + i, next_left);
        }
      }
      if (FP8) {
#pragma unroll
        for (int t = 0; t < T; ++t) {
          acc[t][0] = fmaf(sum[t][0], s_lo, acc[t][0]);
          acc[t][1] = fmaf(sum[t][1], s_lo, acc[t][1]);
          acc[t][2] = fmaf(sum[t][2], s_hi, acc[t][2]);
          acc[t][3] = fmaf(sum[t][3], s_hi, acc[t][3]);
        }
      }
    }
    __syncwarp();                             // every lane has read the stage
    fill();
    if (last_stage || !more) {
      done(a, acc);
#pragma unroll
      for (int t = 0; t < T; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[t][i] = 0.f;
      nt = tiles;
      s = -1;
      ++a;
      if (FP8 && more) scales_of(a);
    }
    ++s;
  }
}

template <bool FP8, bool GLU, int T>
__device__ __forceinline__ void run_layer(const LayerParams& p, const Lists& L, Block& B, Ring& R) {
  using D = Depth<FP8>;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, q = lane & 3;
  const int A = B.n_active, ffu = GLU ? 2 * p.ff : p.ff, warp_total = (p.n + 7) / 8 * 128;

  // ---- up products: a piece is 16 rows of one expert (GLU: 8 gate rows and their 8 up rows), shared by the warps of a team
  constexpr int OUT = GLU ? 8 : 16;
  const int tiles = (p.ff + OUT - 1) / OUT, pieces = A * tiles, depth = (p.d + D::STAGE - 1) / D::STAGE;
  // a team of 2 or 4 warps cuts a piece's k, as long as each has four stages: short pieces end at about the same time everywhere
  const int team_size = depth >= 16 ? 4 : (depth >= 8 ? 2 : 1);
  const int team = warp / team_size, member = warp % team_size;
  const int per = (depth + team_size - 1) / team_size, from = min(depth, member * per), to = min(depth, from + per);
  if (threadIdx.x == 0) B.base = atomicAdd(p.counters, WARPS / team_size);
  __syncthreads();
  int piece = B.base + team, mine = 0;
  while (piece < pieces) {
    int next = 0;
    const int a = piece / tiles, i0 = (piece - a * tiles) * OUT, c0 = L.first[a], cnt = L.first[a + 1] - c0, nt = (cnt + 7) / 8;
    float part[T][4];
#pragma unroll
    for (int t = 0; t < T; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) part[t][i] = 0.f;
    stream<FP8, T, false>(p, L, B, R, a * depth + from, to - from, depth, i0, GLU ? p.ff + i0 : i0 + 8, ffu, p.d, []() {},
                          [&]() {             // not earlier: a CTA that starts first would take the others' first pieces
                            if (member == 0 && lane == 0) next = atomicAdd(p.counters, 1);
                          },
                          [&](int, float (&acc)[T][4]) {
#pragma unroll
                            for (int t = 0; t < T; ++t)
#pragma unroll
                              for (int i = 0; i < 4; ++i) part[t][i] = acc[t][i];
                          });
    if (team_size > 1) {
      if (member != 0) {
#pragma unroll
        for (int t = 0; t < T; ++t)
          if (t < nt) {
#pragma unroll
            for (int i = 0; i < 4; ++i) L.total[(t * 4 + i) * 32 + lane] = part[t][i];
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
              for (int i = 0; i < 4; ++i) part[t][i] += L.total[m * warp_total + (t * 4 + i) * 32 + lane];
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
            const float gv = part[t][i];
            if (i0 + g < p.ff) *u = __float2bfloat16_rn(gv / (1.f + expf(-gv)) * part[t][2 + i]);
          } else {
            if (i0 + g < p.ff) u[0] = __float2bfloat16_rn(gelu_erf(part[t][i]));
            if (i0 + 8 + g < p.ff) u[8] = __float2bfloat16_rn(gelu_erf(part[t][2 + i]));
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
  const int out_pieces = (p.d + 15) / 16, per_expert = (p.ff + D::STAGE - 1) / D::STAGE;
  const int all = A * per_expert, w0 = (int)((long long)all * warp / WARPS), w1 = (int)((long long)all * (warp + 1) / WARPS);
  bool waited = false;
  auto up_done = [&]() {                      // every up piece of every CTA is done
    if (waited) return;
    waited = true;
    if (threadIdx.x == 0) {
      unsigned long long t_from = 0ull;
      for (uint32_t i = 0; !B.stop; ++i) {
        int v;
        asm volatile("ld.acquire.gpu.global.s32 %0, [%1];" : "=r"(v) : "l"(p.counters + 1) : "memory");
        if (v >= pieces) break;
        if ((i & 255u) == 255u) {
          const unsigned long long now = bspec::global_timer();
          if (t_from == 0ull) t_from = now;
          if (now - t_from > WAIT_NS || i >= WAIT_LIMIT || *reinterpret_cast<volatile int*>(p.status) != 0) {
            atomicCAS(p.status, 0, 111);
            B.stop = 1;
          }
        }
      }
      __threadfence();
    }
    __syncthreads();
  };
  while (B.piece < out_pieces) {
    const int n0 = B.piece * 16;
    for (int i = lane; i < p.n * 16; i += 32) L.total[i] = 0.f;
    __syncwarp();
    stream<FP8, T, true>(p, L, B, R, w0, w1 - w0, per_expert, n0, n0 + 8, p.d, p.ff, up_done, []() {}, [&](int a, float (&acc)[T][4]) {
      const int c0 = L.first[a], cnt = L.first[a + 1] - c0;
#pragma unroll
      for (int t = 0; t < T; ++t)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int c = 8 * t + 2 * q + i;
          if (c >= cnt) continue;
          const int slot = L.slot[c0 + c];
          const float w = p.wts[slot];
          float* to = L.total + slot / p.top * 16 + g;
          to[0] = fmaf(w, acc[t][i], to[0]);
          to[8] = fmaf(w, acc[t][2 + i], to[8]);
        }
      __syncwarp();
    });
    __syncthreads();
    if (threadIdx.x == 0) B.base = atomicAdd(p.counters + 2, 1);
    const float* totals = L.total - warp * warp_total;
    if (!B.stop)
      for (int i = threadIdx.x; i < p.n * 16; i += LAYER_THREADS) {
        const int t = i >> 4, col = n0 + (i & 15);
        if (col >= p.d) continue;
        float v = 0.f;
        if (p.add != nullptr) {
          v = to_f32(p.add[(size_t)t * p.d + col]);
          if (p.gate != nullptr) v *= 1.f / (1.f + expf(-p.gate[t]));
        }
#pragma unroll
        for (int w = 0; w < WARPS; ++w) v += totals[w * warp_total + i];
        for (int k = 0; k < p.top; ++k)
          if (p.ids[(size_t)t * p.top + k] >= p.E) v = fmaf(p.wts[(size_t)t * p.top + k], to_f32(p.h[(size_t)t * p.d + col]), v);
        p.out[(size_t)t * p.d + col] = __float2bfloat16_rn(v);
      }
    __syncthreads();
    if (threadIdx.x == 0) B.piece = B.base;
    __syncthreads();
  }
  // after a wait that ran out: copies in flight land (they take microseconds) before the shared memory is given up
  if (B.stop)
    for (int i = 0; i < 1000; ++i) __nanosleep(1000);
}

// bytes of shared memory for the sums, the rings and the lists; a CTA's static shared memory comes on top
__host__ __device__ inline size_t layer_smem(int n, int E, int top, int stages) {
  return (size_t)WARPS * ((n + 7) / 8 * 128 * 4 + stages * STAGE_BYTES) + ((size_t)n * top + 2 * (size_t)most_active(n, E, top) + 1 + E) * 4;
}
constexpr int MAX_STAGES = 4;

template <bool FP8, bool GLU>
__global__ void __launch_bounds__(LAYER_THREADS, 1) moe_layer_experts_kernel(LayerParams p) {
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ Block B;
  __shared__ uint64_t bars[WARPS * MAX_STAGES];
  const int slots = p.n * p.top, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (threadIdx.x < WARPS * MAX_STAGES) mbar_init(bars + threadIdx.x, 1);
  if (threadIdx.x == 0) B.done = B.stop = 0;
  asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  Lists L;
  Ring R;
  R.at = s32(smem) + (uint32_t)(warp * p.stages) * STAGE_BYTES;
  R.bar = bars + warp * MAX_STAGES;
  R.bars = s32(R.bar);
  R.stages = p.stages;
  R.fill = R.use = 0;
  R.phase = 0u;
  unsigned char* at = smem + (size_t)WARPS * p.stages * STAGE_BYTES;
  L.total = reinterpret_cast<float*>(at) + (size_t)warp * ((p.n + 7) / 8 * 128);
  at += (size_t)WARPS * ((p.n + 7) / 8 * 128) * 4;
  L.slot = reinterpret_cast<int*>(at);
  L.active = L.slot + slots;
  L.first = L.active + most_active(p.n, p.E, p.top);
  L.count = L.first + most_active(p.n, p.E, p.top) + 1;
  for (int e = threadIdx.x; e < p.E; e += LAYER_THREADS) L.count[e] = 0;
  __syncthreads();
  bspec::pdl_prologue(85);
  // the entries by expert: counted, then placed
  for (int s = threadIdx.x; s < slots; s += LAYER_THREADS) {
    const int e = p.ids[s];
    if (e < p.E) atomicAdd(L.count + e, 1);
  }
  __syncthreads();
  if (warp == 0) {
    int n_active = 0, run = 0, most = 0;
    for (int e0 = 0; e0 < p.E; e0 += 32) {
      const int e = e0 + lane, c = e < p.E ? L.count[e] : 0, groups = (c + MOST_COLUMNS - 1) / MOST_COLUMNS;
      int upto = c, upto_g = groups;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, upto, o), w = __shfl_up_sync(0xffffffffu, upto_g, o);
        if (lane >= o) upto += v, upto_g += w;
      }
      const int from = run + upto - c;
      for (int i = 0; i < groups; ++i) {
        L.active[n_active + upto_g - groups + i] = e;
        L.first[n_active + upto_g - groups + i] = from + i * MOST_COLUMNS;
      }
      if (c > 0) L.count[e] = from;                               // where the next entry of this expert goes
      most = max(most, c);
      n_active += __shfl_sync(0xffffffffu, upto_g, 31);
      run += __shfl_sync(0xffffffffu, upto, 31);
    }
    most = __reduce_max_sync(0xffffffffu, most);
    if (lane == 0) {
      L.first[n_active] = run;
      B.n_active = n_active;
      B.most = most;
    }
    __syncwarp();
    // placed in the order of their numbers, so that every CTA has the same ones in an expert's first 16
    for (int s0 = 0; s0 < slots; s0 += 32) {
      const int s = s0 + lane, e = s < slots ? p.ids[s] : p.E;
      const unsigned same = __match_any_sync(0xffffffffu, e);
      if (e < p.E) {
        const int from = L.count[e];
        L.slot[from + __popc(same & ((1u << lane) - 1u))] = s;
        __syncwarp(same);
        if (lane == __ffs(same) - 1) L.count[e] = from + __popc(same);
      }
      __syncwarp();
    }
  }
  __syncthreads();
  if (B.most <= 8) run_layer<FP8, GLU, 1>(p, L, B, R);
  else run_layer<FP8, GLU, 2>(p, L, B, R);
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
  const size_t smem = ((size_t)tiles * slices * 16 * ROUTE_TOKENS + (size_t)(ROUTE_WARPS * 3 + 1) * C) * 4;
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
  p.stages = 2;
  while (p.stages < MAX_STAGES && layer_smem(n, E, top, p.stages + 1) <= SMEM_BUDGET) ++p.stages;
  const size_t smem = layer_smem(n, E, top, p.stages);
  if (smem > SMEM_BUDGET) return (int)cudaErrorInvalidValue;
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
