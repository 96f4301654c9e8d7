// Matrix product in 8-bit floating point (e4m3) with a scale for each block of 128, on the 5th-generation tensor cores:
//   C[m, n] = sum over blocks b of 128 k:  xs[m, b] * ws[n / 128, b] * sum over k in b of X[m, k] * W[n, k]
// X [M, K] has a scale per row and block, W [N, K] one per 128 x 128; scales are float32 numbers or powers of two in 8 bits (e8m0).
//
// The products of one block are sums of the tensor core (tcgen05.mma kind::f8f6f4, float32 accumulator in tensor memory); the
// scales differ from block to block, so every block of 128 k gets an accumulator of its own (a ring of them in tensor memory), and
// the epilogue warps read it back, multiply by its scales and add it to float32 sums in registers while the next blocks' products
// run.  The sum over blocks is in ascending k.  Where the product of the two scales alone would leave float32's range, a sum meets them in two factors
// with half of the exponent each, so that small results keep their bits and zeros stay zeros.
//
// Three arrangements, chosen by an estimate of their times (`choose`):
//   few tokens    rows of W on the accumulator's 128 rows, tokens on its columns: every weight is streamed once at full tile efficiency.  K
//                 may be cut into `splits` slices run by the CTAs of one cluster, whose partial tiles are joined in slice order through
//                 distributed shared memory.
//   many tokens   tokens on the rows, 128 rows of W on the columns: one persistent CTA per SM; eight epilogue warps hold the 128 x 128 sums.
//                 What bounds it: a tile asks for 32 KB per 128 k, 512 of the clocks that the L2 (64 bytes a clock) and shared memory have; the
//                 additions are a tenth of the time.  Tiles 192 wide, two CTAs per SM, and pairs of CTAs with rows of W on the accumulator's rows
//                 (whose columns' scales have to be read for every block: 184 us for 118) came no nearer.
//   pairs         many tokens where both scales are powers of two: the tensor cores multiply by the scales and keep the sums of a whole
//                 row, two CTAs share a tile (below).
//
// Measured on B200: 8 x 28,672 x 4,096 in 20.1 us (5.9 TB/s), 61 x 32,000 x 2,048 into float32 in 18.7 us (3.9 TB/s), 1,537 x 4,096 x 14,336 with
// float32 scales in 115 us (1.6 PFLOP/s), 2,048 x 28,672 x 4,096 with e8m0 scales in 177 us (2.7 PFLOP/s; 190 and more once the power limit holds;
// all zeros, which it does not slow down, run at 4.1), into float32 in 229 us.
#include "e4m3.cuh"
#include "umma.cuh"
#include <type_traits>

using namespace bspec;

namespace {

constexpr int KBYTES = 128;            // k per stage: one scale block, one 128-byte swizzle span
constexpr int TILE_ROWS = 128;
constexpr int FEW_THREADS = 192;       // TMA warp, MMA warp, 4 epilogue warps
constexpr int FEW_WINDOW = 16;         // k blocks whose scales wait in shared memory at a time
constexpr int MANY_THREADS = 320;      // TMA warp, MMA warp, 8 epilogue warps
constexpr int MANY_BN = 128, MANY_STAGES = 6;

struct Scales {
  const void* p;
  long long ld;          // from row to row of scales
  int e8m0;              // 1: exponents in 8 bits, 0: float32
};
__device__ __forceinline__ float scale_at(const Scales& s, long long row, int kb) {
  const long long i = row * s.ld + kb;
  return s.e8m0 ? scale_value(reinterpret_cast<const uint8_t*>(s.p)[i]) : reinterpret_cast<const float*>(s.p)[i];
}

struct Fp8Params {
  void* C;               // [M, N]
  int* status;
  Scales xs, ws;
  int M, N, K;
  int out_f32;
  int splits, kblocks_per_split, stages;      // few tokens
  int w_ahead;           // W and its scales may be read before the kernel before this one has ended
  int tiles_m, tiles_n;  // many tokens
};

__device__ __forceinline__ void put(void* C, int out_f32, size_t at, float v) {
  if (out_f32) reinterpret_cast<float*>(C)[at] = v;
  else reinterpret_cast<__nv_bfloat16*>(C)[at] = __float2bfloat16_rn(v);
}
// 16 neighbours in stores of 32 bytes: whole sectors, where stores of 16 bytes would be partial ones.  `to` on a 32-byte boundary.
__device__ __forceinline__ void put32b(void* to, const uint32_t* w) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};"
               ::"l"(to), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7]) : "memory");
}
__device__ __forceinline__ void put16(void* C, int out_f32, size_t at, const float* v) {
  if (out_f32) {
    put32b(reinterpret_cast<float*>(C) + at, reinterpret_cast<const uint32_t*>(v));
    put32b(reinterpret_cast<float*>(C) + at + 8, reinterpret_cast<const uint32_t*>(v + 8));
    return;
  }
  uint32_t w[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * j], v[2 * j + 1]);
    w[j] = *reinterpret_cast<uint32_t*>(&h);
  }
  put32b(reinterpret_cast<__nv_bfloat16*>(C) + at, w);
}
// Let copies in flight land before the CTA gives up its shared memory (after a wait ran out).
__device__ __forceinline__ void drain(uint64_t* full, int armed, int stages) {
  for (int i = max(0, armed - stages); i < armed; ++i) {
    const uint32_t ph = (uint32_t)(i / stages) & 1u;
    for (uint32_t t = 0; t < (1u << 16) && !mbar_try_wait(full + i % stages, ph); ++t) __nanosleep(32);
  }
}

// ------------------------------------------------------------------------------------------------ few tokens
constexpr int FEW_BUFFERS = 4;         // accumulators: two CTAs of an SM share 512 columns

template <int BN>
__global__ void __launch_bounds__(FEW_THREADS)
gemm_fp8_few_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x, Fp8Params p) {
  constexpr int NB = FEW_BUFFERS;
  constexpr uint32_t COLS = NB * BN;                                   // 64, 128 or 256: powers of two
  constexpr int W_BYTES = TILE_ROWS * KBYTES, X_BYTES = BN * KBYTES, STAGE = W_BYTES + X_BYTES;
  extern __shared__ unsigned char smem_dyn[];
  unsigned char* smem = reinterpret_cast<unsigned char*>(((uintptr_t)smem_dyn + 1023) & ~(uintptr_t)1023);
  float* scales = reinterpret_cast<float*>(smem + (size_t)p.stages * STAGE);      // [FEW_WINDOW][BN], xs * ws; and again, what a sum meets before it
  uint64_t* full = reinterpret_cast<uint64_t*>(scales + 2 * FEW_WINDOW * BN);
  uint64_t* empty = full + p.stages;
  uint64_t* acc_full = empty + p.stages;
  uint64_t* acc_empty = acc_full + NB;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_empty + NB);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  float* part = reinterpret_cast<float*>(smem);                        // [BN][128] sums of this K slice, over the stages

  const unsigned long long t_trace = bspec::g_trace_buf != nullptr ? bspec::global_timer() : 0ull;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int tile_n = blockIdx.x, tok0 = blockIdx.y * BN, split = blockIdx.z;
  const int kb_total = (p.K + KBYTES - 1) / KBYTES;
  const int kb0 = split * p.kblocks_per_split;
  const int nkb = min(p.kblocks_per_split, kb_total - kb0);

  if (threadIdx.x == 0) {
    for (int s = 0; s < p.stages; ++s) {
      mbar_init(full + s, 1);
      mbar_init(empty + s, 1);
    }
    for (int b = 0; b < NB; ++b) {
      mbar_init(acc_full + b, 1);
      mbar_init(acc_empty + b, 4);
    }
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(s32(tmem_slot)), "r"(COLS) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  // Not before this CTA holds its tensor memory: that is a wait without a limit, and a CTA of the next kernel that took the columns first would keep
  // them until this kernel has ended.  (Three CTAs of 256 columns fit an SM where K is short.)
  bspec::pdl_launch_dependents();

  float acc[BN];
#pragma unroll
  for (int c = 0; c < BN; ++c) acc[c] = 0.f;

  if (warp == 0) {
    const uint32_t one = elect_one();
    int armed = 0;
    if (!p.w_ahead) bspec::pdl_wait();
    const int pre = min(nkb, p.stages);
    for (int i = 0; i < pre; ++i) {
      mbar_expect_tx_by(one, full + i, (uint32_t)STAGE);
      tma_load_2d_by(one, smem + (size_t)i * STAGE, &map_w, full + i, (kb0 + i) * KBYTES, tile_n * TILE_ROWS);
    }
    bspec::pdl_wait();
    bspec::trace_record(82, t_trace);
    for (int i = 0; i < pre; ++i)
      tma_load_2d_by(one, smem + (size_t)i * STAGE + W_BYTES, &map_x, full + i, (kb0 + i) * KBYTES, tok0);
    armed = pre;
    int s = 0;
    uint32_t phase = 0u;
    for (int i = pre; i < nkb; ++i) {
      if (!warp_wait(empty + s, phase, abort_flag, p.status, 101)) break;
      mbar_expect_tx_by(one, full + s, (uint32_t)STAGE);
      tma_load_2d_by(one, smem + (size_t)s * STAGE, &map_w, full + s, (kb0 + i) * KBYTES, tile_n * TILE_ROWS);
      tma_load_2d_by(one, smem + (size_t)s * STAGE + W_BYTES, &map_x, full + s, (kb0 + i) * KBYTES, tok0);
      armed = i + 1;
      if (++s == p.stages) { s = 0; phase ^= 1u; }
    }
    if (*abort_flag) drain(full, armed, p.stages);
  } else if (warp == 1) {
    const uint32_t one = elect_one();
    const uint32_t idesc = instr_desc_e4m3(BN);
    const uint64_t desc0 = smem_desc(smem);
    int s = 0, b = 0;
    uint32_t phase = 0u, acc_phase = 0u;
    for (int i = 0; i < nkb; ++i) {
      if (!warp_wait(full + s, phase, abort_flag, p.status, 102)) break;
      if (!warp_wait(acc_empty + b, acc_phase ^ 1u, abort_flag, p.status, 103)) break;
      tc_fence_after();
      const uint64_t wd = desc0 + (uint64_t)(s * (STAGE / 16)), xd = wd + W_BYTES / 16;      // addresses count 16 bytes
#pragma unroll
      for (int k = 0; k < KBYTES / 32; ++k) tc_mma_8bit_by(one, tmem_base + b * BN, wd + 2 * k, xd + 2 * k, idesc, k > 0 ? 1u : 0u);
      tc_commit_by(one, empty + s);
      tc_commit_by(one, acc_full + b);
      if (++s == p.stages) { s = 0; phase ^= 1u; }
      if (++b == NB) { b = 0; acc_phase ^= 1u; }
    }
  } else {
    const uint32_t quad = warp & 3;
    const int et = threadIdx.x - 64;                                   // 0 .. 127
    bspec::pdl_wait();
    bool ok = true;
    // whether it holds for any epilogue thread; they meet here
    auto any_of = [](bool mine) {
      uint32_t any;
      asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbarrier.cta.red.or.pred q, 1, 128, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
                   : "=r"(any) : "r"((uint32_t)mine) : "memory");
      return any != 0u;
    };
    int b = 0;
    uint32_t phase = 0u;
    for (int i0 = 0; i0 < nkb; i0 += FEW_WINDOW) {
      // the scales of the next blocks; every epilogue thread comes here, whatever its waits said
      const int nw = min(FEW_WINDOW, nkb - i0);
      asm volatile("bar.sync 1, 128;" ::: "memory");
      bool unusual = false;
      for (int j = et; j < nw * BN; j += 128) {
        const int c = j / nw, k = j - c * nw, tok = tok0 + c;          // neighbours read neighbouring blocks of a token
        const float f = tok < p.M ? scale_at(p.xs, tok, kb0 + i0 + k) * scale_at(p.ws, tile_n, kb0 + i0 + k) : 0.f;
        unusual |= tok < p.M && !is_ordinary(f);
        scales[k * BN + c] = f;
      }
      const bool apart = any_of(unusual);
      if (apart) {
        for (int j = et; j < nw * BN; j += 128) {
          const int c = j / nw, k = j - c * nw, tok = tok0 + c;
          float f = scales[k * BN + c], before = 1.f;
          if (tok < p.M) {
            const float x = scale_at(p.xs, tok, kb0 + i0 + k), w = scale_at(p.ws, tile_n, kb0 + i0 + k);
            if (leaves_range(x, w, f)) split_scales(x, w, before, f);
          }
          scales[k * BN + c] = f;
          scales[(FEW_WINDOW + k) * BN + c] = before;
        }
        asm volatile("bar.sync 1, 128;" ::: "memory");
      }
      auto block = [&](int i, auto in_two) {
        ok = warp_wait(acc_full + b, phase, abort_flag, p.status, 104);
        if (!ok) return;
        tc_fence_after();
        const float4* f = reinterpret_cast<const float4*>(scales + i * BN);
        const uint32_t from = tmem_base + ((quad * 32u) << 16) + (uint32_t)(b * BN);
        // an accumulator is read in one trip, and is free for the next products before its numbers are added
        uint32_t v[BN];
        if constexpr (BN == 16) tc_ld16(from, v);
        else if constexpr (BN == 32) tc_ld32(from, v);
        else tc_ld64(from, v);
        tc_wait_ld();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(acc_empty + b);             // one arrival per warp: those of its lanes would come one after the other
        if (++b == NB) { b = 0; phase ^= 1u; }
        if constexpr (decltype(in_two)::value) {
#pragma unroll
          for (int c = 0; c < BN; ++c) v[c] = __float_as_uint(__uint_as_float(v[c]) * reinterpret_cast<const float*>(f)[FEW_WINDOW * BN + c]);
        }
#pragma unroll
        for (int c = 0; c < BN; c += 4) {
          const float4 g = f[c / 4];
          acc[c] = fmaf(__uint_as_float(v[c]), g.x, acc[c]);
          acc[c + 1] = fmaf(__uint_as_float(v[c + 1]), g.y, acc[c + 1]);
          acc[c + 2] = fmaf(__uint_as_float(v[c + 2]), g.z, acc[c + 2]);
          acc[c + 3] = fmaf(__uint_as_float(v[c + 3]), g.w, acc[c + 3]);
        }
      };
      // two loops, so that the ordinary one is no longer for the other's sake (61 x 32,000 x 2,048: 18.7 us, with a branch in one loop 19.3)
      if (!apart) {
        for (int i = 0; i < nw && ok; ++i) block(i, std::false_type{});
      } else {
        for (int i = 0; i < nw && ok; ++i) block(i, std::true_type{});
      }
    }
    // every product of this slice has completed and every stage has been read: the sums take their place, where few instructions, the same for
    // each token, find them (what is executed once costs the fetch of its code more than its work)
    const int row = (int)quad * 32 + lane, n = tile_n * TILE_ROWS + row;
#pragma unroll
    for (int c = 0; c < BN; ++c) part[c * TILE_ROWS + row] = acc[c];
    if (p.splits == 1 && ok && n < p.N) {
      const int some = min(BN, p.M - tok0);
      size_t at = (size_t)tok0 * p.N + n;
#pragma unroll 4
      for (int c = 0; c < some; ++c, at += p.N) put(p.C, p.out_f32, at, part[c * TILE_ROWS + row]);
    }
  }
  if (p.splits > 1) {
    __syncthreads();
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
    if (warp >= 2 && !*abort_flag) {
      const int row = (warp & 3) * 32 + lane, n = tile_n * TILE_ROWS + row;
      if (n < p.N) {
        uint32_t peer[8];
        const uint32_t mine = s32(part + row);
#pragma unroll
        for (int s = 0; s < 8; ++s)
          if (s < p.splits) asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(peer[s]) : "r"(mine), "r"(s));
        for (int c0 = split; c0 < BN; c0 += 4 * p.splits) {             // four tokens' loads in flight at a time
          float v[4][8];
#pragma unroll
          for (int t = 0; t < 4; ++t) {
            const int c = c0 + t * p.splits;
            if (c < BN && tok0 + c < p.M) {
#pragma unroll
              for (int s = 0; s < 8; ++s)
                if (s < p.splits)
                  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v[t][s]) : "r"(peer[s] + (uint32_t)c * TILE_ROWS * 4u));
            }
          }
#pragma unroll
          for (int t = 0; t < 4; ++t) {
            const int c = c0 + t * p.splits;
            if (c < BN && tok0 + c < p.M) {
              float sum = 0.f;
#pragma unroll
              for (int s = 0; s < 8; ++s)
                if (s < p.splits) sum += v[t][s];
              put(p.C, p.out_f32, (size_t)(tok0 + c) * p.N + n, sum);
            }
          }
        }
      }
    }
    // nobody leaves while a peer may still read its shared memory
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(COLS) : "memory");
  }
}

// ------------------------------------------------------------------------------------------------ many tokens
__global__ void __launch_bounds__(MANY_THREADS, 1)
gemm_fp8_many_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w, Fp8Params p) {
  constexpr int X_BYTES = TILE_ROWS * KBYTES, W_BYTES = MANY_BN * KBYTES, STAGE = X_BYTES + W_BYTES;
  constexpr int NB = 2, COLS = 64;   // accumulators; columns of an epilogue thread
  extern __shared__ unsigned char smem_dyn[];
  unsigned char* smem = reinterpret_cast<unsigned char*>(((uintptr_t)smem_dyn + 1023) & ~(uintptr_t)1023);
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + MANY_STAGES * STAGE);
  uint64_t* empty = full + MANY_STAGES;
  uint64_t* acc_full = empty + MANY_STAGES;
  uint64_t* acc_empty = acc_full + NB;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_empty + NB);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < MANY_STAGES; ++s) {
      mbar_init(full + s, 1);
      mbar_init(empty + s, 1);
    }
    for (int b = 0; b < NB; ++b) {
      mbar_init(acc_full + b, 1);
      mbar_init(acc_empty + b, MANY_BN / 16);
    }
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(s32(tmem_slot)), "r"(512u) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  bspec::pdl_prologue(83);
  const int nkb = (p.K + KBYTES - 1) / KBYTES;
  const long long tiles = (long long)p.tiles_m * p.tiles_n;

  if (warp < 2) {
    const uint32_t one = elect_one();
    if (warp == 0) {
      int s = 0;
      uint32_t phase = 0u;
      bool ok = true;
      for (long long t = blockIdx.x; t < tiles && ok; t += gridDim.x) {
        const int m0 = (int)(t % p.tiles_m) * TILE_ROWS, n0 = (int)(t / p.tiles_m) * MANY_BN;
        for (int kb = 0; kb < nkb; ++kb) {
          if (!(ok = warp_wait(empty + s, phase ^ 1u, abort_flag, p.status, 105))) break;
          mbar_expect_tx_by(one, full + s, (uint32_t)STAGE);
          tma_load_2d_by(one, smem + s * STAGE, &map_x, full + s, kb * KBYTES, m0);
          tma_load_2d_by(one, smem + s * STAGE + X_BYTES, &map_w, full + s, kb * KBYTES, n0);
          if (++s == MANY_STAGES) { s = 0; phase ^= 1u; }
        }
      }
      if (*abort_flag)                       // copies in flight land (they take microseconds) before the CTA ends
        for (int i = 0; i < 1000; ++i) __nanosleep(1000);
    } else {
      const uint32_t idesc = instr_desc_e4m3(MANY_BN);
      const uint64_t desc0 = smem_desc(smem);
      int s = 0, b = 0;
      uint32_t phase = 0u, acc_phase = 0u;
      bool ok = true;
      for (long long t = blockIdx.x; t < tiles && ok; t += gridDim.x) {
        for (int kb = 0; kb < nkb; ++kb) {
          if (!(ok = warp_wait(full + s, phase, abort_flag, p.status, 106))) break;
          if (!(ok = warp_wait(acc_empty + b, acc_phase ^ 1u, abort_flag, p.status, 107))) break;
          tc_fence_after();
          const uint64_t xd = desc0 + (uint64_t)(s * (STAGE / 16)), wd = xd + X_BYTES / 16;
#pragma unroll
          for (int k = 0; k < KBYTES / 32; ++k) tc_mma_8bit_by(one, tmem_base + b * MANY_BN, xd + 2 * k, wd + 2 * k, idesc, k > 0 ? 1u : 0u);
          tc_commit_by(one, empty + s);
          tc_commit_by(one, acc_full + b);
          if (++s == MANY_STAGES) { s = 0; phase ^= 1u; }
          if (++b == NB) { b = 0; acc_phase ^= 1u; }
        }
      }
    }
  } else {
    const uint32_t quad = warp & 3;
    const int group = (warp - 2) >> 2;                                  // columns 64 group .. of the tile: in one row of W's scales
    const uint32_t lane_base = tmem_base + ((quad * 32u) << 16) + (uint32_t)(group * COLS);
    const int row = (int)quad * 32 + lane;
    int b = 0;
    uint32_t phase = 0u;
    bool ok = true;
    for (long long t = blockIdx.x; t < tiles && ok; t += gridDim.x) {
      const int m = (int)(t % p.tiles_m) * TILE_ROWS + row, n0 = (int)(t / p.tiles_m) * MANY_BN + group * COLS;
      const long long srow = min(m, p.M - 1), wrow = min(n0, p.N - 1) / 128;
      float acc[COLS];
#pragma unroll
      for (int c = 0; c < COLS; ++c) acc[c] = 0.f;
      float x_next = scale_at(p.xs, srow, 0), w_next = scale_at(p.ws, wrow, 0);
      // whether a row's product of scales is not a normal number: asked behind the additions, when the next scales have come (before the wait for
      // an accumulator it cost 14 of 118 us of the product of 1,537 x 4,096 x 14,336, here nothing)
      bool apart = __any_sync(0xffffffffu, !is_ordinary(x_next * w_next));
      for (int kb = 0; kb < nkb; ++kb) {
        const float x = x_next, w = w_next;
        if (kb + 1 < nkb) {
          x_next = scale_at(p.xs, srow, kb + 1);
          w_next = scale_at(p.ws, wrow, kb + 1);
        }
        if (!(ok = warp_wait(acc_full + b, phase, abort_flag, p.status, 108))) break;
        tc_fence_after();
        // all columns in one load: what bounds this loop is the number of trips to the tensor memory, not their width
        uint32_t v[COLS];
        tc_ld64(lane_base + (uint32_t)(b * MANY_BN), v);
        tc_wait_ld();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(acc_empty + b);
        if (++b == NB) { b = 0; phase ^= 1u; }
        float f = x * w;
        if (apart) {
          float before = 1.f;
          if (leaves_range(x, w, f)) split_scales(x, w, before, f);
#pragma unroll
          for (int c = 0; c < COLS; ++c) v[c] = __float_as_uint(__uint_as_float(v[c]) * before);
        }
        const uint64_t ff = pack2(f, f);
#pragma unroll
        for (int c = 0; c < COLS; c += 2) {                             // two to an instruction: the loop's time is what it issues
          const uint64_t sum = fma2(pack2(__uint_as_float(v[c]), __uint_as_float(v[c + 1])), ff, pack2(acc[c], acc[c + 1]));
          unpack2(sum, acc[c], acc[c + 1]);
        }
        apart = __any_sync(0xffffffffu, !is_ordinary(x_next * w_next));
      }
      if (ok && m < p.M) {
        const size_t base = (size_t)m * p.N + n0;
        if (p.N % 16 == 0 && n0 + COLS <= p.N) {
#pragma unroll
          for (int c = 0; c < COLS; c += 16) put16(p.C, p.out_f32, base + c, acc + c);
        } else {
#pragma unroll
          for (int c = 0; c < COLS; ++c)
            if (n0 + c < p.N) put(p.C, p.out_f32, base + c, acc[c]);
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(512u) : "memory");
  }
}

// ------------------------------------------------------------------------------------------------ many tokens, powers of two as scales
// Both matrices' scales in 8 bits (e8m0): the tensor cores take them (kind::mxf8f6f4, a scale per 32 k, here the same one four times), nothing is
// added outside of them, and the sums of a whole row stay in tensor memory.  What then bounds a product is the way from the L2 into an SM (64 bytes
// a clock): a 128 x 256 tile of one CTA asks for 48 KB per 128 k, 750 clocks where its products take 512.  So two CTAs work on one tile of
// 256 x PAIR_BN (cta_group::2): each keeps its own 128 rows of X and half the rows of W, 30 KB per 128 k for 448 clocks of products.
//   TMA warp      its CTA's halves of a stage; the bytes are counted on the first CTA's barrier
//   MMA warp      (first CTA) copies the scales of both CTAs into their tensor memory and issues the products for both
//   scale warps   bring the scales of four stages into the form that is copied: 32 lanes x 16 bytes, rows l, l + 32, l + 64, l + 96, a byte per
//                 stage (the products of a stage name its byte)
//   epilogue      eight warps: 128 rows x half the columns, read at once, freed, converted and stored while the next tile's products run
// The tensor cores cut what an addition shifts out, always towards 0: over K products of one sign a sum that stays in them is off by 8.5e-8 of it at
// 512 numbers, 2.0e-7 at 1,024, 5.2e-7 at 2,048, 1.5e-6 at 4,096 (root mean square), where a float32 product in the usual order is off by 5e-8 to
// 2.3e-7.  A bfloat16 result does not notice (its rounding is 2e-3).  For a float32 result (JOIN) the accumulators change every PAIR_JOIN blocks of k, and
// the epilogue adds them up in registers: 1.9e-7 at any K.  2,048 x 28,672 x 4,096 then takes 229 us instead of 200 (every 6 blocks 1.0e-7 and 247 us,
// every 4 blocks 8.5e-8 and 264 us: what counts is the way of an accumulator through the epilogue and back; sums in registers for every block 414).
constexpr int PAIR_JOIN = 8;           // blocks of k
constexpr int PAIR_BN = 224, PAIR_STAGES = 7, PAIR_SF_SLOTS = 4, PAIR_SF_BUFS = 5, PAIR_THREADS = 448;
constexpr int PAIR_X = TILE_ROWS * KBYTES, PAIR_W = PAIR_BN / 2 * KBYTES, PAIR_STAGE = PAIR_X + PAIR_W;
constexpr int PAIR_SF = 512 + 1024;          // the scales of four stages: 128 rows of X, 256 of W
constexpr int PAIR_SF_COL = 2 * PAIR_BN;     // tensor memory columns: two accumulators, then five places for scales, 4 + 8 columns
                                             // each: the stages in flight reach over three of them at most

__device__ __forceinline__ uint32_t in_cta(const void* p, uint32_t rank) {     // the same place in another CTA's shared memory
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(s32(p)), "r"(rank));
  return r;
}
__device__ __forceinline__ void arrive_in(uint32_t bar) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void tma_load_pair(uint32_t one, void* dst, const CUtensorMap* map, uint32_t bar, int x, int y) {
  asm volatile(
      "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %5, 0;\n\t"
      "@q cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];\n\t}"
      ::"r"(s32(dst)), "l"(map), "r"(bar), "r"(x), "r"(y), "r"(one) : "memory");
}
__device__ __forceinline__ void commit_pair(uint32_t one, uint64_t* bar) {
  asm volatile(
      "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %2, 0;\n\t"
      "@q tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;\n\t}"
      ::"r"(s32(bar)), "h"((uint16_t)3), "r"(one) : "memory");
}
__device__ __forceinline__ void copy_scales(uint32_t one, uint32_t tmem, const void* smem) {
  const uint64_t desc = (uint64_t)((s32(smem) & 0x3FFFFu) >> 4) | (8ull << 32) | (1ull << 46);     // 8-row groups 128 bytes apart, no swizzle
  asm volatile(
      "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %2, 0;\n\t"
      "@q tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;\n\t}" ::"r"(tmem), "l"(desc), "r"(one) : "memory");
}
__device__ __forceinline__ void mma_scaled(uint32_t one, uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t sfa,
                                           uint32_t sfb, uint32_t accum) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.b32 p, %6, 0;\n\t"
      "setp.ne.b32 q, %7, 0;\n\t"
      "@q tcgen05.mma.cta_group::2.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%4], [%5], p;\n\t}"
      ::"r"(tmem_d), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accum), "r"(one) : "memory");
}

template <bool JOIN>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(PAIR_THREADS, 1)
gemm_fp8_pair_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w, Fp8Params p) {
  extern __shared__ unsigned char smem_dyn[];
  unsigned char* smem = reinterpret_cast<unsigned char*>(((uintptr_t)smem_dyn + 1023) & ~(uintptr_t)1023);
  unsigned char* sf = smem + PAIR_STAGES * PAIR_STAGE;
  __shared__ uint64_t full[PAIR_STAGES], empty[PAIR_STAGES], sf_full[PAIR_SF_SLOTS], sf_empty[PAIR_SF_SLOTS], acc_full[2], acc_empty[2];
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_word;
  volatile int* abort_flag = &abort_word;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = blockIdx.x & 1;
  if (threadIdx.x == 0) {
    for (int s = 0; s < PAIR_STAGES; ++s) {
      mbar_init(full + s, 1);
      mbar_init(empty + s, 1);
    }
    for (int s = 0; s < PAIR_SF_SLOTS; ++s) {
      mbar_init(sf_full + s, 2);             // a scale warp of each CTA
      mbar_init(sf_empty + s, 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(acc_full + b, 1);
      mbar_init(acc_empty + b, 16);          // the epilogue warps of both CTAs
    }
    abort_word = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(s32(&tmem_slot)), "r"(512u) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  // both CTAs run and have their barriers before one writes to the other
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
  tc_fence_after();
  const uint32_t tmem_base = tmem_slot;
  bspec::pdl_prologue(86);
  const int nkb = (p.K + KBYTES - 1) / KBYTES;
  const long long tiles = (long long)p.tiles_m * p.tiles_n;
  const long long pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;

  if (warp == 0) {
    const uint32_t one = elect_one();
    int st = 0;
    uint32_t phase = 0u;
    bool ok = true;
    for (long long t = pair; t < tiles && ok; t += pairs) {
      const int m0 = (int)(t % p.tiles_m) * 256 + (int)rank * TILE_ROWS, n0 = (int)(t / p.tiles_m) * PAIR_BN + (int)rank * (PAIR_BN / 2);
      for (int kb = 0; kb < nkb; ++kb) {
        if (!(ok = warp_wait(empty + st, phase ^ 1u, abort_flag, p.status, 121))) break;
        if (rank == 0) mbar_expect_tx_by(one, full + st, 2 * PAIR_STAGE);
        const uint32_t bar = in_cta(full + st, 0);
        unsigned char* at = smem + st * PAIR_STAGE;
        tma_load_pair(one, at, &map_x, bar, kb * KBYTES, m0);
        tma_load_pair(one, at + PAIR_X, &map_w, bar, kb * KBYTES, n0);
        if (++st == PAIR_STAGES) { st = 0; phase ^= 1u; }
      }
    }
    if (*abort_flag)                         // copies in flight land (they take microseconds) before the CTA ends
      for (int i = 0; i < 1000; ++i) __nanosleep(1000);
  } else if (warp == 1) {
    if (rank == 0) {
      const uint32_t one = elect_one();
      // float32 sums, e4m3 X and W, e8m0 scales, M = 256, N = PAIR_BN
      const uint32_t idesc = ((uint32_t)(PAIR_BN >> 3) << 17) | (1u << 23) | (16u << 24);
      int st = 0, b = 0, slot = 0, buf = 0;
      uint32_t phase = 0u, acc_phase = 0u, sf_phase = 0u;
      bool ok = true;
      for (long long t = pair; t < tiles && ok; t += pairs) {
        // an accumulator for the whole row or, JOIN, for every PAIR_JOIN blocks of it
        auto next_acc = [&]() {
          ok = __all_sync(0xffffffffu, mbar_wait<true>(acc_empty + b, acc_phase ^ 1u, abort_flag, p.status, 122));
          tc_fence_after();
        };
        next_acc();
        if (!ok) break;
        uint32_t sfa = 0u, sfb = 0u;
        int done = 0;                        // blocks in this accumulator
        for (int kb = 0; kb < nkb; ++kb) {
          if constexpr (JOIN) {
            if (done == PAIR_JOIN) {
              commit_pair(one, acc_full + b);
              if (++b == 2) { b = 0; acc_phase ^= 1u; }
              next_acc();
              if (!ok) break;
              done = 0;
            }
          }
          if ((kb & 3) == 0) {
            if (!(ok = __all_sync(0xffffffffu, mbar_wait<true>(sf_full + slot, sf_phase, abort_flag, p.status, 126)))) break;
            tc_fence_after();
            sfa = tmem_base + PAIR_SF_COL + buf * 12;
            sfb = sfa + 4;
            copy_scales(one, sfa, sf + slot * PAIR_SF);
            copy_scales(one, sfb, sf + slot * PAIR_SF + 512);
            copy_scales(one, sfb + 4, sf + slot * PAIR_SF + 1024);
            commit_pair(one, sf_empty + slot);
            if (++buf == PAIR_SF_BUFS) buf = 0;
            if (++slot == PAIR_SF_SLOTS) { slot = 0; sf_phase ^= 1u; }
          }
          if (!(ok = __all_sync(0xffffffffu, mbar_wait<true>(full + st, phase, abort_flag, p.status, 123)))) break;
          tc_fence_after();
          const uint32_t desc = idesc | ((uint32_t)(kb & 3) << 4) | ((uint32_t)(kb & 3) << 29);
          const uint64_t xd = smem_desc(smem + st * PAIR_STAGE), wd = smem_desc(smem + st * PAIR_STAGE + PAIR_X);
#pragma unroll
          for (int k = 0; k < KBYTES / 32; ++k)
            mma_scaled(one, tmem_base + b * PAIR_BN, xd + 2 * k, wd + 2 * k, desc, sfa, sfb, ((JOIN ? done : kb) > 0 || k > 0) ? 1u : 0u);
          commit_pair(one, empty + st);
          if (++st == PAIR_STAGES) { st = 0; phase ^= 1u; }
          ++done;
        }
        if (!ok) break;
        commit_pair(one, acc_full + b);
        if (++b == 2) { b = 0; acc_phase ^= 1u; }
      }
    }
  } else if (warp < 6) {
    // groups of four stages go round the four warps, each with a place of its own; the next group's loads are on their way while this one waits
    const uint8_t* xs = reinterpret_cast<const uint8_t*>(p.xs.p);
    const uint8_t* ws = reinterpret_cast<const uint8_t*>(p.ws.p);
    const int groups = (nkb + 3) / 4;
    long long t = pair;
    static_assert(PAIR_SF_SLOTS == 4, "a place per warp: one that fills another's would not know its turn by the barrier's parity");
    const int slot = warp - 2;
    int g = slot;
    uint32_t phase = 0u;
    bool ok = true;
    uint32_t v[3][4];                        // X, W up to 128 rows of the tile and behind; rows lane, lane + 32, ...
    auto fetch = [&]() {
      while (g >= groups) {
        g -= groups;
        t += pairs;
      }
      if (t >= tiles) return;
      const int tn = (int)(t / p.tiles_m), tm = (int)(t - (long long)tn * p.tiles_m);
      const int m = tm * 256 + (int)rank * TILE_ROWS + lane, n = tn * PAIR_BN + lane, kb = 4 * g;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint8_t* from[3] = {xs + (long long)min(m + 32 * j, p.M - 1) * p.xs.ld, ws + (long long)(min(n + 32 * j, p.N - 1) / 128) * p.ws.ld,
                                  ws + (long long)(min(n + 128 + 32 * j, p.N - 1) / 128) * p.ws.ld};
#pragma unroll
        for (int i = 0; i < 3; ++i) {
          v[i][j] = 0u;
#pragma unroll
          for (int k = 0; k < 4; ++k) v[i][j] |= (uint32_t)__ldg(from[i] + min(kb + k, nkb - 1)) << (8 * k);
        }
      }
    };
    fetch();
    while (t < tiles && ok) {
      uint4 w[3];
#pragma unroll
      for (int i = 0; i < 3; ++i) w[i] = make_uint4(v[i][0], v[i][1], v[i][2], v[i][3]);
      g += 4;
      fetch();
      if (!(ok = warp_wait(sf_empty + slot, phase ^ 1u, abort_flag, p.status, 124))) break;
      unsigned char* to = sf + slot * PAIR_SF + lane * 16;
#pragma unroll
      for (int i = 0; i < 3; ++i) *reinterpret_cast<uint4*>(to + 512 * i) = w[i];
      fence_async_smem();
      __syncwarp();
      if (lane == 0) arrive_in(in_cta(sf_full + slot, 0));
      phase ^= 1u;
    }
  } else {
    const uint32_t quad = warp & 3;
    const int half = (warp - 6) >> 2;        // columns PAIR_BN / 2 half ..
    constexpr int COLS = PAIR_BN / 2;
    const int row = (int)quad * 32 + lane;
    int b = 0;
    uint32_t phase = 0u;
    bool ok = true;
    for (long long t = pair; t < tiles && ok; t += pairs) {
      const int m = (int)(t % p.tiles_m) * 256 + (int)rank * TILE_ROWS + row, n0 = (int)(t / p.tiles_m) * PAIR_BN + half * COLS;
      float acc[COLS];
      // this thread's columns of an accumulator, which then is free; into the sums or, JOIN, onto them
      auto take = [&]() {
        if (!(ok = warp_wait(acc_full + b, phase, abort_flag, p.status, 125))) return;
        tc_fence_after();
        const uint32_t from = tmem_base + ((quad * 32u) << 16) + (uint32_t)(b * PAIR_BN + half * COLS);
        if constexpr (JOIN) {
#pragma unroll
          for (int c = 0; c < COLS; c += 16) {
            uint32_t v[16];
            tc_ld16(from + c, v);
            tc_wait_ld();
#pragma unroll
            for (int j = 0; j < 16; ++j) acc[c + j] += __uint_as_float(v[j]);
          }
        } else {
#pragma unroll
          for (int c = 0; c < COLS; c += 16) tc_ld16(from + c, *reinterpret_cast<uint32_t(*)[16]>(acc + c));
          tc_wait_ld();
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) arrive_in(in_cta(acc_empty + b, 0));
        if (++b == 2) { b = 0; phase ^= 1u; }
      };
      if constexpr (JOIN) {
#pragma unroll
        for (int c = 0; c < COLS; ++c) acc[c] = 0.f;
#pragma unroll 1
        for (int k0 = 0; k0 < nkb && ok; k0 += PAIR_JOIN) take();
      } else {
        take();
      }
      if (!ok) break;
      if (m < p.M) {
        const size_t base = (size_t)m * p.N + n0;
        if (p.N % 16 == 0 && n0 + COLS <= p.N) {
#pragma unroll
          for (int c = 0; c < COLS; c += 16) put16(p.C, p.out_f32, base + c, acc + c);
        } else {
#pragma unroll
          for (int c = 0; c < COLS; ++c)
            if (n0 + c < p.N) put(p.C, p.out_f32, base + c, acc[c]);
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  // nobody leaves while the other may still use its memory
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(512u) : "memory");
  }
}

// ------------------------------------------------------------------------------------------------ host side
// rows x K bytes, rows `ld` bytes apart; box = box_rows x 128 bytes, 128-byte swizzle; bytes outside read as 0
bool make_map_bytes(CUtensorMap* map, const void* base, long long rows, int K, long long ld, int box_rows) {
  auto fn = encode_fn();
  if (fn == nullptr) return false;
  cuuint64_t dims[2] = {(cuuint64_t)K, (cuuint64_t)rows};
  cuuint64_t strides[1] = {(cuuint64_t)ld};
  cuuint32_t box[2] = {(cuuint32_t)KBYTES, (cuuint32_t)box_rows};
  cuuint32_t elem[2] = {1, 1};
  return fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE,
            CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// slices of k of the arrangement for few tokens: two CTAs share an SM, and K is cut so that the CTAs about fill those slots, at least 4 blocks
// to a slice; 1, 2, 4 or 8, and where the rounding of their lengths leaves the eighth empty (33 to 35, 41, 42 and 49 blocks), seven
int few_splits(long long tiles, int nkb, int sms) {
  long long splits = 2ll * sms / tiles;
  if (splits > nkb / 4) splits = nkb / 4;
  return splits >= 8 ? 8 : (splits >= 4 ? 4 : (splits >= 2 ? 2 : 1));
}

// The arrangement that an estimate of its time takes: a start, and rounds of the tiles over the SMs of so many blocks of k each.  The numbers
// (us) are fits to times on B200: 48 to 1,536 tokens by 4,096 x 4,096, 28,672 x 4,096, 4,096 x 14,336, 2,048 x 2,048 and 1,040 x 720.
// E.g. 4,096 x 14,336, few / many / pairs: 64 tokens 19 / 48 / 42, 256 tokens 51 / 50 / 46, 1,024 tokens - / 98 / 77;
// 4,096 x 4,096: 128 tokens 13 / 17 / 23, 512 tokens 29 / 18 / 24.
enum Form { FEW, MANY, PAIR };
Form choose(int M, int N, int K, bool powers, int sms) {
  const int nkb = (K + KBYTES - 1) / KBYTES;
  const int bn = M <= 16 ? 16 : (M <= 32 ? 32 : 64);
  const long long few_tiles = ((long long)N + TILE_ROWS - 1) / TILE_ROWS * (((long long)M + bn - 1) / bn);
  const int splits = few_splits(few_tiles, nkb, sms);
  auto rounds = [](long long tiles, long long at_once) { return (double)((tiles + at_once - 1) / at_once); };
  const double few = 5.5 + rounds(few_tiles * splits, 2 * sms) * ((nkb + splits - 1) / splits) * (bn == 16 ? 0.45 : (bn == 32 ? 0.6 : 0.87));
  const double many = 6 + rounds(((long long)M + 127) / 128 * (((long long)N + MANY_BN - 1) / MANY_BN), sms) * (0.35 * nkb + 2);
  const double pair = 7 + rounds(((long long)M + 255) / 256 * (((long long)N + PAIR_BN - 1) / PAIR_BN), sms / 2) * (0.27 * nkb + 4);
  const bool fits = ((long long)M + bn - 1) / bn <= 65535;      // a grid's second dimension
  if (fits && few <= many && (!powers || few <= pair)) return FEW;
  return powers && pair < many ? PAIR : MANY;
}

template <int BN>
int launch_few(const CUtensorMap& map_w, const CUtensorMap& map_x, Fp8Params p, int sms, cudaStream_t stream) {
  const int kb_total = (p.K + KBYTES - 1) / KBYTES;
  const int tiles_n = (p.N + TILE_ROWS - 1) / TILE_ROWS, tiles_t = (p.M + BN - 1) / BN;
  const int splits = few_splits((long long)tiles_n * tiles_t, kb_total, sms);
  p.kblocks_per_split = (kb_total + splits - 1) / splits;
  p.splits = (kb_total + p.kblocks_per_split - 1) / p.kblocks_per_split;       // no empty slice
  constexpr int STAGE = (TILE_ROWS + BN) * KBYTES;
  constexpr int FIXED = 1024 + 2 * FEW_WINDOW * BN * 4 + 256;
  int stages = (112 * 1024 - FIXED) / STAGE;
  if (stages > 6) stages = 6;
  // the join's partial tile takes the stages' place
  const int least = (BN * TILE_ROWS * 4 + STAGE - 1) / STAGE;
  if (stages > p.kblocks_per_split + 1) stages = p.kblocks_per_split + 1;
  if (stages < 2) stages = 2;
  if (stages < least) stages = least;
  p.stages = stages;
  const size_t smem = (size_t)stages * STAGE + FIXED;
  static size_t set_dev[bspec::kMaxDevices] = {};
  size_t& set = set_dev[bspec::current_device()];
  if (smem > set) {
    const cudaError_t e = cudaFuncSetAttribute(gemm_fp8_few_kernel<BN>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return (int)e;
    set = smem;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(tiles_n, tiles_t, p.splits);
  cfg.blockDim = dim3(FEW_THREADS);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 1;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = p.splits;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = bspec::pdl_enabled() ? 2 : 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, gemm_fp8_few_kernel<BN>, map_w, map_x, p);
  if (e != cudaSuccess) return (int)e;
  return BSPEC_LAUNCH_CHECK();
}

typedef void (*WholeKernel)(CUtensorMap, CUtensorMap, Fp8Params);
int launch_whole(WholeKernel kernel, const CUtensorMap& map_x, const CUtensorMap& map_w, const Fp8Params& p, long long grid, int threads,
                 size_t smem, cudaStream_t stream) {
  const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  if (e != cudaSuccess) return (int)e;
  (void)bspec::launch(kernel, dim3((unsigned)grid), dim3(threads), smem, stream, map_x, map_w, p);
  return BSPEC_LAUNCH_CHECK();
}

}  // namespace

// C [M, N] = X W^T with block scales.  X, W: e4m3, rows ldx / ldw bytes apart (multiples of 16, bases on 16 bytes); xs [M, ceil(K / 128)]
// and ws [ceil(N / 128), ceil(K / 128)] with rows ldxs / ldws scales apart, float32 or (xs_e8m0, ws_e8m0) 8-bit exponents.
// `w_ahead`: W and ws are complete whatever still runs on the stream.  `status`: one int on the device, 0 unless a bounded wait ran out.
BSPEC_API int bspec_gemm_fp8(const void* X, long long ldx, const void* xs, long long ldxs, int xs_e8m0, const void* W, long long ldw,
                             const void* ws, long long ldws, int ws_e8m0, void* C, int out_f32, int M, int N, int K, int w_ahead,
                             int* status, cudaStream_t stream) {
  if (M <= 0 || N <= 0) return 0;
  if (K <= 0 || K > 0x7fffffff - 256 || N > 0x7fffffff - 512 || M > 0x7fffffff - 512 || ldx % 16 != 0 || ldw % 16 != 0 || ldx < K || ldw < K)
    return (int)cudaErrorInvalidValue;
  Fp8Params p = {};
  p.C = C; p.status = status;
  p.xs = {xs, ldxs, xs_e8m0};
  p.ws = {ws, ldws, ws_e8m0};
  p.M = M; p.N = N; p.K = K; p.out_f32 = out_f32; p.w_ahead = w_ahead;
  const int sms = bspec::sm_count();
  const long long tiles_m = (M + TILE_ROWS - 1) / TILE_ROWS, tiles_n = (N + MANY_BN - 1) / MANY_BN;
  const long long pairs_m = (M + 255) / 256, pairs_n = (N + PAIR_BN - 1) / PAIR_BN;
  const Form form = choose(M, N, K, xs_e8m0 && ws_e8m0, sms);
  CUtensorMap map_x, map_w;
  const int bn = M <= 16 ? 16 : (M <= 32 ? 32 : 64);
  if (!make_map_bytes(&map_x, X, M, K, ldx, form == FEW ? bn : TILE_ROWS) ||
      !make_map_bytes(&map_w, W, N, K, ldw, form == PAIR ? PAIR_BN / 2 : (form == MANY ? MANY_BN : TILE_ROWS)))
    return (int)cudaErrorInvalidValue;
  if (form == FEW) {
    if (bn == 16) return launch_few<16>(map_w, map_x, p, sms, stream);
    if (bn == 32) return launch_few<32>(map_w, map_x, p, sms, stream);
    return launch_few<64>(map_w, map_x, p, sms, stream);
  }
  if (form == MANY) {
    p.tiles_m = (int)tiles_m; p.tiles_n = (int)tiles_n;
    return launch_whole(gemm_fp8_many_kernel, map_x, map_w, p, tiles_m * tiles_n < sms ? tiles_m * tiles_n : sms, MANY_THREADS,
                        1024 + (size_t)MANY_STAGES * (TILE_ROWS + MANY_BN) * KBYTES + 256, stream);
  }
  p.tiles_m = (int)pairs_m; p.tiles_n = (int)pairs_n;
  return launch_whole(out_f32 && (K + KBYTES - 1) / KBYTES > PAIR_JOIN ? gemm_fp8_pair_kernel<true> : gemm_fp8_pair_kernel<false>, map_x, map_w, p, 2 * (pairs_m * pairs_n < sms / 2 ? pairs_m * pairs_n : sms / 2), PAIR_THREADS,
                      1024 + (size_t)PAIR_STAGES * PAIR_STAGE + PAIR_SF_SLOTS * PAIR_SF, stream);
}

BSPEC_DEFINE_TRACE_SETTER(bspec_trace_set_gemm_fp8)
