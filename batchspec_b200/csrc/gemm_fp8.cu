// Matrix product in 8-bit floating point (e4m3) with a scale for each block of 128, on the 5th-generation tensor cores:
//   C[m, n] = sum over blocks b of 128 k:  xs[m, b] * ws[n / 128, b] * sum over k in b of X[m, k] * W[n, k]
// X [M, K] has a scale per row and block, W [N, K] one per 128 x 128; scales are float32 numbers or powers of two in 8 bits (e8m0).
//
// The products of one block are exact sums of the tensor core (tcgen05.mma kind::f8f6f4, float32 accumulator in tensor memory); the
// scales differ from block to block, so every block of 128 k gets an accumulator of its own (a ring of them in tensor memory), and
// the epilogue warps read it back, multiply by its scales and add it to float32 sums in registers while the next blocks' products
// run.  The sum over blocks is in ascending k.
//
// Two arrangements:
//   rows of W on the accumulator's 128 rows, tokens on its columns (few tokens): every weight is streamed once at full tile
//     efficiency.  K may be cut into `splits` slices run by the CTAs of one cluster, whose partial tiles are joined in slice
//     order through distributed shared memory.
//   tokens on the rows, 256 rows of W on the columns (many tokens): one persistent CTA per SM; eight epilogue warps hold the
//     128 x 256 sums.
#include "e4m3.cuh"
#include "umma.cuh"

using namespace bspec;

namespace {

constexpr int KBYTES = 128;            // k per stage: one scale block, one 128-byte swizzle span
constexpr int TILE_ROWS = 128;
constexpr int FEW_THREADS = 192;       // TMA warp, MMA warp, 4 epilogue warps
constexpr int FEW_WINDOW = 32;         // k blocks whose scales wait in shared memory at a time
constexpr int MANY_THREADS = 320;      // TMA warp, MMA warp, 8 epilogue warps
constexpr int MANY_BN = 256, MANY_STAGES = 4;

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

__device__ __forceinline__ void mma_e4m3(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accum) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}"
      ::"r"(tmem_d), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accum) : "memory");
}
// float32 accumulator, e4m3 A and B (format code 0), both K-major, M = 128, N = bn
__device__ __forceinline__ uint32_t e4m3_desc(int bn) {
  return (1u << 4) | ((uint32_t)(bn >> 3) << 17) | ((uint32_t)(TILE_ROWS >> 4) << 24);
}
__device__ __forceinline__ void put(void* C, int out_f32, size_t at, float v) {
  if (out_f32) reinterpret_cast<float*>(C)[at] = v;
  else reinterpret_cast<__nv_bfloat16*>(C)[at] = __float2bfloat16_rn(v);
}
// Let copies in flight land before the CTA gives up its shared memory (after a wait ran out).
__device__ __forceinline__ void drain(uint64_t* full, int armed, int stages) {
  for (int i = max(0, armed - stages); i < armed; ++i) {
    const uint32_t ph = (uint32_t)(i / stages) & 1u;
    for (uint32_t t = 0; t < (1u << 16) && !mbar_try_wait(full + i % stages, ph); ++t) __nanosleep(32);
  }
}

// ------------------------------------------------------------------------------------------------ few tokens
constexpr int few_buffers(int bn) { return bn >= 128 ? 2 : 4; }      // accumulators: two CTAs of an SM share 512 columns

template <int BN>
__global__ void __launch_bounds__(FEW_THREADS)
gemm_fp8_few_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x, Fp8Params p) {
  constexpr int NB = few_buffers(BN);
  constexpr uint32_t COLS = NB * BN;                                   // 64, 128 or 256: powers of two
  constexpr int W_BYTES = TILE_ROWS * KBYTES, X_BYTES = BN * KBYTES, STAGE = W_BYTES + X_BYTES;
  extern __shared__ unsigned char smem_dyn[];
  unsigned char* smem = reinterpret_cast<unsigned char*>(((uintptr_t)smem_dyn + 1023) & ~(uintptr_t)1023);
  float* scales = reinterpret_cast<float*>(smem + (size_t)p.stages * STAGE);      // [FEW_WINDOW][BN], xs * ws
  uint64_t* full = reinterpret_cast<uint64_t*>(scales + FEW_WINDOW * BN);
  uint64_t* empty = full + p.stages;
  uint64_t* acc_full = empty + p.stages;
  uint64_t* acc_empty = acc_full + NB;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_empty + NB);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  float* part = reinterpret_cast<float*>(smem);                        // [BN][128] sums of this K slice, over the stages

  const unsigned long long t_trace = bspec::g_trace_buf != nullptr ? bspec::global_timer() : 0ull;
  bspec::pdl_launch_dependents();
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
      mbar_init(acc_empty + b, 128);
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

  float acc[BN];
#pragma unroll
  for (int c = 0; c < BN; ++c) acc[c] = 0.f;

  if (warp == 0) {
    if (lane == 0) {
      int armed = 0;
      if (!p.w_ahead) bspec::pdl_wait();
      const int pre = min(nkb, p.stages);
      for (int i = 0; i < pre; ++i) {
        mbar_expect_tx(full + i, (uint32_t)STAGE);
        tma_load_2d(smem + (size_t)i * STAGE, &map_w, full + i, (kb0 + i) * KBYTES, tile_n * TILE_ROWS);
      }
      bspec::pdl_wait();
      bspec::trace_record(82, t_trace);
      for (int i = 0; i < pre; ++i)
        tma_load_2d(smem + (size_t)i * STAGE + W_BYTES, &map_x, full + i, (kb0 + i) * KBYTES, tok0);
      armed = pre;
      for (int i = pre; i < nkb; ++i) {
        const int s = i % p.stages;
        if (!mbar_wait(empty + s, ((uint32_t)(i / p.stages) & 1u) ^ 1u, abort_flag, p.status, 101)) break;
        mbar_expect_tx(full + s, (uint32_t)STAGE);
        tma_load_2d(smem + (size_t)s * STAGE, &map_w, full + s, (kb0 + i) * KBYTES, tile_n * TILE_ROWS);
        tma_load_2d(smem + (size_t)s * STAGE + W_BYTES, &map_x, full + s, (kb0 + i) * KBYTES, tok0);
        armed = i + 1;
      }
      if (*abort_flag) drain(full, armed, p.stages);
    }
  } else if (warp == 1) {
    if (lane == 0) {
      const uint32_t idesc = e4m3_desc(BN);
      for (int i = 0; i < nkb; ++i) {
        const int s = i % p.stages, b = i % NB;
        if (!mbar_wait(full + s, (uint32_t)(i / p.stages) & 1u, abort_flag, p.status, 102)) break;
        if (!mbar_wait(acc_empty + b, ((uint32_t)(i / NB) & 1u) ^ 1u, abort_flag, p.status, 103)) break;
        tc_fence_after();
        unsigned char* w_src = smem + (size_t)s * STAGE;
        const uint64_t wd = smem_desc(w_src), xd = smem_desc(w_src + W_BYTES);
#pragma unroll
        for (int k = 0; k < KBYTES / 32; ++k) mma_e4m3(tmem_base + b * BN, wd + 2 * k, xd + 2 * k, idesc, k > 0 ? 1u : 0u);
        tc_commit(empty + s);
        tc_commit(acc_full + b);
      }
    }
  } else {
    const uint32_t quad = warp & 3;
    const int et = threadIdx.x - 64;                                   // 0 .. 127
    bspec::pdl_wait();
    bool ok = true;
    for (int i = 0; i < nkb; ++i) {
      if (i % FEW_WINDOW == 0) {
        // the scales of the next blocks; every epilogue thread comes here, whatever its waits said
        const int nw = min(FEW_WINDOW, nkb - i);
        asm volatile("bar.sync 1, 128;" ::: "memory");
        for (int j = et; j < nw * BN; j += 128) {
          const int c = j / nw, b = j - c * nw, tok = tok0 + c;        // neighbours read neighbouring blocks of a token
          scales[b * BN + c] = tok < p.M ? scale_at(p.xs, tok, kb0 + i + b) * scale_at(p.ws, tile_n, kb0 + i + b) : 0.f;
        }
        asm volatile("bar.sync 1, 128;" ::: "memory");
      }
      const int b = i % NB;
      if (ok) ok = mbar_wait(acc_full + b, (uint32_t)(i / NB) & 1u, abort_flag, p.status, 104);
      if (!ok) continue;
      tc_fence_after();
      const float4* f = reinterpret_cast<const float4*>(scales + (i % FEW_WINDOW) * BN);
#pragma unroll
      for (int c0 = 0; c0 < BN; c0 += 16) {
        uint32_t v[16];
        tc_ld16(tmem_base + ((quad * 32u) << 16) + (uint32_t)(b * BN + c0), v);
        tc_wait_ld();
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float4 g = f[c0 / 4 + j];
          acc[c0 + 4 * j] = fmaf(__uint_as_float(v[4 * j]), g.x, acc[c0 + 4 * j]);
          acc[c0 + 4 * j + 1] = fmaf(__uint_as_float(v[4 * j + 1]), g.y, acc[c0 + 4 * j + 1]);
          acc[c0 + 4 * j + 2] = fmaf(__uint_as_float(v[4 * j + 2]), g.z, acc[c0 + 4 * j + 2]);
          acc[c0 + 4 * j + 3] = fmaf(__uint_as_float(v[4 * j + 3]), g.w, acc[c0 + 4 * j + 3]);
        }
      }
      tc_fence_before();
      mbar_arrive(acc_empty + b);
    }
    const int row = (int)quad * 32 + lane, n = tile_n * TILE_ROWS + row;
    if (p.splits == 1) {
      if (ok && n < p.N) {
#pragma unroll
        for (int c = 0; c < BN; ++c)
          if (tok0 + c < p.M) put(p.C, p.out_f32, (size_t)(tok0 + c) * p.N + n, acc[c]);
      }
    } else {
      // every product of this slice has completed and every stage has been read: the sums take their place
#pragma unroll
      for (int c = 0; c < BN; ++c) part[c * TILE_ROWS + row] = acc[c];
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
  constexpr int NB = 2;
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
      mbar_init(acc_empty + b, 256);
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

  if (warp == 0) {
    if (lane == 0) {
      int armed = 0;
      bool ok = true;
      for (long long t = blockIdx.x; t < tiles && ok; t += gridDim.x) {
        const int m0 = (int)(t % p.tiles_m) * TILE_ROWS, n0 = (int)(t / p.tiles_m) * MANY_BN;
        for (int kb = 0; kb < nkb; ++kb) {
          const int s = armed % MANY_STAGES;
          if (!(ok = mbar_wait(empty + s, ((uint32_t)(armed / MANY_STAGES) & 1u) ^ 1u, abort_flag, p.status, 105))) break;
          mbar_expect_tx(full + s, (uint32_t)STAGE);
          tma_load_2d(smem + s * STAGE, &map_x, full + s, kb * KBYTES, m0);
          tma_load_2d(smem + s * STAGE + X_BYTES, &map_w, full + s, kb * KBYTES, n0);
          ++armed;
        }
      }
      if (*abort_flag) drain(full, armed, MANY_STAGES);
    }
  } else if (warp == 1) {
    if (lane == 0) {
      const uint32_t idesc = e4m3_desc(MANY_BN);
      int i = 0;
      bool ok = true;
      for (long long t = blockIdx.x; t < tiles && ok; t += gridDim.x) {
        for (int kb = 0; kb < nkb; ++kb, ++i) {
          const int s = i % MANY_STAGES, b = i % NB;
          if (!(ok = mbar_wait(full + s, (uint32_t)(i / MANY_STAGES) & 1u, abort_flag, p.status, 106))) break;
          if (!(ok = mbar_wait(acc_empty + b, ((uint32_t)(i / NB) & 1u) ^ 1u, abort_flag, p.status, 107))) break;
          tc_fence_after();
          const uint64_t xd = smem_desc(smem + s * STAGE), wd = smem_desc(smem + s * STAGE + X_BYTES);
#pragma unroll
          for (int k = 0; k < KBYTES / 32; ++k) mma_e4m3(tmem_base + b * MANY_BN, xd + 2 * k, wd + 2 * k, idesc, k > 0 ? 1u : 0u);
          tc_commit(empty + s);
          tc_commit(acc_full + b);
        }
      }
    }
  } else {
    const uint32_t quad = warp & 3;
    const int half = (warp - 2) >> 2;                                   // columns 128 half .. of the tile: one row of W's scales
    const uint32_t lane_base = tmem_base + ((quad * 32u) << 16) + (uint32_t)(half * 128);
    const int row = (int)quad * 32 + lane;
    int i = 0;
    bool ok = true;
    for (long long t = blockIdx.x; t < tiles && ok; t += gridDim.x) {
      const int m = (int)(t % p.tiles_m) * TILE_ROWS + row, n0 = (int)(t / p.tiles_m) * MANY_BN + half * 128;
      const long long srow = min(m, p.M - 1), wrow = min(n0, p.N - 1) / 128;
      uint64_t acc[64];
#pragma unroll
      for (int c = 0; c < 64; ++c) acc[c] = 0ull;
      float f_next = scale_at(p.xs, srow, 0) * scale_at(p.ws, wrow, 0);
      for (int kb = 0; kb < nkb; ++kb, ++i) {
        const float f = f_next;
        if (kb + 1 < nkb) f_next = scale_at(p.xs, srow, kb + 1) * scale_at(p.ws, wrow, kb + 1);
        const uint64_t ff = pack2(f, f);
        const int b = i % NB;
        if (!(ok = mbar_wait(acc_full + b, (uint32_t)(i / NB) & 1u, abort_flag, p.status, 108))) break;
        tc_fence_after();
#pragma unroll
        for (int c0 = 0; c0 < 128; c0 += 32) {
          uint32_t v[32];
          tc_ld32(lane_base + (uint32_t)(b * MANY_BN + c0), v);
          tc_wait_ld();
#pragma unroll
          for (int j = 0; j < 16; ++j)
            acc[c0 / 2 + j] = fma2(pack2(__uint_as_float(v[2 * j]), __uint_as_float(v[2 * j + 1])), ff, acc[c0 / 2 + j]);
        }
        tc_fence_before();
        mbar_arrive(acc_empty + b);
      }
      if (ok && m < p.M) {
        const size_t base = (size_t)m * p.N + n0;
        if (!p.out_f32 && p.N % 8 == 0 && n0 + 128 <= p.N) {
          uint4* dst = reinterpret_cast<uint4*>(reinterpret_cast<__nv_bfloat16*>(p.C) + base);
#pragma unroll
          for (int c = 0; c < 16; ++c) {
            uint32_t w[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              float lo, hi;
              unpack2(acc[4 * c + j], lo, hi);
              __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
              w[j] = *reinterpret_cast<uint32_t*>(&h);
            }
            dst[c] = make_uint4(w[0], w[1], w[2], w[3]);
          }
        } else {
#pragma unroll
          for (int c = 0; c < 64; ++c) {
            float lo, hi;
            unpack2(acc[c], lo, hi);
            if (n0 + 2 * c < p.N) put(p.C, p.out_f32, base + 2 * c, lo);
            if (n0 + 2 * c + 1 < p.N) put(p.C, p.out_f32, base + 2 * c + 1, hi);
          }
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

template <int BN>
int launch_few(const CUtensorMap& map_w, const CUtensorMap& map_x, Fp8Params p, int sms, cudaStream_t stream) {
  const int kb_total = (p.K + KBYTES - 1) / KBYTES;
  const int tiles_n = (p.N + TILE_ROWS - 1) / TILE_ROWS, tiles_t = (p.M + BN - 1) / BN;
  // Two CTAs share an SM: K is cut so that the CTAs about fill those slots, at least 4 blocks to a slice, clusters of a power of two.
  long long splits = 2ll * sms / ((long long)tiles_n * tiles_t);
  if (splits > kb_total / 4) splits = kb_total / 4;
  splits = splits >= 8 ? 8 : (splits >= 4 ? 4 : (splits >= 2 ? 2 : 1));
  p.kblocks_per_split = (kb_total + (int)splits - 1) / (int)splits;
  p.splits = (kb_total + p.kblocks_per_split - 1) / p.kblocks_per_split;       // no empty slice
  constexpr int STAGE = (TILE_ROWS + BN) * KBYTES;
  constexpr int FIXED = 1024 + FEW_WINDOW * BN * 4 + 256;
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
  if (tiles_t > 65535) return (int)cudaErrorInvalidConfiguration;
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
  const bool many = M > 64 && tiles_m * tiles_n * 4 >= 3ll * sms;
  CUtensorMap map_x, map_w;
  const int bn = M <= 16 ? 16 : (M <= 32 ? 32 : (M <= 64 ? 64 : 128));
  if (!make_map_bytes(&map_x, X, M, K, ldx, many ? TILE_ROWS : bn) || !make_map_bytes(&map_w, W, N, K, ldw, many ? MANY_BN : TILE_ROWS))
    return (int)cudaErrorInvalidValue;
  if (!many) {
    if (bn == 16) return launch_few<16>(map_w, map_x, p, sms, stream);
    if (bn == 32) return launch_few<32>(map_w, map_x, p, sms, stream);
    if (bn == 64) return launch_few<64>(map_w, map_x, p, sms, stream);
    return launch_few<128>(map_w, map_x, p, sms, stream);
  }
  p.tiles_m = (int)tiles_m; p.tiles_n = (int)tiles_n;
  const size_t smem = 1024 + (size_t)MANY_STAGES * (TILE_ROWS + MANY_BN) * KBYTES + 256;
  static bool set_dev[bspec::kMaxDevices] = {};
  bool& set = set_dev[bspec::current_device()];
  if (!set) {
    const cudaError_t e = cudaFuncSetAttribute(gemm_fp8_many_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return (int)e;
    set = true;
  }
  const long long tiles = tiles_m * tiles_n;
  BSPEC_LAUNCH((gemm_fp8_many_kernel), (unsigned)(tiles < sms ? tiles : sms), MANY_THREADS, smem, stream, map_x, map_w, p);
  return BSPEC_LAUNCH_CHECK();
}

BSPEC_DEFINE_TRACE_SETTER(bspec_trace_set_gemm_fp8)
