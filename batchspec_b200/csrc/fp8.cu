// Matrices in 8-bit floating point (e4m3: 4 exponent bits, 3 of fraction, largest 448) with one power of two per block:
//   s = the smallest 2^j, j >= -127, with max |x| of the block <= 448 s   (1 where every number is 0)
//   q = x / s, rounded to the nearest e4m3 number, ties to even
// Blocks are 128 numbers of one row (activations) or 128 x 128 numbers (weights); the last ones of a row or column may be
// shorter.  s is kept as its exponent in 8 bits (e8m0: 2^(code - 127)).  A power of two instead of max / 448 costs nothing in
// precision (a floating-point format has the same relative step at every scale; only numbers 2^-15 below the block's largest
// lose bits one doubling earlier), and makes the division exact: every q is one rounding of x, whatever computed it, and
// the products' scales multiply without rounding.  A block that holds an infinity or a NaN has s = NaN and q = NaN throughout, so
// that it shows in every product that reads it.
//
// Bound by memory: one read of x (2 or 4 bytes a number), one write of q.  A block's numbers stay in registers between the
// maximum and the rounding, so x is read once.  Rows: 16 lanes hold a bfloat16 block as 16-byte pieces (a float32 block takes
// 32 lanes); 128 x 128: one thread block each, 64 numbers per thread.
#include "e4m3.cuh"

using namespace bspec;

namespace {

constexpr int FP8_BLOCK = 128;
constexpr int QUANT_THREADS = 256;

// A piece: 16 bytes of x as float32 numbers (8 of bfloat16, 4 of float32); numbers past `left` are 0.
template <typename T> struct Piece;
template <> struct Piece<__nv_bfloat16> { static constexpr int N = 8; };
template <> struct Piece<float> { static constexpr int N = 4; };

template <typename T, bool VEC>
__device__ __forceinline__ void load_piece(const T* __restrict__ p, int left, float* v) {
  constexpr int N = Piece<T>::N;
  if (VEC && left >= N) {
    const uint4 raw = __ldg(reinterpret_cast<const uint4*>(p));
    const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (N == 4) {
        v[i] = __uint_as_float(w[i]);
      } else {
        v[2 * i] = __uint_as_float(w[i] << 16);
        v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = i < left ? to_f32(p[i]) : 0.f;
  }
}
template <int N>
__device__ __forceinline__ void store_piece(uint8_t* q, const float* v, float inv) {
  if (N == 8) *reinterpret_cast<uint2*>(q) = make_uint2(to_e4m3x4(v, inv), to_e4m3x4(v + 4, inv));
  else *reinterpret_cast<uint32_t*>(q) = to_e4m3x4(v, inv);
}
template <int N>
__device__ __forceinline__ uint32_t piece_max(const float* v) {
  uint32_t m = 0u;
#pragma unroll
  for (int i = 0; i < N; ++i) m = max(m, __float_as_uint(v[i]) & 0x7fffffffu);
  return m;
}

// Blocks of 1 x 128.  q rows are `ldq` bytes apart, a multiple of 16, so a piece that ends past the row stays in its padding.
template <typename T, bool VEC, int U>
__global__ void __launch_bounds__(QUANT_THREADS)
quantize_rows_kernel(const T* __restrict__ x, long long ldx, uint8_t* __restrict__ q, long long ldq, uint8_t* __restrict__ s,
                     long long blocks, int K, int KB) {
  bspec::pdl_prologue(80);
  constexpr int N = Piece<T>::N, LANES = FP8_BLOCK / N, AT_ONCE = QUANT_THREADS / LANES;
  const int lane = threadIdx.x % LANES;
  const long long first = (long long)blockIdx.x * AT_ONCE * U + threadIdx.x / LANES;
  float v[U][N];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const long long b = first + u * AT_ONCE;
    const long long row = b / KB;
    const int k = (int)(b - row * KB) * FP8_BLOCK + lane * N;
    load_piece<T, VEC>(x + row * ldx + k, b < blocks ? K - k : 0, v[u]);
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const long long b = first + u * AT_ONCE;
    const long long row = b / KB;
    const int kb = (int)(b - row * KB), k = kb * FP8_BLOCK + lane * N;
    uint32_t m = piece_max<N>(v[u]);
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
    const int code = scale_code(m);
    if (b < blocks) {
      if (k < K) store_piece<N>(q + row * ldq + k, v[u], inverse_scale(code));
      if (lane == 0) s[b] = (uint8_t)code;
    }
  }
}

// Blocks of 128 x 128 of `batch` matrices of R x K numbers; blockIdx.x = block column, y = block row, z = matrix.
template <typename T, bool VEC>
__global__ void __launch_bounds__(QUANT_THREADS)
quantize_blocks_kernel(const T* __restrict__ x, long long ldx, long long mat_x, uint8_t* __restrict__ q, long long ldq,
                       uint8_t* __restrict__ s, int R, int K, int RB) {
  bspec::pdl_prologue(81);
  constexpr int N = Piece<T>::N, LANES = FP8_BLOCK / N, ROWS = QUANT_THREADS / LANES, STEPS = FP8_BLOCK / ROWS;
  __shared__ uint32_t warp_max[QUANT_THREADS / 32];
  const int k = blockIdx.x * FP8_BLOCK + (threadIdx.x % LANES) * N;
  const long long matrix = blockIdx.z + (long long)blockIdx.y / RB;      // the row blocks of all matrices lie along y
  const int r0 = (int)(blockIdx.y % RB) * FP8_BLOCK + threadIdx.x / LANES;
  x += matrix * mat_x;
  q += matrix * R * ldq;
  float v[STEPS][N];
  uint32_t m = 0u;
#pragma unroll
  for (int i = 0; i < STEPS; ++i) {
    const int r = r0 + i * ROWS;
    load_piece<T, VEC>(x + r * ldx + k, r < R ? K - k : 0, v[i]);
  }
#pragma unroll
  for (int i = 0; i < STEPS; ++i) m = max(m, piece_max<N>(v[i]));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
  if ((threadIdx.x & 31) == 0) warp_max[threadIdx.x >> 5] = m;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < QUANT_THREADS / 32; ++w) m = max(m, warp_max[w]);
  const int code = scale_code(m);
  const float inv = inverse_scale(code);
#pragma unroll
  for (int i = 0; i < STEPS; ++i) {
    const int r = r0 + i * ROWS;
    if (r < R && k < K) store_piece<N>(q + r * ldq + k, v[i], inv);
  }
  if (threadIdx.x == 0) s[(size_t)blockIdx.y * gridDim.x + blockIdx.x] = (uint8_t)code;
}

}  // namespace

// x: `batch` matrices of R rows of K numbers, rows `ldx` and matrices `mat_x` numbers apart; q: rows `ldq` bytes apart (a multiple
// of 16), matrices R rows apart; s: e8m0 codes, dense [batch][ceil(R / block_rows)][ceil(K / 128)].  block_rows: 1 (then the
// matrices must be R rows apart) or 128.
BSPEC_API int bspec_quantize_fp8(const void* x, int dtype, long long ldx, long long mat_x, void* q, long long ldq, void* s,
                                 long long batch, long long R, int K, int block_rows, cudaStream_t stream) {
  if (batch <= 0 || R <= 0 || K <= 0) return 0;
  if (ldq % 16 != 0 || ldq < K || R > 0x7fffffff - 128 || K > 0x7fffffff - 256) return (int)cudaErrorInvalidValue;
  const int KB = (K + FP8_BLOCK - 1) / FP8_BLOCK, esz = dtype == BSPEC_F32 ? 4 : 2;
  const bool vec = (reinterpret_cast<uintptr_t>(x) & 15) == 0 && (ldx * esz) % 16 == 0 && (mat_x * esz) % 16 == 0;
  if (block_rows == 1) {
    if (batch > 1 && mat_x != R * ldx) return (int)cudaErrorInvalidValue;
    const long long blocks = batch * R * KB;
    const int at_once = QUANT_THREADS / (FP8_BLOCK * esz / 16);
    // four blocks per lane group keep enough bytes in flight; with fewer blocks than that fills, one each spreads them over the SMs
    const int u = blocks >= (long long)at_once * 4 * 8 * bspec::sm_count() ? 4 : 1;
    const long long grid = (blocks + at_once * u - 1) / (at_once * u);
    if (grid > 0x7fffffff) return (int)cudaErrorInvalidConfiguration;
#define LQ(T, V, U) BSPEC_LAUNCH((quantize_rows_kernel<T, V, U>), (unsigned)grid, QUANT_THREADS, 0, stream, (const T*)x, ldx, \
                                 (uint8_t*)q, ldq, (uint8_t*)s, blocks, K, KB)
#define LV(T, V) do { if (u == 4) LQ(T, V, 4); else LQ(T, V, 1); } while (0)
    if (dtype == BSPEC_F32) { if (vec) LV(float, true); else LV(float, false); }
    else { if (vec) LV(__nv_bfloat16, true); else LV(__nv_bfloat16, false); }
#undef LV
#undef LQ
    return BSPEC_LAUNCH_CHECK();
  }
  if (block_rows != FP8_BLOCK) return (int)cudaErrorInvalidValue;
  const long long RB = (R + FP8_BLOCK - 1) / FP8_BLOCK;
  if (batch * RB > 65535 && RB > 65535) return (int)cudaErrorInvalidConfiguration;
  // grids are at most 65,535 high: whole matrices per launch
  const long long per = 65535 / RB;
  for (long long b0 = 0; b0 < batch; b0 += per) {
    const long long nb = batch - b0 < per ? batch - b0 : per;
    dim3 grid(KB, (unsigned)(nb * RB), 1);
    const size_t xo = (size_t)(b0 * mat_x) * esz;
    uint8_t* qb = (uint8_t*)q + b0 * R * ldq;
    uint8_t* sb = (uint8_t*)s + b0 * RB * KB;
#define LB(T, V) BSPEC_LAUNCH((quantize_blocks_kernel<T, V>), grid, QUANT_THREADS, 0, stream, (const T*)((const char*)x + xo), ldx, mat_x, \
                              qb, ldq, sb, (int)R, K, (int)RB)
    if (dtype == BSPEC_F32) { if (vec) LB(float, true); else LB(float, false); }
    else { if (vec) LB(__nv_bfloat16, true); else LB(__nv_bfloat16, false); }
#undef LB
  }
  return BSPEC_LAUNCH_CHECK();
}

BSPEC_DEFINE_TRACE_SETTER(bspec_trace_set_fp8)
