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
// maximum and the rounding, so x is read once.  Rows: 8 lanes hold a bfloat16 block as 32-byte pieces (a float32 block takes
// 16 lanes); 128 x 128: one thread block each, 64 numbers per thread.
#include "e4m3.cuh"

using namespace bspec;

namespace {

constexpr int FP8_BLOCK = 128;
constexpr int QUANT_THREADS = 256;

// A piece: 32 bytes of x as they lie (16 numbers of bfloat16, 8 of float32); numbers past `left` are 0.  What a piece costs besides its
// numbers (its place, the block's maximum over the lanes, the scale) is shared by as many as one load can bring.
// VEC: 2 one load of 32 bytes, 1 two of 16, 0 number by number.
template <typename T> struct Piece;
template <> struct Piece<__nv_bfloat16> { static constexpr int N = 16; };
template <> struct Piece<float> { static constexpr int N = 8; };

template <typename T, int VEC>
__device__ __forceinline__ void load_piece(const T* __restrict__ p, int left, uint32_t (&w)[8]) {
  constexpr int N = Piece<T>::N;
  if (VEC && left >= N) {
    if (VEC == 2) {
      asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                   : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]), "=r"(w[4]), "=r"(w[5]), "=r"(w[6]), "=r"(w[7]) : "l"(p));
    } else {
      const uint4 a = __ldg(reinterpret_cast<const uint4*>(p)), b = __ldg(reinterpret_cast<const uint4*>(p) + 1);
      w[0] = a.x; w[1] = a.y; w[2] = a.z; w[3] = a.w;
      w[4] = b.x; w[5] = b.y; w[6] = b.z; w[7] = b.w;
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    if (N == 8) {
      w[i] = i < left ? __float_as_uint(to_f32(p[i])) : 0u;
    } else {
      const uint32_t lo = 2 * i < left ? __float_as_uint(to_f32(p[2 * i])) >> 16 : 0u;
      w[i] = lo | (2 * i + 1 < left ? __float_as_uint(to_f32(p[2 * i + 1])) : 0u);
    }
  }
}
// the bits of the largest magnitude as a float32 number; bfloat16 numbers are compared two at a time
template <int N>
__device__ __forceinline__ uint32_t piece_max(const uint32_t (&w)[8]) {
  uint32_t m = 0u;
#pragma unroll
  for (int i = 0; i < 8; ++i) m = N == 8 ? max(m, w[i] & 0x7fffffffu) : __vmaxu2(m, w[i] & 0x7fff7fffu);
  return N == 8 ? m : max(m << 16, m & 0xffff0000u);
}
// x / s as e4m3: a product with a power of two, exact in either type (but for numbers that become 0)
template <int N>
__device__ __forceinline__ void store_piece(uint8_t* q, const uint32_t (&w)[8], float inv) {
  if (N == 8) {
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(w[i]);
    *reinterpret_cast<uint2*>(q) = make_uint2(to_e4m3x4(v, inv), to_e4m3x4(v + 4, inv));
  } else {
    const __nv_bfloat162 inv2 = __float2bfloat162_rn(inv);
    uint32_t out[4];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const __nv_bfloat162 h = __hmul2(*reinterpret_cast<const __nv_bfloat162*>(&w[i]), inv2);
      const uint32_t r = *reinterpret_cast<const uint32_t*>(&h);
      const uint32_t e = to_e4m3x2(__uint_as_float(r << 16), __uint_as_float(r & 0xffff0000u));
      if (i & 1) out[i / 2] |= e << 16;
      else out[i / 2] = e;
    }
    *reinterpret_cast<uint4*>(q) = make_uint4(out[0], out[1], out[2], out[3]);
  }
}

// Blocks of 1 x 128.  q rows are `ldq` bytes apart, a multiple of 16, so a piece that ends past the row stays in its padding.
template <typename T, int VEC, int U, typename I>         // I: the type that counts blocks; 64-bit divisions took half the kernel's time
__global__ void __launch_bounds__(QUANT_THREADS)
quantize_rows_kernel(const T* __restrict__ x, long long ldx, uint8_t* __restrict__ q, long long ldq, uint8_t* __restrict__ s,
                     I blocks, int K, int KB) {
  bspec::pdl_prologue(80);
  constexpr int N = Piece<T>::N, LANES = FP8_BLOCK / N, AT_ONCE = QUANT_THREADS / LANES;
  const int lane = threadIdx.x % LANES;
  const I first = (I)blockIdx.x * (AT_ONCE * U) + threadIdx.x / LANES;
  uint32_t v[U][8];
  I row[U];
  int kb[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const I b = first + u * AT_ONCE;
    row[u] = b / (I)KB;
    kb[u] = (int)(b - row[u] * (I)KB);
    const int k = kb[u] * FP8_BLOCK + lane * N;
    load_piece<T, VEC>(x + (long long)row[u] * ldx + k, b < blocks ? K - k : 0, v[u]);
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const I b = first + u * AT_ONCE;
    const int k = kb[u] * FP8_BLOCK + lane * N;
    uint32_t m = piece_max<N>(v[u]);
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
    const int code = scale_code(m);
    if (b < blocks) {
      if (k < K) store_piece<N>(q + (long long)row[u] * ldq + k, v[u], inverse_scale(code));
      if (lane == 0) s[b] = (uint8_t)code;
    }
  }
}

// Blocks of 128 x 128 of `batch` matrices of R x K numbers; blockIdx.x = block column, y = block row, z = matrix.
template <typename T, int VEC>
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
  uint32_t v[STEPS][8];
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
  const long long places = (long long)reinterpret_cast<uintptr_t>(x) | (ldx * esz) | (mat_x * esz);
  const int vec = places % 32 == 0 ? 2 : (places % 16 == 0 ? 1 : 0);
  if (block_rows == 1) {
    if (batch > 1 && mat_x != R * ldx) return (int)cudaErrorInvalidValue;
    const long long blocks = batch * R * KB;
    const int at_once = QUANT_THREADS / (FP8_BLOCK * esz / 32);
    // four blocks per lane group keep enough bytes in flight; with fewer blocks than that fills, one each spreads them over the SMs
    const int u = blocks >= (long long)at_once * 4 * 8 * bspec::sm_count() ? 4 : 1;
    const long long grid = (blocks + at_once * u - 1) / (at_once * u);
    if (grid > 0x7fffffff) return (int)cudaErrorInvalidConfiguration;
#define LQ(T, V, U, I) BSPEC_LAUNCH((quantize_rows_kernel<T, V, U, I>), (unsigned)grid, QUANT_THREADS, 0, stream, (const T*)x, ldx, \
                                    (uint8_t*)q, ldq, (uint8_t*)s, (I)blocks, K, KB)
#define LV(T, V)                                                                     \
  do {                                                                               \
    if (u == 1) LQ(T, V, 1, uint32_t);                                               \
    else if (blocks < 0x7fffffffll) LQ(T, V, 4, uint32_t);                           \
    else LQ(T, V, 4, unsigned long long);                                            \
  } while (0)
    if (dtype == BSPEC_F32) { if (vec == 2) LV(float, 2); else if (vec == 1) LV(float, 1); else LV(float, 0); }
    else { if (vec == 2) LV(__nv_bfloat16, 2); else if (vec == 1) LV(__nv_bfloat16, 1); else LV(__nv_bfloat16, 0); }
#undef LV
#undef LQ
    return BSPEC_LAUNCH_CHECK();
  }
  if (block_rows != FP8_BLOCK) return (int)cudaErrorInvalidValue;
  const long long RB = (R + FP8_BLOCK - 1) / FP8_BLOCK;
  if (RB > 65535) return (int)cudaErrorInvalidConfiguration;
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
    if (dtype == BSPEC_F32) { if (vec == 2) LB(float, 2); else if (vec == 1) LB(float, 1); else LB(float, 0); }
    else { if (vec == 2) LB(__nv_bfloat16, 2); else if (vec == 1) LB(__nv_bfloat16, 1); else LB(__nv_bfloat16, 0); }
#undef LB
  }
  return BSPEC_LAUNCH_CHECK();
}

BSPEC_DEFINE_TRACE_SETTER(bspec_trace_set_fp8)
