// The router's choice of experts from their scores, by one warp: shared by the router kernel and by the kernels of a whole layer.
#pragma once
#include "common.cuh"

namespace bspec {

// the router's rule: bits 0-1 what the scores are, then options
constexpr int ROUTE_SIGMOID = 0, ROUTE_SOFTMAX_TOP = 1, ROUTE_SOFTMAX = 2, ROUTE_SCORES = 3;
constexpr int ROUTE_GROUP_MAX = 4, ROUTE_RENORMALISE = 8;
constexpr int MAX_EXPERTS = 1024;

// What a logit z and an expert's correction b make of its score and of its choice score (before a softmax over all).
__device__ __forceinline__ void route_score(int rule, float z, float b, float* score, float* choice) {
  const int scores = rule & ROUTE_SCORES;
  const bool softmax_top = scores == ROUTE_SOFTMAX_TOP;
  const float s = softmax_top ? z + b : (scores == ROUTE_SOFTMAX ? z : 1.f / (1.f + expf(-z)));
  *score = s;
  *choice = softmax_top ? s : s + b;
}

// The index of the best of v[0 .. n) (the larger value, the lower index among equals; NaN: taken) or 0x7fffffff, by one warp: every lane
// scans its share, two reductions over the lanes find the largest value, in the order of its bits, and the lowest index that holds it.
// A function of its own: what is executed once per token costs the fetch of its instructions more than anything else.  Four numbers at a time:
// one by one each waits for its load (40 of 1,024 experts for a token 75 us instead of 37; up to 128 experts no difference).
static __device__ __noinline__ int best_of(const float* v, int n) {
  unsigned bv = 0u;
  int bi = 0x7fffffff;
#pragma unroll 4
  for (int i = threadIdx.x & 31; i < n; i += 32) {
    const float x = v[i] + 0.f;                  // one zero
    const unsigned b = __float_as_uint(x), key = isnan(x) ? 0u : ((b & 0x80000000u) ? ~b : (b | 0x80000000u));
    if (key > bv) { bv = key; bi = i; }
  }
  const unsigned most = __reduce_max_sync(0xffffffffu, bv);
  return most == 0u ? 0x7fffffff : __reduce_min_sync(0xffffffffu, bv == most ? bi : 0x7fffffff);
}

// One warp chooses the `top` experts of a token and their weights.  sc, ch [E]: scores and choice scores of route_score, in
// shared memory (changed); hs: room for G numbers.  DISTINCT: where no number is left to compare (NaN logits), the lowest
// expert not taken yet instead of expert 0, so that a token never has an expert twice.
template <bool DISTINCT>
__device__ __forceinline__ void choose_experts(float* sc, float* ch, float* hs, const void* __restrict__ corr, int corr_dtype, int E,
                                               int G, int keep, int top, float scale, int rule, int* __restrict__ ids,
                                               float* __restrict__ w) {
  const int lane = threadIdx.x & 31;
  const int scores = rule & ROUTE_SCORES;
  const bool softmax_top = scores == ROUTE_SOFTMAX_TOP;
  if (scores == ROUTE_SOFTMAX) {
    float mx = -INFINITY, sum = 0.f;
#pragma unroll 1
    for (int i = lane; i < E; i += 32) mx = fmaxf(mx, sc[i]);
    mx = warp_max(mx);
#pragma unroll 1
    for (int i = lane; i < E; i += 32) sum += expf(sc[i] - mx);
    sum = warp_sum(sum);
    // without a correction the logits themselves choose (the softmax keeps their order)
#pragma unroll 1
    for (int i = lane; i < E; i += 32) {
      sc[i] = expf(sc[i] - mx) / sum;
      if (corr != nullptr) ch[i] = sc[i] + load_as_f32(corr, corr_dtype, i);
    }
    __syncwarp();
  }
  if (G > 1 && keep < G) {
    const int per = E / G;
#pragma unroll 1
    for (int g = lane; g < G; g += 32) {          // group scores
      float a = -INFINITY, b = -INFINITY;         // the two largest
#pragma unroll 1
      for (int j = 0; j < per; ++j) {
        const float v = ch[g * per + j];
        if (v > a) { b = a; a = v; } else if (v > b) { b = v; }
      }
      hs[g] = per > 1 && !(rule & ROUTE_GROUP_MAX) ? a + b : a;
    }
    __syncwarp();
#pragma unroll 1
    for (int k = 0; k < keep; ++k) {
      const int best = best_of(hs, G);
      if (lane == 0 && best != 0x7fffffff) hs[best] = NAN;      // NaN marks a kept group
      __syncwarp();
    }
#pragma unroll 1
    for (int i = lane; i < E; i += 32)
      if (!isnan(hs[i / per])) ch[i] = -INFINITY;
    __syncwarp();
  }
  // Lane k keeps choice k (and k + 32 ...: `top` beyond the lanes goes through memory); sums run over the choices in their order.
  int mine = 0;
#pragma unroll 1
  for (int k = 0; k < top; ++k) {
    int best = best_of(ch, E);
    if (best == 0x7fffffff) {
      best = 0;
      if (DISTINCT) {
        if (lane == 0)
          for (int j = 0; j < k;) {
            if (ids[j] == best) { ++best; j = 0; } else ++j;
          }
        best = __shfl_sync(0xffffffffu, best, 0);
      }
    }
    if (lane == (k & 31)) mine = best;
    if (lane == 0) {
      ids[k] = best;
      if (top > 32) w[k] = sc[best] * scale;
      ch[best] = NAN;                             // taken
    }
    __syncwarp();
  }
  const bool renormalise = (rule & ROUTE_RENORMALISE) && !softmax_top;
  if (top <= 32) {
    const float s = lane < top ? sc[mine] : -INFINITY;
    float v = s * scale;
    if (renormalise) {
      float sum = 0.f;
#pragma unroll 1
      for (int k = 0; k < top; ++k) sum += __shfl_sync(0xffffffffu, s, k);
      v = s / (sum + 1e-20f) * scale;
    } else if (softmax_top) {                     // the weights: softmax over the chosen logits alone
      const float e = expf(s - warp_max(s));
      float sum = 0.f;
#pragma unroll 1
      for (int k = 0; k < top; ++k) sum += __shfl_sync(0xffffffffu, e, k);
      v = e / sum * scale;
    }
    if (lane < top) w[lane] = v;
    return;
  }
  if (renormalise && lane == 0) {
    float sum = 0.f;
#pragma unroll 1
    for (int k = 0; k < top; ++k) sum += sc[ids[k]];
#pragma unroll 1
    for (int k = 0; k < top; ++k) w[k] = sc[ids[k]] / (sum + 1e-20f) * scale;
  }
  if (softmax_top && lane == 0) {
    float mx = -INFINITY, sum = 0.f;
#pragma unroll 1
    for (int k = 0; k < top; ++k) mx = fmaxf(mx, sc[ids[k]]);
#pragma unroll 1
    for (int k = 0; k < top; ++k) sum += expf(sc[ids[k]] - mx);
#pragma unroll 1
    for (int k = 0; k < top; ++k) w[k] = expf(sc[ids[k]] - mx) / sum * scale;
  }
}

__device__ __forceinline__ float gelu_erf(float v) { return 0.5f * v * (1.f + erff(v * 0.70710678118654752440f)); }

// D += A B, 16 x 8 x 16, bfloat16 with float32 sums: lane l holds rows l / 4 and l / 4 + 8 of A and column l / 4 of B
__device__ __forceinline__ void mma_bf16_16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                               uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

}  // namespace bspec
