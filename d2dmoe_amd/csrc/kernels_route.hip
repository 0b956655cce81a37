// Routing of tokens to k experts each, from the logits of a learned router, forward and backward.
//
//   s = softmax(z) or 1 / (1 + exp(-z))         scores of the E experts
//   c = s + bias                                what the choice goes by; z itself where neither a bias nor a sum of scores
//                                               enters (the scores rise with z, so the order is the same)
//   groups: E / G consecutive experts each, scored by their largest c or the sum of their two largest; the best stay
//   the k largest c that remain are chosen, ties to the lowest index; experts with z = -inf never; a row with a NaN among
//   its c chooses nothing.  w = scale s, or scale s / (sum of the chosen s).
//
// The choice is made on float64 scores: float32 ones of neighbouring experts coincide or swap about once in ten thousand
// rows, and indices are whole numbers.  The weights are float32.
#include "common.hpp"
#include "launch.hpp"

namespace d2dmoe {

namespace {

constexpr int MAX_E = 1024;
constexpr int PER_LANE = MAX_E / 64;

__device__ inline float wave_sum(float v) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off, kWave);
  return v;
}
__device__ inline double wave_sum(double v) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off, kWave);
  return v;
}
__device__ inline float wave_max(float v) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v = fmaxf(v, __shfl_xor(v, off, kWave));
  return v;
}
__device__ inline bool finite(float v) { return fabsf(v) < INFINITY; }

// One wave per token.
template <typename T>
__global__ __launch_bounds__(64) void route_kernel(const T* __restrict__ logits, const float* __restrict__ bias, T* __restrict__ routing,
                                                   int32_t* __restrict__ indices, float* __restrict__ weights,
                                                   int32_t* __restrict__ counts, int64_t N, int E, int K, int softmax, int G, int kept,
                                                   int top2, int renorm, float scale) {
  __shared__ double s_by[MAX_E];
  __shared__ float s_z[MAX_E];
  __shared__ int s_idx[MAX_E];
  const int lane = threadIdx.x;
  const bool direct = bias == nullptr && !(G > 1 && top2);
  for (int64_t row = blockIdx.x; row < N; row += gridDim.x) {
    const T* zr = logits + row * E;
    float z[PER_LANE];
    double by[PER_LANE];
    bool bad = false;
    float top = -INFINITY;
#pragma unroll
    for (int j = 0; j < PER_LANE; ++j) {
      const int e = lane + 64 * j;
      z[j] = e < E ? Elem<T>::load(zr + e) : -INFINITY;
      if (z[j] != z[j] || (softmax && z[j] == INFINITY)) bad = true;
      top = fmaxf(top, z[j]);
    }
    top = wave_max(top);
    if (!finite(top)) top = 0.f;
    if (direct) {
#pragma unroll
      for (int j = 0; j < PER_LANE; ++j) by[j] = z[j];
    } else {
      double total = 0.0;
#pragma unroll
      for (int j = 0; j < PER_LANE; ++j) {
        by[j] = softmax ? exp((double)z[j] - (double)top) : 1.0 / (1.0 + exp(-(double)z[j]));
        total += by[j];
      }
      if (softmax) total = wave_sum(total);
#pragma unroll
      for (int j = 0; j < PER_LANE; ++j) {
        const int e = lane + 64 * j;
        if (softmax) by[j] /= total;
        if (bias != nullptr && e < E) by[j] += (double)bias[e];
      }
    }
#pragma unroll
    for (int j = 0; j < PER_LANE; ++j) {
      by[j] = (z[j] == -INFINITY) ? -(double)INFINITY : by[j] + 0.0;   // + 0.0: the two zeros are one value
      if (by[j] != by[j]) bad = true;
    }
    if (__ballot(bad) != 0ull) {
#pragma unroll
      for (int j = 0; j < PER_LANE; ++j) by[j] = -(double)INFINITY;
    }
    if (G > 1) {
      const int size = E / G;
      __syncthreads();
#pragma unroll
      for (int j = 0; j < PER_LANE; ++j)
        if (lane + 64 * j < E) s_by[lane + 64 * j] = by[j];
      __syncthreads();
      double of_run[PER_LANE];
#pragma unroll
      for (int j = 0; j < PER_LANE; ++j) {
        const int g = lane + 64 * j;
        double a = -(double)INFINITY, b = a;
        if (g < G)
          for (int i = 0; i < size; ++i) {
            const double v = s_by[g * size + i];
            if (v > a) { b = a; a = v; } else if (v > b) b = v;
          }
        of_run[j] = (top2 && b > -(double)INFINITY) ? a + b : a;
      }
      __syncthreads();
#pragma unroll
      for (int j = 0; j < PER_LANE; ++j)
        if (lane + 64 * j < G) s_by[lane + 64 * j] = of_run[j];
      __syncthreads();
#pragma unroll
      for (int j = 0; j < PER_LANE; ++j) {
        const int e = lane + 64 * j;
        if (e < E) {
          const int g = e / size;
          const double mine = s_by[g];
          int ahead = 0;
          for (int o = 0; o < G; ++o) ahead += (s_by[o] > mine || (s_by[o] == mine && o < g)) ? 1 : 0;
          if (ahead >= kept) by[j] = -(double)INFINITY;
        }
      }
    }
    // the k best, one after the other
    __syncthreads();
    for (int i = 0; i < K; ++i) {
      double v = -(double)INFINITY;
      int at = MAX_E;
#pragma unroll
      for (int j = 0; j < PER_LANE; ++j)
        if (by[j] > v) { v = by[j]; at = lane + 64 * j; }
#pragma unroll
      for (int off = 32; off > 0; off >>= 1) {
        const double ov = __shfl_xor(v, off, kWave);
        const int oa = __shfl_xor(at, off, kWave);
        if (ov > v || (ov == v && oa < at)) { v = ov; at = oa; }
      }
      const bool there = v > -(double)INFINITY;
      if (lane == 0) {
        s_idx[i] = there ? at : -1;
        s_z[i] = there ? Elem<T>::load(zr + at) : -INFINITY;
        if (there && counts != nullptr) atomicAdd(counts + at, 1);
      }
#pragma unroll
      for (int j = 0; j < PER_LANE; ++j)
        if (lane + 64 * j == at) by[j] = -(double)INFINITY;
    }
    __syncthreads();
    // scores of the chosen relative to the best of them (renormalised: no score underflows that way), their sum
    float ref = -INFINITY;
    for (int i = lane; i < K; i += 64) ref = fmaxf(ref, softmax ? s_z[i] : fminf(s_z[i], 0.f));
    ref = wave_max(ref);
    ref = !finite(ref) ? 0.f : ref;
    if (!renorm) ref = softmax ? top : 0.f;
    float part = 0.f;
    for (int i = lane; i < K; i += 64) {
      const float zi = s_z[i];
      const float w = softmax ? expf(zi - ref) : expf(fminf(zi, 0.f) - ref) / (1.f + expf(-fabsf(zi)));
      s_z[i] = s_idx[i] >= 0 ? w : 0.f;
      part += s_z[i];
    }
    float total = 1.f;
    if (renorm) {
      total = wave_sum(part);
    } else if (softmax) {
      float all = 0.f;
#pragma unroll
      for (int j = 0; j < PER_LANE; ++j) all += expf(z[j] - top);
      total = wave_sum(all);
    }
    __syncthreads();
    float mine[PER_LANE];
#pragma unroll
    for (int j = 0; j < PER_LANE; ++j) mine[j] = 0.f;
    for (int i = 0; i < K; ++i) {
      const int at = s_idx[i];
      const float w = at >= 0 ? scale * (s_z[i] / total) : 0.f;
      if (lane == (i & 63)) {
        if (indices) indices[row * K + i] = at;
        if (weights) weights[row * K + i] = w;
      }
#pragma unroll
      for (int j = 0; j < PER_LANE; ++j)
        if (lane + 64 * j == at) mine[j] = w;
    }
    if (routing) {
#pragma unroll
      for (int j = 0; j < PER_LANE; ++j)
        if (lane + 64 * j < E) Elem<T>::store(routing + row * E + lane + 64 * j, mine[j]);
    }
    __syncthreads();
  }
}

// Gradient of the logits from the gradient q of the weights (by expert and / or by place): one wave per token.
//   renormalised: w_j (q_j - sum q_i p_i), p = w / scale, times (1 - s_j) for sigmoid scores; q less its first value, which
//   changes nothing and keeps the difference exact where one expert has nearly all the weight
//   softmax as it is: scale s_j (q_j [chosen] - sum q_i s_i)       sigmoid as it is: scale q_j s_j (1 - s_j)
template <typename T>
__global__ __launch_bounds__(64) void route_grad_kernel(const T* __restrict__ logits, const int32_t* __restrict__ indices,
                                                        const T* __restrict__ g_routing, const float* __restrict__ g_weights,
                                                        T* __restrict__ grad, int64_t N, int E, int K, int softmax, int renorm,
                                                        float scale) {
  __shared__ float s_d[MAX_E];
  const int lane = threadIdx.x;
  for (int64_t row = blockIdx.x; row < N; row += gridDim.x) {
    const T* zr = logits + row * E;
    const int32_t* ir = indices + row * K;
    auto q_of = [&](int i, int at) {
      return (g_routing ? Elem<T>::load(g_routing + row * E + at) : 0.f) + (g_weights ? g_weights[row * K + i] : 0.f);
    };
    auto at_of = [&](int i) { const int at = ir[i]; return (at >= 0 && at < E) ? at : -1; };
    for (int e = lane; e < E; e += 64) s_d[e] = 0.f;
    const int first = at_of(0);
    bool mine = false;
    for (int i = lane; i < K; i += 64) mine = mine || at_of(i) >= 0;
    const bool some = __ballot(mine) != 0ull;
    float ref = -INFINITY, total = 1.f;
    const bool whole = softmax && !renorm;
    if (whole) {
      for (int e = lane; e < E; e += 64) ref = fmaxf(ref, Elem<T>::load(zr + e));
    } else {
      for (int i = lane; i < K; i += 64)
        if (at_of(i) >= 0) ref = fmaxf(ref, softmax ? Elem<T>::load(zr + ir[i]) : fminf(Elem<T>::load(zr + ir[i]), 0.f));
    }
    ref = wave_max(ref);
    if (!finite(ref) || (!softmax && !renorm)) ref = 0.f;
    auto score = [&](float z) { return softmax ? expf(z - ref) : expf(fminf(z, 0.f) - ref) / (1.f + expf(-fabsf(z))); };
    if (whole || renorm) {
      float part = 0.f;
      if (whole) {
        for (int e = lane; e < E; e += 64) part += score(Elem<T>::load(zr + e));
      } else {
        for (int i = lane; i < K; i += 64)
          if (at_of(i) >= 0) part += score(Elem<T>::load(zr + ir[i]));
      }
      total = wave_sum(part);
    }
    const float q0 = (renorm && first >= 0) ? q_of(0, first) : 0.f;
    float dot = 0.f;
    if (whole || renorm) {
      for (int i = lane; i < K; i += 64)
        if (at_of(i) >= 0) dot += score(Elem<T>::load(zr + ir[i])) / total * (q_of(i, ir[i]) - q0);
      dot = wave_sum(dot);
    }
    __syncthreads();
    for (int i = lane; i < K; i += 64)
      if (at_of(i) >= 0) {
        const float z = Elem<T>::load(zr + ir[i]);
        float d = scale * (score(z) / total) * (q_of(i, ir[i]) - q0 - (renorm ? dot : 0.f));
        if (!softmax) d /= 1.f + expf(z);
        atomicAdd(&s_d[ir[i]], d);
      }
    __syncthreads();
    for (int e = lane; e < E; e += 64) {
      float d = s_d[e];
      if (whole && some) d -= scale * (score(Elem<T>::load(zr + e)) / total) * dot;
      Elem<T>::store(grad + row * E + e, d);
    }
    __syncthreads();
  }
}

template <typename T>
hipError_t forward_t(const d2dmoe_route_shape& sh, const void* logits, const float* bias, void* routing, int32_t* indices, float* weights,
                     int32_t* counts, hipStream_t s) {
  const unsigned grid = (unsigned)(sh.n_tokens < (1 << 20) ? sh.n_tokens : (1 << 20));
  hipLaunchKernelGGL(route_kernel<T>, dim3(grid), dim3(64), 0, s, (const T*)logits, bias, (T*)routing, indices, weights, counts,
                     sh.n_tokens, sh.n_experts, sh.k, sh.scoring == D2DMOE_SCORE_SOFTMAX, sh.n_groups, sh.kept_groups,
                     sh.group_score == D2DMOE_GROUP_TOP2, sh.renormalise, sh.scale);
  return hipGetLastError();
}

template <typename T>
hipError_t backward_t(const d2dmoe_route_shape& sh, const void* logits, const int32_t* indices, const void* g_routing,
                      const float* g_weights, void* grad, hipStream_t s) {
  const unsigned grid = (unsigned)(sh.n_tokens < (1 << 20) ? sh.n_tokens : (1 << 20));
  hipLaunchKernelGGL(route_grad_kernel<T>, dim3(grid), dim3(64), 0, s, (const T*)logits, indices, (const T*)g_routing, g_weights,
                     (T*)grad, sh.n_tokens, sh.n_experts, sh.k, sh.scoring == D2DMOE_SCORE_SOFTMAX, sh.renormalise, sh.scale);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_route_topk(const d2dmoe_route_shape& sh, const void* logits, const float* bias, void* routing, int32_t* indices,
                             float* weights, int32_t* counts, hipStream_t s) {
  if (counts != nullptr) {
    const hipError_t e = launch_fill_i32(counts, sh.n_experts, 0, s);
    if (e != hipSuccess || sh.n_tokens == 0) return e;
  }
  switch (sh.dtype) {
    case D2DMOE_F32: return forward_t<float>(sh, logits, bias, routing, indices, weights, counts, s);
    case D2DMOE_BF16: return forward_t<bf16_t>(sh, logits, bias, routing, indices, weights, counts, s);
    default: return forward_t<f16_t>(sh, logits, bias, routing, indices, weights, counts, s);
  }
}

hipError_t launch_route_topk_backward(const d2dmoe_route_shape& sh, const void* logits, const int32_t* indices, const void* g_routing,
                                      const float* g_weights, void* grad, hipStream_t s) {
  switch (sh.dtype) {
    case D2DMOE_F32: return backward_t<float>(sh, logits, indices, g_routing, g_weights, grad, s);
    case D2DMOE_BF16: return backward_t<bf16_t>(sh, logits, indices, g_routing, g_weights, grad, s);
    default: return backward_t<f16_t>(sh, logits, indices, g_routing, g_weights, grad, s);
  }
}

}  // namespace d2dmoe
