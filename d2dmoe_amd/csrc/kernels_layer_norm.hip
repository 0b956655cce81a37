// Layer norm of the rows of h = x (or of x + residual, rounded to the storage type), forward and backward.
//
//   m = mean(h)   v = mean((h - m)^2)   r = 1 / sqrt(v + eps)   n = (h - m) r   out = n * weight + bias
//   u = g * weight   grad = r (u - mean(u) - n mean(u n)) + s      (g: gradient of out, s: gradient of the residual stream)
//   grad_weight = sum over rows of g n      grad_bias = sum over rows of g
//
// All sums, the statistics and every intermediate are float32; what is stored in 16 bits is rounded once (h = x + residual
// is such a value: it is the residual stream, an output, and the norm is taken of what the stream holds).
#include "common.hpp"
#include "launch.hpp"

namespace d2dmoe {

namespace {

constexpr int NT = 256;   // threads per workgroup

__device__ inline float wave_sum(float v) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off, kWave);
  return v;
}

// Sum over the workgroup, the same bits in every thread.  `buf` (NT / 64 floats) may be reused after the next barrier.
__device__ inline float block_sum(float v, float* buf) {
  v = wave_sum(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) buf[threadIdx.x >> 6] = v;
  __syncthreads();
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < NT / 64; ++i) s += buf[i];
  return s;
}

template <typename T, typename P>
__global__ __launch_bounds__(NT) void layer_norm_rows_kernel(const T* __restrict__ x, const T* __restrict__ residual,
                                                             const P* __restrict__ weight, const P* __restrict__ bias,
                                                             T* __restrict__ sum, T* __restrict__ out, float* __restrict__ mean,
                                                             float* __restrict__ rstd, int64_t N, int D, float eps) {
  __shared__ float buf[NT / 64];
  const int t = threadIdx.x;
  for (int64_t row = blockIdx.x; row < N; row += gridDim.x) {
    const T* xr = x + row * D;
    const T* rr = residual ? residual + row * D : nullptr;
    auto h = [&](int d) { return rr ? Elem<T>::round(Elem<T>::load(xr + d) + Elem<T>::load(rr + d)) : Elem<T>::load(xr + d); };
    float s = 0.f;
    for (int d = t; d < D; d += NT) s += h(d);
    const float m = block_sum(s, buf) / (float)D;
    // the mean's own rounding error, from the centred values: it matters where the mean is far larger than the spread
    float e = 0.f, q = 0.f;
    for (int d = t; d < D; d += NT) {
      const float c = h(d) - m;
      e += c;
      q = fmaf(c, c, q);
    }
    const float dm = block_sum(e, buf) / (float)D;
    const float var = block_sum(q, buf) / (float)D - dm * dm;
    const float r = 1.f / sqrtf(fmaxf(var, 0.f) + eps);
    for (int d = t; d < D; d += NT) {
      const float v = h(d);
      if (sum) Elem<T>::store(sum + row * D + d, v);
      float o = (v - m - dm) * r;
      if (weight) o *= Elem<P>::load(weight + d);
      if (bias) o += Elem<P>::load(bias + d);
      Elem<T>::store(out + row * D + d, o);
    }
    if (t == 0) {
      if (mean) mean[row] = m + dm;
      if (rstd) rstd[row] = r;
    }
  }
}

template <typename T, typename P>
__global__ __launch_bounds__(NT) void layer_norm_grad_rows_kernel(const T* __restrict__ g, const T* __restrict__ gs,
                                                                  const T* __restrict__ h, const P* __restrict__ weight,
                                                                  const float* __restrict__ mean, const float* __restrict__ rstd,
                                                                  T* __restrict__ grad, int64_t N, int D) {
  __shared__ float buf[NT / 64];
  const int t = threadIdx.x;
  for (int64_t row = blockIdx.x; row < N; row += gridDim.x) {
    const float m = mean[row], r = rstd[row];
    float a = 0.f, b = 0.f;
    for (int d = t; d < D; d += NT) {
      const float u = Elem<T>::load(g + row * D + d) * (weight ? Elem<P>::load(weight + d) : 1.f);
      a += u;
      b = fmaf(u, (Elem<T>::load(h + row * D + d) - m) * r, b);
    }
    a = block_sum(a, buf) / (float)D;
    b = block_sum(b, buf) / (float)D;
    for (int d = t; d < D; d += NT) {
      const float u = Elem<T>::load(g + row * D + d) * (weight ? Elem<P>::load(weight + d) : 1.f);
      const float n = (Elem<T>::load(h + row * D + d) - m) * r;
      float v = r * (u - a - n * b);
      if (gs) v += Elem<T>::load(gs + row * D + d);
      Elem<T>::store(grad + row * D + d, v);
    }
  }
}

// Column sums of g n and g over a slab of rows: workgroup = (64 columns, slab), four rows at a time.
template <typename T>
__global__ __launch_bounds__(NT) void layer_norm_grad_columns_kernel(const T* __restrict__ g, const T* __restrict__ h,
                                                                     const float* __restrict__ mean, const float* __restrict__ rstd,
                                                                     float* __restrict__ partial, int64_t N, int D, int64_t slab) {
  __shared__ float sw[4][64], sb[4][64];
  const int c = threadIdx.x & 63, q = threadIdx.x >> 6;
  const int d = (int)blockIdx.x * 64 + c;
  const int64_t lo = (int64_t)blockIdx.y * slab, hi = (lo + slab < N) ? lo + slab : N;
  float w = 0.f, b = 0.f;
  if (d < D)
    for (int64_t row = lo + q; row < hi; row += 4) {
      const float gv = Elem<T>::load(g + row * D + d);
      w = fmaf(gv, (Elem<T>::load(h + row * D + d) - mean[row]) * rstd[row], w);
      b += gv;
    }
  sw[q][c] = w;
  sb[q][c] = b;
  __syncthreads();
  if (q == 0 && d < D) {
    float* p = partial + (int64_t)blockIdx.y * 2 * D;
    p[d] = (sw[0][c] + sw[1][c]) + (sw[2][c] + sw[3][c]);
    p[D + d] = (sb[0][c] + sb[1][c]) + (sb[2][c] + sb[3][c]);
  }
}

// The slabs' column sums added in order: thread = column of grad_weight (blockIdx.y == 0) or grad_bias.
template <typename P>
__global__ __launch_bounds__(NT) void layer_norm_grad_finish_kernel(const float* __restrict__ partial, P* __restrict__ gw,
                                                                    P* __restrict__ gb, int slabs, int D) {
  const int d = (int)blockIdx.x * NT + threadIdx.x;
  P* out = blockIdx.y ? gb : gw;
  if (d >= D || out == nullptr) return;
  const float* p = partial + (blockIdx.y ? D : 0) + d;
  float s = 0.f;
  for (int i = 0; i < slabs; ++i) s += p[(int64_t)i * 2 * D];
  Elem<P>::store(out + d, s);
}

inline int slab_count(int64_t N) { return (int)(N < 64 ? 1 : (cdiv64(N, 64) < 256 ? cdiv64(N, 64) : 256)); }

template <typename T, typename P>
hipError_t forward_t(const d2dmoe_norm_shape& sh, const void* x, const void* residual, const void* weight, const void* bias, void* sum,
                     void* out, float* mean, float* rstd, hipStream_t s) {
  const unsigned grid = (unsigned)(sh.n_rows < 65536 ? sh.n_rows : 65536);
  hipLaunchKernelGGL((layer_norm_rows_kernel<T, P>), dim3(grid), dim3(NT), 0, s, (const T*)x, (const T*)residual, (const P*)weight,
                     (const P*)bias, (T*)sum, (T*)out, mean, rstd, sh.n_rows, sh.width, sh.eps);
  return hipGetLastError();
}

template <typename T, typename P>
hipError_t backward_t(const d2dmoe_norm_shape& sh, const void* g, const void* gs, const void* h, const void* weight, const float* mean,
                      const float* rstd, void* grad, void* gw, void* gb, void* workspace, hipStream_t s) {
  const int64_t N = sh.n_rows;
  const int D = sh.width;
  if (N > 0 && grad != nullptr) {
    const unsigned grid = (unsigned)(N < 65536 ? N : 65536);
    hipLaunchKernelGGL((layer_norm_grad_rows_kernel<T, P>), dim3(grid), dim3(NT), 0, s, (const T*)g, (const T*)gs, (const T*)h,
                       (const P*)weight, mean, rstd, (T*)grad, N, D);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  if (gw == nullptr && gb == nullptr) return hipSuccess;
  const int slabs = N > 0 ? slab_count(N) : 0;
  if (slabs > 0) {
    hipLaunchKernelGGL((layer_norm_grad_columns_kernel<T>), dim3((unsigned)((D + 63) / 64), (unsigned)slabs), dim3(NT), 0, s,
                       (const T*)g, (const T*)h, mean, rstd, (float*)workspace, N, D, cdiv64(N, slabs));
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  hipLaunchKernelGGL((layer_norm_grad_finish_kernel<P>), dim3((unsigned)((D + NT - 1) / NT), 2), dim3(NT), 0, s,
                     (const float*)workspace, (P*)gw, (P*)gb, slabs, D);
  return hipGetLastError();
}

}  // namespace

size_t layer_norm_workspace_bytes(const d2dmoe_norm_shape& sh) {
  return sh.n_rows > 0 ? (size_t)slab_count(sh.n_rows) * 2 * sh.width * sizeof(float) : 0;
}

// (activations, parameters): both of one type, or 16-bit activations with float32 parameters
#define D2DMOE_NORM_DISPATCH(CALL)                                                              \
  switch (sh.dtype) {                                                                           \
    case D2DMOE_F32: return CALL(float, float);                                                 \
    case D2DMOE_BF16: return sh.param_dtype == D2DMOE_F32 ? CALL(bf16_t, float) : CALL(bf16_t, bf16_t); \
    default: return sh.param_dtype == D2DMOE_F32 ? CALL(f16_t, float) : CALL(f16_t, f16_t);     \
  }

hipError_t launch_layer_norm(const d2dmoe_norm_shape& sh, const void* x, const void* residual, const void* weight, const void* bias,
                             void* sum, void* out, float* mean, float* rstd, hipStream_t s) {
#define D2DMOE_CALL(T, P) forward_t<T, P>(sh, x, residual, weight, bias, sum, out, mean, rstd, s)
  D2DMOE_NORM_DISPATCH(D2DMOE_CALL)
#undef D2DMOE_CALL
}

hipError_t launch_layer_norm_backward(const d2dmoe_norm_shape& sh, const void* g, const void* gs, const void* h, const void* weight,
                                      const float* mean, const float* rstd, void* grad, void* gw, void* gb, void* workspace,
                                      hipStream_t s) {
#define D2DMOE_CALL(T, P) backward_t<T, P>(sh, g, gs, h, weight, mean, rstd, grad, gw, gb, workspace, s)
  D2DMOE_NORM_DISPATCH(D2DMOE_CALL)
#undef D2DMOE_CALL
}

}  // namespace d2dmoe
