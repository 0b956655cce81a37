// Layer norm of the rows of h = x (or of x + residual, rounded to the storage type), forward and backward.
//
//   m = mean(h)   v = mean((h - m)^2)   r = 1 / sqrt(v + eps)   n = (h - m) r   out = n * weight + bias
//   u = g * weight   grad = r (u - mean(u) - n mean(u n)) + s      (g: gradient of out, s: gradient of the residual stream)
//   grad_weight = sum over rows of g n      grad_bias = sum over rows of g
//
// All sums, the statistics and every intermediate are float32; what is stored in 16 bits is rounded once (h = x + residual
// is such a value: it is the residual stream, an output, and the norm is taken of what the stream holds).
//
// Two kernels per direction: one that keeps a row in registers (from one 16-byte vector up to 32768 16-bit or 16384 float32
// values forward, half of that backward), one that passes over it again for every use (other widths).
#include "launch.hpp"
#include "mfma_common.hpp"
#include "team.hpp"

namespace d2dmoe {

namespace {

constexpr int NT = 256;   // threads per workgroup

// ---------------------------------------------------------------------------------------------------------------------
// A row in registers.  TPR threads per row: a part of a wave (8, 16 or 32 lanes: narrow rows, several per wave), one wave, or a
// whole workgroup of 256, 512 or 1024 (the only ones with a barrier), CH vectors of 16 bytes each.  All but the last of the CH
// are whole; in the last one a thread may lie behind the row's end (it reads the row's first vector and drops it) or across it
// (it reads the row's last whole vector, of which it counts the elements nobody else has; the others are computed twice and
// stored twice, with the same bits).  Rows may begin at any element: the loads and stores make no claim on alignment.
//
// Bound by HBM: a row is read once and written once.  bf16 with residual, 50432 x 768: 60 us, 5.1 TB/s (this card copies at
// 4.9 to 5.5 TB/s); 32768 x 4096 with statistics: 195 us, 5.5 TB/s; 65536 x 64: 6.7 us, 5.0 TB/s.  With one row per workgroup
// and a pass over it for each use the first was 259 us.
// ---------------------------------------------------------------------------------------------------------------------
template <typename T> constexpr int kVec = 16 / (int)sizeof(T);

template <typename T> __device__ __forceinline__ void decode(const uint4& raw, float (&v)[kVec<T>]) {
  const uint32_t q[4] = {raw.x, raw.y, raw.z, raw.w};
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = __uint_as_float(q[i]);
  } else {
    constexpr bool F16 = Elem<T>::dtype == D2DMOE_F16;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = dec16<F16>(q[i] & 0xffffu);
      v[2 * i + 1] = dec16_hi<F16>(q[i]);
    }
  }
}
template <typename T> __device__ __forceinline__ uint4 encode(const float (&v)[kVec<T>]) {
  uint32_t q[4];
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < 4; ++i) q[i] = __float_as_uint(v[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) q[i] = enc16x2<Elem<T>::dtype == D2DMOE_F16>(v[2 * i], v[2 * i + 1]);
  }
  return make_uint4(q[0], q[1], q[2], q[3]);
}
template <typename T> __device__ __forceinline__ uint4 load16(const T* p) {
  uint4 r;
  __builtin_memcpy(&r, p, 16);
  return r;
}
template <typename T> __device__ __forceinline__ void store16(T* p, const uint4& r) { __builtin_memcpy(p, &r, 16); }

// V parameters as float32
template <typename P, int V> __device__ __forceinline__ void load_params(const P* p, float (&v)[V]) {
  P raw[V];
  __builtin_memcpy(raw, p, sizeof(raw));
#pragma unroll
  for (int j = 0; j < V; ++j) v[j] = Elem<P>::load(raw + j);
}

// Sums of two values over the TPR threads of a row.  `turn` alternates between calls: the next call writes the other half of
// buf, and the one after comes behind a barrier that every reader of this half has passed, so one barrier each is enough.
template <int TPR> constexpr int kWaves = TPR > 64 ? TPR / 64 : 1;   // per row
template <int TPR>
__device__ __forceinline__ void row_sum(float& a, float& b, float (*buf)[2][kWaves<TPR>], int& turn) {
  a = team_sum<(TPR < 64 ? TPR : 64)>(a);
  b = team_sum<(TPR < 64 ? TPR : 64)>(b);
  if constexpr (TPR > 64) {
    float (*half)[kWaves<TPR>] = buf[turn];
    turn ^= 1;
    if ((threadIdx.x & 63) == 0) {
      half[0][threadIdx.x >> 6] = a;
      half[1][threadIdx.x >> 6] = b;
    }
    lds_barrier();
    a = b = 0.f;
#pragma unroll
    for (int i = 0; i < TPR / 64; ++i) {
      a += half[0][i];
      b += half[1][i];
    }
  }
}

// The rows of a workgroup: ROWS at a time, RPW of them per wave.  The loop over them is uniform for a wave: `row` is its first
// one, and a lane whose own row lies behind the end works on the last row and stores nothing.
template <int TPR> constexpr int kRows = TPR < NT ? NT / TPR : 1;
template <int TPR> constexpr int kRowsPerWave = TPR < 64 ? 64 / TPR : 1;
template <int TPR> __device__ __forceinline__ int64_t first_row() {
  return (int64_t)blockIdx.x * kRows<TPR> + (TPR < NT ? __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) * kRowsPerWave<TPR> : 0);
}

struct NormForward {
  const void *x, *residual, *weight, *bias;
  void *sum, *out;
  float *mean, *rstd;
  int64_t N;
  int D;
  float eps;
};

template <typename T, typename P, int TPR, int CH, bool RES>
__global__ __launch_bounds__(TPR < NT ? NT : TPR) void layer_norm_kernel(const NormForward A) {
  constexpr int V = kVec<T>, RPW = kRowsPerWave<TPR>;
  __shared__ float buf[2][2][kWaves<TPR>];
  int turn = 0;
  const int t = threadIdx.x % TPR;
  const int D = A.D;
  int at[CH];
#pragma unroll
  for (int c = 0; c < CH; ++c) at[c] = (c * TPR + t) * V;
  const int over = at[CH - 1] + V - D;                      // elements of the last vector behind the row's end
  const int skip = over <= 0 ? 0 : (over >= V ? V : over);  // ... which its first `skip` elements stand for
  if (skip == V) at[CH - 1] = 0;
  else if (skip > 0) at[CH - 1] = D - V;
  float w[CH][V], b[CH][V];
#pragma unroll
  for (int c = 0; c < CH; ++c) {
#pragma unroll
    for (int j = 0; j < V; ++j) { w[c][j] = 1.f; b[c][j] = 0.f; }
    if (A.weight) load_params<P, V>((const P*)A.weight + at[c], w[c]);
    if (A.bias) load_params<P, V>((const P*)A.bias + at[c], b[c]);
  }
  const float inv_d = 1.f / (float)D;
  const int64_t step = (int64_t)gridDim.x * kRows<TPR>;
  const int sub = RPW > 1 ? (threadIdx.x & 63) / TPR : 0;
  uint4 xr[CH], rr[CH];
  auto request = [&](int64_t wave_row) __attribute__((always_inline)) {
    const int64_t r = RPW > 1 && wave_row + sub >= A.N ? A.N - 1 : wave_row + sub;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      xr[c] = load16((const T*)A.x + r * D + at[c]);
      if (RES) rr[c] = load16((const T*)A.residual + r * D + at[c]);
    }
  };
  int64_t wave_row = first_row<TPR>();
  if (wave_row < A.N) request(wave_row);
  for (; wave_row < A.N; wave_row += step) {
    const int64_t row = wave_row + sub;
    const bool live = RPW == 1 || row < A.N;
    float h[CH][V];
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      decode<T>(xr[c], h[c]);
      if (RES) {
        float r[V];
        decode<T>(rr[c], r);
#pragma unroll
        for (int j = 0; j < V; ++j) h[c][j] += r[j];
        const uint4 packed = encode<T>(h[c]);               // the stream as it is stored is what the norm sees
        decode<T>(packed, h[c]);
        if (A.sum && live && (c < CH - 1 || skip < V)) store16((T*)A.sum + row * D + at[c], packed);
      }
    }
    if (wave_row + step < A.N) request(wave_row + step);    // the next row travels while this one is worked on
    float s = 0.f, none = 0.f;
#pragma unroll
    for (int c = 0; c < CH; ++c)
#pragma unroll
      for (int j = 0; j < V; ++j) s += (c < CH - 1 || j >= skip) ? h[c][j] : 0.f;
    row_sum<TPR>(s, none, buf, turn);
    const float m = s * inv_d;
    // the mean's own rounding error, from the centred values: it matters where the mean is far larger than the spread
    float e = 0.f, q = 0.f;
#pragma unroll
    for (int c = 0; c < CH; ++c)
#pragma unroll
      for (int j = 0; j < V; ++j) {
        h[c][j] -= m;
        const float v = (c < CH - 1 || j >= skip) ? h[c][j] : 0.f;
        e += v;
        q = fmaf(v, v, q);
      }
    row_sum<TPR>(e, q, buf, turn);
    const float dm = e * inv_d;
    const float r = 1.f / sqrtf(fmaxf(q * inv_d - dm * dm, 0.f) + A.eps);
#pragma unroll
    for (int c = 0; c < CH; ++c) {
#pragma unroll
      for (int j = 0; j < V; ++j) h[c][j] = fmaf((h[c][j] - dm) * r, w[c][j], b[c][j]);
      if (live && (c < CH - 1 || skip < V)) store16((T*)A.out + row * D + at[c], encode<T>(h[c]));
    }
    if (t == 0 && live) {
      if (A.mean) A.mean[row] = m + dm;
      if (A.rstd) A.rstd[row] = r;
    }
  }
}

struct NormBackward {
  const void *g, *gs, *h, *weight;
  const float *mean, *rstd;
  void* grad;
  float* partial;   // [workgroup][2][D]: column sums of the workgroup's rows, or NULL
  void *gw, *gb;    // a single workgroup's column sums are the result: either may be NULL
  int64_t N;
  int D;
};

// The column sums of grad_weight and grad_bias ride along: every thread owns its columns for all the rows it sees, so they
// cost two accumulators per element and no traffic until the end.  Rows are requested one ahead (the workgroups are as many
// as two per CU hold, so registers are plenty).  Bound by HBM: 32768 x 4096 bf16 with the residual's gradient 210 us, 5.1 TB/s;
// 16384 x 768 22 us, 4.6 TB/s, behind which the finishing launch takes 3.9 us.  Workgroups of eight rows at a time (half as
// many sums to finish) took the same time at 768 and 2 us more at 4097 x 1280, where they are too few to fill the machine.
template <typename T, typename P, int TPR, int CH>
__global__ __launch_bounds__(TPR < NT ? NT : TPR, TPR == 1024 ? 1 : 2) void layer_norm_grad_kernel(const NormBackward A) {
  constexpr int V = kVec<T>, RPW = kRowsPerWave<TPR>, Q = 2 * CH * V / 4;
  constexpr bool AHEAD = TPR < 1024 && CH < 4;   // (registers: the row is requested when it is due)
  __shared__ float buf[2][2][kWaves<TPR>];
  __shared__ float4 sums[TPR <= 64 ? 2 : 1][TPR <= 64 ? Q : 1][64];
  int turn = 0;
  const int t = threadIdx.x % TPR;
  const int D = A.D;
  int at[CH];
#pragma unroll
  for (int c = 0; c < CH; ++c) at[c] = (c * TPR + t) * V;
  const int over = at[CH - 1] + V - D;
  const int skip = over <= 0 ? 0 : (over >= V ? V : over);
  if (skip == V) at[CH - 1] = 0;
  else if (skip > 0) at[CH - 1] = D - V;
  float w[CH][V], cs[2][CH][V];
#pragma unroll
  for (int c = 0; c < CH; ++c) {
#pragma unroll
    for (int j = 0; j < V; ++j) { w[c][j] = 1.f; cs[0][c][j] = 0.f; cs[1][c][j] = 0.f; }
    if (A.weight) load_params<P, V>((const P*)A.weight + at[c], w[c]);
  }
  const float inv_d = 1.f / (float)D;
  const int64_t step = (int64_t)gridDim.x * kRows<TPR>;
  const int sub = RPW > 1 ? (threadIdx.x & 63) / TPR : 0;
  uint4 gr[CH], hr[CH], sr[CH];
  float m, r;
  auto request = [&](int64_t wave_row) __attribute__((always_inline)) {
    const int64_t k = RPW > 1 && wave_row + sub >= A.N ? A.N - 1 : wave_row + sub;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      gr[c] = load16((const T*)A.g + k * D + at[c]);
      hr[c] = load16((const T*)A.h + k * D + at[c]);
    }
    m = A.mean[k];
    r = A.rstd[k];
  };
  int64_t wave_row = first_row<TPR>();
  if (AHEAD && wave_row < A.N) request(wave_row);
  for (; wave_row < A.N; wave_row += step) {
    if (!AHEAD) request(wave_row);
    const bool live = RPW == 1 || wave_row + sub < A.N;
    const int64_t row = live ? wave_row + sub : A.N - 1;
    if (A.gs) {
#pragma unroll
      for (int c = 0; c < CH; ++c) sr[c] = load16((const T*)A.gs + row * D + at[c]);
    }
    float g[CH][V], n[CH][V];
    const float rs = r;
    float a = 0.f, b = 0.f;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      decode<T>(gr[c], g[c]);
      decode<T>(hr[c], n[c]);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        n[c][j] = (n[c][j] - m) * rs;
        cs[0][c][j] = live ? fmaf(g[c][j], n[c][j], cs[0][c][j]) : cs[0][c][j];
        cs[1][c][j] = live ? cs[1][c][j] + g[c][j] : cs[1][c][j];
        g[c][j] *= w[c][j];
        const float u = (c < CH - 1 || j >= skip) ? g[c][j] : 0.f;
        a += u;
        b = (c < CH - 1 || j >= skip) ? fmaf(u, n[c][j], b) : b;
      }
    }
    if (AHEAD && wave_row + step < A.N) request(wave_row + step);
    row_sum<TPR>(a, b, buf, turn);
    a *= inv_d;
    b *= inv_d;
    if (A.grad) {
#pragma unroll
      for (int c = 0; c < CH; ++c) {
        float s[V];
        if (A.gs) decode<T>(sr[c], s);
        if (!AHEAD) {                           // from the row's own registers once more, rather than held across the barrier
          // (the empty asm makes them new values to the compiler, which would otherwise keep the decoded ones)
          asm volatile("" : "+v"(gr[c].x), "+v"(gr[c].y), "+v"(gr[c].z), "+v"(gr[c].w));
          asm volatile("" : "+v"(hr[c].x), "+v"(hr[c].y), "+v"(hr[c].z), "+v"(hr[c].w));
          decode<T>(gr[c], g[c]);
          decode<T>(hr[c], n[c]);
#pragma unroll
          for (int j = 0; j < V; ++j) {
            n[c][j] = (n[c][j] - m) * rs;
            g[c][j] *= w[c][j];
          }
        }
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const float v = rs * (g[c][j] - a - n[c][j] * b);
          g[c][j] = A.gs ? v + s[j] : v;
        }
        if (live && (c < CH - 1 || skip < V)) store16((T*)A.grad + row * D + at[c], encode<T>(g[c]));
      }
    }
  }
  if (A.partial == nullptr && A.gw == nullptr && A.gb == nullptr) return;
  float* flat = &cs[0][0][0];
  if constexpr (TPR <= 64) {
    // the wave's rows first, where it has several
#pragma unroll
    for (int off = TPR; off < 64; off <<= 1)
#pragma unroll
      for (int q = 0; q < 4 * Q; ++q) flat[q] += __shfl_xor(flat[q], off, kWave);
    // the waves' sums: (0 + 2) + (1 + 3), through LDS in the lanes' own order
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    auto leave = [&](int to) __attribute__((always_inline)) {
#pragma unroll
      for (int q = 0; q < Q; ++q) sums[to][q][lane] = make_float4(flat[4 * q], flat[4 * q + 1], flat[4 * q + 2], flat[4 * q + 3]);
    };
    auto add = [&](int from) __attribute__((always_inline)) {
#pragma unroll
      for (int q = 0; q < Q; ++q) {
        const float4 v = sums[from][q][lane];
        flat[4 * q] += v.x; flat[4 * q + 1] += v.y; flat[4 * q + 2] += v.z; flat[4 * q + 3] += v.w;
      }
    };
    if (wave >= 2) leave(wave - 2);
    __syncthreads();
    if (wave < 2) add(wave);
    __syncthreads();
    if (wave == 1) leave(0);
    __syncthreads();
    if (wave != 0 || lane >= TPR) return;
    add(0);
  }
  if (A.partial == nullptr) {
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      P* out = (P*)(k == 0 ? A.gw : A.gb);
      if (out == nullptr) continue;
#pragma unroll
      for (int c = 0; c < CH; ++c)
#pragma unroll
        for (int j = 0; j < V; ++j)
          if (c < CH - 1 || j >= skip) Elem<P>::store(out + at[c] + j, cs[k][c][j]);
    }
    return;
  }
  float* out = A.partial + (int64_t)blockIdx.x * 2 * D;
#pragma unroll
  for (int k = 0; k < 2; ++k)
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      float* p = out + k * D + at[c];
      if (c < CH - 1 || skip == 0) {
        __builtin_memcpy(p, cs[k][c], sizeof(cs[k][c]));
      } else {
#pragma unroll
        for (int j = 0; j < V; ++j)
          if (j >= skip) p[j] = cs[k][c][j];
      }
    }
}

// The workgroups' column sums added in a fixed order.  Workgroup = 32 of the 2 D columns, 32 threads per column: thread q adds
// the workgroups q, q + 32, ...; then the 32 in order.
template <typename P>
__global__ __launch_bounds__(1024) void layer_norm_grad_finish_kernel(const float* __restrict__ partial, P* __restrict__ gw,
                                                                      P* __restrict__ gb, int parts, int D) {
  __shared__ float part[32][33];
  const int c = threadIdx.x & 31, q = threadIdx.x >> 5;
  const int d = (int)blockIdx.x * 32 + c;
  float s = 0.f;
  if (d < 2 * D) {
#pragma unroll 8
    for (int i = q; i < parts; i += 32) s += partial[(int64_t)i * 2 * D + d];
  }
  part[q][c] = s;
  __syncthreads();
  if (threadIdx.x < 32 && d < 2 * D) {
    float v = 0.f;
#pragma unroll
    for (int i = 0; i < 32; ++i) v += part[i][c];
    P* out = d < D ? gw : gb;
    if (out != nullptr) Elem<P>::store(out + (d < D ? d : d - D), v);
  }
}

// ---------------------------------------------------------------------------------------------------------------------
// Any width: one workgroup per row, a pass over it for every use.
// ---------------------------------------------------------------------------------------------------------------------
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

inline int slab_count(int64_t N) { return (int)(N < 64 ? 1 : (cdiv64(N, 64) < 256 ? cdiv64(N, 64) : 256)); }

// Threads per row and vectors per thread for a width, or TPR = 0 where the row does not fit: as few lanes as one vector each is
// enough for (65536 rows of 64 bf16: 23 us with a wave each), then a wave per row as long as `most` vectors per thread are
// enough, then a workgroup of 256, of 1024.  Forward four; backward three, whose sums and the row ahead make 240 of the 256
// registers that two waves per SIMD leave each thread.  There 1024 threads have 128, room for one vector (8192 x 8192 bf16:
// 110 us), and wider rows take 512 threads: 8192 x 12288 bf16 160 us (5.0 TB/s), with 1024 threads of two vectors, which spilled,
// 471; four vectors spill up to 21 registers and wait for their row (8192 x 16384: 250 us, 4.3 TB/s).  Forward, 1024 threads have
// no room for four vectors either (up to 23 registers spilled without a residual, 61 with one): 8192 x 32768 bf16 runs at 4.4 TB/s
// and 3.6 with a residual; three vectors spill with one (up to 17) and reach 5.0 TB/s all the same, two 5.3.
struct RowPlan { int tpr, ch; };
template <typename T> RowPlan row_plan(int D, bool forward) {
  constexpr int V = kVec<T>;
  if (D < V) return {0, 0};
  const int vectors = (D + V - 1) / V, most = forward ? 4 : 3;
  if (vectors <= 32) return {vectors <= 8 ? 8 : vectors <= 16 ? 16 : 32, 1};
  if (vectors <= 64 * most) return {64, (vectors + 63) / 64};
  if (vectors <= 256 * most) return {256, (vectors + 255) / 256};
  if (vectors <= 1024 * (forward ? 4 : 1)) return {1024, (vectors + 1023) / 1024};
  if (!forward && vectors <= 512 * 4) return {512, (vectors + 511) / 512};
  return {0, 0};
}

// Workgroups of the row kernels: enough to fill the machine's 256 CUs, each with as many rows as that leaves it.  (A constant:
// the workspace and the order of the column sums depend on it.)
inline unsigned row_grid(int64_t N, int rows, int per_cu) {
  const int64_t need = cdiv64(N, rows), most = (int64_t)256 * per_cu;
  return (unsigned)(need < most ? need : most);
}
// The gradient's: every workgroup leaves 2 D sums behind, so each takes four rows per wave or row team at least.
inline int grad_parts(const d2dmoe_norm_shape& sh, int tpr) { return (int)row_grid(sh.n_rows, 4 * (tpr < NT ? NT / tpr : 1), tpr >= 512 ? 1 : 2); }

template <typename T, typename P, int TPR, int CH>
hipError_t forward_rows(const NormForward& A, hipStream_t s) {
  constexpr int threads = TPR < NT ? NT : TPR;
  const unsigned grid = row_grid(A.N, kRows<TPR>, TPR == 1024 ? 2 : 5);
  if (A.residual) hipLaunchKernelGGL((layer_norm_kernel<T, P, TPR, CH, true>), dim3(grid), dim3(threads), 0, s, A);
  else hipLaunchKernelGGL((layer_norm_kernel<T, P, TPR, CH, false>), dim3(grid), dim3(threads), 0, s, A);
  return hipGetLastError();
}

template <typename T, typename P, int TPR, int CH>
hipError_t backward_rows(const NormBackward& A, unsigned grid, hipStream_t s) {
  hipLaunchKernelGGL((layer_norm_grad_kernel<T, P, TPR, CH>), dim3(grid), dim3(TPR < NT ? NT : TPR), 0, s, A);
  return hipGetLastError();
}

#define D2DMOE_ROW_DISPATCH(PLAN, CALL, EXTRA)      \
  switch (PLAN.tpr * 8 + PLAN.ch) {                 \
    case 8 * 8 + 1: e = CALL(8, 1); break;          \
    case 16 * 8 + 1: e = CALL(16, 1); break;        \
    case 32 * 8 + 1: e = CALL(32, 1); break;        \
    case 64 * 8 + 1: e = CALL(64, 1); break;        \
    case 64 * 8 + 2: e = CALL(64, 2); break;        \
    case 64 * 8 + 3: e = CALL(64, 3); break;        \
    case 256 * 8 + 1: e = CALL(256, 1); break;      \
    case 256 * 8 + 2: e = CALL(256, 2); break;      \
    case 256 * 8 + 3: e = CALL(256, 3); break;      \
    EXTRA                                           \
    default: e = CALL(1024, 1); break;              \
  }

template <typename T, typename P>
hipError_t forward_t(const d2dmoe_norm_shape& sh, const void* x, const void* residual, const void* weight, const void* bias, void* sum,
                     void* out, float* mean, float* rstd, hipStream_t s) {
  const RowPlan plan = row_plan<T>(sh.width, true);
  hipError_t e;
  if (plan.tpr != 0) {
    const NormForward A{x, residual, weight, bias, sum, out, mean, rstd, sh.n_rows, sh.width, sh.eps};
#define D2DMOE_ROWS(TPR, CH) forward_rows<T, P, TPR, CH>(A, s)
    D2DMOE_ROW_DISPATCH(plan, D2DMOE_ROWS, case 64 * 8 + 4: e = D2DMOE_ROWS(64, 4); break;
                        case 256 * 8 + 4: e = D2DMOE_ROWS(256, 4); break;
                        case 1024 * 8 + 2: e = D2DMOE_ROWS(1024, 2); break; case 1024 * 8 + 3: e = D2DMOE_ROWS(1024, 3); break;
                        case 1024 * 8 + 4: e = D2DMOE_ROWS(1024, 4); break;)
#undef D2DMOE_ROWS
    return e;
  }
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
  const bool columns = gw != nullptr || gb != nullptr;
  int parts = 0;                       // partial column sums in the workspace
  hipError_t e = hipSuccess;
  const RowPlan plan = row_plan<T>(D, false);
  if (N > 0 && plan.tpr != 0) {
    parts = grad_parts(sh, plan.tpr);
    const bool one = parts == 1;       // (16 rows of 768: one launch of two)
    const NormBackward A{g, gs, h, weight, mean, rstd, grad, columns && !one ? (float*)workspace : nullptr, one ? gw : nullptr,
                         one ? gb : nullptr, N, D};
#define D2DMOE_ROWS(TPR, CH) backward_rows<T, P, TPR, CH>(A, (unsigned)parts, s)
    D2DMOE_ROW_DISPATCH(plan, D2DMOE_ROWS, case 512 * 8 + 3: e = D2DMOE_ROWS(512, 3); break;
                        case 512 * 8 + 4: e = D2DMOE_ROWS(512, 4); break;)
#undef D2DMOE_ROWS
  } else if (N > 0) {
    if (grad != nullptr) {
      const unsigned grid = (unsigned)(N < 65536 ? N : 65536);
      hipLaunchKernelGGL((layer_norm_grad_rows_kernel<T, P>), dim3(grid), dim3(NT), 0, s, (const T*)g, (const T*)gs, (const T*)h,
                         (const P*)weight, mean, rstd, (T*)grad, N, D);
      e = hipGetLastError();
    }
    if (e == hipSuccess && columns) {
      parts = slab_count(N);
      hipLaunchKernelGGL((layer_norm_grad_columns_kernel<T>), dim3((unsigned)((D + 63) / 64), (unsigned)parts), dim3(NT), 0, s,
                         (const T*)g, (const T*)h, mean, rstd, (float*)workspace, N, D, cdiv64(N, parts));
      e = hipGetLastError();
    }
  }
  if (e != hipSuccess || !columns || (N > 0 && plan.tpr != 0 && parts == 1)) return e;
  hipLaunchKernelGGL((layer_norm_grad_finish_kernel<P>), dim3((unsigned)((2 * D + 31) / 32)), dim3(1024), 0, s,
                     (const float*)workspace, (P*)gw, (P*)gb, parts, D);
  return hipGetLastError();
}

}  // namespace

size_t layer_norm_workspace_bytes(const d2dmoe_norm_shape& sh) {
  if (sh.n_rows <= 0) return 0;
  const RowPlan plan = sh.dtype == D2DMOE_F32 ? row_plan<float>(sh.width, false) : row_plan<bf16_t>(sh.width, false);
  const int parts = plan.tpr != 0 ? grad_parts(sh, plan.tpr) : slab_count(sh.n_rows);
  return (size_t)parts * 2 * sh.width * sizeof(float);
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
