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
#include "team.hpp"

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
// exp as one multiplication and the hardware's 2^x: relative error (1.5 |v| + 2) u.  For sums over a row and for choices; what
// is stored as a weight goes through expf.
__device__ inline float quick_exp(float v) { return __builtin_amdgcn_exp2f(v * 1.44269504088896341f); }
__device__ inline bool finite(float v) { return fabsf(v) < INFINITY; }

// =====================================================================================================
// Teams: L lanes per token, 64 / L tokens per wave, V consecutive experts per lane (L V >= E, L >= k).
//
// A row is read once, as one or two 16-byte loads per lane.  Each lane sorts its V keys (choice, then lowest index: 32 bits
// that compare as unsigned numbers, 64 for float32 logits); the k best are then the team's largest list head, taken k times: a
// maximum over the team in lane-permute instructions, and the winner's list moves up by one.  Place i ends in lane i, which
// computes its weight; the dense row goes through a zeroed LDS tile of the wave's tokens, so that it leaves as whole 16-byte
// stores.  Waves share nothing, so there are no barriers.
//
// Choices that are not the logits themselves are made on float32 scores first.  With u = 2^-24 a score is off by at most 30 u
// (softmax: its own exponential 3 |v| s + 3 s, the row's sum 44 s -- less than that where s is near 1 -- all of which the
// other score of a pair shares; sigmoid: 4.2 u) and its sum with a bias by u |c| more.  Where two choices whose order matters
// lie within 2^-19 + 2^-22 |c| of each other (sums of two scores: twice that) -- places next to one another in the list, the
// last place and the first one left out, a group that stays and one that goes -- the wave repeats its choice on float64
// scores; and so does a group whose two large biases cancel.  A row or two in a thousand do for logits of spread 1.5 and for
// sigmoid scores.  Their waves finish last: 16384 x 256 takes 16.8 us with a bias, of which 4.5 us are that tail, and 30 us with
// one (all zeros, 16-bit logits) that leaves every wave in doubt.  The doubt does not follow a score's size, so the softmax of
// many small logits, whose scores lie closer together, has about half its waves in it: logits of spread 0.1 with a zero bias take
// 16.4, 29.8 and 49.8 us at 16384 x 128, 256 and 512 float32, logits of spread 1.5 12.1, 17.6 and 25.6 us.
//
// Bound by vector instructions, not by memory: 388 per wave of four tokens at 128 experts and 8 places in bf16, 789 per wave
// of two at 256 in float32 with groups and a bias.  50432 x 128 bf16: 11 us (29 MB: 5.6 us at this card's copy rate);
// 16384 x 256 float32 in groups: 20 us (35 MB: 6.7 us), 131072 x 256: 86 us.  Before: one wave per token with float64
// throughout, 396 us for the first and 206 us for the second.
// =====================================================================================================
constexpr int WAVES = 4;   // per workgroup

// LDS written by some lanes of a wave and read by others of the same wave
__device__ inline void wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

// order-preserving bits of a float; 0 is below every number and stands for "not to be chosen"
__device__ inline uint32_t order_bits(float v) {
  const uint32_t u = __float_as_uint(v);
  return u ^ ((uint32_t)((int32_t)u >> 31) | 0x80000000u);
}
__device__ inline float from_order_bits(uint32_t o) { return __uint_as_float((o & 0x80000000u) ? (o ^ 0x80000000u) : ~o); }

// A lane's V choices as keys that compare as unsigned numbers, the larger choice first and the lower index first among equal
// ones; 0 stands for "not to be chosen".
//   WIDE   a float32 logit: its order-preserving bits and the index, 32 bits each
//   HALF   a 16-bit logit: the same in 32 bits together, exact
//   FIXED  a score (plus bias): 22 bits of fixed point over the row's range and the index in 32 bits; below kNone (a zero in
//          those bits) it stands for "not to be chosen".  A step is 2^-22 of the range, an eighth of what float32 scores leave
//          in doubt anyway where the range is one; choices closer than that doubt and two steps are told apart in float64.
//          The range's ends keep a margin, since the multiplication and addition that makes a step number shares one rounding
//          error of up to a quarter of the doubt among the row's numbers: a doubt of kMargin steps goes to float64 as a whole.
enum { WIDE, HALF, FIXED };
constexpr float kTop = (1 << 22) - 1, kMargin = 1 << 15;
constexpr uint32_t kNone = MAX_E;

template <typename T, int V, int KIND> struct Keys {
  uint32_t hi[V], lo[V];   // (hi: WIDE)
  __device__ __forceinline__ void set(int j, float c, int e) {           // WIDE, HALF
    const bool on = c > -INFINITY;
    if constexpr (KIND == WIDE) {
      hi[j] = on ? order_bits(c) : 0u;
      lo[j] = on ? (uint32_t)(MAX_E - e) : 0u;
    } else {
      uint32_t u;                      // the 16 bits of the logit, on top
      if constexpr (Elem<T>::dtype == D2DMOE_F16) u = (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)c) << 16;
      else u = __float_as_uint(c);
      const uint32_t o = (u ^ ((uint32_t)((int32_t)u >> 31) | 0x80000000u)) & 0xffff0000u;
      lo[j] = on ? (o | (uint32_t)(MAX_E - e)) : 0u;
    }
  }
  __device__ __forceinline__ void set_fixed(int j, float c, int e, float scale, float offset) {   // (-inf and NaN: 0)
    lo[j] = (uint32_t)__builtin_amdgcn_fmed3f(fmaf(c, scale, offset), 0.f, kTop) << 10 | (uint32_t)(MAX_E - 1 - e);
  }
  __device__ __forceinline__ void order(int i, int k) {   // larger key to place i
    const uint32_t al = lo[i], bl = lo[k];
    if constexpr (KIND == WIDE) {
      const uint32_t ah = hi[i], bh = hi[k];
      const bool swap = ((uint64_t)bh << 32 | bl) > ((uint64_t)ah << 32 | al);
      const uint32_t ch = swap ? bh : ah, dh = swap ? ah : bh, cl = swap ? bl : al, dl = swap ? al : bl;
      hi[i] = ch; hi[k] = dh; lo[i] = cl; lo[k] = dl;
    } else {
      const uint32_t big = al > bl ? al : bl, small = al > bl ? bl : al;
      lo[i] = big; lo[k] = small;
    }
  }
  __device__ __forceinline__ void sort() {   // descending (odd-even merge network)
#pragma unroll
    for (int a = 1; a < V; a *= 2)
#pragma unroll
      for (int b = a; b >= 1; b /= 2)
#pragma unroll
        for (int j = b % a; j + b < V; j += 2 * b)
#pragma unroll
          for (int i = 0; i < (b < V - j - b ? b : V - j - b); ++i)
            if ((i + j) / (2 * a) == (i + j + b) / (2 * a)) order(i + j, i + j + b);
  }
  // The team's largest key, which leaves its lane's list.  WIDE: h is its choice, and `won` the lane it was in -- the lowest of
  // those whose list starts with that choice, and so with the lowest index -- found in scalar instructions: the lowest bit
  // of each L-bit field of the ballot (no field is empty, so the subtraction does not borrow from the next); l is the lane's
  // own head.  Otherwise l is the whole key.
  template <int L> __device__ __forceinline__ void take(uint32_t& h, uint32_t& l, bool& won) {
    if constexpr (KIND == WIDE) {
      constexpr uint64_t ones = L == 4 ? 0x1111111111111111ull : L == 8 ? 0x0101010101010101ull : L == 16 ? 0x0001000100010001ull
                                                                      : L == 32 ? 0x0000000100000001ull : 1ull;
      h = team_max_u<L>(hi[0]);
      const uint64_t m = __ballot(hi[0] == h);
      won = __builtin_amdgcn_inverse_ballot_w64(m & ~(m - ones));
      l = lo[0];
    } else {
      h = l = team_max_u<L>(lo[0]);
      won = lo[0] == l;
    }
#pragma unroll
    for (int j = 0; j < V; ++j) {      // (values, not places, to choose from: the lists stay in registers)
      const uint32_t lc = lo[j], ln = j + 1 < V ? lo[j + 1 < V ? j + 1 : j] : 0u;
      lo[j] = won ? ln : lc;
      if constexpr (KIND == WIDE) {
        const uint32_t hc = hi[j], hn = j + 1 < V ? hi[j + 1 < V ? j + 1 : j] : 0u;
        hi[j] = won ? hn : hc;
      }
    }
  }
  static __device__ __forceinline__ int expert(uint32_t l) {
    return KIND == FIXED ? MAX_E - 1 - (int)(l & 1023u) : MAX_E - (int)(KIND == WIDE ? l : (l & 0xffffu));
  }
  static __device__ __forceinline__ float logit(uint32_t h) {            // WIDE, HALF
    if constexpr (KIND == WIDE) {
      return from_order_bits(h);
    } else {
      const uint32_t o = h >> 16;
      const uint16_t u = (uint16_t)((o & 0x8000u) ? (o ^ 0x8000u) : ~o);
      T raw;
      __builtin_memcpy(&raw, &u, 2);
      return Elem<T>::load(&raw);
    }
  }
};

__device__ inline float larger(float a, float b) { return max1(a, b); }
__device__ inline double larger(double a, double b) { return fmax(a, b); }
__device__ inline float smaller(float a, float b) { return min1(a, b); }
__device__ inline double smaller(double a, double b) { return fmin(a, b); }

// V consecutive elements from any address; those at `count` and beyond read as `fill`
template <int V, typename T>
__device__ inline void load_run(const T* p, int count, float fill, float (&v)[V]) {
  if (count >= V) {
    T raw[V];
    __builtin_memcpy(raw, p, sizeof(raw));
#pragma unroll
    for (int j = 0; j < V; ++j) v[j] = Elem<T>::load(raw + j);
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j) v[j] = j < count ? Elem<T>::load(p + j) : fill;
  }
}
template <int V, typename T>
__device__ inline void store_run(T* p, int count, const float (&v)[V]) {
  if (count >= V) {
    T raw[V];
#pragma unroll
    for (int j = 0; j < V; ++j) Elem<T>::store(raw + j, v[j]);
    __builtin_memcpy(p, raw, sizeof(raw));
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j)
      if (j < count) Elem<T>::store(p + j, v[j]);
  }
}

struct RouteArgs {
  const float* bias; int32_t* indices; float* weights; int32_t* counts;
  int64_t N; int E, K, softmax, G, kept, top2, renorm; float scale;
  int size;                             // experts per group
  float inv_size, inv_G, inv_lanes;     // 1 / size, 1 / G, 1 / (lanes per group) where groups are whole lanes
};

// a / b for 0 <= a < 4096 and b <= 1024 from a float32 1 / b: (a + 1/2) / b is at least 1 / (2 b) away from a whole number, the
// product's error below 4096 * 2^-22
__device__ inline int small_div(int a, float inv_b) { return (int)(((float)a + 0.5f) * inv_b); }

// Which of the T G groups of a wave's tokens stay, from their scores: flags in stays[].  NEAR: scores closer than near_abs +
// near_rel |score| leave the order in doubt; returns whether it was (the flags do not matter then).  Otherwise exact, ties to
// the lowest group.
template <typename C, int T, bool NEAR>
__device__ __forceinline__ bool rank_groups(const C* score, uint8_t* stays, const RouteArgs& A, C near_abs, C near_rel) {
  const int lane = threadIdx.x & 63, G = A.G;
  bool doubt = false;
  for (int p = lane; p < T * G; p += 64) {
    const int first = small_div(p, A.inv_G) * G, g = p - first;
    const C* all = score + first;
    const C mine = all[g];
    if constexpr (NEAR) {
      const C size_of = mine < 0 ? -mine : mine;
      const C by = size_of < (C)INFINITY ? near_abs + near_rel * size_of : (C)0;
      const C above = mine + by, below = mine - by;
      int surely = 0, maybe = -1;                       // ahead of this one (which is within its own reach)
#pragma unroll 4
      for (int o = 0; o < G; ++o) {
        const C v = all[o];
        surely += v > above ? 1 : 0;
        maybe += v >= below ? 1 : 0;
      }
      if (mine > -(C)INFINITY && surely < A.kept && maybe >= A.kept) doubt = true;
      stays[p] = surely < A.kept ? 1 : 0;
    } else {
      int ahead = 0;
#pragma unroll 4
      for (int o = 0; o < G; ++o) {
        const C v = all[o];
        ahead += (v > mine || (v == mine && o < g)) ? 1 : 0;
      }
      stays[p] = ahead < A.kept ? 1 : 0;
    }
  }
  return __ballot(doubt) != 0ull;
}

// A group's score from its two largest choices.  (Two of float32's lowest value, as masks use it, overflow: more than none still.)
__device__ inline float add_best(float a, float b) { return max1(a + b, -0x1.fffffep127f); }
__device__ inline double add_best(double a, double b) { return a + b; }
template <typename C>
__device__ __forceinline__ C group_score(const RouteArgs& A, C a, C b) { return (A.top2 && b > -(C)INFINITY) ? add_best(a, b) : a; }
// Two large choices of opposite signs: each is off by u times its own size, which their small sum does not show, so the sum's place
// is in doubt wherever it lies.  Below that line two such scores differ by up to 50 u from the scores they add (see above), 8 u
// and 5 u of the sum's size from its two roundings and the choices': within the 64 u and 8 u of a score that rank_groups asks for.
__device__ __forceinline__ bool cancels(const RouteArgs& A, float a, float b) {
  return A.top2 && b > -INFINITY && fabsf(a) + fabsf(b) > fmaf(1.5f, fabsf(a + b), 4.f);
}
__device__ __forceinline__ bool cancels(const RouteArgs&, double, double) { return false; }   // (the scores that decide)

// The scores of the T G groups from the choices in tile[] (T rows of E); returns whether one of them cancels.
template <typename C, int T>
__device__ __forceinline__ bool score_groups(const C* tile, C* score, const RouteArgs& A) {
  const C low = -(C)INFINITY;
  bool lost = false;
  for (int p = threadIdx.x & 63; p < T * A.G; p += 64) {
    const C* q = tile + p * A.size;       // token-major, groups in order: p counts both
    C a = low, b = low;
    for (int i = 0; i < A.size; ++i) {
      const C v = q[i];
      b = larger(b, smaller(a, v));
      a = larger(a, v);
    }
    score[p] = group_score(A, a, b);
    lost = lost || cancels(A, a, b);
  }
  return lost;
}

// Drops the groups that do not stay from by[] (-inf); returns whether a group's place was in doubt (NEAR).  tile: T E values,
// score: T G values of the wave's own LDS.
template <bool NEAR, int V, int L, typename C>
__device__ __forceinline__ bool keep_groups(C (&by)[V], const RouteArgs& A, C near_abs, C near_rel, C* tile, C* score) {
  constexpr int T = 64 / L;
  const int lane = threadIdx.x & 63, tl = lane & (L - 1), team = lane / L;
  const int size = A.size, G = A.G, e0 = tl * V;
  const C low = -(C)INFINITY;
  bool lost = false;
  wave_sync();
  if (size % V == 0) {
    // whole lanes per group: the two largest of ever longer runs of lanes, up to the group's end, in its first lane
    C a = low, b = low;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      b = larger(b, smaller(a, by[j]));
      a = larger(a, by[j]);
    }
    const int lanes = size / V, of = small_div(tl, A.inv_lanes), pos = tl - of * lanes;
    for (int off = 1; off < lanes; off <<= 1) {
      const C oa = __shfl_down(a, off, kWave), ob = __shfl_down(b, off, kWave);
      if (pos + off < lanes) {
        b = larger(larger(b, ob), smaller(a, oa));
        a = larger(a, oa);
      }
    }
    if (pos == 0 && e0 < A.E) {
      score[team * G + of] = group_score(A, a, b);
      if constexpr (NEAR) lost = cancels(A, a, b);
    }
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j)
      if (e0 + j < A.E) tile[team * A.E + e0 + j] = by[j];
    wave_sync();
    lost = score_groups<C, T>(tile, score, A);
  }
  wave_sync();
  uint8_t* stays = (uint8_t*)tile;
  bool doubt = rank_groups<C, T, NEAR>(score, stays, A, near_abs, near_rel);
  if constexpr (NEAR) doubt = doubt || __ballot(lost) != 0ull;
  wave_sync();
  int g = small_div(e0, A.inv_size);
  if (size % V == 0) {
    const bool out = e0 >= A.E || !stays[team * G + g];
#pragma unroll
    for (int j = 0; j < V; ++j) by[j] = out ? low : by[j];
  } else {
    int r = e0 - g * size;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      if (e0 + j < A.E && !stays[team * G + g]) by[j] = low;
      if (++r == size) { r = 0; ++g; }
    }
  }
  wave_sync();
  return doubt;
}

// The choice on float64 scores: returns place tl's expert (or -1).  Few waves come here, but a launch waits for its last one,
// and the kernel's occupancy is set by its widest part.  So: one exponential at a time (eight interleaved take 100 registers),
// from LDS to LDS, then the choices in registers and the maxima over the team by lane permutes, as in the float32 choice.
// tiles[]: T rows of E, T rows of G scores.
template <int V, int L, bool GROUPS>
__device__ __forceinline__ int choose_exactly(const float (&z)[V], bool row_bad, const RouteArgs& A, double* tiles) {
  constexpr int TOK = 64 / L;
  const int lane = threadIdx.x & 63, tl = lane & (L - 1), team = lane / L, e0 = tl * V;
  const int end = e0 + V < A.E ? e0 + V : A.E;
  const double low = -(double)INFINITY;
  double* tile = tiles + team * A.E;
  wave_sync();
  float top = -INFINITY;
#pragma unroll
  for (int j = 0; j < V; ++j) {
    if (e0 + j < A.E) tile[e0 + j] = (double)z[j];
    top = fmaxf(top, z[j]);
  }
  top = team_max<L>(top);
  if (!finite(top)) top = 0.f;
  double total = 0.0;
#pragma unroll 1
  for (int e = e0; e < end; ++e) {
    const double v = tile[e];
    const double x = exp(A.softmax ? v - (double)top : -v);
    tile[e] = A.softmax ? x : 1.0 / (1.0 + x);
    total += x;
  }
  if (A.softmax) total = team_sum<L>(total);
  double by[V];
  float b[V];
  if (A.bias != nullptr) load_run<V>(A.bias + e0, A.E - e0, 0.f, b);
#pragma unroll
  for (int j = 0; j < V; ++j) {
    double c = e0 + j < A.E ? tile[e0 + j] : 0.0;
    if (A.softmax) c /= total;
    if (A.bias != nullptr) c += (double)b[j];
    by[j] = (z[j] == -INFINITY || row_bad) ? low : c + 0.0;
  }
  if constexpr (GROUPS) keep_groups<false, V, L>(by, A, 0.0, 0.0, tiles, tiles + TOK * A.E);
  int place = -1;
#pragma unroll 1
  for (int i = 0; i < A.K; ++i) {
    double v = low;
    int at = MAX_E;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const double c = by[j];
      at = c > v ? e0 + j : at;
      v = larger(v, c);
    }
    // the team's largest: order-preserving halves, then the lowest index
    const uint64_t u = (uint64_t)__double_as_longlong(v);
    const uint64_t o = u ^ ((uint64_t)((int64_t)u >> 63) | 0x8000000000000000ull);
    const uint32_t h = team_max_u<L>((uint32_t)(o >> 32));
    const bool first = (uint32_t)(o >> 32) == h;
    const uint32_t m = team_max_u<L>(first ? (uint32_t)o : 0u);
    const uint32_t l = team_max_u<L>((first && (uint32_t)o == m && v > low) ? (uint32_t)(2 * MAX_E - at) : 0u);
    const int best = l != 0u ? 2 * MAX_E - (int)l : -1;
    if (tl == i) place = best;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const double c = by[j];
      by[j] = e0 + j == best ? low : c;
    }
  }
  return place;
}

// What the choice goes by, each an instance of its own: the logits (no score, no doubt), or scores (with a bias, or with sums
// of them for the groups); among all experts, or within groups.
enum { BY_LOGIT = 0, BY_SCORE = 1, IN_GROUPS = 2 };

template <typename T, int V, int L, int MODE>
__global__ __launch_bounds__(WAVES * 64) void route_team_kernel(const T* __restrict__ logits, T* __restrict__ routing, const RouteArgs A,
                                                                int wave_lds) {
  extern __shared__ __align__(16) char lds_raw[];
  constexpr int TOK = 64 / L;
  const int lane = threadIdx.x & 63, tl = lane & (L - 1), team = lane / L, e0 = tl * V;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);    // uniform: rows and addresses are scalars
  char* lds = lds_raw + wave * wave_lds;
  if (A.counts != nullptr && blockIdx.x == 0)                 // (filled by the pass over the indices behind this launch)
    for (int e = threadIdx.x; e < A.E; e += WAVES * 64) A.counts[e] = 0;
  constexpr bool direct = !(MODE & BY_SCORE), groups = (MODE & IN_GROUPS) != 0;
  const int have = A.E - e0;                                  // experts from e0 on (<= 0: an idle lane)
  const int64_t tile = (int64_t)blockIdx.x * WAVES + wave;
  if (tile * TOK < A.N) {
    const int rows = (int)((A.N - tile * TOK < TOK) ? A.N - tile * TOK : TOK);
    const bool live = team < rows;
    const T* zt = logits + tile * TOK * A.E;                  // the wave's rows
    const int row_at = team * A.E;
    float z[V];
    load_run<V>(zt + row_at + e0, live ? have : 0, -INFINITY, z);
    bool bad = false;
    float top = -INFINITY;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      bad = bad || z[j] != z[j];
      top = max1(top, z[j]);
    }
    if (A.softmax) bad = bad || top == INFINITY;
    const bool whole = A.softmax && !(A.renorm && direct);    // the row's softmax is needed, not only its order
    float sum = 1.f;
    float p[V];
    if (whole) {
      top = team_max<L>(top);
      if (!finite(top)) top = 0.f;
      sum = 0.f;
#pragma unroll
      for (int j = 0; j < V; ++j) {
        p[j] = quick_exp(z[j] - top);
        sum += p[j];
      }
      sum = team_sum<L>(sum);
    }
    float by[V];
    if (direct) {
#pragma unroll
      for (int j = 0; j < V; ++j) by[j] = z[j] + 0.f;         // + 0: the two zeros are one value
    } else {
      const float inv = __builtin_amdgcn_rcpf(sum);
      float b[V];
      if (A.bias != nullptr) load_run<V>(A.bias + e0, have, 0.f, b);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        float c = A.softmax ? p[j] * inv : __builtin_amdgcn_rcpf(1.f + quick_exp(-z[j]));
        if (A.bias != nullptr) c += b[j];
        by[j] = z[j] == -INFINITY ? -INFINITY : c + 0.f;
        bad = bad || by[j] != by[j];
      }
    }
    bad = team_any<L>(bad);
#pragma unroll
    for (int j = 0; j < V; ++j) by[j] = bad ? -INFINITY : by[j];
    bool doubt = false;
    if constexpr (groups)
      doubt = keep_groups<!direct, V, L>(by, A, 0x1p-18f, 0x1p-21f, (float*)lds, (float*)lds + TOK * A.E);
    using K = Keys<T, V, !direct ? FIXED : (sizeof(T) == 4 ? WIDE : HALF)>;
    K keys;
    float near_by = 0.f;                                      // FIXED: the doubt in steps
    bool windowed = false;
    if constexpr (direct) {
#pragma unroll
      for (int j = 0; j < V; ++j) keys.set(j, by[j], e0 + j);
    } else {
      float most = -INFINITY, least = INFINITY;
#pragma unroll
      for (int j = 0; j < V; ++j) {
        most = max1(most, by[j]);
        least = min1(least, by[j] > -INFINITY ? by[j] : INFINITY);
      }
      most = team_max<L>(most);
      least = -team_max<L>(-least);
      // Further apart than scores are: masks (the type's lowest value, -1e9) in the bias.  Only the uppermost part is told apart
      // then, and a place that falls below it or next to its end is in doubt (16384 x 256 with a tenth masked so: 31 us without, 17 us).
      windowed = !(most - least <= 64.f) && most > -INFINITY;
      least = windowed ? most - 4.f : least;
      const float range = most - least;
      const float scale = fminf((kTop - 2.f * kMargin) * __builtin_amdgcn_rcpf(fmaxf(range, 0x1p-80f)), 0x1p100f);
      const float offset = kMargin - least * scale;
      near_by = (0x1p-19f + 0x1p-22f * fmaxf(fabsf(most), fabsf(least))) * scale + 2.f;
      if (most > -INFINITY && !(near_by < kMargin)) doubt = true;   // (also a NaN: a bias of +inf)
#pragma unroll
      for (int j = 0; j < V; ++j) keys.set_fixed(j, by[j], e0 + j, scale, offset);
    }
    keys.sort();
    uint32_t mine_hi = 0, mine_lo = 0;                        // place tl's key
    uint32_t hi, lo;
    bool won;
    constexpr bool wide = direct && sizeof(T) == 4;
    uint32_t* places = (uint32_t*)lds + team * A.K;           // wide keys: the winner's lane leaves its index here
    if constexpr (wide) wave_sync();
    for (int i = 0; i < A.K; ++i) {
      keys.template take<L>(hi, lo, won);
      if constexpr (wide) {
        if (won) places[i] = lo;
        mine_hi = tl == i ? hi : mine_hi;
      } else {
        mine_lo = tl == i ? lo : mine_lo;
      }
    }
    if constexpr (wide) {
      wave_sync();
      if (tl < A.K) mine_lo = places[tl];
    } else {
      mine_hi = mine_lo;
    }
    int at = (tl < A.K && mine_hi >= (direct ? 1u : kNone)) ? K::expert(mine_lo) : -1;
    float zi = -INFINITY;
    if constexpr (direct) {
      if (at >= 0) zi = K::logit(mine_hi);
    } else {
      // places next to each other, and the last one with the first that was left out
      keys.template take<L>(hi, lo, won);
      const uint32_t after = (uint32_t)__shfl_down((int)mine_lo, 1, kWave);   // (by all lanes: a lane that is switched off gives 0)
      const uint32_t next = tl == A.K - 1 ? lo : after;
      if (tl < A.K && next >= kNone && (float)((mine_lo >> 10) - (next >> 10)) <= near_by) doubt = true;
      if (tl < A.K && windowed && (float)(mine_lo >> 10) <= kMargin + near_by) doubt = true;
      if (__ballot(doubt) != 0ull) at = choose_exactly<V, L, groups>(z, bad, A, (double*)lds);
      // the chosen logits come out of the lanes that hold them through LDS
      float* zs = (float*)lds + team * (L * V);
      wave_sync();
#pragma unroll
      for (int j = 0; j < V; ++j) zs[e0 + j] = z[j];
      wave_sync();
      if (at >= 0) zi = zs[at];
    }
    // place tl's weight
    float ref = A.softmax ? top : 0.f;
    if (A.renorm) {
      ref = team_max<L>(A.softmax ? zi : fminf(zi, 0.f));
      if (!finite(ref)) ref = 0.f;
    }
    float w = expf((A.softmax ? zi : fminf(zi, 0.f)) - ref);
    if (!A.softmax) w = w / (1.f + expf(-fabsf(zi)));
    if (at < 0) w = 0.f;
    float total = A.softmax ? sum : 1.f;
    if (A.renorm) total = team_sum<L>(w);
    w = at >= 0 ? A.scale * (w / total) : 0.f;
    if (tl < A.K && live) {
      const int64_t first = tile * TOK * A.K;
      const int o = team * A.K + tl;
      if (A.indices) (A.indices + first)[o] = at;
      if (A.weights) (A.weights + first)[o] = w;
    }
    if (routing) {
      T* dense = (T*)lds;                                     // [TOK][E], as the rows lie in memory
      constexpr int C = 16 / (int)sizeof(T);
      const int n = rows * A.E;
      wave_sync();
      for (int i = lane * C; i < n; i += 64 * C) *(uint4*)(dense + i) = make_uint4(0, 0, 0, 0);
      wave_sync();
      if (at >= 0) Elem<T>::store(dense + row_at + at, w);
      wave_sync();
      T* out = routing + tile * TOK * A.E;
      for (int i = lane * C; i < n; i += 64 * C) {
        if (i + C <= n) {
          const uint4 v = *(const uint4*)(dense + i);
          __builtin_memcpy(out + i, &v, 16);
        } else {
          for (int j = i; j < n; ++j) out[j] = dense[j];
        }
      }
      wave_sync();
    }
  }
}

// Tokens per expert from the indices.  Integers, so the order of the additions does not show.
__global__ __launch_bounds__(256) void route_count_kernel(const int32_t* __restrict__ indices, int64_t n, int32_t* __restrict__ counts, int E) {
  __shared__ int hist[MAX_E];
  for (int e = threadIdx.x; e < E; e += 256) hist[e] = 0;
  __syncthreads();
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
    const int at = indices[i];
    if (at >= 0) atomicAdd(hist + at, 1);
  }
  __syncthreads();
  for (int e = threadIdx.x; e < E; e += 256)
    if (hist[e] != 0) atomicAdd(counts + e, hist[e]);
}

// Gradient by the same teams: lane i has place i (expert, score, gradient), the places' gradients meet in an LDS tile of the
// wave's rows, and every lane adds the softmax's common term to its V experts where there is one.  The logits are gathered at
// the chosen experts; whole rows of them are read only for softmax scores that are not renormalised.  Places that name the same
// expert add up, in no fixed order (route_topk never returns such places).  Bound by memory latency: one tile per wave, 5 us
// for 16384 x 128 bf16 with the whole softmax (13 MB: 2.4 us at the copy rate).
template <typename T, int V, int L>
__global__ __launch_bounds__(WAVES * 64) void route_grad_team_kernel(const T* __restrict__ logits, const int32_t* __restrict__ indices,
                                                                     const T* __restrict__ g_routing, const float* __restrict__ g_weights,
                                                                     T* __restrict__ grad, int64_t N, int E, int K, int softmax, int renorm,
                                                                     float scale) {
  constexpr int TOK = 64 / L;
  __shared__ __align__(16) float tiles_raw[WAVES][64 * V];
  const int lane = threadIdx.x & 63, tl = lane & (L - 1), team = lane / L, e0 = tl * V;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  float* own = tiles_raw[wave] + team * L * V;                  // this token's row (L V >= E)
  const bool whole = softmax && !renorm;
  const int64_t tile = (int64_t)blockIdx.x * WAVES + wave;
  if (tile * TOK < N) {
    const bool live = team < N - tile * TOK;
    const int64_t row_first = tile * TOK * E, place_first = tile * TOK * K;
    const int row_at = team * E, place = team * K + tl;
    int at = (live && tl < K) ? (indices + place_first)[place] : -1;
    if (at >= E) at = -1;
    float zi = -INFINITY, q = 0.f;
    if (at >= 0) {
      zi = Elem<T>::load(logits + row_first + row_at + at);
      if (g_routing) q = Elem<T>::load(g_routing + row_first + row_at + at);
      if (g_weights) q += (g_weights + place_first)[place];
    }
    float z[V], top = 0.f, sum = 1.f;
    if (whole) {
      load_run<V>(logits + row_first + row_at + e0, live ? E - e0 : 0, -INFINITY, z);
      top = -INFINITY;
#pragma unroll
      for (int j = 0; j < V; ++j) top = fmaxf(top, z[j]);
      top = team_max<L>(top);
      if (!finite(top)) top = 0.f;
      sum = 0.f;
#pragma unroll
      for (int j = 0; j < V; ++j) {
        z[j] = quick_exp(z[j] - top);
        sum += z[j];
      }
      sum = team_sum<L>(sum);
    }
    float ref = top;
    if (renorm) {
      ref = team_max<L>(softmax ? zi : fminf(zi, 0.f));
      if (!finite(ref)) ref = 0.f;
    }
    float s = expf((softmax ? zi : fminf(zi, 0.f)) - ref);
    if (!softmax) s = s / (1.f + expf(-fabsf(zi)));
    if (at < 0) s = 0.f;
    if (renorm) {
      sum = team_sum<L>(s);
      q -= __shfl(at >= 0 ? q : 0.f, lane & ~(L - 1), kWave);   // less the first place's: no effect but on the rounding
    }
    const float p = at >= 0 ? s / sum : 0.f;
    const float dot = (whole || renorm) ? team_sum<L>(at >= 0 ? p * q : 0.f) : 0.f;
    float d = scale * p * (q - (renorm ? dot : 0.f));
    if (!softmax) d = at >= 0 ? d / (1.f + expf(zi)) : 0.f;
    const bool some = team_any<L>(at >= 0);
    wave_sync();
#pragma unroll
    for (int j = 0; j < V; j += 4) *(float4*)(own + e0 + j) = make_float4(0.f, 0.f, 0.f, 0.f);
    wave_sync();
    if (at >= 0) atomicAdd(own + at, d);
    wave_sync();
    float v[V];
#pragma unroll
    for (int j = 0; j < V; j += 4) {
      const float4 f = *(const float4*)(own + e0 + j);
      v[j] = f.x; v[j + 1] = f.y; v[j + 2] = f.z; v[j + 3] = f.w;
    }
    if (whole && some) {
      const float common = scale * dot / sum;
#pragma unroll
      for (int j = 0; j < V; ++j) v[j] -= z[j] * common;
    }
    if (live && e0 < E) store_run<V>(grad + row_first + row_at + e0, E - e0, v);
  }
}

// More than 64 places: one wave per token, float64 throughout.
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
  if (counts != nullptr && blockIdx.x == 0)
    for (int e = lane; e < E; e += 64) counts[e] = 0;
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
// (more than 64 places: one wave per token)
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

// Lanes per token: as many as the places and, at V experts per lane, the experts need.
inline int team_lanes(int E, int V, int K) {
  int lanes = 4;
  while (lanes * V < E || lanes < K) lanes *= 2;
  return lanes;
}

// One tile per wave, no loop over tiles: the compiler would move what a tile computes from E and the lane out of it and hold
// it in registers (130 to 160 of them, three waves per SIMD instead of five).  More workgroups than one launch takes (2^32
// work-items) go in slices of 2^22.
constexpr int64_t SLICE = (int64_t)1 << 22;
inline int64_t team_blocks(int64_t N, int L) { return cdiv64(cdiv64(N, 64 / L), WAVES); }

template <typename T, int V, int L>
hipError_t forward_l(const d2dmoe_route_shape& sh, const T* logits, T* routing, const RouteArgs& A, hipStream_t s) {
  // per wave: the dense tile; with scores the exact choice's T E values, and the chosen logits; with groups also T G scores
  const size_t tok = 64 / L;
  size_t wave = tok * A.E * sizeof(T);
  if (A.G > 1 || A.bias) wave = tok * A.E * sizeof(double) > 64 * V * sizeof(float) ? tok * A.E * sizeof(double) : 64 * V * sizeof(float);
  if (A.G > 1) wave += tok * A.G * sizeof(double);
  wave = (wave + 15) / 16 * 16;
  const size_t lds = WAVES * wave;                            // (64 KB at the most: tok E <= 64 V, G <= E)
  const bool score = A.bias || (A.G > 1 && A.top2);
  const auto kern = A.G > 1 ? (score ? route_team_kernel<T, V, L, BY_SCORE | IN_GROUPS> : route_team_kernel<T, V, L, BY_LOGIT | IN_GROUPS>)
                            : (score ? route_team_kernel<T, V, L, BY_SCORE> : route_team_kernel<T, V, L, BY_LOGIT>);
  constexpr int64_t tokens = SLICE * WAVES * (64 / L);
  for (int64_t done = 0; done < A.N; done += tokens) {
    RouteArgs part = A;
    part.inv_lanes = (float)V * A.inv_size;
    part.N = A.N - done < tokens ? A.N - done : tokens;
    if (A.indices) part.indices += done * A.K;
    if (A.weights) part.weights += done * A.K;
    hipLaunchKernelGGL(kern, dim3((unsigned)team_blocks(part.N, L)), dim3(WAVES * 64), lds, s, logits + done * A.E,
                       routing ? routing + done * A.E : routing, part, (int)wave);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

template <typename T>
hipError_t forward_t(const d2dmoe_route_shape& sh, const void* logits, const float* bias, void* routing, int32_t* indices, float* weights,
                     int32_t* counts, hipStream_t s) {
  const int softmax = sh.scoring == D2DMOE_SCORE_SOFTMAX, top2 = sh.group_score == D2DMOE_GROUP_TOP2;
  if (sh.k <= 64) {
    const RouteArgs A{bias, indices, weights, counts, sh.n_tokens, sh.n_experts, sh.k, softmax, sh.n_groups, sh.kept_groups, top2,
                      sh.renormalise, sh.scale, sh.n_experts / sh.n_groups, (float)sh.n_groups / (float)sh.n_experts,
                      1.f / (float)sh.n_groups, 0.f};
    const T* z = (const T*)logits;
    T* r = (T*)routing;
    if (sh.n_experts > 512) return forward_l<T, 16, 64>(sh, z, r, A, s);
    // fewer experts per lane where the places ask for so many lanes that four each are enough, or two (at eight per lane 2^20
    // rows of 8, two each, take 31 us instead of 20, and 135823 x 48 bf16 in groups with a bias, 12 each, 59 instead of 41)
    const int lanes = team_lanes(1, 8, sh.k);
    if (sh.n_experts <= 4 * lanes) {
      switch (lanes) {
        case 4: return sh.n_experts <= 8 ? forward_l<T, 2, 4>(sh, z, r, A, s) : forward_l<T, 4, 4>(sh, z, r, A, s);
        case 8: return forward_l<T, 4, 8>(sh, z, r, A, s);
        case 16: return forward_l<T, 4, 16>(sh, z, r, A, s);
        case 32: return forward_l<T, 4, 32>(sh, z, r, A, s);
        default: return forward_l<T, 4, 64>(sh, z, r, A, s);
      }
    }
    switch (team_lanes(sh.n_experts, 8, sh.k)) {
      case 4: return forward_l<T, 8, 4>(sh, z, r, A, s);
      case 8: return forward_l<T, 8, 8>(sh, z, r, A, s);
      case 16: return forward_l<T, 8, 16>(sh, z, r, A, s);
      case 32: return forward_l<T, 8, 32>(sh, z, r, A, s);
      default: return forward_l<T, 8, 64>(sh, z, r, A, s);
    }
  }
  const unsigned grid = (unsigned)(sh.n_tokens < (1 << 20) ? sh.n_tokens : (1 << 20));
  hipLaunchKernelGGL(route_kernel<T>, dim3(grid), dim3(64), 0, s, (const T*)logits, bias, (T*)routing, indices, weights, counts,
                     sh.n_tokens, sh.n_experts, sh.k, softmax, sh.n_groups, sh.kept_groups, top2, sh.renormalise, sh.scale);
  return hipGetLastError();
}

template <typename T, int V, int L>
hipError_t backward_l(const d2dmoe_route_shape& sh, const void* logits, const int32_t* indices, const void* g_routing,
                      const float* g_weights, void* grad, hipStream_t s) {
  constexpr int64_t tokens = SLICE * WAVES * (64 / L);
  const int E = sh.n_experts, K = sh.k;
  for (int64_t done = 0; done < sh.n_tokens; done += tokens) {
    const int64_t n = sh.n_tokens - done < tokens ? sh.n_tokens - done : tokens;
    hipLaunchKernelGGL((route_grad_team_kernel<T, V, L>), dim3((unsigned)team_blocks(n, L)), dim3(WAVES * 64), 0, s,
                       (const T*)logits + done * E, indices + done * K, g_routing ? (const T*)g_routing + done * E : nullptr,
                       g_weights ? g_weights + done * K : nullptr, (T*)grad + done * E, n, E, K, sh.scoring == D2DMOE_SCORE_SOFTMAX,
                       sh.renormalise, sh.scale);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

template <typename T>
hipError_t backward_t(const d2dmoe_route_shape& sh, const void* logits, const int32_t* indices, const void* g_routing,
                      const float* g_weights, void* grad, hipStream_t s) {
  if (sh.k <= 64) {
    if (sh.n_experts > 512) return backward_l<T, 16, 64>(sh, logits, indices, g_routing, g_weights, grad, s);
    switch (team_lanes(sh.n_experts, 8, sh.k)) {
      case 4: return backward_l<T, 8, 4>(sh, logits, indices, g_routing, g_weights, grad, s);
      case 8: return backward_l<T, 8, 8>(sh, logits, indices, g_routing, g_weights, grad, s);
      case 16: return backward_l<T, 8, 16>(sh, logits, indices, g_routing, g_weights, grad, s);
      case 32: return backward_l<T, 8, 32>(sh, logits, indices, g_routing, g_weights, grad, s);
      default: return backward_l<T, 8, 64>(sh, logits, indices, g_routing, g_weights, grad, s);
    }
  }
  const unsigned grid = (unsigned)(sh.n_tokens < (1 << 20) ? sh.n_tokens : (1 << 20));
  hipLaunchKernelGGL(route_grad_kernel<T>, dim3(grid), dim3(64), 0, s, (const T*)logits, indices, (const T*)g_routing, g_weights,
                     (T*)grad, sh.n_tokens, sh.n_experts, sh.k, sh.scoring == D2DMOE_SCORE_SOFTMAX, sh.renormalise, sh.scale);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_route_topk(const d2dmoe_route_shape& sh, const void* logits, const float* bias, void* routing, int32_t* indices,
                             float* weights, int32_t* counts, hipStream_t s) {
  if (sh.n_tokens == 0) return counts ? launch_fill_i32(counts, sh.n_experts, 0, s) : hipSuccess;
  hipError_t e;
  switch (sh.dtype) {
    case D2DMOE_F32: e = forward_t<float>(sh, logits, bias, routing, indices, weights, counts, s); break;
    case D2DMOE_BF16: e = forward_t<bf16_t>(sh, logits, bias, routing, indices, weights, counts, s); break;
    default: e = forward_t<f16_t>(sh, logits, bias, routing, indices, weights, counts, s); break;
  }
  if (e != hipSuccess || counts == nullptr) return e;
  const int64_t n = sh.n_tokens * sh.k, blocks = cdiv64(n, 1024);
  hipLaunchKernelGGL(route_count_kernel, dim3((unsigned)(blocks < 256 ? blocks : 256)), dim3(256), 0, s, indices, n, counts, sh.n_experts);
  return hipGetLastError();
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
