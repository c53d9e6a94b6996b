// Group norm with an activation on channels-last activations, forward and backward.
//
//   per sample b and group g (Cg = C/G channels, N = HW*Cg values):
//     mean, rstd = 1/sqrt(var + eps);  xh = (x - mean) rstd;  u = xh gamma + beta;  y = act(u)
//     du = dy act'(u);  dbeta = sum du;  dgamma = sum du xh
//     dx = rstd (du gamma - m1 - xh m2),  m1 = sum(du gamma)/N,  m2 = sum(du gamma xh)/N
//
// HBM-bound: forward reads x and writes y, backward reads x and dy and writes dx.
// A workgroup owns a range of pixels and a slab of at most 256 channel vectors that starts and ends with a group
// (or lies inside one group, when a group is wider); a thread keeps one channel vector and walks the pixels, so a
// wave reads contiguous memory and everything that belongs to a channel stays in registers.
// The statistics are sums of d = x - K and d*d in 64 bits, K the group's first value: mean = K + E[d], var = E[d^2] - E[d]^2.
// K is as near to the mean as the group's values are, so the subtraction is harmless at any mean: a spread of one unit in the
// last place of float32 survives.  On this chip a double add costs what a float add costs.
// Sums over pixels are combined in a fixed order: results repeat bit for bit.
#include <algorithm>

#include "act.h"
#include "common.h"

namespace {

constexpr int GN_THREADS = 256;

// N elements (N * sizeof(T) = 2..16 bytes, aligned to that) <-> floats
template <typename T, int N> struct Bits;
template <typename T> struct Bits<T, 1> { typedef T type; };
template <> struct Bits<bf16, 2> { typedef uint32_t type; };
template <> struct Bits<bf16, 4> { typedef uint2 type; };
template <> struct Bits<bf16, 8> { typedef uint4 type; };
template <> struct Bits<float, 2> { typedef uint2 type; };
template <> struct Bits<float, 4> { typedef uint4 type; };

template <typename T, int V> union Vec {
  typename Bits<T, V>::type u;
  T t[V];
  __device__ Vec() {}
};

struct Shape {
  int64_t HW;
  int C, G, Cg;
  int gps;          // groups per slab (1 when a group needs several slabs)
  int parts;        // slabs per group (1 when a slab holds whole groups)
  int slab_c;       // channels of a full slab
  int CV, PR;       // channel vectors of a full slab, pixels side by side in a workgroup
  int slabs, chunks;
  int64_t ppc;      // pixels per chunk
};

struct Slab {       // of one workgroup
  int c0, nc, g0, ng;
};

__device__ __forceinline__ Slab slab_of(const Shape& s, int i) {
  Slab r;
  if (s.parts == 1) {
    r.g0 = i * s.gps;
    r.ng = min(s.gps, s.G - r.g0);
    r.c0 = r.g0 * s.Cg;
    r.nc = r.ng * s.Cg;
  } else {
    r.g0 = i / s.parts;
    r.ng = 1;
    const int o = (i - r.g0 * s.parts) * s.slab_c;
    r.c0 = r.g0 * s.Cg + o;
    r.nc = min(s.slab_c, s.Cg - o);
  }
  return r;
}

// f(i, group of channel c + i, whether that is another group than channel c + i - 1's) for i < V, with one division.
template <int V, typename F> __device__ __forceinline__ void with_groups(int c, int Cg, F&& f) {
  int g = c / Cg, left = Cg - (c - g * Cg);
#pragma unroll
  for (int i = 0; i < V; i++) {
    const bool other = i > 0 && left == 0;
    if (other) {
      g++;
      left = Cg;
    }
    f(i, g, i == 0 || other);
    left--;
  }
}

// K of group g.  (Where it is not finite the statistics would not be either.)
template <typename T> __device__ __forceinline__ double first_of(const T* __restrict__ sample, int g, int Cg) {
  return (double)to_f32(sample[(int64_t)g * Cg]);
}

// sums[b][chunk*parts + part][g] = (sum d, sum d*d) over the chunk's pixels and the slab's channels of g.
// U: channels of a vector that are sure to share a group (a power of two that divides V and the group), so a thread holds
// V/U pairs of sums and not V: few enough registers for eight waves to a SIMD, which the stream of loads needs.
// Bound by HBM: 16x32x512^2 bf16 (268 MB) in 74 us (72 without K) behind a kernel whose output is still being written back, 3.6
// TB/s; its loop alone reads 7 TB/s.
template <typename T, int V, int U>
__global__ __launch_bounds__(GN_THREADS) void gn_sums_kernel(const T* __restrict__ x, Shape s, double2* __restrict__ sums) {
  constexpr int N = V / U;
  extern __shared__ __attribute__((aligned(16))) char gn_lds[];
  double2* red = (double2*)gn_lds;                       // [PR][CV*N]
  const int b = blockIdx.z, tid = threadIdx.x;
  const Slab sl = slab_of(s, blockIdx.y);
  const int cv = tid % s.CV, pr = tid / s.CV;
  const int64_t p0 = (int64_t)blockIdx.x * s.ppc, p1 = min(p0 + s.ppc, s.HW);
  const bool on = pr < s.PR && cv * V < sl.nc;
  if (on) {
    double a1[N], a2[N], first[N];
    const T* sample = x + (int64_t)b * s.HW * s.C;
    double of_group = 0.0;
    with_groups<N>((sl.c0 + cv * V) / U, s.Cg / U, [&](int k, int g, bool other) {
      if (other) of_group = first_of(sample, g, s.Cg);
      first[k] = of_group;
      a1[k] = a2[k] = 0.0;
    });
    const T* xp = sample + sl.c0 + cv * V;
    auto add = [&](const Vec<T, V>& v) {
#pragma unroll
      for (int k = 0; k < V; k++) {
        const double d = (double)to_f32(v.t[k]) - first[k / U];
        a1[k / U] += d;
        a2[k / U] = fma(d, d, a2[k / U]);
      }
    };
    int64_t p = p0 + pr;
    for (; p + 3 * s.PR < p1; p += 4 * s.PR) {           // four loads ahead of the sums
      Vec<T, V> v[4];
#pragma unroll
      for (int i = 0; i < 4; i++) v[i].u = *(const typename Bits<T, V>::type*)(xp + (p + i * s.PR) * s.C);
#pragma unroll
      for (int i = 0; i < 4; i++) add(v[i]);
    }
    for (; p < p1; p += s.PR) {
      Vec<T, V> v;
      v.u = *(const typename Bits<T, V>::type*)(xp + p * s.C);
      add(v);
    }
#pragma unroll
    for (int k = 0; k < N; k++) red[(pr * s.CV + cv) * N + k] = make_double2(a1[k], a2[k]);
  }
  __syncthreads();
  const int W = s.CV * N, nc = sl.nc / U;
  int n = s.PR;
  while (n > 1) {                                        // pixel rows: halves onto halves
    const int h = (n + 1) >> 1;
    for (int i = tid; i < (n - h) * W; i += GN_THREADS) {
      if (i % W < nc) {
        red[i].x += red[i + h * W].x;
        red[i].y += red[i + h * W].y;
      }
    }
    __syncthreads();
    n = h;
  }
  const int part = s.parts == 1 ? 0 : blockIdx.y % s.parts;
  double2* out = sums + ((int64_t)b * s.chunks * s.parts + (int64_t)blockIdx.x * s.parts + part) * s.G;
  const int gc = (s.parts == 1 ? s.Cg : sl.nc) / U;
  for (int g = tid; g < sl.ng; g += GN_THREADS) {
    double t1 = 0.0, t2 = 0.0;
    for (int c = 0; c < gc; c++) {
      t1 += red[g * gc + c].x;
      t2 += red[g * gc + c].y;
    }
    out[sl.g0 + g] = make_double2(t1, t2);
  }
}

// 64-lane sum of doubles on the DPP path; every lane ends with the total.
template <int CTRL> __device__ __forceinline__ double dpp_move(double v) {
  const uint64_t u = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)u, CTRL, 0xF, 0xF, true);
  const uint32_t hi = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)(u >> 32), CTRL, 0xF, 0xF, true);
  return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
__device__ __forceinline__ double lane_of(double v, int lane) {
  const uint64_t u = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = __builtin_amdgcn_readlane((int)(uint32_t)u, lane), hi = __builtin_amdgcn_readlane((int)(uint32_t)(u >> 32), lane);
  return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
__device__ __forceinline__ double wave_sum64(double v) {
  v += dpp_move<0xB1>(v);
  v += dpp_move<0x4E>(v);
  v += dpp_move<0x141>(v);
  v += dpp_move<0x140>(v);
  return (lane_of(v, 0) + lane_of(v, 16)) + (lane_of(v, 32) + lane_of(v, 48));
}

__device__ __forceinline__ double2 stats_of(double s1, double s2, double first, double count, double eps) {
  const double mean = s1 / count;
  double var = s2 / count - mean * mean;
  if (var < 0.0) var = 0.0;                              // (NaN stays NaN)
  return make_double2(first + mean, 1.0 / sqrt(var + eps));
}

// stats[b][g] = (mean, 1/sqrt(var + eps)); one wave per (b, g); a launch's latency, 3-5 us
template <typename T>
__global__ __launch_bounds__(64) void gn_stats_kernel(const T* __restrict__ x, Shape s, const double2* __restrict__ sums, int rows,
                                                      int G, double count, double eps, double2* __restrict__ stats) {
  const int g = blockIdx.x, b = blockIdx.y, lane = threadIdx.x;
  double t1 = 0.0, t2 = 0.0;
  for (int r = lane; r < rows; r += 64) {
    const double2 v = sums[((int64_t)b * rows + r) * G + g];
    t1 += v.x;
    t2 += v.y;
  }
  t1 = wave_sum64(t1);
  t2 = wave_sum64(t2);
  if (lane == 0) stats[(int64_t)b * G + g] = stats_of(t1, t2, first_of(x + (int64_t)b * s.HW * s.C, g, s.Cg), count, eps);
}

// The mean in two floats: hi + lo.  One float would put x - mean off by up to 2^-25 |mean|, which is all of a spread that is
// far smaller than the mean.
__device__ __forceinline__ float mean_lo(double mean) { return (float)(mean - (double)(float)mean); }

// What a thread holds of its V channels: u = (x - mean) * a + beta, a = rstd * gamma; mean is hi, and lo is in beta.
template <int V> struct Consts {
  float mean[V], a[V], beta[V];
};

template <int V>
__device__ __forceinline__ void load_consts(Consts<V>& k, const double2* __restrict__ stats, const float* __restrict__ gamma,
                                            const float* __restrict__ beta, int c, int Cg) {
  double2 st = make_double2(0.0, 0.0);
  float lo[V];
  with_groups<V>(c, Cg, [&](int i, int g, bool other) {
    if (other) st = stats[g];
    k.mean[i] = (float)st.x;
    lo[i] = mean_lo(st.x);
    k.a[i] = (float)st.y;
  });
#pragma unroll
  for (int i = 0; i < V; i++) k.beta[i] = beta ? beta[c + i] : 0.f;
  if (gamma) {
#pragma unroll
    for (int i = 0; i < V; i++) k.a[i] *= gamma[c + i];
  }
#pragma unroll
  for (int i = 0; i < V; i++) k.beta[i] = fmaf(-lo[i], k.a[i], k.beta[i]);
}

// y from x: 2 passes over memory, 16x32x512^2 bf16 (537 MB) in 88 us, 6.1 TB/s.
// FOLD: the workgroup adds up the rows of `sums` of its own few groups itself (a launch less on the way to y) and the one
// of the first chunk leaves the statistics.  Up to 64 rows: 2x32x128^2 bf16 12.1 -> 9.9 us; at the 128 rows of the large
// tensors every workgroup's start gets longer by more than the launch cost (16x32x512^2 171 -> 178 us).
constexpr int FOLD_GROUPS = 16, FOLD_ROWS = 64;
template <typename T, int V, int ACT, bool FOLD>
__global__ __launch_bounds__(GN_THREADS) void gn_apply_kernel(const T* __restrict__ x, Shape s, const double2* __restrict__ sums,
                                                              double eps, double2* __restrict__ stats_all,
                                                              const float* __restrict__ gamma, const float* __restrict__ beta,
                                                              T* __restrict__ y) {
  __shared__ double2 own[FOLD_GROUPS];
  const int b = blockIdx.z, tid = threadIdx.x;
  const Slab sl = slab_of(s, blockIdx.y);
  const int cv = tid % s.CV, pr = tid / s.CV;
  double2* stats = stats_all + (int64_t)b * s.G;
  if constexpr (FOLD) {
    const int lane = tid & 63, rows = s.chunks * s.parts;
    const double count = (double)s.HW * s.Cg;
    for (int g = tid >> 6; g < sl.ng; g += GN_THREADS / 64) {
      double t1 = 0.0, t2 = 0.0;
#pragma unroll 4
      for (int r = lane; r < rows; r += 64) {
        const double2 v = sums[((int64_t)b * rows + r) * s.G + sl.g0 + g];
        t1 += v.x;
        t2 += v.y;
      }
      const double2 st = stats_of(wave_sum64(t1), wave_sum64(t2), first_of(x + (int64_t)b * s.HW * s.C, sl.g0 + g, s.Cg), count,
                                  eps);
      if (lane == 0) {
        own[g] = st;
        if (blockIdx.x == 0) stats[sl.g0 + g] = st;      // (the parts of one group write the same)
      }
    }
    __syncthreads();
  }
  if (pr >= s.PR || cv * V >= sl.nc) return;
  const int c = sl.c0 + cv * V;
  Consts<V> k;
  load_consts<V>(k, FOLD ? own - sl.g0 : stats, gamma, beta, c, s.Cg);
  const int64_t p0 = (int64_t)blockIdx.x * s.ppc, p1 = min(p0 + s.ppc, s.HW);
  const int64_t base = (int64_t)b * s.HW * s.C + c;
#pragma unroll 4
  for (int64_t p = p0 + pr; p < p1; p += s.PR) {
    Vec<T, V> v;
    v.u = *(const typename Bits<T, V>::type*)(x + base + p * s.C);
#pragma unroll
    for (int i = 0; i < V; i++) v.t[i] = from_f32<T>(act_value<ACT>(fmaf(to_f32(v.t[i]) - k.mean[i], k.a[i], k.beta[i])));
    *(typename Bits<T, V>::type*)(y + base + p * s.C) = v.u;
  }
}

// du = dy act'(u).  ReLU's slope has a jump: where u is within the rounding of its float evaluation of zero (one
// value in a million), its sign is taken from the 64-bit statistics, so that the mask is the definition's.
template <int ACT>
__device__ __forceinline__ float du_of(float x, float dy, float mean, float a, float beta, int c, int Cg,
                                       const double2* __restrict__ stats, const float* __restrict__ gammas,
                                       const float* __restrict__ betas) {
  const float u = fmaf(x - mean, a, beta);
  if constexpr (ACT == MIS_ACT_NONE) {
    return dy;
  } else if constexpr (ACT == MIS_ACT_RELU) {
    bool pos = u > 0.f;
    if (fabsf(u) < 1e-6f * fmaf(fabsf(x) + fabsf(mean), fabsf(a), fabsf(beta))) {
      const double2 st = stats[c / Cg];
      pos = ((double)x - st.x) * st.y * (gammas ? (double)gammas[c] : 1.0) + (betas ? (double)betas[c] : 0.0) > 0.0;
    }
    return pos ? dy : 0.f;
  } else {
    return dy * act_slope<ACT>(u);
  }
}

// rows[b][chunk][2][C] = (sum du, sum du xh) over the chunk's pixels.  Per channel, not per group, since dgamma and dbeta
// need them so and the group's means follow from them.  16x32x512^2 bf16 with ReLU (537 MB) in 131 us, 4.1 TB/s (it starts on
// the write-back of y's gradient).  Float32 over the BWD_RUN pixels at most that a thread walks (plan cuts the chunks so: sums
// of thousands of terms would be 10^-5 off) and pairwise over the workgroup's pixel rows, stored as float32; 64 bits over the
// chunks and samples.
constexpr int BWD_RUN = 64;
template <typename T, int V, int ACT>
__global__ __launch_bounds__(GN_THREADS) void gn_bwd_sums_kernel(const T* __restrict__ x, const T* __restrict__ dy, Shape s,
                                                                 const double2* __restrict__ stats_all,
                                                                 const float* __restrict__ gamma,
                                                                 const float* __restrict__ beta, float* __restrict__ rows) {
  extern __shared__ __attribute__((aligned(16))) char gn_lds[];
  float2* red = (float2*)gn_lds;                         // [PR][CV*V]
  const int b = blockIdx.z, tid = threadIdx.x;
  const Slab sl = slab_of(s, blockIdx.y);
  const int cv = tid % s.CV, pr = tid / s.CV;
  const int64_t p0 = (int64_t)blockIdx.x * s.ppc, p1 = min(p0 + s.ppc, s.HW);
  const double2* stats = stats_all + (int64_t)b * s.G;
  if (pr < s.PR && cv * V < sl.nc) {
    const int c = sl.c0 + cv * V;
    Consts<V> k;
    load_consts<V>(k, stats, gamma, beta, c, s.Cg);
    float a1[V], a2[V];
#pragma unroll
    for (int i = 0; i < V; i++) a1[i] = a2[i] = 0.f;
    const int64_t base = (int64_t)b * s.HW * s.C + c;
#pragma unroll 2
    for (int64_t p = p0 + pr; p < p1; p += s.PR) {
      Vec<T, V> vx, vd;
      vx.u = *(const typename Bits<T, V>::type*)(x + base + p * s.C);
      vd.u = *(const typename Bits<T, V>::type*)(dy + base + p * s.C);
#pragma unroll
      for (int i = 0; i < V; i++) {
        const float xf = to_f32(vx.t[i]);
        const float du = du_of<ACT>(xf, to_f32(vd.t[i]), k.mean[i], k.a[i], k.beta[i], c + i, s.Cg, stats, gamma, beta);
        a1[i] += du;
        a2[i] = fmaf(du, xf - k.mean[i], a2[i]);         // less lo a1, times rstd at the end
      }
    }
    float rstd = 0.f, lo = 0.f;
    with_groups<V>(c, s.Cg, [&](int i, int g, bool other) {
      if (other) {
        rstd = (float)stats[g].y;
        lo = mean_lo(stats[g].x);
      }
      red[(pr * s.CV + cv) * V + i] = make_float2(a1[i], fmaf(-lo, a1[i], a2[i]) * rstd);
    });
  }
  __syncthreads();
  const int W = s.CV * V;
  int n = s.PR;
  while (n > 1) {
    const int h = (n + 1) >> 1;
    for (int i = tid; i < (n - h) * W; i += GN_THREADS) {
      const int r = i / W, c = i - r * W;
      if (c < sl.nc) {
        red[i].x += red[i + h * W].x;
        red[i].y += red[i + h * W].y;
      }
    }
    __syncthreads();
    n = h;
  }
  float* out = rows + ((int64_t)b * s.chunks + blockIdx.x) * 2 * s.C;
  for (int c = tid; c < sl.nc; c += GN_THREADS) {
    out[sl.c0 + c] = red[c].x;
    out[s.C + sl.c0 + c] = red[c].y;
  }
}

// chan[b][2][C] = sums over the chunks; block = 32 channels of one sample, R row lanes; 3-5 us
template <int R>
__global__ __launch_bounds__(32 * R) void gn_bwd_channels_kernel(const float* __restrict__ rows, int chunks, int C,
                                                                 float* __restrict__ chan) {
  __shared__ double2 red[R][33];
  const int lane = threadIdx.x & 31, r = threadIdx.x >> 5, c = blockIdx.x * 32 + lane, b = blockIdx.y;
  double t1 = 0.0, t2 = 0.0;
  if (c < C) {
    const float* p = rows + (int64_t)b * chunks * 2 * C + c;
#pragma unroll 8
    for (int i = r; i < chunks; i += R) {
      t1 += (double)p[(int64_t)i * 2 * C];
      t2 += (double)p[(int64_t)i * 2 * C + C];
    }
  }
  red[r][lane] = make_double2(t1, t2);
  __syncthreads();
  if (r == 0 && c < C) {
#pragma unroll
    for (int i = 1; i < R; i++) {
      t1 += red[i][lane].x;
      t2 += red[i][lane].y;
    }
    chan[(int64_t)b * 2 * C + c] = (float)t1;
    chan[(int64_t)b * 2 * C + C + c] = (float)t2;
  }
}

// The first blocks: dbeta, dgamma = sums of chan over the samples, 64 channels x 4 sample lanes a block.
// The others (launched only if dx is wanted): coef[b][g] = (m1, m2), one wave per (b, g).  3-5 us.
__global__ __launch_bounds__(256) void gn_bwd_finish_kernel(const float* __restrict__ chan, const float* __restrict__ gamma, int B,
                                                            int C, int Cg, int G, double count, int channel_blocks,
                                                            float2* __restrict__ coef, float* __restrict__ dgamma,
                                                            float* __restrict__ dbeta) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  if ((int)blockIdx.x < channel_blocks) {
    __shared__ double2 red[4][64];
    const int c = blockIdx.x * 64 + lane;
    double s1 = 0.0, s2 = 0.0;
    if (c < C) {
#pragma unroll 4
      for (int b = wave; b < B; b += 4) {
        s1 += (double)chan[(int64_t)b * 2 * C + c];
        s2 += (double)chan[(int64_t)b * 2 * C + C + c];
      }
    }
    red[wave][lane] = make_double2(s1, s2);
    __syncthreads();
    if (wave == 0 && c < C) {
      for (int w = 1; w < 4; w++) {
        s1 += red[w][lane].x;
        s2 += red[w][lane].y;
      }
      if (dbeta) dbeta[c] = (float)s1;
      if (dgamma) dgamma[c] = (float)s2;
    }
    return;
  }
  const int64_t bg = ((int64_t)blockIdx.x - channel_blocks) * 4 + wave;
  if (bg >= (int64_t)B * G) return;
  const int b = (int)(bg / G), g = (int)(bg - (int64_t)b * G);
  const float* p = chan + (int64_t)b * 2 * C + (int64_t)g * Cg;
  double t1 = 0.0, t2 = 0.0;
  for (int c = lane; c < Cg; c += 64) {
    const double w = gamma ? (double)gamma[g * Cg + c] : 1.0;
    t1 += w * (double)p[c];
    t2 += w * (double)p[C + c];
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    t1 += __shfl_xor(t1, o, WAVE);
    t2 += __shfl_xor(t2, o, WAVE);
  }
  if (lane == 0) coef[bg] = make_float2((float)(t1 / count), (float)(t2 / count));
}

// dx = du a - rstd m1 - (x - mean) rstd^2 m2 with du formed again from x and dy: reads both, writes dx; 16x32x512^2 bf16
// (805 MB) in 151 us, 5.3 TB/s, a copy's rate.  Adding the sums up here instead of in two launches gained nothing.
template <typename T, int V, int ACT>
__global__ __launch_bounds__(GN_THREADS) void gn_bwd_dx_kernel(const T* __restrict__ x, const T* __restrict__ dy, Shape s,
                                                               const double2* __restrict__ stats_all,
                                                               const float* __restrict__ gamma, const float* __restrict__ beta,
                                                               const float2* __restrict__ coef, T* __restrict__ dx) {
  const int b = blockIdx.z, tid = threadIdx.x;
  const Slab sl = slab_of(s, blockIdx.y);
  const int cv = tid % s.CV, pr = tid / s.CV;
  if (pr >= s.PR || cv * V >= sl.nc) return;
  const double2* stats = stats_all + (int64_t)b * s.G;
  const int c = sl.c0 + cv * V;
  Consts<V> k;
  load_consts<V>(k, stats, gamma, beta, c, s.Cg);
  float q1[V], q2[V];                                    // dx = du a - q1 - (x - hi) q2
  float rstd = 0.f, lo = 0.f;
  float2 m = make_float2(0.f, 0.f);
  with_groups<V>(c, s.Cg, [&](int i, int g, bool other) {
    if (other) {
      rstd = (float)stats[g].y;
      lo = mean_lo(stats[g].x);
      m = coef[(int64_t)b * s.G + g];
    }
    q2[i] = rstd * rstd * m.y;
    q1[i] = fmaf(-lo, q2[i], rstd * m.x);
  });
  const int64_t p0 = (int64_t)blockIdx.x * s.ppc, p1 = min(p0 + s.ppc, s.HW);
  const int64_t base = (int64_t)b * s.HW * s.C + c;
#pragma unroll 2
  for (int64_t p = p0 + pr; p < p1; p += s.PR) {
    Vec<T, V> vx, vd;
    vx.u = *(const typename Bits<T, V>::type*)(x + base + p * s.C);
    vd.u = *(const typename Bits<T, V>::type*)(dy + base + p * s.C);
#pragma unroll
    for (int i = 0; i < V; i++) {
      const float xf = to_f32(vx.t[i]);
      const float du = du_of<ACT>(xf, to_f32(vd.t[i]), k.mean[i], k.a[i], k.beta[i], c + i, s.Cg, stats, gamma, beta);
      vd.t[i] = from_f32<T>(fmaf(du, k.a[i], -fmaf(xf - k.mean[i], q2[i], q1[i])));
    }
    *(typename Bits<T, V>::type*)(dx + base + p * s.C) = vd.u;
  }
}

// ---------------------------------------------------------------------------------------------------------------
// One workgroup holds a slab of whole groups of one sample in registers (RES_THREADS threads, NV vectors each): x (and
// dy) are read once, the forward is one launch.  Vectors never straddle a group here.
// ---------------------------------------------------------------------------------------------------------------
constexpr int RES_THREADS = 512, RES_WAVES = RES_THREADS / 64;
constexpr int RES_WIDE = 256;        // most vectors of a slab side by side

// Sum over all threads of a group of the two values per thread; valid in red_out[group] after the barrier.
// Thread tid holds channel vector tid % CV of pixel row tid / CV; a group is GV neighbouring vectors.
__device__ __forceinline__ void group_sums(double s1, double s2, int CV, int GV, int ng, int PR, double2* red, double2* out) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  red[tid] = make_double2(s1, s2);
  __syncthreads();
  const int n = PR * GV;
  for (int g = wave; g < ng; g += RES_WAVES) {
    double t1 = 0.0, t2 = 0.0;
    for (int e = lane; e < n; e += 64) {
      const int r = e / GV;
      const double2 v = red[r * CV + g * GV + (e - r * GV)];
      t1 += v.x;
      t2 += v.y;
    }
    t1 = wave_sum64(t1);
    t2 = wave_sum64(t2);
    if (lane == 0) out[g] = make_double2(t1, t2);
  }
  __syncthreads();
}

// (sample, slab) of a workgroup: the slabs of a sample, which share its memory lines, run on one XCD (workgroups are dealt
// to the 8 XCDs in turn).
__device__ __forceinline__ bool resident_place(const Shape& s, int B, int& b, int& slab) {
  const int total = B * s.slabs, per = ((int)gridDim.x + 7) / 8, id = ((int)blockIdx.x % 8) * per + (int)blockIdx.x / 8;
  b = id / s.slabs;
  slab = id - b * s.slabs;
  return id < total;
}

// One read of x, one write of y: 16x512x32^2 bf16 (34 MB) in 13 us, 1x64x32^2 in 5: one round of workgroups, each waiting
// for its loads, its two barriers and its stores in turn.
template <typename T, int V, int NV, int ACT>
__global__ __launch_bounds__(RES_THREADS, 2) void gn_resident_kernel(const T* __restrict__ x, Shape s, int B, double eps,
                                                                     const float* __restrict__ gamma,
                                                                     const float* __restrict__ beta, T* __restrict__ y,
                                                                     double2* __restrict__ stats) {
  __shared__ double2 red[RES_THREADS], grp[RES_THREADS];
  int b, slab;
  if (!resident_place(s, B, b, slab)) return;
  const Slab sl = slab_of(s, slab);
  const int tid = threadIdx.x, cv = tid % s.CV, pr = tid / s.CV, HW = (int)s.HW;
  const bool on = pr < s.PR && cv * V < sl.nc;
  const int64_t base = (int64_t)b * s.HW * s.C + sl.c0 + (on ? cv * V : 0);
  Vec<T, V> v[NV];
#pragma unroll
  for (int i = 0; i < NV; i++) {
    const int p = min(pr + i * s.PR, HW - 1);
    v[i].u = *(const typename Bits<T, V>::type*)(x + base + (int64_t)p * s.C);
  }
  const T* sample = x + (int64_t)b * s.HW * s.C;
  const double first = first_of(sample, (sl.c0 + (on ? cv * V : 0)) / s.Cg, s.Cg);
  double s1 = 0.0, s2 = 0.0;
  if (on) {
#pragma unroll
    for (int i = 0; i < NV; i++) {
      if (pr + i * s.PR < HW) {
#pragma unroll
        for (int k = 0; k < V; k++) {
          const double d = (double)to_f32(v[i].t[k]) - first;
          s1 += d;
          s2 = fma(d, d, s2);
        }
      }
    }
  }
  const int GV = s.Cg / V;
  group_sums(s1, s2, s.CV, GV, sl.ng, s.PR, red, grp);
  const double count = (double)s.HW * s.Cg;
  if (tid < sl.ng) {
    const double2 st = stats_of(grp[tid].x, grp[tid].y, first_of(sample, sl.g0 + tid, s.Cg), count, eps);
    grp[tid] = st;
    stats[(int64_t)b * s.G + sl.g0 + tid] = st;
  }
  __syncthreads();
  if (!on) return;
  Consts<V> k;
  load_consts<V>(k, grp - sl.g0, gamma, beta, sl.c0 + cv * V, s.Cg);
#pragma unroll
  for (int i = 0; i < NV; i++) {
    const int p = pr + i * s.PR;
    if (p < HW) {
      Vec<T, V> o;
#pragma unroll
      for (int j = 0; j < V; j++) o.t[j] = from_f32<T>(act_value<ACT>(fmaf(to_f32(v[i].t[j]) - k.mean[j], k.a[j], k.beta[j])));
      *(typename Bits<T, V>::type*)(y + base + (int64_t)p * s.C) = o.u;
    }
  }
}

// Backward of a resident slab: dx, and chan[b][2][C] for gn_bwd_finish_kernel.  Its sums are float32 in short runs: at most 16
// pixels in a thread, 32 and a tree of 16 lanes over the pixel rows, 32 and a tree of 64 over a group's channels.  16x512x32^2 bf16 with SiLU (50 MB) in 21 us.
template <typename T, int V, int NV, int ACT>
__global__ __launch_bounds__(RES_THREADS, 2) void gn_resident_bwd_kernel(const T* __restrict__ x, const T* __restrict__ dy,
                                                                         Shape s, int B, const double2* __restrict__ stats_all,
                                                                         const float* __restrict__ gamma,
                                                                         const float* __restrict__ beta, T* __restrict__ dx,
                                                                         float* __restrict__ chan) {
  __shared__ float red[2 * V * RES_THREADS];             // [channel of the vector][sum][thread]
  __shared__ float2 tot[RES_WIDE * V];                   // by channel of the slab
  __shared__ float2 coef[RES_WIDE];
  int b, slab;
  if (!resident_place(s, B, b, slab)) return;
  const Slab sl = slab_of(s, slab);
  const double2* stats = stats_all + (int64_t)b * s.G;
  const int tid = threadIdx.x, cv = tid % s.CV, pr = tid / s.CV, HW = (int)s.HW;
  const bool on = pr < s.PR && cv * V < sl.nc;
  const int c = sl.c0 + (on ? cv * V : 0);
  const int64_t base = (int64_t)b * s.HW * s.C + c;
  Vec<T, V> vx[NV], vd[NV];
#pragma unroll
  for (int i = 0; i < NV; i++) {
    const int64_t p = min(pr + i * s.PR, HW - 1);
    vx[i].u = *(const typename Bits<T, V>::type*)(x + base + p * s.C);
    vd[i].u = *(const typename Bits<T, V>::type*)(dy + base + p * s.C);
  }
  Consts<V> k;
  load_consts<V>(k, stats, gamma, beta, c, s.Cg);
  const double2 st = stats[c / s.Cg];
  const float rstd = (float)st.y, lo = mean_lo(st.x);
  float a1[V], a2[V];
#pragma unroll
  for (int j = 0; j < V; j++) a1[j] = a2[j] = 0.f;
  if (on) {
#pragma unroll
    for (int i = 0; i < NV; i++) {
      if (pr + i * s.PR < HW) {
#pragma unroll
        for (int j = 0; j < V; j++) {
          const float xf = to_f32(vx[i].t[j]);
          const float du = du_of<ACT>(xf, to_f32(vd[i].t[j]), k.mean[j], k.a[j], k.beta[j], c + j, s.Cg, stats, gamma, beta);
          a1[j] += du;
          a2[j] = fmaf(du, xf - k.mean[j], a2[j]);
        }
      }
    }
  }
#pragma unroll
  for (int j = 0; j < V; j++) {
    red[2 * j * RES_THREADS + tid] = a1[j];
    red[(2 * j + 1) * RES_THREADS + tid] = fmaf(-lo, a1[j], a2[j]) * rstd;
  }
  __syncthreads();
  // pixel rows: 16 lanes to a channel and sum
  float* out = chan + (int64_t)b * 2 * s.C + sl.c0;
  for (int o = tid >> 4; o < 2 * sl.nc; o += RES_THREADS / 16) {
    const int ch = o >> 1, which = o & 1, v = ch / V;
    const float* from = red + (2 * (ch - v * V) + which) * RES_THREADS + v;
    float t = 0.f;
    for (int r = tid & 15; r < s.PR; r += 16) t += from[r * s.CV];
    t = row16_sum(t);
    if ((tid & 15) == 0) {
      (which ? tot[ch].y : tot[ch].x) = t;
      out[which * s.C + ch] = t;
    }
  }
  __syncthreads();
  if (!dx) return;
  const float inv = (float)(1.0 / ((double)s.HW * s.Cg));
  if (s.Cg <= 16) {                                      // a thread per group, else a wave
    for (int g = tid; g < sl.ng; g += RES_THREADS) {
      float t1 = 0.f, t2 = 0.f;
      for (int i = 0; i < s.Cg; i++) {
        const float w = gamma ? gamma[sl.c0 + g * s.Cg + i] : 1.f;
        t1 = fmaf(w, tot[g * s.Cg + i].x, t1);
        t2 = fmaf(w, tot[g * s.Cg + i].y, t2);
      }
      coef[g] = make_float2(t1 * inv, t2 * inv);
    }
  } else {
    for (int g = tid >> 6; g < sl.ng; g += RES_WAVES) {
      float t1 = 0.f, t2 = 0.f;
      for (int i = tid & 63; i < s.Cg; i += 64) {
        const float w = gamma ? gamma[sl.c0 + g * s.Cg + i] : 1.f;
        t1 = fmaf(w, tot[g * s.Cg + i].x, t1);
        t2 = fmaf(w, tot[g * s.Cg + i].y, t2);
      }
      t1 = wave_sum(t1);
      t2 = wave_sum(t2);
      if ((tid & 63) == 0) coef[g] = make_float2(t1 * inv, t2 * inv);
    }
  }
  __syncthreads();
  if (!on) return;
  const float2 m = coef[cv * V / s.Cg];
  const float q2 = rstd * rstd * m.y, q1 = fmaf(-lo, q2, rstd * m.x);
#pragma unroll
  for (int i = 0; i < NV; i++) {
    const int p = pr + i * s.PR;
    if (p < HW) {
      Vec<T, V> o;
#pragma unroll
      for (int j = 0; j < V; j++) {
        const float xf = to_f32(vx[i].t[j]);
        const float du = du_of<ACT>(xf, to_f32(vd[i].t[j]), k.mean[j], k.a[j], k.beta[j], c + j, s.Cg, stats, gamma, beta);
        o.t[j] = from_f32<T>(fmaf(du, k.a[j], -fmaf(xf - k.mean[j], q2, q1)));
      }
      *(typename Bits<T, V>::type*)(dx + base + (int64_t)p * s.C) = o.u;
    }
  }
}

// ---------------------------------------------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------------------------------------------
constexpr int64_t FWD_RUN = (int64_t)1 << 40;           // (its sums are 64-bit: no limit)

// Slabs for vectors of V channels; false when they would not start on a vector.
bool plan_slabs(Shape& s, int V) {
  if (s.C % V) return false;
  const int most = GN_THREADS * V;
  if (s.Cg <= most) {
    s.parts = 1;
    s.gps = most / s.Cg;
    if (s.gps >= s.G) {
      s.gps = s.G;
    } else {
      int step = 1;                                     // groups until a slab start is a multiple of V again
      while ((int64_t)step * s.Cg % V) step++;
      if (s.gps < step) return false;
      s.gps = s.gps / step * step;
    }
    s.slab_c = s.gps * s.Cg;
    s.slabs = cdiv(s.G, s.gps);
  } else {
    if (s.Cg % V) return false;
    s.gps = 1;
    s.slab_c = most;
    s.parts = cdiv(s.Cg, most);
    s.slabs = s.G * s.parts;
  }
  if (s.slab_c % V) return false;
  s.CV = s.slab_c / V;
  s.PR = GN_THREADS / s.CV;
  return true;
}

// The widest vector that the channel count, the slabs and the tensors' addresses allow; chunks so that the launch
// fills the chip eight times over but a thread still walks 4 pixels (one round of its loads), and `run` at most.
int plan(Shape& s, int B, int64_t HW, int C, int G, int esize, uintptr_t addr, int64_t run) {
  s.HW = HW;
  s.C = C;
  s.G = G;
  s.Cg = C / G;
  int V = 16 / esize;
  while (V > 1 && (addr % (V * esize) || !plan_slabs(s, V))) V >>= 1;
  if (V == 1) plan_slabs(s, 1);
  const int64_t most = (HW + (int64_t)s.PR * 4 - 1) / ((int64_t)s.PR * 4);
  int64_t want = (2048 + (int64_t)B * s.slabs - 1) / ((int64_t)B * s.slabs);
  if (want > most) want = most;
  if (want < 1) want = 1;
  if (HW > want * s.PR * run) want = (HW + s.PR * run - 1) / (s.PR * run);
  s.ppc = (HW + want - 1) / want;
  s.chunks = (int)((HW + s.ppc - 1) / s.ppc);
  return V;
}

// Slabs for the resident kernels: whole groups, vectors within a group, at most `most` vectors to a thread.  The widest
// slab that leaves 512 workgroups (or 256 bytes to a pixel) is taken; narrower ones read less of a memory line at a time
// but still meet the others of their sample in the XCD's L2.  Below 16 bytes to a pixel that costs more than the launches
// it saves (16x128x128^2 bf16 in 32 groups, 8 bytes: 74 us against 52), unless a thread holds 8 vectors at most.  Returns
// the vectors to a thread, 0 where the other kernels are to be used.
int plan_resident(Shape& s, int& V, int B, int64_t HW, int C, int G, int esize, uintptr_t addr, int most) {
  s.HW = HW;
  s.C = C;
  s.G = G;
  s.Cg = C / G;
  s.parts = s.chunks = 1;
  s.ppc = HW;
  V = 16 / esize;
  while (V > 1 && (addr % (V * esize) || s.Cg % V)) V >>= 1;
  const int GV = s.Cg / V;
  auto need = [&](int groups) -> int64_t {              // vectors to a thread
    const int CV = groups * GV;
    return CV > RES_WIDE ? INT64_MAX : (HW + RES_THREADS / CV - 1) / (RES_THREADS / CV);
  };
  if (HW > (1 << 20) || need(1) > most) return 0;
  int gps = 1;
  while (gps < G && (int64_t)gps * s.Cg * esize < 256 && need(gps + 1) <= most &&
         ((int64_t)gps * s.Cg * esize < 16 || (int64_t)B * cdiv(G, gps + 1) >= 512))
    gps++;
  if (need(gps) > 8 && gps < G && gps * s.Cg * esize < 16) return 0;
  s.gps = gps;
  s.slab_c = gps * s.Cg;
  s.slabs = cdiv(G, gps);
  s.CV = gps * GV;
  s.PR = RES_THREADS / s.CV;
  return (int)need(gps);
}

bool shape_ok(int dtype, int B, int64_t HW, int C, int G) {
  return (dtype == MIS_F32 || dtype == MIS_BF16) && B >= 1 && B <= 65535 && HW >= 1 && C >= 1 && G >= 1 && C % G == 0 &&
         C <= 65536 && G <= 65535 && HW <= ((int64_t)1 << 40);
}

template <typename F> void with_act(int act, F&& f) {
  switch (act) {
    case MIS_ACT_RELU: f(std::integral_constant<int, MIS_ACT_RELU>()); break;
    case MIS_ACT_SILU: f(std::integral_constant<int, MIS_ACT_SILU>()); break;
    case MIS_ACT_GELU: f(std::integral_constant<int, MIS_ACT_GELU>()); break;
    default: f(std::integral_constant<int, MIS_ACT_NONE>());
  }
}

constexpr int RES_FWD = 32, RES_BWD = 16;               // most vectors to a thread

// f(the next power of two from `n` on, at least 2, as a constant)
template <int MOST, typename F> void with_count(int n, F&& f) {
  if (n <= 2) f(std::integral_constant<int, 2>());
  else if (n <= 4) f(std::integral_constant<int, 4>());
  else if (n <= 8) f(std::integral_constant<int, 8>());
  else if (n <= 16) f(std::integral_constant<int, 16>());
  else f(std::integral_constant<int, MOST>());
}

// f(first sample, samples, workgroups) for each launch: a launch has 2^22 slabs at most (a launch holds below 2^32 threads).
template <typename F> void by_samples(const Shape& s, int B, F&& f) {
  const int most = std::max(1, (1 << 22) / s.slabs);
  for (int b = 0; b < B; b += most) {
    const int n = std::min(most, B - b);
    f((int64_t)b, n, (n * s.slabs + 7) / 8 * 8);
  }
}

template <typename T, int V>
void launch_resident_fwd(const T* x, const Shape& s, int nv, int B, const float* gamma, const float* beta, double eps, int act,
                         T* y, double2* stats, hipStream_t st) {
  const int64_t sample = s.HW * s.C;
  with_act(act, [&](auto a) {
    constexpr int ACT = decltype(a)::value;
    with_count<RES_FWD>(nv, [&](auto n) {
      by_samples(s, B, [&](int64_t b, int nb, int grid) {
        gn_resident_kernel<T, V, decltype(n)::value, ACT><<<grid, RES_THREADS, 0, st>>>(
            x + b * sample, s, nb, eps, gamma, beta, y + b * sample, stats + b * s.G);
      });
    });
  });
}

template <typename T, int V>
void launch_resident_bwd(const T* x, const T* dy, const Shape& s, int nv, int B, const float* gamma, const float* beta, int act,
                         const double2* stats, T* dx, float* dgamma, float* dbeta, float* chan, hipStream_t st) {
  const int64_t sample = s.HW * s.C;
  with_act(act, [&](auto a) {
    constexpr int ACT = decltype(a)::value;
    with_count<RES_BWD>(nv, [&](auto n) {
      by_samples(s, B, [&](int64_t b, int nb, int grid) {
        gn_resident_bwd_kernel<T, V, decltype(n)::value, ACT><<<grid, RES_THREADS, 0, st>>>(
            x + b * sample, dy + b * sample, s, nb, stats + b * s.G, gamma, beta, dx ? dx + b * sample : nullptr,
            chan + b * 2 * s.C);
      });
    });
  });
  if (dgamma || dbeta)
    gn_bwd_finish_kernel<<<cdiv(s.C, 64), 256, 0, st>>>(chan, gamma, B, s.C, s.Cg, s.G, 1.0, cdiv(s.C, 64), nullptr, dgamma, dbeta);
}

template <typename T, int V>
void launch_fwd(const T* x, const Shape& s, int B, const float* gamma, const float* beta, double eps, int act, T* y,
                double2* stats, double2* sums, hipStream_t st) {
  const dim3 grid(s.chunks, s.slabs, B);
  auto sum = [&](auto u) {
    constexpr int U = decltype(u)::value;
    gn_sums_kernel<T, V, U><<<grid, GN_THREADS, (size_t)s.PR * s.CV * (V / U) * sizeof(double2), st>>>(x, s, sums);
  };
  if (s.Cg % V == 0) sum(std::integral_constant<int, V>());
  else if (V >= 4 && s.Cg % (V / 2) == 0) sum(std::integral_constant<int, (V >= 4 ? V / 2 : 1)>());
  else sum(std::integral_constant<int, 1>());
  const bool fold = (s.parts == 1 ? s.gps : 1) <= FOLD_GROUPS && s.chunks * s.parts <= FOLD_ROWS;
  if (!fold) gn_stats_kernel<T><<<dim3(s.G, B), 64, 0, st>>>(x, s, sums, s.chunks * s.parts, s.G, (double)s.HW * s.Cg, eps, stats);
  with_act(act, [&](auto a) {
    constexpr int ACT = decltype(a)::value;
    if (fold) gn_apply_kernel<T, V, ACT, true><<<grid, GN_THREADS, 0, st>>>(x, s, sums, eps, stats, gamma, beta, y);
    else gn_apply_kernel<T, V, ACT, false><<<grid, GN_THREADS, 0, st>>>(x, s, sums, eps, stats, gamma, beta, y);
  });
}

struct BwdBuffers {
  float *rows, *chan;
  float2* coef;
};

template <typename T, int V, int ACT>
void launch_bwd_act(const T* x, const T* dy, const Shape& s, int B, const float* gamma, const float* beta,
                    const double2* stats, T* dx, float* dgamma, float* dbeta, const BwdBuffers& w, hipStream_t st) {
  const dim3 grid(s.chunks, s.slabs, B);
  const size_t lds = (size_t)s.PR * s.CV * V * sizeof(float2);
  gn_bwd_sums_kernel<T, V, ACT><<<grid, GN_THREADS, lds, st>>>(x, dy, s, stats, gamma, beta, w.rows);
  if (s.chunks > 64) gn_bwd_channels_kernel<32><<<dim3(cdiv(s.C, 32), B), 1024, 0, st>>>(w.rows, s.chunks, s.C, w.chan);
  else gn_bwd_channels_kernel<8><<<dim3(cdiv(s.C, 32), B), 256, 0, st>>>(w.rows, s.chunks, s.C, w.chan);
  const int channel_blocks = dgamma || dbeta ? cdiv(s.C, 64) : 0, coef_blocks = dx ? cdiv((int64_t)B * s.G, 4) : 0;
  if (channel_blocks + coef_blocks > 0)
    gn_bwd_finish_kernel<<<channel_blocks + coef_blocks, 256, 0, st>>>(w.chan, gamma, B, s.C, s.Cg, s.G, (double)s.HW * s.Cg,
                                                                      channel_blocks, w.coef, dgamma, dbeta);
  if (dx) gn_bwd_dx_kernel<T, V, ACT><<<grid, GN_THREADS, 0, st>>>(x, dy, s, stats, gamma, beta, w.coef, dx);
}

template <typename T, int V>
void launch_bwd(const T* x, const T* dy, const Shape& s, int B, const float* gamma, const float* beta, int act,
                const double2* stats, T* dx, float* dgamma, float* dbeta, const BwdBuffers& w, hipStream_t st) {
  with_act(act, [&](auto a) {
    launch_bwd_act<T, V, decltype(a)::value>(x, dy, s, B, gamma, beta, stats, dx, dgamma, dbeta, w, st);
  });
}

// Calls f(pointer type tag, vector width) for the planned width.
template <typename F>
void with_vector(int dtype, int V, F&& f) {
  if (dtype == MIS_BF16) {
    if (V == 8) f((bf16*)nullptr, std::integral_constant<int, 8>());
    else if (V == 4) f((bf16*)nullptr, std::integral_constant<int, 4>());
    else if (V == 2) f((bf16*)nullptr, std::integral_constant<int, 2>());
    else f((bf16*)nullptr, std::integral_constant<int, 1>());
  } else {
    if (V == 4) f((float*)nullptr, std::integral_constant<int, 4>());
    else if (V == 2) f((float*)nullptr, std::integral_constant<int, 2>());
    else f((float*)nullptr, std::integral_constant<int, 1>());
  }
}

// Workspace sizes hold for every vector width (a tensor's address may rule the widest out).
size_t fwd_bytes(int dtype, int B, int64_t HW, int C, int G) {
  size_t most = 0;
  for (uintptr_t addr = 2; addr <= 16; addr *= 2) {
    Shape s;
    plan(s, B, HW, C, G, dtype == MIS_BF16 ? 2 : 4, addr, FWD_RUN);
    const size_t n = (size_t)B * s.chunks * s.parts * s.G * sizeof(double2);
    if (n > most) most = n;
  }
  return align256(most);
}

size_t bwd_rows_bytes(int dtype, int B, int64_t HW, int C, int G) {
  size_t most = 0;
  for (uintptr_t addr = 2; addr <= 16; addr *= 2) {
    Shape s;
    plan(s, B, HW, C, G, dtype == MIS_BF16 ? 2 : 4, addr, BWD_RUN);
    const size_t n = (size_t)B * s.chunks * 2 * C * sizeof(float);
    if (n > most) most = n;
  }
  return align256(most);
}

}  // namespace

extern "C" {

size_t mis_group_norm_act_fwd_workspace_bytes(int dtype, int B, int64_t HW, int C, int G) {
  return shape_ok(dtype, B, HW, C, G) ? fwd_bytes(dtype, B, HW, C, G) : 0;
}

int mis_group_norm_act_fwd(const void* x, int dtype, int B, int64_t HW, int C, int G, const float* gamma, const float* beta,
                           double eps, int act, void* y, double* stats, void* workspace, mis_stream_t stream) {
  MIS_REQUIRE(shape_ok(dtype, B, HW, C, G), "group_norm_act_fwd: bad dtype or shape (B=%d HW=%lld C=%d groups=%d)", B,
              (long long)HW, C, G);
  MIS_REQUIRE(x && y && stats && workspace, "group_norm_act_fwd: null pointer");
  MIS_REQUIRE(act >= MIS_ACT_NONE && act <= MIS_ACT_GELU, "group_norm_act_fwd: unknown activation %d", act);
  MIS_REQUIRE(eps >= 0.0, "group_norm_act_fwd: eps must not be negative");
  MIS_REQUIRE((((uintptr_t)x | (uintptr_t)y) & (dtype == MIS_BF16 ? 1 : 3)) == 0 &&
              (((uintptr_t)stats | (uintptr_t)workspace) & 15) == 0, "group_norm_act_fwd: misaligned pointer");
  Shape s;
  const int es = dtype == MIS_BF16 ? 2 : 4;
  const uintptr_t addr = (uintptr_t)x | (uintptr_t)y | 16;
  int V;
  const int nv = plan_resident(s, V, B, HW, C, G, es, addr, RES_FWD);
  if (!nv) V = plan(s, B, HW, C, G, es, addr, FWD_RUN);
  with_vector(dtype, V, [&](auto* t, auto v) {
    typedef std::remove_pointer_t<decltype(t)> T;
    if (nv)
      return launch_resident_fwd<T, decltype(v)::value>((const T*)x, s, nv, B, gamma, beta, eps, act, (T*)y, (double2*)stats,
                                                        (hipStream_t)stream);
    launch_fwd<T, decltype(v)::value>((const T*)x, s, B, gamma, beta, eps, act, (T*)y, (double2*)stats, (double2*)workspace,
                                      (hipStream_t)stream);
  });
  MIS_CHECK_LAUNCH("group_norm_act_fwd");
  return MIS_OK;
}

size_t mis_group_norm_act_bwd_workspace_bytes(int dtype, int B, int64_t HW, int C, int G) {
  if (!shape_ok(dtype, B, HW, C, G)) return 0;
  return bwd_rows_bytes(dtype, B, HW, C, G) + align256((size_t)B * 2 * C * sizeof(float)) +
         align256((size_t)B * G * sizeof(float2));
}

int mis_group_norm_act_bwd(const void* x, const void* dy, int dtype, int B, int64_t HW, int C, int G, const float* gamma,
                           const float* beta, const double* stats, int act, void* dx, float* dgamma, float* dbeta,
                           void* workspace, mis_stream_t stream) {
  MIS_REQUIRE(shape_ok(dtype, B, HW, C, G), "group_norm_act_bwd: bad dtype or shape (B=%d HW=%lld C=%d groups=%d)", B,
              (long long)HW, C, G);
  MIS_REQUIRE(x && dy && stats && workspace, "group_norm_act_bwd: null pointer");
  MIS_REQUIRE(act >= MIS_ACT_NONE && act <= MIS_ACT_GELU, "group_norm_act_bwd: unknown activation %d", act);
  MIS_REQUIRE((((uintptr_t)x | (uintptr_t)dy | (uintptr_t)dx) & (dtype == MIS_BF16 ? 1 : 3)) == 0 &&
              (((uintptr_t)stats | (uintptr_t)workspace) & 15) == 0, "group_norm_act_bwd: misaligned pointer");
  Shape s;
  const int es = dtype == MIS_BF16 ? 2 : 4;
  const uintptr_t addr = (uintptr_t)x | (uintptr_t)dy | (uintptr_t)dx | 16;
  int V;
  const int nv = plan_resident(s, V, B, HW, C, G, es, addr, RES_BWD);
  if (!nv) V = plan(s, B, HW, C, G, es, addr, BWD_RUN);
  BwdBuffers w;
  char* ws = (char*)workspace;
  w.rows = (float*)ws;
  ws += bwd_rows_bytes(dtype, B, HW, C, G);
  w.chan = (float*)ws;
  ws += align256((size_t)B * 2 * C * sizeof(float));
  w.coef = (float2*)ws;
  with_vector(dtype, V, [&](auto* t, auto v) {
    typedef std::remove_pointer_t<decltype(t)> T;
    if (nv)
      return launch_resident_bwd<T, decltype(v)::value>((const T*)x, (const T*)dy, s, nv, B, gamma, beta, act,
                                                        (const double2*)stats, (T*)dx, dgamma, dbeta, w.chan,
                                                        (hipStream_t)stream);
    launch_bwd<T, decltype(v)::value>((const T*)x, (const T*)dy, s, B, gamma, beta, act, (const double2*)stats, (T*)dx,
                                      dgamma, dbeta, w, (hipStream_t)stream);
  });
  MIS_CHECK_LAUNCH("group_norm_act_bwd");
  return MIS_OK;
}

}  // extern "C"
