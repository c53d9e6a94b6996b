// AdamW over many tensors with both moments held in 8 bits, and the total gradient norm it may clip to.
//
//   g *= min(1, max_norm / (|g| + 1e-6));  m = b1 m + (1-b1) g;  v = b2 v + (1-b2) g^2
//   p = p (1 - lr wd) - lr/(1-b1^t) * m / (sqrt(v)/sqrt(1-b2^t) + eps)      with the m, v just formed, not their codes
//
// Storage of the moments: 128 consecutive elements share a byte s, the exponent of their top binade [1, 2) 2^(s-127).
// m: sign, 4 exponent bits, 3 mantissa bits; v: 4 exponent bits, 4 mantissa bits; the lowest binade is linear down to
// zero.  s is the smallest with which no element has to be clamped (0: all elements are zero; 255: one is not finite
// or beyond the top code of the largest binade, and all 128 read back as NaN).  Magnitudes below 2^-126 count as zero.
// Rounding to a code is stochastic: with round-to-nearest the relative step of a second moment, 1 - b2 = 0.001, would
// never move a 4-bit mantissa; a carried random number moves it with the right probability.  The random numbers are
// Philox4x32-10 (Salmon et al. 2011), key = seed, counter = (element / 4, step): one 32-bit word per element, low half
// for m, high half for v; a code depends on nothing but its inputs, the seed and the step.  A second moment that is
// not zero never becomes zero (the update divides by its root).
//
// The moments are formed in 64 bits (as fast as 32 here) and rounded to float once: a code then differs from the
// exact formula's only where 2^-50 decides.
//
// HBM-bound: parameter read and written, gradient read (twice when clipping: the norm comes first), four code bytes
// and a 64th of that in scales per element: 16 (20) bytes per float32 element against 28 (32) with float32 moments.
// At that rate the vector units have about 100 instruction slots per element, so their number is kept down: codes are
// decoded by a table of doubles in LDS, exclusive-ors are three-operand, blocks whose values are too small or not finite
// take a slow way of their own, and a workgroup walks neighbouring chunks with the next one's loads under way.
#include "common.h"

namespace {

constexpr int A8_THREADS = 256;
constexpr int A8_CHUNK = 4096;        // MIS_OPT_CHUNK
constexpr int A8_PARTIALS = 1024;     // partial sums of the norm: few enough for every workgroup to add up
constexpr int A8_GRID = 2048;         // most workgroups of a step: what the chip holds at once, each with a run of chunks

struct Desc8 {
  void* p;
  const void* g;
  int64_t off, n;                     // element offset in the flat moment buffers (a multiple of 128), elements
  int64_t dtype;                      // of p and g
};

struct Step8 {                        // what changes from step to step
  float decay, step_size, inv_bc2;    // 1 - lr wd, lr / (1-b1^t), 1 / sqrt(1-b2^t)
  uint32_t step_lo, step_hi;
};

struct Args8 {
  Step8 s;
  double b1, omb1, b2, omb2;
  float eps;
  double max_norm;
  uint32_t seed_lo, seed_hi;
};

__device__ __forceinline__ int tensor_of(const int* __restrict__ prefix, int n_tensors, int chunk) {
  int lo = 0, hi = n_tensors;         // prefix[lo] <= chunk < prefix[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (prefix[mid] <= chunk) lo = mid; else hi = mid;
  }
  return lo;
}

__device__ __forceinline__ double sum_of_block(double v, double* red) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, WAVE);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  double s = 0.0;
  for (int w = 0; w < A8_THREADS / 64; w++) s += red[w];
  __syncthreads();
  return s;
}

template <typename T>
__device__ __forceinline__ void store8(T* __restrict__ p, int64_t e, int64_t n, bool wide, const float (&f)[8]) {
  if (wide && e + 8 <= n) {
    if constexpr (sizeof(T) == 4) {
      *(float4*)(p + e) = make_float4(f[0], f[1], f[2], f[3]);
      *(float4*)(p + e + 4) = make_float4(f[4], f[5], f[6], f[7]);
    } else {
      bf16x8 a;
#pragma unroll
      for (int i = 0; i < 8; i++) a[i] = (bf16)f[i];
      *(bf16x8*)(p + e) = a;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; i++)
      if (e + i < n) p[e + i] = from_f32<T>(f[i]);
  }
}

// Eight consecutive elements as they lie in memory; those from n on as zeros.
template <typename T> struct Raw8 {
  static constexpr int W = sizeof(T) / 2;
  uint4 u[W];
  __device__ __forceinline__ void load(const T* __restrict__ p, int64_t e, int64_t n, bool wide) {
    if (wide && e + 8 <= n) {
#pragma unroll
      for (int i = 0; i < W; i++) u[i] = ((const uint4*)(p + e))[i];
    } else {
      union { uint4 u[W]; T t[8]; } x;
#pragma unroll
      for (int i = 0; i < 8; i++) x.t[i] = e + i < n ? p[e + i] : (T)0.f;
#pragma unroll
      for (int i = 0; i < W; i++) u[i] = x.u[i];
    }
  }
  __device__ __forceinline__ void floats(float (&f)[8]) const {
    union { uint4 u[W]; T t[8]; } x;
#pragma unroll
    for (int i = 0; i < W; i++) x.u[i] = u[i];
#pragma unroll
    for (int i = 0; i < 8; i++) f[i] = to_f32(x.t[i]);
  }
};

// A workgroup's run of chunks, and the tensor that the current one lies in.
struct Walk {
  const int* prefix;
  int c, end, t;
  __device__ __forceinline__ Walk(const int* prefix_, int n_tensors, int first, int n, int wg, int wgs) : prefix(prefix_) {
    const int per = n / wgs, more = n - per * wgs;       // the first `more` workgroups take one chunk more
    c = first + wg * per + min(wg, more);
    end = c + per + (wg < more ? 1 : 0);
    t = c < end ? tensor_of(prefix, n_tensors, c) : 0;
  }
  __device__ __forceinline__ void next() {
    c++;
    while (c < end && prefix[t + 1] <= c) t++;
  }
};

template <typename T>
__device__ __forceinline__ double chunk_sqsum(const T* __restrict__ g, int64_t e0, int64_t n) {
  constexpr int N = A8_CHUNK / (A8_THREADS * 8);
  const bool wide = ((uintptr_t)g & 15) == 0;
  Raw8<T> r[N];
#pragma unroll
  for (int it = 0; it < N; it++) {
    const int64_t e = e0 + (it * A8_THREADS + threadIdx.x) * 8;
    if (e < n) r[it].load(g, e, n, wide);
    else r[it] = Raw8<T>{};
  }
  double s = 0.0;
#pragma unroll
  for (int it = 0; it < N; it++) {
    float f[8];
    r[it].floats(f);
#pragma unroll
    for (int i = 0; i < 8; i++) s = fma((double)f[i], (double)f[i], s);
  }
  return s;
}

// partials[workgroup] = its share of sum g^2, in 64 bits.  64 M float32 elements (256 MB) 87 us behind a kernel whose output
// is still being written back, 60 at best (4.3 TB/s).
__global__ __launch_bounds__(A8_THREADS) void adamw8_sqsum_kernel(const Desc8* __restrict__ descs,
                                                                  const int* __restrict__ prefix, int n_tensors,
                                                                  int n_chunks, double* __restrict__ partials) {
  __shared__ double red[A8_THREADS / 64];
  double s = 0.0;
  for (Walk w(prefix, n_tensors, 0, n_chunks, blockIdx.x, gridDim.x); w.c < w.end; w.next()) {
    const Desc8 d = descs[w.t];
    const int64_t e0 = (int64_t)(w.c - prefix[w.t]) * A8_CHUNK;
    s += d.dtype == MIS_F32 ? chunk_sqsum((const float*)d.g, e0, d.n) : chunk_sqsum((const bf16*)d.g, e0, d.n);
  }
  s = sum_of_block(s, red);
  if (threadIdx.x == 0) partials[blockIdx.x] = s;
}

__device__ __forceinline__ uint32_t xor3(uint32_t a, uint32_t b, uint32_t c) {
#ifdef __HIP_DEVICE_COMPILE__
  return __builtin_amdgcn_bitop3_b32(a, b, c, 0x96);
#else
  return a ^ b ^ c;
#endif
}

// Philox4x32-10: four words for the counter (c0, c1, c2, c3) under the key (k0, k1).
__device__ __forceinline__ void philox10(uint32_t (&c)[4], uint32_t k0, uint32_t k1) {
#pragma unroll
  for (int r = 0; r < 10; r++) {
    const uint64_t p = (uint64_t)c[0] * 0xD2511F53u, q = (uint64_t)c[2] * 0xCD9E8D57u;
    const uint32_t n0 = xor3((uint32_t)(q >> 32), c[1], k0), n2 = xor3((uint32_t)(p >> 32), c[3], k1);
    c[1] = (uint32_t)q;
    c[3] = (uint32_t)p;
    c[0] = n0;
    c[2] = n2;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
}

// A code shifted to the top of a float's mantissa and exponent fields reads as value * 2^-112 (the linear binade as a
// subnormal float, which the conversion to 64 bits keeps), so the block's factor is 2^(s - 127 + 112).
__device__ __forceinline__ double block_factor(uint32_t s) {
  const uint64_t b = s == 0 ? 0ull : s == 255 ? 0x7FF8000000000000ull : (uint64_t)(s + 1023 - 15) << 52;
  return __builtin_bit_cast(double, b);
}
__device__ __forceinline__ float m_code_float(uint32_t k) {
  return __builtin_bit_cast(float, (k & 0x7Fu) << 20 | (k & 0x80u) << 24);
}
__device__ __forceinline__ float v_code_float(uint32_t k) { return __builtin_bit_cast(float, k << 19); }

__device__ __forceinline__ uint32_t row16_max(uint32_t v) {
  auto step = [](uint32_t a, uint32_t b) { return a > b ? a : b; };
  v = step(v, __builtin_amdgcn_update_dpp(0, v, 0xB1, 0xF, 0xF, true));
  v = step(v, __builtin_amdgcn_update_dpp(0, v, 0x4E, 0xF, 0xF, true));
  v = step(v, __builtin_amdgcn_update_dpp(0, v, 0x141, 0xF, 0xF, true));
  return step(v, __builtin_amdgcn_update_dpp(0, v, 0x140, 0xF, 0xF, true));
}

// |x| as float bits, numbers below 2^-126 as zero
__device__ __forceinline__ uint32_t mag_bits(float x) {
  const uint32_t b = __builtin_bit_cast(uint32_t, x) & 0x7FFFFFFFu;
  return b < 0x00800000u ? 0u : b;
}

// The code of magnitude `b` (float bits) in a block of exponent s, for a code of 23 - DROP mantissa bits; r < 2^DROP.
// Above the lowest binade the code is the float's exponent (rebased) and top mantissa bits, below it the value in
// units of the smallest step: both as integers with DROP bits to be rounded, to which r is added.
template <int DROP>
__device__ __forceinline__ uint32_t code_of(uint32_t b, int s, uint32_t r) {
  const int t = (int)b - ((s - 15) << 23);
  const uint32_t low = (uint32_t)ldexpf(__builtin_bit_cast(float, b), 164 - s);
  return ((b != 0 && t >= (1 << 23) ? (uint32_t)t : low) + r) >> DROP;
}

// The same for SAFE <= s < 255 without the special cases: the mantissa is shifted down to the block's linear binade.
// Zero and numbers below 2^-126 have exponent field 0 and are shifted by at least 24 bits: they give 0 by themselves.
constexpr uint32_t SAFE = 40;
template <int DROP>
__device__ __forceinline__ uint32_t safe_code_of(uint32_t b, uint32_t s, uint32_t r) {
  const int shift = (int)(s - 14) - (int)(b >> 23);
  const uint32_t low = ((b & 0x007FFFFFu) | 0x00800000u) >> min(shift, 31);
  return ((shift > 0 ? low : b - ((s - 15) << 23)) + r) >> DROP;
}

__device__ __forceinline__ uint32_t bytes4(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  return a | b << 8 | c << 16 | d << 24;
}

// What a thread holds of its 8 elements before the update, raw.
template <typename T> struct Item {
  Raw8<T> p, g;
  uint2 m, v;
  uint32_t sm, sv;
  int64_t e;              // first element within the tensor; behind the padded tensor: nothing to do
};

struct Buffers8 {
  uint8_t *m, *ms, *v, *vs;
};

template <typename T>
__device__ __forceinline__ void fetch(Item<T>& x, const Desc8& d, int64_t e, const Buffers8& b) {
  x.e = e;
  if (e >= ((d.n + 127) & ~(int64_t)127)) return;        // (all 16 lanes of a block, or none)
  const int64_t f = d.off + e;
  x.g.load((const T*)d.g, e, d.n, ((uintptr_t)d.g & 15) == 0);
  x.p.load((const T*)d.p, e, d.n, ((uintptr_t)d.p & 15) == 0);
  x.m = *(const uint2*)(b.m + f);
  x.v = *(const uint2*)(b.v + f);
  x.sm = b.ms[f >> 7];
  x.sv = b.vs[f >> 7];
}

// c1 = (1-b1) coef, c2 = (1-b2) coef^2; m_table, v_table: what the codes stand for in a block of exponent 127
template <typename T>
__device__ __forceinline__ void update(const Item<T>& x, const Desc8& d, const Args8& a, const Step8& st, double c1, double c2,
                                       const double* m_table, const double* v_table, const Buffers8& buf) {
  if (x.e >= ((d.n + 127) & ~(int64_t)127)) return;
  const int64_t f = d.off + x.e;
  float p[8], g[8];
  x.p.floats(p);
  x.g.floats(g);
  const double fm = a.b1 * block_factor(x.sm), fv = a.b2 * block_factor(x.sv);
  uint32_t rnd[8];
#pragma unroll
  for (int h = 0; h < 2; h++) {
    const uint64_t q = (uint64_t)(f >> 2) + h;
    uint32_t c[4] = {(uint32_t)q, (uint32_t)(q >> 32), st.step_lo, st.step_hi};
    philox10(c, a.seed_lo, a.seed_hi);
#pragma unroll
    for (int i = 0; i < 4; i++) rnd[4 * h + i] = c[i];
  }
  float m[8], v[8];
  uint32_t mb[8], vb[8], mmax = 0, vmax = 0;
#pragma unroll
  for (int i = 0; i < 8; i++) {
    const uint32_t km = ((i < 4 ? x.m.x : x.m.y) >> 8 * (i & 3)) & 255, kv = ((i < 4 ? x.v.x : x.v.y) >> 8 * (i & 3)) & 255;
    const double gd = (double)g[i];
    m[i] = (float)fma(c1, gd, fm * m_table[km]);
    v[i] = (float)fma(c2, gd * gd, fv * v_table[kv]);
    const float denom = fmaf(__builtin_amdgcn_sqrtf(v[i]), st.inv_bc2, a.eps);
    p[i] = fmaf(p[i], st.decay, -st.step_size * (m[i] * __builtin_amdgcn_rcpf(denom)));
    mb[i] = __builtin_bit_cast(uint32_t, m[i]) & 0x7FFFFFFFu;
    vb[i] = __builtin_bit_cast(uint32_t, v[i]);
    mmax = max(mmax, mb[i]);
    vmax = max(vmax, vb[i]);
  }
  store8((T*)d.p, x.e, d.n, ((uintptr_t)d.p & 15) == 0, p);
  mmax = row16_max(mmax);
  vmax = row16_max(vmax);
  uint32_t sm = min((mmax + 0x000FFFFFu) >> 23, 255u), sv = min((vmax + 0x0007FFFFu) >> 23, 255u);
  uint32_t qm[8], qv[8];
  if (__builtin_expect(sm - SAFE < 255 - SAFE && sv - SAFE < 255 - SAFE, 1)) {
#pragma unroll
    for (int i = 0; i < 8; i++) {
      qm[i] = safe_code_of<20>(mb[i], sm, (rnd[i] << 4 & 0xFFFF0u) | 8u);
      qv[i] = safe_code_of<19>(vb[i], sv, (rnd[i] >> 13 & 0x7FFF8u) | 4u);
      if (vb[i] >= 0x00800000u) qv[i] = max(qv[i], 1u);
      qm[i] |= __builtin_bit_cast(uint32_t, m[i]) >> 24 & 0x80u;
    }
  } else {                                     // tiny, zero or not finite
    mmax = vmax = 0;
#pragma unroll
    for (int i = 0; i < 8; i++) {
      mb[i] = mag_bits(m[i]);
      vb[i] = mag_bits(v[i]);
      mmax = max(mmax, mb[i]);
      vmax = max(vmax, vb[i]);
    }
    sm = min((row16_max(mmax) + 0x000FFFFFu) >> 23, 255u);
    sv = min((row16_max(vmax) + 0x0007FFFFu) >> 23, 255u);
#pragma unroll
    for (int i = 0; i < 8; i++) {
      qm[i] = sm == 255 ? 0u : code_of<20>(mb[i], (int)sm, (rnd[i] << 4 & 0xFFFF0u) | 8u);
      qv[i] = sv == 255 ? 0u : code_of<19>(vb[i], (int)sv, (rnd[i] >> 13 & 0x7FFF8u) | 4u);
      if (qv[i] == 0 && vb[i] != 0 && sv != 255) qv[i] = 1;
      qm[i] |= __builtin_bit_cast(uint32_t, m[i]) >> 24 & 0x80u;
    }
  }
  *(uint2*)(buf.m + f) = make_uint2(bytes4(qm[0], qm[1], qm[2], qm[3]), bytes4(qm[4], qm[5], qm[6], qm[7]));
  *(uint2*)(buf.v + f) = make_uint2(bytes4(qv[0], qv[1], qv[2], qv[3]), bytes4(qv[4], qv[5], qv[6], qv[7]));
  if ((threadIdx.x & 15) == 0) {
    buf.ms[f >> 7] = (uint8_t)sm;
    buf.vs[f >> 7] = (uint8_t)sv;
  }
}

// The chunks of a run that lie in tensors of one type: half a chunk at a time, the next half's loads before the update.
template <typename T>
__device__ __forceinline__ void adamw8_run(Walk& w, Desc8& d, const Desc8* __restrict__ descs, const Args8& a, const Step8& st,
                                           double c1, double c2, const double* m_table, const double* v_table,
                                           const Buffers8& buf) {
  constexpr int HALF = A8_THREADS * 8;
  Item<T> x, y;
  Desc8 dx = d, dy;
  fetch(x, dx, (int64_t)(w.c - w.prefix[w.t]) * A8_CHUNK + threadIdx.x * 8, buf);
  while (true) {
    fetch(y, dx, x.e + HALF, buf);
    update(x, dx, a, st, c1, c2, m_table, v_table, buf);
    const int64_t ey = y.e;
    const int t = w.t;
    w.next();
    const bool more = w.c < w.end;
    dy = dx;
    if (more && w.t != t) d = dy = descs[w.t];
    const bool same = more && dy.dtype == dx.dtype;
    if (same) fetch(x, dy, (int64_t)(w.c - w.prefix[w.t]) * A8_CHUNK + threadIdx.x * 8, buf);
    update(y, dx, a, st, c1, c2, m_table, v_table, buf);
    if (!same) return;
    dx = dy;
  }
}

// 64 M float32 elements (1.03 GB) in 185 to 203 us, 5.1 to 5.5 TB/s, a copy's rate, at 68 vector instructions an element and
// 70 % of the issue slots; 5 M bf16 elements in 22 us; the 2.9 M of a U-Net in 74 tensors in 16 us.
__global__ __launch_bounds__(A8_THREADS) void adamw8_step_kernel(const Desc8* __restrict__ descs,
                                                                 const int* __restrict__ prefix, int n_tensors, int chunk0,
                                                                 int n_chunks, Args8 a, const Step8* __restrict__ dyn,
                                                                 const double* __restrict__ partials, int n_partials,
                                                                 Buffers8 buf, float* __restrict__ norm_out) {
  __shared__ double red[A8_THREADS / 64], m_table[256], v_table[256];
  const Step8 st = dyn ? *dyn : a.s;
  for (int k = threadIdx.x; k < 256; k += A8_THREADS) {
    m_table[k] = (double)m_code_float(k);
    v_table[k] = (double)v_code_float(k);
  }
  double coef = 1.0;
  if (partials) {                              // every workgroup: the same sum in the same order
    double s = 0.0;
    for (int i = threadIdx.x; i < n_partials; i += A8_THREADS) s += partials[i];
    const double norm = sqrt(sum_of_block(s, red));
    coef = a.max_norm / (norm + 1e-6);
    if (coef > 1.0) coef = 1.0;                // (NaN stays NaN)
    if (a.max_norm <= 0.0) coef = 1.0;
    if (norm_out && blockIdx.x == 0 && threadIdx.x == 0) norm_out[0] = (float)norm;
  } else {
    __syncthreads();
  }
  const double c1 = a.omb1 * coef, c2 = a.omb2 * coef * coef;
  Walk w(prefix, n_tensors, chunk0, n_chunks, blockIdx.x, gridDim.x);
  if (w.c >= w.end) return;
  Desc8 d = descs[w.t];
  while (w.c < w.end) {
    if (d.dtype == MIS_F32) adamw8_run<float>(w, d, descs, a, st, c1, c2, m_table, v_table, buf);
    else adamw8_run<bf16>(w, d, descs, a, st, c1, c2, m_table, v_table, buf);
  }
}

// The moments that the codes stand for: 4 elements a thread at a time.  64 M elements (642 MB) in 119 us, 5.4 TB/s.
__global__ __launch_bounds__(A8_THREADS) void adamw8_moments_kernel(const uint32_t* __restrict__ mc, const uint8_t* __restrict__ msc,
                                                                    const uint32_t* __restrict__ vc, const uint8_t* __restrict__ vsc,
                                                                    int64_t n4, float4* __restrict__ m, float4* __restrict__ v) {
  const int64_t stride = (int64_t)gridDim.x * A8_THREADS;
#pragma unroll 2
  for (int64_t i = (int64_t)blockIdx.x * A8_THREADS + threadIdx.x; i < n4; i += stride) {
    const uint32_t km = mc[i], kv = vc[i];
    const int sm = msc[i >> 5], sv = vsc[i >> 5];
    // 2^(s-15) times the code as a float; a factor of NaN or zero for s = 255 and 0
    const float om = sm == 255 ? __builtin_nanf("") : sm == 0 ? 0.f : 1.f, ov = sv == 255 ? __builtin_nanf("") : sv == 0 ? 0.f : 1.f;
    float fm[4], fv[4];
#pragma unroll
    for (int k = 0; k < 4; k++) {
      fm[k] = om * ldexpf(m_code_float(km >> 8 * k & 255), sm - 15);
      fv[k] = ov * ldexpf(v_code_float(kv >> 8 * k & 255), sv - 15);
    }
    m[i] = make_float4(fm[0], fm[1], fm[2], fm[3]);
    v[i] = make_float4(fv[0], fv[1], fv[2], fv[3]);
  }
}

void step_constants(double lr, double b1, double b2, double wd, int64_t step, Step8* s) {
  s->decay = (float)(1.0 - lr * wd);
  s->step_size = (float)(lr / (1.0 - pow(b1, (double)step)));
  s->inv_bc2 = (float)(1.0 / sqrt(1.0 - pow(b2, (double)step)));
  s->step_lo = (uint32_t)step;
  s->step_hi = (uint32_t)((uint64_t)step >> 32);
}

}  // namespace

extern "C" {

size_t mis_adamw8_workspace_bytes(void) { return A8_PARTIALS * sizeof(double); }

int mis_adamw8_sqsum(const void* descs, const int* chunk_prefix, int n_tensors, int n_chunks, void* workspace,
                     mis_stream_t stream) {
  MIS_REQUIRE(descs && chunk_prefix && workspace && n_tensors >= 1 && n_chunks >= 1, "adamw8_sqsum: bad arguments");
  const int grid = n_chunks < A8_PARTIALS ? n_chunks : A8_PARTIALS;
  adamw8_sqsum_kernel<<<grid, A8_THREADS, 0, (hipStream_t)stream>>>((const Desc8*)descs, chunk_prefix, n_tensors, n_chunks,
                                                                    (double*)workspace);
  MIS_CHECK_LAUNCH("adamw8_sqsum");
  return MIS_OK;
}

int mis_adamw8_step_constants(double lr, double beta1, double beta2, double weight_decay, int64_t step, void* host_out) {
  MIS_REQUIRE(host_out && step >= 1, "adamw8_step_constants: bad arguments");
  step_constants(lr, beta1, beta2, weight_decay, step, (Step8*)host_out);
  return MIS_OK;
}

int mis_adamw8_step(const void* descs, const int* chunk_prefix, int n_tensors, int chunk_begin, int chunk_end, int n_chunks,
                    void* exp_avg, void* exp_avg_scale, void* exp_avg_sq, void* exp_avg_sq_scale, const void* norm_workspace,
                    double max_norm, double lr, double beta1, double beta2, double eps, double weight_decay, int64_t step,
                    uint64_t seed, const void* step_constants_dev, float* total_norm, mis_stream_t stream) {
  MIS_REQUIRE(descs && chunk_prefix && n_tensors >= 1 && exp_avg && exp_avg_scale && exp_avg_sq && exp_avg_sq_scale,
              "adamw8_step: null pointer");
  MIS_REQUIRE(((uintptr_t)exp_avg & 7) == 0 && ((uintptr_t)exp_avg_sq & 7) == 0, "adamw8_step: misaligned moment buffers");
  MIS_REQUIRE(0 <= chunk_begin && chunk_begin < chunk_end && chunk_end <= n_chunks, "adamw8_step: bad chunk range");
  MIS_REQUIRE(beta1 >= 0. && beta1 < 1. && beta2 >= 0. && beta2 < 1., "adamw8_step: bad betas");
  MIS_REQUIRE(step_constants_dev || step >= 1, "adamw8_step: bad step");
  Args8 a;
  if (step_constants_dev) a.s = Step8{};
  else step_constants(lr, beta1, beta2, weight_decay, step, &a.s);
  a.b1 = beta1;
  a.omb1 = 1.0 - beta1;
  a.b2 = beta2;
  a.omb2 = 1.0 - beta2;
  a.eps = (float)eps;
  a.max_norm = max_norm;
  a.seed_lo = (uint32_t)seed;
  a.seed_hi = (uint32_t)(seed >> 32);
  const Buffers8 buf{(uint8_t*)exp_avg, (uint8_t*)exp_avg_scale, (uint8_t*)exp_avg_sq, (uint8_t*)exp_avg_sq_scale};
  const int chunks = chunk_end - chunk_begin, grid = chunks < A8_GRID ? chunks : A8_GRID;
  adamw8_step_kernel<<<grid, A8_THREADS, 0, (hipStream_t)stream>>>(
      (const Desc8*)descs, chunk_prefix, n_tensors, chunk_begin, chunks, a, (const Step8*)step_constants_dev,
      (const double*)norm_workspace, n_chunks < A8_PARTIALS ? n_chunks : A8_PARTIALS, buf, total_norm);
  MIS_CHECK_LAUNCH("adamw8_step");
  return MIS_OK;
}

int mis_adamw8_moments(const void* exp_avg, const void* exp_avg_scale, const void* exp_avg_sq, const void* exp_avg_sq_scale,
                       int64_t n_blocks, float* out_avg, float* out_sq, mis_stream_t stream) {
  MIS_REQUIRE(exp_avg && exp_avg_scale && exp_avg_sq && exp_avg_sq_scale && out_avg && out_sq && n_blocks >= 1,
              "adamw8_moments: bad arguments");
  MIS_REQUIRE((((uintptr_t)exp_avg | (uintptr_t)exp_avg_sq) & 7) == 0 && (((uintptr_t)out_avg | (uintptr_t)out_sq) & 15) == 0,
              "adamw8_moments: misaligned pointer");
  const int64_t n4 = n_blocks * 32;
  int64_t grid = (n4 + A8_THREADS - 1) / A8_THREADS;
  if (grid > 16384) grid = 16384;
  adamw8_moments_kernel<<<(int)grid, A8_THREADS, 0, (hipStream_t)stream>>>(
      (const uint32_t*)exp_avg, (const uint8_t*)exp_avg_scale, (const uint32_t*)exp_avg_sq, (const uint8_t*)exp_avg_sq_scale, n4,
      (float4*)out_avg, (float4*)out_sq);
  MIS_CHECK_LAUNCH("adamw8_moments");
  return MIS_OK;
}

}  // extern "C"
