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
#include "common.h"

namespace {

constexpr int A8_THREADS = 256;
constexpr int A8_CHUNK = 4096;        // MIS_OPT_CHUNK
constexpr int A8_PARTIALS = 1024;     // partial sums of the norm: few enough for every workgroup to add up

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

// Eight consecutive elements; those from n on read as zero.
template <typename T>
__device__ __forceinline__ void load8(const T* __restrict__ p, int64_t e, int64_t n, bool wide, float (&f)[8]) {
  if (wide && e + 8 <= n) {
    if constexpr (sizeof(T) == 4) {
      const float4 a = *(const float4*)(p + e), b = *(const float4*)(p + e + 4);
      f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w;
      f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
    } else {
      const bf16x8 a = *(const bf16x8*)(p + e);
#pragma unroll
      for (int i = 0; i < 8; i++) f[i] = (float)a[i];
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; i++) f[i] = e + i < n ? to_f32(p[e + i]) : 0.f;
  }
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

template <typename T>
__device__ __forceinline__ double chunk_sqsum(const T* __restrict__ g, int64_t e0, int64_t n) {
  const bool wide = ((uintptr_t)g & 15) == 0;
  double s = 0.0;
#pragma unroll
  for (int it = 0; it < A8_CHUNK / (A8_THREADS * 8); it++) {
    const int64_t e = e0 + (it * A8_THREADS + threadIdx.x) * 8;
    if (e < n) {
      float f[8];
      load8(g, e, n, wide, f);
#pragma unroll
      for (int i = 0; i < 8; i++) s = fma((double)f[i], (double)f[i], s);
    }
  }
  return s;
}

__global__ __launch_bounds__(A8_THREADS) void adamw8_sqsum_kernel(const Desc8* __restrict__ descs,
                                                                  const int* __restrict__ prefix, int n_tensors,
                                                                  int n_chunks, double* __restrict__ partials) {
  __shared__ double red[A8_THREADS / 64];
  double s = 0.0;
  for (int c = blockIdx.x; c < n_chunks; c += gridDim.x) {
    const int t = tensor_of(prefix, n_tensors, c);
    const Desc8 d = descs[t];
    const int64_t e0 = (int64_t)(c - prefix[t]) * A8_CHUNK;
    s += d.dtype == MIS_F32 ? chunk_sqsum((const float*)d.g, e0, d.n) : chunk_sqsum((const bf16*)d.g, e0, d.n);
  }
  s = sum_of_block(s, red);
  if (threadIdx.x == 0) partials[blockIdx.x] = s;
}

// Philox4x32-10: four words for the counter (c0, c1, c2, c3) under the key (k0, k1).
__device__ __forceinline__ void philox10(uint32_t (&c)[4], uint32_t k0, uint32_t k1) {
#pragma unroll
  for (int r = 0; r < 10; r++) {
    const uint64_t p = (uint64_t)c[0] * 0xD2511F53u, q = (uint64_t)c[2] * 0xCD9E8D57u;
    const uint32_t n0 = (uint32_t)(q >> 32) ^ c[1] ^ k0, n2 = (uint32_t)(p >> 32) ^ c[3] ^ k1;
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

template <typename T>
__device__ __forceinline__ void adamw8_chunk(const Desc8& d, int64_t e0, const Args8& a, const Step8& st, double coef,
                                             uint8_t* __restrict__ mc, uint8_t* __restrict__ msc, uint8_t* __restrict__ vc,
                                             uint8_t* __restrict__ vsc) {
  T* P = (T*)d.p;
  const T* G = (const T*)d.g;
  const bool pw = ((uintptr_t)P & 15) == 0, gw = ((uintptr_t)G & 15) == 0;
  const int64_t padded = (d.n + 127) & ~(int64_t)127;
#pragma unroll
  for (int it = 0; it < A8_CHUNK / (A8_THREADS * 8); it++) {
    const int64_t e = e0 + (it * A8_THREADS + threadIdx.x) * 8;
    if (e >= padded) continue;                 // (all 16 lanes of a block, or none)
    const int64_t f = d.off + e;
    float p[8], g[8];
    load8(G, e, d.n, gw, g);
    load8((const T*)P, e, d.n, pw, p);
    union { uint2 u; uint8_t b[8]; } km, kv;
    km.u = *(const uint2*)(mc + f);
    kv.u = *(const uint2*)(vc + f);
    const double fm = a.b1 * block_factor(msc[f >> 7]), fv = a.b2 * block_factor(vsc[f >> 7]);
    uint32_t rnd[8];
#pragma unroll
    for (int h = 0; h < 2; h++) {
      const uint64_t q = (uint64_t)(f >> 2) + h;
      uint32_t c[4] = {(uint32_t)q, (uint32_t)(q >> 32), st.step_lo, st.step_hi};
      philox10(c, a.seed_lo, a.seed_hi);
#pragma unroll
      for (int i = 0; i < 4; i++) rnd[4 * h + i] = c[i];
    }
    uint32_t mb[8], vb[8], sign[8], mmax = 0, vmax = 0;
#pragma unroll
    for (int i = 0; i < 8; i++) {
      const double gd = (double)g[i] * coef;
      const float m = (float)fma(fm, (double)m_code_float(km.b[i]), a.omb1 * gd);
      const float v = (float)fma(fv, (double)v_code_float(kv.b[i]), a.omb2 * gd * gd);
      const float denom = fmaf(__builtin_amdgcn_sqrtf(v), st.inv_bc2, a.eps);
      p[i] = fmaf(p[i], st.decay, -st.step_size * (m * __builtin_amdgcn_rcpf(denom)));
      mb[i] = mag_bits(m);
      vb[i] = mag_bits(v);
      sign[i] = __builtin_bit_cast(uint32_t, m) >> 31;
      mmax = max(mmax, mb[i]);
      vmax = max(vmax, vb[i]);
    }
    store8(P, e, d.n, pw, p);
    const uint32_t sm = min((row16_max(mmax) + 0x000FFFFFu) >> 23, 255u);
    const uint32_t sv = min((row16_max(vmax) + 0x0007FFFFu) >> 23, 255u);
#pragma unroll
    for (int i = 0; i < 8; i++) {
      const uint32_t qm = code_of<20>(mb[i], (int)sm, (rnd[i] & 0xFFFFu) << 4 | 8u);
      uint32_t qv = code_of<19>(vb[i], (int)sv, (rnd[i] >> 16) << 3 | 4u);
      if (qv == 0 && vb[i] != 0) qv = 1;
      km.b[i] = (uint8_t)((sm == 255 ? 0u : qm) | sign[i] << 7);
      kv.b[i] = (uint8_t)(sv == 255 ? 0u : qv);
    }
    *(uint2*)(mc + f) = km.u;
    *(uint2*)(vc + f) = kv.u;
    if ((threadIdx.x & 15) == 0) {
      msc[f >> 7] = (uint8_t)sm;
      vsc[f >> 7] = (uint8_t)sv;
    }
  }
}

__global__ __launch_bounds__(A8_THREADS) void adamw8_step_kernel(const Desc8* __restrict__ descs,
                                                                 const int* __restrict__ prefix, int n_tensors, int chunk0,
                                                                 Args8 a, const Step8* __restrict__ dyn,
                                                                 const double* __restrict__ partials, int n_partials,
                                                                 uint8_t* __restrict__ mc, uint8_t* __restrict__ msc,
                                                                 uint8_t* __restrict__ vc, uint8_t* __restrict__ vsc,
                                                                 float* __restrict__ norm_out) {
  __shared__ double red[A8_THREADS / 64];
  const Step8 st = dyn ? *dyn : a.s;
  double coef = 1.0;
  if (partials) {                              // every workgroup: the same sum in the same order
    double s = 0.0;
    for (int i = threadIdx.x; i < n_partials; i += A8_THREADS) s += partials[i];
    const double norm = sqrt(sum_of_block(s, red));
    coef = a.max_norm / (norm + 1e-6);
    if (coef > 1.0) coef = 1.0;                // (NaN stays NaN)
    if (a.max_norm <= 0.0) coef = 1.0;
    if (norm_out && blockIdx.x == 0 && threadIdx.x == 0) norm_out[0] = (float)norm;
  }
  const int chunk = chunk0 + blockIdx.x;
  const int t = tensor_of(prefix, n_tensors, chunk);
  const Desc8 d = descs[t];
  const int64_t e0 = (int64_t)(chunk - prefix[t]) * A8_CHUNK;
  if (d.dtype == MIS_F32) adamw8_chunk<float>(d, e0, a, st, coef, mc, msc, vc, vsc);
  else adamw8_chunk<bf16>(d, e0, a, st, coef, mc, msc, vc, vsc);
}

// The moments that the codes stand for.
__global__ __launch_bounds__(A8_THREADS) void adamw8_moments_kernel(const uint8_t* __restrict__ mc, const uint8_t* __restrict__ msc,
                                                                    const uint8_t* __restrict__ vc, const uint8_t* __restrict__ vsc,
                                                                    int64_t n8, float* __restrict__ m, float* __restrict__ v) {
  for (int64_t i = (int64_t)blockIdx.x * A8_THREADS + threadIdx.x; i < n8; i += (int64_t)gridDim.x * A8_THREADS) {
    union { uint2 u; uint8_t b[8]; } km, kv;
    km.u = *(const uint2*)(mc + i * 8);
    kv.u = *(const uint2*)(vc + i * 8);
    const double fm = block_factor(msc[i >> 4]), fv = block_factor(vsc[i >> 4]);
    float om[8], ov[8];
#pragma unroll
    for (int k = 0; k < 8; k++) {
      om[k] = (float)(fm * (double)m_code_float(km.b[k]));
      ov[k] = (float)(fv * (double)v_code_float(kv.b[k]));
    }
    store8(m, i * 8, n8 * 8, true, om);
    store8(v, i * 8, n8 * 8, true, ov);
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
  adamw8_step_kernel<<<chunk_end - chunk_begin, A8_THREADS, 0, (hipStream_t)stream>>>(
      (const Desc8*)descs, chunk_prefix, n_tensors, chunk_begin, a, (const Step8*)step_constants_dev,
      (const double*)norm_workspace, n_chunks < A8_PARTIALS ? n_chunks : A8_PARTIALS, (uint8_t*)exp_avg,
      (uint8_t*)exp_avg_scale, (uint8_t*)exp_avg_sq, (uint8_t*)exp_avg_sq_scale, total_norm);
  MIS_CHECK_LAUNCH("adamw8_step");
  return MIS_OK;
}

int mis_adamw8_moments(const void* exp_avg, const void* exp_avg_scale, const void* exp_avg_sq, const void* exp_avg_sq_scale,
                       int64_t n_blocks, float* out_avg, float* out_sq, mis_stream_t stream) {
  MIS_REQUIRE(exp_avg && exp_avg_scale && exp_avg_sq && exp_avg_sq_scale && out_avg && out_sq && n_blocks >= 1,
              "adamw8_moments: bad arguments");
  MIS_REQUIRE((((uintptr_t)exp_avg | (uintptr_t)exp_avg_sq) & 7) == 0 && (((uintptr_t)out_avg | (uintptr_t)out_sq) & 15) == 0,
              "adamw8_moments: misaligned pointer");
  const int64_t n8 = n_blocks * 16;
  int64_t grid = (n8 + A8_THREADS - 1) / A8_THREADS;
  if (grid > 8192) grid = 8192;
  adamw8_moments_kernel<<<(int)grid, A8_THREADS, 0, (hipStream_t)stream>>>(
      (const uint8_t*)exp_avg, (const uint8_t*)exp_avg_scale, (const uint8_t*)exp_avg_sq, (const uint8_t*)exp_avg_sq_scale, n8,
      out_avg, out_sq);
  MIS_CHECK_LAUNCH("adamw8_moments");
  return MIS_OK;
}

}  // extern "C"
