// Matrix product with bias, activation and residual in its epilogue, forward and backward.
//
//   u = x W^T + b;  y = act(u) + r                    x [M][K], W [N][K], b [N] float32, r and y [M][N]
//   dz = dy act'(u), u formed again;  dx = dz W;  dW = dz^T x;  db = sum over rows of dz;  dr = dy
//
// All products have one form, out[q][p] = sum over r of P(p, r) Q(q, r): the index p that is contiguous in the output
// takes the matrix instruction's row operand, so that a lane's accumulators are consecutive elements of one output row.
// Accumulation is float32; dz is rounded to the tensors' type once, as the operand of its two products (db is summed
// from the unrounded values).
#include "act.h"
#include "common.h"
#include "reduce.h"

namespace {

template <typename T> struct Operand {
  const T* p;
  int64_t s_row, s_k;       // element (row, k) at p[row*s_row + k*s_k]
  int rows;
};

enum Mode { FWD, DZ, STORE, PARTIAL };

template <typename T> struct Epilogue {
  const float* bias;        // [p]
  const T* other;           // residual (FWD, may be null) or dy (DZ): [q][p], row stride ld
  int64_t ld;
  T* out;                   // [q][p] dense
  float* rows;              // DZ: sums over a tile's q, [q tile][p];  PARTIAL: [split][q][p]
  int act;
};

template <typename F> __device__ __forceinline__ void with_act(int act, F&& f) {
  switch (act) {
    case MIS_ACT_RELU: f(std::integral_constant<int, MIS_ACT_RELU>()); break;
    case MIS_ACT_SILU: f(std::integral_constant<int, MIS_ACT_SILU>()); break;
    case MIS_ACT_GELU: f(std::integral_constant<int, MIS_ACT_GELU>()); break;
    default: f(std::integral_constant<int, MIS_ACT_NONE>());
  }
}

template <typename T> struct Mma;
template <> struct Mma<bf16> {
  static constexpr int K = 32, PER = 8;      // a lane holds 8 consecutive k of its row: k = 8 (lane / 16) + i
  typedef bf16x8 Frag;
  static __device__ __forceinline__ f32x4 mul(Frag a, Frag b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
};
template <> struct Mma<float> {
  static constexpr int K = 4, PER = 1;       // k = lane / 16
  typedef float Frag;
  static __device__ __forceinline__ f32x4 mul(Frag a, Frag b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0);
  }
};

// ---------------------------------------------------------------------------------------------------------------
// Any sizes, strides and alignments: 64 x 64 outputs per workgroup, elements staged one by one.
// ---------------------------------------------------------------------------------------------------------------
constexpr int ANY_T = 64, ANY_K = 32, ANY_PITCH = ANY_K + 8;

template <typename T>
__device__ __forceinline__ void any_stage(const Operand<T>& o, int row0, int64_t k0, int64_t k1, T (*tile)[ANY_PITCH]) {
  const int tid = threadIdx.x;
  if (o.s_k == 1) {
    const int row = tid >> 2, kk = (tid & 3) * 8;
#pragma unroll
    for (int i = 0; i < 8; i++) {
      const int64_t k = k0 + kk + i;
      tile[row][kk + i] = row0 + row < o.rows && k < k1 ? o.p[(row0 + row) * o.s_row + k] : (T)0.f;
    }
  } else {
    const int row = tid & 63, kk = (tid >> 6) * 8;
#pragma unroll
    for (int i = 0; i < 8; i++) {
      const int64_t k = k0 + kk + i;
      tile[row][kk + i] = row0 + row < o.rows && k < k1 ? o.p[(row0 + row) * o.s_row + k * o.s_k] : (T)0.f;
    }
  }
}

template <typename T, int MODE>
__global__ __launch_bounds__(256) void lin_any_kernel(Operand<T> P, Operand<T> Q, int64_t R, int64_t r_per_split, Epilogue<T> e) {
  __shared__ __attribute__((aligned(16))) T tp[ANY_T][ANY_PITCH], tq[ANY_T][ANY_PITCH];
  __shared__ float colsum[2][ANY_T];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int wp = (wave & 1) * 32, wq = (wave >> 1) * 32;
  const int p_tiles = (P.rows + ANY_T - 1) / ANY_T, q_tile = blockIdx.x / p_tiles;
  const int p0 = (blockIdx.x - q_tile * p_tiles) * ANY_T, q0 = q_tile * ANY_T;
  const int64_t r0 = (int64_t)blockIdx.y * r_per_split, r1 = min(r0 + r_per_split, R);
  f32x4 acc[2][2] = {};
  for (int64_t k0 = r0; k0 < r1; k0 += ANY_K) {
    any_stage(P, p0, k0, r1, tp);
    any_stage(Q, q0, k0, r1, tq);
    __syncthreads();
#pragma unroll
    for (int k = 0; k < ANY_K; k += Mma<T>::K) {
      typename Mma<T>::Frag a[2], b[2];
      const int kk = k + (lane >> 4) * Mma<T>::PER;
#pragma unroll
      for (int i = 0; i < 2; i++) {
        a[i] = *(const typename Mma<T>::Frag*)&tp[wp + i * 16 + (lane & 15)][kk];
        b[i] = *(const typename Mma<T>::Frag*)&tq[wq + i * 16 + (lane & 15)][kk];
      }
#pragma unroll
      for (int i = 0; i < 2; i++)
#pragma unroll
        for (int j = 0; j < 2; j++) acc[i][j] = Mma<T>::mul(a[i], b[j], acc[i][j]);
    }
    __syncthreads();
  }
  // a lane's values: p = 4 (lane / 16) + r, q = lane % 16 within each 16 x 16 block
  with_act(MODE == FWD || MODE == DZ ? e.act : MIS_ACT_NONE, [&](auto act) {
    constexpr int ACT = decltype(act)::value;
    float cs[2][4] = {};
#pragma unroll
    for (int j = 0; j < 2; j++) {
      const int64_t q = q0 + wq + j * 16 + (lane & 15);
#pragma unroll
      for (int i = 0; i < 2; i++) {
#pragma unroll
        for (int r = 0; r < 4; r++) {
          const int p = p0 + wp + i * 16 + (lane >> 4) * 4 + r;
          if (q >= Q.rows || p >= P.rows) continue;
          float v = acc[i][j][r];
          if constexpr (MODE == FWD || MODE == DZ) v += e.bias ? e.bias[p] : 0.f;
          if constexpr (MODE == FWD) {
            v = act_value<ACT>(v);
            if (e.other) v += to_f32(e.other[q * e.ld + p]);
          }
          if constexpr (MODE == DZ) {
            v = to_f32(e.other[q * e.ld + p]) * act_slope<ACT>(v);
            cs[i][r] += v;
          }
          if constexpr (MODE == PARTIAL) e.rows[((int64_t)blockIdx.y * Q.rows + q) * P.rows + p] = v;
          else e.out[q * P.rows + p] = from_f32<T>(v);
        }
      }
    }
    if constexpr (MODE == DZ) {
#pragma unroll
      for (int i = 0; i < 2; i++)
#pragma unroll
        for (int r = 0; r < 4; r++) {
          const float s = row16_sum(cs[i][r]);
          if ((lane & 15) == 0) colsum[wave >> 1][wp + i * 16 + (lane >> 4) * 4 + r] = s;
        }
    }
  });
  if constexpr (MODE == DZ) {
    __syncthreads();
    if (tid < ANY_T && p0 + tid < P.rows) e.rows[(int64_t)q_tile * P.rows + p0 + tid] = colsum[0][tid] + colsum[1][tid];
  }
}

// out[i] = sum over the splits, in their order
template <typename T>
__global__ __launch_bounds__(256) void lin_join_kernel(const float* __restrict__ part, int splits, int64_t n, T* __restrict__ out) {
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
    float s = 0.f;
    for (int k = 0; k < splits; k++) s += part[k * n + i];
    out[i] = from_f32<T>(s);
  }
}

// rows[chunk][N] = sums of a chunk's rows of d (row stride ld)
constexpr int SUM_ROWS = 256;
template <typename T>
__global__ __launch_bounds__(256) void lin_colsum_kernel(const T* __restrict__ d, int64_t ld, int64_t M, int N,
                                                         float* __restrict__ rows) {
  __shared__ float red[4][64];
  const int c = blockIdx.y * 64 + (threadIdx.x & 63), w = threadIdx.x >> 6;
  const int64_t m1 = min((int64_t)(blockIdx.x + 1) * SUM_ROWS, M);
  float s = 0.f;
  if (c < N)
    for (int64_t m = (int64_t)blockIdx.x * SUM_ROWS + w; m < m1; m += 4) s += to_f32(d[m * ld + c]);
  red[w][threadIdx.x & 63] = s;
  __syncthreads();
  if (w == 0 && c < N) rows[(int64_t)blockIdx.x * N + c] = (red[0][threadIdx.x] + red[1][threadIdx.x]) + (red[2][threadIdx.x] + red[3][threadIdx.x]);
}

// ---------------------------------------------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------------------------------------------
template <typename T, int MODE>
void launch_product(const Operand<T>& P, const Operand<T>& Q, int64_t R, int splits, const Epilogue<T>& e, hipStream_t st) {
  const int64_t per = ((R + splits - 1) / splits + ANY_K - 1) / ANY_K * ANY_K;
  lin_any_kernel<T, MODE><<<dim3(cdiv(P.rows, ANY_T) * cdiv(Q.rows, ANY_T), splits), 256, 0, st>>>(P, Q, R, per, e);
}

// Parts of the long sum of dW: enough workgroups to fill the chip twice, at least 256 rows to a part.
int wgrad_splits(int64_t M, int64_t N, int64_t K) {
  const int64_t tiles = (int64_t)cdiv(N, ANY_T) * cdiv(K, ANY_T);
  int64_t s = (512 + tiles - 1) / tiles;
  const int64_t most = (M + 255) / 256;
  if (s > most) s = most;
  return (int)(s < 1 ? 1 : s);
}

struct BwdPlan {
  size_t dz, rows, part, total;
  int splits;
};

BwdPlan bwd_plan(int dtype, int64_t M, int64_t N, int64_t K, int act) {
  BwdPlan p;
  const size_t es = dtype == MIS_BF16 ? 2 : 4;
  p.splits = wgrad_splits(M, N, K);
  p.dz = act == MIS_ACT_NONE ? 0 : align256((size_t)M * N * es);
  p.rows = align256((size_t)(act == MIS_ACT_NONE ? cdiv(M, SUM_ROWS) : cdiv(M, ANY_T)) * N * sizeof(float));
  p.part = p.splits > 1 ? align256((size_t)p.splits * N * K * sizeof(float)) : 0;
  p.total = p.dz + p.rows + p.part;
  return p;
}

bool sizes_ok(int dtype, int64_t M, int64_t N, int64_t K) {
  return (dtype == MIS_F32 || dtype == MIS_BF16) && M >= 1 && N >= 1 && K >= 1 && N <= 1 << 20 && K <= 1 << 20 &&
         M < ((int64_t)1 << 30) && (M + 63) / 64 * ((N > K ? N : K) + 63) / 64 < ((int64_t)1 << 31);
}

bool aligned(int dtype, std::initializer_list<const void*> ps) {
  uintptr_t m = 0;
  for (const void* p : ps) m |= (uintptr_t)p;
  return (m & (dtype == MIS_BF16 ? 1 : 3)) == 0;
}

template <typename T>
void forward(const T* x, int64_t ldx, const T* w, const float* bias, const T* r, int64_t ldr, int64_t M, int64_t N, int64_t K,
             int act, T* y, hipStream_t st) {
  launch_product<T, FWD>({w, K, 1, (int)N}, {x, ldx, 1, (int)M}, K, 1, {bias, r, ldr, y, nullptr, act}, st);
}

template <typename T>
void backward(const T* x, int64_t ldx, const T* w, const float* bias, const T* dy, int64_t ldd, int dtype, int64_t M, int64_t N,
              int64_t K, int act, T* dx, T* dw, float* db, char* ws, hipStream_t st) {
  const BwdPlan p = bwd_plan(dtype, M, N, K, act);
  T* dz = (T*)ws;
  float* rows = (float*)(ws + p.dz);
  float* part = (float*)(ws + p.dz + p.rows);
  const T* z = dy;
  int64_t ldz = ldd;
  if (act != MIS_ACT_NONE) {
    launch_product<T, DZ>({w, K, 1, (int)N}, {x, ldx, 1, (int)M}, K, 1, {bias, dy, ldd, dz, rows, act}, st);
    z = dz;
    ldz = N;
    if (db) launch_reduce_partials(rows, cdiv(M, ANY_T), (int)N, db, st);
  } else if (db) {
    lin_colsum_kernel<T><<<dim3(cdiv(M, SUM_ROWS), cdiv(N, 64)), 256, 0, st>>>(dy, ldd, M, (int)N, rows);
    launch_reduce_partials(rows, cdiv(M, SUM_ROWS), (int)N, db, st);
  }
  if (dx) launch_product<T, STORE>({w, 1, K, (int)K}, {z, ldz, 1, (int)M}, N, 1, {nullptr, nullptr, 0, dx, nullptr, 0}, st);
  if (dw) {
    const Operand<T> P{x, 1, ldx, (int)K}, Q{z, 1, ldz, (int)N};
    if (p.splits == 1) {
      launch_product<T, STORE>(P, Q, M, 1, {nullptr, nullptr, 0, dw, nullptr, 0}, st);
    } else {
      launch_product<T, PARTIAL>(P, Q, M, p.splits, {nullptr, nullptr, 0, nullptr, part, 0}, st);
      lin_join_kernel<T><<<ew_grid(N * K, 256), 256, 0, st>>>(part, p.splits, N * K, dw);
    }
  }
}

}  // namespace

extern "C" {

int mis_linear_act_fwd(const void* x, int64_t ldx, const void* w, const float* bias, const void* residual, int64_t ldr, int dtype,
                       int64_t M, int64_t N, int64_t K, int act, void* y, mis_stream_t stream) {
  MIS_REQUIRE(x && w && y, "linear_act_fwd: null pointer");
  MIS_REQUIRE(sizes_ok(dtype, M, N, K), "linear_act_fwd: bad dtype or sizes (M=%lld N=%lld K=%lld)", (long long)M, (long long)N,
              (long long)K);
  MIS_REQUIRE(ldx >= K && (!residual || ldr >= N), "linear_act_fwd: row stride below the row length");
  MIS_REQUIRE(act >= MIS_ACT_NONE && act <= MIS_ACT_GELU, "linear_act_fwd: unknown activation %d", act);
  MIS_REQUIRE(aligned(dtype, {x, w, residual, y}), "linear_act_fwd: misaligned pointer");
  hipStream_t st = (hipStream_t)stream;
  if (dtype == MIS_BF16)
    forward((const bf16*)x, ldx, (const bf16*)w, bias, (const bf16*)residual, ldr, M, N, K, act, (bf16*)y, st);
  else
    forward((const float*)x, ldx, (const float*)w, bias, (const float*)residual, ldr, M, N, K, act, (float*)y, st);
  MIS_CHECK_LAUNCH("linear_act_fwd");
  return MIS_OK;
}

size_t mis_linear_act_bwd_workspace_bytes(int dtype, int64_t M, int64_t N, int64_t K, int act) {
  return sizes_ok(dtype, M, N, K) ? bwd_plan(dtype, M, N, K, act).total : 0;
}

int mis_linear_act_bwd(const void* x, int64_t ldx, const void* w, const float* bias, const void* dy, int64_t ldd, int dtype,
                       int64_t M, int64_t N, int64_t K, int act, void* dx, void* dw, float* db, void* workspace,
                       mis_stream_t stream) {
  MIS_REQUIRE(x && w && dy && workspace, "linear_act_bwd: null pointer");
  MIS_REQUIRE(sizes_ok(dtype, M, N, K), "linear_act_bwd: bad dtype or sizes (M=%lld N=%lld K=%lld)", (long long)M, (long long)N,
              (long long)K);
  MIS_REQUIRE(ldx >= K && ldd >= N, "linear_act_bwd: row stride below the row length");
  MIS_REQUIRE(act >= MIS_ACT_NONE && act <= MIS_ACT_GELU, "linear_act_bwd: unknown activation %d", act);
  MIS_REQUIRE(aligned(dtype, {x, w, dy, dx, dw}) && ((uintptr_t)workspace & 15) == 0, "linear_act_bwd: misaligned pointer");
  hipStream_t st = (hipStream_t)stream;
  if (dtype == MIS_BF16)
    backward((const bf16*)x, ldx, (const bf16*)w, bias, (const bf16*)dy, ldd, dtype, M, N, K, act, (bf16*)dx, (bf16*)dw, db,
             (char*)workspace, st);
  else
    backward((const float*)x, ldx, (const float*)w, bias, (const float*)dy, ldd, dtype, M, N, K, act, (float*)dx, (float*)dw, db,
             (char*)workspace, st);
  MIS_CHECK_LAUNCH("linear_act_bwd");
  return MIS_OK;
}

}  // extern "C"
