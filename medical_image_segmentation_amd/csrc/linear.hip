// Matrix product with bias, activation and residual in its epilogue, forward and backward.
//
//   u = x W^T + b;  y = act(u) + r                    x [M][K], W [N][K], b [N] float32, r and y [M][N]
//   dz = dy act'(u), u formed again;  dx = dz W;  dW = dz^T x;  db = sum over rows of dz;  dr = dy
//
// All products have one form, out[q][p] = sum over r of P(p, r) Q(q, r): the index p that is contiguous in the output
// takes the matrix instruction's row operand, so that a lane's accumulators are consecutive elements of one output row.
// Accumulation is float32; dz is rounded to the tensors' type once, as the operand of its two products (db is summed
// from the unrounded values).  In bf16 that is the price of the matrix instructions: they take no wider operand, and dz as a
// sum of two bf16 would double both products and dz's bytes (16384x512 -> 2048, training, 225 us: by their times about 90 more).
// dx and dW are then off from the exact ones by two roundings in place of one, 1.4 times as far in norm (0.0023 against 0.0017
// for that product).
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
  T* out;                   // [q][p], row stride ld_out; columns from the operand's rows up to `cols` are set to zero
  int64_t ld_out;
  int cols;
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
// Tiles staged straight from memory into LDS (16-byte chunks; sizes, strides and addresses multiples of 16 bytes).
//
// A workgroup of WP x WQ waves owns TP x TQ outputs and walks r in steps of 128 bytes (64 bf16, 32 float32).  Two
// stages of LDS (four for the 64-edge, which is used where few workgroups are left to hide a load behind): while the
// matrix instructions work on one, buffer loads with an LDS destination fill the others; one barrier a stage.  Chunks
// outside the operand get an offset behind the buffer's end and arrive as zeros.
//
// Rows of an operand that is contiguous in r are 128 bytes of LDS; a fragment read takes the same 16-byte chunk of 16
// rows, so chunk c of row i lies at c ^ ((i / 2) % 8): 16 rows, 16 different 16-byte windows of the 256 bytes of banks.
// An operand that is contiguous in its rows ("transposed", for the two products of the backward pass) is staged as
// [r][row].  bf16: ds_read_b64_tr_b16 hands lane i of 16 the column i of a 4 x 16 block; a half-wave reads 8 r-rows of
// 32 bytes, spread over the banks by the r bits that differ between them.  float32: plain 4-byte reads, 64 bytes wide,
// four r-rows apart.
// The loads put an LDS line in the order of the lanes, so the permutation is applied to the addresses they read.
// ---------------------------------------------------------------------------------------------------------------
typedef __attribute__((ext_vector_type(4))) uint32_t u32x4;
typedef __attribute__((address_space(3))) void lds_void;
typedef __attribute__((address_space(3))) bf16x4 lds_bf16x4;
constexpr uint32_t OUTSIDE = 0x80000000u;
constexpr int ROW_BYTES = 128;

// (by value: a __builtin_bit_cast of a vector's element in place takes the first one)
__device__ __forceinline__ float as_float(uint32_t u) { return __builtin_bit_cast(float, u); }
__device__ __forceinline__ uint32_t as_bits(float f) { return __builtin_bit_cast(uint32_t, f); }

__device__ __forceinline__ __amdgpu_buffer_rsrc_t buffer_at(const void* p) {
  return __builtin_amdgcn_make_buffer_rsrc((void*)p, 0, 0x7FFFFFF0, 0x00020000);
}

// 16 bytes per lane from `off` on to consecutive LDS addresses (this wave's from `lds`)
__device__ __forceinline__ void to_lds(__amdgpu_buffer_rsrc_t rs, char* lds, uint32_t off) {
#ifdef __HIP_DEVICE_COMPILE__          // (the host pass does not know the 16-byte form and drops the kernel without a word)
  __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (lds_void*)lds, 16, off, 0, 0, 0);
#endif
}

// Where the 16-byte chunk `c` of r-row `k` lies in a transposed tile W rows wide.
template <typename T, int W>
__device__ __forceinline__ int tr_chunk(int k, int c) {
  if constexpr (sizeof(T) == 2) {               // by 32-byte units
    if constexpr (W * 2 >= 256) return c ^ (((k & 3) | (k >> 1 & 4)) << 1);
    else return c ^ (((k >> 1 & 1) | (k >> 2 & 2)) << 1);
  } else {
    return c ^ ((k >> 2 & 3) << 2);             // by 64-byte units
  }
}

// One operand's share of a stage: TR false: W rows of 128 bytes; true: 128 / sizeof(T) r-rows of W elements.
template <typename T, int W, bool TR, int THREADS> struct Stager {
  static constexpr int BYTES = W * ROW_BYTES, N = BYTES / 16 / THREADS, K = ROW_BYTES / (int)sizeof(T);
  uint32_t off[N];        // byte offset of this thread's chunks from the operand's first staged element
  int k[N];               // their first r within the stage

  __device__ __forceinline__ void init(const Operand<T>& o, int row0) {
#pragma unroll
    for (int i = 0; i < N; i++) {
      const int chunk = i * THREADS + threadIdx.x;
      if constexpr (!TR) {
        const int row = chunk >> 3, c = (chunk & 7) ^ (row >> 1 & 7);
        k[i] = c * (16 / (int)sizeof(T));
        off[i] = row0 + row < o.rows ? (uint32_t)((int64_t)row * o.s_row * sizeof(T)) + c * 16 : OUTSIDE;
      } else {
        constexpr int CR = W * (int)sizeof(T) / 16;           // chunks of an r-row
        k[i] = chunk / CR;
        const int c = tr_chunk<T, W>(k[i], chunk % CR);
        off[i] = row0 + c * (16 / (int)sizeof(T)) < o.rows ? (uint32_t)((int64_t)k[i] * o.s_k * sizeof(T)) + c * 16 : OUTSIDE;
      }
    }
  }

  // `first`: the operand's element (row0, r0 of the stage); left = r elements from there on
  __device__ __forceinline__ void issue(const T* first, int64_t left, char* lds) const {
    const __amdgpu_buffer_rsrc_t rs = buffer_at(first);
    const int wave_base = __builtin_amdgcn_readfirstlane((threadIdx.x & ~63) * 16);
    const bool whole = left >= K;
#pragma unroll
    for (int i = 0; i < N; i++) to_lds(rs, lds + i * THREADS * 16 + wave_base, whole || k[i] < left ? off[i] : OUTSIDE);
  }
};

// The fragment of 16 rows from `row` on, half `h` (64 bytes of r) of a stage.  bf16: k = 32 h + 8 g + e; float32:
// k = 16 h + 4 g + e (e-th instruction), g = lane / 16.
template <typename T, int W, bool TR>
__device__ __forceinline__ u32x4 fragment(const char* tile, int row, int h) {
  const int lane = threadIdx.x & 63, g = lane >> 4, j = lane & 15;
  if constexpr (!TR) {
    const int r = row + j;
    return *(const u32x4*)(tile + r * ROW_BYTES + (((4 * h + g) ^ (r >> 1 & 7)) << 4));
  } else if constexpr (sizeof(T) == 2) {
    union { bf16x4 b[2]; u32x4 u; } f;
#pragma unroll
    for (int i = 0; i < 2; i++) {
      const int k = 32 * h + 8 * g + 4 * i + (j >> 2), col = row + 4 * (j & 3);
      f.b[i] = __builtin_amdgcn_ds_read_tr16_b64_v4bf16(
          (lds_bf16x4*)(tile + k * W * 2 + (tr_chunk<T, W>(k, col >> 3) << 4) + (col & 4) * 2));
    }
    return f.u;
  } else {
    u32x4 f;
#pragma unroll
    for (int e = 0; e < 4; e++) {
      const int k = 16 * h + 4 * g + e, col = row + j;
      f[e] = *(const uint32_t*)(tile + k * W * 4 + (tr_chunk<T, W>(k, col >> 2) << 4) + (col & 3) * 4);
    }
    return f;
  }
}

__device__ __forceinline__ f32x4 multiply(u32x4 a, u32x4 b, f32x4 c, bf16) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 multiply(u32x4 a, u32x4 b, f32x4 c, float) {
#pragma unroll
  for (int e = 0; e < 4; e++) c = __builtin_amdgcn_mfma_f32_16x16x4f32(as_float(a[e]), as_float(b[e]), c, 0, 0, 0);
  return c;
}

// 4 (float32) or 8 (bf16) consecutive elements, 16 bytes
template <typename T> struct Pack {
  static constexpr int N = 16 / sizeof(T);
  float v[N];
  __device__ __forceinline__ void load(const T* p) {
    union { u32x4 u; T t[N]; } x;
    x.u = *(const u32x4*)p;
#pragma unroll
    for (int i = 0; i < N; i++) v[i] = to_f32(x.t[i]);
  }
  __device__ __forceinline__ void store(T* p) const {
    union { u32x4 u; T t[N]; } x;
#pragma unroll
    for (int i = 0; i < N; i++) x.t[i] = from_f32<T>(v[i]);
    *(u32x4*)p = x.u;
  }
};

// Tile number -> (p tile, q tile, split).  Workgroups go round-robin over the 8 XCDs; each XCD gets a run of
// neighbouring tiles (its own L2 then holds a few rows of both operands): QGROUP q tiles side by side, p slower.
constexpr int XCDS = 8, QGROUP = 4;
struct Grid {
  int p_tiles, q_tiles, splits;
  int64_t r_per_split;
  __host__ __device__ int total() const { return p_tiles * q_tiles * splits; }
  __host__ __device__ int launch() const { return (total() + XCDS - 1) / XCDS * XCDS; }
};

// All but the last N loads of this wave have arrived, its LDS reads are done, and all waves are here.
template <int N> __device__ __forceinline__ void wait_and_meet() {
#ifdef __HIP_DEVICE_COMPILE__
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
#endif
}

// Measured, bf16: 8192x4096 -> 4096 with ReLU and residual 237 us, 1.16 PFLOP/s with the 256-edge: the matrix units are busy in
// 54 % of the cycles, at 2.02 GHz; of the waves' cycles 33 % go to waits (the barrier of a stage and its loads), 47 % to waiting
// for an issue slot, no LDS bank conflicts.  With sums of a few hundred the epilogue's stores, which the workgroups of a round
// make at the same time, take as long as the products: 16384x512 -> 2048 with GELU 62 us (550 TFLOP/s), dz 79, dx 42 (810),
// dW 46 + 9 for the join.  float32: 4551x100 -> 252 in 12 us.
template <typename T, int TP, int TQ, int WP, int WQ, int STAGES, bool PTR, bool QTR, int MODE, bool WIDE>
__global__ __launch_bounds__(64 * WP * WQ, 2) void lin_tile_kernel(Operand<T> P, Operand<T> Q, int64_t R, Grid grid,
                                                                   Epilogue<T> e) {
  constexpr int THREADS = 64 * WP * WQ, BP = TP / WP / 16, BQ = TQ / WQ / 16, K = ROW_BYTES / (int)sizeof(T);
  static_assert(BP >= BQ, "the second half's fragments of both operands are read in BP steps");
  constexpr int STAGE = (TP + TQ) * ROW_BYTES;
  extern __shared__ __attribute__((aligned(1024))) char lds[];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g = lane >> 4;
  const int wp = (wave % WP) * (TP / WP), wq = (wave / WP) * (TQ / WQ);

  const int total = grid.total(), per = grid.launch() / XCDS;
  const int id = ((int)blockIdx.x % XCDS) * per + (int)blockIdx.x / XCDS;
  if (id >= total) return;
  const int tiles = grid.p_tiles * grid.q_tiles, split = id / tiles;
  int t = id - split * tiles;
  const int group = t / (QGROUP * grid.p_tiles), gq = min(QGROUP, grid.q_tiles - group * QGROUP);
  t -= group * QGROUP * grid.p_tiles;
  const int q_tile = group * QGROUP + t % gq, p_tile = t / gq;
  const int p0 = p_tile * TP, q0 = q_tile * TQ;
  const int64_t r0 = (int64_t)split * grid.r_per_split, r1 = min(r0 + grid.r_per_split, R);

  Stager<T, TP, PTR, THREADS> sp;
  Stager<T, TQ, QTR, THREADS> sq;
  sp.init(P, p0);
  sq.init(Q, q0);
  const T* pp = P.p + (int64_t)p0 * P.s_row + r0 * P.s_k;
  const T* qp = Q.p + (int64_t)q0 * Q.s_row + r0 * Q.s_k;

  f32x4 acc[BP][BQ] = {};
  int64_t left = r1 - r0;                   // from the next stage to be loaded on; stages behind the end are loaded as zeros
  auto load = [&](int buf) {
    sp.issue(pp, left, lds + buf * STAGE);
    sq.issue(qp, left, lds + buf * STAGE + TP * ROW_BYTES);
    pp += K * P.s_k;
    qp += K * Q.s_k;
    left -= K;
  };
#pragma unroll
  for (int i = 0; i < STAGES - 1; i++) load(i);
  int cur = 0;
  for (int64_t r = r0; r < r1; r += K) {
    wait_and_meet<(STAGES - 2) * (sp.N + sq.N)>();       // this stage is here; nobody reads the one before it any more
    load(cur == 0 ? STAGES - 1 : cur - 1);
    const char* tp = lds + cur * STAGE;
    const char* tq = tp + TP * ROW_BYTES;
    // The second half's fragments are read between the products of the first: the compiler on its own reads each just
    // before its use (8192x4096->4096 forward and its two backward products 238, 265, 247 -> 232, 247, 234 us).
    u32x4 a[2][BP], b[2][BQ];
#pragma unroll
    for (int j = 0; j < BQ; j++) b[0][j] = fragment<T, TQ, QTR>(tq, wq + 16 * j, 0);
#pragma unroll
    for (int i = 0; i < BP; i++) a[0][i] = fragment<T, TP, PTR>(tp, wp + 16 * i, 0);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < BP; i++) {
#pragma unroll
      for (int j = 0; j < BQ; j++) acc[i][j] = multiply(a[0][i], b[0][j], acc[i][j], T());
      a[1][i] = fragment<T, TP, PTR>(tp, wp + 16 * i, 1);
      if (i < BQ) b[1][i] = fragment<T, TQ, QTR>(tq, wq + 16 * i, 1);
      __builtin_amdgcn_sched_barrier(0);
    }
#pragma unroll
    for (int i = 0; i < BP; i++)
#pragma unroll
      for (int j = 0; j < BQ; j++) acc[i][j] = multiply(a[1][i], b[1][j], acc[i][j], T());
    cur = cur + 1 == STAGES ? 0 : cur + 1;
  }
  wait_and_meet<0>();                       // (no load may reach LDS that this workgroup no longer owns)

  // A lane has p = 4 g + 0..3 of every 16 x 16 block, q = lane % 16.  For 16-byte accesses in bf16 the lanes of two
  // neighbouring blocks trade halves (v_permlane16_swap): 8 consecutive p of one block each.
  // WIDE false: some row or column does not fit 16-byte accesses; the same values, element by element.
  constexpr bool TRADE = sizeof(T) == 2 && MODE != PARTIAL;
  constexpr int NV = TRADE ? 8 : 4, PAIRS = TRADE ? BP / 2 : BP;
  const int cols = MODE == PARTIAL ? P.rows : e.cols;
  with_act(MODE == FWD || MODE == DZ ? e.act : MIS_ACT_NONE, [&](auto act) {
    constexpr int ACT = decltype(act)::value;
#pragma unroll
    for (int i = 0; i < PAIRS; i++) {
      const int pl = wp + (TRADE ? 32 * i + 16 * (g & 1) + 8 * (g >> 1) : 16 * i + 4 * g), p = p0 + pl;
      float bias[NV], cs[NV];
#pragma unroll
      for (int k = 0; k < NV; k++) {
        bias[k] = 0.f;
        cs[k] = 0.f;
      }
      if constexpr (MODE == FWD || MODE == DZ)
        if (e.bias && p < P.rows)
#pragma unroll
          for (int k = 0; k < NV; k++) bias[k] = WIDE || p + k < P.rows ? e.bias[p + k] : 0.f;
#pragma unroll
      for (int j = 0; j < BQ; j++) {
        float v[NV];
        if constexpr (TRADE) {
#pragma unroll
          for (int k = 0; k < 4; k++) {
            const auto s = __builtin_amdgcn_permlane16_swap(as_bits(acc[2 * i][j][k]), as_bits(acc[2 * i + 1][j][k]), false, false);
            v[k] = as_float(s[0]);
            v[k + 4] = as_float(s[1]);
          }
        } else {
#pragma unroll
          for (int k = 0; k < 4; k++) v[k] = acc[i][j][k];
        }
        const int64_t q = q0 + wq + 16 * j + (lane & 15);
        if (p >= cols || q >= Q.rows) continue;
        auto value = [&](int k, float x) {                   // x: the residual or dy
          if constexpr (MODE == FWD) return act_value<ACT>(v[k] + bias[k]) + x;
          if constexpr (MODE == DZ) {
            const float d = x * act_slope<ACT>(v[k] + bias[k]);
            cs[k] += d;
            return d;
          }
          return v[k];
        };
        if constexpr (WIDE) {
          if constexpr (MODE == PARTIAL) {
            *(f32x4*)(e.rows + ((int64_t)split * Q.rows + q) * P.rows + p) = f32x4{v[0], v[1], v[2], v[3]};
          } else {
            Pack<T> o, x;
#pragma unroll
            for (int k = 0; k < NV; k++) x.v[k] = 0.f;
            if constexpr (MODE == FWD)
              if (e.other) x.load(e.other + q * e.ld + p);
            if constexpr (MODE == DZ) x.load(e.other + q * e.ld + p);
#pragma unroll
            for (int k = 0; k < NV; k++) o.v[k] = value(k, x.v[k]);
            o.store(e.out + q * e.ld_out + p);
          }
        } else {
#pragma unroll
          for (int k = 0; k < NV; k++) {
            if (p + k >= cols) continue;
            const bool in = p + k < P.rows;
            if constexpr (MODE == PARTIAL) {
              e.rows[((int64_t)split * Q.rows + q) * P.rows + p + k] = v[k];
            } else {
              float x = 0.f;
              if constexpr (MODE == FWD || MODE == DZ)
                if (e.other && in) x = to_f32(e.other[q * e.ld + p + k]);
              e.out[q * e.ld_out + p + k] = in ? from_f32<T>(value(k, x)) : (T)0.f;
            }
          }
        }
      }
      if constexpr (MODE == DZ) {
        float* colsum = (float*)lds;                         // [WQ][TP]; the stages are done
#pragma unroll
        for (int k = 0; k < NV; k++) {
          const float s = row16_sum(cs[k]);
          if ((lane & 15) == 0) colsum[(wave / WP) * TP + pl + k] = s;
        }
      }
    }
  });
  if constexpr (MODE == DZ) {
    const float* colsum = (const float*)lds;
    __syncthreads();
    for (int c = threadIdx.x; c < TP && p0 + c < P.rows; c += THREADS) {
      float s = 0.f;
#pragma unroll
      for (int w = 0; w < WQ; w++) s += colsum[w * TP + c];
      e.rows[(int64_t)q_tile * P.rows + p0 + c] = s;
    }
  }
}

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

// Bound by its element loads: a stage of 128 bytes takes 2 to 6 us where the staged kernel takes 0.2 to 0.5.  For products
// too small to pay for padded copies (4x25 -> 678: 6 us), and for rows that are whole 16-byte chunks long but start or step off
// 16 bytes, which get no copy whatever their size: 8192x4096 -> 4096 bf16 from rows three elements off takes 5.9 ms, 0.25 from a
// contiguous copy.
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
          if (q >= Q.rows || p >= (MODE == PARTIAL ? P.rows : e.cols)) continue;
          float v = acc[i][j][r];
          if (p >= P.rows) {
            v = 0.f;
          } else {
            if constexpr (MODE == FWD || MODE == DZ) v += e.bias ? e.bias[p] : 0.f;
            if constexpr (MODE == FWD) {
              v = act_value<ACT>(v);
              if (e.other) v += to_f32(e.other[q * e.ld + p]);
            }
            if constexpr (MODE == DZ) {
              v = to_f32(e.other[q * e.ld + p]) * act_slope<ACT>(v);
              cs[i][r] += v;
            }
          }
          if constexpr (MODE == PARTIAL) e.rows[((int64_t)blockIdx.y * Q.rows + q) * P.rows + p] = v;
          else e.out[q * e.ld_out + p] = from_f32<T>(v);
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

// The epilogue for a product whose sum was split: part [splits][Q][P] added up in a fixed order.  Block = 64 consecutive
// p x LANES, rows_per_block q rows one after another: few splits: a lane to a q row; many (LANES = 16): the lanes share
// the splits of one q row.  DZ leaves rows[block of JOIN_Q q][p].
// A million outputs from 8 parts (34 MB) 9 us, a quarter of that from 32 parts (34 MB) 15 us; with the border at 32 the
// second gained 2 us and sums of few outputs lost (16x2048 -> 2048 float32, dz and db, 22 -> 31 us).
constexpr int JOIN_Q = 16, JOIN_FEW = 8;
template <typename T, int MODE, bool FEW>
__global__ __launch_bounds__(FEW ? 256 : 1024) void lin_join_kernel(const float* __restrict__ part, int splits, int P, int Q,
                                                                    int rows_per_block, Epilogue<T> e) {
  constexpr int LANES = FEW ? 4 : 16;
  __shared__ float red[LANES][64];
  const int p_blocks = (e.cols + 63) / 64, q_block = blockIdx.x / p_blocks, c = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int p = (blockIdx.x - q_block * p_blocks) * 64 + c;
  const int64_t n = (int64_t)P * Q;
  const int qa = q_block * rows_per_block, qb = min(qa + rows_per_block, Q);
  const bool in = p < P;
  const float bias = (MODE == FWD || MODE == DZ) && e.bias && in ? e.bias[p] : 0.f;
  float cs = 0.f;
  with_act(MODE == FWD || MODE == DZ ? e.act : MIS_ACT_NONE, [&](auto act) {
    constexpr int ACT = decltype(act)::value;
    auto finish = [&](int q, float v) {
      if constexpr (MODE == FWD) {
        v = act_value<ACT>(v + bias);
        if (e.other) v += to_f32(e.other[q * e.ld + p]);
      }
      if constexpr (MODE == DZ) {
        v = to_f32(e.other[q * e.ld + p]) * act_slope<ACT>(v + bias);
        cs += v;
      }
      e.out[q * e.ld_out + p] = from_f32<T>(v);
    };
    if (!in && p < e.cols)
      for (int q = qa + w; q < qb; q += LANES) e.out[q * e.ld_out + p] = (T)0.f;
    if constexpr (FEW) {
      if (in)
        for (int q = qa + w; q < qb; q += LANES) {
          float v = 0.f;
#pragma unroll
          for (int k = 0; k < JOIN_FEW; k++)
            if (k < splits) v += part[k * n + (int64_t)q * P + p];
          finish(q, v);
        }
    } else {
      for (int q = qa; q < qb; q++) {
        float v = 0.f;
        if (in) {
#pragma unroll 8
          for (int k = w; k < splits; k += LANES) v += part[k * n + (int64_t)q * P + p];
        }
        red[w][c] = v;
        __syncthreads();
        if (w == 0 && in) {
#pragma unroll
          for (int k = 1; k < LANES; k++) v += red[k][c];
          finish(q, v);
        }
        __syncthreads();
      }
    }
  });
  if constexpr (MODE == DZ) {
    red[w][c] = cs;
    __syncthreads();
    if (w == 0 && in) {
#pragma unroll
      for (int k = 1; k < LANES; k++) cs += red[k][c];
      e.rows[(int64_t)q_block * P + p] = cs;
    }
  }
}

// dst [rows][ld_dst] = src [rows][cols] with zeros behind each row, 16 bytes a thread: operands whose rows are not whole
// 16-byte chunks long are brought into that form once a call.
template <typename T>
__global__ __launch_bounds__(256) void lin_pad_kernel(const T* __restrict__ src, int64_t ld, int64_t rows, int cols, int ld_dst,
                                                      T* __restrict__ dst) {
  constexpr int V = 16 / sizeof(T);
  const int per_row = ld_dst / V;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < rows * per_row; i += (int64_t)gridDim.x * 256) {
    const int64_t r = i / per_row;
    const int c = (int)(i - r * per_row) * V;
    union { u32x4 u; T t[V]; } x;
#pragma unroll
    for (int k = 0; k < V; k++) x.t[k] = c + k < cols ? src[r * ld + c + k] : (T)0.f;
    *(u32x4*)(dst + r * ld_dst + c) = x.u;
  }
}

// rows[chunk][N] = sums of a chunk's rows of d (row stride ld); a thread has V neighbouring columns, up to 64 threads side
// by side, the others take rows in turn.  Chunks of 256 rows, shorter down to 32 while there are fewer than 1024 blocks.
int sum_rows(int64_t M, int64_t N) {
  int rows = 256;
  while (rows > 32 && (int64_t)cdiv(M, rows) * cdiv(N, 512) < 1024) rows /= 2;
  return rows;
}
template <typename T, int V>
__global__ __launch_bounds__(256) void lin_colsum_kernel(const T* __restrict__ d, int64_t ld, int64_t M, int N, int side,
                                                         int chunk, float* __restrict__ rows) {
  __shared__ float red[256 * V];
  const int cx = threadIdx.x % side, w = threadIdx.x / side, lanes = 256 / side;
  const int c = (blockIdx.y * side + cx) * V;
  const int64_t m1 = min((int64_t)(blockIdx.x + 1) * chunk, M);
  float s[V];
#pragma unroll
  for (int k = 0; k < V; k++) s[k] = 0.f;
  if (c < N && w < lanes) {
#pragma unroll 8
    for (int64_t m = (int64_t)blockIdx.x * chunk + w; m < m1; m += lanes) {
      if constexpr (V == 1) {
        s[0] += to_f32(d[m * ld + c]);
      } else {
        Pack<T> x;
        x.load(d + m * ld + c);
#pragma unroll
        for (int k = 0; k < V; k++) s[k] += x.v[k];
      }
    }
  }
#pragma unroll
  for (int k = 0; k < V; k++) red[k * 256 + threadIdx.x] = s[k];
  __syncthreads();
  for (int i = threadIdx.x; i < side * V; i += 256) {
    const int x = i / V, k = i - x * V, col = (blockIdx.y * side + x) * V + k;
    float t = 0.f;
    for (int l = 0; l < lanes; l++) t += red[k * 256 + l * side + x];
    if (col < N) rows[(int64_t)blockIdx.x * N + col] = t;
  }
}

template <typename T>
void launch_colsum(const T* d, int64_t ld, int64_t M, int64_t N, float* rows, float* out, hipStream_t st) {
  constexpr int V = 16 / sizeof(T);
  const bool wide = ((uintptr_t)d & 15) == 0 && ld % V == 0 && N % V == 0;
  const int per = wide ? V : 1, side = (int)(N / per < 64 ? (N + per - 1) / per : 64);
  const int chunk = sum_rows(M, N);
  const dim3 grid(cdiv(M, chunk), cdiv(N, (int64_t)side * per));
  if (wide) lin_colsum_kernel<T, V><<<grid, 256, 0, st>>>(d, ld, M, (int)N, side, chunk, rows);
  else lin_colsum_kernel<T, 1><<<grid, 256, 0, st>>>(d, ld, M, (int)N, side, chunk, rows);
  launch_reduce_partials(rows, cdiv(M, chunk), (int)N, out, st);
}

// ---------------------------------------------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------------------------------------------
enum Tile { ANY64, T64, T128, T256 };
int tile_edge(Tile t) { return t == T256 ? 256 : t == T128 ? 128 : 64; }

// How a product is cut up: the edge of the output tiles, and parts of the sum (joined by a second launch).
struct Cut {
  Tile tile;
  int splits;
  int64_t per;          // r per split, a multiple of a stage
  double us;            // the model's time
  int row_tiles() const { return splits > 1 ? JOIN_Q : tile_edge(tile); }      // q rows behind a row of partial sums
};

// The cheapest by a model of the time in microseconds: rounds of workgroups over the chip's 256 CUs; a round = start,
// epilogue and its stages, a stage at the matrix rate of the tile (shared by the workgroups of a CU) or, for a lone
// workgroup, at the time a load takes; for a split sum the second launch, and the parts written and read.  The constants
// are fitted to 160 products of 1 to 10^6 rows and 24 to 4096 columns, forward and the three backward ones, bf16 and
// float32, each measured in all cuts: the choice is 2 % slower than the best cut on average, 29 % at worst (14 us for 11).
// It ranks cuts; as a time it is short where the epilogue is dear, for which it has no term (16384x512 -> 2048: 31 us, measured 45
// bare and 62 with GELU; 4551x104 -> 252 float32: 3.6 and 11.7).
// ANY64's are from nine odd products (a stage of 2.2 to 6.4 us alone and 2 to 3.5 shared, in either type): 1000 x 2001 -> 1001
// in bf16 takes 132 us there and 27 as padded copies, 25 x 1087 -> 15 in float32 75 and 15; 4 x 25 -> 678 stays at 6.
Cut pick_cut(int esize, bool staged, int64_t p, int64_t q, int64_t r) {
  struct Rate { double full, alone, per_output; int at_a_time; };
  static const Rate rates[] = {{2.5, 4.0, 3e-5, 3}, {0.057, 0.45, 3e-5, 3}, {0.41, 0.745, 3e-5, 2}, {1.06, 0.2, 7e-5, 1}};   // by Tile
  const int K = ROW_BYTES / esize;
  const int64_t stages = (r + K - 1) / K;
  Cut best{ANY64, 1, stages * K, 1e300};
  for (int t = staged ? T64 : ANY64; t <= (staged ? T256 : ANY64); t++) {
    const int edge = tile_edge((Tile)t), slots = 256 * rates[t].at_a_time;
    const int64_t tiles = (int64_t)cdiv(p, edge) * cdiv(q, edge);
    auto round_us = [&](int64_t wgs, int64_t per) {
      const double share = wgs > 256 ? wgs / 256.0 : 1.0, full = rates[t].full * (esize == 4 && t != ANY64 ? 1.84 : 1.0) * share;
      return 2.6 + rates[t].per_output * edge * edge * share + per * (full > rates[t].alone ? full : rates[t].alone);
    };
    for (int s = 1; s <= 1024; s *= 2) {
      const int64_t per = (stages + s - 1) / s;
      const int splits = (int)((stages + per - 1) / per);
      if (s > 1 && (splits == 1 || per < 2 || tiles * splits > 4096)) break;
      const int64_t wgs = tiles * splits, rounds = (wgs + slots - 1) / slots;
      double us = (rounds - 1) * round_us(slots, per) + round_us(wgs - (rounds - 1) * slots, per);
      if (splits > 1) us += 2.6 + 3.1e-6 * splits * p * q;
      if (us < best.us) best = Cut{(Tile)t, splits, per * K, us};
    }
  }
  return best;
}

// Whether a tensor [..][cols] with this row stride is whole 16-byte chunks, as the staged kernels read it.
template <typename T> bool chunked(const T* p, int64_t cols, int64_t ld) {
  constexpr int V = 16 / sizeof(T);
  return ((uintptr_t)p & 15) == 0 && cols % V == 0 && ld % V == 0 && ld * (int64_t)sizeof(T) * 256 < 0x7FFFFF00;
}

template <typename T> bool wide_epilogue(const Operand<T>& P, const Epilogue<T>& e, int mode) {
  constexpr int V = 16 / sizeof(T);
  if (mode == PARTIAL) return P.rows % 4 == 0;
  return e.cols == P.rows && P.rows % V == 0 && e.ld_out % V == 0 && (((uintptr_t)e.other | (uintptr_t)e.out) & 15) == 0 &&
         (!e.other || e.ld % V == 0);
}

template <typename T, int TP, int TQ, int WP, int WQ, int STAGES, bool PTR, bool QTR, int MODE, bool WIDE>
int launch_tile(const Operand<T>& P, const Operand<T>& Q, int64_t R, const Cut& cut, const Epilogue<T>& e, hipStream_t st) {
  constexpr int LDS = STAGES * (TP + TQ) * ROW_BYTES;
  if constexpr (LDS > 65536) {
    static thread_local bool raised[64] = {};
    int dev = 0;
    if (hipGetDevice(&dev) != hipSuccess || dev >= 64) return 1;
    if (!raised[dev]) {
      if (hipFuncSetAttribute((const void*)lin_tile_kernel<T, TP, TQ, WP, WQ, STAGES, PTR, QTR, MODE, WIDE>,
                              hipFuncAttributeMaxDynamicSharedMemorySize, LDS) != hipSuccess)
        return 1;
      raised[dev] = true;
    }
  }
  const Grid g{cdiv(P.rows, TP), cdiv(Q.rows, TQ), cut.splits, cut.per};
  lin_tile_kernel<T, TP, TQ, WP, WQ, STAGES, PTR, QTR, MODE, WIDE><<<g.launch(), 64 * WP * WQ, LDS, st>>>(P, Q, R, g, e);
  return 0;
}

template <typename T, bool PTR, bool QTR, int MODE, bool WIDE>
int launch_staged(const Operand<T>& P, const Operand<T>& Q, int64_t R, const Cut& cut, const Epilogue<T>& e, hipStream_t st) {
  if (cut.tile == T256) return launch_tile<T, 256, 256, 2, 4, 2, PTR, QTR, MODE, WIDE>(P, Q, R, cut, e, st);
  if (cut.tile == T128) return launch_tile<T, 128, 128, 2, 2, 2, PTR, QTR, MODE, WIDE>(P, Q, R, cut, e, st);
  return launch_tile<T, 64, 64, 2, 2, 4, PTR, QTR, MODE, WIDE>(P, Q, R, cut, e, st);
}

template <typename T, bool PTR, bool QTR, int MODE>
int launch_cut(const Operand<T>& P, const Operand<T>& Q, int64_t R, const Cut& cut, const Epilogue<T>& e, hipStream_t st) {
  switch (cut.tile) {
    case T256: case T128: case T64:
      return wide_epilogue(P, e, MODE) ? launch_staged<T, PTR, QTR, MODE, true>(P, Q, R, cut, e, st)
                                       : launch_staged<T, PTR, QTR, MODE, false>(P, Q, R, cut, e, st);
    default:
      lin_any_kernel<T, MODE><<<dim3(cdiv(P.rows, ANY_T) * cdiv(Q.rows, ANY_T), cut.splits), 256, 0, st>>>(P, Q, R, cut.per, e);
      return 0;
  }
}

// out = epilogue(P Q^T); `e.rows` takes DZ's partial sums, `part` the parts of a split sum.
template <typename T, bool PTR, bool QTR, int MODE>
int product(const Operand<T>& P, const Operand<T>& Q, int64_t R, const Cut& cut, Epilogue<T> e, float* part, hipStream_t st) {
  if (cut.splits == 1) return launch_cut<T, PTR, QTR, MODE>(P, Q, R, cut, e, st);
  const Epilogue<T> partial{nullptr, nullptr, 0, nullptr, 0, 0, part, MIS_ACT_NONE};
  if (launch_cut<T, PTR, QTR, PARTIAL>(P, Q, R, cut, partial, st)) return 1;
  const int rpb = MODE == DZ ? JOIN_Q : cut.splits <= JOIN_FEW ? 4 : 1, grid = cdiv(e.cols, 64) * cdiv(Q.rows, rpb);
  if (cut.splits <= JOIN_FEW) lin_join_kernel<T, MODE, true><<<grid, 256, 0, st>>>(part, cut.splits, P.rows, Q.rows, rpb, e);
  else lin_join_kernel<T, MODE, false><<<grid, 1024, 0, st>>>(part, cut.splits, P.rows, Q.rows, rpb, e);
  return 0;
}

// Scratch of one call, handed out in order; with base 0 the same calls add up its size.
struct Scratch {
  uintptr_t base;
  size_t used;
  template <typename T> T* take(size_t n) {
    T* p = (T*)(base + used);
    used += align256(n * sizeof(T));
    return p;
  }
};

template <typename T> int64_t padded(int64_t n) {
  constexpr int V = 16 / sizeof(T);
  return (n + V - 1) / V * V;
}

// Parts of a split sum, whichever kernel takes it (that depends on addresses the size query does not know).
size_t part_floats(int esize, int64_t p, int64_t q, int64_t r) {
  size_t most = 0;
  for (int staged = 0; staged < 2; staged++) {
    const Cut c = pick_cut(esize, staged, p, q, r);
    if (c.splits > 1 && (size_t)c.splits * p * q > most) most = (size_t)c.splits * p * q;
  }
  return most;
}

// A copy with padded rows costs a launch and its bytes.
double pad_us(int64_t rows, int64_t cols, int esize) { return 3.0 + 5e-7 * rows * cols * esize; }

template <typename T>
const T* pad(const T* src, int64_t rows, int64_t cols, int64_t ld, T* dst, hipStream_t st) {
  const int64_t ld_dst = padded<T>(cols);
  lin_pad_kernel<T><<<ew_grid(rows * ld_dst / (16 / (int)sizeof(T)), 256), 256, 0, st>>>(src, ld, rows, (int)cols, (int)ld_dst, dst);
  return dst;
}

// The buffers of a call, in the order the code below uses them.  Rows that are not whole 16-byte chunks long get a padded copy
// where that pays; sizes are for the case that it does.
template <typename T> struct Buffers {
  T *x, *w, *z;
  float *rows, *part;
  Buffers(Scratch& s, int64_t M, int64_t N, int64_t K, int act, bool backward) {
    const int64_t Kp = padded<T>(K), Np = padded<T>(N);
    x = s.take<T>(Kp != K ? M * Kp : 0);
    w = s.take<T>(Kp != K ? N * Kp : 0);
    z = s.take<T>(!backward ? 0 : act != MIS_ACT_NONE || Np != N ? M * Np : 0);       // dz, or a padded dy
    size_t most = part_floats(sizeof(T), N, M, K), few_rows = most ? JOIN_Q : 64;
    rows = s.take<float>(!backward ? 0 : act == MIS_ACT_NONE ? (size_t)cdiv(M, sum_rows(M, N)) * N : (M + few_rows - 1) / few_rows * N);
    if (backward)
      for (size_t n : {part_floats(sizeof(T), K, M, N), part_floats(sizeof(T), K, N, M)})
        if (n > most) most = n;
    part = s.take<float>(most);
  }
};

bool sizes_ok(int dtype, int64_t M, int64_t N, int64_t K) {
  return (dtype == MIS_F32 || dtype == MIS_BF16) && M >= 1 && N >= 1 && K >= 1 && N <= 1 << 20 && K <= 1 << 20 &&
         M < ((int64_t)1 << 30) &&
         (M + 63) / 64 * (((N > K ? N : K) + 63) / 64) <= (1 << 24) - 8;      // tiles of 256 threads: a launch holds below 2^32
}

bool aligned(int dtype, std::initializer_list<const void*> ps) {
  uintptr_t m = 0;
  for (const void* p : ps) m |= (uintptr_t)p;
  return (m & (dtype == MIS_BF16 ? 1 : 3)) == 0;
}

template <typename T>
int forward(const T* x, int64_t ldx, const T* w, const float* bias, const T* r, int64_t ldr, int64_t M, int64_t N, int64_t K,
            int act, T* y, void* ws, hipStream_t st) {
  Scratch scratch{(uintptr_t)ws, 0};
  const Buffers<T> buf(scratch, M, N, K, act, false);
  const Cut any = pick_cut(sizeof(T), false, N, M, K), fast = pick_cut(sizeof(T), true, N, M, K);
  int64_t ldw = K;
  bool staged = chunked(x, K, ldx) && chunked(w, K, ldw);
  if (padded<T>(K) != K && fast.us + pad_us(M, K, sizeof(T)) + pad_us(N, K, sizeof(T)) < any.us) {
    x = pad(x, M, K, ldx, buf.x, st);
    w = pad(w, N, K, ldw, buf.w, st);
    ldx = ldw = padded<T>(K);
    staged = true;
  }
  const Epilogue<T> e{bias, r, ldr, y, N, (int)N, nullptr, act};
  return product<T, false, false, FWD>({w, ldw, 1, (int)N}, {x, ldx, 1, (int)M}, K, staged ? fast : any, e, buf.part, st);
}

template <typename T>
int backward(const T* x, int64_t ldx, const T* w, const float* bias, const T* dy, int64_t ldd, int64_t M, int64_t N, int64_t K,
             int act, T* dx, T* dw, float* db, void* ws, hipStream_t st) {
  Scratch scratch{(uintptr_t)ws, 0};
  const Buffers<T> buf(scratch, M, N, K, act, true);
  const bool again = act != MIS_ACT_NONE;
  const int64_t Kp = padded<T>(K), Np = padded<T>(N);
  Cut dz_cut[2], dx_cut[2], dw_cut[2];                   // [staged]
  double us[2] = {0.0, 0.0};
  for (int i = 0; i < 2; i++) {
    dz_cut[i] = pick_cut(sizeof(T), i, N, M, K);
    dx_cut[i] = pick_cut(sizeof(T), i, K, M, N);
    dw_cut[i] = pick_cut(sizeof(T), i, K, N, M);
    us[i] = (again ? dz_cut[i].us : 0.0) + (dx ? dx_cut[i].us : 0.0) + (dw ? dw_cut[i].us : 0.0);
  }
  const bool pad_k = Kp != K, pad_dy = Np != N && !again;
  const bool use_x = again || dw, use_w = again || dx;
  int64_t ldw = K;
  bool staged = (pad_k || ((!use_x || chunked(x, K, ldx)) && (!use_w || chunked(w, K, ldw)))) &&
                (again || pad_dy || chunked(dy, N, ldd));
  if (staged && (pad_k || pad_dy)) {
    double extra = 0.0;
    if (pad_k) extra += (use_x ? pad_us(M, K, sizeof(T)) : 0.0) + (use_w ? pad_us(N, K, sizeof(T)) : 0.0);
    if (pad_dy) extra += pad_us(M, N, sizeof(T));
    staged = us[1] + extra < us[0];
    if (staged && pad_k) {
      if (use_x) x = pad(x, M, K, ldx, buf.x, st);
      if (use_w) w = pad(w, N, K, ldw, buf.w, st);
      ldx = ldw = Kp;
    }
  }
  const T* z = dy;
  int64_t ldz = ldd;
  if (again) {
    const Epilogue<T> e{bias, dy, ldd, buf.z, Np, (int)Np, buf.rows, act};
    const Cut& cut = dz_cut[staged];
    if (product<T, false, false, DZ>({w, ldw, 1, (int)N}, {x, ldx, 1, (int)M}, K, cut, e, buf.part, st)) return 1;
    z = buf.z;
    ldz = Np;
    if (db) launch_reduce_partials(buf.rows, cdiv(M, cut.row_tiles()), (int)N, db, st);
  } else if (db) {
    launch_colsum(dy, ldd, M, N, buf.rows, db, st);
  }
  if (staged && pad_dy && (dx || dw)) {
    z = pad(dy, M, N, ldd, buf.z, st);
    ldz = Np;
  }
  if (dx) {
    const Epilogue<T> e{nullptr, nullptr, 0, dx, K, (int)K, nullptr, MIS_ACT_NONE};
    if (product<T, true, false, STORE>({w, 1, ldw, (int)K}, {z, ldz, 1, (int)M}, N, dx_cut[staged], e, buf.part, st)) return 1;
  }
  if (dw) {
    const Epilogue<T> e{nullptr, nullptr, 0, dw, K, (int)K, nullptr, MIS_ACT_NONE};
    if (product<T, true, true, STORE>({x, 1, ldx, (int)K}, {z, 1, ldz, (int)N}, M, dw_cut[staged], e, buf.part, st)) return 1;
  }
  return 0;
}

template <typename T> size_t bytes_of(int64_t M, int64_t N, int64_t K, int act, bool backward) {
  Scratch s{0, 0};
  Buffers<T>(s, M, N, K, act, backward);
  return s.used ? s.used : 256;
}

}  // namespace

extern "C" {

size_t mis_linear_act_fwd_workspace_bytes(int dtype, int64_t M, int64_t N, int64_t K) {
  if (!sizes_ok(dtype, M, N, K)) return 0;
  return dtype == MIS_BF16 ? bytes_of<bf16>(M, N, K, MIS_ACT_NONE, false) : bytes_of<float>(M, N, K, MIS_ACT_NONE, false);
}

int mis_linear_act_fwd(const void* x, int64_t ldx, const void* w, const float* bias, const void* residual, int64_t ldr, int dtype,
                       int64_t M, int64_t N, int64_t K, int act, void* y, void* workspace, mis_stream_t stream) {
  MIS_REQUIRE(sizes_ok(dtype, M, N, K), "linear_act_fwd: bad dtype or sizes (M=%lld N=%lld K=%lld)", (long long)M, (long long)N,
              (long long)K);
  MIS_REQUIRE(x && w && y && workspace, "linear_act_fwd: null pointer");
  MIS_REQUIRE(ldx >= K && (!residual || ldr >= N), "linear_act_fwd: row stride below the row length");
  MIS_REQUIRE(act >= MIS_ACT_NONE && act <= MIS_ACT_GELU, "linear_act_fwd: unknown activation %d", act);
  MIS_REQUIRE(aligned(dtype, {x, w, residual, y}) && ((uintptr_t)workspace & 15) == 0, "linear_act_fwd: misaligned pointer");
  hipStream_t st = (hipStream_t)stream;
  int rc;
  if (dtype == MIS_BF16)
    rc = forward((const bf16*)x, ldx, (const bf16*)w, bias, (const bf16*)residual, ldr, M, N, K, act, (bf16*)y,
                 workspace, st);
  else
    rc = forward((const float*)x, ldx, (const float*)w, bias, (const float*)residual, ldr, M, N, K, act, (float*)y,
                 workspace, st);
  MIS_REQUIRE(rc == 0, "linear_act_fwd: the device refuses the kernel's shared memory");
  MIS_CHECK_LAUNCH("linear_act_fwd");
  return MIS_OK;
}

size_t mis_linear_act_bwd_workspace_bytes(int dtype, int64_t M, int64_t N, int64_t K, int act) {
  if (!sizes_ok(dtype, M, N, K)) return 0;
  return dtype == MIS_BF16 ? bytes_of<bf16>(M, N, K, act, true) : bytes_of<float>(M, N, K, act, true);
}

int mis_linear_act_bwd(const void* x, int64_t ldx, const void* w, const float* bias, const void* dy, int64_t ldd, int dtype,
                       int64_t M, int64_t N, int64_t K, int act, void* dx, void* dw, float* db, void* workspace,
                       mis_stream_t stream) {
  MIS_REQUIRE(sizes_ok(dtype, M, N, K), "linear_act_bwd: bad dtype or sizes (M=%lld N=%lld K=%lld)", (long long)M, (long long)N,
              (long long)K);
  MIS_REQUIRE(x && w && dy && workspace, "linear_act_bwd: null pointer");
  MIS_REQUIRE(ldx >= K && ldd >= N, "linear_act_bwd: row stride below the row length");
  MIS_REQUIRE(act >= MIS_ACT_NONE && act <= MIS_ACT_GELU, "linear_act_bwd: unknown activation %d", act);
  MIS_REQUIRE(aligned(dtype, {x, w, dy, dx, dw}) && ((uintptr_t)workspace & 15) == 0, "linear_act_bwd: misaligned pointer");
  hipStream_t st = (hipStream_t)stream;
  int rc;
  if (dtype == MIS_BF16)
    rc = backward((const bf16*)x, ldx, (const bf16*)w, bias, (const bf16*)dy, ldd, M, N, K, act, (bf16*)dx, (bf16*)dw, db,
             workspace, st);
  else
    rc = backward((const float*)x, ldx, (const float*)w, bias, (const float*)dy, ldd, M, N, K, act, (float*)dx, (float*)dw, db,
             workspace, st);
  MIS_REQUIRE(rc == 0, "linear_act_bwd: the device refuses the kernel's shared memory");
  MIS_CHECK_LAUNCH("linear_act_bwd");
  return MIS_OK;
}

}  // extern "C"
