// Device helpers of the transformer-block operators: element types,
// activations with their derivatives, and the launchers shared between the
// operators' files.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "block.h"
#include "common.cuh"

namespace pet {
namespace blk {

inline bool aligned16(const void *p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }
// Rows of p can be read or written in 16-byte pieces.
inline bool rows16(const void *p, int64_t ld, int dt) {
  return aligned16(p) && (ld * static_cast<int64_t>(dtype_size(dt))) % 16 == 0;
}
// SMs of the current device.
int sm_count();
// Device error words count the waits given up and are never cleared, so that
// none is lost beside a check: whether there are new ones, after the work on s,
// since the last time this was asked of `word` on the current device.
bool new_errors(const int &word, cudaStream_t s);
// A wait given up: into the caller's error word, which is 1 then, or the file's.
__device__ __forceinline__ void raise_error(int *callers, int &files) {
  if (callers) atomicExch(callers, 1);
  else atomicAdd(&files, 1);
}
// of the norms' rings (block_norm.cu)
bool norm_error(cudaStream_t s);
void norm_wait_bound(uint64_t ns);

__device__ __forceinline__ float to_f(float x) { return x; }
__device__ __forceinline__ float to_f(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_f(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T>
__device__ __forceinline__ T from_f(float x);
template <>
__device__ __forceinline__ float from_f<float>(float x) { return x; }
template <>
__device__ __forceinline__ __half from_f<__half>(float x) { return __float2half_rn(x); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

// 16 bytes of T <-> floats
template <typename T>
struct Vec {
  static constexpr int n = 16 / sizeof(T);
};
template <typename T>
__device__ __forceinline__ void unpack(const uint4 &u, float (&v)[16 / sizeof(T)]) {
  const T *t = reinterpret_cast<const T *>(&u);
#pragma unroll
  for (int j = 0; j < Vec<T>::n; ++j) v[j] = to_f(t[j]);
}
template <typename T>
__device__ __forceinline__ uint4 pack(const float (&v)[16 / sizeof(T)]) {
  uint4 u;
  T *t = reinterpret_cast<T *>(&u);
#pragma unroll
  for (int j = 0; j < Vec<T>::n; ++j) t[j] = from_f<T>(v[j]);
  return u;
}

// 1 / (1 + e^-z) by the intrinsics: a few ulp of fp32, and 2^-23 |z| of
// e^-z, which no result sees where |z| is large.  Below z = -87 e^-z passes 2^126
// or is infinite and the quotient 0, so nothing is clamped (a clamp by fmaxf
// would turn NaN into a number).
__device__ __forceinline__ float logistic(float z) { return __fdividef(1.f, 1.f + __expf(-z)); }

// a = act(z), da = act'(z)
template <int ACT>
__device__ __forceinline__ void act_pair(float z, float &a, float &da) {
  if (ACT == ACT_SIGMOID) {
    a = logistic(z);
    da = a * (1.f - a);
  } else if (ACT == ACT_SILU) {
    const float p = logistic(z);
    a = z * p;
    da = p * (1.f + z * (1.f - p));
  } else if (ACT == ACT_GELU) {
    const float c = normcdff(z);
    a = z * c;
    da = c + z * __expf(-0.5f * z * z) * 0.3989422804014327f;
  } else if (ACT == ACT_GELU_TANH) {
    const float p = logistic(1.5957691216057308f * (z + 0.044715f * z * z * z)), q = z * p * (1.f - p);
    a = z * p;
    // (q is 0 from about |z| = 10 on; z^2 passes fp32's range later)
    da = q == 0.f ? p : p + q * 1.5957691216057308f * (1.f + 0.134145f * z * z);
  } else if (ACT == ACT_RELU) {
    a = z > 0.f ? z : (z == z ? 0.f : z);
    da = z > 0.f ? 1.f : 0.f;
  } else {
    a = z;
    da = 1.f;
  }
}
template <int V>
struct Const {
  static constexpr int value = V;
};
// f(Const<act>{}) for the run-time activation (one uniform branch)
template <typename F>
__device__ __forceinline__ void with_act(int act, F &&f) {
  switch (act) {
    case ACT_SIGMOID: f(Const<ACT_SIGMOID>{}); break;
    case ACT_SILU: f(Const<ACT_SILU>{}); break;
    case ACT_GELU: f(Const<ACT_GELU>{}); break;
    case ACT_GELU_TANH: f(Const<ACT_GELU_TANH>{}); break;
    case ACT_RELU: f(Const<ACT_RELU>{}); break;
    default: f(Const<ACT_IDENTITY>{}); break;
  }
}
// Element j of a vector of run-time type.
__device__ __forceinline__ float load_dt(const void *p, int dt, int64_t j) {
  if (dt == DT_F32) return static_cast<const float *>(p)[j];
  if (dt == DT_F16) return __half2float(static_cast<const __half *>(p)[j]);
  return __bfloat162float(static_cast<const __nv_bfloat16 *>(p)[j]);
}
__device__ __forceinline__ void store_dt(void *p, int dt, int64_t j, float v) {
  if (dt == DT_F32) static_cast<float *>(p)[j] = v;
  else if (dt == DT_F16) static_cast<__half *>(p)[j] = __float2half_rn(v);
  else static_cast<__nv_bfloat16 *>(p)[j] = __float2bfloat16_rn(v);
}

// ReLU's derivative jumps at 0, where fp32 sums of different orders disagree
// about the sign of z, or cancel to 0 with a remainder below their last bit.
// Elements within kNear of the largest beside them (5 or more of those sums'
// largest errors) get z from a dot product in 64 bits, all lanes of the warp on
// one element at a time: about one in 100,000.  What bounds that work: more than
// kNearMost of a 32 x 32 block (kNearRow of a warp's 32 elements) that are near 0
// are rows or features of a smaller scale than the others', whose own sums are as
// exact; a block's row of zeros is a row of zeros in x (padding), a column of them
// costs one product if its weights are zeros, and more than kZeroMost others are
// such rows and columns in number.  All of these are left as they are.  Measured
// for dz, dWg, dWv, dx of 8192 x 1024 x 4096 in bf16: 340 us, with the smooth silu
// 324; one column of zero weights in each 32: 510.
constexpr float kNear = 1.f / 262144.f;
constexpr unsigned kNearMost = 32, kZeroMost = 64;
constexpr int kNearRow = 2;
// z = x w^T + b of the elements in doubt
struct NearZero {
  const void *x, *w, *b;
  int64_t ldx, ldw, k;
};
// dead: the columns c0 + bit that have turned out to have no weights.
template <typename T>
__device__ __forceinline__ float settled(const NearZero &e, bool flag, int64_t row, int64_t col, float z, int lane,
                                         unsigned &dead, int64_t c0) {
  unsigned todo = __ballot_sync(0xffffffffu, flag && !(dead >> (col - c0) & 1));
  while (todo) {
    const int src = __ffs(todo) - 1;
    todo &= todo - 1;
    const int64_t r = __shfl_sync(0xffffffffu, row, src), c = __shfl_sync(0xffffffffu, col, src);
    const T *x = static_cast<const T *>(e.x) + r * e.ldx, *w = static_cast<const T *>(e.w) + c * e.ldw;
    double t = 0.0;
    bool live = false;
    int64_t k = lane;
    for (; k + 7 * 32 < e.k; k += 8 * 32) {  // 16 loads in flight: latency is all it costs
      T a[8], b[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) a[i] = x[k + i * 32], b[i] = w[k + i * 32];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        t = fma(static_cast<double>(to_f(a[i])), static_cast<double>(to_f(b[i])), t);
        live |= to_f(b[i]) != 0.f;
      }
    }
    for (; k < e.k; k += 32) {
      t = fma(static_cast<double>(to_f(x[k])), static_cast<double>(to_f(w[k])), t);
      live |= to_f(w[k]) != 0.f;
    }
    if (!__any_sync(0xffffffffu, live)) {
      dead |= 1u << (c - c0);
      todo &= ~__ballot_sync(0xffffffffu, col == c);
    }
    t = warp_sum_d(t);
    if (e.b) t += static_cast<double>(to_f(static_cast<const T *>(e.b)[c]));
    if (lane == src) z = t > 0.0 ? fmaxf(static_cast<float>(t), 1e-37f) : fminf(static_cast<float>(t), 0.f);
  }
  return z;
}
// The same for one element a lane (there: it has one), of columns from lane 0's on.
template <typename T>
__device__ __forceinline__ float settled_row(const NearZero &e, bool there, float near, int64_t row, int64_t col,
                                             float z, int lane, int most = kNearRow) {
  const bool flag = there && fabsf(z) <= near, nonzero = flag && z != 0.f;
  const bool all = __popc(__ballot_sync(0xffffffffu, flag)) <= most;
  if (!all && __popc(__ballot_sync(0xffffffffu, nonzero)) > most) return z;
  unsigned dead = 0;
  return settled<T>(e, all ? flag : nonzero, row, col, z, lane, dead, __shfl_sync(0xffffffffu, col, 0));
}

// ---- few rows (block_rows.cu) ---------------------------------------------
// At most kFewRows rows (forward of 16-bit aligned ones: 16): each weight read
// once with plain loads, every sum and gradient in fp32.
constexpr int kFewRows = 8;
struct FewRows {
  int dt, act, M;
  int64_t K, N;
  const void *x, *w0, *w1;  // w1 null: linear
  int64_t ldx, ldw0, ldw1;
  const void *b0, *b1;
  float scale;
  const void *in;           // residual (linear forward) or upstream gradient (backward)
  int64_t ldin;
  void *out;                // forward: the result; null in a backward
  int64_t ldo;
  // backward: gradients out unless null; dz: few_rows_floats() floats
  void *dx, *dw0, *dw1, *db0, *db1;
  int64_t lddx, lddw0, lddw1;
  float *dz;
};
bool few_rows_fit(const FewRows &a);  // forward
void few_rows(const FewRows &a, cudaStream_t s);
size_t few_rows_floats(const FewRows &a);
void few_rows_bwd(const FewRows &a, cudaStream_t s);

// Column sums of a 16-bit [M, N] matrix in fp32 over column_strips(M) strips of
// rows: part [strip][N].
int column_strips(int64_t M);
void column_sums(const void *p, int dt, int64_t ld, int64_t M, int64_t N, float *part, cudaStream_t s);
// out[c] = scale sum over p < P of part[p][c], in a fixed order; part is used up.
void column_join(float *part, int64_t P, int64_t N, float scale, void *out, int dt, cudaStream_t s);

}  // namespace blk
}  // namespace pet
