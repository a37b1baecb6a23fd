// Operators of a transformer block on device tensors: the gated feed-forward
// projection, the dense layer with its epilogue and the residual update
// between two norms, forward and backward.  Host entry points, shared by the
// C API (api.cpp) and the PET model (model.cu).
//
// Matrices are row-major with a leading dimension in elements.  All tensors
// of a call have one type; sums, norms and activations run in fp32.  Working
// memory comes from a Workspace: a call made with a sizing workspace (null
// base) launches nothing and only counts the bytes.
#pragma once

#include <cuda_runtime.h>

#include <cstddef>
#include <cstdint>

namespace pet {

enum DType : int { DT_F32 = 0, DT_F16 = 1, DT_BF16 = 2 };
enum Activation : int {
  ACT_IDENTITY = 0,
  ACT_SIGMOID = 1,
  ACT_SILU = 2,
  ACT_GELU = 3,       // z Phi(z)
  ACT_GELU_TANH = 4,  // z sigmoid(2 sqrt(2 / pi) (z + 0.044715 z^3))
  ACT_RELU = 5,
  ACT_COUNT = 6,
};
enum NormKind : int { NORM_NONE = 0, NORM_RMS = 1, NORM_LAYER = 2, NORM_COUNT = 3 };

inline size_t dtype_size(int dt) { return dt == DT_F32 ? 4 : 2; }

struct Workspace {
  char *base = nullptr;
  size_t cap = 0, off = 0;
  bool sizing() const { return base == nullptr; }
  // 256-byte aligned block of the caller's memory (null while sizing)
  void *take(size_t bytes);
};

struct Mat {
  const void *p = nullptr;
  int64_t ld = 0;
};
struct MutMat {
  void *p = nullptr;
  int64_t ld = 0;
};

// h = act(x Wg^T + bg) * (x Wv^T + bv): x [M, K], Wg and Wv [F, K], h [M, F].
struct GatedLinear {
  int dtype = DT_F32, act = ACT_SILU;
  int64_t M = 0, K = 0, F = 0;
  Mat x, wg, wv;
  const void *bg = nullptr, *bv = nullptr;
  MutMat h;
  // backward: dh in; each gradient out unless its pointer is null
  Mat dh;
  MutMat dx, dwg, dwv;
  void *dbg = nullptr, *dbv = nullptr;
  // f32 only, optional: the weights already in split-fp16 form (one scale
  // exponent per matrix).  products 1 multiplies the hi parts alone (the
  // model's reduced-precision mode).
  struct SplitWeight {
    const uint16_t *hi = nullptr, *lo = nullptr;
    int scale = 0;
  } wg_split, wv_split;
  int products = 3;
  int *err = nullptr;  // device error word (null: the one of block_status)
};
void gated_linear_fwd(const GatedLinear &a, Workspace &ws, cudaStream_t s);
void gated_linear_bwd(const GatedLinear &a, Workspace &ws, cudaStream_t s);

// y = residual + scale act(x W^T + b): x [M, K], W [N, K], y [M, N].
struct Linear {
  int dtype = DT_F32, act = ACT_IDENTITY;
  int64_t M = 0, K = 0, N = 0;
  Mat x, w, residual;
  const void *b = nullptr;
  float scale = 1.f;
  MutMat y;
  // backward: dy in; each gradient out unless its pointer is null
  Mat dy;
  MutMat dx, dw;
  void *db = nullptr;
};
void linear_fwd(const Linear &a, Workspace &ws, cudaStream_t s);
void linear_bwd(const Linear &a, Workspace &ws, cudaStream_t s);

// u = post(y); stream = scale residual + gate u; out = norm(stream), rows of
// d elements.  post and norm: none, RMS (x / sqrt(mean x^2 + eps)) or layer
// ((x - mean) / sqrt(var + eps)), times weight, plus bias (each optional).
// y null: stream = scale residual.  gate null: 1; gate.ld 0: one row [d].
struct ResidualNorm {
  int dtype = DT_F32, norm = NORM_RMS, post = NORM_NONE;
  int64_t M = 0;
  int d = 0;
  float scale = 1.f, eps = 1e-5f;
  Mat residual, y, gate;
  const void *w = nullptr, *b = nullptr, *pw = nullptr, *pb = nullptr;
  MutMat stream, out;  // each optional
  // backward: dstream and dout in (null: zero); gradients out unless null
  Mat dstream, dout;
  MutMat dresidual, dy, dgate;
  void *dw = nullptr, *db = nullptr, *dpw = nullptr, *dpb = nullptr;
  int *err = nullptr;  // device error word (null: the one of block_status)
};
void residual_norm_fwd(const ResidualNorm &a, Workspace &ws, cudaStream_t s);
void residual_norm_bwd(const ResidualNorm &a, Workspace &ws, cudaStream_t s);
constexpr int kMaxNormDim = 16384;

// Whether a bounded wait of the operators' pipelines on the current device has
// run out since the last call.  Synchronises `s`.
bool block_status(cudaStream_t s);
// Bound on the waits of the operators' pipelines (0: the default).
void set_block_wait_bound_ns(uint64_t ns);
// Test hook: the next norm launch with a ring withholds the copies of its first
// rows, so that their waits run out.
void inject_norm_stall();
bool norm_stall_armed();

}  // namespace pet
