// The residual update between two norms, forward and backward:
//   u = post(y),  stream = scale r + gate u,  out = norm(stream).
// A row stays in registers from its one read to its one write, so the passes
// over memory are the inputs and the outputs, and HBM is what bounds both
// directions.  Means, variances and all gradients run in fp32 (variances in
// two passes over the registers), and `out` comes from the unrounded stream.
//
// The backward recomputes both norms from r and y: it reads r, y, dstream and
// dout and writes dr and dy, with no statistics stored by the forward.
//   dn = dout w,     dstream' = dstream + norm'(dn)
//   dr = scale dstream',  dgate = dstream' u,  dp = gate dstream' pw
//   dy = post'(dp)
// where norm'(dn) = (dn - [mean dn] - n mean(dn n)) / sigma.  The gradients
// of the vectors (weights, biases, a gate of one row) are summed per CTA over
// its rows in registers, written once per CTA and added in a fixed order by a
// second kernel.
//
// A row takes 32 threads (up to 512 or 1,024 columns; eight rows per CTA) or
// a CTA.  Rows of 16-byte-aligned tensors move in 16-byte pieces, others by
// elements.
#include <algorithm>

#include "block.cuh"
#include "split16.cuh"

namespace pet {
namespace blk {

namespace {

struct NormArgs {
  int64_t M;
  int d, norm, post;
  float scale, eps;
  const void *r, *y, *gate;
  int64_t ldr, ldy, ldg;
  const void *w, *b, *pw, *pb;
  void *stream, *out;
  int64_t lds, ldo;
  Split16View split;
  const void *ds, *dout;
  int64_t ldds, lddo;
  void *dr, *dy, *dgate;       // dgate: the gate of each row
  int64_t lddr, lddy, lddg;
  float *part;                 // [CTA][vector][d] of the vectors' gradients
  int want;                    // bit v: vector v wanted (0 w, 1 b, 2 pw, 3 pb, 4 gate)
};

// Column of element j of chunk i of thread t (VEC: 16-byte chunks).
template <typename T, int TPR, bool VEC>
struct Row {
  static constexpr int V = VEC ? 16 / static_cast<int>(sizeof(T)) : 1;
  static __device__ __forceinline__ int col(int i, int t) { return (i * TPR + t) * V; }
  // zeros past d (VEC: d is a multiple of V)
  static __device__ __forceinline__ void load(const void *p, int64_t off, int c, int d, float (&v)[V]) {
    const T *q = static_cast<const T *>(p) + off + c;
    if (VEC) {
      uint4 u = make_uint4(0u, 0u, 0u, 0u);
      if (c < d) u = *reinterpret_cast<const uint4 *>(q);
      float f[16 / sizeof(T)];
      unpack<T>(u, f);
#pragma unroll
      for (int j = 0; j < V; ++j) v[j] = f[j];
    } else {
      v[0] = c < d ? to_f(*q) : 0.f;
    }
  }
  static __device__ __forceinline__ void store(void *p, int64_t off, int c, int d, const float (&v)[V]) {
    if (c >= d) return;
    T *q = static_cast<T *>(p) + off + c;
    if (VEC) {
      float f[16 / sizeof(T)];
#pragma unroll
      for (int j = 0; j < V; ++j) f[j] = v[j];
      *reinterpret_cast<uint4 *>(q) = pack<T>(f);
    } else {
      *q = from_f<T>(v[0]);
    }
  }
};

// Sums over the threads of a row.  Two slots in turn, so one barrier each:
// a slot is written again only after every thread has passed the barrier
// that follows its last read.
template <int TPR>
struct Sum {
  float2 *slots;
  int k;
  __device__ __forceinline__ float2 two(float a, float b) {
    a = warp_sum(a);
    b = warp_sum(b);
    if (TPR == 32) return make_float2(a, b);
    float2 *s = slots + (k & 1) * 32;
    k ^= 1;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (lane == 0) s[warp] = make_float2(a, b);
    __syncthreads();
    float2 v = lane < TPR / 32 ? s[lane] : make_float2(0.f, 0.f);
    return make_float2(warp_sum(v.x), warp_sum(v.y));
  }
  __device__ __forceinline__ float one(float a) {
    a = warp_sum(a);
    if (TPR == 32) return a;
    float2 *s = slots + (k & 1) * 32;
    k ^= 1;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (lane == 0) s[warp].x = a;
    __syncthreads();
    return warp_sum(lane < TPR / 32 ? s[lane].x : 0.f);
  }
};

// x -> its normalised row (columns past d stay 0); returns 1 / sigma.
template <typename R, int TPR, int NV>
__device__ __forceinline__ float normalise(int kind, float eps, int d, int t, Sum<TPR> &sum, float (&x)[NV][R::V]) {
  if (kind == NORM_LAYER) {
    float a = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < R::V; ++j) a += x[i][j];
    const float mean = sum.one(a) / static_cast<float>(d);
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < R::V; ++j)
        if (R::col(i, t) < d) x[i][j] -= mean;
  }
  float q = 0.f;
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int j = 0; j < R::V; ++j) q = fmaf(x[i][j], x[i][j], q);
  const float inv = 1.f / sqrtf(sum.one(q) / static_cast<float>(d) + eps);
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int j = 0; j < R::V; ++j) x[i][j] *= inv;
  return inv;
}

template <int TPR>
constexpr int block_threads() { return TPR == 32 ? 256 : TPR; }

template <typename T, int TPR, int E, bool VEC>
__global__ void __launch_bounds__(block_threads<TPR>()) k_norm_fwd(const NormArgs a) {
  using R = Row<T, TPR, VEC>;
  constexpr int V = R::V, NV = E / V;
  __shared__ float2 slots[64];
  const int t = TPR == 32 ? (threadIdx.x & 31) : threadIdx.x;
  const int64_t row = TPR == 32 ? static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5) : blockIdx.x;
  if (row >= a.M) return;
  Sum<TPR> sum{slots, 0};
  const int d = a.d;
  float x[NV][V];
#pragma unroll
  for (int i = 0; i < NV; ++i) R::load(a.r, row * a.ldr, R::col(i, t), d, x[i]);
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int j = 0; j < V; ++j) x[i][j] *= a.scale;
  if (a.y) {
    float u[NV][V];
#pragma unroll
    for (int i = 0; i < NV; ++i) R::load(a.y, row * a.ldy, R::col(i, t), d, u[i]);
    if (a.post != NORM_NONE) normalise<R, TPR, NV>(a.post, a.eps, d, t, sum, u);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = R::col(i, t);
      float f[V];
      if (a.pw) {
        R::load(a.pw, 0, c, d, f);
#pragma unroll
        for (int j = 0; j < V; ++j) u[i][j] *= f[j];
      }
      if (a.pb) {
        R::load(a.pb, 0, c, d, f);
#pragma unroll
        for (int j = 0; j < V; ++j) u[i][j] += f[j];
      }
      if (a.gate) {
        R::load(a.gate, row * a.ldg, c, d, f);
#pragma unroll
        for (int j = 0; j < V; ++j) u[i][j] *= f[j];
      }
#pragma unroll
      for (int j = 0; j < V; ++j) x[i][j] += u[i][j];
    }
  }
  if (a.stream) {
#pragma unroll
    for (int i = 0; i < NV; ++i) R::store(a.stream, row * a.lds, R::col(i, t), d, x[i]);
  }
  if (!a.out && !a.split.hi) return;
  if (a.norm != NORM_NONE) normalise<R, TPR, NV>(a.norm, a.eps, d, t, sum, x);
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = R::col(i, t);
    float f[V];
    if (a.w) {
      R::load(a.w, 0, c, d, f);
#pragma unroll
      for (int j = 0; j < V; ++j) x[i][j] *= f[j];
    }
    if (a.b) {
      R::load(a.b, 0, c, d, f);
#pragma unroll
      for (int j = 0; j < V; ++j) x[i][j] += f[j];
    }
    if (a.out) R::store(a.out, row * a.ldo, c, d, x[i]);
    if (sizeof(T) == 4 && VEC) {
      // a warp's 16-byte chunks are one 128-column block
      if (a.split.hi && c / 128 * 128 < d)
        warp_split_block(a.split, static_cast<int>(row), c / 128,
                         make_float4(x[i][0], x[i][V > 1 ? 1 : 0], x[i][V > 2 ? 2 : 0], x[i][V > 3 ? 3 : 0]),
                         threadIdx.x & 31);
    }
  }
}

// One row's four inputs as they lie in memory, read a row ahead.
template <typename T, int TPR, int E, bool VEC>
struct Raw {
  using R = Row<T, TPR, VEC>;
  static constexpr int V = R::V, NV = E / V;
  struct alignas(VEC ? 16 : sizeof(T)) Piece {
    T e[V];
  };
  Piece p[4][NV];
  __device__ __forceinline__ void load(const NormArgs &a, int64_t row, int t) {
    const void *src[4] = {a.r, a.y, a.ds, a.dout};
    const int64_t ld[4] = {a.ldr, a.ldy, a.ldds, a.lddo};
#pragma unroll
    for (int k = 0; k < 4; ++k)
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int c = R::col(i, t);
        if (src[k] && c < a.d)
          p[k][i] = *reinterpret_cast<const Piece *>(static_cast<const T *>(src[k]) + row * ld[k] + c);
        else
#pragma unroll
          for (int j = 0; j < V; ++j) p[k][i].e[j] = from_f<T>(0.f);
      }
  }
};

template <typename T, int TPR, int E, bool VEC>
__global__ void __launch_bounds__(block_threads<TPR>()) k_norm_bwd(const NormArgs a) {
  using R = Row<T, TPR, VEC>;
  constexpr int V = R::V, NV = E / V;
  __shared__ float2 slots[64];
  const int warp = threadIdx.x >> 5;
  const int t = TPR == 32 ? (threadIdx.x & 31) : threadIdx.x;
  const int64_t step = TPR == 32 ? static_cast<int64_t>(gridDim.x) * 8 : gridDim.x;
  const int d = a.d;
  const float rd = 1.f / static_cast<float>(d);
  Sum<TPR> sum{slots, 0};
  float acc[5][NV][V];
#pragma unroll
  for (int v = 0; v < 5; ++v)
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < V; ++j) acc[v][i][j] = 0.f;
  int64_t row = TPR == 32 ? static_cast<int64_t>(blockIdx.x) * 8 + warp : blockIdx.x;
  Raw<T, TPR, E, VEC> raw;
  if (row < a.M) raw.load(a, row, t);
  for (; row < a.M; row += step) {
    float n[NV][V], u[NV][V], g[NV][V], o[NV][V];
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < V; ++j) {
        n[i][j] = to_f(raw.p[0][i].e[j]) * a.scale;
        u[i][j] = to_f(raw.p[1][i].e[j]);
        g[i][j] = to_f(raw.p[2][i].e[j]);
        o[i][j] = to_f(raw.p[3][i].e[j]);
      }
    if (row + step < a.M) raw.load(a, row + step, t);
    // u: post's normalised row; n: the stream, then its normalised row
    float pinv = 1.f, inv = 1.f;
    if (a.y) {
      if (a.post != NORM_NONE) pinv = normalise<R, TPR, NV>(a.post, a.eps, d, t, sum, u);
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int c = R::col(i, t);
        float w[V], b[V], gt[V];
#pragma unroll
        for (int j = 0; j < V; ++j) {
          w[j] = 1.f;
          b[j] = 0.f;
          gt[j] = 1.f;
        }
        if (a.pw) R::load(a.pw, 0, c, d, w);
        if (a.pb) R::load(a.pb, 0, c, d, b);
        if (a.gate) R::load(a.gate, row * a.ldg, c, d, gt);
#pragma unroll
        for (int j = 0; j < V; ++j)
          if (c < d) n[i][j] = fmaf(gt[j], fmaf(u[i][j], w[j], b[j]), n[i][j]);
      }
    }
    if (a.dout) {
      if (a.norm != NORM_NONE) inv = normalise<R, TPR, NV>(a.norm, a.eps, d, t, sum, n);
      float s0 = 0.f, s1 = 0.f;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int c = R::col(i, t);
        float w[V];
#pragma unroll
        for (int j = 0; j < V; ++j) w[j] = 1.f;
        if (a.w) R::load(a.w, 0, c, d, w);
#pragma unroll
        for (int j = 0; j < V; ++j) {
          acc[0][i][j] = fmaf(o[i][j], n[i][j], acc[0][i][j]);
          acc[1][i][j] += o[i][j];
          o[i][j] *= w[j];
          s0 += o[i][j];
          s1 = fmaf(o[i][j], n[i][j], s1);
        }
      }
      if (a.norm != NORM_NONE) {
        const float2 m = sum.two(s0, s1);
        const float m0 = a.norm == NORM_LAYER ? m.x * rd : 0.f, m1 = m.y * rd;
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
          for (int j = 0; j < V; ++j) g[i][j] += (o[i][j] - m0 - n[i][j] * m1) * inv;
      } else {
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
          for (int j = 0; j < V; ++j) g[i][j] += o[i][j];
      }
    }
    // g: the stream's gradient
    if (a.dr) {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        float v[V];
#pragma unroll
        for (int j = 0; j < V; ++j) v[j] = g[i][j] * a.scale;
        R::store(a.dr, row * a.lddr, R::col(i, t), d, v);
      }
    }
    if (!a.y) continue;
    float s0 = 0.f, s1 = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = R::col(i, t);
      float w[V], b[V], gt[V], dg[V];
#pragma unroll
      for (int j = 0; j < V; ++j) {
        w[j] = 1.f;
        b[j] = 0.f;
        gt[j] = 1.f;
      }
      if (a.pw) R::load(a.pw, 0, c, d, w);
      if (a.gate) {
        if (a.pb) R::load(a.pb, 0, c, d, b);
        R::load(a.gate, row * a.ldg, c, d, gt);
      }
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const bool in = c < d;
        const float gj = in ? g[i][j] : 0.f;
        dg[j] = gj * fmaf(u[i][j], w[j], b[j]);
        acc[4][i][j] += dg[j];
        const float du = gj * gt[j];
        acc[2][i][j] = fmaf(du, u[i][j], acc[2][i][j]);
        acc[3][i][j] += du;
        g[i][j] = du * w[j];
        s0 += g[i][j];
        s1 = fmaf(g[i][j], u[i][j], s1);
      }
      if (a.dgate) R::store(a.dgate, row * a.lddg, c, d, dg);
    }
    if (a.dy) {
      if (a.post != NORM_NONE) {
        const float2 m = sum.two(s0, s1);
        const float m0 = a.post == NORM_LAYER ? m.x * rd : 0.f, m1 = m.y * rd;
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
          for (int j = 0; j < V; ++j) g[i][j] = (g[i][j] - m0 - u[i][j] * m1) * pinv;
      }
#pragma unroll
      for (int i = 0; i < NV; ++i) R::store(a.dy, row * a.lddy, R::col(i, t), d, g[i]);
    }
  }
  // this CTA's sums of the wanted vectors
  if (!a.part) return;
  if (TPR == 32) {
    __shared__ float total[TPR == 32 ? 32 * E : 1];
    int slot = 0;
    for (int v = 0; v < 5; ++v) {
      if (!((a.want >> v) & 1)) continue;
      for (int w = 0; w < 8; ++w) {
        if (warp == w) {
#pragma unroll
          for (int k = 0; k < 5; ++k)
            if (k == v)
#pragma unroll
              for (int i = 0; i < NV; ++i)
#pragma unroll
                for (int j = 0; j < V; ++j) {
                  const int c = R::col(i, t) + j;
                  total[c] = w ? total[c] + acc[k][i][j] : acc[k][i][j];
                }
        }
        __syncthreads();
      }
      float *dst = a.part + (static_cast<size_t>(slot) * gridDim.x + blockIdx.x) * d;
      for (int c = threadIdx.x; c < d; c += 256) dst[c] = total[c];
      __syncthreads();
      ++slot;
    }
  } else {
    int slot = 0;
#pragma unroll
    for (int v = 0; v < 5; ++v) {
      if (!((a.want >> v) & 1)) continue;
      float *dst = a.part + (static_cast<size_t>(slot) * gridDim.x + blockIdx.x) * d;
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const int c = R::col(i, t) + j;
          if (c < d) dst[c] = acc[v][i][j];
        }
      ++slot;
    }
  }
}

template <typename T, int TPR, int E, bool VEC, bool BWD>
void launch(const NormArgs &a, int grid, cudaStream_t s) {
  if constexpr (BWD) k_norm_bwd<T, TPR, E, VEC><<<grid, block_threads<TPR>(), 0, s>>>(a);
  else k_norm_fwd<T, TPR, E, VEC><<<grid, block_threads<TPR>(), 0, s>>>(a);
  CUDA_LAUNCH_CHECK();
}

// Threads per row of the backward (8 elements each, 16 at the ends of the
// range): its gradients' sums take five registers per element.
int bwd_threads(int d) { return d <= 512 ? 32 : d <= 1024 ? 128 : d <= 2048 ? 256 : d <= 4096 ? 512 : 1024; }
// CTAs of the backward: as many as are resident at once, each with its own
// share of the rows and one set of sums.
int bwd_grid(int64_t M, int d) {
  const int tpr = bwd_threads(d);
  const int64_t rows = tpr == 32 ? (M + 7) / 8 : M;
  const int per_sm = tpr <= 128 ? 4 : tpr == 256 ? 2 : 1;
  return static_cast<int>(std::min<int64_t>(rows, static_cast<int64_t>(per_sm) * sm_count()));
}

template <typename T, bool VEC>
void fwd(const NormArgs &a, cudaStream_t s) {
  const int d = a.d;
  const int64_t M = a.M;
  const int warps = static_cast<int>((M + 7) / 8), rows = static_cast<int>(M);
  if (d <= 256) launch<T, 32, 8, VEC, false>(a, warps, s);
  else if (d <= 512) launch<T, 32, 16, VEC, false>(a, warps, s);
  else if (d <= 1024) launch<T, 32, 32, VEC, false>(a, warps, s);
  else if (d <= 2048) launch<T, 128, 16, VEC, false>(a, rows, s);
  else if (d <= 4096) launch<T, 256, 16, VEC, false>(a, rows, s);
  else if (d <= 8192) launch<T, 256, 32, VEC, false>(a, rows, s);
  else launch<T, 512, 32, VEC, false>(a, rows, s);
}
template <typename T, bool VEC>
void bwd(const NormArgs &a, cudaStream_t s) {
  const int d = a.d, grid = bwd_grid(a.M, a.d);
  if (d <= 256) launch<T, 32, 8, VEC, true>(a, grid, s);
  else if (d <= 512) launch<T, 32, 16, VEC, true>(a, grid, s);
  else if (d <= 1024) launch<T, 128, 8, VEC, true>(a, grid, s);
  else if (d <= 2048) launch<T, 256, 8, VEC, true>(a, grid, s);
  else if (d <= 4096) launch<T, 512, 8, VEC, true>(a, grid, s);
  else if (d <= 8192) launch<T, 1024, 8, VEC, true>(a, grid, s);
  else launch<T, 1024, 16, VEC, true>(a, grid, s);
}
template <bool BWD>
void by_type(int dt, bool vec, const NormArgs &a, cudaStream_t s) {
  auto go = [&](auto tag, auto v) {
    using T = decltype(tag);
    if constexpr (BWD) bwd<T, decltype(v)::value != 0>(a, s);
    else fwd<T, decltype(v)::value != 0>(a, s);
  };
  if (dt == DT_F32) vec ? go(float{}, Const<1>{}) : go(float{}, Const<0>{});
  else if (dt == DT_F16) vec ? go(__half{}, Const<1>{}) : go(__half{}, Const<0>{});
  else vec ? go(__nv_bfloat16{}, Const<1>{}) : go(__nv_bfloat16{}, Const<0>{});
}

// Every tensor of the call can move in 16-byte pieces.
bool vectorised(const ResidualNorm &a) {
  if ((a.d * dtype_size(a.dtype)) % 16) return false;
  const Mat m[] = {a.residual, a.y, a.gate, a.dstream, a.dout, {a.stream.p, a.stream.ld}, {a.out.p, a.out.ld},
                   {a.dresidual.p, a.dresidual.ld}, {a.dy.p, a.dy.ld}, {a.dgate.p, a.dgate.ld}};
  for (const Mat &x : m)
    if (x.p && !rows16(x.p, x.ld, a.dtype)) return false;
  for (const void *v : {a.w, a.b, a.pw, a.pb})
    if (v && !aligned16(v)) return false;
  return true;
}

NormArgs args_of(const ResidualNorm &a) {
  NormArgs n{};
  n.M = a.M;
  n.d = a.d;
  n.norm = a.norm;
  n.post = a.post;
  n.scale = a.scale;
  n.eps = a.eps;
  n.r = a.residual.p;
  n.ldr = a.residual.ld;
  n.y = a.y.p;
  n.ldy = a.y.ld;
  n.gate = a.gate.p;
  n.ldg = a.gate.ld;
  n.w = a.w;
  n.b = a.b;
  n.pw = a.pw;
  n.pb = a.pb;
  return n;
}

}  // namespace
}  // namespace blk

using namespace blk;

void residual_norm_fwd(const ResidualNorm &a, Workspace &ws, cudaStream_t s) {
  if (a.M == 0 || ws.sizing()) return;
  NormArgs n = args_of(a);
  n.stream = a.stream.p;
  n.lds = a.stream.ld;
  n.out = a.out.p;
  n.ldo = a.out.ld;
  const bool vec = vectorised(a);
  if (a.out_split) {
    if (a.dtype != DT_F32 || !vec || a.d % 128) throw Error(kErrInternal, "residual_norm: split output needs aligned f32 rows");
    n.split = *a.out_split;
  }
  by_type<false>(a.dtype, vec, n, s);
}

void residual_norm_bwd(const ResidualNorm &a, Workspace &ws, cudaStream_t s) {
  // the vectors' gradients, in the order of NormArgs::want
  void *const grads[5] = {a.dw, a.db, a.dpw, a.dpb, a.dgate.p && a.gate.ld == 0 ? a.dgate.p : nullptr};
  if (a.M == 0) {
    for (void *g : grads)
      if (g && !ws.sizing()) CUDA_CHECK(cudaMemsetAsync(g, 0, a.d * dtype_size(a.dtype), s));
    return;
  }
  NormArgs n = args_of(a);
  int count = 0;
  for (int v = 0; v < 5; ++v)
    if (grads[v]) {
      n.want |= 1 << v;
      ++count;
    }
  const int grid = bwd_grid(a.M, a.d);
  if (count) n.part = static_cast<float *>(ws.take(4 * static_cast<size_t>(count) * grid * a.d));
  if (ws.sizing()) return;
  n.ds = a.dstream.p;
  n.ldds = a.dstream.ld;
  n.dout = a.dout.p;
  n.lddo = a.dout.ld;
  n.dr = a.dresidual.p;
  n.lddr = a.dresidual.ld;
  n.dy = a.dy.p;
  n.lddy = a.dy.ld;
  if (a.gate.ld != 0) {
    n.dgate = a.dgate.p;
    n.lddg = a.dgate.ld;
  }
  by_type<true>(a.dtype, vectorised(a), n, s);
  int slot = 0;
  for (int v = 0; v < 5; ++v)
    if (grads[v]) {
      column_join(n.part + static_cast<size_t>(slot) * grid * a.d, grid, a.d, 1.f, grads[v], a.dtype, s);
      ++slot;
    }
}

}  // namespace pet
