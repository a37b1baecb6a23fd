// The residual update between two norms, forward and backward:
//   u = post(y),  stream = scale r + gate u,  out = norm(stream).
// A row stays in registers from its one read to its one write, so the passes
// over memory are the inputs and the outputs, and HBM is what bounds both
// directions.  Means, variances and all gradients run in fp32 (variances in
// two passes over the registers), and `out` comes from the unrounded stream.
//
// The backward recomputes both norms from r and y: it reads r, y, dstream and
// dout and writes dr and dy, with no statistics stored by the forward.
//   dn = dout w,     g = dstream + norm'(dn)
//   dr = scale g,  dgate = g u,  dp = gate g pw,  dy = post'(dp)
// where norm'(dn) = (dn - [mean dn] - n mean(dn n)) / sigma.  The gradients
// of the vectors (weights, biases, a gate of one row) come from two sums over
// rows per column, four with biases (k_norm_vectors): kept per CTA over its
// rows in registers, written once per CTA and added in a fixed order.
//
// A CTA of 256 or more threads holds one or more groups of threads that take
// a row each, 8 or 16 elements a thread.  A group is persistent: the inputs of
// its next rows come into a ring in shared memory with bulk copies while it
// works on one, so that loads need no registers and the reductions' latency
// (two to six a row) is covered by the other groups and CTAs of the SM.  What
// has rows that are not 16-byte aligned, or too long for the ring, is read
// directly.
//
// Outputs leave L2 before anything else (__stcs): the inputs of later rows are
// still to be read there.  16,383 x 4096 f16 forward: 101 us a call, without 106.
//
// Measured: 16,383 x 4096 f16 forward in 98 us (5.5 TB/s), 8192 x 4096 bf16
// backward in 101 us (4.0 TB/s: four reductions a row and only two CTAs an SM,
// since a row's values and its column sums take 110 registers a thread).  Rows
// that are not 16-byte multiples, an element at a time and with spills, take 2.4
// and 3.1 times as long (4095 columns).
#include <algorithm>
#include <atomic>
#include <type_traits>

#include "block.cuh"
#include "tc_common.cuh"

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
  const void *ds, *dout;
  int64_t ldds, lddo;
  void *dr, *dy, *dgate;       // dgate: the gate of each row
  int64_t lddr, lddy, lddg;
  float *part;                 // [sum][CTA][d] of the vectors' gradients, or null
  bool hb;                     // a bias or its gradient is there
  int *err;                    // error word, or null for the file's own
};

// 16 bytes of T <-> pairs of floats
template <typename T>
__device__ __forceinline__ void open16(const uint4 &v, float2 *x) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
  if constexpr (sizeof(T) == 4) {
    x[0] = make_float2(__uint_as_float(w[0]), __uint_as_float(w[1]));
    x[1] = make_float2(__uint_as_float(w[2]), __uint_as_float(w[3]));
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if constexpr (std::is_same<T, __half>::value) x[k] = __half22float2(*reinterpret_cast<const __half2 *>(&w[k]));
      else x[k] = make_float2(__uint_as_float(w[k] << 16), __uint_as_float(w[k] & 0xffff0000u));
    }
  }
}
template <typename T>
__device__ __forceinline__ uint4 close16(const float2 *x) {
  uint32_t w[4];
  if constexpr (sizeof(T) == 4) {
    w[0] = __float_as_uint(x[0].x);
    w[1] = __float_as_uint(x[0].y);
    w[2] = __float_as_uint(x[1].x);
    w[3] = __float_as_uint(x[1].y);
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if constexpr (std::is_same<T, __half>::value) {
        const __half2 h = __floats2half2_rn(x[k].x, x[k].y);
        w[k] = *reinterpret_cast<const uint32_t *>(&h);
      } else {
        const __nv_bfloat162 h = __floats2bfloat162_rn(x[k].x, x[k].y);
        w[k] = *reinterpret_cast<const uint32_t *>(&h);
      }
    }
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// A thread's share of a row: E elements as E / 2 pairs (the pair forms of the
// fp32 instructions take one issue slot for two elements).  VEC: element e is
// in 16-byte chunk e / V, chunks of a row dealt out over its TPR threads;
// otherwise the elements are dealt out one by one.
// FULL: the row has exactly TPR * E columns, so nothing needs a bound.
template <typename T, int TPR, int E, bool VEC, bool FULL = false>
struct Row {
  static constexpr int V = VEC ? 16 / static_cast<int>(sizeof(T)) : 1;
  static constexpr int P = E / 2;
  static __device__ __forceinline__ int col(int i, int t) { return (i * TPR + t) * V; }
  // elements of one row at p + off; zeros past d (VEC: d is a multiple of V)
  static __device__ __forceinline__ void load(const void *p, int64_t off, int t, int d, float2 (&x)[P]) {
    const T *q = static_cast<const T *>(p) + off;
    if constexpr (VEC) {
#pragma unroll
      for (int i = 0; i < E / V; ++i) {
        uint4 v = make_uint4(0u, 0u, 0u, 0u);
        if (FULL || col(i, t) < d) v = *reinterpret_cast<const uint4 *>(q + col(i, t));
        open16<T>(v, &x[i * V / 2]);
      }
    } else {
#pragma unroll
      for (int k = 0; k < P; ++k) {
        const int c0 = col(2 * k, t), c1 = col(2 * k + 1, t);
        x[k] = make_float2(c0 < d ? to_f(q[c0]) : 0.f, c1 < d ? to_f(q[c1]) : 0.f);
      }
    }
  }
  static __device__ __forceinline__ void store(void *p, int64_t off, int t, int d, const float2 (&x)[P]) {
    T *q = static_cast<T *>(p) + off;
    if constexpr (VEC) {
#pragma unroll
      for (int i = 0; i < E / V; ++i)
        if (FULL || col(i, t) < d) __stcs(reinterpret_cast<uint4 *>(q + col(i, t)), close16<T>(&x[i * V / 2]));
    } else {
#pragma unroll
      for (int k = 0; k < P; ++k) {
        const int c0 = col(2 * k, t), c1 = col(2 * k + 1, t);
        if (c0 < d) q[c0] = from_f<T>(x[k].x);
        if (c1 < d) q[c1] = from_f<T>(x[k].y);
      }
    }
  }
  // fp32 copy of a vector in shared memory (VEC), zeros from d on, in the
  // order in which a warp reads it 16 bytes a lane: place of column c
  static constexpr int kCopy = TPR * E;
  static __device__ __forceinline__ int place(int c) {
    const int i = c / (TPR * V), t = c / V % TPR, j = c % V;
    return ((i * (V / 4) + j / 4) * TPR + t) * 4 + j % 4;
  }
  static __device__ __forceinline__ void load_copy(const float *p, int t, float2 (&x)[P]) {
#pragma unroll
    for (int k = 0; k < P; k += 2) {
      const float4 v = *reinterpret_cast<const float4 *>(p + (k / 2 * TPR + t) * 4);
      x[k] = make_float2(v.x, v.y);
      x[k + 1] = make_float2(v.z, v.w);
    }
  }
  // zeros into the columns past d
  static __device__ __forceinline__ void trim(int t, int d, float2 (&x)[P]) {
    if constexpr (!FULL) {
#pragma unroll
      for (int k = 0; k < P; ++k) {
        if (col(2 * k / V, t) >= d) x[k].x = 0.f;
        if (col((2 * k + 1) / V, t) >= d) x[k].y = 0.f;
      }
    }
  }
};

__device__ __forceinline__ float2 both(float a) { return make_float2(a, a); }
template <int P>
__device__ __forceinline__ float dot(const float2 (&a)[P], const float2 (&b)[P]) {
  float2 s = __fmul2_rn(a[0], b[0]);
#pragma unroll
  for (int k = 1; k < P; ++k) s = __ffma2_rn(a[k], b[k], s);
  return s.x + s.y;
}
template <int P>
__device__ __forceinline__ float total(const float2 (&a)[P]) {
  float2 s = a[0];
#pragma unroll
  for (int k = 1; k < P; ++k) s = __fadd2_rn(a[k], s);
  return s.x + s.y;
}

// The threads of one row: TPR of a CTA's, at a barrier of their own.
template <int TPR>
__device__ __forceinline__ void group_sync(int group) {
  if (TPR == 32) __syncwarp();
  else asm volatile("bar.sync %0, %1;" ::"r"(1 + group), "n"(TPR) : "memory");
}

// Sums over the threads of a row, in a fixed order.  Two slots in turn, so
// one barrier each: a slot is written again only after every thread has
// passed the barrier that follows its last read.
template <int TPR>
struct Sum {
  static constexpr int W = TPR / 32;  // warps of a row
  float *slots;                       // [2][32] of this group, 16-byte aligned
  int group, k;
  __device__ __forceinline__ float operator()(float a) {
    a = warp_sum(a);
    if (TPR == 32) return a;
    float *s = slots + (k & 1) * 32;
    k ^= 1;
    if ((threadIdx.x & 31) == 0) s[(threadIdx.x >> 5) % W] = a;
    group_sync<TPR>(group);
    if (W == 2) return s[0] + s[1];
    float4 v = *reinterpret_cast<const float4 *>(s);
#pragma unroll
    for (int i = 4; i < (W > 4 ? W : 4); i += 4) {
      const float4 u = *reinterpret_cast<const float4 *>(s + i);
      v.x += u.x;
      v.y += u.y;
      v.z += u.z;
      v.w += u.w;
    }
    return (v.x + v.y) + (v.z + v.w);
  }
};

// x -> its normalised row (columns past d stay 0); returns 1 / sigma.
template <typename R, int TPR>
__device__ __forceinline__ float normalise(int kind, float eps, int d, float rd, int t, Sum<TPR> &sum, float2 (&x)[R::P]) {
  if (kind == NORM_LAYER) {
    const float mean = sum(total(x)) * rd;
#pragma unroll
    for (int k = 0; k < R::P; ++k) x[k] = __fadd2_rn(x[k], both(-mean));
    R::trim(t, d, x);
  }
  const float inv = rsqrtf(fmaf(sum(dot(x, x)), rd, eps));  // 2 ulp
#pragma unroll
  for (int k = 0; k < R::P; ++k) x[k] = __fmul2_rn(x[k], both(inv));
  return inv;
}

__device__ int g_norm_err = 0;

constexpr int kMaxStages = 4;
constexpr int kInputs = 5;  // rows of a stage: r, y, dstream, dout, gate

// Shared memory of a CTA: fp32 copies of the vectors there are (Vectors),
// then per group a ring of `stages` stages of `inputs` rows.
struct Ring {
  int stages, inputs;  // stages 0: rows are read directly
  int row_bytes, vector_bytes;
  bool stall;  // test hook: the first group of the first CTA issues no copies
  int bytes(int groups) const { return vector_bytes + row_bytes * groups * stages * inputs; }
};

// One group's ring: `take` waits for the next row's inputs.  A thread whose
// wait runs out records the error and waits no more: the results are void.  The
// one that issues the copies issues no further ones, so that no barrier is armed
// again in an unfinished phase (the others run into their own bounds, once each),
// and waits at its end, with the default bound, for those on their way: no CTA
// ends while something is written to its shared memory.
template <int TPR>
struct Feed {
  const NormArgs &a;
  const Ring &ring;
  uint64_t *bars;
  char *base;
  int64_t row, step;
  int t, stage, phase;
  int lost;  // 1 + rows since the wait that ran out, or 0
  __device__ __forceinline__ void issue(int s, int64_t at) {
    const void *src[kInputs] = {a.r, a.y, a.ds, a.dout, a.ldg ? a.gate : nullptr};
    const int64_t ld[kInputs] = {a.ldr, a.ldy, a.ldds, a.lddo, a.ldg};
    const uint32_t bar = tc::smem_u32(bars + s);
    const int64_t es = ring.row_bytes / a.d;
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(ring.inputs * ring.row_bytes) : "memory");
    char *dst = base + static_cast<size_t>(s) * ring.inputs * ring.row_bytes;
#pragma unroll
    for (int k = 0; k < kInputs; ++k) {
      if (!src[k]) continue;
      asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                   ::"r"(tc::smem_u32(dst)), "l"(static_cast<const char *>(src[k]) + at * ld[k] * es),
                     "r"(ring.row_bytes), "r"(bar) : "memory");
      dst += ring.row_bytes;
    }
  }
  __device__ __forceinline__ bool stalled() const { return ring.stall && blockIdx.x == 0 && threadIdx.x < TPR; }
  __device__ __forceinline__ void start() {
    if (t == 0 && !stalled())
      for (int s = 0; s < ring.stages && row + s * step < a.M; ++s) issue(s, row + s * step);
  }
  __device__ __forceinline__ const char *take() {
    const uint32_t bar = tc::smem_u32(bars + stage);
    if (!lost && !tc::mbar_try_wait(bar, phase) && !tc::wait_within(bar, phase)) {
      lost = 1;
      raise_error(a.err, g_norm_err);
    }
    return base + static_cast<size_t>(stage) * ring.inputs * ring.row_bytes;
  }
  // every thread of the group has read the stage (after a group barrier)
  __device__ __forceinline__ void give(int64_t at) {
    if (t == 0 && !lost && at + ring.stages * step < a.M) issue(stage, at + ring.stages * step);
    lost += lost != 0;
    if (++stage == ring.stages) {
      stage = 0;
      phase ^= 1;
    }
  }
  // after the last row: the row of the wait that ran out and the ring's next
  // ones, as far as there were rows, had been issued
  __device__ __forceinline__ void end() {
    if (!lost || t != 0 || stalled()) return;
    const int n = ring.stages, rows = lost - 1, first = phase * n + stage - rows % (2 * n) + 2 * n;
    for (int i = 0; i < min(n, rows); ++i) {
      const int at = (first + i) % (2 * n);
      tc::wait_bounded(tc::smem_u32(bars + at % n), at / n);
    }
  }
};

// What a row is multiplied with and shifted by after post (gw, gb, with the
// gate where it is one row for all) and after norm (w, b): in shared memory
// in fp32 (RING) or the tensors themselves.
template <typename R, typename T, bool RING>
struct Vectors {
  const NormArgs &a;
  const float *w = nullptr, *b = nullptr, *gw = nullptr, *gb = nullptr;
  static __host__ __device__ int count(const NormArgs &a) {
    const bool row = a.gate && !a.ldg;
    return (a.w ? 1 : 0) + (a.b ? 1 : 0) + (a.pw || row ? 1 : 0) + (a.pb ? 1 : 0);
  }
  // all threads of the CTA; returns the end of the copies
  __device__ __forceinline__ void copy(float *dst) {
    const T *gate = a.ldg ? nullptr : static_cast<const T *>(a.gate);
    auto one = [&](const void *p, const T *times, const float *&out) {
      if (!p && !times) return;
      const T *q = static_cast<const T *>(p);
      for (int c = threadIdx.x; c < R::kCopy; c += blockDim.x)
        dst[R::place(c)] = c < a.d ? (q ? to_f(q[c]) : 1.f) * (times ? to_f(times[c]) : 1.f) : 0.f;
      out = dst;
      dst += R::kCopy;
    };
    one(a.w, nullptr, w);
    one(a.b, nullptr, b);
    one(a.pw, gate, gw);
    if (a.pb) one(a.pb, gate, gb);
  }
  __device__ __forceinline__ void scale(const float *in, const void *p, const void *times, int t, float2 (&x)[R::P], bool add) const {
    float2 f[R::P];
    if (RING) {
      if (!in) return;
      R::load_copy(in, t, f);
    } else {
      if (!p && !times) return;
      if (p) R::load(p, 0, t, a.d, f);
      if (times) {
        float2 g[R::P];
        R::load(times, 0, t, a.d, g);
#pragma unroll
        for (int k = 0; k < R::P; ++k) f[k] = p ? __fmul2_rn(f[k], g[k]) : g[k];
      }
    }
#pragma unroll
    for (int k = 0; k < R::P; ++k) x[k] = add ? __fadd2_rn(x[k], f[k]) : __fmul2_rn(x[k], f[k]);
  }
  __device__ __forceinline__ const void *row_gate() const { return a.ldg ? nullptr : a.gate; }
  __device__ __forceinline__ void times_w(int t, float2 (&x)[R::P]) const { scale(w, a.w, nullptr, t, x, false); }
  __device__ __forceinline__ void plus_b(int t, float2 (&x)[R::P]) const { scale(b, a.b, nullptr, t, x, true); }
  __device__ __forceinline__ void times_gw(int t, float2 (&x)[R::P]) const { scale(gw, a.pw, row_gate(), t, x, false); }
  __device__ __forceinline__ void plus_gb(int t, float2 (&x)[R::P]) const {
    if (a.pb) scale(gb, a.pb, row_gate(), t, x, true);
  }
};

// What both directions set up: this thread's group, its first row, its ring
// and the vectors.
#define PET_NORM_SETUP                                                                                     \
  extern __shared__ __align__(128) char smem[];                                                            \
  __shared__ alignas(16) float slots[NG][64];                                                              \
  __shared__ uint64_t bars[NG][kMaxStages];                                                                \
  const int t = threadIdx.x % TPR, group = threadIdx.x / TPR, d = a.d;                                     \
  const float rd = 1.f / static_cast<float>(d);                                                            \
  const int64_t step = static_cast<int64_t>(gridDim.x) * NG;                                               \
  int64_t row = static_cast<int64_t>(blockIdx.x) * NG + group;                                             \
  Sum<TPR> sum{slots[group], group, 0};                                                                    \
  Vectors<R, T, RING> vec{a};                                                                              \
  Feed<TPR> feed{a, ring, bars[group], nullptr, row, step, t, 0, 0, 0};                                    \
  if (RING) {                                                                                              \
    if (threadIdx.x == 0) {                                                                                \
      for (int g = 0; g < NG; ++g)                                                                         \
        for (int s = 0; s < ring.stages; ++s) tc::mbar_init(tc::smem_u32(&bars[g][s]), 1);                 \
      asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");                                   \
    }                                                                                                      \
    __syncthreads();                                                                                       \
    feed.base = smem + ring.vector_bytes + static_cast<size_t>(ring.row_bytes) * group * ring.stages * ring.inputs; \
    feed.start();                                                                                          \
    vec.copy(reinterpret_cast<float *>(smem));                                                             \
    __syncthreads();                                                                                       \
  }

// NT threads, NT / TPR groups.  MODE 0: single elements, 1: 16-byte pieces,
// 2: with the inputs' rows in the ring, 3: and FULL rows.
template <typename T, int TPR, int NT, int E, int MODE>
__global__ void __launch_bounds__(NT, 1024 / NT) k_norm_fwd(const NormArgs a, const Ring ring) {
  using R = Row<T, TPR, E, MODE != 0, MODE == 3>;
  constexpr int P = R::P, NG = NT / TPR;
  constexpr bool RING = MODE >= 2;
  PET_NORM_SETUP
  for (; row < a.M; row += step) {
    float2 x[P];
    const char *in = nullptr;
    if (RING) in = feed.take();
    if (RING) R::load(in, 0, t, d, x);
    else R::load(a.r, row * a.ldr, t, d, x);
#pragma unroll
    for (int k = 0; k < P; ++k) x[k] = __fmul2_rn(x[k], both(a.scale));
    if (a.y) {
      float2 u[P];
      if (RING) R::load(in + ring.row_bytes, 0, t, d, u);
      else R::load(a.y, row * a.ldy, t, d, u);
      if (a.post != NORM_NONE) normalise<R, TPR>(a.post, a.eps, d, rd, t, sum, u);
      vec.times_gw(t, u);
      vec.plus_gb(t, u);
      if (a.ldg) {
        float2 f[P];
        if (RING) R::load(in + 2 * ring.row_bytes, 0, t, d, f);
        else R::load(a.gate, row * a.ldg, t, d, f);
#pragma unroll
        for (int k = 0; k < P; ++k) x[k] = __ffma2_rn(u[k], f[k], x[k]);
      } else {
#pragma unroll
        for (int k = 0; k < P; ++k) x[k] = __fadd2_rn(x[k], u[k]);
      }
    }
    if (RING) {
      group_sync<TPR>(group);
      feed.give(row);
    }
    if (a.stream) R::store(a.stream, row * a.lds, t, d, x);
    if (!a.out) continue;
    if (a.norm != NORM_NONE) normalise<R, TPR>(a.norm, a.eps, d, rd, t, sum, x);
    vec.times_w(t, x);
    vec.plus_b(t, x);
    if (a.out) R::store(a.out, row * a.ldo, t, d, x);
  }
  if (RING) feed.end();
}

// HB: a bias or its gradient is there (its sums take E registers each).
template <typename T, int TPR, int NT, int E, int MODE, bool HB>
__global__ void __launch_bounds__(NT, NT == 256 ? 2 : 1) k_norm_bwd(const NormArgs a, const Ring ring) {
  using R = Row<T, TPR, E, MODE != 0, MODE == 3>;
  constexpr int P = R::P, NG = NT / TPR;
  constexpr bool RING = MODE >= 2;
  PET_NORM_SETUP
  const bool each = a.ldg != 0;  // a gate for every row
  // sums over rows of do n, q u (and do, q), where q is the stream's
  // gradient, times the gate if each row has its own
  constexpr int NA = HB ? 4 : 2;
  float2 acc[NA][P];
#pragma unroll
  for (int v = 0; v < NA; ++v)
#pragma unroll
    for (int k = 0; k < P; ++k) acc[v][k] = both(0.f);
  for (; row < a.M; row += step) {
    float2 n[P], u[P], g[P], f[P];
    const char *in[kInputs] = {};
    if (RING) {
      const char *p = feed.take();
      const void *there[kInputs] = {a.r, a.y, a.ds, a.dout, each ? a.gate : nullptr};
#pragma unroll
      for (int k = 0; k < kInputs; ++k) {
        in[k] = p;
        if (there[k]) p += ring.row_bytes;
      }
    }
    auto input = [&](int k, const void *p, int64_t ld, float2(&x)[P]) {
      if (RING) R::load(in[k], 0, t, d, x);
      else R::load(p, row * ld, t, d, x);
    };
    // times the row's own gate
    auto gated = [&](float2(&x)[P]) {
      if (!each) return;
      input(4, a.gate, a.ldg, f);
#pragma unroll
      for (int k = 0; k < P; ++k) x[k] = __fmul2_rn(x[k], f[k]);
    };
    // u: post's normalised row; n: the stream, then its normalised row
    input(0, a.r, a.ldr, n);
#pragma unroll
    for (int k = 0; k < P; ++k) n[k] = __fmul2_rn(n[k], both(a.scale));
    float pinv = 1.f;
    if (a.y) {
      input(1, a.y, a.ldy, u);
      if (a.post != NORM_NONE) pinv = normalise<R, TPR>(a.post, a.eps, d, rd, t, sum, u);
#pragma unroll
      for (int k = 0; k < P; ++k) g[k] = u[k];
      vec.times_gw(t, g);
      if (HB) vec.plus_gb(t, g);
      gated(g);
#pragma unroll
      for (int k = 0; k < P; ++k) n[k] = __fadd2_rn(n[k], g[k]);
    }
    float inv = 1.f;
    if (a.dout) {
      float2 (&o)[P] = g;
      if (a.norm != NORM_NONE) inv = normalise<R, TPR>(a.norm, a.eps, d, rd, t, sum, n);
      input(3, a.dout, a.lddo, o);
#pragma unroll
      for (int k = 0; k < P; ++k) {
        acc[0][k] = __ffma2_rn(o[k], n[k], acc[0][k]);
        if (HB) acc[NA / 2][k] = __fadd2_rn(acc[NA / 2][k], o[k]);
      }
      vec.times_w(t, o);
      if (a.norm != NORM_NONE) {
        if (a.norm == NORM_LAYER) {
          const float m0 = sum(total(o)) * rd;
          // (the mean of n is 0: what follows does not see the shift)
#pragma unroll
          for (int k = 0; k < P; ++k) o[k] = __fadd2_rn(o[k], both(-m0));
          R::trim(t, d, o);
        }
        const float m1 = -sum(dot(o, n)) * rd;
#pragma unroll
        for (int k = 0; k < P; ++k) o[k] = __fmul2_rn(__ffma2_rn(n[k], both(m1), o[k]), both(inv));
      }
    } else {
#pragma unroll
      for (int k = 0; k < P; ++k) g[k] = both(0.f);
    }
    if (a.ds) {
      input(2, a.ds, a.ldds, f);
#pragma unroll
      for (int k = 0; k < P; ++k) g[k] = __fadd2_rn(g[k], f[k]);
    }
    // g: the stream's gradient
    if (a.dr) {
#pragma unroll
      for (int k = 0; k < P; ++k) f[k] = __fmul2_rn(g[k], both(a.scale));
      R::store(a.dr, row * a.lddr, t, d, f);
    }
    if (a.y) {
      if (a.dgate) {  // (the gate is the row's own: gw and gb are pw and pb)
        float2 (&v)[P] = n;
#pragma unroll
        for (int k = 0; k < P; ++k) v[k] = u[k];
        vec.times_gw(t, v);
        if (HB) vec.plus_gb(t, v);
#pragma unroll
        for (int k = 0; k < P; ++k) v[k] = __fmul2_rn(v[k], g[k]);
        R::store(a.dgate, row * a.lddg, t, d, v);
      }
      gated(g);
#pragma unroll
      for (int k = 0; k < P; ++k) {
        acc[1][k] = __ffma2_rn(g[k], u[k], acc[1][k]);
        if (HB) acc[NA - 1][k] = __fadd2_rn(acc[NA - 1][k], g[k]);
      }
      vec.times_gw(t, g);
    }
    if (RING) {
      group_sync<TPR>(group);
      feed.give(row);
    }
    if (a.dy) {
      if (a.post != NORM_NONE) {
        if (a.post == NORM_LAYER) {
          const float m0 = sum(total(g)) * rd;
#pragma unroll
          for (int k = 0; k < P; ++k) g[k] = __fadd2_rn(g[k], both(-m0));
          R::trim(t, d, g);
        }
        const float m1 = -sum(dot(g, u)) * rd;
#pragma unroll
        for (int k = 0; k < P; ++k) g[k] = __fmul2_rn(__ffma2_rn(u[k], both(m1), g[k]), both(pinv));
      }
      R::store(a.dy, row * a.lddy, t, d, g);
    }
  }
  if (RING) feed.end();
  // this CTA's sums, each [CTA][d], the groups' added in order
  if (!a.part) return;
#pragma unroll
  for (int v = 0; v < NA; ++v) {
    float *dst = a.part + (static_cast<size_t>(v) * gridDim.x + blockIdx.x) * d;
    if constexpr (NG == 1) {
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const int c = R::col(e / R::V, t) + e % R::V;
        if (c < d) dst[c] = e % 2 ? acc[v][e / 2].y : acc[v][e / 2].x;
      }
    } else {
      __shared__ float sums[NG > 1 ? TPR * E : 1];
      for (int i = 0; i < NG; ++i) {
        if (group == i) {
#pragma unroll
          for (int e = 0; e < E; ++e) {
            const int c = R::col(e / R::V, t) + e % R::V;
            const float x = e % 2 ? acc[v][e / 2].y : acc[v][e / 2].x;
            sums[c] = i ? sums[c] + x : x;
          }
        }
        __syncthreads();
      }
      for (int c = threadIdx.x; c < d; c += NT) dst[c] = sums[c];
      __syncthreads();
    }
  }
}

// The vectors' gradients from the CTAs' sums, in a fixed order; block: 32
// columns x 32 interleaved shares.
//   dw = sum do n, db = sum do;  with one gate for all rows (or none)
//   dpw = gate sum q u, dpb = gate sum q, dgate = pw sum q u + pb sum q.
struct VectorGrads {
  const float *part;
  int P, d, dt;
  bool hb;
  const void *pw, *pb, *gate;  // gate: of one row, or null
  void *dw, *db, *dpw, *dpb, *dgate;
};
__global__ void __launch_bounds__(1024) k_norm_vectors(const VectorGrads a) {
  __shared__ float sums[4][32][33];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int c = blockIdx.x * 32 + lane, na = a.hb ? 4 : 2;
  for (int v = 0; v < na; ++v) {
    float s = 0.f;
    if (c < a.d) {
      const float *p = a.part + static_cast<size_t>(v) * a.P * a.d + c;
#pragma unroll 8
      for (int q = warp; q < a.P; q += 32) s += p[static_cast<size_t>(q) * a.d];
    }
    sums[v][warp][lane] = s;
  }
  __syncthreads();
  if (warp || c >= a.d) return;
  float s[4] = {0.f, 0.f, 0.f, 0.f};
  for (int v = 0; v < na; ++v)
#pragma unroll
    for (int i = 0; i < 32; ++i) s[v] += sums[v][i][lane];
  const float gate = a.gate ? load_dt(a.gate, a.dt, c) : 1.f;
  if (a.dw) store_dt(a.dw, a.dt, c, s[0]);
  if (a.db) store_dt(a.db, a.dt, c, s[2]);
  if (a.dpw) store_dt(a.dpw, a.dt, c, gate * s[1]);
  if (a.dpb) store_dt(a.dpb, a.dt, c, gate * s[3]);
  if (a.dgate) {
    const float pw = a.pw ? load_dt(a.pw, a.dt, c) : 1.f, pb = a.pb ? load_dt(a.pb, a.dt, c) : 0.f;
    store_dt(a.dgate, a.dt, c, pw * s[1] + pb * s[3]);
  }
}

constexpr int kSmemPerSm = 224 * 1024;

// How a call is laid out: threads per row and per CTA, CTAs per SM and the
// ring.  16-bit rows take 16 elements a thread and two CTAs of 256 threads an
// SM (128 registers a thread hold a row's values and its column sums); f32
// rows 8 and one of 512, since their ring is twice as large.  The grid is what
// is resident at once.
struct Layout {
  int tpr, nt, grid;
  Ring ring;
};
Layout layout_of(const NormArgs &a, int dt, bool vec, bool bwd) {
  const int es = static_cast<int>(dtype_size(dt)), e = dt == DT_F32 ? 8 : 16;
  Layout l{32, dt == DT_F32 ? 512 : 256, 0, {0, 0, a.d * es, Vectors<Row<float, 32, 8, true>, float, true>::count(a), false}};
  while (l.tpr * e < a.d && l.tpr < 1024) l.tpr *= 2;
  l.ring.vector_bytes *= 4 * l.tpr * (l.tpr == 1024 ? 16 : e);
  l.nt = std::max(l.nt, l.tpr);
  const int groups = l.nt / l.tpr;
  // forwards hold half the registers
  int per_sm = std::max(1, (bwd ? 512 : 1024) / l.nt);
  if (vec) {
    Ring &r = l.ring;
    for (const void *p : {a.r, a.y, a.ds, a.dout, a.ldg ? a.gate : nullptr}) r.inputs += p ? 1 : 0;
    // the kernels' own arrays (slots, barriers, the groups' sums) and what the
    // system keeps of each CTA's shared memory
    const int fixed = 2048 + 320 * groups + (bwd && groups > 1 ? 4 * l.tpr * e : 0);
    // at least two stages, fewer CTAs rather than fewer stages
    for (; per_sm >= 1; --per_sm) {
      const int room = kSmemPerSm / per_sm - fixed - r.vector_bytes;
      r.stages = std::min(kMaxStages, room / (groups * r.inputs * r.row_bytes));
      if (r.stages >= 2) break;
    }
    if (per_sm < 1) {
      r.stages = 0;
      per_sm = std::max(1, (bwd ? 512 : 1024) / l.nt);
    }
  }
  l.grid = static_cast<int>(std::min<int64_t>((a.M + groups - 1) / groups, static_cast<int64_t>(per_sm) * sm_count()));
  return l;
}

std::atomic<bool> g_norm_stall{false};

template <typename T, int TPR, int NT, int E, int MODE, bool BWD>
void launch(const NormArgs &a, const Layout &l, cudaStream_t s) {
  const int smem = MODE >= 2 ? l.ring.bytes(NT / TPR) : 0;
  Ring ring = l.ring;
  ring.stall = MODE >= 2 && norm_stall_armed() && g_norm_stall.exchange(false);
  auto go = [&](auto *kernel) {
    if (smem) CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    kernel<<<l.grid, NT, smem, s>>>(a, ring);
    CUDA_LAUNCH_CHECK();
  };
  if constexpr (!BWD) go(k_norm_fwd<T, TPR, NT, E, MODE>);
  else if (a.hb) go(k_norm_bwd<T, TPR, NT, E, MODE, true>);
  else go(k_norm_bwd<T, TPR, NT, E, MODE, false>);
}
template <typename T, int TPR, int NT, int E, bool BWD>
void by_feed(const NormArgs &a, const Layout &l, bool vec, cudaStream_t s) {
  if (l.ring.stages && a.d == TPR * E) launch<T, TPR, NT, E, 3, BWD>(a, l, s);
  else if (l.ring.stages) launch<T, TPR, NT, E, 2, BWD>(a, l, s);
  else if (vec) launch<T, TPR, NT, E, 1, BWD>(a, l, s);
  else launch<T, TPR, NT, E, 0, BWD>(a, l, s);
}
template <typename T, bool BWD>
void by_width(const NormArgs &a, const Layout &l, bool vec, cudaStream_t s) {
  constexpr int E = sizeof(T) == 4 ? 8 : 16, NT = sizeof(T) == 4 ? 512 : 256;
  switch (l.tpr) {
    case 32: by_feed<T, 32, NT, E, BWD>(a, l, vec, s); break;
    case 64: by_feed<T, 64, NT, E, BWD>(a, l, vec, s); break;
    case 128: by_feed<T, 128, NT, E, BWD>(a, l, vec, s); break;
    case 256: by_feed<T, 256, NT, E, BWD>(a, l, vec, s); break;
    case 512: by_feed<T, 512, 512, E, BWD>(a, l, vec, s); break;
    default: by_feed<T, 1024, 1024, 16, BWD>(a, l, vec, s); break;  // up to 16,384
  }
}
template <bool BWD>
void by_type(int dt, bool vec, const NormArgs &a, const Layout &l, cudaStream_t s) {
  if (dt == DT_F32) by_width<float, BWD>(a, l, vec, s);
  else if (dt == DT_F16) by_width<__half, BWD>(a, l, vec, s);
  else by_width<__nv_bfloat16, BWD>(a, l, vec, s);
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
  n.ldg = a.gate.p ? a.gate.ld : 0;
  n.w = a.w;
  n.b = a.b;
  n.pw = a.pw;
  n.pb = a.pb;
  n.err = a.err;
  return n;
}

}  // namespace
}  // namespace blk

using namespace blk;

bool blk::norm_error(cudaStream_t s) { return new_errors(g_norm_err, s); }
void blk::norm_wait_bound(uint64_t ns) { CUDA_CHECK(cudaMemcpyToSymbol(tc::g_wait_ns, &ns, sizeof(ns))); }

void inject_norm_stall() { g_norm_stall.store(true); }
bool norm_stall_armed() { return g_norm_stall.load(std::memory_order_relaxed); }

void residual_norm_fwd(const ResidualNorm &a, Workspace &ws, cudaStream_t s) {
  if (a.M == 0 || ws.sizing()) return;
  NormArgs n = args_of(a);
  n.stream = a.stream.p;
  n.lds = a.stream.ld;
  n.out = a.out.p;
  n.ldo = a.out.ld;
  const bool vec = vectorised(a);
  by_type<false>(a.dtype, vec, n, layout_of(n, a.dtype, vec, false), s);
}

void residual_norm_bwd(const ResidualNorm &a, Workspace &ws, cudaStream_t s) {
  void *const dgate = a.dgate.ld == 0 ? a.dgate.p : nullptr;  // of one row
  if (a.M == 0) {
    for (void *g : {a.dw, a.db, a.dpw, a.dpb, dgate})
      if (g && !ws.sizing()) CUDA_CHECK(cudaMemsetAsync(g, 0, a.d * dtype_size(a.dtype), s));
    return;
  }
  NormArgs n = args_of(a);
  n.hb = a.pb || a.db || a.dpb;
  n.ds = a.dstream.p;
  n.ldds = a.dstream.ld;
  n.dout = a.dout.p;
  n.lddo = a.dout.ld;
  n.dr = a.dresidual.p;
  n.lddr = a.dresidual.ld;
  n.dy = a.dy.p;
  n.lddy = a.dy.ld;
  if (n.ldg != 0) {
    n.dgate = a.dgate.p;
    n.lddg = a.dgate.ld;
  }
  const bool vec = vectorised(a), vectors = a.dw || a.db || a.dpw || a.dpb || dgate;
  const Layout l = layout_of(n, a.dtype, vec, true);
  if (vectors) n.part = static_cast<float *>(ws.take(4 * static_cast<size_t>(n.hb ? 4 : 2) * l.grid * a.d));
  if (ws.sizing()) return;
  by_type<true>(a.dtype, vec, n, l, s);
  if (!vectors) return;
  const VectorGrads v{n.part, l.grid, a.d, a.dtype, n.hb, a.pw, a.pb, a.gate.ld == 0 ? a.gate.p : nullptr,
                      a.dw, a.db, a.dpw, a.dpb, dgate};
  k_norm_vectors<<<ceil_div(a.d, 32), 1024, 0, s>>>(v);
  CUDA_LAUNCH_CHECK();
}

}  // namespace pet
