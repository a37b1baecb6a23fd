// Transformer-block operators for a handful of rows (single tokens), and the
// column sums of the bias gradients.
//
// With at most 8 rows the dense forward is the time it takes to read the
// weights once: one to eight warps per output feature stream its weight rows
// with 16-byte loads, several in flight per lane, and multiply them with every
// row of x, which stays in L1.  The sums run in fp32 FMAs; the tensor cores
// would idle behind the same loads, and a 128-row tile would leave most SMs
// without work.
//
// The backward of so few rows is the same for the weights (read once for dz,
// once for dx, and their gradients written once): dz in fp32 by the forward's
// kernel, dW = dz^T x and db as one pass of stores, dx = dz W in strips of W's
// rows whose fp32 sums a last kernel adds in order.
#include <algorithm>

#include "block.cuh"

namespace pet {
namespace blk {

namespace {

constexpr int kDepth = 4;  // loads in flight per lane and weight (8 cost more in resident warps)

template <typename T, int MR, bool DUAL, bool VEC>
__global__ void __launch_bounds__(256) k_few_rows(const FewRows a, int wpr) {
  constexpr int V = VEC ? 16 / static_cast<int>(sizeof(T)) : 1;
  constexpr int NS = DUAL ? 2 * MR : MR;
  __shared__ float part[8][NS];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t n = static_cast<int64_t>(blockIdx.x) * (8 / wpr) + warp / wpr;
  const int sub = warp % wpr;
  float sum[NS];
#pragma unroll
  for (int i = 0; i < NS; ++i) sum[i] = 0.f;
  if (n < a.N) {
    const T *x = static_cast<const T *>(a.x);
    const T *w0 = static_cast<const T *>(a.w0) + n * a.ldw0;
    const T *w1 = DUAL ? static_cast<const T *>(a.w1) + n * a.ldw1 : nullptr;
    const int64_t step = static_cast<int64_t>(wpr) * 32 * V;
    for (int64_t k0 = (static_cast<int64_t>(sub) * 32 + lane) * V; k0 < a.K; k0 += kDepth * step) {
      if (VEC) {
        uint4 r0[kDepth], r1[kDepth];
#pragma unroll
        for (int u = 0; u < kDepth; ++u) {
          const int64_t k = k0 + u * step;
          r0[u] = r1[u] = make_uint4(0u, 0u, 0u, 0u);
          if (k < a.K) {
            r0[u] = __ldg(reinterpret_cast<const uint4 *>(w0 + k));
            if (DUAL) r1[u] = __ldg(reinterpret_cast<const uint4 *>(w1 + k));
          }
        }
#pragma unroll
        for (int u = 0; u < kDepth; ++u) {
          const int64_t k = k0 + u * step;
          if (k >= a.K) break;
          float f0[16 / sizeof(T)], f1[16 / sizeof(T)];
          unpack<T>(r0[u], f0);
          if (DUAL) unpack<T>(r1[u], f1);
#pragma unroll
          for (int m = 0; m < MR; ++m) {
            if (m >= a.M) break;
            float xv[16 / sizeof(T)];
            unpack<T>(__ldg(reinterpret_cast<const uint4 *>(x + m * a.ldx + k)), xv);
#pragma unroll
            for (int j = 0; j < V; ++j) {
              sum[m] = fmaf(xv[j], f0[j], sum[m]);
              if (DUAL) sum[MR * (DUAL ? 1 : 0) + m] = fmaf(xv[j], f1[j], sum[MR * (DUAL ? 1 : 0) + m]);
            }
          }
        }
      } else {
#pragma unroll
        for (int u = 0; u < kDepth; ++u) {
          const int64_t k = k0 + u * step;
          if (k >= a.K) break;
          const float f0 = to_f(w0[k]), f1 = DUAL ? to_f(w1[k]) : 0.f;
#pragma unroll
          for (int m = 0; m < MR; ++m) {
            if (m >= a.M) break;
            const float xv = to_f(x[m * a.ldx + k]);
            sum[m] = fmaf(xv, f0, sum[m]);
            if (DUAL) sum[MR * (DUAL ? 1 : 0) + m] = fmaf(xv, f1, sum[MR * (DUAL ? 1 : 0) + m]);
          }
        }
      }
    }
  }
#pragma unroll
  for (int i = 0; i < NS; ++i) sum[i] = warp_sum(sum[i]);
  if (wpr > 1) {
    if (lane == 0) {
#pragma unroll
      for (int i = 0; i < NS; ++i) part[warp][i] = sum[i];
    }
    __syncthreads();
    if (sub) return;
#pragma unroll
    for (int i = 0; i < NS; ++i) {
      float t = 0.f;
      for (int w = 0; w < wpr; ++w) t += part[warp + w][i];
      sum[i] = t;
    }
  }
  // lane m finishes row m
  float v = 0.f, w = 0.f;
#pragma unroll
  for (int m = 0; m < MR; ++m)
    if (lane == m) {
      v = sum[m];
      if (DUAL) w = sum[MR * (DUAL ? 1 : 0) + m];
    }
  if (n >= a.N || lane >= a.M) return;
  if (a.b0) v += to_f(static_cast<const T *>(a.b0)[n]);
  if (DUAL && a.b1) w += to_f(static_cast<const T *>(a.b1)[n]);
  const float in = a.in ? to_f(static_cast<const T *>(a.in)[lane * a.ldin + n]) : 0.f;
  float da;
  with_act(a.act, [&](auto A) { act_pair<decltype(A)::value>(v, v, da); });
  if (!a.out) {  // backward: [product][row][feature]
    a.dz[lane * a.N + n] = DUAL ? da * w * in : da * a.scale * in;
    if (DUAL) a.dz[(a.M + lane) * a.N + n] = v * in;
    return;
  }
  if (DUAL) v *= w;
  else v = v * a.scale + in;
  static_cast<T *>(a.out)[lane * a.ldo + n] = from_f<T>(v);
}

template <typename T, int MR, bool DUAL>
void launch_rows(const FewRows &a, cudaStream_t s) {
  constexpr int V = 16 / static_cast<int>(sizeof(T));
  const bool vec = a.K % V == 0 && rows16(a.x, a.ldx, a.dt) && rows16(a.w0, a.ldw0, a.dt) &&
                   (!DUAL || rows16(a.w1, a.ldw1, a.dt));
  // warps per output feature: enough of them for every SM to have 16, as
  // long as each has a full load of its own
  int wpr = 1;
  const int64_t step = 32LL * (vec ? V : 1);
  while (wpr < 8 && a.N * wpr < 16LL * sm_count() && a.K > 2 * step * wpr) wpr *= 2;
  const unsigned grid = static_cast<unsigned>((a.N + 8 / wpr - 1) / (8 / wpr));
  if (vec) k_few_rows<T, MR, DUAL, true><<<grid, 256, 0, s>>>(a, wpr);
  else k_few_rows<T, MR, DUAL, false><<<grid, 256, 0, s>>>(a, wpr);
  CUDA_LAUNCH_CHECK();
}
template <typename T, bool DUAL>
void rows_of(const FewRows &a, cudaStream_t s) {
  if (a.M == 1) launch_rows<T, 1, DUAL>(a, s);
  else if (a.M <= 4) launch_rows<T, 4, DUAL>(a, s);
  else launch_rows<T, kFewRows, DUAL>(a, s);
}

// dz of a linear layer without an activation.
template <typename T>
__global__ void __launch_bounds__(256) k_rows_dz(const FewRows a) {
  const int64_t all = a.M * a.N;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < all; i += static_cast<int64_t>(gridDim.x) * 256) {
    const int64_t m = i / a.N;
    a.dz[i] = a.scale * to_f(static_cast<const T *>(a.in)[m * a.ldin + (i - m * a.N)]);
  }
}

// dW[n][k] = sum over m of dz[m][n] x[m][k]; db[n] = sum of dz[m][n].  Block:
// kStrip features n, 32 V columns k a warp and 8 of those; blockIdx.z: product.
constexpr int kStrip = 16;
template <typename T, bool VEC>
__global__ void __launch_bounds__(256) k_rows_dw(const FewRows a) {
  constexpr int V = VEC ? 16 / static_cast<int>(sizeof(T)) : 1;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  T *dw = static_cast<T *>(blockIdx.z ? a.dw1 : a.dw0);
  T *db = static_cast<T *>(blockIdx.z ? a.db1 : a.db0);
  const int64_t ld = blockIdx.z ? a.lddw1 : a.lddw0;
  const float *dz = a.dz + blockIdx.z * a.M * a.N;
  if (db && blockIdx.x == 0)
    for (int64_t n = static_cast<int64_t>(blockIdx.y) * 256 + threadIdx.x; n < a.N; n += static_cast<int64_t>(gridDim.y) * 256) {
      float t = 0.f;
      for (int m = 0; m < a.M; ++m) t += dz[m * a.N + n];
      db[n] = from_f<T>(t);
    }
  const int64_t k = ((static_cast<int64_t>(blockIdx.x) * 8 + warp) * 32 + lane) * V;
  if (!dw || k >= a.K) return;
  float x[kFewRows][V];
#pragma unroll
  for (int m = 0; m < kFewRows; ++m) {
    const T *p = static_cast<const T *>(a.x) + m * a.ldx + k;
#pragma unroll
    for (int j = 0; j < V; ++j) x[m][j] = 0.f;
    if (m >= a.M) continue;
    if constexpr (VEC) {
      float f[16 / sizeof(T)];
      unpack<T>(__ldg(reinterpret_cast<const uint4 *>(p)), f);
#pragma unroll
      for (int j = 0; j < V; ++j) x[m][j] = f[j];
    } else {
      x[m][0] = to_f(*p);
    }
  }
  for (int64_t n0 = static_cast<int64_t>(blockIdx.y) * kStrip; n0 < a.N; n0 += static_cast<int64_t>(gridDim.y) * kStrip)
  for (int64_t n = n0; n < min(a.N, n0 + kStrip); ++n) {
    float v[VEC ? 16 / sizeof(T) : 1];
#pragma unroll
    for (int j = 0; j < V; ++j) v[j] = 0.f;
#pragma unroll
    for (int m = 0; m < kFewRows; ++m) {
      if (m >= a.M) break;
      const float g = __ldg(dz + m * a.N + n);
#pragma unroll
      for (int j = 0; j < V; ++j) v[j] = fmaf(g, x[m][j], v[j]);
    }
    if constexpr (VEC) *reinterpret_cast<uint4 *>(dw + n * ld + k) = pack<T>(v);
    else dw[n * ld + k] = from_f<T>(v[0]);
  }
}

// part[strip][m][k] = sum over the strip's features n of dz[m][n] W[n][k], over
// both products; a strip of W's rows in eight interleaved shares, one a warp.
template <typename T, bool VEC>
__global__ void __launch_bounds__(256) k_rows_dx(const FewRows a, int64_t strip, float *part) {
  constexpr int V = VEC ? 16 / static_cast<int>(sizeof(T)) : 1;
  __shared__ float sums[8][32 * V];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t k0 = static_cast<int64_t>(blockIdx.x) * 32 * V, k = k0 + lane * V;
  const int64_t n0 = blockIdx.y * strip, n1 = min(a.N, n0 + strip);
  float acc[kFewRows][V];
#pragma unroll
  for (int m = 0; m < kFewRows; ++m)
#pragma unroll
    for (int j = 0; j < V; ++j) acc[m][j] = 0.f;
  for (int q = 0; q < (a.w1 ? 2 : 1); ++q) {
    const T *w = static_cast<const T *>(q ? a.w1 : a.w0) + k;
    const int64_t ld = q ? a.ldw1 : a.ldw0;
    const float *dz = a.dz + q * a.M * a.N;
    if (k < a.K) {
#pragma unroll 4
      for (int64_t n = n0 + warp; n < n1; n += 8) {
        float f[VEC ? 16 / sizeof(T) : 1];
        if constexpr (VEC) unpack<T>(__ldg(reinterpret_cast<const uint4 *>(w + n * ld)), f);
        else f[0] = to_f(w[n * ld]);
#pragma unroll
        for (int m = 0; m < kFewRows; ++m) {
          if (m >= a.M) break;
          const float g = __ldg(dz + m * a.N + n);
#pragma unroll
          for (int j = 0; j < V; ++j) acc[m][j] = fmaf(g, f[j], acc[m][j]);
        }
      }
    }
  }
#pragma unroll
  for (int m = 0; m < kFewRows; ++m) {
    if (m >= a.M) break;
    __syncthreads();
#pragma unroll
    for (int j = 0; j < V; ++j) sums[warp][lane * V + j] = acc[m][j];
    __syncthreads();
    for (int i = threadIdx.x; i < 32 * V; i += 256) {
      if (k0 + i >= a.K) continue;
      float t = 0.f;
#pragma unroll
      for (int w8 = 0; w8 < 8; ++w8) t += sums[w8][i];
      part[(static_cast<int64_t>(blockIdx.y) * a.M + m) * a.K + k0 + i] = t;
    }
  }
}
template <typename T>
__global__ void __launch_bounds__(256) k_rows_join(const FewRows a, int strips, const float *part) {
  const int64_t all = a.M * a.K;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < all; i += static_cast<int64_t>(gridDim.x) * 256) {
    float t = 0.f;
#pragma unroll 8
    for (int s = 0; s < strips; ++s) t += part[s * all + i];
    const int64_t m = i / a.K;
    static_cast<T *>(a.dx)[m * a.lddx + (i - m * a.K)] = from_f<T>(t);
  }
}

// Strips of W's rows for dx: enough blocks for every SM to have four, at least
// 32 rows each.
int dx_strips(const FewRows &a) {
  const int64_t cols = (a.K + 255) / 256;  // blocks of 32 16-byte pieces, about
  return static_cast<int>(std::max<int64_t>(1, std::min<int64_t>((a.N + 31) / 32, (4LL * sm_count() + cols - 1) / cols)));
}

int blocks_for(int64_t threads) {
  return static_cast<int>(std::max<int64_t>(1, std::min<int64_t>((threads + 255) / 256, 8LL * sm_count())));
}

template <typename T>
void bwd_of(const FewRows &a, cudaStream_t s) {
  constexpr int V = 16 / static_cast<int>(sizeof(T));
  if (a.w1 || a.act != ACT_IDENTITY) {
    FewRows z = a;
    z.out = nullptr;
    a.w1 ? rows_of<T, true>(z, s) : rows_of<T, false>(z, s);
  } else {
    k_rows_dz<T><<<blocks_for(a.M * a.N), 256, 0, s>>>(a);
    CUDA_LAUNCH_CHECK();
  }
  if (a.dw0 || a.dw1 || a.db0 || a.db1) {
    const bool vec = a.K % V == 0 && rows16(a.x, a.ldx, a.dt) && (!a.dw0 || rows16(a.dw0, a.lddw0, a.dt)) &&
                     (!a.dw1 || rows16(a.dw1, a.lddw1, a.dt));
    const int64_t span = 256LL * (vec ? V : 1);
    const int64_t strips = (a.N + kStrip - 1) / kStrip;
    const dim3 g(static_cast<unsigned>((a.K + span - 1) / span), static_cast<unsigned>(std::min<int64_t>(strips, 65535)),
                 a.w1 ? 2 : 1);
    if (vec) k_rows_dw<T, true><<<g, 256, 0, s>>>(a);
    else k_rows_dw<T, false><<<g, 256, 0, s>>>(a);
    CUDA_LAUNCH_CHECK();
  }
  if (!a.dx) return;
  const bool vec = a.K % V == 0 && rows16(a.w0, a.ldw0, a.dt) && (!a.w1 || rows16(a.w1, a.ldw1, a.dt));
  const int y = dx_strips(a);
  const int64_t strip = (a.N + y - 1) / y, span = 32LL * (vec ? V : 1);
  float *part = a.dz + (a.w1 ? 2 : 1) * a.M * a.N;
  const dim3 g(static_cast<unsigned>((a.K + span - 1) / span), y);
  if (vec) k_rows_dx<T, true><<<g, 256, 0, s>>>(a, strip, part);
  else k_rows_dx<T, false><<<g, 256, 0, s>>>(a, strip, part);
  CUDA_LAUNCH_CHECK();
  k_rows_join<T><<<blocks_for(a.M * a.K), 256, 0, s>>>(a, y, part);
  CUDA_LAUNCH_CHECK();
}

// Sums of columns over a strip of rows, a fixed share of it per warp.
template <typename T, bool VEC>
__global__ void __launch_bounds__(256) k_column_part(const T *__restrict__ p, int64_t ld, int64_t M, int64_t N,
                                                     int64_t strip, float *part) {
  constexpr int V = VEC ? 16 / static_cast<int>(sizeof(T)) : 1;
  __shared__ float sums[8][32 * V];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t c = (static_cast<int64_t>(blockIdx.x) * 32 + lane) * V;
  const int64_t r0 = blockIdx.y * strip, r1 = min(M, r0 + strip);
  float acc[V];
#pragma unroll
  for (int j = 0; j < V; ++j) acc[j] = 0.f;
  if (c < N) {
#pragma unroll 4
    for (int64_t r = r0 + warp; r < r1; r += 8) {
      if (VEC) {
        float v[16 / sizeof(T)];
        unpack<T>(__ldg(reinterpret_cast<const uint4 *>(p + r * ld + c)), v);
#pragma unroll
        for (int j = 0; j < V; ++j) acc[j] += v[j];
      } else {
        acc[0] += to_f(p[r * ld + c]);
      }
    }
  }
#pragma unroll
  for (int j = 0; j < V; ++j) sums[warp][lane * V + j] = acc[j];
  __syncthreads();
  for (int i = threadIdx.x; i < 32 * V; i += 256) {
    const int64_t col = static_cast<int64_t>(blockIdx.x) * 32 * V + i;
    if (col >= N) continue;
    float t = 0.f;
#pragma unroll
    for (int w = 0; w < 8; ++w) t += sums[w][i];
    part[blockIdx.y * N + col] = t;
  }
}

// Sums rows p, p + stride, .. of each group of kFold into the group's first.
constexpr int kFold = 64;
__global__ void __launch_bounds__(256) k_column_fold(float *part, int64_t P, int64_t stride, int64_t N) {
  __shared__ float sums[8][33];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t c = static_cast<int64_t>(blockIdx.x) * 32 + lane;
  for (int64_t g = blockIdx.y; g * kFold < P; g += gridDim.y) {
    float acc = 0.f;
    if (c < N) {
#pragma unroll
      for (int i = 0; i < kFold / 8; ++i) {
        const int64_t q = g * kFold + i * 8 + warp;
        if (q < P) acc += part[q * stride * N + c];
      }
    }
    __syncthreads();
    sums[warp][lane] = acc;
    __syncthreads();
    if (warp == 0 && c < N) {
      float t = 0.f;
#pragma unroll
      for (int w = 0; w < 8; ++w) t += sums[w][lane];
      part[g * kFold * stride * N + c] = t;
    }
  }
}

// out[c] = scale sum over p < P of part[p stride][c], in 8 interleaved shares.
__global__ void __launch_bounds__(256) k_column_join(const float *__restrict__ part, int64_t P, int64_t stride, int64_t N,
                                                     float scale, void *out, int dt) {
  __shared__ float sums[8][33];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t c = static_cast<int64_t>(blockIdx.x) * 32 + lane;
  float acc = 0.f;
  if (c < N) {
#pragma unroll 8
    for (int64_t q = warp; q < P; q += 8) acc += part[q * stride * N + c];
  }
  sums[warp][lane] = acc;
  __syncthreads();
  if (warp == 0 && c < N) {
    float t = 0.f;
#pragma unroll
    for (int w = 0; w < 8; ++w) t += sums[w][lane];
    store_dt(out, dt, c, t * scale);
  }
}

template <typename T>
void column_parts(const void *p, int dt, int64_t ld, int64_t M, int64_t N, int y, float *part, cudaStream_t s) {
  constexpr int V = 16 / static_cast<int>(sizeof(T));
  const int64_t strip = (M + y - 1) / y;
  const T *t = static_cast<const T *>(p);
  if (N % V == 0 && rows16(p, ld, dt)) {
    const dim3 g(static_cast<unsigned>((N + 32 * V - 1) / (32 * V)), y);
    k_column_part<T, true><<<g, 256, 0, s>>>(t, ld, M, N, strip, part);
  } else {
    const dim3 g(static_cast<unsigned>((N + 31) / 32), y);
    k_column_part<T, false><<<g, 256, 0, s>>>(t, ld, M, N, strip, part);
  }
  CUDA_LAUNCH_CHECK();
}

}  // namespace

void few_rows(const FewRows &a, cudaStream_t s) {
  if (a.dt == DT_F32) a.w1 ? rows_of<float, true>(a, s) : rows_of<float, false>(a, s);
  else if (a.dt == DT_F16) a.w1 ? rows_of<__half, true>(a, s) : rows_of<__half, false>(a, s);
  else a.w1 ? rows_of<__nv_bfloat16, true>(a, s) : rows_of<__nv_bfloat16, false>(a, s);
}

size_t few_rows_floats(const FewRows &a) {
  return static_cast<size_t>(a.M) * ((a.w1 ? 2 : 1) * a.N + dx_strips(a) * a.K);
}

void few_rows_bwd(const FewRows &a, cudaStream_t s) {
  if (a.dt == DT_F32) bwd_of<float>(a, s);
  else if (a.dt == DT_F16) bwd_of<__half>(a, s);
  else bwd_of<__nv_bfloat16>(a, s);
}

int column_strips(int64_t M) { return static_cast<int>(std::min<int64_t>(128, (M + 63) / 64)); }

void column_join(float *part, int64_t P, int64_t N, float scale, void *out, int dt, cudaStream_t s) {
  const unsigned gx = static_cast<unsigned>((N + 31) / 32);
  int64_t stride = 1;
  for (; P > 2 * kFold; P = (P + kFold - 1) / kFold, stride *= kFold) {
    k_column_fold<<<dim3(gx, static_cast<unsigned>(std::min<int64_t>((P + kFold - 1) / kFold, 65535))), 256, 0, s>>>(
        part, P, stride, N);
    CUDA_LAUNCH_CHECK();
  }
  k_column_join<<<gx, 256, 0, s>>>(part, P, stride, N, scale, out, dt);
  CUDA_LAUNCH_CHECK();
}

void column_sums(const void *p, int dt, int64_t ld, int64_t M, int64_t N, float *part, cudaStream_t s) {
  const int y = column_strips(M);
  if (dt == DT_F16) column_parts<__half>(p, dt, ld, M, N, y, part, s);
  else column_parts<__nv_bfloat16>(p, dt, ld, M, N, y, part, s);
}

}  // namespace blk
}  // namespace pet
