// Transformer-block operators for a handful of rows (single tokens), and the
// column sums of the bias gradients.
//
// With a handful of rows a dense layer is the time it takes to read the weights
// once, so everything is arranged around 16-byte weight loads, several in flight
// per lane.
//
//  * 16-bit: one CTA per 16 output features, its eight warps along K.  A warp
//    multiplies a 16 x 16 piece of the weight with up to 8 (16) rows of x by one
//    (two) mma.sync: a lane's 16 bytes of a weight row and of a row of x are the
//    fragments as they come, with the contraction index permuted alike on both
//    sides.  With FMAs the same loads cost 130 instructions for 32 bytes of
//    weight at 8 rows, and took 33 us where this takes 11 (two 5632 x 2048
//    weights); a tcgen05 tile of 128 rows took 18.
//  * f32, and rows that are not 16-byte aligned: one to eight warps per output
//    feature, fp32 FMAs.  Every feature's warp reads all of x, so the same two
//    weights in f32 take 16, 31 and 61 us at 1, 4 and 8 rows (bytes alone: 14).
//
// The backward of so few rows is the same for the weights (read once for dz,
// once for dx, and their gradients written once): dz in fp32 by the forward's
// kernels, dW = dz^T x and db as one pass of stores, dx = dz W in strips of W's
// rows whose fp32 sums a last kernel adds in order.
#include <algorithm>
#include <type_traits>

#include "block.cuh"

namespace pet {
namespace blk {

namespace {

constexpr int kDepth = 4;  // loads in flight per lane and weight (8 cost more in resident warps)

// The epilogue of one result: row m, feature n, both products, the first with its
// bias.  dz of a backward goes out as [product][feature][8 rows], the rows past M
// zeros.
constexpr int kRowPad = 8;
template <typename T, bool DUAL>
__device__ __forceinline__ void finish(const FewRows &a, int m, int64_t n, float v, float w) {
  if (DUAL && a.b1) w += to_f(static_cast<const T *>(a.b1)[n]);
  const float in = a.in ? to_f(static_cast<const T *>(a.in)[m * a.ldin + n]) : 0.f;
  float da;
  with_act(a.act, [&](auto A) { act_pair<decltype(A)::value>(v, v, da); });
  if (a.out) {
    if (DUAL) v *= w;
    else v = v * a.scale + in;
    static_cast<T *>(a.out)[m * a.ldo + n] = from_f<T>(v);
  } else {
    a.dz[n * kRowPad + m] = DUAL ? da * w * in : da * a.scale * in;
    if (DUAL) a.dz[(a.N + n) * kRowPad + m] = v * in;
  }
}

__device__ __forceinline__ NearZero near_of(const FewRows &a) { return {a.x, a.w0, a.b0, a.ldx, a.ldw0, a.K}; }

// D += A B with A 16 x 16 (four registers a lane), B 16 x 8 (two).
template <typename T>
__device__ __forceinline__ void mma16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                      uint32_t b1) {
  if constexpr (std::is_same<T, __half>::value)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// 16-bit rows, 16-byte aligned, K a multiple of 8; M <= 8 NT.  Lane (g, t) of a
// warp holds weight rows g and g + 8 and rows g (and g + 8) of x, eight elements
// at 8 t of each 32: two MMAs, of its first and its last four.
template <typename T, int NT, bool DUAL>
__global__ void __launch_bounds__(256) k_few_mma(const FewRows a) {
  constexpr int NP = DUAL ? 2 : 1;
  constexpr int U = DUAL || NT > 1 ? 2 : 4;  // 32-element steps in flight
  __shared__ float part[8][NP][NT][16 * 8];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int64_t n0 = static_cast<int64_t>(blockIdx.x) * 16;
  const T *w[NP][2], *x[NT];
#pragma unroll
  for (int q = 0; q < NP; ++q)
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const int64_t n = min(n0 + g + 8 * r, a.N - 1);  // (rows past N are computed and not stored)
      w[q][r] = static_cast<const T *>(q ? a.w1 : a.w0) + n * (q ? a.ldw1 : a.ldw0);
    }
#pragma unroll
  for (int i = 0; i < NT; ++i) x[i] = g + 8 * i < a.M ? static_cast<const T *>(a.x) + (g + 8 * i) * a.ldx : nullptr;
  float d[NP][NT][4];
#pragma unroll
  for (int q = 0; q < NP; ++q)
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) d[q][i][j] = 0.f;
  for (int64_t k0 = warp * 32 + t * 8; k0 - t * 8 < a.K; k0 += U * 256) {
    uint4 wr[U][NP][2], xr[U][NT];
    const uint4 zero = make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t k = k0 + u * 256;
      const bool in = k < a.K;
#pragma unroll
      for (int q = 0; q < NP; ++q)
#pragma unroll
        for (int r = 0; r < 2; ++r) wr[u][q][r] = in ? __ldg(reinterpret_cast<const uint4 *>(w[q][r] + k)) : zero;
#pragma unroll
      for (int i = 0; i < NT; ++i) xr[u][i] = in && x[i] ? __ldg(reinterpret_cast<const uint4 *>(x[i] + k)) : zero;
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int q = 0; q < NP; ++q)
#pragma unroll
        for (int i = 0; i < NT; ++i) {
          mma16<T>(d[q][i], wr[u][q][0].x, wr[u][q][1].x, wr[u][q][0].y, wr[u][q][1].y, xr[u][i].x, xr[u][i].y);
          mma16<T>(d[q][i], wr[u][q][0].z, wr[u][q][1].z, wr[u][q][0].w, wr[u][q][1].w, xr[u][i].z, xr[u][i].w);
        }
  }
  // d[.][i][j]: feature g + 8 (j / 2), row 8 i + 2 t + j % 2; the warps' shares
  // are added in order
#pragma unroll
  for (int q = 0; q < NP; ++q)
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) part[warp][q][i][(2 * t + j % 2) * 16 + g + 8 * (j / 2)] = d[q][i][j];
  __syncthreads();
  for (int i = threadIdx.x; i < NT * 128; i += 256) {  // (whole warps)
    const int m = i / 16;
    const int64_t n = n0 + i % 16;
    const bool there = n < a.N && m < a.M;
    if (n < a.N && m >= a.M && !a.out && m < kRowPad) {
      a.dz[n * kRowPad + m] = 0.f;
      if (DUAL) a.dz[(a.N + n) * kRowPad + m] = 0.f;
    }
    float v[2] = {0.f, 0.f}, top = 0.f;
#pragma unroll
    for (int q = 0; q < NP; ++q)
#pragma unroll
      for (int s = 0; s < 8; ++s) {
        const float t = part[s][q][m / 8][(m % 8) * 16 + i % 16];
        v[q] += t;
        if (q == 0) top = fmaxf(top, fabsf(t));
      }
    if (there && a.b0) v[0] += to_f(static_cast<const T *>(a.b0)[n]);
    if (!a.out && a.act == ACT_RELU)
      v[0] = settled_row<T>(near_of(a), there, warp_max(there ? top : 0.f) * kNear, m, n, v[0], lane);
    if (there) finish<T, DUAL>(a, m, n, v[0], v[1]);
  }
}

template <typename T, int MR, bool DUAL, bool VEC>
__global__ void __launch_bounds__(256) k_few_rows(const FewRows a, int wpr) {
  constexpr int V = VEC ? 16 / static_cast<int>(sizeof(T)) : 1;
  constexpr int NS = DUAL ? 2 * MR : MR;
  __shared__ float part[8][NS];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t n = static_cast<int64_t>(blockIdx.x) * (8 / wpr) + warp / wpr;
  const int sub = warp % wpr;
  // sums of even and of odd elements (VEC): two to an instruction
  float2 pair[NS];
#pragma unroll
  for (int i = 0; i < NS; ++i) pair[i] = make_float2(0.f, 0.f);
  constexpr int D1 = DUAL ? MR : 0;  // the second product's sums
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
            for (int j = 0; j + 1 < V; j += 2) {
              const float2 x2 = make_float2(xv[j], xv[j + 1]);
              pair[m] = __ffma2_rn(x2, make_float2(f0[j], f0[j + 1]), pair[m]);
              if (DUAL) pair[D1 + m] = __ffma2_rn(x2, make_float2(f1[j], f1[j + 1]), pair[D1 + m]);
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
            pair[m].x = fmaf(xv, f0, pair[m].x);
            if (DUAL) pair[D1 + m].x = fmaf(xv, f1, pair[D1 + m].x);
          }
        }
      }
    }
  }
  float sum[NS];
#pragma unroll
  for (int i = 0; i < NS; ++i) sum[i] = warp_sum(pair[i].x + pair[i].y);
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
      if (DUAL) w = sum[D1 + m];
    }
  if (n >= a.N) return;
  if (!a.out && lane >= a.M && lane < kRowPad) {
    a.dz[n * kRowPad + lane] = 0.f;
    if (DUAL) a.dz[(a.N + n) * kRowPad + lane] = 0.f;
  }
  if (a.b0) v += to_f(static_cast<const T *>(a.b0)[n]);
  if (!a.out && a.act == ACT_RELU) {
    // the partial sums of this warp's lanes stand for those of all
    float top = 0.f;
#pragma unroll
    for (int m = 0; m < MR; ++m) top = fmaxf(top, fmaxf(fabsf(pair[m].x), fabsf(pair[m].y)));
    v = settled_row<T>(near_of(a), lane < a.M, warp_max(top) * kNear, lane, n, v, lane, kFewRows);
  }
  if (lane >= a.M) return;
  finish<T, DUAL>(a, lane, n, v, w);
}

// (K: as in the tiled products, the truncations of one of the eight warps' sums,
// 2^-23 for each 16 terms, must not pass half a rounding of the result)
bool few_mma(const FewRows &a) {
  return a.dt != DT_F32 && a.K % 8 == 0 && a.K <= (a.dt == DT_F16 ? 262144 : 2097152) && rows16(a.x, a.ldx, a.dt) &&
         rows16(a.w0, a.ldw0, a.dt) && (!a.w1 || rows16(a.w1, a.ldw1, a.dt));
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
  if constexpr (sizeof(T) == 2) {
    if (few_mma(a)) {
      const unsigned grid = static_cast<unsigned>((a.N + 15) / 16);
      if (a.M <= 8) k_few_mma<T, 1, DUAL><<<grid, 256, 0, s>>>(a);
      else k_few_mma<T, 2, DUAL><<<grid, 256, 0, s>>>(a);
      CUDA_LAUNCH_CHECK();
      return;
    }
  }
  if (a.M == 1) launch_rows<T, 1, DUAL>(a, s);
  else if (a.M <= 4) launch_rows<T, 4, DUAL>(a, s);
  else launch_rows<T, kFewRows, DUAL>(a, s);
}

// dz of feature n: the first MR rows.
template <int MR>
__device__ __forceinline__ void load_dz(const float *dz, int64_t n, float (&z)[MR]) {
  if constexpr (MR == 1) {
    z[0] = __ldg(dz + n * kRowPad);
  } else {
#pragma unroll
    for (int m = 0; m < MR; m += 4) {
      const float4 a = __ldg(reinterpret_cast<const float4 *>(dz + n * kRowPad + m));
      z[m] = a.x;
      z[m + 1] = a.y;
      z[m + 2] = a.z;
      z[m + 3] = a.w;
    }
  }
}

// dz of a linear layer without an activation.
template <typename T>
__global__ void __launch_bounds__(256) k_rows_dz(const FewRows a) {
  const int64_t all = kRowPad * a.N;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < all; i += static_cast<int64_t>(gridDim.x) * 256) {
    const int64_t n = i / kRowPad, m = i % kRowPad;
    a.dz[i] = m < a.M ? a.scale * to_f(static_cast<const T *>(a.in)[m * a.ldin + n]) : 0.f;
  }
}

// dW[n][k] = sum over m of dz[m][n] x[m][k]; db[n] = sum of dz[m][n].  Block:
// kStrip features n, 32 V columns k a warp and 8 of those; blockIdx.z: product.
constexpr int kStrip = 16;
template <typename T, int MR, bool VEC>
__global__ void __launch_bounds__(256) k_rows_dw(const FewRows a) {
  constexpr int V = VEC ? 16 / static_cast<int>(sizeof(T)) : 1;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  T *dw = static_cast<T *>(blockIdx.z ? a.dw1 : a.dw0);
  T *db = static_cast<T *>(blockIdx.z ? a.db1 : a.db0);
  const int64_t ld = blockIdx.z ? a.lddw1 : a.lddw0;
  const float *dz = a.dz + blockIdx.z * a.N * kRowPad;
  if (db && blockIdx.x == 0)
    for (int64_t n = static_cast<int64_t>(blockIdx.y) * 256 + threadIdx.x; n < a.N; n += static_cast<int64_t>(gridDim.y) * 256) {
      float t = 0.f;
      for (int m = 0; m < a.M; ++m) t += dz[n * kRowPad + m];
      db[n] = from_f<T>(t);
    }
  const int64_t k = ((static_cast<int64_t>(blockIdx.x) * 8 + warp) * 32 + lane) * V;
  if (!dw || k >= a.K) return;
  constexpr int P = V > 1 ? V / 2 : 1;  // pairs of columns (V = 1: .y unused)
  float2 x[MR][P];
#pragma unroll
  for (int m = 0; m < MR; ++m) {
#pragma unroll
    for (int j = 0; j < P; ++j) x[m][j] = make_float2(0.f, 0.f);
    if (m >= a.M) continue;
    const T *p = static_cast<const T *>(a.x) + m * a.ldx + k;
    if constexpr (VEC) {
      float f[16 / sizeof(T)];
      unpack<T>(__ldg(reinterpret_cast<const uint4 *>(p)), f);
#pragma unroll
      for (int j = 0; j < P; ++j) x[m][j] = make_float2(f[2 * j], f[2 * j + 1]);
    } else {
      x[m][0].x = to_f(*p);
    }
  }
  for (int64_t s0 = static_cast<int64_t>(blockIdx.y) * kStrip; s0 < a.N; s0 += static_cast<int64_t>(gridDim.y) * kStrip) {
    const int64_t s1 = min(a.N, s0 + kStrip);
#pragma unroll 4
    for (int64_t n = s0; n < s1; ++n) {
      float z[MR];
      load_dz<MR>(dz, n, z);
      float2 v[P];
#pragma unroll
      for (int j = 0; j < P; ++j) v[j] = make_float2(0.f, 0.f);
#pragma unroll
      for (int m = 0; m < MR; ++m)
#pragma unroll
        for (int j = 0; j < P; ++j) v[j] = __ffma2_rn(make_float2(z[m], z[m]), x[m][j], v[j]);
      if constexpr (VEC) {
        float f[16 / sizeof(T)];
#pragma unroll
        for (int j = 0; j < P; ++j) {
          f[2 * j] = v[j].x;
          f[2 * j + 1] = v[j].y;
        }
        *reinterpret_cast<uint4 *>(dw + n * ld + k) = pack<T>(f);
      } else {
        dw[n * ld + k] = from_f<T>(v[0].x);
      }
    }
  }
}

// part[strip][m][k] = sum over the strip's features n of dz[m][n] W[n][k], over
// both products; a strip of W's rows in eight interleaved shares, one a warp.
template <typename T, int MR, bool VEC>
__global__ void __launch_bounds__(256, 2) k_rows_dx(const FewRows a, int64_t strip, float *part) {
  constexpr int V = VEC ? 16 / static_cast<int>(sizeof(T)) : 1;
  __shared__ float sums[8][32 * V];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t k0 = static_cast<int64_t>(blockIdx.x) * 32 * V, k = k0 + lane * V;
  const int64_t n0 = blockIdx.y * strip, n1 = min(a.N, n0 + strip);
  constexpr int P = V > 1 ? V / 2 : 1;
  float2 acc[MR][P];
#pragma unroll
  for (int m = 0; m < MR; ++m)
#pragma unroll
    for (int j = 0; j < P; ++j) acc[m][j] = make_float2(0.f, 0.f);
  for (int q = 0; q < (a.w1 ? 2 : 1); ++q) {
    const T *w = static_cast<const T *>(q ? a.w1 : a.w0) + k;
    const int64_t ld = q ? a.ldw1 : a.ldw0;
    const float *dz = a.dz + q * a.N * kRowPad;
    if (k < a.K) {
#pragma unroll 4
      for (int64_t n = n0 + warp; n < n1; n += 8) {
        float2 f[P];
        if constexpr (VEC) {
          float u[16 / sizeof(T)];
          unpack<T>(__ldg(reinterpret_cast<const uint4 *>(w + n * ld)), u);
#pragma unroll
          for (int j = 0; j < P; ++j) f[j] = make_float2(u[2 * j], u[2 * j + 1]);
        } else {
          f[0] = make_float2(to_f(w[n * ld]), 0.f);
        }
        float z[MR];
        load_dz<MR>(dz, n, z);
#pragma unroll
        for (int m = 0; m < MR; ++m)
#pragma unroll
          for (int j = 0; j < P; ++j) acc[m][j] = __ffma2_rn(make_float2(z[m], z[m]), f[j], acc[m][j]);
      }
    }
  }
#pragma unroll
  for (int m = 0; m < MR; ++m) {
    if (m >= a.M) break;
    __syncthreads();
#pragma unroll
    for (int j = 0; j < V; ++j) sums[warp][lane * V + j] = j % 2 ? acc[m][j / 2].y : acc[m][j / 2].x;
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
// dx from the strips' sums, in 32 interleaved shares; block: 32 elements.
template <typename T>
__global__ void __launch_bounds__(1024) k_rows_join(const FewRows a, int strips, const float *part) {
  __shared__ float sums[32][33];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t all = a.M * a.K;
  for (int64_t i0 = static_cast<int64_t>(blockIdx.x) * 32; i0 < all; i0 += static_cast<int64_t>(gridDim.x) * 32) {
    const int64_t i = i0 + lane;
    float t = 0.f;
    if (i < all)
      for (int s = warp; s < strips; s += 32) t += part[s * all + i];
    __syncthreads();
    sums[warp][lane] = t;
    __syncthreads();
    // row `warp` of the transpose: the shares of one element
    t = warp_sum(sums[lane][warp]);
    const int64_t o = i0 + warp, m = o / a.K;
    if (lane == 0 && o < all) static_cast<T *>(a.dx)[m * a.lddx + (o - m * a.K)] = from_f<T>(t);
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

template <typename T, int MR>
void bwd_of(const FewRows &a, cudaStream_t s) {
  constexpr int V = 16 / static_cast<int>(sizeof(T));
  if (a.w1 || a.act != ACT_IDENTITY) {
    FewRows z = a;
    z.out = nullptr;
    a.w1 ? rows_of<T, true>(z, s) : rows_of<T, false>(z, s);
  } else {
    k_rows_dz<T><<<blocks_for(kRowPad * a.N), 256, 0, s>>>(a);
    CUDA_LAUNCH_CHECK();
  }
  if (a.dw0 || a.dw1 || a.db0 || a.db1) {
    const bool vec = a.K % V == 0 && rows16(a.x, a.ldx, a.dt) && (!a.dw0 || rows16(a.dw0, a.lddw0, a.dt)) &&
                     (!a.dw1 || rows16(a.dw1, a.lddw1, a.dt));
    const int64_t span = 256LL * (vec ? V : 1);
    const int64_t strips = (a.N + kStrip - 1) / kStrip;
    const dim3 g(static_cast<unsigned>((a.K + span - 1) / span), static_cast<unsigned>(std::min<int64_t>(strips, 65535)),
                 a.w1 ? 2 : 1);
    if (vec) k_rows_dw<T, MR, true><<<g, 256, 0, s>>>(a);
    else k_rows_dw<T, MR, false><<<g, 256, 0, s>>>(a);
    CUDA_LAUNCH_CHECK();
  }
  if (!a.dx) return;
  const bool vec = a.K % V == 0 && rows16(a.w0, a.ldw0, a.dt) && (!a.w1 || rows16(a.w1, a.ldw1, a.dt));
  const int y = dx_strips(a);
  const int64_t strip = (a.N + y - 1) / y, span = 32LL * (vec ? V : 1);
  float *part = a.dz + (a.w1 ? 2 : 1) * a.N * kRowPad;
  const dim3 g(static_cast<unsigned>((a.K + span - 1) / span), y);
  if (vec) k_rows_dx<T, MR, true><<<g, 256, 0, s>>>(a, strip, part);
  else k_rows_dx<T, MR, false><<<g, 256, 0, s>>>(a, strip, part);
  CUDA_LAUNCH_CHECK();
  k_rows_join<T><<<static_cast<unsigned>(std::min<int64_t>((a.M * a.K + 31) / 32, 16LL * sm_count())), 1024, 0, s>>>(a, y, part);
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

bool few_rows_fit(const FewRows &a) { return a.M <= (few_mma(a) ? 16 : kFewRows); }

void few_rows(const FewRows &a, cudaStream_t s) {
  if (a.dt == DT_F32) a.w1 ? rows_of<float, true>(a, s) : rows_of<float, false>(a, s);
  else if (a.dt == DT_F16) a.w1 ? rows_of<__half, true>(a, s) : rows_of<__half, false>(a, s);
  else a.w1 ? rows_of<__nv_bfloat16, true>(a, s) : rows_of<__nv_bfloat16, false>(a, s);
}

size_t few_rows_floats(const FewRows &a) {
  return static_cast<size_t>(a.w1 ? 2 : 1) * a.N * kRowPad + static_cast<size_t>(a.M) * dx_strips(a) * a.K;
}

void few_rows_bwd(const FewRows &a, cudaStream_t s) {
  auto go = [&](auto tag) {
    using T = decltype(tag);
    if (a.M == 1) bwd_of<T, 1>(a, s);
    else if (a.M <= 4) bwd_of<T, 4>(a, s);
    else bwd_of<T, kRowPad>(a, s);
  };
  if (a.dt == DT_F32) go(float{});
  else if (a.dt == DT_F16) go(__half{});
  else go(__nv_bfloat16{});
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
