// Dense products of the transformer-block operators on the 5th-generation
// tensor cores: C = A B^T with fused epilogues, for f16 / bf16 operands read
// where they lie and for f32 operands in split-fp16 form.
//
// One persistent CTA per SM, ten warps: a TMA producer, an MMA issuer and
// eight accumulator warps.  A stage holds 64 contraction elements of 128 rows
// of A and BN rows of B in the 128-byte-swizzled layout that the MMA reads.
// Either operand may be stored with its contraction contiguous (K-major) or
// with its rows contiguous (MN-major, for the products that contract over
// tokens or over a weight's output features), so that no product of a
// backward pass needs a transposed copy.
//
//  * 16-bit: one kind::f16 product, fp32 accumulation in tensor memory over
//    the whole contraction (divided where its truncations could show, see
//    run); BN = 256 (one 128 x 256 tile, two accumulators) or 128 (four
//    accumulators) when 256-wide tiles would leave SMs idle.
//  * f32: A = 2^-s (hi + lo) and B = 2^-t (hi + lo) with one scale per row (the
//    output's row or column) and 128 contraction elements (one for all of a
//    model's weight, split when it was loaded) in the way of split16.cuh;
//    A_lo B_hi + A_hi B_lo + A_hi B_hi per step.  With one scale per 128 x
//    128 block of B, features 2^-36 below their block's largest were a quarter
//    off; the scales per column cost 0.5 to 3% of a call of 65,202 rows.  The
//    tensor core truncates when it adds to its accumulator, so every 128
//    contraction elements the accumulator warps add the partial sum to fp32
//    registers with round-to-nearest.
//
// Pairs (16-bit): where there are enough rows, two SMs take a tile of 256 x 256
// together (cta_group::2).  Each loads its own 128 rows of A and half of B's
// rows, the leader issues M = 256 MMAs that read both halves and leave each SM
// its own rows' accumulator: a third fewer bytes in and out of shared memory
// for a product.
//
// Forms of a launch: `dual` (the gated projections: a tile's accumulator
// holds BN / 2 columns of x Wg^T beside the same columns of x Wv^T, so the
// epilogue has both in one thread), `kcat` (two pairs of operands along the
// contraction: dx = dg Wg + dv Wv), `batch2` (two products that share a
// shape: dWg = dg^T x, dWv = dv^T x) and `splits` (the contraction divided
// over CTAs, partial sums to the workspace and a second kernel that adds them
// in order and runs the epilogue, for outputs of few tiles).
//
// What bounds it: 16-bit, 8192 x 1024 x 8192 bf16 in 99 us (1.39 PFLOP/s, 72% of
// the tensor pipe): 128 pair tiles in two waves of 74.  With the gated backward's
// epilogue (two outputs, an input and the activation for every two columns) the
// same work takes 129 us.  f32: 128 x 128 tiles read 128 bytes of shared memory a
// cycle for the MMAs and write 85 more by TMA, so 65,202 x 512 x 2048 takes 365 us
// (59% of the pipe, 375 TFLOP/s of fp32-accurate products).
//
// Every wait is bounded; on expiry the CTA records an error, waits for its
// own loads and MMAs, frees its tensor memory and returns.
#include <cuda.h>
#include <cudaTypedefs.h>

#include <algorithm>
#include <cstring>
#include <map>
#include <mutex>
#include <utility>

#include "block.cuh"
#include "split16.cuh"
#include "tc_common.cuh"

namespace pet {

using namespace tc;

namespace blk {

namespace {

constexpr int BM = 128, BK = 64;
constexpr int kTile = BM * 128;  // bytes of 128 rows x 64 16-bit elements

constexpr int kAccWarps = 8;  // two per quarter of the tensor-memory lanes
constexpr int kThreads = 64 + 32 * kAccWarps;
constexpr int kStageFloats = 32 * 32;  // turning block of one accumulator warp

// (E_RELU beside E_*_BWD: a variant that settles the sign of z near 0, whose
// registers cost the other activations' launches 2 to 9%)
enum Epi : int { E_LINEAR = 0, E_LINEAR_BWD = 1, E_GATED = 2, E_GATED_BWD = 3, E_PARTIAL = 4, E_RELU = 8 };

// MODE: 16-bit operands (one product, planes = 1) or split-fp16 (planes = 2).
template <bool F32, int BN, bool PAIR>
struct Cfg {
  static constexpr int Planes = F32 ? 2 : 1;
  static constexpr int BRows = PAIR ? BN / 2 : BN;  // rows of B that one CTA loads
  static constexpr int BTile = BRows * 128;
  static constexpr int StageBytes = Planes * (kTile + BTile);
  static constexpr int Stages = 192 * 1024 / StageBytes;

  static constexpr int Bufs = 512 / BN;
  static constexpr int Chunk = F32 ? 2 : 1 << 30;  // k tiles per accumulator pass
  static constexpr int BarBytes = 256;
  static constexpr int Smem = 1024 + Stages * StageBytes + kAccWarps * kStageFloats * 4 + BarBytes;
};
static_assert(Cfg<false, 256, false>::Smem <= 232448 && Cfg<false, 128, false>::Smem <= 232448 &&
                  Cfg<true, 128, false>::Smem <= 232448 && Cfg<false, 256, true>::Smem <= 232448,
              "shared memory of one CTA");

struct EpiArgs {
  const void *b0, *b1;    // biases
  const void *in;         // residual (E_LINEAR) or upstream gradient (E_*_BWD)
  int64_t ldin;
  void *out0, *out1;      // out1: E_GATED_BWD's dv, batch2's second product
  int64_t ldo;
  int act;
  float scale;
  float *sums0, *sums1;   // E_*_BWD, or null: column sums of each 32 rows of the
                          // results before they are rounded, [row / 32][N]
  NearZero near;          // E_*_BWD of a ReLU: what z (the gate) comes from (x null: not asked for)
  bool vin, vout;         // rows movable in 16-byte pieces
  float *part;            // E_PARTIAL: [batch][split][M][nacc]
  int64_t nacc;
};

struct Params {
  int M, N;                        // output rows and columns (dual: of each half)
  int kt0, kt;                     // k tiles of the first pair of operands, of all
  int tiles_m, tiles_n, splits, kt_split, batch;
  int a_mn, b_mn, dual, bf16, products;
  int *err;                        // error word, or null for the file's own
  // f32: scales 2^-s, the upper halves of the floats, of A [block][row] and of
  // B [block][column] (or null: one pair of them)
  const uint16_t *sc[2], *bs[2];
  int64_t scld[2], bsld[2];
  uint16_t bsc[2];
  EpiArgs e;
};

struct Maps {
  CUtensorMap a[2], b[2];
};

__device__ int g_block_err = 0;

// One thread of the warp, in the form that lets the compiler keep what it
// issues to the tensor core and to TMA in uniform registers (a test of the
// lane left the MMA issue, not the MMAs, as the limit: 60 against 68 us for
// 8192 x 4096 x 1024 in bf16).
__device__ __forceinline__ bool elect_one() {
  uint32_t e;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(e));
  return e != 0;
}

__device__ __forceinline__ void tma3(uint32_t dst, const CUtensorMap *map, uint32_t bar, int x, int y, int z) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
      ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(x), "r"(y), "r"(z)
      : "memory");
}
// into this CTA's shared memory, completing on a barrier of the pair's leader
__device__ __forceinline__ void tma3_pair(uint32_t dst, const CUtensorMap *map, uint32_t bar, int x, int y, int z) {
  asm volatile(
      "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
      ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(x), "r"(y), "r"(z)
      : "memory");
}
__device__ __forceinline__ void expect_tx(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}

// One tile's coordinates from its number: groups of 8 row tiles, columns
// outer and rows inner within a group, so that the CTAs at work at one time
// share both operands' tiles in L2.
struct Item {
  int batch, split, tm, tn;
};
__device__ __forceinline__ Item item_of(const Params &p, int it) {
  Item o;
  const int tiles = p.tiles_m * p.tiles_n;
  o.batch = it / (tiles * p.splits);
  it -= o.batch * tiles * p.splits;
  o.split = it / tiles;
  it -= o.split * tiles;
  const int per = 8 * p.tiles_n, g = it / per, r = it - g * per;
  const int gm = min(8, p.tiles_m - 8 * g);
  o.tn = r / gm;
  o.tm = 8 * g + r - o.tn * gm;
  return o;
}

// One warp's 32 x 32 block of a tile, read from tensor memory a row a lane,
// is turned through shared memory to the layout of its loads and stores: a
// lane has V consecutive columns (16 bytes of T) of row i * 32 / L + lane / L,
// i < L.  16-byte piece k of row r lies at place k ^ (r % 8), which keeps both
// accesses free of bank conflicts.
template <typename T>
struct Turned {
  static constexpr int V = 16 / static_cast<int>(sizeof(T)), L = 32 / V;
  float x[L][V];
  static __device__ __forceinline__ float4 *piece(float *st, int r, int k) {
    return reinterpret_cast<float4 *>(st + r * 32 + ((k ^ (r & 7)) << 2));
  }
  static __device__ __forceinline__ int row(int i, int lane) { return i * (32 / L) + lane / L; }
  static __device__ __forceinline__ int col(int lane) { return (lane % L) * V; }
  __device__ __forceinline__ void turn(float *st, int lane, const float (&v)[32]) {
    __syncwarp();  // the block before has been read
#pragma unroll
    for (int j = 0; j < 32; j += 4)
      *piece(st, lane, j / 4) = make_float4(v[j], v[j + 1], v[j + 2], v[j + 3]);
    __syncwarp();
#pragma unroll
    for (int i = 0; i < L; ++i)
#pragma unroll
      for (int j = 0; j < V; j += 4) {
        const float4 u = *piece(st, row(i, lane), (col(lane) + j) / 4);
        x[i][j] = u.x;
        x[i][j + 1] = u.y;
        x[i][j + 2] = u.z;
        x[i][j + 3] = u.w;
      }
  }
  // V elements of a bias from column c on, zeros past N
  static __device__ __forceinline__ void bias(const void *p, int c, int N, float (&b)[V]) {
    const T *q = static_cast<const T *>(p) + c;
#pragma unroll
    for (int j = 0; j < V; ++j) b[j] = c + j < N ? to_f(__ldg(q + j)) : 0.f;
  }
};

// The block's elements of the epilogue's input (residual or upstream
// gradient), requested ahead of the accumulator they are combined with.
template <typename T>
struct Input {
  using U = Turned<T>;
  uint4 v[U::L];
  __device__ __forceinline__ void fetch(const Params &p, int lane, int row0, int col0) {
    const T *in = static_cast<const T *>(p.e.in);
    const int c = col0 + U::col(lane);
#pragma unroll
    for (int i = 0; i < U::L; ++i) {
      const int r = row0 + U::row(i, lane);
      v[i] = make_uint4(0u, 0u, 0u, 0u);
      if (r >= p.M || c >= p.N) continue;
      const T *q = in + static_cast<size_t>(r) * p.e.ldin + c;  // (`in` may be `out`: no read-only loads)
      if (p.e.vin && c + U::V <= p.N) {
        v[i] = *reinterpret_cast<const uint4 *>(q);
      } else {
        T *t = reinterpret_cast<T *>(&v[i]);
#pragma unroll
        for (int j = 0; j < U::V; ++j)
          if (c + j < p.N) t[j] = q[j];
      }
    }
  }
};

// Rows that are not 16-byte aligned go out a row at a time, a column a lane,
// after another turn through `st`.
template <typename T>
__device__ __forceinline__ void block_store(const Turned<T> &b, T *out, int64_t ldo, bool vec, float *st, int lane,
                                            int row0, int col0, int M, int N) {
  using U = Turned<T>;
  const int c = col0 + U::col(lane);
  if (!vec) {
    __syncwarp();
#pragma unroll
    for (int i = 0; i < U::L; ++i)
#pragma unroll
      for (int j = 0; j < U::V; j += 4)
        *U::piece(st, U::row(i, lane), (U::col(lane) + j) / 4) =
            make_float4(b.x[i][j], b.x[i][j + 1], b.x[i][j + 2], b.x[i][j + 3]);
    __syncwarp();
    if (col0 + lane < N)
      for (int r = 0; r < 32 && row0 + r < M; ++r)
        out[static_cast<size_t>(row0 + r) * ldo + col0 + lane] =
            from_f<T>(reinterpret_cast<const float *>(U::piece(st, r, lane / 4))[lane % 4]);
    return;
  }
#pragma unroll
  for (int i = 0; i < U::L; ++i) {
    const int r = row0 + U::row(i, lane);
    if (r >= M || c >= N) continue;
    T *q = out + static_cast<size_t>(r) * ldo + c;
    if (c + U::V <= N) {
      *reinterpret_cast<uint4 *>(q) = pack<T>(b.x[i]);
    } else {
#pragma unroll
      for (int j = 0; j < U::V; ++j)
        if (c + j < N) q[j] = from_f<T>(b.x[i][j]);
    }
  }
}

// Sums of the block's columns (bias gradients), in a fixed order: rows past M
// are zeros.
template <typename T>
__device__ __forceinline__ void block_sums(const Turned<T> &b, float *sums, int lane, int row0, int col0, int N) {
  using U = Turned<T>;
  float s[U::V];
#pragma unroll
  for (int j = 0; j < U::V; ++j) {
    s[j] = b.x[0][j];
#pragma unroll
    for (int i = 1; i < U::L; ++i) s[j] += b.x[i][j];
#pragma unroll
    for (int k = U::L; k < 32; k *= 2) s[j] += __shfl_xor_sync(0xffffffffu, s[j], k);
  }
  const int c = col0 + U::col(lane);
  if (lane >= U::L) return;
#pragma unroll
  for (int j = 0; j < U::V; ++j)
    if (c + j < N) sums[static_cast<size_t>(row0 / 32) * N + c + j] = s[j];
}

// The epilogue of one block: v (and w, the value half of the gated forms) as
// they come from the accumulator, `in` from the rows' input.
template <int EPI, bool RELU, typename T>
__device__ __forceinline__ void epilogue(const Params &p, int batch, float *st, int lane, int row0, int col0,
                                         const float (&v)[32], const float (&w)[32], const Input<T> &in) {
  using U = Turned<T>;
  constexpr bool kDual = EPI == E_GATED || EPI == E_GATED_BWD;
  const EpiArgs &e = p.e;
  const int c = col0 + U::col(lane);
  U a, b;
  a.turn(st, lane, v);
  if (kDual) b.turn(st, lane, w);
  if (e.b0) {
    float f[U::V];
    U::bias(e.b0, c, p.N, f);
#pragma unroll
    for (int i = 0; i < U::L; ++i)
#pragma unroll
      for (int j = 0; j < U::V; ++j) a.x[i][j] += f[j];
  }
  if (RELU) {
    float top = 0.f;
#pragma unroll
    for (int i = 0; i < U::L; ++i)
#pragma unroll
      for (int j = 0; j < U::V; ++j)
        if (row0 + U::row(i, lane) < p.M && c + j < p.N) top = fmaxf(top, fabsf(a.x[i][j]));
    const float near = warp_max(top) * kNear;
    unsigned flags = 0, zeros = 0;
#pragma unroll
    for (int i = 0; i < U::L; ++i)
#pragma unroll
      for (int j = 0; j < U::V; ++j)
        if (fabsf(a.x[i][j]) <= near && row0 + U::row(i, lane) < p.M && c + j < p.N)
          (a.x[i][j] == 0.f ? zeros : flags) |= 1u << (i * U::V + j);
    // (one vote of the warp where nothing is in doubt)
    const unsigned count = __reduce_add_sync(0xffffffffu, __popc(flags) | __popc(zeros) << 16);
    if (count) {
      if ((count & 0xffffu) > kNearMost) flags = 0;
      if ((count >> 16) && p.N - col0 >= 8) {  // (fewer columns say nothing about a row)
        const unsigned mine = ((1u << U::L) - 1) << (lane / U::L * U::L);  // lanes of this row
#pragma unroll
        for (int i = 0; i < U::L; ++i) {
          bool all = true;
#pragma unroll
          for (int j = 0; j < U::V; ++j) all &= (zeros >> (i * U::V + j) & 1) || c + j >= p.N;
          if ((__ballot_sync(0xffffffffu, all) & mine) == mine) zeros &= ~(((1u << U::V) - 1) << (i * U::V));
        }
      }
      if (__reduce_add_sync(0xffffffffu, __popc(zeros)) <= kZeroMost) flags |= zeros;
      // through `st`, so that the product's code is there once
      unsigned any = __reduce_or_sync(0xffffffffu, flags), dead = 0;
      if (any) {
        __syncwarp();
#pragma unroll 1
        for (; any; any &= any - 1) {
          const int k = __ffs(any) - 1, i = k / U::V, j = k % U::V;
          st[k * 32 + lane] = settled<T>(e.near, flags >> k & 1, row0 + U::row(i, lane), c + j, 0.f, lane, dead, col0);
        }
#pragma unroll
        for (int i = 0; i < U::L; ++i)
#pragma unroll
          for (int j = 0; j < U::V; ++j)
            if (flags >> (i * U::V + j) & 1) a.x[i][j] = st[(i * U::V + j) * 32 + lane];
      }
    }
  }
  if (kDual && e.b1) {
    float f[U::V];
    U::bias(e.b1, c, p.N, f);
#pragma unroll
    for (int i = 0; i < U::L; ++i)
#pragma unroll
      for (int j = 0; j < U::V; ++j) b.x[i][j] += f[j];
  }
  with_act(e.act, [&](auto A) {
    constexpr int ACT = decltype(A)::value;
#pragma unroll
    for (int i = 0; i < U::L; ++i) {
      float u[U::V];
      if (EPI == E_LINEAR || EPI == E_LINEAR_BWD || EPI == E_GATED_BWD) unpack<T>(in.v[i], u);
#pragma unroll
      for (int j = 0; j < U::V; ++j) {
        float y, dy;
        act_pair<ACT>(a.x[i][j], y, dy);
        if (EPI == E_LINEAR) {
          a.x[i][j] = fmaf(y, e.scale, u[j]);
        } else if (EPI == E_GATED) {
          a.x[i][j] = y * b.x[i][j];
        } else if (EPI == E_LINEAR_BWD) {
          a.x[i][j] = dy * e.scale * u[j];
        } else {
          a.x[i][j] = dy * b.x[i][j] * u[j];
          b.x[i][j] = y * u[j];
        }
      }
    }
  });
  if (EPI == E_LINEAR_BWD || EPI == E_GATED_BWD) {
    if (e.sums0) block_sums<T>(a, e.sums0, lane, row0, col0, p.N);
    if (EPI == E_GATED_BWD && e.sums1) block_sums<T>(b, e.sums1, lane, row0, col0, p.N);
  }
  block_store<T>(a, static_cast<T *>(batch ? e.out1 : e.out0), e.ldo, e.vout, st, lane, row0, col0, p.M, p.N);
  if (EPI == E_GATED_BWD) block_store<T>(b, static_cast<T *>(e.out1), e.ldo, e.vout, st, lane, row0, col0, p.M, p.N);
}

template <bool F32, int BN, bool PAIR, int FORM, typename T>
__global__ void __launch_bounds__(kThreads, 1) k_block_gemm(const __grid_constant__ Maps maps, const Params p) {
  using C = Cfg<F32, BN, PAIR>;
  constexpr int EPI = FORM & ~E_RELU;
  constexpr bool kDual = EPI == E_GATED || EPI == E_GATED_BWD;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw), base = (raw + 1023u) & ~1023u;
  uint8_t *gbase = smem_raw + (base - raw);
  float *staging = reinterpret_cast<float *>(gbase + C::Stages * C::StageBytes);
  uint8_t *tail = gbase + C::Stages * C::StageBytes + kAccWarps * kStageFloats * 4;
  const uint32_t bars = smem_u32(tail);
  const uint32_t full0 = bars, empty0 = full0 + 8 * C::Stages, accf0 = empty0 + 8 * C::Stages,
                 acce0 = accf0 + 8 * C::Bufs, drain = acce0 + 8 * C::Bufs;
  static_assert(16 * C::Stages + 16 * C::Bufs + 8 <= 224, "mbarrier area");
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(tail + 224);
  volatile int *abort_flag = reinterpret_cast<volatile int *>(tail + 232);

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int rank = PAIR ? static_cast<int>(cluster_rank()) : 0;
  if (warp == 1) {
    if (PAIR) {
      asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                   "r"(512));
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
    } else {
      asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                   "r"(512));
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
  }
  if (tid == 0) {
    for (int s = 0; s < C::Stages; ++s) {
      mbar_init(full0 + 8 * s, 1);
      mbar_init(empty0 + 8 * s, 1);
    }
    for (int b = 0; b < C::Bufs; ++b) {
      mbar_init(accf0 + 8 * b, 1);
      mbar_init(acce0 + 8 * b, (PAIR ? 2 : 1) * kAccWarps);  // of the pair, at the leader
    }
    mbar_init(drain, 1);
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  tc_fence_before();
  if (PAIR) cluster_sync();  // both CTAs' barriers and tensor memory exist
  else __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const int first = PAIR ? static_cast<int>(cluster_id_x()) : static_cast<int>(blockIdx.x);
  const int step = PAIR ? static_cast<int>(num_clusters_x()) : static_cast<int>(gridDim.x);
  constexpr int TM = PAIR ? 2 * BM : BM;  // rows of a tile
  const int items = p.batch * p.splits * p.tiles_m * p.tiles_n;
  const int out_n = p.dual ? BN / 2 : BN;  // output columns of a tile
  const int planes = F32 ? (p.products == 1 ? 1 : 2) : 1;
  int issued = 0;

  if (warp == 0) {
    // ---------------- TMA producer ----------------
    if (elect_one()) {
      int it = 0;
      bool ok = true;
      // one k tile of an item: the pair of operands and the place in them
      struct At {
        const CUtensorMap *a, *b0, *b1;
        int x, m0, nb0, nb1;
      };
      auto locate = [&](const Item &t, int kt) {
        const int m0 = t.tm * TM + rank * BM, n0 = t.tn * out_n;
        const int seg = kt >= p.kt0 ? 1 : 0;
        At o;
        o.x = (kt - (seg ? p.kt0 : 0)) * BK;
        o.m0 = m0;
        // this CTA's rows of B: two boxes of BRows / 2, in the dual form one of
        // each weight, or (pair) both of this CTA's weight
        o.nb0 = n0 + (PAIR && !p.dual ? rank * C::BRows : 0);
        o.nb1 = p.dual && !PAIR ? n0 : o.nb0 + C::BRows / 2;
        o.a = &maps.a[t.batch | seg];
        o.b0 = &maps.b[PAIR && p.dual ? rank : seg];
        o.b1 = &maps.b[p.dual ? (PAIR ? rank : 1) : seg];
        return o;
      };
      // every box of the tile, in the order of shared memory
      auto boxes = [&](const At &o, auto &&load) {
        for (int z = 0; z < planes; ++z) {
          const uint32_t sa = z * kTile, sb = C::Planes * kTile + z * C::BTile;
          if (p.a_mn) {
            load(sa, o.a, o.m0, o.x, z);
            load(sa + 8192, o.a, o.m0 + 64, o.x, z);
          } else {
            load(sa, o.a, o.x, o.m0, z);
          }
          if (p.b_mn) {
            for (int c = 0; c < C::BRows / 64; ++c) load(sb + 8192 * c, o.b0, o.nb0 + 64 * c, o.x, z);
          } else {
            load(sb, o.b0, o.x, o.nb0, z);
            load(sb + C::BTile / 2, o.b1, o.x, o.nb1, z);
          }
        }
      };
      for (int item = first; item < items && ok; item += step) {
        const Item t = item_of(p, item);
        const int k_end = min(p.kt, (t.split + 1) * p.kt_split);
        for (int kt = t.split * p.kt_split; kt < k_end; ++kt, ++it) {
          const int s = it % C::Stages;
          if (!wait_or_abort(empty0 + 8 * s, ((it / C::Stages) & 1) ^ 1, abort_flag)) {
            ok = false;
            break;
          }
          const uint32_t st = base + s * C::StageBytes;
          const uint32_t fb = PAIR ? map_to_rank(full0 + 8 * s, 0) : full0 + 8 * s;
          if (rank == 0) expect_tx(full0 + 8 * s, (PAIR ? 2 : 1) * planes * (kTile + C::BTile));
          boxes(locate(t, kt), [&](uint32_t off, const CUtensorMap *map, int cx, int cy, int cz) {
            if (PAIR) tma3_pair(st + off, map, fb, cx, cy, cz);
            else tma3(st + off, map, fb, cx, cy, cz);
          });
        }
      }
      // (pair) the commits that free the last stages have arrived here before
      // this CTA ends
      if (PAIR)
        for (int i = it; ok && i < it + C::Stages; ++i)
          ok = wait_or_abort(empty0 + 8 * (i % C::Stages), ((i / C::Stages) & 1) ^ 1, abort_flag);
      issued = it;
    }
    __syncwarp();
  } else if (warp == 1) {
    // ---------------- MMA issuer ----------------
    if (rank == 0 && elect_one()) {
      const uint32_t fmt = (!F32 && p.bf16) ? (1u << 7) | (1u << 10) : 0u;
      const uint32_t idesc = idesc_f16(TM, BN) | fmt | (static_cast<uint32_t>(p.a_mn) << 15) |
                             (static_cast<uint32_t>(p.b_mn) << 16);
      // Operand descriptors (tc_common.cuh: kmajor_desc): the upper word is the
      // same for both ways round; the lower one is the address / 16 and, for
      // an MN-major tile of 64-row chunks ([64 k][64 rows], 128-byte rows), the
      // 8 KB between chunks.  Addresses stay below 2^18, so stages and steps
      // are plain additions to it.  One MMA step is 16 k: 32 bytes along a
      // K-major row, 16 rows of 128 bytes of an MN-major chunk.
      const uint32_t lo_a = (base >> 4) | (p.a_mn ? (8192u >> 4) << 16 : 1u << 16);
      const uint32_t lo_b = ((base + C::Planes * kTile) >> 4) | (p.b_mn ? (8192u >> 4) << 16 : 1u << 16);
      const uint32_t ka = p.a_mn ? 2048u >> 4 : 32u >> 4, kb = p.b_mn ? 2048u >> 4 : 32u >> 4;
      auto desc = [](uint32_t lo) {
        constexpr uint32_t hi = (1024u >> 4) | (1u << 14) | (2u << 29);
        uint64_t d;
        asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "r"(lo), "n"(hi));
        return d;
      };
      auto mma = [&](uint32_t d, uint64_t a, uint64_t b, uint32_t acc) {
        if (PAIR) mma_f16_pair(d, a, b, idesc, acc);
        else mma_f16(d, a, b, idesc, acc);
      };
      auto commit = [&](uint32_t bar) {
        if (PAIR) mma_commit_pair(bar);
        else mma_commit(bar);
      };
      int it = 0, pass = 0;
      bool ok = true;
      for (int item = first; item < items && ok; item += step) {
        const Item t = item_of(p, item);
        const int k_end = min(p.kt, (t.split + 1) * p.kt_split);
        for (int kt0 = t.split * p.kt_split; kt0 < k_end && ok; ++pass) {
          const int b = pass % C::Bufs;
          if (!wait_or_abort(acce0 + 8 * b, ((pass / C::Bufs) & 1) ^ 1, abort_flag)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t d = tmem + static_cast<uint32_t>(b * BN);
          const int p_end = (F32 && kt0 + C::Chunk < k_end) ? kt0 + C::Chunk : k_end;
          for (int kt = kt0; kt < p_end; ++kt, ++it) {
            const int s = it % C::Stages;
            if (!wait_or_abort(full0 + 8 * s, (it / C::Stages) & 1, abort_flag)) {
              ok = false;
              break;
            }
            tc_fence_after();
            const uint32_t da = lo_a + s * (C::StageBytes >> 4), db = lo_b + s * (C::StageBytes >> 4);
#pragma unroll
            for (int kk = 0; kk < BK / 16; ++kk) {
              const uint32_t more = (kt > kt0 || kk > 0) ? 1u : 0u;
              if (F32 && p.products == 3) {
                mma(d, desc(da + (kTile >> 4) + kk * ka), desc(db + kk * kb), more);
                mma(d, desc(da + kk * ka), desc(db + (C::BTile >> 4) + kk * kb), 1u);
              } else {
                mma(d, desc(da + kk * ka), desc(db + kk * kb), more);
              }
            }
            // the large products after the small ones, so that fewer additions
            // are truncated at the sum's full size
            if (F32 && p.products == 3) {
#pragma unroll
              for (int kk = 0; kk < BK / 16; ++kk) mma(d, desc(da + kk * ka), desc(db + kk * kb), 1u);
            }
            commit(empty0 + 8 * s);
          }
          if (ok) commit(accf0 + 8 * b);
          kt0 = p_end;
        }
      }
    }
    __syncwarp();
  } else {
    // ------- accumulators and epilogue: warp -> (lane quarter q, share h) -------
    // A warp's columns are two groups of G of the accumulator: in the gated
    // forms the gate and the value of the same outputs.
    constexpr int G = BN / 4;
    const int q = warp & 3, h = (warp - 2) / 4;
    const int cb[2] = {kDual ? h * G : h * 2 * G, kDual ? BN / 2 + h * G : h * 2 * G + G};
    float *st = staging + (warp - 2) * kStageFloats;
    const uint32_t tq = tmem + (static_cast<uint32_t>(q * 32) << 16);
    // this warp has read accumulator b
    auto release = [&](int b) {
      tc_fence_before();
      __syncwarp();
      if (lane) return;
      if (PAIR) mbar_arrive_cluster(map_to_rank(acce0 + 8 * b, 0));
      else mbar_arrive(acce0 + 8 * b);
    };
    int pass = 0;
    bool ok = true;
    for (int item = first; item < items && ok; item += step) {
      const Item t = item_of(p, item);
      const int row0 = t.tm * TM + rank * BM + q * 32, row = row0 + lane, n0 = t.tn * out_n;
      const int k0 = t.split * p.kt_split, k_end = min(p.kt, k0 + p.kt_split);
      constexpr int GA = F32 ? G : 1;
      // output columns a warp finishes, in blocks of 32; column of block i / 32
      constexpr int kCols = kDual ? G : 2 * G;
      constexpr bool kIn = EPI == E_LINEAR || EPI == E_LINEAR_BWD || EPI == E_GATED_BWD;
      auto col_of = [&](int i) {
        const int c = kDual ? h * G + i : cb[i / G] + i % G;
        return n0 + c - ((EPI == E_PARTIAL && p.dual) ? h * (BN / 2) : 0);
      };
      Input<T> next;
      if (kIn) {
        if (p.e.in) {
          next.fetch(p, lane, row0, col_of(0));
        } else {
#pragma unroll
          for (int i = 0; i < Turned<T>::L; ++i) next.v[i] = make_uint4(0u, 0u, 0u, 0u);
        }
      }
      float acc[2][GA];  // f32: the running sums
      int b = 0;
      if (F32) {
#pragma unroll
        for (int gi = 0; gi < 2; ++gi)
#pragma unroll
          for (int j = 0; j < GA; ++j) acc[gi][j] = 0.f;
        // scales of this thread's row and of column `lane` of each group in one
        // pass, requested a pass ahead and not touched before it
        uint32_t sa = 0, sb[2] = {p.bsc[0], p.bsc[p.dual ? 1 : 0]};
        auto scales = [&](int kt) {
          const int seg = kt >= p.kt0 ? 1 : 0, o = t.batch | seg;
          const int blk = (kt - (seg ? p.kt0 : 0)) / C::Chunk;
          if (row < p.M) sa = p.sc[o][static_cast<size_t>(blk) * p.scld[o] + row];
#pragma unroll
          for (int gi = 0; gi < 2; ++gi) {
            const int half = p.dual && cb[gi] >= BN / 2 ? 1 : 0, bi = p.dual ? half : seg;
            const int col = min(n0 + cb[gi] - half * (BN / 2) + lane, p.N - 1);
            sb[gi] = p.bs[bi] ? p.bs[bi][static_cast<size_t>(blk) * p.bsld[bi] + col] : p.bsc[bi];
          }
        };
        scales(k0);
        for (int kt = k0; kt < k_end; kt += C::Chunk, ++pass) {
          const float fa = __uint_as_float(sa << 16);
          // columns of one scale (of ordinary sizes, by k_split's choice) need
          // one factor; others theirs, by way of `st`
          float f[2];
          bool even[2];
          __syncwarp();  // the pass before has been read
#pragma unroll
          for (int gi = 0; gi < 2; ++gi) {
            const float fb = __uint_as_float(sb[gi] << 16);
            f[gi] = fa * __shfl_sync(0xffffffffu, fb, 0);
            even[gi] = __all_sync(0xffffffffu, sb[gi] == __shfl_sync(0xffffffffu, sb[gi], 0));
            if (!even[gi]) st[gi * 32 + lane] = fb;
          }
          __syncwarp();
          if (kt + C::Chunk < k_end) scales(kt + C::Chunk);
          b = pass % C::Bufs;
          if (!__all_sync(0xffffffffu, wait_or_abort(accf0 + 8 * b, (pass / C::Bufs) & 1, abort_flag))) {
            ok = false;
            break;
          }
          tc_fence_after();
          static_assert(!F32 || G == 32, "a group is 32 columns");
#pragma unroll
          for (int gi = 0; gi < 2; ++gi) {
            float v[32];
            tmem_ld32(tq + static_cast<uint32_t>(b * BN + cb[gi]), v);
            if (gi) release(b);
            if (even[gi]) {
#pragma unroll
              for (int j = 0; j < 32; ++j) acc[gi][F32 ? j : 0] = __fmaf_rn(v[j], f[gi], acc[gi][F32 ? j : 0]);
            } else {  // (the two scales first: either may be far from 1)
#pragma unroll
              for (int j = 0; j < 32; ++j)
                acc[gi][F32 ? j : 0] = __fmaf_rn(v[j], fa * st[gi * 32 + j], acc[gi][F32 ? j : 0]);
            }
          }
        }
        if (!ok) break;
      } else {
        b = pass % C::Bufs;
        if (!__all_sync(0xffffffffu, wait_or_abort(accf0 + 8 * b, (pass / C::Bufs) & 1, abort_flag))) {
          ok = false;
          break;
        }
        tc_fence_after();
        ++pass;
      }
      auto get = [&](int gi, int c, float(&v)[32]) {
        if constexpr (F32) {
#pragma unroll
          for (int j = 0; j < 32; ++j) v[j] = acc[gi][c + j];
        } else {
          tmem_ld32(tq + static_cast<uint32_t>(b * BN + cb[gi] + c), v);
        }
      };
      auto chunk = [&](int i) {
        const int gi = i / G, c = i % G;
        float v[32], w[32];
        get(gi, c, v);
        if (kDual) get(1, c, w);
        const int col = col_of(i);
        if constexpr (EPI == E_PARTIAL) {
          if (col >= p.N || row0 >= p.M) return;
          Turned<float> o;
          o.turn(st, lane, v);
          float *dst = p.e.part + (static_cast<size_t>(t.batch) * p.splits + t.split) * p.M * p.e.nacc +
                       (p.dual ? h * p.N : 0);
          block_store<float>(o, dst, p.e.nacc, p.e.vout, st, lane, row0, col, p.M, p.N);
        } else {
          const Input<T> cur = next;
          if (kIn && p.e.in && i + 32 < kCols) next.fetch(p, lane, row0, col_of(i + 32));
          if (col >= p.N || row0 >= p.M) return;
          epilogue<EPI, (FORM & E_RELU) != 0, T>(p, t.batch, st, lane, row0, col, v, w, cur);
        }
      };
      if (F32) {  // register arrays: constant indices
#pragma unroll
        for (int i = 0; i < kCols; i += 32) chunk(i);
      } else {
#pragma unroll 1
        for (int i = 0; i < kCols; i += 32) chunk(i);
        release(b);
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (*abort_flag) {
    // this CTA's own loads and MMAs complete before it ends; a pair's loads
    // report to the leader's barriers, so both CTAs allow them 10 ms instead
    if (PAIR) {
      const uint64_t t0 = globaltimer();
      while (tid == 0 && globaltimer() - t0 < 10000000ull) {
      }
    } else if (warp == 0 && issued) {
      for (int j = issued > C::Stages ? issued - C::Stages : 0; j < issued; ++j)
        wait_bounded(full0 + 8 * (j % C::Stages), (j / C::Stages) & 1);
    }
    if (warp == 1 && rank == 0 && elect_one()) {
      if (PAIR) mma_commit_pair(drain);
      else mma_commit(drain);
      wait_bounded(drain, 0);
    }
    __syncthreads();
    if (tid == 0) raise_error(p.err, g_block_err);
  }
  if (PAIR) {
    cluster_sync();  // neither CTA leaves while the other may still signal it
    tc_fence_after();
    if (warp == 1) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512));
  } else if (warp == 1) {
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512));
  }
}

// Sums the partial products of a split launch in order and runs the epilogue.
// Block: 32 columns x 32 rows, four rows a thread.
template <int EPI, typename T>
__global__ void __launch_bounds__(256) k_join(const Params p) {
  __shared__ float part[2][8][32];
  const EpiArgs &e = p.e;
  const int lane = threadIdx.x & 31, w8 = threadIdx.x >> 5;
  const int64_t nb = (p.N + 31) / 32, mb = (p.M + 31) / 32, all = nb * mb * p.batch;
  for (int64_t id = blockIdx.x; id < all; id += gridDim.x) {
    const int batch = static_cast<int>(id / (nb * mb));
    const int64_t strip = (id - batch * nb * mb) / nb, col = (id % nb) * 32 + lane;
    float s0 = 0.f, s1 = 0.f;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int64_t row = strip * 32 + k * 8 + w8;
      const bool there = row < p.M && col < p.N;
      float v = 0.f, w = 0.f, in = 0.f, top = 0.f;
      if (there) {
        const float *src = e.part + static_cast<size_t>(batch) * p.splits * p.M * e.nacc + row * e.nacc + col;
        const size_t step = static_cast<size_t>(p.M) * e.nacc;
        for (int s = 0; s < p.splits; ++s) {
          v += src[s * step];
          top = fmaxf(top, fabsf(src[s * step]));
        }
        if (p.dual)
          for (int s = 0; s < p.splits; ++s) w += src[s * step + p.N];
        if (e.b0) v += to_f(static_cast<const T *>(e.b0)[col]);
        if (p.dual && e.b1) w += to_f(static_cast<const T *>(e.b1)[col]);
        if (e.in) in = to_f(static_cast<const T *>(e.in)[row * e.ldin + col]);
      }
      if ((EPI == E_LINEAR_BWD || EPI == E_GATED_BWD) && e.near.x) {
        const float near = warp_max(top) * kNear;  // (of the whole warp: lanes past the edges bring 0)
        v = settled_row<T>(e.near, there, near, row, col, v, lane);
      }
      if (!there) continue;
      T *o = static_cast<T *>(batch ? e.out1 : e.out0) + row * e.ldo + col;
      with_act(e.act, [&](auto A) {
        constexpr int ACT = decltype(A)::value;
        float a, da;
        act_pair<ACT>(v, a, da);
        if (EPI == E_LINEAR) {
          *o = from_f<T>(fmaf(a, e.scale, in));
        } else if (EPI == E_LINEAR_BWD) {
          const float r = da * e.scale * in;
          s0 += r;
          *o = from_f<T>(r);
        } else if (EPI == E_GATED) {
          *o = from_f<T>(a * w);
        } else {
          const float r = da * w * in, q = a * in;
          s0 += r;
          s1 += q;
          *o = from_f<T>(r);
          static_cast<T *>(e.out1)[row * e.ldo + col] = from_f<T>(q);
        }
      });
    }
    if ((EPI == E_LINEAR_BWD || EPI == E_GATED_BWD) && (e.sums0 || e.sums1)) {
      __syncthreads();
      part[0][w8][lane] = s0;
      part[1][w8][lane] = s1;
      __syncthreads();
      float *const sums = w8 == 0 ? e.sums0 : w8 == 1 ? e.sums1 : nullptr;
      if (sums && col < p.N) {
        float t = 0.f;
#pragma unroll
        for (int k = 0; k < 8; ++k) t += part[w8][k][lane];
        sums[strip * p.N + col] = t;
      }
    }
  }
}

// ---------------------------------------------------------------------------
// Operand preparation
// ---------------------------------------------------------------------------
// |x|, 0 for infinities and NaN: these must not set the scale of the finite
// elements beside them.
__device__ __forceinline__ float finite_abs(float x) {
  const float a = fabsf(x);
  return a < INFINITY ? a : 0.f;
}

// f32 matrices -> split-fp16 operands, all of a step in one launch; a CTA
// takes a 128 x 128 block of one of them, reads it once into registers and
// writes each form that a product needs of it:
//   rows    one scale per row and 128 columns, [column block][row]
//   cols    one scale per column and 128 rows, [row block][column]
// (2^-s: the upper half of the float).  Of a B operand, whose scales the product
// applies to columns, the rows (columns) within 2^-kEven of their block's largest
// take its scale: an element keeps 2^-40 of what its scale is for, 2^-32 of its
// own row's (column's) largest, far below the 2^-22 that it is good to.
// and, for bias gradients, the sums of its columns, [row block][column].
// All forms are [R][lp] hi, then lo.
struct SplitForm {
  uint16_t *hi, *sc;
  int64_t scld;
  bool even;
};
struct SplitJob {
  const float *src;
  int64_t ld;
  int R, C, lp, first;  // first: number of the job's first block
  bool vec;
  SplitForm rows, cols;
  float *sums;
};
// 2^-s as the upper half of a float
__host__ __device__ __forceinline__ uint16_t scale_bits(int s) { return static_cast<uint16_t>((127 - s) << 7); }
constexpr int kEven = 8;
constexpr int kMaxJobs = 4;
struct SplitJobs {
  SplitJob job[kMaxJobs];
  int n, total;
};
__global__ void __launch_bounds__(256, 2) k_split(const SplitJobs all) {
  __shared__ float part[8][128];
  const int w = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int id = blockIdx.x; id < all.total; id += gridDim.x) {
    int ji = 0;
    while (ji + 1 < all.n && id >= all.job[ji + 1].first) ++ji;
    const SplitJob &q = all.job[ji];
    const int nb = (q.C + 127) / 128, rb = (id - q.first) / nb, cb = (id - q.first) % nb;
    const int c = cb * 128 + 4 * lane, r0 = rb * 128 + w * 16;
    float v[16][4];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const float *p = q.src + static_cast<size_t>(r0 + i) * q.ld + c;
#pragma unroll
      for (int j = 0; j < 4; ++j) v[i][j] = 0.f;
      if (r0 + i >= q.R) continue;
      if (q.vec && c + 4 <= q.C) {
        const float4 u = *reinterpret_cast<const float4 *>(p);
        v[i][0] = u.x;
        v[i][1] = u.y;
        v[i][2] = u.z;
        v[i][3] = u.w;
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (c + j < q.C) v[i][j] = p[j];
      }
    }
    const int64_t plane = static_cast<int64_t>(q.R) * q.lp;
    // one row of the block in split form, each column by its own scale
    auto put = [&](uint16_t *hi, int i, const float (&f)[4]) {
      if (r0 + i >= q.R || c >= q.lp) return;
      uint32_t h[2], l[2];
#pragma unroll
      for (int j = 0; j < 2; ++j) split2(v[i][2 * j] * f[2 * j], v[i][2 * j + 1] * f[2 * j + 1], 1.f, h[j], l[j]);
      uint16_t *o = hi + static_cast<size_t>(r0 + i) * q.lp + c;
      if (c + 4 <= q.lp) {
        *reinterpret_cast<uint2 *>(o) = make_uint2(h[0], h[1]);
        *reinterpret_cast<uint2 *>(o + plane) = make_uint2(l[0], l[1]);
      }
    };
    // maximum (or sum) over the block's rows, per column, in a fixed order
    auto over_rows = [&](const float (&x)[4], bool add, float (&out)[4]) {
      __syncthreads();
      *reinterpret_cast<float4 *>(&part[w][4 * lane]) = make_float4(x[0], x[1], x[2], x[3]);
      __syncthreads();
#pragma unroll
      for (int j = 0; j < 4; ++j) out[j] = 0.f;
#pragma unroll
      for (int k = 0; k < 8; ++k)
#pragma unroll
        for (int j = 0; j < 4; ++j) out[j] = add ? out[j] + part[k][4 * lane + j] : fmaxf(out[j], part[k][4 * lane + j]);
    };
    // exponent of one row (column) by its largest element, given the block's
    // least (kNone: nothing but zeros)
    constexpr int kNone = 1 << 20;
    auto exponent = [](float m) { return m > 0.f ? split_scale_exponent(m) : kNone; };
    auto choose = [](int s, int least, bool even) {
      if (s == kNone) return least == kNone ? 0 : least;
      return even && s - least <= kEven ? least : s;
    };
    if (q.rows.hi) {
      int s[16], least = kNone;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        float m = 0.f;
#pragma unroll
        for (int j = 0; j < 4; ++j) m = fmaxf(m, finite_abs(v[i][j]));
        s[i] = exponent(warp_max(m));
        least = min(least, s[i]);
      }
      if (q.rows.even) {
        __syncthreads();
        if (lane == 0) part[w][0] = __int_as_float(least);
        __syncthreads();
#pragma unroll
        for (int k = 0; k < 8; ++k) least = min(least, __float_as_int(part[k][0]));
      }
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int si = choose(s[i], least, q.rows.even);
        const float e = pow2f(si), f[4] = {e, e, e, e};
        put(q.rows.hi, i, f);
        if (lane == 0 && r0 + i < q.R) q.rows.sc[static_cast<size_t>(cb) * q.rows.scld + r0 + i] = scale_bits(si);
      }
    }
    if (q.cols.hi) {
      float m[4] = {0.f, 0.f, 0.f, 0.f}, top[4];
#pragma unroll
      for (int i = 0; i < 16; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) m[j] = fmaxf(m[j], finite_abs(v[i][j]));
      over_rows(m, false, top);
      int s[4], least = kNone;
      float f[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        s[j] = exponent(top[j]);
        least = min(least, s[j]);
      }
      least = __reduce_min_sync(0xffffffffu, least);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        s[j] = choose(s[j], least, q.cols.even);
        f[j] = pow2f(s[j]);
      }
#pragma unroll
      for (int i = 0; i < 16; ++i) put(q.cols.hi, i, f);
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (w == 0 && c + j < q.lp) q.cols.sc[static_cast<size_t>(rb) * q.cols.scld + c + j] = scale_bits(s[j]);
    }
    if (q.sums) {
      float m[4] = {0.f, 0.f, 0.f, 0.f}, sum[4];
#pragma unroll
      for (int i = 0; i < 16; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) m[j] += v[i][j];
      over_rows(m, true, sum);
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (w == 0 && c + j < q.C) q.sums[static_cast<size_t>(rb) * q.C + c + j] = sum[j];
    }
  }
}

// 16-bit matrices whose address or stride TMA cannot take -> rows of cp
// elements, all of a step in one launch; eight elements a thread.
struct PackJob {
  const uint16_t *src;
  uint16_t *dst;
  int64_t ld, rows, first;  // first: number of the job's first piece
  int C, cp;
};
struct PackJobs {
  PackJob job[4];
  int n;
  int64_t total;
};
__global__ void __launch_bounds__(256) k_pack(const PackJobs all) {
  for (int64_t id = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; id < all.total; id += static_cast<int64_t>(gridDim.x) * 256) {
    int ji = 0;
    while (ji + 1 < all.n && id >= all.job[ji + 1].first) ++ji;
    const PackJob &q = all.job[ji];
    const int64_t i = id - q.first, nc = q.cp / 8, r = i / nc;
    const int c = static_cast<int>(i - r * nc) * 8;
    const uint16_t *p = q.src + r * q.ld + c;
    uint32_t v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = c + j < q.C ? p[j] : 0u;
    *reinterpret_cast<uint4 *>(q.dst + r * q.cp + c) =
        make_uint4(v[0] | v[1] << 16, v[2] | v[3] << 16, v[4] | v[5] << 16, v[6] | v[7] << 16);
  }
}

int grid_for(int64_t threads) {
  const int64_t b = (threads + 255) / 256, top = 16LL * sm_count();
  return static_cast<int>(std::max<int64_t>(1, std::min(b, top)));
}

// A matrix [rows, cols] as an operand of the tensor-core kernel.
struct Operand {
  const uint16_t *p = nullptr;
  int64_t rows = 0, cols = 0, ld = 0;
  int planes = 1;
  int64_t plane = 0;           // elements between hi and lo
  const uint16_t *sc = nullptr;  // f32: scales
  int64_t scld = 0;              // ... between the contraction's blocks of 128
  int scale = 0;                 // f32 B without sc: one exponent
};

// Prepares operands: 16-bit ones where they lie (or packed), f32 ones in split
// form, by one launch each, issued by go().
enum Form { FORM_NONE, FORM_ROWS, FORM_COLS };
class Operands {
 public:
  Operands(int dt, Workspace &ws, cudaStream_t s) : dt_(dt), ws_(ws), s_(s) {}

  // `m` for a product that contracts its columns (FORM_ROWS) or rows (FORM_COLS);
  // even: as the B operand
  Operand add(const Mat &m, int64_t rows, int64_t cols, Form form, bool even = false) {
    if (dt_ != DT_F32) return packed(m, rows, cols);
    Operand o;
    o.rows = rows;
    o.cols = cols;
    o.ld = (cols + 7) / 8 * 8;
    o.planes = 2;
    o.plane = rows * o.ld;
    uint16_t *d = static_cast<uint16_t *>(ws_.take(4 * rows * o.ld));
    const int64_t rb = (rows + 127) / 128, cb = (cols + 127) / 128;
    o.scld = form == FORM_ROWS ? rows : o.ld;
    uint16_t *sc = static_cast<uint16_t *>(ws_.take(2 * (form == FORM_ROWS ? cb : rb) * o.scld));
    o.p = d;
    o.sc = sc;
    if (ws_.sizing()) return o;
    of(job(m, rows, cols, form), form) = SplitForm{d, sc, o.scld, even};
    return o;
  }
  // f32: sums of the columns of each 128 rows of `m` into part [rows / 128][cols]
  void sums(const Mat &m, int64_t rows, int64_t cols, float *part) {
    if (!ws_.sizing()) job(m, rows, cols, FORM_NONE).sums = part;
  }
  void go() {
    if (pack_.n) {
      k_pack<<<grid_for(pack_.total), 256, 0, s_>>>(pack_);
      CUDA_LAUNCH_CHECK();
      pack_ = PackJobs{};
    }
    if (!all_.n) return;
    all_.total = 0;
    for (int i = 0; i < all_.n; ++i) {
      SplitJob &j = all_.job[i];
      j.first = all_.total;
      const int64_t blocks = static_cast<int64_t>(ceil_div(j.R, 128)) * ceil_div(j.C, 128);
      if (blocks > INT32_MAX / 2 - all_.total) throw Error(kErrInvalidParameter, "the operands have too many blocks");
      all_.total += static_cast<int>(blocks);
    }
    k_split<<<std::min(all_.total, 8 * sm_count()), 256, 0, s_>>>(all_);
    CUDA_LAUNCH_CHECK();
    all_.n = 0;
  }

 private:
  static SplitForm &of(SplitJob &j, Form f) { return f == FORM_ROWS ? j.rows : j.cols; }
  // the job that reads `m`: one for all forms of one matrix (a second one if
  // it has this form already, as when both weights are the same tensor)
  SplitJob &job(const Mat &m, int64_t rows, int64_t cols, Form form) {
    for (int i = 0; i < all_.n; ++i) {
      SplitJob &j = all_.job[i];
      if (j.src == m.p && j.ld == m.ld && j.R == rows && j.C == cols && (form == FORM_NONE || !of(j, form).hi)) return j;
    }
    if (all_.n == kMaxJobs) throw Error(kErrInternal, "too many operands in one step");
    SplitJob &j = all_.job[all_.n++];
    j = SplitJob{};
    j.src = static_cast<const float *>(m.p);
    j.ld = m.ld;
    j.R = static_cast<int>(rows);
    j.C = static_cast<int>(cols);
    j.lp = static_cast<int>((cols + 7) / 8 * 8);
    j.vec = rows16(m.p, m.ld, DT_F32);
    return j;
  }
  Operand packed(const Mat &m, int64_t rows, int64_t cols) {
    Operand o;
    o.rows = rows;
    o.cols = cols;
    if (rows16(m.p, m.ld, dt_)) {
      o.p = static_cast<const uint16_t *>(m.p);
      o.ld = m.ld;
      return o;
    }
    o.ld = (cols + 7) / 8 * 8;
    uint16_t *d = static_cast<uint16_t *>(ws_.take(2 * rows * o.ld));
    o.p = d;
    if (!ws_.sizing()) {
      if (pack_.n == 4) throw Error(kErrInternal, "too many operands in one step");
      pack_.job[pack_.n++] = PackJob{static_cast<const uint16_t *>(m.p), d, m.ld, rows, pack_.total,
                                     static_cast<int>(cols), static_cast<int>(o.ld)};
      pack_.total += rows * (o.ld / 8);
    }
    return o;
  }
  int dt_;
  Workspace &ws_;
  cudaStream_t s_;
  SplitJobs all_{};
  PackJobs pack_{};
};

// ---------------------------------------------------------------------------
// Launch
// ---------------------------------------------------------------------------
PFN_cuTensorMapEncodeTiled_v12000 encoder() {
  static const PFN_cuTensorMapEncodeTiled_v12000 f = [] {
    void *fn = nullptr;
    cudaDriverEntryPointQueryResult q;
    CUDA_CHECK(cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &q));
    if (!fn || q != cudaDriverEntryPointSuccess) throw Error(kErrBackend, "cuTensorMapEncodeTiled unavailable");
    return reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(fn);
  }();
  return f;
}

// Boxes of 64 columns x box_rows rows of one plane, zeros outside.
CUtensorMap map_of(const Operand &o, bool bf16, int box_rows) {
  CUtensorMap m;
  const cuuint64_t dims[3] = {static_cast<cuuint64_t>(o.cols), static_cast<cuuint64_t>(o.rows),
                              static_cast<cuuint64_t>(o.planes)};
  const cuuint64_t strides[2] = {static_cast<cuuint64_t>(o.ld) * 2,
                                 static_cast<cuuint64_t>(o.planes > 1 ? o.plane : o.ld) * 2};
  const cuuint32_t box[3] = {64, static_cast<cuuint32_t>(box_rows), 1}, es[3] = {1, 1, 1};
  const CUresult r =
      encoder()(&m, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3,
                const_cast<uint16_t *>(o.p), dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
                CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) throw Error(kErrBackend, "cuTensorMapEncodeTiled failed (" + std::to_string(r) + ")");
  return m;
}

struct Product {
  int dt = DT_F32, epi = E_LINEAR, products = 3;
  int *err = nullptr;
  int64_t M = 0, N = 0, K = 0;  // K: contraction of each pair of operands
  Operand a[2], b[2];
  bool a_mn = false, b_mn = false, dual = false, kcat = false, batch2 = false;
  EpiArgs e{};
};

template <bool F32, int BN, bool PAIR, int EPI, typename T>
void launch(const Maps &maps, const Params &p, cudaStream_t s) {
  constexpr int smem = Cfg<F32, BN, PAIR>::Smem;
  auto *kernel = k_block_gemm<F32, BN, PAIR, EPI, T>;
  CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
  const int items = p.batch * p.splits * p.tiles_m * p.tiles_n;
  if (!PAIR) {
    kernel<<<std::min(items, sm_count()), kThreads, smem, s>>>(maps, p);
    CUDA_LAUNCH_CHECK();
    return;
  }
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(2 * std::min(items, sm_count() / 2));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  CUDA_CHECK(cudaLaunchKernelEx(&cfg, kernel, maps, p));
  ::pet::g_kernel_launches.fetch_add(1, std::memory_order_relaxed);
}
// How a product is tiled.
struct Tiling {
  int bn;
  bool pair;
};
template <int EPI, typename T>
void launch_16(Tiling t, const Maps &maps, const Params &p, cudaStream_t s) {
  if (t.pair) launch<false, 256, true, EPI, T>(maps, p, s);
  else if (t.bn == 256) launch<false, 256, false, EPI, T>(maps, p, s);
  else launch<false, 128, false, EPI, T>(maps, p, s);
}
template <int EPI>
void launch_epi(int dt, Tiling t, const Maps &maps, const Params &p, cudaStream_t s) {
  if (dt == DT_F16) launch_16<EPI, __half>(t, maps, p, s);
  else if (dt == DT_BF16) launch_16<EPI, __nv_bfloat16>(t, maps, p, s);
  else launch<true, 128, false, EPI, float>(maps, p, s);
}
template <int EPI>
void join_epi(int dt, const Params &p, cudaStream_t s) {
  const int64_t blocks = static_cast<int64_t>(ceil_div(p.M, 32)) * ceil_div(p.N, 32) * p.batch;
  const int g = static_cast<int>(std::min<int64_t>(blocks, 8LL * sm_count()));
  if (dt == DT_F32) k_join<EPI, float><<<g, 256, 0, s>>>(p);
  else if (dt == DT_F16) k_join<EPI, __half><<<g, 256, 0, s>>>(p);
  else k_join<EPI, __nv_bfloat16><<<g, 256, 0, s>>>(p);
  CUDA_LAUNCH_CHECK();
}

void run(const Product &g, Workspace &ws, cudaStream_t s) {
  const bool f32 = g.dt == DT_F32;
  const int sms = sm_count();
  Params p{};
  p.M = static_cast<int>(g.M);
  p.N = static_cast<int>(g.N);
  const int unit = f32 ? 2 : 1;  // k tiles that share a scale
  p.kt0 = static_cast<int>((g.K + BK * unit - 1) / (BK * unit)) * unit;
  p.kt = g.kcat ? 2 * p.kt0 : p.kt0;
  p.batch = g.batch2 ? 2 : 1;
  p.a_mn = g.a_mn;
  p.b_mn = g.b_mn;
  p.dual = g.dual;
  p.bf16 = g.dt == DT_BF16;
  p.products = g.products;
  p.err = g.err;
  p.e = g.e;
  // tiles of bm rows of `bn` accumulator columns
  auto count = [&](int bm, int bn) {
    const int on = g.dual ? bn / 2 : bn;
    return (g.M + bm - 1) / bm * ((g.N + on - 1) / on) * p.batch;
  };
  // f32 takes 128 x 128 tiles of one SM (256-wide ones leave no registers for
  // the epilogue beside the running sums).  16-bit: time in waves over the
  // SMs, in units of one SM's 128 x 256 tile; a pair's 256 x 256 tile takes
  // kPair of one, a 128-wide one kNarrow, not half (it needs more
  // shared-memory traffic for a product).  Measured in bf16: 8192 x 1024 x 8192
  // in 100 (pair), 107 and 145 us, 1024 x 4096 x 8192 in 56, 59 and 76.
  constexpr double kPair = 0.93, kNarrow = 0.66;
  auto waves = [&](int64_t tiles, int at_once) { return static_cast<double>((tiles + at_once - 1) / at_once); };
  Tiling tile{128, false};
  if (!f32) {
    const double narrow = kNarrow * waves(count(BM, 128), sms), wide = waves(count(BM, 256), sms),
                 pair = kPair * waves(count(2 * BM, 256), sms / 2);
    if (g.M > BM && pair < narrow && pair < wide) tile = {256, true};
    else if (wide < narrow) tile = {256, false};
  }
  const int bm = tile.pair ? 2 * BM : BM, bn = tile.bn;
  const int64_t tiles = count(bm, bn);
  p.tiles_m = static_cast<int>((g.M + bm - 1) / bm);
  p.tiles_n = static_cast<int>(tiles / p.tiles_m / p.batch);
  // few tiles and a long contraction: divided over the SMs, where that saves
  // 20 k tiles or more (0.2 us each of 128 x 128 in f16, more of wider tiles and
  // of f32) against the 6 us of the second kernel.  128 x 128 outputs in f16:
  // 16, 24, 32 and 64 k tiles in 8.3, 11.7, 9.9 and 11.2 us
  const int at_once = tile.pair ? sms / 2 : sms;
  int splits = 1;
  if (tiles * 2 <= at_once && p.kt >= 16) {
    splits = static_cast<int>(std::min<int64_t>(at_once / tiles, p.kt / 4));
    if (p.kt - (p.kt + splits - 1) / splits < 20) splits = 1;
  }
  // 16-bit: an accumulator takes each 16 terms with one truncation of at most
  // 2^-23 of the sum (f32 joins in registers instead).  Beyond this many all of
  // them together could pass half a rounding of the result: divided further.
  if (!f32) {
    // (2^11 steps of 2^-23 against 2^-11 / 2 in f16, 2^14 against 2^-8 / 2 in bf16)
    const int most = (g.dt == DT_F16 ? 32768 : 262144) / BK;
    splits = std::max(splits, (p.kt + most - 1) / most);
  }
  p.kt_split = (p.kt + splits - 1) / splits;
  p.kt_split = (p.kt_split + unit - 1) / unit * unit;
  p.splits = splits = (p.kt + p.kt_split - 1) / p.kt_split;
  if (tiles * splits > INT32_MAX / 2) throw Error(kErrInvalidParameter, "the product has too many tiles");
  p.e.vin = !g.e.in || rows16(g.e.in, g.e.ldin, g.dt);
  p.e.vout = rows16(g.e.out0, g.e.ldo, g.dt) && (!g.e.out1 || aligned16(g.e.out1));
  Params q = p;  // the partial launch's
  if (splits > 1) {
    q.e.nacc = p.e.nacc = g.dual ? 2 * g.N : g.N;
    q.e.part = p.e.part = static_cast<float *>(ws.take(4 * static_cast<size_t>(p.batch) * splits * g.M * p.e.nacc));
    q.e.vout = p.e.nacc % 4 == 0 && g.N % 4 == 0;
  }
  if (ws.sizing()) return;
  Maps maps;
  std::memset(&maps, 0, sizeof(maps));
  const bool bf = g.dt == DT_BF16;
  for (int i = 0; i < 2; ++i) {
    const Operand &a = g.a[i].p ? g.a[i] : g.a[0], &b = g.b[i].p ? g.b[i] : g.b[0];
    maps.a[i] = map_of(a, bf, g.a_mn ? 64 : BM);
    maps.b[i] = map_of(b, bf, g.b_mn ? 64 : (tile.pair ? bn / 4 : bn / 2));
    q.sc[i] = a.sc;
    q.scld[i] = a.scld;
    q.bs[i] = b.sc;
    q.bsld[i] = b.scld;
    q.bsc[i] = scale_bits(b.scale);
  }
  if (splits > 1) {
    launch_epi<E_PARTIAL>(g.dt, tile, maps, q, s);
    switch (g.epi) {
      case E_LINEAR: join_epi<E_LINEAR>(g.dt, p, s); break;
      case E_LINEAR_BWD: join_epi<E_LINEAR_BWD>(g.dt, p, s); break;
      case E_GATED: join_epi<E_GATED>(g.dt, p, s); break;
      default: join_epi<E_GATED_BWD>(g.dt, p, s); break;
    }
    return;
  }
  switch (g.epi) {
    case E_LINEAR: launch_epi<E_LINEAR>(g.dt, tile, maps, q, s); break;
    case E_LINEAR_BWD:
      if (g.e.near.x) launch_epi<E_LINEAR_BWD | E_RELU>(g.dt, tile, maps, q, s);
      else launch_epi<E_LINEAR_BWD>(g.dt, tile, maps, q, s);
      break;
    case E_GATED: launch_epi<E_GATED>(g.dt, tile, maps, q, s); break;
    default:
      if (g.e.near.x) launch_epi<E_GATED_BWD | E_RELU>(g.dt, tile, maps, q, s);
      else launch_epi<E_GATED_BWD>(g.dt, tile, maps, q, s);
      break;
  }
}

void zero_rows(void *p, int64_t ld, int64_t rows, int64_t cols, int dt, cudaStream_t s) {
  if (p && rows > 0)
    CUDA_CHECK(cudaMemset2DAsync(p, ld * dtype_size(dt), 0, cols * dtype_size(dt), rows, s));
}

EpiArgs plain_out(const MutMat &m) {
  EpiArgs e{};
  e.out0 = m.p;
  e.ldo = m.ld;
  e.act = ACT_IDENTITY;
  e.scale = 1.f;
  return e;
}

}  // namespace

int sm_count() {
  // every device of a node has the same count
  static const int n = [] {
    int dev = 0, v = 0;
    CUDA_CHECK(cudaGetDevice(&dev));
    CUDA_CHECK(cudaDeviceGetAttribute(&v, cudaDevAttrMultiProcessorCount, dev));
    return v;
  }();
  return n;
}

bool new_errors(const int &word, cudaStream_t s) {
  static std::mutex mutex;
  static std::map<std::pair<const int *, int>, int> seen;
  int dev = 0, v = 0;
  CUDA_CHECK(cudaGetDevice(&dev));
  CUDA_CHECK(cudaStreamSynchronize(s));  // (not while others wait for the lock)
  std::lock_guard<std::mutex> lock(mutex);
  CUDA_CHECK(cudaMemcpyFromSymbolAsync(&v, word, sizeof(v), 0, cudaMemcpyDeviceToHost, s));
  CUDA_CHECK(cudaStreamSynchronize(s));
  int &last = seen[{&word, dev}];
  const bool fresh = v != last;
  last = v;
  return fresh;
}

}  // namespace blk

using namespace blk;

void *Workspace::take(size_t bytes) {
  const size_t b = (bytes + 255) / 256 * 256;
  void *p = base ? base + off : nullptr;
  off += b;
  if (base && off > cap) throw Error(kErrInvalidParameter, "the workspace is too small");
  return p;
}

bool block_status(cudaStream_t s) {
  const bool a = new_errors(g_block_err, s), b = norm_error(s);
  return a || b;
}

void set_block_wait_bound_ns(uint64_t ns) {
  const uint64_t v = ns ? ns : tc::kWaitNs;
  CUDA_CHECK(cudaMemcpyToSymbol(tc::g_wait_ns, &v, sizeof(v)));
  norm_wait_bound(v);
}

namespace {
Operand split_weight(const GatedLinear::SplitWeight &w, int64_t rows, int64_t cols) {
  Operand o;
  o.p = w.hi;
  o.rows = rows;
  o.cols = o.ld = cols;
  o.planes = w.lo ? 2 : 1;
  o.plane = w.lo ? w.lo - w.hi : 0;
  o.scale = w.scale;
  return o;
}

}  // namespace

namespace {
FewRows few_of(const GatedLinear &a) {
  FewRows f{};
  f.dt = a.dtype;
  f.act = a.act;
  f.M = static_cast<int>(std::min<int64_t>(a.M, INT32_MAX));
  f.K = a.K;
  f.N = a.F;
  f.x = a.x.p;
  f.ldx = a.x.ld;
  f.w0 = a.wg.p;
  f.w1 = a.wv.p;
  f.ldw0 = a.wg.ld;
  f.ldw1 = a.wv.ld;
  f.b0 = a.bg;
  f.b1 = a.bv;
  f.scale = 1.f;
  return f;
}
FewRows few_of(const Linear &a) {
  FewRows f{};
  f.dt = a.dtype;
  f.act = a.act;
  f.M = static_cast<int>(std::min<int64_t>(a.M, INT32_MAX));
  f.K = a.K;
  f.N = a.N;
  f.x = a.x.p;
  f.ldx = a.x.ld;
  f.w0 = a.w.p;
  f.ldw0 = a.w.ld;
  f.b0 = a.b;
  f.scale = a.scale;
  return f;
}
void few_bwd(FewRows &f, Workspace &ws, cudaStream_t s) {
  f.dz = static_cast<float *>(ws.take(4 * few_rows_floats(f)));
  if (!ws.sizing()) few_rows_bwd(f, s);
}
}  // namespace

void gated_linear_fwd(const GatedLinear &a, Workspace &ws, cudaStream_t s) {
  if (a.M == 0) return;
  if (FewRows f = few_of(a); few_rows_fit(f)) {
    if (ws.sizing()) return;
    f.out = a.h.p;
    f.ldo = a.h.ld;
    few_rows(f, s);
    return;
  }
  Operands prep(a.dtype, ws, s);
  Product g;
  g.dt = a.dtype;
  g.epi = E_GATED;
  g.products = a.products;
  g.err = a.err;
  g.M = a.M;
  g.N = a.F;
  g.K = a.K;
  g.dual = true;
  g.a[0] = prep.add(a.x, a.M, a.K, FORM_ROWS);
  g.b[0] = a.wg_split.hi ? split_weight(a.wg_split, a.F, a.K) : prep.add(a.wg, a.F, a.K, FORM_ROWS, true);
  g.b[1] = a.wv_split.hi ? split_weight(a.wv_split, a.F, a.K) : prep.add(a.wv, a.F, a.K, FORM_ROWS, true);
  g.e = plain_out(a.h);
  g.e.act = a.act;
  g.e.b0 = a.bg;
  g.e.b1 = a.bv;
  prep.go();
  run(g, ws, s);
}

// dg = dh v act'(g) and dv = dh act(g) from the recomputed projections g and
// v (kept in neither direction: writing and reading both would cost 4 M F
// elements of traffic and memory and, in 16 bits, a rounding of each), rounded
// to the operands' type for the products that follow.
void gated_linear_bwd(const GatedLinear &a, Workspace &ws, cudaStream_t s) {
  if (a.M == 0) {
    if (ws.sizing()) return;
    zero_rows(a.dwg.p, a.dwg.ld, a.F, a.K, a.dtype, s);
    zero_rows(a.dwv.p, a.dwv.ld, a.F, a.K, a.dtype, s);
    zero_rows(a.dbg, a.F, 1, a.F, a.dtype, s);
    zero_rows(a.dbv, a.F, 1, a.F, a.dtype, s);
    return;
  }
  const bool weights = a.dwg.p || a.dwv.p;
  if (!a.dx.p && !weights && !a.dbg && !a.dbv) return;
  if (a.M <= kFewRows) {
    FewRows f = few_of(a);
    f.in = a.dh.p;
    f.ldin = a.dh.ld;
    f.dx = a.dx.p;
    f.lddx = a.dx.ld;
    f.dw0 = a.dwg.p;
    f.dw1 = a.dwv.p;
    f.lddw0 = a.dwg.ld;
    f.lddw1 = a.dwv.ld;
    f.db0 = a.dbg;
    f.db1 = a.dbv;
    few_bwd(f, ws, s);
    return;
  }
  const bool f32 = a.dtype == DT_F32;
  const size_t es = dtype_size(a.dtype);
  const int64_t fp = (a.F + 7) / 8 * 8;
  char *buf = static_cast<char *>(ws.take(2 * a.M * fp * es));
  const MutMat dz[2] = {{buf, fp}, {ws.sizing() ? nullptr : buf + a.M * fp * es, fp}};
  Operands prep(a.dtype, ws, s);
  // the weights contract their inputs for the projections, their features for
  // dx; only f32 tells the two apart
  Operand w[2], wc[2], xb;
  const Mat wm[2] = {a.wg, a.wv};
  const GatedLinear::SplitWeight *const split[2] = {&a.wg_split, &a.wv_split};
  for (int i = 0; i < 2; ++i) {
    w[i] = split[i]->hi ? split_weight(*split[i], a.F, a.K) : prep.add(wm[i], a.F, a.K, FORM_ROWS, true);
    wc[i] = f32 && a.dx.p && !split[i]->hi ? prep.add(wm[i], a.F, a.K, FORM_COLS, true) : w[i];
  }
  Product g;
  g.dt = a.dtype;
  g.products = a.products;
  g.err = a.err;
  g.a[0] = prep.add(a.x, a.M, a.K, FORM_ROWS);
  if (weights) xb = f32 ? prep.add(a.x, a.M, a.K, FORM_COLS, true) : g.a[0];
  g.epi = E_GATED_BWD;
  g.M = a.M;
  g.N = a.F;
  g.K = a.K;
  g.dual = true;
  g.b[0] = w[0];
  g.b[1] = w[1];
  g.e = plain_out(dz[0]);
  g.e.out1 = dz[1].p;
  g.e.act = a.act;
  g.e.b0 = a.bg;
  g.e.b1 = a.bv;
  g.e.in = a.dh.p;
  g.e.ldin = a.dh.ld;
  if (a.act == ACT_RELU) g.e.near = {a.x.p, a.wg.p, a.bg, a.x.ld, a.wg.ld, a.K};
  // bias gradients from the unrounded dz: 16-bit in the epilogue (each 32
  // rows), f32 where dz is split (each 128)
  void *const db[2] = {a.dbg, a.dbv};
  const int64_t strips = ceil_div(a.M, f32 ? 128 : 32);
  float *part[2] = {nullptr, nullptr};
  for (int i = 0; i < 2; ++i)
    if (db[i]) part[i] = static_cast<float *>(ws.take(4 * strips * a.F));
  if (!f32) {
    g.e.sums0 = part[0];
    g.e.sums1 = part[1];
  }
  prep.go();
  run(g, ws, s);

  const Mat m[2] = {{dz[0].p, fp}, {dz[1].p, fp}};
  void *const dw[2] = {a.dwg.p, a.dwv.p};
  const int64_t lddw[2] = {a.dwg.ld, a.dwv.ld};
  Operand rows[2], cols[2];
  for (int i = 0; i < 2; ++i) {
    if (a.dx.p) rows[i] = prep.add(m[i], a.M, a.F, FORM_ROWS);
    if (dw[i]) cols[i] = f32 || !a.dx.p ? prep.add(m[i], a.M, a.F, FORM_COLS) : rows[i];
    if (db[i] && f32) prep.sums(m[i], a.M, a.F, part[i]);
  }
  prep.go();
  if (a.dx.p) {
    Product q;
    q.dt = a.dtype;
    q.products = a.products;
    q.err = a.err;
    q.M = a.M;
    q.N = a.K;
    q.K = a.F;
    q.kcat = true;
    q.b_mn = true;
    for (int i = 0; i < 2; ++i) {
      q.a[i] = rows[i];
      q.b[i] = wc[i];
    }
    q.e = plain_out(a.dx);
    run(q, ws, s);
  }
  if (weights) {
    Product q;
    q.dt = a.dtype;
    q.products = a.products;
    q.err = a.err;
    q.M = a.F;
    q.N = a.K;
    q.K = a.M;
    q.a_mn = q.b_mn = true;
    q.b[0] = xb;
    if (dw[0] && dw[1] && lddw[0] == lddw[1]) {
      q.batch2 = true;
      q.a[0] = cols[0];
      q.a[1] = cols[1];
      q.e = plain_out(a.dwg);
      q.e.out1 = dw[1];
      run(q, ws, s);
    } else {
      for (int i = 0; i < 2; ++i) {
        if (!dw[i]) continue;
        q.a[0] = cols[i];
        q.e = plain_out(MutMat{dw[i], lddw[i]});
        run(q, ws, s);
      }
    }
  }
  for (int i = 0; i < 2; ++i)
    if (db[i] && !ws.sizing()) column_join(part[i], strips, a.F, 1.f, db[i], a.dtype, s);
}

void linear_fwd(const Linear &a, Workspace &ws, cudaStream_t s) {
  if (a.M == 0) return;
  if (FewRows f = few_of(a); few_rows_fit(f)) {
    if (ws.sizing()) return;
    f.in = a.residual.p;
    f.ldin = a.residual.ld;
    f.out = a.y.p;
    f.ldo = a.y.ld;
    few_rows(f, s);
    return;
  }
  Operands prep(a.dtype, ws, s);
  Product g;
  g.dt = a.dtype;
  g.M = a.M;
  g.N = a.N;
  g.K = a.K;
  g.a[0] = prep.add(a.x, a.M, a.K, FORM_ROWS);
  g.b[0] = prep.add(a.w, a.N, a.K, FORM_ROWS, true);
  g.e = plain_out(a.y);
  g.e.act = a.act;
  g.e.scale = a.scale;
  g.e.b0 = a.b;
  g.e.in = a.residual.p;
  g.e.ldin = a.residual.ld;
  prep.go();
  run(g, ws, s);
}

// dz = scale dy act'(z) with z recomputed; without an activation dz is dy and
// the scale goes into the products' epilogues.
void linear_bwd(const Linear &a, Workspace &ws, cudaStream_t s) {
  if (a.M == 0) {
    if (ws.sizing()) return;
    zero_rows(a.dw.p, a.dw.ld, a.N, a.K, a.dtype, s);
    zero_rows(a.db, a.N, 1, a.N, a.dtype, s);
    return;
  }
  if (!a.dx.p && !a.dw.p && !a.db) return;
  if (a.M <= kFewRows) {
    FewRows f = few_of(a);
    f.in = a.dy.p;
    f.ldin = a.dy.ld;
    f.dx = a.dx.p;
    f.lddx = a.dx.ld;
    f.dw0 = a.dw.p;
    f.lddw0 = a.dw.ld;
    f.db0 = a.db;
    few_bwd(f, ws, s);
    return;
  }
  const bool id = a.act == ACT_IDENTITY, f32 = a.dtype == DT_F32;
  Operands prep(a.dtype, ws, s);
  Operand wr, wc, xr, xb;  // as in gated_linear_bwd
  if (!id) wr = prep.add(a.w, a.N, a.K, FORM_ROWS, true);
  if (a.dx.p) wc = f32 || id ? prep.add(a.w, a.N, a.K, FORM_COLS, true) : wr;
  if (!id) xr = prep.add(a.x, a.M, a.K, FORM_ROWS);
  if (a.dw.p) xb = f32 || id ? prep.add(a.x, a.M, a.K, FORM_COLS, true) : xr;
  Mat dz = a.dy;
  // bias gradient: without an activation the sums of dy itself, else as in
  // gated_linear_bwd
  const int64_t strips = id && !f32 ? column_strips(a.M) : ceil_div(a.M, f32 ? 128 : 32);
  float *part = a.db ? static_cast<float *>(ws.take(4 * strips * a.N)) : nullptr;
  if (!id) {
    const int64_t np = (a.N + 7) / 8 * 8;
    const MutMat out{ws.take(a.M * np * dtype_size(a.dtype)), np};
    Product g;
    g.dt = a.dtype;
    g.epi = E_LINEAR_BWD;
    g.M = a.M;
    g.N = a.N;
    g.K = a.K;
    g.a[0] = xr;
    g.b[0] = wr;
    g.e = plain_out(out);
    g.e.act = a.act;
    g.e.scale = a.scale;
    g.e.b0 = a.b;
    g.e.in = a.dy.p;
    g.e.ldin = a.dy.ld;
    if (a.act == ACT_RELU) g.e.near = {a.x.p, a.w.p, a.b, a.x.ld, a.w.ld, a.K};
    if (!f32) g.e.sums0 = part;
    prep.go();
    run(g, ws, s);
    dz = Mat{out.p, np};
  }
  const float scale = id ? a.scale : 1.f;
  Operand rows, cols;
  if (a.dx.p) rows = prep.add(dz, a.M, a.N, FORM_ROWS);
  if (a.dw.p) cols = f32 || !a.dx.p ? prep.add(dz, a.M, a.N, FORM_COLS) : rows;
  if (a.db && f32) prep.sums(dz, a.M, a.N, part);
  prep.go();
  if (a.dx.p) {
    Product g;
    g.dt = a.dtype;
    g.M = a.M;
    g.N = a.K;
    g.K = a.N;
    g.b_mn = true;
    g.a[0] = rows;
    g.b[0] = wc;
    g.e = plain_out(a.dx);
    g.e.scale = scale;
    run(g, ws, s);
  }
  if (a.dw.p) {
    Product g;
    g.dt = a.dtype;
    g.M = a.N;
    g.N = a.K;
    g.K = a.M;
    g.a_mn = g.b_mn = true;
    g.a[0] = cols;
    g.b[0] = xb;
    g.e = plain_out(a.dw);
    g.e.scale = scale;
    run(g, ws, s);
  }
  if (a.db && !ws.sizing()) {
    if (id && !f32) column_sums(dz.p, a.dtype, dz.ld, a.M, a.N, part, s);
    column_join(part, strips, a.N, scale, a.db, a.dtype, s);
  }
}

}  // namespace pet
