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
//    the whole contraction; BN = 256 (one 128 x 256 tile, two accumulators)
//    or 128 (four accumulators) when 256-wide tiles would leave SMs idle.
//  * f32: A = 2^-s (hi + lo) with one scale per row and 128 contraction
//    elements, B = 2^-t (hi + lo) with one scale per matrix (split16.cuh);
//    A_lo B_hi + A_hi B_lo + A_hi B_hi per step.  The tensor core truncates
//    when it adds to its accumulator, so every 128 contraction elements the
//    accumulator warps add the partial sum to fp32 registers with
//    round-to-nearest.
//
// Forms of a launch: `dual` (the gated projections: a tile's accumulator
// holds BN / 2 columns of x Wg^T beside the same columns of x Wv^T, so the
// epilogue has both in one thread), `kcat` (two pairs of operands along the
// contraction: dx = dg Wg + dv Wv), `batch2` (two products that share a
// shape: dWg = dg^T x, dWv = dv^T x) and `splits` (the contraction divided
// over CTAs, partial sums to the workspace and a second kernel that adds them
// in order and runs the epilogue, for outputs of few tiles).
//
// Every wait is bounded; on expiry the CTA records an error, waits for its
// own loads and MMAs, frees its tensor memory and returns.
#include <cuda.h>
#include <cudaTypedefs.h>

#include <algorithm>
#include <cmath>
#include <cstring>

#include "block.cuh"
#include "split16.cuh"
#include "tc_common.cuh"

namespace pet {

using namespace tc;

namespace blk {

namespace {

constexpr int BM = 128, BK = 64;
constexpr int kTile = BM * 128;  // bytes of 128 rows x 64 16-bit elements
constexpr int kAccWarps = 8;
constexpr int kThreads = 64 + 32 * kAccWarps;
constexpr int kStageFloats = 32 * 33;  // staging of one accumulator warp

enum Epi : int { E_LINEAR = 0, E_LINEAR_BWD = 1, E_GATED = 2, E_GATED_BWD = 3, E_PARTIAL = 4 };

// MODE: 16-bit operands (one product, planes = 1) or split-fp16 (planes = 2).
template <bool F32, int BN>
struct Cfg {
  static constexpr int Planes = F32 ? 2 : 1;
  static constexpr int BTile = BN * 128;
  static constexpr int StageBytes = Planes * (kTile + BTile);
  static constexpr int Stages = F32 ? 3 : (BN == 256 ? 4 : 6);
  static constexpr int Bufs = 512 / BN;
  static constexpr int Chunk = F32 ? 2 : 1 << 30;  // k tiles per accumulator pass
  static constexpr int BarBytes = 256;
  static constexpr int Smem = 1024 + Stages * StageBytes + kAccWarps * kStageFloats * 4 + BarBytes;
};
static_assert(Cfg<false, 256>::Smem <= 232448 && Cfg<false, 128>::Smem <= 232448 && Cfg<true, 128>::Smem <= 232448,
              "shared memory of one CTA");

struct EpiArgs {
  const void *b0, *b1;    // biases
  const void *in;         // residual (E_LINEAR) or upstream gradient (E_*_BWD)
  int64_t ldin;
  void *out0, *out1;      // out1: E_GATED_BWD's dv, batch2's second product
  int64_t ldo;
  int dt, act;
  float scale;
  bool vin, vout;         // rows movable in 16-byte pieces
  float *part;            // E_PARTIAL: [batch][split][M][nacc]
  int64_t nacc;
};

struct Params {
  int M, N;                        // output rows and columns (dual: of each half)
  int kt0, kt;                     // k tiles of the first pair of operands, of all
  int tiles_m, tiles_n, splits, kt_split, batch;
  int a_mn, b_mn, dual, bf16, products;
  const int8_t *sc[2];             // f32: scale exponents of A, [block][row]
  int64_t scld[2];
  const float *bs[2];              // f32: 2^-t of B on the device, or null
  float bsc[2];                    // ... else this
  EpiArgs e;
};

struct Maps {
  CUtensorMap a[2], b[2];
};

__device__ int g_block_err = 0;

__device__ __forceinline__ void tma3(uint32_t dst, const CUtensorMap *map, uint32_t bar, int x, int y, int z) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
      ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(x), "r"(y), "r"(z)
      : "memory");
}
__device__ __forceinline__ void expect_tx(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}

// MN-major operand of 64-row chunks, each [64 k][64 rows] in 128-byte rows:
// 8 KB between chunks, 1 KB between groups of 8 k.
__device__ __forceinline__ uint64_t mn_desc(uint32_t start) {
  return static_cast<uint64_t>((start >> 4) & 0x3FFFu) | (static_cast<uint64_t>(8192 >> 4) << 16) |
         (static_cast<uint64_t>(1024 >> 4) << 32) | (1ull << 46) | (2ull << 61);
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

// Staged 32 x 32 block -> rows row0.., columns col0.. of `out`, in 16-byte
// pieces of a row per lane.  HOW: 0 plain, 1 adds `in`, 2 multiplies by `in`.
template <typename T, int HOW>
__device__ __forceinline__ void block_out(const float *st, int lane, int row0, int col0, int M, int N, const T *in,
                                          int64_t ldin, bool vin, T *out, int64_t ldo, bool vout) {
  constexpr int V = 16 / sizeof(T), L = 32 / V;  // elements a lane, lanes a row
  if (vout && (HOW == 0 || vin)) {
    const int c = (lane % L) * V;
#pragma unroll
    for (int r0 = 0; r0 < 32; r0 += 32 / L) {
      const int r = r0 + lane / L, row = row0 + r, col = col0 + c;
      if (row >= M || col >= N) continue;
      float v[V];
#pragma unroll
      for (int j = 0; j < V; ++j) v[j] = st[r * 33 + c + j];
      const size_t io = static_cast<size_t>(row) * ldin + col, oo = static_cast<size_t>(row) * ldo + col;
      if (col + V <= N) {
        if (HOW) {
          float u[V];
          unpack<T>(*reinterpret_cast<const uint4 *>(in + io), u);  // `in` may be `out`
#pragma unroll
          for (int j = 0; j < V; ++j) v[j] = HOW == 1 ? v[j] + u[j] : v[j] * u[j];
        }
        *reinterpret_cast<uint4 *>(out + oo) = pack<T>(v);
      } else {
#pragma unroll
        for (int j = 0; j < V; ++j)
          if (col + j < N) {
            const float u = HOW ? to_f(in[io + j]) : 0.f;
            out[oo + j] = from_f<T>(HOW == 0 ? v[j] : HOW == 1 ? v[j] + u : v[j] * u);
          }
      }
    }
  } else {
    const int col = col0 + lane;
    if (col < N)
      for (int r = 0; r < 32 && row0 + r < M; ++r) {
        const float v = st[r * 33 + lane];
        const float u = HOW ? to_f(in[static_cast<size_t>(row0 + r) * ldin + col]) : 0.f;
        out[static_cast<size_t>(row0 + r) * ldo + col] = from_f<T>(HOW == 0 ? v : HOW == 1 ? v + u : v * u);
      }
  }
}

// One warp's 32 x 32 block of a tile through the epilogue.  v (and w, the
// value half of the gated forms): this lane's row, 32 consecutive columns.
template <int EPI, typename T, bool kFast>
__device__ __forceinline__ void epilogue(const Params &p, int batch, float *st, int lane, int row0, int col0,
                                         float (&v)[32], float (&w)[32]) {
  const EpiArgs &e = p.e;
  const T *in = static_cast<const T *>(e.in);
  T *out0 = static_cast<T *>(batch ? e.out1 : e.out0);
  if (e.b0) {
#pragma unroll
    for (int j = 0; j < 32; ++j) v[j] += col0 + j < p.N ? to_f(__ldg(static_cast<const T *>(e.b0) + col0 + j)) : 0.f;
  }
  if ((EPI == E_GATED || EPI == E_GATED_BWD) && e.b1) {
#pragma unroll
    for (int j = 0; j < 32; ++j) w[j] += col0 + j < p.N ? to_f(__ldg(static_cast<const T *>(e.b1) + col0 + j)) : 0.f;
  }
  with_act(e.act, [&](auto A) {
    constexpr int ACT = decltype(A)::value;
#pragma unroll
    for (int j = 0; j < 32; ++j) {
      if (EPI == E_LINEAR) {
        v[j] = act_only<ACT, kFast>(v[j]) * e.scale;
      } else if (EPI == E_GATED) {
        v[j] = act_only<ACT, kFast>(v[j]) * w[j];
      } else {
        float a, da;
        act_pair<ACT, kFast>(v[j], a, da);
        if (EPI == E_LINEAR_BWD) {
          v[j] = da * e.scale;
        } else {
          v[j] = da * w[j];
          w[j] = a;
        }
      }
    }
  });
  float *mine = st + lane * 33;
#pragma unroll
  for (int j = 0; j < 32; ++j) mine[j] = v[j];
  __syncwarp();
  if (EPI == E_LINEAR) {
    if (in) block_out<T, 1>(st, lane, row0, col0, p.M, p.N, in, e.ldin, e.vin, out0, e.ldo, e.vout);
    else block_out<T, 0>(st, lane, row0, col0, p.M, p.N, in, e.ldin, e.vin, out0, e.ldo, e.vout);
  } else if (EPI == E_GATED) {
    block_out<T, 0>(st, lane, row0, col0, p.M, p.N, in, e.ldin, e.vin, out0, e.ldo, e.vout);
  } else {
    block_out<T, 2>(st, lane, row0, col0, p.M, p.N, in, e.ldin, e.vin, out0, e.ldo, e.vout);
  }
  __syncwarp();
  if (EPI == E_GATED_BWD) {
#pragma unroll
    for (int j = 0; j < 32; ++j) mine[j] = w[j];
    __syncwarp();
    block_out<T, 2>(st, lane, row0, col0, p.M, p.N, in, e.ldin, e.vin, static_cast<T *>(e.out1), e.ldo, e.vout);
    __syncwarp();
  }
}

template <bool F32, int BN, int EPI, typename T>
__global__ void __launch_bounds__(kThreads, 1) k_block_gemm(const __grid_constant__ Maps maps, const Params p) {
  using C = Cfg<F32, BN>;
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
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                 "r"(512));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  if (tid == 0) {
    for (int s = 0; s < C::Stages; ++s) {
      mbar_init(full0 + 8 * s, 1);
      mbar_init(empty0 + 8 * s, 1);
    }
    for (int b = 0; b < C::Bufs; ++b) {
      mbar_init(accf0 + 8 * b, 1);
      mbar_init(acce0 + 8 * b, 32 * kAccWarps);
    }
    mbar_init(drain, 1);
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const int items = p.batch * p.splits * p.tiles_m * p.tiles_n;
  const int out_n = p.dual ? BN / 2 : BN;  // output columns of a tile
  const int planes = F32 ? (p.products == 1 ? 1 : 2) : 1;
  int issued = 0;

  if (warp == 0) {
    // ---------------- TMA producer ----------------
    if (lane == 0) {
      int it = 0;
      bool ok = true;
      for (int item = blockIdx.x; item < items && ok; item += gridDim.x) {
        const Item t = item_of(p, item);
        const int m0 = t.tm * BM, n0 = t.tn * out_n;
        const int k_end = min(p.kt, (t.split + 1) * p.kt_split);
        for (int kt = t.split * p.kt_split; kt < k_end; ++kt, ++it) {
          const int s = it % C::Stages;
          if (!wait_or_abort(empty0 + 8 * s, ((it / C::Stages) & 1) ^ 1, abort_flag)) {
            ok = false;
            break;
          }
          const int seg = kt >= p.kt0 ? 1 : 0, x = (kt - (seg ? p.kt0 : 0)) * BK;
          const CUtensorMap *ma = &maps.a[t.batch | seg];
          const uint32_t fb = full0 + 8 * s, st = base + s * C::StageBytes;
          expect_tx(fb, planes * (kTile + C::BTile));
          for (int z = 0; z < planes; ++z) {
            const uint32_t sa = st + z * kTile, sb = st + C::Planes * kTile + z * C::BTile;
            if (p.a_mn) {
              tma3(sa, ma, fb, m0, x, z);
              tma3(sa + 8192, ma, fb, m0 + 64, x, z);
            } else {
              tma3(sa, ma, fb, x, m0, z);
            }
            if (p.b_mn) {
              for (int c = 0; c < BN / 64; ++c) tma3(sb + 8192 * c, &maps.b[seg], fb, n0 + 64 * c, x, z);
            } else {
              // two halves of BN / 2 rows: both weights' rows n0.. (dual), or
              // 2 x BN / 2 consecutive rows
              tma3(sb, &maps.b[seg], fb, x, n0, z);
              tma3(sb + C::BTile / 2, &maps.b[p.dual ? 1 : seg], fb, x, p.dual ? n0 : n0 + BN / 2, z);
            }
          }
        }
      }
      issued = it;
    }
    __syncwarp();
  } else if (warp == 1) {
    // ---------------- MMA issuer ----------------
    if (lane == 0) {
      const uint32_t fmt = (!F32 && p.bf16) ? (1u << 7) | (1u << 10) : 0u;
      const uint32_t idesc = idesc_f16(BM, BN) | fmt | (static_cast<uint32_t>(p.a_mn) << 15) |
                             (static_cast<uint32_t>(p.b_mn) << 16);
      // one MMA step is 16 k: 32 bytes along a K-major row, 16 rows of 128
      // bytes of an MN-major chunk
      const uint32_t ka = p.a_mn ? 2048u : 32u, kb = p.b_mn ? 2048u : 32u;
      auto desc_a = [&](uint32_t a) { return p.a_mn ? mn_desc(a) : sw128_desc(a); };
      auto desc_b = [&](uint32_t a) { return p.b_mn ? mn_desc(a) : sw128_desc(a); };
      int it = 0, pass = 0;
      bool ok = true;
      for (int item = blockIdx.x; item < items && ok; item += gridDim.x) {
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
            const uint32_t sa = base + s * C::StageBytes, sb = sa + C::Planes * kTile;
#pragma unroll
            for (int kk = 0; kk < BK / 16; ++kk) {
              const uint32_t first = (kt > kt0 || kk > 0) ? 1u : 0u;
              const uint64_t ah = desc_a(sa + kk * ka), bh = desc_b(sb + kk * kb);
              if (F32 && p.products == 3) {
                mma_f16(d, desc_a(sa + kTile + kk * ka), bh, idesc, first);
                mma_f16(d, ah, desc_b(sb + C::BTile + kk * kb), idesc, 1u);
                mma_f16(d, ah, bh, idesc, 1u);
              } else {
                mma_f16(d, ah, bh, idesc, first);
              }
            }
            mma_commit(empty0 + 8 * s);
          }
          if (ok) mma_commit(accf0 + 8 * b);
          kt0 = p_end;
        }
      }
    }
    __syncwarp();
  } else {
    // ------- accumulators and epilogue: warp -> (lane quarter q, half h) -------
    // A warp's columns are two groups of BN / 4 of the accumulator: in the
    // gated forms the gate and the value of the same outputs.
    constexpr int G = BN / 4;
    const int q = warp & 3, h = (warp - 2) / 4;
    const int cb[2] = {kDual ? h * G : h * 2 * G, kDual ? BN / 2 + h * G : h * 2 * G + G};
    float *st = staging + (warp - 2) * kStageFloats;
    const uint32_t tq = tmem + (static_cast<uint32_t>(q * 32) << 16);
    int pass = 0;
    bool ok = true;
    for (int item = blockIdx.x; item < items && ok; item += gridDim.x) {
      const Item t = item_of(p, item);
      const int row0 = t.tm * BM + q * 32, row = row0 + lane, n0 = t.tn * out_n;
      const int k0 = t.split * p.kt_split, k_end = min(p.kt, k0 + p.kt_split);
      constexpr int GA = F32 ? G : 1;
      float acc[2][GA];  // f32: the running sums
      int b = 0;
      if (F32) {
#pragma unroll
        for (int gi = 0; gi < 2; ++gi)
#pragma unroll
          for (int j = 0; j < GA; ++j) acc[gi][j] = 0.f;
        for (int kt = k0; kt < k_end; kt += C::Chunk, ++pass) {
          const int seg = kt >= p.kt0 ? 1 : 0, o = t.batch | seg;
          const int blk = (kt - (seg ? p.kt0 : 0)) / C::Chunk;
          const float sa = row < p.M ? pow2f(-static_cast<int>(p.sc[o][static_cast<size_t>(blk) * p.scld[o] + row])) : 0.f;
          b = pass % C::Bufs;
          if (!__all_sync(0xffffffffu, wait_or_abort(accf0 + 8 * b, (pass / C::Bufs) & 1, abort_flag))) {
            ok = false;
            break;
          }
          tc_fence_after();
#pragma unroll
          for (int gi = 0; gi < 2; ++gi) {
            const int bi = p.dual ? (cb[gi] >= BN / 2 ? 1 : 0) : seg;
            const float f = sa * (p.bs[bi] ? __ldg(p.bs[bi]) : p.bsc[bi]);
#pragma unroll
            for (int c = 0; c < G; c += 32) {
              float v[32];
              tmem_ld32(tq + static_cast<uint32_t>(b * BN + cb[gi] + c), v);
#pragma unroll
              for (int j = 0; j < 32; ++j) acc[gi][F32 ? c + j : 0] = __fmaf_rn(v[j], f, acc[gi][F32 ? c + j : 0]);
            }
          }
          tc_fence_before();
          mbar_arrive(acce0 + 8 * b);
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
        if (F32) {
#pragma unroll
          for (int j = 0; j < 32; ++j) v[j] = acc[gi][F32 ? c + j : 0];
        } else {
          tmem_ld32(tq + static_cast<uint32_t>(b * BN + cb[gi] + c), v);
        }
      };
      auto chunk = [&](int gi, int c) {
        float v[32], w[32];
        get(gi, c, v);
        if (kDual) get(1, c, w);
        if (EPI == E_PARTIAL) {
          const int half = p.dual ? h : 0;
          const int col = n0 + cb[gi] + c - half * (BN / 2);
          if (col >= p.N) return;
          float *mine = st + lane * 33;
#pragma unroll
          for (int j = 0; j < 32; ++j) mine[j] = v[j];
          __syncwarp();
          float *dst = p.e.part + (static_cast<size_t>(t.batch) * p.splits + t.split) * p.M * p.e.nacc + half * p.N;
          block_out<float, 0>(st, lane, row0, col, p.M, p.N, nullptr, 0, true, dst, p.e.nacc, p.e.vout);
          __syncwarp();
        } else {
          const int col = n0 + (kDual ? h * G : cb[gi]) + c;
          if (col >= p.N || row0 >= p.M) return;
          epilogue<EPI, T, !F32>(p, t.batch, st, lane, row0, col, v, w);
        }
      };
      if (F32) {  // register arrays: constant indices
#pragma unroll
        for (int gi = 0; gi < (kDual ? 1 : 2); ++gi)
#pragma unroll
          for (int c = 0; c < G; c += 32) chunk(gi, c);
      } else {
#pragma unroll 1
        for (int i = 0; i < (kDual ? 1 : 2) * G; i += 32) chunk(i / G, i % G);
        tc_fence_before();
        mbar_arrive(acce0 + 8 * b);
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (*abort_flag) {
    // this CTA's own loads and MMAs complete before it ends
    if (warp == 0 && lane == 0)
      for (int j = issued > C::Stages ? issued - C::Stages : 0; j < issued; ++j)
        wait_bounded(full0 + 8 * (j % C::Stages), (j / C::Stages) & 1);
    if (warp == 1 && lane == 0) {
      mma_commit(drain);
      wait_bounded(drain, 0);
    }
    __syncthreads();
    if (tid == 0) atomicExch(&g_block_err, 1);
  }
  if (warp == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512));
}

// Sums the partial products of a split launch in order and runs the epilogue.
template <int EPI, typename T>
__global__ void __launch_bounds__(256) k_join(const Params p) {
  const EpiArgs &e = p.e;
  const int64_t per = static_cast<int64_t>(p.M) * p.N, all = per * p.batch;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < all; i += static_cast<int64_t>(gridDim.x) * 256) {
    const int batch = static_cast<int>(i / per);
    const int64_t j = i - batch * per, row = j / p.N, col = j - row * p.N;
    const float *src = e.part + static_cast<size_t>(batch) * p.splits * p.M * e.nacc + row * e.nacc + col;
    const size_t step = static_cast<size_t>(p.M) * e.nacc;
    float v = 0.f, w = 0.f;
    for (int s = 0; s < p.splits; ++s) v += src[s * step];
    if (p.dual)
      for (int s = 0; s < p.splits; ++s) w += src[s * step + p.N];
    if (e.b0) v += to_f(static_cast<const T *>(e.b0)[col]);
    if (p.dual && e.b1) w += to_f(static_cast<const T *>(e.b1)[col]);
    const float in = e.in ? to_f(static_cast<const T *>(e.in)[row * e.ldin + col]) : 0.f;
    T *o = static_cast<T *>(batch ? e.out1 : e.out0) + row * e.ldo + col;
    with_act(e.act, [&](auto A) {
      constexpr int ACT = decltype(A)::value;
      constexpr bool kFast = sizeof(T) == 2;
      float a, da;
      act_pair<ACT, kFast>(v, a, da);
      if (EPI == E_LINEAR) *o = from_f<T>(a * e.scale + in);
      else if (EPI == E_LINEAR_BWD) *o = from_f<T>(da * e.scale * in);
      else if (EPI == E_GATED) *o = from_f<T>(a * w);
      else {
        *o = from_f<T>(da * w * in);
        static_cast<T *>(e.out1)[row * e.ldo + col] = from_f<T>(a * in);
      }
    });
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

// f32 rows -> split form with one scale per row and 128 columns; warp per
// (row, block).  Columns past C are written as zeros up to the block's end.
__global__ void __launch_bounds__(256) k_split_rows(const float *__restrict__ src, int64_t ld, int R, int C, bool vec,
                                                    Split16View o) {
  const int nb = o.cols / 128, lane = threadIdx.x & 31;
  const int64_t n = static_cast<int64_t>(R) * nb, step = static_cast<int64_t>(gridDim.x) * 8;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5); i < n; i += step) {
    const int row = static_cast<int>(i / nb), blk = static_cast<int>(i - static_cast<int64_t>(row) * nb);
    const int c = blk * 128 + lane * 4;
    const float *p = src + static_cast<size_t>(row) * ld + c;
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    if (vec && c + 4 <= C) {
      v = __ldg(reinterpret_cast<const float4 *>(p));
    } else {
      if (c < C) v.x = p[0];
      if (c + 1 < C) v.y = p[1];
      if (c + 2 < C) v.z = p[2];
      if (c + 3 < C) v.w = p[3];
    }
    float mx = fmaxf(fmaxf(finite_abs(v.x), finite_abs(v.y)), fmaxf(finite_abs(v.z), finite_abs(v.w)));
    const int s = split_scale_exponent(warp_max(mx));
    const float f = pow2f(s);
    uint32_t h0, h1, l0, l1;
    split2(v.x, v.y, f, h0, l0);
    split2(v.z, v.w, f, h1, l1);
    const size_t off = static_cast<size_t>(row) * o.cols + c;
    *reinterpret_cast<uint2 *>(o.hi + off) = make_uint2(h0, h1);
    *reinterpret_cast<uint2 *>(o.lo + off) = make_uint2(l0, l1);
    if (lane == 0) o.sc[static_cast<size_t>(blk) * split_ld(o) + row] = static_cast<int8_t>(s);
  }
}

// f32 [R, C] -> split form in the same layout [R, cp] (cp a multiple of 64)
// with one scale per column and 128 rows (scales [row block][column]): the A
// operand of a product that contracts over rows.  CTA: 128 rows x 64 columns
// at a time.
__global__ void __launch_bounds__(256) k_split_cols(const float *__restrict__ src, int64_t ld, int R, int C,
                                                    uint16_t *hi, uint16_t *lo, int cp, int8_t *sc) {
  __shared__ float mx[8][64];
  const int w = threadIdx.x >> 5, lane = threadIdx.x & 31, c = blockIdx.x * 64 + 2 * lane;
  for (int blk = blockIdx.y; blk * 128 < R; blk += gridDim.y) {
    const int r0 = blk * 128 + w * 16;
    float a[16], b[16], ma = 0.f, mb = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const bool in = r0 + i < R;
      const float *p = src + static_cast<size_t>(r0 + i) * ld + c;
      a[i] = in && c < C ? p[0] : 0.f;
      b[i] = in && c + 1 < C ? p[1] : 0.f;
      ma = fmaxf(ma, finite_abs(a[i]));
      mb = fmaxf(mb, finite_abs(b[i]));
    }
    __syncthreads();  // the last block's maxima have been read
    mx[w][2 * lane] = ma;
    mx[w][2 * lane + 1] = mb;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      ma = fmaxf(ma, mx[i][2 * lane]);
      mb = fmaxf(mb, mx[i][2 * lane + 1]);
    }
    const int sa = split_scale_exponent(ma), sb = split_scale_exponent(mb);
    if (w == 0) {
      sc[static_cast<size_t>(blk) * cp + c] = static_cast<int8_t>(sa);
      sc[static_cast<size_t>(blk) * cp + c + 1] = static_cast<int8_t>(sb);
    }
    const float fa = pow2f(sa), fb = pow2f(sb);
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      if (r0 + i >= R) continue;
      uint32_t ha, la, hb, lb;
      split2(a[i], 0.f, fa, ha, la);
      split2(b[i], 0.f, fb, hb, lb);
      const size_t off = static_cast<size_t>(r0 + i) * cp + c;
      *reinterpret_cast<uint32_t *>(hi + off) = (ha & 0xffffu) | (hb << 16);
      *reinterpret_cast<uint32_t *>(lo + off) = (la & 0xffffu) | (lb << 16);
    }
  }
}

// Largest finite |element| as fp32 bits (ordered like the values, so an
// integer maximum, whose result does not depend on the order).
__global__ void __launch_bounds__(256) k_absmax(const float *__restrict__ src, int64_t ld, int64_t R, int64_t C,
                                                unsigned *out) {
  unsigned m = 0;
  const int64_t n = R * C;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < n; i += static_cast<int64_t>(gridDim.x) * 256) {
    const int64_t r = i / C;
    const unsigned u = __float_as_uint(src[r * ld + (i - r * C)]) & 0x7fffffffu;
    if (u < 0x7f800000u) m = max(m, u);
  }
#pragma unroll
  for (int k = 16; k > 0; k >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, k));
  if ((threadIdx.x & 31) == 0 && m) atomicMax(out, m);
}

// f32 [R, C] -> split form [R, cp] with the scale of *mx; writes 2^-s.
__global__ void __launch_bounds__(256) k_split_whole(const float *__restrict__ src, int64_t ld, int64_t R, int C, int cp,
                                                     const unsigned *mx, uint16_t *hi, uint16_t *lo, float *inv) {
  const int s = split_scale_exponent(__uint_as_float(*mx));
  const float f = pow2f(s);
  const int64_t nc = cp / 2, n = R * nc;
  const int64_t i0 = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (i0 == 0) *inv = pow2f(-s);
  for (int64_t i = i0; i < n; i += static_cast<int64_t>(gridDim.x) * 256) {
    const int64_t r = i / nc;
    const int c = static_cast<int>(i - r * nc) * 2;
    const float *p = src + r * ld + c;
    uint32_t h, l;
    split2(c < C ? p[0] : 0.f, c + 1 < C ? p[1] : 0.f, f, h, l);
    *reinterpret_cast<uint32_t *>(hi + r * cp + c) = h;
    *reinterpret_cast<uint32_t *>(lo + r * cp + c) = l;
  }
}

// 16-bit rows whose address or stride TMA cannot take -> rows of cp elements.
__global__ void __launch_bounds__(256) k_pack(const uint16_t *__restrict__ src, int64_t ld, int64_t R, int C, int cp,
                                              uint16_t *dst) {
  const int64_t nc = cp / 2, n = R * nc;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < n; i += static_cast<int64_t>(gridDim.x) * 256) {
    const int64_t r = i / nc;
    const int c = static_cast<int>(i - r * nc) * 2;
    const uint32_t a = c < C ? src[r * ld + c] : 0u, b = c + 1 < C ? src[r * ld + c + 1] : 0u;
    *reinterpret_cast<uint32_t *>(dst + r * cp + c) = a | (b << 16);
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
  int64_t plane = 0;            // elements between hi and lo
  const int8_t *sc = nullptr;   // f32 A: scales [block][row]
  int64_t scld = 0;
  const float *bs = nullptr;    // f32 B: 2^-s on the device
  float bsc = 1.f;
};

Operand from_split(const Split16View &v) {
  Operand o;
  o.p = v.hi;
  o.rows = v.rows;
  o.cols = o.ld = v.cols;
  o.planes = v.lo ? 2 : 1;
  o.plane = v.lo ? v.lo - v.hi : 0;
  o.sc = v.sc;
  o.scld = split_ld(v);
  return o;
}

Operand packed(const Mat &m, int64_t rows, int64_t cols, int dt, Workspace &ws, cudaStream_t s) {
  Operand o;
  o.rows = rows;
  o.cols = cols;
  if (rows16(m.p, m.ld, dt)) {
    o.p = static_cast<const uint16_t *>(m.p);
    o.ld = m.ld;
    return o;
  }
  o.ld = (cols + 7) / 8 * 8;
  uint16_t *d = static_cast<uint16_t *>(ws.take(2 * rows * o.ld));
  o.p = d;
  if (!ws.sizing()) {
    k_pack<<<grid_for(rows * o.ld / 2), 256, 0, s>>>(static_cast<const uint16_t *>(m.p), m.ld, rows,
                                                     static_cast<int>(cols), static_cast<int>(o.ld), d);
    CUDA_LAUNCH_CHECK();
  }
  return o;
}

// A operand.  over_rows: the product contracts over the matrix's rows.
Operand operand_a(const Mat &m, int64_t rows, int64_t cols, int dt, bool over_rows, Workspace &ws, cudaStream_t s) {
  if (dt != DT_F32) return packed(m, rows, cols, dt, ws, s);
  Operand o;
  o.rows = rows;
  o.cols = cols;
  o.ld = (cols + 127) / 128 * 128;
  o.planes = 2;
  o.plane = rows * o.ld;
  uint16_t *d = static_cast<uint16_t *>(ws.take(4 * rows * o.ld));
  const int64_t nblk = over_rows ? (rows + 127) / 128 : o.ld / 128;
  o.scld = over_rows ? o.ld : rows;
  int8_t *sc = static_cast<int8_t *>(ws.take(nblk * o.scld));
  o.p = d;
  o.sc = sc;
  if (ws.sizing()) return o;
  const float *src = static_cast<const float *>(m.p);
  if (over_rows) {
    const dim3 grid(static_cast<unsigned>(o.ld / 64), static_cast<unsigned>(std::min<int64_t>(nblk, 65535)));
    k_split_cols<<<grid, 256, 0, s>>>(src, m.ld, static_cast<int>(rows), static_cast<int>(cols), d, d + o.plane,
                                      static_cast<int>(o.ld), sc);
  } else {
    Split16View v;
    v.hi = d;
    v.lo = d + o.plane;
    v.sc = sc;
    v.rows = static_cast<int>(rows);
    v.cols = static_cast<int>(o.ld);
    k_split_rows<<<grid_for(rows * (o.ld / 128) * 32), 256, 0, s>>>(src, m.ld, static_cast<int>(rows),
                                                                    static_cast<int>(cols), rows16(m.p, m.ld, dt), v);
  }
  CUDA_LAUNCH_CHECK();
  return o;
}

// B operand (either way round).
Operand operand_b(const Mat &m, int64_t rows, int64_t cols, int dt, Workspace &ws, cudaStream_t s) {
  if (dt != DT_F32) return packed(m, rows, cols, dt, ws, s);
  Operand o;
  o.rows = rows;
  o.cols = cols;
  o.ld = (cols + 7) / 8 * 8;
  o.planes = 2;
  o.plane = rows * o.ld;
  uint16_t *d = static_cast<uint16_t *>(ws.take(4 * rows * o.ld));
  unsigned *word = static_cast<unsigned *>(ws.take(8));
  o.p = d;
  o.bs = reinterpret_cast<const float *>(word + 1);
  if (ws.sizing()) return o;
  CUDA_CHECK(cudaMemsetAsync(word, 0, 4, s));
  const float *src = static_cast<const float *>(m.p);
  k_absmax<<<grid_for(rows * cols), 256, 0, s>>>(src, m.ld, rows, cols, word);
  CUDA_LAUNCH_CHECK();
  k_split_whole<<<grid_for(rows * o.ld / 2), 256, 0, s>>>(src, m.ld, rows, static_cast<int>(cols),
                                                          static_cast<int>(o.ld), word, d, d + o.plane,
                                                          reinterpret_cast<float *>(word + 1));
  CUDA_LAUNCH_CHECK();
  return o;
}

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
  int64_t M = 0, N = 0, K = 0;  // K: contraction of each pair of operands
  Operand a[2], b[2];
  bool a_mn = false, b_mn = false, dual = false, kcat = false, batch2 = false;
  EpiArgs e{};
};

template <bool F32, int BN, int EPI, typename T>
void launch(const Maps &maps, const Params &p, cudaStream_t s) {
  constexpr int smem = Cfg<F32, BN>::Smem;
  CUDA_CHECK(cudaFuncSetAttribute(k_block_gemm<F32, BN, EPI, T>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
  const int items = p.batch * p.splits * p.tiles_m * p.tiles_n;
  k_block_gemm<F32, BN, EPI, T><<<std::min(items, sm_count()), kThreads, smem, s>>>(maps, p);
  CUDA_LAUNCH_CHECK();
}
template <int EPI>
void launch_epi(int dt, int bn, const Maps &maps, const Params &p, cudaStream_t s) {
  if (dt == DT_F32) launch<true, 128, EPI, float>(maps, p, s);
  else if (dt == DT_F16 && bn == 256) launch<false, 256, EPI, __half>(maps, p, s);
  else if (dt == DT_F16) launch<false, 128, EPI, __half>(maps, p, s);
  else if (bn == 256) launch<false, 256, EPI, __nv_bfloat16>(maps, p, s);
  else launch<false, 128, EPI, __nv_bfloat16>(maps, p, s);
}
template <int EPI>
void join_epi(int dt, const Params &p, cudaStream_t s) {
  const int g = grid_for(static_cast<int64_t>(p.M) * p.N * p.batch);
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
  p.e = g.e;
  p.e.dt = g.dt;
  auto count = [&](int bn) {
    const int64_t tn = (g.N + (g.dual ? bn / 2 : bn) - 1) / (g.dual ? bn / 2 : bn);
    return (g.M + BM - 1) / BM * tn * p.batch;
  };
  // 256-wide tiles read a third less shared memory for a product, as long as
  // they still give every SM a tile
  const int bn = !f32 && count(256) >= sms ? 256 : 128;
  const int64_t tiles = count(bn);
  p.tiles_m = static_cast<int>((g.M + BM - 1) / BM);
  p.tiles_n = static_cast<int>(tiles / p.tiles_m / p.batch);
  // few tiles and a long contraction: divided over the SMs, at least four k
  // tiles each
  int splits = 1;
  if (tiles * 2 <= sms && p.kt >= 8) splits = static_cast<int>(std::min<int64_t>(sms / tiles, p.kt / 4));
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
    maps.b[i] = map_of(b, bf, g.b_mn ? 64 : bn / 2);
    q.sc[i] = a.sc;
    q.scld[i] = a.scld;
    q.bs[i] = b.bs;
    q.bsc[i] = b.bsc;
  }
  if (splits > 1) {
    launch_epi<E_PARTIAL>(g.dt, bn, maps, q, s);
    switch (g.epi) {
      case E_LINEAR: join_epi<E_LINEAR>(g.dt, p, s); break;
      case E_LINEAR_BWD: join_epi<E_LINEAR_BWD>(g.dt, p, s); break;
      case E_GATED: join_epi<E_GATED>(g.dt, p, s); break;
      default: join_epi<E_GATED_BWD>(g.dt, p, s); break;
    }
    return;
  }
  switch (g.epi) {
    case E_LINEAR: launch_epi<E_LINEAR>(g.dt, bn, maps, q, s); break;
    case E_LINEAR_BWD: launch_epi<E_LINEAR_BWD>(g.dt, bn, maps, q, s); break;
    case E_GATED: launch_epi<E_GATED>(g.dt, bn, maps, q, s); break;
    default: launch_epi<E_GATED_BWD>(g.dt, bn, maps, q, s); break;
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

}  // namespace blk

using namespace blk;

void *Workspace::take(size_t bytes) {
  const size_t b = (bytes + 255) / 256 * 256;
  void *p = base ? base + off : nullptr;
  off += b;
  if (base && off > cap) throw Error(kErrInvalidParameter, "the workspace is too small");
  return p;
}

int block_status(cudaStream_t s) {
  int v = 0;
  CUDA_CHECK(cudaMemcpyFromSymbolAsync(&v, g_block_err, sizeof(v), 0, cudaMemcpyDeviceToHost, s));
  CUDA_CHECK(cudaStreamSynchronize(s));
  if (v) {
    const int zero = 0;
    CUDA_CHECK(cudaMemcpyToSymbolAsync(g_block_err, &zero, sizeof(zero), 0, cudaMemcpyHostToDevice, s));
    CUDA_CHECK(cudaStreamSynchronize(s));
  }
  return v;
}

namespace {
Operand split_weight(const GatedLinear::SplitWeight &w, int64_t rows, int64_t cols) {
  Operand o;
  o.p = w.hi;
  o.rows = rows;
  o.cols = o.ld = cols;
  o.planes = w.lo ? 2 : 1;
  o.plane = w.lo ? w.lo - w.hi : 0;
  o.bsc = std::ldexp(1.f, -w.scale);
  return o;
}
}  // namespace

void gated_linear_fwd(const GatedLinear &a, Workspace &ws, cudaStream_t s) {
  if (a.M == 0) return;
  if (a.M <= kFewRows && !a.x_split) {
    if (ws.sizing()) return;
    FewRows f{a.dtype, a.act, static_cast<int>(a.M), a.K, a.F, a.x.p, a.wg.p, a.wv.p, a.x.ld, a.wg.ld, a.wv.ld,
              a.bg, a.bv, nullptr, 0, 1.f, a.h.p, a.h.ld};
    few_rows(f, s);
    return;
  }
  Product g;
  g.dt = a.dtype;
  g.epi = E_GATED;
  g.products = a.products;
  g.M = a.M;
  g.N = a.F;
  g.K = a.K;
  g.dual = true;
  g.a[0] = a.x_split ? from_split(*a.x_split) : operand_a(a.x, a.M, a.K, a.dtype, false, ws, s);
  g.b[0] = a.wg_split.hi ? split_weight(a.wg_split, a.F, a.K) : operand_b(a.wg, a.F, a.K, a.dtype, ws, s);
  g.b[1] = a.wv_split.hi ? split_weight(a.wv_split, a.F, a.K) : operand_b(a.wv, a.F, a.K, a.dtype, ws, s);
  g.e = plain_out(a.h);
  g.e.act = a.act;
  g.e.b0 = a.bg;
  g.e.b1 = a.bv;
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
  if (!a.dx.p && !a.dwg.p && !a.dwv.p && !a.dbg && !a.dbv) return;
  const size_t es = dtype_size(a.dtype);
  const int64_t fp = (a.F + 7) / 8 * 8;
  MutMat dz{ws.take(2 * a.M * fp * es), fp}, dzv{ws.sizing() ? nullptr : static_cast<char *>(dz.p) + a.M * fp * es, fp};
  const Operand wg = a.wg_split.hi ? split_weight(a.wg_split, a.F, a.K) : operand_b(a.wg, a.F, a.K, a.dtype, ws, s);
  const Operand wv = a.wv_split.hi ? split_weight(a.wv_split, a.F, a.K) : operand_b(a.wv, a.F, a.K, a.dtype, ws, s);
  {
    Product g;
    g.dt = a.dtype;
    g.epi = E_GATED_BWD;
    g.products = a.products;
    g.M = a.M;
    g.N = a.F;
    g.K = a.K;
    g.dual = true;
    g.a[0] = a.x_split ? from_split(*a.x_split) : operand_a(a.x, a.M, a.K, a.dtype, false, ws, s);
    g.b[0] = wg;
    g.b[1] = wv;
    g.e = plain_out(dz);
    g.e.out1 = dzv.p;
    g.e.act = a.act;
    g.e.b0 = a.bg;
    g.e.b1 = a.bv;
    g.e.in = a.dh.p;
    g.e.ldin = a.dh.ld;
    run(g, ws, s);
  }
  const Mat mg{dz.p, fp}, mv{dzv.p, fp};
  if (a.dx.p) {
    Product g;
    g.dt = a.dtype;
    g.products = a.products;
    g.M = a.M;
    g.N = a.K;
    g.K = a.F;
    g.kcat = true;
    g.b_mn = true;
    g.a[0] = operand_a(mg, a.M, a.F, a.dtype, false, ws, s);
    g.a[1] = operand_a(mv, a.M, a.F, a.dtype, false, ws, s);
    g.b[0] = wg;
    g.b[1] = wv;
    g.e = plain_out(a.dx);
    run(g, ws, s);
  }
  if (a.dwg.p || a.dwv.p) {
    Product g;
    g.dt = a.dtype;
    g.products = a.products;
    g.M = a.F;
    g.N = a.K;
    g.K = a.M;
    g.a_mn = g.b_mn = true;
    g.b[0] = operand_b(a.x, a.M, a.K, a.dtype, ws, s);
    const bool both = a.dwg.p && a.dwv.p;
    g.a[0] = operand_a(a.dwg.p ? mg : mv, a.M, a.F, a.dtype, true, ws, s);
    g.e = plain_out(a.dwg.p ? a.dwg : a.dwv);
    if (both && a.dwg.ld == a.dwv.ld) {
      g.batch2 = true;
      g.a[1] = operand_a(mv, a.M, a.F, a.dtype, true, ws, s);
      g.e.out1 = a.dwv.p;
      run(g, ws, s);
    } else {
      run(g, ws, s);
      if (both) {
        g.a[0] = operand_a(mv, a.M, a.F, a.dtype, true, ws, s);
        g.e = plain_out(a.dwv);
        run(g, ws, s);
      }
    }
  }
  for (int i = 0; i < 2; ++i) {
    void *db = i ? a.dbv : a.dbg;
    if (!db) continue;
    float *part = static_cast<float *>(ws.take(4 * column_sum_floats(a.M, a.F)));
    if (!ws.sizing()) column_sum(i ? mv.p : mg.p, a.dtype, fp, a.M, a.F, 1.f, db, a.dtype, part, s);
  }
}

void linear_fwd(const Linear &a, Workspace &ws, cudaStream_t s) {
  if (a.M == 0) return;
  if (a.M <= kFewRows) {
    if (ws.sizing()) return;
    FewRows f{a.dtype, a.act, static_cast<int>(a.M), a.K, a.N, a.x.p, a.w.p, nullptr, a.x.ld, a.w.ld, 0, a.b, nullptr,
              a.residual.p, a.residual.ld, a.scale, a.y.p, a.y.ld};
    few_rows(f, s);
    return;
  }
  Product g;
  g.dt = a.dtype;
  g.M = a.M;
  g.N = a.N;
  g.K = a.K;
  g.a[0] = operand_a(a.x, a.M, a.K, a.dtype, false, ws, s);
  g.b[0] = operand_b(a.w, a.N, a.K, a.dtype, ws, s);
  g.e = plain_out(a.y);
  g.e.act = a.act;
  g.e.scale = a.scale;
  g.e.b0 = a.b;
  g.e.in = a.residual.p;
  g.e.ldin = a.residual.ld;
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
  const bool id = a.act == ACT_IDENTITY;
  Operand w;
  if (!id || a.dx.p) w = operand_b(a.w, a.N, a.K, a.dtype, ws, s);
  Mat dz = a.dy;
  if (!id) {
    const int64_t np = (a.N + 7) / 8 * 8;
    MutMat out{ws.take(a.M * np * dtype_size(a.dtype)), np};
    Product g;
    g.dt = a.dtype;
    g.epi = E_LINEAR_BWD;
    g.M = a.M;
    g.N = a.N;
    g.K = a.K;
    g.a[0] = operand_a(a.x, a.M, a.K, a.dtype, false, ws, s);
    g.b[0] = w;
    g.e = plain_out(out);
    g.e.act = a.act;
    g.e.scale = a.scale;
    g.e.b0 = a.b;
    g.e.in = a.dy.p;
    g.e.ldin = a.dy.ld;
    run(g, ws, s);
    dz = Mat{out.p, np};
  }
  const float scale = id ? a.scale : 1.f;
  if (a.dx.p) {
    Product g;
    g.dt = a.dtype;
    g.M = a.M;
    g.N = a.K;
    g.K = a.N;
    g.b_mn = true;
    g.a[0] = operand_a(dz, a.M, a.N, a.dtype, false, ws, s);
    g.b[0] = w;
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
    g.a[0] = operand_a(dz, a.M, a.N, a.dtype, true, ws, s);
    g.b[0] = operand_b(a.x, a.M, a.K, a.dtype, ws, s);
    g.e = plain_out(a.dw);
    g.e.scale = scale;
    run(g, ws, s);
  }
  if (a.db) {
    float *part = static_cast<float *>(ws.take(4 * column_sum_floats(a.M, a.N)));
    if (!ws.sizing()) column_sum(dz.p, a.dtype, dz.ld, a.M, a.N, scale, a.db, a.dtype, part, s);
  }
}

}  // namespace pet
