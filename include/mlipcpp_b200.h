/*
 * Extensions of the mlipcpp C API provided by the B200 backend.
 *
 * The reference exposes batched prediction only through C++
 * (PETModel::predict_batch, src/models/pet/pet.h:140-143); it is made
 * available to C callers here.  The remaining entry points serve
 * benchmarking and MD drivers that keep positions on the GPU.
 */
#ifndef MLIPCPP_B200_H
#define MLIPCPP_B200_H

#include "mlipcpp.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Predict a batch of independent structures in one call
 * (PETModel::predict_batch, src/models/pet/pet.cpp:125-694).  Non-periodic
 * structures are evaluated together; periodic ones one after another.
 * results[k] receives a handle that owns its data (valid until freed with
 * mlipcpp_result_free). */
mlipcpp_error_t mlipcpp_predict_batch(mlipcpp_model_t model, int32_t n_systems,
                                      const mlipcpp_system_t *systems,
                                      const mlipcpp_predict_options_t *options,
                                      mlipcpp_result_t *results);

/* The same batch from packed arrays, with the results written straight into
 * the caller's arrays (no result handles), for callers that hold many
 * structures as one block (data loaders, screening loops).  Structure k has
 * n_atoms[k] > 0 atoms; its positions ([3 n_atoms[k]] float) and atomic
 * numbers follow those of structure k - 1 in `positions` and `numbers`.
 * cells: [9 n_systems] row-major lattices, or NULL when every structure is
 * non-periodic; pbc: [3 n_systems], or NULL for periodic along all axes when
 * cells are given.  Out: energies [n_systems]; forces [3 sum n_atoms] (NULL:
 * not copied out); stress [6 n_systems], Voigt (NULL: not copied out).
 * Outputs the options do not ask for, and stress of a non-periodic
 * structure, are written as zeros. */
mlipcpp_error_t mlipcpp_b200_predict_packed(mlipcpp_model_t model, int32_t n_systems, const int32_t *n_atoms,
                                            const float *positions, const int32_t *numbers, const float *cells,
                                            const bool *pbc, const mlipcpp_predict_options_t *options,
                                            float *energies, float *forces, float *stress);

/* Predict one structure whose positions are already in device memory
 * (d_positions: device pointer to [3n] float).  atomic_numbers, cell and pbc
 * are host pointers.  Forces are copied back only when copy_forces is true.
 * Same result-handle semantics as mlipcpp_predict. */
mlipcpp_error_t mlipcpp_b200_predict_device(mlipcpp_model_t model, int32_t n_atoms,
                                            const float *d_positions,
                                            const int32_t *atomic_numbers, const float *cell,
                                            const bool *pbc,
                                            const mlipcpp_predict_options_t *options,
                                            bool copy_forces, mlipcpp_result_t *result);

/* No counterpart in the reference (its Python MD loop copies positions and
 * forces through the host each step, python/mlipcpp/ase.py:123-183).  As
 * mlipcpp_b200_predict_device, but the forces stay on the device: they are
 * written to d_forces (device, [3n] float, may be NULL) and the energy
 * (eV, composition included) to *energy; stress (host [6], Voigt, may be
 * NULL) and *has_stress (may be NULL) as in the result of
 * mlipcpp_predict_with_options.  Forces asked for from a model that cannot
 * give them (use_nc_forces without force heads, compute_forces off) return
 * MLIPCPP_ERROR_INVALID_PARAMETER when d_forces is set.  For MD drivers that
 * keep positions, velocities and forces on the GPU. */
mlipcpp_error_t mlipcpp_b200_predict_device_forces(mlipcpp_model_t model, int32_t n_atoms,
                                                   const float *d_positions, const int32_t *atomic_numbers,
                                                   const float *cell, const bool *pbc,
                                                   const mlipcpp_predict_options_t *options, float *d_forces,
                                                   double *energy, float stress[6], bool *has_stress);

/* Verlet neighbour list for repeated single-structure predictions (MD):
 * the reference builds a new list every call (PETModel::predict_batch,
 * src/models/pet/pet.cpp:125-694).  With skin > 0 (Angstrom) the list is
 * built with cutoff + skin and kept across calls, its vectors and distances
 * recomputed from the new positions, until an atom has moved more than
 * skin / 2 since the build (a move by a lattice vector along a periodic
 * axis, as when an integrator wraps positions into the cell, does not
 * count), the atom count, cell or pbc change, or a batch or another call
 * rebuilds the list.  The extra pairs lie beyond the cutoff, where the
 * smooth cutoff is 0 and the key mask -inf, like the reference's padding,
 * so results agree with fresh lists to rounding.  A kept list also keeps
 * the shapes, so the model's kernels replay from a CUDA graph.  0 (the
 * default) rebuilds every call.  A skin that is negative or not finite is
 * MLIPCPP_ERROR_INVALID_PARAMETER. */
mlipcpp_error_t mlipcpp_b200_set_neighbor_skin(mlipcpp_model_t model, float skin);

/* Neighbour lists this model has built so far (kept lists count once);
 * -1 for an invalid or unloaded model. */
int64_t mlipcpp_b200_neighbor_builds(mlipcpp_model_t model);

/* Enable per-phase CUDA-event timing of later predictions. */
mlipcpp_error_t mlipcpp_b200_set_timing(mlipcpp_model_t model, bool enable);

/* Phase times (ms) of the last prediction: h2d, neighbour list, graph prep,
 * forward, backward, reductions, d2h, total. */
mlipcpp_error_t mlipcpp_b200_last_timings(mlipcpp_model_t model, float times_ms[8]);

/* Size of the last prediction: atoms, edges, max neighbours, device bytes
 * held by the model (MiB). */
mlipcpp_error_t mlipcpp_b200_last_shape(mlipcpp_model_t model, int64_t shape[4]);

/* Full neighbour list (no self pairs) of one structure computed on the GPU,
 * bit-identical to the reference's NeighborListBuilder
 * (src/core/neighbor_list.cpp:118-297), in its enumeration order.  Host
 * pointers in and out; writes at most `cap` pairs into the (optional)
 * arrays and returns the total pair count, or -(error code) on failure, so
 * a call with cap = 0 sizes the buffers.  shifts: [3 * pairs] int32,
 * vectors: [3 * pairs] float, distances: [pairs] float. */
int64_t mlipcpp_b200_neighbor_list(int32_t n_atoms, const float *positions, const float *cell,
                                   const bool *pbc, float cutoff, int64_t cap, int32_t *centers,
                                   int32_t *neighbors, int32_t *shifts, float *vectors,
                                   float *distances);

/* No counterpart in the reference.  The periodic (or partially periodic)
 * neighbour list of mlipcpp_b200_neighbor_list, same pairs in the same
 * order, for callers that cannot let a library allocate GPU memory: an MD
 * engine or host framework that hands out every device buffer from its own
 * pool, and code running where a cudaMalloc would stall other streams or is
 * not permitted.  It allocates nothing.  `d_positions` ([3 n_atoms] float)
 * and the five pair arrays are the caller's device buffers on the calling
 * thread's current device; `cell` and `pbc` are host arrays as in
 * mlipcpp_b200_neighbor_list (cell is required).  The working memory is a
 * fixed static device array of 2.6 MB inside this library, which limits a
 * call to at most 65536 atoms and 65536 cutoff-sized bins; larger requests
 * return -MLIPCPP_ERROR_INVALID_PARAMETER with a message naming the limit,
 * before any device work; so do a cutoff that is not finite and positive,
 * one that spans more than 511 cell widths along an axis, and a list that
 * could exceed 2^31 - 1 pairs.  The first call on each device looks up that
 * array's address (cudaGetSymbolAddress), so make it before any stream
 * capture.  All calls on one device share the array, and each call clears
 * the parts that must start at zero: calls that overlap in time (from
 * several host threads or streams) race, so serialise them.
 * Work runs on `stream` (NULL: the legacy default stream).  Every call
 * copies the pair count to the host and synchronises `stream` before it
 * returns, so its work there has finished by then.  Returns the total pair
 * count; the arrays are written only when it is at most `cap` (else call
 * again with larger arrays), or -(error code) on failure. */
int64_t mlipcpp_b200_neighbor_list_noalloc(int32_t n_atoms, const float *d_positions, const float *cell,
                                           const bool *pbc, float cutoff, int64_t cap, int32_t *d_centers,
                                           int32_t *d_neighbors, int32_t *d_shifts, float *d_vectors,
                                           float *d_distances, void *stream);

/* ---- Spatial domain decomposition of one periodic cell (no counterpart in
 * the reference, which evaluates a structure on one device:
 * PETModel::predict_batch, src/models/pet/pet.cpp:125-694) ----------------
 * One rank per GPU, each with its own model.  The cell is split into
 * grid[0] x grid[1] x grid[2] fractional slabs; rank r owns slab
 * (r % g0, r / g0 % g1, r / (g0 g1)) and the atoms assigned to it.  Every
 * step: owned atoms within cutoff + skin of another slab are sent there as
 * ghosts (periodic images included); each rank runs both GNN layers and the
 * readout on its owned atoms only; a layer-1 message that needs the layer-0
 * token of an edge held by another rank gets it from that rank, and the
 * token's gradient goes back; forces on ghosts return to their owners; the
 * energy and virial are summed over the ranks.  The exchanges are the
 * caller's collectives (mlipcpp_b200_comm_t), e.g. torch.distributed over
 * NCCL: alltoallv sends rank r the send_counts[r] elements of elem_bytes
 * bytes of d_send's r-th segment and receives recv_counts[r] elements from
 * rank r into d_recv's r-th segment (segments in rank order);
 * allreduce_sum_f64 sums n doubles in place.  Buffers are device memory of
 * the model's device; both calls must be ordered on `stream` (a cudaStream_t)
 * and return 0 on success.  Every call of domain_step is collective. */
typedef struct {
  void *user;
  int32_t (*alltoallv)(void *user, const void *d_send, const int64_t *send_counts, void *d_recv,
                       const int64_t *recv_counts, int64_t elem_bytes, void *stream);
  int32_t (*allreduce_sum_f64)(void *user, double *d_buf, int64_t n, void *stream);
} mlipcpp_b200_comm_t;

typedef struct mlipcpp_b200_domain_impl *mlipcpp_b200_domain_t;

/* This rank's domain.  cell: row-major lattice of the whole cell (periodic);
 * skin: halo width beyond the cutoff (A) for atoms that moved since
 * ownership was assigned.  Returns NULL on failure (message in
 * mlipcpp_get_last_error), e.g. when a slab is not wider than twice the
 * cutoff plus skin. */
mlipcpp_b200_domain_t mlipcpp_b200_domain_create(mlipcpp_model_t model, const float cell[9],
                                                 const int32_t grid[3], int32_t rank, float skin,
                                                 const mlipcpp_b200_comm_t *comm);
void mlipcpp_b200_domain_free(mlipcpp_b200_domain_t domain);
/* The owned atoms' atomic numbers (host), in the order of the positions of
 * every step.  An unknown Z returns MLIPCPP_ERROR_COMPUTATION. */
mlipcpp_error_t mlipcpp_b200_domain_set_atoms(mlipcpp_b200_domain_t domain, int32_t n_owned,
                                              const int32_t *atomic_numbers);
/* One evaluation: d_positions [3 n_owned] f32 device; d_forces [3 n_owned]
 * f32 device (may be NULL); energy (eV, composition included) and virial
 * (Voigt xx yy zz yz xz xy, sum_e e (x) dE/de, not divided by the volume)
 * over the whole cell, on every rank. */
mlipcpp_error_t mlipcpp_b200_domain_step(mlipcpp_b200_domain_t domain, const float *d_positions,
                                         float *d_forces, bool compute_forces, double *energy,
                                         double virial[6]);
/* Last step: device ms of halo, neighbour list + requests, model (with the
 * token exchanges), reverse force halo, sum over ranks, whole step; host ms
 * of the call; then owned atoms, ghosts, edges, token rows received, token
 * rows sent, halo copies sent -> stats[0..12]. */
mlipcpp_error_t mlipcpp_b200_domain_stats(mlipcpp_b200_domain_t domain, double stats[13]);

/* ---- Transformer-block operators on device tensors -----------------------
 * No counterpart in the reference, whose layers exist only inside its graph
 * (src/models/pet/pet_layers.cpp:242-492).  The pieces of a pre-norm block
 * with a gated feed-forward part, on the caller's own device memory, forward
 * and backward: for models built or trained around the library's, and called
 * by its own PET models of that form.
 *
 * Matrices are row-major; ld* is the distance between rows in elements, at
 * least the row's length (any value where there is at most one row).  All
 * tensors of a call have the type `dtype` and lie on the calling thread's
 * current device, aligned to their elements; rows whose address and stride
 * are multiples of 16 bytes are read where they lie, others cost a copy.  A
 * call may have no rows (gradients of weights are then zeros); features are
 * at least 1, and both at most 2147482624.  Outputs must not overlap
 * inputs, but for a residual that is also the output with the same stride.
 *
 * Products accumulate in fp32; activations, norms and sums run in fp32 and
 * each output is rounded once.  f32 products from 9 rows on take their
 * operands in two halves of 22 bits together, with a scale for each row of
 * either operand (each row and column of the result) and 128 elements of the
 * sum: an element is good to 2^-22 of itself and to 2^-32 of the largest of
 * those 128, and rows and features may differ in size by any factor (results:
 * 4e-7 to 8e-7 of their norm).  An infinite element then makes its row or
 * column of a product NaN.
 *
 * A backward call recomputes what it needs from the forward's inputs;
 * gradients that enter a product are rounded to the call's type first (from 9
 * rows on; in f16 they are infinite beyond 65,504 and lost below 6e-8).  The
 * derivative of relu at 0 is 0.  Results do not depend on timing: no sum's
 * order varies.
 *
 * `workspace`: device memory of at least the bytes that the matching
 * *_workspace call gives for the same arguments, 256-byte aligned (NULL where
 * that is 0), free for reuse once the work on `stream` is done; calls that
 * may run at the same time need one each.  Work is ordered on `stream` (NULL:
 * the legacy default stream); nothing is allocated and nothing waited for, so
 * calls can be captured into a graph.  Errors found before the launch are
 * returned; mlipcpp_b200_ops_status reports a pipeline whose bounded wait
 * ran out since. */
typedef enum {
  MLIPCPP_B200_DTYPE_F32 = 0,
  MLIPCPP_B200_DTYPE_F16 = 1,
  MLIPCPP_B200_DTYPE_BF16 = 2
} mlipcpp_b200_dtype_t;

typedef enum {
  MLIPCPP_B200_ACT_IDENTITY = 0,
  MLIPCPP_B200_ACT_SIGMOID = 1,
  MLIPCPP_B200_ACT_SILU = 2,
  MLIPCPP_B200_ACT_GELU = 3,      /* z Phi(z) */
  MLIPCPP_B200_ACT_GELU_TANH = 4, /* its tanh approximation */
  MLIPCPP_B200_ACT_RELU = 5
} mlipcpp_b200_activation_t;

typedef enum {
  MLIPCPP_B200_NORM_NONE = 0,
  MLIPCPP_B200_NORM_RMS = 1,  /* x / sqrt(mean(x^2) + eps) */
  MLIPCPP_B200_NORM_LAYER = 2 /* (x - mean) / sqrt(var + eps) */
} mlipcpp_b200_norm_t;

/* h = act(x w_gate^T + b_gate) * (x w_value^T + b_value):
 * x [rows, in_features], w_gate and w_value [hidden, in_features], h and dh
 * [rows, hidden]; biases [hidden] or NULL.  Forward reads the inputs and
 * writes h; backward reads them and dh and writes each of dx, dw_gate,
 * dw_value, db_gate and db_value that is not NULL. */
typedef struct {
  int32_t dtype, activation;
  int64_t rows, in_features, hidden;
  const void *x, *w_gate, *w_value, *b_gate, *b_value;
  int64_t ldx, ldw_gate, ldw_value;
  void *h;
  int64_t ldh;
  const void *dh;
  int64_t lddh;
  void *dx, *dw_gate, *dw_value, *db_gate, *db_value;
  int64_t lddx, lddw_gate, lddw_value;
} mlipcpp_b200_gated_linear_t;
int64_t mlipcpp_b200_gated_linear_workspace(const mlipcpp_b200_gated_linear_t *args, bool backward);
mlipcpp_error_t mlipcpp_b200_gated_linear(const mlipcpp_b200_gated_linear_t *args, void *workspace,
                                          int64_t workspace_bytes, void *stream);
mlipcpp_error_t mlipcpp_b200_gated_linear_backward(const mlipcpp_b200_gated_linear_t *args, void *workspace,
                                                   int64_t workspace_bytes, void *stream);

/* y = residual + scale act(x w^T + b): x [rows, in_features], w
 * [out_features, in_features], residual (or NULL), y and dy [rows,
 * out_features], b [out_features] or NULL.  Backward writes each of dx, dw
 * and db that is not NULL (the residual's gradient is dy). */
typedef struct {
  int32_t dtype, activation;
  int64_t rows, in_features, out_features;
  float scale;
  const void *x, *w, *b, *residual;
  int64_t ldx, ldw, ldresidual;
  void *y;
  int64_t ldy;
  const void *dy;
  int64_t lddy;
  void *dx, *dw, *db;
  int64_t lddx, lddw;
} mlipcpp_b200_linear_t;
int64_t mlipcpp_b200_linear_workspace(const mlipcpp_b200_linear_t *args, bool backward);
mlipcpp_error_t mlipcpp_b200_linear(const mlipcpp_b200_linear_t *args, void *workspace, int64_t workspace_bytes,
                                    void *stream);
mlipcpp_error_t mlipcpp_b200_linear_backward(const mlipcpp_b200_linear_t *args, void *workspace,
                                             int64_t workspace_bytes, void *stream);

/* stream = scale residual + gate * post(y), out = norm(stream), on rows of
 * `features` <= 16384 elements: post and norm are none, RMS or layer norms
 * (eps > 0) with an optional weight and bias [features]; y NULL leaves
 * scale * residual; gate NULL is 1 (ldgate is not read then), ldgate 0 is one
 * row for all, else a gate for every row.  Forward writes each of stream and
 * out that is not NULL.  Backward reads residual, y and the gradients dstream
 * and dout (NULL: zero) and writes each gradient that is not NULL (dgate:
 * [features] where ldgate is 0, else rows of stride lddgate). */
typedef struct {
  int32_t dtype, norm, post_norm;
  int64_t rows, features;
  float scale, eps;
  const void *residual, *y, *weight, *bias, *post_weight, *post_bias, *gate;
  int64_t ldresidual, ldy, ldgate;
  void *stream, *out;
  int64_t ldstream, ldout;
  const void *dstream, *dout;
  int64_t lddstream, lddout;
  void *dresidual, *dy, *dweight, *dbias, *dpost_weight, *dpost_bias, *dgate;
  int64_t lddresidual, lddy, lddgate;
} mlipcpp_b200_residual_norm_t;
int64_t mlipcpp_b200_residual_norm_workspace(const mlipcpp_b200_residual_norm_t *args, bool backward);
mlipcpp_error_t mlipcpp_b200_residual_norm(const mlipcpp_b200_residual_norm_t *args, void *workspace,
                                           int64_t workspace_bytes, void *stream);
mlipcpp_error_t mlipcpp_b200_residual_norm_backward(const mlipcpp_b200_residual_norm_t *args, void *workspace,
                                                    int64_t workspace_bytes, void *stream);

/* Waits for `stream`; MLIPCPP_ERROR_COMPUTATION (once) if an operator on the
 * current device has given up a wait since the last call. */
mlipcpp_error_t mlipcpp_b200_ops_status(void *stream);

/* Number of CUDA kernels this library has launched in this process. */
int64_t mlipcpp_b200_kernel_launches(void);

/* Number of device allocations (cudaMalloc calls) this library has made in
 * this process. */
int64_t mlipcpp_b200_device_allocations(void);

/* Failure-detection test hooks (no counterpart in the reference).  Every
 * wait of the tensor-core GEMM pipelines and of the norms' rings is bounded;
 * on expiry the CTA stops (a norm: goes on without waiting), lets its own
 * copies and MMAs complete, frees its tensor memory and records a device error
 * that the call returns as MLIPCPP_ERROR_COMPUTATION (an operator: that
 * mlipcpp_b200_ops_status returns); the model stays usable.  set_wait_bound_ns
 * sets that bound on the current device (0: the default of 1 s).
 * inject_gemm_stall makes the next GEMM launch with a plain store epilogue
 * withhold the operand loads of its first CTA, inject_norm_stall the next norm
 * whose rows are aligned to 16 bytes those of its first rows, so that their
 * waits run out. */
mlipcpp_error_t mlipcpp_b200_set_wait_bound_ns(uint64_t ns);
mlipcpp_error_t mlipcpp_b200_inject_gemm_stall(void);
mlipcpp_error_t mlipcpp_b200_inject_norm_stall(void);

/* CUDA device ordinal used by models created afterwards (default: the
 * calling thread's current device). */
mlipcpp_error_t mlipcpp_b200_set_device(int32_t device);

/* Time every GEMM and attention launch with CUDA events on the model's
 * stream (also resets the statistics). */
mlipcpp_error_t mlipcpp_b200_set_kernel_profiling(mlipcpp_model_t model, bool enable);

/* Cumulative per-class statistics since profiling was enabled: for classes
 * 3xTF32 tensor-core GEMM, SIMT GEMM, attention, neighbour list, other,
 * 3xFP16 tensor-core GEMM (with its row-scale pre-pass):
 * {launches, total ms, algorithmic FLOPs, algorithmic HBM bytes}
 * -> stats[4 * class + 0..3]. */
mlipcpp_error_t mlipcpp_b200_kernel_stats(mlipcpp_model_t model, double stats[24]);

#ifdef __cplusplus
}
#endif

#endif /* MLIPCPP_B200_H */
