/*
 * swarp_b200 — C ABI of the B200 (sm_100a) differentiable batched physics step.
 *
 * This is the boundary the Python layer (swarp_b200.interop / swarp_b200.core) calls
 * through ctypes. Every entry point takes plain pointers and sizes, allocates nothing,
 * launches on the caller's CUDA stream, never aborts, and returns SWARP_OK (0) or a
 * negative error code (see swarp_error_string). All device pointers address
 * contiguous row-major arrays in the dtype named by swarp_world_t.dtype.
 *
 * What each entry point replaces in the reference (ddebenedittis/swarp):
 *   swarp_rollout_fwd  -> the forward half of swarp/interop/autograd.py:341-369
 *                         (rollout: T x warp_step, each Stepper.launch_substeps at
 *                         swarp/core/stepper.py:784-1011: neighbor build
 *                         swarp/core/neighbors.py:76-97, collision_forces_kernel
 *                         swarp/core/collisions.py:818-881, obstacle_dynamics_kernel
 *                         swarp/core/bodies.py:367-569, integrate_kernel
 *                         swarp/dynamics/kernels.py:812-971)
 *   swarp_rollout_bwd  -> the backward half: _WarpStepFn.backward
 *                         swarp/interop/autograd.py:277-296 (wp.Tape.backward replay of
 *                         Warp's generated adjoints), T times in reverse
 *   swarp_neighbors    -> NeighborGrid brute build + overflow view
 *                         swarp/core/neighbors.py:76-97, 465-492, 709-714
 */
#ifndef SWARP_B200_H
#define SWARP_B200_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define SWARP_OK 0
#define SWARP_ERR_INVALID_ARG (-1)   /* null pointer, bad size or inconsistent config */
#define SWARP_ERR_UNSUPPORTED (-2)   /* model / option this build does not run       */
#define SWARP_ERR_TOO_MANY_AGENTS (-3) /* n_agents above SWARP_MAX_AGENTS            */
#define SWARP_ERR_CUDA (-4)          /* a CUDA launch or attribute call failed       */
#define SWARP_ERR_WORKSPACE (-5)     /* workspace pointer null or too small          */
#define SWARP_ERR_SCRATCH_LIMIT (-6) /* swarp_rollout_noalloc: rollout needs more workspace
                                        than SWARP_NOALLOC_SCRATCH_BYTES                 */

/* Agents per env. Envs of up to SWARP_MAX_CTA_AGENTS agents run in one CTA; larger envs
 * run one env per thread-block cluster of up to 8 CTAs (2-D disc fleets: no movable
 * bodies, box agents or drones, which return SWARP_ERR_UNSUPPORTED there). The reference
 * has no per-env agent limit (swarp/core/neighbors.py:135-254 grids any count). */
#define SWARP_MAX_AGENTS 4096
#define SWARP_MAX_CTA_AGENTS 1024
#define SWARP_NUM_PARAMS 22

/* worlds take SWARP_F32 and SWARP_F64; the 16-bit types are those of the policy operators */
typedef enum { SWARP_F32 = 0, SWARP_F64 = 1, SWARP_BF16 = 2, SWARP_F16 = 3 } swarp_dtype_t;
typedef enum { SWARP_BOUNDS_NONE = 0, SWARP_BOUNDS_SOFT = 1, SWARP_BOUNDS_CLAMP = 2 } swarp_bounds_t;

/* The five live 2-D agent fields, structure of arrays. For a state at one time the
 * shapes are pos/vel [E, A, 2] and theta/speed/ang_vel [E, A]; for a trajectory a
 * leading [T] is added. A NULL field means "absent" where the entry point says so. */
typedef struct {
  void* pos;
  void* theta;
  void* vel;
  void* speed;
  void* ang_vel;
  /* 6-DOF drone fields (swarp/core/state.py WorldState.z/vz/attitude/body_rates); read and
   * written only in worlds with drone agents (fleet_models bit 3), NULL otherwise */
  void* z;          /* [.., E, A]    */
  void* vz;         /* [.., E, A]    */
  void* attitude;   /* [.., E, A, 4] unit quaternion (x, y, z, w), body to world */
  void* body_rates; /* [.., E, A, 3] */
} swarp_state_t;

/* Obstacle set (E envs, N shapes). Poses and motion are per env, extents per shape.
 * Movable compound bodies (kind == 1) are integrated inside the substep loop. */
typedef struct {
  int32_t n_obstacles;   /* N; 0 = no obstacles (all other fields ignored) */
  const void* pos;       /* [E, N, 2] */
  const void* angle;     /* [E, N]    */
  const void* vel;       /* [E, N, 2] */
  const void* ang_vel;   /* [E, N]    */
  const void* radius;    /* [N]       */
  const void* half;      /* [N, 2]    */
  const int32_t* shape;  /* [N] 0 circle, 1 box, 2 segment */
  const int32_t* kind;   /* [N] 0 immovable, 1 movable */
  const void* mass;      /* [N] */
  const void* inertia;   /* [N] */
  const int32_t* body;   /* [N] body root index of each shape */
  const void* body_off;  /* [N, 2] shape placement in its body frame */
  int32_t any_movable;   /* 1 when any kind == 1 (host-known; selects the body pass) */
  int32_t bodies_move;   /* 0 freezes movable bodies (the reference's taped-step rule) */
  int32_t movable_shapes; /* host-known bitmask (1 << shape) over the shapes of movable
                             bodies; the adjoint differentiates circle bodies only */
  int32_t poses_from_bodies; /* 1: moving shapes start at the poses placed from the bodies'
                                initial state (a continuing rollout); 0: at the installed
                                pos/angle/vel/ang_vel (the first substep after an install) */
} swarp_obstacles_t;

/* Movable-body state per shape slot (only body-root slots are meaningful):
 * pos/vel [E, N, 2], angle/ang_vel [E, N]; a trajectory adds a leading [T]. */
typedef struct {
  void* pos;
  void* angle;
  void* vel;
  void* ang_vel;
} swarp_bodies_t;

typedef struct {
  int32_t dtype;          /* swarp_dtype_t */
  int32_t n_envs;         /* E */
  int32_t n_agents;       /* A, 1..SWARP_MAX_AGENTS */
  int32_t act_dim;        /* action slots per agent, >= 2 (slots past 2 are ignored) */
  int32_t substeps;       /* >= 1 */
  double dt;              /* env step; the substep is dt / substeps */
  int32_t collisions;     /* agent-agent contacts on/off */
  double k, c, margin, max_overlap;
  double neighbor_radius; /* R of the within-radius lists */
  int32_t max_neighbors;  /* K, list cap (first K by agent index) */
  int32_t bounds_mode;    /* swarp_bounds_t */
  double bounds[4];       /* x_min, x_max, y_min, y_max */
  double lin_damping, ang_damping; /* movable-body drag */
  const void* params;     /* [A, 22] shared, or [E, A, 22] per env */
  int64_t params_env_stride; /* elements between consecutive envs' rows; 0 = shared */
  const int32_t* model_tag;  /* [A] DynamicsModel (0..2 run here) */
  const int32_t* ctrl_mode;  /* [A] ControlMode */
  int32_t fleet_models;      /* host-known bitmask of the DynamicsModel values in model_tag */
  int32_t fleet_modes;       /* host-known bitmask of the ControlMode values in ctrl_mode */
  swarp_obstacles_t obstacles;
  int32_t integrator;        /* 0 semi-implicit Euler, 1 classic RK4 (dynamics/kernels.py:521-793) */
  int32_t box_agents;        /* host-known: some params row has shape BOX (P_SHAPE = 1); the
                                oriented-box contacts of swarp/core/collisions.py:262-690 */
} swarp_world_t;

/* The fused goal loss L = sum over envs and agents of |pos_T - goal|^2 (pos_T: the
 * positions after the last step). goal [E, A, 2] in the world's dtype, NULL = no loss.
 * swarp_rollout_fwd writes L (one scalar of the world's dtype) to `loss`, reduced in a
 * fixed order from per-CTA partials in the workspace's tail; swarp_rollout_bwd adds
 * loss_grad[0] * dL/dpos_T (loss_grad: one device scalar, dL'/dL of the caller's loss)
 * to the final-position cotangent. This is a fused fast path of the library: the
 * reference's callers form such losses in torch after the rollout. */
typedef struct {
  const void* goal;
  void* loss;             /* swarp_rollout_fwd output */
  const void* loss_grad;  /* swarp_rollout_bwd input  */
} swarp_goal_loss_t;

/* Bytes of device workspace for this world and horizon: the contact checkpoint that
 * swarp_rollout_fwd fills and swarp_rollout_bwd reads, then the adjoint's per-CTA
 * partial sums for adj_actions_sqnorm (0 for an invalid world). */
size_t swarp_rollout_workspace_bytes(const swarp_world_t* w, int32_t horizon);

/* Forward rollout of `horizon` steps from `init`.
 *   actions   [T, E, A, act_dim]
 *   traj      out: the state after every step, [T, E, A(,2)] (all five fields required)
 *   final     out (fields may be NULL): the state after the last step
 *   true_count_max  out [E, A] int32 or NULL: max over all substeps of the uncapped
 *             within-radius neighbor count (overflow <=> > max_neighbors)
 *   bodies_init / bodies_traj: movable-body state at t=0 and after every step
 *             (required only when obstacles.any_movable)
 *   goal_loss: the fused goal loss (goal NULL = none; loss required with a goal)
 *   workspace: device scratch of swarp_rollout_workspace_bytes() bytes, kept for the
 *             matching swarp_rollout_bwd call. */
int swarp_rollout_fwd(const swarp_world_t* w, int32_t horizon, swarp_state_t init,
                      const void* actions, swarp_state_t traj, swarp_state_t final_out,
                      int32_t* true_count_max, swarp_bodies_t bodies_init,
                      swarp_bodies_t bodies_traj, swarp_goal_loss_t goal_loss,
                      void* workspace, size_t workspace_bytes, void* stream);

/* Adjoint of swarp_rollout_fwd (same world, horizon, init, actions, traj, bodies and
 * workspace). Cotangents: adj_traj [T, ...] and adj_final (any field may be NULL =
 * zero), adj_bodies_final (fields may be NULL; body pos/angle/vel/ang_vel after the
 * last step). Outputs: adj_actions [T, E, A, act_dim] and adj_init (all five fields
 * required); adj_actions_sqnorm (NULL = not computed): one scalar of the world's dtype,
 * the sum of squares of adj_actions, reduced in the kernel's epilogue (the per-CTA
 * partials go to the workspace's tail) instead of a second pass over adj_actions.
 * Deterministic: no atomics, fixed summation order. Moving bodies are differentiated
 * when all their shapes are circles (SWARP_ERR_UNSUPPORTED otherwise). The fused norm
 * has no counterpart in the reference (its callers compute it from the gradient).
 * goal_loss: with a goal, loss_grad (required) seeds the goal loss's cotangent. */
int swarp_rollout_bwd(const swarp_world_t* w, int32_t horizon, swarp_state_t init,
                      const void* actions, swarp_state_t traj, swarp_state_t adj_traj,
                      swarp_state_t adj_final, swarp_bodies_t bodies_init,
                      swarp_bodies_t bodies_traj, swarp_bodies_t adj_bodies_final,
                      void* adj_actions, swarp_state_t adj_init, void* adj_actions_sqnorm,
                      swarp_goal_loss_t goal_loss, void* workspace, size_t workspace_bytes,
                      void* stream);

/* Padded within-radius neighbor lists of positions pos [E, A, 2] (brute force, ascending
 * agent index, capped at max_neighbors): idx [E, A, K] int32 (unused slots untouched),
 * count [E, A], true_count [E, A] (uncapped). */
int swarp_neighbors(const swarp_world_t* w, const void* pos, int32_t* idx, int32_t* count,
                    int32_t* true_count, void* stream);

/* Allocation-free BPTT rollout: swarp_rollout_fwd followed by swarp_rollout_bwd in one
 * call, for callers that cannot allocate device memory (a plugin under another
 * runtime's memory manager, such as an XLA/JAX custom call, must not allocate behind
 * that manager's back; a real-time control loop cannot wait on cudaMalloc, which may
 * synchronize the device). This entry point has no counterpart in the reference. The two kernels' shared
 * workspace lives in a static device array of SWARP_NOALLOC_SCRATCH_BYTES that the
 * library owns (one per GPU that loads it, held until the process exits); nothing else
 * is allocated. Arguments mean what they mean for swarp_rollout_fwd / _bwd (final_out,
 * adj_traj, adj_final fields may be NULL); movable bodies are not accepted here.
 * Returns SWARP_ERR_SCRATCH_LIMIT when swarp_rollout_workspace_bytes() exceeds
 * SWARP_NOALLOC_SCRATCH_BYTES. The first call on each device resolves the array's
 * device address (cudaGetSymbolAddress) with that device current: make it before any
 * stream capture. The address is kept for the life of the process: after a
 * cudaDeviceReset of a device, do not call this entry point on that device again. All
 * calls share the array, so calls that overlap on one GPU race on it; serialize them. */
#define SWARP_NOALLOC_SCRATCH_BYTES (16u << 20)
int swarp_rollout_noalloc(const swarp_world_t* w, int32_t horizon, swarp_state_t init,
                          const void* actions, swarp_state_t traj, swarp_state_t final_out,
                          swarp_state_t adj_traj, swarp_state_t adj_final, void* adj_actions,
                          swarp_state_t adj_init, void* stream);

/* Strided asynchronous copy of `rows` rows of `row_bytes` each, between any two of host
 * (pinned) and device memory (cudaMemcpy2DAsync, direction from the pointers), on
 * `stream`. This is host plumbing with no counterpart in the reference: it moves one env
 * slice of a [T, E, ...] array (T rows, one per step) in one call, which the streamed
 * BPTT front end (swarp_b200.interop.streamed) uses to pipeline host inputs and gradients
 * against the kernels env chunk by env chunk. */
int swarp_copy_rows(void* dst, size_t dst_pitch, const void* src, size_t src_pitch,
                    size_t row_bytes, size_t rows, void* stream);

/* ---- Policy training: what a trainer runs on the rollouts ---------------------------
 * Advantages of a rollout, the clipped policy loss with its gradient, and the AdamW step.
 * None of them has a counterpart on the reference's step path (its trainer forms them in
 * torch). All launch on `stream`, allocate nothing and are deterministic: the same inputs
 * give the same bits. */

/* A batch of rows, each a categorical distribution over `vocab` tokens given by logits, and
 * the token taken in each row. With lp the log probability of the row's token, r =
 * exp(lp - old_logp), A its advantage, d = ref_logp - lp and H the row's entropy:
 *   row loss = -min(r A, clip(r, 1 - clip_low, 1 + clip_high) A)
 *              + kl_coef (e^d - d - 1) - entropy_coef H
 * and the loss is its mean over the rows that mask admits (mean != 0) or its sum. A row
 * that mask leaves out adds nothing, whatever it holds: its logp, entropy and gradient are 0. A
 * logit of -inf is a token of probability 0; a row of nothing else has logp -inf, entropy 0
 * and no loss or gradient (it still counts). A token outside [0, vocab) gives NaN. With no
 * row admitted the loss is 0. A wait inside a launch that runs out gives a NaN loss too. */
typedef struct {
  int32_t dtype;           /* of logits and grad: SWARP_F32, SWARP_BF16 or SWARP_F16 */
  int32_t tokens_64;       /* tokens are int64 (else int32) */
  int64_t rows, vocab;     /* >= 0, >= 1 */
  /* row i of logits starts at (i / inner) * stride_outer + (i % inner) * stride_inner
   * elements; its vocab elements are adjacent */
  int64_t inner, stride_outer, stride_inner;
  const void* logits;
  const void* tokens;      /* [rows] */
  const float* old_logp;   /* [rows] */
  const float* advantages; /* [rows] */
  const float* ref_logp;   /* [rows] or NULL (no KL term) */
  const uint8_t* mask;     /* [rows], 0 = left out; or NULL */
  float clip_low, clip_high, kl_coef, entropy_coef;
  int32_t mean;
  float grad_scale;        /* grad is that of grad_scale * loss */
  float* logp;             /* out [rows] */
  float* entropy;          /* out [rows] */
  float* loss;             /* out [1] */
  float* stats;            /* out [4]: the mean (or sum) over the admitted rows of the clipped
                              term, e^d - d - 1, H and (1 where the clip cut) */
  void* grad;              /* out [rows, vocab] contiguous, or NULL */
} swarp_policy_t;

/* Bytes of device workspace of one swarp_policy_loss or swarp_policy_grad call (0 for an
 * invalid batch). */
size_t swarp_policy_workspace_bytes(const swarp_policy_t* p);

/* The loss, and with `grad` its gradient in the same pass over the logits. */
int swarp_policy_loss(const swarp_policy_t* p, void* workspace, size_t workspace_bytes,
                      void* stream);

/* The gradient alone, of cotangent[0] * grad_scale * loss (cotangent: one float on the
 * device). With skip_unit the call writes nothing when cotangent[0] is 1: `grad` then
 * holds the gradient that swarp_policy_loss left there. logp, entropy, loss and stats are
 * not used. */
int swarp_policy_grad(const swarp_policy_t* p, const float* cotangent, int32_t skip_unit,
                      void* workspace, size_t workspace_bytes, void* stream);

/* Log probabilities of the tokens and entropies alone: rows, vocab, strides, logits,
 * tokens, logp and entropy are used. */
int swarp_token_logp(const swarp_policy_t* p, void* workspace, size_t workspace_bytes,
                     void* stream);

/* Generalised advantage estimates of a rollout of `steps` steps over `columns` agents:
 *   A_t = r_t + gamma V'_t - V_t + gamma lambda A_{t+1},  returns_t = A_t + V_t
 * V'_t is next_values[t], or without it values[t + 1] (last_values after the last step); it
 * is dropped, whatever it holds, where terminated[t]. A_{t+1} is dropped where
 * terminated[t] or truncated[t]. rewards, values, next_values, advantages, returns
 * [steps, columns] and last_values [columns] are SWARP_F32 or SWARP_F64; terminated and
 * truncated are [steps, columns / columns_per_flag] bytes, or NULL. */
typedef struct {
  int32_t dtype;
  int32_t columns_per_flag; /* >= 1, divides columns */
  int64_t steps, columns;   /* >= 0 */
  const void* rewards;
  const void* values;
  const void* next_values; /* or NULL */
  const void* last_values; /* or NULL where next_values is given */
  const uint8_t* terminated;
  const uint8_t* truncated;
  double gamma, lambda;
  void* advantages;
  void* returns;
} swarp_gae_t;

/* Bytes of device workspace of the call with this very g (its addresses count: aligned columns
 * are taken several at a time); 0 where none is needed or g is invalid. */
size_t swarp_gae_workspace_bytes(const swarp_gae_t* g);
int swarp_gae(const swarp_gae_t* g, void* workspace, size_t workspace_bytes, void* stream);

/* One parameter tensor of `n` contiguous elements and its AdamW state. */
typedef struct {
  int64_t n;
  void* param;          /* swarp_adamw_t.dtype, updated */
  const void* grad;     /* the same dtype */
  float* master;        /* the parameter in 32 bits, updated; required for 16-bit dtypes
                           (param is then its rounding), NULL for SWARP_F32 */
  void* exp_avg;        /* float [n], or with 8-bit moments bytes [n] */
  void* exp_avg_sq;
  uint8_t* exp_avg_exp; /* 8-bit moments: one exponent per SWARP_MOMENT_BLOCK elements */
  uint8_t* exp_avg_sq_exp;
} swarp_adamw_tensor_t;

/* 8-bit moments are kept in blocks of SWARP_MOMENT_BLOCK elements that share one exponent
 * E, the float32 exponent field of the block's largest magnitude. With q(x) = (bits(|x|) +
 * (R << 4)) >> 20, that is the exponent and three mantissa bits of x rounded up or down at
 * random by the 16 random bits R, the first moment is a sign bit and seven bits f = q -
 * (8 E - 112), zero below f = 8, and the second moment eight bits q - (8 E - 247), at
 * least 1 where it is not zero. R is a hash of (seed, step, tensor index, element): the
 * low half word for the first moment, the high for the second. */
#define SWARP_MOMENT_BLOCK 256

typedef struct {
  int32_t dtype;        /* of param and grad: SWARP_F32, SWARP_BF16 or SWARP_F16 */
  int32_t moment_bits;  /* 32 or 8 */
  int64_t step;         /* counted from 1 */
  double lr, beta1, beta2, eps, weight_decay; /* eps below 1e-19 counts as 1e-19 */
  uint32_t seed;        /* of the 8-bit rounding */
  uint32_t first_tensor; /* index of tensors[0] in the rounding's hash */
  /* clipping: gradients are scaled by min(1, max_norm / (norm + 1e-6)) with norm the root
   * of the sum of `norm_partials`; NULL = no clipping */
  const double* norm_partials;
  int64_t n_norm_partials;
  double max_norm;
  float* grad_norm;     /* out: one float, the norm; required with norm_partials */
} swarp_adamw_t;

/* Number of doubles that swarp_grad_norm_partials writes for n_tensors tensors. */
int64_t swarp_grad_norm_partials_count(int64_t n_tensors);

/* Sums of squares of the gradients (n and grad of each entry are used), one per CTA. */
int swarp_grad_norm_partials(int32_t dtype, const swarp_adamw_tensor_t* tensors,
                             int64_t n_tensors, double* partials, void* stream);

/* One decoupled-weight-decay Adam step over all tensors (host array):
 *   m = b1 m + (1 - b1) g;  v = b2 v + (1 - b2) g^2
 *   p = p (1 - lr wd) - lr / (1 - b1^step) * m / (sqrt(v / (1 - b2^step)) + eps)
 * No two tensors may overlap. `step` is part of the launch: a captured call repeats it. */
int swarp_adamw_step(const swarp_adamw_t* opt, const swarp_adamw_tensor_t* tensors,
                     int64_t n_tensors, void* stream);

/* The values that n 8-bit moments stand for, as SWARP_F32 or SWARP_BF16 (both exact). */
int swarp_moment8_values(const uint8_t* codes, const uint8_t* exponents, int64_t n,
                         int32_t is_signed, int32_t dtype, void* out, void* stream);

/* Static description of a return code. */
const char* swarp_error_string(int code);

/* ABI version of this library (bumped on any signature change). */
int32_t swarp_abi_version(void);

#ifdef __cplusplus
}
#endif
#endif /* SWARP_B200_H */
