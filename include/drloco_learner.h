/*
 * drloco_learner.h -- C-ABI of the learner-side operators (drloco_amd/csrc/libdrloco_learner.so).
 *
 * The rollout side of the library (drloco_hip.h) produces time-major buffers [T, N, ...] with episode-start flags; the
 * entry points here are what a learner runs over them next to dl_gae: the gated memory of a recurrent policy with its
 * gradients, and the orthogonalised weight update of its matrices.  Conventions as in drloco_hip.h:
 *
 *   - plain C, no exceptions across the boundary; 0 on success or a negative DL_E_* code, dl_learner_last_error()
 *     returns the text of the last failure on the calling thread;
 *   - array pointers are DEVICE pointers of the current device, owned by the caller; work is enqueued on `stream`
 *     (a hipStream_t as void*, NULL = the null stream), nothing synchronises with the host, nothing is allocated;
 *   - no handle and no state between calls: two calls may run at the same time if their outputs and workspaces differ;
 *   - every call may be captured into a HIP graph (kernels only, no memset or copy nodes).
 */
#ifndef DRLOCO_LEARNER_H
#define DRLOCO_LEARNER_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define DL_LEARNER_ABI_VERSION 1

#ifndef DRLOCO_HIP_H   /* the same codes as drloco_hip.h */
#define DL_OK 0
#define DL_E_INVAL (-1)
#define DL_E_HIP (-3)
#endif

/* element types */
#define DL_F32 0
#define DL_BF16 1
#define DL_F16 2

const char* dl_learner_last_error(void);
int dl_learner_abi_version(void);

/* ---- gated memory -----------------------------------------------------------------------------------------------
 * For every walker n and channel d, over the control steps t = 0 .. T-1 of a rollout:
 *
 *     a[t] = sigmoid(gate[t])
 *     h[t] = a[t] * (starts[t] ? 0 : h[t-1]) + (1 - a[t]) * x[t],        h[-1] = state (NULL: zeros)
 *
 * starts: uint8 [T, N], nonzero = an episode begins at t and nothing of the memory before it is read (a NaN or an
 * infinity there does not leak; within an episode an infinity leaves its channel infinite or NaN until the next one begins); NULL: none.  Elements of x, gate, h and of the gradients have `dtype`; states, sums and
 * gradients of states are float.  Strides are in elements, for the first two axes; the last axis is contiguous; a stride
 * of 0 (a broadcast input) is allowed for inputs.  h, dx and dgate are contiguous [T, N, D], states [N, D]. */
typedef struct dl_memory_shape {
    int64_t T, N, D;
    int64_t x_t, x_n;             /* x[t, n, d] at t * x_t + n * x_n + d */
    int64_t gate_t, gate_n;
    int64_t starts_t, starts_n;
    int64_t grad_t, grad_n;       /* grad_h (dl_memory_backward) */
    int32_t dtype;
    int32_t reserved;             /* 0 */
} dl_memory_shape;

/* Steps between two saved states: dl_memory_forward writes marks[k] = the state before step DL_MEMORY_MARK * k, float
 * [ceil(T / DL_MEMORY_MARK), N, D]; dl_memory_backward recomputes the steps between from x and gate in 32 bits. */
#define DL_MEMORY_MARK 16

/* Bytes of device workspace dl_memory_forward / dl_memory_backward need for this shape (0 is possible), or a DL_E_ code.  Aligned to 16 bytes;
 * what it holds before a call does not matter. */
int64_t dl_memory_workspace_bytes(const dl_memory_shape* shape);

/* h: [T, N, D]; state_out: float [N, D] = h[T-1] before rounding (may be NULL; may not overlap state); marks may be NULL. */
int dl_memory_forward(const dl_memory_shape* shape, const void* x, const void* gate, const uint8_t* starts,
                      const float* state, void* h, float* state_out, float* marks, void* workspace, void* stream);

/* Gradients of sum(h * grad_h) + sum(state_out * grad_state): dx, dgate [T, N, D] of `dtype`, dstate float [N, D] (NULL:
 * not wanted).  grad_h or grad_state may be NULL (zeros).  marks as dl_memory_forward left them for the same inputs. */
int dl_memory_backward(const dl_memory_shape* shape, const void* x, const void* gate, const uint8_t* starts,
                       const float* marks, const void* grad_h, const float* grad_state, void* dx, void* dgate,
                       float* dstate, void* workspace, void* stream);

/* One control step (T = 1) with the state kept by the caller: x, gate, h [N, D], starts [N]; shape->*_n are the strides.
 * state_out may be state itself. */
int dl_memory_step(const dl_memory_shape* shape, const void* x, const void* gate, const uint8_t* starts,
                   const float* state, void* h, float* state_out, void* stream);

/* ---- orthogonalised updates --------------------------------------------------------------------------------------
 * The orthogonal factor of a gradient, approached by `steps` Newton-Schulz products (the update of the Muon optimiser, Jordan
 * et al. 2024), and the weight update built on it, for `batch` matrices [rows, cols]:
 *
 *     U = grad                                            without momentum (momentum == NULL)
 *     M' = beta M + grad,  U = grad + beta M' | M'        with momentum: nesterov | not;  M' goes to momentum_out
 *     X = U / |U|_F   (zeros stay zeros);   steps times:  A = X X',  X = (a I + b A + c A A) X      from the short side
 *     out = weight_keep * weight + gain * X               weight == NULL: out = gain * X
 *
 * Products are exact to about 2^-22 of their operands and summed in 32 bits, norms in 64; out is rounded once.  A NaN or an
 * infinity anywhere in U makes the whole of its matrix NaN.  The coefficients have to keep X, A and a I + b A + c A A
 * of every step below 60 in size, whatever singular values in [0, 1] a matrix has (those of the Muon optimiser, 3.4445 -4.7750 2.0315, and of
 * the classic cubic, 1.5 -0.5 0, keep them below 3.5); dl_orth_update refuses others.  Strides are in elements: of a matrix in its batch and of a row; rows are contiguous. */
typedef struct dl_orth_shape {
    int64_t batch, rows, cols;
    int64_t grad_b, grad_r;
    int64_t momentum_b, momentum_r;          /* momentum, float */
    int64_t momentum_out_b, momentum_out_r;
    int64_t weight_b, weight_r;
    int64_t out_b, out_r;
    double a, b, c;                          /* coefficients of a step */
    double beta, weight_keep, gain;
    int32_t steps, nesterov;
    int32_t grad_type, weight_type, out_type, reserved;
} dl_orth_shape;

/* DL_OK if `steps` steps with these coefficients stay in that range, or DL_E_INVAL. */
int dl_orth_check_coefficients(int32_t steps, double a, double b, double c);

/* Bytes of device workspace dl_orth_update needs for this shape, or a DL_E_ code. */
int64_t dl_orth_workspace_bytes(const dl_orth_shape* shape);

/* momentum_out may be momentum, out may be weight (in place, with the same strides) or grad; no other overlap. */
int dl_orth_update(const dl_orth_shape* shape, const void* grad, const float* momentum, float* momentum_out,
                   const void* weight, void* out, void* workspace, void* stream);

#ifdef __cplusplus
}
#endif
#endif /* DRLOCO_LEARNER_H */
