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
 * infinity there does not leak); NULL: none.  Elements of x, gate, h and of the gradients have `dtype`; states, sums and
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

/* Bytes of device workspace dl_memory_forward / dl_memory_backward need for this shape (0 is possible), or a DL_E_ code. */
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

#ifdef __cplusplus
}
#endif
#endif /* DRLOCO_LEARNER_H */
