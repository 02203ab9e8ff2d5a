/*
 * plast_b200_optim.h — optimiser steps of the plast runtime on sm_100a: one multi-tensor launch
 * updates every parameter of a step (bandwidth-bound elementwise work, like the rest of this
 * library).
 *
 * Replaces src/optimizers/cuda/{sgd,adam,adamw}.cu. The reference's sgd_step_cuda launches one
 * scalar kernel per parameter (sgd.cu:11-32); its adam_step_cuda and adamw_step_cuda are empty
 * functions (adam.cu:17-18, adamw.cu:20-21), so the arithmetic contract is the CPU path:
 * src/optimizers/cpu/sgd.c:11-32, adam.c:22-72, adamw.c:21-74. Parameters, gradients and moments
 * are treated as flat float arrays of numel(param) elements, as the CPU loops do; parameters
 * that are NULL or have no grad are skipped.
 *
 * SGD, Adam and AdamW restate include/optimizers/{sgd,adam,adamw}.h; define
 * PLAST_B200_USE_REFERENCE_TYPES to compile against the reference's own headers instead.
 */
#ifndef PLAST_B200_OPTIM_H
#define PLAST_B200_OPTIM_H

#include "plast_b200.h"

#ifdef PLAST_B200_USE_REFERENCE_TYPES
#include "optimizers/adam.h"
#include "optimizers/adamw.h"
#include "optimizers/sgd.h"
#else

struct Arena;

/* include/optimizers/sgd.h:5-7 */
typedef struct {
  float lr;
} SGD;

/* include/optimizers/adam.h:5-15 — 56 bytes: lr@0 beta1@4 beta2@8 epsilon@12 t@16 m@24 v@32 */
typedef struct {
  float lr;
  float beta1;
  float beta2;
  float epsilon;
  int t;
  Tensor **m;
  Tensor **v;
  struct Arena *data_arena;
  struct Arena *optimizer_arena;
} Adam;

/* include/optimizers/adamw.h:5-16 — 56 bytes: ... weight_decay@16 t@20 m@24 v@32 */
typedef struct {
  float lr;
  float beta1;
  float beta2;
  float epsilon;
  float weight_decay;
  int t;
  Tensor **m;
  Tensor **v;
  struct Arena *data_arena;
  struct Arena *optimizer_arena;
} AdamW;

#endif /* PLAST_B200_USE_REFERENCE_TYPES */

#ifdef __cplusplus
extern "C" {
#endif

/* data[j] -= lr * grad[j] (src/optimizers/cpu/sgd.c:28-30); product and difference each
 * rounded to fp32. */
void sgd_step_cuda(SGD *optimizer, Tensor **parameters, int num_parameters);

/* optimizer->t is incremented first; on the first step the moment tensors are created, zeroed,
 * and stored in optimizer->m / optimizer->v (the CPU path takes them from the optimizer's
 * arenas, adam.c:30-46; here the library owns them: one device allocation for all moments and
 * host Tensor structs, freed by plast_b200_adam_state_release). Then, with
 *   lr_t = lr * sqrt(1 - beta2^t) / (1 - beta1^t)   (computed on the host exactly as adam.c:48-49)
 * every element does, each operation rounded to fp32 (adam.c:62-66):
 *   m = beta1 * m + (1 - beta1) * g;  v = beta2 * v + (1 - beta2) * g * g;
 *   data -= lr_t * m / (sqrtf(v) + epsilon)
 * AdamW first applies data -= lr * weight_decay * data (adamw.c:65-66). */
void adam_step_cuda(Adam *optimizer, Tensor **parameters, int num_parameters);
void adamw_step_cuda(AdamW *optimizer, Tensor **parameters, int num_parameters);

/* Frees moments created by adam_step_cuda / adamw_step_cuda (pass optimizer->m, optimizer->v)
 * and leaves nothing behind; unknown pointers are ignored. No reference counterpart: the
 * reference releases its arenas as a whole. */
void plast_b200_adam_state_release(Tensor **m, Tensor **v);

/* Muon: momentum whose update is orthogonalised, for weight matrices (biases, norms and embeddings
 * take one of the optimisers above). No counterpart in the reference. */
#define PLAST_MUON_SCALE_ASPECT 0 /* s = sqrt(max(1, rows / cols)) */
#define PLAST_MUON_SCALE_RMS 1    /* s = 0.2 sqrt(max(rows, cols)): an update of AdamW's size */
#define PLAST_MUON_SCALE_NONE 2   /* s = 1 */
#define PLAST_MUON_MAX_STEPS 32
#define PLAST_MUON_MAX_DIM 262144
typedef struct {
  float lr;
  float momentum;     /* typically 0.95 */
  float weight_decay; /* decoupled */
  float epsilon;      /* added to the Frobenius norm, typically 1e-7 */
  int nesterov;       /* 0 / 1 */
  int ns_steps;       /* Newton-Schulz steps, typically 5 */
  int scale;          /* PLAST_MUON_SCALE_* */
  Tensor **m;         /* momenta; NULL before the first step */
} Muon;

/* One step over a list of contiguous FLOAT32 parameters of two or more dims, each a matrix of
 * shape[0] rows (at most PLAST_MUON_MAX_DIM rows or columns); entries that are NULL or have no grad
 * are skipped. Per matrix, with gradient g:
 *   m = momentum m + g,  u = nesterov ? g + momentum m : m
 *   data = data (1 - lr weight_decay) - lr s orthogonalised(u)
 * optimizer->m holds one momentum per parameter, contiguous and of its size; where it is NULL the
 * first step creates zeros for the list (freed by plast_b200_muon_state_release, like Adam's), so a
 * first step cannot be captured into a graph and is refused there. No parameter or momentum may overlap another buffer of the
 * call. A call that is refused changes nothing. */
void muon_step_cuda(Muon *optimizer, Tensor **parameters, int num_parameters);
void plast_b200_muon_state_release(Tensor **m);

/* The orthogonalisation alone, for `count` matrices at once: X = x / (|x|_F + epsilon), then `steps`
 * times (0 to PLAST_MUON_MAX_STEPS) X <- a X + (b A + c A A) X with A = X X^T (of the smaller side)
 * and (a, b, c) = (3.4445, -4.7750, 2.0315). Contiguous FLOAT32 tensors as above; an output may be
 * its own input and overlaps no other tensor of the call. The norm is summed in 64 bits. The values of
 * X, X X^T and the polynomial are kept in 22 bits, below 2^-14 with an absolute error of 2^-39 (X begins
 * with norm 1, or |x|_F / epsilon where that is less). A matrix whose rows and columns are of like size
 * comes out as accurate as with products in fp32; a row of 1e-5 of the others about 1e-4 off, relative to
 * itself; and after five steps no element is known better than to 1e-9. A matrix of zeros gives zeros
 * if epsilon > 0 (else 0 / 0, NaN); a NaN or an infinity makes its matrix NaN. */
void plast_b200_orthogonalise(const Tensor **inputs, Tensor **outputs, int count, int steps, float epsilon);

/* Every wait inside the product kernels is limited to about two seconds. Where one runs out (which
 * takes a broken GPU or library) what the call could not compute of its results is NaN instead of
 * wrong (the momenta of a step have moved), and this returns 1 once; later calls are not affected.
 * 0 = all is well since the last look, -1 = a CUDA error. Waits for the library stream; a call on
 * another stream of the device is told of when it has ended. */
int plast_b200_muon_status(void);

#ifdef __cplusplus
}
#endif

#endif /* PLAST_B200_OPTIM_H */
