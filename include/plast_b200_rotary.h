/*
 * plast_b200_rotary.h — rotary position embedding, alone and together with the norm of query and key
 * heads. No counterpart in the reference (its layers stop short of attention); the calling rules are
 * the library's: host Tensor structs, device data, the caller allocates outputs, forward overwrites,
 * backward adds to the gradients of inputs that require them.
 *
 * Tensors of heads have any number of leading dims and any strides: [batch, time, heads, head] and
 * [batch, heads, time, head] are both fine. positions (INT32) broadcasts, NumPy rules, against the
 * dims before the last one: [batch, time, 1] or [time, 1] for the former, [time] or [batch, 1, time]
 * for the latter. inv_freq (FLOAT32, one dim) holds the angle per position of every pair; its length
 * n sets the rotated part of the head: the first 2 n elements, the rest is passed on unchanged.
 * A head has at most PLAST_ROTARY_MAX_HEAD elements.
 *
 * Pair i of a head is turned by position * inv_freq[i] (computed in 64 bits, so that far positions
 * keep their angle): (a, b) -> amplitude * (a cos - b sin, a sin + b cos).
 */
#ifndef PLAST_B200_ROTARY_H
#define PLAST_B200_ROTARY_H

#include "plast_b200.h"

#ifdef __cplusplus
extern "C" {
#endif

#define PLAST_ROTARY_HALVES 0      /* pair i = elements i and n + i */
#define PLAST_ROTARY_INTERLEAVED 1 /* pair i = elements 2 i and 2 i + 1 */
#define PLAST_ROTARY_MAX_HEAD 1024

/* rotary as an op of the table: inputs = {x, positions, inv_freq}, params.dim = the pair layout,
 * params.fval = the amplitude (positive; 1 unless a scaling asks for more). The output may be x
 * itself (same data and strides); no other overlap. Backward turns the other way: x->grad += amplitude * R(-angle)
 * output->grad; positions and inv_freq receive no gradient (requires_grad on them is refused). */
void rotary_cuda_forward(const Tensor **inputs, Tensor *output, KernelParams params);
void rotary_cuda_backward(Tensor **inputs, const Tensor *output, KernelParams params);

/* The table for rotary: frequency i of a head's `rotated` elements is base^(-2 i / rotated), changed
 * for contexts longer than the trained one as `kind` says; `factor` >= 1 is the extension.
 *   NONE      as it is
 *   LINEAR    every frequency / factor (positions interpolated)
 *   BASE      base * factor^(rotated / (rotated - 2)): the slowest pair is slowed by the factor, the
 *             fastest stays
 *   PARTS     pairs that make more than `fast` turns over the trained context stay, those that make
 *             fewer than `slow` are divided by the factor, a linear ramp over the pair index between;
 *             the amplitude becomes 0.1 log(factor) + 1
 *   BANDS     pairs whose wavelength is below context / fast stay, above context / slow are divided
 *             by the factor, between them the frequency is blended in proportion to context / wavelength
 * Host arithmetic in 64 bits; writes rotated / 2 floats to host memory and, unless NULL, the
 * amplitude. Returns PLAST_B200_OK or an error code (also readable with plast_b200_last_error()). */
typedef enum PlastRotaryScalingKind {
  PLAST_ROTARY_SCALING_NONE = 0,
  PLAST_ROTARY_SCALING_LINEAR = 1,
  PLAST_ROTARY_SCALING_BASE = 2,
  PLAST_ROTARY_SCALING_PARTS = 3,
  PLAST_ROTARY_SCALING_BANDS = 4
} PlastRotaryScalingKind;
typedef struct PlastRotaryScaling {
  int kind;     /* PlastRotaryScalingKind */
  float factor;
  float slow;   /* PARTS: turns (typically 1); BANDS: typically 1 */
  float fast;   /* PARTS: turns (typically 32); BANDS: typically 4 */
  u64 context;  /* trained context length (PARTS, BANDS) */
} PlastRotaryScaling;
int plast_b200_rotary_frequencies(const PlastRotaryScaling *scaling, u64 rotated, float base,
                                  float *host_inv_freq, float *amplitude);

/* Root-mean-square norm of every query and key head, its weight, and the rotation, in one launch:
 *   n = x / sqrt(mean(x^2) + epsilon),  u = weight * n,  out = rotary(u)
 * q and k may have different numbers of heads (and shapes) but the same head size; k, k_weight and
 * k_out may be NULL together (one tensor alone). A weight is FLOAT32 with head-size elements along
 * its last dim ([head], [1, head], ...), or NULL for none. An output may be its own input (same data and
 * strides) and shares no element with any other tensor of the call, nor does the gradient of an input
 * in backward but with the gradient of its own output.
 * Backward recomputes the norm from q and k, reads q_out->grad and k_out->grad and adds to the
 * gradients of q, k and the weights, each where requires_grad is set; weight gradients are summed in
 * a fixed order. The sum of squares is held in 32 bits: a head whose elements pass about 10^18 overflows
 * it and gives zeros. (A forward that ran in place has overwritten what backward needs.) Inside a
 * plast_b200_peer_reduce_begin / _end bracket the weight gradients are refused: this call does not
 * combine them across ranks. */
typedef struct PlastQkNormParams {
  float epsilon;
  float amplitude; /* of the rotation, positive */
  int layout;      /* PLAST_ROTARY_HALVES / PLAST_ROTARY_INTERLEAVED */
} PlastQkNormParams;
void plast_b200_qk_norm_rotary(const Tensor *q, const Tensor *k, const Tensor *q_weight,
                               const Tensor *k_weight, const Tensor *positions, const Tensor *inv_freq,
                               Tensor *q_out, Tensor *k_out, PlastQkNormParams params);
void plast_b200_qk_norm_rotary_backward(Tensor *q, Tensor *k, Tensor *q_weight, Tensor *k_weight,
                                        const Tensor *positions, const Tensor *inv_freq,
                                        const Tensor *q_out, const Tensor *k_out, PlastQkNormParams params);

#ifdef __cplusplus
}
#endif

#endif /* PLAST_B200_ROTARY_H */
