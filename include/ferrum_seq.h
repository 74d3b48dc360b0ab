/*
 * ferrum_seq.h — C ABI of the sequence operators: causal filters along a
 * sequence (short convolution, long convolution through the FFT, selective
 * state space scan, gated recurrence), the norms around a sequence block,
 * dropout, and the loss against a vocabulary. They have no counterpart in
 * the reference; they follow the conventions of ferrum_fft.h:
 * plain pointers and sizes, a status code, ferrum_last_error() for the
 * message, device memory on the handle's device, calls asynchronous on
 * `stream`, workspaces from the device's stream-ordered pool.
 *
 * Each call takes a pointer to an argument block. `struct_size` is
 * sizeof(the block); zero the block, then set what the call uses. Strides are
 * in elements. NULL marks an absent optional array. Activations ("data") have
 * type `dtype`; parameters, scan states and parameter gradients are float32 (but
 * a vocabulary matrix and its gradient, of type `dtype`).
 * Sums, recurrences and statistics run in float32; each output is rounded
 * once to its type (the loss's gradient says what else it rounds). No result depends on the order in which blocks run.
 * An array that a call writes shares no memory with its other arrays, except
 * where a block says so; the C entries take the caller's word for it.
 *
 * `lengths` (int32, one per sequence, optional) are the valid lengths of a
 * padded batch. A length is clamped to [0, length]. Steps past it are not
 * read; their outputs (and input gradients) are written as zero, and final
 * states are those after the last valid step.
 */
#ifndef FERRUM_SEQ_H
#define FERRUM_SEQ_H

#include "ferrum_fft.h"

#ifdef __cplusplus
extern "C" {
#endif

enum { FERRUM_F32 = 0, FERRUM_F16 = 1, FERRUM_BF16 = 2 };
enum { FERRUM_NORM_RMS = 0, FERRUM_NORM_LAYER = 1 };

/* Largest number of taps of the short convolution. */
#define FERRUM_CONV1D_MAX_TAPS 8
/* Largest number of states per channel of the scan. */
#define FERRUM_SCAN_MAX_STATES 64
/* Steps between the states the scan saves for its gradient. */
#define FERRUM_SCAN_SAVE_STEPS 16
/* Steps between the states the recurrence saves for its gradient. */
#define FERRUM_RECURRENCE_SAVE_STEPS 16
/* Longest sequence of the long convolution. */
#define FERRUM_LONG_CONV_MAX_LENGTH (1 << 25)
/* Widest rows of the loss's gradient in 16-bit types. */
#define FERRUM_LOSS_BWD_MAX_WIDTH_16 (1 << 16)

/* A (batch, length, channels) array: element (b, t, d) is at
 * ptr[b * batch_stride + t * row_stride + d]. Single-token calls use
 * row_stride 0. */
typedef struct {
  void *ptr;
  int64_t batch_stride, row_stride;
} ferrum_rows;

/* ---------------------------------------------------------------------------
 * Short causal depthwise convolution, taps K in [1, 8]:
 *   p[b,t,d] = bias[d] + sum_j weight[d,j] * x[b, t-K+1+j, d]
 *   y = silu ? p * sigmoid(p) : p
 * x before the first step comes from initial_state (batch, K-1, channels,
 * contiguous, oldest first, type `dtype`), or is zero.
 */
typedef struct {
  size_t struct_size;
  int dtype, taps, silu;
  size_t batch, length, channels;
  const float *weight, *bias; /* (channels, taps) contiguous; (channels) */
  const void *initial_state;
  const int32_t *lengths;
  ferrum_rows x, y;
  void *final_state;          /* optional; may be initial_state */
  /* gradients (ferrum_causal_conv1d_bwd) */
  ferrum_rows dy, dx;
  const void *dfinal_state;   /* optional, as final_state */
  float *dweight, *dbias;     /* dbias optional */
  void *dinitial_state;       /* optional */
} ferrum_conv1d_args;

ferrum_status ferrum_causal_conv1d(ferrum_device *dev, const ferrum_conv1d_args *args, void *stream);
/* Uses x, dy, weight, bias, initial_state, lengths, dfinal_state. */
ferrum_status ferrum_causal_conv1d_bwd(ferrum_device *dev, const ferrum_conv1d_args *args,
                                       void *stream);
/* One step of every sequence (length 1, no lengths): initial_state is the state
 * before, final_state the state after (may be the same array). */
ferrum_status ferrum_causal_conv1d_step(ferrum_device *dev, const ferrum_conv1d_args *args,
                                        void *stream);

/* ---------------------------------------------------------------------------
 * Selective state space scan, N states per channel, N in [1, 64]:
 *   s  = delta[b,t,d] + delta_bias[d];  dt = delta_softplus ? log(1 + e^s) : s
 *   h[n] = exp(dt * A[d,n]) * h[n] + dt * u[b,t,d] * B[b,t,g,n]
 *   y  = sum_n h[n] * C[b,t,g,n] + D[d] * u[b,t,d]
 *   out = z ? y * z * sigmoid(z) : y
 * Channel d belongs to group g = d / (channels / groups). Row strides must fit
 * 32 bits.
 */
typedef struct {
  size_t struct_size;
  int dtype, delta_softplus;
  size_t batch, length, channels, states, groups;
  ferrum_rows u, delta, z, out;             /* z optional */
  ferrum_rows B, C;                         /* element (b, t, g, n): + g * group_stride + n */
  int64_t B_group_stride, C_group_stride;
  const float *A, *D, *delta_bias;          /* (channels, N); (channels); D, delta_bias optional */
  const float *initial_state;               /* (batch, channels, N), optional (zeros) */
  float *final_state;                       /* (batch, channels, N), optional */
  const int32_t *lengths;
  /* (batch, ceil(length / 16), channels, N): the state in front of every 16th
   * step. Optional output of the scan, needed by its gradient. */
  float *saved_states;
  /* gradients (ferrum_selective_scan_bwd) */
  ferrum_rows dout, du, ddelta, dz;         /* dz with z */
  const float *dfinal_state;                /* optional */
  void *dB, *dC;                            /* (batch, length, groups, N) contiguous, type dtype */
  float *dA, *dD, *ddelta_bias;             /* dD, ddelta_bias optional */
  float *dinitial_state;                    /* optional */
} ferrum_scan_args;

ferrum_status ferrum_selective_scan(ferrum_device *dev, const ferrum_scan_args *args, void *stream);
ferrum_status ferrum_selective_scan_bwd(ferrum_device *dev, const ferrum_scan_args *args,
                                        void *stream);
/* One step of every sequence (length 1, no lengths): initial_state (required)
 * before, final_state (required, may be the same array) after. */
ferrum_status ferrum_selective_scan_step(ferrum_device *dev, const ferrum_scan_args *args,
                                         void *stream);

/* ---------------------------------------------------------------------------
 * Norms around a block, over rows of `channels` values (row stride in
 * elements, values contiguous); a normalised row has at most 32768 values. N(v) = v / sqrt(mean(v^2) + eps) (RMS) or
 * (v - mean) / sqrt(var + eps) (LAYER).
 *
 * In front:  r = residual + scale * x (either part optional);
 *            y = N(r) * weight + bias
 * `residual` and `r` have type `residual_dtype` (float32 or dtype).
 *
 * Behind:    gate_inside:  p = N(x * silu(gate)) * weight + bias
 *            otherwise:    p = (N(x) * weight + bias) * silu(gate)
 *            y = residual + scale * p
 * with N over each of `groups` equal parts of a row; gate, residual, scale
 * and bias optional; residual has type residual_dtype, y type dtype.
 */
typedef struct {
  size_t struct_size;
  int dtype, residual_dtype, kind, gate_inside;
  size_t rows, channels, groups;
  float eps;
  const float *weight, *bias, *scale;
  const void *x, *gate, *residual;
  void *y, *r;
  int64_t x_stride, gate_stride, residual_stride, y_stride, r_stride;
  /* gradients */
  const void *dy, *dr;                 /* dr (in front): gradient of r, optional */
  void *dx, *dgate, *dresidual;
  int64_t dy_stride, dr_stride, dx_stride, dgate_stride, dresidual_stride;
  float *dweight, *dbias, *dscale;     /* dbias, dscale optional */
} ferrum_norm_args;

ferrum_status ferrum_norm_before(ferrum_device *dev, const ferrum_norm_args *args, void *stream);
/* Uses r, dy, dr, weight, scale and (for dscale) x. dx optional. */
ferrum_status ferrum_norm_before_bwd(ferrum_device *dev, const ferrum_norm_args *args, void *stream);
ferrum_status ferrum_norm_after(ferrum_device *dev, const ferrum_norm_args *args, void *stream);
/* Uses x, gate, dy, weight, bias, scale. The gradient of residual is dy. */
ferrum_status ferrum_norm_after_bwd(ferrum_device *dev, const ferrum_norm_args *args, void *stream);

/* ---------------------------------------------------------------------------
 * Long causal convolution along the last axis of (batch, channels, length):
 *   y[b,d,t] = sum_{s <= min(t, kernel_length - 1)} kernel[d,s] * x[b,d,t-s]
 *              + skip[d] * x[b,d,t]
 * Element (b, d, t) is at ptr[b * batch_stride + d * row_stride + t * step],
 * x_step being that of x, and so on. A step of 1 is fastest; arrays of other
 * steps (channel-last ones) go through contiguous rows in a workspace.
 * kernel_length in [1, length]. Lengths above a short limit go through the
 * FFT, which mixes all steps of a row: an infinity or NaN in x reaches every
 * output of its row (never another row).
 */
typedef struct {
  size_t struct_size;
  int dtype;
  size_t batch, channels, length, kernel_length;
  const float *kernel, *skip;          /* (channels, kernel_length); (channels) optional */
  ferrum_rows x, y;
  int64_t x_step, y_step;
  /* gradients */
  ferrum_rows dy, dx;
  int64_t dy_step, dx_step;
  float *dkernel, *dskip;              /* dskip optional */
  /* one token: x and y are (batch, channels) (row_stride unused);
   * history (batch, channels, length), positions (batch) int32: x is stored
   * at history[b, :, positions[b]] and y taken there. A position outside
   * [0, length) stores nothing and its y is zero. */
  ferrum_rows history;
  const int32_t *positions;
} ferrum_long_conv_args;

ferrum_status ferrum_long_conv(ferrum_device *dev, const ferrum_long_conv_args *args, void *stream);
ferrum_status ferrum_long_conv_bwd(ferrum_device *dev, const ferrum_long_conv_args *args,
                                   void *stream);
ferrum_status ferrum_long_conv_step(ferrum_device *dev, const ferrum_long_conv_args *args,
                                    void *stream);

/* ---------------------------------------------------------------------------
 * Gated linear recurrence, one state per channel:
 *   a = exp(-decay[d] * sigmoid(recurrence_gate[b,t,d]))
 *   h = a * h + sqrt(1 - a^2) * sigmoid(input_gate[b,t,d]) * x[b,t,d];  out = h
 * decay is not negative (a negative one makes its channel NaN); where 1 - a^2 is
 * not above 0 (or below 2^-126), the root and the gradient through it are 0. An
 * infinite state stays infinite; gradients that it or an infinite dout reaches are
 * infinite or NaN.
 */
typedef struct {
  size_t struct_size;
  int dtype;
  size_t batch, length, channels;
  ferrum_rows x, input_gate, recurrence_gate, out;
  const float *decay;                       /* (channels) */
  const float *initial_state;               /* (batch, channels), optional (zeros) */
  float *final_state;                       /* (batch, channels), optional */
  const int32_t *lengths;
  /* (batch, ceil(length / 16), channels): the state in front of every 16th
   * step. Optional output of the recurrence, needed by its gradient. */
  float *saved_states;
  /* gradients (ferrum_gated_recurrence_bwd) */
  ferrum_rows dout, dx, dinput_gate, drecurrence_gate;
  const float *dfinal_state;                /* optional */
  float *ddecay;
  float *dinitial_state;                    /* optional */
} ferrum_recurrence_args;

ferrum_status ferrum_gated_recurrence(ferrum_device *dev, const ferrum_recurrence_args *args,
                                      void *stream);
ferrum_status ferrum_gated_recurrence_bwd(ferrum_device *dev, const ferrum_recurrence_args *args,
                                          void *stream);
/* One step of every sequence (length 1, no lengths): initial_state (required)
 * before, final_state (required, may be the same array) after. */
ferrum_status ferrum_gated_recurrence_step(ferrum_device *dev, const ferrum_recurrence_args *args,
                                           void *stream);

/* ---------------------------------------------------------------------------
 * Dropout, over rows of `channels` values (strides in elements, values
 * contiguous):
 *   y = residual + (keep ? x / (1 - p) : 0)     (residual optional)
 * Element i = row * channels + channel is kept where word i % 4 of
 * Philox4x32-10 (Salmon et al., "Parallel random numbers: as easy as 1, 2,
 * 3", SC 2011), with the counter (i / 4, offset) and the key seed, each 64 bits
 * in two words, low word first, is not below p * 2^32. No mask is stored: the
 * gradient draws the same words. y and residual have type residual_dtype
 * (float32 or dtype).
 */
typedef struct {
  size_t struct_size;
  int dtype, residual_dtype;
  size_t rows, channels;
  double p;                             /* in [0, 1]; 1 keeps nothing */
  uint64_t seed, offset;
  const uint64_t *seed_ptr;             /* on the device, instead of seed; optional */
  const void *x, *residual;
  void *y;
  int64_t x_stride, residual_stride, y_stride;
  /* gradients: dx (type dtype) from dy (type residual_dtype) */
  const void *dy;
  void *dx;
  int64_t dy_stride, dx_stride;
} ferrum_dropout_args;

ferrum_status ferrum_dropout(ferrum_device *dev, const ferrum_dropout_args *args, void *stream);
/* The gradient of x; that of residual is dy. */
ferrum_status ferrum_dropout_bwd(ferrum_device *dev, const ferrum_dropout_args *args, void *stream);

/* ---------------------------------------------------------------------------
 * Softmax cross entropy of rows against a vocabulary matrix:
 *   l[t,v] = sum_d x[t,d] * weight[v,d]
 *   lse[t] = log(sum_v exp(l[t,v]));  loss[t] = lse[t] - l[t, target[t]]
 * x, weight, dx and dweight have type `dtype`. The logits are never stored as a
 * whole. A row whose target lies outside [0, vocab) has no loss: its loss, lse and
 * gradients are 0, whatever its values.
 * In 16-bit types the gradient takes rows of up to FERRUM_LOSS_BWD_MAX_WIDTH_16
 * values and rounds the logits' gradients to 16 bits between its products: dx and
 * dweight are up to 1.4 times as far from the exact ones as their own rounding
 * leaves them.
 * Workspace of the loss: 8 bytes for each token and 128 words, and a copy of x or
 * weight whose rows do not begin at multiples of 16 bytes. Of the gradient: the
 * logits' gradients of a piece of the vocabulary (256 MiB, or 4096 words if that
 * is more), a copy of x, one of weight as above, and float32 sums of dx
 * (tokens * width) and dweight where their products are split.
 */
typedef struct {
  size_t struct_size;
  int dtype;
  size_t tokens, width, vocab;
  const void *x, *weight;               /* (tokens, width), (vocab, width) */
  int64_t x_stride, weight_stride;      /* of rows, in elements */
  const int64_t *targets;               /* (tokens) */
  float *loss, *lse;                    /* (tokens); lse is an input of the gradient */
  /* gradients */
  const float *dloss, *dlse;            /* (tokens); each optional */
  void *dx, *dweight;
  int64_t dx_stride, dweight_stride;
} ferrum_cross_entropy_args;

ferrum_status ferrum_linear_cross_entropy(ferrum_device *dev, const ferrum_cross_entropy_args *args,
                                          void *stream);
ferrum_status ferrum_linear_cross_entropy_bwd(ferrum_device *dev,
                                              const ferrum_cross_entropy_args *args, void *stream);

#ifdef __cplusplus
}
#endif

#endif /* FERRUM_SEQ_H */
