/*
 * ttsx_seq.h - C ABI of the sequence operators of libttsx.so (MI355X, gfx950): the gated linear recurrence and the
 * low-rank adapters of many voices.  No counterpart in the reference, whose recurrences step serially
 * (Tacotron2/TTS/models.py:419-427) and whose voices differ by one added embedding (:838-849).
 *
 * Conventions are those of ttsx.h (device pointers, explicit stream, TTSX_OK or a negative code, no exception, message
 * by ttsx_last_error_string), with these additions:
 *   - activations are 32-bit floats or one of two 16-bit kinds (TTSX_F32 / _BF16 / _F16); what is summed, scanned or
 *     kept from step to step is fp32;
 *   - an activation [B,T,D] has its last axis contiguous and two strides, of the batch and of the row, in ELEMENTS;
 *     inputs may overlap or repeat (a stride of 0), and with T = 1 the row stride is not looked at; a pointer is
 *     aligned to its element, no further;
 *   - nothing is allocated and nothing synchronises: working memory comes from the caller, the calls can be captured
 *     into a graph, and calls that share no output and no workspace can run at the same time;
 *   - lengths [B] int32 or NULL (= T) is read on the device and clamped to 0..T; rows at positions >= length are not
 *     read.
 */
#ifndef TTSX_SEQ_H
#define TTSX_SEQ_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define TTSX_F32 0
#define TTSX_BF16 1
#define TTSX_F16 2

/* The largest calls: channels or columns and elements between two rows; requests, and steps or positions; voices.  A launch
 * counts its threads in 32 bits: a call of more (2^24 workgroups, such as tiles of 32 positions, or in
 * ttsx_adapter_backward voices times ranks times 1024 columns) returns TTSX_ERR_ARG before anything is queued. */
#define TTSX_SEQ_MAX_WIDTH (1 << 20)
#define TTSX_SEQ_MAX_ROWS (1 << 30)
#define TTSX_SEQ_MAX_VOICES (1 << 24)

/* Steps between two states that ttsx_gated_scan keeps for its backward pass. */
#define TTSX_STATE_BLOCK 64

/* ------------------------------------------------------------------ gated linear recurrence
 *   f_t = sigmoid(g_t)      h_t = f_t h_{t-1} + (1 - f_t) x_t
 * per channel, over the rows 0 .. length-1 of each request, or from row length-1 down to 0 where `reverse` is set.
 *   x, g     [B,T,D]  values and gate logits (may be two slices of one projection); D and the row strides up to
 *                    TTSX_SEQ_MAX_WIDTH
 *   h0       [B,D] fp32 state in front of the first step, or NULL (= 0)
 *   h        [B,T,D] contiguous, of x's type; rows at positions >= length are zero
 *   h_last   [B,D] fp32 state behind the last step (h0 for an empty request)
 *   states   [B,ceil(T/64),D] fp32 or NULL: the state in front of step 64 k (behind the last step where the request
 *            is shorter), for ttsx_gated_scan_backward
 *   workspace  ttsx_gated_scan_workspace(B, T, D, dtype, 0) bytes, aligned to 4; may be NULL where that is 0 */
int ttsx_gated_scan(const void* x, int64_t x_batch_stride, int64_t x_row_stride, const void* g, int64_t g_batch_stride,
                    int64_t g_row_stride, const float* h0, const int32_t* lengths, int B, int T, int D, int dtype,
                    int reverse, void* h, float* h_last, float* states, void* workspace, size_t workspace_bytes,
                    void* stream);

/* Gradients of ttsx_gated_scan, from x, g and the states it kept:
 *   dh       [B,T,D]  gradient of h;  dh_last [B,D] fp32 gradient of h_last, or NULL (= 0)
 *   dx, dg   [B,T,D] contiguous, of x's type; rows at positions >= length are zero
 *   dh0      [B,D] fp32 (dh_last for an empty request)
 *   workspace  ttsx_gated_scan_workspace(B, T, D, dtype, 1) bytes, aligned to 4; may be NULL where that is 0 */
int ttsx_gated_scan_backward(const void* dh, int64_t dh_batch_stride, int64_t dh_row_stride, const void* x,
                             int64_t x_batch_stride, int64_t x_row_stride, const void* g, int64_t g_batch_stride,
                             int64_t g_row_stride, const float* states, const float* dh_last, const int32_t* lengths,
                             int B, int T, int D, int dtype, int reverse, void* dx, void* dg, float* dh0,
                             void* workspace, size_t workspace_bytes, void* stream);

/* Bytes of working memory of the two calls above (0 where the batch alone fills the chip), or a negative code. */
long ttsx_gated_scan_workspace(int B, int T, int D, int dtype, int backward);

/* One step of B requests: x, g [B,D] with a batch stride; h [B,D] fp32 contiguous state; y [B,D] contiguous, the new
 * state in x's type; h_out [B,D] fp32 the new state itself (may be h: the update is in place). */
int ttsx_gated_step(const void* x, int64_t x_batch_stride, const void* g, int64_t g_batch_stride, const float* h, int B,
                    int D, int dtype, void* y, float* h_out, void* stream);

/* ------------------------------------------------------------------ low-rank adapters of many voices
 * Beside a shared projection y = x W^T, each request of a batch adds the adapter of its own voice:
 *   out[b,t,:] = y[b,t,:] + scale[v] (x[b,t,:] down[v]^T) up[v]        v = voices[b]
 *   y, out   [B,T,N]   out may be y itself (in place), and overlaps no other argument
 *   x        [B,T,K]
 *   down     [V,R,K], up [V,R,N], contiguous, of x's type; 1 <= R <= TTSX_ADAPTER_MAX_RANK; K, N and the row strides
 *            up to TTSX_SEQ_MAX_WIDTH, V to TTSX_SEQ_MAX_VOICES
 *   voices   [B] int32; a voice outside 0..V-1 has no adapter
 *   scale    [V] fp32 or NULL (= 1)
 * Rows without an adapter (no voice, or at positions >= length) are y's.  x down^T and the sum are fp32; out is
 * rounded once. */
#define TTSX_ADAPTER_MAX_RANK 64
int ttsx_adapter_add(const void* y, int64_t y_batch_stride, int64_t y_row_stride, const void* x, int64_t x_batch_stride,
                     int64_t x_row_stride, const void* down, const void* up, const int32_t* voices, const float* scale,
                     const int32_t* lengths, int B, int T, int K, int N, int R, int V, int dtype, void* out,
                     int64_t out_batch_stride, int64_t out_row_stride, void* stream);

/* Gradients of ttsx_adapter_add from dy [B,T,N], the gradient of out (that of y is dy itself):
 *   dx       [B,T,K] contiguous; zero in rows without an adapter
 *   ddown    [V,R,K], dup [V,R,N] contiguous, of x's type: sums over the rows of each voice in the order of the
 *            batch (two runs agree to the bit); zero for a voice that no request has
 *   workspace  ttsx_adapter_backward_workspace(B, T, K, N, R, dtype) bytes, aligned to 16 */
int ttsx_adapter_backward(const void* dy, int64_t dy_batch_stride, int64_t dy_row_stride, const void* x,
                          int64_t x_batch_stride, int64_t x_row_stride, const void* down, const void* up,
                          const int32_t* voices, const float* scale, const int32_t* lengths, int B, int T, int K, int N,
                          int R, int V, int dtype, void* dx, void* ddown, void* dup, void* workspace,
                          size_t workspace_bytes, void* stream);
long ttsx_adapter_backward_workspace(int B, int T, int K, int N, int R, int dtype);

#ifdef __cplusplus
}
#endif
#endif /* TTSX_SEQ_H */
