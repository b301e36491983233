/* haste_b200 C ABI: fused RNN layers (LSTM, GRU, IndRNN and their LayerNorm
 * variants) for NVIDIA B200 (sm_100a).
 *
 * Each entry point replaces one `haste::v0::<cell>::{ForwardPass,BackwardPass}<T>::Run`
 * of lmnt-com/haste (file:line cited per function).  Conventions shared by all:
 *
 *   - Every pointer is a DEVICE pointer owned by the caller, including scratch.
 *     Tensors are dense, row-major, rightmost index fastest
 *     (T steps, N batch, C input size, H hidden size), as in lib/haste.h:18-26.
 *   - `dtype` selects the storage type of EVERY tensor of the call:
 *     HASTE_B200_F32 (float), HASTE_B200_BF16 (__nv_bfloat16; all arithmetic,
 *     carries and accumulators stay fp32) or, for the GRU entry points and
 *     haste_b200_gemm, HASTE_B200_F16 (__half, same rule).
 *   - `h`/`c` are [T+1,N,H]; slot 0 holds the initial state and is filled by the
 *     caller.  Gate order: i,g,f,o (LSTM), z,r,g (GRU).
 *   - Outputs documented as "accumulated" are added to and must be zeroed by the
 *     caller (dW, dR, db*, du, dgamma*, dbeta*, dh, dc); `dx` is assigned.
 *   - `zoneout_mask` may be NULL: zoneout is applied only if zoneout_prob != 0
 *     and the mask is non-NULL.
 *   - Backward entry points take `transposed_inputs`: non-zero means x, W and R
 *     are passed pre-transposed exactly as the reference wants them
 *     (x_t [C,T,N], W_t [G*H,C], R_t [G*H,H]); zero means they are passed in their
 *     forward layout (x [T,N,C], W [C,G*H], R [H,G*H]) and no copy is made.
 *   - `stream` is a cudaStream_t (NULL = default stream).  All work is issued on
 *     it, in order; nothing blocks the host.  Any number of threads may call, on the same
 *     stream too: a call's launches go out together.
 *   - Return value: HASTE_B200_OK or an error code; haste_b200_last_error()
 *     returns a thread-local message.  No exceptions cross this boundary.
 */
#ifndef HASTE_B200_H_
#define HASTE_B200_H_

#ifdef __cplusplus
extern "C" {
#endif

enum {
  HASTE_B200_OK = 0,
  HASTE_B200_ERR_INVALID = 1,     /* bad shape, NULL pointer, unknown dtype */
  HASTE_B200_ERR_CUDA = 2,        /* a CUDA runtime call failed */
  HASTE_B200_ERR_TIMEOUT = 3,     /* a bounded in-kernel wait ran out */
  HASTE_B200_ERR_UNSUPPORTED = 4  /* shape outside what a kernel supports */
};

/* HASTE_B200_F16 (__half storage, fp32-grade arithmetic on exact bf16 (hi, lo) splits of the
 * stored values): GRU entry points and haste_b200_gemm only - the one reduced-precision type
 * the reference ships (lib/gru_forward_gpu.cu.cc:373). */
enum { HASTE_B200_F32 = 0, HASTE_B200_BF16 = 1, HASTE_B200_F16 = 2,
       /* LayerNormLSTM entry points only.  Tensors the caller exchanges with the layer are
        * __nv_bfloat16 exactly as with HASTE_B200_BF16 (x, W, R, b, gamma*, beta_h, h, c,
        * zoneout_mask, dh_new, dc_new and every gradient), but everything the forward pass
        * leaves for the backward pass is FLOAT: act_Wx, act_Wx_norm, act_Rh, act_c_norm,
        * tmp_Rh and the three caches must be float buffers of the documented shapes, and h and
        * c are carried in fp32 from step to step (only the returned copies are rounded).
        * Three LayerNorms per step amplify the rounding of a bf16-stored x.W, LN(x.W) or
        * running h to 2e-2 .. 1e-1 of the result; this mode stays within 2e-2 of fp32
        * arithmetic on the same bf16 inputs.  It runs the fp32 kernels on converted operands,
        * i.e. at fp32 speed with bf16 interface traffic. */
       HASTE_B200_BF16_WIDE = 3 };

const char* haste_b200_last_error(void);
const char* haste_b200_version(void);

/* Selects the implementation of the recurrence / contractions for subsequent
 * calls of the calling process (debug and test knob; 0 = automatic). */
enum {
  HASTE_B200_PATH_AUTO = 0,
  HASTE_B200_PATH_STEPWISE = 1,   /* one launch sequence per time step */
  HASTE_B200_PATH_PERSISTENT = 2, /* one persistent kernel per layer pass */
  HASTE_B200_PATH_NO_TENSOR_CORE = 3 /* automatic, but without the tcgen05 recurrence */
};
int haste_b200_set_recurrence_path(int path);
/* Limits the number of SMs one persistent recurrence launch of the calling process occupies
 * (0 = the whole GPU, the default).  With half the GPU per launch the two directions of a
 * bidirectional layer, issued on two streams, are co-resident and run concurrently.  Honoured by
 * the LSTM and GRU recurrences and by the LayerNorm ones on clusters; no reference counterpart. */
int haste_b200_set_sm_budget(int sms);
/* The same for the calls of this thread alone, in front of the process's setting while not 0.
 * Returns what it was, so that a caller who sets it for a call can put it back. */
int haste_b200_exchange_sm_budget(int sms);
/* The budget that holds for this thread's calls. */
int haste_b200_sm_budget(void);
enum { HASTE_B200_GEMM_AUTO = 0, HASTE_B200_GEMM_SIMT = 1, HASTE_B200_GEMM_TCGEN05 = 2,
       HASTE_B200_GEMM_TCGEN05_SINGLE = 3 /* tensor cores, never the CTA-pair kernel */ };
int haste_b200_set_gemm_path(int path);
/* Number of kernels this library has launched in the calling process. */
long long haste_b200_launch_count(void);
/* Device-side timing by phase (CUDA events on each call's stream).  After
 * haste_b200_profile_enable(1), haste_b200_profile_read fills ms[0..n) with the
 * milliseconds spent since the previous read in: 0 input projection, 1 forward
 * recurrence, 2 backward recurrence, 3 weight-gradient contractions, 4 input-gradient
 * contraction, 5 everything else.  Reading synchronises with the recorded work. */
/* Waits for the work queued on `stream` and reports whether any kernel of this library
 * abandoned a bounded wait since the last check (HASTE_B200_ERR_TIMEOUT) - the
 * asynchronous entry points cannot report that themselves. */
int haste_b200_sync_check(void* stream);
int haste_b200_profile_enable(int on);
/* Measurement aid, no reference counterpart: runs `steps` steps of the forward recurrence's
 * inter-CTA hand-off alone (publish tagged words, wait for all of them, CTA barrier; no
 * contraction, no gate math, no activation traffic) with the tiling a recurrence of batch N
 * and H hidden units uses, waits for it, and returns the device time per step in
 * microseconds.  N*H must fit one CTA per SM (16 rows x 16 units per CTA). */
int haste_b200_probe_exchange_latency(int N, int H, int steps, float* us_per_step, void* stream);
int haste_b200_profile_read(float* ms, int n);

/* While on, the sequence backward entry points called from this thread ASSIGN the parameter
 * gradients, dh and dc instead of accumulating into them, so that a caller with fresh buffers need
 * not zero them first.  Off by default (the reference's contract). */
int haste_b200_set_assign_gradients(int on);
int haste_b200_exchange_assign_gradients(int on); /* the same; returns what it was */

/* ---- LSTM -------------------------------------------------------------- */
/* Replaces lstm::ForwardPass<T>::Run  (lib/haste/lstm.h:118-129,
 * lib/lstm_forward_gpu.cu.cc:313-366).
 *   W [C,4H]  R [H,4H]  b [4H]  x [T,N,C]  h,c [T+1,N,H]
 *   v [T,N,4H] receives the gate activations when training (may be NULL otherwise)
 *   tmp_Rh [N,4H] scratch  zoneout_mask [T,N,H] or NULL */
int haste_b200_lstm_forward(int dtype, int training, int T, int N, int C, int H,
                            const void* W, const void* R, const void* b, const void* x,
                            void* h, void* c, void* v, void* tmp_Rh,
                            float zoneout_prob, const void* zoneout_mask, void* stream);

/* Replaces lstm::BackwardPass<T>::Run  (lib/haste/lstm.h:248-265,
 * lib/lstm_backward_gpu.cu.cc:319-405).
 *   dh_new, dc_new [T+1,N,H] (slot 0 is never read; dc_new may be NULL: no gradient of c)
 *   dx [T,N,C] assigned (NULL: not wanted)
 *   dW [C,4H] dR [H,4H] db [4H] dh,dc [N,H] accumulated;  v is overwritten. */
int haste_b200_lstm_backward(int dtype, int transposed_inputs, int T, int N, int C, int H,
                             const void* W, const void* R, const void* b, const void* x,
                             const void* h, const void* c, const void* dh_new,
                             const void* dc_new, void* dx, void* dW, void* dR, void* db,
                             void* dh, void* dc, void* v, const void* zoneout_mask,
                             void* stream);

/* ---- GRU --------------------------------------------------------------- */
/* Replaces gru::ForwardPass<T>::Run  (lib/haste/gru.h:86-98,
 * lib/gru_forward_gpu.cu.cc:310-371).
 *   W [C,3H] R [H,3H] bx,br [3H]  v [T,N,4H] = [z,r,g,Rh_g+br_g] when training
 *   tmp_Wx [T,N,3H], tmp_Rh [N,3H] scratch */
int haste_b200_gru_forward(int dtype, int training, int T, int N, int C, int H,
                           const void* W, const void* R, const void* bx, const void* br,
                           const void* x, void* h, void* v, void* tmp_Wx, void* tmp_Rh,
                           float zoneout_prob, const void* zoneout_mask, void* stream);

/* Replaces gru::BackwardPass<T>::Run  (lib/haste/gru.h:191-209,
 * lib/gru_backward_gpu.cu.cc:322-409).  dp,dq [T,N,3H] scratch (written). */
int haste_b200_gru_backward(int dtype, int transposed_inputs, int T, int N, int C, int H,
                            const void* W, const void* R, const void* bx, const void* br,
                            const void* x, const void* h, const void* v, const void* dh_new,
                            void* dx, void* dW, void* dR, void* dbx, void* dbr, void* dh,
                            void* dp, void* dq, const void* zoneout_mask, void* stream);

/* ---- single-step forms (the reference's Iterate, for autoregressive use) -- */
/* One time step with the state in separate [N,H] buffers; same arithmetic as T == 1 of the
 * sequence entry points, no scratch beyond the arguments.  x [N,C]; v, tmp_* sized for one step.
 * Replaces lstm::ForwardPass<T>::Iterate (lib/haste/lstm.h:73-86,
 * lib/lstm_forward_gpu.cu.cc:141-208). */
int haste_b200_lstm_forward_iterate(int dtype, int training, int N, int C, int H,
                                    const void* W, const void* R, const void* b, const void* x,
                                    const void* h, const void* c, void* h_out, void* c_out,
                                    void* v, void* tmp_Rh, float zoneout_prob,
                                    const void* zoneout_mask, void* stream);
/* Replaces lstm::BackwardPass<T>::Iterate (lib/haste/lstm.h:201-219,
 * lib/lstm_backward_gpu.cu.cc:144-243).  h, c: state before the step; c_new: cell state the
 * step produced; dh_new, dc_new [N,H]: gradient arriving at the step's outputs; dh, dc [N,H]
 * in/out carries; dW, dR, db accumulate; dx [N,C] assigned; v [N,4H] is overwritten.
 * With transposed_inputs, x is [C,N] and W, R are [4H,C], [4H,H]. */
int haste_b200_lstm_backward_iterate(int dtype, int transposed_inputs, int N, int C, int H,
                                     const void* W, const void* R, const void* b, const void* x,
                                     const void* h, const void* c, const void* c_new,
                                     const void* dh_new, const void* dc_new, void* dx, void* dW,
                                     void* dR, void* db, void* dh, void* dc, void* v,
                                     const void* zoneout_mask, void* stream);
/* Replaces gru::ForwardPass<T>::Iterate (lib/haste/gru.h:72-84,
 * lib/gru_forward_gpu.cu.cc:160-212).  v [N,4H] (may be null when not training),
 * tmp_Wx, tmp_Rh [N,3H]. */
int haste_b200_gru_forward_iterate(int dtype, int training, int N, int C, int H, const void* W,
                                   const void* R, const void* bx, const void* br, const void* x,
                                   const void* h, void* h_out, void* v, void* tmp_Wx,
                                   void* tmp_Rh, float zoneout_prob, const void* zoneout_mask,
                                   void* stream);
/* Replaces gru::BackwardPass<T>::Iterate (lib/haste/gru.h:172-189,
 * lib/gru_backward_gpu.cu.cc:168-250).  dp, dq [N,3H] scratch (written). */
int haste_b200_gru_backward_iterate(int dtype, int transposed_inputs, int N, int C, int H,
                                    const void* W, const void* R, const void* bx, const void* br,
                                    const void* x, const void* h, const void* v,
                                    const void* dh_new, void* dx, void* dW, void* dR, void* dbx,
                                    void* dbr, void* dh, void* dp, void* dq,
                                    const void* zoneout_mask, void* stream);

/* ---- IndRNN ------------------------------------------------------------ */
/* Replaces indrnn::ForwardPass<T>::Run  (lib/haste/indrnn.h:38-47,
 * lib/indrnn_forward_gpu.cu.cc:126-210).  W [C,H] u,b [H] workspace [T,N,H]. */
int haste_b200_indrnn_forward(int dtype, int training, int T, int N, int C, int H,
                              const void* W, const void* u, const void* b, const void* x,
                              void* h, void* workspace, float zoneout_prob,
                              const void* zoneout_mask, void* stream);

/* Replaces indrnn::BackwardPass<T>::Run  (lib/haste/indrnn.h:66-80,
 * lib/indrnn_backward_gpu.cu.cc:134-207).  dW [C,H] is ASSIGNED (the reference
 * uses beta=0 here); du, db [H], dh [N,H] accumulated. */
int haste_b200_indrnn_backward(int dtype, int transposed_inputs, int T, int N, int C, int H,
                               const void* W, const void* u, const void* b, const void* x,
                               const void* h, const void* dh_new, void* dx, void* dW,
                               void* du, void* db, void* dh, void* workspace,
                               const void* zoneout_mask, void* stream);

/* ---- LayerNorm --------------------------------------------------------- */
/* Replaces layer_norm::ForwardPass<T>::Run/RunPartial  (lib/haste/layer_norm.h:30-49,
 * lib/layer_norm_forward_gpu.cu.cc:22-150).  Row LayerNorm over `width` with
 * biased variance and eps 1e-5; beta may be NULL; cache [rows,2] = (mean, invstd). */
int haste_b200_layer_norm_forward(int dtype, int rows, int width, const void* gamma,
                                  const void* beta, const void* x, void* y, void* cache,
                                  void* stream);

/* Replaces layer_norm::BackwardPass<T>::Run/RunPartial  (lib/haste/layer_norm.h:63-79,
 * lib/layer_norm_backward_gpu.cu.cc:23-165).  dx may alias dy.  dgamma [width]
 * (and dbeta if non-NULL) accumulated. */
int haste_b200_layer_norm_backward(int dtype, int rows, int width, const void* gamma,
                                   const void* x, const void* dy, void* dx, void* dgamma,
                                   void* dbeta, const void* cache, void* stream);

/* No counterpart in the reference.  The same computation as
 * haste_b200_layer_norm_backward, for callers that cannot let the library allocate: a
 * process whose own arena already owns all device memory, code inside a stream-capture
 * region, or a latency-critical loop that must not hit cudaMalloc's device-wide
 * synchronisation.  The reduction scratch lives in a fixed 2 MiB array inside the library
 * image (held by every GPU that loads the library until the process exits) instead of the
 * grow-only pool, so this call never allocates or frees.
 *   - width must be <= 4096; larger widths return HASTE_B200_ERR_UNSUPPORTED with a message.
 *   - The first call on each device looks up the array's device address (the device of the
 *     pointers must be current); make that first call before starting any stream capture.
 *   - All calls on a device share the one array.  Nothing in it needs to start at zero (each
 *     call overwrites what it later reads), but two calls that overlap on the GPU - different
 *     streams, no ordering between them - race on it and give wrong gradients. */
int haste_b200_layer_norm_backward_noalloc(int dtype, int rows, int width, const void* gamma,
                                           const void* x, const void* dy, void* dx,
                                           void* dgamma, void* dbeta, const void* cache,
                                           void* stream);

/* ---- LayerNormLSTM ----------------------------------------------------- */
/* Replaces layer_norm_lstm::ForwardPass<T>::Run  (lib/haste/layer_norm_lstm.h:75-92,
 * lib/layer_norm_lstm_forward_gpu.cu.cc:276-340).
 *   gamma_Wx, gamma_Rh [4H] (the two rows of the module's [2,4H] gamma: the first
 *   normalises x.W, the second h.R)  gamma_h, beta_h [H]
 *   act_Wx, act_Wx_norm, act_Rh [T,N,4H]  act_c_norm [T,N,H]
 *   cache_Wx, cache_Rh, cache_c [T,N,2]  tmp_Rh [N,4H] */
int haste_b200_layer_norm_lstm_forward(
    int dtype, int training, int T, int N, int C, int H, const void* W, const void* R,
    const void* b, const void* gamma_Wx, const void* gamma_Rh, const void* gamma_h,
    const void* beta_h, const void* x,
    void* h, void* c, void* act_Wx, void* act_Wx_norm, void* cache_Wx, void* act_Rh,
    void* cache_Rh, void* act_c_norm, void* cache_c, void* tmp_Rh, float zoneout_prob,
    const void* zoneout_mask, void* stream);

/* Replaces layer_norm_lstm::BackwardPass<T>::Run  (lib/haste/layer_norm_lstm.h:160-183,
 * lib/layer_norm_lstm_backward_gpu.cu.cc:255-352).  dgamma_Wx, dgamma_Rh [4H], dgamma_h,
 * dbeta_h [H] accumulated; act_Wx, act_Wx_norm, act_Rh, act_c_norm are overwritten. */
int haste_b200_layer_norm_lstm_backward(
    int dtype, int transposed_inputs, int T, int N, int C, int H, const void* W, const void* R,
    const void* b, const void* gamma_Wx, const void* gamma_Rh, const void* gamma_h,
    const void* beta_h, const void* x,
    const void* h, const void* c, const void* dh_new, const void* dc_new, void* dx, void* dW,
    void* dR, void* db, void* dgamma_Wx, void* dgamma_Rh, void* dgamma_h, void* dbeta_h, void* dh,
    void* dc,
    void* act_Wx, void* act_Wx_norm, const void* cache_Wx, void* act_Rh, const void* cache_Rh,
    void* act_c_norm, const void* cache_c, const void* zoneout_mask, void* stream);

/* ---- LayerNormGRU ------------------------------------------------------ */
/* Replaces layer_norm_gru::ForwardPass<T>::Run  (lib/haste/layer_norm_gru.h:72-88,
 * lib/layer_norm_gru_forward_gpu.cu.cc:243-305).  gamma_Wx, gamma_Rh [3H];
 * act_Wx, tmp_Wx_norm [T,N,3H]; act_Rh [T,N,3H]; tmp_Rh_norm [N,3H]. */
int haste_b200_layer_norm_gru_forward(
    int dtype, int training, int T, int N, int C, int H, const void* W, const void* R,
    const void* bx, const void* br, const void* gamma_Wx, const void* gamma_Rh, const void* x,
    void* h, void* v, void* act_Wx, void* cache_Wx, void* tmp_Wx_norm, void* act_Rh, void* cache_Rh,
    void* tmp_Rh_norm, float zoneout_prob, const void* zoneout_mask, void* stream);

/* Replaces layer_norm_gru::BackwardPass<T>::Run  (lib/haste/layer_norm_gru.h:164-184,
 * lib/layer_norm_gru_backward_gpu.cu.cc:246-310).  dgamma_Wx, dgamma_Rh [3H] accumulated;
 * act_Rh is overwritten (it receives the gradient of h.R). */
int haste_b200_layer_norm_gru_backward(
    int dtype, int transposed_inputs, int T, int N, int C, int H, const void* W, const void* R,
    const void* bx, const void* br, const void* gamma_Wx, const void* gamma_Rh, const void* x,
    const void* h, const void* v, const void* dh_new, void* dx, void* dW, void* dR, void* dbx,
    void* dbr, void* dgamma_Wx, void* dgamma_Rh, void* dh, void* dp, void* dq, const void* act_Wx, const void* cache_Wx,
    void* act_Rh, const void* cache_Rh, const void* zoneout_mask, void* stream);

/* ---- LayerNormIndRNN --------------------------------------------------- */
/* Replaces layer_norm_indrnn::ForwardPass<T>::Run  (lib/haste/layer_norm_indrnn.h:38-49,
 * lib/layer_norm_indrnn_forward_gpu.cu.cc:128-213).  gamma [H] (row 0 of the
 * module's [2,H] parameter); act_Wx, workspace [T,N,H]. */
int haste_b200_layer_norm_indrnn_forward(
    int dtype, int training, int T, int N, int C, int H, const void* W, const void* u,
    const void* b, const void* gamma, const void* x, void* h, void* workspace, void* act_Wx,
    void* cache_Wx, float zoneout_prob, const void* zoneout_mask, void* stream);

/* Replaces layer_norm_indrnn::BackwardPass<T>::Run  (lib/haste/layer_norm_indrnn.h:68-83,
 * lib/layer_norm_indrnn_backward_gpu.cu.cc:136-209).  dW assigned. */
int haste_b200_layer_norm_indrnn_backward(
    int dtype, int transposed_inputs, int T, int N, int C, int H, const void* W, const void* u,
    const void* b, const void* gamma, const void* x, const void* h, const void* dh_new,
    void* dx, void* dW, void* du, void* db, void* dgamma, void* dh, void* workspace,
    const void* act_Wx, const void* cache_Wx, const void* zoneout_mask, void* stream);

/* ---- Selective state space operators ------------------------------------ */
/* No counterpart in the reference.  The parts of a state space block, next to the recurrences
 * above: a short causal convolution along time, a scan whose decay and input depend on the data,
 * and a norm fused with the block's gate and residual.
 *
 * Their arguments come in one block each, zeroed by the caller before it is filled; a pointer that
 * is NULL means that the tensor is absent.  A sequence is a view: element (t,n,j) lies at
 * data[t * t_stride + n * n_stride + j] (strides in elements, j unit-strided), so halves of a
 * projection and batch-first tensors are taken as they lie.  Outputs must not overlap inputs,
 * except where said.  dtype is the storage of all sequences (HASTE_B200_F32, BF16 or F16),
 * arithmetic and sums are fp32.  Steps lie less than 2^31 elements apart, T is at most 2^30.  `lengths` [N] (device, 64-bit) ends each row early: from step
 * lengths[n] on (values are clamped to 0..T) inputs are not read, outputs are zero, and the final
 * state is the one after lengths[n] steps.
 * These entry points allocate nothing and keep no state: scratch comes from the caller, so calls
 * may be captured into graphs and issued on any number of streams at once. */
typedef struct {
  void* data;
  long long t_stride, n_stride;
} haste_b200_sequence;

/* y_t[d] = act(bias[d] + sum_k weight[d,k] x_{t-(W-1)+k}[d]), act = SiLU if `silu`, else identity.
 * The steps before the first are `state` (zeros if NULL).  W is 2, 3 or 4.
 *   x, y [T,N,D]  weight [D,W]  bias [D]  state, final_state [N,W-1,D] dense, dtype
 *   final_state may be the same buffer as state.
 * backward: dy, dx [T,N,D], dfinal_state, dstate [N,W-1,D], dweight, dbias like their parameters;
 * dx, dstate and dbias may be NULL.  scratch: haste_b200_causal_conv1d_scratch() floats, aligned to
 * 16 bytes. */
typedef struct {
  int dtype, param_dtype; /* param_dtype: of weight, bias and their gradients; F32 or dtype */
  int T, N, D, W, silu;
  haste_b200_sequence x, y, dy, dx;
  const void *weight, *bias, *state;
  void* final_state;
  const long long* lengths;
  const void* dfinal_state;
  void *dstate, *dweight, *dbias;
  float* scratch;
} haste_b200_causal_conv1d;
int haste_b200_causal_conv1d_forward(const haste_b200_causal_conv1d* args, void* stream);
int haste_b200_causal_conv1d_backward(const haste_b200_causal_conv1d* args, void* stream);
long long haste_b200_causal_conv1d_scratch(const haste_b200_causal_conv1d* args);

/* delta = softplus(dt + dt_bias) (without softplus if `softplus` is 0),
 * h_t[d,s] = exp(delta_t[d] A[d,s]) h_{t-1}[d,s] + delta_t[d] x_t[d] B_t[g,s],  g = d / (D/G),
 * y_t[d] = (sum_s C_t[g,s] h_t[d,s] + skip[d] x_t[d]) * silu(z_t[d]).
 *   x, dt, z, y [T,N,D]   B, C [T,N,G,S]: element (t,n,g,s) at t_stride, n_stride and B_g, C_g
 *   A [D,S], skip [D], dt_bias [D]: float   state, final_state [N,D,S]: float, dense; may be the
 *   same buffer.  S is 1..128, G divides D.
 * checkpoints: what the backward pass starts its pieces from, haste_b200_selective_scan_checkpoints()
 * floats; NULL if there will be none.
 * backward: reads checkpoints, dy and dfinal_state; writes dx, ddt, dz (if z), dB, dC (sequences
 * like B and C with dB_g, dC_g), dA, dskip, ddt_bias (float, like their parameters) and dstate
 * (may be NULL).  scratch: haste_b200_selective_scan_scratch() floats. */
typedef struct {
  int dtype, T, N, D, G, S, softplus;
  haste_b200_sequence x, dt, z, y, B, C;
  long long B_g, C_g;
  const float *A, *skip, *dt_bias, *state;
  float* final_state;
  const long long* lengths;
  float* checkpoints;
  haste_b200_sequence dy, dx, ddt, dz, dB, dC;
  long long dB_g, dC_g;
  const float* dfinal_state;
  float *dA, *dskip, *ddt_bias, *dstate;
  float* scratch;
} haste_b200_selective_scan;
int haste_b200_selective_scan_forward(const haste_b200_selective_scan* args, void* stream);
int haste_b200_selective_scan_backward(const haste_b200_selective_scan* args, void* stream);
long long haste_b200_selective_scan_checkpoints(const haste_b200_selective_scan* args);
/* Floats of scratch that the forward (backward != 0: backward) call needs.  The forward call does without
 * if `scratch` is NULL, at a cost in time where there are few channels. */
long long haste_b200_selective_scan_scratch(const haste_b200_selective_scan* args, int backward);

/* u = x * silu(gate);  r = residual + scale * u;  y = norm(r) * weight + bias
 * (norm: root mean square, or mean and variance if `layer_norm`; eps inside the root).
 *   x, gate, y [T,N,H] dtype   residual, r [T,N,H] residual_dtype (F32 or dtype; without a residual
 *   pass dtype)   scale, weight, bias [H] param_dtype (F32 or dtype); scale needs a residual
 *   stats [T,N,2] float: mean (0 without layer_norm) and 1 / deviation; NULL if there will be no
 *   backward pass; aligned to 8 bytes.  r may be NULL, or the same buffer as residual.  H is 1..8192.
 * backward: reads dy and dr (may be NULL: no gradient of r); writes dx, dgate, dresidual, dscale,
 * dweight, dbias like their tensors.  Any of dx, dgate, dresidual may be NULL.
 * scratch: haste_b200_fused_norm_scratch() floats. */
typedef struct {
  int dtype, residual_dtype, param_dtype, T, N, H, layer_norm;
  float eps;
  haste_b200_sequence x, gate, residual, y, r;
  const void *scale, *weight, *bias;
  float* stats;
  haste_b200_sequence dy, dr, dx, dgate, dresidual;
  void *dscale, *dweight, *dbias;
  float* scratch;
} haste_b200_fused_norm;
int haste_b200_fused_norm_forward(const haste_b200_fused_norm* args, void* stream);
int haste_b200_fused_norm_backward(const haste_b200_fused_norm* args, void* stream);
long long haste_b200_fused_norm_scratch(const haste_b200_fused_norm* args);

/* ---- Gated linear recurrence ---------------------------------------------- */
/* r = sigmoid(gate); with decay: log a = min(decay[d], 0) r, w = sqrt(1 - a^2), without: a = r, w = 1 - a;
 * h_t = a_t h_{t-1} + w_t x_t sigmoid(input_gate_t),  y_t = h_t.  No counterpart in the reference; arguments,
 * sequences, `lengths` and scratch as in the state space operators above.
 *   x, gate, input_gate (may be absent), y [T,N,D]   decay [D] (may be NULL), state, final_state [N,D]: float,
 *   dense; final_state may be the same buffer as state.
 * checkpoints: what the backward pass starts its pieces from, haste_b200_gated_scan_checkpoints() floats; NULL if
 * there will be none.
 * backward: reads checkpoints, dy and dfinal_state; writes dx, dgate, dinput_gate (if input_gate), ddecay (if decay)
 * and dstate (may be NULL); 1 / w is taken as 1 / sqrt(w^2 + 1e-30), and a decay of zero leaves w constant.  scratch: haste_b200_gated_scan_scratch() floats, aligned to 8 bytes. */
typedef struct {
  int dtype, T, N, D;
  haste_b200_sequence x, gate, input_gate, y;
  const float *decay, *state;
  float* final_state;
  const long long* lengths;
  float* checkpoints;
  haste_b200_sequence dy, dx, dgate, dinput_gate;
  const float* dfinal_state;
  float *ddecay, *dstate;
  float* scratch;
} haste_b200_gated_scan;
int haste_b200_gated_scan_forward(const haste_b200_gated_scan* args, void* stream);
int haste_b200_gated_scan_backward(const haste_b200_gated_scan* args, void* stream);
long long haste_b200_gated_scan_checkpoints(const haste_b200_gated_scan* args);
/* Floats of scratch that the forward (backward != 0: backward) call needs.  The forward call does without
 * if `scratch` is NULL, at a cost in time where there are few channels. */
long long haste_b200_gated_scan_scratch(const haste_b200_gated_scan* args, int backward);

/* ---- Projections ---------------------------------------------------------- */
/* y[m,h] = act(sum_c x[m,c] weight[h,c] + bias[h]) + residual[m,h], on the tensor cores, sums in fp32 (fp32 operands:
 * accurate to fp32 rounding, those below 2^-110 to within 2^-134; an infinite one makes NaN of its row's or column's sums
 * from nine rows on and in gradients, what the formula has in up to eight).  No counterpart in the reference, whose
 * layers project inside.
 *   x [M,C], residual, y [M,H]: rows x_ld, residual_ld, y_ld elements apart, elements of a row next to each other
 *   weight [H,C] dense, dtype; C and H are 1 to 2^20 - 1, M is at most 2^30   bias [H] param_dtype (F32 or dtype; may be NULL)
 *   residual (may be NULL) and y have out_dtype: F32 or dtype.  residual may be the same buffer as y, with the same rows.
 *   pre [M,H] dense, dtype: the sums with bias, written for the backward pass (where one is infinite, or beyond dtype's
 *   range, slopes are their limits, 0 or 1); NULL if there will be none, or if activation is HASTE_B200_IDENTITY.
 * backward: dy [M,H] out_dtype, rows dy_ld apart; its product with the slopes is rounded to dtype.  Writes dx [M,C] (rows
 * dx_ld apart; may be NULL), dweight [H,C] (may be NULL) in dtype and dbias [H] in param_dtype (may be NULL).  The
 * residual's gradient is dy.
 * scratch: haste_b200_linear_scratch() bytes, aligned to 256, asked for with all other members set (backward: dx,
 * dweight, dbias not NULL if they will be written).  The calls keep nothing and may be captured. */
#define HASTE_B200_IDENTITY 0
#define HASTE_B200_RELU 1
#define HASTE_B200_SILU 2
#define HASTE_B200_GELU 3 /* x Phi(x), the normal distribution's own */
#define HASTE_B200_TANH 4
#define HASTE_B200_SIGMOID 5
typedef struct {
  int dtype, param_dtype, out_dtype, activation;
  int M, C, H;
  const void *x, *weight, *bias, *residual;
  long long x_ld, residual_ld;
  void* y;
  long long y_ld;
  void* pre;
  const void* dy;
  long long dy_ld;
  void* dx;
  long long dx_ld;
  void *dweight, *dbias;
  void* scratch;
} haste_b200_linear;
int haste_b200_linear_forward(const haste_b200_linear* args, void* stream);
int haste_b200_linear_backward(const haste_b200_linear* args, void* stream);
long long haste_b200_linear_scratch(const haste_b200_linear* args, int backward);

/* ---- Gradient norm and clipping ------------------------------------------- */
/* norm = sqrt(sum over all gradients of their squares);  out = data * min(1, max_norm / (norm + 1e-6)), with a factor
 * of 1 where max_norm is infinite.  No counterpart in the reference.
 * `gradients` is host memory, read before the call returns; data, out and norm (one float) are on the device.  A
 * gradient is `numel` elements that lie next to each other; out (of out_dtype) may be data itself, of its own type, and
 * must otherwise overlap no gradient and no other out.  A norm that is not finite scales as the formula says: infinite ones to zero
 * (and infinite values to NaN), a NaN to NaN.  scratch: haste_b200_grad_norm_scratch() floats, aligned to 8 bytes.
 * The calls allocate nothing, keep nothing and may be captured. */
typedef struct {
  const void* data;
  void* out;
  long long numel;
  int dtype, out_dtype;
} haste_b200_gradient;
int haste_b200_grad_norm(const haste_b200_gradient* gradients, int count, float* norm, float* scratch, void* stream);
int haste_b200_clip_gradients(const haste_b200_gradient* gradients, int count, float max_norm, float* norm,
                              float* scratch, void* stream);
long long haste_b200_grad_norm_scratch(const haste_b200_gradient* gradients, int count);

/* ---- Dense contraction (exposed for tests and benchmarks) --------------- */
/* C[m,n] (+)= sum_k A(m,k) B(k,n);  A(m,k) at a[m*a_rs + k*a_cs],
 * B(k,n) at b[k*b_rs + n*b_cs], C row-major with leading dimension ldc.
 * This is the library's replacement for the cuBLAS calls of lib/blas.h:48-61. */
int haste_b200_gemm(int dtype, int M, int N, int K, const void* a, long long a_rs,
                    long long a_cs, const void* b, long long b_rs, long long b_cs, void* c,
                    long long ldc, int accumulate, void* stream);

#ifdef __cplusplus
}
#endif
#endif /* HASTE_B200_H_ */
