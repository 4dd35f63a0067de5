/*
 * salt_b200 — C ABI of the B200 (sm_100a) implementation of SALT's integer event-driven
 * forward pass and its float chunked affine scan.
 *
 * The reference (Salt-Shio/Spiking-Affine-Lazy-Training) is pure Python/JAX; it has no C
 * interface.  Each entry point below replaces one reference Python call (cited per entry);
 * a host binding (ctypes here, a jax.ffi custom-call handler or cgo elsewhere) passes plain
 * device pointers and sizes.  No torch, JAX or C++ types cross this boundary.
 *
 * Conventions
 *   - All array pointers are DEVICE pointers unless a comment says "host".
 *   - Batch-major layouts: a stream is (batch, capacity) row-major; per-neuron arrays are
 *     (batch, n_neurons) with neuron = oc * h_out * w_out + oy * w_out + ox for conv layers
 *     (salt_core/layers/conv.py:104-112).
 *   - Every call is asynchronous on `stream` (a cudaStream_t) and returns a status; argument
 *     errors are reported before anything is enqueued.  Capacity overflow is NOT an error: it
 *     is reported through `fits` / `needed_queue` / `n_real`, as salt_core/capacity.py:60-63.
 *   - Streams written by this library do not materialise their pad entries: entries at or
 *     beyond min(n_real, capacity) are pads whose time is 1e12 and source 0
 *     (salt_core/stream.py:42-45).  `virtual_pads = 1` tells a consumer to read them that way.
 */
#ifndef SALT_B200_H
#define SALT_B200_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

typedef int32_t salt_status;
enum {
  SALT_OK = 0,
  SALT_BAD_ARG = 1,          /* invalid geometry, bit widths, sizes or null pointers */
  SALT_CUDA_ERROR = 2,       /* a CUDA runtime call failed; see salt_last_error() */
  SALT_NO_DEVICE = 3,        /* no sm_100 device is visible */
  SALT_WORKSPACE_TOO_SMALL = 4
};

enum { SALT_ROUND = 0, SALT_TRUNCATE = 1 };  /* salt_core/quant/fixed_point.py:20-23 */
enum { SALT_WRAP = 0, SALT_SATURATE = 1 };   /* salt_core/quant/fixed_point.py:26-29 */

/* Fixed-point settings of one quantised layer (salt_core/quant/params.py:9-21). */
typedef struct {
  int32_t f_a, f_V, i_V;   /* f_a <= 15, i_V + f_V <= 30 (fixed_point.py:15-17) */
  int32_t round_mode;      /* SALT_ROUND / SALT_TRUNCATE (network-wide in the reference) */
  int32_t overflow_mode;   /* SALT_WRAP / SALT_SATURATE */
  int32_t lut_len;         /* length of decay_table_int */
  int32_t has_vth;         /* 0: v_th_int is None, the layer never fires */
  int32_t q_bits;          /* 8 / 16 when every weight code fits int8 / int16, else 32; lets
                              the kernels stage narrower weights in shared memory */
  int32_t needs_tail;      /* 1 when some v_th_int <= 0 or some decay code is outside
                              [0, 2^f_a): only then can catch-up/identity/pad columns fire, and
                              the kernels must walk them (salt_core/quant/scan.py:65-80 applies
                              every column).  Setting it when not needed is always correct. */
} salt_quant_desc;

/* ConvLayer geometry and capacity (salt_core/layers/conv.py:23-99). */
typedef struct {
  int32_t ic, h_in, w_in, oc, k, s, p;
  int32_t max_queue_len, max_out_spikes, max_extra_steps;
} salt_conv_desc;

/* FCLayer geometry and capacity (salt_core/layers/fc.py:23-41). */
typedef struct {
  int32_t n_in, n_out;
  int32_t max_out_spikes, max_extra_steps;
} salt_fc_desc;

/* Input event stream of a layer: (batch, capacity) times/sources plus n_real per sample.
 * salt_core/stream.py:16-21 EventStream (event_gain is identically 1 on the integer path). */
typedef struct {
  const float *times;
  const int32_t *src;
  const int32_t *n_real;
  int32_t capacity;
  int32_t virtual_pads;
} salt_stream_in;

/* Output stream of a layer, capacity = the layer's max_out_spikes.  n_real[b] is the total
 * spike count (not clipped), exactly as stream.py:61 reports it. */
typedef struct {
  float *times;
  int32_t *src;
  int32_t *n_real;
} salt_stream_out;

/* Per-sample diagnostics of one layer (batch entries each).  Any pointer may be NULL.
 *   spike_count  LayerDiag.spike_count (layers/base.py:73-79)
 *   needed_queue LayerDiag.needed["max_queue_len"] = max n_real + 1 (layers/conv.py:137-141)
 *   overflowed   any(QuantLayerResult.overflowed) (example/quant_run.py:88-89)
 *   vmin / vmax  min/max of v_unfitted_min/max over neurons (example/quant_run.py:90-93)
 *   fits         Capacity.fits (capacity.py:60-63) */
typedef struct {
  int32_t *spike_count, *needed_queue, *overflowed, *vmin, *vmax, *fits;
} salt_layer_stats;

/* ---------------------------------------------------------------- conv layer
 * Replaces ConvLayer.forward with QuantBackend (salt_core/layers/conv.py:124-149 calling
 * build_conv_structure connectivity/conv.py:128-172, QuantBackend.scan quant/backend.py:31-53,
 * extract_output_events_conv stream.py:84-100, _layer_diag layers/base.py:73-79).
 *   q    (oc, ic, k, k) int32 weight codes      lut (lut_len) int32 decay_table_int
 *   vth  (oc*h_out*w_out) int32, or NULL when has_vth == 0
 *   v_final (batch, n_neurons) int32 register values after the queue (QuantLayerResult.v_final)
 * The workspace must be at least salt_conv_layer_workspace_size() bytes, 256-byte aligned. */
salt_status salt_conv_layer_workspace_size(const salt_conv_desc *layer, const salt_quant_desc *quant,
                                           int32_t batch, int32_t in_capacity, size_t *bytes);
salt_status salt_conv_layer_forward(const salt_conv_desc *layer, const salt_quant_desc *quant,
                                    const int32_t *q, const int32_t *lut, const int32_t *vth,
                                    int32_t batch, const salt_stream_in *in, salt_stream_out *out,
                                    int32_t *v_final, const salt_layer_stats *stats,
                                    void *workspace, size_t workspace_bytes, void *stream);

/* Size of the library's fixed device scratch (64 MiB), the largest conv workspace that
 * salt_conv_layer_forward_noalloc accepts. */
#define SALT_NOALLOC_SCRATCH_BYTES ((size_t)64 << 20)

/* salt_conv_layer_forward without a caller workspace, for callers that cannot allocate device
 * memory at call time (a plugin host that hands out no scratch buffers, a loop that must not
 * call cudaMalloc).  No counterpart in the reference: there JAX owns every buffer.
 *   - Same arguments, results and errors as salt_conv_layer_forward minus the workspace; the
 *     layer's scratch lives in a fixed SALT_NOALLOC_SCRATCH_BYTES device array inside the
 *     library, and the call allocates no device memory.
 *   - A layer whose salt_conv_layer_workspace_size exceeds SALT_NOALLOC_SCRATCH_BYTES is
 *     rejected with SALT_WORKSPACE_TOO_SMALL before anything is enqueued.
 *   - Nothing has to start at zero: every call clears the counters it uses, on `stream`.
 *   - The first call on a device does a one-time setup (it looks up the scratch's device
 *     address, which loads the module holding it); make that first call before any stream
 *     capture.  The address is kept for the life of the process: a context reset
 *     (cudaDeviceReset) reloads the library's device code and leaves the kept address stale, so
 *     do not call this entry point on a device after resetting it.
 *   - All calls on one device share the one scratch: calls that may overlap in time (other
 *     streams, other host threads) race and corrupt each other's results.  Order them on one
 *     stream, or with events. */
salt_status salt_conv_layer_forward_noalloc(const salt_conv_desc *layer,
                                            const salt_quant_desc *quant, const int32_t *q,
                                            const int32_t *lut, const int32_t *vth, int32_t batch,
                                            const salt_stream_in *in, salt_stream_out *out,
                                            int32_t *v_final, const salt_layer_stats *stats,
                                            void *stream);

/* ---------------------------------------------------------------- traces
 * Replace QuantBackend.scan with trace=True (salt_core/quant/backend.py:31-53 ->
 * run_layer_traced quant/scan.py:83-94) and the event times of salt_core/trace.py:25-55: for
 * every neuron of every sample, the register after each of its L queue columns (conv: L =
 * max_queue_len; fc: L = the input stream capacity), whether it fired there and the time of the
 * column's event (NaN for columns at or past the neuron's real events).  v_steps / spike_mask /
 * event_ms are (batch, n_neurons, L) or NULL.  per_neuron (optional, each pointer optional,
 * (batch, n_neurons) each) gives the first overflowing column (-1: none) with the register before
 * and after it, whether that column fired and its event time — the fields example/quant_run.py
 * (overflow_events, :189-214) reports — plus the unfitted extremes, v_final and the spike count.
 * An analysis path: one thread per neuron rebuilds its queue from the stream. */
typedef struct {
  int32_t *first_overflow;
  int32_t *v_before, *v_after;
  int32_t *spiked;
  float *time_ms;
  int32_t *v_min, *v_max;
  int32_t *v_final, *spike_count;
} salt_neuron_trace;

salt_status salt_conv_layer_trace(const salt_conv_desc *layer, const salt_quant_desc *quant,
                                  const int32_t *q, const int32_t *lut, const int32_t *vth,
                                  int32_t batch, const salt_stream_in *in, int32_t *v_steps,
                                  uint8_t *spike_mask, float *event_ms,
                                  const salt_neuron_trace *per_neuron, void *stream);
salt_status salt_fc_layer_trace(const salt_fc_desc *layer, const salt_quant_desc *quant,
                                const int32_t *q, const int32_t *lut, const int32_t *vth,
                                int32_t batch, const salt_stream_in *in, int32_t *v_steps,
                                uint8_t *spike_mask, float *event_ms,
                                const salt_neuron_trace *per_neuron, void *stream);

/* ---------------------------------------------------------------- fc layer
 * Replaces FCLayer.forward with QuantBackend (salt_core/layers/fc.py:84-101 calling
 * build_fc_structure connectivity/fc.py:20-33, fc_weight_codes :54-61, QuantBackend.scan,
 * extract_output_events_fc stream.py:67-81).
 *   q (n_out, n_in) int32 weight codes; vth (n_out) or NULL; v_final (batch, n_out). */
salt_status salt_fc_layer_workspace_size(const salt_fc_desc *layer, const salt_quant_desc *quant,
                                         int32_t batch, int32_t in_capacity, size_t *bytes);
salt_status salt_fc_layer_forward(const salt_fc_desc *layer, const salt_quant_desc *quant,
                                  const int32_t *q, const int32_t *lut, const int32_t *vth,
                                  int32_t batch, const salt_stream_in *in, salt_stream_out *out,
                                  int32_t *v_final, const salt_layer_stats *stats,
                                  void *workspace, size_t workspace_bytes, void *stream);

/* ---------------------------------------------------------------- dense scan
 * Replaces quant.scan.run_layer (salt_core/quant/scan.py:65-80, :97-132) on materialised
 * (n, L) queues — the Backend.scan plug-in point of salt_core/backend.py:64-74.
 *   a_int (n, L) int32, is_identity (n, L) uint8, q_int (n, L) int32, vth (n) or NULL
 *   spike_mask / overflowed (n, L) uint8 (may be NULL); v_final, vmin, vmax (n) int32. */
salt_status salt_quant_scan_dense(const salt_quant_desc *quant, int32_t n, int32_t L,
                                  const int32_t *a_int, const uint8_t *is_identity,
                                  const int32_t *q_int, const int32_t *vth, uint8_t *spike_mask,
                                  uint8_t *overflowed, int32_t *v_final, int32_t *vmin,
                                  int32_t *vmax, void *stream);

/* The same scan with trace=True (run_layer_traced, salt_core/quant/scan.py:83-94, as
 * QuantBackend.scan calls it, salt_core/quant/backend.py:41-43): v_steps (n, L) int32 receives
 * the register after each column (after a spike's reset); its last column equals v_final. */
salt_status salt_quant_scan_dense_trace(const salt_quant_desc *quant, int32_t n, int32_t L,
                                        const int32_t *a_int, const uint8_t *is_identity,
                                        const int32_t *q_int, const int32_t *vth,
                                        uint8_t *spike_mask, uint8_t *overflowed,
                                        int32_t *v_final, int32_t *vmin, int32_t *vmax,
                                        int32_t *v_steps, void *stream);

/* ---------------------------------------------------------------- network plan
 * A native runtime object that chains layers on the device (salt_core/network.py:93-122
 * run_network, vmapped over the batch as Network.apply_batched :179-183) with every
 * intermediate stream kept in the workspace, optionally replayed as one CUDA graph.
 * Layer parameters are HOST pointers copied to the device at creation. */
typedef struct {
  int32_t kind;            /* 0 conv, 1 fc */
  salt_conv_desc conv;
  salt_fc_desc fc;
  salt_quant_desc quant;
  const int32_t *q_host;   /* weight codes (layout as above) */
  const int32_t *lut_host;
  const int32_t *vth_host; /* per-neuron thresholds, NULL when has_vth == 0 */
} salt_layer_spec;

typedef struct salt_network salt_network;

salt_status salt_network_create(const salt_layer_spec *layers, int32_t n_layers,
                                salt_network **out);
salt_status salt_network_destroy(salt_network *net);
salt_status salt_network_workspace_size(const salt_network *net, int32_t batch,
                                        int32_t in_capacity, size_t *bytes);
/* Runs every layer.  Outputs (device, may be NULL except logits):
 *   logits      (batch, n_last) int32: v_final of the last layer (register values)
 *   spike_count (n_layers, batch) int32, overflowed (n_layers, batch) int32,
 *   vmin/vmax   (n_layers, batch) int32, needed_queue (n_layers, batch) int32,
 *   fits        (batch) int32: AND of Capacity.fits over layers (network.py:116-119). */
salt_status salt_network_forward(salt_network *net, int32_t batch, const salt_stream_in *in,
                                 int32_t *logits, int32_t *spike_count, int32_t *overflowed,
                                 int32_t *vmin, int32_t *vmax, int32_t *needed_queue,
                                 int32_t *fits, void *workspace, size_t workspace_bytes,
                                 void *stream);
/* Part of a forward (no reference counterpart: lets a caller overlap the input transfer with the
 * first layer): layers [layer_begin, layer_end) on rows [row0, row0 + rows) of a batch-`batch`
 * forward planned for first-layer input capacity in_capacity, with that forward's workspace and
 * full-batch output arrays (same layouts as salt_network_forward; only the rows' entries are
 * written).  layer_begin == 0 reads `in` (rows rows, capacity in_capacity); otherwise the part
 * reads what layer layer_begin - 1 left in the workspace for these rows, so parts run in layer
 * order on one stream.  logits and fits are written when layer_end is the last layer.  Running
 * layer 0 on row slices and then the remaining layers on all rows gives the results of
 * salt_network_forward. */
salt_status salt_network_forward_part(salt_network *net, int32_t batch, int32_t in_capacity,
                                      int32_t row0, int32_t rows, int32_t layer_begin,
                                      int32_t layer_end, const salt_stream_in *in,
                                      int32_t *logits, int32_t *spike_count, int32_t *overflowed,
                                      int32_t *vmin, int32_t *vmax, int32_t *needed_queue,
                                      int32_t *fits, void *workspace, size_t workspace_bytes,
                                      void *stream);
/* Number of kernel launches the last salt_network_forward enqueued (for launch accounting). */
int32_t salt_network_last_launch_count(const salt_network *net);
/* Kernel timing of the forwards enqueued while profiling is on: CUDA events are recorded on the
 * launching stream around every conv layer's fused bucket+scan kernel (the dominant kernel) and
 * around every whole layer.  salt_network_profile_read synchronises on those events and writes,
 * per layer, the summed milliseconds of the fused kernel (fused_ms, 0 for FC layers) and of the
 * whole layer (layer_ms), and the number of timed forwards (launches); reset clears them. */
salt_status salt_network_set_profiling(salt_network *net, int32_t enable);
salt_status salt_network_profile_read(salt_network *net, float *fused_ms, float *layer_ms,
                                      int32_t *launches, int32_t reset);

/* ---------------------------------------------------------------- float FC layer
 * Replaces FCLayer.forward with FloatBackend (salt_core/layers/fc.py:84-106 calling
 * build_fc_structure connectivity/fc.py:20-33, fc_float_values :36-51, FloatBackend.scan
 * float/backend.py:16-31 -> float.scan.run_layer float/scan.py:34-50 over process_chunk
 * float/affine.py:99-126, extract_output_events_fc stream.py:67-81, extra_steps_upper_bound
 * float/affine.py:57-88) — the forward values.
 *   w (n_out, n_in) float32 as FCLayer holds it; decay_base (n_out) = float32(1 - 1/tau) per
 *   neuron (all equal for the reference's scalar tau; per-neuron values extend it).
 *   in_gain (batch, capacity) event gains or NULL for all ones (the forward s_spike of an upstream
 *   float layer is 1).  v_final (batch, n_out).  The output stream's gains are 1 for every real
 *   entry and are not written.
 *   stats (optional, each pointer optional): spike_count (batch) = Σ spike_mask;
 *   needed_extra_steps (batch) = LayerDiag.needed["max_extra_steps"]; fits (batch).
 * v_th must be > 0 (a threshold <= 0 fires on padding, which only the reference's fixed step
 * count bounds).  Float results follow the reference within float32 rounding: the scan runs the
 * recurrence v = a*v + b in event order, where the reference composes each chunk's maps first. */
typedef struct {
  int32_t n_in, n_out;
  int32_t chunk_size;       /* FCLayer.chunk_size */
  int32_t max_out_spikes;   /* FCLayer.max_out_spikes */
  int32_t max_extra_steps;  /* FCLayer.max_extra_steps */
  float v_th;               /* FCLayer.v_th */
} salt_float_fc_desc;

typedef struct {
  int32_t *spike_count;
  int32_t *needed_extra_steps;
  int32_t *fits;
} salt_float_layer_stats;

salt_status salt_float_fc_layer_workspace_size(const salt_float_fc_desc *layer, int32_t batch,
                                               int32_t in_capacity, int32_t has_gain,
                                               size_t *bytes);
salt_status salt_float_fc_layer_forward(const salt_float_fc_desc *layer, const float *w,
                                        const float *decay_base, int32_t batch,
                                        const salt_stream_in *in, const float *in_gain,
                                        salt_stream_out *out, float *v_final,
                                        const salt_float_layer_stats *stats, void *workspace,
                                        size_t workspace_bytes, void *stream);

/* ---------------------------------------------------------------- float conv layer
 * Replaces ConvLayer.forward with FloatBackend (salt_core/layers/conv.py:124-149): the queue of
 * build_conv_structure (connectivity/conv.py:128-172), conv_float_values (:187-206), the chunked
 * scan (float/scan.py:67-116, float/affine.py:99-126), spike_step_upper_bound's need
 * (affine.py:57-88) and extract_output_events_conv (stream.py:84-100).  The float forward of the
 * quantisation pipeline: with chunk_size 1 it is the calibration forward of
 * example/quant_run.py:30-44.  w is (oc, ic, k, k) float32; decay_base = float32(1 - 1/tau);
 * in_gain (batch, capacity) may be NULL (all ones).  The output stream's real entries carry gain
 * 1 (the forward value of s_spike), so it has no gain array.  v_th must be finite and > 0. */
typedef struct {
  int32_t ic, h_in, w_in, oc, k, s, p;
  int32_t max_queue_len;    /* ConvLayer.max_queue_len */
  int32_t max_out_spikes;   /* ConvLayer.max_out_spikes */
  int32_t max_extra_steps;  /* ConvLayer.max_extra_steps */
  int32_t chunk_size;       /* ConvLayer.chunk_size */
  float v_th;               /* ConvLayer.v_th */
} salt_float_conv_desc;

typedef struct {
  int32_t *spike_count;         /* (batch) spikes, not clipped to max_out_spikes */
  int32_t *needed_queue;        /* (batch) largest real taps of a position + 1 */
  int32_t *needed_extra_steps;  /* (batch) */
  int32_t *fits;                /* (batch) every need within its knob */
} salt_float_conv_stats;

/* Per-step traces of a float layer (run_layer_traced, float/scan.py:53-64, with trace.py:13-55)
 * and its potential ranges (quant/calibrate.py:16-36 reduces v_steps to these); any pointer may
 * be NULL.  max_steps = ceil(L / chunk_size) + max_extra_steps, L = max_queue_len (conv) or the
 * input capacity (FC).  Ranges are over every step and, for conv layers, every position of a
 * channel; an FC neuron is its own channel. */
typedef struct {
  float *v_steps;       /* (batch, n_neurons, max_steps) potential after each step */
  float *event_ms;      /* (batch, n_neurons, max_steps) first event time of the step; NaN idle */
  uint8_t *spike_mask;  /* (batch, n_neurons, max_steps) */
  float *v_max;         /* (batch, channels) */
  float *v_min;         /* (batch, channels) */
} salt_float_trace;

salt_status salt_float_conv_layer_workspace_size(const salt_float_conv_desc *layer, int32_t batch,
                                                 int32_t in_capacity, size_t *bytes);
salt_status salt_float_conv_layer_forward(const salt_float_conv_desc *layer, const float *w,
                                          float decay_base, int32_t batch,
                                          const salt_stream_in *in, const float *in_gain,
                                          salt_stream_out *out, float *v_final,
                                          const salt_float_conv_stats *stats,
                                          const salt_float_trace *trace, void *workspace,
                                          size_t workspace_bytes, void *stream);

/* Per-step traces and potential ranges of a float FC layer (FCLayer.forward with FloatBackend and
 * trace=True, salt_core/layers/fc.py:84-106); v_final (batch, n_out) may be NULL.  The layer's
 * output stream comes from salt_float_fc_layer_forward. */
salt_status salt_float_fc_layer_trace(const salt_float_fc_desc *layer, const float *w,
                                      const float *decay_base, int32_t batch,
                                      const salt_stream_in *in, const float *in_gain,
                                      float *v_final, const salt_float_trace *trace, void *stream);

/* ---------------------------------------------------------------- sequence operators
 * No reference counterpart: the dense, trained counterpart of the event-driven affine scan.  A
 * token mixer for sequences of feature vectors (binned spike counts, tokens) is a root-mean-square
 * norm, a short causal convolution and a selective state space scan, an affine recurrence
 * h = a h + b whose a and b depend on the token.  Each runs over whole rows of tokens, for single
 * tokens on a pool of states, and backward.
 *
 * Conventions of this section
 *   - Activations are (batch, len, dim); channels are contiguous, batch and token strides are
 *     given in elements, so that slices of one projection need no copy.  They hold SALT_F32,
 *     SALT_F16 or SALT_BF16 (`type`); all arithmetic, sums and states are 32-bit floats, with
 *     exponentials and reciprocals good to about 2 units in the last place.
 *   - n_real (batch, may be NULL = len) gives each row's tokens, clamped to [0, len].  Inputs past
 *     them are never read; outputs past them are written as zero.  A row without tokens returns its
 *     initial state (zero where none is given).
 *   - Arrays without a stride here are contiguous.  batch, len or rows may be 0: a call then does
 *     what is left (weight gradients become zero).
 *   - Gradients of weights are sums over rows in an order fixed by the sizes: no atomics, the same
 *     inputs give the same bits.  `workspace` needs the bytes the matching *_workspace_size
 *     returns (256-byte aligned; may be NULL when that is 0) and no initialisation.
 *   - Outputs may not overlap inputs unless a comment says so, nor may an output's rows overlap
 *     each other (strides that let them are refused). */
enum { SALT_F32 = 0, SALT_F16 = 1, SALT_BF16 = 2 };

/* Root-mean-square norm with the residual's addition, over rows of `dim` <= 16384 elements:
 *   r = x + residual (r = x without one);  residual_out = r;  rstd = 1 / sqrt(mean(r^2) + eps);
 *   out = r * rstd * weight.
 * `type` holds x and out, `residual_type` (`type` or SALT_F32) residual and residual_out,
 * `weight_type` (`type` or SALT_F32) the weight (dim).  r is rounded only where it is stored.
 * residual_out and rstd (rows) may be NULL; residual_out may be residual itself, out may be x.
 * With `scale` given, out is 8 bits (e4m3) instead: each group of `group` (32, 64, 128, 256, or
 * 0 = the whole row) neighbouring elements has scale = max|out| / 448 (at least 2^-149, float32's
 * smallest value; 1 where the group is zero) and out = the nearest e4m3 of value / scale, ties to
 * even, both of them quotients rounded to float32; scale is (rows, ceil(dim / group)) float32. */
typedef struct {
  int32_t rows, dim;
  int32_t type, residual_type, weight_type;
  int32_t group;
  float eps;
  int64_t x_stride, residual_stride, out_stride, residual_out_stride;
  const void *x, *residual, *weight;
  void *out, *residual_out;
  float *rstd, *scale;
} salt_rms_norm_args;

salt_status salt_rms_norm(const salt_rms_norm_args *args, void *stream);

/* Its gradient.  x (`residual_type`) is what was normalised (residual_out), rstd (rows) from the
 * forward; dresidual (may be NULL) is the gradient that reaches residual_out from elsewhere.
 *   h = x * rstd;  dx = rstd * (w dy - h * mean(w dy h)) + dresidual;  dweight = sum_rows dy h.
 * dx (`residual_type`) is the gradient of x and of residual alike, and may be dresidual itself;
 * dweight (dim) float32, may be NULL. */
typedef struct {
  int32_t rows, dim;
  int32_t type, residual_type, weight_type;
  int32_t pad;
  int64_t dy_stride, x_stride, dresidual_stride, dx_stride;
  const void *dy, *x, *weight;
  const float *rstd;
  const void *dresidual;
  void *dx;
  float *dweight;
} salt_rms_norm_backward_args;

salt_status salt_rms_norm_backward_workspace_size(const salt_rms_norm_backward_args *args,
                                                  size_t *bytes);
salt_status salt_rms_norm_backward(const salt_rms_norm_backward_args *args, void *workspace,
                                   size_t workspace_bytes, void *stream);

/* Causal convolution of each channel with `width` (1 to 8) taps:
 *   p[t] = bias + sum_k weight[k] x[t - width + 1 + k];  out = p, or p * sigmoid(p) with silu.
 * Tokens before the row come from initial_state (batch, dim, width - 1), oldest first, zero when
 * NULL; final_state (same shape, may be NULL or initial_state itself) receives the last
 * width - 1 inputs.  weight (dim, width) and bias (dim, may be NULL) hold `weight_type` (`type` or
 * SALT_F32); states hold `type`. */
typedef struct {
  int32_t batch, len, dim, width;
  int32_t type, weight_type;
  int32_t silu, pad;
  int64_t x_batch_stride, x_stride, out_batch_stride, out_stride;
  const void *x, *weight, *bias;
  const int32_t *n_real;
  const void *initial_state;
  void *out, *final_state;
} salt_causal_conv_args;

salt_status salt_causal_conv(const salt_causal_conv_args *args, void *stream);

/* One token for each of `batch` rows: row b uses and shifts state[slots[b]] of a pool
 * (n_slots, dim, width - 1); slots NULL = row b is slot b.  A slot outside [0, n_slots) is an
 * empty row: its out is zero and no state changes.  No slot may appear twice. */
typedef struct {
  int32_t batch, dim, width, n_slots;
  int32_t type, weight_type;
  int32_t silu, pad;
  int64_t x_stride, out_stride;
  const void *x, *weight, *bias;
  const int32_t *slots;
  void *state, *out;
} salt_causal_conv_step_args;

salt_status salt_causal_conv_step(const salt_causal_conv_step_args *args, void *stream);

/* Gradient of salt_causal_conv for the gradient dy of out.  dweight (dim, width) and dbias (dim)
 * are float32; dx and dinitial (batch, dim, width - 1) hold `type`; dinitial and dbias may be
 * NULL.  A gradient of final_state is the caller's to add: that state holds inputs as they are, the
 * row's last width - 1 tokens (in front of them, in shorter rows, initial_state's entries). */
typedef struct {
  int32_t batch, len, dim, width;
  int32_t type, weight_type;
  int32_t silu, pad;
  int64_t dy_batch_stride, dy_stride, x_batch_stride, x_stride, dx_batch_stride, dx_stride;
  const void *dy, *x, *weight, *bias;
  const int32_t *n_real;
  const void *initial_state;
  void *dx, *dinitial;
  float *dweight, *dbias;
} salt_causal_conv_backward_args;

salt_status salt_causal_conv_backward_workspace_size(const salt_causal_conv_backward_args *args,
                                                     size_t *bytes);
salt_status salt_causal_conv_backward(const salt_causal_conv_backward_args *args, void *workspace,
                                      size_t workspace_bytes, void *stream);

/* Selective state space scan.  With s[t] = delta[t] + delta_bias, put through
 * softplus(s) = log(1 + exp(s)) with softplus set:
 *   h[t] = exp(s[t] A) h[t-1] + s[t] x[t] B[t];  y = sum_n C[t] h[t] + D x[t];
 *   out = y, or y * z * sigmoid(z) where z is given.
 * h is (dim, state) per row, `state` 1 to 64; A (dim, state, finite), D (dim, may be NULL) and
 * delta_bias (dim, may be NULL) are float32; B and C are (batch, len, groups, state) with contiguous
 * (groups, state), and channel d reads group d / (dim / groups).  initial_state and final_state
 * (batch, dim, state) float32 may be NULL, or be the same array.
 * checkpoints (may be NULL) receives what the backward pass restarts from, the state in front of
 * every SALT_SCAN_CHECKPOINT-th token: (batch, ceil(len / SALT_SCAN_CHECKPOINT), dim, state)
 * float32. */
#define SALT_SCAN_CHECKPOINT 16
typedef struct {
  int32_t batch, len, dim, state, groups;
  int32_t type, softplus, pad;
  int64_t x_batch_stride, x_stride, delta_batch_stride, delta_stride, z_batch_stride, z_stride,
      B_batch_stride, B_stride, C_batch_stride, C_stride, out_batch_stride, out_stride;
  const void *x, *delta, *z, *B, *C;
  const float *A, *D, *delta_bias;
  const int32_t *n_real;
  const float *initial_state;
  void *out;
  float *final_state, *checkpoints;
} salt_selective_scan_args;

salt_status salt_selective_scan_workspace_size(const salt_selective_scan_args *args,
                                               size_t *bytes);
salt_status salt_selective_scan(const salt_selective_scan_args *args, void *workspace,
                                size_t workspace_bytes, void *stream);

/* One token for each of `batch` rows on a pool (n_slots, dim, state) of float32 states; slots as
 * in salt_causal_conv_step. */
typedef struct {
  int32_t batch, dim, state, groups, n_slots;
  int32_t type, softplus, pad;
  int64_t x_stride, delta_stride, z_stride, B_stride, C_stride, out_stride;
  const void *x, *delta, *z, *B, *C;
  const float *A, *D, *delta_bias;
  const int32_t *slots;
  float *pool;
  void *out;
} salt_selective_scan_step_args;

salt_status salt_selective_scan_step(const salt_selective_scan_step_args *args, void *stream);

/* Gradient of salt_selective_scan for the gradient dy of out and dfinal (batch, dim, state;
 * may be NULL) of final_state, from the forward's inputs and checkpoints.  dx, ddelta, dz hold
 * `type` and share one batch and token stride per array; dB and dC are contiguous
 * (batch, len, groups, state) of `type`; dA, dD, ddelta_bias and dinitial are float32.  dz is
 * needed exactly where z is; dD, ddelta_bias and dinitial may be NULL. */
typedef struct {
  int32_t batch, len, dim, state, groups;
  int32_t type, softplus, pad;
  int64_t x_batch_stride, x_stride, delta_batch_stride, delta_stride, z_batch_stride, z_stride,
      B_batch_stride, B_stride, C_batch_stride, C_stride, dy_batch_stride, dy_stride,
      dx_batch_stride, dx_stride, ddelta_batch_stride, ddelta_stride, dz_batch_stride, dz_stride;
  const void *x, *delta, *z, *B, *C, *dy;
  const float *A, *D, *delta_bias;
  const int32_t *n_real;
  const float *checkpoints, *dfinal;
  void *dx, *ddelta, *dz, *dB, *dC;
  float *dA, *dD, *ddelta_bias, *dinitial;
} salt_selective_scan_backward_args;

salt_status salt_selective_scan_backward_workspace_size(
    const salt_selective_scan_backward_args *args, size_t *bytes);
salt_status salt_selective_scan_backward(const salt_selective_scan_backward_args *args,
                                         void *workspace, size_t workspace_bytes, void *stream);

/* Linear attention with a decay for each head: an affine recurrence whose state is a matrix,
 *   S[t] = exp(log_decay[h]) S[t-1] + k[t]^T v[t];  out[t] = scale * q[t] S[t],
 * with S (dim_k, dim_v) for each row and head.  q is (batch, len, heads, dim_k), k and v are
 * (batch, len, kv_heads, dim_k or dim_v), out (batch, len, heads, dim_v), all with contiguous
 * (heads, dim); head h reads key head h / (heads / kv_heads).  dim_k and dim_v are 1 to 128.
 * log_decay (heads) is float32 and at most 0: greater values count as 0, values under -200 as -200
 * (a decay that float32 rounds to 0).  Rows past n_real have to be memory, whatever it holds.  A NaN
 * or infinity in any input makes those outputs not finite that the recurrence makes so, and no others
 * (no token before it, no head that does not read it): a v its column of out and of the state from its
 * token on.  An infinity, or what overflows float32 on the way, may come out as NaN.  initial_state
 * and final_state (batch, heads, dim_k, dim_v) float32 may be NULL, or be the same array.
 * The workspace, of which the query gives the size, holds
 *   - a copy in parts of bfloat16 of each array (in backward of dout, too) that is not bfloat16 on
 *     boundaries of 16 bytes (address, strides, dim): 2 (bfloat16), 4 (float16) or 6 (float32) bytes
 *     for each of batch * len * heads * dim values, with dim rounded up to 8 and whole even where a
 *     stride is 0;
 *   - where batch * heads is too small to fill the GPU, up to 64 states for each;
 *   - in backward with shared key heads, 4 * batch * len * heads * max(dim_k, dim_v) bytes. */
typedef struct {
  int32_t batch, len, heads, kv_heads, dim_k, dim_v;
  int32_t type;
  float scale;
  int64_t q_batch_stride, q_stride, k_batch_stride, k_stride, v_batch_stride, v_stride,
      out_batch_stride, out_stride;
  const void *q, *k, *v;
  const float *log_decay;
  const int32_t *n_real;
  const float *initial_state;
  void *out;
  float *final_state;
} salt_linear_attention_args;

salt_status salt_linear_attention_workspace_size(const salt_linear_attention_args *args,
                                                 size_t *bytes);
salt_status salt_linear_attention(const salt_linear_attention_args *args, void *workspace,
                                  size_t workspace_bytes, void *stream);

/* One token for each of `batch` rows on a pool (n_slots, heads, dim_k, dim_v) of float32 states;
 * slots as in salt_causal_conv_step. */
typedef struct {
  int32_t batch, heads, kv_heads, dim_k, dim_v, n_slots;
  int32_t type;
  float scale;
  int64_t q_stride, k_stride, v_stride, out_stride;
  const void *q, *k, *v;
  const float *log_decay;
  const int32_t *slots;
  float *pool;
  void *out;
} salt_linear_attention_step_args;

salt_status salt_linear_attention_step(const salt_linear_attention_step_args *args, void *stream);

/* Gradient of salt_linear_attention for the gradient dout of out and dfinal (batch, heads, dim_k,
 * dim_v; may be NULL) of final_state, from the forward's inputs.  With D[t] the gradient of S[t],
 *   dq[t] = scale * S[t] dout[t];  D[t] = scale * q[t]^T dout[t] + exp(log_decay) D[t+1];
 *   dk[t] = D[t] v[t];  dv[t] = k[t] D[t];  dinitial = exp(log_decay) D[0],
 * dk and dv summed over the heads that share a key head.  dq, dk and dv hold `type` with
 * contiguous (heads, dim); dinitial (float32) may be NULL.  log_decay is a constant of the head:
 * it has no gradient here. */
typedef struct {
  int32_t batch, len, heads, kv_heads, dim_k, dim_v;
  int32_t type;
  float scale;
  int64_t q_batch_stride, q_stride, k_batch_stride, k_stride, v_batch_stride, v_stride,
      dout_batch_stride, dout_stride, dq_batch_stride, dq_stride, dk_batch_stride, dk_stride,
      dv_batch_stride, dv_stride;
  const void *q, *k, *v, *dout;
  const float *log_decay;
  const int32_t *n_real;
  const float *initial_state, *dfinal;
  void *dq, *dk, *dv;
  float *dinitial;
} salt_linear_attention_backward_args;

salt_status salt_linear_attention_backward_workspace_size(
    const salt_linear_attention_backward_args *args, size_t *bytes);
salt_status salt_linear_attention_backward(const salt_linear_attention_backward_args *args,
                                           void *workspace, size_t workspace_bytes, void *stream);

/* An array of rows (rows, dim) of `type`, or its transpose, in 8 bits (e4m3) with float32 scales.
 * The output is (rows, dim), or (dim, rows) with `transposed`; each SALT_Q8_GROUP neighbours of an
 * output row share a scale, or with `blocks` each SALT_Q8_GROUP x SALT_Q8_GROUP block of the output
 * does.  Scale and values are those of salt_rms_norm's 8-bit form: max|x| / 448 and the nearest e4m3
 * of x / scale.  scale is (output rows, or blocks of them; ceil(output dim / SALT_Q8_GROUP)),
 * contiguous; out_stride is that of the output's rows. */
#define SALT_Q8_GROUP 128
typedef struct {
  int32_t rows, dim;
  int32_t type, blocks, transposed, pad;
  int64_t x_stride, out_stride;
  const void *x;
  void *out;
  float *scale;
} salt_quantize_q8_args;

salt_status salt_quantize_q8(const salt_quantize_q8_args *args, void *stream);

/* Product of two matrices in 8 bits (e4m3) with a float32 scale for every SALT_Q8_GROUP of the
 * depth k:
 *   out[m][j] = bias[j] + sum_i (x[m][i] x_scale[m][i / G]) (weight[j][i] w[j][i / G]).
 * x is (rows, k) with x_scale (rows, ceil(k / G)), as salt_rms_norm and salt_quantize_q8 write
 * them; weight is (n, k), and w[j] row j / G of weight_scale (ceil(n / G), ceil(k / G)) (blocks),
 * or with `weight_rows` row j of weight_scale (n, ceil(k / G)).  out (rows, n) holds `type`, bias
 * (n, may be NULL) `bias_type` (`type` or SALT_F32).  Products of a group are added up by the
 * tensor cores in 32 bits, groups in float32.  Rows of x and weight that do not start on 16-byte
 * boundaries (address or stride) are first copied, into the workspace. */
typedef struct {
  int32_t rows, n, k;
  int32_t type, bias_type, weight_rows;
  int64_t x_stride, weight_stride, out_stride;
  const void *x;
  const float *x_scale;
  const void *weight;
  const float *weight_scale;
  const void *bias;
  void *out;
} salt_matmul_q8_args;

salt_status salt_matmul_q8_workspace_size(const salt_matmul_q8_args *args, size_t *bytes);
salt_status salt_matmul_q8(const salt_matmul_q8_args *args, void *workspace,
                           size_t workspace_bytes, void *stream);

/* ---------------------------------------------------------------- stream transfer
 * No reference counterpart (the reference's input lives in XLA buffers): copies a batch of event
 * streams from PINNED host memory to the device, moving each sample's row only up to
 * min(n_real, capacity).  host_times / host_src: (batch, host_pitch) rows in page-locked memory
 * (cudaHostAlloc / cudaMallocHost / cudaHostRegister; rejected with SALT_BAD_ARG otherwise);
 * n_real: (batch) DEVICE array (copy it first); dev_times / dev_src: (batch, capacity) device
 * rows, whose pad entries are left as they were.  Exact whenever no layer reads pad entries: true
 * unless the first layer has needs_tail set (then copy the full rows instead). */
salt_status salt_stream_h2d_real(const float *host_times, const int32_t *host_src,
                                 int64_t host_pitch, const int32_t *n_real, int32_t batch,
                                 int32_t capacity, float *dev_times, int32_t *dev_src,
                                 void *stream);

/* Optional timing of the float FC layers that the calling thread enqueues: with profiling on,
 * CUDA events are recorded on the launching stream around each layer's speculative segment
 * kernel (the dominant kernel) and around the whole layer.  salt_float_fc_profile_read
 * synchronises on them and writes the summed milliseconds and the number of timed layers;
 * reset clears the sums. */
salt_status salt_float_fc_set_profiling(int32_t enable);
salt_status salt_float_fc_profile_read(float *segment_ms, float *layer_ms, int32_t *layers,
                                       int32_t reset);

/* ---------------------------------------------------------------- runtime plumbing
 * No reference counterpart: under JAX, XLA owns the buffers, streams and executables.  A host
 * that calls this library without XLA (the Python package, a C or cgo caller) takes device
 * memory, pinned host memory, streams, events and graph replay from these thin wrappers of the
 * CUDA runtime, so that nothing else on the host side needs a GPU framework.
 *   - salt_malloc / salt_free: stream-ordered device memory (cudaMallocAsync / cudaFreeAsync on
 *     `stream`; the device's default pool keeps freed memory cached for reuse).  A pointer may
 *     be used on another stream only after that stream waits for `stream`.
 *   - salt_host_alloc / salt_host_free: page-locked host memory, mapped into the device's address
 *     space (what salt_stream_h2d_real reads).
 *   - salt_memcpy_async: any direction (cudaMemcpyDefault: unified addressing tells host from
 *     device); salt_memset_async: bytes.
 *   - streams are created non-blocking (no implicit ordering with the legacy default stream,
 *     which is `stream` = NULL).
 *   - salt_graph_*: records everything enqueued on `stream` between begin and end (a
 *     non-default stream; nothing may synchronise meanwhile) and replays it with one launch. */
salt_status salt_malloc(size_t bytes, void *stream, void **ptr);
salt_status salt_free(void *ptr, void *stream);
salt_status salt_host_alloc(size_t bytes, void **ptr);
salt_status salt_host_free(void *ptr);
salt_status salt_memcpy_async(void *dst, const void *src, size_t bytes, void *stream);
salt_status salt_memset_async(void *ptr, int32_t value, size_t bytes, void *stream);
salt_status salt_device_count(int32_t *count);
salt_status salt_set_device(int32_t device);
salt_status salt_get_device(int32_t *device);
salt_status salt_device_synchronize(void);
salt_status salt_stream_create(void **stream);
/* A non-blocking stream whose blocks the scheduler prefers (the device's greatest priority):
 * for transfers that must overlap a kernel already filling the GPU. */
salt_status salt_stream_create_high_priority(void **stream);
salt_status salt_stream_destroy(void *stream);
salt_status salt_stream_synchronize(void *stream);
salt_status salt_stream_wait_event(void *stream, void *event);
salt_status salt_event_create(int32_t timing, void **event);
salt_status salt_event_destroy(void *event);
salt_status salt_event_record(void *event, void *stream);
salt_status salt_event_synchronize(void *event);
/* *done = 1 when the work before the event's last record has finished, else 0 (no waiting). */
salt_status salt_event_query(void *event, int32_t *done);
salt_status salt_event_elapsed_ms(void *start, void *stop, float *ms);
salt_status salt_graph_begin_capture(void *stream);
salt_status salt_graph_end_capture(void *stream, void **graph_exec);
salt_status salt_graph_launch(void *graph_exec, void *stream);
salt_status salt_graph_destroy(void *graph_exec);

/* Library facts and errors (host). */
const char *salt_last_error(void);
const char *salt_version(void);
/* Kernel launches enqueued by this thread since the last reset (for launch accounting). */
int64_t salt_launch_counter(int32_t reset);

#ifdef __cplusplus
}
#endif
#endif /* SALT_B200_H */
