/*
 * voxtral_tts_hip.h - C ABI of the MI355X (gfx950) backend for the
 * voxtral-tts.c LLM-backbone / acoustic-transformer hot path.
 *
 * The entry points mirror, one for one, the GPU backend interface of the
 * reference (voxtral_tts_cuda.h:89-185): same argument order and meaning,
 * same host-pointer / device-pointer conventions, same `int` 0 / -1 results
 * for init and uploads and `void` compute entry points.  The reference
 * declaration each one replaces is cited at its prototype.  Entry points with
 * no counterpart in the reference are grouped at the end and say so.
 *
 * Plain C, no HIP or torch types in any signature: device memory is passed as
 * `void *` / `float *` addresses obtained from tts_hip_alloc (or from any
 * other allocator of the same HIP device).
 *
 * One global context, not thread-safe, one internal stream; every entry
 * point that takes host pointers is synchronous, every entry point that
 * takes device pointers is asynchronous on the internal stream (call
 * tts_hip_sync) - the conventions of the reference backend.
 */
#ifndef VOXTRAL_TTS_HIP_H
#define VOXTRAL_TTS_HIP_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define TTS_HIP_DEC_LAYERS 26
#define TTS_HIP_AC_LAYERS  3

/* ---- host-side weight structs consumed through `void *` -------------------
 * Field order and types are the upload ABI: they equal tts_dec_layer_t /
 * tts_decoder_t (voxtral_tts.h:101-125) and tts_ac_layer_t / tts_acoustic_t
 * (voxtral_tts.h:131-165), so a pointer to the reference's structs can be
 * passed unchanged. */
typedef struct {
    uint16_t *wq_bf16;        /* [4096, 3072] */
    uint16_t *wk_bf16;        /* [1024, 3072] */
    uint16_t *wv_bf16;        /* [1024, 3072] */
    uint16_t *wo_bf16;        /* [3072, 4096] */
    float *attention_norm;    /* [3072] */
    uint16_t *w1_bf16;        /* [9216, 3072] gate */
    uint16_t *w2_bf16;        /* [3072, 9216] down */
    uint16_t *w3_bf16;        /* [9216, 3072] up */
    float *ffn_norm;          /* [3072] */
} tts_hip_host_layer_t;

typedef struct {
    uint16_t *tok_embeddings_bf16;                    /* [131072, 3072] or NULL */
    tts_hip_host_layer_t layers[TTS_HIP_DEC_LAYERS];
    float *norm;                                      /* [3072] */
} tts_hip_host_decoder_t;

typedef struct {
    float *time_inv_freq;              /* [1536] */
    uint16_t *input_proj_bf16;         /* [3072, 36] */
    uint16_t *time_proj_bf16;          /* [3072, 3072] */
    uint16_t *llm_proj_bf16;           /* [3072, 3072] */
    uint16_t *semantic_out_bf16;       /* [8320, 3072] */
    float *semantic_out_bias;          /* [8320] or NULL */
    uint16_t *acoustic_out_bf16;       /* [36, 3072] */
    float *norm;                       /* [3072] */
    tts_hip_host_layer_t layers[TTS_HIP_AC_LAYERS];
} tts_hip_host_acoustic_t;

/* Audio codec decoder weights: field order and types equal tts_conv_t / tts_codec_layer_t /
 * tts_codec_t (voxtral_tts.h:172-225), so a pointer to the reference's struct can be passed
 * unchanged.  All tensors fp32 (weight norm already folded, voxtral_tts_codec.c:38-57). */
typedef struct {
    float *weight;            /* conv1d [out_ch, in_ch, kernel]; transposed [in_ch, out_ch, kernel] */
    float *bias;              /* [out_ch] or NULL */
    int in_ch, out_ch, kernel, stride, is_transpose;
} tts_hip_host_conv_t;

typedef struct {
    float *wq, *wk, *wv, *wo; /* [1024, 1024] */
    float *q_norm, *k_norm;   /* [1024] or NULL */
    float *attention_norm;    /* [1024] */
    float *w1, *w2, *w3;      /* [4096, 1024] [1024, 4096] [4096, 1024] */
    float *ffn_norm;          /* [1024] */
    float *attn_scale, *ffn_scale;   /* [1024] layer scale, or NULL */
    int window_size;
} tts_hip_host_codec_layer_t;

typedef struct {
    float *semantic_embedding;                 /* [8192, 256] */
    tts_hip_host_conv_t input_conv;            /* 292 -> 1024, k 3, s 1 */
    tts_hip_host_codec_layer_t transformers[8];
    tts_hip_host_conv_t stage_convs[4];        /* 3 used: transposed 1024 -> 1024, k 4, s 2 */
    tts_hip_host_conv_t output_proj;           /* 1024 -> 240, k 7, s 1 */
    float alibi_slopes[8];
} tts_hip_host_codec_t;

/* ---- exported context (replaces the fields of `g_cuda` that code outside the
 * backend touches: voxtral_tts_cuda.h:51-54,78 read at voxtral_tts_llm.c:380-381) */
typedef struct {
    float *kv_cache_k_gpu;    /* f32 [26, kv_cache_max, 1024] */
    float *kv_cache_v_gpu;
    int kv_cache_max;
    int initialized;
    int n_cu;                 /* compute units of the device */
    int dec_layers_uploaded;
    int ac_layers_uploaded;
} tts_hip_ctx_t;

extern tts_hip_ctx_t g_hip;

/* ---- init / upload / teardown -------------------------------------------- */

/* replaces tts_cuda_init (voxtral_tts_cuda.h:89). Idempotent. 0 / -1. */
int tts_hip_init(int kv_cache_max);
/* replaces tts_cuda_upload_llm_weights (voxtral_tts_cuda.h:92); decoder_ptr is a
 * tts_decoder_t * / tts_hip_host_decoder_t *.  Copies; the host keeps ownership. */
int tts_hip_upload_llm_weights(void *decoder_ptr);
/* replaces tts_cuda_upload_acoustic_weights (voxtral_tts_cuda.h:93). */
int tts_hip_upload_acoustic_weights(void *acoustic_ptr);
/* replaces tts_cuda_free (voxtral_tts_cuda.h:96). */
void tts_hip_free(void);
/* replaces tts_cuda_available (voxtral_tts_cuda.h:99). */
int tts_hip_available(void);

/* ---- linear ---------------------------------------------------------------- */

/* replaces tts_cuda_linear_bf16 (voxtral_tts_cuda.h:109-111): y = x W^T, x and y
 * each host or device, W_gpu device bf16 [out_dim, in_dim]; W_gpu == NULL
 * uploads W_bf16 from the host for the call. */
void tts_hip_linear_bf16(float *y, const float *x, const uint16_t *W_bf16,
                         int seq_len, int in_dim, int out_dim, const void *W_gpu);

/* ---- kernel-level operators on device pointers ---------------------------- */

/* replaces tts_cuda_rms_norm (voxtral_tts_cuda.h:118-119) */
void tts_hip_rms_norm(float *d_out, const float *d_x, const float *d_weight,
                      int seq_len, int dim, float eps);
/* replaces tts_cuda_apply_rope (voxtral_tts_cuda.h:122-123); d_freqs is
 * f32 [seq, head_dim/2, 2] (cos, sin) and IS honoured (the reference ignores it). */
void tts_hip_apply_rope(float *d_x, const float *d_freqs, int seq, int heads, int head_dim);
/* replaces tts_cuda_compute_rope_freqs (voxtral_tts_cuda.h:126-127), a stub in
 * the reference; here it fills d_freqs for positions start_pos..start_pos+seq-1. */
void tts_hip_compute_rope_freqs(float *d_freqs, int start_pos, int seq, int dim, float theta);
/* replaces tts_cuda_silu_mul (voxtral_tts_cuda.h:130) */
void tts_hip_silu_mul(float *d_gate, const float *d_up, int n);
/* replaces tts_cuda_add_inplace (voxtral_tts_cuda.h:133) */
void tts_hip_add_inplace(float *d_a, const float *d_b, int n);
/* replaces tts_cuda_causal_attention_decode (voxtral_tts_cuda.h:136-139);
 * kv_cache_stride is the row stride in floats (0 = n_kv_heads*head_dim). */
void tts_hip_causal_attention_decode(float *d_out, const float *d_Q, const float *d_K_cache,
                                     const float *d_V_cache, int seq_k, int n_heads,
                                     int n_kv_heads, int head_dim, float scale,
                                     int kv_cache_stride);
/* replaces tts_cuda_causal_attention_prefill (voxtral_tts_cuda.h:142-145).  With the model's head
 * counts and 8 or more queries it runs on the matrix cores, from tile images of K and V that a first
 * kernel writes into a buffer of the library's own (8 x ceil((start_pos + seq_len) / 32) x 32 KB,
 * allocated when a call needs more than any before it). */
void tts_hip_causal_attention_prefill(float *d_out, const float *d_Q, const float *d_K,
                                      const float *d_V, int seq_len, int start_pos,
                                      int n_heads, int n_kv_heads, int head_dim, float scale);
/* replaces tts_cuda_bidirectional_attention (voxtral_tts_cuda.h:148-150) */
void tts_hip_bidirectional_attention(float *d_out, const float *d_Q, const float *d_K,
                                     const float *d_V, int seq_len, int n_heads,
                                     int n_kv_heads, int head_dim, float scale);
/* replaces tts_cuda_embed_token (voxtral_tts_cuda.h:153-154) */
void tts_hip_embed_token(float *d_out, const void *d_embeddings_bf16, int token_id, int dim);

/* ---- backbone --------------------------------------------------------------- */

/* replaces tts_cuda_llm_forward (voxtral_tts_cuda.h:161-162): one decode step
 * at cache position pos; host pointers; synchronous. */
void tts_hip_llm_forward(float *out_hidden, const float *input_embed, int pos);
/* replaces tts_cuda_llm_prefill (voxtral_tts_cuda.h:165): fills cache rows
 * start_pos..start_pos+seq_len-1 on the device; host pointer; synchronous. */
void tts_hip_llm_prefill(const float *embeds, int seq_len, int start_pos);

/* ---- acoustic transformer -------------------------------------------------- */

/* replaces tts_cuda_predict_velocity (voxtral_tts_cuda.h:172-174) */
void tts_hip_predict_velocity(float *out_velocity, const float *x_t,
                              const float *llm_hidden, float t_val);

/* ---- transfers --------------------------------------------------------------- */

/* replace tts_cuda_to_device / to_host / memset / alloc / free_ptr / sync
 * (voxtral_tts_cuda.h:180-185) */
void tts_hip_to_device(void *d_dst, const void *h_src, size_t bytes);
void tts_hip_to_host(void *h_dst, const void *d_src, size_t bytes);
void tts_hip_memset(void *d_ptr, int value, size_t bytes);
void *tts_hip_alloc(size_t bytes);
void tts_hip_free_ptr(void *d_ptr);
void tts_hip_sync(void);

/* ==== entry points with no counterpart in the reference ===================== */

/* Upload only the first n_layers decoder layers (1..26); used for one-layer
 * and few-layer configurations.  Sources may be host or device pointers. */
int tts_hip_upload_llm_weights_n(void *decoder_ptr, int n_layers);
/* Upload one decoder layer (index 0..25) from host or device pointers. */
int tts_hip_upload_llm_layer(int layer, const tts_hip_host_layer_t *src);
/* Final-norm weights f32 [3072], host or device pointer. */
int tts_hip_upload_llm_norm(const float *norm);

/* One decode step on device-resident buffers, asynchronous on the internal
 * stream: d_input_embed f32 [3072] -> d_out_hidden f32 [3072]. */
void tts_hip_llm_forward_device(float *d_out_hidden, const float *d_input_embed, int pos);
/* One decoder layer at batch 1 on a device-resident hidden state (in place),
 * appending row pos of that layer's cache.  Asynchronous. */
void tts_hip_layer_decode(int layer, float *d_hidden, int pos);
/* Prefill that also returns the residual stream after the last layer
 * ([seq_len, 3072], host pointer, may be NULL). */
void tts_hip_llm_prefill_out(const float *embeds, int seq_len, int start_pos, float *out_x);

/* Conditional + unconditional velocity in one batch-2 pass (classifier-free
 * guidance): equals predict_velocity(x_t, llm_hidden, t) and
 * predict_velocity(x_t, 0, t) (voxtral_tts_acoustic.c:345-348). */
void tts_hip_predict_velocity_cfg(float *out_v_cond, float *out_v_uncond, const float *x_t,
                                  const float *llm_hidden, float t_val);
/* One audio frame on the device: semantic head + argmax, 7 Euler steps with
 * CFG from the caller's noise x0[36], FSQ quantisation -> codes[37]
 * (voxtral_tts_acoustic.c:268-373).  Host pointers; synchronous.  out_x
 * (optional) receives the final latent; another NULL is refused. */
void tts_hip_acoustic_frame(int *out_codes, const float *llm_hidden, const float *x0,
                            float *out_x);

/* Audio-code embedding table bf16 [total_rows, 3072] and the first row of each of the 37
 * codebooks (tts_audio_embed_t, voxtral_tts.h:226-236; tts_audio_embed_load,
 * voxtral_tts_voice.c:251-290).  Host or device pointers; copies.  0 / -1. */
int tts_hip_upload_audio_embeddings(const uint16_t *emb_bf16, int total_rows, const int *offsets);
/* replaces tts_audio_embed_forward (voxtral_tts_voice.c:292-315): host codes [37] -> host
 * embedding [3072], the 37 rows summed in codebook order; synchronous. */
void tts_hip_audio_embed(float *out_embed, const int *codes);
/* One turn of the generation loop of voxtral_tts.c:301-321 on the device: backbone step at
 * cache position pos on d_embed (device, f32 [3072]) -> frame of 37 codes from the noise x0
 * (host, f32 [36]) -> embedding of the codes written back to d_embed.  Synchronous; returns
 * the codes (END_AUDIO: codes[0] == 1, the rest 2). */
void tts_hip_generate_frame(int *out_codes, float *d_embed, const float *x0, int pos);

/* Audio codec decoder on the device (the reference runs it on the CPU only).  Upload: codec_ptr
 * is a tts_codec_t * / tts_hip_host_codec_t * (tts_codec_load fills it, voxtral_tts_codec.c:
 * 177-270); tensors may be host or device memory; copies.  0 / -1. */
int tts_hip_upload_codec_weights(void *codec_ptr);
/* replaces tts_codec_decode (voxtral_tts_codec.c:389-503): host codes [n_frames, 37] ->
 * *out_samples, a malloc'ed waveform of *out_n_samples = n_frames * 1920 floats that the caller
 * frees (NULL / 0 on failure); synchronous.  At most 4096 frames per call. */
void tts_hip_codec_decode(const int *codes, int n_frames, float **out_samples, int *out_n_samples);
/* The same with device buffers (d_codes [n_frames, 37], d_samples [n_frames * 1920]), queued
 * on the library's stream without synchronising; 0 / -1. */
int tts_hip_codec_decode_device(const int *d_codes, int n_frames, float *d_samples);

/* Checkpoint file -> device in one call, in place of the host-side loading that precedes
 * the uploads in the reference (safetensors_open / safetensors_find / safetensors_data,
 * voxtral_tts_safetensors.c:204-405; tts_decoder_load, voxtral_tts_llm.c:45-100;
 * tts_acoustic_load, voxtral_tts_acoustic.c:40-130; tts_audio_embed_load,
 * voxtral_tts_voice.c:251-290).  Maps the .safetensors file and uploads what it holds under
 * the reference's tensor names: backbone layers 0..n-1 (as many consecutive ones as are
 * present) with norm.weight and the token embeddings, the acoustic transformer, the
 * audio-code embedding table, the codec decoder (tts_codec_load, voxtral_tts_codec.c:177-270,
 * weight norm folded).  Returns a bit mask (1 backbone, 2 acoustic, 4 audio-code embeddings,
 * 8 codec decoder) or -1; tts_hip_init first. */
int tts_hip_load_safetensors(const char *path);
/* Looks one tensor of a .safetensors file up without touching the GPU (safetensors_find,
 * voxtral_tts_safetensors.c:330-345): 0 and dtype (8 chars), rank, shape (4 entries) and
 * byte size; 1 if the file has no such tensor; -1 if the file cannot be read. */
int tts_hip_safetensors_probe(const char *path, const char *name, char *dtype8, int *rank,
                              long long *shape4, long long *nbytes);

/* y[seq_len, out_dim] = x[seq_len, in_dim] W[out_dim, in_dim]^T on device pointers, like
 * tts_hip_linear_bf16 with device buffers and the same kernels, for callers that cannot allocate
 * device memory (code under HIP graph capture, tight serving loops, harnesses that forbid it).  No
 * counterpart in the reference.  The work area of the matrix-core path (two bf16 planes of x and
 * the partial planes of a K cut) is a fixed array of 16 MiB that every GPU the library runs on
 * holds until the process ends; a product that needs more is refused with an error (use
 * tts_hip_linear_bf16).  Calls no hipMalloc / hipFree.  All calls on one GPU share the array:
 * calls that overlap on one GPU race.  Asynchronous on the library's stream; 0 / -1. */
int tts_hip_linear_bf16_noalloc(float *d_y, const float *d_x, int seq_len, int in_dim, int out_dim,
                                const void *d_W);

/* The table the loader uses when a checkpoint has no `time_embedding.inv_freq`: out[i] =
 * expf(-logf(10000) * i / half_dim) for i < half_dim (the fallback of tts_acoustic_load,
 * voxtral_tts_acoustic.c:48-60).  Host pointer; touches no GPU state. */
void tts_hip_default_time_inv_freq(float *out, int half_dim);

/* Decode schedule: 0 = persistent whole-step kernel (default; a device on which its grid cannot be
 * resident at once runs schedule 1 instead), 1 = one kernel per phase.  Other values are an error
 * and leave the schedule as it is. */
void tts_hip_set_decode_mode(int mode);
/* Prefill schedule: 0 (default) or 1; both run one launch per product and row pass.  (1 used to choose one
 * persistent launch per layer for everything behind the attention, with the same results bit for bit; its
 * dependency waits made it 3-9 % slower at every length, and it is gone.)  Other values are an error.  No
 * counterpart in the reference. */
void tts_hip_set_prefill_mode(int mode);
/* Spin budget of one grid barrier of the whole-step kernel, in ticks of the 100 MHz wall clock
 * (0 = the default of 0.2 s).  When it runs out every workgroup leaves the kernel and the result is
 * invalid.  Entry points with host pointers (tts_hip_llm_forward, tts_hip_generate_frame) report
 * that themselves; after the asynchronous ones (tts_hip_llm_forward_device, tts_hip_layer_decode)
 * it is reported, once, by the next call that waits for the stream: tts_hip_sync, tts_hip_to_host,
 * tts_hip_to_device, tts_hip_memset.
 * The report resets the barrier; the next step starts clean. */
void tts_hip_set_barrier_timeout(unsigned long long ticks);
/* Workgroups of the backbone's whole-step decode kernel: 0 (the default) = the CU count rounded down to
 * a multiple of 8, else a multiple of 8 from 72 up to that.  Waits for the library's stream.  Results
 * agree to rounding, not bit for bit (the attention's key chunks follow the grid).  No counterpart in
 * the reference. */
void tts_hip_set_decode_grid(int workgroups);
/* Workgroups of the acoustic transformer's product kernels: 0 (the default) = one per CU, else
 * 1 .. the CU count.  The results do not depend on it, bit for bit (a unit of 12 weight rows is summed the
 * same way whichever workgroup takes it); a smaller grid leaves CUs to other work and makes a workgroup
 * walk more units.  No counterpart in the reference. */
void tts_hip_set_acoustic_grid(int workgroups);
/* Number of failed calls since init, and the text of the last failure. */
int tts_hip_error_count(void);
const char *tts_hip_last_error(void);

/* The activation format of the sequence-level products: n fp32 values (n even, device pointers,
 * 8-byte aligned) -> two bf16 planes, hi = bf16(x) rounded to nearest even and lo = bf16(x - hi),
 * so that hi + lo carries x to about 2^-17 relative (tts_hip_llm_prefill multiplies every weight tile
 * with both planes, and so does tts_hip_linear_bf16 with seq_len >= 8, out_dim a multiple of 128 and
 * in_dim of 64; except for up to 16 rows with in_dim a multiple of 512 and seq_len * in_dim <= 49152,
 * whose products are fp32 like those of all other shapes).  No counterpart in the
 * reference, whose CPU products read the fp32 activations directly (voxtral_tts_kernels.c:127-138);
 * exported so that the format can be checked bit for bit.  Returns 0, or -1 on error. */
int tts_hip_split_planes(uint16_t *d_hi, uint16_t *d_lo, const float *d_x, size_t n);

/* ==== 4 bits: linear layers and a key/value cache in microscaled floats ====
 * No counterpart in the reference.  The format is MXFP4 of the OCP microscaling specification: a block of
 * 32 consecutive values of a row is 32 codes e2m1 (0, 0.5, 1, 1.5, 2, 3, 4, 6 and a sign) and one scale
 * e8m0, 2^(s - 127).  s = floor(log2 of the block's largest magnitude) - 2 + 127, at least 0; a code is the
 * nearest value's, of two equally near ones the even code, 6 for what lies beyond 6.  A block with an
 * infinity or a NaN in it is held as s = 255 and stands for 32 NaN.
 * A matrix [rows, cols] is d_codes [rows, 64 P] and d_scales [rows, 4 P] bytes with P = cols / 128 rounded
 * up: two codes a byte, the first in its low half, zeros behind the last column.  Codes lie on 16 bytes,
 * scales on 4.  Device pointers only; asynchronous on the library's stream; 0 / -1. */

/* values [rows, cols], x_stride of them apart from row to row (0: cols), fp32 or, with x_bf16, bf16 -> codes
 * and scales.  Values may lie on any multiple of their size; rows up to 2^30, cols up to 2^27. */
int tts_hip_mx4_quantize(uint8_t *d_codes, uint8_t *d_scales, const void *d_x, int x_bf16,
                         int rows, int cols, int x_stride);
/* codes and scales -> the values that they stand for, fp32, exactly; the room between rows is left as it was. */
int tts_hip_mx4_dequantize(float *d_x, const uint8_t *d_codes, const uint8_t *d_scales,
                           int rows, int cols, int x_stride);
/* y[seq_len, out_dim] = x[seq_len, in_dim] W^T, W [out_dim, in_dim] in 4 bits, x and y fp32 and dense: what
 * tts_hip_linear_bf16 is for bf16 weights.  x enters to 2^-21 of the largest of its 32 neighbours at the worst,
 * 2e-8 of a row's norm on values of a normal distribution; sums are fp32: results are off by 1e-7 of their norm.
 * A row of x with an infinity or a NaN in it gives NaN, a sum that leaves fp32 NaN or an infinity of either sign;
 * blocks of x all below 2^-106 lose bits.  y and x do not overlap.
 * seq_len and out_dim up to 2^30, in_dim up to 2^23.  More than a few rows use the library's work area, which
 * grows by allocation when a call needs more than any before it. */
int tts_hip_linear_mx4(float *d_y, const float *d_x, const uint8_t *d_codes, const uint8_t *d_scales,
                       int seq_len, int in_dim, int out_dim);

/* One layer's key/value cache in 4 bits: codes [n_kv_heads, max_rows, head_dim / 2] and scales
 * [n_kv_heads, max_rows, head_dim / 32], the caller's device memory.  head_dim 64, 128, 192 or 256.  Only the
 * struct is read from host memory, during the call. */
typedef struct {
    uint8_t *k_codes, *k_scales, *v_codes, *v_scales;
    int max_rows, n_kv_heads, head_dim;
} tts_hip_kv4_t;

/* K and V rows [n_rows, n_kv_heads * head_dim] fp32, `stride` floats apart (0: dense), into the cache's rows
 * pos .. pos + n_rows - 1; the others stay as they were. */
int tts_hip_kv4_append(const tts_hip_kv4_t *cache, const float *d_K, const float *d_V,
                       int n_rows, int pos, int stride);
/* The cache's rows pos .. pos + n_rows - 1 back as the fp32 values that they stand for. */
int tts_hip_kv4_read(float *d_K, float *d_V, const tts_hip_kv4_t *cache, int n_rows, int pos, int stride);
/* Causal attention over the cache: query i of Q [seq_len, n_heads * head_dim] sees the rows 0 .. start_pos + i,
 * which hold its own keys and values too (append first); out like Q, on 16 bytes both.  n_heads is a multiple
 * of n_kv_heads.  A decode step is seq_len 1; what tts_hip_causal_attention_decode and _prefill are for an
 * fp32 cache.  A row that a query does not see changes nothing in its result, whatever it holds; a query with
 * an infinity or a NaN in it, and one that sees such a key, gives NaN, a value's NaN the 32 values of its block.
 * Q times scale is formed first, in fp32; a score that leaves fp32 makes NaN, also where it is a large negative
 * one.  Sums are fp32; a weight enters to 2^-22 of itself and no finer than 2^-39 of the column's largest, and
 * values below 2^-124 may count as 0.  Values whose magnitudes differ by more than 2^36 within a head go through
 * fp32 arithmetic, far slower, with the queries that share their work: rounding, not more, may differ with what a
 * later query of the call sees.  out and Q do not overlap.  At most 2^24 rows, 65535 kv heads and 2^19 heads on
 * each.  Where several workgroups share a head's rows their parts meet in the library's work area (70 MB for 2000
 * queries of 32 heads on 8), which grows by allocation when a call needs more than any before it and stays. */
int tts_hip_kv4_attention(float *d_out, const float *d_Q, const tts_hip_kv4_t *cache, int seq_len,
                          int start_pos, int n_heads, float scale);

/* ==== several sequences over one paged key/value cache ====
 * No counterpart in the reference, which serves one utterance at a time.  A pool is bf16 [n_pages, n_kv_heads, page_rows, head_dim], one for K
 * and one for V, the caller's device memory on 16 bytes, a pair of them for every layer.  Row p of a sequence lies in row p % page_rows of
 * the page that the sequence's table names at p / page_rows.  A batch is a number of sequences with their new rows, one token each or a chunk, one
 * sequence's rows behind the other's in every matrix that a call takes; rows behind the last one are left as they were.  A program describes
 * a step once (tts_hip_paged_set) and runs every layer's calls on that.  Values x are fp32 or, with x_bf16, bf16. */
typedef struct {
    int n_pages, page_rows;              /* page_rows: a power of two, 16 .. 2^20 */
    int n_heads, n_kv_heads, head_dim;   /* head_dim 64, 128, 192 or 256; up to 4096 heads on a kv head */
    int window;                          /* a query sees the last `window` rows, its own among them; 0: all */
} tts_hip_paged_shape_t;
typedef struct tts_hip_paged tts_hip_paged_t;

/* A handle for batches of up to max_seqs sequences with max_rows new rows and max_table pages in all.  NULL: refused.  Touches no GPU
 * state; the first tts_hip_paged_set allocates.  tts_hip_paged_free waits for the device. */
tts_hip_paged_t *tts_hip_paged_create(const tts_hip_paged_shape_t *shape, int max_seqs, int max_rows, int max_table);
void tts_hip_paged_free(tts_hip_paged_t *batch);
/* The batch to come: sequence i has rows[i] new rows (none is allowed) behind past[i] cached ones and the pages tables[i * table_stride] ..,
 * host memory that is read during the call.  Page numbers are checked, up to 2^30 rows a sequence; entries of pages that no new row sees are not looked at.
 * Sequences may share pages that they read; a page that new rows go into twice is refused.  The description is on its way to the device when the
 * call returns, behind everything that was queued before; a refused one leaves the handle without a batch.  The call waits for the copy of the
 * handle's last description, and so for what was queued ahead of that one; beside that it takes the host some 6 us for a few sequences,
 * 27 for 64 of them and 120 for 32768 new rows. */
int tts_hip_paged_set(tts_hip_paged_t *batch, int n_seqs, const int *past, const int *rows, const int *tables, int table_stride);
/* The new rows' positions, one after the other (device memory of the handle), for tts_hip_rotary; NULL: no batch. */
const int *tts_hip_paged_positions(const tts_hip_paged_t *batch);

/* How heads are turned by their positions.  rot_dim values of each head turn, the first ones, in pairs: (2 i, 2 i + 1), or with half
 * (i, i + rot_dim / 2); the others pass.  Pair i turns by 2 pi position d_turns[i] (device memory, rot_dim / 2 of them), times
 * `magnitude`.  With d_gain (fp32 [head_dim], device) a head is divided by its root mean square first, sqrt(mean of squares + eps), and
 * multiplied by the gains.  rot_dim 0: only that.  The struct is read from host memory during the call. */
typedef struct {
    const double *d_turns;
    const float *d_gain;
    int rot_dim, half;
    float magnitude, eps;
} tts_hip_rotary_t;

/* d_turns[i] = theta^(-2 i / rot_dim) / 2 pi for i < rot_dim / 2, stretched by `factor` (1: not): a pair that makes fewer than low_turns
 * turns in original_rows positions is divided by it, one that makes more than high_turns is not, in between the share goes with the turns.  original_rows 0
 * and a low_turns above 0 divide all of them.  Each is right to some 2^-52, an angle of it to 2^-24 at positions of 2^28 and 2^-21 at 2^31.
 * The share goes with the turns themselves.  Models are also trained with one that goes with the pair's number i between two bounds: for such
 * a model, or with any other rule, a program fills d_turns itself. */
int tts_hip_rotary_turns(double *d_turns, int rot_dim, double theta, double factor, int original_rows, double low_turns, double high_turns);
/* x [rows, n_heads, head_dim] -> out of the same type, x_stride and out_stride values from row to row (0: dense); row r at position
 * d_positions[r] (any int; device).  out may be x with the same stride, else they do not overlap.  Any alignment that the type allows; rows on
 * four values, head_dim a multiple of 8 and, with half, rot_dim too are fastest.  head_dim even, 2 .. 512.  Angles, position times the turns
 * given, are as exact as fp32 holds them at any position, sums fp32, bf16 results are rounded once.  Values that do not turn and are not normed
 * come out bit for bit, a NaN as a NaN. */
int tts_hip_rotary(void *d_out, const void *d_x, int x_bf16, int rows, int n_heads, int head_dim, int out_stride, int x_stride,
                   const int *d_positions, const tts_hip_rotary_t *how);

/* The new rows' keys and values [rows, n_kv_heads * head_dim], `stride` values from row to row for both (0: dense), into their pages: keys
 * turned and normed as `how` says (NULL: as they are), values as they are, each rounded to bf16 once.  Nothing else in a page changes. */
int tts_hip_paged_append(const tts_hip_paged_t *batch, void *d_k_pages, void *d_v_pages, const void *d_K, const void *d_V, int x_bf16,
                         int stride, const tts_hip_rotary_t *how);
/* Causal attention of the new rows over their sequences: the query at position p sees the rows 0 .. p, or the last `window` of them, its own
 * among them (append first).  Q [rows, n_heads * head_dim], q_stride values from row to row (0: dense, else a multiple of 8), out dense and of
 * Q's type, both on 16 bytes; they do not overlap.  scale > 0.
 * What a query does not see changes nothing in its result, whatever it holds: rows of its pages behind the last one are not even read.  A query
 * with an infinity or a NaN in it, and one that sees a key with a NaN, gives NaN; a key's infinity makes NaN too, or, where the score is
 * -infinity, may leave the key without weight.  A value's infinity or NaN that a query sees makes that value of its result infinite or NaN.
 * Sums and softmax statistics are fp32.  A score that leaves that gives NaN or infinity, and a value times its weight below 2^-126 may count as 0.
 * A mean of finite values is finite: a query whose sums leave fp32 is summed once more with smaller weights (and what counts as 0 is then below
 * 2^-86).  fp32: queries times scale and weights enter to 24 bits, results are off by some 1e-7 of their norm.  bf16: weights enter to 16 bits, and
 * results are rounded once.  A call's results are the same bits each time; beside other sequences in the batch the same query's may differ by
 * these roundings, as the kernel and the parts that its rows are read in are chosen for the batch.  Where several workgroups share a
 * sequence's rows their parts meet in the library's work area, which grows by allocation when a call needs more than any before it and
 * stays. */
int tts_hip_paged_attention(void *d_out, const void *d_Q, int x_bf16, int q_stride, const tts_hip_paged_t *batch, const void *d_k_pages,
                            const void *d_v_pages, float scale);

#ifdef __cplusplus
}
#endif
#endif /* VOXTRAL_TTS_HIP_H */
