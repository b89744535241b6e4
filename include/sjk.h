/* sjk.h - C ABI of the MI355X (gfx950) SJ-KVaRN codec library, libsjk.so.
 *
 * Two layers, both plain C (no torch or HIP C++ types; hipStream_t is passed as void *):
 *
 * 1. The sj_kvarn.h API, same names, types and argument meaning (reference sj_kvarn.h:177-453), so
 *    an engine written against the reference header links against this library unchanged. The codec
 *    routines run as HIP kernels on the current device; the cache objects (layer, pool, sequence)
 *    keep their sink, staging ring and sealed body in device memory (HBM) with the reference's byte
 *    layout, while the rows, queries and outputs handed across the API stay host arrays as in the
 *    reference. One documented difference: sj_kvarn_layer_record() and the ring/sink/body members
 *    of sj_kvarn_layer / sj_kvarn_pool are DEVICE addresses.
 *
 * 2. sjk_hip_*: the device entry points the engine's hot path calls (device pointers, explicit
 *    stream, batched over records, rows, positions and layers). They replace the reference's CUDA
 *    kernels and launcher in sj_kvarn_cuda.cuh:27-151 and the per-layer loops of sj_kvarn.h.
 *
 * Status codes: the SJKVARN_* space of the reference (sj_kvarn.h:332-361) plus SJK_ERR_DEVICE
 * (a HIP call failed) and SJK_ERR_UNSUPPORTED (a shape the kernels are not built for).
 * Every function that returns a status leaves its outputs untouched when it fails before launching.
 */
#ifndef SJK_H
#define SJK_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* ---- format constants (sj_kvarn.h:114-131) ---- */
#define SJKVARN_GROUP_DEFAULT     128
#define SJKVARN_SINK_DEFAULT      128
#define SJKVARN_TAIL_DEFAULT      4096
#define SJKVARN_TAIL_MAX_DEFAULT  8192
#define SJKVARN_ITERS_DEFAULT     16
#define SJKVARN_RED_LANES         8
#define SJKVARN_TQ6_QK            128
#define SJKVARN_TQ6_BLOCK_BYTES   98
#define SJKVARN_TRELLIS_SEQ       128
#define SJKVARN_TRELLIS_HIST_BITS 6
#define SJKVARN_TRELLIS_NSTATE    64
#define SJKVARN_NO_POS            UINT32_MAX
#define SJKVARN_NO_BLOCK          UINT32_MAX
#define SJKVARN_STATE_HEADER_BYTES 128
#define SJKVARN_ROTATION_HADAMARD 1

typedef enum sj_kvarn_body { SJKVARN_BODY_SCALAR = 0, SJKVARN_BODY_TRELLIS = 1, SJKVARN_BODY_AUTO = 2 } sj_kvarn_body;
typedef enum sj_kvarn_staging { SJKVARN_STAGING_TQ6_0 = 0, SJKVARN_STAGING_F16 = 1 } sj_kvarn_staging;
typedef enum sj_kvarn_sink_type { SJKVARN_SINK_F16 = 0, SJKVARN_SINK_INHERIT = 1 } sj_kvarn_sink_type;

/* 98-byte staging block (sj_kvarn.h:146-154) */
typedef struct sj_kvarn_tq6_block {
    uint16_t norm;
    uint8_t  qs[64];
    uint8_t  qh[32];
} sj_kvarn_tq6_block;

/* record layout (sj_kvarn.h:170-175) */
typedef struct sj_kvarn_layout {
    int D, G, bits_k, bits_v, body;
    uint32_t k_payload, v_payload;
    uint32_t k_scale, k_zero, k_tok, v_ch, v_scale, v_zero;
    uint32_t bytes;
} sj_kvarn_layout;

/* journal policy (sj_kvarn.h:228-234) */
typedef struct sj_kvarn_policy {
    uint32_t sink, tail, tail_max, group, flush_chunk;
    uint32_t B, B_prev, B_pending;
    int      draining;
} sj_kvarn_policy;

/* cache configuration (sj_kvarn.h:279-291) */
typedef struct sj_kvarn_config {
    int      head_dim, n_head_kv, group, bits_k, bits_v, body, iters, staging, sink_type;
    uint32_t sink, tail, tail_max, flush_chunk, n_ubatch, n_ctx;
} sj_kvarn_config;

/* per-layer cache (sj_kvarn.h:293-309); ring, sink and body are device memory here */
typedef struct sj_kvarn_layer {
    sj_kvarn_config cfg;
    sj_kvarn_layout lay;
    uint32_t cap, n_groups;
    size_t   stage_bytes;
    uint8_t * ring;            /* device: [cap][n_head_kv][K row | V row] */
    uint8_t * sink;            /* device: f16 [sink][n_head_kv][K D | V D] fp16, inherit: staging rows */
    uint8_t * body;            /* device: [n_groups][n_head_kv][lay.bytes] (or a pool slab) */
    void    * work;            /* the HIP seal needs no workspace: pool mode keeps the device copy of the
                                  sequence's block table here, NULL otherwise */
    uint16_t * kstage;         /* DEVICE workspace of the layer's attention calls (sjk_hip_workspace_bytes;
                                  the layers of a sequence share their first layer's), not host staging */
    uint16_t * vstage;         /* the library's private runtime of the cache object (a layer of layer_init, or a
                                  sequence, kept with its first layer): its stream, truncation run table and state
                                  transfer buffers; opaque, set by init, freed by free (the device seal reads the
                                  ring directly and needs no host staging) */
    const uint32_t * blocks;   /* host block table (pool mode), NULL = contiguous body */
    int       owns_body;
} sj_kvarn_layer;

/* status codes (sj_kvarn.h:333-359) */
enum {
    SJKVARN_OK = 0,
    SJKVARN_ERR_ARG = -100, SJKVARN_ERR_NOMEM = -101, SJKVARN_ERR_BUFFER = -102, SJKVARN_ERR_TRUNCATED = -103,
    SJKVARN_ERR_MAGIC = -104, SJKVARN_ERR_VERSION = -105, SJKVARN_ERR_FORMAT = -106, SJKVARN_ERR_CORRUPT = -107,
    SJKVARN_ERR_PENDING = -108, SJKVARN_ERR_CAPACITY = -109, SJKVARN_ERR_POOL_FULL = -110,
    SJKVARN_ERR_HEAD_DIM = -120, SJKVARN_ERR_N_HEAD_KV = -121, SJKVARN_ERR_GROUP = -122, SJKVARN_ERR_SINK = -123,
    SJKVARN_ERR_BITS = -124, SJKVARN_ERR_BODY = -125, SJKVARN_ERR_ITERS = -126, SJKVARN_ERR_STAGING = -127,
    SJKVARN_ERR_TAIL = -128, SJKVARN_ERR_ROTATION = -129, SJKVARN_ERR_CODEBOOK = -130, SJKVARN_ERR_N_LAYERS = -131,
    /* this library only: */
    SJK_ERR_DEVICE = -140,      /* a HIP runtime call or kernel launch failed */
    SJK_ERR_UNSUPPORTED = -141  /* shape outside what the kernels are built for (see sjk_hip_supported) */
};

/* ---- pool / sequence / state (sj_kvarn.h:366-442) ---- */
typedef struct sj_kvarn_pool {
    sj_kvarn_config cfg;
    sj_kvarn_layout lay;
    int       n_layers;
    uint32_t  n_blocks;
    uint8_t * body;            /* device: [n_layers][n_blocks][n_head_kv][lay.bytes] */
    uint32_t * free_ids;       /* host */
    uint32_t  n_free;
} sj_kvarn_pool;

typedef struct sj_kvarn_seq {
    sj_kvarn_config  cfg;
    int              n_layers;
    sj_kvarn_layer * layers;
    sj_kvarn_policy  pol;
    uint32_t         n;
    sj_kvarn_pool  * pool;
    uint32_t       * blocks;   /* host block table */
} sj_kvarn_seq;

typedef struct sj_kvarn_state_info {
    uint32_t state_version, format_version;
    sj_kvarn_config cfg;
    uint32_t rotation, rotation_n;
    uint64_t codebook_id;
    int      n_layers;
    uint32_t n, B, B_prev, draining;
    size_t   total_bytes;
} sj_kvarn_state_info;

/* ================================================================================================ */
/* 1. sj_kvarn.h API                                                                                */
/* ================================================================================================ */

/* fp16 conversion, host scalar helpers (sj_kvarn.h:181-182) */
uint16_t sj_kvarn_f32_to_f16(float f);
float    sj_kvarn_f16_to_f32(uint16_t h);

/* rotation (sj_kvarn.h:184-185): runs on the device, for any power-of-two n (the reference's stages read past
 * the end of x for other n; here such a call leaves x as it is) */
void sj_kvarn_hadamard(float * x, int n);
void sj_kvarn_rotate_heads(float * x, int n_heads, int head_dim);

/* record layout (sj_kvarn.h:188-195): host integer logic */
int      sj_kvarn_body_resolve(int body, int bits_k, int bits_v);
int      sj_kvarn_layout_init(sj_kvarn_layout * l, int D, int G, int bits_k, int bits_v, int body);
size_t   sj_kvarn_record_bytes(int D, int G, int bits_k, int bits_v);
double   sj_kvarn_body_bits_per_element(const sj_kvarn_layout * l);
uint32_t sj_kvarn_code_bit(const sj_kvarn_layout * l, int t, int d, int is_v);
int      sj_kvarn_k_ch_idx(const sj_kvarn_layout * l, int d);
int      sj_kvarn_v_ch_idx(const sj_kvarn_layout * l, int d);

/* seal / decode (sj_kvarn.h:199-208): run on the device; rows, rec and out are host arrays.
 * The HIP seal needs no workspace: sj_kvarn_seal_workspace_bytes() returns the reference's figure
 * for ABI compatibility and `work` is ignored. */
size_t sj_kvarn_seal_workspace_bytes(const sj_kvarn_layout * l);
void   sj_kvarn_seal_group(const sj_kvarn_layout * l, const uint16_t * K, const uint16_t * V, size_t row_stride,
                           int iters, uint8_t * rec, void * work);
void   sj_kvarn_decode_k_row(const sj_kvarn_layout * l, const uint8_t * rec, int t, float * out);
void   sj_kvarn_decode_v_row(const sj_kvarn_layout * l, const uint8_t * rec, int t, float * out);

/* staging (sj_kvarn.h:212-216): run on the device */
void   sj_kvarn_tq6_quantize_row(const float * x, sj_kvarn_tq6_block * y, int n);
void   sj_kvarn_tq6_dequantize_row(const sj_kvarn_tq6_block * y, float * x, int n);
size_t sj_kvarn_stage_row_bytes(int staging, int D);
void   sj_kvarn_stage_row(int staging, const float * x_rot, void * dst, int D);
void   sj_kvarn_unstage_row(int staging, const void * src, float * x_rot, int D);

/* attention helpers (sj_kvarn.h:220-222): run on the device */
void sj_kvarn_record_scores(const sj_kvarn_layout * l, const uint8_t * rec, const float * q, int n, float * scores);
void sj_kvarn_record_accum_v(const sj_kvarn_layout * l, const uint8_t * rec, const float * w, int n, float * acc);

/* journal policy, truncation, ring (sj_kvarn.h:236-274): host integer logic */
void     sj_kvarn_policy_init(sj_kvarn_policy * p, uint32_t sink, uint32_t tail, uint32_t tail_max, uint32_t group,
                              uint32_t flush_chunk);
void     sj_kvarn_policy_reset(sj_kvarn_policy * p);
uint32_t sj_kvarn_policy_begin_ubatch(sj_kvarn_policy * p, uint32_t pos0, uint32_t n_tokens);
void     sj_kvarn_policy_commit(sj_kvarn_policy * p);
uint32_t sj_kvarn_policy_idle(sj_kvarn_policy * p, uint32_t end, uint32_t keep_recent);
uint32_t sj_kvarn_group_floor(uint32_t sink, uint32_t group, uint32_t pos);
uint32_t sj_kvarn_policy_trunc_floor(const sj_kvarn_policy * p, uint32_t pos);
uint32_t sj_kvarn_policy_truncate(sj_kvarn_policy * p, uint32_t pos, uint32_t * n_dropped);
uint32_t sj_kvarn_ring_capacity(uint32_t tail, uint32_t tail_max, uint32_t group, uint32_t n_ubatch);
uint32_t sj_kvarn_ring_slot(uint32_t sink, uint32_t cap, uint32_t pos);

/* per-layer cache (sj_kvarn.h:311-330): device-resident buffers, host rows at the API */
sj_kvarn_config sj_kvarn_config_default(int head_dim, int n_head_kv, uint32_t n_ctx, uint32_t n_ubatch);
int       sj_kvarn_layer_init(sj_kvarn_layer * L, const sj_kvarn_config * cfg);
void      sj_kvarn_layer_free(sj_kvarn_layer * L);
void      sj_kvarn_layer_store(sj_kvarn_layer * L, uint32_t pos, const float * k_rot, const float * v_rot);
void      sj_kvarn_layer_seal(sj_kvarn_layer * L, uint32_t B_from, uint32_t B_to);
void      sj_kvarn_layer_kv_row(const sj_kvarn_layer * L, uint32_t B, uint32_t pos, int h, float * k, float * v);
void      sj_kvarn_layer_attend_row(const sj_kvarn_layer * L, uint32_t B, uint32_t N, const float * q_rot, int h,
                                    uint32_t qpos, float scale, float * out_rot);
uint8_t * sj_kvarn_layer_record(const sj_kvarn_layer * L, uint32_t g, int h);   /* DEVICE address */
void      sj_kvarn_layer_truncate(sj_kvarn_layer * L, uint32_t B_old, uint32_t B_new, uint32_t n_old, uint32_t resume);
const char * sj_kvarn_strerror(int code);

/* pool / sequence / state (sj_kvarn.h:378-442) */
int      sj_kvarn_pool_init(sj_kvarn_pool * pool, const sj_kvarn_config * cfg, int n_layers, uint32_t n_blocks);
void     sj_kvarn_pool_free(sj_kvarn_pool * pool);
uint32_t sj_kvarn_pool_alloc(sj_kvarn_pool * pool);
void     sj_kvarn_pool_release(sj_kvarn_pool * pool, uint32_t id);
int      sj_kvarn_seq_init(sj_kvarn_seq * s, const sj_kvarn_config * cfg, int n_layers, sj_kvarn_pool * pool);
void     sj_kvarn_seq_free(sj_kvarn_seq * s);
void     sj_kvarn_seq_reset(sj_kvarn_seq * s);
/* seq_begin_ubatch / seq_idle: a due commit seals [B, B_pending) of every layer in one launch on the sequence's own
 * stream, after the work enqueued on the null stream and on the streams its device stores used
 * (sjk_hip_seq_store, _batch), and waits for that seal only, not for the rest of the device. */
int      sj_kvarn_seq_begin_ubatch(sj_kvarn_seq * s, uint32_t pos0, uint32_t n_tokens);
void     sj_kvarn_seq_store(sj_kvarn_seq * s, uint32_t pos, const float * k_rot, const float * v_rot);
int      sj_kvarn_seq_idle(sj_kvarn_seq * s, uint32_t keep_recent);
uint32_t sj_kvarn_seq_truncate(sj_kvarn_seq * s, uint32_t pos);
void     sj_kvarn_seq_attend_row(const sj_kvarn_seq * s, int il, const float * q_rot, int h, uint32_t qpos, float scale,
                                 float * out_rot);
size_t   sj_kvarn_seq_state_size(const sj_kvarn_seq * s);
size_t   sj_kvarn_state_size_max(const sj_kvarn_config * cfg, int n_layers);
int      sj_kvarn_seq_state_write(const sj_kvarn_seq * s, void * dst, size_t dst_size, size_t * written);
int      sj_kvarn_state_peek(const void * src, size_t size, sj_kvarn_state_info * info);
/* seq_state_read: every check of the reference (sj_kvarn.h:1949-2034) runs, and the transfer buffers are
 * allocated, before the sequence is touched; a rejected stream leaves it unchanged. A device failure during
 * the copy itself returns SJK_ERR_DEVICE with the sequence reset (empty). */
int      sj_kvarn_seq_state_read(sj_kvarn_seq * s, const void * src, size_t size);

/* ================================================================================================ */
/* 2. device entry points (device pointers, stream = hipStream_t or NULL for the null stream)       */
/* ================================================================================================ */

/* Device view of one layer's cache, byte layout of sj_kvarn_layer (sj_kvarn_cuda.cuh:27-42), plus
 * an optional device block table: record (g, h) at body + ((blocks ? blocks[g] : g)*n_head_kv + h)*lay.bytes. */
typedef struct sjk_hip_view {
    sj_kvarn_layout lay;
    int       n_head_kv;
    int       staging;
    int       sink_type;
    uint32_t  S, cap;
    size_t    stage_bytes;
    uint8_t * sink;
    uint8_t * ring;
    uint8_t * body;
    const uint32_t * blocks;
    void    * work;            /* device workspace of the attention calls on this view (their partial results, the plan
                                  of a 4/4 sjk_hip_attend_dyn call, the staging of the host-array layer calls):
                                  sjk_hip_workspace_bytes() bytes. sjk_layer_view
                                  fills it with the layer's own; a hand-built view brings one. Calls that
                                  share a workspace must be ordered (one stream, or the caller's
                                  synchronisation), as for the cache itself. */
    size_t    work_bytes;
} sjk_hip_view;

/* 1 when the kernels are built for this layout (D in {128, 256}, G = 128), else 0 */
int sjk_hip_supported(const sj_kvarn_layout * l);

/* Bytes of device workspace that attention calls on a view with this layout and KV head count need
 * (sjk_hip_view.work); sized on the current device. No counterpart in the reference (whose attention keeps its
 * state in registers of one thread per row and head, sj_kvarn_cuda.cuh:102-135). */
size_t sjk_hip_workspace_bytes(const sj_kvarn_layout * l, int n_head_kv);

/* Seal n_groups*n_head_kv records from fp16 rows: record r = g*n_head_kv + h reads the G rows
 * k + g*G*row_stride + h*D (+ t*row_stride) and writes body + r*l->bytes.
 * Replaces sj_kvarn_cuda_seal (sj_kvarn_cuda.cuh:142-151); needs no workspace. */
int sjk_hip_seal(const sj_kvarn_layout * l, const uint16_t * d_k, const uint16_t * d_v, size_t row_stride,
                 int n_head_kv, int n_groups, int iters, uint8_t * d_body, void * stream);

/* Decode n_rec records to fp32 rows out_k/out_v [n_rec][G][D] (sj_kvarn_cuda.cuh:57-66). */
int sjk_hip_decode(const sj_kvarn_layout * l, const uint8_t * d_body, int n_rec, float * d_out_k, float * d_out_v,
                   void * stream);

/* Stage / unstage n_rows rows of D values (sj_kvarn_cuda.cuh:68-80). */
int sjk_hip_stage(int staging, const float * d_x, uint8_t * d_dst, int D, size_t dst_row_bytes, int n_rows, void * stream);
int sjk_hip_unstage(int staging, const uint8_t * d_src, size_t src_row_bytes, float * d_x, int D, int n_rows,
                    void * stream);

/* In-place orthonormal Hadamard of n_rows rows of D floats, D any power of two (sj_kvarn_rotate_heads,
 * sj_kvarn.h:754-759); SJKVARN_ERR_ARG for other D. */
int sjk_hip_rotate(float * d_x, int n_rows, int D, void * stream);

/* The rotation folded into the projection weights at load time (the reference's INTEGRATION_LLAMACPP.md:46: "the
 * rotation can also be folded into the Q/K/V/O weights at load time"; the fork's fused Q / output rotation,
 * README.md:45-54), so that a decode step needs no sj_kvarn_rotate_heads on q, k, v and none on the attention
 * output. R = the Hadamard of sj_kvarn_hadamard (H / sqrt(D), symmetric, its own inverse); device memory, fp32,
 * row-major, in place, any power-of-two D.
 * sjk_hip_fold_rotation_out: W is [n_heads * head_dim][cols] (W_q, W_k or W_v; a bias with cols = 1): every column's
 *   head_dim-blocks become R times them, W' = blockdiag(R) W, so W' x is the rotated projection, value for value the
 *   reference's sj_kvarn_rotate_heads(W x) up to the rounding of the product (then store with rotate = 0).
 * sjk_hip_fold_rotation_in: W is [rows][n_heads * head_dim] (W_o): every row's head segments become R times them,
 *   W' = W blockdiag(R), so W' takes the attention's rotated output directly.
 * Each folded vector is bit for bit sj_kvarn_hadamard of the original. No counterpart function in the reference,
 * which describes the folding without shipping it. */
int sjk_hip_fold_rotation_out(float * d_w, int n_heads, int head_dim, int cols, void * stream);
int sjk_hip_fold_rotation_in(float * d_w, int rows, int n_heads, int head_dim, void * stream);

/* Append n_pos positions pos0.. to a layer (sj_kvarn_layer_store, sj_kvarn.h:1475-1492, batched):
 * d_k, d_v are [n_pos][n_head_kv][D] floats. rotate != 0 applies the Hadamard first (the engine's
 * sj_kvarn_rotate_heads fused into the append); rotate == 0 expects rotated rows. */
int sjk_hip_layer_store(const sjk_hip_view * v, uint32_t pos0, uint32_t n_pos, const float * d_k, const float * d_v,
                        int rotate, void * stream);

/* sjk_hip_layer_store with pos0 = d_desc[SJK_DESC_QPOS0] read on the device when the kernel runs, so a captured
 * HIP graph stores every decode step's rows (the reference's staged write ggml_set_rows_stage,
 * INTEGRATION_LLAMACPP.md:47, whose row indices are a graph input). A negative entry stores nothing. */
int sjk_hip_layer_store_dyn(const sjk_hip_view * v, const int32_t * d_desc, uint32_t n_pos, const float * d_k,
                            const float * d_v, int rotate, void * stream);

/* Commit: seal groups [B_from, B_to) of every KV head of n_layers layers straight out of their
 * staging rings in one launch (sj_kvarn_layer_seal, sj_kvarn.h:1494-1514, for each layer). */
int sjk_hip_commit(const sjk_hip_view * views, int n_layers, uint32_t B_from, uint32_t B_to, int iters, void * stream);

/* Run-time descriptor of a commit: 16 int32 in device memory, at the indices of the reference's seal_dyn
 * descriptor (INTEGRATION_LLAMACPP.md:51-71). sjk_hip_commit_dyn reads SJK_DESC_B_OLD and SJK_DESC_B. */
enum {
    SJK_DESC_S = 0, SJK_DESC_CAP = 1, SJK_DESC_B = 2, SJK_DESC_N = 3, SJK_DESC_QPOS0 = 4, SJK_DESC_G = 5,
    SJK_DESC_D = 6, SJK_DESC_RECBYTES = 7, SJK_DESC_HKV = 8, SJK_DESC_B_OLD = 9, SJK_DESC_TYPE_K = 10,
    SJK_DESC_TYPE_V = 11, SJK_DESC_BODY_TYPE = 12, SJK_DESC_SINK_TYPE = 13, SJK_DESC_N_ENTRIES = 16
};

/* The commit of sjk_hip_commit with its range [d_desc[SJK_DESC_B_OLD], d_desc[SJK_DESC_B]) read on the device
 * when the kernel runs, launched for n_groups_max groups per layer: the launch does not depend on the range,
 * so a captured HIP graph replays every commit (the reference's ggml_sjkvarn_seal_dyn,
 * INTEGRATION_LLAMACPP.md:48). Groups past the range exit at once. Refused, sealing nothing: a negative
 * entry, an empty or misaligned range, and a range of more than n_groups_max groups (sealing a part would
 * leave records that attention reads unsealed). The range must lie in the views' groups, as for
 * sjk_hip_commit. */
int sjk_hip_commit_dyn(const sjk_hip_view * views, int n_layers, const int32_t * d_desc, int n_groups_max, int iters,
                       void * stream);

/* Causal attention for n_q query rows at positions qpos0.. over [0, min(N, qpos+1)) with sealed end B
 * (sj_kvarn_cuda.cuh:102-135). d_q, d_out: [n_q][n_head][D] fp32, rotated basis; GQA maps query head
 * hq to KV head hq / (n_head / n_head_kv). Any n_q and n_head (a prefill ubatch as well as a decode step):
 * the n_q x n_head / n_head_kv query rows of a KV head are cut into tiles of 16 rows, and a launch takes up to
 * 8 jobs side by side (sharing its workgroups in proportion to their work; each job reads the context); a 4/4
 * call of more than 256 rows (or of 256 and 8 KV heads) whose output does not lie over its queries runs in one launch
 * of 32-row tiles. The
 * partial results go to v->work (SJKVARN_ERR_ARG without one). Every layout a layer can have runs
 * on a matrix-core kernel; a hand-built view outside them (another group size, head dimension or record
 * layout) is refused with SJK_ERR_UNSUPPORTED and a message (sjk_last_error), as are the batched, no-alloc and
 * descriptor forms below. */
int sjk_hip_attend(const sjk_hip_view * v, uint32_t B, uint32_t N, uint32_t qpos0, int n_q, int n_head,
                   const float * d_q, float scale, float * d_out, void * stream);

/* sjk_hip_attend for callers that cannot allocate device memory (code under stream capture, serving loops
 * that forbid hipMalloc): the same kernels and results, with v->work ignored and the partial results in a
 * static device array of 16 MiB per device, held until the process ends. Views whose workspace would be larger
 * (sjk_hip_workspace_bytes > 16 MiB) are refused with SJKVARN_ERR_CAPACITY (sjk_last_error says why). All
 * calls on one device share the array: calls that overlap on a device (two streams, two threads) race. No
 * counterpart in the reference; it is for callers that cannot allocate. */
int sjk_hip_attend_noalloc(const sjk_hip_view * v, uint32_t B, uint32_t N, uint32_t qpos0, int n_q, int n_head,
                           const float * d_q, float scale, float * d_out, void * stream);

/* sjk_hip_attend with B, N and qpos0 read from the device descriptor d_desc (SJK_DESC_B, SJK_DESC_N,
 * SJK_DESC_QPOS0) when the kernels run, on a launch shape that does not depend on them, so a captured HIP
 * graph replays every decode step (the reference's region-aware flash_attn_ext,
 * ggml_flash_attn_ext_set_sjkvarn, INTEGRATION_LLAMACPP.md:49; n_max plays its n_kv_pad: the positions the
 * view's buffers hold). Every layout sjk_hip_attend takes (D = 128 or 256; every scalar body and the 3/3, 3/2,
 * 2/2 trellis bodies). Results equal sjk_hip_attend's bit for bit. A descriptor
 * the view cannot hold (a negative entry, B misaligned or past N, N past n_max, a tail longer than the ring)
 * writes NaN rows. The call is planned on the device from the descriptor: a 16-row call of the trellis and other
 * scalar bodies in its workgroups, a 4/4 call and any call of more than 16 rows per KV head by a one-workgroup
 * plan kernel that writes the launch's job table into v->work. The table and the partial results live in v->work,
 * which the layer allocated when it was created, so a capture sees no allocation. Any number of query rows per
 * KV head (n_q x n_head / n_head_kv): as in sjk_hip_attend, 16-row tiles, up to 8 a launch, shared out by the
 * same arithmetic, a launch and its combine per 8 tiles, or the 32-row tiles of a large 4/4 call, with no plan
 * kernel; in stream order, all on the one stream a capture records. */
int sjk_hip_attend_dyn(const sjk_hip_view * v, const int32_t * d_desc, uint32_t n_max, int n_q, int n_head,
                       const float * d_q, float scale, float * d_out, void * stream);

/* Batched attention: n_jobs independent calls (each a layer view with its B, N, qpos0, d_q, d_out as in
 * sjk_hip_attend) that share n_q, n_head and scale, e.g. one layer of every sequence of a decode
 * batch. Jobs of one record layout, KV head count and staging type run in one launch (8 per launch);
 * others run one call each. No counterpart in the reference (whose attention is one row and head per
 * call, sj_kvarn.h:1535-1564); each job's result equals its sjk_hip_attend result. */
typedef struct sjk_hip_attend_job {
    sjk_hip_view  v;
    uint32_t      B, N, qpos0;
    const float * d_q;
    float       * d_out;
} sjk_hip_attend_job;
int sjk_hip_attend_batch(const sjk_hip_attend_job * jobs, int n_jobs, int n_q, int n_head, float scale, void * stream);

/* Batched append: n_jobs independent sjk_hip_layer_store calls of n_pos positions each (job = view,
 * pos0, d_k, d_v) in one launch (16 per launch). No counterpart in the reference. */
typedef struct sjk_hip_store_job {
    sjk_hip_view  v;
    uint32_t      pos0;
    const float * d_k;
    const float * d_v;
} sjk_hip_store_job;
int sjk_hip_store_batch(const sjk_hip_store_job * jobs, int n_jobs, uint32_t n_pos, int rotate, void * stream);

/* ---- rows between a layer's projections and its cache (no counterpart in the reference, whose API takes rows that are
 * normed, turned and rotated already, sj_kvarn.h:1475-1492) ---- */

/* element types of the rows an engine hands over */
enum { SJK_F32 = 0, SJK_F16 = 1, SJK_BF16 = 2 };

/* Frequencies of rotary positions: pair i of the n_rot / 2 turned pairs of channels has f_i = base^(-2 i / n_rot) radians
 * per position, divided by divisors[i] where that list is given, then scaled for contexts longer than the trained one:
 *   SJK_ROPE_PLAIN   as it is
 *   SJK_ROPE_LINEAR  f_i / factor
 *   SJK_ROPE_NTK     base * factor^(n_rot / (n_rot - 2)) in place of base (n_rot = 2: f_0 / factor)
 *   SJK_ROPE_RAMP    between f_i / factor and f_i along i: f_i up to the pair that turns `high` times in n_orig positions,
 *                    f_i / factor from the pair that turns `low` times on (pair indices floor and ceil of
 *                    n_rot ln(n_orig / (2 pi turns)) / (2 ln base), cut to 0 and n_rot - 1); magnitude 0.1 ln(factor) + 1
 *   SJK_ROPE_BANDS   between them by turns r = n_orig f_i / 2 pi: f_i from r = high on, f_i / factor up to r = low */
enum { SJK_ROPE_PLAIN = 0, SJK_ROPE_LINEAR = 1, SJK_ROPE_NTK = 2, SJK_ROPE_RAMP = 3, SJK_ROPE_BANDS = 4 };
typedef struct sjk_rope_config {
    int            n_rot;       /* turned channels of a head, even */
    int            scaling;     /* SJK_ROPE_* */
    double         base;        /* > 1 */
    double         factor;      /* > 0; for RAMP >= 1 */
    double         n_orig;      /* RAMP, BANDS: the trained context, > 0 */
    double         low, high;   /* RAMP, BANDS: turns in n_orig positions, 0 < low < high */
    const double * divisors;    /* NULL, or n_rot / 2 values > 0 (host) */
} sjk_rope_config;

/* The table that the calls below read: turns[i] = f_i / 2 pi, n_rot / 2 doubles (host; a program copies it to the device
 * once), and *mscale, the factor that the scaling puts on sines and cosines (1 but for RAMP). Host arithmetic, no GPU call.
 * SJKVARN_ERR_ARG, writing nothing, for values outside the ranges above. */
int sjk_rope_turns(const sjk_rope_config * c, double * turns, float * mscale);

/* A turn of rotary positions. Channels behind n_rot pass through. With a pair (a, b) at position p, u = p turns[i]:
 * (a, b) -> mscale (a cos 2 pi u - b sin 2 pi u, a sin 2 pi u + b cos 2 pi u); the angle is reduced in 64 bits, so far
 * positions lose nothing. inverse: the sine's sign turned, which is the turn's gradient (for mscale = 1 also the way back). */
enum { SJK_ROPE_HALVES = 0 /* pairs (i, i + n_rot / 2) */, SJK_ROPE_PAIRS = 1 /* pairs (2 i, 2 i + 1) */ };
typedef struct sjk_hip_rope {
    int            layout;      /* SJK_ROPE_HALVES or SJK_ROPE_PAIRS */
    int            n_rot;       /* even, 0 (no turn) to the head's width */
    int            inverse;
    float          mscale;
    const double * d_turns;     /* device, n_rot / 2 */
} sjk_hip_rope;

/* One set of heads of sjk_hip_head_rows: rows x[pos][head][D] of x_type at d_x + pos * x_pos + head * x_head (strides in
 * elements, any; the channels of a head adjacent) to rows of out_type at d_out. In order, each where asked for: the norm
 * x / sqrt(mean(x^2) + eps) * w (d_norm: fp32 weights [D] of head h at d_norm + h * norm_head, 0 = shared), the turn
 * (rope != 0), the orthonormal Hadamard (rotate != 0; D = 64, 128, 256 or 512), one rounding to out_type. */
typedef struct sjk_hip_head_job {
    const void  * d_x;
    void        * d_out;        /* may be d_x, with the same type and strides; no other overlap */
    int64_t       x_pos, x_head, out_pos, out_head;
    int           x_type, out_type, n_heads, rope, rotate;
    float         eps;          /* where d_norm is given: normal, finite, > 0 */
    const float * d_norm;       /* NULL: no norm */
    int64_t       norm_head;
} sjk_hip_head_job;

/* n_pos positions of every job's heads (the queries and the keys of a layer, say) in one launch for up to three jobs of one
 * x_type (several where a call has more rows than a launch takes, 2^29 of up to 64 channels and one head). Head widths 1 to 512,
 * fewer than 2^31 rows in all jobs. Position i is d_pos[i] (device, int32) or, with d_pos NULL, pos0 + i, below 2^32 - 1. rope may
 * be NULL if no job turns. Sums, angles and products in 32 bits or more. */
int sjk_hip_head_rows(const sjk_hip_head_job * jobs, int n_jobs, uint32_t n_pos, int D, const sjk_hip_rope * rope,
                      uint32_t pos0, const int32_t * d_pos, void * stream);

/* What a layer's projection rows are, the same for each of its calls: q [n_pos][n_head][D], k and v [n_pos][n_head_kv][D]
 * of one type with strides in elements (views of one fused output, or three tensors). */
typedef struct sjk_hip_qkv {
    int           type;         /* SJK_F32, _F16, _BF16 */
    int           n_head;       /* query heads; 0: no queries, keys and values only */
    int           rotate_qk;    /* the Hadamard on queries and keys: 1 unless the caller has rotated them */
    int           rotate_v;     /* the Hadamard on values: 0 where it is folded into W_v (a turn or a norm lies between W_q,
                                   W_k and the cache, so there it cannot be folded) */
    float         eps;
    int64_t       q_pos, q_head, k_pos, k_head, v_pos, v_head;
    const float * d_q_norm;     /* NULL or fp32 weights, as sjk_hip_head_job.d_norm */
    const float * d_k_norm;
    int64_t       norm_head;
    sjk_hip_rope  rope;         /* n_rot = 0: no turn */
} sjk_hip_qkv;

/* Queries, keys and values of positions pos0 .. pos0 + n_pos - 1 from a layer's projections in one launch: queries normed,
 * turned and rotated to d_q_out [n_pos][n_head][D] fp32, as sjk_hip_attend takes them; keys the same, values rotated,
 * both staged into the view's sink and ring at the positions' slots. The bytes are those of sjk_hip_head_rows to fp32
 * followed by sjk_hip_layer_store. d_pos (device, int32): positions of the turn other than pos0 + i; the slots stay those of
 * pos0 + i. d_q_out may be d_q (fp32 rows [n_pos][n_head][D]); no other overlap. n_pos beyond what sink and ring hold at
 * once is SJKVARN_ERR_CAPACITY (positions would share a slot). D = 128 or 256, as layers have. */
int sjk_hip_store_qkv(const sjk_hip_view * v, uint32_t pos0, uint32_t n_pos, const sjk_hip_qkv * m, const int32_t * d_pos,
                      const void * d_q, const void * d_k, const void * d_v, float * d_q_out, void * stream);

/* The same with pos0 = d_desc[SJK_DESC_QPOS0] read on the device when the kernel runs (sjk_hip_layer_store_dyn): one
 * captured graph takes every step. A negative entry writes nothing, d_q_out included. SJKVARN_ERR_ARG for more rows than one launch
 * holds (2^27 positions of one KV head of 128). */
int sjk_hip_store_qkv_dyn(const sjk_hip_view * v, const int32_t * d_desc, uint32_t n_pos, const sjk_hip_qkv * m,
                          const int32_t * d_pos, const void * d_q, const void * d_k, const void * d_v, float * d_q_out,
                          void * stream);

/* n_jobs independent sjk_hip_store_qkv calls of n_pos positions each, 32 a launch where the views agree in KV heads, staging
 * and sink type. Two jobs on one ring are refused (SJKVARN_ERR_ARG). */
typedef struct sjk_hip_qkv_job {
    sjk_hip_view    v;
    uint32_t        pos0;
    const int32_t * d_pos;
    const void    * d_q;
    const void    * d_k;
    const void    * d_v;
    float         * d_q_out;
} sjk_hip_qkv_job;
int sjk_hip_store_qkv_batch(const sjk_hip_qkv_job * jobs, int n_jobs, uint32_t n_pos, const sjk_hip_qkv * m, void * stream);

/* The same for layer il of several sequences (a decode batch), as sjk_hip_seq_store_batch: each sequence's position count
 * is extended. SJKVARN_ERR_ARG for a bad layer index, a gap before pos0 or a sequence given twice; SJKVARN_ERR_CAPACITY where the
 * staged positions (from the sealed end on) would not fit the ring, and for positions of the sealed part whose ring slots hold
 * staged ones. A refused call stores nothing. */
typedef struct sjk_hip_seq_qkv_job {
    sj_kvarn_seq  * seq;
    uint32_t        pos0;
    const int32_t * d_pos;
    const void    * d_q;
    const void    * d_k;
    const void    * d_v;
    float         * d_q_out;
} sjk_hip_seq_qkv_job;
int sjk_hip_seq_store_qkv_batch(const sjk_hip_seq_qkv_job * jobs, int n_jobs, int il, uint32_t n_pos, const sjk_hip_qkv * m,
                                void * stream);

/* K and V rows (fp32, rotated) of positions pos0 .. pos0+n_pos-1 of KV head h with sealed end B:
 * d_k, d_v [n_pos][D] (the region resolver of sj_kvarn_layer_kv_row, sj_kvarn.h:1516-1533, and of
 * sj_kvarn_cuda_kv_row, sj_kvarn_cuda.cuh:82-100) */
int sjk_hip_kv_rows(const sjk_hip_view * v, uint32_t B, uint32_t pos0, uint32_t n_pos, int h, float * d_k, float * d_v,
                    void * stream);

/* scores[t] = dot(q, K[t]) and acc[d] += sum_t w[t] V[t,d] for the first n tokens of one device record,
 * sequential fp32 sums as in the reference (sj_kvarn.h:1288-1311) */
int sjk_hip_record_scores(const sj_kvarn_layout * l, const uint8_t * d_rec, const float * d_q, int n, float * d_scores,
                          void * stream);
int sjk_hip_record_accum_v(const sj_kvarn_layout * l, const uint8_t * d_rec, const float * d_w, int n, float * d_acc,
                           void * stream);

/* Device twins of sj_kvarn_seq_store (sj_kvarn.h:407, 1779-1792) and sj_kvarn_seq_attend_row
 * (sj_kvarn.h:414, 1806-1809), one layer il per call: sjk_hip_seq_store appends n_pos positions
 * pos0.. (pos0 <= the sequence's position count) to layer il as sjk_hip_layer_store does and extends
 * the position count; sjk_hip_seq_attend is sjk_hip_attend over layer il with the sequence's sealed
 * end and position count. SJKVARN_ERR_ARG for a bad layer index or a gap before pos0. */
int sjk_hip_seq_store(sj_kvarn_seq * s, int il, uint32_t pos0, uint32_t n_pos, const float * d_k, const float * d_v,
                      int rotate, void * stream);
int sjk_hip_seq_attend(const sj_kvarn_seq * s, int il, uint32_t qpos0, int n_q, int n_head, const float * d_q,
                       float scale, float * d_out, void * stream);

/* The same for layer il of several sequences in one launch each (a decode batch): job k appends n_pos
 * positions from pos0 to seq (sjk_hip_seq_store_batch, d_k / d_v) or runs the n_q query rows at
 * positions pos0.. over it (sjk_hip_seq_attend_batch, d_q / d_out; pos0 + n_q <= the position count). */
typedef struct sjk_hip_seq_job {
    sj_kvarn_seq * seq;
    uint32_t       pos0;
    const float  * d_k;
    const float  * d_v;
    const float  * d_q;
    float        * d_out;
} sjk_hip_seq_job;
int sjk_hip_seq_store_batch(const sjk_hip_seq_job * jobs, int n_jobs, int il, uint32_t n_pos, int rotate, void * stream);

/* Stream-ordered twins of sj_kvarn_seq_begin_ubatch and sj_kvarn_seq_idle (sj_kvarn.h:408-410, 1760-1777): the
 * same policy step and commit, with the seal of [B, B_pending) (every layer, one launch per 64 layers) and the
 * copy of the new block-table entries enqueued on `stream` after what the caller enqueued there before (its
 * stores of earlier positions), and no wait: work the caller enqueues on `stream` afterwards sees the new records.
 * The reference's seal reads only positions below pos0 and may run on a side stream (README.md:351-352): an engine
 * that stores on another stream orders the two itself. A failed launch returns its status with the policy as it
 * was. No counterpart in the reference's C API. */
int sjk_hip_seq_begin_ubatch(sj_kvarn_seq * s, uint32_t pos0, uint32_t n_tokens, void * stream);
int sjk_hip_seq_idle(sj_kvarn_seq * s, uint32_t keep_recent, void * stream);

/* Asynchronous state save and restore (README.md:609 plans "device-to-host copies overlapped with decoding"; no
 * counterpart in the reference's C API). The stream bytes are those of sj_kvarn_seq_state_write / _read.
 *   _write_begin: the checks and header of sj_kvarn_seq_state_write; the sequence's device pieces (sink, records,
 *     ring rows of every layer) are gathered into a device snapshot by one launch before it returns, so the caller
 *     may store into, commit and attend the sequence right away; a host thread then copies the snapshot to dst
 *     (pinned chunks on a stream of the sequence's own) and appends the checksum. dst stays valid until _finish.
 *   _read_begin: the header checks of sj_kvarn_seq_state_read (all but the checksum); a host thread checks the
 *     checksum and uploads the payload into the device snapshot. The sequence is left as it was; the caller does
 *     not use it until _finish, which checks the pool again, resets the sequence and scatters the snapshot into
 *     it with one launch (a rejected stream leaves the sequence unchanged; a device failure in the scatter leaves
 *     it reset, as sj_kvarn_seq_state_read).
 *   _poll: 1 when no transfer is in flight or it has ended, 0 while it runs (never blocks).
 *   _finish: waits for the transfer and returns its status (*written: the stream bytes of a save).
 * One transfer per sequence at a time: state calls on a sequence with one in flight return SJKVARN_ERR_PENDING;
 * sj_kvarn_seq_free waits for it. The snapshot (one stream payload of device memory) is kept with the sequence. */
int sjk_hip_seq_state_write_begin(const sj_kvarn_seq * s, void * dst, size_t dst_size);
int sjk_hip_seq_state_read_begin(sj_kvarn_seq * s, const void * src, size_t size);
int sjk_hip_seq_state_poll(const sj_kvarn_seq * s);
int sjk_hip_seq_state_finish(sj_kvarn_seq * s, size_t * written);
int sjk_hip_seq_attend_batch(const sjk_hip_seq_job * jobs, int n_jobs, int il, int n_q, int n_head, float scale,
                             void * stream);

/* ---- part of a long context, and drafted tokens (no counterpart in the reference, whose attention reads the whole context and
 * whose positions follow each other) ---- */

/* Attention over some of the sealed groups. For every query position and KV head, sjk_hip_select_groups lists the `top` groups
 * whose keys can reach the highest scores, and sjk_hip_attend_groups attends over the sink, the listed groups and the
 * staged tail (positions from B on, causal among themselves).
 *
 * A group's score comes from its record's scale tables alone. With codes in [c0, c1] (0 and 2^bits - 1, or the K codebook's
 * least and greatest value) a key is K[t, d] = (c Kscale[d] + Kzero[d]) Ktok[t], so with
 *   u = sum_d q_d Kzero_d + w_d Kscale_d,   w_d = c1 q_d for q_d > 0, else c0 q_d,
 * no token's product with q is above u max Ktok (u >= 0) or u min Ktok (u < 0). The score is the largest such bound of the KV head's
 * query heads, in 64 bits (for scores that are multiplied by a scale above zero). The greatest scores are taken, of equal ones the lower
 * group; a score that is not a number is above all others. d_sel [n_q][n_head_kv][top] (int32) is in ascending order, -1 where there are fewer
 * groups than top.
 *
 * sjk_hip_attend_groups takes any ascending list, longer than the groups are many or not: an entry that is no sealed group, or not above the
 * entry before it, adds nothing, wherever it stands.
 * With all groups listed the result is sjk_hip_attend's up to rounding. d_out [n_q][n_head][D] of out_type (SJK_F32, _F16, _BF16), rotated
 * basis. Sums and statistics have 32 bits; weights keep 22 bits, those of SJK_BF16 outputs on scalar records are rounded to
 * fp16 once. A row that sees nothing is zero. Infinities and NaNs of staged positions that a row does not see do not reach it.
 *
 * Query positions lie behind the sealed part: with B > S, qpos0 + 1 >= B, N >= B, and B at a group's end (SJKVARN_ERR_ARG otherwise).
 * d_q is fp32 [n_q][n_head][D], 16-byte aligned, and does not overlap d_out. Both use v->work as sjk_hip_attend does. A selection's
 * scores lie there too: SJKVARN_ERR_CAPACITY where one position's (8 bytes a group and KV head) do not fit. More
 * staged positions than the ring holds are SJKVARN_ERR_CAPACITY. Views outside the attention kernels: SJK_ERR_UNSUPPORTED. */
int sjk_hip_select_groups(const sjk_hip_view * v, uint32_t B, uint32_t N, uint32_t qpos0, int n_q, int n_head, const float * d_q,
                          int top, int32_t * d_sel, void * stream);
int sjk_hip_attend_groups(const sjk_hip_view * v, uint32_t B, uint32_t N, uint32_t qpos0, int n_q, int n_head, const float * d_q,
                          float scale, const int32_t * d_sel, int top, int out_type, void * d_out, void * stream);

/* The same with B, N and qpos0 from the device descriptor (SJK_DESC_B, _N, _QPOS0) when the kernels run, on a launch that does not
 * depend on them: one captured graph takes every step. n_max bounds N. A descriptor that the view cannot hold, or whose
 * positions do not lie behind the sealed part, gives lists of -1 and NaN rows. */
int sjk_hip_select_groups_dyn(const sjk_hip_view * v, const int32_t * d_desc, uint32_t n_max, int n_q, int n_head, const float * d_q,
                              int top, int32_t * d_sel, void * stream);
int sjk_hip_attend_groups_dyn(const sjk_hip_view * v, const int32_t * d_desc, uint32_t n_max, int n_q, int n_head, const float * d_q,
                              float scale, const int32_t * d_sel, int top, int out_type, void * d_out, void * stream);

/* n_jobs independent calls with one n_q, n_head and top in as few launches as the kernels take: up to 16 jobs a selection, as many as
 * have room for their scores in the workspaces that they share (one that does not fit alone: SJKVARN_ERR_CAPACITY, nothing is
 * launched); up to 13 tiles of 16 query rows an attention, where a list's tile is one position. Views of a selection agree in layout
 * and KV heads. d_out is not used by a selection. */
typedef struct sjk_hip_groups_job {
    sjk_hip_view  v;
    uint32_t      B, N, qpos0;
    const float * d_q;
    int32_t     * d_sel;
    void        * d_out;
} sjk_hip_groups_job;
int sjk_hip_select_groups_batch(const sjk_hip_groups_job * jobs, int n_jobs, int n_q, int n_head, int top, void * stream);
int sjk_hip_attend_groups_batch(const sjk_hip_groups_job * jobs, int n_jobs, int n_q, int n_head, float scale, int top, int out_type,
                                void * stream);

/* The same for layer il of several sequences: positions pos0 .. pos0 + n_q - 1 of seq, which are stored (pos0 + n_q <= its count). */
typedef struct sjk_hip_seq_groups_job {
    sj_kvarn_seq * seq;
    uint32_t       pos0;
    const float  * d_q;
    int32_t      * d_sel;
    void         * d_out;
} sjk_hip_seq_groups_job;
int sjk_hip_seq_select_groups_batch(const sjk_hip_seq_groups_job * jobs, int n_jobs, int il, int n_q, int n_head, int top, void * stream);
int sjk_hip_seq_attend_groups_batch(const sjk_hip_seq_groups_job * jobs, int n_jobs, int il, int n_q, int n_head, float scale, int top,
                                    int out_type, void * stream);

/* Attention of drafted nodes. A tree (or any set) of n_nodes drafted tokens is stored behind the context like positions base ..
 * base + n_nodes - 1 (sjk_hip_store_qkv, whose d_pos turns each node by its depth). Query row i sees positions [0, base) and those nodes j
 * whose bit is set in d_seen: bit j % 64 of word i * ceil(n_nodes / 64) + j / 64 (uint64, device), its ancestors and itself say;
 * bits past the nodes are ignored. Rows and nodes need not be the same tokens: n_q rows may be the last level of a tree, and a row may see
 * no node. Sealed groups are read whole; base is not below the sealed end (B > S: base >= B, SJKVARN_ERR_ARG otherwise). Everything else is as for
 * sjk_hip_attend_groups; the values of a node reach no row that does not see it, whatever they are. */
int sjk_hip_attend_tree(const sjk_hip_view * v, uint32_t B, uint32_t base, int n_nodes, int n_q, int n_head, const float * d_q, float scale,
                        const uint64_t * d_seen, int out_type, void * d_out, void * stream);

/* The same with B and base = d_desc[SJK_DESC_QPOS0] read on the device (SJK_DESC_N is not read); n_max bounds base + n_nodes. */
int sjk_hip_attend_tree_dyn(const sjk_hip_view * v, const int32_t * d_desc, uint32_t n_max, int n_nodes, int n_q, int n_head,
                            const float * d_q, float scale, const uint64_t * d_seen, int out_type, void * d_out, void * stream);

typedef struct sjk_hip_tree_job {
    sjk_hip_view     v;
    uint32_t         B, base;
    const uint64_t * d_seen;
    const float    * d_q;
    void           * d_out;
} sjk_hip_tree_job;
int sjk_hip_attend_tree_batch(const sjk_hip_tree_job * jobs, int n_jobs, int n_nodes, int n_q, int n_head, float scale, int out_type,
                              void * stream);

/* The same for layer il of several sequences whose nodes are stored (base + n_nodes <= the position count). */
typedef struct sjk_hip_seq_tree_job {
    sj_kvarn_seq   * seq;
    uint32_t         base;
    const uint64_t * d_seen;
    const float    * d_q;
    void           * d_out;
} sjk_hip_seq_tree_job;
int sjk_hip_seq_attend_tree_batch(const sjk_hip_seq_tree_job * jobs, int n_jobs, int il, int n_nodes, int n_q, int n_head, float scale,
                                  int out_type, void * stream);

/* The accepted path becomes the context: in every one of n_layers layers the stored row of node d_path[i] (device, int32) moves to position
 * base + i, in place, one launch for up to 160 layers. The path ascends; it ends at n_path entries or at the first that is no node
 * above the entry before it (-1, say), so a launch need not know its length. Rows of the positions behind it stay as they are. The views agree
 * in heads, staging, sink and capacity. A row that moves from a ring of 6-bit rows into an fp16 sink becomes the fp16 values of what
 * the ring holds. SJKVARN_ERR_CAPACITY for more staged nodes than the ring has slots. _dyn: base = d_desc[SJK_DESC_QPOS0], a negative
 * one moves nothing. */
int sjk_hip_accept(const sjk_hip_view * views, int n_layers, uint32_t base, int n_nodes, const int32_t * d_path, int n_path, void * stream);
int sjk_hip_accept_dyn(const sjk_hip_view * views, int n_layers, const int32_t * d_desc, int n_nodes, const int32_t * d_path, int n_path,
                       void * stream);

/* The same for a sequence whose last positions, from base on, are drafted nodes: path is a host array, and the position count becomes
 * base + n_path (n_path 0: all nodes are dropped). Enqueued on `stream` with no host wait; nothing is cleared. SJKVARN_ERR_ARG for a path
 * that does not ascend or leaves the nodes, and for base past the count or below the sealed end; SJKVARN_ERR_PENDING while a
 * state restore of the sequence is in flight. A refused call changes nothing. */
int sjk_hip_seq_accept(sj_kvarn_seq * s, uint32_t base, const int32_t * path, int n_path, void * stream);

/* ---- pages: from one sequence to another, and from place to place in a pool (no counterpart in the reference, whose
 * sequences own their blocks alone) ----
 *
 * A sealed record never changes, so sequences of one pool can hold the same block: a pool of sj_kvarn_pool_init counts the
 * holders of its blocks. sj_kvarn_pool_release takes one holder off and frees the block with the last one; seq_truncate,
 * seq_reset, seq_free and a state restore release the blocks they drop in that way and clear only those that no one else holds
 * (sj_kvarn_layer_truncate on a pool sequence's layer knows no holders and clears every dropped record: use seq_truncate).
 * The blocks of a pool that its caller put together have one holder each: forks on it copy the records.
 * These calls change the pool on the host: the caller orders them with each other and with commits on that pool. */

/* The sink entries [0, min(N, S)) and the staged rows of positions [B, N) of n_layers layers copied from src's buffers to dst's
 * slots of the same positions, in one launch for up to 64 layers; nothing else in dst is written. Records are not copied: dst's
 * view brings its own body or block table. The views agree in layout, KV heads, staging, sink type and S (capacities may
 * differ), buffers 4-byte aligned, and no buffer of dst (S sink entries, cap ring slots) overlaps another of dst or one of src.
 * SJKVARN_ERR_ARG otherwise and for B < S, B inside a group or N < B with B > S; SJKVARN_ERR_CAPACITY where [B, N) does not fit
 * a ring. */
int sjk_hip_fork(const sjk_hip_view * dst, const sjk_hip_view * src, int n_layers, uint32_t B, uint32_t N, void * stream);

/* Blocks src_ids[i] of one pool's slab to blocks dst_ids[i] of another's (or the same) in every layer: block id of layer il lies
 * at base + il * layer_bytes + id * block_bytes. Ids are host arrays, read before the call returns; 448 pairs a launch. One
 * source may go to several destinations. SJKVARN_ERR_ARG for an id outside its slab, a destination twice, a destination that is
 * also a source of the same slab, slabs that overlap without being one, or addresses and sizes that are no multiples of 4. */
int sjk_hip_copy_blocks(uint8_t * d_dst, size_t dst_layer_bytes, uint32_t dst_blocks, const uint8_t * d_src, size_t src_layer_bytes,
                        uint32_t src_blocks, int n_layers, size_t block_bytes, const uint32_t * src_ids,
                        const uint32_t * dst_ids, uint32_t n, void * stream);

/* child goes on from parent's first pos positions (parallel samples, beams, a shared prompt). On one pool the child holds the
 * parent's sealed blocks with it; otherwise (another pool, or no pool on either side) their records are copied. Sink and staged
 * rows are copied. Everything is enqueued on `stream` after what the caller enqueued there, with no host wait; the caller orders
 * other streams. Where pos lies inside the sealed part the child starts at the group boundary below it, as
 * sj_kvarn_seq_truncate does; *kept (may be NULL) is the child's position count. The child is a new or reset sequence with the
 * parent's configuration (the status codes of sj_kvarn_seq_state_read otherwise; n_ctx and n_ubatch may differ:
 * SJKVARN_ERR_CAPACITY where the positions do not fit). SJKVARN_ERR_ARG for a child that is not empty or is the parent, or
 * pos past the parent's positions; SJKVARN_ERR_PENDING while a seal or a state restore of the parent, or any transfer of the child, is
 * pending; SJKVARN_ERR_POOL_FULL. A refused call changes nothing. */
int sjk_hip_seq_fork(sj_kvarn_seq * child, sj_kvarn_seq * parent, uint32_t pos, uint32_t * kept, void * stream);

/* Holders of a block of a pool of sj_kvarn_pool_init (0: free or no block of it) */
uint32_t sjk_hip_pool_refs(const sj_kvarn_pool * pool, uint32_t id);

/* Move the pool's live blocks to its lowest ids: afterwards ids [0, n_blocks - n_free) are held and the rest are free, lowest
 * first. seqs: every sequence that holds blocks of the pool, each once. Records are moved and the sequences' device block
 * tables rewritten on `stream`; the caller orders other streams that use these sequences. What the vacated blocks hold stays in
 * them. *moved (may be NULL): the blocks moved. SJKVARN_ERR_ARG, changing nothing, where a live block is not held by the
 * sequences given alone; SJKVARN_ERR_PENDING while a restore of one of them is in flight. */
int sjk_hip_pool_compact(sj_kvarn_pool * pool, sj_kvarn_seq * const * seqs, int n_seqs, uint32_t * moved, void * stream);

/* The log-domain scale update of the seal's variance balance, element-wise over device arrays: with
 * s = clamp(d_sd[i], 1e-3, 1e3), d_acc[i] = clamp(d_acc[i] + log((double) s), -0.3, 10) and d_scale[i] =
 * (float) exp(d_acc[i]) (sj_kvarn.h:1000-1002, 1006-1008). It is the seal's own device code, exported so that
 * the device's double log / exp can be compared with the host libm the reference calls. */
int sjk_hip_balance_step(const float * d_sd, double * d_acc, float * d_scale, int n, void * stream);

/* device view of a layer created by sj_kvarn_layer_init / sj_kvarn_seq_init (pool mode: the view
 * carries the sequence's device copy of its block table) */
sjk_hip_view sjk_layer_view(const sj_kvarn_layer * L);

/* last HIP error text seen by the library (for SJK_ERR_DEVICE) */
const char * sjk_last_error(void);

#ifdef __cplusplus
}
#endif
#endif /* SJK_H */
