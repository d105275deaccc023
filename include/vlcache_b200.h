/*
 * vlcache_b200 — C ABI of the B200-native (sm_100a) warm-prefill attention path
 * for Qwen2.5-VL in VLCache / nano-vllm.
 *
 * Every entry point takes plain device pointers, element strides, int32
 * metadata and a CUDA stream (passed as `void*`, NULL = legacy default stream),
 * and returns an int status (VLC_OK = 0).  No entry point allocates device
 * memory: callers own the KV cache, metadata, outputs and workspaces.
 * Argument errors are reported before any launch; data-dependent errors found
 * on the device (e.g. an out-of-range slot) are recorded in a device error
 * word that vlc_get_device_error() reads.
 *
 * Layout conventions (all bf16 unless stated):
 *   q        [num_tokens, num_heads, head_dim]      token stride given, head stride = head_dim
 *   key/value[num_tokens, num_kv_heads, head_dim]   token stride given (views of the QKV split)
 *   k_cache/v_cache per layer [num_slots, num_kv_heads, head_dim] contiguous,
 *            num_slots = num_blocks * block_size  (nano-vllm: [num_blocks, 256, Hk, D])
 *   block_tables [num_seqs, block_table_stride] int32, padded with -1
 *   slot_mapping [num_tokens] int32, -1 = skip
 */
#ifndef VLCACHE_B200_H
#define VLCACHE_B200_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* ---- status codes (host side) ---- */
#define VLC_OK 0
#define VLC_ERR_NULL 1        /* required pointer is NULL */
#define VLC_ERR_SHAPE 2       /* unsupported or inconsistent sizes */
#define VLC_ERR_STRIDE 3      /* stride/contiguity requirement violated */
#define VLC_ERR_ALIGN 4       /* pointer/stride not 16-byte aligned */
#define VLC_ERR_UNSUPPORTED 5 /* e.g. head_dim != 128 */
#define VLC_ERR_WORKSPACE 6   /* workspace missing or too small */
#define VLC_ERR_CUDA 7        /* a CUDA runtime/driver call failed */
#define VLC_ERR_PLAN 8        /* plan buffer malformed or too small */
#define VLC_ERR_METADATA 9    /* cu_seqlens / lengths inconsistent */

/* ---- device error codes (recorded by kernels, read by vlc_get_device_error) ---- */
#define VLC_DEV_ERR_SLOT_RANGE 101   /* slot >= num_slots or < -1 */
#define VLC_DEV_ERR_BLOCK_RANGE 102  /* block table entry out of range where a key is needed */
#define VLC_DEV_ERR_POSITION 103     /* rotary position outside the cos/sin cache */
#define VLC_DEV_ERR_LENGTH 104       /* a device length exceeds the host-side bound the grid was sized for */
#define VLC_DEV_ERR_PAGES 105        /* a free list without the pages that are needed (or without room for more) */
#define VLC_DEV_ERR_TOKEN 106        /* a drafted token past the vocabulary */
#define VLC_DEV_ERR_TIMEOUT 110      /* an mbarrier wait hit its bound (base; +role id) */

/* Library version (major*10000 + minor*100 + patch). */
int vlc_version(void);

/* Human-readable text for a status code. */
const char* vlc_status_string(int status);

/* Synchronises the current device and returns its device error word (0 = none).
 * reset != 0 clears the word afterwards. */
int vlc_get_device_error(int reset);

/* Number of SMs of the current device (used by the planners). */
int vlc_num_sms(void);

/* Self-test of the bounded waits every kernel uses (no fault, no hang): one warp
 * waits on a shared-memory barrier that is completed (arrive != 0) or never
 * completed (arrive == 0).  In the second case the wait gives up after
 * limit_cycles (1 .. about 4e9) and records VLC_DEV_ERR_TIMEOUT + VLC_SELFTEST_ROLE
 * in the device error word; the kernel returns and the context stays usable. */
#define VLC_SELFTEST_ROLE 31
int vlc_selftest_bounded_wait(long long limit_cycles, int arrive, void* stream);

/* --------------------------------------------------------------------------
 * KV scatter.
 * Replaces nanovllm/layers/attention.py:10-40 (store_kvcache_kernel + store_kvcache):
 *   k_cache.view(-1, D)[slot_mapping[i]] = key[i];  v_cache likewise;  slot -1 skipped.
 * key/value rows are row_elems = num_kv_heads*head_dim contiguous bf16 elements;
 * key_stride/value_stride are token strides in elements.  Bit-exact copy.
 * ------------------------------------------------------------------------ */
int vlc_store_kvcache(const void* key, int64_t key_stride, const void* value, int64_t value_stride,
                      void* k_cache, void* v_cache, const int32_t* slot_mapping, int num_tokens,
                      int row_elems, int64_t num_slots, void* stream);

/* --------------------------------------------------------------------------
 * Rotary embedding fused with the KV scatter.
 * Replaces RotaryEmbedding.forward (nanovllm/layers/rotary_embedding.py:37-48,
 * rotate-half apply_rotary_emb :6-14) followed by store_kvcache (attention.py:10-40):
 *   q_out[i] = rope(q[i], positions[i])        (q_out may be q: in place)
 *   slot_mapping != NULL: rope(key[i]) and value[i] to k_cache / v_cache row
 *                         slot_mapping[i] (-1 skipped; rows of num_kv_heads*head_dim)
 *   slot_mapping == NULL: rope(key[i]) to k_out[i] (value, caches unused)
 * positions: int64 [num_tokens]; cos_sin_cache: fp32 [max_position, head_dim]
 * (first half cos, second half sin, as the reference's buffer); head_dim ==
 * rotary_dim == 128.  Strides are token strides in elements.  fp32 math with each
 * product and sum rounded separately, bf16 round-to-nearest-even output.
 * ------------------------------------------------------------------------ */
int vlc_rope_store_kvcache(const int64_t* positions, const void* q, int64_t q_stride, void* q_out,
                           int64_t q_out_stride, const void* key, int64_t key_stride, const void* value,
                           int64_t value_stride, const float* cos_sin_cache, int64_t max_position,
                           int rotary_dim, void* k_cache, void* v_cache, const int32_t* slot_mapping,
                           int64_t num_slots, void* k_out, int64_t k_out_stride, int num_tokens,
                           int num_heads, int num_kv_heads, int head_dim, void* stream);

/* --------------------------------------------------------------------------
 * M-RoPE position shift of reused vision K (new capability; replaces the
 * verbatim row copy of nanovllm/engine/model_runner.py:170-180 copy_image_kv,
 * driven by nanovllm/engine/llm_engine.py:58-89).
 * For each of num_layers layers (layer l at k_cache + l*layer_stride elements)
 * and each row i: K row at src_slots[i] is rotated by the per-section position
 * delta (delta_thw[0..2] for the t/h/w sections of mrope_section[0..2] pairs)
 * and written to dst_slots[i] (dst_slots == NULL: in place).  When v_cache is
 * non-NULL and dst_slots is non-NULL, the V row is copied verbatim too.
 * RoPE convention: rotate-half pairs (j, j + head_dim/2), inv_freq[j] =
 * theta^(-2j/head_dim) (HF transformers modeling_qwen2_5_vl.py:627-665).
 * Math in fp32 with a host-built cos/sin table; bf16 storage.
 * src/dst rows must be disjoint sets (or dst == src in place).
 * ------------------------------------------------------------------------ */
int vlc_mrope_shift(void* k_cache, void* v_cache, int64_t layer_stride, int num_layers,
                    int64_t num_slots, int num_kv_heads, int head_dim, const int32_t* src_slots,
                    const int32_t* dst_slots, int num_rows, const int32_t* delta_thw,
                    const int32_t* mrope_section, float rope_theta, void* stream);

/* --------------------------------------------------------------------------
 * Warm-prefill attention plan (host-only, no CUDA calls).
 * Replaces the work decomposition flash-attn derives inside
 * flash_attn_varlen_func (called at nanovllm/layers/attention.py:64-70).
 * Inputs are HOST copies of cu_seqlens_q / cu_seqlens_k ([num_seqs+1]).
 * Query row i of sequence b has logical position
 *   k_len_b - q_len_b + i   (causal, bottom-right aligned, as flash-attn).
 * Writes an int32 plan into plan_out (capacity plan_capacity ints) and returns
 * VLC_OK; *plan_len receives the number of ints used.  num_sms = 0 queries the
 * current device (falls back to 148 without a device).
 * ------------------------------------------------------------------------ */
int vlc_prefill_plan(const int32_t* cu_seqlens_q, const int32_t* cu_seqlens_k, int num_seqs,
                     int num_heads, int num_kv_heads, int head_dim, int num_sms,
                     int32_t* plan_out, int64_t plan_capacity, int64_t* plan_len);

/* Upper bound (ints) of the plan for these sequences. */
int64_t vlc_prefill_plan_capacity(const int32_t* cu_seqlens_q, const int32_t* cu_seqlens_k,
                                  int num_seqs, int num_heads, int num_kv_heads, int num_sms);

/* The same plan for the general varlen attention: causal != 0 is vlc_prefill_plan;
 * causal == 0 lets every query row of a sequence see all k_len keys of it, as
 * flash_attn_varlen_func(..., causal=False) in the vision tower's window and full
 * attention (nanovllm/models/qwen2_5_vl.py:202-211).  head_dim: 64 < d <= 128,
 * a multiple of 16 (Qwen2.5-VL's vision heads: 80).  vlc_prefill_plan(...) equals
 * vlc_attention_plan(..., causal = 1, ...). */
int vlc_attention_plan(const int32_t* cu_seqlens_q, const int32_t* cu_seqlens_k, int num_seqs, int num_heads,
                       int num_kv_heads, int head_dim, int causal, int num_sms, int32_t* plan_out,
                       int64_t plan_capacity, int64_t* plan_len);
int64_t vlc_attention_plan_capacity(const int32_t* cu_seqlens_q, const int32_t* cu_seqlens_k, int num_seqs,
                                    int num_heads, int num_kv_heads, int causal, int num_sms);

/* Unit kind of the prefill plans built from now on (process-wide): 1 = pairs of query
 * tiles sharing each K/V block on one SM; 2 = quads of tiles on CTA pairs (clusters of 2,
 * tcgen05.mma.cta_group::2; each SM loads half of every K/V block); 0 = the default (1).
 * Packed plans always use pairs.  A plan records its kind; vlc_prefill_attn follows it. */
int vlc_prefill_set_kernel(int mode);

/* Workspace bytes vlc_prefill_attn needs for a given (host) plan. */
int64_t vlc_prefill_workspace_size(const int32_t* plan_host);

/* --------------------------------------------------------------------------
 * Sparse-query paged prefill attention (tcgen05 / TMEM / TMA, sm_100a).
 * Replaces flash_attn_varlen_func(q, k, v, cu_seqlens_q, cu_seqlens_k,
 * max_seqlen_q, max_seqlen_k, softmax_scale, causal=True, block_table=...)
 * at nanovllm/layers/attention.py:64-70, both of its branches:
 *   paged      (block_tables != NULL): k/v are one layer's caches, key j of
 *              sequence b lives at row block_tables[b][j / block_size] *
 *              block_size + j % block_size (block_size a multiple of 128);
 *   contiguous (block_tables == NULL): key j of sequence b is row
 *              cu_seqlens_k[b] + j of k/v (the in-flight K/V of a cold prefill).
 *   o[i, h, :] = softmax(scale * q[i,h,:] . K[j, h/G, :]^T, j <= pos(i)) V
 * with GQA group G = num_heads / num_kv_heads.  k_row_stride / v_row_stride
 * are the element strides between consecutive key rows (num_kv_heads*head_dim
 * for a cache); num_kv_rows is the number of rows addressable through k/v.
 * plan_dev is the plan from vlc_prefill_plan copied to device memory;
 * plan_host is the same plan on the host (only its header is read).
 * out: [total_q, num_heads, head_dim] bf16 with token stride out_token_stride.
 * head_dim: 64 < d <= 128, a multiple of 16, equal to the plan's (q/k/v tiles are
 * zero-padded to 128 columns on load; outputs are written for the d real ones).
 * The plan's causal flag selects the mask (vlc_attention_plan).
 * Launch order: the attention is a programmatic dependent launch of the kernel
 * enqueued just before it on `stream` (its setup overlaps that kernel's tail).
 * That kernel may write q, k, v and block_tables (vlc_step_metadata makes them on the
 * device); plan_dev must have been written by a copy or by an earlier kernel.
 * ------------------------------------------------------------------------ */
int vlc_prefill_attn(const void* q, int64_t q_token_stride, int total_q, int num_heads,
                     const void* k, const void* v, int64_t k_row_stride, int64_t v_row_stride,
                     int64_t num_kv_rows, int num_kv_heads, int head_dim,
                     const int32_t* block_tables, int block_table_stride, int block_size,
                     const int32_t* plan_dev, const int32_t* plan_host, float softmax_scale,
                     void* out, int64_t out_token_stride, void* workspace,
                     int64_t workspace_bytes, void* stream);

/* Same as vlc_prefill_attn, plus the step's in-flight K/V: k_new / v_new hold the
 * rows the projection produced for the queries ([num_new_rows >= total_q, num_kv_heads,
 * head_dim], row strides kn_row_stride / vn_row_stride; row i is the key / value of query
 * row i, before store_kvcache copies it into the cache).  A sequence whose q_len equals
 * its k_len attends over exactly its own rows (a warm request's first sub-sequence:
 * model_runner.py:237-242 builds Q = K = tokens [0, img_start + R)), so its keys are read
 * from these rows instead of the cache and its work does not wait for the kernel
 * launched just before; the other sequences' K/V loads do.  That kernel may only write
 * the paged cache (the KV scatter), and must be an ordinary stream-ordered launch: q,
 * k_new, v_new complete and out / workspace free when it starts. */
int vlc_prefill_attn_inflight(const void* q, int64_t q_token_stride, int total_q, int num_heads,
                              const void* k, const void* v, int64_t k_row_stride, int64_t v_row_stride,
                              int64_t num_kv_rows, int num_kv_heads, int head_dim,
                              const int32_t* block_tables, int block_table_stride, int block_size,
                              const int32_t* plan_dev, const int32_t* plan_host, float softmax_scale,
                              void* out, int64_t out_token_stride, void* workspace,
                              int64_t workspace_bytes, const void* k_new, const void* v_new,
                              int64_t kn_row_stride, int64_t vn_row_stride, int64_t num_new_rows,
                              void* stream);

/* --------------------------------------------------------------------------
 * Split-K paged flash-decode.
 * Replaces flash_attn_with_kvcache(q.unsqueeze(1), k_cache, v_cache,
 * cache_seqlens=context_lens, block_table=block_tables, softmax_scale, causal=True)
 * at nanovllm/layers/attention.py:71-74 (one query token per sequence).
 * q: [num_seqs, num_heads, head_dim] (token stride q_seq_stride); out likewise.
 * context_lens [num_seqs] int32 on device; max_context_len is a host-side upper
 * bound used only to size the grid (graph-capture safe: no host reads).  A
 * context length above the keys that grid covers is recorded as
 * VLC_DEV_ERR_LENGTH and only the covered keys are attended (no access outside
 * the workspace).
 * ------------------------------------------------------------------------ */
int vlc_decode_attn(const void* q, int64_t q_seq_stride, int num_seqs, int num_heads,
                    const void* k_cache, const void* v_cache, int64_t num_slots, int num_kv_heads,
                    int head_dim, const int32_t* block_tables, int block_table_stride,
                    int block_size, const int32_t* context_lens, int max_context_len,
                    float softmax_scale, void* out, int64_t out_seq_stride, void* workspace,
                    int64_t workspace_bytes, void* stream);

/* Workspace bytes vlc_decode_attn needs. */
int64_t vlc_decode_workspace_size(int num_seqs, int num_heads, int num_kv_heads,
                                  int max_context_len);

/* --------------------------------------------------------------------------
 * Decode that allocates nothing.  No counterpart in the reference: it exists for
 * callers that cannot allocate device memory (a runtime with a fixed memory budget,
 * a process that may not call cudaMalloc after start-up).  Same arguments and
 * result as vlc_decode_attn minus the workspace: the split partials go to a
 * library-owned device array of vlc_decode_noalloc_scratch_bytes() (8 MiB) that
 * every GPU loading the library holds until exit.  Requests needing more
 * (vlc_decode_workspace_size() larger than that) return VLC_ERR_WORKSPACE without
 * launching.  Calls on one device share the array: calls that overlap on the GPU
 * race.  The first call on each device looks up the array's device address; make
 * it before any stream capture.
 * ------------------------------------------------------------------------ */
int vlc_decode_attn_noalloc(const void* q, int64_t q_seq_stride, int num_seqs, int num_heads,
                            const void* k_cache, const void* v_cache, int64_t num_slots,
                            int num_kv_heads, int head_dim, const int32_t* block_tables,
                            int block_table_stride, int block_size, const int32_t* context_lens,
                            int max_context_len, float softmax_scale, void* out,
                            int64_t out_seq_stride, void* stream);

/* Size in bytes of the built-in scratch array used by vlc_decode_attn_noalloc. */
int64_t vlc_decode_noalloc_scratch_bytes(void);

/* --------------------------------------------------------------------------
 * Warm-prefill metadata on the device.  Replaces the O(tokens) host loops of
 * nanovllm/engine/model_runner.py:160-168 (_compute_slots), :182-192 (padded block
 * tables), :232-276 (warm branch of prepare_prefill: positions, slot_mapping) and
 * nanovllm/engine/llm_engine.py:75-89 (_do_image_kv_copy: old/new slots of the
 * reused image rows).  The host lists O(requests) descriptors (device int32):
 *   vseq_desc[num_vseqs][7]  = {q_begin, q_len, first position, block-table offset
 *                               into block_tables_flat, block-table length, first
 *                               slot_mapping row (-1: none), output block-table row
 *                               (-1: none)}; a warm request is two virtual sequences,
 *                               [0, img_start + R) and [img_end, seqlen);
 *   reuse_desc[num_reuse][8] = {output offset, rows, first new position, new table
 *                               offset, new table length, first old position, old
 *                               table offset, old table length}.
 * Outputs (device; positions / slot_mapping / block_tables may be NULL):
 *   positions[q] (int64), slot_mapping[q] (int32), block_tables[num_vseqs][width]
 *   (int32, -1 padded), src_slots / dst_slots[rows] (int32).
 * slot(p) = table[p / block_size] * block_size + p % block_size; a page index past
 * the table's length writes -1 and records VLC_DEV_ERR_BLOCK_RANGE.  One launch. */
int vlc_warm_metadata(const int32_t* vseq_desc, int num_vseqs, const int32_t* reuse_desc, int num_reuse,
                      const int32_t* block_tables_flat, int block_size, int64_t* positions,
                      int32_t* slot_mapping, int32_t* block_tables, int block_table_width,
                      int32_t* src_slots, int32_t* dst_slots, void* stream);

/* --------------------------------------------------------------------------
 * Linear layers of the recomputed rows (tcgen05 GEMM, sm_100a).  All take
 * x [m, k] bf16 (row stride ldx) and a weight [rows, k] bf16 (row stride ldw,
 * nn.Linear layout), compute in fp32 and write bf16.  k, strides and output
 * columns must be multiples of 8; pointers 16-byte aligned.
 *
 * Workspace (optional, all three): with workspace != NULL the K-block work may
 * be split evenly over one CTA per SM (stream-K), which keeps every SM busy when
 * the output has fewer 128 x 256 tiles than the GPU has SMs and each tile is
 * long (>= 64 K blocks: down_proj of the recomputed rows); the library uses the
 * split only there and otherwise leaves the workspace untouched.  Size: vlc_linear_workspace_size(kind,
 * m, n, k) bytes, 256-byte aligned, ZEROED before its first use; each launch
 * leaves it reusable (its tickets back at zero).  Launches sharing one
 * workspace must not overlap on the GPU.  After a recorded device error, zero
 * it again.  workspace == NULL: whole output tiles per CTA.
 * kind: 0 vlc_linear, 1 vlc_linear_silu_mul (n = intermediate), 2 vlc_qkv_*
 * (n = (num_heads + 2 num_kv_heads) * head_dim).
 *
 * vlc_linear: out[m, n] = x . weight^T (+ bias[n]).
 *   Replaces F.linear in RowParallelLinear / ColumnParallelLinear
 *   (nanovllm/layers/linear.py:73, :154; o_proj and down_proj of
 *   nanovllm/models/qwen3.py:86, :116).
 * ------------------------------------------------------------------------ */
int64_t vlc_linear_workspace_size(int kind, int m, int n, int k);

/* Which GEMM kernel the linear entry points use, process-wide: 0 automatic (default: a
 * cost model fitted on B200 picks per shape), 1 single-SM 128 x 256 tiles (with the
 * stream-K split where it pays), 2 CTA pairs (clusters of 2, tcgen05.mma.cta_group::2,
 * 256 x 256 tiles), 3 single-SM 128 x 128 tiles, 4 single-SM 128 x 224 tiles (vlc_linear
 * only; the fused epilogues use the automatic choice).  A tuning and test switch; results
 * agree within the GEMM tolerance. */
int vlc_linear_set_kernel(int mode);

int vlc_linear(const void* x, int64_t ldx, const void* weight, int64_t ldw, const void* bias, void* out,
               int64_t ldo, int m, int n, int k, void* workspace, int64_t workspace_bytes, void* stream);

/* vlc_linear_silu_mul: gate_up_weight is [2 * intermediate, k] (gate rows, then up
 * rows, MergedColumnParallelLinear's layout); out[m, intermediate] =
 * silu(g) * u with g, u the bf16-rounded gate / up outputs, evaluated in fp32.
 *   Replaces gate_up_proj + SiluAndMul (nanovllm/models/qwen3.py:112-114,
 *   nanovllm/layers/activation.py:8-14). */
int vlc_linear_silu_mul(const void* x, int64_t ldx, const void* gate_up_weight, int64_t ldw, void* out,
                        int64_t ldo, int m, int intermediate, int k, void* workspace, int64_t workspace_bytes,
                        void* stream);

/* vlc_qkv_rope_store_kvcache: the QKV projection of the recomputed rows with its
 * bias, the rotary embedding and the KV scatter in one kernel.  qkv_weight is
 * [(num_heads + 2 num_kv_heads) * head_dim, hidden] (q rows, k rows, v rows,
 * QKVParallelLinear's layout).  Row i: qkv = bf16(x[i] . W^T + bias); q and k
 * heads rotated at positions[i] as vlc_rope_store_kvcache does (cos_sin_cache
 * [max_position, 128] fp32); q to q_out[i] ([m, num_heads, 128], row stride
 * q_out_stride); k and v rows to k_cache / v_cache row slot_mapping[i] (-1:
 * not stored; rows of num_kv_heads * 128).  head_dim must be 128.
 *   Replaces qkv_proj -> rotary_emb -> store_kvcache
 *   (nanovllm/models/qwen3.py:75-84, rotary_embedding.py:37-48, attention.py:10-40).
 * Out-of-range slots / positions are recorded as VLC_DEV_ERR_SLOT_RANGE /
 * VLC_DEV_ERR_POSITION and the row's stores skipped.  Whole output tiles only:
 * the workspace arguments are accepted and left untouched. */
int vlc_qkv_rope_store_kvcache(const void* x, int64_t ldx, const void* qkv_weight, int64_t ldw,
                               const void* qkv_bias, const int64_t* positions, const float* cos_sin_cache,
                               int64_t max_position, void* q_out, int64_t q_out_stride, void* k_cache,
                               void* v_cache, const int32_t* slot_mapping, int64_t num_slots, int m, int hidden,
                               int num_heads, int num_kv_heads, int head_dim, void* workspace,
                               int64_t workspace_bytes, void* stream);

/* --------------------------------------------------------------------------
 * Content hash of encoder-cache inputs.  Replaces EncoderCacheManager.compute_hash
 * (nanovllm/engine/encoder_cache_manager.py:24-29: XXH64 of grid_thw bytes then
 * pixel bytes, on the host, called per image at nanovllm/engine/llm_engine.py:52)
 * with a tree of XXH64 whose leaves hash in parallel (same bytes -> same key):
 *   d1[i] = XXH64(data[1024 i, 1024 (i+1)), seed 1)      (last chunk shorter)
 *   d2[j] = XXH64(d1 as little-endian bytes [512 j, 512 (j+1)), seed 2)
 *   d3[k] = XXH64(d2 as little-endian bytes [1024 k, 1024 (k+1)), seed 3)
 *   digest = XXH64(little-endian uint64 words {header_len, header zero-padded to a
 *            multiple of 8 bytes, nbytes, n1 = #d1, d3...}, seed 4)
 * header: the caller's bytes (e.g. grid_thw as int64 x 3), at most 256.
 *
 * vlc_content_hash_device: data in device memory; digest (one uint64) written to
 *   device memory `digest` on `stream` (two launches); workspace of
 *   vlc_content_hash_workspace_size(nbytes) bytes, 16-byte aligned.
 * vlc_content_hash_host: data in host memory, level 1 split over num_threads
 *   threads (<= 0: all hardware threads); digest written to *digest.
 * vlc_xxh64: plain XXH64 of a host buffer (the tree's primitive). */
int64_t vlc_content_hash_workspace_size(int64_t nbytes);
int vlc_content_hash_device(const void* data, int64_t nbytes, const void* header, int header_bytes, void* workspace,
                            int64_t workspace_bytes, uint64_t* digest, void* stream);
int vlc_content_hash_host(const void* data, int64_t nbytes, const void* header, int header_bytes, int num_threads,
                          uint64_t* digest);
uint64_t vlc_xxh64(const void* data, int64_t nbytes, uint64_t seed);

/* --------------------------------------------------------------------------
 * Rotary embedding at positions with several axes (time, height, width) fused with the
 * KV scatter.  No counterpart in the reference (get_rope ignores rope_scaling,
 * nanovllm/layers/rotary_embedding.py:51-71); the rotation is HF transformers'
 * apply_multimodal_rotary_pos_emb (modeling_qwen2_5_vl.py:627-665).
 *   positions [num_axes][axis_stride] int64, num_axes 1 .. 4 (axis_stride 0: one row for
 *   every axis); sections[num_axes] pairs per axis, in order, summing to head_dim / 2:
 *   rotate-half pair j takes the position of the axis whose section holds it.
 * Everything else as vlc_rope_store_kvcache, whose result it gives, bit for bit, when a
 * row's positions are equal on all axes.  A row with a position outside the table on any
 * axis is recorded (VLC_DEV_ERR_POSITION) and its q and k are not stored.
 * ------------------------------------------------------------------------ */
int vlc_mrope_store_kvcache(const int64_t* positions, int64_t axis_stride, int num_axes, const int32_t* sections,
                            const void* q, int64_t q_stride, void* q_out, int64_t q_out_stride, const void* key,
                            int64_t key_stride, const void* value, int64_t value_stride,
                            const float* cos_sin_cache, int64_t max_position, void* k_cache, void* v_cache,
                            const int32_t* slot_mapping, int64_t num_slots, void* k_out, int64_t k_out_stride,
                            int num_tokens, int num_heads, int num_kv_heads, int head_dim, void* stream);

/* --------------------------------------------------------------------------
 * The KV cache in 4 bits.  No counterpart in the reference.
 * A head's row of 128 dims is 8 groups of 16; a group holds one e4m3 scale s and 16 e2m1
 * codes (two per byte, the even dim in the low nibble).  With g a power of two per cache
 * (k_scale, v_scale; 2^-64 .. 2^64):
 *   s = e4m3(min(max|x / g| / 6, 448)),  code = e2m1(x / g / s),  value = g * s * code,
 * rounded to nearest even; codes are 0 where s is 0, magnitudes above 6 become 6, a NaN
 * makes its whole group NaN.  Every value is exact in bf16.  Choose g so that max|x| / g
 * stays below 2688 and the small groups' max|x| / g above 6 * 2^-6.
 * Page of one layer's K or V: [num_kv_heads][block_size * 64 code bytes | block_size * 8
 * scale bytes], block_size a multiple of 64, at most 2^20; caches [num_pages] such pages,
 * contiguous.  The slots that one call writes differ.
 * Slot -> page slot / block_size, row slot % block_size, as in the bf16 cache.
 *
 * vlc_rope_store_kvcache_fp4: vlc_mrope_store_kvcache with its k and v rows quantised into
 *   such a cache (num_axes = 1, sections = {64}: the one-axis rotation).  The key is
 *   rounded to bf16 first, as the bf16 cache holds it.
 * vlc_store_kvcache_fp4: the rows without a rotation (vlc_store_kvcache's contract).
 * vlc_gather_kvcache_fp4: the values of keys 0 .. len_b - 1 of every sequence, row
 *   cu_seqlens_k[b] + j of k_out / v_out ([total_k, num_kv_heads, 128] bf16, row stride
 *   out_row_stride elements), for num_layers layers (layer l of the caches at
 *   l * layer_stride bytes, of the outputs at l * out_layer_stride elements).
 *   cu_seqlens_k: device, num_seqs + 1.  Keys of a bad table entry read as 0, as in the bf16
 *   prefill (the 4-bit decode leaves them out), and are recorded (VLC_DEV_ERR_BLOCK_RANGE);
 *   rows past total_k are recorded (VLC_DEV_ERR_LENGTH) and not written.
 * vlc_gather_seen_kvcache_fp4: the same for an attention with a window (vlc_attention_plan_window): of each
 *   sequence, keys from the sinks up to lows[b] (device; the first key that its first row's window
 *   shows) are seen by no row, and lows[b] < 0 says that none is seen (no rows): tiles of 64 keys of
 *   them are not read, their table entries may be -1, and their rows of the outputs stay as they were.
 * vlc_mrope_shift_fp4: vlc_mrope_shift in such a cache: K rows of src_slots rotated by the
 *   delta, rounded to bf16, quantised again, written to dst_slots (NULL: in place); V rows
 *   copied when dst_slots is given.  A group whose 16 pairs the delta does not turn keeps
 *   its bits.  layer_stride in bytes.
 * vlc_decode_attn_fp4: vlc_decode_attn over such a cache: f16 products of exact K / V
 *   values with q (scaled per head by a power of two) and P, fp32 sums.  Keys of a chunk of
 *   64 whose table entry is bad are left out and recorded.  A head whose q holds an infinity or a
 *   NaN gives NaN, unless its sequence has no key (zeros).  The workspace, 32-byte aligned,
 *   holds the parts of keys split over the grid; calls that may overlap take one each.
 * ------------------------------------------------------------------------ */
int vlc_rope_store_kvcache_fp4(const int64_t* positions, int64_t axis_stride, int num_axes, const int32_t* sections,
                               const void* q, int64_t q_stride, void* q_out, int64_t q_out_stride, const void* key,
                               int64_t key_stride, const void* value, int64_t value_stride,
                               const float* cos_sin_cache, int64_t max_position, void* k_cache, void* v_cache,
                               const int32_t* slot_mapping, int64_t num_pages, int block_size, float k_scale,
                               float v_scale, int num_tokens, int num_heads, int num_kv_heads, int head_dim,
                               void* stream);
int vlc_store_kvcache_fp4(const void* key, int64_t key_stride, const void* value, int64_t value_stride, void* k_cache,
                          void* v_cache, const int32_t* slot_mapping, int64_t num_pages, int block_size,
                          float k_scale, float v_scale, int num_tokens, int num_kv_heads, int head_dim, void* stream);
int vlc_gather_kvcache_fp4(const void* k_cache, const void* v_cache, int64_t layer_stride, int num_layers,
                           int64_t num_pages, int block_size, int num_kv_heads, int head_dim,
                           const int32_t* block_tables, int64_t block_table_stride, int block_table_width,
                           const int32_t* cu_seqlens_k, int num_seqs, int64_t total_k, float k_scale, float v_scale,
                           void* k_out, void* v_out, int64_t out_row_stride, int64_t out_layer_stride, void* stream);
int vlc_gather_seen_kvcache_fp4(const void* k_cache, const void* v_cache, int64_t layer_stride, int num_layers,
                                int64_t num_pages, int block_size, int num_kv_heads, int head_dim,
                                const int32_t* block_tables, int64_t block_table_stride, int block_table_width,
                                const int32_t* cu_seqlens_k, int num_seqs, int64_t total_k, float k_scale, float v_scale,
                                void* k_out, void* v_out, int64_t out_row_stride, int64_t out_layer_stride,
                                const int32_t* lows, int sinks, void* stream);
int vlc_mrope_shift_fp4(void* k_cache, void* v_cache, int64_t layer_stride, int num_layers, int64_t num_pages,
                        int block_size, int num_kv_heads, int head_dim, const int32_t* src_slots,
                        const int32_t* dst_slots, int num_rows, const int32_t* delta_thw,
                        const int32_t* mrope_section, float rope_theta, void* stream);
int vlc_decode_attn_fp4(const void* q, int64_t q_seq_stride, int num_seqs, int num_heads, const void* k_cache,
                        const void* v_cache, int64_t num_pages, int block_size, int num_kv_heads, int head_dim,
                        const int32_t* block_tables, int64_t block_table_stride, int block_table_width,
                        const int32_t* context_lens, int max_context_len, float softmax_scale, float k_scale,
                        float v_scale, void* out, int64_t out_seq_stride, void* workspace, int64_t workspace_bytes,
                        void* stream);
int64_t vlc_decode_fp4_workspace_size(int num_seqs, int num_heads, int num_kv_heads, int max_context_len);

/* --------------------------------------------------------------------------
 * Pages.  vlc_copy_pages: in each of num_planes planes (one layer's K or V: num_pages
 * pages of page_bytes, planes plane_stride bytes apart) page dst_pages[i] becomes a copy
 * of page src_pages[i] (device lists; a pair of -1 is skipped).  All in one launch and in
 * no order: destinations differ, and none is another pair's source.  An index out of
 * range is recorded (VLC_DEV_ERR_BLOCK_RANGE) and its pair skipped.
 * vlc_remap_block_tables: every entry p of a table (row stride row_stride) becomes
 * page_map[p]; -1 stays, an entry out of range is recorded and stays.
 * ------------------------------------------------------------------------ */
int vlc_copy_pages(void* base, int64_t plane_stride, int num_planes, int64_t page_bytes, int64_t num_pages,
                   const int32_t* src_pages, const int32_t* dst_pages, int num_pairs, void* stream);
int vlc_remap_block_tables(int32_t* block_tables, int64_t row_stride, int num_rows, int width,
                           const int32_t* page_map, int num_pages, void* stream);

/* --------------------------------------------------------------------------
 * A decode step with drafted tokens over a windowed cache.
 *
 * The mask of all of them: the row at position t of a sequence sees key j iff j <= t and
 * (window == 0 or j > t - window or j < sinks).  Pages that no row sees are not read: their
 * block-table entries may be -1.  A NaN or an infinity in V of a key that one row sees and
 * another row of its tile does not reaches both (0 * NaN); keys that no row sees may hold anything.
 *
 * vlc_attention_plan_window: vlc_attention_plan with that mask (causal plans; capacity and
 *   workspace as there); vlc_prefill_attn and vlc_prefill_attn_inflight follow the plan, and
 *   take a positive softmax_scale only.  A window that no sequence outgrows, and a window of 0, give the
 *   plan without one, unless tiles are split there: parts of split tiles keep 32 bits in windowed plans.
 * vlc_decode_attn_window: the last num_tokens tokens of each sequence (its key and value rows
 *   are in the cache, context_lens counts them): q / out [num_seqs * num_tokens, num_heads, 128]
 *   with any token stride, row i num_tokens + r being token context_lens[i] - num_tokens + r of
 *   sequence i.  At most 128 rows num_tokens * num_heads / num_kv_heads; block_size a multiple of
 *   32.  Tokens before a sequence's first and sequences of length 0 give zeros, a query row with
 *   an infinity or a NaN gives NaN.  Keys of a bad page that a row sees count as zeros and are
 *   recorded (VLC_DEV_ERR_BLOCK_RANGE), a length past max_context_len is cut to it and recorded
 *   (VLC_DEV_ERR_LENGTH).  Sizes come from host values, so the launches can be captured; workspace:
 *   vlc_decode_window_workspace_size bytes, 16-byte aligned, one per call in flight.
 * vlc_step_metadata: sequence i of context_lens[i] tokens takes new_lens[i] more (a context_lens[i] below 0: an
 *   idle place of the batch, whose new_lens[i] rows have position 0 and slot -1, and which takes no page and
 *   has length 0 after).  Block-table entries below 0 where they fall are filled from the end
 *   of the free list (free_pages[0 .. *num_free), the k-th missing page of the batch being
 *   free_pages[*num_free - 1 - k], sequences in order), then pages wholly behind the window of
 *   the first new row and behind the sinks go back to its end, in order, and their entries become
 *   -1.  Writes positions and slots of the new rows one sequence after another (position 0 and
 *   slot -1 in the rows behind the last, up to total_rows), their running sums cu_seqlens_q and
 *   those of the lengths with them cu_seqlens_k (num_seqs + 1 each, below 2^31), and the lengths
 *   new_context_lens.  Recorded, with slots of -1: pages that the list does not have
 *   (VLC_DEV_ERR_PAGES), positions past the table (VLC_DEV_ERR_BLOCK_RANGE); with the rows left
 *   out: more than total_rows (VLC_DEV_ERR_LENGTH).  The tables hold pages of their own: one that
 *   several tables share would be given back by each.  new_context_lens is no input's memory.
 * vlc_verify_drafts: draft i of a sequence (drafts[seq][i], -1: none from there on) is accepted iff
 *   u[i] * draft_probs[i][d] < target_probs[i][d], up to the first refusal; then a token is sampled
 *   from max(target - draft, 0) at the refused draft, or from the target's row behind the last
 *   accepted one, at the random number u_last: probability x counts floor(clamp(x, 0, 1) 2^42), and
 *   the token is the first whose running count passes floor(floor(u_last 2^24) total / 2^24).
 *   tokens[seq] = accepted drafts, that token, -1 ..; emitted[seq] = accepted drafts + 1, which
 *   context_lens[seq] (unless NULL, or below 0: an idle place) is moved on by.  Without
 *   draft_probs (NULL) a draft has probability 1, and refused it counts 0.  A difference without a
 *   positive value is replaced by the target's row; a row without one gives token -1.  target_probs
 *   [num_seqs][num_drafts + 1][vocab], draft_probs [num_seqs][num_drafts][vocab], strides in
 *   elements, dtype 0 fp32, 1 bf16, 2 fp16; at most 31 drafts and 2^18 tokens.  A draft past the
 *   vocabulary is recorded (VLC_DEV_ERR_TOKEN) and ends the drafts.  Every row of the step counts as stored.
 * vlc_verify_stored_drafts: the same of rows that have a page: row r of a sequence (its last token, then its
 *   drafts) is at position context_lens[seq] + r, and from the first on whose entry of the step's
 *   block tables is below 0 or past their width nothing is in the cache.  A draft there is none, and a sequence
 *   whose first row is there emits nothing: emitted 0, tokens -1, its length stays, and its next step
 *   begins with the same token.  So the lengths count stored tokens only, whatever the step's free list lacked.
 * ------------------------------------------------------------------------ */
int vlc_attention_plan_window(const int32_t* cu_seqlens_q, const int32_t* cu_seqlens_k, int num_seqs, int num_heads,
                              int num_kv_heads, int head_dim, int causal, int window, int sinks, int num_sms,
                              int32_t* plan_out, int64_t plan_capacity, int64_t* plan_len);
int vlc_decode_attn_window(const void* q, int64_t q_token_stride, int num_seqs, int num_tokens, int num_heads,
                           const void* k_cache, const void* v_cache, int64_t num_pages, int block_size,
                           int num_kv_heads, int head_dim, const int32_t* block_tables, int64_t block_table_stride,
                           int block_table_width, const int32_t* context_lens, int max_context_len, int window,
                           int sinks, float softmax_scale, void* out, int64_t out_token_stride, void* workspace,
                           int64_t workspace_bytes, void* stream);
int64_t vlc_decode_window_workspace_size(int num_seqs, int num_tokens, int num_heads, int num_kv_heads,
                                         int max_context_len, int window, int sinks);
int vlc_step_metadata(const int32_t* context_lens, const int32_t* new_lens, int num_seqs, int32_t* block_tables,
                      int64_t block_table_stride, int block_table_width, int block_size, int window, int sinks,
                      int32_t* free_pages, int free_capacity, int32_t* num_free, int64_t* positions,
                      int32_t* slot_mapping, int total_rows, int32_t* cu_seqlens_q, int32_t* cu_seqlens_k,
                      int32_t* new_context_lens, void* stream);
int vlc_verify_drafts(const int64_t* drafts, int64_t draft_stride, int num_seqs, int num_drafts,
                      const void* target_probs, int64_t target_seq_stride, int64_t target_row_stride,
                      const void* draft_probs, int64_t draft_seq_stride, int64_t draft_row_stride, int vocab, int dtype,
                      const float* u, int64_t u_stride, const float* u_last, int64_t* tokens, int32_t* emitted,
                      int32_t* context_lens, void* stream);
int vlc_verify_stored_drafts(const int64_t* drafts, int64_t draft_stride, int num_seqs, int num_drafts,
                             const void* target_probs, int64_t target_seq_stride, int64_t target_row_stride,
                             const void* draft_probs, int64_t draft_seq_stride, int64_t draft_row_stride, int vocab,
                             int dtype, const float* u, int64_t u_stride, const float* u_last, int64_t* tokens,
                             int32_t* emitted, int32_t* context_lens, const int32_t* block_tables,
                             int64_t block_table_stride, int block_table_width, int block_size, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* VLCACHE_B200_H */
