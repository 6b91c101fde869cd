/*
 * ipl_b200.h - C ABI of the B200 (sm_100a) fused add+RMSNorm and SiLU-and-mul library, and of its
 * paged KV cache (rotary positions, attention, pages).
 *
 * Plain pointers and sizes only; no torch types cross this boundary. Every entry point is
 * stream-ordered: it validates its arguments on the host, enqueues its kernels (at most one for
 * the norm, SiLU and rotary calls) on `stream` (a cudaStream_t; NULL means the legacy default
 * stream) of the CURRENT device and returns without synchronising. Device pointers must be memory
 * of the current device. Nothing is allocated on the device: calls that need scratch memory take
 * it as a workspace, which may be reused by later work on the same stream.
 *
 * Element type is bfloat16 (passed as raw 16-bit words); arithmetic is fp32.
 *
 * Errors: every function returns IPL_SUCCESS (0) or a nonzero ipl_status. The message of the
 * last failure on the calling thread is available from ipl_last_error(); the messages repeat
 * the reference's STD_TORCH_CHECK texts where an equivalent check exists.
 *
 * Shared library: libipl_b200.so (link with -lipl_b200, or dlopen it).
 */
#ifndef IPL_B200_H_
#define IPL_B200_H_

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define IPL_ABI_VERSION 1

#if defined(__GNUC__)
#define IPL_API __attribute__((visibility("default")))
#else
#define IPL_API
#endif

typedef int ipl_status;

#define IPL_SUCCESS 0
#define IPL_ERROR_INVALID_VALUE 1 /* bad size, null pointer, non-positive epsilon */
#define IPL_ERROR_MISALIGNED 2    /* packed entry point given a pointer or width it cannot vectorise */
#define IPL_ERROR_TOO_LARGE 3     /* a dimension beyond what the kernels index */
#define IPL_ERROR_CUDA 4          /* a CUDA runtime call or kernel launch failed */

/*
 * Fused residual add + RMSNorm, in place, over `rows` rows of `hidden_size` bf16 elements:
 *
 *   v        = fp32(x) + fp32(residual)                (fp32, round to nearest)
 *   residual = bf16(v)                                 (bit-exact with the reference)
 *   x        = bf16(v * rsqrt(mean(v^2) + epsilon) * fp32(weight))
 *
 * x, residual: [rows, hidden_size] contiguous, distinct; weight: [hidden_size].
 * Any alignment of the three pointers is accepted. rows == 0 is a no-op.
 *
 * Replaces fused_add_rms_norm_cuda(Tensor& x, Tensor& residual, const Tensor& weight,
 * double epsilon) at csrc/fused_add_rms_norm_kernel.cu:276-329 of the reference, the body of
 * torch.ops.inference_performance_lab.fused_add_rms_norm (csrc/torch_ops.cpp:13,19).
 */
IPL_API ipl_status ipl_fused_add_rms_norm_bf16(void* x, void* residual, const void* weight, int64_t rows,
                                       int64_t hidden_size, double epsilon, void* stream);

/*
 * RMSNorm without a residual, out of place (output may equal input):
 *
 *   output = bf16((fp32(input) * rsqrt(mean(fp32(input)^2) + epsilon)) * fp32(weight))
 *
 * input, output: [rows, hidden_size] contiguous; weight: [hidden_size]. Any alignment is
 * accepted (output sharing input's offset modulo 16 bytes keeps the vectorised kernels).
 *
 * No counterpart in the reference's C++ sources: it is the plain rms_norm of the vLLM IR that
 * the reference's plugin targets (vllm/ir/ops/layernorm.py:9-21 of vLLM 0.22, the op before the
 * first and after the last decoder layer), with vLLM's torch.ops._C.rms_norm(out, input, weight,
 * epsilon) argument order and the reference oracle's fp32 arithmetic
 * (src/inference_performance_lab/kernels/reference.py:18-23 with a zero residual).
 */
IPL_API ipl_status ipl_rms_norm_bf16(void* output, const void* input, const void* weight, int64_t rows,
                                     int64_t hidden_size, double epsilon, void* stream);

/*
 * Fused residual add + RMSNorm with a statically scaled fp8 (e4m3) output:
 *
 *   v        = fp32(input) + fp32(residual)
 *   residual = bf16(v)                                            (bit-exact, in place)
 *   output   = e4m3(((v * rsqrt(mean(v^2) + epsilon)) * fp32(weight)) / *scale)
 *
 * e4m3 is OCP E4M3FN (bias 7, max 448, no infinities), round to nearest even, saturating to
 * +-448. input is read only. output: [rows, hidden_size] bytes; scale: one fp32 on the device.
 *
 * No counterpart in the reference's C++ sources: it is the fused variant the reference's scope
 * lists next (add+RMSNorm feeding an fp8 GEMM), with vLLM's
 * torch.ops._C.fused_add_rms_norm_static_fp8_quant(result, input, residual, weight, scale,
 * epsilon) argument order and the reference oracle's arithmetic up to the quantisation
 * (src/inference_performance_lab/kernels/reference.py:18-21).
 */
IPL_API ipl_status ipl_fused_add_rms_norm_static_fp8_quant(void* output, const void* input, void* residual,
                                                           const void* weight, const float* scale, int64_t rows,
                                                           int64_t hidden_size, double epsilon, void* stream);

/*
 * SiLU-and-multiply: output[r, c] = bf16(silu(fp32(input[r, c])) * fp32(input[r, I + c])),
 * I = intermediate_size, input [rows, 2*I] and output [rows, I], both contiguous. Any width and
 * alignment is accepted; aligned widths take the vector path. rows * I == 0 is a no-op.
 *
 * Replaces silu_and_mul_cuda(Tensor& output, const Tensor& input) at
 * csrc/silu_and_mul_kernel.cu:85-127 (torch.ops.inference_performance_lab.silu_and_mul,
 * csrc/torch_ops.cpp:14,20).
 */
IPL_API ipl_status ipl_silu_and_mul_bf16(void* output, const void* input, int64_t rows,
                                 int64_t intermediate_size, void* stream);

/*
 * Same computation with the reference's packed contract: intermediate_size must be a multiple
 * of 8 and both pointers 16-byte aligned, else IPL_ERROR_MISALIGNED with the reference's
 * message ("the output width must be divisible by 8", "input and output must be 16-byte
 * aligned"); no fallback path is taken.
 *
 * Replaces silu_and_mul_packed_cuda(Tensor& output, const Tensor& input) at
 * csrc/silu_and_mul_kernel.cu:129-180 (torch.ops.inference_performance_lab.silu_and_mul_packed,
 * csrc/torch_ops.cpp:15,21).
 */
IPL_API ipl_status ipl_silu_and_mul_packed_bf16(void* output, const void* input, int64_t rows,
                                        int64_t intermediate_size, void* stream);

/*
 * Rotary position embedding. For pair i of the first rotary_dim elements of every head, at position
 * p = positions[token]:
 *
 *   (a, b) := (a cos - b sin, b cos + a sin),  cos = cos_sin_cache[p][i],
 *                                              sin = cos_sin_cache[p][rotary_dim / 2 + i]
 *
 * with a, b = x[i], x[rotary_dim / 2 + i] (is_neox != 0) or x[2 i], x[2 i + 1]; fp32 arithmetic, one
 * rounding. Scaling for long contexts is folded into the table. query is [num_tokens, num_heads,
 * head_size], key [num_tokens, num_kv_heads, head_size], with the given strides in elements (the last
 * dimension contiguous). A token whose position is outside the table is skipped and bit 3 of the
 * device fault word set.
 *
 * ipl_rotary_embedding_bf16 rotates query and key in place (the members from value on are ignored).
 * ipl_rotary_embedding_cache_bf16 rotates query in place and writes the rotated key and the value to
 * slot slot_mapping[token] of the caches (page slot / page_size, row slot % page_size); key itself is
 * not modified. A negative slot writes nothing (query is still rotated); a token whose slot lies past
 * the cache is skipped and bit 3 of the fault word set. Slots of one call must differ.
 *
 * No counterpart in the reference's C++ sources, which leave the decoder layer between its two norms
 * to vLLM; the table is laid out as vLLM's cos_sin_cache.
 */
typedef struct ipl_rotary_args {
    const int64_t* positions;
    const float* cos_sin_cache; /* [max_position, rotary_dim] */
    void* query;
    void* key;
    int64_t num_tokens, num_heads, num_kv_heads, head_size, rotary_dim, max_position;
    int64_t query_token_stride, query_head_stride, key_token_stride, key_head_stride;
    int is_neox;
    const void* value;
    void* key_cache;
    void* value_cache;
    const int64_t* slot_mapping;
    int64_t value_token_stride, value_head_stride;
    int64_t num_pages, page_size;
    int64_t key_cache_page_stride, key_cache_token_stride, key_cache_head_stride;
    int64_t value_cache_page_stride, value_cache_token_stride, value_cache_head_stride;
} ipl_rotary_args;

IPL_API ipl_status ipl_rotary_embedding_bf16(const ipl_rotary_args* args, void* stream);
IPL_API ipl_status ipl_rotary_embedding_cache_bf16(const ipl_rotary_args* args, void* stream);

/*
 * Attention of new tokens over a paged KV cache. Sequence s owns the tokens query_start_loc[s] to
 * query_start_loc[s + 1] - 1 of query (none: it is skipped) and has seq_lens[s] tokens in the cache,
 * the new ones included. New token j of n sits at position P = seq_lens[s] - n + j and sees the keys at
 * positions t <= P, with window > 0 only those with t > P - window:
 *
 *   output = sum_t w_t v_t / sum_t w_t,   w_t = exp(scale q.k_t - max_t scale q.k_t)
 *
 * with fp32 scores, statistics and sums, rounded to bf16 once; the weights enter the product with the
 * values rounded to bf16 (their fp32 sum is the denominator), and are off by up to 1e-4 of themselves
 * before that (approximate exponentials). Equal calls give equal bits; which keys are summed together
 * depends on all sequences of a call, so in another call a sequence's last bits may differ. A token that sees no key gives 0, and so
 * does one all of whose scores are -infinity; NaN and +infinity among its scores give NaN. Query head h
 * reads key head h / (num_heads / num_kv_heads). Key t lies in page block_tables[s][t / page_size], row
 * t % page_size; table entries past a sequence's pages are never read, rows past its length never
 * matter, whatever they hold. Keys at masked positions never matter either; values that one token of a
 * sequence sees must be finite for its other tokens to be. A page number outside 0..num_pages-1
 * contributes nothing and sets bit 3 of the fault word; so do keys past the table's row or past 2^31 -
 * 256. Rows of query that belong to no sequence are not written.
 *
 * Strides are in elements; the last dimension is contiguous; output overlaps none of the inputs.
 * max_query_len and max_seq_len are upper bounds of the lengths, known on the host: they choose the
 * kernels and the split of long rows.
 * Sequences longer than the bounds are computed all the same, more slowly. The workspace
 * (ipl_paged_attention_workspace bytes, 16-byte aligned) holds the parts of split rows.
 *
 * No counterpart in the reference's C++ sources (see the rotary calls).
 */
typedef struct ipl_paged_attention_args {
    void* output;
    const void* query;
    const void* key_cache;
    const void* value_cache;
    const int32_t* block_tables;    /* [num_seqs, table_width], row stride table_stride */
    const int32_t* query_start_loc; /* [num_seqs + 1], non-decreasing from 0 */
    const int32_t* seq_lens;        /* [num_seqs] */
    int64_t num_tokens, num_seqs, num_heads, num_kv_heads, head_size;
    int64_t num_pages, page_size, table_width, table_stride;
    int64_t output_token_stride, output_head_stride, query_token_stride, query_head_stride;
    int64_t key_cache_page_stride, key_cache_token_stride, key_cache_head_stride;
    int64_t value_cache_page_stride, value_cache_token_stride, value_cache_head_stride;
    int64_t max_query_len, max_seq_len;
    int64_t window; /* 0: none */
    double scale;
    void* workspace;
    size_t workspace_bytes;
} ipl_paged_attention_args;

IPL_API ipl_status ipl_paged_attention_bf16(const ipl_paged_attention_args* args, void* stream);
/* Bytes of workspace the call needs (0: none); pointers are only looked at for their alignment. */
IPL_API ipl_status ipl_paged_attention_workspace(const ipl_paged_attention_args* args, size_t* bytes);
/* Names of the kernels the call launches, as the other plan queries. */
IPL_API const char* ipl_paged_attention_plan(const ipl_paged_attention_args* args);

/*
 * Pages of a KV cache, managed on the device. The pool's state is a block table per row (entry j: the
 * page of tokens j * page_size and on, -1 where there is none), a length per row and a reference count
 * per page; a page is free when its count is 0. Claims take the lowest-numbered free pages in order, so
 * equal states give equal results. The caches (K and V of every layer) are opaque: num_caches bases in
 * a host array, page i of each at i * page_stride_bytes, page_bytes long (16-byte multiples; bases
 * 16-byte aligned).
 *
 * status receives 0, or the number of free pages lacking, or -1 for an entry out of range (a row, a
 * length, a row given twice, a child that holds tokens); unless it is 0 nothing has changed. A call
 * takes up to 16384 rows. Lengths and tables change through these calls alone: a claim writes the
 * entries past a row's length, and a page that still stood there keeps its reference for good.
 *
 * ipl_copy_pages: page pairs[2 i] to page pairs[2 i + 1] in every cache; negative entries are skipped.
 *   No target may be the source or target of another pair.
 * ipl_reserve_pages: rows[i] gets pages up to new_lens[i] tokens, and that length if it was shorter.
 * ipl_fork_sequences: children[i] (empty) becomes a copy of parents[i]: it shares the whole pages and
 *   gets a page of its own with a copy of a partly filled last one.
 * ipl_release_sequences: the pages of rows[i] lose one reference each, the row becomes empty.
 * ipl_compact_pages: the pages in use past the first `live` numbers move, in order, to the free numbers
 *   below. The renumbered tables ([num_rows, width] contiguous) and counts are written beside the old
 *   ones, which stay valid for work in flight: moved pages keep their data until they are claimed. The
 *   workspace (ipl_compact_pages_workspace bytes, 4-byte aligned) may be reused by later work on the stream.
 */
typedef struct ipl_page_pool {
    int32_t* block_tables;
    int32_t* seq_lens;
    int32_t* ref_counts;
    int64_t num_rows, width, table_stride, num_pages, page_size;
} ipl_page_pool;

typedef struct ipl_page_caches {
    void* const* caches;
    int64_t num_caches, page_stride_bytes, page_bytes;
} ipl_page_caches;

IPL_API ipl_status ipl_copy_pages(const ipl_page_caches* caches, int64_t num_pages, const int32_t* pairs,
                                  int64_t count, void* stream);
IPL_API ipl_status ipl_reserve_pages(const ipl_page_pool* pool, const int32_t* rows, const int32_t* new_lens,
                                     int64_t count, int32_t* status, void* stream);
IPL_API ipl_status ipl_fork_sequences(const ipl_page_caches* caches, const ipl_page_pool* pool, const int32_t* parents,
                                      const int32_t* children, int64_t count, int32_t* status, void* stream);
IPL_API ipl_status ipl_release_sequences(const ipl_page_pool* pool, const int32_t* rows, int64_t count, void* stream);
IPL_API ipl_status ipl_compact_pages_workspace(int64_t num_pages, size_t* bytes);
IPL_API ipl_status ipl_compact_pages(const ipl_page_caches* caches, const ipl_page_pool* pool,
                                     int32_t* new_block_tables, int32_t* new_ref_counts, int32_t* live,
                                     void* workspace, size_t workspace_bytes, void* stream);

/* Message of the last failing call on this thread ("" if none). Valid until the next call. */
IPL_API const char* ipl_last_error(void);

/* Static name of a status code. */
IPL_API const char* ipl_status_string(ipl_status status);

/* IPL_ABI_VERSION of the loaded library. */
IPL_API int ipl_abi_version(void);

/*
 * Device-side fault word of `device`: bit flags that a kernel sets when one of its bounded
 * waits on a shared-memory barrier runs out (the kernel then stops early and its outputs are
 * incomplete), and bit 3, set when a paged-cache kernel skipped a position, slot, page or row
 * outside its range. 0 means that neither has happened on that device. Reading it synchronises the
 * device. The waits never run out on a healthy GPU.
 */
IPL_API ipl_status ipl_device_fault_flags(int device, uint32_t* flags);

/* Clears the fault word of `device` (synchronous). */
IPL_API ipl_status ipl_clear_device_fault_flags(int device);

/*
 * Name of the kernel that ipl_fused_add_rms_norm_bf16 / ipl_rms_norm_bf16 /
 * ipl_fused_add_rms_norm_static_fp8_quant / ipl_silu_and_mul_bf16 would launch for these
 * arguments on the current device (no launch; the device's SM count and shared-memory limit are
 * read as a call reads them). Where no CUDA device can be queried, a B200's limits are assumed
 * (148 SMs, 232448 bytes of opt-in shared memory per block). Static string; "none" for an empty
 * batch, "invalid" when the arguments would be rejected.
 */
IPL_API const char* ipl_fused_add_rms_norm_plan(const void* x, const void* residual, const void* weight,
                                        int64_t rows, int64_t hidden_size);
IPL_API const char* ipl_rms_norm_plan(const void* output, const void* input, const void* weight,
                                      int64_t rows, int64_t hidden_size);
IPL_API const char* ipl_fused_add_rms_norm_static_fp8_quant_plan(const void* output, const void* input,
                                                                 const void* residual, const void* weight,
                                                                 int64_t rows, int64_t hidden_size);
IPL_API const char* ipl_silu_and_mul_plan(const void* output, const void* input, int64_t rows,
                                  int64_t intermediate_size);

#ifdef __cplusplus
}
#endif

#endif /* IPL_B200_H_ */
