// Stable-LibTorch-ABI registration of the ops, a thin shim over the C ABI in ipl_b200.h.
//
// Namespace, schemas and in-place signatures are those of the reference
// (csrc/torch_ops.cpp:12-22): fused_add_rms_norm(Tensor(a!) x, Tensor(b!) residual,
// Tensor weight, float epsilon) -> (), silu_and_mul(Tensor(a!) output, Tensor input) -> (),
// silu_and_mul_packed(Tensor(a!) output, Tensor input) -> (). The tensor checks repeat the
// reference's (csrc/fused_add_rms_norm_kernel.cu:277-301, csrc/silu_and_mul_kernel.cu:86-106,
// :130-158) with the same messages, so callers see the same RuntimeError texts. The kernel runs
// on the current stream of the tensors' device, under a device guard; nothing synchronises.
#include <torch/csrc/stable/accelerator.h>
#include <torch/csrc/stable/library.h>
#include <torch/csrc/stable/tensor.h>
#include <torch/headeronly/core/ScalarType.h>
#include <torch/headeronly/util/Exception.h>

#include <torch/csrc/stable/ops.h>

#include <cstdint>
#include <limits>
#include <vector>

#include "ipl_b200.h"

// Declared by torch's C shim under USE_CUDA; the symbol lives in libtorch_cuda.
extern "C" AOTITorchError aoti_torch_get_current_cuda_stream(int32_t device_index, void** ret_stream);

namespace ts = torch::stable;

namespace {

void* current_stream(int32_t device_index) {
    void* stream = nullptr;
    const AOTITorchError err = aoti_torch_get_current_cuda_stream(device_index, &stream);
    STD_TORCH_CHECK(err == AOTI_TORCH_SUCCESS, "failed to query the current CUDA stream");
    return stream;
}

void raise_on_error(ipl_status status) {
    STD_TORCH_CHECK(status == IPL_SUCCESS, ipl_last_error());
}

void check_silu_tensors(const ts::Tensor& output, const ts::Tensor& input) {
    STD_TORCH_CHECK(input.is_cuda() && output.is_cuda(), "input and output must be CUDA tensors");
    STD_TORCH_CHECK(input.scalar_type() == torch::headeronly::ScalarType::BFloat16 &&
                        output.scalar_type() == torch::headeronly::ScalarType::BFloat16,
                    "input and output must use bfloat16");
    STD_TORCH_CHECK(input.is_contiguous() && output.is_contiguous(), "input and output must be contiguous");
    STD_TORCH_CHECK(input.device() == output.device(), "input and output must be on the same device");
    STD_TORCH_CHECK(input.dim() >= 1 && input.size(-1) % 2 == 0, "the final input dimension must be even");
    STD_TORCH_CHECK(output.dim() == input.dim(), "input and output must have the same rank");
    const int64_t intermediate_size = input.size(-1) / 2;
    STD_TORCH_CHECK(output.size(-1) == intermediate_size, "the output width must be half the input width");
    for (int64_t dimension = 0; dimension < input.dim() - 1; ++dimension) {
        STD_TORCH_CHECK(output.size(dimension) == input.size(dimension),
                        "input and output leading dimensions must match");
    }
}

void run_silu(ts::Tensor& output, const ts::Tensor& input, bool packed) {
    check_silu_tensors(output, input);
    if (output.numel() == 0) {
        return;
    }
    const int64_t intermediate_size = input.size(-1) / 2;
    const int64_t rows = output.numel() / intermediate_size;
    const int32_t device = input.get_device_index();
    const ts::accelerator::DeviceGuard device_guard(device);
    void* stream = current_stream(device);
    void* out = output.mutable_data_ptr();
    const void* in = input.const_data_ptr();
    raise_on_error(packed ? ipl_silu_and_mul_packed_bf16(out, in, rows, intermediate_size, stream)
                          : ipl_silu_and_mul_bf16(out, in, rows, intermediate_size, stream));
}

}  // namespace

void fused_add_rms_norm_cuda(ts::Tensor& x, ts::Tensor& residual, const ts::Tensor& weight, double epsilon) {
    STD_TORCH_CHECK(x.is_cuda(), "x must be a CUDA tensor");
    STD_TORCH_CHECK(residual.is_cuda(), "residual must be a CUDA tensor");
    STD_TORCH_CHECK(weight.is_cuda(), "weight must be a CUDA tensor");

    STD_TORCH_CHECK(x.scalar_type() == torch::headeronly::ScalarType::BFloat16, "x must use bfloat16");
    STD_TORCH_CHECK(residual.scalar_type() == torch::headeronly::ScalarType::BFloat16, "residual must use bfloat16");
    STD_TORCH_CHECK(weight.scalar_type() == torch::headeronly::ScalarType::BFloat16, "weight must use bfloat16");

    STD_TORCH_CHECK(x.is_contiguous(), "x must be contiguous");
    STD_TORCH_CHECK(residual.is_contiguous(), "residual must be contiguous");
    STD_TORCH_CHECK(weight.is_contiguous(), "weight must be contiguous");

    STD_TORCH_CHECK(x.sizes().equals(residual.sizes()), "x and residual must have identical shapes");
    STD_TORCH_CHECK(x.device() == residual.device() && x.device() == weight.device(),
                    "x, residual, and weight must be on the same device");
    STD_TORCH_CHECK(x.dim() >= 1, "x must have at least one dimension");
    STD_TORCH_CHECK(weight.dim() == 1, "weight must be one-dimensional");
    STD_TORCH_CHECK(weight.size(0) == x.size(-1), "weight must match the final tensor dimension");
    STD_TORCH_CHECK(epsilon > 0.0, "epsilon must be positive");

    const int64_t hidden_size = x.size(-1);
    if (x.numel() == 0) {
        // Nothing to normalise (the reference launches an empty grid here and fails).
        return;
    }
    const int64_t rows = x.numel() / hidden_size;

    STD_TORCH_CHECK(hidden_size <= std::numeric_limits<int>::max(), "hidden dimension is too large");
    STD_TORCH_CHECK(rows <= std::numeric_limits<int>::max(), "number of rows is too large");

    const int32_t device = x.get_device_index();
    const ts::accelerator::DeviceGuard device_guard(device);
    void* stream = current_stream(device);
    raise_on_error(ipl_fused_add_rms_norm_bf16(x.mutable_data_ptr(), residual.mutable_data_ptr(),
                                               weight.const_data_ptr(), rows, hidden_size, epsilon, stream));
}

void rms_norm_cuda(ts::Tensor& output, const ts::Tensor& input, const ts::Tensor& weight, double epsilon) {
    STD_TORCH_CHECK(output.is_cuda() && input.is_cuda() && weight.is_cuda(),
                    "output, input, and weight must be CUDA tensors");
    STD_TORCH_CHECK(output.scalar_type() == torch::headeronly::ScalarType::BFloat16 &&
                        input.scalar_type() == torch::headeronly::ScalarType::BFloat16 &&
                        weight.scalar_type() == torch::headeronly::ScalarType::BFloat16,
                    "output, input, and weight must use bfloat16");
    STD_TORCH_CHECK(output.is_contiguous() && input.is_contiguous() && weight.is_contiguous(),
                    "output, input, and weight must be contiguous");
    STD_TORCH_CHECK(output.sizes().equals(input.sizes()), "output and input must have identical shapes");
    STD_TORCH_CHECK(output.device() == input.device() && input.device() == weight.device(),
                    "output, input, and weight must be on the same device");
    STD_TORCH_CHECK(input.dim() >= 1, "input must have at least one dimension");
    STD_TORCH_CHECK(weight.dim() == 1, "weight must be one-dimensional");
    STD_TORCH_CHECK(weight.size(0) == input.size(-1), "weight must match the final tensor dimension");
    STD_TORCH_CHECK(epsilon > 0.0, "epsilon must be positive");
    if (input.numel() == 0) {
        return;
    }
    const int64_t hidden_size = input.size(-1);
    const int64_t rows = input.numel() / hidden_size;
    const int32_t device = input.get_device_index();
    const ts::accelerator::DeviceGuard device_guard(device);
    void* stream = current_stream(device);
    raise_on_error(ipl_rms_norm_bf16(output.mutable_data_ptr(), input.const_data_ptr(), weight.const_data_ptr(),
                                     rows, hidden_size, epsilon, stream));
}

void fused_add_rms_norm_static_fp8_quant_cuda(ts::Tensor& result, const ts::Tensor& input, ts::Tensor& residual,
                                              const ts::Tensor& weight, const ts::Tensor& scale, double epsilon) {
    STD_TORCH_CHECK(result.is_cuda() && input.is_cuda() && residual.is_cuda() && weight.is_cuda() && scale.is_cuda(),
                    "result, input, residual, weight, and scale must be CUDA tensors");
    STD_TORCH_CHECK(result.scalar_type() == torch::headeronly::ScalarType::Float8_e4m3fn,
                    "result must use float8_e4m3fn");
    STD_TORCH_CHECK(input.scalar_type() == torch::headeronly::ScalarType::BFloat16 &&
                        residual.scalar_type() == torch::headeronly::ScalarType::BFloat16 &&
                        weight.scalar_type() == torch::headeronly::ScalarType::BFloat16,
                    "input, residual, and weight must use bfloat16");
    STD_TORCH_CHECK(scale.scalar_type() == torch::headeronly::ScalarType::Float && scale.numel() == 1,
                    "scale must be a single float32");
    STD_TORCH_CHECK(result.is_contiguous() && input.is_contiguous() && residual.is_contiguous() &&
                        weight.is_contiguous(),
                    "result, input, residual, and weight must be contiguous");
    STD_TORCH_CHECK(input.sizes().equals(residual.sizes()) && input.sizes().equals(result.sizes()),
                    "result, input, and residual must have identical shapes");
    STD_TORCH_CHECK(input.device() == residual.device() && input.device() == weight.device() &&
                        input.device() == result.device() && input.device() == scale.device(),
                    "all tensors must be on the same device");
    STD_TORCH_CHECK(input.dim() >= 1, "input must have at least one dimension");
    STD_TORCH_CHECK(weight.dim() == 1, "weight must be one-dimensional");
    STD_TORCH_CHECK(weight.size(0) == input.size(-1), "weight must match the final tensor dimension");
    STD_TORCH_CHECK(epsilon > 0.0, "epsilon must be positive");
    if (input.numel() == 0) {
        return;
    }
    const int64_t hidden_size = input.size(-1);
    const int64_t rows = input.numel() / hidden_size;
    const int32_t device = input.get_device_index();
    const ts::accelerator::DeviceGuard device_guard(device);
    void* stream = current_stream(device);
    raise_on_error(ipl_fused_add_rms_norm_static_fp8_quant(
        result.mutable_data_ptr(), input.const_data_ptr(), residual.mutable_data_ptr(), weight.const_data_ptr(),
        static_cast<const float*>(scale.const_data_ptr()), rows, hidden_size, epsilon, stream));
}

void silu_and_mul_cuda(ts::Tensor& output, const ts::Tensor& input) { run_silu(output, input, false); }

void silu_and_mul_packed_cuda(ts::Tensor& output, const ts::Tensor& input) { run_silu(output, input, true); }

// ---- paged KV cache (not in the reference library) -----------------------------------------------

namespace {

using torch::headeronly::ScalarType;

void check_same_device(const ts::Tensor& first, const ts::Tensor& other, const char* message) {
    STD_TORCH_CHECK(other.is_cuda() && other.get_device_index() == first.get_device_index(), message);
}

// [tokens, heads, head_size] in bfloat16, the last dimension contiguous.
void check_heads(const ts::Tensor& t, const char* message) {
    STD_TORCH_CHECK(t.scalar_type() == ScalarType::BFloat16 && t.dim() == 3 && (t.numel() == 0 || t.stride(2) == 1 || t.size(2) == 1),
                    message);
}

// [pages, page_size, kv_heads, head_size] in bfloat16, the last dimension contiguous.
void check_cache(const ts::Tensor& t, const char* message) {
    STD_TORCH_CHECK(t.scalar_type() == ScalarType::BFloat16 && t.dim() == 4 && (t.numel() == 0 || t.stride(3) == 1 || t.size(3) == 1),
                    message);
}

void check_ints(const ts::Tensor& t, int64_t dim, const char* message) {
    STD_TORCH_CHECK(t.scalar_type() == ScalarType::Int && t.dim() == dim && (t.numel() == 0 || t.size(-1) <= 1 || t.stride(-1) == 1),
                    message);
}

ts::Tensor new_ints(const ts::Tensor& like, int64_t count) {
    const int64_t size[1] = {count};
    return ts::new_empty(like, torch::headeronly::IntHeaderOnlyArrayRef(size, 1), ScalarType::Int);
}

ipl_rotary_args rotary_args(const ts::Tensor& positions, ts::Tensor& query, const ts::Tensor& key,
                            const ts::Tensor& cos_sin_cache, bool is_neox) {
    STD_TORCH_CHECK(query.is_cuda(), "query must be a CUDA tensor");
    check_same_device(query, key, "query and key must be on the same device");
    check_same_device(query, positions, "query and positions must be on the same device");
    check_same_device(query, cos_sin_cache, "query and cos_sin_cache must be on the same device");
    check_heads(query, "query must be bfloat16 [tokens, heads, head_size] with a contiguous last dimension");
    check_heads(key, "key must be bfloat16 [tokens, kv_heads, head_size] with a contiguous last dimension");
    STD_TORCH_CHECK(positions.scalar_type() == ScalarType::Long && positions.dim() == 1 && positions.is_contiguous(),
                    "positions must be contiguous int64 [tokens]");
    STD_TORCH_CHECK(cos_sin_cache.scalar_type() == ScalarType::Float && cos_sin_cache.dim() == 2 &&
                        cos_sin_cache.is_contiguous(),
                    "cos_sin_cache must be contiguous float32 [positions, rotary_dim]");
    STD_TORCH_CHECK(key.size(0) == query.size(0) && positions.size(0) == query.size(0),
                    "positions, query and key must have the same number of tokens");
    STD_TORCH_CHECK(key.size(2) == query.size(2), "query and key must have the same head size");
    ipl_rotary_args a = {};
    a.positions = static_cast<const int64_t*>(positions.const_data_ptr());
    a.cos_sin_cache = static_cast<const float*>(cos_sin_cache.const_data_ptr());
    a.query = query.mutable_data_ptr();
    a.key = const_cast<void*>(key.const_data_ptr());
    a.num_tokens = query.size(0);
    a.num_heads = query.size(1);
    a.num_kv_heads = key.size(1);
    a.head_size = query.size(2);
    a.rotary_dim = cos_sin_cache.size(1);
    a.max_position = cos_sin_cache.size(0);
    a.query_token_stride = query.stride(0);
    a.query_head_stride = query.stride(1);
    a.key_token_stride = key.stride(0);
    a.key_head_stride = key.stride(1);
    a.is_neox = is_neox;
    return a;
}

ipl_page_pool page_pool(const ts::Tensor& tables, const ts::Tensor& ref_counts) {
    STD_TORCH_CHECK(tables.is_cuda(), "block_tables must be a CUDA tensor");
    check_same_device(tables, ref_counts, "block_tables and ref_counts must be on the same device");
    check_ints(tables, 2, "block_tables must be int32 [rows, width] with contiguous rows");
    check_ints(ref_counts, 1, "ref_counts must be contiguous int32 [pages]");
    ipl_page_pool pool = {};
    pool.block_tables = static_cast<int32_t*>(const_cast<void*>(tables.const_data_ptr()));
    pool.ref_counts = static_cast<int32_t*>(const_cast<void*>(ref_counts.const_data_ptr()));
    pool.num_rows = tables.size(0);
    pool.width = tables.size(1);
    pool.table_stride = tables.stride(0);
    pool.num_pages = ref_counts.size(0);
    pool.page_size = 1;
    return pool;
}

void add_rows(ipl_page_pool& pool, const ts::Tensor& tables, const ts::Tensor& seq_lens, const ts::Tensor& rows,
              const char* rows_message) {
    check_same_device(tables, seq_lens, "block_tables and seq_lens must be on the same device");
    check_same_device(tables, rows, "block_tables and the lists of rows must be on the same device");
    check_ints(seq_lens, 1, "seq_lens must be contiguous int32 [rows]");
    check_ints(rows, 1, rows_message);
    STD_TORCH_CHECK(seq_lens.size(0) == pool.num_rows, "seq_lens must have a length for each row of block_tables");
    pool.seq_lens = static_cast<int32_t*>(const_cast<void*>(seq_lens.const_data_ptr()));
}

// The caches of a call: alike in shape, type and strides, each [pages, page_size, ...], a page either
// its tokens one after the other or (four dimensions) its heads one after the other.
struct Caches {
    std::vector<void*> bases;
    ipl_page_caches args = {};
    int64_t num_pages = 0, page_size = 1;

    explicit Caches(std::vector<ts::Tensor>& caches, int32_t device) {
        bases.reserve(caches.size());
        for (size_t i = 0; i < caches.size(); ++i) {
            ts::Tensor& c = caches[i];
            STD_TORCH_CHECK(c.is_cuda() && c.get_device_index() == device, "caches and block_tables must be on the same device");
            STD_TORCH_CHECK(c.dim() >= 2, "caches must be [pages, page_size, ...]");
            if (i > 0) {
                STD_TORCH_CHECK(c.scalar_type() == caches[0].scalar_type() && c.sizes().equals(caches[0].sizes()) &&
                                    c.strides().equals(caches[0].strides()),
                                "caches must have the same type, shape and strides");
            }
            bases.push_back(c.mutable_data_ptr());
        }
        args.caches = bases.data();
        args.num_caches = static_cast<int64_t>(bases.size());
        if (caches.empty()) return;
        const ts::Tensor& c = caches[0];
        const int64_t element = static_cast<int64_t>(c.element_size());
        num_pages = c.size(0);
        page_size = c.size(1);
        STD_TORCH_CHECK(page_size >= 1, "caches must have a page size of at least one token");
        int64_t token = 1;
        for (int64_t d = 2; d < c.dim(); ++d) token *= c.size(d);
        args.page_bytes = page_size * token * element;
        args.page_stride_bytes = num_pages > 1 ? c.stride(0) * element : args.page_bytes;
        const bool tokens_follow = page_size == 1 || c.stride(1) == token;
        bool dense = true;
        int64_t expect = 1;
        for (int64_t d = c.dim() - 1; d >= 2; --d) {
            dense = dense && (c.size(d) == 1 || c.stride(d) == expect);
            expect *= c.size(d);
        }
        const bool heads_follow = c.dim() == 4 && (c.size(3) == 1 || c.stride(3) == 1) &&
                                  (page_size == 1 || c.stride(1) == c.size(3)) &&
                                  (c.size(2) == 1 || c.stride(2) == c.size(3) * page_size);
        STD_TORCH_CHECK(token == 0 || num_pages == 0 || (dense && tokens_follow) || heads_follow,
                        "the pages of a cache must be contiguous, tokens or heads one after the other");
    }
};

const int32_t* int_ptr(const ts::Tensor& t) { return static_cast<const int32_t*>(t.const_data_ptr()); }
int32_t* mutable_int_ptr(ts::Tensor& t) { return static_cast<int32_t*>(t.mutable_data_ptr()); }

}  // namespace

void rotary_embedding_cuda(const ts::Tensor& positions, ts::Tensor& query, ts::Tensor& key,
                           const ts::Tensor& cos_sin_cache, bool is_neox) {
    const ipl_rotary_args a = rotary_args(positions, query, key, cos_sin_cache, is_neox);
    const int32_t device = query.get_device_index();
    const ts::accelerator::DeviceGuard device_guard(device);
    raise_on_error(ipl_rotary_embedding_bf16(&a, current_stream(device)));
}

void rotary_embedding_cache_cuda(const ts::Tensor& positions, ts::Tensor& query, const ts::Tensor& key,
                                 const ts::Tensor& value, const ts::Tensor& cos_sin_cache, ts::Tensor& key_cache,
                                 ts::Tensor& value_cache, const ts::Tensor& slot_mapping, bool is_neox) {
    ipl_rotary_args a = rotary_args(positions, query, key, cos_sin_cache, is_neox);
    check_same_device(query, value, "query and value must be on the same device");
    check_same_device(query, key_cache, "query and key_cache must be on the same device");
    check_same_device(query, value_cache, "query and value_cache must be on the same device");
    check_same_device(query, slot_mapping, "query and slot_mapping must be on the same device");
    check_heads(value, "value must be bfloat16 [tokens, kv_heads, head_size] with a contiguous last dimension");
    STD_TORCH_CHECK(value.sizes().equals(key.sizes()), "key and value must have identical shapes");
    check_cache(key_cache, "key_cache must be bfloat16 [pages, page_size, kv_heads, head_size] with a contiguous last dimension");
    check_cache(value_cache, "value_cache must be bfloat16 [pages, page_size, kv_heads, head_size] with a contiguous last dimension");
    STD_TORCH_CHECK(key_cache.sizes().equals(value_cache.sizes()), "key_cache and value_cache must have identical shapes");
    STD_TORCH_CHECK(key_cache.size(2) == key.size(1) && key_cache.size(3) == key.size(2),
                    "the caches must have the heads and head size of key");
    STD_TORCH_CHECK(slot_mapping.scalar_type() == ScalarType::Long && slot_mapping.dim() == 1 &&
                        slot_mapping.is_contiguous() && slot_mapping.size(0) == query.size(0),
                    "slot_mapping must be contiguous int64 [tokens]");
    a.value = value.const_data_ptr();
    a.key_cache = key_cache.mutable_data_ptr();
    a.value_cache = value_cache.mutable_data_ptr();
    a.slot_mapping = static_cast<const int64_t*>(slot_mapping.const_data_ptr());
    a.value_token_stride = value.stride(0);
    a.value_head_stride = value.stride(1);
    a.num_pages = key_cache.size(0);
    a.page_size = key_cache.size(1);
    a.key_cache_page_stride = key_cache.stride(0);
    a.key_cache_token_stride = key_cache.stride(1);
    a.key_cache_head_stride = key_cache.stride(2);
    a.value_cache_page_stride = value_cache.stride(0);
    a.value_cache_token_stride = value_cache.stride(1);
    a.value_cache_head_stride = value_cache.stride(2);
    const int32_t device = query.get_device_index();
    const ts::accelerator::DeviceGuard device_guard(device);
    raise_on_error(ipl_rotary_embedding_cache_bf16(&a, current_stream(device)));
}

void paged_attention_cuda(ts::Tensor& output, const ts::Tensor& query, const ts::Tensor& key_cache,
                          const ts::Tensor& value_cache, const ts::Tensor& block_tables,
                          const ts::Tensor& query_start_loc, const ts::Tensor& seq_lens, int64_t max_query_len,
                          int64_t max_seq_len, double scale, int64_t window) {
    STD_TORCH_CHECK(query.is_cuda(), "query must be a CUDA tensor");
    check_same_device(query, output, "query and output must be on the same device");
    check_same_device(query, key_cache, "query and key_cache must be on the same device");
    check_same_device(query, value_cache, "query and value_cache must be on the same device");
    check_same_device(query, block_tables, "query and block_tables must be on the same device");
    check_same_device(query, query_start_loc, "query and query_start_loc must be on the same device");
    check_same_device(query, seq_lens, "query and seq_lens must be on the same device");
    check_heads(query, "query must be bfloat16 [tokens, heads, head_size] with a contiguous last dimension");
    check_heads(output, "output must be bfloat16 [tokens, heads, head_size] with a contiguous last dimension");
    check_cache(key_cache, "key_cache must be bfloat16 [pages, page_size, kv_heads, head_size] with a contiguous last dimension");
    check_cache(value_cache, "value_cache must be bfloat16 [pages, page_size, kv_heads, head_size] with a contiguous last dimension");
    check_ints(block_tables, 2, "block_tables must be int32 [sequences, width] with contiguous rows");
    check_ints(query_start_loc, 1, "query_start_loc must be contiguous int32 [sequences + 1]");
    check_ints(seq_lens, 1, "seq_lens must be contiguous int32 [sequences]");
    STD_TORCH_CHECK(output.sizes().equals(query.sizes()), "output and query must have identical shapes");
    STD_TORCH_CHECK(key_cache.sizes().equals(value_cache.sizes()), "key_cache and value_cache must have identical shapes");
    STD_TORCH_CHECK(key_cache.size(3) == query.size(2), "query and the caches must have the same head size");
    STD_TORCH_CHECK(block_tables.size(0) == seq_lens.size(0) && query_start_loc.size(0) == seq_lens.size(0) + 1,
                    "block_tables, query_start_loc and seq_lens must describe the same sequences");
    ipl_paged_attention_args a = {};
    a.output = output.mutable_data_ptr();
    a.query = query.const_data_ptr();
    a.key_cache = key_cache.const_data_ptr();
    a.value_cache = value_cache.const_data_ptr();
    a.block_tables = int_ptr(block_tables);
    a.query_start_loc = int_ptr(query_start_loc);
    a.seq_lens = int_ptr(seq_lens);
    a.num_tokens = query.size(0);
    a.num_heads = query.size(1);
    a.head_size = query.size(2);
    a.num_seqs = seq_lens.size(0);
    a.num_kv_heads = key_cache.size(2);
    a.num_pages = key_cache.size(0);
    a.page_size = key_cache.size(1);
    a.table_width = block_tables.size(1);
    a.table_stride = block_tables.stride(0);
    a.output_token_stride = output.stride(0);
    a.output_head_stride = output.stride(1);
    a.query_token_stride = query.stride(0);
    a.query_head_stride = query.stride(1);
    a.key_cache_page_stride = key_cache.stride(0);
    a.key_cache_token_stride = key_cache.stride(1);
    a.key_cache_head_stride = key_cache.stride(2);
    a.value_cache_page_stride = value_cache.stride(0);
    a.value_cache_token_stride = value_cache.stride(1);
    a.value_cache_head_stride = value_cache.stride(2);
    a.max_query_len = max_query_len;
    a.max_seq_len = max_seq_len;
    a.window = window;
    a.scale = scale;
    const int32_t device = query.get_device_index();
    const ts::accelerator::DeviceGuard device_guard(device);
    raise_on_error(ipl_paged_attention_workspace(&a, &a.workspace_bytes));
    if (a.workspace_bytes == 0) {
        raise_on_error(ipl_paged_attention_bf16(&a, current_stream(device)));
        return;
    }
    ts::Tensor workspace = new_ints(query, static_cast<int64_t>((a.workspace_bytes + 3) / 4));
    a.workspace = workspace.mutable_data_ptr();
    raise_on_error(ipl_paged_attention_bf16(&a, current_stream(device)));
}

void copy_pages_cuda(std::vector<ts::Tensor> caches, const ts::Tensor& pairs) {
    STD_TORCH_CHECK(pairs.is_cuda(), "pairs must be a CUDA tensor");
    STD_TORCH_CHECK(pairs.scalar_type() == ScalarType::Int && pairs.dim() == 2 && pairs.size(1) == 2 && pairs.is_contiguous(),
                    "pairs must be contiguous int32 [pairs, 2]");
    const int32_t device = pairs.get_device_index();
    const Caches c(caches, device);
    const ts::accelerator::DeviceGuard device_guard(device);
    raise_on_error(ipl_copy_pages(&c.args, c.num_pages, int_ptr(pairs), pairs.size(0), current_stream(device)));
}

ts::Tensor reserve_pages_cuda(ts::Tensor& block_tables, ts::Tensor& seq_lens, ts::Tensor& ref_counts,
                              const ts::Tensor& rows, const ts::Tensor& new_lens, int64_t page_size) {
    ipl_page_pool pool = page_pool(block_tables, ref_counts);
    add_rows(pool, block_tables, seq_lens, rows, "rows must be contiguous int32 [rows]");
    check_same_device(block_tables, new_lens, "block_tables and new_lens must be on the same device");
    check_ints(new_lens, 1, "new_lens must be contiguous int32 [rows]");
    STD_TORCH_CHECK(new_lens.size(0) == rows.size(0), "rows and new_lens must have the same length");
    pool.page_size = page_size;
    const int32_t device = block_tables.get_device_index();
    const ts::accelerator::DeviceGuard device_guard(device);
    ts::Tensor status = new_ints(block_tables, 1);
    raise_on_error(ipl_reserve_pages(&pool, int_ptr(rows), int_ptr(new_lens), rows.size(0), mutable_int_ptr(status),
                                     current_stream(device)));
    return status;
}

ts::Tensor fork_sequences_cuda(std::vector<ts::Tensor> caches, ts::Tensor& block_tables, ts::Tensor& seq_lens,
                               ts::Tensor& ref_counts, const ts::Tensor& parents, const ts::Tensor& children) {
    ipl_page_pool pool = page_pool(block_tables, ref_counts);
    add_rows(pool, block_tables, seq_lens, parents, "parents must be contiguous int32 [rows]");
    check_same_device(block_tables, children, "block_tables and the lists of rows must be on the same device");
    check_ints(children, 1, "children must be contiguous int32 [rows]");
    STD_TORCH_CHECK(parents.size(0) == children.size(0), "parents and children must have the same length");
    const int32_t device = block_tables.get_device_index();
    const Caches c(caches, device);
    STD_TORCH_CHECK(!caches.empty(), "caches must not be empty");
    STD_TORCH_CHECK(c.num_pages == pool.num_pages, "ref_counts must have a count for each page of the caches");
    pool.page_size = c.page_size;
    const ts::accelerator::DeviceGuard device_guard(device);
    ts::Tensor status = new_ints(block_tables, 1);
    raise_on_error(ipl_fork_sequences(&c.args, &pool, int_ptr(parents), int_ptr(children), parents.size(0),
                                      mutable_int_ptr(status), current_stream(device)));
    return status;
}

void release_sequences_cuda(ts::Tensor& block_tables, ts::Tensor& seq_lens, ts::Tensor& ref_counts,
                            const ts::Tensor& rows) {
    ipl_page_pool pool = page_pool(block_tables, ref_counts);
    add_rows(pool, block_tables, seq_lens, rows, "rows must be contiguous int32 [rows]");
    const int32_t device = block_tables.get_device_index();
    const ts::accelerator::DeviceGuard device_guard(device);
    raise_on_error(ipl_release_sequences(&pool, int_ptr(rows), rows.size(0), current_stream(device)));
}

void compact_pages_cuda(std::vector<ts::Tensor> caches, const ts::Tensor& block_tables, const ts::Tensor& ref_counts,
                        ts::Tensor& new_block_tables, ts::Tensor& new_ref_counts, ts::Tensor& live) {
    ipl_page_pool pool = page_pool(block_tables, ref_counts);
    check_same_device(block_tables, new_block_tables, "block_tables and new_block_tables must be on the same device");
    check_same_device(block_tables, new_ref_counts, "block_tables and new_ref_counts must be on the same device");
    check_same_device(block_tables, live, "block_tables and live must be on the same device");
    check_ints(new_block_tables, 2, "new_block_tables must be contiguous int32 [rows, width]");
    check_ints(new_ref_counts, 1, "new_ref_counts must be contiguous int32 [pages]");
    check_ints(live, 1, "live must be int32 [1]");
    STD_TORCH_CHECK(new_block_tables.sizes().equals(block_tables.sizes()) && new_block_tables.is_contiguous(),
                    "new_block_tables must be contiguous int32 [rows, width]");
    STD_TORCH_CHECK(new_ref_counts.size(0) == pool.num_pages && live.size(0) == 1,
                    "new_ref_counts must have a count for each page, live one element");
    const int32_t device = block_tables.get_device_index();
    const Caches c(caches, device);
    STD_TORCH_CHECK(!caches.empty(), "caches must not be empty");
    STD_TORCH_CHECK(c.num_pages == pool.num_pages, "ref_counts must have a count for each page of the caches");
    pool.page_size = c.page_size;
    const ts::accelerator::DeviceGuard device_guard(device);
    size_t bytes = 0;
    raise_on_error(ipl_compact_pages_workspace(pool.num_pages, &bytes));
    ts::Tensor workspace = new_ints(block_tables, static_cast<int64_t>(bytes / sizeof(int32_t)));
    raise_on_error(ipl_compact_pages(&c.args, &pool, mutable_int_ptr(new_block_tables), mutable_int_ptr(new_ref_counts),
                                     mutable_int_ptr(live), workspace.mutable_data_ptr(), bytes, current_stream(device)));
}

STABLE_TORCH_LIBRARY(inference_performance_lab, library) {
    library.def("fused_add_rms_norm(Tensor(a!) x, Tensor(b!) residual, Tensor weight, float epsilon) -> ()");
    library.def("silu_and_mul(Tensor(a!) output, Tensor input) -> ()");
    library.def("silu_and_mul_packed(Tensor(a!) output, Tensor input) -> ()");
    // Not in the reference library: plain RMSNorm (vLLM's _C.rms_norm argument order).
    library.def("rms_norm(Tensor(a!) output, Tensor input, Tensor weight, float epsilon) -> ()");
    // Not in the reference library: add+RMSNorm with a static fp8 output (vLLM's argument order).
    library.def(
        "fused_add_rms_norm_static_fp8_quant(Tensor(a!) result, Tensor input, Tensor(b!) residual, "
        "Tensor weight, Tensor scale, float epsilon) -> ()");
    // Not in the reference library: a paged KV cache.
    library.def(
        "rotary_embedding(Tensor positions, Tensor(a!) query, Tensor(b!) key, Tensor cos_sin_cache, bool is_neox) -> ()");
    library.def(
        "rotary_embedding_cache(Tensor positions, Tensor(a!) query, Tensor key, Tensor value, Tensor cos_sin_cache, "
        "Tensor(b!) key_cache, Tensor(c!) value_cache, Tensor slot_mapping, bool is_neox) -> ()");
    library.def(
        "paged_attention(Tensor(a!) output, Tensor query, Tensor key_cache, Tensor value_cache, Tensor block_tables, "
        "Tensor query_start_loc, Tensor seq_lens, int max_query_len, int max_seq_len, float scale, int window) -> ()");
    library.def("copy_pages(Tensor(a!)[] caches, Tensor pairs) -> ()");
    library.def(
        "reserve_pages(Tensor(a!) block_tables, Tensor(b!) seq_lens, Tensor(c!) ref_counts, Tensor rows, "
        "Tensor new_lens, int page_size) -> Tensor");
    library.def(
        "fork_sequences(Tensor(a!)[] caches, Tensor(b!) block_tables, Tensor(c!) seq_lens, Tensor(d!) ref_counts, "
        "Tensor parents, Tensor children) -> Tensor");
    library.def(
        "release_sequences(Tensor(a!) block_tables, Tensor(b!) seq_lens, Tensor(c!) ref_counts, Tensor rows) -> ()");
    library.def(
        "compact_pages(Tensor(a!)[] caches, Tensor block_tables, Tensor ref_counts, Tensor(b!) new_block_tables, "
        "Tensor(c!) new_ref_counts, Tensor(d!) live) -> ()");
}

STABLE_TORCH_LIBRARY_IMPL(inference_performance_lab, CUDA, library) {
    library.impl("fused_add_rms_norm", TORCH_BOX(&fused_add_rms_norm_cuda));
    library.impl("silu_and_mul", TORCH_BOX(&silu_and_mul_cuda));
    library.impl("silu_and_mul_packed", TORCH_BOX(&silu_and_mul_packed_cuda));
    library.impl("rms_norm", TORCH_BOX(&rms_norm_cuda));
    library.impl("fused_add_rms_norm_static_fp8_quant", TORCH_BOX(&fused_add_rms_norm_static_fp8_quant_cuda));
    library.impl("rotary_embedding", TORCH_BOX(&rotary_embedding_cuda));
    library.impl("rotary_embedding_cache", TORCH_BOX(&rotary_embedding_cache_cuda));
    library.impl("paged_attention", TORCH_BOX(&paged_attention_cuda));
    library.impl("copy_pages", TORCH_BOX(&copy_pages_cuda));
    library.impl("reserve_pages", TORCH_BOX(&reserve_pages_cuda));
    library.impl("fork_sequences", TORCH_BOX(&fork_sequences_cuda));
    library.impl("release_sequences", TORCH_BOX(&release_sequences_cuda));
    library.impl("compact_pages", TORCH_BOX(&compact_pages_cuda));
}
