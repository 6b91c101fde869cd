// Host side of the paged-cache entry points of ipl_b200.h: argument checks, kernel selection, launch.
#pragma once

#include "cache_pages.cuh"
#include "ipl_host.cuh"
#include "paged_attention.cuh"
#include "paged_attention_short.cuh"
#include "paged_attention_tile.cuh"
#include "rotary.cuh"

namespace ipl {
namespace {

int64_t round_up(int64_t value, int64_t multiple) { return (value + multiple - 1) / multiple * multiple; }

bool aligned(const void* p, uintptr_t bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }

ipl_status launch_status(cudaError_t err, const char* what) {
    if (err == cudaSuccess) return IPL_SUCCESS;
    return fail(IPL_ERROR_CUDA, "%s kernel launch failed: %s", what, cudaGetErrorString(err));
}

// ------------------------------------------------------------------------------------------
// rotary positions

ipl_status check_rotary_args(const ipl_rotary_args* a, bool append) {
    if (a == nullptr) return fail(IPL_ERROR_INVALID_VALUE, "args must be non-null");
    if (a->num_tokens < 0) return fail(IPL_ERROR_INVALID_VALUE, "number of tokens must be non-negative");
    if (a->num_heads < 1 || a->num_kv_heads < 1 || a->head_size < 1) {
        return fail(IPL_ERROR_INVALID_VALUE, "number of heads and head size must be positive");
    }
    if (a->rotary_dim < 2 || a->rotary_dim % 2 != 0 || a->rotary_dim > a->head_size) {
        return fail(IPL_ERROR_INVALID_VALUE, "rotary dimension must be even, positive and at most the head size");
    }
    if (a->max_position < 1) return fail(IPL_ERROR_INVALID_VALUE, "cos_sin_cache must have at least one position");
    if (a->num_tokens > INT_MAX) return fail(IPL_ERROR_TOO_LARGE, "number of tokens is too large");
    if (a->num_heads > 65536 || a->num_kv_heads > 65536 || a->head_size > 4096) {
        return fail(IPL_ERROR_TOO_LARGE, "number of heads or head size is too large");
    }
    if (append) {
        if (a->page_size < 1 || a->num_pages < 0) {
            return fail(IPL_ERROR_INVALID_VALUE, "page size must be positive and number of pages non-negative");
        }
        if (a->page_size > INT_MAX || a->num_pages > INT_MAX / a->page_size) {
            return fail(IPL_ERROR_TOO_LARGE, "the cache holds too many slots");
        }
    }
    if (a->num_tokens == 0) return IPL_SUCCESS;
    if (a->positions == nullptr || a->cos_sin_cache == nullptr || a->query == nullptr || a->key == nullptr) {
        return fail(IPL_ERROR_INVALID_VALUE, "positions, query, key and cos_sin_cache must be non-null");
    }
    if (append && (a->value == nullptr || a->slot_mapping == nullptr ||
                   (a->num_pages > 0 && (a->key_cache == nullptr || a->value_cache == nullptr)))) {
        return fail(IPL_ERROR_INVALID_VALUE, "value, key_cache, value_cache and slot_mapping must be non-null");
    }
    if (!aligned(a->positions, 8) || !aligned(a->cos_sin_cache, 4) || (append && !aligned(a->slot_mapping, 8))) {
        return fail(IPL_ERROR_INVALID_VALUE, "positions, slot_mapping and cos_sin_cache must be aligned to their types");
    }
    if (!aligned(a->query, 2) || !aligned(a->key, 2) ||
        (append && !(aligned(a->value, 2) && aligned(a->key_cache, 2) && aligned(a->value_cache, 2)))) {
        return fail(IPL_ERROR_INVALID_VALUE, "bfloat16 pointers must be 2-byte aligned");
    }
    return IPL_SUCCESS;
}

// Whether every 16-byte chunk of the call is 16-byte aligned and holds whole pairs' halves.
bool rotary_vectorises(const ipl_rotary_args& a, bool append) {
    int64_t strides = a.query_token_stride | a.query_head_stride | a.key_token_stride | a.key_head_stride;
    bool pointers = aligned(a.query, 16) && aligned(a.key, 16) && aligned(a.cos_sin_cache, 16);
    if (append) {
        strides |= a.value_token_stride | a.value_head_stride | a.key_cache_page_stride | a.key_cache_token_stride |
                   a.key_cache_head_stride | a.value_cache_page_stride | a.value_cache_token_stride |
                   a.value_cache_head_stride | a.head_size;
        pointers = pointers && aligned(a.value, 16) && aligned(a.key_cache, 16) && aligned(a.value_cache, 16);
    }
    return pointers && strides % 8 == 0 && a.rotary_dim % (a.is_neox ? 16 : 8) == 0;
}

template <bool kAppend>
ipl_status run_rotary(const ipl_rotary_args* a, cudaStream_t stream) {
    const ipl_status st = check_rotary_args(a, kAppend);
    if (st != IPL_SUCCESS || a->num_tokens == 0) return st;
    int device = 0;
    DeviceInfo* info = nullptr;
    const ipl_status found = current_device(&device, &info);
    if (found != IPL_SUCCESS) return found;
    const bool vector = rotary_vectorises(*a, kAppend);
    RotaryParams p = {};
    p.positions = a->positions;
    p.cos_sin = a->cos_sin_cache;
    p.max_position = a->max_position;
    p.rot = static_cast<int>(a->rotary_dim);
    p.tokens = static_cast<uint32_t>(a->num_tokens);
    p.q = static_cast<uint16_t*>(a->query);
    p.k = static_cast<uint16_t*>(a->key);
    p.q_token = a->query_token_stride, p.q_head = a->query_head_stride;
    p.k_token = a->key_token_stride, p.k_head = a->key_head_stride;
    p.q_heads = static_cast<uint32_t>(a->num_heads);
    const uint32_t kv_heads = static_cast<uint32_t>(a->num_kv_heads);
    const int64_t chunks = !vector ? a->rotary_dim / 2 : a->is_neox ? a->rotary_dim / 16 : a->rotary_dim / 8;
    const int64_t pass = (a->head_size - a->rotary_dim) / (vector ? 8 : 1);
    const int64_t v_chunks = a->head_size / (vector ? 8 : 1);
    p.rotated_items = (p.q_heads + kv_heads) * static_cast<uint32_t>(chunks);
    p.items = p.rotated_items;
    p.rot_chunks = make_fast_div32(static_cast<uint32_t>(chunks));
    if (kAppend) {
        p.v = static_cast<const uint16_t*>(a->value);
        p.slots = a->slot_mapping;
        p.num_slots = a->num_pages * a->page_size;
        p.page_size = make_fast_div32(static_cast<uint32_t>(a->page_size));
        p.key_cache = static_cast<uint16_t*>(a->key_cache);
        p.value_cache = static_cast<uint16_t*>(a->value_cache);
        p.v_token = a->value_token_stride, p.v_head = a->value_head_stride;
        p.key_page = a->key_cache_page_stride, p.key_token = a->key_cache_token_stride;
        p.key_head = a->key_cache_head_stride;
        p.value_page = a->value_cache_page_stride, p.value_token = a->value_cache_token_stride;
        p.value_head = a->value_cache_head_stride;
        p.passed_items = kv_heads * static_cast<uint32_t>(pass);
        p.pass_chunks = make_fast_div32(static_cast<uint32_t>(pass > 0 ? pass : 1));
        p.v_chunks = make_fast_div32(static_cast<uint32_t>(v_chunks));
        p.items += p.passed_items + kv_heads * static_cast<uint32_t>(v_chunks);
    }
    p.items_div = make_fast_div32(p.items);
    // CTAs of 128 threads once the items are more than about four times the threads the GPU holds.
    const bool large = a->num_tokens * p.items > 4 * int64_t{kThreadsPerSm} * info->sm_count.load(std::memory_order_relaxed);
    uint32_t threads = large ? 128 : 256;
    if (!large && p.items > threads) threads = p.items < kRotaryMaxThreads ? (p.items + 31) / 32 * 32 : kRotaryMaxThreads;
    p.tokens_per_cta = p.items < threads ? threads / p.items : 1;
    const unsigned grid = (p.tokens + p.tokens_per_cta - 1) / p.tokens_per_cta;
    cudaError_t err;
    if (vector) {
        err = a->is_neox ? launch(rotary_kernel<true, true, kAppend>, grid, threads, 0, stream, p)
                         : launch(rotary_kernel<true, false, kAppend>, grid, threads, 0, stream, p);
    } else {
        err = a->is_neox ? launch(rotary_kernel<false, true, kAppend>, grid, threads, 0, stream, p)
                         : launch(rotary_kernel<false, false, kAppend>, grid, threads, 0, stream, p);
    }
    return launch_status(err, "rotary embedding");
}

// ------------------------------------------------------------------------------------------
// attention

ipl_status check_attention_args(const ipl_paged_attention_args* a) {
    if (a == nullptr) return fail(IPL_ERROR_INVALID_VALUE, "args must be non-null");
    if (a->num_tokens < 0 || a->num_seqs < 0 || a->num_pages < 0 || a->table_width < 0) {
        return fail(IPL_ERROR_INVALID_VALUE, "sizes must be non-negative");
    }
    if (a->num_heads < 1 || a->num_kv_heads < 1 || a->head_size < 1 || a->page_size < 1) {
        return fail(IPL_ERROR_INVALID_VALUE, "number of heads, head size and page size must be positive");
    }
    if (a->num_heads % a->num_kv_heads != 0) {
        return fail(IPL_ERROR_INVALID_VALUE, "number of query heads must be a multiple of the number of key heads");
    }
    if (a->max_query_len < 0 || a->max_seq_len < 0 || a->window < 0) {
        return fail(IPL_ERROR_INVALID_VALUE, "max_query_len, max_seq_len and window must be non-negative");
    }
    if (!(a->scale > 0.0) || a->scale > 1e30) return fail(IPL_ERROR_INVALID_VALUE, "scale must be positive and finite");
    if (a->head_size > kAttentionMaxDim) {
        return fail(IPL_ERROR_TOO_LARGE, "head size must be at most %d", kAttentionMaxDim);
    }
    if (a->num_tokens > INT_MAX / 2 || a->num_seqs > INT_MAX / 2 || a->num_heads > 65536 || a->num_pages > INT_MAX ||
        a->page_size > INT_MAX || a->table_width > INT_MAX || a->max_seq_len > INT_MAX / 2 ||
        a->num_tokens > INT64_MAX / 65536 / 256 || a->num_tokens * a->num_heads > INT64_C(4) * INT_MAX) {
        return fail(IPL_ERROR_TOO_LARGE, "a size is too large");
    }
    if (a->num_tokens == 0 || a->num_seqs == 0) return IPL_SUCCESS;
    if (a->output == nullptr || a->query == nullptr || a->block_tables == nullptr || a->query_start_loc == nullptr ||
        a->seq_lens == nullptr || (a->num_pages > 0 && (a->key_cache == nullptr || a->value_cache == nullptr))) {
        return fail(IPL_ERROR_INVALID_VALUE,
                    "output, query, key_cache, value_cache, block_tables, query_start_loc and seq_lens must be non-null");
    }
    if (!aligned(a->output, 2) || !aligned(a->query, 2) || !aligned(a->key_cache, 2) || !aligned(a->value_cache, 2)) {
        return fail(IPL_ERROR_INVALID_VALUE, "bfloat16 pointers must be 2-byte aligned");
    }
    if (!aligned(a->block_tables, 4) || !aligned(a->query_start_loc, 4) || !aligned(a->seq_lens, 4)) {
        return fail(IPL_ERROR_INVALID_VALUE, "int32 pointers must be 4-byte aligned");
    }
    return IPL_SUCCESS;
}

AttentionParams attention_params(const ipl_paged_attention_args& a) {
    AttentionParams p = {};
    p.out = static_cast<uint16_t*>(a.output);
    p.q = static_cast<const uint16_t*>(a.query);
    p.key_cache = static_cast<const uint16_t*>(a.key_cache);
    p.value_cache = static_cast<const uint16_t*>(a.value_cache);
    p.tables = a.block_tables;
    p.starts = a.query_start_loc;
    p.lens = a.seq_lens;
    p.num_tokens = static_cast<int>(a.num_tokens);
    p.num_seqs = static_cast<int>(a.num_seqs);
    p.heads = static_cast<int>(a.num_heads);
    p.kv_heads = static_cast<int>(a.num_kv_heads);
    p.group = p.heads / p.kv_heads;
    p.dim = static_cast<int>(a.head_size);
    p.page_size = static_cast<int>(a.page_size);
    p.num_pages = static_cast<int>(a.num_pages);
    p.table_width = static_cast<int>(a.table_width);
    p.window = a.window > 0 && a.window < INT_MAX ? static_cast<int>(a.window) : INT_MAX;
    p.table_row = a.table_stride;
    p.out_token = a.output_token_stride, p.out_head = a.output_head_stride;
    p.q_token = a.query_token_stride, p.q_head = a.query_head_stride;
    p.key_page = a.key_cache_page_stride, p.key_token = a.key_cache_token_stride, p.key_head = a.key_cache_head_stride;
    p.value_page = a.value_cache_page_stride, p.value_token = a.value_cache_token_stride;
    p.value_head = a.value_cache_head_stride;
    p.scale_log2 = static_cast<float>(a.scale * 1.4426950408889634);
    p.page_blocks = make_fast_div32(static_cast<uint32_t>(p.page_size >= kAttentionBlock ? p.page_size / kAttentionBlock : 1));
    p.group_div = make_fast_div32(static_cast<uint32_t>(p.group));
    return p;
}

// cuTensorMapEncodeTiled, from the driver the runtime has loaded (the library links no libcuda).
using EncodeTensorMap = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                     const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                     CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeTensorMap encode_tensor_map() {
    static const EncodeTensorMap encode = [] {
        void* f = nullptr;
        cudaDriverEntryPointQueryResult found = cudaDriverEntryPointSymbolNotFound;
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &f, 12000, cudaEnableDefault, &found) != cudaSuccess ||
            found != cudaDriverEntryPointSuccess) {
            (void)cudaGetLastError();
            f = nullptr;
        }
        return reinterpret_cast<EncodeTensorMap>(f);
    }();
    return encode;
}

// Map of bf16 elements, boxes of 64 elements in 128-byte swizzled rows; places outside read as 0.
// strides in elements, of the dimensions after the first.
ipl_status make_tensor_map(CUtensorMap* map, const void* base, int rank, const int64_t* sizes, const int64_t* strides,
                           const int* box) {
    const EncodeTensorMap encode = encode_tensor_map();
    if (encode == nullptr) return fail(IPL_ERROR_CUDA, "the CUDA driver has no cuTensorMapEncodeTiled");
    cuuint64_t dims[4], bytes[3];
    cuuint32_t boxes[4], steps[4];
    for (int i = 0; i < rank; ++i) {
        dims[i] = static_cast<cuuint64_t>(sizes[i]);
        boxes[i] = static_cast<cuuint32_t>(box[i]);
        steps[i] = 1;
        if (i > 0) bytes[i - 1] = static_cast<cuuint64_t>(strides[i - 1]) * 2;
    }
    const CUresult err = encode(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, static_cast<cuuint32_t>(rank), const_cast<void*>(base),
                                dims, bytes, boxes, steps, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                                CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (err != CUDA_SUCCESS) return fail(IPL_ERROR_CUDA, "cuTensorMapEncodeTiled failed: error %d", static_cast<int>(err));
    return IPL_SUCCESS;
}

// Which kernels a call runs, a pure function of its sizes, strides, alignment and the SM count.
struct AttentionPlan {
    bool vector = false;  // the short and tile kernels; else a warp per row
    int dim = 0;          // head size padded to 64 or 128
    bool tile = false;    // the tile kernel takes the sequences of more than short_rows rows
    int short_rows = 0;
    int tiles = 0;        // short kernels: column tiles of 8 rows; 0: not launched
    int cluster = 0;      // CTAs a sequence, key head and row tile of the short kernel; 0: the shared kernel
    int row_tiles = 1;
    int tile_ctas = 0, shared_ctas = 0;
    size_t tile_workspace = 0, workspace = 0;  // the tile kernel's at the beginning
};

// 16-byte chunks of every row, and 16 keys of a block in one page.
bool attention_vectorises(const ipl_paged_attention_args& a) {
    const int64_t strides = a.output_token_stride | a.output_head_stride | a.query_token_stride | a.query_head_stride |
                            a.key_cache_page_stride | a.key_cache_token_stride | a.key_cache_head_stride |
                            a.value_cache_page_stride | a.value_cache_token_stride | a.value_cache_head_stride;
    return a.head_size % 8 == 0 && a.head_size <= 128 && a.page_size % kAttentionBlock == 0 && strides % 8 == 0 &&
           aligned(a.output, 16) && aligned(a.query, 16) && aligned(a.key_cache, 16) && aligned(a.value_cache, 16);
}

// Workspace of the parts that `ctas` CTAs leave.
size_t parts_bytes(int64_t ctas, int64_t slot_rows, int64_t dim) {
    return static_cast<size_t>(round_up(2 * ctas * (slot_rows * (dim * 4 + 8) + static_cast<int64_t>(sizeof(AttentionPart))), 16));
}
AttentionParts attention_parts(void* workspace, int64_t ctas, int slot_rows, int64_t dim, int tile_rows, int tile_tokens) {
    AttentionParts parts;
    float* const base = static_cast<float*>(workspace);
    // The tile kernel stores sums 32 bytes at once, a workspace lies on 16: the sums begin at the next 32 bytes. They
    // end 16 bytes late then, in the last slot's, which nothing is written to: no CTA comes after the last one.
    parts.sums = aligned(base, 32) ? base : base + 4;
    parts.stats = reinterpret_cast<float2*>(base + 2 * ctas * slot_rows * dim);
    parts.parts = reinterpret_cast<AttentionPart*>(parts.stats + 2 * ctas * slot_rows);
    parts.slot_rows = slot_rows;
    parts.tile_rows = tile_rows;
    parts.tile_tokens = tile_tokens;
    return parts;
}

// Turns of a CTA of the short kernel over `keys` keys, a block a warp.
int64_t key_turns(int64_t keys) { return (keys + kShortWarps * kAttentionBlock - 1) / (kShortWarps * kAttentionBlock); }

// CTAs of the short kernel that the GPU holds in clusters of this size: a cluster stays within a part of the GPU,
// which leaves some SMs out (72 clusters of 4 and 36 of 8 took a second wave on 296 places, 116 of 2 did not).
int64_t short_resident(int sm_count, int cluster) {
    const int64_t places = static_cast<int64_t>(sm_count) * kShortCtas;
    return cluster == 1 ? places : cluster <= 4 ? places * 7 / 8 : places * 3 / 4;
}

// CTAs a cluster: as many as the GPU holds of all of them, up to one for each turn.
int short_cluster(int64_t units, int64_t keys, int sm_count) {
    int cluster = 1;
    while (cluster < kShortCluster && cluster < key_turns(keys) && units * cluster * 2 <= short_resident(sm_count, cluster * 2)) {
        cluster *= 2;
    }
    return cluster;
}

// Estimates of the two kernels' times in ns, within a fifth of those measured at 1-256 tokens a sequence, 1-148
// sequences and 36-8192 keys, all of one layout: 28 and 4 heads of 128. Others go by the same constants.
int64_t short_time(int64_t units, int64_t keys, int sm_count, int cluster) {
    const int64_t held = short_resident(sm_count, cluster), waves = (units * cluster + held - 1) / held;
    return 3000 + waves * (2500 + 1300 * ((key_turns(keys) + cluster - 1) / cluster));
}
int64_t tile_time(int64_t pairs, int64_t keys, int sm_count) {
    return 16000 + 1900 * (pairs * (keys / kTileKeys + 2) / sm_count);
}

constexpr int kMostRowTiles = 4096;

AttentionPlan plan_attention(const ipl_paged_attention_args& a, int sm_count) {
    AttentionPlan plan;
    if (!attention_vectorises(a)) return plan;
    plan.vector = true;
    plan.dim = a.head_size <= 64 ? 64 : 128;
    const int64_t group = a.num_heads / a.num_kv_heads;
    // The bounds may be any numbers; beyond the tokens there are, and for a window beyond the keys, they bound nothing.
    const int64_t most_new = a.max_query_len < a.num_tokens ? a.max_query_len : a.num_tokens;
    const int64_t rows = most_new * group;
    plan.tiles = rows <= 8 ? 1 : 2;
    plan.short_rows = INT_MAX;
    int64_t keys = a.max_seq_len > 1 ? a.max_seq_len : 1;
    if (a.window > 0 && a.window < keys && a.window + most_new < keys) keys = a.window + most_new;
    // TMA takes strides of up to 2^40 bytes and no zero ones.
    const int64_t strides[] = {a.query_token_stride, a.query_head_stride, a.key_cache_page_stride, a.key_cache_token_stride,
                               a.key_cache_head_stride, a.value_cache_page_stride, a.value_cache_token_stride, a.value_cache_head_stride};
    bool mappable = a.num_pages > 0;
    for (const int64_t s : strides) mappable = mappable && s > 0 && s < (INT64_C(1) << 38);
    if (rows > 16) {
        // Small calls stay with the short kernel, its row tiles side by side.
        const int64_t most = (rows + 15) / 16, tiles = a.num_tokens * group / 16 + a.num_seqs;
        const int64_t units = (tiles < most * a.num_seqs ? tiles : most * a.num_seqs) * a.num_kv_heads;
        const int64_t pairs = (a.num_tokens * group / (2 * kTileRows) + a.num_seqs) * a.num_kv_heads;
        if (group <= kTileRows && mappable && short_time(units, keys, sm_count, short_cluster(units, keys, sm_count)) > tile_time(pairs, keys, sm_count)) {
            plan.tile = true;
            plan.tiles = group <= 8 ? 1 : 2;
            plan.short_rows = plan.tiles * 8;
            // Sequences of one length have no short one among them.
            if (group > 16 || a.num_tokens == most_new * a.num_seqs) {
                plan.tiles = 0;
                plan.short_rows = 0;
            }
        } else {
            plan.row_tiles = static_cast<int>(most < kMostRowTiles ? most : kMostRowTiles);
        }
    }
    // The short kernels count a sequence's rows, and a turn of its row tiles past them, in 32 bits.
    if (!plan.tile && a.num_tokens * group > INT_MAX - 16 * kMostRowTiles) return AttentionPlan{};
    if (plan.tile) {
        plan.tile_ctas = sm_count;
        plan.tile_workspace = parts_bytes(plan.tile_ctas, 2 * kTileRows, plan.dim);
        plan.workspace = plan.tile_workspace;
    }
    if (plan.tiles > 0) {
        // A cluster for each sequence, key head and row tile where the GPU holds all of them and no warp has more
        // than 16 blocks of keys; otherwise equal shares (row tiles: clusters all the same, they are not cut). Those
        // are cut from a sum of blocks in 32 bits, which the tables' width bounds.
        const int64_t longest = a.table_width < INT_MAX / a.page_size ? a.table_width * a.page_size : INT_MAX;
        const bool countable = a.num_seqs <= INT_MAX / (longest / kAttentionBlock + 1 + kShortPairCost);
        const int64_t units = a.num_seqs * a.num_kv_heads * plan.row_tiles;
        const int64_t resident = static_cast<int64_t>(sm_count) * shared_ctas(plan.tiles);
        plan.cluster = short_cluster(units, keys, sm_count);
        if (plan.row_tiles == 1 && countable && (units * plan.cluster > resident || key_turns(keys) > 16 * plan.cluster)) {
            plan.cluster = 0;
            plan.shared_ctas = static_cast<int>(resident);
            plan.workspace += parts_bytes(plan.shared_ctas, 8 * plan.tiles, plan.dim);
        }
    }
    return plan;
}

template <int kDim>
ipl_status launch_short(const AttentionPlan& plan, const AttentionParams& p, char* workspace, DeviceInfo* info, cudaStream_t stream) {
    if (plan.cluster > 0) {
        const uint32_t bit = 1u << (kDim == 64 ? 28 : 29);
        if (plan.cluster > 8 && !(info->smem_configured.load(std::memory_order_acquire) & bit)) {
            cudaError_t err = cudaFuncSetAttribute(attention_short_kernel<kDim, 1>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
            if (err == cudaSuccess) {
                err = cudaFuncSetAttribute(attention_short_kernel<kDim, 2>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
            }
            if (err != cudaSuccess) return fail(IPL_ERROR_CUDA, "paged attention kernel setup failed: %s", cudaGetErrorString(err));
            info->smem_configured.fetch_or(bit, std::memory_order_acq_rel);
        }
        const int64_t ctas = static_cast<int64_t>(p.num_seqs) * p.kv_heads * plan.row_tiles * plan.cluster;
        if (ctas > INT_MAX) return fail(IPL_ERROR_TOO_LARGE, "too many sequences and heads");
        const unsigned cluster = static_cast<unsigned>(plan.cluster), grid = static_cast<unsigned>(ctas);
        return launch_status(
            plan.tiles == 1 ? launch_clustered(attention_short_kernel<kDim, 1>, grid, cluster, kShortThreads, 0, stream, p)
                            : launch_clustered(attention_short_kernel<kDim, 2>, grid, cluster, kShortThreads, 0, stream, p),
            "paged attention");
    }
    const AttentionParts parts = attention_parts(workspace, plan.shared_ctas, 8 * plan.tiles, kDim, 8 * plan.tiles, 8 * plan.tiles);
    const unsigned grid = static_cast<unsigned>(plan.shared_ctas);
    const ipl_status st = launch_status(
        plan.tiles == 1 ? launch(attention_shared_kernel<kDim, 1>, grid, kShortThreads, 0, stream, p, parts)
                        : launch(attention_shared_kernel<kDim, 2>, grid, kShortThreads, 0, stream, p, parts),
        "paged attention");
    if (st != IPL_SUCCESS) return st;
    return launch_status(launch_2d(attention_join_parts_kernel<kDim>, grid, 4u * plan.tiles, 2 * kJoinSplit * kWarpSize, stream, p, parts),
                         "paged attention");
}

template <int kDim>
ipl_status launch_tile(const ipl_paged_attention_args& a, const AttentionPlan& plan, const AttentionParams& p,
                       DeviceInfo* info, cudaStream_t stream) {
    using Layout = TileLayout<kDim>;
    const uint32_t bit = 1u << (kDim == 64 ? 30 : 31);
    if (!(info->smem_configured.load(std::memory_order_acquire) & bit)) {
        const cudaError_t err = cudaFuncSetAttribute(attention_tile_kernel<kDim>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                     static_cast<int>(Layout::kDynamic));
        if (err != cudaSuccess) return fail(IPL_ERROR_CUDA, "paged attention kernel setup failed: %s", cudaGetErrorString(err));
        info->smem_configured.fetch_or(bit, std::memory_order_acq_rel);
    }
    TileParams t;
    t.a = p;
    t.tile_tokens = kTileRows / p.group;
    t.box_keys = kAttentionBlock;
    while (t.box_keys < kTileKeys && p.page_size % (2 * t.box_keys) == 0) t.box_keys *= 2;
    t.units = p.num_tokens / (2 * t.tile_tokens) + p.num_seqs;
    t.pair_tokens = make_fast_div32(static_cast<uint32_t>(2 * t.tile_tokens));
    t.page_size = make_fast_div32(static_cast<uint32_t>(p.page_size));
    t.group_reciprocal = 65536 / p.group + 1;
    t.wide_out = p.dim % 16 == 0 && (p.out_token | p.out_head) % 16 == 0 && aligned(p.out, 32);
    t.parts = attention_parts(a.workspace, plan.tile_ctas, 2 * kTileRows, kDim, kTileRows, t.tile_tokens);
    CUtensorMap q, k, v;
    const int64_t q_sizes[3] = {p.dim, p.heads, p.num_tokens}, q_strides[2] = {p.q_head, p.q_token};
    const int q_box[3] = {64, p.group, t.tile_tokens};
    ipl_status st = make_tensor_map(&q, a.query, 3, q_sizes, q_strides, q_box);
    const int64_t sizes[4] = {p.dim, p.kv_heads, p.page_size, p.num_pages};
    const int box[4] = {64, 1, t.box_keys, 1};
    const int64_t k_strides[3] = {p.key_head, p.key_token, p.key_page};
    const int64_t v_strides[3] = {p.value_head, p.value_token, p.value_page};
    if (st == IPL_SUCCESS) st = make_tensor_map(&k, a.key_cache, 4, sizes, k_strides, box);
    if (st == IPL_SUCCESS) st = make_tensor_map(&v, a.value_cache, 4, sizes, v_strides, box);
    if (st != IPL_SUCCESS) return st;
    const unsigned ctas = static_cast<unsigned>(plan.tile_ctas);
    st = launch_status(launch(attention_tile_kernel<kDim>, ctas, kTileThreads, Layout::kDynamic, stream, t, q, k, v),
                       "paged attention");
    if (st != IPL_SUCCESS) return st;
    // Parts a pair, on average at least.
    const bool split = ctas > 4 * static_cast<int64_t>(t.units) * p.kv_heads;
    const unsigned blocks = 2 * kTileRows / kJoinRows;
    return launch_status(split ? launch_2d(attention_join_rows_kernel<kDim, true>, ctas, blocks, kJoinWarps * kWarpSize, stream, p, t.parts)
                               : launch_2d(attention_join_rows_kernel<kDim, false>, ctas, blocks / kJoinWarps, kJoinWarps * kWarpSize,
                                           stream, p, t.parts),
                         "paged attention");
}

template <int kDim>
ipl_status launch_attention(const ipl_paged_attention_args& a, const AttentionPlan& plan, const AttentionParams& p,
                            DeviceInfo* info, cudaStream_t stream) {
    ipl_status st = IPL_SUCCESS;
    if (plan.tile) st = launch_tile<kDim>(a, plan, p, info, stream);
    if (st == IPL_SUCCESS && plan.tiles > 0) st = launch_short<kDim>(plan, p, static_cast<char*>(a.workspace) + plan.tile_workspace, info, stream);
    return st;
}

ipl_status run_attention(const ipl_paged_attention_args* a, cudaStream_t stream) {
    ipl_status st = check_attention_args(a);
    if (st != IPL_SUCCESS || a->num_tokens == 0 || a->num_seqs == 0) return st;
    int device = 0;
    DeviceInfo* info = nullptr;
    st = current_device(&device, &info);
    if (st != IPL_SUCCESS) return st;
    const AttentionPlan plan = plan_attention(*a, info->sm_count.load(std::memory_order_relaxed));
    AttentionParams p = attention_params(*a);
    if (!plan.vector) {
        const int64_t rows = a->num_tokens * a->num_heads;
        const unsigned grid = static_cast<unsigned>((rows + kAttentionRowWarps - 1) / kAttentionRowWarps);
        return launch_status(launch(attention_row_kernel, grid, kAttentionRowWarps * kWarpSize, 0, stream, p), "paged attention");
    }
    if (a->workspace_bytes < plan.workspace) return fail(IPL_ERROR_INVALID_VALUE, "workspace is too small");
    if (plan.workspace > 0 && (a->workspace == nullptr || !aligned(a->workspace, 16))) {
        return fail(IPL_ERROR_INVALID_VALUE, "workspace must be non-null and 16-byte aligned");
    }
    p.short_rows = plan.short_rows;
    p.row_tiles = plan.row_tiles;
    return plan.dim == 64 ? launch_attention<64>(*a, plan, p, info, stream) : launch_attention<128>(*a, plan, p, info, stream);
}

// ------------------------------------------------------------------------------------------
// pages

ipl_status check_pool(const ipl_page_pool* pool) {
    if (pool == nullptr) return fail(IPL_ERROR_INVALID_VALUE, "pool must be non-null");
    if (pool->num_rows < 0 || pool->width < 0 || pool->num_pages < 0 || pool->page_size < 1) {
        return fail(IPL_ERROR_INVALID_VALUE, "sizes of the pool must be non-negative and its page size positive");
    }
    if (pool->num_rows > INT_MAX || pool->width > INT_MAX || pool->num_pages > INT_MAX / 2 || pool->page_size > INT_MAX) {
        return fail(IPL_ERROR_TOO_LARGE, "a size of the pool is too large");
    }
    if ((pool->num_rows > 0 && pool->width > 0 && pool->block_tables == nullptr) ||
        (pool->num_pages > 0 && pool->ref_counts == nullptr)) {
        return fail(IPL_ERROR_INVALID_VALUE, "block_tables and ref_counts must be non-null");
    }
    if (!aligned(pool->block_tables, 4) || !aligned(pool->seq_lens, 4) || !aligned(pool->ref_counts, 4)) {
        return fail(IPL_ERROR_INVALID_VALUE, "int32 pointers must be 4-byte aligned");
    }
    return IPL_SUCCESS;
}

ipl_status check_rows(const ipl_page_pool* pool, const void* rows, const void* other, int64_t count) {
    if (count < 0) return fail(IPL_ERROR_INVALID_VALUE, "number of rows must be non-negative");
    if (count > INT_MAX / 2) return fail(IPL_ERROR_TOO_LARGE, "number of rows is too large");
    if (count > 0 && (rows == nullptr || other == nullptr)) {
        return fail(IPL_ERROR_INVALID_VALUE, "the lists of rows must be non-null");
    }
    if (pool->num_rows > 0 && pool->seq_lens == nullptr) {
        return fail(IPL_ERROR_INVALID_VALUE, "seq_lens must be non-null");
    }
    if (!aligned(rows, 4) || !aligned(other, 4)) return fail(IPL_ERROR_INVALID_VALUE, "int32 pointers must be 4-byte aligned");
    return IPL_SUCCESS;
}

ipl_status check_caches(const ipl_page_caches* c) {
    if (c == nullptr) return fail(IPL_ERROR_INVALID_VALUE, "caches must be non-null");
    if (c->num_caches < 0 || c->page_bytes < 0 || c->page_stride_bytes < c->page_bytes) {
        return fail(IPL_ERROR_INVALID_VALUE, "sizes of the caches must be non-negative and pages must not overlap");
    }
    if (c->num_caches > 65536) return fail(IPL_ERROR_TOO_LARGE, "too many caches");
    if (c->num_caches > 0 && c->caches == nullptr) return fail(IPL_ERROR_INVALID_VALUE, "caches must be non-null");
    bool ok = (c->page_bytes | c->page_stride_bytes) % 16 == 0;
    for (int64_t i = 0; i < c->num_caches; ++i) {
        if (c->caches[i] == nullptr && c->page_bytes > 0) return fail(IPL_ERROR_INVALID_VALUE, "caches must be non-null");
        ok = ok && aligned(c->caches[i], 16);
    }
    if (!ok) return fail(IPL_ERROR_MISALIGNED, "pages must be 16-byte aligned multiples of 16 bytes");
    return IPL_SUCCESS;
}

PageState page_state(const ipl_page_pool& pool) {
    PageState s;
    s.tables = pool.block_tables;
    s.table_row = pool.table_stride;
    s.lens = pool.seq_lens;
    s.ref_counts = pool.ref_counts;
    s.num_rows = static_cast<int>(pool.num_rows);
    s.width = static_cast<int>(pool.width);
    s.num_pages = static_cast<int>(pool.num_pages);
    s.page_size = static_cast<int>(pool.page_size);
    return s;
}

PageLayout page_layout(const ipl_page_caches& c) {
    PageLayout page = {c.page_stride_bytes, c.page_bytes, (c.page_stride_bytes | c.page_bytes) % 32 == 0};
    for (int64_t i = 0; i < c.num_caches; ++i) page.wide = page.wide && aligned(c.caches[i], 32);
    return page;
}

// The caches from number `from` on, as many as one launch takes.
int cache_list(const ipl_page_caches& c, int64_t from, CacheList* list) {
    int n = 0;
    for (; n < kMaxCachesPerLaunch && from + n < c.num_caches; ++n) list->cache[n] = static_cast<char*>(c.caches[from + n]);
    return n;
}

// Workspace of a compaction: three lists of num_pages, then a count.
size_t compact_workspace_bytes(int64_t num_pages) { return static_cast<size_t>(3 * num_pages + 1) * sizeof(int32_t); }

ipl_status check_claim(const ipl_page_pool* pool, const void* rows, const void* other, int64_t count, const int32_t* status) {
    ipl_status st = check_pool(pool);
    if (st == IPL_SUCCESS) st = check_rows(pool, rows, other, count);
    if (st != IPL_SUCCESS) return st;
    if (count > kMaxClaimRows) return fail(IPL_ERROR_TOO_LARGE, "number of rows must be at most %d", kMaxClaimRows);
    if (status == nullptr || !aligned(status, 4)) {
        return fail(IPL_ERROR_INVALID_VALUE, "status must be non-null and 4-byte aligned");
    }
    return IPL_SUCCESS;
}

template <bool kFork>
ipl_status launch_claim(const ClaimParams& p, cudaStream_t stream) {
    const size_t smem = 2 * sizeof(int) * static_cast<size_t>(p.count);
    if (smem > 40 * 1024) {
        const cudaError_t err = cudaFuncSetAttribute(page_claim_kernel<kFork>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                     2 * sizeof(int) * kMaxClaimRows);
        if (err != cudaSuccess) return fail(IPL_ERROR_CUDA, "page claim kernel setup failed: %s", cudaGetErrorString(err));
    }
    return launch_status(launch(page_claim_kernel<kFork>, 1, kPlanThreads, smem, stream, p), "page claim");
}

}  // namespace
}  // namespace ipl

extern "C" {

ipl_status ipl_rotary_embedding_bf16(const ipl_rotary_args* args, void* stream) {
    return ipl::run_rotary<false>(args, static_cast<cudaStream_t>(stream));
}

ipl_status ipl_rotary_embedding_cache_bf16(const ipl_rotary_args* args, void* stream) {
    return ipl::run_rotary<true>(args, static_cast<cudaStream_t>(stream));
}

ipl_status ipl_paged_attention_bf16(const ipl_paged_attention_args* args, void* stream) {
    return ipl::run_attention(args, static_cast<cudaStream_t>(stream));
}

ipl_status ipl_paged_attention_workspace(const ipl_paged_attention_args* args, size_t* bytes) {
    using namespace ipl;
    if (bytes == nullptr) return fail(IPL_ERROR_INVALID_VALUE, "bytes must be non-null");
    const ipl_status st = check_attention_args(args);
    if (st != IPL_SUCCESS) return st;
    int sms = 0, smem = 0;
    plan_limits(&sms, &smem);
    *bytes = args->num_tokens == 0 || args->num_seqs == 0 ? 0 : plan_attention(*args, sms).workspace;
    return IPL_SUCCESS;
}

const char* ipl_paged_attention_plan(const ipl_paged_attention_args* args) {
    using namespace ipl;
    if (check_attention_args(args) != IPL_SUCCESS) return "invalid";
    if (args->num_tokens == 0 || args->num_seqs == 0) return "none";
    int sms = 0, smem = 0;
    plan_limits(&sms, &smem);
    const AttentionPlan plan = plan_attention(*args, sms);
    if (!plan.vector) return "attention_row_kernel";
    static const char* const kNames[2][5] = {
        {"invalid", "attention_short_kernel<1>", "attention_short_kernel<2>", "attention_shared_kernel<1> + attention_join_parts_kernel",
         "attention_shared_kernel<2> + attention_join_parts_kernel"},
        {"attention_tile_kernel + attention_join_rows_kernel", "attention_tile_kernel + attention_join_rows_kernel + attention_short_kernel<1>",
         "attention_tile_kernel + attention_join_rows_kernel + attention_short_kernel<2>",
         "attention_tile_kernel + attention_join_rows_kernel + attention_shared_kernel<1> + attention_join_parts_kernel",
         "attention_tile_kernel + attention_join_rows_kernel + attention_shared_kernel<2> + attention_join_parts_kernel"}};
    return kNames[plan.tile ? 1 : 0][plan.tiles == 0 ? 0 : plan.tiles + (plan.cluster > 0 ? 0 : 2)];
}

ipl_status ipl_compact_pages_workspace(int64_t num_pages, size_t* bytes) {
    using namespace ipl;
    if (bytes == nullptr || num_pages < 0 || num_pages > INT_MAX / 2) {
        return fail(IPL_ERROR_INVALID_VALUE, "bytes must be non-null and the number of pages a non-negative 31-bit number");
    }
    *bytes = compact_workspace_bytes(num_pages);
    return IPL_SUCCESS;
}

ipl_status ipl_copy_pages(const ipl_page_caches* caches, int64_t num_pages, const int32_t* pairs, int64_t count,
                          void* stream) {
    using namespace ipl;
    ipl_status st = check_caches(caches);
    if (st != IPL_SUCCESS) return st;
    if (num_pages < 0 || count < 0) return fail(IPL_ERROR_INVALID_VALUE, "sizes must be non-negative");
    if (num_pages > INT_MAX || count > INT_MAX / kMaxCachesPerLaunch) return fail(IPL_ERROR_TOO_LARGE, "a size is too large");
    if (count == 0 || caches->page_bytes == 0) return IPL_SUCCESS;
    if (pairs == nullptr || !aligned(pairs, 4)) {
        return fail(IPL_ERROR_INVALID_VALUE, "pairs must be non-null and 4-byte aligned");
    }
    const PageLayout layout = page_layout(*caches);
    for (int64_t from = 0; from < caches->num_caches; from += kMaxCachesPerLaunch) {
        CopyPagesParams p = {};
        p.num_caches = cache_list(*caches, from, &p.caches);
        p.count = static_cast<int>(count);
        p.pairs = pairs;
        p.num_pages = static_cast<int>(num_pages);
        p.page = layout;
        const unsigned grid = static_cast<unsigned>(count * p.num_caches);
        st = launch_status(launch(page_copy_kernel, grid, kPageCopyThreads, 0, static_cast<cudaStream_t>(stream), p), "page copy");
        if (st != IPL_SUCCESS) return st;
    }
    return IPL_SUCCESS;
}

ipl_status ipl_reserve_pages(const ipl_page_pool* pool, const int32_t* rows, const int32_t* new_lens, int64_t count,
                             int32_t* status, void* stream) {
    using namespace ipl;
    const ipl_status st = check_claim(pool, rows, new_lens, count, status);
    if (st != IPL_SUCCESS) return st;
    const ClaimParams p = {page_state(*pool), nullptr, rows, new_lens, static_cast<int>(count), status};
    return launch_claim<false>(p, static_cast<cudaStream_t>(stream));
}

ipl_status ipl_fork_sequences(const ipl_page_caches* caches, const ipl_page_pool* pool, const int32_t* parents,
                              const int32_t* children, int64_t count, int32_t* status, void* stream) {
    using namespace ipl;
    ipl_status st = check_caches(caches);
    if (st == IPL_SUCCESS) st = check_claim(pool, children, parents, count, status);
    if (st != IPL_SUCCESS) return st;
    const ClaimParams claim = {page_state(*pool), parents, children, nullptr, static_cast<int>(count), status};
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    st = launch_claim<true>(claim, s);
    if (st != IPL_SUCCESS || count == 0) return st;
    const PageLayout layout = page_layout(*caches);
    int64_t from = 0;
    do {
        ForkParams p = {};
        p.num_caches = cache_list(*caches, from, &p.caches);
        p.count = static_cast<int>(count);
        p.with_tables = from == 0;
        p.state = claim.state;
        p.parents = parents;
        p.children = children;
        p.status = status;
        p.page = layout;
        if (p.num_caches == 0) p.num_caches = 1, p.page.bytes = 0;  // tables alone
        const unsigned grid = static_cast<unsigned>(count * p.num_caches);
        st = launch_status(launch(page_fork_kernel, grid, kPageCopyThreads, 0, s, p), "page fork");
        if (st != IPL_SUCCESS) return st;
        from += kMaxCachesPerLaunch;
    } while (from < caches->num_caches);
    return IPL_SUCCESS;
}

ipl_status ipl_release_sequences(const ipl_page_pool* pool, const int32_t* rows, int64_t count, void* stream) {
    using namespace ipl;
    ipl_status st = check_pool(pool);
    if (st == IPL_SUCCESS) st = check_rows(pool, rows, rows, count);
    if (st != IPL_SUCCESS || count == 0) return st;
    return launch_status(launch(page_release_kernel, static_cast<unsigned>(count), kReleaseThreads, 0,
                                static_cast<cudaStream_t>(stream), page_state(*pool), rows),
                         "page release");
}

ipl_status ipl_compact_pages(const ipl_page_caches* caches, const ipl_page_pool* pool, int32_t* new_block_tables,
                             int32_t* new_ref_counts, int32_t* live, void* workspace, size_t workspace_bytes,
                             void* stream) {
    using namespace ipl;
    ipl_status st = check_caches(caches);
    if (st == IPL_SUCCESS) st = check_pool(pool);
    if (st != IPL_SUCCESS) return st;
    if (workspace == nullptr || !aligned(workspace, 4)) {
        return fail(IPL_ERROR_INVALID_VALUE, "workspace must be non-null and 4-byte aligned");
    }
    if (workspace_bytes < compact_workspace_bytes(pool->num_pages)) {
        return fail(IPL_ERROR_INVALID_VALUE, "workspace is too small");
    }
    if ((pool->num_rows > 0 && pool->width > 0 && new_block_tables == nullptr) ||
        (pool->num_pages > 0 && new_ref_counts == nullptr) || live == nullptr) {
        return fail(IPL_ERROR_INVALID_VALUE, "new_block_tables, new_ref_counts and live must be non-null");
    }
    if (!aligned(new_block_tables, 4) || !aligned(new_ref_counts, 4) || !aligned(live, 4)) {
        return fail(IPL_ERROR_INVALID_VALUE, "int32 pointers must be 4-byte aligned");
    }
    if (pool->num_rows > 0 && pool->num_pages > 0 &&
        (new_block_tables == pool->block_tables || new_ref_counts == pool->ref_counts)) {
        return fail(IPL_ERROR_INVALID_VALUE, "the new tables and counts must not alias the old ones");
    }
    int device = 0;
    DeviceInfo* info = nullptr;
    st = current_device(&device, &info);
    if (st != IPL_SUCCESS) return st;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    CompactPlanParams plan = {};
    plan.ref_counts = pool->ref_counts;
    plan.new_ref_counts = new_ref_counts;
    plan.num_pages = static_cast<int>(pool->num_pages);
    plan.live = live;
    plan.map = static_cast<int32_t*>(workspace);
    plan.holes = plan.map + pool->num_pages;
    plan.movers = plan.holes + pool->num_pages;
    plan.moves = plan.movers + pool->num_pages;
    st = launch_status(launch(page_compact_plan_kernel, 1, kPlanThreads, 0, s, plan), "page compaction plan");
    if (st != IPL_SUCCESS) return st;
    const PageLayout layout = page_layout(*caches);
    int64_t from = 0;
    do {
        CompactMoveParams p = {};
        p.num_caches = cache_list(*caches, from, &p.caches);
        p.tables = from == 0 && pool->num_rows > 0 ? pool->block_tables : nullptr;
        p.new_tables = new_block_tables;
        p.table_row = pool->table_stride;
        p.num_rows = static_cast<int>(pool->num_rows);
        p.width = static_cast<int>(pool->width);
        p.num_pages = plan.num_pages;
        p.moves = plan.moves;
        p.map = plan.map;
        p.holes = plan.holes;
        p.movers = plan.movers;
        p.page = layout;
        // At most half the pages move; the kernel's loop covers what the grid does not.
        const int64_t most = pool->num_pages / 2 * p.num_caches;
        const int64_t entries = (pool->num_rows * pool->width + kPageMoveThreads - 1) / kPageMoveThreads;
        const int64_t cap = static_cast<int64_t>(info->sm_count.load(std::memory_order_relaxed)) * 8;
        int64_t grid = most > entries ? most : entries;
        grid = grid < 1 ? 1 : grid > cap ? cap : grid;
        if (p.num_caches == 0) p.num_caches = 1, p.page.bytes = 0;
        st = launch_status(launch(page_compact_move_kernel, static_cast<unsigned>(grid), kPageMoveThreads, 0, s, p),
                           "page compaction");
        if (st != IPL_SUCCESS) return st;
        from += kMaxCachesPerLaunch;
    } while (from < caches->num_caches);
    return IPL_SUCCESS;
}

}  // extern "C"
