// Attention of new tokens over a paged KV cache, for sm_100a.
//
// Token j of the n new ones of a sequence of L tokens (its own keys and values already in the cache)
// sits at position P = L - n + j and sees the keys t with max(0, P - window + 1) <= t <= P:
//
//   out = sum_t exp(scale q.k_t - m) v_t / sum_t exp(scale q.k_t - m),   m = max_t scale q.k_t
//
// in one pass over the keys with a running m and sum (fp32). A token that sees no key gives 0.
// Query head h reads key head h / (heads / kv_heads). Key t of a sequence lies in page
// table[t / page_size], row t % page_size.
#pragma once

#include "ipl_common.cuh"
#include "silu_and_mul.cuh"

namespace ipl {

constexpr int kAttentionMaxDim = 256;

struct AttentionParams {
    uint16_t* out;
    const uint16_t* q;
    const uint16_t* key_cache;
    const uint16_t* value_cache;
    const int32_t* tables;
    const int32_t* starts;
    const int32_t* lens;
    int num_tokens, num_seqs, heads, kv_heads, group, dim, page_size, num_pages, table_width;
    int window;  // INT_MAX without one
    int64_t table_row;
    int64_t out_token, out_head, q_token, q_head;
    int64_t key_page, key_token, key_head, value_page, value_token, value_head;
    float scale_log2;  // scale * log2(e): the exponentials are powers of two
    // Sequences of at most short_rows rows (new tokens x group) belong to the short kernels, the others
    // to the tile kernel. The short kernels count rows in 32 bits, the tile kernel only those of a tile.
    int short_rows;
    FastDiv32 page_blocks;  // blocks of 16 keys a page (fast kernels)
    FastDiv32 group_div;
    int row_tiles;  // row tiles of a sequence that the short kernel takes at the same time
};

// Rows whose keys several CTAs share. The CTAs take equal stretches of all the work, laid end to end, so CTA c
// leaves at most two parts: in slot 2 c the end (or a middle stretch) of rows that the CTA before began, in slot
// 2 c + 1 the beginning of rows that it leaves to the next. A slot holds sums [slot_rows][padded dim], not yet
// divided, and (maximum, sum of weights) [slot_rows].
struct AttentionPart {
    int tokens;  // 0: nothing in the slot
    int token, kv_head;  // first token (row of query), key head
    int last;            // the end of the rows' keys
};
struct AttentionParts {
    float* sums;
    float2* stats;
    AttentionPart* parts;
    int slot_rows;
    // A row of a slot: token row / tile_rows * tile_tokens + row % tile_rows / group, head row % tile_rows % group.
    int tile_rows, tile_tokens;
};

constexpr int kAttentionBlock = 16;  // keys a warp takes at once; a page holds a multiple of them

// The keys that a sequence's new tokens see, by its first and its last one: [first, stop).
struct KeyRange {
    int first, stop;
};
__device__ __forceinline__ KeyRange visible_keys(const AttentionParams& p, int len, int new_tokens) {
    const int from = len - new_tokens;  // position of the first new token
    KeyRange r;
    r.first = from >= p.window ? from - p.window + 1 : 0;
    r.stop = max(len, 0);
    return r;
}

__device__ __forceinline__ float exp2_approx(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// The sequence that token `token` belongs to: the last s with starts[s] <= token.
__device__ __forceinline__ int sequence_of_token(const int32_t* starts, int num_seqs, int token) {
    int lo = 0, hi = num_seqs - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (starts[mid] <= token) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

// The longest sequence whose keys, and those of a block or tile that begins below its end, 32 bits count.
constexpr int kMostKeys = INT32_MAX - 255;

// A sequence's length as far as its row of the block table and the count of keys reach.
__device__ __forceinline__ int table_bounded_length(const AttentionParams& p, int seq) {
    const int64_t most = min(static_cast<int64_t>(p.table_width) * p.page_size, static_cast<int64_t>(kMostKeys));
    const int len = p.lens[seq];
    if (len > most) {
        atomicOr(&g_fault_word, kFaultIndexOutOfRange);
        return static_cast<int>(most);
    }
    return len;
}

// a / b of non-negative numbers, in 32 bits where they fit (a 64-bit division takes several hundred cycles).
__device__ __forceinline__ int64_t divide(int64_t a, int64_t b) {
    if ((a | b) >> 32 == 0) return static_cast<uint32_t>(a) / static_cast<uint32_t>(b);
    return a / b;
}

__device__ __forceinline__ float warp_max(float value) {
#pragma unroll
    for (int offset = kWarpSize / 2; offset > 0; offset >>= 1) {
        value = fmaxf(value, __shfl_xor_sync(0xffffffffu, value, offset));
    }
    return value;
}

// Adds the parts. The first of some rows' parts is in slot 2 c + 1; the others follow in slots 2 (c + 1), 2 (c + 2),
// ..., up to the last, as far as those CTAs have a share. join_slots(base): of the slots of CTAs base to base + 31,
// one a lane, those that belong to the rows (bits); `last` says whether that is all.
__device__ __forceinline__ uint32_t join_slots(const AttentionParts& parts, int cta, int base, int lane, int& slot, bool& last) {
    slot = base + lane == cta ? 2 * cta + 1 : 2 * (base + lane);
    const bool there = base + lane < static_cast<int>(gridDim.x) && parts.parts[slot].tokens != 0;
    const uint32_t ends = __ballot_sync(0xffffffffu, there && parts.parts[slot].last != 0);
    last = ends != 0;
    return __ballot_sync(0xffffffffu, there && (ends == 0 || lane < __ffs(ends)));
}

// Output row of row `row` of a slot; null for padding.
__device__ __forceinline__ uint16_t* join_output(const AttentionParams& p, const AttentionParts& parts, const AttentionPart& part, int row) {
    const int in_tile = row % parts.tile_rows, token_in_tile = in_tile / p.group;
    const int token = row / parts.tile_rows * parts.tile_tokens + token_in_tile;
    if (token_in_tile >= parts.tile_tokens || token >= part.tokens) return nullptr;
    const int head = part.kv_head * p.group + in_tile - token_in_tile * p.group;
    return p.out + static_cast<int64_t>(part.token + token) * p.out_token + head * p.out_head;
}

template <int kMine>
__device__ __forceinline__ void load_part(const float* from, float (&x)[kMine]) {
    if constexpr (kMine == 4) {
        const float4 y = *reinterpret_cast<const float4*>(from);
        x[0] = y.x, x[1] = y.y, x[2] = y.z, x[3] = y.w;
    } else {
        const float2 y = *reinterpret_cast<const float2*>(from);
        x[0] = y.x, x[1] = y.y;
    }
}

template <int kMine>
__device__ __forceinline__ void write_joined(uint16_t* out, float weight, const float (&total)[kMine]) {
    const float inverse = weight > 0.0f || weight != weight ? 1.0f / weight : 0.0f;
#pragma unroll
    for (int i = 0; i < kMine; i += 2) {
        *reinterpret_cast<uint32_t*>(out + i) = pack_bf16x2(total[i] * inverse, total[i + 1] * inverse);
    }
}

// The tile kernel's parts, kDim / 32 elements a lane. Many pairs in few parts each (kSplit false): block (c, y) takes 64
// rows, a warp 8 of them at once; with a row a warp the blocks were four waves of start-up latency (19 us after 147
// cut pairs). Few pairs in many parts: block (c, y) takes 8 rows, its warps share the parts (18
// tokens on 8192 keys, the whole call: 22.7 us, one after the other 35.1; 23.1 since).
constexpr int kJoinRows = 8, kJoinWarps = 8;

template <int kDim, bool kSplit>
__global__ void __launch_bounds__(kJoinWarps * kWarpSize, 2) attention_join_rows_kernel(const AttentionParams p, const AttentionParts parts) {
    grid_dependency_wait();
    grid_launch_dependents();
    constexpr int kMine = kDim / kWarpSize;
    __shared__ float sums[kSplit ? kJoinWarps : 1][kJoinRows][kDim];
    __shared__ float2 stats[kSplit ? kJoinWarps : 1][kJoinRows];
    const int warp = threadIdx.x / kWarpSize, lane = threadIdx.x % kWarpSize;
    const int row0 = (kSplit ? blockIdx.y : blockIdx.y * kJoinWarps + warp) * kJoinRows;
    const AttentionPart part = parts.parts[2 * blockIdx.x + 1];
    if (row0 / parts.tile_rows * parts.tile_tokens + row0 % parts.tile_rows / p.group >= part.tokens) return;
    float m[kJoinRows], l[kJoinRows], total[kJoinRows][kMine] = {};
#pragma unroll
    for (int r = 0; r < kJoinRows; ++r) m[r] = -INFINITY, l[r] = 0.0f;
    bool last = false;
    int before = 0;
    for (int base = blockIdx.x; base < static_cast<int>(gridDim.x) && !last; base += kWarpSize) {
        int slot;
        for (uint32_t set = join_slots(parts, blockIdx.x, base, lane, slot, last); set != 0; set &= set - 1, ++before) {
            if (kSplit && before % kJoinWarps != warp) continue;
            const int64_t at = static_cast<int64_t>(__shfl_sync(0xffffffffu, slot, __ffs(set) - 1)) * parts.slot_rows + row0;
            const float2 own = lane < kJoinRows ? parts.stats[at + lane] : make_float2(0.0f, 0.0f);
            float x[kJoinRows][kMine];
#pragma unroll
            for (int r = 0; r < kJoinRows; ++r) load_part(parts.sums + (at + r) * kDim + lane * kMine, x[r]);
#pragma unroll
            for (int r = 0; r < kJoinRows; ++r) {
                const float there = __shfl_sync(0xffffffffu, own.x, r), top = fmaxf(m[r], there);
                const float shift = top == -INFINITY ? 0.0f : top;
                const float keep = exp2_approx(m[r] - shift), add = exp2_approx(there - shift);
                m[r] = top;
                l[r] = l[r] * keep + __shfl_sync(0xffffffffu, own.y, r) * add;
#pragma unroll
                for (int i = 0; i < kMine; ++i) total[r][i] = total[r][i] * keep + x[r][i] * add;
            }
        }
    }
    if constexpr (kSplit) {
#pragma unroll
        for (int r = 0; r < kJoinRows; ++r) {
#pragma unroll
            for (int i = 0; i < kMine; ++i) sums[warp][r][lane * kMine + i] = total[r][i];
            if (lane == 0) stats[warp][r] = make_float2(m[r], l[r]);
        }
        __syncthreads();
        // A row a warp.
        float top = -INFINITY, weight = 0.0f, sum[kMine] = {};
#pragma unroll
        for (int w = 0; w < kJoinWarps; ++w) top = fmaxf(top, stats[w][warp].x);
        const float shift = top == -INFINITY ? 0.0f : top;
#pragma unroll
        for (int w = 0; w < kJoinWarps; ++w) {
            const float f = exp2_approx(stats[w][warp].x - shift);
            weight += f * stats[w][warp].y;
#pragma unroll
            for (int i = 0; i < kMine; ++i) sum[i] += f * sums[w][warp][lane * kMine + i];
        }
        uint16_t* out = join_output(p, parts, part, row0 + warp);
        if (out != nullptr && lane * kMine < p.dim) write_joined(out + lane * kMine, weight, sum);
        return;
    }
    if (lane * kMine >= p.dim) return;
#pragma unroll
    for (int r = 0; r < kJoinRows; ++r) {
        uint16_t* out = join_output(p, parts, part, row0 + r);
        if (out != nullptr) write_joined(out + lane * kMine, l[r], total[r]);
    }
}

// Few rows in many parts (the shared kernel's): block (c, y) takes two rows, 8 warps share a row's parts.
constexpr int kJoinSplit = 8;

template <int kDim>
__global__ void __launch_bounds__(2 * kJoinSplit * kWarpSize) attention_join_parts_kernel(const AttentionParams p, const AttentionParts parts) {
    constexpr int kMine = kDim / kWarpSize;
    __shared__ float sums[2 * kJoinSplit][kDim];
    __shared__ float2 stats[2 * kJoinSplit];
    grid_dependency_wait();
    grid_launch_dependents();
    const AttentionPart part = parts.parts[2 * blockIdx.x + 1];
    if (2 * static_cast<int>(blockIdx.y) >= part.tokens * p.group) return;
    const int warp = threadIdx.x / kWarpSize, lane = threadIdx.x % kWarpSize;
    const int row = 2 * blockIdx.y + warp / kJoinSplit, turn = warp % kJoinSplit;
    float m = -INFINITY, l = 0.0f, total[kMine] = {};
    bool last = false;
    for (int base = blockIdx.x; base < static_cast<int>(gridDim.x) && !last; base += kWarpSize) {
        int slot;
        const uint32_t set = join_slots(parts, blockIdx.x, base, lane, slot, last);
        const bool mine = (set >> lane & 1u) != 0 && lane % kJoinSplit == turn;
        const int64_t at = static_cast<int64_t>(slot) * parts.slot_rows + row;
        const float2 own = mine ? parts.stats[at] : make_float2(-INFINITY, 0.0f);
        const float top = fmaxf(m, warp_max(own.x)), shift = top == -INFINITY ? 0.0f : top;
        const float keep = exp2_approx(m - shift), add = exp2_approx(own.x - shift);
        l = l * keep + warp_sum(own.y * add);
        m = top;
#pragma unroll
        for (int i = 0; i < kMine; ++i) total[i] *= keep;
#pragma unroll
        for (int j = 0; j < kWarpSize / kJoinSplit; ++j) {
            const int from = j * kJoinSplit + turn;
            const float f = __shfl_sync(0xffffffffu, add, from);
            const int64_t there = __shfl_sync(0xffffffffu, at, from);
            if (!(set >> from & 1u)) continue;
            float x[kMine];
            load_part(parts.sums + there * kDim + lane * kMine, x);
#pragma unroll
            for (int i = 0; i < kMine; ++i) total[i] += x[i] * f;
        }
    }
#pragma unroll
    for (int i = 0; i < kMine; ++i) sums[warp][lane * kMine + i] = total[i];
    if (lane == 0) stats[warp] = make_float2(m, l);
    __syncthreads();
    if (turn != 0) return;
#pragma unroll
    for (int w = 1; w < kJoinSplit; ++w) {
        const float2 other = stats[warp + w];
        const float top = fmaxf(m, other.x), shift = top == -INFINITY ? 0.0f : top;
        const float keep = exp2_approx(m - shift), add = exp2_approx(other.x - shift);
        l = l * keep + other.y * add;
        m = top;
#pragma unroll
        for (int i = 0; i < kMine; ++i) total[i] = total[i] * keep + sums[warp + w][lane * kMine + i] * add;
    }
    uint16_t* out = join_output(p, parts, part, row);
    if (out != nullptr && lane * kMine < p.dim) write_joined(out + lane * kMine, l, total);
}

// ---- everything else --------------------------------------------------------------------------------
//
// Any head size up to 256, page size, stride and alignment: a warp for each (token, head), a key a
// lane for the scores, an element a lane (and every 32nd further) for the sum of values.
constexpr int kAttentionRowWarps = 4;

__global__ void __launch_bounds__(kAttentionRowWarps * kWarpSize) attention_row_kernel(const AttentionParams p) {
    __shared__ float q_rows[kAttentionRowWarps][kAttentionMaxDim];
    grid_dependency_wait();
    grid_launch_dependents();
    const int warp = threadIdx.x / kWarpSize, lane = threadIdx.x % kWarpSize;
    const int64_t row = static_cast<int64_t>(blockIdx.x) * kAttentionRowWarps + warp;
    if (row >= static_cast<int64_t>(p.num_tokens) * p.heads) return;
    const int token = static_cast<int>(row / p.heads), head = static_cast<int>(row % p.heads);
    const int seq = sequence_of_token(p.starts, p.num_seqs, token);
    const int begin = p.starts[seq], end = min(p.starts[seq + 1], p.num_tokens);
    if (begin < 0 || token < begin || token >= end) return;  // padding
    float* q = q_rows[warp];
    for (int d = lane; d < p.dim; d += kWarpSize) {
        q[d] = bf16_bits_to_float(p.q[token * p.q_token + head * p.q_head + d]);
    }
    __syncwarp();
    const int len = table_bounded_length(p, seq);
    const int position = p.lens[seq] - (end - begin) + (token - begin);
    const int stop = min(position + 1, len);
    const int first = position >= p.window ? position - p.window + 1 : 0;
    const int32_t* table = p.tables + seq * p.table_row;
    const int kv_head = head / p.group;

    constexpr int kSlots = kAttentionMaxDim / kWarpSize;
    float acc[kSlots] = {};
    float top = -INFINITY, sum = 0.0f;
    for (int base = first; base < stop; base += kWarpSize) {
        const int key = base + lane;
        int page = -1;
        float score = -INFINITY;
        if (key < stop) {
            page = table[key / p.page_size];
            if (page < 0 || page >= p.num_pages) {
                atomicOr(&g_fault_word, kFaultIndexOutOfRange);
                page = -1;
            } else {
                const uint16_t* k = p.key_cache + page * p.key_page + (key % p.page_size) * p.key_token + kv_head * p.key_head;
                float dot = 0.0f;
                for (int d = 0; d < p.dim; ++d) dot += q[d] * bf16_bits_to_float(k[d]);
                score = dot * p.scale_log2;
            }
        }
        if (!__any_sync(0xffffffffu, page >= 0)) continue;
        // The maximum passes over NaN scores; their weights do not.
        const float new_top = fmaxf(top, warp_max(score)), shift = new_top == -INFINITY ? 0.0f : new_top;
        const float weight = exp2f(score - shift);
        const float keep = exp2f(top - shift);
        sum = sum * keep + warp_sum(weight);
        top = new_top;
#pragma unroll
        for (int i = 0; i < kSlots; ++i) acc[i] *= keep;
        for (int j = 0; j < kWarpSize; ++j) {
            const float w = __shfl_sync(0xffffffffu, weight, j);
            const int from = __shfl_sync(0xffffffffu, page, j);
            if (from < 0) continue;
            const int t = base + j;
            const uint16_t* v = p.value_cache + from * p.value_page + (t % p.page_size) * p.value_token + kv_head * p.value_head;
#pragma unroll
            for (int i = 0; i < kSlots; ++i) {
                const int d = lane + i * kWarpSize;
                if (d < p.dim) acc[i] += w * bf16_bits_to_float(v[d]);
            }
        }
    }
    const float inverse = sum > 0.0f || sum != sum ? 1.0f / sum : 0.0f;
#pragma unroll
    for (int i = 0; i < kSlots; ++i) {
        const int d = lane + i * kWarpSize;
        if (d < p.dim) p.out[token * p.out_token + head * p.out_head + d] = float_to_bf16_bits(acc[i] * inverse);
    }
}

}  // namespace ipl
