// Attention of few rows over a paged KV cache, for sm_100a: the formula of paged_attention.cuh.
//
// For the at most 8 kTiles rows (token, head of a group) that share a key head. Bound by the bytes of the
// cache: a warp loads blocks of 16 keys straight into the operand registers of mma.m16n8k16 (16-byte
// loads, no shared memory) and works on the transposed products, keys and head elements along M, rows
// along N = 8, so that seven heads of a group waste one column of eight:
//   S^T = K Q^T:  the sum over head elements does not care for their order, so lane (g, t) = (lane / 4,
//     lane % 4) takes the 16-byte chunks t, t + 4, ... of keys g and g + 8, and of row g of Q;
//   O^T = V^T P^T:  lane (g, t) takes chunk g of keys 2t, 2t + 1, 2t + 8, 2t + 9 and pairs the keys'
//     elements by byte permutes; P^T comes from the score registers by movmatrix.
// The loads of the next block are issued as soon as the registers are free, keys behind S^T, values behind
// O^T. The warps of a CTA take blocks in turn and are joined through shared memory. Two kernels share that:
// * attention_short_kernel: a cluster of 1 to 16 CTAs for each sequence, key head and tile of rows, joined through
//   distributed shared memory: one launch, no workspace, for small calls;
// * attention_shared_kernel: CTAs that fill the GPU once take equal stretches of all the blocks, laid end to end;
//   rows that a border cuts leave parts for attention_join_parts_kernel. No last wave, whatever the lengths.
#pragma once

#include "paged_attention.cuh"

namespace ipl {

constexpr int kShortWarps = 4;
constexpr int kShortCluster = 16;  // CTAs a cluster, at most (above 8 a kernel has to be allowed them)

__device__ __forceinline__ void mma_bf16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose_8x8(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
// 16 bytes, or zeros where the place holds nothing to read.
__device__ __forceinline__ U32x4 ld_stream_v4_or_zero(const uint16_t* p, bool there) {
    U32x4 r;
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %5, 0;\n\t"
        "mov.b32 %0, 0;\n\tmov.b32 %1, 0;\n\tmov.b32 %2, 0;\n\tmov.b32 %3, 0;\n\t"
        "@p ld.global.nc.L1::no_allocate.v4.b32 {%0,%1,%2,%3}, [%4];\n\t}"
        : "=&r"(r.v[0]), "=&r"(r.v[1]), "=&r"(r.v[2]), "=&r"(r.v[3])
        : "l"(p), "r"(static_cast<uint32_t>(there)));
    return r;
}

// A sequence as the short kernels see it.
struct ShortSequence {
    int begin, new_tokens, rows, true_len, len;
    int first;                // key that the first new token sees first
    int first_block, blocks;  // of 16 keys
};

__device__ __forceinline__ bool short_sequence(const AttentionParams& p, int seq, ShortSequence& s) {
    s.begin = p.starts[seq];
    s.new_tokens = min(p.starts[seq + 1], p.num_tokens) - s.begin;
    const int64_t rows = static_cast<int64_t>(s.new_tokens) * p.group;
    if (s.begin < 0 || s.new_tokens <= 0 || rows > p.short_rows) return false;
    s.rows = static_cast<int>(rows);
    s.true_len = p.lens[seq];
    s.len = table_bounded_length(p, seq);
    const KeyRange range = visible_keys(p, s.true_len, s.new_tokens);
    s.first = range.first;
    s.first_block = range.first / kAttentionBlock;
    s.blocks = max(0, (min(range.stop, s.len) + kAttentionBlock - 1) / kAttentionBlock - s.first_block);
    return true;
}

template <int kDim, int kTiles>
struct ShortShared {
    static constexpr int kRows = 8 * kTiles;
    alignas(16) float joined[kShortWarps][kRows][kDim + 4];
    float2 stats[kShortWarps][kRows];
    float2 cta_stats[kRows];
};

// Rows row0 and on of a sequence against its blocks block_begin to block_end, each warp's maxima, sums of weights
// and sums in shared memory. The whole CTA; ends with a barrier. kDim: the head size padded to 64 or 128; kTiles:
// column tiles of 8 rows; kBlocks: adjacent blocks a warp takes at once.
template <int kDim, int kTiles, int kBlocks>
__device__ __forceinline__ void short_rows(const AttentionParams& p, const ShortSequence& s, int seq, int kv_head, int row0,
                                           int block_begin, int block_end, ShortShared<kDim, kTiles>& shared) {
    constexpr int kRows = 8 * kTiles;
    constexpr int kChunks = kDim / 32;  // 16-byte chunks of a row a lane takes
    constexpr int kPasses = kDim / 64;  // 64-element halves of a value row
    constexpr int kMmas = kDim / 16;    // products of 16 head elements
    const int warp = threadIdx.x / kWarpSize, lane = threadIdx.x % kWarpSize;
    const int g = lane >> 2, t = lane & 3;
    const int32_t* table = p.tables + seq * p.table_row;
    const uint16_t* key_base = p.key_cache + kv_head * p.key_head;
    const uint16_t* value_base = p.value_cache + kv_head * p.value_head;

    // Q: row row0 + 8 n + g.
    uint32_t q[kTiles][kChunks][4];
#pragma unroll
    for (int n = 0; n < kTiles; ++n) {
        const int row = row0 + 8 * n + g;
        const int in_seq = static_cast<int>(fast_div(static_cast<uint32_t>(row), p.group_div));
        const int token = s.begin + in_seq, head = kv_head * p.group + row - in_seq * p.group;
        const uint16_t* src = p.q + token * p.q_token + head * p.q_head;
#pragma unroll
        for (int c = 0; c < kChunks; ++c) {
            const int d = 8 * (t + 4 * c);
            const U32x4 v = ld_stream_v4_or_zero(src + d, row < s.rows && d < p.dim);
#pragma unroll
            for (int i = 0; i < 4; ++i) q[n][c][i] = v.v[i];
        }
    }
    // Positions of the rows 2t, 2t + 1 of each tile (columns of the products).
    int position[kTiles][2];
#pragma unroll
    for (int n = 0; n < kTiles; ++n) {
#pragma unroll
        for (int j = 0; j < 2; ++j) position[n][j] = s.true_len - s.new_tokens + static_cast<int>(fast_div(static_cast<uint32_t>(row0 + 8 * n + 2 * t + j), p.group_div));
    }
    const int lowest = s.true_len - s.new_tokens + static_cast<int>(fast_div(static_cast<uint32_t>(row0), p.group_div));
    const int highest = s.true_len - s.new_tokens + static_cast<int>(fast_div(static_cast<uint32_t>(row0 + kRows - 1), p.group_div));

    float o[kTiles][kMmas][4] = {};
    float top[kTiles][2], sum[kTiles][2];
#pragma unroll
    for (int n = 0; n < kTiles; ++n) top[n][0] = top[n][1] = -INFINITY, sum[n][0] = sum[n][1] = 0.0f;

    // Page numbers of this warp's next 32 blocks, one a lane.
    constexpr int kTurn = kShortWarps * kBlocks, kTurns = kWarpSize / kBlocks;
    int pages = -1;
    const auto fetch_pages = [&](int block) {
        const int mine = block + lane / kBlocks * kTurn + lane % kBlocks;
        pages = -1;
        if (mine < block_end) {
            pages = table[fast_div(static_cast<uint32_t>(s.first_block + mine), p.page_blocks)];
            if (pages < 0 || pages >= p.num_pages) {
                atomicOr(&g_fault_word, kFaultIndexOutOfRange);
                pages = -1;
            }
        }
    };
    const auto in_page = [&](int block) {  // the block's first token in its page
        const uint32_t number = static_cast<uint32_t>(s.first_block + block);
        return static_cast<int64_t>(number - fast_div(number, p.page_blocks) * p.page_blocks.divisor) * kAttentionBlock;
    };
    uint32_t k[kBlocks][kChunks][2][4];  // chunk, key g or g + 8
    U32x4 v[kBlocks][kPasses][4];        // half of the row, key 2t, 2t + 1, 2t + 8, 2t + 9
    const auto load_keys = [&](int block, const int (&page)[kBlocks]) {
#pragma unroll
        for (int u = 0; u < kBlocks; ++u) {
            const int key0 = (s.first_block + block + u) * kAttentionBlock;
            const int64_t at = page[u] * p.key_page + in_page(block + u) * p.key_token;
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                const int key = g + 8 * r;
                const bool there = page[u] >= 0 && key0 + key < s.len;
                const uint16_t* src = key_base + at + key * p.key_token;
#pragma unroll
                for (int c = 0; c < kChunks; ++c) {
                    const int d = 8 * (t + 4 * c);
                    const U32x4 x = ld_stream_v4_or_zero(src + d, there && d < p.dim);
#pragma unroll
                    for (int i = 0; i < 4; ++i) k[u][c][r][i] = x.v[i];
                }
            }
        }
    };
    const auto load_values = [&](int block, const int (&page)[kBlocks]) {
#pragma unroll
        for (int u = 0; u < kBlocks; ++u) {
            const int key0 = (s.first_block + block + u) * kAttentionBlock;
            const int64_t at = page[u] * p.value_page + in_page(block + u) * p.value_token;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int key = 2 * t + (r & 1) + 4 * (r & 2);
                // Rows that no token sees may hold anything, NaN included: they count as zeros.
                const bool there = page[u] >= 0 && key0 + key < s.len && key0 + key >= s.first;
                const uint16_t* src = value_base + at + key * p.value_token;
#pragma unroll
                for (int h = 0; h < kPasses; ++h) {
                    const int d = 64 * h + 8 * g;
                    v[u][h][r] = ld_stream_v4_or_zero(src + d, there && d < p.dim);
                }
            }
        }
    };

    int block = block_begin + warp * kBlocks;
    int turn = 0, page[kBlocks], next_page[kBlocks];
    const auto take_pages = [&](int (&to)[kBlocks]) {  // -1 past block_end
#pragma unroll
        for (int u = 0; u < kBlocks; ++u) to[u] = __shfl_sync(0xffffffffu, pages, turn * kBlocks + u);
    };
    fetch_pages(block);
    take_pages(page);
    if (block < block_end) {
        load_keys(block, page);
        load_values(block, page);
    }
    for (; block < block_end; block += kTurn) {
        const int next = block + kTurn;
        turn = (turn + 1) % kTurns;
        if (turn == 0) fetch_pages(next);
        take_pages(next_page);

        float score[kBlocks][kTiles][4];
#pragma unroll
        for (int u = 0; u < kBlocks; ++u) {
#pragma unroll
            for (int n = 0; n < kTiles; ++n) {
                float even[4] = {}, odd[4] = {};
#pragma unroll
                for (int c = 0; c < kChunks; ++c) {
                    const uint32_t a0[4] = {k[u][c][0][0], k[u][c][1][0], k[u][c][0][1], k[u][c][1][1]};
                    const uint32_t a1[4] = {k[u][c][0][2], k[u][c][1][2], k[u][c][0][3], k[u][c][1][3]};
                    mma_bf16(even, a0, q[n][c][0], q[n][c][1]);
                    mma_bf16(odd, a1, q[n][c][2], q[n][c][3]);
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) score[u][n][i] = (even[i] + odd[i]) * p.scale_log2;
            }
        }
        if (next < block_end) load_keys(next, next_page);

        // score[u][n][2 r + j]: key g + 8 r of block u, row 2t + j.
#pragma unroll
        for (int u = 0; u < kBlocks; ++u) {
            const int key0 = (s.first_block + block + u) * kAttentionBlock;
            if (page[u] < 0 || key0 + kAttentionBlock > min(lowest + 1, s.len) || highest - key0 >= p.window) {
#pragma unroll
                for (int n = 0; n < kTiles; ++n) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int key = key0 + g + 4 * (i & 2), at = position[n][i & 1];
                        if (page[u] < 0 || key >= s.len || key > at || at - key >= p.window) score[u][n][i] = -INFINITY;
                    }
                }
            }
        }
        uint32_t weights[kBlocks][kTiles][2];
#pragma unroll
        for (int n = 0; n < kTiles; ++n) {
            float keep[2], shift[2];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                float m = top[n][j];
#pragma unroll
                for (int u = 0; u < kBlocks; ++u) m = fmaxf(m, fmaxf(score[u][n][j], score[u][n][2 + j]));
#pragma unroll
                for (int offset = 4; offset < kWarpSize; offset *= 2) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, offset));
                shift[j] = m == -INFINITY ? 0.0f : m;
                keep[j] = exp2_approx(top[n][j] - shift[j]);
                top[n][j] = m;
                sum[n][j] *= keep[j];
            }
#pragma unroll
            for (int m = 0; m < kMmas; ++m) {
#pragma unroll
                for (int i = 0; i < 4; ++i) o[n][m][i] *= keep[i & 1];
            }
#pragma unroll
            for (int u = 0; u < kBlocks; ++u) {
                float w[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    w[i] = exp2_approx(score[u][n][i] - shift[i & 1]);
                    sum[n][i & 1] += w[i];
                }
                // The weights of 16 bits for the product; their sum above is of the unrounded ones.
                weights[u][n][0] = transpose_8x8(pack_bf16x2(w[0], w[1]));
                weights[u][n][1] = transpose_8x8(pack_bf16x2(w[2], w[3]));
            }
        }
        // Product tile m: head elements 8g + m and 64 + 8g + m (kDim 128), 8g + 2m and 8g + 2m + 1 (64).
#pragma unroll
        for (int u = 0; u < kBlocks; ++u) {
#pragma unroll
            for (int m = 0; m < kMmas; ++m) {
                uint32_t a[4];
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    const int h = kPasses == 2 ? r : 0, e = kPasses == 2 ? m : 2 * m + r;
                    const uint32_t pick = e & 1 ? 0x7632u : 0x5410u;
                    a[r] = __byte_perm(v[u][h][0].v[e >> 1], v[u][h][1].v[e >> 1], pick);
                    a[2 + r] = __byte_perm(v[u][h][2].v[e >> 1], v[u][h][3].v[e >> 1], pick);
                }
#pragma unroll
                for (int n = 0; n < kTiles; ++n) mma_bf16(o[n][m], a, weights[u][n][0], weights[u][n][1]);
            }
        }
        if (next < block_end) load_values(next, next_page);
#pragma unroll
        for (int u = 0; u < kBlocks; ++u) page[u] = next_page[u];
    }

    // Join the warps: sums over their maxima, then one rescaled sum.
#pragma unroll
    for (int n = 0; n < kTiles; ++n) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            float l = sum[n][j];
#pragma unroll
            for (int offset = 4; offset < kWarpSize; offset *= 2) l += __shfl_xor_sync(0xffffffffu, l, offset);
            const int row = 8 * n + 2 * t + j;
            if (g == 0) shared.stats[warp][row] = make_float2(top[n][j], l);
#pragma unroll
            for (int m = 0; m < kMmas; ++m) {
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    const int d = kPasses == 2 ? 64 * r + 8 * g + m : 8 * g + 2 * m + r;
                    shared.joined[warp][row][d] = o[n][m][2 * r + j];
                }
            }
        }
    }
    __syncthreads();
}

// Four elements from `d` of a row, joined over the CTA's warps.
template <int kDim, int kTiles>
__device__ __forceinline__ float4 join_warps(const ShortShared<kDim, kTiles>& shared, int local, int d, float& m, float& l) {
    m = -INFINITY, l = 0.0f;
#pragma unroll
    for (int w = 0; w < kShortWarps; ++w) m = fmaxf(m, shared.stats[w][local].x);
    const float shift = m == -INFINITY ? 0.0f : m;
    float4 total = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
    for (int w = 0; w < kShortWarps; ++w) {
        const float2 part = shared.stats[w][local];
        const float f = exp2_approx(part.x - shift);
        const float4 x = *reinterpret_cast<const float4*>(&shared.joined[w][local][d]);
        l += f * part.y;
        total.x += f * x.x, total.y += f * x.y, total.z += f * x.z, total.w += f * x.w;
    }
    return total;
}

__device__ __forceinline__ void write_short(const AttentionParams& p, const ShortSequence& s, int kv_head, int row, int d, float l,
                                            float4 total) {
    const float inverse = l > 0.0f || l != l ? 1.0f / l : 0.0f;
    const int token = static_cast<int>(fast_div(static_cast<uint32_t>(row), p.group_div)), head = kv_head * p.group + row - token * p.group;
    st_v2(p.out + static_cast<int64_t>(s.begin + token) * p.out_token + head * p.out_head + d,
          pack_bf16x2(total.x * inverse, total.y * inverse), pack_bf16x2(total.z * inverse, total.w * inverse));
}

constexpr int kShortThreads = kShortWarps * kWarpSize;
// Where a warp has few turns, latency counts: it takes two blocks a turn for 8 rows, of which two CTAs fit an SM (255
// registers). Where the GPU is full three CTAs of one block a turn (168 registers) have as much in flight.
constexpr int short_blocks(int tiles) { return tiles == 1 ? 2 : 1; }
constexpr int kShortCtas = 2;
constexpr int shared_ctas(int tiles) { return tiles == 1 ? 3 : 2; }

template <int kDim, int kTiles>
__global__ void __launch_bounds__(kShortThreads, kShortCtas) attention_short_kernel(const AttentionParams p) {
    constexpr int kRows = 8 * kTiles;
    __shared__ ShortShared<kDim, kTiles> shared;
    grid_dependency_wait();
    grid_launch_dependents();
    const uint32_t rank = cluster_ctarank(), ctas = cluster_nctarank();
    const int unit = blockIdx.x / ctas, pair = unit / p.row_tiles, seq = pair / p.kv_heads, kv_head = pair - seq * p.kv_heads;
    ShortSequence s;
    // The CTAs of a cluster leave together.
    if (!short_sequence(p, seq, s)) return;
    const int block_begin = static_cast<int>(static_cast<int64_t>(s.blocks) * rank / ctas);
    const int block_end = static_cast<int>(static_cast<int64_t>(s.blocks) * (rank + 1) / ctas);
    for (int row0 = (unit - pair * p.row_tiles) * kRows; row0 < s.rows; row0 += p.row_tiles * kRows) {
        short_rows<kDim, kTiles, short_blocks(kTiles)>(p, s, seq, kv_head, row0, block_begin, block_end, shared);
        for (int e = threadIdx.x; e < kRows * (kDim / 4); e += kShortThreads) {
            const int local = e / (kDim / 4), d = e % (kDim / 4) * 4;
            float m, l;
            const float4 total = join_warps(shared, local, d, m, l);
            if (ctas > 1) {  // the CTA's sum takes the place of warp 0's
                *reinterpret_cast<float4*>(&shared.joined[0][local][d]) = total;
                if (d == 0) shared.cta_stats[local] = make_float2(m, l);
            } else if (row0 + local < s.rows && d < p.dim) {
                write_short(p, s, kv_head, row0 + local, d, l, total);
            }
        }
        if (ctas == 1) {
            __syncthreads();
            continue;
        }
        __syncwarp();
        cluster_arrive_release();
        cluster_wait_acquire();
        // Every CTA writes its share of the elements.
        const uint32_t sums_at = smem_addr(shared.joined), stats_at = smem_addr(shared.cta_stats);
        for (uint32_t e = rank * kShortThreads + threadIdx.x; e < kRows * (kDim / 4); e += ctas * kShortThreads) {
            const int local = e / (kDim / 4), d = e % (kDim / 4) * 4;
            float2 part[kShortCluster];
            float4 x[kShortCluster];
            float m = -INFINITY, l = 0.0f;
#pragma unroll
            for (uint32_t c = 0; c < kShortCluster; ++c) {
                part[c] = make_float2(-INFINITY, 0.0f);
                x[c] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                if (c < ctas) {
                    part[c] = ld_shared_cluster_f32x2(map_shared_to_rank(stats_at, c) + 8u * local);
                    x[c] = ld_shared_cluster_f32x4(map_shared_to_rank(sums_at, c) + 4u * (local * (kDim + 4) + d));
                }
            }
#pragma unroll
            for (int c = 0; c < kShortCluster; ++c) m = fmaxf(m, part[c].x);
            const float shift = m == -INFINITY ? 0.0f : m;
            float4 total = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
            for (int c = 0; c < kShortCluster; ++c) {
                const float f = exp2_approx(part[c].x - shift);
                l += f * part[c].y;
                total.x += f * x[c].x, total.y += f * x[c].y, total.z += f * x[c].z, total.w += f * x[c].w;
            }
            if (row0 + local < s.rows && d < p.dim) write_short(p, s, kv_head, row0 + local, d, l, total);
        }
        // No CTA's shared memory goes, or is written again, while another reads it.
        __syncwarp();
        cluster_arrive_release();
        cluster_wait_acquire();
    }
}

constexpr int kShortPairCost = 8;   // of a sequence and key head beside its blocks, in blocks
constexpr int kShortLeast = 24;     // of a stretch, in blocks: shorter ones cost more parts than they save time

template <int kDim, int kTiles>
__global__ void __launch_bounds__(kShortThreads, shared_ctas(kTiles)) attention_shared_kernel(const AttentionParams p,
                                                                                          const AttentionParts parts) {
    constexpr int kRows = 8 * kTiles;
    __shared__ ShortShared<kDim, kTiles> shared;
    __shared__ int sums[kShortWarps + 2];
    grid_dependency_wait();
    grid_launch_dependents();
    const int warp = threadIdx.x / kWarpSize, lane = threadIdx.x % kWarpSize;
    if (threadIdx.x < 2) parts.parts[2 * blockIdx.x + threadIdx.x].tokens = 0;

    // This CTA's stretch of the blocks: of each sequence in turn, key head after key head.
    const auto weight = [&](int seq) {
        ShortSequence s;
        return seq < p.num_seqs && short_sequence(p, seq, s) ? s.blocks + kShortPairCost : 0;
    };
    int mine = 0;
    for (int seq = threadIdx.x; seq < p.num_seqs; seq += kShortThreads) mine += weight(seq);
    mine = __reduce_add_sync(0xffffffffu, mine);
    if (lane == 0) sums[warp] = mine;
    __syncthreads();
    int head_weight = 0;
    for (int w = 0; w < kShortWarps; ++w) head_weight += sums[w];
    const int64_t all_weight = static_cast<int64_t>(head_weight) * p.kv_heads, share = max(divide(all_weight + gridDim.x - 1, gridDim.x), int64_t{kShortLeast});
    const int64_t share_begin = share * blockIdx.x, share_end = min(share_begin + share, all_weight);
    if (share_begin >= share_end) return;
    for (int base = 0, before = 0; base < p.num_seqs; base += kShortThreads) {
        const int w = weight(base + threadIdx.x);
        int through = w;
#pragma unroll
        for (int offset = 1; offset < kWarpSize; offset *= 2) {
            const int below = __shfl_up_sync(0xffffffffu, through, offset);
            if (lane >= offset) through += below;
        }
        __syncthreads();
        if (lane == kWarpSize - 1) sums[warp] = through;
        __syncthreads();
        int total = before;
        for (int i = 0; i < kShortWarps; ++i) {
            if (i == warp) through += total;
            total += sums[i];
        }
        const int64_t after = static_cast<int64_t>(through) * p.kv_heads, from = static_cast<int64_t>(through - w) * p.kv_heads;
        if (share_begin < after && share_begin >= from) {
            sums[kShortWarps] = base + threadIdx.x;
            sums[kShortWarps + 1] = through - w;
        }
        before = total;
        if (share_begin < static_cast<int64_t>(total) * p.kv_heads) break;
    }
    __syncthreads();
    int seq = sums[kShortWarps];
    ShortSequence s = {};
    bool exists = short_sequence(p, seq, s);
    int64_t left = share_end - share_begin;
    const int64_t into = share_begin - static_cast<int64_t>(sums[kShortWarps + 1]) * p.kv_heads;
    int kv_head = static_cast<int>(divide(into, s.blocks + kShortPairCost));
    int skip = static_cast<int>(into - static_cast<int64_t>(kv_head) * (s.blocks + kShortPairCost));
    while (left > 0) {
        if (!exists || kv_head == p.kv_heads) {
            kv_head = 0;
            if (++seq >= p.num_seqs) break;
            exists = short_sequence(p, seq, s);
            continue;
        }
        const int own_weight = s.blocks + kShortPairCost;
        const int take = static_cast<int>(left < own_weight - skip ? left : own_weight - skip);
        int block_begin = max(skip - kShortPairCost, 0), block_end = max(skip + take - kShortPairCost, 0);
        bool work = s.blocks > 0 ? block_end > block_begin : skip == 0;
        if (s.rows > kRows) {
            // More rows than a slot holds (a sequence longer than max_query_len): not cut, but done by the CTA
            // whose stretch has its beginning.
            work = skip == 0;
            block_begin = 0, block_end = s.blocks;
        }
        const int slot = block_end - block_begin < s.blocks ? 2 * static_cast<int>(blockIdx.x) + (block_begin == 0 ? 1 : 0) : -1;
        left -= take;
        skip = 0;
        for (int row0 = 0; work && row0 < s.rows; row0 += kRows) {
            short_rows<kDim, kTiles, 1>(p, s, seq, kv_head, row0, block_begin, block_end, shared);
            for (int e = threadIdx.x; e < kRows * (kDim / 4); e += kShortThreads) {
                const int local = e / (kDim / 4), d = e % (kDim / 4) * 4;
                float m, l;
                const float4 total = join_warps(shared, local, d, m, l);
                if (row0 + local >= s.rows || d >= p.dim) continue;
                if (slot < 0) {
                    write_short(p, s, kv_head, row0 + local, d, l, total);
                } else {
                    const int64_t at = static_cast<int64_t>(slot) * kRows + local;
                    *reinterpret_cast<float4*>(parts.sums + at * kDim + d) = total;
                    if (d == 0) parts.stats[at] = make_float2(m, l);
                }
            }
            __syncthreads();
        }
        if (work && slot >= 0 && threadIdx.x == 0) parts.parts[slot] = AttentionPart{s.new_tokens, s.begin, kv_head, block_end == s.blocks};
        ++kv_head;
    }
}

}  // namespace ipl
