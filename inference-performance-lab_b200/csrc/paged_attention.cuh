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
    // Sequences of at most short_rows rows (new tokens x group) belong to the short kernel, the others
    // to the tile kernel.
    int short_rows;
    int splits;     // clusters along a sequence's keys, at most
    int split_len;  // keys each takes, a multiple of kAttentionBlock (the last one: all that are left)
    // Parts of rows whose keys several clusters share: for split s of row r = token * heads + head, at
    // s * num_tokens * heads + r, the unnormalised sum [padded dim] and (maximum, sum of weights).
    float* part_sums;
    float2* part_stats;
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

// A sequence's length as far as its row of the block table reaches.
__device__ __forceinline__ int table_bounded_length(const AttentionParams& p, int seq) {
    const int64_t most = static_cast<int64_t>(p.table_width) * p.page_size;
    const int len = p.lens[seq];
    if (len > most) {
        atomicOr(&g_fault_word, kFaultIndexOutOfRange);
        return static_cast<int>(most);
    }
    return len;
}

__device__ __forceinline__ float warp_max(float value) {
#pragma unroll
    for (int offset = kWarpSize / 2; offset > 0; offset >>= 1) {
        value = fmaxf(value, __shfl_xor_sync(0xffffffffu, value, offset));
    }
    return value;
}

// ---- few rows: the cache streams through registers ------------------------------------------------
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
// O^T. The warps of a CTA take blocks in turn and are joined through shared memory at the end. Where sequences
// and key heads are few, a cluster of up to 8 CTAs shares a sequence's keys and adds its parts through
// distributed shared memory, which needs no workspace and no second launch; where even that leaves SMs idle,
// several clusters do, and attention_join_kernel adds theirs.

constexpr int kShortWarps = 4;
constexpr int kShortCluster = 8;  // CTAs a cluster, at most

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

// kDim: the head size padded to 64 or 128; kTiles: column tiles of 8 rows.
template <int kDim, int kTiles>
__global__ void __launch_bounds__(kShortWarps * kWarpSize, kTiles == 1 ? 3 : 2) attention_short_kernel(const AttentionParams p) {
    constexpr int kRows = 8 * kTiles;
    constexpr int kChunks = kDim / 32;   // 16-byte chunks of a row a lane takes
    constexpr int kPasses = kDim / 64;   // 64-element halves of a value row
    constexpr int kMmas = kDim / 16;     // products of 16 head elements
    constexpr int kThreads = kShortWarps * kWarpSize;
    __shared__ __align__(16) float joined[kShortWarps][kRows][kDim + 4];
    __shared__ float2 stats[kShortWarps][kRows], cta_stats[kRows];
    grid_dependency_wait();
    grid_launch_dependents();

    const uint32_t rank = cluster_ctarank(), ctas = cluster_nctarank();
    const uint32_t unit = blockIdx.x / ctas;
    const uint32_t pair = unit % (static_cast<uint32_t>(p.num_seqs) * p.kv_heads);
    const int split = unit / (static_cast<uint32_t>(p.num_seqs) * p.kv_heads);
    const int seq = pair / p.kv_heads, kv_head = pair - seq * p.kv_heads;
    const int begin = p.starts[seq], new_tokens = min(p.starts[seq + 1], p.num_tokens) - begin;
    const int rows = new_tokens * p.group;
    // The CTAs of a cluster leave together: here and below the conditions are the same for all of them.
    if (begin < 0 || new_tokens <= 0 || rows > p.short_rows) return;
    const int true_len = p.lens[seq];
    const int len = table_bounded_length(p, seq);
    const KeyRange range = visible_keys(p, true_len, new_tokens);
    const int first_block = range.first / kAttentionBlock;
    const int blocks = max(0, (min(range.stop, len) + kAttentionBlock - 1) / kAttentionBlock - first_block);
    const int split_blocks = p.split_len / kAttentionBlock;
    const int used = min(p.splits, max(1, (blocks + split_blocks - 1) / split_blocks));
    if (split >= used) return;
    const int share_begin = split * split_blocks, share = (split == used - 1 ? blocks : share_begin + split_blocks) - share_begin;
    const int block_begin = share_begin + static_cast<int>(static_cast<int64_t>(share) * rank / ctas);
    const int block_end = share_begin + static_cast<int>(static_cast<int64_t>(share) * (rank + 1) / ctas);

    const int warp = threadIdx.x / kWarpSize, lane = threadIdx.x % kWarpSize;
    const int g = lane >> 2, t = lane & 3;
    const int32_t* table = p.tables + seq * p.table_row;
    const uint16_t* key_base = p.key_cache + kv_head * p.key_head;
    const uint16_t* value_base = p.value_cache + kv_head * p.value_head;
    const int blocks_per_page = p.page_size / kAttentionBlock;

    for (int row0 = 0; row0 < rows; row0 += kRows) {
        // Q: row row0 + 8 n + g.
        uint32_t q[kTiles][kChunks][4];
#pragma unroll
        for (int n = 0; n < kTiles; ++n) {
            const int row = row0 + 8 * n + g;
            const int token = begin + row / p.group, head = kv_head * p.group + row % p.group;
            const uint16_t* src = p.q + token * p.q_token + head * p.q_head;
#pragma unroll
            for (int c = 0; c < kChunks; ++c) {
                const int d = 8 * (t + 4 * c);
                const U32x4 v = ld_stream_v4_or_zero(src + d, row < rows && d < p.dim);
#pragma unroll
                for (int i = 0; i < 4; ++i) q[n][c][i] = v.v[i];
            }
        }
        // Positions of the rows 2t, 2t + 1 of each tile (columns of the products).
        int position[kTiles][2];
#pragma unroll
        for (int n = 0; n < kTiles; ++n) {
#pragma unroll
            for (int j = 0; j < 2; ++j) position[n][j] = true_len - new_tokens + (row0 + 8 * n + 2 * t + j) / p.group;
        }
        const int lowest = true_len - new_tokens + row0 / p.group;
        const int highest = true_len - new_tokens + (row0 + kRows - 1) / p.group;

        float o[kTiles][kMmas][4] = {};
        float top[kTiles][2], sum[kTiles][2];
#pragma unroll
        for (int n = 0; n < kTiles; ++n) top[n][0] = top[n][1] = -INFINITY, sum[n][0] = sum[n][1] = 0.0f;

        // Page numbers of this warp's next 32 blocks, one a lane.
        int pages = -1;
        const auto fetch_pages = [&](int block) {
            const int mine = block + lane * kShortWarps;
            pages = -1;
            if (mine < block_end) {
                pages = table[(first_block + mine) / blocks_per_page];
                if (pages < 0 || pages >= p.num_pages) {
                    atomicOr(&g_fault_word, kFaultIndexOutOfRange);
                    pages = -1;
                }
            }
        };
        uint32_t k[kChunks][2][4];  // chunk, key g or g + 8
        U32x4 v[kPasses][4];        // half of the row, key 2t, 2t + 1, 2t + 8, 2t + 9
        const auto load_keys = [&](int block, int page) {
            const int key0 = (first_block + block) * kAttentionBlock;
            const int64_t at = page * p.key_page + static_cast<int64_t>((first_block + block) % blocks_per_page * kAttentionBlock) * p.key_token;
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                const int key = g + 8 * r;
                const bool there = page >= 0 && key0 + key < len;
                const uint16_t* src = key_base + at + key * p.key_token;
#pragma unroll
                for (int c = 0; c < kChunks; ++c) {
                    const int d = 8 * (t + 4 * c);
                    const U32x4 x = ld_stream_v4_or_zero(src + d, there && d < p.dim);
#pragma unroll
                    for (int i = 0; i < 4; ++i) k[c][r][i] = x.v[i];
                }
            }
        };
        const auto load_values = [&](int block, int page) {
            const int key0 = (first_block + block) * kAttentionBlock;
            const int64_t at = page * p.value_page + static_cast<int64_t>((first_block + block) % blocks_per_page * kAttentionBlock) * p.value_token;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int key = 2 * t + (r & 1) + 4 * (r & 2);
                // Rows that no token sees may hold anything, NaN included: they count as zeros.
                const bool there = page >= 0 && key0 + key < len && key0 + key >= range.first;
                const uint16_t* src = value_base + at + key * p.value_token;
#pragma unroll
                for (int h = 0; h < kPasses; ++h) {
                    const int d = 64 * h + 8 * g;
                    v[h][r] = ld_stream_v4_or_zero(src + d, there && d < p.dim);
                }
            }
        };

        int block = block_begin + warp;
        int turn = 0;
        fetch_pages(block);
        int page = __shfl_sync(0xffffffffu, pages, 0);
        if (block < block_end) {
            load_keys(block, page);
            load_values(block, page);
        }
        for (; block < block_end; block += kShortWarps) {
            const int next = block + kShortWarps;
            turn = (turn + 1) & 31;
            if (turn == 0) fetch_pages(next);
            const int next_page = __shfl_sync(0xffffffffu, pages, turn);

            float s[kTiles][4];
#pragma unroll
            for (int n = 0; n < kTiles; ++n) {
                float even[4] = {}, odd[4] = {};
#pragma unroll
                for (int c = 0; c < kChunks; ++c) {
                    const uint32_t a0[4] = {k[c][0][0], k[c][1][0], k[c][0][1], k[c][1][1]};
                    const uint32_t a1[4] = {k[c][0][2], k[c][1][2], k[c][0][3], k[c][1][3]};
                    mma_bf16(even, a0, q[n][c][0], q[n][c][1]);
                    mma_bf16(odd, a1, q[n][c][2], q[n][c][3]);
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) s[n][i] = (even[i] + odd[i]) * p.scale_log2;
            }
            if (next < block_end) load_keys(next, next_page);

            const int key0 = (first_block + block) * kAttentionBlock;
            // s[n][2 r + j]: key g + 8 r, row 2t + j.
            if (page < 0 || key0 + kAttentionBlock > min(lowest + 1, len) || highest - key0 >= p.window) {
#pragma unroll
                for (int n = 0; n < kTiles; ++n) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int key = key0 + g + 4 * (i & 2), at = position[n][i & 1];
                        if (page < 0 || key >= len || key > at || at - key >= p.window) s[n][i] = -INFINITY;
                    }
                }
            }
            uint32_t weights[kTiles][2];
#pragma unroll
            for (int n = 0; n < kTiles; ++n) {
                float keep[2], shift[2];
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    float m = fmaxf(s[n][j], s[n][2 + j]);
#pragma unroll
                    for (int offset = 4; offset < kWarpSize; offset *= 2) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, offset));
                    m = fmaxf(m, top[n][j]);
                    shift[j] = m == -INFINITY ? 0.0f : m;
                    keep[j] = exp2_approx(top[n][j] - shift[j]);
                    top[n][j] = m;
                }
                float w[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) w[i] = exp2_approx(s[n][i] - shift[i & 1]);
#pragma unroll
                for (int j = 0; j < 2; ++j) sum[n][j] = sum[n][j] * keep[j] + (w[j] + w[2 + j]);
#pragma unroll
                for (int m = 0; m < kMmas; ++m) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) o[n][m][i] *= keep[i & 1];
                }
                // The weights of 16 bits for the product; their sum above is of the unrounded ones.
                weights[n][0] = transpose_8x8(pack_bf16x2(w[0], w[1]));
                weights[n][1] = transpose_8x8(pack_bf16x2(w[2], w[3]));
            }
            // Product tile m: head elements 8g + m and 64 + 8g + m (kDim 128), 8g + 2m and 8g + 2m + 1 (64).
#pragma unroll
            for (int m = 0; m < kMmas; ++m) {
                uint32_t a[4];
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    const int h = kPasses == 2 ? r : 0, e = kPasses == 2 ? m : 2 * m + r;
                    const uint32_t pick = e & 1 ? 0x7632u : 0x5410u;
                    a[r] = __byte_perm(v[h][0].v[e >> 1], v[h][1].v[e >> 1], pick);
                    a[2 + r] = __byte_perm(v[h][2].v[e >> 1], v[h][3].v[e >> 1], pick);
                }
#pragma unroll
                for (int n = 0; n < kTiles; ++n) mma_bf16(o[n][m], a, weights[n][0], weights[n][1]);
            }
            if (next < block_end) load_values(next, next_page);
            page = next_page;
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
                if (g == 0) stats[warp][row] = make_float2(top[n][j], l);
#pragma unroll
                for (int m = 0; m < kMmas; ++m) {
#pragma unroll
                    for (int r = 0; r < 2; ++r) {
                        const int d = kPasses == 2 ? 64 * r + 8 * g + m : 8 * g + 2 * m + r;
                        joined[warp][row][d] = o[n][m][2 * r + j];
                    }
                }
            }
        }
        __syncthreads();
        const auto write = [&](int local, int d, float m, float l, float4 total) {
            const int row = row0 + local;
            if (row >= rows || d >= p.dim) return;
            const int token = begin + row / p.group, head = kv_head * p.group + row % p.group;
            if (used > 1) {
                const int64_t at = (static_cast<int64_t>(split) * p.num_tokens + token) * p.heads + head;
                *reinterpret_cast<float4*>(p.part_sums + at * kDim + d) = total;
                if (d == 0) p.part_stats[at] = make_float2(m, l);
            } else {
                const float inverse = l > 0.0f || l != l ? 1.0f / l : 0.0f;
                st_v2(p.out + token * p.out_token + head * p.out_head + d, pack_bf16x2(total.x * inverse, total.y * inverse),
                      pack_bf16x2(total.z * inverse, total.w * inverse));
            }
        };
        // Four elements a thread, from all the warps; in a cluster the sum takes the place of warp 0's.
        for (int e = threadIdx.x; e < kRows * (kDim / 4); e += kThreads) {
            const int local = e / (kDim / 4), d = e % (kDim / 4) * 4;
            float m = -INFINITY;
#pragma unroll
            for (int w = 0; w < kShortWarps; ++w) m = fmaxf(m, stats[w][local].x);
            const float shift = m == -INFINITY ? 0.0f : m;
            float l = 0.0f;
            float4 total = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
            for (int w = 0; w < kShortWarps; ++w) {
                const float2 part = stats[w][local];
                const float f = exp2_approx(part.x - shift);
                const float4 x = *reinterpret_cast<const float4*>(&joined[w][local][d]);
                l += f * part.y;
                total.x += f * x.x, total.y += f * x.y, total.z += f * x.z, total.w += f * x.w;
            }
            if (ctas > 1) {
                *reinterpret_cast<float4*>(&joined[0][local][d]) = total;
                if (d == 0) cta_stats[local] = make_float2(m, l);
            } else {
                write(local, d, m, l, total);
            }
        }
        if (ctas > 1) {
            __syncwarp();
            cluster_arrive_release();
            cluster_wait_acquire();
            // Every CTA writes its share of the elements.
            const uint32_t sums_at = smem_addr(joined), stats_at = smem_addr(cta_stats);
            for (uint32_t e = rank * kThreads + threadIdx.x; e < kRows * (kDim / 4); e += ctas * kThreads) {
                const int local = e / (kDim / 4), d = e % (kDim / 4) * 4;
                float2 part[kShortCluster];
                float4 x[kShortCluster];
                float m = -INFINITY, l = 0.0f;
#pragma unroll
                for (uint32_t c = 0; c < kShortCluster; ++c) {
                    if (c >= ctas) {
                        part[c] = make_float2(-INFINITY, 0.0f);
                        x[c] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                        continue;
                    }
                    part[c] = ld_shared_cluster_f32x2(map_shared_to_rank(stats_at, c) + 8u * local);
                    x[c] = ld_shared_cluster_f32x4(map_shared_to_rank(sums_at, c) + 4u * (local * (kDim + 4) + d));
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
                write(local, d, m, l, total);
            }
            // No CTA's shared memory goes, or is written again, while another reads it.
            __syncwarp();
            cluster_arrive_release();
            cluster_wait_acquire();
        } else {
            __syncthreads();
        }
    }
}

// Adds the parts of split rows: a CTA for each sequence and key head, a warp for each row in turn, kDim / 32
// elements a lane.
constexpr int kJoinWarps = 8;

template <int kDim>
__global__ void __launch_bounds__(kJoinWarps * kWarpSize) attention_join_kernel(const AttentionParams p) {
    grid_dependency_wait();
    grid_launch_dependents();
    constexpr int kMine = kDim / kWarpSize;
    const int lane = threadIdx.x % kWarpSize;
    const int seq = blockIdx.x / p.kv_heads, kv_head = blockIdx.x - seq * p.kv_heads;
    const int64_t rows = static_cast<int64_t>(p.num_tokens) * p.heads;
    const int begin = p.starts[seq], new_tokens = min(p.starts[seq + 1], p.num_tokens) - begin;
    if (begin < 0 || new_tokens <= 0 || new_tokens * p.group > p.short_rows) return;
    const KeyRange range = visible_keys(p, p.lens[seq], new_tokens);
    const int first_block = range.first / kAttentionBlock;
    const int stop = min(range.stop, table_bounded_length(p, seq));
    const int blocks = max(0, (stop + kAttentionBlock - 1) / kAttentionBlock - first_block);
    const int split_blocks = p.split_len / kAttentionBlock;
    const int used = min(p.splits, max(1, (blocks + split_blocks - 1) / split_blocks));
    if (used == 1) return;  // written already
    for (int mine = threadIdx.x / kWarpSize; mine < new_tokens * p.group; mine += kJoinWarps) {
        const int token = begin + mine / p.group, head = kv_head * p.group + mine % p.group;
        const int64_t row = static_cast<int64_t>(token) * p.heads + head;
        float m = -INFINITY;
        for (int s = lane; s < used; s += kWarpSize) m = fmaxf(m, p.part_stats[s * rows + row].x);
        m = warp_max(m);
        const float shift = m == -INFINITY ? 0.0f : m;
        float l = 0.0f, total[kMine] = {};
#pragma unroll 4
        for (int s = 0; s < used; ++s) {
            const float2 part = p.part_stats[s * rows + row];
            const float f = exp2_approx(part.x - shift);
            l += f * part.y;
            const float* x = p.part_sums + (s * rows + row) * kDim + lane * kMine;
            if constexpr (kMine == 4) {
                const float4 y = *reinterpret_cast<const float4*>(x);
                total[0] += f * y.x, total[1] += f * y.y, total[2] += f * y.z, total[3] += f * y.w;
            } else {
                const float2 y = *reinterpret_cast<const float2*>(x);
                total[0] += f * y.x, total[1] += f * y.y;
            }
        }
        const float inverse = l > 0.0f || l != l ? 1.0f / l : 0.0f;
        const int d = lane * kMine;
        if (d >= p.dim) continue;
        uint16_t* out = p.out + token * p.out_token + head * p.out_head + d;
        if constexpr (kMine == 4) {
            st_v2(out, pack_bf16x2(total[0] * inverse, total[1] * inverse), pack_bf16x2(total[2] * inverse, total[3] * inverse));
        } else {
            *reinterpret_cast<uint32_t*>(out) = pack_bf16x2(total[0] * inverse, total[1] * inverse);
        }
    }
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
        const float new_top = fmaxf(top, warp_max(score));
        if (new_top == -INFINITY) continue;
        const float weight = exp2f(score - new_top);
        const float keep = exp2f(top - new_top);
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
    const float inverse = sum > 0.0f ? 1.0f / sum : 0.0f;
#pragma unroll
    for (int i = 0; i < kSlots; ++i) {
        const int d = lane + i * kWarpSize;
        if (d < p.dim) p.out[token * p.out_token + head * p.out_head + d] = float_to_bf16_bits(acc[i] * inverse);
    }
}

}  // namespace ipl
