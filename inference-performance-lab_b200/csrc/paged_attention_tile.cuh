// Attention of many rows over a paged KV cache on the tensor cores (tcgen05), for sm_100a: the formula
// of paged_attention.cuh.
//
// A tile is 128 rows (token, head) that share a key head: floor(128 / group) tokens times the heads of
// the group, so that a group reads its keys once. A CTA takes two tiles of adjacent tokens and walks over
// their keys, 128 at a time:
//   S_t = Q_t K^T (tensor memory)  ->  P_t = exp2(scale S_t - m) (registers)  ->  O_t += P_t V
// with the scores of one tile in the softmax while the tensor core works on the other. Roles:
//   warps 0-3, 4-7   softmax of tile 0 and 1, a row a thread (a lane of tensor memory): no shuffles;
//   warp 8           one thread issues the products;
//   warp 9           loads K and V page by page (TMA) into a ring of shared-memory stages.
// P overwrites the first half of its S; the products are issued in the order P_t V (step j), Q_t K^T (step
// j + 1), which the tensor core keeps, so nothing is overwritten early. The running maximum is only moved
// when it has grown by more than 2^8, which then rescales O in tensor memory: the result is the same, as
// any reference point within the exponents' range is (weights of at most 2^8 lose nothing in 16 bits).
#pragma once

#include "paged_attention.cuh"
#include "tensor_core.cuh"

namespace ipl {

constexpr int kTileRows = 128;
constexpr int kTileKeys = 128;
constexpr int kTileThreads = 384;  // three warpgroups, among which the registers are split
// Registers a thread: launched with 65536 / 384 rounded down to 168 (64512 in all), of which the two
// softmax warpgroups take 208 and the third keeps 88 (64512 again).
constexpr int kSoftmaxRegisters = 208, kOtherRegisters = 88;
constexpr int kTilePolynomial = 0;  // of 16 pairs of weights, by the polynomial
constexpr int kTileBoxes = kTileKeys / kAttentionBlock;  // boxes of at least 16 keys a tile

struct TileParams {
    AttentionParams a;
    int tile_tokens;  // tokens a tile: 128 / group
    int box_keys;     // keys a TMA box: the largest power of two up to 128 that divides the page size
    int pairs;        // upper bound of the tile pairs of all sequences
};

// Shared memory: the two Q tiles, the stages, the barriers. A tile of kDim 128 is two halves of 64
// elements (128-byte rows), one after the other.
template <int kDim>
struct TileLayout {
    static constexpr int kHalves = kDim / 64;
    static constexpr uint32_t kHalfBytes = kTileRows * 128;
    static constexpr uint32_t kTileBytes = kHalves * kHalfBytes;
    static constexpr int kStages = kDim == 128 ? 5 : 8;
    static constexpr uint32_t kStageBase = 2 * kTileBytes;
    static constexpr uint32_t kBarrierBase = kStageBase + kStages * kTileBytes;
    static constexpr uint32_t kItemBase = kBarrierBase + 384;
    static constexpr uint32_t kBytes = kItemBase + 128;
    static constexpr uint32_t kDynamic = kBytes + 1024;  // room to align to 1024
};

// Powers of two of a pair. The special-function units give 16 a cycle and SM, as many as the products of a
// step have scores for each of their cycles, so a part of the pairs is computed on the FMA pipes:
// 2^x = 2^n 2^r, n = x rounded (by adding 1.5 2^23, which leaves n in the low bits), r in [-1/2, 1/2],
// with the polynomial of degree 3 of least relative error for 2^r (7.5e-5 by the Remez exchange, a fiftieth
// of the rounding of a weight to bf16). x is held above -126, so a vanishing weight is 2^-126, not 0.
__device__ __forceinline__ F32x2 exp2_pair_units(F32x2 x) {
    float a, b;
    f32x2_split(x, a, b);
    return f32x2_make(exp2_approx(a), exp2_approx(b));
}
__device__ __forceinline__ F32x2 exp2_pair_polynomial(F32x2 x) {
    float a, b;
    f32x2_split(x, a, b);
    x = f32x2_make(fmaxf(a, -126.0f), fmaxf(b, -126.0f));
    const F32x2 magic = f32x2_make(12582912.0f, 12582912.0f), minus = f32x2_make(-12582912.0f, -12582912.0f);
    const F32x2 n = f32x2_add(x, magic);
    const F32x2 r = f32x2_fma(f32x2_add(n, minus), f32x2_make(-1.0f, -1.0f), x);
    F32x2 y = f32x2_fma(r, f32x2_make(0.05517166852951050f, 0.05517166852951050f), f32x2_make(0.2426111251115799f, 0.2426111251115799f));
    y = f32x2_fma(y, r, f32x2_make(0.6932609677314758f, 0.6932609677314758f));
    y = f32x2_fma(y, r, f32x2_make(0.9999280571937561f, 0.9999280571937561f));
    float na, nb;
    f32x2_split(n, na, nb);
    f32x2_split(y, a, b);
    return f32x2_make(__uint_as_float(__float_as_uint(a) + (__float_as_uint(na) << 23)),
                      __uint_as_float(__float_as_uint(b) + (__float_as_uint(nb) << 23)));
}

// The largest of three, NaN if one is.
__device__ __forceinline__ float max3(float a, float b, float c) {
    float m;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(m) : "f"(a), "f"(b), "f"(c));
    return m;
}

// Weights of 32 scores: 2^(score scale - shift), rounded to bf16 pairs; their unrounded sum is added up.
// kPolynomial: of every 16 pairs, this many by the polynomial.
template <int kPolynomial>
__device__ __forceinline__ void tile_weights(const float (&s)[32], F32x2 scale, F32x2 minus_shift, uint32_t (&w)[16], F32x2 (&sums)[2]) {
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const F32x2 x = f32x2_fma(f32x2_make(s[2 * i], s[2 * i + 1]), scale, minus_shift);
        const bool polynomial = (i + 1) * kPolynomial / 16 > i * kPolynomial / 16;
        const F32x2 y = polynomial ? exp2_pair_polynomial(x) : exp2_pair_units(x);
        sums[i & 1] = f32x2_add(sums[i & 1], y);
        w[i] = f32x2_to_bf16x2(y);
    }
}

// Tensor memory columns.
constexpr uint32_t kTmemScores = 0;     // tile t at 128 t
constexpr uint32_t kTmemOutput = 256;   // tile t at 256 + 128 t

// What a CTA works on; in shared memory, read where it is used, so that it takes no registers.
struct TileItem {
    int work;  // 0: nothing
    int seq, begin, new_tokens, true_len, len, first;
    int kv_head;
    int token0;     // of the pair, in the sequence
    int tiles;      // 1 or 2
    int key0;       // of step 0, a multiple of 128
    int steps;
};

__device__ __forceinline__ TileItem tile_item(const TileParams& p) {
    TileItem item = {};
    const AttentionParams& a = p.a;
    const uint32_t unit = blockIdx.x / a.kv_heads;
    item.kv_head = blockIdx.x - unit * a.kv_heads;
    // Pair numbers are laid out so that sequence s starts at starts[s] / (tokens a pair) + s, which leaves it
    // room for its own rounded up. The last pairs, which see the most keys, come first.
    const int pair_tokens = 2 * p.tile_tokens;
    const int u = p.pairs - 1 - static_cast<int>(unit);
    int lo = 0, hi = a.num_seqs - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (a.starts[mid] / pair_tokens + mid <= u) lo = mid;
        else hi = mid - 1;
    }
    item.seq = lo;
    item.begin = a.starts[lo];
    item.new_tokens = min(a.starts[lo + 1], a.num_tokens) - item.begin;
    item.token0 = (u - (item.begin / pair_tokens + lo)) * pair_tokens;
    if (item.begin < 0 || item.token0 < 0 || item.token0 >= item.new_tokens || item.new_tokens * a.group <= a.short_rows) return item;
    item.tiles = item.token0 + p.tile_tokens < item.new_tokens ? 2 : 1;
    item.true_len = a.lens[lo];
    item.len = table_bounded_length(a, lo);
    const int from = item.true_len - item.new_tokens + item.token0;  // position of the pair's first token
    const int last = item.true_len - item.new_tokens + min(item.token0 + pair_tokens, item.new_tokens) - 1;
    item.first = from >= a.window ? from - a.window + 1 : 0;
    const int stop = min(last + 1, item.len);
    item.key0 = item.first / kTileKeys * kTileKeys;
    item.steps = stop > item.key0 ? (stop - item.key0 + kTileKeys - 1) / kTileKeys : 0;
    item.work = 1;
    return item;
}

template <int kDim>
__global__ void __launch_bounds__(kTileThreads, 1) attention_tile_kernel(const __grid_constant__ TileParams p,
                                                                         const __grid_constant__ CUtensorMap q_map,
                                                                         const __grid_constant__ CUtensorMap k_map,
                                                                         const __grid_constant__ CUtensorMap v_map) {
    using L = TileLayout<kDim>;
    extern __shared__ uint8_t dynamic_smem[];
    const uint32_t smem = (smem_addr(dynamic_smem) + 1023u) & ~1023u;
    const uint32_t bars = smem + L::kBarrierBase;
    const uint32_t stage_full = bars, stage_empty = bars + 8 * L::kStages;
    const uint32_t q_full = bars + 16 * L::kStages, s_full = q_full + 16, p_ready = s_full + 16, o_full = p_ready + 32,
                   drain = o_full + 16;
    const uint32_t tmem_slot = drain + 8;
    volatile int* const abort = reinterpret_cast<volatile int*>(dynamic_smem + (tmem_slot + 4 - smem_addr(dynamic_smem)));
    // Blocks of 16 keys of step j whose page is in the cache, at j % 8: the ring is shorter than that.
    volatile uint32_t* const block_masks = reinterpret_cast<volatile uint32_t*>(dynamic_smem + (tmem_slot + 8 - smem_addr(dynamic_smem)));

    const int warp = threadIdx.x / kWarpSize, lane = threadIdx.x % kWarpSize;
    const AttentionParams& a = p.a;
    if (threadIdx.x == 0) {
        for (int i = 0; i < L::kStages; ++i) {
            mbar_init(stage_full + 8 * i, 1);
            mbar_init(stage_empty + 8 * i, 1);
        }
        for (int t = 0; t < 2; ++t) {
            mbar_init(q_full + 8 * t, 1);
            mbar_init(s_full + 8 * t, 1);
            mbar_init(p_ready + 16 * t, 4);
            mbar_init(p_ready + 16 * t + 8, 4);
            mbar_init(o_full + 8 * t, 1);
        }
        mbar_init(drain, 1);
        *abort = 0;
        fence_mbar_init();
    }
    if (warp == 9 && lane == 0) {
        prefetch_tensor_map(&q_map);
        prefetch_tensor_map(&k_map);
        prefetch_tensor_map(&v_map);
    }
    if (warp == 8) tmem_alloc(tmem_slot);
    grid_dependency_wait();
    grid_launch_dependents();
    TileItem* const shared_item = reinterpret_cast<TileItem*>(dynamic_smem + (smem + L::kItemBase - smem_addr(dynamic_smem)));
    if (threadIdx.x == 0) *shared_item = tile_item(p);
    tcgen05_fence_before();
    __syncthreads();
    tcgen05_fence_after();
    const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(dynamic_smem + (tmem_slot - smem_addr(dynamic_smem)));

    const volatile TileItem& item = *shared_item;
    const bool work = item.work != 0;
    if (warp >= 8) {
      warpgroup_leave_registers<kOtherRegisters>();
      if (work && warp == 9) {
        // Producer. Lane l loads box l % boxes, half l / boxes of a stage.
        const int boxes = kTileKeys / p.box_keys;
        const uint32_t box_bytes = static_cast<uint32_t>(p.box_keys) * 128u;
        const int32_t* table = a.tables + item.seq * a.table_row;
        if (lane == 0 && item.steps > 0) {
            const uint32_t rows = static_cast<uint32_t>(p.tile_tokens) * a.group;
            for (int t = 0; t < item.tiles; ++t) {
                mbar_arrive_expect_tx(q_full + 8 * t, L::kHalves * rows * 128u);
                for (int h = 0; h < L::kHalves; ++h) {
                    tma_load_3d(smem + t * L::kTileBytes + h * L::kHalfBytes, &q_map, 64 * h, item.kv_head * a.group,
                                item.begin + item.token0 + t * p.tile_tokens, q_full + 8 * t);
                }
            }
        }
        bool ok = true;
        int loads = 0;
        for (int step = 0; step < item.steps && ok; ++step) {
            const int key0 = item.key0 + step * kTileKeys;
            const int box = lane % boxes, half = lane / boxes;
            const int key = key0 + box * p.box_keys;
            int page = -1;
            const bool wanted = key < item.len && key + p.box_keys > item.first;
            if (wanted) {
                page = table[key / a.page_size];
                if (page < 0 || page >= a.num_pages) {
                    atomicOr(&g_fault_word, kFaultIndexOutOfRange);
                    page = -1;
                }
            }
            // One bit a block of 16 keys: set unless the box's page is missing.
            const uint32_t per_box = p.box_keys / kAttentionBlock;
            uint32_t mask = wanted && page < 0 ? ((1u << per_box) - 1u) << (box * per_box) : 0u;
            mask = ~__reduce_or_sync(0xffffffffu, mask) & ((1u << kTileBoxes) - 1u);
            const uint32_t count = __popc(__ballot_sync(0xffffffffu, page >= 0 && lane < boxes)) * L::kHalves;
            if (lane == 0) block_masks[step % 8] = mask;
            const int in_page = key % a.page_size;
            for (int which = 0; which < 2; ++which, ++loads) {
                const int stage = loads % L::kStages;
                ok = mbar_wait_bounded(stage_empty + 8 * stage, ((loads / L::kStages) & 1) ^ 1, abort, kFaultEmptyBarrierTimeout);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                const uint32_t full = stage_full + 8 * stage;
                if (lane == 0) mbar_arrive_expect_tx(full, count * box_bytes);
                __syncwarp();
                if (page >= 0 && half < L::kHalves) {
                    const uint32_t dst = smem + L::kStageBase + stage * L::kTileBytes + half * L::kHalfBytes + box * box_bytes;
                    tma_load_4d(dst, which == 0 ? &k_map : &v_map, 64 * half, item.kv_head, in_page, page, full);
                }
            }
        }
        if (*abort) {
            // Let every copy issued land before the CTA may leave.
            for (int i = loads - L::kStages > 0 ? loads - L::kStages : 0; i < loads; ++i) {
                mbar_wait_timed(stage_full + 8 * (i % L::kStages), (i / L::kStages) & 1, kFaultCopyDrainTimeout);
            }
            for (int t = 0; t < item.tiles && item.steps > 0; ++t) mbar_wait_timed(q_full + 8 * t, 0, kFaultCopyDrainTimeout);
        }
      } else if (work && warp == 8) {
        // Issuer: the whole warp walks, one elected lane issues.
        const int steps = __shfl_sync(0xffffffffu, item.steps, 0), tiles = __shfl_sync(0xffffffffu, item.tiles, 0);
        constexpr uint32_t kScores = mma_descriptor(kTileRows, kTileKeys, false);
        constexpr uint32_t kOutput = mma_descriptor(kTileRows, kDim, true);
        constexpr uint32_t kHigh = smem_descriptor_high(1024);
        const uint32_t q_low = smem_descriptor_low(smem, 16);
        const uint32_t k_low = smem_descriptor_low(smem + L::kStageBase, 16);
        const uint32_t v_low = smem_descriptor_low(smem + L::kStageBase, L::kHalfBytes);
        bool ok = true;
        const auto wait = [&](uint32_t bar, uint32_t parity) {
            ok = ok && mbar_wait_bounded(bar, parity, abort, kFaultFullBarrierTimeout);
            ok = __all_sync(0xffffffffu, ok);
            tcgen05_fence_after();
            return ok;
        };
        const auto scores = [&](int t, int stage) {
            const uint32_t q = q_low + t * (L::kTileBytes >> 4), k = k_low + stage * (L::kTileBytes >> 4);
            if (elect_lane()) {
#pragma unroll
                for (int i = 0; i < kDim / 16; ++i) {
                    const uint32_t at = (i / 4) * (L::kHalfBytes >> 4) + (i % 4) * 2u;
                    mma_smem(tmem + kTmemScores + 128 * t, smem_descriptor(q + at, kHigh), smem_descriptor(k + at, kHigh), kScores,
                             i > 0);
                }
                mma_commit(s_full + 8 * t);
            }
            __syncwarp();
        };
        const auto output = [&](int t, int stage, int half, bool first) {
            const uint32_t v = v_low + stage * (L::kTileBytes >> 4);
            if (elect_lane()) {
#pragma unroll
                for (int j = 0; j < kTileKeys / 32; ++j) {
                    const int i = half * (kTileKeys / 32) + j;
                    mma_tmem(tmem + kTmemOutput + 128 * t, tmem + kTmemScores + 128 * t + 8 * i,
                             smem_descriptor(v + i * (2048u >> 4), kHigh), kOutput, !first || j > 0);
                }
            }
            __syncwarp();
        };
        const auto commit = [&](uint32_t bar) {
            if (elect_lane()) mma_commit(bar);
            __syncwarp();
        };
        if (steps > 0 && wait(stage_full, 0)) {
            for (int t = 0; t < tiles; ++t) {
                if (!wait(q_full + 8 * t, 0)) break;
                scores(t, 0);
            }
            if (ok && steps > 1) commit(stage_empty);
        }
        int v_stage = 1, v_phase = 0;
        for (int step = 0; step < steps && ok; ++step) {
            const bool more = step + 1 < steps;
            int k_stage = v_stage + 1, k_phase = v_phase;
            if (k_stage == L::kStages) k_stage = 0, k_phase ^= 1;
            if (!wait(stage_full + 8 * v_stage, v_phase)) break;
            if (more && !wait(stage_full + 8 * k_stage, k_phase)) break;
            for (int t = 0; t < tiles; ++t) {
                if (!wait(p_ready + 16 * t, step & 1)) break;
                output(t, v_stage, 0, step == 0);
                if (!wait(p_ready + 16 * t + 8, step & 1)) break;
                output(t, v_stage, 1, false);
                if (more) scores(t, k_stage);
                else commit(o_full + 8 * t);
            }
            // None after the last step's: an arrival must not outlive the CTA.
            if (ok && more) {
                commit(stage_empty + 8 * v_stage);
                commit(stage_empty + 8 * k_stage);
            }
            v_stage = k_stage + 1, v_phase = k_phase;
            if (v_stage == L::kStages) v_stage = 0, v_phase ^= 1;
        }
        if (*abort) {
            commit(drain);
            mbar_wait_timed(drain, 0, kFaultCopyDrainTimeout);
        }
      }
    } else {
      warpgroup_take_registers<kSoftmaxRegisters>();
      if (work) {
        // Softmax of tile t; this thread's row is r = token (in the tile) * group + head.
        const int t = warp >> 2;
        if (t < item.tiles) {
            const int r = (warp & 3) * kWarpSize + lane;
            const uint32_t lanes = static_cast<uint32_t>(warp & 3) << 21;
            const uint32_t s_tmem = tmem + lanes + kTmemScores + 128 * t, o_tmem = tmem + lanes + kTmemOutput + 128 * t;
            const int in_tile = r / a.group;
            const int token = min(item.token0 + t * p.tile_tokens + in_tile, item.new_tokens - 1);
            const bool real = in_tile < p.tile_tokens && item.token0 + t * p.tile_tokens + in_tile < item.new_tokens;
            const int position = item.true_len - item.new_tokens + token;
            const int see_first = position >= a.window ? position - a.window + 1 : 0;
            const int see_stop = min(position + 1, item.len);
            float top = -INFINITY, sum = 0.0f;
            bool ok = true;
            for (int step = 0; step < item.steps; ++step) {
                ok = mbar_wait_bounded(s_full + 8 * t, step & 1, abort, kFaultFullBarrierTimeout);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                tcgen05_fence_after();
                float s[4][32];
#pragma unroll
                for (int c = 0; c < 4; ++c) tmem_load_32(s_tmem + 32 * c, s[c]);
                const int key0 = item.key0 + step * kTileKeys;
                const int begin = see_first - key0, end = see_stop - key0;
                const uint32_t mask = block_masks[step % 8];
                const bool partial = begin > 0 || end < kTileKeys || mask != (1u << kTileBoxes) - 1u;
                tmem_wait_loads();
                const bool any_partial = __any_sync(0xffffffffu, partial);
                if (any_partial) {
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
#pragma unroll
                        for (int i = 0; i < 32; ++i) {
                            const int key = 32 * c + i;
                            if (key < begin || key >= end || !(mask >> (key / kAttentionBlock) & 1u)) s[c][i] = -INFINITY;
                        }
                    }
                }
                float m4[4];
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    m4[c] = s[c][0];
#pragma unroll
                    for (int i = 1; i < 31; i += 2) m4[c] = max3(m4[c], s[c][i], s[c][i + 1]);
                    m4[c] = max3(m4[c], s[c][31], s[c][31]);
                }
                const float m = max3(max3(m4[0], m4[1], m4[2]), m4[3], m4[3]) * a.scale_log2;
                // Move the reference point when it is left behind by more than 2^8, and to NaN if a score is.
                const bool move = real && !(m <= top + 8.0f);
                if (__any_sync(0xffffffffu, move)) {
                    const float keep = move ? exp2_approx(top - m) : 1.0f;
                    if (move) {
                        sum *= keep;
                        top = m;
                    }
                    if (step > 0) {
#pragma unroll
                        for (int c = 0; c < kDim / 32; ++c) {
                            float o[32];
                            tmem_load_32(o_tmem + 32 * c, o);
                            tmem_wait_loads();
#pragma unroll
                            for (int i = 0; i < 32; ++i) o[i] *= keep;
                            tmem_store_32(o_tmem + 32 * c, o);
                        }
                    }
                }
                const float shift = top == -INFINITY ? 0.0f : top;
                if (t == 0 && (key0 < item.first || key0 + kTileKeys > item.len || mask != (1u << kTileBoxes) - 1u)) {
                    // Value rows that no token sees may hold anything, NaN included: they become zeros before
                    // the product, which would carry a NaN into every row.
                    const int load = 2 * step + 1, stage = load % L::kStages;
                    ok = mbar_wait_bounded(stage_full + 8 * stage, (load / L::kStages) & 1, abort, kFaultFullBarrierTimeout);
                    ok = __all_sync(0xffffffffu, ok);
                    if (!ok) break;
                    const int key = key0 + r;
                    if (key < item.first || key >= item.len || !(mask >> (r / kAttentionBlock) & 1u)) {
                        const uint32_t row = smem + L::kStageBase + stage * L::kTileBytes + r * 128u;
#pragma unroll
                        for (int h = 0; h < L::kHalves; ++h) {
#pragma unroll
                            for (int i = 0; i < 8; ++i) sts_pairs(row + h * L::kHalfBytes + 16u * i, 0ull, 0ull);
                        }
                    }
                    fence_async_shared();
                }
                const F32x2 scale = f32x2_make(a.scale_log2, a.scale_log2), minus_shift = f32x2_make(-shift, -shift);
                F32x2 sums[2] = {0ull, 0ull};
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    uint32_t w[16];
                    if (any_partial) tile_weights<0>(s[c], scale, minus_shift, w, sums);
                    else tile_weights<kTilePolynomial>(s[c], scale, minus_shift, w, sums);
                    tmem_store_16(s_tmem + 16 * c, w);
                    if (c & 1) {
                        // Half of the weights are there: their product can begin.
                        tmem_wait_stores();
                        tcgen05_fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(p_ready + 16 * t + 8 * (c >> 1));
                    }
                }
                float parts[4];
                f32x2_split(sums[0], parts[0], parts[1]);
                f32x2_split(sums[1], parts[2], parts[3]);
                sum += (parts[0] + parts[1]) + (parts[2] + parts[3]);
            }
            if (ok && item.steps > 0) {
                ok = mbar_wait_bounded(o_full + 8 * t, 0, abort, kFaultFullBarrierTimeout);
                ok = __all_sync(0xffffffffu, ok);
                tcgen05_fence_after();
            }
            if (ok) {
                const float inverse = sum > 0.0f || sum != sum ? 1.0f / sum : 0.0f;
                const int head = item.kv_head * a.group + r - in_tile * a.group;
                uint16_t* out = a.out + static_cast<int64_t>(item.begin + token) * a.out_token + head * a.out_head;
#pragma unroll
                for (int c = 0; c < kDim / 32; ++c) {
                    float o[32] = {};
                    if (item.steps > 0) {
                        tmem_load_32(o_tmem + 32 * c, o);
                        tmem_wait_loads();
                    }
                    if (!real) continue;
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        if (32 * c + 8 * i >= a.dim) break;
                        U32x4 v;
#pragma unroll
                        for (int j = 0; j < 4; ++j) v.v[j] = pack_bf16x2(o[8 * i + 2 * j] * inverse, o[8 * i + 2 * j + 1] * inverse);
                        st_v4(out + 32 * c + 8 * i, v);
                    }
                }
            }
            tmem_wait_stores();
        }
    }
    }
    tcgen05_fence_before();
    __syncthreads();
    tcgen05_fence_after();
    if (warp == 8) tmem_free(tmem);
}

}  // namespace ipl
