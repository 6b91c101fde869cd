// Attention of many rows over a paged KV cache on the tensor cores (tcgen05), for sm_100a: the formula
// of paged_attention.cuh.
//
// A tile is 128 rows (token, head) that share a key head: floor(128 / group) tokens times the heads of
// the group, so that a group reads its keys once. A CTA takes two tiles of adjacent tokens and walks over
// their keys, 128 at a time:
//   S_t = Q_t K^T (tensor memory)  ->  P_t = exp2(scale S_t - m) (registers)  ->  O_t += P_t V
// with the scores of one tile in the softmax while the tensor core works on the other. Roles:
//   warps 0-3, 4-7   softmax of tile 0 and 1, a row a thread (a lane of tensor memory): no shuffles;
//   warp 8           issues the products;
//   warps 9, 11      load Q and K, and V, page by page (TMA), into a ring of shared-memory stages;
//   warp 10          hands out the work.
// A CTA on every SM takes an equal share of the steps of all pairs of tiles and key heads, laid end to end;
// a pair that a share's border cuts leaves parts in the workspace, which attention_join_rows_kernel adds.
// Against a CTA for each pair, that evens out the last wave (57 pairs x 4 heads on 148 SMs are 1.54 waves)
// and hides each pair's first loads behind the pair before.
// P overwrites the first half of its S; the products are issued in the order P_t V (step j), Q_t K^T (step
// j + 1), which the tensor core keeps, so nothing is overwritten early. The running maximum is only moved
// when it has grown by more than 2^8, which then rescales O in tensor memory: the result is the same, as
// any reference point within the exponents' range is (weights of at most 2^8 lose nothing in 16 bits).
#pragma once

#include "paged_attention.cuh"
#include "silu_and_mul.cuh"
#include "tensor_core.cuh"

namespace ipl {

constexpr int kTileRows = 128;
constexpr int kTileKeys = 128;
constexpr int kTileThreads = 384;  // three warpgroups, among which the registers are split
// Registers a thread: launched with 65536 / 384 rounded down to 168 (64512 in all), of which the two
// softmax warpgroups take 208 and the third keeps 88 (64512 again).
constexpr int kSoftmaxRegisters = 208, kOtherRegisters = 88;
constexpr int kTileHeadKeys = 96;   // weights of a step handed over first, so that their product begins early
constexpr int kTilePolynomial = 2;  // of 16 pairs of weights, by the polynomial (0: 1 % slower, 4: 2 to 5 %, 6: 4 to 6 %)
constexpr int kTileBoxes = kTileKeys / kAttentionBlock;  // boxes of at least 16 keys a tile
constexpr uint32_t kAllBlocks = (1u << kTileBoxes) - 1u;

#ifndef IPL_TEST_TILE_PAIR_COST
#define IPL_TEST_TILE_PAIR_COST 2  // test builds: a cost at which few pairs weigh more than 2^31
#endif
constexpr int kTilePairCost = IPL_TEST_TILE_PAIR_COST;  // of a pair beside its steps (first scores, output), in steps
constexpr int kTileItems = 4;     // ring of work items

struct TileParams {
    AttentionParams a;
    int tile_tokens;  // tokens a tile: 128 / group
    FastDiv32 pair_tokens, page_size;
    int group_reciprocal;  // 65536 / group + 1: row / group of a row below 128 is the product's high half
    int box_keys;     // keys a TMA box: the largest power of two up to 128 that divides the page size
    int units;        // upper bound of the tile pairs of all sequences
    int wide_out;     // rows of output are whole 32-byte sectors
    AttentionParts parts;  // of pairs that several CTAs share
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
    static constexpr uint32_t kItemBase = kBarrierBase + 512;
    static constexpr uint32_t kBytes = kItemBase + kTileItems * 96;
    static constexpr uint32_t kDynamic = kBytes + 1024;  // room to align to 1024
};

// Powers of two of a pair. The special-function units give 16 a cycle and SM, as many as the products of a
// step have scores for each of their cycles, so a part of the pairs is computed on the FMA pipes:
// 2^x = 2^n 2^r, n = x rounded (by adding 1.5 2^23, which leaves n in the low bits), r in [-1/2, 1/2],
// with the polynomial of degree 3 of least relative error for 2^r (7.5e-5 by the Remez exchange, a fiftieth
// of the rounding of a weight to bf16). x is held above -126, so a vanishing weight is 2^-126, not 0, and so is that of
// NaN: rows whose maximum is not finite are seen to where it is taken and at their end.
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

// The lowest n bits (none for n <= 0, all from 32 on).
__device__ __forceinline__ uint32_t bits_below(int n) { return n >= 32 ? ~0u : n <= 0 ? 0u : (1u << n) - 1u; }

// Bit 31 - i: key 32 c + i of a step is seen, one from `begin` to `end` whose block's page is there.
__device__ __forceinline__ uint32_t seen_bits(int c, int begin, int end, uint32_t blocks) {
    const uint32_t there = (blocks >> (2 * c) & 1u ? 0x0000ffffu : 0u) | (blocks >> (2 * c) & 2u ? 0xffff0000u : 0u);
    return __brev(there & bits_below(end - 32 * c) & ~bits_below(begin - 32 * c));
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

// A stretch of steps of a pair. In shared memory, read where it is used, so that it takes no registers.
struct TileItem {
    int work;  // 0: no more
    int seq, first, len;  // keys [first, len) of the sequence may be read
    int kv_head;
    int token, tokens;  // first token of the pair (row of query), number of tokens
    int position;       // of the first token
    int tiles;          // 1 or 2
    int key0;           // of the first step, a multiple of 128
    int steps;
    int slot;           // for parts; -1: the whole pair
    // Running counts before this item, for the phases of the barriers: stage loads, and for each tile steps
    // and items with steps.
    int loads, tile_steps[2], tile_items[2];
};
static_assert(sizeof(TileItem) <= 96, "fits its place in shared memory");

// A pair of tiles as its sequence defines it.
struct TilePair {
    int seq, token, tokens, position, first, len, key0, steps;
};

// Pair number u: sequence s starts at number starts[s] / (tokens a pair) + s, which leaves it room for its own
// rounded up. Returns false for a number that no pair has.
__device__ __forceinline__ bool tile_pair(const TileParams& p, int u, TilePair& pair) {
    const AttentionParams& a = p.a;
    const int pair_tokens = 2 * p.tile_tokens;
    int lo = 0, hi = a.num_seqs - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        // starts[mid] / pair_tokens + mid <= u
        if (a.starts[mid] < static_cast<int64_t>(u - mid + 1) * pair_tokens) lo = mid;
        else hi = mid - 1;
    }
    const int begin = a.starts[lo], new_tokens = min(a.starts[lo + 1], a.num_tokens) - begin;
    const int token0 = (u - (static_cast<int>(fast_div(static_cast<uint32_t>(max(begin, 0)), p.pair_tokens)) + lo)) * pair_tokens;
    if (u >= p.units || begin < 0 || token0 < 0 || token0 >= new_tokens || static_cast<int64_t>(new_tokens) * a.group <= a.short_rows) return false;
    pair.seq = lo;
    pair.token = begin + token0;
    pair.tokens = min(pair_tokens, new_tokens - token0);
    pair.position = a.lens[lo] - new_tokens + token0;
    pair.len = table_bounded_length(a, lo);
    pair.first = pair.position >= a.window ? pair.position - a.window + 1 : 0;
    const int stop = min(pair.position + pair.tokens, pair.len);
    pair.key0 = pair.first / kTileKeys * kTileKeys;
    pair.steps = stop > pair.key0 ? (stop - pair.key0 + kTileKeys - 1) / kTileKeys : 0;
    return true;
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
    const uint32_t q_full = bars + 16 * L::kStages, q_empty = q_full + 16, s_full = q_empty + 8, p_ready = s_full + 16;
    const uint32_t o_full = p_ready + 32, item_full = o_full + 16, item_empty = item_full + 8 * kTileItems;
    const uint32_t drain = item_empty + 8 * kTileItems, tmem_slot = drain + 8;
    const auto at = [&](uint32_t address) { return dynamic_smem + (address - smem_addr(dynamic_smem)); };
    volatile int* const abort = reinterpret_cast<volatile int*>(at(tmem_slot + 4));
    // Blocks of 16 keys of a step whose page is in the cache, at its number % 8: the ring is shorter than that.
    volatile uint32_t* const block_masks = reinterpret_cast<volatile uint32_t*>(at(tmem_slot + 8));
    volatile int* const issued = reinterpret_cast<volatile int*>(at(tmem_slot + 40));  // one past the last load of K and of V, loads of Q's tiles
    volatile TileItem* const items = reinterpret_cast<volatile TileItem*>(at(smem + L::kItemBase));

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
        for (int i = 0; i < kTileItems; ++i) {
            mbar_init(item_full + 8 * i, 1);
            mbar_init(item_empty + 8 * i, 11);
        }
        mbar_init(q_empty, 1);
        mbar_init(drain, 1);
        *abort = 0;
        for (int i = 0; i < 4; ++i) issued[i] = 0;
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

    // This CTA's share of the steps: of the pairs of one key head in their order, then of the next head. The
    // items' memory serves the sums. Pair u weighs its steps and kTilePairCost, all pairs more than 31 bits hold.
    int64_t* const scratch = reinterpret_cast<int64_t*>(at(smem + L::kItemBase));
    int* const found = reinterpret_cast<int*>(scratch + kTileThreads / kWarpSize);  // the pair the share begins in, and its weight before it
    if (threadIdx.x < a.num_seqs) {
        // The searches below go through these one load after the other: bring them near at once.
        asm volatile("prefetch.global.L1 [%0];" ::"l"(a.starts + threadIdx.x));
        asm volatile("prefetch.global.L1 [%0];" ::"l"(a.lens + threadIdx.x));
    }
    const auto weight = [&](int u, TilePair& pair) { return u < p.units && tile_pair(p, u, pair) ? pair.steps + kTilePairCost : 0; };
    // Sum over the CTA up to and with this thread; `total` gets all of it. Over a warp in the value's type: 32 bits
    // hold the weights of 32 pairs.
    const auto sum_through = [&](auto value, int64_t& total) -> int64_t {
        auto in_warp = value;
#pragma unroll
        for (int offset = 1; offset < kWarpSize; offset *= 2) {
            const auto below = __shfl_up_sync(0xffffffffu, in_warp, offset);
            if (lane >= offset) in_warp += below;
        }
        __syncthreads();
        if (lane == kWarpSize - 1) scratch[warp] = in_warp;
        __syncthreads();
        int64_t through = in_warp;
        total = 0;
        for (int i = 0; i < kTileThreads / kWarpSize; ++i) {
            if (i == warp) through += total;
            total += scratch[i];
        }
        return through;
    };
    // In the common case every thread has one pair, whose weight serves both sums.
    TilePair pair = {};
    int own = weight(threadIdx.x, pair);
    int64_t more = 0;
    for (int u = threadIdx.x + kTileThreads; u < p.units; u += kTileThreads) {
        TilePair other;
        more += weight(u, other);
    }
    int64_t through, head_weight;
    if (p.units <= kTileThreads) {
        through = sum_through(own, head_weight);
    } else {
        sum_through(own + more, head_weight);
    }
    const int64_t all_weight = head_weight * a.kv_heads;
    const int64_t share_begin = divide(all_weight * blockIdx.x, gridDim.x), share_end = divide(all_weight * (blockIdx.x + 1), gridDim.x);
    const int begin_head = head_weight > 0 ? static_cast<int>(divide(share_begin, head_weight)) : 0;
    const int64_t begin_weight = share_begin - begin_head * head_weight;
    int64_t before = 0;
    for (int base = 0; share_begin < share_end && base < p.units; base += kTileThreads) {
        int64_t total = 0;
        if (p.units > kTileThreads) {
            own = weight(base + threadIdx.x, pair);
            through = before + sum_through(own, total);
        }
        if (begin_weight < through && begin_weight >= through - own) {
            found[0] = base + threadIdx.x;
            found[1] = static_cast<int>(begin_weight - (through - own));
        }
        before += total;
        if (begin_weight < before) break;
    }
    // The pairs from there on, for the warp that hands out the work: in the last stage, which is loaded into later.
    TilePair* const first_pairs = reinterpret_cast<TilePair*>(at(smem + L::kStageBase + (L::kStages - 1) * L::kTileBytes));
    __syncthreads();
    const int begin_unit = found[0], begin_skip = found[1];
    if (p.units <= kTileThreads && share_begin < share_end) {
        const int place = static_cast<int>(threadIdx.x) - begin_unit;
        if (place >= 0 && place < kWarpSize) {
            pair.seq = own > 0 ? pair.seq : -1;
            first_pairs[place] = pair;
        }
    }
    fence_async_shared();
    tcgen05_fence_before();
    __syncthreads();
    tcgen05_fence_after();
    const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(at(tmem_slot));

    if (warp >= 8) {
      warpgroup_leave_registers<kOtherRegisters>();
      if (warp == 10) {
        // Work: 32 pairs at a time, one a lane; lane 0 writes the items.
        if (lane < 2) p.parts.parts[2 * blockIdx.x + lane].tokens = 0;
        __syncwarp();
        int n = 0;
        const auto put = [&](const TileItem& item) {
            const int place = n % kTileItems;
            bool ok = mbar_poll_bounded(item_empty + 8 * place, ((n / kTileItems) & 1) ^ 1, abort, kFaultEmptyBarrierTimeout);
            ok = __all_sync(0xffffffffu, ok);
            if (ok && lane == 0) {
                volatile int* to = reinterpret_cast<volatile int*>(items + place);
                const int* from = reinterpret_cast<const int*>(&item);
#pragma unroll
                for (int i = 0; i < static_cast<int>(sizeof(TileItem) / 4); ++i) to[i] = from[i];
                mbar_arrive(item_full + 8 * place);
            }
            __syncwarp();
            ++n;
            return ok;
        };
        int64_t left = share_end - share_begin;
        int skip = begin_skip, head = begin_head;
        TileItem item = {};
        bool ok = true;
        for (int base = begin_unit; left > 0 && ok; base += kWarpSize) {
            if (base >= p.units) base = 0, ++head;
            if (head >= a.kv_heads) break;
            TilePair pair = {};
            bool exists;
            if (base == begin_unit && head == begin_head && p.units <= kTileThreads) {
                pair = first_pairs[lane];
                exists = base + lane < kTileThreads && pair.seq >= 0;
            } else {
                exists = tile_pair(p, base + lane, pair);
            }
            for (uint32_t set = __ballot_sync(0xffffffffu, exists); set != 0 && left > 0 && ok; set &= set - 1) {
                const int from = __ffs(set) - 1;
                const int steps = __shfl_sync(0xffffffffu, pair.steps, from), weight = steps + kTilePairCost;
                if (skip >= weight) {
                    skip -= weight;
                    continue;
                }
                const int take = static_cast<int>(left < weight - skip ? left : weight - skip);
                const int step_begin = max(skip - kTilePairCost, 0), step_end = max(skip + take - kTilePairCost, 0);
                const bool mine = steps > 0 ? step_end > step_begin : skip == 0;
                skip = 0;
                left -= take;
                if (!mine) continue;
                item.work = 1;
                item.kv_head = head;
                item.seq = __shfl_sync(0xffffffffu, pair.seq, from);
                item.first = __shfl_sync(0xffffffffu, pair.first, from);
                item.len = __shfl_sync(0xffffffffu, pair.len, from);
                item.token = __shfl_sync(0xffffffffu, pair.token, from);
                item.tokens = __shfl_sync(0xffffffffu, pair.tokens, from);
                item.position = __shfl_sync(0xffffffffu, pair.position, from);
                item.tiles = item.tokens > p.tile_tokens ? 2 : 1;
                item.key0 = __shfl_sync(0xffffffffu, pair.key0, from) + step_begin * kTileKeys;
                item.steps = step_end - step_begin;
                item.slot = -1;
                if (item.steps < steps) {
                    item.slot = 2 * blockIdx.x + (step_begin == 0 ? 1 : 0);
                    if (lane == 0) {
                        p.parts.parts[item.slot] = AttentionPart{item.tokens, item.token, head, step_end == steps};
                    }
                }
                ok = put(item);
                item.loads += 2 * item.steps;
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    if (t < item.tiles) item.tile_steps[t] += item.steps, item.tile_items[t] += item.steps > 0;
                }
            }
        }
        item.work = 0;
        if (ok) put(item);
      } else if (warp == 9 || warp == 11) {
        // Producers of K (and Q) and of V. Lane l loads box l % boxes, half l / boxes of a stage.
        const bool keys = warp == 9;
        const CUtensorMap* const map = keys ? &k_map : &v_map;
        const int boxes = kTileKeys / p.box_keys;
        const uint32_t box_bytes = static_cast<uint32_t>(p.box_keys) * 128u;
        const uint32_t q_bytes = L::kHalves * static_cast<uint32_t>(p.tile_tokens) * a.group * 128u;
        bool ok = true;
        int loads = keys ? 0 : 1, q_loads = 0;  // the next load: K's are the even ones
        const auto load_q = [&](const volatile TileItem& item) {
            bool free = mbar_poll_bounded(q_empty, (q_loads & 1) ^ 1, abort, kFaultEmptyBarrierTimeout);
            free = __all_sync(0xffffffffu, free);
            if (!free) return false;
            ++q_loads;
            const int tiles = item.tiles, head = item.kv_head * a.group, token = item.token;
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                if (t >= tiles) break;
                if (lane == 0) {
                    issued[2 + t] = item.tile_items[t] + 1;
                    mbar_arrive_expect_tx(q_full + 8 * t, q_bytes);
                    for (int h = 0; h < L::kHalves; ++h) {
                        tma_load_3d(smem + t * L::kTileBytes + h * L::kHalfBytes, &q_map, 64 * h, head, token + t * p.tile_tokens,
                                    q_full + 8 * t);
                    }
                }
            }
            __syncwarp();
            return true;
        };
        for (int n = 0;; ++n) {
            const volatile TileItem& item = items[n % kTileItems];
            ok = ok && mbar_poll_bounded(item_full + 8 * (n % kTileItems), (n / kTileItems) & 1, abort, kFaultFullBarrierTimeout);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok || item.work == 0) break;
            const int32_t* table = a.tables + item.seq * a.table_row;
            const int len = item.len, first = item.first, steps = item.steps, kv_head = item.kv_head;
            if (keys && n == 0 && steps > 0) ok = load_q(item);
            for (int step = 0; step < steps && ok; ++step, loads += 2) {
                const int key0 = item.key0 + step * kTileKeys;
                const int box = lane % boxes, half = lane / boxes;
                const int key = key0 + box * p.box_keys;
                int page = -1;
                const int key_page = static_cast<int>(fast_div(static_cast<uint32_t>(key), p.page_size));
                const bool wanted = key < len && key + p.box_keys > first;
                if (wanted) {
                    page = table[key_page];
                    if (page < 0 || page >= a.num_pages) {
                        atomicOr(&g_fault_word, kFaultIndexOutOfRange);
                        page = -1;
                    }
                }
                // One bit a block of 16 keys: set unless the box's page is missing.
                const uint32_t per_box = p.box_keys / kAttentionBlock;
                uint32_t mask = wanted && page < 0 ? ((1u << per_box) - 1u) << (box * per_box) : 0u;
                mask = ~__reduce_or_sync(0xffffffffu, mask) & kAllBlocks;
                const uint32_t count = __popc(__ballot_sync(0xffffffffu, page >= 0 && lane < boxes)) * L::kHalves;
                if (keys && lane == 0) block_masks[(loads / 2) % 8] = mask;
                const int in_page = key - key_page * a.page_size;
#ifdef IPL_TEST_TILE_SKIP_LOAD
                // Test builds: CTA 0 never issues this load, so the waits for it run out.
                if (blockIdx.x == 0 && loads == IPL_TEST_TILE_SKIP_LOAD) continue;
#endif
                const int stage = loads % L::kStages;
                ok = mbar_poll_bounded(stage_empty + 8 * stage, ((loads / L::kStages) & 1) ^ 1, abort, kFaultEmptyBarrierTimeout);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                const uint32_t full = stage_full + 8 * stage;
                if (lane == 0) {
                    issued[keys ? 0 : 1] = loads + 1;
                    mbar_arrive_expect_tx(full, count * box_bytes);
                }
                __syncwarp();
                if (page >= 0 && half < L::kHalves) {
                    const uint32_t dst = smem + L::kStageBase + stage * L::kTileBytes + half * L::kHalfBytes + box * box_bytes;
                    tma_load_4d(dst, map, 64 * half, kv_head, in_page, page, full);
                }
                if (keys && step == 0 && n > 0) {
                    // Q behind the first keys: its place is free when the item before is done with its scores.
                    ok = load_q(item);
                    if (!ok) {
                        loads += 2;
                        break;
                    }
                }
            }
            if (ok && lane == 0) mbar_arrive(item_empty + 8 * (n % kTileItems));
            __syncwarp();
        }
      } else if (warp == 8) {
        // Issuer: the whole warp walks, one elected lane issues.
        constexpr uint32_t kScores = mma_descriptor(kTileRows, kTileKeys, false);
        constexpr uint32_t kOutput = mma_descriptor(kTileRows, kDim, true);
        constexpr uint32_t kHigh = smem_descriptor_high(1024);
        const uint32_t q_low = smem_descriptor_low(smem, 16);
        const uint32_t k_low = smem_descriptor_low(smem + L::kStageBase, 16);
        const uint32_t v_low = smem_descriptor_low(smem + L::kStageBase, L::kHalfBytes);
        bool ok = true;
        const auto wait = [&](uint32_t bar, uint32_t parity) {
            ok = ok && mbar_poll_bounded(bar, parity, abort, kFaultFullBarrierTimeout);
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
        // The products of 16 keys each with weights that are there: from 0 to 5 and 6, 7.
        const auto output = [&](int t, int stage, bool head, bool first) {
            const uint32_t v = v_low + stage * (L::kTileBytes >> 4);
            if (elect_lane()) {
#pragma unroll
                for (int i = 0; i < kTileKeys / 16; ++i) {
                    if ((i < kTileHeadKeys / 16) != head) continue;
                    mma_tmem(tmem + kTmemOutput + 128 * t, tmem + kTmemScores + 128 * t + 8 * i,
                             smem_descriptor(v + i * (2048u >> 4), kHigh), kOutput, !first || i > 0);
                }
            }
            __syncwarp();
        };
        const auto commit = [&](uint32_t bar) {
            if (elect_lane()) mma_commit(bar);
            __syncwarp();
        };
        int stage = 0, phase = 0;  // of the next load to be consumed
        const auto next_stage = [&](int& s, int& f) {
            if (++s == L::kStages) s = 0, f ^= 1;
        };
        int tile_steps[2] = {0, 0}, tile_items[2] = {0, 0};
        for (int n = 0;; ++n) {
            const volatile TileItem& item = items[n % kTileItems];
            if (!wait(item_full + 8 * (n % kTileItems), (n / kTileItems) & 1) || item.work == 0) break;
            const int steps = __shfl_sync(0xffffffffu, item.steps, 0), tiles = __shfl_sync(0xffffffffu, item.tiles, 0);
            if (steps > 0 && wait(stage_full + 8 * stage, phase)) {
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    if (t >= tiles) break;
                    if (!wait(q_full + 8 * t, tile_items[t] & 1)) break;
                    ++tile_items[t];
                    scores(t, stage);
                }
                if (ok) commit(stage_empty + 8 * stage);
                if (ok && steps == 1) commit(q_empty);
                next_stage(stage, phase);
            }
            for (int step = 0; step < steps && ok; ++step) {
                const bool more = step + 1 < steps;
                int k_stage = stage, k_phase = phase;
                next_stage(k_stage, k_phase);
                if (!wait(stage_full + 8 * stage, phase)) break;
                if (more && !wait(stage_full + 8 * k_stage, k_phase)) break;
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    if (t >= tiles) break;
                    if (!wait(p_ready + 16 * t, tile_steps[t] & 1)) break;
                    output(t, stage, true, step == 0);
                    if (!wait(p_ready + 16 * t + 8, tile_steps[t] & 1)) break;
                    ++tile_steps[t];
                    output(t, stage, false, false);
                    if (more) scores(t, k_stage);
                    else commit(o_full + 8 * t);
                }
                if (!ok) break;
                commit(stage_empty + 8 * stage);
                next_stage(stage, phase);
                if (more) {
                    commit(stage_empty + 8 * k_stage);
                    if (step + 2 == steps) commit(q_empty);
                    next_stage(stage, phase);
                }
            }
            if (!ok) break;
            if (lane == 0) mbar_arrive(item_empty + 8 * (n % kTileItems));
            __syncwarp();
        }
        // No product and no arrival outlives the CTA.
        commit(drain);
        mbar_wait_timed(drain, 0, kFaultCopyDrainTimeout);
      }
      __syncwarp();
      // Once the issuer is through, every copy has landed, unless a wait ran out: then let those issued land before the
      // CTA leaves, the last load of each stage, K's (even) or V's (odd), and Q's.
      named_barrier_sync(1, 4 * kWarpSize);
      if (*abort && threadIdx.x == 8 * kWarpSize) {
        for (int stage = 0; stage < L::kStages; ++stage) {
            int last = -1;
            for (int i = stage; i < max(issued[0], issued[1]); i += L::kStages) {
#ifdef IPL_TEST_TILE_SKIP_LOAD
                if (blockIdx.x == 0 && i == IPL_TEST_TILE_SKIP_LOAD) continue;
#endif
                if (i < issued[i & 1]) last = i;
            }
            if (last >= 0) mbar_wait_timed(stage_full + 8 * stage, (last / L::kStages) & 1, kFaultCopyDrainTimeout);
        }
        for (int t = 0; t < 2; ++t) {
            if (issued[2 + t] > 0) mbar_wait_timed(q_full + 8 * t, (issued[2 + t] - 1) & 1, kFaultCopyDrainTimeout);
        }
      }
    } else {
      warpgroup_take_registers<kSoftmaxRegisters>();
      // Softmax of tile t; this thread's row is r = token (in the tile) * group + head.
      const int t = warp >> 2;
      const auto row = [&] {  // of the tile; computed anew where it is used, so that it takes no registers between
          uint32_t tid;
          asm volatile("mov.u32 %0, %%tid.x;" : "=r"(tid));
          return static_cast<int>(tid) % kTileRows;
      };
      const auto row_token = [&](int r) { return r * p.group_reciprocal >> 16; };
      const uint32_t lanes = static_cast<uint32_t>(warp & 3) << 21;
      const uint32_t s_tmem = tmem + lanes + kTmemScores + 128 * t, o_tmem = tmem + lanes + kTmemOutput + 128 * t;
      bool ok = true;
      for (int n = 0;; ++n) {
        const volatile TileItem& item = items[n % kTileItems];
        ok = mbar_poll_bounded(item_full + 8 * (n % kTileItems), (n / kTileItems) & 1, abort, kFaultFullBarrierTimeout);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok || item.work == 0) break;
        if (t < item.tiles) {
            const int tokens = item.tokens, row_in_tile = row_token(row()), in_pair = t * p.tile_tokens + row_in_tile;
            const bool padding = row_in_tile >= p.tile_tokens || in_pair >= tokens;
            const int position = item.position + min(in_pair, tokens - 1);
            const int see_first = position >= a.window ? position - a.window + 1 : 0;
            const int see_stop = min(position + 1, item.len);
            // A row of padding holds anything; its reference point never moves.
            float top = padding ? INFINITY : -INFINITY, sum = 0.0f;
            for (int step = 0; step < item.steps; ++step) {
                const auto key0 = [&] { return item.key0 + step * kTileKeys; };
                const bool edge = __any_sync(0xffffffffu, see_first > key0() || see_stop < key0() + kTileKeys);
                const bool hole = t == 0 && (key0() < item.first || key0() + kTileKeys > item.len);
                ok = mbar_poll_bounded(s_full + 8 * t, (item.tile_steps[t] + step) & 1, abort, kFaultFullBarrierTimeout);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                tcgen05_fence_after();
                // The second half arrives while the first one is searched.
                float s[4][32];
                tmem_load_32(s_tmem, s[0]);
                tmem_load_32(s_tmem + 32, s[1]);
                const uint32_t mask = block_masks[(item.loads / 2 + step) % 8];
                const bool partial = edge || mask != kAllBlocks;
                tmem_wait_loads();
                tmem_load_32(s_tmem + 64, s[2]);
                tmem_load_32(s_tmem + 96, s[3]);
                if (partial) {
                    tmem_wait_loads();
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        uint32_t seen = seen_bits(c, see_first - key0(), see_stop - key0(), mask);
                        // Shifted along, so that each test is of the same bit.
#pragma unroll
                        for (int i = 0; i < 32; ++i) {
                            const uint32_t keep = static_cast<uint32_t>(static_cast<int>(seen) >> 31);
                            s[c][i] = __uint_as_float((__float_as_uint(s[c][i]) & keep) | (0xff800000u & ~keep));
                            seen += seen;
                        }
                    }
                }
                float m4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    if (h == 1) tmem_wait_loads();
#pragma unroll
                    for (int i = 0; i < 64; i += 2) {
                        float& m = m4[(i / 2) % 4];
                        m = max3(m, s[2 * h + i / 32][i % 32], s[2 * h + i / 32][i % 32 + 1]);
                    }
                }
                const float m = max3(max3(m4[0], m4[1], m4[2]), m4[3], m4[3]) * a.scale_log2;
                // Move the reference point when it is left behind by more than 2^8, and to NaN if a score is.
                const bool move = top < INFINITY && !(m <= top + 8.0f);
                if (__any_sync(0xffffffffu, move)) {
                    const float keep = move ? exp2_approx(top - m) : 1.0f;
                    sum = sum * keep + (move ? m - m : 0.0f);  // the polynomial hides +inf and NaN, this does not
                    top = move ? m : top;
                    __syncwarp();
                    if (step > 0) {
#pragma unroll
                        for (int c = 0; c < kDim / 16; ++c) {
                            uint32_t o[16];
                            tmem_load_16(o_tmem + 16 * c, o);
                            tmem_wait_loads();
#pragma unroll
                            for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * keep);
                            tmem_store_16(o_tmem + 16 * c, o);
                        }
                    }
                }
                const float shift = top == -INFINITY ? 0.0f : top;
                if (hole || (t == 0 && mask != kAllBlocks)) {
                    // Value rows that no token sees may hold anything, NaN included: they become zeros before
                    // the product, which would carry a NaN into every row.
                    const int load = item.loads + 2 * step + 1, stage = load % L::kStages;
                    ok = mbar_poll_bounded(stage_full + 8 * stage, (load / L::kStages) & 1, abort, kFaultFullBarrierTimeout);
                    ok = __all_sync(0xffffffffu, ok);
                    if (!ok) break;
                    const int r = row(), key = key0() + r;
                    if (key < item.first || key >= item.len || !(mask >> (r / kAttentionBlock) & 1u)) {
                        const uint32_t row = smem + L::kStageBase + stage * L::kTileBytes + r * 128u;
#pragma unroll
                        for (int h = 0; h < L::kHalves; ++h) {
#pragma unroll
                            for (int i = 0; i < 8; ++i) sts_pairs(row + h * L::kHalfBytes + 16u * ((i + r) % 8), 0ull, 0ull);
                        }
                    }
                    fence_async_shared();
                    __syncwarp();
                }
                const F32x2 scale = f32x2_make(a.scale_log2, a.scale_log2), minus_shift = f32x2_make(-shift, -shift);
                F32x2 sums[2] = {0ull, 0ull};
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    uint32_t w[16];
                    if (partial) tile_weights<0>(s[c], scale, minus_shift, w, sums);
                    else tile_weights<kTilePolynomial>(s[c], scale, minus_shift, w, sums);
                    tmem_store_16(s_tmem + 16 * c, w);
                    if (c >= kTileHeadKeys / 32 - 1) {
                        // The weights of the first keys are there: their product can begin.
                        tmem_wait_stores();
                        tcgen05_fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(p_ready + 16 * t + 8 * (c - (kTileHeadKeys / 32 - 1)));
                        __syncwarp();
                    }
                }
                float parts[4];
                f32x2_split(sums[0], parts[0], parts[1]);
                f32x2_split(sums[1], parts[2], parts[3]);
                sum += (parts[0] + parts[1]) + (parts[2] + parts[3]);
            }
            if (ok && item.steps > 0) {
                ok = mbar_poll_bounded(o_full + 8 * t, item.tile_items[t] & 1, abort, kFaultFullBarrierTimeout);
                ok = __all_sync(0xffffffffu, ok);
                tcgen05_fence_after();
            }
            if (!ok) break;
            // At least 1 where a score was above -inf; what the polynomial adds for -inf alone stays below 2^-64.
            const float inverse = sum > 0x1p-64f || sum != sum ? 1.0f / sum : 0.0f;
            const int r = row(), in_tile = row_token(r);
            const bool real = in_tile < p.tile_tokens && t * p.tile_tokens + in_tile < item.tokens;
            const int slot = item.slot;
            const int64_t part = static_cast<int64_t>(slot) * (2 * kTileRows) + t * kTileRows + r;
            if (slot >= 0) p.parts.stats[part] = make_float2(top, sum);
            uint16_t* out = a.out + static_cast<int64_t>(item.token + t * p.tile_tokens + in_tile) * a.out_token +
                            (item.kv_head * a.group + r - in_tile * a.group) * a.out_head;
#pragma unroll
            for (int c = 0; c < kDim / 32; ++c) {
                float o[32] = {};
                __syncwarp();  // the rows' stores part the warp, tensor memory is read by all of it
                if (item.steps > 0) {
                    tmem_load_32(o_tmem + 32 * c, o);
                    tmem_wait_loads();
                }
                if (!real) continue;
                // 32 bytes a store, whole sectors. (Chunks exchanged between threads, so that a store of the warp
                // wrote 128 bytes a row, took as long: the instructions count here, not the sectors.)
                if (slot >= 0) {
                    float* to = p.parts.sums + part * kDim + 32 * c;
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        U32x8 v;
#pragma unroll
                        for (int j = 0; j < 8; ++j) v.v[j] = __float_as_uint(o[8 * i + j]);
                        st_v8(to + 8 * i, v);
                    }
                    continue;
                }
                U32x8 v[2];
#pragma unroll
                for (int i = 0; i < 16; ++i) v[i / 8].v[i % 8] = pack_bf16x2(o[2 * i] * inverse, o[2 * i + 1] * inverse);
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    uint16_t* to = out + 32 * c + 16 * i;
                    if (p.wide_out) {
                        if (32 * c + 16 * i < a.dim) st_v8(to, v[i]);
                    } else {
                        if (32 * c + 16 * i < a.dim) st_v4(to, U32x4{v[i].v[0], v[i].v[1], v[i].v[2], v[i].v[3]});
                        if (32 * c + 16 * i + 8 < a.dim) st_v4(to + 8, U32x4{v[i].v[4], v[i].v[5], v[i].v[6], v[i].v[7]});
                    }
                }
            }
        }
        // The output has been read before the next item's first product overwrites it: that waits for weights
        // which these threads write later.
        tcgen05_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(item_empty + 8 * (n % kTileItems));
      }
      tmem_wait_stores();
    }
    tcgen05_fence_before();
    __syncthreads();
    tcgen05_fence_after();
    if (warp == 8) tmem_free(tmem);
}

}  // namespace ipl
