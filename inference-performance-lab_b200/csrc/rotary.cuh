// Rotary position embedding for sm_100a, in place or fused with the write of k and v into the pages
// of a KV cache.
//
// Pair i of a head's first R elements turns by the angle of its token's position p:
//   (a, b) := (a cos(p f_i) - b sin(p f_i), b cos(p f_i) + a sin(p f_i)),
// a, b = x[i], x[i + R/2] (half layout) or x[2i], x[2i + 1] (interleaved); cos and sin come from row p
// of an fp32 table [positions, R] (cosines, then sines), in which any scaling for long contexts is
// folded. Elements past R stay as they are. The arithmetic is fp32, each result rounded to bf16 once.
#pragma once

#include "ipl_common.cuh"
#include "silu_and_mul.cuh"

namespace ipl {

constexpr int kRotaryThreads = 256;

struct RotaryParams {
    const int64_t* positions;
    const float* cos_sin;
    int64_t max_position;
    int rot;
    uint32_t tokens;
    uint32_t tokens_per_cta;
    uint16_t* q;
    uint16_t* k;
    const uint16_t* v;  // append only, like everything down to value_*
    const int64_t* slots;
    int64_t num_slots;
    FastDiv32 page_size;
    uint16_t* key_cache;
    uint16_t* value_cache;
    int64_t q_token, q_head, k_token, k_head, v_token, v_head;
    int64_t key_page, key_token, key_head, value_page, value_token, value_head;
    // A token's work in items of one chunk each: the rotated chunks of every q head and k head, then
    // (append) the chunks of k past R and the chunks of v.
    uint32_t q_heads;
    uint32_t rotated_items, passed_items, items;
    FastDiv32 items_div, rot_chunks, pass_chunks, v_chunks;
};

// Turns kPairs pairs: a[i], b[i] by c[i], s[i].
template <int kPairs>
__device__ __forceinline__ void turn_pairs(float* a, float* b, const float* c, const float* s) {
#pragma unroll
    for (int i = 0; i < kPairs; ++i) {
        const float x = a[i], y = b[i];
        a[i] = x * c[i] - y * s[i];
        b[i] = y * c[i] + x * s[i];
    }
}

// kVector: 16-byte chunks (pointers and strides a multiple of 8 elements; R a multiple of 16 in the
// half layout, of 8 interleaved); otherwise one pair (or one element to copy) an item.
template <bool kVector, bool kHalf, bool kAppend>
__global__ void __launch_bounds__(kRotaryThreads) rotary_kernel(const RotaryParams p) {
    constexpr int kChunk = kVector ? 8 : 1;
    grid_dependency_wait();
    grid_launch_dependents();
    const uint32_t first = blockIdx.x * p.tokens_per_cta;
    const uint32_t here = min(p.tokens_per_cta, p.tokens - first);
    for (uint32_t e = threadIdx.x; e < here * p.items; e += kRotaryThreads) {
        const uint32_t local = fast_div(e, p.items_div);
        uint32_t item = e - local * p.items;
        const int64_t token = first + local;
        const int64_t position = p.positions[token];
        if (position < 0 || position >= p.max_position) {
            atomicOr(&g_fault_word, kFaultIndexOutOfRange);
            continue;
        }
        uint16_t* key_row = nullptr;
        int64_t value_offset = 0;
        if constexpr (kAppend) {
            const int64_t slot = p.slots[token];
            if (slot >= p.num_slots) {
                atomicOr(&g_fault_word, kFaultIndexOutOfRange);
                continue;
            }
            if (slot >= 0) {
                const uint32_t page = fast_div(static_cast<uint32_t>(slot), p.page_size);
                const uint32_t offset = static_cast<uint32_t>(slot) - page * p.page_size.divisor;
                key_row = p.key_cache + page * p.key_page + offset * p.key_token;
                value_offset = page * p.value_page + offset * p.value_token;
            }
        }
        if (item < p.rotated_items) {
            uint32_t head = fast_div(item, p.rot_chunks);
            const uint32_t chunk = item - head * p.rot_chunks.divisor;
            uint16_t* src;
            uint16_t* dst;
            if (head < p.q_heads) {
                src = dst = p.q + token * p.q_token + head * p.q_head;
            } else {
                head -= p.q_heads;
                src = dst = p.k + token * p.k_token + head * p.k_head;
                if constexpr (kAppend) {
                    if (key_row == nullptr) continue;
                    dst = key_row + head * p.key_head;
                }
            }
            const float* cos = p.cos_sin + position * p.rot;
            const float* sin = cos + p.rot / 2;
            if constexpr (kVector && kHalf) {
                const uint32_t at = chunk * 8, other = at + p.rot / 2;
                const U32x4 lo = ld_v4(src + at), hi = ld_v4(src + other);
                const U32x4 c0 = ld_shared_ro_v4(cos + at), c1 = ld_shared_ro_v4(cos + at + 4);
                const U32x4 s0 = ld_shared_ro_v4(sin + at), s1 = ld_shared_ro_v4(sin + at + 4);
                float a[8], b[8], c[8], s[8];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    a[2 * i] = bf16_lo(lo.v[i]), a[2 * i + 1] = bf16_hi(lo.v[i]);
                    b[2 * i] = bf16_lo(hi.v[i]), b[2 * i + 1] = bf16_hi(hi.v[i]);
                    c[i] = __uint_as_float(c0.v[i]), c[i + 4] = __uint_as_float(c1.v[i]);
                    s[i] = __uint_as_float(s0.v[i]), s[i + 4] = __uint_as_float(s1.v[i]);
                }
                turn_pairs<8>(a, b, c, s);
                U32x4 out_lo, out_hi;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    out_lo.v[i] = pack_bf16x2(a[2 * i], a[2 * i + 1]);
                    out_hi.v[i] = pack_bf16x2(b[2 * i], b[2 * i + 1]);
                }
                st_v4(dst + at, out_lo);
                st_v4(dst + other, out_hi);
            } else if constexpr (kVector) {
                const U32x4 x = ld_v4(src + chunk * 8);
                const U32x4 c4 = ld_shared_ro_v4(cos + chunk * 4), s4 = ld_shared_ro_v4(sin + chunk * 4);
                U32x4 out;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    float a = bf16_lo(x.v[i]), b = bf16_hi(x.v[i]);
                    const float c = __uint_as_float(c4.v[i]), s = __uint_as_float(s4.v[i]);
                    turn_pairs<1>(&a, &b, &c, &s);
                    out.v[i] = pack_bf16x2(a, b);
                }
                st_v4(dst + chunk * 8, out);
            } else {
                const uint32_t at = kHalf ? chunk : 2 * chunk;
                const uint32_t other = kHalf ? chunk + p.rot / 2 : 2 * chunk + 1;
                float a = bf16_bits_to_float(src[at]), b = bf16_bits_to_float(src[other]);
                turn_pairs<1>(&a, &b, cos + chunk, sin + chunk);
                dst[at] = float_to_bf16_bits(a);
                dst[other] = float_to_bf16_bits(b);
            }
            continue;
        }
        if constexpr (kAppend) {
            if (key_row == nullptr) continue;
            item -= p.rotated_items;
            const uint16_t* src;
            uint16_t* dst;
            if (item < p.passed_items) {
                const uint32_t head = fast_div(item, p.pass_chunks);
                const uint32_t at = p.rot + (item - head * p.pass_chunks.divisor) * kChunk;
                src = p.k + token * p.k_token + head * p.k_head + at;
                dst = key_row + head * p.key_head + at;
            } else {
                item -= p.passed_items;
                const uint32_t head = fast_div(item, p.v_chunks);
                const uint32_t at = (item - head * p.v_chunks.divisor) * kChunk;
                src = p.v + token * p.v_token + head * p.v_head + at;
                dst = p.value_cache + value_offset + head * p.value_head + at;
            }
            if constexpr (kVector) {
                st_v4(dst, ld_v4(src));
            } else {
                *dst = *src;
            }
        }
    }
}

}  // namespace ipl
