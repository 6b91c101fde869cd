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

constexpr int kRotaryMaxThreads = 512;

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
    // A token's work in items of a chunk each: the rotated chunks of the q heads and the k heads, then (append) the
    // chunks of k past R and the chunks of v.
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

// kVector: 16-byte chunks (pointers and strides a multiple of 8 elements; R a multiple of 16 in the half layout, of 8
// interleaved); otherwise one pair (or one element to copy) an item. Bound by HBM in large launches, by the chain of
// loads (position, then its row of the table) in small ones: the elements are loaded ahead of the position. Small
// launches give a token's items a thread each in one CTA; large ones use CTAs of 128 threads, which retire more
// evenly (8192 tokens of 28 + 4 heads of 128, written to pages: 27.3 to 28.0 us, 0.84 to 0.86 of the copy peak, with 256 threads
// 31.7; 64 tokens: 1.9 us, with 128 threads 2.65). Four heads a thread, sharing cosines and sines, measured the same.
template <bool kVector, bool kHalf, bool kAppend>
__global__ void __launch_bounds__(kRotaryMaxThreads) rotary_kernel(const RotaryParams p) {
    constexpr int kChunk = kVector ? 8 : 1;
    grid_dependency_wait();
    grid_launch_dependents();
    const uint32_t first = blockIdx.x * p.tokens_per_cta;
    const uint32_t here = min(p.tokens_per_cta, p.tokens - first);
    for (uint32_t e = threadIdx.x; e < here * p.items; e += blockDim.x) {
        const uint32_t local = fast_div(e, p.items_div);
        uint32_t item = e - local * p.items;
        const int64_t token = first + local;
        const int64_t* position_at = p.positions + token;
        const int64_t* slot_at = p.slots + token;
        uint16_t* key_row = nullptr;
        int64_t value_offset = 0;
        // Whether the token is written: its position and slot are in range. Reads both, sets the places of a slot.
        int64_t position = 0;
        const auto place = [&] {
            position = *position_at;
            bool ok = position >= 0 && position < p.max_position;
            if constexpr (kAppend) {
                const int64_t slot = *slot_at;
                ok = ok && slot < p.num_slots;
                if (ok && slot >= 0) {
                    const uint32_t page = fast_div(static_cast<uint32_t>(slot), p.page_size);
                    const uint32_t offset = static_cast<uint32_t>(slot) - page * p.page_size.divisor;
                    key_row = p.key_cache + page * p.key_page + offset * p.key_token;
                    value_offset = page * p.value_page + offset * p.value_token;
                }
            }
            if (!ok) atomicOr(&g_fault_word, kFaultIndexOutOfRange);
            return ok;
        };
        if (item < p.rotated_items) {
            uint32_t head = fast_div(item, p.rot_chunks);
            const uint32_t chunk = item - head * p.rot_chunks.divisor;
            const bool is_key = head >= p.q_heads;
            if (is_key) head -= p.q_heads;
            uint16_t* const src = is_key ? p.k + token * p.k_token + head * p.k_head : p.q + token * p.q_token + head * p.q_head;
            const auto target = [&]() -> uint16_t* {
                if (!kAppend || !is_key) return src;
                return key_row == nullptr ? nullptr : key_row + head * p.key_head;
            };
            if constexpr (kVector && kHalf) {
                const uint32_t at = chunk * 8, other = at + p.rot / 2;
                const U32x4 lo = ld_v4(src + at), hi = ld_v4(src + other);
                if (!place()) continue;
                const float* cos = p.cos_sin + position * p.rot;
                const float* sin = cos + p.rot / 2;
                const U32x4 c0 = ld_shared_ro_v4(cos + at), c1 = ld_shared_ro_v4(cos + at + 4);
                const U32x4 s0 = ld_shared_ro_v4(sin + at), s1 = ld_shared_ro_v4(sin + at + 4);
                uint16_t* const dst = target();
                if (dst == nullptr) continue;
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
                if (!place()) continue;
                const float* cos = p.cos_sin + position * p.rot;
                const U32x4 c4 = ld_shared_ro_v4(cos + chunk * 4), s4 = ld_shared_ro_v4(cos + p.rot / 2 + chunk * 4);
                uint16_t* const dst = target();
                if (dst == nullptr) continue;
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
                if (!place()) continue;
                uint16_t* const dst = target();
                if (dst == nullptr) continue;
                const float* cos = p.cos_sin + position * p.rot;
                const uint32_t at = kHalf ? chunk : 2 * chunk;
                const uint32_t other = kHalf ? chunk + p.rot / 2 : 2 * chunk + 1;
                float a = bf16_bits_to_float(src[at]), b = bf16_bits_to_float(src[other]);
                turn_pairs<1>(&a, &b, cos + chunk, cos + p.rot / 2 + chunk);
                dst[at] = float_to_bf16_bits(a);
                dst[other] = float_to_bf16_bits(b);
            }
            continue;
        }
        if constexpr (kAppend) {
            item -= p.rotated_items;
            const bool pass = item < p.passed_items;
            if (!pass) item -= p.passed_items;
            const uint32_t head = fast_div(item, pass ? p.pass_chunks : p.v_chunks);
            const uint32_t at = (item - head * (pass ? p.pass_chunks : p.v_chunks).divisor) * kChunk + (pass ? p.rot : 0);
            const uint16_t* src = pass ? p.k + token * p.k_token + head * p.k_head : p.v + token * p.v_token + head * p.v_head;
            if constexpr (kVector) {
                const U32x4 x = ld_v4(src + at);
                if (!place() || key_row == nullptr) continue;
                st_v4((pass ? key_row + head * p.key_head : p.value_cache + value_offset + head * p.value_head) + at, x);
            } else {
                if (!place() || key_row == nullptr) continue;
                (pass ? key_row + head * p.key_head : p.value_cache + value_offset + head * p.value_head)[at] = src[at];
            }
        }
    }
}

}  // namespace ipl
