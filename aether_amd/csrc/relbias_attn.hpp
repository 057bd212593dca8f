// What the forward and the backward pass of attention with a relative position bias share: arguments, the bias table in LDS, the key mask.
#pragma once
#include "common.hpp"

namespace aether {

constexpr int RB_D = 64;              // head dimension
constexpr int RB_KV = 64;             // keys of a tile
constexpr int RB_TILE = RB_KV * RB_D * 2;
constexpr int RB_MAX_BORDERS = 64;
constexpr int RB_MAX_REACH = 1024;    // largest distance whose bucket may differ from the farthest one's
constexpr int RB_MAX_S = 65536;
constexpr float RB_LOG2E = 1.4426950408889634f;

// [B, S, H, 64] with any strides (elements); the last one is 1
struct RbTensor { const bf16_t* p; long sb, ss, sh; };

struct RbArgs {
    RbTensor q, k, v;
    const bf16_t* table; int H;       // [2 * half][H]
    const unsigned char* mask; long mask_sb;   // [B][S], 0 = the key does not count; or null
    int B, S;
    float c;                          // scale · log2(e): scores are kept in the log2 domain
    // bucket of d = key - query: n = |d|;  (d > 0 ? half : 0) + (n < near ? n : near + #{border <= n})
    int half, near_n, n_border, reach;   // reach: from this distance on the bucket is the last one
    int border[RB_MAX_BORDERS];
    int nqb;                          // query blocks per (batch, head)
};

// The bias of one head over d, in LDS in log2 units: tab[d + reach + pad], d in [-reach - pad, reach + pad]; the pad lets a tile that straddles the
// reach read past it without a clamp.
template <int PAD>
AE_DEV void rb_fill_table(const RbArgs& p, int h, float* tab, int nthreads) {
    const int n_tab = 2 * (p.reach + PAD) + 1;
    for (int i = threadIdx.x; i < n_tab; i += nthreads) {
        const int d = i - p.reach - PAD, n = d < 0 ? -d : d;
        int b = n;
        if (n >= p.near_n) {
            b = p.near_n;
            for (int j = 0; j < p.n_border; ++j) b += p.border[j] <= n;
        }
        b += d > 0 ? p.half : 0;
        tab[i] = (float)p.table[(size_t)b * p.H + h] * RB_LOG2E;
    }
}

// One bit per key, 64 keys a word.  A lane reads eight mask bytes and writes their bits as one byte.
AE_DEV void rb_fill_words(const unsigned char* mask, int S, unsigned char* words, int nthreads) {
    for (int i = threadIdx.x; i < (S + 63) / 64 * 8; i += nthreads) {
        unsigned bits = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const int key = i * 8 + e;
            bits |= (key < S && mask[min(key, S - 1)] != 0 ? 1u : 0u) << e;
        }
        words[i] = (unsigned char)bits;
    }
}

AE_DEV uint64_t rb_uniform(uint64_t w) {
    return (uint64_t)(unsigned)__builtin_amdgcn_readfirstlane((int)(unsigned)w) | (uint64_t)(unsigned)__builtin_amdgcn_readfirstlane((int)(unsigned)(w >> 32)) << 32;
}

// the keys of tile j that count
AE_DEV uint64_t rb_word(const RbArgs& p, const uint64_t* words, int j) {
    if (p.mask) return rb_uniform(words[j]);
    const int left = p.S - j * RB_KV;
    return left >= 64 ? ~0ull : (1ull << left) - 1;
}

// (d, e) of the transposing LDS read: within 16 lanes, lane 4r + c names row r, elements 4c .. 4c + 3 of a 4 x 16 piece, and lane i receives column i
typedef short s16x4 __attribute__((ext_vector_type(4)));
AE_DEV bf16x8 rb_read_tr(const char* a, const char* b) {
    const s16x4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)a);
    const s16x4 y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)b);
    typedef short s16x8 __attribute__((ext_vector_type(8)));
    const s16x8 v = {x[0], x[1], x[2], x[3], y[0], y[1], y[2], y[3]};
    return __builtin_bit_cast(bf16x8, v);
}

}  // namespace aether
