// What the forward and the backward pass of attention with a relative position bias share: arguments, the bias table in LDS, the key mask, the layout
// of a tile.
#pragma once
#include "common.hpp"
#include "turned_tile.hpp"

namespace aether {

constexpr int RB_D = 64;              // head dimension
constexpr int RB_KV = 64;             // keys of a tile
constexpr int RB_TILE = RB_KV * RB_D * 2;
constexpr int RB_MAX_BORDERS = 64;
constexpr int RB_MAX_REACH = 1024;    // largest distance whose bucket may differ from the farthest one's
constexpr int RB_MAX_S = 65536;
constexpr int RB_BUF = 2 * RB_TILE;   // two tiles that are staged together
constexpr int RB_PAD = 96;            // >= 31 + 63: a wave's 32 rows against the 64 of a tile
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

// The bias of one head over d, in LDS in log2 units: tab[d + reach + pad], d in [-reach - pad, reach + pad] (pad = RB_PAD); the pad lets a tile that straddles the
// reach read past it without a clamp.
AE_DEV void rb_fill_table(const RbArgs& p, int h, float* tab, int nthreads) {
    const int n_tab = 2 * (p.reach + RB_PAD) + 1;
    for (int i0 = threadIdx.x; i0 < n_tab; i0 += 2 * nthreads) {          // two entries at a time: their loads travel together
        bf16_t v[2];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const int d = min(i0 + k * nthreads, n_tab - 1) - p.reach - RB_PAD, n = d < 0 ? -d : d;
            int b = n;
            if (n >= p.near_n) {
                b = p.near_n;
                for (int j = 0; j < p.n_border; ++j) b += p.border[j] <= n;
            }
            b += d > 0 ? p.half : 0;
            v[k] = p.table[(size_t)b * p.H + h];
        }
#pragma unroll
        for (int k = 0; k < 2; ++k)
            if (i0 + k * nthreads < n_tab) {
                const float t = (float)v[k];                              // a finite entry stays finite in log2 units: rows that hold only the type's lowest value are uniform
                tab[i0 + k * nthreads] = fabsf(t) < INFINITY ? fminf(fmaxf(t * RB_LOG2E, -3.3e38f), 3.3e38f) : t;
            }
    }
}

// One bit per key, 64 keys a word.  A lane reads eight mask bytes and writes their bits as one byte.
AE_DEV void rb_fill_words(const unsigned char* mask, int S, unsigned char* words, int nthreads) {
    for (int i = threadIdx.x; i < (S + 63) / 64 * 8; i += nthreads) {
        unsigned char m[8];                                               // all eight loads before the first is looked at
#pragma unroll
        for (int e = 0; e < 8; ++e) m[e] = mask[min(i * 8 + e, S - 1)];
        unsigned bits = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) bits |= (m[e] != 0 && i * 8 + e < S ? 1u : 0u) << e;
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

// the row of a 32-row half that feeds MFMA row i: the 16 results of a lane are then rows 16(r >> 3) + 8hi + (r & 7), in register order the B operand
// of a product over these rows
AE_DEV int rb_pi(int i) { return 16 * (i >> 4) + 8 * ((i >> 2) & 1) + 4 * ((i >> 3) & 1) + (i & 3); }

// offsets of a lane's A fragments from a tile: rows in the order pi, 16 ks + 8 hi ... + 7
AE_DEV void rb_row_offsets(int lane, int (&off)[4]) {
    const int r = rb_pi(lane & 31), hi = lane >> 5;
#pragma unroll
    for (int ks = 0; ks < 4; ++ks) off[ks] = r * 128 + (((2 * ks + hi) ^ tt_swz(r)) << 4);
}
// Makes the wait for a fragment's loads happen here.  Left to its first use inside a loop, the compiler counts it together with the loop's own tile loads
// and waits for those too.
AE_DEV void rb_arrived(bf16x8 (&f)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) asm volatile("" : "+v"(f[i]));
}

// zeroes the elements of a fragment of eight rows whose bit is not set
AE_DEV bf16x8 rb_keep(bf16x8 f, unsigned bits) {
    uint4 u = __builtin_bit_cast(uint4, f);
    u.x &= (bits & 1 ? 0xffffu : 0u) | (bits & 2 ? 0xffff0000u : 0u);
    u.y &= (bits & 4 ? 0xffffu : 0u) | (bits & 8 ? 0xffff0000u : 0u);
    u.z &= (bits & 16 ? 0xffffu : 0u) | (bits & 32 ? 0xffff0000u : 0u);
    u.w &= (bits & 64 ? 0xffffu : 0u) | (bits & 128 ? 0xffff0000u : 0u);
    return __builtin_bit_cast(bf16x8, u);
}

// a lane's column of a 64 x 32 result (rows d = 32dt + 8(r >> 2) + 4hi + (r & 3)) times `f` -> 64 bf16 at `row`, in 16-byte pieces
AE_DEV void rb_store(const f32x16 (&o)[2], float f, bf16_t* row, int hi, bool ok) {
#pragma unroll
    for (int dt = 0; dt < 2; ++dt) {
        unsigned pk[4][2];
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            pk[g][0] = pack_bf16x2(o[dt][4 * g + 0] * f, o[dt][4 * g + 1] * f);
            pk[g][1] = pack_bf16x2(o[dt][4 * g + 2] * f, o[dt][4 * g + 3] * f);
        }
#pragma unroll
        for (int g = 0; g < 4; g += 2) {
            auto r0 = __builtin_amdgcn_permlane32_swap(pk[g][0], pk[g + 1][0], false, false);
            auto r1 = __builtin_amdgcn_permlane32_swap(pk[g][1], pk[g + 1][1], false, false);
            if (ok) *(uint4*)(row + 32 * dt + 8 * g + 8 * hi) = make_uint4(r0[0], r1[0], r0[1], r1[1]);
        }
    }
}

// The transposed fragments of 32 rows of a tile: f[s][dt] holds column 32 dt + (lane & 31), rows 16 s + 8hi ... + 7.  The transposing LDS read moves a 4 x 16 piece
// per 16 lanes: lane 4r + c names row r, elements 4c ... 4c + 3, and lane i receives column i.
AE_DEV void rb_read_tr(bf16x8 (&f)[2][2], const char* at, const int (&off)[2][2]) {
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
        for (int dt = 0; dt < 2; ++dt) f[s][dt] = tt_read(at + 2048 * s, off[dt]);
}

// Three buffers of two tiles: while one is worked on, the next one is complete or arriving, and the one after it is issued.
constexpr int RB_RING = 3 * RB_BUF;
AE_DEV int rb_next(int buf) { return buf == 2 * RB_BUF ? 0 : buf + RB_BUF; }   // buffers by their offsets
AE_DEV void rb_reads_done_barrier() {
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

}  // namespace aether

struct AetherRelbias;
namespace aether {
inline size_t rb_table_bytes(int reach) { return (size_t)((2 * (reach + RB_PAD) + 1) * 4 + 15) / 16 * 16; }
inline size_t rb_words_bytes(const RbArgs& p) { return p.mask ? (size_t)(p.S + 63) / 64 * 8 : 0; }
int rb_setup(RbArgs& p, const AetherRelbias* d);   // fills the arguments; an error code and its message where the call is refused
int rb_tensor(RbTensor& t, const void* ptr, const long* strides, int S);
// waves of a workgroup (32 rows each): four where that still gives every CU a workgroup or the sequence is long enough for the pipelined loop, else fewer
inline int rb_waves(const RbArgs& p) { return p.S <= 32 ? 1 : p.S >= 448 || (p.S > 64 && (long)p.B * p.H * ((p.S + 127) / 128) >= 256) ? 4 : 2; }
}  // namespace aether
