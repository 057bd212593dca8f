// Gated feed-forward product:  h = act(x Wgᵀ) ⊙ (x Wuᵀ),  x [M, K], Wg and Wu [F, K] (rows are output features), h bf16 [M, F]; act = tanh-GELU or
// SiLU; operands in bf16, or in e4m3 with one scale per row of x, Wg and Wu.  And its backward pass.
//
// One kernel: the W tile of a workgroup holds, for each group of 32 output columns, 32 rows of Wg and the same 32 rows of Wu, so that both products of an
// element end up in the same lane's accumulators; activation, product and rounding happen in registers and neither projection goes to memory
// (for a backward pass both are also written, in fp32: rounding them to bf16 there would cost the gradients as much again as rounding the
// gradients does).
//
// Main loop: 8 waves as WM x WN; a wave owns MT·32 rows and 32 pairs of columns on v_mfma_f32_32x32x16_bf16, or v_mfma_..._32x32x64_f8f6f4 for e4m3.  A K tile is
// 128 bytes of every row either way.  Tiles come by 16-byte LDS-DMA into two buffers; 128-byte LDS rows are XOR-swizzled in 16-byte chunks.  The two
// waves that share a SIMD alternate: one reads its next fragments and issues the next tile's DMA while the other feeds the matrix pipe.
// Measured, F = 10240, K = 4096: 14464 rows in e4m3 930 ... 963 µs, 2520 ... 2610 TFLOP/s (a large library product in 8 bits: 2440); 3616 rows in bf16 500 µs, 1210 TFLOP/s
// (library 1390), and 610 µs writing both projections, 296 MB.
#include <algorithm>
#include <type_traits>
#include "common.hpp"
#include "turned_tile.hpp"
#include "../../include/aether_hip.h"

namespace aether {

typedef unsigned char u8_t;
typedef int i32x8 __attribute__((ext_vector_type(8)));

struct FfArgs {
    const void* x; long ldx;             // elements
    const void* wg; const void* wu; long ldw;
    const float* sx; const float* sg; const float* su;   // e4m3: scale of each row
    bf16_t* h; long ldh;
    float* gu;                           // fp32 [M][2F]: both projections, or null
    int M, F, K;
    unsigned x_bytes, w_bytes;
    int tiles_m, tiles_n;
};

enum { ACT_GELU_TANH = AETHER_ACT_GELU_TANH, ACT_SILU = AETHER_ACT_SILU };

// sigma(t) = 1 / (1 + e^-t)
AE_DEV float ff_sigmoid(float t) { return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-1.4426950408889634f * t)); }
// tanh-GELU(g) = g · sigma(2u), u = sqrt(2/pi) (g + 0.044715 g³): the argument of sigma, and its slope in g
AE_DEV float ff_gelu_arg(float g) { return 1.5957691216057308f * (g + 0.044715f * g * g * g); }
template <int ACT>
AE_DEV float ff_act(float g) {
    return g * ff_sigmoid(ACT == ACT_SILU ? g : ff_gelu_arg(g));
}
// act(g) and act'(g) = s + g s (1 − s) t'(g) with s = sigma(t(g)); where s is 0 or 1 the second term is 0 whatever t' is
template <int ACT>
AE_DEV void ff_act_slope(float g, float& a, float& slope) {
    const float s = ff_sigmoid(ACT == ACT_SILU ? g : ff_gelu_arg(g));
    const float dt = ACT == ACT_SILU ? 1.0f : 1.5957691216057308f * (1.0f + 0.134145f * g * g);
    const float c = s * (1.0f - s);
    a = g * s;
    slope = s + (c == 0.f ? 0.f : g * c * dt);
}

template <class ET> struct FfType;
template <> struct FfType<bf16_t> { static constexpr int SIZE = 2, SLOTS = 4, CHUNKS = 1; };   // per K tile: MFMA steps, 16-byte chunks a lane reads per step
template <> struct FfType<u8_t> { static constexpr int SIZE = 1, SLOTS = 2, CHUNKS = 2; };

AE_DEV f32x16 ff_mfma(const i32x4 (&a)[1], const i32x4 (&b)[1], f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a[0]), __builtin_bit_cast(bf16x8, b[0]), c, 0, 0, 0);
}
AE_DEV f32x16 ff_mfma(const i32x4 (&a)[2], const i32x4 (&b)[2], f32x16 c) {
    const i32x8 x = {a[0][0], a[0][1], a[0][2], a[0][3], a[1][0], a[1][1], a[1][2], a[1][3]};
    const i32x8 y = {b[0][0], b[0][1], b[0][2], b[0][3], b[1][0], b[1][1], b[1][2], b[1][3]};
    return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(x, y, c, 0, 0, 0, 0x7f7f7f7f, 0, 0x7f7f7f7f);   // block scales 2^0
}

// (g, u) of one lane: 16 rows' worth of a 32 x 32 result, column (= row of x) l32, n = 8(r >> 2) + 4hi + (r & 3)
template <class ET, int ACT>
AE_DEV void ff_finish(const FfArgs& p, f32x16 g, f32x16 u, int m, int n0, int hi) {
    const bool ok = m < p.M;
    const size_t row = (size_t)min(m, p.M - 1);
    if constexpr (std::is_same<ET, u8_t>::value) {
        const float sx = p.sx[row];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const f32x4 a = *(const f32x4*)(p.sg + n0 + 8 * q + 4 * hi), b = *(const f32x4*)(p.su + n0 + 8 * q + 4 * hi);
#pragma unroll
            for (int e = 0; e < 4; ++e) { g[4 * q + e] *= sx * a[e]; u[4 * q + e] *= sx * b[e]; }
        }
    }
    if (p.gu && ok) {
        float* const gp = p.gu + row * (2 * (size_t)p.F) + n0 + 4 * hi;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            *(f32x4*)(gp + 8 * q) = f32x4{g[4 * q], g[4 * q + 1], g[4 * q + 2], g[4 * q + 3]};
            *(f32x4*)(gp + p.F + 8 * q) = f32x4{u[4 * q], u[4 * q + 1], u[4 * q + 2], u[4 * q + 3]};
        }
    }
    unsigned pk[4][2];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        pk[q][0] = pack_bf16x2(ff_act<ACT>(g[4 * q]) * u[4 * q], ff_act<ACT>(g[4 * q + 1]) * u[4 * q + 1]);
        pk[q][1] = pack_bf16x2(ff_act<ACT>(g[4 * q + 2]) * u[4 * q + 2], ff_act<ACT>(g[4 * q + 3]) * u[4 * q + 3]);
    }
#pragma unroll
    for (int q = 0; q < 4; q += 2) {
        auto r0 = __builtin_amdgcn_permlane32_swap(pk[q][0], pk[q + 1][0], false, false);
        auto r1 = __builtin_amdgcn_permlane32_swap(pk[q][1], pk[q + 1][1], false, false);
        if (ok) *(uint4*)(p.h + row * p.ldh + n0 + 8 * q + 8 * hi) = make_uint4(r0[0], r1[0], r0[1], r1[1]);
    }
}

template <class ET, int WM, int WN, int MT, int ACT>
__global__ __launch_bounds__(512) void gated_ff_kernel(FfArgs p) {
    static_assert(WM * WN == 8, "8 wavefronts per workgroup");
    constexpr int BM = WM * MT * 32, BN = WN * 32;                    // rows, pairs of columns
    constexpr int X_TILE = BM * 128, W_TILE = WN * 64 * 128, BUF = X_TILE + W_TILE;
    constexpr int X_ROUNDS = BM / 64, W_ROUNDS = WN;
    constexpr int SLOTS = FfType<ET>::SLOTS, CH = FfType<ET>::CHUNKS, ES = FfType<ET>::SIZE;
    __shared__ __attribute__((aligned(16))) char smem[2 * BUF];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, wm = wave / WN, wn = wave % WN, hi = lane >> 5, l32 = lane & 31;
    const int wave_s = __builtin_amdgcn_readfirstlane(wave);
    // XCD-aware remap, then groups of four row tiles x all column tiles, row tile fastest: neighbours share W tiles in their L2
    int tile_m, tile_n;
    {
        const int id = xcd_remap((int)blockIdx.x, p.tiles_m * p.tiles_n);
        const int group = id / (4 * p.tiles_n), gsz = min(4, p.tiles_m - group * 4), in = id - group * 4 * p.tiles_n;
        tile_m = group * 4 + in % gsz;
        tile_n = in / gsz;
    }
    const int m0 = tile_m * BM, n0 = tile_n * BN;

    // ---- staging: a wave-instruction moves 8 rows x 128 bytes; waves 0-3 carry rows of Wg, waves 4-7 the same rows of Wu ----
    const int srow = wave * 8 + (lane >> 3);
    const unsigned schunk = ((lane & 7) ^ ((srow >> 1) & 7)) * 16;
    unsigned x_off[X_ROUNDS], w_off[W_ROUNDS];
#pragma unroll
    for (int r = 0; r < X_ROUNDS; ++r) x_off[r] = (unsigned)min(m0 + r * 64 + srow, p.M - 1) * (unsigned)(p.ldx * ES) + schunk;
#pragma unroll
    for (int r = 0; r < W_ROUNDS; ++r) w_off[r] = (unsigned)min(n0 + r * 32 + (srow & 31), p.F - 1) * (unsigned)(p.ldw * ES) + schunk;
    const buf_rsrc_t x_rsrc = make_buf_rsrc(p.x, p.x_bytes), w_rsrc = make_buf_rsrc(wave_s < 4 ? p.wg : p.wu, p.w_bytes);
    char* const lds_stage = smem + wave_s * 1024;
    const int nk = p.K * ES / 128;
    constexpr int NP = X_ROUNDS + W_ROUNDS, NPART = SLOTS > 2 ? 3 : 1;
    // past the last K tile the staging fetches that tile again, into the buffer that nobody reads any more: no branch, the same counts of loads
    auto stage_part = [&](int kt, int buf, int part, int nparts) {
        const unsigned soff = 128u * (unsigned)min(kt, nk - 1);
        char* const dst = lds_stage + buf * BUF;
#pragma unroll
        for (int r = 0; r < X_ROUNDS; ++r)
            if (r * nparts / NP == part) bglds16(x_rsrc, x_off[r], soff, dst + r * 8192);
#pragma unroll
        for (int r = 0; r < W_ROUNDS; ++r)
            if ((X_ROUNDS + r) * nparts / NP == part) bglds16(w_rsrc, w_off[r], soff, dst + X_TILE + r * 8192);
    };
    // ---- fragments ----
    const int swz = (lane >> 1) & 7;
    const int x_row = (wm * MT * 32 + l32) * 128, w_row = X_TILE + (wn * 64 + l32) * 128;
    i32x4 wf[2][CH], xf[MT][CH];
    auto load_frags = [&](const char* base, int slot) {
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            const int off = ((2 * (slot * CH + c) + hi) ^ swz) << 4;
#pragma unroll
            for (int t = 0; t < 2; ++t) wf[t][c] = *(const i32x4*)(base + w_row + t * 4096 + off);
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) xf[mt][c] = *(const i32x4*)(base + x_row + mt * 4096 + off);
        }
    };
    f32x16 acc[MT][2];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int i = 0; i < 16; ++i) { acc[mt][0][i] = 0.f; acc[mt][1][i] = 0.f; }
    auto mma = [&]() {
        __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int t = 0; t < 2; ++t) acc[mt][t] = ff_mfma(wf[t], xf[mt], acc[mt][t]);
        __builtin_amdgcn_s_setprio(0);
    };
    auto slot_end = [&]() {
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        __builtin_amdgcn_sched_barrier(0);
    };
    stage_part(0, 0, 0, 1);
    drain_and_barrier();
    // Waves 0-3 load in slots 0, 2, 4 ... and compute in 1, 3, 5 ...; waves 4-7 one slot later.  With 2·SLOTS slots a tile, the last read of tile kt − 1 lies in
    // slot 2·SLOTS·kt − 1: its buffer is free for all of tile kt.  The DMA of tile kt + 1 is waited for before the barrier that ends tile kt.
    if (wave_s < 4) {
        for (int kt = 0; kt < nk; ++kt) {
            const char* base = smem + (kt & 1) * BUF;
#pragma unroll
            for (int sl = 0; sl < SLOTS; ++sl) {
                load_frags(base, sl);
                if (sl < NPART) stage_part(kt + 1, (kt + 1) & 1, sl, NPART);
                asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
                slot_end();
                mma();
                if (sl == SLOTS - 1) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
                slot_end();
            }
        }
    } else {
        for (int kt = 0; kt < nk; ++kt) {
            const char* base = smem + (kt & 1) * BUF;
            if (kt > 0) mma();
            slot_end();
#pragma unroll
            for (int sl = 0; sl < SLOTS; ++sl) {
                load_frags(base, sl);
                if (sl < NPART) stage_part(kt + 1, (kt + 1) & 1, sl, NPART);
                if (sl == SLOTS - 1) asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
                else asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
                slot_end();
                if (sl < SLOTS - 1) {
                    mma();
                    slot_end();
                }
            }
        }
        mma();
    }
    const int n = n0 + wn * 32;
    if (n >= p.F) return;                                             // F % 32 == 0: a wave's columns are all in or all out
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) ff_finish<ET, ACT>(p, acc[mt][0], acc[mt][1], m0 + (wm * MT + mt) * 32 + l32, n, hi);
}

// ---- few rows: 16 pairs of columns a workgroup, straight from memory ----------------------------------------------------------------------------
// Bound by reading the weights: every lane loads its 16 bytes of a weight row in the matrix unit's operand layout, with no LDS and no barrier in between.
// A K tile is 128 bytes of 16 rows of Wg and of Wu; the workgroup's waves take every NW-th tile, many loads in flight each, and add up at the end through
// LDS in the order of the waves.  x comes from the caches: MB blocks of 16 rows on v_mfma_f32_16x16x32_bf16 / v_mfma_..._16x16x128_f8f6f4; rows behind the last one
// repeat it.  Measured, 16 rows, F = 8192, K = 2048: 67 MB of weights in 14.5 µs, 4.6 TB/s.
typedef f32x4 FfAcc;
AE_DEV FfAcc ff_mfma16(const i32x4 (&a)[2], const i32x4 (&b)[2], FfAcc c, bf16_t*) {
#pragma unroll
    for (int s = 0; s < 2; ++s) c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a[s]), __builtin_bit_cast(bf16x8, b[s]), c, 0, 0, 0);
    return c;
}
AE_DEV FfAcc ff_mfma16(const i32x4 (&a)[2], const i32x4 (&b)[2], FfAcc c, u8_t*) {
    const i32x8 x = {a[0][0], a[0][1], a[0][2], a[0][3], a[1][0], a[1][1], a[1][2], a[1][3]};
    const i32x8 y = {b[0][0], b[0][1], b[0][2], b[0][3], b[1][0], b[1][1], b[1][2], b[1][3]};
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(x, y, c, 0, 0, 0, 0x7f7f7f7f, 0, 0x7f7f7f7f);
}

template <class ET, int MB, int ACT>      // MB: blocks of 16 rows
__global__ __launch_bounds__(256) void gated_ff_rows_kernel(FfArgs p) {
    constexpr int NW = 4, ES = FfType<ET>::SIZE, UNROLL = MB == 1 ? 4 : 2;
    __shared__ __attribute__((aligned(16))) float part[NW][2][MB][64][4];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l16 = lane & 15, quad = lane >> 4;
    const int n0 = blockIdx.x * 16;
    const int nk = p.K * ES / 128;
    // 16-byte chunks 4s + quad of a 128-byte tile (bf16: k = 32s + 8 quad ... of step s; e4m3: any order will do, the same in both operands)
    const char* const g = (const char*)p.wg + (size_t)(n0 + l16) * p.ldw * ES + quad * 16;
    const char* const u = (const char*)p.wu + (size_t)(n0 + l16) * p.ldw * ES + quad * 16;
    const char* x[MB];
#pragma unroll
    for (int b = 0; b < MB; ++b) x[b] = (const char*)p.x + (size_t)min(b * 16 + l16, p.M - 1) * p.ldx * ES + quad * 16;
    FfAcc ag[MB], au[MB];
#pragma unroll
    for (int b = 0; b < MB; ++b) { ag[b] = FfAcc{0.f, 0.f, 0.f, 0.f}; au[b] = ag[b]; }
    auto step = [&](int kt, auto n_tag) {
        constexpr int N = decltype(n_tag)::value;
        i32x4 wg[N][2], wu[N][2], xv[N][MB][2];
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const size_t at = (size_t)(kt + i * NW) * 128;
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                wg[i][s] = *(const i32x4*)(g + at + 64 * s);
                wu[i][s] = *(const i32x4*)(u + at + 64 * s);
            }
#pragma unroll
            for (int b = 0; b < MB; ++b)
#pragma unroll
                for (int s = 0; s < 2; ++s) xv[i][b][s] = *(const i32x4*)(x[b] + at + 64 * s);
        }
#pragma unroll
        for (int i = 0; i < N; ++i)
#pragma unroll
            for (int b = 0; b < MB; ++b) {
                ag[b] = ff_mfma16(wg[i], xv[i][b], ag[b], (ET*)nullptr);
                au[b] = ff_mfma16(wu[i], xv[i][b], au[b], (ET*)nullptr);
            }
    };
    int kt = wave;
    for (; kt + (UNROLL - 1) * NW < nk; kt += UNROLL * NW) step(kt, std::integral_constant<int, UNROLL>{});
    for (; kt < nk; kt += NW) step(kt, std::integral_constant<int, 1>{});
    // lane (token l16 of block b, columns 4 quad ... + 3)
#pragma unroll
    for (int b = 0; b < MB; ++b) {
        *(FfAcc*)part[wave][0][b][lane] = ag[b];
        *(FfAcc*)part[wave][1][b][lane] = au[b];
    }
    __syncthreads();
    for (int i = threadIdx.x; i < MB * 64; i += 256) {
        const int b = i >> 6, l = i & 63, m = b * 16 + (l & 15), n = n0 + 4 * (l >> 4);
        if (m >= p.M) continue;
        FfAcc a = *(const FfAcc*)part[0][0][b][l], c = *(const FfAcc*)part[0][1][b][l];
#pragma unroll
        for (int w = 1; w < NW; ++w) { a += *(const FfAcc*)part[w][0][b][l]; c += *(const FfAcc*)part[w][1][b][l]; }
        if constexpr (std::is_same<ET, u8_t>::value) {
            const float sx = p.sx[m];
#pragma unroll
            for (int e = 0; e < 4; ++e) { a[e] *= sx * p.sg[n + e]; c[e] *= sx * p.su[n + e]; }
        }
        if (p.gu) {
            *(FfAcc*)(p.gu + (size_t)m * 2 * p.F + n) = a;
            *(FfAcc*)(p.gu + (size_t)m * 2 * p.F + p.F + n) = c;
        }
        *(uint2*)(p.h + (size_t)m * p.ldh + n) = make_uint2(pack_bf16x2(ff_act<ACT>(a[0]) * c[0], ff_act<ACT>(a[1]) * c[1]),
                                                            pack_bf16x2(ff_act<ACT>(a[2]) * c[2], ff_act<ACT>(a[3]) * c[3]));
    }
}

// ---- some rows: small tiles ------------------------------------------------------------------------------------------------------------------------
// 4 or 8 waves as WM x WN over (WM MT 32) rows x (WN 32) pairs of columns; a ring of NS tiles, one barrier a tile.
// Measured, F = 10240, K = 4096 (168 MB of weights): one row 33 µs, 5.1 TB/s, bound by reading them; 226 rows 59 µs, 2.8 TB/s: one round of 160 workgroups, which
// leaves 96 CUs idle and reads x in every one (80 workgroups of this size go through a K tile in 0.5 µs, 160 in 0.9: 8 TB/s of tiles out of the L2s, where the
// kernel above takes 10 with larger tiles).  K split over the idle CUs is not built.  Tried at 226 rows without gain: rings of 2 ... 6 tiles for the weights with
// loading waves of their own, and 256 x 48 tiles, so that 214 CUs share the work (57 µs).
template <class ET, int WM, int WN, int MT, int NS, int ACT>
__global__ __launch_bounds__(WM * WN * 64) void gated_ff_small_kernel(FfArgs p) {
    constexpr int NW = WM * WN;
    static_assert(NW == 4 || NW == 8, "4 or 8 wavefronts per workgroup");
    constexpr int BM = WM * MT * 32, BN = WN * 32;
    constexpr int X_TILE = BM * 128, W_TILE = WN * 64 * 128, BUF = X_TILE + W_TILE;
    constexpr int X_ROUNDS = BM / (8 * NW), W_ROUNDS = WN * 8 / NW;   // 8 rows a wave-instruction
    constexpr int SLOTS = FfType<ET>::SLOTS, CH = FfType<ET>::CHUNKS, ES = FfType<ET>::SIZE;
    extern __shared__ __attribute__((aligned(16))) char smem_small[];
    char* const smem = smem_small;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, wm = wave / WN, wn = wave % WN, hi = lane >> 5, l32 = lane & 31;
    const int wave_s = __builtin_amdgcn_readfirstlane(wave);
    const int id = xcd_remap((int)blockIdx.x, p.tiles_m * p.tiles_n);
    const int tile_n = id / p.tiles_m, tile_m = id - tile_n * p.tiles_m;   // the row tiles of a column tile one after the other: its weights are read once
    const int m0 = tile_m * BM, n0 = tile_n * BN;
    const int srow = wave * 8 + (lane >> 3);
    const unsigned schunk = ((lane & 7) ^ ((srow >> 1) & 7)) * 16;
    unsigned x_off[X_ROUNDS], w_off[W_ROUNDS];
#pragma unroll
    for (int r = 0; r < X_ROUNDS; ++r) x_off[r] = (unsigned)min(m0 + r * (8 * NW) + srow, p.M - 1) * (unsigned)(p.ldx * ES) + schunk;
    // rows 64 c ... + 31 of the W tile are rows 32 c ... of Wg, + 32 ... + 63 the same of Wu: a wave-instruction carries rows of one of them
#pragma unroll
    for (int r = 0; r < W_ROUNDS; ++r) {
        const int row = r * (8 * NW) + srow;
        w_off[r] = (unsigned)min(n0 + (row >> 6) * 32 + (row & 31), p.F - 1) * (unsigned)(p.ldw * ES) + schunk;
    }
    const buf_rsrc_t x_rsrc = make_buf_rsrc(p.x, p.x_bytes), g_rsrc = make_buf_rsrc(p.wg, p.w_bytes), u_rsrc = make_buf_rsrc(p.wu, p.w_bytes);
    const int nk = p.K * ES / 128;
    // The K tile that is fetched next.  The column tiles begin at places of their own and wrap around: one K tile of rows that lie a power of two apart is a few
    // memory channels' work, and all workgroups would ask for the same ones (F = 10240, K = 4096: 48 rows 37.7 -> 36.0 µs, 120 rows 47.7 -> 43.6, 226 58.9 -> 57.7).
    int at = (int)((long)tile_n * nk / p.tiles_n);
    auto stage = [&](int buf) {
        const unsigned soff = 128u * (unsigned)at;
        at = at == nk - 1 ? 0 : at + 1;
        char* const dst = smem + buf * BUF + wave_s * 1024;
#pragma unroll
        for (int r = 0; r < W_ROUNDS; ++r) {
            const bool up = ((r * NW + wave_s) & 4) != 0;
            bglds16(up ? u_rsrc : g_rsrc, w_off[r], soff, dst + X_TILE + r * (NW * 1024));
        }
#pragma unroll
        for (int r = 0; r < X_ROUNDS; ++r) bglds16(x_rsrc, x_off[r], soff, dst + r * (NW * 1024));
    };
    const int swz = (lane >> 1) & 7;
    const int x_row = (wm * MT * 32 + l32) * 128, w_row = X_TILE + (wn * 64 + l32) * 128;
    f32x16 acc[MT][2];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int i = 0; i < 16; ++i) { acc[mt][0][i] = 0.f; acc[mt][1][i] = 0.f; }
    // a ring of NS buffers; past the last K tile the first ones come again, into buffers that nobody reads any more, so that the counts of loads stay the same
    constexpr int PIECES = W_ROUNDS + X_ROUNDS;
#pragma unroll
    for (int i = 0; i < NS - 1; ++i) stage(i);
    int buf = 0;
    for (int kt = 0; kt < nk; ++kt) {
        wait_vmcnt<(NS - 2) * PIECES>();                              // this wave's part of tile kt has landed
        block_barrier();                                              // everybody's; and tile kt - 1 has been read by all
        stage(buf == 0 ? NS - 1 : buf - 1);
        const char* base = smem + buf * BUF;
        buf = buf == NS - 1 ? 0 : buf + 1;
#pragma unroll
        for (int sl = 0; sl < SLOTS; ++sl) {
            i32x4 wf[2][CH], xf[MT][CH];
#pragma unroll
            for (int c = 0; c < CH; ++c) {
                const int off = ((2 * (sl * CH + c) + hi) ^ swz) << 4;
#pragma unroll
                for (int t = 0; t < 2; ++t) wf[t][c] = *(const i32x4*)(base + w_row + t * 4096 + off);
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) xf[mt][c] = *(const i32x4*)(base + x_row + mt * 4096 + off);
            }
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                for (int t = 0; t < 2; ++t) acc[mt][t] = ff_mfma(wf[t], xf[mt], acc[mt][t]);
        }
        wait_lgkmcnt0();
    }
    wait_vmcnt<0>();                                                  // nothing arrives in LDS behind the workgroup's end
    const int n = n0 + wn * 32;
    if (n >= p.F) return;
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) ff_finish<ET, ACT>(p, acc[mt][0], acc[mt][1], m0 + (wm * MT + mt) * 32 + l32, n, hi);
}

// ---- backward ------------------------------------------------------------------------------------------------------------------------------
// dg = dh u act'(g), du = dh act(g), each rounded to bf16 once, as the products' operands (error of the gradients against 64 bits 0.0023, the outputs' own rounding
// 0.0017), as [M][2F] for the product with the weights and transposed, [2F][Mp], for the one with x.  A workgroup turns a 64 x 64 piece through LDS.  Columns
// M ... Mp − 1 of the transposed form are zeros.
template <int ACT>
__global__ __launch_bounds__(256) void gated_ff_dgu_kernel(const float* __restrict__ gu, const bf16_t* __restrict__ dh, long lddh, int M, int F, int Mp,
                                                           bf16_t* __restrict__ dgu, bf16_t* __restrict__ dgut) {
    __shared__ unsigned short t[2][64][66];
    const int nf = (F + 63) / 64, m0 = blockIdx.x / nf * 64, f0 = blockIdx.x % nf * 64;   // (one axis: the others hold 65535 pieces)
    for (int i = threadIdx.x; i < 64 * 16; i += 256) {                // four columns at a time
        const int r = i >> 4, c = (i & 15) * 4, m = m0 + r, f = f0 + c;
        unsigned short g4[4] = {0, 0, 0, 0}, u4[4] = {0, 0, 0, 0};
        if (m < M && f < F) {
            const f32x4 g = *(const f32x4*)(gu + (size_t)m * 2 * F + f), u = *(const f32x4*)(gu + (size_t)m * 2 * F + F + f);
            const u16x4 d = *(const u16x4*)((const unsigned short*)dh + (size_t)m * lddh + f);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                float a, slope;
                ff_act_slope<ACT>(g[e], a, slope);
                const float dd = bf16_bits_to_f32(d[e]);
                g4[e] = f32_to_bf16_bits(dd * u[e] * slope);
                u4[e] = f32_to_bf16_bits(dd * a);
            }
            *(u16x4*)((unsigned short*)dgu + (size_t)m * 2 * F + f) = u16x4{g4[0], g4[1], g4[2], g4[3]};
            *(u16x4*)((unsigned short*)dgu + (size_t)m * 2 * F + F + f) = u16x4{u4[0], u4[1], u4[2], u4[3]};
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) { t[0][r][c + e] = g4[e]; t[1][r][c + e] = u4[e]; }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < 2 * 64 * 16; i += 256) {
        const int which = i >> 10, c = (i >> 4) & 63, r = (i & 15) * 4;
        if (f0 + c >= F) continue;
        u16x4 v;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = t[which][r + e][c];
        *(u16x4*)((unsigned short*)dgut + ((size_t)which * F + f0 + c) * Mp + m0 + r) = v;
    }
}

// out[c][r] = in[r][c] for r < rows, 0 for rows <= r < fill
__global__ __launch_bounds__(256) void transpose_bf16_kernel(const bf16_t* __restrict__ in, long ldi, int rows, int cols, bf16_t* __restrict__ out, long ldo, int fill) {
    __shared__ unsigned short t[64][66];
    const int nc = (cols + 63) / 64, r0 = blockIdx.x / nc * 64, c0 = blockIdx.x % nc * 64;
    for (int i = threadIdx.x; i < 64 * 16; i += 256) {
        const int r = i >> 4, c = (i & 15) * 4;
        u16x4 v = {0, 0, 0, 0};
        if (r0 + r < rows && c0 + c < cols) v = *(const u16x4*)((const unsigned short*)in + (size_t)(r0 + r) * ldi + c0 + c);
#pragma unroll
        for (int e = 0; e < 4; ++e) t[r][c + e] = v[e];
    }
    __syncthreads();
    for (int i = threadIdx.x; i < 64 * 16; i += 256) {
        const int c = i >> 4, r = (i & 15) * 4;
        if (c0 + c >= cols || r0 + r >= fill) continue;        // (fill is a multiple of 4)
        u16x4 v;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = t[r + e][c];
        *(u16x4*)((unsigned short*)out + (size_t)(c0 + c) * ldo + r0 + r) = v;
    }
}

// dx = [dg du] [Wg; Wu] for few rows, without turned copies of the weights: dx[m][c] = Σ_r dgu[m][r] W[r][c], r < F in Wg, the rest in Wu.  The weights' tile, 64 rows
// of BC columns, goes into LDS as it lies in memory and is read transposed; dgu's rows are read as they are.  The sum over r is split over workgroups so
// that all CUs work; their parts, in fp32, are added in order by ff_dx_join_kernel.  Bound by reading the weights: F = 10240, K = 4096, 60 rows 29 µs for
// 168 MB (and 6 to join), 226 rows 56 (and 6).
struct FfDxArgs {
    const bf16_t* dgu;                   // [M][2F]
    const bf16_t *wg, *wu; long ldw;
    bf16_t* dx; long lddx;
    float* part;                         // [splits][M][K], or null: dx itself
    int M, F, K, tiles_m, tiles_c, splits;
    unsigned dgu_bytes, w_bytes;
};
template <int WM, int WC, int MT, int CT>
__global__ __launch_bounds__(WM * WC * 64) void gated_ff_dx_kernel(FfDxArgs p) {
    constexpr int NW = WM * WC, NS = 3, BM = WM * MT * 32, BC = WC * CT * 32;
    constexpr int G_TILE = BM * 128, W_TILE = BC * 128, BUF = G_TILE + W_TILE;
    constexpr int G_ROUNDS = BM / 8 / NW, W_ROUNDS = BC / 8 / NW;
    static_assert(BM % (8 * NW) == 0 && BC % (8 * NW) == 0 && BC % 64 == 0 && NW % 2 == 0, "whole wave-instructions");
    extern __shared__ __attribute__((aligned(16))) char smem_dx[];
    char* const smem = smem_dx;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, hi = lane >> 5, l32 = lane & 31;
    const int wave_s = __builtin_amdgcn_readfirstlane(wave), wm = wave_s / WC, wc = wave_s % WC;
    const int id = xcd_remap((int)blockIdx.x, p.tiles_m * p.tiles_c * p.splits);
    const int tile_m = id % p.tiles_m, rest = id / p.tiles_m;         // the row tiles of one piece of the weights one after the other
    const int tile_c = rest % p.tiles_c, split = rest / p.tiles_c;
    const int m0 = tile_m * BM, c0 = tile_c * BC;
    const int steps = p.F / 32;                                       // of 64 rows of [Wg; Wu]
    const int from = (int)((long)steps * split / p.splits), to = (int)((long)steps * (split + 1) / p.splits);
    const i32x4 g_rsrc = tt_rsrc(p.dgu, p.dgu_bytes), wg_rsrc = tt_rsrc(p.wg, p.w_bytes), wu_rsrc = tt_rsrc(p.wu, p.w_bytes);
    unsigned g_off[G_ROUNDS], w_off[W_ROUNDS];
#pragma unroll
    for (int r = 0; r < G_ROUNDS; ++r) {
        const int row = (r * NW + wave) * 8 + (lane >> 3);
        g_off[r] = (unsigned)min(m0 + row, p.M - 1) * (unsigned)(p.F * 4) + (((lane & 7) ^ ((row >> 1) & 7)) << 4);
    }
#pragma unroll
    for (int r = 0; r < W_ROUNDS; ++r) {                              // piece r NW + wave: 8 rows of 64 columns; columns behind the last ones repeat them
        const int piece = r * NW + wave, row = (piece & 7) * 8 + (lane >> 3);
        w_off[r] = (unsigned)(lane >> 3) * (unsigned)(p.ldw * 2) + (unsigned)min(c0 + (piece >> 3) * 64, p.K - 64) * 2 + (((lane & 7) ^ tt_swz(row)) << 4);
    }
    auto stage = [&](int step, int buf) __attribute__((always_inline)) {
        const int s = min(step, to - 1);                              // past the last one it is fetched again, into a buffer that nobody reads any more
        const unsigned dst = tt_lds(smem) + buf * BUF + wave_s * 1024;
#pragma unroll
        for (int r = 0; r < W_ROUNDS; ++r) {
            const int row = s * 64 + ((r * NW + wave_s) & 7) * 8;     // (F is a multiple of 32: eight rows are of one of the two)
            const bool up = row >= p.F;
            tt_dma16(up ? wu_rsrc : wg_rsrc, w_off[r], (unsigned)(up ? row - p.F : row) * (unsigned)(p.ldw * 2), dst + G_TILE + r * (NW * 1024));
        }
#pragma unroll
        for (int r = 0; r < G_ROUNDS; ++r) tt_dma16(g_rsrc, g_off[r], (unsigned)s * 128u, dst + r * (NW * 1024));
    };
    int toff[2][2];
    tt_offsets(lane, toff);
    const int g_row = (wm * MT * 32 + l32) * 128, swz = (lane >> 1) & 7;
    f32x16 acc[CT][MT];
#pragma unroll
    for (int ct = 0; ct < CT; ++ct)
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int i = 0; i < 16; ++i) acc[ct][mt][i] = 0.f;
#pragma unroll
    for (int i = 0; i < NS - 1; ++i) stage(from + i, i);
    int buf = 0;
    for (int step = from; step < to; ++step) {
        wait_vmcnt<(NS - 2) * (G_ROUNDS + W_ROUNDS)>();               // this wave's part of the tile has landed
        block_barrier();                                              // everybody's; and the tile before it has been read by all
        stage(step + NS - 1, buf == 0 ? NS - 1 : buf - 1);
        const char* const base = smem + buf * BUF;
        buf = buf == NS - 1 ? 0 : buf + 1;
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            bf16x8 w[CT], g[MT];
#pragma unroll
            for (int ct = 0; ct < CT; ++ct) {
                const int col = wc * CT + ct;                         // of 32 columns
                const char* const at = base + G_TILE + (col >> 1) * 8192 + 2048 * s;
                if constexpr (CT == 2) w[ct] = tt_read(at, toff[ct]);
                else {
                    const int off[2] = {wc & 1 ? toff[1][0] : toff[0][0], wc & 1 ? toff[1][1] : toff[0][1]};
                    w[ct] = tt_read(at, off);
                }
            }
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) g[mt] = *(const bf16x8*)(base + g_row + mt * 4096 + (((2 * s + hi) ^ swz) << 4));
#pragma unroll
            for (int ct = 0; ct < CT; ++ct)
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) acc[ct][mt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(w[ct], g[mt], acc[ct][mt], 0, 0, 0);
        }
        wait_lgkmcnt0();
    }
    wait_vmcnt<0>();                                                  // nothing arrives in LDS behind the workgroup's end
    // acc[ct][mt][r]: row m of dx, column 8(r >> 2) + 4hi + (r & 3) of 32
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
        const int c = c0 + (wc * CT + ct) * 32;
        if (c >= p.K) continue;
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
            const int m = m0 + (wm * MT + mt) * 32 + l32;
            if (m >= p.M) continue;
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const f32x4 v = {acc[ct][mt][4 * q], acc[ct][mt][4 * q + 1], acc[ct][mt][4 * q + 2], acc[ct][mt][4 * q + 3]};
                if (p.part) *(f32x4*)(p.part + ((size_t)split * p.M + m) * p.K + c + 8 * q + 4 * hi) = v;
                else *(uint2*)(p.dx + (size_t)m * p.lddx + c + 8 * q + 4 * hi) = make_uint2(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]));
            }
        }
    }
}

__global__ __launch_bounds__(256) void ff_dx_join_kernel(const float* __restrict__ part, int splits, int M, int K, bf16_t* __restrict__ dx, long lddx) {
    const size_t i = ((size_t)blockIdx.x * 256 + threadIdx.x) * 4, n = (size_t)M * K;
    if (i >= n) return;
    f32x4 a = {0.f, 0.f, 0.f, 0.f};
    for (int s0 = 0; s0 < splits; s0 += 8) {                          // eight loads on their way together
        f32x4 v[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = *(const f32x4*)(part + min(s0 + k, splits - 1) * n + i);
#pragma unroll
        for (int k = 0; k < 8; ++k)
            if (s0 + k < splits) a += v[k];
    }
    const size_t m = i / K, c = i - m * K;
    *(uint2*)(dx + m * lddx + c) = make_uint2(pack_bf16x2(a[0], a[1]), pack_bf16x2(a[2], a[3]));
}

// rows of the tile: few rows a small one; the split that fills the CUs (two workgroups of the smallest tile fit one), as far as the parts fit the place of the
// turned weights
// Against a large product on turned copies of the weights (F = 10240, K = 4096, µs, copies included): 226 rows 62 against 505, 1800 rows 339 against 505, 3616 rows
// 631 against 560.  This kernel's tiles are half as wide, so it stays as long as they need one round of the CUs.
static bool ff_dx_direct(int M, int K) { return (long)((M + 255) / 256) * ((K + 127) / 128) <= 256; }
struct FfDxPlan { int rows, splits; };
static FfDxPlan ff_dx_plan(int M, int F, int K) {
    FfDxPlan q;
    q.rows = M <= 64 ? 64 : M <= 128 ? 128 : 256;
    const long tiles = (long)((M + q.rows - 1) / q.rows) * ((K + 127) / 128), want = q.rows == 64 ? 512 : 256;
    const long most = std::max(1l, std::min({(long)F / M, (long)F / 32 / 4, 64l}));
    q.splits = (int)std::min(most, std::max(1l, want / tiles));
    return q;
}

static int ff_check(const void* x, long ldx, const void* wg, const void* wu, long ldw, int M, int F, int K, int act, int size) {
    if (act != ACT_GELU_TANH && act != ACT_SILU) return aether_set_error(AETHER_ERR_ARG, "gated_ff: unknown activation");
    if (M < 0 || F <= 0 || K <= 0) return aether_set_error(AETHER_ERR_SHAPE, "gated_ff: M must not be negative, F and K must be positive");
    if (F % 32 || (long)K * size % 128) return aether_set_error(AETHER_ERR_SHAPE, "gated_ff: F must be a multiple of 32, K of 64 (bf16) or 128 (e4m3)");
    if (M > (1 << 30) || (size_t)M * F >= (1ull << 46)) return aether_set_error(AETHER_ERR_SHAPE, "gated_ff: too many rows");
    if (M == 0) return AETHER_OK;
    if (!x || !wg || !wu) return aether_set_error(AETHER_ERR_ARG, "gated_ff: null operand");
    if (ldx < K || ldw < K) return aether_set_error(AETHER_ERR_SHAPE, "gated_ff: a leading dimension is shorter than a row");
    if (ldx * size % 16 || ldw * size % 16 || (((uintptr_t)x | (uintptr_t)wg | (uintptr_t)wu) & 15)) return aether_set_error(AETHER_ERR_ALIGN, "gated_ff: rows must be 16-byte aligned");
    if ((size_t)F * ldw * size >= (1ull << 32)) return aether_set_error(AETHER_ERR_SHAPE, "gated_ff: a weight must be below 4 GiB (the reach of a buffer descriptor)");
    if ((size_t)ldx * size * 256 >= (1ull << 32)) return aether_set_error(AETHER_ERR_SHAPE, "gated_ff: a row of x is too far from the next");
    return AETHER_OK;
}

// what the products of the backward pass reach; asked for where the projections are written, too
static int ff_bwd_check(int M, int F, int K) {
    const size_t Mp = ((size_t)M + 63) / 64 * 64;
    if (Mp * 2 * F * 2 >= (1ull << 32) || (size_t)2 * F * K * 2 >= (1ull << 32))
        return aether_set_error(AETHER_ERR_SHAPE, "gated_ff: the backward pass takes M·2F and 2F·K elements of 16 bits below 4 GiB each");
    return AETHER_OK;
}

// Which kernel, from the sizes alone.  A tile kernel runs its workgroups in rounds of one a CU; a round's time is that of one workgroup's K loop, measured per
// K tile of 128 bytes (K = 4096, F = 1024 ... 10240, µs): 64 x 64 (rows x pairs of columns) 0.42, 128 x 64 0.6, 128 x 128 and 256 x 64 0.9, the 256 x 128
// kernel with alternating waves 1.45.  The least rounds x time wins; for instance, bf16, F = 10240: 64 rows 36 µs (256 x 128: 91), 128 rows 44 (91), 226 rows
// 58 (92), 300 rows 64 (96), 400 rows 95 with 256 x 128 (the others 110 and more), 1024 rows 184 (199), 2048 rows 300.
// The same times choose for e4m3, whose K tile holds twice the depth: only their ratios count there, and they were not measured for it (F = 10240, K = 4096, µs: 1 row 15, 226 rows 31, 400 rows 41).
// The kernel without tiles splits K over its waves and needs no round: up to 32 rows it is ahead where F / 64 workgroups of the smallest tile leave most CUs
// idle (F = 2048, K = 4096: 1 row 12 µs against 23, 32 rows 18.5 against 23.5; F = 8192, K = 2048: 16 rows 14.5 against 15.3, 32 rows 18.6 against 15.6).
enum FfVariant { FF_ROWS_16, FF_ROWS_32, FF_64X64, FF_128X64, FF_128X128, FF_256X64, FF_256X128 };
static FfVariant ff_variant(int M, int F) {
    if (M <= 16 && F <= 8192) return FF_ROWS_16;
    if (M <= 32 && F <= 4096) return FF_ROWS_32;
    static const struct { FfVariant v; int rows, pairs; float us; } tile[] = {
        {FF_64X64, 64, 64, 0.42f}, {FF_128X64, 128, 64, 0.6f}, {FF_256X64, 256, 64, 0.9f}, {FF_128X128, 128, 128, 0.9f}, {FF_256X128, 256, 128, 1.45f}};
    FfVariant best = FF_256X128;
    float least = 3e38f;
    for (const auto& t : tile) {
        const long groups = (long)((M + t.rows - 1) / t.rows) * ((F + t.pairs - 1) / t.pairs);
        const float us = (float)((groups + 255) / 256) * t.us;
        if (us < least) { least = us; best = t.v; }
    }
    return best;
}

template <class ET>
static int ff_forward(FfArgs p, int act, hipStream_t s) {
    constexpr int ES = FfType<ET>::SIZE;
    p.w_bytes = (unsigned)(((size_t)(p.F - 1) * p.ldw + p.K) * ES);
    // rows in launches whose part of x a buffer descriptor reaches
    const int M = p.M, most = (int)((((1ull << 32) - 1) / ((size_t)p.ldx * ES)) / 256 * 256);
    const FfArgs whole = p;
    for (int m = 0; m < M; m += most) {
        p.M = M - m < most ? M - m : most;
        p.x = (const char*)whole.x + (size_t)m * p.ldx * ES;
        p.sx = whole.sx ? whole.sx + m : nullptr;
        p.h = whole.h + (size_t)m * p.ldh;
        p.gu = whole.gu ? whole.gu + (size_t)m * 2 * p.F : nullptr;
        p.x_bytes = (unsigned)(((size_t)(p.M - 1) * p.ldx + p.K) * ES);
#define FF_LAUNCH(WM, WN, MT)                                                                                                          \
    do {                                                                                                                               \
        p.tiles_m = (p.M + WM * MT * 32 - 1) / (WM * MT * 32);                                                                         \
        p.tiles_n = (p.F + WN * 32 - 1) / (WN * 32);                                                                                   \
        const dim3 grid(p.tiles_m * p.tiles_n);                                                                                        \
        if (act == ACT_SILU) hipLaunchKernelGGL((gated_ff_kernel<ET, WM, WN, MT, ACT_SILU>), grid, dim3(512), 0, s, p);                \
        else hipLaunchKernelGGL((gated_ff_kernel<ET, WM, WN, MT, ACT_GELU_TANH>), grid, dim3(512), 0, s, p);                           \
    } while (0)
#define FF_SMALL(WM, WN, MT)                                                                                                           \
    do {                                                                                                                               \
        constexpr int NS = 3, LDS = NS * (WM * MT * 32 + WN * 64) * 128;                                                               \
        p.tiles_m = (p.M + WM * MT * 32 - 1) / (WM * MT * 32);                                                                         \
        p.tiles_n = (p.F + WN * 32 - 1) / (WN * 32);                                                                                   \
        const dim3 grid(p.tiles_m * p.tiles_n), block(WM * WN * 64);                                                                   \
        const void* f = act == ACT_SILU ? (const void*)gated_ff_small_kernel<ET, WM, WN, MT, NS, ACT_SILU>                             \
                                        : (const void*)gated_ff_small_kernel<ET, WM, WN, MT, NS, ACT_GELU_TANH>;                       \
        if (LDS > 64 * 1024 && hipFuncSetAttribute(f, hipFuncAttributeMaxDynamicSharedMemorySize, LDS) != hipSuccess) {                \
            (void)hipGetLastError();                                                                                                   \
            return aether_set_error(AETHER_ERR_LAUNCH, "gated_ff: the workgroup's LDS could not be set");                              \
        }                                                                                                                              \
        if (act == ACT_SILU) hipLaunchKernelGGL((gated_ff_small_kernel<ET, WM, WN, MT, NS, ACT_SILU>), grid, block, LDS, s, p);        \
        else hipLaunchKernelGGL((gated_ff_small_kernel<ET, WM, WN, MT, NS, ACT_GELU_TANH>), grid, block, LDS, s, p);                   \
    } while (0)
#define FF_ROWS(MB)                                                                                                                    \
    do {                                                                                                                               \
        const dim3 grid(p.F / 16);                                                                                                     \
        if (act == ACT_SILU) hipLaunchKernelGGL((gated_ff_rows_kernel<ET, MB, ACT_SILU>), grid, dim3(256), 0, s, p);                   \
        else hipLaunchKernelGGL((gated_ff_rows_kernel<ET, MB, ACT_GELU_TANH>), grid, dim3(256), 0, s, p);                              \
    } while (0)
        switch (ff_variant(p.M, p.F)) {
            case FF_ROWS_16: FF_ROWS(1); break;
            case FF_ROWS_32: FF_ROWS(2); break;
            case FF_64X64: FF_SMALL(2, 2, 1); break;
            case FF_128X64: FF_SMALL(4, 2, 1); break;
            case FF_128X128: FF_SMALL(2, 4, 2); break;
            case FF_256X64: FF_SMALL(4, 2, 2); break;
            default: FF_LAUNCH(2, 4, 4); break;
        }
#undef FF_ROWS
#undef FF_SMALL
#undef FF_LAUNCH
        int rc = aether_check_launch("gated_ff");
        if (rc) return rc;
    }
    return AETHER_OK;
}

}  // namespace aether

using namespace aether;

extern "C" int aether_gated_ff(const void* x, long ldx, const void* wg, const void* wu, long ldw, void* h, long ldh, float* gu, int M, int F, int K, int act, void* stream) {
    int rc = ff_check(x, ldx, wg, wu, ldw, M, F, K, act, 2);
    if (rc || M == 0) return rc;
    if (!h) return aether_set_error(AETHER_ERR_ARG, "gated_ff: null output");
    if (ldh < F || ldh % 8 || (((uintptr_t)h | (uintptr_t)gu) & 15)) return aether_set_error(AETHER_ERR_ALIGN, "gated_ff: rows of the output must be 16-byte aligned");
    if (gu && (rc = ff_bwd_check(M, F, K)) != AETHER_OK) return rc;
    FfArgs p = {x, ldx, wg, wu, ldw, nullptr, nullptr, nullptr, (bf16_t*)h, ldh, gu, M, F, K};
    return ff_forward<bf16_t>(p, act, (hipStream_t)stream);
}

extern "C" int aether_gated_ff_e4m3(const void* x, long ldx, const float* x_scale, const void* wg, const float* wg_scale, const void* wu, const float* wu_scale, long ldw,
                                    void* h, long ldh, int M, int F, int K, int act, void* stream) {
    int rc = ff_check(x, ldx, wg, wu, ldw, M, F, K, act, 1);
    if (rc || M == 0) return rc;
    if (!h || !x_scale || !wg_scale || !wu_scale) return aether_set_error(AETHER_ERR_ARG, "gated_ff_e4m3: null output or scale");
    if (ldh < F || ldh % 8 || (((uintptr_t)h | (uintptr_t)wg_scale | (uintptr_t)wu_scale) & 15) || ((uintptr_t)x_scale & 3))
        return aether_set_error(AETHER_ERR_ALIGN, "gated_ff_e4m3: rows of the output and the weights' scales must be 16-byte aligned");
    FfArgs p = {x, ldx, wg, wu, ldw, x_scale, wg_scale, wu_scale, (bf16_t*)h, ldh, nullptr, M, F, K};
    return ff_forward<u8_t>(p, act, (hipStream_t)stream);
}

extern "C" size_t aether_gated_ff_bwd_workspace_bytes(int M, int F, int K) {
    if (M <= 0 || F <= 0 || K <= 0) return 0;
    const size_t Mp = ((size_t)M + 63) / 64 * 64;
    return 2 * ((size_t)M * 2 * F + 2 * (size_t)F * Mp + (size_t)K * Mp + (size_t)K * 2 * F) + 4 * 256;
}

extern "C" int aether_gated_ff_bwd(const void* dh, long lddh, const void* x, long ldx, const void* wg, const void* wu, long ldw, const float* gu, void* dx, long lddx,
                                   void* dw, int M, int F, int K, int act, void* workspace, size_t workspace_bytes, void* stream) {
    int rc = ff_check(x, ldx, wg, wu, ldw, M, F, K, act, 2);
    if (rc) return rc;
    if ((!dx && !dw) || (M > 0 && (!dh || !gu))) return aether_set_error(AETHER_ERR_ARG, "gated_ff_bwd: null operand");
    if (M == 0) return aether_set_error(AETHER_ERR_SHAPE, "gated_ff_bwd: no rows");
    if (lddh < F || lddh % 8 || (dx && (lddx < K || lddx % 8)) || (((uintptr_t)dh | (uintptr_t)gu | (uintptr_t)dx | (uintptr_t)dw | (uintptr_t)workspace) & 15))
        return aether_set_error(AETHER_ERR_ALIGN, "gated_ff_bwd: rows must be 16-byte aligned");
    if (dx && lddx > 0x7fffffffl) return aether_set_error(AETHER_ERR_SHAPE, "gated_ff_bwd: a row of dx is too far from the next (aether_gemm_bf16 takes 32 bits)");
    rc = ff_bwd_check(M, F, K);
    if (rc) return rc;
    const size_t Mp = ((size_t)M + 63) / 64 * 64;
    if (!workspace || workspace_bytes < aether_gated_ff_bwd_workspace_bytes(M, F, K)) return aether_set_error(AETHER_ERR_ARG, "gated_ff_bwd: workspace too small (aether_gated_ff_bwd_workspace_bytes)");
    hipStream_t s = (hipStream_t)stream;
    auto up = [](char* p) { return (char*)(((uintptr_t)p + 255) & ~(uintptr_t)255); };
    char* w = up((char*)workspace);
    bf16_t* dgu = (bf16_t*)w; w = up(w + (size_t)M * 2 * F * 2);
    bf16_t* dgut = (bf16_t*)w; w = up(w + 2 * (size_t)F * Mp * 2);
    bf16_t* xt = (bf16_t*)w; w = up(w + (size_t)K * Mp * 2);
    bf16_t* wt = (bf16_t*)w;
    auto pieces = [](size_t rows, size_t cols) { return dim3((unsigned)((rows + 63) / 64 * ((cols + 63) / 64))); };   // of 64 x 64
    const dim3 eg = pieces(M, F);
    if (act == ACT_SILU) hipLaunchKernelGGL((gated_ff_dgu_kernel<ACT_SILU>), eg, dim3(256), 0, s, gu, (const bf16_t*)dh, lddh, M, F, (int)Mp, dgu, dgut);
    else hipLaunchKernelGGL((gated_ff_dgu_kernel<ACT_GELU_TANH>), eg, dim3(256), 0, s, gu, (const bf16_t*)dh, lddh, M, F, (int)Mp, dgu, dgut);
    rc = aether_check_launch("gated_ff_bwd");
    if (!rc && dx && ff_dx_direct(M, K)) {
        const FfDxPlan plan = ff_dx_plan(M, F, K);
        FfDxArgs a = {dgu, (const bf16_t*)wg, (const bf16_t*)wu, ldw, (bf16_t*)dx, lddx, plan.splits > 1 ? (float*)wt : nullptr, M, F, K, (M + plan.rows - 1) / plan.rows, (K + 127) / 128,
                      plan.splits, (unsigned)((size_t)M * 4 * F), (unsigned)(((size_t)(F - 1) * ldw + K) * 2)};
        const dim3 grid((unsigned)((long)a.tiles_m * a.tiles_c * a.splits));
#define FF_DX(WM, WC, MT, CT)                                                                                                          \
    do {                                                                                                                               \
        constexpr int LDS = 3 * (WM * MT * 32 + WC * CT * 32) * 128;                                                                   \
        if (hipFuncSetAttribute((const void*)gated_ff_dx_kernel<WM, WC, MT, CT>, hipFuncAttributeMaxDynamicSharedMemorySize, LDS) != hipSuccess) { \
            (void)hipGetLastError();                                                                                                   \
            return aether_set_error(AETHER_ERR_LAUNCH, "gated_ff_bwd: the workgroup's LDS could not be set");                          \
        }                                                                                                                              \
        hipLaunchKernelGGL((gated_ff_dx_kernel<WM, WC, MT, CT>), grid, dim3(WM * WC * 64), LDS, s, a);                                 \
    } while (0)
        if (plan.rows == 64) FF_DX(1, 4, 2, 1);
        else if (plan.rows == 128) FF_DX(2, 2, 2, 2);
        else FF_DX(4, 2, 2, 2);
#undef FF_DX
        rc = aether_check_launch("gated_ff_dx");
        if (!rc && plan.splits > 1) {
            hipLaunchKernelGGL(ff_dx_join_kernel, dim3((unsigned)(((size_t)M * K / 4 + 255) / 256)), dim3(256), 0, s, (const float*)wt, plan.splits, M, K, (bf16_t*)dx, lddx);
            rc = aether_check_launch("ff_dx_join");
        }
    } else if (!rc && dx) {
        hipLaunchKernelGGL(transpose_bf16_kernel, pieces(F, K), dim3(256), 0, s, (const bf16_t*)wg, ldw, F, K, wt, 2 * (long)F, F);
        hipLaunchKernelGGL(transpose_bf16_kernel, pieces(F, K), dim3(256), 0, s, (const bf16_t*)wu, ldw, F, K, wt + F, 2 * (long)F, F);
        rc = aether_check_launch("gated_ff_bwd (weights turned)");
        if (!rc) rc = aether_gemm_bf16(dgu, 2 * F, wt, 2 * F, dx, (int)lddx, M, K, 2 * F, nullptr, AETHER_EPI_BIAS, nullptr, 0, nullptr, nullptr, 0, 0, 0, nullptr, 0, 0, stream);
    }
    if (!rc && dw) {
        hipLaunchKernelGGL(transpose_bf16_kernel, pieces(M, K), dim3(256), 0, s, (const bf16_t*)x, ldx, M, K, xt, (long)Mp, (int)Mp);
        rc = aether_check_launch("gated_ff_bwd (input turned)");
        // columns in launches whose part of the turned x a buffer descriptor reaches: whole tiles of them, and 64 at least (Mp is below 2^25)
        const size_t reach = ((1ull << 32) - 1) / (2 * Mp), most = std::min((size_t)K, reach >= 256 ? reach / 256 * 256 : reach / 64 * 64);
        for (size_t c = 0; !rc && c < (size_t)K; c += most)
            rc = aether_gemm_bf16(dgut, (int)Mp, xt + c * Mp, (int)Mp, (bf16_t*)dw + c, K, 2 * F, (int)std::min(most, (size_t)K - c), (int)Mp, nullptr, AETHER_EPI_BIAS, nullptr, 0, nullptr, nullptr, 0, 0, 0,
                                  nullptr, 0, 0, stream);
    }
    return rc;
}
