// Self-attention with a learned bias by bucket of the relative position, forward pass, head dimension 64:
//
//   S_ij = scale · q_i·k_j + T[bucket(j − i), h]  where key j counts,   P = softmax_j(S),   O = P V;   a row without keys gives 0, and one whose keys all score −inf.
//
// gfx950 design
//   * A wave owns 32 queries, a workgroup NW waves of one (batch, head); tiles of 64 keys, K and V by 16-byte LDS-DMA into a ring of three, one barrier a tile.
//     Sᵀ = K·Qᵀ on v_mfma_f32_32x32x16_bf16: a lane holds 32 scores of ONE query.  K rows enter in the order pi, so that the exponentiated scores are, in
//     register order, the B operand of Oᵀ += Vᵀ·Pᵀ; Vᵀ comes out of the row-major tile by ds_read_b64_tr_b16.
//   * The bias depends on key − query alone and is constant beyond `reach` (91 positions for 32 buckets up to 128): a tile that lies beyond it adds ONE
//     number, folded into the fma that scales the scores.  Only the few tiles along the diagonal look their bias up, in a table of 2·reach + 1 floats
//     in LDS, whose addresses are consecutive over the lanes (no bank conflicts).
//   * Soft-max over one pass: the shift of a row is the maximum of its first 32 scores that holds one above -inf; later scores are exponentiated against it
//     and checked afterwards (a lane's partial sum above 2^40, or NaN, makes the wave compute these scores again and take the classic online step).  Any
//     shift gives the same soft-max; the check keeps P·V inside fp32 for |v| up to 1e22.  Sums are fp32; P is rounded to bf16 once, as the operand of P·V
//     (the matrix unit's fp32 products run at a sixteenth of the rate), and without TRAIN the sum adds the rounded values, so that a row of equal values comes out exact.  Relative L2 error
//     against 64 bits 0.0018 ... 0.0021, of which the output's own rounding is 0.0017.
//   * For a backward pass the output is needed beyond bf16: δ = dO·O is subtracted from numbers that may be nearly equal to it.  TRAIN multiplies V with P in
//     two bf16 parts (P = hi + lo to 2^-17) and also stores what the rounding of O left (o_low), so that O + o_low is good to 2^-16.
//   * Keys that do not count: whole tiles are skipped; in a tile that holds some, their scores become −inf and their V elements 0 (a NaN or an infinity
//     behind the mask reaches nothing).
//
// What bounds it.  Long sequences: the matrix and the vector pipe together, about 45% of the former's cycles, with two waves a SIMD (1 x 7993 x 16 heads: 262 GFLOP in
// 287 µs, 910 TFLOP/s where a large library product reaches 1390; tile by tile it took 359).  Many short ones: memory, at 60% of a copy's rate (16 x
// 226 x 64 heads, ragged: 91 MB in 39 µs against 18.5; a workgroup lives for four tiles, of which the first waits for memory, the table and the mask).
#include <type_traits>
#include "relbias_attn.hpp"
#include "../../include/aether_hip.h"

namespace aether {

struct RbFwdArgs { RbArgs a; bf16_t* o; bf16_t* o_low; float* lse; };   // o_low, lse: for a backward pass

// tiles from which the pipelined loop is used: its start and end cost about two tiles' time, its registers the third wave of a SIMD
constexpr int RB_PIPE_TILES = 7;

// beyond this a row's shift is taken off the rounded sum of score and bias, as it was found, so that all of a row's scores round alike
constexpr float RB_FAR_SHIFT = 16384.f;

template <int NW, bool TRAIN, bool PIPE>
__global__ __launch_bounds__(NW * 64) __attribute__((amdgpu_waves_per_eu(PIPE || NW == 1 ? 2 : 3, PIPE || NW == 1 ? 2 : 3))) void relbias_attn_fwd_kernel(RbFwdArgs args) {
    extern __shared__ __attribute__((aligned(16))) char smem[];
    const RbArgs& p = args.a;
    float* const tab = (float*)(smem + RB_RING);
    unsigned char* const words8 = (unsigned char*)(smem + RB_RING + ((2 * (p.reach + RB_PAD) + 1) * 4 + 15) / 16 * 16);
    const uint64_t* const words = (const uint64_t*)words8;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, hi = lane >> 5, l32 = lane & 31;
    const int wave_s = __builtin_amdgcn_readfirstlane(wave);
    const int S = p.S;
    const int wgid = xcd_remap((int)blockIdx.x, p.B * p.H * p.nqb);   // the query blocks of a head share an L2
    const int bh = wgid / p.nqb, qb = wgid - bh * p.nqb;
    const int b = bh / p.H, h = bh - b * p.H;
    const int q0 = qb * (NW * 32) + wave_s * 32;                      // this wave's first query
    const int qrow = q0 + l32;

    bf16x8 qf[4];
    {
        const bf16_t* qp = p.q.p + (size_t)b * p.q.sb + (size_t)h * p.q.sh + (size_t)min(qrow, S - 1) * p.q.ss;
#pragma unroll
        for (int ks = 0; ks < 4; ++ks) qf[ks] = *(const bf16x8*)(qp + 16 * ks + 8 * hi);
    }
    // ---- staging: a wave-instruction moves 8 rows x 128 bytes; rows at or beyond S are outside the descriptor and their keys do not count ----
    const unsigned k_row = (unsigned)p.k.ss * 2, v_row = (unsigned)p.v.ss * 2;
    const i32x4 k_rsrc = tt_rsrc(p.k.p + (size_t)b * p.k.sb + (size_t)h * p.k.sh, (unsigned)(S - 1) * k_row + 128);
    const i32x4 v_rsrc = tt_rsrc(p.v.p + (size_t)b * p.v.sb + (size_t)h * p.v.sh, (unsigned)(S - 1) * v_row + 128);
    unsigned k_off[8 / NW], v_off[8 / NW];
#pragma unroll
    for (int ps = 0; ps < 8 / NW; ++ps) {
        const int r = (ps * NW + wave) * 8 + (lane >> 3), ch = lane & 7;
        k_off[ps] = r * k_row + ((ch ^ tt_swz(r)) << 4);
        v_off[ps] = r * v_row + ((ch ^ tt_swz(r)) << 4);
    }
    auto stage_k = [&](int j, int buf) {
        const unsigned dst = tt_lds(smem) + buf + wave_s * 1024;
#pragma unroll
        for (int ps = 0; ps < 8 / NW; ++ps) tt_dma16(k_rsrc, k_off[ps], (unsigned)j * (RB_KV * k_row), dst + ps * (NW * 1024));
    };
    auto stage_v = [&](int j, int buf) {
        const unsigned dst = tt_lds(smem) + buf + RB_TILE + wave_s * 1024;
#pragma unroll
        for (int ps = 0; ps < 8 / NW; ++ps) tt_dma16(v_rsrc, v_off[ps], (unsigned)j * (RB_KV * v_row), dst + ps * (NW * 1024));
    };
    auto stage = [&](int j, int buf) {
        stage_k(j, buf);
        stage_v(j, buf);
    };
    const int nkv = (S + RB_KV - 1) / RB_KV;
    stage(0, 0);                                                      // on their way while the table and the mask are read; whether their keys count shows later
    if (nkv > 1) stage(1, RB_BUF);
    rb_fill_table(p, h, tab, NW * 64);
    if (p.mask) rb_fill_words(p.mask + (size_t)b * p.mask_sb, S, words8, NW * 64);
    int koff[4], voff[2][2];
    rb_row_offsets(lane, koff);
    tt_offsets(lane, voff);

    f32x16 o[2];
#pragma unroll
    for (int i = 0; i < 16; ++i) { o[0][i] = 0.f; o[1][i] = 0.f; }
    float m_run = 0.f, l_run = 0.f;
    bool started = false, fresh = true;                               // (of the wave) a key was met; (of the row) only scores of -inf were

    rb_arrived(qf);
    drain_and_barrier();                                              // table and words are there, and the first two tiles
    const float far_r = tab[2 * (p.reach + RB_PAD)], far_l = tab[0];
    auto next_tile = [&](int j, uint64_t& w) {                        // the next tile from j on that holds a key, nkv if none does
        for (; j < nkv; ++j)
            if ((w = rb_word(p, words, j)) != 0) break;
        return j;
    };
    // Tile by tile from `first` on, any tile: the tiles in front of it are done.  staged: tiles 0 and 1 are in the first two buffers.
    auto sweep = [&](int first, bool staged) {
        uint64_t w = 0, w1 = 0, w2 = 0;
        int j = next_tile(first, w), j1 = next_tile(j + 1, w1);
        int buf = 0;
        if (!staged || j != 0 || j1 != 1) {                            // not the tiles that were staged at the start
            if (j < nkv) stage(j, 0);
            if (j1 < nkv) stage(j1, RB_BUF);
            drain_and_barrier();
        }
        while (j < nkv) {
            const char* base = smem + buf;
            const int j2 = next_tile(j1 + 1, w2);
            f32x16 x[2];
    #pragma unroll
            for (int i = 0; i < 16; ++i) { x[0][i] = 0.f; x[1][i] = 0.f; }
    #pragma unroll
            for (int t = 0; t < 2; ++t)
    #pragma unroll
                for (int ks = 0; ks < 4; ++ks)
                    x[t] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(*(const bf16x8*)(base + t * 4096 + koff[ks]), qf[ks], x[t], 0, 0, 0);
            // x[t][r]: query l32, key 64j + 32t + 16(r >> 3) + 8hi + (r & 7)
            const int d_lo = j * RB_KV - (q0 + 31), d_hi = j * RB_KV + 63 - q0;
            const bool right = d_lo >= p.reach, left = d_hi <= -p.reach;
            const bool part = w != ~0ull;
            // One half of the tile: soft-max, then its share of Oᵀ += Vᵀ·Pᵀ.  The first half's soft-max runs behind the second half's scores on the matrix pipe,
            // the second half's behind the first half's products.
            auto half = [&](auto t_tag) {
                constexpr int t = decltype(t_tag)::value;
                const unsigned wt = (unsigned)(w >> (32 * t));
                if (part && wt == 0) return;                              // (wave-uniform) no key in this half
                auto weigh = [&](float shift) __attribute__((always_inline)) {   // scale, bias and shift, -inf at keys that do not count
                    if (right || left) {
                        const float add = (right ? far_r : far_l) - shift;
    #pragma unroll
                        for (int r = 0; r < 16; ++r) x[t][r] = fmaf(x[t][r], p.c, add);
                    } else {
                        // |d| <= reach + 94 here: inside the padded table.  A query row beyond the last one reads inside it too (its wave's own range).
                        const float* tb = tab + (j * RB_KV + 32 * t + 8 * hi - qrow + p.reach + RB_PAD);
    #pragma unroll
                        for (int r = 0; r < 16; ++r) x[t][r] = fmaf(x[t][r], p.c, tb[16 * (r >> 3) + (r & 7)] - shift);
                    }
                    if (__builtin_expect(part, 0)) {
                        const unsigned mine = wt >> (8 * hi);
    #pragma unroll
                        for (int r = 0; r < 16; ++r)
                            if (!((mine >> (16 * (r >> 3) + (r & 7))) & 1)) x[t][r] = -INFINITY;
                    }
                };
                if (__builtin_expect(__any(fabsf(m_run) > RB_FAR_SHIFT) != 0, 0)) {   // bias - shift would keep digits that the shift, a sum with the bias, lost
                    weigh(0.f);
    #pragma unroll
                    for (int r = 0; r < 16; ++r) x[t][r] -= m_run;
                } else weigh(m_run);
                unsigned pf[2][4], pl[2][4];
                float tsum = 0.f;
                auto expo = [&]() {
                    float s0 = 0.f, s1 = 0.f;
    #pragma unroll
                    for (int s = 0; s < 2; ++s)
    #pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const float pa = __builtin_amdgcn_exp2f(x[t][8 * s + 2 * e]), pb = __builtin_amdgcn_exp2f(x[t][8 * s + 2 * e + 1]);
                            pf[s][e] = pack_bf16x2(pa, pb);
                            if constexpr (TRAIN) {
                                pl[s][e] = pack_bf16x2(pa - __uint_as_float(pf[s][e] << 16), pb - __uint_as_float(pf[s][e] & 0xffff0000u));
                                s0 += pa;
                                s1 += pb;
                            } else {                                      // the sum of the rounded values: numerator and denominator round alike, one instruction a pair
                                bf16x2 ones;
                                ones[0] = (__bf16)1.0f; ones[1] = (__bf16)1.0f;
                                if (e & 1) s1 = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, pf[s][e]), ones, s1, false);
                                else s0 = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, pf[s][e]), ones, s0, false);
                            }
                        }
                    tsum = s0 + s1;
                };
                bool redo = !started;
                if (!redo) {
                    expo();
                    redo = __any(fresh || !(tsum <= 1.099511627776e12f)) != 0;   // 2^40
                }
                if (__builtin_expect(redo, 0)) {
                    if (started) {                                        // the scores once more: shifted far, they have lost digits
    #pragma unroll
                        for (int r = 0; r < 16; ++r) x[t][r] = 0.f;
    #pragma unroll
                        for (int ks = 0; ks < 4; ++ks)
                            x[t] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(*(const bf16x8*)(base + t * 4096 + koff[ks]), qf[ks], x[t], 0, 0, 0);
                        weigh(0.f);
                    }
                    float top = x[t][0];
    #pragma unroll
                    for (int r = 1; r < 16; ++r) top = fmaxf(top, x[t][r]);
                    top = fmaxf(top, __shfl_xor(top, 32, 64));
                    const float to = fresh ? (top == -INFINITY ? 0.f : top) : fmaxf(m_run, top);
                    if (started) {
                        const float alpha = fresh ? 1.f : __builtin_amdgcn_exp2f(m_run - to);
    #pragma unroll
                        for (int i = 0; i < 16; ++i) { o[0][i] *= alpha; o[1][i] *= alpha; }
                        l_run *= alpha;
                    }
                    m_run = to;
                    fresh = fresh && top == -INFINITY;
    #pragma unroll
                    for (int i = 0; i < 16; ++i) x[t][i] -= to;
                    expo();
                    started = true;
                }
                l_run += tsum;
                bf16x8 vf[2][2];
                rb_read_tr(vf, base + RB_TILE + t * 4096, voff);
                if (__builtin_expect(part, 0)) {
    #pragma unroll
                    for (int s = 0; s < 2; ++s)
    #pragma unroll
                        for (int dt = 0; dt < 2; ++dt) vf[s][dt] = rb_keep(vf[s][dt], (wt >> (16 * s + 8 * hi)) & 0xffu);
                }
    #pragma unroll
                for (int s = 0; s < 2; ++s)
    #pragma unroll
                    for (int dt = 0; dt < 2; ++dt) {
                        o[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vf[s][dt], __builtin_bit_cast(bf16x8, make_uint4(pf[s][0], pf[s][1], pf[s][2], pf[s][3])), o[dt], 0, 0, 0);
                        if constexpr (TRAIN)
                            o[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vf[s][dt], __builtin_bit_cast(bf16x8, make_uint4(pl[s][0], pl[s][1], pl[s][2], pl[s][3])), o[dt], 0, 0, 0);
                    }
            };
            half(std::integral_constant<int, 0>{});
            half(std::integral_constant<int, 1>{});
            tt_landed();                                            // tile j1, issued one tile ago
            if (j2 < nkv) stage(j2, rb_next(rb_next(buf)));               // its buffer was last read before the previous barrier
            rb_reads_done_barrier();
            j = j1; w = w1;
            j1 = j2; w1 = w2;
            buf = rb_next(buf);
        }
    };

    // ---- the run of whole tiles at the front, in a pipeline --------------------------------------------------------------------------------------------
    // VALU issued between a wave's own matrix instructions runs behind them, that of the SIMD's other waves mostly does not: the soft-max of one half of a tile
    // is spread over eight matrix instructions, four of the other half's scores and four of the previous half's products.  Iteration j:
    //   scores of (j, half 1) and products of (j − 1, half 1)  behind them the soft-max of (j, half 0)
    //   products of (j, half 0) and scores of (j + 1, half 0)   behind them the soft-max of (j, half 1)
    // K runs one tile ahead of V.  The shift is the maximum of the row's first 32 scores throughout; whether an exp2 left fp32's range shows in the finished
    // row (a sum or an output that is not finite): the workgroup then starts over with the tile-by-tile loop.
    auto pipeline = [&](int n) {
        constexpr int KO = 0, VO = RB_TILE;
        int kb = 0, kb1 = RB_BUF, kb2 = 2 * RB_BUF;                   // buffers of K(j), K(j + 1), K(j + 2); V(j) is in the same as K(j)
        if (n > 2) stage_k(2, kb2);                                   // tiles 0 and 1 are there
        f32x16 x0, x1;
        bf16x8 ka[4], kc[4], va[2][2], vc[2][2];                      // fragments for the first and the second half of an iteration
        unsigned p0[2][4], p1[2][4], l0[2][4], l1[2][4];
        auto scores = [&](int ks, const bf16x8& k, f32x16& x) {
            if (ks == 0) {
#pragma unroll
                for (int i = 0; i < 16; ++i) x[i] = 0.f;
            }
            x = __builtin_amdgcn_mfma_f32_32x32x16_bf16(k, qf[ks], x, 0, 0, 0);
        };
        auto frag = [&](const unsigned (&f)[4]) { return __builtin_bit_cast(bf16x8, make_uint4(f[0], f[1], f[2], f[3])); };
        auto product = [&](int i, const bf16x8 (&v)[2][2], const unsigned (&p)[2][4], const unsigned (&l)[2][4]) {   // i: 2 s + dt
            o[i & 1] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(v[i >> 1][i & 1], frag(p[i >> 1]), o[i & 1], 0, 0, 0);
            if constexpr (TRAIN) o[i & 1] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(v[i >> 1][i & 1], frag(l[i >> 1]), o[i & 1], 0, 0, 0);
        };
        float s0 = 0.f, s1 = 0.f;
        auto soft = [&](int e, const f32x16& x, unsigned (&p)[2][4], unsigned (&l)[2][4], float add, auto near_tag) {   // elements 2e, 2e + 1
            const bool NEAR = decltype(near_tag)::value;
            const float a = __builtin_amdgcn_exp2f(NEAR ? x[2 * e] : fmaf(x[2 * e], args.a.c, add));
            const float b = __builtin_amdgcn_exp2f(NEAR ? x[2 * e + 1] : fmaf(x[2 * e + 1], args.a.c, add));
            const unsigned pk = pack_bf16x2(a, b);
            p[e >> 2][e & 3] = pk;
            if constexpr (TRAIN) {
                l[e >> 2][e & 3] = pack_bf16x2(a - __uint_as_float(pk << 16), b - __uint_as_float(pk & 0xffff0000u));
                s0 += a;
                s1 += b;
            } else {
                bf16x2 ones;
                ones[0] = (__bf16)1.0f; ones[1] = (__bf16)1.0f;
                if (e & 1) s1 = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, pk), ones, s1, false);
                else s0 = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, pk), ones, s0, false);
            }
        };
        auto biased = [&](f32x16& x, int at) {                        // scale, bias and shift of 16 scores near the diagonal
            const float* tb = tab + (at + 8 * hi - qrow + p.reach + RB_PAD);
#pragma unroll
            for (int r = 0; r < 16; ++r) x[r] = fmaf(x[r], p.c, tb[16 * (r >> 3) + (r & 7)] - m_run);
        };
        auto sides = [&](int j, bool& right, bool& left) {
            right = j * RB_KV - (q0 + 31) >= p.reach;
            left = j * RB_KV + 63 - q0 <= -p.reach;
        };
        // scores of (0, half 0): their maximum is the rows' shift
#pragma unroll
        for (int ks = 0; ks < 4; ++ks) scores(ks, *(const bf16x8*)(smem + kb + KO + koff[ks]), x0);
        {
            f32x16 y = x0;
            bool right, left;
            sides(0, right, left);
            if (right || left) {
#pragma unroll
                for (int r = 0; r < 16; ++r) y[r] = fmaf(y[r], p.c, right ? far_r : far_l);
            } else biased(y, 0);
            float top = y[0];
#pragma unroll
            for (int r = 1; r < 16; ++r) top = fmaxf(top, y[r]);
            m_run = fmaxf(top, __shfl_xor(top, 32, 64));
        }
#pragma unroll
        for (int ks = 0; ks < 4; ++ks) ka[ks] = *(const bf16x8*)(smem + kb + KO + 4096 + koff[ks]);
#pragma unroll
        for (int i = 0; i < 4; ++i) va[i >> 1][i & 1] = bf16x8{};
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int e = 0; e < 4; ++e) { p1[s][e] = 0; l1[s][e] = 0; }   // (0, half 1) has no predecessor: zeros times zeros
        auto turn = [&](int j, float add, auto near_tag) {
            if constexpr (decltype(near_tag)::value) biased(x0, j * RB_KV);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                vc[i >> 1][i & 1] = tt_read(smem + kb + VO + 2048 * (i >> 1), voff[i & 1]);      // for the second half of the iteration
                kc[i] = *(const bf16x8*)(smem + kb1 + KO + koff[i]);
                scores(i, ka[i], x1);
                soft(2 * i, x0, p0, l0, add, near_tag);
                __builtin_amdgcn_sched_barrier(0);
                product(i, va, p1, l1);
                soft(2 * i + 1, x0, p0, l0, add, near_tag);
                __builtin_amdgcn_sched_barrier(0);
            }
            if constexpr (decltype(near_tag)::value) biased(x1, j * RB_KV + 32);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                va[i >> 1][i & 1] = tt_read(smem + kb + VO + 4096 + 2048 * (i >> 1), voff[i & 1]);   // for the next iteration's first half
                ka[i] = *(const bf16x8*)(smem + kb1 + KO + 4096 + koff[i]);
                product(i, vc, p0, l0);
                soft(2 * i, x1, p1, l1, add, near_tag);
                __builtin_amdgcn_sched_barrier(0);
                scores(i, kc[i], x0);
                soft(2 * i + 1, x1, p1, l1, add, near_tag);
                __builtin_amdgcn_sched_barrier(0);
            }
            // K(j + 2) and V(j + 1) have landed.  V(j)'s and K(j + 1)'s reads above may still be on their way; K(j)'s and V(j - 1)'s, whose buffers are
            // filled now, have been used.
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            block_barrier();
            if (j + 3 < n) stage_k(j + 3, kb);
            if (j + 2 < n) stage_v(j + 2, kb2);
            const int was = kb;
            kb = kb1; kb1 = kb2; kb2 = was;
        };
        // three loops, so that each has one body: tiles left of the wave's diagonal, along it, right of it.  The workgroup's waves change over at
        // different tiles; every iteration has the same one barrier.
        const int near_from = min(n, max(0, (q0 - p.reach - 63) / RB_KV + (q0 - p.reach - 63 >= 0 ? 1 : 0)));   // the first tile with 64j + 63 - q0 > -reach
        const int near_to = min(n, (q0 + 31 + p.reach + RB_KV - 1) / RB_KV);                                    // the first with 64j - q0 - 31 >= reach
        int j = 0;
        for (; j < near_from; ++j) turn(j, far_l - m_run, std::false_type{});
        for (; j < near_to; ++j) turn(j, 0.f, std::true_type{});
        for (; j < n; ++j) turn(j, far_r - m_run, std::false_type{});
#pragma unroll
        for (int i = 0; i < 4; ++i) product(i, va, p1, l1);
        l_run = s0 + s1;
        started = true;
        fresh = false;
        drain_and_barrier();
    };
    int whole = 0;                                                    // tiles at the front whose keys all count
    if (PIPE && p.mask == nullptr) whole = S / RB_KV;
    else if (PIPE) {
        for (int at = 0;; at += 64) {
            const uint64_t less = __ballot(at + lane >= nkv || words[min(at + lane, nkv - 1)] != ~0ull);
            if (less) { whole = at + __builtin_ctzll(less); break; }
        }
    }
    if (PIPE && whole >= RB_PIPE_TILES) {
        pipeline(whole);
        if (whole < nkv) sweep(whole, false);
        const float l_row = l_run + __shfl_xor(l_run, 32, 64);        // the row's sum: two finite halves may add up to more than fp32 holds
        float worst = fabsf(l_row);
        if (fabsf(m_run) > RB_FAR_SHIFT) worst = INFINITY;
#pragma unroll
        for (int i = 0; i < 16; ++i) worst = fmaxf(worst, fmaxf(fabsf(o[0][i]), fabsf(o[1][i])));
        bool bad = !(worst <= 3.4e38f);
#pragma unroll
        for (int i = 0; i < 16; ++i) bad |= o[0][i] != o[0][i] || o[1][i] != o[1][i];   // (fmaxf passes over a NaN)
        bad |= l_row != l_row;
        if (__syncthreads_or(bad ? 1 : 0)) {
#pragma unroll
            for (int i = 0; i < 16; ++i) { o[0][i] = 0.f; o[1][i] = 0.f; }
            m_run = 0.f;
            l_run = 0.f;
            started = false;
            fresh = true;
            sweep(0, false);
        }
    } else sweep(0, true);
    // ---- epilogue: O[b][q][h][d], d = 32dt + 8(r >> 2) + 4hi + (r & 3) ----
    const float l_tot = l_run + __shfl_xor(l_run, 32, 64);
    const float inv = started && l_tot != 0.f ? 1.0f / l_tot : 0.f;   // (a sum of 0: the keys that count all score -inf)
    const size_t at = (((size_t)b * S + min(qrow, S - 1)) * p.H + h) * RB_D;
    if constexpr (TRAIN) {
        if (hi == 0 && qrow < S) {            // +inf: the backward pass gets P = 0 everywhere in such a row; beyond 2^20 a log-sum's digits do not tell P any more
            const float l = m_run + __builtin_amdgcn_logf(l_tot);
            args.lse[(size_t)bh * S + qrow] = !started || fabsf(l) > 1048576.f ? INFINITY : l;
        }
        f32x16 low[2];
#pragma unroll
        for (int dt = 0; dt < 2; ++dt)
#pragma unroll
            for (int i = 0; i < 16; ++i) low[dt][i] = o[dt][i] * inv - (float)(bf16_t)(o[dt][i] * inv);
        rb_store(low, 1.f, args.o_low + at, hi, qrow < S);
    }
    rb_store(o, inv, args.o + at, hi, qrow < S);
}

// One head's rows go through a 32-bit buffer descriptor, and the tile behind the last row is addressed (not fetched) too.
int rb_tensor(RbTensor& t, const void* ptr, const long* st, int S) {
    if (!ptr) return aether_set_error(AETHER_ERR_ARG, "relbias_attn: null operand");
    if ((uintptr_t)ptr & 15 || st[0] % 8 || st[1] % 8 || st[2] % 8) return aether_set_error(AETHER_ERR_ALIGN, "relbias_attn: rows of [B, S, H, 64] operands must be 16-byte aligned");
    if (st[0] < 0 || st[1] < 0 || st[2] < 0 || ((long)S + RB_KV) * st[1] * 2 + 128 >= (1l << 32))
        return aether_set_error(AETHER_ERR_SHAPE, "relbias_attn: S times the row stride must stay below 4 GiB, and no stride may be negative");
    t = RbTensor{(const bf16_t*)ptr, st[0], st[1], st[2]};
    return AETHER_OK;
}

int rb_setup(RbArgs& p, const AetherRelbias* d) {
    auto fail = [](int code, const char* msg) { return aether_set_error(code, msg); };
    if (!d) return fail(AETHER_ERR_ARG, "relbias_attn: null descriptor");
    if (d->B < 0 || d->S < 0 || d->H < 1) return fail(AETHER_ERR_SHAPE, "relbias_attn: B and S must not be negative, H must be positive");
    if (d->S > RB_MAX_S) return fail(AETHER_ERR_SHAPE, "relbias_attn: S must be at most 65536");
    if (d->num_buckets < 4 || d->num_buckets % 2 != 0 || d->num_buckets > 128) return fail(AETHER_ERR_SHAPE, "relbias_attn: num_buckets must be an even number in [4, 128]");
    const int half = d->num_buckets / 2, near_n = half / 2;
    if (!d->borders || d->n_borders != half - near_n - 1) return fail(AETHER_ERR_ARG, "relbias_attn: borders must name where each bucket behind the first logarithmic one begins");
    int last = near_n;
    for (int i = 0; i < d->n_borders; ++i) {
        if (d->borders[i] < last) return fail(AETHER_ERR_ARG, "relbias_attn: borders must not fall, nor lie below num_buckets / 4");
        last = d->borders[i];
        p.border[i] = last;
    }
    if (last > RB_MAX_REACH) return fail(AETHER_ERR_SHAPE, "relbias_attn: the last bucket must begin at 1024 or before");
    if (!(d->scale == 0.f || (fabsf(d->scale) >= 1e-20f && fabsf(d->scale) <= 1e20f)))    // (a backward pass divides by it)
        return fail(AETHER_ERR_ARG, "relbias_attn: the scale must be 0 or of a magnitude in [1e-20, 1e20]");
    p.B = d->B; p.S = d->S; p.H = d->H;
    p.half = half; p.near_n = near_n; p.n_border = d->n_borders; p.reach = last;
    p.c = d->scale * RB_LOG2E;
    p.table = (const bf16_t*)d->table;
    p.mask = (const unsigned char*)d->mask; p.mask_sb = d->mask_sb;
    // a grid of 2^32 threads or more is cut short without an error  (the backward pass takes as many waves or fewer)
    const int nw = rb_waves(p);
    if ((size_t)d->B * d->H * ((d->S + nw * 32 - 1) / (nw * 32)) >= (1ull << 32) / (nw * 64)) return fail(AETHER_ERR_SHAPE, "relbias_attn: too many query blocks for one launch");
    if (d->B == 0 || d->S == 0) return AETHER_OK;
    if (!d->table) return fail(AETHER_ERR_ARG, "relbias_attn: null table");
    int rc = rb_tensor(p.q, d->q, d->q_strides, d->S);
    if (!rc) rc = rb_tensor(p.k, d->k, d->k_strides, d->S);
    if (!rc) rc = rb_tensor(p.v, d->v, d->v_strides, d->S);
    if (rc) return rc;
    return AETHER_OK;
}

}  // namespace aether

using namespace aether;

extern "C" int aether_relbias_attn(const AetherRelbias* d, void* o, void* o_low, float* lse, void* stream) {
    RbFwdArgs args = {};
    int rc = rb_setup(args.a, d);
    if (rc) return rc;
    if (d->B == 0 || d->S == 0) return AETHER_OK;
    if (!o) return aether_set_error(AETHER_ERR_ARG, "relbias_attn: null output");
    if ((o_low != nullptr) != (lse != nullptr)) return aether_set_error(AETHER_ERR_ARG, "relbias_attn: o_low and lse are given together");
    if (((uintptr_t)o | (uintptr_t)o_low) & 15) return aether_set_error(AETHER_ERR_ALIGN, "relbias_attn: the output must be 16-byte aligned");
    args.o = (bf16_t*)o;
    args.o_low = (bf16_t*)o_low;
    args.lse = lse;
    RbArgs& p = args.a;
    const size_t lds = RB_RING + rb_table_bytes(p.reach) + rb_words_bytes(p);
    const int nw = rb_waves(p);
    p.nqb = (p.S + nw * 32 - 1) / (nw * 32);
    const dim3 grid((unsigned)((long)p.B * p.H * p.nqb));
    hipStream_t s = (hipStream_t)stream;
    // ring, table and mask words pass 64 KiB where S, the mask and the reach are all near their limits
#define RB_LAUNCH(NW, PIPE)                                                                                          \
    do {                                                                                                             \
        const void* f = lse ? (const void*)relbias_attn_fwd_kernel<NW, true, PIPE> : (const void*)relbias_attn_fwd_kernel<NW, false, PIPE>; \
        if (lds > 64 * 1024 && hipFuncSetAttribute(f, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds) != hipSuccess) { \
            (void)hipGetLastError();                                                                                 \
            return aether_set_error(AETHER_ERR_LAUNCH, "relbias_attn: the workgroup's LDS could not be set");        \
        }                                                                                                            \
        if (lse) hipLaunchKernelGGL((relbias_attn_fwd_kernel<NW, true, PIPE>), grid, dim3(NW * 64), lds, s, args);   \
        else hipLaunchKernelGGL((relbias_attn_fwd_kernel<NW, false, PIPE>), grid, dim3(NW * 64), lds, s, args);      \
    } while (0)
    switch (nw) {
        case 4:
            if (p.S >= RB_PIPE_TILES * RB_KV) RB_LAUNCH(4, true);
            else RB_LAUNCH(4, false);
            break;
        case 2: RB_LAUNCH(2, false); break;
        default: RB_LAUNCH(1, false); break;
    }
#undef RB_LAUNCH
    return aether_check_launch("relbias_attn");
}
