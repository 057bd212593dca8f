// Self-attention with a learned bias by bucket of the relative position, forward pass, head dimension 64:
//
//   S_ij = scale · q_i·k_j + T[bucket(j − i), h]  where key j counts,   P = softmax_j(S),   O = P V;   a row without keys gives 0.
//
// gfx950 design
//   * A wave owns 32 queries, a workgroup NW waves of one (batch, head); tiles of 64 keys, K and V by 16-byte LDS-DMA into two buffers, one barrier
//     per tile.  Sᵀ = K·Qᵀ on v_mfma_f32_32x32x16_bf16: a lane holds 32 scores of ONE query.  K rows enter in the order pi, so that the
//     exponentiated scores are, in register order, the B operand of Oᵀ += Vᵀ·Pᵀ; Vᵀ comes out of the row-major tile by ds_read_b64_tr_b16.
//   * The bias depends on key − query alone and is constant beyond `reach` (91 positions for 32 buckets up to 128): a tile that lies beyond it adds ONE
//     number, folded into the fma that scales the scores.  Only the few tiles along the diagonal look their bias up, in a table of 2·reach + 1 floats
//     in LDS, whose addresses are consecutive over the lanes (no bank conflicts).
//   * Soft-max over one pass: the shift of a row is the true maximum of its first tile; later tiles are exponentiated against it and checked
//     afterwards (a lane's partial sum above 2^100, or NaN, makes the wave take the classic online step on the scores it still holds).  Any shift
//     gives the same soft-max; the check keeps exp2 inside fp32.  Sums are fp32; P is rounded to bf16 once, as the operand of P·V.
//   * For a backward pass the output is needed beyond bf16: δ = dO·O is subtracted from numbers that may be nearly equal to it.  TRAIN multiplies V with P in
//     two bf16 parts (P = hi + lo to 2^-17) and also stores what the rounding of O left (o_low), so that O + o_low is good to 2^-16.
//   * Keys that do not count: whole tiles are skipped; in a tile that holds some, their scores become −inf and their V elements 0 (a NaN or an infinity
//     behind the mask reaches nothing).
#include <type_traits>
#include "relbias_attn.hpp"
#include "../../include/aether_hip.h"

namespace aether {

struct RbFwdArgs { RbArgs a; bf16_t* o; bf16_t* o_low; float* lse; };   // o_low, lse: for a backward pass

template <int NW, bool TRAIN>
__global__ __launch_bounds__(NW * 64) __attribute__((amdgpu_waves_per_eu(3, 3))) void relbias_attn_fwd_kernel(RbFwdArgs args) {
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

    rb_fill_table(p, h, tab, NW * 64);
    if (p.mask) rb_fill_words(p.mask + (size_t)b * p.mask_sb, S, words8, NW * 64);

    bf16x8 qf[4];
    {
        const bf16_t* qp = p.q.p + (size_t)b * p.q.sb + (size_t)h * p.q.sh + (size_t)min(qrow, S - 1) * p.q.ss;
#pragma unroll
        for (int ks = 0; ks < 4; ++ks) qf[ks] = *(const bf16x8*)(qp + 16 * ks + 8 * hi);
    }
    // ---- staging: a wave-instruction moves 8 rows x 128 bytes; rows at or beyond S are outside the descriptor and their keys do not count ----
    const unsigned k_row = (unsigned)p.k.ss * 2, v_row = (unsigned)p.v.ss * 2;
    const buf_rsrc_t k_rsrc = make_buf_rsrc(p.k.p + (size_t)b * p.k.sb + (size_t)h * p.k.sh, (unsigned)(S - 1) * k_row + 128);
    const buf_rsrc_t v_rsrc = make_buf_rsrc(p.v.p + (size_t)b * p.v.sb + (size_t)h * p.v.sh, (unsigned)(S - 1) * v_row + 128);
    unsigned k_off[8 / NW], v_off[8 / NW];
#pragma unroll
    for (int ps = 0; ps < 8 / NW; ++ps) {
        const int r = (ps * NW + wave) * 8 + (lane >> 3), ch = lane & 7;
        k_off[ps] = r * k_row + ((ch ^ rb_swz(r)) << 4);
        v_off[ps] = r * v_row + ((ch ^ rb_swz(r)) << 4);
    }
    auto stage = [&](int j, int buf) {
        char* const dst = smem + buf + wave_s * 1024;
#pragma unroll
        for (int ps = 0; ps < 8 / NW; ++ps) {
            bglds16(k_rsrc, k_off[ps], (unsigned)j * (RB_KV * k_row), dst + ps * (NW * 1024));
            bglds16(v_rsrc, v_off[ps], (unsigned)j * (RB_KV * v_row), dst + RB_TILE + ps * (NW * 1024));
        }
    };
    int koff[4], voff[2][2];
    rb_row_offsets(lane, koff);
    rb_tr_offsets(lane, voff);

    f32x16 o[2];
#pragma unroll
    for (int i = 0; i < 16; ++i) { o[0][i] = 0.f; o[1][i] = 0.f; }
    float m_run = 0.f, l_run = 0.f;
    bool started = false;

    rb_arrived(qf);
    __syncthreads();                                                  // table and words are there
    const float far_r = tab[2 * (p.reach + RB_PAD)], far_l = tab[0];
    const int nkv = (S + RB_KV - 1) / RB_KV;
    auto next_tile = [&](int j, uint64_t& w) {                        // the next tile from j on that holds a key, nkv if none does
        for (; j < nkv; ++j)
            if ((w = rb_word(p, words, j)) != 0) break;
        return j;
    };
    uint64_t w = 0, w1 = 0, w2 = 0;
    int j = next_tile(0, w), j1 = next_tile(j + 1, w1);
    int buf = 0;
    if (j < nkv) stage(j, 0);
    if (j1 < nkv) stage(j1, RB_BUF);
    drain_and_barrier();
    while (j < nkv) {
        const char* base = smem + buf;
        const int j2 = next_tile(j1 + 1, w2);
        f32x16 x[2];
#pragma unroll
        for (int i = 0; i < 16; ++i) { x[0][i] = 0.f; x[1][i] = 0.f; }
        __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int ks = 0; ks < 4; ++ks)
                x[t] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(*(const bf16x8*)(base + t * 4096 + koff[ks]), qf[ks], x[t], 0, 0, 0);
        __builtin_amdgcn_s_setprio(0);
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
            if (right || left) {
                const float add = (right ? far_r : far_l) - m_run;
#pragma unroll
                for (int r = 0; r < 16; ++r) x[t][r] = fmaf(x[t][r], p.c, add);
            } else {
                // |d| <= reach + 94 here: inside the padded table.  A query row beyond the last one reads inside it too (its wave's own range).
                const float* tb = tab + (j * RB_KV + 32 * t + 8 * hi - qrow + p.reach + RB_PAD);
#pragma unroll
                for (int r = 0; r < 16; ++r) x[t][r] = fmaf(x[t][r], p.c, tb[16 * (r >> 3) + (r & 7)] - m_run);
            }
            if (__builtin_expect(part, 0)) {
                const unsigned mine = wt >> (8 * hi);
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    if (!((mine >> (16 * (r >> 3) + (r & 7))) & 1)) x[t][r] = -INFINITY;
            }
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
                redo = __any(!(tsum <= 1.2676506e30f)) != 0;          // 2^100
            }
            if (__builtin_expect(redo, 0)) {
                float top = x[t][0];
#pragma unroll
                for (int r = 1; r < 16; ++r) top = fmaxf(top, x[t][r]);
                top = fmaxf(top, __shfl_xor(top, 32, 64));
                const float up = started ? fmaxf(top, 0.f) : top == -INFINITY ? 0.f : top;
                if (started) {
                    const float alpha = __builtin_amdgcn_exp2f(-up);
#pragma unroll
                    for (int i = 0; i < 16; ++i) { o[0][i] *= alpha; o[1][i] *= alpha; }
                    l_run *= alpha;
                }
                m_run += up;
#pragma unroll
                for (int i = 0; i < 16; ++i) x[t][i] -= up;
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
            __builtin_amdgcn_s_setprio(1);
#pragma unroll
            for (int s = 0; s < 2; ++s)
#pragma unroll
                for (int dt = 0; dt < 2; ++dt) {
                    o[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vf[s][dt], __builtin_bit_cast(bf16x8, make_uint4(pf[s][0], pf[s][1], pf[s][2], pf[s][3])), o[dt], 0, 0, 0);
                    if constexpr (TRAIN)
                        o[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vf[s][dt], __builtin_bit_cast(bf16x8, make_uint4(pl[s][0], pl[s][1], pl[s][2], pl[s][3])), o[dt], 0, 0, 0);
                }
            __builtin_amdgcn_s_setprio(0);
        };
        half(std::integral_constant<int, 0>{});
        half(std::integral_constant<int, 1>{});
        rb_tiles_landed();                                            // tile j1, issued one tile ago
        if (j2 < nkv) stage(j2, rb_next(rb_next(buf)));               // its buffer was last read before the previous barrier
        rb_reads_done_barrier();
        j = j1; w = w1;
        j1 = j2; w1 = w2;
        buf = rb_next(buf);
    }
    // ---- epilogue: O[b][q][h][d], d = 32dt + 8(r >> 2) + 4hi + (r & 3) ----
    const float l_tot = l_run + __shfl_xor(l_run, 32, 64);
    const float inv = started ? 1.0f / l_tot : 0.f;
    const size_t at = (((size_t)b * S + min(qrow, S - 1)) * p.H + h) * RB_D;
    if constexpr (TRAIN) {
        if (hi == 0 && qrow < S)              // +inf: the backward pass gets P = 0 everywhere in such a row
            args.lse[(size_t)bh * S + qrow] = started ? m_run + __builtin_amdgcn_logf(l_tot) : INFINITY;
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
    p.B = d->B; p.S = d->S; p.H = d->H;
    p.half = half; p.near_n = near_n; p.n_border = d->n_borders; p.reach = last;
    p.c = d->scale * RB_LOG2E;
    p.table = (const bf16_t*)d->table;
    p.mask = (const unsigned char*)d->mask; p.mask_sb = d->mask_sb;
    if ((long)d->B * d->H * ((d->S + 31) / 32) > 0x7fffffffl) return fail(AETHER_ERR_SHAPE, "relbias_attn: too many query blocks");
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
#define RB_LAUNCH(NW)                                                                                                \
    do {                                                                                                             \
        if (lse) hipLaunchKernelGGL((relbias_attn_fwd_kernel<NW, true>), grid, dim3(NW * 64), lds, s, args);         \
        else hipLaunchKernelGGL((relbias_attn_fwd_kernel<NW, false>), grid, dim3(NW * 64), lds, s, args);            \
    } while (0)
    switch (nw) {
        case 4: RB_LAUNCH(4); break;
        case 2: RB_LAUNCH(2); break;
        default: RB_LAUNCH(1); break;
    }
#undef RB_LAUNCH
    return aether_check_launch("relbias_attn");
}
