// Backward pass of attention with a relative position bias (relbias_attn.hip), head dimension 64.  From O (in two bf16 parts), dO and the rows' log-sums L
// (base 2):
//
//   P_ij = 2^(S_ij − L_i),   δ_i = dO_i·O_i,   dP_ij = dO_i·v_j,   dS_ij = P_ij (dP_ij − δ_i)
//   dq_i = scale Σ_j dS_ij k_j,   dk_j = scale Σ_i dS_ij q_i,   dv_j = Σ_i P_ij dO_i,   dT[b, h] = Σ of dS_ij over the pairs whose bucket is b
//
// Two sweeps instead of one with atomics: the first owns queries (δ, dq, dT), the second owns keys (dk, dv).  The scores and dP are computed twice
// (7 products instead of 5), and every sum has an order that depends on the sizes alone.  A lane holds 16 scores of ONE query (first sweep) or of
// ONE key (second) at a time, and dS / P leave the registers as the B operand of the next product; the transposed A operands come out of
// row-major tiles by ds_read_b64_tr_b16.
// Where one key alone counts, P is 1 whatever its score and dS is 0: those gradients are set to 0 instead of the difference of two roundings of one number.
// dT: beyond `reach` a tile's dS go into one number per lane.  Near the diagonal dS is summed along its diagonals in registers: the 16 values of a lane are
// rotated over the 32 queries by their key's place (ds_swizzle, a constant each), which brings a diagonal into one lane; what wraps around joins the next
// 32 keys' diagonals, so that every entry of a wave's table of distances is stored once, by plain stores.  (LDS float atomics in their place: 200 cycles an
// instruction, three quarters of this kernel's time at 16 x 226 x 64 heads.)  Keys that do not count: their
// P and dS are 0 whatever k and v hold there, and so are dk and dv.
// P and dS become bf16 once, as operands of the products (the matrix unit's fp32 products run at a sixteenth of the rate); dT is summed from dS before that.  Relative L2 error of the
// gradients against 64 bits 0.0024, of which the outputs' own rounding is 0.0017.
//
// What bounds it.  2 x 2039 x 32 heads: the pass takes 282 µs, its sweeps 142 and 149 under the profiler, a third (first) to 45% (second) of the matrix pipe's cycles; the vector work (an exponential,
// a product and two roundings an element) takes nearly as many and hides behind the products only in part.  Deeper rings, fragments read further ahead and a
// pipeline over half tiles changed nothing.  16 x 226 x 64 heads: 75 + 61 µs for 207 + 178 MB, 2.8 TB/s: reading q, k, v and dO in two sweeps instead of one
// is what this split costs there.
#include <type_traits>
#include <utility>
#include "relbias_attn.hpp"
#include "../../include/aether_hip.h"

namespace aether {

struct RbBwdArgs {
    RbArgs a;
    RbTensor o, go, dq, dk, dv;
    const bf16_t* o_low;              // [B, S, H, 64]
    const float* lse;
    float* delta;                     // [B, H, S]
    float* part;                      // [B·H·nqb][2·half]: a workgroup's share of dT; or null
    float scale;
};

template <int... Is, class F> AE_DEV void rb_static_for_impl(F&& f, std::integer_sequence<int, Is...>) { (f(std::integral_constant<int, Is>{}), ...); }
template <int N, class F> AE_DEV void rb_static_for(F&& f) { rb_static_for_impl(f, std::make_integer_sequence<int, N>{}); }

template <int NW>
__global__ __launch_bounds__(NW * 64) __attribute__((amdgpu_waves_per_eu(2, 2))) void relbias_attn_dq_kernel(RbBwdArgs args) {
    extern __shared__ __attribute__((aligned(16))) char smem[];
    const RbArgs& p = args.a;
    const int n_tab = 2 * (p.reach + RB_PAD) + 1;
    const int tab_bytes = (n_tab * 4 + 15) / 16 * 16;
    float* const tab = (float*)(smem + RB_RING);
    float* const hist = (float*)(smem + RB_RING + tab_bytes);              // [wave][hi][n_tab]
    unsigned char* const words8 = (unsigned char*)(smem + RB_RING + tab_bytes * (args.part ? 1 + 2 * NW : 1));
    const uint64_t* const words = (const uint64_t*)words8;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, hi = lane >> 5, l32 = lane & 31;
    const int wave_s = __builtin_amdgcn_readfirstlane(wave);
    const int S = p.S;
    const int wgid = xcd_remap((int)blockIdx.x, p.B * p.H * p.nqb);
    const int bh = wgid / p.nqb, qb = wgid - bh * p.nqb;
    const int b = bh / p.H, h = bh - b * p.H;
    const int q0 = qb * (NW * 32) + wave_s * 32;
    const int qrow = q0 + l32, qc = min(qrow, S - 1);

    float* const my_hist = hist + (wave * 2 + hi) * (tab_bytes / 4);

    bf16x8 qf[4], gf[4];
    float delta = 0.f;
    {
        const bf16_t* qp = p.q.p + (size_t)b * p.q.sb + (size_t)h * p.q.sh + (size_t)qc * p.q.ss;
        const bf16_t* gp = args.go.p + (size_t)b * args.go.sb + (size_t)h * args.go.sh + (size_t)qc * args.go.ss;
        const bf16_t* op = args.o.p + (size_t)b * args.o.sb + (size_t)h * args.o.sh + (size_t)qc * args.o.ss;
        const bf16_t* lp = args.o_low + (((size_t)b * S + qc) * p.H + h) * RB_D;
        f32x16 og;                                                    // og[r]: O of query 8(r >> 2) + 4hi + (r & 3) times dO of query l32
#pragma unroll
        for (int i = 0; i < 16; ++i) og[i] = 0.f;
#pragma unroll
        for (int ks = 0; ks < 4; ++ks) {
            qf[ks] = *(const bf16x8*)(qp + 16 * ks + 8 * hi);
            gf[ks] = *(const bf16x8*)(gp + 16 * ks + 8 * hi);
            og = __builtin_amdgcn_mfma_f32_32x32x16_bf16(*(const bf16x8*)(op + 16 * ks + 8 * hi), gf[ks], og, 0, 0, 0);
        }
#pragma unroll
        for (int ks = 0; ks < 4; ++ks) og = __builtin_amdgcn_mfma_f32_32x32x16_bf16(*(const bf16x8*)(lp + 16 * ks + 8 * hi), gf[ks], og, 0, 0, 0);
#pragma unroll
        for (int r = 0; r < 16; ++r) delta = 8 * (r >> 2) + 4 * hi + (r & 3) == l32 ? og[r] : delta;
        const float other = __shfl_xor(delta, 32, 64);                // the diagonal's element is in one of the two halves
        delta = ((l32 >> 2) & 1) == hi ? delta : other;
    }
    if (hi == 0 && qrow < S) args.delta[(size_t)bh * S + qrow] = delta;
    const float lse = qrow < S ? args.lse[(size_t)bh * S + qc] : INFINITY;   // rows behind the last one: P = 0, they add nothing to dT

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
    auto stage = [&](int j, int buf) __attribute__((always_inline)) {
        const unsigned dst = tt_lds(smem) + buf + wave_s * 1024;
#pragma unroll
        for (int ps = 0; ps < 8 / NW; ++ps) {
            tt_dma16(k_rsrc, k_off[ps], (unsigned)j * (RB_KV * k_row), dst + ps * (NW * 1024));
            tt_dma16(v_rsrc, v_off[ps], (unsigned)j * (RB_KV * v_row), dst + RB_TILE + ps * (NW * 1024));
        }
    };
    const int nkv = (S + RB_KV - 1) / RB_KV;
    stage(0, 0);                                                      // on their way while the table and the mask are read; whether their keys count shows later
    if (nkv > 1) stage(1, RB_BUF);
    rb_fill_table(p, h, tab, NW * 64);
    if (p.mask) rb_fill_words(p.mask + (size_t)b * p.mask_sb, S, words8, NW * 64);
    if (args.part)
        for (int i = tid; i < tab_bytes / 4 * 2 * NW; i += NW * 64) hist[i] = 0.f;
    int roff[4], toff[2][2];
    rb_row_offsets(lane, roff);
    tt_offsets(lane, toff);

    rb_arrived(qf);
    rb_arrived(gf);
    f32x16 dq[2], minus_delta;                                        // dP starts from −δ
#pragma unroll
    for (int i = 0; i < 16; ++i) { dq[0][i] = 0.f; dq[1][i] = 0.f; minus_delta[i] = -delta; }
    float sum_r = 0.f, sum_l = 0.f, far_sum[2] = {0.f, 0.f};                    // dS beyond the reach, on either side
    float carry = 0.f;                                                // diagonals that go on into the keys from carry_at on (wave-uniform; < 0: none)
    int carry_at = -1;
    auto put = [&](int at, float v) {
        if (at < n_tab) my_hist[at] = v;                              // (beyond it there are only zeros: no pair of the wave is that far apart)
    };

    drain_and_barrier();                                              // table, words and tables of distances are there, and the first two tiles
    const float far_r = tab[2 * (p.reach + RB_PAD)], far_l = tab[0];
    bool lone = S == 1;
    if (p.mask) {
        int n = 0;
        for (int i = lane; i < nkv; i += 64) n += __popcll(words[i]);
        lone = wave_sum((float)n) == 1.f;
    }
    auto next_tile = [&](int j, uint64_t& w) {
        for (; j < nkv; ++j)
            if ((w = rb_word(p, words, j)) != 0) break;
        return j;
    };
    uint64_t w = 0, w1 = 0, w2 = 0;
    int j = next_tile(0, w), j1 = next_tile(j + 1, w1);
    int buf = 0;
    if (j != 0 || j1 != 1) {                                          // not the tiles that were staged at the start
        if (j < nkv) stage(j, 0);
        if (j1 < nkv) stage(j1, RB_BUF);
        drain_and_barrier();
    }
    // dS of one half, near the diagonal: summed along its diagonals
    auto diagonals = [&](const f32x16& ds, int k_at) __attribute__((always_inline)) {
        // element (query l32, key k_at + kr + 8hi), kr = 16(r >> 3) + (r & 7): rotated by kr it is in lane i = l32 - kr of its half (of 32 lanes), distance
        // k_at + 8hi - q0 - i; or, wrapped, in lane i = l32 - kr + 32, distance 32 more
        float whole = 0.f, wrap = 0.f;
        rb_static_for<16>([&](auto r_tag) __attribute__((always_inline)) {
            constexpr int r = decltype(r_tag)::value, kr = 16 * (r >> 3) + (r & 7);
            const float y = kr ? __int_as_float(__builtin_amdgcn_ds_swizzle(__float_as_int(ds[r]), 0xc000 | (kr << 5))) : ds[r];
            const float z = l32 > 31 - kr ? y : 0.f;
            wrap += z;
            whole += y - z;
        });
        if (k_at != carry_at) {                                       // the diagonals carried here do not continue where this begins
            if (carry_at >= 0) put(carry_at + 8 * hi - q0 - l32 + p.reach + RB_PAD, carry);
            carry = 0.f;
        }
        put(k_at + 8 * hi - q0 - l32 + p.reach + RB_PAD, whole + carry);
        carry = wrap;
        carry_at = k_at + 32;
    };
    // One tile.  VALU issued between a wave's own matrix instructions runs behind them: the first half's dS is spread over the second half's scores and dP, the
    // second half's over the first half's products.
    auto tile = [&](float add, auto near_tag, auto part_tag) __attribute__((always_inline)) {
        constexpr bool NEAR = decltype(near_tag)::value, PART = decltype(part_tag)::value;
        const char* const base = smem + buf;
        // the A fragment of matrix instruction i of 24: scores and dP of the first half, of the second half, products of the first, of the second
        auto fragment = [&](auto i_tag) __attribute__((always_inline)) -> bf16x8 {
            constexpr int i = decltype(i_tag)::value;
            if constexpr (i < 16) return *(const bf16x8*)(base + (i & 1) * RB_TILE + (i >> 3) * 4096 + roff[(i >> 1) & 3]);
            else if constexpr (PART)
                return rb_keep(tt_read(base + ((i >> 2) & 1) * 4096 + 2048 * ((i >> 1) & 1), toff[i & 1]), (unsigned)(w >> (32 * ((i >> 2) & 1) + 16 * ((i >> 1) & 1) + 8 * hi)) & 0xffu);
            else return tt_read(base + ((i >> 2) & 1) * 4096 + 2048 * ((i >> 1) & 1), toff[i & 1]);
        };
        f32x16 x[2], dp[2];                                           // x[t][r], dp[t][r]: query l32, key 64j + 32t + 16(r >> 3) + 8hi + (r & 7)
        unsigned df[2][2][4];
        const float* const tb = tab + (j * RB_KV + 8 * hi - qrow + p.reach + RB_PAD);
        const unsigned keep0 = (unsigned)w >> (8 * hi), keep1 = (unsigned)(w >> 32) >> (8 * hi);
        auto weigh = [&](auto e_tag, auto t_tag) __attribute__((always_inline)) {                    // elements 2e, 2e + 1
            constexpr int e = decltype(e_tag)::value, t = decltype(t_tag)::value, at = 16 * (e >> 2) + 2 * (e & 3);
            float d0 = __builtin_amdgcn_exp2f(fmaf(x[t][2 * e], p.c, NEAR ? tb[32 * t + at] + add : add)) * dp[t][2 * e];
            float d1 = __builtin_amdgcn_exp2f(fmaf(x[t][2 * e + 1], p.c, NEAR ? tb[32 * t + at + 1] + add : add)) * dp[t][2 * e + 1];
            if constexpr (PART) {
                d0 = ((t ? keep1 : keep0) >> at) & 1 ? d0 : 0.f;
                d1 = ((t ? keep1 : keep0) >> (at + 1)) & 1 ? d1 : 0.f;
            }
            x[t][2 * e] = d0;
            x[t][2 * e + 1] = d1;
            const unsigned pk = pack_bf16x2(d0, d1);
            df[t][e >> 2][e & 3] = pk;
            if constexpr (!NEAR) {                                    // a far bucket's share.  (A row's dS add up to 0: summed after their rounding, the far ones of a long row
                far_sum[0] += d0;                                     // lose what they differ by from the near ones.)
                far_sum[1] += d1;
            }
        };
        constexpr int AHEAD = 3;                                      // fragments are read this many instructions before they are used
        bf16x8 f[AHEAD + 1];
        rb_static_for<AHEAD>([&](auto i_tag) { f[decltype(i_tag)::value] = fragment(i_tag); });
        rb_static_for<24>([&](auto i_tag) __attribute__((always_inline)) {
            constexpr int i = decltype(i_tag)::value, t = (i >> 3) & 1, ks = (i >> 1) & 3;
            if constexpr (i + AHEAD < 24) f[(i + AHEAD) % (AHEAD + 1)] = fragment(std::integral_constant<int, i + AHEAD>{});
            const bf16x8& a = f[i % (AHEAD + 1)];
            if constexpr (i < 16 && (i & 1) == 0) {
                if constexpr (ks == 0) {
#pragma unroll
                    for (int r = 0; r < 16; ++r) x[t][r] = 0.f;
                }
                x[t] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, qf[ks], x[t], 0, 0, 0);
            } else if constexpr (i < 16) {
                dp[t] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, gf[ks], ks == 0 ? minus_delta : dp[t], 0, 0, 0);
            } else {
                constexpr int ht = (i >> 2) & 1, s = (i >> 1) & 1, dt = i & 1;
                dq[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, __builtin_bit_cast(bf16x8, make_uint4(df[ht][s][0], df[ht][s][1], df[ht][s][2], df[ht][s][3])), dq[dt], 0, 0, 0);
            }
            if constexpr (i >= 8 && i < 16) weigh(std::integral_constant<int, i - 8>{}, std::integral_constant<int, 0>{});
            if constexpr (i >= 16 && i < 20) {
                weigh(std::integral_constant<int, 2 * (i - 16)>{}, std::integral_constant<int, 1>{});
                weigh(std::integral_constant<int, 2 * (i - 16) + 1>{}, std::integral_constant<int, 1>{});
            }
            __builtin_amdgcn_sched_barrier(0);
        });
        if constexpr (NEAR) {
            if (args.part) {
                diagonals(x[0], j * RB_KV);
                diagonals(x[1], j * RB_KV + 32);
            }
        }
    };
    auto advance = [&]() __attribute__((always_inline)) {
        const int j2 = next_tile(j1 + 1, w2);
        tt_landed();                                            // tile j1, issued one tile ago
        if (j2 < nkv) stage(j2, rb_next(rb_next(buf)));               // its buffer was last read before the previous barrier
        rb_reads_done_barrier();
        j = j1; w = w1;
        j1 = j2; w1 = w2;
        buf = rb_next(buf);
    };
    // three loops: keys left of the wave's queries, around them, right of them.  The workgroup's waves change over at different tiles; every iteration has the
    // same one barrier.
    const int near_from = q0 - p.reach - 63 >= 0 ? (q0 - p.reach - 63) / RB_KV + 1 : 0;   // the first tile with 64j + 63 - q0 > -reach
    const int near_to = (q0 + 31 + p.reach + RB_KV - 1) / RB_KV;                          // the first with 64j - q0 - 31 >= reach
    auto far = [&](float add) __attribute__((always_inline)) {
        if (__builtin_expect(w != ~0ull, 0)) tile(add, std::false_type{}, std::true_type{});
        else tile(add, std::false_type{}, std::false_type{});
        advance();
    };
    while (j < min(near_from, nkv)) far(far_l - lse);
    sum_l = far_sum[0] + far_sum[1];
    far_sum[0] = far_sum[1] = 0.f;
    while (j < min(near_to, nkv)) {
        if (__builtin_expect(w != ~0ull, 0)) tile(-lse, std::true_type{}, std::true_type{});
        else tile(-lse, std::true_type{}, std::false_type{});
        advance();
    }
    while (j < nkv) far(far_r - lse);
    sum_r = far_sum[0] + far_sum[1];
    if (lone) {
#pragma unroll
        for (int i = 0; i < 16; ++i) { dq[0][i] = 0.f; dq[1][i] = 0.f; }
    }
    rb_store(dq, args.scale, const_cast<bf16_t*>(args.dq.p) + (size_t)b * args.dq.sb + (size_t)h * args.dq.sh + (size_t)qc * args.dq.ss, hi, qrow < S);

    if (args.part == nullptr) return;
    // ---- dT of this workgroup: the far sums join the outermost entries, then the copies are added up, then each bucket's run of distances ----
    if (carry_at >= 0) put(carry_at + 8 * hi - q0 - l32 + p.reach + RB_PAD, carry);
    sum_r = wave_sum(sum_r);
    sum_l = wave_sum(sum_l);
    if (lane == 0) {                                                  // (wave-private, and behind the wave's own adds)
        my_hist[0] += sum_l;
        my_hist[n_tab - 1] += sum_r;
    }
    __syncthreads();
    for (int i = tid; i < n_tab; i += NW * 64) {
        float s = 0.f;
#pragma unroll
        for (int c = 0; c < 2 * NW; ++c) s += hist[c * (tab_bytes / 4) + i];
        tab[i] = s;
    }
    __syncthreads();
    float* const out = args.part + (size_t)wgid * (2 * p.half);
    const int sub = tid & 7;                                          // eight lanes a bucket
    for (int bk = tid >> 3; bk < 2 * p.half; bk += NW * 8) {
        const int n = bk >= p.half ? bk - p.half : bk;                // bucket of its side: distances [from, to]
        const int from = n <= p.near_n ? n : p.border[n - p.near_n - 1];
        const int to = n < p.near_n ? n : n == p.half - 1 ? p.reach + RB_PAD : p.border[n - p.near_n] - 1;
        float s = 0.f;
        for (int d = from + sub; d <= to; d += 8) s += tab[(bk >= p.half ? d : -d) + p.reach + RB_PAD];
        if (bk >= p.half && from == 0 && sub == 0) s = 0.f;           // distance 0 belongs to the other side
        s += __shfl_xor(s, 1, 64);
        s += __shfl_xor(s, 2, 64);
        s += __shfl_xor(s, 4, 64);
        if (sub == 0) out[bk] = lone ? 0.f : s;
    }
}

// dT[b, h] = Σ over the batch and the query blocks, every eighth in order and then these eight.  One workgroup per head.
__global__ __launch_bounds__(1024) void relbias_attn_dtable_kernel(const float* __restrict__ part, int B, int H, int nqb, int nb, bf16_t* __restrict__ dtable) {
    __shared__ float red[8][128];
    const int h = blockIdx.x, bk = threadIdx.x & 127, g = threadIdx.x >> 7;
    float s = 0.f;
    if (bk < nb)
        for (int i = g; i < B * nqb; i += 8) {
            const int b = i / nqb;
            s += part[(((size_t)b * H + h) * nqb + (i - b * nqb)) * nb + bk];
        }
    red[g][bk] = s;
    __syncthreads();
    if (g == 0 && bk < nb) {
#pragma unroll
        for (int i = 1; i < 8; ++i) s += red[i][bk];
        dtable[(size_t)bk * H + h] = (bf16_t)s;
    }
}

template <int NW>
__global__ __launch_bounds__(NW * 64) __attribute__((amdgpu_waves_per_eu(2, 2))) void relbias_attn_dkv_kernel(RbBwdArgs args) {
    extern __shared__ __attribute__((aligned(16))) char smem[];
    const RbArgs& p = args.a;
    float* const rows = (float*)(smem + RB_RING);                  // [buffer of three][−L / c | −δ][64]
    float* const tab = (float*)(smem + RB_RING + 1536);
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, hi = lane >> 5, l32 = lane & 31;
    const int wave_s = __builtin_amdgcn_readfirstlane(wave);
    const int S = p.S;
    const int wgid = xcd_remap((int)blockIdx.x, p.B * p.H * p.nqb);
    const int bh = wgid / p.nqb, kb = wgid - bh * p.nqb;
    const int b = bh / p.H, h = bh - b * p.H;
    const int k0 = kb * (NW * 32) + wave_s * 32;
    const int key = k0 + l32, kc = min(key, S - 1);
    const bool counts = key < S && (p.mask == nullptr || p.mask[(size_t)b * p.mask_sb + kc] != 0);
    const bool some = __any(counts) != 0;                             // of this wave; the others keep it company at the barriers
    int mine = 0;                                                     // keys of the batch item that count, as far as this thread looked
    if (p.mask)
        for (int i = tid; i < S; i += NW * 64) mine += p.mask[(size_t)b * p.mask_sb + i] != 0;
    bf16_t* const dkp = const_cast<bf16_t*>(args.dk.p) + (size_t)b * args.dk.sb + (size_t)h * args.dk.sh + (size_t)kc * args.dk.ss;
    bf16_t* const dvp = const_cast<bf16_t*>(args.dv.p) + (size_t)b * args.dv.sb + (size_t)h * args.dv.sh + (size_t)kc * args.dv.ss;

    bf16x8 kf[4], vf[4];
    {
        const bf16_t* kp = p.k.p + (size_t)b * p.k.sb + (size_t)h * p.k.sh + (size_t)kc * p.k.ss;
        const bf16_t* vp = p.v.p + (size_t)b * p.v.sb + (size_t)h * p.v.sh + (size_t)kc * p.v.ss;
        const bf16x8 zero = {};
#pragma unroll
        for (int ks = 0; ks < 4; ++ks) {                              // what stands at a key that does not count is not looked at
            kf[ks] = counts && p.c != 0.f ? *(const bf16x8*)(kp + 16 * ks + 8 * hi) : zero;
            vf[ks] = counts ? *(const bf16x8*)(vp + 16 * ks + 8 * hi) : zero;
        }
    }
    // a scale of 0 is a scale of 1 on keys of 0
    const float c = p.c != 0.f ? p.c : 1.f, inv_c = 1.f / c;
    f32x16 dk[2], dv[2];
#pragma unroll
    for (int i = 0; i < 16; ++i) { dk[0][i] = 0.f; dk[1][i] = 0.f; dv[0][i] = 0.f; dv[1][i] = 0.f; }

    const bool lone = p.mask ? __syncthreads_count(mine != 0) == 1 && !__syncthreads_or(mine > 1) : S == 1;
    if (__syncthreads_or(some ? 1 : 0)) {
        const unsigned q_row = (unsigned)p.q.ss * 2, g_row = (unsigned)args.go.ss * 2;
        const i32x4 q_rsrc = tt_rsrc(p.q.p + (size_t)b * p.q.sb + (size_t)h * p.q.sh, (unsigned)(S - 1) * q_row + 128);
        const i32x4 g_rsrc = tt_rsrc(args.go.p + (size_t)b * args.go.sb + (size_t)h * args.go.sh, (unsigned)(S - 1) * g_row + 128);
        float next_l = 0.f, next_d = 0.f;
        // rows behind the last one repeat it: their P is 0 (L = +inf), and what they are multiplied with has to be a number
        auto stage = [&](int j, int buf) __attribute__((always_inline)) {
            const unsigned dst = tt_lds(smem) + buf + wave_s * 1024;
#pragma unroll
            for (int ps = 0; ps < 8 / NW; ++ps) {
                const int r = (ps * NW + wave) * 8 + (lane >> 3), sw = ((lane & 7) ^ tt_swz(r)) << 4;
                const unsigned row = min(j * RB_KV + r, S - 1);
                tt_dma16(q_rsrc, row * q_row + sw, 0u, dst + ps * (NW * 1024));
                tt_dma16(g_rsrc, row * g_row + sw, 0u, dst + RB_TILE + ps * (NW * 1024));
            }
            if (tid < RB_KV) {
                const int row = j * RB_KV + tid;
                next_l = row < S ? args.lse[(size_t)bh * S + row] : INFINITY;
                next_d = row < S ? args.delta[(size_t)bh * S + row] : 0.f;
            }
        };
        auto put_rows = [&](int buf) {
            if (tid < RB_KV) {
                float* const to = rows + buf / RB_BUF * 128 + tid;
                to[0] = next_l * -inv_c;
                to[64] = -next_d;
            }
        };
        const int nq = (S + RB_KV - 1) / RB_KV;
        stage(0, 0);
        const float first_l = next_l, first_d = next_d;
        if (nq > 1) stage(1, RB_BUF);
        rb_fill_table(p, h, tab, NW * 64);
        if (tid < RB_KV) {
            rows[tid] = first_l * -inv_c;
            rows[64 + tid] = -first_d;
        }
        rb_arrived(kf);
        rb_arrived(vf);
        int roff[4], toff[2][2];
        rb_row_offsets(lane, roff);
        tt_offsets(lane, toff);
        drain_and_barrier();
        const float far_r = tab[2 * (p.reach + RB_PAD)], far_l = tab[0];
        // One tile of 64 queries.  The scores start from −L / c, so that one fma with the bias gives the exponent, and dP from −δ.  VALU issued between a wave's own matrix
        // instructions runs behind them: the first half's P and dS are spread over the second half's scores and dP, the second half's over the first half's
        // products.
        const float off = counts ? 0.f : -INFINITY;
        int buf = 0;
        auto tile = [&](int j, float add, auto near_tag) __attribute__((always_inline)) {             // add: what every score of the tile gets, −inf at keys that do not count
            constexpr bool NEAR = decltype(near_tag)::value;
            const char* const base = smem + buf;
            const float* const lp = rows + buf / RB_BUF * 128 + 8 * hi;
            // x[r], dp[r] of half t: key l32, query 64j + 32t + 16(r >> 3) + 8hi + (r & 7)
            auto begin = [&](int t, f32x16& x, f32x16& dp) {
#pragma unroll
                for (int s = 0; s < 2; ++s) {
                    const f32x4 l0 = *(const f32x4*)(lp + 32 * t + 16 * s), l1 = *(const f32x4*)(lp + 32 * t + 16 * s + 4);
                    const f32x4 e0 = *(const f32x4*)(lp + 64 + 32 * t + 16 * s), e1 = *(const f32x4*)(lp + 64 + 32 * t + 16 * s + 4);
#pragma unroll
                    for (int e = 0; e < 4; ++e) { x[8 * s + e] = l0[e]; x[8 * s + 4 + e] = l1[e]; dp[8 * s + e] = e0[e]; dp[8 * s + 4 + e] = e1[e]; }
                }
            };
            // the A fragment of matrix instruction i of 32: scores and dP of the first half, of the second half, products of the first, of the second
            auto fragment = [&](int i) {
                if (i < 16) return *(const bf16x8*)(base + (i & 1) * RB_TILE + (i >> 3) * 4096 + roff[(i >> 1) & 3]);
                return tt_read(base + (i & 1 ? 0 : RB_TILE) + ((i >> 3) & 1) * 4096 + 2048 * ((i >> 2) & 1), toff[(i >> 1) & 1]);
            };
            auto score = [&](int i, const bf16x8& a, f32x16& x, f32x16& dp) {
                if (i & 1) dp = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, vf[(i >> 1) & 3], dp, 0, 0, 0);
                else x = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, kf[(i >> 1) & 3], x, 0, 0, 0);
            };
            auto product = [&](int i, const bf16x8& a, const unsigned (&pf)[2][4], const unsigned (&df)[2][4]) {
                const int s = (i >> 2) & 1, dt = (i >> 1) & 1;
                const unsigned (&f)[4] = i & 1 ? df[s] : pf[s];
                const bf16x8 v = __builtin_bit_cast(bf16x8, make_uint4(f[0], f[1], f[2], f[3]));
                if (i & 1) dk[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, v, dk[dt], 0, 0, 0);
                else dv[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, v, dv[dt], 0, 0, 0);
            };
            auto weigh = [&](int e, int t, const f32x16& x, const f32x16& dp, unsigned (&pf)[2][4], unsigned (&df)[2][4]) {   // elements 2e, 2e + 1
                const float* const tb = tab + (key - (j * RB_KV + 32 * t + 8 * hi) - 23 + p.reach + RB_PAD);   // of the last of the 16 queries
                float pr[2], ds[2];
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const int r = 2 * e + i;
                    pr[i] = __builtin_amdgcn_exp2f(fmaf(x[r], c, NEAR ? tb[23 - 16 * (r >> 3) - (r & 7)] + add : add));
                    ds[i] = pr[i] * dp[r];
                }
                pf[e >> 2][e & 3] = pack_bf16x2(pr[0], pr[1]);
                df[e >> 2][e & 3] = pack_bf16x2(ds[0], ds[1]);
            };
            f32x16 x0, dp0, x1, dp1;
            unsigned p0[2][4], d0[2][4], p1[2][4], d1[2][4];
            constexpr int AHEAD = 3;                                  // fragments are read this many instructions before they are used
            bf16x8 f[AHEAD + 1];
#pragma unroll
            for (int i = 0; i < AHEAD; ++i) f[i] = fragment(i);
            begin(0, x0, dp0);
            rb_static_for<32>([&](auto i_tag) __attribute__((always_inline)) {
                constexpr int i = decltype(i_tag)::value;
                if constexpr (i + AHEAD < 32) f[(i + AHEAD) % (AHEAD + 1)] = fragment(i + AHEAD);
                const bf16x8& a = f[i % (AHEAD + 1)];
                if constexpr (i < 8) score(i, a, x0, dp0);
                else if constexpr (i < 16) score(i, a, x1, dp1);
                else if constexpr (i < 24) product(i, a, p0, d0);
                else product(i, a, p1, d1);
                if constexpr (i == 5) begin(1, x1, dp1);
                if constexpr (i >= 8 && i < 16) weigh(i - 8, 0, x0, dp0, p0, d0);
                if constexpr (i >= 16 && i < 24) weigh(i - 16, 1, x1, dp1, p1, d1);
                __builtin_amdgcn_sched_barrier(0);
            });
        };
        auto advance = [&](int j) __attribute__((always_inline)) {
            tt_landed();                                        // tile j + 1, issued one tile ago, and its rows' L and δ
            put_rows(rb_next(buf));
            if (j + 2 < nq) stage(j + 2, rb_next(rb_next(buf)));      // its buffer was last read before the previous barrier
            rb_reads_done_barrier();
            buf = rb_next(buf);
        };
        // three loops, so that each has one body: queries left of the wave's keys, around them, right of them.  The workgroup's waves change over at different
        // tiles; every iteration has the same one barrier.
        const int near_from = k0 - 63 - p.reach >= 0 ? min(nq, (k0 - 63 - p.reach) / RB_KV + 1) : 0;   // the first tile with k0 - 64j - 63 < reach
        const int near_to = min(nq, (k0 + 31 + p.reach + RB_KV - 1) / RB_KV);                          // the first with k0 + 31 - 64j <= -reach
        int j = 0;
        for (; j < near_from; ++j) {
            if (some) tile(j, far_r + off, std::false_type{});
            advance(j);
        }
        for (; j < near_to; ++j) {
            if (some) tile(j, off, std::true_type{});
            advance(j);
        }
        for (; j < nq; ++j) {
            if (some) tile(j, far_l + off, std::false_type{});
            advance(j);
        }
    }
    // a key that does not count has P = dS = 0; times a NaN of some row's dO that would be a NaN
#pragma unroll
    for (int i = 0; i < 16; ++i)
#pragma unroll
        for (int dt = 0; dt < 2; ++dt) { dk[dt][i] = counts && !lone ? dk[dt][i] : 0.f; dv[dt][i] = counts ? dv[dt][i] : 0.f; }
    rb_store(dk, args.scale, dkp, hi, key < S);
    rb_store(dv, 1.f, dvp, hi, key < S);
}

static int rb_bwd_waves(const RbArgs& p, bool dtable) {
    // a wave's two tables of the distances have to fit beside the tiles
    int nw = rb_waves(p);
    while (dtable && nw > 1 && RB_RING + rb_table_bytes(p.reach) * (1 + 2 * nw) + rb_words_bytes(p) > 160 * 1024) nw /= 2;
    return nw;
}

}  // namespace aether

using namespace aether;

extern "C" size_t aether_relbias_attn_bwd_workspace_bytes(const AetherRelbias* d, int need_dtable) {
    RbArgs p = {};
    if (!d) return 0;
    AetherRelbias dd = *d;
    if (rb_setup(p, &dd)) return 0;
    const size_t rows = (size_t)p.B * p.H * p.S;
    const int nw = rb_bwd_waves(p, need_dtable != 0);
    return rows * 4 + (need_dtable ? (size_t)p.B * p.H * ((p.S + nw * 32 - 1) / (nw * 32)) * (2 * p.half) * 4 : 0);
}

extern "C" int aether_relbias_attn_bwd(const AetherRelbias* d, const void* go, const long* go_strides, const void* o, const long* o_strides, const void* o_low,
                                       const float* lse, void* dq, const long* dq_strides, void* dk, const long* dk_strides, void* dv, const long* dv_strides, void* dtable,
                                       void* workspace, size_t workspace_bytes, void* stream) {
    RbBwdArgs args = {};
    int rc = rb_setup(args.a, d);
    if (rc) return rc;
    RbArgs& p = args.a;
    hipStream_t s = (hipStream_t)stream;
    const bool empty = p.B == 0 || p.S == 0;
    int nw = 1;
    if (!empty) {
        if (!lse || !o_low) return aether_set_error(AETHER_ERR_ARG, "relbias_attn_bwd: null lse or o_low");
        if ((uintptr_t)o_low & 15) return aether_set_error(AETHER_ERR_ALIGN, "relbias_attn_bwd: o_low must be 16-byte aligned");
        rc = rb_tensor(args.go, go, go_strides, p.S);
        if (!rc) rc = rb_tensor(args.o, o, o_strides, p.S);
        if (!rc) rc = rb_tensor(args.dq, dq, dq_strides, p.S);
        if (!rc) rc = rb_tensor(args.dk, dk, dk_strides, p.S);
        if (!rc) rc = rb_tensor(args.dv, dv, dv_strides, p.S);
        if (rc) return rc;
        if (!workspace || ((uintptr_t)workspace & 15) || workspace_bytes < aether_relbias_attn_bwd_workspace_bytes(d, dtable != nullptr))
            return aether_set_error(AETHER_ERR_ARG, "relbias_attn_bwd: workspace too small or misaligned (aether_relbias_attn_bwd_workspace_bytes)");
        args.lse = lse;
        args.o_low = (const bf16_t*)o_low;
        args.delta = (float*)workspace;
        args.part = dtable ? args.delta + (size_t)p.B * p.H * p.S : nullptr;
        args.scale = d->scale;
        nw = rb_bwd_waves(p, dtable != nullptr);
        p.nqb = (p.S + nw * 32 - 1) / (nw * 32);
        const dim3 grid((unsigned)((long)p.B * p.H * p.nqb));
        const size_t lds_q = RB_RING + rb_table_bytes(p.reach) * (dtable ? 1 + 2 * nw : 1) + rb_words_bytes(p);
        const size_t lds_k = RB_RING + 1536 + rb_table_bytes(p.reach);
#define RB_LAUNCH(NW)                                                                                       \
    do {                                                                                                    \
        if (lds_q > 64 * 1024 && hipFuncSetAttribute((const void*)relbias_attn_dq_kernel<NW>, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds_q) != hipSuccess) { \
            (void)hipGetLastError();                                                                        \
            return aether_set_error(AETHER_ERR_LAUNCH, "relbias_attn_bwd: the workgroup's LDS could not be set"); \
        }                                                                                                   \
        hipLaunchKernelGGL((relbias_attn_dq_kernel<NW>), grid, dim3(NW * 64), lds_q, s, args);              \
        rc = aether_check_launch("relbias_attn_dq");                                                        \
        if (rc) return rc;                                                                                  \
        hipLaunchKernelGGL((relbias_attn_dkv_kernel<NW>), grid, dim3(NW * 64), lds_k, s, args);             \
    } while (0)
        switch (nw) {
            case 4: RB_LAUNCH(4); break;
            case 2: RB_LAUNCH(2); break;
            default: RB_LAUNCH(1); break;
        }
#undef RB_LAUNCH
        rc = aether_check_launch("relbias_attn_dkv");
        if (rc) return rc;
    }
    if (dtable) {
        hipLaunchKernelGGL(relbias_attn_dtable_kernel, dim3(p.H), dim3(1024), 0, s, args.part, empty ? 0 : p.B, p.H, p.nqb, 2 * p.half, (bf16_t*)dtable);
        rc = aether_check_launch("relbias_attn_dtable");
    }
    return rc;
}
