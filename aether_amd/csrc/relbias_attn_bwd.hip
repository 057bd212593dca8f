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
// δ is a product with O on the matrix pipe like dP is one with v, in the same order of sums: a row that has one key has O = v, so that its dP − δ is 0, not the
// difference of two roundings.
// dT: beyond `reach` a tile's dS go into one number per lane.  Near the diagonal dS is summed along its diagonals in registers: the 16 values of a lane are
// rotated over the 32 queries by their key's place (ds_swizzle, a constant each), which brings a diagonal into one lane; what wraps around joins the next
// 32 keys' diagonals, so that every entry of a wave's table of distances is stored once, by plain stores.  (LDS float atomics in their place: 200 cycles an
// instruction, three quarters of this kernel's time at 16 x 226 x 64 heads.)  Keys that do not count: their
// P and dS are 0 whatever k and v hold there, and so are dk and dv.
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
    const i32x4 k_rsrc = rb_rsrc(p.k.p + (size_t)b * p.k.sb + (size_t)h * p.k.sh, (unsigned)(S - 1) * k_row + 128);
    const i32x4 v_rsrc = rb_rsrc(p.v.p + (size_t)b * p.v.sb + (size_t)h * p.v.sh, (unsigned)(S - 1) * v_row + 128);
    unsigned k_off[8 / NW], v_off[8 / NW];
#pragma unroll
    for (int ps = 0; ps < 8 / NW; ++ps) {
        const int r = (ps * NW + wave) * 8 + (lane >> 3), ch = lane & 7;
        k_off[ps] = r * k_row + ((ch ^ rb_swz(r)) << 4);
        v_off[ps] = r * v_row + ((ch ^ rb_swz(r)) << 4);
    }
    auto stage = [&](int j, int buf) {
        const unsigned dst = rb_lds(smem) + buf + wave_s * 1024;
#pragma unroll
        for (int ps = 0; ps < 8 / NW; ++ps) {
            rb_dma16(k_rsrc, k_off[ps], (unsigned)j * (RB_KV * k_row), dst + ps * (NW * 1024));
            rb_dma16(v_rsrc, v_off[ps], (unsigned)j * (RB_KV * v_row), dst + RB_TILE + ps * (NW * 1024));
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
    rb_tr_offsets(lane, toff);

    rb_arrived(qf);
    rb_arrived(gf);
    f32x16 dq[2];
#pragma unroll
    for (int i = 0; i < 16; ++i) { dq[0][i] = 0.f; dq[1][i] = 0.f; }
    float sum_r = 0.f, sum_l = 0.f;                                   // dS beyond the reach, on either side
    float carry = 0.f;                                                // diagonals that go on into the keys from carry_at on (wave-uniform; < 0: none)
    int carry_at = -1;
    auto put = [&](int at, float v) {
        if (at < n_tab) my_hist[at] = v;                              // (beyond it there are only zeros: no pair of the wave is that far apart)
    };

    drain_and_barrier();                                              // table, words and tables of distances are there, and the first two tiles
    const float far_r = tab[2 * (p.reach + RB_PAD)], far_l = tab[0];
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
    while (j < nkv) {
        const int j2 = next_tile(j1 + 1, w2);
        const char* base = smem + buf;
        const bool part = w != ~0ull;
        const int d_lo = j * RB_KV - (q0 + 31), d_hi = j * RB_KV + 63 - q0;
        const bool right = d_lo >= p.reach, left = d_hi <= -p.reach;
        f32x16 x[2], dp[2];
#pragma unroll
        for (int i = 0; i < 16; ++i) { x[0][i] = 0.f; x[1][i] = 0.f; dp[0][i] = 0.f; dp[1][i] = 0.f; }
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int ks = 0; ks < 4; ++ks) {
                x[t] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(*(const bf16x8*)(base + t * 4096 + roff[ks]), qf[ks], x[t], 0, 0, 0);
                dp[t] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(*(const bf16x8*)(base + RB_TILE + t * 4096 + roff[ks]), gf[ks], dp[t], 0, 0, 0);
            }
        // x[t][r], dp[t][r]: query l32, key 64j + 32t + 16(r >> 3) + 8hi + (r & 7)
        auto half = [&](auto t_tag) {
            constexpr int t = decltype(t_tag)::value;
            const unsigned wt = (unsigned)(w >> (32 * t));
            if (part && wt == 0) return;                              // (wave-uniform) no key in this half
            const int k_at = j * RB_KV + 32 * t;
            const int d0 = k_at + 8 * hi - qrow + p.reach + RB_PAD;   // the distance of r = 0, as an index of tab
            f32x16& ds = x[t];
            if (right || left) {
                const float add = (right ? far_r : far_l) - lse;
#pragma unroll
                for (int r = 0; r < 16; ++r) ds[r] = fmaf(ds[r], p.c, add);
            } else {
#pragma unroll
                for (int r = 0; r < 16; ++r) ds[r] = fmaf(ds[r], p.c, tab[d0 + 16 * (r >> 3) + (r & 7)] - lse);
            }
#pragma unroll
            for (int r = 0; r < 16; ++r) ds[r] = __builtin_amdgcn_exp2f(ds[r]) * (dp[t][r] - delta);
            if (__builtin_expect(part, 0)) {
                const unsigned mine = wt >> (8 * hi);
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    if (!((mine >> (16 * (r >> 3) + (r & 7))) & 1)) ds[r] = 0.f;
            }
            if (args.part) {
                if (right || left) {
                    float s0 = 0.f, s1 = 0.f;
#pragma unroll
                    for (int r = 0; r < 16; r += 2) { s0 += ds[r]; s1 += ds[r + 1]; }
                    if (right) sum_r += s0 + s1;
                    else sum_l += s0 + s1;
                } else {
                    // element (query l32, key k_at + kr + 8hi), kr = 16(r >> 3) + (r & 7): rotated by kr it is in lane i = l32 - kr of its half (of 32
                    // lanes), distance k_at + 8hi - q0 - i; or, wrapped, in lane i = l32 - kr + 32, distance 32 more
                    float whole = 0.f, wrap = 0.f;
                    rb_static_for<16>([&](auto r_tag) {
                        constexpr int r = decltype(r_tag)::value, kr = 16 * (r >> 3) + (r & 7);
                        const float y = kr ? __int_as_float(__builtin_amdgcn_ds_swizzle(__float_as_int(ds[r]), 0xc000 | (kr << 5))) : ds[r];
                        const float z = l32 > 31 - kr ? y : 0.f;
                        wrap += z;
                        whole += y - z;
                    });
                    if (k_at != carry_at) {                           // the diagonals carried here do not continue where this begins
                        if (carry_at >= 0) put(carry_at + 8 * hi - q0 - l32 + p.reach + RB_PAD, carry);
                        carry = 0.f;
                    }
                    put(d0 + qrow - q0 - l32, whole + carry);
                    carry = wrap;
                    carry_at = k_at + 32;
                }
            }
            bf16x8 kf[2][2];
            rb_read_tr(kf, base + t * 4096, toff);
            if (__builtin_expect(part, 0)) {
#pragma unroll
                for (int s = 0; s < 2; ++s)
#pragma unroll
                    for (int dt = 0; dt < 2; ++dt) kf[s][dt] = rb_keep(kf[s][dt], (wt >> (16 * s + 8 * hi)) & 0xffu);
            }
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                const bf16x8 df = __builtin_bit_cast(bf16x8, make_uint4(pack_bf16x2(ds[8 * s], ds[8 * s + 1]), pack_bf16x2(ds[8 * s + 2], ds[8 * s + 3]),
                                                                        pack_bf16x2(ds[8 * s + 4], ds[8 * s + 5]), pack_bf16x2(ds[8 * s + 6], ds[8 * s + 7])));
#pragma unroll
                for (int dt = 0; dt < 2; ++dt) dq[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf[s][dt], df, dq[dt], 0, 0, 0);
            }
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
        if (sub == 0) out[bk] = s;
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
    float* const rows = (float*)(smem + RB_RING);                  // [buffer of three][L | δ][64]
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
    bf16_t* const dkp = const_cast<bf16_t*>(args.dk.p) + (size_t)b * args.dk.sb + (size_t)h * args.dk.sh + (size_t)kc * args.dk.ss;
    bf16_t* const dvp = const_cast<bf16_t*>(args.dv.p) + (size_t)b * args.dv.sb + (size_t)h * args.dv.sh + (size_t)kc * args.dv.ss;

    bf16x8 kf[4], vf[4];
    {
        const bf16_t* kp = p.k.p + (size_t)b * p.k.sb + (size_t)h * p.k.sh + (size_t)kc * p.k.ss;
        const bf16_t* vp = p.v.p + (size_t)b * p.v.sb + (size_t)h * p.v.sh + (size_t)kc * p.v.ss;
        const bf16x8 zero = {};
#pragma unroll
        for (int ks = 0; ks < 4; ++ks) {                              // what stands at a key that does not count is not looked at
            kf[ks] = counts ? *(const bf16x8*)(kp + 16 * ks + 8 * hi) : zero;
            vf[ks] = counts ? *(const bf16x8*)(vp + 16 * ks + 8 * hi) : zero;
        }
    }
    f32x16 dk[2], dv[2];
#pragma unroll
    for (int i = 0; i < 16; ++i) { dk[0][i] = 0.f; dk[1][i] = 0.f; dv[0][i] = 0.f; dv[1][i] = 0.f; }

    if (__syncthreads_or(some ? 1 : 0)) {
        const unsigned q_row = (unsigned)p.q.ss * 2, g_row = (unsigned)args.go.ss * 2;
        const i32x4 q_rsrc = rb_rsrc(p.q.p + (size_t)b * p.q.sb + (size_t)h * p.q.sh, (unsigned)(S - 1) * q_row + 128);
        const i32x4 g_rsrc = rb_rsrc(args.go.p + (size_t)b * args.go.sb + (size_t)h * args.go.sh, (unsigned)(S - 1) * g_row + 128);
        float next_l = 0.f, next_d = 0.f;
        // rows behind the last one repeat it: their P is 0 (L = +inf), and what they are multiplied with has to be a number
        auto stage = [&](int j, int buf) {
            const unsigned dst = rb_lds(smem) + buf + wave_s * 1024;
#pragma unroll
            for (int ps = 0; ps < 8 / NW; ++ps) {
                const int r = (ps * NW + wave) * 8 + (lane >> 3), sw = ((lane & 7) ^ rb_swz(r)) << 4;
                const unsigned row = min(j * RB_KV + r, S - 1);
                rb_dma16(q_rsrc, row * q_row + sw, 0u, dst + ps * (NW * 1024));
                rb_dma16(g_rsrc, row * g_row + sw, 0u, dst + RB_TILE + ps * (NW * 1024));
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
                to[0] = next_l;
                to[64] = next_d;
            }
        };
        const int nq = (S + RB_KV - 1) / RB_KV;
        stage(0, 0);
        const float first_l = next_l, first_d = next_d;
        if (nq > 1) stage(1, RB_BUF);
        rb_fill_table(p, h, tab, NW * 64);
        if (tid < RB_KV) {
            rows[tid] = first_l;
            rows[64 + tid] = first_d;
        }
        rb_arrived(kf);
        rb_arrived(vf);
        int roff[4], toff[2][2];
        rb_row_offsets(lane, roff);
        rb_tr_offsets(lane, toff);
        drain_and_barrier();
        const float far_r = tab[2 * (p.reach + RB_PAD)], far_l = tab[0];
        int buf = 0;
        for (int j = 0; j < nq; ++j) {
            if (some) {
                const char* base = smem + buf;
                const int d_lo = k0 - (j * RB_KV + 63), d_hi = k0 + 31 - j * RB_KV;
                const bool right = d_lo >= p.reach, left = d_hi <= -p.reach;
                const float far = right ? far_r : far_l;
                auto half = [&](auto t_tag, auto far_tag) {
                    constexpr int t = decltype(t_tag)::value;
                    constexpr bool FAR = decltype(far_tag)::value;
                    // x[r], dp[r]: key l32, query 64j + 32t + 16(r >> 3) + 8hi + (r & 7)
                    f32x16 x, dp;
#pragma unroll
                    for (int i = 0; i < 16; ++i) { x[i] = 0.f; dp[i] = 0.f; }
#pragma unroll
                    for (int ks = 0; ks < 4; ++ks) {
                        x = __builtin_amdgcn_mfma_f32_32x32x16_bf16(*(const bf16x8*)(base + t * 4096 + roff[ks]), kf[ks], x, 0, 0, 0);
                        dp = __builtin_amdgcn_mfma_f32_32x32x16_bf16(*(const bf16x8*)(base + RB_TILE + t * 4096 + roff[ks]), vf[ks], dp, 0, 0, 0);
                    }
                    const float* lp = rows + buf / RB_BUF * 128 + 32 * t + 8 * hi;
                    const float* tb = tab + (key - (j * RB_KV + 32 * t + 8 * hi) - 23 + p.reach + RB_PAD);   // of the last of the 16 queries
                    unsigned pf[2][4], df[2][4];
#pragma unroll
                    for (int s = 0; s < 2; ++s) {
                        const f32x4 l0 = *(const f32x4*)(lp + 16 * s), l1 = *(const f32x4*)(lp + 16 * s + 4);
                        const f32x4 e0 = *(const f32x4*)(lp + 64 + 16 * s), e1 = *(const f32x4*)(lp + 64 + 16 * s + 4);
#pragma unroll
                        for (int e = 0; e < 8; e += 2) {
                            float pr[2], ds[2];
#pragma unroll
                            for (int i = 0; i < 2; ++i) {
                                const int r = 8 * s + e + i;
                                const float l = e < 4 ? l0[e + i] : l1[e + i - 4], dl = e < 4 ? e0[e + i] : e1[e + i - 4];
                                const float bias = FAR ? far : tb[23 - 16 * s - e - i];
                                pr[i] = __builtin_amdgcn_exp2f(counts ? fmaf(x[r], p.c, bias - l) : -INFINITY);
                                ds[i] = pr[i] * (dp[r] - dl);
                            }
                            pf[s][e / 2] = pack_bf16x2(pr[0], pr[1]);
                            df[s][e / 2] = pack_bf16x2(ds[0], ds[1]);
                        }
                    }
                    bf16x8 qt[2][2], gt[2][2];
                    rb_read_tr(gt, base + RB_TILE + t * 4096, toff);
                    rb_read_tr(qt, base + t * 4096, toff);
#pragma unroll
                    for (int s = 0; s < 2; ++s) {
                        const bf16x8 pv = __builtin_bit_cast(bf16x8, make_uint4(pf[s][0], pf[s][1], pf[s][2], pf[s][3]));
                        const bf16x8 dv_ = __builtin_bit_cast(bf16x8, make_uint4(df[s][0], df[s][1], df[s][2], df[s][3]));
#pragma unroll
                        for (int dt = 0; dt < 2; ++dt) {
                            dv[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(gt[s][dt], pv, dv[dt], 0, 0, 0);
                            dk[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(qt[s][dt], dv_, dk[dt], 0, 0, 0);
                        }
                    }
                };
                if (right || left) {
                    half(std::integral_constant<int, 0>{}, std::true_type{});
                    half(std::integral_constant<int, 1>{}, std::true_type{});
                } else {
                    half(std::integral_constant<int, 0>{}, std::false_type{});
                    half(std::integral_constant<int, 1>{}, std::false_type{});
                }
            }
            rb_tiles_landed();                                        // tile j + 1, issued one tile ago, and its rows' L and δ
            put_rows(rb_next(buf));
            if (j + 2 < nq) stage(j + 2, rb_next(rb_next(buf)));      // its buffer was last read before the previous barrier
            rb_reads_done_barrier();
            buf = rb_next(buf);
        }
    }
    // a key that does not count has P = dS = 0; times a NaN of some row's dO that would be a NaN
#pragma unroll
    for (int i = 0; i < 16; ++i)
#pragma unroll
        for (int dt = 0; dt < 2; ++dt) { dk[dt][i] = counts ? dk[dt][i] : 0.f; dv[dt][i] = counts ? dv[dt][i] : 0.f; }
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
        if (lds_q > 64 * 1024 && hipFuncSetAttribute((const void*)relbias_attn_dq_kernel<NW>, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds_q) != hipSuccess) \
            return aether_set_error(AETHER_ERR_LAUNCH, "relbias_attn_bwd: the workgroup's LDS could not be set"); \
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
