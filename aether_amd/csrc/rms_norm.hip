// Root-mean-square norm of a residual stream, with the residual's addition, an output in bf16 or in 8 bits, and the backward pass.
//
//   h = x + delta                      (x: the stream, fp32 or bf16; delta: a block's output, bf16; h goes back into the stream)
//   y = h · r · w,   r = (mean(h²) + eps)^-1/2
//   8 bits:  s = the smallest power of two with max|y| / s <= 448,  q = e4m3(y / s)      (one s per row)
//   backward, n = dy · w, ĥ = h · r:   dx = r (n − ĥ · mean(n ĥ)) + dres,   ddelta = dx,   dw = Σ_rows dy · ĥ
//
// A power of two as scale makes the division exact, so that e4m3's rounding is the only one; e4m3 is a floating format, a scale that is up to
// twice as large as max/448 costs it precision only among its subnormals (values below max · 2^-14).
// The norm is taken of the fp32 sum, before it is rounded into a bf16 stream.  All statistics are fp32.
//
// What bounds it: HBM.  A row stays in registers between its statistics and its output, so every tensor is read and written once.  A workgroup
// owns whole rows and walks rows g, g + G, ...: w stays in its registers, and the next row is requested before the present one is reduced.
// WPR waves share a row (1 up to 1024 elements, 4 above), NCH chunks of 8 elements a lane: D <= WPR·64·8·NCH.
//
// Measured (a large copy on this card moves 4.9 TB/s): 14464 x 4096, fp32 stream with delta, e4m3 out: 652 MB in 124 µs, 5.3 TB/s; 3616 x 4096 forward and backward:
// 415 MB in 79 µs, 5.3 TB/s; 226 x 4096: 10.6 µs, what a call costs on the host (the kernel itself 4.4).
#include "common.hpp"
#include "../../include/aether_hip.h"

namespace aether {

typedef unsigned char u8_t;

struct RmsArgs {
    const void* x; long ldx;           // stream in
    const bf16_t* delta; long ldd;     // or null
    void* res; long ldr;               // stream out, or null
    const float* w;
    void* y; long ldy;                 // bf16, or e4m3
    float* scale;                      // e4m3: one per row
    int rows, D;
    float eps, inv_d;
};

struct RmsBwdArgs {
    const bf16_t* dy; long lddy;
    const void* res; long ldr;         // h as the forward pass stored it; with delta the stream before the addition
    const bf16_t* delta; long ldd;     // or null
    const void* dres; long lddr;       // the gradient that reaches h from elsewhere, stream type, or null
    const float* w;
    void* dx; long lddx;               // stream type
    bf16_t* ddelta; long ldds;         // or null
    float* part;                       // [gridDim.x · 4/WPR][D]: Σ dy·ĥ over the rows that one row slot of the grid walked
    int rows, D;
    float eps, inv_d;
};

// eight elements of a row, from a stream of either type, as fp32
template <class T> struct Raw8;
template <> struct Raw8<float> { f32x4 a, b; };
template <> struct Raw8<bf16_t> { u16x8 a; };
AE_DEV void load8(Raw8<float>& r, const float* p) { r.a = *(const f32x4*)p; r.b = *(const f32x4*)(p + 4); }
AE_DEV void load8(Raw8<bf16_t>& r, const bf16_t* p) { r.a = *(const u16x8*)p; }
AE_DEV float get8(const Raw8<float>& r, int e) { return e < 4 ? r.a[e] : r.b[e - 4]; }
AE_DEV float get8(const Raw8<bf16_t>& r, int e) { return bf16_bits_to_f32(r.a[e]); }
AE_DEV void store8(float* p, const float (&v)[8]) {
    *(f32x4*)p = f32x4{v[0], v[1], v[2], v[3]};
    *(f32x4*)(p + 4) = f32x4{v[4], v[5], v[6], v[7]};
}
AE_DEV void store8(bf16_t* p, const float (&v)[8]) {
    *(uint4*)p = make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7]));
}
AE_DEV unsigned wave_max_u32(unsigned v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v = max(v, (unsigned)__shfl_xor((int)v, o, 64));
    return v;
}

// Two sums over the WPR waves of a row, the same in every lane.  `slot` alternates between calls, so that one barrier per call is enough: a wave that
// writes slot s again has passed the barrier of the call in between, which every reader of the first use reached after its reads.
template <int WPR>
AE_DEV void row_sums(float& a, float& b, float (&lds)[2][8], int& slot, int wave) {
    a = wave_sum(a);
    b = wave_sum(b);
    if constexpr (WPR > 1) {
        if ((threadIdx.x & 63) == 0) { lds[slot][wave] = a; lds[slot][4 + wave] = b; }
        __syncthreads();
        a = (lds[slot][0] + lds[slot][1]) + (lds[slot][2] + lds[slot][3]);
        b = (lds[slot][4] + lds[slot][5]) + (lds[slot][6] + lds[slot][7]);
        slot ^= 1;
    }
}
template <int WPR>
AE_DEV float row_sum(float a, float (&lds)[2][8], int& slot, int wave) {
    a = wave_sum(a);
    if constexpr (WPR > 1) {
        if ((threadIdx.x & 63) == 0) lds[slot][wave] = a;
        __syncthreads();
        a = (lds[slot][0] + lds[slot][1]) + (lds[slot][2] + lds[slot][3]);
        slot ^= 1;
    }
    return a;
}
template <int WPR>
AE_DEV unsigned row_max_u32(unsigned v, float (&lds)[2][8], int& slot, int wave) {
    v = wave_max_u32(v);
    if constexpr (WPR > 1) {
        if ((threadIdx.x & 63) == 0) lds[slot][wave] = __uint_as_float(v);
        __syncthreads();
        v = max(max(__float_as_uint(lds[slot][0]), __float_as_uint(lds[slot][1])), max(__float_as_uint(lds[slot][2]), __float_as_uint(lds[slot][3])));
        slot ^= 1;
    }
    return v;
}

// The scale of a row whose largest magnitude has the bits `top`: the smallest power of two with value / scale <= 448, not below 2^-126.
// 448 = 1.75 · 2^8: the exponent of top / 448, one up where its mantissa is above 1.75.  A row that holds an infinity or a NaN (as unsigned numbers
// both are above every finite magnitude) has no scale: it becomes NaN throughout, as one such element makes every product with the row.
struct RowScale {
    int e;
    bool bad;
    AE_DEV explicit RowScale(unsigned top) : e(max((int)(top >> 23) - 127 - 8 + ((top & 0x7fffffu) > 0x600000u ? 1 : 0), -126)), bad(top >= 0x7f800000u) {}
    AE_DEV float value() const { return bad ? __uint_as_float(0x7fc00000u) : __uint_as_float((unsigned)(127 + e) << 23); }
    AE_DEV uint2 pack(const float (&v)[8]) const {              // rounds to nearest even
        const float inv = bad ? __uint_as_float(0x7fc00000u) : __uint_as_float((unsigned)(127 - e) << 23);
        int lo = 0, hi = 0;
        lo = __builtin_amdgcn_cvt_pk_fp8_f32(v[0] * inv, v[1] * inv, lo, false);
        lo = __builtin_amdgcn_cvt_pk_fp8_f32(v[2] * inv, v[3] * inv, lo, true);
        hi = __builtin_amdgcn_cvt_pk_fp8_f32(v[4] * inv, v[5] * inv, hi, false);
        hi = __builtin_amdgcn_cvt_pk_fp8_f32(v[6] * inv, v[7] * inv, hi, true);
        return bad ? make_uint2(0x7f7f7f7fu, 0x7f7f7f7fu) : make_uint2((unsigned)lo, (unsigned)hi);
    }
};

template <class XT, int WPR, int NCH, bool E4M3>
__global__ __launch_bounds__(256) void rms_norm_kernel(RmsArgs p) {
    __shared__ float red[2][8];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int d0 = ((WPR == 1 ? 0 : wave * 64) + lane) * 8;
    constexpr int STEP = WPR * 512;                            // elements between a lane's chunks
    constexpr int RPB = 4 / WPR;                               // rows of a workgroup at a time
    const int rstep = gridDim.x * RPB;
    int slot = 0;
    float w[NCH][8];
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
        const int d = d0 + c * STEP;
#pragma unroll
        for (int e = 0; e < 8; ++e) w[c][e] = 0.f;
        if (d < p.D) {
            const f32x4 a = *(const f32x4*)(p.w + d), b = *(const f32x4*)(p.w + d + 4);
#pragma unroll
            for (int e = 0; e < 4; ++e) { w[c][e] = a[e]; w[c][e + 4] = b[e]; }
        }
    }
    Raw8<XT> x[NCH];
    u16x8 dl[NCH];
    auto fetch = [&](int row) {
#pragma unroll
        for (int c = 0; c < NCH; ++c) {
            const int d = d0 + c * STEP;
            if (d < p.D) {
                load8(x[c], (const XT*)p.x + (size_t)row * p.ldx + d);
                if (p.delta) dl[c] = *(const u16x8*)((const unsigned short*)p.delta + (size_t)row * p.ldd + d);
            }
        }
    };
    int row = (int)blockIdx.x * RPB + (WPR == 1 ? wave : 0);
    if (row < p.rows) fetch(row);
    // with WPR == 4 `row` is the same in all waves, so that they meet at the same barriers; with WPR == 1 there are none
    for (; row < p.rows; row += rstep) {
        float h[NCH][8];
        float sq = 0.f;
#pragma unroll
        for (int c = 0; c < NCH; ++c) {
            const bool in = d0 + c * STEP < p.D;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                float v = in ? get8(x[c], e) : 0.f;
                if (p.delta && in) v += bf16_bits_to_f32(dl[c][e]);
                h[c][e] = v;
                sq += v * v;
            }
        }
        if (row + rstep < p.rows) fetch(row + rstep);
        const float r = rsqrtf(row_sum<WPR>(sq, red, slot, wave) * p.inv_d + p.eps);
        if (p.res) {
#pragma unroll
            for (int c = 0; c < NCH; ++c) {
                const int d = d0 + c * STEP;
                if (d < p.D) store8((XT*)p.res + (size_t)row * p.ldr + d, h[c]);
            }
        }
#pragma unroll
        for (int c = 0; c < NCH; ++c)
#pragma unroll
            for (int e = 0; e < 8; ++e) h[c][e] = h[c][e] * r * w[c][e];
        if constexpr (!E4M3) {
#pragma unroll
            for (int c = 0; c < NCH; ++c) {
                const int d = d0 + c * STEP;
                if (d < p.D) store8((bf16_t*)p.y + (size_t)row * p.ldy + d, h[c]);
            }
        } else {
            // the largest |y| as an unsigned number: infinities and NaN are above every finite value, so that they are not lost
            unsigned top = 0;
#pragma unroll
            for (int c = 0; c < NCH; ++c)
#pragma unroll
                for (int e = 0; e < 8; ++e) top = max(top, d0 + c * STEP < p.D ? __float_as_uint(h[c][e]) & 0x7fffffffu : 0u);
            top = row_max_u32<WPR>(top, red, slot, wave);
            const RowScale sc(top);
            if (WPR == 1 ? lane == 0 : threadIdx.x == 0) p.scale[row] = sc.value();
#pragma unroll
            for (int c = 0; c < NCH; ++c) {
                const int d = d0 + c * STEP;
                if (d < p.D) *(uint2*)((u8_t*)p.y + (size_t)row * p.ldy + d) = sc.pack(h[c]);
            }
        }
    }
}

template <class XT, int WPR, int NCH, bool SUM>      // SUM: h is taken from the stream and delta
__global__ __launch_bounds__(256) void rms_norm_bwd_kernel(RmsBwdArgs p) {
    __shared__ float red[2][8];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int d0 = ((WPR == 1 ? 0 : wave * 64) + lane) * 8;
    constexpr int STEP = WPR * 512;
    constexpr int RPB = 4 / WPR;
    const int rstep = gridDim.x * RPB;
    const int first = (int)blockIdx.x * RPB + (WPR == 1 ? wave : 0);
    int slot = 0;
    float w[NCH][8], dw[NCH][8];
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
        const int d = d0 + c * STEP;
#pragma unroll
        for (int e = 0; e < 8; ++e) { w[c][e] = 0.f; dw[c][e] = 0.f; }
        if (d < p.D) {
            const f32x4 a = *(const f32x4*)(p.w + d), b = *(const f32x4*)(p.w + d + 4);
#pragma unroll
            for (int e = 0; e < 4; ++e) { w[c][e] = a[e]; w[c][e + 4] = b[e]; }
        }
    }
    Raw8<XT> x[NCH], dr[NCH];
    u16x8 g[NCH], dl[NCH];
    auto fetch = [&](int row) {
#pragma unroll
        for (int c = 0; c < NCH; ++c) {
            const int d = d0 + c * STEP;
            if (d < p.D) {
                load8(x[c], (const XT*)p.res + (size_t)row * p.ldr + d);
                g[c] = *(const u16x8*)((const unsigned short*)p.dy + (size_t)row * p.lddy + d);
                if (p.dres) load8(dr[c], (const XT*)p.dres + (size_t)row * p.lddr + d);
                if constexpr (SUM) dl[c] = *(const u16x8*)((const unsigned short*)p.delta + (size_t)row * p.ldd + d);
            }
        }
    };
    if (first < p.rows) fetch(first);
    for (int row = first; row < p.rows; row += rstep) {
        float h[NCH][8], n[NCH][8], o[NCH][8];                  // h, then dy, then what reaches h from elsewhere
        float sq = 0.f, dot = 0.f;                              // Σ h², Σ dy·w·h
#pragma unroll
        for (int c = 0; c < NCH; ++c) {
            const bool in = d0 + c * STEP < p.D;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                h[c][e] = in ? get8(x[c], e) : 0.f;
                if constexpr (SUM) h[c][e] += in ? bf16_bits_to_f32(dl[c][e]) : 0.f;
                n[c][e] = in ? bf16_bits_to_f32(g[c][e]) : 0.f;
                o[c][e] = in && p.dres ? get8(dr[c], e) : 0.f;
                sq += h[c][e] * h[c][e];
                dot += n[c][e] * w[c][e] * h[c][e];
            }
        }
        if (row + rstep < p.rows) fetch(row + rstep);
        row_sums<WPR>(sq, dot, red, slot, wave);
        const float r = rsqrtf(sq * p.inv_d + p.eps);
        const float mean = dot * r * p.inv_d;                   // mean(n ĥ)
#pragma unroll
        for (int c = 0; c < NCH; ++c) {
            const int d = d0 + c * STEP;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float hh = h[c][e] * r;
                dw[c][e] += n[c][e] * hh;
                o[c][e] += r * (n[c][e] * w[c][e] - hh * mean);
            }
            if (d < p.D) {
                store8((XT*)p.dx + (size_t)row * p.lddx + d, o[c]);
                if (p.ddelta) store8(p.ddelta + (size_t)row * p.ldds + d, o[c]);
            }
        }
    }
    // a slot without a row writes its zeros: the sum below reads all of them
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
        const int d = d0 + c * STEP;
        if (d < p.D) store8(p.part + (size_t)first * p.D + d, dw[c]);
    }
}

// dw[d] = Σ_s part[s][d], s ascending inside each of the 32 thread rows and then over them: the order depends on the sizes alone
__global__ __launch_bounds__(1024) void rms_norm_dw_kernel(const float* __restrict__ part, int slots, int D, float* __restrict__ dw) {
    __shared__ float red[32][33];
    const int c = threadIdx.x & 31, g = threadIdx.x >> 5;
    const int d = blockIdx.x * 32 + c;
    float s = 0.f;
    if (d < D)
        for (int i0 = g; i0 < slots; i0 += 8 * 32) {           // eight loads on their way together
            float v[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) v[k] = part[(size_t)min(i0 + 32 * k, slots - 1) * D + d];
#pragma unroll
            for (int k = 0; k < 8; ++k)
                if (i0 + 32 * k < slots) s += v[k];
        }
    red[g][c] = s;
    __syncthreads();
    if (g == 0 && d < D) {
        float t = 0.f;
#pragma unroll
        for (int i = 0; i < 32; ++i) t += red[i][c];
        dw[d] = t;
    }
}

// q = e4m3(x / s), s per row as in the norm above: the form in which gated_ff takes a weight matrix in 8 bits.  One workgroup per row, two passes
// over it (the second hits the caches); run once when weights are laid out: 10240 x 4096 in 25 µs, 126 MB at 5.0 TB/s.  A grid of 2^32 threads or more
// is cut short without an error, so a workgroup of a large matrix takes several rows.
constexpr int QUANT_WG = 1 << 20;
__global__ __launch_bounds__(256) void quantize_rows_kernel(const bf16_t* __restrict__ x, long ldx, u8_t* __restrict__ q, long ldq, float* __restrict__ scale, int rows, int K) {
    __shared__ float red[2][8];
    int slot = 0;
    for (int row = blockIdx.x; row < rows; row += gridDim.x) {
        const unsigned short* xr = (const unsigned short*)x + (size_t)row * ldx;
        unsigned top = 0;
        for (int k = threadIdx.x * 8; k < K; k += 2048) {
            const u16x8 v = *(const u16x8*)(xr + k);
#pragma unroll
            for (int e = 0; e < 8; ++e) top = max(top, ((unsigned)v[e] & 0x7fffu) << 16);
        }
        top = row_max_u32<4>(top, red, slot, threadIdx.x >> 6);
        const RowScale s(top);
        if (threadIdx.x == 0) scale[row] = s.value();
        for (int k = threadIdx.x * 8; k < K; k += 2048) {
            const u16x8 v = *(const u16x8*)(xr + k);
            float f[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) f[e] = bf16_bits_to_f32(v[e]);
            *(uint2*)(q + (size_t)row * ldq + k) = s.pack(f);
        }
    }
}

constexpr int RMS_MAX_D = 16384;
// workgroups of the backward pass: each leaves one partial row of dw per row slot
constexpr int RMS_BWD_WG = 512;

static int rms_grid(int rows, int rpb, int most) { return min((rows + rpb - 1) / rpb, most); }

static int rms_check(const void* x, int x_dtype, long rows, int D, const char* who) {
    if (x_dtype != AETHER_STREAM_BF16 && x_dtype != AETHER_STREAM_FP32) return aether_set_error(AETHER_ERR_ARG, "rms_norm: the stream is bf16 or fp32");
    if (rows < 0 || rows > (1l << 30)) return aether_set_error(AETHER_ERR_SHAPE, "rms_norm: rows must be in [0, 2^30]");
    if (D <= 0 || D % 8 != 0 || D > RMS_MAX_D) return aether_set_error(AETHER_ERR_SHAPE, "rms_norm: D must be a multiple of 8 up to 16384");
    if (rows > 0 && !x) return aether_set_error(AETHER_ERR_ARG, who);
    return AETHER_OK;
}

}  // namespace aether

using namespace aether;

// D -> waves per row and chunks per lane: one wave up to 1024 elements (no barrier), four above.  3616 rows, fp32: forward 5.1 ... 6.5 TB/s at 4096 ... 16384
// elements; backward 5.0 at 4096, 4.7 at 8192, 3.3 above, where a lane of four waves a row holds 64 elements of six vectors, more than its registers
// (eight waves a row are not built).
#define RMS_PICK(D, CALL)                     \
    do {                                      \
        if ((D) <= 512) { CALL(1, 1); }       \
        else if ((D) <= 1024) { CALL(1, 2); } \
        else if ((D) <= 2048) { CALL(4, 1); } \
        else if ((D) <= 4096) { CALL(4, 2); } \
        else if ((D) <= 8192) { CALL(4, 4); } \
        else { CALL(4, 8); }                  \
    } while (0)

extern "C" int aether_rms_norm(const void* x, int x_dtype, long ldx, const void* delta, long ldd, void* res, long ldr, const float* w, float eps,
                               void* y, long ldy, float* scale, int rows, int D, void* stream) {
    int rc = rms_check(x, x_dtype, rows, D, "rms_norm: null stream");
    if (rc) return rc;
    if (rows == 0) return AETHER_OK;
    if (!w || !y) return aether_set_error(AETHER_ERR_ARG, "rms_norm: null weight or output");
    if (delta && !res) return aether_set_error(AETHER_ERR_ARG, "rms_norm: a sum with delta needs a place (res)");
    if (ldx % 8 || (delta && ldd % 8) || (res && ldr % 8) || ldy % 8) return aether_set_error(AETHER_ERR_ALIGN, "rms_norm: leading dimensions must be multiples of 8");
    if (((uintptr_t)x | (uintptr_t)delta | (uintptr_t)res | (uintptr_t)w | (scale ? 0 : (uintptr_t)y)) & 15 || ((uintptr_t)y & 7))
        return aether_set_error(AETHER_ERR_ALIGN, "rms_norm: pointers must be 16-byte aligned");
    RmsArgs p = {x, ldx, (const bf16_t*)delta, ldd, res, ldr, w, y, ldy, scale, rows, D, eps, 1.0f / (float)D};
    hipStream_t s = (hipStream_t)stream;
#define RMS_FWD(WPR, NCH)                                                                                                       \
    do {                                                                                                                        \
        dim3 grid(rms_grid(rows, 4 / WPR, 2048));                                                                               \
        if (x_dtype == AETHER_STREAM_FP32) {                                                                                    \
            if (scale) hipLaunchKernelGGL((rms_norm_kernel<float, WPR, NCH, true>), grid, dim3(256), 0, s, p);                  \
            else hipLaunchKernelGGL((rms_norm_kernel<float, WPR, NCH, false>), grid, dim3(256), 0, s, p);                       \
        } else {                                                                                                                \
            if (scale) hipLaunchKernelGGL((rms_norm_kernel<bf16_t, WPR, NCH, true>), grid, dim3(256), 0, s, p);                 \
            else hipLaunchKernelGGL((rms_norm_kernel<bf16_t, WPR, NCH, false>), grid, dim3(256), 0, s, p);                      \
        }                                                                                                                       \
    } while (0)
    RMS_PICK(D, RMS_FWD);
#undef RMS_FWD
    return aether_check_launch("rms_norm");
}

extern "C" size_t aether_rms_norm_bwd_workspace_bytes(int rows, int D) {
    if (rows <= 0 || D <= 0 || D % 8 != 0 || D > RMS_MAX_D) return 0;
    const int rpb = D <= 1024 ? 4 : 1;
    return (size_t)rms_grid(rows, rpb, RMS_BWD_WG) * rpb * D * sizeof(float);
}

extern "C" int aether_rms_norm_bwd(const void* dy, long lddy, const void* res, int x_dtype, long ldr, const void* delta, long ldd, const void* dres, long lddr,
                                   const float* w, float eps, void* dx, long lddx, void* ddelta, long ldds, float* dw, int rows, int D, void* workspace, size_t workspace_bytes, void* stream) {
    int rc = rms_check(res, x_dtype, rows, D, "rms_norm_bwd: null stream");
    if (rc) return rc;
    if (!w || !dw) return aether_set_error(AETHER_ERR_ARG, "rms_norm_bwd: null weight or weight gradient");
    if (rows > 0 && (!dy || !dx)) return aether_set_error(AETHER_ERR_ARG, "rms_norm_bwd: null gradient");
    if (lddy % 8 || ldr % 8 || (delta && ldd % 8) || (dres && lddr % 8) || lddx % 8 || (ddelta && ldds % 8)) return aether_set_error(AETHER_ERR_ALIGN, "rms_norm_bwd: leading dimensions must be multiples of 8");
    if (((uintptr_t)dy | (uintptr_t)res | (uintptr_t)delta | (uintptr_t)dres | (uintptr_t)w | (uintptr_t)dx | (uintptr_t)ddelta | (uintptr_t)workspace) & 15)
        return aether_set_error(AETHER_ERR_ALIGN, "rms_norm_bwd: pointers must be 16-byte aligned");
    if (rows > 0 && (!workspace || workspace_bytes < aether_rms_norm_bwd_workspace_bytes(rows, D)))
        return aether_set_error(AETHER_ERR_ARG, "rms_norm_bwd: workspace too small (aether_rms_norm_bwd_workspace_bytes)");
    hipStream_t s = (hipStream_t)stream;
    int slots = 0;
    if (rows > 0) {
        RmsBwdArgs p = {(const bf16_t*)dy, lddy, res, ldr, (const bf16_t*)delta, ldd, dres, lddr, w, dx, lddx, (bf16_t*)ddelta, ldds, (float*)workspace, rows, D, eps, 1.0f / (float)D};
#define RMS_BWD(WPR, NCH)                                                                                                       \
    do {                                                                                                                        \
        dim3 grid(rms_grid(rows, 4 / WPR, RMS_BWD_WG));                                                                         \
        slots = grid.x * (4 / WPR);                                                                                             \
        if (x_dtype == AETHER_STREAM_FP32) {                                                                                    \
            if (delta) hipLaunchKernelGGL((rms_norm_bwd_kernel<float, WPR, NCH, true>), grid, dim3(256), 0, s, p);              \
            else hipLaunchKernelGGL((rms_norm_bwd_kernel<float, WPR, NCH, false>), grid, dim3(256), 0, s, p);                   \
        } else {                                                                                                                \
            if (delta) hipLaunchKernelGGL((rms_norm_bwd_kernel<bf16_t, WPR, NCH, true>), grid, dim3(256), 0, s, p);             \
            else hipLaunchKernelGGL((rms_norm_bwd_kernel<bf16_t, WPR, NCH, false>), grid, dim3(256), 0, s, p);                  \
        }                                                                                                                       \
    } while (0)
        RMS_PICK(D, RMS_BWD);
#undef RMS_BWD
        rc = aether_check_launch("rms_norm_bwd");
        if (rc) return rc;
    }
    hipLaunchKernelGGL(rms_norm_dw_kernel, dim3((D + 31) / 32), dim3(1024), 0, s, (const float*)workspace, slots, D, dw);
    return aether_check_launch("rms_norm_dw");
}

extern "C" int aether_quantize_rows_e4m3(const void* x, long ldx, void* q, long ldq, float* scale, int rows, int K, void* stream) {
    if (rows < 0 || rows > (1 << 30) || K <= 0 || K % 8 != 0 || K > (1 << 30)) return aether_set_error(AETHER_ERR_SHAPE, "quantize_rows: K must be a positive multiple of 8 up to 2^30, rows in [0, 2^30]");
    if (rows == 0) return AETHER_OK;
    if (!x || !q || !scale) return aether_set_error(AETHER_ERR_ARG, "quantize_rows: null operand");
    if (ldx % 8 || ldq % 8 || ((uintptr_t)x & 15) || ((uintptr_t)q & 7)) return aether_set_error(AETHER_ERR_ALIGN, "quantize_rows: rows must be 16-byte (x) and 8-byte (q) aligned");
    hipLaunchKernelGGL(quantize_rows_kernel, dim3(min(rows, QUANT_WG)), dim3(256), 0, (hipStream_t)stream, (const bf16_t*)x, ldx, (u8_t*)q, ldq, scale, rows, K);
    return aether_check_launch("quantize_rows");
}
