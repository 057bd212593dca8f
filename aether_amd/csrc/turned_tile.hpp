// 64 x 64 tiles of bf16 in LDS whose columns feed the matrix unit: LDS-DMA in, transposing reads out.
#pragma once
#include "common.hpp"

namespace aether {

// 16-byte LDS-DMA as in common.hpp (LDS destination: wave-uniform base + lane · 16; bytes beyond the descriptor are not fetched), in assembly: the compiler
// waits for every LDS-DMA it knows of before a transposing LDS read, the next tile's included.  The loops wait for their tiles themselves.
typedef int i32x4 __attribute__((ext_vector_type(4)));
AE_DEV i32x4 tt_rsrc(const void* base, unsigned bytes) {
    const uint64_t a = (uint64_t)base;
    return i32x4{__builtin_amdgcn_readfirstlane((int)(unsigned)a), __builtin_amdgcn_readfirstlane((int)(unsigned)(a >> 32) & 0xffff), __builtin_amdgcn_readfirstlane((int)bytes), 0x00020000};
}
AE_DEV unsigned tt_lds(const void* p) { return (unsigned)(uintptr_t)(const __attribute__((address_space(3))) char*)p; }
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"       // (that m0 is not preserved is what is meant)
AE_DEV void tt_dma16(i32x4 rsrc, unsigned voff, unsigned soff, unsigned lds_wave_base) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds" ::"s"(lds_wave_base), "v"(voff), "s"(rsrc), "s"(soff) : "memory", "m0");
}
#pragma clang diagnostic pop

// A 64 x 64 tile in LDS: 128-byte rows, the 16-byte chunk c of row r stands at c ^ swz(r).  swz takes all eight values over r's bits 1 ... 3, so that 32 rows
// read at one chunk spread over the banks; and rows r, r + 2 differ in its bit 1, so that the 4 x 32-byte pieces of a transposing read do too.
AE_DEV int tt_swz(int r) { return (((r >> 1) & 3) << 1) | ((r >> 3) & 1); }

// offsets of a lane's transposed fragments: column 32 dt + (lane & 31), rows 8hi + 4f ... + 3 of 16; 16 rows further the swizzle is the same
AE_DEV void tt_offsets(int lane, int (&off)[2][2]) {
    const int i = lane & 15, hi = lane >> 5;
#pragma unroll
    for (int dt = 0; dt < 2; ++dt)
#pragma unroll
        for (int f = 0; f < 2; ++f) {
            const int r = 8 * hi + 4 * f + (i >> 2), chunk = dt * 4 + ((lane >> 4) & 1) * 2 + ((i & 3) >> 1);
            off[dt][f] = r * 128 + ((chunk ^ tt_swz(r)) << 4) + (i & 1) * 8;
        }
}

// One transposed fragment: 16 rows from `at`, columns by off (tt_offsets of a 32-column half)
AE_DEV bf16x8 tt_read(const char* at, const int (&off)[2]) {
    typedef short s16x4 __attribute__((ext_vector_type(4)));
    typedef short s16x8 __attribute__((ext_vector_type(8)));
    const s16x4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(at + off[0]));
    const s16x4 y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(at + off[1]));
    return __builtin_bit_cast(bf16x8, s16x8{x[0], x[1], x[2], x[3], y[0], y[1], y[2], y[3]});
}

AE_DEV void tt_landed() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

}  // namespace aether
