// What the kernels of latent attention share (latent_attend.hip, latent_flash.hip): rows from memory to LDS, the
// transposing read of values, values that are not finite.
#pragma once

#include "common.h"

namespace latent {

// A raw buffer of 32-bit data from `base` (wave-uniform) up, its bounds left to the caller's offsets.
TS_DEV u32x4 rows_buffer(const void *base) {
    const uint64_t a = (uint64_t)(uintptr_t)base;
    return u32x4{(uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)a),
                 (uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)(a >> 32)) & 0xffffu, 0xffffffffu, 0x00020000u};
}
TS_DEV uint32_t lds_address(const void *p) { return (uint32_t)(uintptr_t)(ts_lds *)p; }

// 16 bytes a lane from `buf` (byte offset `at`, a lane's) straight to LDS: the lane lands at `lds` + 16 lane. Written out,
// because with the builtin's load on its way the compiler waits for all loads before a transposing read of LDS, whatever
// it reads. Nothing but LDS (and m0, which nothing else of these kernels uses) is written, and only the caller's own
// waits (vmcnt) tell when: a barrier after them, before any read. (Five wait states between a vector instruction that writes
// a scalar register and a load that reads it are the program's to keep, and the compiler does not look into the text.)
TS_DEV void rows_to_lds16(u32x4 buf, uint32_t lds, uint32_t at) {
#ifdef __HIP_DEVICE_COMPILE__
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds"
                 :: "s"(lds), "v"(at), "s"(buf)
                 : "memory");
#endif
}

typedef short ts_v4i16 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) ts_v4i16 lds_v4i16;
// Four keys of one d, from the 8-byte pieces of four rows (lane 4 e + c of 16: row e, d 4 c ..).
TS_DEV u32x2 read_vt4(const char *a) {
    return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4i16 *)a));
}

// The bits of the bf16 values of a pair that are not finite. (All ones are a NaN.)
TS_DEV uint32_t odd_mask(uint32_t x) {
    return ((x & 0x7f80u) == 0x7f80u ? 0xffffu : 0u) | ((x & 0x7f800000u) == 0x7f800000u ? 0xffff0000u : 0u);
}

// c, or NaN once a pair of bf16 values holds one that is not finite (0 times it).
TS_DEV float odd_sum(uint32_t x, float c) {
    return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(ts_bf16x2, x), __builtin_bit_cast(ts_bf16x2, 0u), c, false);
}

// A lane's number that what follows is computed from where it is used: rare steps' addresses would otherwise be
// computed ahead of the loops, and push what the common ones use out of the registers.
TS_DEV uint32_t again(uint32_t v) {
    asm volatile("" : "+v"(v));
    return v;
}
// A value worked out here, not where it is used.
TS_DEV void pinned(float &v) { asm volatile("" : "+v"(v)); }
TS_DEV void pinned(uint32_t &v) { asm volatile("" : "+v"(v)); }

}  // namespace latent
