// Kept blocks: kept rows in 8 bits. A block is 16 positions of one kv head, e4m3 codes times a
// power of two for K and another for V:
//   k       [blocks][kv_heads][16 positions][128]
//   v       [blocks][kv_heads][128][16 positions]
//   scales  [blocks][kv_heads rounded up to even][2: K's, V's] f32
// A block's head is 2 KiB in one piece, so a kv head's keys stream in whole lines whatever the
// other heads do, and V stands with its positions innermost because that is the matrix unit's
// operand of P V. A power of two scales a code to bf16 exactly, on the conversion instruction
// itself, and lets an append move a begun block to a wider scale without rounding its codes anew
// (but for those that turn subnormal). scales are padded to even heads so that a page's scales
// are whole 16-byte pieces, as the page copies want.
#pragma once

#include "common.h"

namespace kept8 {

constexpr uint32_t kBlock = 16, kWidth = 128, kBlockBytes = kBlock * kWidth;
constexpr int kLeast = -100, kMost = 119;  // exponents of a scale: codes times it stay normal bf16 values

TS_DEV uint32_t scale_heads(uint32_t kv_heads) { return (kv_heads + 1) & ~1u; }

// The least e with amax <= 448 * 2^e (448 = 1.75 * 2^8), within the bounds.
TS_DEV int scale_exponent(float amax) {
    const uint32_t u = __float_as_uint(amax);
    const int e = (int)(u >> 23) - 127 - 8 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0);
    return min(max(e, kLeast), kMost);
}
// The exponent of a stored scale, whatever its other bits hold.
TS_DEV int stored_exponent(float scale) {
    return min(max((int)((__float_as_uint(scale) >> 23) & 255u) - 127, kLeast), kMost);
}
TS_DEV float two_to(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

// The position's place: page table entry (or the dense row), then the block of 16 within it.
struct Place {
    const uint32_t *table;  // NULL: dense, slot * keys + position
    uint32_t keys, slot_count, kept_pages, page_shift, pages;
};

// Whether (slot, pos) is one that the kept rows hold.
TS_DEV bool holds(const Place &p, uint32_t slot, uint32_t pos) {
    return pos < p.keys && slot < p.slot_count && (!p.table || (pos >> p.page_shift) < p.kept_pages);
}
// First kept row of the page (or dense 16 rows) that (slot, pos) is in, then pos's own row; false
// where the table names a page that the buffers do not hold. Only for places that hold.
TS_DEV bool row_of(const Place &p, uint32_t slot, uint32_t pos, uint64_t &row) {
    if (!p.table) {
        row = (uint64_t)slot * p.keys + pos;
        return true;
    }
    const uint32_t id = p.table[(uint64_t)slot * p.kept_pages + (pos >> p.page_shift)];
    const bool ok = id < p.pages;
    row = ((uint64_t)(ok ? id : 0) << p.page_shift) | (pos & ((1u << p.page_shift) - 1));
    return ok;
}

// Two e4m3 codes (the low or the high half of w) times a power of two, as packed bf16: exact.
template <bool HIGH>
TS_DEV uint32_t code_pair(uint32_t w, float scale) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, HIGH));
}
// Eight codes (two words) as a matrix operand.
TS_DEV bf16x8 codes8(uint32_t a, uint32_t b, float scale) {
    return as_bf16x8(u32x4{code_pair<false>(a, scale), code_pair<true>(a, scale), code_pair<false>(b, scale),
                           code_pair<true>(b, scale)});
}

// A byte of 0x80 for each NaN code (0x7f or 0xff) of w.
TS_DEV uint32_t nan_codes(uint32_t w) { return ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u; }

}  // namespace kept8

namespace ts {
// The argument checks that appends and the attention over kept blocks share (append.hip): the
// table, its page and how many pages and slots there are.
int kept_check(const char *rule, const uint32_t *table, uint32_t page, uint32_t keys, uint32_t slot_count,
               uint32_t kept_pages, uint32_t pages, bool blocks);
}  // namespace ts
