// New rows into the kept rows: q and k pass through RmsNorm per head (with gains) and the rotation
// of their position (with an angle table), k and v are kept in bf16 rows or in e4m3 blocks.
//
//   y = x * gain / sqrt(mean(x^2) + eps)         (a, b) -> (a cos - b sin, a sin + b cos)
//   blocks: scale = 2^e, e the least with amax <= 448 * 2^e over the block's values;
//           code = e4m3(y / scale), round to nearest even
//
// No counterpart in the reference, whose kept rows are bf16 and whose append follows separate
// norm and rotation stages (engine/models/src/shared.rs:109-145, engine/ir/interp/src/
// run.rs:122-198).
//
// A head's row is 16 lanes' work, eight values each (four pairs of the rotation), so a wave takes four rows at
// once, in 16-byte loads, and a row's sum of squares needs no step across rows of lanes.
//
// The unit of work for k and v is a segment: rows r, r + 1, ... of the call that are consecutive positions
// of one slot within one block of 16. One wave owns a segment's kv head, lane group g (16 lanes) the block's
// positions 4 g .. 4 g + 3: it sees all new values of the block's head, so the scale, the codes and
// (where the scale grows) the codes already there are settled without another launch or an atomic, and
// four positions of a d are one word of V's block. The rows of a call that meet in a block must
// therefore stand together; a later segment of the same block is refused (TS_STATUS_TWICE), found by
// looking through the rows before it.
//
// Many rows are bound by HBM: 6 ragged prompts of up to 2048 f32 rows, 16 + 2 x 8 heads, into blocks, 250 MB: 52 to
// 64 us, 3.9 to 4.8 TB/s. Few by a chain of loads (position, page, row, scale, held codes): one row 4.6 us, 200 into
// bf16 rows 5.9, 48 x 5 into begun blocks 10.4.
// The look through the rows before grows with the square of the rows: a prompt of 32768 rows takes 221 us (186 at the
// rate of a large copy), of 65536 508 (372), of 131072 1290 (744). Longer ones are best appended in parts.
#include "kept8.h"

namespace {

using namespace kept8;

struct AppendParams {
    const void *q, *k, *v;
    const float *q_gain, *k_gain;
    const float2 *turns;
    void *q_out, *k_kept, *v_kept;
    float *scales;
    const uint32_t *slots, *positions;
    uint32_t *status;
    Place place;
    uint32_t rows, heads, kv_heads, q_stride, k_stride, v_stride;
    uint32_t window, kv_groups;      // rows a kv group looks at, and how many such groups there are
    uint32_t q_rows, head_quads;     // rows a wave of q heads takes, fours of q heads a row
    float eps;
    int q_out_bf16;
    int fours;  // slots and positions are 16-byte aligned
};

constexpr uint32_t kQRows = 4;

// The lane's eight values of a 128-wide row, in memory order: 4 l .. and 64 + 4 l .. (pairs (j, j + 64)), or
// 8 l .. (pairs (2j, 2j + 1)); pair k is values pa(k), pb(k), its angle 4 l + k.
template <bool HALVES>
struct Lanes {
    static TS_DEV uint32_t at(uint32_t l, uint32_t half) { return HALVES ? 4 * l + 64 * half : 8 * l + 4 * half; }
    static TS_DEV constexpr int pa(int k) { return HALVES ? k : 2 * k; }
    static TS_DEV constexpr int pb(int k) { return HALVES ? k + 4 : 2 * k + 1; }
};

// The lane's values of a row `row` elements past x (uniform, so that the address is a scalar base and a
// 32-bit offset).
template <bool XBF16, bool HALVES>
TS_DEV void load8(const void *x, uint32_t row, uint32_t l, float (&v)[8]) {
#pragma unroll
    for (int half = 0; half < 2; half++) {
        const uint32_t at = row + Lanes<HALVES>::at(l, half);
        if (XBF16) {
            const u32x2 w = *(const u32x2 *)((const char *)x + (uint32_t)(at * 2));
            v[4 * half] = lo_bf16(w.x);
            v[4 * half + 1] = hi_bf16(w.x);
            v[4 * half + 2] = lo_bf16(w.y);
            v[4 * half + 3] = hi_bf16(w.y);
        } else {
            const f32x4 w = *(const f32x4 *)((const char *)x + (uint32_t)(at * 4));
#pragma unroll
            for (int e = 0; e < 4; e++) v[4 * half + e] = w[e];
        }
    }
}
// Element `row` rows of `stride` on, as load8's uniform base.
template <bool XBF16>
TS_DEV const void *row_base(const void *x, uint32_t row, uint32_t stride) {
    return (const char *)x + (size_t)row * stride * (XBF16 ? 2 : 4);
}

template <bool HALVES>
TS_DEV void store8_bf16(uint16_t *row, uint32_t l, const float (&v)[8]) {
#pragma unroll
    for (int half = 0; half < 2; half++)
        *(u32x2 *)(row + Lanes<HALVES>::at(l, half)) =
            u32x2{pack_bf16x2(v[4 * half], v[4 * half + 1]), pack_bf16x2(v[4 * half + 2], v[4 * half + 3])};
}

// RmsNorm of a head's row over its 16 lanes; of pairs (j, j + 64) in the order, and to the bits, of
// tessera_hip_qk_norm_rope_append.
template <bool HALVES>
TS_DEV void norm8(float (&v)[8], const float (&gain)[8], float eps) {
    float s[4];
#pragma unroll
    for (int k = 0; k < 4; k++) {
        const float a = v[Lanes<HALVES>::pa(k)], b = v[Lanes<HALVES>::pb(k)];
        s[k] = a * a + b * b;
    }
    const float inv = 1.0f / sqrtf(row16_sum((s[0] + s[1]) + (s[2] + s[3])) / 128.0f + eps);
#pragma unroll
    for (int k = 0; k < 8; k++) v[k] = v[k] * (inv * gain[k]);
}

// The rotation, each value rounded as tessera_hip_qk_norm_rope_append's.
template <bool HALVES>
TS_DEV void turn8(float (&v)[8], const f32x4 (&cs)[2]) {
#pragma unroll
    for (int k = 0; k < 4; k++) {
        const float c = cs[k / 2][2 * (k % 2)], sn = cs[k / 2][2 * (k % 2) + 1];
        float &a = v[Lanes<HALVES>::pa(k)], &b = v[Lanes<HALVES>::pb(k)];
        const float x = a, y = b;
        a = fmaf(x, c, -(y * sn));
        b = fmaf(y, c, x * sn);
    }
}

// Rows that become codes are normed and rotated in f64 and come back as f32 rounded to odd (cut off, the last bit
// set where anything was), so that the code is the nearest to the formula's value and the scale the least for it:
// from f32 steps one code in a million or so is its neighbour, an eighth away. (6 prompts of up to 2048 rows: 63 us,
// in f32 61.)
TS_DEV float to_odd(double d) {
    const float f = (float)d;
    const uint64_t off = __builtin_bit_cast(uint64_t, d - (double)f);
    const uint32_t high = (uint32_t)(off >> 32), u = __float_as_uint(f);
    const uint32_t inexact = min((high & 0x7fffffffu) | (uint32_t)off, 1u), away = (high ^ u) >> 31;
    const uint32_t odd = (u - (away & inexact)) | inexact;
    return fabs(d) < __builtin_inf() ? __uint_as_float(odd) : f;  // (past f32's range its largest, cut off)
}
template <bool HALVES>
TS_DEV void norm_turn8(float (&v)[8], bool norm, const float (&gain)[8], float eps, bool turn, const f32x4 (&cs)[2]) {
    double inv = 1.0;
    if (norm) {
        double sum = 0.0;
#pragma unroll
        for (int k = 0; k < 8; k++) sum = __builtin_fma((double)v[k], (double)v[k], sum);
        const double mean = row16_total(sum) * (1.0 / 128.0) + (double)eps;
        inv = __builtin_amdgcn_rsq(mean);  // refined to 1e-15; 0 for infinity, as it is
        const double e = __builtin_fma(-mean * inv, inv, 1.0);
        inv = mean < __builtin_inf() ? __builtin_fma(inv * e, __builtin_fma(e, 0.375, 0.5), inv) : inv;
    }
#pragma unroll
    for (int k = 0; k < 4; k++) {  // (a pair at a time: all of them side by side in f64 would spill)
        float &a = v[Lanes<HALVES>::pa(k)], &b = v[Lanes<HALVES>::pb(k)];
        asm volatile("" : "+v"(a), "+v"(b));
        double x = a, y = b;
        if (norm) {
            x *= inv * (double)gain[Lanes<HALVES>::pa(k)];
            y *= inv * (double)gain[Lanes<HALVES>::pb(k)];
        }
        if (turn) {
            const double c = cs[k / 2][2 * (k % 2)], sn = cs[k / 2][2 * (k % 2) + 1];
            const double z = __builtin_fma(x, c, -(y * sn));
            y = __builtin_fma(y, c, x * sn);
            x = z;
        }
        a = to_odd(x);
        b = to_odd(y);
        asm volatile("" : "+v"(a), "+v"(b));
    }
}

template <bool HALVES>
TS_DEV void load_gain(const float *gain, uint32_t l, float (&g)[8]) {
#pragma unroll
    for (int half = 0; half < 2; half++) {
        const float *from = gain + Lanes<HALVES>::at(l, half);
#pragma unroll
        for (int e = 0; e < 4; e++) g[4 * half + e] = from[e];
    }
}

// The lane's four (cos, sin) `rows` rows past the table's uniform row.
TS_DEV void load_turns(const float2 *row, uint32_t rows, uint32_t l, f32x4 (&cs)[2]) {
    const char *from = (const char *)row;
    cs[0] = *(const f32x4 *)(from + (rows * 512 + l * 32));
    cs[1] = *(const f32x4 *)(from + (rows * 512 + l * 32 + 16));
}

TS_DEV float finite_abs(float x) {
    const float a = fabsf(x);
    return a < __builtin_inff() ? a : 0.0f;  // infinities and NaN take no part in the scale
}

// Four codes of x * inv, `inv` = 1 / scale: beyond the range the largest, NaN for infinities and NaN (the
// format has no infinity).
TS_DEV float coded(float x, float inv) {
    const float y = fminf(fmaxf(x * inv, -448.0f), 448.0f);
    return fabsf(x) < __builtin_inff() ? y : __builtin_nanf("");
}
TS_DEV uint32_t codes4(float a, float b, float c, float d, float inv) {
    const int w = __builtin_amdgcn_cvt_pk_fp8_f32(coded(a, inv), coded(b, inv), 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(coded(c, inv), coded(d, inv), w, true);
}

// Four codes held under one scale as codes under another (factor = old / new, a power of two <= 1).
TS_DEV uint32_t rebase4(uint32_t w, float factor) {
    float f[4];
    e4m3x4_to_f32(w, f);
    const int r = __builtin_amdgcn_cvt_pk_fp8_f32(f[0] * factor, f[1] * factor, 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(f[2] * factor, f[3] * factor, r, true);
}

// The segment's row at block position `at`, or the nearest: rows off .. off + n - 1 are written.
TS_DEV uint32_t segment_row(uint32_t at, uint32_t off, uint32_t n) {
    return (uint32_t)min(max((int)at - (int)off, 0), (int)n - 1);
}

// A segment of one row (a decode step's): 16 lanes a kv head's k or v, four of them a wave. A short way, as a
// step's few groups spend most of their time fetching code.
template <bool XBF16, bool KEPT8, bool HALVES>
TS_DEV void append_one(const AppendParams &p, uint64_t row0, uint32_t pos, uint32_t unit, uint32_t r, uint32_t l) {
    const uint32_t h = unit >> 1, is_v = unit & 1;
    if (h >= p.kv_heads) return;  // (16 lanes together)
    const void *k = row_base<XBF16>(p.k, r, p.k_stride), *from = row_base<XBF16>(p.v, r, p.v_stride);
    float v[8], x[8];
    load8<XBF16, HALVES>(is_v ? from : k, h * 128, l, v);
#pragma unroll
    for (int e = 0; e < 8; e++) x[e] = v[e];
    if (KEPT8 && (p.k_gain || p.turns)) {
        float gain[8] = {};
        f32x4 cs[2] = {};
        if (p.k_gain) load_gain<HALVES>(p.k_gain, l, gain);
        if (p.turns) load_turns(p.turns + (size_t)pos * 64, 0, l, cs);
        norm_turn8<HALVES>(x, p.k_gain, gain, p.eps, p.turns, cs);
    }
    if (!KEPT8 && p.k_gain) {
        float gain[8];
        load_gain<HALVES>(p.k_gain, l, gain);
        norm8<HALVES>(x, gain, p.eps);
    }
    if (!KEPT8 && p.turns) {
        f32x4 cs[2];
        load_turns(p.turns + (size_t)pos * 64, 0, l, cs);
        turn8<HALVES>(x, cs);
    }
#pragma unroll
    for (int e = 0; e < 8; e++) v[e] = is_v ? v[e] : x[e];
    if (!KEPT8) {
        store8_bf16<HALVES>((uint16_t *)(is_v ? p.v_kept : p.k_kept) + (row0 * p.kv_heads + h) * 128, l, v);
        return;
    }
    float amax = 0.0f;
#pragma unroll
    for (int k = 0; k < 8; k++) amax = fmaxf(amax, finite_abs(v[k]));
    amax = row16_max(amax);
    const uint32_t off = (uint32_t)row0 & (kBlock - 1);
    const uint64_t block = row0 / kBlock;
    float *scale_at = p.scales + (block * scale_heads(p.kv_heads) + h) * 2 + is_v;
    uint8_t *to = (uint8_t *)(is_v ? p.v_kept : p.k_kept) + (block * p.kv_heads + h) * kBlockBytes;
    int e = scale_exponent(amax), grow = 0;
    if (off) {  // positions are there: the scale only grows
        const int was = stored_exponent(*scale_at);
        e = max(e, was);
        grow = e - was;
    }
    if (grow) {  // all of the block; the new position's bytes are written after it
        const float factor = two_to(max(-grow, -126));
        u32x4 *at = (u32x4 *)to + l;
#pragma unroll 1
        for (uint32_t i = 0; i < kBlockBytes / 256; i++, at += 16) {
            const u32x4 w = *at;
            *at = u32x4{rebase4(w.x, factor), rebase4(w.y, factor), rebase4(w.z, factor), rebase4(w.w, factor)};
        }
        // Other lanes' words of the new position must be there before its bytes.
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    }
    const float inv = two_to(-e);
    const uint32_t lo = codes4(v[0], v[1], v[2], v[3], inv), hi = codes4(v[4], v[5], v[6], v[7], inv);
    if (!is_v) {
        *(uint32_t *)(to + off * kWidth + Lanes<HALVES>::at(l, 0)) = lo;
        *(uint32_t *)(to + off * kWidth + Lanes<HALVES>::at(l, 1)) = hi;
    } else {
#pragma unroll
        for (int k = 0; k < 8; k++)
            to[(Lanes<HALVES>::at(l, k / 4) + k % 4) * kBlock + off] = (uint8_t)((k < 4 ? lo : hi) >> (8 * (k % 4)));
    }
    if (l == 0) *scale_at = two_to(e);
}

// One segment of n rows of one kv head's k (or v), rows from r on, the first at kept row `row0`: x[i] is
// position 4 g + i, of the row's own values where the segment writes it, else of one of its rows (not used).
template <bool KEPT8, bool HALVES, bool IS_V>
TS_DEV void append_segment(const AppendParams &p, uint64_t row0, uint32_t pos, uint32_t n, uint32_t h, uint32_t lane,
                           float (&x)[4][8]) {
    const uint32_t g = lane >> 4, l = lane & 15, off = pos & (kBlock - 1);
    const uint32_t mine = (((1u << n) - 1) << off) >> (4 * g) & 15;
    const uint64_t first = row0 - off;  // kept row of the 16's position 0
    if (!IS_V && !KEPT8) {
        if (p.k_gain) {
            float gain[8];
            load_gain<HALVES>(p.k_gain, l, gain);
#pragma unroll
            for (uint32_t i = 0; i < 4; i++) norm8<HALVES>(x[i], gain, p.eps);
        }
        if (p.turns) {
            const float2 *row = p.turns + (size_t)pos * 64;
#pragma unroll
            for (uint32_t i = 0; i < 4; i++) {
                f32x4 cs[2];
                load_turns(row, segment_row(4 * g + i, off, n), l, cs);
                turn8<HALVES>(x[i], cs);
            }
        }
    } else if (!IS_V && (p.k_gain || p.turns)) {
        float gain[8] = {};
        if (p.k_gain) load_gain<HALVES>(p.k_gain, l, gain);
        const float2 *row = p.turns + (size_t)pos * 64;
#pragma unroll
        for (uint32_t i = 0; i < 4; i++) {
            f32x4 cs[2] = {};
            if (p.turns) load_turns(row, segment_row(4 * g + i, off, n), l, cs);
            norm_turn8<HALVES>(x[i], p.k_gain, gain, p.eps, p.turns, cs);
        }
    }
    if (!KEPT8) {
        char *to = (char *)(IS_V ? p.v_kept : p.k_kept) + (first * p.kv_heads + h) * 256;
#pragma unroll
        for (uint32_t i = 0; i < 4; i++)
            if (mine >> i & 1) store8_bf16<HALVES>((uint16_t *)(to + (4 * g + i) * (p.kv_heads * 256)), l, x[i]);
        return;
    }
    float amax = 0.0f;
#pragma unroll
    for (uint32_t i = 0; i < 4; i++)  // (positions not written hold one of the segment's rows)
#pragma unroll
        for (int k = 0; k < 8; k++) amax = fmaxf(amax, finite_abs(x[i][k]));
    amax = wave_max(amax);
    const uint64_t block = first / kBlock;
    float *scale_at = p.scales + (block * scale_heads(p.kv_heads) + h) * 2 + (IS_V ? 1 : 0);
    int e = scale_exponent(amax), grow = 0;
    if (off) {  // positions are there: the scale only grows
        const int was = stored_exponent(*scale_at);
        e = max(e, was);
        grow = e - was;
    }
    const float inv = two_to(-e), factor = two_to(max(-grow, -126));
    uint8_t *to = (uint8_t *)(IS_V ? p.v_kept : p.k_kept) + (block * p.kv_heads + h) * kBlockBytes;
    if (!IS_V) {
#pragma unroll
        for (uint32_t i = 0; i < 4; i++)
#pragma unroll
            for (int half = 0; half < 2; half++) {
                uint32_t *at = (uint32_t *)(to + (4 * g + i) * kWidth + Lanes<HALVES>::at(l, half));
                const float *v = x[i] + 4 * half;
                const uint32_t w = codes4(v[0], v[1], v[2], v[3], inv);
                if (mine >> i & 1)
                    *at = w;
                else if (grow)
                    *at = rebase4(*at, factor);
            }
    } else if (mine || grow) {  // the lane's eight d, four positions of each a word
        const uint32_t bytes = (mine & 1 ? 0xffu : 0) | (mine & 2 ? 0xff00u : 0) | (mine & 4 ? 0xff0000u : 0) |
                               (mine & 8 ? 0xff000000u : 0);
#pragma unroll
        for (int k = 0; k < 8; k++) {
            uint32_t *at = (uint32_t *)(to + (Lanes<HALVES>::at(l, k / 4) + k % 4) * kBlock + 4 * g);
            uint32_t w = codes4(x[0][k], x[1][k], x[2][k], x[3][k], inv) & bytes;
            if (mine != 15) {
                uint32_t held = *at;
                if (grow) held = rebase4(held, factor);
                w |= held & ~bytes;
            }
            *at = w;
        }
    }
    if (lane == 0) *scale_at = two_to(e);
}

constexpr uint32_t kWaves = 4;

template <bool XBF16, bool KEPT8, bool HALVES>
__global__ __launch_bounds__(64 * kWaves, KEPT8 ? 4 : 5) void append_kernel(AppendParams p) {
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    if (blockIdx.x >= p.kv_groups) {  // four q heads of q_rows rows a wave
        const uint32_t u = (blockIdx.x - p.kv_groups) * kWaves + wave, r0 = u / p.head_quads * p.q_rows, l = lane & 15;
        const uint32_t h = u % p.head_quads * 4 + (lane >> 4);
        if (r0 >= p.rows || h >= p.heads) return;  // (16 lanes together)
        float v[kQRows][8], gain[8];
        f32x4 cs[kQRows][2];
        bool held[kQRows];
        const uint32_t n = min(p.q_rows, p.rows - r0);
#pragma unroll
        for (uint32_t i = 0; i < kQRows; i++) {
            if (i >= n) continue;
            load8<XBF16, HALVES>(row_base<XBF16>(p.q, r0 + i, p.q_stride), h * 128, l, v[i]);
            const uint32_t slot = p.slots[r0 + i], pos = p.positions[r0 + i];
            if (p.turns) load_turns(p.turns + (pos < p.place.keys ? (size_t)pos * 64 : 0), 0, l, cs[i]);
            uint64_t row;  // (its page is asked for beside the angles)
            held[i] = holds(p.place, slot, pos) && row_of(p.place, slot, pos, row);
        }
        if (p.q_gain) load_gain<HALVES>(p.q_gain, l, gain);
#pragma unroll
        for (uint32_t i = 0; i < kQRows; i++) {
            if (i >= n) continue;
            if (p.q_gain) norm8<HALVES>(v[i], gain, p.eps);
            if (p.turns) turn8<HALVES>(v[i], cs[i]);
            if (!held[i]) {
#pragma unroll
                for (int k = 0; k < 8; k++) v[i][k] = __builtin_nanf("");
            }
            const size_t at = ((size_t)(r0 + i) * p.heads + h) * 128;
            if (p.q_out_bf16) {
                store8_bf16<HALVES>((uint16_t *)p.q_out + at, l, v[i]);
            } else {
#pragma unroll
                for (int half = 0; half < 2; half++)
                    *(f32x4 *)((float *)p.q_out + at + Lanes<HALVES>::at(l, half)) =
                        f32x4{v[i][4 * half], v[i][4 * half + 1], v[i][4 * half + 2], v[i][4 * half + 3]};
            }
        }
        return;
    }
    // k and v: the segments that begin among the window's rows, a wave a kv head's k or v.
    const uint32_t groups = (2 * p.kv_heads + kWaves - 1) / kWaves, first_unit = blockIdx.x % groups * kWaves;
    const uint32_t unit = first_unit + wave, h = unit >> 1, w0 = blockIdx.x / groups * p.window;
    const bool is_v = unit & 1, mine = h < p.kv_heads;
    const void *from = is_v ? p.v : p.k;
    const uint32_t stride = is_v ? p.v_stride : p.k_stride;
    // Lane i holds row w0 - 1 + i, of the window, the row before it and the 15 after it. A segment begins
    // where a row does not go on from the one before it, or begins a block.
    const uint32_t at = w0 + lane, ri = min(max(at, 1u) - 1, p.rows - 1), si = p.slots[ri], pi = p.positions[ri];
    const bool there = at >= 1 && at - 1 < p.rows;
    const uint32_t sb = __shfl_up((int)si, 1, 64), pb = __shfl_up((int)pi, 1, 64);  // (by every lane)
    const bool goes_on = lane && at >= 2 && sb == si && pb + 1 == pi && (pi & (kBlock - 1)) != 0;
    const uint64_t begins = __builtin_amdgcn_ballot_w64(there && !goes_on);
    // Of the window's own rows, lanes 1 .. window.
    uint64_t todo = begins & (((uint64_t)2 << p.window) - 2);
    while (todo) {
        const uint32_t li = __builtin_ctzll(todo), r = w0 + li - 1;
        todo &= todo - 1;
        const uint32_t slot = __builtin_amdgcn_readlane(si, li), pos = __builtin_amdgcn_readlane(pi, li);
        const uint32_t off = pos & (kBlock - 1);
        // It ends where the next one begins, or the rows do.
        const uint64_t next = begins >> li >> 1;
        const uint32_t count = min(next ? __builtin_ctzll(next) + 1 : kBlock, min(p.rows - r, kBlock - off));
        // Rows that a slot cannot hold: nothing is kept of them.
        uint32_t n = holds(p.place, slot, pos) ? min(count, p.place.keys - pos) : 0;
        uint32_t bad = n < count ? TS_STATUS_POSITION : 0;
        if (slot >= p.place.slot_count) bad = TS_STATUS_PAGE;
        const bool one = n == 1;  // 16 units a group instead of 4: the first groups do them all
        if (one && first_unit * 4 >= 2 * p.kv_heads) continue;
        float x[4][8];
        if (n && mine && !one) {
            const void *base = row_base<XBF16>(from, r, stride);
#pragma unroll
            for (uint32_t i = 0; i < 4; i++)
                load8<XBF16, HALVES>(base, segment_row(4 * (lane >> 4) + i, off, n) * stride + h * 128, lane & 15, x[i]);
        }
        uint64_t row0 = 0;
        if (n && !row_of(p.place, slot, pos, row0)) {
            bad |= TS_STATUS_PAGE;
            n = 0;
        }
        // A segment of the same block before this one in the call: the two would race. (Looked for while
        // the rows come.)
        bool twice = false;
        auto meets = [&](uint32_t sj, uint32_t pj) { return sj == slot && pj / kBlock == pos / kBlock; };
        const uint32_t whole = p.fours ? r & ~3u : 0;  // rows looked at four at a time
#pragma unroll 2
        for (uint32_t j = threadIdx.x * 4; j < whole; j += 256 * kWaves) {
            const u32x4 a = *(const u32x4 *)(p.slots + j), b = *(const u32x4 *)(p.positions + j);
#pragma unroll
            for (uint32_t e = 0; e < 4; e++) twice |= meets(a[e], b[e]);
        }
        for (uint32_t j = whole + threadIdx.x; j < r; j += 64 * kWaves) twice |= meets(p.slots[j], p.positions[j]);
        if (r && __syncthreads_or(twice)) {
            bad |= TS_STATUS_TWICE;
            n = 0;
        }
        if (bad && p.status && threadIdx.x == 0) atomicOr(p.status, bad);
        if (!n) continue;
        if (one)
            append_one<XBF16, KEPT8, HALVES>(p, row0, pos, 4 * unit + (lane >> 4), r, lane & 15);
        else if (!mine)
            continue;
        else if (is_v)
            append_segment<KEPT8, HALVES, true>(p, row0, pos, n, h, lane, x);
        else
            append_segment<KEPT8, HALVES, false>(p, row0, pos, n, h, lane, x);
    }
}

}  // namespace

int ts::kept_check(const char *rule, const uint32_t *table, uint32_t page, uint32_t keys, uint32_t slot_count,
                   uint32_t kept_pages, uint32_t pages, bool blocks) {
    TS_REQUIRE(keys >= 1 && slot_count >= 1, "%s: %u positions a slot, %u slots", rule, keys, slot_count);
    TS_REQUIRE(page >= 16 && (page & (page - 1)) == 0, "%s: page %u must be a power of two >= 16", rule, page);
    if (table) {
        TS_REQUIRE(kept_pages >= 1 && pages >= 1, "%s: %u table entries a slot, %u pages", rule, kept_pages, pages);
    } else {
        TS_REQUIRE(!blocks || keys % 16 == 0, "%s: dense blocks need %u positions a slot to be whole blocks", rule, keys);
        TS_REQUIRE((uint64_t)slot_count * keys <= (uint64_t)pages * page, "%s: %u slots of %u positions, kept rows hold %llu",
                   rule, slot_count, keys, (unsigned long long)pages * page);
    }
    return TS_OK;
}

extern "C" int tessera_hip_append_rows(const ts_append_args *a, void *stream) {
    TS_REQUIRE(a, "append_rows: null args");
    const bool some = a->rows != 0;  // (what has an element a row may be NULL without rows)
    TS_REQUIRE(a->k_kept && a->v_kept && (!some || (a->k && a->v && a->slots && a->positions)), "append_rows: null pointer");
    TS_REQUIRE(a->width == 128, "append_rows: head width %u (128 supported)", a->width);
    TS_REQUIRE(a->kv_heads >= 1 && a->kv_heads <= 1024, "append_rows: %u kv heads", a->kv_heads);
    TS_REQUIRE(a->x_dtype == TS_F32 || a->x_dtype == TS_BF16, "append_rows: rows f32 or bf16 supported");
    TS_REQUIRE(a->kv_dtype == TS_BF16 || a->kv_dtype == TS_E4M3, "append_rows: kept rows bf16 or e4m3 blocks supported");
    const bool blocks = a->kv_dtype == TS_E4M3;
    TS_REQUIRE(!blocks || a->scales, "append_rows: e4m3 blocks need their scales");
    int rc = ts::kept_check("append_rows", a->kept_table, a->page, a->keys, a->slot_count, a->kept_pages, a->pages, blocks);
    if (rc) return rc;
    TS_REQUIRE(!a->rope_table || a->rope_rows >= a->keys, "append_rows: positions up to %u but the angle table has %u rows",
               a->keys - 1, a->rope_rows);
    const uint32_t unit = a->x_dtype == TS_F32 ? 4 : 8;  // 16 bytes
    TS_REQUIRE(a->k_stride >= a->kv_heads * 128 && a->v_stride >= a->kv_heads * 128 && a->k_stride % unit == 0 &&
                   a->v_stride % unit == 0,
               "append_rows: rows %u and %u apart must hold %u kv heads and be whole 16-byte pieces", a->k_stride,
               a->v_stride, a->kv_heads);
    TS_REQUIRE(a->k_stride <= 1u << 26 && a->v_stride <= 1u << 26, "append_rows: rows %u and %u apart", a->k_stride,
               a->v_stride);  // (16 rows within a 32-bit offset)
    TS_REQUIRE(ts::aligned(a->k, 16) && ts::aligned(a->v, 16) && ts::aligned(a->k_kept, 16) && ts::aligned(a->v_kept, 16) &&
                   ts::aligned(a->scales, 16) && ts::aligned(a->rope_table, 8),
               "append_rows: k, v, kept rows and scales must be 16-byte aligned, the angle table 8");
    const bool q = a->q != nullptr;
    if (q) {
        TS_REQUIRE(a->q_out || !some, "append_rows: q without q_out");
        TS_REQUIRE(a->heads >= 1 && a->heads <= 16384, "append_rows: %u heads", a->heads);
        TS_REQUIRE(a->q_stride >= a->heads * 128 && a->q_stride % unit == 0,
                   "append_rows: q rows %u apart must hold %u heads and be whole 16-byte pieces", a->q_stride, a->heads);
        TS_REQUIRE(a->q_out_dtype == TS_F32 || a->q_out_dtype == TS_BF16, "append_rows: q out f32 or bf16 supported");
        TS_REQUIRE(ts::aligned(a->q, 16) && ts::aligned(a->q_out, 16), "append_rows: q must be 16-byte aligned");
        TS_REQUIRE(a->q_out != a->q || (a->q_out_dtype == a->x_dtype && a->q_stride == a->heads * 128),
                   "append_rows: q in place needs rows back to back of the same type");
    }
    if (!some) return TS_OK;
    AppendParams p;
    p.q = a->q; p.k = a->k; p.v = a->v; p.q_gain = a->q_gain; p.k_gain = a->k_gain;
    p.turns = (const float2 *)a->rope_table;
    p.q_out = a->q_out; p.k_kept = a->k_kept; p.v_kept = a->v_kept; p.scales = a->scales;
    p.slots = a->slots; p.positions = a->positions; p.status = a->status;
    p.place.table = a->kept_table; p.place.keys = a->keys; p.place.slot_count = a->slot_count;
    p.place.kept_pages = a->kept_pages; p.place.page_shift = (uint32_t)__builtin_ctz(a->page);
    p.place.pages = a->pages;
    p.rows = a->rows; p.heads = a->heads; p.kv_heads = a->kv_heads;
    p.q_stride = a->q_stride; p.k_stride = a->k_stride; p.v_stride = a->v_stride;
    p.eps = a->eps; p.q_out_bf16 = a->q_out_dtype == TS_BF16;
    p.fours = ts::aligned(a->slots, 16) && ts::aligned(a->positions, 16);
    // Few rows are taken for a decode step, a segment each: a group looks at one row. Of many, most
    // go on from the row before them, and a group looks at 16; and a wave of q heads takes four rows,
    // whose loads are in flight together. (A group looking at one row, or at 16, into blocks: 256 decode rows 12 and
    // 53 us, 1024 36 and 57, 2048 68 and 82, 4096 150 and 143; 128 x 9 drafted rows 21 and 29, 200 x 9 32 and 33, 512 x
    // 9 87 and 70. A prompt by itself, which the count does not tell from them, takes 12 and 8 at 256 rows, 26 and 12
    // at 1024, 46 and 16 at 2048.)
    const bool few = a->rows <= 1024;
    p.window = few ? 1 : 16;
    p.q_rows = few ? 1 : kQRows;
    const uint64_t kv = (uint64_t)((a->rows + p.window - 1) / p.window) * ((2 * a->kv_heads + kWaves - 1) / kWaves);
    p.head_quads = (a->heads + 3) / 4;
    const uint64_t units = q ? (uint64_t)((a->rows + p.q_rows - 1) / p.q_rows) * p.head_quads : 0;
    const uint64_t all = kv + (units + kWaves - 1) / kWaves;
    TS_REQUIRE(all <= 0x7fffffffull, "append_rows: %u rows in one launch", a->rows);
    p.kv_groups = (uint32_t)kv;
    const int pick = (a->x_dtype == TS_BF16 ? 4 : 0) | (blocks ? 2 : 0) | (a->halves ? 1 : 0);
    void (*const kernels[8])(AppendParams) = {
        append_kernel<false, false, false>, append_kernel<false, false, true>, append_kernel<false, true, false>,
        append_kernel<false, true, true>,   append_kernel<true, false, false>, append_kernel<true, false, true>,
        append_kernel<true, true, false>,   append_kernel<true, true, true>};
    hipLaunchKernelGGL(kernels[pick], dim3((uint32_t)all), dim3(64 * kWaves), 0, (hipStream_t)stream, p);
    TS_CHECK_LAUNCH("append_rows launch");
    return TS_OK;
}
