// What the kernels of the attention over kept blocks share (kept8.hip: a wave streams its own keys;
// kept8_rows.hip: a group's waves share them): tiles of columns, the softmax's pieces, partial results.
#pragma once

#include "kept8.h"

namespace kept8 {

constexpr uint32_t kStep = 64;           // keys a wave takes at a time
constexpr uint32_t kPart = 132;          // floats of a column's partial result: max, sum, 2 unused, 128
constexpr float kSlack = 8.0f;           // base-2 headroom of the softmax reference point

struct AttendParams {
    const void *q;
    const uint8_t *k, *v;
    const float *scales;
    void *out;
    // Where the keys are split: results of groups for a tile that an earlier group began, then for one that a
    // later group goes on with, each [groups][kv_heads][columns][kPart]; and each row tile's groups (first,
    // count). NULL: a group a tile.
    float *partials;
    uint32_t *shares;
    const uint32_t *slots, *positions;
    uint32_t *status;
    Place place;
    uint32_t rows, heads, kv_heads, group, back, max_position;
    uint32_t tile_rows, tiles, groups;  // rows a tile, row tiles, and groups a kv head
    float scale;
    int out_bf16;
};

// Tile gi: tile_rows rows from row0 and the q heads of one kv head, its columns row by row.
struct Tile {
    uint32_t row0, kvh;
    // Column c's row and q head; false where it has none.
    TS_DEV bool column(const AttendParams &p, uint32_t c, uint32_t &r, uint32_t &h) const {
        const uint32_t ri = c / p.group;
        r = row0 + ri;
        h = kvh * p.group + c % p.group;
        return ri < p.tile_rows && r < p.rows;
    }
};
TS_DEV float rows4_sum(float x) {
    const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = __uint_as_float(a[0]) + __uint_as_float(a[1]);
    const auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}
TS_DEV float rows4_max(float x) {
    const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    const auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}

// The least of the 16 lanes of a row, by DPP moves; uniform where the four rows hold the same.
template <int CTRL>
TS_DEV uint32_t dpp_u(uint32_t v) { return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xF, 0xF, false); }
TS_DEV uint32_t row16_least(uint32_t v) {
    v = min(v, dpp_u<0xB1>(v));
    v = min(v, dpp_u<0x4E>(v));
    v = min(v, dpp_u<0x141>(v));
    v = min(v, dpp_u<0x140>(v));
    return __builtin_amdgcn_readfirstlane(v);
}

TS_DEV void store4(const AttendParams &p, size_t at, f32x4 v) {
    if (p.out_bf16)
        *(u32x2 *)((uint16_t *)p.out + at) = u32x2{pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3])};
    else
        *(f32x4 *)((float *)p.out + at) = v;
}

// Bytes of a word of four positions pos .. pos + 3 that lie in [lo, hi].
TS_DEV uint32_t within4(uint32_t w, uint32_t pos, uint32_t lo, uint32_t hi) {
    uint32_t m = 0;
#pragma unroll
    for (uint32_t i = 0; i < 4; i++) m |= (pos + i >= lo && pos + i <= hi) ? 0xffu << (8 * i) : 0u;
    return w & m;
}

// Two f32 as packed bf16, rounded to nearest even; NaN stays NaN.
TS_DEV uint32_t bf16_pair(float a, float b) {
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(ts_f32x2{a, b}, ts_bf16x2));
}
// P parts of two f32 values: bf16 values that add up to them (24 bits in three parts, 16 in two, 8 in one).
template <uint32_t P>
TS_DEV void split_pair(float a, float b, uint32_t (&w)[P]) {
#pragma unroll
    for (uint32_t e = 0; e < P; e++) {
        w[e] = bf16_pair(a, b);
        if (e + 1 < P) {
            a -= lo_bf16(w[e]);
            b -= hi_bf16(w[e]);
        }
    }
}

// The table and the scales are read by scalar loads (their addresses are uniform), which return
// beside the codes' vector loads instead of behind them.
typedef const __attribute__((address_space(4))) uint32_t const_u32;
typedef const __attribute__((address_space(4))) float const_f32;
template <class T>
TS_DEV T in_constant(const void *p) { return (T)(uintptr_t)p; }

// Keeps what follows from being computed earlier: eight registers of codes at a time are widened,
// where the compiler would widen all of a step's and spill.
TS_DEV void pin(u32x4 &v) { asm volatile("" : "+v"(v)); }

// The kept block of key `key` of a slot, whose page is `id`; a page that is not held is lost, and page 0
// stands in its place.
TS_DEV uint32_t block_in(const Place &p, uint32_t slot, uint32_t id, uint32_t key, bool &lost) {
    lost = false;
    if (!p.table) return slot * (p.keys / kBlock) + key / kBlock;
    lost = id >= p.pages;
    if (lost) id = 0;
    return (id << (p.page_shift - 4)) + (key & ((1u << p.page_shift) - 1)) / kBlock;
}
TS_DEV uint32_t block_of(const Place &p, uint32_t slot, uint32_t key, bool &lost) {
    const_u32 *t = in_constant<const_u32 *>(p.table + (size_t)slot * p.kept_pages);
    return block_in(p, slot, p.table ? t[key >> p.page_shift] : 0, key, lost);
}

// Shared keys: a row tile is as many units of UNIT keys as its rows see, and the units of all tiles, one
// behind the other, are dealt to a kv head's groups in equal runs, so that all groups end together however
// the sequences differ in length. (A run's first and last tile are joined with other groups' by a second
// kernel.)
constexpr uint32_t kMaxShared = 256;  // tiles
struct Share {
    uint32_t unit, end, each;  // the group's units, and those of a group
    uint32_t tile;             // the tile of the first
};
// Group u's share, false where nothing is left for it. starts[t], in LDS, becomes tile t's first unit. Every
// wave works it out for itself, lane i for tiles i, i + 64 ..; a tile's units are told from its first and
// last row (those of one sequence, consecutive, or of two).
template <uint32_t UNIT>
TS_DEV bool share_of(const AttendParams &p, uint32_t u, uint32_t lane, uint32_t *starts, Share &s) {
    if (!p.partials) {
        s = Share{0, 1, 1, u};
        return true;
    }
    uint32_t end[4], all = 0;
#pragma unroll
    for (uint32_t k = 0; k < 4; k++) {
        end[k] = 0xffffffffu;
        if (64 * k >= p.tiles) break;
        const uint32_t t = 64 * k + lane;
        uint32_t n = 0;
        if (t < p.tiles) {
            const uint32_t r0 = t * p.tile_rows, r1 = min(r0 + p.tile_rows, p.rows) - 1;
            const uint32_t most = min(p.max_position, p.place.keys - 1);
            const uint32_t p0 = min(p.positions[r0], most), p1 = min(p.positions[r1], most);
            const uint32_t from0 = p0 > p.back ? p0 - p.back : 0, from1 = p1 > p.back ? p1 - p.back : 0;
            auto units = [](uint32_t lo, uint32_t hi) { return (hi - (lo & ~(kBlock - 1))) / UNIT + 1; };
            n = p.slots[r0] == p.slots[r1] ? units(min(from0, from1), max(p0, p1)) : units(from0, p0) + units(from1, p1);
            n = min(n, 1u << 22);
        }
        uint32_t upto = n;  // and the lanes' before
        upto += dpp_u<0x111>(upto);
        upto += dpp_u<0x112>(upto);
        upto += dpp_u<0x114>(upto);
        upto += dpp_u<0x118>(upto);
        const uint32_t a = __builtin_amdgcn_readlane(upto, 15), b = a + __builtin_amdgcn_readlane(upto, 31),
                       c = b + __builtin_amdgcn_readlane(upto, 47);
        upto += all + (lane < 16 ? 0 : lane < 32 ? a : lane < 48 ? b : c);
        all = __builtin_amdgcn_readlane(upto, 63);
        if (t < p.tiles) {
            end[k] = upto;
            starts[t + 1] = upto;
        }
    }
    starts[0] = 0;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");  // (each wave reads what it has written itself)
    s.each = (all + p.groups - 1) / p.groups;
    s.unit = u * s.each;
    s.end = min(s.unit + s.each, all);
    s.tile = 0;
#pragma unroll
    for (uint32_t k = 0; k < 4; k++) {
        if (64 * k >= p.tiles) break;
        s.tile += __builtin_popcountll(__builtin_amdgcn_ballot_w64(end[k] <= s.unit));
    }
    return s.unit < all;
}
// A group's part of a tile: units [a, b) of its n.
struct Part {
    uint32_t a, b, n, row0;
    float *partial;  // the columns' results, or NULL: out
};
TS_DEV Part part_of(const AttendParams &p, uint32_t u, uint32_t lane, uint32_t kvh, uint32_t columns,
                    const uint32_t *starts, const Share &s) {
    if (!p.partials) return Part{0, 1, 1, s.tile * p.tile_rows, nullptr};
    const uint32_t t0 = __builtin_amdgcn_readfirstlane(starts[s.tile]);
    const uint32_t t1 = __builtin_amdgcn_readfirstlane(starts[s.tile + 1]);
    Part part = {s.unit - t0, min(s.end, t1) - t0, t1 - t0, s.tile * p.tile_rows, nullptr};
    if (part.a || part.b < part.n)
        part.partial = p.partials + ((size_t)((part.a ? 0 : p.groups) + u) * p.kv_heads + kvh) * columns * kPart;
    if (part.a == 0 && lane == 0) {  // (by every wave and kv head alike)
        p.shares[2 * s.tile] = u;
        p.shares[2 * s.tile + 1] = (t1 - 1) / s.each - u + 1;
    }
    return part;
}
// Unit x of a tile's n, in a pass over np units of one slot: a tile of several slots is taken a slot at a time,
// each in the same proportion.
TS_DEV uint32_t pass_unit(uint32_t x, uint32_t n, uint32_t np) {
    if (x >= n) return np;
    if (n == np) return x;
    return min(np, (uint32_t)((float)x * ((float)np * __builtin_amdgcn_rcpf((float)n))));
}

// Which of a lane's 16 keys key0 .. key0 + 15 lie in [from, pos], a bit each.
TS_DEV uint32_t seen_keys(uint32_t key0, uint32_t from, uint32_t pos) {
    const int first = max((int)(from - key0), 0), end = min((int)(pos - key0) + 1, 16);
    const uint32_t upto = end <= 0 ? 0u : (1u << end) - 1;
    return first < 16 ? upto & (0xffffu << first) : 0u;
}

// The softmax of one column over a step's 64 keys: the lane's 16 raw scores (scaled by sl > 0 to base 2,
// -inf where masked) to weights 2^(score - m) in P bf16 parts, as the second product takes them
// (operand x: positions 8 x .. 8 x + 7 of the lane's block). m moves only when a score passes it by
// 2^kSlack, so most steps leave the sum and O as they are and no weight passes 2^kSlack; l adds up the
// lane's own keys. O (NO tiles) is rescaled when some column of the wave moved.
template <uint32_t P, int NO>
TS_DEV void weigh(const f32x4 (&s)[4], float sl, float &m, float &l, f32x4 (&o)[NO], bf16x8 (&w)[2][P]) {
    float mx = s[0][0];
#pragma unroll
    for (int t = 0; t < 4; t++)
#pragma unroll
        for (int e = 0; e < 4; e++) mx = fmaxf(mx, s[t][e]);
    mx = rows4_max(mx) * sl;
    const bool raise = mx > m + kSlack;
    const float mn = raise ? mx : m;
    const float mo = mn == -INFINITY ? 0.0f : mn;
    float sum = 0.0f;
    uint32_t pw[8][P];
#pragma unroll
    for (int t = 0; t < 4; t++)
#pragma unroll
        for (int e = 0; e < 4; e += 2) {
            const float a = __builtin_amdgcn_exp2f(fmaf(s[t][e], sl, -mo));
            const float c = __builtin_amdgcn_exp2f(fmaf(s[t][e + 1], sl, -mo));
            sum += a + c;
            split_pair<P>(a, c, pw[2 * t + e / 2]);
        }
#pragma unroll
    for (int x = 0; x < 2; x++)
#pragma unroll
        for (uint32_t e = 0; e < P; e++)
            w[x][e] = as_bf16x8(u32x4{pw[4 * x][e], pw[4 * x + 1][e], pw[4 * x + 2][e], pw[4 * x + 3][e]});
    if (__builtin_amdgcn_ballot_w64(raise) != 0) {
        const float alpha = raise ? __builtin_amdgcn_exp2f(m - mn) : 1.0f;
        l *= alpha;
        m = mn;
#pragma unroll
        for (int dt = 0; dt < NO; dt++) o[dt] *= alpha;
    }
    l += sum;
}

// The q operands of one column (dead ones zero): operand j holds d 64 (j / 2) + 16 grp + 8 (j % 2) ..,
// kParts parts of f32 q; the scale's sign goes into q, exactly.
template <bool QF32, uint32_t P>
TS_DEV void load_q(const AttendParams &p, bool live, size_t at, uint32_t grp, bf16x8 (&q)[4][P]) {
    const uint32_t qsign = p.scale < 0.0f ? 0x80008000u : 0u;
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const uint32_t d = 64 * (j >> 1) + 16 * grp + 8 * (j & 1);
        if (!QF32) {
            u32x4 w = *(const u32x4 *)((const uint16_t *)p.q + at + d);
            w = live ? w ^ qsign : u32x4{0, 0, 0, 0};
            q[j][0] = as_bf16x8(w);
        } else {
            const f32x4 x = *(const f32x4 *)((const float *)p.q + at + d);
            const f32x4 y = *(const f32x4 *)((const float *)p.q + at + d + 4);
            uint32_t w[4][P];
#pragma unroll
            for (int e = 0; e < 4; e++) {
                float a = e < 2 ? x[2 * e] : y[2 * e - 4], b = e < 2 ? x[2 * e + 1] : y[2 * e - 3];
                if (qsign) { a = -a; b = -b; }
                split_pair<P>(live ? a : 0.0f, live ? b : 0.0f, w[e]);
            }
#pragma unroll
            for (uint32_t e = 0; e < P; e++) q[j][e] = as_bf16x8(u32x4{w[0][e], w[1][e], w[2][e], w[3][e]});
        }
    }
}
// The scale to base 2, positive: a zero one becomes 2^-100, which keeps masked scores -inf and every
// weight 1 within f32 rounding.
TS_DEV float base2_scale(float scale) { return scale == 0.0f ? 0x1p-100f : fabsf(scale) * 1.4426950408889634f; }

}  // namespace kept8

namespace ts {
// The kernel whose waves share their keys (kept8_rows.hip), for tiles of 64, 128 or (bf16 q) 256 columns.
int kept8_rows_launch(const kept8::AttendParams &p, uint32_t columns, bool qf32, uint32_t groups, void *stream);
}  // namespace ts
