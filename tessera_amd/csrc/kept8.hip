// Attention over kept blocks (kept8.h): decode rows, several drafted rows of a sequence, prompts.
//
// Row r (slot s, position p) sees the keys at [max(0, p - back), p] of its slot: w = softmax(q . k *
// scale), out = sum of w v (engine/ir/interp/src/cpu.rs:293-351 over bf16 rows; no counterpart in the
// reference for blocks).
//
// A tile is the q heads of one kv head for R rows that stand together, its (row, head) pairs the columns
// of 16-wide matrix products: S^T = K q^T and O^T = V^T P^T, so the scores of a column stay in its
// lanes and P^T is the second product's operand as it stands. Each wave takes steps of 64 keys, four
// blocks:
//  * K: tile t of the four 16-key tiles takes positions 4t .. 4t + 3 of each block, so that a lane's
//    16 scores are the 16 positions of one block (block lane / 16), the order V's operand has them in.
//    A lane reads 16 bytes of a key (d 64 s + 16 (lane / 16) ..), two operands' worth.
//  * V: 16 bytes are the 16 positions of one d of block lane / 16, again two operands.
//  Nothing passes through LDS: codes go from memory to registers, through the conversion that applies
//  the block's scale, into the matrix unit; the next step's are asked for as soon as this step's are used.
//  The four waves of a group, and the groups that share a tile's keys (share_of), are joined by their maxima
//  and sums, the former in LDS, the latter by a second kernel.
// HBM bounds it: 32 rows of 512 .. 8192 keys, 8 kv heads, 286 MB: 56 us and 5 for the join, 5.1 TB/s of codes;
// 2 rows of 131000 keys, 4 kv heads: 43 and 5 us, 6 TB/s. A step costs a wave about 2.2 us with two waves a SIMD; a
// group's first is done after some 8 us, which is what one row of 4000 keys takes (9.5 and 4 us).
#include <algorithm>

#include "kept8_attend.h"

namespace {

using namespace kept8;

constexpr uint32_t kWaves = 4;
constexpr uint32_t kRound = kStep * kWaves;  // keys of a group's waves at a time, and its unit of shared keys

template <bool QF32>
__global__ __launch_bounds__(256, 2) void attend_kept8_kernel(AttendParams p) {
    // The weights of bf16 q in two parts (16 bits): in one the outputs' error against 64 bits is 2.3e-3 of them, in two
    // 1.6e-3, what rounding them to bf16 makes; the keys' bytes hide most of it (2 rows of 131000 keys 58.1 -> 58.4 us,
    // 32 of 8192 65.2 -> 65.9, 8 of 4096 17.9 -> 18.5).
    constexpr uint32_t kCols = 16, kParts = QF32 ? 3 : 1, kWeights = QF32 ? 3 : 2;
    extern __shared__ __attribute__((aligned(16))) float joined[];  // [kWaves][kCols][kPart]
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const uint32_t col = lane & 15, grp = lane >> 4;
    __shared__ uint32_t starts[kMaxShared + 1];
    const uint32_t u = blockIdx.x / p.kv_heads, kvh = blockIdx.x % p.kv_heads;
    Share share;
    if (!share_of<kRound>(p, u, lane, starts, share)) return;
    for (;;) {
        const Part part = part_of(p, u, lane, kvh, kCols, starts, share);
        const Tile tile = {part.row0, kvh};

        // The lane's column, a (row, head) pair of the tile.
        uint32_t r, h;
        const bool there = tile.column(p, col, r, h);
        const uint32_t pos = there ? p.positions[r] : 0, slot = there ? p.slots[r] : 0;
        const bool live = there && pos <= p.max_position && holds(p.place, slot, pos);
        if (there && !live && p.status && part.a == 0 && wave == 0 && grp == 0)
            atomicOr(p.status, slot >= p.place.slot_count ? TS_STATUS_PAGE : TS_STATUS_POSITION);
        const uint32_t from = pos > p.back ? pos - p.back : 0;
        const size_t q_at = live ? ((size_t)r * p.heads + h) * 128 : 0;

        // A pass over the keys for each slot among the columns (one, where rows of a slot stand together): its
        // active columns see keys in [lo, hi], all of them those in [all_lo, all_hi].
        struct Pass {
            uint32_t now, lo, hi, all_lo, all_hi;
            bool act;
        } s;
        bool wait = live;
        auto next_pass = [&] {
            const uint64_t b = __builtin_amdgcn_ballot_w64(wait);
            if (!b) return false;
            s.now = __builtin_amdgcn_readlane(slot, __builtin_ctzll(b));
            s.act = wait && slot == s.now;
            wait = wait && !s.act;
            s.lo = row16_least(s.act ? from : 0xffffffffu);
            s.hi = ~row16_least(s.act ? ~pos : 0xffffffffu);
            s.all_lo = ~row16_least(s.act ? ~from : live ? 0u : 0xffffffffu);  // (a column not active sees none)
            s.all_hi = row16_least(s.act ? pos : 0xffffffffu);
            return true;
        };
        // Of a pass, the wave's next step is the keys from base0 + off on, its last one's off at most `last`.
        uint32_t base0, off, last;
        auto next_keys = [&] {
            if (!next_pass()) return false;
            base0 = s.lo & ~(kBlock - 1);
            const uint32_t span = s.hi - base0, np = span / kRound + 1;
            const uint32_t a = pass_unit(part.a, part.n, np), b = pass_unit(part.b, part.n, np);
            off = a * kRound + wave * kStep;
            last = a < b ? min(b * kRound - 1, span) : 0;
            if (a >= b) off = 1;
            return true;
        };
        bool more_passes = next_keys();

        // The blocks of a step; bit j of `lost`: block j's page is not held.
        struct Blocks {
            uint32_t at[4], lost;
        } b;
        auto look = [&](uint32_t base) {
            b.lost = 0;
#pragma unroll
            for (uint32_t j = 0; j < 4; j++) {
                bool gone;
                b.at[j] = block_of(p.place, s.now, min(base / kBlock + j, s.hi / kBlock) * kBlock, gone);
                b.lost |= gone ? 1u << j : 0u;
            }
        };
        // Lane value j of four uniform ones.
        auto choose = [](uint32_t j, auto a, auto b, auto c, auto d) {
            const auto x = j & 1 ? b : a, y = j & 1 ? d : c;
            return j & 2 ? y : x;
        };
        u32x4 kf[4][2], vf[8];
        float ks = 0.0f, vs = 0.0f;
        const_f32 *scales = in_constant<const_f32 *>(p.scales + tile.kvh * 2);
        const size_t scale_row = scale_heads(p.kv_heads) * 2;
        auto load_k = [&] {
            const uint32_t block = choose(col >> 2, b.at[0], b.at[1], b.at[2], b.at[3]);
            const uint8_t *at = p.k + ((size_t)block * p.kv_heads + tile.kvh) * kBlockBytes + (col & 3) * kWidth + 16 * grp;
#pragma unroll
            for (int t = 0; t < 4; t++)
#pragma unroll
                for (int x = 0; x < 2; x++) kf[t][x] = *(const u32x4 *)(at + 4 * t * kWidth + 64 * x);
            ks = choose(col >> 2, scales[b.at[0] * scale_row], scales[b.at[1] * scale_row], scales[b.at[2] * scale_row],
                        scales[b.at[3] * scale_row]);
        };
        auto load_v = [&] {
            const uint32_t block = choose(grp, b.at[0], b.at[1], b.at[2], b.at[3]);
            const uint8_t *at = p.v + ((size_t)block * p.kv_heads + tile.kvh) * kBlockBytes + col * kBlock;
#pragma unroll
            for (int dt = 0; dt < 8; dt++) vf[dt] = *(const u32x4 *)(at + dt * 16 * kBlock);
            vs = choose(grp, scales[b.at[0] * scale_row + 1], scales[b.at[1] * scale_row + 1],
                        scales[b.at[2] * scale_row + 1], scales[b.at[3] * scale_row + 1]);
        };

        // The first step's K is asked for before q, its V after.
        const bool early = more_passes && off <= last;
        if (early) {
            look(base0 + off);
            load_k();
        }
        const float sl = base2_scale(p.scale);
        bf16x8 q[4][kParts];
        load_q<QF32, kParts>(p, live, q_at, grp, q);
        if (early) load_v();
        float m = -INFINITY, l = 0.0f;
        f32x4 o[8];  // O^T: lane's column, d 16 dt + 4 grp + i
#pragma unroll
        for (int dt = 0; dt < 8; dt++) o[dt] = f32x4{0, 0, 0, 0};

        for (bool first = true; more_passes; first = false, more_passes = next_keys()) {
            if (!first && off <= last) {
                look(base0 + off);
                load_k();
                load_v();
            }
            for (bool more = off <= last; more;) {
                const uint32_t base = base0 + off, lost = b.lost;
                off += kRound;
                more = off <= last;
                // (The last step's codes are asked for once more, from the caches: a branch around the
                // loads would keep two copies of them in registers.)
                look(more ? base0 + off : base);
                f32x4 sc[4];
#pragma unroll
                for (int t = 0; t < 4; t++) {
                    pin(kf[t][0]);
                    pin(kf[t][1]);
                    sc[t] = f32x4{0, 0, 0, 0};
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        const u32x4 w = kf[t][j >> 1];
                        const bf16x8 kc = codes8(j & 1 ? w.z : w.x, j & 1 ? w.w : w.y, ks);
#pragma unroll
                        for (uint32_t e = 0; e < kParts; e++) sc[t] = mfma16(kc, q[j][e], sc[t]);
                    }
                }
                load_k();

                // A step that meets a window's edge, or a block that is lost.
                if (base < s.all_lo || base + (kStep - 1) > s.all_hi || lost) {
                    const uint32_t key0 = base + kBlock * grp;
                    const bool gone = lost >> grp & 1;
                    if (lost && p.status && lane == 0) atomicOr(p.status, TS_STATUS_PAGE);
                    const uint32_t seen = s.act ? seen_keys(key0, from, pos) : 0u;
#pragma unroll
                    for (int t = 0; t < 4; t++)
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            const float x = gone ? __builtin_nanf("") : sc[t][e];
                            sc[t][e] = seen >> (4 * t + e) & 1 ? x : -INFINITY;
                        }
                    // Codes outside [lo, hi] may be anything: as zeros they add nothing.
                    uint32_t nan = 0;
#pragma unroll
                    for (int dt = 0; dt < 8; dt++) {
                        vf[dt] = u32x4{within4(vf[dt].x, key0, s.lo, s.hi), within4(vf[dt].y, key0 + 4, s.lo, s.hi),
                                       within4(vf[dt].z, key0 + 8, s.lo, s.hi), within4(vf[dt].w, key0 + 12, s.lo, s.hi)};
                        nan |= nan_codes(vf[dt].x) | nan_codes(vf[dt].y) | nan_codes(vf[dt].z) | nan_codes(vf[dt].w);
                    }
                    // A NaN code at a key that some columns see and some do not: a weight of 0 times NaN
                    // must not reach the latter. Such codes become 0, and what they reach is marked by a
                    // product of (code is NaN) with (column sees the key).
                    if (__builtin_amdgcn_ballot_w64(nan != 0) != 0) {
#pragma unroll
                        for (int dt = 0; dt < 8; dt++) {
                            uint32_t ones[4];  // e4m3 1.0 (0x38) at each NaN code
#pragma unroll
                            for (int e = 0; e < 4; e++) {
                                const uint32_t at = nan_codes(vf[dt][e]) >> 7;
                                ones[e] = at * 0x38u;
                                vf[dt][e] &= ~(at * 0xffu);
                            }
                            f32x4 hit = f32x4{0, 0, 0, 0};
#pragma unroll
                            for (int x = 0; x < 2; x++) {
                                uint32_t sw[4];
#pragma unroll
                                for (int e = 0; e < 4; e++) {
                                    const uint32_t two = seen >> (8 * x + 2 * e);
                                    sw[e] = (two & 1 ? 0x3f80u : 0u) | (two & 2 ? 0x3f800000u : 0u);
                                }
                                hit = mfma16(codes8(ones[2 * x], ones[2 * x + 1], 1.0f),
                                             as_bf16x8(u32x4{sw[0], sw[1], sw[2], sw[3]}), hit);
                            }
#pragma unroll
                            for (int e = 0; e < 4; e++)
                                if (hit[e] > 0.0f) o[dt][e] = __builtin_nanf("");
                        }
                    }
                }
                bf16x8 w[2][kWeights];
                weigh<kWeights, 8>(sc, sl, m, l, o, w);
#pragma unroll
                for (int dt = 0; dt < 8; dt++) {
                    pin(vf[dt]);
#pragma unroll
                    for (int x = 0; x < 2; x++) {
                        const bf16x8 vc = codes8(x ? vf[dt].z : vf[dt].x, x ? vf[dt].w : vf[dt].y, vs);
#pragma unroll
                        for (uint32_t e = 0; e < kWeights; e++) o[dt] = mfma16(vc, w[x][e], o[dt]);
                    }
                }
                load_v();
            }
        }

        // The waves' results joined, a thread four d of a column at a time.
        {
            float *at = joined + (wave * kCols + col) * kPart;
            const float sum = rows4_sum(l);
            if (grp == 0) {
                at[0] = m;
                at[1] = live ? sum : __builtin_nanf("");  // a refused column passed unmasked with the others
            }
#pragma unroll
            for (int dt = 0; dt < 8; dt++) *(f32x4 *)(at + 4 + 16 * dt + 4 * grp) = o[dt];
        }
        __syncthreads();
        for (uint32_t e = threadIdx.x; e < kCols * 32; e += 256) {
            const uint32_t c = e / 32, d = e % 32 * 4;
            if (!tile.column(p, c, r, h)) continue;
            float M = -INFINITY;
#pragma unroll
            for (uint32_t w = 0; w < kWaves; w++) M = fmaxf(M, joined[(w * kCols + c) * kPart]);
            float L = 0.0f;
            f32x4 O = f32x4{0, 0, 0, 0};
#pragma unroll
            for (uint32_t w = 0; w < kWaves; w++) {
                const float *at = joined + (w * kCols + c) * kPart;
                const float f = at[0] == -INFINITY ? (at[1] == 0.0f ? 0.0f : 1.0f) : __builtin_amdgcn_exp2f(at[0] - M);
                L += at[1] * f;
                O += *(const f32x4 *)(at + 4 + d) * f;
            }
            if (part.partial) {
                float *at = part.partial + c * kPart;
                if (d == 0) {
                    at[0] = M;
                    at[1] = L;
                }
                *(f32x4 *)(at + 4 + d) = O;
            } else {
                store4(p, ((size_t)r * p.heads + h) * 128 + d, O / L);  // 0 / 0 of a refused row: NaN
            }
        }
        share.unit += part.b - part.a;
        share.tile++;
        if (share.unit >= share.end) return;
        __syncthreads();  // (the results joined are read, the next tile's may be written)
    }
}

// The parts of a tile's columns joined: S lane groups of 32 (four d a lane) take a column's parts in turn, four
// at a time, 8 / S columns a group of 256. (One lane group walking 128 parts by itself waits 20 us; up to four
// parts are one step of one.)
template <uint32_t S>
__global__ __launch_bounds__(256) void join_kept8_kernel(AttendParams p, uint32_t cols, uint32_t pieces) {
    __shared__ float smax[8], ssum[8];
    __shared__ f32x4 so[8][32];
    constexpr uint32_t kBatch = 4;
    const uint32_t gi = blockIdx.x / pieces, lg = threadIdx.x / 32, d = threadIdx.x % 32;
    const Tile tile = {gi / p.kv_heads * p.tile_rows, gi % p.kv_heads};
    const uint32_t parts = p.shares[gi / p.kv_heads * 2 + 1];
    if (parts == 1) return;  // (its group has written the rows)
    const uint32_t c = blockIdx.x % pieces * (8 / S) + lg / S, j1 = lg % S;
    uint32_t r, h;
    const bool there = c < cols && tile.column(p, c, r, h);
    // Part 0 is of a group that a later one goes on from, the others of groups that an earlier one began for.
    const size_t next = (size_t)p.kv_heads * cols * kPart;  // from a group's results to the next's
    const float *rest = p.partials + p.shares[gi / p.kv_heads * 2] * next +
                        ((size_t)tile.kvh * cols + (there ? c : 0)) * kPart;
    float M = -INFINITY, L = 0.0f;
    f32x4 O = f32x4{0, 0, 0, 0};
    // A maximum of -inf: an empty part, or a refused column's (whose sum is NaN): as it is.
    auto factor = [](float m, float to) { return m == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m - to); };
    for (uint32_t j0 = j1; j0 < parts; j0 += S * kBatch) {
        float mq[kBatch], lq[kBatch], top = M;
        f32x4 oq[kBatch];
#pragma unroll
        for (uint32_t j = 0; j < kBatch; j++) {  // past the end: read, not used
            const uint32_t part = min(j0 + S * j, parts - 1);
            const float *at = rest + (part ? part : p.groups) * next;
            mq[j] = at[0];
            lq[j] = at[1];
            oq[j] = *(const f32x4 *)(at + 4 + 4 * d);
        }
#pragma unroll
        for (uint32_t j = 0; j < kBatch; j++)
            if (j0 + S * j < parts) top = fmaxf(top, mq[j]);
        const float f = factor(M, top);
        M = top;
        L *= f;
        O *= f;
#pragma unroll
        for (uint32_t j = 0; j < kBatch; j++) {
            if (j0 + S * j >= parts) continue;
            const float g = factor(mq[j], M);
            L += lq[j] * g;
            O += oq[j] * g;
        }
    }
    if (S > 1) {
        so[lg][d] = O;
        if (d == 0) {
            smax[lg] = M;
            ssum[lg] = L;
        }
        __syncthreads();
        if (j1) return;
#pragma unroll
        for (uint32_t s = 1; s < S; s++) M = fmaxf(M, smax[lg + s]);
        const float f = factor(smax[lg], M);
        L *= f;
        O *= f;
#pragma unroll
        for (uint32_t s = 1; s < S; s++) {
            const float g = factor(smax[lg + s], M);
            L += ssum[lg + s] * g;
            O += so[lg + s][d] * g;
        }
    }
    if (there) store4(p, ((size_t)r * p.heads + h) * 128 + 4 * d, O / L);
}

// How a call runs: `columns` (row, q head) pairs a tile; 16: the kernel above, more: kept8_rows.hip's.
struct Plan {
    uint32_t columns, tile_rows, tiles, groups, most;  // row tiles; groups a kv head; parts a tile at most
};

Plan plan(const ts_kept8_args *k) {
    const ts_rows_args *a = &k->rows;
    const uint32_t G = a->heads / a->kv_heads;
    const bool f32 = a->q_dtype == TS_F32;
    Plan s;
    const uint32_t run = std::max(1u, std::min(k->run, a->rows));
    const uint64_t wanted = (uint64_t)run * G;
    // f32 q, in three parts, leaves a wave of the shared kernel 16 columns. 256 columns widen the codes for fewer
    // waves twice, but fill a CU with one group: only where there are one and a half groups a CU to even them out
    // (prompts of 2048 rows, 16 heads over 8: 4 of them 105 us, 128 columns 119; 3, the border, 81 and 92; 2 81 and
    // 75. Between one and one and a half groups either may win: 3 of 1600 86 and 64, 9 of 512 36 and 41.)
    const uint64_t wide = (a->rows + 256 / G - 1) / (256 / G) * (uint64_t)a->kv_heads;
    s.columns = wanted <= 16 ? 16 : wanted <= 64 ? 64 : wanted <= 128 || f32 || wide < 384 ? 128 : 256;
    s.tile_rows = std::min(run, s.columns / G);
    s.tiles = (a->rows + s.tile_rows - 1) / s.tile_rows;
    s.groups = s.tiles;
    s.most = 1;
    // Keys are shared out over as many groups as run at once (a CU's two of four waves, with 64 columns of bf16 q
    // three, or one of eight): more would each cost 8 us before the first step is done, fewer leave CUs idle.
    // Up to 64 columns always: 32 sequences of 512 .. 8192, 8 kv heads, 68 us, a group a tile 116; 24 x 5 drafted rows
    // 73 and 197; 128 sequences of up to 4096, beyond the groups at once, 127 and 138 (but 250 of up to 2000 143 and
    // 135, 100 x 5 drafted rows 141 and 125). Wide tiles, whose partial results are large, only where there are fewer
    // tiles than groups: 2 chunks of 700 f32 rows behind 4300 145 us, a group a tile 313; 1 of 1024 bf16 rows behind
    // 7168 130 and 229. From as many on, a group a tile, the widest first: 1 of 2048 bf16 rows 68, shared 89; 2 of
    // them behind 2048 142 and 213 (but 4 chunks of 700 f32 rows behind 4300, 44 tiles for 32 groups, 484 and 277).
    const uint32_t at_once = (s.columns == 64 && !f32 ? 768 : s.columns <= 64 ? 512 : 256) / a->kv_heads;
    const uint32_t unit = s.columns == 16 ? kRound : kStep;
    const uint64_t span = std::min<uint64_t>(std::min<uint64_t>((uint64_t)a->max_position + 1, a->keys),
                                             (uint64_t)a->back + s.tile_rows + kBlock);
    const uint64_t units = (span + unit - 1) / unit + 1;
    if (at_once > 1 && s.tiles <= (s.columns <= 64 ? kMaxShared : std::min(kMaxShared, at_once - 1)) && span > unit) {
        s.groups = (uint32_t)std::min<uint64_t>(at_once, s.tiles * units);
        s.most = (uint32_t)std::min<uint64_t>(units, s.groups);
    }
    return s;
}

size_t partial_bytes(const ts_kept8_args *k, const Plan &s) {
    return s.most <= 1 ? 0 : (size_t)s.groups * 2 * k->rows.kv_heads * s.columns * kPart * sizeof(float);
}
size_t share_bytes(const Plan &s) { return s.most <= 1 ? 0 : (size_t)s.tiles * 2 * sizeof(uint32_t); }

int check(const ts_kept8_args *k) {
    TS_REQUIRE(k, "attend_kept8: null args");
    const ts_rows_args *a = &k->rows;
    TS_REQUIRE(a->k && a->v && k->scales && (a->rows == 0 || (a->q && a->out && a->slots && a->positions)),
               "attend_kept8: null pointer");
    TS_REQUIRE(a->width == 128, "attend_kept8: head width %u (128 supported)", a->width);
    TS_REQUIRE(a->kv_heads >= 1 && a->kv_heads <= 1024 && a->heads >= 1 && a->heads % a->kv_heads == 0 &&
                   a->heads / a->kv_heads <= 64,
               "attend_kept8: %u heads over %u kv heads (at most 64 each)", a->heads, a->kv_heads);
    TS_REQUIRE((a->q_dtype == TS_F32 || a->q_dtype == TS_BF16) && a->kv_dtype == TS_E4M3 &&
                   (a->out_dtype == TS_F32 || a->out_dtype == TS_BF16),
               "attend_kept8: q and out f32 or bf16, kept rows e4m3 blocks supported");
    int rc = ts::kept_check("attend_kept8", a->kept_table, a->page, a->keys, k->slot_count, a->kept_pages, k->pages, true);
    if (rc) return rc;
    TS_REQUIRE(a->keys <= 1u << 30, "attend_kept8: %u positions a slot", a->keys);
    TS_REQUIRE((uint64_t)k->pages * a->page <= 1ull << 36, "attend_kept8: %u pages of %u rows", k->pages, a->page);
    TS_REQUIRE(ts::aligned(a->k, 16) && ts::aligned(a->v, 16) && ts::aligned(a->q, 16) && ts::aligned(a->out, 16) &&
                   ts::aligned(k->scales, 16),
               "attend_kept8: q, k, v, scales and out must be 16-byte aligned");
    return TS_OK;
}

template <bool QF32>
int launch(const AttendParams &p, uint32_t groups, void *stream) {
    constexpr uint32_t kLds = kWaves * 16 * kPart * sizeof(float);
    hipLaunchKernelGGL(attend_kept8_kernel<QF32>, dim3(groups), dim3(256), kLds, (hipStream_t)stream, p);
    TS_CHECK_LAUNCH("attend_kept8 launch");
    return TS_OK;
}

}  // namespace

extern "C" size_t tessera_hip_attend_kept8_workspace(const ts_kept8_args *k) {
    if (!k || k->rows.kv_heads == 0 || k->rows.heads == 0 || k->rows.heads % k->rows.kv_heads ||
        k->rows.heads / k->rows.kv_heads > 64 || k->rows.rows == 0)
        return 0;
    const Plan s = plan(k);
    return partial_bytes(k, s) + share_bytes(s);
}

extern "C" int tessera_hip_attend_kept8(const ts_kept8_args *k, void *stream) {
    int rc = check(k);
    if (rc) return rc;
    const ts_rows_args *a = &k->rows;
    if (a->rows == 0) return TS_OK;
    const Plan s = plan(k);
    TS_REQUIRE((uint64_t)s.groups * a->kv_heads <= 0x7fffffffull / 128, "attend_kept8: %u rows in one launch", a->rows);
    const size_t partials = partial_bytes(k, s), need = partials + share_bytes(s);
    if (need && (!a->workspace || a->workspace_bytes < need || !ts::aligned(a->workspace, 16)))
        return ts::fail(TS_ERR_WORKSPACE, "attend_kept8: workspace of %zu bytes, 16-byte aligned, needed", need);
    AttendParams p;
    p.q = a->q; p.k = (const uint8_t *)a->k; p.v = (const uint8_t *)a->v; p.scales = k->scales; p.out = a->out;
    p.partials = need ? (float *)a->workspace : nullptr;
    p.shares = need ? (uint32_t *)((char *)a->workspace + partials) : nullptr;
    p.slots = a->slots; p.positions = a->positions; p.status = a->status;
    p.place.table = a->kept_table; p.place.keys = a->keys; p.place.slot_count = k->slot_count;
    p.place.kept_pages = a->kept_pages; p.place.page_shift = (uint32_t)__builtin_ctz(a->page); p.place.pages = k->pages;
    p.rows = a->rows; p.heads = a->heads; p.kv_heads = a->kv_heads; p.group = a->heads / a->kv_heads;
    p.back = a->back; p.max_position = a->max_position;
    p.tile_rows = s.tile_rows; p.tiles = s.tiles; p.groups = s.groups;
    p.scale = a->scale; p.out_bf16 = a->out_dtype == TS_BF16;
    const uint32_t groups = s.groups * a->kv_heads;
    const bool f32 = a->q_dtype == TS_F32;
    if (s.columns > 16)
        rc = ts::kept8_rows_launch(p, s.columns, f32, groups, stream);
    else
        rc = f32 ? launch<true>(p, groups, stream) : launch<false>(p, groups, stream);
    if (rc || s.most == 1) return rc;
    const uint32_t used = s.tile_rows * p.group, parts = std::min(s.most, s.groups / s.tiles + 2);
    const uint32_t S = parts <= 4 ? 1 : parts <= 8 ? 2 : 8;
    const uint32_t pieces = (used * S + 7) / 8;
    const auto join = S == 1 ? join_kept8_kernel<1> : S == 2 ? join_kept8_kernel<2> : join_kept8_kernel<8>;
    hipLaunchKernelGGL(join, dim3(s.tiles * a->kv_heads * pieces), dim3(256), 0, (hipStream_t)stream, p, s.columns,
                       pieces);
    TS_CHECK_LAUNCH("attend_kept8 join launch");
    return TS_OK;
}
