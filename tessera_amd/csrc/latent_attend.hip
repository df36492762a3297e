// The absorbed form of latent attention: every head of row r (slot s, position p) sees the kept rows of its slot at
// [max(0, p - back), p], w = softmax(q . row * scale), out = sum of w row[: RANK].
//
// A tile is the heads of R rows that stand together, its (row, head) pairs the columns of 16-wide matrix products
// S^T = K q^T and O^T = V^T P^T, so a column's scores stay in its lanes and P^T is the second product's operand as
// it stands. Keys and values are one row, which goes from memory to LDS once, 32 keys a step, without passing
// registers; K's operand is 16 bytes of a row, V^T's comes through the transposing LDS read. A wave holds 16
// columns: 128 (RANK 512) registers of O and 72 of q.
//  * WC waves share a step's keys, 16 columns each; the teams of a group take steps in turn, and are joined in LDS at
//    the end. With WC = 1 each wave streams keys of its own and waits for no other.
//  * Keys are dealt to the groups, the tiles' one behind the other, so that groups end together however the sequences
//    differ in length; a tile that several groups have is joined by a second kernel. Few tiles: each in equal parts of
//    its own, a group one of them, which spares groups a second start (24 sequences of 3 to 5 rows, 32 heads, 1000 ..
//    9001 keys: 73 us against 81; 32 sequences of 16 heads, 512 .. 8192 keys: 48 against 54).
//  * A weight enters the product in two bf16 parts with 16 columns, which leave the matrix unit time for it, in one else. Two
//    there would bring the error against 64 bits (2-norm) from 2.0e-3 to 1.66e-3, the output's own rounding, and take 48 us for
//    46 with 32 columns (32 sequences of 32 heads, 4000 keys), 77 for 70 with 64 (32 sequences of 128 heads, 512 .. 8192 keys;
//    24 x 5 drafts of 32 heads 70 for 65), 191 for 149 with 128 (two chunks of 512 rows, 16 heads, 2500 and 4600 keys).
//
// 32 sequences of 16 heads, 32000 keys each: 5.3 TB/s, what a copy reaches. 8 prompts' chunks of 512 rows behind 8000 keys,
// 16 heads: 1000 to 1050 TFLOP/s. A round of 32 keys and 128 columns takes some 4700 cycles: its loads 600 (the vector cache
// takes 64 bytes a cycle), scores 1300, softmax 350, values 1300, the barrier 500 and more; the matrix unit is busy for 46% of
// the cycles, LDS for 48% (a wave's 16 columns read a step's whole rows, 68 KB; 32 columns a wave do not fit the registers), at
// a clock of 1.9 GHz. Short calls are bound by a group's start (positions, pages, q and the first keys come one after the
// other, 7 us) and by the join (5 us, 22 for the chunks' 128 columns).
#include <algorithm>

#include "kept8_attend.h"
#include "latent.h"
#include "places.h"

namespace {

using namespace kept8;
using namespace latent;

constexpr uint32_t kKeys = 32;         // keys of a step
constexpr uint32_t kMaxTiles = 1024;   // row tiles whose keys are shared
constexpr uint32_t kWholeTiles = 128;  // and those of which each group has one
constexpr uint32_t kCutRows = 512;     // rows whose tiles are cut where slots change
constexpr uint32_t kJoinThreads = 256;

struct LatentParams {
    const uint16_t *q, *kept;
    uint16_t *out;
    // Where keys are shared: results of groups for a tile that an earlier group began, then for one that a later
    // group goes on with, each [groups][blocks] of a tile's columns; and each row tile's groups and rows (first and count of
    // both), then how many tiles there are.
    float *partials;
    uint32_t *shares;
    const uint32_t *slots, *positions;
    uint32_t *status;
    Place place;
    uint32_t rows, heads, back, max_position;
    uint32_t tile_rows, tiles, groups;  // rows a tile, row tiles (cut ones: their most), and groups a block of heads
    int whole;                          // where keys are shared: a group has keys of one tile only
    int cut;                            // and: a tile's rows are one slot's
    uint32_t block_heads, blocks;       // a row's heads in a tile, and the blocks they make
    float scale;
};

// Column c's row and head of a tile of n rows; false where it has none.
TS_DEV bool column_of(const LatentParams &p, uint32_t row0, uint32_t n, uint32_t block, uint32_t c, uint32_t &r, uint32_t &h) {
    const uint32_t ri = c / p.block_heads;
    r = row0 + ri;
    h = block * p.block_heads + c % p.block_heads;
    return ri < n && h < p.heads;
}

// A column's partial result: RANK / 4 times [columns] of four sums, then [columns] maxima and sums.
template <uint32_t RANK>
constexpr uint32_t part_floats(uint32_t columns) { return columns * (RANK + 2); }

// The XOR of a row's 16-byte pieces in LDS: among eight where rows begin 128 bytes apart (modulo the 256 that LDS
// serves at a time), among four where 64. It keeps the lanes that are served together in 16 places: of K's read
// lanes 0-3 and 12-15 of one 16 and 4-11 of the next, of V^T's the two pieces of eight rows.
template <uint32_t CH>
TS_DEV uint32_t swap_of(uint32_t row) {
    const uint32_t i = CH % 16 == 8 ? row >> 1 & 7 : row >> 2 & 3;
    if (CH % 16 == 8) return (i & 1) << 2 | ((i ^ i >> 1) & 2) | i >> 2;
    return ((i ^ i >> 1) & 1) << 1 | i >> 1;
}

// The least over a wave, uniform; the total; and the lanes' sums up to each.
TS_DEV uint32_t wave_least(uint32_t v) {
    const auto a = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    const uint32_t x = min((uint32_t)a[0], (uint32_t)a[1]);
    const auto b = __builtin_amdgcn_permlane16_swap(x, x, false, false);
    return row16_least(min((uint32_t)b[0], (uint32_t)b[1]));
}
TS_DEV uint32_t wave_upto(uint32_t v, uint32_t lane) {
    v += dpp_u<0x111>(v);
    v += dpp_u<0x112>(v);
    v += dpp_u<0x114>(v);
    v += dpp_u<0x118>(v);
    const uint32_t a = __builtin_amdgcn_readlane(v, 15), b = a + __builtin_amdgcn_readlane(v, 31),
                   c = b + __builtin_amdgcn_readlane(v, 47);
    return v + (lane < 16 ? 0 : lane < 32 ? a : lane < 48 ? b : c);
}
TS_DEV uint32_t rows4_total(uint32_t v) {  // over the four lanes of a column
    const auto a = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    const uint32_t x = (uint32_t)a[0] + (uint32_t)a[1];
    const auto b = __builtin_amdgcn_permlane16_swap(x, x, false, false);
    return (uint32_t)b[0] + (uint32_t)b[1];
}
TS_DEV uint32_t wave_total(uint32_t v) { return __builtin_amdgcn_readlane(wave_upto(v, threadIdx.x & 63), 63); }

// 2^(a - b) of maxima, 0 where a has seen nothing.
TS_DEV float weight_of(float a, float b) { return a == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(a - b); }

template <uint32_t RANK, uint32_t ROPE, uint32_t WC>
struct Shape {
    static constexpr uint32_t kWidth = RANK + ROPE, kRow = 2 * kWidth, kPieces = kWidth / 8;
    static constexpr uint32_t kWaves = WC < 4 ? 4 : 8, kTeams = kWaves / WC;
    static constexpr uint32_t kRing = 4 / kTeams;                // rounds of kTeams steps in LDS
    static constexpr uint32_t kTile = kKeys * kRow, kLds = 4 * kTile;
    static constexpr uint32_t kUnit = kKeys * kTeams;            // keys of a round
    static constexpr uint32_t kParts = kTile / 1024;             // loads of a step, dealt to the team's waves
    static constexpr uint32_t kLoads = (kParts + WC - 1) / WC, kLeast = kParts / WC;
    static constexpr uint32_t kOwn = kLoads < 9 ? kLoads : 9;    // those of different places within a block
    static constexpr uint32_t kCols = 16 * WC, kWeights = WC == 1 ? 2 : 1;
    static constexpr uint32_t kAhead = WC == 8 ? 3 : 2;          // operands read ahead of their products
    static constexpr uint32_t kQ = kWidth / 32, kD = RANK / 16;  // operands of q, tiles of O
    static constexpr uint32_t kIds = WC == 1 ? 2 : 2 * kTeams;   // blocks whose pages a wave looks up
    static constexpr uint32_t kXor = kPieces % 16 == 8 ? 8 : 4;  // pieces that the XOR permutes
    static constexpr bool kAside = RANK == 512;                  // the loads' places are kept in LDS: registers are few
};

template <uint32_t RANK, uint32_t ROPE, uint32_t WC>
__global__ __launch_bounds__((64 * Shape<RANK, ROPE, WC>::kWaves), 2) void attend_latent_kernel(LatentParams p) {
    using S = Shape<RANK, ROPE, WC>;
    constexpr uint32_t kThreads = 64 * S::kWaves;
    extern __shared__ __attribute__((aligned(16))) char stage[];
    __shared__ uint32_t rows_at[2][128];  // the tile's rows' positions and slots (each wave writes all, the same)
    // (starts: with cut tiles the second half holds their first rows.)
    __shared__ uint32_t starts[kMaxTiles + 2], firsts[2][kWholeTiles], words[8], odd_met[S::kWaves], found;
    __shared__ uint16_t from_aside[S::kAside ? S::kOwn : 1][S::kAside ? kThreads : 1];
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const uint32_t col = lane & 15, grp = lane >> 4, team = wave / WC, mine = wave % WC;
    // Groups go to the eight XCDs in turn. Those of a tile's parts, which read the same q, and of its blocks of heads,
    // which read the same keys, belong to one.
    const uint32_t block = (blockIdx.x >> 3) % p.blocks, u = (blockIdx.x & 7) * ((p.groups + 7) / 8) + (blockIdx.x >> 3) / p.blocks;
    if (u >= p.groups) return;

    // The group's part of the keys: units [a, b) of a row tile's. A tile has as many as its rows see, told from its first
    // and last row. All groups work the division out alike, every wave for itself but for the tiles' units.
    uint32_t tile = u, a = 0, b = 1, units = 1, unit = 0, end = 1, each = 1;
    float *partial = nullptr;
    auto part = [&](bool some) {
        partial = !some ? nullptr : p.partials + ((size_t)((a ? 0 : p.groups) + u) * p.blocks + block) * part_floats<RANK>(S::kCols);
    };
    const bool cut = WC > 1 && p.cut;
    uint32_t tiles = p.tiles;
    uint32_t *const cuts = starts + kCutRows + 1;
    auto row_of = [&](uint32_t tile) { return cut ? (uint32_t)__builtin_amdgcn_readfirstlane(cuts[tile]) : tile * p.tile_rows; };
    auto rows_of = [&](uint32_t tile) {
        return cut ? (uint32_t)__builtin_amdgcn_readfirstlane(cuts[tile + 1] - cuts[tile])
                     : min(p.tile_rows, p.rows - tile * p.tile_rows);
    };
    auto share = [&](uint32_t first, uint32_t count) {
        if (a == 0 && block == 0 && threadIdx.x == 0) {
            p.shares[4 * tile] = first;
            p.shares[4 * tile + 1] = count;
            p.shares[4 * tile + 2] = row_of(tile);
            p.shares[4 * tile + 3] = rows_of(tile);
        }
    };
    if (p.partials) {
        if (cut) {
            // Tiles begin where the slot changes, where tile_rows rows are full, and every 64 rows (a wave's).
            constexpr uint32_t kOwn = kCutRows / 64 / S::kWaves;
            uint64_t begins[kOwn];
#pragma unroll
            for (uint32_t i = 0; i < kOwn; i++) {
                const uint32_t r = (wave + i * S::kWaves) * 64 + lane;
                const uint32_t slot = p.slots[min(r, p.rows - 1)], before = p.slots[min(max(r, 1u) - 1, p.rows - 1)];
                const uint64_t change = __builtin_amdgcn_ballot_w64(lane == 0 || slot != before);
                const uint32_t since = lane - (63 - __builtin_clzll(change & (~0ull >> (63 - lane))));
                begins[i] = __builtin_amdgcn_ballot_w64(r < p.rows && since % p.tile_rows == 0);
                words[wave + i * S::kWaves] = __builtin_popcountll(begins[i]);
            }
            __syncthreads();
            uint32_t n[kCutRows / 64];
            tiles = 0;
#pragma unroll
            for (uint32_t i = 0; i < kCutRows / 64; i++) tiles += n[i] = __builtin_amdgcn_readfirstlane(words[i]);
#pragma unroll
            for (uint32_t i = 0; i < kOwn; i++) {
                uint32_t at = __builtin_amdgcn_mbcnt_hi((uint32_t)(begins[i] >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)begins[i], 0));
#pragma unroll
                for (uint32_t e = 0; e < kCutRows / 64; e++)
                    if (e < wave + i * S::kWaves) at += n[e];
                if (begins[i] >> lane & 1) cuts[at] = (wave + i * S::kWaves) * 64 + lane;
            }
            if (threadIdx.x == 0) {
                cuts[tiles] = p.rows;
                if (u == 0 && block == 0) p.shares[4 * p.tiles] = tiles;
            }
            __syncthreads();
        }
#pragma unroll 1
        for (uint32_t t = threadIdx.x; t < (p.whole ? kWholeTiles : cut ? kCutRows : kMaxTiles); t += kThreads) {
            uint32_t n = 0;
            if (t < tiles) {
                const uint32_t r0 = cut ? cuts[t] : t * p.tile_rows;
                const uint32_t r1 = (cut ? cuts[t + 1] : min(r0 + p.tile_rows, p.rows)) - 1;
                const uint32_t most = min(p.max_position, p.place.keys - 1);
                const uint32_t first = p.positions[r0], slot = p.slots[r0];
                const uint32_t p0 = min(first, most), p1 = min(p.positions[r1], most);
                const uint32_t from0 = p0 > p.back ? p0 - p.back : 0, from1 = p1 > p.back ? p1 - p.back : 0;
                auto units = [](uint32_t lo, uint32_t hi) { return (hi - (lo & ~(kBlock - 1))) / S::kUnit + 1; };
                n = slot == p.slots[r1] ? units(min(from0, from1), max(p0, p1)) : units(from0, p0) + units(from1, p1);
                n = min(n, 1u << 21);
                if (t < kWholeTiles) {
                    firsts[0][t] = first;
                    firsts[1][t] = slot;
                }
            }
            starts[t] = n;
        }
        __syncthreads();
        if (p.whole) {
            // Each tile's keys in as many equal parts as leave none longer than `each`: the shortest `each` (of 16 tried,
            // one a column's lanes) whose parts are no more than the groups.
            uint32_t m[kWholeTiles / 64], all = 0;
#pragma unroll
            for (uint32_t i = 0; i < kWholeTiles / 64; i++) all += m[i] = starts[64 * i + lane];
            all = wave_total(all);
            const float least = (float)all / (float)p.groups, most = (float)all / (float)(p.groups - tiles) + 1.0f;
            const float by = __builtin_amdgcn_rcpf(least + (most - least) * (float)col * (1.0f / 15.0f));
            auto parts_of = [](uint32_t n, float by) { return min(max((uint32_t)ceilf((float)n * by), 1u), n); };
            uint32_t parts = 0;
#pragma unroll 4
            for (uint32_t t = grp; t < tiles; t += 4) parts += parts_of(starts[t], by);
            parts = rows4_total(parts);
            const uint64_t fit = __builtin_amdgcn_ballot_w64(parts <= p.groups);
            const float chosen = fit ? __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(by), __builtin_ctzll(fit))) : 0.0f;
            uint32_t before = 0;
            bool mine_found = false;
#pragma unroll
            for (uint32_t i = 0; i < kWholeTiles / 64; i++) {
                const uint32_t own = 64 * i + lane < tiles ? parts_of(m[i], chosen) : 0, upto = before + wave_upto(own, lane);
                const uint64_t here = __builtin_amdgcn_ballot_w64(u < upto && u >= upto - own);
                before = __builtin_amdgcn_readlane(upto, 63);
                if (!here) continue;
                const uint32_t at = __builtin_ctzll(here), count = __builtin_amdgcn_readlane(own, at);
                const uint32_t first = __builtin_amdgcn_readlane(upto, at) - count;
                mine_found = true;
                tile = 64 * i + at;
                units = __builtin_amdgcn_readlane(m[i], at);
                a = units * (u - first) / count;
                b = units * (u - first + 1) / count;
                part(count > 1);
                share(first, count);
            }
            if (!mine_found) return;
        } else {
            // All tiles' units, one behind the other, in equal runs.
            constexpr uint32_t kEach = kMaxTiles / kThreads;
            uint32_t n[kEach], sum = 0;
#pragma unroll
            for (uint32_t i = 0; i < kEach; i++) sum += n[i] = threadIdx.x * kEach + i < tiles ? starts[threadIdx.x * kEach + i] : 0;
            const uint32_t upto = wave_upto(sum, lane);
            if (lane == 63) words[wave] = upto;
            __syncthreads();
            uint32_t all = 0, before = 0;
#pragma unroll
            for (uint32_t w = 0; w < S::kWaves; w++) {
                if (w < wave) before += words[w];
                all += words[w];
            }
            all = __builtin_amdgcn_readfirstlane(all);
            each = (all + p.groups - 1) / p.groups;
            unit = u * each;
            end = min(unit + each, all);
            if (unit >= all) return;
            uint32_t at = before + upto - sum;
#pragma unroll
            for (uint32_t i = 0; i < kEach; i++) {
                const uint32_t t = threadIdx.x * kEach + i;
                if (t >= tiles) break;
                starts[t] = at;
                if (unit >= at && unit < at + n[i]) found = t;
                at += n[i];
            }
            if (threadIdx.x == 0) starts[tiles] = all;
            __syncthreads();
            tile = __builtin_amdgcn_readfirstlane(found);
        }
    }

    // A tile's rows, two a lane, for what all waves agree on, and the lane's column. (Columns that are not there, or are
    // refused, go along with what is loaded for them.)
    uint32_t row_pos[2], row_slot[2], pos, slot, cut_row, cut_rows;
    bool there;
    const uint16_t *q_at;
    const uint32_t qsign = p.scale < 0.0f ? 0x80008000u : 0u;
    // The tile's first row and rows. (With 16 columns, where registers are fewest, from the tile's number each time.)
    auto tile_row = [&]() { return WC > 1 ? cut_row : tile * p.tile_rows; };
    auto tile_rows = [&]() { return WC > 1 ? cut_rows : min(p.tile_rows, p.rows - tile * p.tile_rows); };
    auto one_row = [&]() { return WC > 1 ? cut_rows == 1 : p.tile_rows == 1; };
    auto fetch = [&]() {
        const uint32_t l0 = again(lane);
        if (WC > 1) {
            cut_row = row_of(tile);
            cut_rows = rows_of(tile);
        }
        const uint32_t row0 = tile_row(), rows = tile_rows();
        uint32_t r = row0, h = block * p.block_heads;
        if (one_row()) {
            pos = p.whole ? firsts[0][tile] : p.positions[row0];
            slot = p.whole ? firsts[1][tile] : p.slots[row0];
            row_pos[0] = row_pos[1] = pos;
            row_slot[0] = row_slot[1] = slot;
            const uint32_t c = 16 * mine + (l0 & 15);
            there = c < p.block_heads && h + c < p.heads;
            if (there) h += c;
        } else {
#pragma unroll
            for (uint32_t i = 0; i < 2; i++) {
                const uint32_t r = row0 + min(l0 + 64 * i, rows - 1);
                row_pos[i] = p.positions[r];
                row_slot[i] = p.slots[r];
            }
            there = column_of(p, row0, rows, block, 16 * mine + (l0 & 15), r, h);
            if (!there) r = row0, h = 0;
            pos = p.positions[r];
            slot = p.slots[r];
        }
        q_at = p.q + ((size_t)r * p.heads + h) * S::kWidth + 8 * (l0 >> 4);
    };
    fetch();

    // Where the lane's 16 bytes of the wave's loads of a step come from, in their block of 16 rows (LDS holds rows back
    // to back). They repeat after nine loads: in the other block, or (WC = 1) eight rows on, where the XOR differs by 3.
    uint32_t from_at[S::kAside ? 1 : S::kOwn];
    {
        constexpr uint32_t kStep = 64 * WC;
        uint32_t row = (64 * mine + lane) / S::kPieces, piece = (64 * mine + lane) % S::kPieces;
#pragma unroll S::kAside ? 3 : S::kOwn
        for (uint32_t i = 0; i < S::kOwn; i++) {
            const uint32_t at = row * S::kRow + (piece ^ swap_of<S::kPieces>(row)) * 16;
            if (S::kAside)
                from_aside[i][threadIdx.x] = (uint16_t)at;
            else
                from_at[S::kAside ? 0 : i] = at;
            piece += kStep % S::kPieces;
            row += kStep / S::kPieces;
            if (piece >= S::kPieces) piece -= S::kPieces, row++;
            row &= kBlock - 1;
        }
    }
    // LDS offsets of the lane's operands: K piece grp of row `col`, and V^T d 8 (lane / 2 % 2) + 4 (lane % 2) .. of keys
    // 4 grp + lane / 4 % 4; others by the XOR of their piece.
    const uint32_t koff = col * S::kRow + (grp ^ swap_of<S::kPieces>(col)) * 16;
    const uint32_t vrow = 4 * grp + (lane >> 2 & 3);
    const uint32_t voff = vrow * S::kRow + ((lane >> 1 & 1) ^ swap_of<S::kPieces>(vrow)) * 16 + (lane & 1) * 8;
    const float sl = base2_scale(p.scale);
    const uint32_t page_blocks = p.place.table ? p.place.page_shift - 4 : 0;  // (the logarithm)
    const uint32_t page_mask = p.place.table ? (1u << page_blocks) - 1 : 0xffffffffu;
    const uint32_t page_count = p.place.table ? p.place.pages : 0xffffffffu;

    for (;;) {
        if (p.partials && !p.whole) {
            const uint32_t t0 = __builtin_amdgcn_readfirstlane(starts[tile]);
            const uint32_t t1 = __builtin_amdgcn_readfirstlane(starts[tile + 1]);
            a = unit - t0;
            b = min(end, t1) - t0;
            units = t1 - t0;
            part(a || b < units);
            share(u, (t1 - 1) / each - u + 1);
        }
        auto lives = [&](uint32_t pos, uint32_t slot) { return pos <= p.max_position && holds(p.place, slot, pos); };
        uint64_t row_waits[2], row_live[2];
        {
            const uint32_t l0 = again(lane);
#pragma unroll
            for (uint32_t i = 0; i < 2; i++) {
                rows_at[0][64 * i + l0] = row_pos[i];
                rows_at[1][64 * i + l0] = row_slot[i];
                const bool here = 64 * i + l0 < tile_rows();
                row_waits[i] = row_live[i] = __builtin_amdgcn_ballot_w64(here && lives(row_pos[i], row_slot[i]));
            }
            if (there && !lives(pos, slot) && p.status && a == 0 && team == 0 && l0 < 16)
                atomicOr(p.status, slot >= p.place.slot_count ? TS_STATUS_PAGE : TS_STATUS_POSITION);
        }
        const bool live = there && lives(pos, slot);
        const uint32_t from = pos > p.back ? pos - p.back : 0;
        bool wait = live;
        float m = -INFINITY, l = 0.0f;
        f32x4 o[S::kD];
#pragma unroll
        for (uint32_t d = 0; d < S::kD; d++) o[d] = f32x4{0, 0, 0, 0};

        // A pass over the keys for each slot among the columns (one, where rows of a slot stand together).
        for (;;) {
            if (!(row_waits[0] | row_waits[1])) break;
            const uint32_t l0 = again(lane);
            const uint32_t now = __builtin_amdgcn_readfirstlane(
                rows_at[1][row_waits[0] ? __builtin_ctzll(row_waits[0]) : 64 + __builtin_ctzll(row_waits[1])]);
            // Keys that some row sees, [lo, hi], and those that all rows see alike, [same_lo, same_hi]; those of the wave's
            // columns, [wlo, whi] and [all_lo, all_hi].
            const bool act = wait && slot == now;
            wait = wait && !act;
            uint32_t lo, hi, same_lo, same_hi, wlo, whi, all_lo, all_hi;
            if (one_row()) {
                row_waits[0] = 0;
                lo = same_lo = all_lo = __builtin_amdgcn_readfirstlane(from);
                hi = same_hi = all_hi = __builtin_amdgcn_readfirstlane(pos);
                const bool any = __builtin_amdgcn_ballot_w64(act) != 0;
                wlo = any ? lo : 0xffffffffu;
                whi = any ? hi : 0;
            } else {
                uint32_t least[4] = {0xffffffffu, 0xffffffffu, 0xffffffffu, 0xffffffffu};
#pragma unroll
                for (uint32_t i = 0; i < 2; i++) {
                    const uint32_t row_pos = rows_at[0][64 * i + l0], since = row_pos > p.back ? row_pos - p.back : 0;
                    const bool here = (row_waits[i] >> l0 & 1) && rows_at[1][64 * i + l0] == now;
                    row_waits[i] &= ~__builtin_amdgcn_ballot_w64(here);
                    if (here) {
                        least[0] = min(least[0], since);
                        least[1] = min(least[1], ~row_pos);
                        least[2] = min(least[2], ~since);
                        least[3] = min(least[3], row_pos);
                    } else if (row_live[i] >> l0 & 1) {
                        least[2] = least[3] = 0;
                    }
                }
                lo = wave_least(least[0]);
                hi = ~wave_least(least[1]);
                same_lo = ~wave_least(least[2]);
                same_hi = wave_least(least[3]);
                wlo = row16_least(act ? from : 0xffffffffu);
                whi = ~row16_least(act ? ~pos : 0xffffffffu);
                all_lo = ~row16_least(act ? ~from : live ? 0u : 0xffffffffu);
                all_hi = row16_least(act ? pos : live ? 0u : 0xffffffffu);
            }
            auto differ = [&](uint32_t here, uint32_t n) { return max(here, lo) < same_lo || min(here + n - 1, hi) > same_hi; };
            const uint32_t base0 = lo & ~(kBlock - 1), last = hi / kBlock, np = (hi - base0) / S::kUnit + 1;
            const uint32_t unit0 = pass_unit(a, units, np), unit1 = pass_unit(b, units, np);
            if (unit0 >= unit1) continue;

            // Where the blocks of the rounds from r0 on are held, those of kChunk rounds one a lane, and which are not. (A block
            // that is not held is the first in the loads, and cleared. Without a table a slot is one page.)
            constexpr uint32_t kChunk = 64 / S::kIds;
            bf16x8 q[S::kQ];
            uint32_t r0, place;
            uint64_t lost_of;
            const_u32 *pages = in_constant<const_u32 *>(p.place.table + (size_t)now * p.place.kept_pages);
            auto look = [&](uint32_t round, bool first) {
                const uint32_t l0 = again(lane);
                const uint32_t block = min(base0 / kBlock + (WC == 1 ? 2 * wave : 0) +
                                               (round + l0 / S::kIds) * (S::kUnit / kBlock) + l0 % S::kIds, last);
                uint32_t page = now * (p.place.keys / kBlock);
                if (p.place.table) page = pages[block >> page_blocks];
                if (first) {
                    // q is asked for behind the pages, which the first keys wait for, and before those. (The pages' own wait is
                    // here, where q's loads are known to be younger.)
#pragma unroll
                    for (uint32_t j = 0; j < S::kQ; j++) q[j] = *(const bf16x8 *)(q_at + 32 * j);
                    asm volatile("; pages" : "+v"(page));
                    if (qsign)
#pragma unroll
                        for (uint32_t j = 0; j < S::kQ; j++) q[j] = as_bf16x8(__builtin_bit_cast(u32x4, q[j]) ^ qsign);
                }
                const bool lost = page >= page_count;
                place = ((lost ? 0 : page) << page_blocks) + (block & page_mask);
                lost_of = __builtin_amdgcn_ballot_w64(lost);
                r0 = round;
            };
            // The blocks of a round that are not held, a bit each.
            auto gone_of = [&](uint32_t round) { return (uint32_t)(lost_of >> (round - r0) * S::kIds) & ((1u << S::kIds) - 1); };
            auto issue = [&](uint32_t round, uint32_t slot_of_ring) {
                uint32_t from[S::kOwn];
#pragma unroll
                for (uint32_t i = 0; i < S::kOwn; i++) from[i] = S::kAside ? from_aside[i][threadIdx.x] : from_at[S::kAside ? 0 : i];
                const uint32_t to = lds_address(stage) + (slot_of_ring * S::kTeams + team) * S::kTile;
                u32x4 buf[2];
#pragma unroll
                for (uint32_t i = 0; i < 2; i++) {
                    const uint32_t block = __builtin_amdgcn_readlane(place, (round - r0) * S::kIds + (WC == 1 ? i : 2 * team + i));
                    buf[i] = rows_buffer((const char *)p.kept + (size_t)block * (kBlock * S::kRow));
                }
#pragma unroll
                for (uint32_t i = 0; i < S::kLoads; i++) {
                    const uint32_t part = mine + i * WC;
                    if (S::kLoads != S::kLeast && part >= S::kParts) break;
                    const bool on = WC == 1 && S::kParts == 36 && (i / 9 & 1);
                    rows_to_lds16(part < S::kParts / 2 ? buf[0] : buf[1], to + part * 1024,
                                  on ? (from[i % S::kOwn] ^ 48) + 8 * S::kRow : from[i % S::kOwn]);
                }
            };

            // A step is the wave's columns against the keys here .. here + 31 at `at`. Its scores: register i of s[t] is key
            // 16 t + 4 grp + i. Operands are read kAhead products ahead: left to itself, the compiler reads all it has
            // registers for, or one at a time and waits for each.
            auto scores = [&](const char *at, f32x4 (&s)[2]) {
                const uint32_t k0 = again(koff);
                bf16x8 ring[S::kAhead + 1];
                auto read_k = [&](uint32_t i) {
                    const uint32_t j = i / 2, t = i % 2;
                    ring[i % (S::kAhead + 1)] = *(const bf16x8 *)(at + (k0 ^ j % (S::kXor / 4) * 64) +
                                                               j / (S::kXor / 4) * (S::kXor * 16) + t * kBlock * S::kRow);
                };
                s[0] = s[1] = f32x4{0, 0, 0, 0};
#pragma unroll
                for (uint32_t i = 0; i < S::kAhead; i++) read_k(i);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (uint32_t i = 0; i < 2 * S::kQ; i++) {
                    if (i + S::kAhead < 2 * S::kQ) read_k(i + S::kAhead);
                    s[i % 2] = mfma16(ring[i % (S::kAhead + 1)], q[i / 2], s[i % 2]);
                    __builtin_amdgcn_sched_barrier(0);
                }
            };
            auto masked = [&](uint32_t here, uint32_t gone, f32x4 (&s)[2]) {
                if (here >= all_lo && here + (kKeys - 1) <= all_hi && !gone) return;
                const int upto = act ? (int)(pos - here) - 4 * (int)grp : -1, since = (int)(from - here) - 4 * (int)grp;
#pragma unroll
                for (int t = 0; t < 2; t++)
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const bool seen = 16 * t + i <= upto && 16 * t + i >= since;
                        s[t][i] = seen ? (gone >> t & 1 ? __builtin_nanf("") : s[t][i]) : -INFINITY;
                    }
            };
            // The softmax of a step: weights 2^(score - m) in bf16 parts. m moves only when a score passes it by 2^kSlack, so
            // most steps leave the sum and O as they are and no weight passes 2^kSlack.
            float mn, sum;
            uint32_t pw[4][S::kWeights];
            auto soft = [&](const f32x4 (&s)[2]) {
                const float mx = rows4_max(fmaxf(fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[0][2], s[0][3])),
                                                 fmaxf(fmaxf(s[1][0], s[1][1]), fmaxf(s[1][2], s[1][3])))) * sl;
                mn = mx > m + kSlack ? mx : m;
                const float mo = mn == -INFINITY ? 0.0f : mn;
                sum = 0.0f;
#pragma unroll
                for (uint32_t i = 0; i < 4; i++) {
                    const float x = __builtin_amdgcn_exp2f(fmaf(s[i / 2][i % 2 * 2], sl, -mo));
                    const float y = __builtin_amdgcn_exp2f(fmaf(s[i / 2][i % 2 * 2 + 1], sl, -mo));
                    sum += x + y;
                    split_pair<S::kWeights>(x, y, pw[i]);
                }
            };
            // The step's weights times its values, onto O.
            auto product = [&](uint32_t here, char *at, bool apart) {
                if (__builtin_amdgcn_ballot_w64(mn > m) != 0) {
                    const float alpha = mn > m ? __builtin_amdgcn_exp2f(m - mn) : 1.0f;
                    l *= alpha;
                    m = mn;
#pragma unroll
                    for (uint32_t d = 0; d < S::kD; d++) o[d] *= alpha;
                }
                l += sum;
                u32x4 w[S::kWeights];
#pragma unroll
                for (uint32_t e = 0; e < S::kWeights; e++) w[e] = u32x4{pw[0][e], pw[1][e], pw[2][e], pw[3][e]};
                if (apart) {
                    // Some key here is one column's and not another's. A value that is not finite must reach the former
                    // alone, and the product's 0 times it would be NaN: such values are looked for, become NaN where they
                    // are seen (their key's score is infinite or NaN as well, so the column's sum can be nothing else), and
                    // are cleared. (By all waves of the group together, but where each has keys of its own.)
                    uint32_t odd = 0;
#pragma unroll 2
                    for (uint32_t g = mine * 64 + again(lane); g < kKeys * RANK / 8; g += 64 * WC) {
                        const u32x4 x = *(const u32x4 *)(at + g / (RANK / 8) * S::kRow + g % (RANK / 8) * 16);
#pragma unroll
                        for (uint32_t e = 0; e < 4; e++) odd |= odd_mask(x[e]);
                    }
                    uint32_t any = __builtin_amdgcn_ballot_w64(odd != 0) != 0;
                    if (WC > 1) {
                        odd_met[wave] = any;
                        lds_barrier();
#pragma unroll
                        for (uint32_t i = 0; i < S::kWaves; i++) any |= __builtin_amdgcn_readfirstlane(odd_met[i]);
                    }
                    if (any) {
#pragma unroll 1
                        for (uint32_t k = 0; k < kKeys; k++) {
                            const uint32_t swap = swap_of<S::kPieces>(k), g = again(grp);
                            const uint32_t keep = act && here + k <= pos && here + k >= from ? 0xffffffffu : 0u;
                            const char *row = at + k * S::kRow + 8 * (g & 1);
#pragma unroll
                            for (uint32_t d = 0; d < S::kD; d++) {
                                u32x2 x = *(const u32x2 *)(row + ((2 * d + (g >> 1)) ^ swap) * 16);
                                x = u32x2{odd_mask(x[0]), odd_mask(x[1])} & keep;
                                o[d] += f32x4{lo_bf16(x[0]), hi_bf16(x[0]), lo_bf16(x[1]), hi_bf16(x[1])};
                                __builtin_amdgcn_sched_barrier(0);
                            }
                        }
                        if (WC > 1) lds_barrier();
#pragma unroll 1
                        for (uint32_t k = mine; k < kKeys; k += WC) {
                            uint32_t *x = (uint32_t *)(at + k * S::kRow) + again(lane) * (RANK / 128);
#pragma unroll
                            for (uint32_t e = 0; e < RANK / 128; e++) x[e] &= ~odd_mask(x[e]);
                        }
                        if (WC > 1) lds_barrier();
                    }
                }
                // V^T: d 16 dt + col of keys 4 grp .. and 16 + 4 grp .. (eight of them).
                const uint32_t v0 = again(voff);
                u32x4 ring[S::kAhead + 1];
                auto read_v = [&](uint32_t d) {
                    const char *v = at + d / (S::kXor / 2) * (S::kXor * 16) + (v0 ^ d % (S::kXor / 2) * 32);
                    const u32x2 lo4 = read_vt4(v), hi4 = read_vt4(v + kBlock * S::kRow);
                    ring[d % (S::kAhead + 1)] = u32x4{lo4.x, lo4.y, hi4.x, hi4.y};
                };
#pragma unroll
                for (uint32_t i = 0; i < S::kAhead; i++) read_v(i);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (uint32_t i = 0; i < S::kD; i++) {
                    if (i + S::kAhead < S::kD) read_v(i + S::kAhead);
#pragma unroll
                    for (uint32_t e = 0; e < S::kWeights; e++)
                        o[i] = mfma16(as_bf16x8(ring[i % (S::kAhead + 1)]), as_bf16x8(w[e]), o[i]);
                    __builtin_amdgcn_sched_barrier(0);
                }
            };
            auto step = [&](uint32_t here, char *at, uint32_t gone, bool apart) {
                f32x4 s[2];
                scores(at, s);
                masked(here, gone, s);
                soft(s);
                product(here, at, apart);
            };
            // Rows of a step that no column of the pass sees, or of no page, are zero in the products.
            auto clear = [&](uint32_t here, char *at, uint32_t gone) {
                for (uint32_t g = mine * 64 + again(lane); g < kKeys * S::kPieces; g += 64 * WC) {
                    const uint32_t row = g / S::kPieces, key = here + row;
                    if (key < lo || key > hi || gone >> (row / kBlock) & 1) *(u32x4 *)(at + g * 16) = u32x4{0, 0, 0, 0};
                }
                // (Rows that stand apart may leave keys of the pass that none of them sees.)
                if (gone && p.status && act && ((gone & 1 && here <= pos && here + (kBlock - 1) >= from) ||
                                                (gone & 2 && here + kBlock <= pos && here + (kKeys - 1) >= from)))
                    atomicOr(p.status, TS_STATUS_PAGE);
            };

            if (WC == 1) {
                char *at = stage + team * S::kTile;
                uint32_t round = unit0;
                look(round, true);
                for (; round < unit1; round++) {
                    const uint32_t here = base0 + round * S::kUnit + kKeys * wave;
                    if (here > hi) break;
                    if (round - r0 == kChunk) look(round, false);
                    const uint32_t gone = gone_of(round);
                    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the last step's reads
                    issue(round, 0);
                    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
                    if (here < lo || here + (kKeys - 1) > hi || gone) clear(here, at, gone);
                    step(here, at, gone, differ(here, kKeys));
                }
            } else {
                // kRing - 1 rounds on their way.
                constexpr uint32_t kLater = (S::kRing - 2) * S::kLeast;
                uint32_t gone[S::kRing], n = 0;
                look(unit0, true);
#pragma unroll
                for (uint32_t r = 0; r + 1 < S::kRing; r++) {
                    gone[r] = gone_of(unit0 + r);
                    if (unit0 + r < unit1) issue(unit0 + r, r);
                }
                for (uint32_t round = unit0; round < unit1; round++) {
                    if (unit1 - round >= S::kRing - 1)
                        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(kLater) : "memory");
                    else
                        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
                    const uint32_t next = round + S::kRing - 1;
                    gone[S::kRing - 1] = 0;
                    if (next < unit1) {
                        if (next - r0 == kChunk) look(next, false);
                        gone[S::kRing - 1] = gone_of(next);
                        issue(next, (n + S::kRing - 1) % S::kRing);
                    }
                    const uint32_t here = base0 + round * S::kUnit;
                    const uint32_t at_here = here + team * kKeys, lost = gone[0] >> (2 * team) & 3;
                    char *at = stage + (n * S::kTeams + team) * S::kTile;
                    if (here < lo || here + (S::kUnit - 1) > hi || gone[0]) {
                        clear(at_here, at, lost);
                        lds_barrier();
                    }
                    const bool apart = differ(here, S::kUnit);
                    n = n + 1 == S::kRing ? 0 : n + 1;
                    if (apart || (at_here <= whi && at_here + (kKeys - 1) >= wlo)) step(at_here, at, lost, apart);
#pragma unroll
                    for (uint32_t i = 0; i + 1 < S::kRing; i++) gone[i] = gone[i + 1];
                }
                lds_barrier();  // the last reads, before the next pass's loads
            }
        }

        // The teams' results joined: each team sums its share of O's tiles, which the others give it in LDS.
        constexpr uint32_t kShare = S::kD / S::kTeams;
        const uint32_t l0 = again(lane), c = 16 * mine + (l0 & 15), g = l0 >> 4;
        float most = m, sum = rows4_sum(l), weight[S::kTeams];
        weight[0] = 1.0f;
        char *given = stage + mine * ((S::kTeams - 1) * S::kD * 1024) + l0 * 16;
        if (S::kTeams > 1) {
            float *ml = (float *)(stage + WC * (S::kTeams - 1) * S::kD * 1024) + mine * S::kTeams * 32 + (l0 & 15);
            __syncthreads();
#pragma unroll
            for (uint32_t t = 0; t < S::kTeams; t++)
                if (t != team)
#pragma unroll
                    for (uint32_t d = 0; d < kShare; d++)
                        *(f32x4 *)(given + ((t * (S::kTeams - 1) + (team < t ? team : team - 1)) * kShare + d) * 1024) = o[t * kShare + d];
            if (g == 0) {
                ml[team * 32] = m;
                ml[team * 32 + 16] = sum;
            }
            __syncthreads();
#pragma unroll
            for (uint32_t t = 0; t < S::kTeams; t++) most = fmaxf(most, ml[t * 32]);
            sum = 0.0f;
#pragma unroll
            for (uint32_t t = 0; t < S::kTeams; t++) {
                weight[t] = weight_of(ml[t * 32], most);
                // (A part that has met nothing but NaN has no maximum either.)
                const float x = ml[t * 32 + 16];
                sum += x != x ? x : x * weight[t];
            }
        }
        if (!live) sum = __builtin_nanf("");
        // The wave's share of O, one team's code after the other (registers have no index): four sums of a column a lane.
        auto each_of = [&](auto put) {
#pragma unroll
            for (uint32_t t = 0; t < S::kTeams; t++) {
                if (t != team) continue;
#pragma unroll
                for (uint32_t d = t * kShare; d < (t + 1) * kShare; d++) {
                    f32x4 x = o[d] * weight[t];
#pragma unroll
                    for (uint32_t e = 0; e < S::kTeams; e++)
                        if (e != t)
                            x += weight[e] * *(const f32x4 *)(given + ((t * (S::kTeams - 1) + (e < t ? e : e - 1)) * kShare +
                                                                       d - t * kShare) * 1024);
                    put(d, x);
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
        };
        uint32_t r, h;
        if (column_of(p, tile_row(), tile_rows(), block, c, r, h)) {
            if (partial) {
                float *to = partial + (g * S::kCols + c) * 4;
                each_of([&](uint32_t d, f32x4 x) { *(f32x4 *)(to + 4 * d * S::kCols * 4) = x; });
                if (team == 0 && g == 0) {
                    partial[RANK * S::kCols + c] = most;
                    partial[RANK * S::kCols + S::kCols + c] = sum;
                }
            } else {
                uint16_t *to = p.out + ((size_t)r * p.heads + h) * RANK + 4 * g;
                const float by = 1.0f / sum;
                each_of([&](uint32_t d, f32x4 x) {
                    *(u32x2 *)(to + 16 * d) = u32x2{bf16_pair(x[0] * by, x[1] * by), bf16_pair(x[2] * by, x[3] * by)};
                });
            }
        }
        unit += b - a;
        tile++;
        if (p.whole || unit >= end) return;
        fetch();
        __syncthreads();
    }
}

// The parts of tiles that several groups have: a group takes 16 columns and 64 values of O, a thread four of one
// column. Tiles that one group had alone are out already.
template <uint32_t RANK>
__global__ __launch_bounds__(kJoinThreads) void join_latent_kernel(LatentParams p, uint32_t columns) {
    uint32_t u = blockIdx.x;
    const uint32_t piece = u % (RANK / 64), c0 = u / (RANK / 64) % (columns / 16) * 16;
    u /= RANK / 64 * (columns / 16);
    const uint32_t block = u % p.blocks, tile = u / p.blocks;
    const u32x4 share = *(const u32x4 *)(p.shares + 4 * tile);
    const uint32_t tiles = p.cut ? p.shares[4 * p.tiles] : p.tiles;
    const uint32_t first = __builtin_amdgcn_readfirstlane(share[0]), parts = __builtin_amdgcn_readfirstlane(share[1]);
    if (tile >= tiles || parts < 2) return;
    const uint32_t c = c0 + (threadIdx.x & 15), quad = piece * 16 + (threadIdx.x >> 4);
    uint32_t r, h;
    if (!column_of(p, __builtin_amdgcn_readfirstlane(share[2]), __builtin_amdgcn_readfirstlane(share[3]), block, c, r, h)) return;
    auto part_at = [&](uint32_t j) {
        return p.partials + ((size_t)((j ? 0 : p.groups) + first + j) * p.blocks + block) * part_floats<RANK>(columns);
    };
    float most = -INFINITY, sum = 0.0f;
    f32x4 o = {0, 0, 0, 0};
    constexpr uint32_t kBatch = 16;
    for (uint32_t j0 = 0; j0 < parts; j0 += kBatch) {
        float mq[kBatch], lq[kBatch];
        f32x4 oq[kBatch];
#pragma unroll
        for (uint32_t j = 0; j < kBatch; j++) {
            mq[j] = -INFINITY;
            if (j0 + j >= parts) continue;  // (all lanes alike)
            const float *at = part_at(j0 + j);
            mq[j] = at[RANK * columns + c];
            lq[j] = at[RANK * columns + columns + c];
            oq[j] = *(const f32x4 *)(at + (quad * columns + c) * 4);
        }
        float top = most;
#pragma unroll
        for (uint32_t j = 0; j < kBatch; j++) top = fmaxf(top, mq[j]);
        const float f = weight_of(most, top);
        most = top;
        sum *= f;
        o *= f;
#pragma unroll
        for (uint32_t j = 0; j < kBatch; j++) {
            if (j0 + j >= parts) continue;
            const float g = weight_of(mq[j], top);
            // (A part that has seen nothing of the column holds no sums, but one that met a NaN has no maximum either.)
            sum += mq[j] == -INFINITY ? lq[j] : lq[j] * g;
            o += mq[j] == -INFINITY ? oq[j] : oq[j] * g;
        }
    }
    o /= sum;
    *(u32x2 *)(p.out + ((size_t)r * p.heads + h) * RANK + 4 * quad) = u32x2{pack_bf16x2(o[0], o[1]), pack_bf16x2(o[2], o[3])};
}

struct Plan {
    uint32_t columns, block_heads, blocks, tile_rows, tiles, groups;
    bool shared, whole, cut;
};

// How many columns a group has, and how the keys are divided. A group takes some time for its q, its partial sums and
// their share of the join, and some for each key it reads; both grow with its columns, a key's less than they do. Of 16, 32,
// 64 and 128 columns those are taken whose groups are done first. The constants are times of the kernels' earlier forms, a key's
// of 256 + 32 values half the others'; as the kernels are (us of graph replays, about 5 of them the graph's; sequences x heads x
// keys; 16, 32, 64, 128 columns):
//   512 + 64: 1 x 16 x 4000 23, 26, 26, 32; 1 x 128 x 4000 26, 32, 35, 47; 4 x 128 x 4000 32, 32, 37, 46; 32 x 64 x 4000 59, 54,
//   49, 50; 32 x 128 x 512 .. 8192 138, 97, 70, 72; 2 x 512 rows of 16 heads x 2500, 4600 322, 241, 164, 150; the last two with
//   a window of 1000 54, 47, 39, 47 and 124, 98, 65, 74.
//   256 + 32: 18, 22, 22, 29; 21, 27, 27, 38; 24, 31, 30, 36; 34, 34, 34, 37; 58, 47, 46, 46; 130, 105, 99, 93; 35, 30, 29, 32
//   and 53, 42, 40, 50.
// Of 38 shapes the columns taken are within 10% of the best, but for drafts of 24 x 3 to 5 rows: of 16 heads x 4000 keys 73
// (16 columns) for 47 (64), and 256 + 32 values, 32 heads, a window of 1000 34 (16) for 29 (32).
//
// Rows of a tile that belong to two slots take two passes over keys, one after the other. So tiles are cut where slots change,
// which a group looks for among up to kCutRows rows; of more rows, and in 16 columns, a tile has no more than a fourth of those
// that stand together. (24 sequences of 3 to 5 rows, 32 heads, 1000 .. 9001 keys: 73 us, with a row a tile 98; 4 heads, 4000
// keys: 43 and 70.)
Plan plan(const ts_latent_args *k) {
    const ts_rows_args *a = &k->rows;
    constexpr double kStart[2][4] = {{19, 22, 29, 40}, {14.5, 19.5, 20, 29}};                // us (512 + 64 values; 256 + 32)
    constexpr double kKey[2][4] = {{0.020, 0.032, 0.033, 0.0565}, {0.010, 0.016, 0.0165, 0.028}};
    const uint32_t of = k->rank == 512 ? 0 : 1;
    const uint32_t run = std::max(1u, std::min(k->run, a->rows));
    Plan best = {};
    double least = INFINITY;
    for (uint32_t i = 0; i < 4; i++) {
        Plan s;
        s.columns = 16u << i;
        s.block_heads = std::min(a->heads, s.columns);
        s.blocks = (a->heads - 1) / s.block_heads + 1;
        s.tile_rows = std::max(1u, std::min(run, s.columns / s.block_heads));
        const uint32_t at_once = std::max(1u, (k->rank == 512 || s.columns >= 64 ? 256u : 512u) / s.blocks);  // a CU's one or two
        const uint32_t unit = kKeys * (s.columns == 16 ? 4 : s.columns == 128 ? 1 : 2);
        const uint64_t span = std::min<uint64_t>(std::min<uint64_t>((uint64_t)a->max_position + 1, a->keys),
                                                 (uint64_t)a->back + s.tile_rows + kBlock);
        auto shared = [&](uint32_t tiles) { return at_once > 1 && tiles <= std::min(kMaxTiles, 4 * at_once) && span > unit; };
        s.cut = s.columns > 16 && s.tile_rows > 1 && a->rows <= kCutRows && shared(a->rows);
        if (!s.cut) s.tile_rows = std::max(1u, std::min(run / 4, s.tile_rows));
        s.tiles = s.cut ? a->rows : (a->rows - 1) / s.tile_rows + 1;
        // (Cut tiles: as many as full runs make.)
        const uint32_t tiles = s.cut ? (a->rows * ((run - 1) / s.tile_rows + 1) - 1) / run + 1 : s.tiles;
        s.shared = shared(s.tiles);
        s.groups = s.shared ? (uint32_t)std::min<uint64_t>(at_once, s.tiles * ((span + unit - 1) / unit + 1)) : s.tiles;
        s.whole = s.shared && s.tiles <= kWholeTiles && s.tiles < s.groups && 3 * tiles <= s.groups;
        const double keys = (double)span * tiles * s.blocks / 256.0;  // a CU's
        const double takes = kStart[of][i] + keys * kKey[of][i];
        if (takes < least) least = takes, best = s;
    }
    return best;
}

size_t partial_bytes(const ts_latent_args *k, const Plan &s) {
    return s.shared ? (size_t)s.groups * 2 * s.blocks * s.columns * (k->rank + 2) * sizeof(float) : 0;
}
size_t share_bytes(const Plan &s) { return s.shared ? ((size_t)s.tiles * 4 + 1) * sizeof(uint32_t) : 0; }

bool wide(const ts_latent_args *k) { return k->rank == 512 && k->rows.width == 576; }
bool narrow(const ts_latent_args *k) { return k->rank == 256 && k->rows.width == 288; }

int check(const ts_latent_args *k) {
    TS_REQUIRE(k, "attend_latent: null args");
    const ts_rows_args *a = &k->rows;
    TS_REQUIRE(a->k && (a->rows == 0 || (a->q && a->out && a->slots && a->positions)), "attend_latent: null pointer");
    TS_REQUIRE(wide(k) || narrow(k), "attend_latent: rows of %u values, %u of them latent (576 and 512, or 288 and 256)",
               a->width, k->rank);
    TS_REQUIRE(a->kv_heads == 1 && a->heads >= 1 && a->heads <= 1024, "attend_latent: %u heads over %u rows a position",
               a->heads, a->kv_heads);
    TS_REQUIRE(a->q_dtype == TS_BF16 && a->kv_dtype == TS_BF16 && a->out_dtype == TS_BF16,
               "attend_latent: q, kept rows and out bf16 supported");
    int rc = ts::kept_check("attend_latent", a->kept_table, a->page, a->keys, k->slot_count, a->kept_pages, k->pages, true);
    if (rc) return rc;
    TS_REQUIRE(a->keys <= 1u << 30, "attend_latent: %u positions a slot", a->keys);
    TS_REQUIRE((uint64_t)k->pages * a->page <= 1ull << 36, "attend_latent: %u pages of %u rows", k->pages, a->page);
    TS_REQUIRE(ts::aligned(a->k, 16) && ts::aligned(a->q, 16) && ts::aligned(a->out, 16),
               "attend_latent: q, kept rows and out must be 16-byte aligned");
    return TS_OK;
}

template <uint32_t RANK, uint32_t ROPE, uint32_t WC>
int launch(const LatentParams &p, uint32_t groups, void *stream) {
    using S = Shape<RANK, ROPE, WC>;
    static const hipError_t attr = hipFuncSetAttribute((const void *)attend_latent_kernel<RANK, ROPE, WC>,
                                                       hipFuncAttributeMaxDynamicSharedMemorySize, S::kLds);
    if (attr != hipSuccess) return ts::hip_status(attr, "attend_latent: shared memory attribute");
    hipLaunchKernelGGL((attend_latent_kernel<RANK, ROPE, WC>), dim3(groups), dim3(64 * S::kWaves), S::kLds, (hipStream_t)stream, p);
    TS_CHECK_LAUNCH("attend_latent launch");
    return TS_OK;
}
template <uint32_t RANK, uint32_t ROPE>
int launch(const LatentParams &p, const Plan &s, void *stream) {
    const uint32_t groups = (s.groups + 7) / 8 * 8 * s.blocks;
    const int rc = s.columns == 16 ? launch<RANK, ROPE, 1>(p, groups, stream)
                   : s.columns == 32 ? launch<RANK, ROPE, 2>(p, groups, stream)
                   : s.columns == 64 ? launch<RANK, ROPE, 4>(p, groups, stream)
                                     : launch<RANK, ROPE, 8>(p, groups, stream);
    if (rc || !s.shared) return rc;
    hipLaunchKernelGGL(join_latent_kernel<RANK>, dim3(s.tiles * s.blocks * (s.columns / 16) * (RANK / 64)), dim3(kJoinThreads), 0,
                       (hipStream_t)stream, p, s.columns);
    TS_CHECK_LAUNCH("attend_latent join launch");
    return TS_OK;
}

}  // namespace

extern "C" size_t tessera_hip_attend_latent_workspace(const ts_latent_args *k) {
    if (!k || k->rows.heads == 0 || k->rows.rows == 0 || !(wide(k) || narrow(k))) return 0;
    const Plan s = plan(k);
    return partial_bytes(k, s) + share_bytes(s);
}

extern "C" int tessera_hip_attend_latent(const ts_latent_args *k, void *stream) {
    const int rc = check(k);
    if (rc) return rc;
    const ts_rows_args *a = &k->rows;
    if (a->rows == 0) return TS_OK;
    const Plan s = plan(k);
    TS_REQUIRE(((uint64_t)s.groups + 7) * s.blocks < 1u << 23, "attend_latent: %u rows in one launch", a->rows);  // (2^32 threads)
    const size_t partials = partial_bytes(k, s), need = partials + share_bytes(s);
    if (need && (!a->workspace || a->workspace_bytes < need || !ts::aligned(a->workspace, 16)))
        return ts::fail(TS_ERR_WORKSPACE, "attend_latent: workspace of %zu bytes, 16-byte aligned, needed", need);
    const uint64_t of = (uint64_t)a->rows * a->heads * 2;
    const uint64_t held = a->kept_table ? (uint64_t)k->pages * a->page : (uint64_t)k->slot_count * a->keys;
    const int over = ts::outputs_apart("attend_latent", {{"out", a->out, of * k->rank}},
                                       {{"q", a->q, of * a->width},
                                        {"kept", a->k, held * a->width * 2},
                                        {"slots", a->slots, (uint64_t)a->rows * 4},
                                        {"positions", a->positions, (uint64_t)a->rows * 4},
                                        {"the page table", a->kept_table, (uint64_t)k->slot_count * a->kept_pages * 4},
                                        {"the workspace", a->workspace, need}});
    if (over) return over;
    LatentParams p;
    p.q = (const uint16_t *)a->q; p.kept = (const uint16_t *)a->k; p.out = (uint16_t *)a->out;
    p.partials = need ? (float *)a->workspace : nullptr;
    p.shares = need ? (uint32_t *)((char *)a->workspace + partials) : nullptr;
    p.slots = a->slots; p.positions = a->positions; p.status = a->status;
    p.place.table = a->kept_table; p.place.keys = a->keys; p.place.slot_count = k->slot_count;
    p.place.kept_pages = a->kept_pages; p.place.page_shift = (uint32_t)__builtin_ctz(a->page); p.place.pages = k->pages;
    p.rows = a->rows; p.heads = a->heads; p.back = a->back; p.max_position = a->max_position;
    p.tile_rows = s.tile_rows; p.tiles = s.tiles; p.groups = s.groups;
    p.block_heads = s.block_heads; p.blocks = s.blocks;
    p.whole = s.shared && s.whole;
    p.cut = s.cut;
    p.scale = a->scale;
    return k->rank == 512 ? launch<512, 64>(p, s, stream) : launch<256, 32>(p, s, stream);
}
