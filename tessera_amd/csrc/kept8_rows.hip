// Attention over kept blocks (kept8.h) where a tile has more than 16 columns: prompts, chunks of them,
// and drafted rows under many q heads. Semantics and tiles as in kept8.hip, whose waves each stream keys
// of their own; here the waves of a group have columns of their own (16 or 32 each) and share the keys.
//
//  * A step is 64 keys, four blocks. Their codes are loaded a step ahead (16 or 32 bytes of K and of V a
//    thread), widened to bf16 once, with their scale, and put into LDS: one of two buffers and a barrier a step, or
//    one buffer and two barriers (buffers()). Widening per wave would cost each of the waves the 128
//    conversions that they share here.
//  * K lies in LDS as rows of 256 bytes, V^T (as the blocks hold it) as rows of 128; the 16-byte
//    chunks of a row are permuted by XOR so that the 16 rows of an operand read meet 16 places.
//  * The score, softmax and product steps of a wave are kept8.hip's, but the weights of bf16 q enter the product as
//    one bf16 part: in two the error against 64 bits falls from 2.1e-3 .. 2.3e-3 of the outputs to the 1.65e-3 of their
//    own rounding, but 24 x 5 drafted rows go from 77 to 87 us, 4 prompts of 2048 rows from 100 to 121.
//  * A tile's cost grows with its position, and a tile of 8 waves fills a CU: tiles are taken widest
//    first (by their last row's position), heads fastest, so that consecutive groups, which go to
//    different XCDs, leave each XCD one kv head's keys. Fewer tiles than groups share their keys (share_of).
// A wave's step is a chain (K from LDS, scores, softmax, V from LDS, product) that two or three waves a SIMD overlap
// in part. 4 prompts of 2048 rows, 16 heads over 8: 95 us one pass after the other, 720 TFLOP/s (104 us each by
// itself); vector work takes 54% of the cycles, the matrix unit 31%. 24 x 5 drafted rows, 64 heads over 8, 1000 .. 9001
// keys: 58 us and 6 for the join, 4.3 TB/s of codes; vector 43%, matrix 20%, LDS conflicts 14%. f32 chunks of up to 700
// rows with a window of 1000, 16 heads over 8: 54 and 8 us; vector 43%, matrix 38%.
#include <algorithm>

#include "kept8_attend.h"

namespace {

using namespace kept8;

constexpr uint32_t kKBytes = kStep * 256, kVBytes = 128 * kStep * 2, kStage = kKBytes + kVBytes;
constexpr uint32_t kMaxOrder = 256;  // tiles of rows that are ordered by cost

// A wave-uniform value over the group's W waves, joined by `f`.
template <int W, class F>
TS_DEV uint32_t over_waves(uint32_t *mine, uint32_t wave, uint32_t v, F f) {
    __syncthreads();
    mine[wave] = v;
    __syncthreads();
    uint32_t r = mine[0];
#pragma unroll
    for (int w = 1; w < W; w++) r = f(r, mine[w]);
    return __builtin_amdgcn_readfirstlane(r);
}

// The XOR of a V^T row's eight chunks: distinct for the rows of one parity among 16, which share half the
// banks, and so that lanes 0-3, 12-15 of one 16 and 4-11 of the next, which LDS serves together, meet no two either.
TS_DEV uint32_t v_swap(uint32_t d) {
    const uint32_t i = d >> 1;
    return (i & 1) | (i >> 1 & 2) | ((i ^ i << 1) & 4);
}

// One buffer of codes, and two barriers a step, where the registers let three groups of four waves onto a CU, whose
// LDS two buffers would fill with two (24 x 5 rows: 79 us, 87 with two buffers).
template <int QT, int W, bool QF32>
constexpr uint32_t buffers() { return QT == 1 && W == 4 && !QF32 ? 1 : 2; }

template <int QT, int W, bool QF32>
__global__ __launch_bounds__(64 * W, (buffers<QT, W, QF32>() == 1 ? 3 : 2)) void attend_kept8_rows_kernel(AttendParams p) {
    constexpr uint32_t kCols = 16 * QT * W, kParts = QF32 ? 3 : 1, kThreads = 64 * W;
    constexpr uint32_t kBuffers = buffers<QT, W, QF32>();
    // Operands read ahead (with one buffer four would spill: 81 us for 77).
    constexpr uint32_t kAhead = kBuffers == 1 ? 2 : 4;
    constexpr uint32_t kEach = 512 / kThreads;  // 16-byte pieces of K (and V) codes a thread and step
    extern __shared__ __attribute__((aligned(16))) char stage[];  // kBuffers of kStage
    __shared__ uint32_t shared_words[W], starts[kMaxShared + 1];
    // Per buffer and d: which of the step's 64 keys hold a NaN in V; and whether there has been any.
    __shared__ uint64_t nan_keys[kBuffers][128];
    __shared__ uint32_t nan_met;
    if (threadIdx.x == 0) nan_met = 0;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, t = threadIdx.x;
    const uint32_t col = lane & 15, grp = lane >> 4;

    // What the steps read from uniform addresses goes through vector loads: a scalar load on its way would make
    // every wait for LDS wait for it too.
    uint32_t zero = 0;
    asm volatile("" : "+v"(zero));

    // Whole tiles: the widest first. Shared keys: all groups at once (share_of).
    uint32_t u = blockIdx.x / p.kv_heads;
    const uint32_t kvh = blockIdx.x % p.kv_heads;
    if (!p.partials && p.tiles > 1 && p.tiles <= kMaxOrder) {
        uint32_t *cost = (uint32_t *)stage;
        for (uint32_t i = t; i < p.tiles; i += kThreads) {
            const uint32_t pos = p.positions[min((i + 1) * p.tile_rows, p.rows) - 1];
            cost[i] = min(min(pos, p.max_position), p.back);
        }
        if (t == 0) shared_words[0] = 0;
        __syncthreads();
        for (uint32_t i = t; i < p.tiles; i += kThreads) {
            const uint32_t c = cost[i];
            uint32_t before = 0;
            for (uint32_t j = 0; j < p.tiles; j++) {
                const uint32_t d = cost[j];
                before += (d > c) | ((d == c) & (j < i));
            }
            if (before == u) shared_words[0] = i;
        }
        __syncthreads();
        u = __builtin_amdgcn_readfirstlane(shared_words[0]);
    }
    Share share;
    if (!share_of<kStep>(p, u, lane, starts, share)) return;
    for (;;) {
        const Part part = part_of(p, u, lane, kvh, kCols, starts, share);
        const Tile tile = {part.row0, kvh};

        uint32_t pos[QT], from[QT], slot[QT];
        bool live[QT], wait[QT];
        bf16x8 q[QT][4][kParts];
        const float sl = base2_scale(p.scale);
        float m[QT], l[QT];
        f32x4 o[QT][8];  // O^T: lane's column, d 16 dt + 4 grp + i
#pragma unroll
        for (int qt = 0; qt < QT; qt++) {
            uint32_t r, h;
            const bool there = tile.column(p, 16 * (QT * wave + qt) + col, r, h);
            pos[qt] = there ? p.positions[r] : 0;
            slot[qt] = there ? p.slots[r] : 0;
            live[qt] = there && pos[qt] <= p.max_position && holds(p.place, slot[qt], pos[qt]);
            if (there && !live[qt] && p.status && part.a == 0 && grp == 0)
                atomicOr(p.status, slot[qt] >= p.place.slot_count ? TS_STATUS_PAGE : TS_STATUS_POSITION);
            from[qt] = pos[qt] > p.back ? pos[qt] - p.back : 0;
            load_q<QF32, kParts>(p, live[qt], live[qt] ? ((size_t)r * p.heads + h) * 128 : 0, grp, q[qt]);
            wait[qt] = live[qt];
            m[qt] = -INFINITY;
            l[qt] = 0.0f;
#pragma unroll
            for (int dt = 0; dt < 8; dt++) o[qt][dt] = f32x4{0, 0, 0, 0};
        }

        // LDS byte offsets of the lane's operands: K row (block col / 4, position 4 t + col % 4), chunk
        // 8 (j / 2) + 2 grp + j % 2; V^T row 16 dt + col, chunk 2 grp + x.
        uint32_t koff[4], voff[2];
#pragma unroll
        for (int j = 0; j < 4; j++)
            koff[j] = (16 * (col >> 2) + (col & 3)) * 256 + (((8 * (j >> 1) + 2 * grp + (j & 1)) ^ col) << 4);
#pragma unroll
        for (int x = 0; x < 2; x++) voff[x] = kKBytes + col * 128 + (((2 * grp + x) ^ v_swap(col)) << 4);

        for (;;) {
            // The slot of this pass: the first column's that still waits.
            uint32_t first = 0xffffffffu;
#pragma unroll
            for (int qt = QT - 1; qt >= 0; qt--) {
                const uint64_t b = __builtin_amdgcn_ballot_w64(wait[qt]);
                if (b) first = __builtin_amdgcn_readlane(slot[qt], __builtin_ctzll(b));
            }
            const uint32_t now = over_waves<W>(shared_words, wave, first, [](uint32_t a, uint32_t b) { return min(a, b); });
            if (now == 0xffffffffu) break;  // (a served slot is below slot_count)
            bool act[QT];
            uint32_t lo = 0xffffffffu, hi = 0, all_lo = 0, all_hi = 0xffffffffu;
#pragma unroll
            for (int qt = 0; qt < QT; qt++) {
                act[qt] = wait[qt] && slot[qt] == now;
                wait[qt] = wait[qt] && !act[qt];
                if (act[qt]) {
                    lo = min(lo, from[qt]);
                    hi = max(hi, pos[qt]);
                    all_lo = max(all_lo, from[qt]);
                    all_hi = min(all_hi, pos[qt]);
                } else if (live[qt]) {
                    all_lo = 0xffffffffu;
                }
            }
            // The wave's own keys [wlo, whi] (none: wlo above whi), the group's [lo, hi].
            const uint32_t wlo = row16_least(lo), whi = ~row16_least(~hi);
            all_lo = ~row16_least(~all_lo);
            all_hi = row16_least(all_hi);
            lo = over_waves<W>(shared_words, wave, wlo, [](uint32_t a, uint32_t b) { return min(a, b); });
            hi = over_waves<W>(shared_words, wave, whi, [](uint32_t a, uint32_t b) { return max(a, b); });
            const uint32_t base0 = lo & ~(kBlock - 1), last = hi / kBlock, np = (hi - base0) / kStep + 1;
            const uint32_t unit0 = pass_unit(part.a, part.n, np), unit1 = pass_unit(part.b, part.n, np);
            if (unit0 >= unit1) continue;
            uint32_t base = base0 + unit0 * kStep;
            const uint32_t end = base0 + (unit1 - 1) * kStep;  // the last step's

            // A thread's pieces: number t + i kThreads of the step's 512, block (t + i kThreads) / 128 (the
            // wave's own), 16 bytes of K and 16 of V. The page's id is asked for a step before the codes.
            u32x4 kraw[kEach], vraw[kEach];
            ts_f32x2 scale[kEach];
            uint32_t id[kEach], gone;  // gone: bit i: piece i's page is not held
            auto key_of = [&](uint32_t base, uint32_t i) {
                return min(base / kBlock + ((wave + i * W) >> 1), last) * kBlock;
            };
            const uint32_t *pages = p.place.table + (size_t)now * p.place.kept_pages + zero;
            auto look = [&](uint32_t base) {
#pragma unroll
                for (uint32_t i = 0; i < kEach; i++)
                    id[i] = p.place.table ? pages[key_of(base, i) >> p.place.page_shift] : 0;
            };
            auto fetch = [&](uint32_t base) {
                uint32_t block[kEach];
                gone = 0;
#pragma unroll
                for (uint32_t i = 0; i < kEach; i++) {
                    bool lost;
                    block[i] = block_in(p.place, now, __builtin_amdgcn_readfirstlane(id[i]), key_of(base, i), lost);
                    gone |= lost ? 1u << i : 0u;
                }
                look(min(base + kStep, end));
#pragma unroll
                for (uint32_t i = 0; i < kEach; i++) {
                    const size_t at_scale = ((size_t)block[i] * scale_heads(p.kv_heads) + kvh) * 2;
                    scale[i] = *(const ts_f32x2 *)(p.scales + at_scale + zero);
                    const size_t at =
                        ((size_t)block[i] * p.kv_heads + kvh) * kBlockBytes + ((t + i * kThreads) & 127) * 16;
                    kraw[i] = *(const u32x4 *)(p.k + at);
                    vraw[i] = *(const u32x4 *)(p.v + at);
                }
            };
            auto stash = [&](uint32_t buffer, uint32_t base) {
                if (gone) {  // NaN keys for the rows that see them (put in here: at the loads it would wait for them)
#pragma unroll
                    for (uint32_t i = 0; i < kEach; i++)
                        if (gone >> i & 1) {
                            kraw[i] = u32x4{0x7f7f7f7fu, 0x7f7f7f7fu, 0x7f7f7f7fu, 0x7f7f7f7fu};
                            vraw[i] = u32x4{0, 0, 0, 0};
                        }
                    if (p.status && lane == 0) atomicOr(p.status, TS_STATUS_PAGE);
                }
                char *to = stage + buffer * kStage;
#pragma unroll
                for (uint32_t i = 0; i < kEach; i++) {
                    const uint32_t j = (wave + i * W) >> 1, c = (t + i * kThreads) & 127;
                    const uint32_t key = c >> 3, chunk = 2 * (c & 7), swap = (key & 3) | (j << 2);
                    char *row = to + (16 * j + key) * 256;
                    *(bf16x8 *)(row + ((chunk ^ swap) << 4)) = codes8(kraw[i].x, kraw[i].y, scale[i].x);
                    *(bf16x8 *)(row + (((chunk + 1) ^ swap) << 4)) = codes8(kraw[i].z, kraw[i].w, scale[i].x);
                    u32x4 v = vraw[i];
                    if (base < lo || base + (kStep - 1) > hi) {  // codes outside [lo, hi] may be anything
                        const uint32_t key0 = base + kBlock * j;
                        v = u32x4{within4(v.x, key0, lo, hi), within4(v.y, key0 + 4, lo, hi), within4(v.z, key0 + 8, lo, hi),
                                  within4(v.w, key0 + 12, lo, hi)};
                    }
                    // A NaN is 0 in the products, and reaches what sees it by itself (below): a weight of 0 times
                    // NaN must not reach the columns that do not.
                    const u32x4 nan = {nan_codes(v.x), nan_codes(v.y), nan_codes(v.z), nan_codes(v.w)};
                    uint32_t keys = 0;
                    if (__builtin_amdgcn_ballot_w64((nan.x | nan.y | nan.z | nan.w) != 0) != 0) {
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            v[e] &= ~((nan[e] >> 7) * 0xffu);
                            keys |= ((nan[e] >> 7) * 0x10204080u >> 28 & 0xfu) << (4 * e);
                        }
                        if (lane == 0) nan_met = 1;
                    }
                    ((uint16_t *)nan_keys[buffer])[4 * c + j] = keys;
                    row = to + kKBytes + c * 128;
                    *(bf16x8 *)(row + (((2 * j) ^ v_swap(c)) << 4)) = codes8(v.x, v.y, scale[i].y);
                    *(bf16x8 *)(row + (((2 * j + 1) ^ v_swap(c)) << 4)) = codes8(v.z, v.w, scale[i].y);
                }
            };

            look(base);
            fetch(base);
            uint32_t next = base;  // the step whose codes are in registers
            if (kBuffers == 2) {
                stash(0, base);
                next = min(base + kStep, end);
                fetch(next);
            }
            for (uint32_t buffer = 0;; buffer ^= kBuffers - 1) {
                lds_barrier();  // two buffers: this step's codes are in; the readers of the other are done
                const bool go = base < end;
                const uint32_t here = base;
                if (kBuffers == 1 || go) {
                    stash(buffer ^ (kBuffers - 1), next);
                    base = kBuffers == 1 ? min(base + kStep, end) : next;
                    next = kBuffers == 1 ? base : min(base + kStep, end);
                    fetch(next);
                }
                if (kBuffers == 1) lds_barrier();
                if (here <= whi && here + (kStep - 1) >= wlo) {
                    const char *kb = stage + buffer * kStage, *vb = kb;
                    const uint32_t nan = __builtin_amdgcn_readfirstlane(nan_met);
                    // Operands are read a few products ahead: left to itself, the compiler reads one at a time and
                    // waits for each (4 prompts of 2048 rows 105 -> 100 us, f32 chunks 68 -> 61).
                    f32x4 s[QT][4];
                    bf16x8 ahead[2][kAhead];
                    auto read_k = [&](uint32_t x) {
#pragma unroll
                        for (uint32_t i = 0; i < kAhead; i++)
                            ahead[x & 1][i] =
                                *(const bf16x8 *)(kb + koff[(x * kAhead + i) % 4] + (x * kAhead + i) / 4 * 1024);
                        __builtin_amdgcn_sched_barrier(0);
                    };
#pragma unroll
                    for (int x = 0; x < 4; x++)
#pragma unroll
                        for (int qt = 0; qt < QT; qt++) s[qt][x] = f32x4{0, 0, 0, 0};
                    read_k(0);
#pragma unroll
                    for (uint32_t x = 0; x < 16 / kAhead; x++) {
                        if (x + 1 < 16 / kAhead) read_k(x + 1);
#pragma unroll
                        for (uint32_t i = 0; i < kAhead; i++)
#pragma unroll
                            for (int qt = 0; qt < QT; qt++) {
                                const uint32_t j = (x * kAhead + i) % 4;
                                f32x4 &to = s[qt][(x * kAhead + i) / 4];
#pragma unroll
                                for (uint32_t e = 0; e < kParts; e++) to = mfma16(ahead[x & 1][i], q[qt][j][e], to);
                            }
                        __builtin_amdgcn_sched_barrier(0);
                    }
                    if (here < all_lo || here + (kStep - 1) > all_hi) {
#pragma unroll
                        for (int qt = 0; qt < QT; qt++) {
                            const uint32_t seen = act[qt] ? seen_keys(here + kBlock * grp, from[qt], pos[qt]) : 0u;
#pragma unroll
                            for (int x = 0; x < 4; x++)
#pragma unroll
                                for (int e = 0; e < 4; e++)
                                    s[qt][x][e] = seen >> (4 * x + e) & 1 ? s[qt][x][e] : -INFINITY;
                        }
                    }
                    bf16x8 w[QT][2][kParts];
#pragma unroll
                    for (int qt = 0; qt < QT; qt++) weigh<kParts, 8>(s[qt], sl, m[qt], l[qt], o[qt], w[qt]);
                    auto read_v = [&](uint32_t x) {
#pragma unroll
                        for (uint32_t i = 0; i < kAhead; i++)
                            ahead[x & 1][i] = *(const bf16x8 *)(vb + voff[i % 2] + (x * kAhead + i) / 2 * 2048);
                        __builtin_amdgcn_sched_barrier(0);
                    };
                    read_v(0);
#pragma unroll
                    for (uint32_t x = 0; x < 16 / kAhead; x++) {
                        if (x + 1 < 16 / kAhead) read_v(x + 1);
#pragma unroll
                        for (uint32_t i = 0; i < kAhead; i++)
#pragma unroll
                            for (int qt = 0; qt < QT; qt++) {
                                f32x4 &to = o[qt][(x * kAhead + i) / 2];
#pragma unroll
                                for (uint32_t e = 0; e < kParts; e++) to = mfma16(ahead[x & 1][i], w[qt][i % 2][e], to);
                            }
                        __builtin_amdgcn_sched_barrier(0);
                    }
                    if (nan) {
#pragma unroll
                        for (int qt = 0; qt < QT; qt++) {
                            uint64_t seen = 0;
#pragma unroll
                            for (int j = 0; j < 4; j++)
                                if (act[qt]) seen |= (uint64_t)seen_keys(here + kBlock * j, from[qt], pos[qt]) << (16 * j);
#pragma unroll
                            for (int dt = 0; dt < 8; dt++)
#pragma unroll
                                for (int e = 0; e < 4; e++)
                                    if (nan_keys[buffer][16 * dt + 4 * grp + e] & seen) o[qt][dt][e] = __builtin_nanf("");
                        }
                    }
                }
                if (!go) break;
            }
        }

        // A column is one wave's: O / l, or the part's result. Refused rows are NaN.
#pragma unroll
        for (int qt = 0; qt < QT; qt++) {
            const uint32_t c = 16 * (QT * wave + qt) + col;
            uint32_t r, h;
            const float sum = live[qt] ? rows4_sum(l[qt]) : __builtin_nanf("");
            if (!tile.column(p, c, r, h)) continue;
            if (part.partial) {
                float *at = part.partial + c * kPart;
                if (grp == 0) {
                    at[0] = m[qt];
                    at[1] = sum;
                }
#pragma unroll
                for (int dt = 0; dt < 8; dt++) *(f32x4 *)(at + 4 + 16 * dt + 4 * grp) = o[qt][dt];
            } else {
#pragma unroll
                for (int dt = 0; dt < 8; dt++)
                    store4(p, ((size_t)r * p.heads + h) * 128 + 16 * dt + 4 * grp, o[qt][dt] / sum);
            }
        }
        share.unit += part.b - part.a;
        share.tile++;
        if (share.unit >= share.end) return;
    }
}

template <int QT, int W, bool QF32>
int launch(const AttendParams &p, uint32_t groups, void *stream) {
    constexpr uint32_t kLds = buffers<QT, W, QF32>() * kStage;
    static const hipError_t attr = hipFuncSetAttribute((const void *)attend_kept8_rows_kernel<QT, W, QF32>,
                                                       hipFuncAttributeMaxDynamicSharedMemorySize, kLds);
    if (attr != hipSuccess) return ts::hip_status(attr, "attend_kept8: shared memory attribute");
    hipLaunchKernelGGL((attend_kept8_rows_kernel<QT, W, QF32>), dim3(groups), dim3(64 * W), kLds, (hipStream_t)stream, p);
    TS_CHECK_LAUNCH("attend_kept8 rows launch");
    return TS_OK;
}

}  // namespace

int ts::kept8_rows_launch(const AttendParams &p, uint32_t columns, bool qf32, uint32_t groups, void *stream) {
    if (columns == 64) return qf32 ? launch<1, 4, true>(p, groups, stream) : launch<1, 4, false>(p, groups, stream);
    if (columns == 128) return qf32 ? launch<1, 8, true>(p, groups, stream) : launch<2, 4, false>(p, groups, stream);
    return launch<2, 8, false>(p, groups, stream);
}
