// The expanded form of latent attention over whole sequences packed back to back: row i of a sequence of n rows and m
// keys stands at m - n + i, w = softmax((q . k + q' . r) * scale) over the keys [position - back, position], out = sum
// of w v; every head has keys k and values v of its own, the rotated part r is all heads'.
//
// A wave has 32 rows of one head, the columns of S^T = K q^T and O^T = V^T P^T on the 32-wide matrix products, so a
// row's scores stay in two lanes and P^T is the second product's operand as it stands. The four waves of a group have
// 128 neighbouring rows and share the keys, 64 a step: k, r and v rows go from memory straight to LDS, a step ahead of
// their use; V^T comes through the transposing LDS read. Two groups share a CU (all of its LDS: there is none besides
// the steps'), so that one's softmax runs under the other's products.
//
// 4 prompts of 2048 rows, 16 heads of 128 + 64 and 128 values: 107 us, 800 TFLOP/s (132 us before a step's halves took turns
// and tiles of a head shared an XCD, 117 with a step's loads before its products); one of 16384 rows 1000 TFLOP/s. The
// matrix unit is busy for 50% of the cycles and the vector unit for 47%, at the clock of 1.7 GHz that the card then keeps; LDS
// for a quarter. Small grids are bound by a wave's steps in turn, some 1.4 us each (5 sequences of up to 900 rows, 5 heads of
// 64 + 32 and 64 values: 25 us; one prompt of 2048 rows and 8 heads 46 us). Weights enter their product in one bf16 part: two bring
// the error against 64 bits (2-norm) from 2.1e-3 (2.3e-3 with 64 values) to the output's own rounding, 1.6e-3, and take the 4
// prompts from 108 to 134 us, the 5 sequences from 28 to 31 (graph replays).
#include "latent.h"
#include "places.h"

namespace {

using namespace latent;

constexpr uint32_t kWaves = 4, kThreads = 64 * kWaves, kRows = 32 * kWaves, kKeys = 64, kRing = 2;
constexpr uint32_t kAhead = 4;       // operands read ahead of their products
constexpr int kCostBits = 12;  // of the steps that tiles are ordered by
constexpr float kSlack = 8.0f;       // base-2 headroom of the softmax reference point

struct FlashParams {
    const uint16_t *q, *k, *v, *r;
    uint16_t *out;
    const uint32_t *first, *key_first;
    uint32_t rows, key_rows, seqs, heads, tiles;
    uint32_t q_stride, k_stride, k_head, v_stride, v_head, r_stride, back;
    float scale;
};

// Sequence s: n rows from row0 on, m keys from key0 on; n 0 where its bounds are not in order or in the tensors.
struct Sequence {
    uint32_t row0, n, key0, m;
};
TS_DEV Sequence sequence_of(const FlashParams &p, uint32_t s) {
    Sequence q = {0, p.rows, 0, p.key_rows};
    const uint32_t *kf = p.key_first ? p.key_first : p.first;
    if (p.first) {
        const uint32_t a = p.first[s], b = p.first[s + 1];
        q.row0 = a;
        q.n = a <= b && b <= p.rows ? b - a : 0;
    }
    if (kf) {
        const uint32_t a = kf[s], b = kf[s + 1];
        q.key0 = a;
        q.m = b - a;
        if (a > b || b > p.key_rows) q.n = 0;
    }
    return q;
}
TS_DEV uint32_t tiles_of(const Sequence &q) { return q.n / kRows + (q.n % kRows != 0); }
// Sequence s (a lane's own; none past the last), its n tiles, and those of it and the lanes' before it.
TS_DEV uint32_t tiles_upto(const FlashParams &p, uint32_t s, Sequence &q, uint32_t &n) {
    q = Sequence{0, 0, 0, 0};
    if (s < p.seqs) q = sequence_of(p, s);
    n = tiles_of(q);
    uint32_t upto = n;
    for (uint32_t d = 1; d < 64; d <<= 1) {
        const uint32_t x = __shfl_up((int)upto, d, 64);
        if ((threadIdx.x & 63) >= d) upto += x;
    }
    return upto;
}
// The steps that a sequence's tile t takes (as far as kCostBits tell), and one.
TS_DEV uint32_t cost_of(const FlashParams &p, const Sequence &q, uint32_t t) {
    const int64_t last = (int64_t)q.m - q.n + min((t + 1) * kRows, q.n);
    const uint32_t keys = last <= 0 ? 0 : (uint32_t)min(last, (int64_t)p.back + kRows);
    return min(keys / kKeys, (1u << kCostBits) - 2) + 1;
}
TS_DEV float halves_max(float x) {
    const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
}
TS_DEV float halves_sum(float x) {
    const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(a[0]) + __uint_as_float(a[1]);
}
TS_DEV uint32_t bf16_pair(float a, float b) {
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(ts_f32x2{a, b}, ts_bf16x2));
}
// The XOR of a row's 16-byte pieces in LDS, of P pieces: the 16 rows that an operand's read serves at once meet 16
// places (LDS serves 256 bytes at a time); the four rows by four pieces of a transposing read likewise.
template <uint32_t P>
TS_DEV uint32_t key_swap(uint32_t row) {
    return P == 16 ? row & 15 : P == 8 ? row >> 1 & 7 : row >> 2 & 3;
}
template <uint32_t P>
TS_DEV uint32_t value_swap(uint32_t row) {
    return P == 16 ? (row & 3) << 2 : (row >> 1 & 1) << 2;
}

template <uint32_t NOPE, uint32_t ROPE, uint32_t VALUE>
__global__ __launch_bounds__(kThreads, 2) void flash_latent_kernel(FlashParams p) {
    constexpr uint32_t kPk = NOPE / 8, kPr = ROPE / 8, kPv = VALUE / 8;  // pieces of a row
    constexpr uint32_t kK = kKeys * NOPE * 2, kR = kKeys * ROPE * 2, kV = kKeys * VALUE * 2, kStage = kK + kR + kV;
    constexpr uint32_t kD = VALUE / 32;
    extern __shared__ __attribute__((aligned(16))) char stage[];  // kRing of kStage: k, r, v rows
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const uint32_t col = lane & 31, half = lane >> 5;
    // Groups go to the eight XCDs in turn: where heads are whole eights, a head's tiles go to one, one head after the other,
    // so that the tiles that run at once share their keys in its L2.
    const uint32_t x = blockIdx.x & 7, y = blockIdx.x >> 3;
    const bool eights = p.heads % 8 == 0;
    const uint32_t h = eights ? y / p.tiles * 8 + x : blockIdx.x % p.heads;
    uint32_t t = eights ? y % p.tiles : blockIdx.x / p.heads;

    // The group's row tile: those of all sequences, one behind the other, 64 at a time the widest first. Every wave works
    // it out for itself.
    uint32_t n;
    Sequence q;
    uint32_t upto = tiles_upto(p, lane, q, n);
    if (p.tiles > 1) {
        // The costs of the 64 into LDS (the same by every wave, at any time), one a lane; 0: no tile.
        uint32_t *cost = (uint32_t *)stage, before = 0;
        const uint32_t base = t & ~63u;
        t &= 63;
        for (uint32_t s0 = 0;;) {
            if (p.seqs <= 16) {  // a sequence after the other, a tile a lane
                for (uint32_t s = 0; s < p.seqs; s++) {
                    const Sequence x = {0, (uint32_t)__builtin_amdgcn_readlane(q.n, s), 0, (uint32_t)__builtin_amdgcn_readlane(q.m, s)};
                    const uint32_t all = tiles_of(x), first = __builtin_amdgcn_readlane(upto, s) - all, y = base + lane - first;
                    if (base + lane >= first && y < all) cost[lane] = cost_of(p, x, y);
                }
            } else {
                const uint32_t first = before + upto - n;
                for (uint32_t y = first < base ? base - first : 0; y < n && first + y < base + 64; y++)
                    cost[first + y - base] = cost_of(p, q, y);
            }
            before += __builtin_amdgcn_readlane(upto, 63);
            s0 += 64;
            if (s0 >= p.seqs || before >= base + 64) break;
            upto = tiles_upto(p, s0 + lane, q, n);
        }
        if (base + lane >= before) cost[lane] = 0;
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        // The cost of rank t, bit by bit from the highest; then the t-th of those that cost as much, in order.
        const uint32_t c = cost[lane];
        uint32_t want = 0;
#pragma unroll
        for (int bit = kCostBits - 1; bit >= 0; bit--) {
            const uint32_t with = want | 1u << bit;
            const uint32_t more = __builtin_popcountll(__builtin_amdgcn_ballot_w64(c >> bit == with >> bit));
            if (t < more)
                want = with;
            else
                t -= more;
        }
        const uint64_t same = __builtin_amdgcn_ballot_w64(c == want);
        const uint32_t rank = __builtin_amdgcn_mbcnt_hi((uint32_t)(same >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)same, 0));
        t = base + __builtin_ctzll(__builtin_amdgcn_ballot_w64(c == want && rank == t));
        __syncthreads();  // (before the first step's rows)
        if (p.seqs > 64) upto = tiles_upto(p, lane, q, n);
    }
    for (uint32_t s0 = 64;; s0 += 64) {
        const uint64_t here = __builtin_amdgcn_ballot_w64(t < upto);
        if (here) {
            const uint32_t at = __builtin_ctzll(here);
            t -= __builtin_amdgcn_readlane(upto - n, at);
            q = Sequence{(uint32_t)__builtin_amdgcn_readlane(q.row0, at), (uint32_t)__builtin_amdgcn_readlane(q.n, at),
                         (uint32_t)__builtin_amdgcn_readlane(q.key0, at), (uint32_t)__builtin_amdgcn_readlane(q.m, at)};
            break;
        }
        if (s0 >= p.seqs) return;
        t -= __builtin_amdgcn_readlane(upto, 63);
        upto = tiles_upto(p, s0 + lane, q, n);
    }
    t = __builtin_amdgcn_readfirstlane(t);
    q = Sequence{(uint32_t)__builtin_amdgcn_readfirstlane(q.row0), (uint32_t)__builtin_amdgcn_readfirstlane(q.n),
                 (uint32_t)__builtin_amdgcn_readfirstlane(q.key0), (uint32_t)__builtin_amdgcn_readfirstlane(q.m)};
    const uint32_t i0 = t * kRows;
    // Position of the group's row i: shift + i, negative where it sees nothing.
    const int32_t shift = (int32_t)((int64_t)q.m - q.n);
    const uint32_t i = i0 + 32 * wave + col;
    const bool there = i < q.n;
    const int32_t pos = shift + (int32_t)min(i, q.n - 1);
    const uint32_t row = q.row0 + min(i, q.n - 1);
    // The scale to base 2, positive: its sign goes into q, exactly.
    const float sl = p.scale == 0.0f ? 0x1p-100f : fabsf(p.scale) * 1.4426950408889634f;
    const uint32_t qsign = p.scale < 0.0f ? 0x80008000u : 0u;
    constexpr uint32_t kQ = (NOPE + ROPE) / 16;
    bf16x8 qv[kQ];
    {
        const uint16_t *at = p.q + (size_t)row * p.q_stride + h * (NOPE + ROPE) + 8 * half;
#pragma unroll
        for (uint32_t j = 0; j < kQ; j++) qv[j] = as_bf16x8(*(const u32x4 *)(at + 16 * j) ^ qsign);
    }
    auto from_of = [&](int32_t pos) { return pos > 0 && (uint32_t)pos > p.back ? pos - (int32_t)p.back : 0; };
    const int32_t from = from_of(pos);
    // Keys [lo, hi] that some row of the group (of the wave) sees, and those that all do.
    const int32_t p0 = shift + (int32_t)i0, p1 = shift + (int32_t)min(i0 + kRows, q.n) - 1;
    const int32_t w0 = shift + (int32_t)min(i0 + 32 * wave, q.n - 1), w1 = shift + (int32_t)min(i0 + 32 * wave + 31, q.n - 1);
    const int32_t lo = from_of(p0), hi = p1, same_lo = from_of(p1), same_hi = p0;
    const int32_t wlo = from_of(w0), whi = i0 + 32 * wave < q.n ? w1 : -1, wsame_lo = from_of(w1), wsame_hi = w0;

    float m = -INFINITY, l = 0.0f;
    f32x16 o[kD];
#pragma unroll
    for (uint32_t d = 0; d < kD; d++)
#pragma unroll
        for (int e = 0; e < 16; e++) o[d][e] = 0.0f;

    // LDS offsets of the lane's operands: piece `half` of key `col` (others by the XOR of their piece), and V^T d 16
    // (lane / 16 % 2) + 4 (lane % 4) .. of keys 4 half + lane / 4 % 4 (and 8 more).
    const uint32_t koff = col * (2 * NOPE) + (half ^ key_swap<kPk>(col)) * 16;
    const uint32_t roff = kK + col * (2 * ROPE) + (half ^ key_swap<kPr>(col)) * 16;
    const uint32_t vrow = 4 * half + (lane >> 2 & 3);
    const uint32_t voff = kK + kR + vrow * (2 * VALUE) + (((lane >> 4 & 1) * 2 + (lane >> 1 & 1)) ^ value_swap<kPv>(vrow)) * 16 +
                          (lane & 1) * 8;

    const int32_t base = lo & ~31;
    const uint32_t steps = hi < 0 ? 0 : (uint32_t)(hi - base) / kKeys + 1;
    // Where the lane's 16 bytes of each of the wave's loads of a step come from.
    constexpr uint32_t kPartsK = kK / 1024 / kWaves, kPartsR = kR / 1024 / kWaves, kPartsV = kV / 1024 / kWaves;
    uint32_t kplace[kPartsK], rplace[kPartsR], vplace[kPartsV];
#pragma unroll
    for (uint32_t x = 0; x < kPartsK; x++) {
        const uint32_t g = 64 * (x * kWaves + wave) + lane, r = g / kPk;
        kplace[x] = r * p.k_stride * 2 + (g % kPk ^ key_swap<kPk>(r)) * 16;
    }
#pragma unroll
    for (uint32_t x = 0; x < kPartsR; x++) {
        const uint32_t g = 64 * (x * kWaves + wave) + lane, r = g / kPr;
        rplace[x] = r * p.r_stride * 2 + (g % kPr ^ key_swap<kPr>(r)) * 16;
    }
#pragma unroll
    for (uint32_t x = 0; x < kPartsV; x++) {
        const uint32_t g = 64 * (x * kWaves + wave) + lane, r = g / kPv;
        vplace[x] = r * p.v_stride * 2 + (g % kPv ^ value_swap<kPv>(r)) * 16;
    }
    // A step's rows, a KiB a load, of which a wave has kLoads; keys past the last are the last again. The vector cache
    // takes 64 bytes a cycle, so that a step's loads one behind the other keep a wave for 640 cycles: they go between
    // the products.
    constexpr uint32_t kLoads = kPartsK + kPartsR + kPartsV;
    const char *kat = (const char *)(p.k + (size_t)(q.key0 + base) * p.k_stride + (size_t)h * p.k_head);
    const char *vat = (const char *)(p.v + (size_t)(q.key0 + base) * p.v_stride + (size_t)h * p.v_head);
    const char *rat = (const char *)(p.r + (size_t)(q.key0 + base) * p.r_stride);
    uint32_t most = (uint32_t)(hi - base);  // keys behind the step's first
    auto last = [&]() {
        if (most >= kKeys - 1) return;
        auto ends = [&](uint32_t &at, uint32_t row0, uint32_t pieces, uint32_t stride) {
            const uint32_t row = row0 + again(lane) / pieces;
            at -= row > most ? (row - most) * stride * 2 : 0;
        };
#pragma unroll
        for (uint32_t x = 0; x < kPartsK; x++) ends(kplace[x], (x * kWaves + wave) * (64 / kPk), kPk, p.k_stride);
#pragma unroll
        for (uint32_t x = 0; x < kPartsR; x++) ends(rplace[x], (x * kWaves + wave) * (64 / kPr), kPr, p.r_stride);
#pragma unroll
        for (uint32_t x = 0; x < kPartsV; x++) ends(vplace[x], (x * kWaves + wave) * (64 / kPv), kPv, p.v_stride);
    };
    auto onward = [&]() {
        kat += (size_t)p.k_stride * (2 * kKeys);
        vat += (size_t)p.v_stride * (2 * kKeys);
        rat += (size_t)p.r_stride * (2 * kKeys);
        most -= kKeys;
        last();
    };
    struct Next {
        u32x4 k, v, r;
        uint32_t land;
    };
    auto rows_to = [&](uint32_t slot) { return Next{rows_buffer(kat), rows_buffer(vat), rows_buffer(rat), lds_address(stage) + slot * kStage}; };
    auto load = [&](const Next &next, uint32_t x) {
        if (x < kPartsK)
            rows_to_lds16(next.k, next.land + (x * kWaves + wave) * 1024, kplace[x]);
        else if (x < kPartsK + kPartsR)
            rows_to_lds16(next.r, next.land + kK + ((x - kPartsK) * kWaves + wave) * 1024, rplace[x - kPartsK]);
        else
            rows_to_lds16(next.v, next.land + kK + kR + ((x - kPartsK - kPartsR) * kWaves + wave) * 1024,
                          vplace[x - kPartsK - kPartsR]);
    };
    if (steps) {
        last();
        const Next next = rows_to(0);
#pragma unroll
        for (uint32_t x = 0; x < kLoads; x++) load(next, x);
    }
    // The operands' places by their piece; those of a step's buffer are a constant further.
    uint32_t kx[NOPE / 16], rx[ROPE / 16], vx[kD];
#pragma unroll
    for (uint32_t j = 0; j < NOPE / 16; j++) kx[j] = koff ^ 32 * j;
#pragma unroll
    for (uint32_t j = 0; j < ROPE / 16; j++) rx[j] = roff ^ 32 * j;
#pragma unroll
    for (uint32_t d = 0; d < kD; d++) vx[d] = voff ^ 64 * d;
    auto step = [&](uint32_t n, auto slot) {
        char *const at = stage + slot() * kStage;
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
        // (Behind the last step, its rows once more: nobody reads them.)
        if (n + 1 < steps) onward();
        const Next next = rows_to(1 - slot());
        const int32_t here = base + (int32_t)(n * kKeys), end = here + (int32_t)kKeys - 1;
        const bool apart = here < same_lo || end > same_hi;  // some key is one row's and not another's, or no key
        const bool work = here <= whi && end >= wlo;
        if (!apart && !work) {
#pragma unroll
            for (uint32_t x = 0; x < kLoads; x++) load(next, x);
            return;
        }

        // Half t of the step, 32 keys: its scores, register e key 32 t + 8 (e / 4) + 4 half + e % 4; its softmax; its
        // values. The first half's softmax runs beside the second's scores, the second's beside the first's values, in
        // pieces between the products (a wave's instructions issue in order). Operands are read kAhead products ahead.
        f32x16 s[2];
        bf16x8 ring[kAhead + 1];
        auto scores = [&](uint32_t t, auto beside) {
            auto read_k = [&](uint32_t j) {
                ring[j % (kAhead + 1)] = j < NOPE / 16 ? *(const bf16x8 *)(at + t * 32 * (2 * NOPE) + kx[j < NOPE / 16 ? j : 0])
                                                       : *(const bf16x8 *)(at + t * 32 * (2 * ROPE) + rx[j < NOPE / 16 ? 0 : j - NOPE / 16]);
            };
#pragma unroll
            for (int e = 0; e < 16; e++) s[t][e] = 0.0f;
#pragma unroll
            for (uint32_t j = 0; j < kAhead; j++) read_k(j);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (uint32_t j = 0; j < kQ; j++) {
                if (j + kAhead < kQ) read_k(j + kAhead);
                s[t] = mfma32(ring[j % (kAhead + 1)], qv[j], s[t]);
                beside(j);
                __builtin_amdgcn_sched_barrier(0);
            }
        };
        auto masked = [&](uint32_t t) {
            if (here >= wsame_lo && end <= wsame_hi) return;
            const int32_t upto = pos - here - 4 * (int32_t)half, since = from - here - 4 * (int32_t)half;
#pragma unroll
            for (int e = 0; e < 16; e++) {
                const int32_t x = 32 * t + 8 * (e / 4) + e % 4;
                s[t][e] = x <= upto && x >= since ? s[t][e] : -INFINITY;
            }
        };
        // The softmax in kSoft pieces. m moves only when a score passes it by 2^kSlack, so most steps leave the sum and O as
        // they are and no weight passes 2^kSlack.
        constexpr uint32_t kSoft = 13;
        float mx, mn, mo, sum, arg[2], weight[2];
        uint32_t w[2][8];
        auto soft = [&](uint32_t t, uint32_t i) {
            if (i < 2) {
                // (A NaN may come out: the row's sum is one as well.)
                float x = __builtin_elementwise_maximum(s[t][8 * i], s[t][8 * i + 1]);
#pragma unroll
                for (int e = 2; e < 8; e++) x = __builtin_elementwise_maximum(x, s[t][8 * i + e]);
                mx = i ? __builtin_elementwise_maximum(mx, x) : x;
                pinned(mx);
            } else if (i == 2) {
                mx = halves_max(mx) * sl;
                mn = mx > m + kSlack ? mx : m;
                mo = mn == -INFINITY ? 0.0f : mn;
                sum = 0.0f;
                pinned(mn);
                pinned(mo);
            } else {
                // Pair j's arguments, the pair's before it weights, and those of one more before into the sum: none waits for
                // another.
                const uint32_t j = i - 3;
                if (j >= 2) {
                    sum += weight[0] + weight[1];
                    w[t][j - 2] = bf16_pair(weight[0], weight[1]);
                    pinned(sum);
                    pinned(w[t][j - 2]);
                }
#pragma unroll
                for (uint32_t e = 0; e < 2; e++) {
                    if (j >= 1 && j < 9) {
                        weight[e] = __builtin_amdgcn_exp2f(arg[e]);
                        pinned(weight[e]);
                    }
                    if (j < 8) {
                        arg[e] = fmaf(s[t][2 * j + e], sl, -mo);
                        pinned(arg[e]);
                    }
                }
            }
        };
        // The pieces that belong to product i of n.
        auto pieces = [&](uint32_t t, uint32_t i, uint32_t n) {
#pragma unroll
            for (uint32_t x = 0; x < kSoft; x++)
                if (x * n / kSoft == i) soft(t, x);
        };
        auto raised = [&]() {
            if (__builtin_amdgcn_ballot_w64(mn > m) != 0) {
                // (Not 0, which would make a NaN of an infinite sum.)
                const float alpha = mn > m ? fmaxf(__builtin_amdgcn_exp2f(m - mn), 0x1p-126f) : 1.0f;
                l *= alpha;
                m = mn;
#pragma unroll
                for (uint32_t d = 0; d < kD; d++) o[d] *= alpha;
            }
            l += sum;
        };
        auto values = [&](uint32_t t, auto beside) {
            // Product i: keys 32 t + 16 (i / kD) .., d 32 (i % kD) .. . (Eight rows on the XOR is the same.)
            auto read_v = [&](uint32_t i) {
                const char *v = at + (32 * t + i / kD * 16) * (2 * VALUE) + vx[i % kD];
                const u32x2 lo4 = read_vt4(v), hi4 = read_vt4(v + 8 * (2 * VALUE));
                ring[i % (kAhead + 1)] = as_bf16x8(u32x4{lo4.x, lo4.y, hi4.x, hi4.y});
            };
#pragma unroll
            for (uint32_t i = 0; i < kAhead && i < 2 * kD; i++) read_v(i);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (uint32_t i = 0; i < 2 * kD; i++) {
                if (i + kAhead < 2 * kD) read_v(i + kAhead);
                const uint32_t x = 4 * (i / kD);
                o[i % kD] = mfma32(ring[i % (kAhead + 1)], as_bf16x8(u32x4{w[t][x], w[t][x + 1], w[t][x + 2], w[t][x + 3]}),
                                   o[i % kD]);
                beside(i);
                __builtin_amdgcn_sched_barrier(0);
            }
        };
        scores(0, [&](uint32_t i) {
#pragma unroll
            for (uint32_t x = 0; x < kLoads; x++)
                if (x * kQ / kLoads == i) load(next, x);
        });
        masked(0);
        scores(1, [&](uint32_t i) { pieces(0, i, kQ); });
        masked(1);
        raised();
        if (apart) {
            // A value that is not finite must reach the rows that see it alone, and the product's 0 times it would be
            // NaN: such values are looked for, added by themselves, and cleared, by all waves of the group alike.
            float odd = 0.0f;
#pragma unroll 4
            for (uint32_t g = again(lane); g < kV / 16; g += 64) {
                const u32x4 x = *(const u32x4 *)(at + kK + kR + g * 16);
#pragma unroll
                for (uint32_t e = 0; e < 4; e++) odd = odd_sum(x[e], odd);
            }
            if (__builtin_amdgcn_ballot_w64(odd != odd) != 0) {
#pragma unroll 1
                for (uint32_t k = 0; k < kKeys; k++) {
                    const uint32_t swap = value_swap<kPv>(k), g = again(half);
                    const uint32_t keep = here + (int32_t)k <= pos && here + (int32_t)k >= from ? 0xffffffffu : 0u;
                    const char *vk = at + kK + kR + k * (2 * VALUE) + 8 * g;
#pragma unroll
                    for (uint32_t d = 0; d < kD; d++)
#pragma unroll
                        for (uint32_t e = 0; e < 4; e++) {
                            u32x2 x = *(const u32x2 *)(vk + ((4 * d + e) ^ swap) * 16);
                            x = u32x2{x[0] & odd_mask(x[0]), x[1] & odd_mask(x[1])} & keep;
                            o[d][4 * e] += lo_bf16(x[0]);
                            o[d][4 * e + 1] += hi_bf16(x[0]);
                            o[d][4 * e + 2] += lo_bf16(x[1]);
                            o[d][4 * e + 3] += hi_bf16(x[1]);
                            __builtin_amdgcn_sched_barrier(0);
                        }
                }
                lds_barrier();
                for (uint32_t g = wave * 64 + again(lane); g < kV / 16; g += kThreads) {
                    u32x4 x = *(const u32x4 *)(at + kK + kR + g * 16);
#pragma unroll
                    for (uint32_t e = 0; e < 4; e++) x[e] &= ~odd_mask(x[e]);
                    *(u32x4 *)(at + kK + kR + g * 16) = x;
                }
                lds_barrier();
            }
        }
        values(0, [&](uint32_t i) { pieces(1, i, 2 * kD); });
        raised();
        values(1, [](uint32_t) {});
    };
    for (uint32_t n = 0; n < steps; n += 2) {
        step(n, [] { return 0u; });
        if (n + 1 < steps) step(n + 1, [] { return 1u; });
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    if (!there) return;
    // A row that sees no key is zero.
    const float sum = halves_sum(l), by = pos < 0 ? 0.0f : 1.0f / sum;
    uint16_t *to = p.out + ((size_t)row * p.heads + h) * VALUE + 4 * half;
#pragma unroll
    for (uint32_t d = 0; d < kD; d++)
#pragma unroll
        for (uint32_t e = 0; e < 4; e++)
            *(u32x2 *)(to + 32 * d + 8 * e) = u32x2{bf16_pair(o[d][4 * e] * by, o[d][4 * e + 1] * by),
                                                    bf16_pair(o[d][4 * e + 2] * by, o[d][4 * e + 3] * by)};
}

template <uint32_t NOPE, uint32_t ROPE, uint32_t VALUE>
int launch(const FlashParams &p, uint32_t groups, void *stream) {
    constexpr uint32_t kLds = kRing * kKeys * 2 * (NOPE + ROPE + VALUE);
    const auto kernel = flash_latent_kernel<NOPE, ROPE, VALUE>;
    static const hipError_t attr =
        hipFuncSetAttribute((const void *)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, kLds);
    if (attr != hipSuccess) return ts::hip_status(attr, "flash_latent: shared memory attribute");
    hipLaunchKernelGGL(kernel, dim3(groups), dim3(kThreads), kLds, (hipStream_t)stream, p);
    TS_CHECK_LAUNCH("flash_latent launch");
    return TS_OK;
}

}  // namespace

extern "C" int tessera_hip_flash_latent(const ts_flash_latent_args *a, void *stream) {
    TS_REQUIRE(a, "flash_latent: null args");
    const bool wide = a->nope == 128 && a->rope == 64 && a->value == 128;
    TS_REQUIRE(wide || (a->nope == 64 && a->rope == 32 && a->value == 64),
               "flash_latent: heads of %u + %u and %u values (128 + 64 and 128, or 64 + 32 and 64)", a->nope, a->rope, a->value);
    TS_REQUIRE(a->heads >= 1 && a->heads <= 1024, "flash_latent: %u heads", a->heads);
    TS_REQUIRE(a->rows <= 1u << 28 && a->key_rows <= 1u << 28, "flash_latent: %u rows, %u keys", a->rows, a->key_rows);
    TS_REQUIRE(a->seqs <= 1u << 20 && (a->first || a->seqs <= 1), "flash_latent: %u sequences without their bounds", a->seqs);
    TS_REQUIRE(a->first || !a->key_first, "flash_latent: bounds of the keys without those of the rows");
    TS_REQUIRE((a->q_stride == 0 || a->q_stride >= a->heads * (a->nope + a->rope)) && a->q_stride % 8 == 0,
               "flash_latent: q rows %u apart must hold %u heads and be whole 16-byte pieces", a->q_stride, a->heads);
    TS_REQUIRE(a->k_stride % 8 == 0 && a->k_head % 8 == 0 && a->v_stride % 8 == 0 && a->v_head % 8 == 0 && a->r_stride % 8 == 0,
               "flash_latent: rows and heads of k, v and r must be whole 16-byte pieces apart");
    if (a->rows == 0 || a->seqs == 0) return TS_OK;
    TS_REQUIRE(a->q && a->out && (a->key_rows == 0 || (a->k && a->v && a->r)), "flash_latent: null pointer");
    TS_REQUIRE(ts::aligned(a->q, 16) && ts::aligned(a->k, 16) && ts::aligned(a->v, 16) && ts::aligned(a->r, 16) &&
                   ts::aligned(a->out, 16),
               "flash_latent: q, k, v, r and out must be 16-byte aligned");
    // (64 keys within a 32-bit offset.)
    TS_REQUIRE(a->k_stride <= 1u << 25 && a->v_stride <= 1u << 25 && a->r_stride <= 1u << 25,
               "flash_latent: keys %u, %u and %u elements apart", a->k_stride, a->v_stride, a->r_stride);
    FlashParams p;
    p.q = (const uint16_t *)a->q; p.k = (const uint16_t *)a->k; p.v = (const uint16_t *)a->v; p.r = (const uint16_t *)a->r;
    p.out = (uint16_t *)a->out; p.first = a->first; p.key_first = a->key_first;
    p.rows = a->rows; p.key_rows = a->key_rows; p.seqs = a->first ? a->seqs : 1; p.heads = a->heads;
    p.q_stride = a->q_stride; p.k_stride = a->k_stride; p.k_head = a->k_head; p.v_stride = a->v_stride;
    p.v_head = a->v_head; p.r_stride = a->r_stride; p.back = a->back; p.scale = a->scale;
    // Whole tiles and a begun one a sequence at most.
    p.tiles = a->rows / kRows + (p.seqs < a->rows ? p.seqs : a->rows);
    const uint64_t groups = (uint64_t)p.tiles * a->heads;
    TS_REQUIRE(groups < (1ull << 32) / kThreads, "flash_latent: %u rows in one launch", a->rows);
    const uint64_t bounds = a->first ? ((uint64_t)a->seqs + 1) * 4 : 0;
    const int over = ts::outputs_apart("flash_latent", {{"out", a->out, (uint64_t)a->rows * a->heads * a->value * 2}},
                                       {{"q", a->q, 2ull * a->heads * (a->nope + a->rope), a->rows, 2ull * a->q_stride},
                                        {"k", a->k, 2ull * a->nope, a->key_rows, 2ull * a->k_stride, a->heads, 2ull * a->k_head},
                                        {"v", a->v, 2ull * a->value, a->key_rows, 2ull * a->v_stride, a->heads, 2ull * a->v_head},
                                        {"r", a->r, 2ull * a->rope, a->key_rows, 2ull * a->r_stride},
                                        {"first", a->first, bounds},
                                        {"key_first", a->key_first, bounds}});
    if (over) return over;
    return wide ? launch<128, 64, 128>(p, (uint32_t)groups, stream) : launch<64, 32, 64>(p, (uint32_t)groups, stream);
}
