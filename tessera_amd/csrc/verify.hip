// Verification of drafted tokens (speculative decoding) against the target's distribution, from given
// uniform numbers: draft t of a sequence is taken while u_t q_t(draft) < p_t(draft), and the token after
// the taken ones is drawn from max(p - q, 0) (after a refusal) or p by inverting the running sum in index
// order. (Rejection sampling keeps the target's distribution: Leviathan et al., Chen et al., 2023.) No
// counterpart in the reference, which decodes greedily, one token a step.
//
//   p_i = e_i / Z,  e_i = exp((x_i - M) / temperature),  M = max x,  Z = sum of e
//
// Two launches:
//   1. rows: every row in chunks of a few pieces of 2048, a group each: the chunk's maximum, its first
//      index, and its sum of e against that maximum;
//   2. draw: each group works out its sequence's verdict from the rows' chunks (a few hundred values, 3 us),
//      then weighs its share of the row to draw from, a wave a run of 256 indices at a time. The
//      group that is last of a sequence to do so finds the run where the running sum passes u times the
//      whole, and one wave the index in it.
// Code that runs once costs its fetch, so nothing here is unrolled or inlined twice that need not be.
// Sums are in f64 and exponentials good to 33 bits (the vector unit's f64 rate is f32's here): the draw compares u
// with running sums. Over rows of 151936 logits the exponentials' error moves their borders by up to 6e-12 of the
// whole and, all borders together, decides about one draw in two million; f32 exponentials would move them by up to
// 2e-8 and decide one draw in a thousand.
// 32 sequences of up to 4 drafts with the drafter's probabilities, 81 rows of 151936 f32 logits: rows 19 us, draw 16.
// The rows' 49 MB are 10 us at a large copy's rate; their 29 vector instructions a logit keep the vector unit busy for
// 79% of the cycles in which a CU has waves, and a CU has them for some 60% of the kernel's time. The draw reads the
// drawn row again and the drafter's (39 MB, 8 us), after the verdict (3 us) and before the last group's search; the
// vector unit is busy for half of it. One greedy sequence of 4 drafts: 4 and 3 us.
#include <algorithm>

#include "common.h"

namespace {

constexpr uint32_t kEach = 8, kWaves = 4, kPiece = 64 * kWaves * kEach;  // the rows' kernel: 2048 indices a piece
constexpr uint32_t kMostPieces = 8;                // pieces a chunk at most
constexpr uint32_t kRun = 256, kDrawWaves = 16;    // the draw's: indices a run, waves a group

struct Chunk {  // of one row
    double sum;
    float most;
    uint32_t at;  // first index of `most`, or width where the chunk holds none
};

struct Verdict {  // of one sequence
    double whole;  // Z of the row to draw from
    float most;    // its M
    uint32_t row;  // in logits
    uint32_t accepted;
    uint32_t refused;  // 1: a draft was refused
    uint32_t pick;     // greedy: the token
};

struct VerifyParams {
    const void *logits;
    const uint32_t *drafts, *counts, *first;
    const float *uniforms, *probs, *temperatures;
    uint32_t *tokens, *accepted, *status;
    Chunk *chunks;      // [seqs][most + 1][parts]
    double *sums;       // [seqs][runs]: weights of runs of 256 indices
    uint32_t *done;     // [seqs]: groups of the second kernel that have left their sum
    uint32_t seqs, most, rows, width, stride;
    uint32_t pieces, parts;  // of the rows' kernel: pieces a chunk, chunks a row
    uint32_t runs, groups;   // of the draw's: runs a row, groups a sequence
    float temperature;
};

// A constant in scalar registers: as an addend it would otherwise be copied to vector ones each time.
TS_DEV double scalar(double c) {
    asm("" : "+s"(c));
    return c;
}

// 2^t for -1200 < t <= 0: t = n + f, |f| <= 1/2, n out of the low bits of t + 1.5 * 2^52, and 2^f = 1 + f g(f)
// with g, of degree 6, through (2^f - 1) / f at the Chebyshev points: 1.1e-10 off at most, 2^0 exact. (f32
// would be 6e-8 off. The series up to the 10th power, 3e-13, cost an eighth of both kernels.)
TS_DEV double exp2_neg(double t) {
    const double k = t + scalar(6755399441055744.0), f = t - (k - scalar(6755399441055744.0));
    double r = __builtin_fma(f, scalar(1.5297324125640444e-05), scalar(0.00015461444699635));
    r = __builtin_fma(r, f, scalar(0.0013333502384966778));
    r = __builtin_fma(r, f, scalar(0.009618056678521874));
    r = __builtin_fma(r, f, scalar(0.05550410883910522));
    r = __builtin_fma(r, f, scalar(0.24022650922288763));
    r = __builtin_fma(r, f, scalar(0.6931471805599453));
    r = __builtin_fma(r, f, 1.0);
    return __builtin_amdgcn_ldexp(r, (int)(uint32_t)__builtin_bit_cast(uint64_t, k));  // (0 below 2^-1074)
}

// e of logits side by side, `by` = log2(e) / temperature: 1 at the maximum (+inf too), 0 for NaN and -inf
// (whose t is -inf or NaN; fmax takes its other operand).
template <int N>
TS_DEV void weights(float (&x)[N], float most, double by, double (&w)[N]) {
    if (most == __builtin_inff()) {
        most = 0.0f;
#pragma unroll
        for (int j = 0; j < N; j++) x[j] = x[j] == __builtin_inff() ? 0.0f : -__builtin_inff();
    }
#pragma unroll
    for (int j = 0; j < N; j++) w[j] = exp2_neg(fmax(((double)x[j] - (double)most) * by, -1100.0));
}
TS_DEV double per_unit(float temperature) { return 1.4426950408889634 / (double)temperature; }

template <bool BF16>
TS_DEV float logit(const VerifyParams &p, uint32_t row, uint32_t i) {
    const size_t at = (size_t)row * p.stride + i;
    return BF16 ? bf16_float(((const uint16_t *)p.logits)[at]) : ((const float *)p.logits)[at];
}

// Four consecutive logits of a row (or probabilities); past the row, its last. VEC: they are one load, and the width
// a multiple of four. No branch and no use of a value here: either would make a loop that asks for the next ones
// before it uses these wait for both (32 x 4 drafts 36 us, 35 so).
template <bool BF16, bool VEC>
TS_DEV void load4(const void *row, uint32_t i, uint32_t width, uint32_t (&x)[4]) {
    if (VEC) {
        const uint32_t at = min(i, width - 4);
        if (BF16) {
            const u32x2 w = *(const u32x2 *)((const uint16_t *)row + at);
            x[0] = w.x;
            x[1] = w.y;
        } else {
            const u32x4 w = *(const u32x4 *)((const uint32_t *)row + at);
#pragma unroll
            for (int e = 0; e < 4; e++) x[e] = w[e];
        }
    } else {
#pragma unroll
        for (uint32_t e = 0; e < 4; e++) {
            const uint32_t at = min(i + e, width - 1);
            x[e] = BF16 ? ((const uint16_t *)row)[at] : ((const uint32_t *)row)[at];
        }
    }
}
// What load4 has brought, as f32: indices past the width as `past`, where the wave has any (`edge`).
template <bool BF16, bool VEC>
TS_DEV void values4(const uint32_t (&x)[4], uint32_t i, uint32_t width, bool edge, float past, float *v) {
#pragma unroll
    for (uint32_t e = 0; e < 4; e++)
        v[e] = !BF16 ? __uint_as_float(x[e]) : !VEC ? lo_bf16(x[e]) : e % 2 ? hi_bf16(x[e / 2]) : lo_bf16(x[e / 2]);
    if (edge) {
#pragma unroll
        for (uint32_t e = 0; e < 4; e++) v[e] = i + e < width ? v[e] : past;
    }
}
template <bool BF16>
TS_DEV const void *row_of(const VerifyParams &p, uint32_t row) {
    return (const char *)p.logits + (size_t)row * p.stride * (BF16 ? 2 : 4);
}

// A sequence's drafts, first row of logits and temperature (<= 0: greedy); false where it is out of range.
struct Seq {
    uint32_t count, first;
    float temperature;
    bool good, greedy;
};
TS_DEV Seq seq_of(const VerifyParams &p, uint32_t s) {
    Seq q;
    q.count = p.counts ? p.counts[s] : p.most;
    q.first = p.first ? p.first[s] : s * (p.most + 1);
    q.good = q.count <= p.most && (uint64_t)q.first + q.count < p.rows;
    q.temperature = p.temperatures ? p.temperatures[s] : p.temperature;
    q.greedy = !p.uniforms || !(q.temperature > 0.0f);
    return q;
}

// The sum over the wave, in every lane: within rows of 16 lanes, then by the permlane swaps across them
// (through LDS, two exchanges a step of a double, the six steps take five times as long).
TS_DEV double wave_total(double v) {
    v = row16_total(v);
    uint64_t b = __builtin_bit_cast(uint64_t, v);
    const auto l32 = __builtin_amdgcn_permlane32_swap((uint32_t)b, (uint32_t)b, false, false);
    const auto h32 = __builtin_amdgcn_permlane32_swap((uint32_t)(b >> 32), (uint32_t)(b >> 32), false, false);
    v = __builtin_bit_cast(double, (uint64_t)h32[0] << 32 | l32[0]) + __builtin_bit_cast(double, (uint64_t)h32[1] << 32 | l32[1]);
    b = __builtin_bit_cast(uint64_t, v);
    const auto l16 = __builtin_amdgcn_permlane16_swap((uint32_t)b, (uint32_t)b, false, false);
    const auto h16 = __builtin_amdgcn_permlane16_swap((uint32_t)(b >> 32), (uint32_t)(b >> 32), false, false);
    return __builtin_bit_cast(double, (uint64_t)h16[0] << 32 | l16[0]) + __builtin_bit_cast(double, (uint64_t)h16[1] << 32 | l16[1]);
}

// A chunk's pieces, the next one's logits asked for before this one's are weighed. Each lane keeps a
// maximum and a sum of its own; they meet once, at the end. A lane has two fours of consecutive indices
// of a piece, 256 apart.
template <bool BF16, bool VEC>
__global__ __launch_bounds__(64 * kWaves) void verify_rows_kernel(VerifyParams p) {
    __shared__ Chunk waves[kWaves];
    const uint32_t part = blockIdx.x % p.parts, sr = blockIdx.x / p.parts;
    const uint32_t s = sr / (p.most + 1), t = sr % (p.most + 1), wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const Seq q = seq_of(p, s);
    if (!q.good || t > q.count) return;
    if (p.done && part == 0 && t == 0 && threadIdx.x == 0) p.done[s] = 0;
    const double by = per_unit(q.temperature);
    const uint32_t first = part * p.pieces, end = min(first + p.pieces, (p.width + kPiece - 1) / kPiece);
    const uint32_t mine = wave * (kPiece / kWaves) + lane * 4;
    const void *row = row_of<BF16>(p, q.first + t);
    float most = -__builtin_inff();
    uint32_t at = p.width, raw[2][4];
    double sum = 0.0;
    auto load = [&](uint32_t piece, uint32_t (&to)[2][4]) {
        load4<BF16, VEC>(row, piece * kPiece + mine, p.width, to[0]);
        load4<BF16, VEC>(row, piece * kPiece + mine + 256, p.width, to[1]);
    };
    load(first, raw);
    for (uint32_t piece = first; piece < end; piece++) {
        uint32_t next[2][4];
        load(min(piece + 1, end - 1), next);  // (the last piece's again, not used)
        float x[kEach];
        const bool edge = (piece + 1) * kPiece > p.width;
#pragma unroll
        for (uint32_t h = 0; h < 2; h++)
            values4<BF16, VEC>(raw[h], piece * kPiece + mine + 256 * h, p.width, edge, -__builtin_inff(), x + 4 * h);
        float top = x[0];
#pragma unroll
        for (uint32_t j = 1; j < kEach; j++) top = fmaxf(top, x[j]);  // (NaN: the other operand)
        float was[1] = {most};
        const bool raise = top > most;
        most = raise ? top : most;
        if (q.greedy) {
            if (raise) {
#pragma unroll
                for (int j = kEach - 1; j >= 0; j--)  // the first: the lane's places ascend
                    if (x[j] == most) at = piece * kPiece + mine + (j / 4) * 256 + j % 4;
            }
        } else {
            double w[kEach];
            if (__builtin_amdgcn_ballot_w64(raise) != 0) {
                double f[1];
                weights(was, most, by, f);
                sum *= f[0];
            }
            weights(x, most, by, w);
#pragma unroll
            for (uint32_t j = 0; j < kEach; j++) sum += w[j];
        }
#pragma unroll
        for (uint32_t j = 0; j < kEach; j++) raw[j / 4][j % 4] = next[j / 4][j % 4];
    }
    float own[1] = {most};
    double scale[1];
    most = wave_max(most);
    at = own[0] == most ? at : p.width;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) at = min(at, (uint32_t)__shfl_xor((int)at, o, 64));
    if (!q.greedy) {
        weights(own, most, by, scale);
        sum = wave_total(sum * scale[0]);
    }
    if (lane == 0) waves[wave] = Chunk{sum, most, at};
    __syncthreads();
    if (threadIdx.x == 0) {
        Chunk c = waves[0];
        for (uint32_t w = 1; w < kWaves; w++)
            if (waves[w].most > c.most || (waves[w].most == c.most && waves[w].at < c.at)) {
                c.most = waves[w].most;
                c.at = waves[w].at;
            }
        if (!q.greedy) {
            float m[kWaves];
            double f[kWaves];
            c.sum = 0.0;
            for (uint32_t w = 0; w < kWaves; w++) m[w] = waves[w].most;
            weights(m, c.most, by, f);
            for (uint32_t w = 0; w < kWaves; w++) c.sum += waves[w].sum * f[w];
        }
        p.chunks[(size_t)sr * p.parts + part] = c;
    }
}

constexpr uint32_t kMostDrafts = 64;

// The sequence's verdict, by the whole group, 16 lanes a row; in every thread. Reads the rows' chunks.
template <bool BF16>
TS_DEV Verdict decide(const VerifyParams &p, uint32_t s, const Seq &q) {
    __shared__ Verdict rows[kMostDrafts + 1];
    __shared__ uint32_t taken[kMostDrafts + 1];
    const uint32_t l16 = threadIdx.x & 15;
    const double by = per_unit(q.temperature);
    for (uint32_t t = threadIdx.x >> 4; t <= q.count; t += blockDim.x / 16) {
        const size_t sr = (size_t)s * (p.most + 1) + t;
        // What the test of the draft needs is asked for before the row's chunks.
        const uint32_t draft = t < q.count ? p.drafts[(size_t)s * p.most + t] : p.width;
        float x = 0.0f, chance = 1.0f, u = 0.0f;
        if (!q.greedy && draft < p.width) {
            x = logit<BF16>(p, q.first + t, draft);
            u = p.uniforms[sr];
            if (p.probs) chance = p.probs[((size_t)s * p.most + t) * p.width + draft];
        }
        const Chunk *c = p.chunks + sr * p.parts;
        float most = -__builtin_inff();
        uint32_t at = p.width;
        double z = 0.0;
        for (uint32_t j0 = l16; j0 < p.parts; j0 += 64) {
            Chunk four[4];
#pragma unroll
            for (uint32_t j = 0; j < 4; j++) four[j] = c[min(j0 + 16 * j, p.parts - 1)];  // past the end: not used
            float m[5];
            double f[5];
            m[4] = most;
#pragma unroll
            for (uint32_t j = 0; j < 4; j++) {
                m[j] = j0 + 16 * j < p.parts ? four[j].most : -__builtin_inff();
                if (m[j] > most) { most = m[j]; at = four[j].at; }
            }
            if (q.greedy) continue;
            weights(m, most, by, f);
            z *= f[4];
#pragma unroll
            for (uint32_t j = 0; j < 4; j++) z += f[j] > 0.0 ? four[j].sum * f[j] : 0.0;
        }
        float whole = most;
#pragma unroll
        for (int o = 1; o < 16; o <<= 1) {
            const float w = __shfl_xor(whole, o, 64);
            const uint32_t b = __shfl_xor(at, o, 64);
            if (w > whole || (w == whole && b < at)) { whole = w; at = b; }
        }
        double e = 0.0;
        if (!q.greedy) {
            float m[2] = {most, x};
            double f[2];
            weights(m, whole, by, f);
            z *= f[0];
            e = f[1];
            z = row16_total(z);
        }
        if (l16 == 0) {
            chance = chance > 0.0f ? chance : 0.0f;
            taken[t] = draft < p.width && (q.greedy ? draft == at : (double)u * (double)chance * z < e);
            rows[t] = Verdict{z, whole, q.first + t, t, t < q.count, at};
        }
    }
    __syncthreads();
    uint32_t n = 0;
    while (n < q.count && taken[n]) n++;
    return rows[n];
}

// The sequence's tokens: the accepted drafts, the pick, `width` in the rest.
TS_DEV void answer(const VerifyParams &p, uint32_t s, bool good, uint32_t accepted, uint32_t pick) {
    for (uint32_t t = threadIdx.x; t <= p.most; t += blockDim.x)
        p.tokens[(size_t)s * (p.most + 1) + t] = !good           ? p.width
                                                 : t < accepted  ? p.drafts[(size_t)s * p.most + t]
                                                 : t == accepted ? pick
                                                                 : p.width;
    if (threadIdx.x == 0) p.accepted[s] = good ? accepted : 0;
    if (threadIdx.x == 0 && !good && p.status) atomicOr(p.status, TS_STATUS_POSITION);
}

// All greedy: the verdict is the answer.
template <bool BF16>
__global__ __launch_bounds__(256) void verify_greedy_kernel(VerifyParams p) {
    const uint32_t s = blockIdx.x;
    const Seq q = seq_of(p, s);
    if (!q.good) {
        answer(p, s, false, 0, 0);
        return;
    }
    const Verdict v = decide<BF16>(p, s, q);
    answer(p, s, true, v.accepted, v.pick);
}

// The draw. Runs of 256 indices, four consecutive ones a lane.
template <bool BF16, bool VEC>
__global__ __launch_bounds__(64 * kDrawWaves) void verify_draw_kernel(VerifyParams p) {
    __shared__ uint32_t before, found[2];
    __shared__ double ends[kDrawWaves], starts[2];
    const uint32_t part = blockIdx.x % p.groups, s = blockIdx.x / p.groups;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const Seq q = seq_of(p, s);
    if (!q.good) {
        if (part == 0) answer(p, s, false, 0, 0);
        return;
    }
    const Verdict v = decide<BF16>(p, s, q);
    if (q.greedy) {
        if (part == 0) answer(p, s, true, v.accepted, v.pick);
        return;
    }
    const double by = per_unit(q.temperature);
    const uint32_t draft = v.refused ? p.drafts[(size_t)s * p.most + v.accepted] : 0;
    const float *probs = p.probs ? p.probs + ((size_t)s * p.most + v.accepted) * p.width : nullptr;
    const double u = (double)p.uniforms[(size_t)s * (p.most + 1) + p.most];
    double *sums = p.sums + (size_t)s * p.runs;
    // The weights are max(e - q Z, 0) after a refusal, e otherwise; one pass over the runs for all
    // groups together, and should the former all be zero, one for e by the last group alone.
    bool residual = v.refused;
    uint32_t r0 = part * kDrawWaves + wave, apart = p.groups * kDrawWaves, run = 0xffffffffu;
    double w[4], target = 0.0, start = 0.0;
    bool alone = false, searching = false;
    const void *row = row_of<BF16>(p, v.row);
    // (Without probabilities the logits are read in their place, from the caches, and not used.)
    const bool rest = v.refused && probs;
    const void *beside = rest ? (const void *)probs : row;
    auto load = [&](uint32_t r, uint32_t (&x)[4], uint32_t (&c)[4]) {
        load4<BF16, VEC>(row, r * kRun + lane * 4, p.width, x);
        if (BF16 && !rest)
            load4<true, VEC>(beside, r * kRun + lane * 4, p.width, c);
        else
            load4<false, VEC>(beside, r * kRun + lane * 4, p.width, c);
    };
    for (;;) {
        uint32_t raw[4], rawc[4];
        uint32_t r = r0;
        if (r < p.runs) load(r, raw, rawc);
        while (r < p.runs) {
            const uint32_t next = searching ? p.runs : r + apart;
            uint32_t nx[4], nc[4];
            load(min(next, p.runs - 1), nx, nc);  // (past the last: not used)
            float x[4], c[4];
            const uint32_t i = r * kRun + lane * 4;
            const bool edge = (r + 1) * kRun > p.width;
            values4<BF16, VEC>(raw, i, p.width, edge, -__builtin_inff(), x);
            values4<false, VEC>(rawc, i, p.width, edge, 0.0f, c);
            if (!rest || !residual) {
#pragma unroll
                for (uint32_t e = 0; e < 4; e++) c[e] = 0.0f;
            }
            weights(x, v.most, by, w);
#pragma unroll
            for (uint32_t e = 0; e < 4; e++) {
                if (residual) {
                    if (!probs && r * kRun + lane * 4 + e == draft) w[e] = 0.0;
                    w[e] -= (c[e] > 0.0f ? (double)c[e] : 0.0) * v.whole;
                    w[e] = w[e] > 0.0 ? w[e] : 0.0;
                }
            }
            if (!searching) {
                const double sum = wave_total((w[0] + w[1]) + (w[2] + w[3]));
                // Past the XCD's own L2, where the sequence's last group reads it. (Its loads pass their L2 too. So
                // stores that have arrived, the wait below, before the group's add to `done`, are what whoever sees
                // that add reads: no release of the whole L2, which would cost microseconds, is needed.)
                if (lane == 0) __hip_atomic_store(sums + r, sum, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            }
            r = next;
#pragma unroll
            for (uint32_t e = 0; e < 4; e++) {
                raw[e] = nx[e];
                rawc[e] = nc[e];
            }
        }
        if (searching) break;  // wave 0 has the weights of the run found
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // the sums have arrived
        __syncthreads();
        if (!alone) {
            if (threadIdx.x == 0) before = __hip_atomic_fetch_add(p.done + s, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            __syncthreads();
            if (before + 1 != p.groups) return;
            alone = true;
        }
        // The last group: running sums over the runs, a thread a block of consecutive ones.
        const uint32_t each = (p.runs + 64 * kDrawWaves - 1) / (64 * kDrawWaves);
        const uint32_t j0 = threadIdx.x * each, j1 = min(j0 + each, p.runs);
        double mine = 0.0;
        for (uint32_t j = j0; j < j1; j++) mine += __hip_atomic_load(sums + j, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        double upto = mine;
#pragma unroll 1
        for (int o = 1; o < 64; o <<= 1) {
            const double up = __shfl_up(upto, o, 64);
            if ((int)lane >= o) upto += up;
        }
        if (lane == 63) ends[wave] = upto;
        if (threadIdx.x < 2) found[threadIdx.x] = threadIdx.x ? 0u : 0xffffffffu;
        __syncthreads();
        double whole = 0.0;
#pragma unroll 1
        for (uint32_t j = 0; j < kDrawWaves; j++) {
            if (j < wave) upto += ends[j];
            whole += ends[j];
        }
        if (residual && !(whole > 0.0)) {  // (uniform over the group)
            residual = false;
            r0 = wave;
            apart = kDrawWaves;
            continue;
        }
        // The first run whose running sum passes the target; without one (rounding, or u not below 1) the
        // last that weighs anything.
        target = u * whole;
        uint32_t over = 0xffffffffu, weighs = 0xffffffffu;
        double over_start = 0.0, weighs_start = 0.0, at = upto - mine;
        for (uint32_t j = j0; j < j1; j++) {
            const double c = __hip_atomic_load(sums + j, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            if (c > 0.0) {
                weighs = j;
                weighs_start = at;
                if (over == 0xffffffffu && at + c > target) {
                    over = j;
                    over_start = at;
                }
            }
            at += c;
        }
        // (One lane a wave: the first with one over, the last that weighs.)
        const uint64_t overs = __builtin_amdgcn_ballot_w64(over != 0xffffffffu);
        const uint64_t all = __builtin_amdgcn_ballot_w64(weighs != 0xffffffffu);
        if (overs && lane == __builtin_ctzll(overs)) atomicMin(&found[0], over);
        if (all && lane == 63 - __builtin_clzll(all)) atomicMax(&found[1], weighs);
        __syncthreads();
        run = found[0] != 0xffffffffu ? found[0] : found[1];
        if (run == over) starts[0] = over_start;
        if (run == weighs) starts[1] = weighs_start;
        __syncthreads();
        start = found[0] != 0xffffffffu ? starts[0] : starts[1];
        if (wave != 0) return;
        searching = true;
        r0 = run;
    }
    // The run's index, by one wave: the first whose running sum passes the target, or the last that
    // weighs anything; `width` where nothing does.
    double upto = (w[0] + w[1]) + (w[2] + w[3]);
#pragma unroll 1
    for (int o = 1; o < 64; o <<= 1) {
        const double up = __shfl_up(upto, o, 64);
        if ((int)lane >= o) upto += up;
    }
    const double left = __shfl_up(upto, 1, 64);
    double at = start + (lane ? left : 0.0);
    uint32_t over = 0xffffffffu, last = 0xffffffffu;
#pragma unroll
    for (uint32_t e = 0; e < 4; e++) {
        at += w[e];
        const uint32_t i = run * kRun + lane * 4 + e;
        if (w[e] > 0.0) {
            last = i;
            if (over == 0xffffffffu && at > target) over = i;
        }
    }
    const uint64_t overs = __builtin_amdgcn_ballot_w64(over != 0xffffffffu);
    const uint64_t lasts = __builtin_amdgcn_ballot_w64(last != 0xffffffffu);
    const uint32_t pick = overs   ? __builtin_amdgcn_readlane(over, __builtin_ctzll(overs))
                          : lasts ? __builtin_amdgcn_readlane(last, 63 - __builtin_clzll(lasts))
                                  : p.width;
    for (uint32_t t = lane; t <= p.most; t += 64) {
        const uint32_t kept = t < v.accepted ? p.drafts[(size_t)s * p.most + t] : p.width;
        p.tokens[(size_t)s * (p.most + 1) + t] = t == v.accepted ? pick : kept;
    }
    if (lane == 0) p.accepted[s] = v.accepted;
}

// How the rows are cut.
struct Cut {
    uint32_t pieces, parts, runs, groups;
};
Cut cut(const ts_verify_args *a) {
    Cut c;
    // The rows' kernel: pieces a chunk so that the groups fill the chip once (8 of 4 waves a CU), a
    // chunk's later pieces loading under the work on its earlier ones.
    const uint32_t all = (a->width + kPiece - 1) / kPiece;
    const uint64_t rows = (uint64_t)a->seqs * (a->most + 1);
    c.pieces = (uint32_t)std::min<uint64_t>(kMostPieces, std::max<uint64_t>(1, all * rows / 2048));
    c.parts = (all + c.pieces - 1) / c.pieces;
    // The draw: about a group a CU (16 waves, four a SIMD), a run a wave at least.
    c.runs = (a->width + kRun - 1) / kRun;
    c.groups = std::min((c.runs + kDrawWaves - 1) / kDrawWaves, std::max(1u, 256 / std::max(1u, a->seqs)));
    return c;
}

struct Sizes {
    size_t chunks, sums, done;  // bytes
    size_t whole() const { return chunks + sums + done; }
};
Sizes sizes(const ts_verify_args *a) {
    const Cut c = cut(a);
    Sizes z;
    z.chunks = (size_t)a->seqs * (a->most + 1) * c.parts * sizeof(Chunk);
    z.sums = a->uniforms ? (size_t)a->seqs * c.runs * sizeof(double) : 0;
    z.done = a->uniforms ? (size_t)a->seqs * sizeof(uint32_t) : 0;
    return z;
}

int check(const ts_verify_args *a) {
    TS_REQUIRE(a, "verify: null args");
    TS_REQUIRE(a->seqs == 0 || ((a->logits || a->rows == 0) && a->tokens && a->accepted && (a->drafts || a->most == 0)),
               "verify: null pointer");
    TS_REQUIRE(a->most <= kMostDrafts, "verify: %u drafts a sequence (at most %u)", a->most, kMostDrafts);
    TS_REQUIRE(a->logits_dtype == TS_F32 || a->logits_dtype == TS_BF16, "verify: logits f32 or bf16 supported");
    TS_REQUIRE(a->width >= 1 && a->width <= 1u << 28 && a->stride >= a->width, "verify: rows of %u logits, %u apart",
               a->width, a->stride);
    TS_REQUIRE(a->first || (uint64_t)a->seqs * (a->most + 1) <= a->rows, "verify: %u sequences of %u rows, %u rows given",
               a->seqs, a->most + 1, a->rows);
    TS_REQUIRE((uint64_t)a->seqs * (a->most + 1) * ((a->width + kPiece - 1) / kPiece) <= 0x7fffffffull,
               "verify: %u sequences in one launch", a->seqs);
    const uint32_t one = a->logits_dtype == TS_BF16 ? 2 : 4;
    TS_REQUIRE(ts::aligned(a->logits, one), "verify: logits must be %u-byte aligned", one);
    return TS_OK;
}

template <bool BF16>
int launch(const VerifyParams &p, bool vec_x, bool vec_q, hipStream_t stream) {
    const auto rows = vec_x ? verify_rows_kernel<BF16, true> : verify_rows_kernel<BF16, false>;
    const auto draw = vec_x && vec_q ? verify_draw_kernel<BF16, true> : verify_draw_kernel<BF16, false>;
    hipLaunchKernelGGL(rows, dim3(p.seqs * (p.most + 1) * p.parts), dim3(64 * kWaves), 0, stream, p);
    TS_CHECK_LAUNCH("verify rows launch");
    if (p.uniforms)
        hipLaunchKernelGGL(draw, dim3(p.seqs * p.groups), dim3(64 * kDrawWaves), 0, stream, p);
    else
        hipLaunchKernelGGL(verify_greedy_kernel<BF16>, dim3(p.seqs), dim3(256), 0, stream, p);
    TS_CHECK_LAUNCH("verify draw launch");
    return TS_OK;
}

}  // namespace

extern "C" size_t tessera_hip_verify_workspace(const ts_verify_args *a) { return a && a->width ? sizes(a).whole() : 0; }

extern "C" int tessera_hip_verify(const ts_verify_args *a, void *stream) {
    int rc = check(a);
    if (rc) return rc;
    if (a->seqs == 0) return TS_OK;
    const Sizes z = sizes(a);
    if (!a->workspace || a->workspace_bytes < z.whole() || !ts::aligned(a->workspace, 16))
        return ts::fail(TS_ERR_WORKSPACE, "verify: workspace of %zu bytes, 16-byte aligned, needed", z.whole());
    VerifyParams p;
    p.logits = a->logits; p.drafts = a->drafts; p.counts = a->counts; p.first = a->first;
    p.uniforms = a->uniforms; p.probs = a->draft_probs; p.temperatures = a->temperatures;
    p.tokens = a->tokens; p.accepted = a->accepted; p.status = a->status;
    char *w = (char *)a->workspace;
    p.chunks = (Chunk *)w;
    p.sums = (double *)(w + z.chunks);
    p.done = a->uniforms ? (uint32_t *)(w + z.chunks + z.sums) : nullptr;
    p.seqs = a->seqs; p.most = a->most; p.rows = a->rows; p.width = a->width; p.stride = a->stride;
    const Cut c = cut(a);
    p.pieces = c.pieces; p.parts = c.parts; p.runs = c.runs; p.groups = c.groups;
    p.temperature = a->temperature;
    // Four consecutive logits, and probabilities, are one aligned load.
    const bool bf16 = a->logits_dtype == TS_BF16;
    const bool vec_x = a->width % 4 == 0 && a->stride % 4 == 0 && ts::aligned(a->logits, bf16 ? 8 : 16);
    const bool vec_q = ts::aligned(a->draft_probs, 16);
    return bf16 ? launch<true>(p, vec_x, vec_q, (hipStream_t)stream) : launch<false>(p, vec_x, vec_q, (hipStream_t)stream);
}
