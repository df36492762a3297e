// Verification of drafted tokens (speculative decoding) against the target's distribution, from given
// uniform numbers: draft t of a sequence is taken while u_t q_t(draft) < p_t(draft), and the token after
// the taken ones is drawn from max(p - q, 0) (after a refusal) or p by inverting the running sum in index
// order. (Rejection sampling keeps the target's distribution: Leviathan et al., Chen et al., 2023.) No
// counterpart in the reference, which decodes greedily, one token a step.
//
//   p_i = e_i / Z,  e_i = exp((x_i - M) / temperature),  M = max x,  Z = sum of e
//
// The vocabulary is cut into chunks of 2048, a group each:
//   1. every row's chunks: maximum, its first index, and the sum of e against the chunk's own maximum;
//   2. each sequence's decision, from its rows' chunk results (every group of a sequence works it out
//      for itself: a few hundred values), the weights' sum over each chunk of the row to draw from, and,
//      by the group that is last to leave its sum, the draw: the chunk by the chunks' sums, then the
//      index within it.
// Exponentials and sums are in f64 (the vector unit's f64 rate is f32's here): the draw compares u with
// running sums whose borders lie 1 / 150,000 apart and closer, and f32 would move them by 1e-7 of the whole.
#include "common.h"

namespace {

constexpr uint32_t kWaves = 4, kThreads = 64 * kWaves, kEach = 8, kChunk = kThreads * kEach;
constexpr uint32_t kRuns = kEach / 4;  // runs of 256 indices a wave takes of a chunk
// A lane has four consecutive indices of each run: its value j is index place(wave, lane, j) of the chunk,
// in index order by (wave, j / 4, lane, j % 4).
TS_DEV uint32_t place(uint32_t wave, uint32_t lane, uint32_t j) {
    return (wave * kRuns + j / 4) * 256 + lane * 4 + j % 4;
}

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
    double *sums;       // [seqs][parts]
    uint32_t *done;     // [seqs]: groups of the second kernel that have left their sum
    uint32_t seqs, most, rows, width, stride, parts;
    float temperature;
    int whole_x, whole_q;  // four consecutive logits, or probabilities, are one aligned load
};

// A constant in scalar registers: as an addend it would otherwise be copied to vector ones each time.
TS_DEV double scalar(double c) {
    asm("" : "+s"(c));
    return c;
}

// 2^t for t <= 0: t = n + f, |f| <= 1/2, the series of 2^f = e^(f ln 2) up to the 10th power (the 11th is
// 3e-13 at most, at |f| = 1/2). 0 for NaN and t below -1074.
TS_DEV double exp2_neg(double t) {
    t = fmax(t, -1500.0);
    const double n = __builtin_rint(t), f = t - n;
    double r = __builtin_fma(f, scalar(7.054911620801123e-09), scalar(1.01780860092397e-07));
    r = __builtin_fma(r, f, scalar(1.321548679014431e-06));
    r = __builtin_fma(r, f, scalar(1.5252733804059841e-05));
    r = __builtin_fma(r, f, scalar(0.0001540353039338161));
    r = __builtin_fma(r, f, scalar(0.0013333558146428443));
    r = __builtin_fma(r, f, scalar(0.009618129107628477));
    r = __builtin_fma(r, f, scalar(0.05550410866482158));
    r = __builtin_fma(r, f, scalar(0.24022650695910072));
    r = __builtin_fma(r, f, scalar(0.6931471805599453));
    r = __builtin_fma(r, f, 1.0);
    return __builtin_amdgcn_ldexp(r, (int)n);
}

// e of logit x against the maximum: 1 at the maximum (+inf too), 0 for NaN and -inf. `by`: log2(e) /
// temperature.
TS_DEV double weight(float x, float most, double by) {
    if (!(most < __builtin_inff())) return x == most ? 1.0 : 0.0;
    const double e = exp2_neg(((double)x - (double)most) * by);
    return x > -__builtin_inff() ? e : 0.0;
}
// Of a thread's logits side by side (x as load_logits leaves them, `most` finite or +inf; -inf gives 0).
template <int N>
TS_DEV void weights(const float (&x)[N], float most, double by, double (&w)[N]) {
    if (!(most < __builtin_inff())) {
#pragma unroll
        for (int j = 0; j < N; j++) w[j] = x[j] == most ? 1.0 : 0.0;
        return;
    }
#pragma unroll
    for (int j = 0; j < N; j++) w[j] = exp2_neg(((double)x[j] - (double)most) * by);
}
TS_DEV double per_unit(float temperature) { return 1.4426950408889634 / (double)temperature; }

template <bool BF16>
TS_DEV float logit(const VerifyParams &p, uint32_t row, uint32_t i) {
    const size_t at = (size_t)row * p.stride + i;
    return BF16 ? bf16_float(((const uint16_t *)p.logits)[at]) : ((const float *)p.logits)[at];
}

// The thread's 16 logits of a chunk, NaN and indices past the row as -inf.
template <bool BF16>
TS_DEV void load_logits(const VerifyParams &p, uint32_t row, uint32_t chunk, float (&x)[kEach]) {
    const uint32_t wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
#pragma unroll
    for (uint32_t v = 0; v < kEach; v += 4) {
        const uint32_t i = chunk * kChunk + place(wave, lane, v);
        if (p.whole_x && i + 3 < p.width) {
            const size_t at = (size_t)row * p.stride + i;
            if (BF16) {
                const u32x2 w = *(const u32x2 *)((const uint16_t *)p.logits + at);
                x[v] = lo_bf16(w.x);
                x[v + 1] = hi_bf16(w.x);
                x[v + 2] = lo_bf16(w.y);
                x[v + 3] = hi_bf16(w.y);
            } else {
                const f32x4 w = *(const f32x4 *)((const float *)p.logits + at);
#pragma unroll
                for (int e = 0; e < 4; e++) x[v + e] = w[e];
            }
        } else {
#pragma unroll
            for (uint32_t e = 0; e < 4; e++)
                x[v + e] = i + e < p.width ? logit<BF16>(p, row, i + e) : -__builtin_inff();
        }
    }
#pragma unroll
    for (uint32_t j = 0; j < kEach; j++) x[j] = x[j] > -__builtin_inff() ? x[j] : -__builtin_inff();
}

// The drafter's probabilities at the same indices, NaN and negative ones as 0.
TS_DEV void load_probs(const VerifyParams &p, size_t row, uint32_t chunk, float (&q)[kEach]) {
    const uint32_t wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const float *from = p.probs + row * p.width;
#pragma unroll
    for (uint32_t v = 0; v < kEach; v += 4) {
        const uint32_t i = chunk * kChunk + place(wave, lane, v);
        if (p.whole_q && i + 3 < p.width) {
            const f32x4 w = *(const f32x4 *)(from + i);
#pragma unroll
            for (int e = 0; e < 4; e++) q[v + e] = w[e];
        } else {
#pragma unroll
            for (uint32_t e = 0; e < 4; e++) q[v + e] = i + e < p.width ? from[i + e] : 0.0f;
        }
    }
#pragma unroll
    for (uint32_t j = 0; j < kEach; j++) q[j] = q[j] > 0.0f ? q[j] : 0.0f;
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

TS_DEV double wave_total(double v) {
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) v += __shfl_xor(v, o, 64);
    return v;
}

TS_DEV double group_total(double v) {
    __shared__ double ss[4];
    v = wave_total(v);
    if ((threadIdx.x & 63) == 0) ss[threadIdx.x >> 6] = v;
    __syncthreads();
    return (ss[0] + ss[1]) + (ss[2] + ss[3]);
}

// The larger value, at equal ones the lower index, over the wave.
TS_DEV void wave_best(float &v, uint32_t &at) {
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const float w = __shfl_xor(v, o, 64);
        const uint32_t b = __shfl_xor(at, o, 64);
        if (w > v || (w == v && b < at)) { v = w; at = b; }
    }
}

// A wave takes its maximum and sums against it by itself; the four meet once, at the end.
template <bool BF16>
__global__ __launch_bounds__(256) void verify_rows_kernel(VerifyParams p) {
    __shared__ Chunk waves[4];
    const uint32_t part = blockIdx.x % p.parts, sr = blockIdx.x / p.parts;
    const uint32_t s = sr / (p.most + 1), t = sr % (p.most + 1), wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const Seq q = seq_of(p, s);
    if (!q.good || t > q.count) return;
    if (p.done && part == 0 && t == 0 && threadIdx.x == 0) p.done[s] = 0;
    float x[kEach];
    load_logits<BF16>(p, q.first + t, part, x);
    const double by = per_unit(q.temperature);
    float most = x[0];
#pragma unroll
    for (uint32_t j = 1; j < kEach; j++) most = fmaxf(most, x[j]);
    most = wave_max(most);
    uint32_t at = p.width;
#pragma unroll
    for (int j = kEach - 1; j >= 0; j--)
        if (x[j] == most) at = part * kChunk + place(wave, lane, j);  // the lane's first (its places ascend)
    if (!(most > -__builtin_inff())) at = p.width;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) at = min(at, (uint32_t)__shfl_xor((int)at, o, 64));
    double sum = 0.0;
    if (!q.greedy) {
        double w[kEach];
        weights(x, most, by, w);
#pragma unroll
        for (uint32_t j = 0; j < kEach; j++) sum += w[j];
        sum = most > -__builtin_inff() ? wave_total(sum) : 0.0;
    }
    if (lane == 0) waves[wave] = Chunk{sum, most, at};
    __syncthreads();
    if (threadIdx.x == 0) {
        Chunk c = waves[0];
        for (int w = 1; w < 4; w++)
            if (waves[w].most > c.most) { c.most = waves[w].most; c.at = waves[w].at; }  // ties: the lower wave's
        if (!q.greedy) {
            c.sum = 0.0;
            for (int w = 0; w < 4; w++) c.sum += waves[w].sum * weight(waves[w].most, c.most, by);
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
    for (uint32_t t = threadIdx.x >> 4; t <= q.count; t += kThreads / 16) {
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
            const float was = most;
#pragma unroll
            for (uint32_t j = 0; j < 4; j++)
                if (j0 + 16 * j < p.parts && four[j].most > most) { most = four[j].most; at = four[j].at; }
            if (q.greedy) continue;
            z *= weight(was, most, by);
#pragma unroll
            for (uint32_t j = 0; j < 4; j++)
                if (j0 + 16 * j < p.parts) z += four[j].sum * weight(four[j].most, most, by);
        }
        float whole = most;
#pragma unroll
        for (int o = 1; o < 16; o <<= 1) {
            const float w = __shfl_xor(whole, o, 64);
            const uint32_t b = __shfl_xor(at, o, 64);
            if (w > whole || (w == whole && b < at)) { whole = w; at = b; }
        }
        if (!q.greedy) {
            z *= weight(most, whole, by);
#pragma unroll
            for (int o = 1; o < 16; o <<= 1) z += __shfl_xor(z, o, 64);
        }
        if (l16 == 0) {
            chance = chance > 0.0f ? chance : 0.0f;
            taken[t] = draft < p.width && (q.greedy ? draft == at : (double)u * (double)chance * z < weight(x, whole, by));
            rows[t] = Verdict{z, whole, q.first + t, t, t < q.count, at};
        }
    }
    __syncthreads();
    uint32_t n = 0;
    while (n < q.count && taken[n]) n++;
    return rows[n];
}

// The weights that a draw gives the thread's 16 indices of a chunk of the verdict's row.
template <bool BF16>
TS_DEV void draw_weights(const VerifyParams &p, uint32_t s, const Verdict &v, double by, bool residual, uint32_t draft,
                         uint32_t chunk, double (&w)[kEach]) {
    float x[kEach], q[kEach];
    load_logits<BF16>(p, v.row, chunk, x);
    const bool probs = residual && p.probs;
    if (probs) load_probs(p, (size_t)s * p.most + v.accepted, chunk, q);
    weights(x, v.most, by, w);
#pragma unroll
    for (uint32_t j = 0; j < kEach; j++) {
        if (probs) {
            w[j] -= (double)q[j] * v.whole;
            w[j] = w[j] > 0.0 ? w[j] : 0.0;
        } else if (residual && chunk * kChunk + place(threadIdx.x >> 6, threadIdx.x & 63, j) == draft) {
            w[j] = 0.0;
        }
    }
}

// The sequence's tokens: the accepted drafts, the pick, `width` in the rest.
TS_DEV void answer(const VerifyParams &p, uint32_t s, bool good, uint32_t accepted, uint32_t pick) {
    for (uint32_t t = threadIdx.x; t <= p.most; t += kThreads)
        p.tokens[(size_t)s * (p.most + 1) + t] = !good           ? p.width
                                                 : t < accepted  ? p.drafts[(size_t)s * p.most + t]
                                                 : t == accepted ? pick
                                                                 : p.width;
    if (threadIdx.x == 0) p.accepted[s] = good ? accepted : 0;
    if (threadIdx.x == 0 && !good && p.status) atomicOr(p.status, TS_STATUS_POSITION);
}

// Inclusive running sums over the 256 threads' values in thread order, and the whole.
TS_DEV double running(double v, double &whole) {
    __shared__ double ends[4];
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const double w = __shfl_up(v, o, 64);
        if ((int)lane >= o) v += w;
    }
    __syncthreads();
    if (lane == 63) ends[wave] = v;
    __syncthreads();
    double before = 0.0;
    whole = 0.0;
    for (uint32_t w = 0; w < 4; w++) {
        if (w < wave) before += ends[w];
        whole += ends[w];
    }
    return before + v;
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

// The draw: a group a chunk leaves its chunk's weight, the last of a sequence to do so picks the token.
template <bool BF16>
__global__ __launch_bounds__(256) void verify_draw_kernel(VerifyParams p) {
    __shared__ uint32_t found, last, before;
    __shared__ double under, runs[kWaves * kRuns];
    const uint32_t part = blockIdx.x % p.parts, s = blockIdx.x / p.parts;
    const uint32_t wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
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
    bool residual = v.refused;
    const uint32_t draft = v.refused ? p.drafts[(size_t)s * p.most + v.accepted] : 0;
    const Chunk *own = p.chunks + ((size_t)s * (p.most + 1) + v.accepted) * p.parts;
    if (!residual) {  // from p itself: its chunks' weights are there
        if (part != 0) return;
    } else {
        double w[kEach], sum = 0.0;
        draw_weights<BF16>(p, s, v, by, true, draft, part, w);
#pragma unroll
        for (uint32_t j = 0; j < kEach; j++) sum += w[j];
        sum = group_total(sum);
        // The sum is stored and counted past the XCDs' own L2s; the last group sees every one.
        if (threadIdx.x == 0) {
            __hip_atomic_store(p.sums + (size_t)s * p.parts + part, sum, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            before = __hip_atomic_fetch_add(p.done + s, 1u, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT);
        }
        __syncthreads();
        if (before + 1 != p.parts) return;
    }
    // Chunk sums: of the residual, or of p should the residual be zero everywhere.
    auto chunk_sum = [&](uint32_t j) {
        return residual ? __hip_atomic_load(p.sums + (size_t)s * p.parts + j, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT)
                        : own[j].sum * weight(own[j].most, v.most, by);
    };
    const uint32_t per = (p.parts + kThreads - 1) / kThreads, j0 = threadIdx.x * per, j1 = min(j0 + per, p.parts);
    double whole, mine, upto;
    auto total = [&] {
        mine = 0.0;
        for (uint32_t j = j0; j < j1; j++) mine += chunk_sum(j);
        upto = running(mine, whole);
    };
    total();
    if (residual && !(whole > 0.0)) {
        residual = false;
        total();
    }
    // The first chunk whose running sum passes the target; without one (rounding, or u not below
    // 1) the last chunk that weighs anything.
    const double target = (double)p.uniforms[(size_t)s * (p.most + 1) + p.most] * whole;
    if (threadIdx.x == 0) { found = 0xffffffffu; last = 0; under = 0.0; }
    __syncthreads();
    uint32_t over = 0xffffffffu, weighs = 0;  // the thread's own such chunks, and the sums before them
    double before_over = 0.0, before_weighs = 0.0, c = upto - mine;
    for (uint32_t j = j0; j < j1; j++) {
        const double w = chunk_sum(j);
        if (w > 0.0) {
            weighs = j;
            before_weighs = c;
            if (over == 0xffffffffu && c + w > target) {
                over = j;
                before_over = c;
            }
        }
        c += w;
    }
    if (over != 0xffffffffu) atomicMin(&found, over);
    if (weighs) atomicMax(&last, weighs);
    __syncthreads();
    const bool passes = found != 0xffffffffu;
    const uint32_t chunk = passes ? found : last;
    if (chunk >= j0 && chunk < j1) under = passes ? before_over : before_weighs;
    __syncthreads();
    const double start = under;
    if (threadIdx.x == 0) { found = 0xffffffffu; last = 0; }
    __syncthreads();
    // Within it: the sums of the runs of 256 indices, then each thread's own four of each run.
    double w[kEach], ends[kRuns];
    draw_weights<BF16>(p, s, v, by, residual, draft, chunk, w);
#pragma unroll
    for (uint32_t run = 0; run < kRuns; run++) {
        double c = (w[4 * run] + w[4 * run + 1]) + (w[4 * run + 2] + w[4 * run + 3]);
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const double up = __shfl_up(c, o, 64);
            if ((int)lane >= o) c += up;
        }
        ends[run] = c;
        if (lane == 63) runs[wave * kRuns + run] = c;
    }
    __syncthreads();
    uint32_t first = 0xffffffffu, end = 0;  // end: past the last index that weighs anything
    upto = start;
    for (uint32_t run = 0; run < wave * kRuns; run++) upto += runs[run];
#pragma unroll
    for (uint32_t run = 0; run < kRuns; run++) {
        c = __shfl_up(ends[run], 1, 64);
        c = upto + (lane ? c : 0.0);
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const uint32_t i = chunk * kChunk + place(wave, lane, 4 * run + e);
            c += w[4 * run + e];
            if (first == 0xffffffffu && w[4 * run + e] > 0.0 && c > target) first = i;
            if (w[4 * run + e] > 0.0) end = i + 1;
        }
        upto += runs[wave * kRuns + run];
    }
    if (first != 0xffffffffu) atomicMin(&found, first);
    atomicMax(&last, end);
    __syncthreads();
    answer(p, s, true, v.accepted, found != 0xffffffffu ? found : last ? last - 1 : p.width);
}

struct Sizes {
    size_t chunks, sums, done;  // bytes
    size_t whole() const { return chunks + sums + done; }
};

Sizes sizes(const ts_verify_args *a) {
    const size_t parts = ((size_t)a->width + kChunk - 1) / kChunk;
    Sizes z;
    z.chunks = (size_t)a->seqs * (a->most + 1) * parts * sizeof(Chunk);
    z.sums = a->uniforms ? a->seqs * parts * sizeof(double) : 0;
    z.done = a->uniforms ? (size_t)a->seqs * sizeof(uint32_t) : 0;
    return z;
}

int check(const ts_verify_args *a) {
    TS_REQUIRE(a && a->logits && a->tokens && a->accepted, "verify: null pointer");
    TS_REQUIRE(a->drafts || a->most == 0, "verify: null pointer");
    TS_REQUIRE(a->most <= kMostDrafts, "verify: %u drafts a sequence (at most %u)", a->most, kMostDrafts);
    TS_REQUIRE(a->logits_dtype == TS_F32 || a->logits_dtype == TS_BF16, "verify: logits f32 or bf16 supported");
    TS_REQUIRE(a->width >= 1 && a->width <= 1u << 28 && a->stride >= a->width, "verify: rows of %u logits, %u apart",
               a->width, a->stride);
    TS_REQUIRE(a->first || (uint64_t)a->seqs * (a->most + 1) <= a->rows, "verify: %u sequences of %u rows, %u rows given",
               a->seqs, a->most + 1, a->rows);
    TS_REQUIRE((uint64_t)a->seqs * (a->most + 1) * ((a->width + kChunk - 1) / kChunk) <= 0x7fffffffull,
               "verify: %u sequences in one launch", a->seqs);
    TS_REQUIRE(ts::aligned(a->logits, 4), "verify: logits must be 4-byte aligned");
    return TS_OK;
}

template <bool BF16>
int launch(const VerifyParams &p, hipStream_t stream) {
    hipLaunchKernelGGL(verify_rows_kernel<BF16>, dim3(p.seqs * (p.most + 1) * p.parts), dim3(kThreads), 0, stream, p);
    TS_CHECK_LAUNCH("verify rows launch");
    if (p.uniforms)
        hipLaunchKernelGGL(verify_draw_kernel<BF16>, dim3(p.seqs * p.parts), dim3(kThreads), 0, stream, p);
    else
        hipLaunchKernelGGL(verify_greedy_kernel<BF16>, dim3(p.seqs), dim3(kThreads), 0, stream, p);
    TS_CHECK_LAUNCH("verify draw launch");
    return TS_OK;
}

}  // namespace

extern "C" size_t tessera_hip_verify_workspace(const ts_verify_args *a) { return a ? sizes(a).whole() : 0; }

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
    p.parts = (a->width + kChunk - 1) / kChunk;
    p.temperature = a->temperature;
    p.whole_x = a->stride % 4 == 0 && ts::aligned(a->logits, a->logits_dtype == TS_BF16 ? 8 : 16);
    p.whole_q = a->width % 4 == 0 && ts::aligned(a->draft_probs, 16);
    return a->logits_dtype == TS_BF16 ? launch<true>(p, (hipStream_t)stream) : launch<false>(p, (hipStream_t)stream);
}
