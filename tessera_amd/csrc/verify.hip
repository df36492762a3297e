// Verification of drafted tokens (speculative decoding) against the target's distribution, from given
// uniform numbers: draft t of a sequence is taken while u_t q_t(draft) < p_t(draft), and the token after
// the taken ones is drawn from max(p - q, 0) (after a refusal) or p by inverting the running sum in index
// order. (Rejection sampling keeps the target's distribution: Leviathan et al., Chen et al., 2023.) No
// counterpart in the reference, which decodes greedily, one token a step.
//
//   p_i = e_i / Z,  e_i = exp((x_i - M) / temperature),  M = max x,  Z = sum of e
//
// The vocabulary is cut into chunks of 4096, a group each:
//   1. every row's chunks: maximum, its first index, and the sum of e against the chunk's own maximum;
//   2. each sequence's decision, from its rows' chunk results (every group of a sequence works it out
//      for itself: a few hundred values), and the weights' sum over each chunk of the row to draw from;
//   3. the draw: the chunk by the chunks' sums, then the index within it.
// Exponentials and sums are in f64 (the vector unit's f64 rate is f32's here): the draw compares u with
// running sums whose borders lie 1 / 150,000 apart and closer, and f32 would move them by 1e-7 of the whole.
#include "common.h"

namespace {

constexpr uint32_t kChunk = 4096, kThreads = 256, kEach = kChunk / kThreads;

struct Chunk {  // of one row
    double sum;
    float most;
    uint32_t at;  // first index of `most`, or width where the chunk holds none
};

struct Verdict {  // of one sequence
    double whole;       // Z of the row to draw from
    float most;         // its M
    uint32_t row;       // in logits
    uint32_t accepted;
    uint32_t refused;   // 1: a draft was refused
    uint32_t good;      // 0: the sequence's sizes are out of range
    uint32_t pick;      // greedy: the token
};

struct VerifyParams {
    const void *logits;
    const uint32_t *drafts, *counts, *first;
    const float *uniforms, *probs, *temperatures;
    uint32_t *tokens, *accepted, *status;
    Chunk *chunks;      // [seqs][most + 1][parts]
    double *sums;       // [seqs][parts]
    Verdict *verdicts;  // [seqs]
    uint32_t seqs, most, rows, width, stride, parts;
    float temperature;
};

// 2^t for t = y log2(e), y <= 0 (-inf: 0): n + f, |f| <= 1/2, the series of 2^f in f ln 2 up to the 12th
// power (the 13th is below 2e-16 there). log2(e) in two parts, so that f keeps its bits when n is large.
TS_DEV double exp_neg(double y) {
    constexpr double hi = 1.4426950408889634, lo = 2.0355273740931033e-17;
    const double t = y * hi, n = __builtin_rint(t);
    const double f = ((t - n) + (__builtin_fma(y, hi, -t) + y * lo)) * 0.6931471805599453;
    double r = 1.0 / 479001600.0;
    r = __builtin_fma(r, f, 1.0 / 39916800.0);
    r = __builtin_fma(r, f, 1.0 / 3628800.0);
    r = __builtin_fma(r, f, 1.0 / 362880.0);
    r = __builtin_fma(r, f, 1.0 / 40320.0);
    r = __builtin_fma(r, f, 1.0 / 5040.0);
    r = __builtin_fma(r, f, 1.0 / 720.0);
    r = __builtin_fma(r, f, 1.0 / 120.0);
    r = __builtin_fma(r, f, 1.0 / 24.0);
    r = __builtin_fma(r, f, 1.0 / 6.0);
    r = __builtin_fma(r, f, 0.5);
    r = __builtin_fma(r, f, 1.0);
    r = __builtin_fma(r, f, 1.0);
    return t > -1000.0 ? __builtin_amdgcn_ldexp(r, (int)n) : 0.0;
}

// e of logit x against the maximum: 1 at the maximum (+inf too), 0 for NaN and -inf.
TS_DEV double weight(float x, float most, double by) {
    if (!(x > -__builtin_inff())) return 0.0;
    return x == most ? 1.0 : exp_neg(((double)x - (double)most) * by);
}

template <bool BF16>
TS_DEV float logit(const VerifyParams &p, uint32_t row, uint32_t i) {
    const size_t at = (size_t)row * p.stride + i;
    return BF16 ? bf16_float(((const uint16_t *)p.logits)[at]) : ((const float *)p.logits)[at];
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

// The larger value, at equal ones the lower index, over the group; the result in every thread.
TS_DEV void group_best(float &v, uint32_t &at) {
    __shared__ float sv[4];
    __shared__ uint32_t sa[4];
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const float w = __shfl_xor(v, o, 64);
        const uint32_t b = __shfl_xor(at, o, 64);
        if (w > v || (w == v && b < at)) { v = w; at = b; }
    }
    if ((threadIdx.x & 63) == 0) { sv[threadIdx.x >> 6] = v; sa[threadIdx.x >> 6] = at; }
    __syncthreads();
    v = sv[0];
    at = sa[0];
#pragma unroll
    for (int w = 1; w < 4; w++)
        if (sv[w] > v || (sv[w] == v && sa[w] < at)) { v = sv[w]; at = sa[w]; }
}
TS_DEV double group_total(double v) {
    __shared__ double ss[4];
    v = wave_total(v);
    if ((threadIdx.x & 63) == 0) ss[threadIdx.x >> 6] = v;
    __syncthreads();
    return (ss[0] + ss[1]) + (ss[2] + ss[3]);
}

template <bool BF16>
__global__ __launch_bounds__(256) void verify_rows_kernel(VerifyParams p) {
    const uint32_t part = blockIdx.x % p.parts, sr = blockIdx.x / p.parts;
    const uint32_t s = sr / (p.most + 1), t = sr % (p.most + 1);
    const Seq q = seq_of(p, s);
    if (!q.good || t > q.count) return;
    const uint32_t base = part * kChunk;
    float x[kEach];
#pragma unroll
    for (uint32_t j = 0; j < kEach; j++) {
        const uint32_t i = base + j * kThreads + threadIdx.x;
        const float v = logit<BF16>(p, q.first + t, min(i, p.width - 1));
        x[j] = i < p.width && v > -__builtin_inff() ? v : -__builtin_inff();  // NaN too
    }
    float most = -__builtin_inff();
    uint32_t at = p.width;
#pragma unroll
    for (uint32_t j = 0; j < kEach; j++)
        if (x[j] > most) { most = x[j]; at = base + j * kThreads + threadIdx.x; }
    group_best(most, at);
    double sum = 0.0;
    if (!q.greedy) {
        const double by = 1.0 / (double)q.temperature;
#pragma unroll
        for (uint32_t j = 0; j < kEach; j++) sum += weight(x[j], most, by);
        sum = group_total(sum);
    }
    if (threadIdx.x == 0) p.chunks[(size_t)sr * p.parts + part] = Chunk{sum, most, at};
}

// A row's maximum, its first index and Z from its chunks, by one wave; in every lane.
TS_DEV void row_total(const VerifyParams &p, uint32_t sr, double by, bool greedy, float &most, uint32_t &at, double &z) {
    const Chunk *c = p.chunks + (size_t)sr * p.parts;
    const uint32_t lane = threadIdx.x & 63;
    most = -__builtin_inff();
    at = p.width;
    for (uint32_t j = lane; j < p.parts; j += 64)
        if (c[j].most > most) { most = c[j].most; at = c[j].at; }
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const float w = __shfl_xor(most, o, 64);
        const uint32_t b = __shfl_xor(at, o, 64);
        if (w > most || (w == most && b < at)) { most = w; at = b; }
    }
    z = 0.0;
    if (greedy) return;
    for (uint32_t j = lane; j < p.parts; j += 64) z += c[j].sum * weight(c[j].most, most, by);
    z = wave_total(z);
}

constexpr uint32_t kMostDrafts = 64;

// The sequence's verdict, by the whole group; in every thread. Uses no memory but the rows' chunks.
template <bool BF16>
TS_DEV Verdict decide(const VerifyParams &p, uint32_t s, const Seq &q) {
    __shared__ Verdict rows[kMostDrafts + 1];
    __shared__ uint32_t taken[kMostDrafts + 1];
    const uint32_t wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    Verdict v = {0.0, 0.0f, 0, 0, 0, 0, p.width};
    if (!q.good) return v;
    const double by = 1.0 / (double)q.temperature;
    for (uint32_t t = wave; t <= q.count; t += 4) {
        Verdict r = {0.0, 0.0f, q.first + t, t, t < q.count, 1, 0};
        row_total(p, s * (p.most + 1) + t, by, q.greedy, r.most, r.pick, r.whole);
        if (lane == 0) {
            uint32_t take = 0;
            if (t < q.count) {
                const uint32_t draft = p.drafts[(size_t)s * p.most + t];
                if (draft >= p.width)
                    take = 0;
                else if (q.greedy)
                    take = draft == r.pick;
                else {
                    const double e = weight(logit<BF16>(p, q.first + t, draft), r.most, by);
                    float chance = 1.0f;
                    if (p.probs) {
                        chance = p.probs[((size_t)s * p.most + t) * p.width + draft];
                        chance = chance > 0.0f ? chance : 0.0f;
                    }
                    take = (double)p.uniforms[(size_t)s * (p.most + 1) + t] * (double)chance * r.whole < e;
                }
            }
            taken[t] = take;
            rows[t] = r;
        }
    }
    __syncthreads();
    uint32_t n = 0;
    while (n < q.count && taken[n]) n++;
    return rows[n];
}

// The weight that a draw gives index i of the verdict's row.
template <bool BF16>
TS_DEV double draw_weight(const VerifyParams &p, uint32_t s, const Verdict &v, double by, bool residual, uint32_t draft,
                          uint32_t i) {
    const double e = weight(logit<BF16>(p, v.row, i), v.most, by);
    if (!residual) return e;
    if (!p.probs) return i == draft ? 0.0 : e;
    float chance = p.probs[((size_t)s * p.most + v.accepted) * p.width + i];
    chance = chance > 0.0f ? chance : 0.0f;
    const double w = e - (double)chance * v.whole;
    return w > 0.0 ? w : 0.0;
}

template <bool BF16>
__global__ __launch_bounds__(256) void verify_sums_kernel(VerifyParams p) {
    const uint32_t part = blockIdx.x % p.parts, s = blockIdx.x / p.parts;
    const Seq q = seq_of(p, s);
    const Verdict v = decide<BF16>(p, s, q);
    if (part == 0 && threadIdx.x == 0) p.verdicts[s] = v;
    if (!q.good || q.greedy) return;
    const double by = 1.0 / (double)q.temperature;
    if (!v.refused) {  // the draw is from p itself: its chunk sums are there
        const Chunk c = p.chunks[((size_t)s * (p.most + 1) + v.accepted) * p.parts + part];
        if (threadIdx.x == 0) p.sums[(size_t)s * p.parts + part] = c.sum * weight(c.most, v.most, by);
        return;
    }
    const uint32_t draft = p.drafts[(size_t)s * p.most + v.accepted];
    double sum = 0.0;
#pragma unroll 4
    for (uint32_t j = 0; j < kEach; j++) {
        const uint32_t i = part * kChunk + j * kThreads + threadIdx.x;
        if (i < p.width) sum += draw_weight<BF16>(p, s, v, by, true, draft, i);
    }
    sum = group_total(sum);
    if (threadIdx.x == 0) p.sums[(size_t)s * p.parts + part] = sum;
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

template <bool BF16>
__global__ __launch_bounds__(256) void verify_draw_kernel(VerifyParams p) {
    __shared__ uint32_t found, last;
    __shared__ double under;
    const uint32_t s = blockIdx.x;
    const Seq q = seq_of(p, s);
    const bool decided = !p.uniforms;  // all greedy: no kernel before this one has judged
    const Verdict v = decided ? decide<BF16>(p, s, q) : p.verdicts[s];
    uint32_t pick = v.pick;
    if (q.good && !q.greedy) {
        const double by = 1.0 / (double)q.temperature;
        bool residual = v.refused;
        const uint32_t draft = v.refused ? p.drafts[(size_t)s * p.most + v.accepted] : 0;
        const Chunk *own = p.chunks + ((size_t)s * (p.most + 1) + v.accepted) * p.parts;
        const double u = (double)p.uniforms[(size_t)s * (p.most + 1) + p.most];
        // Chunk sums: of the residual, or of p should the residual be zero everywhere.
        auto chunk_sum = [&](uint32_t j) {
            if (j >= p.parts) return 0.0;
            return residual ? p.sums[(size_t)s * p.parts + j] : own[j].sum * weight(own[j].most, v.most, by);
        };
        double whole = 0.0;
        auto total = [&] {
            whole = 0.0;
            for (uint32_t j0 = 0; j0 < p.parts; j0 += kThreads) {
                double w;
                running(chunk_sum(j0 + threadIdx.x), w);
                whole += w;
            }
        };
        total();
        if (residual && !(whole > 0.0)) {
            residual = false;
            total();
        }
        // The first chunk whose running sum passes the target; without one (rounding, or u not below
        // 1) the last chunk that weighs anything.
        const double target = u * whole;
        if (threadIdx.x == 0) { found = 0xffffffffu; last = 0; under = 0.0; }
        double before = 0.0;
        for (uint32_t j0 = 0; j0 < p.parts; j0 += kThreads) {
            double w;
            const double c = chunk_sum(j0 + threadIdx.x), upto = before + running(c, w);
            if (upto > target) atomicMin(&found, j0 + threadIdx.x);
            if (c > 0.0) atomicMax(&last, j0 + threadIdx.x);
            before += w;
        }
        __syncthreads();
        const uint32_t chunk = found != 0xffffffffu ? found : last;
        before = 0.0;
        for (uint32_t j0 = 0; j0 < p.parts; j0 += kThreads) {
            double w;
            const double c = chunk_sum(j0 + threadIdx.x), upto = before + running(c, w);
            if (j0 + threadIdx.x + 1 == chunk) under = upto;  // the sum before the chunk
            before += w;
        }
        __syncthreads();
        const double start = under;
        if (threadIdx.x == 0) { found = 0xffffffffu; last = 0; }
        __syncthreads();
        // Within it, 16 consecutive indices a thread.
        const uint32_t i0 = chunk * kChunk + threadIdx.x * kEach;
        double w[kEach], mine = 0.0, all;
#pragma unroll 4
        for (uint32_t j = 0; j < kEach; j++) {
            w[j] = i0 + j < p.width ? draw_weight<BF16>(p, s, v, by, residual, draft, i0 + j) : 0.0;
            mine += w[j];
        }
        double upto = start + (running(mine, all) - mine);
        uint32_t first = 0xffffffffu, end = 0;  // end: past the last index that weighs anything
#pragma unroll
        for (uint32_t j = 0; j < kEach; j++) {
            upto += w[j];
            if (first == 0xffffffffu && w[j] > 0.0 && upto > target) first = i0 + j;
            if (w[j] > 0.0) end = i0 + j + 1;
        }
        if (first != 0xffffffffu) atomicMin(&found, first);
        atomicMax(&last, end);
        __syncthreads();
        pick = found != 0xffffffffu ? found : last ? last - 1 : p.width;
    }
    if (threadIdx.x == 0 && !q.good && p.status) atomicOr(p.status, TS_STATUS_POSITION);
    for (uint32_t t = threadIdx.x; t <= p.most; t += kThreads)
        p.tokens[(size_t)s * (p.most + 1) + t] = !q.good             ? p.width
                                                 : t < v.accepted    ? p.drafts[(size_t)s * p.most + t]
                                                 : t == v.accepted   ? pick
                                                                     : p.width;
    if (threadIdx.x == 0) p.accepted[s] = q.good ? v.accepted : 0;
}

struct Sizes {
    size_t chunks, verdicts, sums;  // bytes
    size_t whole() const { return chunks + verdicts + sums; }
};

Sizes sizes(const ts_verify_args *a) {
    const size_t parts = ((size_t)a->width + kChunk - 1) / kChunk;
    Sizes z;
    z.chunks = (size_t)a->seqs * (a->most + 1) * parts * sizeof(Chunk);
    z.verdicts = a->uniforms ? (size_t)a->seqs * sizeof(Verdict) : 0;
    z.sums = a->uniforms ? a->seqs * parts * sizeof(double) : 0;
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
    if (p.uniforms) {
        hipLaunchKernelGGL(verify_sums_kernel<BF16>, dim3(p.seqs * p.parts), dim3(kThreads), 0, stream, p);
        TS_CHECK_LAUNCH("verify sums launch");
    }
    hipLaunchKernelGGL(verify_draw_kernel<BF16>, dim3(p.seqs), dim3(kThreads), 0, stream, p);
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
    p.verdicts = (Verdict *)(w + z.chunks);
    p.sums = (double *)(w + z.chunks + z.verdicts);
    p.seqs = a->seqs; p.most = a->most; p.rows = a->rows; p.width = a->width; p.stride = a->stride;
    p.parts = (a->width + kChunk - 1) / kChunk;
    p.temperature = a->temperature;
    return a->logits_dtype == TS_BF16 ? launch<true>(p, (hipStream_t)stream) : launch<false>(p, (hipStream_t)stream);
}
