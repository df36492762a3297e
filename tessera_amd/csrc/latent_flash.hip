// The expanded form of latent attention over whole sequences packed back to back: row i of a sequence of n rows and m
// keys stands at m - n + i, w = softmax((q . k + q' . r) * scale) over the keys [position - back, position], out = sum
// of w v; every head has keys k and values v of its own, the rotated part r is all heads'.
//
// A wave has 32 rows of one head, the columns of S^T = K q^T and O^T = V^T P^T on the 32-wide matrix products, so a
// row's scores stay in two lanes and P^T is the second product's operand as it stands. The four waves of a group have
// 128 neighbouring rows and share the keys, 32 a step: k, r and v rows go from memory straight to LDS, two steps ahead
// of their use; V^T comes through the transposing LDS read. Two groups share a CU, so that one's softmax runs under the
// other's products.
#include "common.h"

namespace {

constexpr uint32_t kWaves = 4, kThreads = 64 * kWaves, kRows = 32 * kWaves, kKeys = 32, kRing = 3;
constexpr uint32_t kMaxOrder = 256;  // row tiles that are ordered by cost
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
// How many keys the rows of a sequence's tile t see (of its last row, at most `back` and its own).
TS_DEV uint32_t span_of(const FlashParams &p, const Sequence &q, uint32_t t) {
    const int64_t last = (int64_t)q.m - q.n + min((t + 1) * kRows, q.n);
    return last <= 0 ? 0 : (uint32_t)min(last, (int64_t)p.back + kRows);
}

typedef short ts_v4i16 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) ts_v4i16 lds_v4i16;
// Four keys of one d, from the 8-byte pieces of four rows (lane 4 e + c of 16: row e, d 4 c ..).
TS_DEV u32x2 read_vt4(const char *a) {
    return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4i16 *)a));
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
// The bits of the bf16 values of a pair that are not finite.
TS_DEV uint32_t odd_mask(uint32_t x) {
    return ((x & 0x7f80u) == 0x7f80u ? 0xffffu : 0u) | ((x & 0x7f800000u) == 0x7f800000u ? 0xffff0000u : 0u);
}
TS_DEV uint32_t again(uint32_t v) {  // (keeps rare steps' addresses from being computed ahead of the loop)
    asm volatile("" : "+v"(v));
    return v;
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
    __shared__ uint32_t cost[kMaxOrder], chosen, odd_keys[kWaves];
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const uint32_t col = lane & 31, half = lane >> 5;
    const uint32_t h = blockIdx.x % p.heads;

    // The group's row tile: those of all sequences, one behind the other, the widest first.
    uint32_t t = blockIdx.x / p.heads;
    if (p.tiles > 1 && p.tiles <= kMaxOrder) {
        for (uint32_t i = threadIdx.x; i < kMaxOrder; i += kThreads) cost[i] = 0;
        if (threadIdx.x == 0) chosen = 0;
        __syncthreads();
        uint32_t before = 0;
        for (uint32_t s0 = 0; s0 < p.seqs; s0 += 64) {
            Sequence q;
            uint32_t n;
            const uint32_t upto = before + tiles_upto(p, s0 + lane, q, n);
            if (wave == 0)
                for (uint32_t t = 0; t < n && upto - n + t < kMaxOrder; t++) cost[upto - n + t] = span_of(p, q, t) + 1;
            before = __builtin_amdgcn_readlane(upto, 63);
        }
        __syncthreads();
        for (uint32_t i = threadIdx.x; i < p.tiles; i += kThreads) {
            const uint32_t c = cost[i];
            uint32_t ahead = 0;
            for (uint32_t j = 0; j < p.tiles; j++) {
                const uint32_t d = cost[j];
                ahead += (d > c) | ((d == c) & (j < i));
            }
            if (ahead == t) chosen = i;
        }
        __syncthreads();
        t = __builtin_amdgcn_readfirstlane(chosen);
    }
    Sequence q;
    for (uint32_t s0 = 0;; s0 += 64) {
        if (s0 >= p.seqs) return;
        uint32_t n;
        const uint32_t upto = tiles_upto(p, s0 + lane, q, n);
        const uint64_t here = __builtin_amdgcn_ballot_w64(t < upto);
        if (here) {
            const uint32_t at = __builtin_ctzll(here);
            t -= __builtin_amdgcn_readlane(upto - n, at);
            q = Sequence{(uint32_t)__builtin_amdgcn_readlane(q.row0, at), (uint32_t)__builtin_amdgcn_readlane(q.n, at),
                         (uint32_t)__builtin_amdgcn_readlane(q.key0, at), (uint32_t)__builtin_amdgcn_readlane(q.m, at)};
            break;
        }
        t -= __builtin_amdgcn_readlane(upto, 63);
    }
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

    const uint32_t steps = hi < 0 ? 0 : (uint32_t)(hi - (lo & ~31)) / kKeys + 1;
    const int32_t base = lo & ~31;
    // One step's rows, a KiB a load; keys past the last are the last again.
    auto issue = [&](uint32_t n, uint32_t slot) {
        char *to = stage + slot * kStage;
        const uint32_t key0 = base + n * kKeys, most = (uint32_t)hi - key0;
        const auto kbuf = raw_buffer(p.k + (size_t)(q.key0 + key0) * p.k_stride + (size_t)h * p.k_head);
        const auto vbuf = raw_buffer(p.v + (size_t)(q.key0 + key0) * p.v_stride + (size_t)h * p.v_head);
        const auto rbuf = raw_buffer(p.r + (size_t)(q.key0 + key0) * p.r_stride);
        auto load = [&](auto buf, char *at, uint32_t part, uint32_t pieces, uint32_t stride, uint32_t swap_kind) {
            const uint32_t g = 64 * part + lane, r = g / pieces, pc = g % pieces;
            const uint32_t swap = swap_kind == 0 ? (pieces == 16 ? key_swap<16>(r) : pieces == 8 ? key_swap<8>(r) : key_swap<4>(r))
                                                 : (pieces == 16 ? value_swap<16>(r) : value_swap<8>(r));
            buffer_to_lds16(buf, at + part * 1024, min(r, most) * stride * 2 + (pc ^ swap) * 16, 0);
        };
#pragma unroll
        for (uint32_t x = 0; x < kK / 1024; x += kWaves)
            if (x + kWaves <= kK / 1024 || wave + x < kK / 1024) load(kbuf, to, x + wave, kPk, p.k_stride, 0);
#pragma unroll
        for (uint32_t x = 0; x < kR / 1024; x += kWaves)
            if (x + kWaves <= kR / 1024 || wave + x < kR / 1024) load(rbuf, to + kK, x + wave, kPr, p.r_stride, 0);
#pragma unroll
        for (uint32_t x = 0; x < kV / 1024; x += kWaves)
            if (x + kWaves <= kV / 1024 || wave + x < kV / 1024) load(vbuf, to + kK + kR, x + wave, kPv, p.v_stride, 1);
    };
    // Loads of a step by the wave with the fewest.
    constexpr uint32_t kLeast = kK / 1024 / kWaves + kR / 1024 / kWaves + kV / 1024 / kWaves;

#pragma unroll
    for (uint32_t n = 0; n + 1 < kRing; n++)
        if (n < steps) issue(n, n);
    for (uint32_t n = 0, slot = 0; n < steps; n++) {
        if (steps - n >= kRing - 1)
            asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"((kRing - 2) * kLeast) : "memory");
        else
            asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
        if (n + kRing - 1 < steps) issue(n + kRing - 1, (slot + kRing - 1) % kRing);
        char *at = stage + slot * kStage;
        slot = slot + 1 == kRing ? 0 : slot + 1;
        const int32_t here = base + (int32_t)(n * kKeys), end = here + (int32_t)kKeys - 1;
        const bool apart = here < same_lo || end > same_hi;  // some key is one row's and not another's, or no key
        const bool work = here <= whi && end >= wlo;
        if (!apart && !work) continue;

        f32x16 s;
#pragma unroll
        for (int e = 0; e < 16; e++) s[e] = 0.0f;
        const uint32_t k0 = again(koff), r0 = again(roff), v0 = again(voff);
#pragma unroll
        for (uint32_t j = 0; j < kQ; j++) {
            const bf16x8 a = j < NOPE / 16 ? *(const bf16x8 *)(at + (k0 ^ 32 * j))
                                           : *(const bf16x8 *)(at + (r0 ^ 32 * (j - NOPE / 16)));
            s = mfma32(a, qv[j], s);
        }
        // Register e of a lane: key 8 (e / 4) + 4 half + e % 4.
        if (here < wsame_lo || end > wsame_hi) {
            const int32_t upto = pos - here - 4 * (int32_t)half, since = from - here - 4 * (int32_t)half;
#pragma unroll
            for (int e = 0; e < 16; e++) {
                const int32_t x = 8 * (e / 4) + e % 4;
                s[e] = x <= upto && x >= since ? s[e] : -INFINITY;
            }
        }
        float mx = s[0];
#pragma unroll
        for (int e = 1; e < 16; e++) mx = fmaxf(mx, s[e]);
        mx = halves_max(mx) * sl;
        const bool raise = mx > m + kSlack;
        const float mn = raise ? mx : m, mo = mn == -INFINITY ? 0.0f : mn;
        uint32_t w[8];
        float sum = 0.0f;
#pragma unroll
        for (int e = 0; e < 16; e += 2) {
            const float x = __builtin_amdgcn_exp2f(fmaf(s[e], sl, -mo)), y = __builtin_amdgcn_exp2f(fmaf(s[e + 1], sl, -mo));
            sum += x + y;
            w[e / 2] = bf16_pair(x, y);
        }
        if (__builtin_amdgcn_ballot_w64(raise) != 0) {
            const float alpha = raise ? __builtin_amdgcn_exp2f(m - mn) : 1.0f;
            l *= alpha;
            m = mn;
#pragma unroll
            for (uint32_t d = 0; d < kD; d++) o[d] *= alpha;
        }
        l += sum;
        if (apart) {
            // A value that is not finite must reach the rows that see it alone, and the product's 0 times it would be
            // NaN: such values are looked for, added by themselves, and cleared, by all waves of the group together.
            uint32_t bad = 0;  // keys that hold one
#pragma unroll 1
            for (uint32_t k = wave; k < kKeys; k += kWaves) {
                const uint32_t l0 = again(lane);
                const uint32_t x = *(const uint32_t *)(at + kK + kR + k * (2 * VALUE) + (l0 % (VALUE / 2)) * 4);
                bad |= __builtin_amdgcn_ballot_w64(odd_mask(x) != 0) != 0 ? 1u << k : 0u;
            }
            odd_keys[wave] = bad;
            lds_barrier();
            bad = 0;
#pragma unroll
            for (uint32_t x = 0; x < kWaves; x++) bad |= __builtin_amdgcn_readfirstlane(odd_keys[x]);
            for (uint32_t left = bad; left;) {
                const uint32_t k = __builtin_ctz(left), swap = value_swap<kPv>(k), g = again(half);
                left &= left - 1;
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
            if (bad) {
                lds_barrier();
#pragma unroll 1
                for (uint32_t k = wave; k < kKeys; k += kWaves) {
                    const uint32_t l0 = again(lane);
                    uint32_t *x = (uint32_t *)(at + kK + kR + k * (2 * VALUE)) + l0;
                    if (l0 < VALUE / 2) *x &= ~odd_mask(*x);
                }
                lds_barrier();
            }
        }
#pragma unroll
        for (uint32_t x = 0; x < kKeys / 16; x++)
#pragma unroll
            for (uint32_t d = 0; d < kD; d++) {
                const char *v = at + (v0 ^ d * 64) + x * 16 * (2 * VALUE);
                const u32x2 lo4 = read_vt4(v);
                // (Eight rows on the XOR is the same.)
                const u32x2 hi4 = read_vt4(v + 8 * (2 * VALUE));
                o[d] = mfma32(as_bf16x8(u32x4{lo4.x, lo4.y, hi4.x, hi4.y}),
                              as_bf16x8(u32x4{w[4 * x], w[4 * x + 1], w[4 * x + 2], w[4 * x + 3]}), o[d]);
            }
    }
    if (!there) return;
    // A row that sees no key is zero.
    const float sum = halves_sum(l), by = pos < 0 ? 0.0f : 1.0f / sum;
    uint16_t *to = p.out + ((size_t)row * p.heads + h) * VALUE + 4 * half;
#pragma unroll
    for (uint32_t d = 0; d < kD; d++)
#pragma unroll
        for (uint32_t e = 0; e < 4; e++)
            *(u32x2 *)(to + 32 * d + 8 * e) = u32x2{pack_bf16x2(o[d][4 * e] * by, o[d][4 * e + 1] * by),
                                                    pack_bf16x2(o[d][4 * e + 2] * by, o[d][4 * e + 3] * by)};
}

template <uint32_t NOPE, uint32_t ROPE, uint32_t VALUE>
int launch(const FlashParams &p, uint32_t groups, void *stream) {
    constexpr uint32_t kLds = kRing * kKeys * 2 * (NOPE + ROPE + VALUE);
    static const hipError_t attr = hipFuncSetAttribute((const void *)flash_latent_kernel<NOPE, ROPE, VALUE>,
                                                       hipFuncAttributeMaxDynamicSharedMemorySize, kLds);
    if (attr != hipSuccess) return ts::hip_status(attr, "flash_latent: shared memory attribute");
    hipLaunchKernelGGL((flash_latent_kernel<NOPE, ROPE, VALUE>), dim3(groups), dim3(kThreads), kLds, (hipStream_t)stream, p);
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
    TS_REQUIRE(a->q_stride >= a->heads * (a->nope + a->rope) && a->q_stride % 8 == 0,
               "flash_latent: q rows %u apart must hold %u heads and be whole 16-byte pieces", a->q_stride, a->heads);
    TS_REQUIRE(a->k_stride % 8 == 0 && a->k_head % 8 == 0 && a->v_stride % 8 == 0 && a->v_head % 8 == 0 && a->r_stride % 8 == 0,
               "flash_latent: rows and heads of k, v and r must be whole 16-byte pieces apart");
    if (a->rows == 0 || a->seqs == 0) return TS_OK;
    TS_REQUIRE(a->q && a->out && (a->key_rows == 0 || (a->k && a->v && a->r)), "flash_latent: null pointer");
    TS_REQUIRE(ts::aligned(a->q, 16) && ts::aligned(a->k, 16) && ts::aligned(a->v, 16) && ts::aligned(a->r, 16) &&
                   ts::aligned(a->out, 16),
               "flash_latent: q, k, v, r and out must be 16-byte aligned");
    // (32 keys within a 32-bit offset.)
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
    TS_REQUIRE(groups <= 0x7fffffffull, "flash_latent: %u rows in one launch", a->rows);
    return wide ? launch<128, 64, 128>(p, (uint32_t)groups, stream) : launch<64, 32, 64>(p, (uint32_t)groups, stream);
}
