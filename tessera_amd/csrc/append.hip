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
// The unit of work is a segment: rows r, r + 1, ... of the call that are consecutive positions of
// one slot within one block of 16. One wave owns a segment's kv head: it sees all new values of
// the block's head, so the scale, the codes and (where the scale grows) the codes already there
// are settled without another launch or an atomic. The rows of a call that meet in a block must
// therefore stand together; a later segment of the same block is refused (TS_STATUS_TWICE), found
// by looking through the rows before it.
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
    uint32_t window, kv_groups, head_groups;  // rows a kv group looks at; groups of 4 kv heads; of 16 q heads
    float eps;
    int q_out_bf16;
};

constexpr uint32_t kQBatch = 4;  // q heads a wave

// The lane's pair of a 128-wide row: (j, j + 64) or (2j, 2j + 1).
template <bool XBF16, bool HALVES>
TS_DEV void load_pair(const void *x, size_t at, uint32_t lane, float &a, float &b) {
    if (XBF16) {
        const uint16_t *r = (const uint16_t *)x + at;
        if (HALVES) {
            a = bf16_float(r[lane]);
            b = bf16_float(r[lane + 64]);
        } else {
            const uint32_t w = *(const uint32_t *)(r + 2 * lane);
            a = lo_bf16(w);
            b = hi_bf16(w);
        }
    } else {
        const float *r = (const float *)x + at;
        if (HALVES) {
            a = r[lane];
            b = r[lane + 64];
        } else {
            const float2 w = *(const float2 *)(r + 2 * lane);
            a = w.x;
            b = w.y;
        }
    }
}

template <bool HALVES>
TS_DEV void store_pair_bf16(uint16_t *r, uint32_t lane, float a, float b) {
    if (HALVES) {
        r[lane] = bf16_bits(a);
        r[lane + 64] = bf16_bits(b);
    } else {
        *(uint32_t *)(r + 2 * lane) = pack_bf16x2(a, b);
    }
}

TS_DEV void norm_pair(float &a, float &b, float ga, float gb, float eps) {
    const float inv = 1.0f / sqrtf(wave_sum(a * a + b * b) / 128.0f + eps);
    a = a * (inv * ga);
    b = b * (inv * gb);
}

// Rounded as tessera_hip_qk_norm_rope_append's rotation.
TS_DEV void turn_pair(float &a, float &b, float2 cs) {
    const float x = a, y = b;
    a = fmaf(x, cs.x, -(y * cs.y));
    b = fmaf(y, cs.x, x * cs.y);
}

TS_DEV float finite_abs(float x) {
    const float a = fabsf(x);
    return a < __builtin_inff() ? a : 0.0f;  // infinities and NaN take no part in the scale
}

// The code of x / scale, `inv` = 1 / scale: beyond the range the largest, NaN for infinities and NaN
// (the format has no infinity).
TS_DEV float coded(float x, float inv) {
    const float y = fminf(fmaxf(x * inv, -448.0f), 448.0f);
    return fabsf(x) < __builtin_inff() ? y : __builtin_nanf("");
}
TS_DEV uint32_t code_of(float a) { return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(a, a, 0, false) & 0xffu; }

// Four codes held under one scale as codes under another (factor = old / new, a power of two <= 1).
TS_DEV uint32_t rebase4(uint32_t w, float factor) {
    float f[4];
    e4m3x4_to_f32(w, f);
    int r = __builtin_amdgcn_cvt_pk_fp8_f32(f[0] * factor, f[1] * factor, 0, false);
    r = __builtin_amdgcn_cvt_pk_fp8_f32(f[2] * factor, f[3] * factor, r, true);
    return (uint32_t)r;
}
TS_DEV u32x4 rebase16(u32x4 w, float factor) {
    return u32x4{rebase4(w.x, factor), rebase4(w.y, factor), rebase4(w.z, factor), rebase4(w.w, factor)};
}

// One segment of one kv head: N rows at most (1 or 16), n of them, from row r, the first at kept row
// `row0`.
template <bool XBF16, bool KEPT8, bool HALVES, int N>
TS_DEV void append_segment(const AppendParams &p, uint32_t r, uint32_t n, uint64_t row0, uint32_t pos, uint32_t h,
                           uint32_t lane) {
    float ka[N], kb[N], va[N], vb[N];
    float2 cs[N];
#pragma unroll
    for (int i = 0; i < N; i++) {
        const size_t row = r + min((uint32_t)i, n - 1);  // past the end: read, not used
        load_pair<XBF16, HALVES>(p.k, row * p.k_stride + h * 128, lane, ka[i], kb[i]);
        load_pair<XBF16, HALVES>(p.v, row * p.v_stride + h * 128, lane, va[i], vb[i]);
        if (p.turns) cs[i] = p.turns[(size_t)(pos + min((uint32_t)i, n - 1)) * 64 + lane];
    }
    if (p.k_gain) {
        const float ga = p.k_gain[HALVES ? lane : 2 * lane], gb = p.k_gain[HALVES ? lane + 64 : 2 * lane + 1];
#pragma unroll
        for (int i = 0; i < N; i++) norm_pair(ka[i], kb[i], ga, gb, p.eps);
    }
    if (p.turns) {
#pragma unroll
        for (int i = 0; i < N; i++) turn_pair(ka[i], kb[i], cs[i]);
    }
    if (!KEPT8) {
#pragma unroll
        for (int i = 0; i < N; i++) {
            if ((uint32_t)i >= n) continue;
            const size_t at = ((row0 + i) * p.kv_heads + h) * 128;
            store_pair_bf16<HALVES>((uint16_t *)p.k_kept + at, lane, ka[i], kb[i]);
            store_pair_bf16<HALVES>((uint16_t *)p.v_kept + at, lane, va[i], vb[i]);
        }
        return;
    }
    float ak = 0.0f, av = 0.0f;
#pragma unroll
    for (int i = 0; i < N; i++) {  // rows past the end repeat the last one
        ak = fmaxf(ak, fmaxf(finite_abs(ka[i]), finite_abs(kb[i])));
        av = fmaxf(av, fmaxf(finite_abs(va[i]), finite_abs(vb[i])));
    }
    ak = wave_max(ak);
    av = wave_max(av);
    const uint32_t off = (uint32_t)(row0 & (kBlock - 1));
    const uint64_t block = row0 / kBlock;
    float2 *scale_at = (float2 *)p.scales + block * scale_heads(p.kv_heads) + h;
    int ek = scale_exponent(ak), ev = scale_exponent(av), wask = ek, wasv = ev;
    if (off) {  // rows are there: the scale only grows
        const float2 was = *scale_at;
        wask = stored_exponent(was.x);
        wasv = stored_exponent(was.y);
        ek = max(ek, wask);
        ev = max(ev, wasv);
    }
    const float ik = two_to(-ek), iv = two_to(-ev);
    uint8_t *kb8 = (uint8_t *)p.k_kept + (block * p.kv_heads + h) * kBlockBytes;
    uint8_t *vb8 = (uint8_t *)p.v_kept + (block * p.kv_heads + h) * kBlockBytes;
    if (off && ek > wask) {  // four lanes a row of K: the rows not written now move to the new scale
        const uint32_t row = lane >> 2;
        if (row < off || row >= off + n) {
            u32x4 *at = (u32x4 *)(kb8 + lane * 32);
            const u32x4 w0 = at[0], w1 = at[1];
            const float factor = two_to(wask - ek > -126 ? wask - ek : -126);
            at[0] = rebase16(w0, factor);
            at[1] = rebase16(w1, factor);
        }
    }
#pragma unroll
    for (int i = 0; i < N; i++) {
        if ((uint32_t)i >= n) continue;
        uint8_t *at = kb8 + (off + i) * kWidth;
        const int w = __builtin_amdgcn_cvt_pk_fp8_f32(coded(ka[i], ik), coded(kb[i], ik), 0, false);
        if (HALVES) {
            at[lane] = (uint8_t)w;
            at[lane + 64] = (uint8_t)(w >> 8);
        } else {
            *(uint16_t *)(at + 2 * lane) = (uint16_t)w;
        }
    }
    // V: 16 positions of a d are one 16-byte piece; the lane's two.
    typedef unsigned __int128 u128;
    const u128 ones = ~(u128)0;
    const u128 mask = (n == kBlock ? ones : (((u128)1 << (8 * n)) - 1)) << (8 * off);
    const float fv = two_to(wasv - ev > -126 ? wasv - ev : -126);
#pragma unroll
    for (int e = 0; e < 2; e++) {
        u128 fresh = 0;
#pragma unroll
        for (int i = 0; i < N; i++)
            fresh |= (u128)code_of(coded(e ? vb[i] : va[i], iv)) << (8 * i);
        u128 *at = (u128 *)(vb8 + (HALVES ? lane + 64 * e : 2 * lane + e) * kBlock);
        u128 all = fresh << (8 * off);
        if (n < kBlock) {
            u32x4 held = *(const u32x4 *)at;
            if (off && ev > wasv) held = rebase16(held, fv);
            all = (all & mask) | (__builtin_bit_cast(u128, held) & ~mask);
        }
        *(u32x4 *)at = __builtin_bit_cast(u32x4, all);
    }
    if (lane == 0) *scale_at = make_float2(two_to(ek), two_to(ev));
}

template <bool XBF16, bool KEPT8, bool HALVES>
__global__ __launch_bounds__(256) void append_kernel(AppendParams p) {
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    if (blockIdx.x >= p.kv_groups) {  // q heads of one row
        const uint32_t g = blockIdx.x - p.kv_groups, r = g / p.head_groups;
        const uint32_t h0 = (g % p.head_groups) * 4 * kQBatch + wave;
        if (h0 >= p.heads) return;
        const uint32_t pos = p.positions[r];
        const bool held = pos < p.place.keys;
        float a[kQBatch], b[kQBatch];
#pragma unroll
        for (uint32_t i = 0; i < kQBatch; i++)  // past the end: read, not used
            load_pair<XBF16, HALVES>(p.q, (size_t)r * p.q_stride + min(h0 + 4 * i, p.heads - 1) * 128, lane, a[i], b[i]);
        float2 cs = make_float2(1.0f, 0.0f);
        if (p.turns && held) cs = p.turns[(size_t)pos * 64 + lane];
        float ga = 1.0f, gb = 1.0f;
        if (p.q_gain) {
            ga = p.q_gain[HALVES ? lane : 2 * lane];
            gb = p.q_gain[HALVES ? lane + 64 : 2 * lane + 1];
        }
#pragma unroll
        for (uint32_t i = 0; i < kQBatch; i++) {
            const uint32_t h = h0 + 4 * i;
            if (h >= p.heads) break;
            if (p.q_gain) norm_pair(a[i], b[i], ga, gb, p.eps);
            if (p.turns) turn_pair(a[i], b[i], cs);
            if (!held) a[i] = b[i] = __builtin_nanf("");
            const size_t at = ((size_t)r * p.heads + h) * 128;
            if (p.q_out_bf16) {
                store_pair_bf16<HALVES>((uint16_t *)p.q_out + at, lane, a[i], b[i]);
            } else {
                float *o = (float *)p.q_out + at;
                if (HALVES) {
                    o[lane] = a[i];
                    o[lane + 64] = b[i];
                } else {
                    *(float2 *)(o + 2 * lane) = make_float2(a[i], b[i]);
                }
            }
        }
        return;
    }
    // k and v: the segments that begin among the window's rows, a wave a kv head.
    const uint32_t groups = (p.kv_heads + 3) / 4, h = blockIdx.x % groups * 4 + wave;
    const uint32_t w0 = blockIdx.x / groups * p.window;
    // Lane i looks at row w0 + i: a segment begins where the row does not go on from the one before
    // it, or begins a block.
    bool begins = false;
    if (lane < p.window && w0 + lane < p.rows) {
        const uint32_t r = w0 + lane, pos = p.positions[r];
        begins = r == 0 || (pos & (kBlock - 1)) == 0 || p.slots[r - 1] != p.slots[r] || p.positions[r - 1] + 1 != pos;
    }
    uint64_t todo = __builtin_amdgcn_ballot_w64(begins);
    while (todo) {
        const uint32_t r = w0 + __builtin_ctzll(todo);
        todo &= todo - 1;
        const uint32_t slot = __builtin_amdgcn_readfirstlane(p.slots[r]);
        const uint32_t pos = __builtin_amdgcn_readfirstlane(p.positions[r]);
        bool on = false;  // lane i: row r + i belongs to the segment
        if (lane < kBlock && r + lane < p.rows)
            on = p.slots[r + lane] == slot && p.positions[r + lane] == pos + lane && (pos & (kBlock - 1)) + lane < kBlock;
        const uint32_t count = __builtin_ctzll(~__builtin_amdgcn_ballot_w64(on));
        // Rows that a slot cannot hold: nothing is kept of them.
        uint32_t n = holds(p.place, slot, pos) ? min(count, p.place.keys - pos) : 0;
        uint32_t bad = n < count ? TS_STATUS_POSITION : 0;
        uint64_t row0 = 0;
        if (n && !row_of(p.place, slot, pos, row0)) {
            bad |= TS_STATUS_PAGE;
            n = 0;
        }
        if (slot >= p.place.slot_count) bad = TS_STATUS_PAGE;
        // A segment of the same block before this one in the call: the two would race.
        bool twice = false;
        for (uint32_t j = threadIdx.x; j < r; j += 256)
            twice |= p.slots[j] == slot && p.positions[j] / kBlock == pos / kBlock;
        if (__syncthreads_or(twice)) {
            bad |= TS_STATUS_TWICE;
            n = 0;
        }
        if (bad && p.status && threadIdx.x == 0) atomicOr(p.status, bad);
        if (n == 0 || h >= p.kv_heads) continue;
        if (n == 1)
            append_segment<XBF16, KEPT8, HALVES, 1>(p, r, n, row0, pos, h, lane);
        else
            append_segment<XBF16, KEPT8, HALVES, 16>(p, r, n, row0, pos, h, lane);
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
    TS_REQUIRE(a && a->k && a->v && a->k_kept && a->v_kept && a->slots && a->positions, "append_rows: null pointer");
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
    TS_REQUIRE(ts::aligned(a->k, 16) && ts::aligned(a->v, 16) && ts::aligned(a->k_kept, 16) && ts::aligned(a->v_kept, 16) &&
                   ts::aligned(a->scales, 16) && ts::aligned(a->rope_table, 8),
               "append_rows: k, v, kept rows and scales must be 16-byte aligned, the angle table 8");
    const bool q = a->q != nullptr;
    if (q) {
        TS_REQUIRE(a->q_out, "append_rows: q without q_out");
        TS_REQUIRE(a->heads >= 1 && a->heads <= 16384, "append_rows: %u heads", a->heads);
        TS_REQUIRE(a->q_stride >= a->heads * 128 && a->q_stride % unit == 0,
                   "append_rows: q rows %u apart must hold %u heads and be whole 16-byte pieces", a->q_stride, a->heads);
        TS_REQUIRE(a->q_out_dtype == TS_F32 || a->q_out_dtype == TS_BF16, "append_rows: q out f32 or bf16 supported");
        TS_REQUIRE(ts::aligned(a->q, 16) && ts::aligned(a->q_out, 16), "append_rows: q must be 16-byte aligned");
        TS_REQUIRE(a->q_out != a->q || (a->q_out_dtype == a->x_dtype && a->q_stride == a->heads * 128),
                   "append_rows: q in place needs rows back to back of the same type");
    }
    if (a->rows == 0) return TS_OK;
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
    // Few rows are taken for a decode step, a segment each: a group looks at one row. Of many, most
    // go on from the row before them, and a group looks at 16.
    p.window = a->rows <= 1024 ? 1 : 16;
    const uint64_t kv = (uint64_t)((a->rows + p.window - 1) / p.window) * ((a->kv_heads + 3) / 4);
    p.head_groups = (a->heads + 4 * kQBatch - 1) / (4 * kQBatch);
    const uint64_t all = kv + (q ? (uint64_t)a->rows * p.head_groups : 0);
    TS_REQUIRE(all <= 0x7fffffffull, "append_rows: %u rows in one launch", a->rows);
    p.kv_groups = (uint32_t)kv;
    const int pick = (a->x_dtype == TS_BF16 ? 4 : 0) | (blocks ? 2 : 0) | (a->halves ? 1 : 0);
    void (*const kernels[8])(AppendParams) = {
        append_kernel<false, false, false>, append_kernel<false, false, true>, append_kernel<false, true, false>,
        append_kernel<false, true, true>,   append_kernel<true, false, false>, append_kernel<true, false, true>,
        append_kernel<true, true, false>,   append_kernel<true, true, true>};
    hipLaunchKernelGGL(kernels[pick], dim3((uint32_t)all), dim3(256), 0, (hipStream_t)stream, p);
    TS_CHECK_LAUNCH("append_rows launch");
    return TS_OK;
}
