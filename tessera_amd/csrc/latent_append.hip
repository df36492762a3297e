// New rows of latent attention into their kept rows: RmsNorm of the latent, rotation of the shared key part,
// and the rotation of q's part of it.
//
//   kept[row] = bf16(c[: rank] / sqrt(mean(c[: rank]^2) + eps) * gain | rot(c[rank :])),  q_out = rot(q)
//
// A wave takes one row of c, or the q parts of one row that 64 lanes hold at eight values each (eight heads of
// 64). A lane's eight values are neighbours, whole 16-byte pieces of every tensor: pairs (2j, 2j + 1) rotate
// within it, pairs (j, j + rope / 2) with the lane rope / 16 further. Waves are many and their loads independent
// but for the row's place, so nothing is kept in LDS and no wave waits for another. Bytes bound many rows: 12288 bf16 rows of
// 512 + 64 values with 16 heads' q parts in 16.6 us, 4.3 TB/s; few rows the chain of place, row, angles and store (one row
// 2.5 us, 128 f32 rows with 128 heads 4.7 us, 1.4 TB/s).
#include "kept8.h"
#include "places.h"

namespace {

using kept8::Place;

constexpr uint32_t kWaves = 4, kMostRank = 1024;

struct LatentRows {
    const void *c, *q;
    const float *gain, *turns;
    void *q_out, *kept, *c_out, *r_out;
    const uint32_t *slots, *positions;
    uint32_t *status;
    Place place;
    uint32_t rows, heads, rank, rope, c_stride, q_stride, q_head, q_out_stride, q_out_head;
    uint32_t c_groups;     // groups that take rows of c; the others q
    uint32_t head_shift;   // log2 of the heads a wave takes
    uint32_t head_units;   // waves a row's heads are
    float eps;
    int q_out_bf16;
};

template <bool BF16>
TS_DEV void load8(const void *from, uint64_t at, float (&v)[8]) {
    if (BF16) {
        const u32x4 w = *(const u32x4 *)((const uint16_t *)from + at);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            v[2 * i] = lo_bf16(w[i]);
            v[2 * i + 1] = hi_bf16(w[i]);
        }
    } else {
        const f32x4 a = *(const f32x4 *)((const float *)from + at), b = *(const f32x4 *)((const float *)from + at + 4);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            v[i] = a[i];
            v[4 + i] = b[i];
        }
    }
}
TS_DEV u32x4 as_bf16(const float (&v)[8]) {
    return u32x4{pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7])};
}
TS_DEV void store8(void *to, uint64_t at, bool bf16, const float (&v)[8]) {
    if (bf16) {
        *(u32x4 *)((uint16_t *)to + at) = as_bf16(v);
    } else {
        *(f32x4 *)((float *)to + at) = f32x4{v[0], v[1], v[2], v[3]};
        *(f32x4 *)((float *)to + at + 4) = f32x4{v[4], v[5], v[6], v[7]};
    }
}
TS_DEV void all_nan(float (&v)[8]) {
#pragma unroll
    for (int i = 0; i < 8; i++) v[i] = __builtin_nanf("");
}

// The angles of the lane's values, piece `l` of the rotated part: a (cos, sin) for each pair (2j, 2j + 1), or for
// each value of a half.
template <bool HALVES>
struct Turns {
    f32x4 cs[HALVES ? 4 : 2];
    TS_DEV void load(const float *row, uint32_t l, uint32_t rope) {
        const float *from = row + (HALVES ? (16 * l) & (rope - 1) : 8 * l);
#pragma unroll
        for (int i = 0; i < (HALVES ? 4 : 2); i++) cs[i] = *(const f32x4 *)(from + 4 * i);
    }
    // (By all lanes of a part together.)
    TS_DEV void turn(float (&v)[8], uint32_t l, uint32_t rope) const {
        if (!HALVES) {
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const float cos = cs[i / 2][2 * (i % 2)], sin = cs[i / 2][2 * (i % 2) + 1], a = v[2 * i], b = v[2 * i + 1];
                v[2 * i] = a * cos - b * sin;
                v[2 * i + 1] = a * sin + b * cos;
            }
        } else {
            const bool second = 16 * l >= rope;
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const float cos = cs[i / 2][2 * (i % 2)], sin = cs[i / 2][2 * (i % 2) + 1];
                const float other = __shfl_xor(v[i], (int)(rope >> 4), 64);
                v[i] = second ? other * sin + v[i] * cos : v[i] * cos - other * sin;
            }
        }
    }
};

template <bool XBF16, bool HALVES>
__global__ __launch_bounds__(64 * kWaves) void append_latent_kernel(LatentRows p) {
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    Turns<HALVES> turns;
    if (blockIdx.x >= p.c_groups) {
        const uint32_t u = (blockIdx.x - p.c_groups) * kWaves + wave, r = u / p.head_units;
        if (r >= p.rows) return;
        const uint32_t pieces = p.rope >> 3, l = lane & (pieces - 1);
        const uint32_t h = (u % p.head_units << p.head_shift) + lane / pieces;
        if (h >= p.heads) return;  // (a head's lanes together)
        float v[8];
        load8<XBF16>(p.q, (uint64_t)r * p.q_stride + (uint64_t)h * p.q_head + 8 * l, v);
        const uint32_t slot = p.slots[r], pos = p.positions[r];
        if (p.turns) {
            turns.load(p.turns + (pos < p.place.keys ? (uint64_t)pos * p.rope : 0), l, p.rope);
            turns.turn(v, l, p.rope);
        }
        uint64_t row;
        if (!holds(p.place, slot, pos) || !row_of(p.place, slot, pos, row)) all_nan(v);
        store8(p.q_out, (uint64_t)r * p.q_out_stride + (uint64_t)h * p.q_out_head + 8 * l, p.q_out_bf16, v);
        return;
    }
    const uint32_t r = blockIdx.x * kWaves + wave;
    if (r >= p.rows) return;
    constexpr uint32_t kPasses = kMostRank / 512;
    const uint64_t from = (uint64_t)r * p.c_stride;
    const bool turned = 8 * lane < p.rope;
    float v[kPasses][8], t[8];
#pragma unroll
    for (uint32_t i = 0; i < kPasses; i++) {
        const uint32_t d = 512 * i + 8 * lane;
        if (d < p.rank)
            load8<XBF16>(p.c, from + d, v[i]);
        else
#pragma unroll
            for (int k = 0; k < 8; k++) v[i][k] = 0.0f;
    }
    if (turned) load8<XBF16>(p.c, from + p.rank + 8 * lane, t);
    const uint32_t slot = p.slots[r], pos = p.positions[r];
    if (turned && p.turns) turns.load(p.turns + (pos < p.place.keys ? (uint64_t)pos * p.rope : 0), lane, p.rope);
    uint64_t row = 0;
    const bool fits = holds(p.place, slot, pos), held = fits && row_of(p.place, slot, pos, row);
    if (!held && p.status && lane == 0)
        atomicOr(p.status, fits || slot >= p.place.slot_count ? TS_STATUS_PAGE : TS_STATUS_POSITION);
    if (p.gain) {
        float sum = 0.0f;
#pragma unroll
        for (uint32_t i = 0; i < kPasses; i++)
#pragma unroll
            for (int k = 0; k < 8; k++) sum = fmaf(v[i][k], v[i][k], sum);
        sum = wave_sum(sum);
        float by = 1.0f / sqrtf(sum / (float)p.rank + p.eps);
        if (sum == INFINITY) {
            // Squares past f32's range: those of the values by 2^-72 hold, and half of it goes to the values (a root of 2^59 or
            // more takes what that makes subnormal to 0). A value that is infinite still makes the others 0 and itself NaN.
            sum = 0.0f;
#pragma unroll
            for (uint32_t i = 0; i < kPasses; i++)
#pragma unroll
                for (int k = 0; k < 8; k++) {
                    v[i][k] *= 0x1p-36f;
                    sum = fmaf(v[i][k] * 0x1p-36f, v[i][k] * 0x1p-36f, sum);
                }
            by = 0x1p-36f / sqrtf(wave_sum(sum) / (float)p.rank + p.eps * 0x1p-72f * 0x1p-72f);
        }
#pragma unroll
        for (uint32_t i = 0; i < kPasses; i++) {
            const uint32_t d = 512 * i + 8 * lane;
            if (d >= p.rank) continue;
            float g[8];
            load8<false>(p.gain, d, g);
#pragma unroll
            for (int k = 0; k < 8; k++) v[i][k] = v[i][k] * by * g[k];
        }
    }
    if (turned && p.turns) turns.turn(t, lane, p.rope);
    if (!held) {
#pragma unroll
        for (uint32_t i = 0; i < kPasses; i++) all_nan(v[i]);
        all_nan(t);
    }
    uint16_t *kept = (uint16_t *)p.kept + row * (p.rank + p.rope);
#pragma unroll
    for (uint32_t i = 0; i < kPasses; i++) {
        const uint32_t d = 512 * i + 8 * lane;
        if (d >= p.rank) continue;
        const u32x4 w = as_bf16(v[i]);
        if (held) *(u32x4 *)(kept + d) = w;
        if (p.c_out) *(u32x4 *)((uint16_t *)p.c_out + (uint64_t)r * p.rank + d) = w;
    }
    if (turned) {
        const u32x4 w = as_bf16(t);
        if (held) *(u32x4 *)(kept + p.rank + 8 * lane) = w;
        if (p.r_out) *(u32x4 *)((uint16_t *)p.r_out + (uint64_t)r * p.rope + 8 * lane) = w;
    }
}

}  // namespace

extern "C" int tessera_hip_append_latent(const ts_append_latent_args *a, void *stream) {
    TS_REQUIRE(a, "append_latent: null args");
    const bool some = a->rows != 0;  // (what has an element a row may be NULL without rows)
    TS_REQUIRE(a->kept && (!some || (a->c && a->slots && a->positions)), "append_latent: null pointer");
    TS_REQUIRE(a->rank >= 8 && a->rank % 8 == 0 && a->rank <= kMostRank, "append_latent: rank %u (a multiple of 8 up to %u)",
               a->rank, kMostRank);
    TS_REQUIRE(a->rope == 16 || a->rope == 32 || a->rope == 64 || a->rope == 128,
               "append_latent: %u rotated values (16, 32, 64 or 128)", a->rope);
    TS_REQUIRE(a->x_dtype == TS_F32 || a->x_dtype == TS_BF16, "append_latent: rows f32 or bf16 supported");
    int rc = ts::kept_check("append_latent", a->kept_table, a->page, a->keys, a->slot_count, a->kept_pages, a->pages, false);
    if (rc) return rc;
    TS_REQUIRE(!a->rope_table || a->rope_rows >= a->keys, "append_latent: positions up to %u but the angle table has %u rows",
               a->keys - 1, a->rope_rows);
    const uint32_t unit = a->x_dtype == TS_F32 ? 4 : 8;  // 16 bytes
    TS_REQUIRE(a->c_stride >= a->rank + a->rope && a->c_stride % unit == 0,
               "append_latent: rows %u apart must hold %u values and be whole 16-byte pieces", a->c_stride,
               a->rank + a->rope);
    TS_REQUIRE(ts::aligned(a->c, 16) && ts::aligned(a->kept, 16) && ts::aligned(a->gain, 16) && ts::aligned(a->rope_table, 16) &&
                   ts::aligned(a->c_out, 16) && ts::aligned(a->r_out, 16),
               "append_latent: rows, kept rows, gain and the angle table must be 16-byte aligned");
    const bool q = a->q != nullptr;
    if (q) {
        TS_REQUIRE(a->q_out || !some, "append_latent: q without q_out");
        TS_REQUIRE(a->heads >= 1 && a->heads <= 16384, "append_latent: %u heads", a->heads);
        TS_REQUIRE(a->q_out_dtype == TS_F32 || a->q_out_dtype == TS_BF16, "append_latent: q out f32 or bf16 supported");
        const uint32_t out_unit = a->q_out_dtype == TS_F32 ? 4 : 8;
        TS_REQUIRE(a->q_stride % unit == 0 && a->q_head % unit == 0 && a->q_out_stride % out_unit == 0 &&
                       a->q_out_head % out_unit == 0,
                   "append_latent: q's rows and heads must be whole 16-byte pieces apart");
        TS_REQUIRE(a->q_out_head >= a->rope || a->heads == 1, "append_latent: q out's heads %u apart", a->q_out_head);
        TS_REQUIRE(ts::beside(a->rows, a->q_out_stride, a->heads, a->q_out_head, a->rope),
                   "append_latent: q out's rows %u and heads %u apart meet", a->q_out_stride, a->q_out_head);
        TS_REQUIRE(ts::aligned(a->q, 16) && ts::aligned(a->q_out, 16), "append_latent: q must be 16-byte aligned");
        TS_REQUIRE(a->q_out != a->q || (a->q_out_dtype == a->x_dtype && a->q_stride == a->q_out_stride &&
                                        a->q_head == a->q_out_head),
                   "append_latent: q in place needs one layout and type");
    }
    if (!some) return TS_OK;
    LatentRows p;
    p.c = a->c; p.q = a->q; p.gain = a->gain; p.turns = a->rope_table;
    p.q_out = a->q_out; p.kept = a->kept; p.c_out = a->c_out; p.r_out = a->r_out;
    p.slots = a->slots; p.positions = a->positions; p.status = a->status;
    p.place.table = a->kept_table; p.place.keys = a->keys; p.place.slot_count = a->slot_count;
    p.place.kept_pages = a->kept_pages; p.place.page_shift = (uint32_t)__builtin_ctz(a->page);
    p.place.pages = a->pages;
    p.rows = a->rows; p.heads = a->heads; p.rank = a->rank; p.rope = a->rope;
    p.c_stride = a->c_stride; p.q_stride = a->q_stride; p.q_head = a->q_head;
    p.q_out_stride = a->q_out_stride; p.q_out_head = a->q_out_head;
    p.eps = a->eps; p.q_out_bf16 = a->q_out_dtype == TS_BF16;
    p.head_shift = 9 - (uint32_t)__builtin_ctz(a->rope);
    p.head_units = q ? (a->heads + (1u << p.head_shift) - 1) >> p.head_shift : 0;
    p.c_groups = (a->rows - 1) / kWaves + 1;
    const uint64_t all = p.c_groups + ((uint64_t)a->rows * p.head_units + kWaves - 1) / kWaves;
    TS_REQUIRE(all < (1ull << 32) / (64 * kWaves), "append_latent: %u rows in one launch", a->rows);
    const uint64_t size = a->x_dtype == TS_F32 ? 4 : 2, out = a->q_out_dtype == TS_F32 ? 4 : 2, width = a->rank + a->rope;
    const uint64_t held = a->kept_table ? (uint64_t)a->pages * a->page : (uint64_t)a->slot_count * a->keys;
    const uint32_t heads = q ? a->heads : 0;
    rc = ts::outputs_apart(
        "append_latent",
        {{"q_out", a->q_out, a->rope * out, a->rows, a->q_out_stride * out, heads, a->q_out_head * out},
         {"c_out", a->c_out, (uint64_t)a->rows * a->rank * 2},
         {"r_out", a->r_out, (uint64_t)a->rows * a->rope * 2},
         {"kept", a->kept, held * width * 2}},
        {{"c", a->c, width * size, a->rows, a->c_stride * size},
         {"q", a->q_out == a->q ? nullptr : a->q, a->rope * size, a->rows, a->q_stride * size, heads, a->q_head * size},
         {"gain", a->gain, (uint64_t)a->rank * 4},
         {"the angle table", a->rope_table, (uint64_t)a->rope_rows * a->rope * 4},
         {"slots", a->slots, (uint64_t)a->rows * 4},
         {"positions", a->positions, (uint64_t)a->rows * 4},
         {"the page table", a->kept_table, (uint64_t)a->slot_count * a->kept_pages * 4}});
    if (rc) return rc;
    const auto kernel = a->x_dtype == TS_BF16 ? a->halves ? append_latent_kernel<true, true> : append_latent_kernel<true, false>
                                              : a->halves ? append_latent_kernel<false, true> : append_latent_kernel<false, false>;
    hipLaunchKernelGGL(kernel, dim3((uint32_t)all), dim3(64 * kWaves), 0, (hipStream_t)stream, p);
    TS_CHECK_LAUNCH("append_latent launch");
    return TS_OK;
}
