// A product a head: out[r, h, n] = sum_k x[r, h, k] w[h, n, k] (q into a latent space, latent sums out of it).
//
// 2 n k flops against 2 (n + k) bytes of x and out: at k or n of 128 at most 128 flops a byte, a fifth of what the
// matrix unit needs for each byte from HBM, so bytes bound it (few rows: the weights'). A chunk of 64 k of a group's rows
// of x and w, 128 or 256 bytes of each, goes straight to LDS, one or two chunks ahead of the products: reads of whole lines, where
// operands taken from memory as they lie (32 rows, 32 bytes of each) were bound by the vector cache's tags.
// 1024 rows of 32 heads, 512 -> 128 to f32: 13.5 us, 4.0 TB/s (from memory to registers 27.5 us); 32 rows of 128 heads,
// 128 -> 512: 5.5 us, 4.0 TB/s (7.6 us); 8192 rows of 16 heads, 512 -> 128: 34 us, 6.0 TB/s. What is left is the start
// of each group, before its first chunk has come, and its end; f32 rows are bound by three products for one and the vector work before them (24 us, 3.7 TB/s).
#include <algorithm>

#include "common.h"
#include "places.h"

namespace {

constexpr uint32_t kChunk = 64;

struct HeadsParams {
    const void *x;
    const uint16_t *w;
    void *out;
    uint32_t rows, n, k, x_stride, x_head, out_stride, out_head;
    uint64_t w_head;
    uint32_t row_tiles, col_tiles, groups;
    int out_bf16, fours;  // fours: four columns of out are one aligned store
};

// Three bf16 parts of f32 values that add up to them: the upper 8 bits of what is left each time. (Nothing is left
// of an infinity, and NaN stays NaN.)
TS_DEV void split8(const f32x4 &a, const f32x4 &b, bf16x8 (&to)[3]) {
    u32x4 w[3];
    auto rest = [](float x, float part) { return x == part ? 0.0f : x - part; };
#pragma unroll
    for (int i = 0; i < 4; i++) {
        float lo = i < 2 ? a[2 * i] : b[2 * i - 4], hi = i < 2 ? a[2 * i + 1] : b[2 * i - 3];
#pragma unroll
        for (int e = 0; e < 3; e++) {
            const uint32_t pair = __builtin_amdgcn_perm(__float_as_uint(hi), __float_as_uint(lo), 0x07060302u);
            w[e][i] = pair;
            lo = rest(lo, lo_bf16(pair));
            hi = rest(hi, hi_bf16(pair));
        }
    }
#pragma unroll
    for (int e = 0; e < 3; e++) to[e] = as_bf16x8(w[e]);
}

// 16 bytes a lane from `from` straight to LDS, where the lane lands at `lds` + 16 lane. Nothing but LDS (and m0) is
// written, and only the caller's own waits (vmcnt) and barrier tell when. (Beside the builtin's loads the compiler waits
// for all of them before any read of LDS.)
TS_DEV void row_to_lds16(const char *from, uint32_t lds) {
#ifdef __HIP_DEVICE_COMPILE__
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(lds), "v"(from) : "memory");
#endif
}

// NW waves along the columns, 32 MN each, and RW along the rows, 32 MT each.
template <bool XBF16, uint32_t NW, uint32_t RW, uint32_t MT, uint32_t MN>
struct Tile {
    static constexpr uint32_t kWaves = NW * RW, kThreads = 64 * kWaves, kRows = 32 * MT * RW, kCols = 32 * MN * NW;
    static constexpr uint32_t kXRow = kChunk * (XBF16 ? 2 : 4), kWRow = kChunk * 2;
    static constexpr uint32_t kX = kRows * kXRow, kStage = kX + kCols * kWRow;
    static constexpr uint32_t kXLoads = kX / 1024 / kWaves, kWLoads = kCols * kWRow / 1024 / kWaves;  // a wave's
    static constexpr uint32_t kStages = NW == 2 && MN == 2 ? 2 : 3;  // chunks in LDS: two of the largest leave a CU two groups
    static constexpr uint32_t kOutRow = kCols * 4 + 16, kOut = kRows * kOutRow;
    static_assert(kX % (1024 * kWaves) == 0 && kCols * kWRow % (1024 * kWaves) == 0, "equal loads for all waves");
};

template <bool XBF16, uint32_t NW, uint32_t RW, uint32_t MT, uint32_t MN>
__global__ __launch_bounds__(64 * NW * RW, 2) void linear_heads_kernel(HeadsParams p) {
    using T = Tile<XBF16, NW, RW, MT, MN>;
    constexpr uint32_t kWaves = T::kWaves;
    extern __shared__ __attribute__((aligned(16))) char stage[];
    __shared__ uint32_t odd_met[XBF16 ? 1 : kWaves];
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const uint32_t col = lane & 31, half = lane >> 5;
    // Groups go to the eight XCDs in turn: those of a head, which read the same x or w, belong to one.
    uint32_t u = (blockIdx.x & 7) * ((p.groups + 7) / 8) + (blockIdx.x >> 3);
    if (u >= p.groups) return;
    const uint32_t n0 = u % p.col_tiles * T::kCols;
    u /= p.col_tiles;
    const uint32_t r0 = u % p.row_tiles * T::kRows, h = u / p.row_tiles;

    // LDS holds a chunk's rows back to back, their pieces of 16 bytes permuted by an XOR that has the 16 lanes of a read,
    // one piece of 16 rows, meet all banks. Rows and columns past the last are the last again, and are not stored.
    auto swap_w = [](uint32_t row) { return row >> 1 & 7; };
    auto swap_x = [](uint32_t row) { return XBF16 ? row >> 1 & 7 : row & 15; };
    const char *x[T::kXLoads], *w[T::kWLoads];
    uint32_t x_k[T::kXLoads], w_k[T::kWLoads];  // the first k of the lane's piece
#pragma unroll
    for (uint32_t i = 0; i < T::kXLoads; i++) {
        const uint32_t at = (wave + i * kWaves) * 64 + lane, row = at / (T::kXRow / 16);
        x_k[i] = (at % (T::kXRow / 16) ^ swap_x(row)) * (XBF16 ? 8 : 4);
        x[i] = (const char *)p.x + ((uint64_t)min(r0 + row, p.rows - 1) * p.x_stride + (uint64_t)h * p.x_head) * (XBF16 ? 2 : 4);
    }
#pragma unroll
    for (uint32_t i = 0; i < T::kWLoads; i++) {
        const uint32_t at = (wave + i * kWaves) * 64 + lane, row = at / 8;
        w_k[i] = (at % 8 ^ swap_w(row)) * 8;
        w[i] = (const char *)(p.w + h * p.w_head + (uint64_t)min(n0 + row, p.n - 1) * p.k);
    }
    // (Pieces past the last k are the row's first, and zero in the products.)
    auto issue = [&](uint32_t k0, uint32_t to) {
        const uint32_t lds = (uint32_t)(uintptr_t)(ts_lds *)stage + to * T::kStage + wave * 1024;
#pragma unroll
        for (uint32_t i = 0; i < T::kXLoads; i++)
            row_to_lds16(x[i] + (k0 + x_k[i] < p.k ? (k0 + x_k[i]) * (XBF16 ? 2 : 4) : 0), lds + i * (kWaves * 1024));
#pragma unroll
        for (uint32_t i = 0; i < T::kWLoads; i++)
            row_to_lds16(w[i] + (k0 + w_k[i] < p.k ? (k0 + w_k[i]) * 2 : 0), lds + T::kX + i * (kWaves * 1024));
    };

    f32x16 acc[MT][MN];
#pragma unroll
    for (uint32_t m = 0; m < MT; m++)
#pragma unroll
        for (uint32_t j = 0; j < MN; j++)
#pragma unroll
            for (int i = 0; i < 16; i++) acc[m][j][i] = 0.0f;
    const uint32_t n1 = wave % NW * (32 * MN), r1 = wave / NW * (32 * MT);
    // Four steps of 16 k: the lane has the eight of its half of column `col` of w (the left operand) and of row `col` of x.
    auto products = [&](const char *at, uint32_t left) {
        const uint32_t row_w = n1 + col, row_x = r1 + col;  // (32 more rows have the same XOR)
#pragma unroll
        for (uint32_t s = 0; s < kChunk / 16; s++) {
            if (16 * s >= left) break;
            const uint32_t keep = 16 * s + 8 * half < left ? 0xffffffffu : 0u, piece = 2 * s + half;
            bf16x8 a[MN];
#pragma unroll
            for (uint32_t j = 0; j < MN; j++)
                a[j] = as_bf16x8(*(const u32x4 *)(at + T::kX + (row_w + 32 * j) * T::kWRow + (piece ^ swap_w(row_w)) * 16) & keep);
#pragma unroll
            for (uint32_t m = 0; m < MT; m++) {
                const char *row = at + (row_x + 32 * m) * T::kXRow;
                bf16x8 part[XBF16 ? 1 : 3];
                if constexpr (XBF16)
                    part[0] = as_bf16x8(*(const u32x4 *)(row + (piece ^ swap_x(row_x)) * 16) & keep);
                else
                    split8(__builtin_bit_cast(f32x4, *(const u32x4 *)(row + (2 * piece ^ swap_x(row_x)) * 16) & keep),
                           __builtin_bit_cast(f32x4, *(const u32x4 *)(row + ((2 * piece + 1) ^ swap_x(row_x)) * 16) & keep), part);
#pragma unroll
                for (uint32_t e = 0; e < (XBF16 ? 1 : 3); e++)
#pragma unroll
                    for (uint32_t j = 0; j < MN; j++) acc[m][j] = mfma32(a[j], part[e], acc[m][j]);
            }
        }
    };
    constexpr uint32_t kLoads = T::kXLoads + T::kWLoads;
    issue(0, 0);
    if (T::kStages == 3 && kChunk < p.k) issue(kChunk, 1);
    uint32_t now = 0;
    for (uint32_t k0 = 0; k0 < p.k; k0 += kChunk) {
        if (T::kStages == 3 && k0 + kChunk < p.k)
            asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(kLoads) : "memory");
        else
            asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
        const uint32_t next = k0 + (T::kStages - 1) * kChunk;
        if (next < p.k) issue(next, now ? now - 1 : T::kStages - 1);
        if (n0 + n1 < p.n) {
            if (k0 + kChunk <= p.k)
                products(stage + now * T::kStage, kChunk);
            else
                products(stage + now * T::kStage, p.k - k0);
        }
        now = now + 1 == T::kStages ? 0 : now + 1;
    }
    // Sums change places in LDS, so that a store has whole rows' columns: register 4 q + i of a lane is column
    // 8 q + 4 half + i of row `col`.
    if (!XBF16) {
        float odd = 0.0f;  // NaN where a sum is not finite
#pragma unroll
        for (uint32_t m = 0; m < MT; m++)
#pragma unroll
            for (uint32_t j = 0; j < MN; j++)
#pragma unroll
                for (int i = 0; i < 16; i++) odd = fmaf(acc[m][j][i], 0.0f, odd);
        odd_met[wave] = __builtin_amdgcn_ballot_w64(odd != odd) != 0;
    }
    lds_barrier();
#pragma unroll
    for (uint32_t m = 0; m < MT; m++)
#pragma unroll
        for (uint32_t q = 0; q < 4 * MN; q++) {
            const f32x16 &v = acc[m][q / 4];
            *(f32x4 *)(stage + (r1 + 32 * m + col) * T::kOutRow + (n1 + 8 * q + 4 * half) * 4) =
                f32x4{v[q % 4 * 4], v[q % 4 * 4 + 1], v[q % 4 * 4 + 2], v[q % 4 * 4 + 3]};
        }
    lds_barrier();
    const uint64_t out = (uint64_t)h * p.out_head + n0;
    if (p.fours) {
#pragma unroll 4
        for (uint32_t e = threadIdx.x; e < T::kRows * T::kCols / 4; e += T::kThreads) {
            const uint32_t row = e / (T::kCols / 4), n = e % (T::kCols / 4) * 4;
            if (r0 + row >= p.rows || n0 + n >= p.n) continue;
            const f32x4 v = *(const f32x4 *)(stage + row * T::kOutRow + n * 4);
            const uint64_t at = out + (uint64_t)(r0 + row) * p.out_stride + n;
            if (p.out_bf16)
                *(u32x2 *)((uint16_t *)p.out + at) = u32x2{pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3])};
            else
                *(f32x4 *)((float *)p.out + at) = v;
        }
    } else {
        for (uint32_t e = threadIdx.x; e < T::kRows * T::kCols; e += T::kThreads) {
            const uint32_t row = e / T::kCols, n = e % T::kCols;
            if (r0 + row >= p.rows || n0 + n >= p.n) continue;
            const float v = *(const float *)(stage + row * T::kOutRow + n * 4);
            const uint64_t at = out + (uint64_t)(r0 + row) * p.out_stride + n;
            if (p.out_bf16)
                ((uint16_t *)p.out)[at] = bf16_bits(v);
            else
                ((float *)p.out)[at] = v;
        }
    }
    if (XBF16) return;
    // A sum of parts may be NaN only because one of them is 0 and its weight infinite: those are summed anew, of whole values.
    uint32_t any = 0;
#pragma unroll
    for (uint32_t i = 0; i < kWaves; i++) any |= __builtin_amdgcn_readfirstlane(odd_met[i]);
    if (!any) return;
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // the stores of the same places
    lds_barrier();
#pragma unroll 1
    for (uint32_t e = threadIdx.x; e < T::kRows * T::kCols; e += T::kThreads) {
        const uint32_t row = e / T::kCols, n = e % T::kCols;
        if (r0 + row >= p.rows || n0 + n >= p.n) continue;
        float v = *(const float *)(stage + row * T::kOutRow + n * 4);
        if (v == v) continue;
        const float *a = (const float *)p.x + (uint64_t)(r0 + row) * p.x_stride + (uint64_t)h * p.x_head;
        const uint16_t *b = p.w + h * p.w_head + (uint64_t)(n0 + n) * p.k;
        v = 0.0f;
#pragma unroll 1
        for (uint32_t k = 0; k < p.k && v == v; k++) v = fmaf(a[k], lo_bf16(b[k]), v);
        const uint64_t at = out + (uint64_t)(r0 + row) * p.out_stride + n;
        if (p.out_bf16)
            ((uint16_t *)p.out)[at] = bf16_bits(v);
        else
            ((float *)p.out)[at] = v;
    }
}

int out_apart(const ts_heads_args *a) {
    const uint64_t x = a->x_dtype == TS_F32 ? 4 : 2, out = a->out_dtype == TS_F32 ? 4 : 2;
    return ts::outputs_apart("linear_heads",
                             {{"out", a->out, a->n * out, a->rows, a->out_stride * out, a->heads, a->out_head * out}},
                             {{"x", a->x, a->k * x, a->rows, a->x_stride * x, a->heads, a->x_head * x},
                              {"w", a->w, 2ull * a->n * a->k, a->heads, 2ull * a->w_head}});
}

template <bool XBF16, uint32_t NW, uint32_t RW, uint32_t MT, uint32_t MN>
int launch(HeadsParams &p, const ts_heads_args *a, void *stream) {
    using T = Tile<XBF16, NW, RW, MT, MN>;
    const auto kernel = linear_heads_kernel<XBF16, NW, RW, MT, MN>;
    constexpr uint32_t kMost = std::max(T::kStages * T::kStage, T::kOut);
    p.row_tiles = (p.rows - 1) / T::kRows + 1;
    p.col_tiles = (p.n - 1) / T::kCols + 1;
    const uint64_t all = (uint64_t)p.row_tiles * p.col_tiles * a->heads;
    TS_REQUIRE(all < (1ull << 32) / T::kThreads - 8, "linear_heads: %u rows in one launch", p.rows);
    const int rc = out_apart(a);
    if (rc) return rc;
    p.groups = (uint32_t)all;
    static const hipError_t attr =
        hipFuncSetAttribute((const void *)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, kMost);
    if (attr != hipSuccess) return ts::hip_status(attr, "linear_heads: shared memory attribute");
    const uint32_t stages = std::min(T::kStages, (p.k - 1) / kChunk + 1);  // (fewer: more groups a CU)
    hipLaunchKernelGGL(kernel, dim3((p.groups + 7) / 8 * 8), dim3(T::kThreads), std::max(stages * T::kStage, T::kOut),
                       (hipStream_t)stream, p);
    TS_CHECK_LAUNCH("linear_heads launch");
    return TS_OK;
}

}  // namespace

extern "C" int tessera_hip_linear_heads(const ts_heads_args *a, void *stream) {
    TS_REQUIRE(a, "linear_heads: null args");
    TS_REQUIRE(a->w && (a->rows == 0 || (a->x && a->out)), "linear_heads: null pointer");
    TS_REQUIRE(a->x_dtype == TS_F32 || a->x_dtype == TS_BF16, "linear_heads: x f32 or bf16 supported");
    TS_REQUIRE(a->out_dtype == TS_F32 || a->out_dtype == TS_BF16, "linear_heads: out f32 or bf16 supported");
    TS_REQUIRE(a->heads >= 1 && a->heads <= 16384, "linear_heads: %u heads", a->heads);
    TS_REQUIRE(a->n >= 1 && a->n <= 1u << 20, "linear_heads: n %u", a->n);
    TS_REQUIRE(a->k >= 8 && a->k % 8 == 0 && a->k <= 1u << 20, "linear_heads: k %u must be a multiple of 8", a->k);
    const uint32_t unit = a->x_dtype == TS_F32 ? 4 : 8;  // 16 bytes
    TS_REQUIRE(a->x_stride % unit == 0 && a->x_head % unit == 0 && a->w_head % 8 == 0,
               "linear_heads: x's rows and heads and w's heads must be whole 16-byte pieces apart");
    TS_REQUIRE(a->heads == 1 || a->w_head >= (uint64_t)a->n * a->k, "linear_heads: heads of w %llu apart",
               (unsigned long long)a->w_head);
    TS_REQUIRE(ts::beside(a->rows, a->out_stride, a->heads, a->out_head, a->n),
               "linear_heads: out's rows %u and heads %u apart meet", a->out_stride, a->out_head);
    TS_REQUIRE(ts::aligned(a->x, 16) && ts::aligned(a->w, 16), "linear_heads: x and w must be 16-byte aligned");
    const uint32_t size = a->out_dtype == TS_F32 ? 4 : 2;
    TS_REQUIRE(ts::aligned(a->out, size), "linear_heads: out must be aligned to its type");
    if (a->rows == 0) return TS_OK;
    HeadsParams p;
    p.x = a->x; p.w = (const uint16_t *)a->w; p.out = a->out;
    p.rows = a->rows; p.n = a->n; p.k = a->k;
    p.x_stride = a->x_stride; p.x_head = a->x_head; p.out_stride = a->out_stride; p.out_head = a->out_head;
    p.w_head = a->w_head;
    p.out_bf16 = a->out_dtype == TS_BF16;
    p.fours = a->n % 4 == 0 && a->out_stride % 4 == 0 && a->out_head % 4 == 0 && ts::aligned(a->out, 4 * size);
    const bool bf16 = a->x_dtype == TS_BF16;
    // Up to 64 rows a tile has 32 of them and more groups share the chip (33 rows, 128 heads, 512 -> 128: 6.7 us against 7.8
    // with 64 rows; 64 rows of f32 14.0 against 19.4; but 1024 rows of 32 heads 16.0 against 13.5), and 64 columns where
    // 128 would leave CUs without a group (1 row, 16 heads, 128 -> 512: 3.9 us against 4.6).
    if (a->rows <= 64) {
        if ((uint64_t)a->heads * ((a->n - 1) / 128 + 1) * ((a->rows - 1) / 32 + 1) < 256)
            return bf16 ? launch<true, 2, 1, 1, 1>(p, a, stream) : launch<false, 2, 1, 1, 1>(p, a, stream);
        return bf16 ? launch<true, 4, 1, 1, 1>(p, a, stream) : launch<false, 4, 1, 1, 1>(p, a, stream);
    }
    // 64 columns have a tile of their own (1000 rows of 16 heads, 256 -> 64: 5.3 us against 6.2).
    if (a->n <= 64) return bf16 ? launch<true, 2, 2, 1, 1>(p, a, stream) : launch<false, 1, 4, 1, 2>(p, a, stream);
    // Many rows of bf16: 128 a tile, 64 x 64 a wave, two chunks in LDS (8192 rows of 16 heads, 512 -> 128: 34 us against 39 with 64
    // rows; 32000 rows, 640 -> 640: 46 against 53; but of one chunk, 2000 rows of 16 heads, 8 -> 640: 19 against 17).
    if (bf16 && a->k > kChunk && (uint64_t)a->heads * ((a->n - 1) / 128 + 1) * ((a->rows - 1) / 128 + 1) >= 1024)
        return launch<true, 2, 2, 2, 2>(p, a, stream);
    // f32 rows are taken apart by each wave that reads them, and are twice the bytes in LDS: two waves along the columns and
    // two chunks (1024 rows of 32 heads, 512 -> 128: 23.6 us; one wave along them and a group a CU 24.8, four 29.5).
    return bf16 ? launch<true, 4, 1, 2, 1>(p, a, stream) : launch<false, 2, 2, 1, 2>(p, a, stream);
}
