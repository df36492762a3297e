// A product a head: out[r, h, n] = sum_k x[r, h, k] w[h, n, k] (q into a latent space, latent sums out of it).
//
// 2 n k flops against 2 (n + k) bytes of x and out: at k or n of 128 at most 128 flops a byte, a fifth of what the
// matrix unit needs for each byte from HBM, so bytes bound it (few rows: the weights') and operands go from memory
// to registers as they lie: a lane's 16 bytes are eight neighbouring k of one row of w (the left operand, 32
// columns of out) or of x (the right one, 32 rows of out). A wave has 32 columns and MT times 32 rows; the four
// waves of a group have neighbouring columns and the same rows, whose second to fourth reads the vector cache
// serves. Loads run a chunk of 64 k ahead of the matrix unit.
#include "common.h"

namespace {

constexpr uint32_t kWaves = 4, kSteps = 4;  // steps of 16 k a chunk

struct HeadsParams {
    const void *x;
    const uint16_t *w;
    void *out;
    uint32_t rows, heads, n, k, x_stride, x_head, out_stride, out_head;
    uint64_t w_head;
    uint32_t row_tiles, col_groups;
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

template <bool XBF16, int MT>
__global__ __launch_bounds__(64 * kWaves) void linear_heads_kernel(HeadsParams p) {
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const uint32_t col = lane & 31, half = lane >> 5;
    uint32_t u = blockIdx.x;
    const uint32_t cg = u % p.col_groups;
    u /= p.col_groups;
    const uint32_t h = u % p.heads, r0 = u / p.heads * (32 * MT);
    const uint32_t n0 = (cg * kWaves + wave) * 32;
    if (n0 >= p.n) return;
    // Rows and columns past the last are the last again, and are not stored.
    const uint16_t *w = p.w + h * p.w_head + (uint64_t)min(n0 + col, p.n - 1) * p.k + 8 * half;
    const char *x[MT];
#pragma unroll
    for (int m = 0; m < MT; m++)
        x[m] = (const char *)p.x + ((uint64_t)min(r0 + 32 * m + col, p.rows - 1) * p.x_stride +
                                    (uint64_t)h * p.x_head + 8 * half) * (XBF16 ? 2 : 4);
    struct Chunk {
        u32x4 w[kSteps];
        u32x4 x[MT][kSteps][XBF16 ? 1 : 2];
    };
    // Step j's k: 16 j + 8 half .. + 7, zero past the last.
    auto load = [&](uint32_t j0, Chunk &c) {
#pragma unroll
        for (uint32_t s = 0; s < kSteps; s++) {
            const uint32_t at = 16 * (j0 + s);
            const bool in = at + 8 * half < p.k;
            const uint32_t d = in ? at : 0;
            const uint32_t keep = in ? 0xffffffffu : 0u;
            c.w[s] = *(const u32x4 *)(w + (in ? d : 0)) & keep;
#pragma unroll
            for (int m = 0; m < MT; m++) {
                c.x[m][s][0] = *(const u32x4 *)(x[m] + d * (XBF16 ? 2 : 4)) & keep;
                if (!XBF16) c.x[m][s][XBF16 ? 0 : 1] = *(const u32x4 *)(x[m] + d * 4 + 16) & keep;
            }
        }
    };
    f32x16 acc[MT];
#pragma unroll
    for (int m = 0; m < MT; m++)
#pragma unroll
        for (int i = 0; i < 16; i++) acc[m][i] = 0.0f;
    const uint32_t steps = (p.k + 15) / 16;
    Chunk c, next;
    load(0, c);
    for (uint32_t j = 0;;) {
        const bool more = j + kSteps < steps;
        if (more) load(j + kSteps, next);
#pragma unroll
        for (uint32_t s = 0; s < kSteps; s++) {
            const bf16x8 a = as_bf16x8(c.w[s]);
#pragma unroll
            for (int m = 0; m < MT; m++) {
                if (XBF16) {
                    acc[m] = mfma32(a, as_bf16x8(c.x[m][s][0]), acc[m]);
                } else {
                    bf16x8 part[3];
                    split8(__builtin_bit_cast(f32x4, c.x[m][s][0]), __builtin_bit_cast(f32x4, c.x[m][s][XBF16 ? 0 : 1]), part);
#pragma unroll
                    for (int e = 0; e < 3; e++) acc[m] = mfma32(a, part[e], acc[m]);
                }
            }
        }
        if (!more) break;
        c = next;
        j += kSteps;
    }
#pragma unroll
    for (int m = 0; m < MT; m++) {
        const uint32_t r = r0 + 32 * m + col;
        if (r >= p.rows) continue;
        const uint64_t at = (uint64_t)r * p.out_stride + (uint64_t)h * p.out_head;
#pragma unroll
        for (int q = 0; q < 4; q++) {
            const uint32_t n = n0 + 8 * q + 4 * half;
            const f32x4 v = {acc[m][4 * q], acc[m][4 * q + 1], acc[m][4 * q + 2], acc[m][4 * q + 3]};
            if (p.fours) {
                if (n >= p.n) continue;
                if (p.out_bf16)
                    *(u32x2 *)((uint16_t *)p.out + at + n) = u32x2{pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3])};
                else
                    *(f32x4 *)((float *)p.out + at + n) = v;
            } else {
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    if (n + i >= p.n) continue;
                    if (p.out_bf16)
                        ((uint16_t *)p.out)[at + n + i] = bf16_bits(v[i]);
                    else
                        ((float *)p.out)[at + n + i] = v[i];
                }
            }
        }
    }
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
    TS_REQUIRE((a->heads == 1 || a->out_head >= a->n) && (a->rows <= 1 || a->out_stride >= a->n),
               "linear_heads: out's rows %u and heads %u apart meet", a->out_stride, a->out_head);
    TS_REQUIRE(ts::aligned(a->x, 16) && ts::aligned(a->w, 16), "linear_heads: x and w must be 16-byte aligned");
    const uint32_t size = a->out_dtype == TS_F32 ? 4 : 2;
    TS_REQUIRE(ts::aligned(a->out, size), "linear_heads: out must be aligned to its type");
    if (a->rows == 0) return TS_OK;
    HeadsParams p;
    p.x = a->x; p.w = (const uint16_t *)a->w; p.out = a->out;
    p.rows = a->rows; p.heads = a->heads; p.n = a->n; p.k = a->k;
    p.x_stride = a->x_stride; p.x_head = a->x_head; p.out_stride = a->out_stride; p.out_head = a->out_head;
    p.w_head = a->w_head;
    p.out_bf16 = a->out_dtype == TS_BF16;
    p.fours = a->n % 4 == 0 && a->out_stride % 4 == 0 && a->out_head % 4 == 0 && ts::aligned(a->out, 4 * size);
    const int mt = a->rows <= 32 ? 1 : 2;
    p.row_tiles = (a->rows - 1) / (32 * mt) + 1;
    p.col_groups = (a->n - 1) / (32 * kWaves) + 1;
    const uint64_t all = (uint64_t)p.row_tiles * p.col_groups * a->heads;
    TS_REQUIRE(all <= 0x7fffffffull, "linear_heads: %u rows in one launch", a->rows);
    const bool bf16 = a->x_dtype == TS_BF16;
    const auto kernel = mt == 1 ? bf16 ? linear_heads_kernel<true, 1> : linear_heads_kernel<false, 1>
                                : bf16 ? linear_heads_kernel<true, 2> : linear_heads_kernel<false, 2>;
    hipLaunchKernelGGL(kernel, dim3((uint32_t)all), dim3(64 * kWaves), 0, (hipStream_t)stream, p);
    TS_CHECK_LAUNCH("linear_heads launch");
    return TS_OK;
}
