// ppocr_matvec_q4: a few rows of x times a matrix of 4-bit weights, and its
// form for three rows and more, and for fewer where k_q4_int.cu is no faster.
//
// A weight becomes q - z, a small integer that f16 and bf16 hold exactly; its
// scale multiplies each group's f32 sum. x enters exactly too: f16 and bf16
// as they are, e4m3 as f16, f32 as three bf16 columns (8 bits of the mantissa
// each) whose sums are added at the end. Bound by the unpacking of the
// weights (11 instructions a word of 8) and, past 16 columns, by the matrix
// instructions; small products by latency. 16 rows f16, 120 x 18 710, groups of
// 32: 4.9 us (2.6 MB, 0.4 us of HBM; an empty launch 2.2); 16 rows e4m3, 4096 x
// 4096, groups of 64: 11.6 us (9.4 MB, 1.4 us).
// Three rows of f32 and more cost most: 16 rows, 4096 x 1024, groups of 64: 21 us,
// f16 6.5, for three columns a row and the taking apart of x in each warp.
#include <type_traits>

#include "q4.cuh"

namespace ppocr {

namespace {

// How x's type enters the matrix instruction: as which type, in how many
// columns a row, and what the weights' power of two leaves to the scale.
template <class XT>
struct Enter {
    using M = XT;
    static constexpr int PARTS = 1;
    static constexpr float SCALE = std::is_same<XT, __nv_bfloat16>::value ? 65536.0f : 1.0f;
};
template <>
struct Enter<float> {
    using M = __nv_bfloat16;
    static constexpr int PARTS = 3;
    static constexpr float SCALE = 65536.0f;
};
template <>
struct Enter<e4m3> {
    using M = __half;
    static constexpr int PARTS = 1;
    static constexpr float SCALE = 1.0f;
};

// 8 weights of a word, less the zero point z, as pairs (0, 4), (1, 5),
// (2, 6), (3, 7).
template <class M>
__device__ __forceinline__ void unpack(uint32_t w, uint32_t z, uint32_t out[4]);

// (w & mask) | magic in one instruction: two constants in registers.
__device__ __forceinline__ uint32_t pick(uint32_t w, uint32_t mask, uint32_t magic) {
    uint32_t v;
    asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(v) : "r"(w), "r"(mask), "r"(magic));
    return v;
}

// f16: 0x6400 | q is 1024 + q, 0x6400 | q << 4 is 1024 + 16 q; both less their
// offset are exact (a small integer in the low bits of a float of a fixed exponent: a
// published way from integers to floats without a conversion).
template <>
__device__ __forceinline__ void unpack<__half>(uint32_t w, uint32_t z, uint32_t out[4]) {
    const uint32_t z1 = (0x6400u + z) * 0x10001u;          // 1024 + z, twice
    const uint32_t z16 = (0xD400u + (z << 4)) * 0x10001u;  // -(64 + z), twice
    const uint32_t sixteenth = 0x2C002C00u;                // 1 / 16
    const uint32_t w8 = w >> 8;
    const uint32_t a = pick(w, 0x000F000Fu, 0x64006400u), b = pick(w, 0x00F000F0u, 0x64006400u);
    const uint32_t c = pick(w8, 0x000F000Fu, 0x64006400u), d = pick(w8, 0x00F000F0u, 0x64006400u);
    const auto h2 = [](const uint32_t &v) { return *reinterpret_cast<const __half2 *>(&v); };
    const auto u = [](const __half2 &v) { return *reinterpret_cast<const uint32_t *>(&v); };
    out[0] = u(__hsub2(h2(a), h2(z1)));
    out[1] = u(__hfma2(h2(b), h2(sixteenth), h2(z16)));
    out[2] = u(__hsub2(h2(c), h2(z1)));
    out[3] = u(__hfma2(h2(d), h2(sixteenth), h2(z16)));
}

// bf16: 0x3B00 | q is (128 + q) 2^-16. The power of two keeps a group's sum of
// products with the largest x finite (x itself may be anything f32 holds); the
// scale takes it back.
template <>
__device__ __forceinline__ void unpack<__nv_bfloat16>(uint32_t w, uint32_t z, uint32_t out[4]) {
    const uint32_t z1 = (0x3B00u + z) * 0x10001u;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const uint32_t v = pick(w >> (4 * i), 0x000F000Fu, 0x3B003B00u);
        const __nv_bfloat162 r =
            __hsub2(*reinterpret_cast<const __nv_bfloat162 *>(&v), *reinterpret_cast<const __nv_bfloat162 *>(&z1));
        out[i] = *reinterpret_cast<const uint32_t *>(&r);
    }
}

// The part of an f32 x that column `part` of its row holds: the top 8 bits of the mantissa, the next 8, the last 8, each exact in bf16; an
// infinity or NaN stays whole in the first.
__device__ __forceinline__ float part_of(float x, int part) {
    if (!(fabsf(x) < INFINITY)) return part == 0 ? x : 0.0f;
    const float hi = __uint_as_float(__float_as_uint(x) & 0xFFFF0000u), rest = x - hi;
    const float mid = __uint_as_float(__float_as_uint(rest) & 0xFFFF0000u);
    return part == 0 ? hi : part == 1 ? mid : rest - mid;
}


// CT: 8-column tiles of x; BPG: 32-k blocks a weight group (4, 2, or 1,
// which serves every multiple of 32).
template <int CT>
struct Q4Tile {
    // a row of partial sums, padded so that 16 rows' columns lie in different banks
    static constexpr int COLS = 8 * CT, WIDE = COLS + 2, SL = CT == 1 ? 2 : 1, DEPTH = 4 / SL;
    // 64 registers of x a lane with four column tiles: half the warps
    static constexpr int WARPS = CT == 4 ? 8 : 16;
    static constexpr int SHARED = 200 * 1024;
};

template <class XT, int CT, int BPG, bool ZEROS>
__global__ void __launch_bounds__(Q4Tile<CT>::WARPS * 32, 1) q4_kernel(const __grid_constant__ Q4Args a) {
    using M = typename Enter<XT>::M;
    using Q = Q4Tile<CT>;
    constexpr int PARTS = Enter<XT>::PARTS, WIDE = Q::WIDE, SL = Q::SL, DEPTH = Q::DEPTH;
    extern __shared__ __align__(16) float red[];  // [list of the batch][tile of the item][warp][16][WIDE], then the cluster's sums
    const Place at(a);
    const int warps = int(blockDim.x) / 32;
    const int m0 = blockIdx.y * a.cols_rows, rows = min(a.cols_rows, a.m - m0);
    if (a.ks > 1) cluster_arrive();
    Stream<SL, DEPTH, BPG, ZEROS> in;
    in.begin(a, at);
    uint4 xf[SL][4][CT];
    const auto load = [&](int c0) {
        const auto k_of = [&](int c, int u) { return (c0 + c) * 128 + (BPG == 4 ? at.t * 32 + u * 8 : u * 32 + at.t * 8); };
#pragma unroll
        for (int c = 0; c < SL; c++)
#pragma unroll
            for (int u = 0; u < 4; u++) {
                float v[PARTS == 1 ? 1 : CT][8] = {};
#pragma unroll
                for (int ct = 0; ct < CT; ct++) {
                    const int r = (ct * 8 + at.g) / PARTS;
                    const bool there = r < rows && c0 + c < at.c_hi;
                    if constexpr (PARTS == 1)
                        xf[c][u][ct] = take_x<XT>(a, m0 + r, k_of(c, u), there);
                    else if (there)
                        load_x<XT>(a, m0 + r, k_of(c, u), v[ct]);
                }
                if constexpr (PARTS > 1) {
#pragma unroll
                    for (int ct = 0; ct < CT; ct++) {
                        const int part = (ct * 8 + at.g) % PARTS;
                        uint32_t p[4];
#pragma unroll
                        for (int i = 0; i < 4; i++) p[i] = pack2<M>(part_of(v[ct][i], part), part_of(v[ct][i + 4], part));
                        xf[c][u][ct] = make_uint4(p[0], p[1], p[2], p[3]);
                    }
                }
            }
        if constexpr (PARTS == 1) {
#pragma unroll
            for (int c = 0; c < SL; c++)
#pragma unroll
                for (int u = 0; u < 4; u++)
#pragma unroll
                    for (int ct = 0; ct < CT; ct++) xf[c][u][ct] = pairs_of<XT>(xf[c][u][ct]);
        }
    };
    const auto value = [&](int l, int tile, int m, int r) {
        const float *from = red + (((l * a.depth + tile % a.depth) * warps + tile / a.depth * a.wk) * 16 + r) * WIDE + m * PARTS;
        float y = 0.0f;
        for (int p = PARTS - 1; p >= 0; p--)
            for (int w = 0; w < a.wk; w++) y += from[w * 16 * WIDE + p];
        return y;
    };
    const auto finish = [&](int m, int n, float y, float bias, float scale) { put_y(a, m0 + m, n, fmaf(y, scale, bias)); };
    for (int b0 = 0; b0 < at.lists; b0 += a.batch) {
        const int count = min(a.batch, at.lists - b0);
        for (int lap = 0; lap < a.laps; lap++) {
            const int c0 = at.c_lo + (lap * a.wk + at.k_warp) * SL;
            if (a.laps > 1 || b0 == 0) load(c0);
            for (int i = 0; i < count; i++) {
                in.aim(a, at);
                const bool more = in.rows > 0;  // there is another item to take
#pragma unroll
                for (int d = 0; d < DEPTH; d++) {
                    if (d >= a.depth) break;
                    float acc[CT][4] = {}, sum[CT][4];
                    float s[SL][4 / BPG][2];
                    uint32_t z[SL][4 / BPG][2];
#pragma unroll
                    for (int j = 0; j < SL * 4 / BPG; j++)
#pragma unroll
                        for (int h = 0; h < 2; h++) {
                            s[j / (4 / BPG)][j % (4 / BPG)][h] = in.scale(a, d, j, at.g + 8 * h) * Enter<XT>::SCALE;
                            z[j / (4 / BPG)][j % (4 / BPG)][h] = in.zero(d, j, at.g + 8 * h);
                        }
                    if (more) in.scales(a, at, d);
#pragma unroll
                    for (int c = 0; c < SL; c++) {
                        uint4 u0 = in.w[d][c][0], u1 = in.w[d][c][1];
                        if constexpr (BPG < 4) {
                            transpose(u0, at.t);
                            transpose(u1, at.t);
                        }
                        const uint32_t w0[4] = {u0.x, u0.y, u0.z, u0.w}, w1[4] = {u1.x, u1.y, u1.z, u1.w};
#pragma unroll
                        for (int u = 0; u < 4; u++) {
                            const int j = u / BPG;
                            if (u % BPG == 0) {
#pragma unroll
                                for (int ct = 0; ct < CT; ct++) sum[ct][0] = sum[ct][1] = sum[ct][2] = sum[ct][3] = 0.0f;
                            }
                            uint32_t p0[4], p1[4];
                            unpack<M>(w0[u], z[c][j][0], p0);
                            unpack<M>(w1[u], z[c][j][1], p1);
                            const uint32_t lo[4] = {p0[0], p1[0], p0[1], p1[1]}, hi[4] = {p0[2], p1[2], p0[3], p1[3]};
#pragma unroll
                            for (int ct = 0; ct < CT; ct++) {
                                mma16<M>(sum[ct], lo, xf[c][u][ct].x, xf[c][u][ct].y);
                                mma16<M>(sum[ct], hi, xf[c][u][ct].z, xf[c][u][ct].w);
                            }
                            if (u % BPG == BPG - 1) {
#pragma unroll
                                for (int ct = 0; ct < CT; ct++) {
                                    float f0 = 1.0f, f1 = 1.0f;
                                    if (sizeof(XT) == 1 && a.x_groups > 1) {
                                        const int group = ((c0 + c) * 4 + u) * 32 / a.group, m = ct * 8 + at.t * 2;
                                        if (group < a.groups) {
                                            if (m < rows) f0 = __ldg(a.x_scales + int64_t(m0 + m) * a.x_groups + group);
                                            if (m + 1 < rows) f1 = __ldg(a.x_scales + int64_t(m0 + m + 1) * a.x_groups + group);
                                        }
                                    }
                                    acc[ct][0] = fmaf(sum[ct][0], s[c][j][0] * f0, acc[ct][0]);
                                    acc[ct][1] = fmaf(sum[ct][1], s[c][j][0] * f1, acc[ct][1]);
                                    acc[ct][2] = fmaf(sum[ct][2], s[c][j][1] * f0, acc[ct][2]);
                                    acc[ct][3] = fmaf(sum[ct][3], s[c][j][1] * f1, acc[ct][3]);
                                }
                            }
                        }
                        if (more) in.chunk(a, at, d, c);
                    }
                    const float bias[2] = {in.b[d][0], in.b[d][1]};
                    if (more) in.biases(a, at, d);
                    if (PARTS == 1 && a.direct) {
                        // this warp's sums are whole: out with them
                        const int n0 = at.row(a, b0 + i, at.r_warp) + d * 16 + at.g;
#pragma unroll
                        for (int ct = 0; ct < CT; ct++)
#pragma unroll
                            for (int e = 0; e < 4; e++) {
                                const int n = n0 + 8 * (e >> 1), m = ct * 8 + at.t * 2 + (e & 1);
                                if (n >= a.n || m >= rows) continue;
                                const float scale = sizeof(XT) == 1 && a.x_groups == 1 ? __ldg(a.x_scales + m0 + m) : 1.0f;
                                finish(m, n, acc[ct][e], bias[e >> 1], scale);
                            }
                        continue;
                    }
                    float *mine = red + (((i * a.depth + d) * warps + at.warp) * 16 + at.g) * WIDE + at.t * 2;
#pragma unroll
                    for (int ct = 0; ct < CT; ct++)
#pragma unroll
                        for (int h = 0; h < 2; h++) {
                            float2 *to = reinterpret_cast<float2 *>(mine + h * 8 * WIDE + ct * 8);
                            float2 v = make_float2(acc[ct][2 * h], acc[ct][2 * h + 1]);
                            if (lap > 0) v.x += to->x, v.y += to->y;
                            *to = v;
                        }
                }
                in.next(a, at);
            }
        }
        if (!a.direct) join(a, at, m0, rows, b0, count, red + a.red_floats, value, finish);
    }
}

template <class XT, int CT, int BPG, bool ZEROS>
cudaError_t start(Q4Args a, cudaStream_t stream) {
    using Q = Q4Tile<CT>;
    const cudaError_t e = raise_shared<q4_kernel<XT, CT, BPG, ZEROS>>(Q::SHARED);
    if (e != cudaSuccess) return e;
    a.cols_rows = Q::COLS / Enter<XT>::PARTS < a.m ? Q::COLS / Enter<XT>::PARTS : a.m;
    return launch_q4(reinterpret_cast<const void *>(q4_kernel<XT, CT, BPG, ZEROS>), a, Q::WARPS, Q::SL, Q::DEPTH, BPG, Q::WIDE, 0,
                     Q::SHARED, Enter<XT>::PARTS == 1, Enter<XT>::PARTS == 1, stream);
}

template <class XT, int BPG, bool ZEROS>
cudaError_t start_m(const Q4Args &a, cudaStream_t s) {
    const int cols = a.m * Enter<XT>::PARTS;
    if constexpr (Enter<XT>::PARTS == 1)
        if (cols <= 8) return start<XT, 1, BPG, ZEROS>(a, s);
    if (cols <= 16) return start<XT, 2, BPG, ZEROS>(a, s);
    return start<XT, 4, BPG, ZEROS>(a, s);
}

template <class XT>
cudaError_t start_x(const Q4Args &a, cudaStream_t s) {
    if (a.group % 128 == 0) return a.zeros ? start_m<XT, 4, true>(a, s) : start_m<XT, 4, false>(a, s);
    if (a.group % 64 == 0) return a.zeros ? start_m<XT, 2, true>(a, s) : start_m<XT, 2, false>(a, s);
    return a.zeros ? start_m<XT, 1, true>(a, s) : start_m<XT, 1, false>(a, s);
}

}  // namespace

}  // namespace ppocr

using namespace ppocr;

extern "C" int ppocr_matvec_q4(const ppocr_matvec_q4_shape *s, const void *x, const float *x_scales, const uint8_t *w,
                               const void *scales, const uint8_t *zeros, const float *bias, void *y, void *stream) {
    static const char *me = "ppocr_matvec_q4";
    clear_error();
    if (!s) return refuse(PPOCR_E_ARG, me, "null shape");
    if (s->x_type != PPOCR_F32 && s->x_type != PPOCR_F16 && s->x_type != PPOCR_BF16 && s->x_type != PPOCR_E4M3)
        return refuse(PPOCR_E_ARG, me, "x_type must be PPOCR_F32, PPOCR_F16, PPOCR_BF16 or PPOCR_E4M3");
    if (s->y_type != PPOCR_F32 && s->y_type != PPOCR_F16 && s->y_type != PPOCR_BF16)
        return refuse(PPOCR_E_ARG, me, "y_type must be PPOCR_F32, PPOCR_F16 or PPOCR_BF16");
    if (s->scale_type != PPOCR_F32 && s->scale_type != PPOCR_F16 && s->scale_type != PPOCR_BF16)
        return refuse(PPOCR_E_ARG, me, "scale_type must be PPOCR_F32, PPOCR_F16 or PPOCR_BF16");
    if (!s->group || s->group % 32 || s->group > (1u << 20)) return refuse(PPOCR_E_ARG, me, "group must be a multiple of 32, at most 2^20");
    if (s->rows > 32) return refuse(PPOCR_E_SIZE, me, "more than 32 rows of x: split the call");
    if (!s->k || s->k > (1u << 20) || s->n > (1u << 24)) return refuse(PPOCR_E_SIZE, me, "k must be between 1 and 2^20, n at most 2^24");
    const uint64_t most = uint64_t(1) << 32;
    if (s->x_row > most || s->y_row > most || s->w_row > most) return refuse(PPOCR_E_SIZE, me, "a stride above 2^32");
    if (!s->rows || !s->n) return PPOCR_OK;
    if (!x || !w || !scales || !y) return refuse(PPOCR_E_ARG, me, "null buffer");
    const uint64_t groups = (uint64_t(s->k) + s->group - 1) / s->group;
    if (s->x_type == PPOCR_E4M3) {
        if (!x_scales) return refuse(PPOCR_E_ARG, me, "e4m3 rows need x_scales");
        if (s->x_group != 0 && s->x_group != s->group) return refuse(PPOCR_E_ARG, me, "x_group must be 0 (a row) or the weights' group");
    } else if (x_scales) {
        return refuse(PPOCR_E_ARG, me, "x_scales belong to e4m3 rows");
    }
    const size_t xs = type_size(s->x_type), ys = type_size(s->y_type), ss = type_size(s->scale_type);
    if (!aligned(x, xs) || !aligned(y, ys) || !aligned(scales, ss) || !aligned(x_scales, 4) || !aligned(bias, 4))
        return refuse(PPOCR_E_ARG, me, "a buffer is not aligned to its type");
    Q4Args a{};
    a.x = x, a.x_scales = x_scales, a.w = w, a.scales = scales, a.zeros = zeros, a.bias = bias, a.y = y;
    a.m = int(s->rows), a.k = int(s->k), a.n = int(s->n), a.group = int(s->group), a.groups = int(groups);
    a.x_row = int64_t(s->x_row ? s->x_row : s->k), a.y_row = int64_t(s->y_row ? s->y_row : s->n);
    a.w_row = int64_t(s->w_row ? s->w_row : (uint64_t(s->k) + 1) / 2);
    if (a.w_row < (int64_t(s->k) + 1) / 2 || (s->rows > 1 && a.y_row < int64_t(s->n)))
        return refuse(PPOCR_E_ARG, me, "rows of w or y overlap");
    const auto rows = [](const void *p, uint64_t n, uint64_t row, uint64_t each, uint64_t bytes) {
        return Rows{p, p ? ((n - 1) * row + each) * bytes : 0, each * bytes, row * bytes};
    };
    const Rows yr = rows(y, s->rows, uint64_t(a.y_row), s->n, ys);
    const uint64_t x_groups = s->x_group ? groups : 1;
    if (overlap(yr, rows(x, s->rows, uint64_t(a.x_row), s->k, xs)) ||
        overlap(yr, rows(w, s->n, uint64_t(a.w_row), (uint64_t(s->k) + 1) / 2, 1)) || overlap(yr, rows(scales, s->n, groups, groups, ss)) ||
        overlap(yr, rows(zeros, s->n, groups, groups, 1)) || overlap(yr, rows(bias, 1, s->n, s->n, 4)) ||
        overlap(yr, rows(x_scales, s->rows, x_groups, x_groups, 4)))
        return refuse(PPOCR_E_ARG, me, "y overlaps another buffer");
    if (const int bad = check_buffers(me, {x, x_scales, w, scales, zeros, bias, y})) return bad;
    a.scale_type = s->scale_type, a.y_type = s->y_type;
    // one group in all is the row's scale
    a.x_groups = !x_scales ? 0 : s->x_group ? int(groups) : 1;
    a.w_vec = aligned(w, 16) && a.w_row % 16 == 0;
    a.x_vec = uint64_t(a.x_row) * xs % (xs == 1 ? 8 : 16) == 0 && aligned(x, xs == 1 ? 8 : 16);
    const auto str = static_cast<cudaStream_t>(stream);
    // in whole numbers: one or two rows of f32 (two rows, groups of 128, 4096 x 4096 and 8192 x
    // 28 672: 9.4 and 41 us; one row 7.8 and 27, where three parts take 157), and one row of
    // another type from 2^26 weights on (bf16, 8192 x 4096, 8192 and 28 672, groups of 128
    // without zero points: 9.4, 13.4 and 27 us, 9.3, 16.0 and 40 the other way; groups of 64
    // with them: 13.4, 22.5 and 56, 12.1, 22.7 and 61; two rows 18 and 16, 40 and 40)
    const bool whole = s->x_type == PPOCR_F32 ? a.m <= 2 : a.m == 1 && s->n * uint64_t(s->k) >= uint64_t(1) << 26;
    const cudaError_t e = whole                     ? launch_q4_int(a, s->x_type, str)
                          : s->x_type == PPOCR_F32  ? start_x<float>(a, str)
                          : s->x_type == PPOCR_F16  ? start_x<__half>(a, str)
                          : s->x_type == PPOCR_BF16 ? start_x<__nv_bfloat16>(a, str)
                                                    : start_x<e4m3>(a, str);
    return e == cudaSuccess ? int(PPOCR_OK) : refuse(PPOCR_E_DEVICE, me, cudaGetErrorString(e));
}
