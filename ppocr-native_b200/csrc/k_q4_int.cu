// ppocr_matvec_q4 for one and two rows of x: the sums in whole numbers.
//
// x enters as fixed point of 31 bits below the largest magnitude of its
// warp's slice, as four columns of signed bytes (base 256, digits -128 to
// 127), and the weights as the unsigned bytes that one mask makes of them:
// 3 instructions a word of 8 where f16 or bf16 weights take 9 and 11, and half
// the matrix instructions (k 32 a piece, at f16's rate of instructions). Sums of
// a group are exact; its zero point comes off as z times the group's sum of
// x, before the f32 scale. What the fixed point drops of an x is at most
// 2^-31 of its slice's largest: less than f32 sums round away, save where all
// weights of values far above the rest (2^10 times and more) are zero. A slice with an
// infinity or NaN gives NaN, and such results are done again the plain way.
// Bound by HBM and, with zero points or small groups, by the groups' sums: one
// row bf16, 8192 x 28 672, groups of 128: 25 to 28 us, 121 MB at 4.3 to 4.8 TB/s
// (18.6 us at a plain copy's rate, the rest launch, x and join); groups of 64
// with zero points 54 us, of 32 80 us.
#include <type_traits>

#include "q4.cuh"

namespace ppocr {

namespace {

// y[m][n] in plain f32 arithmetic, by one thread.
template <class XT>
__device__ __noinline__ float plain_q4(const Q4Args &a, int m, int n) {
    float y = 0.0f;
    for (int k = 0; k < a.k; k++) {
        float x;
        if constexpr (sizeof(XT) == 1) {
            x = __half2float(__half(__nv_cvt_fp8_to_halfraw(__nv_fp8_storage_t(static_cast<const uint8_t *>(a.x)[m * a.x_row + k]), __NV_E4M3)));
            x *= a.x_scales[int64_t(m) * a.x_groups + (a.x_groups > 1 ? k / a.group : 0)];
        } else {
            x = to_f32(static_cast<const XT *>(a.x)[m * a.x_row + k]);
        }
        const int64_t at = int64_t(n) * a.groups + k / a.group;
        const int q = (a.w[int64_t(n) * a.w_row + k / 2] >> (4 * (k & 1))) & 15, z = a.zeros ? a.zeros[at] & 15 : 8;
        y = fmaf(x, float(q - z) * load_scale(a, at), y);
    }
    return y;
}

template <int BPG>
struct IntTile {
    // two chunks where every 32 k have their own sums: registers
    static constexpr int SL = BPG == 1 ? 2 : 4, DEPTH = 4 / SL, WARPS = 16, SHARED = 128 * 1024;
};

template <class XT, int BPG, bool ZEROS, int ROWS_X>
__global__ void __launch_bounds__(IntTile<BPG>::WARPS * 32, 1) q4_int_kernel(const __grid_constant__ Q4Args a) {
    using Q = IntTile<BPG>;
    constexpr int SL = Q::SL, DEPTH = Q::DEPTH, GPC = 4 / BPG;  // groups a chunk
    // a group's sum is below 2^19 in magnitude; added to these bits, 1.5 * 2^23's,
    // it is that number as a float plus 1.5 * 2^23
    constexpr int MAGIC = 0x4B400000;
    extern __shared__ __align__(16) float red[];  // [list of the batch][tile of the item][warp][row of x][16], the cluster's sums, x's stage
    const Place at(a);
    const int warps = int(blockDim.x) / 32;
    if (a.ks > 1) cluster_arrive();
    Stream<SL, DEPTH, BPG, ZEROS> in;
    in.begin(a, at);

    uint32_t xe[SL][4], xo[SL][4];  // column g % COLS: byte g % 4 of row g / 4, the even and the odd k
    int xc[SL][GPC][2];             // columns 2t and 2t + 1: what a group's sum starts from (or its sum of x)
    float back0 = 0.0f, back1 = 0.0f;  // 2^-up of the row of columns 2t, in two factors; NaN where x is not finite
    const auto load = [&](int c0) {
        // each lane converts a piece of 8 k of every eighth unit (32 k); the
        // columns' owners get them through this warp's shared memory
        constexpr int UNITS = SL * 4, MINE = (UNITS + 7) / 8, COLS = 4 * ROWS_X;
        uint2 *stage = reinterpret_cast<uint2 *>(red + a.stage_floats) + at.warp * UNITS * COLS * 4;  // [unit][column][t]
        __syncwarp();
#pragma unroll
        for (int row = 0; row < ROWS_X; row++) {
            float v[MINE][8];
            uint32_t top = 0;  // as bits: an infinity or NaN shows
#pragma unroll
            for (int x = 0; x < MINE; x++) {
                const int unit = at.g + 8 * x, c = c0 + unit / 4, u = unit % 4;
                const int k = c * 128 + (BPG == 4 ? at.t * 32 + u * 8 : u * 32 + at.t * 8);
#pragma unroll
                for (int i = 0; i < 8; i++) v[x][i] = 0.0f;
                if (unit >= UNITS || c >= at.c_hi) continue;
                load_x<XT>(a, row, k, v[x]);
                if constexpr (sizeof(XT) == 1) {
                    const float f = k < a.k ? __ldg(a.x_scales + int64_t(row) * a.x_groups + (a.x_groups > 1 ? k / a.group : 0)) : 0.0f;
#pragma unroll
                    for (int i = 0; i < 8; i++) v[x][i] *= f;
                }
#pragma unroll
                for (int i = 0; i < 8; i++) top = max(top, __float_as_uint(v[x][i]) & 0x7fffffffu);
            }
            top = __reduce_max_sync(0xffffffffu, top);
            const bool odd = top >= 0x7f800000u;
            const int up = top == 0 || odd ? 0 : 29 - ilogbf(__uint_as_float(top));  // x * 2^up is below 2^30
            const float up0 = ldexpf(1.0f, up / 2), up1 = ldexpf(1.0f, up - up / 2);
            if (ROWS_X == 1 || (at.t >> 1) == row) back0 = odd ? NAN : ldexpf(1.0f, -(up / 2)), back1 = ldexpf(1.0f, -(up - up / 2));
#pragma unroll
            for (int x = 0; x < MINE; x++) {
                const int unit = at.g + 8 * x;
                uint32_t n[8];
#pragma unroll
                for (int i = 0; i < 8; i++)  // plus 128 in each of the lower digits: its bytes are the digits plus 128
                    n[i] = uint32_t((odd ? 0 : __float2int_rn(v[x][i] * up0 * up1)) + 0x00808080);
                // byte b of four numbers in word b, for the even k and the odd
                uint32_t word[2][4];
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    const uint32_t l0 = __byte_perm(n[h], n[2 + h], 0x5140), l1 = __byte_perm(n[4 + h], n[6 + h], 0x5140);
                    const uint32_t h0 = __byte_perm(n[h], n[2 + h], 0x7362), h1 = __byte_perm(n[4 + h], n[6 + h], 0x7362);
                    word[h][0] = __byte_perm(l0, l1, 0x5410) ^ 0x80808080u;
                    word[h][1] = __byte_perm(l0, l1, 0x7632) ^ 0x80808080u;
                    word[h][2] = __byte_perm(h0, h1, 0x5410) ^ 0x80808080u;
                    word[h][3] = __byte_perm(h0, h1, 0x7632);
                }
                if (unit < UNITS)
#pragma unroll
                    for (int b = 0; b < 4; b++) stage[(unit * COLS + row * 4 + b) * 4 + at.t] = make_uint2(word[0][b], word[1][b]);
            }
        }
        __syncwarp();
#pragma unroll
        for (int c = 0; c < SL; c++) {
            int sum[GPC] = {};
#pragma unroll
            for (int u = 0; u < 4; u++) {
                const uint2 v = stage[((c * 4 + u) * COLS + at.g % COLS) * 4 + at.t];
                xe[c][u] = v.x, xo[c][u] = v.y;
                sum[u / BPG] = __dp4a(int(v.x), 0x01010101, __dp4a(int(v.y), 0x01010101, sum[u / BPG]));
            }
#pragma unroll
            for (int j = 0; j < GPC; j++) {
                int v = sum[j];
                v += __shfl_xor_sync(0xffffffffu, v, 1);
                v += __shfl_xor_sync(0xffffffffu, v, 2);
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    const int other = __shfl_sync(0xffffffffu, v, (at.t * 2 + h) * 4);
                    xc[c][j][h] = ZEROS ? other : MAGIC - 8 * other;
                }
            }
        }
    };
    const auto value = [&](int l, int tile, int m, int r) {
        const float *from = red + ((l * a.depth + tile % a.depth) * warps + tile / a.depth * a.wk) * ROWS_X * 16 + m * 16 + r;
        float y = 0.0f;
        for (int w = 0; w < a.wk; w++) y += from[w * ROWS_X * 16];
        return y;
    };
    const auto finish = [&](int m, int n, float y, float bias, float) {
        if (!(fabsf(y) < INFINITY)) y = plain_q4<XT>(a, m, n);
        put_y(a, m, n, y + bias);
    };
    for (int b0 = 0; b0 < at.lists; b0 += a.batch) {
        const int count = min(a.batch, at.lists - b0);
        for (int lap = 0; lap < a.laps; lap++) {
            if (a.laps > 1 || b0 == 0) load(at.c_lo + (lap * a.wk + at.k_warp) * SL);
            for (int i = 0; i < count; i++) {
                in.aim(a, at);
                const bool more = in.rows > 0;  // there is another item to take
#pragma unroll
                for (int d = 0; d < DEPTH; d++) {
                    if (d >= a.depth) break;
                    float acc[4] = {};
                    float s[SL * GPC][2];
                    uint32_t z[SL * GPC][2];
#pragma unroll
                    for (int j = 0; j < SL * GPC; j++)
#pragma unroll
                        for (int h = 0; h < 2; h++) {
                            s[j][h] = in.scale(a, d, j, at.g + 8 * h);
                            z[j][h] = in.zero(d, j, at.g + 8 * h);
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
                        int v[4];
#pragma unroll
                        for (int u = 0; u < 4; u++) {
                            const int j = c * GPC + u / BPG;
                            if (u % BPG == 0) {
                                if constexpr (ZEROS) {
                                    v[0] = MAGIC - int(z[j][0]) * xc[c][u / BPG][0], v[1] = MAGIC - int(z[j][0]) * xc[c][u / BPG][1];
                                    v[2] = MAGIC - int(z[j][1]) * xc[c][u / BPG][0], v[3] = MAGIC - int(z[j][1]) * xc[c][u / BPG][1];
                                } else {
                                    v[0] = v[2] = xc[c][u / BPG][0], v[1] = v[3] = xc[c][u / BPG][1];
                                }
                            }
                            asm volatile(
                                "mma.sync.aligned.m16n8k32.row.col.s32.u8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                                : "+r"(v[0]), "+r"(v[1]), "+r"(v[2]), "+r"(v[3])
                                : "r"(w0[u] & 0x0F0F0F0Fu), "r"(w1[u] & 0x0F0F0F0Fu), "r"((w0[u] >> 4) & 0x0F0F0F0Fu),
                                  "r"((w1[u] >> 4) & 0x0F0F0F0Fu), "r"(xe[c][u]), "r"(xo[c][u]));
                            if (u % BPG == BPG - 1) {
                                acc[0] = fmaf(__int_as_float(v[0]) - 12582912.0f, s[j][0], acc[0]);
                                acc[1] = fmaf(__int_as_float(v[1]) - 12582912.0f, s[j][0], acc[1]);
                                acc[2] = fmaf(__int_as_float(v[2]) - 12582912.0f, s[j][1], acc[2]);
                                acc[3] = fmaf(__int_as_float(v[3]) - 12582912.0f, s[j][1], acc[3]);
                            }
                        }
                        if (more) in.chunk(a, at, d, c);
                    }
                    const float bias[2] = {in.b[d][0], in.b[d][1]};
                    if (more) in.biases(a, at, d);
                    // columns 2t and 2t + 1 are bytes 0, 1 (t even) or 2, 3 of a row: one number
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        float y = fmaf(acc[2 * h + 1], 256.0f, acc[2 * h]);
                        if (at.t & 1) y *= 65536.0f;
                        y += __shfl_xor_sync(0xffffffffu, y, 1);
                        y = y * back0 * back1;
                        const int m = at.t >> 1;
                        if ((at.t & 1) == 0 && m < ROWS_X && a.direct) {
                            const int n = at.row(a, b0 + i, at.r_warp) + d * 16 + at.g + 8 * h;
                            if (n < a.n) finish(m, n, y, bias[h], 1.0f);
                        } else if ((at.t & 1) == 0 && m < ROWS_X) {
                            float *to = red + (((i * a.depth + d) * warps + at.warp) * ROWS_X + m) * 16 + at.g + 8 * h;
                            *to = lap > 0 ? *to + y : y;
                        }
                    }
                }
                in.next(a, at);
            }
        }
        if (!a.direct) join(a, at, 0, ROWS_X, b0, count, red + a.red_floats, value, finish);
    }
}

template <class XT, int BPG, bool ZEROS, int ROWS_X>
cudaError_t start(Q4Args a, cudaStream_t stream) {
    using Q = IntTile<BPG>;
    const cudaError_t e = raise_shared<q4_int_kernel<XT, BPG, ZEROS, ROWS_X>>(Q::SHARED);
    if (e != cudaSuccess) return e;
    a.cols_rows = a.m;
    return launch_q4(reinterpret_cast<const void *>(q4_int_kernel<XT, BPG, ZEROS, ROWS_X>), a, Q::WARPS, Q::SL, Q::DEPTH, BPG, ROWS_X,
                     Q::SL * 4 * 4 * ROWS_X * 32, Q::SHARED, true, false, stream);
}

template <class XT, int BPG>
cudaError_t start_g(const Q4Args &a, cudaStream_t s) {
    if (a.m == 1) return a.zeros ? start<XT, BPG, true, 1>(a, s) : start<XT, BPG, false, 1>(a, s);
    return a.zeros ? start<XT, BPG, true, 2>(a, s) : start<XT, BPG, false, 2>(a, s);
}

template <class XT>
cudaError_t start_x(const Q4Args &a, cudaStream_t s) {
    return a.group % 128 == 0 ? start_g<XT, 4>(a, s) : a.group % 64 == 0 ? start_g<XT, 2>(a, s) : start_g<XT, 1>(a, s);
}

}  // namespace

cudaError_t launch_q4_int(const Q4Args &a, int x_type, cudaStream_t stream) {
    if (x_type == PPOCR_F32) return start_x<float>(a, stream);
    if (x_type == PPOCR_F16) return start_x<__half>(a, stream);
    if (x_type == PPOCR_BF16) return start_x<__nv_bfloat16>(a, stream);
    return start_x<e4m3>(a, stream);
}

}  // namespace ppocr
