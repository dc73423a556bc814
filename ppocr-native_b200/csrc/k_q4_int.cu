// ppocr_matvec_q4 for one and two rows of f32, and one of another type times many
// weights: the sums in whole numbers.
//
// x enters as fixed point of 62 bits below the largest magnitude of its
// warp's slice, a row as eight columns of signed bytes (base 256, digits -128 to
// 127; the matrix instruction has eight columns, so the bits cost nothing), and the
// weights as the unsigned bytes that one mask makes of them:
// 3 instructions a word of 8 where f16 or bf16 weights take 9 and 11, and half
// the matrix instructions (k 32 a piece, at f16's rate of instructions). Sums of
// a group are exact; its zero point comes off as z times the group's sum of
// x, before the f32 scale. f16 enters exactly, f32 down to 2^-38 and bf16 to 2^-54 of the
// slice's largest, values below to 2^-62 of it (four columns, 31 bits, lost what stood
// beside a value 2^14 times as large whose weight is zero). A slice with an
// infinity or NaN gives NaN, and such results are done again the plain way.
// Bound by HBM and, with zero points or small groups, by the groups' sums: one
// row bf16, 8192 x 28 672, groups of 128: 27 us, 121 MB at 4.5 TB/s
// (18.6 us at a plain copy's rate, the rest launch, x and join); groups of 64
// with zero points 54 to 58 us, of 32 80 us; two rows f32 41, 67 and 122 us.
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

template <int BPG, int ROWS_X>
struct IntTile {
    // two chunks where every 32 k have their own sums: registers. Two rows' columns take half
    // the warps with twice the tiles each (8192 x 28 672, groups of 128 and 64: 40 and 67 us,
    // in 16 warps of two chunks 50 and 74), save for groups of 32, where half the k a
    // block holds would leave more to the cluster's join (122 us, 178 in 8 warps)
    static constexpr bool WIDE = ROWS_X == 2 && BPG > 1;
    static constexpr int SL = BPG == 1 ? 2 : 4, DEPTH = (WIDE ? 8 : 4) / SL, WARPS = WIDE ? 8 : 16, SHARED = 128 * 1024;
    static constexpr int COLS = 8 * ROWS_X, STAGE = SL * 4 * COLS * 4 * 8;  // columns of x; bytes of its stage a warp
};

// Bytes 0 to 3 of four words, byte b of each in word b.
__device__ __forceinline__ void bytes_of(uint32_t a, uint32_t b, uint32_t c, uint32_t d, uint32_t out[4]) {
    const uint32_t l0 = __byte_perm(a, b, 0x5140), l1 = __byte_perm(c, d, 0x5140);
    const uint32_t h0 = __byte_perm(a, b, 0x7362), h1 = __byte_perm(c, d, 0x7362);
    out[0] = __byte_perm(l0, l1, 0x5410);
    out[1] = __byte_perm(l0, l1, 0x7632);
    out[2] = __byte_perm(h0, h1, 0x5410);
    out[3] = __byte_perm(h0, h1, 0x7632);
}

template <class XT, int BPG, bool ZEROS, int ROWS_X>
__global__ void __launch_bounds__(IntTile<BPG, ROWS_X>::WARPS * 32, 1) q4_int_kernel(const __grid_constant__ Q4Args a) {
    using Q = IntTile<BPG, ROWS_X>;
    constexpr int SL = Q::SL, DEPTH = Q::DEPTH, GPC = 4 / BPG, COLS = Q::COLS;  // GPC: groups a chunk
    // a group's sum is below 2^19 in magnitude; added to these bits, 1.5 * 2^23's,
    // it is that number as a float plus 1.5 * 2^23
    constexpr int MAGIC = 0x4B400000;
    extern __shared__ __align__(16) float red[];  // [list of the batch][tile of the item][warp][row of x][16], the cluster's sums, x's stage
    const Place at(a);
    const int warps = int(blockDim.x) / 32;
    if (a.ks > 1) cluster_arrive();
    Stream<SL, DEPTH, BPG, ZEROS> in;
    in.begin(a, at);

    uint32_t xe[ROWS_X][SL][4], xo[ROWS_X][SL][4];  // column g: byte g of the row, the even and the odd k
    int xc[ROWS_X][SL][GPC][2];                     // columns 2t and 2t + 1: what a group's sum starts from (or its sum of x)
    float back[ROWS_X][2];                          // 2^(16 t - up) in two factors; NaN where x is not finite
    const auto load = [&](int c0) {
        // each lane converts a piece of 8 k of every eighth unit (32 k); the
        // columns' owners get them through this warp's shared memory
        constexpr int UNITS = SL * 4, MINE = (UNITS + 7) / 8;
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
            const int up = top == 0 || odd ? 0 : 61 - ilogbf(__uint_as_float(top));  // x * 2^up is below 2^62
            const float up0 = ldexpf(1.0f, up / 2), up1 = ldexpf(1.0f, up - up / 2);
            const int down = 16 * at.t - up;
            back[row][0] = odd ? NAN : ldexpf(1.0f, down / 2), back[row][1] = ldexpf(1.0f, down - down / 2);
#pragma unroll
            for (int x = 0; x < MINE; x++) {
                const int unit = at.g + 8 * x;
                uint32_t lo[8], hi[8];
#pragma unroll
                for (int i = 0; i < 8; i++) {  // plus 128 in each digit but the highest: its bytes are the digits plus 128
                    const unsigned long long n = (unsigned long long)(odd ? 0 : __float2ll_rn(v[x][i] * up0 * up1)) + 0x0080808080808080ull;
                    lo[i] = uint32_t(n), hi[i] = uint32_t(n >> 32);
                }
                // byte b of four numbers in word b, for the even k and the odd
                uint32_t word[2][8];
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    bytes_of(lo[h], lo[2 + h], lo[4 + h], lo[6 + h], word[h]);
                    bytes_of(hi[h], hi[2 + h], hi[4 + h], hi[6 + h], word[h] + 4);
#pragma unroll
                    for (int b = 0; b < 7; b++) word[h][b] ^= 0x80808080u;
                }
                if (unit < UNITS)
#pragma unroll
                    for (int b = 0; b < 8; b++) stage[(unit * COLS + row * 8 + b) * 4 + at.t] = make_uint2(word[0][b], word[1][b]);
            }
        }
        __syncwarp();
#pragma unroll
        for (int row = 0; row < ROWS_X; row++)
#pragma unroll
            for (int c = 0; c < SL; c++) {
                int sum[GPC] = {};
#pragma unroll
                for (int u = 0; u < 4; u++) {
                    const uint2 v = stage[((c * 4 + u) * COLS + row * 8 + at.g) * 4 + at.t];
                    xe[row][c][u] = v.x, xo[row][c][u] = v.y;
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
                        xc[row][c][j][h] = ZEROS ? other : MAGIC - 8 * other;
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
                    float acc[ROWS_X][4] = {};
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
                        int v[ROWS_X][4];
#pragma unroll
                        for (int u = 0; u < 4; u++) {
                            const int j = c * GPC + u / BPG;
                            const uint32_t lo0 = w0[u] & 0x0F0F0F0Fu, lo1 = w1[u] & 0x0F0F0F0Fu;
                            const uint32_t hi0 = (w0[u] >> 4) & 0x0F0F0F0Fu, hi1 = (w1[u] >> 4) & 0x0F0F0F0Fu;
#pragma unroll
                            for (int r = 0; r < ROWS_X; r++) {
                                const int *x = xc[r][c][u / BPG];
                                if (u % BPG == 0) {
                                    if constexpr (ZEROS) {
                                        v[r][0] = MAGIC - int(z[j][0]) * x[0], v[r][1] = MAGIC - int(z[j][0]) * x[1];
                                        v[r][2] = MAGIC - int(z[j][1]) * x[0], v[r][3] = MAGIC - int(z[j][1]) * x[1];
                                    } else {
                                        v[r][0] = v[r][2] = x[0], v[r][1] = v[r][3] = x[1];
                                    }
                                }
                                asm volatile(
                                    "mma.sync.aligned.m16n8k32.row.col.s32.u8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                                    : "+r"(v[r][0]), "+r"(v[r][1]), "+r"(v[r][2]), "+r"(v[r][3])
                                    : "r"(lo0), "r"(lo1), "r"(hi0), "r"(hi1), "r"(xe[r][c][u]), "r"(xo[r][c][u]));
                                if (u % BPG == BPG - 1) {
#pragma unroll
                                    for (int e = 0; e < 4; e++)
                                        acc[r][e] = fmaf(__int_as_float(v[r][e]) - 12582912.0f, s[j][e >> 1], acc[r][e]);
                                }
                            }
                        }
                        if (more) in.chunk(a, at, d, c);
                    }
                    const float bias[2] = {in.b[d][0], in.b[d][1]};
                    if (more) in.biases(a, at, d);
                    // columns 2t and 2t + 1 are bytes 2t, 2t + 1 of a row: one number, in every lane
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        float y[ROWS_X];
#pragma unroll
                        for (int r = 0; r < ROWS_X; r++) {
                            y[r] = fmaf(acc[r][2 * h + 1], 256.0f, acc[r][2 * h]) * back[r][0] * back[r][1];
                            y[r] += __shfl_xor_sync(0xffffffffu, y[r], 1);
                            y[r] += __shfl_xor_sync(0xffffffffu, y[r], 2);
                        }
                        const int m = at.t;  // lane m of a row's four has row m of x
                        if (m < ROWS_X) {
                            const float mine = y[ROWS_X == 2 && m ? ROWS_X - 1 : 0];
                            if (a.direct) {
                                const int n = at.row(a, b0 + i, at.r_warp) + d * 16 + at.g + 8 * h;
                                if (n < a.n) finish(m, n, mine, bias[h], 1.0f);
                            } else {
                                float *to = red + (((i * a.depth + d) * warps + at.warp) * ROWS_X + m) * 16 + at.g + 8 * h;
                                *to = lap > 0 ? *to + mine : mine;
                            }
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
    using Q = IntTile<BPG, ROWS_X>;
    const cudaError_t e = raise_shared<q4_int_kernel<XT, BPG, ZEROS, ROWS_X>>(Q::SHARED);
    if (e != cudaSuccess) return e;
    a.cols_rows = a.m;
    return launch_q4(reinterpret_cast<const void *>(q4_int_kernel<XT, BPG, ZEROS, ROWS_X>), a, Q::WARPS, Q::SL, Q::DEPTH, BPG, ROWS_X,
                     Q::STAGE, Q::SHARED, true, false, stream);
}

template <class XT, int BPG>
cudaError_t start_g(const Q4Args &a, cudaStream_t s) {
    if constexpr (sizeof(XT) == 4)  // two rows of the other types are k_q4.cu's
        if (a.m == 2) return a.zeros ? start<XT, BPG, true, 2>(a, s) : start<XT, BPG, false, 2>(a, s);
    return a.zeros ? start<XT, BPG, true, 1>(a, s) : start<XT, BPG, false, 1>(a, s);
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
