// ppocr_matvec_q4: a few rows of x times a matrix of 4-bit weights,
//
//     y[m][n] = sum_k x[m][k] (q[n][k] - z[n][k / G]) s[n][k / G] + b[n].
//
// The weights are the matrix instruction's A operand (16 of their rows, one
// warp), x its B operand (8 columns: rows of x), so few rows of x cost the
// same weight traffic as one and sums stay in f32. A weight becomes q - z, a
// small integer that f16 and bf16 hold exactly; its scale multiplies each
// group's f32 sum. x enters exactly too: f16 and bf16 as they are, e4m3 as
// f16, f32 as three bf16 columns (8 bits of the mantissa each) whose sums
// are added at the end. The instruction sums over k in any order as long as
// both operands agree, so a lane's four k slots of two instructions are 8
// consecutive weights, one 32-bit word, and x is staged in that order.
//
// A block of 8 warps takes 8 / WK row tiles at a time, WK warps a tile, each
// every WK-th step of 128 k; weights come through a ring of cp.async stages
// per warp that runs on across tiles, x lies in shared memory (in chunks of
// k where it does not fit), and the WK partial sums meet there in a fixed
// order. Bound by the weights' bytes.
#include <cuda_fp8.h>

#include <type_traits>

#include "block.cuh"

namespace ppocr {

namespace {

constexpr int WARPS = 8, THREADS = WARPS * 32;
constexpr int STEP = 128;               // k a warp takes at a time: 64 bytes of each of 16 rows
constexpr int STAGES = 4;
constexpr int W_BYTES = 16 * 64;        // a stage's weights
constexpr int S_BYTES = 16 * 4 * 8;     // a stage's (scale, zero point) per row and 32 k
constexpr int RING = STAGES * (W_BYTES + S_BYTES);
// Staged x: two blocks an SM with up to 16 columns, one with 32 (whose 8 warps'
// turn of x takes 64 KB).
constexpr int x_bytes_of(int ct) { return (ct <= 2 ? 40 : 64) * 1024; }

struct Q4Args {
    const void *x;
    const float *x_scales;
    const uint8_t *w;
    const void *scales;
    const uint8_t *zeros;
    const float *bias;
    void *y;
    int64_t x_row, y_row, w_row;
    int m, k, n, group, groups;
    int scale_type, y_type;
    int x_groups;   // scales a row of x has (e4m3): 0 none, 1 the row's, else one a group
    int wk;         // warps that share a row tile
    int steps, chunk_steps, cols_rows;  // steps of k in all and per staged chunk; rows of x a pass takes
    bool w_vec, x_vec;
};

struct e4m3 {
    uint8_t bits;
};

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

// f16: 0x6400 | q is 1024 + q, 0x6400 | q << 4 is 1024 + 16 q; both less their
// offset are exact.
template <>
__device__ __forceinline__ void unpack<__half>(uint32_t w, uint32_t z, uint32_t out[4]) {
    const uint32_t z1 = (0x6400u + z) * 0x10001u;          // 1024 + z, twice
    const uint32_t z16 = (0xD400u + (z << 4)) * 0x10001u;  // -(64 + z), twice
    const uint32_t sixteenth = 0x2C002C00u;                // 1 / 16
    const uint32_t w8 = w >> 8;
    const uint32_t a = (w & 0x000F000Fu) | 0x64006400u, b = (w & 0x00F000F0u) | 0x64006400u;
    const uint32_t c = (w8 & 0x000F000Fu) | 0x64006400u, d = (w8 & 0x00F000F0u) | 0x64006400u;
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
        const uint32_t v = ((w >> (4 * i)) & 0x000F000Fu) | 0x3B003B00u;
        const __nv_bfloat162 r =
            __hsub2(*reinterpret_cast<const __nv_bfloat162 *>(&v), *reinterpret_cast<const __nv_bfloat162 *>(&z1));
        out[i] = *reinterpret_cast<const uint32_t *>(&r);
    }
}

__device__ __forceinline__ float load_scale(const Q4Args &a, int64_t at) {
    if (a.scale_type == PPOCR_F16) return __half2float(static_cast<const __half *>(a.scales)[at]);
    if (a.scale_type == PPOCR_BF16) return __bfloat162float(static_cast<const __nv_bfloat16 *>(a.scales)[at]);
    return static_cast<const float *>(a.scales)[at];
}

// Eight values of x as f32 (exact for every type); zeros past k.
template <class XT>
__device__ __forceinline__ void load_x(const Q4Args &a, int row, int k, float v[8]) {
    const XT *p = static_cast<const XT *>(a.x) + row * a.x_row + k;
    if (a.x_vec && k + 8 <= a.k) {
        if constexpr (sizeof(XT) == 4) {
            const float4 lo = __ldg(reinterpret_cast<const float4 *>(p)), hi = __ldg(reinterpret_cast<const float4 *>(p) + 1);
            v[0] = lo.x, v[1] = lo.y, v[2] = lo.z, v[3] = lo.w, v[4] = hi.x, v[5] = hi.y, v[6] = hi.z, v[7] = hi.w;
        } else if constexpr (sizeof(XT) == 2) {
            const uint4 u = __ldg(reinterpret_cast<const uint4 *>(p));
            const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const uint16_t h = uint16_t(w[i / 2] >> (16 * (i & 1)));
                v[i] = to_f32(*reinterpret_cast<const XT *>(&h));
            }
        } else {
            const uint2 u = __ldg(reinterpret_cast<const uint2 *>(p));
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const __nv_fp8_storage_t b = __nv_fp8_storage_t((i < 4 ? u.x : u.y) >> (8 * (i & 3)));
                v[i] = __half2float(__half(__nv_cvt_fp8_to_halfraw(b, __NV_E4M3)));
            }
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < 8; i++) {
        v[i] = 0.0f;
        if (k + i < a.k) {
            if constexpr (sizeof(XT) == 1)
                v[i] = __half2float(__half(__nv_cvt_fp8_to_halfraw(__nv_fp8_storage_t(p[i].bits), __NV_E4M3)));
            else
                v[i] = to_f32(p[i]);
        }
    }
}

// The part of x that column `part` of its row holds. f32 in three: the top 8
// bits of the mantissa, the next 8, the last 8, each exact in bf16; an
// infinity or NaN stays whole in the first.
template <class XT>
__device__ __forceinline__ float part_of(float x, int part) {
    if constexpr (Enter<XT>::PARTS == 1) return x;
    if (!(fabsf(x) < INFINITY)) return part == 0 ? x : 0.0f;
    const float hi = __uint_as_float(__float_as_uint(x) & 0xFFFF0000u), rest = x - hi;
    const float mid = __uint_as_float(__float_as_uint(rest) & 0xFFFF0000u);
    return part == 0 ? hi : part == 1 ? mid : rest - mid;
}

// BPG: 32-k blocks a weight group, 1, 2 or 4 (1 serves every multiple of 32).
template <class XT, int CT, int BPG, bool ZEROS>
__global__ void __launch_bounds__(THREADS, CT <= 2 ? 2 : 1) q4_kernel(const __grid_constant__ Q4Args a) {
    using M = typename Enter<XT>::M;
    constexpr int PARTS = Enter<XT>::PARTS, COLS = 8 * CT;
    extern __shared__ __align__(16) unsigned char smem[];
    const int tid = threadIdx.x, warp = tid / 32, lane = tid & 31, g = lane >> 2, t = lane & 3;
    unsigned char *ring = smem + warp * RING;
    float *red = reinterpret_cast<float *>(smem + WARPS * RING);          // [2][WARPS][16][COLS]
    unsigned char *xs = smem + WARPS * RING + 2 * WARPS * 16 * COLS * 4;  // [block][cols][t] of 16 bytes
    const uint32_t ring_s = shared_u32(ring), xs_s = shared_u32(xs);

    const int wr = WARPS / a.wk, k_warp = warp % a.wk, r_warp = warp / a.wk;
    const int tiles = (a.n + 15) / 16, turns = (a.steps + a.wk - 1) / a.wk;
    const int m0 = blockIdx.y * a.cols_rows, rows = min(a.cols_rows, a.m - m0), cols = rows * PARTS;
    const bool once = a.chunk_steps >= a.steps;

    // x's chunk from step `s0` on into shared memory
    const auto stage_x = [&](int s0) {
        const int blocks = min(a.chunk_steps, a.steps - s0) * 4;
        for (int e = tid; e < blocks * rows * 4; e += THREADS) {
            const int q = e & 3, r = (e >> 2) % rows, b = (e >> 2) / rows;
            float v[8];
            load_x<XT>(a, m0 + r, (s0 * 4 + b) * 32 + q * 8, v);
#pragma unroll
            for (int part = 0; part < PARTS; part++) {
                uint32_t u[4];
#pragma unroll
                for (int i = 0; i < 4; i++) u[i] = pack2<M>(part_of<XT>(v[i], part), part_of<XT>(v[i + 4], part));
                *reinterpret_cast<uint4 *>(xs + ((b * cols + r * PARTS + part) * 4 + q) * 16) = make_uint4(u[0], u[1], u[2], u[3]);
            }
        }
    };

    // this warp's u-th step: tile (u / turns) of its block's list, turn u % turns
    const int first_tile = blockIdx.x * wr + r_warp, tile_step = gridDim.x * wr;
    const int groups_of_tiles = (tiles + wr - 1) / wr;
    const int my_groups = groups_of_tiles > int(blockIdx.x) ? (groups_of_tiles - int(blockIdx.x) + int(gridDim.x) - 1) / int(gridDim.x) : 0;

    // prefetch cursor
    int f_tile = first_tile, f_turn = 0, f_left = my_groups * turns;
    float2 held[2] = {};  // scales and zero points on their way to shared memory
    const auto fetch = [&](int slot) {
        if (f_left > 0) {
            const int step = f_turn * a.wk + k_warp;
            const bool on = f_tile < tiles && step < a.steps;
            if (on) {
                const uint32_t to = ring_s + slot * (W_BYTES + S_BYTES);
                const int half_k = (a.k + 1) / 2;
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    const int r = (lane >> 2) + 8 * i, c = lane & 3, n = f_tile * 16 + r, at = step * 64 + c * 16;
                    int valid = n < a.n ? half_k - at : 0;
                    valid = valid < 0 ? 0 : valid > 16 ? 16 : valid;
                    const uint8_t *from = valid ? a.w + int64_t(n) * a.w_row + at : a.w;
                    const int place = r * 64 + ((c ^ ((r >> 1) & 3)) * 16);
                    if (a.w_vec) {
                        copy_async<16>(to + place, from, valid);
                    } else {
                        for (int j = 0; j < 16; j++) ring[slot * (W_BYTES + S_BYTES) + place + j] = j < valid ? from[j] : 0;
                    }
                }
                const int n = f_tile * 16 + (lane >> 1);
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    const int group = ((step * 4 + (lane & 1) * 2 + i) * 32) / a.group;
                    held[i] = make_float2(0.0f, __uint_as_float(8u));
                    if (n < a.n && group < a.groups) {
                        const int64_t at = int64_t(n) * a.groups + group;
                        held[i].x = load_scale(a, at) * Enter<XT>::SCALE;
                        if constexpr (ZEROS) held[i].y = __uint_as_float(uint32_t(a.zeros[at]) & 15u);
                    }
                }
            }
            f_left--;
            if (++f_turn == turns) f_turn = 0, f_tile += tile_step;
        }
        copy_commit();
    };
    const auto put_scales = [&](int slot) {
        float2 *s = reinterpret_cast<float2 *>(ring + slot * (W_BYTES + S_BYTES) + W_BYTES);
        s[(lane >> 1) * 4 + (lane & 1) * 2] = held[0];
        s[(lane >> 1) * 4 + (lane & 1) * 2 + 1] = held[1];
    };
#pragma unroll
    for (int s = 0; s < STAGES - 1; s++) {
        fetch(s);
        put_scales(s);
    }
    if (once) {
        stage_x(0);
        __syncthreads();
    }

    int slot = 0, buf = 0;
    for (int list = 0; list < my_groups; list++) {
        const int tile = first_tile + list * tile_step;
        float acc[CT][4] = {};
        for (int turn = 0; turn < turns; turn++) {
            const int step = turn * a.wk + k_warp;
            if (!once && (turn * a.wk) % a.chunk_steps == 0) {
                __syncthreads();
                stage_x(turn * a.wk);
                __syncthreads();
            }
            copy_wait<STAGES - 2>();
            __syncwarp();
            const int next = slot == 0 ? STAGES - 1 : slot - 1;
            fetch(next);
            if (tile < tiles && step < a.steps) {
                const unsigned char *ws = ring + slot * (W_BYTES + S_BYTES);
                const float2 *ss = reinterpret_cast<const float2 *>(ws + W_BYTES);
                const int b0 = (once ? step : step % a.chunk_steps) * 4;
#pragma unroll
                for (int b = 0; b < 4; b += BPG) {
                    float sum[CT][4] = {};
                    const float2 s0 = ss[g * 4 + b], s1 = ss[(g + 8) * 4 + b];
                    const uint32_t z0 = ZEROS ? __float_as_uint(s0.y) : 8u, z1 = ZEROS ? __float_as_uint(s1.y) : 8u;
#pragma unroll
                    for (int c = b; c < b + BPG; c++) {
                        const int at = ((c ^ ((g >> 1) & 3)) * 16) + t * 4;
                        const uint32_t w0 = *reinterpret_cast<const uint32_t *>(ws + g * 64 + at);
                        const uint32_t w1 = *reinterpret_cast<const uint32_t *>(ws + (g + 8) * 64 + at);
                        uint32_t p0[4], p1[4];
                        unpack<M>(w0, z0, p0);
                        unpack<M>(w1, z1, p1);
                        const uint32_t lo[4] = {p0[0], p1[0], p0[1], p1[1]}, hi[4] = {p0[2], p1[2], p0[3], p1[3]};
#pragma unroll
                        for (int ct = 0; ct < CT; ct++) {
                            const int col = ct * 8 + g;
                            uint4 xf = make_uint4(0, 0, 0, 0);
                            if (col < cols)
                                asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];"
                                             : "=r"(xf.x), "=r"(xf.y), "=r"(xf.z), "=r"(xf.w)
                                             : "r"(xs_s + uint32_t((((b0 + c) * cols + col) * 4 + t) * 16)));
                            mma16<M>(sum[ct], lo, xf.x, xf.y);
                            mma16<M>(sum[ct], hi, xf.z, xf.w);
                        }
                    }
#pragma unroll
                    for (int ct = 0; ct < CT; ct++) {
                        float f0 = 1.0f, f1 = 1.0f;
                        if (sizeof(XT) == 1 && a.x_groups > 1) {
                            const int group = (step * 4 + b) * 32 / a.group, c0 = ct * 8 + t * 2;
                            if (group < a.groups) {
                                if (c0 < rows) f0 = __ldg(a.x_scales + int64_t(m0 + c0) * a.x_groups + group);
                                if (c0 + 1 < rows) f1 = __ldg(a.x_scales + int64_t(m0 + c0 + 1) * a.x_groups + group);
                            }
                        }
                        acc[ct][0] = fmaf(sum[ct][0], s0.x * f0, acc[ct][0]);
                        acc[ct][1] = fmaf(sum[ct][1], s0.x * f1, acc[ct][1]);
                        acc[ct][2] = fmaf(sum[ct][2], s1.x * f0, acc[ct][2]);
                        acc[ct][3] = fmaf(sum[ct][3], s1.x * f1, acc[ct][3]);
                    }
                }
            }
            put_scales(next);
            slot = slot == STAGES - 1 ? 0 : slot + 1;
        }
        // the warps' partial sums: [warp][row of the tile][column]
        float *mine = red + (buf * WARPS + warp) * 16 * COLS;
#pragma unroll
        for (int ct = 0; ct < CT; ct++) {
            *reinterpret_cast<float2 *>(mine + g * COLS + ct * 8 + t * 2) = make_float2(acc[ct][0], acc[ct][1]);
            *reinterpret_cast<float2 *>(mine + (g + 8) * COLS + ct * 8 + t * 2) = make_float2(acc[ct][2], acc[ct][3]);
        }
        __syncthreads();
        if (tile < tiles) {
            const float *from = red + (buf * WARPS + r_warp * a.wk) * 16 * COLS;
            for (int e = k_warp * 32 + lane; e < 16 * rows; e += a.wk * 32) {
                const int r = e & 15, m = e >> 4, n = tile * 16 + r;
                if (n >= a.n) continue;
                float y = 0.0f;
                for (int p = PARTS - 1; p >= 0; p--)
                    for (int w = 0; w < a.wk; w++) y += from[(w * 16 + r) * COLS + m * PARTS + p];
                if (sizeof(XT) == 1 && a.x_groups == 1) y *= __ldg(a.x_scales + m0 + m);
                if (a.bias) y += __ldg(a.bias + n);
                const int64_t at = int64_t(m0 + m) * a.y_row + n;
                if (a.y_type == PPOCR_F32)
                    static_cast<float *>(a.y)[at] = y;
                else if (a.y_type == PPOCR_F16)
                    static_cast<__half *>(a.y)[at] = __float2half_rn(y);
                else
                    static_cast<__nv_bfloat16 *>(a.y)[at] = __float2bfloat16_rn(y);
            }
        }
        buf ^= 1;  // the next tile's sums go elsewhere: one barrier a tile
    }
    copy_wait<0>();
}

template <class XT, int CT, int BPG, bool ZEROS>
cudaError_t start(Q4Args a, cudaStream_t stream) {
    constexpr int PARTS = Enter<XT>::PARTS, COLS = 8 * CT;
    constexpr int X_BYTES = x_bytes_of(CT), FIXED = WARPS * RING + 2 * WARPS * 16 * COLS * 4;
    const cudaError_t e = raise_shared<q4_kernel<XT, CT, BPG, ZEROS>>(FIXED + X_BYTES);
    if (e != cudaSuccess) return e;
    a.cols_rows = COLS / PARTS < a.m ? COLS / PARTS : a.m;
    const int passes = (a.m + a.cols_rows - 1) / a.cols_rows;
    // chunks of whole turns: a step of x takes 256 bytes a column
    const int fit = X_BYTES / (256 * a.cols_rows * PARTS);
    a.chunk_steps = fit >= a.steps ? a.steps : fit / a.wk * a.wk;
    const int x_bytes = a.chunk_steps * 256 * a.cols_rows * PARTS;
    const int wr = WARPS / a.wk, lists = ((a.n + 15) / 16 + wr - 1) / wr;
    const int most = sm_count() * (CT <= 2 ? 2 : 1);
    q4_kernel<XT, CT, BPG, ZEROS><<<dim3(unsigned(lists < most ? lists : most), unsigned(passes)), THREADS, FIXED + x_bytes, stream>>>(a);
    return cudaGetLastError();
}

template <class XT, int CT>
cudaError_t start_g(const Q4Args &a, cudaStream_t s) {
    if (a.group % 128 == 0) return a.zeros ? start<XT, CT, 4, true>(a, s) : start<XT, CT, 4, false>(a, s);
    if (a.group % 64 == 0) return a.zeros ? start<XT, CT, 2, true>(a, s) : start<XT, CT, 2, false>(a, s);
    return a.zeros ? start<XT, CT, 1, true>(a, s) : start<XT, CT, 1, false>(a, s);
}

template <class XT>
cudaError_t start_x(const Q4Args &a, cudaStream_t s) {
    const int cols = a.m * Enter<XT>::PARTS;
    if (cols <= 8) return start_g<XT, 1>(a, s);
    if (cols <= 16) return start_g<XT, 2>(a, s);
    return start_g<XT, 4>(a, s);
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
    const uint64_t yn = ((s->rows - 1) * uint64_t(a.y_row) + s->n) * ys, wn = (s->n - 1) * uint64_t(a.w_row) + (uint64_t(s->k) + 1) / 2;
    if (overlap(y, yn, x, ((s->rows - 1) * uint64_t(a.x_row) + s->k) * xs) || overlap(y, yn, w, wn) ||
        overlap(y, yn, scales, s->n * groups * ss) || (zeros && overlap(y, yn, zeros, s->n * groups)) ||
        (bias && overlap(y, yn, bias, s->n * uint64_t(4))) ||
        (x_scales && overlap(y, yn, x_scales, s->rows * (s->x_group ? groups : 1) * 4)))
        return refuse(PPOCR_E_ARG, me, "y overlaps another buffer");
    a.scale_type = s->scale_type, a.y_type = s->y_type;
    // one group in all is the row's scale
    a.x_groups = !x_scales ? 0 : s->x_group ? int(groups) : 1;
    a.steps = (a.k + STEP - 1) / STEP;
    a.wk = 1;
    while (a.wk < WARPS && a.wk * 2 <= a.steps) a.wk *= 2;
    a.w_vec = aligned(w, 16) && a.w_row % 16 == 0;
    a.x_vec = uint64_t(a.x_row) * xs % (xs == 1 ? 8 : 16) == 0 && aligned(x, xs == 1 ? 8 : 16);
    const auto str = static_cast<cudaStream_t>(stream);
    const cudaError_t e = s->x_type == PPOCR_F32    ? start_x<float>(a, str)
                          : s->x_type == PPOCR_F16  ? start_x<__half>(a, str)
                          : s->x_type == PPOCR_BF16 ? start_x<__nv_bfloat16>(a, str)
                                                    : start_x<e4m3>(a, str);
    return e == cudaSuccess ? int(PPOCR_OK) : refuse(PPOCR_E_DEVICE, me, cudaGetErrorString(e));
}
