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
// A block of 8 warps takes 8 / wk row tiles at a time, wk warps a tile, each
// every wk-th step of k; weights come through a ring of cp.async stages per
// warp that runs on across tiles, x lies in shared memory, and the wk partial
// sums meet there in a fixed order. Where x is too much for one block, or the
// tiles are too few for the card, a cluster's blocks share k and their sums
// meet through distributed shared memory (past eight blocks' worth of x, it
// is staged in chunks). Bound by the weights' bytes.
#include <cuda_fp8.h>

#include <type_traits>

#include "block.cuh"

namespace ppocr {

namespace {

constexpr int WARPS = 8, THREADS = WARPS * 32;

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
    int cols_rows;  // rows of x a pass takes
    int ks, wk;     // blocks of a cluster, and warps of a block, that share a row tile
    int steps, share_steps, chunk_steps;  // of k: in all, a block's share, staged at a time
    int keep;       // lists of tiles whose partial sums a cluster gathers before it joins them
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

__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ float peer_load(const float *p, uint32_t rank) {
    uint32_t at;
    float v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(shared_u32(p)), "r"(rank));
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(at) : "memory");
    return v;
}
__device__ __forceinline__ uint4 lds128(uint32_t a) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a));
    return v;
}
__device__ __forceinline__ uint32_t lds32(uint32_t a) {
    uint32_t v;
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(a));
    return v;
}

// A step: 256 k, 128 bytes of each of a tile's 16 rows of weights, swizzled as
// the tensor copies do (16-byte chunk c of row r at c ^ (r % 8)).
constexpr int STEP = 256, BLOCKS = STEP / 32, ROW = STEP / 2, W_BYTES = 16 * ROW;

// Sizes of one variant. CT: 8-column tiles of x; BPG: 32-k blocks a weight
// group (4, 2, or 1, which serves every multiple of 32).
template <int CT, int BPG, bool ZEROS>
struct Q4Tile {
    static constexpr int COLS = 8 * CT;
    static constexpr int SB = BLOCKS / BPG;  // scales a row and step
    static constexpr int SPL = SB / 2;       // of which a lane fetches
    static constexpr int S_BYTES = 16 * SB * (ZEROS ? 8 : 4);
    static constexpr int STAGES = CT <= 2 ? 3 : 4;
    // weights of every warp and stage first (the swizzle wants 1 KB borders),
    // then the scales, the partial sums, the barriers, 64 zeros and x
    static constexpr int SCALES = WARPS * STAGES * W_BYTES, RED = SCALES + WARPS * STAGES * S_BYTES;
    static constexpr int BARS = RED + 2 * WARPS * 16 * COLS * 4, ZERO = BARS + WARPS * STAGES * 8, FIXED = ZERO + 64;
    // staged x and, behind it, a cluster's partial results (one list at least);
    // two blocks an SM up to 16 columns
    static constexpr int X_BYTES = (CT == 1 ? 24 : CT == 2 ? 16 : 64) * 1024, PART_BYTES = (CT == 4 ? 16 : 8) * 1024;
    static_assert(CT > 2 || FIXED + X_BYTES + PART_BYTES <= 113 * 1024, "two blocks an SM");
    static_assert(PART_BYTES >= WARPS * 16 * COLS * 4, "one list of partial results");
};

template <class XT, int CT, int BPG, bool ZEROS>
__global__ void __launch_bounds__(THREADS, CT <= 2 ? 2 : 1)
    q4_kernel(const __grid_constant__ Q4Args a, const __grid_constant__ CUtensorMap map) {
    using M = typename Enter<XT>::M;
    using Q = Q4Tile<CT, BPG, ZEROS>;
    constexpr int PARTS = Enter<XT>::PARTS, COLS = Q::COLS, STAGES = Q::STAGES, SB = Q::SB;
    extern __shared__ __align__(1024) unsigned char smem[];
    const int tid = threadIdx.x, warp = tid / 32, lane = tid & 31, g = lane >> 2, t = lane & 3;
    unsigned char *ring = smem + warp * STAGES * W_BYTES, *sring = smem + Q::SCALES + warp * STAGES * Q::S_BYTES;
    float *red = reinterpret_cast<float *>(smem + Q::RED);  // [2][WARPS][16][COLS]
    unsigned char *xs = smem + Q::FIXED;                    // [block][column][t] of 16 bytes
    const uint32_t ring_s = shared_u32(ring), bars = shared_u32(smem + Q::BARS) + warp * STAGES * 8;

    // this block's share of k (one of a cluster's blocks) and of the tiles
    const int ks = a.ks, rank = ks > 1 ? int(blockIdx.x) % ks : 0, team = int(blockIdx.x) / ks, teams = int(gridDim.x) / ks;
    const int s_lo = rank * a.share_steps, s_hi = min(a.steps, s_lo + a.share_steps);
    const int wr = WARPS / a.wk, k_warp = warp % a.wk, r_warp = warp / a.wk;
    const int tiles = (a.n + 15) / 16, turns = (a.share_steps + a.wk - 1) / a.wk;
    const int m0 = blockIdx.y * a.cols_rows, rows = min(a.cols_rows, a.m - m0);
    // x's columns: as many as there are for one column tile, else whole tiles
    const int cols = CT == 1 ? rows * PARTS : COLS;
    const bool once = a.chunk_steps >= a.share_steps;
    const int lists = (tiles + wr - 1) / wr, my_lists = lists > team ? (lists - team + teams - 1) / teams : 0;
    float *part = reinterpret_cast<float *>(xs + a.chunk_steps * BLOCKS * 64 * cols);

    if (lane == 0)
        for (int s = 0; s < STAGES; s++) bar_init(bars + s * 8, 1);
    if (tid < 16) reinterpret_cast<uint32_t *>(smem + Q::ZERO)[tid] = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    __syncthreads();

    // x's chunk of steps from `s0` on into shared memory. Groups of 128 k: a
    // lane's four words of a row are 32 consecutive weights, so k is staged in
    // that order (one 16-byte load a row); else a lane's word is its 8 k of a block.
    const auto stage_x = [&](int s0) {
        const int blocks = max(0, min(a.chunk_steps, s_hi - s0)) * BLOCKS, q = tid & 3;
        for (int b = tid >> 2; b < blocks; b += THREADS / 4) {
            const int k = s0 * STEP + (BPG == 4 ? (b >> 2) * 128 + q * 32 + (b & 3) * 8 : b * 32 + q * 8);
            for (int r = 0; r < (CT == 1 ? rows : COLS / PARTS); r++) {
                float v[8] = {};
                if (r < rows) load_x<XT>(a, m0 + r, k, v);
#pragma unroll
                for (int p = 0; p < PARTS; p++) {
                    uint32_t u[4];
#pragma unroll
                    for (int i = 0; i < 4; i++) u[i] = pack2<M>(part_of<XT>(v[i], p), part_of<XT>(v[i + 4], p));
                    *reinterpret_cast<uint4 *>(xs + ((b * cols + r * PARTS + p) * 4 + q) * 16) = make_uint4(u[0], u[1], u[2], u[3]);
                }
            }
            if constexpr (CT > 1 && COLS % PARTS != 0)
                for (int c = COLS / PARTS * PARTS; c < COLS; c++)
                    *reinterpret_cast<uint4 *>(xs + ((b * cols + c) * 4 + q) * 16) = make_uint4(0, 0, 0, 0);
        }
    };

    // the prefetch cursor: the tile it is at, this lane's scales there
    const int s_row = lane >> 1, s_col = (lane & 1) * Q::SPL;
    int f_tile = team * wr + r_warp, f_turn = 0, f_left = my_lists * turns;
    float held[Q::SPL] = {};
    uint32_t held_z[Q::SPL] = {};
    const auto fetch = [&](int slot) {
        if (f_left <= 0) return;
        const int step = s_lo + f_turn * a.wk + k_warp;
        if (f_tile < tiles && step < s_hi) {
            if (a.w_vec) {
                if (lane == 0) {
                    arrive_expect(bars + slot * 8, W_BYTES);
                    tma_load_2d(ring_s + slot * W_BYTES, &map, step * ROW, f_tile * 16, bars + slot * 8);
                }
            } else {
                const int half_k = (a.k + 1) / 2, at = step * ROW;
                for (int e = lane; e < W_BYTES; e += 32) {
                    const int r = e / ROW, c = e % ROW, n = f_tile * 16 + r;
                    ring[slot * W_BYTES + r * ROW + (((c >> 4) ^ (r & 7)) << 4) + (c & 15)] =
                        n < a.n && at + c < half_k ? a.w[int64_t(n) * a.w_row + at + c] : 0;
                }
            }
            const int n = f_tile * 16 + s_row;
            const int64_t row = int64_t(n) * a.groups;
#pragma unroll
            for (int i = 0; i < Q::SPL; i++) {
                const int b = step * SB + s_col + i, group = a.group == 32 * BPG ? b : b * BPG * 32 / a.group;
                held[i] = 0.0f;
                held_z[i] = 8;
                if (n < a.n && group < a.groups) {
                    held[i] = load_scale(a, row + group) * Enter<XT>::SCALE;
                    if constexpr (ZEROS) held_z[i] = uint32_t(__ldg(a.zeros + row + group)) & 15u;
                }
            }
        }
        f_left--;
        if (++f_turn == turns) {
            f_turn = 0;
            f_tile += teams * wr;
        }
    };
    const auto put_scales = [&](int slot) {
        unsigned char *s = sring + slot * Q::S_BYTES;
#pragma unroll
        for (int i = 0; i < Q::SPL; i++) {
            if constexpr (ZEROS)
                reinterpret_cast<float2 *>(s)[s_row * SB + s_col + i] = make_float2(held[i], __uint_as_float(held_z[i]));
            else
                reinterpret_cast<float *>(s)[s_row * SB + s_col + i] = held[i];
        }
    };
#pragma unroll
    for (int s = 0; s < STAGES - 1; s++) {
        fetch(s);
        put_scales(s);
    }
    if (once) {
        stage_x(s_lo);
        __syncthreads();
    }

    // one output value: the row's scale, the bias, the type
    const auto finish = [&](int m, int n, float y) {
        if (sizeof(XT) == 1 && a.x_groups == 1) y *= __ldg(a.x_scales + m0 + m);
        if (a.bias) y += __ldg(a.bias + n);
        const int64_t at = int64_t(m0 + m) * a.y_row + n;
        if (a.y_type == PPOCR_F32)
            static_cast<float *>(a.y)[at] = y;
        else if (a.y_type == PPOCR_F16)
            static_cast<__half *>(a.y)[at] = __float2half_rn(y);
        else
            static_cast<__nv_bfloat16 *>(a.y)[at] = __float2bfloat16_rn(y);
    };

    // the instruction's rows g and g + 8 are the tile's rows `my` and my + 8: an
    // order in which the rows that one phase of a 16-byte load reads lie in different banks
    const int my = (g >> 1) | ((g & 1) << 2);
    const uint32_t w_at = uint32_t(my * ROW), key = uint32_t(my) << 4;
    // lanes with no column of x (one column tile) read zeros
    const bool has_x = CT > 1 || g < cols;
    const uint32_t x_at = has_x ? shared_u32(xs) + uint32_t(g * 64 + t * 16) : shared_u32(smem + Q::ZERO);
    const uint32_t x_step = has_x ? uint32_t(cols * 64) : 0;
    int slot = 0, buf = 0, kept = 0;
    uint32_t phase = 0;  // bit s: the parity stage s's next copy completes
    bool late = false;   // a copy that never came: the results say so
    for (int list = 0; list < my_lists; list++) {
        const int tile = (team + list * teams) * wr + r_warp;
        float acc[CT][4] = {};
        for (int turn = 0; turn < turns; turn++) {
            const int step = s_lo + turn * a.wk + k_warp;
            if (!once && (turn * a.wk) % a.chunk_steps == 0) {
                __syncthreads();
                stage_x(s_lo + turn * a.wk);
                __syncthreads();
            }
            const bool on = tile < tiles && step < s_hi;
            __syncwarp();  // the stage before is read, its scales' successors written
            const int next = slot == 0 ? STAGES - 1 : slot - 1;
            fetch(next);
            if (on) {
                if (a.w_vec) {
                    if (!late && !wait_copy(bars + slot * 8, (phase >> slot) & 1u)) late = true;
                    phase ^= 1u << slot;
                }
                const uint32_t ws = ring_s + uint32_t(slot * W_BYTES) + w_at;
                const unsigned char *ss = sring + slot * Q::S_BYTES;
                int in = step - s_lo;
                if (!once) in %= a.chunk_steps;
                uint32_t xb = x_at + uint32_t(in * BLOCKS) * x_step;
                const int blocks = min(BLOCKS, (a.k - step * STEP + 31) / 32);
#pragma unroll
                for (int b = 0; b < BLOCKS; b += BPG) {
                    if (b > 0 && b >= blocks) break;
                    float sum[CT][4] = {};
                    float s0, s1;
                    uint32_t z0 = 8, z1 = 8;
                    if constexpr (ZEROS) {
                        const float2 u0 = reinterpret_cast<const float2 *>(ss)[my * SB + b / BPG];
                        const float2 u1 = reinterpret_cast<const float2 *>(ss)[(my + 8) * SB + b / BPG];
                        s0 = u0.x, s1 = u1.x, z0 = __float_as_uint(u0.y), z1 = __float_as_uint(u1.y);
                    } else {
                        s0 = reinterpret_cast<const float *>(ss)[my * SB + b / BPG];
                        s1 = reinterpret_cast<const float *>(ss)[(my + 8) * SB + b / BPG];
                    }
                    uint32_t w0[BPG], w1[BPG];
                    if constexpr (BPG == 4) {
                        const uint32_t at = ws + (uint32_t((b + t) << 4) ^ key);
                        const uint4 u0 = lds128(at), u1 = lds128(at + 8 * ROW);
                        w0[0] = u0.x, w0[1] = u0.y, w0[2] = u0.z, w0[3] = u0.w;
                        w1[0] = u1.x, w1[1] = u1.y, w1[2] = u1.z, w1[3] = u1.w;
                    } else {
#pragma unroll
                        for (int c = 0; c < BPG; c++) {
                            const uint32_t at = ws + (uint32_t((b + c) << 4) ^ key) + t * 4;
                            w0[c] = lds32(at);
                            w1[c] = lds32(at + 8 * ROW);
                        }
                    }
#pragma unroll
                    for (int c = 0; c < BPG; c++) {
                        uint32_t p0[4], p1[4];
                        unpack<M>(w0[c], z0, p0);
                        unpack<M>(w1[c], z1, p1);
                        const uint32_t lo[4] = {p0[0], p1[0], p0[1], p1[1]}, hi[4] = {p0[2], p1[2], p0[3], p1[3]};
#pragma unroll
                        for (int ct = 0; ct < CT; ct++) {
                            const uint4 xf = lds128(CT == 1 ? xb : xb + uint32_t(((b + c) * COLS + ct * 8) * 64));
                            mma16<M>(sum[ct], lo, xf.x, xf.y);
                            mma16<M>(sum[ct], hi, xf.z, xf.w);
                        }
                        if constexpr (CT == 1) xb += x_step;
                    }
#pragma unroll
                    for (int ct = 0; ct < CT; ct++) {
                        float f0 = 1.0f, f1 = 1.0f;
                        if (sizeof(XT) == 1 && a.x_groups > 1) {
                            const int group = (step * BLOCKS + b) * 32 / a.group, c0 = ct * 8 + t * 2;
                            if (group < a.groups) {
                                if (c0 < rows) f0 = __ldg(a.x_scales + int64_t(m0 + c0) * a.x_groups + group);
                                if (c0 + 1 < rows) f1 = __ldg(a.x_scales + int64_t(m0 + c0 + 1) * a.x_groups + group);
                            }
                        }
                        acc[ct][0] = fmaf(sum[ct][0], s0 * f0, acc[ct][0]);
                        acc[ct][1] = fmaf(sum[ct][1], s0 * f1, acc[ct][1]);
                        acc[ct][2] = fmaf(sum[ct][2], s1 * f0, acc[ct][2]);
                        acc[ct][3] = fmaf(sum[ct][3], s1 * f1, acc[ct][3]);
                    }
                }
            }
            put_scales(next);
            slot = slot == STAGES - 1 ? 0 : slot + 1;
        }
        if (late) acc[0][0] = acc[0][1] = acc[0][2] = acc[0][3] = NAN;
        // the warps' partial sums: [warp][row of the tile][column]
        float *mine = red + (buf * WARPS + warp) * 16 * COLS;
#pragma unroll
        for (int ct = 0; ct < CT; ct++) {
            *reinterpret_cast<float2 *>(mine + my * COLS + ct * 8 + t * 2) = make_float2(acc[ct][0], acc[ct][1]);
            *reinterpret_cast<float2 *>(mine + (my + 8) * COLS + ct * 8 + t * 2) = make_float2(acc[ct][2], acc[ct][3]);
        }
        __syncthreads();
        const float *from = red + (buf * WARPS + r_warp * a.wk) * 16 * COLS;
        for (int e = k_warp * 32 + lane; e < 16 * rows; e += a.wk * 32) {
            const int r = e & 15, m = e >> 4, n = tile * 16 + r;
            float y = 0.0f;
            for (int p = PARTS - 1; p >= 0; p--)
                for (int w = 0; w < a.wk; w++) y += from[(w * 16 + r) * COLS + m * PARTS + p];
            if (ks > 1)
                part[(kept * wr + r_warp) * 16 * rows + e] = y;
            else if (n < a.n)
                finish(m, n, y);
        }
        buf ^= 1;  // the next tile's sums go elsewhere: one barrier a tile
        if (ks > 1 && (++kept == a.keep || list + 1 == my_lists)) {
            // the cluster's sums over k, in rank order; block `rank` joins every
            // ks-th value
            cluster_sync();
            const int first = team + (list + 1 - kept) * teams;
            for (int e = rank * THREADS + tid; e < kept * wr * 16 * rows; e += ks * THREADS) {
                const int in = e % (16 * rows), at = e / (16 * rows);
                const int n = ((first + at / wr * teams) * wr + at % wr) * 16 + (in & 15);
                float y = 0.0f;
                for (int x = 0; x < ks; x++) y += peer_load(part + e, uint32_t(x));
                if (n < a.n) finish(in >> 4, n, y);
            }
            cluster_sync();
            kept = 0;
        }
    }
}

template <class XT, int CT, int BPG, bool ZEROS>
cudaError_t start(Q4Args a, cudaStream_t stream) {
    using Q = Q4Tile<CT, BPG, ZEROS>;
    constexpr int PARTS = Enter<XT>::PARTS;
    const cudaError_t e = raise_shared<q4_kernel<XT, CT, BPG, ZEROS>>(Q::FIXED + Q::X_BYTES + Q::PART_BYTES);
    if (e != cudaSuccess) return e;
    CUtensorMap map{};
    if (a.w_vec) {
        const EncodeTiled encode = tensor_map_encoder();
        const cuuint64_t dims[2] = {cuuint64_t(a.k + 1) / 2, cuuint64_t(a.n)}, strides[1] = {cuuint64_t(a.w_row)};
        const cuuint32_t box[2] = {ROW, 16}, each[2] = {1, 1};
        a.w_vec = encode && encode(&map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<uint8_t *>(a.w), dims, strides, box, each,
                                   CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                                   CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
    }
    a.cols_rows = Q::COLS / PARTS < a.m ? Q::COLS / PARTS : a.m;
    const int passes = (a.m + a.cols_rows - 1) / a.cols_rows, tiles = (a.n + 15) / 16;
    const int step_bytes = BLOCKS * 64 * (CT == 1 ? a.cols_rows * PARTS : Q::COLS), fit = Q::X_BYTES / step_bytes;
    const int most = sm_count() * (CT <= 2 ? 2 : 1);
    a.steps = (a.k + STEP - 1) / STEP;
    // split k over a cluster's blocks until each one's share of x fits, or
    // (few tiles) the card is full and each warp has one step
    a.ks = 1;
    while (a.ks < 8 && a.steps > a.ks && (a.steps > fit * a.ks || (a.steps >= 2 * a.ks && tiles * a.ks * 2 <= most))) a.ks *= 2;
    a.share_steps = (a.steps + a.ks - 1) / a.ks;
    a.wk = 1;
    while (a.wk < WARPS && a.wk * 2 <= a.share_steps && a.wk * 2 <= fit) a.wk *= 2;
    // chunks of whole turns where even a share of x is too much
    a.chunk_steps = fit >= a.share_steps ? a.share_steps : fit / a.wk * a.wk;
    const int wr = WARPS / a.wk, lists = (tiles + wr - 1) / wr;
    a.keep = Q::PART_BYTES / (wr * 16 * a.cols_rows * 4);
    int teams = most / a.ks;
    teams = lists < teams ? lists : teams;
    cudaLaunchConfig_t c{};
    c.gridDim = dim3(unsigned(teams * a.ks), unsigned(passes));
    c.blockDim = dim3(THREADS);
    c.dynamicSmemBytes = Q::FIXED + a.chunk_steps * step_bytes + (a.ks > 1 ? Q::PART_BYTES : 0);
    c.stream = stream;
    cudaLaunchAttribute at{};
    at.id = cudaLaunchAttributeClusterDimension;
    at.val.clusterDim.x = unsigned(a.ks);
    at.val.clusterDim.y = at.val.clusterDim.z = 1;
    c.attrs = &at;
    c.numAttrs = a.ks > 1 ? 1 : 0;
    return cudaLaunchKernelEx(&c, q4_kernel<XT, CT, BPG, ZEROS>, a, map);
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
    a.w_vec = aligned(w, 16) && a.w_row % 16 == 0;
    a.x_vec = uint64_t(a.x_row) * xs % (xs == 1 ? 8 : 16) == 0 && aligned(x, xs == 1 ? 8 : 16);
    const auto str = static_cast<cudaStream_t>(stream);
    const cudaError_t e = s->x_type == PPOCR_F32    ? start_x<float>(a, str)
                          : s->x_type == PPOCR_F16  ? start_x<__half>(a, str)
                          : s->x_type == PPOCR_BF16 ? start_x<__nv_bfloat16>(a, str)
                                                    : start_x<e4m3>(a, str);
    return e == cudaSuccess ? int(PPOCR_OK) : refuse(PPOCR_E_DEVICE, me, cudaGetErrorString(e));
}
