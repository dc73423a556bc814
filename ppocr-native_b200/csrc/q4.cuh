// The 4-bit product's shared part: its arguments, how a warp's weights and
// scales come in, and how partial sums are joined.
//
//     y[m][n] = sum_k x[m][k] (q[n][k] - z[n][k / G]) s[n][k / G] + b[n]
//
// A warp owns a slice of k (SL chunks of 128) for the whole launch: its part of
// x stays in registers as the matrix instruction's B operand, and the weights
// stream past, DEPTH tiles of 16 of their rows at a time (an item), from
// global memory straight into the A operand's registers: no staging, no
// barrier, no address arithmetic in between. An item's four chunks (4 KB a
// warp) are in flight while the one before is worked on. The matrix instruction sums over k in any
// order as long as both operands agree, so the k of lane t's slots are those
// of the bytes it loaded.
//
// The wk warps that share a tile leave their sums in shared memory; every
// few tiles a block adds them up in warp order, and where a cluster's blocks
// share k (ks of them) their sums meet through distributed shared memory in
// rank order: the same order every time.
#pragma once

#include <cuda_fp8.h>

#include <type_traits>

#include "block.cuh"

namespace ppocr {

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
    bool w_vec, x_vec;
    // the split, set by the launch
    int cols_rows;            // rows of x a pass takes
    int ks, wk;               // blocks of a cluster, and warps of a block, that share a tile
    int chunks, share, laps;  // chunks of 128 k in all and in a block's share; slices a warp takes of it
    bool direct;              // a warp has the whole sum of its tiles: no join
    int depth;                // tiles of an item
    int batch;                // lists of tiles between two joins
    int red_floats, stage_floats;  // of partial sums in shared memory before the cluster's, and before what else a warp keeps there
    uint32_t per_mul;         // ceil(2^31 / (group / (32 * BPG))): n * per_mul >> 31 divides n < 2^15 exactly
};

cudaError_t launch_q4_int(const Q4Args &a, int x_type, cudaStream_t stream);

namespace {

struct e4m3 {
    uint8_t bits;
};

// A scale's bits, and the number they are: the bits are taken ahead, the number
// where it is used, so that no load is waited for before it is needed.
__device__ __forceinline__ uint32_t scale_bits(const Q4Args &a, int64_t at) {
    if (a.scale_type == PPOCR_F32) return __ldg(static_cast<const uint32_t *>(a.scales) + at);
    return __ldg(static_cast<const unsigned short *>(a.scales) + at);
}
__device__ __forceinline__ float scale_of(const Q4Args &a, uint32_t bits) {
    if (a.scale_type == PPOCR_F16) return __half2float(__ushort_as_half((unsigned short)bits));
    return __uint_as_float(a.scale_type == PPOCR_BF16 ? bits << 16 : bits);
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

// Eight values of x as they lie in memory, of a type that enters in one part
// (zeros past k), and as pairs (0, 4), (1, 5), (2, 6), (3, 7) of the matrix
// instruction's type: two steps, so that a warp's loads all go out first.
template <class XT>
__device__ __forceinline__ uint4 take_x(const Q4Args &a, int row, int k, bool there) {
    uint4 v = make_uint4(0, 0, 0, 0);
    if (!there || k >= a.k) return v;
    const XT *p = static_cast<const XT *>(a.x) + row * a.x_row + k;
    if (a.x_vec && k + 8 <= a.k) {
        if constexpr (sizeof(XT) == 2) {
            v = __ldg(reinterpret_cast<const uint4 *>(p));
        } else {
            const uint2 u = __ldg(reinterpret_cast<const uint2 *>(p));
            v.x = u.x, v.y = u.y;
        }
        return v;
    }
    uint32_t u[4] = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < 8; i++)
        if (k + i < a.k) {
            if constexpr (sizeof(XT) == 2)
                u[i / 2] |= uint32_t(reinterpret_cast<const unsigned short *>(p)[i]) << (16 * (i & 1));
            else
                u[i / 4] |= uint32_t(reinterpret_cast<const unsigned char *>(p)[i]) << (8 * (i & 3));
        }
    return make_uint4(u[0], u[1], u[2], u[3]);
}
template <class XT>
__device__ __forceinline__ uint4 pairs_of(const uint4 &v) {
    uint32_t u[4] = {v.x, v.y, v.z, v.w};  // pairs (0, 1), (2, 3), (4, 5), (6, 7)
    if constexpr (sizeof(XT) == 1) {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(__nv_fp8x2_storage_t((i < 2 ? v.x : v.y) >> (16 * (i & 1))), __NV_E4M3);
            u[i] = *reinterpret_cast<const uint32_t *>(&h);
        }
    }
    return make_uint4(__byte_perm(u[0], u[2], 0x5410), __byte_perm(u[0], u[2], 0x7632), __byte_perm(u[1], u[3], 0x5410),
                      __byte_perm(u[1], u[3], 0x7632));
}

// This block has started: another's shared memory may be written once all blocks of the
// cluster have said so (cluster_wait).
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// 16 bytes of weights, each read once: past L1.
__device__ __forceinline__ uint4 load_once(const uint8_t *p) {
    uint4 v;
    asm volatile("ld.global.nc.L1::no_allocate.L2::256B.v4.u32 {%0,%1,%2,%3}, [%4];"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                 : "l"(p));
    return v;
}

// The first `valid` of 16 bytes, any alignment: 16 loads at once.
__device__ __noinline__ uint4 load_bytes(const uint8_t *p, int valid) {
    uint32_t b[16];
#pragma unroll
    for (int i = 0; i < 16; i++) b[i] = i < valid ? uint32_t(__ldg(p + i)) : 0;
    uint32_t v[4];
#pragma unroll
    for (int i = 0; i < 4; i++) v[i] = b[4 * i] | b[4 * i + 1] << 8 | b[4 * i + 2] << 16 | b[4 * i + 3] << 24;
    return make_uint4(v[0], v[1], v[2], v[3]);
}

// Which tiles and which share of k this warp has. An item is a.depth tiles,
// a list what a block takes at a time: wr items, one a group of wk warps.
struct Place {
    int warp, lane, g, t;             // g = lane / 4, t = lane % 4
    int rank, team, teams;            // block of the cluster; cluster; clusters
    int wr, k_warp, r_warp;           // items of a list; this warp's part of k and item
    int lists, c_lo, c_hi;            // this block's lists; its chunks
    __device__ __forceinline__ Place(const Q4Args &a) {
        warp = threadIdx.x / 32, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
        rank = a.ks > 1 ? int(blockIdx.x) % a.ks : 0, team = int(blockIdx.x) / a.ks, teams = int(gridDim.x) / a.ks;
        wr = int(blockDim.x) / 32 / a.wk, k_warp = warp % a.wk, r_warp = warp / a.wk;
        const int rows = wr * a.depth * 16, all = (a.n + rows - 1) / rows;
        lists = all > team ? (all - team + teams - 1) / teams : 0;
        c_lo = rank * a.share, c_hi = min(a.chunks, c_lo + a.share);
    }
    // the first row of item `r` of this block's list `list`
    __device__ __forceinline__ int row(const Q4Args &a, int list, int r) const {
        return ((team + list * teams) * wr + r) * a.depth * 16;
    }
};

// A warp's stream of weights and scales: an item in registers. The sequence
// is batches of lists, in each the laps over k, in each the batch's lists.
template <int SL, int DEPTH, int BPG, bool ZEROS>
struct Stream {
    static constexpr int NG = SL * 4 / BPG;         // groups a slice
    static constexpr int NS = NG < 2 ? 1 : NG / 2;  // scales a lane holds of a tile: row lane % 16
    uint4 w[DEPTH][SL][2];
    uint32_t s[DEPTH][NS], z[DEPTH][ZEROS ? NS : 1];  // their bits
    float b[DEPTH][2];                                // biases of rows g and g + 8 (one warp a tile)
    // the cursor: the item to be loaded next
    int b0 = 0, lap = 0, i = 0;
    const uint8_t *p, *p8;     // rows g and g + 8 of its first tile at this lane's first byte
    int n0, rows, left;        // its first row; rows and bytes of k left from there on
    bool full;                 // all there, in whole vectors: the loads need no checks
    int64_t sp;                // where this lane's row of scales begins
    int group0;                // and its group

    __device__ __forceinline__ void aim(const Q4Args &a, const Place &at) {
        const int list = b0 + i, first = at.c_lo + (lap * a.wk + at.k_warp) * SL;
        const int byte = first * 64 + at.t * 16;
        n0 = at.row(a, list, at.r_warp);
        rows = list < at.lists && first < at.c_hi ? a.n - n0 : 0;
        left = (a.k + 1) / 2 - byte;
        full = a.w_vec && rows >= a.depth * 16 && (first + SL) * 64 <= (a.k + 1) / 2;
        p = a.w + int64_t(n0 + at.g) * a.w_row + byte;
        p8 = p + 8 * a.w_row;
        group0 = first * (4 / BPG) + (at.lane >> 4);
        sp = int64_t(n0 + (at.lane & 15)) * a.groups;
    }
    __device__ __forceinline__ uint4 bytes(const Q4Args &a, const uint8_t *from, int rows_left, int c) const {
        const int n = rows_left > 0 ? left - c * 64 : 0;
        // past its k a row may be read as far as its stride goes (x is zero
        // there), the matrix's last row not
        if (a.w_vec && (n >= 16 || (n > 0 && rows_left > 1 && a.w_row - (a.k + 1) / 2 + n >= 16))) return load_once(from);
        return n > 0 ? load_bytes(from, n < 16 ? n : 16) : make_uint4(0, 0, 0, 0);
    }
    __device__ __forceinline__ void chunk(const Q4Args &a, const Place &at, int d, int c) {
        const int64_t down = int64_t(d) * 16 * a.w_row;
        if (full) {
            w[d][c][0] = load_once(p + down + c * 64);
            w[d][c][1] = load_once(p8 + down + c * 64);
        } else {
            w[d][c][0] = bytes(a, p + down + c * 64, rows - d * 16 - at.g, c);
            w[d][c][1] = bytes(a, p8 + down + c * 64, rows - d * 16 - at.g - 8, c);
        }
    }
    __device__ __forceinline__ void scales(const Q4Args &a, const Place &at, int d) {
        const bool there = rows > d * 16 + (at.lane & 15);
#pragma unroll
        for (int x = 0; x < NS; x++) {
            const int group = int((uint64_t(uint32_t(group0 + 2 * x)) * a.per_mul) >> 31);
            s[d][x] = 0;
            if constexpr (ZEROS) z[d][x] = 8;
            if (there && (NG > 1 || at.lane < 16) && group < a.groups) {
                const int64_t q = sp + int64_t(d) * 16 * a.groups + group;
                s[d][x] = scale_bits(a, q);
                if constexpr (ZEROS) z[d][x] = __ldg(a.zeros + q);
            }
        }
    }
    __device__ __forceinline__ void biases(const Q4Args &a, const Place &at, int d) {
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const int r = d * 16 + at.g + 8 * h;
            b[d][h] = a.direct && a.bias && rows > r ? __ldg(a.bias + n0 + r) : 0.0f;
        }
    }
    __device__ __forceinline__ void next(const Q4Args &a, const Place &at) {
        if (++i == min(a.batch, at.lists - b0)) {
            i = 0;
            if (++lap == a.laps) lap = 0, b0 += a.batch;
        }
    }
    __device__ __forceinline__ void begin(const Q4Args &a, const Place &at) {
        aim(a, at);
#pragma unroll
        for (int d = 0; d < DEPTH; d++) {
            if (d >= a.depth) break;
#pragma unroll
            for (int c = 0; c < SL; c++) chunk(a, at, d, c);
            scales(a, at, d);
            biases(a, at, d);
        }
        next(a, at);
    }
    // group j's scale (zero point) of tile row r, in every lane
    __device__ __forceinline__ float scale(const Q4Args &a, int d, int j, int r) const {
        return scale_of(a, __shfl_sync(0xffffffffu, s[d][j >> 1], r | ((j & 1) << 4)));
    }
    __device__ __forceinline__ uint32_t zero(int d, int j, int r) const {
        if constexpr (ZEROS) return __shfl_sync(0xffffffffu, z[d][j >> 1], r | ((j & 1) << 4)) & 15u;
        return 8;
    }
};

// A row's four words in lane t (k t * 32 + 8 i of a chunk, i = 0..3) to the
// words at k i * 32 + 8 t: a 4 x 4 transposition among the lanes of a row,
// for groups smaller than a chunk (the words of one instruction then lie in
// one group).
__device__ __forceinline__ void transpose(uint4 &u, int t) {
    uint32_t a0 = u.x, a1 = u.y, a2 = u.z, a3 = u.w;
    const bool odd = t & 1, high = t & 2;
    uint32_t p = __shfl_xor_sync(0xffffffffu, odd ? a0 : a1, 1), q = __shfl_xor_sync(0xffffffffu, odd ? a2 : a3, 1);
    if (odd)
        a0 = p, a2 = q;
    else
        a1 = p, a3 = q;
    p = __shfl_xor_sync(0xffffffffu, high ? a0 : a2, 2), q = __shfl_xor_sync(0xffffffffu, high ? a1 : a3, 2);
    if (high)
        a0 = p, a1 = q;
    else
        a2 = p, a3 = q;
    u = make_uint4(a0, a1, a2, a3);
}

// One output value in its type.
__device__ __forceinline__ void put_y(const Q4Args &a, int m, int n, float y) {
    const int64_t at = int64_t(m) * a.y_row + n;
    if (a.y_type == PPOCR_F32)
        static_cast<float *>(a.y)[at] = y;
    else if (a.y_type == PPOCR_F16)
        static_cast<__half *>(a.y)[at] = __float2half_rn(y);
    else
        static_cast<__nv_bfloat16 *>(a.y)[at] = __float2bfloat16_rn(y);
}

__device__ __forceinline__ void peer_store(float *p, uint32_t rank, float v) {
    uint32_t at;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(shared_u32(p)), "r"(rank));
    asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(at), "f"(v) : "memory");
}

// The join of `count` lists from `list0` on, in pieces of 32 values (a tile's 16
// rows for two rows of x): value(list of the batch, tile of the list, row of
// x, row of the tile) adds up the block's warps; in a cluster piece p goes to
// block p mod ks, which adds the blocks' in rank order; finish(m, n, y, bias,
// scale) takes the sum. The kernel has called cluster_arrive() before its first load.
template <class V, class F>
__device__ __forceinline__ void join(const Q4Args &a, const Place &at, int m0, int rows, int list0, int count, float *part,
                                     const V &value, const F &finish) {
    __syncthreads();
    const int each = at.wr * a.depth, pieces = (rows + 1) / 2, all = count * each * pieces, warps = int(blockDim.x) / 32;
    const int r = at.lane & 15, mine = (all + a.ks - 1) / a.ks;
    const auto end = [&](int p, float y) {
        const int tile = p / pieces, m = (p - tile * pieces) * 2 + (at.lane >> 4);
        const int n = at.row(a, list0 + tile / each, 0) + tile % each * 16 + r;
        if (m >= rows || n >= a.n) return;
        finish(m, n, y, a.bias ? __ldg(a.bias + n) : 0.0f, a.x_groups == 1 ? __ldg(a.x_scales + m0 + m) : 1.0f);
    };
    if (a.ks > 1 && list0 == 0) cluster_wait();  // every block has started: its shared memory is there
    for (int p = at.warp; p < all; p += warps) {
        const int tile = p / pieces, m = (p - tile * pieces) * 2 + (at.lane >> 4);
        const float y = m < rows ? value(tile / each, tile % each, m, r) : 0.0f;
        if (a.ks > 1)
            peer_store(part + (at.rank * mine + p / a.ks) * 32 + at.lane, uint32_t(p % a.ks), y);
        else
            end(p, y);
    }
    if (a.ks == 1) {
        __syncthreads();
        return;
    }
    cluster_sync();
    for (int q = at.warp; q * a.ks + at.rank < all; q += warps) {
        float y = 0.0f;
        for (int x = 0; x < a.ks; x++) y += part[(x * mine + q) * 32 + at.lane];
        end(q * a.ks + at.rank, y);
    }
    if (list0 + count < at.lists) cluster_sync();  // the next batch's pieces come to the same place
}

// Splits the work and launches: blocks of up to `warps` warps, items of up to
// `depth` tiles by `sl` chunks, `cols` partial sums a tile row and warp,
// `stage` bytes of shared memory a warp besides, `direct` where a warp alone can
// write its tiles' results, `laps` where laps cost little.
cudaError_t launch_q4(const void *kernel, Q4Args a, int warps, int sl, int depth, int bpg, int cols, int stage, int shared_most,
                      bool direct, bool laps, cudaStream_t stream) {
    const int passes = (a.m + a.cols_rows - 1) / a.cols_rows, sms = sm_count();
    a.chunks = (a.k + 127) / 128;
    const uint32_t per = uint32_t(a.group) / (32 * bpg);
    a.per_mul = ((1u << 31) + per - 1) / per;
    // k over one block's warps, then over a cluster's blocks, then in laps; where a
    // slice of x comes in as it is (`laps`), in laps before a cluster's join holds up
    // more tiles than there are SMs (16 rows f16 or bf16, k 16384: n 256 in clusters
    // 11.8 us, in laps 22.5; n 2048 28.4 and 22.8; 32 rows, k 8192, n 4096 65 and 38;
    // f32, whose slices are taken apart each lap, 61 and 240, 129 and 258, 181 and 295)
    const int slices = (a.chunks + sl - 1) / sl;
    a.wk = 1;
    while (a.wk < warps && a.wk < slices) a.wk *= 2;
    a.ks = 1;
    while (a.ks < 8 && a.ks * a.wk < slices && (!laps || int64_t((a.n + 15) / 16) * passes * a.ks * 2 <= sms)) a.ks *= 2;
    a.share = (slices + a.ks - 1) / a.ks * sl;
    a.laps = (a.share + a.wk * sl - 1) / (a.wk * sl);
    // fewer tiles an item, then fewer items a block, as long as every item still
    // has a warp, and every block an SM, at once (16 rows, 120 x 18 710: 4.9 us, 9.6
    // with items as they are, 5.6 with blocks as they are; 120 x 360: 4.5, 5.9, 5.7)
    const int64_t room = int64_t(sms) * (warps / a.wk) / (passes * a.ks);
    const auto items_of = [&](int d) { return (a.n + d * 16 - 1) / (d * 16); };
    while (depth > 1 && items_of(depth / 2) <= room) depth /= 2;
    a.depth = depth;
    const int items = items_of(depth);
    const auto blocks_of = [&](int w) { return int64_t((items + w / a.wk - 1) / (w / a.wk)) * passes * a.ks; };
    while (warps > a.wk && blocks_of(warps / 2) <= sms) warps /= 2;
    const int wr = warps / a.wk, lists = (items + wr - 1) / wr;
    int teams = sms / a.ks;
    teams = lists < teams ? lists : teams;
    const int list_floats = warps * depth * 16 * cols, part_floats = a.ks > 1 ? wr * depth * (a.cols_rows + 1) / 2 * 32 + a.ks * 32 : 0;
    const int fit = (shared_most - warps * stage) / 4 / (list_floats + part_floats), mine = (lists + teams - 1) / teams;
    a.batch = fit < mine ? fit : mine;
    a.red_floats = a.batch * list_floats;
    // whole sums leave at once (16 rows, 120 x 18 710: 4.9 us, through the join 10.8)
    a.direct = direct && a.wk == 1 && a.ks == 1 && a.laps == 1;
    a.stage_floats = a.batch * (list_floats + part_floats);
    cudaLaunchConfig_t c{};
    c.gridDim = dim3(unsigned(teams * a.ks), unsigned(passes));
    c.blockDim = dim3(unsigned(warps * 32));
    c.dynamicSmemBytes = size_t(a.stage_floats) * 4 + warps * stage;
    c.stream = stream;
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = unsigned(a.ks);
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    c.attrs = &attr;
    c.numAttrs = a.ks > 1 ? 1 : 0;
    void *args[1] = {&a};
    return cudaLaunchKernelExC(&c, kernel, args);
}

}  // namespace

}  // namespace ppocr
