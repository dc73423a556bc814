// Window attention for few queries a lane (single steps over a cache): the
// keys are split, and joined in the same launch.
//
// Rows of a tile are the queries that read one key head (query i, head h of
// its group), up to 16. A cluster of up to eight blocks takes one tile; its
// 4 * blocks warps take the key tiles in turn, each with a ring of its own
// filled by cp.async and a softmax state of its own (m, l, o). A block's four
// states become one in its shared memory, with weights 2^(m_i - max m), and the
// cluster's meet through distributed shared memory: row r is joined by block
// r mod cluster. No workspace, nothing to clear.
// Bound by the keys' and values' bytes; a single lane by latency. 64 lanes of
// one query behind 300 to 12 000 keys, 32 heads over 8 of 128, window 4096, bf16:
// 155 us, 919 MB at 5.9 TB/s (0.9 of a plain copy's rate). One lane, 516 keys, 16
// heads over 4 of 64: 6.4 us, of which an empty launch is 2.2.
#include "attn.cuh"

namespace ppocr {

namespace {

constexpr int WARPS = 4, THREADS = WARPS * 32, STAGES = 3, MOST_BLOCKS = 8, SORT_LANES = 256;

template <class T, int DP>
struct SplitTile {
    static constexpr int BK = sizeof(T) == 4 ? 16 : 32;  // keys a warp takes at a time
    static constexpr int STRIDE = TileOf<T, DP>::STRIDE;
    static constexpr int Q_BYTES = 16 * STRIDE * int(sizeof(T)), K_BYTES = BK * STRIDE * int(sizeof(T));
    static constexpr int RING = STAGES * 2 * K_BYTES;  // one warp's
    // a warp's joined state reuses its ring: o[16][DP], m[16], l[16]
    static_assert(RING >= (16 * DP + 32) * 4, "the state fits the ring");
    static constexpr int JOIN = (16 * DP + 32) * 4;  // the block's joined state
    static constexpr int SHARED = Q_BYTES + WARPS * RING + JOIN;
};

__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ uint32_t cluster_size() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t peer_addr(uint32_t addr, uint32_t rank) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
    return r;
}
__device__ __forceinline__ float peer_load(uint32_t addr) {
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ float lds(uint32_t addr) {
    float v;
    asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ float4 lds4(uint32_t addr) {
    float4 v;
    asm volatile("ld.shared.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ void sts2(uint32_t addr, float x, float y) {
    asm volatile("st.shared.v2.f32 [%0], {%1,%2};" ::"r"(addr), "f"(x), "f"(y) : "memory");
}
__device__ __forceinline__ void sts(uint32_t addr, float v) {
    asm volatile("st.shared.f32 [%0], %1;" ::"r"(addr), "f"(v) : "memory");
}

template <class T, int DP>
__global__ void __launch_bounds__(THREADS) attn_split_kernel(const __grid_constant__ AttnArgs a) {
    using R = SplitTile<T, DP>;
    constexpr int BK = R::BK, STRIDE = R::STRIDE;
    extern __shared__ __align__(16) unsigned char smem[];
    const int tid = threadIdx.x, warp = tid / 32, lane = tid & 31;
    const uint32_t qs = shared_u32(smem), rings = qs + R::Q_BYTES, ring = rings + warp * R::RING, joined = rings + WARPS * R::RING;
    const int blocks = int(cluster_size()), rank = int(cluster_rank()), workers = blocks * WARPS;
    // more tiles than blocks that run at once: the lanes with most keys first, so
    // that the last to start are short (64 lanes of 300 to 12 000 keys in a window
    // of 4096: 197 us in the lanes' order, 180 us so)
    __shared__ int keys[SORT_LANES], pick;
    int mine_z = blockIdx.z;
    if (a.sort) {
        for (int b = tid; b < a.lanes; b += THREADS) {
            const Lane l = read_lane(a, b);
            keys[b] = a.left < 0 ? l.nk : int(min(int64_t(l.nk), int64_t(a.left) + l.nq + a.sinks));
        }
        __syncthreads();
        for (int b = tid; b < a.lanes; b += THREADS) {
            const int k = keys[b];
            int rank = 0;
            for (int x = 0; x < a.lanes; x++) rank += keys[x] > k || (keys[x] == k && x < b);
            if (rank == int(blockIdx.z)) pick = b;
        }
        __syncthreads();
        mine_z = pick;
    }
    const Lane ln = read_lane(a, mine_z);
    const int kvh = blockIdx.y;
    const T *k = static_cast<const T *>(a.k) + ln.k0 * a.k_row + kvh * a.k_head;
    const T *v = static_cast<const T *>(a.v) + ln.k0 * a.v_row + kvh * a.v_head;
    const int64_t total = int64_t(ln.nq) * a.share;

    for (int64_t base = int64_t(blockIdx.x) / blocks * 16; base < total; base += int64_t(gridDim.x) / blocks * 16) {
        const int rows = int(total - base < 16 ? total - base : 16);
        const int shift = ln.nk - ln.nq;
        const int p0 = int(base / a.share) + shift, p1 = int((base + rows - 1) / a.share) + shift;
        const int pr[2] = {int((base + (lane >> 2)) / a.share) + shift, int((base + (lane >> 2) + 8) / a.share) + shift};
        KeyTiles kt;
        kt.plan<BK>(a, p0, p1, ln.nk);
        const auto fetch = [&](int it, int slot) {
            if (it < kt.n) {
                const int j = kt.first<BK>(it), n = min(BK, kt.end(it) - j);
                const uint32_t to = ring + uint32_t(slot * 2 * R::K_BYTES);
                load_rows<T, BK, DP, STRIDE, 32>(to, k + j * a.k_row, a.k_row, n, a.d, a.k_bytes, lane);
                load_rows<T, BK, DP, STRIDE, 32>(to + R::K_BYTES, v + j * a.v_row, a.v_row, n, a.d, a.v_bytes, lane);
            }
            copy_commit();
        };
        for (int r = warp; r < 16; r += WARPS) {
            const int64_t i = (base + r) / a.share, h = kvh * a.share + (base + r) % a.share;
            const T *src = static_cast<const T *>(a.q) + (r < rows ? (ln.q0 + i) * a.q_row + h * a.q_head : 0);
            load_rows<T, 1, DP, STRIDE, 32>(qs + uint32_t(r * STRIDE * int(sizeof(T))), src, 0, r < rows ? 1 : 0, a.d, a.q_bytes,
                                            lane);
        }
        copy_commit();
        const int first = rank * WARPS + warp;
#pragma unroll
        for (int s = 0; s < STAGES - 1; s++) fetch(first + s * workers, s);
        copy_wait<STAGES - 1>();
        __syncthreads();  // every warp's rows of q are there

        WarpAttn<T, DP> w;
        w.clear();
        int slot = 0;
        for (int it = first; it < kt.n; it += workers) {
            copy_wait<STAGES - 2>();
            __syncwarp();
            fetch(it + (STAGES - 1) * workers, slot == 0 ? STAGES - 1 : slot - 1);
            const uint32_t ks = ring + uint32_t(slot * 2 * R::K_BYTES), vs = ks + R::K_BYTES;
            const int j0 = kt.first<BK>(it), jend = kt.end(it);
            float s[BK / 8][4];
            w.template scores<BK / 8>(s, qs, ks, lane);
            const bool whole = j0 + BK <= jend && (a.right < 0 || j0 + BK - 1 <= p0 + a.right) &&
                               (a.left < 0 || j0 >= p1 - a.left || j0 + BK <= a.sinks);
            if (!whole) {
#pragma unroll
                for (int n = 0; n < BK / 8; n++)
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const int j = j0 + n * 8 + (lane & 3) * 2 + (e & 1);
                        if (j >= jend || !sees(a, pr[e >> 1], j)) s[n][e] = -INFINITY;
                    }
            }
            w.template soften<BK / 8>(s, a.scale_log2);
            w.template gather<BK / 8>(s, vs, lane);
            slot = slot == STAGES - 1 ? 0 : slot + 1;
        }
        copy_wait<0>();
        __syncwarp();  // the ring is free: this warp's state goes there
#pragma unroll
        for (int r = 0; r < 2; r++) {
            w.l[r] += __shfl_xor_sync(0xffffffffu, w.l[r], 1);
            w.l[r] += __shfl_xor_sync(0xffffffffu, w.l[r], 2);
            const int row = (lane >> 2) + 8 * r;
            if (row >= rows) continue;
            if ((lane & 3) == 0) {
                sts(ring + uint32_t((16 * DP + row) * 4), w.m[r]);
                sts(ring + uint32_t((16 * DP + 16 + row) * 4), w.l[r]);
            }
#pragma unroll
            for (int n = 0; n < DP / 8; n++)
                sts2(ring + uint32_t((row * DP + n * 8 + (lane & 3) * 2) * 4), w.o[n][2 * r], w.o[n][2 * r + 1]);
        }
        __syncthreads();
        // the block's four states as one, a quarter of a warp's lanes' values
        // (4 columns) a thread
        constexpr int Q4 = DP / 4;
        for (int e = tid; e < rows * Q4; e += THREADS) {
            const int r = e / Q4, c = e % Q4 * 4;
            float m[WARPS], top = -INFINITY, sum = 0.0f;
            float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
            for (int x = 0; x < WARPS; x++) {
                m[x] = lds(rings + uint32_t(x * R::RING + (16 * DP + r) * 4));
                top = fmaxf(top, m[x]);
            }
#pragma unroll
            for (int x = 0; x < WARPS; x++) {
                const float f = exp2_fast(m[x] - (top == -INFINITY ? 0.0f : top));
                const float4 o = lds4(rings + uint32_t(x * R::RING + (r * DP + c) * 4));
                sum = fmaf(f, lds(rings + uint32_t(x * R::RING + (16 * DP + 16 + r) * 4)), sum);
                acc = make_float4(fmaf(f, o.x, acc.x), fmaf(f, o.y, acc.y), fmaf(f, o.z, acc.z), fmaf(f, o.w, acc.w));
            }
            sts2(joined + uint32_t((r * DP + c) * 4), acc.x, acc.y);
            sts2(joined + uint32_t((r * DP + c + 2) * 4), acc.z, acc.w);
            if (c == 0) {
                sts(joined + uint32_t((16 * DP + r) * 4), top);
                sts(joined + uint32_t((16 * DP + 16 + r) * 4), sum);
            }
        }
        if (blocks > 1)
            cluster_sync();
        else
            __syncthreads();

        // then the cluster's: row r by block r mod blocks, a warp a row
        for (int r = rank + warp * blocks; r < rows; r += workers) {
            float m[MOST_BLOCKS], top = -INFINITY, sum = 0.0f;
            uint32_t from[MOST_BLOCKS];
#pragma unroll
            for (int x = 0; x < MOST_BLOCKS; x++) {
                from[x] = x < blocks ? peer_addr(joined, uint32_t(x)) : 0;
                m[x] = x < blocks ? peer_load(from[x] + uint32_t((16 * DP + r) * 4)) : -INFINITY;
            }
            float part[MOST_BLOCKS];
#pragma unroll
            for (int x = 0; x < MOST_BLOCKS; x++) {
                part[x] = x < blocks ? peer_load(from[x] + uint32_t((16 * DP + 16 + r) * 4)) : 0.0f;
                top = fmaxf(top, m[x]);
            }
#pragma unroll
            for (int x = 0; x < MOST_BLOCKS; x++) {
                m[x] = exp2_fast(m[x] - (top == -INFINITY ? 0.0f : top));
                sum = fmaf(m[x], part[x], sum);
            }
            constexpr int E = (DP + 31) / 32;
            float acc[E] = {};
#pragma unroll
            for (int x = 0; x < MOST_BLOCKS; x++)
#pragma unroll
                for (int e = 0; e < E; e++)
                    if (x < blocks && lane + 32 * e < DP)
                        acc[e] = fmaf(m[x], peer_load(from[x] + uint32_t((r * DP + lane + 32 * e) * 4)), acc[e]);
            const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
            const int i = int((base + r) / a.share), h = kvh * a.share + int((base + r) % a.share);
            bool bad = sum == 0.0f;  // it sees no key, or scores that overflowed
#pragma unroll
            for (int e = 0; e < E; e++) {
                acc[e] *= inv;
                bad |= !(fabsf(acc[e]) < INFINITY);
            }
            if (__any_sync(0xffffffffu, bad) && !no_numbers<T>(a, sum)) {
                row_alone<T>(a, ln, i, h);
            } else {
                T *out = static_cast<T *>(a.out) + (ln.q0 + i) * a.out_row + h * a.out_head;
#pragma unroll
                for (int e = 0; e < E; e++)
                    if (lane + 32 * e < a.d) out[lane + 32 * e] = from_f32<T>(acc[e]);
            }
        }
        if (blocks > 1)
            cluster_sync();  // no block overwrites or leaves what another still reads
        else
            __syncthreads();
    }
}

template <class T, int DP>
cudaError_t start_split(AttnArgs a, uint32_t max_q, uint32_t max_keys, cudaStream_t stream) {
    using R = SplitTile<T, DP>;
    cudaError_t e = raise_shared<attn_split_kernel<T, DP>>(R::SHARED);
    if (e != cudaSuccess) return e;
    const uint64_t rows = uint64_t(max_q) * a.share, tiles = rows ? (rows + 15) / 16 : 1;
    const uint64_t alone = tiles * a.lanes * a.kv_heads;
    // blocks a tile: while all clusters run at once and every warp has a key tile
    // (4 lanes of one query and 8 key heads of 64, window 1024: 9.2 us with 4, 22.5
    // with 8 blocks, which are more than the SMs)
    uint32_t blocks = 1;
    while (blocks < MOST_BLOCKS && alone * blocks * 2 <= uint64_t(sm_count()) && uint64_t(blocks) * WARPS * R::BK < max_keys) blocks *= 2;
    a.sort = alone * blocks > uint64_t(sm_count()) && a.lanes > 1 && a.lanes <= SORT_LANES;
    cudaLaunchConfig_t c{};
    c.gridDim = dim3(unsigned(tiles * blocks), unsigned(a.kv_heads), unsigned(a.lanes));
    c.blockDim = dim3(THREADS);
    c.dynamicSmemBytes = R::SHARED;
    c.stream = stream;
    cudaLaunchAttribute at{};
    at.id = cudaLaunchAttributeClusterDimension;
    at.val.clusterDim.x = blocks;
    at.val.clusterDim.y = at.val.clusterDim.z = 1;
    c.attrs = &at;
    c.numAttrs = 1;
    return cudaLaunchKernelEx(&c, attn_split_kernel<T, DP>, a);
}

template <class T>
cudaError_t start_split_d(const AttnArgs &a, uint32_t max_q, uint32_t max_keys, cudaStream_t stream) {
    if (a.d <= 16) return start_split<T, 16>(a, max_q, max_keys, stream);
    if (a.d <= 32) return start_split<T, 32>(a, max_q, max_keys, stream);
    if (a.d <= 64) return start_split<T, 64>(a, max_q, max_keys, stream);
    return start_split<T, 128>(a, max_q, max_keys, stream);
}

}  // namespace

cudaError_t launch_attn_split(const AttnArgs &a, int type, uint32_t max_q, uint32_t max_keys, cudaStream_t stream) {
    if (type == PPOCR_F32) return start_split_d<float>(a, max_q, max_keys, stream);
    if (type == PPOCR_F16) return start_split_d<__half>(a, max_q, max_keys, stream);
    return start_split_d<__nv_bfloat16>(a, max_q, max_keys, stream);
}

}  // namespace ppocr
