// Window attention over whole lanes on the 5th-generation tensor cores (f16
// and bf16, rows and heads on 16-byte borders).
//
// A block takes 128 queries of one head (a thread a row) and walks the key
// tiles they see: the sinks, then up to 64 keys at a time from the window's
// first key on, the last tile in steps of 16. Per tile:
//     S = Q K^T      tcgen05.mma, Q and K in shared memory (TMA, 128-byte
//                    swizzle), S in tensor memory
//     softmax        four warps: a row's 64 scores in registers, P back into
//                    S's place in 16 bits
//     O += P V       tcgen05.mma, P from tensor memory, V as it lies in shared
//                    memory (its head dimension is the instruction's N)
// One warp issues the products, one the copies. S, K and V have two buffers, so
// that the next tile's scores are there when a tile's softmax ends; two
// blocks share an SM (256 columns of tensor memory and 96 KB of shared memory
// each) for the rest. Tiles of 128 keys leave no room for a second S beside
// an O of 128 columns, and were slower though a product of N = 64 costs 48
// cycles where half of one of N = 128 costs 32.
//
// O is rescaled only when a row's maximum has grown by more than 2^8 since
// the last time (the weights stay below 2^8, their sums in f32), which is rare
// after the first tile: a published way to leave most of a running softmax's
// corrections out. Bound by the latency of a tile's product, softmax and product one
// after another, of which two blocks an SM cover about half: 8192 queries, 16 heads of
// 128, window 1024, bf16: 89 to 96 us from card to card replayed, 101 called one by one,
// 64.7 GFLOP at 640 to 730 TFLOP/s (40 us at the library's matrix rate; tensor pipe
// 43% busy, exponentials 41%, issue 39%), where warp-level products
// (k_attn.cu) take 275. 12 lanes of 1 to 1500 queries, 8 heads of 40, window
// 257, f16: 35 us and 47. Up to head size 64: tiles of 32 keys and four blocks
// an SM (34 us, with tiles of 64 and two blocks 37 to 40).
#include <type_traits>

#include "attn.cuh"
#include "devmath.cuh"

namespace ppocr {

namespace {

constexpr int BQ = 128, SOFTMAX_WARPS = 4, MMA_WARP = SOFTMAX_WARPS, COPY_WARP = SOFTMAX_WARPS + 1, THREADS = SOFTMAX_WARPS * 32 + 64;
constexpr int BOX = 32;                    // rows a copy brings: 4 KB of one 64-column panel
constexpr int BOX_BYTES = BOX * 128;
constexpr unsigned long long DRAIN_NS = 200ull * 1000 * 1000;
constexpr float GROW = 8.0f;               // log2 of how far a maximum may grow before O is rescaled

struct Maps {
    CUtensorMap q, k, v;
};

__device__ __forceinline__ uint64_t desc(uint32_t addr, uint32_t lead, uint32_t stride) {
    // shared-memory matrix descriptor: start, leading and stride offsets in
    // 16-byte units, version 1, 128-byte swizzle (2)
    return uint64_t((addr >> 4) & 0x3FFF) | uint64_t((lead >> 4) & 0x3FFF) << 16 | uint64_t((stride >> 4) & 0x3FFF) << 32 |
           uint64_t(1) << 46 | uint64_t(2) << 61;
}

// kind::f16: D f32, A and B f16 (0) or bf16 (1), M = 128, N = n; B's major
// dimension: 0 k, 1 n.
template <class T>
__device__ __forceinline__ uint32_t idesc(int n, int b_major) {
    constexpr uint32_t F = std::is_same<T, __half>::value ? 0 : 1;
    return (1u << 4) | (F << 7) | (F << 10) | (uint32_t(b_major) << 16) | (uint32_t(n >> 3) << 17) | (uint32_t(BQ >> 4) << 24);
}

__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t id, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d), "l"(a), "l"(b), "r"(id), "r"(acc));
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t id, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}\n" ::"r"(d), "r"(a), "l"(b), "r"(id), "r"(acc));
}

// The products of one tile, their number known at compile time and nothing
// between them: 32 + N / 4 cycles each with both operands in shared memory (its
// bandwidth), N / 2 with one in tensor memory; a branch or a predicate a
// product cost 11 to 43 more.
template <int STEPS, int BK>
__device__ __forceinline__ void score_steps(uint32_t d, uint64_t q, uint64_t k, uint32_t id) {
#pragma unroll
    for (int kk = 0; kk < STEPS; kk++)  // the descriptors' addresses count 16 bytes: 16 columns are 2, a panel all its rows
        mma_ss(d, q + (kk >> 2) * (BQ * 128 / 16) + (kk & 3) * 2, k + (kk >> 2) * (BK * 128 / 16) + (kk & 3) * 2, id, kk > 0);
}
template <int BK>
__device__ __forceinline__ void score_product(int steps, uint32_t d, uint64_t q, uint64_t k, uint32_t id) {
    switch (steps) {
    case 1: return score_steps<1, BK>(d, q, k, id);
    case 2: return score_steps<2, BK>(d, q, k, id);
    case 3: return score_steps<3, BK>(d, q, k, id);
    case 4: return score_steps<4, BK>(d, q, k, id);
    case 5: return score_steps<5, BK>(d, q, k, id);
    case 6: return score_steps<6, BK>(d, q, k, id);
    case 7: return score_steps<7, BK>(d, q, k, id);
    default: return score_steps<8, BK>(d, q, k, id);
    }
}
template <int STEPS>
__device__ __forceinline__ void value_steps(uint32_t d, uint32_t p, uint64_t v, uint32_t id, uint32_t acc) {
#pragma unroll
    for (int kk = 0; kk < STEPS; kk++) mma_ts(d, p + kk * 8, v + kk * 128, id, kk > 0 ? 1 : acc);
}
__device__ __forceinline__ void value_product(int steps, uint32_t d, uint32_t p, uint64_t v, uint32_t id, uint32_t acc) {
    switch (steps) {
    case 1: return value_steps<1>(d, p, v, id, acc);
    case 2: return value_steps<2>(d, p, v, id, acc);
    case 3: return value_steps<3>(d, p, v, id, acc);
    default: return value_steps<4>(d, p, v, id, acc);
    }
}

__device__ __forceinline__ void commit(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}

__device__ __forceinline__ void tmem_load32(uint32_t addr, float *v) {
    uint32_t *r = reinterpret_cast<uint32_t *>(v);
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
          "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]),
          "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]),
          "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(addr));
}
__device__ __forceinline__ void tmem_load16(uint32_t addr, float *v) {
    uint32_t *r = reinterpret_cast<uint32_t *>(v);
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
          "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(addr));
}
__device__ __forceinline__ void tmem_store16(uint32_t addr, const uint32_t *r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(addr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
        "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}
__device__ __forceinline__ void tmem_wait_load() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_store() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// True in one lane of a whole warp.
__device__ __forceinline__ bool elect_one() {
    uint32_t e;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.b32 %0, 1, 0, p;\n\t}" : "=r"(e));
    return e != 0;
}

__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
__device__ __forceinline__ float2 fadd2(float2 a, float2 b) {
    float2 d;
    asm("{.reg .b64 ra, rb, rd;\n\tmov.b64 ra, {%2, %3};\n\tmov.b64 rb, {%4, %5};\n\tadd.rn.f32x2 rd, ra, rb;\n\t"
        "mov.b64 {%0, %1}, rd;}"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}
// The slow half of a wait; a lane that was told to give up says so to all.
__device__ __noinline__ bool wait_long(uint32_t bar, uint32_t parity, volatile int *give_up) {
    if (*give_up) return false;
    if (wait_copy(bar, parity)) return true;
    *give_up = 1;
    return false;
}

// Bits 0 to n - 1.
__device__ __forceinline__ uint32_t below(int n) { return n <= 0 ? 0u : n >= 32 ? ~0u : (1u << n) - 1; }

// The tiles of one query tile: the sinks below the window, then the window.
template <int BK>
struct Tiles {
    int sink_end, lo, hi, n_sink, n;
    __device__ __forceinline__ Tiles(const AttnArgs &a, int p0, int p1, int nk) {
        hi = max(0, a.right < 0 ? nk : min(nk, p1 + a.right + 1));
        lo = a.left < 0 ? 0 : min(max(0, p0 - a.left), hi);
        sink_end = min(a.sinks, lo);
        n_sink = (sink_end + BK - 1) / BK;
        n = n_sink + (hi - lo + BK - 1) / BK;
    }
    __device__ __forceinline__ int first(int it) const { return it < n_sink ? it * BK : lo + (it - n_sink) * BK; }
    __device__ __forceinline__ int count(int it) const {
        return it < n_sink ? min(BK, sink_end - it * BK) : min(BK, hi - lo - (it - n_sink) * BK);
    }
};

// The query tiles of a block that gave up behind the one at i0, the plain way (it
// has some where max_q was too small).
template <class T>
__device__ __noinline__ void rest_alone(const AttnArgs &a, int64_t i0) {
    const Lane ln = read_lane(a, blockIdx.z);
    while ((i0 += int64_t(gridDim.x) * BQ) < ln.nq)
        for (int r = threadIdx.x / 32; r < BQ && i0 + r < ln.nq; r += THREADS / 32) row_alone<T>(a, ln, int(i0) + r, blockIdx.y);
}

// BK keys a tile. Head sizes above 64: 64 keys, 256 columns of tensor memory (two
// S and P in their places, then 128 of O), two blocks an SM; up to 64: 32 keys,
// 128 columns (O has 64), four.
template <class T, int BK>
__global__ void __launch_bounds__(THREADS, BK == 64 ? 2 : 4) attn_tc_kernel(const __grid_constant__ AttnArgs a, const __grid_constant__ Maps maps) {
    constexpr int O_COL = 2 * BK, TMEM_COLS = BK == 64 ? 256 : 128;
    extern __shared__ __align__(1024) unsigned char smem[];
    // Q has come; then a pair each, used in turn: K and V have come, S is done, P
    // is there, O is done
    __shared__ uint64_t bars[11];
    __shared__ uint32_t tmem_s;
    __shared__ int give_up_s;
    // the warp's number and the tensor memory's address by a shuffle, which the
    // compiler knows to be the same in every lane: the products' operands then
    // stay in uniform registers (64 cycles a product of 128 x 128 x 16; 110 with
    // each operand moved there first)
    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid / 32, 0), lane = tid & 31;
    const int panels = (a.d + 63) / 64, dn = (a.d + 15) / 16 * 16;  // 64-column panels; head size in steps of 16
    const uint32_t tile_bytes = uint32_t(panels * (BK * 128));      // of one K or V buffer
    const uint32_t q_s = shared_u32(smem), k_s = q_s + panels * (BQ * 128), v_s = k_s + 2 * tile_bytes;
    const uint32_t q_bar = shared_u32(bars), k_bar = q_bar + 8, v_bar = q_bar + 24, s_bar = q_bar + 40, p_bar = q_bar + 56,
                   o_bar = q_bar + 72;
    volatile int *give_up = &give_up_s;
    // the lane first: most blocks of a ragged batch's grid have no queries
    if (tid == 32) {
        asm volatile("prefetch.tensormap [%0];" ::"l"(&maps.q) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&maps.k) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&maps.v) : "memory");
    }
    Lane ln = read_lane(a, blockIdx.z);
    ln.q0 = __shfl_sync(0xffffffffu, ln.q0, 0), ln.k0 = __shfl_sync(0xffffffffu, ln.k0, 0);
    ln.nq = __shfl_sync(0xffffffffu, ln.nq, 0), ln.nk = __shfl_sync(0xffffffffu, ln.nk, 0);
    if (int64_t(blockIdx.x) * BQ >= ln.nq) return;
    if (tid == 0) {
        for (int i = 0; i < 11; i++) bar_init(q_bar + 8 * i, i == 7 || i == 8 ? SOFTMAX_WARPS : 1);
        give_up_s = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == MMA_WARP) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(shared_u32(&tmem_s)), "r"(TMEM_COLS));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = __shfl_sync(0xffffffffu, tmem_s, 0);
    const bool one = elect_one();
    // a wait that ran out of time ends every role's; the rows are done again the plain way
    const auto wait = [&](uint32_t bar, uint32_t parity) {
        return try_wait(bar, parity) || wait_long(bar, parity, give_up);
    };

    const int h = blockIdx.y, kvh = h / a.share;
    // query tiles with keys, and key tiles, so far: tile x uses buffer x % 2 in its phase x / 2 % 2
    uint32_t turn = 0, done = 0;
    for (int64_t i0 = int64_t(blockIdx.x) * BQ; i0 < ln.nq; i0 += int64_t(gridDim.x) * BQ) {
        const int rows = int(ln.nq - i0 < BQ ? ln.nq - i0 : BQ);
        const int p0 = int(i0) + ln.nk - ln.nq;
        const Tiles<BK> tl(a, p0, p0 + rows - 1, ln.nk);
        const auto buf = [&](int it) { return (done + uint32_t(it)) & 1u; };
        const auto phase = [&](int it) { return (done + uint32_t(it)) >> 1 & 1u; };
        if (warp == COPY_WARP) {
            if (tl.n > 0) {
                const auto load = [&](const CUtensorMap *map, uint32_t to, uint32_t panel, int head, int64_t row, int n, uint32_t bar) {
                    const int boxes = (n + BOX - 1) / BOX;
                    if (!one) return;
                    arrive_expect(bar, uint32_t(boxes * panels * BOX_BYTES));
                    for (int p = 0; p < panels; p++)
                        for (int b = 0; b < boxes; b++)
                            tma_load_3d(to + p * panel + uint32_t(b * BOX_BYTES), map, p * 64, head, int(row) + b * BOX, bar);
                };
                const auto load_k = [&](int it) {
                    load(&maps.k, k_s + buf(it) * tile_bytes, BK * 128, kvh, ln.k0 + tl.first(it), tl.count(it), k_bar + buf(it) * 8);
                };
                const auto load_v = [&](int it) {
                    load(&maps.v, v_s + buf(it) * tile_bytes, BK * 128, kvh, ln.k0 + tl.first(it), tl.count(it), v_bar + buf(it) * 8);
                };
                load(&maps.q, q_s, BQ * 128, h, ln.q0 + i0, rows, q_bar);
                load_k(0);
                if (tl.n > 1) load_k(1);
                load_v(0);
                if (tl.n > 1) load_v(1);
                int k_end = min(tl.n, 2), v_end = k_end;
                for (int it = 2; it < tl.n; it++) {
                    if (!__all_sync(0xffffffffu, wait(s_bar + buf(it) * 8, phase(it - 2)))) break;  // K is read
                    load_k(it);
                    k_end = it + 1;
                    if (!__all_sync(0xffffffffu, wait(o_bar + buf(it) * 8, phase(it - 2)))) break;  // V is read
                    load_v(it);
                    v_end = it + 1;
                }
                if (v_end < tl.n) {  // given up: not before the copies in flight have landed
                    drain(q_bar, turn & 1, DRAIN_NS);
                    for (int it = max(0, k_end - 2); it < k_end; it++) drain(k_bar + buf(it) * 8, phase(it), DRAIN_NS);
                    for (int it = max(0, v_end - 2); it < v_end; it++) drain(v_bar + buf(it) * 8, phase(it), DRAIN_NS);
                }
            }
            __syncwarp();
        } else if (warp == MMA_WARP) {
            if (tl.n > 0) {
                const uint64_t q_desc = desc(q_s, 16, 1024), k_desc = desc(k_s, 16, 1024), v_desc = desc(v_s, BK * 128, 1024);
                const uint64_t next = tile_bytes / 16;  // the descriptors' addresses count 16 bytes
                const uint32_t id_o = idesc<T>(dn, 1);
                const int steps = dn / 16;
                // The tensor core runs one thread's products in order: S of tile it + 1 goes
                // ahead of tile it's second product, and takes the place of P two tiles
                // back behind the product that read it. No early way out of the loop: its
                // control stays the same in every lane, and after a wait that ran out no
                // product is issued.
                bool on = __all_sync(0xffffffffu, wait(q_bar, turn & 1));
                const auto scores = [&](int it) {
                    on &= __all_sync(0xffffffffu, wait(k_bar + buf(it) * 8, phase(it)));
                    fence_after();
                    const uint32_t id_s = idesc<T>((tl.count(it) + 15) / 16 * 16, 0);
                    if (one && on) {
                        score_product<BK>(steps, tmem + buf(it) * BK, q_desc, k_desc + buf(it) * next, id_s);
                        commit(s_bar + buf(it) * 8);
                    }
                };
                scores(0);
                int s_end = on, o_end = 0;  // tiles whose products were issued
                for (int it = 0; it < tl.n; it++) {
                    if (it + 1 < tl.n) {
                        scores(it + 1);
                        s_end += on;
                    }
                    const int n = (tl.count(it) + 15) / 16;
                    on &= __all_sync(0xffffffffu, wait(v_bar + buf(it) * 8, phase(it)) && wait(p_bar + buf(it) * 8, phase(it)));
                    fence_after();
                    if (one && on) {
                        value_product(n, tmem + O_COL, tmem + buf(it) * BK, v_desc + buf(it) * next, id_o, it > 0);
                        commit(o_bar + buf(it) * 8);
                    }
                    o_end += on;
                }
                if (!on) {  // given up: not before the products in flight are done
                    if (s_end > 0) drain(s_bar + buf(s_end - 1) * 8, phase(s_end - 1), DRAIN_NS);
                    if (o_end > 0) drain(o_bar + buf(o_end - 1) * 8, phase(o_end - 1), DRAIN_NS);
                }
            }
            __syncwarp();
        } else {
            const int row = warp * 32 + lane, p = p0 + row;
            const uint32_t mine = tmem + (uint32_t(warp * 32) << 16), o_at = mine + O_COL;
            float m = -INFINITY, l = 0.0f;
            bool ok = true;  // a wait that ran out spoils the rows, not the warp's common way
            // rows of V past the lane's keys, up to the product's step of 16:
            // whatever lies there, zero
            const auto clear_v = [&](int it, int n) {
                if ((n & 15) == 0) return;
                ok &= wait(v_bar + buf(it) * 8, phase(it));
                unsigned char *v = smem + (v_s - q_s) + buf(it) * tile_bytes;
                const int gap = 16 - (n & 15);
                for (int e = row; e < gap * panels * 8; e += SOFTMAX_WARPS * 32) {
                    const int r = n + e / (panels * 8), c = e % (panels * 8);
                    *reinterpret_cast<uint4 *>(v + (c >> 3) * (BK * 128) + r * 128 + (c & 7) * 16) = make_uint4(0, 0, 0, 0);
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            };
            const auto arrive_p = [&](int it) {
                tmem_wait_store();
                fence_before();
                __syncwarp();
                if (lane == 0) arrive(p_bar + buf(it) * 8);
            };
            // the tiles that every row of this warp sees whole, and those behind the
            // sinks that any sees at all
            const int pw = p0 + warp * 32;
            const int whole_from = tl.n_sink + (a.left < 0 ? 0 : max(0, pw + 31 - a.left - tl.lo + BK - 1) / BK);
            const int whole_to = tl.n_sink + (min(tl.hi, a.right < 0 ? tl.hi : pw + a.right + 1) - tl.lo) / BK;
            const int some_from = tl.n_sink + (a.left < 0 || tl.lo < a.sinks ? 0 : max(0, pw - a.left - tl.lo) / BK);
            const int some_to = tl.n_sink + (a.right < 0 ? tl.n : max(0, pw + 32 + a.right - tl.lo + BK - 1) / BK);
            for (int it = 0; it < tl.n; it++) {
                const uint32_t s_at = mine + buf(it) * BK;
                const int j0 = tl.first(it), n = tl.count(it);
                ok &= wait(s_bar + buf(it) * 8, phase(it));
                fence_after();
                if (it >= tl.n_sink && (it < some_from || it >= some_to)) {  // no weight here
                    const uint32_t w[16] = {};
#pragma unroll
                    for (int c = 0; c < BK / 32; c++) tmem_store16(s_at + c * 16, w);
                    clear_v(it, n);
                    arrive_p(it);
                    continue;
                }
                float s[BK];
                tmem_load32(s_at, s);
                if (n > 32) tmem_load32(s_at + 32, s + 32);
                tmem_wait_load();
                float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
                if (it < whole_from || it >= whole_to) {
#pragma unroll
                    for (int c = 0; c < BK / 32; c++) {
                        // this row's keys of these 32: a run, and below the sinks' end all that
                        // the right side leaves
                        const int j = j0 + c * 32, left = n - c * 32;
                        const uint32_t seen = below(a.right < 0 ? left : min(left, p + a.right + 1 - j)) &
                                              (a.left < 0 ? ~0u : ~below(p - a.left - j) | below(a.sinks - j));
                        if (__all_sync(0xffffffffu, seen == ~0u)) continue;
#pragma unroll
                        for (int x = 0; x < 32; x++)
                            if (!(seen >> x & 1u)) s[c * 32 + x] = -INFINITY;
                    }
                }
#pragma unroll
                for (int c = 0; c < BK / 32; c++)
                    if (c * 32 < n) {
#pragma unroll
                        for (int x = 0; x < 32; x += 2) top[x / 2 & 3] = max3(top[x / 2 & 3], s[c * 32 + x], s[c * 32 + x + 1]);
                    }
                const float now = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])) * a.scale_log2;
                const bool grown = now > m + GROW;
                if (__any_sync(0xffffffffu, grown)) {
                    // O's row is zero while no key was seen: nothing to rescale then
                    float keep = 1.0f;
                    if (grown) {
                        keep = m == -INFINITY ? 1.0f : exp2_fast(m - now);
                        m = now;
                    }
                    if (__any_sync(0xffffffffu, keep != 1.0f)) {
                        ok &= wait(o_bar + buf(it + 1) * 8, phase(it - 1));  // the product before is in O
                        fence_after();
                        __syncwarp();
                        l *= keep;
                        for (int c = 0; c < dn; c += 16) {
                            float o[16];
                            tmem_load16(o_at + c, o);
                            tmem_wait_load();
#pragma unroll
                            for (int x = 0; x < 16; x++) o[x] *= keep;
                            tmem_store16(o_at + c, reinterpret_cast<const uint32_t *>(o));
                        }
                    }
                }
                clear_v(it, n);
                const float base = m == -INFINITY ? 0.0f : -m;
                const float2 scale2 = make_float2(a.scale_log2, a.scale_log2), base2 = make_float2(base, base);
                float2 sum[2] = {make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f)};
#pragma unroll
                for (int c = 0; c < BK / 32; c++)
                    if (c * 32 < n) {
                        uint32_t w[16];
#pragma unroll
                        for (int x = 0; x < 16; x++) {
                            float2 e = ffma2(make_float2(s[c * 32 + 2 * x], s[c * 32 + 2 * x + 1]), scale2, base2);
                            e = make_float2(exp2_fast(e.x), exp2_fast(e.y));
                            sum[x & 1] = fadd2(sum[x & 1], e);
                            w[x] = pack2<T>(e.x, e.y);
                        }
                        tmem_store16(s_at + c * 16, w);
                    }
                l += (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
                arrive_p(it);
            }
            if (tl.n > 0) ok &= wait(o_bar + buf(tl.n - 1) * 8, phase(tl.n - 1));
            ok = __all_sync(0xffffffffu, ok);
            fence_after();
            const float inv = l == 0.0f ? 0.0f : 1.0f / l;
            bool bad = !ok || !(l < INFINITY) || (l == 0.0f && sees_any(a, p, ln.nk));
            T *out = static_cast<T *>(a.out) + (ln.q0 + i0 + row) * a.out_row + h * a.out_head;
            if (ok) {
                for (int c = 0; c < dn; c += 16) {
                    float o[16];
                    tmem_load16(o_at + c, o);
                    tmem_wait_load();
#pragma unroll
                    for (int x = 0; x < 16; x++) {
                        o[x] = tl.n == 0 ? 0.0f : o[x] * inv;  // no tile: O was never written
                        bad |= !(fabsf(o[x]) < INFINITY);
                    }
                    if (row < rows) {
                        if (a.out_vec == 2 && c + 16 <= a.d) {
                            uint32_t w[8];
#pragma unroll
                            for (int x = 0; x < 8; x++) w[x] = pack2<T>(o[2 * x], o[2 * x + 1]);
                            reinterpret_cast<uint4 *>(out + c)[0] = make_uint4(w[0], w[1], w[2], w[3]);
                            reinterpret_cast<uint4 *>(out + c)[1] = make_uint4(w[4], w[5], w[6], w[7]);
                        } else {
#pragma unroll
                            for (int x = 0; x < 16; x++)
                                if (c + x < a.d) out[c + x] = from_f32<T>(o[x]);
                        }
                    }
                }
            }
            __syncwarp();
            unsigned again = __ballot_sync(0xffffffffu, bad && row < rows && !(ok && no_numbers<T>(a, l)));
            while (again) {
                const int r = __ffs(again) - 1;
                again &= again - 1;
                row_alone<T>(a, ln, int(i0) + warp * 32 + r, h);
            }
            fence_before();
        }
        done += tl.n;
        turn += tl.n > 0;
        __syncthreads();  // O is read: the next query tile's product may overwrite it
        fence_after();
        if (*give_up) {
            rest_alone<T>(a, i0);
            break;
        }
    }
    fence_before();
    __syncthreads();
    if (warp == MMA_WARP) {
        fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(TMEM_COLS));
    }
}

bool map_rows(CUtensorMap *map, const void *p, int type, int64_t rows, int64_t row, int heads, int64_t head, int d) {
    const EncodeTiled encode = tensor_map_encoder();
    // rows or heads that are all the same one: a stride that no document allows
    if ((heads > 1 && head == 0) || (rows > 1 && row == 0)) return false;
    // a single head's stride is never used, but has to be a valid one
    const cuuint64_t dims[3] = {cuuint64_t(d), cuuint64_t(heads), cuuint64_t(rows)};
    const cuuint64_t strides[2] = {cuuint64_t(heads > 1 ? head : (d + 7) / 8 * 8) * 2, cuuint64_t(rows > 1 ? row : (d + 7) / 8 * 8) * 2};
    const cuuint32_t box[3] = {64, 1, BOX}, each[3] = {1, 1, 1};
    return encode && encode(map, type == PPOCR_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3,
                            const_cast<void *>(p), dims, strides, box, each, CU_TENSOR_MAP_INTERLEAVE_NONE,
                            CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <class T, int BK>
cudaError_t start(const AttnArgs &a, const Maps &maps, uint32_t max_q, cudaStream_t stream) {
    const int panels = (a.d + 63) / 64, shared = panels * 128 * (BQ + 4 * BK);
    const cudaError_t e = raise_shared<attn_tc_kernel<T, BK>>((BK == 64 ? 2 : 1) * 128 * (BQ + 4 * BK));
    if (e != cudaSuccess) return e;
    const uint32_t tiles = max_q ? (max_q + BQ - 1) / BQ : 1;
    attn_tc_kernel<T, BK><<<dim3(tiles, unsigned(a.heads), unsigned(a.lanes)), THREADS, shared, stream>>>(a, maps);
    return cudaGetLastError();
}

template <class T>
cudaError_t start_d(const AttnArgs &a, const Maps &maps, uint32_t max_q, cudaStream_t stream) {
    return a.d > 64 ? start<T, 64>(a, maps, max_q, stream) : start<T, 32>(a, maps, max_q, stream);
}

}  // namespace

cudaError_t launch_attn_tc(const AttnArgs &a, int type, uint32_t max_q, bool *taken, cudaStream_t stream) {
    *taken = false;
    if (type == PPOCR_F32 || a.q_bytes != 16 || a.k_bytes != 16 || a.v_bytes != 16) return cudaSuccess;
    Maps maps;
    if (!map_rows(&maps.q, a.q, type, a.q_rows, a.q_row, a.heads, a.q_head, a.d) ||
        !map_rows(&maps.k, a.k, type, a.kv_rows, a.k_row, a.kv_heads, a.k_head, a.d) ||
        !map_rows(&maps.v, a.v, type, a.kv_rows, a.v_row, a.kv_heads, a.v_head, a.d))
        return cudaSuccess;  // strides the encoder does not take
    *taken = true;
    return type == PPOCR_F16 ? start_d<__half>(a, maps, max_q, stream) : start_d<__nv_bfloat16>(a, maps, max_q, stream);
}

}  // namespace ppocr
