// Window attention over whole lanes (many queries a lane), any type, head
// size and alignment: ppocr_attention_window's general form, and its entry
// point.
//
// A block of four warps takes 64 queries of one head, 16 a warp, and walks
// the key tiles they see (sinks, then the window), 64 keys a tile, two
// buffers filled by cp.async while the other is used (32 in f32, whose
// products are three each: a finer step leaves less of a narrow window's tiles
// hidden, and more blocks an SM; 2000 queries of 8 heads of 128, window 256: 72
// us, 103 with 64); tiles outside every query's window are never read, those
// outside a warp's are skipped, tiles inside every window skip the masks.
//
// Bound by the issue of instructions: f32 takes three products a pair and the
// splitting of their operands. 44 lines of 10 to 200 queries, 8 heads of 15 in
// f32, window 49: 19.3 us (8.4 MB, 1.3 us of HBM; 20.0 before warps skipped the tiles
// in front of their windows).
#include <cmath>

#include "attn.cuh"

namespace ppocr {

namespace {

constexpr int BQ = 64, ROW_THREADS = 128;

template <class T, int DP>
struct RowTile {
    static constexpr int BK = sizeof(T) == 4 ? 32 : 64;
    static constexpr int BLOCKS = DP <= 32 ? 5 : DP <= 64 ? 3 : 2;  // an SM, by registers
    static constexpr int STRIDE = TileOf<T, DP>::STRIDE;
    static constexpr int Q_BYTES = BQ * STRIDE * int(sizeof(T)), K_BYTES = BK * STRIDE * int(sizeof(T));
    static constexpr int SHARED = Q_BYTES + 4 * K_BYTES;
};

template <class T, int DP>
__global__ void __launch_bounds__(ROW_THREADS, RowTile<T, DP>::BLOCKS) attn_rows_kernel(const __grid_constant__ AttnArgs a) {
    using R = RowTile<T, DP>;
    constexpr int BK = R::BK, STRIDE = R::STRIDE;
    extern __shared__ __align__(16) unsigned char smem[];
    const uint32_t qs = shared_u32(smem), kv = qs + R::Q_BYTES;
    const int tid = threadIdx.x, warp = tid / 32, lane = tid & 31;
    const Lane ln = read_lane(a, blockIdx.z);
    const int h = blockIdx.y, kvh = h / a.share;
    const T *k = static_cast<const T *>(a.k) + ln.k0 * a.k_row + kvh * a.k_head;
    const T *v = static_cast<const T *>(a.v) + ln.k0 * a.v_row + kvh * a.v_head;

    for (int64_t i0 = int64_t(blockIdx.x) * BQ; i0 < ln.nq; i0 += int64_t(gridDim.x) * BQ) {
        const int rows = int(ln.nq - i0 < BQ ? ln.nq - i0 : BQ);
        const int p0 = int(i0) + ln.nk - ln.nq, p1 = p0 + rows - 1;
        KeyTiles kt;
        kt.plan<BK>(a, p0, p1, ln.nk);
        const auto fetch = [&](int it, int buf) {
            const int j = kt.first<BK>(it), n = min(BK, kt.end(it) - j);
            load_rows<T, BK, DP, STRIDE, ROW_THREADS>(kv + buf * 2 * R::K_BYTES, k + j * a.k_row, a.k_row, n, a.d, a.k_bytes, tid);
            load_rows<T, BK, DP, STRIDE, ROW_THREADS>(kv + (buf * 2 + 1) * R::K_BYTES, v + j * a.v_row, a.v_row, n, a.d, a.v_bytes, tid);
        };
        __syncthreads();  // the last tile's readers are done
        load_rows<T, BQ, DP, STRIDE, ROW_THREADS>(qs, static_cast<const T *>(a.q) + (ln.q0 + i0) * a.q_row + h * a.q_head, a.q_row,
                                                  rows, a.d, a.q_bytes, tid);
        if (kt.n > 0) fetch(0, 0);
        copy_commit();

        WarpAttn<T, DP> w;
        w.clear();
        const int pw = p0 + warp * 16;  // this warp's first position
        const uint32_t qw = qs + uint32_t(warp * 16 * STRIDE * int(sizeof(T)));
        for (int it = 0; it < kt.n; it++) {
            copy_wait<0>();
            __syncthreads();
            if (it + 1 < kt.n) fetch(it + 1, (it + 1) & 1);
            copy_commit();
            const uint32_t ks = kv + (it & 1) * 2 * R::K_BYTES, vs = ks + R::K_BYTES;
            const int j0 = kt.first<BK>(it), jend = kt.end(it);
            // nothing here for this warp's rows
            if ((a.right >= 0 && j0 > pw + 15 + a.right) || (a.left >= 0 && min(jend, j0 + BK) <= pw - a.left && j0 >= a.sinks)) continue;
            float s[BK / 8][4];
            w.template scores<BK / 8>(s, qw, ks, lane);
            const bool whole = j0 + BK <= jend && (a.right < 0 || j0 + BK - 1 <= pw + a.right) &&
                               (a.left < 0 || j0 >= pw + 15 - a.left || j0 + BK <= a.sinks);
            if (!whole) {
#pragma unroll
                for (int n = 0; n < BK / 8; n++)
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const int j = j0 + n * 8 + (lane & 3) * 2 + (e & 1), p = pw + (lane >> 2) + (e >> 1) * 8;
                        if (j >= jend || !sees(a, p, j)) s[n][e] = -INFINITY;
                    }
            }
            w.template soften<BK / 8>(s, a.scale_log2);
            w.template gather<BK / 8>(s, vs, lane);
        }
        copy_wait<0>();

        // rows g and g + 8: the sums over the row's four lanes, the output
        bool bad[2] = {false, false};
        float inv[2];
#pragma unroll
        for (int r = 0; r < 2; r++) {
            w.l[r] += __shfl_xor_sync(0xffffffffu, w.l[r], 1);
            w.l[r] += __shfl_xor_sync(0xffffffffu, w.l[r], 2);
            inv[r] = w.l[r] == 0.0f ? 0.0f : 1.0f / w.l[r];
            bad[r] = w.l[r] == 0.0f;  // it sees no key, or scores that overflowed
        }
#pragma unroll
        for (int n = 0; n < DP / 8; n++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                w.o[n][e] *= inv[e >> 1];
                bad[e >> 1] |= !(fabsf(w.o[n][e]) < INFINITY);
            }
#pragma unroll
        for (int r = 0; r < 2; r++) {
            bad[r] = bad[r] && !no_numbers<T>(a, w.l[r]);
            const unsigned any = __ballot_sync(0xffffffffu, bad[r]);
            const int row = warp * 16 + r * 8 + (lane >> 2);
            bad[r] = (any >> (lane & 28)) & 15u;
            if (row < rows && !bad[r]) {
                T *out = static_cast<T *>(a.out) + (ln.q0 + i0 + row) * a.out_row + h * a.out_head;
#pragma unroll
                for (int n = 0; n < DP / 8; n++) {
                    const int c = n * 8 + (lane & 3) * 2;
                    if (a.out_vec && c + 1 < a.d) {
                        if constexpr (sizeof(T) == 2)
                            *reinterpret_cast<uint32_t *>(out + c) = pack2<T>(w.o[n][2 * r], w.o[n][2 * r + 1]);
                        else
                            *reinterpret_cast<float2 *>(out + c) = make_float2(w.o[n][2 * r], w.o[n][2 * r + 1]);
                    } else {
                        if (c < a.d) out[c] = from_f32<T>(w.o[n][2 * r]);
                        if (c + 1 < a.d) out[c + 1] = from_f32<T>(w.o[n][2 * r + 1]);
                    }
                }
            }
            for (int x = 0; x < 8; x++)
                if ((any >> (4 * x)) & 15u) {
                    const int again = warp * 16 + r * 8 + x;
                    if (again < rows) row_alone<T>(a, ln, int(i0) + again, h);
                }
        }
    }
}

template <class T, int DP>
cudaError_t start_rows(const AttnArgs &a, uint32_t max_q, cudaStream_t stream) {
    constexpr int shared = RowTile<T, DP>::SHARED;
    const cudaError_t e = raise_shared<attn_rows_kernel<T, DP>>(shared);
    if (e != cudaSuccess) return e;
    const uint32_t tiles = max_q ? (max_q + BQ - 1) / BQ : 1;
    attn_rows_kernel<T, DP><<<dim3(tiles, unsigned(a.heads), unsigned(a.lanes)), ROW_THREADS, shared, stream>>>(a);
    return cudaGetLastError();
}

template <class T>
cudaError_t start_rows_d(const AttnArgs &a, uint32_t max_q, cudaStream_t stream) {
    if (a.d <= 16) return start_rows<T, 16>(a, max_q, stream);
    if (a.d <= 32) return start_rows<T, 32>(a, max_q, stream);
    if (a.d <= 64) return start_rows<T, 64>(a, max_q, stream);
    return start_rows<T, 128>(a, max_q, stream);
}

// The widest copy that every row and head of a tensor allows.
int copy_bytes(const void *p, uint64_t row, uint64_t head, size_t size) {
    const uint64_t all = reinterpret_cast<uintptr_t>(p) | row * size | head * size;
    return all % 16 == 0 ? 16 : all % 4 == 0 ? 4 : 2;
}

}  // namespace

cudaError_t launch_attn_rows(const AttnArgs &a, int type, uint32_t max_q, cudaStream_t stream) {
    if (type == PPOCR_F32) return start_rows_d<float>(a, max_q, stream);
    if (type == PPOCR_F16) return start_rows_d<__half>(a, max_q, stream);
    return start_rows_d<__nv_bfloat16>(a, max_q, stream);
}

}  // namespace ppocr

using namespace ppocr;

extern "C" int ppocr_attention_window(const ppocr_attention_shape *s, const void *q, const void *k, const void *v,
                                      void *out, const int64_t *q_offsets, const int64_t *k_begin,
                                      const int32_t *k_len, void *stream) {
    static const char *me = "ppocr_attention_window";
    clear_error();
    if (!s) return refuse(PPOCR_E_ARG, me, "null shape");
    if (s->type != PPOCR_F32 && s->type != PPOCR_F16 && s->type != PPOCR_BF16)
        return refuse(PPOCR_E_ARG, me, "type must be PPOCR_F32, PPOCR_F16 or PPOCR_BF16");
    if (!s->heads || !s->kv_heads || s->heads % s->kv_heads)
        return refuse(PPOCR_E_ARG, me, "heads must be a multiple of kv_heads");
    if (s->left < -1 || s->right < -1) return refuse(PPOCR_E_ARG, me, "left and right are -1 (no limit) or more");
    if (!std::isfinite(s->scale) || s->scale < 0.0f) return refuse(PPOCR_E_ARG, me, "scale must be finite and not negative");
    if (!s->head_dim || s->head_dim > 128) return refuse(PPOCR_E_SIZE, me, "head_dim must be between 1 and 128");
    if (s->heads > 65535 || s->lanes > 65535) return refuse(PPOCR_E_SIZE, me, "more than 65535 heads or lanes");
    const uint64_t most = uint64_t(1) << 40, rows_most = uint64_t(1) << 29;
    if (s->q_rows > rows_most || s->kv_rows > rows_most) return refuse(PPOCR_E_SIZE, me, "more than 2^29 rows");
    if (s->q_row > most || s->q_head > most || s->k_row > most || s->k_head > most || s->v_row > most ||
        s->v_head > most || s->out_row > most || s->out_head > most)
        return refuse(PPOCR_E_SIZE, me, "a stride above 2^40 elements");
    if (!s->lanes || !s->q_rows) return PPOCR_OK;
    if (!q || !out || !q_offsets) return refuse(PPOCR_E_ARG, me, "null buffer");
    if (s->kv_rows && (!k || !v)) return refuse(PPOCR_E_ARG, me, "null buffer");
    if (!k_begin != !k_len) return refuse(PPOCR_E_ARG, me, "k_begin and k_len come together");
    const size_t size = type_size(s->type);
    if (!aligned(q, size) || !aligned(k, size) || !aligned(v, size) || !aligned(out, size) || !aligned(q_offsets, 8) ||
        !aligned(k_begin, 8) || !aligned(k_len, 4))
        return refuse(PPOCR_E_ARG, me, "a buffer is not aligned to its type");
    // rows and heads of the output may not share elements
    const uint64_t d = s->head_dim;
    const bool apart = (s->out_head >= d || s->heads == 1) && (s->out_row >= uint64_t(s->heads - 1) * s->out_head + d || s->q_rows == 1);
    const bool apart2 = (s->out_row >= d || s->q_rows == 1) && (s->out_head >= (s->q_rows - 1) * s->out_row + d || s->heads == 1);
    if (!apart && !apart2) return refuse(PPOCR_E_ARG, me, "output rows or heads overlap");
    // 2^29 rows x 2^40 elements fit neither the card nor 64 bits of bytes
    const auto span = [&](uint64_t rows, uint64_t row, uint64_t heads, uint64_t head) {
        const double n = (rows ? double(rows - 1) : 0.0) * double(row) + double(heads - 1) * double(head) + double(d);
        return n > 1e15 ? uint64_t(0) : rows ? ((rows - 1) * row + (heads - 1) * head + d) * size : uint64_t(1);
    };
    const uint64_t qn = span(s->q_rows, s->q_row, s->heads, s->q_head), on = span(s->q_rows, s->out_row, s->heads, s->out_head);
    const uint64_t kn = span(s->kv_rows, s->k_row, s->kv_heads, s->k_head), vn = span(s->kv_rows, s->v_row, s->kv_heads, s->v_head);
    if (!qn || !on || !kn || !vn) return refuse(PPOCR_E_SIZE, me, "a tensor spans more than 10^15 elements");
    // rows of all their heads, where these lie side by side
    const auto rows = [&](const void *p, uint64_t n, uint64_t row, uint64_t heads, uint64_t head) {
        return Rows{p, n, ((heads - 1) * head + d) * size, row * size};
    };
    const Rows outs = rows(out, on, s->out_row, s->heads, s->out_head);
    if (overlap(outs, rows(q, qn, s->q_row, s->heads, s->q_head)) ||
        (s->kv_rows && (overlap(outs, rows(k, kn, s->k_row, s->kv_heads, s->k_head)) || overlap(outs, rows(v, vn, s->v_row, s->kv_heads, s->v_head)))))
        return refuse(PPOCR_E_ARG, me, "out overlaps q, k or v");

    bool local = false;
    if (const int bad = check_buffers(me, {q, s->kv_rows ? k : nullptr, s->kv_rows ? v : nullptr, out, q_offsets, k_begin, k_len}, &local)) return bad;

    AttnArgs a{};
    a.q = q, a.k = k, a.v = v, a.out = out;
    a.q_offsets = q_offsets, a.k_begin = k_begin, a.k_len = k_len;
    a.q_rows = int64_t(s->q_rows), a.kv_rows = int64_t(s->kv_rows);
    a.q_row = int64_t(s->q_row), a.q_head = int64_t(s->q_head), a.k_row = int64_t(s->k_row), a.k_head = int64_t(s->k_head);
    a.v_row = int64_t(s->v_row), a.v_head = int64_t(s->v_head), a.out_row = int64_t(s->out_row), a.out_head = int64_t(s->out_head);
    a.lanes = int(s->lanes), a.heads = int(s->heads), a.kv_heads = int(s->kv_heads), a.share = a.heads / a.kv_heads;
    a.d = int(s->head_dim);
    // positions lie below 2^29 in size, so these limits cut nothing and sums stay in 32 bits
    const int32_t far = int32_t(1) << 29;
    a.left = s->left, a.right = s->right < far ? s->right : far;
    a.left = a.left < far ? a.left : far;
    a.sinks = int(s->sinks < uint32_t(far) ? s->sinks : uint32_t(far));
    // a scale of zero would turn a hidden score's minus infinity into NaN
    a.scale_log2 = s->scale * 1.4426950408889634f;
    if (a.scale_log2 < 1.2e-38f) a.scale_log2 = 1.2e-38f;
    a.q_bytes = copy_bytes(q, s->q_row, s->q_head, size);
    a.k_bytes = copy_bytes(k, s->k_row, s->k_head, size);
    a.v_bytes = copy_bytes(v, s->v_row, s->v_head, size);
    a.out_vec = copy_bytes(out, s->out_row, s->out_head, size) == 16 ? 2 : (reinterpret_cast<uintptr_t>(out) | s->out_row * size | s->out_head * size) % (2 * size) == 0 ? 1 : 0;

    const uint32_t max_q = s->max_q ? uint32_t(s->max_q < s->q_rows ? s->max_q : s->q_rows) : uint32_t(s->q_rows);
    uint64_t keys = s->max_k && s->max_k < s->kv_rows ? s->max_k : s->kv_rows;
    if (a.left >= 0 && a.right >= 0) {
        const uint64_t seen = uint64_t(a.left) + uint64_t(a.right) + max_q + uint64_t(a.sinks);
        keys = keys < seen ? keys : seen;
    }
    const auto str = static_cast<cudaStream_t>(stream);
    // The split form walks a tile's keys with 4 to 32 warps and takes the heads that
    // share a key head as rows of one tile; the others walk them alone, 64 or 128
    // queries of a head at a time. Split, then,
    // - where its tiles fill the card at most once and there are keys to split (8 key
    //   heads of 64, window 1024, a query: 7.6 us where the others take 20 in bf16 and 79
    //   in f32; 17 keys: 5.8 us, 4.7 and 5.9; 16 lanes of 16 queries: 15, 28 and 80 us);
    // - where its tiles are half as many as the others' blocks or fewer (32 lanes of
    //   4 heads a key head: 27 us, 63 and 358);
    // - in f32 with keys to split, up to twice as many tiles as blocks or SMs (32 lanes
    //   of 32 queries, head sizes 16, 64 and 128: 30, 93 and 238 us, 48, 116 and 216
    //   the other way; of 64 queries: 50, 182 and 415 and 49, 119 and 223).
    // Beyond, in bf16, head sizes 64 and 128: 27 and 35 us for 32 lanes of one query
    // and head where the others take 30 and 29.
    const bool f32 = s->type == PPOCR_F32;
    const uint64_t sms = uint64_t(sm_count()), per_head = uint64_t(a.lanes) * a.kv_heads;
    const uint64_t tiles = (uint64_t(max_q) * a.share + 15) / 16 * per_head;
    const uint64_t blocks = (uint64_t(max_q) + 63) / 64 * a.share * per_head;
    if ((tiles <= sms && keys >= (f32 ? 64 : 256)) || (2 * tiles <= blocks && blocks > sms) ||
        (f32 && tiles <= 2 * (blocks > sms ? blocks : sms) && keys >= 256)) {
        const cudaError_t e = launch_attn_split(a, s->type, max_q, uint32_t(keys), str);
        return e == cudaSuccess ? int(PPOCR_OK) : refuse(PPOCR_E_DEVICE, me, cudaGetErrorString(e));
    }
    // (tensor copies of the device's own memory alone: no document promises them of the host's)
    bool taken = false;
    cudaError_t e = local ? launch_attn_tc(a, s->type, max_q, &taken, str) : cudaSuccess;
    if (!taken) e = launch_attn_rows(a, s->type, max_q, str);
    return e == cudaSuccess ? int(PPOCR_OK) : refuse(PPOCR_E_DEVICE, me, cudaGetErrorString(e));
}
