// Window attention: the arguments and the warp-level pieces that its kernels
// share.
//
// Lane b has queries i in [0, nq) and keys j in [0, nk); query i stands at
// key position p = i + nk - nq. It sees key j when
//     j <= p + right  and  (j >= p - left  or  j < sinks),
// a negative left or right meaning no limit, and its output is
//     sum_j softmax_j(scale * q_i . k_j) v_j   over the keys it sees,
// zero when it sees none. The softmax runs in one pass: a running maximum m
// and sum l per row in f32, the accumulator scaled by 2^(m_old - m_new)
// whenever the maximum moves, scores in units of log2 (scale * log2 e).
#pragma once

#include "block.cuh"

namespace ppocr {

struct AttnArgs {
    const void *q, *k, *v;
    void *out;
    const int64_t *q_offsets, *k_begin;
    const int32_t *k_len;
    int64_t q_rows, kv_rows;
    int64_t q_row, q_head, k_row, k_head, v_row, v_head, out_row, out_head;  // elements
    int lanes, heads, kv_heads, share, d;
    int left, right, sinks;  // left, right -1: no limit
    float scale_log2;  // the scale times log2 e
    int q_bytes, k_bytes, v_bytes;  // widest copy each tensor's rows allow: 16, 4 or 2 bytes
    int sort;                        // split form: take the lanes by their keys, most first
    int out_vec;                     // 1 when pairs of outputs may be stored together, 2 when 16 bytes may
};

namespace {

struct Lane {
    int64_t q0, k0;  // first row of its queries and of its keys
    int nq, nk;
};

// A lane's rows, cut to the rows the tensors hold whatever the arrays say.
__device__ __forceinline__ Lane read_lane(const AttnArgs &a, int b) {
    Lane l;
    int64_t q0 = __ldg(a.q_offsets + b), q1 = __ldg(a.q_offsets + b + 1);
    q0 = q0 < 0 ? 0 : q0 > a.q_rows ? a.q_rows : q0;
    q1 = q1 < q0 ? q0 : q1 > a.q_rows ? a.q_rows : q1;
    int64_t k0 = q0, n = q1 - q0;
    if (a.k_begin) {
        k0 = __ldg(a.k_begin + b);
        n = __ldg(a.k_len + b);
    }
    k0 = k0 < 0 ? 0 : k0 > a.kv_rows ? a.kv_rows : k0;
    n = n < 0 ? 0 : n > a.kv_rows - k0 ? a.kv_rows - k0 : n;
    l.q0 = q0;
    l.nq = int(q1 - q0);
    l.k0 = k0;
    l.nk = int(n);
    return l;
}

__device__ __forceinline__ bool sees(const AttnArgs &a, int p, int j) {
    return (a.right < 0 || j <= p + a.right) && (a.left < 0 || j >= p - a.left || j < a.sinks);
}

// Whether position p sees any of nk keys.
__device__ __forceinline__ bool sees_any(const AttnArgs &a, int p, int nk) {
    const int hi = a.right < 0 ? nk : min(nk, p + a.right + 1), lo = a.left < 0 ? 0 : max(0, p - a.left);
    return hi > 0 && (lo < hi || a.sinks > 0);
}

// The key tiles that queries at positions [p0, p1] need: the sinks below the
// window first, then the window from a multiple of the tile size on.
struct KeyTiles {
    int sink_end, lo, hi, n_sink, n;
    template <int BK>
    __device__ __forceinline__ void plan(const AttnArgs &a, int p0, int p1, int nk) {
        hi = a.right < 0 ? nk : min(nk, p1 + a.right + 1);
        hi = max(hi, 0);
        lo = a.left < 0 ? 0 : max(0, p0 - a.left);
        lo = min(lo / BK * BK, hi);
        sink_end = min(a.sinks, lo);
        n_sink = (sink_end + BK - 1) / BK;
        n = n_sink + (hi - lo + BK - 1) / BK;
    }
    // tile `it`: its keys are [first, end), fewer than BK at the ends
    template <int BK>
    __device__ __forceinline__ int first(int it) const {
        return it < n_sink ? it * BK : lo + (it - n_sink) * BK;
    }
    __device__ __forceinline__ int end(int it) const { return it < n_sink ? sink_end : hi; }
};

// Rows [0, rows) of a tensor's one head into a shared tile of ROWS rows of
// STRIDE elements, zeros past `rows` and past d, by THREADS threads.
template <class T, int ROWS, int DP, int STRIDE, int W, int THREADS>
__device__ __forceinline__ void load_rows_w(uint32_t dst, const T *src, int64_t row_stride, int rows, int d, int tid) {
    constexpr int E = W / int(sizeof(T)), CPR = DP / E;
    if constexpr (W >= 4 && THREADS % CPR == 0 && ROWS % (THREADS / CPR) == 0) {
        // a thread's copies lie in one column, THREADS / CPR rows apart
        constexpr int STEP = THREADS / CPR;
        const int r0 = tid / CPR, c = tid % CPR * E;
        const int left = (d - c) * int(sizeof(T)), valid = left < 0 ? 0 : left > W ? W : left;
        const T *from = src + r0 * row_stride + c;
        uint32_t to = dst + uint32_t((r0 * STRIDE + c) * int(sizeof(T)));
        const int64_t step = STEP * row_stride;
        if (rows == ROWS && d == DP) {
#pragma unroll
            for (int i = 0; i < ROWS / STEP; i++, from += step) copy_async<W>(to + uint32_t(i * STEP * STRIDE * int(sizeof(T))), from, W);
        } else {
#pragma unroll
            for (int i = 0; i < ROWS / STEP; i++, from += step) {
                const int v = r0 + i * STEP < rows ? valid : 0;
                copy_async<W>(to + uint32_t(i * STEP * STRIDE * int(sizeof(T))), v ? from : src, v);
            }
        }
    } else {
        for (int e = tid; e < ROWS * CPR; e += THREADS) {
            const int r = e / CPR, c = e % CPR;
            const int left = r < rows ? (d - c * E) * int(sizeof(T)) : 0;
            const int valid = left < 0 ? 0 : left > W ? W : left;
            const T *from = valid ? src + r * row_stride + c * E : src;
            const uint32_t to = dst + uint32_t((r * STRIDE + c * E) * int(sizeof(T)));
            if constexpr (W >= 4) {
                copy_async<W>(to, from, valid);
            } else {
                uint16_t v = 0;
                if (valid) v = __ldg(reinterpret_cast<const uint16_t *>(from));
                asm volatile("st.shared.u16 [%0], %1;" ::"r"(to), "h"(v) : "memory");
            }
        }
    }
}
template <class T, int ROWS, int DP, int STRIDE, int THREADS>
__device__ __forceinline__ void load_rows(uint32_t dst, const T *src, int64_t row_stride, int rows, int d, int bytes, int tid) {
    if (bytes == 16)
        load_rows_w<T, ROWS, DP, STRIDE, 16, THREADS>(dst, src, row_stride, rows, d, tid);
    else if (sizeof(T) == 4 || bytes == 4)
        load_rows_w<T, ROWS, DP, STRIDE, 4, THREADS>(dst, src, row_stride, rows, d, tid);
    else if constexpr (sizeof(T) == 2)
        load_rows_w<T, ROWS, DP, STRIDE, 2, THREADS>(dst, src, row_stride, rows, d, tid);
}

// Row strides of the shared tiles, padded so that a fragment's 32 accesses
// fall into 32 banks.
template <class T, int DP>
struct TileOf {
    static constexpr int STRIDE = sizeof(T) == 4 ? DP + 4 : DP + 8;
};

// One warp's 16 query rows against tiles of keys. Scores and output use the
// matrix instruction's layout: this lane holds rows g and g + 8 (g = lane /
// 4) and columns 2t, 2t + 1 of each 8 (t = lane % 4).
//
// f16 and bf16: m16n8k16 with f32 accumulation; the probabilities are
// rounded to the type for the second product (2^-9 or 2^-12 of each, the
// size of the output's own rounding), the sum l keeps them unrounded.
// f32: each product as three tf32 ones (hi*hi + hi*lo + lo*hi), the sums of a tile
// apart from those of the lane.
template <class T, int DP>
struct WarpAttn {
    static constexpr int STRIDE = TileOf<T, DP>::STRIDE;
    static constexpr int ND = DP / 8;
    float o[ND][4];
    float m[2], l[2], keep[2];

    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int n = 0; n < ND; n++) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.0f;
        m[0] = m[1] = -INFINITY;
        l[0] = l[1] = 0.0f;
    }

    // s[nt] = q (16 rows from qs) . the 8 * NT keys at ks
    template <int NT>
    __device__ __forceinline__ void scores(float (*s)[4], uint32_t qs, uint32_t ks, int lane) const {
#pragma unroll
        for (int n = 0; n < NT; n++) s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.0f;
        if constexpr (sizeof(T) == 2) {
            const uint32_t qa = qs + uint32_t(((lane & 15) * STRIDE + (lane >> 4) * 8) * 2);
            const uint32_t ka = ks + uint32_t((((lane & 7) + (lane >> 4) * 8) * STRIDE + ((lane >> 3) & 1) * 8) * 2);
#pragma unroll
            for (int kk = 0; kk < DP / 16; kk++) {
                uint32_t qf[4];
                ldmatrix4(qf, qa + kk * 32);
#pragma unroll
                for (int n = 0; n < NT; n += 2) {
                    uint32_t kf[4];
                    ldmatrix4(kf, ka + uint32_t(n * 8 * STRIDE * 2) + kk * 32);
                    mma16<T>(s[n], qf, kf[0], kf[1]);
                    mma16<T>(s[n + 1], qf, kf[2], kf[3]);
                }
            }
        } else {
            const int g = lane >> 2, t = lane & 3;
            const uint32_t qa = qs + uint32_t((g * STRIDE + t) * 4), ka = ks + uint32_t((g * STRIDE + t) * 4);
            // The matrix units cut a sum's low bits where f32 addition rounds them, always
            // toward zero: the small products go into sums of their own.
            float small[NT][4];
#pragma unroll
            for (int n = 0; n < NT; n++) small[n][0] = small[n][1] = small[n][2] = small[n][3] = 0.0f;
            // unrolled by two only: more would spill
#pragma unroll 2
            for (int kk = 0; kk < DP / 8; kk++) {
                uint32_t qh[4], ql[4];
                split_tf32(lds(qa + kk * 32), qh[0], ql[0]);
                split_tf32(lds(qa + kk * 32 + 8 * STRIDE * 4), qh[1], ql[1]);
                split_tf32(lds(qa + kk * 32 + 16), qh[2], ql[2]);
                split_tf32(lds(qa + kk * 32 + 8 * STRIDE * 4 + 16), qh[3], ql[3]);
#pragma unroll
                for (int n = 0; n < NT; n++) {
                    uint32_t h0, h1, l0, l1;
                    split_tf32(lds(ka + uint32_t(n * 8 * STRIDE * 4) + kk * 32), h0, l0);
                    split_tf32(lds(ka + uint32_t(n * 8 * STRIDE * 4) + kk * 32 + 16), h1, l1);
                    mma8_tf32(small[n], ql, h0, h1);
                    mma8_tf32(small[n], qh, l0, l1);
                    mma8_tf32(s[n], qh, h0, h1);
                }
            }
#pragma unroll
            for (int n = 0; n < NT; n++)
#pragma unroll
                for (int e = 0; e < 4; e++) s[n][e] += small[n][e];
        }
    }

    static __device__ __forceinline__ float lds(uint32_t a) {
        float v;
        asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(a));
        return v;
    }

    // The softmax step over 8 * NT scores (masked ones are -inf): p in place.
    template <int NT>
    __device__ __forceinline__ void soften(float (*s)[4], float scale_log2) {
        float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
        for (int n = 0; n < NT; n++) {
            top[0] = fmaxf(top[0], fmaxf(s[n][0], s[n][1]));
            top[1] = fmaxf(top[1], fmaxf(s[n][2], s[n][3]));
        }
        float from[2];
#pragma unroll
        for (int r = 0; r < 2; r++) {
            top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 1));
            top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 2));
            const float now = fmaxf(m[r], top[r] * scale_log2);
            from[r] = now == -INFINITY ? 0.0f : now;  // no key seen yet: every p is 2^-inf
            keep[r] = exp2_fast(m[r] - from[r]);
            m[r] = now;
        }
        float sum[2] = {0.0f, 0.0f};
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                s[n][e] = exp2_fast(fmaf(s[n][e], scale_log2, -from[e >> 1]));
                sum[e >> 1] += s[n][e];
            }
        l[0] = fmaf(l[0], keep[0], sum[0]);
        l[1] = fmaf(l[1], keep[1], sum[1]);
        // (f32's sums take the factor as they take the tile)
        if (sizeof(T) == 2 && __any_sync(0xffffffffu, keep[0] != 1.0f || keep[1] != 1.0f)) {
#pragma unroll
            for (int n = 0; n < ND; n++) {
                o[n][0] *= keep[0];
                o[n][1] *= keep[0];
                o[n][2] *= keep[1];
                o[n][3] *= keep[1];
            }
        }
    }

    // o += p . the 8 * NT rows at vs
    template <int NT>
    __device__ __forceinline__ void gather(float (*s)[4], uint32_t vs, int lane) {
        if constexpr (sizeof(T) == 2) {
            const uint32_t va = vs + uint32_t((((lane & 7) + ((lane >> 3) & 1) * 8) * STRIDE + (lane >> 4) * 8) * 2);
#pragma unroll
            for (int n = 0; n < NT; n += 2) {
                const uint32_t pf[4] = {pack2<T>(s[n][0], s[n][1]), pack2<T>(s[n][2], s[n][3]),
                                        pack2<T>(s[n + 1][0], s[n + 1][1]), pack2<T>(s[n + 1][2], s[n + 1][3])};
#pragma unroll
                for (int c = 0; c < ND; c += 2) {
                    uint32_t vf[4];
                    ldmatrix4_t(vf, va + uint32_t((n * 8 * STRIDE + c * 8) * 2));
                    mma16<T>(o[c], pf, vf[0], vf[1]);
                    mma16<T>(o[c + 1], pf, vf[2], vf[3]);
                }
            }
        } else {
            // key slots t and t + 4 of the instruction stand for keys 2t and
            // 2t + 1, where this lane's probabilities are
            const int g = lane >> 2, t = lane & 3;
            const uint32_t va = vs + uint32_t((2 * t * STRIDE + g) * 4);
            uint32_t ph[NT][4], pl[NT][4];
#pragma unroll
            for (int n = 0; n < NT; n++) {
                split_tf32(s[n][0], ph[n][0], pl[n][0]);
                split_tf32(s[n][2], ph[n][1], pl[n][1]);
                split_tf32(s[n][1], ph[n][2], pl[n][2]);
                split_tf32(s[n][3], ph[n][3], pl[n][3]);
            }
            // the tile's sums by themselves, then into o by a rounded addition
#pragma unroll
            for (int c = 0; c < ND; c++) {
                float sum[4] = {}, small[4] = {};
#pragma unroll
                for (int n = 0; n < NT; n++) {
                    uint32_t h0, h1, l0, l1;
                    split_tf32(lds(va + uint32_t((n * 8 * STRIDE + c * 8) * 4)), h0, l0);
                    split_tf32(lds(va + uint32_t(((n * 8 + 1) * STRIDE + c * 8) * 4)), h1, l1);
                    mma8_tf32(small, pl[n], h0, h1);
                    mma8_tf32(small, ph[n], l0, l1);
                    mma8_tf32(sum, ph[n], h0, h1);
                }
#pragma unroll
                for (int e = 0; e < 4; e++) o[c][e] = fmaf(o[c][e], keep[e >> 1], sum[e] + small[e]);
            }
        }
    }
};

// q . k of one head's row, in f32; 16 bytes at a time where both rows allow it.
template <class T>
__device__ __forceinline__ float dot_row(const AttnArgs &a, const T *q, const T *k) {
    constexpr int E = 16 / int(sizeof(T));
    float s = 0.0f;
    int c = 0;
    if (a.q_bytes == 16 && a.k_bytes == 16) {
        float part[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
        for (; c + E <= a.d; c += E) {
            const uint4 qv = __ldg(reinterpret_cast<const uint4 *>(q + c)), kv = __ldg(reinterpret_cast<const uint4 *>(k + c));
            const T *x = reinterpret_cast<const T *>(&qv), *y = reinterpret_cast<const T *>(&kv);
#pragma unroll
            for (int e = 0; e < E; e++) part[e & 3] = fmaf(to_f32(x[e]), to_f32(y[e]), part[e & 3]);
        }
        s = (part[0] + part[1]) + (part[2] + part[3]);
    }
    for (; c < a.d; c++) s = fmaf(to_f32(q[c]), to_f32(k[c]), s);
    return s;
}

// Whether a row whose sum of weights is `sum` is known not to be numbers: hidden scores
// are minus infinity and weigh nothing, so a NaN comes from a score that the row sees.
// Not so in f32, where an infinity's tf32 remainder is NaN, nor where finite
// scores overflow in units of log2.
template <class T>
__device__ __forceinline__ bool no_numbers(const AttnArgs &a, float sum) {
    return sizeof(T) == 2 && sum != sum && a.scale_log2 <= 1.0f;
}

// One output row the plain way, by a whole warp, in f32 and over the keys it
// sees alone: for rows that came out infinite or NaN above, since there a
// masked key's zero weight times an infinity or NaN in its values is NaN, and
// values near the largest number overflow where the weights, not yet divided by
// their sum, exceed one (here the output is divided by the sum at every step); and for
// rows that see keys whose weights all came out as zeros, since a score above 0.69 of the
// largest number overflows in units of log2 (here the difference to the maximum is
// taken first, halved lest it overflow). A key a lane, 32 at a time, then channels a lane:
// 4000 causal queries of 8 heads of 64 that all see an infinity, bf16: 17 ms (199 with
// a key at a time); one NaN score ends a row.
template <class T>
__device__ __noinline__ void row_alone(const AttnArgs &a, const Lane &ln, int i, int h) {
    const int lane = threadIdx.x & 31, p = i + ln.nk - ln.nq, kvh = h / a.share;
    const T *q = static_cast<const T *>(a.q) + (ln.q0 + i) * a.q_row + h * a.q_head;
    const T *k = static_cast<const T *>(a.k) + ln.k0 * a.k_row + kvh * a.k_head;
    const T *v = static_cast<const T *>(a.v) + ln.k0 * a.v_row + kvh * a.v_head;
    const int hi = max(0, a.right < 0 ? ln.nk : min(ln.nk, p + a.right + 1)), lo = a.left < 0 ? 0 : min(max(0, p - a.left), hi);
    const int sink_end = min(a.sinks, lo);
    // channels: 16 bytes of them a lane, so that 32 / across keys are taken at once; or
    // lane, lane + 32 and so on
    constexpr int E = 16 / int(sizeof(T));
    const bool wide = a.v_bytes == 16 && a.d % E == 0;
    int across = 1;
    while (across * E < a.d) across *= 2;
    const int c0 = (lane & (across - 1)) * E;
    float acc[E] = {}, top = -INFINITY, sum = 0.0f;
    bool seen = false;
    // 2^(the scores' difference)
    const auto weight = [&](float s, float from) { return exp2_fast((0.5f * s - 0.5f * from) * (2.0f * a.scale_log2)); };
    for (int j0 = sink_end > 0 ? 0 : lo; j0 < hi; j0 = j0 < sink_end && j0 + 32 >= sink_end ? lo : j0 + 32) {
        const int n = min(32, (j0 < sink_end ? sink_end : hi) - j0);
        const float s = lane < n ? dot_row(a, q, k + int64_t(j0 + lane) * a.k_row) : -INFINITY;
        seen = true;
        float high = s;
#pragma unroll
        for (int x = 16; x; x >>= 1) high = fmaxf(high, __shfl_xor_sync(0xffffffffu, high, x));
        if (__any_sync(0xffffffffu, s != s) || high == INFINITY) {
            sum = NAN;
            break;
        }
        if (high == -INFINITY) continue;  // nothing here, unless nothing is anywhere
        const float now = fmaxf(top, high), keep = top == -INFINITY ? 0.0f : weight(top, now);
        float w = lane < n ? weight(s, now) : 0.0f, add = w;
#pragma unroll
        for (int x = 16; x; x >>= 1) add += __shfl_xor_sync(0xffffffffu, add, x);
        const float before = sum * keep;
        sum = before + add, top = now;
        w /= sum;
#pragma unroll
        for (int e = 0; e < E; e++) acc[e] *= before / sum;
        if (wide) {
#pragma unroll 4
            for (int x0 = 0; x0 < n; x0 += 32 / across) {
                const int x = x0 + lane / across;
                const float wx = __shfl_sync(0xffffffffu, w, x);
                if (x >= n || c0 >= a.d) continue;
                const uint4 vv = __ldg(reinterpret_cast<const uint4 *>(v + (j0 + x) * a.v_row + c0));
                const T *y = reinterpret_cast<const T *>(&vv);
#pragma unroll
                for (int e = 0; e < E; e++) acc[e] = fmaf(wx, to_f32(y[e]), acc[e]);
            }
        } else {
            for (int x = 0; x < n; x++) {
                const float wx = __shfl_sync(0xffffffffu, w, x);
                const T *row = v + (j0 + x) * a.v_row;
#pragma unroll
                for (int e = 0; e < 4; e++)
                    if (lane + 32 * e < a.d) acc[e] = fmaf(wx, to_f32(row[lane + 32 * e]), acc[e]);
            }
        }
    }
    // a sum of NaN, or keys that all score minus infinity
    const bool none = sum != sum || (seen && sum == 0.0f);
    T *out = static_cast<T *>(a.out) + (ln.q0 + i) * a.out_row + h * a.out_head;
    if (wide) {
        for (int x = across; x < 32; x *= 2)
#pragma unroll
            for (int e = 0; e < E; e++) acc[e] += __shfl_xor_sync(0xffffffffu, acc[e], x);
#pragma unroll
        for (int e = 0; e < E; e++)
            if (lane < across && c0 < a.d) out[c0 + e] = from_f32<T>(none ? NAN : acc[e]);
    } else {
#pragma unroll
        for (int e = 0; e < 4; e++)
            if (lane + 32 * e < a.d) out[lane + 32 * e] = from_f32<T>(none ? NAN : acc[e]);
    }
}

}  // namespace

// Each returns a CUDA error; the grid covers any lane lengths, the hints
// only size it.
cudaError_t launch_attn_rows(const AttnArgs &a, int type, uint32_t max_q, cudaStream_t stream);
// *taken says whether this form takes the call (types, alignment).
cudaError_t launch_attn_tc(const AttnArgs &a, int type, uint32_t max_q, bool *taken, cudaStream_t stream);
cudaError_t launch_attn_split(const AttnArgs &a, int type, uint32_t max_q, uint32_t max_keys, cudaStream_t stream);

}  // namespace ppocr
