// ppocr_rms_norm_e4m3: the residual's addition, the root-mean-square norm and
// its 8-bit output, one pass over the row.
//
//     s = x + r;  n = s * rsqrt(mean(s^2) + eps) * gamma
//     scale_g = max |n| over group g / 448;  y = e4m3(n / scale_g)
//
// A row lies in the registers of its threads (8 consecutive channels a
// chunk, up to four chunks a thread), so x and r are read once and nothing
// is read again: s leaves rounded to the type, the norm uses the f32 s. The
// sum of squares is kept in f32: lane sums, a shuffle tree, then the warps'
// sums in order (the same order every time). Bound by HBM bytes.
#include <cuda_fp8.h>

#include <cmath>

#include "block.cuh"

namespace ppocr {

namespace {

struct RmsArgs {
    const void *x, *r;
    const float *gamma;
    void *sum;
    uint8_t *y;
    float *scales;
    int64_t rows, x_row, r_row, sum_row, y_row;
    int channels, group, groups;
    float eps;
};

template <class T>
__device__ __forceinline__ void load8(const T *p, int n, bool vec, float v[8]) {
    if (vec) {
        if constexpr (sizeof(T) == 4) {
            const float4 a = __ldcs(reinterpret_cast<const float4 *>(p)), b = __ldcs(reinterpret_cast<const float4 *>(p) + 1);
            v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
        } else {
            const uint4 a = __ldcs(reinterpret_cast<const uint4 *>(p));
            const uint32_t u[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const uint16_t lo = uint16_t(u[i] & 0xffff), hi = uint16_t(u[i] >> 16);
                v[2 * i] = to_f32(*reinterpret_cast<const T *>(&lo));
                v[2 * i + 1] = to_f32(*reinterpret_cast<const T *>(&hi));
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = i < n ? to_f32(p[i]) : 0.0f;
    }
}

template <class T>
__device__ __forceinline__ void store8(T *p, int n, bool vec, const float v[8]) {
    if (vec) {
        if constexpr (sizeof(T) == 4) {
            reinterpret_cast<float4 *>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
            reinterpret_cast<float4 *>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
        } else {
            *reinterpret_cast<uint4 *>(p) =
                make_uint4(pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]), pack2<T>(v[4], v[5]), pack2<T>(v[6], v[7]));
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++)
            if (i < n) p[i] = from_f32<T>(v[i]);
    }
}

// |v| as bits: as integers they order as the magnitudes do, infinity above
// every number and NaN above infinity, so a NaN is never lost.
__device__ __forceinline__ uint32_t mag(float v) { return __float_as_uint(v) & 0x7fffffffu; }

// TPR threads a row, CH chunks of 8 channels a thread. Rows narrower than a
// warp's reach share a block of 128 threads, four rows to it.
template <class T, int TPR, int CH, bool VEC>
__global__ void __launch_bounds__(TPR < 128 ? 128 : TPR) rms_norm_kernel(const __grid_constant__ RmsArgs a) {
    constexpr int THREADS = TPR < 128 ? 128 : TPR, ROWS = THREADS / TPR, WARPS = TPR / 32;
    __shared__ float part[WARPS];
    __shared__ uint32_t peak[WARPS];
    const int t = threadIdx.x % TPR, lane = threadIdx.x & 31, warp = t / 32;
    for (int64_t row0 = int64_t(blockIdx.x) * ROWS; row0 < a.rows; row0 += int64_t(gridDim.x) * ROWS) {
        const int64_t row = row0 + threadIdx.x / TPR;
        const bool live = row < a.rows;
        float s[CH][8], square = 0.0f;
        const T *x = static_cast<const T *>(a.x) + row * a.x_row, *r = static_cast<const T *>(a.r) + row * a.r_row;
        T *sum = static_cast<T *>(a.sum) + row * a.sum_row;
#pragma unroll
        for (int c = 0; c < CH; c++) {
            const int at = (c * TPR + t) * 8, n = live ? min(8, a.channels - at) : 0;
            const bool vec = VEC && n == 8;
            if (n > 0) {
                load8<T>(x + at, n, vec, s[c]);
                if (a.r) {
                    float v[8];
                    load8<T>(r + at, n, vec, v);
#pragma unroll
                    for (int i = 0; i < 8; i++) s[c][i] += v[i];
                }
            } else {
#pragma unroll
                for (int i = 0; i < 8; i++) s[c][i] = 0.0f;
            }
        }
#pragma unroll
        for (int c = 0; c < CH; c++) {
            const int at = (c * TPR + t) * 8, n = live ? min(8, a.channels - at) : 0;
            if (a.sum && n > 0) store8<T>(sum + at, n, VEC && n == 8, s[c]);
#pragma unroll
            for (int i = 0; i < 8; i++) square = fmaf(s[c][i], s[c][i], square);
        }
#pragma unroll
        for (int d = 16; d; d >>= 1) square += __shfl_xor_sync(0xffffffffu, square, d);
        if constexpr (WARPS > 1) {
            __syncthreads();  // the row before is done with part and peak
            if (lane == 0) part[warp] = square;
            __syncthreads();
            square = 0.0f;
#pragma unroll
            for (int w = 0; w < WARPS; w++) square += part[w];
        }
        const float inv = 1.0f / sqrtf(square / float(a.channels) + a.eps);
        uint32_t top[CH], all = 0;
#pragma unroll
        for (int c = 0; c < CH; c++) {
            const int at = (c * TPR + t) * 8;
            top[c] = 0;
#pragma unroll
            for (int i = 0; i < 8; i++) {
                s[c][i] = at + i < a.channels ? s[c][i] * inv * __ldg(a.gamma + at + i) : 0.0f;
                top[c] = max(top[c], mag(s[c][i]));
            }
            all = max(all, top[c]);
        }
        float *scales = a.scales + row * a.groups;
        if (a.group == 0) {
            all = __reduce_max_sync(0xffffffffu, all);
            if constexpr (WARPS > 1) {
                if (lane == 0) peak[warp] = all;
                __syncthreads();
                all = 0;
#pragma unroll
                for (int w = 0; w < WARPS; w++) all = max(all, peak[w]);
            }
            if (live && t == 0) scales[0] = __uint_as_float(all) / 448.0f;
#pragma unroll
            for (int c = 0; c < CH; c++) top[c] = all;
        } else {
            // a group of 32, 64 or 128 channels is 4, 8 or 16 neighbouring lanes' chunks
#pragma unroll
            for (int c = 0; c < CH; c++) {
                top[c] = max(top[c], __shfl_xor_sync(0xffffffffu, top[c], 1));
                top[c] = max(top[c], __shfl_xor_sync(0xffffffffu, top[c], 2));
                if (a.group > 32) top[c] = max(top[c], __shfl_xor_sync(0xffffffffu, top[c], 4));
                if (a.group > 64) top[c] = max(top[c], __shfl_xor_sync(0xffffffffu, top[c], 8));
                const int at = (c * TPR + t) * 8;
                if (live && at < a.channels && at % a.group == 0) scales[at / a.group] = __uint_as_float(top[c]) / 448.0f;
            }
        }
        uint8_t *y = a.y + row * a.y_row;
#pragma unroll
        for (int c = 0; c < CH; c++) {
            const int at = (c * TPR + t) * 8, n = live ? min(8, a.channels - at) : 0;
            const float scale = __uint_as_float(top[c]) / 448.0f;
            uint32_t packed[2] = {0, 0};
#pragma unroll
            for (int i = 0; i < 8; i++) {
                // a scale of zero (all zeros, or too small for f32): zeros
                const float v = scale == 0.0f ? 0.0f : s[c][i] / scale;
                packed[i / 4] |= uint32_t(__nv_cvt_float_to_fp8(v, __NV_SATFINITE, __NV_E4M3)) << (8 * (i % 4));
            }
            if (VEC && n == 8) {
                *reinterpret_cast<uint2 *>(y + at) = make_uint2(packed[0], packed[1]);
            } else {
#pragma unroll
                for (int i = 0; i < 8; i++)
                    if (i < n) y[at + i] = uint8_t(packed[i / 4] >> (8 * (i % 4)));
            }
        }
    }
}

template <class T, int TPR, int CH, bool VEC>
cudaError_t start(const RmsArgs &a, cudaStream_t stream) {
    constexpr int THREADS = TPR < 128 ? 128 : TPR, ROWS = THREADS / TPR;
    const int64_t want = (a.rows + ROWS - 1) / ROWS, most = int64_t(sm_count()) * (2048 / THREADS);
    rms_norm_kernel<T, TPR, CH, VEC><<<unsigned(want < most ? want : most), THREADS, 0, stream>>>(a);
    return cudaGetLastError();
}

template <class T, bool VEC>
cudaError_t start_c(const RmsArgs &a, cudaStream_t stream) {
    // two chunks a thread where the row allows it, four only past 1024 threads
    const int chunks = (a.channels + 7) / 8;
    if (chunks <= 32) return start<T, 32, 1, VEC>(a, stream);
    if (chunks <= 64) return start<T, 32, 2, VEC>(a, stream);
    if (chunks <= 256) return start<T, 128, 2, VEC>(a, stream);
    if (chunks <= 512) return start<T, 256, 2, VEC>(a, stream);
    if (chunks <= 1024) return start<T, 512, 2, VEC>(a, stream);
    if (chunks <= 2048) return start<T, 1024, 2, VEC>(a, stream);
    return start<T, 1024, 4, VEC>(a, stream);
}

template <class T>
cudaError_t start_t(const RmsArgs &a, bool vec, cudaStream_t stream) {
    return vec ? start_c<T, true>(a, stream) : start_c<T, false>(a, stream);
}

}  // namespace

}  // namespace ppocr

using namespace ppocr;

extern "C" int ppocr_rms_norm_e4m3(const ppocr_rms_norm_shape *s, const void *x, const void *residual,
                                   const float *gamma, void *sum, uint8_t *y, float *scales, void *stream) {
    static const char *me = "ppocr_rms_norm_e4m3";
    clear_error();
    if (!s) return refuse(PPOCR_E_ARG, me, "null shape");
    if (s->type != PPOCR_F32 && s->type != PPOCR_F16 && s->type != PPOCR_BF16)
        return refuse(PPOCR_E_ARG, me, "type must be PPOCR_F32, PPOCR_F16 or PPOCR_BF16");
    if (s->group != 0 && s->group != 32 && s->group != 64 && s->group != 128)
        return refuse(PPOCR_E_ARG, me, "group must be 0 (a row), 32, 64 or 128");
    if (!(s->eps >= 0.0f) || !std::isfinite(s->eps)) return refuse(PPOCR_E_ARG, me, "eps must be finite and not negative");
    if (!s->channels || s->channels > 32768) return refuse(PPOCR_E_SIZE, me, "channels must be between 1 and 32768");
    const uint64_t most = uint64_t(1) << 32, c = s->channels;
    if (s->rows > most || s->x_row > most || s->residual_row > most || s->sum_row > most || s->y_row > most)
        return refuse(PPOCR_E_SIZE, me, "more than 2^32 rows, or a stride above 2^32 elements");
    if (!s->rows) return PPOCR_OK;
    if (!x || !gamma || !y || !scales) return refuse(PPOCR_E_ARG, me, "null buffer");
    const size_t size = type_size(s->type);
    if (!aligned(x, size) || !aligned(residual, size) || !aligned(sum, size) || !aligned(gamma, 4) || !aligned(scales, 4))
        return refuse(PPOCR_E_ARG, me, "a buffer is not aligned to its type");
    RmsArgs a{};
    a.x = x, a.r = residual, a.gamma = gamma, a.sum = sum, a.y = y, a.scales = scales;
    a.rows = int64_t(s->rows);
    a.x_row = int64_t(s->x_row ? s->x_row : c), a.r_row = int64_t(s->residual_row ? s->residual_row : c);
    a.sum_row = int64_t(s->sum_row ? s->sum_row : c), a.y_row = int64_t(s->y_row ? s->y_row : c);
    if (s->rows > 1 && (a.sum_row < int64_t(c) || a.y_row < int64_t(c)))
        return refuse(PPOCR_E_ARG, me, "output rows overlap");
    a.channels = int(c), a.group = int(s->group), a.groups = s->group ? int((c + s->group - 1) / s->group) : 1;
    a.eps = s->eps;
    // outputs may meet the inputs only as x or residual updated in place
    const auto span = [&](int64_t row) { return (s->rows - 1) * uint64_t(row) + c; };
    const uint64_t xn = span(a.x_row) * size, rn = residual ? span(a.r_row) * size : 0, sn = sum ? span(a.sum_row) * size : 0;
    const uint64_t yn = span(a.y_row), gn = c * 4, cn = s->rows * uint64_t(a.groups) * 4;
    const bool over_x = overlap(sum, sn, x, xn) && !(sum == x && a.sum_row == a.x_row);
    const bool over_r = overlap(sum, sn, residual, rn) && !(sum == residual && a.sum_row == a.r_row);
    if (over_x || over_r || overlap(sum, sn, gamma, gn) || overlap(sum, sn, y, yn) || overlap(sum, sn, scales, cn) ||
        overlap(y, yn, x, xn) || overlap(y, yn, residual, rn) || overlap(y, yn, gamma, gn) || overlap(y, yn, scales, cn) ||
        overlap(scales, cn, x, xn) || overlap(scales, cn, residual, rn) || overlap(scales, cn, gamma, gn))
        return refuse(PPOCR_E_ARG, me, "an output overlaps another buffer");
    const auto wide = [&](const void *p, int64_t row) { return !p || (aligned(p, 16) && uint64_t(row) * size % 16 == 0); };
    const bool vec = wide(x, a.x_row) && wide(residual, a.r_row) && wide(sum, a.sum_row) && aligned(y, 8) && a.y_row % 8 == 0;
    const auto str = static_cast<cudaStream_t>(stream);
    const cudaError_t e = s->type == PPOCR_F32   ? start_t<float>(a, vec, str)
                          : s->type == PPOCR_F16 ? start_t<__half>(a, vec, str)
                                                 : start_t<__nv_bfloat16>(a, vec, str);
    return e == cudaSuccess ? int(PPOCR_OK) : refuse(PPOCR_E_DEVICE, me, cudaGetErrorString(e));
}
