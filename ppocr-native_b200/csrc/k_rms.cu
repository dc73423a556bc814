// ppocr_rms_norm_e4m3: the residual's addition, the root-mean-square norm and
// its 8-bit output, one pass over the row.
//
//     s = x + r;  n = s * rsqrt(mean(s^2) + eps) * gamma
//     scale_g = max |n| over group g / 448;  y = e4m3(n / scale_g)
//
// A row lies in the registers of its threads (8 channels a chunk, up to
// four chunks a thread), so x and r are read once and nothing is read again: s
// leaves rounded to the type, the norm uses the f32 s. The sum of squares is kept
// in f32: lane sums, a shuffle tree, then the warps' sums in order (the same
// order every time), squares that leave its range in sums of scaled values; the next
// row's loads are out while a row is worked on, and a row costs one barrier. Bound
// by HBM bytes: 16 384 rows of 4096 in bf16, groups of 128: 83 us, 472 MB at 5.7 TB/s
// (0.86 of a plain copy's rate; 81 us without the test for squares out of range and
// what follows it, 184 without the loads ahead). Rows that no vector width divides are
// read an element at a time, 32 lanes side by side: 1009 rows of 1111 in f16 6.8 us
// (7.9 MB, 1.2 us of HBM); 4096 channels so read would take 284 us.
#include <cuda_fp8.h>

#include <cmath>
#include <type_traits>

#include "block.cuh"
#include "devmath.cuh"

namespace ppocr {

namespace {

struct RmsArgs {
    const void *x, *r;
    const float *gamma;
    void *sum;
    uint8_t *y;
    float *scales;
    int64_t rows, x_row, r_row, sum_row, y_row;
    int channels, group, group_log2, groups;
    float eps, inv_channels;
};

// A lane's 8 channels of one chunk as they lie in memory.
template <class T>
struct Eight {
    static constexpr int W = sizeof(T) == 4 ? 2 : 1;
    uint4 u[W];

    // from 8 consecutive channels at a 16-byte border
    __device__ __forceinline__ void load(const T *p) {
#pragma unroll
        for (int i = 0; i < W; i++) u[i] = __ldcs(reinterpret_cast<const uint4 *>(p) + i);
    }
    // from channels 32 apart, n of the run left from p on
    __device__ __forceinline__ void load_apart(const T *p, int n) {
        if constexpr (sizeof(T) == 4) {
            uint32_t *w = reinterpret_cast<uint32_t *>(u);
#pragma unroll
            for (int i = 0; i < 8; i++) w[i] = i * 32 < n ? __float_as_uint(p[i * 32]) : 0;
        } else {
            uint32_t *w = reinterpret_cast<uint32_t *>(u);
            const unsigned short *q = reinterpret_cast<const unsigned short *>(p);
            uint32_t h[8];
#pragma unroll
            for (int i = 0; i < 8; i++) h[i] = i * 32 < n ? q[i * 32] : 0;
#pragma unroll
            for (int i = 0; i < 4; i++) w[i] = h[2 * i] | h[2 * i + 1] << 16;
        }
    }
    __device__ __forceinline__ void get(float v[8]) const {
        const uint32_t *w = reinterpret_cast<const uint32_t *>(u);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            if constexpr (sizeof(T) == 4) {
                v[i] = __uint_as_float(w[i]);
                v[i + 4] = __uint_as_float(w[i + 4]);
            } else if constexpr (std::is_same<T, __half>::value) {
                const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(w + i));
                v[2 * i] = f.x, v[2 * i + 1] = f.y;
            } else {
                v[2 * i] = __uint_as_float(w[i] << 16);
                v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
            }
        }
    }
    __device__ __forceinline__ void put(const float v[8]) {
        uint32_t *w = reinterpret_cast<uint32_t *>(u);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            if constexpr (sizeof(T) == 4) {
                w[i] = __float_as_uint(v[i]);
                w[i + 4] = __float_as_uint(v[i + 4]);
            } else {
                w[i] = pack2<T>(v[2 * i], v[2 * i + 1]);
            }
        }
    }
    __device__ __forceinline__ void store(T *p) const {
#pragma unroll
        for (int i = 0; i < W; i++) reinterpret_cast<uint4 *>(p)[i] = u[i];
    }
    __device__ __forceinline__ void store_apart(T *p, int n) const {
        const uint32_t *w = reinterpret_cast<const uint32_t *>(u);
#pragma unroll
        for (int i = 0; i < 8; i++)
            if (i * 32 < n) {
                if constexpr (sizeof(T) == 4)
                    p[i * 32] = __uint_as_float(w[i]);
                else
                    reinterpret_cast<unsigned short *>(p)[i * 32] = (unsigned short)(w[i / 2] >> (16 * (i & 1)));
            }
    }
};

// The larger magnitude of three; a NaN is never lost, and as an integer lies
// above every other magnitude's bits.
__device__ __forceinline__ float peak3(float top, float a, float b) {
    float d;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(top), "f"(fabsf(a)), "f"(fabsf(b)));
    return d;
}
__device__ __forceinline__ float peak2(float a, float b) {
    float d;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
    return d;
}

// Two values as e4m3, the first in the low byte.
__device__ __forceinline__ uint32_t e4m3_pair(float lo, float hi) {
    return __nv_cvt_float2_to_fp8x2(make_float2(lo, hi), __NV_SATFINITE, __NV_E4M3);
}

// Factors that leave the squares of the largest f32 numbers, and of the least, in f32.
constexpr float BIG = 0x1p-75f, TINY = 0x1p90f;

// What the chunk's v = s * gamma are multiplied by for their 8 bits, from their
// group's peak magnitude of n = v * inv: inv * 448 / peak. Where that quotient
// leaves the quick division's range (or there is none: zeros, NaN), v becomes
// n first; a scale that f32 rounds to zero gives zeros.
__device__ __forceinline__ float steps_of(float peak, float inv, float v[8]) {
    if (peak > 1e-30f && peak < 1e37f) return __fdividef(448.0f, peak) * inv;
#pragma unroll
    for (int i = 0; i < 8; i++) v[i] *= inv;
    if (peak <= 1e-30f) return peak * (1.0f / 448.0f) == 0.0f ? 0.0f : fminf(1.0f / (peak * (1.0f / 448.0f)), 3e38f);
    return 448.0f / peak;
}

// TPR threads a row, CH chunks of 8 channels a thread. Rows narrower than a
// warp's reach share a block of 128 threads, four rows to it. A block walks
// rows gridDim apart and has the next row's loads in flight while it works
// on this one.
//
// The 8 bits are those of v = s * gamma over its own peak: the root-mean-square
// reaches the scale alone, so a row needs one barrier, for the sum of squares
// and (one scale a row) the peak together.
//
// VEC: a chunk is 8 consecutive channels, 16-byte loads; else (rows, strides
// or bases that 16 bytes do not divide) channels 32 apart, so that a warp's
// loads lie side by side.
//
// Threads an SM: 1024 (64 registers), fewer where a thread holds two chunks and more.
template <class T, int TPR, int CH, bool VEC>
constexpr int at_least = TPR == 1024 || CH == 1 ? 1024 / (TPR < 128 ? 128 : TPR)
                                                : (!VEC ? 512 : sizeof(T) == 4 ? 768 : TPR == 32 ? 896 : 1024) / (TPR < 128 ? 128 : TPR);

template <class T, int TPR, int CH, bool VEC>
__global__ void __launch_bounds__(TPR < 128 ? 128 : TPR, at_least<T, TPR, CH, VEC>) rms_norm_kernel(const __grid_constant__ RmsArgs a) {
    constexpr int THREADS = TPR < 128 ? 128 : TPR, ROWS = THREADS / TPR, WARPS = TPR / 32;
    // two rows' in turn: between two writes of one lies the other's barrier
    __shared__ float part[2][WARPS], peak[2][WARPS];
    __shared__ float3 wide[2][WARPS];  // where part is not a number
    const int t = threadIdx.x % TPR, lane = threadIdx.x & 31, warp = t / 32;
    const auto place = [&](int c) { return VEC ? (c * TPR + t) * 8 : (c * TPR + (t & ~31)) * 8 + lane; };
    const T *x = static_cast<const T *>(a.x), *r = static_cast<const T *>(a.r);
    Eight<T> nx[CH], nr[CH];
    const auto fetch = [&](int64_t row) {
        if (row >= a.rows) return;
        const T *xr = x + row * a.x_row, *rr = r + row * a.r_row;
#pragma unroll
        for (int c = 0; c < CH; c++) {
            const int at = place(c);
            if constexpr (VEC) {
                if (at < a.channels) {
                    nx[c].load(xr + at);
                    if (r) nr[c].load(rr + at);
                }
            } else {
                nx[c].load_apart(xr + at, a.channels - at);
                if (r) nr[c].load_apart(rr + at, a.channels - at);
            }
        }
    };
    int64_t row = int64_t(blockIdx.x) * ROWS + threadIdx.x / TPR;
    fetch(row);
    int turn = 0;
    for (int64_t row0 = int64_t(blockIdx.x) * ROWS; row0 < a.rows; row0 += int64_t(gridDim.x) * ROWS) {
        const int channels = row < a.rows ? a.channels : 0;  // of this row: none past the last
        float v[CH][8], top[CH][VEC ? 1 : 8];
        float2 square2 = make_float2(0.0f, 0.0f);
        T *sum = static_cast<T *>(a.sum) + row * a.sum_row;
#pragma unroll
        for (int c = 0; c < CH; c++) {
            const int at = place(c);
            if constexpr (VEC) top[c][0] = 0.0f;
            if (at < channels) {
                nx[c].get(v[c]);
                if (r) {
                    float w[8];
                    nr[c].get(w);
#pragma unroll
                    for (int i = 0; i < 8; i++) v[c][i] += w[i];
                }
                if (a.sum) {
                    Eight<T> e;
                    e.put(v[c]);
                    if constexpr (VEC)
                        e.store(sum + at);
                    else
                        e.store_apart(sum + at, channels - at);
                }
                float gamma[8];
                if constexpr (VEC) {
                    const float4 g0 = __ldg(reinterpret_cast<const float4 *>(a.gamma + at));
                    const float4 g1 = __ldg(reinterpret_cast<const float4 *>(a.gamma + at) + 1);
                    gamma[0] = g0.x, gamma[1] = g0.y, gamma[2] = g0.z, gamma[3] = g0.w;
                    gamma[4] = g1.x, gamma[5] = g1.y, gamma[6] = g1.z, gamma[7] = g1.w;
                } else {
#pragma unroll
                    for (int i = 0; i < 8; i++) gamma[i] = at + i * 32 < channels ? __ldg(a.gamma + at + i * 32) : 0.0f;
                }
#pragma unroll
                for (int i = 0; i < 8; i += 2) {
                    const float2 s = make_float2(v[c][i], v[c][i + 1]);
                    square2 = ffma2(s, s, square2);
                    v[c][i] *= gamma[i];
                    v[c][i + 1] *= gamma[i + 1];
                    if constexpr (VEC)
                        top[c][0] = peak3(top[c][0], v[c][i], v[c][i + 1]);
                    else
                        top[c][i] = fabsf(v[c][i]), top[c][i + 1] = fabsf(v[c][i + 1]);
                }
            } else {
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    v[c][i] = 0.0f;
                    if constexpr (!VEC) top[c][i] = 0.0f;
                }
            }
        }
        float square = square2.x + square2.y;
        // between 2^-80 and 2^100, or f32 may not hold this thread's squares (f16's lie between
        // 2^-48 and 2^34): then they are taken again, of values times BIG or TINY, and square is
        // not a number until the row's sum is made. Zeros have no squares to hold.
        float3 apart = make_float3(0.0f, 0.0f, 0.0f);  // sums of squares as they are, times BIG^2, times TINY^2
        const bool lost = place(0) < channels && __float_as_uint(square) - 0x17800000u >= 0x5A000000u;
        const bool far = !std::is_same<T, __half>::value && __any_sync(0xffffffffu, lost);
        if (far) {
            const float by = square < 1.0f ? TINY : BIG;
            float again = 0.0f;
#pragma unroll
            for (int c = 0; c < CH; c++) {
                if (!lost || place(c) >= channels) continue;
                float x8[8], r8[8];
                nx[c].get(x8);
                if (r) nr[c].get(r8);
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const float w = (r ? x8[i] + r8[i] : x8[i]) * by;
                    again = fmaf(w, w, again);
                }
            }
            apart = make_float3(lost ? 0.0f : square, square < 1.0f ? 0.0f : again, square < 1.0f ? again : 0.0f);
        }
        fetch(row + int64_t(gridDim.x) * ROWS);
        if (far) {
#pragma unroll
            for (int d = 16; d; d >>= 1) {
                apart.x += __shfl_xor_sync(0xffffffffu, apart.x, d);
                apart.y += __shfl_xor_sync(0xffffffffu, apart.y, d);
                apart.z += __shfl_xor_sync(0xffffffffu, apart.z, d);
            }
            square = apart.y != 0.0f || apart.z != 0.0f ? NAN : apart.x;
        } else {
#pragma unroll
            for (int d = 16; d; d >>= 1) square += __shfl_xor_sync(0xffffffffu, square, d);
            apart.x = square;
        }
        float all = 0.0f;
        if (a.group == 0) {
#pragma unroll
            for (int c = 0; c < CH; c++) {
                if constexpr (VEC)
                    all = peak2(all, top[c][0]);
                else
#pragma unroll
                    for (int i = 0; i < 8; i += 2) all = peak3(all, top[c][i], top[c][i + 1]);
            }
            all = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(all)));
        } else {
#pragma unroll
            for (int c = 0; c < CH; c++) {
                if constexpr (VEC) {
                    // a group of 32, 64 or 128 channels is 4, 8 or 16 neighbouring lanes' chunks
                    float &m = top[c][0];
                    m = peak2(m, __shfl_xor_sync(0xffffffffu, m, 1));
                    m = peak2(m, __shfl_xor_sync(0xffffffffu, m, 2));
                    if (a.group > 32) m = peak2(m, __shfl_xor_sync(0xffffffffu, m, 4));
                    if (a.group > 64) m = peak2(m, __shfl_xor_sync(0xffffffffu, m, 8));
                } else {
                    // 1, 2 or 4 of the warp's 32-channel runs
#pragma unroll
                    for (int i = 0; i < 8; i++) top[c][i] = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(top[c][i])));
#pragma unroll
                    for (int i = 0; i < 8; i += 2)
                        if (a.group > 32) top[c][i] = top[c][i + 1] = peak2(top[c][i], top[c][i + 1]);
#pragma unroll
                    for (int i = 0; i < 8; i += 4)
                        if (a.group > 64) top[c][i] = top[c][i + 1] = top[c][i + 2] = top[c][i + 3] = peak2(top[c][i], top[c][i + 2]);
                }
            }
        }
        if constexpr (WARPS > 1) {
            if (lane == 0) part[turn][warp] = square, peak[turn][warp] = all;
            if (lane == 0 && square != square) wide[turn][warp] = apart;
            __syncthreads();
            square = 0.0f;
#pragma unroll
            for (int w = 0; w < WARPS; w++) square += part[turn][w];
            if (a.group == 0) {
#pragma unroll
                for (int w = 0; w < WARPS; w++) all = peak2(all, peak[turn][w]);
            }
        }
        // by: an exact factor that brings values far from one nearer
        float mean = fmaf(square, a.inv_channels, a.eps), by = 1.0f;
        if (!(mean > 0x1p-80f && mean < 0x1p100f)) {
            // (a mean of zero or of no number goes through as it is)
            if constexpr (WARPS > 1) {
                // a warp's sums a lane: no loop here, which would end the wait for the loads in flight early
                apart = make_float3(0.0f, 0.0f, 0.0f);
                if (lane < WARPS) {
                    apart.x = part[turn][lane];
                    if (apart.x != apart.x) apart = wide[turn][lane];
                }
#pragma unroll
                for (int d = 16; d; d >>= 1) {
                    apart.x += __shfl_xor_sync(0xffffffffu, apart.x, d);
                    apart.y += __shfl_xor_sync(0xffffffffu, apart.y, d);
                    apart.z += __shfl_xor_sync(0xffffffffu, apart.z, d);
                }
            }
            mean = fmaf(fmaf(apart.z * (1 / TINY), 1 / TINY, apart.x), a.inv_channels, a.eps);
            if (apart.y != 0.0f) {
                by = BIG, mean = fmaf(fmaf(apart.x * BIG, BIG, apart.y), a.inv_channels, a.eps * BIG * BIG);
            } else if (mean < 0x1p-75f) {
                by = TINY, mean = fmaf(apart.x * a.inv_channels * TINY, TINY, apart.z * a.inv_channels) + a.eps * TINY * TINY;
            }
#pragma unroll
            for (int c = 0; c < CH; c++) {
#pragma unroll
                for (int i = 0; i < 8; i++) v[c][i] *= by;
#pragma unroll
                for (int i = 0; i < (VEC ? 1 : 8); i++) top[c][i] *= by;
            }
            all *= by;
        }
        turn ^= 1;
        const float inv = rsqrtf(mean);
        float *scales = a.scales + row * a.groups;
        uint8_t *y = a.y + row * a.y_row;
        if (a.group == 0 && channels && t == 0) scales[0] = all * inv * (1.0f / 448.0f);
#pragma unroll
        for (int c = 0; c < CH; c++) {
            const int at = place(c), n = channels - at;
            if (n <= 0) continue;
            if constexpr (VEC) {
                const float p = (a.group ? top[c][0] : all) * inv;
                if (a.group && (at & (a.group - 1)) == 0) scales[at >> a.group_log2] = p * (1.0f / 448.0f);
                const float f = steps_of(p, inv, v[c]);
                uint32_t w[2];
#pragma unroll
                for (int i = 0; i < 2; i++)
                    w[i] = e4m3_pair(v[c][4 * i] * f, v[c][4 * i + 1] * f) |
                           e4m3_pair(v[c][4 * i + 2] * f, v[c][4 * i + 3] * f) << 16;
                *reinterpret_cast<uint2 *>(y + at) = make_uint2(w[0], w[1]);
            } else {
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    if (i * 32 >= n) continue;
                    const float p = (a.group ? top[c][i] : all) * inv;
                    if (a.group && lane == 0 && ((at + i * 32) & (a.group - 1)) == 0) scales[(at + i * 32) >> a.group_log2] = p * (1.0f / 448.0f);
                    float one[8] = {v[c][i]};
                    const float f = steps_of(p, inv, one);
                    y[at + i * 32] = uint8_t(e4m3_pair(one[0] * f, 0.0f));
                }
            }
        }
        row += int64_t(gridDim.x) * ROWS;
    }
}

template <class T, int TPR, int CH, bool VEC>
cudaError_t start(const RmsArgs &a, cudaStream_t stream) {
    static_assert(TPR == 32 || TPR >= 128, "a row is one warp's or a whole block's");
    constexpr int THREADS = TPR < 128 ? 128 : TPR, ROWS = THREADS / TPR;
    // all blocks at once where a thread has little to fetch ahead, else twice as many
    // (bf16, 1024 channels: 42.6 us, 43.2 with twice as many; f32, 2048: 137 us, 164 with half)
    constexpr int AT_ONCE = sizeof(T) == 2 && CH == 1 && TPR > 32 ? 1024 : 2048;
    const int64_t want = (a.rows + ROWS - 1) / ROWS, most = int64_t(sm_count()) * (AT_ONCE / THREADS);
    rms_norm_kernel<T, TPR, CH, VEC><<<unsigned(want < most ? want : most), THREADS, 0, stream>>>(a);
    return cudaGetLastError();
}

template <class T, bool VEC>
cudaError_t start_c(const RmsArgs &a, cudaStream_t stream) {
    const int chunks = (a.channels + 7) / 8;
    if (chunks <= 32) return start<T, 32, 1, VEC>(a, stream);
    if (chunks <= 64) return start<T, 32, 2, VEC>(a, stream);
    if constexpr (sizeof(T) == 2) {
        // a chunk a thread up to 2048 channels, then two (bf16, 1024 and 2048 channels:
        // 41.0 and 79.3 us where two take 47.1 and 89.6; 4096 and 8192: 82.6 and 96.8
        // us where two take 79.3 and 85.5)
        if (chunks <= 128) return start<T, 128, 1, VEC>(a, stream);
        if (chunks <= 256) return start<T, 256, 1, VEC>(a, stream);
        if (chunks <= 512) return start<T, 256, 2, VEC>(a, stream);
        if (chunks <= 1024) return start<T, 512, 2, VEC>(a, stream);
    } else {
        // a chunk is 32 bytes: two a thread up to 4096 channels, then one as far as
        // threads go (f32, 2048 and 4096 channels: 137 and 141 us where one takes 141
        // and 157; 8192: 154 us where two take 177)
        if (chunks <= 256) return start<T, 128, 2, VEC>(a, stream);
        if (chunks <= 512) return start<T, 256, 2, VEC>(a, stream);
        if (chunks <= 1024) return start<T, 1024, 1, VEC>(a, stream);
    }
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
    a.group_log2 = s->group == 128 ? 7 : s->group == 64 ? 6 : 5;
    a.eps = s->eps, a.inv_channels = 1.0f / float(c);
    // outputs may meet the inputs only as x or residual updated in place
    const auto rows = [&](const void *p, int64_t row, uint64_t each, uint64_t bytes) {
        return Rows{p, p ? ((s->rows - 1) * uint64_t(row) + each) * bytes : 0, each * bytes, uint64_t(row) * bytes};
    };
    const Rows xs = rows(x, a.x_row, c, size), rs = rows(residual, a.r_row, c, size), ss = rows(sum, a.sum_row, c, size);
    const Rows ys = rows(y, a.y_row, c, 1), gs{gamma, c * 4, c * 4, 0}, cs = rows(scales, a.groups, uint64_t(a.groups), 4);
    const bool over_x = overlap(ss, xs) && !(sum == x && a.sum_row == a.x_row);
    const bool over_r = overlap(ss, rs) && !(sum == residual && a.sum_row == a.r_row);
    if (over_x || over_r || overlap(ss, gs) || overlap(ss, ys) || overlap(ss, cs) || overlap(ys, xs) || overlap(ys, rs) ||
        overlap(ys, gs) || overlap(ys, cs) || overlap(cs, xs) || overlap(cs, rs) || overlap(cs, gs))
        return refuse(PPOCR_E_ARG, me, "an output overlaps another buffer");
    if (const int bad = check_buffers(me, {x, residual, gamma, sum, y, scales})) return bad;
    const auto wide = [&](const void *p, int64_t row) { return !p || (aligned(p, 16) && uint64_t(row) * size % 16 == 0); };
    const bool vec = c % 8 == 0 && aligned(gamma, 16) && wide(x, a.x_row) && wide(residual, a.r_row) && wide(sum, a.sum_row) && aligned(y, 8) && a.y_row % 8 == 0;
    const auto str = static_cast<cudaStream_t>(stream);
    const cudaError_t e = s->type == PPOCR_F32   ? start_t<float>(a, vec, str)
                          : s->type == PPOCR_F16 ? start_t<__half>(a, vec, str)
                                                 : start_t<__nv_bfloat16>(a, vec, str);
    return e == cudaSuccess ? int(PPOCR_OK) : refuse(PPOCR_E_DEVICE, me, cudaGetErrorString(e));
}
