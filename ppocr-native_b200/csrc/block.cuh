// Shared pieces of the transformer-block operators (window attention, the
// 8-bit RMS norm, the 4-bit product): element types, warp-level matrix
// instructions, asynchronous copies, and the checks of their C entry points.
#pragma once

#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <atomic>
#include <cstdint>
#include <initializer_list>
#include <string>

#include "../../include/ppocr_cuda.h"
#include "async.cuh"

namespace ppocr {

void set_last_error(const std::string &msg);

namespace {

// ------------------------------------------------------------ host checks

// Records `what: why` and returns `code`; never throws across the C entry
// (a message that cannot be stored is dropped).
int refuse(int code, const char *what, const char *why) noexcept {
    try {
        set_last_error(std::string(what) + ": " + why);
    } catch (...) {
    }
    return code;
}

void clear_error() noexcept {
    try {
        set_last_error(std::string());
    } catch (...) {
    }
}

// 0 when every buffer (NULL ones aside) is memory that the current device's
// kernels may read and write as it is: this device's, managed, or page-locked
// host memory. Another device's and plain host memory would fault there.
// About 0.05 us a buffer. *local: whether all are this device's own memory.
int check_buffers(const char *what, std::initializer_list<const void *> buffers, bool *local = nullptr) noexcept {
    int here = 0;
    if (local) *local = true;
    cudaError_t e = cudaGetDevice(&here);
    for (const void *p : buffers) {
        if (!p || e != cudaSuccess) continue;
        cudaPointerAttributes at{};
        e = cudaPointerGetAttributes(&at, p);
        if (e == cudaErrorInvalidValue) {
            cudaGetLastError();
            return refuse(PPOCR_E_ARG, what, "a buffer is not device memory");
        }
        if (e != cudaSuccess) break;
        if (at.type == cudaMemoryTypeUnregistered) return refuse(PPOCR_E_ARG, what, "a buffer is not device memory");
        if (at.type == cudaMemoryTypeDevice && at.device != here)
            return refuse(PPOCR_E_ARG, what, "a buffer is another device's than the current one");
        if (local && at.type != cudaMemoryTypeDevice) *local = false;
    }
    if (e == cudaSuccess) return PPOCR_OK;
    cudaGetLastError();
    return refuse(PPOCR_E_DEVICE, what, cudaGetErrorString(e));
}

inline bool aligned(const void *p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

// The number of SMs of the current device (one query per device).
inline int sm_count() {
    static std::atomic<int> known[64];
    int d = 0;
    if (cudaGetDevice(&d) != cudaSuccess) return 148;
    if (d < 64 && known[d] > 0) return known[d];
    int n = 0;
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, d) != cudaSuccess || n < 1) n = 148;
    if (d < 64) known[d] = n;
    return n;
}

// Raises a kernel's dynamic shared-memory limit, once per device (a
// per-device bit remembers; a race only repeats the call).
template <auto KERNEL>
cudaError_t raise_shared(int bytes) {
    static std::atomic<uint64_t> done{0};
    int d = 0;
    cudaError_t e = cudaGetDevice(&d);
    if (e != cudaSuccess) return e;
    const uint64_t bit = d < 64 ? uint64_t(1) << d : 0;
    if (done.load(std::memory_order_relaxed) & bit) return cudaSuccess;
    e = cudaFuncSetAttribute(KERNEL, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e == cudaSuccess) done.fetch_or(bit, std::memory_order_relaxed);
    return e;
}

// The driver's tensor-map encoder (NULL where it has none).
using EncodeTiled = CUresult (*)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *,
                                 const cuuint64_t *, const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave,
                                 CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

inline EncodeTiled tensor_map_encoder() {
    static const EncodeTiled fn = [] {
        void *p = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &q) != cudaSuccess ||
            q != cudaDriverEntryPointSuccess)
            p = nullptr;
        return reinterpret_cast<EncodeTiled>(p);
    }();
    return fn;
}

inline size_t type_size(int type) { return type == PPOCR_F32 ? 4 : type == PPOCR_E4M3 ? 1 : 2; }

// True when the byte ranges [a, a + an) and [b, b + bn) meet.
inline bool overlap(const void *a, uint64_t an, const void *b, uint64_t bn) {
    const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
    return an && bn && x < y + bn && y < x + an;
}

// The bytes that rows of a tensor lie in: all of them, and each row's.
struct Rows {
    const void *p;
    uint64_t all, each, step;  // bytes from the first to the last; of a row; from row to row
};

// True when two tensors' elements may meet: their ranges do, unless rows of one step lie
// beside one another (columns of one buffer).
inline bool overlap(const Rows &a, const Rows &b) {
    if (!overlap(a.p, a.all, b.p, b.all)) return false;
    if (a.step != b.step || !a.step) return true;
    const uint64_t from = reinterpret_cast<uintptr_t>(b.p) - reinterpret_cast<uintptr_t>(a.p);
    const uint64_t off = b.p >= a.p ? from % a.step : (a.step - (0 - from) % a.step) % a.step;
    return off < a.each || off + b.each > a.step;
}

// ------------------------------------------------------------ device pieces

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }

template <class T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

template <class T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&h);
}
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&h);
}

// 2^x with the special-function unit (2 ulp; 0 for -inf).
__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ uint32_t shared_u32(const void *p) {
    return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}

// N bytes to shared memory, the last N - valid of them zeros.
template <int N>
__device__ __forceinline__ void copy_async(uint32_t dst, const void *src, int valid) {
    if constexpr (N == 16)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(valid) : "memory");
    else
        asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(dst), "l"(src), "n"(N), "r"(valid) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// A wait on an mbarrier's phase that ends by itself: a copy takes
// microseconds, and after two seconds the caller is told so (false).
__device__ __forceinline__ bool wait_copy(uint32_t bar, uint32_t parity) {
    if (try_wait(bar, parity)) return true;
    const unsigned long long t0 = global_ns();
    while (!try_wait_sleep(bar, parity, 20000u))
        if (global_ns() - t0 > 2000000000ull) return false;
    return true;
}

__device__ __forceinline__ void ldmatrix4(uint32_t r[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr));
}
__device__ __forceinline__ void ldmatrix4_t(uint32_t r[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr));
}

// c (16 x 8, f32) += a (16 x 16) * b (16 x 8), operands f16 or bf16.
template <class T>
__device__ __forceinline__ void mma16(float c[4], const uint32_t a[4], uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma16<__half>(float c[4], const uint32_t a[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma16<__nv_bfloat16>(float c[4], const uint32_t a[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// c (16 x 8, f32) += a (16 x 8) * b (8 x 8) in tf32.
__device__ __forceinline__ void mma8_tf32(float c[4], const uint32_t a[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// An f32 value as its tf32 neighbour (in whole-number steps: rounded to nearest,
// 19.6 us on the page lines' attention where cvt.rna took 23.2) and the exact
// remainder, of which the matrix instruction reads 11 bits: hi*hi + hi*lo + lo*hi
// loses about 2^-22 of a product. An infinity's remainder is NaN.
__device__ __forceinline__ void split_tf32(float x, uint32_t &hi, uint32_t &lo) {
    hi = (__float_as_uint(x) + 0x1000u) & 0xFFFFE000u;
    lo = __float_as_uint(x - __uint_as_float(hi));
}

}  // namespace

}  // namespace ppocr
