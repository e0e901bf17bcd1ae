// layers.h -- what the layer operators on device data share (rms_norm.hip, dense_w4.hip, window_attention.hip): element types, loads of any
// alignment, and the two checks every entry point makes.
#pragma once
#include "common.h"

namespace shodh {

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef int32_t i32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// A vector of N elements at an address that is a multiple of one element only (odd row lengths, views into wider rows): global memory takes
// 16-byte accesses at any such address, so these compile to the same wide instructions as aligned ones.
template <class T, int N>
__device__ __forceinline__ void load_any(T (&dst)[N], const T *src) { __builtin_memcpy(dst, __builtin_assume_aligned(src, sizeof(T)), sizeof(T) * N); }
template <class T, int N>
__device__ __forceinline__ void store_any(T *dst, const T (&src)[N]) { __builtin_memcpy(__builtin_assume_aligned(dst, sizeof(T)), src, sizeof(T) * N); }

// Between a wave's stores to LDS and loads of what its other lanes stored: LDS serves a wave's accesses in their order, so only the compiler has to be held,
// which may move a lane's load over stores of its own that it knows to lie elsewhere.
__device__ __forceinline__ void wave_lds_order() { __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront", "local"); }

inline size_t dtype_bytes(uint32_t t) { return t == SHODH_DTYPE_FP32 ? 4 : t == SHODH_DTYPE_INT8 || t == SHODH_DTYPE_E4M3 ? 1 : 2; }
inline bool is_float_dtype(uint32_t t) { return t == SHODH_DTYPE_FP32 || t == SHODH_DTYPE_BF16 || t == SHODH_DTYPE_FP16; }
inline bool aligned_to(const void *p, size_t bytes) { return ((uintptr_t)p & (bytes - 1)) == 0; }

// The bytes of an operand: runs of `width` bytes, n[0] x n[1] of them at distances step[0] and step[1] (bytes). Null, or none of them: no bytes.
struct Region {
    const void *p;
    uint64_t width, n[2], step[2];
    Region(const void *p, uint64_t width, uint64_t n0 = 1, uint64_t step0 = 0, uint64_t n1 = 1, uint64_t step1 = 0) : p(p), width(width), n{n0, n1}, step{step0, step1} {}
    bool empty() const { return !p || !width || !n[0] || !n[1]; }
    // where the runs lie modulo m (0: not modulo anything), as a length from p on
    unsigned __int128 span(uint64_t m) const {
        unsigned __int128 s = width;
        for (int i = 0; i < 2; ++i)
            if (n[i] > 1 && (m == 0 || step[i] % m != 0)) s += (unsigned __int128)(n[i] - 1) * step[i];
        return s;
    }
};
inline bool same_place(const Region &a, const Region &b) {
    if (a.p != b.p || a.width != b.width) return false;
    for (int i = 0; i < 2; ++i)
        if (a.n[i] != b.n[i] || (a.n[i] > 1 && a.step[i] != b.step[i])) return false;
    return true;
}
// False only where the two have no byte in common: they lie one behind the other, or in different places of the rows (heads, tokens) of one buffer.
inline bool may_overlap(const Region &a, const Region &b) {
    if (a.empty() || b.empty()) return false;
    const uintptr_t x = (uintptr_t)a.p, y = (uintptr_t)b.p;
    if (x + a.span(0) <= y || y + b.span(0) <= x) return false;
    for (const Region *r : {&a, &b})
        for (int i = 0; i < 2; ++i) {
            const uint64_t m = r->n[i] > 1 ? r->step[i] : 0;
            if (m == 0 || a.span(m) > m || b.span(m) > m) continue;
            const uint64_t apart = y >= x ? (uint64_t)(y - x) % m : (m - (uint64_t)(x - y) % m) % m;
            if (apart >= a.span(m) && apart + b.span(m) <= m) return false;
        }
    return true;
}

// The calling thread's current device is the caller's (torch keeps its own idea of it): it is switched for the call and put back.
struct DeviceScope {
    int before = -1;
    bool changed = false;
    int enter(int device) {
        if (hipGetDevice(&before) != hipSuccess) { set_error("no HIP device: libshodh_hip has no CPU fallback"); return SHODH_ERR_DEVICE; }
        if (before == device) return SHODH_OK;
        if (hipSetDevice(device) != hipSuccess) { (void)hipGetLastError(); set_error("device %d not present", device); return SHODH_ERR_DEVICE; }
        changed = true;
        return SHODH_OK;
    }
    ~DeviceScope() { if (changed) (void)hipSetDevice(before); }
};

// Allocations and frees of calls that are not captured themselves: a capture of another thread neither refuses them nor is ended by them.
struct BesideCaptures {
    hipStreamCaptureMode mode = hipStreamCaptureModeRelaxed;
    BesideCaptures() { (void)hipThreadExchangeStreamCaptureMode(&mode); }
    ~BesideCaptures() { (void)hipThreadExchangeStreamCaptureMode(&mode); }
    BesideCaptures(const BesideCaptures &) = delete;
};
// ... and a stream of its own for a call on host data (work on the default stream ends a capture)
struct OwnStream {
    hipStream_t st = nullptr;
    int make() { SHODH_HIP_TRY(hipStreamCreateWithFlags(&st, hipStreamNonBlocking)); return SHODH_OK; }
    ~OwnStream() { if (st) { (void)hipStreamSynchronize(st); (void)hipStreamDestroy(st); } }
};

int compute_units(int device);      // of an existing device; asked once per device

}  // namespace shodh
