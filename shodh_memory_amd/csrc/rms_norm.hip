// rms_norm.hip -- root-mean-square norm with the residual's addition, and its output in 8 bits with scales.
//
//   h = x + residual            (f32; written back rounded to the tensors' type: the residual stream of the next layer)
//   y = h / sqrt(mean(h^2) + eps) * weight                                     (f32; written rounded, if asked for)
//   s = max |y| / 127 or / 448, q = round_to_nearest_even(y / s) per row or per group of a row, as int8 or e4m3 (if asked for)
//
// One pass over the data: a row stays in the registers of the 64, 256 or 1024 threads that own it (8 neighbouring values a thread and step),
// so x and residual are read once and everything else is written from registers. A group of 32 .. 256 values lies in 4 .. 32 neighbouring
// lanes of one wave: its maximum is a few lane exchanges and no barrier. Bound: HBM for many rows (32768 x 4096 bf16 with residual, sum and e4m3:
// 944 MB in 155 us, 6.1 TB/s), one launch for few (one row of 384: 3 us on the device).
// Sums and statistics are f32. h^2 passes f32's range when |h| is over 2^63 or so (bf16 and f32 hold such values): that row is summed again
// with h scaled by 2^-96, which loses nothing that counts next to the value that overflowed.
#include "layers.h"

#pragma clang fp contract(off)

namespace shodh {

struct RmsArgs {
    const void *x, *residual, *weight;
    void *sum, *y, *q;
    float *scale;
    uint64_t rows, x_stride, residual_stride, sum_stride, y_stride, q_stride;
    uint32_t dim, group_lanes /* lanes of 8 values per group; 0 = the scale of a whole row */, groups;
    uint32_t weight_f32, q_dtype /* 0 = none */;
    float eps;
};

typedef uint32_t u32x4_any __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t u32x2_any __attribute__((ext_vector_type(2), aligned(1)));

// 8 values (n of them at a row's end). STREAM: past the caches, for data that is larger than they are.
template <bool STREAM, class T>
__device__ __forceinline__ void load8(float (&v)[8], const T *p, uint32_t n) {
    T t[8];
    if (n >= 8) {
        if constexpr (STREAM) {
#pragma unroll
            for (int k = 0; k < (int)sizeof(T) / 2; ++k) {
                const u32x4_any w = __builtin_nontemporal_load(reinterpret_cast<const u32x4_any *>(p) + k);
                __builtin_memcpy(t + 16 / sizeof(T) * k, &w, 16);
            }
        } else load_any(t, p);
    } else
        for (int i = 0; i < 8; ++i) t[i] = (uint32_t)i < n ? p[i] : (T)0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = (float)t[i];
}
template <bool STREAM, class T>
__device__ __forceinline__ void store8(T *p, const float (&v)[8], uint32_t n) {
    T t[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) t[i] = (T)v[i];
    if (n >= 8) {
        if constexpr (STREAM) {
#pragma unroll
            for (int k = 0; k < (int)sizeof(T) / 2; ++k) {
                u32x4_any w;
                __builtin_memcpy(&w, t + 16 / sizeof(T) * k, 16);
                __builtin_nontemporal_store(w, reinterpret_cast<u32x4_any *>(p) + k);
            }
        } else store_any(p, t);
    } else
        for (int i = 0; i < 8; ++i) if ((uint32_t)i < n) p[i] = t[i];
}

__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
    return v;
}
__device__ __forceinline__ uint32_t wave_max(uint32_t v, int lanes) {
    for (int o = 1; o < lanes; o <<= 1) v = max(v, (uint32_t)__shfl_xor((int)v, o));
    return v;
}

// TPR threads own a row of at most TPR * 8 * C values; a workgroup of max(TPR, 256) threads holds 256 / TPR rows (TPR = 64) or one.
template <class T, int TPR, int C, bool STREAM>
__global__ __launch_bounds__(TPR < 256 ? 256 : TPR) void rms_norm_kernel(const RmsArgs a) {
    constexpr int WAVES = TPR / 64, ROWS = TPR < 256 ? 256 / TPR : 1;
    __shared__ float part[2][WAVES];
    __shared__ uint32_t part_max[2][WAVES];
    constexpr bool HELD = C * TPR < 4096;       // the weights wait in registers for the row's sum; of the longest rows there is no room for them
                                                // (8192 x 32768 bf16 380 -> 354 us)
    const int t = threadIdx.x % TPR, wave = t >> 6;
    float w[HELD ? C : 1][8];
    uint32_t left[C];           // values of the row from this thread's place on: 8 or more where a step is whole
    auto weight = [&](int c, float (&v)[8]) {
        if (a.weight_f32) load8<false>(v, (const float *)a.weight + (c * TPR + t) * 8, left[c]);
        else load8<false>(v, (const T *)a.weight + (c * TPR + t) * 8, left[c]);
    };
#pragma unroll
    for (int c = 0; c < C; ++c) {
        const uint32_t at = (uint32_t)(c * TPR + t) * 8;
        left[c] = at < a.dim ? a.dim - at : 0;
        if constexpr (HELD) weight(c, w[c]);
    }
    auto row_sum = [&](float v, int slot) -> float {
        v = wave_sum(v);
        if constexpr (WAVES > 1) {
            if ((t & 63) == 0) part[slot][wave] = v;
            __syncthreads();
            v = 0.0f;
#pragma unroll
            for (int i = 0; i < WAVES; ++i) v += part[slot][i];
        }
        return v;
    };
    int slot = 0;
    for (uint64_t row = (uint64_t)blockIdx.x * ROWS + threadIdx.x / TPR; row < a.rows; row += (uint64_t)gridDim.x * ROWS) {
        float h[C][8];
        float ss = 0.0f;
#pragma unroll
        for (int c = 0; c < C; ++c) load8<STREAM>(h[c], (const T *)a.x + row * a.x_stride + (c * TPR + t) * 8, left[c]);
        if (a.residual) {
#pragma unroll
            for (int c = 0; c < C; ++c) {
                float r[8];
                load8<STREAM>(r, (const T *)a.residual + row * a.residual_stride + (c * TPR + t) * 8, left[c]);
#pragma unroll
                for (int i = 0; i < 8; ++i) h[c][i] += r[i];
            }
        }
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
            for (int i = 0; i < 8; ++i) ss = __builtin_fmaf(h[c][i], h[c][i], ss);
        if (a.sum)
#pragma unroll
            for (int c = 0; c < C; ++c) store8<STREAM>((T *)a.sum + row * a.sum_stride + (c * TPR + t) * 8, h[c], left[c]);
        ss = row_sum(ss, slot);
        slot ^= 1;
        float eps = a.eps;
        if (!(ss < __builtin_inff())) {        // the whole row takes this branch (every thread holds the same sum)
            ss = 0.0f;
#pragma unroll
            for (int c = 0; c < C; ++c)
#pragma unroll
                for (int i = 0; i < 8; ++i) { h[c][i] *= 0x1p-96f; ss = __builtin_fmaf(h[c][i], h[c][i], ss); }
            eps = 0.0f;                        // 2^-192 eps: nothing next to a mean that is over 2^-100 here
            ss = row_sum(ss, slot);
            slot ^= 1;
        }
        const float rstd = 1.0f / __builtin_sqrtf(ss / (float)a.dim + eps);
#pragma unroll
        for (int c = 0; c < C; ++c) {
            if constexpr (!HELD) weight(c, w[0]);
#pragma unroll
            for (int i = 0; i < 8; ++i) h[c][i] = h[c][i] * rstd * w[HELD ? c : 0][i];
        }
        if (a.y)
#pragma unroll
            for (int c = 0; c < C; ++c) store8<STREAM>((T *)a.y + row * a.y_stride + (c * TPR + t) * 8, h[c], left[c]);
        if (a.q_dtype) {
            // |y| as bits: for magnitudes the order of unsigned integers is that of the numbers, with infinity and then NaN above all of them
            uint32_t m[C];
#pragma unroll
            for (int c = 0; c < C; ++c) {
                m[c] = 0;
#pragma unroll
                for (int i = 0; i < 8; ++i) m[c] = max(m[c], __float_as_uint(h[c][i]) & 0x7FFFFFFFu);       // (0 behind the row's end)
            }
            if (a.group_lanes) {
#pragma unroll
                for (int c = 0; c < C; ++c) m[c] = wave_max(m[c], a.group_lanes);
            } else {
#pragma unroll
                for (int c = 1; c < C; ++c) m[0] = max(m[0], m[c]);
                m[0] = wave_max(m[0], 64);
                if constexpr (WAVES > 1) {
                    if ((t & 63) == 0) part_max[slot][wave] = m[0];
                    __syncthreads();
#pragma unroll
                    for (int i = 0; i < WAVES; ++i) m[0] = max(m[0], part_max[slot][i]);
                }
#pragma unroll
                for (int c = 1; c < C; ++c) m[c] = m[0];
            }
            const float top = a.q_dtype == SHODH_DTYPE_INT8 ? 127.0f : 448.0f;
#pragma unroll
            for (int c = 0; c < C; ++c) {
                const uint32_t at = (uint32_t)(c * TPR + t) * 8;
                if (at >= a.dim) continue;
                const float amax = __uint_as_float(m[c]);
                // a group with a NaN or an infinity reads as NaN throughout; one below 2^-100 as zeros (448 / amax would pass f32's range)
                const bool bad = m[c] >= 0x7F800000u, none = amax < 0x1p-100f;
                const float scale = bad ? __builtin_nanf("") : none ? 0.0f : amax / top, inv = bad || none ? 0.0f : top / amax;
                if (a.group_lanes ? (t & (a.group_lanes - 1)) == 0 : t == 0 && c == 0)
                    a.scale[row * a.groups + (a.group_lanes ? (uint32_t)(c * TPR + t) / a.group_lanes : 0)] = scale;
                float v[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] = bad ? 0.0f : fminf(fmaxf(h[c][i] * inv, -top), top);
                uint8_t b[8];
                if (a.q_dtype == SHODH_DTYPE_INT8) {
#pragma unroll
                    for (int i = 0; i < 8; ++i) b[i] = (uint8_t)(int8_t)(int)__builtin_rintf(v[i]);
                } else {
                    int lo = 0, hi = 0;
                    lo = __builtin_amdgcn_cvt_pk_fp8_f32(v[0], v[1], lo, false);
                    lo = __builtin_amdgcn_cvt_pk_fp8_f32(v[2], v[3], lo, true);
                    hi = __builtin_amdgcn_cvt_pk_fp8_f32(v[4], v[5], hi, false);
                    hi = __builtin_amdgcn_cvt_pk_fp8_f32(v[6], v[7], hi, true);
                    __builtin_memcpy(b, &lo, 4);
                    __builtin_memcpy(b + 4, &hi, 4);
                }
                uint8_t *dst = (uint8_t *)a.q + row * a.q_stride + at;
                if (left[c] >= 8) {
                    if constexpr (STREAM) {
                        u32x2_any w;
                        __builtin_memcpy(&w, b, 8);
                        __builtin_nontemporal_store(w, reinterpret_cast<u32x2_any *>(dst));
                    } else store_any(dst, b);
                } else
                    for (int i = 0; i < 8; ++i) if ((uint32_t)i < left[c]) dst[i] = b[i];
            }
        }
    }
}

template <class T, bool STREAM>
static int launch_rms(const RmsArgs &a, hipStream_t st) {
    // one workgroup for every one or four rows: its neighbours on the CU hide its waits (a loop over rows with the weights kept: 213 instead of 198 us
    // for 32768 x 4096 bf16 with residual, sum and e4m3)
    auto go = [&](auto kern, int threads, int rows_per_wg) {
        const uint64_t wgs = ceil_div(a.rows, rows_per_wg), most = (1u << 31) / threads;        // (a launch has fewer than 2^32 threads; further rows in turns)
        hipLaunchKernelGGL(kern, dim3((uint32_t)(wgs < most ? wgs : most)), dim3(threads), 0, st, a);
    };
    if (a.dim <= 512) go(rms_norm_kernel<T, 64, 1, STREAM>, 256, 4);
    else if (a.dim <= 1024) go(rms_norm_kernel<T, 64, 2, STREAM>, 256, 4);
    else if (a.dim <= 2048) go(rms_norm_kernel<T, 256, 1, STREAM>, 256, 1);
    else if (a.dim <= 4096) go(rms_norm_kernel<T, 256, 2, STREAM>, 256, 1);
    else if (a.dim <= 8192) go(rms_norm_kernel<T, 256, 4, STREAM>, 256, 1);
    else if (a.dim <= 16384) go(rms_norm_kernel<T, 1024, 2, STREAM>, 1024, 1);
    else go(rms_norm_kernel<T, 1024, 4, STREAM>, 1024, 1);
    SHODH_HIP_TRY(hipGetLastError());
    return SHODH_OK;
}

int compute_units(int device) {
    static int known[64];       // (a race writes the same number twice)
    if (device >= 0 && device < 64 && known[device]) return known[device];
    int n = 0;
    if (hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, device) != hipSuccess || n <= 0) n = 256;
    if (device >= 0 && device < 64) known[device] = n;
    return n;
}

}  // namespace shodh

using namespace shodh;

extern "C" {

void shodh_rms_norm_cfg_default(shodh_rms_norm_cfg *cfg) {
    if (!cfg) return;
    memset(cfg, 0, sizeof *cfg);
    cfg->dtype = cfg->weight_dtype = SHODH_DTYPE_BF16;
    cfg->q_dtype = SHODH_DTYPE_INT8;
    cfg->eps = 1e-6f;
}

int shodh_rms_norm_device(int device, const shodh_rms_norm_cfg *cfg, const void *d_x, const void *d_residual, const void *d_weight, void *d_sum, void *d_y,
                          void *d_q, float *d_scale, void *stream) {
    if (!cfg || !d_weight) { set_error("null argument"); return SHODH_ERR_INVALID; }
    if (!is_float_dtype(cfg->dtype)) { set_error("rms_norm: dtype %u is none of fp32, bf16, fp16", cfg->dtype); return SHODH_ERR_INVALID; }
    if (cfg->weight_dtype != SHODH_DTYPE_FP32 && cfg->weight_dtype != cfg->dtype) { set_error("rms_norm: the weight is fp32 or of x's type"); return SHODH_ERR_INVALID; }
    if (cfg->dim == 0 || cfg->dim > 32768) { set_error("rms_norm: dim %u is not in 1 .. 32768", cfg->dim); return cfg->dim ? SHODH_ERR_UNSUPPORTED : SHODH_ERR_INVALID; }
    if (!(cfg->eps >= 1e-30f) || cfg->eps > 3.0e38f) { set_error("rms_norm: eps has to be a number of 1e-30 or more"); return SHODH_ERR_INVALID; }
    if (cfg->rows == 0) return SHODH_OK;
    if ((d_q == nullptr) != (d_scale == nullptr)) { set_error("rms_norm: q and its scales come together"); return SHODH_ERR_INVALID; }
    if (!d_sum && !d_y && !d_q) { set_error("rms_norm: no output is asked for"); return SHODH_ERR_INVALID; }
    if (d_sum && !d_residual) { set_error("rms_norm: the sum is that of x and a residual: there is none"); return SHODH_ERR_INVALID; }
    if (d_q && cfg->q_dtype != SHODH_DTYPE_INT8 && cfg->q_dtype != SHODH_DTYPE_E4M3) { set_error("rms_norm: q_dtype %u is neither int8 nor e4m3", cfg->q_dtype); return SHODH_ERR_INVALID; }
    if (d_q && cfg->q_group != 0 && cfg->q_group != 32 && cfg->q_group != 64 && cfg->q_group != 128 && cfg->q_group != 256) {
        set_error("rms_norm: q_group %u is none of 0 (a row), 32, 64, 128, 256", cfg->q_group); return SHODH_ERR_UNSUPPORTED;
    }
    const uint64_t dim = cfg->dim;
    const uint64_t xs = cfg->x_stride ? cfg->x_stride : dim, rs = cfg->residual_stride ? cfg->residual_stride : dim, ss = cfg->sum_stride ? cfg->sum_stride : dim,
                   ys = cfg->y_stride ? cfg->y_stride : dim, qs = cfg->q_stride ? cfg->q_stride : dim;
    if (cfg->rows > 1 && (ss < dim || ys < dim || qs < dim)) { set_error("rms_norm: an output's rows overlap (stride below dim %u)", cfg->dim); return SHODH_ERR_INVALID; }
    const size_t b = dtype_bytes(cfg->dtype);
    if (!aligned_to(d_x, b) || !aligned_to(d_residual, b) || !aligned_to(d_sum, b) || !aligned_to(d_y, b) || !aligned_to(d_weight, dtype_bytes(cfg->weight_dtype)) || !aligned_to(d_scale, 4)) {
        set_error("rms_norm: a pointer is not a multiple of its element's size"); return SHODH_ERR_INVALID;
    }
    if (!d_x) { set_error("null argument"); return SHODH_ERR_INVALID; }
    const uint32_t groups = cfg->q_group ? (uint32_t)ceil_div(dim, cfg->q_group) : 1;
    {   // sum and y are written element for element by the threads that read x and residual there: in place, but not beside it
        const uint64_t n = cfg->rows;
        const Region x(d_x, dim * b, n, xs * b), res(d_residual, dim * b, n, rs * b), weight(d_weight, dim * dtype_bytes(cfg->weight_dtype)),
            out[4] = {Region(d_sum, dim * b, n, ss * b), Region(d_y, dim * b, n, ys * b), Region(d_q, dim, n, qs), Region(d_scale, groups * 4ull, n, groups * 4ull)};
        for (int i = 0; i < 4; ++i) {
            bool bad = may_overlap(out[i], weight);
            for (const Region *in : {&x, &res}) bad |= !(i < 2 && same_place(out[i], *in)) && may_overlap(out[i], *in);
            for (int j = 0; j < i; ++j) bad |= may_overlap(out[i], out[j]);
            if (bad) { set_error("rms_norm: %s overlaps another operand (sum and y may be x or residual themselves)", i == 0 ? "sum" : i == 1 ? "y" : i == 2 ? "q" : "scale"); return SHODH_ERR_INVALID; }
        }
    }
    DeviceScope scope;
    SHODH_TRY(scope.enter(device));
    RmsArgs a;
    a.x = d_x; a.residual = d_residual; a.weight = d_weight; a.sum = d_sum; a.y = d_y; a.q = d_q; a.scale = d_scale;
    a.rows = cfg->rows; a.x_stride = xs; a.residual_stride = rs; a.sum_stride = ss; a.y_stride = ys; a.q_stride = qs;
    a.dim = cfg->dim; a.group_lanes = cfg->q_group / 8; a.groups = groups;
    a.weight_f32 = cfg->weight_dtype == SHODH_DTYPE_FP32; a.q_dtype = d_q ? cfg->q_dtype : 0; a.eps = cfg->eps;
    hipStream_t st = (hipStream_t)stream;
    // 16-bit types, whole 16-byte pieces: past the caches from 256 MiB on, the size of the last level (what is written does not stay there anyway).
    // With residual, sum and e4m3, us through / past them: 65536 x 1024 bf16 102 / 79, 16384 x 4096 102 / 80, 32768 x 4096 198 / 155; f32 65536 x 1024
    // 163 / 168; rows of 771, 16384 of them, 24.5 / 26.7.
    const uint64_t each = b * (1 + (d_residual ? 1 : 0) + (d_sum ? 1 : 0) + (d_y ? 1 : 0)) + (d_q ? 1 : 0);
    const bool past = cfg->rows * dim * each > (256ull << 20) && ((dim | xs | rs | ss | ys | qs) & 7) == 0;
    if (cfg->dtype == SHODH_DTYPE_FP32) return launch_rms<float, false>(a, st);
    if (cfg->dtype == SHODH_DTYPE_BF16) return past ? launch_rms<__bf16, true>(a, st) : launch_rms<__bf16, false>(a, st);
    return past ? launch_rms<_Float16, true>(a, st) : launch_rms<_Float16, false>(a, st);
}

}  // extern "C"
