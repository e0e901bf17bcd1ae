// dense_w4.hip -- dense layers for few rows on 4-bit weights with group scales (and zero points).
//
//   y[m][n] = (sum_k x[m][k] * (q[n][k] - z[n][g]) * s[n][g]) * x_scale[m] + bias[n],   g = k / group, q and z in 0 .. 15
//
// Bound: the weights' bytes (half a byte a weight) for up to 16 rows; a launch for small layers; waits for 64 rows (28672 x 4096, bf16: 28 us, 65 MB at 2.3 TB/s:
// CUs are busy for 65 % of it -- 224 workgroups for 256 CUs, a barrier a block -- and in that the vector unit for 52 %, the matrix unit for 30 %). One fp16 row
// x 14336 x 4096: 8.8 us with the call where the last-level cache holds the 31 MB of weights, 10.3 (3.0 TB/s) where they come from HBM.
// Everything follows from that:
//  * weights are laid out once, in records of 16 outputs x 128 inputs (1 KiB of 4-bit numbers, 16 B a lane, then the record's scales and zero
//    points): a wave's load of a record is one contiguous KiB and lands where the matrix instruction wants it;
//  * a 4-bit number becomes a matrix operand with a shift and an and-or per PAIR: or-ed into the mantissa of 16.0 it reads as 16 + q, in bf16 as in
//    fp16, exactly. sum x (16 + q) - (16 + z) sum x is the group's sum; sum x comes from the same matrix instruction with ones for weights, in the same
//    order. int8 rows multiply q as a byte: sums exact in int32, (q - z) likewise;
//  * f32 rows are split into three bf16 parts (8 + 8 + 8 bits, by truncation, exact): three products with q - z itself, sums in f32. 16-bit rows with an f32
//    result are multiplied with q - z too;
//  * scales multiply the f32 sum of a group, so no weight is rounded to 16 bits on the way.
// A row of x that holds a NaN or an infinity gives NaN in all its outputs (16 x - 16 x; f32 parts x - x); 16-bit rows with an f32 result what x (q - z) gives.
#include "layers.h"

#include <cstddef>
#include <new>
#include <type_traits>
#include <vector>

#pragma clang fp contract(off)

struct shodh_w4_weight {
    int device = 0;
    uint32_t N = 0, K = 0, group = 0, scale_dtype = 0, zeros = 0, tiles = 0, blocks = 0, record = 0;
    uint8_t *data = nullptr;
};

namespace shodh {

constexpr int W4_TN = 16, W4_TK = 128;        // outputs and inputs of a record

static uint32_t record_bytes(uint32_t group, bool zeros) { return 1024u + (W4_TK / group) * (32u + (zeros ? 16u : 0u)); }

// ---- laying out -----------------------------------------------------------------------------------------------------------------
// Record: [lane 64][step 4] words; word (lane, step) holds inputs 32 step + 8 (lane >> 4) + e, e = 0 .. 7, of output lane & 15, element e in the 4 bits
// number (e >> 1) + 4 (e & 1): a shift by 4 i and a mask leave elements 2 i and 2 i + 1 in the two halves of the word. Then [group][16 outputs] scales of
// two bytes, then [group][16] bytes 16 + z.
template <class S>
__global__ __launch_bounds__(256) void w4_pack_kernel(const uint8_t *__restrict__ q, const float *__restrict__ scale, const uint8_t *__restrict__ zero, uint32_t N, uint32_t K,
                                                      uint32_t group, uint32_t blocks, uint32_t record, uint8_t *__restrict__ out, uint32_t *__restrict__ bad) {
    const uint32_t tile = blockIdx.y, block = blockIdx.x, t = threadIdx.x;
    uint8_t *rec = out + ((size_t)tile * blocks + block) * record;
    const uint32_t lane = t >> 2, step = t & 3, n = tile * W4_TN + (lane & 15), k0 = block * W4_TK + 32 * step + 8 * (lane >> 4);
    const size_t pitch = (K + 1) / 2;
    uint32_t word = 0;
    for (uint32_t e = 0; e < 8; ++e) {
        uint32_t v = 0;          // (behind the matrix: x reads as zero there, or the output is not written)
        if (n < N && k0 + e < K) { const uint32_t b = q[n * pitch + ((k0 + e) >> 1)]; v = ((k0 + e) & 1) ? b >> 4 : b & 15u; }
        word |= v << (4 * ((e >> 1) + 4 * (e & 1)));
    }
    reinterpret_cast<uint32_t *>(rec)[t] = word;
    const uint32_t per = W4_TK / group, groups = (K + group - 1) / group;
    if (t < per * 16) {
        const uint32_t gl = t >> 4, g = block * per + gl, m = tile * W4_TN + (t & 15);
        const bool in = m < N && g < groups;
        const float s = in ? scale[(size_t)m * groups + g] : 0.0f;
        const S r = (S)s;
        if (!(__builtin_fabsf((float)r) < __builtin_inff())) atomicOr(bad, 1u);
        else if (__builtin_fabsf((float)r - s) > __builtin_fabsf(s) * (std::is_same_v<S, _Float16> ? 0x1p-11f : 0x1p-8f)) atomicOr(bad, 8u);       // more than its half step: too small for S
        reinterpret_cast<S *>(rec + 1024)[t] = r;
        if (zero) {
            const uint32_t z = in ? zero[(size_t)m * groups + g] : 8u;
            if (z > 15u) atomicOr(bad, 2u);
            rec[1024 + per * 32 + t] = (uint8_t)(16u + (z & 15u));
        }
    }
}

// a group's scale and zero point from its floats (one wave a group), then its 4-bit numbers
template <class S>
__global__ __launch_bounds__(64) void w4_quantize_kernel(const float *__restrict__ w, uint32_t N, uint32_t K, uint32_t group, uint32_t zeros, uint8_t *__restrict__ q /* one a byte */,
                                                         float *__restrict__ scale, uint8_t *__restrict__ zero, uint32_t *__restrict__ bad) {
    const uint32_t groups = (K + group - 1) / group, g = blockIdx.x, n = blockIdx.y + gridDim.y * blockIdx.z;
    if (n >= N) return;
    const uint32_t k0 = g * group, k1 = min(K, k0 + group);
    float lo = 0.0f, hi = 0.0f;
    bool odd = false;
    for (uint32_t k = k0 + threadIdx.x; k < k1; k += 64) {
        const float v = w[(size_t)n * K + k];
        odd |= !(__builtin_fabsf(v) < __builtin_inff());
        lo = fminf(lo, v); hi = fmaxf(hi, v);
    }
    for (int o = 32; o > 0; o >>= 1) { lo = fminf(lo, __shfl_xor(lo, o)); hi = fmaxf(hi, __shfl_xor(hi, o)); }
    if (odd) atomicOr(bad, 4u);
    const float s = (float)(S)(zeros ? (hi - lo) / 15.0f : fmaxf(-lo, hi) / 7.0f);
    const bool none = !(s > 0.0f);
    const float z = zeros ? (none ? 0.0f : fminf(fmaxf(__builtin_rintf(-lo / s), 0.0f), 15.0f)) : 8.0f;
    for (uint32_t k = k0 + threadIdx.x; k < k1; k += 64) {
        const float v = none ? z : __builtin_rintf(w[(size_t)n * K + k] / s) + z;
        q[(size_t)n * K + k] = (uint8_t)(int)fminf(fmaxf(v, 0.0f), 15.0f);
    }
    if (threadIdx.x == 0) { scale[(size_t)n * groups + g] = s; if (zeros) zero[(size_t)n * groups + g] = (uint8_t)(int)z; }
}
__global__ __launch_bounds__(256) void w4_pairs_kernel(const uint8_t *__restrict__ q, uint32_t N, uint32_t K, uint8_t *__restrict__ out) {
    const size_t pitch = (K + 1) / 2, total = (size_t)N * pitch;
    for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (size_t)gridDim.x * 256) {
        const size_t n = i / pitch, k = (i - n * pitch) * 2;
        const uint32_t lo = q[n * K + k], hi = k + 1 < K ? q[n * K + k + 1] : 0u;
        out[i] = (uint8_t)(lo | (hi << 4));
    }
}
template <class S>
__global__ __launch_bounds__(256) void w4_unpack_kernel(const uint8_t *__restrict__ data, uint32_t N, uint32_t K, uint32_t group, uint32_t blocks, uint32_t record, uint32_t zeros,
                                                        float *__restrict__ out) {
    const uint32_t tile = blockIdx.y, block = blockIdx.x, t = threadIdx.x;
    const uint8_t *rec = data + ((size_t)tile * blocks + block) * record;
    const uint32_t lane = t >> 2, step = t & 3, n = tile * W4_TN + (lane & 15), kk = 32 * step + 8 * (lane >> 4), per = W4_TK / group;
    const uint32_t word = reinterpret_cast<const uint32_t *>(rec)[t];
    for (uint32_t e = 0; e < 8; ++e) {
        const uint32_t k = block * W4_TK + kk + e, g = (kk + e) / group;
        if (n >= N || k >= K) continue;
        const float v = (float)((word >> (4 * ((e >> 1) + 4 * (e & 1)))) & 15u);
        const float z = zeros ? (float)rec[1024 + per * 32 + g * 16 + (n & 15)] - 16.0f : 8.0f;
        out[(size_t)n * K + k] = (v - z) * (float)reinterpret_cast<const S *>(rec + 1024)[g * 16 + (n & 15)];
    }
}

// ---- the product ------------------------------------------------------------------------------------------------------------------
struct W4Args {
    const uint8_t *w;
    const void *x;
    const float *x_scale, *bias;
    void *y;
    uint64_t x_stride, y_stride;
    uint32_t M, N, K, blocks, record, y_dtype;
    uint32_t f16_mask;          // all ones: scales are fp16; 0: bf16
    uint32_t zero_at, zero_mask, zero_else;     // place of the zero points in a record, or (mask 0) of anything, and what stands in for them
};

enum { W4_BF16 = 0, W4_F16 = 1, W4_F32 = 2, W4_I8 = 3, W4_BF16_TO_F32 = 4, W4_F16_TO_F32 = 5 };      // type of x (and, of 16 bits, of y)
constexpr bool w4_half(int x) { return x == W4_F16 || x == W4_F16_TO_F32; }
// Weights as q - z themselves: f32 rows, and 16-bit rows whose result keeps 32 bits. (16 + q) would leave it the rounding of terms that are 16 times and more as
// large where large values of x meet small weights; a 16-bit result rounds that away. 14336 x 4096, f32 result, 16 + q / q - z (us): one fp16 row 8.0 / 8.1, 64
// fp16 rows 19.9 / 18.2; one bf16 row 8.1 / 10.2, 64 bf16 rows 19.9 / 21.2 (no packed subtraction in bf16).
constexpr bool w4_exact(int x) { return x == W4_F32 || x == W4_BF16_TO_F32 || x == W4_F16_TO_F32; }

// One lane's 8 neighbouring inputs of one row as matrix operands: one for 16-bit types and int8, three for f32.
template <int X> struct XFrag;
template <> struct XFrag<W4_BF16> { static constexpr int P = 1; using E = __bf16; u32x4 v[1]; };
template <> struct XFrag<W4_F16> { static constexpr int P = 1; using E = _Float16; u32x4 v[1]; };
template <> struct XFrag<W4_F32> { static constexpr int P = 3; using E = float; u32x4 v[3]; };
template <> struct XFrag<W4_BF16_TO_F32> : XFrag<W4_BF16> {};
template <> struct XFrag<W4_F16_TO_F32> : XFrag<W4_F16> {};
template <> struct XFrag<W4_I8> { static constexpr int P = 1; using E = int8_t; u32x2 v[1]; };

template <int X>
__device__ __forceinline__ void x_convert(XFrag<X> &f, const typename XFrag<X>::E (&e)[8]) {
    if constexpr (X == W4_F32) {
        uint32_t u[3][8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const uint32_t b0 = __float_as_uint(e[i]);
            const float r1 = e[i] - __uint_as_float(b0 & 0xFFFF0000u);
            const uint32_t b1 = __float_as_uint(r1);
            const float r2 = r1 - __uint_as_float(b1 & 0xFFFF0000u);
            u[0][i] = b0; u[1][i] = b1; u[2][i] = __float_as_uint(r2);
        }
#pragma unroll
        for (int p = 0; p < 3; ++p)
#pragma unroll
            for (int i = 0; i < 4; ++i) f.v[p][i] = __builtin_amdgcn_perm(u[p][2 * i + 1], u[p][2 * i], 0x07060302u);     // the high halves of two words
    } else if constexpr (X != W4_I8) __builtin_memcpy(&f.v[0], e, 16);
    else {
        // in the order in which a word of 4-bit numbers leaves its bytes: 0 4 1 5 | 2 6 3 7
        uint32_t lo, hi;
        __builtin_memcpy(&lo, e, 4);
        __builtin_memcpy(&hi, e + 4, 4);
        f.v[0][0] = __builtin_amdgcn_perm(hi, lo, 0x05010400u);
        f.v[0][1] = __builtin_amdgcn_perm(hi, lo, 0x07030602u);
    }
}
// A block of 128 inputs of a row is PLACES pieces of 16 bytes, loaded by neighbouring lanes (a wave's load of fragments straight from memory would be 64
// separate lines) and turned into fragments through LDS. There a piece's place is exchanged by the row's number, so that 16 rows' same place meets on
// no LDS banks.
template <int X>
struct Piece {
    using E = typename XFrag<X>::E;
    static constexpr int PER = 16 / (int)sizeof(E), ROW = W4_TK * (int)sizeof(E), PLACES = ROW / 16;
    static __device__ __forceinline__ int place(int row, int c) { return sizeof(E) == 1 ? c ^ ((row >> 1) & 7) : sizeof(E) == 2 ? c ^ (row & 15) : c ^ ((row & 15) << 1); }
    static __device__ __forceinline__ u32x4 load(const E *row, uint32_t k0, int c) {          // of a block within the row
        E v[PER];
        load_any(v, row + k0 + c * PER);
        return __builtin_bit_cast(u32x4, v);
    }
    static __device__ __forceinline__ u32x4 load_part(const E *row, uint32_t k0, int c, uint32_t K) {      // of the last block: zeros behind the row's end
        const uint32_t k = k0 + c * PER;
        E v[PER];
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const E w = row[min(k + i, K - 1)];
            v[i] = k + i < K ? w : (E)0;
        }
        return __builtin_bit_cast(u32x4, v);
    }
    static __device__ __forceinline__ void store(unsigned char *xs, int row, int c, u32x4 v) { *reinterpret_cast<u32x4 *>(xs + row * ROW + place(row, c) * 16) = v; }
    // the lane's 8 inputs of step s of a row
    static __device__ __forceinline__ XFrag<X> fragment(const unsigned char *xs, int row, int s, int quad) {
        E e[8];
        const unsigned char *r = xs + row * ROW;
        if constexpr (sizeof(E) == 1) __builtin_memcpy(e, r + place(row, 2 * s + (quad >> 1)) * 16 + (quad & 1) * 8, 8);
        else if constexpr (sizeof(E) == 2) __builtin_memcpy(e, r + place(row, 4 * s + quad) * 16, 16);
        else __builtin_memcpy(e, r + place(row, 2 * (4 * s + quad)) * 16, 32);
        XFrag<X> f;
        x_convert<X>(f, e);
        return f;
    }
};

template <int X> struct WFrag { u32x4 v; };
template <> struct WFrag<W4_I8> { u32x2 v; };
template <int X>
__device__ __forceinline__ WFrag<X> w_expand(uint32_t w) {
    WFrag<X> f;
    if constexpr (X == W4_I8) { f.v[0] = w & 0x0F0F0F0Fu; f.v[1] = (w >> 4) & 0x0F0F0F0Fu; }
    else if constexpr (X == W4_F16) {
        uint32_t base = 0x4C004C00u;
        asm("" : "+v"(base));             // (in a vector register: and and or are one instruction then)
        f.v[0] = ((w << 6) & 0x03C003C0u) | base; f.v[1] = ((w << 2) & 0x03C003C0u) | base;
        f.v[2] = ((w >> 2) & 0x03C003C0u) | base; f.v[3] = ((w >> 6) & 0x03C003C0u) | base;
    } else {
        uint32_t base = 0x41804180u;
        asm("" : "+v"(base));
        f.v[0] = ((w << 3) & 0x00780078u) | base; f.v[1] = ((w >> 1) & 0x00780078u) | base;
        f.v[2] = ((w >> 5) & 0x00780078u) | base; f.v[3] = ((w >> 9) & 0x00780078u) | base;
    }
    return f;
}
// the weights' own numbers q - z (exact in bf16 and fp16), so that nothing cancels; zero = 16 + z of the lane's output
template <int X>
__device__ __forceinline__ WFrag<X> w_expand_exact(uint32_t w, float zero) {
    WFrag<X> r;
    if constexpr (w4_half(X)) {
        const WFrag<W4_F16> f = w_expand<W4_F16>(w);
        const f16x2 z = {(_Float16)zero, (_Float16)zero};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t pair = f.v[i];          // (a bit cast of a vector's element itself takes the first one)
            r.v[i] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(f16x2, pair) - z);
        }
    } else {
        const WFrag<W4_BF16> f = w_expand<W4_BF16>(w);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float lo = __uint_as_float(f.v[i] << 16) - zero, hi = __uint_as_float(f.v[i] & 0xFFFF0000u) - zero;
            r.v[i] = __builtin_amdgcn_perm(__float_as_uint(hi), __float_as_uint(lo), 0x07060302u);
        }
    }
    return r;
}
template <int X>
__device__ __forceinline__ WFrag<X> w_ones() {
    WFrag<X> f;
    const uint32_t one = X == W4_I8 ? 0x01010101u : X == W4_F16 ? 0x3C003C00u : 0x3F803F80u;
    for (int i = 0; i < (X == W4_I8 ? 2 : 4); ++i) f.v[i] = one;
    return f;
}
template <int X> struct Acc { using V = f32x4; };
template <> struct Acc<W4_I8> { using V = i32x4; };
template <int X>
__device__ __forceinline__ typename Acc<X>::V mma(const WFrag<X> &a, const XFrag<X> &b, typename Acc<X>::V c) {
    if constexpr (X == W4_I8) return __builtin_amdgcn_mfma_i32_16x16x32_i8(__builtin_bit_cast(long, a.v), __builtin_bit_cast(long, b.v[0]), c, 0, 0, 0);
    else if constexpr (w4_half(X)) return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a.v), __builtin_bit_cast(f16x8, b.v[0]), c, 0, 0, 0);
    else {
#pragma unroll
        for (int p = XFrag<X>::P - 1; p >= 0; --p) c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a.v), __builtin_bit_cast(bf16x8, b.v[p]), c, 0, 0, 0);
        return c;
    }
}

// What a wave holds of NT records of one block of inputs.
template <int X, int GROUP, int MT, int NT>
struct Block {
    static constexpr int PER = W4_TK / GROUP, STEPS = GROUP / 32;       // groups of a record; steps of 32 inputs of a group
    static constexpr bool EXACT = w4_exact(X);
    u32x4 w[NT];
    u32x2 s[NT][PER];
    uint32_t z[NT][PER];

    __device__ __forceinline__ void load_w(const W4Args &a, const uint8_t *const (&rec)[NT], size_t at, int lane) {
        const int quad = lane >> 4;
#pragma unroll
        for (int j = 0; j < NT; ++j) {
            const uint8_t *r = rec[j] + at;
            w[j] = *reinterpret_cast<const u32x4 *>(r + lane * 16);
#pragma unroll
            for (int g = 0; g < PER; ++g) {
                s[j][g] = *reinterpret_cast<const u32x2 *>(r + 1024 + g * 32 + quad * 8);
                z[j][g] = (EXACT ? (uint32_t)r[a.zero_at + g * 16 + (lane & 15)] : *reinterpret_cast<const uint32_t *>(r + a.zero_at + g * 16 + quad * 4)) & a.zero_mask | a.zero_else;
            }
        }
    }
    // fragment(t, i): x's step t of tile i; total(g, i): the sum of x over group g for the lane's row of tile i, or nullptr: it is made here
    template <class Fragment, class Total>
    __device__ __forceinline__ void multiply(const W4Args &a, f32x4 (&acc)[NT][MT], Fragment fragment, Total total) const {
        using V = typename Acc<X>::V;
        constexpr bool OWN = std::is_same_v<Total, std::nullptr_t>;
#pragma unroll
        for (int g = 0; g < PER; ++g) {
            V d[NT][MT], sum[MT];
#pragma unroll
            for (int i = 0; i < MT; ++i) {
                sum[i] = V{0, 0, 0, 0};
                if constexpr (!OWN && !EXACT) sum[i][0] = total(g, i);
#pragma unroll
                for (int j = 0; j < NT; ++j) d[j][i] = V{0, 0, 0, 0};
            }
#pragma unroll
            for (int t = g * STEPS; t < (g + 1) * STEPS; ++t) {
                XFrag<X> x[MT];
#pragma unroll
                for (int i = 0; i < MT; ++i) x[i] = fragment(t, i);
#pragma unroll
                for (int j = 0; j < NT; ++j) {
                    WFrag<X> wf;
                    if constexpr (EXACT) wf = w_expand_exact<X>(w[j][t], (float)(z[j][g] & 255u));
                    else wf = w_expand<X>(w[j][t]);
#pragma unroll
                    for (int i = 0; i < MT; ++i) d[j][i] = mma<X>(wf, x[i], d[j][i]);
                }
                if constexpr (!EXACT && OWN)
#pragma unroll
                    for (int i = 0; i < MT; ++i) sum[i] = mma<X>(w_ones<X>(), x[i], sum[i]);
                if constexpr (X == W4_F16_TO_F32 && GROUP == 64 && MT == 4) __builtin_amdgcn_sched_barrier(0);          // (registers for one step's operands: with two's some spill)
            }
            if constexpr (PER > 1) __builtin_amdgcn_sched_barrier(0);          // (groups one after another: side by side they would only cost registers)
#pragma unroll
            for (int j = 0; j < NT; ++j)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const uint16_t h = (uint16_t)(s[j][g][r >> 1] >> (16 * (r & 1)));
                    const float scale = __uint_as_float((__float_as_uint((float)__builtin_bit_cast(_Float16, h)) & a.f16_mask) | (((uint32_t)h << 16) & ~a.f16_mask));
                    const int zero = (int)((z[j][g] >> (8 * r)) & 255u);
#pragma unroll
                    for (int i = 0; i < MT; ++i) {
                        float v;
                        if constexpr (X == W4_I8) v = (float)(d[j][i][r] - (zero - 16) * sum[i][0]);          // (a row's sum: the same for all outputs)
                        else if constexpr (EXACT) v = d[j][i][r];
                        else v = __builtin_fmaf(-(float)zero, sum[i][0], d[j][i][r]);
                        acc[j][i][r] = __builtin_fmaf(v, scale, acc[j][i][r]);
                    }
                }
        }
    }
};

// The waves' sums in their order (through LDS), the row's scale, the bias, the output's type. `first` of `parts` waves that share outputs; t of nt threads.
template <int X, int MT, int NT>
__device__ __forceinline__ void finish(const W4Args &a, const f32x4 (&acc)[NT][MT], float *sums /* [parts][NT][MT][64][4], free when called */, int part, int parts, int t, int nt, uint32_t m0,
                                       uint32_t tile0, int lane) {
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int i = 0; i < MT; ++i) *reinterpret_cast<f32x4 *>(sums + (((part * NT + j) * MT + i) * 64 + lane) * 4) = acc[j][i];
    __syncthreads();
    for (int e = t; e < NT * MT * 64; e += nt) {
        f32x4 v = *reinterpret_cast<const f32x4 *>(sums + e * 4);
        for (int w2 = 1; w2 < parts; ++w2) v += *reinterpret_cast<const f32x4 *>(sums + (w2 * NT * MT * 64 + e) * 4);
        const uint32_t m = m0 + ((e >> 6) % MT) * 16 + (e & 15), n = (tile0 + (e >> 6) / MT) * W4_TN + ((e & 63) >> 4) * 4;
        if (m >= a.M || n >= a.N) continue;
        const float xs = X == W4_I8 ? a.x_scale[m] : 1.0f;
        float o[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) o[r] = (X == W4_I8 ? v[r] * xs : v[r]) + (a.bias && n + r < a.N ? a.bias[n + r] : 0.0f);
        const uint64_t to = (uint64_t)m * a.y_stride + n;
        auto put = [&](auto *y) {
            using Y = std::remove_reference_t<decltype(*y)>;
            Y t[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) t[r] = (Y)o[r];
            if (n + 4 <= a.N) store_any(y + to, t);
            else
                for (int r = 0; r < 4; ++r) if (n + r < a.N) y[to + r] = t[r];
        };
        if (a.y_dtype == SHODH_DTYPE_FP32) put((float *)a.y);
        else if (a.y_dtype == SHODH_DTYPE_BF16) put((__bf16 *)a.y);
        else put((_Float16 *)a.y);
    }
}

// A workgroup of `waves` waves: NT x 16 outputs, MT x 16 rows; wave i takes the blocks of 128 inputs i, i + waves, ..., and the waves' sums are added in
// their order. Matrix layouts: operand lane = output (weights) or row (x) lane & 15, inputs 8 (lane >> 4) ..; result lane = row lane & 15,
// outputs 4 (lane >> 4) .. + 3. U blocks are asked for before the first is multiplied; with U = 1 the next one is on its way meanwhile.
// FEW: there are no more rows than one piece a lane covers (2, 4 or 8 by type): the others' columns hold whatever LDS held, and are not written.
template <int X, int GROUP, int MT, int NT, int U, bool FEW>
__global__ __launch_bounds__(512, FEW && GROUP != 32 && (X == W4_F32 || !w4_exact(X)) ? 6 : MT == 1 && (FEW || X != W4_F32 || GROUP == 128) ? 4 : 2) void w4_dense_kernel(const W4Args a) {
    using P = Piece<X>;
    using E = typename P::E;
    constexpr int STEP = 64 / P::PLACES, PIECES = FEW ? 1 : MT * 16 / STEP, TILE = MT * 16 * P::ROW;         // rows between a lane's pieces of a block, their number
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];           // [waves][TILE]; then the sums
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
    const uint32_t m0 = blockIdx.y * (MT * 16u), tiles = (a.N + W4_TN - 1) / W4_TN;
    unsigned char *xs = smem + wave * TILE;
    const int piece_row = lane / P::PLACES, piece_place = lane % P::PLACES;
    const uint8_t *rec[NT];
#pragma unroll
    for (int j = 0; j < NT; ++j) rec[j] = a.w + (size_t)min(blockIdx.x * NT + j, tiles - 1) * a.blocks * a.record;
    f32x4 acc[NT][MT];
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int i = 0; i < MT; ++i) acc[j][i] = f32x4{0, 0, 0, 0};
    auto x_row = [&](int i) { return (const E *)a.x + (uint64_t)min(m0 + i * STEP + piece_row, a.M - 1) * a.x_stride; };     // (rows behind the last repeat it: not written)
    auto load = [&](u32x4 (&v)[PIECES], Block<X, GROUP, MT, NT> &w, uint32_t block) {
        w.load_w(a, rec, (size_t)block * a.record, lane);
#pragma unroll
        for (int i = 0; i < PIECES; ++i) v[i] = P::load(x_row(i), block * W4_TK, piece_place);
    };
    auto store_x = [&](const u32x4 (&v)[PIECES]) {          // (LDS serves a wave's accesses in order: only the compiler has to be held, from its loads of memory too: 9.1 us, and 9.6 with a fence for LDS alone)
        asm volatile("" ::: "memory");
#pragma unroll
        for (int i = 0; i < PIECES; ++i) P::store(xs, i * STEP + piece_row, piece_place, v[i]);
        asm volatile("" ::: "memory");
    };
    auto fragment = [&](int s, int i) { return P::fragment(xs, i * 16 + (lane & 15), s, lane >> 4); };
    u32x4 x[U][PIECES];
    Block<X, GROUP, MT, NT> b[U];
    const uint32_t full = a.K / W4_TK;         // blocks that no row ends in; loads of these are never behind a branch: a wait after one would be for all of them
    uint32_t at = wave;
    if constexpr (U > 1) {
        for (; at + (U - 1) * waves < full; at += U * waves) {
#pragma unroll
            for (int u = 0; u < U; ++u) load(x[u], b[u], at + u * waves);
#pragma unroll
            for (int u = 0; u < U; ++u) { store_x(x[u]); b[u].multiply(a, acc, fragment, nullptr); }
        }
    }
    if (at < full) {
        load(x[0], b[0], at);
        for (; at < full; at += waves) {
            store_x(x[0]);
            const Block<X, GROUP, MT, NT> cur = b[0];
            load(x[0], b[0], min(at + waves, full - 1));          // (the last one once more: not used)
            cur.multiply(a, acc, fragment, nullptr);
        }
    }
    if (at < a.blocks) {
        b[0].load_w(a, rec, (size_t)at * a.record, lane);
#pragma unroll
        for (int i = 0; i < PIECES; ++i) x[0][i] = P::load_part(x_row(i), at * W4_TK, piece_place, a.K);
        store_x(x[0]);
        b[0].multiply(a, acc, fragment, nullptr);
    }
    __syncthreads();
    finish<X, MT, NT>(a, acc, reinterpret_cast<float *>(smem), wave, waves, threadIdx.x, blockDim.x, m0, blockIdx.x * NT, lane);
}

// More than 16 rows and many outputs: x's blocks are shared by WN waves of 2 x 16 outputs each; WK such sets of waves take every WK-th block. A wave
// brings MT * 16 / WN rows of a block to LDS, a block ahead of the multiplying, and makes those rows' sums there for all (a third of the matrix
// instructions, were each wave to make its own: 28672 x 4096, 64 rows 29.9 us, 27.1 so). Blocks are asked for two rounds ahead, x's three.
template <int X, int GROUP, int MT, int WN, int WK>
__global__ __launch_bounds__(512, 2) void w4_dense_shared_kernel(const W4Args a) {
    using P = Piece<X>;
    using E = typename P::E;
    using V = typename Acc<X>::V;
    using S = std::conditional_t<X == W4_I8, int, float>;
    constexpr int NT = 2, ROWS = MT * 16, TILE = ROWS * P::ROW, MINE = ROWS / WN, STEP = 64 / P::PLACES, N = MINE / STEP, PER = W4_TK / GROUP, COLS = MINE < 16 ? MINE : 16;
    static_assert(WN * WK == 8 && N >= 1, "");
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];           // [WK][2][TILE]; [WK][2][PER][ROWS] sums of x; then the outputs' sums
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wn = wave % WN, wk = wave / WN;
    const uint32_t m0 = blockIdx.y * (MT * 16u), tiles = (a.N + W4_TN - 1) / W4_TN, tile0 = (blockIdx.x * WN + wn) * NT;
    const int piece_row = wn * MINE + lane / P::PLACES, piece_place = lane % P::PLACES;
    const uint8_t *rec[NT];
#pragma unroll
    for (int j = 0; j < NT; ++j) rec[j] = a.w + (size_t)min(tile0 + j, tiles - 1) * a.blocks * a.record;
    f32x4 acc[NT][MT];
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int i = 0; i < MT; ++i) acc[j][i] = f32x4{0, 0, 0, 0};
    unsigned char *xs = smem + wk * 2 * TILE;
    S *totals = reinterpret_cast<S *>(smem + WK * 2 * TILE) + wk * 2 * PER * ROWS;
    u32x4 x[2][N];
    Block<X, GROUP, MT, NT> b[2];
    const uint32_t full = a.K / W4_TK;         // blocks that no row ends in; loads of these are never behind a branch: a wait after one would be for all of them
    auto x_row = [&](int i) { return (const E *)a.x + (uint64_t)min(m0 + i * STEP + piece_row, a.M - 1) * a.x_stride; };
    auto nth = [&](uint32_t r) { return min(r * WK + wk, full - 1); };              // (past the end the last one once more: not used)
    auto load_w = [&](Block<X, GROUP, MT, NT> &w, uint32_t r) { w.load_w(a, rec, (size_t)nth(r) * a.record, lane); };
    auto load_x = [&](u32x4 (&v)[N], uint32_t r) {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = P::load(x_row(i), nth(r) * W4_TK, piece_place);
    };
    auto store = [&](const u32x4 (&v)[N], int half) {
#pragma unroll
        for (int i = 0; i < N; ++i) P::store(xs + half * TILE, i * STEP + piece_row, piece_place, v[i]);
        if constexpr (w4_exact(X)) return;
        wave_lds_order();
#pragma unroll
        for (int c = 0; c < MINE; c += COLS)
#pragma unroll
            for (int g = 0; g < PER; ++g) {
                V sum = V{0, 0, 0, 0};
#pragma unroll
                for (int s = g * GROUP / 32; s < (g + 1) * GROUP / 32; ++s) sum = mma<X>(w_ones<X>(), P::fragment(xs + half * TILE, wn * MINE + c + lane % COLS, s, lane >> 4), sum);
                if (lane < COLS) totals[(half * PER + g) * ROWS + wn * MINE + c + lane] = sum[0];
            }
    };
    auto multiply = [&](const Block<X, GROUP, MT, NT> &w, int half) {
        w.multiply(a, acc, [&](int s, int i) { return P::fragment(xs + half * TILE, i * 16 + (lane & 15), s, lane >> 4); },
                   [&](int g, int i) { return totals[(half * PER + g) * ROWS + i * 16 + (lane & 15)]; });
    };
    auto round = [&](u32x4 (&next)[N], Block<X, GROUP, MT, NT> &w, int half, uint32_t r) {
        __syncthreads();
        const Block<X, GROUP, MT, NT> cur = w;
        load_w(w, r + 2);
        store(next, half ^ 1);
        load_x(next, r + 3);
        if (r * WK + wk < full) multiply(cur, half);
    };
    if (full) {
        load_x(x[0], 0);
        load_w(b[0], 0);
        load_x(x[1], 1);
        load_w(b[1], 1);
        store(x[0], 0);
        load_x(x[0], 2);
        const uint32_t rounds = (full + WK - 1) / WK;
        for (uint32_t r = 0; r < rounds; r += 2) {
            round(x[1], b[0], 0, r);
            round(x[0], b[1], 1, r + 1);
        }
    }
    if (full < a.blocks) {
        const bool turn = (int)(full % WK) == wk;
        if (turn) {
            b[0].load_w(a, rec, (size_t)full * a.record, lane);
#pragma unroll
            for (int i = 0; i < N; ++i) x[0][i] = P::load_part(x_row(i), full * W4_TK, piece_place, a.K);
            store(x[0], 0);              // (the last round read the other half)
        }
        __syncthreads();
        if (turn) multiply(b[0], 0);
    }
    __syncthreads();
    finish<X, MT, NT>(a, acc, reinterpret_cast<float *>(smem) + wn * WK * NT * MT * 256, wk, WK, wk * 64 + lane, WK * 64, m0, tile0, lane);
}

// Which kernel. Up to 16 rows own pieces; measured at 4096 inputs, group 128, bf16 (us; weights cold): rows that one piece a lane covers (4 in 16 bits),
// 4096 outputs 5.3, 14336 outputs 10.8 (all rows' pieces loaded: 9.1 and 29); 16 rows: 6.2 and 16. Beyond them the workgroups are counted in rounds over
// the CUs, a round of each kernel by what it takes. Measured there (us):
//   rows x outputs     32 x 4096   7168  10240  14336  20480  28672    64 x 4096   7168  10240  14336  20480  28672    256 x 4096  14336  28672
//     own pieces             7.9   11.5   14.8   23.1   25.5   38.3         11.6   20.1   27.4   39.0   47.2   66.5          37.7  123.6  242.8
//     shared by 2 waves     12.4   12.6   12.5   14.4   24.4   25.9         18.7   18.8   19.0   21.0   37.1   39.1          19.6   72.0  128.8
//     shared by 4 waves     18.8   18.7   18.6   19.7   19.5   20.6         25.7   25.9   25.9   26.6   26.7   27.9          25.8   51.6  100.8
//   int8 rows: 64 x 7168 15.7 / 17.7 / 29.1; 64 x 28672 51.3 / 35.5 / 30.7; 256 x 10240 62.6 / 49.7 / 56.7
// At 1024 inputs the order is the same. Groups of 32 (64 rows, 28672 outputs): 90 / - / 55, of 64: 81 / 47 / 38.
template <int X, int GROUP>
static int launch_w4(const W4Args &a, uint32_t tiles, int cus, hipStream_t st) {
    auto own = [&](auto kern, uint32_t mt) -> int {
        uint32_t waves = 1;
        while (waves < 8 && waves * 2 <= a.blocks) waves *= 2;
        const size_t lds = (size_t)waves * mt * 16 * Piece<X>::ROW;          // (more than the sums)
        SHODH_TRY(ensure_dynamic_lds((const void *)kern, lds));
        hipLaunchKernelGGL(kern, dim3(tiles, (a.M + 16 * mt - 1) / (16 * mt)), dim3(64 * waves), lds, st, a);
        SHODH_HIP_TRY(hipGetLastError());
        return SHODH_OK;
    };
    if (a.M <= 64 / Piece<X>::PLACES) return own(w4_dense_kernel<X, GROUP, 1, 1, 2, true>, 1);
    if (a.M <= 16) return own(w4_dense_kernel<X, GROUP, 1, 1, X == W4_F32 ? 1 : 2, false>, 1);
    if constexpr (X == W4_F32) return own(w4_dense_kernel<X, GROUP, 2, 1, 1, false>, 2);           // (three parts of each value: registers for no more)
    else {
        auto shared = [&](auto kern, uint32_t mt, uint32_t wn) -> int {
            const size_t x = (size_t)(8 / wn) * 2 * mt * 16 * (Piece<X>::ROW + W4_TK / GROUP * 4), sums = (size_t)8 * 2 * mt * 1024, lds = x > sums ? x : sums;
            SHODH_TRY(ensure_dynamic_lds((const void *)kern, lds));
            hipLaunchKernelGGL(kern, dim3((tiles + 2 * wn - 1) / (2 * wn), (a.M + 16 * mt - 1) / (16 * mt)), dim3(512), lds, st, a);
            SHODH_HIP_TRY(hipGetLastError());
            return SHODH_OK;
        };
        const uint32_t mt = a.M <= 32 ? 2 : 4, row_tiles = (a.M + 16 * mt - 1) / (16 * mt);
        auto cost = [&](uint32_t per /* tiles of a workgroup */, uint32_t round) { return (((uint64_t)(tiles + per - 1) / per * row_tiles + cus - 1) / cus) * round; };
        constexpr uint32_t TWO = X == W4_I8 ? (GROUP == 128 ? 8 : 10) : (GROUP == 128 ? 7 : 8);
        constexpr uint32_t FOUR = X == W4_I8 ? (GROUP == 128 ? 13 : GROUP == 64 ? 16 : 23) : (GROUP == 128 ? 10 : GROUP == 64 ? 12 : 16);
        const uint64_t one = cost(1, mt == 2 ? 3 : 4), two = GROUP == 32 ? ~0ull /* (12 or more: never the least) */ : cost(4, TWO), four = cost(8, FOUR);
        auto pick = [&](auto MT) -> int {
            if (one <= two && one <= four) return own(w4_dense_kernel<X, GROUP, MT.value, 1, 1, false>, MT.value);
            if constexpr (GROUP > 32)
                if (two <= four) return shared(w4_dense_shared_kernel<X, GROUP, MT.value, 2, 4>, MT.value, 2);
            return shared(w4_dense_shared_kernel<X, GROUP, MT.value, 4, 2>, MT.value, 4);
        };
        return mt == 2 ? pick(std::integral_constant<int, 2>{}) : pick(std::integral_constant<int, 4>{});
    }
}
template <int X>
static int pick_w4(const W4Args &a, const shodh_w4_weight *w, hipStream_t st) {
    const int cus = compute_units(w->device);
    return w->group == 32 ? launch_w4<X, 32>(a, w->tiles, cus, st) : w->group == 64 ? launch_w4<X, 64>(a, w->tiles, cus, st) : launch_w4<X, 128>(a, w->tiles, cus, st);
}

static int check_w4(uint32_t N, uint32_t K, uint32_t group, uint32_t scale_dtype, shodh_w4_weight **out) {
    if (!out) { set_error("null argument"); return SHODH_ERR_INVALID; }
    *out = nullptr;
    if (N == 0 || K == 0 || N > (1u << 20) - 16 || K > (1u << 24)) { set_error("w4: %u outputs, %u inputs out of range (1 .. 1048560, 1 .. 16777216)", N, K); return SHODH_ERR_INVALID; }
    if (group != 32 && group != 64 && group != 128) { set_error("w4: group %u is none of 32, 64, 128", group); return SHODH_ERR_UNSUPPORTED; }
    if (scale_dtype != SHODH_DTYPE_FP16 && scale_dtype != SHODH_DTYPE_BF16) { set_error("w4: scales are kept in fp16 or bf16 (got dtype %u)", scale_dtype); return SHODH_ERR_INVALID; }
    return SHODH_OK;
}

// `q` packed two to a byte, `scale`, `zero`: device data. Waits for the stream: the handle is ready when the call returns.
static int lay_out(int device, const uint8_t *q, const float *scale, const uint8_t *zero, uint32_t N, uint32_t K, uint32_t group, uint32_t scale_dtype, uint32_t *d_bad,
                   hipStream_t st, shodh_w4_weight **out) {
    shodh_w4_weight *w = new (std::nothrow) shodh_w4_weight();
    if (!w) { set_error("out of memory"); return SHODH_ERR_OOM; }
    w->device = device; w->N = N; w->K = K; w->group = group; w->scale_dtype = scale_dtype; w->zeros = zero != nullptr;
    w->tiles = (N + W4_TN - 1) / W4_TN; w->blocks = (K + W4_TK - 1) / W4_TK; w->record = record_bytes(group, w->zeros);
    if (dev_alloc(&w->data, (size_t)w->tiles * w->blocks * w->record) != hipSuccess) { (void)hipGetLastError(); delete w; set_error("out of HBM for 4-bit weights"); return SHODH_ERR_OOM; }
    const dim3 grid(w->blocks, w->tiles);
    if (scale_dtype == SHODH_DTYPE_FP16) hipLaunchKernelGGL((w4_pack_kernel<_Float16>), grid, dim3(256), 0, st, q, scale, zero, N, K, group, w->blocks, w->record, w->data, d_bad);
    else hipLaunchKernelGGL((w4_pack_kernel<__bf16>), grid, dim3(256), 0, st, q, scale, zero, N, K, group, w->blocks, w->record, w->data, d_bad);
    uint32_t bad = 0;
    hipError_t e = hipGetLastError();
    if (e == hipSuccess) e = hipMemcpyAsync(&bad, d_bad, 4, hipMemcpyDeviceToHost, st);
    if (e == hipSuccess) e = hipStreamSynchronize(st);
    if (e != hipSuccess || bad) {
        (void)dev_free(w->data); delete w;
        if (e != hipSuccess) { set_error("w4: laying out failed: %s", hipGetErrorString(e)); return SHODH_ERR_DEVICE; }
        if (bad & 2u) { set_error("w4: a zero point is over 15"); return SHODH_ERR_INVALID; }
        if ((bad & 13u) == 8u) { set_error("w4: a scale is not 0 but below what its 16-bit type holds%s", scale_dtype == SHODH_DTYPE_FP16 ? " (bf16 reaches further)" : ""); return SHODH_ERR_INVALID; }
        set_error(bad & 4u ? "w4: a weight is a NaN or an infinity" : "w4: a scale is no finite number of its 16-bit type"); return SHODH_ERR_NONFINITE;
    }
    *out = w;
    return SHODH_OK;
}

struct Buffers {           // device scratch of one create call
    std::vector<void *> held;
    template <class T> T *take(size_t n) {
        void *p = nullptr;
        if (dev_alloc(&p, n * sizeof(T)) != hipSuccess) { (void)hipGetLastError(); return nullptr; }
        held.push_back(p);
        return (T *)p;
    }
    ~Buffers() { for (void *p : held) (void)dev_free(p); }
};

}  // namespace shodh

using namespace shodh;

extern "C" {

int shodh_w4_weight_create_device(int device, const uint8_t *d_q, const float *d_scale, const uint8_t *d_zero, uint32_t N, uint32_t K, uint32_t group, uint32_t scale_dtype,
                                  void *stream, shodh_w4_weight **out) {
    SHODH_TRY(check_w4(N, K, group, scale_dtype, out));
    if (!d_q || !d_scale) { set_error("null argument"); return SHODH_ERR_INVALID; }
    DeviceScope scope;
    SHODH_TRY(scope.enter(device));
    hipStreamCaptureStatus capture = hipStreamCaptureStatusNone;
    SHODH_HIP_TRY(hipStreamIsCapturing((hipStream_t)stream, &capture));
    if (capture != hipStreamCaptureStatusNone) { set_error("w4: weights are not laid out while their stream is captured"); return SHODH_ERR_STATE; }
    const BesideCaptures beside;
    try {
        Buffers b;
        uint32_t *bad = b.take<uint32_t>(1);
        if (!bad) { set_error("out of HBM"); return SHODH_ERR_OOM; }
        SHODH_HIP_TRY(hipMemsetAsync(bad, 0, 4, (hipStream_t)stream));
        return lay_out(device, d_q, d_scale, d_zero, N, K, group, scale_dtype, bad, (hipStream_t)stream, out);
    } catch (const std::exception &ex) { set_error("w4: %s", ex.what()); return SHODH_ERR_OOM; }
}

int shodh_w4_weight_create(int device, const uint8_t *q, const float *scale, const uint8_t *zero, uint32_t N, uint32_t K, uint32_t group, uint32_t scale_dtype, shodh_w4_weight **out) {
    SHODH_TRY(check_w4(N, K, group, scale_dtype, out));
    if (!q || !scale) { set_error("null argument"); return SHODH_ERR_INVALID; }
    DeviceScope scope;
    SHODH_TRY(scope.enter(device));
    const BesideCaptures beside;
    try {
        Buffers b;
        OwnStream own;             // (ends before the buffers do)
        SHODH_TRY(own.make());
        const size_t nq = (size_t)N * ((K + 1) / 2), ng = (size_t)N * ((K + group - 1) / group);
        uint8_t *dq = b.take<uint8_t>(nq), *dz = zero ? b.take<uint8_t>(ng) : nullptr;
        float *ds = b.take<float>(ng);
        if (!dq || !ds || (zero && !dz)) { set_error("out of HBM"); return SHODH_ERR_OOM; }
        SHODH_HIP_TRY(hipMemcpyAsync(dq, q, nq, hipMemcpyHostToDevice, own.st));
        SHODH_HIP_TRY(hipMemcpyAsync(ds, scale, ng * 4, hipMemcpyHostToDevice, own.st));
        if (zero) SHODH_HIP_TRY(hipMemcpyAsync(dz, zero, ng, hipMemcpyHostToDevice, own.st));
        return shodh_w4_weight_create_device(device, dq, ds, dz, N, K, group, scale_dtype, own.st, out);
    } catch (const std::exception &ex) { set_error("w4: %s", ex.what()); return SHODH_ERR_OOM; }
}

int shodh_w4_weight_quantize(int device, const float *w, uint32_t N, uint32_t K, uint32_t group, uint32_t zeros, uint32_t scale_dtype, shodh_w4_weight **out) {
    SHODH_TRY(check_w4(N, K, group, scale_dtype, out));
    if (!w) { set_error("null argument"); return SHODH_ERR_INVALID; }
    DeviceScope scope;
    SHODH_TRY(scope.enter(device));
    const BesideCaptures beside;
    try {
        Buffers b;
        OwnStream own;
        SHODH_TRY(own.make());
        const size_t n = (size_t)N * K, ng = (size_t)N * ((K + group - 1) / group), pairs = (size_t)N * ((K + 1) / 2);
        float *dw = b.take<float>(n), *ds = b.take<float>(ng);
        uint8_t *d1 = b.take<uint8_t>(n), *dq = b.take<uint8_t>(pairs), *dz = zeros ? b.take<uint8_t>(ng) : nullptr;
        uint32_t *bad = b.take<uint32_t>(1);
        if (!dw || !ds || !d1 || !dq || (zeros && !dz) || !bad) { set_error("out of HBM"); return SHODH_ERR_OOM; }
        SHODH_HIP_TRY(hipMemcpyAsync(dw, w, n * 4, hipMemcpyHostToDevice, own.st));
        SHODH_HIP_TRY(hipMemsetAsync(bad, 0, 4, own.st));
        const uint32_t ny = N < 32768 ? N : 32768;
        const dim3 grid((K + group - 1) / group, ny, (N + ny - 1) / ny);
        if (scale_dtype == SHODH_DTYPE_FP16) hipLaunchKernelGGL((w4_quantize_kernel<_Float16>), grid, dim3(64), 0, own.st, dw, N, K, group, zeros, d1, ds, dz, bad);
        else hipLaunchKernelGGL((w4_quantize_kernel<__bf16>), grid, dim3(64), 0, own.st, dw, N, K, group, zeros, d1, ds, dz, bad);
        hipLaunchKernelGGL(w4_pairs_kernel, dim3((uint32_t)(ceil_div(pairs, 256) < 8192 ? ceil_div(pairs, 256) : 8192)), dim3(256), 0, own.st, d1, N, K, dq);
        SHODH_HIP_TRY(hipGetLastError());
        return lay_out(device, dq, ds, dz, N, K, group, scale_dtype, bad, own.st, out);
    } catch (const std::exception &ex) { set_error("w4: %s", ex.what()); return SHODH_ERR_OOM; }
}

void shodh_w4_weight_destroy(shodh_w4_weight *w) {
    if (!w) return;
    DeviceScope scope;
    const BesideCaptures beside;
    if (scope.enter(w->device) == SHODH_OK) (void)dev_free(w->data);
    delete w;
}

int shodh_w4_weight_dequantize(const shodh_w4_weight *w, float *out) {
    if (!w || !out) { set_error("null argument"); return SHODH_ERR_INVALID; }
    DeviceScope scope;
    SHODH_TRY(scope.enter(w->device));
    const BesideCaptures beside;
    try {
        Buffers b;
        OwnStream own;
        SHODH_TRY(own.make());
        const size_t n = (size_t)w->N * w->K;
        float *d = b.take<float>(n);
        if (!d) { set_error("out of HBM"); return SHODH_ERR_OOM; }
        const dim3 grid(w->blocks, w->tiles);
        if (w->scale_dtype == SHODH_DTYPE_FP16) hipLaunchKernelGGL((w4_unpack_kernel<_Float16>), grid, dim3(256), 0, own.st, w->data, w->N, w->K, w->group, w->blocks, w->record, w->zeros, d);
        else hipLaunchKernelGGL((w4_unpack_kernel<__bf16>), grid, dim3(256), 0, own.st, w->data, w->N, w->K, w->group, w->blocks, w->record, w->zeros, d);
        SHODH_HIP_TRY(hipGetLastError());
        SHODH_HIP_TRY(hipMemcpyAsync(out, d, n * 4, hipMemcpyDeviceToHost, own.st));
        SHODH_HIP_TRY(hipStreamSynchronize(own.st));
        return SHODH_OK;
    } catch (const std::exception &ex) { set_error("w4: %s", ex.what()); return SHODH_ERR_OOM; }
}

int shodh_w4_weight_shape(const shodh_w4_weight *w, uint32_t *N, uint32_t *K, uint32_t *group, uint64_t *bytes) {
    if (!w) { set_error("null argument"); return SHODH_ERR_INVALID; }
    if (N) *N = w->N;
    if (K) *K = w->K;
    if (group) *group = w->group;
    if (bytes) *bytes = (uint64_t)w->tiles * w->blocks * w->record;
    return SHODH_OK;
}

int shodh_w4_dense_device(const shodh_w4_weight *w, const void *d_x, uint32_t x_dtype, uint64_t x_stride, const float *d_x_scale, uint32_t rows, const float *d_bias, void *d_y,
                          uint32_t y_dtype, uint64_t y_stride, void *stream) {
    if (!w) { set_error("null argument"); return SHODH_ERR_INVALID; }
    if (!is_float_dtype(x_dtype) && x_dtype != SHODH_DTYPE_INT8) { set_error("w4: x of dtype %u: fp32, bf16, fp16 or int8 are taken", x_dtype); return SHODH_ERR_INVALID; }
    if (!is_float_dtype(y_dtype)) { set_error("w4: y of dtype %u: fp32, bf16 or fp16", y_dtype); return SHODH_ERR_INVALID; }
    if (rows == 0) return SHODH_OK;
    if (!d_x || !d_y) { set_error("null argument"); return SHODH_ERR_INVALID; }
    if ((x_dtype == SHODH_DTYPE_INT8) != (d_x_scale != nullptr)) { set_error("w4: int8 rows come with a scale each, others with none"); return SHODH_ERR_INVALID; }
    const uint64_t xs = x_stride ? x_stride : w->K, ys = y_stride ? y_stride : w->N;
    if (rows > 1 && ys < w->N) { set_error("w4: y's rows overlap (stride %llu below %u)", (unsigned long long)ys, w->N); return SHODH_ERR_DIM; }
    if (!aligned_to(d_x, dtype_bytes(x_dtype)) || !aligned_to(d_y, dtype_bytes(y_dtype)) || !aligned_to(d_x_scale, 4) || !aligned_to(d_bias, 4)) {
        set_error("w4: a pointer is not a multiple of its element's size"); return SHODH_ERR_INVALID;
    }
    const size_t xb = dtype_bytes(x_dtype), yb = dtype_bytes(y_dtype);
    const Region y(d_y, w->N * yb, rows, ys * yb);
    if (may_overlap(y, Region(d_x, w->K * xb, rows, xs * xb)) || may_overlap(y, Region(d_x_scale, rows * 4ull)) || may_overlap(y, Region(d_bias, w->N * 4ull)) ||
        may_overlap(y, Region(w->data, (uint64_t)w->tiles * w->blocks * w->record))) {
        set_error("w4: y overlaps another operand"); return SHODH_ERR_INVALID;
    }
    DeviceScope scope;
    SHODH_TRY(scope.enter(w->device));
    W4Args a;
    a.w = w->data; a.bias = d_bias; a.x_stride = xs; a.y_stride = ys; a.N = w->N; a.K = w->K; a.blocks = w->blocks; a.record = w->record; a.y_dtype = y_dtype;
    a.f16_mask = w->scale_dtype == SHODH_DTYPE_FP16 ? 0xFFFFFFFFu : 0u;
    a.zero_at = w->zeros ? 1024 + (W4_TK / w->group) * 32 : 1024; a.zero_mask = w->zeros ? 0xFFFFFFFFu : 0u; a.zero_else = w->zeros ? 0u : 0x18181818u;
    hipStream_t st = (hipStream_t)stream;
    // A launch has at most 65535 workgroups of 32 rows or more, and fewer than 2^31 threads (512 for each tile of outputs): further rows in turns.
    const uint32_t most = 0x7FFFFFFFu / (w->tiles * 512u), turn = 32u * (most < 65535u ? most : 65535u);
    for (uint64_t r = 0; r < rows; r += turn) {
        a.x = (const uint8_t *)d_x + r * xs * xb; a.y = (uint8_t *)d_y + r * ys * yb; a.x_scale = d_x_scale ? d_x_scale + r : nullptr;
        a.M = (uint32_t)(rows - r < turn ? rows - r : turn);
        const bool wide = y_dtype == SHODH_DTYPE_FP32;
        switch (x_dtype) {
            case SHODH_DTYPE_BF16: SHODH_TRY(wide ? pick_w4<W4_BF16_TO_F32>(a, w, st) : pick_w4<W4_BF16>(a, w, st)); break;
            case SHODH_DTYPE_FP16: SHODH_TRY(wide ? pick_w4<W4_F16_TO_F32>(a, w, st) : pick_w4<W4_F16>(a, w, st)); break;
            case SHODH_DTYPE_FP32: SHODH_TRY(pick_w4<W4_F32>(a, w, st)); break;
            default: SHODH_TRY(pick_w4<W4_I8>(a, w, st));
        }
    }
    return SHODH_OK;
}

}  // extern "C"
