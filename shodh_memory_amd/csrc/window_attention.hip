// window_attention.hip -- attention with a sliding window and a few first tokens that stay visible (sinks), over ragged batches, with grouped heads,
// for whole texts as for single tokens at the end of a cache.
//
//   query i of a sequence (Lq new tokens, Lk keys) stands at p = i + Lk - Lq and sees key j iff  j <= p + right  and  (j >= p - left or j < sinks)
//   out = sum_j softmax_j(scale q k_j) v_j over the visible keys;  lse = log sum_j exp(scale q k_j);  no visible key: zeros and -inf
//
// Everything is computed transposed, so that a lane owns one query: S^T = K Q^T (matrix instruction 32 x 32 x 16: rows = keys, columns = queries), softmax
// down the lane's own registers, O^T = V^T P^T with P straight from those registers. The order in which the first product hands keys to a lane
// (register r of half h holds key (r & 3) + 8 (r >> 2) + 4 h of 32) is taken as the order of the second product's inner index; V^T in that order is what
// the transposing LDS read returns for four neighbouring keys. One pass over the keys, with a running maximum and sum in f32. The reference maximum is
// only raised when a tile's maximum is more than 8 (in powers of two) above its place: until then the accumulator is not scaled again. P is rounded to the
// inputs' 16-bit type, because that is what the matrix instruction multiplies; the sum is of unrounded values. fp16 has no number below 2^-24, so there
// the reference lies 7 below the maximum: the largest P is 2^7 .. 2^15 and one step of the smallest is 2^-31 of it or less, which keeps what a sink with
// nearly all the weight leaves to 4096 others (17.5 above them: within 0.02 %; with the reference at the maximum an eighth to all of it was lost). bf16 needs no such room.
//
// A row of work is one (query token, head of a group): the heads that share a key head read the same tile. Two forms:
//  * tiles (texts, prompts): 4 waves x 32 rows, K and V tiles of 64 keys straight to LDS, the next tile on its way meanwhile. Bound: the matrix unit, with
//    the softmax hidden under it but for a tenth, and the first and last tiles of a window. 8192 tokens, 32 over 8 heads of 128, 2048 keys each (bf16):
//    258 - 265 us, 0.92 PFLOP/s (a large matrix product: 1.27). Of 272 us, before sinks shared a tile, it took 238 with the products alone (213 without
//    their tiles' transfers) and 40 with no tile at all (q and out: 134 MB). 96 texts of up to 512 tokens, 12 heads of 32: 20 us, half of it one launch and its first loads.
//  * split (few rows): one tile of 32 rows, the 4 waves take different blocks of 32 keys through LDS of their own, and further workgroups other parts of
//    the key range; parts are added in a fixed order. Bound: HBM (the visible keys are read once). 48 single tokens over caches of up to 32768 keys,
//    32 over 8 heads of 128 (bf16): 109 us, 477 MB, 4.4 TB/s; one token over 4096 keys: 8 us and 5 for the parts' join. 900 tokens over 32768 keys: 1.82 ms.
// Heads are computed as 32, 64 or 128 features: of 40 and 72 .. 96 they cost what the next of these does and up to a tenth more (tiles of them are not whole: 8192
// tokens 179 us for 40, 153 for 64, 290 for 96, 260 for 128).
// Masked places may hold anything: scores there are replaced, and where a tile is partly masked its V is looked through for a NaN or an infinity: such
// values are taken out of the tile, and put into the rows that see them at the end.
#include "glds.h"
#include "layers.h"

#pragma clang fp contract(off)

namespace shodh {

struct AttnArgs {
    const void *q, *k, *v;
    void *out;
    float *lse;
    const int32_t *cu;
    const int64_t *kv_start;
    const int32_t *kv_len;
    float *part;               // split form, the workspace: 16 bytes (number of rows to be joined, per key head), [kv_heads][list_room] of these rows,
                               // [kv_heads][room][DP] parts' sums, [kv_heads][room][2] maxima and sums
    uint64_t q_stride, q_head, k_stride, k_head, v_stride, v_head, o_stride, o_head;
    int64_t q_tokens, kv_tokens;
    uint32_t heads, kv_heads, group, dim, seqs, slots, splits, chunk /* blocks of 32 keys of a part */, sinks;
    uint32_t room, list_room, coarser;       // (AttnPlan)
    int32_t left, right;       // negative: no bound
    float scale2;              // |scale| * log2(e)
    uint32_t sign;             // 0, or the sign bits of two 16-bit numbers
    int shift;                 // log2(group), or -1
    __device__ __forceinline__ uint32_t over_group(uint32_t x) const { return shift >= 0 ? x >> shift : x / group; }
    __device__ __forceinline__ u32x4 *list() const { return reinterpret_cast<u32x4 *>(part) + 1; }          // of a row: its place in lse (64 bits), its first part, their number
    __device__ __forceinline__ float *sums() const { return reinterpret_cast<float *>(list() + (uint64_t)kv_heads * list_room); }
    __device__ __forceinline__ float *stats(int dp) const { return sums() + (uint64_t)kv_heads * room * dp; }
};

constexpr float NEG_INF = -__builtin_inff();

__device__ __forceinline__ float half_max(float x) {        // over a lane and its partner in the other half of the wave
    const auto s = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(s[0]), __uint_as_float(s[1]));
}
__device__ __forceinline__ float half_sum(float x) {
    const auto s = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(s[0]) + __uint_as_float(s[1]);
}

// (BELOW: how far the reference maximum lies below the largest score, in powers of two)
template <class T> struct Vec8;
template <> struct Vec8<__bf16> { using V = bf16x8; using V2 = bf16x2; static constexpr uint32_t EXP = 0x7F807F80u, ONE = 0x00800080u; static constexpr float BELOW = 0.0f; };
template <> struct Vec8<_Float16> { using V = f16x8; using V2 = f16x2; static constexpr uint32_t EXP = 0x7C007C00u, ONE = 0x04000400u; static constexpr float BELOW = 7.0f; };
__device__ __forceinline__ f32x16 mma32(bf16x8 a, bf16x8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x16 mma32(f16x8 a, f16x8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }

// Does a wave find a value that is no number in BYTES of V in LDS?
template <class T, int BYTES>
__device__ __forceinline__ bool find_values(const unsigned char *Vs, int lane) {
    uint32_t m = 0;
#pragma unroll 8
    for (int e = 0; e < BYTES; e += 1024) {
        const u32x4 w = *reinterpret_cast<const u32x4 *>(Vs + e + lane * 16);
#pragma unroll
        for (int i = 0; i < 4; ++i) m |= (w[i] & Vec8<T>::EXP) + Vec8<T>::ONE;          // an exponent of all ones carries into the sign's place
    }
    return __any((m & 0x80008000u) != 0);
}
// Takes them out, by NT threads.
template <class T, int NT>
__device__ __forceinline__ void clear_values(unsigned char *Vs, int bytes, int t) {
    for (int e = t * 16; e < bytes; e += NT * 16) {
        u32x4 w = *reinterpret_cast<const u32x4 *>(Vs + e);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t bad = ((w[i] & Vec8<T>::EXP) + Vec8<T>::ONE) & 0x80008000u;
            w[i] &= (bad & 0x8000u ? 0u : 0x0000FFFFu) | (bad & 0x80000000u ? 0u : 0xFFFF0000u);
        }
        *reinterpret_cast<u32x4 *>(Vs + e) = w;
    }
}

// 16-byte places of a row of DP values, exchanged so that neither 16 rows' same place (a fragment of K) nor 4 rows' same four places (of V, read across)
// meet on LDS banks, which repeat every 256 bytes: 1, 2 or 4 rows
template <int DP> __device__ __forceinline__ int k_place(int row, int c) { return DP == 32 ? c ^ ((row >> 2) & 3) : DP == 64 ? c ^ ((row >> 1) & 7) : c ^ (row & 15); }
template <int DP> __device__ __forceinline__ int v_place(int row, int c) { return DP == 32 ? c : DP == 64 ? c ^ ((row & 2) << 1) : c ^ ((row & 3) << 2); }

typedef short s16x4 __attribute__((ext_vector_type(4)));

// Sequence of a tile slot: the largest b with cu[b] * group / BM + b <= slot (those starts rise strictly), and its tokens [t0, t1).
__device__ __forceinline__ int find_seq(const AttnArgs &a, int64_t slot, int bm, int &t0, int &t1) {
    const int lane = threadIdx.x & 63, seqs = (int)a.seqs;
    auto starts_by = [&](int b, int c) { return ((int64_t)(c < 0 ? 0 : min((int64_t)c, a.q_tokens)) * a.group) / bm + b <= slot; };
    if (seqs < 256) {                       // all of cu at once
        int c[4], got = 0;
#pragma unroll
        for (int u = 0; u < 4; ++u) c[u] = u * 64 <= seqs ? a.cu[min(u * 64 + lane, seqs)] : 0;
#pragma unroll
        for (int u = 0; u < 4; ++u) got += __popcll(__ballot(u * 64 + lane < seqs && starts_by(u * 64 + lane, c[u])));
        const int b = max(got, 1) - 1;
        t0 = t1 = 0;
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int x = __builtin_amdgcn_readlane(c[u], b & 63), y = __builtin_amdgcn_readlane(c[u], (b + 1) & 63);
            t0 = (b >> 6) == u ? x : t0;
            t1 = ((b + 1) >> 6) == u ? y : t1;
        }
        return b;
    }
    int lo = 0, n = seqs;                   // the answer is in [lo, lo + n); 64 probes at a time
    while (n > 1) {
        const int step = (n + 63) / 64, b = lo + lane * step;
        const int got = __popcll(__ballot(lane * step < n && starts_by(b, a.cu[min(b, seqs)])));       // (lane 0's start is never above the slot)
        const int at = got > 0 ? got - 1 : 0;
        lo += at * step;
        n = min(step, n - at * step);
    }
    lo = __builtin_amdgcn_readfirstlane(lo);
    t0 = __builtin_amdgcn_readfirstlane(a.cu[lo]); t1 = __builtin_amdgcn_readfirstlane(a.cu[lo + 1]);
    return lo;
}

__device__ __forceinline__ int64_t uniform64(int64_t x) {       // a number that all lanes hold alike, in scalar registers
    return (int64_t)(((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(x >> 32)) << 32) | (uint32_t)__builtin_amdgcn_readfirstlane((int)x));
}
constexpr int MOST_KEYS = 0x7FFFFF00;          // (a place behind the last tile is a number too)
struct Seq {
    int64_t q0, k0;
    int nq, nk;
};
__device__ __forceinline__ Seq seq_at(const AttnArgs &a, int b, int64_t t0, int64_t t1) {        // of the tokens [t0, t1)
    Seq s;
    if (t0 < 0 || t1 < t0 || t1 > a.q_tokens) t0 = t1 = 0;            // no such rows: nothing is done for them
    s.q0 = t0; s.nq = (int)(t1 - t0);
    if (a.kv_start) {
        s.k0 = a.kv_start[b]; s.nk = a.kv_len[b];
        if (s.k0 < 0 || s.nk < 0 || s.k0 > a.kv_tokens || s.nk > a.kv_tokens - s.k0 || s.nk > MOST_KEYS) { s.k0 = 0; s.nk = 0; }      // no such keys: none is seen
    } else { s.k0 = t0; s.nk = s.nq; }
    return s;
}
__device__ __forceinline__ Seq seq_of(const AttnArgs &a, int b, int t0, int t1) {           // all alike in all lanes
    Seq s = seq_at(a, b, t0, t1);
    s.q0 = uniform64(s.q0); s.k0 = uniform64(s.k0);
    s.nq = __builtin_amdgcn_readfirstlane(s.nq); s.nk = __builtin_amdgcn_readfirstlane(s.nk);
    return s;
}

// One wave's 32 rows: positions, running statistics, accumulators.
template <class T, int DP>
struct Rows {
    using V8 = typename Vec8<T>::V;
    int lane;                  // (kept apart from threadIdx: what is formed from it is not kept in registers around a loop over items)
    V8 q[DP / 16];
    f32x16 o[DP / 32];
    float m, l;                // reference maximum (powers of two) and this half's part of the sum
    int lo, hi;                // the lane's query sees [lo, hi) and the sinks below hi
    bool live;
    uint32_t token, head;      // of the lane's row (token within the sequence)
    uint32_t at_k[DP / 16], at_v[DP / 32];      // LDS offsets of the lane's fragments in a block

    __device__ __forceinline__ void init(const AttnArgs &a, const Seq &s, uint32_t kvh, int64_t row) {
        lane = threadIdx.x & 63;
        asm volatile("" : "+v"(lane));
        const int half = lane >> 5;
        const uint32_t r = (uint32_t)row + (lane & 31);          // (a sequence has fewer than 2^31 rows)
        live = r < (uint32_t)s.nq * a.group;
        token = live ? a.over_group(r) : 0;
        head = kvh * a.group + (live ? r - token * a.group : 0);
        const int64_t p = (int64_t)token + s.nk - s.nq;
        const int64_t h = a.right < 0 ? s.nk : p + a.right + 1, w = a.left < 0 ? 0 : p - a.left;
        hi = live ? (int)(h < 0 ? 0 : h > s.nk ? s.nk : h) : 0;
        lo = (int)(w < 0 ? 0 : w > s.nk ? s.nk : w);
        load_q(a, s);
#pragma unroll
        for (int t = 0; t < DP / 32; ++t)
#pragma unroll
            for (int r2 = 0; r2 < 16; ++r2) o[t][r2] = 0.0f;
        m = NEG_INF; l = 0.0f;
        const int l31 = lane & 31, sub = lane & 15;
#pragma unroll
        for (int i = 0; i < DP / 16; ++i) {
            at_k[i] = l31 * (DP * 2) + k_place<DP>(l31, 2 * i + half) * 16;
            asm volatile("" : "+v"(at_k[i]));
        }
#pragma unroll
        for (int t = 0; t < DP / 32; ++t) {
            const int row = half * 4 + (sub >> 2);
            at_v[t] = row * (DP * 2) + v_place<DP>(row, t * 4 + ((lane >> 4) & 1) * 2 + ((sub & 3) >> 1)) * 16 + (sub & 1) * 8;
            asm volatile("" : "+v"(at_v[t]));
        }
    }
    __device__ __forceinline__ void load_q(const AttnArgs &a, const Seq &s) {
        const int half = lane >> 5;
        const T *src = (const T *)a.q + (uint64_t)(s.q0 + token) * a.q_stride + (uint64_t)head * a.q_head;
#pragma unroll
        for (int i = 0; i < DP / 16; ++i) {
            const uint32_t d = i * 16 + half * 8;
            T e[8];
            if (live && d < a.dim) load_any(e, src + d);
            else
                for (int x = 0; x < 8; ++x) e[x] = (T)0.0f;
            u32x4 w;
            __builtin_memcpy(&w, e, 16);
            w ^= a.sign;                // a negative scale: its sign goes to q (exact), so that the largest score has the largest product
            __builtin_memcpy(&q[i], &w, 16);
        }
    }

    // Scores of NB blocks of 32 keys in LDS at Ks; `meanwhile` is called while their fragments are on their way.
    template <int NB, class Meanwhile>
    __device__ __forceinline__ void scores(const unsigned char *Ks, f32x16 (&s)[NB], Meanwhile meanwhile) const {
        V8 k[NB][DP / 16];
#pragma unroll
        for (int i = 0; i < DP / 16; ++i)
#pragma unroll
            for (int b = 0; b < NB; ++b) k[b][i] = *reinterpret_cast<const V8 *>(Ks + at_k[i] + b * (32 * DP * 2));
        if constexpr (NB > 1) __builtin_amdgcn_sched_barrier(0);          // (all of them on their way before the first is waited for)
        meanwhile();
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int r = 0; r < 16; ++r) s[b][r] = 0.0f;
#pragma unroll
        for (int i = 0; i < DP / 16; ++i)
#pragma unroll
            for (int b = 0; b < NB; ++b) s[b] = mma32(k[b][i], q[i], s[b]);
    }
    // The same for one block, with the queries' fragments in LDS: [DP / 16][64 lanes] x 16 bytes at Qs.
    __device__ __forceinline__ void scores_lds(const unsigned char *Ks, const unsigned char *Qs, f32x16 &s) const {
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] = 0.0f;
#pragma unroll
        for (int i = 0; i < DP / 16; ++i)
            s = mma32(*reinterpret_cast<const V8 *>(Ks + at_k[i]), *reinterpret_cast<const V8 *>(Qs + i * 1024 + lane * 16), s);
    }
    // Scores to probabilities. Block b begins at key[b]; keys from limit[b] on belong to no one here; masked: some row does not see some key of these.
    template <int NB>
    __device__ __forceinline__ void softmax(const AttnArgs &a, f32x16 (&s)[NB], V8 (&p)[NB][2], const int (&key)[NB], const int (&limit)[NB], bool masked) {
        if (masked) {
            const int half = lane >> 5;
            auto first = [](int n) { return n <= 0 ? 0u : n >= 32 ? 0xFFFFFFFFu : (1u << n) - 1u; };
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                // a bit for each of the block's keys that the row sees; in the order of the registers after a shift by the half's 4
                const int j = key[b], end = min(hi, limit[b]);
                const uint32_t seen = (first(end - j) & (~first(lo - j) | first((int)a.sinks - j))) >> (4 * half);
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const uint32_t keep = (uint32_t)((int)(seen << (31 - (r & 3) - 8 * (r >> 2))) >> 31);
                    s[b][r] = __uint_as_float((__float_as_uint(s[b][r]) & keep) | (~keep & 0xFF800000u));
                }
            }
        }
        float tops[4] = {NEG_INF, NEG_INF, NEG_INF, NEG_INF};
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int r = 0; r < 16; ++r) tops[r & 3] = fmaxf(tops[r & 3], s[b][r]);
        const float top = half_max(fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]))) * a.scale2;
        const bool raise = top > m + (8.0f + Vec8<T>::BELOW);      // (m = -inf: any finite score); a row's own affair: its neighbours change nothing in it
        if (__any(raise)) {
            const float next = raise ? top - Vec8<T>::BELOW : m, c = raise ? __builtin_amdgcn_exp2f(m - next) : 1.0f;
            m = next;
            l *= c;
#pragma unroll
            for (int t = 0; t < DP / 32; ++t)
#pragma unroll
                for (int r = 0; r < 16; ++r) o[t][r] *= c;
        }
        const float base = m == NEG_INF ? 0.0f : m;
        float ls[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int r = 0; r < 16; r += 2) {
                f32x2 v;
                v[0] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[b][r], a.scale2, -base));
                v[1] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[b][r + 1], a.scale2, -base));
                ls[r & 3] += v[0];
                ls[(r & 3) + 1] += v[1];
                const auto c = __builtin_convertvector(v, typename Vec8<T>::V2);
                p[b][r >> 3][r & 7] = c[0];
                p[b][r >> 3][(r & 7) + 1] = c[1];
            }
        l += (ls[0] + ls[1]) + (ls[2] + ls[3]);
    }
    // Probabilities times values in LDS at Vs.
    template <int NB>
    __device__ __forceinline__ void values(const unsigned char *Vs, const V8 (&p)[NB][2]) {
        V8 f[2][DP / 32];           // the fragments of 16 keys are on their way while those of the 16 before them are multiplied
#pragma unroll
        for (int t = 0; t < DP / 32; ++t) f[0][t] = v_frag(Vs, 0, 0, t);
#pragma unroll
        for (int x = 0; x < 2 * NB; ++x) {
            if (x + 1 < 2 * NB)
#pragma unroll
                for (int t = 0; t < DP / 32; ++t) f[(x + 1) & 1][t] = v_frag(Vs, (x + 1) >> 1, (x + 1) & 1, t);
#pragma unroll
            for (int t = 0; t < DP / 32; ++t) o[t] = mma32(f[x & 1][t], p[x >> 1][x & 1], o[t]);
        }
    }

    // V^T of 16 keys (inner order as above) and 32 features
    __device__ __forceinline__ V8 v_frag(const unsigned char *Vs, int b, int u, int t) const {
        s16x4 v[2];
#pragma unroll
        for (int x = 0; x < 2; ++x)
            v[x] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4 *)(Vs + at_v[t] + (b * 32 + u * 16 + x * 8) * (DP * 2)));
        V8 f;
        __builtin_memcpy(&f, v, 16);
        return f;
    }

    // Values that are no numbers were taken out of the tiles that some row sees in part (clear_values): here they go into the rows that do see them, as
    // what they make of any sum. (A row that took one in already is what it is.)
    __device__ __forceinline__ void spoil(const AttnArgs &a, const T *vb, int j0, int j1, int limit) {
        const int half = lane >> 5, end = min(hi, limit);
        for (int j = j0; j < j1; ++j) {
            const T *v = vb + (uint64_t)j * a.v_stride;
            bool bad = false;
            for (uint32_t d = lane; d < a.dim; d += 64) bad |= !(__builtin_fabsf((float)v[d]) < __builtin_inff());
            if (!__any(bad)) continue;
            const bool sees = j < end && (j >= lo || j < (int)a.sinks);
            const T *mine = v + half * 4;
#pragma unroll
            for (int t = 0; t < DP / 32; ++t)
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    if ((uint32_t)(t * 32 + g * 8) >= a.dim) continue;
                    T e[4];
                    load_any(e, mine + t * 32 + g * 8);
#pragma unroll
                    for (int x = 0; x < 4; ++x) {
                        const float f = (float)e[x];
                        o[t][4 * g + x] += sees && !(__builtin_fabsf(f) < __builtin_inff()) ? f : 0.0f;
                    }
                    asm volatile("" ::: "memory");       // (four at a time: registers for this would be taken from the loop before)
                }
        }
    }

    // 32 features (of tile t), and what goes with a row
    __device__ __forceinline__ void store(const AttnArgs &a, const Seq &s, const f32x16 &v, int t, float total) const {
        const float inv = total > 0.0f || total != total ? 1.0f / total : 0.0f;
        T *dst = (T *)a.out + (uint64_t)(s.q0 + token) * a.o_stride + (uint64_t)head * a.o_head;
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const uint32_t d = t * 32 + g * 8 + (lane >> 5) * 4;
            T e[4];
#pragma unroll
            for (int x = 0; x < 4; ++x) e[x] = (T)(total == 0.0f ? 0.0f : v[4 * g + x] * inv);
            if (d < a.dim) store_any(dst + d, e);
        }
    }
    __device__ __forceinline__ void store_lse(const AttnArgs &a, const Seq &s, float total) const {
        if (a.lse) a.lse[(uint64_t)(s.q0 + token) * a.heads + head] = total == 0.0f ? NEG_INF : (m + __builtin_amdgcn_logf(total)) * 0.69314718055994530942f;
    }
};

// What the live rows [r0, r1) of a sequence see: the last begin and the first end (everybody's), the first begin and the last end (anybody's). No such rows: nothing.
struct Bounds {
    int lo_max, hi_min, lo_min, hi_max;
};
__device__ __forceinline__ Bounds bounds_of(const AttnArgs &a, const Seq &s, int64_t r0, int64_t r1) {
    const int64_t rows = (int64_t)s.nq * a.group;
    if (r1 > rows) r1 = rows;
    if (r0 >= r1) return Bounds{0, 0x7FFFFFFF, 0x7FFFFFFF, 0};
    const int64_t p0 = (int64_t)(a.over_group((uint32_t)r0)) + s.nk - s.nq, p1 = (int64_t)(a.over_group((uint32_t)(r1 - 1))) + s.nk - s.nq;
    auto clamped = [&](int64_t x) { return (int)(x < 0 ? 0 : x > s.nk ? s.nk : x); };
    return Bounds{a.left < 0 ? 0 : clamped(p1 - a.left), a.right < 0 ? s.nk : clamped(p0 + a.right + 1), a.left < 0 ? 0 : clamped(p0 - a.left), a.right < 0 ? s.nk : clamped(p1 + a.right + 1)};
}
// Range of keys that the rows [r0, r1) of a sequence see: sinks [0, first) and [begin, end); a multiple of 32 begins the second.
struct Range {
    int first, begin, end;
};
__device__ __forceinline__ Range range_of(const AttnArgs &a, const Seq &s, int64_t r0, int64_t r1) {
    const int64_t rows = (int64_t)s.nq * a.group;
    r1 = r1 < rows ? r1 : rows;
    const int64_t p0 = (int64_t)(a.over_group((uint32_t)r0)) + s.nk - s.nq, p1 = (int64_t)(a.over_group((uint32_t)(r1 - 1))) + s.nk - s.nq;
    int64_t end = a.right < 0 ? s.nk : p1 + a.right + 1, begin = a.left < 0 ? 0 : p0 - a.left;
    end = end < 0 ? 0 : end > s.nk ? s.nk : end;
    begin = begin < 0 ? 0 : begin > end ? end : begin;
    Range g;
    g.end = (int)end;
    g.begin = (int)begin & ~31;
    g.first = (int)a.sinks < g.begin ? (int)a.sinks : g.begin;
    return g;
}

// KEYS rows of K or V to LDS by NT threads (t of them is this one). DMA: straight from memory, 16 bytes a lane, in flight when the call returns; every
// place of LDS fetches what belongs there, places behind the head's features are left alone (they were cleared once). Rows and heads that do not
// begin at multiples of 16 bytes go through registers instead, and are there when the call returns. Rows behind the last valid one repeat it: their
// scores are replaced, and what V holds there counts as any masked place does.
template <class T, int DP, int KEYS, int NT, bool DMA, class Place>
__device__ __forceinline__ void stage(unsigned char *lds, const T *base, uint64_t stride, int last, uint32_t dim, int t, Place place) {
    constexpr int N = KEYS * DP / 8 / NT;          // 16-byte places of a thread
    auto to = [&](int i) { return (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)(uintptr_t)(__attribute__((address_space(3))) unsigned char *)(lds + (size_t)(i * NT + (t & ~63)) * 16)); };
    int t2 = t;
    asm volatile("" : "+v"(t2));           // (addresses are formed here, not kept in registers through the loop around)
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int e = i * NT + t2, row = e / (DP / 8), x = e % (DP / 8), c = place(row, x);      // (an exchange is its own inverse)
        const uint32_t from = (uint32_t)min(row, last);
        const bool in = (uint32_t)(c * 8) < dim;
        if constexpr (DMA) {
            if (in) glds16(uniform_ptr((const unsigned char *)base), (from * (uint32_t)stride + c * 8) * 2, to(i));
        } else {
            T v[8];
            load_any(v, base + (uint64_t)from * stride + (in ? c * 8 : 0));
            u32x4 w;
            __builtin_memcpy(&w, v, 16);
            if (!in) w = u32x4{0, 0, 0, 0};
            *reinterpret_cast<u32x4 *>(lds + e * 16) = w;
        }
    }
}
// 1 .. 4 transfers of 16 bytes a lane from one base to LDS places `step` bytes apart, as one statement
template <int N>
__device__ __forceinline__ void glds16_n(const void *base, const uint32_t (&off)[N], uint32_t lds, uint32_t step) {
    unsigned keep;
    if constexpr (N == 1)
        asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %3\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2\n\ts_mov_b32 m0, %0" : "=&s"(keep) : "v"(off[0]), "s"(base), "s"(lds) : "memory");
    else if constexpr (N == 2)
        asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %4\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %3\n\ts_add_u32 m0, m0, %5\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %2, %3\n\ts_mov_b32 m0, %0"
                     : "=&s"(keep) : "v"(off[0]), "v"(off[1]), "s"(base), "s"(lds), "s"(step) : "memory", "scc");
    else {
        static_assert(N == 4, "");
        asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %6\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %5\n\ts_add_u32 m0, m0, %7\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %2, %5\n\t"
                     "s_add_u32 m0, m0, %7\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %3, %5\n\ts_add_u32 m0, m0, %7\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %4, %5\n\ts_mov_b32 m0, %0"
                     : "=&s"(keep) : "v"(off[0]), "v"(off[1]), "v"(off[2]), "v"(off[3]), "s"(base), "s"(lds), "s"(step) : "memory", "scc");
    }
}
// the same with one lane offset and a base that moves on by `rows` bytes
template <int N>
__device__ __forceinline__ void glds16_rows(const void *base, uint32_t off, uint32_t rows, uint32_t lds) {
    unsigned keep;
    uint64_t b = (uint64_t)base;
    if constexpr (N == 1)
        asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %3\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %2, %1\n\ts_mov_b32 m0, %0" : "=&s"(keep), "+s"(b) : "v"(off), "s"(lds) : "memory");
    else
#pragma unroll
        for (int i = 0; i < N; i += 2) {
            uint64_t b2 = b + rows;
            asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %4\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %3, %1\n\ts_add_u32 m0, m0, 0x400\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %3, %2\n\ts_mov_b32 m0, %0"
                         : "=&s"(keep) : "s"(b), "s"(b2), "v"(off), "s"(lds + i * 1024) : "memory", "scc");
            b = b2 + rows;
        }
}
__device__ __forceinline__ uint32_t lds_address(const void *p) { return (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) unsigned char *)p; }
template <int DP> struct KPlace { __device__ __forceinline__ int operator()(int row, int c) const { return k_place<DP>(row, c); } };
template <int DP> struct VPlace { __device__ __forceinline__ int operator()(int row, int c) const { return v_place<DP>(row, c); } };

// ---- tiles: 128 rows, tiles of 64 keys --------------------------------------------------------------------------------------------------
template <class T, int DP, bool DMA>
__global__ __launch_bounds__(256, 2) void attn_tile_kernel(const AttnArgs a) {
    constexpr int BM = 128, KT = 64, TILE = KT * DP * 2;
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];      // [2][K | V]
    const uint32_t items = gridDim.x;
    // neighbouring items (tiles of one key head) on one XCD: it takes every eighth workgroup
    const uint32_t per = items / 8, xcd = blockIdx.x & 7, item = blockIdx.x < per * 8 ? xcd * per + (blockIdx.x >> 3) : blockIdx.x;
    const uint32_t kvh = item / a.slots, slot = a.slots - 1 - item % a.slots;          // later tiles, that tend to see more keys, first: 8192 tokens 292 -> 286 us, 96 texts 22.9 -> 21.2
    int t0, t1;
    const int b = find_seq(a, slot, BM, t0, t1);
    const Seq s = seq_of(a, b, t0, t1);
    const int64_t row0 = ((int64_t)slot - (s.q0 * a.group / BM + b)) * BM;
    if (row0 < 0 || row0 >= (int64_t)s.nq * a.group) return;
    const int t = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(t >> 6);
    const Range g = range_of(a, s, row0, row0 + BM);
    // Up to 32 sinks share a tile with the window's first 32 keys: tile 0, of two blocks that begin at 0 and at g.begin. The tiles behind begin at w0.
    const bool mixed = g.first > 0 && g.first <= 32;
    const int n_first = (g.first + KT - 1) / KT, w0 = g.begin + (mixed ? 32 : 0), n = n_first + max(0, g.end - w0 + KT - 1) / KT;
    const Bounds own = bounds_of(a, s, row0 + wave * 32, row0 + wave * 32 + 32), all = bounds_of(a, s, row0, row0 + BM);
    const T *kb = (const T *)a.k + (uint64_t)s.k0 * a.k_stride + (uint64_t)kvh * a.k_head, *vb = (const T *)a.v + (uint64_t)s.k0 * a.v_stride + (uint64_t)kvh * a.v_head;
    auto start_of = [&](int i) { return i < n_first ? i * KT : w0 + (i - n_first) * KT; };
    auto limit_of = [&](int i) { return i < n_first ? g.first : g.end; };
    // whole tiles: the lane's offsets from a base that moves on with the tiles
    constexpr int N = KT * DP / 8 / 256, STEP = 256 / (DP / 8);
    uint32_t off_k[N], off_v[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int row = i * STEP + t / (DP / 8), x = t % (DP / 8);
        off_k[i] = ((uint32_t)row * (uint32_t)a.k_stride + k_place<DP>(row, x) * 8) * 2;
        off_v[i] = ((uint32_t)row * (uint32_t)a.v_stride + v_place<DP>(row, x) * 8) * 2;
    }
    const uint32_t lds0 = (uint32_t)__builtin_amdgcn_readfirstlane((int)(lds_address(smem) + wave * 1024));
    const T *kn = kb + (n_first ? 0 : (uint64_t)w0 * a.k_stride), *vn = vb + (n_first ? 0 : (uint64_t)w0 * a.v_stride);       // the next tile's
    const uint64_t k_step = (uint64_t)KT * a.k_stride, v_step = (uint64_t)KT * a.v_stride;
    const bool whole = a.dim == DP;
    auto fetch = [&](int i) {
        const int last = min(KT, limit_of(i) - start_of(i)) - 1;
        if (mixed && i == 0) {              // half of the threads a block
            const int b = wave >> 1, first = b ? g.begin : 0, last_b = (b ? min(32, g.end - g.begin) : g.first) - 1;
            unsigned char *Ks = smem + b * (TILE / 2);
            if (last_b >= 0) {
                stage<T, DP, 32, 128, DMA>(Ks, kb + (uint64_t)first * a.k_stride, a.k_stride, last_b, a.dim, t & 127, KPlace<DP>());
                stage<T, DP, 32, 128, DMA>(Ks + TILE, vb + (uint64_t)first * a.v_stride, a.v_stride, last_b, a.dim, t & 127, VPlace<DP>());
            }
        } else if (DMA && whole && last == KT - 1) {
            const uint32_t to = lds0 + (i & 1) * 2 * TILE;
            glds16_n(uniform_ptr((const unsigned char *)kn), off_k, to, 4096);
            glds16_n(uniform_ptr((const unsigned char *)vn), off_v, to + TILE, 4096);
        } else {
            unsigned char *Ks = smem + (i & 1) * 2 * TILE;
            stage<T, DP, KT, 256, DMA>(Ks, kn, a.k_stride, last, a.dim, t, KPlace<DP>());
            stage<T, DP, KT, 256, DMA>(Ks + TILE, vn, a.v_stride, last, a.dim, t, VPlace<DP>());
        }
        if (i + 1 == n_first) { kn = kb + (uint64_t)w0 * a.k_stride; vn = vb + (uint64_t)w0 * a.v_stride; }
        else { kn += k_step; vn += v_step; }
    };
    if (DMA && a.dim < DP) {
        for (int e = t; e < 4 * TILE / 16; e += 256) *reinterpret_cast<u32x4 *>(smem + e * 16) = u32x4{0, 0, 0, 0};
        __syncthreads();
    }
    bool spoiled = false;
    if (n > 0) fetch(0);
    Rows<T, DP> rows;
    rows.init(a, s, kvh, row0 + wave * 32);
    // Tiles [plain0, plain1) are whole and every row of the workgroup sees all of each: no masks, no looking through, no arithmetic but the rows'
    // (8192 tokens, 2048 keys each, 32 over 8 heads of 128: 270 -> 266 us; of 32: 125 -> 120 us)
    const int seen = min(all.hi_min, g.end) - w0;
    const int plain0 = n_first + max(0, (all.lo_max - w0 + KT - 1) / KT), plain1 = DMA && whole && seen > 0 ? n_first + seen / KT : 0;
    for (int i = 0; i < n; ++i) {
        if (i >= plain0)
            for (; i + 1 < plain1; ++i) {
                asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
                const unsigned char *Ks = smem + (i & 1) * 2 * TILE;
                f32x16 sc[KT / 32];
                typename Rows<T, DP>::V8 p[KT / 32][2];
                rows.scores(Ks, sc, [&] {
                    const uint32_t to = lds0 + (~i & 1) * 2 * TILE;
                    glds16_n(uniform_ptr((const unsigned char *)kn), off_k, to, 4096);
                    glds16_n(uniform_ptr((const unsigned char *)vn), off_v, to + TILE, 4096);
                    kn += k_step; vn += v_step;
                });
                rows.softmax(a, sc, p, {0, 0}, {0, 0}, false);
                rows.values(Ks + TILE, p);
            }
        // this tile has arrived, for every wave; nobody reads the other buffer any more
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
        if (i + 1 < n) fetch(i + 1);
        unsigned char *Ks = smem + (i & 1) * 2 * TILE;
        const int j = start_of(i), limit = limit_of(i);
        const bool two = mixed && i == 0;
        if (two || !(j + KT <= min(all.hi_min, limit) && (j >= all.lo_max || j + KT <= (int)a.sinks))) {        // some row of the workgroup sees it in part
            if (__builtin_expect(find_values<T, TILE>(Ks + TILE, t & 63), 0)) {       // (every wave looks through all of it: all find the same)
                __syncthreads();
                clear_values<T, 256>(Ks + TILE, TILE, t);
                __syncthreads();
                spoiled = true;
            }
        }
        if (j < own.hi_max && (j + KT > own.lo_min || j < (int)a.sinks)) {
            const bool masked = two || !(j + KT <= min(own.hi_min, limit) && (j >= own.lo_max || j + KT <= (int)a.sinks));
            f32x16 sc[KT / 32];
            typename Rows<T, DP>::V8 p[KT / 32][2];
            rows.scores(Ks, sc, [] {});
            rows.softmax(a, sc, p, {j, two ? g.begin : j + 32}, {limit, two ? g.end : limit}, masked);
            rows.values(Ks + TILE, p);
        }
    }
    if (spoiled) { rows.spoil(a, vb, 0, g.first, g.first); rows.spoil(a, vb, g.begin, g.end, g.end); }
    const float total = half_sum(rows.l);
    if (!rows.live) return;
#pragma unroll
    for (int t2 = 0; t2 < DP / 32; ++t2) rows.store(a, s, rows.o[t2], t2, total);
    if (rows.lane < 32) rows.store_lse(a, s, total);
}

// ---- split: 32 rows, every wave its own blocks of 32 keys, every workgroup its own part of them ------------------------------------------------
template <class T, int DP, bool DMA>
__global__ __launch_bounds__(256, 2) void attn_split_kernel(const AttnArgs a) {
    constexpr int BM = 32, KT = 32, TILE = KT * DP * 2;
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];      // [4 waves][K | V]; then the waves' sums
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    // Items of work: (sequence, tile of its rows, part of its keys) x key head, counted off over the sequences, 64 of them at a time in a table: a
    // workgroup takes every gridDim.x-th of them, so that short sequences cost what they are.
    struct Table {
        int64_t q0[64], k0[64];
        int nq[64], nk[64], parts[64];
        uint32_t begin[64], end[64];             // items of sequences base .. : [begin, end)
        uint32_t first[64], listed[64];          // places of a key head's parts and listed rows
        uint32_t parts_before, rows_before, fewer, pad;        // places and listed rows of the sequences before base + 64
    };
    static_assert(sizeof(Table) == 64 * 44 + 16, "");
    Table &table = *reinterpret_cast<Table *>(smem + 8 * TILE + 1024);
    // A sequence is wanted in so many parts; `fewer` of these are one, where the places would not do for all: then its rows that are cut have two parts at
    // least, and 2 / fewer of what was wanted at most.
    constexpr uint32_t MOST = 1u << 24;            // (more than any room: counts stop there, and 64 of them and MOST are below 2^32)
    auto wanted = [&](const Seq &s) {
        int64_t seen = s.nk;
        if (a.left >= 0 && a.right >= 0) seen = min(seen, (int64_t)a.left + a.right + 1 + BM + 64 + (int64_t)a.sinks);
        return min(a.splits, max(1u, ((uint32_t)((seen + 31) >> 5) + a.chunk - 1) / a.chunk));
    };
    auto places = [&](const Seq &s, uint32_t parts) { return parts > 1 ? (uint32_t)min((int64_t)s.nq * a.group * parts, (int64_t)MOST) : 0u; };
    if (a.coarser) {                               // (every workgroup finds the same number)
        uint64_t sum = 0;
        for (int64_t b = threadIdx.x; b < (int64_t)a.seqs; b += 256) {
            const Seq s = seq_at(a, (int)b, a.cu[b], a.cu[b + 1]);
            sum += places(s, wanted(s));
        }
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) sum += (uint64_t)(uint32_t)__shfl_xor((int)(sum >> 32), o) << 32 | (uint32_t)__shfl_xor((int)sum, o);
        uint64_t *sums = reinterpret_cast<uint64_t *>(smem);
        if (lane == 0) sums[wave] = sum;
        __syncthreads();
        if (threadIdx.x == 0) {
            const uint64_t f = (2 * (sums[0] + sums[1] + sums[2] + sums[3]) + a.room - 1) / a.room;
            table.fewer = f < 1 ? 1u : f > 64 ? 64u : (uint32_t)f;           // (64: no sequence has more)
        }
        __syncthreads();
    } else if (wave == 0) table.fewer = 1;
    auto running = [&](auto &x) {                  // sums over the lanes up to this one, side by side
#pragma unroll
        for (int o = 1; o < 64; o <<= 1)
#pragma unroll
            for (uint32_t &v : x) { const uint32_t u = (uint32_t)__shfl_up((int)v, o); v += lane >= o ? u : 0u; }
    };
    auto count = [&](int base) {          // by wave 0; the items of 64 sequences
        const int b = base + lane;
        Seq s = {0, 0, 0, 0};
        if (b < (int)a.seqs) s = seq_at(a, b, a.cu[b], a.cu[b + 1]);
        const int64_t rows = (int64_t)s.nq * a.group;
        const uint32_t tiles = (uint32_t)((rows + BM - 1) / BM);          // (below 2^26: 64 times that fits)
        uint32_t parts = 1, items = tiles, end;
        if (a.splits > 1) {
            parts = table.fewer == 1 ? wanted(s) : (wanted(s) + table.fewer - 1) / table.fewer;
            const uint32_t p = places(s, parts);
            uint32_t r = parts > 1 ? (uint32_t)rows : 0u;
            items = tiles * parts;
            uint32_t sums[3] = {p, r, items};
            running(sums);
            const uint32_t p_end = (base ? table.parts_before : 0u) + sums[0];
            if (__any(p_end > a.room)) {           // (only where cu is out of order: what has no places is not cut)
                if (p_end > a.room) { parts = 1; r = 0; items = tiles; }
                sums[1] = r; sums[2] = items;
                running(sums);
            }
            const uint32_t r_end = (base ? table.rows_before : 0u) + sums[1];
            end = sums[2];
            table.first[lane] = p_end - p; table.listed[lane] = r_end - r;
            if (lane == 63) { table.parts_before = min(p_end, MOST); table.rows_before = r_end; }
        } else {
            uint32_t sums[1] = {items};
            running(sums);
            end = sums[0];
        }
        table.q0[lane] = s.q0; table.k0[lane] = s.k0; table.nq[lane] = s.nq; table.nk[lane] = s.nk; table.parts[lane] = (int)parts;
        table.begin[lane] = end - items; table.end[lane] = end;
    };
    int base = 0;
    uint32_t before = 0;                 // items of the sequences before base
    if (wave == 0) count(0);
    __syncthreads();
    for (uint32_t id = blockIdx.x, next;; id = next) {
    next = id + gridDim.x;
    // (heads in turn, shifted from item to item: an XCD, which takes every eighth workgroup, sees all of them)
    const uint32_t item = id / a.kv_heads, kvh = (id + (item >> 1)) % a.kv_heads;
    while (item - before >= table.end[63]) {
        before += table.end[63];
        base += 64;
        if (base >= (int)a.seqs) {
            if (a.splits > 1 && blockIdx.x == 0 && threadIdx.x == 0) *reinterpret_cast<uint32_t *>(a.part) = table.rows_before;
            return;
        }
        __syncthreads();
        if (wave == 0) count(base);
        __syncthreads();
    }
    const int at_lane = __ffsll((unsigned long long)__ballot(table.end[lane] > item - before)) - 1;
    const int within = __builtin_amdgcn_readfirstlane((int)(item - before - table.begin[at_lane])), parts = __builtin_amdgcn_readfirstlane(table.parts[at_lane]), split = within % parts;
    Seq s;
    s.q0 = uniform64(table.q0[at_lane]); s.k0 = uniform64(table.k0[at_lane]);
    s.nq = __builtin_amdgcn_readfirstlane(table.nq[at_lane]); s.nk = __builtin_amdgcn_readfirstlane(table.nk[at_lane]);
    const int64_t row0 = (int64_t)(within / parts) * BM;
    Rows<T, DP> rows;
    rows.init(a, s, kvh, row0);
    unsigned char *Qs = smem + 8 * TILE + 1024 + sizeof(Table);          // the queries' fragments, the same for all four waves (registers for them would spill)
    if (wave == 0)
#pragma unroll
        for (int i = 0; i < DP / 16; ++i) *reinterpret_cast<typename Rows<T, DP>::V8 *>(Qs + i * 1024 + rows.lane * 16) = rows.q[i];
    __syncthreads();
    const Range g = range_of(a, s, row0, row0 + BM);
    const int n_first = (g.first + KT - 1) / KT, n = n_first + (g.end - g.begin + KT - 1) / KT;
    const int i0 = (int)((int64_t)n * split / parts), i1 = (int)((int64_t)n * (split + 1) / parts);
    const Bounds own = bounds_of(a, s, row0, row0 + BM);
    const T *kb = (const T *)a.k + (uint64_t)s.k0 * a.k_stride + (uint64_t)kvh * a.k_head, *vb = (const T *)a.v + (uint64_t)s.k0 * a.v_stride + (uint64_t)kvh * a.v_head;
    unsigned char *Ks = smem + wave * 2 * TILE, *Vs = Ks + TILE;
    auto start_of = [&](int i) { return i < n_first ? i * KT : g.begin + (i - n_first) * KT; };
    auto limit_of = [&](int i) { return i < n_first ? g.first : g.end; };
    // Whole blocks: DP / 16 transfers of 512 / DP rows each. K's exchange of places repeats after DP / 32 of them, V's is the same in all: so many lane
    // offsets, and bases that move on by rows.
    constexpr int RPT = 512 / DP, VAR = DP / 32;
    uint32_t off_k[VAR], off_v;
    {
        const int x = rows.lane % (DP / 8), r = rows.lane / (DP / 8);
#pragma unroll
        for (int i = 0; i < VAR; ++i) off_k[i] = ((uint32_t)(i * RPT + r) * (uint32_t)a.k_stride + k_place<DP>(i * RPT + r, x) * 8) * 2;
        off_v = ((uint32_t)r * (uint32_t)a.v_stride + v_place<DP>(r, x) * 8) * 2;
    }
    const uint32_t lds_k = (uint32_t)__builtin_amdgcn_readfirstlane((int)lds_address(Ks)), lds_v = lds_k + TILE;
    const bool whole = a.dim == DP;
    auto fetch_k = [&](int i) {
        const int j = start_of(i), last = min(KT, limit_of(i) - j) - 1;
        const T *p = kb + (uint64_t)j * a.k_stride;
        if (DMA && whole && last == KT - 1) {
            glds16_n(uniform_ptr((const unsigned char *)p), off_k, lds_k, 1024);
            glds16_n(uniform_ptr((const unsigned char *)(p + (uint64_t)(VAR * RPT) * a.k_stride)), off_k, lds_k + VAR * 1024, 1024);
        } else stage<T, DP, KT, 64, DMA>(Ks, p, a.k_stride, last, a.dim, rows.lane, KPlace<DP>());
    };
    auto fetch_v = [&](int i) {
        const int j = start_of(i), last = min(KT, limit_of(i) - j) - 1;
        const T *p = vb + (uint64_t)j * a.v_stride;
        if (DMA && whole && last == KT - 1) {
#pragma unroll
            for (int u = 0; u < 2; ++u)
                glds16_rows<VAR>(uniform_ptr((const unsigned char *)(p + (uint64_t)(u * VAR * RPT) * a.v_stride)), off_v, (uint32_t)a.v_stride * (RPT * 2), lds_v + u * VAR * 1024);
        } else stage<T, DP, KT, 64, DMA>(Vs, p, a.v_stride, last, a.dim, rows.lane, VPlace<DP>());
    };
    if (DMA && a.dim < DP) {
        for (int e = rows.lane; e < 2 * TILE / 16; e += 64) *reinterpret_cast<u32x4 *>(Ks + e * 16) = u32x4{0, 0, 0, 0};
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    }
    // K's next block is fetched while this one's values are multiplied, V's next while the next scores are: each wait leaves the other's loads (one
    // per 64 lanes x 16 bytes: DP / 16 of them) in flight. (With a head smaller than DP some are left out: there all are waited for.)
    auto arrived = [&](bool all) {
        if (DMA && whole && !all) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(DP / 16) : "memory");
        else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_wave_barrier();
    };
    bool spoiled = false;
    if (i0 + wave < i1) { fetch_k(i0 + wave); fetch_v(i0 + wave); }
    for (int i = i0 + wave; i < i1; i += 4) {
        const int j = start_of(i), limit = limit_of(i);
        const bool masked = !(j + KT <= min(own.hi_min, limit) && (j >= own.lo_max || j + KT <= (int)a.sinks)), more = i + 4 < i1;
        f32x16 sc[1];
        typename Rows<T, DP>::V8 p[1][2];
        arrived(false);                       // K
        rows.scores_lds(Ks, Qs, sc[0]);
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        if (more) fetch_k(i + 4);
        rows.softmax(a, sc, p, {j}, {limit}, masked);
        arrived(!more);                       // V
        if (masked && __builtin_expect(find_values<T, TILE>(Vs, rows.lane), 0)) {
            clear_values<T, 64>(Vs, TILE, rows.lane);
            wave_lds_order();
            spoiled = true;
        }
        rows.values(Vs, p);
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        if (more) fetch_v(i + 4);
    }
    if (spoiled)
        for (int i = i0 + wave; i < i1; i += 4) rows.spoil(a, vb, start_of(i), min(start_of(i) + KT, limit_of(i)), limit_of(i));
    // the four waves' parts, in their order: statistics first, then the sums, 32 features at a time
    float *stat = reinterpret_cast<float *>(smem + 8 * TILE);       // [4][32][2]
    const float part = half_sum(rows.l);
    if (rows.lane < 32) { stat[(wave * 32 + rows.lane) * 2] = rows.m; stat[(wave * 32 + rows.lane) * 2 + 1] = part; }
    __syncthreads();
    float top = NEG_INF, total = 0.0f;
#pragma unroll
    for (int w = 0; w < 4; ++w) top = fmaxf(top, stat[(w * 32 + (rows.lane & 31)) * 2]);
    const float base = top == NEG_INF ? 0.0f : top;
#pragma unroll
    for (int w = 0; w < 4; ++w) total += stat[(w * 32 + (rows.lane & 31)) * 2 + 1] * __builtin_amdgcn_exp2f(stat[(w * 32 + (rows.lane & 31)) * 2] - base);
    const float mine = __builtin_amdgcn_exp2f(rows.m - base);
    // (every wave's tiles are done with at the barrier above: their place takes the sums, 32 features of which each wave adds up)
    float *sums = reinterpret_cast<float *>(smem);                  // [4 waves][DP / 32][16][64]
#pragma unroll
    for (int t = 0; t < DP / 32; ++t)
#pragma unroll
        for (int r = 0; r < 16; ++r) sums[((wave * (DP / 32) + t) * 16 + r) * 64 + rows.lane] = rows.o[t][r] * mine;
    __syncthreads();
    const uint32_t r = (uint32_t)row0 + (rows.lane & 31), place = kvh * a.room + table.first[at_lane] + r * (uint32_t)parts + split;
    rows.m = top;
    if (wave == 0 && rows.live && rows.lane < 32) {
        if (parts > 1) {
            float *stats = a.stats(DP) + (uint64_t)place * 2;
            stats[0] = top; stats[1] = total;
            const uint64_t at = (uint64_t)(s.q0 + rows.token) * a.heads + rows.head;
            if (split == 0) a.list()[(uint64_t)kvh * a.list_room + table.listed[at_lane] + r] = u32x4{(uint32_t)at, (uint32_t)(at >> 32), place, (uint32_t)parts};
        } else rows.store_lse(a, s, total);
    }
    if (wave < DP / 32 && rows.live) {
        f32x16 o;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            float v = 0.0f;
#pragma unroll
            for (int w = 0; w < 4; ++w) v += sums[((w * (DP / 32) + wave) * 16 + r) * 64 + rows.lane];
            o[r] = v;
        }
        if (parts == 1) rows.store(a, s, o, wave, total);
        else {
            float *dst = a.sums() + (uint64_t)place * DP + wave * 32 + (rows.lane >> 5) * 4;
#pragma unroll
            for (int gq = 0; gq < 4; ++gq) {
                f32x4 e;
#pragma unroll
                for (int x = 0; x < 4; ++x) e[x] = o[4 * gq + x];
                *reinterpret_cast<f32x4 *>(dst + gq * 8) = e;
            }
        }
    }
    if (next < id) {                     // (only where cu is out of order: the items of valid sequences are fewer than 2^32)
        if (a.splits > 1 && blockIdx.x == 0 && threadIdx.x == 0) *reinterpret_cast<uint32_t *>(a.part) = 0;
        return;
    }
    __syncthreads();                     // the sums' place is the next item's tiles'
    }
}

// the parts of the listed rows, in their order: one wave a row
template <class T, int DP>
__global__ __launch_bounds__(256) void attn_join_kernel(const AttnArgs a) {
    const int lane = threadIdx.x & 63;
    const uint32_t used = *reinterpret_cast<const uint32_t *>(a.part);
    const float *sums = a.sums(), *stats = a.stats(DP);
    for (uint32_t e = blockIdx.x * 4 + (threadIdx.x >> 6); e < used * a.kv_heads; e += gridDim.x * 4) {
    const u32x4 row = a.list()[(uint64_t)(e / used) * a.list_room + e % used];
    const uint64_t at = (uint64_t)row[1] << 32 | row[0];
    const uint32_t first = row[2], parts = row[3];
    float m = NEG_INF, l = 0.0f;
    if ((uint32_t)lane < parts) { m = stats[(uint64_t)(first + lane) * 2]; l = stats[(uint64_t)(first + lane) * 2 + 1]; }
    float top = m;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o));
    const float base = top == NEG_INF ? 0.0f : top, w = __builtin_amdgcn_exp2f(m - base);
    float total = l * w;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) total += __shfl_xor(total, o);
    constexpr int PER = DP >= 64 ? DP / 64 : 1;
    float v[PER] = {};
    const int d = lane * PER;
    for (uint32_t i = 0; i < parts; i += 8) {          // eight parts' loads on their way at once; those behind the last repeat it with weight 0
        float r[8][PER];
#pragma unroll
        for (int u = 0; u < 8; ++u)
#pragma unroll
            for (int x = 0; x < PER; ++x) r[u][x] = sums[(uint64_t)(first + min(i + u, parts - 1)) * DP + (d < DP ? d : 0) + x];
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            const float c = __shfl(w, (int)min(i + u, 63u));
#pragma unroll
            for (int x = 0; x < PER; ++x) v[x] += i + u < parts ? c * r[u][x] : 0.0f;
        }
    }
    T *dst = (T *)a.out + (at / a.heads) * a.o_stride + (at % a.heads) * a.o_head;
#pragma unroll
    for (int x = 0; x < PER; ++x)
        if ((uint32_t)(d + x) < a.dim) dst[d + x] = (T)(total == 0.0f ? 0.0f : v[x] / total);
    if (a.lse && lane == 0) a.lse[at] = total == 0.0f ? NEG_INF : (top + __builtin_amdgcn_logf(total)) * 0.69314718055994530942f;
    }
}

static int padded_dim(uint32_t d) { return d <= 32 ? 32 : d <= 64 ? 64 : 128; }

struct AttnPlan {
    bool split;
    uint32_t slots, splits, chunk, grid;
    uint32_t room, list_room;  // places of a key head's parts, of its rows that are joined
    bool coarser;              // there may be more parts than places: then they are made larger
    uint64_t workspace;
};
// Which form, and into how many parts the keys are cut. How long each sequence is stands in device memory: the longest may have all keys, or every one of
// them (shared keys). The workspace holds no more than 8 rounds of resident workgroups' parts, 32 rows each; where places for every row at the largest number of
// parts would take more, the kernel counts what the sequences want, and makes parts larger until they fit. (With a place for each 10000 texts of 30 tokens,
// 32 heads x 128, took 298 GiB, now 66 MiB; 900 tokens over 32768 keys, 32 / 8 heads x 128, 915 MiB and 2.53 ms, now 66 and 1.82.)
static AttnPlan plan_attention(const shodh_attention_cfg *c, int cus) {
    AttnPlan p;
    const uint64_t group = c->heads / c->kv_heads, rows = c->q_tokens * group;
    const uint64_t tiles = (rows / 128 + c->seqs) * c->kv_heads;
    p.split = rows <= 32ull * c->seqs || tiles < (uint64_t)cus;
    p.slots = (uint32_t)(rows / (p.split ? 32 : 128) + c->seqs);
    p.splits = p.chunk = p.grid = 1;
    p.room = p.list_room = 0;
    p.coarser = false;
    p.workspace = 0;
    if (p.split) {
        uint64_t seen = c->kv_tokens;
        if (c->left >= 0 && c->right >= 0) {
            const uint64_t w = (uint64_t)c->left + (uint64_t)c->right + 1 + c->sinks + 32;
            if (w < seen) seen = w;
        }
        // A part is 256 KiB of K and V (a workgroup's share of the bandwidth for some 25 us), less where that leaves CUs without work, 128 keys at least.
        const uint64_t groups = (uint64_t)p.slots * c->kv_heads, blocks = ceil_div(seen ? seen : 1, 32), dp = padded_dim(c->head_dim);
        uint64_t chunk = blocks * groups / (4ull * cus);
        const uint64_t most = 2048 / dp;
        chunk = chunk < 4 ? 4 : chunk > most ? most : chunk;
        const uint64_t n = ceil_div(blocks, chunk);
        p.splits = (uint32_t)(n > 64 ? 64 : n);
        p.chunk = (uint32_t)chunk;
        const uint64_t items = groups * p.splits, resident = (uint64_t)cus * (dp == 128 ? 2 : 4);
        p.grid = (uint32_t)(items < resident ? items : resident);
        if (p.splits > 1) {
            const uint64_t most = 8 * resident * 32 / c->kv_heads + 2, each = rows * p.splits;
            p.coarser = each > most;
            p.room = (uint32_t)(p.coarser ? most : each);
            p.list_room = p.room / 2;          // (a row that is joined has two parts or more)
            p.workspace = 16 + c->kv_heads * (16ull * p.list_room + (uint64_t)p.room * (dp + 2) * 4);
        }
    }
    return p;
}

static int check_attention(const shodh_attention_cfg *c) {
    if (!c) { set_error("null argument"); return SHODH_ERR_INVALID; }
    if (c->dtype != SHODH_DTYPE_BF16 && c->dtype != SHODH_DTYPE_FP16) { set_error("attention: dtype %u is neither bf16 nor fp16", c->dtype); return SHODH_ERR_UNSUPPORTED; }
    if (c->heads == 0 || c->kv_heads == 0 || c->heads % c->kv_heads != 0) { set_error("attention: %u heads over %u key heads", c->heads, c->kv_heads); return SHODH_ERR_INVALID; }
    if (c->head_dim == 0 || c->head_dim % 8 != 0 || c->head_dim > 128) { set_error("attention: head_dim %u is no multiple of 8 up to 128", c->head_dim); return SHODH_ERR_UNSUPPORTED; }
    if (!(c->scale == c->scale) || c->scale > 2.0e38f || c->scale < -2.0e38f /* (times log2 e, in f32) */) { set_error("attention: scale is no number, or too large"); return SHODH_ERR_INVALID; }
    if (c->q_tokens > (uint64_t)MOST_KEYS / (c->heads / c->kv_heads) || c->kv_tokens > (1ull << 40) || c->heads > 65535u || c->seqs > 0x3FFFFFFFu || c->sinks > 0x7FFFFFFFu) { set_error("attention: a size is out of range"); return SHODH_ERR_UNSUPPORTED; }
    const uint64_t rows = c->q_tokens * (c->heads / c->kv_heads);
    if (rows / 32 + c->seqs > 0x7FFFFFFFull / c->kv_heads || (rows > 32ull * c->seqs && (rows / 128 + c->seqs) * c->kv_heads >= (1u << 24) /* of 256 threads: a launch has fewer than 2^32 */)) { set_error("attention: too many rows for one launch"); return SHODH_ERR_UNSUPPORTED; }
    return SHODH_OK;
}

template <class T, int DP, bool DMA>
static int launch_attention(const AttnArgs &a, const AttnPlan &p, hipStream_t st) {
    const uint64_t tiles = (uint64_t)p.slots * a.kv_heads;
    if (!p.split) {
        constexpr size_t lds = 4 * 64 * DP * 2;
        SHODH_TRY(ensure_dynamic_lds((const void *)attn_tile_kernel<T, DP, DMA>, lds));
        hipLaunchKernelGGL((attn_tile_kernel<T, DP, DMA>), dim3((uint32_t)tiles), dim3(256), lds, st, a);
        SHODH_HIP_TRY(hipGetLastError());
        return SHODH_OK;
    }
    constexpr size_t lds = 8 * 32 * DP * 2 + 1024 + 64 * 44 + 16 + DP * 64;          // tiles or sums, statistics, the table of sequences, queries
    SHODH_TRY(ensure_dynamic_lds((const void *)attn_split_kernel<T, DP, DMA>, lds));
    hipLaunchKernelGGL((attn_split_kernel<T, DP, DMA>), dim3(p.grid), dim3(256), lds, st, a);
    SHODH_HIP_TRY(hipGetLastError());
    if (p.splits > 1) {
        const uint64_t rows = (uint64_t)a.q_tokens * a.heads, listed = (uint64_t)p.list_room * a.kv_heads, joins = ceil_div(rows < listed ? rows : listed, 4);
        hipLaunchKernelGGL((attn_join_kernel<T, DP>), dim3((uint32_t)(joins < 4096 ? joins : 4096)), dim3(256), 0, st, a);
        SHODH_HIP_TRY(hipGetLastError());
    }
    return SHODH_OK;
}
template <class T, bool DMA>
static int pick_dim(const AttnArgs &a, const AttnPlan &p, hipStream_t st) {
    return a.dim <= 32 ? launch_attention<T, 32, DMA>(a, p, st) : a.dim <= 64 ? launch_attention<T, 64, DMA>(a, p, st) : launch_attention<T, 128, DMA>(a, p, st);
}
template <class T>
static int pick_attention(const AttnArgs &a, const AttnPlan &p, hipStream_t st) {
    // 16-byte pieces straight to LDS: every row and head at a multiple of 16 bytes, a tile's rows within a 32-bit offset
    const bool dma = aligned_to(a.k, 16) && aligned_to(a.v, 16) && ((a.k_stride | a.v_stride | a.k_head | a.v_head) & 7) == 0 && a.k_stride < (1u << 24) && a.v_stride < (1u << 24);
    return dma ? pick_dim<T, true>(a, p, st) : pick_dim<T, false>(a, p, st);
}

}  // namespace shodh

using namespace shodh;

extern "C" {

void shodh_attention_cfg_default(shodh_attention_cfg *cfg) {
    if (!cfg) return;
    memset(cfg, 0, sizeof *cfg);
    cfg->dtype = SHODH_DTYPE_BF16;
    cfg->left = cfg->right = -1;
}

int shodh_window_attention_workspace(int device, const shodh_attention_cfg *cfg, uint64_t *bytes) {
    if (!bytes) { set_error("null argument"); return SHODH_ERR_INVALID; }
    *bytes = 0;
    SHODH_TRY(check_attention(cfg));
    if (cfg->seqs == 0 || cfg->q_tokens == 0) return SHODH_OK;
    *bytes = plan_attention(cfg, compute_units(device)).workspace;
    return SHODH_OK;
}

int shodh_window_attention_device(int device, const shodh_attention_cfg *cfg, const void *d_q, const void *d_k, const void *d_v, const int32_t *d_cu, const int64_t *d_kv_start,
                                  const int32_t *d_kv_len, void *d_out, float *d_lse, void *d_workspace, uint64_t workspace_bytes, void *stream) {
    SHODH_TRY(check_attention(cfg));
    if (cfg->seqs == 0 || cfg->q_tokens == 0) return SHODH_OK;
    if (!d_q || !d_cu || !d_out || (cfg->kv_tokens && (!d_k || !d_v))) { set_error("null argument"); return SHODH_ERR_INVALID; }
    if ((d_kv_start == nullptr) != (d_kv_len == nullptr)) { set_error("attention: kv_start and kv_len come together"); return SHODH_ERR_INVALID; }
    if (!d_kv_start && cfg->kv_tokens != cfg->q_tokens) { set_error("attention: without kv_start and kv_len the keys are those of the queries' tokens (%llu tokens, %llu keys)",
                                                                    (unsigned long long)cfg->q_tokens, (unsigned long long)cfg->kv_tokens); return SHODH_ERR_DIM; }
    const uint64_t d = cfg->head_dim, H = cfg->heads;
    AttnArgs a;
    a.q_head = cfg->q_head_stride ? cfg->q_head_stride : d; a.q_stride = cfg->q_stride ? cfg->q_stride : H * d;
    a.k_head = cfg->k_head_stride ? cfg->k_head_stride : d; a.k_stride = cfg->k_stride ? cfg->k_stride : cfg->kv_heads * d;
    a.v_head = cfg->v_head_stride ? cfg->v_head_stride : d; a.v_stride = cfg->v_stride ? cfg->v_stride : cfg->kv_heads * d;
    a.o_head = cfg->out_head_stride ? cfg->out_head_stride : d; a.o_stride = cfg->out_stride ? cfg->out_stride : H * d;
    // rows of the output that lie over one another: neither [token][head] nor [head][token] with room for each
    if (a.o_head < d || a.o_stride < d || (H > 1 && cfg->q_tokens > 1 && a.o_stride < (H - 1) * a.o_head + d && a.o_head < (cfg->q_tokens - 1) * a.o_stride + d)) {
        set_error("attention: the output's rows overlap"); return SHODH_ERR_DIM;
    }
    if (!aligned_to(d_q, 2) || !aligned_to(d_k, 2) || !aligned_to(d_v, 2) || !aligned_to(d_out, 2) || !aligned_to(d_lse, 4) || !aligned_to(d_cu, 4) || !aligned_to(d_kv_start, 8) ||
        !aligned_to(d_kv_len, 4) || !aligned_to(d_workspace, 16)) {
        set_error("attention: a pointer is not a multiple of its element's size (the workspace: of 16)"); return SHODH_ERR_INVALID;
    }
    const uint64_t n = cfg->q_tokens, kn = cfg->kv_tokens, KV = cfg->kv_heads;
    const Region q(d_q, d * 2, n, a.q_stride * 2, H, a.q_head * 2), out(d_out, d * 2, n, a.o_stride * 2, H, a.o_head * 2), lse(d_lse, n * H * 4),
        in[6] = {q, Region(d_k, d * 2, kn, a.k_stride * 2, KV, a.k_head * 2), Region(d_v, d * 2, kn, a.v_stride * 2, KV, a.v_head * 2), Region(d_cu, (cfg->seqs + 1ull) * 4),
                 Region(d_kv_start, cfg->seqs * 8ull), Region(d_kv_len, cfg->seqs * 4ull)};
    bool bad = may_overlap(out, lse);
    for (const Region &r : in) bad |= (!(&r == in && same_place(out, q)) && may_overlap(out, r)) || may_overlap(lse, r);
    if (bad) { set_error("attention: out or lse overlaps another operand (out may be q itself)"); return SHODH_ERR_INVALID; }
    DeviceScope scope;
    SHODH_TRY(scope.enter(device));
    const AttnPlan p = plan_attention(cfg, compute_units(device));
    const Region work(d_workspace, p.workspace);
    bad = may_overlap(work, out) || may_overlap(work, lse);
    for (const Region &r : in) bad |= may_overlap(work, r);
    if (bad) { set_error("attention: the workspace overlaps another operand"); return SHODH_ERR_INVALID; }
    if (p.workspace && (!d_workspace || workspace_bytes < p.workspace)) {
        set_error("attention: a workspace of %llu bytes is needed (%llu given)", (unsigned long long)p.workspace, (unsigned long long)(d_workspace ? workspace_bytes : 0)); return SHODH_ERR_INVALID;
    }
    a.q = d_q; a.k = d_k; a.v = d_v; a.out = d_out; a.lse = d_lse; a.cu = d_cu; a.kv_start = d_kv_start; a.kv_len = d_kv_len; a.part = (float *)d_workspace;
    a.q_tokens = (int64_t)cfg->q_tokens; a.kv_tokens = (int64_t)cfg->kv_tokens;
    a.heads = cfg->heads; a.kv_heads = cfg->kv_heads; a.group = cfg->heads / cfg->kv_heads; a.shift = (a.group & (a.group - 1)) == 0 ? __builtin_ctz(a.group) : -1; a.dim = cfg->head_dim; a.seqs = cfg->seqs;
    a.slots = p.slots; a.splits = p.splits; a.chunk = p.chunk; a.room = p.room; a.list_room = p.list_room; a.coarser = p.coarser; a.sinks = cfg->sinks; a.left = cfg->left; a.right = cfg->right;
    const float scale = cfg->scale == 0.0f ? 1.0f / __builtin_sqrtf((float)d) : cfg->scale;
    a.scale2 = __builtin_fabsf(scale) * 1.44269504088896340736f;
    a.sign = scale < 0.0f ? 0x80008000u : 0u;
    hipStream_t st = (hipStream_t)stream;
    return cfg->dtype == SHODH_DTYPE_BF16 ? pick_attention<__bf16>(a, p, st) : pick_attention<_Float16>(a, p, st);
}

}  // extern "C"
