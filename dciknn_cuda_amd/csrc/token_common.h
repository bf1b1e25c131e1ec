// What the token operators share: element types, 16-byte pieces of rows that may start at any
// element, ids of 4 or 8 bytes, the running statistics of a softmax, and the launch interface.
#pragma once

#include "common.h"

namespace dcih {

// Element types as they stand in memory; values are computed with in 32 bits.
struct F32 { using raw = float; };
struct F16 { using raw = _Float16; };
struct BF16 { using raw = __bf16; };

// Bytes of an element of type code `dtype` (DCIH_F32, ..), 0 for no such type.
inline int type_bytes(int dtype) { return dtype == 0 ? 4 : dtype == 1 || dtype == 2 ? 2 : 0; }

// ---- what the entry points (token_api.hip) hand to embed.hip and logits.hip --------
// Type codes are DCIH_F32, DCIH_F16, DCIH_BF16; ids are 4 or 8 bytes wide.

constexpr int kMaxTop = 64;       // alternatives of a row
constexpr int kTeacherSlots = 1024;   // slots of a teacher's row
constexpr int kMaxSplits = 64;    // workgroups that share a row

struct LogitArgs {
    const void* z;                // logits: row r at z + r * stride (elements)
    int64_t n, stride, first;     // `first`: the first row of a launch
    int vocab;
    float c2, c2_rest;            // log2(e) / temperature and what it is rounded by
    float inv_t, half_t;          // 1 / temperature, temperature / 2
    const void* ids;              // targets [n], or the teacher's ids [n][slots]
    bool wide_ids;
    int splits, per_split;        // workgroups of a row, 16-byte pieces of each
    float4* stats;                // [n] (max, sum, entropy / ln 2, -) or (max, sum, teacher's max, 1 / teacher's sum)
    float4* part;                 // [n][splits] statistics of splits
    unsigned long long* part_top; // [n][splits][top] their best pieces
    // log probabilities
    int top;
    float *logprobs, *entropy;
    int32_t* top_ids;
    float* top_logprobs;
    // distillation
    const void* teacher;          // [n][slots]
    int teacher_dtype, slots;
    float* losses;
    // gradients
    const float *grad_logprobs, *grad_entropy, *weights;
    void* grad;
    int64_t grad_stride;
};
int logit_splits(int64_t n, int vocab, int dtype);
int logit_stats(LogitArgs a, int dtype, bool distill, hipStream_t s);
int logit_grad(const LogitArgs& a, int dtype, bool distill, hipStream_t s);
bool distill_by_rows(const LogitArgs& a, int dtype);                             // loss and gradient by one workgroup a row
int distill_rows(const LogitArgs& a, int dtype, hipStream_t s);

struct EmbedArgs {
    const void* rows;             // the table, or the gradients of the rows looked up
    int64_t num_rows, stride;     // rows of the table; distance of rows in `rows` (elements)
    int dim;
    const void* ids;
    bool wide_ids;
    int64_t n;                    // ids
    float scale;
    void* out;                    // contiguous
    bool accumulate;              // (gradient) added to what `out` holds
    void* work;
};
int embed_rows(const EmbedArgs& a, int dtype, hipStream_t s);
size_t embed_grad_bytes(int64_t n, int dim, int64_t num_rows);
int embed_grad(const EmbedArgs& a, int dtype, int out_dtype, hipStream_t s);

#if defined(__HIPCC__)

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
// Sixteen bytes at any element's address: rows of odd lengths start on no boundary, and the
// memory system takes such accesses (a wavefront's 1 KB then touches one line more).
typedef uint32_t u32x4_any __attribute__((ext_vector_type(4), aligned(2)));

template <class T> struct Piece {          // one 16-byte piece of a row
    static constexpr int kLen = 16 / (int)sizeof(typename T::raw);
    typedef typename T::raw vec __attribute__((ext_vector_type(kLen)));
    typedef float fvec __attribute__((ext_vector_type(kLen)));

    __device__ static u32x4 load(const typename T::raw* p) {
        return *reinterpret_cast<const u32x4_any*>(p);
    }
    // Rows that are read or written once: not to displace what the caches hold.
    __device__ static u32x4 load_once(const typename T::raw* p) {
        return __builtin_nontemporal_load(reinterpret_cast<const u32x4_any*>(p));
    }
    // Elements [i, i + kLen) of a row of `len`, `fill` beyond its end.
    __device__ static u32x4 load_part(const typename T::raw* row, int i, int len, float fill) {
        vec v;
#pragma unroll
        for (int k = 0; k < kLen; k++) v[k] = i + k < len ? row[i + k] : (typename T::raw)fill;
        return __builtin_bit_cast(u32x4, v);
    }
    __device__ static u32x4 filled(float y) {
        vec v;
#pragma unroll
        for (int k = 0; k < kLen; k++) v[k] = (typename T::raw)y;
        return __builtin_bit_cast(u32x4, v);
    }
    __device__ static void unpack(u32x4 x, float (&z)[kLen]) {
        const fvec f = __builtin_convertvector(__builtin_bit_cast(vec, x), fvec);
#pragma unroll
        for (int k = 0; k < kLen; k++) z[k] = f[k];
    }
    // Rounded to the nearest, ties to even.
    __device__ static u32x4 pack(const float (&z)[kLen]) {
        fvec f;
#pragma unroll
        for (int k = 0; k < kLen; k++) f[k] = z[k];
        return __builtin_bit_cast(u32x4, __builtin_convertvector(f, vec));
    }
    __device__ static void store(typename T::raw* p, u32x4 x) { *reinterpret_cast<u32x4_any*>(p) = x; }
    __device__ static void store_once(typename T::raw* p, u32x4 x) {
        __builtin_nontemporal_store((u32x4_any)x, reinterpret_cast<u32x4_any*>(p));
    }
    __device__ static void store_part(typename T::raw* row, int i, int len, u32x4 x) {
        const vec v = __builtin_bit_cast(vec, x);
#pragma unroll
        for (int k = 0; k < kLen; k++)
            if (i + k < len) row[i + k] = v[k];
    }
};

// A row of logits as whole 16-byte pieces and, as one more, what is left behind them.
template <class T> struct Row {
    using raw_t = typename T::raw;
    static constexpr int kLen = Piece<T>::kLen;
    const raw_t* z;
    int pieces, len;
    bool odd;           // elements of two bytes that start within a word
    __device__ Row(const void* logits, int64_t row, int64_t stride, int len_) : z((const raw_t*)logits + row * stride), len(len_) {
        pieces = len / kLen;
        odd = sizeof(raw_t) == 2 && ((uintptr_t)z & 2);
    }
    // Whole pieces piece, piece + step, .. of each lane, one behind that of the lane before.  Rows within words are
    // read by whole words (by accesses within words: 4.9 TB/s instead of 6.0) and shifted; the first and the
    // last word of a run are shared with what stands beside it.
    template <int U> __device__ void load_runs(int piece, int step, u32x4 (&raw)[U]) const {
        if (sizeof(raw_t) == 4 || !odd) {
#pragma unroll
            for (int u = 0; u < U; u++) raw[u] = Piece<T>::load_once(z + (int64_t)(piece + u * step) * kLen);
            return;
        }
        // (rounded down as a number: a scalar load drops the low bits of its base and of its offset each, so a base of
        // z - 1 with the odd z in a register would miss by a word)
        const uint32_t* w = (const uint32_t*)((uintptr_t)z & ~(uintptr_t)3);
        const int behind = __builtin_amdgcn_readfirstlane(piece) + kWave;        // the piece behind the last lane's
        uint32_t last[U];
#pragma unroll
        for (int u = 0; u < U; u++) {
            raw[u] = __builtin_nontemporal_load((const u32x4_any*)(w + (int64_t)(piece + u * step) * 4));
            last[u] = w[(int64_t)(behind + u * step) * 4];
        }
#pragma unroll
        for (int u = 0; u < U; u++) {
            const u32x4 x = raw[u];
            const uint32_t next = (uint32_t)__builtin_amdgcn_update_dpp((int)last[u], (int)x[0], 0x130, 0xf, 0xf, false);      // wave_shl:1
            raw[u] = u32x4{__builtin_amdgcn_alignbit(x[1], x[0], 16), __builtin_amdgcn_alignbit(x[2], x[1], 16),
                           __builtin_amdgcn_alignbit(x[3], x[2], 16), __builtin_amdgcn_alignbit(next, x[3], 16)};
        }
    }
    // Any piece: what is left for the one behind the whole ones, -inf beyond the row.
    __device__ u32x4 load(int piece) const {
        if (piece < pieces) return Piece<T>::load_once(z + (int64_t)piece * kLen);
        return Piece<T>::load_part(z, piece == pieces ? pieces * kLen : len, len, -__builtin_huge_valf());
    }
    // To the same place of another row.
    __device__ void store(raw_t* to, int piece, u32x4 x) const {
        if (piece < pieces) Piece<T>::store_once(to + (int64_t)piece * kLen, x);
        else Piece<T>::store_part(to, pieces * kLen, len, x);
    }
};

__device__ inline int64_t id_at(const void* ids, bool wide, int64_t i) {
    return wide ? ((const int64_t*)ids)[i] : (int64_t)((const int32_t*)ids)[i];
}

// The same for an index that all lanes share and ids that the kernel does not write: through the scalar cache.
__device__ inline int64_t id_of_all(const void* ids, bool wide, int64_t i) {
    return wide ? ((const __attribute__((address_space(4))) int64_t*)ids)[i] : (int64_t)((const __attribute__((address_space(4))) int32_t*)ids)[i];
}

__device__ inline float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }   // v_exp_f32, 1 ulp
__device__ inline float log2_fast(float x) { return __builtin_amdgcn_logf(x); }    // v_log_f32, 1 ulp

constexpr float kNoLogit = -__builtin_huge_valf();
constexpr float kLn2 = 0.693147180559945309f;
constexpr float kLog2e = 1.44269504088896341f;

// Below 2^-256 nothing is left in 32 bits: exponents are cut off there wherever they are a
// factor themselves, so that a ruled-out entry adds 0 * -256 and not 0 * -inf.
constexpr float kFloor2 = -256.f;

// Set bits of `mask` below this lane's.
__device__ inline int lanes_below(unsigned long long mask) {
    return __builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0));
}

// What one lane wrote to the wavefront's own part of LDS the others may read after this.  (It orders the compiler:
// the wavefront's accesses to LDS are in their order as they are.)
__device__ inline void wave_fence() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// What lane (this one ^ O) holds, without the wait for LDS that lane_xor's swizzles by 4, 8 and 16 are.
template <int O> __device__ inline uint32_t other_lane(uint32_t v) {
    if constexpr (O == 4) {           // of 8 lanes in reverse, each four in reverse
        return (uint32_t)__builtin_amdgcn_mov_dpp(__builtin_amdgcn_mov_dpp((int)v, 0x141, 0xf, 0xf, true), 0x1B, 0xf, 0xf, true);
    } else if constexpr (O == 8) {    // of 16 lanes by a rotation
        return (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x128, 0xf, 0xf, true);
    } else if constexpr (O == 16) {   // [0] holds the even rows of 16 lanes twice each, [1] the odd ones
        const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
        return lane_id() & 16 ? r[0] : r[1];
    } else {
        return lane_xor_u32<O>(v);
    }
}
template <int O> __device__ inline float other_lane(float v) {
    return __builtin_bit_cast(float, other_lane<O>(__builtin_bit_cast(uint32_t, v)));
}
template <int O> __device__ inline unsigned long long other_lane(unsigned long long v) {
    return (unsigned long long)other_lane<O>((uint32_t)(v >> 32)) << 32 | other_lane<O>((uint32_t)v);
}

__device__ inline float max_of_lanes(float v) {
    v = fmaxf(v, other_lane<32>(v)); v = fmaxf(v, other_lane<16>(v)); v = fmaxf(v, other_lane<8>(v));
    v = fmaxf(v, other_lane<4>(v)); v = fmaxf(v, other_lane<2>(v)); v = fmaxf(v, other_lane<1>(v));
    return v;
}
__device__ inline float sum_of_lanes(float v) {
    v += other_lane<32>(v); v += other_lane<16>(v); v += other_lane<8>(v);
    v += other_lane<4>(v); v += other_lane<2>(v); v += other_lane<1>(v);
    return v;
}

// Running statistics of a softmax over entries z at temperature T, exponents to the base 2
// (c2 = log2(e) / T):  m = max z,  s = sum 2^((z - m) c2),  a = sum (z - m) c2 2^((z - m) c2).
// The difference z - m is formed before the factor: a product that is beyond 32 bits, as the type's
// lowest value gives, is -inf and 2 to it 0, as it should be.  With m = -inf nothing but -inf was seen and s = a = 0; a NaN or +inf leaves s = NaN.
struct Softmax {
    float m, s, a;

    __device__ static Softmax none() { return Softmax{kNoLogit, 0.f, 0.f}; }

    // The statistics of both parts.  (fmaxf(NaN, floor) = floor covers -inf - -inf.)
    __device__ void join(const Softmax& o, float c2) {
        const float top = fmaxf(m, o.m);
        const float d1 = fmaxf((m - top) * c2, kFloor2), d2 = fmaxf((o.m - top) * c2, kFloor2);
        const float f1 = exp2_fast(d1), f2 = exp2_fast(d2);
        a = f1 * (a + d1 * s) + f2 * (o.a + d2 * o.s);
        s = s * f1 + o.s * f2;
        m = top;
    }
    // Adds N entries.
    template <int N, bool kEntropy>
    __device__ void add(const float (&z)[N], float c2) {
        float top = z[0];
#pragma unroll
        for (int k = 1; k < N; k++) top = fmaxf(top, z[k]);
        add<N, kEntropy>(z, top, c2);
    }
    // `top` is the largest of them.  Many are added up by themselves first: a thread has a thousand terms of a long row, and their
    // sum one after the other was twice as far off as one in parts.
    template <int N, bool kEntropy>
    __device__ void add(const float (&z)[N], float top, float c2) {
        constexpr bool kInParts = N > 8;
        top = fmaxf(top, m);
        const float ref = top == kNoLogit ? 0.f : top;
        const float d = fmaxf((m - ref) * c2, kFloor2), f = exp2_fast(d);
        const float a0 = f * (a + d * s), s0 = s * f;
        if (kEntropy) a = kInParts ? 0.f : a0;
        s = kInParts ? 0.f : s0;
        m = top;
#pragma unroll
        for (int k = 0; k < N; k++) {
            const float x = (z[k] - ref) * c2, e = exp2_fast(x);
            s += e;
            if (kEntropy) a = __builtin_fmaf(fmaxf(x, kFloor2), e, a);
        }
        if (kInParts) s += s0;
        if (kInParts && kEntropy) a += a0;
    }
    // Over a wavefront; every lane gets the result.
    template <bool kEntropy>
    __device__ void join_wave(float c2) {
        const float top = max_of_lanes(m), d = fmaxf((m - top) * c2, kFloor2), f = exp2_fast(d);
        if (kEntropy) a = sum_of_lanes(f * (a + d * s));
        s = sum_of_lanes(s * f);
        m = top;
    }
};

#endif  // __HIPCC__
}  // namespace dcih
