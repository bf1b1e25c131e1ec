// Operators on rows of logits z[row][0 .. vocab): log probabilities of given tokens with
// entropies and best alternatives, the loss against a teacher's top logits, and the gradients
// of both by the logits.
//
//   x_v = (z_v - max z) / T,  Z = sum_v exp x_v,  log p_v = x_v - log Z,
//   H   = log Z - sum_v x_v exp(x_v) / Z
//   d/dz_v (g log p_t + h H) = ( g ([v = t] - p_v) - h p_v (log p_v + H) ) / T
//   q_j = softmax over a row's filled slots of t_j / T,  loss = sum_j q_j (log q_j - log p_{id_j})
//   d/dz_v (w loss) = (w / T) (p_v - sum_{j: id_j = v} q_j)
//
// All of them are bound by memory: a row is read once for its statistics (max, sum and, for the
// entropy, weighted sum are kept running per thread and joined at the end), and read and written
// once more for a gradient.  Everything between is in 32 bits; a gradient is rounded once.
#include <algorithm>

#include "../../include/dci_hip.h"
#include "token_common.h"

namespace dcih {
namespace {

constexpr int kThreads = 256;
constexpr int64_t kMaxGrid = 1 << 22; // workgroups of one launch (their threads are counted in 32 bits)
constexpr int kTopWait = 8;          // candidates that a wavefront gathers before it puts them in order
constexpr int kTopRoom = 520;        // room for candidates: those and eight rounds of 64
static_assert(kTopRoom >= kTopWait + 8 * kWave, "room for eight rounds of candidates");

enum { kLogprobs = 0, kLogprobsTop = 1, kDistill = 2 };

typedef unsigned long long u64;

// One entry of a candidate list: larger logits first, ties to the lower index (of an element or a piece).
__device__ inline u64 entry_of(float z, int index) {
    return (u64)f2ord(z + 0.f) << 32 | (0xffffffffu - (uint32_t)index);      // (-0 and 0 tie)
}
__device__ inline float entry_logit(u64 e) { return ord2f((uint32_t)(e >> 32)); }
__device__ inline int entry_index(u64 e) { return (int)(0xffffffffu - (uint32_t)e); }

// One step of a bitonic sort over the lanes, larger ones first: towards runs of SIZE.
template <int SIZE, int STRIDE, class V>
__device__ inline void sort_step(V& v) {
    const V o = other_lane<STRIDE>(v);
    const bool larger = ((lane_id() & STRIDE) == 0) == (SIZE == kWave || (lane_id() & SIZE) == 0);
    v = (o > v) == larger ? o : v;
}
template <int SIZE, int STRIDE, class V>
__device__ inline void sort_steps(V& v) {
    sort_step<SIZE, STRIDE>(v);
    if constexpr (STRIDE > 1) sort_steps<SIZE, STRIDE / 2>(v);
}

// The k-th largest (k = 1 .. 64) of the lanes' values, on every lane.
__device__ inline uint32_t kth_of_lanes(uint32_t v, int k) {
    sort_steps<2, 1>(v); sort_steps<4, 2>(v); sort_steps<8, 4>(v);
    sort_steps<16, 8>(v); sort_steps<32, 16>(v); sort_steps<64, 32>(v);
    return (uint32_t)__builtin_amdgcn_readlane((int)v, k - 1);
}
__device__ inline u64 of_lane(u64 v, int lane) {
    return (u64)(uint32_t)__builtin_amdgcn_readlane((int)(v >> 32), lane) << 32 | (uint32_t)__builtin_amdgcn_readlane((int)v, lane);
}

// The k best pieces a wavefront has met, or elements: lane i holds the i-th best of them.  Candidates wait in
// LDS until there are more than a few, after eight rounds of up to 64 at the latest, so that any order of
// the row and any number of ties is taken.  No entry is 0 (index 2^32 - 1 does not exist).
struct WaveTop {
    u64* wait;         // kTopRoom entries
    int k, count = 0;  // of those that wait
    u64 best = 0;
    u64 least = 0;     // what an entry has to exceed

    __device__ WaveTop(u64* b, int k_) : wait(b), k(k_) {}

    __device__ void push(bool want, u64 e) {
        const u64 mask = __ballot(want && e > least);
        if (mask >> lane_id() & 1) wait[count + lanes_below(mask)] = e;
        count += __popcll(mask);
    }
    // `other`: another list, its best on the last lane.
    __device__ void merge_reversed(u64 other) {
        best = best > other ? best : other;        // the best 64 of both, rising and falling
        sort_steps<kWave, kWave / 2>(best);
    }
    __device__ void settle() {
        wave_fence();
        for (int first = 0; first < count; first += kWave) {
            u64 e = first + lane_id() < count ? wait[first + lane_id()] : 0;
            sort_steps<2, 1>(e); sort_steps<4, 2>(e); sort_steps<8, 4>(e);
            if (count - first > 8) sort_steps<16, 8>(e);               // (the other lanes hold nothing)
            if (count - first > 16) {
                sort_steps<32, 16>(e); sort_steps<64, 32>(e);
            }
            if (of_lane(best, 0)) merge_reversed(__shfl(e, kWave - 1 - lane_id()));
            else best = e;
        }
        wave_fence();
        count = 0;
        least = max(least, of_lane(best, k - 1));
    }
    __device__ void tidy() {
        if (count > kTopWait) settle();
    }
    __device__ int held() const { return min(k, (int)__popcll(__ballot(best != 0))); }
};

__device__ inline float teacher_at(const LogitArgs& a, int64_t i) {
    switch (a.teacher_dtype) {
        case DCIH_F32: return ((const float*)a.teacher)[i];
        case DCIH_F16: return (float)((const _Float16*)a.teacher)[i];
        default: return (float)((const __bf16*)a.teacher)[i];
    }
}

// (z - m) / T - log Z in 32 bits, what is returned of a logit: infinite only where the value itself is beyond them.  (The
// difference of halves holds any two logits; a factor log2(e) / T, as the exponents have, is beyond 1 and would take
// the lowest value to -inf.)
__device__ inline float log_share(float z, float m, float half_t, float log_sum) { return (0.5f * z - 0.5f * m) / half_t - log_sum; }

// 2^((z - m) c2) with what the difference and the product are rounded by made good: a teacher's weight is a factor of all that
// its token adds to a loss and a gradient, and the two roundings of an exponent of 10 would take it 1e-6 from its value.
__device__ inline float power_of(float z, float m, float c2, float c2_rest) {
    const float d = z - m, x = d * c2, e = exp2_fast(x);
    const float b = d - z, lost = (z - (d - b)) - (m + b);             // z - m = d + lost
    const float rest = __builtin_fmaf(d, c2, -x) + __builtin_fmaf(d, c2_rest, lost * c2);
    return e == 0.f ? 0.f : __builtin_fmaf(e, rest * kLn2, e);
}

// Half of q (log q - log p), with the teacher's logit y, its maximum ym, the student's z and zm, `log_ratio` the logarithm of the
// teacher's sum over the student's.  (The weight comes ahead of the temperature: log p may be beyond 32 bits where their product is
// not, and a small weight by a large temperature is not to be 0 times a difference that is infinite.)
__device__ inline float half_loss(float q, float y, float ym, float z, float zm, float inv_t, float log_ratio) {
    const float d = (0.5f * y - 0.5f * ym) - (0.5f * z - 0.5f * zm);
    return q * d * inv_t - 0.5f * q * log_ratio;
}
// A loss from its half.  One that is beyond 32 bits by no more than a sum's rounding is the largest number: q_j that are 1 together
// but for their rounding, all of them of tokens at the type's lowest value, are not to give infinity.
__device__ inline float loss_of_half(float half) {
    return half > 0.5f * __FLT_MAX__ && half <= 0.5f * __FLT_MAX__ * (1.f + 0x1p-18f) ? __FLT_MAX__ : half + half;
}

// Whether a row of logits holds nothing but -inf.
__device__ inline bool nothing_left(const Softmax& f) { return f.m == kNoLogit && f.s == 0.f; }

// The maximum that is kept of a row: -inf for one without entries and for no other (one of nothing
// but NaN keeps 0 beside its sum, NaN).
__device__ inline float kept_max(const Softmax& f) { return nothing_left(f) ? kNoLogit : f.m == kNoLogit ? 0.f : f.m; }

// From the k best pieces of a row by their largest elements (the k best elements are in them: every piece
// before an element's own holds a better one) to its k best elements.  Fewer than k: all that are above -inf.
template <class T>
__device__ void best_of_pieces(const LogitArgs& a, int64_t row, WaveTop& top) {
    using P = Piece<T>;
    const bool have = lane_id() < top.k && top.best;
    const int piece = have ? entry_index(top.best) : 0;
    const u64 last = of_lane(top.best, top.k - 1);
    const float bar = last ? entry_logit(last) : -__FLT_MAX__;
    float x[P::kLen];
    P::unpack(Row<T>(a.z, row, a.stride, a.vocab).load(piece), x);
    top.best = top.least = 0;
#pragma unroll
    for (int k = 0; k < P::kLen; k++) top.push(have && x[k] >= bar, entry_of(x[k], piece * P::kLen + k));
    top.settle();
}

// One wavefront: what is returned of a row of log probabilities.  `top`: its best pieces.
template <class T>
__device__ void finish_logprobs(const LogitArgs& a, int64_t row, const Softmax& f, WaveTop& top, int64_t t, float z_t) {
    const typename T::raw* z = (const typename T::raw*)a.z + row * a.stride;
    const bool none = nothing_left(f);
    const float log_s = logf(f.s);
    const float entropy = none ? 0.f : log_s - f.a / f.s * kLn2;
    if (lane_id() == 0) {
        float lp = 0.f;
        if (t >= a.vocab) lp = __builtin_nanf("");
        else if (t >= 0) lp = none ? kNoLogit : log_share(z_t, f.m, a.half_t, log_s);
        a.logprobs[row] = lp;
        a.entropy[row] = entropy;
        if (a.stats) a.stats[row] = make_float4(kept_max(f), f.s, entropy * kLog2e, 0.f);
    }
    const int k = a.top;
    if (!k) return;
    best_of_pieces<T>(a, row, top);
    int count = top.held();
    int32_t* ids = a.top_ids + row * k;
    float* lps = a.top_logprobs + row * k;
    if (lane_id() < count) {
        const u64 e = top.best;
        ids[lane_id()] = entry_index(e);
        lps[lane_id()] = log_share(entry_logit(e), f.m, a.half_t, log_s);
    }
    // what is ruled out (or no number) follows in order of its index
    const float rest = f.s != f.s ? f.s : kNoLogit;
    for (int first = 0; count < k && first < a.vocab; first += kWave) {
        const int i = first + lane_id();
        const bool gone = i < a.vocab && !((float)z[i] > kNoLogit);
        const u64 mask = __ballot(gone);
        const int at = count + lanes_below(mask);
        if (gone && at < k) {
            ids[at] = i;
            lps[at] = rest;
        }
        count += __popcll(mask);
    }
}

// One wavefront: the loss of a row against its teacher.
template <class T>
__device__ void finish_distill(const LogitArgs& a, int64_t row, const Softmax& f) {
    const typename T::raw* z = (const typename T::raw*)a.z + row * a.stride;
    const int64_t at = row * a.slots;
    Softmax t = Softmax::none();
    bool wrong = false;
    for (int j = lane_id(); j < a.slots; j += kWave) {
        const int64_t id = id_at(a.ids, a.wide_ids, at + j);
        float y[1] = {id < 0 ? kNoLogit : teacher_at(a, at + j)};
        wrong |= id >= a.vocab && y[0] != kNoLogit;
        t.add<1, false>(y, a.c2);
    }
    t.join_wave<false>(a.c2);
    wrong = __ballot(wrong) != 0;
    const bool empty = nothing_left(t), none = nothing_left(f);
    const float share = 1.f / t.s, log_ratio = logf(t.s) - (none ? 0.f : logf(f.s));
    float sum = 0.f;      // of halves
    for (int j = lane_id(); j < a.slots; j += kWave) {
        const int64_t id = id_at(a.ids, a.wide_ids, at + j);
        const float y = id < 0 ? kNoLogit : teacher_at(a, at + j);
        if (y == kNoLogit || id >= a.vocab) continue;
        const float q = power_of(y, t.m, a.c2, a.c2_rest) * share;
        if (!(q == 0.f)) sum += half_loss(q, y, t.m, (float)z[id], none ? 0.f : f.m, a.inv_t, log_ratio);
    }
    sum = loss_of_half(sum_of_lanes(sum));
    wrong |= t.s != t.s;
    if (wrong) sum = __builtin_nanf("");
    if (empty) sum = 0.f;
    if (lane_id() == 0) {
        a.losses[row] = sum;
        if (a.stats) a.stats[row] = make_float4(kept_max(f), wrong ? __builtin_nanf("") : f.s, kept_max(t), share);
    }
}

// Statistics of rows, each by `splits` workgroups.  Threads keep their own running statistics over
// every kRowThreads-th piece; a wavefront keeps its best pieces, too, and what one of them
// finds to be the least that can still be among the best bounds the others' as well.  (Keeping
// elements instead of pieces doubled the arithmetic, which is what bounds this kernel with alternatives.)
// Without alternatives bound by memory: 8192 x 32000 f32 160 us (6.5 TB/s read), 4096 x 50000 bf16 70 us (5.9); with five of
// them by its instructions: 78 us there, 84 for 4096 x 50001 f16, of which every second row starts within a word.
template <class T, int kMode, int kRowThreads, int U>
__global__ __launch_bounds__(kRowThreads, 8) void logit_stats_kernel(LogitArgs a) {
    using P = Piece<T>;
    constexpr int kWaves = kRowThreads / kWave, N = U * P::kLen;
    constexpr bool kTop = kMode == kLogprobsTop;
    __shared__ u64 s_top[kTop ? kWaves * kTopRoom : 1];
    __shared__ u64 s_least;
    __shared__ Softmax s_part[kWaves];
    const int64_t at_row = a.first + blockIdx.x / (uint32_t)a.splits;
    const int split = (int)(blockIdx.x % (uint32_t)a.splits);
    const Row<T> row(a.z, at_row, a.stride, a.vocab);
    const int tid = threadIdx.x, wave = tid / kWave;
    const int end = min(row.pieces + 1, (split + 1) * a.per_split);
    const int64_t t = kMode == kDistill ? -1 : id_of_all(a.ids, a.wide_ids, at_row);
    Softmax f = Softmax::none();
    WaveTop top(s_top + (kTop ? wave * kTopRoom : 0), a.top);
    if (kTop && kWaves > 1) {
        if (tid == 0) s_least = 0;
        __syncthreads();
    }
    bool first = true;
    for (int base = split * a.per_split; base < end; base += kRowThreads * U) {
        u32x4 raw[U];
        if (base + kRowThreads * U <= min(end, row.pieces)) {
            row.load_runs(base + tid, kRowThreads, raw);
        } else {
#pragma unroll
            for (int u = 0; u < U; u++) {
                const int i = base + u * kRowThreads + tid;
                raw[u] = row.load(i < end ? i : row.pieces + 1);
            }
        }
        float x[N], most = kNoLogit, largest[U];
#pragma unroll
        for (int u = 0; u < U; u++) {
            float y[P::kLen];
            P::unpack(raw[u], y);
            largest[u] = y[0];
#pragma unroll
            for (int k = 0; k < P::kLen; k++) {
                x[u * P::kLen + k] = y[k];
                largest[u] = fmaxf(largest[u], y[k]);
            }
            most = fmaxf(most, largest[u]);
        }
        if constexpr (kTop) {
            if (kWaves > 1) top.least = max(top.least, __hip_atomic_load(&s_least, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP));
            // The k-th largest of the lanes' largest values has k pieces at or above it: none
            // below it is among the k best.
            if (first) top.least = max(top.least, (u64)kth_of_lanes(f2ord(most + 0.f), a.top) << 32);
            first = false;
            const float bar = fmaxf(entry_logit(top.least), -__FLT_MAX__);
            if (__any(most >= bar)) {
#pragma unroll
                for (int u = 0; u < U; u++)
                    if (__any(largest[u] >= bar)) top.push(largest[u] >= bar, entry_of(largest[u], base + u * kRowThreads + tid));
                top.tidy();           // (what is best of them bounds what comes)
                if (kWaves > 1 && lane_id() == 0) atomicMax(&s_least, top.least);
            }
        }
        f.add<N, kMode != kDistill>(x, most, a.c2);
    }
    // (asked for now, used at the end)
    const typename T::raw z_t = kMode != kDistill && a.splits == 1 ? row.z[t >= 0 && t < a.vocab ? t : 0] : (typename T::raw)0.f;
    f.join_wave<kMode != kDistill>(a.c2);
    if constexpr (kTop) top.settle();
    if constexpr (kWaves > 1) {
        if (lane_id() == 0) s_part[wave] = f;
        if constexpr (kTop) s_top[wave * kTopRoom + lane_id()] = top.best;
        __syncthreads();
        if (wave) return;
        f = s_part[0];
#pragma unroll
        for (int w = 1; w < kWaves; w++) {
            f.join(s_part[w], a.c2);
            if constexpr (kTop) top.merge_reversed(s_top[w * kTopRoom + kWave - 1 - lane_id()]);
        }
    }
    if (a.splits > 1) {
        const int64_t at = at_row * a.splits + split;
        if (lane_id() == 0) a.part[at] = make_float4(f.m, f.s, f.a, 0.f);
        if (kTop && lane_id() < a.top) a.part_top[at * a.top + lane_id()] = top.best;
        return;
    }
    if constexpr (kMode == kDistill) finish_distill<T>(a, at_row, f);
    else finish_logprobs<T>(a, at_row, f, top, t, (float)z_t);
}

// Joins the splits (up to 64) of a row: one wavefront each.  Bound by waits: 6.2 us for 4 rows of 64 splits with 20
// alternatives, as long as logit_stats_kernel takes for their 131072 bf16 each.
template <class T, int kMode>
__global__ __launch_bounds__(kWave) void logit_join_kernel(LogitArgs a) {
    __shared__ u64 s_top[kMode == kLogprobsTop ? kTopRoom : 1];
    const int64_t row = a.first + blockIdx.x;
    const int lane = lane_id();
    const int64_t t = kMode == kDistill ? -1 : id_of_all(a.ids, a.wide_ids, row);
    Softmax f = Softmax::none();
    if (lane < a.splits) {
        const float4 p = a.part[row * a.splits + lane];
        f.m = p.x; f.s = p.y; f.a = p.z;
    }
    const typename T::raw z_t = kMode == kDistill ? (typename T::raw)0.f : ((const typename T::raw*)a.z + row * a.stride)[t >= 0 && t < a.vocab ? t : 0];
    f.join_wave<kMode != kDistill>(a.c2);
    if constexpr (kMode == kDistill) {
        finish_distill<T>(a, row, f);
    } else {
        WaveTop top(s_top, a.top);
        if constexpr (kMode == kLogprobsTop) {
            const u64* lists = a.part_top + (row * a.splits + min(lane, a.splits - 1)) * a.top;
            // The lists are in order: with k lists or more, the k-th largest of their first entries bounds
            // from below, and where no list has an entry above the bound at a place none has one behind it.
            constexpr int kAhead = 8;
            u64 e[kAhead], next[kAhead];
            auto load = [&](u64 (&x)[kAhead], int p) {
#pragma unroll
                for (int j = 0; j < kAhead; j++) x[j] = lane < a.splits && p + j < a.top ? lists[p + j] : 0;
            };
            load(next, 0);
            for (int p = 0; p < a.top; p += kAhead) {
#pragma unroll
                for (int j = 0; j < kAhead; j++) e[j] = next[j];
                load(next, p + kAhead);
                if (p == 0) {
                    const uint32_t kth = kth_of_lanes((uint32_t)(e[0] >> 32), a.top);
                    if (a.top <= a.splits) top.least = (u64)kth << 32;
                }
                if (!__any(e[0] > top.least)) break;
#pragma unroll
                for (int j = 0; j < kAhead; j++)
                    if (__any(e[j] > top.least)) top.push(e[j] != 0, e[j]);
                top.settle();
            }
            top.settle();
        }
        finish_logprobs<T>(a, row, f, top, t, (float)z_t);
    }
}

// What the slots that name `token` add up to, in their order.  Slots that name the same one get the same bits, and may all
// write what they make of them.  `fours`: slots by fours, those beyond the last named by no token.
__device__ inline float slots_of_token(const int* s_id, const float* s_q, int fours, int token) {
    float sum = 0.f;
#pragma unroll 4
    for (int i = 0; i < fours; i++) {
        const int4 id = reinterpret_cast<const int4*>(s_id)[i];
        const float4 q = reinterpret_cast<const float4*>(s_q)[i];
        sum += id.x == token ? q.x : 0.f;
        sum += id.y == token ? q.y : 0.f;
        sum += id.z == token ? q.z : 0.f;
        sum += id.w == token ? q.w : 0.f;
    }
    return sum;
}

// Gradients by the logits from a row's statistics, one tile of a row per workgroup: nothing is to be joined, so the
// tiles are small and many.  Bound by memory: 8192 x 32000 f32 340 us (6.2 TB/s read and written; 362 with one or four pieces
// a thread instead of two).
template <class T, int kMode, int U>
__global__ __launch_bounds__(kThreads) void logit_grad_kernel(LogitArgs a) {
    using P = Piece<T>;
    constexpr int kTile = kThreads * U;                  // pieces
    constexpr int kOwn = kTeacherSlots / kThreads;
    __shared__ alignas(16) int s_id[kMode == kDistill ? kTeacherSlots : 1];
    __shared__ alignas(16) float s_q[kMode == kDistill ? kTeacherSlots : 1];
    const int64_t at_row = a.first + blockIdx.x / (uint32_t)a.splits;
    const int tile = (int)(blockIdx.x % (uint32_t)a.splits) * kTile, tid = threadIdx.x;
    const Row<T> row(a.z, at_row, a.stride, a.vocab);
    typename T::raw* dz = (typename T::raw*)a.grad + at_row * a.grad_stride;
    const float4 st = a.stats[at_row];
    // What a gradient is made of: dz = p (c0 + c1 log2 p) + at_target, with p = 2^x / sum.  (The sum as a factor: its logarithm
    // in the exponent, a number of 10 to 20, would bring a rounding of 1e-6 into every p.)
    float c0, c1 = 0.f, at_target = 0.f;
    const float log2s = log2_fast(st.y);
    int64_t target = -1;
    bool zero = st.x == kNoLogit;
    if constexpr (kMode == kDistill) {
        c0 = (a.weights ? a.weights[at_row] : 1.f) * a.inv_t;
        zero |= c0 == 0.f || st.z == kNoLogit;
    } else {
        target = id_at(a.ids, a.wide_ids, at_row);
        const float g = a.grad_logprobs && target >= 0 ? a.grad_logprobs[at_row] * a.inv_t : 0.f;
        const float h = a.grad_entropy ? a.grad_entropy[at_row] * a.inv_t : 0.f;
        zero |= g == 0.f && h == 0.f;
        c0 = -(g + h * st.z * kLn2);
        c1 = -h * kLn2;
        at_target = g;
        if (target >= a.vocab && g != 0.f) c0 = __builtin_nanf("");
    }
    const float share0 = c0 / st.y, share1 = c1 / st.y;
    float own_z[kMode == kDistill ? kOwn : 1];
    bool here = false;
    if constexpr (kMode == kDistill) {
        if (!zero) {
            if (tid < 4) s_id[(a.slots - 1) / 4 * 4 + tid] = -1;       // (those beyond the last)
            __syncthreads();
#pragma unroll
            for (int o = 0; o < kOwn; o++) {
                const int j = o * kThreads + tid;
                if (j >= a.slots) break;
                const int64_t id = id_at(a.ids, a.wide_ids, at_row * a.slots + j);
                const float y = teacher_at(a, at_row * a.slots + j);
                const bool in = id >= 0 && id < a.vocab && id / P::kLen >= tile && id / P::kLen < tile + kTile && y != kNoLogit;
                s_id[j] = in ? (int)id : -1;
                s_q[j] = power_of(y, st.z, a.c2, a.c2_rest) * st.w;
                if (in) own_z[o] = (float)row.z[id];       // before it is written over
                here |= in;
            }
        }
        here = __syncthreads_or(here);
    }
#pragma unroll
    for (int u = 0; u < U; u++) {
        const int i = tile + u * kThreads + tid;
        if (i > row.pieces) continue;
        float y[P::kLen];
        if (zero) {
#pragma unroll
            for (int k = 0; k < P::kLen; k++) y[k] = 0.f;
        } else {
            P::unpack(row.load(i), y);
#pragma unroll
            for (int k = 0; k < P::kLen; k++) {
                const float x = (y[k] - st.x) * a.c2, e = exp2_fast(x);
                if constexpr (kMode == kDistill) y[k] = e * share0;
                else y[k] = e * __builtin_fmaf(share1, fmaxf(x - log2s, kFloor2), share0);
            }
            if (kMode != kDistill && target / P::kLen == i) {
#pragma unroll
                for (int k = 0; k < P::kLen; k++) y[k] += i * P::kLen + k == target ? at_target : 0.f;
            }
        }
        row.store(dz, i, P::pack(y));
    }
    if constexpr (kMode == kDistill) {
        if (!here) return;
        __syncthreads();
        // the teacher's tokens
#pragma unroll
        for (int o = 0; o < kOwn; o++) {
            const int j = o * kThreads + tid;
            if (j >= a.slots) break;
            const int id = s_id[j];
            if (id < 0) continue;
            const float q = slots_of_token(s_id, s_q, (a.slots + 3) / 4, id);
            dz[id] = (typename T::raw)(share0 * exp2_fast((own_z[o] - st.x) * a.c2) - c0 * q);
        }
    }
}

// Loss and gradient of a row by one workgroup: the row is read once, kept in registers as it came
// (NV pieces a thread) and written once.  A workgroup goes on to another row as soon as the gradient's
// pieces leave: the next row's loads take their registers and travel beside the stores.  Memory
// operations are waited for in their order and counted where their number is known, so there are no branches about
// them: beyond the row's end a thread reads (and writes, the same values again) the last piece once more.
// Bound by memory: 8192 x 131072 bf16 842 us (5.1 TB/s read and written; a copy reaches 4.8); 1001 x 100003 f16
// 112 us (3.6 TB/s: with four rows a workgroup the first one's loads and the last one's stores are alone).
template <class T, int kRowThreads, int NV>
__global__ __launch_bounds__(kRowThreads) void distill_rows_kernel(LogitArgs a) {
    using P = Piece<T>;
    using raw_t = typename T::raw;
    constexpr int kRowWaves = kRowThreads / kWave;
    __shared__ alignas(16) int s_id[kRowThreads];
    __shared__ alignas(16) float s_q[kRowThreads];
    __shared__ float s_y[kRowThreads];
    __shared__ float s_max[kRowWaves], s_sum[kRowWaves];
    __shared__ float s_loss[kRowWaves];                  // (not s_sum: a wavefront behind may still read that one)
    __shared__ float4 s_teacher;                         // max, 1 / sum, log sum, 0 without one and NaN if its ids or logits are unsound
    const int tid = threadIdx.x, wave = tid / kWave;
    // whole pieces, and behind them less than one whose elements a thread each takes
    const int pieces = a.vocab / P::kLen, end = pieces * P::kLen + tid;
    const uint32_t end_at = (uint32_t)min(end, a.vocab - 1) * (uint32_t)sizeof(raw_t);
    auto row_of = [&](int64_t row) { return (const char*)a.z + row * a.stride * (int64_t)sizeof(raw_t); };
    auto load_end = [&](const char* z) { return *(const raw_t*)(z + end_at); };
    // (the thread's number is made to look new each time: the compiler would keep, and spill, an offset for every piece)
    auto piece_of = [&](int u) {
        int i = tid;
        asm volatile("" : "+v"(i));
        return i + u * kRowThreads;
    };
    auto at_piece = [&](int u, int most) { return (uint32_t)min(piece_of(u), most) * 16u; };
    auto load = [&](const char* z, int u, int most) { return P::load_once((const raw_t*)(z + at_piece(u, most))); };
    // a thread's slot: the id (-1: empty; vocab: beyond it), the teacher's logit and the student's there
    uint32_t id_lo, id_hi;
    uint16_t y_lo, y_hi;
    raw_t there;
    const int id_size = a.wide_ids ? 8 : 4, y_size = a.teacher_dtype == DCIH_F32 ? 4 : 2;
    auto load_slots = [&](int64_t row) {
        const uint32_t j = (uint32_t)min(tid, a.slots - 1);
        const char* id = (const char*)a.ids + row * a.slots * id_size + j * id_size;
        const char* y = (const char*)a.teacher + row * a.slots * y_size + j * y_size;
        id_lo = *(const uint32_t*)id;
        id_hi = *(const uint32_t*)(id + id_size - 4);
        y_lo = *(const uint16_t*)y;
        y_hi = *(const uint16_t*)(y + y_size - 2);
    };
    auto id_of = [&]() {
        const int64_t id = a.wide_ids ? (int64_t)((uint64_t)id_hi << 32 | id_lo) : (int64_t)(int32_t)id_lo;
        return tid >= a.slots || id < 0 ? -1 : (int)min(id, (int64_t)a.vocab);
    };
    auto y_of = [&]() {
        const float y = a.teacher_dtype == DCIH_F16 ? (float)__builtin_bit_cast(_Float16, y_lo)
                                                    : __builtin_bit_cast(float, (uint32_t)y_hi << 16 | (y_size == 4 ? y_lo : 0));
        return id_of() < 0 ? kNoLogit : y;
    };
    auto load_there = [&](const char* z) {
        asm volatile("" : "+v"(id_lo), "+v"(id_hi));         // (not to be waited for before this place)
        const int id = id_of();
        there = ((const raw_t*)z)[id >= 0 && id < a.vocab ? id : 0];
    };
    int64_t row = blockIdx.x;
    const char* z = row_of(row);
    u32x4 raw[NV];
    load_slots(row);
    raw_t raw_end = load_end(z);
    load_there(z);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int u = 0; u < NV; u++) raw[u] = load(z, u, pieces - 1);
    while (true) {
        s_id[tid] = y_of() == kNoLogit ? -1 : id_of();
        s_y[tid] = y_of();
        __syncthreads();
        if (wave == 0) {      // while the row arrives
            Softmax t = Softmax::none();
            bool wrong = false;
            for (int j = lane_id(); j < a.slots; j += kWave) {
                const float y[1] = {s_y[j]};
                wrong |= s_id[j] == a.vocab;
                t.add<1, false>(y, a.c2);
            }
            t.join_wave<false>(a.c2);
            wrong = __ballot(wrong) != 0 || t.s != t.s;
            if (lane_id() == 0) s_teacher = make_float4(kept_max(t), 1.f / t.s, log2_fast(t.s) * kLn2, nothing_left(t) ? 0.f : wrong ? __builtin_nanf("") : 1.f);
        }
        Softmax f = Softmax::none();
#pragma unroll
        for (int u = 0; u < NV; u++) {
            float x[P::kLen];
            const u32x4 none = P::filled(kNoLogit);
            const bool in = piece_of(u) < pieces;
            u32x4 piece = raw[u];
#pragma unroll
            for (int k = 0; k < 4; k++) piece[k] = in ? piece[k] : none[k];
            P::unpack(piece, x);
            f.add<P::kLen, false>(x, a.c2);
            __builtin_amdgcn_sched_barrier(0);           // (one piece unpacked at a time)
        }
        {
            const float x[1] = {end < a.vocab ? (float)raw_end : kNoLogit};
            f.add<1, false>(x, a.c2);
        }
        f.join_wave<false>(a.c2);
        if (lane_id() == 0) {
            s_max[wave] = f.m;
            s_sum[wave] = f.s;
        }
        __syncthreads();
        f = Softmax::none();
        if (lane_id() < kRowWaves) {
            f.m = s_max[lane_id()];
            f.s = s_sum[lane_id()];
        }
        f.join_wave<false>(a.c2);
        const float4 t = s_teacher;
        const bool none = nothing_left(f), empty = t.w == 0.f, wrong = t.w != t.w;
        const float m = kept_max(f), sum_z = wrong ? __builtin_nanf("") : f.s;
        // (read through the scalar cache: no vector load to wait for)
        const float weight = a.weights ? ((const __attribute__((address_space(4))) float*)a.weights)[row] : 1.f;
        const float w = none || empty ? 0.f : weight * a.inv_t;
        char* dz = (char*)a.grad + row * a.grad_stride * (int64_t)sizeof(raw_t);
        const float share = w / sum_z;                       // the row's factor / the sum of the powers
        // (a row without weight has gradient 0 whatever it holds: by the bits)
        const uint32_t kept = w == 0.f ? 0u : ~0u;
        auto gradient = [&](float x) { return share * exp2_fast((x - m) * a.c2); };
        auto put = [&](int u) {
            asm volatile("" : "+v"(raw[u]));             // (keeps the pieces packed: not the 32-bit values of the sums)
            float x[P::kLen];
            P::unpack(raw[u], x);
#pragma unroll
            for (int k = 0; k < P::kLen; k++) x[k] = gradient(x[k]);
            u32x4 out = P::pack(x);
#pragma unroll
            for (int k = 0; k < 4; k++) out[k] &= kept;
            P::store_once((raw_t*)(dz + at_piece(u, pieces - 1)), out);
        };
        // (without a next row one piece of this one is read instead, by all)
        const bool more = row + gridDim.x < a.n;
        const int64_t next = more ? row + gridDim.x : row;
        const int most = more ? pieces - 1 : 0;
        z = row_of(next);
        const raw_t was_end = raw_end;
        const float zy = (float)there;
        load_slots(next);
        raw_end = load_end(z);
#pragma unroll
        for (int u = 0; u < NV; u++) {
            put(u);
            raw[u] = load(z, u, most);
            if (u == (NV - 1) / 4) load_there(z);
            __builtin_amdgcn_sched_barrier(0);
        }
        if (end < a.vocab) ((raw_t*)dz)[end] = (raw_t)(kept ? gradient((float)was_end) : 0.f);
        // the teacher's part: the loss, and its tokens
        const int token = s_id[tid];
        float q = 0.f, loss = 0.f;                           // (half of it)
        if (__any(token >= 0)) {          // (logf, half as far off, in the place of the logarithms here and above: 113 instead of 111 us for 1001 x 100003)
            const float y = s_y[tid];
            q = token < 0 ? 0.f : power_of(y, t.x, a.c2, a.c2_rest) * t.y;
            loss = q == 0.f ? 0.f : half_loss(q, y, t.x, zy, none ? 0.f : m, a.inv_t, t.z - (none ? 0.f : log2_fast(f.s) * kLn2));
            loss = sum_of_lanes(loss);
        }
        s_q[tid] = q;
        if (lane_id() == 0) s_loss[wave] = loss;
        __syncthreads();
        if (tid == 0) {
            loss = 0.f;
            for (int v = 0; v < kRowWaves; v++) loss += s_loss[v];
            a.losses[row] = empty ? 0.f : wrong ? __builtin_nanf("") : loss_of_half(loss);
            if (a.stats) a.stats[row] = make_float4(none ? kNoLogit : m, sum_z, empty ? kNoLogit : t.x, t.y);
        }
        if (w != 0.f && token >= 0 && token < a.vocab) {
            const float sum = slots_of_token(s_id, s_q, (a.slots + 3) / 4, token);
            ((raw_t*)dz)[token] = (raw_t)(share * exp2_fast((zy - m) * a.c2) - w * sum);
        }
        __syncthreads();
        if (!more) return;
        row = next;
    }
}

template <class T, int kMode, int kRowThreads>
int stats_by(LogitArgs a, hipStream_t s) {
    constexpr int U = sizeof(typename T::raw) == 4 || kRowThreads == kWave ? 4 : 2;      // loads in flight
    for (int64_t most = kMaxGrid / a.splits; a.first < a.n; a.first += most) {
        const uint32_t rows = (uint32_t)std::min(most, a.n - a.first);
        logit_stats_kernel<T, kMode, kRowThreads, U><<<rows * a.splits, kRowThreads, 0, s>>>(a);
        DCIH_HIP(hipGetLastError());
        if (a.splits > 1) {
            logit_join_kernel<T, kMode><<<rows, kWave, 0, s>>>(a);
            DCIH_HIP(hipGetLastError());
        }
    }
    return 0;
}

// With alternatives one wavefront takes a row where there are rows enough to fill the device, or rows too short for more:
// each wavefront of a row has best pieces of its own to find.  One and four, us, with 5 alternatives in bf16:
//   rows of   1024         2048          3000          4096          8192
//     9000    13.7  12.9   16.6  18.9    19.8  25.1    23.0  31.4    38.1  56.1
//    50001    42.7  33.2   54.0  52.1    66.7  72.8    82.0  91.3     151   173
//   131072    88.6  61.5    108   101     140   147     180   193     344   372
// (f32: 40.2 and 26.7 for 1024 x 32000, 83.8 and 86.8 for 4096; 1024 x 1000 7.1 and 8.8.)  Without, four take 81 us and one 85.
template <class T, int kMode>
int stats_of(const LogitArgs& a, hipStream_t s) {
    if constexpr (kMode == kLogprobsTop) {
        const bool few = a.vocab <= 4 * kWave * Piece<T>::kLen;
        if (a.splits == 1 && (a.n >= 4096 || few)) return stats_by<T, kMode, kWave>(a, s);
    }
    return stats_by<T, kMode, kThreads>(a, s);
}

template <class T, int kRowThreads, int NV>
int distill_rows_by(const LogitArgs& a, int per_unit, hipStream_t s) {      // per_unit: workgroups that a compute unit holds
    const uint32_t groups = (uint32_t)std::min<int64_t>(a.n, 256 * per_unit);
    distill_rows_kernel<T, kRowThreads, NV><<<groups, kRowThreads, 0, s>>>(a);
    DCIH_HIP(hipGetLastError());
    return 0;
}

constexpr int kMostPieces = 16 * 1024;       // of a row in registers

// The fewest threads that hold a row in 16 pieces each and a slot each: several rows are on a compute unit then,
// and one's sums run while others' bytes travel.  (1024 threads for all: 16384 x 2000 bf16 379 us instead of 33, 8192 x 16000
// 251 instead of 120, 4096 x 50000 233 instead of 187.)  Fewer pieces where they do: what a thread does not need it reads
// again, which costs most where rows start off a boundary.  16 pieces for all instead of these, f16: 4 pieces 8192 x 1900 40 us
// instead of 20, 8 pieces 8192 x 9000 143 instead of 85, 10 pieces 1001 x 81001 119 instead of 87, 13 pieces 1001 x 53001 65
// instead of 56 and x 100003 125 instead of 109.
template <class T>
int distill_rows_of(const LogitArgs& a, hipStream_t s) {
    const int pieces = a.vocab / Piece<T>::kLen;
    if (a.slots <= 64) {
        if (pieces <= 4 * 64) return distill_rows_by<T, 64, 4>(a, 24, s);
        if (pieces <= 8 * 64) return distill_rows_by<T, 64, 8>(a, 20, s);
        // (few rows wait for one wavefront's 16 pieces: 64 x 8000 bf16 7.7 us, 5.0 by four; 1000 x 8000 9.7 and 9.4, 4000 26 and 27)
        if (pieces <= 16 * 64 && a.n >= 1024) return distill_rows_by<T, 64, 16>(a, 16, s);
    }
    if (a.slots <= 256) {
        if (pieces <= 4 * 256) return distill_rows_by<T, 256, 4>(a, 6, s);
        if (pieces <= 8 * 256) return distill_rows_by<T, 256, 8>(a, 5, s);
        if (pieces <= 16 * 256) return distill_rows_by<T, 256, 16>(a, 4, s);
    }
    if (a.slots <= 512) {
        if (pieces <= 8 * 512) return distill_rows_by<T, 512, 8>(a, 2, s);
        if (pieces <= 13 * 512) return distill_rows_by<T, 512, 13>(a, 2, s);
        if (pieces <= 16 * 512) return distill_rows_by<T, 512, 16>(a, 2, s);
    }
    if (pieces <= 4 * 1024) return distill_rows_by<T, 1024, 4>(a, 1, s);
    if (pieces <= 8 * 1024) return distill_rows_by<T, 1024, 8>(a, 1, s);
    if (pieces <= 10 * 1024) return distill_rows_by<T, 1024, 10>(a, 1, s);
    if (pieces <= 13 * 1024) return distill_rows_by<T, 1024, 13>(a, 1, s);
    return distill_rows_by<T, 1024, 16>(a, 1, s);
}

template <class T, int kMode>
int grad_of(LogitArgs a, hipStream_t s) {
    constexpr int U = 2, kTile = kThreads * U * Piece<T>::kLen;      // elements
    a.splits = a.vocab / kTile + 1;           // (what is left of a row is a piece more)
    for (int64_t most = std::max<int64_t>(1, kMaxGrid / a.splits); a.first < a.n; a.first += most) {
        logit_grad_kernel<T, kMode, U><<<(uint32_t)std::min(most, a.n - a.first) * a.splits, kThreads, 0, s>>>(a);
        DCIH_HIP(hipGetLastError());
    }
    return 0;
}

}  // namespace

// Workgroups a row is split over: enough of them in all to fill the device, each with a round of loads of all its threads
// at least, and none of rows that are done before splits could be joined (4 rows of 16000 bf16: 4.2 us by a workgroup each,
// 4.9 by 8 and the join, with 10 alternatives 11.9 and 12.5; 800: 8.4 and 10.2; but 4 of 50000 8.3 and 4.8, 500 16.3 and 15.1).
int logit_splits(int64_t n, int vocab, int dtype) {
    const int64_t pieces = ((int64_t)vocab * type_bytes(dtype) + 15) / 16;
    if (pieces <= 8 * kThreads) return 1;
    const int64_t most = (pieces + kThreads - 1) / kThreads, want = (1024 + n - 1) / n;
    return (int)std::min<int64_t>(std::min(most, std::max<int64_t>(want, 1)), kMaxSplits);
}

int logit_stats(LogitArgs a, int dtype, bool distill, hipStream_t s) {
    const int len = 16 / type_bytes(dtype), pieces = a.vocab / len + 1;
    a.per_split = (pieces + a.splits - 1) / a.splits;
    if (distill) {
        switch (dtype) {
            case DCIH_F32: return stats_of<F32, kDistill>(a, s);
            case DCIH_F16: return stats_of<F16, kDistill>(a, s);
            default: return stats_of<BF16, kDistill>(a, s);
        }
    }
    switch (dtype * 2 + (a.top > 0)) {
        case DCIH_F32 * 2: return stats_of<F32, kLogprobs>(a, s);
        case DCIH_F32 * 2 + 1: return stats_of<F32, kLogprobsTop>(a, s);
        case DCIH_F16 * 2: return stats_of<F16, kLogprobs>(a, s);
        case DCIH_F16 * 2 + 1: return stats_of<F16, kLogprobsTop>(a, s);
        case DCIH_BF16 * 2: return stats_of<BF16, kLogprobs>(a, s);
        default: return stats_of<BF16, kLogprobsTop>(a, s);
    }
}

// Rows that fit a workgroup's registers, by one workgroup each; where they are long, only if there are enough of
// them to give a compute unit in three one: one of 131072 bf16 takes 21 us by one workgroup and 13 by three launches over
// the device, 64 22 and 20, 80 22.4 and 22.1, 96 23 and 24, 128 24 and 28; one of 32000 takes 8.6 and 9.6.  (Shorter ones part
// earlier: of 60000 f32 1 takes 14 and 10, 32 15.2 and 14.9, 64 16 and 18; of 65536 bf16 1 takes 12.3 and 12.1, 64 14 and 17.)
bool distill_by_rows(const LogitArgs& a, int dtype) {
    const int len = 16 / type_bytes(dtype), pieces = a.vocab / len;
    return pieces >= 1 && pieces <= kMostPieces && (pieces <= 4096 || a.n >= 96);
}

int distill_rows(const LogitArgs& a, int dtype, hipStream_t s) {
    switch (dtype) {
        case DCIH_F32: return distill_rows_of<F32>(a, s);
        case DCIH_F16: return distill_rows_of<F16>(a, s);
        default: return distill_rows_of<BF16>(a, s);
    }
}

int logit_grad(const LogitArgs& a, int dtype, bool distill, hipStream_t s) {
    if (distill) {
        switch (dtype) {
            case DCIH_F32: return grad_of<F32, kDistill>(a, s);
            case DCIH_F16: return grad_of<F16, kDistill>(a, s);
            default: return grad_of<BF16, kDistill>(a, s);
        }
    }
    switch (dtype) {
        case DCIH_F32: return grad_of<F32, kLogprobs>(a, s);
        case DCIH_F16: return grad_of<F16, kLogprobs>(a, s);
        default: return grad_of<BF16, kLogprobs>(a, s);
    }
}

}  // namespace dcih
