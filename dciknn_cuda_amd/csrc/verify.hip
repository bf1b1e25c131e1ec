// Drafted tokens t_i of a sequence against the model's probabilities p_i = softmax(z_i / temperature), from given random
// numbers u: t_i stands while u_i q_i(t_i) < p_i(t_i), with q_i what it was drawn from (1 for a draft that was named for
// certain).  Where the first does not, a token is drawn from max(p_i - q_i, 0), behind the last one from p_i: the first with
// u_k (sum of all weights) < (sum of the weights up to it).
//
// A token is right or wrong: everything that decides on one is in 64 bits, exponentials included, so that a random number has to
// be within 1e-13 of a border to be taken to its wrong side (in 32 bits the borders of 131072 tokens cover some hundredths of [0, 1)).
// Behind a refused draft borders are parts of what is left of the row: a border there is 1e-13 of the row off while a thousandth or more is
// left, 1e-14 of it where less is (see choose_kernel).  Taking off leaves nothing of an entry where it leaves as little as those roundings.
#include "../../include/dci_hip.h"
#include "verify.h"

#include <algorithm>

namespace dcih {
namespace {

constexpr int kThreads = 256, kWaves = kThreads / kWave;
constexpr int kChunk = 2048;                   // entries of a row that one wavefront adds up
constexpr int kSumWaves = 6;                   // of a SIMD (512 x 131072 bf16 with the choice 44.7 us; 4, as the registers would have it, 47.5; 8 50)
constexpr int kChoosers = 512, kChooserWaves = kChoosers / kWave;
constexpr int64_t kMaxGrid = 1 << 23;

struct alignas(16) Sum { double s; float m; float pad; };        // sum of 2^((z - m) c2), m = 0 or max z

// 2^x to 1e-15 of it: n whole, 2^f by its series.  0 for x = -inf, NaN for NaN.
__device__ inline double exp2_wide(double x) {
    const double n = __builtin_rint(x), f = x - n;
    double p = 2.5678435993488196e-11;          // ln(2)^12 / 12!
    p = __builtin_fma(p, f, 4.44553827187081e-10);
    p = __builtin_fma(p, f, 7.054911620801121e-09);
    p = __builtin_fma(p, f, 1.0178086009239696e-07);
    p = __builtin_fma(p, f, 1.3215486790144305e-06);
    p = __builtin_fma(p, f, 1.5252733804059838e-05);
    p = __builtin_fma(p, f, 0.00015403530393381606);
    p = __builtin_fma(p, f, 0.0013333558146428441);
    p = __builtin_fma(p, f, 0.009618129107628477);
    p = __builtin_fma(p, f, 0.055504108664821576);
    p = __builtin_fma(p, f, 0.2402265069591007);
    p = __builtin_fma(p, f, 0.6931471805599453);
    p = __builtin_fma(p, f, 1.0);
    const double y = __builtin_ldexp(p, (int)__builtin_fmax(n, -2000.0));
    return x < -1100.0 ? 0.0 : y;
}
// The weight of an entry beside the largest.  The difference is formed before the factor: of the type's lowest values it is exact.
__device__ inline double weight_of(float z, double c2, double m) { return exp2_wide(((double)z - m) * c2); }
// What weights are relative to, for a row of nothing but -inf too.
__device__ inline double base_of(float m) { return (double)(m == kNoLogit ? 0.f : m); }

template <int O> __device__ inline double other_lane(double v) {
    return __builtin_bit_cast(double, dcih::other_lane<O>(__builtin_bit_cast(unsigned long long, v)));
}
__device__ inline double lanes_sum(double v) {
    v += other_lane<32>(v); v += other_lane<16>(v); v += other_lane<8>(v);
    v += other_lane<4>(v); v += other_lane<2>(v); v += other_lane<1>(v);
    return v;
}
// Sums over the lanes up to and including each one's.
template <int kControl, int kRows> __device__ inline double add_shifted(double v) {
    const unsigned long long w = __builtin_bit_cast(unsigned long long, v);
    const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)w, kControl, kRows, 0xf, false);
    const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(w >> 32), kControl, kRows, 0xf, false);
    return v + __builtin_bit_cast(double, (unsigned long long)hi << 32 | lo);
}
__device__ inline double lanes_scan(double v) {
    v = add_shifted<0x111, 0xf>(v);      // row_shr:1
    v = add_shifted<0x112, 0xf>(v);
    v = add_shifted<0x114, 0xf>(v);
    v = add_shifted<0x118, 0xf>(v);
    v = add_shifted<0x142, 0xa>(v);      // row_bcast:15 into rows 1 and 3
    return add_shifted<0x143, 0xc>(v);   // row_bcast:31 into rows 2 and 3
}

// 2^(i / 256), i below 256, as 2^x is put together for whole rows: less i / 256 in its exponent's place, so that adding all of n / 256 there
// leaves 2^(n / 256), n = i mod 256.
constexpr int kParts = 256;
// 2^(f / 256), |f| <= 1/2, by its series to f^3, with 0.207 f^2 for f^4: 2.5e-14 off at most, and 1 at 0, so that a certain token's share is 1
constexpr double kC1 = 0.0027076061740622863, kC2 = 3.665566060704036e-06, kC3 = 3.3083026805413713e-09;
constexpr int kPart = 20 - 8;
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
__device__ inline void fill_table(u32x2* s_table) {
    static_assert(kParts == kThreads, "a part for each thread");
    u32x2 part = __builtin_bit_cast(u32x2, exp2_wide((double)threadIdx.x / kParts));
    part.y -= threadIdx.x << kPart;
    s_table[threadIdx.x] = part;
}
// s + 2^(d scale / 256): 2^(whole / 256) 2^(rest / 256).  The sum with 1.5 2^52 holds `whole` in its low word.
__device__ inline double add_power(double d, double scale, double s, const u32x2* s_table) {
    constexpr double kMagic = 6755399441055744.0;
    const double t = __builtin_fma(d, scale, kMagic), f = __builtin_fma(d, scale, -(t - kMagic));
    const uint32_t whole = (uint32_t)__builtin_bit_cast(unsigned long long, t);
    double q = kC3;
    q = __builtin_fma(q, f, kC2);
    q = __builtin_fma(q, f, kC1);
    q = __builtin_fma(q, f, 1.0);
    u32x2 part = s_table[whole & (kParts - 1)];
    part.y += whole << kPart;
    return __builtin_fma(__builtin_bit_cast(double, part), q, s);
}

// A wavefront adds up `per` chunks of a row, one after the other.  Rows behind a sequence's last draft are asked for by nobody.
// Weights are relative to 1 where 64 bits have room for that, as logits have it: no look for the largest first.  A sum that says otherwise
// is formed again, relative to the chunk's largest.
// Bound by its instructions: 9 of 64 bits and 6 others an entry, 512 x 131072 bf16 35 us (the bytes alone take 25).  By a table of 64 and
// one more term, relative to each chunk's largest: 43.
template <class T>
__global__ __launch_bounds__(kThreads, kSumWaves) void sums_kernel(VerifyArgs a, Sum* sums, int chunks, int per, int64_t first) {
    using P = Piece<T>;
    constexpr int U = kChunk / kWave / P::kLen;
    __shared__ u32x2 s_table[kParts];
    const int splits = (chunks + per - 1) / per, lane = lane_id();
    const int64_t item = first + (int64_t)blockIdx.x * kWaves + __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int64_t row = item / splits, b = row / (a.drafts + 1);
    const int i = b < a.n ? (int)(row - b * (a.drafts + 1)) : 0, from = (int)(item - row * splits) * per, to = min(chunks, from + per);
    int64_t draft = lane < i ? id_at(a.ids, a.wide_ids, b * a.drafts + lane) : 0;
    fill_table(s_table);
    __syncthreads();
    if (b >= a.n) return;
    for (int j = lane;;) {
        if (__any(draft < 0)) return;
        j += kWave;
        if (!__any(j < i)) break;
        draft = j < i ? id_at(a.ids, a.wide_ids, b * a.drafts + j) : 0;
    }
    const Row<T> r(a.z, row, a.stride, a.vocab);
    const double scale = a.c2 * kParts;
    const double deepest = -1000.0 / a.c2;                 // weights of less than 2^-1000 are that
    const bool plain = a.c2 > 1e-27 && a.c2 < 1e30;        // `most` is far from the ends of its type
    const float most = (float)(900.0 / a.c2);
    for (int c = from; c < to; c++) {
        u32x4 raw[U];
        const int piece = c * (kChunk / P::kLen) + lane;
        if ((c + 1) * (kChunk / P::kLen) <= r.pieces) {
            r.load_runs(piece, kWave, raw);
        } else {
#pragma unroll
            for (int u = 0; u < U; u++) raw[u] = r.load(piece + u * kWave);
        }
        float m = 0.f;
        bool bad = false;
        double s = 0.0;
        if (plain) {
#pragma unroll
            for (int u = 0; u < U; u++) {
                float z[P::kLen];
                P::unpack(raw[u], z);
#pragma unroll
                for (int k = 0; k < P::kLen; k++) {
                    bad |= z[k] != z[k];
                    s = add_power((double)__builtin_amdgcn_fmed3f(z[k], -most, most), scale, s, s_table);
                }
            }
            s = lanes_sum(s);
        }
        if (!(s > 0x1p-800 && s < 0x1p890)) {              // nothing of -inf counts, nothing was cut
            m = kNoLogit;
#pragma unroll
            for (int u = 0; u < U; u++) {
                float z[P::kLen];
                P::unpack(raw[u], z);
#pragma unroll
                for (int k = 0; k < P::kLen; k++) {
                    m = fmaxf(m, z[k]);
                    bad |= z[k] != z[k];
                }
            }
            m = max_of_lanes(m);
            const double base = base_of(m);
            s = 0.0;
#pragma unroll
            for (int u = 0; u < U; u++) {
                float z[P::kLen];
                P::unpack(raw[u], z);
#pragma unroll
                for (int k = 0; k < P::kLen; k++) s = add_power(__builtin_fmax((double)z[k] - base, deepest), scale, s, s_table);
            }
            s = lanes_sum(s);
            if (m == kNoLogit) s = 0.0;
        }
        if (__any(bad) || m == -kNoLogit) s = __builtin_nan("");
        if (lane == 0) sums[row * chunks + c] = Sum{s, m, 0.f};
    }
}

// Sums up to and including each thread's, in the order of the threads.
__device__ inline double scan_threads(double v, double* s_part) {
    const int lane = lane_id(), wave = threadIdx.x / kWave;
    v = lanes_scan(v);
    __syncthreads();
    if (lane == kWave - 1) s_part[wave] = v;
    __syncthreads();
    double before = 0.0;
    for (int w = 0; w < wave; w++) before += s_part[w];
    return before + v;
}

// The largest thread that says yes and what it brings, which grows with the threads.  (By the last lane of each wavefront: an atomic operation of 64
// lanes takes them one by one, 1.5 us.)
__device__ inline void last_that(bool yes, int value, int* s_last) {
    const unsigned long long lanes = __ballot(yes);
    if (lanes && lane_id() == kWave - 1 - __builtin_clzll(lanes)) atomicMax(s_last, value);
}

__device__ inline float teacher_at(const VerifyArgs& a, int64_t i) {
    switch (a.teacher_dtype) {
        case DCIH_F32: return ((const float*)a.teacher)[i];
        case DCIH_F16: return (float)((const _Float16*)a.teacher)[i];
        default: return (float)((const __bf16*)a.teacher)[i];
    }
}

constexpr int kSlots = 1024, kNearChunks = 256;      // chunks whose amounts are added up beside the slots
constexpr double kLog2eWide = 1.44269504088896340736, kLn2Wide = 0.693147180559945309417;

// 11.3 us of 64 sequences with 7 drafts of 64 slots each, 7.6 of 4 with 4 drafts for certain: a chain of loads, exponentials and joined sums that wait
// for one another.
// One workgroup a sequence: a wavefront a row joins its sums and says whether the draft stands; then all of them draw the next token
// from the row that it comes from, by chunks, then among the entries of one.
template <class T>
__global__ __launch_bounds__(kChoosers) void choose_kernel(VerifyArgs a, Sum* sums, int chunks, int64_t first) {
    constexpr int kPer = kChunk / kChoosers;
    __shared__ double s_total[kMaxDrafts + 1], s_part[kChooserWaves], s_weight[kChunk], s_gone[kSlots], s_target;
    __shared__ unsigned long long s_fixed[kSlots], s_taken[kNearChunks];
    __shared__ float s_max[kMaxDrafts + 1], s_z[kMaxDrafts + 1];
    __shared__ int s_kept[kMaxDrafts], s_id[kSlots], s_chunk_of[kSlots], s_chunk, s_token, s_last, s_slots;
    const int64_t b = first + blockIdx.x;
    const int k = a.drafts, lane = lane_id(), wave = threadIdx.x / kWave, tid = threadIdx.x;
    const float u = a.uniforms[b * (k + 1) + k];
    const double c2 = a.c2;
    const typename T::raw* logits = (const typename T::raw*)a.z + b * (k + 1) * a.stride;
    auto draft_at = [&](int i) { return id_at(a.ids, a.wide_ids, b * k + i); };
    // what a row takes from memory, for the first one of a wavefront before it is known whether there is such a draft
    struct Asked { Sum part; int64_t draft, id; float number, teacher; };
    auto ask = [&](int i) {
        Asked r{Sum{0.0, kNoLogit, 0.f}, -1, -1, 0.f, kNoLogit};
        if (i <= k && lane < chunks) r.part = sums[(b * (k + 1) + i) * chunks + lane];
        if (i >= k) return r;
        r.draft = draft_at(i);
        r.number = a.uniforms[b * (k + 1) + i];
        if (a.slot_ids && lane < a.slots) {
            r.id = id_at(a.slot_ids, a.wide_slots, (b * k + i) * a.slots + lane);
            r.teacher = teacher_at(a, (b * k + i) * a.slots + lane);
        }
        return r;
    };
    Asked r = ask(wave);
    // how many drafts there are
    if (tid == 0) {
        s_slots = k;                                  // (for the moment)
        s_chunk = s_token = s_last = -1;
    }
    __syncthreads();
    for (int i = tid; i < k; i += kChoosers)
        if (draft_at(i) < 0) atomicMin(&s_slots, i);
    __syncthreads();
    const int given = s_slots;
    for (int i = wave; i <= given; i += kChooserWaves, r = ask(i)) {
        const float z = i < given && r.draft < a.vocab ? (float)logits[i * a.stride + r.draft] : kNoLogit;
        const Sum* part = sums + (b * (k + 1) + i) * chunks;
        float m = r.part.m;
        for (int c = lane + kWave; c < chunks; c += kWave) m = fmaxf(m, part[c].m);
        m = max_of_lanes(m);
        const double base = base_of(m);
        auto share_of = [&](const Sum& p) { return p.s == 0.0 ? 0.0 : p.s * weight_of(p.m, c2, base); };
        double s = share_of(r.part);
        for (int c = lane + kWave; c < chunks; c += kWave) s += share_of(part[c]);
        s = lanes_sum(s);
        if (lane == 0) {
            s_total[i] = s;
            s_max[i] = m;
            s_z[i] = z;
        }
        if (i == given) continue;
        // the probability that it was drawn with: its / all
        double its = 1.0, all = 1.0;
        if (a.slot_ids) {
            const int64_t at = (b * k + i) * a.slots;
            float top = r.id >= 0 ? r.teacher : kNoLogit;
            for (int j = lane + kWave; j < a.slots; j += kWave)
                if (id_at(a.slot_ids, a.wide_slots, at + j) >= 0) top = fmaxf(top, teacher_at(a, at + j));
            top = max_of_lanes(top);
            const double top_base = base_of(top);
            all = r.id < 0 ? 0.0 : weight_of(r.teacher, kLog2eWide, top_base);
            its = r.id == r.draft ? all : 0.0;
            for (int j = lane + kWave; j < a.slots; j += kWave) {
                const int64_t id = id_at(a.slot_ids, a.wide_slots, at + j);
                const double w = id < 0 ? 0.0 : weight_of(teacher_at(a, at + j), kLog2eWide, top_base);
                all += w;
                its += id == r.draft ? w : 0.0;
            }
            all = lanes_sum(all);
            its = lanes_sum(its);
        }
        const double p = weight_of(z, c2, base);
        // (without slots it is none of what was drawn from: 0 < p, if the row has probabilities and the number is one)
        if (lane == 0) s_kept[i] = p > 0.0 && (double)r.number * its * s < p * (all == 0.0 ? 1.0 : all);
    }
    __syncthreads();
    int kept = 0;
    while (kept < given && s_kept[kept]) kept++;
    // row `kept` names the next token
    const double total = s_total[kept], base = base_of(s_max[kept]);
    const typename T::raw* row = logits + kept * a.stride;
    Sum* part = sums + (b * (k + 1) + kept) * chunks;
    bool fine = total > 0.0 && total < __builtin_huge_val();
    // what is taken off its weights: ids and amounts, each id once.  (What several threads add up are whole numbers of 2^-52 of
    // the largest, or of 2^-60 of the total: their order does not matter.)
    const int each = (chunks + kChoosers - 1) / kChoosers, begin = min(chunks, tid * each), end = min(chunks, begin + each);
    Sum mine{};
    if (begin < end) mine = part[begin];
    int slots = 0;
    if (kept < given && fine) {
        for (int c = tid; c < kNearChunks; c += kChoosers) s_taken[c] = 0;
        if (!a.slot_ids) {
            slots = 1;
            if (tid == 0) {
                const int64_t t = draft_at(kept);
                s_id[0] = t < a.vocab ? (int)t : -1;
                s_gone[0] = total;
            }
        } else {
            slots = a.slots;
            const int64_t at = (b * k + kept) * a.slots;
            constexpr int E = kSlots / kChoosers;
            int id[E];
            float z[E], top = kNoLogit;
#pragma unroll
            for (int e = 0; e < E; e++) {
                const int j = tid + e * kChoosers;
                id[e] = -2;
                z[e] = kNoLogit;
                if (j >= slots) continue;
                const int64_t wide = id_at(a.slot_ids, a.wide_slots, at + j);
                z[e] = teacher_at(a, at + j);
                id[e] = wide < 0 ? -1 : wide < a.vocab ? (int)wide : a.vocab;
                z[e] = wide < 0 ? kNoLogit : z[e];
                top = fmaxf(top, z[e]);
            }
            top = max_of_lanes(top);
            if (lane == 0) s_part[wave] = top;
#pragma unroll
            for (int e = 0; e < E; e++) {
                const int j = tid + e * kChoosers;
                s_id[j] = id[e];
                s_fixed[j] = 0;
            }
            __syncthreads();
            for (int w = 0; w < kChooserWaves; w++) top = fmaxf(top, (float)s_part[w]);
            const double top_base = base_of(top);
            bool bad = false;
            double amount[E];
#pragma unroll
            for (int e = 0; e < E; e++) {
                const int j = tid + e * kChoosers;
                amount[e] = 0.0;
                if (id[e] < 0) continue;
                const double w = weight_of(z[e], kLog2eWide, top_base);
                bad |= !(w <= 1.0);
                // a token of several slots stands in the first of them
                int lead = j;
                for (int o = 0; o < j; o += 8) {
                    int found = j;
#pragma unroll
                    for (int i = 7; i >= 0; i--) found = s_id[o + i] == id[e] && o + i < j ? o + i : found;
                    lead = found < lead ? found : lead;
                }
                if (lead == j) amount[e] = w;
                else if (!bad) atomicAdd(&s_fixed[lead], (unsigned long long)(w * 0x1p52));
            }
            fine = !__syncthreads_or(bad);
            double all = 0.0;
#pragma unroll
            for (int e = 0; e < E; e++) {
                amount[e] += (double)s_fixed[tid + e * kChoosers] * 0x1p-52;
                all += amount[e];
            }
            all = lanes_sum(all);
            __syncthreads();
            if (lane == 0) s_part[wave] = all;
            __syncthreads();
            all = 0.0;
            for (int w = 0; w < kChooserWaves; w++) all += s_part[w];
            const double share = all == 0.0 ? 0.0 : total / all;
#pragma unroll
            for (int e = 0; e < E; e++) {
                const int j = tid + e * kChoosers;
                s_gone[j] = amount[e] * share;
                if (id[e] == a.vocab || amount[e] == 0.0) s_id[j] = -1;
            }
        }
    }
    __syncthreads();
    // What is left of an entry, nothing where that is within the roundings of what is taken off.
    double rounding = 1e-13;
    auto left_of = [&](double w, double gone) {
        const double left = w - gone;
        return left > gone * rounding ? left : 0.0;
    };
    const double to_fixed = 0x1p60 / total;
    for (int j = tid; j < (slots + 7) / 8 * 8; j += kChoosers) {           // what entry s_id[j] weighs less than in p
        const int id = j < slots ? s_id[j] : -1;
        const double w = id >= 0 ? weight_of((float)row[id], c2, base) : 0.0, less = id >= 0 ? w - left_of(w, s_gone[j]) : 0.0;
        s_fixed[j] = (unsigned long long)(less * to_fixed);
        s_chunk_of[j] = id >= 0 ? id / kChunk : -1;
        if (id >= 0 && id / kChunk < kNearChunks) atomicAdd(&s_taken[id / kChunk], s_fixed[j]);
    }
    __syncthreads();
    fine = fine && u == u;
    // The weights of a chunk's entries, less what is taken off; to be read behind the next barrier.  (Between the last read of others and this stands
    // a barrier in each place: that of the sum or of the scan over them.)
    auto weigh = [&](int from, bool all_of_them) {
#pragma unroll
        for (int e = 0; e < kPer; e++) {
            const int i = e * kChoosers + tid;
            s_weight[i] = from + i < a.vocab ? weight_of((float)row[from + i], c2, base) : 0.0;
        }
        if (all_of_them) return;
        __syncthreads();
        for (int j = tid; j < slots; j += kChoosers)
            if (s_id[j] >= from && s_id[j] < from + kChunk) s_weight[s_id[j] - from] = left_of(s_weight[s_id[j] - from], s_gone[j]);
    };
    auto sum_of_weights = [&] {
        __syncthreads();
        double sum = 0.0;
#pragma unroll
        for (int e = 0; e < kPer; e++) sum += s_weight[tid * kPer + e];
        scan_threads(sum, s_part);
        sum = 0.0;
        for (int w = 0; w < kChooserWaves; w++) sum += s_part[w];
        return sum;
    };
    // the chunk: a run of chunks for each thread
    bool settled = false;                // what is left of a chunk stands in the place of its sum
    auto chunk_sum = [&](int c) -> double {
        const Sum p = c == begin ? mine : part[c];
        const double s = p.s == 0.0 ? 0.0 : p.s * weight_of(p.m, c2, base);
        unsigned long long taken = 0;
        if (!slots || settled) return s;
        if (c < kNearChunks) taken = s_taken[c];
        else
            for (int o = 0; o < slots; o++) taken += s_chunk_of[o] == c ? s_fixed[o] : 0;
        return __builtin_fmax(s - (double)taken * (total * 0x1p-60), 0.0);
    };
    double all = 0.0, before = 0.0, own = 0.0;
    auto sum_up = [&] {
        own = 0.0;
        for (int c = begin; c < end; c++) own += chunk_sum(c);
        before = scan_threads(own, s_part);
        all = 0.0;
        for (int w = 0; w < kChooserWaves; w++) all += s_part[w];
    };
    auto put = [&](int c, double sum) {
        if (tid == 0) part[c] = Sum{sum, s_max[kept], 0.f};
    };
    auto put_done = [&] {
        __syncthreads();
        if (begin < end) mine = part[begin];
    };
    if (fine) sum_up();
    // Sums are 2.5e-14 off, each entry 1e-15.  Where little is left that is not small beside it: chunks that something is taken off are formed again
    // from their entries, so that what is left is as near as 1e-14 of the row.
    if (__builtin_expect(fine && slots && !(all >= total * 0x1p-10), 0)) {
        rounding = 1e-14;
        bool leads[kSlots / kChoosers];
#pragma unroll
        for (int e = 0; e < kSlots / kChoosers; e++) {
            const int j = tid + e * kChoosers;
            leads[e] = j < slots && s_chunk_of[j] >= 0;
            for (int o = 0; leads[e] && o < j; o++) leads[e] = s_chunk_of[o] != s_chunk_of[j];
        }
        __syncthreads();
#pragma unroll
        for (int e = 0; e < kSlots / kChoosers; e++)
            if (tid + e * kChoosers < slots && !leads[e]) s_chunk_of[tid + e * kChoosers] = -1;
        __syncthreads();
        settled = true;
        for (int j = 0; j < slots; j++) {
            const int c = s_chunk_of[j];
            if (c < 0) continue;
            weigh(c * kChunk, true);
            const double sum = sum_of_weights();
            if (tid == 0) s_fixed[j] = __builtin_bit_cast(unsigned long long, sum);
            put(c, sum);
        }
        put_done();
        sum_up();
        const double more = all / total;
        for (int j = tid; j < slots; j += kChoosers) s_gone[j] *= more;
        for (int j = 0; j < slots; j++) {
            const int c = s_chunk_of[j];
            if (c < 0) continue;
            weigh(c * kChunk, false);
            put(c, sum_of_weights());
        }
        put_done();
        sum_up();
        if (!(all > 0.0)) {              // nothing is left: drawn from p itself
            for (int j = 0; j < slots; j++)
                if (s_chunk_of[j] >= 0) put(s_chunk_of[j], __builtin_bit_cast(double, s_fixed[j]));
            put_done();
            slots = 0;
            sum_up();
        }
    }
    // (a chunk of which there is a sum, of roundings, and no entry counts as nothing: the next one is looked for)
    while (fine && all > 0.0) {
        const double target = min(max((double)u, 0.0), 1.0) * all;
        last_that(own > 0.0 && before - own <= target, tid, &s_last);      // (with weights below the target)
        __syncthreads();
        if (tid == s_last) {
            double sum = before - own;
            int at = -1;
            double rest = target - sum;
            if (end - begin == 1) at = begin;
            for (int c = begin; end - begin > 1 && c < end; c++) {
                const double s = chunk_sum(c);
                if (s > 0.0 && sum <= target) {
                    at = c;
                    rest = target - sum;
                }
                sum += s;
            }
            s_chunk = at;
            s_target = rest;
        }
        __syncthreads();
        // the entry
        const int chunk = s_chunk, from = chunk * kChunk;
        if (chunk < 0) break;
        weigh(from, false);
        if (tid == 0) s_last = -1;
        __syncthreads();
        double w[kPer], sum = 0.0;
#pragma unroll
        for (int e = 0; e < kPer; e++) {
            w[e] = s_weight[tid * kPer + e];
            sum += w[e];
        }
        sum = scan_threads(sum, s_part) - sum;
        int found = -1;
#pragma unroll
        for (int e = 0; e < kPer; e++) {
            if (w[e] > 0.0 && sum <= s_target) found = tid * kPer + e;
            sum += w[e];
        }
        last_that(found >= 0, found, &s_last);
        __syncthreads();
        if (s_last >= 0) {
            if (tid == 0) s_token = from + s_last;
            break;
        }
        put(chunk, 0.0);
        put_done();
        sum_up();
        if (tid == 0) s_last = -1;
        __syncthreads();
    }
    __syncthreads();
    const int token = s_token;
    for (int i = tid; i <= k; i += kChoosers) {
        const int64_t t = i < kept ? draft_at(i) : i == kept ? token : -1;
        float logp = 0.f;
        if (i <= kept) {
            const float z = i < kept ? s_z[i] : t >= 0 ? (float)row[t] : __builtin_nanf("");
            logp = (float)(((double)z - base_of(s_max[i])) * c2 * kLn2Wide - log(s_total[i]));
        }
        a.tokens[b * (k + 1) + i] = (int32_t)t;
        a.logprobs[b * (k + 1) + i] = logp;
    }
    if (tid == 0) a.accepted[b] = kept;
}

int chunks_of(int vocab) { return (vocab + kChunk - 1) / kChunk; }

template <class T>
int run(const VerifyArgs& a, hipStream_t s) {
    const int chunks = chunks_of(a.vocab);
    const int64_t rows = a.n * (a.drafts + 1);
    // wavefronts that fill the device
    const int per = (int)std::min<int64_t>(chunks, std::max<int64_t>(1, rows * chunks / 16384));
    const int64_t items = rows * ((chunks + per - 1) / per), most = kMaxGrid * kWaves;
    for (int64_t first = 0; first < items; first += most) {
        sums_kernel<T><<<(uint32_t)((std::min(most, items - first) + kWaves - 1) / kWaves), kThreads, 0, s>>>(a, (Sum*)a.work, chunks, per, first);
        DCIH_HIP(hipGetLastError());
    }
    for (int64_t first = 0; first < a.n; first += kMaxGrid) {
        choose_kernel<T><<<(uint32_t)std::min(kMaxGrid, a.n - first), kChoosers, 0, s>>>(a, (Sum*)a.work, chunks, first);
        DCIH_HIP(hipGetLastError());
    }
    return 0;
}

}  // namespace

int64_t verify_work_bytes(int64_t rows, int vocab, int) { return rows * chunks_of(vocab) * (int64_t)sizeof(Sum); }

int verify(const VerifyArgs& a, int dtype, hipStream_t s) {
    switch (dtype) {
        case DCIH_F32: return run<F32>(a, s);
        case DCIH_F16: return run<F16>(a, s);
        default: return run<BF16>(a, s);
    }
}

}  // namespace dcih
