// Rows of a table by ids, times a factor, and the gradient of that by the table:
//
//   out[i, :] = scale * W[id_i, :]            dW[v, :] = scale * sum over i with id_i = v of G[i, :]
//
// Both are bound by memory.  The gradient's sums are formed without atomics on values, in the
// order of the tokens whatever the schedule: the tokens are first grouped by their row (chunk_kernel,
// bucket_kernel), then summed in pieces of up to kPiece tokens of one row (sum_kernel); the pieces of rows with more
// tokens than that are joined by a third launch (join_kernel).  Sums are in 32 bits, rounded once.
#include "../../include/dci_hip.h"
#include "token_common.h"

#include <algorithm>
#include <type_traits>

namespace dcih {
namespace {

constexpr int kThreads = 256;

// ---- lookup ------------------------------------------------------------------------------
// `lanes` (a power of two up to 256) neighbouring threads take one row.
template <class T>
__global__ __launch_bounds__(kThreads) void lookup_kernel(EmbedArgs a, int lanes, int64_t first) {
    using P = Piece<T>;
    const int64_t i = first + (int64_t)blockIdx.x * (kThreads / lanes) + threadIdx.x / lanes;
    if (i >= a.n) return;
    const int64_t id = id_at(a.ids, a.wide_ids, i);
    typename T::raw* out = (typename T::raw*)a.out + i * a.dim;
    // an empty slot is a row of zeros; a row that does not exist is not passed over in silence
    const float fill = id < 0 ? 0.f : __builtin_nanf("");
    const bool real = id >= 0 && id < a.num_rows;
    const typename T::raw* row = (const typename T::raw*)a.rows + (real ? id : 0) * a.stride;
    for (int c = (threadIdx.x % lanes) * P::kLen; c < a.dim; c += lanes * P::kLen) {
        const bool whole = c + P::kLen <= a.dim;
        float y[P::kLen];
        if (real) {
            P::unpack(whole ? P::load(row + c) : P::load_part(row, c, a.dim, 0.f), y);
#pragma unroll
            for (int k = 0; k < P::kLen; k++) y[k] *= a.scale;
        } else {
#pragma unroll
            for (int k = 0; k < P::kLen; k++) y[k] = fill;
        }
        const u32x4 x = P::pack(y);
        if (whole) P::store(out + c, x);
        else P::store_part(out, c, a.dim, x);
    }
}

// ---- tokens by rows ----------------------------------------------------------------------
// One token in the grouped order: its row, its place among all tokens, its place among the row's
// tokens, and how many the row has.
struct alignas(16) Token { uint32_t row, at, rank, count; };
struct alignas(8) Placed { uint32_t row, at; };

constexpr int kChunk = 2048;                             // tokens that one workgroup puts in order of their buckets
constexpr int kGroupThreads = 512, kGroupWaves = kGroupThreads / kWave;
constexpr int kPerLane = kChunk / kGroupThreads;
constexpr int kMinBucketBits = 8, kMaxBucketBits = 11;   // a bucket for each compute unit; what chunk_kernel counts on chip
constexpr int kBins = 1024;                              // rows that bucket_kernel counts at a time
constexpr int kPiece = 32;                               // tokens of a row that are summed by one group of lanes

// The call's workspace.
struct Work {
    uint32_t* total;        // tokens with a row
    Placed* placed;         // [chunks][kChunk]: each chunk's tokens in order of (bucket, place)
    uint16_t* starts;       // [chunks][buckets + 1]: where a bucket's begin
    Token* tokens;          // [n] in the grouped order
    unsigned long long* present;   // [buckets][words]: bit r mod 64 of word r / 64 for the r-th row of a bucket
    float* part;            // [2 * windows][width]: see sum_kernel
    int64_t chunks, windows;
    int bucket_bits, words, width;
};
__host__ inline size_t lay_out(Work& w, void* mem, int64_t n, int dim, int64_t num_rows) {
    w.chunks = (n + kChunk - 1) / kChunk;
    w.windows = (n + kPiece - 1) / kPiece;
    w.width = (dim + 7) & ~7;
    w.bucket_bits = kMinBucketBits;
    while (w.bucket_bits < kMaxBucketBits && num_rows > (int64_t)kBins << w.bucket_bits) w.bucket_bits++;
    const int64_t buckets = 1 << w.bucket_bits;
    w.words = (int)(((num_rows + buckets - 1) / buckets + 63) / 64);
    size_t at = 0;
    auto take = [&](auto*& p, int64_t count) {
        p = (std::remove_reference_t<decltype(p)>)((char*)mem + at);
        at += (count * sizeof(*p) + 255) / 256 * 256;
    };
    take(w.total, 1);
    take(w.placed, w.chunks * kChunk);
    take(w.starts, w.chunks * (buckets + 1));
    take(w.tokens, n);
    take(w.present, buckets * w.words);
    take(w.part, w.windows * 2 * w.width);
    return at;
}

__device__ inline int lanes_below(unsigned long long mask) {
    return __builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0));
}

// The lanes of `in` whose keys (of `bits` bits) are the same as this one's.
__device__ inline unsigned long long same_key(unsigned long long in, uint32_t key, int bits) {
    for (int b = 0; b < bits; b++) {
        const bool one = key >> b & 1;
        const unsigned long long ones = __ballot(one);
        in &= one ? ones : ~ones;
    }
    return in;
}

// Exclusive sums over the workgroup's threads of one value each, behind `before`; *all: the sum of all.
__device__ inline uint32_t group_scan(uint32_t v, uint32_t before, uint32_t* s_wave, uint32_t* all) {
    const uint32_t upto = wave_scan_u32(v);
    __syncthreads();
    if (lane_id() == kWave - 1) s_wave[threadIdx.x / kWave] = upto;
    __syncthreads();
    uint32_t start = before + upto - v, sum = 0;
    for (int w = 0; w < kGroupWaves; w++) {
        if (w < (int)threadIdx.x / kWave) start += s_wave[w];
        sum += s_wave[w];
    }
    *all = sum;
    return start;
}

// Grouping, first half.  Bucket b holds the rows r with r mod buckets = b (neighbouring rows, often alike in
// their number of tokens, go to different ones).  A workgroup puts a chunk of the tokens in order
// of their buckets, those of a bucket in their own order: a wavefront takes a run of them, counts
// them by buckets as it goes, and the counts of the wavefronts before it give its places.
__global__ __launch_bounds__(kGroupThreads) void chunk_kernel(const void* ids, bool wide, int64_t n, int64_t num_rows, Work w) {
    extern __shared__ uint32_t s_count[];                // [kGroupWaves][buckets]
    __shared__ uint32_t s_wave[kGroupWaves];
    const int tid = threadIdx.x, wave = tid / kWave, lane = lane_id(), buckets = 1 << w.bucket_bits;
    const int64_t base = (int64_t)blockIdx.x * kChunk;
    int64_t id[kPerLane];
    uint32_t rank[kPerLane];
#pragma unroll
    for (int j = 0; j < kPerLane; j++) {
        const int64_t i = base + (wave * kPerLane + j) * kWave + lane;
        id[j] = i < n ? id_at(ids, wide, i) : -1;
    }
    for (int i = tid; i < kGroupWaves * buckets; i += kGroupThreads) s_count[i] = 0;
    __syncthreads();
    uint32_t* mine = s_count + wave * buckets;
#pragma unroll
    for (int j = 0; j < kPerLane; j++) {
        const bool real = id[j] >= 0 && id[j] < num_rows;
        if (!real) id[j] = -1;
        const uint32_t bucket = (uint32_t)id[j] & (buckets - 1);
        const unsigned long long same = same_key(__ballot(real), bucket, w.bucket_bits);
        if (real) {
            const uint32_t have = mine[bucket];
            rank[j] = have + lanes_below(same);
            if (lanes_below(same) == 0) mine[bucket] = have + __popcll(same);
        }
    }
    __syncthreads();
    uint32_t before = 0;
    uint16_t* starts = w.starts + blockIdx.x * (int64_t)(buckets + 1);
    for (int b0 = 0; b0 < buckets; b0 += kGroupThreads) {
        const int b = b0 + tid;
        uint32_t len = 0, all;
        if (b < buckets)
            for (int v = 0; v < kGroupWaves; v++) len += s_count[v * buckets + b];
        uint32_t start = group_scan(len, before, s_wave, &all);
        if (b < buckets) {
            starts[b] = (uint16_t)start;
            for (int v = 0; v < kGroupWaves; v++) {
                const uint32_t c = s_count[v * buckets + b];
                s_count[v * buckets + b] = start;
                start += c;
            }
        }
        before += all;
    }
    if (tid == 0) starts[buckets] = (uint16_t)before;
    __syncthreads();
#pragma unroll
    for (int j = 0; j < kPerLane; j++) {
        if (id[j] < 0) continue;
        const uint32_t at = mine[(uint32_t)id[j] & (buckets - 1)] + rank[j];
        w.placed[base + at] = Placed{(uint32_t)id[j], (uint32_t)(base + (wave * kPerLane + j) * kWave + lane)};
    }
}

// Calls f(token, whether it is one) for a bucket's tokens in chunks [from, to), in order, by whole wavefronts.
template <class F>
__device__ inline void for_tokens(const Work& w, int bucket, int64_t from, int64_t to, F f) {
    const int lane = lane_id(), row = (1 << w.bucket_bits) + 1;
    for (int64_t c0 = from; c0 < to; c0 += kWave) {
        uint32_t o0 = 0, o1 = 0;
        if (c0 + lane < to) {
            o0 = w.starts[(c0 + lane) * row + bucket];
            o1 = w.starts[(c0 + lane) * row + bucket + 1];
        }
        const int many = (int)min((int64_t)kWave, to - c0);
        constexpr int kAhead = 4;
        for (int j0 = 0; j0 < many; j0 += kAhead) {
            Placed p[kAhead];
            int first[kAhead], last[kAhead];
#pragma unroll
            for (int j = 0; j < kAhead; j++) {
                const int from_lane = min(j0 + j, many - 1);
                first[j] = __builtin_amdgcn_readlane((int)o0, from_lane);
                last[j] = j0 + j < many ? __builtin_amdgcn_readlane((int)o1, from_lane) : first[j];
                p[j] = Placed{0, 0};
                if (first[j] + lane < last[j]) p[j] = w.placed[(c0 + j0 + j) * kChunk + first[j] + lane];
            }
#pragma unroll
            for (int j = 0; j < kAhead; j++) {
                if (first[j] < last[j]) f(p[j], first[j] + lane < last[j]);
                for (int t = first[j] + kWave; t < last[j]; t += kWave) {
                    const bool real = t + lane < last[j];
                    f(real ? w.placed[(c0 + j0 + j) * kChunk + t + lane] : Placed{0, 0}, real);
                }
            }
        }
    }
}

// Second half: a workgroup takes a bucket, its wavefronts runs of the chunks.  What the chunks hold of the
// buckets before it is where its part of the order starts; its rows are counted up to kBins at a time.
__global__ __launch_bounds__(kGroupThreads) void bucket_kernel(int64_t num_rows, Work w) {
    __shared__ uint32_t s_count[kGroupWaves][kBins];
    __shared__ uint32_t s_start[kBins], s_len[kBins];
    __shared__ uint32_t s_wave[kGroupWaves], s_before[kGroupWaves], s_total[kGroupWaves];
    const int tid = threadIdx.x, wave = tid / kWave, lane = lane_id(), bucket = blockIdx.x, buckets = 1 << w.bucket_bits;
    const int64_t run = (w.chunks + kGroupWaves - 1) / kGroupWaves, from = min(w.chunks, wave * run), to = min(w.chunks, from + run);
    uint32_t before = 0, total = 0;
    for (int64_t c = from + lane; c < to; c += kWave) {
        before += w.starts[c * (buckets + 1) + bucket];
        total += w.starts[c * (buckets + 1) + buckets];
    }
    before = wave_sum_u32(before);
    total = wave_sum_u32(total);
    if (lane == 0) {
        s_before[wave] = before;
        s_total[wave] = total;
    }
    __syncthreads();
    before = total = 0;
    for (int v = 0; v < kGroupWaves; v++) {
        before += s_before[v];
        total += s_total[v];
    }
    if (bucket == 0 && tid == 0) *w.total = total;
    const int64_t rows = (num_rows - bucket + buckets - 1) >> w.bucket_bits;       // of this bucket
    for (int64_t bin0 = 0; bin0 < rows; bin0 += kBins) {
        for (int i = tid; i < kGroupWaves * kBins; i += kGroupThreads) (&s_count[0][0])[i] = 0;
        __syncthreads();
        for_tokens(w, bucket, from, to, [&](Placed p, bool real) {
            const uint32_t bin = (p.row >> w.bucket_bits) - (uint32_t)bin0;
            if (real && bin < kBins) atomicAdd(&s_count[wave][bin], 1u);
        });
        __syncthreads();
        for (int b0 = 0; b0 < kBins; b0 += kGroupThreads) {
            const int b = b0 + tid;
            uint32_t len = 0, all;
            for (int v = 0; v < kGroupWaves; v++) {
                const uint32_t c = s_count[v][b];
                s_count[v][b] = len;
                len += c;
            }
            s_start[b] = group_scan(len, before, s_wave, &all);
            s_len[b] = len;
            before += all;
            const unsigned long long have = __ballot(len != 0);
            const int64_t word = (bin0 + b) / kWave;
            if (lane == 0 && word < w.words) w.present[(int64_t)bucket * w.words + word] = have;
        }
        __syncthreads();
        for_tokens(w, bucket, from, to, [&](Placed p, bool real) {
            const uint32_t bin = (p.row >> w.bucket_bits) - (uint32_t)bin0;
            const bool mine = real && bin < kBins;
            const unsigned long long same = same_key(__ballot(mine), bin, 10);       // 2^10 = kBins
            if (mine) {
                const uint32_t rank = s_count[wave][bin] + lanes_below(same);
                if (lanes_below(same) == 0) s_count[wave][bin] = rank + __popcll(same);
                w.tokens[s_start[bin] + rank] = Token{p.row, p.at, rank, s_len[bin]};
            }
        });
        __syncthreads();
    }
}

// ---- sums --------------------------------------------------------------------------------
// Writes N sums of columns c .. c + N - 1 of row `row`.
template <class O, int N>
__device__ inline void put_sums(const EmbedArgs& a, uint32_t row, int c, const float (&sum)[N]) {
    using P = Piece<O>;
    typename O::raw* out = (typename O::raw*)a.out + (int64_t)row * a.dim;
    constexpr int kStep = N < P::kLen ? N : P::kLen;
    if (N >= P::kLen && c + N <= a.dim) {
#pragma unroll
        for (int j = 0; j < N; j += kStep) {
            float y[P::kLen];
            if (a.accumulate) {
                P::unpack(P::load(out + c + j), y);
#pragma unroll
                for (int k = 0; k < kStep; k++) y[k] += sum[j + k] * a.scale;
            } else {
#pragma unroll
                for (int k = 0; k < kStep; k++) y[k] = sum[j + k] * a.scale;
            }
            P::store(out + c + j, P::pack(y));
        }
        return;
    }
#pragma unroll
    for (int k = 0; k < N; k++) {
        if (c + k >= a.dim) continue;
        const float y = sum[k] * a.scale;
        out[c + k] = (typename O::raw)(a.accumulate ? (float)out[c + k] + y : y);
    }
}

template <class O, int N>
__device__ inline void put_zeros(const EmbedArgs& a, int64_t row, int c) {
    using P = Piece<O>;
    typename O::raw* out = (typename O::raw*)a.out + row * a.dim;
    const u32x4 none = {0, 0, 0, 0};
    if (c + N <= a.dim) {
#pragma unroll
        for (int j = 0; j < N; j += P::kLen) P::store(out + c + j, none);
    } else {
        for (int k = c; k < a.dim; k++) out[k] = (typename O::raw)0.f;
    }
}

// `lanes` (a power of two up to 64) neighbouring lanes take one window of kPiece tokens in one slice of
// the columns: they sum the pieces that START in the window, up to kPiece tokens of one row each.
// Rows of up to kPiece tokens are one piece and final; the first piece of a longer one goes to
// place 2 w + 1 of `part`, a later one to 2 w (a window w has at most one of each).
//
// Behind the windows' groups come those that write the rows without tokens: one takes the 64 rows
// of a word of `present` in one slice.  Every row is written once, and these writes fill the gaps of the reads.
template <class T, class O>
__global__ __launch_bounds__(kThreads) void sum_kernel(EmbedArgs a, Work w, int lanes, int slices, int64_t first) {
    using P = Piece<T>;
    constexpr int kAhead = 8;
    const int64_t unit = first + (int64_t)blockIdx.x * (kThreads / lanes) + threadIdx.x / lanes;
    const int64_t window = unit / slices, total = *w.total;
    if (window >= w.windows) {
        const int64_t word = window - w.windows;
        const int c = ((int)(unit % slices) * lanes + threadIdx.x % lanes) * P::kLen;
        if (a.accumulate || word >= (int64_t)w.words << w.bucket_bits || c >= a.dim) return;
        const int64_t row0 = (word % w.words * 64 << w.bucket_bits) + word / w.words;
        for (unsigned long long left = ~w.present[word]; left; left &= left - 1) {
            const int64_t row = row0 + ((int64_t)__builtin_ctzll(left) << w.bucket_bits);
            if (row >= a.num_rows) break;
            put_zeros<O, P::kLen>(a, row, c);
        }
        return;
    }
    const int64_t begin = window * kPiece, end = min(total, begin + kPiece);
    if (begin >= end) return;
    const int c = ((int)(unit % slices) * lanes + threadIdx.x % lanes) * P::kLen;
    if (c >= a.dim) return;
    const bool whole = c + P::kLen <= a.dim;
    // the pieces that start here are tokens [t, stop): behind the rest of an earlier one, and up to
    // the end of the piece of the window's last token
    const Token e0 = w.tokens[begin], e1 = w.tokens[end - 1];
    int64_t t = begin;
    if (e0.rank % kPiece) t += min(kPiece - e0.rank % kPiece, e0.count - e0.rank);
    if (t >= end) return;
    const int64_t stop = end - 1 + min(kPiece - e1.rank % kPiece, e1.count - e1.rank);
    float sum[P::kLen];
#pragma unroll
    for (int k = 0; k < P::kLen; k++) sum[k] = 0.f;
    for (; t < stop; t += kAhead) {
        Token e[kAhead];
        u32x4 x[kAhead];
#pragma unroll
        for (int j = 0; j < kAhead; j++) e[j] = w.tokens[min(t + j, stop - 1)];
#pragma unroll
        for (int j = 0; j < kAhead; j++) {
            const typename T::raw* row = (const typename T::raw*)a.rows + (int64_t)e[j].at * a.stride;
            x[j] = whole ? P::load(row + c) : P::load_part(row, c, a.dim, 0.f);
        }
#pragma unroll
        for (int j = 0; j < kAhead; j++) {
            if (t + j >= stop) break;
            float y[P::kLen];
            P::unpack(x[j], y);
#pragma unroll
            for (int k = 0; k < P::kLen; k++) sum[k] += y[k];
            if (e[j].rank + 1 < e[j].count && (e[j].rank + 1) % kPiece) continue;
            if (e[j].count <= kPiece) {
                put_sums<O, P::kLen>(a, e[j].row, c, sum);
            } else {
                const int64_t began = t + j - e[j].rank % kPiece;
                float* part = w.part + (2 * (began / kPiece) + (e[j].rank < kPiece)) * w.width + c;
#pragma unroll
                for (int k = 0; k < P::kLen; k += 4)
                    *reinterpret_cast<float4*>(part + k) = make_float4(sum[k], sum[k + 1], sum[k + 2], sum[k + 3]);
            }
#pragma unroll
            for (int k = 0; k < P::kLen; k++) sum[k] = 0.f;
        }
    }
}

// Rows of more than kPiece tokens: a workgroup looks for them among 256 tokens, and its wavefronts
// add the pieces of each, every fourth one, in 256 columns.
template <class O>
__global__ __launch_bounds__(kThreads) void join_kernel(EmbedArgs a, Work w, int slices, int64_t first) {
    constexpr int kWaves = kThreads / kWave;
    __shared__ float s_sum[kWaves][kWave * 4];
    __shared__ int s_found[kThreads / kPiece + 1];
    __shared__ int s_n;
    const int64_t unit = first + blockIdx.x, total = *w.total;
    const int64_t base = unit / slices * kThreads;
    if (base >= total) return;
    const int c = (int)(unit % slices) * kWave * 4 + lane_id() * 4;
    const int tid = threadIdx.x, wave = tid / kWave;
    if (tid == 0) s_n = 0;
    __syncthreads();
    if (base + tid < total) {
        const Token e = w.tokens[base + tid];
        if (e.rank == 0 && e.count > kPiece) s_found[atomicAdd(&s_n, 1)] = tid;      // (in any order)
    }
    __syncthreads();
    for (int f = 0; f < s_n; f++) {
        const int64_t at = base + s_found[f], window = at / kPiece;
        const Token e = w.tokens[at];
        const int pieces = (int)((e.count + kPiece - 1) / kPiece);
        float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
        if (c < a.dim) {
#pragma unroll 4
            for (int p = wave; p < pieces; p += kWaves) {
                const float4 x = *reinterpret_cast<const float4*>(w.part + (2 * (window + p) + (p == 0)) * w.width + c);
                sum.x += x.x; sum.y += x.y; sum.z += x.z; sum.w += x.w;
            }
        }
        *reinterpret_cast<float4*>(&s_sum[wave][lane_id() * 4]) = sum;
        __syncthreads();
        if (wave == 0 && c < a.dim) {
            float y[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int v = 0; v < kWaves; v++)
#pragma unroll
                for (int k = 0; k < 4; k++) y[k] += s_sum[v][lane_id() * 4 + k];
            put_sums<O, 4>(a, e.row, c, y);
        }
        __syncthreads();
    }
}

constexpr int64_t kMaxGrid = 1 << 22;     // workgroups of one launch (their threads are counted in 32 bits)

// The smallest power of two that is no less than n, at most `most`.
int lanes_for(int n, int most) {
    int l = 1;
    while (l < n && l < most) l *= 2;
    return l;
}

template <class T>
int lookup(const EmbedArgs& a, hipStream_t s) {
    const int lanes = lanes_for((a.dim + Piece<T>::kLen - 1) / Piece<T>::kLen, kThreads), per = kThreads / lanes;
    for (int64_t first = 0; first < a.n; first += kMaxGrid * per) {
        const int64_t groups = std::min(kMaxGrid, (a.n - first + per - 1) / per);
        lookup_kernel<T><<<(uint32_t)groups, kThreads, 0, s>>>(a, lanes, first);
        DCIH_HIP(hipGetLastError());
    }
    return 0;
}

// Room on the chip for chunk_kernel's counts, once for each device.
int room_for_counts() {
    static DeviceOnce once;
    return once.run([] {
        DCIH_HIP(hipFuncSetAttribute((const void*)chunk_kernel, hipFuncAttributeMaxDynamicSharedMemorySize,
                                     kGroupWaves * (int)sizeof(uint32_t) << kMaxBucketBits));
        return 0;
    });
}

template <class T, class O>
int grad(const EmbedArgs& a, hipStream_t s) {
    Work w;
    lay_out(w, a.work, a.n, a.dim, a.num_rows);
    if (a.n) {
        if (int rc = room_for_counts()) return rc;
        chunk_kernel<<<(uint32_t)w.chunks, kGroupThreads, kGroupWaves * sizeof(uint32_t) << w.bucket_bits, s>>>(a.ids, a.wide_ids, a.n, a.num_rows, w);
        DCIH_HIP(hipGetLastError());
    }
    bucket_kernel<<<1u << w.bucket_bits, kGroupThreads, 0, s>>>(a.num_rows, w);
    DCIH_HIP(hipGetLastError());
    const int pieces = (a.dim + Piece<T>::kLen - 1) / Piece<T>::kLen, lanes = lanes_for(pieces, kWave);
    int slices = (pieces + lanes - 1) / lanes;
    const int per = kThreads / lanes;
    int64_t units = (w.windows + (a.accumulate ? 0 : (int64_t)w.words << w.bucket_bits)) * slices;
    for (int64_t first = 0; first < units; first += kMaxGrid * per) {
        const int64_t groups = std::min(kMaxGrid, (units - first + per - 1) / per);
        sum_kernel<T, O><<<(uint32_t)groups, kThreads, 0, s>>>(a, w, lanes, slices, first);
        DCIH_HIP(hipGetLastError());
    }
    if (a.n <= kPiece) return 0;
    slices = (a.dim + kWave * 4 - 1) / (kWave * 4);
    units = (a.n + kThreads - 1) / kThreads * slices;
    for (int64_t first = 0; first < units; first += kMaxGrid) {
        join_kernel<O><<<(uint32_t)std::min(kMaxGrid, units - first), kThreads, 0, s>>>(a, w, slices, first);
        DCIH_HIP(hipGetLastError());
    }
    return 0;
}

}  // namespace

int embed_rows(const EmbedArgs& a, int dtype, hipStream_t s) {
    switch (dtype) {
        case DCIH_F32: return lookup<F32>(a, s);
        case DCIH_F16: return lookup<F16>(a, s);
        default: return lookup<BF16>(a, s);
    }
}

size_t embed_grad_bytes(int64_t n, int dim, int64_t num_rows) {
    Work w;
    return lay_out(w, nullptr, n, dim, num_rows);
}

int embed_grad(const EmbedArgs& a, int dtype, int out_dtype, hipStream_t s) {
    switch (dtype) {
        case DCIH_F32: return grad<F32, F32>(a, s);
        case DCIH_F16: return out_dtype == DCIH_F32 ? grad<F16, F32>(a, s) : grad<F16, F16>(a, s);
        default: return out_dtype == DCIH_F32 ? grad<BF16, F32>(a, s) : grad<BF16, BF16>(a, s);
    }
}

}  // namespace dcih
