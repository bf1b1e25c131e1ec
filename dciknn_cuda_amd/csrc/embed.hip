// Rows of a table by ids, times a factor, and the gradient of that by the table:
//
//   out[i, :] = scale * W[id_i, :]            dW[v, :] = scale * sum over i with id_i = v of G[i, :]
//
// Both are bound by memory (figures are of one MI355X, whose copies reach 4.8 TB/s).  The gradient's sums are formed
// without atomics on values, in the order of the tokens whatever the schedule: the tokens are first grouped by their
// row (chunk_kernel, bucket_kernel), then summed in pieces of up to 16 tokens of one row (sum_kernel); the pieces of
// rows with more tokens than that are joined by a third launch (join_kernel).  Sums are in 32 bits, rounded once.
#include "../../include/dci_hip.h"
#include "token_common.h"

#include <algorithm>
#include <type_traits>

namespace dcih {
namespace {

constexpr int kThreads = 256;

// ---- lookup ------------------------------------------------------------------------------
// `lanes` (up to 256) neighbouring threads take one row: as many as it has pieces, so that few are idle.  Bound by
// memory: 32768 tokens of text by 131072 x 4096 bf16 78 us (268 MB written, 98 MB of different rows read: 4.7 TB/s),
// 100000 x 128 f32 20 us (5.1 TB/s), 32 x 4096 bf16 4.2 us (a launch).
template <class T>
__global__ __launch_bounds__(kThreads) void lookup_kernel(EmbedArgs a, int lanes, int64_t first) {
    using P = Piece<T>;
    const int per = kThreads / lanes, group = threadIdx.x / lanes;
    const int64_t i = first + (int64_t)blockIdx.x * per + group;
    if (group >= per || i >= a.n) return;
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
constexpr int kWide = 16;                                // pieces from which a row's sums are joined by groups
// Elements from which pieces of 16 tokens fill the device: fewer parts to join (65536 x 32 f32 40 us, 45 with pieces of 8,
// 65536 x 1024 101 and 110; but 5000 x 100 26 and 24, 20000 x 64 28 and 27).
constexpr int64_t kManySums = 1 << 21;

// The call's workspace.
struct Work {
    uint32_t* total;        // [3]: tokens with a row; rows with more tokens than a piece, and than kWide pieces
    Placed* placed;         // [chunks][kChunk]: each chunk's tokens in order of (bucket, place)
    uint16_t* starts;       // [chunks][buckets + 1]: where a bucket's begin
    Token* tokens;          // [n] in the grouped order
    uint32_t* common;       // [2][n / piece]: where the rows with more tokens than a piece, and than kWide pieces, begin
    float* part;            // [2 * windows][width]: see sum_kernel
    int64_t chunks, windows;
    int64_t cleared;        // rows that chunk_kernel writes zeros to: all or none
    int piece;              // tokens of a row that are summed by one group of lanes
    int bucket_bits, width;
};

// Bucket b holds the rows r with r mod buckets = b: rows are often alike in their number of tokens where
// they are near (with runs of 8 rows the commonest bucket took 30 us instead of 16 for 65536 tokens of text).
__device__ inline uint32_t bucket_of(const Work& w, uint32_t row) { return row & ((1u << w.bucket_bits) - 1); }
__device__ inline uint32_t bin_of(const Work& w, uint32_t row) { return row >> w.bucket_bits; }
__device__ inline int64_t row_of(const Work& w, int64_t bucket, int64_t bin) { return (bin << w.bucket_bits) + bucket; }

__host__ inline size_t lay_out(Work& w, void* mem, int64_t n, int dim, int64_t num_rows) {
    w.chunks = (n + kChunk - 1) / kChunk;
    w.piece = n * dim >= kManySums ? 16 : 8;
    w.windows = (n + w.piece - 1) / w.piece;
    w.width = (dim + 7) & ~7;
    w.bucket_bits = kMinBucketBits;
    while (w.bucket_bits < kMaxBucketBits && num_rows > (int64_t)kBins << w.bucket_bits) w.bucket_bits++;
    const int64_t buckets = 1 << w.bucket_bits;
    size_t at = 0;
    auto take = [&](auto*& p, int64_t count) {
        p = (std::remove_reference_t<decltype(p)>)((char*)mem + at);
        at += (count * sizeof(*p) + 255) / 256 * 256;
    };
    take(w.total, 3);
    take(w.placed, w.chunks * kChunk);
    take(w.starts, w.chunks * (buckets + 1));
    take(w.tokens, n);
    take(w.common, 2 * (n / w.piece));
    take(w.part, w.windows * 2 * w.width);
    return at;
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
template <int kWaves>
__device__ inline uint32_t group_scan(uint32_t v, uint32_t before, uint32_t* s_wave, uint32_t* all) {
    const uint32_t upto = wave_scan_u32(v);
    __syncthreads();
    if (lane_id() == kWave - 1) s_wave[threadIdx.x / kWave] = upto;
    __syncthreads();
    uint32_t start = before + upto - v, sum = 0;
    for (int w = 0; w < kWaves; w++) {
        if (w < (int)threadIdx.x / kWave) start += s_wave[w];
        sum += s_wave[w];
    }
    *all = sum;
    return start;
}

// Grouping, first half.  A workgroup puts a chunk of the tokens in order
// of their buckets, those of a bucket in their own order: a wavefront takes a run of them, counts
// them by buckets as it goes, and the counts of the wavefronts before it give its places.  Bound by the
// waits of its few steps: 5.6 us for 65536 tokens, 8.2 for 100000 by 1024 buckets (With one launch in
// which every workgroup read all ids, 65536 tokens by 50001 x 2048 bf16 took 80 us more.)
// More workgroups write zeros to the table's first w.cleared rows, 16 bytes a thread in the order of the launch: the one
// order that reaches 6.9 TB/s (rows in turn, or more bytes a thread: 4.4 to 6.1).
template <class O>
__global__ __launch_bounds__(kGroupThreads) void chunk_kernel(EmbedArgs a, Work w) {
    extern __shared__ uint32_t s_count[];                // [kGroupWaves][buckets]
    __shared__ uint32_t s_wave[kGroupWaves];
    if (blockIdx.x >= w.chunks) {
        const int64_t at = ((blockIdx.x - w.chunks) * kGroupThreads + threadIdx.x) * Piece<O>::kLen, end = w.cleared * a.dim;
        if (at + Piece<O>::kLen <= end) Piece<O>::store((typename O::raw*)a.out + at, u32x4{0, 0, 0, 0});
        else
            for (int64_t i = at; i < end; i++) ((typename O::raw*)a.out)[i] = (typename O::raw)0.f;
        return;
    }
    const int64_t n = a.n, num_rows = a.num_rows;
    const int tid = threadIdx.x, wave = tid / kWave, lane = lane_id(), buckets = 1 << w.bucket_bits;
    const int64_t base = (int64_t)blockIdx.x * kChunk;
    int64_t id[kPerLane];
    uint32_t rank[kPerLane];
#pragma unroll
    for (int j = 0; j < kPerLane; j++) {
        const int64_t i = base + (wave * kPerLane + j) * kWave + lane;
        id[j] = i < n ? id_at(a.ids, a.wide_ids, i) : -1;
    }
    for (int i = tid; i < kGroupWaves * buckets; i += kGroupThreads) s_count[i] = 0;
    __syncthreads();
    uint32_t* mine = s_count + wave * buckets;
#pragma unroll
    for (int j = 0; j < kPerLane; j++) {
        const bool real = id[j] >= 0 && id[j] < num_rows;
        if (!real) id[j] = -1;
        const uint32_t bucket = bucket_of(w, (uint32_t)id[j]);
        const unsigned long long same = same_key(__ballot(real), bucket, w.bucket_bits);
        if (real) {
            const uint32_t have = mine[bucket];
            rank[j] = have + lanes_below(same);
            if (lanes_below(same) == 0) mine[bucket] = have + __popcll(same);
        }
        wave_fence();
    }
    __syncthreads();
    uint32_t before = 0;
    uint16_t* starts = w.starts + blockIdx.x * (int64_t)(buckets + 1);
    for (int b0 = 0; b0 < buckets; b0 += kGroupThreads) {
        const int b = b0 + tid;
        uint32_t len = 0, all;
        if (b < buckets)
            for (int v = 0; v < kGroupWaves; v++) len += s_count[v * buckets + b];
        uint32_t start = group_scan<kGroupWaves>(len, before, s_wave, &all);
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
    if (tid == 0 && blockIdx.x == 0) w.total[1] = w.total[2] = 0;
    if (tid == 0) starts[buckets] = (uint16_t)before;
    __syncthreads();
#pragma unroll
    for (int j = 0; j < kPerLane; j++) {
        if (id[j] < 0) continue;
        const uint32_t at = mine[bucket_of(w, (uint32_t)id[j])] + rank[j];
        w.placed[base + at] = Placed{(uint32_t)id[j], (uint32_t)(base + (wave * kPerLane + j) * kWave + lane)};
    }
}

// Calls f(token, whether it is one) for a bucket's tokens in up to 64 chunks from `chunk` on, in order, by whole
// wavefronts; a lane has the bounds [o0, o1) in one chunk.  The tokens are taken as one sequence, 64 at a
// time whatever their chunks hold.  (A chunk at a time: 16 us instead of 20 for the grouping of 65536 tokens of text, but 28
// instead of 16 for 100000 tokens spread evenly, two in a chunk.)
template <class F>
__device__ inline void for_tokens(const Work& w, int64_t chunk, uint32_t o0, uint32_t o1, F f) {
    constexpr int kAhead = 4;
    const uint32_t upto = wave_scan_u32(o1 - o0), total = (uint32_t)__builtin_amdgcn_readlane((int)upto, kWave - 1);
    const uint32_t mine = upto - (o1 - o0);          // tokens in the lanes before
    for (uint32_t t = 0; t < total; t += kAhead * kWave) {
        Placed p[kAhead];
#pragma unroll
        for (int j = 0; j < kAhead; j++) {
            const uint32_t at = t + j * kWave + lane_id();
            // the lane that holds it is the last one that starts at or before it: often the same one for all 64
            int lane = __popcll(__ballot(mine <= t + j * kWave)) - 1;
            uint32_t first, before;
            if (lane == __popcll(__ballot(mine <= t + j * kWave + kWave - 1)) - 1) {
                first = (uint32_t)__builtin_amdgcn_readlane((int)o0, lane);
                before = (uint32_t)__builtin_amdgcn_readlane((int)mine, lane);
            } else {
                lane = 0;
#pragma unroll
                for (int step = kWave / 2; step; step /= 2)
                    if ((uint32_t)__shfl((int)mine, lane + step) <= at) lane += step;
                first = (uint32_t)__shfl((int)o0, lane);
                before = (uint32_t)__shfl((int)mine, lane);
            }
            p[j] = Placed{0, 0};
            if (at < total) p[j] = w.placed[(chunk + lane) * kChunk + first + (at - before)];
        }
#pragma unroll
        for (int j = 0; j < kAhead; j++)
            if (t + j * kWave < total) f(p[j], t + j * kWave + lane_id() < total);
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
            P::store_once(out + c + j, P::pack(y));
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

// (Plain stores: rows that start off a line's boundary are written in parts of lines, which the caches put together.
// 10241 tokens by 49752 x 1593 f32: 91 us, 125 with non-temporal ones.)
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

// Second half of the grouping: a workgroup takes a bucket.  What the chunks hold of the buckets before it is where
// its part of the order starts.  Eight wavefronts read the bucket's tokens, in runs of the chunks, once to count them
// by rows (up to kBins at a time) and once to put them into their places.  Eight more meanwhile write the rows
// without tokens, whose bytes hide the waits of the first, unless there is nothing to be written or chunk_kernel has
// done it.  Bound by its own instructions in the bucket of the commonest row: 31 us for 65536 tokens of text with 142
// MB of zeros, 101 where 65536 of 131072 tokens have one row; or by the waits of its steps, where buckets are many:
// without zeros four workgroups are on a compute unit at once (100000 tokens added to 1M x 128 f32: 52 us in all, 63
// with one at a time).
template <class O, bool kZeros>
__global__ __launch_bounds__((kZeros ? 2 : 1) * kGroupThreads, kZeros ? 4 : 8) void bucket_kernel(EmbedArgs a, Work w, int lanes) {
    constexpr int kAllThreads = (kZeros ? 2 : 1) * kGroupThreads, kAllWaves = kAllThreads / kWave;
    __shared__ uint32_t s_count[kGroupWaves][kBins];
    __shared__ uint32_t s_start[kBins + 1];
    __shared__ uint32_t s_wave[kAllWaves], s_before[kGroupWaves], s_total[kGroupWaves];
    static_assert(kBins % kAllThreads == 0, "as many rows for each thread");
    const int tid = threadIdx.x, wave = tid / kWave, lane = lane_id(), bucket = blockIdx.x, buckets = 1 << w.bucket_bits;
    const bool reads = !kZeros || wave < kGroupWaves;
    const int64_t run = (w.chunks + kGroupWaves - 1) / kGroupWaves;
    const int64_t from = reads ? min(w.chunks, wave * run) : 0, to = reads ? min(w.chunks, from + run) : 0;
    uint32_t before = 0, total = 0, o0 = 0, o1 = 0;
    auto bounds = [&](int64_t c) {
        o0 = c < to ? w.starts[c * (buckets + 1) + bucket] : 0;
        o1 = c < to ? w.starts[c * (buckets + 1) + bucket + 1] : 0;
    };
    auto each_token = [&](auto f) {
        for (int64_t c = from; c < to; c += kWave) {
            if (run > kWave) bounds(c + lane);
            for_tokens(w, c, o0, o1, f);
        }
    };
    for (int64_t c = from + lane; c - lane < to; c += kWave) {
        bounds(c);
        before += o0;
        if (bucket == 0 && c < to) total += w.starts[c * (buckets + 1) + buckets];
    }
    before = wave_sum_u32(before);
    total = wave_sum_u32(total);
    if (reads && lane == 0) {
        s_before[wave] = before;
        s_total[wave] = total;
    }
    __syncthreads();
    before = total = 0;
    for (int v = 0; v < kGroupWaves; v++) {
        before += s_before[v];
        total += s_total[v];
    }
    if (bucket == 0 && tid == 0) w.total[0] = total;
    const int64_t rows = (a.num_rows - bucket + buckets - 1) >> w.bucket_bits;       // of this bucket
    for (int64_t bin0 = 0; bin0 < rows; bin0 += kBins) {
        for (int i = tid; i < kGroupWaves * kBins; i += kAllThreads) (&s_count[0][0])[i] = 0;
        __syncthreads();
        each_token([&](Placed p, bool real) {
            const uint32_t bin = bin_of(w, p.row) - (uint32_t)bin0;
            const bool mine = real && bin < kBins;
            // the first lane's row by one addition for all its tokens: a bucket of many has mostly one row
            const uint32_t lead = (uint32_t)__builtin_amdgcn_readfirstlane((int)bin);
            const unsigned long long same = __ballot(mine && bin == lead);
            if (mine && (bin != lead || lanes_below(same) == 0)) atomicAdd(&s_count[wave][bin], bin == lead ? (uint32_t)__popcll(same) : 1u);
        });
        __syncthreads();
        for (int bin = tid; bin < kBins; bin += kAllThreads) {
            uint32_t len = 0, all;
            for (int v = 0; v < kGroupWaves; v++) {
                const uint32_t c = s_count[v][bin];
                s_count[v][bin] = len;
                len += c;
            }
            const uint32_t start = group_scan<kAllWaves>(len, before, s_wave, &all);
            before += all;
            s_start[bin] = start;
            if (bin == kBins - 1) s_start[kBins] = start + len;
            if (len > (uint32_t)w.piece) {      // (in any order)
                const int wide = len > (uint32_t)(w.piece * kWide);
                w.common[wide * (a.n / w.piece) + atomicAdd(&w.total[1 + wide], 1u)] = start;
            }
        }
        __syncthreads();
        if (reads) {
            each_token([&](Placed p, bool real) {
                const uint32_t bin = bin_of(w, p.row) - (uint32_t)bin0;
                const bool mine = real && bin < kBins;
                const unsigned long long here = __ballot(mine), led = __ballot(mine && bin == (uint32_t)__builtin_amdgcn_readfirstlane((int)bin));
                const unsigned long long same = here == led ? here : same_key(here, bin, 10);       // 2^10 = kBins
                if (mine) {
                    const uint32_t rank = s_count[wave][bin] + lanes_below(same);
                    if (lanes_below(same) == 0) s_count[wave][bin] = rank + __popcll(same);
                    w.tokens[s_start[bin] + rank] = Token{p.row, p.at, rank, s_start[bin + 1] - s_start[bin]};
                }
                wave_fence();
            });
        } else if (kZeros) {
            const int64_t many = min((int64_t)kBins, rows - bin0);
            const int id = tid - kGroupThreads, groups = kGroupThreads / lanes;
            for (int64_t r = id / lanes < groups ? id / lanes : many; r < many; r += groups) {
                if (s_start[r + 1] != s_start[r]) continue;
                for (int c = id % lanes * Piece<O>::kLen; c < a.dim; c += lanes * Piece<O>::kLen)
                    put_zeros<O, Piece<O>::kLen>(a, row_of(w, bucket, bin0 + r), c);
            }
        }
        __syncthreads();
    }
}

// `lanes` (up to 64) neighbouring threads take one window of w.piece tokens in one slice of
// the columns: they sum the pieces that START in the window, up to as many tokens of one row each.
// Rows of up to w.piece tokens are one piece and final; the first piece of a longer one goes to
// place 2 w + 1 of `part`, a later one to 2 w (a window w has at most one of each).  Windows, not rows, are
// what a group takes: a tenth of a text's tokens are one row's.  Bound by memory: 65536 tokens by 50001 x 2048
// bf16 70 us (268 MB read, 82 MB written: 5.0 TB/s).
template <class T, class O, bool kByWaves>
__global__ __launch_bounds__(kThreads) void sum_kernel(EmbedArgs a, Work w, int lanes, int slices, int64_t first) {
    using P = Piece<T>;
    constexpr int kAhead = 8;
    if (kByWaves) lanes = kWave;
    const int per = kThreads / lanes, group = kByWaves ? __builtin_amdgcn_readfirstlane(threadIdx.x / kWave) : threadIdx.x / lanes;
    if (group >= per) return;
    // (With a wavefront for a window its tokens are read through the scalar cache, and half the registers do: 70 us for what
    // takes 73 otherwise.)
    auto token = [&](int64_t i) {
        if (!kByWaves) return w.tokens[i];
        const u32x4 x = ((const __attribute__((address_space(4))) u32x4*)w.tokens)[i];
        return Token{x[0], x[1], x[2], x[3]};
    };
    const int64_t unit = first + (int64_t)blockIdx.x * per + group;
    const int64_t window = unit / slices, total = *w.total;
    const int piece = w.piece;
    const int64_t begin = window * piece, end = min(total, begin + piece);
    if (begin >= end) return;
    const int c = ((int)(unit % slices) * lanes + threadIdx.x % lanes) * P::kLen;
    if (c >= a.dim) return;
    const bool whole = c + P::kLen <= a.dim;
    // the pieces that start here are tokens [t, stop): behind the rest of an earlier one, and up to
    // the end of the piece of the window's last token
    const Token e0 = token(begin), e1 = token(end - 1);
    int64_t t = begin;
    if (e0.rank & (piece - 1)) t += min(piece - (e0.rank & (piece - 1)), e0.count - e0.rank);
    if (t >= end) return;
    const int64_t stop = end - 1 + min(piece - (e1.rank & (piece - 1)), e1.count - e1.rank);
    float sum[P::kLen];
#pragma unroll
    for (int k = 0; k < P::kLen; k++) sum[k] = 0.f;
    for (; t < stop; t += kAhead) {
        Token e[kAhead];
        u32x4 x[kAhead];
#pragma unroll
        for (int j = 0; j < kAhead; j++) e[j] = token(min(t + j, stop - 1));
#pragma unroll
        for (int j = 0; j < kAhead; j++) {
            const typename T::raw* row = (const typename T::raw*)a.rows + (int64_t)e[j].at * a.stride;
            x[j] = whole ? P::load_once((const typename T::raw*)((const char*)row + (uint32_t)c * (uint32_t)sizeof(typename T::raw))) : P::load_part(row, c, a.dim, 0.f);
        }
#pragma unroll
        for (int j = 0; j < kAhead; j++) {
            if (t + j >= stop) break;
            float y[P::kLen];
            P::unpack(x[j], y);
#pragma unroll
            for (int k = 0; k < P::kLen; k++) sum[k] += y[k];
            if (e[j].rank + 1 < e[j].count && (e[j].rank + 1) & (piece - 1)) continue;
            if (e[j].count <= (uint32_t)piece) {
                put_sums<O, P::kLen>(a, e[j].row, c, sum);
            } else {
                const int64_t began = t + j - (e[j].rank & (piece - 1));
                float* part = w.part + (2 * (began / (uint32_t)piece) + (e[j].rank < (uint32_t)piece)) * w.width + c;
#pragma unroll
                for (int k = 0; k < P::kLen; k += 4)
                    *reinterpret_cast<float4*>(part + k) = make_float4(sum[k], sum[k + 1], sum[k + 2], sum[k + 3]);
            }
#pragma unroll
            for (int k = 0; k < P::kLen; k++) sum[k] = 0.f;
        }
    }
}

// Rows of more tokens than a piece.  Up to kWide pieces: a thread adds the pieces of one in four columns.
// More: sixteen groups of 16 lanes add every sixteenth piece of one in 64 columns.  (Sixteen groups for all
// of them: 17 us for the 400 such rows of 65536 tokens of text, nearly all of it the waits of many small workgroups.)
// Bound by the waits for a row's loads: 7.6 us there, 22 for a row of 4096 pieces.
template <class O, bool kIsWide>
__device__ void join_row(const EmbedArgs& a, const Work& w, uint32_t at, int slice, float4 (*s_sum)[16]) {
    constexpr int kLanes = kIsWide ? 16 : kThreads, kGroups = kThreads / kLanes, kAhead = 8;
    const int group = threadIdx.x / kLanes, lane = threadIdx.x % kLanes, c = (slice * kLanes + lane) * 4;
    const uint32_t window = at / (uint32_t)w.piece;
    const Token e = w.tokens[at];
    const int pieces = (int)((e.count + w.piece - 1) / (uint32_t)w.piece);
    float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
    if (c < a.dim) {
        for (int p0 = group; p0 < pieces; p0 += kGroups * kAhead) {
            float4 x[kAhead];
#pragma unroll
            for (int j = 0; j < kAhead; j++) {
                const int p = min(p0 + j * kGroups, pieces - 1);
                x[j] = *reinterpret_cast<const float4*>(w.part + (2 * ((int64_t)window + p) + (p == 0)) * w.width + c);
            }
#pragma unroll
            for (int j = 0; j < kAhead; j++) {
                // (no branch: the compiler would move the loads behind it, to wait for one at a time)
                const bool in = p0 + j * kGroups < pieces;
                sum.x += in ? x[j].x : 0.f; sum.y += in ? x[j].y : 0.f; sum.z += in ? x[j].z : 0.f; sum.w += in ? x[j].w : 0.f;
            }
        }
    }
    if (kIsWide) {
        s_sum[group][lane % 16] = sum;
        __syncthreads();
        if (group == 0) {
#pragma unroll
            for (int v = 1; v < kGroups; v++) {
                const float4 x = s_sum[v][lane % 16];
                sum.x += x.x; sum.y += x.y; sum.z += x.z; sum.w += x.w;
            }
        }
        __syncthreads();
    }
    if (group == 0 && c < a.dim) {
        const float y[4] = {sum.x, sum.y, sum.z, sum.w};
        put_sums<O, 4>(a, e.row, c, y);
    }
}
template <class O>
__global__ __launch_bounds__(kThreads) void join_kernel(EmbedArgs a, Work w, int wide_groups, int groups) {
    __shared__ float4 s_sum[16][16];
    int block = blockIdx.x;
    const int wide_slices = (a.dim + 63) / 64, slices = (a.dim + kThreads * 4 - 1) / (kThreads * 4);
    if (block < wide_groups * wide_slices) {
        const uint32_t many = w.total[2];
        for (uint32_t f = block / wide_slices; f < many; f += wide_groups)
            join_row<O, true>(a, w, w.common[a.n / w.piece + f], block % wide_slices, s_sum);
        return;
    }
    block -= wide_groups * wide_slices;
    const uint32_t many = w.total[1];
    for (uint32_t f = block / slices; f < many; f += groups)
        join_row<O, false>(a, w, w.common[f], block % slices, s_sum);
}

// ---- few tokens --------------------------------------------------------------------------
// (By one launch, and by four: 512 tokens by 3000 x 100 f32 6 and 18 us, 4096 17 and 21; 4096 by 32000 x 1024 33 and 44, by
// 50000 x 2048 108 and 101.  Four bytes each they are what a workgroup keeps on the chip beside its counts.)
constexpr int kFew = 4096, kFewLanes = kFew / kGroupThreads;
constexpr int kFewRows = 256;        // rows of a workgroup at most

// Up to kFew tokens by one launch: a workgroup reads all ids, puts the tokens of its up to `rows` rows in
// order of (row, place) in LDS and sums them in one slice of the columns.  The workgroups of a slice take runs of
// 2^run_bits neighbouring rows in turn: the commonest tokens are often neighbours (4096 tokens of text by 50000 x 512
// f16, 98 neighbouring rows each: 54 us instead of 18), while a run is to be worth a write.  `lanes` lanes are a group; each takes
// the same share of the tokens, and the sum of a row that reaches over several shares is put together
// by the group it starts in.  Bound by the waits of its steps (1000 tokens by 3000 x 100 f32: 6.6 us; four launches took 18),
// by its zeros where the table is large (100 by 1M x 256 f16: 96 us, 5.3 TB/s).
template <class T, class O>
__global__ __launch_bounds__(kGroupThreads) void few_kernel(EmbedArgs a, bool clears, int rows, int run_bits, int64_t blocks, int lanes, int64_t first) {
    using P = Piece<T>;
    constexpr int kAhead = 8;
    __shared__ uint32_t s_count[kGroupWaves * kFewRows], s_wave[kGroupWaves], s_start[kFewRows + 1];
    __shared__ uint32_t s_token[kFew];                              // bin << 16 | place among all tokens
    __shared__ float s_head[kGroupThreads * P::kLen];
    const int tid = threadIdx.x, wave = tid / kWave, lane = lane_id();
    const int64_t block = first + blockIdx.x;
    const uint32_t run = (1u << run_bits) - 1;
    auto row_of_bin = [&](int bin) { return (((int64_t)(bin >> run_bits) * blocks + block) << run_bits) + (bin & run); };
    const int n = (int)a.n, per = (n + kGroupThreads - 1) / kGroupThreads;      // rounds of 64 tokens for each wavefront
    int bin[kFewLanes], rank[kFewLanes];
#pragma unroll
    for (int j = 0; j < kFewLanes; j++) {
        const int i = (wave * per + j) * kWave + lane;
        const int64_t id = j < per && i < n ? id_at(a.ids, a.wide_ids, i) : -1;
        bin[j] = -1;
        if (id >= 0 && id < a.num_rows) {
            const uint32_t r = (uint32_t)id >> run_bits, turn = r / (uint32_t)blocks;
            if (r - turn * (uint32_t)blocks == (uint32_t)block) bin[j] = (int)(turn << run_bits | ((uint32_t)id & run));
        }
    }
    // all of its rows are zeros first, few are written again: nothing is waited for before these bytes leave
    const int group = tid / lanes, groups = kGroupThreads / lanes, c = ((int)blockIdx.y * lanes + tid % lanes) * P::kLen;
    const bool in = c < a.dim && group < groups, whole = c + P::kLen <= a.dim;
    if (in && clears)
        for (int r = group; r < rows; r += groups)
            if (row_of_bin(r) < a.num_rows) put_zeros<O, P::kLen>(a, row_of_bin(r), c);
    bool any = false;
#pragma unroll
    for (int j = 0; j < kFewLanes; j++) any |= bin[j] >= 0;
    for (int i = tid; i < kGroupWaves * kFewRows; i += kGroupThreads) s_count[i] = 0;
    if (!__syncthreads_or(any)) return;
    uint32_t* mine = s_count + wave * kFewRows;
#pragma unroll
    for (int j = 0; j < kFewLanes; j++) {
        if (j >= per) break;
        const unsigned long long here = __ballot(bin[j] >= 0);
        if (!here) continue;
        const unsigned long long same = same_key(here, (uint32_t)bin[j], 8);         // 2^8 = kFewRows
        if (bin[j] >= 0) {
            const uint32_t have = mine[bin[j]];
            rank[j] = have + lanes_below(same);
            if (lanes_below(same) == 0) mine[bin[j]] = have + __popcll(same);
        }
        wave_fence();
    }
    __syncthreads();
    uint32_t len = 0, all;
    if (tid < kFewRows)
        for (int v = 0; v < kGroupWaves; v++) len += s_count[v * kFewRows + tid];
    uint32_t start = group_scan<kGroupWaves>(len, 0, s_wave, &all);
    if (tid < kFewRows) {
        s_start[tid] = start;
        for (int v = 0; v < kGroupWaves; v++) {
            const uint32_t c = s_count[v * kFewRows + tid];
            s_count[v * kFewRows + tid] = start;
            start += c;
        }
        if (tid == kFewRows - 1) s_start[kFewRows] = start;
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < kFewLanes; j++)
        if (bin[j] >= 0) s_token[mine[bin[j]] + rank[j]] = (uint32_t)bin[j] << 16 | (uint32_t)((wave * per + j) * kWave + lane);
    __syncthreads();
    const int share = ((int)all + groups - 1) / groups;
    const int from = min((int)all, group * share), to = min((int)all, from + share);
    float sum[P::kLen];
#pragma unroll
    for (int k = 0; k < P::kLen; k++) sum[k] = 0.f;
    for (int t = from; t < to; t += kAhead) {
        uint32_t e[kAhead];
        u32x4 x[kAhead];
#pragma unroll
        for (int j = 0; j < kAhead; j++) e[j] = s_token[min(t + j, to - 1)];
#pragma unroll
        for (int j = 0; j < kAhead; j++) {
            const typename T::raw* row = (const typename T::raw*)a.rows + (int64_t)(e[j] & 0xffff) * a.stride;
            x[j] = u32x4{0, 0, 0, 0};
            if (whole) x[j] = P::load(row + c);
            else if (in) x[j] = P::load_part(row, c, a.dim, 0.f);
        }
#pragma unroll
        for (int j = 0; j < kAhead; j++) {
            if (t + j >= to) break;
            float y[P::kLen];
            P::unpack(x[j], y);
#pragma unroll
            for (int k = 0; k < P::kLen; k++) sum[k] += y[k];
            const int r = (int)(e[j] >> 16), last = (int)s_start[r + 1] - 1;
            if (t + j < last && t + j + 1 < to) continue;
            // the row ends here, or the share
            if ((int)s_start[r] < from) {
#pragma unroll
                for (int k = 0; k < P::kLen; k++) s_head[tid * P::kLen + k] = sum[k];
            } else if (t + j == last) {
                if (in) put_sums<O, P::kLen>(a, (uint32_t)row_of_bin(r), c, sum);
            } else {
                continue;                                          // the others' parts are to come
            }
#pragma unroll
            for (int k = 0; k < P::kLen; k++) sum[k] = 0.f;
        }
    }
    __syncthreads();
    if (from >= to || !in) return;
    const int r = (int)(s_token[to - 1] >> 16), end = (int)s_start[r + 1];
    if ((int)s_start[r] < from || end <= to) return;
    for (int g = group + 1; g * share < end; g++)
#pragma unroll
        for (int k = 0; k < P::kLen; k++) sum[k] += s_head[(g * lanes + tid % lanes) * P::kLen + k];
    put_sums<O, P::kLen>(a, (uint32_t)row_of_bin(r), c, sum);
}

constexpr int64_t kMaxGrid = 1 << 22;     // workgroups of one launch (their threads are counted in 32 bits)

// Lanes for a row of n pieces, or for a share of it in whole lines of 128 bytes each of the fewest times: up to `most`
// (a multiple of 8).  A line that two workgroups write in part costs both a line: 1 token by 250000 x 960 f32 262 us with
// shares of 60 pieces, 180 with 64.
int lanes_for(int n, int most) {
    const int times = (n + most - 1) / most;
    return times == 1 ? n : ((n + times - 1) / times + 7) / 8 * 8;
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
template <class O>
int room_for_counts() {
    static DeviceOnce once;
    return once.run([] {
        DCIH_HIP(hipFuncSetAttribute((const void*)chunk_kernel<O>, hipFuncAttributeMaxDynamicSharedMemorySize,
                                     kGroupWaves * (int)sizeof(uint32_t) << kMaxBucketBits));
        return 0;
    });
}

// The launch of chunk_kernel, which groups (w.chunks) and clears (w.cleared).
template <class O>
int group_and_clear(const EmbedArgs& a, const Work& w, hipStream_t s) {
    constexpr int kCleared = kGroupThreads * Piece<O>::kLen;       // elements, by a workgroup
    const int64_t clearing = (w.cleared * a.dim + kCleared - 1) / kCleared;
    const size_t room = w.chunks ? kGroupWaves * sizeof(uint32_t) << w.bucket_bits : 0;
    chunk_kernel<O><<<(uint32_t)(w.chunks + clearing), kGroupThreads, room, s>>>(a, w);
    DCIH_HIP(hipGetLastError());
    return 0;
}
template <class O>
bool one_launch_clears(const EmbedArgs& a) { return a.num_rows <= kMaxGrid * kGroupThreads * Piece<O>::kLen / a.dim; }

template <class T, class O>
int grad_of_few(const EmbedArgs& a, hipStream_t s) {
    // a row of up to 128 pieces is not shared by workgroups (4000 tokens by 50000 x 520 f16 22 us, 26 in two slices), longer
    // ones are by 64 (by 50000 x 2048 39 us, 42 with 128)
    const int pieces = (a.dim + Piece<T>::kLen - 1) / Piece<T>::kLen, lanes = lanes_for(pieces, pieces <= 2 * kWave ? 2 * kWave : kWave);
    // runs of 512 bytes or more; 512 workgroups to fill the device, each of which reads all ids (83 tokens by 5130 x
    // 1872 f32 11 us, 19 with as many for each of the 8 slices, 4000 by 32000 x 4096 f16 65 and 91); where rows share
    // lines and few tokens can be one workgroup's, of 4096 (32 tokens by 410256 x 624 f16: 107 us, 142 with runs of a
    // row)
    const int64_t row_bytes = (int64_t)a.dim * (int)sizeof(typename O::raw), run_bytes = a.n <= 256 && row_bytes % 128 ? 4096 : 512;
    int run_bits = 0;
    while (run_bits < 3 && row_bytes << run_bits < run_bytes) run_bits++;
    const int64_t runs = ((a.num_rows - 1) >> run_bits) + 1;
    const int64_t slices = (pieces + lanes - 1) / lanes;
    const int64_t turns = std::min<int64_t>(kFewRows >> run_bits, std::max<int64_t>(std::max(1, 8 >> run_bits), (runs * slices + 511) / 512));
    const int64_t blocks = (runs + turns - 1) / turns;
    const int rows = (int)(turns << run_bits);
    // tables of 768 MB and more are cleared by a launch of their own (100 tokens by 1M x 256 f32 175 us, 190 by few_kernel alone;
    // by half of that table 102 and 98)
    bool clears = !a.accumulate;
    if (clears && a.num_rows * row_bytes >= (int64_t)768 << 20 && one_launch_clears<O>(a)) {
        Work w{};
        w.cleared = a.num_rows;
        if (int rc = group_and_clear<O>(a, w, s)) return rc;
        clears = false;
    }
    const int64_t most = std::max<int64_t>(1, kMaxGrid / slices);
    for (int64_t first = 0; first < blocks; first += most) {
        few_kernel<T, O><<<dim3((uint32_t)std::min(most, blocks - first), (uint32_t)slices), kGroupThreads, 0, s>>>(a, clears, rows, run_bits, blocks, lanes, first);
        DCIH_HIP(hipGetLastError());
    }
    return 0;
}

template <class T, class O>
int grad(const EmbedArgs& a, hipStream_t s) {
    if (a.n <= kFew) return grad_of_few<T, O>(a, s);
    Work w;
    lay_out(w, a.work, a.n, a.dim, a.num_rows);
    if (int rc = room_for_counts<O>()) return rc;
    // Tables that stay empty for the most part are cleared first: 100000 tokens by 1M x 128 f32 125 us instead of 129, 20000 110
    // instead of 120; but 65536 by 262144 x 512 f16 73 instead of 71.
    w.cleared = !a.accumulate && a.num_rows >= 8 * a.n && one_launch_clears<O>(a) ? a.num_rows : 0;
    if (int rc = group_and_clear<O>(a, w, s)) return rc;
    const int out_lanes = lanes_for((a.dim + Piece<O>::kLen - 1) / Piece<O>::kLen, kWave);
    if (a.accumulate || w.cleared) bucket_kernel<O, false><<<1u << w.bucket_bits, kGroupThreads, 0, s>>>(a, w, out_lanes);
    else bucket_kernel<O, true><<<1u << w.bucket_bits, 2 * kGroupThreads, 0, s>>>(a, w, out_lanes);
    DCIH_HIP(hipGetLastError());
    const int pieces = (a.dim + Piece<T>::kLen - 1) / Piece<T>::kLen, lanes = lanes_for(pieces, kWave);
    const int slices = (pieces + lanes - 1) / lanes, per = kThreads / lanes;
    const int64_t units = w.windows * slices;
    for (int64_t first = 0; first < units; first += kMaxGrid * per) {
        const int64_t groups = std::min(kMaxGrid, (units - first + per - 1) / per);
        if (lanes == kWave) sum_kernel<T, O, true><<<(uint32_t)groups, kThreads, 0, s>>>(a, w, lanes, slices, first);
        else sum_kernel<T, O, false><<<(uint32_t)groups, kThreads, 0, s>>>(a, w, lanes, slices, first);
        DCIH_HIP(hipGetLastError());
    }
    // groups of workgroups that fill the device, no more than there can be such rows
    const int wide = (int)std::min<int64_t>(a.n / (w.piece * kWide + 1), 16), groups = (int)std::min<int64_t>(a.n / (w.piece + 1), 1024);
    const int64_t blocks = (int64_t)wide * ((a.dim + 63) / 64) + (int64_t)groups * ((a.dim + kThreads * 4 - 1) / (kThreads * 4));
    join_kernel<O><<<(uint32_t)blocks, kThreads, 0, s>>>(a, w, wide, groups);
    DCIH_HIP(hipGetLastError());
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
    return n <= kFew ? 16 : lay_out(w, nullptr, n, dim, num_rows);
}

int embed_grad(const EmbedArgs& a, int dtype, int out_dtype, hipStream_t s) {
    switch (dtype) {
        case DCIH_F32: return grad<F32, F32>(a, s);
        case DCIH_F16: return out_dtype == DCIH_F32 ? grad<F16, F32>(a, s) : grad<F16, F16>(a, s);
        default: return out_dtype == DCIH_F32 ? grad<BF16, F32>(a, s) : grad<BF16, BF16>(a, s);
    }
}

}  // namespace dcih
