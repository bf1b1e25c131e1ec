// Rows of a table by ids, times a factor, and the gradient of that by the table:
//
//   out[i, :] = scale * W[id_i, :]            dW[v, :] = scale * sum over i with id_i = v of G[i, :]
//
// Both are bound by memory.  The gradient's sums are formed without atomics on values, in the
// order of the tokens whatever the schedule: the tokens are first grouped by their row (group_kernel),
// then summed in pieces of up to kPiece tokens of one row (sum_kernel); the pieces of rows with more
// tokens than that are joined by a third launch (join_kernel).  Sums are in 32 bits, rounded once.
#include "../../include/dci_hip.h"
#include "token_common.h"

#include <algorithm>

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

constexpr int kGroupThreads = 1024, kGroupWaves = kGroupThreads / kWave;
constexpr int kBins = 1024;          // rows of one bucket
constexpr int kPiece = 32;           // tokens of a row that are summed by one group of lanes

struct Work {
    uint32_t* total;        // tokens with a row
    Token* tokens;          // [n]
    float* part;            // [2 * windows][width]: see sum_kernel
    int64_t windows;
    int width;
};
__host__ __device__ inline Work work_of(void* mem, int64_t n, int dim) {
    Work w;
    w.total = (uint32_t*)mem;
    w.tokens = (Token*)((char*)mem + 256);
    w.part = (float*)((char*)mem + 256 + n * sizeof(Token));
    w.windows = (n + kPiece - 1) / kPiece;
    w.width = (dim + 7) & ~7;
    return w;
}

__device__ inline int lanes_below(unsigned long long mask) {
    return __builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0));
}

// Bucket b holds the rows r with r mod buckets = b (a power of two: neighbouring rows, often alike in
// their number of tokens, go to different buckets).  Each workgroup reads all ids: once to count
// its rows' tokens and those of the buckets before it, which is where its part of the output starts,
// and once to put its tokens into their places.  A wavefront takes a run of the tokens, so that
// its counts in front of the places give the order of the tokens.
__global__ __launch_bounds__(kGroupThreads) void group_kernel(const void* ids, bool wide, int64_t n, int64_t num_rows, int bucket_bits,
                                                              Token* tokens, uint32_t* total) {
    __shared__ uint32_t s_count[kGroupWaves][kBins];
    __shared__ uint32_t s_start[kBins], s_len[kBins];
    __shared__ uint32_t s_wave[kGroupWaves], s_before[kGroupWaves];
    const int tid = threadIdx.x, lane = lane_id(), wave = tid / kWave;
    const uint32_t bucket = blockIdx.x, mask_bits = (1u << bucket_bits) - 1;
    for (int w = 0; w < kGroupWaves; w++) s_count[w][tid] = 0;
    static_assert(kBins == kGroupThreads, "a thread per bin");
    __syncthreads();
    const int64_t run = ((n + kGroupThreads - 1) / kGroupThreads) * kWave;
    const int64_t from = min(n, wave * run), to = min(n, from + run);
    uint32_t before = 0;
    for (int64_t i = from + lane; i - lane < to; i += kWave) {
        const int64_t id = i < to ? id_at(ids, wide, i) : -1;
        const bool real = id >= 0 && id < num_rows;
        const uint32_t in = (uint32_t)id & mask_bits;
        before += real && in < bucket;
        if (real && in == bucket) atomicAdd(&s_count[wave][(uint32_t)id >> bucket_bits], 1u);
    }
    before = wave_sum_u32(before);
    if (lane == 0) s_before[wave] = before;
    __syncthreads();
    // counts become the places of a wavefront's tokens among their row's
    uint32_t len = 0;
#pragma unroll
    for (int w = 0; w < kGroupWaves; w++) {
        const uint32_t c = s_count[w][tid];
        s_count[w][tid] = len;
        len += c;
    }
    const uint32_t upto = wave_scan_u32(len);
    if (lane == kWave - 1) s_wave[wave] = upto;
    __syncthreads();
    uint32_t start = upto - len;
    for (int w = 0; w < kGroupWaves; w++) {
        start += s_before[w];
        if (w < wave) start += s_wave[w];
    }
    s_start[tid] = start;
    s_len[tid] = len;
    if (bucket == mask_bits && tid == kBins - 1) *total = start + len;
    __syncthreads();
    for (int64_t i = from + lane; i - lane < to; i += kWave) {
        const int64_t id = i < to ? id_at(ids, wide, i) : -1;
        const bool mine = id >= 0 && id < num_rows && ((uint32_t)id & mask_bits) == bucket;
        unsigned long long same = __ballot(mine);
        if (!same) continue;
        const uint32_t bin = mine ? (uint32_t)id >> bucket_bits : 0;
#pragma unroll
        for (int b = 0; b < 10; b++) {                // 2^10 = kBins
            const unsigned long long ones = __ballot(bin >> b & 1);
            same &= bin >> b & 1 ? ones : ~ones;
        }
        if (mine) {
            const uint32_t rank = s_count[wave][bin] + lanes_below(same);
            if (lanes_below(same) == 0) s_count[wave][bin] = rank + __popcll(same);
            tokens[s_start[bin] + rank] = Token{(uint32_t)id, (uint32_t)i, rank, s_len[bin]};
        }
    }
}

// ---- sums --------------------------------------------------------------------------------
template <class O>
__global__ __launch_bounds__(kThreads) void zero_kernel(typename O::raw* out, int64_t n) {
    using P = Piece<O>;
    const u32x4 none = {0, 0, 0, 0};
    for (int64_t i = ((int64_t)blockIdx.x * kThreads + threadIdx.x) * P::kLen; i < n; i += (int64_t)gridDim.x * kThreads * P::kLen) {
        if (i + P::kLen <= n) P::store(out + i, none);
        else for (int64_t j = i; j < n; j++) out[j] = (typename O::raw)0.f;
    }
}

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

// `lanes` (a power of two up to 64) neighbouring lanes take one window of kPiece tokens in one slice of
// the columns: they sum the pieces that START in the window, up to kPiece tokens of one row each.
// Rows of up to kPiece tokens are one piece and final; the first piece of a longer one goes to
// place 2 w + 1 of `part`, a later one to 2 w (a window w has at most one of each).
template <class T, class O>
__global__ __launch_bounds__(kThreads) void sum_kernel(EmbedArgs a, Work w, int lanes, int slices, int64_t first) {
    using P = Piece<T>;
    constexpr int kAhead = 8;
    const int64_t unit = first + (int64_t)blockIdx.x * (kThreads / lanes) + threadIdx.x / lanes;
    const int64_t window = unit / slices, total = *w.total;
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

template <class T, class O>
int grad(const EmbedArgs& a, hipStream_t s) {
    const Work w = work_of(a.work, a.n, a.dim);
    if (!a.accumulate) {
        const int64_t cells = a.num_rows * a.dim, per = (int64_t)kThreads * Piece<O>::kLen;
        zero_kernel<O><<<(uint32_t)std::min<int64_t>(8192, (cells + per - 1) / per), kThreads, 0, s>>>((typename O::raw*)a.out, cells);
        DCIH_HIP(hipGetLastError());
    }
    if (!a.n) return 0;
    int bits = 0;
    while (a.num_rows > (int64_t)kBins << bits) bits++;
    group_kernel<<<1u << bits, kGroupThreads, 0, s>>>(a.ids, a.wide_ids, a.n, a.num_rows, bits, w.tokens, w.total);
    DCIH_HIP(hipGetLastError());
    const int pieces = (a.dim + Piece<T>::kLen - 1) / Piece<T>::kLen, lanes = lanes_for(pieces, kWave);
    int slices = (pieces + lanes - 1) / lanes;
    const int per = kThreads / lanes;
    int64_t units = w.windows * slices;
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

size_t embed_grad_bytes(int64_t n, int dim) {
    const Work w = work_of(nullptr, n, dim);
    return 256 + (size_t)n * sizeof(Token) + (size_t)w.windows * 2 * w.width * sizeof(float);
}

int embed_grad(const EmbedArgs& a, int dtype, int out_dtype, hipStream_t s) {
    switch (dtype) {
        case DCIH_F32: return grad<F32, F32>(a, s);
        case DCIH_F16: return out_dtype == DCIH_F32 ? grad<F16, F32>(a, s) : grad<F16, F16>(a, s);
        default: return out_dtype == DCIH_F32 ? grad<BF16, F32>(a, s) : grad<BF16, BF16>(a, s);
    }
}

}  // namespace dcih
