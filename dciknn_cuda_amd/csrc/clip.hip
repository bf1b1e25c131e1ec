// The norm of all gradients of a model, and gradients times a factor that bounds it:
//
//   norm = |scale| sqrt(sum of g^2),      out = g * scale * min(1, max_norm / norm)
//
// Squares are summed in 64 bits: no value of any type overflows or vanishes there, and the vector units form as many of these
// as of 32 bits.  The sum's order depends on the spans alone.  Tables of spans go to the kernels as arguments, kSpans a launch: nothing
// is copied to the device, so a recorded call reads nothing of the host.
#include "../../include/dci_hip.h"
#include "clip.h"

#include <algorithm>
#include <cmath>

namespace dcih {
namespace {

constexpr int kThreads = 256;
constexpr int kRead = 240, kWritten = 160;      // spans of a launch: 3.9 KB of arguments
constexpr int64_t kMaxUnit = 65536;             // elements that a workgroup takes at a time, 2048 at least
constexpr int64_t kUnits = 8192;                // in all, where units are not the largest yet
constexpr int64_t kFewSums = kThreads;          // up to here every workgroup joins the sums itself
constexpr int64_t kMaxSpan = (int64_t)1 << 31;  // elements of an entry: longer spans are several
constexpr int64_t kMaxGrid = 1 << 23;
constexpr uint32_t kBlocks = 1024;              // workgroups of a launch that writes (that one with 4096 660 us)

// Where spans lie. A type is kept beside the address, which has 57 bits.
struct Place {
    uint64_t bits;
    __host__ void set(const void* p, int dtype) { bits = (uint64_t)(uintptr_t)p | (uint64_t)dtype << 60; }
    __device__ int dtype() const { return (int)(bits >> 60); }
    template <class T> __device__ typename T::raw* at(int64_t i) const { return (typename T::raw*)(uintptr_t)(bits & ((1ull << 60) - 1)) + i; }
};
struct Entry { Place in; uint32_t count, first; };          // `first`: the first unit of the launch
struct ReadTable {
    int spans;
    uint32_t units, unit;
    Entry e[kRead];
    __host__ void set(int i, const void* data, int dtype, const void*, int) { e[i].in.set(data, dtype); }
    static constexpr int kRoom = kRead;
};
struct WriteTable {
    int spans;
    uint32_t units, unit;
    bool moves;                 // something is written to another place
    Entry e[kWritten];
    Place out[kWritten];
    __host__ void set(int i, const void* data, int dtype, void* to, int out_dtype) {
        e[i].in.set(data, dtype);
        out[i].set(to, out_dtype);
        moves = (i && moves) || e[i].in.bits != out[i].bits;
    }
    static constexpr int kRoom = kWritten;
};

// The span of a unit: the last that begins at it or before.
template <class Table> __device__ inline int span_of(const Table& t, uint32_t unit) {
    int lo = 0, hi = t.spans;
    while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (t.e[mid].first <= unit) lo = mid;
        else hi = mid;
    }
    return lo;
}

__device__ inline double sum_of_lanes(double v) {
#pragma unroll
    for (int o = kWave / 2; o; o /= 2) v += __builtin_bit_cast(double, lane_xor_any(__builtin_bit_cast(unsigned long long, v), o));
    return v;
}
// Over a workgroup, in one order; every thread gets it.
__device__ inline double sum_of_threads(double v, double* s_part) {
    v = sum_of_lanes(v);
    if (lane_id() == 0) s_part[threadIdx.x / kWave] = v;
    __syncthreads();
    v = 0.0;
    for (int w = 0; w < (int)blockDim.x / kWave; w++) v += s_part[w];
    return v;
}

template <class T> __device__ double squares(const typename T::raw* p, int64_t n) {
    using P = Piece<T>;
    constexpr int U = 8;
    const int64_t pieces = n / P::kLen;
    double sum[2] = {0.0, 0.0};
    auto add = [&](u32x4 x) {
        float z[P::kLen];
        P::unpack(x, z);
#pragma unroll
        for (int k = 0; k < P::kLen; k++) sum[k & 1] = __builtin_fma((double)z[k], (double)z[k], sum[k & 1]);
    };
    int64_t i = threadIdx.x;
    for (; i + (U - 1) * kThreads < pieces; i += U * kThreads) {
        u32x4 x[U];
#pragma unroll
        for (int u = 0; u < U; u++) x[u] = P::load(p + (i + u * kThreads) * P::kLen);
#pragma unroll
        for (int u = 0; u < U; u++) add(x[u]);
    }
    for (; i < pieces; i += kThreads) add(P::load(p + i * P::kLen));
    const int64_t rest = pieces * P::kLen + threadIdx.x;
    if (rest < n) sum[0] = __builtin_fma((double)(float)p[rest], (double)(float)p[rest], sum[0]);
    return sum[0] + sum[1];
}

// One pass over all gradients, bound by memory: 564M bf16 181 us (6.2 TB/s), 382M f32 255 us (6.0); of 1000 f16 tensors of 1 to 1M elements
// five launches of 10 us, more than their bytes take, for each has to fill the device by itself.
__global__ __launch_bounds__(kThreads) void squares_kernel(ReadTable t, double* sums) {
    __shared__ double s_part[kThreads / kWave];
    const uint32_t unit = blockIdx.x;
    const Entry e = t.e[span_of(t, unit)];
    const int64_t from = (int64_t)(unit - e.first) * t.unit, n = min((int64_t)t.unit, (int64_t)e.count - from);
    double sum;
    switch (e.in.dtype()) {
        case DCIH_F32: sum = squares<F32>(e.in.at<F32>(from), n); break;
        case DCIH_F16: sum = squares<F16>(e.in.at<F16>(from), n); break;
        default: sum = squares<BF16>(e.in.at<BF16>(from), n);
    }
    sum = sum_of_threads(sum, s_part);
    if (threadIdx.x == 0) sums[unit] = sum;
}

__device__ inline double sum_of(const double* sums, int64_t n, double* s_part) {
    double sum = 0.0;
    for (int64_t i = threadIdx.x; i < n; i += blockDim.x) sum += sums[i];
    return sum_of_threads(sum, s_part);
}

// The sum of the units' sums, behind them, and the norm.
__global__ __launch_bounds__(1024) void norm_kernel(double* sums, int64_t n, double scale, float* norm) {
    __shared__ double s_part[1024 / kWave];
    const double sum = sum_of(sums, n, s_part);
    if (threadIdx.x) return;
    sums[n] = sum;
    *norm = (float)(sqrt(sum) * scale);
}

// L elements in the place of L others: 16 bytes of what is written, so that a wavefront's stores are whole lines.  (564M bf16 into f32 645 us,
// 5.2 TB/s; with 16 bytes of what is read, and every second piece of 16 bytes written at a time, 1024.)
template <class T, class O> __device__ void scaled(const typename T::raw* p, typename O::raw* out, int64_t n, float factor) {
    constexpr int U = 8, L = Piece<O>::kLen;
    typedef typename T::raw in_vec __attribute__((ext_vector_type(L)));
    typedef in_vec in_vec_any __attribute__((aligned(sizeof(typename T::raw))));
    typedef float float_vec __attribute__((ext_vector_type(L)));
    const int64_t pieces = n / L;
    auto get = [&](int64_t i) -> in_vec { return *(const in_vec_any*)(p + i * L); };
    auto put = [&](int64_t i, in_vec x) {
        const float_vec y = __builtin_convertvector(x, float_vec) * factor;
        float z[L];
#pragma unroll
        for (int k = 0; k < L; k++) z[k] = y[k];
        Piece<O>::store_once(out + i * L, Piece<O>::pack(z));
    };
    int64_t i = threadIdx.x;
    for (; i + (U - 1) * kThreads < pieces; i += U * kThreads) {
        in_vec x[U];
#pragma unroll
        for (int u = 0; u < U; u++) x[u] = get(i + u * kThreads);
#pragma unroll
        for (int u = 0; u < U; u++) put(i + u * kThreads, x[u]);
    }
    for (; i < pieces; i += kThreads) put(i, get(i));
    const int64_t rest = pieces * L + threadIdx.x;
    if (rest < n) out[rest] = (typename O::raw)((float)p[rest] * factor);
}

// The tables come in reverse: what the sums read last is in the caches still.  Where nothing is clipped or scaled and the
// gradients stay in their place there is nothing to do.
__global__ __launch_bounds__(kThreads) void clip_kernel(WriteTable t, const double* sums, int64_t n, bool joined, double scale, double max_norm, float* norm) {
    __shared__ double s_part[kThreads / kWave];
    const double total = (joined ? sums[n] : sum_of(sums, n, s_part)), length = sqrt(total) * fabs(scale);
    if (norm && blockIdx.x == 0 && threadIdx.x == 0) *norm = (float)length;
    // (a norm that is no number, or infinite as it is returned, clips nothing)
    const float factor = (float)(length > max_norm && (float)length < __builtin_huge_valf() ? max_norm / length * scale : scale);
    if (factor == 1.f && !t.moves) return;
    for (uint32_t unit = blockIdx.x; unit < t.units; unit += gridDim.x) {
        const int i = span_of(t, unit);
        const Entry e = t.e[i];
        const Place out = t.out[i];
        if (factor == 1.f && e.in.bits == out.bits) continue;
        const int64_t from = (int64_t)(unit - e.first) * t.unit, left = min((int64_t)t.unit, (int64_t)e.count - from);
        switch (3 * e.in.dtype() + out.dtype()) {
            case 3 * DCIH_F32 + DCIH_F32: scaled<F32, F32>(e.in.at<F32>(from), out.at<F32>(from), left, factor); break;
            case 3 * DCIH_F16 + DCIH_F16: scaled<F16, F16>(e.in.at<F16>(from), out.at<F16>(from), left, factor); break;
            case 3 * DCIH_F16 + DCIH_F32: scaled<F16, F32>(e.in.at<F16>(from), out.at<F32>(from), left, factor); break;
            case 3 * DCIH_BF16 + DCIH_F32: scaled<BF16, F32>(e.in.at<BF16>(from), out.at<F32>(from), left, factor); break;
            default: scaled<BF16, BF16>(e.in.at<BF16>(from), out.at<BF16>(from), left, factor);
        }
    }
}

int64_t units_of(int64_t count, int64_t unit) { return (count + unit - 1) / unit; }

// Elements of a unit, a power of two: as few as give no more than about kUnits of them.
int64_t unit_for(const dcih_span* spans, int64_t n, int64_t& units) {
    int64_t all = 0;
    for (int64_t i = 0; i < n; i++) all += spans[i].count;
    int bits = 11;
    while (((int64_t)1 << bits) < kMaxUnit && (all >> bits) + n > kUnits) bits++;
    units = 0;
    for (int64_t i = 0; i < n; i++) units += (spans[i].count + ((int64_t)1 << bits) - 1) >> bits;
    return (int64_t)1 << bits;
}

// Calls `launch` with tables of the spans in order, or with the same ones from the last to the first.
template <class Table, class Launch>
int by_tables(const dcih_span* spans, int64_t n, int64_t unit, bool reverse, Launch launch) {
    // (parts of spans: of kMaxSpan elements each but the last)
    auto parts_of = [&](int64_t i) { return (spans[i].count + kMaxSpan - 1) / kMaxSpan; };
    int64_t i = reverse ? n - 1 : 0, part = reverse && n ? parts_of(i) - 1 : 0, before = 0;
    auto more = [&] { return reverse ? i >= 0 : i < n; };
    auto next = [&] {
        if (reverse) {
            if (--part < 0 && --i >= 0) part = parts_of(i) - 1;
        } else if (++part >= parts_of(i)) {
            i++;
            part = 0;
        }
    };
    Table t;
    t.unit = (uint32_t)unit;
    while (more()) {
        t.spans = 0;
        t.units = 0;
        for (; more() && t.spans < Table::kRoom; next()) {
            if (part < 0 || part >= parts_of(i)) continue;          // an empty span
            const int64_t from = part * kMaxSpan, count = std::min(kMaxSpan, spans[i].count - from);
            t.set(t.spans, (const char*)spans[i].data + from * type_bytes(spans[i].dtype), spans[i].dtype,
                  (char*)spans[i].out + from * type_bytes(spans[i].out_dtype), spans[i].out_dtype);
            t.e[t.spans].count = (uint32_t)count;
            t.e[t.spans++].first = t.units;
            t.units += (uint32_t)units_of(count, unit);
        }
        if (t.spans)
            if (int rc = launch(t, before)) return rc;
        before += t.units;
    }
    return 0;
}

int sum_up(const dcih_span* spans, int64_t n, int64_t unit, double* sums, hipStream_t s) {
    return by_tables<ReadTable>(spans, n, unit, false, [&](const ReadTable& t, int64_t at) {
        squares_kernel<<<t.units, kThreads, 0, s>>>(t, sums + at);
        DCIH_HIP(hipGetLastError());
        return 0;
    });
}

int join(double* sums, int64_t units, double scale, float* norm, hipStream_t s) {
    norm_kernel<<<1, 1024, 0, s>>>(sums, units, fabs(scale), norm);
    DCIH_HIP(hipGetLastError());
    return 0;
}

}  // namespace

int64_t clip_work_bytes(const dcih_span* spans, int64_t n) {
    int64_t units;
    unit_for(spans, n, units);
    return (units + 2) * 8;
}

bool clip_fits(const dcih_span* spans, int64_t n) {
    int64_t units;
    unit_for(spans, n, units);
    return units <= kMaxGrid;
}

int grad_norm(const dcih_span* spans, int64_t n, double scale, float* norm, void* work, hipStream_t s) {
    int64_t units;
    const int64_t unit = unit_for(spans, n, units);
    if (int rc = sum_up(spans, n, unit, (double*)work, s)) return rc;
    return join((double*)work, units, scale, norm, s);
}

int clip_grads(const dcih_span* spans, int64_t n, double max_norm, double scale, float* norm, void* work, hipStream_t s) {
    int64_t units;
    const int64_t unit = unit_for(spans, n, units);
    double* sums = (double*)work;
    if (int rc = sum_up(spans, n, unit, sums, s)) return rc;
    const bool joined = units > kFewSums || !units;
    if (joined)
        if (int rc = join(sums, units, scale, norm, s)) return rc;
    bool first = !joined;
    return by_tables<WriteTable>(spans, n, unit, true, [&](const WriteTable& t, int64_t) {
        clip_kernel<<<std::min(t.units, kBlocks), kThreads, 0, s>>>(t, sums, units, joined, scale, max_norm, first ? norm : nullptr);
        DCIH_HIP(hipGetLastError());
        first = false;
        return 0;
    });
}

}  // namespace dcih
