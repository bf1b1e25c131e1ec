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
constexpr int kSpans = 120;                     // of a launch: 3.8 KB of arguments
constexpr int64_t kMinUnit = 2048, kMaxUnit = 65536;     // elements that a workgroup takes
constexpr int64_t kUnits = 4096;                // in all, where units are not the largest yet
constexpr int64_t kFewSums = kThreads;          // up to here every workgroup joins the sums itself
constexpr int64_t kMaxGrid = 1 << 23;

struct Table {
    const void* in[kSpans];
    void* out[kSpans];
    int64_t count[kSpans];
    uint32_t first[kSpans];                     // a span's first unit of the launch
    uint8_t types[kSpans];                      // 3 * type + type of what is written
    int spans;
    uint32_t units;
    int64_t unit;                               // elements
};

// The span of a unit: the last that begins at it or before.
__device__ inline int span_of(const Table& t, uint32_t unit) {
    int lo = 0, hi = t.spans;
    while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (t.first[mid] <= unit) lo = mid;
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

// One pass over all gradients, bound by memory.
__global__ __launch_bounds__(kThreads) void squares_kernel(Table t, double* sums) {
    __shared__ double s_part[kThreads / kWave];
    const uint32_t unit = blockIdx.x;
    const int i = span_of(t, unit);
    const int64_t from = (int64_t)(unit - t.first[i]) * t.unit, n = min(t.unit, t.count[i] - from);
    double sum;
    switch (t.types[i] / 3) {
        case DCIH_F32: sum = squares<F32>((const float*)t.in[i] + from, n); break;
        case DCIH_F16: sum = squares<F16>((const _Float16*)t.in[i] + from, n); break;
        default: sum = squares<BF16>((const __bf16*)t.in[i] + from, n);
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

template <class T, class O> __device__ void scaled(const typename T::raw* p, typename O::raw* out, int64_t n, float factor) {
    using P = Piece<T>;
    constexpr int U = 8, L = P::kLen, K = Piece<O>::kLen;
    const int64_t pieces = n / L;
    auto put = [&](int64_t i, u32x4 x) {
        float z[L];
        P::unpack(x, z);
#pragma unroll
        for (int k = 0; k < L; k++) z[k] *= factor;
#pragma unroll
        for (int k = 0; k < L; k += K) {
            float y[K];
#pragma unroll
            for (int j = 0; j < K; j++) y[j] = z[k + j];
            Piece<O>::store_once(out + i * L + k, Piece<O>::pack(y));
        }
    };
    int64_t i = threadIdx.x;
    for (; i + (U - 1) * kThreads < pieces; i += U * kThreads) {
        u32x4 x[U];
#pragma unroll
        for (int u = 0; u < U; u++) x[u] = P::load(p + (i + u * kThreads) * L);
#pragma unroll
        for (int u = 0; u < U; u++) put(i + u * kThreads, x[u]);
    }
    for (; i < pieces; i += kThreads) put(i, P::load(p + i * L));
    const int64_t rest = pieces * L + threadIdx.x;
    if (rest < n) out[rest] = (typename O::raw)((float)p[rest] * factor);
}

// The last units first: what the sums read last is in the caches still.  Where nothing is clipped or scaled and the
// gradients stay in their place there is nothing to do.
__global__ __launch_bounds__(kThreads) void clip_kernel(Table t, const double* sums, int64_t n, bool joined, double scale, double max_norm, float* norm) {
    __shared__ double s_part[kThreads / kWave];
    const double total = (joined ? sums[n] : sum_of(sums, n, s_part)), length = sqrt(total) * fabs(scale);
    if (norm && blockIdx.x == 0 && threadIdx.x == 0) *norm = (float)length;
    // (a norm that is no number, or infinite as it is returned, clips nothing)
    const float factor = (float)(length > max_norm && (float)length < __builtin_huge_valf() ? max_norm / length * scale : scale);
    const uint32_t unit = t.units - 1 - blockIdx.x;
    const int i = span_of(t, unit);
    if (factor == 1.f && t.in[i] == t.out[i]) return;
    const int64_t from = (int64_t)(unit - t.first[i]) * t.unit, left = min(t.unit, t.count[i] - from);
    switch (t.types[i]) {
        case 3 * DCIH_F32 + DCIH_F32: scaled<F32, F32>((const float*)t.in[i] + from, (float*)t.out[i] + from, left, factor); break;
        case 3 * DCIH_F16 + DCIH_F16: scaled<F16, F16>((const _Float16*)t.in[i] + from, (_Float16*)t.out[i] + from, left, factor); break;
        case 3 * DCIH_F16 + DCIH_F32: scaled<F16, F32>((const _Float16*)t.in[i] + from, (float*)t.out[i] + from, left, factor); break;
        case 3 * DCIH_BF16 + DCIH_F32: scaled<BF16, F32>((const __bf16*)t.in[i] + from, (float*)t.out[i] + from, left, factor); break;
        default: scaled<BF16, BF16>((const __bf16*)t.in[i] + from, (__bf16*)t.out[i] + from, left, factor);
    }
}

int64_t units_of(int64_t count, int64_t unit) { return (count + unit - 1) / unit; }

// Elements of a unit: as few as give no more than kUnits of them.
int64_t unit_for(const dcih_span* spans, int64_t n, int64_t& units) {
    for (int64_t unit = kMinUnit;; unit *= 2) {
        units = 0;
        for (int64_t i = 0; i < n; i++) units += units_of(spans[i].count, unit);
        if (units <= kUnits || unit == kMaxUnit) return unit;
    }
}

// Calls `launch` with tables of the spans in order, or in reverse.
template <class Launch>
int by_tables(const dcih_span* spans, int64_t n, int64_t unit, bool reverse, Launch launch) {
    int64_t before = 0, all = 0;
    for (int64_t i = 0; i < n; i++) all += units_of(spans[i].count, unit);
    Table t;
    t.unit = unit;
    t.spans = 0;
    t.units = 0;
    auto flush = [&](int64_t at) {
        const int rc = t.spans ? launch(t, at) : 0;
        t.spans = 0;
        t.units = 0;
        return rc;
    };
    // (a table holds spans [from, to) in ascending order in both directions)
    int64_t from = 0, to = reverse ? n : 0;
    while (reverse ? to > 0 : from < n) {
        if (reverse) {
            from = to;
            for (int taken = 0; from > 0 && taken < kSpans; ) taken += spans[--from].count > 0;
        } else {
            to = from;
            for (int taken = 0; to < n && taken < kSpans; ) taken += spans[to++].count > 0;
        }
        for (int64_t i = from; i < to; i++) {
            if (!spans[i].count) continue;
            t.in[t.spans] = spans[i].data;
            t.out[t.spans] = spans[i].out;
            t.count[t.spans] = spans[i].count;
            t.types[t.spans] = (uint8_t)(3 * spans[i].dtype + spans[i].out_dtype);
            t.first[t.spans++] = t.units;
            t.units += (uint32_t)units_of(spans[i].count, unit);
        }
        const int64_t taken = t.units;
        if (int rc = flush(reverse ? all - before - taken : before)) return rc;
        before += taken;
        if (reverse) to = from;
        else from = to;
    }
    return 0;
}

int sum_up(const dcih_span* spans, int64_t n, int64_t unit, double* sums, hipStream_t s) {
    return by_tables(spans, n, unit, false, [&](const Table& t, int64_t at) {
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
    return by_tables(spans, n, unit, true, [&](const Table& t, int64_t) {
        clip_kernel<<<t.units, kThreads, 0, s>>>(t, sums, units, joined, scale, max_norm, first ? norm : nullptr);
        DCIH_HIP(hipGetLastError());
        first = false;
        return 0;
    });
}

}  // namespace dcih
