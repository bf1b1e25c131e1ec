// A gated linear recurrence over the tokens of sequences, each channel by itself, and its gradient:
//
//   a_t = 1 / (1 + e^-g_t),  h_t = a_t h_(t-1) + (1 - a_t) x_t        (gates)
//   a_t = g_t,               h_t = a_t h_(t-1) + x_t                  (decays)
//
//   l_t = dh_t + a_(t+1) l_(t+1)        the gradient that reaches h_t
//   gates:  dx_t = (1 - a_t) l_t,  dg_t = a_t (1 - a_t) l_t (h_(t-1) - x_t)
//   decays: dx_t = l_t,            dg_t = l_t h_(t-1);        both: by the first state a_1 l_1
//
// Both directions are compositions of maps s -> A s + B, which are associative: a tile of 128 or 256 tokens by kLanes pieces
// of 16 bytes is one workgroup's, in registers; each group of lanes composes its few tokens, the groups are joined in
// shared memory, and a tile's map is joined to that of the tiles before it while these still run (see carry_of; a scan in a single pass, with a
// look back).  So every element is read and written once, but for few long chains, whose tokens are read a second time when their maps are joined
// (see link_kernel; in the gradient dh and the gates).  The gradient forms h_(t-1) again, from x, g and the state before each tile, which
// the forward call keeps in 32 bits: less to read than h itself, and not rounded.
#include "../../include/dci_hip.h"
#include "scan.h"

#include <algorithm>
#include <type_traits>

namespace dcih {
namespace {

constexpr int kThreads = 256;
constexpr int kLanes = 8;                          // pieces of 16 bytes that a tile is wide: a line (two: 65536 x 4096 bf16 374 us, 351 so)
// Tokens of a tile, with pieces of `len` elements: as many as the gradient's registers hold.  (8 x 4096 x 1024 f32 with gradients 230 us, with 256
// tokens 241 to 253; with shared gates 139 either way, and a chain of 20000 tokens by 64 has half the tiles: 18 and 21 us instead of 26 and 27.)
constexpr int tile_of(int len, bool shared) { return len == 8 || (len == 4 && !shared) ? 128 : 256; }
// Wavefronts of a SIMD: registers enough for a tile, tiles enough to hide one another's waits (one more each way spills: 8 x 4096 x 2048
// with gradients 262 us instead of 238; one less is as fast).
constexpr int kWaves = 4, kBackWaves = 3;
// Tokens that one thread takes in any case.  Of longer rows it takes all where pieces are many, kManyPieces for each token up to kEnoughPieces: 512 x 40 x
// 2048 bf16 42 us, 53 by tiles; 512 x 48 x 1024 29 and 40, 128 x 48 x 1024 24 and 12; 256 x 130 x 2048 85 and 154, 256 x 300 x 2048 206 and 241, 64 x 300 x
// 2048 132 and 58.  But not where a tile is full to 7/8 or more and has no other to wait for: there either is within a tenth of the other (bf16 512 x 128 x
// 1024 80 and 72, 512 x 128 x 2048 159 and 167, f32 256 x 116 x 1024 59 and 58).
constexpr int kShort = 32;
constexpr int64_t kManyPieces = 1280, kEnoughPieces = 1 << 16;
// Up to so many channels each has a thread, not a piece of them: a wavefront's arithmetic for 8 channels takes 0.4 us a token (32 x 16 x 1024 bf16 4.7 us,
// 9.2 by pieces; 32 x 32 x 1024 7.4 and 16.3; but 512 x 8 x 1024 8.7 and 6.5).  Twice as many where sequences are longer than kSteps.
constexpr int64_t kSingles = 1 << 17;
constexpr int kSteps = 16;
// Up to so many chains of so many tiles or more each are joined by a launch of their own (see link_kernel): 1 x 262144 x 64 bf16 81 us, with gradients 178,
// chained 200 and 398; x 256 171 and 427, 221 and 453; x 384 237 and 582, 245 and 525; 1 x 16384 x 64 19 and 21, with gradients 69 and 63, the host's two
// launches more.
constexpr int kFewChains = 4, kManyTiles = 192;
constexpr int kApart = 32;                         // words from one chain's counter to the next: a line takes an atomic operation in 11 ns
constexpr int64_t kMaxGrid = 1 << 23;
constexpr uint32_t kUnset = 0xffffffffu;           // what the workspace is filled with; no value that is published has these bits
constexpr uint32_t kMapSet = 1, kStateSet = 2;
// Decays beyond 1: where those of a tile could make something 2^100 times as large the product of all of them says too little in 32 bits (it may overflow
// in front of a state of 0, which stays 0), and the tile's tokens are gone through one after the other by a thread a channel, 24 us a tile of a chain
// (20000 x 64 f32 of nothing but such 3.8 ms, else 26 us; in a chain that is joined at once 55).  Below that a product may lose 2^-149 of
// what the state was, 2^-49 where that grows as much again.  In units of 2^(1 / kFine).
constexpr int kFine = 256, kSteep = 100 * kFine;
constexpr uint32_t kSteepMap = 0xfffffffeu;        // (in a map's A) no map: the tile's tokens say what is behind it

typedef uint32_t u32x4_float __attribute__((ext_vector_type(4), aligned(4)));

// Makes the compiler take a register's contents for others: what was computed from it before is computed again, not kept in more
// registers from one loop over a group's tokens to the next.
template <class V> __device__ __forceinline__ void renew(V& v) { asm volatile("" : "+v"(v)); }

// L elements of a row: a 16-byte piece, or (L = 1, rows shorter than that) one.
template <class T, int L> struct Span {
    using raw_t = typename T::raw;
    using P = Piece<T>;
    u32x4 bits;
    static_assert(L == P::kLen, "a piece");
    __device__ void load(const raw_t* p) { bits = P::load(p); }
    __device__ void load_once(const raw_t* p) { bits = P::load_once(p); }
    __device__ void get(float (&z)[L]) const { P::unpack(bits, z); }
    __device__ void clear() { bits = u32x4{0, 0, 0, 0}; }
    __device__ void renew() { dcih::renew(bits); }
    __device__ static void store(raw_t* p, const float (&z)[L]) { P::store_once(p, P::pack(z)); }
};
template <class T> struct Span<T, 1> {
    using raw_t = typename T::raw;
    raw_t bits;
    __device__ void load(const raw_t* p) { bits = *p; }
    __device__ void load_once(const raw_t* p) { bits = *p; }
    __device__ void get(float (&z)[1]) const { z[0] = (float)bits; }
    __device__ void clear() { bits = (raw_t)0.f; }
    __device__ void renew() {}
    __device__ static void store(raw_t* p, const float (&z)[1]) { *p = (raw_t)z[0]; }
};

template <int L> __device__ inline void load_floats(const float* p, float (&z)[L]) {
    if constexpr (L % 4 == 0) {
#pragma unroll
        for (int k = 0; k < L; k += 4) {
            const u32x4 v = *reinterpret_cast<const u32x4_float*>(p + k);
#pragma unroll
            for (int i = 0; i < 4; i++) z[k + i] = __builtin_bit_cast(float, (uint32_t)v[i]);
        }
    } else {
#pragma unroll
        for (int k = 0; k < L; k++) z[k] = p[k];
    }
}
template <int L> __device__ inline void store_floats(float* p, const float (&z)[L]) {
    if constexpr (L % 4 == 0) {
#pragma unroll
        for (int k = 0; k < L; k += 4) {
            u32x4 v;
#pragma unroll
            for (int i = 0; i < 4; i++) v[i] = __builtin_bit_cast(uint32_t, z[k + i]);
            *reinterpret_cast<u32x4_float*>(p + k) = v;
        }
    } else {
#pragma unroll
        for (int k = 0; k < L; k++) p[k] = z[k];
    }
}

// e^-|g|.  log2(e) in two parts, the first of so few bits that its product with 16-bit types is exact.
template <class T> __device__ inline float exp_below(float g) {
    const float y = -__builtin_fabsf(g);
    if constexpr (sizeof(typename T::raw) == 2) {
        constexpr float kHigh = std::is_same<T, BF16>::value ? 47274.f / 32768.f : 5909.f / 4096.f;
        constexpr float kRest = (float)((1.44269504088896340736 - kHigh) * 0.693147180559945309417);
        const float e = exp2_fast(y * kHigh);
        return __builtin_fmaf(e, fmaxf(y * kRest, -1.f), e);        // (0 for y = -inf, NaN for NaN)
    } else {
        const float z = y < -150.f ? -150.f : y;                    // (nothing is left there; NaN stays)
        const float t = z * kLog2e, rest = __builtin_fmaf(z, 1.92596299e-8f, __builtin_fmaf(z, kLog2e, -t));
        const float e = exp2_fast(t);
        return __builtin_fmaf(e * kLn2, rest, e);
    }
}

// a and 1 - a of a gate.  The smaller of the two is computed, the other is what is missing to 1: a channel that forgets over
// thousands of tokens keeps the digits of 1 - a.
struct Gate { float a, keep; };
template <class T> __device__ inline float lesser_of(float g) {
    const float e = exp_below<T>(g);
    return e * __builtin_amdgcn_rcpf(1.f + e);
}
__device__ inline Gate gate_by(float small, float sign) {
    const float big = 1.f - small;
    const bool holds = __builtin_bit_cast(int, sign) >= 0;
    return Gate{holds ? big : small, holds ? small : big};
}
// A token's factor of the state and what is added to it, of a gate and an input.
template <class T, bool kDecay> __device__ inline Gate coefs_of(float g) {
    if (kDecay) return Gate{g, 1.f};
    return gate_by(lesser_of<T>(g), g);
}
// Where one register has to do: the smaller one with the gate's sign (decays as they are).
template <class T, bool kDecay> __device__ inline float packed_of(float g) { return kDecay ? g : __builtin_copysignf(lesser_of<T>(g), g); }
template <bool kDecay> __device__ inline Gate coefs_of(float packed) {
    if (kDecay) return Gate{packed, 1.f};
    return gate_by(__builtin_fabsf(packed), packed);
}
template <bool kDecay> __device__ inline float step(float h, float x, Gate c) { return __builtin_fmaf(c.a, h, kDecay ? x : c.keep * x); }

// ---- one thread a channel ----------------------------------------------------------------
// A server's step, or its drafts, few tokens of many sequences; rows of any length where they are many.  The state may be written where it is read.  Bound by the launch (32 x 1 x 4096 bf16
// 2.7 us replayed), then by the chain of a wavefront's tokens (8: 4.0), then memory (1024 x 8 x 4096 39 us, 6 TB/s).
template <class T, int L, bool kDecay, int U, int kTile>
__global__ __launch_bounds__(kThreads) void short_kernel(ScanArgs a, int pieces, int64_t first) {
    constexpr bool kStates = kTile > 0;
    const int64_t strips = (pieces + kLanes - 1) / kLanes, tiles = kStates ? (a.length + kTile - 1) / max(kTile, 1) : 0;
    using raw_t = typename T::raw;
    const int64_t i = first + (int64_t)blockIdx.x * kThreads + threadIdx.x;
    const int64_t b = i / pieces;
    if (b >= a.rows) return;
    const int piece = (int)(i - b * pieces), own = piece * L, c0 = min(own, a.dim - L), length = (int)a.length;
    int64_t len = length;
    if (a.bounds) len = min(max(id_at(a.bounds, a.wide_bounds, b), (int64_t)0), len);
    const raw_t *x = (const raw_t*)a.x + b * a.x_row + c0, *g = (const raw_t*)a.gates + (a.shared ? 0 : b * a.g_row) + c0;
    raw_t* out = (raw_t*)a.h + b * length * a.dim + c0;
    float h[L];
#pragma unroll
    for (int k = 0; k < L; k++) h[k] = 0.f;
    if (a.state) load_floats<L>(a.state + b * a.dim + c0, h);
    int64_t t0 = 0;
    for (; t0 < len; t0 += U) {
        // what the gradient takes for the state before a tile
        if (kStates && t0 % kTile == 0) store_floats<L>(a.states + ((b * strips + piece / kLanes) * tiles + t0 / kTile) * (kLanes * L) + piece % kLanes * L, h);
        Span<T, L> xs[U], gs[U];
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int64_t t = min(t0 + u, len - 1);
            xs[u].load(x + t * a.x_step);
            gs[u].load(g + t * a.g_step);
        }
#pragma unroll
        for (int u = 0; u < U; u++) {
            if (t0 + u >= length) break;
            const bool in = t0 + u < len;
            float xv[L], c[L], y[L];
            xs[u].get(xv);
            gs[u].get(c);
#pragma unroll
            for (int k = 0; k < L; k++) {
                const float next = step<kDecay>(h[k], xv[k], coefs_of<T, kDecay>(c[k]));
                h[k] = in ? next : h[k];
                y[k] = in ? next : 0.f;
            }
            raw_t* to = out + (t0 + u) * a.dim;
            if (c0 == own) {
                Span<T, L>::store(to, y);
            } else {           // the row's last piece: what it shares with the one before is that one's, whose state may be written already
#pragma unroll
                for (int k = 0; k < L; k++)
                    if (c0 + k >= own) to[k] = (raw_t)y[k];
            }
        }
    }
    float none[L];
#pragma unroll
    for (int k = 0; k < L; k++) none[k] = 0.f;
    for (; t0 < length; t0++) Span<T, L>::store(out + t0 * a.dim, none);
    if (!a.last) return;
    float* last = a.last + b * a.dim + c0;
    if (c0 == own) {
        store_floats<L>(last, h);
    } else {
#pragma unroll
        for (int k = 0; k < L; k++)
            if (c0 + k >= own) last[k] = h[k];
    }
}

// ---- tiles -------------------------------------------------------------------------------
// A chain is a strip of kLanes pieces of one row of tokens; its tiles follow one another.  Workgroups take tiles by counters, those of a
// chain in order: what a tile waits for was taken before it, by a workgroup that waits for nothing taken later.
enum Phase { kChained, kMaps, kApply };              // all at once; or maps alone, then (behind link_kernel) what they lead to
struct Chains {
    int pieces, strips, slots;         // pieces of a row; strips of them; channels of a strip, those beyond the row included
    int64_t tiles, count;              // tiles of a chain, chains
    bool once;                         // tokens are read past the caches
    bool apart;                        // rows are whole lines: strips share none
    uint32_t *tickets, *flags;         // what was taken; [count][tiles] what is set: a hint of what to wait for
    uint64_t* maps;                    // [count][tiles][slots] (A, B)
    uint32_t* states;                  // [count][tiles][slots] the state behind a tile
    int32_t* from;                     // (kPacked) [tiles] the last sequence that begins before a tile
    float* sums;                       // [count][tiles][slots] (gradient of shared gates)
    Phase phase;
};

int span_len(int dim, int dtype) {
    const int len = dtype == DCIH_F32 ? 4 : 8;
    return dim >= len ? len : 1;
}

__host__ inline int64_t lay_out(Chains& c, void* mem, int64_t rows, int64_t length, int dim, int dtype, bool gradient, bool shared) {
    const int len = span_len(dim, dtype);
    c.pieces = (dim + len - 1) / len;
    c.strips = (c.pieces + kLanes - 1) / kLanes;
    c.slots = kLanes * len;
    const int tile = tile_of(len, shared);
    c.tiles = (length + tile - 1) / tile;
    c.count = rows * c.strips;
    int64_t at = 0;
    auto take = [&](int64_t bytes) {
        char* p = (char*)mem + at;
        at += (bytes + 255) / 256 * 256;
        return p;
    };
    const int64_t cells = c.count * c.tiles * c.slots, chained = c.tiles > 1 ? 1 : 0;
    c.tickets = (uint32_t*)take(chained * c.count * kApart * 4);
    c.flags = (uint32_t*)take(chained * c.count * c.tiles * 4);
    c.maps = (uint64_t*)take(chained * cells * 8);
    c.states = (uint32_t*)take(chained * cells * 4);
    c.from = (int32_t*)take(chained * c.tiles * 4);
    c.sums = (float*)take(gradient && shared ? cells * 4 : 0);
    return at;
}

// The last sequence that begins before a token, by `bound`, which cuts offsets to [0, length].
template <class Bound> __device__ inline int64_t last_before(int64_t sequences, int64_t token, Bound bound) {
    int64_t from = 0, to = sequences;
    while (to - from > 1) {
        const int64_t mid = from + (to - from) / 2;
        if (bound(mid) < token) from = mid;
        else to = mid;
    }
    return from;
}
__device__ inline int64_t cut(const ScanArgs& a, int64_t o) { return min(max(o, (int64_t)0), a.length); }

// The mark of what is not posted yet, and by the workgroups behind the first `blocks` where each tile looks for its sequences: there
// every workgroup would look for itself, ten steps that wait for one another.
__global__ __launch_bounds__(kThreads) void fill_kernel(u32x4* p, int64_t n, int64_t blocks, ScanArgs a, int32_t* from, int64_t tiles, int tokens) {
    if (blockIdx.x < blocks) {
        const int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x;
        if (i < n) p[i] = u32x4{kUnset, kUnset, kUnset, kUnset};
        return;
    }
    const int64_t i = ((int64_t)blockIdx.x - blocks) * kThreads + threadIdx.x;
    if (i < tiles) from[i] = (int32_t)last_before(a.sequences, i * tokens, [&](int64_t s) { return cut(a, id_at(a.bounds, a.wide_bounds, s)); });
}
__global__ __launch_bounds__(kThreads) void copy_kernel(const float* from, float* to, int64_t n) {
    const int64_t step = (int64_t)gridDim.x * kThreads;
    for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < n; i += step) to[i] = from ? from[i] : 0.f;
}

// Sequences without tokens: what reaches their end is what they began with.  By workgroups of their own behind those of the tiles.
constexpr int kEmpty = 16;                          // sequences of a workgroup, up to kEmptyGrid workgroups
constexpr int64_t kEmptyGrid = 4096;
__device__ inline void pass_empty(const ScanArgs& a, int64_t block, int64_t blocks, const float* from, float* to) {
    const int waves = kThreads / kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    for (int64_t s = block * waves + wave; s < a.sequences; s += blocks * waves) {
        int64_t lo = 0, hi = id_of_all(a.bounds, a.wide_bounds, a.form == kPacked ? s + 1 : s);
        if (a.form == kPacked) lo = max(id_of_all(a.bounds, a.wide_bounds, s), (int64_t)0);
        if (a.form == kPacked) hi = min(hi, a.length);
        if (hi > lo) continue;
        for (int c = lane_id(); c < a.dim; c += kWave) to[s * a.dim + c] = from ? from[s * a.dim + c] : 0.f;
    }
}

__device__ inline uint32_t peek(const uint32_t* p) { return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
__device__ inline uint64_t peek(const uint64_t* p) { return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
template <class V> __device__ inline void post(V* p, V v) { __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
__device__ inline int64_t uniform(int64_t v) {
    return (int64_t)((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(v >> 32)) << 32 | (uint32_t)__builtin_amdgcn_readfirstlane((int)v));
}
__device__ inline uint32_t word_of(float v) {
    const uint32_t w = __builtin_bit_cast(uint32_t, v);
    return w >= kSteepMap ? 0x7fc00000u : w;           // (NaN for NaN)
}

// Item i of all is the next tile of a chain, in the direction of the scan, and each chain has as many items as tiles.  Neighbouring
// items run on different XCDs.  From one round to the next the strips go on by one: an XCD that always had the same ones would use a
// few of its cache's channels only (65536 x 4096 bf16 packed 351 us, 403 so).  Strips that share lines with their neighbours stand 8
// items from them, so that most of them are on one XCD and close in time (30011 x 1023 f16 with gradients 202 us, 239 apart; with
// rows of whole lines 375 and 351 of the first case).  By one thread; returns chain * tiles + place.
__device__ inline int64_t take_tile(const Chains& c, Phase phase, int64_t i) {
    if (c.tiles == 1) return i;
    const int64_t round = i / c.count, at = i - round * c.count, row = at / c.strips;
    int strip = (int)(at - row * c.strips);
    if (!c.apart) {
        const int xcd = strip % 8, rest = c.strips % 8;
        strip = xcd * (c.strips / 8) + min(xcd, rest) + strip / 8;
    }
    const int64_t chain = row * c.strips + (strip + round) % c.strips;
    if (phase != kChained) return chain * c.tiles + round;
    return chain * c.tiles + (atomicAdd(&c.tickets[chain * kApart], 1u) - kUnset);        // the counter begins at kUnset
}

// The state that enters tile `at` of a chain in channel `slot`.  A tile posts its map as soon as it has it, and the state
// behind it when it knows the one before; a wavefront looks for the nearest tile before its own whose state is there and goes on from it by the
// maps in between, in their order: that is what those tiles do themselves, so the bits do not depend on who was how far.
// Words are waited for themselves; the flags only say which are worth a look.
__device__ float carry_of(const Chains& c, int64_t chain, int64_t at, int slot) {
    const uint32_t* flags = c.flags + chain * c.tiles;
    const int64_t last = (chain * c.tiles + at - 1) * c.slots + slot;
    const int lane = lane_id();
    const int64_t tile = at - 1 - lane;
    int behind;                                     // tiles between the one whose state is there and this one
    uint32_t w;
    for (;;) {
        w = peek(c.states + last);
        const uint32_t f = tile >= 0 ? peek(flags + tile) : kUnset;
        if (__all(w != kUnset)) return __builtin_bit_cast(float, w);
        const unsigned long long full = __ballot(f == kStateSet), some = __ballot(f != kUnset);
        behind = full ? __builtin_ctzll(full) : -1;
        if (full && (~some & ((1ull << behind) - 1)) == 0) break;
        __builtin_amdgcn_s_sleep(1);
    }
    const int64_t base = last - (int64_t)behind * c.slots;
    const uint64_t* maps = c.maps + base + c.slots;
    constexpr int U = 16;
    uint64_t m[U];
    auto load_maps = [&](int i) {
#pragma unroll
        for (int u = 0; u < U; u++) m[u] = i + u < behind ? peek(maps + (int64_t)(i + u) * c.slots) : 0;
    };
    load_maps(0);
    while ((w = peek(c.states + base)) == kUnset) {}
    float h = __builtin_bit_cast(float, w);
    for (int i = 0; i < behind; i += U) {
        if (i) load_maps(i);
#pragma unroll
        for (int u = 0; u < U; u++) {
            if (i + u < behind) {
                while ((uint32_t)m[u] == kUnset || (uint32_t)(m[u] >> 32) == kUnset) m[u] = peek(maps + (int64_t)(i + u) * c.slots);
                h = __builtin_fmaf(__builtin_bit_cast(float, (uint32_t)m[u]), h, __builtin_bit_cast(float, (uint32_t)(m[u] >> 32)));
            }
        }
    }
    return h;
}

// How much a thread's decays may make of something, at most in any of its channels, is counted.  Whole numbers: the order does not matter.
template <int R, int L> __device__ __forceinline__ void count_growth(const float (&as)[R][L], int times, int& s_growth, uint32_t& s_steep) {
    float most = 0.f;
#pragma unroll
    for (int u = 0; u < R; u++)
#pragma unroll
        for (int k = 0; k < L; k++) most = fmaxf(most, __builtin_fabsf(as[u][k]));
    if (!(most > 1.f)) return;
    most = 1.f;
#pragma unroll
    for (int k = 0; k < L; k++) {
        float grows = 1.f;
#pragma unroll
        for (int u = 0; u < R; u++) grows *= fmaxf(__builtin_fabsf(as[u][k]), 1.f);
        most = fmaxf(most, grows);
    }
    const int by = (int)fminf(log2_fast(most) * kFine + 1.f, 1e6f) * times;
    if (atomicAdd(&s_growth, by) + by > kSteep) s_steep = 1;
}

// A channel's groups joined, by one thread: map (A, B) of each in the direction of the scan, `resets` those whose result does not
// depend on what enters.  Leaves in B what enters each group.  Where a tile is steep, `go` goes through the tokens of a group without such.
template <int kGroups, bool kBack, class Go>
__device__ void join_groups(const Chains& c, Phase phase, int64_t chain, int64_t at, int slot, uint32_t resets, const float* s_a, float* s_b, bool steep, Go go) {
    auto place = [&](int g) { return (kBack ? kGroups - 1 - g : g) * c.slots + slot; };
    float in = 0.f;
    if (steep) {
        const int64_t cell = chain * c.tiles + at, word = cell * c.slots + slot;
        const bool follows = at + 1 < c.tiles && phase == kChained;
        if (at && phase != kMaps) in = phase == kApply ? __builtin_bit_cast(float, c.states[word - c.slots]) : carry_of(c, chain, at, slot);
        for (int i = 0; i < kGroups; i++) {
            const int g = kBack ? kGroups - 1 - i : i;
            const float gb = s_b[place(i)];
            s_b[place(i)] = in;
            in = resets >> g & 1 ? gb : go(g, slot, in);
        }
        if (phase == kMaps) c.maps[word] = (uint64_t)word_of(in) << 32 | (resets ? kUnset : kSteepMap);
        if (follows) post(c.states + word, word_of(in));
        if (follows && slot == 0) post(c.flags + cell, kStateSet);
        return;
    }
    if (c.tiles > 1) {
        float A = 1.f, B = 0.f;
#pragma unroll 8
        for (int g = 0; g < kGroups; g++) {
            const float ga = s_a[place(g)], gb = s_b[place(g)];
            const bool reset = resets >> (kBack ? kGroups - 1 - g : g) & 1;
            B = reset ? gb : __builtin_fmaf(ga, B, gb);
            A *= ga;
        }
        const int64_t cell = chain * c.tiles + at, word = cell * c.slots + slot;
        const bool follows = at + 1 < c.tiles && phase == kChained;
        if (phase == kMaps) {
            c.maps[word] = (uint64_t)word_of(B) << 32 | (resets ? kUnset : word_of(A));
            return;
        }
        if (resets) {
            if (follows) post(c.states + word, word_of(B));
            if (follows && slot == 0) post(c.flags + cell, kStateSet);
        } else if (follows) {
            post(c.maps + word, (uint64_t)word_of(B) << 32 | word_of(A));
            if (slot == 0) post(c.flags + cell, kMapSet);
        }
        if (at) in = phase == kApply ? __builtin_bit_cast(float, c.states[word - c.slots]) : carry_of(c, chain, at, slot);
        if (!resets && follows) {
            post(c.states + word, word_of(__builtin_fmaf(A, in, B)));
            if (slot == 0) post(c.flags + cell, kStateSet);
        }
    }
    float h = in;
#pragma unroll 8
    for (int g = 0; g < kGroups; g++) {
        const float ga = s_a[place(g)], gb = s_b[place(g)];
        const bool reset = resets >> (kBack ? kGroups - 1 - g : g) & 1;
        s_b[place(g)] = h;
        h = reset ? gb : __builtin_fmaf(ga, h, gb);
    }
}

// Where sequences begin and end among the tokens of a tile.  In groups of tokens without either, and with all of them
// in one sequence, nobody asks.
struct Marks {
    int64_t row, length;              // a row of tokens, and how many it has
    int64_t t0;                       // the tile's first token
    int64_t lo, hi;                   // tokens [lo, hi) of the row are of sequences
    const int *first, *end;           // (kPacked) for each token of the tile the sequence that begins or ends there, -1: none

    __device__ Marks(const ScanArgs& a, int64_t row_, int64_t t0_) : row(row_), length(a.length), t0(t0_) {
        if (a.form == kFlat) length = min(length, a.total - row * a.length);
    }
    __device__ static int64_t length_of(const ScanArgs& a, int64_t s, int64_t most) {
        return a.bounds ? min(max(id_at(a.bounds, a.wide_bounds, s), (int64_t)0), most) : most;
    }
    // (kFlat) the sequence of a token, and its place there
    __device__ int64_t of(const ScanArgs& a, int64_t t, int& place) const {
        const uint32_t each = (uint32_t)a.each, s = (uint32_t)t / each;
        place = (int)((uint32_t)t - s * each);
        return row * ((uint32_t)a.length / each) + s;
    }
    __device__ bool in(const ScanArgs& a, int64_t t) const {
        if (t < lo || t >= hi) return false;
        if (a.form != kFlat || !a.bounds) return true;
        int place;
        const int64_t s = of(a, t, place);
        return place < length_of(a, s, a.each);
    }
    __device__ int64_t begins(const ScanArgs& a, int64_t t) const {
        if (a.form == kPacked) return first[t - t0];
        if (a.form == kRows) return t ? -1 : row;
        int place;
        const int64_t s = of(a, t, place);
        return place ? -1 : s;
    }
    __device__ int64_t ends(const ScanArgs& a, int64_t t) const {
        if (a.form == kPacked) return end[t - t0];
        if (a.form == kRows) return t == hi - 1 ? row : -1;
        int place;
        const int64_t s = of(a, t, place);
        return place == length_of(a, s, a.each) - 1 ? s : -1;
    }
};

// (kRows) How many tokens of a row are its sequence's.
__device__ inline int64_t row_end(const ScanArgs& a, int64_t row) {
    return a.bounds ? min(max(id_of_all(a.bounds, a.wide_bounds, row), (int64_t)0), a.length) : a.length;
}

// A tile behind the end of a row's sequence: zeros, without a look at the tokens.  What enters the next tile is zero too.
template <class T, int L>
__device__ inline void write_zeros(const Chains& c, Phase phase, int64_t item, int64_t at, typename T::raw* out, int64_t step, int64_t tokens, bool live) {
    float zeros[L];
#pragma unroll
    for (int k = 0; k < L; k++) zeros[k] = 0.f;
    if (out && live)
        for (int64_t u = 0; u < tokens; u++) Span<T, L>::store(out + u * step, zeros);
    if (at >= c.tiles || threadIdx.x >= c.slots) return;
    const int64_t cell = item - item % c.tiles + at, word = cell * c.slots + threadIdx.x;
    if (phase == kMaps) c.maps[word] = kUnset;
    if (phase == kChained && at + 1 < c.tiles) {
        post(c.states + word, 0u);
        if (threadIdx.x == 0) post(c.flags + cell, kStateSet);
    }
}

// What finds the sequences of a tile (kPacked): the first of them that may begin or end there, and each thread's bounds, asked for ahead
// of the tokens (what the vector memory answers comes in order).
struct Found {
    int64_t from = 0, lo = 0, hi = 0;
    __device__ Found(const ScanArgs& a, const Chains& c, int64_t tile, int64_t t0) {
        if (a.form != kPacked) return;
        if (c.tiles > 1) from = ((const __attribute__((address_space(4))) int32_t*)c.from)[tile];
        else from = last_before(a.sequences, t0, [&](int64_t s) { return cut(a, id_of_all(a.bounds, a.wide_bounds, s)); });
        ask(a, from);
    }
    __device__ void ask(const ScanArgs& a, int64_t s) {
        const int64_t mine = s + threadIdx.x;
        lo = hi = 0;
        if (mine >= a.sequences) return;
        lo = cut(a, id_at(a.bounds, a.wide_bounds, mine));
        hi = cut(a, id_at(a.bounds, a.wide_bounds, mine + 1));
    }
};
// By all threads; `s_first`, `s_end` and `s_marked` (a bit for each `per` tokens) are ready behind the next barrier.
template <int kTokens>
__device__ inline void find_marks(const ScanArgs& a, Found f, Marks& m, int per, int (&s_first)[kTokens], int (&s_end)[kTokens], uint32_t& s_marked) {
    m.lo = 0;
    m.hi = m.length;
    if (a.form == kRows) m.hi = row_end(a, m.row);
    if (a.form != kPacked) return;
    auto bound_of_all = [&](int64_t i) { return cut(a, id_of_all(a.bounds, a.wide_bounds, i)); };
    m.lo = bound_of_all(0);
    m.hi = bound_of_all(a.sequences);
    m.first = s_first;
    m.end = s_end;
    for (int i = threadIdx.x; i < kTokens; i += blockDim.x) s_first[i] = s_end[i] = -1;
    if (threadIdx.x == 0) s_marked = 0;
    __syncthreads();
    for (int64_t s = f.from;;) {
        const int mine = (int)(s + threadIdx.x);
        if (f.hi > f.lo) {
            if (f.lo >= m.t0 && f.lo < m.t0 + kTokens) {
                s_first[f.lo - m.t0] = mine;
                atomicOr(&s_marked, 1u << ((int)(f.lo - m.t0) / per));
            }
            if (f.hi - 1 >= m.t0 && f.hi - 1 < m.t0 + kTokens) {
                s_end[f.hi - 1 - m.t0] = mine;
                atomicOr(&s_marked, 1u << ((int)(f.hi - 1 - m.t0) / per));
            }
        }
        s += blockDim.x;
        if (s >= a.sequences || bound_of_all(s) >= m.t0 + kTokens) break;
        f.ask(a, s);
    }
}

// What a group of `per` tokens from `t` on has to know of them, a bit for each: which are of a sequence, its first, its last.  Tokens
// of no sequence are zeros that begin and end at zero.  (No lane leaves the loops over the tokens early: hipcc 7.2 lost a
// factor of A there.)
struct Bits {
    uint32_t in, first, end;
    bool any;                         // some group of the wavefront has other tokens than those in the middle of a sequence

    __device__ Bits(const ScanArgs& a, const Marks& m, int64_t t, int per, int group, uint32_t s_marked) : in(~0u), first(0), end(0) {
        bool marked = a.form == kFlat || t < m.lo || t + per > m.hi;
        if (a.form == kRows) marked |= t == 0 || t + per == m.hi;
        if (a.form == kPacked) marked |= s_marked >> group & 1;
        any = __any(marked);
        if (!any) return;
        in = 0;
        for (int u = 0; u < per; u++) {
            const bool inside = m.in(a, t + u);
            in |= (uint32_t)inside << u;
            first |= (uint32_t)(inside && m.begins(a, t + u) >= 0) << u;
            end |= (uint32_t)(inside && m.ends(a, t + u) >= 0) << u;
        }
    }
    __device__ bool is_in(int u) const { return in >> u & 1; }
    __device__ bool is_end(int u) const { return end >> u & 1; }
    __device__ bool is_first(int u) const { return first >> u & 1; }
    __device__ bool starts(int u) const { return (first | ~in) >> u & 1; }      // what comes from the token before does not enter
    __device__ bool stops(int u) const { return (end | ~in) >> u & 1; }         // nor what comes back from the one behind
    __device__ bool starts_any(int per) const { return (first | ~in) & ((1u << per) - 1); }
    __device__ bool stops_any(int per) const { return (end | ~in) & ((1u << per) - 1); }
};

// A kernel's first argument, read again for what is hardly ever done: kept for that, its fields would take the scalar registers that the tiles need
// (by which the gradient had 31 of them in vector registers).
__device__ inline const ScanArgs& args_again() {
    const ScanArgs* a = (const ScanArgs*)__builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(a));
    return *a;
}
// The channel of a slot of a strip.
template <int L> __device__ inline int channel_of(const ScanArgs& a, int strip, int slot) {
    return min(min(strip * kLanes + slot / L, (a.dim - 1) / L) * L, a.dim - L) + slot % L;
}
// Tokens [t, t + n) of a row's channel one after the other, all of them in the middle of a sequence, by decays; or back through them.
template <class T, int kUnroll> __device__ inline float go_forward(const ScanArgs& a, int64_t row, int channel, int64_t t, int n, float h) {
    using raw_t = typename T::raw;
    const raw_t *x = (const raw_t*)a.x + row * a.x_row + channel, *g = (const raw_t*)a.gates + (a.shared ? 0 : row * a.g_row) + channel;
#pragma unroll kUnroll
    for (int64_t i = t; i < t + n; i++) h = __builtin_fmaf((float)g[a.shared ? 0 : i * a.g_step], h, (float)x[i * a.x_step]);
    return h;
}
template <class T, int kUnroll> __device__ inline float go_back(const ScanArgs& a, int64_t row, int channel, int64_t t, int n, float l) {
    using raw_t = typename T::raw;
    const raw_t *dh = (const raw_t*)a.dh + row * a.length * a.dim + channel, *g = (const raw_t*)a.gates + (a.shared ? 0 : row * a.g_row) + channel;
#pragma unroll kUnroll
    for (int64_t i = t + n - 1; i >= t; i--) l = (float)g[a.shared ? 0 : i * a.g_step] * ((a.dh ? (float)dh[i * a.dim] : 0.f) + l);
    return l;
}

// Runs `body` as the wavefront has marks or not: without them there is no branch about a token.
template <class Body> __device__ __forceinline__ void by_marks(bool any, Body body) {
    if (any) body(std::true_type{});
    else body(std::false_type{});
}

// A tile, read and written once (twice read in the chains of link_kernel): bound by memory (65536 x 4096 bf16 355 us, 1.61 GB at 4.5 TB/s; 8 x 4096 x 2048 88 us) where chains are many or long,
// by the wait for the tile before where one short row is all there is (20000 x 64 f32, 79 tiles: 18 us).  Without that wait the
// second took 92 us of 113 at the time, without the gates' arithmetic 106.
template <class T, int L, bool kDecay, bool kShared, bool kPhased>
__global__ __launch_bounds__(kThreads, kWaves) void scan_kernel(ScanArgs a, Chains c, int64_t first, int64_t empty) {
    constexpr int kTile = tile_of(L, kShared), kGroups = kThreads / kLanes, U = kTile / kGroups, kSlots = kLanes * L;
    static_assert(kGroups <= 32, "a bit for each group");
    using raw_t = typename T::raw;
    const Phase phase = kPhased ? c.phase : kChained;
    __shared__ float s_a[kGroups * kSlots], s_b[kGroups * kSlots];
    __shared__ int s_first[kTile], s_end[kTile];
    __shared__ uint32_t s_marked, s_resets, s_steep;
    __shared__ int s_growth[kLanes];
    __shared__ int64_t s_item;
    if (first + blockIdx.x >= c.count * c.tiles) return pass_empty(a, first + blockIdx.x - c.count * c.tiles, empty, a.state, a.last);
    const int lane = threadIdx.x % kLanes, group = threadIdx.x / kLanes;
    if (kDecay && threadIdx.x < kLanes) s_growth[threadIdx.x] = 0;
    if (threadIdx.x == 0) {
        s_resets = s_steep = 0;
        s_item = take_tile(c, phase, first + blockIdx.x);
    }
    __syncthreads();
    const int64_t item = uniform(s_item), chain = item / c.tiles, at = item - chain * c.tiles, row = chain / c.strips;
    const int64_t t0 = at * kTile, t = t0 + group * U;
    Marks m(a, row, t0);
    const int piece = (int)(chain - row * c.strips) * kLanes + lane, c0 = min(min(piece, c.pieces - 1) * L, a.dim - L);
    const bool live = piece < c.pieces;
    if (a.form == kRows && a.bounds && t0 >= row_end(a, row))
        return write_zeros<T, L>(c, phase, item, at, phase == kMaps ? nullptr : (raw_t*)a.h + (row * a.length + t) * a.dim + c0, a.dim, min((int64_t)U, m.length - t), live);
    const raw_t* x = (const raw_t*)a.x + row * a.x_row + c0;
    const raw_t* g = (const raw_t*)a.gates + (kShared ? 0 : row * a.g_row) + c0;
    const Found found(a, c, at, t0);
    Span<T, L> xs[U], gs[kShared ? 1 : U];
    if (kShared) gs[0].load(g);
    if (c.once) {
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int64_t from = min(t + u, m.length - 1);
            xs[u].load_once(x + from * a.x_step);
            if (!kShared) gs[kShared ? 0 : u].load_once(g + from * a.g_step);
        }
    } else {
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int64_t from = min(t + u, m.length - 1);
            xs[u].load(x + from * a.x_step);
            if (!kShared) gs[kShared ? 0 : u].load(g + from * a.g_step);
        }
    }
    find_marks(a, found, m, U, s_first, s_end, s_marked);
    __syncthreads();
    const Bits bits(a, m, t, U, group, s_marked);
    if (bits.any)
#pragma unroll
        for (int u = 0; u < U; u++)
            if (!bits.is_in(u)) {
                xs[u].clear();
                if (!kShared) gs[kShared ? 0 : u].clear();
            }
    auto start = [&](int u, float (&h)[L]) {
#pragma unroll
        for (int k = 0; k < L; k++) h[k] = 0.f;
        if (a.state && bits.is_in(u)) load_floats<L>(a.state + m.begins(a, t + u) * a.dim + c0, h);
    };
    // the tokens' maps, and the group's
    float as[kShared ? 1 : U][L], bs[U][L], A[L], B[L];
#pragma unroll
    for (int k = 0; k < L; k++) { A[k] = 1.f; B[k] = 0.f; }
#pragma unroll
    for (int u = 0; u < U; u++) {          // (a shared gate's are the same for every u: formed once)
        float g[L];
        gs[kShared ? 0 : u].get(g);
        xs[u].get(bs[u]);
#pragma unroll
        for (int k = 0; k < L; k++) {
            const Gate co = coefs_of<T, kDecay>(g[k]);
            as[kShared ? 0 : u][k] = co.a;
            if (!kDecay) bs[u][k] *= co.keep;
            A[k] *= co.a;
        }
    }
    by_marks(bits.any, [&](auto asks) {
#pragma unroll
        for (int u = 0; u < U; u++) {
            if (asks && bits.starts(u)) start(u, B);
#pragma unroll
            for (int k = 0; k < L; k++) B[k] = __builtin_fmaf(as[kShared ? 0 : u][k], B[k], bs[u][k]);
        }
    });
    if (lane == 0 && bits.starts_any(U)) atomicOr(&s_resets, 1u << group);
    if (kDecay) count_growth(as, kShared ? U : 1, s_growth[lane], s_steep);
    const int slot = lane * L, mine = group * kSlots + slot;
#pragma unroll
    for (int k = 0; k < L; k++) { s_a[mine + k] = A[k]; s_b[mine + k] = B[k]; }
    __syncthreads();
    if (threadIdx.x < kSlots) {
        join_groups<kGroups, false>(c, phase, chain, at, threadIdx.x, s_resets, s_a, s_b, kDecay && s_steep, [&](int g, int own, float h) {
            const ScanArgs& args = args_again();
            return go_forward<T, 1>(args, row, channel_of<L>(args, (int)(chain - row * c.strips), own), t0 + g * U, U, h);
        });
        if (a.states && phase != kMaps) a.states[item * kSlots + threadIdx.x] = s_b[threadIdx.x];
    }
    if (phase == kMaps) return;
    __syncthreads();
    if (!live) return;
    float h[L];
#pragma unroll
    for (int k = 0; k < L; k++) h[k] = s_b[mine + k];
    raw_t* out = (raw_t*)a.h + (row * a.length + t) * a.dim + c0;
    by_marks(bits.any, [&](auto asks) {
#pragma unroll
        for (int u = 0; u < U; u++) {
            if (asks && bits.starts(u)) start(u, h);
#pragma unroll
            for (int k = 0; k < L; k++) h[k] = __builtin_fmaf(as[kShared ? 0 : u][k], h[k], bs[u][k]);
            if (asks && kShared && !bits.is_in(u))            // (whatever the gate holds)
#pragma unroll
                for (int k = 0; k < L; k++) h[k] = 0.f;
            if (!asks || t + u < m.length) Span<T, L>::store(out + (int64_t)u * a.dim, h);
            if (asks && bits.is_end(u) && a.last) store_floats<L>(a.last + m.ends(a, t + u) * a.dim + c0, h);
        }
    });
}

// The gradient of a tile: 8 x 4096 x 2048 bf16 155 us (671 MB at 4.3 TB/s; 133 with neither waits nor sums).  The states go forward from the one kept, the gradient that reaches them goes back from the tile
// behind: its maps are s -> A s + Q of the same A.
template <class T, int L, bool kDecay, bool kShared, bool kPhased>
__global__ __launch_bounds__(kThreads, kBackWaves) void scan_grad_kernel(ScanArgs a, Chains c, int64_t first, int64_t empty) {
    constexpr int kTile = tile_of(L, kShared), kGroups = kThreads / kLanes, U = kTile / kGroups, kSlots = kLanes * L;
    static_assert(kGroups <= 32 && 2 * kSlots <= kThreads, "a bit for each group, threads for both directions");
    using raw_t = typename T::raw;
    const Phase phase = kPhased ? c.phase : kChained;
    __shared__ float s_a[kGroups * kSlots], s_b[kGroups * kSlots], s_q[kGroups * kSlots];
    __shared__ int s_first[kTile], s_end[kTile];
    __shared__ uint32_t s_marked, s_resets, s_back_resets, s_steep;
    __shared__ int s_growth[kLanes];
    __shared__ int64_t s_item;
    if (first + blockIdx.x >= c.count * c.tiles) return pass_empty(a, first + blockIdx.x - c.count * c.tiles, empty, a.dlast, a.dstate);
    const int lane = threadIdx.x % kLanes, group = threadIdx.x / kLanes;
    if (kDecay && threadIdx.x < kLanes) s_growth[threadIdx.x] = 0;
    if (threadIdx.x == 0) {
        s_resets = s_back_resets = s_steep = 0;
        s_item = take_tile(c, phase, first + blockIdx.x);
    }
    __syncthreads();
    const int64_t item = uniform(s_item), chain = item / c.tiles, at = item - chain * c.tiles, row = chain / c.strips;
    const int strip = (int)(chain - row * c.strips);
    const int64_t tile = c.tiles - 1 - at, t0 = tile * kTile, t = t0 + group * U;
    Marks m(a, row, t0);
    const int piece = strip * kLanes + lane, c0 = min(min(piece, c.pieces - 1) * L, a.dim - L);
    const bool live = piece < c.pieces;
    const raw_t* x = (const raw_t*)a.x + row * a.x_row + c0;
    const raw_t* g = (const raw_t*)a.gates + (kShared ? 0 : row * a.g_row) + c0;
    if (a.form == kRows && a.bounds && t0 >= row_end(a, row)) {
        const int64_t place = (row * a.length + t) * a.dim + c0, own = min((int64_t)U, m.length - t);
        write_zeros<T, L>(c, phase, item, at, a.dx && phase != kMaps ? (raw_t*)a.dx + place : nullptr, a.dim, own, live);
        if (phase == kMaps) return;
        if (!kShared && a.dgates) write_zeros<T, L>(c, phase, item, c.tiles, (raw_t*)a.dgates + place, a.dim, own, live);
        if (kShared && a.dgates && threadIdx.x < kSlots) c.sums[(chain * c.tiles + tile) * kSlots + threadIdx.x] = 0.f;
        return;
    }
    const raw_t* dh = a.dh ? (const raw_t*)a.dh + row * a.length * a.dim + c0 : x;
    const int64_t dh_step = a.dh ? a.dim : a.x_step, x_step = phase == kMaps ? dh_step : a.x_step;
    if (phase == kMaps) x = dh;            // (the maps of what goes back take nothing of x)
    const Found found(a, c, tile, t0);
    Span<T, L> xs[U], gs[kShared ? 1 : U], ds[U];
    if (kShared) gs[0].load(g);
    if (c.once) {
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int64_t from = min(t + u, m.length - 1);
            xs[u].load_once(x + from * x_step);
            if (!kShared) gs[kShared ? 0 : u].load_once(g + from * a.g_step);
            ds[u].load_once(dh + from * dh_step);
        }
    } else {
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int64_t from = min(t + u, m.length - 1);
            xs[u].load(x + from * x_step);
            if (!kShared) gs[kShared ? 0 : u].load(g + from * a.g_step);
            ds[u].load(dh + from * dh_step);
        }
    }
    find_marks(a, found, m, U, s_first, s_end, s_marked);
    __syncthreads();
    const Bits bits(a, m, t, U, group, s_marked);
    if (bits.any)
#pragma unroll
        for (int u = 0; u < U; u++)
            if (!bits.is_in(u)) {
                xs[u].clear();
                ds[u].clear();
                if (!kShared) gs[kShared ? 0 : u].clear();
            }
    if (!a.dh)
#pragma unroll
        for (int u = 0; u < U; u++) ds[u].clear();
    auto start = [&](int u, float (&h)[L]) {
#pragma unroll
        for (int k = 0; k < L; k++) h[k] = 0.f;
        if (a.state && bits.is_in(u)) load_floats<L>(a.state + m.begins(a, t + u) * a.dim + c0, h);
    };
    auto stop = [&](int u, float (&l)[L]) {
#pragma unroll
        for (int k = 0; k < L; k++) l[k] = 0.f;
        if (a.dlast && bits.is_in(u)) load_floats<L>(a.dlast + m.ends(a, t + u) * a.dim + c0, l);
    };
    float cs[kShared ? 1 : U][L], A[L], B[L], Q[L];
    auto again = [&] {
#pragma unroll
        for (int u = 0; u < U; u++) {
            xs[u].renew();
            ds[u].renew();
            if (!kShared || !u)
#pragma unroll
                for (int k = 0; k < L; k++) renew(cs[kShared ? 0 : u][k]);
        }
    };
#pragma unroll
    for (int k = 0; k < L; k++) { A[k] = 1.f; B[k] = 0.f; Q[k] = 0.f; }
#pragma unroll
    for (int u = 0; u < (kShared ? 1 : U); u++) {
        gs[u].get(cs[u]);
#pragma unroll
        for (int k = 0; k < L; k++) cs[u][k] = packed_of<T, kDecay>(cs[u][k]);
    }
    if (kDecay) count_growth(cs, kShared ? U : 1, s_growth[lane], s_steep);
    again();
#pragma unroll
    for (int u = 0; u < U; u++) {
        if (bits.starts(u)) start(u, B);
        float xv[L];
        xs[u].get(xv);
#pragma unroll
        for (int k = 0; k < L; k++) {
            const Gate c = coefs_of<kDecay>(cs[kShared ? 0 : u][k]);
            A[k] *= c.a;
            B[k] = step<kDecay>(B[k], xv[k], c);
        }
    }
    again();
#pragma unroll
    for (int u = U - 1; u >= 0; u--) {
        if (bits.stops(u)) stop(u, Q);
        float d[L];
        ds[u].get(d);
#pragma unroll
        for (int k = 0; k < L; k++) Q[k] = coefs_of<kDecay>(cs[kShared ? 0 : u][k]).a * (d[k] + Q[k]);
    }
    again();
    if (lane == 0 && bits.starts_any(U)) atomicOr(&s_resets, 1u << group);
    if (lane == 0 && bits.stops_any(U)) atomicOr(&s_back_resets, 1u << group);
    const int slot = lane * L, mine = group * kSlots + slot;
#pragma unroll
    for (int k = 0; k < L; k++) { s_a[mine + k] = A[k]; s_b[mine + k] = B[k]; s_q[mine + k] = Q[k]; }
    __syncthreads();
    // the states by some wavefronts, the gradients by others
    if (phase == kMaps && threadIdx.x >= kSlots) return;
    if (threadIdx.x < kSlots) {
        join_groups<kGroups, true>(c, phase, chain, at, threadIdx.x, s_back_resets, s_a, s_q, kDecay && s_steep, [&](int g, int own, float l) {
            const ScanArgs& args = args_again();
            return go_back<T, 1>(args, row, channel_of<L>(args, strip, own), t0 + g * U, U, l);
        });
        if (phase == kMaps) return;
    } else if (threadIdx.x < 2 * kSlots) {
        const int own = threadIdx.x - kSlots;
        float h = tile ? a.states[(chain * c.tiles + tile) * kSlots + own] : 0.f;      // (a row begins with a sequence, or with tokens of none)
        if (kDecay && s_steep) {
            const ScanArgs& args = args_again();
            for (int i = 0; i < kGroups; i++) {
                const float gb = s_b[i * kSlots + own];
                s_b[i * kSlots + own] = h;
                h = s_resets >> i & 1 ? gb : go_forward<T, 1>(args, row, channel_of<L>(args, strip, own), t0 + i * U, U, h);
            }
        } else {
#pragma unroll 8
            for (int i = 0; i < kGroups; i++) {
                const float ga = s_a[i * kSlots + own], gb = s_b[i * kSlots + own];
                s_b[i * kSlots + own] = h;
                h = s_resets >> i & 1 ? gb : __builtin_fmaf(ga, h, gb);
            }
        }
    }
    __syncthreads();
    float h[L], l[L], before[U][L], sum[L];
#pragma unroll
    for (int k = 0; k < L; k++) {
        h[k] = s_b[mine + k];
        l[k] = s_q[mine + k];
        sum[k] = 0.f;
    }
    const int64_t place = (row * a.length + t) * a.dim + c0;
    raw_t *dx = a.dx ? (raw_t*)a.dx + place : nullptr, *dg = a.dgates && !kShared ? (raw_t*)a.dgates + place : nullptr;
#pragma unroll
    for (int u = 0; u < U; u++) {
        if (bits.starts(u)) start(u, h);
        float xv[L];
        xs[u].get(xv);
#pragma unroll
        for (int k = 0; k < L; k++) {
            before[u][k] = h[k];
            h[k] = step<kDecay>(h[k], xv[k], coefs_of<kDecay>(cs[kShared ? 0 : u][k]));
        }
    }
    again();
#pragma unroll
    for (int u = U - 1; u >= 0; u--) {
        if (bits.stops(u)) stop(u, l);
        float d[L], xv[L], by_x[L], by_g[L];
        ds[u].get(d);
        xs[u].get(xv);
#pragma unroll
        for (int k = 0; k < L; k++) {
            const Gate c = coefs_of<kDecay>(cs[kShared ? 0 : u][k]);
            const float reaches = d[k] + l[k];
            by_x[k] = kDecay ? reaches : reaches * c.keep;
            l[k] = c.a * reaches;
            by_g[k] = kDecay ? reaches * before[u][k] : l[k] * c.keep * (before[u][k] - xv[k]);
            if (kShared && !bits.is_in(u)) by_x[k] = by_g[k] = 0.f;
            if (kShared) sum[k] += by_g[k];
        }
        if (live && t + u < m.length) {
            if (dx) Span<T, L>::store(dx + (int64_t)u * a.dim, by_x);
            if (dg) Span<T, L>::store(dg + (int64_t)u * a.dim, by_g);
        }
        if (bits.is_first(u) && live && a.dstate) store_floats<L>(a.dstate + m.begins(a, t + u) * a.dim + c0, l);
    }
    if (!kShared || !a.dgates) return;
    // (s_a is read by nobody any more)
#pragma unroll
    for (int k = 0; k < L; k++) s_a[mine + k] = sum[k];
    __syncthreads();
    if (threadIdx.x < kSlots) {
        float total = 0.f;
#pragma unroll 8
        for (int i = 0; i < kGroups; i++) total += s_a[i * kSlots + threadIdx.x];
        c.sums[(chain * c.tiles + tile) * kSlots + threadIdx.x] = total;
    }
}

// Few chains of many tiles: a chain's wait from tile to tile, 0.1 us, is longer than their tokens take.  So their maps are formed by a launch of their own,
// joined here, and the tokens read again.  One wavefront goes from map to map, in the order and by the steps of tiles that wait for one another: equal
// bits.  What it reads comes by all of them, a round ahead, and leaves by all of them, a round behind (by that one alone stores wait for stores); a
// workgroup has 16 channels (2048 tiles of 64 channels 43 us; with all of them 51, of which one CU reads and writes 30).
constexpr int kLinkers = 1024, kLinkWords = 8, kLinkRound = kLinkers * kLinkWords;
constexpr int link_width(int slots) { return slots < 16 ? slots : 16; }
template <class T, int kSlots, bool kDecay>
__global__ __launch_bounds__(kLinkers) void link_kernel(Chains c, ScanArgs a, bool gradient, int tokens) {
    constexpr int U = 8, kWidth = link_width(kSlots), kParts = kSlots / kWidth;
    struct alignas(8) Map { uint32_t a, b; };         // a's place is the state's once it is joined
    __shared__ Map s_maps[2][kLinkRound + U * kWidth];
    __shared__ uint32_t s_steep;
    const int64_t words = c.tiles * kWidth, own = (int64_t)(blockIdx.x / kParts) * c.tiles * kSlots + blockIdx.x % kParts * kWidth;
    const uint64_t* maps = c.maps + own;
    uint32_t* states = c.states + own;
    auto place = [](int64_t word) { return word / kWidth * kSlots + word % kWidth; };
    uint64_t m[kLinkWords];
    auto load = [&](int64_t from) {
#pragma unroll
        for (int i = 0; i < kLinkWords; i++) m[i] = maps[place(min(from + i * kLinkers + (int)threadIdx.x, words - 1))];
    };
    auto leave = [&](int64_t from, int half) {
#pragma unroll
        for (int i = 0; i < kLinkWords; i++) {
            const int at = i * kLinkers + threadIdx.x;
            if (from + at < words) states[place(from + at)] = word_of(__builtin_bit_cast(float, s_maps[half][at].a));
        }
    };
    // What is behind a tile without a map, whose tokens are all of one sequence.
    auto go_through = [&](int64_t at, float h) {
        const int64_t chain = blockIdx.x / kParts, row = chain / c.strips;
        const int channel = channel_of<kSlots / kLanes>(a, (int)(chain - row * c.strips), blockIdx.x % kParts * kWidth + threadIdx.x);
        return gradient ? go_back<T, 4>(a, row, channel, (c.tiles - 1 - at) * tokens, tokens, h) : go_forward<T, 4>(a, row, channel, at * tokens, tokens, h);
    };
    load(0);
    if (kDecay) {
        if (threadIdx.x == 0) s_steep = 0;
        __syncthreads();
    }
    float h = 0.f;
    int half = 0;
    for (int64_t from = 0; from < words; from += kLinkRound, half ^= 1) {
        // (each thread's own places, whose states it has taken away before)
        bool steep = false;
#pragma unroll
        for (int i = 0; i < kLinkWords; i++) {
            s_maps[half][i * kLinkers + threadIdx.x] = Map{(uint32_t)m[i], (uint32_t)(m[i] >> 32)};
            steep |= kDecay && (uint32_t)m[i] == kSteepMap;
        }
        if (steep) s_steep = 1;
        __syncthreads();
        if (from) leave(from - kLinkRound, half ^ 1);
        if (from + kLinkRound < words) load(from + kLinkRound);
        if (threadIdx.x >= kWidth) continue;
        // (behind the last tile maps of no use are joined, whose states go nowhere)
        const int tiles = (int)(min((int64_t)kLinkRound, words - from) / kWidth);
        Map *at = s_maps[half] + threadIdx.x, next[U];
        if (kDecay && __builtin_expect(s_steep != 0, 0)) {
            for (int i = 0; i < tiles; i++, at += kWidth) {
                const float b = __builtin_bit_cast(float, at->b);
                if (at->a == kSteepMap) h = go_through(from / kWidth + i, h);
                else h = at->a == kUnset ? b : __builtin_fmaf(__builtin_bit_cast(float, at->a), h, b);
                at->a = __builtin_bit_cast(uint32_t, h);
            }
            continue;
        }
        // (in this order: in another the loop's first wait is for all that is under way, and those of a round are for each other)
#pragma unroll
        for (int u = 0; u < U; u++) {
            next[u] = at[u * kWidth];
            if (u % 2) __builtin_amdgcn_sched_barrier(0);
        }
#pragma unroll 2
        for (int i = 0; i < tiles; i += U, at += U * kWidth) {
            Map map[U];
#pragma unroll
            for (int u = 0; u < U; u++) {
                map[u] = next[u];
                next[u] = at[(U + u) * kWidth];
            }
#pragma unroll
            for (int u = 0; u < U; u++) {
                const float b = __builtin_bit_cast(float, map[u].b);
                h = map[u].a == kUnset ? b : __builtin_fmaf(__builtin_bit_cast(float, map[u].a), h, b);
                at[u * kWidth].a = __builtin_bit_cast(uint32_t, h);
            }
        }
    }
    __syncthreads();
    const int64_t from = (words - 1) / kLinkRound * kLinkRound;
    leave(from, (int)(from / kLinkRound % 2));
}

// The tiles' sums of a shared gate's gradient, in 64 bits and one order.
constexpr int kSumChannels = 16;
template <class T>
__global__ __launch_bounds__(1024) void sum_kernel(ScanArgs a, Chains c, int len) {
    __shared__ double s_sum[1024];
    const int own = threadIdx.x % kSumChannels, part = threadIdx.x / kSumChannels, parts = 1024 / kSumChannels;
    const int channel = blockIdx.x * kSumChannels + own;
    double sum = 0.0;
    if (channel < a.dim) {
        const int piece = channel / len, strip = piece / kLanes;
        // (of the last piece's channels the first are those of the one before)
        const int slot = piece % kLanes * len + channel - min(piece * len, a.dim - len);
        const int64_t cells = a.rows * c.tiles;
        for (int64_t i = part; i < cells; i += parts)
            sum += c.sums[((i / c.tiles * c.strips + strip) * c.tiles + i % c.tiles) * c.slots + slot];
    }
    s_sum[threadIdx.x] = sum;
    for (int half = parts / 2; half; half /= 2) {
        __syncthreads();
        if (part < half) s_sum[threadIdx.x] += s_sum[threadIdx.x + half * kSumChannels];
    }
    __syncthreads();
    if (part == 0 && channel < a.dim) ((typename T::raw*)a.dgates)[channel] = (typename T::raw)(float)s_sum[threadIdx.x];
}

// ---- launches ----------------------------------------------------------------------------
int fill(const ScanArgs& a, const Chains& c, int tokens, hipStream_t s) {
    if (c.tiles <= 1) return 0;
    const int64_t words = c.phase == kChained ? ((char*)c.from - (char*)c.tickets) / 16 : 0, blocks = (words + kThreads - 1) / kThreads;
    const int64_t more = a.form == kPacked ? (c.tiles + kThreads - 1) / kThreads : 0;
    if (!(blocks + more)) return 0;
    fill_kernel<<<(uint32_t)(blocks + more), kThreads, 0, s>>>((u32x4*)c.tickets, words, blocks, a, c.from, c.tiles, tokens);
    DCIH_HIP(hipGetLastError());
    return 0;
}

template <class T, int L, bool kDecay, bool kShared>
int run(const ScanArgs& a, int dtype, bool gradient, hipStream_t s) {
    Chains c{};
    lay_out(c, a.work, a.rows, a.length, a.dim, dtype, gradient, a.shared);
    constexpr int kSize = sizeof(typename T::raw), kLine = 128;
    c.apart = a.x_step * kSize % kLine == 0 && (uintptr_t)a.x % kLine == 0 && a.dim * kSize % kLine == 0;
    // what the caches hold is read through them: 30011 x 1024 f16 with gradients 164 us, 171 past them; what they do not, past them
    // (65536 x 4096 bf16 packed 351 us, 366)
    c.once = c.apart && a.rows * a.length * a.dim * kSize * (kShared ? 1 : 2) > (int64_t)256 << 20;
    c.phase = c.count <= kFewChains && c.tiles >= kManyTiles ? kMaps : kChained;
    if (int rc = fill(a, c, tile_of(L, kShared), s)) return rc;
    const int64_t tiles = c.count * c.tiles;
    auto launch = [&](auto phased, int64_t empty) {
        constexpr bool kPhased = decltype(phased)::value;
        for (int64_t first = 0; first < tiles + empty; first += kMaxGrid) {
            const uint32_t grid = (uint32_t)std::min(kMaxGrid, tiles + empty - first);
            if (gradient) scan_grad_kernel<T, L, kDecay, kShared, kPhased><<<grid, kThreads, 0, s>>>(a, c, first, empty);
            else scan_kernel<T, L, kDecay, kShared, kPhased><<<grid, kThreads, 0, s>>>(a, c, first, empty);
            DCIH_HIP(hipGetLastError());
        }
        return 0;
    };
    // (workgroups that pass on the states of sequences without tokens)
    const int64_t empty = a.bounds && (gradient ? a.dstate : a.last) ? std::min((a.sequences + kEmpty - 1) / kEmpty, kEmptyGrid) : 0;
    if (c.phase == kMaps) {
        if (int rc = launch(std::true_type{}, 0)) return rc;
        link_kernel<T, kLanes * L, kDecay><<<(uint32_t)(c.count * (kLanes * L / link_width(kLanes * L))), kLinkers, 0, s>>>(c, a, gradient, tile_of(L, kShared));
        DCIH_HIP(hipGetLastError());
        c.phase = kApply;
        if (int rc = launch(std::true_type{}, empty)) return rc;
    } else if (int rc = launch(std::false_type{}, empty)) {
        return rc;
    }
    if (gradient && kShared && a.dgates) {
        sum_kernel<T><<<(uint32_t)((a.dim + kSumChannels - 1) / kSumChannels), 1024, 0, s>>>(a, c, L);
        DCIH_HIP(hipGetLastError());
    }
    return 0;
}

template <class T, int L, bool kDecay>
int run_short(const ScanArgs& a, hipStream_t s) {
    const int pieces = (a.dim + L - 1) / L;
    const int64_t threads = a.rows * pieces, most = kMaxGrid * kThreads;
    for (int64_t first = 0; first < threads; first += most) {
        const uint32_t grid = (uint32_t)((std::min(most, threads - first) + kThreads - 1) / kThreads);
        if (a.states && a.length > tile_of(L, a.shared)) {
            if (tile_of(L, a.shared) == 128) short_kernel<T, L, kDecay, 8, 128><<<grid, kThreads, 0, s>>>(a, pieces, first);
            else short_kernel<T, L, kDecay, 8, 256><<<grid, kThreads, 0, s>>>(a, pieces, first);
        } else if (a.length > 4) {
            short_kernel<T, L, kDecay, 8, 0><<<grid, kThreads, 0, s>>>(a, pieces, first);
        } else {
            short_kernel<T, L, kDecay, 4, 0><<<grid, kThreads, 0, s>>>(a, pieces, first);
        }
        DCIH_HIP(hipGetLastError());
    }
    return 0;
}

template <class T, int L>
int by_gates(const ScanArgs& a, int dtype, bool gradient, hipStream_t s) {
    if (!gradient && scan_is_short(a, dtype)) {
        if (L > 1 && (a.length > kShort || a.rows * a.dim > kSingles * (a.length > kSteps ? 2 : 1))) return a.decay ? run_short<T, L, true>(a, s) : run_short<T, L, false>(a, s);
        return a.decay ? run_short<T, 1, true>(a, s) : run_short<T, 1, false>(a, s);
    }
    if (a.decay) return a.shared ? run<T, L, true, true>(a, dtype, gradient, s) : run<T, L, true, false>(a, dtype, gradient, s);
    return a.shared ? run<T, L, false, true>(a, dtype, gradient, s) : run<T, L, false, false>(a, dtype, gradient, s);
}

template <class T>
int by_length(const ScanArgs& a, int dtype, bool gradient, hipStream_t s) {
    if (span_len(a.dim, dtype) == 1) return by_gates<T, 1>(a, dtype, gradient, s);
    return by_gates<T, Piece<T>::kLen>(a, dtype, gradient, s);
}

// Short sequences that stand one behind the other share tiles: as many as one holds.
ScanArgs flattened(ScanArgs a, int tile) {
    auto flat = [&](int64_t row, int64_t step) { return row == a.length * step; };
    if (a.form != kRows || 2 * a.length > tile || a.rows == 1 || !flat(a.x_row, a.x_step) || (!a.shared && !flat(a.g_row, a.g_step)))
        return a;
    const int64_t together = tile / a.length;
    a.form = kFlat;
    a.each = a.length;
    a.total = a.rows * a.length;
    a.length *= together;
    a.rows = (a.rows + together - 1) / together;
    a.x_row *= together;
    a.g_row *= together;
    a.states = nullptr;               // (rows begin with sequences)
    return a;
}

int dispatch(const ScanArgs& a, int dtype, bool gradient, hipStream_t s) {
    switch (dtype) {
        case DCIH_F32: return by_length<F32>(a, dtype, gradient, s);
        case DCIH_F16: return by_length<F16>(a, dtype, gradient, s);
        default: return by_length<BF16>(a, dtype, gradient, s);
    }
}

}  // namespace

int64_t scan_state_floats(int64_t rows, int64_t length, int dim, int dtype) {
    Chains c{};
    lay_out(c, nullptr, rows, length, dim, dtype, false, false);
    return c.count * c.tiles * c.slots;
}

int64_t scan_work_bytes(int64_t rows, int64_t length, int dim, int dtype) {
    Chains c{};
    return std::max(lay_out(c, nullptr, rows, length, dim, dtype, true, true), lay_out(c, nullptr, rows, length, dim, dtype, true, false));
}

bool scan_is_short(const ScanArgs& a, int dtype) {
    if (a.form != kRows || a.length <= kShort) return a.form == kRows;
    const int len = span_len(a.dim, dtype), tile = tile_of(len, a.shared);
    if (a.length <= tile && 8 * a.length >= 7 * tile) return false;
    return a.rows * ((a.dim + len - 1) / len) >= std::min(kManyPieces * a.length, kEnoughPieces);
}

int scan(const ScanArgs& a, int dtype, hipStream_t s) { return dispatch(scan_is_short(a, dtype) ? a : flattened(a, tile_of(span_len(a.dim, dtype), a.shared)), dtype, false, s); }
int scan_grad(const ScanArgs& a, int dtype, hipStream_t s) { return dispatch(flattened(a, tile_of(span_len(a.dim, dtype), a.shared)), dtype, true, s); }

int scan_copy(const float* from, float* to, int64_t n, hipStream_t s) {
    copy_kernel<<<(uint32_t)std::min<int64_t>((n + kThreads - 1) / kThreads, 2048), kThreads, 0, s>>>(from, to, n);
    DCIH_HIP(hipGetLastError());
    return 0;
}

}  // namespace dcih
