// Optimiser-step operators over lists of tensors: the global gradient norm, clipping by it, and the Adam update that takes
// the clipped gradient (C ABI: include/mbrl.h).
//
// Mathematics, over the values x of all tensors of a list:
//   norm   s = (sum |x|^p)^(1/p), p = 1, 2 or infinity
//   clip   x <- c x,  c = min(1, max_norm / (s + 1e-6))
//   Adam   g <- c g (+ wd x)          m <- b1 m + (1 - b1) g      v <- b2 v + (1 - b2) g^2
//          x <- x (1 - lr wd) - lr / (1 - b1^t)  m / (sqrt(v / (1 - b2^t)) + eps)
//
// Layout.  Every tensor is cut into units of 2^shift values, a unit belongs to one wave, and the units of the whole list are
// spread over the waves of a launch.  The list travels in the kernel arguments (at most 4 KB), so a call uploads nothing,
// can be captured into a graph, and keeps nothing of one call for the next; a longer list takes several launches.  A wave
// finds its unit's tensor by comparing 64 unit ends at once (owner()).  Sums are float64 in every case: squares of float32
// and bfloat16 values cannot overflow there, and each partial sum has a fixed place and is added in a fixed order, so the
// norm is a function of the values, sizes and types alone: not of which wave is done first (no atomics) and not of addresses.
//
// What bounds it.  Memory, from some 10 MB on: a multiplication or two a value for the norm and clipping, some 60
// instructions (a division and a root among them) for the update.  Measured on an MI355X, where a copy of 4 GiB runs at 4.8
// TB/s and x *= c at 5.9, 10 float32 tensors of as many values in all, every launch included:
//   values    norm               clip (scaled)       Adam                Adam, clipped
//   8e3       3.5 us             5.1 us              6.2 us              8.3 us         one launch
//   5e5       4.8 us             6.7 us              6.2 us              8.1 us         two launches
//   8e6       6.6 us, 4.9 TB/s   14.7 us, 6.5 TB/s   40 us, 5.6 TB/s     46 us          from the cache
//   268e6     164 us, 6.5 TB/s   525 us, 6.1 TB/s    1.22 ms, 6.2 TB/s   1.37 ms        from memory
// (clip: two reads and a write).  Below that it is the launches: an empty one takes 2.2 us of the device and 3.7 us of the
// host, so small lists are done in one.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <cstdio>
#include <new>
#include <type_traits>
#include <vector>

#include "../../include/mbrl.h"
#include "abi_error.hpp"

namespace {
using mbrl::report;

constexpr int kWave = 64, kThreads = 256, kWaves = kThreads / kWave;

// Bytes that one block of 16 waves takes on alone, in one launch (of gradients; of all four tensors for Adam).  Against the two
// launches of longer lists, device / host time in us for float32: norm of 64e3 values 4.7 / 5.0 for 4.6 / 8.1, clipping of
// 24e3 6.7 / 6.9 for 6.0 / 8.7, Adam of 12e3 6.5 / 6.9 for 5.1 / 8.7 and clipped 8.8 / 9.2 for 7.0 / 9.6.  Twice as much is slower
// both ways for the last two (24e3: 10.8 / 11.2 for 5.5 / 8.8, clipped 13.5 / 13.9 for 7.4 / 9.8).  The bounds go by the host's time,
// that of a call; a replayed graph pays the device's alone, and would be better off with two launches near them.
constexpr int64_t kSmallNorm = 256 << 10, kSmallClip = 96 << 10, kSmallAdam = 192 << 10;
// And tensors, of which a wave takes 1 in 16 one after another: clipping of 64 (4000 values) 8.8 / 9.3 for 7.2 / 10.5, of 96 11.6 /
// 12.1 for 7.3 / 11.3; the norm of 128 8.1 / 8.9 for 5.3 / 10.3, of 160 9.5 / 10.2 for 5.3 / 11.5.
constexpr int kSmallNormCount = 128, kSmallClipCount = 64;
constexpr int kSmallThreads = 1024, kSmallWaves = kSmallThreads / kWave;
constexpr int kSmallShift = 8;            // units of one 1 KB load a wave: 800-value tensors 6.2 us for 6.7 with twice that (Adam)

// Middle lists: up to kMaxBlocks blocks (4 a CU) stay and take units of 2^9 values or more.  Clipping and norm walk a wave's units
// one after another (walk()): 8e6 values 7.0 us for 10.2 dealt out in turn, 16e6 13.4 for 15.4.  Two units a wave at least:
// 2e6 values 5.5 us for 5.9 with one.
constexpr int kMaxBlocks = 1024, kUnits = 2;
constexpr int kMinShift = 9, kMaxShift = 12;
constexpr int kMaxParts = 2048;           // partial sums that every block of a second launch joins for itself, not a launch between

// Large lists: what does not stay in the 256 MB last-level cache is read and written past it (nontemporal), and the scaling and
// the update take short units in blocks that do not stay, so that what is under way at a time lies together.  268e6 float32
// values: norm 161 us for 180, scaling 357 for 440, Adam 1226 for 1505.  From a quarter of the cache on it pays for data that
// was not in it (float32, other tensors used between: clipping of 32e6 values 67 us for 81, Adam of 8e6 43 for 51; of 4e6 26
// for 28) and costs little for data that was (65 -> 71, 38 -> 41).  Sums gain from half of it on (a norm
// of 32e6: 25.2 us for 27.1; 16e6: 17.3 for 17.0), before a scaling too, though it finds less in the cache then, if there is one:
// 50e6 values 39.5 us for 42.8 untouched and 105 for 100 scaled, 117e6 of bfloat16 44 for 48.5 and 119 for 116.  Before an
// update, which reads the gradients in any case, what is read stays in the cache, up to its size (50e6: 244 us for 258).
constexpr int64_t kCache = int64_t(256) << 20;
// Values of a unit.  Of the update one load a lane and tensor (268e6 float32 values: 1.23 ms for 1.30 with two, bfloat16 0.93 for
// 1.04; 128e6 of float64, half as many a load: 1.19 for 1.25), compiled for that alone: 72 registers for 117 leave room for 7
// waves for 4 (bfloat16 0.93 ms for 1.08).  Of the scaling four loads (496 us for 548 with two, 514 with eight), and two units
// a wave, for lists that need no scaling: its blocks alone take 11 us for 22 with one.
constexpr int kAdamShift = 8, kAdamShift64 = 7, kScaleShift = 10, kScaleShift16 = 11;
constexpr int kStreamBlocks = 1 << 22;    // HIP counts a launch's threads in 32 bits

// ---- element types: what is stored, what is computed with, values in 16 bytes ----
struct F64 { using T = double; using C = double; static constexpr int V = 2; };
struct F32 { using T = float; using C = float; static constexpr int V = 4; };
struct B16 { using T = __bf16; using C = float; static constexpr int V = 8; };
struct F16 { using T = _Float16; using C = float; static constexpr int V = 8; };

// Vectors with the alignment of their elements: a tensor may start at any element (a slice of a bucket), and the memory
// system takes a 16-byte access at any such address, so there is one path for all alignments.
template <class T, int V> struct Pack { T v[V]; };
template <int kBytes, int kAlign> struct Raw { typedef uint32_t type __attribute__((ext_vector_type(kBytes / 4), aligned(kAlign), may_alias)); };
template <bool kStream, int V, class T>
__device__ __forceinline__ Pack<T, V> load(const T *p) {
    using R = typename Raw<int(sizeof(Pack<T, V>)), int(sizeof(T))>::type;
    const R *q = reinterpret_cast<const R *>(p);
    return __builtin_bit_cast(Pack<T, V>, kStream ? __builtin_nontemporal_load(q) : *q);
}
template <bool kStream, int V, class T>
__device__ __forceinline__ void store(T *p, const Pack<T, V> &r) {
    using R = typename Raw<int(sizeof(Pack<T, V>)), int(sizeof(T))>::type;
    R *q = reinterpret_cast<R *>(p);
    if (kStream) __builtin_nontemporal_store(__builtin_bit_cast(R, r), q);
    else *q = __builtin_bit_cast(R, r);
}

// Calls f(the element type) for a type code, which is the same in all lanes.
template <class F>
__device__ __forceinline__ void by_type(int code, F &&f) {
    if (code == MBRL_DT_FLOAT) f(F32{});
    else if (code == MBRL_DT_DOUBLE) f(F64{});
    else if (code == MBRL_DT_BFLOAT) f(B16{});
    else f(F16{});
}

// ---- lists in kernel arguments ----
// A list of up to kFew tensors has a size of its own: filling 4 KB of arguments takes the host 0.5 us more than 350 bytes.  The
// others hold as many as can be in the 4 KB of a launch, and are packed for it (device addresses have 48 bits): 400 tensors take
// 2 launches for their sums and 4 for their update instead of 3 and 5 with fields of 8 bytes (8e6 float32 values: norm 14.3 us ->
// 11.6, clipping 31.2 -> 25.2, Adam clipped 79 -> 73).  Unpacking is waited for where one block does it all: 16 tensors of
// 500 values 5.65 us for 5.05 (Adam, with the hardware's root and quotient).
constexpr int kFew = 16;
__host__ __device__ __forceinline__ void *address(uint32_t lo, uint32_t hi) { return reinterpret_cast<void *>(uint64_t(hi) << 32 | lo); }
__host__ __forceinline__ uint32_t upper(const void *p) { return uint32_t(uintptr_t(p) >> 32); }

template <int K_, bool = (K_ > kFew)> struct Units {
    static constexpr int K = K_;
    uint32_t end[K];      // units of the tensors up to and including this one
    uint32_t n[K];        // values, the lower 32 bits
    uint32_t rest[K];     // the upper 6 | type code << 6 | head << 8; the upper half is the list's
    int count, shift;
    uint32_t units;
    __device__ __forceinline__ int64_t values(int t) const { return int64_t(rest[t] & 63) << 32 | n[t]; }
    __device__ __forceinline__ int type(int t) const { return rest[t] >> 6 & 3; }
    __device__ __forceinline__ int head(int t) const { return rest[t] >> 8 & 63; }
    void put(int t, int64_t values, int type, int64_t head) {
        n[t] = uint32_t(values);
        rest[t] = uint32_t(values >> 32) | uint32_t(type) << 6 | uint32_t(head) << 8;
    }
};
template <int K_> struct Units<K_, false> {
    static constexpr int K = K_;
    uint64_t n[K];        // values << 8 | head << 2 | type code
    uint32_t end[K];
    int count, shift;
    uint32_t units;
    __device__ __forceinline__ int64_t values(int t) const { return n[t] >> 8; }
    __device__ __forceinline__ int type(int t) const { return n[t] & 3; }
    __device__ __forceinline__ int head(int t) const { return n[t] >> 2 & 63; }
    void put(int t, int64_t values, int type, int64_t head) { n[t] = uint64_t(values) << 8 | uint64_t(head) << 2 | uint64_t(type); }
};
// Lists of one tensor each (x), and of a gradient with its parameter, m and v; put() comes after the units' own.
template <int K, bool = (K > kFew)> struct Ones {
    Units<K> u;
    uint32_t lo[K];
    __device__ __forceinline__ void *x(int t) const { return address(lo[t], u.rest[t] >> 16); }
    void put(int t, const void *p) {
        lo[t] = uint32_t(uintptr_t(p));
        u.rest[t] |= upper(p) << 16;
    }
};
template <int K> struct Ones<K, false> {
    Units<K, false> u;
    const void *at[K];
    __device__ __forceinline__ void *x(int t) const { return const_cast<void *>(at[t]); }
    void put(int t, const void *p) { at[t] = p; }
};
template <int K, bool = (K > kFew)> struct Fours {
    Units<K> u;
    struct { uint32_t lo[4], hi[2]; } at[K];
    template <int I> __device__ __forceinline__ void *get(int t) const { return address(at[t].lo[I], at[t].hi[I / 2] >> I % 2 * 16 & 0xffff); }
    void put(int t, const void *g, const void *p, const void *m, const void *v) {
        const void *a[4] = {g, p, m, v};
        for (int i = 0; i < 4; i++) at[t].lo[i] = uint32_t(uintptr_t(a[i]));
        for (int i = 0; i < 2; i++) at[t].hi[i] = upper(a[2 * i]) | upper(a[2 * i + 1]) << 16;
    }
    __device__ __forceinline__ void *x(int t) const { return get<0>(t); }
};
template <int K> struct Fours<K, false> {
    Units<K, false> u;
    const void *at[4][K];
    template <int I> __device__ __forceinline__ void *get(int t) const { return const_cast<void *>(at[I][t]); }
    void put(int t, const void *g, const void *p, const void *m, const void *v) { at[0][t] = g, at[1][t] = p, at[2][t] = m, at[3][t] = v; }
    __device__ __forceinline__ void *x(int t) const { return get<0>(t); }
};
template <int K> using NormList = Ones<K>;
template <int K> using UpdateList = Fours<K>;
template <int K> using SmallNorm = Ones<K, false>;        // for one block
template <int K> struct BeginList : Ones<K> { float *step[K]; double lr[K], wd[K]; };        // of the gradients
template <int K> struct SmallAdam { Fours<K, false> l; float *step[K]; double lr[K], wd[K]; };          // both, for one block
// Steps alone.  Their rates come from few groups: the list holds each pair once.
constexpr int kCountList = 416, kRates = 64;
struct CountList {
    double lr[kRates], wd[kRates];
    uint32_t lo[kCountList];
    uint16_t hi[kCountList];
    uint8_t rate[kCountList];
    int count, rates;
    // false: full
    bool put(float *step, double lr_, double wd_) {
        int k = 0;
        while (k < rates && !(lr[k] == lr_ && wd[k] == wd_)) k++;
        if (count == kCountList || k == kRates) return false;
        if (k == rates) lr[k] = lr_, wd[k] = wd_, rates++;
        lo[count] = uint32_t(uintptr_t(step));
        hi[count] = uint16_t(upper(step));
        rate[count++] = uint8_t(k);
        return true;
    }
};
constexpr int kNormList = 246, kBeginList = 98, kAdamList = 109, kSmallAdamCount = 58;
static_assert(sizeof(NormList<kNormList>) <= 3968 && sizeof(BeginList<kBeginList>) <= 3968 && sizeof(UpdateList<kAdamList>) <= 3968 &&
              sizeof(SmallAdam<kSmallAdamCount>) <= 3968 && sizeof(CountList) <= 3968, "kernel arguments are 4 KB");

// What the update of one tensor multiplies with.
struct Scalars { double size, root, keep, l2; };

__device__ __forceinline__ uint32_t wave_of_block() { return __builtin_amdgcn_readfirstlane(threadIdx.x / kWave); }
__device__ __forceinline__ uint32_t wave_of_grid() { return blockIdx.x * kWaves + wave_of_block(); }
__device__ __forceinline__ uint32_t waves_of_grid() { return gridDim.x * kWaves; }

// The tensor that unit `unit` belongs to: as many as end at or before it come first.  All ends are on their way at once.
template <class U>
__device__ __forceinline__ int owner(const U &u, uint32_t unit) {
    const int lane = threadIdx.x % kWave;
    uint32_t end[(U::K + kWave - 1) / kWave];
#pragma unroll
    for (int k = 0; k < U::K; k += kWave) end[k / kWave] = u.end[min(k + lane, u.count - 1)];
    int t = 0;
#pragma unroll
    for (int k = 0; k < U::K; k += kWave) t += __popcll(__ballot(k + lane < u.count && end[k / kWave] <= unit));
    return __builtin_amdgcn_readfirstlane(t);
}

// Values of one tensor, one after another: n from `first` on, which begins a cache line, and where the tensor begins the `head`
// before the first line.
struct Piece { int t, type, head; int64_t first; int n; };

// Units `unit` to `stop` of the list, as far as they lie in tensor t; moves `unit` past them.
template <class U>
__device__ __forceinline__ Piece piece(const U &u, int t, uint32_t &unit, uint32_t stop) {
    Piece p;
    p.t = t;
    const uint32_t end = min(stop, u.end[t]), skipped = unit - (t ? u.end[t - 1] : 0);
    const int head = u.head(t);
    p.type = u.type(t);
    p.head = skipped ? 0 : head;
    p.first = head + (int64_t(skipped) << u.shift);
    p.n = int(min(u.values(t) - p.first, int64_t(end - unit) << u.shift));
    unit = end;
    return p;
}

// The share of wave `wave` of `waves`: every waves-th unit, so that waves that run together read what lies together.
template <class U, class F>
__device__ __forceinline__ void dealt(const U &u, uint32_t wave, uint32_t waves, F f) {
    for (uint32_t i = wave; i < u.units; i += waves) {
        uint32_t unit = i;
        f(piece(u, owner(u, unit), unit, unit + 1));
    }
}
// The same, but units one after another, so that a wave has few tensors to find.
template <class U, class F>
__device__ __forceinline__ void shared_out(const U &u, uint32_t wave, uint32_t waves, F f) {
    const uint32_t each = (u.units + waves - 1) / waves, stop = min(u.units, (wave + 1) * each);
    uint32_t unit = wave * each;
    if (unit >= stop) return;
    for (int t = owner(u, unit); unit < stop; t++)
        if (u.end[t] > unit) f(piece(u, t, unit, stop));        // an empty tensor ends where it begins
}
template <bool kStream, class U, class F>
__device__ __forceinline__ void walk(const U &u, F f) {
    if constexpr (kStream) dealt(u, wave_of_grid(), waves_of_grid(), f);
    else shared_out(u, wave_of_grid(), waves_of_grid(), f);
}

// ---- norm ----
// P == 0 is the largest |x|: an order on the bits of |x|, in which NaN is larger than infinity, so that a NaN stays.
__device__ __forceinline__ double larger(double a, double b) {
    const uint64_t x = __double_as_longlong(a), y = __double_as_longlong(b);
    return __longlong_as_double(x > y ? x : y);
}
template <int P>
__device__ __forceinline__ double join(double a, double b) {
    if constexpr (P == MBRL_NORM_INF) return larger(a, b);
    return a + b;
}
template <int P>
__device__ __forceinline__ double add(double acc, double x) {
    if constexpr (P == MBRL_NORM_TWO) return fma(x, x, acc);
    if constexpr (P == MBRL_NORM_ONE) return acc + fabs(x);
    return larger(acc, fabs(x));
}

// Every thread gets the join of all threads' values; W: waves of the block.
template <int P, int W>
__device__ __forceinline__ double block_join(double a) {
    __shared__ double part[W];
    for (int d = kWave / 2; d; d /= 2) a = join<P>(a, __shfl_xor(a, d));
    __syncthreads();
    if (threadIdx.x % kWave == 0) part[threadIdx.x / kWave] = a;
    __syncthreads();
    a = part[0];
    for (int w = 1; w < W; w++) a = join<P>(a, part[w]);
    return a;
}

template <int P, bool kStream, class E>
__device__ __forceinline__ double piece_norm(E, const void *base, const Piece &p, double acc) {
    using T = typename E::T;
    constexpr int V = E::V, kStep = kWave * V;
    const T *x = static_cast<const T *>(base) + p.first;
    const int lane = threadIdx.x % kWave, n = p.n;
    int i = lane * V;
    double a[2] = {acc, 0.0};
    for (; i + 3 * kStep + V <= n; i += 4 * kStep) {
        Pack<T, V> r[4];
#pragma unroll
        for (int k = 0; k < 4; k++) r[k] = load<kStream, V>(x + i + k * kStep);
#pragma unroll
        for (int k = 0; k < 4; k++)
#pragma unroll
            for (int j = 0; j < V; j++) a[j % 2] = add<P>(a[j % 2], double(typename E::C(r[k].v[j])));
    }
    for (; i + V <= n; i += kStep) {
        const Pack<T, V> r = load<kStream, V>(x + i);
#pragma unroll
        for (int j = 0; j < V; j++) a[j % 2] = add<P>(a[j % 2], double(typename E::C(r.v[j])));
    }
    const int tail = n / V * V + lane;        // the last n % V values, one a lane, and those of the head
    if (tail < n) a[1] = add<P>(a[1], double(typename E::C(x[tail])));
    if (lane < p.head) a[1] = add<P>(a[1], double(typename E::C(static_cast<const T *>(base)[lane])));
    return join<P>(a[0], a[1]);
}


template <int P, bool kStream, class L>
__device__ __forceinline__ double grid_norm(const L &l) {
    double acc = 0.0;
    walk<kStream>(l.u, [&](const Piece &p) {
        by_type(p.type, [&](auto e) { acc = piece_norm<P, kStream>(e, l.x(p.t), p, acc); });
    });
    return block_join<P, kWaves>(acc);
}
template <int P, class L>
__device__ __forceinline__ double small_norm(const L &l) {
    double acc = 0.0;
    shared_out(l.u, wave_of_block(), kSmallWaves, [&](const Piece &p) {
        by_type(p.type, [&](auto e) { acc = piece_norm<P, false>(e, l.x(p.t), p, acc); });
    });
    return block_join<P, kSmallWaves>(acc);
}

template <int P, bool kStream, class L>
__global__ __launch_bounds__(kThreads) void norm_partials(const L l, double *part) {
    const double acc = grid_norm<P, kStream>(l);
    if (threadIdx.x == 0) part[blockIdx.x] = acc;
}

template <int P> __device__ __forceinline__ double root_of(double acc) { return P == MBRL_NORM_TWO ? sqrt(acc) : acc; }

// What clipping multiplies with.  A norm that is not a number makes it NaN (the comparisons are false), an infinite one 0, unless
// the bound is infinite too: every number is within that.
__device__ __forceinline__ double factor_of(double norm, double max_norm) {
    if (max_norm == HUGE_VAL && norm <= max_norm) return 1.0;
    const double c = max_norm / (norm + 1e-6);
    return c > 1.0 ? 1.0 : c;
}

// The partial sums in their order.
template <int P>
__device__ __forceinline__ double join_partials(const double *part, int parts) {
    if (parts == 1) return part[0];
    double acc = 0.0;
    for (int i = threadIdx.x; i < parts; i += 4 * kThreads) {        // four on their way at once: other dies wrote them, it is far
        double x[4];
#pragma unroll
        for (int k = 0; k < 4; k++) x[k] = i + k * kThreads < parts ? part[i + k * kThreads] : 0.0;
#pragma unroll
        for (int k = 0; k < 4; k++) acc = join<P>(acc, x[k]);
    }
    return block_join<P, kWaves>(acc);
}

template <int P>
__global__ __launch_bounds__(kThreads) void norm_finish(const double *part, int parts, double *total, double *norm) {
    const double acc = join_partials<P>(part, parts);
    if (threadIdx.x == 0) {
        *total = acc;
        *norm = root_of<P>(acc);
    }
}

// ---- clip ----
// Multiplies by the clipping factor in the type that the values are computed with: float32 for all but float64 ones, so the
// factor is rounded (2^-24) and so is the product.  A factor below float32's normal range would lose digits: it is taken in
// two, the second a power of 2.  2^-64 keeps the first one normal down to 2^-190; below that 2^-149 does to 2^-275, where a product
// with the largest value is at most 4 steps of subnormal ones, and the first product cannot overflow (2^-41 2^128).
template <class C> struct Factor {
    C first, second;
    explicit __device__ __forceinline__ Factor(double c) {
        const bool tiny = sizeof(C) == 4 && c < 0x1p-126, least = c < 0x1p-190;
        first = C(tiny ? c * (least ? 0x1p149 : 0x1p64) : c);
        second = C(tiny ? (least ? 0x1p-149 : 0x1p-64) : 1.0);
    }
    __device__ __forceinline__ C operator()(C x) const { return x * first * second; }
};

template <bool kStream, class E>
__device__ __forceinline__ void piece_scale(E, void *base, const Piece &p, double c) {
    using T = typename E::T;
    constexpr int V = E::V, kStep = kWave * V;
    T *x = static_cast<T *>(base) + p.first;
    const Factor<typename E::C> f(c);
    const int lane = threadIdx.x % kWave, n = p.n;
    int i = lane * V;
    for (; i + 3 * kStep + V <= n; i += 4 * kStep) {
        Pack<T, V> r[4];
#pragma unroll
        for (int k = 0; k < 4; k++) r[k] = load<kStream, V>(x + i + k * kStep);
#pragma unroll
        for (int k = 0; k < 4; k++) {
#pragma unroll
            for (int j = 0; j < V; j++) r[k].v[j] = T(f(r[k].v[j]));
            store<kStream, V>(x + i + k * kStep, r[k]);
        }
    }
    for (; i + V <= n; i += kStep) {
        Pack<T, V> r = load<kStream, V>(x + i);
#pragma unroll
        for (int j = 0; j < V; j++) r.v[j] = T(f(r.v[j]));
        store<kStream, V>(x + i, r);
    }
    const int tail = n / V * V + lane;
    if (tail < n) x[tail] = T(f(x[tail]));
    if (lane < p.head) x[lane - p.first] = T(f(x[lane - p.first]));
}

// Every block of a middle list joins the partial sums for itself: 0.5 us instead of a launch between.  x * 1 is x: a factor of
// 1 leaves nothing to read or write.
template <int P, bool kStream, class L>
__global__ __launch_bounds__(kThreads) void clip_scale(const L l, const double *part, int parts, double max_norm, double *norm) {
    const double s = root_of<P>(join_partials<P>(part, parts)), c = factor_of(s, max_norm);
    if (blockIdx.x == 0 && threadIdx.x == 0) *norm = s;
    if (c == 1.0) return;
    walk<kStream>(l.u, [&](const Piece &p) {
        by_type(p.type, [&](auto e) { piece_scale<kStream>(e, l.x(p.t), p, c); });
    });
}

// A small list in one launch of one block.
template <int P, bool kClip, class L>
__global__ __launch_bounds__(kSmallThreads) void norm_small(const L l, double max_norm, double *norm) {
    const double s = root_of<P>(small_norm<P>(l));
    if (threadIdx.x == 0) *norm = s;
    if constexpr (kClip) {
        const double c = factor_of(s, max_norm);
        if (c == 1.0) return;
        shared_out(l.u, wave_of_block(), kSmallWaves, [&](const Piece &p) {
            by_type(p.type, [&](auto e) { piece_scale<false>(e, l.x(p.t), p, c); });
        });
    }
}

// ---- Adam ----
// up: a power of 2 that root, eps and with them the denominator are multiplied by, and size for it, so that an eps beyond the
// ends of float32 counts there, and the quotient of a small one does not overflow before it is multiplied (scale_of()).
struct Betas { double b1, b2, log_b1, log_b2, eps, up; };

// Counts a tensor's step and turns it into what the update multiplies with, in float64.
__device__ __forceinline__ Scalars count_step(float *count, double lr, double wd, const Betas &b, int decoupled) {
    const float step = *count + 1.0f;
    *count = step;
    const double t = step;
    Scalars s;
    s.size = b.up * lr / -expm1(t * b.log_b1);        // 1 - b^t without the cancellation
    s.root = b.up / sqrt(-expm1(t * b.log_b2));
    s.keep = decoupled ? 1.0 - lr * wd : 1.0;
    s.l2 = decoupled ? 0.0 : wd;
    return s;
}

// In float32 (float64 for float64 tensors); the state is float32 or wider, and a 16-bit parameter is rounded once, on
// its way back.  Root and quotient are correctly rounded for every list, so that a tensor's new values do not hang on what else is
// in its list, and hold where the parameter is near 0 and the update is the result.  The hardware's own, each within a step
// instead of half a one, are 7 instructions for 25; where one block does the update, or data come from the cache, it waits for
// them (float32, device time: 8e3 values 6.2 us for 5.2, 24e3 5.5 for 5.1, 5e5 6.2 for 5.9, 8e6 40 for 39; nothing beyond the cache).
template <class C> struct Update {
    C b1, a1, b2, a2, eps, size, scale, keep, l2;
    Factor<C> clip;
    __device__ __forceinline__ C operator()(C x, C g, C &m, C &v) const {
        g = clip(g);
        if (l2 != C(0)) g = fma(l2, x, g);        // not 0 * x, which an infinite x makes NaN
        m = fma(b1, m, a1 * g);
        v = fma(b2, v, a2 * g * g);
        return fma(-size, m / fma(C(sqrt(v)), scale, eps), x * keep);
    }
};

template <bool kStream, class E, class L>
__device__ __forceinline__ void piece_adam(E, const L &l, const Piece &q, const Betas &b, const Scalars &s, double clip) {
    using T = typename E::T;
    using C = typename E::C;
    constexpr int V = sizeof(C) == 8 ? 2 : 4, kStep = kWave * V;
    T *p = static_cast<T *>(l.template get<1>(q.t)) + q.first;
    const T *g = static_cast<const T *>(l.x(q.t)) + q.first;
    C *m = static_cast<C *>(l.template get<2>(q.t)) + q.first, *v = static_cast<C *>(l.template get<3>(q.t)) + q.first;
    const Update<C> f{C(b.b1), C(1.0 - b.b1), C(b.b2), C(1.0 - b.b2), C(b.eps), C(s.size), C(s.root), C(s.keep), C(s.l2), Factor<C>(clip)};
    const int lane = threadIdx.x % kWave, n = q.n;
    auto some = [&](int i, auto count) {        // `count` vectors a lane, all on their way at once
        constexpr int N = count;
        Pack<T, V> rp[N], rg[N];
        Pack<C, V> rm[N], rv[N];
#pragma unroll
        for (int k = 0; k < N; k++) {
            rg[k] = load<kStream, V>(g + i + k * kStep);
            rm[k] = load<kStream, V>(m + i + k * kStep);
            rv[k] = load<kStream, V>(v + i + k * kStep);
            rp[k] = load<kStream, V>(p + i + k * kStep);
        }
#pragma unroll
        for (int k = 0; k < N; k++) {
#pragma unroll
            for (int j = 0; j < V; j++) rp[k].v[j] = T(f(C(rp[k].v[j]), C(rg[k].v[j]), rm[k].v[j], rv[k].v[j]));
            store<kStream, V>(m + i + k * kStep, rm[k]);
            store<kStream, V>(v + i + k * kStep, rv[k]);
            store<kStream, V>(p + i + k * kStep, rp[k]);
        }
    };
    int i = lane * V;
    if constexpr (!kStream)        // where units have one vector a lane, two at once would only take registers, and with them waves
        for (; i + kStep + V <= n; i += 2 * kStep) some(i, std::integral_constant<int, 2>{});
    for (; i + V <= n; i += kStep) some(i, std::integral_constant<int, 1>{});
    auto one = [&](int64_t i) { p[i] = T(f(C(p[i]), C(g[i]), m[i], v[i])); };
    const int tail = n / V * V + lane;
    if (tail < n) one(tail);
    if (lane < q.head) one(lane - q.first);
}

constexpr int kNoClip = -1;        // P of an update that does not clip

// First launch of a step: the steps are counted (every block of the update needs what follows from them, so it cannot be
// done there), and the gradients' partial sums made if they are to be clipped.
template <int P, bool kStream, class L>
__global__ __launch_bounds__(kThreads) void adam_begin(const L l, const Betas b, int decoupled, Scalars *scalars, double *part) {
    if (blockIdx.x == 0)
        for (int i = threadIdx.x; i < l.u.count; i += kThreads) scalars[i] = count_step(l.step[i], l.lr[i], l.wd[i], b, decoupled);
    if constexpr (P != kNoClip) {
        const double acc = grid_norm<P, kStream>(l);
        if (threadIdx.x == 0) part[blockIdx.x] = acc;
    }
}

// For lists too long for that: the steps apart, the norm as of any list.
__global__ __launch_bounds__(kThreads) void adam_count(const CountList l, const Betas b, int decoupled, Scalars *scalars) {
    const int i = blockIdx.x * kThreads + threadIdx.x;
    if (i >= l.count) return;
    const int k = l.rate[i];
    scalars[i] = count_step(static_cast<float *>(address(l.lo[i], l.hi[i])), l.lr[k], l.wd[k], b, decoupled);
}

// Streaming: 7 waves a SIMD, by the compiler's own choice or not (kAdamShift; two registers too many leave 6: bfloat16, 268e6 values
// clipped: 1.03 ms for 1.01).
template <int P, bool kStream, class L>
__global__ __launch_bounds__(kThreads, kStream ? 7 : 1) void adam_update(const L l, const Betas b, const Scalars *scalars, const double *part, int parts,
                                                        double max_norm, double *norm) {
    double clip = 1.0;
    if constexpr (P != kNoClip) {
        const double s = root_of<P>(join_partials<P>(part, parts));
        if (blockIdx.x == 0 && threadIdx.x == 0) *norm = s;
        clip = factor_of(s, max_norm);
    }
    dealt(l.u, wave_of_grid(), waves_of_grid(), [&](const Piece &q) {
        by_type(q.type, [&](auto e) { piece_adam<kStream>(e, l, q, b, scalars[q.t], clip); });
    });
}

template <int P, class L>
__global__ __launch_bounds__(kSmallThreads) void adam_small(const L a, const Betas b, int decoupled, double max_norm, double *norm) {
    __shared__ Scalars scalars[decltype(a.l.u)::K];
    static_assert(decltype(a.l.u)::K <= kWave, "one thread of one wave a tensor");
    const int i = int(threadIdx.x) - (kSmallThreads - kWave);        // the last wave: where there is little to do, it has nothing else
    if (i >= 0 && i < a.l.u.count) scalars[i] = count_step(a.step[i], a.lr[i], a.wd[i], b, decoupled);
    double clip = 1.0;
    if constexpr (P != kNoClip) {
        const double s = root_of<P>(small_norm<P>(a.l));
        if (threadIdx.x == 0) *norm = s;
        clip = factor_of(s, max_norm);
    }
    __syncthreads();
    shared_out(a.l.u, wave_of_block(), kSmallWaves, [&](const Piece &q) {
        by_type(q.type, [&](auto e) { piece_adam<false>(e, a.l, q, b, scalars[q.t], clip); });
    });
}

// ---- host ----
const int kSize[4] = {8, 4, 2, 2};

// Units small enough to fill the blocks that stay, and large enough that finding a unit's tensor does not count.
int unit_shift(int64_t values) {
    int shift = kMinShift;
    while (shift < kMaxShift && (values >> shift) > 4 * kMaxBlocks * kWaves) shift++;
    return shift;
}

int64_t total(int64_t count, const int64_t *numel) {
    int64_t n = 0;
    for (int64_t i = 0; i < count; i++) n += numel[i];
    return n;
}

int64_t total_bytes(int64_t count, const int64_t *numel, const int *dtype) {
    int64_t n = 0;
    for (int64_t i = 0; i < count; i++) n += numel[i] * kSize[dtype[i]];
    return n;
}

int64_t adam_bytes(int64_t count, const int64_t *numel, const int *dtype) {        // of all four tensors
    int64_t n = 0;
    for (int64_t i = 0; i < count; i++) n += numel[i] * (kSize[dtype[i]] == 8 ? 32 : 8 + 2 * kSize[dtype[i]]);
    return n;
}

// Puts tensors `from` to `to` of a call into a list: fill(place, tensor).  Empty ones have a place and no units.  Units begin at
// the tensor's first value (head(i) of 0, for sums), or behind its first head(i) values, at a cache line.
template <class List, class Head, class Fill>
void fill_list(List &l, int64_t from, int64_t to, const int64_t *numel, const int *dtype, int shift, Head head, Fill fill) {
    uint32_t units = 0;
    for (int64_t i = from; i < to; i++) {
        const int at = int(i - from);
        const int64_t h = std::min<int64_t>(numel[i], head(i));
        if (numel[i]) units += uint32_t(std::max<int64_t>((numel[i] - h + (int64_t(1) << shift) - 1) >> shift, 1));
        l.u.end[at] = units;
        l.u.put(at, numel[i], dtype[i], h);
        fill(at, i);
    }
    l.u.count = int(to - from);
    l.u.shift = shift;
    l.u.units = units;
}
// Values of `size` bytes before the first cache line that begins in a tensor.  What is written is aligned to them: 402 tensors of
// a bucket, which begin anywhere, are updated in 261 us for 281 us from their first values on.
int64_t before_line(const void *p, int64_t size) { return int64_t(-uintptr_t(p) & 127) / size; }
int64_t from_first(int64_t) { return 0; }

template <class U> int grid_of(const U &u, int most = kMaxBlocks, int each = 1) {
    return int(std::min<int64_t>((int64_t(u.units) + kWaves * each - 1) / (kWaves * each), most));
}

template <class F>
void by_norm(int kind, F &&f) {
    if (kind == MBRL_NORM_TWO) f(std::integral_constant<int, MBRL_NORM_TWO>{});
    else if (kind == MBRL_NORM_ONE) f(std::integral_constant<int, MBRL_NORM_ONE>{});
    else if (kind == MBRL_NORM_INF) f(std::integral_constant<int, MBRL_NORM_INF>{});
    else f(std::integral_constant<int, kNoClip>{});
}

// A float32 denominator lies between eps and the largest root, 2^64, times its scale, at most 2^27: 2^32 more does not overflow.
// An eps under float32's subnormal values counts from 2^-181 on.
double scale_of(double eps) { return eps > 0.0 && eps < 0x1p-126 ? 0x1p32 : eps >= 0x1p64 ? 0x1p-64 : 1.0; }

constexpr int64_t kMaxValues = int64_t(1) << 37;        // of a call: units are counted in 32 bits

int check_list(const char *what, int64_t count, const int64_t *numel, const int *dtype) {
    static thread_local char text[160];
    auto bad = [&](int code, const char *why) { snprintf(text, sizeof text, "%s: %s", what, why); return report(code, text); };
    if (count < 0 || count > (int64_t(1) << 24)) return bad(-6, "the number of tensors is out of range");
    if (count && (!numel || !dtype)) return bad(-1, "null argument");
    int64_t n = 0;
    for (int64_t i = 0; i < count; i++) {
        if (numel[i] < 0 || numel[i] > kMaxValues || (n += numel[i]) > kMaxValues) return bad(-6, "a number of values is out of range");
        if (dtype[i] < 0 || dtype[i] > 3) return bad(-7, "unknown element type");
    }
    return 0;
}

// Whether a list can hold the address of a tensor with values.
bool usable(const void *p) { return p && !(uintptr_t(p) >> 48); }

// Memory that is written must not be any other memory of the call.
struct Ranges {
    struct Range { uintptr_t lo, hi; bool written; };
    std::vector<Range> r;
    std::vector<size_t> lists;        // where each list ends
    void add(const void *p, int64_t bytes, bool written) {
        if (bytes) r.push_back({uintptr_t(p), uintptr_t(p) + uintptr_t(bytes), written});
    }
    void close() { lists.push_back(r.size()); }
    bool disjoint() const {
        uintptr_t read_end = 0, write_end = 0;
        auto next = [&](const Range &x) {
            if (x.lo < write_end || (x.written && x.lo < read_end)) return false;
            uintptr_t &end = x.written ? write_end : read_end;
            end = std::max(end, x.hi);
            return true;
        };
        // Addresses have 48 bits: with the place behind them they are sorted as plain numbers, four times as fast as the ranges
        // themselves.  Lists mostly lie in order, or nearly so, and are only merged then (402 tensors and their four others: 1
        // to 5 us for 14 to 20, which a step would wait for).
        std::vector<uint64_t> order(r.size());
        const bool packed = r.size() <= 0x10000;
        for (size_t i = 0; i < r.size(); i++) order[i] = packed ? uint64_t(r[i].lo) << 16 | i : i;
        const auto begin = order.begin();
        if (packed) {
            size_t from = 0;
            for (size_t to : lists) {
                if (!std::is_sorted(begin + from, begin + to)) std::sort(begin + from, begin + to);
                if (from && from < to && order[from] < order[from - 1]) std::inplace_merge(begin, begin + from, begin + to);
                from = to;
            }
        } else
            std::sort(begin, order.end(), [&](uint64_t a, uint64_t b) { return r[a].lo < r[b].lo; });
        for (uint64_t i : order)
            if (!next(r[packed ? i & 0xffff : i])) return false;
        return true;
    }
};

int launched(const char *what) {
    const hipError_t e = hipGetLastError();
    if (e == hipSuccess) return 0;
    static thread_local char text[160];
    snprintf(text, sizeof text, "%s: launch failed (hip error %d)", what, int(e));
    return report(-10, text);
}

// Whether one block takes a list on alone.
bool small(int op, int64_t count, const int64_t *numel, const int *dtype) {
    if (op == MBRL_OP_ADAM) return count <= kSmallAdamCount && adam_bytes(count, numel, dtype) <= kSmallAdam;
    const bool clip = op == MBRL_OP_CLIP;
    return count <= (clip ? kSmallClipCount : kSmallNormCount) && total_bytes(count, numel, dtype) <= (clip ? kSmallClip : kSmallNorm);
}

// Workspace of the others: [total, unused][partial sums][Scalars of each tensor]
int64_t partials(int64_t count) { return (count + kNormList - 1) / kNormList * kMaxBlocks; }
struct Space {
    double *total, *part;
    Scalars *scalars;
    Space(void *p, int64_t count) {
        total = static_cast<double *>(p);
        part = total + 2;
        scalars = reinterpret_cast<Scalars *>(part + partials(count));
    }
    static int64_t bytes(int op, int64_t count, const int64_t *numel, const int *dtype) {
        return small(op, count, numel, dtype) ? 0 : 16 + 8 * partials(count) + int64_t(sizeof(Scalars)) * count;
    }
};

// The gradients of a call.
struct Gradients {
    int64_t count, values, bytes;
    void *const *x;
    const int64_t *numel;
    const int *dtype;
    Gradients(int64_t count_, void *const *xs, const int64_t *ns, const int *types)
        : count(count_), values(total(count_, ns)), bytes(total_bytes(count_, ns, types)), x(xs), numel(ns), dtype(types) {}

    template <class L, class Head, class Go> void lists(L &l, int shift, Head head, Go go) const {
        constexpr int K = decltype(l.u)::K;
        l.u.count = l.u.units = 0;
        for (int64_t i = 0; i < count; i += K) {
            fill_list(l, i, std::min<int64_t>(count, i + K), numel, dtype, shift, head, [&](int at, int64_t k) { l.put(at, x[k]); });
            go();
        }
    }
};

// For scaling it is all one where a tensor ends: neighbours in memory of one type become one, and a bucket of many tensors takes
// one launch instead of one for each kNormList.  Not for sums, whose order, and with it their last bit, must not hang on
// where tensors lie: every rank of a sharded run clips by the same factor.
struct Runs : Gradients {
    std::vector<void *> x_;
    std::vector<int64_t> numel_;
    std::vector<int> dtype_;
    explicit Runs(const Gradients &g) : Gradients(g) {
        auto follows = [&](int64_t i) {
            return g.dtype[i] == g.dtype[i - 1] && g.numel[i - 1] && static_cast<char *>(g.x[i - 1]) + g.numel[i - 1] * kSize[g.dtype[i]] == g.x[i];
        };
        int64_t runs = count ? 1 : 0;
        for (int64_t i = 1; i < count; i++) runs += !follows(i);
        if (runs == count) return;
        x_.reserve(runs), numel_.reserve(runs), dtype_.reserve(runs);
        for (int64_t i = 0; i < count; i++) {
            if (i && follows(i)) {
                numel_.back() += g.numel[i];
                continue;
            }
            x_.push_back(g.x[i]), numel_.push_back(g.numel[i]), dtype_.push_back(g.dtype[i]);
        }
        count = runs;
        x = x_.data(), numel = numel_.data(), dtype = dtype_.data();
    }
    Runs(const Runs &) = delete;
};

// Calls f(the flag as a constant).
template <class F> void by_flag(bool flag, F &&f) { flag ? f(std::true_type{}) : f(std::false_type{}); }
// Calls f(a list of the smallest size).
template <template <int> class List, int K, class F>
void by_count(int64_t count, F &&f) {
    if (count <= kFew) f(List<kFew>{});
    else f(List<K>{});
}

// Joins the partial sums in a launch of its own where `finish` says so, they are too many for every block of the next launch, or
// there are none (all tensors are empty: the next launch may have no block that would write the norm).
struct Parts { const double *part; int parts; };
template <int P>
Parts launch_finish(int parts, bool finish, const Space &ws, double *norm, hipStream_t st) {
    if (!finish && parts && parts <= kMaxParts) return {ws.part, parts};
    hipLaunchKernelGGL((norm_finish<P>), dim3(1), dim3(kThreads), 0, st, ws.part, parts, ws.total, norm);
    return {ws.total, 1};
}

// Launches the partial sums of a list.
template <int P>
Parts launch_partials(const Gradients &g, bool stream, bool finish, const Space &ws, double *norm, hipStream_t st) {
    int parts = 0;
    by_flag(stream, [&](auto stream_) {
        constexpr bool kStream = stream_;
        by_count<NormList, kNormList>(g.count, [&](auto l) {
            g.lists(l, unit_shift(g.values), from_first, [&] {
                if (const int grid = grid_of(l.u, kMaxBlocks, kStream ? 1 : kUnits)) {
                    hipLaunchKernelGGL((norm_partials<P, kStream, decltype(l)>), dim3(grid), dim3(kThreads), 0, st, l, ws.part + parts);
                    parts += grid;
                }
            });
        });
    });
    return launch_finish<P>(parts, finish, ws, norm, st);
}

// The norm of a list, and the scaling where kClip.
template <bool kClip>
void launch_norm(int kind, const Gradients &g, const Space &ws, double max_norm, double *norm, hipStream_t st) {
    by_norm(kind, [&](auto P_) {
        constexpr int P = P_;
        if constexpr (P != kNoClip) {
            if (small(kClip ? MBRL_OP_CLIP : MBRL_OP_NORM, g.count, g.numel, g.dtype)) {
                by_count<SmallNorm, kSmallNormCount>(g.count, [&](auto l) {
                    g.lists(l, kSmallShift, from_first, [] {});
                    hipLaunchKernelGGL((norm_small<P, kClip, decltype(l)>), dim3(1), dim3(kSmallThreads), 0, st, l, max_norm, norm);
                });
                return;
            }
            const bool stream = g.bytes > kCache / 4;
            const Parts sum = launch_partials<P>(g, g.bytes > kCache / 2, !kClip || stream, ws, norm, st);
            if constexpr (kClip) {
                const Runs runs(g);
                auto head = [&](int64_t i) { return before_line(runs.x[i], kSize[runs.dtype[i]]); };
                by_flag(stream, [&](auto stream_) {
                    constexpr bool kStream = stream_;
                    by_count<NormList, kNormList>(runs.count, [&](auto l) {
                        runs.lists(l, !kStream ? unit_shift(g.values) : g.bytes == 2 * g.values ? kScaleShift16 : kScaleShift, head, [&] {
                            if (const int grid = grid_of(l.u, kStream ? kStreamBlocks : kMaxBlocks, kUnits))
                                hipLaunchKernelGGL((clip_scale<P, kStream, decltype(l)>), dim3(grid), dim3(kThreads), 0, st, l, sum.part, sum.parts,
                                                   max_norm, norm);
                        });
                    });
                });
            }
        }
    });
}

template <class F>
int guarded(const char *what, F &&f) {
    try {
        return f();
    } catch (const std::bad_alloc &) {
        return report(-5, "out of host memory");
    } catch (...) {
        return report(-10, what);
    }
}
}  // namespace

extern "C" {

int64_t mbrl_optim_workspace_bytes(int op, int64_t count, const int64_t *numel, const int *dtype) {
    if (int rc = check_list("mbrl_optim_workspace_bytes", count, numel, dtype)) return rc;
    if (op != MBRL_OP_NORM && op != MBRL_OP_CLIP && op != MBRL_OP_ADAM) return report(-7, "mbrl_optim_workspace_bytes: unknown operator");
    return Space::bytes(op, count, numel, dtype);
}

int mbrl_grad_norm(int64_t count, const void *const *grads, const int64_t *numel, const int *dtype, int norm_type, void *workspace,
                   int64_t workspace_bytes, double *norm, void *hip_stream) {
    return guarded("mbrl_grad_norm: failed", [&] {
        if (int rc = check_list("mbrl_grad_norm", count, numel, dtype)) return rc;
        if (norm_type < MBRL_NORM_INF || norm_type > MBRL_NORM_TWO) return report(-7, "mbrl_grad_norm: unknown norm type");
        const int64_t need = Space::bytes(MBRL_OP_NORM, count, numel, dtype);
        if (!norm || (need && !workspace) || (count && !grads)) return report(-1, "mbrl_grad_norm: null argument");
        if (workspace_bytes < need) return report(-8, "mbrl_grad_norm: workspace too small (mbrl_optim_workspace_bytes)");
        for (int64_t i = 0; i < count; i++)
            if (numel[i] && !usable(grads[i])) return report(-1, "mbrl_grad_norm: null tensor, or no device address");
        launch_norm<false>(norm_type, Gradients(count, const_cast<void *const *>(grads), numel, dtype), Space(workspace, count), 0.0, norm,
                           (hipStream_t)hip_stream);
        return launched("mbrl_grad_norm");
    });
}

int mbrl_clip_grad_norm(int64_t count, void *const *grads, const int64_t *numel, const int *dtype, int norm_type, double max_norm,
                        void *workspace, int64_t workspace_bytes, double *norm, void *hip_stream) {
    return guarded("mbrl_clip_grad_norm: failed", [&] {
        if (int rc = check_list("mbrl_clip_grad_norm", count, numel, dtype)) return rc;
        if (norm_type < MBRL_NORM_INF || norm_type > MBRL_NORM_TWO) return report(-7, "mbrl_clip_grad_norm: unknown norm type");
        if (!(max_norm >= 0.0)) return report(-7, "mbrl_clip_grad_norm: max_norm must not be negative");
        const int64_t need = Space::bytes(MBRL_OP_CLIP, count, numel, dtype);
        if (!norm || (need && !workspace) || (count && !grads)) return report(-1, "mbrl_clip_grad_norm: null argument");
        if (workspace_bytes < need) return report(-8, "mbrl_clip_grad_norm: workspace too small (mbrl_optim_workspace_bytes)");
        Ranges r;
        r.r.reserve(count);
        for (int64_t i = 0; i < count; i++) {
            if (numel[i] && !usable(grads[i])) return report(-1, "mbrl_clip_grad_norm: null tensor, or no device address");
            r.add(grads[i], numel[i] * kSize[dtype[i]], true);
        }
        r.close();
        if (!r.disjoint()) return report(-7, "mbrl_clip_grad_norm: two of the tensors share memory");
        launch_norm<true>(norm_type, Gradients(count, grads, numel, dtype), Space(workspace, count), max_norm, norm, (hipStream_t)hip_stream);
        return launched("mbrl_clip_grad_norm");
    });
}

int mbrl_adam_step(int64_t count, void *const *params, const void *const *grads, void *const *exp_avgs, void *const *exp_avg_sqs,
                   float *const *steps, const int64_t *numel, const int *dtype, const double *lr, const double *weight_decay,
                   double beta_one, double beta_two, double eps, int decoupled, int norm_type, double max_norm, void *workspace,
                   int64_t workspace_bytes, double *norm, void *hip_stream) {
    return guarded("mbrl_adam_step: failed", [&] {
        if (int rc = check_list("mbrl_adam_step", count, numel, dtype)) return rc;
        const bool clip = norm != nullptr;
        if (clip && (norm_type < MBRL_NORM_INF || norm_type > MBRL_NORM_TWO)) return report(-7, "mbrl_adam_step: unknown norm type");
        if (clip && !(max_norm >= 0.0)) return report(-7, "mbrl_adam_step: max_norm must not be negative");
        if (!(beta_one >= 0.0 && beta_one < 1.0 && beta_two >= 0.0 && beta_two < 1.0)) return report(-7, "mbrl_adam_step: betas must be in [0, 1)");
        if (!(eps >= 0.0)) return report(-7, "mbrl_adam_step: eps must not be negative");
        const int64_t need = Space::bytes(MBRL_OP_ADAM, count, numel, dtype);
        if ((need && !workspace) || (count && (!params || !grads || !exp_avgs || !exp_avg_sqs || !steps || !lr || !weight_decay)))
            return report(-1, "mbrl_adam_step: null argument");
        if (workspace_bytes < need) return report(-8, "mbrl_adam_step: workspace too small (mbrl_optim_workspace_bytes)");
        for (int64_t i = 0; i < count; i++)
            if (!usable(steps[i]) || (numel[i] && !(usable(params[i]) && usable(grads[i]) && usable(exp_avgs[i]) && usable(exp_avg_sqs[i]))))
                return report(-1, "mbrl_adam_step: null tensor, or no device address");
        Ranges r;
        r.r.reserve(5 * count);
        auto add = [&](auto x, bool written, auto bytes) {
            for (int64_t i = 0; i < count; i++) r.add(x[i], bytes(i), written);
            r.close();
        };
        auto own = [&](int64_t i) { return numel[i] * kSize[dtype[i]]; };
        auto wide = [&](int64_t i) { return numel[i] * (kSize[dtype[i]] == 8 ? 8 : 4); };
        add(params, true, own);
        add(grads, false, own);
        add(exp_avgs, true, wide);
        add(exp_avg_sqs, true, wide);
        add(steps, true, [](int64_t) { return 4; });
        if (!r.disjoint()) return report(-7, "mbrl_adam_step: a tensor that is written shares memory with another one");
        const hipStream_t st = (hipStream_t)hip_stream;
        const Space ws(workspace, count);
        const double up = scale_of(eps);
        const Betas b{beta_one, beta_two, std::log1p(beta_one - 1.0), std::log1p(beta_two - 1.0), up * eps, up};        // b - 1 is exact from 0.5 on
        const int64_t values = total(count, numel);
        const int64_t bytes = adam_bytes(count, numel, dtype);
        auto lists = [&](auto &l, int shift, auto head, auto fill, auto go) {
            constexpr int K = std::decay_t<decltype(l.u)>::K;
            l.u.count = l.u.units = 0;
            for (int64_t i = 0; i < count; i += K) {
                fill_list(l, i, std::min<int64_t>(count, i + K), numel, dtype, shift, head, fill);
                go(i);
            }
        };
        auto tensors = [&](auto &l) { return [&](int at, int64_t k) { l.put(at, grads[k], params[k], exp_avgs[k], exp_avg_sqs[k]); }; };
        auto counters = [&](auto &l) { return [&](int at, int64_t k) { l.step[at] = steps[k]; l.lr[at] = lr[k]; l.wd[at] = weight_decay[k]; }; };
        by_norm(clip ? norm_type : kNoClip, [&](auto P_) {
            constexpr int P = P_;
            constexpr bool kClip = P != kNoClip;
            if (small(MBRL_OP_ADAM, count, numel, dtype)) {
                by_count<SmallAdam, kSmallAdamCount>(count, [&](auto l) {
                    lists(l.l, kSmallShift, from_first, [&](int at, int64_t k) { tensors(l.l)(at, k); counters(l)(at, k); }, [](int64_t) {});
                    hipLaunchKernelGGL((adam_small<P, decltype(l)>), dim3(1), dim3(kSmallThreads), 0, st, l, b, decoupled, max_norm, norm);
                });
                return;
            }
            const bool stream = bytes > kCache / 4;
            const int shift = unit_shift(values);
            auto head = [&](int64_t i) { return before_line(exp_avgs[i], kSize[dtype[i]] == 8 ? 8 : 4); };
            Parts sum{nullptr, 0};
            if (count <= kBeginList) {
                by_flag(kClip && total_bytes(count, numel, dtype) > kCache, [&](auto stream_) {
                    constexpr bool kStream = kClip && stream_;
                    by_count<BeginList, kBeginList>(count, [&](auto l) {
                        lists(l, shift, from_first, [&](int at, int64_t k) { l.put(at, grads[k]); counters(l)(at, k); }, [&](int64_t) {
                            const int grid = kClip ? std::max(grid_of(l.u), 1) : 1;
                            hipLaunchKernelGGL((adam_begin<P, kStream, decltype(l)>), dim3(grid), dim3(kThreads), 0, st, l, b, decoupled,
                                               ws.scalars, ws.part);
                            if constexpr (kClip) sum = launch_finish<P>(grid, stream, ws, norm, st);
                        });
                    });
                });
            } else {
                CountList l;
                for (int64_t i = 0, from = 0; from < count; from = i) {
                    l.count = l.rates = 0;
                    while (i < count && l.put(steps[i], lr[i], weight_decay[i])) i++;
                    hipLaunchKernelGGL(adam_count, dim3((l.count + kThreads - 1) / kThreads), dim3(kThreads), 0, st, l, b, decoupled, ws.scalars + from);
                }
                if constexpr (kClip) {
                    const Gradients g(count, const_cast<void *const *>(grads), numel, dtype);
                    sum = launch_partials<P>(g, g.bytes > kCache, stream, ws, norm, st);
                }
            }
            by_flag(stream, [&](auto stream_) {
                constexpr bool kStream = stream_;
                by_count<UpdateList, kAdamList>(count, [&](auto l) {
                    lists(l, !kStream ? shift : bytes == 32 * values ? kAdamShift64 : kAdamShift, head, tensors(l), [&](int64_t i) {
                        if (const int grid = std::max(grid_of(l.u, kStream ? kStreamBlocks : kMaxBlocks), kClip && i == 0 ? 1 : 0))        // one block at least writes the norm
                            hipLaunchKernelGGL((adam_update<P, kStream, decltype(l)>), dim3(grid), dim3(kThreads), 0, st, l, b, ws.scalars + i,
                                               sum.part, sum.parts, max_norm, norm);
                    });
                });
            });
        });
        return launched("mbrl_adam_step");
    });
}

}  // extern "C"
