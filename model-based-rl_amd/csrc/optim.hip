// Optimiser-step operators over lists of tensors: the global gradient norm, clipping by it, and the Adam update that takes
// the clipped gradient (C ABI: include/mbrl.h).
//
// Mathematics, over the values x of all tensors of a list:
//   norm   s = (sum |x|^p)^(1/p), p = 1, 2 or infinity
//   clip   x <- c x,  c = min(1, max_norm / (s + 1e-6))
//   Adam   g <- c g (+ wd x)          m <- b1 m + (1 - b1) g      v <- b2 v + (1 - b2) g^2
//          x <- x (1 - lr wd) - lr / (1 - b1^t)  m / (sqrt(v / (1 - b2^t)) + eps)
//
// Layout.  Every tensor is cut into units of 2^shift values, a unit belongs to one wave, and the units of the whole list
// are dealt out to the waves of a launch in turn.  The list travels in the kernel arguments (at most 4 KB), so a call
// uploads nothing, can be captured into a graph, and keeps nothing of one call for the next; a longer list takes several
// launches.  A wave finds its unit's tensor by comparing 64 unit ends at once (owner()).  Sums are float64 in every
// case: squares of float32 and bfloat16 values cannot overflow there, and each partial sum has a fixed place and is
// added in a fixed order, so the norm does not depend on which wave is done first (no atomics).
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
constexpr int kMaxBlocks = 1024;          // of a launch: 4 blocks of 4 waves a CU
constexpr int kMinShift = 9, kMaxShift = 12;

// ---- element types: what is stored, what is computed with, values in 16 bytes ----
struct F64 { using T = double; using C = double; static constexpr int V = 2; };
struct F32 { using T = float; using C = float; static constexpr int V = 4; };
struct B16 { using T = __bf16; using C = float; static constexpr int V = 8; };
struct F16 { using T = _Float16; using C = float; static constexpr int V = 8; };

// Vectors with the alignment of their elements: a tensor may start at any element (a slice of a bucket), and the memory
// system takes a 16-byte access at any such address, so there is one path for all alignments.
template <class T, int V> struct Pack { T v[V]; };
template <class T, int V>
__device__ __forceinline__ Pack<T, V> load(const T *p) {
    Pack<T, V> r;
    __builtin_memcpy(&r, p, sizeof r);
    return r;
}
template <class T, int V>
__device__ __forceinline__ void store(T *p, const Pack<T, V> &r) { __builtin_memcpy(p, &r, sizeof r); }

// Calls f(integral_constant-like element type) for a stored type code; wave-uniform.
template <class F>
__device__ __forceinline__ void by_type(int code, F &&f) {
    if (code == MBRL_DT_FLOAT) f(F32{});
    else if (code == MBRL_DT_DOUBLE) f(F64{});
    else if (code == MBRL_DT_BFLOAT) f(B16{});
    else f(F16{});
}

// ---- lists in kernel arguments ----
template <int K> struct Units {
    uint64_t n[K];        // values << 2 | type code
    uint32_t end[K];      // units of the tensors up to and including this one
    int count, shift;
    uint32_t units;
};
constexpr int kNormList = 192, kAdamList = 80, kStepList = 160;
struct NormList { Units<kNormList> u; void *x[kNormList]; };
struct AdamList { Units<kAdamList> u; void *p[kAdamList]; const void *g[kAdamList]; void *m[kAdamList], *v[kAdamList]; uint32_t s[kAdamList]; };
struct StepList { float *step[kStepList]; double lr[kStepList], wd[kStepList]; int count; };
static_assert(sizeof(NormList) <= 3968 && sizeof(AdamList) <= 3968 && sizeof(StepList) <= 3968, "kernel arguments are 4 KB");

// What the update of one tensor multiplies with (adam_scalars).
struct Scalars { double size, root, keep, l2; };

__device__ __forceinline__ uint32_t wave_of_block() { return __builtin_amdgcn_readfirstlane(threadIdx.x / kWave); }

// The tensor that unit `unit` belongs to: as many as end at or before it come first.
template <int K>
__device__ __forceinline__ int owner(const Units<K> &u, uint32_t unit) {
    const int lane = threadIdx.x % kWave;
    int t = 0;
    for (int k = 0; k < u.count; k += kWave)
        t += __popcll(__ballot(k + lane < u.count && u.end[k + lane < u.count ? k + lane : 0] <= unit));
    return __builtin_amdgcn_readfirstlane(t);
}

// One unit of a list: its tensor, its first value and how many it has.
struct Piece { int t, type; int64_t first; int n; };
template <int K>
__device__ __forceinline__ Piece piece(const Units<K> &u, uint32_t unit) {
    Piece p;
    p.t = owner(u, unit);
    const uint64_t n = u.n[p.t];
    p.type = int(n & 3);
    p.first = int64_t(unit - (p.t ? u.end[p.t - 1] : 0)) << u.shift;
    const int64_t left = int64_t(n >> 2) - p.first;
    p.n = int(left < (int64_t(1) << u.shift) ? left : (int64_t(1) << u.shift));
    return p;
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

template <int P>
__device__ __forceinline__ double block_join(double a) {
    __shared__ double part[kWaves];
    for (int d = kWave / 2; d; d /= 2) a = join<P>(a, __shfl_xor(a, d));
    __syncthreads();
    if (threadIdx.x % kWave == 0) part[threadIdx.x / kWave] = a;
    __syncthreads();
    a = part[0];
    for (int w = 1; w < kWaves; w++) a = join<P>(a, part[w]);
    return a;
}

template <int P, class E>
__device__ __forceinline__ double unit_norm(E, const void *base, int64_t first, int n, double acc) {
    using T = typename E::T;
    constexpr int V = E::V, kStep = kWave * V;
    const T *x = static_cast<const T *>(base) + first;
    const int lane = threadIdx.x % kWave;
    int i = lane * V;
    double a[2] = {acc, 0.0};
    for (; i + 3 * kStep + V <= n; i += 4 * kStep) {
        Pack<T, V> r[4];
#pragma unroll
        for (int k = 0; k < 4; k++) r[k] = load<T, V>(x + i + k * kStep);
#pragma unroll
        for (int k = 0; k < 4; k++)
#pragma unroll
            for (int j = 0; j < V; j++) a[j % 2] = add<P>(a[j % 2], double(typename E::C(r[k].v[j])));
    }
    for (; i + V <= n; i += kStep) {
        const Pack<T, V> r = load<T, V>(x + i);
#pragma unroll
        for (int j = 0; j < V; j++) a[j % 2] = add<P>(a[j % 2], double(typename E::C(r.v[j])));
    }
    const int tail = n / V * V + lane;        // the last n % V values, one a lane
    if (tail < n) a[1] = add<P>(a[1], double(typename E::C(x[tail])));
    return join<P>(a[0], a[1]);
}

template <int P>
__global__ __launch_bounds__(kThreads) void norm_partials(const NormList l, double *part) {
    double acc = 0.0;
    for (uint32_t unit = blockIdx.x * kWaves + wave_of_block(); unit < l.u.units; unit += gridDim.x * kWaves) {
        const Piece p = piece(l.u, unit);
        by_type(p.type, [&](auto e) { acc = unit_norm<P>(e, l.x[p.t], p.first, p.n, acc); });
    }
    acc = block_join<P>(acc);
    if (threadIdx.x == 0) part[blockIdx.x] = acc;
}

// The partial sums in their order -> the norm, and the factor that clipping multiplies with.  A norm that is not a number
// makes the factor NaN (the comparison is false), an infinite one makes it 0.
template <int P>
__global__ __launch_bounds__(kThreads) void norm_finish(const double *part, int count, double max_norm, double *norm, double *factor) {
    double acc = 0.0;
    for (int i = threadIdx.x; i < count; i += kThreads) acc = join<P>(acc, part[i]);
    acc = block_join<P>(acc);
    if (threadIdx.x == 0) {
        const double s = P == MBRL_NORM_TWO ? sqrt(acc) : acc;
        *norm = s;
        if (factor) {
            const double c = max_norm / (s + 1e-6);
            *factor = c > 1.0 ? 1.0 : c;
        }
    }
}

// ---- clip ----
// float32 values are multiplied in float64 and rounded once; 16-bit ones in float32, whose rounding of the factor is
// 2^-16 of theirs.
template <class E>
__device__ __forceinline__ typename E::T scaled(typename E::T x, double c) {
    using C = std::conditional_t<sizeof(typename E::T) == 2, float, double>;
    return typename E::T(C(x) * C(c));
}

template <class E>
__device__ __forceinline__ void unit_scale(E, void *base, int64_t first, int n, double c) {
    using T = typename E::T;
    constexpr int V = E::V, kStep = kWave * V;
    T *x = static_cast<T *>(base) + first;
    const int lane = threadIdx.x % kWave;
    int i = lane * V;
    for (; i + 3 * kStep + V <= n; i += 4 * kStep) {
        Pack<T, V> r[4];
#pragma unroll
        for (int k = 0; k < 4; k++) r[k] = load<T, V>(x + i + k * kStep);
#pragma unroll
        for (int k = 0; k < 4; k++) {
#pragma unroll
            for (int j = 0; j < V; j++) r[k].v[j] = scaled<E>(r[k].v[j], c);
            store<T, V>(x + i + k * kStep, r[k]);
        }
    }
    for (; i + V <= n; i += kStep) {
        Pack<T, V> r = load<T, V>(x + i);
#pragma unroll
        for (int j = 0; j < V; j++) r.v[j] = scaled<E>(r.v[j], c);
        store<T, V>(x + i, r);
    }
    const int tail = n / V * V + lane;
    if (tail < n) x[tail] = scaled<E>(x[tail], c);
}

__global__ __launch_bounds__(kThreads) void clip_scale(const NormList l, const double *factor) {
    const double c = *factor;
    if (c == 1.0) return;          // x * 1 is x: nothing to read or write
    for (uint32_t unit = blockIdx.x * kWaves + wave_of_block(); unit < l.u.units; unit += gridDim.x * kWaves) {
        const Piece p = piece(l.u, unit);
        by_type(p.type, [&](auto e) { unit_scale(e, l.x[p.t], p.first, p.n, c); });
    }
}

// ---- Adam ----
// One thread a tensor: counts the step and turns it into what the update multiplies with, in float64.  A launch before the update, because every block of the update needs them.
__global__ void adam_scalars(const StepList l, double b1, double b2, int decoupled, Scalars *out) {
    const int i = threadIdx.x;
    if (i >= l.count) return;
    const float step = *l.step[i] + 1.0f;
    *l.step[i] = step;
    const double t = step;
    Scalars s;
    s.size = l.lr[i] / -expm1(t * log1p(b1 - 1.0));        // 1 - b^t without the cancellation (b - 1 is exact from 0.5 on)
    s.root = 1.0 / sqrt(-expm1(t * log1p(b2 - 1.0)));
    s.keep = decoupled ? 1.0 - l.lr[i] * l.wd[i] : 1.0;
    s.l2 = decoupled ? 0.0 : l.wd[i];
    out[i] = s;
}

// In float32 (float64 for float64 tensors); the state is float32 or wider, and a 16-bit parameter is rounded once, on
// its way back.
template <class C> struct Update {
    C b1, a1, b2, a2, eps, clip, size, root, keep, l2;
    __device__ __forceinline__ C operator()(C x, C g, C &m, C &v) const {
        g = g * clip;
        if (l2 != C(0)) g = fma(l2, x, g);        // not 0 * x, which an infinite x makes NaN
        m = fma(b1, m, a1 * g);
        v = fma(b2, v, a2 * g * g);
        const C d = fma(sqrt(v), root, eps);
        return fma(-size, m / d, x * keep);
    }
};

struct Betas { double b1, b2, eps; };

template <class E>
__device__ __forceinline__ void unit_adam(E, void *pp, const void *gg, void *mm, void *vv, int64_t first, int n, const Betas &b,
                                          const Scalars &s, double clip) {
    using T = typename E::T;
    using C = typename E::C;
    constexpr int V = sizeof(C) == 8 ? 2 : 4, kStep = kWave * V;
    T *p = static_cast<T *>(pp) + first;
    const T *g = static_cast<const T *>(gg) + first;
    C *m = static_cast<C *>(mm) + first, *v = static_cast<C *>(vv) + first;
    const Update<C> f{C(b.b1), C(1.0 - b.b1), C(b.b2), C(1.0 - b.b2), C(b.eps), C(clip), C(s.size), C(s.root), C(s.keep), C(s.l2)};
    const int lane = threadIdx.x % kWave;
    for (int i = lane * V; i + V <= n; i += kStep) {
        Pack<T, V> rp = load<T, V>(p + i);
        const Pack<T, V> rg = load<T, V>(g + i);
        Pack<C, V> rm = load<C, V>(m + i), rv = load<C, V>(v + i);
#pragma unroll
        for (int j = 0; j < V; j++) rp.v[j] = T(f(C(rp.v[j]), C(rg.v[j]), rm.v[j], rv.v[j]));
        store<T, V>(p + i, rp);
        store<C, V>(m + i, rm);
        store<C, V>(v + i, rv);
    }
    const int tail = n / V * V + lane;
    if (tail < n) p[tail] = T(f(C(p[tail]), C(g[tail]), m[tail], v[tail]));
}

__global__ __launch_bounds__(kThreads) void adam_update(const AdamList l, const Betas b, const Scalars *scalars, const double *factor) {
    const double clip = factor ? *factor : 1.0;
    for (uint32_t unit = blockIdx.x * kWaves + wave_of_block(); unit < l.u.units; unit += gridDim.x * kWaves) {
        const Piece q = piece(l.u, unit);
        const Scalars s = scalars[l.s[q.t]];
        by_type(q.type, [&](auto e) { unit_adam(e, l.p[q.t], l.g[q.t], l.m[q.t], l.v[q.t], q.first, q.n, b, s, clip); });
    }
}

// ---- host ----
// Values of a unit: small enough that the units of the list fill the chip's waves, large enough that finding a unit's
// tensor does not count.
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

// Runs through the tensors that have values, K at a time: fill(list, at, i) puts tensor i at place `at`, go(list, grid).
template <int K, class List, class Fill, class Go>
void in_lists(int64_t count, const int64_t *numel, const int *dtype, int shift, Fill fill, Go go) {
    List l;
    int at = 0;
    uint32_t units = 0;
    auto flush = [&] {
        if (!at) return;
        l.u.count = at;
        l.u.shift = shift;
        l.u.units = units;
        go(l, int(std::min<int64_t>((int64_t(units) + kWaves - 1) / kWaves, kMaxBlocks)));
        at = 0;
        units = 0;
    };
    for (int64_t i = 0; i < count; i++) {
        if (!numel[i]) continue;
        units += uint32_t((numel[i] + (int64_t(1) << shift) - 1) >> shift);
        l.u.n[at] = uint64_t(numel[i]) << 2 | uint64_t(dtype[i]);
        l.u.end[at] = units;
        fill(l, at, i);
        if (++at == K) flush();
    }
    flush();
}

constexpr int64_t kMaxValues = int64_t(1) << 40;

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

const int kSize[4] = {8, 4, 2, 2};

// Memory that is written must not be any other memory of the call.
struct Range { uintptr_t lo, hi; bool written; };
bool disjoint(std::vector<Range> &r) {
    std::sort(r.begin(), r.end(), [](const Range &a, const Range &b) { return a.lo < b.lo; });
    uintptr_t read_end = 0, write_end = 0;
    for (const Range &x : r) {
        if (x.lo < write_end || (x.written && x.lo < read_end)) return false;
        uintptr_t &end = x.written ? write_end : read_end;
        end = std::max(end, x.hi);
    }
    return true;
}

int launched(const char *what) {
    const hipError_t e = hipGetLastError();
    if (e == hipSuccess) return 0;
    static thread_local char text[160];
    snprintf(text, sizeof text, "%s: launch failed (hip error %d)", what, int(e));
    return report(-10, text);
}

int64_t partials(int64_t count) { return (count + kNormList - 1) / kNormList * kMaxBlocks; }

// Workspace: [factor, unused][partial sums][Scalars of each tensor]
struct Space {
    double *factor, *part;
    Scalars *scalars;
    Space(void *p, int64_t count) {
        factor = static_cast<double *>(p);
        part = factor + 2;
        scalars = reinterpret_cast<Scalars *>(part + partials(count));
    }
    static int64_t bytes(int64_t count) { return 16 + 8 * partials(count) + int64_t(sizeof(Scalars)) * count; }
};

template <int P>
void launch_norm_as(int64_t count, const void *const *x, const int64_t *numel, const int *dtype, const Space &ws, double max_norm,
                    double *norm, double *factor, hipStream_t st) {
    int parts = 0;
    in_lists<kNormList, NormList>(count, numel, dtype, unit_shift(total(count, numel)),
        [&](NormList &l, int at, int64_t i) { l.x[at] = const_cast<void *>(x[i]); },
        [&](const NormList &l, int grid) {
            hipLaunchKernelGGL((norm_partials<P>), dim3(grid), dim3(kThreads), 0, st, l, ws.part + parts);
            parts += grid;
        });
    hipLaunchKernelGGL((norm_finish<P>), dim3(1), dim3(kThreads), 0, st, ws.part, parts, max_norm, norm, factor);
}

void launch_norm(int kind, int64_t count, const void *const *x, const int64_t *numel, const int *dtype, const Space &ws, double max_norm,
                 double *norm, double *factor, hipStream_t st) {
    if (kind == MBRL_NORM_TWO) launch_norm_as<MBRL_NORM_TWO>(count, x, numel, dtype, ws, max_norm, norm, factor, st);
    else if (kind == MBRL_NORM_ONE) launch_norm_as<MBRL_NORM_ONE>(count, x, numel, dtype, ws, max_norm, norm, factor, st);
    else launch_norm_as<MBRL_NORM_INF>(count, x, numel, dtype, ws, max_norm, norm, factor, st);
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

int64_t mbrl_optim_workspace_bytes(int64_t count) {
    if (count < 0 || count > (int64_t(1) << 24)) return report(-6, "mbrl_optim_workspace_bytes: the number of tensors is out of range");
    return Space::bytes(count);
}

int mbrl_grad_norm(int64_t count, const void *const *grads, const int64_t *numel, const int *dtype, int norm_type, void *workspace,
                   int64_t workspace_bytes, double *norm, void *hip_stream) {
    return guarded("mbrl_grad_norm: failed", [&] {
        if (int rc = check_list("mbrl_grad_norm", count, numel, dtype)) return rc;
        if (norm_type < MBRL_NORM_INF || norm_type > MBRL_NORM_TWO) return report(-7, "mbrl_grad_norm: unknown norm type");
        if (!norm || !workspace || (count && !grads)) return report(-1, "mbrl_grad_norm: null argument");
        if (workspace_bytes < Space::bytes(count)) return report(-8, "mbrl_grad_norm: workspace too small (mbrl_optim_workspace_bytes)");
        for (int64_t i = 0; i < count; i++)
            if (numel[i] && !grads[i]) return report(-1, "mbrl_grad_norm: null tensor");
        launch_norm(norm_type, count, grads, numel, dtype, Space(workspace, count), 0.0, norm, nullptr, (hipStream_t)hip_stream);
        return launched("mbrl_grad_norm");
    });
}

int mbrl_clip_grad_norm(int64_t count, void *const *grads, const int64_t *numel, const int *dtype, int norm_type, double max_norm,
                        void *workspace, int64_t workspace_bytes, double *norm, void *hip_stream) {
    return guarded("mbrl_clip_grad_norm: failed", [&] {
        if (int rc = check_list("mbrl_clip_grad_norm", count, numel, dtype)) return rc;
        if (norm_type < MBRL_NORM_INF || norm_type > MBRL_NORM_TWO) return report(-7, "mbrl_clip_grad_norm: unknown norm type");
        if (!(max_norm >= 0.0)) return report(-7, "mbrl_clip_grad_norm: max_norm must not be negative");
        if (!norm || !workspace || (count && !grads)) return report(-1, "mbrl_clip_grad_norm: null argument");
        if (workspace_bytes < Space::bytes(count)) return report(-8, "mbrl_clip_grad_norm: workspace too small (mbrl_optim_workspace_bytes)");
        std::vector<Range> r;
        r.reserve(count);
        for (int64_t i = 0; i < count; i++) {
            if (!numel[i]) continue;
            if (!grads[i]) return report(-1, "mbrl_clip_grad_norm: null tensor");
            const uintptr_t lo = uintptr_t(grads[i]);
            r.push_back({lo, lo + uintptr_t(numel[i]) * kSize[dtype[i]], true});
        }
        if (!disjoint(r)) return report(-7, "mbrl_clip_grad_norm: two of the tensors share memory");
        const hipStream_t st = (hipStream_t)hip_stream;
        const Space ws(workspace, count);
        launch_norm(norm_type, count, grads, numel, dtype, ws, max_norm, norm, ws.factor, st);
        in_lists<kNormList, NormList>(count, numel, dtype, unit_shift(total(count, numel)),
            [&](NormList &l, int at, int64_t i) { l.x[at] = grads[i]; },
            [&](const NormList &l, int grid) { hipLaunchKernelGGL(clip_scale, dim3(grid), dim3(kThreads), 0, st, l, ws.factor); });
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
        if (!workspace || (count && (!params || !grads || !exp_avgs || !exp_avg_sqs || !steps || !lr || !weight_decay)))
            return report(-1, "mbrl_adam_step: null argument");
        if (workspace_bytes < Space::bytes(count)) return report(-8, "mbrl_adam_step: workspace too small (mbrl_optim_workspace_bytes)");
        std::vector<Range> r;
        r.reserve(5 * count);
        for (int64_t i = 0; i < count; i++) {
            if (!steps[i] || (numel[i] && (!params[i] || !grads[i] || !exp_avgs[i] || !exp_avg_sqs[i])))
                return report(-1, "mbrl_adam_step: null tensor");
            const int64_t size = kSize[dtype[i]], wide = size == 8 ? 8 : 4;
            auto range = [&](const void *p, int64_t bytes, bool written) {
                if (bytes) r.push_back({uintptr_t(p), uintptr_t(p) + uintptr_t(bytes), written});
            };
            range(params[i], numel[i] * size, true);
            range(grads[i], numel[i] * size, false);
            range(exp_avgs[i], numel[i] * wide, true);
            range(exp_avg_sqs[i], numel[i] * wide, true);
            range(steps[i], 4, true);
        }
        if (!disjoint(r)) return report(-7, "mbrl_adam_step: a tensor that is written shares memory with another one");
        const hipStream_t st = (hipStream_t)hip_stream;
        const Space ws(workspace, count);
        for (int64_t i = 0; i < count; i += kStepList) {
            StepList l;
            l.count = int(std::min<int64_t>(kStepList, count - i));
            for (int k = 0; k < l.count; k++) l.step[k] = steps[i + k], l.lr[k] = lr[i + k], l.wd[k] = weight_decay[i + k];
            hipLaunchKernelGGL(adam_scalars, dim3(1), dim3(kStepList), 0, st, l, beta_one, beta_two, decoupled, ws.scalars + i);
        }
        if (clip) launch_norm(norm_type, count, grads, numel, dtype, ws, max_norm, norm, ws.factor, st);
        const Betas b{beta_one, beta_two, eps};
        in_lists<kAdamList, AdamList>(count, numel, dtype, unit_shift(total(count, numel)),
            [&](AdamList &l, int at, int64_t i) { l.p[at] = params[i]; l.g[at] = grads[i]; l.m[at] = exp_avgs[i]; l.v[at] = exp_avg_sqs[i]; l.s[at] = uint32_t(i); },
            [&](const AdamList &l, int grid) {
                hipLaunchKernelGGL(adam_update, dim3(grid), dim3(kThreads), 0, st, l, b, ws.scalars, clip ? ws.factor : nullptr);
            });
        return launched("mbrl_adam_step");
    });
}

}  // extern "C"
