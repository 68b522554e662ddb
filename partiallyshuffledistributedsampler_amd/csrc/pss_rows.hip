// pss_rows.hip -- what a batch's rows go through after the sampler picked them: dropout keyed by
// row ids, routing to experts, dispatch into expert order and combination by weight (pss_rows.h).
#include <math.h>

#include <algorithm>

#include "pss_common.h"
#include "pss_device.h"
#include "pss_rows.h"

namespace pss {
namespace {

// ---- values --------------------------------------------------------------------------------------
// Eight values of a row at a time (one Philox block, 16 bytes of a 16-bit type).  Rows of odd width
// start at any multiple of the value's size, which global loads and stores of this target take.
template <typename T> struct Value;
template <> struct Value<float> {
    static __device__ __forceinline__ float up(float v) { return v; }
    static __device__ __forceinline__ float down(float v) { return v; }
};
template <> struct Value<__bf16> {
    static __device__ __forceinline__ float up(__bf16 v) { return (float)v; }
    static __device__ __forceinline__ __bf16 down(float v) { return (__bf16)v; }
};
template <> struct Value<_Float16> {
    static __device__ __forceinline__ float up(_Float16 v) { return (float)v; }
    static __device__ __forceinline__ _Float16 down(float v) { return (_Float16)v; }
};

// N values as one vector of the value's alignment: one wide load or store (an array of values is taken
// apart by the compiler and its first value's access shared with the branch for a row's end).
template <typename T, int N> struct Pack { typedef T V __attribute__((ext_vector_type(N), aligned(sizeof(T)))); };
template <typename T> struct Pack<T, 1> { typedef T V; };
__device__ __forceinline__ float at(float v, int) { return v; }
__device__ __forceinline__ __bf16 at(__bf16 v, int) { return v; }
__device__ __forceinline__ _Float16 at(_Float16 v, int) { return v; }
template <typename V> __device__ __forceinline__ auto at(const V &v, int i) { return v[i]; }

template <typename T, int N>
__device__ __forceinline__ void load(const T *p, int64_t left, float (&v)[N]) {
    if (left >= N) {
        typedef typename Pack<T, N>::V V;
        const V a = *(const V *)p;
#pragma unroll
        for (int i = 0; i < N; i++) v[i] = Value<T>::up(at(a, i));
    } else {
#pragma unroll
        for (int i = 0; i < N; i++) v[i] = i < left ? Value<T>::up(p[i]) : 0.f;
    }
}

template <typename T, int N>
__device__ __forceinline__ void store(T *p, int64_t left, const float (&v)[N]) {
    if (left >= N) {
        if constexpr (N == 1) {
            *p = Value<T>::down(v[0]);
        } else {
            typename Pack<T, N>::V a;
#pragma unroll
            for (int i = 0; i < N; i++) a[i] = Value<T>::down(v[i]);
            *(typename Pack<T, N>::V *)p = a;
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; i++)
            if (i < left) p[i] = Value<T>::down(v[i]);
    }
}

// Eight values of a row of D, from column c (a multiple of 8) on, 0 past the end.  A lane at the end reads
// the row's last eight and shifts them down: every lane makes the same wide load and several rows' loads
// stay on their way, where a branch that reads the end value by value waits for each (combine of 8 rows
// of 4095 bf16 of 8194 tokens: 169 -> 112 us; dropout of 16386 x 8191 bf16: 156 -> 119).  raw8 is the load
// (NT: nontemporal, past the caches), open8 the rest.  WHOLE (gather and dropout): D % 8 is 0, and
// no branch stands between the load and the Philox block (a call of gather of 65536 x 2048 bf16: 162 -> 99).
template <bool NT = false, bool WHOLE = false, typename T>
__device__ __forceinline__ typename Pack<T, 8>::V raw8(const T *row, int64_t c, int64_t D) {
    typedef typename Pack<T, 8>::V V;
    if (WHOLE) return NT ? __builtin_nontemporal_load((const V *)(row + c)) : *(const V *)(row + c);
    if (D >= 8) {
        const V *p = (const V *)(row + (c <= D - 8 ? c : D - 8));
        return NT ? __builtin_nontemporal_load(p) : *p;
    }
    V a;
#pragma unroll
    for (int i = 0; i < 8; i++) a[i] = i < D ? row[i] : (T)0.f;
    return a;
}
template <typename T, bool WHOLE = false, typename V>
__device__ __forceinline__ void open8(const V &a, int64_t c, int64_t D, float (&v)[8]) {
#pragma unroll
    for (int i = 0; i < 8; i++) v[i] = Value<T>::up(a[i]);
    if (!WHOLE && D > 8 && D % 8) {
        const int by = c > D - 8 ? (int)(c - (D - 8)) : 0;
#pragma unroll
        for (int s = 1; s < 8; s *= 2)
#pragma unroll
            for (int i = 0; i < 8; i++) v[i] = !(by & s) ? v[i] : i + s < 8 ? v[i + s] : 0.f;
    }
}
template <bool NT = false, bool WHOLE = false, typename T>
__device__ __forceinline__ void load8(const T *row, int64_t c, int64_t D, float (&v)[8]) {
    open8<T, WHOLE>(raw8<NT, WHOLE>(row, c, D), c, D, v);
}
// and the values back: what is left of a row in pieces of 4, 2 and 1
template <bool NT = false, bool WHOLE = false, typename T>
__device__ __forceinline__ void store8(T *row, int64_t c, int64_t D, const float (&v)[8]) {
    typename Pack<T, 8>::V a;
#pragma unroll
    for (int i = 0; i < 8; i++) a[i] = Value<T>::down(v[i]);
    T *p = row + c;
    const int left = WHOLE || D - c >= 8 ? 8 : (int)(D - c);
    if (left == 8) {
        if (NT) __builtin_nontemporal_store(a, (typename Pack<T, 8>::V *)p);
        else *(typename Pack<T, 8>::V *)p = a;
    } else {
        if (left & 4) {
            *(typename Pack<T, 4>::V *)p = __builtin_shufflevector(a, a, 0, 1, 2, 3);
            p += 4;
        }
        const auto b = left & 4 ? __builtin_shufflevector(a, a, 4, 5, 6, 6) : __builtin_shufflevector(a, a, 0, 1, 2, 2);
        if (left & 2) {
            *(typename Pack<T, 2>::V *)p = __builtin_shufflevector(b, b, 0, 1);
            p += 2;
        }
        if (left & 1) *p = left & 2 ? b[2] : b[0];
    }
}

// ---- dropout -------------------------------------------------------------------------------------
__device__ __forceinline__ int64_t drop_row(const Drop &d, int64_t i) {
    const uint64_t id = !d.ids ? (uint64_t)i : d.per_row ? (uint64_t)d.ids[i] : (uint64_t)d.ids[0] + (uint64_t)i;
    return (int64_t)((uint64_t)d.row0 + id);        // (modulo 2^64)
}

// The eight draws of a block of columns of the row with id r.
struct Draw { uint32_t w[4]; };
__device__ __forceinline__ Draw draw8(const Drop &d, int64_t r, uint32_t block) {
    uint32_t c0 = block, c1 = (uint32_t)r, c2 = (uint32_t)((uint64_t)r >> 32), c3 = DOM_DROPOUT;
    philox4x32_10(c0, c1, c2, c3, d.key0, d.key1);
    return Draw{{c0, c1, c2, c3}};
}

// v * scale (+ add, in one rounding as the CPU mode's fma) where kept; an exact 0 (add) where not,
// also of an infinity or a NaN.
template <bool ADD>
__device__ __forceinline__ void drop8(const Drop &d, const Draw &u, float (&v)[8], const float (&add)[8]) {
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const uint32_t x = (i & 1) ? u.w[i >> 1] >> 16 : u.w[i >> 1] & 0xFFFFu;
        v[i] = x >= d.drop ? (ADD ? fmaf(v[i], d.scale, add[i]) : v[i] * d.scale) : (ADD ? add[i] : 0.f);
    }
}

// y = dropout(x) (+ residual).  Bound by memory: a value is read (twice with a residual) and written, and
// 20 32 x 32-bit products per 8 values hide behind that.  One thread per block of 8 columns, over rows and
// blocks as one range, so that odd widths leave no lanes idle; (row, block) are stepped, not divided.
// 16384 x 8192 bf16: 135 us with a residual (6.0 TB/s), 91 without (5.9); x 8191, whose rows start at
// any 2 bytes, 178 and 126; 4093 x 1537 fp32, from the Infinity Cache: 14 and 9.
template <typename T, bool RES, bool NT, bool WHOLE>
__global__ __launch_bounds__(256) void k_dropout(const T *__restrict__ x, int64_t ldx, const T *__restrict__ res,
                                                 int64_t ldr, T *__restrict__ y, int64_t rows, int64_t cols,
                                                 uint32_t nb, Drop d) {
    const int64_t step = (int64_t)gridDim.x * blockDim.x;
    const int64_t at = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    int64_t row = at / nb;
    uint32_t b = (uint32_t)(at - row * nb);
    const int64_t drow = step / nb;
    const uint32_t db = (uint32_t)(step - drow * nb);
    while (row < rows) {
        const int64_t c = (int64_t)b * 8;
        float v[8];
        load8<NT, WHOLE>(x + row * ldx, c, cols, v);
        float r[8];
        Draw dr;
        if (d.drop) dr = draw8(d, drop_row(d, row), b);
        if (RES) load8<NT, WHOLE>(res + row * ldr, c, cols, r);     // after the block: 140 -> 133 us
        if (d.drop) {
            drop8<RES>(d, dr, v, r);
        } else if (RES) {
#pragma unroll
            for (int i = 0; i < 8; i++) v[i] += r[i];
        }
        store8<NT, WHOLE>(y + row * cols, c, cols, v);
        row += drow;
        b += db;
        if (b >= nb) { b -= nb; row++; }
    }
}

// ---- routing -------------------------------------------------------------------------------------
// The lanes of a segment (4, 8, 16, 32 or 64 of a wave) share one row; reductions stay inside the segment.  Step
// i joins lanes that hold the same after the steps before: 1 and 2 apart, then the halves of 8 and 16
// mirrored (DPP, no LDS), then 16 and 32 apart.
template <int CTRL> __device__ __forceinline__ uint32_t dpp_mov(uint32_t x) {
    return (uint32_t)__builtin_amdgcn_update_dpp((int)x, (int)x, CTRL, 0xF, 0xF, true);
}
template <int I> __device__ __forceinline__ uint32_t partner32(uint32_t x) {
    if constexpr (I == 0) return dpp_mov<0xB1>(x);
    else if constexpr (I == 1) return dpp_mov<0x4E>(x);
    else if constexpr (I == 2) return dpp_mov<0x141>(x);
    else if constexpr (I == 3) return dpp_mov<0x140>(x);
    else return (uint32_t)__shfl_xor((int)x, 1 << I, 64);
}
template <int I, typename T> __device__ __forceinline__ T partner(T x) {
    if constexpr (sizeof(T) == 4) {
        uint32_t u;
        __builtin_memcpy(&u, &x, 4);
        u = partner32<I>(u);
        __builtin_memcpy(&x, &u, 4);
    } else {
        static_assert(sizeof(T) == 8);
        uint32_t u[2];
        __builtin_memcpy(u, &x, 8);
        u[0] = partner32<I>(u[0]);
        u[1] = partner32<I>(u[1]);
        __builtin_memcpy(&x, u, 8);
    }
    return x;
}
template <int L, typename T, typename F>
__device__ __forceinline__ T seg_reduce(T v, F f) {
    v = f(v, partner<0>(v));
    v = f(v, partner<1>(v));
    if constexpr (L >= 8) v = f(v, partner<2>(v));
    if constexpr (L >= 16) v = f(v, partner<3>(v));
    if constexpr (L >= 32) v = f(v, partner<4>(v));
    if constexpr (L == 64) v = f(v, partner<5>(v));
    return v;
}
struct Max { template <typename T> __device__ T operator()(T a, T b) const { return a > b ? a : b; } };
struct Min { template <typename T> __device__ T operator()(T a, T b) const { return a < b ? a : b; } };
struct Sum { template <typename T> __device__ T operator()(T a, T b) const { return a + b; } };
struct Or { template <typename T> __device__ T operator()(T a, T b) const { return a | b; } };
template <int L> __device__ __forceinline__ float seg_max(float v) {
    return seg_reduce<L>(v, [](float a, float b) { return fmaxf(a, b); });
}
template <int L> __device__ __forceinline__ float seg_min(float v) {
    return seg_reduce<L>(v, [](float a, float b) { return fminf(a, b); });
}

__device__ __forceinline__ void wave_lds_sync() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// N <= E logits of row t from expert e0 on, -inf past the last.  A lane whose values run past the end
// reads the row's last N and shifts them down: no branch, no loads one by one.
template <typename T, int N>
__device__ __forceinline__ void load_end(const T *row, int e0, int E, float (&l)[N]) {
    const int left = E - e0;
    load(row + (left >= N ? e0 : left > 0 ? E - N : 0), N, l);
    if (E % N) {
        const int by = left >= N ? 0 : N - left;
#pragma unroll
        for (int s = 1; s < N; s *= 2)
#pragma unroll
            for (int i = 0; i < N; i++) l[i] = !(by & s) ? l[i] : i + s < N ? l[i + s] : -INFINITY;
    }
    if (left <= 0)
#pragma unroll
        for (int i = 0; i < N; i++) l[i] = -INFINITY;
}
template <int N>
__device__ __forceinline__ void load_logits(const RouteArgs &a, int64_t t, int e0, float (&l)[N]) {
    const int64_t i = t * a.ld;
    if (a.dtype == 0) load_end((const float *)a.logits + i, e0, a.E, l);
    else if (a.dtype == 1) load_end((const __bf16 *)a.logits + i, e0, a.E, l);
    else load_end((const _Float16 *)a.logits + i, e0, a.E, l);
}
__device__ __forceinline__ float one_logit(const RouteArgs &a, int64_t t, int e) {
    const int64_t i = t * a.ld + e;
    if (a.dtype == 0) return ((const float *)a.logits)[i];
    if (a.dtype == 1) return (float)((const __bf16 *)a.logits)[i];
    return (float)((const _Float16 *)a.logits)[i];
}

// exp of a difference of logits (<= 0): off by 2^-24 of the exponent and one unit of the result
__device__ __forceinline__ float fast_exp(float x) { return __builtin_amdgcn_exp2f(x * 1.44269504f); }

// Sorted lists (falling) of unsigned keys, in registers.
__device__ __forceinline__ void order2(uint32_t &a, uint32_t &b) {
    const uint32_t hi = a > b ? a : b, lo = a > b ? b : a;
    a = hi;
    b = lo;
}
template <int N> __device__ __forceinline__ void bitonic(uint32_t *x) {   // a bitonic list into falling order
#pragma unroll
    for (int h = N / 2; h; h >>= 1)
#pragma unroll
        for (int i = 0; i < N; i++)
            if (!(i & h)) order2(x[i], x[i + h]);
}
// x[0, N) any -> falling: bitonic, and for 8 the network of 19 comparisons (the fewest)
template <int N> __device__ __forceinline__ void sort_falling(uint32_t *x) {
    if constexpr (N == 8) {
        order2(x[0], x[2]); order2(x[1], x[3]); order2(x[4], x[6]); order2(x[5], x[7]);
        order2(x[0], x[4]); order2(x[1], x[5]); order2(x[2], x[6]); order2(x[3], x[7]);
        order2(x[0], x[1]); order2(x[2], x[3]); order2(x[4], x[5]); order2(x[6], x[7]);
        order2(x[2], x[4]); order2(x[3], x[5]);
        order2(x[1], x[4]); order2(x[3], x[6]);
        order2(x[1], x[2]); order2(x[3], x[4]); order2(x[5], x[6]);
    } else if constexpr (N > 1) {
        sort_falling<N / 2>(x);
        sort_falling<N / 2>(x + N / 2);
        // two falling halves: the larger of each mirrored pair first
#pragma unroll
        for (int i = 0; i < N / 2; i++) order2(x[i], x[N - 1 - i]);
        bitonic<N / 2>(x);
        bitonic<N / 2>(x + N / 2);
    }
}
// the KP largest of two falling lists
template <int KP> __device__ __forceinline__ void merge_top(uint32_t *x, const uint32_t *y) {
#pragma unroll
    for (int i = 0; i < KP; i++) x[i] = x[i] > y[KP - 1 - i] ? x[i] : y[KP - 1 - i];
    bitonic<KP>(x);
}
// the KP largest keys of a segment, falling, in every lane; each lane's less `first` (0 stays 0)
template <int L, int V, int KP>
__device__ __forceinline__ void seg_top(const uint32_t *key, uint32_t first, uint32_t *top) {
    if constexpr (V <= KP) {
#pragma unroll
        for (int i = 0; i < KP; i++) top[i] = i < V ? key[i] : 0u;
        sort_falling<V>(top);
    } else {
#pragma unroll
        for (int i = 0; i < KP; i++) top[i] = key[i];
        sort_falling<KP>(top);
#pragma unroll
        for (int b = KP; b < V; b += KP) {
            uint32_t more[KP];
#pragma unroll
            for (int i = 0; i < KP; i++) more[i] = key[b + i];
            sort_falling<KP>(more);
            merge_top<KP>(top, more);
        }
    }
#pragma unroll
    for (int i = 0; i < KP; i++) top[i] = top[i] ? top[i] - first : 0u;
    auto step = [&](auto I) {
        uint32_t other[KP];
#pragma unroll
        for (int i = 0; i < KP; i++) other[i] = partner32<decltype(I)::value>(top[i]);
        merge_top<KP>(top, other);
    };
    step(std::integral_constant<int, 0>());
    step(std::integral_constant<int, 1>());
    if constexpr (L >= 16) {
        step(std::integral_constant<int, 2>());
        step(std::integral_constant<int, 3>());
    }
    if constexpr (L == 64) {
        step(std::integral_constant<int, 4>());
        step(std::integral_constant<int, 5>());
    }
}

constexpr double kDead = -INFINITY;   // an expert that cannot be chosen
constexpr double kLast = -1e300;      // a live one whose choice value is no number: after all others

// the maximum of a wave: inside rows of 16 lanes, then of the four rows
__device__ __forceinline__ uint32_t wave_max(uint32_t v) {
    v = seg_reduce<16>(v, Max());
    const uint32_t a = __builtin_amdgcn_readlane(v, 0), b = __builtin_amdgcn_readlane(v, 16);
    const uint32_t c = __builtin_amdgcn_readlane(v, 32), d = __builtin_amdgcn_readlane(v, 48);
    return std::max(std::max(a, b), std::max(c, d));
}

// The choice of a row's experts from values in 64 bits, one at a time, by a whole wave: lane j's expert.
// It is the definition of the choice, and what the 32-bit choice leaves to it where its values are too
// close to tell the order, too far from the best, or no numbers.  l[v], bias[v]: of expert 64 * v + lane
// (l is -inf past the last, bias 0 without one); m: the logits' maximum; sum: of their exponentials, set here if `exps`; value:
// E + G doubles of LDS (groups).  One row is 5 us of latency, which a launch sees once, at its end.
template <int V>
__device__ __forceinline__ int choose64(const RouteArgs &a, bool by_logit, bool exps, int lane, const float (&l)[V],
                                        const float (&bias)[V], float m, double &sum, double *value) {
    const int E = a.E, G = a.groups, S = E / G;
    double c[V];
#pragma unroll
    for (int v = 0; v < V; v++) c[v] = (double)l[v];
    sum = 1.0;
    if (!by_logit || exps) {
        // exponentials, two at a time
        double t[V];
#pragma unroll
        for (int v = 0; v < V; v++) t[v] = a.score == 0 ? c[v] - (double)m : -c[v];
        if (V < 2) {
            t[0] = exp(t[0]);
        } else {
#pragma unroll
            for (int v = 0; v + 1 < V; v += 2) {
                const double x = exp(t[v]), y = exp(t[v + 1]);
                t[v] = x;
                t[v + 1] = y;
            }
            if (V % 2) t[V - 1] = exp(t[V - 1]);
        }
        if (exps) {
            sum = 0.0;
#pragma unroll
            for (int v = 0; v < V; v++) sum += l[v] == -INFINITY ? 0.0 : t[v];
            sum = seg_reduce<64>(sum, Sum());
        }
        if (!by_logit)
#pragma unroll
            for (int v = 0; v < V; v++) {
                // t / sum, or 1 / (1 + t)
                const double x = (a.score == 0 ? t[v] : 1.0) / (a.score == 0 ? sum : 1.0 + t[v]);
                c[v] = a.bias ? x + (double)bias[v] : x;
            }
    }
#pragma unroll
    for (int v = 0; v < V; v++) c[v] = l[v] == -INFINITY || bias[v] == -INFINITY ? kDead : c[v] >= kLast ? c[v] : kLast;
    if (G > 1) {
        double *score = value + E;
#pragma unroll
        for (int v = 0; v < V; v++)
            if (64 * v + lane < E) value[64 * v + lane] = c[v];
        wave_lds_sync();
        double mine = kDead;
        if (lane < G) {
            double b2 = kDead;
#pragma unroll 8
            for (int s = 0; s < S; s++) {
                const double x = value[lane * S + s];
                b2 = x > mine ? mine : x > b2 ? x : b2;
                mine = x > mine ? x : mine;
            }
            if (a.group_sum == 2 && b2 > kDead) mine += b2;
            score[lane] = mine;
        }
        wave_lds_sync();
        int before = 0;         // a group is kept if fewer than top_groups come before it
#pragma unroll 8
        for (int o = 0; o < G; o++) {
            const double x = score[o];
            before += x > mine || (x == mine && o < lane);
        }
        const uint64_t kept = __ballot(lane < G && before < a.top_groups);
        wave_lds_sync();
#pragma unroll
        for (int v = 0; v < V; v++) c[v] = kept >> ((uint32_t)(64 * v + lane) / (uint32_t)S & 63) & 1 ? c[v] : kDead;
    }
    int my_e = -1;
    for (int j = 0; j < a.k; j++) {
        double best = kDead;
        int be = 1 << 20;
#pragma unroll
        for (int v = 0; v < V; v++) {
            be = c[v] > best ? 64 * v + lane : be;
            best = c[v] > best ? c[v] : best;
        }
        // the wave's maximum as ordered bits, high word first; of equal values the lowest expert
        uint64_t u;
        best += 0.0;            // -0 is 0
        __builtin_memcpy(&u, &best, 8);
        u ^= (uint64_t)((int64_t)u >> 63) | 0x8000000000000000ull;
        const uint32_t hi = (uint32_t)(u >> 32), lo = (uint32_t)u, top = wave_max(hi);
        bool on = hi == top;
        uint64_t who = __ballot(on);
        if (who & (who - 1)) {
            const uint32_t low = wave_max(on ? lo : 0u);
            on = on && lo == low;
            who = __ballot(on);
        }
        int won = __builtin_amdgcn_readlane(be, __builtin_ctzll(who));
        if (who & (who - 1)) won = (int)~wave_max(on ? ~(uint32_t)be : 0u);
        if (lane == j) my_e = won < E ? won : -1;
#pragma unroll
        for (int v = 0; v < V; v++) c[v] = 64 * v + lane == won ? kDead : c[v];
    }
    return my_e;
}

// A group's value as an unsigned key of its order, the lowest 6 bits the index (lower first); and back,
// to within those bits.  -0 is 0.
__device__ __forceinline__ uint32_t group_key(float x, uint32_t g) {
    uint32_t u = __float_as_uint(x + 0.f);
    u ^= (uint32_t)((int32_t)u >> 31) | 0x80000000u;
    return (u & ~63u) | (63u - g);
}
__device__ __forceinline__ float group_value(uint32_t key) {
    uint32_t u = key & ~63u;
    u ^= u & 0x80000000u ? 0x80000000u : 0xFFFFFFFFu;
    return __uint_as_float(u);
}

// The two best of the values of aligned runs of lanes: a lane stands for `unit` values, a run for `all`
// (both powers of two), the lanes hold their own two best.
template <int L> __device__ __forceinline__ void join_best(int unit, int all, float &b1, float &b2) {
    auto join = [&](auto I) {
        if ((unit << decltype(I)::value) < all) {
            const float o1 = partner<decltype(I)::value>(b1), o2 = partner<decltype(I)::value>(b2);
            b2 = fmaxf(fminf(b1, o1), fmaxf(b2, o2));
            b1 = fmaxf(b1, o1);
        }
    };
    join(std::integral_constant<int, 0>());
    join(std::integral_constant<int, 1>());
    if constexpr (L >= 16) {
        join(std::integral_constant<int, 2>());
        join(std::integral_constant<int, 3>());
    }
    if constexpr (L == 64) {
        join(std::integral_constant<int, 4>());
        join(std::integral_constant<int, 5>());
    }
}

constexpr int kPlaceThreads = 512;

// Exclusive scan of v[0, E) in LDS by all NT threads; returns the total.
template <int NT> __device__ __forceinline__ int32_t scan_lds(int32_t *v, int E, uint32_t *scan_tmp) {
    uint32_t run = 0;
    for (int e0 = 0; e0 < E; e0 += NT) {
        const int e = e0 + threadIdx.x;
        uint32_t total;
        const uint32_t x = e < E ? (uint32_t)v[e] : 0u;
        const uint32_t pre = block_excl_scan<NT>(x, scan_tmp, total);
        if (e < E) v[e] = (int32_t)(run + pre);
        run += total;
    }
    __syncthreads();
    return (int32_t)run;
}

// Places of the slots of one chunk of up to 64 rows: rows of an expert in the order of the rows (mask[e]: the
// chunk's rows that have it, base[e]: where its rows of this chunk begin), slots without an expert from
// unused0 on.  All NT threads, at most kRouteChunk * kRouteMaxK / NT slots each; `first` holds 64 words.
template <int NT>
__device__ __forceinline__ void place_chunk(const RouteArgs &a, int64_t t0, int nt, const uint64_t *mask,
                                            const int32_t *base, int32_t unused0, uint32_t *first) {
    constexpr int kPer = kRouteChunk * kRouteMaxK / NT;
    const int k = a.k, n = nt * k;
    int e[kPer];
    bool none = false;
#pragma unroll
    for (int q = 0; q < kPer; q++) {
        const int i = threadIdx.x + q * NT;
        e[q] = i < n ? a.experts[t0 * k + i] : 0;
        none |= e[q] < 0;
    }
    if (__syncthreads_or(none)) {
        if (threadIdx.x < 64) {     // slots without an expert in the rows before
            const int t = threadIdx.x;
            uint32_t un = 0;
            if (t < nt)
                for (int j = 0; j < k; j++) un += a.experts[(t0 + t) * k + j] < 0;
            const uint32_t incl = wave_incl_scan(un);
            first[t] = incl - un - (k - un);        // + j = the slot's rank: they are a row's last slots
        }
        __syncthreads();
    }
#pragma unroll
    for (int q = 0; q < kPer; q++) {
        const int i = threadIdx.x + q * NT;
        if (i >= n) break;
        const int t = i / k, j = i - t * k;
        const int64_t slot = t0 * k + i;
        const int32_t p = e[q] < 0 ? unused0 + (int32_t)(first[t] + j)
                                   : base[e[q]] + __popcll(mask[e[q]] & ((1ull << t) - 1));
        a.pos[slot] = p;
        a.src[p] = (int32_t)slot;
    }
}

// Weight of the slot of a thread, KP threads a row: e its expert (0xFFFF: none); m, sum: the row's softmax
// statistics (scores not renormalised).  Softmax is exp(l - max) / sum, renormalised over the chosen
// alone; so are sigmoids, exp(min(l, 0)) / (1 + exp(-|l|)), with the best one's exp(min(l, 0)) taken out of
// all: neither under- nor overflows.  k values a row, so the library's expf (fast_exp is off by 60 u at
// 87 below the best).
template <int KP>
__device__ __forceinline__ void finish_slot(const RouteArgs &a, int64_t t, int i, int j, int e, bool nan, float m,
                                            float sum, uint64_t *mask) {
    const bool used = j < a.k && e != 0xFFFF;
    const float lw = used ? one_logit(a, t, e) : -INFINITY;
    float w = 0.f;
    if (a.renorm) {
        const float best = seg_max<KP>(lw);
        if (used) w = a.score == 0 ? expf(lw - best) : expf(fminf(lw, 0.f) - fminf(best, 0.f)) / (1.f + expf(-fabsf(lw)));
        const float ws = seg_reduce<KP>(w, Sum());
        w = used ? w / ws * a.scale : 0.f;
    } else if (used) {
        w = a.scale * (a.score == 0 ? expf(lw - m) / sum : 1.f / (1.f + expf(-lw)));
    }
    if (used && nan) w = NAN;
    if (j < a.k) {
        const int64_t slot = t * a.k + j;
        a.experts[slot] = used ? e : -1;
        a.weights[slot] = w;
        // 1 - sigmoid, for the gradient: its rows would else be read again for k values each
        if (a.slopes) a.slopes[slot] = used ? 1.f / (1.f + expf(lw)) : 0.f;
        if (used) atomicOr((unsigned long long *)&mask[e], 1ull << i);
    }
}

// The choice of the experts and their weights.  Bound by vector instructions, about 1000 a wave and four
// rows of 256 experts (a third of them scores, a quarter the sorting networks); k rounds of a maximum over
// 64-bit values took 166 us where this takes 45 (65536 rows, 8 of 256 experts in 16 groups, sigmoid and
// bias, bf16; reading the logits alone: 7).
//
// One workgroup routes a chunk of up to 64 rows, L lanes a row and V experts a lane.  The choice runs on
// 32-bit keys that hold value and expert (unique, so that maxima need no ties): of 16-bit logits the
// order-preserving bits themselves, else the value's distance from a floor below the row's best, in 24
// bits (22 beyond 256 experts).  Sorting networks of the KP >= k largest keys run in registers and
// across lanes.  A row where two neighbours of the result, or the last chosen and the first not, are
// nearer than the keys' and the scores' error is left to choose64 after the others.  Weights come last,
// KP threads a row.
template <int L, int V, int KP, int kThreads>
__global__ __launch_bounds__(kThreads, L == 64 ? 4 : 6) void k_route(RouteArgs a) {
    extern __shared__ __align__(16) uint64_t lds[];
    __shared__ uint32_t scan_tmp[kThreads / 64], first[64];
    __shared__ unsigned long long odd_rows, nan_rows;
    __shared__ __align__(16) uint16_t chosen[kRouteChunk * KP];
    __shared__ float2 stat[kRouteChunk];
    __shared__ uint32_t steep;  // 1 + the largest |bias|, 0 without biases, as the bits of a float
    constexpr int kIndex = L * V <= 256 ? 8 : 10;
    constexpr uint32_t kIndexMask = (1u << kIndex) - 1, kExactMask = 0x1FFFu;
    const int E = a.E, k = a.k, G = a.groups, S = E / G;
    int lane = threadIdx.x & (L - 1);
    const int seg = threadIdx.x / L;
    uint64_t *mask = lds;                                                  // [E]
    double *room = (double *)(mask + (E + 1) / 2 * 2);                     // 16-byte aligned; groups alone:
    const int Gp = (G + 3) & ~3;
    uint32_t *score = (uint32_t *)room + (size_t)seg * Gp;                 // [segments][Gp], the last ones 0
    float *value = (float *)room + (size_t)(kThreads / L) * Gp + (size_t)seg * (L * V);  // [segments][L * V]
    const int64_t t0 = (int64_t)blockIdx.x * a.chunk;
    const int nt = (int)(a.T - t0 < a.chunk ? a.T - t0 : a.chunk);
    const bool by_logit = !a.bias && (G == 1 || a.group_sum == 1);
    const bool exact = by_logit && a.dtype != 0;                           // keys that lose nothing
    const bool exps = a.score == 0 && !(by_logit && a.renorm);             // softmax statistics wanted
    const uint32_t inv = ((1u << 20) + S - 1) / S;                         // e / S = e * inv >> 20, e < 1024
    for (int i = threadIdx.x; i < E; i += kThreads) mask[i] = 0;
    if (G > 1)
        for (int i = threadIdx.x; i < kThreads / L * Gp; i += kThreads) ((uint32_t *)room)[i] = 0;
    if (threadIdx.x == 0) { odd_rows = nan_rows = 0; steep = 0; }
    __syncthreads();
    // (in LDS, value v of lane x at v / 4 * 4 * L + 4 * x + v % 4: registers are what limits the waves)
    __shared__ float bias[L * V < 64 ? 64 : L * V];
    constexpr int kVec = V < 4 ? V : 4;
    if (a.bias) {
        float far = 0.f;
        for (int e = threadIdx.x; e < L * V; e += kThreads) {
            const int x = e / V, v = e % V;
            const float b = e < E ? a.bias[e] : 0.f;
            bias[(v / kVec * L + x) * kVec + v % kVec] = b;
            // (a bias that is no number leaves every row's groups to choose64)
            if (b != 0.f) far = fmaxf(far, fabsf(b) < 1e30f ? 1.f + fabsf(b) : INFINITY);
        }
        if (G > 1) {
            far = seg_max<64>(far);
            if ((threadIdx.x & 63) == 0) atomicMax(&steep, __float_as_uint(far));
        }
    }
    auto add_bias = [&](float (&c)[V]) {
#pragma unroll
        for (int v = 0; v < V; v++) c[v] += bias[(v / kVec * L + lane) * kVec + v % kVec];
    };
    __syncthreads();
    for (int i0 = 0; i0 < nt; i0 += kThreads / L) {
        asm volatile("" : "+v"(lane));      // what depends on the lane is made anew for every row, not kept
        const int i = i0 + seg;
        const bool row = i < nt;
        const int64_t t = t0 + (row ? i : 0);
        const bool on = row && (!a.valid || a.valid[t]);
        // c: a NaN or -inf where the expert is masked (0 * l is a NaN for l = -inf; the maxima below
        // leave a NaN out, and its key is 0).  A row that has a NaN or +inf is left to choose64.
        float c[V];
        load_logits(a, t, lane * V, c);
        bool odd = false;
        float m = -INFINITY, sum = 1.f, eps = 0.f;
#pragma unroll
        for (int v = 0; v < V; v++) odd |= __builtin_amdgcn_classf(c[v], 0x203);
        if (exps) {
#pragma unroll
            for (int v = 0; v < V; v++) m = fmaxf(m, c[v]);
            m = seg_max<L>(m);
            const float mm = m == -INFINITY ? 0.f : m;
            float s[V];
            sum = 0.f;
#pragma unroll
            for (int v = 0; v < V; v++) {
                s[v] = fast_exp(c[v] - mm);
                sum += s[v];
            }
            sum = seg_reduce<L>(sum, Sum());
            if (!by_logit) {
                // off by 2e-6 at most: the exponent's rounding, and the sum over the row
                eps = 2e-6f;
                const float r = __builtin_amdgcn_rcpf(sum);
#pragma unroll
                for (int v = 0; v < V; v++) c[v] = fmaf(c[v], 0.f, s[v] * r);
                if (a.bias) add_bias(c);
            }
        } else if (!by_logit) {
            // off by 5e-7: the exponent's rounding times s (1 - s), and a unit each of exp, sum, reciprocal
            eps = 5e-7f;
#pragma unroll
            for (int v = 0; v < V; v++) c[v] = fmaf(c[v], 0.f, __builtin_amdgcn_rcpf(1.f + fast_exp(-c[v])));
            if (a.bias) add_bias(c);
        }
        if (G > 1) {
            const float far = __uint_as_float(steep);
            odd |= far >= 1e30f;
#pragma unroll
            for (int v = 0; v < V; v++) c[v] = fmaxf(c[v], -INFINITY);      // (a median takes no NaN)
            // the two best of every group: a lane's values one by one, then across lanes, or through LDS
            if ((S & (S - 1)) == 0) {
                float b1 = -INFINITY, b2 = -INFINITY;
                auto flush = [&](int e) {       // of expert e's group
                    const uint32_t g = ((uint32_t)e * inv) >> 20;
                    score[g] = group_key(a.group_sum == 2 && b2 > -INFINITY ? b1 + b2 : b1, g);
                };
#pragma unroll
                for (int v = 0; v < V; v++) {
                    b2 = __builtin_amdgcn_fmed3f(b1, b2, c[v]);
                    b1 = fmaxf(b1, c[v]);
                    if (((v + 1) & (S - 1)) == 0) {
                        if (lane * V + v < E) flush(lane * V + v);
                        b1 = b2 = -INFINITY;
                    }
                }
                join_best<L>(V, S, b1, b2);
                if (S > V && ((lane * V) & (S - 1)) == 0 && lane * V < E) flush(lane * V);
            } else {
#pragma unroll
                for (int v = 0; v < V; v++) value[lane * V + v] = c[v];
                wave_lds_sync();
                // `share` lanes a group
                int share = 1;
                while (2 * share * G <= L) share *= 2;
                for (int g0 = 0; g0 < G; g0 += L / share) {
                    const int g = g0 + lane / share;
                    float b1 = -INFINITY, b2 = -INFINITY;
                    if (g < G) {
#pragma unroll 4
                        for (int s = lane & (share - 1); s < S; s += share) {
                            const float x = value[g * S + s];
                            b2 = __builtin_amdgcn_fmed3f(b1, b2, x);
                            b1 = fmaxf(b1, x);
                        }
                    }
                    join_best<L>(1, share, b1, b2);
                    if (g < G && !(lane & (share - 1)))
                        score[g] = group_key(a.group_sum == 2 && b2 > -INFINITY ? b1 + b2 : b1, g);
                }
            }
            wave_lds_sync();
            // a group is kept if fewer than top_groups keys are larger
            uint64_t kept = 0;
            uint32_t least = 0xFFFFFFFFu, most = 0;       // of the groups kept, and of the others
            for (int g = lane; g < G; g += L) {
                const uint32_t x = score[g];
                int before = 0;
                for (int o = 0; o < G; o += 4) {
                    const uint4 y = *(const uint4 *)(score + o);
                    before += (y.x > x) + (y.y > x) + (y.z > x) + (y.w > x);
                }
                if (before < a.top_groups) {
                    kept |= 1ull << g;
                    least = std::min(least, x);
                } else {
                    most = std::max(most, x);
                }
            }
            kept = seg_reduce<L>(kept, Or());
            if (!exact) {
                least = seg_reduce<L>(least, Min());
                most = seg_reduce<L>(most, Max());
                // two scores' errors on either side, of the sums the roundings and the keys' 64 units, and half a
                // step of each of the four summands: biases of opposite sign leave a sum far below them
                const float p = group_value(least), q = group_value(most);
                const float apart = 4.f * eps + (a.group_sum == 2 ? 0x1p-22f * far : 0.f) + 0x1.4p-17f * fmaxf(fabsf(p), fabsf(q));
                if (most) odd |= !(p - q > apart) && q > -INFINITY;
            }
            wave_lds_sync();
            const uint32_t g0 = ((uint32_t)(lane * V) * inv) >> 20;
            const uint32_t from = (uint32_t)(kept >> (g0 & 63));           // bit 0: the first value's group
            if (S >= V && (S & (S - 1)) == 0) {
#pragma unroll
                for (int v = 0; v < V; v++) c[v] = from & 1 ? c[v] : -INFINITY;
            } else {
                const uint32_t r0 = lane * V - g0 * S;
#pragma unroll
                for (int v = 0; v < V; v++) c[v] = from >> (((r0 + v) * inv) >> 20) & 1 ? c[v] : -INFINITY;
            }
        }
        // (a key holds the place in the lane until the lane's own are sorted: fewer registers)
        uint32_t key[V];
        if (exact) {
#pragma unroll
            for (int v = 0; v < V; v++) {
                uint32_t u = __float_as_uint(c[v] + 0.f);       // -0 is 0
                u ^= (uint32_t)((int32_t)u >> 31) | 0x80000000u;
                u = (u & ~kExactMask) | (kExactMask - v);
                key[v] = c[v] == -INFINITY ? 0u : u;
            }
        } else {
            float top = -INFINITY;
#pragma unroll
            for (int v = 0; v < V; v++) top = fmaxf(top, c[v]);
            top = seg_max<L>(top);
            // scores span less than 2 unless a bias does more; values at or below the floor have key 0
            // and, where one of them is chosen, choose64 tells them apart and from masked ones
            // (the conversion makes 0 of what is negative, and of a NaN)
            constexpr float kSteps = (float)((1 << (32 - kIndex)) - 8);
            const float scale = by_logit ? kSteps / 16.f : kSteps / 2.f;
            odd |= !(fabsf(top) < 1e6f) && top > -INFINITY;
            eps = fminf(2.f * scale * (eps > 0.f ? eps + 0x1p-23f * fmaxf(fabsf(top), 1.f) : 0.f) + 5.f, 0x1p30f);
#pragma unroll
            for (int v = 0; v < V; v++) {
                uint32_t q;
                asm("v_cvt_u32_f32 %0, %1" : "=v"(q) : "v"(fmaf(c[v] - top, scale, kSteps)));
                key[v] = q << kIndex | (kIndexMask - v);
            }
        }
        uint32_t top[KP];
        seg_top<L, V, KP>(key, lane * V, top);
        const uint32_t near = (uint32_t)eps;        // keys of less distance do not tell the order
        uint32_t pairs = 0, last = 0;               // bit j: choices j - 1 and j are near; the last choice
        bool edge = false;                          // the best key that was not chosen is near the last
        if (!exact) {
#pragma unroll
            for (int j = 0; j < KP; j++) {
                const uint32_t q = top[j] >> kIndex;
                if (j < k) {
                    if (j) pairs |= (last >> kIndex) - q < near ? 1u << j : 0u;
                    odd |= q == 0;                  // at the floor, or no expert at all
                    last = top[j];
                }
            }
            uint32_t rest = 0;
            const uint32_t below = last + lane * V;
#pragma unroll
            for (int v = 0; v < V; v++) {
                const uint32_t x = key[v] < below ? key[v] : 0u;
                rest = x > rest ? x : rest;
            }
            rest = seg_reduce<L>(rest, Max());
            edge = (last >> kIndex) - (rest >> kIndex) < near;
        }
        odd = seg_reduce<L>((int)odd, Or()) != 0 && on;
        if (row && lane == 0) {
            // (odd rows' experts are choose64's)
            const uint32_t field = exact ? kExactMask : kIndexMask;
            uint32_t pair[KP / 2];
#pragma unroll
            for (int j = 0; j < KP; j += 2) {
                const uint32_t e = on && top[j] ? field - (top[j] & field) : 0xFFFFu;
                const uint32_t f = on && top[j + 1] ? field - (top[j + 1] & field) : 0xFFFFu;
                pair[j / 2] = e | f << 16;
            }
            __builtin_memcpy(__builtin_assume_aligned(chosen + i * KP, KP >= 8 ? 16 : 8), pair, sizeof(pair));
            if (exps) stat[i] = make_float2(m, sum);
        }
        if (__any((pairs || edge) && on && !odd)) {
            // Near ones of the same logit and bias are equal, and stand in the order of their indexes already
            // (16-bit logits and biases that move in steps make many of them); others make the row odd.
            wave_lds_sync();
            if (!on || odd) pairs = 0, edge = false;
            auto same = [&](int e, int f) {
                bool eq = one_logit(a, t, e) == one_logit(a, t, f);
                if (a.bias) eq = eq && bias[(e % V / kVec * L + e / V) * kVec + e % V % kVec] ==
                                           bias[(f % V / kVec * L + f / V) * kVec + f % V % kVec];
                return eq;
            };
            for (; pairs; pairs &= pairs - 1) {
                const int j = __builtin_ctz(pairs);
                if (!same(chosen[i * KP + j - 1], chosen[i * KP + j])) { odd = true; break; }
            }
            if (edge && !odd) {
                uint32_t close = 0;
                const uint32_t below = last + lane * V;
#pragma unroll
                for (int v = 0; v < V; v++)
                    close |= key[v] < below && (last >> kIndex) - (key[v] >> kIndex) < near ? 1u << v : 0u;
                const int e = chosen[i * KP + k - 1];
                for (; close; close &= close - 1) {
                    const int f = lane * V + __builtin_ctz(close);
                    if (f < E && !same(e, f)) { odd = true; break; }
                }
            }
            odd = seg_reduce<L>((int)odd, Or()) != 0;
        }
        if (odd && lane == 0) atomicOr(&odd_rows, 1ull << i);
    }
    __syncthreads();
    // the rows left, a wave each
    const int wave = threadIdx.x >> 6, wl = threadIdx.x & 63;
    const int odds = __popcll(odd_rows);
    double *row64 = room + (size_t)wave * (E + G);
    for (int n0 = wave; n0 < odds; n0 += kThreads / 64) {
        unsigned long long left = odd_rows;
        for (int n = 0; n < n0; n++) left &= left - 1;
        const int i = __ffsll(left) - 1;
        const int64_t t = t0 + i;
        constexpr int VX = (L * V + 63) / 64;
        float l[VX], bx[VX], m = -INFINITY;
        bool nan = false;
#pragma unroll
        for (int v = 0; v < VX; v++) {
            const int e = 64 * v + wl;
            l[v] = one_logit(a, t, e < E ? e : 0);
            bx[v] = a.bias && e < E ? bias[(e % V / kVec * L + e / V) * kVec + e % V % kVec] : 0.f;
        }
#pragma unroll
        for (int v = 0; v < VX; v++) {
            if (64 * v + wl >= E) l[v] = -INFINITY;
            nan |= l[v] != l[v];
            m = fmaxf(m, l[v]);
        }
        nan = __any(nan);
        m = seg_max<64>(m);
        double sum;
        const int my_e = choose64<VX>(a, by_logit, exps, wl, l, bx, m, sum, row64);
        if (wl < KP) chosen[i * KP + wl] = (uint16_t)(wl < k && my_e >= 0 ? my_e : 0xFFFF);
        if (wl == 0) {
            if (exps) stat[i] = make_float2(m, (float)sum);
            if (nan) atomicOr(&nan_rows, 1ull << i);
        }
    }
    __syncthreads();
    for (int x = threadIdx.x; x < nt * KP; x += kThreads) {
        const int i = x / KP, j = x % KP;
        const float2 ms = exps ? stat[i] : make_float2(0.f, 1.f);
        finish_slot<KP>(a, t0 + i, i, j, chosen[x], nan_rows >> i & 1, ms.x, ms.y, mask);
    }
    __syncthreads();
    if (a.mask) {
        for (int e = threadIdx.x; e < E; e += kThreads) a.mask[(int64_t)blockIdx.x * E + e] = mask[e];
        return;
    }
    // the only chunk: places at once
    int32_t *base = (int32_t *)(mask + E);
    for (int e = threadIdx.x; e < E; e += kThreads) base[e] = __popcll(mask[e]);
    __syncthreads();
    const int32_t total = scan_lds<kThreads>(base, E, scan_tmp);
    for (int e = threadIdx.x; e < E; e += kThreads) a.offsets[e] = base[e];
    if (threadIdx.x == 0) a.offsets[E] = total;
    place_chunk<kThreads>(a, t0, nt, mask, base, total, first);
}

// Rows of every expert in the chunks before each chunk, and in all chunks: a workgroup takes 8 experts,
// 128 threads of each over the chunks (two passes; the masks of the second come from L2).  Bound by the
// latency of those passes: 5.6 us for 1024 chunks of 256 experts (2 MB), 4 for 256 of 60.
__global__ __launch_bounds__(1024) void k_route_scan(const uint64_t *__restrict__ mask, int32_t *__restrict__ before,
                                                     int32_t *__restrict__ total, int64_t chunks, int E) {
    __shared__ int32_t part[8][129];
    const int x = threadIdx.x & 7, y = threadIdx.x >> 3, e = blockIdx.x * 8 + x;
    const int64_t per = (chunks + 127) / 128, lo = y * per, hi = lo + per < chunks ? lo + per : chunks;
    int32_t n = 0;
    if (e < E) {
#pragma unroll 8
        for (int64_t c = lo; c < hi; c++) n += __popcll(mask[c * E + e]);
    }
    part[x][y] = n;
    __syncthreads();
    // a wave per expert scans its 128 parts
    const int w = threadIdx.x >> 6, lane = threadIdx.x & 63;
    if (w < 8) {
        const int32_t p = part[w][2 * lane], q = part[w][2 * lane + 1];
        const int32_t incl = (int32_t)wave_incl_scan((uint32_t)(p + q));
        part[w][2 * lane] = incl - p - q;
        part[w][2 * lane + 1] = incl - q;
        if (lane == 63 && blockIdx.x * 8 + w < E) total[blockIdx.x * 8 + w] = incl;
    }
    __syncthreads();
    if (e < E) {
        n = part[x][y];
#pragma unroll 8
        for (int64_t c = lo; c < hi; c++) {
            const int32_t rows = __popcll(mask[c * E + e]);
            before[c * E + e] = n;
            n += rows;
        }
    }
}

// Places of one chunk's slots: the chunk's masks and sums, one scan over the experts, then a popcount a
// slot.  Bound by latency: 8 us for 65536 x 8 slots, 4 for 16381 x 4.  Without the sums of k_route_scan
// a workgroup counts all chunks itself.
__global__ __launch_bounds__(kPlaceThreads) void k_route_place(RouteArgs a, const int32_t *__restrict__ before,
                                                               const int32_t *__restrict__ totals) {
    extern __shared__ __align__(16) uint64_t lds[];
    __shared__ uint64_t scan_tmp[kPlaceThreads / 64];
    __shared__ uint32_t first[64];
    const int E = a.E;
    uint64_t *mask = lds;                       // [E]
    int32_t *base = (int32_t *)(mask + E);      // [E]
    const int64_t c = blockIdx.x, t0 = c * a.chunk;
    const int nt = (int)(a.T - t0 < a.chunk ? a.T - t0 : a.chunk);
    // exclusive sums over the experts: all their rows, and (high half) this chunk's predecessors' rows
    uint64_t run = 0;
    for (int e0 = 0; e0 < E; e0 += kPlaceThreads) {
        const int e = e0 + threadIdx.x;
        uint32_t all = 0, prev = 0;
        if (e < E) {
            mask[e] = a.mask[c * E + e];
            if (before) {
                all = (uint32_t)totals[e];
                prev = (uint32_t)before[c * E + e];
            } else {
#pragma unroll 8
                for (int64_t b = 0; b < gridDim.x; b++) {
                    const uint32_t n = __popcll(a.mask[b * E + e]);
                    all += n;
                    prev += b < c ? n : 0u;
                }
            }
        }
        uint64_t sum;
        const uint64_t pre = run + block_excl_scan<kPlaceThreads>((uint64_t)prev << 32 | all, scan_tmp, sum);
        run += sum;
        if (e < E) {
            base[e] = (int32_t)((uint32_t)pre + prev);
            if (c == 0) a.offsets[e] = (int32_t)(uint32_t)pre;
        }
    }
    const int32_t total = (int32_t)(uint32_t)run, used_all = (int32_t)(run >> 32);
    if (c == 0 && threadIdx.x == 0) a.offsets[E] = total;
    __syncthreads();
    // slots without an expert in the chunks before: all of theirs less the used ones
    place_chunk<kPlaceThreads>(a, t0, nt, mask, base, (int32_t)(total + t0 * a.k - used_all), first);
}

// dlogits of one row from the chosen slots' gradients: with a = w / scale,
//   softmax:                s_i * (scale * g_i [chosen] - sum scale * g_j * s_j)
//   softmax, renormalised:  scale * a_i * (g_i - sum g_j * a_j) at the chosen
//   sigmoid:                w_i * (1 - s_i) * g_i at the chosen (renormalised: g_i - sum g_j * a_j)
// L lanes a row; the slots' values go through LDS to the lanes that store them, so that the row leaves in
// wide stores.  Bound by writing every value, nearly all of them 0: 12.4 us for 65536 x 256 bf16 (33.6 MB).
constexpr int kGradThreads = 512;
template <typename T, int L, int V>
__global__ __launch_bounds__(kGradThreads) void k_route_grad(RouteArgs a, const float *__restrict__ dweights,
                                                              T *__restrict__ dlogits) {
    extern __shared__ __align__(16) uint64_t lds[];
    const int E = a.E, k = a.k;
    const int lane = threadIdx.x & (L - 1), seg = threadIdx.x / L;
    float *d = (float *)lds + (size_t)seg * (L * V);
    const bool full = a.score == 0 && !a.renorm;
    for (int64_t i0 = (int64_t)blockIdx.x * (kGradThreads / L); i0 < a.T;
         i0 += (int64_t)gridDim.x * (kGradThreads / L)) {
        const int64_t t = i0 + seg;
        const bool row = t < a.T;
        const int64_t tt = row ? t : 0;
        const T *lp = (const T *)a.logits + tt * a.ld;
        int e = -1;
        float w = 0.f, g = 0.f;
        if (row && lane < k) {
            e = a.experts[tt * k + lane];
            if (e >= 0) { w = a.weights[tt * k + lane]; g = dweights[tt * k + lane]; }
        }
        // (w / scale is exactly 1 for the only expert of a renormalised row, whose gradient is exactly 0)
        const float dot = seg_reduce<L>(g * (a.renorm ? w / a.scale : w), Sum());
        float x = w * (a.renorm ? g - dot : g);
        if (a.score == 1 && e >= 0) x *= a.slopes[tt * k + lane];
#pragma unroll
        for (int v = 0; v < V; v++) d[v * L + lane] = 0.f;
        wave_lds_sync();
        if (e >= 0) d[e] = x;
        wave_lds_sync();
        float o[V];
#pragma unroll
        for (int v = 0; v < V; v++) o[v] = d[lane * V + v];
        if (full) {
            float l[V];
            load(lp + lane * V, E - lane * V, l);
            float m = -INFINITY, sum = 0.f;
#pragma unroll
            for (int v = 0; v < V; v++)
                if (lane * V + v < E) m = fmaxf(m, l[v]);
            m = seg_max<L>(m);
            float s[V];
#pragma unroll
            for (int v = 0; v < V; v++) {
                s[v] = lane * V + v < E && l[v] != -INFINITY ? expf(l[v] - m) : 0.f;
                sum += s[v];
            }
            sum = seg_reduce<L>(sum, Sum());
            // (a row without an expert has dot 0, and its logits may hold anything; else a NaN makes dot one)
            const float f = dot != 0.f ? dot / sum : 0.f;
#pragma unroll
            for (int v = 0; v < V; v++)
                if (s[v] != 0.f && f != 0.f) o[v] -= s[v] * f;
        }
        if (row && lane * V < E) store(dlogits + t * E + lane * V, E - lane * V, o);
        wave_lds_sync();
    }
}

// ---- rows moved: gather, dispatch, combine -------------------------------------------------------
// L lanes of a 256-thread workgroup share one row (16, 32, 64 or all 256), eight columns a lane and step;
// gridDim.y workgroups share its columns where there are few rows.  A place outside the T * k rows (a
// plan that route did not make) is taken as a slot without an expert, and nothing is written there.
template <int L>
__device__ __forceinline__ int64_t first_row() {
    const int sub = L >= 64 ? __builtin_amdgcn_readfirstlane(threadIdx.x / L) : (int)threadIdx.x / L;
    return (int64_t)blockIdx.x * (256 / L) + sub;
}
template <int L> __device__ __forceinline__ int64_t row_step() { return (int64_t)gridDim.x * (256 / L); }
template <int L> __device__ __forceinline__ int64_t first_col() { return ((int64_t)blockIdx.y * L + threadIdx.x % L) * 8; }
template <int L> __device__ __forceinline__ int64_t col_step() { return (int64_t)gridDim.y * L * 8; }
// f(row, column of its eight values) over all of them; L = 0: a thread per eight values over rows and
// columns as one range, so that no lane of a narrow row is idle ((row, block) are stepped, not divided)
template <int L, typename F>
__device__ __forceinline__ void each8(int64_t rows, int64_t cols, F f) {
    if constexpr (L) {
        for (int64_t r = first_row<L>(); r < rows; r += row_step<L>())
            for (int64_t c = first_col<L>(); c < cols; c += col_step<L>()) f(r, c);
    } else {
        const uint32_t nb = (uint32_t)((cols + 7) / 8), at = blockIdx.x * 256 + threadIdx.x, step = gridDim.x * 256;
        const uint32_t dr = step / nb, db = step - dr * nb;
        int64_t r = at / nb;
        uint32_t b = at % nb;
        while (r < rows) {
            f(r, (int64_t)b * 8);
            r += dr;
            b += db;
            if (b >= nb) { b -= nb; r++; }
        }
    }
}

// out[r] = dropout(row base[order[f_r]] + off_r of the data).  Bound by memory, a row's index loads first:
// they are the same for the lanes of a row (scalar loads), and rows of other waves cover them.
// 65536 rows of 2048 bf16: 88 us (6.1 TB/s), of 2047 112.
template <typename T, int L, bool NT, bool WHOLE>
__global__ __launch_bounds__(256) void k_gather_drop(const T *__restrict__ data, T *__restrict__ out, int64_t rows,
                                                     int64_t cols, Drop d, RowGather g) {
    each8<L>(rows, cols, [&](int64_t r, int64_t c) {
        const int32_t f = g.fpos[r] < 0 ? -1 - g.fpos[r] : g.fpos[r];
        const T *x = data + (g.base[g.order[f]] + g.off[r]) * cols;
        const int64_t id = drop_row(d, r);
        const auto a = raw8<NT, WHOLE>(x, c, cols);
        Draw dr;
        if (d.drop) dr = draw8(d, id, (uint32_t)(c >> 3));      // while the values come
        float v[8];
        open8<T, WHOLE>(a, c, cols, v);
        if (d.drop) drop8<false>(d, dr, v, v);
        store8<NT, WHOLE>(out + r * cols, c, cols, v);
    });
}

// xs[pos[t, j]] = x[t].  Bound by the k writes of a row, which is read once (a gather by place would read
// it k times).  16384 rows of 4096 bf16 to 8 experts each: 247 us (4.9 TB/s).
template <typename T, int L>
__global__ __launch_bounds__(256) void k_dispatch(MoveArgs m, const T *__restrict__ x, int64_t ldx, T *__restrict__ xs) {
    const uint32_t places = (uint32_t)(m.T * m.k);
    each8<L>(m.T, m.D, [&](int64_t t, int64_t c) {
        const int32_t *e = m.experts + t * m.k, *pos = m.pos + t * m.k;
        float v[8];
        const float zero[8] = {0, 0, 0, 0, 0, 0, 0, 0};
        load8(x + t * ldx, c, m.D, v);
        for (int j = 0; j < m.k; j++) {
            if ((uint32_t)pos[j] >= places) continue;
            T *to = xs + (int64_t)pos[j] * m.D;
            if (e[j] >= 0) store8(to, c, m.D, v);
            else store8(to, c, m.D, zero);
        }
    });
}

// out[t] = residual[t] + dropout(sum of w[t, j] * y[pos[t, j]]), the gradient of k_dispatch without weights
// and residual.  Bound by the reads of k rows: KU of them are on their way at a time, and the Philox block
// is computed meanwhile.  16384 x 8 rows of 4096 bf16: 219 us (5.5 TB/s), with residual and dropout
// 242; 8194 x 8 of 4095 112 (5.4).  A slot without an expert is read like any other (its place is a row of
// y) and left out of the sum whatever it holds.
template <typename T, int L, int KU, bool NT>
__global__ __launch_bounds__(256) void k_combine(MoveArgs m, const T *__restrict__ y, const float *__restrict__ w,
                                                 const T *__restrict__ res, int64_t ldr, Drop d, T *__restrict__ out) {
    const uint32_t places = (uint32_t)(m.T * m.k);
    each8<L>(m.T, m.D, [&](int64_t t, int64_t c) {
        const int32_t *e = m.experts + t * m.k, *pos = m.pos + t * m.k;
        const int64_t id = d.drop ? drop_row(d, t) : 0;
        float acc[8] = {0, 0, 0, 0, 0, 0, 0, 0}, r[8] = {0, 0, 0, 0, 0, 0, 0, 0};
        if (res) load8<NT>(res + t * ldr, c, m.D, r);
        Draw dr;
        for (int j0 = 0; j0 < m.k; j0 += KU) {
            typename Pack<T, 8>::V raw[KU];
#pragma unroll
            for (int u = 0; u < KU; u++) {
                const int j = j0 + u < m.k ? j0 + u : j0;
                const uint32_t at = (uint32_t)pos[j] < places ? (uint32_t)pos[j] : 0u;
                raw[u] = raw8<NT>(y + (int64_t)at * m.D, c, m.D);
            }
            if (d.drop && j0 == 0) dr = draw8(d, id, (uint32_t)(c >> 3));   // while the rows come
#pragma unroll
            for (int u = 0; u < KU; u++) {
                const int j = j0 + u < m.k ? j0 + u : j0;
                const bool on = j0 + u < m.k && e[j] >= 0 && (uint32_t)pos[j] < places;
                const float wj = w ? w[t * m.k + j] : 1.f;
                float v[8];
                open8<T>(raw[u], c, m.D, v);
#pragma unroll
                for (int i = 0; i < 8; i++) acc[i] = on ? fmaf(wj, v[i], acc[i]) : acc[i];
            }
        }
        if (d.drop) {
            drop8<true>(d, dr, acc, r);
        } else if (res) {
#pragma unroll
            for (int i = 0; i < 8; i++) acc[i] += r[i];
        }
        store8<NT>(out + t * m.D, c, m.D, acc);
    });
}

// One pass over g = dropout(dout): KU products with rows of y and KU rows of dy at a time.  The lanes
// of a row hold partial products of all its slots; they are joined after the last column.  Bound by the
// k rows read and k written of a row.  16384 x 8 x 4096 bf16: 473 us (4.8 TB/s; a plain copy 4.95).
template <typename T, int L, int KM, bool NT>
__global__ __launch_bounds__(256) void k_combine_grad(MoveArgs m, const int32_t *__restrict__ experts,
                                                      const int32_t *__restrict__ places, const T *__restrict__ dout, int64_t ldo,
                                                      const T *__restrict__ y, const float *__restrict__ w, Drop d,
                                                      T *__restrict__ dy, float *__restrict__ dw) {
    constexpr int KU = KM < 8 ? KM : 8;
    const uint32_t rows = (uint32_t)(m.T * m.k);
    __shared__ float part[L > 64 ? 4 : 1][KM];
    for (int64_t t = first_row<L>(); t < m.T; t += row_step<L>()) {
        const int64_t id = d.drop ? drop_row(d, t) : 0;
        float dot[KM], wt[KM];
        int32_t pos[KM];
        bool on[KM], in[KM];
#pragma unroll
        for (int j = 0; j < KM; j++) {
            const int64_t slot = t * m.k + (j < m.k ? j : 0);
            const uint32_t at = (uint32_t)places[slot];
            on[j] = experts[slot] >= 0 && at < rows;
            in[j] = at < rows;
            pos[j] = at < rows ? (int32_t)at : 0;
            wt[j] = w[slot];
            dot[j] = 0.f;
        }
        for (int64_t c = first_col<L>(); c < m.D; c += col_step<L>()) {
            float g[8];
            load8(dout + t * ldo, c, m.D, g);
            if (d.drop) drop8<false>(d, draw8(d, id, (uint32_t)(c >> 3)), g, g);
#pragma unroll
            for (int j0 = 0; j0 < KM; j0 += KU) {
                if (j0 >= m.k) break;
                if (dw) {
                    typename Pack<T, 8>::V raw[KU];
#pragma unroll
                    for (int u = 0; u < KU; u++) raw[u] = raw8<NT>(y + (int64_t)pos[j0 + u] * m.D, c, m.D);
#pragma unroll
                    for (int u = 0; u < KU; u++) {
                        float v[8];
                        open8<T>(raw[u], c, m.D, v);
#pragma unroll
                        for (int i = 0; i < 8; i++) dot[j0 + u] = fmaf(g[i], v[i], dot[j0 + u]);
                    }
                }
                if (dy) {
#pragma unroll
                    for (int u = 0; u < KU; u++) {
                        if (j0 + u >= m.k) break;
                        if (!in[j0 + u]) continue;
                        float o[8];
#pragma unroll
                        for (int i = 0; i < 8; i++) o[i] = on[j0 + u] ? wt[j0 + u] * g[i] : 0.f;
                        store8(dy + (int64_t)pos[j0 + u] * m.D, c, m.D, o);
                    }
                }
            }
        }
        if (!dw) continue;
#pragma unroll
        for (int j = 0; j < KM; j++) dot[j] = seg_reduce<(L < 64 ? L : 64)>(dot[j], Sum());
        if (L > 64) {
            __syncthreads();
            if ((threadIdx.x & 63) == 0)
#pragma unroll
                for (int j = 0; j < KM; j++) part[threadIdx.x >> 6][j] = dot[j];
            __syncthreads();
            const int j = threadIdx.x;
            if (j < m.k) dw[t * m.k + j] = experts[t * m.k + j] >= 0 && (uint32_t)places[t * m.k + j] < rows ? (part[0][j] + part[1][j]) + (part[2][j] + part[3][j]) : 0.f;
        } else {
#pragma unroll
            for (int j = 0; j < KM; j++)
                if ((threadIdx.x & (L - 1)) == (j & (L - 1)) && j < m.k) dw[t * m.k + j] = on[j] ? dot[j] : 0.f;
        }
    }
}

template <typename F>
hipError_t by_type(int32_t dtype, F f) {
    switch (dtype) {
        case 0: f((float *)nullptr); break;
        case 1: f((__bf16 *)nullptr); break;
        case 2: f((_Float16 *)nullptr); break;
        default: return hipErrorInvalidValue;
    }
    return hipGetLastError();
}

// Lanes and values per lane of a row of E experts.  Up to 64 experts and many rows: 4 lanes, whose own
// sorting networks do more of the work (123580 rows, 36 experts in groups, with gradient: 71 -> 50 us);
// few rows rather take 16 for their latency.  V <= E: a lane past the end reads the row's last V values.
template <typename F>
void by_width(int E, int64_t T, F f) {
    using std::integral_constant;
    if (E >= 4 && E <= 64 && T > 8192) {
        if (E <= 16) f(integral_constant<int, 4>(), integral_constant<int, 4>());
        else if (E <= 32) f(integral_constant<int, 4>(), integral_constant<int, 8>());
        else f(integral_constant<int, 4>(), integral_constant<int, 16>());
    } else if (E <= 16) f(integral_constant<int, 16>(), integral_constant<int, 1>());
    else if (E <= 32) f(integral_constant<int, 16>(), integral_constant<int, 2>());
    else if (E <= 64) f(integral_constant<int, 16>(), integral_constant<int, 4>());
    else if (E <= 128) f(integral_constant<int, 16>(), integral_constant<int, 8>());
    else if (E <= 256) f(integral_constant<int, 16>(), integral_constant<int, 16>());
    else if (E <= 512) f(integral_constant<int, 64>(), integral_constant<int, 8>());
    else f(integral_constant<int, 64>(), integral_constant<int, 16>());
}

}  // namespace

// Whether a pass over so many bytes goes past the caches: beyond the 256 MB of the Infinity Cache
// nothing of it can be found there later.  Measured past / through, in one run each: dropout 16384 x 8192 bf16 with
// residual 131 / 157 us, without 91 / 98; fp32 without 224 / 204, so that it goes through them; gather of
// 65536 x 2048 bf16 99 / 125; combine of 16384 x 8 x 4096 bf16 233 / 281; combine of 2039 x 3 x 1001 fp16
// (17 MB) 7.8 / 7.4; the reads of y of the combine's gradient (16384 x 8 x 4096) 480 / 495.  Rows written
// for one read are slower past them (dispatch 249 / 223, the gradient's writes 525 / 495).
static bool past_caches(int64_t bytes) { return bytes > ((int64_t)256 << 20); }

template <typename F>
static void by_flag(bool b, F f) {
    if (b) f(std::true_type());
    else f(std::false_type());
}

// Lanes of a row of `cols` values, and the launch of `rows` such rows.  256 lanes where two thirds of them
// have work (dispatch and combine of 8 rows of 20000 tokens, 256 / 64 lanes: 1030 bf16 216 / 208 us, 1400
// 226 / 273, 2047 of 16384 298 / 335) and the row has `wide` blocks of eight.  Gather's loads of its
// indexes come before a row's values, and 64 lanes in steps wait for them once, which is what counts for
// the fewer bytes of 16-bit rows of up to 256 blocks (65536 rows of bf16, 256 / 64 lanes: 1368 88 / 79,
// 1449 143 / 96, 1920 98 / 94, 2047 170 / 121, 2048 100 / 98; the one range that loses is 2000 to 2040 in
// whole blocks, 104 / 121; from 2049 on even, 3584 162 / 177), not for 32 bits (32768 rows: 1536 87 / 97,
// 1921 117 / 128, 2047 121 / 135, 2048 110 / 126, 4096 232 / 252).
template <typename F>
static void by_row(int64_t rows, int64_t cols, int64_t wide, F f) {
    const int64_t blocks = (cols + 7) / 8, all = (blocks + 255) / 256 * 256;
    const int L = blocks <= 16 ? 16 : blocks <= 32 ? 32 : blocks < wide || 3 * blocks < 2 * all ? 64 : 256;
    int64_t x = (rows + 256 / L - 1) / (256 / L), y = 1;
    if (x < 2048) {      // few rows: their columns over several workgroups
        y = (cols + L * 8 - 1) / (L * 8);
        if (y > 2048 / x) y = 2048 / x;
        if (y < 1) y = 1;
    }
    const dim3 grid((unsigned)(x < (1 << 20) ? x : 1 << 20), (unsigned)y);
    if (L == 16) f(std::integral_constant<int, 16>(), grid);
    else if (L == 32) f(std::integral_constant<int, 32>(), grid);
    else if (L == 64) f(std::integral_constant<int, 64>(), grid);
    else f(std::integral_constant<int, 256>(), grid);
}

// The same where a row's lanes need not meet: rows of less than `narrow` values as one range of blocks.
// Row by row / as one range: gather of 65536 rows of 130 bf16 24 / 17 us, 300 39 / 26, 515 51 / 35,
// 1000 53 / 63;
// combine of 8 rows of 72 of 466000 tokens 285 / 201, 130 of 258000 328 / 223, 200 of 168000 209 / 174,
// 300 of 32768 (with its dispatch) 106 / 117.  Dispatch is no faster so (128: 134 / 150, 200: 188 / 197).
template <typename F>
static void by_block(int64_t rows, int64_t cols, int64_t narrow, int64_t wide, F f) {
    if (cols >= narrow) return by_row(rows, cols, wide, f);
    const int64_t x = (rows * ((cols + 7) / 8) + 255) / 256;
    f(std::integral_constant<int, 0>(), dim3((unsigned)(x < 8192 ? x : 8192)));
}

template <typename F>
static void by_slots(int k, F f) {
    if (k <= 1) f(std::integral_constant<int, 1>());
    else if (k <= 2) f(std::integral_constant<int, 2>());
    else if (k <= 4) f(std::integral_constant<int, 4>());
    else if (k <= 8) f(std::integral_constant<int, 8>());
    else f(std::integral_constant<int, 16>());
}

hipError_t launch_dropout(const void *x, int64_t ldx, const void *residual, int64_t ldr, void *y, int64_t rows,
                          int64_t cols, int32_t dtype, const Drop &d, hipStream_t s) {
    if (rows <= 0 || cols <= 0) return hipSuccess;
    const int64_t nb = (cols + 7) / 8, n = rows * nb;
    const int64_t blocks = (n + 255) / 256;
    const dim3 grid((unsigned)(blocks < 8192 ? blocks : 8192));
    return by_type(dtype, [&](auto *p) {
        using T = std::remove_pointer_t<decltype(p)>;
        by_flag((residual || sizeof(T) == 2) && past_caches(rows * cols * (int64_t)sizeof(T) * (residual ? 3 : 2)), [&](auto NT) {
            by_flag(residual != nullptr, [&](auto RES) {
                by_flag(cols % 8 == 0, [&](auto WHOLE) {
                    hipLaunchKernelGGL((k_dropout<T, decltype(RES)::value, decltype(NT)::value, decltype(WHOLE)::value>),
                                       grid, dim3(256), 0, s, (const T *)x, ldx, (const T *)residual, ldr, (T *)y, rows,
                                       cols, (uint32_t)nb, d);
                });
            });
        });
    });
}

hipError_t launch_gather_dropout(const void *data, void *out, int64_t rows, int64_t cols, int32_t dtype, const Drop &d,
                                 const RowGather &g, hipStream_t s) {
    if (rows <= 0 || cols <= 0) return hipSuccess;
    return by_type(dtype, [&](auto *p) {
        using T = std::remove_pointer_t<decltype(p)>;
        by_block(rows, cols, 640, sizeof(T) == 2 ? 257 : 0, [&](auto L, dim3 grid) {
            by_flag(past_caches(2 * rows * cols * (int64_t)sizeof(T)), [&](auto NT) {
                by_flag(cols % 8 == 0, [&](auto WHOLE) {
                    hipLaunchKernelGGL((k_gather_drop<T, decltype(L)::value, decltype(NT)::value, decltype(WHOLE)::value>),
                                       grid, dim3(256), 0, s, (const T *)data, (T *)out, rows, cols, d, g);
                });
            });
        });
    });
}

hipError_t launch_route(const RouteArgs &a, hipStream_t s) {
    const int64_t chunks = route_chunks(a.T, a.E);
    const int S = a.E / a.groups;
    hipError_t err = hipSuccess;
    by_width(a.E, a.T, [&](auto L, auto V) {
        constexpr int kThreads = decltype(L)::value == 4 ? 256 : 512;
        // masks; the bases (one chunk); the groups' keys and, for groups of no power of two, the values of
        // every row at once; or a row's values and its groups' in 64 bits for every wave
        const size_t rows = kThreads / decltype(L)::value, E = a.E, G = a.groups;
        size_t room = 4 * E;
        if (G > 1) room = std::max(std::max(room, kThreads / 64 * 8 * (E + G)), rows * 4 * ((G + 3) / 4 * 4 + (S & (S - 1) ? (size_t)(L * V) : 0)));
        const size_t lds = 8 * ((E + 1) / 2 * 2) + room;
        if (decltype(V)::value > a.E || decltype(L)::value * decltype(V)::value < a.E) {
            err = hipErrorInvalidValue;     // (no width does)
            return;
        }
        auto go = [&](auto KP) {
            const auto kern = k_route<decltype(L)::value, decltype(V)::value, decltype(KP)::value, kThreads>;
            if (lds > 64 * 1024)
                err = hipFuncSetAttribute((const void *)kern, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
            if (err == hipSuccess) hipLaunchKernelGGL(kern, dim3((unsigned)chunks), dim3(kThreads), lds, s, a);
        };
        if (a.k <= 4) go(std::integral_constant<int, 4>());
        else if (a.k <= 8) go(std::integral_constant<int, 8>());
        else go(std::integral_constant<int, 16>());
    });
    if (err == hipSuccess) err = hipGetLastError();
    if (err != hipSuccess || !a.mask) return err;
    // few chunks: every workgroup of the last kernel sums them, one launch less
    // (a call with 2048 rows and 64 experts 11.4 us, with 2049 rows 14.1)
    const bool sums = chunks > 32;
    if (sums)
        hipLaunchKernelGGL(k_route_scan, dim3((unsigned)((a.E + 7) / 8)), dim3(1024), 0, s, a.mask, a.before, a.totals,
                           chunks, a.E);
    hipLaunchKernelGGL(k_route_place, dim3((unsigned)chunks), dim3(kPlaceThreads), 12 * (size_t)a.E, s, a,
                       sums ? a.before : nullptr, a.totals);
    return hipGetLastError();
}

hipError_t launch_route_grad(const RouteArgs &a, const float *dweights, void *dlogits, hipStream_t s) {
    if (a.T <= 0) return hipSuccess;
    return by_type(a.dtype, [&](auto *p) {
        using T = std::remove_pointer_t<decltype(p)>;
        by_width(a.E, 0, [&](auto L, auto V) {
            if constexpr (decltype(L)::value >= 16) {       // (a lane for each of up to 16 slots)
                const int64_t blocks = (a.T + kGradThreads / L - 1) / (kGradThreads / L);
                hipLaunchKernelGGL((k_route_grad<T, decltype(L)::value, decltype(V)::value>),
                                   dim3((unsigned)(blocks < 4096 ? blocks : 4096)), dim3(kGradThreads),
                                   4 * (size_t)kGradThreads * V, s, a, dweights, (T *)dlogits);
            }
        });
    });
}

hipError_t launch_dispatch(const MoveArgs &m, const void *x, int64_t ldx, void *xs, hipStream_t s) {
    if (m.T <= 0 || m.D <= 0) return hipSuccess;
    return by_type(m.dtype, [&](auto *p) {
        using T = std::remove_pointer_t<decltype(p)>;
        by_row(m.T, m.D, 0, [&](auto L, dim3 grid) {
            hipLaunchKernelGGL((k_dispatch<T, decltype(L)::value>), grid, dim3(256), 0, s, m, (const T *)x, ldx, (T *)xs);
        });
    });
}

hipError_t launch_combine(const MoveArgs &m, const void *y, const float *w, const void *residual, int64_t ldr,
                          const Drop &d, void *out, hipStream_t s) {
    if (m.T <= 0 || m.D <= 0) return hipSuccess;
    return by_type(m.dtype, [&](auto *p) {
        using T = std::remove_pointer_t<decltype(p)>;
        by_block(m.T, m.D, 257, 0, [&](auto L, dim3 grid) {
            by_slots(m.k < 8 ? m.k : 8, [&](auto KU) {
                by_flag(past_caches(m.T * (m.k + 2) * m.D * (int64_t)sizeof(T)), [&](auto NT) {
                    hipLaunchKernelGGL((k_combine<T, decltype(L)::value, decltype(KU)::value, decltype(NT)::value>), grid,
                                       dim3(256), 0, s, m, (const T *)y, w, (const T *)residual, ldr, d, (T *)out);
                });
            });
        });
    });
}

hipError_t launch_combine_grad(const MoveArgs &m, const void *dout, int64_t ldo, const void *y, const float *w,
                               const Drop &d, void *dy, float *dw, hipStream_t s) {
    if (m.T <= 0) return hipSuccess;
    return by_type(m.dtype, [&](auto *p) {
        using T = std::remove_pointer_t<decltype(p)>;
        by_row(m.T, m.D, 0, [&](auto L, dim3 grid) {
            grid.y = 1;     // the products run over all columns
            by_slots(m.k, [&](auto KM) {
                by_flag(past_caches(m.T * (2 * m.k + 1) * m.D * (int64_t)sizeof(T)), [&](auto NT) {
                    hipLaunchKernelGGL((k_combine_grad<T, decltype(L)::value, decltype(KM)::value, decltype(NT)::value>),
                                       grid, dim3(256), 0, s, m, m.experts, m.pos, (const T *)dout, ldo, (const T *)y,
                                       w, d, (T *)dy, dw);
                });
            });
        });
    });
}

}  // namespace pss
