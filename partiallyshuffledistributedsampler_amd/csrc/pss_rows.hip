// pss_rows.hip -- what a batch's rows go through after the sampler picked them: dropout keyed by
// row ids, routing to experts, dispatch into expert order and combination by weight (pss_rows.h).
#include <math.h>

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

// NT: past the caches (nontemporal)
template <bool NT = false, typename T, int N>
__device__ __forceinline__ void load(const T *p, int64_t left, float (&v)[N]) {
    if (left >= N) {
        typedef typename Pack<T, N>::V V;
        const V a = NT ? __builtin_nontemporal_load((const V *)p) : *(const V *)p;
#pragma unroll
        for (int i = 0; i < N; i++) v[i] = Value<T>::up(at(a, i));
    } else {
#pragma unroll
        for (int i = 0; i < N; i++) v[i] = i < left ? Value<T>::up(p[i]) : 0.f;
    }
}

template <bool NT = false, typename T, int N>
__device__ __forceinline__ void store(T *p, int64_t left, const float (&v)[N]) {
    if (left >= N) {
        if constexpr (N == 1) {
            *p = Value<T>::down(v[0]);
        } else {
            typename Pack<T, N>::V a;
#pragma unroll
            for (int i = 0; i < N; i++) a[i] = Value<T>::down(v[i]);
            if (NT) __builtin_nontemporal_store(a, (typename Pack<T, N>::V *)p);
            else *(typename Pack<T, N>::V *)p = a;
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; i++)
            if (i < left) p[i] = Value<T>::down(v[i]);
    }
}

// ---- dropout -------------------------------------------------------------------------------------
__device__ __forceinline__ int64_t drop_row(const Drop &d, int64_t i) {
    if (!d.ids) return d.row0 + i;
    return d.row0 + (d.per_row ? d.ids[i] : d.ids[0] + i);
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

// One thread per block of 8 columns, walking over (row, block) without a division per step.
template <typename T, bool RES, bool NT>
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
        const int64_t c = (int64_t)b * 8, left = cols - c;
        float v[8];
        load<NT>(x + row * ldx + c, left, v);
        float r[8];
        if (RES) load<NT>(res + row * ldr + c, left, r);
        if (d.drop) {
            drop8<RES>(d, draw8(d, drop_row(d, row), b), v, r);
        } else if (RES) {
#pragma unroll
            for (int i = 0; i < 8; i++) v[i] += r[i];
        }
        store<NT>(y + row * cols + c, left, v);
        row += drow;
        b += db;
        if (b >= nb) { b -= nb; row++; }
    }
}

// ---- routing -------------------------------------------------------------------------------------
// The lanes of a segment (16 or 64 of a wave) share one row; reductions stay inside the segment.
template <int L, typename T, typename F>
__device__ __forceinline__ T seg_reduce(T v, F f) {
#pragma unroll
    for (int m = L / 2; m; m >>= 1) v = f(v, __shfl_xor(v, m, 64));
    return v;
}

__device__ __forceinline__ void wave_lds_sync() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

constexpr double kDead = -INFINITY;   // an expert that cannot be chosen
constexpr double kLast = -1e300;      // a live one whose choice value is no number: after all others

// Places of a chunk's slots: rows of an expert in the order of the rows (bits of `mask`, one per
// row of the chunk), slots without an expert after all experts' rows.
__device__ __forceinline__ int32_t rank_in_chunk(const uint64_t *mask, int E, int e, int t) {
    const int w = t >> 6;
    int n = 0;
    for (int i = 0; i < w; i++) n += __popcll(mask[i * E + e]);
    return n + __popcll(mask[w * E + e] & ((1ull << (t & 63)) - 1));
}

constexpr int kRouteThreads = 512;
constexpr int kWords = kRouteChunk / 64;

// Places of one chunk from its masks, the expert bases and the rows' slot counts; all threads.
__device__ __forceinline__ void place_chunk(const RouteArgs &a, int64_t t0, int nt, const uint64_t *mask,
                                            const int32_t *base, int32_t unused0, uint32_t *scan_tmp) {
    // the chunk's slots without an expert, in order
    const int t = threadIdx.x;
    uint32_t un = 0;
    if (t < nt)
        for (int j = 0; j < a.k; j++) un += a.experts[(t0 + t) * a.k + j] < 0;
    uint32_t total;
    uint32_t at = block_excl_scan<kRouteThreads>(un, scan_tmp, total);
    if (t < nt) {
        for (int j = 0; j < a.k; j++) {
            const int64_t slot = (t0 + t) * a.k + j;
            const int e = a.experts[slot];
            const int32_t p = e < 0 ? unused0 + (int32_t)at++ : base[e] + rank_in_chunk(mask, a.E, e, t);
            a.pos[slot] = p;
            a.src[p] = (int32_t)slot;
        }
    }
}

// Exclusive scan of v[0, E) in LDS by all threads; returns the total.
__device__ __forceinline__ int32_t scan_lds(int32_t *v, int E, uint32_t *scan_tmp) {
    uint32_t run = 0;
    for (int e0 = 0; e0 < E; e0 += kRouteThreads) {
        const int e = e0 + threadIdx.x;
        uint32_t total;
        const uint32_t x = e < E ? (uint32_t)v[e] : 0u;
        const uint32_t pre = block_excl_scan<kRouteThreads>(x, scan_tmp, total);
        if (e < E) v[e] = (int32_t)(run + pre);
        run += total;
    }
    __syncthreads();
    return (int32_t)run;
}

template <typename T, int L, int V>
__global__ __launch_bounds__(kRouteThreads) void k_route(RouteArgs a) {
    extern __shared__ uint64_t lds[];
    __shared__ uint32_t scan_tmp[kRouteThreads / 64];
    const int E = a.E, k = a.k, G = a.groups;
    uint64_t *mask = lds;                                             // [kWords][E]
    double *choice = (double *)(mask + (size_t)kWords * E);           // [segments][E] (groups)
    const int lane = threadIdx.x & (L - 1), seg = threadIdx.x / L;
    const int64_t t0 = (int64_t)blockIdx.x * kRouteChunk;
    const int nt = (int)(a.T - t0 < kRouteChunk ? a.T - t0 : kRouteChunk);
    for (int i = threadIdx.x; i < kWords * E; i += kRouteThreads) mask[i] = 0;
    __syncthreads();
    for (int i0 = 0; i0 < kRouteChunk; i0 += kRouteThreads / L) {
        if (i0 >= nt) break;
        const int i = i0 + seg;
        const bool row = i < nt;
        const int64_t t = t0 + (row ? i : 0);
        const T *lp = (const T *)a.logits + t * a.ld;
        const bool on = row && (!a.valid || a.valid[t]);
        float l[V];
        load(lp + lane * V, E - lane * V, l);
        // row statistics of the softmax
        bool nan = false;
        float m = -INFINITY;
#pragma unroll
        for (int v = 0; v < V; v++)
            if (lane * V + v < E) { nan |= l[v] != l[v]; m = fmaxf(m, l[v]); }
        nan = seg_reduce<L>((int)nan, [](int x, int y) { return x | y; });
        m = seg_reduce<L>(m, [](float x, float y) { return fmaxf(x, y); });
        double sum = 1.0;
        if (a.score == 0) {
            sum = 0.0;
#pragma unroll
            for (int v = 0; v < V; v++)
                if (lane * V + v < E && l[v] != -INFINITY) sum += exp((double)l[v] - (double)m);
            sum = seg_reduce<L>(sum, [](double x, double y) { return x + y; });
        }
        // choice values
        const bool by_logit = !a.bias && (G == 1 || a.group_sum == 1);
        double c[V];
#pragma unroll
        for (int v = 0; v < V; v++) {
            const int e = lane * V + v;
            c[v] = kDead;
            if (e < E && on && l[v] != -INFINITY) {
                double x = (double)l[v];
                if (!by_logit) {
                    x = a.score == 0 ? exp(x - (double)m) / sum : 1.0 / (1.0 + exp(-x));
                    if (a.bias) x += (double)a.bias[e];
                }
                c[v] = x >= kLast ? x : kLast;
            }
        }
        if (G > 1) {
            const int S = E / G;
            double *mine = choice + (size_t)seg * E;
#pragma unroll
            for (int v = 0; v < V; v++)
                if (lane * V + v < E) mine[lane * V + v] = c[v];
            wave_lds_sync();
            double gs[kRouteMaxGroups / 16];
            for (int n = 0, g = lane; g < G; n++, g += L) {
                double b1 = kDead, b2 = kDead;
                for (int s = 0; s < S; s++) {
                    const double x = mine[g * S + s];
                    if (x > b1) { b2 = b1; b1 = x; }
                    else if (x > b2) b2 = x;
                }
                if (a.group_sum == 2 && b2 > kDead) b1 += b2;
                gs[n] = b1;
            }
            wave_lds_sync();
            for (int n = 0, g = lane; g < G; n++, g += L) mine[g] = gs[n];
            wave_lds_sync();
            uint64_t kept = 0;      // groups kept: fewer than top_groups come before them
            for (int g = lane; g < G; g += L) {
                const double x = mine[g];
                int before = 0;
                for (int o = 0; o < G; o++) before += mine[o] > x || (mine[o] == x && o < g);
                if (before < a.top_groups) kept |= 1ull << g;
            }
            kept = seg_reduce<L>(kept, [](uint64_t x, uint64_t y) { return x | y; });
            wave_lds_sync();
#pragma unroll
            for (int v = 0; v < V; v++) {
                const int e = lane * V + v;
                if (e < E && !((kept >> (e / S)) & 1)) c[v] = kDead;
            }
        }
        // the k best, ties to the lowest index; lane j keeps the j-th
        int my_e = -1;
        for (int j = 0; j < k; j++) {
            double best = kDead;
            int be = 1 << 20;
#pragma unroll
            for (int v = 0; v < V; v++)
                if (c[v] > best) { best = c[v]; be = lane * V + v; }
#pragma unroll
            for (int s = L / 2; s; s >>= 1) {
                const double ob = __shfl_xor(best, s, 64);
                const int oe = __shfl_xor(be, s, 64);
                if (ob > best || (ob == best && oe < be)) { best = ob; be = oe; }
            }
            if (lane == j) my_e = best > kDead ? be : -1;
#pragma unroll
            for (int v = 0; v < V; v++)
                if (lane * V + v == be) c[v] = kDead;
        }
        // weights: softmax as exp(l - max) / sum, renormalised over the chosen alone; the chosen
        // sigmoids' ratio from their logarithms, which neither under- nor overflow
        float w = 0.f;
        const bool used = my_e >= 0 && lane < k;
        const float lw = used ? Value<T>::up(lp[my_e]) : -INFINITY;
        if (a.renorm) {
            const float z = !used ? -INFINITY : a.score == 0 ? lw : fminf(lw, 0.f) - log1pf(expf(-fabsf(lw)));
            const float zm = seg_reduce<L>(z, [](float x, float y) { return fmaxf(x, y); });
            w = used ? expf(z - zm) : 0.f;
            const float ws = seg_reduce<L>(w, [](float x, float y) { return x + y; });
            w = used ? w / ws * a.scale : 0.f;
        } else if (used) {
            w = a.scale * (a.score == 0 ? expf(lw - m) / (float)sum : 1.f / (1.f + expf(-lw)));
        }
        if (used && nan) w = NAN;
        if (row && lane < k) {
            a.experts[t * k + lane] = my_e;
            a.weights[t * k + lane] = w;
            if (my_e >= 0) atomicOr((unsigned long long *)&mask[(i >> 6) * E + my_e], 1ull << (i & 63));
        }
    }
    __syncthreads();
    if (a.hist) {
        for (int e = threadIdx.x; e < E; e += kRouteThreads) {
            int n = 0;
            for (int w = 0; w < kWords; w++) n += __popcll(mask[w * E + e]);
            a.hist[(int64_t)blockIdx.x * E + e] = (uint16_t)n;
        }
        return;
    }
    // the only chunk: places at once
    int32_t *base = (int32_t *)(mask + (size_t)kWords * E);
    for (int e = threadIdx.x; e < E; e += kRouteThreads) {
        int n = 0;
        for (int w = 0; w < kWords; w++) n += __popcll(mask[w * E + e]);
        base[e] = n;
    }
    __syncthreads();
    const int32_t total = scan_lds(base, E, scan_tmp);
    for (int e = threadIdx.x; e < E; e += kRouteThreads) a.offsets[e] = base[e];
    if (threadIdx.x == 0) a.offsets[E] = total;
    place_chunk(a, t0, nt, mask, base, total, scan_tmp);
}

// Places of every chunk: each workgroup sums the chunks' counts before its own and in all.
__global__ __launch_bounds__(kRouteThreads) void k_route_place(RouteArgs a, int64_t chunks) {
    extern __shared__ uint64_t lds[];
    __shared__ uint32_t scan_tmp[kRouteThreads / 64];
    const int E = a.E, k = a.k;
    uint64_t *mask = lds;                                    // [kWords][E]
    int32_t *base = (int32_t *)(mask + (size_t)kWords * E);  // [E] all counts, then the bases
    int32_t *prev = base + E;                                // [E] counts of the chunks before
    const int64_t c = blockIdx.x, t0 = c * kRouteChunk;
    const int nt = (int)(a.T - t0 < kRouteChunk ? a.T - t0 : kRouteChunk);
    for (int i = threadIdx.x; i < kWords * E; i += kRouteThreads) mask[i] = 0;
    for (int e = threadIdx.x; e < 2 * E; e += kRouteThreads) base[e] = 0;
    __syncthreads();
    // threads share the experts; with few experts several threads share one, over the chunks
    const int per = E >= kRouteThreads ? 1 : kRouteThreads / E;
    const int part = E >= kRouteThreads ? 0 : threadIdx.x / E;
    if (part < per) {
        for (int e = E >= kRouteThreads ? threadIdx.x : threadIdx.x % E; e < E; e += kRouteThreads) {
            int32_t before = 0, all = 0;
            for (int64_t b = part; b < chunks; b += per) {
                const int32_t n = a.hist[b * E + e];
                all += n;
                before += b < c ? n : 0;
            }
            atomicAdd(&base[e], all);
            atomicAdd(&prev[e], before);
        }
    }
    for (int i = threadIdx.x; i < nt * k; i += kRouteThreads) {
        const int e = a.experts[t0 * k + i], t = i / k;
        if (e >= 0) atomicOr((unsigned long long *)&mask[(t >> 6) * E + e], 1ull << (t & 63));
    }
    __syncthreads();
    const int32_t total = scan_lds(base, E, scan_tmp);
    if (c == 0) {
        for (int e = threadIdx.x; e < E; e += kRouteThreads) a.offsets[e] = base[e];
        if (threadIdx.x == 0) a.offsets[E] = total;
    }
    // slots without an expert in the chunks before
    uint32_t used = 0, used_all;
    for (int e = threadIdx.x; e < E; e += kRouteThreads) used += prev[e];
    block_excl_scan<kRouteThreads>(used, scan_tmp, used_all);
    __syncthreads();
    for (int e = threadIdx.x; e < E; e += kRouteThreads) base[e] += prev[e];
    __syncthreads();
    place_chunk(a, t0, nt, mask, base, (int32_t)(total + t0 * k - used_all), scan_tmp);
}

// dlogits of one row from the chosen slots' gradients: with a = w / scale,
//   softmax:                s_i * (scale * g_i [chosen] - sum scale * g_j * s_j)
//   softmax, renormalised:  scale * a_i * (g_i - sum g_j * a_j) at the chosen
//   sigmoid:                w_i * (1 - s_i) * g_i at the chosen (renormalised: g_i - sum g_j * a_j)
template <typename T, int L, int V>
__global__ __launch_bounds__(kRouteThreads) void k_route_grad(RouteArgs a, const float *__restrict__ dweights,
                                                              T *__restrict__ dlogits) {
    extern __shared__ uint64_t lds[];
    const int E = a.E, k = a.k;
    const int lane = threadIdx.x & (L - 1), seg = threadIdx.x / L;
    float *d = (float *)lds + (size_t)seg * (L * V);
    const bool full = a.score == 0 && !a.renorm;
    for (int64_t i0 = (int64_t)blockIdx.x * (kRouteThreads / L); i0 < a.T;
         i0 += (int64_t)gridDim.x * (kRouteThreads / L)) {
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
        const float dot = seg_reduce<L>(g * w, [](float x, float y) { return x + y; });
        float x = w * (a.renorm ? g - dot / a.scale : g);
        if (a.score == 1 && e >= 0) x /= 1.f + expf(Value<T>::up(lp[e]));
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
            m = seg_reduce<L>(m, [](float p, float q) { return fmaxf(p, q); });
            float s[V];
#pragma unroll
            for (int v = 0; v < V; v++) {
                s[v] = lane * V + v < E && l[v] != -INFINITY ? expf(l[v] - m) : 0.f;
                sum += s[v];
            }
            sum = seg_reduce<L>(sum, [](float p, float q) { return p + q; });
            const float f = sum != 0.f ? dot / sum : 0.f;
#pragma unroll
            for (int v = 0; v < V; v++)
                if (s[v] != 0.f) o[v] -= s[v] * f;
        }
        if (row && lane * V < E) store(dlogits + t * E + lane * V, E - lane * V, o);
        wave_lds_sync();
    }
}

// ---- rows moved: gather, dispatch, combine -------------------------------------------------------
// L lanes of a 256-thread workgroup share one row (16, 64 or all 256), eight columns a lane and step;
// gridDim.y workgroups share its columns where there are few rows.
template <int L>
__device__ __forceinline__ int64_t first_row() {
    const int sub = L >= 64 ? __builtin_amdgcn_readfirstlane(threadIdx.x / L) : (int)threadIdx.x / L;
    return (int64_t)blockIdx.x * (256 / L) + sub;
}
template <int L> __device__ __forceinline__ int64_t row_step() { return (int64_t)gridDim.x * (256 / L); }
template <int L> __device__ __forceinline__ int64_t first_col() { return ((int64_t)blockIdx.y * L + threadIdx.x % L) * 8; }
template <int L> __device__ __forceinline__ int64_t col_step() { return (int64_t)gridDim.y * L * 8; }

template <typename T, int L, bool NT>
__global__ __launch_bounds__(256) void k_gather_drop(const T *__restrict__ data, T *__restrict__ out, int64_t rows,
                                                     int64_t cols, Drop d, RowGather g) {
    for (int64_t r = first_row<L>(); r < rows; r += row_step<L>()) {
        const int32_t f = g.fpos[r] < 0 ? -1 - g.fpos[r] : g.fpos[r];
        const T *x = data + (g.base[g.order[f]] + g.off[r]) * cols;
        const int64_t id = drop_row(d, r);
        for (int64_t c = first_col<L>(); c < cols; c += col_step<L>()) {
            float v[8];
            load<NT>(x + c, cols - c, v);
            if (d.drop) drop8<false>(d, draw8(d, id, (uint32_t)(c >> 3)), v, v);
            store<NT>(out + r * cols + c, cols - c, v);
        }
    }
}

template <typename T, int L>
__global__ __launch_bounds__(256) void k_dispatch(MoveArgs m, const T *__restrict__ x, int64_t ldx, T *__restrict__ xs) {
    for (int64_t t = first_row<L>(); t < m.T; t += row_step<L>()) {
        const int32_t *e = m.experts + t * m.k, *pos = m.pos + t * m.k;
        for (int64_t c = first_col<L>(); c < m.D; c += col_step<L>()) {
            float v[8];
            const float zero[8] = {0, 0, 0, 0, 0, 0, 0, 0};
            load(x + t * ldx + c, m.D - c, v);
            for (int j = 0; j < m.k; j++) {
                T *to = xs + (int64_t)pos[j] * m.D + c;
                if (e[j] >= 0) store(to, m.D - c, v);
                else store(to, m.D - c, zero);
            }
        }
    }
}

// KU rows of y are on their way at a time.  A slot without an expert is read like any other (its place
// is a row of y) and left out of the sum whatever it holds.
template <typename T, int L, int KU, bool NT>
__global__ __launch_bounds__(256) void k_combine(MoveArgs m, const T *__restrict__ y, const float *__restrict__ w,
                                                 const T *__restrict__ res, int64_t ldr, Drop d, T *__restrict__ out) {
    for (int64_t t = first_row<L>(); t < m.T; t += row_step<L>()) {
        const int32_t *e = m.experts + t * m.k, *pos = m.pos + t * m.k;
        const int64_t id = d.drop ? drop_row(d, t) : 0;
        for (int64_t c = first_col<L>(); c < m.D; c += col_step<L>()) {
            float acc[8] = {0, 0, 0, 0, 0, 0, 0, 0}, r[8] = {0, 0, 0, 0, 0, 0, 0, 0};
            if (res) load<NT>(res + t * ldr + c, m.D - c, r);
            Draw dr;
            for (int j0 = 0; j0 < m.k; j0 += KU) {
                float v[KU][8];
#pragma unroll
                for (int u = 0; u < KU; u++) {
                    const int j = j0 + u < m.k ? j0 + u : j0;
                    load<NT>(y + (int64_t)pos[j] * m.D + c, m.D - c, v[u]);
                }
                if (d.drop && j0 == 0) dr = draw8(d, id, (uint32_t)(c >> 3));   // while the rows come
#pragma unroll
                for (int u = 0; u < KU; u++) {
                    const int j = j0 + u < m.k ? j0 + u : j0;
                    const bool on = j0 + u < m.k && e[j] >= 0;
                    const float wj = w ? w[t * m.k + j] : 1.f;
#pragma unroll
                    for (int i = 0; i < 8; i++) acc[i] = on ? fmaf(wj, v[u][i], acc[i]) : acc[i];
                }
            }
            if (d.drop) {
                drop8<true>(d, dr, acc, r);
            } else if (res) {
#pragma unroll
                for (int i = 0; i < 8; i++) acc[i] += r[i];
            }
            store<NT>(out + t * m.D + c, m.D - c, acc);
        }
    }
}

// One pass over g = dropout(dout): KU products with rows of y and KU rows of dy at a time.  The lanes
// of a row hold partial products of all its slots; they are joined after the last column.
template <typename T, int L, int KM>
__global__ __launch_bounds__(256) void k_combine_grad(MoveArgs m, const int32_t *__restrict__ experts,
                                                      const int32_t *__restrict__ places, const T *__restrict__ dout, int64_t ldo,
                                                      const T *__restrict__ y, const float *__restrict__ w, Drop d,
                                                      T *__restrict__ dy, float *__restrict__ dw) {
    constexpr int KU = KM < 8 ? KM : 8;
    __shared__ float part[L > 64 ? 4 : 1][KM];
    for (int64_t t = first_row<L>(); t < m.T; t += row_step<L>()) {
        const int64_t id = d.drop ? drop_row(d, t) : 0;
        float dot[KM], wt[KM];
        int32_t pos[KM];
        bool on[KM];
#pragma unroll
        for (int j = 0; j < KM; j++) {
            const int64_t slot = t * m.k + (j < m.k ? j : 0);
            on[j] = experts[slot] >= 0;
            pos[j] = places[slot];
            wt[j] = w[slot];
            dot[j] = 0.f;
        }
        for (int64_t c = first_col<L>(); c < m.D; c += col_step<L>()) {
            float g[8];
            load(dout + t * ldo + c, m.D - c, g);
            if (d.drop) drop8<false>(d, draw8(d, id, (uint32_t)(c >> 3)), g, g);
#pragma unroll
            for (int j0 = 0; j0 < KM; j0 += KU) {
                if (j0 >= m.k) break;
                if (dw) {
                    float v[KU][8];
#pragma unroll
                    for (int u = 0; u < KU; u++) load(y + (int64_t)pos[j0 + u] * m.D + c, m.D - c, v[u]);
#pragma unroll
                    for (int u = 0; u < KU; u++)
#pragma unroll
                        for (int i = 0; i < 8; i++) dot[j0 + u] = fmaf(g[i], v[u][i], dot[j0 + u]);
                }
                if (dy) {
#pragma unroll
                    for (int u = 0; u < KU; u++) {
                        if (j0 + u >= m.k) break;
                        float o[8];
#pragma unroll
                        for (int i = 0; i < 8; i++) o[i] = on[j0 + u] ? wt[j0 + u] * g[i] : 0.f;
                        store(dy + (int64_t)pos[j0 + u] * m.D + c, m.D - c, o);
                    }
                }
            }
        }
        if (!dw) continue;
#pragma unroll
        for (int j = 0; j < KM; j++) dot[j] = seg_reduce<(L < 64 ? L : 64)>(dot[j], [](float a, float b) { return a + b; });
        if (L > 64) {
            __syncthreads();
            if ((threadIdx.x & 63) == 0)
#pragma unroll
                for (int j = 0; j < KM; j++) part[threadIdx.x >> 6][j] = dot[j];
            __syncthreads();
            const int j = threadIdx.x;
            if (j < m.k) dw[t * m.k + j] = experts[t * m.k + j] >= 0 ? (part[0][j] + part[1][j]) + (part[2][j] + part[3][j]) : 0.f;
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

// lanes and values per lane of a row of E experts
template <typename F>
void by_width(int E, F f) {
    if (E <= 16) f(std::integral_constant<int, 16>(), std::integral_constant<int, 1>());
    else if (E <= 32) f(std::integral_constant<int, 16>(), std::integral_constant<int, 2>());
    else if (E <= 64) f(std::integral_constant<int, 16>(), std::integral_constant<int, 4>());
    else if (E <= 128) f(std::integral_constant<int, 16>(), std::integral_constant<int, 8>());
    else if (E <= 256) f(std::integral_constant<int, 16>(), std::integral_constant<int, 16>());
    else if (E <= 512) f(std::integral_constant<int, 64>(), std::integral_constant<int, 8>());
    else f(std::integral_constant<int, 64>(), std::integral_constant<int, 16>());
}

}  // namespace

// Whether a pass over so many bytes goes past the caches: beyond the 256 MB of the Infinity Cache
// nothing of it can be found there later.  Measured past / through: dropout 16384 x 8192 bf16 with
// residual 131 / 157 us, without 91 / 94; gather of 65536 x 2048 bf16 99 / 125; combine of
// 16384 x 8 x 4096 bf16 233 / 281; combine of 2039 x 3 x 1001 fp16 (17 MB) 7.8 / 7.4.  Dispatch and
// the combine's gradient write eight rows for one read and are slower past them (249 / 223, 474 / 458).
static bool past_caches(int64_t bytes) { return bytes > ((int64_t)256 << 20); }

template <typename F>
static void by_flag(bool b, F f) {
    if (b) f(std::true_type());
    else f(std::false_type());
}

// lanes of a row of `cols` values, and the launch of `rows` such rows
template <typename F>
static void by_row(int64_t rows, int64_t cols, F f) {
    const int L = cols <= 128 ? 16 : cols <= 1024 ? 64 : 256;
    int64_t x = (rows + 256 / L - 1) / (256 / L), y = 1;
    if (x < 2048) {      // few rows: their columns over several workgroups
        y = (cols + L * 8 - 1) / (L * 8);
        if (y > 2048 / x) y = 2048 / x;
        if (y < 1) y = 1;
    }
    const dim3 grid((unsigned)(x < (1 << 20) ? x : 1 << 20), (unsigned)y);
    if (L == 16) f(std::integral_constant<int, 16>(), grid);
    else if (L == 64) f(std::integral_constant<int, 64>(), grid);
    else f(std::integral_constant<int, 256>(), grid);
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
        by_flag(past_caches(rows * cols * (int64_t)sizeof(T) * (residual ? 3 : 2)), [&](auto NT) {
            by_flag(residual != nullptr, [&](auto RES) {
                hipLaunchKernelGGL((k_dropout<T, decltype(RES)::value, decltype(NT)::value>), grid, dim3(256), 0, s,
                                   (const T *)x, ldx, (const T *)residual, ldr, (T *)y, rows, cols, (uint32_t)nb, d);
            });
        });
    });
}

hipError_t launch_gather_dropout(const void *data, void *out, int64_t rows, int64_t cols, int32_t dtype, const Drop &d,
                                 const RowGather &g, hipStream_t s) {
    if (rows <= 0 || cols <= 0) return hipSuccess;
    return by_type(dtype, [&](auto *p) {
        using T = std::remove_pointer_t<decltype(p)>;
        by_row(rows, cols, [&](auto L, dim3 grid) {
            by_flag(past_caches(2 * rows * cols * (int64_t)sizeof(T)), [&](auto NT) {
                hipLaunchKernelGGL((k_gather_drop<T, decltype(L)::value, decltype(NT)::value>), grid, dim3(256), 0, s,
                                   (const T *)data, (T *)out, rows, cols, d, g);
            });
        });
    });
}

hipError_t launch_route(const RouteArgs &a, hipStream_t s) {
    const int64_t chunks = route_chunks(a.T);
    hipError_t err = hipSuccess;
    const hipError_t e = by_type(a.dtype, [&](auto *p) {
        using T = std::remove_pointer_t<decltype(p)>;
        by_width(a.E, [&](auto L, auto V) {
            size_t lds = 8 * (size_t)kWords * a.E + 4 * (size_t)a.E;
            if (a.groups > 1) lds = 8 * (size_t)kWords * a.E + 8 * (size_t)(kRouteThreads / L) * a.E;
            auto kern = k_route<T, decltype(L)::value, decltype(V)::value>;
            if (lds > 64 * 1024)
                err = hipFuncSetAttribute((const void *)kern, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
            if (err == hipSuccess) hipLaunchKernelGGL(kern, dim3((unsigned)chunks), dim3(kRouteThreads), lds, s, a);
        });
    });
    if (err != hipSuccess) return err;
    if (e != hipSuccess || chunks == 1) return e;
    hipLaunchKernelGGL(k_route_place, dim3((unsigned)chunks), dim3(kRouteThreads),
                       8 * (size_t)kWords * a.E + 8 * (size_t)a.E, s, a, chunks);
    return hipGetLastError();
}

hipError_t launch_route_grad(const RouteArgs &a, const float *dweights, void *dlogits, hipStream_t s) {
    if (a.T <= 0) return hipSuccess;
    return by_type(a.dtype, [&](auto *p) {
        using T = std::remove_pointer_t<decltype(p)>;
        by_width(a.E, [&](auto L, auto V) {
            const int64_t blocks = (a.T + kRouteThreads / L - 1) / (kRouteThreads / L);
            hipLaunchKernelGGL((k_route_grad<T, decltype(L)::value, decltype(V)::value>),
                               dim3((unsigned)(blocks < 4096 ? blocks : 4096)), dim3(kRouteThreads),
                               4 * (size_t)kRouteThreads * V, s, a, dweights, (T *)dlogits);
        });
    });
}

hipError_t launch_dispatch(const MoveArgs &m, const void *x, int64_t ldx, void *xs, hipStream_t s) {
    if (m.T <= 0 || m.D <= 0) return hipSuccess;
    return by_type(m.dtype, [&](auto *p) {
        using T = std::remove_pointer_t<decltype(p)>;
        by_row(m.T, m.D, [&](auto L, dim3 grid) {
            hipLaunchKernelGGL((k_dispatch<T, decltype(L)::value>), grid, dim3(256), 0, s, m, (const T *)x, ldx, (T *)xs);
        });
    });
}

hipError_t launch_combine(const MoveArgs &m, const void *y, const float *w, const void *residual, int64_t ldr,
                          const Drop &d, void *out, hipStream_t s) {
    if (m.T <= 0 || m.D <= 0) return hipSuccess;
    return by_type(m.dtype, [&](auto *p) {
        using T = std::remove_pointer_t<decltype(p)>;
        by_row(m.T, m.D, [&](auto L, dim3 grid) {
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
        by_row(m.T, m.D, [&](auto L, dim3 grid) {
            grid.y = 1;     // the products run over all columns
            by_slots(m.k, [&](auto KM) {
                hipLaunchKernelGGL((k_combine_grad<T, decltype(L)::value, decltype(KM)::value>), grid, dim3(256), 0, s,
                                   m, m.experts, m.pos, (const T *)dout, ldo, (const T *)y, w, d, (T *)dy, dw);
            });
        });
    });
}

}  // namespace pss
