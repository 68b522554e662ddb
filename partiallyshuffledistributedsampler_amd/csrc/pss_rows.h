// pss_rows.h -- launch interface of the batch-row operators (pss_rows.hip): dropout keyed by row
// ids (alone, with a residual, or fused in the gather of device-resident files), routing of rows
// to experts, and the dispatch / combine of the routed rows.  Stream-ordered and allocation-free.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace pss {

// Dropout of one call: value (row id r, column c) is kept iff u >= drop, u the 16-bit half c % 8
// of the Philox block (c / 8, r lo, r hi, DOM_DROPOUT) under the key.  r = row0 + ids[i] for row i
// (per_row), row0 + ids[0] + i (one id), or row0 + i (no ids).
struct Drop {
    uint32_t key0, key1;
    uint32_t drop;          // 0 .. 65536
    float scale;            // 65536 / (65536 - drop); 0 if everything is dropped
    int64_t row0;
    const int64_t *ids;
    int32_t per_row;
};

// x -> y (+ residual); strides in values
hipError_t launch_dropout(const void *x, int64_t ldx, const void *residual, int64_t ldr, void *y, int64_t rows,
                          int64_t cols, int32_t dtype, const Drop &d, hipStream_t s);
// row i: row base[order[f_i]] + off_i of the data, f_i the file position (reflected: < 0)
struct RowGather {
    const int64_t *base;
    const int32_t *order, *fpos, *off;
};
hipError_t launch_gather_dropout(const void *data, void *out, int64_t rows, int64_t cols, int32_t dtype, const Drop &d,
                                 const RowGather &g, hipStream_t s);

struct RouteArgs {
    const void *logits;
    int64_t ld;
    int64_t T;
    int32_t E, k, dtype;
    int32_t chunk;          // rows of a workgroup
    int32_t score;          // 0 softmax, 1 sigmoid
    int32_t renorm;
    float scale;
    const float *bias;      // [E] or NULL
    const uint8_t *valid;   // [T] or NULL
    int32_t groups, top_groups, group_sum;
    int32_t *experts;       // [T, k]
    float *weights;         // [T, k]
    float *slopes;          // [T, k] 1 - sigmoid of the chosen, or NULL
    int32_t *offsets;       // [E + 1]
    int32_t *pos, *src;     // [T * k]
    // workspace (NULL with one chunk): rows of each chunk and expert, rows before, rows in all
    uint64_t *mask;         // [chunks, E]
    int32_t *before;        // [chunks, E]
    int32_t *totals;        // [E]
};
constexpr int kRouteChunk = 64;     // rows of a workgroup at most: one bit of a 64-bit mask each
// More than 256 experts take a wave a row, eight rows at once: with few rows 16 to a workgroup (700 rows,
// 368 experts in groups: 33 us, 63 with 64), else 64, the masks and sums then being fewer.
static inline int route_chunk(int64_t T, int32_t E) { return E > 256 && T <= 8192 ? 16 : kRouteChunk; }
constexpr int kRouteMaxE = 1024, kRouteMaxK = 16, kRouteMaxGroups = 64;
static inline int64_t route_chunks(int64_t T, int32_t E) {
    const int c = route_chunk(T, E);
    return T <= c ? 1 : (T + c - 1) / c;
}
hipError_t launch_route(const RouteArgs &a, hipStream_t s);
// dweights [T, k] -> dlogits [T, E] (contiguous); reads experts, weights, slopes (sigmoid) or logits
// (softmax not renormalised) of `a`
hipError_t launch_route_grad(const RouteArgs &a, const float *dweights, void *dlogits, hipStream_t s);

struct MoveArgs {           // rows between their own order (T) and the experts' (T * k)
    int64_t T, D;
    int32_t k, dtype;
    const int32_t *experts, *pos;
};
// xs[pos[t, j]] = x[t], 0 where slot (t, j) has no expert
hipError_t launch_dispatch(const MoveArgs &m, const void *x, int64_t ldx, void *xs, hipStream_t s);
// out[t] = residual[t] + dropout(sum over used j of w[t, j] * y[pos[t, j]]); w NULL: weights 1
hipError_t launch_combine(const MoveArgs &m, const void *y, const float *w, const void *residual, int64_t ldr,
                          const Drop &d, void *out, hipStream_t s);
// g = dropout(dout): dy[pos[t, j]] = w[t, j] * g[t] (0 where unused; dy NULL: not wanted),
// dw[t, j] = <g[t], y[pos[t, j]]> (0 where unused; dw NULL: not wanted)
hipError_t launch_combine_grad(const MoveArgs &m, const void *dout, int64_t ldo, const void *y, const float *w,
                               const Drop &d, void *dy, float *dw, hipStream_t s);

// argument checks of the entries in pss_rows.cpp, shared with pss_gather_dropout
int make_drop(double p, uint64_t key, int64_t row0, const int64_t *ids, int64_t n_ids, int64_t rows, Drop *d);
int check_rows(const void *x, int64_t ldx, const void *y, int64_t rows, int64_t cols, int32_t dtype);

namespace cpu {
// launch_dropout (g NULL) and launch_gather_dropout on host memory
void dropout(const void *x, int64_t ldx, const void *residual, int64_t ldr, void *y, int64_t rows, int64_t cols,
             int32_t dtype, const Drop &d, const RowGather *g);
}  // namespace cpu

// error text of the C entries (pss_runtime.cpp)
int set_error(int code, const char *msg);

}  // namespace pss
