// pss_rows.cpp -- the C entries of the batch-row operators (include/pss.h) that need no sampler
// handle, and their CPU mode: dropout keyed by row ids on host memory, from the same Philox
// definition as the kernels (pss_common.h), bit-identical to them.
#include <hip/hip_runtime.h>

#include <cmath>
#include <cstring>
#include <string>

#include "../../include/pss.h"
#include "pss_common.h"
#include "pss_cpu.h"
#include "pss_rows.h"

namespace {

using pss::set_error;

#define ROWS_HIP(call)                                                                        \
    do {                                                                                      \
        hipError_t e_ = (call);                                                               \
        if (e_ != hipSuccess) return set_error(PSS_EHIP, hipGetErrorString(e_));              \
    } while (0)

// ---- host values ---------------------------------------------------------------------------------
float up(const void *p, int64_t i, int32_t dtype) {
    if (dtype == PSS_F32) return ((const float *)p)[i];
    const uint16_t h = ((const uint16_t *)p)[i];
    uint32_t u;
    if (dtype == PSS_BF16) {
        u = (uint32_t)h << 16;
    } else {
        const uint32_t sign = (uint32_t)(h & 0x8000) << 16, exp = (h >> 10) & 31, man = h & 0x3FF;
        if (exp == 31) u = sign | 0x7F800000u | man << 13;
        else if (exp) u = sign | (exp + 112) << 23 | man << 13;
        else {
            const float f = std::ldexp((float)man, -24);   // subnormal: exact in float
            std::memcpy(&u, &f, 4);
            u |= sign;
        }
    }
    float f;
    std::memcpy(&f, &u, 4);
    return f;
}

// to the nearest, ties to the even value, as the GPU's conversions
void down(void *p, int64_t i, int32_t dtype, float f) {
    if (dtype == PSS_F32) { ((float *)p)[i] = f; return; }
    uint32_t u;
    std::memcpy(&u, &f, 4);
    uint16_t h;
    if (dtype == PSS_BF16) {
        h = f != f ? (uint16_t)(u >> 16 | 0x40) : (uint16_t)((u + 0x7FFF + ((u >> 16) & 1)) >> 16);
    } else {
        const uint16_t sign = (uint16_t)(u >> 16 & 0x8000);
        const uint32_t a = u & 0x7FFFFFFFu;
        if (a > 0x7F800000u) h = sign | 0x7E00 | (uint16_t)(a >> 13 & 0x3FF);
        else if (a >= 0x477FF000u) h = sign | 0x7C00;        // 65520 and above round to infinity
        else if (a >= 0x38800000u) h = sign | (uint16_t)((a - 0x38000000u + 0xFFF + ((a >> 13) & 1)) >> 13);
        else {                                               // below 2^-14: units of 2^-24
            float g;
            std::memcpy(&g, &a, 4);
            h = sign | (uint16_t)std::nearbyint(std::ldexp(g, 24));
        }
    }
    ((uint16_t *)p)[i] = h;
}

}  // namespace

namespace pss {

int make_drop(double p, uint64_t key, int64_t row0, const int64_t *ids, int64_t n_ids, int64_t rows, Drop *d) {
    if (!(p >= 0.0 && p <= 1.0)) return set_error(PSS_EINVAL, "dropout: p must be in [0, 1]");
    if (n_ids < 0 || (n_ids > 1 && n_ids != rows) || (n_ids > 0 && !ids))
        return set_error(PSS_EINVAL, "dropout: row ids are none, one (the first row's) or one per row");
    d->key0 = (uint32_t)key;
    d->key1 = (uint32_t)(key >> 32);
    d->drop = (uint32_t)std::floor(p * 65536.0 + 0.5);
    d->scale = d->drop < 65536 ? (float)(65536.0 / (double)(65536 - d->drop)) : 0.f;
    d->row0 = row0;
    d->ids = n_ids ? ids : nullptr;
    d->per_row = n_ids > 1;
    return PSS_OK;
}

int check_rows(const void *x, int64_t ldx, const void *y, int64_t rows, int64_t cols, int32_t dtype) {
    if (dtype < PSS_F32 || dtype > PSS_F16) return set_error(PSS_EINVAL, "dtype must be PSS_F32, PSS_BF16 or PSS_F16");
    if (rows < 0 || cols < 0) return set_error(PSS_EINVAL, "rows and cols must be >= 0");
    if (cols >= (int64_t)1 << 34) return set_error(PSS_ENOTSUP, "rows of 2^34 values or more");
    if (rows > 0 && cols > 0 && (!x || !y)) return set_error(PSS_EINVAL, "NULL rows");
    if (ldx < 0) return set_error(PSS_EINVAL, "the row stride must be >= 0");
    return PSS_OK;
}

namespace cpu {

void dropout(const void *x, int64_t ldx, const void *residual, int64_t ldr, void *y, int64_t rows, int64_t cols,
             int32_t dtype, const Drop &d, const RowGather *g) {
    for (int64_t r = 0; r < rows; r++) {
        const int64_t id = (int64_t)((uint64_t)d.row0 + (d.ids ? (uint64_t)d.ids[d.per_row ? r : 0] : 0u) +
                                     (d.per_row ? 0u : (uint64_t)r));
        int64_t from = r;
        if (g) {
            const int32_t f = g->fpos[r] < 0 ? -1 - g->fpos[r] : g->fpos[r];
            from = g->base[g->order[f]] + g->off[r];
        }
        uint32_t w[4];
        for (int64_t c = 0; c < cols; c++) {
            if ((c & 7) == 0 && d.drop) {
                w[0] = (uint32_t)(c >> 3); w[1] = (uint32_t)id; w[2] = (uint32_t)((uint64_t)id >> 32); w[3] = DOM_DROPOUT;
                philox4x32_10(w[0], w[1], w[2], w[3], d.key0, d.key1);
            }
            float v = up(x, from * ldx + c, dtype);
            const bool drop = d.drop && ((w[(c & 7) >> 1] >> (c & 1 ? 16 : 0)) & 0xFFFF) < d.drop;
            if (residual) {
                const float q = up(residual, r * ldr + c, dtype);
                v = drop ? q : d.drop ? std::fma(v, d.scale, q) : v + q;
            } else {
                v = drop ? 0.f : d.drop ? v * d.scale : v;
            }
            down(y, r * cols + c, dtype, v);
        }
    }
}

}  // namespace cpu
}  // namespace pss

using namespace pss;

extern "C" {

int pss_dropout_key(uint64_t seed, int64_t epoch, int32_t rank, int32_t site, uint64_t *key) {
    if (!key) return set_error(PSS_EINVAL, "key is NULL");
    *key = mix64(epoch_key(seed, epoch) ^ ((uint64_t)(uint32_t)rank << 32 | (uint32_t)site));
    return PSS_OK;
}

int pss_dropout(const void *x, int64_t ldx, const void *residual, int64_t ldr, void *y, int64_t rows, int64_t cols,
                int32_t dtype, double p, uint64_t key, int64_t row0, const int64_t *row_ids, int64_t n_ids,
                int32_t host, void *stream) {
    Drop d;
    int rc = check_rows(x, ldx, y, rows, cols, dtype);
    if (rc == PSS_OK) rc = make_drop(p, key, row0, row_ids, n_ids, rows, &d);
    if (rc) return rc;
    if (ldr < 0) return set_error(PSS_EINVAL, "the row stride must be >= 0");
    if (host) {
        cpu::dropout(x, ldx, residual, ldr, y, rows, cols, dtype, d, nullptr);
        return PSS_OK;
    }
    ROWS_HIP(launch_dropout(x, ldx, residual, ldr, y, rows, cols, dtype, d, (hipStream_t)stream));
    return PSS_OK;
}

static int route_args(RouteArgs *a, const void *logits, int64_t ld, int64_t tokens, int32_t experts, int32_t k,
                      int32_t dtype, int32_t score, int32_t renorm, double scale) {
    if (dtype < PSS_F32 || dtype > PSS_F16) return set_error(PSS_EINVAL, "dtype must be PSS_F32, PSS_BF16 or PSS_F16");
    if (tokens < 0 || experts < 1 || k < 1 || k > experts)
        return set_error(PSS_EINVAL, "route: tokens >= 0 and 1 <= k <= experts");
    if (experts > kRouteMaxE || k > kRouteMaxK)
        return set_error(PSS_ENOTSUP, "route: at most 1024 experts, 16 of them for a row");
    if (tokens >= (int64_t)1 << 28 || tokens * k >= (int64_t)1 << 31)
        return set_error(PSS_ENOTSUP, "route: 2^28 rows, or 2^31 slots, or more");
    if (tokens > 0 && !logits) return set_error(PSS_EINVAL, "route: NULL logits");
    if (ld < 0) return set_error(PSS_EINVAL, "the row stride must be >= 0");
    if (score != PSS_SOFTMAX && score != PSS_SIGMOID) return set_error(PSS_EINVAL, "route: score must be PSS_SOFTMAX or PSS_SIGMOID");
    if (!(std::fabs(scale) >= 1e-18 && std::fabs(scale) <= 1e18))
        return set_error(PSS_EINVAL, "route: scale must be a number between 1e-18 and 1e18 in magnitude");
    *a = RouteArgs{};
    a->logits = logits;
    a->ld = ld;
    a->T = tokens;
    a->E = experts;
    a->chunk = route_chunk(tokens, experts);
    a->k = k;
    a->dtype = dtype;
    a->score = score;
    a->renorm = renorm != 0;
    a->scale = (float)scale;
    return PSS_OK;
}

int64_t pss_route_workspace(int64_t tokens, int32_t experts) {
    if (tokens < 0 || experts < 1) return 0;
    const int64_t n = route_chunks(tokens, experts);
    return n > 1 ? (n * 12 + 4) * experts : 0;
}

int pss_route(const void *logits, int64_t ld, int64_t tokens, int32_t experts, int32_t k, int32_t dtype, int32_t score,
              const float *bias, const uint8_t *valid, int32_t groups, int32_t top_groups, int32_t group_sum,
              int32_t renorm, double scale, int32_t *out_experts, float *out_weights, float *slopes, int32_t *offsets,
              int32_t *pos, int32_t *src, void *ws, int64_t ws_bytes, void *stream) {
    RouteArgs a;
    const int rc = route_args(&a, logits, ld, tokens, experts, k, dtype, score, renorm, scale);
    if (rc) return rc;
    if (groups < 1 || experts % groups || top_groups < 1 || top_groups > groups)
        return set_error(PSS_EINVAL, "route: groups divide the experts, 1 <= top_groups <= groups");
    if (groups > kRouteMaxGroups) return set_error(PSS_ENOTSUP, "route: at most 64 groups");
    if ((int64_t)top_groups * (experts / groups) < k)
        return set_error(PSS_EINVAL, "route: the chosen groups hold fewer than k experts");
    if (group_sum != 1 && group_sum != 2) return set_error(PSS_EINVAL, "route: group_sum is 1 or 2");
    if (!offsets || (tokens > 0 && (!out_experts || !out_weights || !pos || !src)))
        return set_error(PSS_EINVAL, "route: NULL output");
    const int64_t need = pss_route_workspace(tokens, experts);
    if (need > 0 && (!ws || ws_bytes < need || (uintptr_t)ws % 8))
        return set_error(PSS_EINVAL, "route: the workspace is too small, or not 8-byte aligned");
    a.bias = bias;
    a.valid = valid;
    a.groups = groups;
    a.top_groups = top_groups;
    a.group_sum = group_sum;
    a.experts = out_experts;
    a.weights = out_weights;
    a.slopes = score == PSS_SIGMOID ? slopes : nullptr;
    a.offsets = offsets;
    a.pos = pos;
    a.src = src;
    if (need > 0) {
        const int64_t n = route_chunks(tokens, experts) * experts;
        a.mask = (uint64_t *)ws;
        a.before = (int32_t *)(a.mask + n);
        a.totals = a.before + n;
    }
    ROWS_HIP(launch_route(a, (hipStream_t)stream));
    return PSS_OK;
}

int pss_route_grad(const void *logits, int64_t ld, int64_t tokens, int32_t experts, int32_t k, int32_t dtype,
                   int32_t score, int32_t renorm, double scale, const int32_t *chosen, const float *weights,
                   const float *slopes, const float *dweights, void *dlogits, void *stream) {
    RouteArgs a;
    // the logits are read for a softmax that was not renormalised alone
    const bool full = score == PSS_SOFTMAX && !renorm;
    const int rc = route_args(&a, full ? logits : dlogits, ld, tokens, experts, k, dtype, score, renorm, scale);
    if (rc) return rc;
    if (tokens > 0 && (!chosen || !weights || !dweights || !dlogits || (score == PSS_SIGMOID && !slopes)))
        return set_error(PSS_EINVAL, "route_grad: NULL argument");
    a.slopes = const_cast<float *>(slopes);
    a.experts = const_cast<int32_t *>(chosen);
    a.weights = const_cast<float *>(weights);
    ROWS_HIP(launch_route_grad(a, dweights, dlogits, (hipStream_t)stream));
    return PSS_OK;
}

static int move_args(MoveArgs *m, int64_t tokens, int32_t k, int64_t cols, int32_t dtype, const int32_t *experts,
                     const int32_t *pos) {
    if (dtype < PSS_F32 || dtype > PSS_F16) return set_error(PSS_EINVAL, "dtype must be PSS_F32, PSS_BF16 or PSS_F16");
    if (tokens < 0 || cols < 0 || k < 1) return set_error(PSS_EINVAL, "tokens and cols >= 0, k >= 1");
    if (k > kRouteMaxK) return set_error(PSS_ENOTSUP, "at most 16 experts for a row");
    if (tokens * k >= ((int64_t)1 << 31)) return set_error(PSS_ENOTSUP, "2^31 slots or more");
    if (cols >= (int64_t)1 << 34) return set_error(PSS_ENOTSUP, "rows of 2^34 values or more");
    if (tokens > 0 && (!experts || !pos)) return set_error(PSS_EINVAL, "NULL plan");
    *m = MoveArgs{tokens, cols, k, dtype, experts, pos};
    return PSS_OK;
}

int pss_dispatch(const void *x, int64_t ldx, int64_t tokens, int32_t k, int64_t cols, int32_t dtype,
                 const int32_t *experts, const int32_t *pos, void *xs, void *stream) {
    MoveArgs m;
    const int rc = move_args(&m, tokens, k, cols, dtype, experts, pos);
    if (rc) return rc;
    if (ldx < 0) return set_error(PSS_EINVAL, "the row stride must be >= 0");
    if (tokens > 0 && cols > 0 && (!x || !xs)) return set_error(PSS_EINVAL, "NULL rows");
    ROWS_HIP(launch_dispatch(m, x, ldx, xs, (hipStream_t)stream));
    return PSS_OK;
}

int pss_combine(const void *y, int64_t tokens, int32_t k, int64_t cols, int32_t dtype, const int32_t *experts,
                const int32_t *pos, const float *weights, const void *residual, int64_t ldr, double p, uint64_t key,
                int64_t row0, const int64_t *row_ids, int64_t n_ids, void *out, void *stream) {
    MoveArgs m;
    Drop d;
    int rc = move_args(&m, tokens, k, cols, dtype, experts, pos);
    if (rc == PSS_OK) rc = make_drop(p, key, row0, row_ids, n_ids, tokens, &d);
    if (rc) return rc;
    if (ldr < 0) return set_error(PSS_EINVAL, "the row stride must be >= 0");
    if (tokens > 0 && cols > 0 && (!y || !out)) return set_error(PSS_EINVAL, "NULL rows");
    ROWS_HIP(launch_combine(m, y, weights, residual, ldr, d, out, (hipStream_t)stream));
    return PSS_OK;
}

int pss_combine_grad(const void *dout, int64_t ldo, const void *y, int64_t tokens, int32_t k, int64_t cols,
                     int32_t dtype, const int32_t *experts, const int32_t *pos, const float *weights, double p,
                     uint64_t key, int64_t row0, const int64_t *row_ids, int64_t n_ids, void *dy, float *dweights,
                     void *stream) {
    MoveArgs m;
    Drop d;
    int rc = move_args(&m, tokens, k, cols, dtype, experts, pos);
    if (rc == PSS_OK) rc = make_drop(p, key, row0, row_ids, n_ids, tokens, &d);
    if (rc) return rc;
    if (ldo < 0) return set_error(PSS_EINVAL, "the row stride must be >= 0");
    if (tokens > 0 && (!weights || (cols > 0 && (!dout || (dweights && !y))))) return set_error(PSS_EINVAL, "NULL argument");
    ROWS_HIP(launch_combine_grad(m, dout, ldo, y, weights, d, dy, dweights, (hipStream_t)stream));
    return PSS_OK;
}

}  // extern "C"
