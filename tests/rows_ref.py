"""The batch-row operators in 64 bits (numpy), written from their definitions in include/pss.h."""
import numpy as np

M32 = np.uint64(0xFFFFFFFF)


def philox(counter, key):
    """Philox4x32-10 of counters [..., 4] (uint64 arrays of 32-bit words) -> [..., 4]."""
    c = [counter[..., i].astype(np.uint64) for i in range(4)]
    k = [np.uint64(key & 0xFFFFFFFF), np.uint64(key >> 32)]
    for _ in range(10):
        p0, p1 = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(p1 >> np.uint64(32)) ^ c[1] ^ k[0], p1 & M32, (p0 >> np.uint64(32)) ^ c[3] ^ k[1], p0 & M32]
        k = [(k[0] + np.uint64(0x9E3779B9)) & M32, (k[1] + np.uint64(0xBB67AE85)) & M32]
    return np.stack(c, -1)


def halves(ids, cols, key):
    """The 16-bit draw of every value of rows `ids` (python ints of 64 bits)."""
    ids = np.array([i % (1 << 64) for i in ids], dtype=np.uint64)
    nb = (cols + 7) // 8
    ctr = np.zeros((len(ids), nb, 4), dtype=np.uint64)
    ctr[..., 0] = np.arange(nb, dtype=np.uint64)
    ctr[..., 1] = (ids & M32)[:, None]
    ctr[..., 2] = (ids >> np.uint64(32))[:, None]
    ctr[..., 3] = 6
    w = philox(ctr, key)
    u = np.stack([w & np.uint64(0xFFFF), w >> np.uint64(16)], -1).reshape(len(ids), nb * 8)
    return u[:, :cols].astype(np.int64)


def factor(ids, cols, p, key):
    """What dropout multiplies every value by; NaN-safe users select by factor != 0."""
    t = int(np.floor(p * 65536 + 0.5))
    if t == 0:
        return np.ones((len(ids), cols))
    keep = halves(ids, cols, key) >= t
    return np.where(keep, 65536.0 / (65536 - t) if t < 65536 else 0.0, 0.0)


def drop(v, f):
    return np.where(f != 0, v * np.where(f != 0, f, 1.0), 0.0)


def scores(l, score):
    l = np.asarray(l, dtype=np.float64)
    with np.errstate(all="ignore"):
        if score == "sigmoid":
            return np.where(l >= 0, 1 / (1 + np.exp(-l)), np.exp(l) / (1 + np.exp(l)))
        m = np.max(l, 1, keepdims=True)
        e = np.exp(l - np.where(np.isneginf(m), 0.0, m))
        s = e.sum(1, keepdims=True)
        return e / np.where(s == 0, 1.0, s)


def route(l, k, score="softmax", bias=None, groups=1, top_groups=1, group_sum=1, renormalise=True, scale=1.0,
          valid=None):
    """(experts, weights, offsets, pos, src) of finite or masked (-inf) logits l [T, E]."""
    l = np.asarray(l, dtype=np.float64)
    T, E = l.shape
    s = scores(l, score) if T else l
    c = l if bias is None and (groups == 1 or group_sum == 1) else s + (0 if bias is None else np.asarray(bias, np.float64))
    c = np.where(np.isneginf(l), -np.inf, c)
    if valid is not None:
        c = np.where(np.asarray(valid)[:, None], c, -np.inf)
    experts = np.full((T, k), -1, dtype=np.int64)
    for t in range(T):
        row = c[t].copy()
        if groups > 1:
            g = row.reshape(groups, -1)
            value = []
            for v in g:
                best = sorted((x for x in v if x > -np.inf), reverse=True)[:group_sum]
                value.append(sum(best) if best else -np.inf)
            kept = sorted(range(groups), key=lambda i: (-value[i], i))[:top_groups]
            for i in range(groups):
                if i not in kept:
                    g[i] = -np.inf
        order = np.argsort(-row, kind="stable")[:k]
        for j, e in enumerate(order):
            if row[e] > -np.inf:
                experts[t, j] = e
    used = experts >= 0
    at = np.where(used, experts, 0)
    if renormalise:     # ratios from the scores' logarithms, which do not underflow
        z = np.take_along_axis(l, at, 1) if T else np.zeros((0, k))
        if score == "sigmoid":
            z = np.minimum(z, 0) - np.log1p(np.exp(-np.abs(z)))
        z = np.where(used, z, -np.inf)
        m = z.max(1, keepdims=True) if T else z
        e = np.where(used, np.exp(z - np.where(np.isneginf(m), 0.0, m)), 0.0)
        w = e / np.where(e.sum(1, keepdims=True) == 0, 1.0, e.sum(1, keepdims=True))
    else:
        w = np.where(used, np.take_along_axis(s, at, 1), 0.0) if T else np.zeros((0, k))
    owner = np.where(used, experts, E).reshape(-1)
    src = np.argsort(owner, kind="stable")
    pos = np.empty(T * k, dtype=np.int64)
    pos[src] = np.arange(T * k)
    offsets = np.searchsorted(owner[src], np.arange(E + 1))
    return experts, w * scale, offsets, pos.reshape(T, k), src


def route_grad(l, experts, w, dw, score, renormalise, scale):
    """(dlogits, the sum of the magnitudes that entered each) in 64 bits."""
    l = np.asarray(l, dtype=np.float64)
    used = experts >= 0
    at = np.where(used, experts, 0)
    g = np.where(used, np.asarray(dw, np.float64), 0.0)
    a = w / scale
    s = scores(l, score)
    rest = scores(-l, score) if score == "sigmoid" else None      # 1 - s, also where s rounds to 1
    rows = np.arange(len(l))[:, None]
    out, mag = np.zeros_like(l), np.zeros_like(l)
    dot, adot = (g * a).sum(1, keepdims=True), np.abs(g * a).sum(1, keepdims=True)
    if renormalise:
        f = np.take_along_axis(rest, at, 1) if score == "sigmoid" else 1.0
        np.add.at(out, (rows, at), scale * a * f * (g - dot) * used)
        np.add.at(mag, (rows, at), np.abs(scale * a * f * (np.abs(g) + adot) * used))
    elif score == "sigmoid":
        d = scale * a * np.take_along_axis(rest, at, 1) * g
        np.add.at(out, (rows, at), d)
        np.add.at(mag, (rows, at), np.abs(d))
    else:
        np.add.at(out, (rows, at), scale * a * g)
        np.add.at(mag, (rows, at), np.abs(scale * a * g))
        out -= s * scale * dot
        mag += np.abs(s * scale * adot)
    return out, mag
