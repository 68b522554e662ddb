"""Batch-row operators on the GPU against their definitions in 64 bits (tests/rows_ref.py): dropout,
gather with dropout, routing, dispatch and combine, forward and backward; masks that leave rows
empty, ties, odd sizes, strides, replayed graphs, streams.

Tolerances: u = 2^-24 is half a step of a 32-bit result.  A stored value is off by at most half a
step of its type on top of what the 32-bit arithmetic before it may be off, which each test bounds
from the number of roundings and the magnitudes that enter."""
import numpy as np
import pytest
import torch

from partiallyshuffledistributedsampler_amd import ops
from partiallyshuffledistributedsampler_amd.engine import IndexEngine
from tests import rows_ref as R
from tests.test_ops_cpu import DT, check

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def dev():
    return torch.device("cuda", 0)


def rnd(seed, *shape, dtype="fp32", scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale).to(DT[dtype]).to(dev())


def f64(t):
    return t.detach().double().cpu().numpy()


# ---- dropout -------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 8), (3, 7), (17, 9), (5, 64), (64, 1000), (33, 1537), (700, 24),
                                       (2, 70001), (20000, 3), (1025, 512), (300, 4100)])
def test_dropout_equals_the_cpu_mode(dtype, rows, cols):
    # the CPU mode is held to the definition in test_ops_cpu.py; the GPU gives the same bits
    x, res = rnd(rows, rows, cols, dtype=dtype), rnd(cols, rows, cols, dtype=dtype)
    key = 0xD1B54A32D192ED03 * rows & (1 << 64) - 1
    for p, row0 in ((0.1, (1 << 32) - 5), (0.5, 0), (0.0, 3), (1.0, 3)):
        for r in (None, res):
            got = ops.dropout(x, p, key, rows=row0, residual=r)
            want = ops.dropout(x.cpu(), p, key, rows=row0, residual=None if r is None else r.cpu())
            assert torch.equal(got.cpu(), want), (p, r is not None)


@pytest.mark.parametrize("dtype", list(DT))
def test_dropout_gradient_ids_and_strides(dtype):
    n, d = 37, 203
    x, res, dy = (rnd(i, n, d, dtype=dtype).requires_grad_() for i in (1, 2, 3))
    ids = torch.randint(0, 1 << 62, (n,))
    f = R.factor(ids.tolist(), d, 0.35, 99)
    y = ops.dropout(x, 0.35, 99, rows=ids.to(dev()), residual=res)
    check(y, R.drop(f64(x), f) + f64(res), DT[dtype], extra=2 * U * (np.abs(f64(x) * f) + np.abs(f64(res))))
    dx, dres = torch.autograd.grad(y, (x, res), dy)
    check(dx, R.drop(f64(dy), f), DT[dtype], extra=U * np.abs(f64(dy) * f))
    assert torch.equal(dres, dy)
    # a linear map: its difference in any direction is the map of that direction
    # strided, transposed, broadcast rows and gradients
    wide = rnd(5, n, d + 9, dtype=dtype)
    for v in (wide[:, 4:4 + d], wide[::3, 1:], wide.t(), wide[:1].expand(8, -1), wide[:, :1].expand(-1, 24)):
        assert torch.equal(ops.dropout(v, 0.5, 7), ops.dropout(v.contiguous(), 0.5, 7))
    y = ops.dropout(x, 0.5, 7)
    y.sum().backward()
    ones = torch.ones(n, d, dtype=DT[dtype], device=dev())
    assert torch.equal(x.grad, ops.dropout(ones, 0.5, 7))


def test_dropout_of_infinities_and_nan():
    x = torch.tensor([float("inf"), float("nan"), -float("inf"), 1.0], device=dev()).repeat(512).reshape(16, 128)
    y = ops.dropout(x, 0.5, 11)
    f = R.factor(range(16), 128, 0.5, 11)
    assert (y.cpu().numpy()[f == 0] == 0).all()
    assert np.array_equal(np.isnan(y.cpu().numpy())[f != 0], np.isnan(x.cpu().numpy())[f != 0])


def test_dropout_more_than_2_31_values():
    # offsets that pass 32 bits: the last rows of a tensor of 2^31 + values equal those rows alone
    rows, cols = (1 << 20) + 3, 2056
    x = torch.ones(rows, cols, dtype=torch.bfloat16, device=dev())
    y = ops.dropout(x, 0.25, 3, rows=10)
    assert torch.equal(y[-5:], ops.dropout(x[-5:], 0.25, 3, rows=10 + rows - 5))
    assert torch.equal(y[:3], ops.dropout(x[:3], 0.25, 3, rows=10))
    del x, y


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("shape", [(8,), (5, 3), (1000,), (257,)])
def test_gather_with_dropout(dtype, shape):
    lens = [50, 31, 97, 1, 41]
    total = sum(lens)
    eng = IndexEngine(lens, total, 1, 16, 2, seed=5, device=0)
    eng.init_iter(2)
    fpos, off = eng.generate_mapped(0, 1)
    data = rnd(8, total, *shape, dtype=dtype)
    base = torch.tensor(np.concatenate([[0], np.cumsum(lens)[:-1]]), device=dev())
    plain = eng.gather(data, base, fpos, off)
    for p in (0.3, 1.0):
        got = eng.gather(data, base, fpos, off, p=p, key=42, rows=1 << 33)
        want = ops.dropout(plain.reshape(total, -1), p, 42, rows=1 << 33).reshape(plain.shape)
        assert torch.equal(got, want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = eng.gather(data, base, fpos[:, ::2], off[:, ::2].long(), p=0.3, key=42, stream=side)
    side.synchronize()
    assert torch.equal(got.reshape(len(got), -1), ops.dropout(plain.reshape(total, -1)[::2], 0.3, 42))
    out = torch.empty_like(plain)
    assert eng.gather(data, base, fpos[:, :7], off[:, :7], out=out[:7], p=0.3, key=42).data_ptr() == out.data_ptr()
    assert torch.equal(out[:7], ops.dropout(plain.reshape(total, -1)[:7], 0.3, 42).reshape(7, *shape))
    with pytest.raises(ValueError, match="out must be"):
        eng.gather(data, base, fpos, off, out=out[:7], p=0.3)
    with pytest.raises(TypeError, match="float32"):
        eng.gather(data.to(torch.float64), base, fpos, off, p=0.3)
    with pytest.raises(ValueError, match="one length"):
        eng.gather(data, base, fpos, off[:, :5], p=0.3)
    with pytest.raises(ValueError, match="one length"):
        eng.gather(data, base[:4], fpos, off, p=0.3)
    eng.close()


def test_gather_with_dropout_is_not_captured():
    # a replay after later epochs would read a file order that is no longer there
    lens = [50, 31, 97, 1, 41]
    eng = IndexEngine(lens, 220, 1, 16, 2, seed=5, device=0)
    base = torch.tensor(np.concatenate([[0], np.cumsum(lens)[:-1]]), device=dev())
    data = rnd(1, 220, 24)
    for epoch in (2, 3, 4):
        eng.init_iter(epoch)
        fpos, off = eng.generate_mapped(0, 1)
        want = ops.dropout(eng.gather(data, base, fpos, off), 0.3, 42)
        torch.cuda.synchronize()
        with pytest.raises(RuntimeError, match="cannot be captured"):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                eng.gather(data, base, fpos, off, p=0.3, key=42)
        assert torch.equal(eng.gather(data, base, fpos, off, p=0.3, key=42), want)
    eng.close()


@pytest.mark.parametrize("dtype,rows,cols", [
    ("fp32", 300, 1375), ("fp32", 300, 2048), ("fp16", 300, 1375), ("bf16", 300, 2047), ("bf16", 300, 2049), ("bf16", 300, 2056), ("fp32", 120, 4099), ("fp16", 2500, 2055), ("bf16", 40000, 2056),
    ("fp32", 20000, 2051), ("bf16", 650000, 40), ("fp16", 560000, 33), ("fp32", 300000, 130)])
def test_gather_with_dropout_of_wide_and_of_many_rows(dtype, rows, cols):
    # wide rows, more bytes than the caches hold, and more blocks of eight than one pass of the workgroups
    lens = [rows // 4, rows // 8, 1, rows - rows // 4 - rows // 8 - 1]
    eng = IndexEngine(lens, rows, 1, 4096, 2, seed=5, device=0)
    eng.init_iter(1)
    fpos, off = eng.generate_mapped(0, 1)
    base = torch.tensor(np.concatenate([[0], np.cumsum(lens)[:-1]]), device=dev())
    data = torch.randn(rows, cols, device=dev(), dtype=torch.float32, generator=torch.Generator(dev()).manual_seed(cols)).to(DT[dtype])
    got = eng.gather(data, base, fpos, off, p=0.3, key=42, rows=7)
    plain = eng.gather(data, base, fpos, off)
    order = torch.from_numpy(eng.file_order().astype(np.int64)).to(dev())
    assert torch.equal(plain, data[base[order[fpos[0].long()]] + off[0].long()])
    # the definition at the first, the last and some rows between
    at = torch.cat([torch.arange(20), torch.arange(rows - 20, rows), torch.randint(0, rows, (60,), generator=torch.Generator().manual_seed(1))])
    f = R.factor([7 + i for i in at.tolist()], cols, 0.3, 42)
    v = f64(plain[at.to(dev())])
    check(got[at.to(dev())], R.drop(v, f), DT[dtype], extra=U * np.abs(v * f))
    assert torch.equal(got, ops.dropout(plain, 0.3, 42, rows=7))
    eng.close()


# ---- routing -------------------------------------------------------------------------------------
def exponents(l, score):
    """[T, 1] the largest exponent that a row's weights go through: differences of logits (exp is 0
    in 32 bits beyond 110 below the maximum), or logarithms of sigmoids."""
    finite = np.isfinite(l)
    top = np.where(finite, l, -np.inf).max(1, keepdims=True, initial=-np.inf)
    low = np.where(finite, l, np.inf).min(1, keepdims=True, initial=np.inf)
    far = np.maximum(np.abs(top), np.abs(low)) * 2 if score == "sigmoid" else np.clip(top - low, 0, 110)
    return np.where(np.isfinite(top), far, 0.0)


def weight_bound(l, k, score, w):
    """How far a weight may be: an exponent z is off by z * u, and every sum, product, quotient and
    function adds a few u: (2 z + 2 k + 40) u of it."""
    return (2 * exponents(l, score) + 2 * k + 40) * U * np.abs(w)


def check_route(logits, k, grad=True, seed=0, **kw):
    logits = logits.detach().requires_grad_(grad)
    r = ops.route(logits, k, **kw)
    l = f64(logits)
    ref = dict(kw)
    for n in ("bias", "valid"):
        if ref.get(n) is not None:
            ref[n] = ref[n].cpu().numpy()
    experts, w, offsets, pos, src = R.route(l, k, **ref)
    assert np.array_equal(r.experts.cpu().numpy(), experts)
    assert np.array_equal(r.offsets.cpu().numpy(), offsets)
    assert np.array_equal(r.pos.cpu().numpy(), pos)
    assert np.array_equal(r.src.cpu().numpy(), src)
    score, renorm, scale = kw.get("score", "softmax"), kw.get("renormalise", True), kw.get("scale", 1.0)
    off = np.abs(f64(r.weights) - w)
    bound = weight_bound(l, k, score, w)
    tiny = 2.0 ** -126 * abs(scale)            # scores below the normal numbers
    assert (off <= bound + tiny).all(), (off - bound).max()
    if grad and logits.shape[0]:
        dw = rnd(seed + 77, *w.shape)
        dl, = torch.autograd.grad(r.weights, logits, dw)
        want, mag = R.route_grad(l, experts, w, f64(dw), score, renorm, scale)
        # (a weight that vanished was at most `tiny`, and stood with the row's |dw| in the gradient)
        lost = tiny * (1 + 2 * np.abs(f64(dw)).sum(1, keepdims=True))
        check(dl, want, logits.dtype, extra=(4 * exponents(l, score) + 6 * k + 120) * U * mag + lost)
    return r


SHAPES = [
    # T, E, k, keywords
    (1, 1, 1, {}), (5, 2, 2, {}), (3, 7, 3, dict(renormalise=False)), (1, 16, 16, {}), (9, 17, 4, dict(score="sigmoid")),
    (8, 64, 4, {}), (255, 60, 6, dict(renormalise=False)), (256, 64, 8, dict(score="sigmoid", renormalise=False)),
    (257, 33, 2, dict(scale=2.5)), (1000, 128, 8, {}), (700, 129, 16, dict(score="sigmoid", scale=0.5)),
    (513, 256, 8, dict(groups=16, top_groups=6, group_sum=2, score="sigmoid", bias=True, scale=2.5)),
    (300, 256, 8, dict(groups=8, top_groups=4, score="softmax")),
    (300, 96, 5, dict(groups=4, top_groups=2, group_sum=2, score="softmax", renormalise=False)),
    (130, 40, 10, dict(groups=40, top_groups=20, group_sum=2, bias=True)),
    (64, 512, 8, dict(groups=64, top_groups=3, group_sum=1, bias=True, score="sigmoid")),
    (70, 320, 12, dict(groups=2, top_groups=1, group_sum=2, bias=True, score="softmax")),
    (150, 394, 1, dict(groups=2, top_groups=1, group_sum=2, bias=True, score="sigmoid", renormalise=False)),
    (150, 36, 3, dict(groups=4, top_groups=3, group_sum=2)), (70, 300, 4, dict(groups=60, top_groups=10, group_sum=2)),
    (70, 264, 4, dict(groups=24, top_groups=10, bias=True)), (70, 90, 4, dict(groups=30, top_groups=4, group_sum=2)),
    (40, 257, 16, dict(bias=True)), (33, 600, 7, dict(score="sigmoid", bias=True, renormalise=False)),
    (20, 1024, 16, dict(groups=32, top_groups=32, group_sum=2, score="sigmoid")), (3, 1024, 1, dict(renormalise=False)),
]


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("T,E,k,kw", SHAPES, ids=str)
def test_route(dtype, T, E, k, kw):
    kw = dict(kw)
    if kw.pop("bias", False):
        kw["bias"] = rnd(4, E, scale=0.1)
    check_route(rnd(T * E, T, E, dtype=dtype), k, **kw)
    # a padded batch with masked experts, an empty row, far and close logits
    l = rnd(T * E + 1, T, E, dtype=dtype, scale=4.0)
    g = torch.Generator().manual_seed(E)
    l = l.masked_fill((torch.rand(T, E, generator=g) < 0.3).to(dev()), float("-inf"))
    l[T // 2] = float("-inf")
    check_route(l, k, valid=(torch.rand(T, generator=g) < 0.8).to(dev()), **kw)


@pytest.mark.parametrize("T", [0, 1, 255, 256, 257, 511, 513, 5000, 40000])
def test_route_order_of_many_rows(T):
    check_route(rnd(T, T, 12), 3, valid=torch.rand(T, generator=torch.Generator().manual_seed(1)).to(dev()) < 0.7)


@pytest.mark.parametrize("E,k,kw", [
    (64, 8, {}), (60, 4, dict(renormalise=False)), (33, 16, dict(score="sigmoid", bias=True)), (30, 3, dict(groups=5, top_groups=2)),
    (32, 8, dict(groups=8, top_groups=5, group_sum=2)), (64, 6, dict(groups=64, top_groups=10, group_sum=2, bias=True)),
    (36, 1, dict(groups=4, top_groups=3, group_sum=2, score="sigmoid")), (16, 16, {}), (9, 2, dict(bias=True)), (5, 5, {}), (4, 3, {}), (3, 2, {}),
    (2, 2, dict(score="sigmoid")), (1, 1, {})],
    ids=str)
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_route_of_many_rows_over_few_experts(E, k, kw, dtype):
    T, kw = 8300, dict(kw)
    if kw.pop("bias", False):
        kw["bias"] = rnd(4, E, scale=0.1)
    l = rnd(T + E, T, E, dtype=dtype, scale=2.0)
    g = torch.Generator().manual_seed(E)
    l = l.masked_fill(((torch.rand(T, 1, generator=g) < 0.1) & (torch.rand(T, E, generator=g) < 0.6)).to(dev()), float("-inf"))
    check_route(l, k, valid=(torch.rand(T, generator=g) < 0.9).to(dev()), **kw)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("T,E,k,kw", [
    (600, 300, 4, {}), (8300, 300, 8, {}), (8300, 520, 3, dict(score="sigmoid", bias=True)),
    (700, 320, 6, dict(groups=10, top_groups=4, group_sum=2, score="sigmoid", bias=True, scale=2.5)),
    (8200, 384, 8, dict(groups=12, top_groups=6, group_sum=2, renormalise=False)),
    (8200, 512, 8, dict(groups=16, top_groups=4, score="sigmoid", renormalise=False)),
    (530, 900, 16, dict(groups=10, top_groups=5, group_sum=2)), (530, 1000, 2, dict(groups=40, top_groups=9, bias=True))],
    ids=str)
def test_route_of_many_rows_over_many_experts(dtype, T, E, k, kw):
    kw = dict(kw)
    if kw.pop("bias", False):
        kw["bias"] = rnd(4, E, scale=0.1)
    l = rnd(T + E, T, E, dtype=dtype, scale=2.0)
    g = torch.Generator().manual_seed(E)
    l = l.masked_fill(((torch.rand(T, 1, generator=g) < 0.1) & (torch.rand(T, E, generator=g) < 0.6)).to(dev()), float("-inf"))
    l[T // 2] = float("-inf")
    check_route(l, k, valid=(torch.rand(T, generator=g) < 0.9).to(dev()), **kw)


def test_route_of_a_million_rows():
    # more rows than one workgroup's counts can hold: the order is checked by its properties
    T, E, k = 1 << 20, 20, 2
    r = ops.route(rnd(2, T, E, dtype="bf16"), k)
    e = r.experts.reshape(-1).long()
    assert torch.equal(r.offsets.long(), torch.cat([e.new_zeros(1), torch.bincount(e, minlength=E).cumsum(0)]))
    assert torch.equal(r.src.long(), torch.sort(e, stable=True)[1])
    assert torch.equal(r.pos.reshape(-1)[r.src.long()].long(), torch.arange(T * k, device=dev()))


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_route_ties_go_to_the_lowest_index(dtype, score):
    l = torch.zeros(7, 50, dtype=DT[dtype], device=dev())
    assert check_route(l, 4, score=score).experts.tolist() == [[0, 1, 2, 3]] * 7
    l[:, 1::2] = -0.0                                    # equal to 0
    assert check_route(l, 4, score=score).experts.tolist() == [[0, 1, 2, 3]] * 7
    g = torch.Generator().manual_seed(3)
    l = torch.randint(-2, 3, (900, 50), generator=g).to(DT[dtype]).to(dev())
    bias = (torch.randint(0, 2, (50,), generator=g).float() * 0.25).to(dev())
    for kw in ({}, dict(bias=bias), dict(groups=10, top_groups=5, group_sum=2), dict(groups=5, top_groups=2, bias=bias),
               dict(groups=25, top_groups=9)):
        check_route(l, 6, score=score, **kw)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("bias", [False, True])
def test_route_close_scores_are_told_apart(score, bias):
    # neighbours in 32 bits, and scores that differ far below 32 bits
    l = torch.full((64, 40), 1.0)
    l += torch.arange(40).flip(0) * 2.0 ** -23
    l[32:] *= -1
    b = torch.full((40,), 0.5, device=dev()) if bias else None
    check_route(l.to(dev()), 8, score=score, bias=b)
    check_route(l.to(dev()), 8, score=score, bias=b, groups=8, top_groups=3, group_sum=2)
    check_route((l + torch.randn(64, 40, generator=torch.Generator().manual_seed(2)) * 1e-6).to(dev()), 8, score=score,
                bias=b, groups=4, top_groups=2, group_sum=2)


@pytest.mark.parametrize("dtype", list(DT))
def test_route_extreme_logits(dtype):
    big = torch.finfo(DT[dtype]).max
    l = rnd(6, 40, 20, dtype=dtype)
    l[0], l[1] = -big, big                               # masks of the type's lowest value
    l[2, 3:] = -big
    l[3, :] = torch.arange(20) * -30.0
    l[4, 5:] = float("-inf")
    kw = dict(score="softmax")
    check_route(l, 4, **kw)
    check_route(l, 4, renormalise=False, **kw)
    small = l.clamp(-60, 60)
    small[4, 5:] = float("-inf")
    check_route(small, 4, score="sigmoid")
    check_route(small, 4, score="sigmoid", renormalise=False)
    # sigmoids that vanish in 32 bits still have ratios
    far = torch.full((2, 4), -200.0)
    far[:, 1] = -201.0
    w = ops.route(far.to(DT[dtype]).to(dev()), 2, score="sigmoid").weights
    assert torch.allclose(w.sum(1), torch.ones(2, device=dev())) and (w > 0.2).all()


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("E", [8, 60, 300])
def test_route_weights_far_below_the_best(dtype, E):
    # The exponents are exact.  expf is within 2 u; the row's sum, of 1 and terms below 5e-5, goes through
    # at most 8 additions in a lane and 6 across lanes, u each; the quotient and the scale are u each: 18 u
    l = torch.full((E, E), -100.0)
    at = torch.arange(E)
    far = -(10.0 + at * 77.0 / E).floor()               # -10 .. -87
    l[:, 0] = 0.0
    l[at[1:], at[1:]] = far[1:]
    l = l.to(DT[dtype]).to(dev())
    ld = f64(l)
    for renorm in (False, True):
        r = ops.route(l, 2, renormalise=renorm)
        w = np.exp(ld)
        w = w / (w.sum(1, keepdims=True) if not renorm else np.sort(w, 1)[:, -2:].sum(1, keepdims=True))
        want = np.take_along_axis(w, r.experts.long().cpu().numpy(), 1)[1:]
        off = np.abs(f64(r.weights)[1:] / want - 1)
        assert (off <= 18 * U).all(), off.max() / U


@pytest.mark.parametrize("renormalise", [False, True])
def test_route_sigmoid_weights_far_below_the_best(renormalise):
    # expf within 2 u, a sum, a quotient (renormalised: two of each) and the scale 1 u each
    n = 78
    l = torch.stack([torch.zeros(n), -torch.arange(10.0, 10 + n)], 1).to(dev()).requires_grad_()
    for shift in (0.0, -60.0 if renormalise else 0.0, 60.0 if renormalise else 0.0):
        ls = (l.detach() + shift).requires_grad_()
        r = ops.route(ls, 2, score="sigmoid", renormalise=renormalise)
        s = R.scores(f64(ls), "sigmoid")
        want = s / s.sum(1, keepdims=True) if renormalise else s
        off = np.abs(f64(r.weights) / want - 1)
        assert (off <= 10 * U).all(), off.max() / U
    # and 1 - s of the gradient, where s is 1 in 32 bits
    up = (-l.detach()).requires_grad_()
    d, = torch.autograd.grad(ops.route(up, 1, score="sigmoid", renormalise=False).weights.sum(), up)
    want = R.scores(-f64(up)[:, 1], "sigmoid") * R.scores(f64(up)[:, 1], "sigmoid")
    off = np.abs(f64(d)[:, 1] / want - 1)
    assert (off <= 12 * U).all(), off.max() / U


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("groups", [1, 4])
def test_route_of_nan_rows_stays_in_range(score, bias, groups):
    l = rnd(3, 12, 16)
    l[1, 4] = float("nan")
    l[2] = float("nan")
    l[3, 7] = float("inf")
    l[4, :15] = float("-inf")
    l[4, 15] = float("nan")
    b = torch.zeros(16, device=dev()) if bias else None
    if bias:
        b[2], b[3] = float("nan"), float("-inf")
    r = ops.route(l, 4, score=score, bias=b, groups=groups, top_groups=max(1, groups // 2), group_sum=2)
    e = r.experts
    assert ((e >= -1) & (e < 16)).all()
    assert e[4].tolist() == [15, -1, -1, -1]
    assert r.weights[1:3].isnan().all() and r.weights[4, 0].isnan() and r.weights[4, 1:].eq(0).all()
    assert r.weights[5:].isfinite().all()
    for row in e.tolist():
        used = [x for x in row if x >= 0]
        assert len(used) == len(set(used))
    if not bias and groups == 1:
        assert 4 not in e[1].tolist() and e[2].tolist() == [0, 1, 2, 3] and e[3, 0] == 7
    assert torch.equal(torch.sort(r.pos.reshape(-1))[0], torch.arange(48, dtype=torch.int32, device=dev()))


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_route_nan_comes_last_of_what_is_not_masked(score):
    nan, inf = float("nan"), float("inf")
    b = torch.tensor([nan, 0.0, 0.25, -inf, 0.0, nan], device=dev())
    l = torch.tensor([[9.0, 1.0, 1.0, 9.0, 3.0, 0.0], [9.0, -inf, 2.0, nan, 1.0, -inf], [-inf, -inf, -inf, 2.0, -inf, -inf]],
                     device=dev())
    r = ops.route(l, 6, score=score, bias=b)
    assert r.experts[0].tolist() == [2, 4, 1, 0, 5, -1]
    assert r.weights[0, :5].isfinite().all() and (r.weights[0, 5] == 0).all()
    # (a softmax with a NaN logit has no number at all: the order of the indexes)
    assert r.experts[1].tolist() == ([2, 4, 0, -1, -1, -1] if score == "sigmoid" else [0, 2, 4, -1, -1, -1])
    assert r.weights[1, :3].isnan().all() and (r.weights[1, 3:] == 0).all()
    assert r.experts[2].tolist() == [-1] * 6 and (r.weights[2] == 0).all()
    assert r.offsets[-1] == 8


def test_route_of_padding_alone_and_of_a_zero_router():
    for T, E, kw in ((300, 40, {}), (9, 7, dict(bias=torch.zeros(7, device=dev()))), (200, 300, dict(groups=4, top_groups=2))):
        l = rnd(T, T, E)
        r = check_route(l, 3, valid=torch.zeros(T, dtype=torch.bool, device=dev()), **kw)
        assert (r.experts == -1).all() and (r.offsets == 0).all() and (r.weights == 0).all()
        check_route(torch.zeros(T, E, device=dev()), 3, **kw)


@pytest.mark.parametrize("bias", [1e9, -1e9, 1e5, 100.0])
@pytest.mark.parametrize("groups", [1, 5])
def test_route_large_biases(bias, groups):
    # experts switched off or forced by their bias
    b = rnd(1, 60, scale=0.1)
    b[::7] += bias
    check_route(rnd(2, 300, 60), 5, bias=b, score="sigmoid", groups=groups, top_groups=max(1, groups // 2), group_sum=2)
    check_route(rnd(3, 300, 60, dtype="bf16"), 5, bias=b, groups=groups, top_groups=max(1, groups // 2))


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("G,S", [(2, 2), (2, 3), (4, 2)])
@pytest.mark.parametrize("bias", [1e3, 1e4])
def test_route_groups_whose_biases_cancel(score, G, S, bias):
    # +B and -B in every group: a group's value is of the scores' size, its terms' rounding of the bias's
    b = torch.full((G, S), -bias)
    b[torch.arange(G), torch.arange(G) % S] = bias
    l = rnd(G * S, 4000, G * S, scale=1e-3)
    check_route(l, 1, score=score, bias=b.reshape(-1).to(dev()), groups=G, top_groups=1, group_sum=2)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("T,E,k,kw", [
    (50, 12, 4, {}), (50, 12, 11, {}), (300, 40, 6, dict(groups=5, top_groups=2, group_sum=2)),
    (300, 40, 6, dict(groups=5, top_groups=4)), (40, 300, 16, dict(groups=60, top_groups=30, group_sum=2)),
    (9000, 24, 3, dict(groups=6, top_groups=3, group_sum=2, renormalise=False))], ids=str)
def test_route_bias_of_minus_infinity_masks_its_expert(dtype, score, T, E, k, kw):
    b = rnd(E, E, scale=0.1)
    b[::3] = float("-inf")
    if "groups" in kw:
        b[:E // kw["groups"]] = float("-inf")           # a whole group
    r = check_route(rnd(T, T, E, dtype=dtype), k, score=score, bias=b, **kw)
    masked = torch.isneginf(b).nonzero().flatten()
    assert not torch.isin(r.experts, masked).any()
    b[:] = float("-inf")
    r = check_route(rnd(T, T, E, dtype=dtype), k, score=score, bias=b, **kw)
    assert (r.experts == -1).all() and (r.weights == 0).all()


def test_plan_that_route_did_not_make_writes_nowhere_else():
    T, k, D = 6, 2, 40
    r = ops.route(rnd(1, T, 4), k)
    x, y = rnd(2, T, D), rnd(3, T * k, D).requires_grad_()
    pos = r.pos.clone()
    pos[2, 1], pos[4, 0] = -5, 1 << 30
    bad = r._replace(pos=pos, weights=r.weights.detach().requires_grad_())
    good = r._replace(experts=r.experts.clone(), weights=r.weights.detach())
    good.experts[2, 1] = good.experts[4, 0] = -1
    xs, want = ops.dispatch(x, bad), ops.dispatch(x, good)
    on = [p for i, p in enumerate(r.pos.reshape(-1).tolist()) if i not in (5, 8)]
    assert torch.equal(xs[on], want[on])
    out = ops.combine(y, bad)
    assert torch.equal(out, ops.combine(y, good))
    dy, dw = torch.autograd.grad(out, (y, bad.weights), torch.ones(T, D, device=dev()))
    assert dw[2, 1] == 0 and dw[4, 0] == 0


def test_route_strided_logits_and_no_gradient():
    wide = rnd(9, 300, 100, dtype="bf16")
    a, b = ops.route(wide[::2, 7:71], 4), ops.route(wide[::2, 7:71].contiguous(), 4)
    for x, y in zip(a, b):
        assert torch.equal(x, y)
    c = ops.route(wide.t(), 4)
    for x, y in zip(c, ops.route(wide.t().contiguous(), 4)):
        assert torch.equal(x, y)
    leaf = wide[::2, 7:71].detach().requires_grad_()
    dw = rnd(1, 4, 150).t()
    d1, = torch.autograd.grad(ops.route(leaf, 4).weights, leaf, dw)
    d2, = torch.autograd.grad(ops.route(leaf.contiguous(), 4).weights, leaf, dw.contiguous())
    assert torch.equal(d1, d2)
    with torch.no_grad():
        assert not ops.route(leaf, 4).weights.requires_grad


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renormalise", [True, False])
@pytest.mark.parametrize("T,E", [(40, 20), (40, 300), (9000, 20)])
def test_route_gradient_ignores_the_logits_of_padding(dtype, score, renormalise, T, E):
    clean = rnd(T + E, T, E, dtype=dtype)
    valid = torch.ones(T, dtype=torch.bool, device=dev())
    valid[::3] = False
    dirty = clean.clone()
    dirty[0, 1], dirty[3, :] = float("nan"), float("nan")
    dirty[6, 2], dirty[9, 3] = float("inf"), float("-inf")
    dirty[12, 0], dirty[12, 1] = float("inf"), float("nan")
    dirty[15, :] = float("-inf")
    dw = rnd(7, T, 3)

    def passes(l):
        l = l.detach().requires_grad_()
        r = ops.route(l, 3, score=score, renormalise=renormalise, valid=valid)
        return tuple(r) + torch.autograd.grad(r.weights, l, dw)

    got, want = passes(dirty), passes(clean)
    assert (got[-1][::3] == 0).all()
    for a, b in zip(got, want):
        assert torch.equal(a, b)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("scale", [1.0, 2.5, 0.3])
def test_route_gradient_of_an_only_expert_is_zero(score, scale):
    # a renormalised weight of one expert is the scale, whatever the logit
    l = rnd(3, 900, 20)
    l[::2, 1:] = float("-inf")
    l.requires_grad_()
    for k in (1, 3):
        r = ops.route(l, k, score=score, scale=scale)
        d, = torch.autograd.grad(r.weights, l, rnd(4, 900, k))
        one = (r.experts >= 0).sum(1) == 1
        assert one.sum() == (900 if k == 1 else 450)
        assert (r.weights[one][:, 0] == torch.tensor(scale, device=dev())).all() and (d[one] == 0).all()
        assert k == 1 or (d[~one] != 0).any()


@pytest.mark.parametrize("kw", [dict(), dict(renormalise=False), dict(score="sigmoid"),
                                dict(score="sigmoid", renormalise=False, scale=2.0)], ids=str)
def test_route_gradient_against_differences(kw):
    # third derivatives of the scores are below 2, so a central difference of step h is off by
    # h^2 / 3 * scale a unit of |dw|, and by the weights' rounding over h
    T, E, k, h = 6, 12, 3, 2.0 ** -6
    l = (torch.arange(E).float() * 0.25)[torch.stack([torch.randperm(E, generator=torch.Generator().manual_seed(i))
                                                      for i in range(T)])].to(dev())   # gaps wider than 2 h
    l.requires_grad_()
    dw = rnd(5, T, k)
    r = ops.route(l, k, **kw)
    dl, = torch.autograd.grad(r.weights, l, dw)
    scale = kw.get("scale", 1.0)
    tol = (h * h / 3 * 8 + 60 * U / h) * scale * dw.abs().sum(1).max().item()
    with torch.no_grad():
        for e in range(E):
            d = torch.zeros(E, device=dev())
            d[e] = h
            up, down = ops.route(l + d, k, **kw), ops.route(l - d, k, **kw)
            assert torch.equal(up.experts, r.experts) and torch.equal(down.experts, r.experts)
            diff = ((up.weights - down.weights) * dw).sum(1) / (2 * h)
            assert (diff - dl[:, e]).abs().max().item() <= tol


# ---- dispatch and combine ------------------------------------------------------------------------
def plan_of(T, E, k, seed, empty=True):
    l = rnd(seed, T, E)
    valid = None
    if empty and T:
        g = torch.Generator().manual_seed(seed)
        l = l.masked_fill((torch.rand(T, E, generator=g) < 0.4).to(dev()), float("-inf"))
        l[T // 2] = float("-inf")
        valid = (torch.rand(T, generator=g) < 0.8).to(dev())
    return ops.route(l, k, valid=valid)


MOVES = [(0, 4, 2, 8), (1, 1, 1, 1), (1, 8, 8, 16), (5, 4, 2, 7), (16, 64, 4, 2048), (33, 10, 3, 1001), (130, 9, 5, 520),
         (300, 16, 16, 24), (64, 6, 1, 9000), (4, 8, 6, 20000), (5000, 4, 2, 40), (2500, 12, 8, 513)]


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("T,E,k,D", MOVES, ids=str)
def test_dispatch_and_combine(dtype, T, E, k, D):
    t = DT[dtype]
    r = plan_of(T, E, k, T + D)
    w = r.weights.detach().requires_grad_()
    r = r._replace(weights=w)
    x, res, dout = rnd(1, T, D, dtype=dtype), rnd(2, T, D, dtype=dtype), rnd(3, T, D, dtype=dtype)
    ys, dxs = rnd(4, T * k, D, dtype=dtype), rnd(5, T * k, D, dtype=dtype)
    for v in (x, res, ys):
        v.requires_grad_()
    p, key, row0 = 0.2, 5, (1 << 32) - 7
    xs = ops.dispatch(x, r)
    out = ops.combine(ys, r, residual=res, p=p, key=key, rows=row0)
    dx, dys, dw, dres = torch.autograd.grad((xs, out), (x, ys, w, res), (dxs, dout))
    used = r.experts.cpu().numpy() >= 0
    pos, wd = r.pos.cpu().numpy(), f64(w)
    f = R.factor([row0 + i for i in range(T)], D, p, key)
    X, Y, DX, G = f64(x), f64(ys), f64(dxs), R.drop(f64(dout), f)
    rows = np.where(used[..., None], Y[pos], 0.0)
    want = np.zeros((T * k, D))
    want[pos[used]] = np.repeat(X[:, None], k, 1)[used]
    assert np.array_equal(f64(xs), want)
    parts = wd[..., None] * rows
    mag = np.abs(parts).sum(1)
    check(out, R.drop(parts.sum(1), f) + f64(res), t, extra=U * ((k + 3) * mag * f + 2 * np.abs(f64(res))))
    g = np.where(used[..., None], DX[pos], 0.0)
    check(dx, g.sum(1), t, extra=U * k * np.abs(g).sum(1))
    want = np.zeros((T * k, D))
    want[pos[used]] = (wd[..., None] * G[:, None])[used]
    check(dys, want, t, extra=3 * U * np.abs(want))
    check(dw, (G[:, None] * rows).sum(2), torch.float32, extra=U * (D + 4) * (np.abs(G)[:, None] * np.abs(rows)).sum(2))
    assert torch.equal(dres, dout)
    # without dropout, residual and gradients
    with torch.no_grad():
        check(ops.combine(ys, r), parts.sum(1), t, extra=U * k * mag)
        assert torch.equal(ops.dispatch(x, r), xs)


def test_combine_gradients_one_at_a_time_and_strides():
    T, E, k, D = 40, 6, 3, 72
    r = plan_of(T, E, k, 3)
    w = r.weights.detach().requires_grad_()
    y, dout = rnd(1, T * k, D).requires_grad_(), rnd(2, T, 2 * D)[:, 3:3 + D]
    both = torch.autograd.grad(ops.combine(y, r._replace(weights=w), p=0.5, key=1), (y, w), dout)
    only_y, = torch.autograd.grad(ops.combine(y, r._replace(weights=w.detach()), p=0.5, key=1), y, dout.contiguous())
    only_w, = torch.autograd.grad(ops.combine(y.detach(), r._replace(weights=w), p=0.5, key=1), w, dout)
    assert torch.equal(both[0], only_y) and torch.equal(both[1], only_w)
    x = rnd(3, T, 2 * D)
    assert torch.equal(ops.dispatch(x[:, 5:5 + D], r), ops.dispatch(x[:, 5:5 + D].contiguous(), r))
    assert torch.equal(ops.combine(y, r, residual=x[:, 5:5 + D]), ops.combine(y, r, residual=x[:, 5:5 + D].contiguous()))
    assert torch.equal(ops.combine(y.t().contiguous().t(), r), ops.combine(y, r))
    shared = rnd(4, 1, D).expand(T, D)                    # one row for all
    assert torch.equal(ops.dispatch(shared, r), ops.dispatch(shared.contiguous(), r))
    # a gradient that is one value for all
    a, = torch.autograd.grad(ops.combine(y, r).sum(), y)
    b, = torch.autograd.grad(ops.combine(y, r), y, torch.ones(T, D, device=dev()))
    assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("D", [8, 9, 10, 11, 12, 13, 14, 15, 121, 129, 135, 255, 257, 263, 509, 513, 1023, 1031, 2055])
def test_a_value_does_not_depend_on_the_width(dtype, D):
    # the first D columns of rows of more of them: the same bits, but for the sums over a row
    T, k, wide, kw = 37, 3, 2304, dict(p=0.3, key=11, rows=5)
    r = plan_of(T, 8, k, D)
    w = r.weights.detach().requires_grad_()
    r = r._replace(weights=w)
    x, res, dout = (rnd(i, T, wide, dtype=dtype) for i in (1, 2, 3))
    ys = rnd(4, T * k, wide, dtype=dtype)
    dout[:, D:] = 0

    def passes(n):
        y = ys[:, :n].contiguous().requires_grad_()
        out = ops.combine(y, r, residual=res[:, :n], **kw)
        dy, dw = torch.autograd.grad(out, (y, w), dout[:, :n])
        a = x[:, :n].contiguous()
        return dw, ops.dropout(a, 0.3, 11), ops.dropout(a, 0.3, 11, residual=res[:, :n]), ops.dispatch(a, r), \
            ops.combine(y, r), out, dy

    got, want = passes(D), passes(wide)
    for a, b in zip(got[1:], want[1:]):
        assert torch.equal(a, b[:, :D])
    # both sums: D roundings of products of g, y and 10/7
    used = (r.experts >= 0)[..., None]
    rows = torch.where(used, ys[:, :D].double()[r.pos.long()], 0.0)
    mag = (dout[:, None, :D].double() * rows).abs().sum(2) * 65536 / 45875
    assert ((got[0].double() - want[0].double()).abs() <= 2 * U * (wide + 4) * mag).all()


def test_dispatch_past_2_31_values():
    T, k, D = 70000, 8, 4096                              # 2.3e9 values of expert-ordered rows
    r = ops.route(rnd(1, T, 16), k)
    x = rnd(2, 1000, D, dtype="bf16").repeat(70, 1)
    xs = ops.dispatch(x, r)
    for t in (0, 34567, T - 1):
        for j in (0, k - 1):
            assert torch.equal(xs[r.pos[t, j].item()], x[t])
    last = int(r.src[-1])
    assert torch.equal(xs[-1], x[last // k])
    out = ops.combine(xs, r)                              # the weights of a row sum to 1
    assert (out[-100:].float() - x[-100:].float()).abs().max().item() <= 2 ** -8 * 6 * 1.01
    del xs, out


@pytest.mark.parametrize("dtype,T,k,D", [
    ("bf16", 300000, 8, 72), ("fp16", 270000, 2, 130), ("bf16", 20000, 4, 1024), ("bf16", 10000, 8, 1025),
    ("fp32", 9000, 16, 520), ("bf16", 140000, 4, 4096)])
def test_combine_and_gradients_of_many_rows(dtype, T, k, D):
    # narrow rows of more blocks than one pass of the workgroups, more bytes than the caches hold, more
    # than 2^31 values; the first, the last and some rows between against the definition
    gen = torch.Generator(dev()).manual_seed(D)

    def big(*shape):
        return torch.randn(*shape, device=dev(), generator=gen, dtype=torch.float32 if T * k * D < 1 << 30 else DT[dtype]).to(DT[dtype])

    r = ops.route(rnd(3, T, 20, dtype="bf16"), k, valid=(torch.rand(T, generator=torch.Generator().manual_seed(2)) < 0.9).to(dev()))
    w = r.weights.detach().requires_grad_()
    r = r._replace(weights=w)
    y, res, dout, x = big(T * k, D).requires_grad_(), big(T, D), big(T, D), big(T, D).requires_grad_()
    out = ops.combine(y, r, residual=res, p=0.2, key=5, rows=11)
    dy, dw = torch.autograd.grad(out, (y, w), dout)
    xs = ops.dispatch(x, r)
    dx, = torch.autograd.grad(xs, x, y.detach())
    at = torch.cat([torch.arange(20), torch.arange(T - 20, T), torch.randint(0, T, (60,), generator=torch.Generator().manual_seed(1))])
    a = at.to(dev())
    f = R.factor([11 + i for i in at.tolist()], D, 0.2, 5)
    used = (r.experts[a] >= 0).cpu().numpy()
    pos, wd = r.pos[a].long(), f64(w[a])
    rows = np.where(used[..., None], f64(y[pos]), 0.0)
    parts = wd[..., None] * rows
    G = R.drop(f64(dout[a]), f)
    check(out[a], R.drop(parts.sum(1), f) + f64(res[a]), DT[dtype],
          extra=U * ((k + 3) * np.abs(parts).sum(1) * f + 2 * np.abs(f64(res[a]))))
    check(dx[a], rows.sum(1), DT[dtype], extra=U * k * np.abs(rows).sum(1))
    want = np.where(used[..., None], wd[..., None] * G[:, None], 0.0)
    check(dy[pos], want, DT[dtype], extra=3 * U * np.abs(want))
    check(dw[a], (G[:, None] * rows).sum(2), torch.float32, extra=U * (D + 4) * (np.abs(G)[:, None] * np.abs(rows)).sum(2))
    assert np.array_equal(f64(xs[pos]), np.where(used[..., None], f64(x[a])[:, None], 0.0))


@pytest.mark.parametrize("T,D", [(5, 0), (0, 0), (0, 7)])
def test_rows_without_values_and_no_rows(T, D):
    r = ops.route(rnd(1, T, 4), 2)
    w = r.weights.detach().requires_grad_()
    r = r._replace(weights=w)
    x, y, res = (torch.zeros(n, D, device=dev(), requires_grad=True) for n in (T, 2 * T, T))
    xs, out = ops.dispatch(x, r), ops.combine(y, r, residual=res, p=0.5, key=1, rows=torch.arange(T, device=dev()))
    assert xs.shape == (2 * T, D) and out.shape == (T, D)
    dx, dy, dw, dres = torch.autograd.grad((xs, out), (x, y, w, res), (torch.zeros_like(xs), torch.zeros_like(out)))
    assert dx.shape == x.shape and dy.shape == y.shape and dres.shape == res.shape and (dw == 0).all() and dw.shape == (T, 2)
    assert ops.dropout(x, 0.5, 1, rows=torch.arange(T, device=dev())).shape == (T, D)


def test_values_whose_sign_torch_still_holds():
    # contiguous views with the sign as a bit, in the place of every tensor of values
    T, E, k, D = 9, 6, 2, 24

    def neg(seed, *shape):
        v = torch._neg_view(rnd(seed, *shape))
        assert v.is_neg()
        return v, v.clone()

    l, b, x, y, res, w = (neg(i, *s) for i, s in enumerate([(T, E), (E,), (T, D), (T * k, D), (T, D), (T, k)]))
    r = ops.route(rnd(9, T, E), k)
    dw, dout = neg(10, T, k), neg(11, T, D)
    dxs = neg(12, T * k, D)

    def passes(i):
        ll, xx, yy, ww = (t[i].detach().requires_grad_() for t in (l, x, y, w))
        q = ops.route(ll, k, bias=b[i], score="sigmoid", renormalise=False)
        xs = ops.dispatch(xx, r)
        out = ops.combine(yy, r._replace(weights=ww), residual=res[i], p=0.3, key=2)
        full = ops.route(ll, k, renormalise=False)
        return tuple(q) + (xs, out) + torch.autograd.grad((q.weights, full.weights, xs, out), (ll, xx, yy, ww),
                                                          (dw[i], dw[i], dxs[i], dout[i]))

    for a, c in zip(passes(0), passes(1)):
        assert torch.equal(a, c)


def test_recorders_of_torch_operations_are_refused():
    from torch.fx.experimental.proxy_tensor import make_fx
    l, x = rnd(1, 6, 8).requires_grad_(), rnd(2, 6, 16).requires_grad_()
    r = ops.route(l, 2)
    plan = r._replace(weights=r.weights.detach())       # (torch refuses a closure over what has a gradient itself)
    y = rnd(3, 12, 16)
    calls = [(lambda v: ops.route(v, 2).weights, l.detach()), (lambda v: ops.dispatch(v, plan), x.detach()),
             (lambda v: ops.combine(v, plan), y)]
    xs = ops.dispatch(x, r)
    for f, v in calls:
        with pytest.raises(RuntimeError, match="cannot be traced"):
            make_fx(f)(v)
        with pytest.raises(RuntimeError, match="cannot be traced"):
            torch.jit.trace(f, v, check_trace=False)
    for out, leaf in ((r.weights, l), (xs, x), (ops.combine(y, r), l)):
        with pytest.raises(RuntimeError, match="cannot be traced"):
            make_fx(lambda g: torch.autograd.grad(out, leaf, g, retain_graph=True))(torch.ones_like(out))
    assert torch.equal(ops.dispatch(x, r), xs)


# ---- together ------------------------------------------------------------------------------------
def layer(x, router, w1, p, key, rows, k=2):
    """A layer of experts: route, dispatch, each expert's product, combine."""
    r = ops.route(x @ router, k)
    xs = ops.dispatch(x, r)
    at = r.offsets.tolist()
    ys = torch.cat([xs[a:b] @ w for a, b, w in zip(at, at[1:], w1)] + [xs[at[-1]:]])
    return ops.combine(ys, r, residual=x, p=p, key=key, rows=rows), r


def test_sampler_batches_through_a_layer_of_experts():
    from partiallyshuffledistributedsampler_amd.DistributedSamplerViaLocallyShuffleV2 import \
        DistributedSamplerViaLocallyShuffle as V2

    class Files:
        files = ["f%d" % i for i in range(9)]

        def reset(self):
            pass

    lens = dict(zip(Files.files, range(20, 110, 10)))
    total = sum(lens.values())
    s = V2(Files(), None, num_replicas=2, rank=1, shuffle_buffer=32, total_size=total, batch_size=50, files_len=lens,
           seed=3, device=0)
    s.set_epoch(4)
    iter(s)
    D, E = 24, 5
    data = rnd(1, total, D)
    base = torch.tensor(np.concatenate([[0], np.cumsum(list(lens.values()))[:-1]]), device=dev())
    router, w1 = rnd(2, D, E).requires_grad_(), rnd(3, E, D, D, scale=0.2).requires_grad_()
    key0, key1, lo = s.dropout_key(), s.dropout_key(site=1), 0
    seen = 0
    for rows, fpos, off in s.device_batches(data, base, p=0.1):
        n = rows.shape[0]
        out, r = layer(rows, router, w1, 0.25, key1, lo)
        dout = rnd(lo, n, D)
        g_router, g_w1 = torch.autograd.grad(out, (router, w1), dout)
        # the same in 64 bits on the CPU, with the kernels' choice of experts
        order = torch.from_numpy(s._engine.file_order().astype(np.int64))
        picked = data.cpu().double()[base.cpu()[order[fpos.cpu().long()]] + off.cpu().long()]
        x = picked * torch.from_numpy(R.factor(range(lo, lo + n), D, 0.1, key0))
        x = x.float().double()                            # the batch is stored in 32 bits
        ro, ww = router.detach().cpu().double().requires_grad_(), w1.detach().cpu().double().requires_grad_()
        e = r.experts.cpu().long()
        w = torch.softmax(torch.gather(x @ ro, 1, e), 1)
        y = torch.einsum("td,tkde->tke", x, ww[e])
        f = torch.from_numpy(R.factor(range(lo, lo + n), D, 0.25, key1))
        want = x + (w.unsqueeze(2) * y).sum(1) * f
        want_router, want_w1 = torch.autograd.grad(want, (ro, ww), dout.cpu().double())
        # 32-bit products of D = 24 terms, logits of size ~6, sums over 50 rows: below 1e-4 of the norm
        for a, b in ((out, want), (g_router, want_router), (g_w1, want_w1)):
            a = a.detach().cpu().double()
            assert (a - b.detach()).norm() <= 1e-4 * b.detach().norm()
        lo += n
        seen += 1
    assert seen == -(-s.num_samples // 50)


def test_captured_passes_replay_with_other_inputs():
    T, E, k, D = 300, 16, 4, 264
    l, x, ys = rnd(1, T, E).requires_grad_(), rnd(2, T, D, dtype="bf16").requires_grad_(), \
        rnd(3, T * k, D, dtype="bf16").requires_grad_()
    dout, dxs, first = rnd(4, T, D, dtype="bf16"), rnd(5, T * k, D, dtype="bf16"), torch.zeros(1, dtype=torch.int64, device=dev())

    def passes():
        r = ops.route(l, k, score="sigmoid")
        xs = ops.dispatch(ops.dropout(x, 0.1, 9, rows=first), r)
        out = ops.combine(ys, r, residual=x, p=0.3, key=8, rows=first)
        # (no autograd graph of the leaves outlives a pass)
        return (r.experts, r.pos, xs.detach(), out.detach()) + torch.autograd.grad((xs, out), (l, x, ys), (dxs, dout))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        passes()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = passes()
    for i in range(5):
        with torch.no_grad():
            l.copy_(rnd(10 + i, T, E))
            x.copy_(rnd(20 + i, T, D, dtype="bf16"))
            first.fill_(1000 * i)
        graph.replay()
        torch.cuda.synchronize()
        want = passes()
        for a, b in zip(got, want):
            assert torch.equal(a, b), i
        torch.cuda.synchronize()


def test_two_streams_at_once():
    T, E, k, D = 4000, 32, 4, 512
    inputs = [(rnd(i, T, E), rnd(i + 10, T, D, dtype="bf16")) for i in range(4)]

    def passes(l, x, i):
        r = ops.route(l, k)
        return ops.combine(ops.dispatch(x, r), r, residual=x, p=0.2, key=i), r.src

    want = [passes(l, x, i) for i, (l, x) in enumerate(inputs)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = []
    for i, (l, x) in enumerate(inputs * 3):
        with torch.cuda.stream(streams[i % 2]):
            got.append(passes(l, x, i % 4))
    torch.cuda.synchronize()
    for i, (a, b) in enumerate(got):
        assert torch.equal(a, want[i % 4][0]) and torch.equal(b, want[i % 4][1]), i


def test_two_graphs_replayed_at_once():
    T, E, k, D = 1000, 24, 3, 128
    graphs, want = [], []
    inputs = [(rnd(i, T, E), rnd(i + 10, T, D)) for i in range(2)]      # (alive as long as the graphs)
    for i, (l, x) in enumerate(inputs):

        def passes():
            r = ops.route(l, k, score="sigmoid", bias=torch.zeros(E, device=dev()))
            return ops.combine(ops.dispatch(x, r), r, residual=x, p=0.2, key=i), r.pos, r.src

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            want.append([t.clone() for t in passes()])
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = passes()
        graphs.append((g, out, side))
    for _ in range(6):
        for g, out, side in graphs:
            with torch.cuda.stream(side):
                for t in out:
                    t.zero_()
                g.replay()
        torch.cuda.synchronize()
        for (g, out, side), w in zip(graphs, want):
            for a, b in zip(out, w):
                assert torch.equal(a, b)


def test_two_threads_at_once():
    import threading
    T, E, k, D = 700, 300, 4, 96
    inputs = [(rnd(i, T, E), rnd(i + 10, T, D), rnd(i + 20, T, D)) for i in range(2)]

    def passes(i):
        l, x, dout = (t.detach().requires_grad_() for t in inputs[i])
        r = ops.route(l, k, score="sigmoid")
        out = ops.combine(ops.dispatch(ops.dropout(x, 0.1, i), r), r, residual=x, p=0.2, key=i + 5)
        return torch.autograd.grad(out, (l, x), dout)

    want = [passes(i) for i in range(2)]
    torch.cuda.synchronize()
    got, errors = [[], []], []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(20):
                    got[i].append(passes(i))
                torch.cuda.current_stream().synchronize()
        except Exception as e:      # noqa: BLE001 -- reported by the main thread
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(60)
    assert not errors and [len(g) for g in got] == [20, 20]
    torch.cuda.synchronize()
    for i in range(2):
        for a in got[i]:
            for x, y in zip(a, want[i]):
                assert torch.equal(x, y)


def test_gpu_refusals():
    l, x = rnd(1, 6, 8), rnd(2, 6, 16)
    r = ops.route(l, 2)
    y = rnd(3, 12, 16)
    with pytest.raises(TypeError, match="float32, bfloat16 or float16"):
        ops.route(l.double(), 2)
    with pytest.raises(ValueError, match=r"\[T, E\]"):
        ops.route(l[0], 2)
    with pytest.raises(ValueError, match="score"):
        ops.route(l, 2, score="tanh")
    for bias in (torch.zeros(7, device=dev()), torch.zeros(8), torch.zeros(8, device=dev(), dtype=torch.float64)):
        with pytest.raises(ValueError, match="bias"):
            ops.route(l, 2, bias=bias)
    for valid in (torch.ones(5, dtype=torch.bool, device=dev()), torch.ones(6, device=dev())):
        with pytest.raises(ValueError, match="valid"):
            ops.route(l, 2, valid=valid)
    for kw in (dict(k=0), dict(k=9), dict(k=2, groups=3), dict(k=2, groups=4, top_groups=5), dict(k=3, groups=4),
               dict(k=2, group_sum=0), dict(k=2, scale=0.0), dict(k=2, scale=float("inf")), dict(k=2, scale=1e-30)):
        with pytest.raises(RuntimeError, match="route"):
            ops.route(l, **kw)
    with pytest.raises(TypeError, match="Routing"):
        ops.dispatch(x, tuple(r))
    with pytest.raises(ValueError, match="of 6 rows, got 5"):
        ops.dispatch(x[:5], r)
    with pytest.raises(ValueError, match="12 rows, got 11"):
        ops.combine(y[:11], r)
    with pytest.raises(ValueError, match="int32"):
        ops.dispatch(x, r._replace(pos=r.pos.long()))
    with pytest.raises(ValueError, match="weights"):
        ops.combine(y, r._replace(weights=r.weights.double()))
    with pytest.raises(ValueError, match="residual"):
        ops.combine(y, r, residual=x[:, :8])
    with pytest.raises(TypeError, match="dtype and device"):
        ops.combine(y, r, residual=x.half())
    with pytest.raises(TypeError, match="device"):
        ops.dropout(x, 0.1, 0, rows=torch.zeros(1, dtype=torch.int64))
    with pytest.raises(RuntimeError, match="differentiated again"):
        xg = x.clone().requires_grad_()
        g, = torch.autograd.grad(ops.dropout(xg, 0.5, 1).square().sum(), xg, create_graph=True)
        g.sum().backward()
    assert torch.equal(ops.dispatch(x, r)[r.pos[3, 1].item()], x[3])      # the device still works
