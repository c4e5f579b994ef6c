"""The full-catalogue softmax loss and its gradients (hpfrec_amd.softmax, hpf_hip_softmax_nll / _grad): refusals on the CPU,
results on the GPU against 64-bit arithmetic, alone and followed by the AdamW step."""
import ctypes
import math
from types import SimpleNamespace

import numpy as np
import pytest
import torch

from hpfrec_amd import _lib, adamw, softmax

U = 2.0 ** -24
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
HALF = {F32: U, BF16: 2.0 ** -8, F16: 2.0 ** -11}   # half a step of each type, relative


# ---------------------------------------------------------------------------------------------
# refusals
# ---------------------------------------------------------------------------------------------
class _Recorder:
    device = torch.device("cpu")

    def __init__(self):
        self.calls = []

    def softmax_nll(self, x, ldx, items, ld_items, *rest):
        self.calls.append((ldx, ld_items))

    def softmax_nll_grad(self, x, ldx, items, ld_items, target, weight, bias, scale, n, v, k, loss, dx, ld_dx, ditems, ld_ditems, dbias):
        self.calls.append((ldx, ld_items, ld_dx, ld_ditems))


def _good(**change):
    a = dict(ops=_Recorder(), x=torch.ones(4, 5), items=torch.ones(7, 5), target=torch.zeros(4, dtype=torch.int64), bias=torch.zeros(7))
    a.update(change)
    return a


def test_row_strides_are_passed_on():
    a = _good(x=torch.ones(4, 32)[:, :5], items=torch.ones(7, 64)[:, :5])
    softmax.softmax_nll(**a)
    softmax.softmax_nll_grad(**a, dx=torch.ones(4, 8)[:, :5])
    assert a["ops"].calls == [(32, 64), (32, 64, 8, 5)]
    a = _good(x=torch.ones(1, 32)[:, :5], target=torch.zeros(1, dtype=torch.int64))
    softmax.softmax_nll(**a)
    empty = _good(x=torch.ones(0, 5), target=torch.zeros(0, dtype=torch.int64))
    loss, lse = softmax.softmax_nll(**empty)
    assert loss.shape == lse.shape == (0,) and empty["ops"].calls == []


_REFUSED = [
    (dict(x=torch.ones(5)), "x must be a matrix"),
    (dict(x=torch.ones(4, 5, dtype=torch.float64)), "x must be of"),
    (dict(items=torch.ones(7, 5, dtype=BF16)), "items must be of"),
    (dict(items=torch.ones(7, 6)), "items has shape"),
    (dict(items=torch.ones(0, 5), bias=None), "items is empty"),
    (dict(x=torch.ones(4, 0), items=torch.ones(7, 0)), "items is empty"),
    (dict(x=torch.ones(5, 4).t()), "contiguous rows"),
    (dict(x=torch.ones(1, 5).expand(4, 5)), "overlap"),
    (dict(x=torch.ones(4, 2 ** 20), items=torch.ones(1, 2 ** 20), bias=None), "2\\^20"),
    (dict(target=torch.zeros(4, dtype=torch.int32)), "target"),
    (dict(target=torch.zeros(3, dtype=torch.int64)), "target"),
    (dict(target=torch.zeros(8, dtype=torch.int64)[::2]), "target"),
    (dict(bias=torch.zeros(6)), "bias"),
    (dict(bias=torch.zeros(7, dtype=torch.float64)), "bias"),
    (dict(scale=float("nan")), "scale"),
    (dict(scale=float("inf")), "scale"),
    (dict(ops=SimpleNamespace(device=torch.device("cuda:0"))), "expected cuda"),
]


@pytest.mark.parametrize("call", [softmax.softmax_nll, softmax.softmax_nll_grad])
@pytest.mark.parametrize("change, words", _REFUSED)
def test_refusals(call, change, words):
    with pytest.raises(ValueError, match=words):
        call(**_good(**change))


@pytest.mark.parametrize("change, words", [
    (dict(weight=torch.ones(5)), "weight"),
    (dict(weight=torch.ones(4, dtype=torch.int64)), "weight"),
    (dict(dx=torch.ones(4, 6)), "dx has shape"),
    (dict(dx=torch.ones(4, 5, dtype=BF16)), "dx must be of"),
    (dict(ditems=torch.ones(5, 7).t()), "ditems must have contiguous rows"),
    (dict(dbias=torch.ones(6)), "dbias"),
    (dict(bias=None, dbias=torch.ones(7)), "dbias without a bias"),
])
def test_refusals_of_the_gradients(change, words):
    with pytest.raises(ValueError, match=words):
        softmax.softmax_nll_grad(**_good(**change))


def test_outputs_that_overlap_are_refused():
    a = _good()
    for name, t in (("dx", a["x"]), ("ditems", a["items"]), ("dbias", a["bias"])):
        with pytest.raises(ValueError, match="overlaps"):
            softmax.softmax_nll_grad(**a, **{name: t})
    both = torch.ones(11, 5)
    with pytest.raises(ValueError, match="overlaps"):
        softmax.softmax_nll_grad(**a, dx=both[:4], ditems=both[3:10])
    softmax.softmax_nll_grad(**a, dx=both[:4], ditems=both[4:])


def test_c_entries_refuse_before_touching_the_gpu():
    L = ctypes.CDLL(_lib.build())
    vp, i64, ci, cf = ctypes.c_void_p, ctypes.c_int64, ctypes.c_int, ctypes.c_float
    L.hpf_hip_softmax_workspace.argtypes, L.hpf_hip_softmax_workspace.restype = [i64, i64, i64, ci, ci, ci], i64
    L.hpf_hip_softmax_nll.argtypes = [vp, i64, vp, i64, vp, vp, cf, i64, i64, i64, ci, vp, vp, vp, i64, ci, vp]
    L.hpf_hip_softmax_nll_grad.argtypes = [vp, i64, vp, i64, vp, vp, vp, cf, i64, i64, i64, ci, vp, vp, i64, vp, i64, vp, vp, i64, ci, vp]
    EINVAL, EUNSUPPORTED = -1, -2
    size = L.hpf_hip_softmax_workspace
    assert size(-1, 5, 5, 0, 0, 256) == EINVAL and size(5, 0, 5, 0, 0, 256) == EINVAL and size(5, 5, 0, 0, 0, 256) == EINVAL
    assert size(2 ** 30, 5, 5, 0, 0, 256) == EINVAL and size(5, 5, 5, 0, 0, 0) == EINVAL
    assert size(5, 5, 5, 3, 0, 256) == EUNSUPPORTED
    assert size(0, 5, 5, 0, 1, 256) == 0 and size(0, 5, 500, 1, 0, 256) == 0
    for k in (1, 50, 256, 257, 5000):
        for kind in (0, 1, 2):
            assert 0 < size(100, 1000, k, kind, 0, 256) < size(100, 1000, k, kind, 1, 256)
    buf = ctypes.create_string_buffer(1024)
    p = (ctypes.addressof(buf) + 255) // 256 * 256

    def nll(x=p, ldx=5, w=p, ldw=5, t=p, n=4, v=7, k=5, kind=0, loss=p, ws=p, wsize=1 << 40, cus=256):
        return L.hpf_hip_softmax_nll(x, ldx, w, ldw, t, None, 1.0, n, v, k, kind, loss, None, ws, wsize, cus, None)

    def grad(x=p, ldx=5, w=p, ldw=5, t=p, bias=None, n=4, v=7, k=5, kind=0, loss=p, dx=p, lddx=5, dw=p, lddw=5, db=None, ws=p, wsize=1 << 40):
        return L.hpf_hip_softmax_nll_grad(x, ldx, w, ldw, t, None, bias, 1.0, n, v, k, kind, loss, dx, lddx, dw, lddw, db, ws, wsize, 256, None)

    for call in (nll, grad):
        for bad in (dict(x=None), dict(w=None), dict(t=None), dict(loss=None), dict(ws=None), dict(ws=p + 16), dict(ldx=4), dict(ldw=4),
                    dict(n=-1), dict(v=0), dict(k=0), dict(wsize=1000)):
            assert call(**bad) == EINVAL, bad
        assert call(kind=3) == EUNSUPPORTED
    assert nll(n=0) == 0 and nll(cus=0) == EINVAL
    for bad in (dict(dx=None), dict(dw=None), dict(lddx=4), dict(lddw=4), dict(bias=p), dict(db=p)):
        assert grad(**bad) == EINVAL, bad


# ---------------------------------------------------------------------------------------------
# in 64 bits, and how far 32-bit (and 16-bit) arithmetic may be from it
# ---------------------------------------------------------------------------------------------
def _exact(x, items, target, weight, bias, scale):
    x, w = x.double(), items.double()
    z = scale * (x @ w.t())
    if bias is not None:
        z = z + bias.double()
    lse = torch.logsumexp(z, dim=1)
    live = target >= 0
    zt = z.gather(1, target.clamp(min=0)[:, None])[:, 0]
    loss = torch.where(live, lse - zt, torch.zeros_like(lse))
    p = torch.exp(z - lse[:, None])
    g = p.clone()
    g.scatter_(1, target.clamp(min=0)[:, None], -(p.scatter(1, target.clamp(min=0)[:, None], 0.0).sum(dim=1))[:, None])
    g = g * (torch.where(live, weight.double() if weight is not None else torch.ones_like(lse), torch.zeros_like(lse)))[:, None]
    return dict(z=z, lse=lse, loss=loss, g=g, dx=scale * (g @ w), ditems=scale * (g.t() @ x), dbias=g.sum(dim=0), x=x, w=w)


def _bounds(e, kind, bias, scale, k, wmax=1.0):
    """A logit: up to (6 products x) 2 ceil(k / 32) matrix instructions, each rounding its running sum (by a whole unit at most);
    what products of parts leave out (each part to 2^-23, low times low 2^-22: 8 U), and 2^-40 of the largest |x| |w|, k times;
    the conversion to base 2 (constant, product, sum: 4 U of the size).
    A share exp(z - lse): twice that error, 2 U of |z - lse| + |lse| for the argument's rounding, 2 U for the function.
    Sums of V shares (or V, N products): independent roundings, 4 sqrt(count) U; joining pieces a few U more; parts 8 U.
    16-bit types: shares are rounded to the type once more, results too.  Shares in half precision (float32's parts too) end at
    2^-39 of the row's, the item's or (rows over 256 wide) the weights' largest, 32-bit matrices at 2^-40 of their column's."""
    steps = (6 if kind == F32 else 1) * 2 * max(1, math.ceil(k / 32)) + 4 + (4 if kind == F32 else 0)
    ax, aw = e["x"].abs(), e["w"].abs()
    size = abs(scale) * (ax @ aw.t())
    b = torch.where(bias > -1e30, bias, torch.zeros_like(bias)).double().abs() if bias is not None else torch.zeros(e["w"].shape[0], dtype=torch.float64, device=e["x"].device)
    ez = (2 * U * steps * size + 4 * U * (size + b)).amax(dim=1)                     # per row
    if kind == F32:
        ez = ez + abs(scale) * k * 2.0 ** -39 * float(ax.max()) * float(aw.max())
    n, v = e["z"].shape
    span = torch.where(e["z"] > -1e30, (e["z"] - e["lse"][:, None]).abs(), torch.zeros_like(e["z"]))
    share = e["g"].abs()
    total = ez + (16 + 4 * math.sqrt(v)) * U + 2 * U * (torch.exp(-span) * span).sum(dim=1)
    lse = total + 4 * U * e["lse"].abs()
    rel = (2 * ez + total + 8 * U * (1 + e["lse"].abs()))[:, None] + 4 * U * span   # of a share, per logit
    coarse = 8 * U if kind == F32 else HALF[kind]
    by_row, by_item = (wmax, wmax) if k > 256 else (share.amax(dim=1, keepdim=True), share.amax(dim=0, keepdim=True))
    least_row, least_item = (0.0, 0.0) if kind == BF16 else (2.0 ** -38 * by_row, 2.0 ** -38 * by_item)
    long_v, long_n = (32 + 4 * math.sqrt(v)) * U, (32 + 4 * math.sqrt(n)) * U
    end = 2.0 ** -39 if kind == F32 else 0.0
    dx = abs(scale) * ((share * (rel + coarse + long_v) + least_row) @ aw + end * share.sum(dim=1, keepdim=True) * aw.amax(dim=0)) + HALF[kind] * e["dx"].abs()
    dw = abs(scale) * ((share * (rel + coarse + long_n) + least_item).t() @ ax + end * share.sum(dim=0)[:, None] * ax.amax(dim=0)) + HALF[kind] * e["ditems"].abs()
    if kind == F16:   # subnormal results
        dx, dw = dx + 2.0 ** -25, dw + 2.0 ** -25
    db = (share * (rel + long_n)).sum(dim=0) + 4 * U * e["dbias"].abs()
    return dict(lse=lse, loss=lse + ez + 4 * U * e["loss"].abs(), dx=dx, ditems=dw, dbias=db)


def _close(got, e, bounds, names, rows=None):
    for name, x in zip(names, got):
        if x is None:
            continue
        off = (x.double() - e[name]).abs() - bounds[name]
        assert bool((off <= 0).all()), (name, float(off.max()), float((off > 0).double().mean()))


# ---------------------------------------------------------------------------------------------
# on the GPU
# ---------------------------------------------------------------------------------------------
@pytest.fixture(scope="module")
def ops():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    from hpfrec_amd.ops_hip import HipOps
    return HipOps("cuda:0")


def _case(n, v, k, kind, bias=True, seed=0, spread=2.0, pad=0):
    gen = torch.Generator(device="cuda:0").manual_seed(seed)
    normal = lambda *s: torch.randn(s, device="cuda:0", generator=gen)  # noqa: E731
    s = (spread / math.sqrt(k)) ** 0.5
    x = torch.full((n, k + pad), 9.0, device="cuda:0").to(kind)[:, :k]
    w = torch.full((v, k + pad), 9.0, device="cuda:0").to(kind)[:, :k]
    x.copy_(normal(n, k) * s)
    w.copy_(normal(v, k) * s)
    target = torch.randint(0, v, (n,), device="cuda:0", generator=gen)
    if n > 4:
        target[::5] = -1
        target[1::5] = v - 1          # the same item many times
    weight = normal(n)
    if n > 4:
        weight[2::7] = 0.0
    return dict(x=x, items=w, target=target, weight=weight, bias=normal(v) if bias else None, scale=1.3)


def _both(ops, c):
    nll = softmax.softmax_nll(ops, **{k: v for k, v in c.items() if k != "weight"})
    grad = softmax.softmax_nll_grad(ops, **c)
    return nll, grad


def _check(ops, c):
    kind, k = c["x"].dtype, c["x"].shape[1]
    e = _exact(**c)
    b = _bounds(e, kind, c["bias"], c["scale"], k, 2 * float(c["weight"].abs().max()) if c["weight"] is not None else 1.0)
    nll, grad = _both(ops, c)
    _close(nll, e, b, ("loss", "lse"))
    _close(grad, e, b, ("loss", "dx", "ditems", "dbias"))


SHAPES = [(1, 1, 1), (1, 7, 3), (2, 33, 31), (31, 31, 32), (33, 1000, 50), (32, 32, 64), (65, 97, 33), (129, 4097, 100), (300, 2000, 128),
          (200, 1500, 200), (77, 640, 256), (40, 500, 257), (100, 1000, 300), (3, 3000, 520), (150, 900, 1000), (66, 400, 90), (80, 390, 160), (70, 333, 180), (50, 300, 224), (1100, 300, 40), (700, 260, 600)]


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [F32, BF16, F16])
@pytest.mark.parametrize("bias", [True, False])
@pytest.mark.parametrize("n, v, k", SHAPES)
def test_against_64_bits(ops, n, v, k, bias, kind):
    _check(ops, _case(n, v, k, kind, bias, seed=n + v + k))


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [F32, BF16])
@pytest.mark.parametrize("k", [50, 300])
@pytest.mark.parametrize("scale", [-1.7, 0.0, 1e-3])
def test_scales_strides_and_no_weights(ops, k, scale, kind):
    c = _case(70, 500, k, kind, True, seed=3, pad=13)
    _check(ops, dict(c, scale=scale))
    _check(ops, dict(c, weight=None))
    _check(ops, dict(c, weight=c["weight"] * 1e-6))
    _check(ops, dict(c, weight=torch.zeros_like(c["weight"])))


@pytest.mark.gpu
@pytest.mark.parametrize("k", [40, 300])
def test_rows_and_columns_of_far_apart_sizes(ops, k):
    """32-bit matrices: tables of very large, very small, zero and mixed magnitudes; columns from 1e-12 to 1e6 (x the other way
    round); items whose shares are 1e-9 and less; a row of zeros."""
    c = _case(90, 700, k, F32, True, seed=21)
    _check(ops, dict(c, x=c["x"] * 1e-25, items=c["items"] * 1e24))
    _check(ops, dict(c, x=c["x"] * 1e-30))
    _check(ops, dict(c, x=torch.zeros_like(c["x"])))
    size = torch.logspace(-2, 2, k, device="cuda:0")
    _check(ops, dict(c, x=c["x"] / size, items=c["items"] * size))
    rows = torch.logspace(-4, 0, 700, device="cuda:0")[torch.randperm(700, device="cuda:0", generator=torch.Generator(device="cuda:0").manual_seed(2))]
    _check(ops, dict(c, items=c["items"] * rows[:, None]))
    _check(ops, dict(c, bias=c["bias"] - 30.0 * (torch.arange(700, device="cuda:0") % 3 > 0)))   # two thirds of the items: shares of 1e-13


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [F32, BF16, F16])
@pytest.mark.parametrize("k", [20, 200, 400])
def test_many_rows_and_long_catalogues(ops, k, kind):
    """Several pieces of both sides, joined."""
    _check(ops, _case(2500, 6000, k, kind, True, seed=5))
    _check(ops, _case(40, 60000, k, kind, False, seed=6))


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [F32, BF16, F16])
@pytest.mark.parametrize("n", [1, 32, 33, 64, 65])
def test_few_rows(ops, n, kind):
    """Loss alone for a few rows: every width class of that path, catalogues that end inside its last tiles, strides and offsets
    that no wide load likes."""
    for k in (1, 2, 31, 33, 50, 64, 65, 100, 112, 113, 128, 129, 200, 209, 256):
        for v in (1, 31, 33, 63, 64, 65, 95, 96, 97, 1000, 5003)[k % 2::2]:
            c = _case(n, v, k, kind, v % 2 == 0, seed=n + k + v, pad=(0, 1, 3, 7)[k % 4])
            if v % 3 == 0:      # a table that begins one value into its storage
                flat = torch.empty(v * (k + 5) + 1, dtype=kind, device="cuda:0")
                flat[1:].view(v, k + 5)[:, :k].copy_(c["items"])
                c["items"] = flat[1:].view(v, k + 5)[:, :k]
            e = _exact(**c)
            b = _bounds(e, kind, c["bias"], c["scale"], k, 4.0)
            _close(softmax.softmax_nll(ops, **{a: x for a, x in c.items() if a != "weight"}), e, b, ("loss", "lse"))


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [F32, BF16, F16])
@pytest.mark.parametrize("n", [1, 32, 33, 64])
def test_few_wide_rows(ops, n, kind):
    """The same for rows that are taken in parts of 64 columns."""
    for k in (129, 192, 257, 320, 1000, 1025):
        for v in (1, 31, 33, 63, 64, 65, 95, 96, 97, 1000, 5003)[k % 2::2]:
            c = _case(n, v, k, kind, v % 2 == 0, seed=n + k + v, pad=(0, 1, 3, 7)[k % 4])
            if v % 3 == 0:
                flat = torch.empty(v * (k + 5) + 1, dtype=kind, device="cuda:0")
                flat[1:].view(v, k + 5)[:, :k].copy_(c["items"])
                c["items"] = flat[1:].view(v, k + 5)[:, :k]
            e = _exact(**c)
            b = _bounds(e, kind, c["bias"], c["scale"], k, 4.0)
            _close(softmax.softmax_nll(ops, **{a: x for a, x in c.items() if a != "weight"}), e, b, ("loss", "lse"))


@pytest.mark.gpu
@pytest.mark.parametrize("k", [50, 300])
@pytest.mark.parametrize("kind", [F32, BF16])
@pytest.mark.parametrize("lowest", [float("-inf"), torch.finfo(torch.float32).min])
def test_masked_items(ops, k, kind, lowest):
    c = _case(64, 300, k, kind, True, seed=8)
    out = torch.zeros(300, dtype=torch.bool, device="cuda:0")
    out[::3] = True
    out[96:160] = True                       # whole tiles
    c["bias"] = torch.where(out, lowest, c["bias"])
    c["target"] = torch.where((c["target"] >= 0) & out[c["target"].clamp(min=0)], 1, c["target"])
    c["target"][0], c["target"][3] = 0, 99   # masked targets
    (loss, lse), (gloss, dx, ditems, dbias) = _both(ops, c)
    gone = torch.zeros(64, dtype=torch.bool, device="cuda:0")
    gone[0] = gone[3] = True
    d = dict(c, bias=torch.where(out, float("-inf"), c["bias"]), target=torch.where(gone, -1, c["target"]))
    e = _exact(**d)
    b = _bounds(e, kind, d["bias"], c["scale"], k, 2 * float(c["weight"].abs().max()))
    assert bool((loss[gone] == float("inf")).all()) and bool((gloss[gone] == float("inf")).all())
    _close((torch.where(gone, 0.0, gloss),), e, b, ("loss",))
    _close((torch.where(gone, 0.0, loss), lse, dx, ditems, dbias), e, b, ("loss", "lse", "dx", "ditems", "dbias"))
    assert not bool(dx[gone].any()) and not bool(ditems[out].any()) and not bool(dbias[out].any())
    # nothing left at all
    c["bias"] = torch.full_like(c["bias"], lowest)
    (loss, lse), (gloss, dx, ditems, dbias) = _both(ops, c)
    live = c["target"] >= 0
    assert bool((lse == float("-inf")).all()) and bool((loss[live] == float("inf")).all()) and not bool(loss[~live].any())
    assert not bool(dx.any()) and not bool(ditems.any()) and not bool(dbias.any())


@pytest.mark.gpu
@pytest.mark.parametrize("k", [50, 300])
@pytest.mark.parametrize("kind", [F32, F16])
def test_nan_and_padding(ops, k, kind):
    c = _case(50, 200, k, kind, True, seed=9)
    clean = _both(ops, c)
    c["x"][0] = float("nan")                 # row 0 has no target: what it holds reaches no gradient
    assert c["target"][0] == -1
    (loss, lse), grad = _both(ops, c)
    assert float(loss[0]) == 0.0 and math.isnan(float(lse[0])) and torch.equal(lse[1:], clean[0][1][1:])
    for x, y in zip(grad, clean[1]):
        assert torch.equal(x, y)
    c["target"][7] = 200                     # no such item
    c["x"][7] = float("inf")
    loss, dx, ditems, dbias = softmax.softmax_nll_grad(ops, **c)
    d = dict(c, target=c["target"].clone(), x=c["x"].clone())
    d["target"][7], d["x"][7] = -1, 0.0
    want = softmax.softmax_nll_grad(ops, **d)
    assert math.isnan(float(loss[7])) and torch.equal(dx, want[1]) and torch.equal(ditems, want[2]) and torch.equal(dbias, want[3])
    c["x"][8, k - 1] = float("nan")          # a live row: its loss and dx, and every item
    loss, dx, ditems, dbias = softmax.softmax_nll_grad(ops, **c)
    assert math.isnan(float(loss[8])) and bool(torch.isnan(dx[8]).all()) and bool(torch.isfinite(dx[9]).all()) and bool(torch.isnan(ditems).any(dim=1).all())
    c["x"][8] = 0.0
    c["items"][5, 0] = float("nan")          # an item: every live row, whether it is the target or not
    c["target"][9] = 5
    loss, dx, _, _ = softmax.softmax_nll_grad(ops, **c)
    live = (c["target"] >= 0)
    assert bool(torch.isnan(loss[live]).all())
    loss, lse = softmax.softmax_nll(ops, **{a: b for a, b in c.items() if a != "weight"})
    assert bool(torch.isnan(loss[live]).all()) and bool(torch.isnan(lse[1:]).all())


@pytest.mark.gpu
@pytest.mark.parametrize("n", [40, 90])
@pytest.mark.parametrize("k", [50, 300])
@pytest.mark.parametrize("kind", [F32, BF16, F16])
def test_what_takes_no_part_may_hold_anything(ops, kind, k, n):
    """Rows and weights without a target, rows with a masked target, masked items: NaN, infinite or as large as the type goes, they
    change no bit of the rest."""
    c = _case(n, 300, k, kind, True, seed=30)
    out = torch.zeros(300, dtype=torch.bool, device="cuda:0")
    out[::7] = True
    out[64:96] = True                        # a whole tile
    c["bias"] = torch.where(out, float("-inf"), c["bias"])
    c["target"] = torch.where((c["target"] >= 0) & out[c["target"].clamp(min=0)], 2, c["target"])
    c["target"][3] = 70                      # masked
    gone = (c["target"] < 0) | (c["target"] == 70)
    big = torch.finfo(kind).max / 4
    filled = lambda value, values: dict(c, x=torch.where(gone[:, None], value, c["x"]), items=torch.where(out[:, None], value, c["items"]),  # noqa: E731
                                        weight=torch.where(gone, values, c["weight"]))
    nll, grad = _both(ops, filled(0.0, 0.0))
    assert bool((nll[0][3] == float("inf")).all()) and bool(torch.isfinite(grad[0][~gone]).all())
    for value in (big, -big, float("inf"), float("nan")):
        (loss, lse), got = _both(ops, filled(value, 1e38 if abs(value) == big else value))
        assert torch.equal(loss, nll[0]) and torch.equal(lse[~gone], nll[1][~gone])
        for a, b in zip(got, grad):
            assert torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("n, v, k", [(2200003, 3, 2), (70001, 40, 1000)])
def test_launches_of_over_65536_workgroups(ops, n, v, k):
    """Results of all rows against the same rows in a call of their own."""
    c = _case(n, v, k, F16, True, seed=31)
    loss, dx, _, dbias = softmax.softmax_nll_grad(ops, **c)
    e = _exact(**{a: b[-500:] if a in ("x", "target", "weight") else b for a, b in c.items()})
    wmax = 2 * float(c["weight"].abs().max())
    b = _bounds(e, F16, c["bias"], c["scale"], k, wmax)
    _close((loss[-500:], dx[-500:]), e, b, ("loss", "dx"))
    g = torch.zeros(v, dtype=torch.float64, device="cuda:0")
    slack = torch.zeros_like(g)
    for i in range(0, n, 200000):
        e = _exact(**{a: b[i:i + 200000] if a in ("x", "target", "weight") else b for a, b in c.items()})
        b = _bounds(e, F16, c["bias"], c["scale"], k, wmax)
        g += e["dbias"]
        slack += b["dbias"] + e["g"].abs().sum(dim=0) * 4 * math.sqrt(n) * U
        _close((loss[i:i + 200000], dx[i:i + 200000]), e, b, ("loss", "dx"))
    assert bool(((dbias.double() - g).abs() <= slack).all())


@pytest.mark.gpu
@pytest.mark.parametrize("k", [16, 272])
def test_a_row_that_is_sure_of_its_target(ops, k):
    """Loss and gradient are far below one and keep their relative accuracy: others / target, not 1 - p."""
    v = 500
    x = torch.zeros(4, k, device="cuda:0")
    items = torch.zeros(v, k, device="cuda:0")
    items[7, 0] = 1.0
    items[:, 1] = torch.linspace(-1, 1, v, device="cuda:0")
    x[:, 0] = torch.tensor([12.0, 25.0, 40.0, 60.0], device="cuda:0")
    x[:, 1] = 0.5
    target = torch.full((4,), 7, device="cuda:0")
    e = _exact(x, items, target, None, None, 1.0)
    others = torch.exp(e["z"] - e["z"][:, 7:8])[:, torch.arange(v, device="cuda:0") != 7].sum(dim=1)
    loss, dx, ditems, _ = softmax.softmax_nll_grad(ops, x, items, target)
    # a logit of 60 is rounded by U of it: 2 x 60 U of the quotient, and some more
    assert bool(((loss.double() / torch.log1p(others) - 1).abs() <= 400 * U).all())
    assert bool(((dx[:, 0].double() / (-others / (1 + others)) - 1).abs() <= 400 * U).all())
    assert bool(((ditems[7, 0].double() / e["ditems"][7, 0] - 1).abs() <= 400 * U))


@pytest.mark.gpu
@pytest.mark.parametrize("k", [24, 290])
def test_gradients_against_differences(ops, k):
    """Along random directions: losses are right to 1e-6 of about 7, so that a difference over 2 h = 0.04 is to 4e-4 of N = 60
    rows' sqrt(60) x 7e-6 / 0.04; third derivatives (of order 1) add h^2 / 6."""
    c = _case(60, 700, k, F32, True, seed=12)
    _, dx, ditems, dbias = softmax.softmax_nll_grad(ops, **c)
    total = lambda d: float((softmax.softmax_nll(ops, **{a: b for a, b in d.items() if a != "weight"})[0].double() * c["weight"].double()).sum())  # noqa: E731
    gen = torch.Generator(device="cuda:0").manual_seed(1)
    for name, g in (("x", dx), ("items", ditems), ("bias", dbias)):
        d = torch.randn(g.shape, device="cuda:0", generator=gen)
        d /= d.norm()
        h = 0.02
        got = (total(dict(c, **{name: c[name] + h * d})) - total(dict(c, **{name: c[name] - h * d}))) / (2 * h)
        want = float((g.double() * d.double()).sum())
        assert abs(got - want) <= 1.5e-3, (name, got, want)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [F32, F16])
@pytest.mark.parametrize("k", [37, 301])
def test_given_outputs(ops, k, kind):
    c = _case(45, 130, k, kind, True, seed=13)
    want = softmax.softmax_nll_grad(ops, **c)
    dx, dw = torch.full((45, k + 9), 5.0, device="cuda:0").to(kind), torch.full((130, k + 3), 5.0, device="cuda:0").to(kind)
    db = torch.empty(130, device="cuda:0")
    got = softmax.softmax_nll_grad(ops, **c, dx=dx[:, :k], ditems=dw[:, :k], dbias=db)
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    assert bool((dx[:, k:] == 5).all()) and bool((dw[:, k:] == 5).all()) and got[3] is db


@pytest.mark.gpu
def test_no_rows(ops):
    for kind in (F32, BF16):
        c = _case(1, 40, 10, kind, True)
        for name in ("x", "target", "weight"):
            c[name] = c[name][:0]
        loss, dx, ditems, dbias = softmax.softmax_nll_grad(ops, **c, ditems=torch.full((40, 12), 3.0, device="cuda:0").to(kind)[:, :10])
        assert loss.shape == (0,) and dx.shape == (0, 10) and not bool(ditems.any()) and not bool(dbias.any())


@pytest.mark.gpu
@pytest.mark.parametrize("kind, k", [(F32, 50), (BF16, 200), (F16, 300)])
def test_equal_calls_streams_and_graphs(ops, kind, k):
    """Equal bits in every call, on another stream, in two calls at once, and in each replay of a captured call with eager
    work and synchronisations between them."""
    c, d = _case(257, 3000, k, kind, True, seed=14), _case(100, 900, k, kind, False, seed=15)
    want, other = softmax.softmax_nll_grad(ops, **c), softmax.softmax_nll_grad(ops, **d)
    torch.cuda.synchronize()
    one, two = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(3):
        with torch.cuda.stream(one):
            a = softmax.softmax_nll_grad(ops, **c)
        with torch.cuda.stream(two):
            b = softmax.softmax_nll_grad(ops, **d)
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(a, want)) and all(torch.equal(x, y) for x, y in zip(b[:3], other))
    inputs = {n: t.clone() if torch.is_tensor(t) else t for n, t in c.items()}
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = softmax.softmax_nll_grad(ops, **inputs)
        nll = softmax.softmax_nll(ops, **{n: t for n, t in inputs.items() if n != "weight"})
    for r in range(3):
        inputs["x"].copy_(c["x"] * (1 + r))
        graph.replay()
        d = dict(c, x=(c["x"] * (1 + r)).contiguous())
        eager, eager_nll = softmax.softmax_nll_grad(ops, **d), softmax.softmax_nll(ops, **{n: t for n, t in d.items() if n != "weight"})
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(got + nll, eager + eager_nll))


@pytest.mark.gpu
@pytest.mark.parametrize("kind, k, bits", [(F32, 30, 32), (F32, 30, 8), (BF16, 260, 32)])
def test_loss_gradients_and_steps_together(ops, kind, k, bits):
    """Three training steps -- loss, gradients, AdamW on both tables and the biases -- against the same in 64 bits.  A step moves a
    value by about lr whatever its gradient's size, so only values whose gradient is far from zero are held: there the
    gradient's relative error is below 1e-3 (32 bits), and three steps of lr = 1e-3 drift apart by less than 3e-3 lr."""
    c = _case(90, 400, k, kind, True, seed=16)
    c["weight"] = c["weight"].abs() + 0.5
    params = [c["x"], c["items"], c["bias"]]
    st = adamw.adamw_state(params, bits)
    wide = [p.double() for p in params]
    wm, wv = [torch.zeros_like(p) for p in wide], [torch.zeros_like(p) for p in wide]
    sure = [torch.ones(p.shape, dtype=torch.bool, device="cuda:0") for p in wide]
    lr, b1, b2, eps, wd = 1e-3, 0.9, 0.999, 1e-8, 0.01
    for t in range(1, 4):
        loss, *grads = softmax.softmax_nll_grad(ops, **c)
        adamw.adamw_step(ops, params, grads, lr=lr, betas=(b1, b2), eps=eps, weight_decay=[wd, wd, 0.0], seed=3, **st)
        e = _exact(wide[0], wide[1], c["target"], c["weight"], wide[2], c["scale"])
        for i, g in enumerate((e["dx"], e["ditems"], e["dbias"])):
            wm[i], wv[i] = b1 * wm[i] + (1 - b1) * g, b2 * wv[i] + (1 - b2) * g * g
            wide[i] = wide[i] * (1 - lr * (wd if i < 2 else 0.0)) - lr * (wm[i] / (1 - b1 ** t)) / (torch.sqrt(wv[i] / (1 - b2 ** t)) + eps)
            sure[i] &= g.abs() > 0.05 * g.abs().mean()
    assert int(st["step"]) == 3 and torch.is_tensor(loss)
    if kind == F32 and bits == 32:
        for i, p in enumerate(params):
            off = (p.double() - wide[i]).abs()
            assert float(sure[i].double().mean()) > 0.5 and float(off[sure[i]].max()) <= 3e-3 * lr + 4 * U * float(wide[i].abs().max())
    else:   # 8-bit moments and 16-bit gradients: every step still moves by at most a few lr
        for i, p in enumerate(params):
            held = p if st["masters"][i] is None else st["masters"][i]
            assert float((held.double() - wide[i]).abs().max()) <= 12 * lr + (HALF[kind] * float(wide[i].abs().max()) if kind != F32 else 0.0)


@pytest.mark.gpu
def test_more_than_2_to_the_32_logits(ops):
    """70,001 rows x 70,001 items: rows and items from all over against 64 bits; and a table of over 2^31 values."""
    n = v = 70001
    c = _case(n, v, 16, BF16, True, seed=17)
    loss, dx, ditems, dbias = softmax.softmax_nll_grad(ops, **c)
    at = torch.tensor([0, 1, 4097, 35000, n - 2, n - 1], device="cuda:0")
    few = dict(c, x=c["x"][at], target=c["target"][at], weight=c["weight"][at])
    e = _exact(**few)
    b = _bounds(e, BF16, c["bias"], c["scale"], 16, 16.0)
    _close((loss[at], dx[at]), e, b, ("loss", "dx"))
    g = torch.zeros(len(at), dtype=torch.float64, device="cuda:0")
    size = torch.zeros_like(g)
    for i in range(0, n, 5000):
        e = _exact(**dict(c, x=c["x"][i:i + 5000], target=c["target"][i:i + 5000], weight=c["weight"][i:i + 5000]))
        g += e["g"][:, at].sum(dim=0)
        size += e["g"][:, at].abs().sum(dim=0)
    assert bool(((dbias[at].double() - g).abs() <= size * (64 + 4 * math.sqrt(n)) * U).all())
    del c, few, e, dx, ditems
    v = 2 ** 26 + 77
    items = torch.zeros((v, 33), dtype=BF16, device="cuda:0")
    gen = torch.Generator(device="cuda:0").manual_seed(1)
    items[-300:] = torch.randn((300, 33), device="cuda:0", generator=gen)
    x = torch.randn((2, 33), device="cuda:0", generator=gen).to(BF16)
    loss, lse = softmax.softmax_nll(ops, x, items, torch.tensor([v - 1, v - 299], device="cuda:0"))
    z = x.double() @ items[-300:].double().t()
    want = torch.log(torch.exp(z).sum(dim=1) + (v - 300))
    assert bool(((lse.double() - want).abs() <= (64 + 4 * math.sqrt(v)) * U).all())
    assert bool(((loss.double() - (want - z[[0, 1], [299, 1]])).abs() <= (64 + 4 * math.sqrt(v)) * U).all())


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [F32, BF16])
@pytest.mark.parametrize("n, v, k", [(5, 40, 5000), (70, 300, 2049), (2, 9, 40000)])
def test_very_wide_rows(ops, n, v, k, kind):
    _check(ops, _case(n, v, k, kind, True, seed=n + k))


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [F32, BF16])
def test_rows_far_apart_and_one_table_for_both(ops, kind):
    """Items 2^24 values apart, and rows that are some of the items themselves."""
    c = _case(40, 40, 50, kind, True, seed=41)
    flat = torch.empty(39 * 2 ** 24 + 50, dtype=kind, device="cuda:0")
    far = flat.as_strided((40, 50), (2 ** 24, 1))
    far.copy_(c["items"])
    _check(ops, dict(c, items=far))
    _check(ops, dict(c, items=far, x=far))
    many = _case(10, 3000, 50, kind, True, seed=42)
    many["x"] = many["items"][1000:1010]
    _check(ops, many)


@pytest.mark.gpu
@pytest.mark.parametrize("kind, n, k", [(F32, 61, 100), (BF16, 61, 100), (F16, 1, 256)])
def test_few_rows_streams_and_graphs(ops, kind, n, k):
    """Equal bits on two streams at once, and in two captured calls' replays with eager work and synchronisations between them."""
    c = {a: b for a, b in _case(n, 5000, k, kind, True, seed=43).items() if a != "weight"}
    want = softmax.softmax_nll(ops, **c)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = []
    for _ in range(4):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(softmax.softmax_nll(ops, **c))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for g in got for a, b in zip(g, want))
    inputs = {a: b.clone() if torch.is_tensor(b) else b for a, b in c.items()}
    graphs, outs = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()], []
    for g in graphs:
        with torch.cuda.graph(g):
            outs.append(softmax.softmax_nll(ops, **inputs))
    for r in range(3):
        inputs["x"].copy_(c["x"] * (1 + r))
        torch.cuda.synchronize()
        for s, g in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
        eager = softmax.softmax_nll(ops, **dict(c, x=c["x"] * (1 + r)))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for o in outs for a, b in zip(o, eager))


@pytest.mark.gpu
@pytest.mark.parametrize("v, k", [(2 ** 26 + 77, 33), (2 ** 22 + 5, 600)])
def test_gradients_of_tables_of_over_2_to_the_31_values(ops, v, k):
    """All items but the last 300 are zeros.  Shares, the matrices' products and the results are each rounded to the type (3 x 2^-8
    of a term); sums of v shares of one size keep 4 sqrt(v) U."""
    n = 70
    gen = torch.Generator(device="cuda:0").manual_seed(2)
    items = torch.zeros((v, k), dtype=BF16, device="cuda:0")
    items[-300:] = torch.randn((300, k), device="cuda:0", generator=gen) * k ** -0.25
    x = (torch.randn((n, k), device="cuda:0", generator=gen) * 3 * k ** -0.25).to(BF16)
    target = v - 1 - torch.randint(0, 300, (n,), device="cuda:0", generator=gen)
    target[0] = 5
    loss, dx, ditems, _ = softmax.softmax_nll_grad(ops, x, items, target)
    w = items[-300:].double()
    z = x.double() @ w.t()
    lse = torch.log(torch.exp(z).sum(dim=1) + (v - 300))
    zt = torch.where(target == 5, 0.0, z.gather(1, (target - (v - 300)).clamp(min=0)[:, None])[:, 0])
    assert bool(((loss.double() - (lse - zt)).abs() <= (64 + 4 * math.sqrt(v) + 40 * k ** 0.5) * U).all())
    g = torch.exp(z - lse[:, None])
    last = target != 5
    g[last, (target - (v - 300))[last]] -= 1.0
    rel = 3 * HALF[BF16] + (64 + 4 * math.sqrt(v)) * U
    assert bool(((dx.double() - g @ w).abs() <= rel * (g.abs() @ w.abs()) + 1e-30).all())
    assert bool(((ditems[-300:].double() - g.t() @ x.double()).abs() <= rel * (g.abs().t() @ x.double().abs())).all())
    other = torch.exp(-lse)
    rest = (other[:, None] * x.double())
    for i in (0, 6, v // 2, v - 301):
        assert bool(((ditems[i].double() - rest.sum(dim=0)).abs() <= rel * rest.abs().sum(dim=0)).all())
    hit = rest.sum(dim=0) - x[0].double()
    assert bool(((ditems[5].double() - hit).abs() <= rel * (rest.abs().sum(dim=0) + x[0].double().abs())).all())


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_a_batch_of_events_that_names_users_twice(ops, bits):
    """Rows gathered from a table, their gradients added up to the table's, one step of all three tensors.  AdamW's first step moves a
    value by lr g / (|g| + eps') -- lr times its gradient's sign, to 1e-4 of it where |g| > 1e4 eps (8-bit moments: the e4m3
    rounding of the next step's moments does not reach this one)."""
    c = _case(90, 400, 40, F32, True, seed=51)
    gen = torch.Generator(device="cuda:0").manual_seed(3)
    users = torch.randn((60, 40), device="cuda:0", generator=gen) * 0.2
    batch = torch.randint(0, 50, (90,), device="cuda:0", generator=gen)
    params = [users, c["items"].contiguous(), c["bias"]]
    before = [p.clone() for p in params]
    state = adamw.adamw_state(params, bits)
    call = dict(c, x=users[batch], items=params[1])
    e = _exact(**call)
    b = _bounds(e, F32, c["bias"], c["scale"], 40)
    loss, dx, ditems, dbias = softmax.softmax_nll_grad(ops, **call)
    _close((loss, dx, ditems, dbias), e, b, ("loss", "dx", "ditems", "dbias"))
    grads = [torch.zeros_like(users).index_add_(0, batch, dx), ditems, dbias]
    want = torch.zeros((60, 40), dtype=torch.float64, device="cuda:0").index_add_(0, batch, e["dx"])
    slack = torch.zeros_like(want).index_add_(0, batch, b["dx"] + 90 * U * e["dx"].abs())
    assert bool(((grads[0].double() - want).abs() <= slack).all())
    adamw.adamw_step(ops, params, grads, lr=1e-2, eps=1e-10, weight_decay=0.0, **state)
    for p, q, g in zip(params, before, grads):
        far = g.abs() > 1e-6
        assert bool(((p - (q - 1e-2 * torch.sign(g)))[far].abs() <= 2e-6 + 4 * U * q[far].abs()).all())
        assert bool((p == q)[g == 0].all())


# finite biases far from zero, above what masks
FAR = (-1e4, -3e7, -5e7, -1e8, -1.5e8, -1e9, -1e20, -5e37)


def _with_far_items(k, kind, weights, seed=61):
    """A third of the items have biases far below the others'; every fifth row's target is one of them, and most are no row's target.
    Returns the case, which items, and in 64 bits what it has to give: shares of exp(-800) are zero there as those of exp(-1e4) are."""
    c = _case(200, 300, k, kind, True, seed=seed)
    far = torch.arange(300, device="cuda:0") % 3 == 0
    c["bias"] = torch.where(far, torch.tensor(FAR, device="cuda:0").repeat(100)[:300], c["bias"])
    c["target"] = torch.where((c["target"] >= 0) & far[c["target"].clamp(min=0)], c["target"] + 1, c["target"])
    c["target"][2::5] = 3 * (torch.arange(40, device="cuda:0") % 25)
    gen = torch.Generator(device="cuda:0").manual_seed(7)
    if weights == "spread":       # of both signs, from 2^-14 to 1
        c["weight"] = torch.exp2(-14 * torch.rand(200, device="cuda:0", generator=gen)) * torch.sign(c["weight"])
    else:
        c["weight"] = torch.ones(200, device="cuda:0")
    e = _exact(**dict(c, bias=torch.where(far, -800.0, c["bias"])))
    # bounds as if the far items' logits were no further away than their row's lse: a share of zero and a target's of one owe nothing to
    # the size of such a bias
    e["z"] = torch.where(far, e["lse"][:, None], e["z"])
    return c, far, e, _bounds(e, kind, torch.where(far, 0.0, c["bias"]), c["scale"], k, 2 * float(c["weight"].abs().max()))


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [F32, BF16, F16])
@pytest.mark.parametrize("k", [50, 200, 300])
@pytest.mark.parametrize("weights", ["ones", "spread"])
def test_targets_with_large_biases(ops, weights, k, kind):
    """A target's share is its row's weight less nothing, however far below the others its item is."""
    c, far, e, b = _with_far_items(k, kind, weights)
    loss, dx, ditems, dbias = softmax.softmax_nll_grad(ops, **c)
    near = (c["target"] < 0) | ~far[c["target"].clamp(min=0)]
    _close((torch.where(near, loss, 0.0), dx), dict(e, loss=torch.where(near, e["loss"], 0.0)), b, ("loss", "dx"))
    t = c["target"][~near]
    z = c["scale"] * (c["x"][~near].double() * c["items"][t].double()).sum(dim=1) + c["bias"][t].double()
    assert bool(((loss[~near].double() / (e["lse"][~near] - z) - 1).abs() <= 8 * U).all())
    hit = torch.zeros(300, dtype=torch.bool, device="cuda:0")
    hit[c["target"][c["target"] >= 0]] = True
    for name, got in (("ditems", ditems), ("dbias", dbias)):
        off = (got.double() - e[name]).abs() - b[name]
        assert bool((off[hit | ~far] <= 0).all()), (name, float(off[hit | ~far].max()))


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [F32, BF16, F16])
@pytest.mark.parametrize("k", [50, 200, 300])
def test_items_far_below_the_others(ops, k, kind):
    """An item that is nobody's target and whose shares are zero in 32 bits gets gradients of zero."""
    c, far, e, b = _with_far_items(k, kind, "spread")
    _, _, ditems, dbias = softmax.softmax_nll_grad(ops, **c)
    far[c["target"][c["target"] >= 0]] = False
    assert int(far.sum()) >= 70 and not bool(ditems[far].any()) and not bool(dbias[far].any())
    # rows none of which has weight to speak of but for these items
    c["weight"] = torch.where(c["weight"].abs() > 0.5, c["weight"], 0.0)
    for x in softmax.softmax_nll_grad(ops, **c)[1:]:
        assert bool(torch.isfinite(x).all())


AWAY = (-2e7, 2e7, -3e7, 5e7, -1e8, 1e8, -1.5e8, 1e9, -1e9, 1e12, -1e30, 1e37)


def _away(n, k, kind, away):
    """Logits that are `away` and a little, which 32 bits round to `away`: every item's share is 1 / v."""
    c = _case(n, 300, k, kind, True, seed=71, spread=1e-3)
    c["bias"] = torch.full((300,), away, device="cuda:0")
    p = torch.full((n, 300), 1 / 300, dtype=torch.float64, device="cuda:0")
    live = c["target"] >= 0
    g = (p - torch.nn.functional.one_hot(c["target"].clamp(min=0), 300)) * (torch.where(live, c["weight"].double(), 0.0))[:, None]
    x, w = c["x"].double(), c["items"].double()
    flat = torch.full((n,), math.log(300.0), dtype=torch.float64, device="cuda:0")
    e = dict(z=torch.zeros_like(g), lse=flat, loss=torch.where(live, flat, 0.0), g=g, dx=c["scale"] * (g @ w), ditems=c["scale"] * (g.t() @ x), dbias=g.sum(dim=0), x=x, w=w)
    return c, e, _bounds(e, kind, None, c["scale"], k, 2 * float(c["weight"].abs().max()))


def _check_away(ops, n, k, kind):
    for away in AWAY:
        c, e, b = _away(n, k, kind, away)
        (loss, lse), grad = _both(ops, c)
        _close((loss,), e, b, ("loss",))
        _close(grad[:2], e, b, ("loss", "dx"))
        assert bool(((lse.double() - away).abs() <= math.log(300.0) + 8 * U * abs(away)).all()), away


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [F32, BF16, F16])
@pytest.mark.parametrize("k", [50, 200])
@pytest.mark.parametrize("n", [40, 150])
def test_rows_whose_logits_are_all_far_from_zero(ops, n, k, kind):
    """Loss and dx know only differences; lse is off by a few units of its own last place."""
    _check_away(ops, n, k, kind)


def _check_products(ops, n, k, kind):
    """One column whose product is far from zero, no bias.  All items are alike, so that logits that are rounded alike differ by nothing;
    half precision's stay where floats are closer than one, and are rounded apart by up to a step each."""
    big = 2.0 ** 7 if kind == F16 else 2.0 ** 14
    step = 4 * U * big * big / 3 if kind == F16 else 0.0
    x, items = torch.zeros((n, k), device="cuda:0", dtype=kind), torch.zeros((290, k), device="cuda:0", dtype=kind)
    x[:, 0], items[:, 0] = big, -big
    x[::2, 0] *= -1
    target = torch.arange(n, device="cuda:0") % 290
    loss, dx, ditems, _ = softmax.softmax_nll_grad(ops, x, items, target, scale=1.0 / 3)
    want = math.log(290.0)
    assert bool(((loss.double() - want).abs() <= 64 * U * want + step).all())
    assert bool(torch.isfinite(dx).all()) and bool(torch.isfinite(ditems).all())
    # all shares are 1 / 290 and the items alike: what is left of dx is rounding
    assert bool((dx[:, 0].double().abs() <= big / 3 * (2 * HALF[kind] + 290 * U + step)).all())


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [F32, BF16, F16])
@pytest.mark.parametrize("n", [40, 150])
def test_rows_far_from_zero_by_their_products(ops, n, kind):
    _check_products(ops, n, 50, kind)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [F32, BF16, F16])
@pytest.mark.parametrize("n", [40, 150])
def test_wide_rows_far_from_zero(ops, n, kind):
    """Rows over 256 wide, whose dx comes from the shares that the items' gradients come from."""
    _check_away(ops, n, 300, kind)
    _check_products(ops, n, 300, kind)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [F32, BF16, F16])
@pytest.mark.parametrize("k", [50, 200, 300])
def test_items_of_rows_far_from_zero(ops, k, kind):
    """The items' gradients too know only differences of logits, and the rows' weights."""
    for away in AWAY + (300.0, -5000.0):
        c, e, b = _away(150, k, kind, away)
        if abs(away) < 1e6:      # (there logits keep their own differences: up to a 32-bit step of `away`, twice)
            b = {name: x + 8 * U * abs(away) * (e["g"].abs().sum(dim=0)[:, None] * 0.1 if name == "ditems" else e["g"].abs().sum(dim=0)) if name in ("ditems", "dbias") else x for name, x in b.items()}
            e = _exact(**c)
        _, _, ditems, dbias = softmax.softmax_nll_grad(ops, **c)
        _close((ditems, dbias), e, b, ("ditems", "dbias"))


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [F32, BF16, F16])
@pytest.mark.parametrize("k", [50, 300])
def test_an_item_far_above_the_others(ops, k, kind):
    """It has every row's share, with its row's weight: what it gets is the sum of the others' weights, to their rounding.  (A logit of z
    is rounded to U z, in both passes by itself; from 1e8 on the products are lost in it, and it is the bias in both.)"""
    for above in (200.0, 5e3, 1e6, 1e8, 1e9, 1e20):
        c = _case(150, 300, k, kind, True, seed=72)
        c["bias"][17] = above
        c["target"][2::5] = 17
        c["weight"] = torch.exp2(torch.round(c["weight"] * 3))
        loss, dx, ditems, dbias = softmax.softmax_nll_grad(ops, **c)
        w = torch.where((c["target"] >= 0) & (c["target"] != 17), c["weight"].double(), 0.0)
        assert bool((loss[c["target"] == 17] == 0).all()) and bool(torch.isfinite(dx).all()) and bool(torch.isfinite(ditems).all())
        step = 4 * U * above if above < 1e7 else 0.0
        assert abs(float(dbias[17]) / float(w.sum()) - 1) <= 64 * U + step, above
        want = c["scale"] * (w @ c["x"].double())
        slack = abs(c["scale"]) * (w @ c["x"].double().abs()) * (64 * U + step + 2 * HALF[kind])
        assert bool(((ditems[17].double() - want).abs() <= slack).all()), above


@pytest.mark.skipif(torch.cuda.is_available(), reason="shows, without a GPU, that nothing is refused ahead of the first launch")
@pytest.mark.parametrize("n, v, k, kind", [(4, 1000, 50, 0), (64, 500, 100, 0), (64, 40, 300, 0), (4, 300, 200, 1), (64, 3000, 300, 2)])
def test_a_workspace_of_the_size_asked_for_is_enough_for_every_stride(n, v, k, kind):
    L = ctypes.CDLL(_lib.build())
    vp, i64, ci, cf = ctypes.c_void_p, ctypes.c_int64, ctypes.c_int, ctypes.c_float
    L.hpf_hip_softmax_workspace.argtypes, L.hpf_hip_softmax_workspace.restype = [i64, i64, i64, ci, ci, ci], i64
    L.hpf_hip_softmax_nll.argtypes = [vp, i64, vp, i64, vp, vp, cf, i64, i64, i64, ci, vp, vp, vp, i64, ci, vp]
    buf = ctypes.create_string_buffer(1024)
    p = (ctypes.addressof(buf) + 255) // 256 * 256
    size = L.hpf_hip_softmax_workspace(n, v, k, kind, 0, 256)
    for ld in (k, 2 ** 24 - 1, 2 ** 24, 2 ** 33):
        rc = L.hpf_hip_softmax_nll(p, k, p, ld, p, None, 1.0, n, v, k, kind, p, None, p, size, 256, None)
        assert rc > 0, ld      # the runtime's word that there is no device; -1 would be a refusal


@pytest.mark.gpu
@pytest.mark.parametrize("n", [4, 64])
@pytest.mark.parametrize("v, k, kind", [(40, 300, F32), (150, 100, F32), (300, 200, BF16), (70, 600, F16), (66, 31, BF16)])
def test_few_rows_of_items_far_apart(ops, n, v, k, kind):
    """Items 2^24 values apart and one value less, for the paths that take a few rows."""
    c = _case(n, v, k, kind, True, seed=n + v + k)
    args = {a: b for a, b in c.items() if a != "weight"}
    e = _exact(**c)
    b = _bounds(e, kind, c["bias"], c["scale"], k, 4.0)
    for ld in (2 ** 24, 2 ** 24 - 1):
        flat = torch.empty((v - 1) * ld + k, dtype=kind, device="cuda:0")
        far = flat.as_strided((v, k), (ld, 1))
        far.copy_(c["items"])
        _close(softmax.softmax_nll(ops, **dict(args, items=far)), e, b, ("loss", "lse"))
        del flat, far


@pytest.mark.parametrize("device", ["cuda", "cuda:0"])
@pytest.mark.parametrize("call", [softmax.softmax_nll, softmax.softmax_nll_grad])
def test_tensors_of_another_device_are_refused(call, device):
    """Also where the operators' device was given without a number, and where one tensor alone is elsewhere."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    ops = _Recorder()
    ops.device = torch.device(device)
    with FakeTensorMode():
        for at in (("cuda:1",) * 4, ("cuda:0", "cuda:1", "cuda:0", "cuda:0"), ("cuda:0", "cuda:0", "cuda:1", "cuda:0"), ("cuda:0",) * 3 + ("cuda:1",)):
            args = dict(x=torch.empty(4, 5, device=at[0]), items=torch.empty(7, 5, device=at[1]), target=torch.empty(4, dtype=torch.int64, device=at[2]),
                        bias=torch.empty(7, device=at[3]))
            with pytest.raises(ValueError, match="expected cuda"):
                call(ops, **args)
    assert ops.calls == []


def test_operators_without_a_device_number_are_those_of_the_current_device(monkeypatch):
    import contextlib
    from hpfrec_amd import ops_hip
    monkeypatch.setattr(torch.cuda, "is_available", lambda: True)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 3)
    monkeypatch.setattr(torch.cuda, "device", lambda d: contextlib.nullcontext())
    monkeypatch.setattr(_lib, "lib", lambda: None)
    monkeypatch.setattr(_lib, "device_info", lambda: (256, "gfx950"))
    for given in (None, "cuda", torch.device("cuda"), "cuda:3"):
        assert ops_hip.HipOps(given).device == torch.device("cuda", 3)
    assert ops_hip.HipOps("cuda:1").device == torch.device("cuda", 1)


@pytest.mark.gpu
@pytest.mark.parametrize("n, k", [(40, 50), (40, 300), (100, 50), (100, 300)])
def test_the_largest_32_bit_values(ops, n, k):
    """Items up to the largest number of the type -- its upper 2^-8 is beyond bfloat16 --, rows small enough for ordinary logits."""
    gen = torch.Generator(device="cuda:0").manual_seed(9)
    items = torch.zeros((200, k), device="cuda:0")
    items[:, 0] = torch.finfo(F32).max * (1 - 2.0 ** -8 * torch.rand(200, device="cuda:0", generator=gen))
    items[::2, 0] *= -1
    items[0, 0] = torch.finfo(F32).max
    x = torch.zeros((n, k), device="cuda:0")
    x[:, 0] = 2.0 ** -125 * (1 + torch.arange(n, device="cuda:0") % 4)     # (one set bit or two: its second part is zero)
    target = torch.arange(n, device="cuda:0") % 200
    e = _exact(x, items, target, None, None, 1.0)
    b = _bounds(e, F32, None, 1.0, k)
    _close(softmax.softmax_nll(ops, x, items, target), e, b, ("loss", "lse"))
    loss, _, ditems, _ = softmax.softmax_nll_grad(ops, x, items, target)
    _close((loss,), e, b, ("loss",))
    assert bool(torch.isfinite(ditems).all())


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [F32, BF16, F16])
@pytest.mark.parametrize("n, k", [(40, 50), (40, 300), (100, 50), (100, 300)])
def test_infinite_values(ops, n, k, kind):
    """32 bits: logits of NaN.  16 bits: what the products are, so that -inf is masked."""
    c = _case(n, 200, k, kind, True, seed=33)
    c["x"][:, 3] = c["x"][:, 3].abs() + 0.25
    live = c["target"] >= 0
    c["target"] = torch.where(live & (c["target"] == 70), 71, c["target"])
    c["items"][70, 3] = -float("inf")
    nll = {a: b for a, b in c.items() if a != "weight"}
    loss, lse = softmax.softmax_nll(ops, **nll)
    if kind == F32:
        assert bool(torch.isnan(loss[live]).all()) and bool(torch.isnan(lse).all())
        assert bool(torch.isnan(softmax.softmax_nll_grad(ops, **c)[0][live]).all())
    else:
        bias = c["bias"].clone()
        bias[70] = -float("inf")
        want = softmax.softmax_nll(ops, **dict(nll, bias=bias))
        assert torch.equal(loss, want[0]) and torch.equal(lse, want[1])
        loss, dx, _, _ = softmax.softmax_nll_grad(ops, **c)
        assert torch.equal(loss, softmax.softmax_nll_grad(ops, **dict(c, bias=bias))[0]) and bool(torch.isnan(dx[live, 3]).all())
    c["items"][70, 3] = float("inf")
    assert bool(torch.isnan(softmax.softmax_nll(ops, **nll)[0][live]).all())
    c["items"][70, 3] = 0.0
    c["x"][6, 3] = float("inf")          # one row alone
    loss = softmax.softmax_nll(ops, **nll)[0]
    assert math.isnan(float(loss[6])) and bool(torch.isfinite(loss[torch.arange(n, device="cuda:0") != 6]).all())


def test_given_outputs_are_known_to_have_changed_and_no_graph_is_made():
    a = _good(x=torch.ones(4, 5, requires_grad=True), items=torch.ones(7, 5, requires_grad=True))
    loss, lse = softmax.softmax_nll(**a)
    out = dict(dx=torch.ones(4, 8)[:, :5], ditems=torch.ones(7, 5), dbias=torch.ones(7))
    got = softmax.softmax_nll_grad(**a, **out)
    assert not any(t.requires_grad for t in (loss, lse) + got)
    assert all(t._version == 1 for t in out.values()) and a["x"]._version == a["items"]._version == a["bias"]._version == 0
    table = torch.full((7, 5), 2.0, requires_grad=True)
    late = (table * table).sum()                # its backward pass needs the table as it was
    with torch.no_grad():
        softmax.softmax_nll_grad(**a, ditems=table)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        late.backward()
    with torch.inference_mode():
        softmax.softmax_nll_grad(**a, ditems=torch.ones(7, 5))


@pytest.mark.parametrize("call", [softmax.softmax_nll, softmax.softmax_nll_grad])
@pytest.mark.parametrize("scale", [1e39, -1e39, 3.5e38, 1e300, 2.0 ** 127, -3e38])
def test_scales_that_32_bits_do_not_hold_are_refused(call, scale):
    a = _good(scale=scale)
    with pytest.raises(ValueError, match="scale"):
        call(**a)
    assert a["ops"].calls == []
    call(**_good(scale=-1.7e38))


def test_c_entries_refuse_such_a_scale():
    if torch.cuda.is_available():
        pytest.skip("shown without a GPU: a call that is not refused would read host addresses")
    L = ctypes.CDLL(_lib.build())
    vp, i64, ci, cf = ctypes.c_void_p, ctypes.c_int64, ctypes.c_int, ctypes.c_float
    L.hpf_hip_softmax_nll.argtypes = [vp, i64, vp, i64, vp, vp, cf, i64, i64, i64, ci, vp, vp, vp, i64, ci, vp]
    L.hpf_hip_softmax_nll_grad.argtypes = [vp, i64, vp, i64, vp, vp, vp, cf, i64, i64, i64, ci, vp, vp, i64, vp, i64, vp, vp, i64, ci, vp]
    buf = ctypes.create_string_buffer(1024)
    p = (ctypes.addressof(buf) + 255) // 256 * 256
    for scale in (float("inf"), -float("inf"), float("nan"), 2.0 ** 127):
        assert L.hpf_hip_softmax_nll(p, 5, p, 5, p, None, scale, 4, 7, 5, 0, p, None, p, 1 << 40, 256, None) == -1
        assert L.hpf_hip_softmax_nll_grad(p, 5, p, 5, p, None, None, scale, 4, 7, 5, 0, p, p, 5, p, 5, None, p, 1 << 40, 256, None) == -1


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [F32, BF16, F16])
@pytest.mark.parametrize("k", [50, 300])
@pytest.mark.parametrize("power", [-120, -100, 98, 110, 125])
def test_weights_of_any_size(ops, power, k, kind):
    """Largest weights of 2^power to 2^(power + 2), and a scale that brings the tables' gradients back to ordinary sizes (logits are biases)."""
    c = _case(90, 300, k, kind, True, seed=81)
    c["weight"] = (c["weight"].clamp(-2, 2) * 2.0 ** power).float()
    c["scale"] = 2.0 ** (-power if power > 0 else 0)
    e = _exact(**c)
    b = _bounds(e, kind, c["bias"], c["scale"], k, 2 * float(c["weight"].abs().max()))
    _, dx, ditems, dbias = softmax.softmax_nll_grad(ops, **c)
    # sums of numbers below the normal ones; and a result below 2^-126 is rounded by up to half of the type's least number, which for
    # bfloat16 (7 bits of mantissa) is 2^-133 (half precision's 2^-24 is in the bounds)
    least = 2.0 ** -149 * 90 + (2.0 ** -134 if kind == BF16 else 0.0)
    _close((dx, ditems, dbias), e, {name: x + least for name, x in b.items()}, ("dx", "ditems", "dbias"))


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [F32, BF16, F16])
@pytest.mark.parametrize("n, k", [(20, 50), (300, 50), (300, 300)])
def test_far_and_near_pieces_of_a_long_catalogue(ops, n, k, kind):
    """Most items far below, a few near zero in one piece of the catalogue alone, the targets among either: shares are those of the
    near ones, and the far pieces' sums vanish beside them.  Then one item far above all: it has every share."""
    v, near = 30000, torch.arange(17000, 17040, device="cuda:0")
    c = _case(n, v, k, kind, True, seed=91)
    bias = torch.full((v,), -1e8, device="cuda:0")
    bias[near] = c["bias"][near]
    live = c["target"] >= 0
    c["target"] = torch.where(live, near[torch.arange(n, device="cuda:0") % 40], c["target"])
    c["target"][7] = 3                       # far, whatever the others
    few = dict(c, items=c["items"][near], bias=bias[near], target=torch.where(live, c["target"] - 17000, c["target"]))
    few["target"][7] = -1
    e = _exact(**few)
    b = _bounds(e, kind, few["bias"], c["scale"], k, 2 * float(c["weight"].abs().max()))
    (loss, lse), (gloss, dx, ditems, dbias) = _both(ops, dict(c, bias=bias))
    rest = torch.arange(n, device="cuda:0") != 7
    _close((torch.where(rest, loss, 0.0), lse), e, b, ("loss", "lse"))
    _close((torch.where(rest, gloss, 0.0), torch.where(rest[:, None], dx, 0.0)), e, b, ("loss", "dx"))
    assert abs(float(loss[7]) / 1e8 - 1) < 1e-6 and bool(torch.isfinite(dx[7]).all())
    g7 = c["weight"][7] * torch.softmax(e["z"][7], 0)       # row 7's shares, which `few` left out
    got = ditems[near].double() - c["scale"] * g7[:, None] * c["x"][7].double()
    assert bool(((got - e["ditems"]).abs() <= b["ditems"] + (2 * HALF[kind] + 1e-4) * (abs(c["scale"]) * g7.abs()[:, None] * c["x"][7].double().abs() + e["ditems"].abs())).all())
    assert bool(((dbias[near].double() - g7 - e["dbias"]).abs() <= b["dbias"] + 1e-4 * g7.abs()).all())
    far = torch.ones(v, dtype=torch.bool, device="cuda:0")
    far[near] = False
    far[3] = False
    assert not bool(ditems[far].any()) and not bool(dbias[far].any())
    assert abs(float(dbias[3]) + float(c["weight"][7])) <= 64 * U * abs(float(c["weight"][7]))
    bias[29990] = 3e8
    (loss, lse), (_, _, ditems, dbias) = _both(ops, dict(c, bias=bias))
    w = torch.where(live, c["weight"].double(), 0.0)
    assert bool(((lse.double() / 3e8 - 1).abs() <= 8 * U).all()) and abs(float(dbias[29990]) - float(w.sum())) <= 64 * U * float(w.abs().sum())
    assert bool(((ditems[29990].double() - c["scale"] * (w @ c["x"].double())).abs() <= abs(c["scale"]) * (w.abs() @ c["x"].double().abs()) * (64 * U + 2 * HALF[kind])).all())
