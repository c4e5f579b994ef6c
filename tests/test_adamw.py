"""The AdamW step (hpfrec_amd.adamw, hpf_hip_adamw_step): refusals on the CPU, results on the GPU against 64-bit arithmetic
and, for the 8-bit moments, code by code against the same roundings in numpy."""
import ctypes
from types import SimpleNamespace

import numpy as np
import pytest
import torch

from hpfrec_amd import _lib, adamw

U = 2.0 ** -24   # half a step of a 32-bit float
F8 = torch.float8_e4m3fn


# ---------------------------------------------------------------------------------------------
# refusals (no GPU: the checks run before any launch)
# ---------------------------------------------------------------------------------------------
class _Recorder:
    device = torch.device("cpu")

    def __init__(self):
        self.calls = []

    def adamw_step(self, tensors, ptype, gtype, bits, step, advance, *rest):
        self.calls.append((len(tensors), ptype, gtype, bits, advance))


def _call(**change):
    p = [torch.ones(5, 3), torch.ones(4, dtype=torch.bfloat16)]
    a = dict(adamw.adamw_state(p), params=p, grads=[torch.ones(5, 3), torch.ones(4, dtype=torch.bfloat16)])
    a.update(change)
    ops = a.pop("ops", None) or _Recorder()
    adamw.adamw_step(ops, **a)
    return ops.calls


def test_calls_of_one_combination_of_types_are_grouped():
    assert _call() == [(1, torch.float32, torch.float32, 32, False), (1, torch.bfloat16, torch.bfloat16, 32, True)]
    none = adamw.adamw_state([torch.ones(1)])["step"]
    assert _call(params=[], grads=[], m=[], v=[], masters=[], m_scale=None, v_scale=None, step=none) == [(0, torch.float32, torch.float32, 32, True)]


@pytest.mark.parametrize("change, words", [
    (dict(grads=[torch.ones(5, 3)]), "entries"),
    (dict(grads=[torch.ones(3, 5), torch.ones(4, dtype=torch.bfloat16)]), "shape"),
    (dict(grads=[torch.ones(3, 5).t(), torch.ones(4, dtype=torch.bfloat16)]), "contiguous"),
    (dict(grads=[torch.ones(5, 3, dtype=torch.float64), torch.ones(4)]), "must be a tensor of"),
    (dict(params=[torch.ones(5, 3, dtype=torch.int32), torch.ones(4)]), "must be a tensor of"),
    (dict(m=[torch.ones(5, 3), torch.ones(4, dtype=torch.bfloat16)]), "must be a tensor of"),
    (dict(m=[torch.ones(5, 3), torch.ones(4).to(F8)]), "v"),
    (dict(masters=None), "masters"),
    (dict(masters=[torch.ones(5, 3), torch.ones(4)]), "has none"),
    (dict(m_scale=[torch.ones(1), None]), "no scales"),
    (dict(m=[torch.ones(5, 3).to(F8), torch.ones(4)], v=[torch.ones(5, 3).to(F8), torch.ones(4)]), "m_scale"),
    (dict(step=torch.zeros(1)), "step"),
    (dict(step=torch.zeros(2, dtype=torch.int64)), "step"),
    (dict(step=0), "step"),
    (dict(lr=-1.0), "lr"),
    (dict(lr=float("nan")), "lr"),
    (dict(lr=torch.ones(1, dtype=torch.float64)), "lr"),
    (dict(betas=(1.0, 0.9)), "betas"),
    (dict(betas=(0.9, -0.1)), "betas"),
    (dict(eps=-1e-8), "eps"),
    (dict(weight_decay=[0.1]), "weight_decay"),
    (dict(weight_decay=float("inf")), "weight_decay"),
    (dict(ops=SimpleNamespace(device=torch.device("cuda:0"))), "expected cuda"),
])
def test_refusals(change, words):
    with pytest.raises(ValueError, match=words):
        _call(**change)


def test_overlapping_tensors_are_refused():
    p = torch.ones(8)
    st = adamw.adamw_state([p, p])
    with pytest.raises(ValueError, match="overlap"):
        _call(params=[p, p], grads=[torch.ones(8), torch.ones(8)], **st)
    st = adamw.adamw_state([p[:4], p[4:]])
    assert len(_call(params=[p[:4], p[4:]], grads=[torch.ones(4), torch.ones(4)], **st)) == 1
    both = torch.ones(12)
    st = adamw.adamw_state([both[:8]])
    with pytest.raises(ValueError, match="gradient overlaps"):
        _call(params=[both[:8]], grads=[both[4:]], **st)
    shared = torch.ones(4)   # one gradient for two parameters is read twice: allowed
    st = adamw.adamw_state([p[:4], p[4:]])
    _call(params=[p[:4], p[4:]], grads=[shared, shared], **st)


def test_state_refusals():
    with pytest.raises(ValueError):
        adamw.adamw_state([torch.ones(3)], 16)
    with pytest.raises(ValueError):
        adamw.adamw_state([])


def test_c_entry_refuses_before_touching_the_gpu():
    from hpfrec_amd.ops_hip import AdamwTensor
    L = ctypes.CDLL(_lib.build())
    vp, ci, cd = ctypes.c_void_p, ctypes.c_int, ctypes.c_double
    L.hpf_hip_adamw_step.argtypes = [vp, ci, ci, ci, ci, vp, ci, vp, cd, cd, cd, cd, ctypes.c_uint64, ci, vp]
    buf = ctypes.create_string_buffer(256)
    p = (ctypes.addressof(buf) + 15) // 16 * 16

    def rc(fields=(p, p, p, p, None, None, None, 3, 0.0, 0, 0), n=1, ptype=0, gtype=0, bits=32, step=p, betas=(0.9, 0.999), eps=1e-8, grid=8):
        d = (AdamwTensor * 1)(fields)
        return L.hpf_hip_adamw_step(d, n, ptype, gtype, bits, step, 1, None, 1e-3, betas[0], betas[1], eps, 0, grid, None)

    EINVAL, EUNSUPPORTED = -1, -2
    assert rc(n=-1) == EINVAL and rc(step=None) == EINVAL and rc(grid=0) == EINVAL
    assert rc(bits=16) == EUNSUPPORTED and rc(ptype=3) == EUNSUPPORTED and rc(gtype=-1) == EUNSUPPORTED
    assert rc(betas=(1.0, 0.9)) == EINVAL and rc(betas=(0.9, float("nan"))) == EINVAL and rc(eps=-1.0) == EINVAL
    for i in range(4):   # a missing pointer
        f = [p, p, p, p, None, None, None, 3, 0.0, 0, 0]
        f[i] = None
        assert rc(tuple(f)) == EINVAL
    assert rc((p, p, p, p, p, None, None, 3, 0.0, 0, 0)) == EINVAL              # a master of a float32 parameter
    assert rc((p, p, p, p, None, None, None, 3, 0.0, 0, 0), ptype=1) == EINVAL  # no master of a bfloat16 one
    assert rc(bits=8) == EINVAL                                                 # no scales
    assert rc((p, p, p, p, None, p, p, 3, 0.0, 0, 0)) == EINVAL                 # scales of 32-bit moments
    assert rc((p + 2, p, p, p, None, None, None, 3, 0.0, 0, 0)) == EINVAL       # misaligned float32
    assert rc((p, p, p, p, None, None, None, -3, 0.0, 0, 0)) == EINVAL


# ---------------------------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------------------------
B1, B2, EPS, LR, WD = 0.9, 0.999, 1e-8, 1e-2, 0.1


def _wide(p, g, m, v, t):
    """One step in 64 bits, and bounds on what 32-bit rounding of each operation may add.  m: constant, two products, sum
    (each U of |b1 m| + |c1 g|); v: constant, square, product, sum; p: 3 U of |p| for factor, product and sum, and for the
    quotient the rounded rate, product, root (half of v's error, its own), the root's and eps' sum, two divisions."""
    p, g, m, v = (x.double() for x in (p, g, m, v))
    m1, v1 = B1 * m + (1 - B1) * g, B2 * v + (1 - B2) * g * g
    size = B1 * m.abs() + (1 - B1) * g.abs()
    den = torch.sqrt(v1 / (1 - B2 ** t)) + EPS
    rate = LR / (1 - B1 ** t)
    p1 = p * (1 - LR * WD) - rate * m1 / den
    tiny = 2.0 ** -148   # below the normal numbers a rounding is absolute
    return (p1, m1, v1), (4 * U * p.abs() + 16 * U * rate * size / den + tiny, 4 * U * size + tiny, 5 * U * v1 + tiny)


def _mix(x):
    with np.errstate(over="ignore"):
        x = x ^ (x >> np.uint32(16))
        x = x * np.uint32(0x9E3779B1)
        x = x ^ (x >> np.uint32(15))
        x = x * np.uint32(0x6A09E669)
        return x ^ (x >> np.uint32(16))


def _words(seed, t, number, n, first=0):
    one = lambda v: np.array([v & 0xFFFFFFFF], np.uint32)  # noqa: E731
    with np.errstate(over="ignore"):
        key = _mix(_mix(_mix(_mix(one(seed)) ^ one(seed >> 32)) + one(t)) + one(number))
        i = np.arange(first, first + n, dtype=np.uint64)
        return _mix(i.astype(np.uint32) + key + (i >> np.uint64(32)).astype(np.uint32) * np.uint32(0x9E3779B1))


_CODES = np.array([float(c) for c in torch.arange(127, dtype=torch.uint8).view(F8).float()])


def _encode(x, chance16, least):
    """float32 x -> (codes' values, scales) by the table of e4m3 and each value's place between its two neighbours."""
    n = x.size
    pad = np.zeros(-(-n // 256) * 256, np.float32)
    pad[:n] = x
    top = np.abs(pad).reshape(-1, 256).max(axis=1).astype(np.float64)
    scale = np.ones_like(top)
    scale[top > 0] = 2.0 ** np.maximum(np.floor(np.log2(top[top > 0])) - 7, -126)
    a = np.abs(x.astype(np.float64)) / scale[np.arange(n) // 256]
    low = np.where(a < 2.0 ** -6, 2.0 ** -6, 0.0)
    a = (a + low).astype(np.float32).astype(np.float64) - low      # below 2^-6 a 32-bit sum with 2^-6 (2^-30 of a step's 2^-9)
    at = np.searchsorted(_CODES, a, side="right") - 1
    part = (a - _CODES[at]) / (_CODES[at + 1] - _CODES[at])
    part = np.floor(part * 2 ** 20) / 2 ** 20
    q = _CODES[at + (part + chance16 / 65536.0 >= 1.0)]
    if least:
        q[(q == 0) & (x > 0)] = 2.0 ** -9
    return np.copysign(q, x), scale


# ---------------------------------------------------------------------------------------------
# on the GPU
# ---------------------------------------------------------------------------------------------
@pytest.fixture(scope="module")
def ops():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    from hpfrec_amd.ops_hip import HipOps
    return HipOps("cuda:0")


def _tensors(shape, ptype, gtype, bits, seed, device="cuda:0"):
    gen = torch.Generator(device=device).manual_seed(seed)
    normal = lambda s: torch.randn(shape, device=device, generator=gen) * s  # noqa: E731
    p = normal(0.5)
    a = dict(params=[p.to(ptype)], grads=[normal(1e-2).to(gtype)], **adamw.adamw_state([p.to(ptype)], bits))
    if ptype != torch.float32:
        a["masters"] = [p]
    a["step"].fill_(4)
    if bits == 32:
        a["m"], a["v"] = [normal(1e-2)], [normal(1e-2).square()]
    else:
        a["m"], a["v"] = [normal(50.0).clamp(-240, 240).to(F8)], [normal(50.0).abs().clamp(max=240).to(F8)]
        a["m_scale"][0].fill_(2.0 ** -13)
        a["v_scale"][0].fill_(2.0 ** -12)
    return a


def _step(ops, a, **more):
    adamw.adamw_step(ops, **a, **dict(dict(lr=LR, betas=(B1, B2), eps=EPS, weight_decay=WD, seed=7), **more))


def _held(a, i=0):
    """float32 values that the step starts from."""
    p = a["params"][i] if a["masters"][i] is None else a["masters"][i]
    m, v = a["m"][i].float(), a["v"][i].float()
    if a["m"][i].dtype == F8:
        n = m.numel()
        m = m * a["m_scale"][i].repeat_interleave(256)[:n].view(m.shape)
        v = (v * a["v_scale"][i].repeat_interleave(256)[:n].view(m.shape)).square()
    return tuple(x.clone() for x in (p, a["grads"][i].float(), m, v))   # (the step works in place)


TYPES = [torch.float32, torch.bfloat16, torch.float16]
SIZES = [1, 3, 255, 256, 257, 4095, 4097, 100003]


@pytest.mark.gpu
@pytest.mark.parametrize("n", SIZES)
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("ptype, gtype", [(p, g) for p in TYPES for g in TYPES])
def test_one_step_against_64_bits(ops, n, bits, ptype, gtype):
    a = _tensors(n, ptype, gtype, bits, n)
    before = _held(a)
    _step(ops, a)
    (p, m, v), (bp, bm, bv) = _wide(*before, t=5)
    new = a["params"][0] if ptype == torch.float32 else a["masters"][0]
    assert int(a["step"]) == 5
    assert bool(((new.double() - p).abs() <= bp).all())
    if ptype != torch.float32:
        assert torch.equal(a["params"][0], new.to(ptype))
    if bits == 32:
        assert bool(((a["m"][0].double() - m).abs() <= bm).all()) and bool(((a["v"][0].double() - v).abs() <= bv).all())
    else:   # within a whole step of e4m3 (rounding is up or down): 2^-3 of the value, 2^-9 of the scale below
        for name, x, bound in (("m", m, bm), ("v", v.sqrt(), bv / (2 * v.sqrt()).clamp(min=1e-30))):
            s = a[name + "_scale"][0].double().repeat_interleave(256)[:n]
            off = (a[name][0].double() * s - x).abs()
            assert bool((off <= torch.maximum(x.abs() / 8, s * 2.0 ** -9) * 1.0000001 + 2 * bound).all())


@pytest.mark.gpu
@pytest.mark.parametrize("n", SIZES)
@pytest.mark.parametrize("ptype, gtype", [(torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16), (torch.float16, torch.float32)])
def test_8_bit_codes_are_the_same_roundings(ops, n, ptype, gtype):
    a = _tensors(n, ptype, gtype, 8, n + 1)
    _, g, m, v = (x.cpu().numpy().astype(np.float32) for x in _held(a))
    _step(ops, a, seed=(5 << 32) + 11)
    f = np.float32
    m1 = m * f(B1) + g * f(1 - B1)
    r1 = np.sqrt(v * f(B2) + (g * g) * f(1 - B2))
    w = _words((5 << 32) + 11, 5, 0, n)
    for name, x, chance, least in (("m", m1, w & np.uint32(0xFFFF), False), ("v", r1, w >> np.uint32(16), True)):
        q, s = _encode(x, chance.astype(np.float64), least)
        assert np.array_equal(a[name + "_scale"][0].cpu().numpy().astype(np.float64), s)
        assert np.array_equal(a[name][0].float().cpu().numpy().astype(np.float64), q)


@pytest.mark.gpu
def test_rounding_is_unbiased_and_lets_a_moment_move(ops):
    """b1 = 0 makes m the gradient itself: the mean of its codes over 400 steps is the gradient within 5 standard errors
    (a value's rounding deviates by at most half an e4m3 step).  And roots under zero gradients fall by sqrt(b2) a step:
    500 steps leave 0.7788 of their mean; the mean of 4096 walks of steps <= 2^-3, each with a variance of at most
    (drift a step) x (one code) -- 500 * 5e-4 * 2^-3 of the square -- deviates by less than 0.18 / 64 = 0.003; 5 of them."""
    n = 4096
    a = _tensors(n, torch.float32, torch.float32, 8, 3)
    g = a["grads"][0].double()
    total = torch.zeros_like(g)
    for _ in range(400):
        _step(ops, a, betas=(0.0, B2))
        total += a["m"][0].double() * a["m_scale"][0].double().repeat_interleave(256)
    scale = a["m_scale"][0].double().repeat_interleave(256)
    step = torch.maximum(g.abs() / 8, scale * 2.0 ** -9)
    assert bool(((total / 400 - g).abs() <= 5 * step / 2 / 20 + step * 2.0 ** -15).all())
    a = _tensors(n, torch.float32, torch.float32, 8, 4)
    a["grads"][0].zero_()
    a["v"][0].copy_(torch.full((n,), 200.0, device="cuda:0").to(F8))
    was = (a["v"][0].float().mean() * a["v_scale"][0][0]).item()
    for _ in range(500):
        _step(ops, a)
    now = (a["v"][0].float() * a["v_scale"][0].repeat_interleave(256)).mean().item()
    assert abs(now / was - 0.999 ** 250) < 0.015


@pytest.mark.gpu
def test_a_root_above_zero_is_never_held_as_zero(ops):
    a = _tensors(256, torch.float32, torch.float32, 8, 5)
    a["m"][0].copy_(torch.zeros(256).to(F8))
    a["v"][0].copy_(torch.zeros(256).to(F8))
    a["grads"][0].fill_(1e-9)
    a["grads"][0][0] = 1e3
    _step(ops, a)
    held = a["v"][0].float()
    assert held[0] >= 128 and bool((held[1:] == 2.0 ** -9).all())
    before = a["params"][0].clone()
    a["grads"][0].zero_()
    _step(ops, a)
    assert bool(((a["params"][0] - before * (1 - LR * WD)).abs()[1:] <= 1e-2).all())


@pytest.mark.gpu
def test_zero_tensors_stay_zero(ops):
    for bits in (32, 8):
        p = [torch.zeros(700, device="cuda:0")]
        st = adamw.adamw_state(p, bits)
        _step(ops, dict(st, params=p, grads=[torch.zeros(700, device="cuda:0")]))
        for x in (p[0], st["m"][0].float(), st["v"][0].float()):
            assert not bool(x.any())
        if bits == 8:
            assert bool((st["m_scale"][0] == 1).all())


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
def test_one_bad_gradient_spoils_its_own_value_alone(ops, bits, bad):
    a, b = (_tensors(600, torch.float32, torch.float32, bits, 6) for _ in range(2))
    for x in (a, b):
        x["grads"][0][300] = 0.0
    a["grads"][0][300] = bad
    _step(ops, a)
    _step(ops, b)
    rest = torch.arange(600, device="cuda:0") != 300
    for name in ("params", "m", "v"):
        x, y = a[name][0].float(), b[name][0].float()
        assert torch.equal(x[rest], y[rest]), name
        assert not bool(torch.isfinite(x[300])), name


@pytest.mark.gpu
def test_many_tensors_of_all_types_in_one_call(ops):
    """95 tensors -- more than one launch holds --, empty ones among them, of every type, with 32- and 8-bit moments."""
    shapes = [(0,), (1,), (7, 5), (300,), (64, 64), (5000,)]
    parts = [_tensors(shapes[i % 6], TYPES[i % 3], TYPES[i // 3 % 3], (32, 8)[i // 9 % 2], 100 + i) for i in range(95)]
    a = {k: [p[k][0] for p in parts] for k in parts[0] if k != "step"}
    a["step"] = parts[0]["step"]
    before = [_held(a, i) for i in range(95)]
    decay = [0.0 if i % 4 == 0 else WD for i in range(95)]
    _step(ops, a, weight_decay=decay)
    assert int(a["step"]) == 5
    for i in range(95):
        (p, _, _), (bp, _, _) = _wide(*before[i], t=5)
        if i % 4 == 0:
            p = p + before[i][0].double() * (LR * WD)
        new = a["params"][i] if a["masters"][i] is None else a["masters"][i]
        assert bool(((new.double() - p).abs() <= bp).all()), i


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("ptype", TYPES)
def test_unaligned_tensors_give_the_same(ops, bits, ptype):
    a, b = (_tensors(3001, ptype, ptype, bits, 9) for _ in range(2))
    for name in ("params", "grads", "m", "v", "masters"):   # views that begin one value into their storage
        x = b[name][0]
        if x is not None:
            raw = torch.zeros((x.numel() + 1) * x.element_size(), dtype=torch.uint8, device="cuda:0")
            y = raw.view(x.dtype)[1:]
            y.view(torch.uint8).copy_(x.view(torch.uint8))
            b[name] = [y]
    _step(ops, a)
    _step(ops, b)
    for name in ("params", "m", "v"):
        assert torch.equal(a[name][0].view(torch.uint8), b[name][0].view(torch.uint8)), name


@pytest.mark.gpu
def test_what_lies_beside_a_tensor_is_left_alone(ops):
    for bits in (32, 8):
        a = _tensors(1030, torch.float32, torch.float32, bits, 10)
        kept = {}
        for name in ("params", "m", "v"):
            x = a[name][0]
            raw = torch.full((1030 * x.element_size() + 64,), 77, dtype=torch.uint8, device="cuda:0")
            y = raw[:1030 * x.element_size()].view(x.dtype)
            y.view(torch.uint8).copy_(x.view(torch.uint8))
            kept[name], a[name] = raw, [y]
        _step(ops, a)
        for raw in kept.values():
            assert bool((raw[-64:] == 77).all())


@pytest.mark.gpu
def test_graph_replays_stream_and_device_side_rate(ops):
    """A captured step replayed three times, eager steps of another state and synchronisations in between, is the eager
    sequence; the rate is read from the device at each replay."""
    for bits in (32, 8):
        a, b, other = (_tensors(5001, torch.bfloat16, torch.bfloat16, bits, 11) for _ in range(3))
        lr = torch.full((1,), LR, device="cuda:0")
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            _step(ops, other, lr=lr)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            _step(ops, a, lr=lr)
        for k in range(3):
            lr.fill_(LR * (k + 1))
            graph.replay()
            _step(ops, b, lr=float(np.float32(LR * (k + 1))))
            _step(ops, other)
            torch.cuda.synchronize()
            for name in ("params", "masters", "m", "v"):
                assert torch.equal(a[name][0].view(torch.uint8), b[name][0].view(torch.uint8)), (bits, k, name)
            assert int(a["step"]) == int(b["step"]) == 5 + k


@pytest.mark.gpu
def test_more_than_2_to_the_32_values(ops):
    """The last values of a tensor whose indexes pass 32 bits: those of a small tensor of the same numbers and bits."""
    n = 2 ** 32 + 300
    if torch.cuda.mem_get_info()[0] < 60 << 30:
        pytest.skip("not enough memory")
    p = torch.full((n,), 0.25, device="cuda:0")
    g = torch.full((n,), 1e-3, device="cuda:0")
    st = adamw.adamw_state([p], 8)
    _step(ops, dict(st, params=[p], grads=[g]))
    f = np.float32
    tail = n - 2 ** 32
    w = _words(7, 1, 0, tail, first=2 ** 32)
    m1 = np.full(tail, f(1e-3) * f(1 - B1), np.float32)
    q, s = _encode(m1, (w & np.uint32(0xFFFF)).astype(np.float64), False)
    assert np.array_equal(st["m"][0][2 ** 32:].float().cpu().numpy().astype(np.float64), q)
    (want, _, _), (bound, _, _) = _wide(torch.tensor(0.25), torch.tensor(f(1e-3)), torch.tensor(0.0), torch.tensor(0.0), t=1)
    for i in (0, 2 ** 31, 2 ** 32 - 1, 2 ** 32, n - 1):
        assert abs(float(p[i]) - float(want)) <= float(bound)


def test_a_step_on_another_device_is_refused():
    from torch._subclasses.fake_tensor import FakeTensorMode
    ops = _Recorder()
    for device in ("cuda", "cuda:0"):
        ops.device = torch.device(device)
        with FakeTensorMode():
            p = [torch.empty(5, 3, device="cuda:1")]
            with pytest.raises(ValueError, match="expected cuda"):
                adamw.adamw_step(ops, p, [torch.empty(5, 3, device="cuda:1")], **adamw.adamw_state(p))
    assert ops.calls == []


def test_c_entry_refuses_a_tensor_that_is_too_large_before_it_moves_any():
    """A tensor of over 2^39 - 2^16 values behind an ordinary one: refused ahead of every launch, which would give the runtime's word
    that there is no device (and on one would read these host addresses)."""
    from hpfrec_amd.ops_hip import AdamwTensor
    L = ctypes.CDLL(_lib.build())
    vp, ci, cd = ctypes.c_void_p, ctypes.c_int, ctypes.c_double
    L.hpf_hip_adamw_step.argtypes = [vp, ci, ci, ci, ci, vp, ci, vp, cd, cd, cd, cd, ctypes.c_uint64, ci, vp]
    buf = ctypes.create_string_buffer(256)
    p = (ctypes.addressof(buf) + 15) // 16 * 16
    if torch.cuda.is_available():
        pytest.skip("shown without a GPU")
    for n in (2 ** 39 - 2 ** 16 + 1, 2 ** 39, 2 ** 62, 2 ** 63 - 1):
        d = (AdamwTensor * 2)((p, p, p, p, None, None, None, 3, 0.0, 0, 0), (p, p, p, p, None, None, None, n, 0.0, 1, 0))
        assert L.hpf_hip_adamw_step(d, 2, 0, 0, 32, p, 1, None, 1e-3, 0.9, 0.999, 1e-8, 0, 8, None) == -2, n


def test_parameters_are_known_to_have_changed():
    p = [torch.full((5, 3), 2.0, requires_grad=True), torch.ones(4, dtype=torch.bfloat16)]
    st = adamw.adamw_state(p)
    late = (p[0] * p[0]).sum()                  # its backward pass needs the parameter as it was
    _call(params=p, grads=[torch.ones(5, 3), torch.ones(4)], **st)
    assert p[0]._version == p[1]._version == st["masters"][1]._version == 1
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        late.backward()
    with torch.inference_mode():
        p = [torch.ones(3)]
        _call(params=p, grads=[torch.ones(3)], **adamw.adamw_state(p))


def test_a_rate_inside_what_the_step_writes_is_refused():
    p = torch.ones(8)
    st = adamw.adamw_state([p])
    for lr in (p[3:4], st["m"][0][:1], st["v"][0][7:]):
        with pytest.raises(ValueError, match="lr overlaps"):
            _call(params=[p], grads=[torch.ones(8)], lr=lr, **st)
    g = torch.full((8,), 1e-3)
    assert len(_call(params=[p], grads=[g], lr=g[:1], **st)) == 1      # read twice: allowed


@pytest.mark.parametrize("number", [np.float32(0.25), np.float64(0.25), np.int64(1), 1, True])
def test_numbers_of_numpy_are_numbers(number):
    assert len(_call(weight_decay=number, lr=number)) == 2
