"""The operators measured beside the framework's own: the full-catalogue softmax loss with its gradients, and the AdamW step.

Plain forms are elementary torch operations in 32 bits; with `own` set, `run` calls hpfrec_amd instead.

softmax_nll       z[n, v] = scale * <x[n], items[v]> + bias[v];  loss[n] = logsumexp_v z[n, v] - z[n, target[n]]
softmax_nll_grad  the same loss and the gradients of  sum_n weight[n] * loss[n]  in x, items and bias
adamw_step        decoupled weight decay, moments in 32 bits or in 8 (e4m3 with one power of two per 256 values)

A negative target is a row of padding: its loss and its gradients are zero.
"""
import math

import torch

own = False

DEV = "cuda"
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BLOCK = 256                     # values that share a scale in an 8-bit moment
PIECE = 32768                   # items that the plain form sums at once
BETAS, EPS, DECAY, LR, SEED = (0.9, 0.999), 1e-8, 0.01, 1e-3, 20240607
MASK32, MUL_A, MUL_B = 0xFFFFFFFF, 0x9E3779B1, 0x6A09E669


def listed():
    return [
        # one event scored against the MovieLens-20M-sized catalogue (27k items, k=50): what a single request pays
        dict(name="nll one event f32", op="nll", n=1, v=27000, k=50, type="f32", bias=False),
        # a small serving batch against the 380k-item catalogue
        dict(name="nll batch bf16", op="nll", n=61, v=380000, k=100, type="bf16", bias=True),
        # held-out evaluation of a whole chunk of events, 32-bit tables in the framework's padded rows
        dict(name="nll evaluation f32", op="nll", n=8192, v=380000, k=50, type="f32", bias=True),
        # the smallest training step: a ragged handful of events on a 1000-item catalogue
        dict(name="grad tiny f32", op="grad", n=33, v=1000, k=50, type="f32", bias=True),
        # an ordinary step on the MovieLens-20M-sized catalogue
        dict(name="grad ordinary f32", op="grad", n=4001, v=27000, k=50, type="f32", bias=True),
        # 16-bit tables, a wider model (k=200), 100k items
        dict(name="grad wide tables bf16", op="grad", n=8192, v=100000, k=200, type="bf16", bias=True),
        # the widest rows the framework takes (k up to 1024), odd on purpose, half precision
        dict(name="grad widest rows f16", op="grad", n=2048, v=50001, k=1000, type="f16", bias=False),
        # the largest: 380k items, k=100, 32 bits
        dict(name="grad largest f32", op="grad", n=8192, v=380000, k=100, type="f32", bias=False),
        # one step over the tables of a debug-sized model (2k users, 1k items, their biases)
        dict(name="adamw tiny f32", op="adamw", users=2001, items=1000, k=50, type="f32", bits=32),
        # the million-user model (1M x 380k, k=50) in 32 bits throughout
        dict(name="adamw million users f32", op="adamw", users=1000000, items=380000, k=50, type="f32", bits=32),
        # MovieLens-20M-sized tables, moments in 8 bits
        dict(name="adamw 8 bits f32", op="adamw", users=138000, items=27000, k=50, type="f32", bits=8),
        # the million-user model at k=100: bf16 tables with 32-bit masters, moments in 8 bits
        dict(name="adamw 8 bits bf16", op="adamw", users=1000000, items=380000, k=100, type="bf16", bits=8),
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["nll", "grad", "adamw"])
    kind = rng.choice(["f32", "bf16", "f16"])
    if op == "adamw":
        return dict(op=op, users=_log_uniform(rng, 100, 1000000), items=_log_uniform(rng, 100, 380000), k=_log_uniform(rng, 5, 100),
                    type=kind, bits=rng.choice([32, 8]))
    while True:
        n, v, k = _log_uniform(rng, 1, 8192), _log_uniform(rng, 100, 380000), _log_uniform(rng, 5, 1000)
        if n * v * max(k, 100) <= 8192 * 380000 * 100:
            return dict(op=op, n=n, v=v, k=k, type=kind, bias=rng.random() < 0.5)


# -- what a program has in hand ----------------------------------------------------------------------------------------


def _rows(n, k, kind, spread, gen):
    """n rows of k values; 32-bit tables in rows padded to a power of two, as the framework lays its tables out."""
    ld = 1 << max(5, (k - 1).bit_length()) if kind == "f32" else k
    t = torch.zeros((n, ld), device=DEV, dtype=TYPES[kind])
    t[:, :k] = torch.randn((n, k), device=DEV, generator=gen).mul_(spread)
    return t[:, :k]


def _shapes(case):
    """One model's parameters: two factor tables and the items' biases."""
    return [(case["users"], case["k"]), (case["items"], case["k"]), (case["items"],)]


def prepare(case, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed * 7919 + 13)
    if case["op"] == "adamw":
        s = dict(op="adamw", step=torch.full((1,), 100, device=DEV, dtype=torch.int64))
        tensors = [_trained_tensor(shape, TYPES[case["type"]], case["bits"], gen) for shape in _shapes(case)]
        for name in tensors[0]:
            got = [t[name] for t in tensors]
            s[name] = None if got[0] is None else got
        return s
    n, v, k = case["n"], case["v"], case["k"]
    # factors whose products have a spread of about 2, as of a trained model; an item's popularity falls as a power of its rank
    spread = (2.0 / math.sqrt(k)) ** 0.5
    s = dict(op=case["op"], scale=1.25, x=_rows(n, k, case["type"], spread, gen), items=_rows(v, k, case["type"], spread, gen))
    rank = torch.randperm(v, device=DEV, generator=gen)
    s["bias"] = -0.8 * torch.log(rank.float() + 10.0) if case["bias"] else None
    popular = (torch.rand(n, device=DEV, generator=gen, dtype=torch.float64).mul_(math.log(v + 1.0)).exp_() - 1.0).long().clamp_(0, v - 1)
    s["target"] = torch.argsort(rank)[popular]
    if n > 8:  # rows of padding
        s["target"][torch.rand(n, device=DEV, generator=gen) < 0.02] = -1
    if case["op"] == "grad":  # an event counts as often as it was seen; half precision is trained with a scaled loss
        seen = 1.0 + torch.floor(-2.0 * torch.log(torch.rand(n, device=DEV, generator=gen).clamp_(min=1e-6)))
        s["weight"] = seen * ((4096.0 if case["type"] == "f16" else 1.0) / n)
    return s


def _trained_tensor(shape, kind, bits, gen):
    """A tensor in the midst of a training: its values, gradient and moments."""
    normal = lambda spread: torch.randn(shape, device=DEV, generator=gen).mul_(spread)  # noqa: E731
    p = normal(0.3)
    s = dict(params=p.to(kind), masters=None if kind == torch.float32 else p, grads=normal(1e-3).to(kind), m_scale=None, v_scale=None)
    if bits == 32:
        return dict(s, m=normal(3e-4), v=normal(1e-3).square_().add_(1e-8))
    power = lambda lo: torch.randint(lo, lo + 3, (-(-p.numel() // BLOCK),), device=DEV, generator=gen).float().exp2_()  # noqa: E731
    return dict(s, m=normal(40.0).clamp_(-250, 250).to(torch.float8_e4m3fn), v=normal(30.0).abs_().add_(20.0).clamp_(max=250).to(torch.float8_e4m3fn),
                m_scale=power(-20), v_scale=power(-17))


# -- one pass ------------------------------------------------------------------------------------------------------------


_ops = None


def _framework():
    global _ops
    if _ops is None:
        from hpfrec_amd.ops_hip import HipOps
        _ops = HipOps()
    return _ops


def run(s):
    if own:
        return _run_own(s)
    return {"nll": _plain_nll, "grad": _plain_grad, "adamw": _plain_adamw}[s["op"]](s)


def _run_own(s):
    ops = _framework()
    if s["op"] == "nll":
        from hpfrec_amd.softmax import softmax_nll
        loss, lse = softmax_nll(ops, s["x"], s["items"], s["target"], bias=s["bias"], scale=s["scale"])
        return dict(loss=loss, lse=lse)
    if s["op"] == "grad":
        from hpfrec_amd.softmax import softmax_nll_grad
        loss, dx, ditems, dbias = softmax_nll_grad(ops, s["x"], s["items"], s["target"], weight=s["weight"], bias=s["bias"], scale=s["scale"])
        return dict(loss=loss, dx=dx, ditems=ditems, dbias=dbias)
    from hpfrec_amd.adamw import adamw_step
    adamw_step(ops, s["params"], s["grads"], s["m"], s["v"], s["step"], masters=s["masters"], m_scale=s["m_scale"], v_scale=s["v_scale"],
               lr=LR, betas=BETAS, eps=EPS, weight_decay=DECAY, seed=SEED)
    return _adamw_outputs(s)


def _adamw_outputs(s):
    # the 8-bit moments come as they are held: float8 values and the 32-bit power of two that each block of them is times
    return {k: s[k] for k in ("params", "masters", "m", "v", "m_scale", "v_scale", "step")}


def _plain_logits(s):
    z = (s["x"].float() @ s["items"].float().t()).mul_(s["scale"])
    return z if s["bias"] is None else z.add_(s["bias"])


def _plain_loss(z, target):
    """loss and log-sum-exp of the rows; z becomes exp(z - its row's largest), `total` its sums."""
    live = target >= 0
    at = z.gather(1, target.clamp(min=0)[:, None])[:, 0]
    top = z.max(dim=1, keepdim=True).values
    z.sub_(top).exp_()
    total = z.sum(dim=1, keepdim=True)
    lse = (top + total.log())[:, 0]
    return torch.where(live, lse - at, torch.zeros_like(lse)), lse, total, live


def _plain_nll(s):
    loss, lse, _, _ = _plain_loss(_plain_logits(s), s["target"])
    return dict(loss=loss, lse=lse)


def _plain_grad(s):
    z = _plain_logits(s)
    loss, _, total, live = _plain_loss(z, s["target"])
    w = torch.where(live, s["weight"], torch.zeros_like(loss))
    z.mul_(w[:, None] / total)
    z.scatter_add_(1, s["target"].clamp(min=0)[:, None], -w[:, None])
    dx = sum(z[:, a:a + PIECE] @ s["items"][a:a + PIECE].float() for a in range(0, z.shape[1], PIECE))   # a long sum, in pieces
    return dict(loss=loss, dx=dx.mul_(s["scale"]).to(s["x"].dtype), ditems=(z.t() @ s["x"].float()).mul_(s["scale"]).to(s["items"].dtype),
                dbias=None if s["bias"] is None else z.sum(dim=0))


def _mix(x):
    """One 32-bit word from another (held in 64): two multiplications by odd constants between shifts."""
    x = x ^ (x >> 16)
    x = (x * MUL_A) & MASK32
    x = x ^ (x >> 15)
    x = (x * MUL_B) & MASK32
    return x ^ (x >> 16)


def _random_words(step, number, count):
    """The 32 random bits of each value of tensor `number` in the step that makes the counter `step`."""
    key = _mix((_mix((_mix(_mix(torch.full_like(step, SEED & MASK32)) ^ (SEED >> 32)) + (step & MASK32)) & MASK32) + number) & MASK32)
    i = torch.arange(count, device=DEV)
    return _mix(((i & MASK32) + key + (i >> 32) * MUL_A) & MASK32)


def _to_e4m3(a, bits16):
    """Non-negative a < 256 in e4m3, rounded up with the probability of its place between two neighbours."""
    low = torch.where(a < 2.0 ** -6, 2.0 ** -6, 0.0)   # puts the subnormals' fixed step at the end of a mantissa
    b = ((a + low).view(torch.int32) + (bits16 << 4).to(torch.int32)) & ~0xFFFFF
    return b.view(torch.float32) - low


def _pack8(x, bits16, least):
    """x in e4m3 and a power of two for each block: its largest finite magnitude becomes one from 128 up to 256."""
    n = x.numel()
    pad = torch.nn.functional.pad(x.reshape(-1), (0, -n % BLOCK)).view(-1, BLOCK)
    top = pad.abs().amax(dim=1)
    up = torch.where(top > 0, torch.frexp(top).exponent - 8, torch.zeros_like(top, dtype=torch.int32)).clamp(min=-126)
    scale = ((up + 127) << 23).view(torch.float32)
    q = (pad / scale[:, None]).reshape(-1)[:n].view(x.shape)
    a = _to_e4m3(q.abs(), bits16)
    if least:   # a root that is not zero keeps the smallest code: a later step divides by it
        a = torch.where((a == 0) & (x > 0), 2.0 ** -9, a)
    return torch.copysign(a, q).to(torch.float8_e4m3fn), scale


def _unpack8(q, scale):
    return q.float() * scale.repeat_interleave(BLOCK)[: q.numel()].view(q.shape)


def _plain_adamw(s):
    s["step"].add_(1)
    [_plain_step(s, i) for i in range(len(s["params"]))]
    return _adamw_outputs(s)


def _plain_step(s, i):
    b1, b2 = BETAS
    g, eight = s["grads"][i].float(), s["m_scale"] is not None
    m, v = s["m"][i], s["v"][i]
    if eight:   # the second moment is held as its root
        m, v = _unpack8(m, s["m_scale"][i]), _unpack8(v, s["v_scale"][i]).square()
    m = m * b1 + g * (1 - b1)
    v = v * b2 + (g * g) * (1 - b2)
    t = s["step"].double()
    rate, root = LR / (1 - b1 ** t), (1 - b2 ** t).sqrt()
    p = s["params"][i] if s["masters"] is None else s["masters"][i]
    p = p * (1 - LR * DECAY) - rate.float() * m / (v.sqrt() / root.float() + EPS)
    if s["masters"] is not None:
        s["masters"][i].copy_(p)
    s["params"][i].copy_(p)
    if eight:
        words = _random_words(s["step"], i, g.numel()).view(g.shape)
        (m, m_scale), (v, v_scale) = _pack8(m, words & 0xFFFF, False), _pack8(v.sqrt(), words >> 16, True)
        s["m_scale"][i].copy_(m_scale)
        s["v_scale"][i].copy_(v_scale)
    s["m"][i].copy_(m)
    s["v"][i].copy_(v)


# -- what it costs at least, and what it is exactly ------------------------------------------------------------------------


def work(case):
    if case["op"] == "adamw":
        count = sum(math.prod(shape) for shape in _shapes(case))
        size = TYPES[case["type"]].itemsize
        each = 2 * (2 * case["bits"] // 8) + size + (2 * size if size == 4 else size + 8)   # moments both ways, gradient, values (masters)
        return dict(bytes=count * each + (count // BLOCK * 16 if case["bits"] == 8 else 0), flops=count * 15)
    n, v, k, size = case["n"], case["v"], case["k"], TYPES[case["type"]].itemsize
    tables, rows = (n + v) * k * size + (4 * v if case["bias"] else 0), n * 16
    if case["op"] == "nll":
        return dict(bytes=tables + rows, flops=2.0 * n * v * k)
    return dict(bytes=2 * tables + rows, flops=6.0 * n * v * k)


def exact(case, seed):
    s = prepare(case, seed)
    if s["op"] == "adamw":
        t = int(s["step"]) + 1
        new = [_exact_step(s, i, t) for i in range(len(s["params"]))]
        return dict({name: [x[name] for x in new] for name in new[0]}, step=t)
    x, items, target = s["x"].double(), s["items"].double(), s["target"]
    n, v = x.shape[0], items.shape[0]
    loss, lse = torch.zeros(n, device=DEV, dtype=torch.float64), torch.zeros(n, device=DEV, dtype=torch.float64)
    dx, ditems, dbias = torch.zeros_like(x), torch.zeros_like(items), torch.zeros(v, device=DEV, dtype=torch.float64)
    for a in range(0, n, 512):
        z = s["scale"] * (x[a:a + 512] @ items.t())
        if s["bias"] is not None:
            z += s["bias"].double()
        lse[a:a + 512] = total = torch.logsumexp(z, dim=1)
        t = target[a:a + 512]
        r, c = torch.nonzero(t >= 0)[:, 0], t[t >= 0]
        loss[a + r] = total[r] - z[r, c]
        if s["op"] == "grad":
            g = torch.exp(z - total[:, None])
            g[r, c] -= 1
            g *= (s["weight"][a:a + 512].double() * (t >= 0))[:, None]
            dx[a:a + 512] = s["scale"] * (g @ items)
            ditems += s["scale"] * (g.t() @ x[a:a + 512])
            dbias += g.sum(dim=0)
    if s["op"] == "nll":
        return dict(loss=loss, lse=lse)
    return dict(loss=loss, dx=dx, ditems=ditems, dbias=None if s["bias"] is None else dbias)


def _exact_step(s, i, t):
    wide = lambda name: s[name][i].reshape(-1).double()  # noqa: E731
    g, (b1, b2), shape, eight = wide("grads"), BETAS, s["grads"][i].shape, s["m_scale"] is not None
    m, v = wide("m"), wide("v")
    block = torch.arange(g.numel(), device=DEV) // BLOCK
    if eight:
        m, v = m * s["m_scale"][i].double()[block], (v * s["v_scale"][i].double()[block]) ** 2
    m, v = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g * g
    p = wide("params" if s["masters"] is None else "masters")
    p = (p - LR * DECAY * p - LR * (m / (1 - b1 ** t)) / (torch.sqrt(v / (1 - b2 ** t)) + EPS)).view(shape)
    new = dict(params=p, masters=None if s["masters"] is None else p, m=m.view(shape), v=v.view(shape), m_scale=None, v_scale=None)
    if eight:
        words = _random_words(s["step"] + 1, i, g.numel())
        for name, x, chance in (("m", m, words % 65536), ("v", torch.sqrt(v), words // 65536)):
            scale = torch.zeros(int(block[-1]) + 1, device=DEV, dtype=torch.float64).scatter_reduce_(0, block, x.abs(), "amax")
            scale = 2.0 ** (torch.floor(torch.log2(scale)) - 7)
            q = x.abs() / scale[block]
            codes = torch.arange(127, device=DEV, dtype=torch.uint8).view(torch.float8_e4m3fn).double()   # 0 to 448, rising
            below = torch.searchsorted(codes, q, right=True) - 1
            part = (q - codes[below]) / (codes[below + 1] - codes[below])
            q = codes[below + (part + chance / 65536 >= 1)]
            new[name] = torch.copysign(q, x).view(shape)   # (of the scales: the last bit of a block's largest value may decide, so they have no value in 64 bits)
    return new
