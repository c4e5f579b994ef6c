"""The softmax likelihood of events against the whole catalogue, and its gradients: beside the Poisson likelihood of listed pairs
(cython_loops_float.calc_llk), what a model is evaluated on and trained with that ranks every item for every event.

Logits are scale * <x[n], items[v]> + bias[v]; they are made and used in pieces and never stored.  Results are torch tensors on
the device of `ops`; calls are asynchronous on the current stream, take their scratch memory from torch's allocator and keep
nothing.  They are no part of autograd's graph: results require no gradients, whatever the inputs do, and
softmax_nll_grad gives them.  The definitions, and what happens to rows without a target, masked items and NaN, are in include/hpf_hip.h
(hpf_hip_softmax_nll, hpf_hip_softmax_nll_grad).
"""
import torch

from .ops_hip import TYPE_CODES, changed


def _matrix(t, name, ops, dtype=None, shape=None):
    """Row stride of a matrix whose rows are contiguous."""
    if not isinstance(t, torch.Tensor) or t.dim() != 2:
        raise ValueError("%s must be a matrix" % name)
    if t.dtype not in TYPE_CODES if dtype is None else t.dtype != dtype:
        raise ValueError("%s must be of %s" % (name, " or ".join(str(d) for d in TYPE_CODES) if dtype is None else dtype))
    rows, k = t.shape
    if shape is not None and (rows, k) != shape:
        raise ValueError("%s has shape %s, expected %s" % (name, (rows, k), shape))
    _on(t, name, ops)
    ld, inner = t.stride()
    if inner != 1 and k > 1:
        raise ValueError("%s must have contiguous rows" % name)
    if ld >= k:
        return ld
    if rows > 1:
        raise ValueError("%s must have rows that do not overlap" % name)
    return k


def _vector(t, name, ops, dtype, n):
    if not isinstance(t, torch.Tensor) or t.dtype != dtype or t.dim() != 1 or len(t) != n or not t.is_contiguous():
        raise ValueError("%s must be a contiguous %s vector of %d" % (name, dtype, n))
    _on(t, name, ops)


def _on(t, name, ops):
    if t.device != ops.device:
        raise ValueError("%s is on %s, expected %s" % (name, t.device, ops.device))


def _inputs(ops, x, items, target, bias, scale):
    ldx = _matrix(x, "x", ops)
    n, k = x.shape
    ldi = _matrix(items, "items", ops, x.dtype)
    v = items.shape[0]
    if items.shape[1] != k:
        raise ValueError("items has shape %s, expected (%d, %d)" % (tuple(items.shape), v, k))
    if v == 0 or k == 0:
        raise ValueError("items is empty")
    if max(n, v) >= 2 ** 30 - 32:
        raise ValueError("more than 2^30 - 33 rows")
    if k >= 2 ** 20:
        raise ValueError("rows of 2^20 values or more")
    _vector(target, "target", ops, torch.int64, n)
    if bias is not None:
        _vector(bias, "bias", ops, torch.float32, v)
    if not abs(scale) < 2.0 ** 127:      # (32 bits hold it times log2(e))
        raise ValueError("scale must be a number below 2^127 in size")
    return n, v, k, ldx, ldi


def softmax_nll(ops, x, items, target, bias=None, scale=1.0):
    """(loss, lse) of each event: lse[n] = log sum_v exp(scale <x[n], items[v]> + bias[v]), loss[n] = lse[n] minus the
    target's logit; float32 vectors.

    x       [n, k] float32, bfloat16 or float16, rows contiguous (a stride between them is allowed: `table[:, :k]`)
    items   [v, k] of the same type
    target  int64 [n]; negative: no target, loss 0.  An id of v or more gives a loss of NaN
    bias    float32 [v] or None; -inf (or the type's lowest value) takes an item out, whatever its row holds.  A masked target's
            loss is +inf"""
    n, v, k, ldx, ldi = _inputs(ops, x, items, target, bias, scale)
    loss = torch.empty(n, dtype=torch.float32, device=x.device)
    lse = torch.empty_like(loss)
    if n:
        ops.softmax_nll(x, ldx, items, ldi, target, bias, float(scale), n, v, k, loss, lse)
    return loss, lse


def _span(t):
    if t is None or t.numel() == 0:
        return None
    return t.data_ptr(), t.data_ptr() + (sum((s - 1) * d for s, d in zip(t.shape, t.stride())) + 1) * t.element_size()


def softmax_nll_grad(ops, x, items, target, weight=None, bias=None, scale=1.0, dx=None, ditems=None, dbias=None):
    """(loss, dx, ditems, dbias): softmax_nll's loss of each event, and the gradients of sum_n weight[n] * loss[n] in x, items and
    (None without a bias) bias.  dx and ditems are of x's type; loss and dbias are float32.  Sums are float32 and results are rounded
    once; with 16-bit tables each event's factor in a sum is rounded to their type before (by up to 2^-8 of it in bfloat16, 2^-11
    in float16), as the tables are.

    weight  float32 [n] or None (ones); any sign
    dx, ditems, dbias  tensors to write to (dx and ditems may have a stride between rows; what lies between is left as it is);
                       None: new ones.  They must not overlap an input or each other

    A row without a target, with an id of v or more, or with a masked target takes no part in the gradients."""
    n, v, k, ldx, ldi = _inputs(ops, x, items, target, bias, scale)
    if weight is not None:
        _vector(weight, "weight", ops, torch.float32, n)
    if bias is None and dbias is not None:
        raise ValueError("dbias without a bias")
    given = [t for t in (dx, ditems, dbias) if t is not None]
    if dx is None:
        dx, lddx = torch.empty((n, k), dtype=x.dtype, device=x.device), k
    else:
        lddx = _matrix(dx, "dx", ops, x.dtype, (n, k))
    if ditems is None:
        ditems, lddi = torch.empty((v, k), dtype=x.dtype, device=x.device), k
    else:
        lddi = _matrix(ditems, "ditems", ops, x.dtype, (v, k))
    if dbias is not None:
        _vector(dbias, "dbias", ops, torch.float32, v)
    elif bias is not None:
        dbias = torch.empty(v, dtype=torch.float32, device=x.device)
    if given:
        outs, ins = [[s for s in map(_span, ts) if s] for ts in (given, (x, items, target, bias, weight))]
        for i, (a, b) in enumerate(outs):
            if any(a < d and c < b for c, d in outs[:i] + ins):
                raise ValueError("dx, ditems or dbias overlaps another tensor of the call")
    loss = torch.empty(n, dtype=torch.float32, device=x.device)
    ops.softmax_nll_grad(x, ldx, items, ldi, target, weight, bias, float(scale), n, v, k, loss, dx, lddx, ditems, lddi, dbias)
    if given:
        changed(given)
    return loss, dx, ditems, dbias
