"""The AdamW step over many tensors at once: the first-order counterpart of the stochastic natural-gradient steps of
svi.py, for tables that are trained by a gradient (softmax.softmax_nll_grad gives one).

Tensors are plain torch device tensors that the caller keeps; nothing is remembered between calls except what the caller
holds (`adamw_state` makes it).  The gradients' and moments' formulas, and the 8-bit form of the moments, are in
include/hpf_hip.h (hpf_hip_adamw_step).
"""
import bisect
import math
import numbers

import torch

from .ops_hip import TYPE_CODES, changed

#: consecutive values of an 8-bit moment that share a scale (HPF_ADAMW_BLOCK)
BLOCK = 256


def adamw_state(params, state_bits=32):
    """What `adamw_step` keeps for `params` (a list of float32, bfloat16 or float16 tensors), as a dict of its arguments:
    zero moments m and v in 32 or 8 bits (8: float8_e4m3fn values and the float32 scale of every 256 of them; the second
    moment is held as its root), a float32 master of each 16-bit parameter, and the counter `step`."""
    if state_bits not in (32, 8):
        raise ValueError("state_bits must be 32 or 8")
    params = list(params)
    if not params:
        raise ValueError("params is empty")
    moment = torch.float32 if state_bits == 32 else torch.float8_e4m3fn

    def zeros(p):   # (a byte tensor seen as float8: every fill is an ordinary one)
        return torch.zeros(p.shape, dtype=torch.float32 if state_bits == 32 else torch.uint8, device=p.device).view(moment)

    def scales(p):
        return torch.ones(-(-p.numel() // BLOCK), dtype=torch.float32, device=p.device) if state_bits == 8 else None

    masters = [None if p.dtype == torch.float32 else p.detach().to(torch.float32) for p in params]
    return dict(m=[zeros(p) for p in params], v=[zeros(p) for p in params], step=torch.zeros(1, dtype=torch.int64, device=params[0].device),
                masters=masters, m_scale=[scales(p) for p in params], v_scale=[scales(p) for p in params])


def _held(t, name, i, shape, dtypes, device):
    if isinstance(t, torch.Tensor) and t.dtype in dtypes and t.shape == shape and t.device == device and t.is_contiguous():
        return t.data_ptr()
    if not isinstance(t, torch.Tensor) or t.dtype not in dtypes:
        raise ValueError("%s[%d] must be a tensor of %s" % (name, i, " or ".join(str(d) for d in dtypes)))
    if t.shape != shape:
        raise ValueError("%s[%d] has shape %s, expected %s" % (name, i, tuple(t.shape), tuple(shape)))
    if not t.is_contiguous():
        raise ValueError("%s[%d] must be contiguous" % (name, i))
    raise ValueError("%s[%d] is on %s, expected %s" % (name, i, t.device, device))


_PARAM_TYPES = tuple(TYPE_CODES)
_MOMENT_TYPES = (torch.float32, torch.float8_e4m3fn)
_F32 = (torch.float32,)


def adamw_step(ops, params, grads, m, v, step, masters=None, m_scale=None, v_scale=None, lr=1e-3, betas=(0.9, 0.999), eps=1e-8,
               weight_decay=0.01, seed=0):
    """One step of AdamW on `params` (in place, with their moments and masters), on the current stream; asynchronous.

    ops           HipOps; every tensor is on its device
    params        list of contiguous tensors: float32, or bfloat16 / float16 with a float32 entry in `masters`
    grads         list of contiguous tensors of the same shapes; float32, bfloat16 or float16 each
    m, v          moments of the same shapes: float32, or float8_e4m3fn (v as its root) with a float32 tensor of
                  ceil(numel / 256) scales in m_scale and v_scale
    step          int64 tensor of one element: steps taken so far, moved on by one (so a captured call counts its replays)
    lr            float, or a float32 device tensor of one element, read when the step runs
    weight_decay  float, or one float per tensor
    seed          with 8-bit moments: the random bits of their rounding are a function of (seed, step, the tensor's place
                  in the list, index) alone, so that equal calls give equal results

    Tensors of different types may share a call; those of one combination of types share launches.  No two of them may
    overlap.  Empty tensors are allowed.  Parameters may require gradients: the step is no part of their graph, but moves
    their version, so that a backward pass that still needs the old values says so."""
    count = len(params)
    for name, x in (("grads", grads), ("m", m), ("v", v), ("masters", masters), ("m_scale", m_scale), ("v_scale", v_scale)):
        if x is not None and len(x) != count:
            raise ValueError("%s has %d entries for %d params" % (name, len(x), count))
    b1, b2 = (float(b) for b in betas)
    if not (0.0 <= b1 < 1.0 and 0.0 <= b2 < 1.0):
        raise ValueError("betas must be in [0, 1)")
    if not (math.isfinite(eps) and eps >= 0.0):
        raise ValueError("eps must be finite and not negative")
    device = step.device if torch.is_tensor(step) else None
    if device is None or step.dtype != torch.int64 or step.numel() != 1:
        raise ValueError("step must be an int64 tensor of one element")
    if device != ops.device:
        raise ValueError("step is on %s, expected %s" % (device, ops.device))
    if torch.is_tensor(lr):
        if lr.dtype != torch.float32 or lr.numel() != 1 or lr.device != device:
            raise ValueError("lr must be a number or a float32 tensor of one element on %s" % device)
    elif not (math.isfinite(lr) and lr >= 0.0):
        raise ValueError("lr must be finite and not negative")
    one = isinstance(weight_decay, (int, float)) or isinstance(weight_decay, numbers.Real)
    decay = [float(weight_decay)] * count if one else [float(w) for w in weight_decay]
    if len(decay) != count or not all(math.isfinite(w) and w >= 0.0 for w in (decay[:1] if one else decay)):
        raise ValueError("weight_decay must be a finite number that is not negative, or one for each of params")
    groups, written, read = {}, [(step.data_ptr(), 8)], [(lr.data_ptr(), 4, "lr")] if torch.is_tensor(lr) else []
    for i in range(count):
        p = params[i]
        at = _held(p, "params", i, getattr(p, "shape", None), _PARAM_TYPES, device)
        shape, n = p.shape, p.numel()
        g = _held(grads[i], "grads", i, shape, _PARAM_TYPES, device)
        at_m, at_v = _held(m[i], "m", i, shape, _MOMENT_TYPES, device), _held(v[i], "v", i, shape, (m[i].dtype,), device)
        eight = m[i].dtype != torch.float32
        master = masters[i] if masters is not None else None
        if p.dtype == torch.float32:
            if master is not None:
                raise ValueError("masters[%d]: a float32 parameter has none" % i)
            at_w = None
        else:
            at_w = _held(master, "masters", i, shape, _F32, device)
        at_ms = at_vs = None
        if eight:
            scales = (-(-n // BLOCK),)
            at_ms = _held(m_scale[i] if m_scale is not None else None, "m_scale", i, scales, _F32, device)
            at_vs = _held(v_scale[i] if v_scale is not None else None, "v_scale", i, scales, _F32, device)
        elif (m_scale is not None and m_scale[i] is not None) or (v_scale is not None and v_scale[i] is not None):
            raise ValueError("m_scale[%d], v_scale[%d]: 32-bit moments have no scales" % (i, i))
        if n == 0:
            continue
        size, moment = (4 if at_w is None else 2) * n, (1 if eight else 4) * n
        written += [(at, size), (at_m, moment), (at_v, moment)]
        if at_w is not None:
            written.append((at_w, 4 * n))
        if eight:
            written += [(at_ms, 4 * scales[0]), (at_vs, 4 * scales[0])]
        read.append((g, (4 if grads[i].dtype == torch.float32 else 2) * n, "a gradient"))
        groups.setdefault((p.dtype, grads[i].dtype, 8 if eight else 32), []).append((at, g, at_m, at_v, at_w, at_ms, at_vs, n, decay[i], i, 0))
    written.sort()
    if any(a + size > b for (a, size), (b, _) in zip(written, written[1:])):
        raise ValueError("two of the tensors that the step writes overlap")
    for a, size, name in read:
        j = bisect.bisect_left(written, (a + size,))
        if j and written[j - 1][0] + written[j - 1][1] > a:
            raise ValueError("%s overlaps a tensor that the step writes" % name)
    if not groups:
        groups[torch.float32, torch.float32, 32] = []   # nothing to move, yet a step
    last = len(groups) - 1
    for j, ((ptype, gtype, bits), tensors) in enumerate(groups.items()):
        ops.adamw_step(tensors, ptype, gtype, bits, step, j == last, lr, b1, b2, eps, seed)
    changed([*params, *masters] if masters is not None else params)
