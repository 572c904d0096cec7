"""The next token of every row of logits, from given random numbers (csrc/kernels/sampling.hip)."""
from __future__ import annotations

import numbers

import torch

from ..framework.tensor import Tensor
from ..ops import _native as N
from .paged import _launch, _u

_MAX_VOCAB, _MAX_ROWS = 1 << 20, 65535


def _setting(v, name, rows, dev, dtype, lo, hi):
    """(tensor or None, number): one value per row, or one for all, checked where the host can see it."""
    if v.__class__ is float or v.__class__ is int:
        number = True
    else:
        v = _u(v)
        number = isinstance(v, numbers.Real)
    if number and lo <= v <= hi and (dtype is not torch.int32 or v == int(v)):
        return None, int(min(v, 2 ** 31 - 1)) if dtype is torch.int32 else float(v)
    if not torch.is_tensor(v):
        raise ValueError(f"sample_tokens: {name} = {v!r} (a number in [{lo}, {hi}] or a tensor of one per row)")
    if v.shape != (rows,) or v.device != dev:
        raise ValueError(f"sample_tokens: {name} {tuple(v.shape)} on {v.device}, expected ({rows},) on {dev}")
    if dtype is torch.int32:
        if v.is_floating_point() or v.dtype is torch.bool:
            raise TypeError(f"sample_tokens: {name} must hold integers")
        if v.dtype is torch.int64:
            v = v.clamp(-1, 2 ** 31 - 1)
    return (v if v.dtype is dtype and v.is_contiguous() else v.detach().to(dtype).contiguous()), 0


def sample_tokens(logits, uniform, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, out=None):
    """Draw one token per row: logits [B, V] (float32, bfloat16, float16) and a random number per row,
    ``uniform`` [B] float32 in [0, 1) -> int64 [B].

    With w_i = exp((x_i - max x) / temperature) and the tokens ordered by logit, equal ones by index:
    ``top_k`` > 0 keeps the first k; ``top_p`` < 1 then keeps the shortest head whose mass reaches top_p of what is left
    (one token at least); ``min_p`` > 0 then keeps w_i >= min_p, that is, tokens at least min_p times as likely as the
    best.  The token is the first, in index order, whose cumulative kept mass exceeds uniform * (kept mass).
    ``temperature`` 0 takes the largest logit, the lowest index among equals.

    Every setting is a number or a tensor of one per row ([B] on the logits' device; a temperature there that is not
    above 0 is greedy, values outside the other ranges act as the nearest bound, NaN as off).  Logits of -inf are never
    drawn, NaN counts as -inf, +inf shares all mass among its like; a row with nothing else gives 0.  A number at or
    above 1 in ``uniform`` draws the last kept token.

    Weights are computed in 64 bits and summed as integers of 2^-min(50, 62 - bits of V) of the largest, so on the GPU the
    token depends on the row, its settings and its number alone: the same in every launch, batch and graph.  A weight is off
    by half of such a unit and 2e-13 of itself, so a number closer to a border than that may fall on its other side than in
    exact arithmetic.  V is at most 1,048,576 on the GPU."""
    wrap = isinstance(logits, Tensor)
    x, u, out = _u(logits), _u(uniform), _u(out)
    shape, dev, dt = x.shape, x.device, x.dtype
    if len(shape) != 2 or shape[1] < 1 or not dt.is_floating_point:
        raise ValueError(f"sample_tokens: logits {tuple(shape)} {dt}")
    B, V = shape
    if u.shape != (B,) or u.dtype is not torch.float32 or u.device != dev:
        raise ValueError(f"sample_tokens: uniform {tuple(u.shape)} {u.dtype} on {u.device}, expected ({B},) float32 on {dev}")
    t = _setting(temperature, "temperature", B, dev, torch.float32, 0.0, 1e30)
    k = _setting(top_k, "top_k", B, dev, torch.int32, -1, 2 ** 63 - 1)
    p = _setting(top_p, "top_p", B, dev, torch.float32, 0.0, 1.0)
    m = _setting(min_p, "min_p", B, dev, torch.float32, 0.0, 1.0)
    if out is None:
        out = torch.empty(B, dtype=torch.int64, device=dev)
    elif out.shape != (B,) or out.dtype is not torch.int64 or out.device != dev or not out.is_contiguous():
        raise ValueError(f"sample_tokens: out {tuple(out.shape)} {out.dtype} on {out.device}")
    if B == 0:
        pass
    elif dev.type == "cuda" and N.use_native(x):
        if dt not in N.DT_CODE or V > _MAX_VOCAB or B > _MAX_ROWS:
            raise ValueError(f"sample_tokens: {B} rows of {dt} logits over {V} tokens (float32, bfloat16 or float16, at most "
                             f"{_MAX_ROWS} rows and {_MAX_VOCAB} tokens)")
        if V > 1 and x.stride(1) != 1:
            x = x.detach().contiguous()
        if not u.is_contiguous():
            u = u.detach().contiguous()
        n = N.native()
        ws = torch.empty(n.sample_workspace(B, V, t[0] is not None, t[1], k[0] is not None, k[1], p[0] is not None, p[1]),
                         dtype=torch.uint8, device=dev)
        _launch(dev, n.sample, N.DT_CODE[dt], x.data_ptr(), x.stride(0), B, V, u.data_ptr(), N.ptr(t[0]), t[1], N.ptr(k[0]),
                k[1], N.ptr(p[0]), p[1], N.ptr(m[0]), m[1], out.data_ptr(), ws.data_ptr())
    else:
        with torch.no_grad():
            out.copy_(_reference(x, u, t, k, p, m))
    return Tensor._wrap(out) if wrap else out


def _reference(x, u, t, k, p, m):
    B, V = x.shape

    def column(s, dtype):
        v = s[0] if s[0] is not None else torch.full((B,), s[1], dtype=dtype, device=x.device)
        return v.to(dtype).double()[:, None]

    t, k, p, m = (column(s, d) for s, d in zip((t, k, p, m), (torch.float32, torch.int32) + (torch.float32,) * 2))
    t, p, m = torch.nan_to_num(t, nan=0.0), torch.nan_to_num(p, nan=1.0), torch.nan_to_num(m, nan=0.0).clamp(max=1.0)
    x = torch.where(torch.isnan(x), float("-inf"), x.double())
    top = x.amax(1, keepdim=True)
    w = torch.exp((x - top) / torch.where(t > 0, t, 1.0))
    w = torch.where(x == top, 1.0, torch.where(torch.isnan(w) | (x == float("-inf")), 0.0, w))
    sx, order = torch.sort(x, dim=1, descending=True, stable=True)
    sw = w.gather(1, order)
    rank = torch.arange(V, device=x.device)[None]
    sw = torch.where((k > 0) & (rank >= k), 0.0, sw)
    before = sw.cumsum(1) - sw
    keep = ((p >= 1) | (before < p * sw.sum(1, keepdim=True)) | (rank == 0)) & (sw >= m)
    kept = torch.zeros_like(w).scatter_(1, order, torch.where(keep, sw, 0.0))
    c = kept.cumsum(1)
    z = c[:, -1:]
    u = torch.nan_to_num(u.double(), nan=0.0).clamp(0.0, 1.0)[:, None]
    token = (c <= u * z).sum(1)
    last = V - 1 - (kept.flip(1) > 0).int().argmax(1)
    token = torch.minimum(token, last)
    return torch.where((t[:, 0] > 0) & (top[:, 0] > float("-inf")), token, x.argmax(1))
