"""The encoder's operators from their definitions in 64 bits, and how far a result may be from them.

A rounding to a type is off by at most half a step, u = eps / 2 relative to the value: 2^-11 for fp16, 2^-8 for bf16, 2^-24 for fp32."""
import math

import torch

HALF = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}  # half the smallest subnormal


def attention_reference(q, k, v, q_start, k_start, q_used=None, k_used=None, window=(-1, -1), scale=None):
    """(out, weight, largest, written) in 64 bits: out like q (NaN where nothing is written); weight = sum p|v| per output; largest
    |score| and largest |v| that a query sees, per query and head."""
    scale = 1 / math.sqrt(q.shape[2]) if scale is None else scale
    Hq, Hkv = q.shape[1], k.shape[1]
    out = torch.full(q.shape, math.nan, dtype=torch.float64, device=q.device)
    weight, zmax, vmax = torch.zeros_like(out), torch.zeros_like(out[..., :1]), torch.zeros_like(out[..., :1])
    for s in range(len(q_start) - 1):
        nq, nk = q_start[s + 1] - q_start[s], k_start[s + 1] - k_start[s]
        if q_used is not None:
            nq = min(nq, max(q_used[s], 0))
        if k_used is not None:
            nk = min(nk, max(k_used[s], 0))
        rows, keys = slice(q_start[s], q_start[s] + nq), slice(k_start[s], k_start[s] + nk)
        place = torch.arange(nq, device=q.device)[:, None] + nk - nq
        j = torch.arange(nk, device=q.device)[None, :]
        seen = torch.ones(nq, nk, dtype=torch.bool, device=q.device)
        if window[0] >= 0:
            seen &= j >= place - window[0]
        if window[1] >= 0:
            seen &= j <= place + window[1]
        for h in range(Hq):
            kk, vv = k[keys, h * Hkv // Hq].double(), v[keys, h * Hkv // Hq].double()
            z = (q[rows, h].double() @ kk.t()) * scale
            z = torch.where(seen, z, -math.inf)
            p = torch.softmax(z, 1) if nk else z
            p = torch.where(seen, p, 0.0)
            p = torch.where(seen.any(1, keepdim=True), p, 0.0)
            if torch.isfinite(vv).all():
                o = p @ vv
            else:  # a key that is not seen has no part, whatever it holds
                o = torch.where(seen[:, :, None], p[:, :, None] * vv[None], 0.0).sum(1)
            out[rows, h] = o
            weight[rows, h] = p.abs() @ vv.abs().nan_to_num(0, 0, 0)
            if nk:
                zmax[rows, h] = torch.where(seen, z.abs(), 0.0).amax(1, keepdim=True)
                vmax[rows, h] = torch.where(seen[:, :, None], vv.abs()[None], 0.0).amax(dim=(1, 2))[:, None] if nq * nk * vv.shape[1] < 1 << 26 else vv.abs().max()
    return out, weight, zmax, vmax


def attention_bound(ref, dtype, keys):
    """How far a result in `dtype` may be from attention_reference's: the result's own rounding; a rounding of every weight p to that
    type on its way into the matrix product (weights are kept at most 2^8 below their row's scale of 1, so that underflow costs at most 2^8 half
    subnormals each); of a score z, fp32 sums and products (relative 2^-22 with head_dim <= 128 terms of like size) and the exponential's
    argument and value, together at most 2^-18 (1 + |z|) of the weight."""
    out, weight, zmax, vmax = ref
    u = HALF[dtype]
    return u * out.abs() + (u + 2.0 ** -18 * (1 + zmax)) * weight * (1 + 2 * u) + keys * 2.0 ** 8 * TINY[dtype] * vmax + TINY[dtype]


def close(got, want, bound):
    """Whether got is want to within bound, NaN and infinities in the same places."""
    got = got.double()
    same = (got == want) | (torch.isnan(got) & torch.isnan(want))
    return bool((same | ((got - want).abs() <= bound)).all())


def starts(lengths, device="cuda"):
    total = [0]
    for n in lengths:
        total.append(total[-1] + n)
    return total, torch.tensor(total, dtype=torch.int32, device=device)


def norm_reference(x, kind, weight=None, bias=None, eps=1e-5, residual=None, residual_scale=1.0):
    """(y, bound): y in 64 bits, and what fp32 arithmetic may be off by: sums of n terms as trees (relative 2^-20 with room), of values up to the row's
    largest |s|, carried through the division by the deviation and the weight."""
    s = x.double()
    if residual is not None:
        s = s + residual_scale * residual.double()
    top = s.abs().amax(1, keepdim=True)
    if residual is not None:
        top = top + (abs(residual_scale) * residual.double().abs()).amax(1, keepdim=True)
    y, factor = s, torch.ones_like(top)
    if kind != "none":
        d = s - s.mean(1, keepdim=True) if kind == "layer" else s
        factor = 1 / torch.sqrt((d * d).mean(1, keepdim=True) + eps)
        y = d * factor
    w = torch.ones(x.shape[1], dtype=torch.float64, device=x.device) if weight is None else weight.double()
    y = y * w
    bound = 2.0 ** -20 * (top * factor * w.abs() + y.abs())
    if bias is not None:
        y = y + bias.double()
        bound = bound + 2.0 ** -22 * (y.abs() + bias.double().abs())
    return y, bound
