"""Plain 64-bit statements of the serving operators, for the tests (any device)."""
import math

import torch

QMAX = {"e4m3": 448.0, "int8": 127.0}


def attention(q, k, v, scale, bias, shift):
    """q [n, h, d], k / v [m, hk, d] in 64 bits; query i sees keys 0 .. i + shift.  Returns the output
    and the same average of |v| (what the rounding of the weights is relative to).  Keys with weight 0
    contribute nothing, whatever they hold."""
    n, h, d = q.shape
    m, hk, _ = k.shape
    out, size = torch.zeros_like(q), torch.zeros_like(q)
    for a in range(h):
        b = a // (h // hk)
        for i in range(n):
            seen = min(m, i + shift + 1)
            if seen <= 0:
                continue
            s = (k[:seen, b] @ q[i, a]) * scale
            if bias is not None:
                dist = i + shift - torch.arange(seen, device=q.device)
                s = s + bias[a].double()[dist.clamp_max(bias.shape[1] - 1)]
            if bool((s == -math.inf).all()):
                continue
            p = torch.softmax(s, 0)
            live = p != 0
            out[i, a] = p[live] @ v[:seen, b][live]
            size[i, a] = p[live] @ v[:seen, b][live].abs()
    return out, size


def attention_fast(q, k, v, scale, bias, shift):
    """The same for finite inputs, one matrix product per head."""
    n, h, d = q.shape
    m, hk, _ = k.shape
    dist = torch.arange(n, device=q.device)[:, None] + shift - torch.arange(m, device=q.device)
    out, size = torch.zeros_like(q), torch.zeros_like(q)
    for a in range(h):
        b = a // (h // hk)
        s = (q[:, a] @ k[:, b].t()) * scale
        if bias is not None:
            s = s + bias[a].double()[dist.clamp(0, bias.shape[1] - 1)]
        s = s.masked_fill(dist < 0, -math.inf)
        p = torch.nan_to_num(torch.softmax(s, 1), nan=0.0)
        out[:, a], size[:, a] = p @ v[:, b], p @ v[:, b].abs()
    return out, size


def attention_bound(out, size, dtype, weight_dtype=None):
    """Half a step of the output, half a step of the 16-bit weights relative to the averaged |v|, and
    2^-13 of that for the scores: products of 32-bit accuracy whose arguments stay below 2^6 leave less
    than 2^-24 * 2^6 * a few operations on every weight."""
    step = torch.finfo(dtype).eps / 2
    weight = torch.finfo(weight_dtype or dtype).eps / 2
    return step * out.abs() + (weight * (1 + step) + 2.0 ** -13) * size + 2.0 ** -25


def quantise(x, fmt):
    """(values of the codes, fp32 scales) of rows x: the nearest code to x / scale, ties to even."""
    x = x.double()
    amax = x.abs().amax(-1).float()                     # a tensor below: a number's reciprocal would be multiplied
    scale = (amax / torch.full_like(amax, QMAX[fmt])).clamp_min(2.0 ** -126)
    y = x / scale.double()[..., None]
    if fmt == "int8":
        return y.round().clamp(-127, 127), scale
    _, e = torch.frexp(y)
    step = torch.exp2((e - 1).clamp_min(-6).double() - 3)
    return ((y / step).round() * step).clamp(-448, 448), scale


def sample_row(row, t, k, p, least, u):
    """(token, logprob) of one row of logits (64-bit, on the CPU); the settings are Python numbers."""
    row = row.double()
    if bool(row.isnan().any()) or bool((row == math.inf).any()) or bool((row == -math.inf).all()) or not 0 <= t < math.inf:
        return -1, math.nan
    if t == 0:
        return int(torch.nonzero(row == row.max())[0, 0]), 0.0
    order = sorted(range(row.numel()), key=lambda i: (-float(row[i]), i))
    if k > 0:
        order = order[:k]
    w = {i: math.exp((float(row[i]) - float(row[order[0]])) / t) for i in order}
    if p < 1:
        z, before, kept = sum(w.values()), 0.0, []
        for i in order:
            if before < p * z or not kept:
                kept.append(i)
            before += w[i]
        order = kept
    if least > 0:
        order = [i for i in order if w[i] >= min(least, 1.0)]
    total, cum = sum(w[i] for i in order), 0.0
    u = min(max(u, 0.0), 1 - 2.0 ** -53)
    last = None
    for i in sorted(order):
        cum += w[i]
        if w[i] > 0:
            last = i
        if cum > u * total:
            return i, math.log(w[i] / total)
    return last, math.log(w[last] / total)
