"""A batched serving step over a paged KV cache, in 64 bits on the CPU, from the operators' definitions: rows of pages,
RoPE and store, decode attention with the account of weights, eviction, sampling.  Loops over sequences and heads; inputs
are tensors on any device, results are CPU tensors."""

from __future__ import annotations

import math

import torch


def e4m3_values() -> torch.Tensor:
    """The 256 E4M3FN codes' values (NaN at 0x7F and 0xFF)."""
    c = torch.arange(256)
    e, f = (c >> 3) & 15, (c & 7).double()
    v = torch.where(e == 0, f * 2.0**-9, (1 + f / 8) * torch.exp2((e - 7).double()))
    v = torch.where((c & 127) == 127, float("nan"), v)
    return torch.where(c >= 128, -v, v)


def code_values(codes: torch.Tensor, kv: str) -> torch.Tensor:
    """Stored rows (..., width) as the numbers that the codes stand for, (..., hd), before the scale."""
    c = codes.cpu()
    if kv == "fp16":
        return c.double()
    c = c.view(torch.uint8).long()
    if kv == "fp8":
        return e4m3_values()[c]
    n = torch.stack([c & 15, c >> 4], -1).flatten(-2)
    return torch.where(n >= 8, n - 16, n).double()


def row_values(codes: torch.Tensor, scales, kv: str) -> torch.Tensor:
    """Stored rows as the dequantizers give them: code times scale, rounded to fp16 once."""
    v = code_values(codes, kv)
    if kv == "fp16":
        return v
    return (v * scales.cpu().double().repeat_interleave(64, -1)).half().double()


def sequence_rows(pages: torch.Tensor, table_row, n: int, h: int) -> torch.Tensor:
    """Rows of slots 0 .. n - 1 of one sequence and KV head: (n, width)."""
    P, _, page, _ = pages.shape
    got = [pages[int(table_row[s // page]), h, s % page] for s in range(n)]
    return torch.stack(got) if got else pages.new_empty(0, pages.size(-1))


def decode(q, k, v, table, lens, ks=None, vs=None, kv="fp16", mass=None):
    """-> (out, bound, mass, mass_bound): 64-bit attention of q (B, Hq, hd), how far an fp16 result with fp32 sums and
    fp16 weights may be off, and the account with its bound.  Bound: half a step of the fp16 result; half a step of every fp16
    weight; and twice (numerator and sum) the error of a weight from its score, whose products are summed in fp32 in
    some order (hd half steps of the sum of magnitudes) and whose exponential is good to 2^-20."""
    q, k, v, table = q.cpu(), k.cpu(), v.cpu(), table.cpu().tolist()
    ks, vs = (None if x is None else x.cpu() for x in (ks, vs))
    B, Hq, hd = q.shape
    Hkv = k.size(1)
    R = Hq // Hkv
    out, bound = torch.zeros(B, Hq, hd, dtype=torch.float64), torch.zeros(B, Hq, hd, dtype=torch.float64)
    new = None if mass is None else mass.cpu().double().clone()
    new_bound = None if mass is None else torch.zeros_like(new)
    for b in range(B):
        n = int(lens[b])
        if n == 0:
            continue
        for h in range(Hkv):
            def rows(pages, scales):
                c = sequence_rows(pages, table[b], n, h)
                return row_values(c, None if scales is None else sequence_rows(scales, table[b], n, h), kv)

            kr, vr = rows(k, ks), rows(v, vs)
            qr = q[b, h * R:(h + 1) * R].double()
            p = torch.softmax(qr @ kr.T / math.sqrt(hd), -1)
            off = (qr.abs() @ kr.abs().T / math.sqrt(hd)).amax(-1, keepdim=True) * hd * 2.0**-24 + 2.0**-20
            o = p @ vr
            out[b, h * R:(h + 1) * R] = o
            bound[b, h * R:(h + 1) * R] = 2.0**-11 * o.abs() + (2.0**-11 + 2 * off) * (p @ vr.abs()) + 2.0**-25
            if mass is not None:
                new[b, h, :n] += p.sum(0)
                new_bound[b, h, :n] = (p * 2 * off).sum(0) + 2.0**-23 * new[b, h, :n].abs()
    return out, bound, new, new_bound


def rope_rows(rows, freqs, positions, n_rotated: int, bias=None):
    """rows (T, heads, hd) -> 64-bit rows, the first n_rotated heads rotated; the bias joins as fp16 + fp16 -> fp16."""
    x = rows.cpu()
    if bias is not None:
        x = (x.float() + bias.cpu().float().view(x.shape[1:])).half()
    x = x.double()
    f = freqs.cpu().double()
    f = f[positions.cpu().long() % f.size(0)][:, None]
    a, b = x[:, :n_rotated, 0::2], x[:, :n_rotated, 1::2]
    y = x.clone()
    y[:, :n_rotated, 0::2] = a * f[..., 0] - b * f[..., 1]
    y[:, :n_rotated, 1::2] = a * f[..., 1] + b * f[..., 0]
    return y


def evict_choice(account, n: int, budget: int, recent: int):
    """Kept slots, in order, of one sequence and head; account: its n values."""
    if n <= budget:
        return list(range(n))
    old = n - recent
    worth = [-math.inf if math.isnan(a) else a for a in account[:old]]
    nan = [math.isnan(a) for a in account[:old]]
    best = sorted(range(old), key=lambda i: (nan[i], -worth[i], i))[:budget - recent]
    return sorted(best) + list(range(old, n))


def sample_row(z, u: float, temperature: float, top_k: int, top_p: float, min_p: float):
    """-> (token, probability) of one row of logits (64-bit sums)."""
    z = z.cpu().double()
    z = torch.where(torch.isnan(z), -math.inf, z)
    if bool((z == -math.inf).all()):
        return -1, 0.0
    order = torch.argsort(z, descending=True, stable=True)
    order = order[z[order] > -math.inf]
    if temperature <= 0:
        return int(order[0]), 1.0
    top = float(z[order[0]])
    if top == math.inf:
        order = order[z[order] == math.inf]
        w = torch.ones(len(order), dtype=torch.float64)
    else:
        w = torch.exp((z[order] - top) / temperature)
    if top_k > 0:
        order, w = order[:top_k], w[:top_k]
    if top_p < 1:
        stay = w.cumsum(0) - w < top_p * w.sum()
        stay[0] = True
        order, w = order[stay], w[stay]
    stay = w >= min_p
    stay[0] = True
    order, w = order[stay], w[stay]
    order, at = torch.sort(order)
    w = w[at]
    run = w.cumsum(0)
    last = int(torch.nonzero(w > 0)[-1])
    i = min(int((run <= u * float(run[-1])).sum()), last)
    return int(order[i]), float(w[i] / run[-1])
