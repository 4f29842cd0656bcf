"""One step of batched serving over a paged key / value cache: what its operators are asked to do, and how to check it.

``attend``  attention of one new token per sequence over a cache held in pages (ragged lengths, grouped heads, fp16 /
            FP8 / INT4 pages), on request adding every cached key's attention weight to a running account;
``write``   bias-free RoPE of the new tokens' queries and keys, and their keys and values stored into the pages;
``evict``   the cache of every layer cut down to a budget: the latest tokens and those with the largest account stay;
``sample``  the next token of every row by temperature, top-k, top-p and min-p from given uniform numbers.

The plain forms are torch expressions in 32 bits (sampling in 64: its borders are sums over the vocabulary).
"""

from __future__ import annotations

import math
import random

import torch

own = False

# (heads, KV heads, head size): the small test model, the 7B shape, the 7B shape with grouped heads, and 32 heads of 64
# on four KV heads.
HEADS = {"c1": (4, 4, 64), "7b": (32, 32, 128), "gqa": (32, 8, 128), "gqa64": (32, 4, 64)}
THETA = 10000.0
E4M3 = torch.float8_e4m3fn


def listed():
    return [
        # One user of the small test model: a few keys, latency is everything.
        {"name": "attend_one", "op": "attend", "shape": "c1", "kv": "fp16", "B": 1, "longest": 100, "page": 16,
         "mass": False},
        # A busy chat server: 48 conversations of very different lengths on a grouped-query model.
        {"name": "attend_chat", "op": "attend", "shape": "gqa", "kv": "fp16", "B": 48, "longest": 4096, "page": 64,
         "mass": False},
        # A few long documents, FP8 pages.
        {"name": "attend_docs_fp8", "op": "attend", "shape": "gqa", "kv": "fp8", "B": 8, "longest": 32768, "page": 128,
         "mass": False},
        # Many short requests on a model with small heads, INT4 pages of 16 tokens.
        {"name": "attend_int4", "op": "attend", "shape": "gqa64", "kv": "int4", "B": 128, "longest": 3001, "page": 16,
         "mass": False},
        # The same step where the server keeps the account that eviction goes by; one KV head per head.
        {"name": "attend_account", "op": "attend", "shape": "7b", "kv": "fp16", "B": 6, "longest": 5003, "page": 32,
         "mass": True},
        # The new token of each of 48 conversations.
        {"name": "write_step", "op": "write", "shape": "gqa", "kv": "fp16", "T": 48, "B": 48, "longest": 4096,
         "page": 64},
        # Prompts of five sequences read at once into FP8 pages.
        {"name": "write_prompts_fp8", "op": "write", "shape": "gqa", "kv": "fp8", "T": 4001, "B": 5, "longest": 4096,
         "page": 16},
        # A single conversation of the small model that reached its limit.
        {"name": "evict_one", "op": "evict", "shape": "c1", "kv": "fp16", "layers": 4, "B": 1, "longest": 300,
         "page": 16, "budget": 128, "recent": 32},
        # A server's cache cut to a quarter: eight sequences, sixteen layers.
        {"name": "evict_server", "op": "evict", "shape": "gqa", "kv": "fp16", "layers": 16, "B": 8, "longest": 4096,
         "page": 64, "budget": 1024, "recent": 256},
        # One user's next token with the usual settings.
        {"name": "sample_one", "op": "sample", "rows": 1, "vocab": 32000, "dtype": "fp16", "filters": "usual"},
        # A batch of a large vocabulary, nucleus sampling.
        {"name": "sample_batch", "op": "sample", "rows": 64, "vocab": 128000, "dtype": "fp16", "filters": "top_p"},
        # Many rows with settings of their own, greedy rows among them, fp32 logits.
        {"name": "sample_mixed", "op": "sample", "rows": 500, "vocab": 50304, "dtype": "fp32", "filters": "mixed"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["attend", "attend", "attend", "write", "evict", "sample", "sample"])
    shape = rng.choice(sorted(HEADS))
    page = rng.choice([16, 32, 64, 128])
    if op == "attend":
        longest = _log(rng, 1, 8192 if shape == "7b" else 32768)
        return {"op": op, "shape": shape, "kv": rng.choice(["fp16", "fp8", "int4"]),
                "B": _log(rng, 1, max(1, min(128, (16384 if shape == "7b" else 65536) // longest))),
                "longest": longest, "page": page, "mass": rng.random() < 0.3}
    if op == "write":
        B = _log(rng, 1, 64)
        T = rng.choice([B, _log(rng, 1, 4000)])
        return {"op": op, "shape": shape, "kv": rng.choice(["fp16", "fp8"]), "T": T, "B": B,
                "longest": max(T, _log(rng, 64, 4096)), "page": page}
    if op == "evict":
        longest = _log(rng, 8, 4096)
        budget = rng.randint(max(1, longest // 8), longest)
        return {"op": op, "shape": shape, "kv": rng.choice(["fp16", "fp8"]), "layers": rng.randint(1, 12),
                "B": rng.randint(1, 6), "longest": longest, "page": page, "budget": budget,
                "recent": rng.randint(0, budget)}
    return {"op": op, "rows": _log(rng, 1, 256), "vocab": _log(rng, 1000, 100000),
            "dtype": rng.choice(["fp16", "fp32"]), "filters": rng.choice(["usual", "top_p", "mixed", "none", "min_p"])}


# ---- sizes ----------------------------------------------------------------------------------------------------------
def _lens(case):
    """Cached tokens of every sequence: the first has the longest, the others are spread below it, one in twelve of a
    larger batch is idle (no token)."""
    rng = random.Random("%s %s %s" % (case["B"], case["longest"], case["page"]))
    n = [case["longest"]]
    for _ in range(case["B"] - 1):
        n.append(0 if case["B"] > 8 and rng.random() < 1 / 12 else _log(rng, max(1, case["longest"] // 16),
                                                                          case["longest"]))
    return n


def _row_bytes(kv, hd):
    return {"fp16": 2 * hd, "fp8": hd + hd // 32, "int4": hd // 2 + hd // 32}[kv]


def _width(kv, hd):
    return hd // 2 if kv == "int4" else hd


# ---- inputs ---------------------------------------------------------------------------------------------------------
class _Rand:
    def __init__(self, seed):
        self.dev = torch.device("cuda", torch.cuda.current_device())
        self.g = torch.Generator(device=self.dev)
        self.g.manual_seed(int(seed))

    def normal(self, *shape, std=1.0):
        return torch.randn(*shape, generator=self.g, device=self.dev) * std

    def uniform(self, *shape):
        return torch.rand(*shape, generator=self.g, device=self.dev)

    def perm(self, n):
        return torch.randperm(n, generator=self.g, device=self.dev)

    def pages(self, kv, shape):
        """Pages (..., hd) of N(0, 1) keys or values, stored as `kv`, and their scales."""
        x = self.normal(*shape).half()
        if kv == "fp16":
            return x, None
        g = x.float().unflatten(-1, (shape[-1] // 64, 64))
        s = (g.abs().amax(-1, keepdim=True) / (448.0 if kv == "fp8" else 7.0)).half()
        c = g / s.float()
        if kv == "fp8":
            return c.flatten(-2).to(E4M3).view(torch.uint8), s[..., 0].contiguous()
        c = c.round().clamp(-8, 7).to(torch.int32).flatten(-2).unflatten(-1, (shape[-1] // 2, 2)) & 15
        return (c[..., 0] | (c[..., 1] << 4)).to(torch.uint8), s[..., 0].contiguous()

    def table(self, lens, page, capacity):
        """Every sequence's pages, scattered over the pool (and two pages of nobody); -1 past its last one."""
        need = [-(-n // page) for n in lens]
        width = -(-capacity // page)
        free = self.perm(sum(need) + 2).to(torch.int32)
        table = torch.full((len(lens), width), -1, dtype=torch.int32, device=self.dev)
        at = 0
        for b, n in enumerate(need):
            table[b, :n] = free[at:at + n]
            at += n
        return table, sum(need) + 2


def prepare(case, seed):
    r = _Rand(seed)
    if case["op"] == "sample":
        return _prepare_sample(case, r)
    H, Hkv, hd = HEADS[case["shape"]]
    kv, page, lens = case["kv"], case["page"], _lens(case)
    st = {"case": case, "lens": torch.tensor(lens, dtype=torch.int32, device=r.dev)}
    if case["op"] == "attend":
        st["table"], P = r.table(lens, page, max(lens))
        st["q"] = r.normal(case["B"], H, hd).half()
        st["k"], st["ks"] = r.pages(kv, (P, Hkv, page, hd))
        st["v"], st["vs"] = r.pages(kv, (P, Hkv, page, hd))
        st["mass"] = None
        if case["mass"]:
            st["mass"] = r.uniform(case["B"], Hkv, st["table"].size(1) * page) ** 4
    elif case["op"] == "write":
        # T new tokens: one each while they last, the rest of them the first sequences' prompts.
        T, B, cap = case["T"], case["B"], case["longest"] + 1
        st["table"], P = r.table([cap] * B, page, cap)
        each = [T // B + (1 if b < T % B else 0) for b in range(B)]
        seq = [b for b in range(B) for _ in range(each[b])]
        start = [min(n, cap - e) for n, e in zip(lens, each)]
        pos = [start[b] + i for b in range(B) for i in range(each[b])]
        st["seq"] = torch.tensor(seq, dtype=torch.int32, device=r.dev)
        st["pos"] = torch.tensor(pos, dtype=torch.int32, device=r.dev)
        st["qkv"] = r.normal(T, (H + 2 * Hkv) * hd).half()
        angle = torch.arange(cap, device=r.dev, dtype=torch.float64)[:, None] * THETA ** (
            -torch.arange(0, hd, 2, device=r.dev, dtype=torch.float64) / hd)
        st["freqs"] = torch.stack([angle.cos(), angle.sin()], -1).float()
        st["k"], st["ks"] = r.pages(kv, (P, Hkv, page, hd))
        st["v"], st["vs"] = r.pages(kv, (P, Hkv, page, hd))
    else:
        L = case["layers"]
        st["table"], P = r.table(lens, page, max(lens))
        st["cache"], st["scales"] = r.pages(kv, (L, 2, P, Hkv, page, hd))
        st["mass"] = r.uniform(L, case["B"], Hkv, st["table"].size(1) * page) ** 4
    return st


def _prepare_sample(case, r):
    """Logits of a language model: N(0, 2.5) with a few likely tokens; settings of one kind, or of every row's own."""
    n, V = case["rows"], case["vocab"]
    z = r.normal(n, V, std=2.5)
    likely = ((r.uniform(n, 1) * V).long() + torch.arange(24, device=r.dev) * (V // 24)) % V
    z.scatter_(1, likely, 6.0 + 3.0 * r.normal(n, 24))
    st = {"case": case, "logits": z.half() if case["dtype"] == "fp16" else z, "u": r.uniform(n)}
    usual = {"usual": (0.8, 50, 0.95, 0.0), "top_p": (1.0, 0, 0.9, 0.0), "none": (0.7, 0, 1.0, 0.0),
             "min_p": (1.2, 0, 1.0, 0.05)}
    if case["filters"] == "mixed":
        t = 0.5 + r.uniform(n)
        st["temperature"] = torch.where(r.uniform(n) < 0.1, torch.zeros_like(t), t)
        st["top_k"] = torch.where(r.uniform(n) < 0.3, 0, (r.uniform(n) ** 3 * 1000).int() + 1).int()
        st["top_p"] = torch.where(r.uniform(n) < 0.3, 1.0, 0.5 + 0.5 * r.uniform(n))
        st["min_p"] = torch.where(r.uniform(n) < 0.5, 0.0, 0.2 * r.uniform(n))
    else:
        st["temperature"], st["top_k"], st["top_p"], st["min_p"] = usual[case["filters"]]
    return st


# ---- one pass -------------------------------------------------------------------------------------------------------
def run(state):
    return {"attend": _attend, "write": _write, "evict": _evict, "sample": _sample}[state["case"]["op"]](state)


def _values(codes, scales, kv):
    """What the stored codes stand for: code times scale as the framework's dequantizers give it, in fp16."""
    if kv == "fp16":
        return codes.float()
    if kv == "fp8":
        c = codes.view(E4M3).float()
    else:
        b = codes.to(torch.int32)
        c = (torch.stack([b & 15, b >> 4], -1).flatten(-2) ^ 8).float() - 8
    return (c.unflatten(-1, (-1, 64)) * scales.float()[..., None]).flatten(-2).half().float()


def _attend(st):
    case = st["case"]
    if own:
        from axiomlm_amd.kernels import gqa_paged_decode

        out = gqa_paged_decode(st["q"], st["k"], st["v"], st["table"], st["lens"], k_scales=st["ks"],
                               v_scales=st["vs"], kv_dtype=case["kv"], mass=st["mass"])
        return {"out": out, "mass": st["mass"]}
    H, Hkv, hd = HEADS[case["shape"]]
    B, kv, t = case["B"], case["kv"], st["table"].clamp(min=0).long()

    def rows(pages, scales):  # (B, pages, Hkv, page, hd) -> (B, Hkv, slots, hd)
        return _values(pages[t], None if scales is None else scales[t], kv).transpose(1, 2).flatten(2, 3)

    k, v = rows(st["k"], st["ks"]), rows(st["v"], st["vs"])
    here = torch.arange(k.size(2), device=k.device) < st["lens"][:, None]
    v = torch.where(here[:, None, :, None], v, 0.0)
    s = torch.matmul(st["q"].float().view(B, Hkv, H // Hkv, hd), k.transpose(2, 3).contiguous()) / math.sqrt(hd)
    s = torch.where(here[:, None, None], s, -math.inf)
    m = s.amax(-1, keepdim=True)
    e = torch.where(here[:, None, None], (s - torch.where(m == -math.inf, 0.0, m)).exp(), 0.0)
    total = e.sum(-1, keepdim=True)
    p = e / torch.where(total == 0, 1.0, total)
    if st["mass"] is not None:
        st["mass"] += p.sum(2)
    return {"out": torch.matmul(p, v).half().view(B, H, hd), "mass": st["mass"]}


def _stored(k, kv):
    return k if kv == "fp16" else k.view(E4M3)


def _write(st):
    case = st["case"]
    H, Hkv, hd = HEADS[case["shape"]]
    kv = case["kv"]
    if own:
        from axiomlm_amd.kernels import rope_paged_kv_cache_write

        rope_paged_kv_cache_write(st["qkv"], st["freqs"], st["k"], st["v"], st["table"], st["pos"], H * hd, Hkv * hd,
                                  hd, seq_ids=st["seq"], k_scales=st["ks"], v_scales=st["vs"], kv_dtype=kv)
    else:
        f = st["freqs"][st["pos"].long()][:, None]  # (T, 1, hd/2, 2)
        x = st["qkv"].float().view(-1, H + 2 * Hkv, hd // 2, 2)
        a, b = x[:, :H + Hkv, :, 0], x[:, :H + Hkv, :, 1]
        c, s = f[..., 0], f[..., 1]
        turned = torch.stack([a * c - b * s, a * s + b * c], -1).flatten(-2).half()
        st["qkv"][:, :H * hd] = turned[:, :H].flatten(1)
        where = st["pos"].long()
        pages, at = st["table"][st["seq"].long(), where // case["page"]].long(), where % case["page"]
        for to, scales, new in ((st["k"], st["ks"], turned[:, H:]),
                                (st["v"], st["vs"], x[:, H + Hkv:].flatten(-2).half())):
            if kv == "fp16":
                to[pages, :, at] = new
                continue
            g = new.float().unflatten(-1, (hd // 64, 64))
            sc = (g.abs().amax(-1, keepdim=True) / 448.0).half()
            scales[pages, :, at] = sc[..., 0]
            to[pages, :, at] = (g / sc.float()).flatten(-2).to(E4M3).view(torch.uint8)
    return {"q": st["qkv"][:, :H * hd], "k": _stored(st["k"], kv), "v": _stored(st["v"], kv), "k_scales": st["ks"],
            "v_scales": st["vs"]}


def _evict(st):
    case = st["case"]
    kv, budget, recent = case["kv"], case["budget"], case["recent"]
    if own:
        from axiomlm_amd.kernels import evict_paged_kv

        kept, lens, mass = evict_paged_kv(st["cache"], st["scales"], st["table"], st["lens"], st["mass"], budget,
                                          recent)
        return {"cache": _stored(st["cache"], kv), "scales": st["scales"], "kept": kept, "lens": lens, "mass": mass}
    L, B, Hkv, C = st["mass"].shape
    dev, page = st["mass"].device, case["page"]
    slot = torch.arange(C, device=dev)
    n = st["lens"].long()[:, None, None]  # (B, 1, 1)
    worth = torch.where(slot >= n - recent, math.inf, st["mass"])
    worth = torch.where(slot < n, worth, -math.inf)
    order = worth.sort(dim=-1, descending=True, stable=True).indices[..., :budget]
    if order.size(-1) < budget:  # a budget past the cache's end
        order = torch.cat([order, order.new_full((L, B, Hkv, budget - order.size(-1)), C)], -1)
    left = n.clamp(max=budget)
    rank = torch.arange(budget, device=dev)
    order = torch.where(rank < left, order, C).sort(-1).values  # (L, B, Hkv, budget): kept slots in order, then C
    kept = torch.where(rank < left, order, -1)
    # Rows that move: those of sequences over the budget.
    l, b, h, to = torch.nonzero((rank < left) & (n > budget) & (kept >= 0), as_tuple=True)
    frm = kept[l, b, h, to]
    t = st["table"].long()
    src, dst = (t[b, frm // page], frm % page), (t[b, to // page], to % page)
    st["cache"][l, :, dst[0], h, dst[1]] = st["cache"][l, :, src[0], h, src[1]]
    if st["scales"] is not None:
        st["scales"][l, :, dst[0], h, dst[1]] = st["scales"][l, :, src[0], h, src[1]]
    padded = torch.cat([st["mass"], st["mass"].new_zeros(L, B, Hkv, 1)], -1)
    mass = torch.zeros_like(st["mass"])
    w = min(budget, C)
    mass[..., :w] = padded.gather(-1, order)[..., :w]
    return {"cache": _stored(st["cache"], kv), "scales": st["scales"], "kept": kept.int(),
            "lens": left[:, 0, 0].int(), "mass": mass}


def _sample(st):
    if own:
        from axiomlm_amd.kernels import sample_tokens

        tokens, probs = sample_tokens(st["logits"], st["u"], st["temperature"], st["top_k"], st["top_p"], st["min_p"],
                                      return_probs=True)
        return {"tokens": tokens, "probs": probs}
    z = st["logits"].double()
    n, V = z.shape

    def column(x):  # settings are held in 32 bits
        x = torch.as_tensor(x, device=z.device)
        return (x.float().double() if x.is_floating_point() else x.long()).expand(n)[:, None]

    temperature, top_k, top_p, min_p = (column(st[k]) for k in ("temperature", "top_k", "top_p", "min_p"))
    greedy = temperature <= 0
    z, index = z.sort(dim=-1, descending=True, stable=True)
    w = ((z - z[:, :1]) / torch.where(greedy, 1.0, temperature)).exp()
    rank = torch.arange(V, device=z.device)
    keep = rank < torch.where(greedy, 1, torch.where(top_k > 0, top_k, V))
    kept = torch.where(keep, w, 0.0)
    keep = keep & ((kept.cumsum(-1) - kept < top_p * kept.sum(-1, keepdim=True)) | (top_p >= 1.0) | (rank == 0))
    keep = keep & (w >= min_p)
    w = torch.zeros_like(w).scatter(-1, index, torch.where(keep, w, 0.0))
    run_sum = w.cumsum(-1)
    total = run_sum[:, -1:]
    last = torch.where(w > 0, rank, 0).amax(-1, keepdim=True)
    token = torch.minimum((run_sum <= st["u"].double()[:, None] * total).sum(-1, keepdim=True), last)
    return {"tokens": token[:, 0], "probs": (w.gather(-1, token) / total).float()[:, 0]}


# ---- work and 64-bit results ----------------------------------------------------------------------------------------
def work(case):
    if case["op"] == "sample":
        n, V = case["rows"], case["vocab"]
        return {"bytes": n * V * (2 if case["dtype"] == "fp16" else 4) + n * 32, "flops": n * V}
    H, Hkv, hd = HEADS[case["shape"]]
    lens, row = _lens(case), _row_bytes(case["kv"], hd)
    if case["op"] == "attend":
        keys = sum(lens)
        return {"bytes": 2 * keys * Hkv * row + 4 * case["B"] * H * hd + (8 * keys * Hkv if case["mass"] else 0) +
                4 * sum(-(-n // case["page"]) for n in lens), "flops": 4 * keys * H * hd}
    if case["op"] == "write":
        T = case["T"]
        return {"bytes": T * ((2 * H + 2 * Hkv) * hd * 2 + 2 * Hkv * row + 4 * hd + 8), "flops": T * 3 * (H + Hkv) * hd}
    L, heads = case["layers"], case["layers"] * Hkv
    moved = sum(case["budget"] for n in lens if n > case["budget"])
    C = -(-max(lens) // case["page"]) * case["page"]
    return {"bytes": heads * (4 * moved * row + 4 * sum(lens) + 4 * case["B"] * (C + case["budget"])),
            "flops": heads * sum(lens)}


def _exact_values(codes, scales, kv):
    """Stored codes in 64 bits, from the formats' definitions."""
    if kv == "fp16":
        return codes.double()
    c = codes.to(torch.int64)
    if kv == "fp8":
        e, f = (c >> 3) & 15, (c & 7).double()
        v = torch.where(e == 0, f * 2.0 ** -9, (1 + f / 8) * torch.exp2((e - 7).double()))
        v = torch.where(c >= 128, -v, v)
    else:
        v = torch.stack([c % 16, c // 16], -1).reshape(*c.shape[:-1], -1).double()
        v = torch.where(v >= 8, v - 16, v)
    return (v * scales.double().repeat_interleave(64, -1)).half().double()


def exact(case, seed):
    st = prepare(case, seed)
    return {"attend": _exact_attend, "write": _exact_write, "evict": _exact_evict,
            "sample": _exact_sample}[case["op"]](case, st)


def _exact_attend(case, st):
    H, Hkv, hd = HEADS[case["shape"]]
    out = torch.zeros(case["B"], H, hd, dtype=torch.float64, device=st["q"].device)
    mass = None if st["mass"] is None else st["mass"].double()
    for b, n in enumerate(_lens(case)):
        if n == 0:
            continue
        pages = st["table"][b, :-(-n // case["page"])].long()
        k, v = (_exact_values(st[x][pages], st[x + "s"][pages] if st[x + "s"] is not None else None, case["kv"])
                .permute(1, 0, 2, 3).reshape(Hkv, -1, hd)[:, :n] for x in ("k", "v"))
        q = st["q"][b].double().view(Hkv, H // Hkv, hd)
        p = torch.softmax((q @ k.transpose(1, 2).contiguous()) * hd ** -0.5, -1)
        out[b] = (p @ v).view(H, hd)
        if mass is not None:
            mass[b, :, :n] += p.sum(1)
    return {"out": out, "mass": mass}


def _exact_write(case, st):
    H, Hkv, hd = HEADS[case["shape"]]
    T = case["T"]
    x = st["qkv"].double().view(T, H + 2 * Hkv, hd)
    z = torch.view_as_complex(x[:, :H + Hkv].reshape(T, H + Hkv, hd // 2, 2).contiguous())
    turn = torch.view_as_complex(st["freqs"].double().contiguous())[st["pos"].long()][:, None]
    turned = torch.view_as_real(z * turn).reshape(T, H + Hkv, hd)
    got = {"q": turned[:, :H].reshape(T, -1)}
    pages = st["table"].long()[st["seq"].long(), st["pos"].long() // case["page"]]
    at = st["pos"].long() % case["page"]
    for name, new in (("k", turned[:, H:]), ("v", x[:, H + Hkv:])):
        if case["kv"] == "fp16":
            to = st[name].double()
            to[pages, :, at] = new
            got[name], got[name + "_scales"] = to, None
            continue
        g = new.half().double().view(T, Hkv, hd // 64, 64)  # what is divided into codes is the fp16 row
        sc = g.abs().amax(-1) / 448
        scales = st[name + "s"].double()
        scales[pages, :, at] = sc
        to = _exact_values(st[name], torch.ones_like(st[name + "s"]), "fp8")
        to[pages, :, at] = (g / sc.half().double()[..., None]).reshape(T, Hkv, hd)
        got[name], got[name + "_scales"] = to, scales
    return got


def _exact_evict(case, st):
    L, B, Hkv, C = st["mass"].shape
    budget, recent, page = case["budget"], case["recent"], case["page"]
    cache = st["cache"].clone()
    scales = None if st["scales"] is None else st["scales"].clone()
    dev = cache.device
    kept = torch.full((L, B, Hkv, budget), -1, dtype=torch.int32)
    mass = torch.zeros(L, B, Hkv, C, dtype=torch.float64)
    account = st["mass"].cpu()
    lens = _lens(case)
    for b, n in enumerate(lens):
        left = min(n, budget)
        old = max(0, n - recent)
        for l in range(L):
            for h in range(Hkv):
                a = account[l, b, h, :n].tolist()
                take = range(n) if n <= budget else sorted(
                    sorted(range(old), key=lambda i: (-a[i], i))[:budget - (n - old)] + list(range(old, n)))
                kept[l, b, h, :left] = torch.tensor(list(take), dtype=torch.int32)
                mass[l, b, h, :left] = torch.tensor([a[i] for i in take], dtype=torch.float64)
        if n <= budget:
            continue
        pages = st["table"][b].long()
        to = torch.arange(left, device=dev)
        for l in range(L):
            for h in range(Hkv):
                frm = kept[l, b, h, :left].to(dev).long()
                for new, was in ((cache, st["cache"]), (scales, st["scales"])):
                    if new is not None:
                        new[l, :, pages[to // page], h, to % page] = was[l, :, pages[frm // page], h, frm % page]
    whole = cache if case["kv"] == "fp16" else cache.view(E4M3)
    return {"cache": whole, "scales": scales, "kept": kept,
            "lens": torch.tensor([min(n, budget) for n in lens], dtype=torch.int32), "mass": mass}


def _exact_sample(case, st):
    n, V = case["rows"], case["vocab"]
    z = st["logits"].double().cpu()
    u = st["u"].double().cpu().tolist()

    def of(name, i):
        x = st[name]
        x = x[i].item() if isinstance(x, torch.Tensor) else x
        return x if isinstance(x, int) else float(torch.tensor(x, dtype=torch.float32))

    tokens, probs = [], []
    for i in range(n):
        t = of("temperature", i)
        order = torch.argsort(z[i], descending=True, stable=True)
        if t <= 0:
            tokens.append(int(order[0]))
            probs.append(1.0)
            continue
        k = of("top_k", i)
        order = order[:k] if k > 0 else order
        w = torch.exp((z[i][order] - z[i][order[0]]) / t)
        p = of("top_p", i)
        if p < 1.0:
            before = torch.cat([torch.zeros(1, dtype=torch.float64), w.cumsum(0)[:-1]])
            stay = before < p * w.sum()
            stay[0] = True
            order, w = order[stay], w[stay]
        stay = w >= of("min_p", i)
        order, w = order[stay], w[stay]
        order, by = torch.sort(order)
        w = w[by]
        c = w.cumsum(0)
        at = min(int((c <= u[i] * c[-1]).sum()), len(w) - 1)
        tokens.append(int(order[at]))
        probs.append(float(w[at] / c[-1]))
    return {"tokens": torch.tensor(tokens), "probs": torch.tensor(probs, dtype=torch.float64)}
