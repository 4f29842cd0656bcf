"""Paged KV cache operators against 64-bit forms (oracle.serving): RoPE + store, decode attention with its account of
weights, eviction; at sizes, lengths, strides and contents where they can go wrong, and their refusals."""

import pytest
import torch

import axiomlm_amd.kernels as K
from oracle import serving

pytestmark = pytest.mark.gpu

WIDTH = {"fp16": lambda hd: hd, "fp8": lambda hd: hd, "int4": lambda hd: hd // 2}


def gen(dev, seed):
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    return g


def make_pages(kv, shape, g, dev, std=1.0):
    """Pages of N(0, std) rows in the pool's format (P, H, page, hd) and their scales, by the framework's packers."""
    x = (torch.randn(*shape, generator=g, device=dev) * std).half()
    if kv == "fp16":
        return x, None
    c, s, _, _ = (K.quantize_kv_fp8 if kv == "fp8" else K.quantize_kv_int4)(x, x)
    return c, s


def make_table(lens, page, g, dev, spare=2, width=None):
    need = [-(-n // page) for n in lens]
    width = width or max(1, max(need))
    order = torch.randperm(sum(need) + spare, generator=g, device=dev).to(torch.int32)
    table = torch.full((len(lens), width), -1, dtype=torch.int32, device=dev)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    return table, sum(need) + spare


def make_case(dev, lens, H, Hkv, hd, kv, page, seed=1):
    g = gen(dev, seed)
    table, P = make_table(lens, page, g, dev)
    k, ks = make_pages(kv, (P, Hkv, page, hd), g, dev)
    v, vs = make_pages(kv, (P, Hkv, page, hd), g, dev)
    q = torch.randn(len(lens), H, hd, generator=g, device=dev).half()
    n = torch.tensor(lens, dtype=torch.int32, device=dev)
    return q, k, v, table, n, ks, vs


def check_decode(q, k, v, table, lens, ks, vs, kv, mass=None, got=None, got_mass=None):
    want, bound, want_mass, mass_bound = serving.decode(q, k, v, table, lens, ks, vs, kv, mass)
    off = (got.cpu().double() - want).abs()
    assert torch.isfinite(got).all()
    assert bool((off <= bound).all()), f"{(off / bound).max().item():.3g} of the bound"
    if mass is not None:
        off = (got_mass.cpu().double() - want_mass).abs()
        assert bool((off <= mass_bound).all()), f"account: {(off / mass_bound).max().item():.3g} of the bound"


# ---- attention ------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("kv", ["fp16", "fp8", "int4"])
@pytest.mark.parametrize("H,Hkv,hd", [(4, 4, 64), (8, 2, 128), (8, 1, 64), (6, 2, 128), (20, 1, 128), (33, 1, 64),
                                      (128, 2, 64)])
def test_ragged_lengths(dev, kv, H, Hkv, hd):
    lens = [1, 0, 7, 16, 17, 129, 300, 33]
    print(f"[paged] {kv} {H}/{Hkv}/{hd}", flush=True)
    q, k, v, table, n, ks, vs = make_case(dev, lens, H, Hkv, hd, kv, 16)
    mass = torch.rand(len(lens), Hkv, table.size(1) * 16, device=dev)
    got_mass = mass.clone()
    got = K.gqa_paged_decode(q, k, v, table, n, ks, vs, kv)
    assert bool((got[1] == 0).all())
    check_decode(q, k, v, table, lens, ks, vs, kv, got=got)
    again = K.gqa_paged_decode(q, k, v, table, n, ks, vs, kv, mass=got_mass)
    check_decode(q, k, v, table, lens, ks, vs, kv, mass, again, got_mass)


@pytest.mark.parametrize("page", [16, 32, 64, 128, 256, 1024])
@pytest.mark.parametrize("kv", ["fp16", "int4"])
def test_page_sizes(dev, kv, page):
    lens = [5, 64, 700, 31]
    q, k, v, table, n, ks, vs = make_case(dev, lens, 8, 2, 64, kv, page, seed=page)
    mass = torch.zeros(len(lens), 2, table.size(1) * page + 3, device=dev)
    got_mass = mass.clone()
    got = K.gqa_paged_decode(q, k, v, table, n, ks, vs, kv, mass=got_mass)
    check_decode(q, k, v, table, lens, ks, vs, kv, mass, got, got_mass)


@pytest.mark.parametrize("kv,lens", [("fp16", [6001]), ("fp8", [9000, 3, 2500]), ("int4", [1, 12345]),
                                     ("fp16", [513] * 40), ("fp8", [130] * 70)])
def test_long_and_many(dev, kv, lens):
    q, k, v, table, n, ks, vs = make_case(dev, lens, 8, 2, 128, kv, 64, seed=3)
    mass = torch.zeros(len(lens), 2, table.size(1) * 64, device=dev)
    got_mass = mass.clone()
    got = K.gqa_paged_decode(q, k, v, table, n, ks, vs, kv, mass=got_mass)
    check_decode(q, k, v, table, lens, ks, vs, kv, mass, got, got_mass)
    # Every row's weights sum to the group's heads.
    total = got_mass.double().sum(-1).cpu()
    assert torch.allclose(total, torch.full_like(total, 4.0), atol=4 * 2.0**-16)


def test_more_sequences_than_a_wave_scans_at_once(dev):
    lens = [(7 * i) % 50 for i in range(300)]
    q, k, v, table, n, ks, vs = make_case(dev, lens, 4, 2, 64, "fp16", 16, seed=4)
    got = K.gqa_paged_decode(q, k, v, table, n, ks, vs)
    check_decode(q, k, v, table, lens, ks, vs, "fp16", got=got)


@pytest.mark.parametrize("kv", ["fp16", "fp8", "int4"])
def test_what_lies_behind_a_sequence_does_not_count(dev, kv):
    """NaN and infinities in the slots behind the last one, in pages of nobody and behind table entries of -1."""
    lens = [1, 40, 0, 130, 16]
    q, k, v, table, n, ks, vs = make_case(dev, lens, 8, 2, 64, kv, 16, seed=5)
    used = torch.zeros(k.size(0), 16, dtype=torch.bool)
    for b, m in enumerate(lens):
        for s in range(m):
            used[int(table[b, s // 16]), s % 16] = True
    idle = ~used.to(dev)[:, None, :, None]
    for t, junk in ((k, float("nan")), (v, float("inf"))) if kv == "fp16" else ((k, 0x7F), (v, 0xFF)):
        t.copy_(torch.where(idle, torch.tensor(junk, dtype=t.dtype, device=dev), t))
    for s in (ks, vs):
        if s is not None:
            s.copy_(torch.where(idle, torch.tensor(float("nan"), dtype=s.dtype, device=dev), s))
    mass = torch.full((5, 2, table.size(1) * 16), 0.5, device=dev)
    got_mass = mass.clone()
    got = K.gqa_paged_decode(q, k, v, table, n, ks, vs, kv, mass=got_mass)
    check_decode(q, k, v, table, lens, ks, vs, kv, mass, got, got_mass)
    for b, m in enumerate(lens):
        assert bool((got_mass[b, :, m:] == 0.5).all())


def test_a_cached_value_that_is_not_finite_is_seen(dev):
    lens = [200, 200]
    q, k, v, table, n, _, _ = make_case(dev, lens, 4, 1, 128, "fp16", 32, seed=6)
    k[int(table[0, 1]), 0, 3, 5] = float("nan")
    got = K.gqa_paged_decode(q, k, v, table, n)
    assert bool(torch.isnan(got[0]).all()) and bool(torch.isfinite(got[1]).all())
    k[int(table[0, 1]), 0, 3, 5] = 1.0
    v[int(table[0, 5]), 0, 7, 9] = float("nan")
    got = K.gqa_paged_decode(q, k, v, table, n)
    assert bool(torch.isnan(got[0, :, 9]).all()) and bool(torch.isfinite(got[1]).all())
    assert bool(torch.isfinite(got[0, :, :9]).all()) and bool(torch.isfinite(got[0, :, 10:]).all())


def test_extreme_scores(dev):
    """Keys of the type's largest values: one key takes all the weight, whichever block it is in."""
    lens = [300, 65]
    q, k, v, table, n, _, _ = make_case(dev, lens, 4, 1, 64, "fp16", 16, seed=7)
    q[0, 0], q[0, 1] = 100.0, -100.0
    k[int(table[0, 17]), 0, 11] = 60000.0
    k[int(table[0, 3]), 0, 1] = -60000.0
    got = K.gqa_paged_decode(q, k, v, table, n)
    assert torch.equal(got[0, 0], v[int(table[0, 17]), 0, 11])
    assert torch.equal(got[0, 1], v[int(table[0, 3]), 0, 1])
    check_decode(q[1:], k, v, table[1:], lens[1:], None, None, "fp16", got=got[1:])


def test_a_page_outside_the_pool_is_left_out(dev):
    lens = [100]
    q, k, v, table, n, _, _ = make_case(dev, lens, 4, 2, 64, "fp16", 16, seed=8)
    for bad in (-7, k.size(0), 2**31 - 1):
        broken = table.clone()
        broken[0, 2] = bad
        mass = torch.zeros(1, 2, table.size(1) * 16, device=dev)
        got = K.gqa_paged_decode(q, k, v, broken, n, mass=mass)
        short = torch.cat([table[:, :2], table[:, 3:]], 1).contiguous()
        want, bound, _, _ = serving.decode(q, k, v, short, [84])
        assert bool(((got.cpu().double() - want).abs() <= bound).all())
        assert bool((mass[..., 32:48] == 0).all())


def test_lengths_past_the_table_are_held_to_it(dev):
    q, k, v, table, n, _, _ = make_case(dev, [64, 48], 4, 2, 64, "fp16", 16, seed=9)
    want = K.gqa_paged_decode(q[:1], k, v, table[:1], n[:1])
    got = K.gqa_paged_decode(q, k, v, table, torch.tensor([10**9, -5], dtype=torch.int32, device=dev))
    assert torch.equal(got[0], want[0]) and bool((got[1] == 0).all())
    got = K.gqa_paged_decode(q, k, v, table, torch.tensor([2**32 + 5, -2**32 + 5], device=dev))
    assert torch.equal(got[0], want[0]) and bool((got[1] == 0).all())


def test_shared_pages_and_repeated_rows(dev):
    """Sequences with a common prefix read the same pages."""
    q, k, v, table, n, _, _ = make_case(dev, [90, 90, 90], 8, 2, 128, "fp16", 16, seed=10)
    table[1, :3] = table[0, :3]
    table[2] = table[0]
    q[2] = q[0]
    got = K.gqa_paged_decode(q, k, v, table, n)
    check_decode(q, k, v, table, [90] * 3, None, None, "fp16", got=got)
    assert torch.equal(got[0], got[2])


@pytest.mark.parametrize("kv", ["fp16", "fp8"])
def test_strided_pages_and_queries(dev, kv):
    """One layer's pages inside a pool whose pages hold every layer, and queries inside a qkv tensor."""
    lens, H, Hkv, hd, page = [50, 3, 170], 8, 2, 64, 16
    g = gen(dev, 11)
    table, P = make_table(lens, page, g, dev)
    pool, scales = make_pages(kv, (P, 3, 2, Hkv, page, hd), g, dev)
    k, v = pool[:, 1, 0], pool[:, 1, 1]
    ks, vs = (None, None) if scales is None else (scales[:, 1, 0], scales[:, 1, 1])
    qkv = torch.randn(3, (H + 2 * Hkv) * hd, generator=g, device=dev).half()
    q = qkv[:, :H * hd].view(3, H, hd)
    n = torch.tensor(lens, dtype=torch.int32, device=dev)
    got = K.gqa_paged_decode(q, k, v, table, n, ks, vs, kv)
    dense = K.gqa_paged_decode(q.contiguous(), k.contiguous(), v.contiguous(), table, n,
                               None if ks is None else ks.contiguous(), None if vs is None else vs.contiguous(), kv)
    assert torch.equal(got, dense)
    check_decode(q, k, v, table, lens, ks, vs, kv, got=got)
    assert torch.equal(K.gqa_paged_decode(q.unsqueeze(2), k, v, table, n, ks, vs, kv).squeeze(2), got)
    # Queries that start off a 16-byte boundary, and transposed ones.
    odd = torch.zeros(3 * H * hd + 4, device=dev, dtype=torch.float16)
    odd[4:] = q.reshape(-1)
    assert torch.equal(K.gqa_paged_decode(odd[4:].view(3, H, hd), k, v, table, n, ks, vs, kv), got)
    turned = q.permute(2, 1, 0).contiguous().permute(2, 1, 0)
    assert torch.equal(K.gqa_paged_decode(turned, k, v, table, n, ks, vs, kv), got)


def test_pool_offsets_past_32_bits(dev):
    """Pages more than 4 GiB into the pool."""
    P, Hkv, page, hd = 2400, 8, 1024, 128
    if torch.cuda.get_device_properties(dev).total_memory < 40 << 30:
        pytest.skip("needs 12 GB of GPU memory")
    k = torch.empty(P, Hkv, page, hd, dtype=torch.float16, device=dev)
    v = torch.empty_like(k)
    g = gen(dev, 12)
    pages = [2399, 1, 2200]
    for p in pages:
        k[p] = torch.randn(Hkv, page, hd, generator=g, device=dev).half()
        v[p] = torch.randn(Hkv, page, hd, generator=g, device=dev).half()
    table = torch.tensor([pages], dtype=torch.int32, device=dev)
    n = torch.tensor([2600], dtype=torch.int32, device=dev)
    q = torch.randn(1, 16, hd, generator=g, device=dev).half()
    got = K.gqa_paged_decode(q, k, v, table, n)
    near = torch.stack([k[p] for p in pages]), torch.stack([v[p] for p in pages])
    want = K.gqa_paged_decode(q, *near, torch.tensor([[0, 1, 2]], dtype=torch.int32, device=dev), n)
    assert torch.equal(got, want)
    qkv = torch.randn(1, (16 + 16) * hd, generator=g, device=dev).half()
    fr = torch.randn(4096, hd // 2, 2, generator=g, device=dev)
    K.rope_paged_kv_cache_write(qkv, fr, k, v, table, n - 1, 16 * hd, 8 * hd, hd)
    assert torch.equal(v[2200, :, 2599 - 2048], qkv[0, 24 * hd:].view(8, hd))


def test_matches_the_contiguous_cache(dev):
    """The same rows in a StaticKVCache layout through gqa_flash_decode_mps."""
    for kv in ("fp16", "fp8", "int4"):
        lens = [777]
        q, k, v, table, n, ks, vs = make_case(dev, lens, 32, 8, 128, kv, 64, seed=13)

        def flat(x):
            return None if x is None else x[table[0].long()].transpose(0, 1).flatten(1, 2)[None].contiguous()

        want = K.gqa_flash_decode_mps(q, flat(k), flat(v), 777, 0, flat(ks), flat(vs), kv)
        got = K.gqa_paged_decode(q, k, v, table, n, ks, vs, kv)
        bound = serving.decode(q, k, v, table, lens, ks, vs, kv)[1]
        assert bool(((got.double() - want.double()).abs().cpu() <= 2 * bound).all())


def test_decode_is_reproducible_and_batch_independent(dev):
    lens = [40, 2000, 0, 333, 129]
    q, k, v, table, n, _, _ = make_case(dev, lens, 8, 2, 128, "fp16", 32, seed=14)
    first = K.gqa_paged_decode(q, k, v, table, n)
    for _ in range(5):
        assert torch.equal(K.gqa_paged_decode(q, k, v, table, n), first)


def test_decode_on_another_stream_and_in_graphs(dev):
    """Two captured graphs of two batches and eager calls between their replays, each replay checked."""
    a = make_case(dev, [40, 900, 0, 333], 8, 2, 64, "fp16", 16, seed=15)
    b = make_case(dev, [1500, 2], 16, 2, 128, "fp8", 32, seed=16)
    stream = torch.cuda.Stream(dev)
    graphs, outs, masses = [], [], []
    for (q, k, v, t, n, ks, vs), kv in ((a, "fp16"), (b, "fp8")):
        mass = torch.zeros(q.size(0), k.size(1), t.size(1) * k.size(2), device=dev)
        stream.wait_stream(torch.cuda.current_stream(dev))
        with torch.cuda.stream(stream):
            K.gqa_paged_decode(q, k, v, t, n, ks, vs, kv, mass=mass)
        torch.cuda.current_stream(dev).wait_stream(stream)
        torch.cuda.synchronize()
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            out = K.gqa_paged_decode(q, k, v, t, n, ks, vs, kv, mass=mass)
        graphs.append(gr)
        outs.append(out)
        masses.append(mass)
    for step in range(4):
        for (q, k, v, t, n, ks, vs), kv, gr, out, mass in zip((a, b), ("fp16", "fp8"), graphs, outs, masses):
            q.copy_(torch.randn(q.shape, device=dev).half())
            n.copy_((n + 1).clamp(max=t.size(1) * k.size(2)) if step % 2 else (n - 1).clamp(min=0))
            # Lengths may grow by one past a page that the table has: keep to owned slots.
            owned = (t >= 0).sum(1).int() * k.size(2)
            n.copy_(torch.minimum(n, owned))
            mass.zero_()
            gr.replay()
            want_mass = torch.zeros_like(mass)
            want = K.gqa_paged_decode(q, k, v, t, n, ks, vs, kv, mass=want_mass)
            torch.cuda.synchronize()
            assert torch.equal(out, want) and torch.equal(mass, want_mass)


def test_decode_refusals(dev):
    q, k, v, table, n, _, _ = make_case(dev, [20, 30], 8, 2, 64, "fp16", 16, seed=17)
    c8, s8 = make_pages("fp8", (3, 2, 16, 64), gen(dev, 1), dev)
    mass = torch.zeros(2, 2, table.size(1) * 16, device=dev)
    bad = [
        (q[:1], k, v, table, n, {}), (q[..., :32], k, v, table, n, {}), (q[:, :7], k, v, table, n, {}),
        (q, k, v[:-1], table, n, {}), (q, k.float(), v.float(), table, n, {}), (q, k, v, table.long(), n, {}),
        (q, k, v, table[0], n, {}), (q, k, v, table, n[:1], {}), (q, k, v, table, n.float(), {}),
        (q, k[:, :, :12], v[:, :, :12], table, n, {}), (q, k.transpose(1, 2), v.transpose(1, 2), table, n, {}),
        (q, k, v, table, n, {"kv_dtype": "fp8"}), (q, k, v, table, n, {"kv_dtype": "fp4"}),
        (q, c8, c8, table, n, {"kv_dtype": "fp8"}), (q, c8, c8, table, n, {"kv_dtype": "fp8", "k_scales": s8}),
        (q, c8, c8, table, n, {"kv_dtype": "fp8", "k_scales": s8, "v_scales": s8[:2]}),
        (q, k, v, table, n, {"mass": mass[:, :, :5]}), (q, k, v, table, n, {"mass": mass.double()}),
        (q, k, v, table, n, {"mass": mass[:, :1]}), (q, k, v, table, n.cpu(), {}), (q, k, v, table.cpu(), n, {}),
    ]
    for args in bad:
        with pytest.raises((ValueError, RuntimeError)):
            K.gqa_paged_decode(*args[:5], **args[5])
    k12 = torch.zeros(4, 2, 24, 64, device=dev, dtype=torch.float16)
    with pytest.raises(RuntimeError, match="power of two"):
        K.gqa_paged_decode(q, k12, k12, table, n)
    k96 = torch.zeros(4, 2, 16, 96, device=dev, dtype=torch.float16)
    with pytest.raises(RuntimeError, match="head_dim"):
        K.gqa_paged_decode(torch.zeros(2, 8, 96, device=dev).half(), k96, k96, table, n)
    with pytest.raises(RuntimeError):
        K.gqa_paged_decode(q.cpu(), k, v, table, n)
    assert K.gqa_paged_decode(q[:0], k, v, table[:0], n[:0]).shape == (0, 8, 64)
    assert bool((K.gqa_paged_decode(q, k, v, table[:, :0], n) == 0).all())


# ---- write ----------------------------------------------------------------------------------------------------------
def check_stored(codes, scales, want, kv):
    """Stored rows (N, width) against 64-bit rows (N, hd): fp16 half a step (and the fp32 products' rounding before it); FP8 /
    INT4 half a step of the code, with the quotient rounded to fp16 before."""
    codes = codes.cpu()
    if kv == "fp16":
        off = (codes.double() - want).abs()
        assert bool((off <= 2.0**-11 * want.abs() + 2.0**-21).all()), off.max()
        return
    g = want.unflatten(-1, (-1, 64))
    sc = scales.cpu().double()
    most = 448.0 if kv == "fp8" else 7.0
    assert bool(((sc - g.abs().amax(-1) / most).abs() <= 2.0**-10 * sc + 2.0**-25).all())
    quot = g / sc[..., None]
    val = serving.code_values(codes, kv).unflatten(-1, (-1, 64))
    step = torch.maximum(2.0**-4 * quot.abs(), torch.tensor(2.0**-10)) if kv == "fp8" else torch.tensor(0.5)
    assert bool(((val - quot).abs() <= step + 2.0**-10 * quot.abs() + 2.0**-12).all())


@pytest.mark.parametrize("kv", ["fp16", "fp8", "int4"])
@pytest.mark.parametrize("H,Hkv,hd,bias", [(4, 4, 64, False), (8, 2, 128, True), (5, 1, 64, True), (3, 3, 128, False)])
def test_write_tokens_of_several_sequences(dev, kv, H, Hkv, hd, bias):
    print(f"[paged write] {kv} {H}/{Hkv}/{hd}", flush=True)
    g = gen(dev, 20)
    page, caps = 16, [70, 40, 16, 100]
    table, P = make_table(caps, page, g, dev)
    k, ks = make_pages(kv, (P, Hkv, page, hd), g, dev)
    v, vs = make_pages(kv, (P, Hkv, page, hd), g, dev)
    # A prompt, single tokens, positions ahead of the slots, padding (slot -1, sequence and slot out of range).
    seq = [0] * 37 + [1, 2, 3, 3] + [1, 9, -1, 2]
    slot = list(range(3, 40)) + [39, 0, 99, 50] + [-1, 3, 4, 400]
    ahead = [0] * 37 + [0, 0, 1000, 500] + [0] * 4
    T = len(seq)
    pos = [max(s, 0) + a for s, a in zip(slot, ahead)]
    qkv = torch.randn(T, (H + 2 * Hkv) * hd, generator=g, device=dev).half()
    b = torch.randn((H + 2 * Hkv) * hd, generator=g, device=dev).half() if bias else None
    freqs = torch.polar(torch.ones(600, hd // 2, device=dev), torch.rand(600, hd // 2, generator=g, device=dev) * 6)
    before = {n: None if t is None else t.clone() for n, t in (("k", k), ("v", v), ("ks", ks), ("vs", vs))}
    rows = qkv.clone()
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    K.rope_paged_kv_cache_write(qkv, freqs, k, v, table, i32(pos), H * hd, Hkv * hd, hd, slots=i32(slot),
                                seq_ids=i32(seq), qkv_bias=b, k_scales=ks, v_scales=vs, kv_dtype=kv)
    real = T - 4
    want = serving.rope_rows(rows.view(T, -1, hd), torch.view_as_real(freqs), i32(pos), H + Hkv, b)
    q = qkv[:real, :H * hd].cpu().double().view(real, H, hd)
    wq = want[:real, :H]
    size = rows[:real, :H * hd].float().abs().view(real, H, hd).amax().item() * 2 + 8
    assert bool(((q - wq).abs() <= 2.0**-11 * wq.abs() + size * 2.0**-22).all())
    assert torch.equal(qkv[:, H * hd:], rows[:, H * hd:])  # keys and values of qkv stay
    assert torch.equal(qkv[real:], rows[real:])            # padding stays
    pages = table.cpu()[torch.tensor(seq[:real]), torch.tensor(slot[:real]) // page].long()
    at = torch.tensor(slot[:real]) % page
    touched = torch.zeros(P, page, dtype=torch.bool)
    touched[pages, at] = True
    for name, t, sc, w in (("k", k, ks, want[:real, H:H + Hkv]), ("v", v, vs, want[:real, H + Hkv:])):
        check_stored(t.cpu()[pages, :, at].reshape(real * Hkv, -1),
                     None if sc is None else sc.cpu()[pages, :, at].reshape(real * Hkv, -1),
                     w.reshape(real * Hkv, hd), kv)
        rest = ~touched
        assert torch.equal(t.cpu().transpose(1, 2)[rest], before[name].cpu().transpose(1, 2)[rest])
        if sc is not None:
            assert torch.equal(sc.cpu().transpose(1, 2)[rest], before[name + "s"].cpu().transpose(1, 2)[rest])


@pytest.mark.parametrize("kv", ["fp16", "fp8", "int4"])
@pytest.mark.parametrize("hd", [64, 128])
def test_write_stores_what_the_contiguous_cache_stores(dev, kv, hd):
    g = gen(dev, 21)
    H, Hkv, page, T = 4, 2, 16, 40
    table, P = make_table([64], page, g, dev)
    z = lambda *s, dtype=torch.uint8: torch.zeros(*s, dtype=dtype, device=dev)  # noqa: E731
    width = WIDTH[kv](hd)
    dt = torch.float16 if kv == "fp16" else torch.uint8
    k, v = z(P, Hkv, page, width, dtype=dt), z(P, Hkv, page, width, dtype=dt)
    ck, cv = z(1, Hkv, 64, width, dtype=dt), z(1, Hkv, 64, width, dtype=dt)
    ks = vs = cks = cvs = None
    if kv != "fp16":
        ks, vs = (z(P, Hkv, page, hd // 64, dtype=torch.float16) for _ in range(2))
        cks, cvs = (z(1, Hkv, 64, hd // 64, dtype=torch.float16) for _ in range(2))
    qkv = torch.randn(T, (H + 2 * Hkv) * hd, generator=g, device=dev).half()
    other = qkv.clone()
    freqs = torch.polar(torch.ones(50, hd // 2, device=dev), torch.rand(50, hd // 2, generator=g, device=dev) * 6)
    bias = torch.randn((H + 2 * Hkv) * hd, generator=g, device=dev).half()
    pos = torch.arange(7, 7 + T, device=dev)  # int64; wraps the 50 rotations
    K.rope_paged_kv_cache_write(qkv, freqs, k, v, table, pos, H * hd, Hkv * hd, hd,
                                seq_ids=torch.zeros(T, dtype=torch.int32, device=dev), qkv_bias=bias, k_scales=ks,
                                v_scales=vs, kv_dtype=kv)
    K.rope_kv_cache_write_quantized(other, freqs, ck, cv, cks, cvs, H * hd, Hkv * hd, hd, 7, 7, kv, bias)
    assert torch.equal(qkv, other)

    def rows(t):
        return t[table[0].long()].transpose(0, 1).flatten(1, 2)[None]

    assert torch.equal(rows(k), ck) and torch.equal(rows(v), cv)
    if ks is not None:
        assert torch.equal(rows(ks), cks) and torch.equal(rows(vs), cvs)


@pytest.mark.parametrize("kv", ["fp8", "int4"])
def test_write_of_zero_and_tiny_rows_stays_finite(dev, kv):
    hd, page = 128, 16
    table = torch.zeros(1, 1, dtype=torch.int32, device=dev)
    width = WIDTH[kv](hd)
    k, v = (torch.full((1, 1, page, width), 0x7F, dtype=torch.uint8, device=dev) for _ in range(2))
    ks, vs = (torch.full((1, 1, page, 2), 9.0, dtype=torch.float16, device=dev) for _ in range(2))
    sizes = [0.0, 6e-8, 1e-6, 1e-5, 1.2e-4, 3e-4, 60000.0]
    qkv = torch.zeros(len(sizes), 3 * hd, device=dev)
    for i, s in enumerate(sizes):
        qkv[i] = s * torch.linspace(-1, 1, 3 * hd, device=dev)
    qkv = qkv.half()
    fr = torch.zeros(64, hd // 2, 2, device=dev)
    fr[..., 0] = 1
    pos = torch.arange(len(sizes), dtype=torch.int32, device=dev)
    K.rope_paged_kv_cache_write(qkv.clone(), fr, k, v, table, pos, hd, hd, hd, seq_ids=torch.zeros_like(pos), k_scales=ks,
                                v_scales=vs, kv_dtype=kv)
    got = (K.dequantize_kv_fp8 if kv == "fp8" else K.dequantize_kv_int4)(v[0, 0, :len(sizes)], vs[0, 0, :len(sizes)])
    x = qkv[:, 2 * hd:].float()
    assert bool(torch.isfinite(got).all())
    # Off by half a code step of the largest, by a scale's step where it is a subnormal fp16, or, where the scale
    # rounds to zero (a largest value under 448 | 7 times 2^-25), by the value itself.
    m = x.abs().amax(-1, keepdim=True)
    most = 448.0 if kv == "fp8" else 7.0
    assert bool(((got.float() - x).abs() <= m * (2.0**-4 if kv == "fp8" else 1 / 14 + 1e-3) + most * 2.0**-25).all())


def test_write_rows_may_be_strided_and_int64(dev):
    g = gen(dev, 22)
    H, Hkv, hd = 4, 2, 64
    table, P = make_table([32, 32], 16, g, dev)
    pool = torch.zeros(P, 2, Hkv, 16, hd, dtype=torch.float16, device=dev)
    k, v = pool[:, 0], pool[:, 1]
    wide = torch.randn(2, (H + 2 * Hkv) * hd + 10, generator=g, device=dev).half()
    qkv = wide[:, :-10]
    fr = torch.randn(100, hd // 2, 2, generator=g, device=dev)
    rows = wide.clone()
    pos = torch.tensor([4, 31], device=dev)
    K.rope_paged_kv_cache_write(qkv, fr, k, v, table, pos, H * hd, Hkv * hd, hd)
    assert torch.equal(wide[:, -10:], rows[:, -10:])
    for t in range(2):
        s = int(pos[t])
        assert torch.equal(v[int(table[t, s // 16]), :, s % 16], rows[t, (H + Hkv) * hd:(H + 2 * Hkv) * hd].view(Hkv, hd))
    # Slots and sequences that 32 bits would bring back into range are padding.
    was, row = pool.clone(), wide.clone()
    K.rope_paged_kv_cache_write(qkv, fr, k, v, table, pos, H * hd, Hkv * hd, hd, slots=torch.tensor([2**32, 5], device=dev),
                                seq_ids=torch.tensor([0, 2**32 + 1], device=dev))
    assert torch.equal(pool, was) and torch.equal(wide, row)


def test_write_refusals(dev):
    g = gen(dev, 23)
    table, P = make_table([32, 32], 16, g, dev)
    k, _ = make_pages("fp16", (P, 2, 16, 64), g, dev)
    v = k.clone()
    qkv = torch.zeros(2, 8 * 64, device=dev).half()
    fr = torch.zeros(40, 32, 2, device=dev)
    pos = torch.zeros(2, dtype=torch.int32, device=dev)
    good = dict(qkv=qkv, freqs_cis=fr, k_cache=k, v_cache=v, block_table=table, positions=pos, q_dim=256, kv_dim=128,
                head_dim=64)
    K.rope_paged_kv_cache_write(**good)
    for change in (dict(qkv=qkv.float()), dict(qkv=qkv[:, :-2]), dict(qkv=qkv.t()), dict(freqs_cis=fr[:, :16]),
                   dict(positions=pos[:1]), dict(positions=pos.float()), dict(slots=pos[:1]), dict(seq_ids=pos.cpu()),
                   dict(kv_dim=64, q_dim=384), dict(head_dim=128), dict(q_dim=250, qkv=qkv[:, :506]),
                   dict(qkv_bias=torch.zeros(3, device=dev)), dict(kv_dtype="fp8"), dict(freqs_cis=fr[:0]),
                   dict(qkv=torch.zeros(2, 514, device=dev).half()[:, 1:513])):
        with pytest.raises((ValueError, RuntimeError)):
            K.rope_paged_kv_cache_write(**{**good, **change})
    K.rope_paged_kv_cache_write(**{**good, "qkv": qkv[:0], "positions": pos[:0]})


# ---- eviction -------------------------------------------------------------------------------------------------------
def make_cache(dev, kv, L, lens, Hkv, hd, page, seed, width=None):
    g = gen(dev, seed)
    table, P = make_table(lens, page, g, dev, width=width)
    cache, scales = make_pages(kv, (L, 2, P, Hkv, page, hd), g, dev)
    mass = torch.rand(L, len(lens), Hkv, table.size(1) * page, generator=g, device=dev)
    return cache, scales, table, torch.tensor(lens, dtype=torch.int32, device=dev), mass


def check_evict(cache, scales, table, lens, mass, budget, recent):
    was = cache.clone(), None if scales is None else scales.clone(), mass.clone()
    kept, new, out = K.evict_paged_kv(cache, scales, table, lens, mass, budget, recent)
    assert torch.equal(mass, was[2]) or bool(torch.isnan(mass).any())
    assert new.tolist() == [min(n, budget) for n in lens.tolist()]
    L, B, H = mass.shape[:3]
    page = cache.size(4)
    want_c, want_s = was[0].cpu().clone(), None if scales is None else was[1].cpu().clone()
    tab, acc = table.cpu(), mass.cpu()
    for b, n in enumerate(lens.tolist()):
        for l in range(L):
            for h in range(H):
                keep = serving.evict_choice(acc[l, b, h, :n].tolist(), n, budget, recent)
                assert kept[l, b, h].tolist() == keep + [-1] * (budget - len(keep)), (l, b, h)
                got = out[l, b, h].cpu()
                ref = torch.zeros_like(got)
                ref[:len(keep)] = acc[l, b, h, keep]
                assert torch.equal(got.nan_to_num(7), ref.nan_to_num(7))
                for to, frm in enumerate(keep):
                    src, dst = (int(tab[b, frm // page]), frm % page), (int(tab[b, to // page]), to % page)
                    want_c[l, :, dst[0], h, dst[1]] = was[0].cpu()[l, :, src[0], h, src[1]] if to != frm else \
                        want_c[l, :, dst[0], h, dst[1]]
                    if want_s is not None and to != frm:
                        want_s[l, :, dst[0], h, dst[1]] = was[1].cpu()[l, :, src[0], h, src[1]]
    assert torch.equal(cache.cpu(), want_c)
    if scales is not None:
        assert torch.equal(scales.cpu(), want_s)


@pytest.mark.parametrize("kv", ["fp16", "fp8", "int4"])
@pytest.mark.parametrize("hd,page,budget,recent", [(64, 16, 20, 5), (128, 32, 1, 0), (64, 16, 33, 33), (128, 16, 64, 0),
                                                   (64, 64, 1, 1)])
def test_evict(dev, kv, hd, page, budget, recent):
    print(f"[evict] {kv} {hd} {page} {budget}/{recent}", flush=True)
    lens = [90, 0, budget, budget + 1, 17, 1]
    check_evict(*make_cache(dev, kv, 2, lens, 2, hd, page, 30), budget, recent)


@pytest.mark.parametrize("n,budget,recent", [(700, 300, 32), (1500, 1499, 700), (2049, 130, 1)])
def test_evict_long(dev, n, budget, recent):
    check_evict(*make_cache(dev, "fp16", 1, [n, 5], 1, 64, 64, 31), budget, recent)


def test_evict_ties_and_odd_accounts(dev):
    """Equal values, signed zeros, infinities, NaN: the lower slot first, NaN behind every number."""
    cache, scales, table, lens, mass = make_cache(dev, "fp16", 1, [300, 300, 300, 300], 1, 64, 16, 32)
    mass[0, 0] = 1.0
    mass[0, 1] = (torch.arange(304, device=dev) % 3).float()
    mass[0, 2, 0, ::2] = 0.0
    mass[0, 2, 0, 1::2] = -0.0
    mass[0, 3, 0, ::5] = float("nan")
    mass[0, 3, 0, 1::5] = float("inf")
    mass[0, 3, 0, 2::5] = -float("inf")
    mass[0, 3, 0, 3::5] = -1.0
    for budget, recent in ((100, 10), (280, 0), (150, 3)):
        check_evict(cache.clone(), scales, table, lens, mass, budget, recent)


def test_evict_budget_past_the_table(dev):
    cache, scales, table, lens, mass = make_cache(dev, "fp8", 2, [30, 11], 2, 64, 16, 33)
    check_evict(cache, scales, table, lens, mass, 500, 100)


def test_evict_strided_layers_and_account(dev):
    """Layers taken out of a larger cache, an account with room behind the table."""
    cache, scales, table, lens, _ = make_cache(dev, "fp8", 4, [50, 70], 2, 64, 16, 34)
    mass = torch.rand(2, 2, 2, table.size(1) * 16 + 7, device=dev)
    whole = cache.clone()
    check_evict(cache[::2], scales[::2], table, lens, mass, 24, 8)
    assert torch.equal(cache[1::2], whole[1::2])


def test_evict_refusals(dev):
    cache, scales, table, lens, mass = make_cache(dev, "fp8", 2, [50, 70], 2, 64, 16, 35)
    for args in ((cache, None, table, lens, mass, 10, 2), (cache[0], scales, table, lens, mass, 10, 2),
                 (cache, scales, table, lens, mass, 0, 0), (cache, scales, table, lens, mass, 10, 11),
                 (cache, scales, table, lens, mass, 10, -1), (cache, scales, table, lens, mass[..., :30], 10, 2),
                 (cache, scales, table, lens, mass.half(), 10, 2), (cache, scales, table, lens[:1], mass, 10, 2),
                 (cache, scales, table.long(), lens, mass, 10, 2), (cache, scales[:1], table, lens, mass, 10, 2),
                 (cache.cpu(), scales, table, lens, mass, 10, 2)):
        with pytest.raises((ValueError, RuntimeError)):
            K.evict_paged_kv(*args)


# ---- together -------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("kv", ["fp16", "fp8"])
def test_a_run_of_them_together(dev, kv):
    """Three sequences decoded over one layer: write, attend with the account, evict when the longest passes the limit,
    sample from a projection of the output; every step against the 64-bit forms."""
    H, Hkv, hd, page, V = 8, 2, 64, 16, 500
    limit, budget, recent = 48, 32, 8
    g = gen(dev, 40)
    B, width = 3, limit // page + 1
    table = torch.randperm(B * width, generator=g, device=dev).to(torch.int32).view(B, width)
    cache, scales = make_pages(kv, (1, 2, B * width, Hkv, page, hd), g, dev)
    mass = torch.zeros(1, B, Hkv, width * page, device=dev)
    k, v = cache[0, 0], cache[0, 1]
    ks, vs = (None, None) if scales is None else (scales[0, 0], scales[0, 1])
    lens = torch.tensor([40, 0, 21], dtype=torch.int32, device=dev)
    position = lens.clone()
    freqs = torch.polar(torch.ones(500, hd // 2, device=dev), torch.rand(500, hd // 2, generator=g, device=dev) * 6)
    head = torch.randn(H * hd, V, generator=g, device=dev).half()
    evictions = 0
    for step in range(20):
        qkv = torch.randn(B, (H + 2 * Hkv) * hd, generator=g, device=dev).half()
        K.rope_paged_kv_cache_write(qkv, freqs, k, v, table, position, H * hd, Hkv * hd, hd, slots=lens, k_scales=ks,
                                    v_scales=vs, kv_dtype=kv)
        lens = lens + 1
        position = position + 1
        was = mass.clone()
        q = qkv[:, :H * hd].view(B, H, hd)
        out = K.gqa_paged_decode(q, k, v, table, lens, ks, vs, kv, mass=mass[0])
        check_decode(q, k, v, table, lens.tolist(), ks, vs, kv, was[0], out, mass[0])
        logits = out.flatten(1).float() @ head.float()
        u = torch.rand(B, generator=g, device=dev)
        tokens, probs = K.sample_tokens(logits, u, 0.8, 40, 0.9, 0.02, return_probs=True)
        for b in range(B):
            t, p = serving.sample_row(logits[b], float(u[b].double()), float(torch.tensor(0.8)), 40,
                                      float(torch.tensor(0.9)), float(torch.tensor(0.02)))
            assert int(tokens[b]) == t and abs(float(probs[b]) - p) < 1e-6
        if int(lens.max()) >= limit:
            check_evict(cache.clone(), None if scales is None else scales.clone(), table, lens, mass, budget, recent)
            _, lens, mass = K.evict_paged_kv(cache, scales, table, lens, mass, budget, recent)
            evictions += 1
    assert evictions == 1 and lens.tolist() == [44, 20, 41]
