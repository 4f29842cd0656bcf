"""PagedKVCache: page bookkeeping, a decoding loop over two layers against 64-bit forms, eviction and reuse of pages,
replay of a captured step, and the registered operators."""

import pytest
import torch

import axiomlm_amd.kernels as K
from axiomlm_amd.cache import PagedKVCache
from oracle import serving

pytestmark = pytest.mark.gpu


def rotations(n, hd, g, dev):
    return torch.polar(torch.ones(n, hd // 2, device=dev), torch.rand(n, hd // 2, generator=g, device=dev) * 6)


def gen(dev, seed):
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    return g


def test_pages_come_and_go(dev):
    c = PagedKVCache(3, 100, 1, 2, 64, n_pages=9, page_size=16, device=dev)
    assert c.max_seq_len == 112 and c.free_pages == 9
    t = c.begin_step([20, 0, 16])
    assert t.seq_ids.tolist() == [0] * 20 + [2] * 16 and t.slots.tolist() == list(range(20)) + list(range(16))
    assert c.free_pages == 6 and c.seq_lens.tolist() == [20, 0, 16]
    used = c.block_table[c.block_table >= 0].tolist()
    assert len(used) == 3 == len(set(used))
    with pytest.raises(RuntimeError, match="pages"):
        c.begin_step([90, 40, 40])
    with pytest.raises(RuntimeError, match="passes"):
        c.begin_step([93, 0, 0])
    with pytest.raises(ValueError):
        c.begin_step([1, 1])
    assert c.lens == [20, 0, 16] and c.free_pages == 6
    c.begin_step([1, 1, 1])
    assert c.free_pages == 4 and c.block_table[2].tolist()[2:] == [-1] * 5
    c.free(0)
    assert c.free_pages == 6 and c.seq_lens.tolist() == [0, 1, 17] and c.block_table[0].tolist() == [-1] * 7
    c.reset()
    assert c.free_pages == 9 and c.seq_lens.tolist() == [0, 0, 0]
    with pytest.raises(RuntimeError, match="account"):
        c.evict(4, 2)


def test_constructor_refusals(dev):
    for bad in (dict(head_dim=96), dict(page_size=24), dict(page_size=8), dict(cache_dtype="fp4"), dict(n_pages=0),
                dict(n_layer=0)):
        with pytest.raises(ValueError):
            PagedKVCache(**{**dict(max_batch_size=2, max_seq_len=64, n_layer=1, n_kv_head=1, head_dim=64, device=dev),
                            **bad})


@pytest.mark.parametrize("kv", ["fp16", "fp8", "int4"])
def test_decoding_with_eviction(dev, kv):
    """A prompt and then single tokens of three sequences over two layers; one ends and its place is taken by another;
    every attention against the 64-bit form over the rows that the cache holds."""
    H, Hkv, hd, L = 4, 2, 64, 2
    g = gen(dev, 50)
    c = PagedKVCache(3, 96, L, Hkv, hd, n_pages=14, page_size=16, device=dev, cache_dtype=kv, account=True)
    freqs = rotations(400, hd, g, dev)
    counts = [[30, 0, 5], [1, 0, 1], [1, 40, 0], [1, 1, 1], [0, 1, 1], [1, 1, 1], [1, 1, 1], [1, 1, 1]]
    for step, n in enumerate(counts):
        if step == 5:
            c.free(2)
        t = c.begin_step(n)
        last = torch.tensor([max([i for i, s in enumerate(t.seq_ids.tolist()) if s == b], default=-1)
                             for b in range(3)])
        for layer in range(L):
            qkv = torch.randn(sum(n), (H + 2 * Hkv) * hd, generator=g, device=dev).half()
            c.write(layer, qkv, freqs, t, H * hd)
            q = torch.randn(3, H, hd, generator=g, device=dev).half()
            for b in range(3):
                if last[b] >= 0:
                    q[b] = qkv[last[b], :H * hd].view(H, hd)
            was = c.mass[layer].clone()
            out = c.attend(layer, q)
            here = [n_b if new else 0 for n_b, new in zip(c.lens, n)]  # an idle sequence's account stays as it is
            want, bound, mass, mass_bound = serving.decode(q, c.k_caches[layer], c.v_caches[layer], c.block_table,
                                                           here, c.k_scales[layer], c.v_scales[layer], kv, was)
            assert bool(((out.cpu().double() - want).abs() <= bound).all())
            assert bool(((c.mass[layer].cpu().double() - mass).abs() <= mass_bound).all())
        if step in (3, 6):
            lens, mass, table = list(c.lens), c.mass.clone(), c.block_table.cpu().clone()
            rows = {}
            for b in range(3):
                for layer in range(L):
                    for h in range(Hkv):
                        rows[b, layer, h] = serving.sequence_rows(c.k_caches[layer].cpu(), table[b], lens[b], h)
            kept = c.evict(20, 6)
            assert c.lens == [min(n, 20) for n in lens] and c.seq_lens.tolist() == c.lens
            assert c.free_pages == 14 - sum(-(-n // 16) for n in c.lens)
            for (b, layer, h), was in rows.items():
                keep = serving.evict_choice(mass[layer, b, h, :lens[b]].tolist(), lens[b], 20, 6)
                assert kept[layer, b, h, :len(keep)].tolist() == keep
                now = serving.sequence_rows(c.k_caches[layer].cpu(), c.block_table.cpu()[b], c.lens[b], h)
                assert torch.equal(now, was[keep])
    assert c.positions[0] == 30 + 6 and c.positions[2] == 3


def test_a_captured_step_replays(dev):
    """write and attend of one layer captured once; begin_step, pages and an eviction between the replays, each against
    eager calls on a second cache."""
    H, Hkv, hd, B = 8, 2, 64, 2
    g = gen(dev, 51)
    freqs = rotations(300, hd, g, dev)
    caches = [PagedKVCache(B, 200, 1, Hkv, hd, page_size=16, device=dev, account=True) for _ in range(2)]
    qkv = torch.zeros(B, (H + 2 * Hkv) * hd, device=dev, dtype=torch.float16)
    tokens = None
    fixed = None
    graph, out = torch.cuda.CUDAGraph(), None
    for step in range(12):
        new = torch.randn(qkv.shape, generator=g, device=dev).half()
        both = [c.begin_step([1, 1]) for c in caches]
        if fixed is None:
            fixed = type(both[0])(*(t.clone() for t in both[0]))
        for to, t in zip(fixed, both[0]):
            to.copy_(t)
        qkv.copy_(new)
        if step == 1:
            torch.cuda.synchronize()
            with torch.cuda.graph(graph):
                caches[0].write(0, qkv, freqs, fixed, H * hd)
                out = caches[0].attend(0, qkv[:, :H * hd].view(B, H, hd))
        if step == 0:
            caches[0].write(0, qkv, freqs, fixed, H * hd)
            got = caches[0].attend(0, qkv[:, :H * hd].view(B, H, hd))
        else:
            graph.replay()
            got = out
        other = new.clone()
        caches[1].write(0, other, freqs, both[1], H * hd)
        want = caches[1].attend(0, other[:, :H * hd].view(B, H, hd))
        torch.cuda.synchronize()
        assert torch.equal(got, want) and torch.equal(qkv, other)
        assert torch.equal(caches[0].mass, caches[1].mass)
        if step == 8:
            a, b = (c.evict(4, 2) for c in caches)
            assert torch.equal(a, b) and caches[0].lens == [4, 4]


def test_registered_operators(dev):
    from axiomlm_amd import torch_ops  # noqa: F401

    A = torch.ops.axiomlm
    H, Hkv, hd = 4, 2, 64
    g = gen(dev, 52)
    c = PagedKVCache(2, 64, 1, Hkv, hd, page_size=16, device=dev, account=True)
    d = PagedKVCache(2, 64, 1, Hkv, hd, page_size=16, device=dev, account=True)
    t, u = c.begin_step([20, 9]), d.begin_step([20, 9])
    qkv = torch.randn(29, (H + 2 * Hkv) * hd, generator=g, device=dev).half()
    other = qkv.clone()
    freqs = torch.view_as_real(rotations(64, hd, g, dev)).contiguous()
    c.write(0, qkv, freqs, t, H * hd)
    A.rope_paged_kv_cache_write(other, freqs, d.k_caches[0], d.v_caches[0], None, None, d.block_table, u.positions,
                                H * hd, Hkv * hd, hd, u.slots, u.seq_ids)
    assert torch.equal(qkv, other) and torch.equal(c.cache, d.cache)
    q = torch.randn(2, H, hd, generator=g, device=dev).half()
    mass = d.mass[0].clone()
    assert torch.equal(c.attend(0, q), A.gqa_paged_decode(q, d.k_caches[0], d.v_caches[0], d.block_table, d.seq_lens,
                                                          mass=mass))
    d.mass[0].copy_(mass)
    assert torch.equal(c.mass, d.mass)
    kept, lens, new = A.evict_paged_kv(d.cache, None, d.block_table, d.seq_lens, d.mass, 8, 3)
    assert torch.equal(c.evict(8, 3), kept) and torch.equal(c.mass, new) and lens.tolist() == [8, 8]
    z = torch.randn(3, 700, generator=g, device=dev)
    r = torch.rand(3, generator=g, device=dev)
    full = lambda x: torch.full((3,), x, device=dev)  # noqa: E731
    got = A.sample_tokens(z, r, full(0.9), full(20), full(0.8), full(0.0))
    want = K.sample_tokens(z, r, 0.9, 20, 0.8, 0.0, return_probs=True)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
