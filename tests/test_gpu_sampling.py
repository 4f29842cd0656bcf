"""sample_tokens against a 64-bit form (oracle.serving.sample_row): types, sizes, settings, ties, masked rows, strides,
graphs, and its refusals."""

import pytest
import torch

import axiomlm_amd.kernels as K
from oracle import serving

pytestmark = pytest.mark.gpu


def f32(x):
    return float(torch.tensor(x, dtype=torch.float32))


def make_logits(dev, rows, V, dtype, seed, std=2.5):
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    z = torch.randn(rows, V, generator=g, device=dev) * std
    return z.to(dtype), torch.rand(rows, generator=g, device=dev)


def check(z, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    tokens, probs = K.sample_tokens(z, u, temperature, top_k, top_p, min_p, return_probs=True)
    assert torch.equal(tokens, K.sample_tokens(z, u, temperature, top_k, top_p, min_p))

    def of(x, i):
        return f32(x[i].item() if isinstance(x, torch.Tensor) else x)

    for i in range(z.size(0)):
        want, p = serving.sample_row(z[i], float(u[i].double()), of(temperature, i), int(of(top_k, i)), of(top_p, i),
                                     of(min_p, i))
        assert int(tokens[i]) == want, (i, int(tokens[i]), want)
        # fp32 of a quotient of sums of weights of 46 bits (39 at the largest vocabularies)
        assert abs(float(probs[i]) - p) <= 2.0**-24 * p + 2.0**-24, (i, float(probs[i]), p)
    return tokens


SETTINGS = [(1.0, 0, 1.0, 0.0), (0.7, 0, 1.0, 0.0), (0.8, 50, 0.95, 0.0), (1.0, 0, 0.9, 0.0), (1.3, 7, 1.0, 0.0),
            (1.0, 1, 1.0, 0.0), (1.2, 0, 1.0, 0.05), (0.6, 1000, 0.5, 0.3), (0.0, 0, 1.0, 0.0), (1.0, 0, 0.0, 0.0),
            (1.0, 0, 1.0, 1.0), (50.0, 0, 0.99, 0.0), (0.01, 0, 0.999, 0.0), (2.0, 300, 0.7, 0.01)]


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V", [1, 2, 63, 64, 1000, 1025, 8191, 32000, 50304])
def test_settings(dev, dtype, V):
    print(f"[sample] {dtype} {V}", flush=True)
    for i, s in enumerate(SETTINGS):
        z, u = make_logits(dev, 3, V, dtype, 10 * V + i)
        check(z, u, s[0], min(s[1], V), s[2], s[3])


@pytest.mark.parametrize("dtype,V", [(torch.float16, 131072), (torch.float16, 131073), (torch.float32, 151001),
                                     (torch.float16, 300007), (torch.bfloat16, 262144)])
def test_large_vocabularies(dev, dtype, V):
    for i, s in enumerate([SETTINGS[0], SETTINGS[2], SETTINGS[3], SETTINGS[6], SETTINGS[7]]):
        z, u = make_logits(dev, 2, V, dtype, V + i)
        check(z, u, *s)


@pytest.mark.parametrize("dtype,V", [(torch.float16, 40960), (torch.float32, 50011), (torch.bfloat16, 65537),
                                     (torch.float16, 131072), (torch.float32, 400003)])
def test_few_rows_of_large_vocabularies_without_top_k(dev, dtype, V):
    """Rows that several workgroups share: every slice with another largest logit, slices of -inf, ties over the slices'
    borders, rows that are left to one workgroup (+inf, huge logits, temperatures near 0, too many ties at the cut)."""
    inf = float("inf")
    for rows, settings in ((1, SETTINGS), (9, SETTINGS[:1] + SETTINGS[3:4] + SETTINGS[6:7] + SETTINGS[10:])):
        z, u = make_logits(dev, rows, V, dtype, V + rows)
        for s in settings:
            check(z, u, s[0], 0, s[2], s[3])
    z, u = make_logits(dev, 12, V, dtype, V)
    z[0] = z[0] + torch.linspace(-9, 9, V, device=dev).to(dtype)
    z[1, : V // 2] = -inf
    z[2, V // 3:] = -inf
    z[3] = -inf
    z[3, V - 1] = -7.0
    z[4] = 0.25
    z[5] = (torch.arange(V, device=dev) % 3).to(dtype)
    z[6, V // 2] = inf
    z[7] = z[7] * 3000
    z[8] = z[8] * 0.001
    z[9] = -inf
    z[10] = z[10] - 300
    z[11, ::7] = float("nan")
    for s in [(1.0, 0.9, 0.0), (0.7, 1.0, 0.0), (1.3, 0.5, 0.02), (1e-3, 0.9, 0.0), (1e-7, 0.99, 0.0), (1e4, 0.3, 0.0),
              (1.0, 0.0, 0.0), (1.0, 1.0, 0.3), (0.0, 0.9, 0.0)]:
        check(z, u, s[0], 0, s[1], s[2])
    check(z, u, torch.tensor([0.9, 0.0, 1.1] * 4, device=dev), V, torch.tensor([0.8, 1.0] * 6, device=dev), 0.01)
    check(z, u, torch.tensor([0.9, 0.0, 1.1] * 4, device=dev), torch.tensor([0, 5] * 6, device=dev),
          torch.tensor([0.8, 1.0] * 6, device=dev), 0.01)


def test_settings_of_every_row(dev):
    rows, V = 40, 5000
    z, u = make_logits(dev, rows, V, torch.float16, 3)
    g = torch.Generator(device=dev)
    g.manual_seed(4)
    r = lambda: torch.rand(rows, generator=g, device=dev)  # noqa: E731
    t = torch.where(r() < 0.2, 0.0, r() + 0.3)
    k = (r() * 200).int() * (r() < 0.7)
    check(z, u, t, k, torch.where(r() < 0.3, 1.0, r()), torch.where(r() < 0.5, 0.0, r() * 0.3))
    check(z, u, t.double(), k.long(), 0.9, r() * 0.1)


def test_more_rows_than_fit_at_once_with_settings_of_their_own(dev):
    rows, V = 300, 41001
    z, u = make_logits(dev, rows, V, torch.float16, 13)
    i = torch.arange(rows, device=dev)
    z[7], z[299] = float("-inf"), float("-inf")
    z[11, 5] = float("inf")
    check(z, u, torch.where(i % 5 == 0, 0.0, 0.6 + (i % 7) / 8.0), (i % 3) * 40, torch.where(i % 4 == 1, 1.0, 0.85), 0.01)
    check(z[:257], u[:257], 0.9, 0, torch.where(i[:257] % 2 == 0, 1.0, 0.7), 0.0)


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_ties(dev, dtype):
    """Equal logits at the borders: the lower index is kept."""
    V = 3000
    for seed, z in enumerate([torch.zeros(4, V), torch.full((4, V), -3.5), (torch.arange(V) % 4).float().repeat(4, 1),
                              (torch.arange(V) % 1000 == 7).float().repeat(4, 1) * 5,
                              torch.randint(-3, 4, (4, V), generator=torch.Generator().manual_seed(1)).float()]):
        z = z.to(dtype).to(dev)
        u = torch.tensor([0.0, 0.3, 0.77, 1 - 2.0**-24], device=dev)
        for s in SETTINGS + [(1.0, 3, 1.0, 0.0), (1.0, 1500, 0.5, 0.0), (1.0, 0, 0.25, 0.0), (1.0, 2999, 1.0, 0.0)]:
            check(z, u, *s)


@pytest.mark.parametrize("k", [63, 64, 65, 100, 128, 129, 255, 256, 257, 500, 1024, 1025, 2047, 2049])
def test_lists_of_all_lengths(dev, k):
    z, u = make_logits(dev, 6, 5003, torch.float32, 14)
    check(z, u, 1.5, k, 0.95, 0.0)
    check((z * 8).round() / 8, u, 2.0, k, 1.0, 0.0)  # ties at the border


def test_top_k_past_32_bits_is_no_filter(dev):
    z, u = make_logits(dev, 3, 500, torch.float16, 12)
    want = K.sample_tokens(z, u)
    assert torch.equal(K.sample_tokens(z, u, top_k=2**32 + 1), want)
    assert torch.equal(K.sample_tokens(z, u, top_k=torch.tensor([2**32 + 1, 2**31, -2**32 + 1], device=dev)), want)


def test_signed_zeros_are_equal(dev):
    z = torch.full((1, 100), -0.0, device=dev)
    z[0, 50:] = 0.0
    for k in (1, 30, 70):
        check(z, torch.tensor([0.999], device=dev), 1.0, k)
    check(z, torch.tensor([0.5], device=dev), 0.0)


def test_masked_rows(dev):
    """-inf and NaN are never taken, the lowest finite value is an ordinary one, +inf is taken alone; a row with nothing
    to take gives -1."""
    inf, nan = float("inf"), float("nan")
    V = 2500
    z, _ = make_logits(dev, 10, V, torch.float16, 5)
    z[0] = -inf
    z[1] = nan
    z[2, :] = -inf
    z[2, 1700] = -65504.0
    z[3, ::2] = -inf
    z[4, ::3] = nan
    z[5, 7] = inf
    z[6, 100:2000:300] = inf
    z[7] = -65504.0
    z[8, 1:] = -inf
    z[9, :-1] = -inf
    for uu in (0.0, 0.5, 0.999):
        u = torch.full((10,), uu, device=dev)
        for s in SETTINGS:
            tokens = check(z, u, *s)
            assert tokens[:2].tolist() == [-1, -1] and tokens[8] == 0 and tokens[9] == V - 1
    z32 = torch.full((1, 50), -3.4e38, device=dev)
    z32[0, 20] = 3.4e38
    assert check(z32, torch.tensor([0.9], device=dev)).item() == 20
    check(z32, torch.tensor([0.9], device=dev), 1e-3, 10, 0.5)
    check(z32, torch.tensor([0.9], device=dev), 1e30, 10, 0.5)


def test_uniform_numbers_at_the_ends(dev):
    z, _ = make_logits(dev, 4, 1000, torch.float32, 6)
    u = torch.tensor([0.0, 2.0**-30, 1 - 2.0**-24, 0.5], device=dev)
    for s in SETTINGS:
        check(z, u, *s)
    top = K.sample_tokens(z, torch.tensor([1.0, 2.0, 1.0, 1.0], device=dev))
    assert bool((top >= 0).all()) and bool((top < 1000).all())


def test_shapes_and_strides(dev):
    z, u = make_logits(dev, 6, 1000, torch.float16, 7)
    want = check(z, u, 0.9, 20, 0.9)
    assert torch.equal(K.sample_tokens(z.view(2, 3, 1000), u.view(2, 3), 0.9, 20, 0.9), want.view(2, 3))
    assert torch.equal(K.sample_tokens(z[0], u[:1], 0.9, 20, 0.9), want[0])
    wide = torch.zeros(6, 1237, device=dev, dtype=torch.float16)
    for at in (0, 1, 8):  # rows of a padded vocabulary, aligned and not
        wide[:, at:at + 1000] = z
        assert torch.equal(K.sample_tokens(wide[:, at:at + 1000], u, 0.9, 20, 0.9), want)
    assert torch.equal(K.sample_tokens(z.t().contiguous().t(), u, 0.9, 20, 0.9), want)
    assert torch.equal(K.sample_tokens(z[::2], u[::2], 0.9, 20, 0.9), want[::2])
    assert K.sample_tokens(z[:0], u[:0]).shape == (0,)
    expanded = z[:1].expand(6, 1000)
    assert torch.equal(K.sample_tokens(expanded, u), K.sample_tokens(expanded.contiguous(), u))


def test_greedy_is_argmax(dev):
    z, u = make_logits(dev, 50, 32000, torch.float16, 8)
    assert torch.equal(K.sample_tokens(z, u, 0.0), K.argmax_last_token(z))
    assert torch.equal(K.sample_tokens(z, u, 1.0, top_k=1), K.argmax_last_token(z))


def test_the_tokens_follow_the_distribution(dev):
    """Uniform numbers on a grid: every token is taken as often as its probability says, to one grid step."""
    z, _ = make_logits(dev, 1, 200, torch.float32, 9, std=1.5)
    n = 1 << 14
    u = (torch.arange(n, device=dev) + 0.5) / n
    tokens = K.sample_tokens(z.expand(n, 200), u, 0.8, 100, 0.95)
    share = torch.bincount(tokens, minlength=200).double().cpu() / n
    w = torch.softmax(z[0].double().cpu() / f32(0.8), -1)
    order = torch.argsort(w, descending=True)[:100]
    w2 = torch.zeros_like(w)
    w2[order] = w[order]
    keep = w2[order].cumsum(0) - w2[order] < f32(0.95) * w2.sum()
    w3 = torch.zeros_like(w)
    w3[order[keep]] = w[order[keep]]
    assert bool(((share - w3 / w3.sum()).abs() <= 1.01 / n).all())


def test_in_a_graph(dev):
    z, u = make_logits(dev, 5, 32000, torch.float16, 10)
    t = torch.full((5,), 0.8, device=dev)
    K.sample_tokens(z, u, t, 50, 0.9)
    torch.cuda.synchronize()
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        out = K.sample_tokens(z, u, t, 50, 0.9)
    for i in range(4):
        z2, u2 = make_logits(dev, 5, 32000, torch.float16, 20 + i)
        z.copy_(z2)
        u.copy_(u2)
        t.fill_(0.5 + 0.2 * i)
        gr.replay()
        assert torch.equal(K.sample_tokens(z, u, t, 50, 0.9), out)
        torch.cuda.synchronize()


def test_refusals(dev):
    z, u = make_logits(dev, 2, 100, torch.float16, 11)
    for args in ((z.double(), u), (z.long(), u), (z, u[:1]), (z, u.double()), (z, u.cpu()), (z[:, :0], u), (z.cpu(), u),
                 (z, u, -1.0), (z, u, float("nan")), (z, u, 1.0, -1), (z, u, 1.0, 0, 1.5), (z, u, 1.0, 0, -0.1),
                 (z, u, 1.0, 5.5), (z, u, 1.0, 0, 1.0, 1.1), (z, u, torch.ones(3, device=dev)), (z, u, torch.ones(2))):
        with pytest.raises((ValueError, RuntimeError)):
            K.sample_tokens(*args)
