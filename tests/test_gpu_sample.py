"""sample_tokens against float64: the same tokens, logprobs within half a step of fp32 (2^-24 of the value;
the quotient inside the logarithm is off by 2^-40 at most)."""
import math

import numpy as np
import pytest
import torch

from oracle import serving as O

pytestmark = pytest.mark.gpu
INF = math.inf


def check(mk, dev, logits, u, **kw):
    on = {k: v.to(dev) if isinstance(v, torch.Tensor) else v for k, v in kw.items()}
    tok, lp = mk.sample_tokens(logits.to(dev), u.to(dev), **on)
    torch.cuda.synchronize()
    want, wlp = O.sample_tokens(logits, u, **{k: v.numpy() if isinstance(v, torch.Tensor) else v for k, v in kw.items()})
    tok, lp = tok.cpu().numpy(), lp.double().cpu().numpy()
    assert np.array_equal(tok, want), [(b, int(tok[b]), int(want[b])) for b in np.flatnonzero(tok != want)[:5]]
    none = want < 0
    assert np.array_equal(lp[none], wlp[none])
    lp, wlp = lp[~none], wlp[~none]
    assert (np.abs(lp - wlp) <= 2.0 ** -24 * np.abs(wlp) + 2.0 ** -36).all()
    return tok


def rows(seed, B, V, std=2.0, peaks=8, dtype=torch.float32):
    g = torch.Generator().manual_seed(seed)
    x = std * torch.randn(B, V, generator=g)
    x += torch.where(torch.rand(B, V, generator=g) < peaks / V, 12 * torch.rand(B, V, generator=g), 0.0)
    return x.to(dtype), torch.rand(B, generator=g)


SETTINGS = [dict(), dict(temperature=0.7, top_k=20, top_p=0.95), dict(top_p=0.5), dict(min_p=0.05), dict(top_k=1),
            dict(temperature=1.6, top_k=300, min_p=0.001), dict(temperature=0.3, top_p=0.9, min_p=0.1, top_k=50),
            dict(temperature=0.0), dict(temperature=5.0, top_p=0.999)]


@pytest.mark.parametrize("V", [1, 2, 63, 1000, 4096, 4097, 50257, 151936])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_sizes_and_settings(mk, dev, V, dtype):
    for i, kw in enumerate(SETTINGS):
        print(f"sample V={V} {dtype} {kw}", flush=True)
        x, u = rows(V + i, 6, V, dtype=dtype)
        check(mk, dev, x, u, **kw)


def test_rows_of_settings(mk, dev):
    B, V = 40, 9001
    g = torch.Generator().manual_seed(1)
    x, u = rows(2, B, V)
    x[torch.rand(B, V, generator=g) < 0.4] = -INF
    t = torch.where(torch.arange(B) % 5 == 0, 0.0, 0.2 + 2 * torch.rand(B, generator=g))
    for it in (torch.int32, torch.int64):
        check(mk, dev, x, u, temperature=t, top_k=torch.randint(0, 60, (B,), generator=g).to(it),
              top_p=torch.rand(B, generator=g) * 1.2, min_p=torch.rand(B, generator=g) * 0.2)


def test_borders_of_equal_logits(mk, dev):
    """Equal logits have exact masses: cuts and random numbers that fall on a border exactly."""
    for V in (4, 4096, 8192, 12288):
        x = torch.zeros(9, V)
        u = torch.tensor([0, 0.25, 0.5, 0.75, 1 - 2.0 ** -24, 0.125, 0.5, 0.5, 0.999])
        for kw in (dict(), dict(top_p=0.5), dict(top_k=3), dict(top_p=0.25, top_k=V // 2), dict(min_p=1.0), dict(top_p=0.0)):
            check(mk, dev, x, u, **kw)


def test_ties_and_orders(mk, dev):
    """Few distinct values (ties across chunks of the vocabulary), falling and rising rows, both zeros."""
    g = torch.Generator().manual_seed(7)
    V = 20000
    few = torch.randint(0, 4, (8, V), generator=g).float() * 0.5 - 3
    ramp = torch.stack([torch.arange(V), -torch.arange(V)]).float().repeat(4, 1) * 1e-3
    zero = torch.where(torch.rand(8, V, generator=g) < 0.5, 0.0, -0.0)
    u = torch.rand(8, generator=g)
    small = (0.03 * torch.randn(8, V, generator=g)).to(torch.bfloat16)      # both signs in one bin
    for x in (few, ramp, zero, few.to(torch.bfloat16), small, small.float()):
        for kw in (dict(), dict(top_k=7777), dict(top_p=0.7), dict(top_k=5001, top_p=0.3), dict(min_p=0.4), dict(temperature=0.05)):
            check(mk, dev, x, u, **kw)


def test_spread_of_magnitudes(mk, dev):
    """Scaled logits hundreds apart, tiny and huge temperatures, adjacent floats."""
    g = torch.Generator().manual_seed(8)
    u = torch.rand(6, generator=g)
    wide = 300 * torch.randn(6, 10000, generator=g)
    near = torch.from_numpy(np.nextafter(np.float32(10), np.float32(11)) * np.ones((6, 10000), np.float32))
    near[:, ::3] = 10.0
    for x in (wide, near, wide * 1e30, wide * 1e-30):
        for kw in (dict(), dict(temperature=1e-6), dict(temperature=1e6, top_k=9999), dict(temperature=30.0, top_p=0.8), dict(min_p=0.3)):
            check(mk, dev, x, u, **kw)


def test_not_finite(mk, dev):
    """-inf and NaN are never chosen, +inf takes all the mass, a row of neither gives -1."""
    x, u = rows(9, 7, 5000)
    x[0] = -INF
    x[1] = float("nan")
    x[2, 4500:] = float("nan")
    x[3, :] = -INF
    x[3, 4321] = -50.0
    x[4, [70, 4200]] = INF
    x[5, ::2] = -INF
    x[6, 5] = -3e38
    for kw in SETTINGS:
        tok = check(mk, dev, x, u, **kw)
        assert tok[0] == -1 and tok[1] == -1 and tok[3] == 4321 and tok[4] in (70, 4200)


def test_infinite_temperature(mk, dev):
    """Tensors of temperatures may hold an infinity: all logits but -inf and NaN weigh the same."""
    x, u = rows(14, 8, 9000)
    x[:, ::3] = -INF
    x[:, 7::5] = float("nan")
    x[1, [4, 8500]] = INF
    for kw in (dict(), dict(top_k=700), dict(top_p=0.3), dict(top_k=9000, top_p=0.9, min_p=0.2)):
        tok, lp = mk.sample_tokens(x.to(dev), u.to(dev), temperature=torch.full((8,), INF, device=dev),
                                   **kw)
        want, wlp = O.sample_tokens(x, u, temperature=2.0 ** 127, **kw)
        assert np.array_equal(tok.cpu().numpy(), want), kw
        assert np.abs(lp.double().cpu().numpy() - wlp).max() <= 2.0 ** -24 * np.abs(wlp).max() + 2.0 ** -36


def test_strides_and_output(mk, dev):
    x, u = rows(10, 5, 3001)
    want, _ = O.sample_tokens(x, u, top_p=0.9)
    wide = torch.zeros(5, 3009, device=dev)
    wide[:, 3:3004] = x.to(dev)                 # rows off 16-byte boundaries
    out = torch.full((7,), -9, dtype=torch.int32, device=dev)
    tok, _ = mk.sample_tokens(wide[:, 3:3004], u.to(dev), top_p=0.9, output=out[1:6])
    assert np.array_equal(out.cpu().numpy(), np.concatenate([[-9], want, [-9]]))
    cols = x.to(dev).t().contiguous().t()       # columns contiguous
    assert np.array_equal(mk.sample_tokens(cols, u.to(dev), top_p=0.9)[0].cpu().numpy(), want)
    one = x[:1].to(dev).expand(5, -1)           # one row of logits, several random numbers
    assert np.array_equal(mk.sample_tokens(one, u.to(dev))[0].cpu().numpy(), O.sample_tokens(x[:1].expand(5, -1), u)[0])
    tok, lp = mk.sample_tokens(x[:0].to(dev), u[:0].to(dev))
    assert tok.numel() == 0 and lp.numel() == 0


def test_largest_vocabulary_and_batch(mk, dev):
    x, u = rows(11, 2, 1 << 20, std=1.0)
    check(mk, dev, x, u)
    check(mk, dev, x, u, top_k=100000, top_p=0.9)
    x, u = rows(12, 3000, 40)
    check(mk, dev, x, u, top_p=0.8)


def test_repeats_streams_and_graph(mk, dev):
    """Equal tokens from run to run, on another stream, and from replays that read new numbers and settings."""
    x, u = rows(13, 16, 151936)
    x, u = x.to(dev), u.to(dev)
    p, t = torch.full((16,), 0.9, device=dev), torch.full((16,), 0.8, device=dev)
    first = mk.sample_tokens(x, u, temperature=t, top_p=p)
    for _ in range(5):
        again = mk.sample_tokens(x, u, temperature=t, top_p=p)
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = mk.sample_tokens(x, u, temperature=t, top_p=p)
    side.synchronize()
    assert torch.equal(first[0], other[0])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        tok, lp = mk.sample_tokens(x, u, temperature=t, top_p=p)
    for i in range(4):
        u.copy_(torch.rand(16, device=dev))
        t.fill_(0.3 * i)
        x.mul_(0.95)
        graph.replay()
        torch.cuda.synchronize()
        want = mk.sample_tokens(x, u, temperature=t, top_p=p)
        assert torch.equal(tok, want[0]) and torch.equal(lp, want[1]), i


def test_distribution(mk, dev):
    """Shares of 200,000 draws against the masses: 5 standard deviations of a binomial."""
    x = torch.tensor([[2.0, 0.5, 1.0, -1.0, 0.0, 1.5]])
    n = 50000
    count = torch.zeros(6, dtype=torch.int64)
    for i in range(4):
        u = torch.rand(n, generator=torch.Generator().manual_seed(i)).to(dev)
        tok, _ = mk.sample_tokens(x.to(dev).expand(n, -1), u, temperature=0.8)
        count += torch.bincount(tok.cpu().long(), minlength=6)
    p = torch.softmax(x[0].double() / 0.8, 0)
    assert ((count / (4 * n) - p).abs() <= 5 * (p * (1 - p) / (4 * n)).sqrt()).all()
