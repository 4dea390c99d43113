"""sample against a 64-bit restatement of its definition, on the GPU. Tokens are compared for equality: a row whose
number u, top-p or min-p lies within 1e-9 of a border between two tokens (in units of the mass) would be left to
rounding, and the inputs here have none (checked)."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from autokernel_amd import kernels

pytestmark = pytest.mark.gpu
sample = kernels.get("sample")
DT = [torch.float32, torch.float16, torch.bfloat16]


def oracle(logits, u, T=1.0, k=0, p=1.0, m=0.0):
    """(tokens, distance of each row to the nearest border)"""
    x = logits.double().cpu().numpy()
    R, V = x.shape

    def col(v):
        v = v.cpu().numpy() if torch.is_tensor(v) else v
        return np.broadcast_to(np.asarray(v, np.float32).astype(np.float64), (R,))
    T, p, m, u = col(T), col(p), col(m), np.clip(np.nan_to_num(col(u)), 0.0, 1 - 2.0 ** -24)
    k = np.broadcast_to(k.cpu().numpy() if torch.is_tensor(k) else k, (R,))
    tokens, margin = np.zeros(R, np.int64), np.full(R, np.inf)
    for r in range(R):
        row = x[r]
        order = np.argsort(-row, kind="stable")
        if np.isnan(row).any() or row.max() == -np.inf or not 0 <= T[r] < np.inf or np.isnan(p[r]) or np.isnan(m[r]):
            tokens[r] = -1
            continue
        if T[r] == 0:
            tokens[r] = order[0]
            continue
        s = row[order]
        with np.errstate(invalid="ignore", over="ignore"):
            w = np.where(s == s[0], 1.0, np.exp((s - s[0]) / T[r]))
        if m[r] > 0:
            keep = w >= min(m[r], 1.0)
            margin[r] = min(margin[r], np.abs(w[w < 1] - min(m[r], 1.0)).min(initial=np.inf))
            order, w = order[keep], w[keep]
        if 0 < k[r]:
            order, w = order[:k[r]], w[:k[r]]
        c = np.cumsum(w)
        if p[r] < 1:
            margin[r] = min(margin[r], np.abs(c / c[-1] - p[r])[:-1].min(initial=np.inf)) if len(set(w)) > 1 else margin[r]
            n = max(1, int((np.concatenate([[0.0], c[:-1]]) < p[r] * c[-1]).sum()))
            order, c, w = order[:n], c[:n], w[:n]
        if len(set(w)) > 1:
            margin[r] = min(margin[r], np.abs(c / c[-1] - u[r])[:-1].min(initial=np.inf))
        tokens[r] = order[min(len(c) - 1, int((c <= u[r] * c[-1]).sum()))]
    return tokens, margin


def check(logits, u, what="", **kw):
    print(f"sample {what} {tuple(logits.shape)} {logits.dtype} "
          f"{ {k: v if not torch.is_tensor(v) else 'rows' for k, v in kw.items()} }", flush=True)
    names = {"temperature": "T", "top_k": "k", "top_p": "p", "min_p": "m"}
    want, margin = oracle(logits, u, **{names[k]: v for k, v in kw.items()})
    got = sample(logits, u, **kw).cpu().numpy()
    clear = margin > 1e-9
    assert clear.mean() > 0.99  # the inputs keep off the borders
    assert (got[clear] == want[clear]).all(), (what, np.flatnonzero(got != want)[:5], got[got != want][:5], want[got != want][:5])
    return got


def zipf(R, V, dt, seed, a=1.5):
    g = torch.Generator().manual_seed(seed)
    x = -a * (torch.rand(R, V, generator=g) * V + 1).log() + 0.3 * torch.randn(R, V, generator=g) + 5
    return x.to(dt).cuda(), torch.rand(R, generator=g).cuda()


SETTINGS = [dict(), dict(temperature=0.0), dict(temperature=0.7), dict(top_k=1), dict(top_k=50), dict(top_p=0.9),
            dict(top_p=0.0), dict(min_p=0.05), dict(min_p=1.0), dict(top_k=40, top_p=0.8), dict(top_k=300, top_p=0.95, min_p=0.01),
            dict(temperature=1.7, top_p=0.99), dict(temperature=0.05), dict(temperature=30.0, top_p=0.7),
            dict(top_k=1 << 30), dict(top_p=1e-9), dict(temperature=1e-30), dict(temperature=1e30)]


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("kw", SETTINGS, ids=str)
def test_settings(gpu, dt, kw):
    for R, V, seed in ((7, 5003, 1), (2, 50257, 2)):
        x, u = zipf(R, V, dt, seed)
        check(x, u, "settings", **kw)


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("V", [1, 2, 3, 7, 8, 9, 63, 64, 65, 1000, 1023, 1024, 1025, 4095, 4097, 8191, 8193, 32000, 131072])
def test_widths(gpu, dt, V):
    x, u = zipf(5, V, dt, V)
    check(x, u, "width")
    check(x, u, "width", top_k=20, top_p=0.9)
    check(x, u, "width", top_p=0.97)


@pytest.mark.parametrize("dt", DT)
def test_largest_vocabulary(gpu, dt):
    # (min_p where the margin of 1e-9 is one: around a weight of 1e-6 it spans 0.002 of x, which holds some hundred of a
    # million elements; around 0.02 it spans 1e-7)
    x, u = zipf(3, 1 << 20, dt, 6, a=1.1)
    for kw in (dict(), dict(top_p=0.8), dict(top_k=100), dict(top_k=100000, min_p=0.02), dict(temperature=0.0)):
        check(x, u, "largest", **kw)


@pytest.mark.parametrize("dt", DT)
def test_rows_of_their_own(gpu, dt):
    R = 90
    x, u = zipf(R, 3001, dt, 5)
    g = torch.Generator().manual_seed(6)
    T = torch.where(torch.rand(R, generator=g) < 0.2, torch.zeros(R), 0.3 + torch.rand(R, generator=g)).cuda()
    k = torch.randint(-3, 200, (R,), generator=g).to(torch.int32).cuda()
    p = (torch.rand(R, generator=g) * 1.2).cuda()
    m = (torch.rand(R, generator=g) * 0.3 - 0.1).cuda()
    check(x, u, "per row", temperature=T, top_k=k, top_p=p, min_p=m)
    check(x, u, "per row", temperature=0.8, top_k=k, top_p=0.9, min_p=m)


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("V", [5000, 50257])
def test_flat_rows(gpu, dt, V):
    """Far more elements at a border than a list holds: equal logits, few levels, a narrow range, a wide one."""
    g = torch.Generator().manual_seed(V)
    u = torch.rand(6, generator=g).cuda()
    x = torch.zeros(6, V, dtype=dt)
    x[1] = torch.randint(0, 3, (V,), generator=g).to(dt)
    x[2] = (torch.randn(V, generator=g) * 0.01).to(dt)
    x[3] = (torch.rand(V, generator=g) * 1e-3 + 7).to(dt)
    x[4] = torch.finfo(dt).min          # all masked with the lowest value
    x[5] = (torch.randn(V, generator=g) * 8).to(dt)
    x[0, 17] = -0.0                     # equal to the zeros around it
    for kw in (dict(), dict(top_k=V - 7), dict(top_k=4500, top_p=0.5), dict(top_p=0.999), dict(min_p=0.9, top_p=0.6),
               dict(top_k=4100), dict(temperature=50.0, top_k=4999)):
        check(x.cuda(), u, "flat", **kw)


@pytest.mark.parametrize("dt", DT)
def test_ties_take_the_lowest_index(gpu, dt):
    x = torch.full((4, 300), -2.0, dtype=dt)
    x[:, [250, 40, 7, 199]] = 3.0
    u = torch.tensor([0.0, 0.3, 0.55, 0.999], device="cuda")
    assert sample(x.cuda(), u, temperature=0.0).tolist() == [7] * 4
    assert sample(x.cuda(), u, top_k=2).tolist() == [7, 7, 40, 40]
    assert sample(x.cuda(), u, top_k=4).tolist() == [7, 40, 199, 250]
    assert sample(x.cuda(), u, min_p=0.5).tolist() == [7, 40, 199, 250]
    assert sample(x.cuda(), u, min_p=0.5, top_p=0.5).tolist() == [7, 7, 40, 40]


@pytest.mark.parametrize("dt", DT)
def test_exact_borders_of_equal_weights(gpu, dt):
    """u = j / V on V equal logits is a border that every format holds exactly: the token is j."""
    V = 4096
    u = (torch.arange(0, V, 37) / V).float().cuda()
    x = torch.full((u.numel(), V), 1.5, dtype=dt, device="cuda")
    assert sample(x, u).tolist() == list(range(0, V, 37))
    assert sample(x, u, top_p=0.5).tolist() == [j // 2 for j in range(0, V, 37)]


@pytest.mark.parametrize("dt", DT)
def test_rows_without_a_token(gpu, dt):
    x, u = zipf(10, 777, dt, 3)
    x[0, 5] = float("nan")
    x[1] = float("-inf")
    x[2] = float("-inf")
    x[2, 700] = -3.0                                  # the only one left
    x[3, [9, 4]] = float("inf")                       # share all the weight
    x[4, ::2] = float("-inf")
    x[5, 1:] = torch.finfo(dt).min
    got = check(x, u, "odd rows")
    assert got[0] == -1 and got[1] == -1 and got[2] == 700 and got[3] in (4, 9) and got[4] % 2 == 1 and got[5] == 0
    check(x, u, "odd rows", top_k=5, top_p=0.9, min_p=0.01)
    assert sample(x, u, temperature=0.0).tolist()[:6] == [-1, -1, 700, 4, int(x[4].argmax()), 0]
    one = torch.ones(10, device="cuda")
    for name, bad in (("temperature", (float("nan"), -1.0, float("inf"))), ("top_p", (float("nan"),)),
                      ("min_p", (float("nan"),))):
        for v in bad:
            s = one.clone() * 0.5
            s[7] = v
            got = sample(x, u, **{name: s}).tolist()
            assert got[7] == -1 and got[8] >= 0 and got[6] >= 0


@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("V", [65535, 65536, 65537, 131072, 200001])
def test_long_runs_of_equal_values(gpu, dt, V):
    """Values that fill most of a row, around and past what 16 bits count: a constant, a masked row whose mask is a
    small number, the lowest finite one or -inf, two values in turn, neighbours in falling order."""
    g = torch.Generator().manual_seed(V)
    rows = []
    for fill in (0.0, 2.5, -3.0, torch.finfo(dt).min, -float("inf"), torch.finfo(dt).max):
        row = torch.full((V,), fill)
        rows.append(row.clone())
        at = torch.randperm(V, generator=g)[:300]
        row[at] = torch.randn(300, generator=g) * 2
        rows.append(row)
    rows.append((torch.arange(V) % 2).float())
    rows.append(torch.where(torch.arange(V) < 70000, -0.0, 0.0))
    x = torch.stack(rows).to(dt).cuda()
    u = torch.rand(len(x), generator=g).cuda()
    check(x, u, f"runs of {V}")
    check(x, u, f"runs of {V}", top_p=0.37)
    check(x, u, f"runs of {V}", top_k=1000, min_p=0.01)
    check(x, u, f"runs of {V}", temperature=torch.rand(len(x), generator=g).cuda() * 2 + 0.1, top_k=70000)
    check(x, u, f"runs of {V}", temperature=0.0)


@pytest.mark.parametrize("dt", DT)
def test_signed_zeros_are_equal(gpu, dt):
    x = torch.full((16, 300), -50.0)
    x[:, 40::7] = 0.0
    x[:, 43::14] = -0.0
    x[8:, 5] = -0.0
    n = int((x[0] == 0).sum())
    x, u = x.to(dt).cuda(), ((torch.arange(16) + 0.5) / 16).cuda()
    check(x, u, "zeros")
    check(x, u, "zeros", top_k=n // 2)
    check(x, u, "zeros", top_p=0.31)
    check(x, u, "zeros", temperature=0.0)


def test_numbers_outside_their_range(gpu):
    x, _ = zipf(6, 500, torch.float32, 4)
    u = torch.tensor([-1.0, float("nan"), 1.0, 7.0, float("inf"), -float("inf")], device="cuda")
    same = torch.tensor([0.0, 0.0, 1 - 2.0 ** -24, 1 - 2.0 ** -24, 1 - 2.0 ** -24, 0.0], device="cuda")
    for kw in (dict(), dict(top_k=9), dict(top_p=0.3)):
        assert torch.equal(sample(x, u, **kw), sample(x, same, **kw))


@pytest.mark.parametrize("V", [40, 5000])
def test_settings_outside_their_range(gpu, V):
    """In a tensor, values below the range count as 0 and top_p, min_p above 1 as 1."""
    x, u = zipf(6, V, torch.float32, 5)

    def rows(*v, dtype=torch.float32):
        return torch.tensor(v, dtype=dtype, device="cuda")
    inf = float("inf")
    low, high = rows(-0.5, -1e-30, -3.0, -1e30, -inf, -0.0), rows(1.0, 1.5, 1e30, inf, 2.0, 1.0)
    one, zero = torch.ones_like(u), torch.zeros_like(u)
    assert torch.equal(sample(x, u, top_p=low), sample(x, u, top_k=1))
    assert torch.equal(sample(x, u, top_p=low, top_k=30), sample(x, u, top_k=1))
    assert torch.equal(sample(x, u, top_p=high), sample(x, u, top_p=one))
    assert torch.equal(sample(x, u, min_p=low), sample(x, u, min_p=zero))
    assert torch.equal(sample(x, u, min_p=high), sample(x, u, min_p=one))
    k = rows(-1, -(1 << 31), 0, V, V + 1, (1 << 31) - 1, dtype=torch.int32)
    assert torch.equal(sample(x, u, top_k=k), sample(x, u))


@pytest.mark.parametrize("dt", DT)
def test_strides_and_shapes(gpu, dt):
    x, u = zipf(6, 1003, dt, 8)
    wide = torch.zeros(6, 1100, dtype=dt, device="cuda")
    for shift in (0, 1, 3, 8):
        wide[:, shift:shift + 1003] = x
        check(wide[:, shift:shift + 1003], u, f"shift {shift}", top_k=30)
    want = sample(x, u)
    assert torch.equal(sample(x.view(2, 3, 1003), u.view(2, 3)), want.view(2, 3))
    assert torch.equal(sample(x[4], u[4]), want[4])
    assert torch.equal(sample(x.t().contiguous().t(), u), want)
    assert torch.equal(sample(x[:1].expand(6, -1), u), sample(x[:1].repeat(6, 1), u))
    assert sample(x[:0], u[:0]).shape == (0,)


def test_frequencies(gpu):
    """Evenly spaced numbers reach each token as often as its weight says, to one count."""
    x = torch.tensor([0.3, -1.0, 2.0, 0.0, 1.1])
    n = 20000
    u = ((torch.arange(n) + 0.5) / n).float().cuda()
    got = torch.bincount(sample(x.cuda().expand(n, -1).contiguous(), u), minlength=5).cpu()
    want = torch.softmax(x.double(), 0) * n
    assert ((got - want).abs() <= 1.5).all()


def test_graph_and_streams(gpu):
    x, u = zipf(16, 32000, torch.bfloat16, 9)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        sample(x, u, top_p=0.9)
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = sample(x, u, top_p=0.9)
    for i in range(4):
        y, v = zipf(16, 32000, torch.bfloat16, 20 + i)
        x.copy_(y)
        u.copy_(v)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, sample(y, v, top_p=0.9))


def test_refusals(gpu):
    x, u = zipf(3, 100, torch.float32, 1)

    def no(match, *a, err=ValueError, **kw):
        with pytest.raises(err, match=match):
            sample(*a, **kw)
    no("no CPU path", x.cpu(), u, err=RuntimeError)
    no("no CPU path", x, u.cpu(), err=RuntimeError)
    no("no CPU path", x, u, top_p=u.cpu(), err=RuntimeError)
    no("dtype", x.double(), u)
    no("u must be", x, u.double())
    no("u must be", x, u[:2])
    no("logits must be", x[:, :0], u)
    no("logits must be", torch.empty(1, (1 << 20) + 1, device="cuda", dtype=torch.float16), u[:1])
    for t in (-0.1, float("nan"), float("inf")):
        no("temperature", x, u, temperature=t)
    for v in (-0.1, 1.1, float("nan")):
        no("top_p", x, u, top_p=v)
        no("min_p", x, u, min_p=v)
    no("top_k", x, u, top_k=-1)
    no("top_k", x, u, top_k=2.5)
    no("top_k", x, u, top_k=torch.ones(3, device="cuda", dtype=torch.int64))
    no("top_p", x, u, top_p=torch.ones(2, device="cuda"))
    no("temperature must be a number", x, u, temperature="hot")
