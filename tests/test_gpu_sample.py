"""Token sampling on the GPU against a plain 64-bit form on the CPU: tokens are equal."""
import math

import pytest
import torch

from bfloat16x_b200 import _lib
from bfloat16x_b200.sampling import sample

pytestmark = pytest.mark.gpu


def plain(logits, u, temperature, top_k, top_p, min_p):
    """One row, by the definition."""
    x = logits.double()
    x = torch.where(x.isnan(), torch.full_like(x, -math.inf), x)
    top = float(x.max())
    if top == -math.inf:
        return -1
    order = sorted(range(len(x)), key=lambda i: (-float(x[i]), i))
    if not temperature > 0 or top_k == 1:
        return order[0]
    w = torch.where(x == top, torch.ones_like(x), torch.exp((x - top) / float(torch.tensor(temperature))))
    if top_k > 0:
        order = order[:top_k]
    if top_p < 1:
        ws = w[order]
        cum = torch.cumsum(ws, 0)
        n = int((cum - ws < float(torch.tensor(top_p)) * float(cum[-1])).sum())
        order = order[:max(n, 1)]
    keep = torch.zeros_like(w)
    keep[order] = 1
    if min_p > 0:
        keep *= w >= float(torch.tensor(min_p))
    w = w * keep
    cum = torch.cumsum(w, 0)
    return int((cum <= float(u) * float(cum[-1])).sum())


def _rows(B, V, seed, kind="normal", dtype=torch.float32):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(B, V, generator=g) * 2.5
    if kind == "ties":
        x = (x * 2).round() / 2
    if kind == "bf16":
        x = x.to(torch.bfloat16).float()
    return x.to(dtype), torch.rand(B, generator=g)


@pytest.mark.parametrize("V", [1, 2, 31, 33, 500, 4099])
@pytest.mark.parametrize("kind,dtype", [("normal", torch.float32), ("ties", torch.float32), ("bf16", torch.bfloat16)])
def test_sample_filters(V, kind, dtype):
    settings = [(1.0, 0, 1.0, 0.0), (0.7, 5, 1.0, 0.0), (1.3, 0, 0.8, 0.0), (1.0, 0, 1.0, 0.1), (0.9, 40, 0.9, 0.02),
                (0.0, 0, 1.0, 0.0), (1.0, 1, 0.5, 0.0), (1.0, 0, 1e-9, 0.0), (1.0, 0, 1.0, 1.0), (5.0, 10 ** 6, 0.999, 0.0),
                (1.0, 3, 0.99, 0.5), (0.02, 0, 0.3, 0.0)]
    for i, (t, k, p, m) in enumerate(settings):
        x, u = _rows(3, V, 17 * V + i, kind, dtype)
        got = sample(x.cuda(), u.cuda(), t, k, p, m)
        want = [plain(x[r], u[r], t, k, p, m) for r in range(3)]
        assert got.tolist() == want, (t, k, p, m)
    _lib.check_device_status()


def test_sample_settings_per_row_and_strides():
    B, V = 23, 1000
    x, u = _rows(B, V, 3, "ties")
    t = [(1.0, 0.0, 0.6, 2.0)[i % 4] for i in range(B)]
    k = [(0, 7, 300)[i % 3] for i in range(B)]
    p = [(1.0, 0.7)[i % 2] for i in range(B)]
    m = [(0.0, 0.05, 0.0, 0.0, 0.3)[i % 5] for i in range(B)]
    want = [plain(x[i], u[i], t[i], k[i], p[i], m[i]) for i in range(B)]
    args = (torch.tensor(t).cuda(), torch.tensor(k, dtype=torch.int32).cuda(), torch.tensor(p).cuda(),
            torch.tensor(m).cuda())
    assert sample(x.cuda(), u.cuda(), *args).tolist() == want
    wide = torch.full((B, V + 37), 50.0).cuda()
    wide[:, 5:5 + V] = x.cuda()
    assert sample(wide[:, 5:5 + V], u.cuda(), *args).tolist() == want
    tr = x.t().contiguous().cuda().t()
    out = torch.empty(B, dtype=torch.int64, device="cuda")
    assert sample(tr, u.cuda(), *args, out=out) is out and out.tolist() == want


def test_sample_special_rows():
    V = 300
    inf = float("inf")
    g = torch.Generator().manual_seed(4)
    rows = [torch.full((V,), -inf), torch.full((V,), float("nan")), torch.full((V,), -3.4028e38), torch.zeros(V)]
    one = torch.full((V,), -inf)
    one[123] = -7.0
    some = torch.randn(V, generator=g)
    some[::2] = -inf
    some[5] = float("nan")
    big = torch.randn(V, generator=g)
    big[[40, 200]] = inf
    tiny = torch.randn(V, generator=g) * 1e-30
    zeros = torch.zeros(V)
    zeros[::3] = -0.0
    mask = torch.randn(V, generator=g)
    mask[50:] = -3.4028234663852886e38
    rows += [one, some, big, tiny, zeros, mask]
    x = torch.stack(rows)
    for t, k, p, m in ((1.0, 0, 1.0, 0.0), (0.5, 3, 1.0, 0.0), (1.0, 0, 0.5, 0.0), (1.0, 4, 0.6, 0.2), (0.0, 0, 1.0, 0.0)):
        for uu in (0.0, 0.37, 0.9999999):
            u = torch.full((len(rows),), uu)
            got = sample(x.cuda(), u.cuda(), t, k, p, m).tolist()
            assert got == [plain(r, uu if uu < 0.99 else float(u[0]), t, k, p, m) for r in x], (t, k, p, m, uu)


@pytest.mark.parametrize("B,V,dtype", [(1, 128256, torch.float32), (2, 73448, torch.bfloat16), (40, 20011, torch.float32),
                                       (160, 9000, torch.float32), (1, 327680, torch.float32)])
def test_sample_large(B, V, dtype):
    x, u = _rows(B, V, V, "bf16" if dtype == torch.bfloat16 else "normal", dtype)
    xd, ud = x.cuda(), u.cuda()
    for t, k, p, m in ((1.0, 0, 1.0, 0.0), (1.2, 0, 0.9, 0.0), (0.8, 50, 0.95, 0.01), (1.0, 5000, 1.0, 0.0)):
        got = sample(xd, ud, t, k, p, m)
        rows = range(B) if B * V < 400000 else (0, B // 2, B - 1)
        want = []
        for r in rows:
            xr = x[r].double()
            s, idx = torch.sort(xr, descending=True, stable=True)
            w = torch.exp((s - s[0]) / float(torch.tensor(t)))
            if k:
                w[k:] = 0
            cum = torch.cumsum(w, 0)
            if p < 1:
                w = w * (cum - w < float(torch.tensor(p)) * cum[-1])
            w = w * (w >= float(torch.tensor(m)))
            full = torch.zeros_like(w)
            full[idx] = w
            cum = torch.cumsum(full, 0)
            want.append(int((cum <= float(u[r]) * cum[-1]).sum()))
        assert [int(got[r]) for r in rows] == want


def test_sample_extreme_temperatures():
    """Too small for a reciprocal in fp32: the largest logit; infinite: every token alike."""
    x, u = _rows(3, 777, 9)
    for t in (1e-45, 4e-39):
        got = sample(x.cuda(), u.cuda(), temperature=torch.full((3,), t, device="cuda"), top_p=0.9)
        assert torch.equal(got.cpu(), x.argmax(1))
    x[:, 5] = float("-inf")
    got = sample(x.cuda(), u.cuda(), temperature=float("inf")).cpu()
    alike = [i for i in range(777) if i != 5]
    assert got.tolist() == [alike[int(float(v) * 776)] for v in u]


def test_sample_distribution_and_graph():
    """Equally spaced numbers draw each token as often as its probability says; a captured call follows its inputs."""
    V, N = 50, 4096
    x = torch.randn(1, V, generator=torch.Generator().manual_seed(8)) * 1.5
    u = (torch.arange(N) + 0.5) / N
    xd = x.expand(N, V).contiguous().cuda()
    got = sample(xd, u.cuda(), 0.9)
    count = torch.bincount(got.cpu(), minlength=V).double() / N
    want = torch.softmax(x[0].double() / float(torch.tensor(0.9)), 0)
    assert float((count - want).abs().max()) <= 1.0 / N + 1e-9
    ud = torch.zeros(N, device="cuda")
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = sample(xd, ud, 0.9)
    ud.copy_(u)
    g.replay()
    assert torch.equal(out, got)


def _plain_fast(x, u, t, k, p, m):
    """plain() for long rows with a temperature above 0."""
    x = x.double()
    s, idx = torch.sort(x, descending=True, stable=True)
    w = torch.where(s == s[0], torch.ones_like(s), torch.exp((s - s[0]) / float(torch.tensor(t))))
    if k:
        w[k:] = 0
    cum = torch.cumsum(w, 0)
    if p < 1:
        keep = cum - w < float(torch.tensor(p)) * cum[-1]
        keep[0] = True
        w = w * keep
    w = w * (w >= float(torch.tensor(m)))
    cum = torch.cumsum(torch.zeros_like(w).scatter_(0, idx, w), 0)
    return int((cum <= float(u) * float(cum[-1])).sum())


@pytest.mark.parametrize("V", [5000, 60001, 200000])
@pytest.mark.parametrize("kind", ["equal", "two", "steps", "wide", "narrow", "flat-bf16"])
def test_sample_many_ties_and_broad_rows(V, kind):
    """Cuts inside bins of more tokens than one CTA sorts, and cuts after thousands of tokens."""
    g = torch.Generator().manual_seed(V)
    x = torch.randn(4, V, generator=g)
    x = {"equal": torch.full_like(x, 2.5), "two": (x > 1).float() * 0.5, "steps": (x * 2).round() / 2, "wide": x * 8,
         "narrow": x * 1e-3, "flat-bf16": (x * 0.3).to(torch.bfloat16).float()}[kind]
    # numbers away from the 64-bit form's own rounding where weights are equal and sums tie exactly
    u = torch.tensor([0.0, 0.2871, 0.7313, 0.99993])
    for t, k, p, m in ((1.0, 0, 0.9, 0.0), (0.7, 3001, 1.0, 0.0), (1.1, 4500, 0.65, 0.0), (1.0, 0, 0.9999999, 0.0),
                       (1.0, 2, 0.5, 0.0), (1.0, 0, 0.0, 0.0), (1.0, V - 1, 0.999, 0.2), (3.0, 1025, 0.3, 0.0)):
        got = sample(x.cuda(), u.cuda(), t, k, p, m).tolist()
        assert got == [_plain_fast(x[i], u[i], t, k, p, m) for i in range(4)], (t, k, p, m)
