"""Router balance and its gradient against 64-bit formulas, automatic differentiation and differences."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
SCORES = ("softmax", "sigmoid", "sqrt_softplus")
TINY = 2.0 ** -126                                       # below it fp32 loses bits, or its functions return 0


def shares(z, score):
    """Shares in float64 (rows whose scores are all zero: zero)."""
    if score == "softmax":
        return torch.softmax(z, 1)
    s = torch.sigmoid(z) if score == "sigmoid" else torch.sqrt(torch.nn.functional.softplus(z, threshold=50.0))
    return s / s.sum(1, keepdim=True)


def balance64(z, ids, score, mask, coef):
    M, E = z.shape
    live = torch.ones(M, dtype=torch.bool) if mask is None else mask
    n = int(live.sum())
    picks = ids[live].reshape(-1)
    counts = torch.bincount(picks[(picks >= 0) & (picks < E)].long(), minlength=E)
    zl = z[live].double().requires_grad_(True)
    p = shares(zl, score)
    prob = p.sum(0) / max(n, 1)
    frac = E * counts.double() / (ids.shape[1] * max(n, 1))
    loss = coef * (frac * prob).sum()
    d = torch.zeros(M, E, dtype=torch.float64)
    scale = torch.zeros(M, E, dtype=torch.float64)       # what the gradient's differences are taken between
    if n:
        d[live] = torch.autograd.grad(loss, zl)[0]
        a = coef * frac / n
        pd = p.detach()
        scale[live] = pd * (a.abs() + (pd * a.abs()).sum(1, keepdim=True))
    return loss.detach(), counts, prob.detach(), d, scale, n


def tol(z, M):
    """Relative error of a share: two steps of exp and its argument's rounding (|z| and the maximum, 2^-24 each), the row's
    sum and reciprocal (at most 32 + 8 additions); of a mean: a chain of at most M / 8 + 40 more."""
    top = float(z[torch.isfinite(z)].abs().max()) if torch.isfinite(z).any() else 0.0
    share = (2 * top + 60) * 2.0 ** -23
    return share, share + (min(M / 8, 80) + 48) * 2.0 ** -23


def compare(exl3, z, ids, score, mask, coef):
    g = torch.tensor([0.75])
    dz, di, dm = z.to(DEV), ids.to(DEV), None if mask is None else mask.to(DEV)
    loss, counts, prob, rows = exl3.route_balance(dz, di, score=score, mask=dm, coef=coef)
    d = exl3.route_balance_grad(dz, counts, rows, ids.shape[1], score=score, mask=dm, coef=coef, grad=g.to(DEV))
    rl, rc, rp, rd, scale, n = balance64(z, ids, score, mask, coef)
    ts, tp = tol(z, z.shape[0])
    assert int(rows) == n and torch.equal(counts.cpu().long(), rc)
    assert ((prob.cpu().double() - rp).abs() <= tp * rp + TINY).all()
    assert abs(float(loss) - float(rl)) <= (tp + 2.0 ** -17) * abs(float(rl)) + TINY   # 512 column blocks of 16 added
    err = (d.cpu().double() - 0.75 * rd).abs()
    assert (err <= 0.75 * (3 * ts * scale) + TINY).all(), float((err / (scale + 1e-300)).max())
    if mask is not None:
        assert (d[~dm] == 0).all()
    return loss, counts, prob, rows, d


def make(M, E, k, seed, wild=False):
    g = torch.Generator().manual_seed(seed)
    z = torch.randn(M, E, generator=g) * (4.0 if wild else 1.5) + torch.randn(E, generator=g)
    ids = torch.stack([torch.randperm(E, generator=g)[:k] for _ in range(M)]) if M else torch.empty(0, k)
    return z, ids.to(torch.int32).reshape(M, k)


@pytest.mark.parametrize("score", SCORES)
@pytest.mark.parametrize("M,E,k", [(1, 1, 1), (1, 2, 2), (3, 8, 2), (16, 160, 8), (32, 60, 4), (33, 64, 6), (100, 65, 3), (257, 129, 8),
                                   (700, 512, 10), (64, 1000, 4), (90, 2048, 8), (9, 2049, 8), (41, 5000, 4), (5, 8192, 32)])
def test_balance(exl3, score, M, E, k):
    z, ids = make(M, E, k, M + E)
    compare(exl3, z, ids, score, None, 0.01)
    mask = torch.rand(M, generator=torch.Generator().manual_seed(1)) < 0.6
    compare(exl3, z, ids, score, mask, 1.0)


@pytest.mark.parametrize("score", SCORES)
def test_balance_many_rows(exl3, score):
    z, ids = make(5000, 96, 4, 7)
    mask = torch.zeros(5000, dtype=torch.bool)
    mask[:4097] = True                                   # a padded tail
    l, c, p, n, d = compare(exl3, z, ids, score, mask, 0.5)
    for _ in range(3):                                   # the same bits every time
        l2, c2, p2, n2 = exl3.route_balance(z.to(DEV), ids.to(DEV), score=score, mask=mask.to(DEV), coef=0.5)
        assert torch.equal(l, l2) and torch.equal(c, c2) and torch.equal(p, p2) and torch.equal(n, n2)


@pytest.mark.parametrize("score", SCORES)
@pytest.mark.parametrize("M", [6, 300])
def test_balance_odd_picks_and_masks(exl3, score, M):
    z, ids = make(M, 40, 5, 11, wild=True)
    ids[::2, 1] = -1
    ids[1::3, 2] = 40
    ids[:, 4] = ids[:, 3]                                # the same expert twice in a row
    compare(exl3, z, ids, score, None, 0.3)
    for mask in (torch.zeros(M, dtype=torch.bool), torch.arange(M) == M - 1):
        l, c, p, n, d = compare(exl3, z, ids, score, mask, 0.3)
        if not mask.any():
            assert float(l) == 0 and int(n) == 0 and (c == 0).all() and (p == 0).all() and (d == 0).all()
    u8 = (torch.arange(M) % 3).to(torch.uint8)           # any non-zero byte is live
    a = exl3.route_balance(z.to(DEV), ids.to(DEV), score=score, mask=u8.to(DEV))
    b = exl3.route_balance(z.to(DEV), ids.to(DEV), score=score, mask=(u8 > 0).to(DEV))
    assert all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize("M", [4, 200])
def test_balance_infinite_logits(exl3, M):
    z, ids = make(M, 70, 3, 13)
    z[:, 5] = float("-inf")                              # a closed expert
    z[2, :] = float("-inf")
    z[2, 3] = 0.0                                        # one expert left: share 1
    compare(exl3, z, ids, "softmax", None, 1.0)
    for score in SCORES:                                 # a row of which nothing is left adds nothing
        z2 = z.clone()
        z2[1, :] = float("-inf")
        l, c, p, n = exl3.route_balance(z2.to(DEV), ids.to(DEV), score=score)
        d = exl3.route_balance_grad(z2.to(DEV), c, n, 3, score=score)
        assert int(n) == M and torch.isfinite(l).all() and torch.isfinite(p).all() and torch.isfinite(d).all()
        assert (d[1] == 0).all() and (d[:, 5] == 0).all()
        keep = torch.arange(M) != 1
        rp = shares(z2[keep].double(), score).sum(0) / M
        assert ((p.cpu().double() - rp).abs() <= tol(z, M)[1] * rp + TINY).all()
    zn = z.clone()
    zn[3, 7] = float("nan")
    l, c, p, n = exl3.route_balance(zn.to(DEV), ids.to(DEV))
    d = exl3.route_balance_grad(zn.to(DEV), c, n, 3)
    assert torch.isnan(l).all() and torch.isnan(d[3]).all() and torch.isfinite(d[:3]).all()


@pytest.mark.parametrize("score", SCORES)
def test_balance_far_logits(exl3, score):
    z, ids = make(24, 33, 2, 17)
    z[:, ::4] -= 60
    z[:, 1::4] += 40
    compare(exl3, z, ids, score, None, 1.0)


@pytest.mark.parametrize("score", SCORES)
def test_gradient_against_differences(exl3, score):
    """Central differences of the 64-bit loss (counts held), step 1e-4: their own error is of the order of 1e-8 of the scale."""
    z, ids = make(5, 12, 3, 19)
    l, c, p, n = exl3.route_balance(z.to(DEV), ids.to(DEV), score=score, coef=2.0)
    d = exl3.route_balance_grad(z.to(DEV), c, n, 3, score=score, coef=2.0).cpu().double()
    frac = 12 * c.cpu().double() / (3 * 5)

    def loss(zz):
        return 2.0 * (frac * shares(zz, score).mean(0)).sum()

    for t in range(5):
        for j in range(12):
            h = torch.zeros(5, 12, dtype=torch.float64)
            h[t, j] = 1e-4
            diff = (loss(z.double() + h) - loss(z.double() - h)) / 2e-4
            assert abs(float(diff) - float(d[t, j])) <= 1e-6


def test_balance_strides_streams_and_in_place(exl3):
    z, ids = make(50, 24, 3, 23)
    buf = torch.full((50, 40), 9.0, device=DEV)
    buf[:, 8:32] = z.to(DEV)
    a = exl3.route_balance(z.to(DEV), ids.to(DEV))
    b = exl3.route_balance(buf[:, 8:32], torch.cat([ids, ids], 1).to(DEV)[:, :3])
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    want = exl3.route_balance_grad(z.to(DEV), a[1], a[3], 3)
    got = exl3.route_balance_grad(buf[:, 8:32], a[1], a[3], 3, out=buf[:, 8:32])       # over its own logits
    assert torch.equal(got, want) and (buf[:, :8] == 9).all() and (buf[:, 32:] == 9).all()
    for bad in (dict(logits=z.to(DEV).double()), dict(score="relu"), dict(mask=torch.ones(49, dtype=torch.bool, device=DEV)),
                dict(topk_ids=ids.long().to(DEV)), dict(topk_ids=ids[:49].to(DEV))):
        kw = dict(dict(logits=z.to(DEV), topk_ids=ids.to(DEV)), **bad)
        with pytest.raises((exl3.Exl3Error, NotImplementedError)):
            exl3.route_balance(**kw)
    e = exl3.route_balance(z[:0].to(DEV), ids[:0].to(DEV))
    assert float(e[0]) == 0 and int(e[3]) == 0 and (e[1] == 0).all() and (e[2] == 0).all()
    assert exl3.route_balance_grad(z[:0].to(DEV), e[1], e[3], 3).shape == (0, 24)


def test_counts_of_several_processes_add_up(exl3):
    """Counts and rows summed over parts of a batch give every part the whole batch's gradient."""
    z, ids = make(90, 32, 4, 29)
    whole = exl3.route_balance(z.to(DEV), ids.to(DEV))
    want = exl3.route_balance_grad(z.to(DEV), whole[1], whole[3], 4)
    parts = [exl3.route_balance(z[i:i + 30].to(DEV), ids[i:i + 30].to(DEV)) for i in (0, 30, 60)]
    c, n = sum(p[1] for p in parts).to(torch.int32), sum(p[3] for p in parts).to(torch.int32)
    got = torch.cat([exl3.route_balance_grad(z[i:i + 30].to(DEV), c, n, 4) for i in (0, 30, 60)])
    assert torch.equal(c, whole[1]) and torch.equal(got, want)


@pytest.mark.parametrize("M", [16, 900])
def test_captured_balance_replays(exl3, M):
    """Routing, balance and gradient in one graph, replayed with eager work between."""
    z, _ = make(M, 48, 4, 31)
    z = z.to(DEV)

    def step():
        ids, w = exl3.route_topk(z, 4)
        l, c, p, n = exl3.route_balance(z, ids, coef=0.1)
        return ids, l, c, p, n, exl3.route_balance_grad(z, c, n, 4, coef=0.1)

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step()
    for r in range(4):
        z.copy_(make(M, 48, 4, 40 + r)[0].to(DEV))
        want = [t.clone() for t in step()]
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want)), r
