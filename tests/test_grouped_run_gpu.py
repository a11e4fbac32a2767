"""The grouped products as they are used together: a routed layer's forward and backward pass, the same layer over 4-bit experts, calls
on several streams, captured and replayed ones."""
import pytest
import torch

from grouped_util import ends_of, spans

pytestmark = pytest.mark.gpu
M, H, I, E, TOPK = 60, 128, 96, 7, 2


def _layer(seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(M, H, device="cuda", generator=g).half()
    logits = torch.randn(M, E, device="cuda", generator=g)
    gate, up = ((torch.randn(E, I, H, device="cuda", generator=g) / H ** 0.5).half() for _ in range(2))
    down = (torch.randn(E, H, I, device="cuda", generator=g) / I ** 0.5).half()
    return x, logits, gate, up, down, torch.randn(M, H, device="cuda", generator=g).half()


def _sorted(exl3, logits):
    """Rows of every pick in the order of their experts, the picks' weights and the experts' ends."""
    ids, w = exl3.route_topk(logits, TOPK)
    counts, tok, pw, _ = exl3.moe_align(ids, w, E)
    return ids, w, tok.long(), pw, counts.cumsum(0, dtype=torch.int32)


def test_routed_layer_forward_and_backward(exl3):
    """moe_align sorts the picks, three grouped products and silu_mul make the layer; its gradients by grouped_mm_dx and grouped_mm_dw
    against autograd in 64 bits. What is rounded in between is rounded in the reference too (fp16: half a step, 2^-11), so the
    results differ by roundings that fall the other way: below two steps of the largest value for every output, of which at most
    seven roundings on the way count."""
    x, logits, gate, up, down, dy = _layer(1)
    ids, w, tok, pw, ends = _sorted(exl3, logits)
    rows = x[tok]
    a, b = exl3.grouped_mm(rows, gate, ends), exl3.grouped_mm(rows, up, ends)
    h = torch.empty_like(a)
    exl3.silu_mul(a, b, h, 0.0)
    y = exl3.grouped_mm(h, down, ends, out_dtype=torch.float32)
    out = torch.zeros(M, H, device="cuda").index_add_(0, tok, y * pw[:, None])

    # backward
    dpick = (dy[tok].float() * pw[:, None]).half()
    dh = exl3.grouped_mm_dx(dpick, down, ends, out_dtype=torch.float32)
    ddown = exl3.grouped_mm_dw(dpick, h, ends, out_dtype=torch.float32)
    s = torch.sigmoid(a.float())
    da = (dh * b.float() * s * (1 + a.float() * (1 - s))).half()
    db = (dh * a.float() * s).half()
    drows = exl3.grouped_mm_dx(da, gate, ends, out_dtype=torch.float32) + exl3.grouped_mm_dx(db, up, ends, out_dtype=torch.float32)
    dgate, dup = exl3.grouped_mm_dw(da, rows, ends, out_dtype=torch.float32), exl3.grouped_mm_dw(db, rows, ends, out_dtype=torch.float32)
    dx = torch.zeros(M, H, device="cuda").index_add_(0, tok, drows)

    x64, gate64, up64, down64 = (t.double().requires_grad_(True) for t in (x, gate, up, down))
    ref = torch.zeros(M, H, dtype=torch.float64, device="cuda")
    for e, lo, hi in spans(ends):
        t = tok[lo:hi]
        r = x64[t]
        u, v = torch.mm(r, gate64[e].t()), torch.mm(r, up64[e].t())
        ref = ref.index_add(0, t, torch.mm(u * torch.sigmoid(u) * v, down64[e].t()) * pw[lo:hi, None].double())
    grads = torch.autograd.grad((ref * dy.double()).sum(), (x64, gate64, up64, down64))
    assert int(ends[-1]) == M * TOPK and len(set(ids.flatten().tolist())) == E
    for got, want in ((out, ref.detach()), (dx, grads[0]), (dgate, grads[1]), (dup, grads[2]), (ddown, grads[3])):
        assert float((got.double() - want).abs().max()) <= 7 * 2.0 ** -11 * float(want.abs().max())

    # a second micro-batch's gradient on top of the first's
    both = dgate.clone()
    exl3.grouped_mm_dw(da, rows, ends, out=both, accumulate=True)
    assert torch.equal(both, 2 * dgate)


def test_routed_layer_over_4_bit_experts(exl3):
    x, logits, *_ = _layer(2)
    _, _, tok, pw, ends = _sorted(exl3, logits)
    g = torch.Generator(device="cuda").manual_seed(5)

    def experts(n, k):
        codes = torch.randint(0, 256, (E, n, k // 2), device="cuda", generator=g, dtype=torch.uint8)
        scales = (torch.rand(E, n, k // 32, device="cuda", generator=g) / (4 * k ** 0.5)).half()
        q = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).double().unflatten(-1, (-1, 32))
        return exl3.G4Tensor(codes, scales), ((q - 8) * scales.double()[..., None]).flatten(-2)

    (gu, gu64), (dn, dn64) = experts(2 * I, H), experts(H, I)
    z = exl3.grouped_mm(x[tok], gu, ends)
    h = torch.empty(len(tok), I, dtype=torch.float16, device="cuda")
    exl3.silu_mul(z[:, :I].contiguous(), z[:, I:].contiguous(), h, 0.0)
    y = exl3.grouped_mm(h, dn, ends, out_dtype=torch.float32)
    out = torch.zeros(M, H, device="cuda").index_add_(0, tok, y * pw[:, None])
    ref = torch.zeros(M, H, dtype=torch.float64, device="cuda")
    for e, lo, hi in spans(ends):
        t = tok[lo:hi]
        u = torch.mm(x[t].double(), gu64[e].t().contiguous())
        h64 = u[:, :I] * torch.sigmoid(u[:, :I]) * u[:, I:]
        ref.index_add_(0, t, torch.mm(h64, dn64[e].t().contiguous()) * pw[lo:hi, None].double())
    # two roundings of the products, one of the activation
    assert float((out.double() - ref).abs().max()) <= 4 * 2.0 ** -11 * float(ref.abs().max())


def _calls(exl3, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    ends = ends_of([300, 0, 21, 500, 3])
    T = 824
    x, dy = torch.randn(T, 256, device="cuda", generator=g).bfloat16(), torch.randn(T, 192, device="cuda", generator=g).bfloat16()
    w = torch.randn(5, 192, 256, device="cuda", generator=g).bfloat16()
    few, few_ends = x[:6].contiguous(), ends_of([1, 2, 0, 2, 1])
    codes = torch.randint(0, 256, (5, 192, 128), device="cuda", generator=g, dtype=torch.uint8)
    scales = torch.rand(5, 192, 4, device="cuda", generator=g).bfloat16()
    t = exl3.G4Tensor(codes, scales)
    one = exl3.G4Linear(exl3.G4Tensor(torch.randint(0, 256, (256, 8192), device="cuda", generator=g, dtype=torch.uint8),
                                      torch.rand(256, 128, device="cuda", generator=g).bfloat16()))
    long = torch.randn(90, 16384, device="cuda", generator=g).bfloat16()
    assert exl3.lib().exl3_g4_linear_scratch(90, 16384, 256, 128) > 0
    long_x, long_dy, long_ends = x.repeat(8, 1)[:, :64].contiguous(), dy.repeat(8, 1)[:, :64].contiguous(), ends_of([6000, 592])
    assert exl3.lib().exl3_grouped_mm_dw_scratch(6592, 64, 64, 2) > 0
    return {"mm": lambda: exl3.grouped_mm(x, w, ends), "few": lambda: exl3.grouped_mm(few, w, few_ends),
            "dx": lambda: exl3.grouped_mm_dx(dy, w, ends), "dw": lambda: exl3.grouped_mm_dw(dy, x, ends),
            "dw_parts": lambda: exl3.grouped_mm_dw(long_dy, long_x, long_ends, out_dtype=torch.float32),
            "g4": lambda: exl3.grouped_mm(x, t, ends), "linear_splits": lambda: one.run_alloc(long, 256, True)}


NAMES = ["mm", "few", "dx", "dw", "dw_parts", "g4", "linear_splits"]


@pytest.mark.parametrize("name", NAMES)
def test_calls_overlap_on_streams(exl3, name):
    calls = [_calls(exl3, s)[name] for s in (10, 20, 30)]
    want = [c() for c in calls]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in calls]
    out = [[] for _ in calls]
    for _ in range(20):
        for s, c, o in zip(streams, calls, out):
            with torch.cuda.stream(s):
                o.append(c())
    torch.cuda.synchronize()
    for w, o in zip(want, out):
        assert all(torch.equal(y, w) for y in o)


@pytest.mark.parametrize("name", NAMES)
def test_graphs_replay_beside_each_other_and_eager_calls(exl3, name):
    calls = [_calls(exl3, s)[name] for s in (10, 20, 30)]
    want = [c() for c in calls]
    torch.cuda.synchronize()
    graphs, outs = [], []
    for c in calls[:2]:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append([c() for _ in range(3)])
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in range(3)]
    for _ in range(5):
        for s, g in zip(streams, graphs):
            with torch.cuda.stream(s):
                for _ in range(3):
                    g.replay()
        with torch.cuda.stream(streams[2]):
            eager = [calls[2]() for _ in range(9)]
        torch.cuda.synchronize()
        assert all(torch.equal(y, want[2]) for y in eager)
        for w, o in zip(want, outs):
            assert all(torch.equal(y, w) for y in o)
            for y in o:
                y.zero_()
        torch.cuda.synchronize()


def test_replays_follow_the_ends(exl3):
    """A captured call reads the ends at each replay."""
    x = torch.randn(64, 128, device="cuda").bfloat16()
    w = torch.randn(3, 72, 128, device="cuda").bfloat16()
    ends = ends_of([10, 20, 30])
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = exl3.grouped_mm(x, w, ends)
        dw = exl3.grouped_mm_dw(y, x, ends)
    for sizes in ([10, 20, 30], [0, 64, 0], [1, 0, 63], [0, 0, 0], [21, 21, 22]):
        ends.copy_(ends_of(sizes))
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, exl3.grouped_mm(x, w, ends)) and torch.equal(dw, exl3.grouped_mm_dw(y, x, ends))
