"""GPU: llmt.embedding and its gradient against float64: types, odd widths, strides, padding, tokens
that repeat, every sort (few positions by rank, more by radix passes).

A gradient row is a sum of c products in fp32 in the positions' order: off by at most c 2^-24 of the
sum of magnitudes, then scaled, added and rounded (2^-23 of the parts' magnitudes) and rounded to the
table's type (eps / 2)."""
import pytest
import torch

import llmt

pytestmark = pytest.mark.gpu
F, H, B = torch.float32, torch.float16, torch.bfloat16


def tokens(T, V, pad=0.1, seed=0):
    g = torch.Generator().manual_seed(seed + T)
    t = ((V + 1.0) ** torch.rand(T, generator=g, dtype=torch.float64) - 1).long().clamp(0, V - 1)
    t[torch.rand(T, generator=g) < pad] = -1
    return t.to(torch.int32)


@pytest.mark.parametrize("wt,ot", [(F, F), (F, B), (H, H), (H, F), (B, B), (B, F), (B, H)])
@pytest.mark.parametrize("V,W", [(1, 1), (7, 3), (100, 64), (300, 1037), (50, 2048), (10, 8200)])
def test_lookup(dev, wt, ot, V, W):
    w = torch.randn(V, W).to(wt).to(dev)
    t = tokens(61, V, 0.2).to(dev)
    t[3] = V                      # as far out as -1
    for scale in (1.0, 3.25):
        x = llmt.embedding(t, w, scale=scale, out_dtype=ot)
        ok = (t >= 0) & (t < V)
        want = torch.where(ok[:, None], w[t.long().clamp(0, V - 1)].float() * scale, 0.0).to(ot)
        assert x.dtype == ot and torch.equal(x, want)


@pytest.mark.parametrize("T,V,W", [(4096, 900, 24), (4097, 900, 24), (9000, 70000, 33), (65535, 300, 8),
                                   (65536, 300, 8), (65537, 600, 5)])
@pytest.mark.parametrize("accumulate", [False, True])
def test_gradient_where_sort_and_chunks_change(dev, accumulate, T, V, W):
    g = torch.Generator().manual_seed(T)
    dout = torch.randn(T, W, generator=g).to(B).to(dev)
    check_grad(dev, tokens(T, V).to(dev), dout, torch.randn(V, W, generator=g).to(dev), 0.5, accumulate)


@pytest.mark.parametrize("T", [1025, 4096, 20000])
@pytest.mark.parametrize("W", [4, 264, 1000])
def test_one_token_at_all_positions(dev, T, W):
    """A run over every chunk, more of them than a workgroup has threads."""
    g = torch.Generator().manual_seed(T)
    dout = torch.randn(T, W, generator=g).to(dev)
    for at, V in ((0, 1), (2, 5)):
        t = torch.full((T,), at, dtype=torch.int32, device=dev)
        check_grad(dev, t, dout, torch.ones(V, W, device=dev), 2.0, False)


def test_lookup_of_strided_rows_and_shapes(dev):
    w = torch.randn(40, 96, device=dev)[:, 5:70]
    t = tokens(24, 40).to(dev).view(2, 3, 4)
    x = llmt.embedding(t, w)
    assert x.shape == (2, 3, 4, 65)
    assert torch.equal(x, torch.where((t >= 0)[..., None], w[t.long().clamp(min=0)], 0.0))
    assert llmt.embedding(t.view(-1)[:0].contiguous(), w).shape == (0, 65)


def check_grad(dev, t, dout, dw, scale, accumulate):
    V, W = dw.shape
    before = dw.clone()
    ok = (t >= 0) & (t < V)
    at = t[ok].long().cpu()
    d = dout.reshape(t.numel(), W)[ok.reshape(-1)].double().cpu()
    z = lambda: torch.zeros(V, W, dtype=torch.float64)
    total, mag = z().index_add_(0, at, d), z().index_add_(0, at, d.abs())
    count = torch.zeros(V, dtype=torch.float64).index_add_(0, at, torch.ones(len(at), dtype=torch.float64))
    want = total * scale
    parts = mag * abs(scale)
    if accumulate:
        want += before.double().cpu()
        parts = parts + before.double().cpu().abs()
    got = llmt.embedding_bwd(t, dout, dw, scale=scale, accumulate=accumulate)
    assert got is dw
    tiny = {F: 0.0, B: 0.0, H: 2.0 ** -25}[dw.dtype]
    u = 0.0 if dw.dtype == F else torch.finfo(dw.dtype).eps / 2
    bound = (count[:, None] + 2) * 2 ** -24 * parts + 2 ** -23 * parts + u * want.abs() + tiny
    off = (dw.double().cpu() - want).abs()
    assert (off <= bound * (1 + 2 ** -10)).all(), (off / (bound + 1e-300)).max()
    if accumulate:
        untouched = (count == 0).nonzero()[:, 0].to(dev)
        assert torch.equal(dw[untouched], before[untouched])


@pytest.mark.parametrize("dt,wt", [(F, F), (B, F), (H, F), (B, B), (H, H), (F, B)])
@pytest.mark.parametrize("accumulate", [False, True])
@pytest.mark.parametrize("T,V,W", [(1, 1, 1), (2, 5, 9), (5, 1, 64), (63, 30, 130), (300, 511, 256),
                                   (1000, 20, 520), (2047, 100000, 17), (2500, 3, 72)])
def test_gradient(dev, dt, wt, accumulate, T, V, W):
    g = torch.Generator().manual_seed(T + V + W)
    dout = torch.randn(T, W, generator=g).to(dt).to(dev)
    dw = torch.randn(V, W, generator=g).to(wt).to(dev)
    check_grad(dev, tokens(T, V).to(dev), dout, dw, 1.5, accumulate)


# by rank with 16 and 8 lanes, by radix of one, two and three digits, more workgroups than one
@pytest.mark.parametrize("T,V", [(8192, 700), (8193, 40000), (16384, 7), (16385, 300), (16385, 511),
                                 (20000, 512), (33333, 151936), (40000, 262144), (17000, 3), (270000, 90)])
@pytest.mark.parametrize("accumulate", [False, True])
def test_gradient_of_many_tokens(dev, T, V, accumulate):
    g = torch.Generator().manual_seed(T + V)
    W = 12
    dout = torch.randn(T, W, generator=g).to(B).to(dev)
    dw = torch.randn(V, W, generator=g).to(dev)
    check_grad(dev, tokens(T, V).to(dev), dout, dw, 1.0, accumulate)


@pytest.mark.parametrize("T", [40, 3000, 20000])
def test_gradient_of_one_token_or_none(dev, T):
    dout = torch.randn(T, 64, device=dev)
    for v in (0, 4, -1, 5):
        t = torch.full((T,), v, dtype=torch.int32, device=dev)
        check_grad(dev, t, dout, torch.ones(5, 64, device=dev), 0.5, True)
        check_grad(dev, t, dout, torch.ones(5, 64, device=dev), 0.5, False)


def test_gradient_of_no_tokens(dev):
    t = torch.zeros(0, dtype=torch.int32, device=dev)
    dw = torch.ones(5, 64, device=dev)
    llmt.embedding_bwd(t, dw[:0], dw, accumulate=True)
    assert (dw == 1).all()
    llmt.embedding_bwd(t, dw[:0].clone(), dw)
    assert not dw.any()


def test_gradient_of_large_vocabularies_has_three_digits(dev):
    V, T = (1 << 18) + 5, 17001
    t = torch.randint(0, V, (T,), dtype=torch.int32)
    t[::7] = V - 1
    check_grad(dev, t.to(dev), torch.randn(T, 3, device=dev), torch.zeros(V, 3, device=dev), 1.0, False)


def test_gradient_into_strided_rows_leaves_the_rest(dev):
    buf = torch.full((30, 100), 9.0, device=dev)
    wide = torch.randn(500, 80, device=dev)
    t = tokens(500, 30).to(dev)
    check_grad(dev, t, wide[:, 3:68], buf[:, 7:72], 1.0, False)
    assert (buf[:, :7] == 9).all() and (buf[:, 72:] == 9).all()
    check_grad(dev, t, wide[:, 3:68], buf[:, 7:72], 1.0, True)


def test_infinities_and_nan_stay_with_their_token(dev):
    t = torch.tensor([1, 2, 3, 2, -1], dtype=torch.int32, device=dev)
    d = torch.ones(5, 8, device=dev)
    d[1, 0], d[2, 1], d[4] = float("inf"), float("nan"), float("nan")
    w = torch.empty(6, 8, device=dev)
    llmt.embedding_bwd(t, d, w)
    assert w[2, 0] == float("inf") and w[3, 1].isnan()
    w[2, 0] = w[3, 1] = 0
    assert w.isfinite().all()


@pytest.mark.parametrize("T,V", [(700, 50), (20000, 3000)])
def test_same_bits_twice_captured_and_on_another_stream(dev, T, V):
    t = tokens(T, V).to(dev)
    d = torch.randn(T, 256, device=dev).to(B)
    w = torch.randn(V, 256, device=dev)
    start = w.clone()
    want = llmt.embedding_bwd(t, d, w.clone(), accumulate=True)
    x = llmt.embedding(t, w.to(B))
    graph = torch.cuda.CUDAGraph()
    table = w.to(B)
    with torch.cuda.graph(graph):
        llmt.embedding_bwd(t, d, w, accumulate=True)
        y = llmt.embedding(t, table)
    for _ in range(3):
        w.copy_(start)
        y.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(w, want) and torch.equal(x, y)
    s = torch.cuda.Stream()
    w.copy_(start)
    s.wait_stream(torch.cuda.current_stream())
    llmt.embedding_bwd(t, d, w, accumulate=True, stream=s)
    s.synchronize()
    assert torch.equal(w, want)
