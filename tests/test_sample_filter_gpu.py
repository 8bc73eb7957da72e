"""Filtered sampling (csrc/sample_filter.hip) against the oracle in 64 bits.

Tokens are equal: the inputs' uniform numbers lie at random, and both sides' sums differ by some 1e-12 of their value, so that a
token at a border differs once in 1e9 rows or so. Log-probabilities: exponentials in fp32 of differences d from the largest
entry, |d| <= 60 where they count; the difference is rounded (2^-24 |d|, 4e-6) and so is the exponential (2^-22): 5e-6 of the sum
of the others, which is what a log-probability near 0 is; the rest of it is rounded to fp32 (2^-24 of its value).
"""
import math

import pytest
import torch

from docagents_amd.ops import reference as R

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(scope="module")
def K():
    from docagents_amd.ops import kernels
    return kernels


def _logits(g, B, V, f32, sigma, ld=None):
    x = torch.randn(B, ld or V, generator=g) * sigma
    x = x if f32 else x.bfloat16()
    return x[:, :V]


def _same(K, x, u, xg=None, **opts):
    """(the tensors of opts lie on the CPU)"""
    xg = x.to(DEV) if xg is None else xg
    tok, lp = K.sample_filtered(xg, u=u.to(DEV), **{k: v.to(DEV) if isinstance(v, torch.Tensor) else v for k, v in opts.items()})
    wt, wl = R.sample_filtered(x, u=u, **opts)
    assert torch.equal(tok.cpu(), wt), (tok.cpu() != wt).nonzero().flatten().tolist()
    lp = lp.cpu()
    fin = wl.isfinite()
    assert torch.equal(lp[~fin], wl[~fin])
    assert ((lp - wl)[fin].abs() <= 1e-5 * wl[fin].abs() + 1e-30).all(), (lp - wl)[fin].abs().max()
    return tok, lp


@pytest.mark.parametrize("f32", [False, True])
@pytest.mark.parametrize("V", [1, 2, 63, 64, 65, 1000, 2047, 2049, 32064, 50257])
@pytest.mark.parametrize("opts", [dict(top_k=1), dict(top_k=7), dict(top_k=40, top_p=0.9), dict(top_p=0.8), dict(min_p=0.1),
                                  dict(top_k=300, top_p=0.99, min_p=0.001), dict(top_p=0.999), dict(top_k=1500), dict()])
def test_filters(K, f32, V, opts):
    g = torch.Generator().manual_seed(V)
    B = 5
    x = _logits(g, B, V, f32, 3.0)
    for T in (0.3, 1.0, 1.7):
        _same(K, x, torch.rand(B, generator=g), temperature=T, **opts)


@pytest.mark.parametrize("V", [33, 5000, 128256])
def test_borders_of_u_and_of_the_options(K, V):
    g = torch.Generator().manual_seed(V)
    u = torch.tensor([0.0, 1 - 2 ** -24, 0.5, 2 ** -24])
    x = _logits(g, 4, V, False, 2.0)
    for opts in (dict(temperature=0.0), dict(temperature=-1.0, top_p=0.5), dict(temperature=0.01, top_k=50), dict(temperature=1.0, top_k=V),
                 dict(temperature=1.0, top_k=10 ** 9, top_p=0.7), dict(temperature=1.0, top_p=0.0), dict(temperature=1.0, top_p=1e-9),
                 dict(temperature=1.0, min_p=1.0), dict(temperature=1.0, min_p=2.0), dict(temperature=50.0), dict(temperature=50.0, top_p=0.5)):
        _same(K, x, u, **opts)


@pytest.mark.parametrize("f32", [False, True])
def test_equal_logits(K, f32):
    """Rows of one value, of two, and of few: the order among equals is the index's."""
    g = torch.Generator().manual_seed(5)
    V, B = 20011, 6
    x = torch.zeros(B, V)
    x[1] = -7.25
    x[2] = torch.where(torch.rand(V, generator=g) < 0.5, 1.0, 2.0)
    x[3] = torch.randint(0, 3, (V,), generator=g).float()
    x[4, ::2] = -0.0
    x[5, 17000:] = 3.0
    x = x if f32 else x.bfloat16()
    for opts in (dict(), dict(top_k=5), dict(top_k=9000), dict(top_p=0.5), dict(top_p=0.25, top_k=8000), dict(min_p=0.9), dict(min_p=1.0), dict(min_p=1.5),
                 dict(top_k=15000, top_p=0.9, min_p=0.3), dict(top_k=15000, top_p=0.9, min_p=1.5)):
        for _ in range(2):
            _same(K, x, torch.rand(B, generator=g), temperature=1.0, **opts)


@pytest.mark.parametrize("opts", [dict(top_k=3), dict(top_p=0.9), dict(), dict(min_p=0.2), dict(top_k=4000, top_p=0.9)])
def test_masked_entries(K, opts):
    """-inf, NaN, +inf and the type's lowest value; rows that a mask leaves one entry or none."""
    g = torch.Generator().manual_seed(9)
    V, B = 9001, 9
    x = torch.randn(B, V, generator=g)
    x[0] = -math.inf
    x[1] = math.nan
    x[2] = -math.inf
    x[2, 8999] = -3.0
    x[3, ::3] = math.nan
    x[4, 100], x[4, 7000] = math.inf, math.inf
    x[5] = torch.finfo(torch.bfloat16).min
    x[6, 1:] = torch.finfo(torch.bfloat16).min
    x[7, torch.rand(V, generator=g) < 0.99] = -math.inf
    x[8] = torch.finfo(torch.bfloat16).max
    for y in (x, x.bfloat16()):
        _same(K, y, torch.rand(B, generator=g), temperature=0.8, **opts)


def test_options_of_each_row(K):
    g = torch.Generator().manual_seed(11)
    B, V = 70, 4001
    x = _logits(g, B, V, False, 2.5)
    pick = lambda *v: torch.tensor(v)[torch.randint(0, len(v), (B,), generator=g)]  # noqa: E731
    _same(K, x, torch.rand(B, generator=g), temperature=pick(0.0, 0.5, 1.0, 2.0), top_k=pick(0, 1, 20, 3000).int(),
          top_p=pick(1.0, 0.2, 0.9, 0.99), min_p=pick(0.0, 0.05, 0.5))


@pytest.mark.parametrize("f32", [False, True])
def test_rows_of_any_stride_and_address(K, f32):
    g = torch.Generator().manual_seed(12)
    for ld, off in ((3003, 1), (3008, 3), (3000, 0)):
        x = _logits(g, 4, 3000 - off, f32, 2.0, ld=ld)
        flat = torch.zeros(4 * ld + off, dtype=x.dtype, device=DEV)
        xg = flat[off:].view(4, ld)[:, :3000 - off]
        xg.copy_(x)
        _same(K, x, torch.rand(4, generator=g), xg=xg, temperature=0.9, top_k=60, top_p=0.95)


@pytest.mark.parametrize("V", [262143, 262144])
def test_the_largest_vocabulary(K, V):
    g = torch.Generator().manual_seed(V)
    for f32 in (False, True):
        x = _logits(g, 2, V, f32, 1.5)
        for opts in (dict(top_k=50, top_p=0.9), dict(top_p=0.99), dict(), dict(top_k=100000)):
            _same(K, x, torch.rand(2, generator=g), temperature=1.1, **opts)
    with pytest.raises(ValueError, match="vocabulary"):
        K.sample_filtered(torch.zeros(1, (1 << 18) + 1, device=DEV), 1.0, top_k=3)


def test_what_is_refused(K):
    x = torch.randn(3, 100, device=DEV)
    for kw in (dict(temperature=torch.ones(3)), dict(temperature=torch.ones(2, device=DEV)), dict(temperature=1.0, top_k=torch.ones(3, device=DEV)),
               dict(temperature=1.0, u=torch.rand(3, device=DEV, dtype=torch.float64)), dict(temperature=1.0, u=torch.rand(3)),
               dict(temperature=1.0, out_tok=torch.zeros(3, device=DEV)), dict(temperature=1.0, conf=torch.zeros(3, 3, device=DEV)),
               dict(temperature=1.0, hist=torch.zeros(3, 4, dtype=torch.int32, device=DEV))):
        with pytest.raises(ValueError):
            K.sample_filtered(x, **kw)
    for y in (x.half(), x.double(), x[:, ::2], x.cpu()):
        with pytest.raises(ValueError):
            K.sample_filtered(y, 1.0, top_k=3)
    tok, lp = K.sample_filtered(x[:0], 1.0, top_k=3)
    assert tok.numel() == lp.numel() == 0


def test_own_numbers_and_bookkeeping(K):
    """Without u: the oracle's counter-based numbers; inactive rows stay as they were."""
    g = torch.Generator().manual_seed(13)
    B, V = 6, 2500
    x = _logits(g, B, V, False, 2.0)
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32)  # noqa: E731
    mk = lambda: dict(out_tok=torch.full((B,), -5, dtype=torch.int32), out_lp=torch.full((B,), 9.0), conf=torch.ones(B, 2),  # noqa: E731
                      active=i32(1, 1, 0, 1, 1, 1), pos=i32(3, 9, 4, 5, 6, 7), lens=i32(4, 10, 5, 6, 7, 8),
                      hist=torch.full((B, 4), -1, dtype=torch.int32), start=i32(3, 6, 4, 5, 5, 4))
    a, b = mk(), {k: v.to(DEV) for k, v in mk().items()}
    for step in range(2):
        R.sample_filtered(x, 0.9, 77, top_k=30, top_p=0.9, ctr=a["pos"], eos=(3, 5), **a)
        K.sample_filtered(x.to(DEV), 0.9, 77, top_k=30, top_p=0.9, ctr=b["pos"], eos=(3, 5), **b)
        for k in a:
            assert torch.allclose(a[k].float(), b[k].cpu().float(), rtol=1e-5, atol=0), k


def test_captured_and_beside_another_stream(K):
    g = torch.Generator().manual_seed(14)
    B, V = 8, 40000
    x = _logits(g, B, V, False, 1.0).to(DEV)
    u = torch.rand(B, generator=g).to(DEV)
    want, lp = K.sample_filtered(x, 1.2, top_p=0.97, u=u)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got, glp = K.sample_filtered(x, 1.2, top_p=0.97, u=u)
    for _ in range(3):
        graph.replay()
        with torch.cuda.stream(s):
            other, _ = K.sample_filtered(x, 1.2, top_p=0.97, u=u)
        K.sample_filtered(x[:2], 0.7, top_k=3)
        torch.cuda.synchronize()
        assert torch.equal(got, want) and torch.equal(glp, lp) and torch.equal(other, want)


def test_drawn_as_often_as_its_probability(K):
    """Even numbers through the whole range draw each entry as often as its share: within one draw of it."""
    V, B = 50, 20000
    x = torch.randn(V, generator=torch.Generator().manual_seed(1)).to(DEV).repeat(B, 1)
    u = ((torch.arange(B) + 0.5) / B).to(DEV)
    tok, _ = K.sample_filtered(x, 1.3, top_k=20, u=u)
    top = x[0].topk(20)
    share = torch.zeros(V, dtype=torch.float64, device=DEV)
    share[top.indices] = torch.softmax(top.values.double() / 1.3, 0)
    assert ((torch.bincount(tok.long(), minlength=V) - share * B).abs() <= 1.01).all()


@pytest.mark.parametrize("f32", [False, True])
@pytest.mark.parametrize("copies", [1, 7, 127, 128, 129, 700])
def test_lists_of_each_length(K, f32, copies):
    """As many entries as each way to sort them takes, all different to all alike."""
    g = torch.Generator().manual_seed(copies)
    V, B = 4000, 3
    x = (torch.randint(0, V // copies + 1, (B, V), generator=g).float() / 64 - 20)
    x = x if f32 else x.bfloat16()
    for k in (63, 64, 65, 127, 128, 129, 300, 1000, 2047, 2048, 2049, 3000):
        _same(K, x, torch.rand(B, generator=g), temperature=7.0, top_k=k)
        _same(K, x, torch.rand(B, generator=g), temperature=7.0, top_k=k, top_p=0.7, min_p=0.01)


@pytest.mark.parametrize("f32", [False, True])
@pytest.mark.parametrize("V", [2500, 30011, 131072])
def test_top_k_of_many_candidates(K, f32, V):
    """k near the number of groups and above it: the bound leaves more entries than the list holds."""
    g = torch.Generator().manual_seed(V + 1)
    B = 4
    for sigma in (0.5, 4.0):
        x = _logits(g, B, V, f32, sigma)
        x[3] = x[3].round()  # thousands of equal ones
        for k in (V // 70, V // 64 + 1, 1500, 2000, 2047, 2048):
            _same(K, x, torch.rand(B, generator=g), temperature=0.9, top_k=k)
            _same(K, x, torch.rand(B, generator=g), temperature=0.9, top_k=k, top_p=0.8)


@pytest.mark.parametrize("f32", [False, True])
@pytest.mark.parametrize("T", [1e-38, 1e-4, 0.05, 1.0, 1e4, 1e30, math.inf])
def test_any_temperature_and_value(K, f32, T):
    """Weights of 1 and of 0 and everything beside them; infinite entries, NaN, the type's largest values."""
    g = torch.Generator().manual_seed(11)
    V = 5003
    x = torch.randn(8, V, generator=g) * 3
    x[1, torch.randperm(V, generator=g)[:1500]] = -math.inf
    x[2, torch.randperm(V, generator=g)[:3000]] = math.nan
    x[3, torch.randperm(V, generator=g)[:200]] = 3e38
    x[4, torch.randperm(V, generator=g)[:200]] = -3e38
    x[5, torch.randperm(V, generator=g)[:3]] = math.inf
    x[6] = torch.where(torch.rand(V, generator=g) < 0.5, -0.0, 0.0)
    x[7] *= 1e-38
    x = x if f32 else x.bfloat16()
    for opts in (dict(), dict(top_k=900), dict(top_k=3000), dict(top_p=0.6), dict(top_k=1200, top_p=0.9, min_p=0.5)):
        _same(K, x, torch.rand(8, generator=g), temperature=T, **opts)


@pytest.mark.parametrize("f32", [False, True])
@pytest.mark.parametrize("V", [1, 3, 7, 8, 9, 57, 64, 120, 511, 2050])
def test_short_rows_at_each_address(K, f32, V):
    g = torch.Generator().manual_seed(V)
    for lead in range(9):
        for ld in (V + 8, V + 9):
            whole = torch.full((3, ld), 99.0)
            whole[:, lead:lead + V] = torch.randn(3, min(V, ld - lead), generator=g) * 2
            whole = whole if f32 else whole.bfloat16()
            on = whole.to(DEV)
            for opts in (dict(top_p=0.9), dict(top_k=max(1, V // 2)), dict()):
                _same(K, whole[:, lead:lead + V], torch.rand(3, generator=g), xg=on[:, lead:lead + V], temperature=0.8, **opts)


@pytest.mark.parametrize("B,V", [(1, 8185), (256, 600), (257, 600), (9, 8186), (32, 9000), (33, 9000), (4, 128256), (5, 128256)])
def test_one_launch_or_two(K, B, V):
    """About the sizes where a row's workgroups begin to share a launch: one after the other, in graphs on one stream and on two."""
    g = torch.Generator().manual_seed(B * V)
    xs = [_logits(g, B, V, f32, 2.0) for f32 in (False, True)]
    us = [torch.rand(B, generator=g) for _ in range(4)]
    want = [[R.sample_filtered(x, 0.9, u=u, top_k=30, top_p=0.9)[0] for u in us[:2]] for x in xs]
    xg, ug = [x.to(DEV) for x in xs], [u.to(DEV) for u in us]
    call = lambda i, j: K.sample_filtered(xg[i], 0.9, u=ug[j], top_k=30, top_p=0.9)[0]  # noqa: E731
    for i in range(2):
        for j in range(2):
            assert torch.equal(call(i, j).cpu(), want[i][j])
    streams, graphs, outs = [torch.cuda.Stream() for _ in range(2)], [], []
    torch.cuda.synchronize()
    for i, s in enumerate(streams):
        with torch.cuda.stream(s):
            call(i, 0)
            s.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=s):
                outs.append([call(i, j) for j in range(2)])
            graphs.append(graph)
    for _ in range(5):  # both on their way at once, and eager calls beside them
        for s, graph in zip(streams, graphs):
            with torch.cuda.stream(s):
                graph.replay()
        eager = call(0, 1)
        torch.cuda.synchronize()
        assert torch.equal(eager.cpu(), want[0][1])
        for i in range(2):
            for j in range(2):
                assert torch.equal(outs[i][j].cpu(), want[i][j])
                outs[i][j].fill_(-7)


@pytest.mark.parametrize("f32", [False, True])
@pytest.mark.parametrize("top", [None, math.inf])
def test_not_numbers_among_more_entries_than_the_list_holds(K, f32, top):
    """NaN is -inf where top-k's bin is looked for, where weights are counted, and beside infinite entries."""
    g = torch.Generator().manual_seed(21)
    B, V = 5, 9000
    x = torch.randn(B, V, generator=g) * 2
    x[torch.rand(B, V, generator=g) < 0.4] = math.nan
    if top is not None:
        x[torch.rand(B, V, generator=g) < 0.3] = top  # thousands
    x = x if f32 else x.bfloat16()
    for opts in (dict(top_k=250), dict(top_k=700, top_p=0.6), dict(top_k=2000), dict(top_p=0.9), dict()):
        for T in (0.8, 5.0):
            _same(K, x, torch.rand(B, generator=g), temperature=T, **opts)
