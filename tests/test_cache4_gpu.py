"""The 4-bit cache's kernels (csrc/cache4.hip) against the oracle in 64 bits, where they can go wrong.

Tolerances. Write, read and eviction move or round values exactly as defined: equal. Attention: the products' operands are exact
in bf16 but for the weights, which are rounded to it (half a step, 2^-8 of a weight's value at most, so of the output in units
of sum p |v|), and the output, rounded once more; scores are sums of D products in fp32 and turn into weights by 2^x: with
|score| <= 64 (bounded below by the inputs) an error of 64 * 2^-22 at most in the exponent, 2e-5 of a weight. So
|out - exact| <= 2^-8 |exact| + (2^-8 + 5e-5) sum p |v|. Accumulated weights stay in fp32: 1e-4 of each is far above the same 2e-5.
"""
import pytest
import torch

from docagents_amd.ops import reference as R

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(scope="module")
def K():
    from docagents_amd.ops import kernels
    return kernels


def _values(g, *shape):
    """bf16 of many magnitudes: blocks of zeros, powers of two, ties between codes, large and tiny ones."""
    x = torch.randn(*shape, generator=g) * torch.exp(2 * torch.randn(*shape[:-1], 1, generator=g))
    ties = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, -0.25, -1.75, 6.0, 7.0])[torch.randint(0, 11, shape, generator=g)]
    x = torch.where(torch.rand(*shape[:-1], 1, generator=g) < 0.3, ties, x)
    x = torch.where(torch.rand(*shape[:-1], 1, generator=g) < 0.1, torch.zeros(()), x)
    return x.bfloat16()


def _filled(K, g, slots, Hkv, max_seq, D, layers=None):
    c = K.new_cache4(slots, Hkv, max_seq, D, "cpu", layers)
    lead = c.k.shape[:-1]
    for codes, scales in ((c.k, c.k_scale), (c.v, c.v_scale)):
        new, sc = R._encode4((torch.randn(*lead, D, generator=g) * (1 + 3 * (torch.rand(D, generator=g) > 0.95))).bfloat16())
        codes.copy_(new); scales.copy_(sc)
    return c, K.Cache4(*(t.to(DEV) for t in c))


@pytest.mark.parametrize("D", [64, 96, 128])
@pytest.mark.parametrize("T,Hkv", [(1, 1), (1, 8), (37, 3), (300, 2)])
def test_write_and_read(K, D, T, Hkv):
    g = torch.Generator().manual_seed(T + D)
    slots, max_seq = 3, 320
    rows = torch.zeros(T, 2 * Hkv * D + 24).bfloat16()  # rows of another stride
    rows[:, 8:8 + 2 * Hkv * D] = _values(g, T, 2 * Hkv * (D // 32), 32).flatten(1)
    if T > 2:
        rows[1, 8] = float("inf")
        rows[2, 8 + Hkv * D + 33] = float("nan")
    slot = torch.randint(0, slots, (T,), generator=g).int()
    at = torch.randperm(max_seq, generator=g)[:T].int()
    if T > 5:
        at[3], at[4], slot[5] = -1, max_seq, slots  # outside: not written
    want = K.new_cache4(slots, Hkv, max_seq, D, "cpu")
    for t in want:
        t.fill_(77)
    got = K.Cache4(*(t.to(DEV) for t in want))
    w = torch.rand(slots, Hkv, max_seq, generator=g)
    wg = w.to(DEV)
    rg = rows.to(DEV)
    part = lambda r, i: r[:, 8 + i * Hkv * D:8 + (i + 1) * Hkv * D]  # noqa: E731
    R.cache4_write(part(rows, 0), part(rows, 1), want, slot, at, w)
    K.cache4_write(part(rg, 0), part(rg, 1), got, slot.to(DEV), at.to(DEV), wg)
    for a, b in zip(want, got):
        assert torch.equal(a, b.cpu())
    assert torch.equal(w, wg.cpu())
    for s in range(slots):
        for n in (0, 1, max_seq):
            for a, b in zip(R.cache4_read(want, s, n), K.cache4_read(got, s, n)):
                assert torch.equal(a.nan_to_num(7e7), b.cpu().nan_to_num(7e7))


def test_codes_read_as_their_values(K):
    """Every code at every scale, and the scale that marks a block as no number."""
    c = K.new_cache4(1, 1, 256, 64, "cpu")
    c.k[:] = torch.arange(256, dtype=torch.uint8).repeat(1, 1, 256, 1)[..., :32].contiguous()
    c.k[0, 0, :, :16] = torch.tensor([i | ((15 - i) << 4) for i in range(16)], dtype=torch.uint8)
    c.k_scale[0, 0, :, 0] = torch.arange(256).to(torch.uint8)
    c.k_scale[0, 0, :, 1] = 127
    k, _ = K.cache4_read(K.Cache4(*(t.to(DEV) for t in c)), 0, 256)
    want, _ = R.cache4_read(c, 0, 256)
    normal = slice(2, 253)  # 2^-125 .. 2^125: no value below the smallest normal bf16, none above the largest
    assert torch.equal(k[0, normal].cpu(), want[0, normal])
    assert k[0, 255, :32].isnan().all() and torch.equal(k[0, 255, 32:].cpu(), want[0, 255, 32:])


@pytest.mark.parametrize("H,Hkv,D", [(4, 4, 96), (8, 2, 64), (6, 1, 128)])
def test_rope_write_is_rope_cache_and_write(K, H, Hkv, D):
    g = torch.Generator().manual_seed(H)
    T, max_seq = 19, 64
    qkv = torch.randn(T, (H + 2 * Hkv) * D, generator=g).bfloat16().to(DEV)
    pos = torch.randint(0, 500, (T,), generator=g).int().to(DEV)
    cs = R.rope_table(512, D, 10000.0, DEV)
    slot, at = torch.ones(T, dtype=torch.int32, device=DEV), torch.arange(T, dtype=torch.int32, device=DEV)
    a, b = K.new_cache4(2, Hkv, max_seq, D, DEV), K.new_cache4(2, Hkv, max_seq, D, DEV)
    one = K.rope_cache4(qkv.clone(), pos, cs, H, Hkv, D, slot, at, a)
    two = K.rope_cache(qkv.clone(), pos, cs, H, Hkv, D)
    K.cache4_write(two[:, H * D:(H + Hkv) * D], two[:, (H + Hkv) * D:], b, slot, at)
    assert torch.equal(one, two)
    for x, y in zip(a, b):
        assert torch.equal(x, y)


def test_positions_outside_the_table(K):
    """Neither rotated nor written; the others are."""
    g = torch.Generator().manual_seed(8)
    H, Hkv, D = 4, 2, 64
    qkv = torch.randn(6, (H + 2 * Hkv) * D, generator=g).bfloat16()
    pos = torch.tensor([3, -1, 31, 32, 10 ** 6, 0], dtype=torch.int32)
    cs, z = R.rope_table(32, D, 10000.0), torch.zeros(6, dtype=torch.int32)
    at = torch.arange(6, dtype=torch.int32)
    c = K.new_cache4(1, Hkv, 8, D, DEV)
    got = K.rope_cache4(qkv.to(DEV), pos.to(DEV), cs.to(DEV), H, Hkv, D, z.to(DEV), at.to(DEV), c)
    bad = [1, 3, 4]
    assert torch.equal(got[bad].cpu(), qkv[bad]) and not c.k[0, :, bad].any() and not c.v_scale[0, :, bad].any()
    assert (got.cpu()[[0, 2]] != qkv[[0, 2]]).any(1).all() and all(c.k[0, 0, i].any() for i in (0, 2, 5))


def _attend(K, g, B, Hkv, G, D, lens, max_seq, max_len, pre=None, weight=False):
    H = Hkv * G
    c, cg = _filled(K, g, B + 1, Hkv, max_seq, D)
    q = torch.randn(B, H * D + 40, generator=g).bfloat16()
    lens = torch.tensor(lens, dtype=torch.int32)
    slot = torch.randperm(B + 1, generator=g)[:B].int()
    # behind a row's end lies what another sequence left: large values and blocks that are no numbers
    for b in range(B):
        n = int(lens[b])
        for t in (c.k_scale, c.v_scale):
            t[slot[b], :, n:, 0], t[slot[b], :, n:, 1] = 255, 230
    cg = K.Cache4(*(t.to(DEV) for t in c))
    w = torch.rand(c.k.shape[:3], generator=g) if weight else None
    wg = w.to(DEV) if weight else None
    if pre is not None:
        pre = torch.tensor([[pre, int(slot[0])]] * B, dtype=torch.int32)
    got = K.decode_attn4(q.to(DEV), cg, lens.to(DEV), slot.to(DEV), H, Hkv, D, max_len, pre=None if pre is None else pre.to(DEV), weight=wg)
    w64 = w.double() if weight else None
    want = R.decode_attn4(q, c, lens, slot, H, Hkv, D, pre=pre, weight=w64, dtype=torch.float64)
    absolute = c._replace(v=c.v & 0x77)  # the magnitudes of v
    most = R.decode_attn4(q, absolute, lens, slot, H, Hkv, D, pre=pre, dtype=torch.float64)
    err = (got.double().cpu() - want).abs()
    assert (err <= 2 ** -8 * want.abs() + (2 ** -8 + 5e-5) * most + 1e-30).all(), (err - 2 ** -8 * want.abs()).max()
    if weight:
        added = w64 - w.double()
        assert ((wg.cpu().double() - w64).abs() <= 1e-4 * added.abs() + 2 ** -23 * w64.abs()).all()
        for b in range(B):
            assert torch.equal(wg[slot[b], :, int(lens[b]):].cpu(), w[slot[b], :, int(lens[b]):])
    return q, cg, lens, slot, got


@pytest.mark.parametrize("D", [64, 96, 128])
@pytest.mark.parametrize("G", [1, 2, 4, 8, 16, 5])
def test_attention_of_ragged_rows(K, D, G):
    g = torch.Generator().manual_seed(D + G)
    lens = [1, 0, 2, 15, 16, 17, 31, 33, 127, 128, 129, 255, 257, 700, 511, 513]
    _attend(K, g, len(lens), 2, G, D, lens, 701, 700, weight=G in (1, 4, 5))


@pytest.mark.parametrize("Hkv,G,D,L", [(1, 8, 128, 9001), (2, 1, 96, 5000), (8, 4, 128, 1), (3, 2, 64, 2047)])
@pytest.mark.parametrize("weight", [False, True])
def test_attention_of_one_row(K, Hkv, G, D, L, weight):
    _attend(K, torch.Generator().manual_seed(L), 1, Hkv, G, D, [L], L + 3, L, weight=weight)


@pytest.mark.parametrize("D,G", [(64, 2), (96, 1), (128, 4)])
@pytest.mark.parametrize("P", [64, 448])
def test_attention_behind_a_shared_head(K, D, G, P):
    lens = [P, P + 1, P + 65, 1200, P + 300]
    _attend(K, torch.Generator().manual_seed(P + D), 5, 2, G, D, lens, 1300, 1290, pre=P)


def test_attention_of_a_capture_and_of_another_stream(K):
    """Replays give the eager call's bits, with eager calls of other sizes between them; so does a call on a stream of its own."""
    g = torch.Generator().manual_seed(3)
    q, c, lens, slot, want = _attend(K, g, 4, 2, 4, 128, [900, 1, 350, 0], 1000, 1000)
    q, lens, slot = q.to(DEV), lens.to(DEV), slot.to(DEV)
    w = torch.zeros(c.k.shape[:3], device=DEV)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        other = K.decode_attn4(q, c, lens, slot, 8, 2, 128, 1000, weight=w)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(other, want)
    graph = torch.cuda.CUDAGraph()
    w2 = torch.zeros_like(w)
    with torch.cuda.graph(graph):
        out = K.decode_attn4(q, c, lens, slot, 8, 2, 128, 1000, weight=w2)
    for i in range(3):
        graph.replay()
        K.decode_attn4(q[:1], c, lens[2:3], slot[2:3], 8, 2, 128, 500)
        torch.cuda.synchronize()
        assert torch.equal(out, want)
    assert torch.allclose(w2, 3 * w, rtol=1e-5, atol=0)


@pytest.mark.parametrize("layers", [None, 3])
@pytest.mark.parametrize("inplace", [True, False])
@pytest.mark.parametrize("D,keep,recent", [(64, 1, 0), (96, 100, 100), (128, 700, 64), (64, 0, 0), (128, 2500, 2000), (96, 5000, 3)])
def test_evict(K, layers, inplace, D, keep, recent):
    g = torch.Generator().manual_seed(keep + D)
    lens = torch.tensor([3000, 0, 1, 701, 1500, 101], dtype=torch.int32)
    B, Hkv, max_seq = len(lens), 2, 3001
    c, cg = _filled(K, g, 2 * B, Hkv, max_seq, D, layers)
    w = torch.rand(c.k.shape[:-1], generator=g)
    w = torch.where(w < 0.5, (w * 16).floor() / 16, w)  # half of them equal to others
    w[..., 5], w[..., 7], w[..., 9], w[..., 11] = float("nan"), float("inf"), -0.0, 0.0
    slots = torch.randperm(2 * B, generator=g).int()
    slot, to = slots[:B], None if inplace else slots[B:]
    wg = w.to(DEV)
    n = K.cache4_evict(cg, wg, lens.to(DEV), slot.to(DEV), keep, recent, to=None if inplace else to.to(DEV))
    want_n = R.cache4_evict(c, w, lens, slot, keep, recent, to)
    assert torch.equal(n.cpu(), want_n)
    for a, b in zip((*c, w.view(torch.int32)), (*cg, wg.view(torch.int32))):
        assert torch.equal(a, b.cpu())


def test_places_past_32_bits(K):
    """A cache whose bytes and rows pass 2^31: the last slot's places."""
    Hkv, D, max_seq, slots = 8, 128, 65536, 70  # 2.3e9 bytes of codes
    c = K.new_cache4(slots, Hkv, max_seq, D, DEV)
    g = torch.Generator().manual_seed(1)
    T = 300
    kv = torch.randn(T, 2 * Hkv * D, generator=g).bfloat16().to(DEV)
    s, at = torch.full((T,), slots - 1, dtype=torch.int32, device=DEV), torch.arange(T, dtype=torch.int32, device=DEV)
    K.cache4_write(kv[:, :Hkv * D], kv[:, Hkv * D:], c, s, at)
    small = K.new_cache4(1, Hkv, 512, D, DEV)
    K.cache4_write(kv[:, :Hkv * D], kv[:, Hkv * D:], small, s * 0, at)
    for a, b in zip(K.cache4_read(c, slots - 1, T), K.cache4_read(small, 0, T)):
        assert torch.equal(a, b)
    q = torch.randn(1, 32 * D, generator=g).bfloat16().to(DEV)
    n = torch.tensor([T], dtype=torch.int32, device=DEV)
    assert torch.equal(K.decode_attn4(q, c, n, s[:1], 32, Hkv, D, 512), K.decode_attn4(q, small, n, s[:1] * 0, 32, Hkv, D, 512))
    w = torch.rand(slots, Hkv, max_seq, device=DEV)
    ws = w[-1:, :, :512].contiguous()
    assert torch.equal(K.cache4_evict(c, w, n, s[:1], 100, 10), K.cache4_evict(small, ws, n, s[:1] * 0, 100, 10))
    for a, b in zip(K.cache4_read(c, slots - 1, 100), K.cache4_read(small, 0, 100)):
        assert torch.equal(a, b)
    assert torch.equal(w[-1, :, :100], ws[0, :, :100])


def test_what_is_refused(K):
    c = K.new_cache4(2, 2, 64, 64, DEV)
    i = torch.zeros(4, dtype=torch.int32, device=DEV)
    x = torch.zeros(4, 128, device=DEV).bfloat16()
    w = torch.zeros(2, 2, 64, device=DEV)
    q = torch.zeros(4, 256, device=DEV).bfloat16()
    bad = [lambda: K.cache4_write(x.float(), x, c, i, i), lambda: K.cache4_write(x, x[:2], c, i, i), lambda: K.cache4_write(x, x, c, i[:3], i),
           lambda: K.cache4_write(x, x, c, i.long(), i), lambda: K.cache4_write(x[:, :64], x, c, i, i), lambda: K.cache4_write(x.cpu(), x, c, i, i),
           lambda: K.cache4_write(x, x, c, i, i, weight=w[:1]), lambda: K.cache4_write(x, x, c._replace(k=c.k[:, :1]), i, i),
           lambda: K.cache4_write(x, x, c._replace(k_scale=c.k_scale[..., :2]), i, i),
           lambda: K.cache4_write(x.view(-1)[4:388].view(3, 128), x[:3], c, i, i),
           lambda: K.cache4_read(c, 2, 1), lambda: K.cache4_read(c, 0, 65), lambda: K.cache4_read(c, -1, 1),
           lambda: K.decode_attn4(q, c, i, i, 4, 2, 128, 64), lambda: K.decode_attn4(q, c, i, i, 3, 2, 64, 64),
           lambda: K.decode_attn4(q, c, i, i, 4, 2, 64, 65), lambda: K.decode_attn4(q, c, i, i, 4, 2, 64, 0),
           lambda: K.decode_attn4(q, c, i[:3], i, 4, 2, 64, 64), lambda: K.decode_attn4(q, c, i, i, 68, 2, 64, 64),
           lambda: K.decode_attn4(q, c, i, i, 4, 2, 64, 64, weight=w, pre=torch.zeros(4, 2, dtype=torch.int32, device=DEV)),
           lambda: K.decode_attn4(q, c, i, i, 4, 2, 64, 64, weight=w.half()), lambda: K.decode_attn4(q, c, i, i, 4, 2, 64, 64, out=q[:, :128]),
           lambda: K.cache4_evict(c, w, i, i, 4, 5), lambda: K.cache4_evict(c, w, i, i, 4, 2, above=3), lambda: K.cache4_evict(c, w, i, i[:2], 4, 2),
           lambda: K.cache4_evict(c, w, i, i, 4, 2, out=i), lambda: K.cache4_evict(c, w[:, :1], i, i, 4, 2)]
    for n, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            print("not refused:", n)
    assert K.decode_attn4(q[:0], c, i[:0], i[:0], 4, 2, 64, 64).shape == (0, 256)
    K.cache4_write(x[:0], x[:0], c, i[:0], i[:0])
    assert K.cache4_evict(c, w, i[:0], i[:0], 4, 2).numel() == 0


def test_new_lengths_do_not_lie_over_the_old_ones(K):
    c, w = K.new_cache4(2, 2, 64, 64, DEV), torch.zeros(2, 2, 64, device=DEV)
    x, slot = torch.tensor([8, 9, 7], dtype=torch.int32, device=DEV), torch.tensor([1, 0], dtype=torch.int32, device=DEV)
    for lens, out in ((x[:2], x[1:]), (x[1:], x[:2])):
        with pytest.raises(ValueError, match="apart from lens"):
            K.cache4_evict(c, w, lens, slot, 4, 2, out=out)
    assert x.tolist() == [8, 9, 7]


def test_evict_leaves_sequences_below_the_line(K):
    g = torch.Generator().manual_seed(4)
    c, cg = _filled(K, g, 3, 1, 300, 64)
    w = torch.rand(3, 1, 300, generator=g)
    lens, slot = torch.tensor([150, 200, 201], dtype=torch.int32), torch.tensor([2, 0, 1], dtype=torch.int32)
    wg = w.to(DEV)
    n = K.cache4_evict(cg, wg, lens.to(DEV), slot.to(DEV), 100, 10, above=200)
    want = R.cache4_evict(c, w, lens, slot, 100, 10, above=200)
    assert n.tolist() == want.tolist() == [150, 200, 100]
    for a, b in zip((*c, w), (*cg, wg)):
        assert torch.equal(a, b.cpu())


def test_blocks_that_are_no_numbers_stay_with_their_row(K):
    """A key's block: its KV head's query heads of that row; a value's: 32 of their elements. Nothing else."""
    g = torch.Generator().manual_seed(6)
    c, cg = _filled(K, g, 3, 2, 200, 128)
    for t in (c.k_scale, cg.k_scale):
        t[0, 1, 77, 2] = 255
    for t in (c.v_scale, cg.v_scale):
        t[1, 0, 130, 3] = 255
    q = torch.randn(3, 8 * 128, generator=g).bfloat16()
    lens, slot = torch.tensor([150, 150, 150], dtype=torch.int32), torch.tensor([0, 1, 2], dtype=torch.int32)
    got = K.decode_attn4(q.to(DEV), cg, lens.to(DEV), slot.to(DEV), 8, 2, 128, 200).cpu().view(3, 8, 128)
    want = torch.zeros(3, 8, 128, dtype=torch.bool)
    want[0, 4:] = True
    want[1, :4, 96:] = True
    assert torch.equal(got.isnan(), want)


@pytest.mark.parametrize("scale", [-0.1, 0.0, 0.5])
def test_any_scale(K, scale):
    g = torch.Generator().manual_seed(7)
    c, cg = _filled(K, g, 2, 2, 300, 64)
    q = torch.randn(2, 4 * 64, generator=g).bfloat16()
    lens, slot = torch.tensor([300, 41], dtype=torch.int32), torch.tensor([1, 0], dtype=torch.int32)
    got = K.decode_attn4(q.to(DEV), cg, lens.to(DEV), slot.to(DEV), 4, 2, 64, 300, scale=scale).cpu().double()
    want = R.decode_attn4(q, c, lens, slot, 4, 2, 64, scale=scale, dtype=torch.float64)
    most = R.decode_attn4(q, c._replace(v=c.v & 0x77), lens, slot, 4, 2, 64, scale=scale, dtype=torch.float64)
    assert ((got - want).abs() <= 2 ** -8 * want.abs() + (2 ** -8 + 5e-5) * most).all()


def test_rows_without_a_slot_give_zeros(K):
    c = K.new_cache4(2, 1, 64, 128, DEV)
    q = torch.randn(3, 128, device=DEV).bfloat16()
    n, s = torch.tensor([5, 64, 0], dtype=torch.int32, device=DEV), torch.tensor([-1, 2, 0], dtype=torch.int32, device=DEV)
    assert not K.decode_attn4(q, c, n, s, 1, 1, 128, 64).any()
