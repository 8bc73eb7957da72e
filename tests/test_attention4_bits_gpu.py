"""The bits that attention over the 4-bit cache keeps of its weights (csrc/cache4.hip), against the oracle in 64 bits.

Tolerance. Keys, values and queries are exact in bf16. A weight is 2^x of a score summed in fp32: with |score| <= 64 its relative
error is 64 * 2^-22 at most, 2e-5 with the exponential's own. It meets the values in two pieces of 8 bits, cut off: 2^-16 of it
is left. Sums in fp32 over the products of a wave, some dozen of them, and their join: 64 *
2^-24 = 4e-6. So what is rounded to the output is within t = 2 (2e-5 + 2^-16 + 4e-6) sum p |v| < 1e-4 sum p |v| of exact (the sum of the
weights has the same errors), and the output between the roundings of exact - t and of exact + t. Weights of 8 bits are off by up to
39e-4 sum p |v|."""
import pytest
import torch

from docagents_amd.ops import reference as R

pytestmark = pytest.mark.gpu
LENS = [2, 3, 7, 16, 33, 64, 65, 129, 300, 1000, 0, 1]


@pytest.mark.parametrize("G", [1, 2, 4, 5, 6, 8, 9, 13, 16])
@pytest.mark.parametrize("D", [64, 96, 128])
@pytest.mark.parametrize("collect", [False, True])
def test_weights_keep_their_bits(D, G, collect):
    from docagents_amd.ops import kernels as K
    g = torch.Generator().manual_seed(100 * G + D)
    Hkv, max_seq, B = 2, 1024, len(LENS)
    c = R.new_cache4(B, Hkv, max_seq, D, "cpu")
    for codes, scales in ((c.k, c.k_scale), (c.v, c.v_scale)):
        new, sc = R._encode4(torch.randn(B, Hkv, max_seq, D, generator=g).bfloat16())
        codes.copy_(new), scales.copy_(sc)
    q = torch.randn(B, Hkv * G * D, generator=g).bfloat16()
    lens, slot = torch.tensor(LENS, dtype=torch.int32), torch.randperm(B, generator=g).int()
    w = torch.zeros(B, Hkv, max_seq) if collect else None
    wg = None if w is None else w.cuda()
    got = K.decode_attn4(q.cuda(), K.Cache4(*(t.cuda() for t in c)), lens.cuda(), slot.cuda(), Hkv * G, Hkv, D, 1000, weight=wg)
    w64 = None if w is None else w.double()
    want = R.decode_attn4(q, c, lens, slot, Hkv * G, Hkv, D, weight=w64, dtype=torch.float64)
    most = R.decode_attn4(q, c._replace(v=c.v & 0x77), lens, slot, Hkv * G, Hkv, D, dtype=torch.float64)
    t, got = 1e-4 * most, got.cpu()
    outside = (got < (want - t).bfloat16()) | (got > (want + t).bfloat16())
    assert not outside.any(), (int(outside.sum()), float(((got.double() - want).abs() / most).nan_to_num(0).max()))
    if collect:
        assert ((wg.cpu().double() - w64).abs() <= 1e-4 * w64).all()


@pytest.mark.parametrize("G", [1, 8, 16])
def test_equal_values_come_back_as_they_are(G):
    """All values of a KV head's element the same: whatever the weights, the output is that value (the sum goes by the same pieces)."""
    from docagents_amd.ops import kernels as K
    g = torch.Generator().manual_seed(G)
    Hkv, D, n = 2, 128, 777
    v = torch.tensor([0.5, 1.0, 1.5, 2.0, 3.0, -4.0, 6.0, -1.0]).repeat(16).bfloat16()
    c = K.new_cache4(1, Hkv, 1024, D, "cuda")
    slot, at = torch.zeros(n, dtype=torch.int32, device="cuda"), torch.arange(n, dtype=torch.int32, device="cuda")
    K.cache4_write((3 * torch.randn(n, Hkv * D, generator=g)).bfloat16().cuda(), v.repeat(n, Hkv).cuda(), c, slot, at)
    q = torch.randn(1, Hkv * G * D, generator=g).bfloat16().cuda()
    out = K.decode_attn4(q, c, slot[:1] + n, slot[:1], Hkv * G, Hkv, D, 1024)
    assert torch.equal(out.cpu().view(-1, D), v.expand(Hkv * G, D))
