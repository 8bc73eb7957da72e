"""Filtered sampling: which rows go in one launch is decided in one place, and rows on either side of each border are the oracle's."""
import pytest
import torch

from docagents_amd.ops import reference as R

pytestmark = pytest.mark.gpu


# a workgroup has 8185 entries of a row and 8192 more for each other one (entries before the first 16 bytes count)
@pytest.mark.parametrize("V,B,tickets", [(8185, 256, 0), (8185, 257, 0), (8186, 32, 32), (8186, 33, 0), (16377, 32, 32), (16371, 22, 22),
                                         (16377, 33, 0), (16378, 21, 21), (16378, 22, 0), (1, 1, 0), (128256, 4, 4), (128256, 5, 0)])
def test_rows_of_one_launch(V, B, tickets):
    from docagents_amd.ops import kernels as K
    assert K._filtered_plan(B, V)[1] == tickets
    g = torch.Generator().manual_seed(V + B)
    x = (2 * torch.randn(B, V + 9, generator=g)).bfloat16()
    u = torch.rand(B, generator=g)
    xg = x.cuda()
    for lead in (0, 7):  # rows at 16 bytes, and with a first entry just before
        tok, lp = K.sample_filtered(xg[:, lead:lead + V], 0.9, top_k=30, top_p=0.95, u=u.cuda())
        want, wl = R.sample_filtered(x[:, lead:lead + V], 0.9, top_k=30, top_p=0.95, u=u)
        assert torch.equal(tok.cpu(), want)
        # exponentials in fp32 of differences up to 60: 5e-6 of what a log-probability is
        assert ((lp.cpu() - wl).abs() <= 1e-5 * wl.abs() + 1e-30).all()
