"""Eviction: where the new lengths may not go."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_new_lengths_lie_over_no_input():
    """Workgroups read lengths and slots while others write the new lengths: what lies over either is refused by the host."""
    from docagents_amd.ops import kernels as K
    c, w = K.new_cache4(4, 2, 64, 64, "cuda"), torch.zeros(4, 2, 64, device="cuda")
    x = torch.tensor([8, 9, 0, 1, 2, 3, 7, 7], dtype=torch.int32, device="cuda")
    lens, slot, to = x[0:2], x[2:4], x[4:6]
    for out in (x[0:2], x[1:3], x[2:4], x[3:5], x[5:7]):
        with pytest.raises(ValueError, match="apart from lens"):
            K.cache4_evict(c, w, lens, slot, 4, 2, to=to, out=out)
    assert x.tolist() == [8, 9, 0, 1, 2, 3, 7, 7]
    assert K.cache4_evict(c, w, lens, slot, 4, 2, to=to, out=x[6:8]).tolist() == [4, 4]
    assert K.cache4_evict(c, w, lens, slot, 4, 2, out=x[4:6]).tolist() == [4, 4]  # (no ``to`` there)
