"""4-bit o_proj of a few tokens with a K that clusters of four and eight CTAs share, at heights whose row tiles the resident clusters
do not divide evenly.  Tolerance: as for every other shape, which ``test_gpu_int4.check`` states."""
import pytest
import torch

from helix_a2a_b200.ops import oproj
from test_gpu_int4 import check, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("tokens", [1, 8, 9, 16])
@pytest.mark.parametrize("hidden,K,group", [(4096, 11008, 128), (4096, 14336, 128), (4096, 16384, 128), (576, 16384, 128), (4736, 16384, 64),
                                            (288, 32768, 64), (544, 28672, 128), (2304, 32768, 32)])
def test_shapes(hidden, K, group, tokens):
    w, full = make(hidden, K, group, True, torch.bfloat16, seed=K)
    x = torch.randn(tokens, K, device="cuda").bfloat16()
    y = check(x, w, full)
    assert all(torch.equal(y, oproj.oproj(x, w)) for _ in range(3))
