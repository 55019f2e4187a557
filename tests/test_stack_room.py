"""What a decode stack says when drafted tokens find no page or no mask bit."""
import pytest
import torch

from helix_a2a_b200.models.llama_decode import HelixDecodeStack, LlamaDecodeConfig

DEVICES = [pytest.param("cpu"), pytest.param("cuda", marks=pytest.mark.gpu)]
CFG = LlamaDecodeConfig.tiny(n_layers=2)


def tokens(rows, device, seed=0):
    gen = torch.Generator().manual_seed(seed)
    return [torch.randn(2, rows, h, 128, generator=gen).bfloat16().to(device) for h in (16, 2, 2)]


def ints(*v, device):
    return torch.tensor(v, dtype=torch.int32, device=device)


@pytest.mark.parametrize("device", DEVICES)
def test_tokens_without_a_page_are_not_forgotten(device):
    # 16 tokens and two spare pages of 16 each: 32 more tokens fit a sequence, and its neighbour's share of the free list
    stack = HelixDecodeStack(CFG, batch=2, local_ctx=16, device=device, draft_tokens=16)
    q, k, v = tokens(20, device)
    start = ints(0, 10, 20, device=device)
    for _ in range(3):                                         # 30 tokens each
        stack.commit(k, v, torch.arange(20, device=device), start)
        stack.check_room()
    stack.commit(k, v, torch.arange(20, device=device), start)
    assert int(stack.plan.missing) == 2
    # later calls that need nothing new do not hide it
    stack.commit(k, v, torch.arange(0, device=device), ints(0, 0, 0, device=device))
    with pytest.raises(RuntimeError, match="outgrown"):
        stack.check_room()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("rows,fits", [(256, True), (257, False)])
def test_tokens_without_a_mask_bit_are_not_forgotten(rows, fits, device):
    stack = HelixDecodeStack(CFG, batch=1, local_ctx=16, device=device, draft_tokens=300)
    stack.verify_step(*tokens(rows, device), ints(0, rows, device=device))
    if fits:
        stack.check_room()
    else:
        with pytest.raises(RuntimeError, match="outgrown"):
            stack.check_room()


@pytest.mark.gpu
def test_replays_count_too():
    stack = HelixDecodeStack(CFG, batch=1, local_ctx=16, draft_tokens=8)                   # 16 + 32 tokens fit
    q, k, v = tokens(8, "cuda")
    start, all_of_them = ints(0, 8, device="cuda"), torch.arange(8, device="cuda")
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            stack.commit(k, v, all_of_them, start)
        for i in range(6):
            g.replay()
            if i < 4:
                stack.check_room()
    with pytest.raises(RuntimeError, match="outgrown"):
        stack.check_room()
