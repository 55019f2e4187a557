"""The most tokens of a step, as the caller of a decode stack knows them: masks and the division of the attention go by it."""
import pytest
import torch

from helix_a2a_b200.models.llama_decode import HelixDecodeStack, LlamaDecodeConfig
from helix_a2a_b200.ops import attention

DEVICES = [pytest.param("cpu"), pytest.param("cuda", marks=pytest.mark.gpu)]
CFG = LlamaDecodeConfig.tiny(n_layers=2)


def tokens(rows, device, seed=0):
    gen = torch.Generator().manual_seed(seed)
    return [torch.randn(2, rows, h, 128, generator=gen).bfloat16().to(device) for h in (16, 2, 2)]


def ints(*v, device):
    return torch.tensor(v, dtype=torch.int32, device=device)


@pytest.mark.parametrize("device", DEVICES)
def test_more_tokens_than_the_caller_said(device):
    stack = HelixDecodeStack(CFG, batch=2, local_ctx=16, device=device, draft_tokens=100)
    data = tokens(90, device)
    y = stack.verify_step(*data, ints(0, 20, 84, device=device), max_new=20)               # 64 of a sequence: still a bit for each
    stack.check_room()
    assert torch.equal(y, stack.verify_step(*data, ints(0, 20, 84, device=device)))
    stack.verify_step(*data, ints(0, 20, 85, device=device), max_new=20)
    with pytest.raises(RuntimeError, match="outgrown"):
        stack.check_room()


@pytest.mark.parametrize("device", DEVICES)
def test_the_step_is_divided_by_its_own_tokens(device, monkeypatch):
    """A stack that is to grow by 2000 tokens, five at a time."""
    stack = HelixDecodeStack(CFG, batch=3, local_ctx=40, device=device, draft_tokens=2000)
    data, start = tokens(15, device), ints(0, 5, 10, 15, device=device)
    seen, call = [], attention.tree_decode

    def spy(*args, **kw):
        seen.append((args[7].shape[1], kw["max_q_len"]))
        return call(*args, **kw)

    monkeypatch.setattr(attention, "tree_decode", spy)
    y = stack.verify_step(*data, start, max_new=5)
    assert seen == [(1, 5)] * 2
    assert torch.equal(y, stack.verify_step(*data, start))              # 40 and 120 rows of a KV head: the same division
    assert seen[2:] == [(1, 15)] * 2


def test_refusals():
    stack = HelixDecodeStack(CFG, batch=1, local_ctx=16, device="cpu", draft_tokens=300)
    data, start = tokens(4, "cpu"), ints(0, 4, device="cpu")
    for bad in (-1, 257, 301):
        with pytest.raises(ValueError):
            stack.verify_step(*data, start, max_new=bad)
    stack = HelixDecodeStack(CFG, batch=1, local_ctx=16, device="cpu", draft_tokens=10)
    with pytest.raises(ValueError):
        stack.verify_step(*data, start, max_new=11)
