"""extend_tables / append_kv on CPU tensors: the oracle against its definition, and the refusals of the Python layer."""
import pytest
import torch

from helix_a2a_b200.ops import paged, reference_math as rm


def ints(*v):
    return torch.tensor(v, dtype=torch.int32)


@pytest.mark.parametrize("cp,il", [(1, 1), (2, 1), (4, 16), (3, 5)])
def test_local_tokens_counts_what_a_rank_holds(cp, il):
    for rank in range(cp):
        held = 0
        for n in range(4 * cp * il + 3):
            assert rm.local_tokens(n, cp, rank, il) == held
            held += n // il % cp == rank
    assert all(sum(rm.local_tokens(n, cp, r, il) for r in range(cp)) == n for n in range(200))


def test_tree_mask_and_positions():
    # -1 -> 0 -> 1 -> 3, 0 -> 2, -1 -> 4
    table, held, used = torch.zeros(1, 4, dtype=torch.int32), ints(1), ints(0)
    plan = paged.extend_tables(table, held, ints(7, 9, 5), used, ints(3), ints(0, 5), rows=6, page_size=4,
                               parents=ints(-1, 0, 0, 1, -1, -1))
    assert plan.mask.flatten().tolist() == [0b1, 0b11, 0b101, 0b1011, 0b10000, 0]
    assert plan.positions.tolist() == [3, 4, 4, 5, 3, 0]
    assert table[0].tolist() == [0, 7, 0, 0] and held.item() == 2 and used.item() == 1
    assert plan.slots.tolist() == [3, 28, 29, 30, 31, -1]
    assert plan.seq_lens.item() == 8 and plan.draft_lens.item() == 5 and plan.missing.item() == 0


def test_ranks_share_the_tokens():
    n0, t, cp = 11, 9, 3
    seen = []
    for rank in range(cp):
        plan = paged.extend_tables(torch.zeros(1, 4, dtype=torch.int32), ints(0), torch.arange(4, dtype=torch.int32), ints(0), ints(n0),
                                   ints(0, t), rows=t, page_size=16, cp_size=cp, cp_rank=rank, interleave=2)
        own = [j for j in range(t) if plan.slots[j] >= 0]
        seen += own
        assert int(plan.draft_lens) == len(own)
        # a chain: the last token sees every local one
        assert int(plan.mask[-1, 0]) == 2 ** len(own) - 1
    assert sorted(seen) == list(range(t))


def test_pages_run_out_in_order():
    table, held, used = torch.zeros(3, 2, dtype=torch.int32), ints(0, 0, 0), ints(1)
    plan = paged.extend_tables(table, held, ints(90, 91, 92, 93), used, ints(0, 0, 0), ints(0, 20, 30, 70), rows=70, page_size=8)
    assert held.tolist() == [2, 1, 0] and used.item() == 4
    assert plan.missing.item() == 1 + 1 + 5
    assert plan.seq_lens.tolist() == [16, 8, 0]
    assert [(plan.slots[a:b] >= 0).sum().item() for a, b in ((0, 20), (20, 30), (30, 70))] == [16, 8, 0]


@pytest.mark.parametrize("layout", ["HND", "NHD"])
def test_append_on_cpu(layout):
    shape = (3, 2, 4, 16) if layout == "HND" else (3, 4, 2, 16)
    kc, vc = torch.zeros(shape), torch.zeros(shape)
    k, v = torch.randn(4, 2, 16), torch.randn(4, 2, 16)
    paged.append_kv(k, v, kc, vc, torch.tensor([9, -1, 0, 12]), layout=layout)
    kn, vn = (c.transpose(1, 2) if layout == "HND" else c for c in (kc, vc))
    assert torch.equal(kn[2, 1], k[0]) and torch.equal(vn[0, 0], v[2])
    assert kc.abs().sum() == k[[0, 2]].abs().sum() or torch.isclose(kc.abs().sum(), k[[0, 2]].abs().sum())
    with pytest.raises(ValueError):
        paged.append_kv(k, v, kc, vc, torch.tensor([0, 1, 2, 3]), layout="DHN")
