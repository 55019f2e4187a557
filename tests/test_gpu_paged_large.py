"""extend_tables where sums over the sequences leave 32 bits: whole numbers, so everything is equal."""
import pytest
import torch

from helix_a2a_b200.ops import paged

pytestmark = pytest.mark.gpu
END = 2 ** 31 - 1


def ints(*v, device="cuda"):
    return torch.tensor(v, dtype=torch.int32, device=device)


def plan_of(ctx, width, free, page, device, rows_each=0):
    """Sequences of nothing but their lengths, without new tokens; the table's entries are made by the caller's device."""
    B = len(ctx)
    table, held, used = torch.zeros(B, width, dtype=torch.int32, device=device), ints(*[0] * B, device=device), ints(0, device=device)
    starts = ints(*[rows_each * i for i in range(B + 1)], device=device)
    plan = paged.extend_tables(table, held, ints(*free, device=device), used, ints(*ctx, device=device), starts, rows=rows_each * B, page_size=page)
    return plan, table, held, used


@pytest.mark.parametrize("ctx,want", [((END, END), END), ((END, END, 9), END), ((END // 2, END // 2, 4), 2 * (END // 2) + 4 - 4), ((2 ** 30, 2 ** 30, 2 ** 30, 2 ** 30), END)])
def test_missing_pages_do_not_wrap(ctx, want):
    """Pages of one token, a table of three, four free pages: all the others are missing."""
    for device in ("cuda", "cpu"):
        plan, table, held, used = plan_of(ctx, 3, (5, 6, 7, 8), 1, device)
        assert int(plan.missing) == min(want, END)
        assert held.tolist() == [3, 1] + [0] * (len(ctx) - 2) and int(used) == 4
        assert table[0].tolist() == [5, 6, 7] and table[1].tolist() == [8, 0, 0]


def test_more_pages_asked_for_than_32_bits_count():
    """Three sequences that each ask for 2^30 pages of a table that wide (13 GB): the few free ones go to the first."""
    n = 2 ** 30
    plan, table, held, used = plan_of((n, n, n), n, (5, 6, 7), 1, "cuda", rows_each=0)
    assert held.tolist() == [3, 0, 0] and int(used) == 3 and table[0, :4].tolist() == [5, 6, 7, 0] and not table[1:, :4].any()
    assert int(plan.missing) == END and plan.seq_lens.tolist() == [3, 0, 0]


@pytest.mark.parametrize("cp_size,interleave", [(1, 2 ** 28 + 1), (4, 2 ** 62), (2 ** 62, 4), (2 ** 33, 2 ** 31), (2 ** 29, 1), (2, 2 ** 28)])
def test_shares_that_leave_32_bits_are_refused(cp_size, interleave):
    """... also where their product is a small number again in 64 bits."""
    with pytest.raises(RuntimeError, match="2\\^28"):
        paged.extend_tables(torch.zeros(1, 4, dtype=torch.int32, device="cuda"), ints(0), ints(1, 2, 3), ints(0), ints(5), ints(0, 2), rows=2,
                            page_size=16, cp_size=cp_size, interleave=interleave)
