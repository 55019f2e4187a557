"""extend_tables / append_kv on the GPU against the token-by-token oracle: whole numbers and copies, so everything is equal."""
import numpy as np
import pytest
import torch

from helix_a2a_b200.ops import paged, reference_math as rm

pytestmark = pytest.mark.gpu


def ints(v):
    return torch.tensor(np.asarray(v), dtype=torch.int32)


def make(seed, batch, new, ctx, page, cp, il, tree, pad=0, spare=8, max_pages=None):
    rng = np.random.default_rng(seed)
    counts = rng.integers(0, new + 1, batch)
    counts[rng.random(batch) < 0.1] = 0
    lens = rng.integers(0, ctx + 1, batch)
    rank = int(rng.integers(cp))
    local = [rm.local_tokens(int(n), cp, rank, il) for n in lens]
    need = [-(-rm.local_tokens(int(n + t), cp, rank, il) // page) for n, t in zip(lens, counts)]
    held = [min(w, -(-n // page) + int(rng.random() < 0.3)) for n, w in zip(local, need)]
    width = max(need + [1]) + 1 if max_pages is None else max_pages
    held = [min(h, width) for h in held]
    ids = rng.permutation(sum(need) + max(spare, 0) + batch)
    table = np.full((batch, width), 12345, dtype=np.int32)
    at = 0
    for b, h in enumerate(held):
        table[b, :h] = ids[at:at + h]
        at += h
    free = ids[at:at + max(sum(need) - at + spare, 0)]
    rows = int(counts.sum()) + pad
    parents = None
    if tree:
        parents = np.concatenate([np.maximum(-1, np.arange(c) - 1 - rng.integers(0, 3, c)) for c in counts] + [np.full(pad, -1)])
    state = dict(block_table=ints(table), held=ints(held), free_pages=ints(free), free_used=ints([0]))
    return state, dict(ctx_lens=ints(lens), q_start=ints(np.concatenate([[0], np.cumsum(counts)]))), dict(
        rows=rows, page_size=page, parents=ints(parents) if tree else None, cp_size=cp, cp_rank=rank, interleave=il)


def run(state, lens, kw, device):
    state = {k: v.clone().to(device) for k, v in state.items()}
    kw = dict(kw, parents=kw["parents"].to(device) if kw["parents"] is not None else None)
    plan = paged.extend_tables(state["block_table"], state["held"], state["free_pages"], state["free_used"], lens["ctx_lens"].to(device),
                               lens["q_start"].to(device), **kw)
    return plan, state


def same(a, b):
    for name, x, y in zip(paged.TablePlan._fields, a[0], b[0]):
        assert x.dtype == y.dtype and torch.equal(x.cpu(), y.cpu()), name
    for k in a[1]:
        assert torch.equal(a[1][k].cpu(), b[1][k].cpu()), k


CASES = [
    dict(batch=1, new=1, ctx=0, page=16, cp=1, il=1, tree=False),
    dict(batch=1, new=16, ctx=300, page=16, cp=1, il=1, tree=True),
    dict(batch=7, new=33, ctx=500, page=32, cp=4, il=16, tree=True, pad=5),
    dict(batch=65, new=64, ctx=4000, page=16, cp=2, il=1, tree=True),
    dict(batch=40, new=64, ctx=1000, page=64, cp=8, il=3, tree=False, pad=3),
    dict(batch=513, new=9, ctx=700, page=16, cp=3, il=5, tree=True),
    dict(batch=600, new=12, ctx=90, page=7, cp=1, il=1, tree=False),
    dict(batch=5, new=2500, ctx=100, page=16, cp=1, il=1, tree=False, pad=100),
    dict(batch=20, new=40, ctx=100, page=16, cp=1, il=1, tree=True, spare=-25),           # the free list runs out
    dict(batch=20, new=40, ctx=100, page=16, cp=2, il=1, tree=False, spare=-300),         # ... before the first sequence
    dict(batch=12, new=60, ctx=300, page=16, cp=1, il=1, tree=True, max_pages=9),         # sequences outgrow the table
    dict(batch=0, new=3, ctx=5, page=16, cp=1, il=1, tree=False, pad=2),
    dict(batch=3, new=0, ctx=50, page=16, cp=1, il=1, tree=True),
]


@pytest.mark.parametrize("words", [0, 1, 4])
@pytest.mark.parametrize("case", CASES, ids=range(len(CASES)))
def test_tables_equal_the_oracle(case, words):
    args = make(words + 1, **case)
    args[2]["mask_words"] = words
    want = run(*args, "cpu")
    got = run(*args, "cuda")
    same(got, want)


def test_tables_of_more_nodes_than_mask_bits():
    state, lens, kw = make(3, 3, 300, 64, 16, 1, 1, True)
    kw["mask_words"] = 4
    assert int(lens["q_start"].diff().max()) > 256 - 64
    same(run(state, lens, kw, "cuda"), run(state, lens, kw, "cpu"))


def test_tables_largest_batch_and_second_call():
    state, lens, kw = make(5, 8192, 3, 50, 16, 2, 1, False)
    want, got = run(state, lens, kw, "cpu"), run(state, lens, kw, "cuda")
    same(got, want)
    same(run(got[1], lens, kw, "cuda"), (want[0][:5] + (torch.zeros(1, dtype=torch.int32),), want[1]))     # nothing left to take


def test_tables_walk_of_malformed_parents_ends():
    state, lens, kw = make(1, 4, 40, 100, 16, 1, 1, True)
    kw["parents"] = torch.randint(-5, 60, kw["parents"].shape, dtype=torch.int32)
    same(run(state, lens, kw, "cuda"), run(state, lens, kw, "cpu"))


@pytest.mark.parametrize("words,cp", [(4, 1), (2, 4), (0, 8)])
def test_a_tree_of_many_nodes(words, cp):
    """Walks to the root of a long chain go on where the warp has been."""
    state, lens, kw = make(words, 3, 1500, 40, 16, cp, 1, True, spare=9)
    kw = dict(kw, mask_words=words)
    same(run(state, lens, kw, "cuda"), run(state, lens, kw, "cpu"))


@pytest.mark.parametrize("tree", [False, True])
def test_lengths_at_the_end_of_32_bits(tree):
    state = dict(block_table=ints([[3, 4, 5], [6, 7, 8]]), held=ints([2, 1]), free_pages=ints([9, 10, 11]), free_used=ints([0]))
    lens = dict(ctx_lens=ints([2**31 - 3, 20]), q_start=ints([0, 8, 16]))
    plan, after = run(state, lens, dict(rows=20, page_size=16, parents=ints(np.arange(20) - 1 - 8 * (np.arange(20) >= 8)) if tree else None), "cuda")
    # the first sequence takes what its table has room for, the second one needs a page
    assert after["block_table"].tolist() == [[3, 4, 9], [6, 10, 8]] and after["held"].tolist() == [3, 2]
    assert plan.slots.tolist() == [-1] * 8 + [10 * 16 + 4 + i for i in range(8)] + [-1] * 4
    assert int(plan.missing) > 0 and plan.seq_lens.tolist() == [48, 28] and plan.draft_lens.tolist() == [0, 8]


def test_tables_in_a_graph_carry_their_state():
    """Replays of one captured call see what the replay before them took, as calls one after the other do."""
    state, lens, kw = make(9, 30, 20, 200, 16, 1, 1, True, spare=400)
    dev = {k: v.cuda() for k, v in state.items()}
    at = {k: v.cuda() for k, v in lens.items()}
    args = (dev["block_table"], dev["held"], dev["free_pages"], dev["free_used"], at["ctx_lens"], at["q_start"])
    kw = dict(kw, parents=kw["parents"].cuda())
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            plan = paged.extend_tables(*args, **kw)
        for _ in range(3):
            g.replay()
            want = run(state, lens, kw | dict(parents=kw["parents"].cpu()), "cpu")
            s.synchronize()
            same((plan, dev), want)
            lens = dict(lens, ctx_lens=lens["ctx_lens"] + 13)
            state = want[1]
            at["ctx_lens"].copy_(lens["ctx_lens"])


def test_tables_refusals():
    state, lens, kw = make(1, 4, 8, 50, 16, 1, 1, True)
    good = dict({k: v.cuda() for k, v in state.items()}, **{k: v.cuda() for k, v in lens.items()})
    kw = dict(kw, parents=kw["parents"].cuda())

    def call(**over):
        a = dict(good, **{k: v for k, v in over.items() if k in good})
        return paged.extend_tables(*a.values(), **dict(kw, **{k: v for k, v in over.items() if k not in good}))

    call()
    for bad in (dict(held=good["held"].long()), dict(held=good["held"][:3]), dict(q_start=good["q_start"][:4]), dict(free_used=good["held"]),
                dict(ctx_lens=good["ctx_lens"].cpu()), dict(parents=kw["parents"][:-1]), dict(mask_words=5), dict(mask_words=-1),
                dict(page_size=0), dict(cp_rank=1), dict(cp_size=0), dict(interleave=0), dict(block_table=good["block_table"].t()),
                dict(rows=-1), dict(free_pages=good["free_pages"].float()),
                dict(rows=2**20 + 1, parents=torch.zeros(2**20 + 1, dtype=torch.int32, device="cuda")), dict(rows=2**30)):
        with pytest.raises(RuntimeError):
            call(**bad)


@pytest.mark.parametrize("rows", [0, 1, 37, 5000])
@pytest.mark.parametrize("layout,heads,dim,dtype", [("HND", 8, 128, torch.bfloat16), ("NHD", 1, 128, torch.float16), ("HND", 3, 64, torch.float32),
                                                    ("NHD", 32, 128, torch.bfloat16), ("HND", 2, 16, torch.uint8), ("NHD", 5, 8, torch.float16)])
def test_append_writes_rows_and_nothing_else(rows, layout, heads, dim, dtype):
    torch.manual_seed(rows)
    page, pool = 16, rows // 8 + 3
    shape = (pool, heads, page, dim) if layout == "HND" else (pool, page, heads, dim)

    def make(*s):
        return torch.randint(0, 100, s, device="cuda").to(dtype)

    kc, vc, qkv = make(*shape), make(*shape), make(rows, 3, heads, dim)
    k, v = qkv[:, 1], qkv[:, 2]                                                           # strided rows
    slots = torch.randperm(pool * page, device="cuda")[:rows]
    if rows > 4:
        slots[::5] = -1
        slots[1::7] = pool * page + torch.arange(len(slots[1::7]), device="cuda")          # behind the cache: left out
        slots[2] = -(1 << 40)
    want = [c.clone() for c in (kc, vc)]
    keep = (slots >= 0) & (slots < pool * page)
    for c, x in zip(want, (k, v)):
        view = c.transpose(1, 2) if layout == "HND" else c
        view[slots[keep] // page, slots[keep] % page] = x[keep]
    paged.append_kv(k, v, kc, vc, slots, layout=layout)
    assert torch.equal(kc, want[0]) and torch.equal(vc, want[1])


def test_append_into_views_of_a_larger_cache_on_another_stream():
    both = torch.zeros(9, 2, 4, 16, 128, dtype=torch.bfloat16, device="cuda")              # K and V of a page together
    kc, vc = both[:, 0], both[:, 1]
    k, v = torch.randn(2, 20, 4, 128, device="cuda").bfloat16()
    slots = torch.randperm(9 * 16, device="cuda")[:20]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        paged.append_kv(k, v, kc, vc, slots)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(kc.transpose(1, 2)[slots // 16, slots % 16], k) and torch.equal(vc.transpose(1, 2)[slots // 16, slots % 16], v)
    assert int((both != 0).any(-1).sum()) == 2 * 20 * 4


def test_append_offsets_beyond_32_bits():
    """A cache of 4.6 GB: byte offsets of its last pages do not fit 32 bits."""
    pool, page = 35000, 16
    kc = torch.zeros(pool, 4, page, 1024, dtype=torch.uint8, device="cuda")
    vc = torch.zeros_like(kc)
    k, v = torch.randint(1, 255, (2, 8, 4, 1024), dtype=torch.uint8, device="cuda")
    slots = pool * page - 1 - 3 * torch.arange(8, device="cuda")
    paged.append_kv(k, v, kc, vc, slots)
    assert torch.equal(kc.transpose(1, 2)[slots // page, slots % page], k) and torch.equal(vc.transpose(1, 2)[slots // page, slots % page], v)
    assert not kc[:pool - 3].any() and not vc[:pool - 3].any()


def test_append_refusals():
    kc = torch.zeros(4, 2, 16, 128, dtype=torch.bfloat16, device="cuda")
    vc, k = kc.clone(), torch.zeros(5, 2, 128, dtype=torch.bfloat16, device="cuda")
    slots = torch.arange(5, device="cuda")
    paged.append_kv(k, k, kc, vc, slots)
    odd = torch.zeros(5, 2, 129, dtype=torch.bfloat16, device="cuda")[..., 1:]
    for args in ((k.half(), k, kc, vc, slots), (k, k[:4], kc, vc, slots), (k, k, kc, vc[:3], slots), (k, k, kc, vc, slots.int()),
                 (k, k, kc, vc, slots[:4]), (k[:, :1], k[:, :1], kc, vc, slots), (odd, k, kc, vc, slots), (k, k, kc, vc, slots.cpu()),
                 (k[..., ::2], k[..., ::2], kc[..., :64], vc[..., :64], slots), (k[..., :4], k[..., :4], kc[..., :4], vc[..., :4], slots)):
        with pytest.raises(RuntimeError):
            paged.append_kv(*args)


def test_append_to_slots_behind_32_bits():
    """A cache of 2^33 slots whose pages all lie on one another."""
    one = [torch.zeros(1, 2, 16, 8, dtype=torch.float16, device="cuda") for _ in range(2)]
    k, v = torch.randn(2, 3, 2, 8, device="cuda").half()
    slots = torch.tensor([2**32 + 5, 2**33 - 1, 2**33], device="cuda")
    paged.append_kv(k, v, one[0].expand(2**29, -1, -1, -1), one[1].expand(2**29, -1, -1, -1), slots)
    for c, x in zip(one, (k, v)):
        want = torch.zeros_like(c)
        want[0, :, 5], want[0, :, 15] = x[0], x[1]
        assert torch.equal(c, want)
