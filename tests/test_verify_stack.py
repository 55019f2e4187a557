"""Drafted tokens through the decode stack: tables, cache writes, tree attention and o_proj together, as they are used.

A plain float64 pass over the same tokens gives o and A = sum_j p_j |v_j|.  The stack's o is off by at most e (A + |o|) + 2e-4 A with e = eps / 2
of bf16 (P and o are rounded), so y = o w^T by at most that times |w|, plus its own rounding e |y| and K fp32 additions.
"""
import math

import pytest
import torch

from helix_a2a_b200 import api, lse_combine
from helix_a2a_b200.models.llama_decode import HelixDecodeStack, LlamaDecodeConfig
from helix_a2a_b200.ops import attention, oproj, paged

E = 2.0 ** -8
DEVICES = [pytest.param("cpu"), pytest.param("cuda", marks=pytest.mark.gpu)]
CFG = LlamaDecodeConfig.tiny(n_layers=2)


def trees(counts, gen):
    par = []
    for c in counts:
        par += [int(torch.randint(-1, j, (1,), generator=gen)) if j else -1 for j in range(c)]
    return torch.tensor(par, dtype=torch.int32)


def plain(q, k, v, seen):
    """q [t, Hq, D], k / v [n, Hkv, D], seen [t, n] -> o, A [t, Hq, D] in float64."""
    g = q.shape[1] // k.shape[1]
    x = torch.einsum("thd,nhd->thn", q.double(), k.double().repeat_interleave(g, 1)) / math.sqrt(q.shape[-1])
    p = torch.softmax(x.masked_fill(~seen[:, None], -math.inf), -1)
    vd = v.double().repeat_interleave(g, 1)
    return torch.einsum("thn,nhd->thd", p, vd), torch.einsum("thn,nhd->thd", p, vd.abs())


def check(y, o, a, w):
    w = w.double()
    k = w.shape[1]
    want = o.flatten(1) @ w.t()
    d_o = (E * (a + o.abs()) + 2e-4 * a).flatten(1)
    tol = d_o @ w.abs().t() + E * want.abs() + k * 2.0 ** -24 * (o.flatten(1).abs() @ w.abs().t())
    assert ((y.double() - want).abs() <= tol).all(), float(((y.double() - want).abs() / tol).max())


def context(stack, l, b, n):
    rows = stack.block_table[b, :-(-n // CFG.page_size)].long()
    return [c[l][rows].transpose(1, 2).flatten(0, 1)[:n] for c in (stack.k_cache, stack.v_cache)]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("w_bits", [16, 4])
def test_verify_then_commit_then_decode(device, w_bits):
    gen = torch.Generator().manual_seed(3)
    counts, ctx = [7, 1, 12, 4], 150
    stack = HelixDecodeStack(CFG, batch=4, local_ctx=ctx, device=device, draft_tokens=16, w_bits=w_bits)
    rows, L = sum(counts) + 2, CFG.n_layers                                     # two rows of padding

    def normal(*s):
        return torch.randn(*s, generator=gen).bfloat16().to(device)

    start = torch.tensor([0, 7, 8, 20, 24], dtype=torch.int32, device=device)
    par = torch.cat([trees(counts, gen), torch.tensor([-1, -1], dtype=torch.int32)])
    w = [oproj.unpack_weight_int4(stack._oproj_weight(l)) if w_bits == 4 else stack.w_o[l] for l in range(L)]
    before = [[context(stack, l, b, ctx) for b in range(4)] for l in range(L)]
    q, k, v = normal(L, rows, 16, 128), normal(L, rows, 2, 128), normal(L, rows, 2, 128)
    for attempt in range(2):                                                    # drafted twice: the second attempt overwrites the first
        y = stack.verify_step(q, k, v, start, par.to(device))
        assert y.shape == (L, rows, CFG.hidden) and not y[:, 24:].any()
        for l in range(L):
            for b, c in enumerate(counts):
                r0 = int(start[b])
                anc = torch.eye(c, dtype=torch.bool)
                for j in range(c):
                    if par[r0 + j] >= 0:
                        anc[j] |= anc[int(par[r0 + j])]
                seen = torch.cat([torch.ones(c, ctx, dtype=torch.bool), anc], 1).to(device)
                kb, vb = (torch.cat([before[l][b][i], x[l, r0:r0 + c]]) for i, x in enumerate((k, v)))
                o, a = plain(q[l, r0:r0 + c], kb, vb, seen)
                check(y[l, r0:r0 + c], o, a, w[l])
        if attempt == 0:
            q, k, v = normal(L, rows, 16, 128), normal(L, rows, 2, 128), normal(L, rows, 2, 128)
    # accept a path of each tree: from a leaf up
    paths = []
    for b, c in enumerate(counts):
        r0, node, path = int(start[b]), c - 1, []
        while node >= 0:
            path.append(r0 + node)
            node = int(par[r0 + node])
        paths.append(path[::-1] if b != 3 else [])                              # of the last sequence nothing is taken
    taken = torch.tensor([r for p in paths for r in p], device=device)
    t_start = torch.tensor([0] + list(torch.tensor([len(p) for p in paths]).cumsum(0)), dtype=torch.int32, device=device)
    stack.commit(k, v, taken, t_start)
    assert stack.seq_lens.tolist() == [ctx + len(p) for p in paths] == stack.ctx_lens.tolist()
    qd = normal(L, 4, 16, 128)
    y = stack.decode_step(qd)
    for l in range(L):
        for b, p in enumerate(paths):
            kb, vb = (torch.cat([before[l][b][i], x[l, p]]) for i, x in enumerate((k, v)))
            o, a = plain(qd[l, b:b + 1], kb, vb, torch.ones(1, len(kb), dtype=torch.bool, device=device))
            check(y[l, b:b + 1], o, a, w[l])


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("cp,il", [(2, 1), (4, 4), (3, 16)])
def test_shards_of_ranks_combine_to_the_whole(device, cp, il):
    """Every rank's tables, cache and partial attention, played one after the other: their combination is the attention of one rank."""
    gen = torch.Generator().manual_seed(cp)
    ctx, counts, page, Hq, Hkv = [37, 0, 100], [9, 5, 1], 16, 8, 2
    rows = sum(counts)

    def normal(*s):
        return torch.randn(*s, generator=gen).bfloat16().to(device)

    def i32(v):
        return torch.tensor(v, dtype=torch.int32, device=device)

    q, k, v = normal(rows, Hq, 128), normal(rows, Hkv, 128), normal(rows, Hkv, 128)
    old = [(normal(n, Hkv, 128), normal(n, Hkv, 128)) for n in ctx]
    par, start = trees(counts, gen).to(device), i32([0, 9, 14, 15])
    outs, lses, seen_slots = [], [], 0
    for rank in range(cp):
        kc, vc = (torch.zeros(24, Hkv, page, 128, dtype=torch.bfloat16, device=device) for _ in range(2))
        table, held, free, used = i32([[0] * 9] * 3), i32([0] * 3), torch.randperm(24, generator=gen).int().to(device), i32([0])
        common = dict(page_size=page, cp_size=cp, cp_rank=rank, interleave=il)
        prompt = paged.extend_tables(table, held, free, used, i32([0] * 3), i32([0, 37, 37, 137]), rows=137, mask_words=0, **common)
        paged.append_kv(torch.cat([o[0] for o in old]), torch.cat([o[1] for o in old]), kc, vc, prompt.slots)
        plan = paged.extend_tables(table, held, free, used, i32(ctx), start, rows=rows, parents=par, **common)
        paged.append_kv(k, v, kc, vc, plan.slots)
        assert int(plan.missing) == 0
        seen_slots += int((plan.slots >= 0).sum())
        o, lse = attention.tree_decode(q, kc, vc, table, plan.seq_lens, start, plan.draft_lens, plan.mask)
        outs.append(o)
        lses.append(lse)
    assert seen_slots == rows
    got = lse_combine(torch.stack(outs), torch.stack(lses)).double()
    for b, c in enumerate(counts):
        r0 = int(start[b])
        anc = torch.eye(c, dtype=torch.bool)
        for j in range(c):
            if par[r0 + j] >= 0:
                anc[j] |= anc[int(par[r0 + j])]
        seen = torch.cat([torch.ones(c, ctx[b], dtype=torch.bool), anc], 1).to(device)
        o, a = plain(q[r0:r0 + c], torch.cat([old[b][0], k[r0:r0 + c]]), torch.cat([old[b][1], v[r0:r0 + c]]), seen)
        # the parts' roundings are weighted like the parts, the combination is rounded once more
        assert ((got[r0:r0 + c] - o).abs() <= 2 * E * (a + o.abs()) + 4e-4 * a).all()


@pytest.mark.parametrize("device", DEVICES)
def test_exchange_and_o_proj_with_four_bits(device, monkeypatch):
    """The call that would be one kernel takes 4-bit weights too, as two."""
    o, lse = torch.randn(5, 8, 128).bfloat16().to(device), torch.randn(5, 8).to(device)
    w = oproj.quantize_weight_int4(torch.randn(256, 512).bfloat16().to(device))
    monkeypatch.setattr(api, "alltoall_combine", lambda o, lse, ws, rank, size, base2=False: o[:, 4 * rank:4 * rank + 4])
    got = api.alltoall_combine_oproj(o, lse, w, None, 1, 2)
    assert torch.equal(got, oproj.oproj(o[:, 4:].reshape(5, 512), w))


@pytest.mark.gpu
def test_captured_verification():
    stack = HelixDecodeStack(CFG, batch=3, local_ctx=200, draft_tokens=8, w_bits=4)
    shape = dict(dtype=torch.bfloat16, device="cuda")
    q, k, v = torch.randn(2, 24, 16, 128, **shape), torch.randn(2, 24, 2, 128, **shape), torch.randn(2, 24, 2, 128, **shape)
    start = torch.tensor([0, 8, 16, 24], dtype=torch.int32, device="cuda")
    eager = stack.verify_step(q, k, v, start).clone()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            y = stack.verify_step(q, k, v, start)
        g.replay()
        s.synchronize()
        assert torch.equal(y, eager)
        start.copy_(torch.tensor([0, 3, 4, 10]))
        g.replay()
        s.synchronize()
    assert torch.equal(y[:, :10], stack.verify_step(q, k, v, start)[:, :10]) and not y[:, 10:].any()


def test_refusals():
    with pytest.raises(ValueError):
        HelixDecodeStack(CFG, batch=1, local_ctx=16, device="cpu", w_bits=8)
    stack = HelixDecodeStack(CFG, batch=1, local_ctx=16, device="cpu")
    z = torch.zeros(2, 1, 16, 128).bfloat16()
    with pytest.raises(RuntimeError):
        stack.verify_step(z, z[:, :, :2], z[:, :, :2], torch.tensor([0, 1], dtype=torch.int32))
    with pytest.raises(RuntimeError):
        stack.commit(z, z, torch.tensor([0]), torch.tensor([0, 1], dtype=torch.int32))
