"""Verification of drafted tokens over this rank's shard of a paged cache, as cases that can be timed.

Every case is one call of a public entry point on one GPU:

* ``tables``  ``ops.paged.extend_tables``: pages, slots, positions, local lengths and tree masks of a step's new tokens
* ``append``  ``ops.paged.append_kv``: the new tokens' K and V rows into their slots
* ``tree``    ``ops.attention.tree_decode``: attention of several drafted tokens per sequence, masked by their tree
* ``int4``    ``ops.oproj.oproj`` with 4-bit weights and group scales

With ``own`` false the same is computed by elementary torch operations in 32 bits.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False


def listed():
    return [
        # the plan of one chat's step: a tree of 16 drafted tokens
        dict(name="tables one chat", op="tables", batch=1, new=16, ragged=False, ctx=2000, page=16, cp=1, rank=0, il=1, tree=True),
        # a serving batch on one of four ranks, every sequence with another tree, pages interleaved over the ranks
        dict(name="tables serving batch", op="tables", batch=256, new=26, ragged=True, ctx=9000, page=32, cp=4, rank=1, il=16,
             tree=True),
        # prompts that enter the cache: slots and pages only
        dict(name="tables prompts", op="tables", batch=64, new=1900, ragged=True, ctx=0, page=16, cp=1, rank=0, il=1, tree=False),
        # a step's drafted tokens of a small batch, and a chunk of prompts
        dict(name="append step", op="append", rows=32, heads=8, page=16, pool=4096, layout="HND", dtype="bf16", gone=0.0),
        dict(name="append prompts", op="append", rows=16384, heads=8, page=32, pool=1024, layout="NHD", dtype="fp16", gone=0.25),
        # one short chat with a small tree: nothing but latency
        dict(name="tree short", op="tree", batch=1, nodes=8, ctx=300, ragged=False, q_heads=64, kv_heads=8, page=16, layout="HND",
             dtype="bf16", cp=1),
        # a mixed serving batch: every sequence another length and another number of drafted tokens
        dict(name="tree ragged batch", op="tree", batch=24, nodes=16, ctx=9000, ragged=True, q_heads=32, kv_heads=8, page=32,
             layout="NHD", dtype="fp16", cp=1),
        # chains of a few drafted tokens over the shards of a large batch: bound by reading the cache
        dict(name="tree chains", op="tree", batch=64, nodes=5, ctx=8192, ragged=False, q_heads=64, kv_heads=8, page=16, layout="HND",
             dtype="bf16", cp=4),
        # a wide tree over one long sequence: bound by the products
        dict(name="tree wide 128k", op="tree", batch=1, nodes=64, ctx=131072, ragged=False, q_heads=64, kv_heads=8, page=16,
             layout="HND", dtype="bf16", cp=1),
        # o_proj: one rank's K-slice of eight for one chat, the whole layer at a decode batch, and the tokens of a verified batch
        dict(name="int4 slice", op="int4", tokens=1, hidden=8192, k=1024, group=128, zeros=False, dtype="bf16"),
        dict(name="int4 decode", op="int4", tokens=8, hidden=8192, k=8192, group=128, zeros=True, dtype="bf16"),
        dict(name="int4 verify", op="int4", tokens=100, hidden=7168, k=8192, group=64, zeros=False, dtype="fp16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["tables", "append", "tree", "tree", "tree", "int4", "int4"])
    if op == "tables":
        cp = rng.choice([1, 1, 2, 4, 8])
        tree = rng.random() < 0.7
        batch = _log(rng, 1, 512 if tree else 64)
        return dict(op=op, batch=batch, new=_log(rng, 1, 64 if tree else 1900), ragged=rng.random() < 0.7, ctx=_log(rng, 1, 20000),
                    page=rng.choice([16, 32, 64]), cp=cp, rank=rng.randrange(cp), il=rng.choice([1, 1, 16, 64]), tree=tree)
    if op == "append":
        rows = _log(rng, 1, 16384)
        page = rng.choice([16, 32, 64])
        return dict(op=op, rows=rows, heads=rng.choice([1, 2, 4, 8]), page=page, pool=2 * (rows // page) + 8,
                    layout=rng.choice(["HND", "NHD"]), dtype=rng.choice(["bf16", "fp16"]), gone=rng.choice([0.0, 0.5]))
    if op == "tree":
        batch = _log(rng, 1, 64)
        kv_heads, group = rng.choice([(8, 8), (8, 4), (4, 8), (2, 8), (8, 1), (4, 5)])
        nodes = _log(rng, 1, 64)
        return dict(op=op, batch=batch, nodes=nodes, ctx=_log(rng, 16, min(131072, (1 << 23) // (batch * nodes))),
                    ragged=rng.random() < 0.6, q_heads=kv_heads * group, kv_heads=kv_heads, page=rng.choice([16, 32, 64]),
                    layout=rng.choice(["HND", "NHD"]), dtype=rng.choice(["bf16", "fp16"]), cp=rng.choice([1, 1, 2, 4]))
    return dict(op=op, tokens=_log(rng, 1, 100), hidden=rng.choice([1024, 2048, 4096, 7168]),
                k=rng.choice([832, 1024, 2048, 4096, 8192]), group=rng.choice([32, 64]), zeros=rng.random() < 0.5,
                dtype=rng.choice(["bf16", "fp16"]))


_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def _spread(case, key, low=1):
    """One number per sequence: all alike, or spread over the range (the same ones whatever the seed)."""
    b, top = case["batch"], case[key]
    if not case["ragged"]:
        return [top] * b
    phase = 0.137 if key == "ctx" else 0.71
    return [max(low, int(math.ceil(top * ((phase + i * 0.6180339887) % 1.0)))) for i in range(b)]


def _parents(nodes, rng):
    """Parents of each sequence's drafted tokens: about two children per token, -1 for those behind the last committed one."""
    out = []
    for t in nodes:
        at = np.arange(t)
        out.append(np.where(rng.random(t) < 0.15, -1, np.maximum(-1, at - 1 - (rng.random(t) * (at // 2 + 1)).astype(np.int64))))
    return out


def _tree_words(parents, cp):
    """Mask words ``[rows, 1]`` over the drafted tokens that a rank with every ``cp``-th of them holds, and their counts."""
    words, counts = [], []
    for par in parents:
        bits = []
        for j, p in enumerate(par):
            bits.append((bits[p] if p >= 0 else 0) | (1 << (j // cp) if j % cp == 0 else 0))
        words += bits
        counts.append(-(-len(par) // cp))
    return np.array(words, dtype=np.uint64).view(np.int64).reshape(-1, 1), counts


def _starts(counts):
    return torch.tensor([0] + list(np.cumsum(counts)), dtype=torch.int32, device="cuda")


def _int4_weights(case, seed):
    """A 4-bit checkpoint's arrays: nibbles ``[hidden, K / 2]`` (even column in the low half), scales, zero points or None."""
    gen = torch.Generator(device="cuda").manual_seed(seed + 1)
    h, k, g, dtype = case["hidden"], case["k"], case["group"], _DTYPES[case["dtype"]]
    w = torch.empty(h, k // g, g, device="cuda").normal_(0, 0.02, generator=gen)
    if case["zeros"]:
        lo, hi = w.amin(-1), w.amax(-1)
        scales = ((hi - lo) / 15).to(dtype)
        zeros = (-lo / scales.float()).round().clamp(0, 15)
    else:
        scales = (w.abs().amax(-1) / 7).to(dtype)
        zeros = torch.full_like(scales, 8, dtype=torch.float32)
    q = (w / scales.float().unsqueeze(-1) + zeros.unsqueeze(-1)).round().clamp(0, 15).to(torch.uint8).view(h, k)
    return q[:, 0::2] | (q[:, 1::2] << 4), scales, zeros.to(torch.uint8) if case["zeros"] else None


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rng = np.random.default_rng(seed)

    def normal(*shape, dtype=torch.bfloat16):
        return torch.empty(*shape, dtype=dtype, device="cuda").normal_(0, 1, generator=gen)

    def ints(values):
        return torch.tensor(values, dtype=torch.int32, device="cuda")

    op = case["op"]
    if op == "tables":
        order = rng.permutation(case["batch"])
        ctx = [_spread(case, "ctx", 0)[i] for i in order]
        new = [_spread(case, "new")[i] for i in order]
        page, cp, il = case["page"], case["cp"], case["il"]
        local = [_local_count(n, case) for n in ctx]
        wants = [-(-_local_count(n + t, case) // page) for n, t in zip(ctx, new)]
        # a sequence holds what its committed tokens need and at times a page of drafted ones that were not taken
        held = [min(w, -(-n // page) + int(rng.random() < 0.3)) for n, w in zip(local, wants)]
        pool = sum(wants) + 8
        ids = rng.permutation(pool)
        table = np.zeros((len(ctx), max(wants) + 2), dtype=np.int32)
        at = 0
        for b, h in enumerate(held):
            table[b, :h] = ids[at:at + h]
            at += h
        rows = sum(new)
        return dict(op=op, table=torch.from_numpy(table).cuda(), held=ints(held), free=ints(ids[at:]), used=ints([0]), ctx=ints(ctx),
                    starts=_starts(new), rows=rows, page=page, cp=cp, rank=case["rank"], il=il, words=1 if case["tree"] else 0,
                    max_new=max(new), parents=ints(np.concatenate(_parents(new, rng))) if case["tree"] else None)
    if op == "append":
        rows, h, page, pool, dtype = case["rows"], case["heads"], case["page"], case["pool"], _DTYPES[case["dtype"]]
        shape = (pool, h, page, 128) if case["layout"] == "HND" else (pool, page, h, 128)
        slots = rng.permutation(pool * page)[:rows]
        slots[rng.random(rows) < case["gone"]] = -1                      # tokens of other ranks
        qkv = normal(rows, 3, h, 128, dtype=dtype)                        # K and V as a projection leaves them, side by side
        return dict(op=op, k=qkv[:, 1], v=qkv[:, 2], kc=normal(*shape, dtype=dtype), vc=normal(*shape, dtype=dtype),
                    slots=torch.from_numpy(slots).cuda(), layout=case["layout"])
    if op == "tree":
        order = rng.permutation(case["batch"])
        ctx = [_spread(case, "ctx")[i] for i in order]
        nodes = [_spread(case, "nodes")[i] for i in order]
        words, drafts = _tree_words(_parents(nodes, rng), case["cp"])
        lens = [n + d for n, d in zip(ctx, drafts)]
        page, h, dtype = case["page"], case["kv_heads"], _DTYPES[case["dtype"]]
        pages = [-(-n // page) for n in lens]
        pool = sum(pages) + 3
        ids = rng.permutation(pool)
        table = np.zeros((len(lens), max(pages)), dtype=np.int32)
        at = 0
        for b, c in enumerate(pages):
            table[b, :c] = ids[at:at + c]
            at += c
        shape = (pool, h, page, 128) if case["layout"] == "HND" else (pool, page, h, 128)
        return dict(op=op, q=normal(sum(nodes), case["q_heads"], 128, dtype=dtype), k=normal(*shape, dtype=dtype),
                    v=normal(*shape, dtype=dtype), table=torch.from_numpy(table).cuda(), lens=ints(lens), starts=_starts(nodes),
                    drafts=ints(drafts), mask=torch.from_numpy(words).cuda(), layout=case["layout"], base2=case["layout"] == "NHD",
                    host=list(zip(nodes, lens, drafts)), max_len=max(lens), max_rows=max(nodes))
    x = normal(case["tokens"], case["k"], dtype=_DTYPES[case["dtype"]])
    qweight, scales, zeros = _int4_weights(case, seed)
    if own:
        from helix_a2a_b200.ops import oproj
        return dict(op=op, x=x, w=oproj.pack_weight_int4(qweight, scales, zeros))
    return dict(op=op, x=x, q=qweight, scales=scales, zeros=zeros, group=case["group"])


def _run_own(s):
    from helix_a2a_b200.ops import attention, oproj, paged
    if s["op"] == "tables":
        plan = paged.extend_tables(s["table"], s["held"], s["free"], s["used"], s["ctx"], s["starts"], rows=s["rows"],
                                   page_size=s["page"], parents=s["parents"], mask_words=s["words"], cp_size=s["cp"],
                                   cp_rank=s["rank"], interleave=s["il"])
        return dict(plan._asdict(), table=s["table"], held=s["held"], used=s["used"])
    if s["op"] == "append":
        paged.append_kv(s["k"], s["v"], s["kc"], s["vc"], s["slots"], layout=s["layout"])
        return s["kc"], s["vc"]
    if s["op"] == "tree":
        return attention.tree_decode(s["q"], s["k"], s["v"], s["table"], s["lens"], s["starts"], s["drafts"], s["mask"],
                                     layout=s["layout"], lse_base2=s["base2"], max_seq_len=s["max_len"], max_q_len=s["max_rows"])
    return oproj.oproj(s["x"], s["w"])


def _tables(s):
    page, cp, rank, il, words = s["page"], s["cp"], s["rank"], s["il"], s["words"]
    table, held, free = s["table"], s["held"].long(), s["free"].long()
    starts, n0 = s["starts"].long(), s["ctx"].long()

    def local(n):
        return n // (il * cp) * il + (n % (il * cp) - rank * il).clamp(0, il)

    n1 = n0 + starts.diff()
    need = (local(n1) + page - 1) // page
    new = (need.clamp(max=table.shape[1]) - held).clamp(min=0)
    first = s["used"].long() + new.cumsum(0) - new
    got = torch.minimum(new, (len(free) - first).clamp(min=0))
    at = torch.arange(table.shape[1], device=table.device) - held.unsqueeze(1)
    taken = (at >= 0) & (at < got.unsqueeze(1))
    if len(free):
        table.copy_(torch.where(taken, free[(first.unsqueeze(1) + at).clamp(0, len(free) - 1)], table))
    missing = (need - held).clamp(min=0).sum().view(1) - got.sum()
    held = held + got
    s["held"].copy_(held)
    s["used"].add_(got.sum())
    lens = torch.minimum(local(n1), held * page)
    row = torch.arange(s["rows"], device=table.device)
    b = torch.searchsorted(starts[1:], row, right=True).clamp(max=len(n0) - 1)
    inside = row < starts[-1]
    node = row - starts[b]
    pos = n0[b] + node
    mine = (pos // il % cp == rank) & inside
    at = local(pos)
    mine &= at < held[b] * page
    slots = torch.where(mine, table[b, (at // page).clamp(max=table.shape[1] - 1)].long() * page + at % page, -1)
    out = dict(slots=slots, seq_lens=lens.int(), draft_lens=(lens - local(n0)).clamp(min=0).int(), missing=missing.int(), table=table,
               held=s["held"], used=s["used"])
    mask = torch.zeros(s["rows"], max(words, 1), dtype=torch.int64, device=table.device)
    depth = torch.zeros_like(row)
    if words:
        up, alive = node.clone(), inside.clone()
        for _ in range(s["max_new"]):
            p = n0[b] + up
            bit = local(p) - local(n0[b])
            seen = alive & (p // il % cp == rank) & (local(p) < held[b] * page) & (bit < 64 * words)
            word = (bit // 64).clamp(0, words - 1).unsqueeze(1)
            value = torch.where(seen, torch.ones_like(bit) << (bit % 64), 0)
            mask.scatter_(1, word, mask.gather(1, word) | value.unsqueeze(1))
            parent = s["parents"][(starts[b] + up).clamp(0, s["rows"] - 1)].long()
            alive = alive & (parent >= 0)
            depth = depth + alive
            up = torch.where(alive, parent, up)
    else:
        depth = node
    return dict(out, positions=torch.where(inside, n0[b] + depth, 0).int(), mask=mask[:, :words])


def _plain_tree(s):
    """Every sequence by itself: its pages put side by side, scores, the mask, softmax and the weighted sum."""
    k, v = (c.transpose(1, 2) if s["layout"] == "HND" else c for c in (s["k"], s["v"]))
    heads, group = k.shape[2], s["q"].shape[1] // k.shape[2]
    outs, lses, at = [], [], 0
    for b, (t, n, d) in enumerate(s["host"]):
        rows = s["table"][b, :-(-n // k.shape[1])].long()
        kb, vb = (c[rows].flatten(0, 1)[:n].float().transpose(0, 1) for c in (k, v))                    # [Hkv, n, 128]
        x = s["q"][at:at + t].float().view(t, heads, group, 128).permute(1, 2, 0, 3) / math.sqrt(128)   # [Hkv, group, t, 128]
        x = (x.reshape(heads, group * t, 128) @ kb.transpose(1, 2)).view(heads, group, t, n)
        hidden = (s["mask"][at:at + t] >> torch.arange(d, device=x.device)) & 1 == 0
        x[..., n - d:].masked_fill_(hidden, -math.inf)
        top = x.amax(-1, keepdim=True).clamp(min=torch.finfo(torch.float32).min)
        p = (x - top).exp_()
        total = p.sum(-1, keepdim=True)
        o = (p.view(heads, group * t, n) @ vb).view(heads, group, t, 128) / total.clamp(min=1e-30)
        outs.append(o.permute(2, 0, 1, 3).reshape(t, -1, 128))
        lses.append((top + total.log()).squeeze(-1).permute(2, 0, 1).reshape(t, -1))
        at += t
    lse = torch.cat(lses)
    return torch.cat(outs).to(s["q"].dtype), lse / math.log(2.0) if s["base2"] else lse


def run(s):
    if own:
        return _run_own(s)
    if s["op"] == "tables":
        return _tables(s)
    if s["op"] == "append":
        page = s["kc"].shape[2 if s["layout"] == "HND" else 1]
        take = s["slots"] >= 0
        slots = s["slots"][take]
        for c, x in ((s["kc"], s["k"]), (s["vc"], s["v"])):
            c = c.transpose(1, 2) if s["layout"] == "HND" else c
            c[slots // page, slots % page] = x[take]
        return s["kc"], s["vc"]
    if s["op"] == "tree":
        return _plain_tree(s)
    h, k = s["q"].shape[0], 2 * s["q"].shape[1]
    q = torch.stack([s["q"] & 15, s["q"] >> 4], -1).view(h, -1, s["group"]).float()
    w = (q - (8 if s["zeros"] is None else s["zeros"].float().unsqueeze(-1))) * s["scales"].float().unsqueeze(-1)
    return (s["x"].float() @ w.view(h, k).t()).to(s["x"].dtype)


def work(case):
    op = case["op"]
    if op == "tables":
        rows, b, words = sum(_spread(case, "new")), case["batch"], 1 if case["tree"] else 0
        pages = sum(_local_count(t, case) for t in _spread(case, "new")) // case["page"]
        return dict(bytes=b * 24 + pages * 8 + rows * (12 + 12 * words), flops=rows * 8)
    if op == "append":
        rows = case["rows"] * (1 - case["gone"])
        return dict(bytes=int(rows * case["heads"] * 4 * 256) + 8 * case["rows"], flops=0)
    if op == "tree":
        nodes, hq = _spread(case, "nodes"), case["q_heads"]
        lens = [n + -(-t // case["cp"]) for n, t in zip(_spread(case, "ctx"), nodes)]
        return dict(bytes=sum(lens) * case["kv_heads"] * 512 + sum(nodes) * (hq * (512 + 4) + 8),
                    flops=4 * 128 * hq * sum(n * t for n, t in zip(lens, nodes)))
    t, h, k = case["tokens"], case["hidden"], case["k"]
    return dict(bytes=h * k // 2 + h * (k // case["group"]) * (3 if case["zeros"] else 2) + 2 * t * (h + k), flops=2 * t * h * k)


def _local_count(n, case):
    """How many of a sequence's first ``n`` tokens this rank holds."""
    il, cp = case["il"], case["cp"]
    return sum(1 for p in range(n // (il * cp) * il * cp, n) if p // il % cp == case["rank"]) + n // (il * cp) * il


def _exact_tables(s):
    page, cp, rank, il = s["page"], s["cp"], s["rank"], s["il"]
    table, held, free = (s[k].cpu().numpy().copy() for k in ("table", "held", "free"))
    ctx, starts, used = s["ctx"].tolist(), s["starts"].tolist(), int(s["used"])
    parents = s["parents"].tolist() if s["parents"] is not None else None
    out = dict(slots=[], positions=[], seq_lens=[], draft_lens=[], mask=[])
    missing = 0
    for b, n0 in enumerate(ctx):
        t = starts[b + 1] - starts[b]
        before = _local_count(n0, dict(il=il, cp=cp, rank=rank))
        mine = [j for j in range(t) if (n0 + j) // il % cp == rank]
        need = -(-(before + len(mine)) // page)
        while held[b] < need:
            if held[b] == table.shape[1] or used == len(free):
                missing += need - held[b]
                break
            table[b, held[b]] = free[used]
            held[b] += 1
            used += 1
        room = int(held[b]) * page
        here = {j: before + i for i, j in enumerate(mine) if before + i < room}
        out["seq_lens"].append(min(before + len(mine), room))
        out["draft_lens"].append(len(here))
        out["slots"] += [int(table[b, here[j] // page]) * page + here[j] % page if j in here else -1 for j in range(t)]
        words, depths = [], []
        for j in range(t):
            p = parents[starts[b] + j] if parents is not None else j - 1
            depths.append(0 if p < 0 else depths[p] + 1)
            if parents is not None:
                words.append((words[p] if p >= 0 else 0) | (1 << (here[j] - before) if j in here else 0))
        out["positions"] += [n0 + d for d in depths]
        out["mask"] += words
    res = {k: torch.tensor(v) for k, v in out.items() if k != "mask"}
    res["mask"] = torch.from_numpy(np.array(out["mask"], dtype=np.uint64).view(np.int64).reshape(len(res["slots"]), -1))
    res.update(missing=torch.tensor([missing]), table=torch.from_numpy(table), held=torch.from_numpy(held), used=torch.tensor([used]))
    return {k: v.cuda() for k, v in res.items()}


def exact(case, seed):
    """What ``run`` returns, from the definitions in 64 bits."""
    s = prepare(case, seed)
    if s["op"] == "tables":
        return _exact_tables(s)
    if s["op"] == "append":
        out = []
        for c, x in ((s["kc"], s["k"]), (s["vc"], s["v"])):
            flat = (c.transpose(1, 2) if s["layout"] == "HND" else c).double().flatten(0, 1)             # [slots, heads, 128]
            rows = torch.full((len(flat),), -1, device=c.device)
            at = torch.arange(len(s["slots"]), device=c.device)[s["slots"] >= 0]
            rows[s["slots"][at]] = at
            flat = torch.where((rows >= 0).view(-1, 1, 1), x.double()[rows], flat)
            flat = flat.view(c.shape[0], -1, *flat.shape[1:])
            out.append(flat.transpose(1, 2).contiguous() if s["layout"] == "HND" else flat)
        return tuple(out)
    if s["op"] == "tree":
        o = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
        lse = torch.empty(s["q"].shape[:2], dtype=torch.float64, device="cuda")
        hnd, group = s["layout"] == "HND", case["q_heads"] // case["kv_heads"]
        at = 0
        for b, (t, n, d) in enumerate(s["host"]):
            token = torch.arange(n, device="cuda")
            pages, tip = s["table"][b].long()[token // case["page"]], token % case["page"]
            seen = torch.ones(t, n, dtype=torch.bool, device="cuda")
            for i in range(d):
                seen[:, n - d + i] = (s["mask"][at:at + t, 0] >> i) % 2 != 0
            for h in range(case["q_heads"]):
                kb, vb = (c[pages, h // group, tip] if hnd else c[pages, tip, h // group] for c in (s["k"], s["v"]))
                x = s["q"][at:at + t, h].double() @ kb.double().t() / math.sqrt(128)
                x = torch.where(seen, x, -math.inf)
                lse[at:at + t, h] = torch.logsumexp(x, -1)
                o[at:at + t, h] = torch.softmax(x, -1).nan_to_num(0) @ vb.double()
            at += t
        return o, lse / math.log(2.0) if s["base2"] else lse
    q, scales, zeros = _int4_weights(case, seed)
    w = torch.empty(case["hidden"], case["k"], dtype=torch.float64, device="cuda")
    w[:, 0::2], w[:, 1::2] = (q % 16).double(), (q // 16).double()
    w -= 8 if zeros is None else zeros.double().repeat_interleave(case["group"], 1)
    w *= scales.double().repeat_interleave(case["group"], 1)
    return s["x"].double() @ w.t()
