"""tree_decode against softmax attention in float64, row by row masked.

Tolerances, with A = sum_j p_j |v_j| / sum_j p_j and e = eps / 2 of the type: P rounded to the type moves an output by at most e A, the
output's own rounding by e |o|; fp32 scores of 128 products are off by less than 128 * 2^-24 * sum |q k| * scale < 1e-4, i.e. 1e-4 A, and
fp32 sums over n tokens by at most n 2^-24 A.  The LSE is not rounded: 2e-4 covers the scores and one fp32 step of values up to 1000.
"""
import math

import numpy as np
import pytest
import torch

from helix_a2a_b200.ops import attention
from helix_a2a_b200.ops.oproj import check_compute_status

pytestmark = pytest.mark.gpu
DT = {"bf16": torch.bfloat16, "fp16": torch.float16}


def make(lens, drafts, counts, hq, hkv, page, layout, dtype, words=1, pad=0, seed=0, density=0.5, extra_pages=3):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rng = np.random.default_rng(seed)

    def normal(*s):
        return torch.empty(*s, device="cuda", dtype=DT[dtype]).normal_(0, 1, generator=gen)

    need = [-(-n // page) for n in lens]
    pool = sum(need) + extra_pages
    ids = rng.permutation(pool)
    table = np.full((len(lens), max(need + [1]) + 1), -7, dtype=np.int32)              # entries that must not be read
    at = 0
    for b, c in enumerate(need):
        table[b, :c] = ids[at:at + c]
        at += c
    rows = sum(counts) + pad
    mask = rng.integers(0, 2 ** 64, (rows, max(words, 1)), dtype=np.uint64)
    if density < 0.5:
        mask &= rng.integers(0, 2 ** 64, mask.shape, dtype=np.uint64) & rng.integers(0, 2 ** 64, mask.shape, dtype=np.uint64)
    shape = (pool, hkv, page, 128) if layout == "HND" else (pool, page, hkv, 128)

    def i32(v):
        return torch.tensor(np.asarray(v), dtype=torch.int32, device="cuda")

    return dict(q=normal(rows, hq, 128), k_cache=normal(*shape), v_cache=normal(*shape), block_table=i32(table), seq_lens=i32(lens),
                q_start=i32(np.concatenate([[0], np.cumsum(counts)])), draft_lens=i32(drafts),
                mask=torch.from_numpy(mask.view(np.int64)).cuda()[:, :words])


def exact(s, layout, scale=None, base2=False):
    """o, lse and A in float64."""
    scale = 1 / math.sqrt(128) if scale is None else scale
    k, v = (c.transpose(1, 2) if layout == "HND" else c for c in (s["k_cache"], s["v_cache"]))
    hkv, page = k.shape[2], k.shape[1]
    rows, hq, _ = s["q"].shape
    o = torch.zeros(rows, hq, 128, dtype=torch.float64, device="cuda")
    a, lse = o.clone(), torch.full((rows, hq), -math.inf, dtype=torch.float64, device="cuda")
    starts = s["q_start"].tolist()
    for b, (n, d) in enumerate(zip(s["seq_lens"].tolist(), s["draft_lens"].tolist())):
        r0, r1 = starts[b], starts[b + 1]
        if n == 0 or r0 == r1:
            continue
        pages = s["block_table"][b, :-(-n // page)].long()
        kb, vb = (c[pages].flatten(0, 1)[:n].double() for c in (k, v))
        seen = torch.ones(r1 - r0, n, dtype=torch.bool, device="cuda")
        for i in range(d):
            w = i // 64
            seen[:, n - d + i] = (s["mask"][r0:r1, w] >> (i % 64)) & 1 != 0 if w < s["mask"].shape[1] else False
        for h in range(hkv):
            g = slice(h * (hq // hkv), (h + 1) * (hq // hkv))
            x = torch.einsum("rgd,nd->rgn", s["q"][r0:r1, g].double(), kb[:, h]) * scale
            x = torch.where(seen[:, None], x, -math.inf)
            top = x.amax(-1, keepdim=True)
            p = torch.where(seen[:, None], (x - torch.where(top == -math.inf, 0, top)).exp(), 0)
            total = p.sum(-1, keepdim=True)
            p = torch.where(total > 0, p / total, 0) if not torch.isnan(total).any() else p / total
            vz = vb[:, h]
            finite = torch.isfinite(vz)
            o[r0:r1, g] = torch.einsum("rgn,nd->rgd", p, torch.where(finite, vz, 0))
            a[r0:r1, g] = torch.einsum("rgn,nd->rgd", p, torch.where(finite, vz, 0).abs())
            for j in (~finite).any(-1).nonzero().flatten().tolist():                     # only to the rows that see the token
                bad = torch.where(finite[j], 0, vz[j])
                o[r0:r1, g] += torch.where(seen[:, j, None, None], bad, 0)
            lse[r0:r1, g] = (top + total.log()).squeeze(-1)
    return o, lse / math.log(2) if base2 else lse, a


def check(s, layout, dtype, **kw):
    o, lse = attention.tree_decode(s["q"], s["k_cache"], s["v_cache"], s["block_table"], s["seq_lens"], s["q_start"], s["draft_lens"],
                                   s["mask"], layout=layout, **{k: v for k, v in kw.items() if k != "base2"}, lse_base2=kw.get("base2", False))
    check_compute_status(s["q"])
    want, want_lse, a = exact(s, layout, kw.get("scale"), kw.get("base2", False))
    e = torch.finfo(DT[dtype]).eps / 2
    n = int(s["seq_lens"].max()) if s["seq_lens"].numel() else 0
    assert o.dtype == DT[dtype] and lse.dtype == torch.float32 and o.shape == s["q"].shape
    tol = e * (a + want.abs()) + (1e-4 + n * 2.0 ** -24) * a
    same = (o.double() == want) | (torch.isnan(want) & torch.isnan(o))
    bad = ~((o.double() - want).abs() <= tol) & ~same
    assert not bad.any(), (bad.nonzero()[:5].tolist(), int(bad.sum()), float((o.double() - want).abs().nan_to_num().max()))
    same = (lse.double() == want_lse) | (torch.isnan(want_lse) & torch.isnan(lse))
    bad = ~((lse.double() - want_lse).abs() <= 2e-4) & ~same
    assert not bad.any(), (bad.nonzero()[:5].tolist(), lse[bad][:3], want_lse[bad][:3])
    return o, lse


@pytest.mark.parametrize("layout,dtype", [("HND", "bf16"), ("NHD", "fp16")])
@pytest.mark.parametrize("hq,hkv", [(64, 8), (8, 8), (10, 2), (32, 1)])
@pytest.mark.parametrize("n,d,t", [(1, 1, 1), (1, 0, 1), (16, 5, 5), (127, 3, 9), (128, 8, 16), (129, 16, 16), (300, 26, 26), (1000, 64, 64),
                                   (70, 64, 33)])
def test_one_sequence(n, d, t, hq, hkv, layout, dtype):
    s = make([n], [d], [t], hq, hkv, 16, layout, dtype, seed=n + d)
    check(s, layout, dtype, max_seq_len=n, max_q_len=t)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("page", [16, 32, 48, 64, 256])
@pytest.mark.parametrize("t,hq,hkv", [(7, 16, 2), (40, 16, 2), (1, 8, 8)])
def test_ragged_batch(t, hq, hkv, page, dtype):
    rng = np.random.default_rng(page + t)
    lens = [int(x) for x in rng.integers(1, 2000, 9)] + [0, 5, 0, 3000]
    counts = [int(x) for x in rng.integers(0, t + 1, 13)]
    counts[9], counts[10] = 3, 2                              # a sequence without a token here, rows that see drafted tokens only
    drafts = [min(n, int(x)) for n, x in zip(lens, rng.integers(0, t + 1, 13))]
    drafts[10] = 5
    s = make(lens, drafts, counts, hq, hkv, page, "NHD", dtype, pad=3, seed=t)
    o, lse = check(s, "NHD", dtype, max_seq_len=3000, max_q_len=t, base2=True)
    assert not o[-3:].any() and (lse[-3:] == -math.inf).all()
    check(s, "NHD", dtype, max_seq_len=1, max_q_len=1)        # hints that are too low, or unknown, only cost time
    check(s, "NHD", dtype)


def test_rows_that_see_nothing():
    s = make([40, 9], [40, 9], [6, 5], 16, 2, 16, "HND", "bf16")
    s["mask"][1] = 0
    s["mask"][3] = 1 << 50                                    # a bit of no token
    s["mask"][8:] = 0
    o, lse = check(s, "HND", "bf16", max_seq_len=40, max_q_len=6)
    for r in (1, 3, 8, 9, 10):
        assert not o[r].any() and (lse[r] == -math.inf).all()


@pytest.mark.parametrize("t", [9, 70])
@pytest.mark.parametrize("words,d", [(0, 4), (1, 64), (1, 100), (2, 128), (3, 140), (4, 256), (4, 300)])
def test_mask_words(words, d, t):
    s = make([500, 300], [d, d], [t, 2], 8, 2, 16, "HND", "fp16", words=words, seed=d)
    check(s, "HND", "fp16", max_seq_len=500, max_q_len=t)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("hq,t", [(8, 12), (64, 40)])
def test_masked_places_hold_anything(hq, t, dtype):
    """NaN and infinities behind the sequence and in drafted tokens reach nobody who does not see them."""
    lens, drafts = [200, 130, 77], [t, t, t]
    s = make(lens, drafts, [t, t, t], hq, 8, 32, "HND", dtype, seed=3, density=0.2)
    for b, (n, d) in enumerate(zip(lens, drafts)):
        last = int(s["block_table"][b, (n - 1) // 32])
        for c in (s["k_cache"], s["v_cache"]):
            if n % 32:
                c[last, :, n % 32:] = float("nan")            # the rest of the last page
            c[last, :, -1] = float("inf") if n % 32 else c[last, :, -1]
    check(s, "HND", dtype, max_seq_len=200, max_q_len=t)
    for b, (n, d) in enumerate(zip(lens, drafts)):
        for j, val in ((1, float("inf")), (4, float("-inf")), (5, float("nan"))):
            tok = n - d + j
            at = s["v_cache"][int(s["block_table"][b, tok // 32]), :, tok % 32]
            at[:, 3 * j:3 * j + 20] = val
        s["mask"][b * t:b * t + t // 2] &= ~0b110010          # half of the rows see none of the three
    check(s, "HND", dtype, max_seq_len=200, max_q_len=t)
    tok = lens[0] - drafts[0] + 2
    s["k_cache"][int(s["block_table"][0, tok // 32]), :, tok % 32] = float("nan")
    s["mask"][:t] &= ~0b100
    check(s, "HND", dtype, max_seq_len=200, max_q_len=t)


def test_nan_that_is_seen_stays():
    s = make([150], [4], [4], 8, 1, 16, "HND", "bf16")
    s["q"][2, 3] = float("nan")
    s["k_cache"][int(s["block_table"][0, 0]), 0, 5] = 1e30    # scores far beyond the others, of either sign (fp32 holds them; 3e38 overflows it)
    o, lse = attention.tree_decode(*s.values())
    assert torch.isnan(o[2, 3]).all() and torch.isnan(lse[2, 3])
    rest = torch.ones(4, 8, dtype=torch.bool, device="cuda")
    rest[2, 3] = False
    s2 = dict(s, q=s["q"].nan_to_num())
    want, want_lse, _ = exact(s2, "HND")
    big = torch.isfinite(want_lse) & rest & (want_lse.abs() < 1e30)
    assert torch.allclose(o[big].double(), want[big], atol=2e-2)


@pytest.mark.parametrize("scale", [0.02, 1.0, 30.0])
def test_scales_and_peaked_scores(scale):
    s = make([700, 90], [5, 5], [5, 5], 16, 2, 16, "HND", "fp16", seed=8)
    if scale < 2:
        check(s, "HND", "fp16", scale=scale, max_seq_len=700, max_q_len=5)
        return
    # one token takes nearly all: scores up to 1000, so fp32 scores are off by up to 1000 * 2^-17
    o, lse = attention.tree_decode(*s.values(), scale=scale)
    want, want_lse, a = exact(s, "HND", scale)
    assert ((lse.double() - want_lse).abs() <= 1e-5 * want_lse.abs() + 0.02).all()
    assert ((o.double() - want).abs() <= 0.05 * (a + want.abs()) + 0.05).all()


def test_many_sequences():
    rng = np.random.default_rng(1)
    lens = [int(x) for x in rng.integers(0, 90, 700)]
    counts = [int(x) for x in rng.integers(0, 4, 700)]
    s = make(lens, [min(n, c) for n, c in zip(lens, counts)], counts, 8, 2, 16, "HND", "bf16")
    check(s, "HND", "bf16", max_seq_len=90, max_q_len=3)


@pytest.mark.parametrize("t,hq", [(2, 8), (9, 64)])
def test_short_units_one_after_the_other(t, hq):
    """Segments of one KV tile, many to a CTA, in which one of the two streams has nothing to do; with longer ones between."""
    lens = [1 + 7 * i % 128 for i in range(400)] + [128 * (1 + i % 3) - i % 2 for i in range(60)] + [5] * 40
    s = make(lens, [min(n, t) for n in lens], [t] * len(lens), hq, hq // 8, 16, "HND", "fp16", seed=t)
    first = check(s, "HND", "fp16", max_seq_len=384, max_q_len=t)
    for _ in range(20):
        again = attention.tree_decode(*s.values(), max_seq_len=384, max_q_len=t)
        assert torch.equal(again[0], first[0]) and torch.equal(again[1], first[1])


def test_long_sequence_and_shards_of_it():
    """The shards' outputs, combined, are the attention over the whole."""
    from helix_a2a_b200 import lse_combine
    t = 24
    s = make([20000], [t], [t], 16, 2, 16, "HND", "bf16", seed=5)
    whole = check(s, "HND", "bf16", max_seq_len=20000, max_q_len=t)
    part = []
    table = s["block_table"]
    for pages, d in ((slice(0, 400), 0), (slice(400, 1250), t)):
        bt = table[:, pages].contiguous()
        n = min(20000, pages.stop * 16) - pages.start * 16
        part.append(attention.tree_decode(s["q"], s["k_cache"], s["v_cache"], bt, torch.tensor([n], dtype=torch.int32, device="cuda"), s["q_start"],
                                          torch.tensor([d], dtype=torch.int32, device="cuda"), s["mask"]))
    o = lse_combine(torch.stack([p[0] for p in part]), torch.stack([p[1] for p in part]))
    # three outputs, each within 2^-8 (A + |o|) and A <= 5 of N(0, 1) values at 20000 tokens
    assert (o.float() - whole[0].float()).abs().max() < 3 * 2 ** -8 * 2


def test_strides_and_views():
    s = make([260, 31], [6, 6], [6, 6], 16, 2, 16, "NHD", "bf16", seed=2)
    want = attention.tree_decode(*s.values(), layout="NHD")
    qkv = torch.randn(12, 40, 128, device="cuda").bfloat16()
    qkv[:, :16] = s["q"]
    both = torch.randn(*s["k_cache"].shape[:2], 2, 2, 128, device="cuda").bfloat16()
    both[:, :, 0], both[:, :, 1] = s["k_cache"], s["v_cache"]
    wide = torch.full((2, 50), -1, dtype=torch.int32, device="cuda")
    wide[:, 3:3 + s["block_table"].shape[1]] = s["block_table"]
    masks = torch.zeros(12, 3, dtype=torch.int64, device="cuda")
    masks[:, :1] = s["mask"]
    got = attention.tree_decode(qkv[:, :16], both[:, :, 0], both[:, :, 1], wide[:, 3:3 + s["block_table"].shape[1]], s["seq_lens"], s["q_start"],
                                s["draft_lens"], masks[:, :1], layout="NHD")
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("page", [16, 32, 128])
@pytest.mark.parametrize("layout,hkv", [("HND", 1), ("HND", 3), ("NHD", 1), ("NHD", 3)])
def test_caches_whose_pages_and_heads_lie_apart(layout, hkv, page):
    """Gaps between tokens, heads and pages, one page only, a page that is not there."""
    for ctx in ([700, 90], [min(page, 90)] * 1):
        n = len(ctx)
        s = make(ctx, [5] * n, [5] * n, 4 * hkv, hkv, page, layout, "bf16", seed=page + hkv)
        want = attention.tree_decode(*s.values(), layout=layout)
        for pad in ((0, 1, 0, 0), (0, 0, 1, 0), (1, 0, 0, 0), (0, 1, 1, 0), (0, 0, 0, 8)):
            c = {}
            for i, name in enumerate(("k_cache", "v_cache")):
                shape = s[name].shape
                room = torch.full([a + b for a, b in zip(shape, pad)], float("nan"), dtype=torch.bfloat16, device="cuda")
                c[name] = room[tuple(slice(0, x) for x in shape)]
                c[name].copy_(s[name])
            got = attention.tree_decode(*dict(s, **c).values(), layout=layout)
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    # pages outside the cache are pages of zeros, and what lies behind the cache in memory is not read
    s = make([3 * page], [0], [2], hkv, hkv, page, layout, "bf16")
    for bad in (s["k_cache"].shape[0], 2 ** 28 + 1, 2 ** 31 - 1, -1):
        t = dict(s, block_table=s["block_table"].clone(), k_cache=torch.cat([s["k_cache"], torch.full_like(s["k_cache"], 1e30)])[:len(s["k_cache"])])
        t["block_table"][0, 1] = bad
        zero = dict(s, k_cache=torch.cat([s["k_cache"], torch.zeros_like(s["k_cache"][:1])]), v_cache=torch.cat([s["v_cache"], torch.zeros_like(s["v_cache"][:1])]),
                    block_table=s["block_table"].clone())
        zero["block_table"][0, 1] = s["k_cache"].shape[0]
        got, want = attention.tree_decode(*t.values(), layout=layout), attention.tree_decode(*zero.values(), layout=layout)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_rows_before_the_first_sequence():
    s = make([90, 40], [4, 4], [4, 4], 16, 2, 16, "HND", "bf16", pad=7)
    t = {k: torch.cat([torch.randn_like(v[:3]) if v.is_floating_point() else v[:3], v]) if k in ("q", "mask") else v for k, v in s.items()}
    t["q_start"] = s["q_start"] + 3
    torch.full((1 << 22,), float("nan"), device="cuda")                     # what fresh memory may hold
    o, lse = check(t, "HND", "bf16")
    assert not o[:3].any() and (lse[:3] == -math.inf).all()


def test_graph_replays_follow_their_inputs():
    s = make([900, 400, 130], [9, 9, 9], [9, 9, 9], 32, 4, 16, "HND", "bf16", seed=4)
    eager = attention.tree_decode(*s.values(), max_seq_len=900, max_q_len=9)
    st = torch.cuda.Stream()
    with torch.cuda.stream(st):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            o, lse = attention.tree_decode(*s.values(), max_seq_len=900, max_q_len=9)
        g.replay()
    st.synchronize()
    assert torch.equal(o, eager[0]) and torch.equal(lse, eager[1])
    s["seq_lens"].copy_(torch.tensor([901 - 120, 9, 129]))
    s["q_start"].copy_(torch.tensor([0, 9, 12, 20]))           # fewer rows: the rest are padding
    g.replay()
    torch.cuda.synchronize()
    want, want_lse, a = exact(s, "HND")
    assert ((o.double() - want).abs() <= 2 ** -8 * (a + want.abs()) + 2e-4 * a).all()
    assert not o[20:].any() and (lse[20:] == -math.inf).all()


def test_calls_at_once():
    """Split calls on two streams, and graphs of both replayed together, have each its own scratch."""
    kw = dict(max_seq_len=6000, max_q_len=20)
    inputs = [make([6000, 3000], [20, 20], [20, 20], 32, 4, 16, "HND", "bf16", seed=s) for s in (1, 2)]
    want = [attention.tree_decode(*s.values(), **kw) for s in inputs]
    streams, graphs, outs = [torch.cuda.Stream() for _ in inputs], [], []
    torch.cuda.synchronize()
    for _ in range(10):
        got = []
        for s, st in zip(inputs, streams):
            with torch.cuda.stream(st):
                got.append(attention.tree_decode(*s.values(), **kw))
        torch.cuda.synchronize()
        for g, w in zip(got, want):
            assert torch.equal(g[0], w[0]) and torch.equal(g[1], w[1])
    for s, st in zip(inputs, streams):
        with torch.cuda.stream(st):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=st):
                outs.append([attention.tree_decode(*s.values(), **kw) for _ in range(3)])
            graphs.append(g)
    torch.cuda.synchronize()
    for _ in range(5):
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
        eager = attention.tree_decode(*inputs[0].values(), **kw)
        torch.cuda.synchronize()
        for o, w in zip(outs, want):
            for x in o:
                assert torch.equal(x[0], w[0]) and torch.equal(x[1], w[1])
        assert torch.equal(eager[0], want[0][0])


@pytest.mark.parametrize("lens,counts,hq,hkv", [([9000], [64], 64, 8), ([5000, 3000, 700], [40, 40, 40], 64, 8), ([4000, 4100], [33, 60], 64, 8), ([6000], [150], 32, 4),
                                                ([3000, 0, 2000], [50, 9, 50], 96, 4), ([2500], [256], 64, 1), ([20000], [37], 56, 8),
                                                ([1000] * 150, [40] * 150, 8, 1)])
def test_groups_of_rows_side_by_side(lens, counts, hq, hkv):
    """Sequences with several groups of 256 rows each: as many for all of them, or not, and numbers that do not divide the CTAs."""
    drafts = [min(n, c) for n, c in zip(lens, counts)]
    s = make(lens, drafts, counts, hq, hkv, 16, "HND", "bf16", words=4, pad=3, seed=len(lens))
    check(s, "HND", "bf16", max_seq_len=max(lens), max_q_len=max(counts))
    check(s, "HND", "bf16")


def test_same_call_same_bits():
    s = make([5000, 17, 2600], [30, 10, 30], [30, 10, 30], 64, 8, 16, "HND", "bf16", seed=6)
    first = attention.tree_decode(*s.values(), max_seq_len=5000, max_q_len=30)
    for _ in range(5):
        again = attention.tree_decode(*s.values(), max_seq_len=5000, max_q_len=30)
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


def test_cache_beyond_32_bit_offsets():
    """Pages whose byte offsets need more than 32 bits, and drafted values that are read from the cache itself there."""
    pool = 150000                                               # 16 tokens x 2 heads x 256 bytes: 1.2 GB each, 9 times
    k = torch.zeros(pool * 4, 2, 16, 128, dtype=torch.bfloat16, device="cuda")
    v = torch.zeros_like(k)
    s = make([100], [6], [6], 4, 2, 16, "HND", "bf16", seed=11)
    table = s["block_table"].clone()
    for i in range(7):
        old, new = int(table[0, i]), pool * 4 - 1 - 3 * i
        k[new], v[new] = s["k_cache"][old], s["v_cache"][old]
        table[0, i] = new
    tok = 100 - 6 + 2
    v[int(table[0, tok // 16]), :, tok % 16, 7] = float("inf")
    s.update(k_cache=k, v_cache=v, block_table=table)
    assert k.numel() * 2 > 2 ** 32
    check(s, "HND", "bf16", max_seq_len=100, max_q_len=6)


def test_bad_pages_are_not_read():
    """Page ids outside the cache count as pages of zeros; lengths that outgrow the table end there."""
    s = make([64], [0], [2], 8, 1, 16, "HND", "bf16")
    s["block_table"][0, 1] = 10 ** 9
    s["block_table"][0, 2] = -5
    o, lse = attention.tree_decode(*s.values())
    assert torch.isfinite(o).all() and torch.isfinite(lse).all()
    s["seq_lens"].fill_(10 ** 9)
    s["block_table"].zero_()
    o, lse = attention.tree_decode(*s.values())
    assert torch.isfinite(o).all()
    check_compute_status(o)


def test_refusals():
    s = make([50], [4], [4], 16, 2, 16, "HND", "bf16")

    def call(layout="HND", scale=None, **over):
        return attention.tree_decode(*dict(s, **over).values(), layout=layout, scale=scale)

    call()
    for bad in (dict(q=s["q"].half()), dict(q=s["q"].float()), dict(k_cache=s["k_cache"].half(), v_cache=s["v_cache"].half()), dict(q=s["q"][..., :64]),
                dict(q=s["q"][:, :15]), dict(k_cache=s["k_cache"][:, :1]), dict(seq_lens=s["seq_lens"].long()), dict(q_start=s["q_start"][:1]),
                dict(draft_lens=s["draft_lens"].cpu()), dict(mask=s["mask"].int()), dict(mask=s["mask"][:3]), dict(mask=s["mask"].repeat(1, 5)),
                dict(block_table=s["block_table"].repeat(2, 1)), dict(block_table=s["block_table"].long()), dict(scale=0.0), dict(scale=-1.0),
                dict(scale=float("nan")), dict(scale=float("inf")), dict(k_cache=s["k_cache"][:, :, :15], v_cache=s["v_cache"][:, :, :15])):
        with pytest.raises(RuntimeError):
            call(**bad)
    with pytest.raises(ValueError):
        call(layout="hnd")


def test_no_rows_and_no_sequences():
    s = make([50], [4], [4], 16, 2, 16, "HND", "bf16")
    o, lse = attention.tree_decode(s["q"][:0], s["k_cache"], s["v_cache"], s["block_table"], s["seq_lens"], s["q_start"] * 0, s["draft_lens"], s["mask"][:0])
    assert o.shape == (0, 16, 128) and lse.shape == (0, 16)
    o, lse = attention.tree_decode(s["q"], s["k_cache"], s["v_cache"], s["block_table"][:0], s["seq_lens"][:0], s["q_start"][:1], s["draft_lens"][:0], s["mask"])
    assert not o.any() and (lse == -math.inf).all()
