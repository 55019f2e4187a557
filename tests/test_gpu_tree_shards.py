"""tree_decode over the shards of a long sequence, shard by shard and combined, with drafted tokens that take a visible part of the softmax.

Tolerances, with e = eps / 2 of bf16, A = sum_j p_j |v_j| and S = scale * max_j sum_d |q_d k_jd|: fp32 scores of 128 products are off by at
most D = 128 * 2^-24 S, and 1e-4 covers the exponentials and sums as in test_gpu_tree_decode.  Probabilities are then off by a factor of
at most exp(2 (D + 1e-4)), which moves an output by less than 3 (D + 1e-4) A; P's rounding moves it by e A and its own by e |o|.  The LSE is off by
D + 2e-4.  Combined, the shards' errors are weighted like the shards, the weights themselves are off like the LSEs, and one rounding is added.
"""
import math

import pytest
import torch

from helix_a2a_b200 import lse_combine
from helix_a2a_b200.ops import attention
from helix_a2a_b200.ops.oproj import check_compute_status
from test_gpu_tree_decode import exact, make

pytestmark = pytest.mark.gpu
E = 2.0 ** -8


def score_error(s, hkv):
    k = s["k_cache"].double().abs().transpose(0, 1).flatten(1, 2)                           # [hkv, tokens of the cache, 128]
    q = s["q"].double().abs().unflatten(1, (hkv, -1))
    most = torch.stack([(q[:, h] @ k[h].t()).amax(-1) for h in range(hkv)], 1)
    return 128 * 2.0 ** -24 * most.flatten(1) / math.sqrt(128)


def compare(got, s, hkv):
    """Check o and lse of one call against float64; returns both and the tolerance of o."""
    o, lse, a = exact(s, "HND")
    d = score_error(s, hkv)
    tol = E * (a + o.abs()) + 3 * (d[..., None] + 1e-4) * a
    assert ((got[0].double() - o).abs() <= tol).all()
    assert ((got[1].double() - lse).abs() <= d + 2e-4).all()
    return o, lse, a, tol, d


@pytest.mark.parametrize("t,hq,hkv", [(24, 16, 2), (5, 8, 1), (40, 32, 4)])
@pytest.mark.parametrize("cut", [400, 1240])
def test_shards_and_their_combination(cut, t, hq, hkv):
    n, page = 20000, 16
    s = make([n], [t], [t], hq, hkv, page, "HND", "bf16", seed=5 + t)
    for j in range(n - t, n):                                                               # the drafted tokens: scores of N(0, 144)
        s["k_cache"][int(s["block_table"][0, j // page]), :, j % page] *= 12
    s["mask"][0::2], s["mask"][1::2] = 0x5555555555555555, 0x2AAAAAAAAAAAAAAA                # every other one
    kw = dict(max_seq_len=n, max_q_len=t)
    whole = attention.tree_decode(*s.values(), **kw)
    o, lse, a, tol, d = compare(whole, s, hkv)

    parts = []
    for pages, drafts in ((slice(0, cut), 0), (slice(cut, n // page), t)):
        i32 = dict(dtype=torch.int32, device="cuda")
        shard = dict(s, block_table=s["block_table"][:, pages].contiguous(), seq_lens=torch.tensor([(pages.stop - pages.start) * page], **i32),
                     draft_lens=torch.tensor([drafts], **i32))
        got = attention.tree_decode(*shard.values(), **kw)
        parts.append((got, compare(got, shard, hkv)))
    # what the test is for: had the second shard seen none or all of its drafted tokens, or other ones, it would show in every row
    right = parts[1][1][0]
    for mask in (torch.zeros_like(s["mask"]), torch.full_like(s["mask"], -1), s["mask"] << 1):
        wrong = exact(dict(shard, mask=mask), "HND")[0]
        assert ((wrong - right).abs() > 4 * parts[1][1][3]).flatten(1).any(1).all()

    combined, combined_lse = lse_combine(torch.stack([p[0][0] for p in parts]), torch.stack([p[0][1] for p in parts]), return_lse=True)
    weights = [torch.exp(p[1][1] - lse)[..., None] for p in parts]
    tol = sum(w * p[1][3] for w, p in zip(weights, parts)) + E * o.abs() + 3 * (d[..., None] + 2e-4) * a
    assert ((combined.double() - o).abs() <= tol).all()
    assert ((combined_lse.double() - lse).abs() <= d + 4e-4).all()
    check_compute_status(s["q"])
