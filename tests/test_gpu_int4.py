"""o_proj with 4-bit weights against float64.

Tolerance: products and sums are fp32, at most K + 2 K / group roundings of 2^-24 of the sum of magnitudes; the output is rounded once, eps / 2.
"""
import pytest
import torch

from helix_a2a_b200.ops import oproj

pytestmark = pytest.mark.gpu


def make(hidden, K, group, zeros, dtype, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    q = torch.randint(0, 16, (hidden, K), generator=g, dtype=torch.uint8, device="cuda")
    s = (torch.rand(hidden, K // group, generator=g, device="cuda") * 0.02 + 1e-3).to(dtype)
    s[1:2] *= -1
    z = torch.randint(0, 16, s.shape, generator=g, dtype=torch.uint8, device="cuda") if zeros else None
    w = oproj.pack_weight_int4(q[:, 0::2] | (q[:, 1::2] << 4), s, z)
    full = (q.double() - (8 if z is None else z.double().repeat_interleave(group, 1))) * s.double().repeat_interleave(group, 1)
    return w, full


def check(x, w, full):
    y = oproj.oproj(x, w)
    assert y.dtype == x.dtype and y.shape == (x.shape[0], w.hidden) and y.is_contiguous()
    want, mag = x.double() @ full.t(), x.double().abs() @ full.abs().t()
    tol = torch.finfo(x.dtype).eps / 2 * want.abs() + (w.K + 2 * w.K // w.group) * 2.0 ** -24 * mag
    bad = (y.double() - want).abs() > tol
    assert not bad.any(), (bad.nonzero()[:4].tolist(), int(bad.sum()), float((y.double() - want).abs().max()))
    return y


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("tokens", [1, 7, 8, 9, 16, 17, 33, 64, 65, 100, 128, 129, 300])
def test_types_groups_and_tokens(tokens, group, zeros, dtype):
    w, full = make(256, 1024, group, zeros, dtype)
    check(torch.randn(tokens, 1024, device="cuda").to(dtype), w, full)


@pytest.mark.parametrize("tokens", [1, 16, 40, 100])
@pytest.mark.parametrize("hidden,K,group", [(16, 64, 64), (16, 64, 32), (48, 192, 64), (1, 128, 128), (100, 256, 128), (130, 448, 64), (4096, 832, 32), (144, 4160, 32), (2048, 2048, 128), (8192, 1024, 128),
                                            (1024, 8192, 64), (32, 16384, 128), (48, 32768, 64), (20000, 320, 64), (7168, 4096, 128), (7168, 16384, 64),
                                            (9600, 32768, 32), (28672, 8192, 128)])
def test_shapes(hidden, K, group, tokens):
    w, full = make(hidden, K, group, True, torch.bfloat16, seed=K)
    check(torch.randn(tokens, K, device="cuda").bfloat16(), w, full)


@pytest.mark.parametrize("tokens", [3, 20])
def test_strided_rows_other_stream_and_graph(tokens):
    w, full = make(512, 2048, 128, False, torch.float16)
    wide = torch.randn(tokens, 2048 + 64, device="cuda").half()
    y = check(wide[:, 32:2080], w, full)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            out = oproj.oproj(wide[:, 32:2080], w)
        g.replay()
        s.synchronize()
        assert torch.equal(out, y)
        wide.mul_(-1)
        g.replay()
        s.synchronize()
        assert torch.equal(out, -y)


def test_infinities_and_nan_stay_in_their_row():
    w, full = make(64, 512, 64, True, torch.bfloat16)
    x = torch.randn(12, 512, device="cuda").bfloat16()
    clean = oproj.oproj(x, w)
    x[3, 17] = float("nan")
    x[9, 500] = float("inf")
    y = oproj.oproj(x, w)
    assert torch.isnan(y[3]).all() and not torch.isfinite(y[9]).any()
    rest = [i for i in range(12) if i not in (3, 9)]
    assert torch.equal(y[rest], clean[rest])


def test_same_call_same_bits():
    w, _ = make(7168, 8192, 128, True, torch.bfloat16)
    for tokens in (2, 48):
        x = torch.randn(tokens, 8192, device="cuda").bfloat16()
        first = oproj.oproj(x, w)
        assert all(torch.equal(first, oproj.oproj(x, w)) for _ in range(5))


def test_quantised_matrix():
    m = (torch.randn(512, 1024, device="cuda") * 0.02).bfloat16()
    x = torch.randn(6, 1024, device="cuda").bfloat16()
    for zp in (False, True):
        w = oproj.quantize_weight_int4(m, 128, zero_points=zp)
        check(x, w, oproj.unpack_weight_int4(w).double())


def test_no_tokens_and_refusals():
    w, _ = make(64, 256, 64, True, torch.bfloat16)
    assert oproj.oproj(torch.zeros(0, 256, dtype=torch.bfloat16, device="cuda"), w).shape == (0, 64)
    x = torch.zeros(4, 256, dtype=torch.bfloat16, device="cuda")
    oproj.oproj(x, w)
    odd = torch.zeros(4 * 264 + 1, dtype=torch.bfloat16, device="cuda")[1:].view(4, 264)
    for bad in (x.half(), x.float(), x[:, :128], x[0], odd[:, :256], torch.zeros(4, 257, dtype=torch.bfloat16, device="cuda")[:, :256], x.t()):
        with pytest.raises(RuntimeError):
            oproj.oproj(bad, w)
    for key, bad in (("packed", w.packed[:-16]), ("packed", w.packed.cpu()), ("packed", w.packed.view(torch.int32)), ("zeros", False), ("group", 32),
                     ("hidden", 160), ("group", 256), ("dtype", torch.float16), ("packed", torch.cat([w.packed[:1], w.packed])[1:])):
        broken = oproj.Int4OprojWeight(w.packed, w.hidden, w.K, w.group, w.dtype, w.zeros)
        setattr(broken, key, bad)
        with pytest.raises(RuntimeError):
            oproj.oproj(x, broken)
