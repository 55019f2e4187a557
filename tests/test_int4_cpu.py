"""4-bit weights on the CPU: packing, quantisation and refusals."""
import pytest
import torch

from helix_a2a_b200.ops import oproj


def arrays(hidden, K, group, zeros, dtype=torch.bfloat16, seed=0):
    g = torch.Generator().manual_seed(seed)
    q = torch.randint(0, 16, (hidden, K), generator=g, dtype=torch.uint8)
    s = (torch.rand(hidden, K // group, generator=g) + 0.1).to(dtype)
    z = torch.randint(0, 16, s.shape, generator=g, dtype=torch.uint8) if zeros else None
    return q, s, z


@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("hidden,K,group", [(16, 64, 32), (16, 64, 64), (48, 192, 64), (32, 256, 128), (128, 832, 32), (300, 384, 128), (1, 64, 32)])
def test_pack_and_unpack(hidden, K, group, zeros):
    q, s, z = arrays(hidden, K, group, zeros)
    w = oproj.pack_weight_int4(q[:, 0::2] | (q[:, 1::2] << 4), s, z)
    assert w.shape == (hidden, K) and w.group == group and w.packed.numel() == -(-hidden // 128) * 128 * (K // 2 + K // group * (3 if zeros else 2))
    want = (q.float() - (z.float() if zeros else torch.full(s.shape, 8.0)).repeat_interleave(group, 1)) * s.float().repeat_interleave(group, 1)
    assert torch.equal(oproj.unpack_weight_int4(w), want)
    x = torch.randn(3, K).bfloat16()
    assert torch.equal(oproj.oproj(x, w), (x.float() @ want.t()).bfloat16())


def test_layout():
    """The layout that csrc/oproj_int4.h states, nibble by nibble."""
    q, s, z = arrays(256, 192, 64, True)
    w = oproj.pack_weight_int4(q[:, 0::2] | (q[:, 1::2] << 4), s, z)
    slab = 192 * 64 + 3 * 384
    for row, col in ((0, 0), (0, 1), (5, 31), (127, 32), (130, 63), (255, 64), (200, 127), (129, 128), (250, 191)):
        rec, c = col // 128, col % 128
        at = row // 128 * slab + rec * (128 * 64 + 2 * 384) + row % 128 // 16 * (256 if rec else 512) * 2 + c // 32 * 256 + row % 16 * 16 + c % 32 // 8 * 4
        word = int.from_bytes(bytes(w.packed[at:at + 4].tolist()), "little")
        assert word >> (4 * (c % 8 // 2 + 4 * (c % 2))) & 15 == int(q[row, col])
    scale_at = slab + 128 * 64 + 256                       # slab 1, record 0, group 1
    order = [16 * tile + g + 8 * half for tile in range(8) for g in range(8) for half in range(2)]
    assert torch.equal(w.packed[scale_at:scale_at + 256].view(torch.bfloat16), s[128:, 1][order])
    zero_at = slab + 128 * 64 + 2 * 384 + 64 * 64 + 256    # slab 1, record 1, group 2
    assert torch.equal(w.packed[zero_at:zero_at + 128], z[128:, 2][order])


@pytest.mark.parametrize("zero_points", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_quantisation_is_off_by_half_a_step(dtype, zero_points):
    w = (torch.randn(64, 256) * 0.02 + 0.01).to(dtype)
    w[3] = 0
    w[4, :64] = 0.5
    pw = oproj.quantize_weight_int4(w, 64, zero_points=zero_points)
    step = torch.cat([sc[0, :, :4].permute(1, 3, 2, 0).reshape(64, -1) for _, _, sc, _ in pw.records()], 1).float().repeat_interleave(64, 1)
    # half a step for the rounding; the scale and the zero point are rounded too, which the ends of the range feel (up to 7.5 steps
    # eps / 2 each, and with zero points another half step where the range is clamped)
    tol = step * (0.5 + 8 * torch.finfo(dtype).eps + (0.5 if zero_points else 0))
    assert ((oproj.unpack_weight_int4(pw) - w.float()).abs() <= tol).all()
    assert not oproj.unpack_weight_int4(pw)[3].any()


def test_refusals():
    q, s, z = arrays(32, 128, 64, True)
    b = q[:, 0::2] | (q[:, 1::2] << 4)
    for bad in ((b.int(), s, z), (b, s.float(), z), (b, s[:, :1].repeat(1, 3), z), (b, s, z[:16]), (b, s, z.int()), (b, s, z + 16),
                (b[:, :16], s, z), (b[:0], s[:0], None)):
        with pytest.raises(ValueError):
            oproj.pack_weight_int4(*bad)
    w = torch.zeros(32, 128, dtype=torch.bfloat16)
    for bad in (w.float(), w[:0], w[:, :96], w[0]):
        with pytest.raises(ValueError):
            oproj.quantize_weight_int4(bad, 64)
    with pytest.raises(ValueError):
        oproj.quantize_weight_int4(w, 16)
