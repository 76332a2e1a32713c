"""The cache in 4 bits, what needs no device: its form, how near its values are, and refusals."""
import pytest
import torch

from plain import kv4_plain as P


def test_values_are_near():
    """A number is off by half a step of its group's range, by what the two scales' roundings move the steps, and by the value's own rounding."""
    g = torch.Generator().manual_seed(0)
    for offset in (0.0, 1.0, 30.0):
        x = torch.randn((50, 2, 128), generator=g).double() + offset
        codes, a, b = P.encode(x)
        assert codes.min() == 0 and codes.max() == 15
        w = x.view(50, 2, 4, 32)
        reach, top = w.amax(-1) - w.amin(-1), w.abs().amax(-1)
        err = (P.decode(codes, a, b).view(50, 2, 4, 32) - w).abs().amax(-1)
        assert (err <= reach / 30 + 2.0 ** -8 * (top + 3 * reach)).all()


@pytest.mark.parametrize("d", [64, 128, 192, 256])
def test_a_page_has_every_code_once(d):
    g = torch.Generator().manual_seed(d)
    x = [P.encode(torch.randn((64, d), generator=g).double()) for _ in range(2)]
    data = P.page_bytes(*x)
    assert data.numel() == 80 * d and data.dtype == torch.uint8
    for i, (codes, _, _) in enumerate(x):
        part = data[i * 32 * d:(i + 1) * 32 * d].long()
        # (turning bytes or words and moving pieces keeps how often a bit is set)
        assert sum(int((part >> k & 1).sum()) for k in range(8)) == sum(int((codes >> k & 1).sum()) for k in range(4))


def test_without_a_device_calls_are_refused():
    from wick_b200 import ops
    kv, i32 = torch.zeros((3, 2, 80 * 64), dtype=torch.uint8), torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ops.KernelError):
        ops.kv4_read(kv, 64, i32.view(1, 2), i32, i32)
    with pytest.raises(ops.KernelError):
        ops.kv4_read(kv, 80, i32.view(1, 2), i32, i32)
    with pytest.raises(ops.KernelError):
        ops.qk_norm_rope_append_kv4(torch.zeros((2, 8 * 64)), 4, 2, 64, q_weight=None, k_weight=None, eps=0.0, cos=None, sin=None, kv=kv,
                                    page_table=i32.view(1, 2), seq_of_token=i32, positions=i32)
    with pytest.raises(ops.KernelError):
        ops.attention_kv4(torch.zeros((2, 4, 64)), kv, None, 0.1)
