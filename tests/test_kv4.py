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


def test_storage_holds_five_bits_a_number():
    from wick_b200.cache import PAGE, Cache, PagedKV4
    from wick_b200.parts.base import CacheNeed
    need = CacheNeed("paged_kv4", kv_heads=3, head_dim=64, dtype=torch.uint8)
    c = Cache([need, need], max_tokens=640, dtype=torch.float32, device="cpu")
    store = c.groups[0].store
    assert isinstance(store, PagedKV4) and store.tensor.shape == (2, 11, 3, 80 * 64) and store.tensor.dtype == torch.uint8
    assert c.bytes_per_token() == 2 * 3 * 2 * 64 * 5 // 8 and c.read_bytes(70, 2) == 70 * c.bytes_per_token()
    assert c.storage_bytes() == 11 * PAGE * c.bytes_per_token()
    store.tensor[:, 3] = 7
    c.copy_pages(torch.tensor([3]), torch.tensor([5]))
    assert (store.tensor[:, 5] == 7).all() and (store.tensor[:, 4] == 0).all() and not c.cannot_copy()
    for bad in (dict(dtype=torch.float32), dict(dtype=torch.uint8, v_head_dim=128), dict(dtype=torch.uint8, window=5)):
        with pytest.raises(ValueError):
            Cache([CacheNeed("paged_kv4", kv_heads=3, head_dim=64, **bad)], max_tokens=64, dtype=torch.float32, device="cpu", allocate=False)


def test_a_model_says_which_of_its_parts_do_not_take_part():
    import wick_b200 as wick
    from helpers import CONFIGS
    from wick_b200.models.qwen3 import build_spec
    spec = build_spec(wick.config_from_json(CONFIGS["D"]))
    m = wick.Model(spec, torch.bfloat16, "cpu", cache_bits=4)
    assert all(n.kind == "paged_kv4" for n in m.cache_needs())
    assert all(n.kind == "paged_kv" for n in wick.Model(spec, torch.bfloat16, "cpu").cache_needs())
    from test_nibotar_config import CONFIG
    cfg = wick.config_from_json(CONFIG)
    with pytest.raises(ValueError, match="do not keep their cache in 4 bits"):
        wick.Model(wick.get_architecture(cfg.architecture).build_spec(cfg), torch.bfloat16, "cpu", cache_bits=4)
    with pytest.raises(ValueError, match="2 bits"):
        wick.Model(spec, torch.bfloat16, "cpu", cache_bits=2)
    with pytest.raises(ValueError, match="head sizes"):
        wick.Model(build_spec(wick.config_from_json(CONFIGS["A"])), torch.bfloat16, "cpu", cache_bits=4)


def test_command_line_option():
    from wick_b200 import cli
    assert cli.parse_args(["run", "d", "--cache-bits", "4"]).cache_bits == 4 and cli.parse_args(["run", "d"]).cache_bits is None
    with pytest.raises(cli.UsageError):
        cli.parse_args(["run", "d", "--cache-bits", "8"])


@pytest.mark.parametrize("d", [64, 256])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_scratch_is_enough_for_shorter_sequences(d, dtype):
    """A longer sequence may be cut into fewer pieces than a shorter one: a step has places for those of all lengths up to its bound."""
    import types
    from wick_b200 import ops
    for kv in (1, 2, 8, 32, 80):
        before = 0
        for pages in list(range(1, 90)) + list(range(90, 3000, 37)):
            b = types.SimpleNamespace(n_tokens=3, n_seqs=2, table_width=pages, max_q_len=2, kv_bound=64 * pages)
            words = ops.attention_kv4_scratch(b, 4 * kv, kv, d, dtype, kind="plain" if dtype == torch.float32 else "records")
            assert words >= before, (kv, pages)
            before = words
