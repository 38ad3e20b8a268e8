"""The 8-bit KV cache away from the kernels: planning, snapshots of a slot, refusals."""
import pytest
import torch

from helexa_b200.config import get_preset
from helexa_b200.ops.kv8 import BLOCK, KV8, bytes_per_token, tail_bytes
from helexa_b200.runtime.context_limit import ContextProfile, derive_limit


def test_profile_counts_codes_scales_and_tails():
    cfg = get_preset("qwen3-8b")
    a, b = ContextProfile.from_config(cfg), ContextProfile.from_config(cfg, 1, "int8")
    assert b.kv_bytes_per_token == 36 * 2 * 8 * (128 * 32 + 4) // 32
    assert b.state_bytes_per_seq == a.state_bytes_per_seq + 36 * 2 * 8 * BLOCK * 128 * 2
    free = 40 << 30
    la, lb = (derive_limit(p, free, concurrent=64) for p in (a, b))
    assert 1.9 * la.context < lb.context <= 2 * la.context  # twice the context, less scales and tails


def test_pool_size_is_what_planning_counts():
    for hkv, D, L in ((8, 128, 4096), (2, 256, 320), (2, 64, 32)):
        c = KV8.alloc(3, hkv, L, D, "fp8", "cpu")
        assert c.nbytes() == 3 * (L * bytes_per_token(hkv, D) + tail_bytes(hkv, D))
        assert c.head_dim == D


@pytest.mark.parametrize("D,dtype", [(96, "int8"), (32, "fp8"), (128, "bf16"), (128, "fp4")])
def test_alloc_refuses(D, dtype):
    with pytest.raises(ValueError):
        KV8.alloc(1, 1, 64, D, dtype, "cpu")


def _filled(dtype="int8"):
    c = KV8.alloc(2, 2, 160, 64, dtype, "cpu")
    g = torch.Generator().manual_seed(1)
    for t in c:
        t.view(torch.uint8).random_(0, 127, generator=g)
    return c


@pytest.mark.parametrize("length,held", [(0, 0), (0, 70), (64, 70), (65, 70), (70, 70), (96, 96), (90, 96), (32, 128)])
def test_snapshot_restores_what_a_continuation_reads(length, held):
    c = _filled()
    saved = c.snapshot(0, length, held)
    other = KV8.alloc(2, 2, 160, 64, "int8", "cpu")
    other.restore(1, saved)
    n = length // BLOCK
    for a, b in zip(c[:4], other[:4]):
        assert torch.equal(a[0, :, :n].view(torch.uint8), b[1, :, :n].view(torch.uint8))
        assert not b[0].any() and not b[1, :, n:].any()
    for a, b in zip(c[4:], other[4:]):
        assert torch.equal(a[0].view(torch.uint8), b[1].view(torch.uint8))
    c[0][0].zero_()  # a copy, not a view
    assert n == 0 or saved[0].any()


@pytest.mark.parametrize("length,held", [(33, 70), (63, 64), (1, 33), (71, 70), (-1, 5)])
def test_snapshot_refuses_cuts_whose_rows_are_gone(length, held):
    if (length, held) == (63, 64):  # inside the last block, which is complete: its rows are still there
        _filled().snapshot(0, length, held)
        return
    with pytest.raises(ValueError):
        _filled().snapshot(0, length, held)


def test_model_refuses():
    from helexa_b200.models.fast import DeviceError, FastModel
    cfg = get_preset("tiny-qwen3")
    for kv in ("int8", "int3"):
        with pytest.raises(ValueError):
            FastModel(cfg, [], torch.zeros(1), torch.zeros(1), torch.zeros(1), None, torch.device("cpu"), kv_dtype=kv)
    assert "position" in str(DeviceError(6001)) and "wait" in str(DeviceError(7004))
    assert "peer 3" in str(DeviceError(1003))


def test_node_refuses_kv_dtype():
    from helexa_b200.runtime.registry import LoadError, ModelSpec, build_served_model
    for kv in ("int8", "q4"):
        with pytest.raises(LoadError) as e:
            build_served_model(ModelSpec("m", "preset:tiny-qwen3", device="cpu", kv_dtype=kv))
        assert e.value.code == "bad_kv_dtype"
