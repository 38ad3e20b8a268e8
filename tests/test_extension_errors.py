"""A failed argument check of the extension reaches Python as an exception."""
import pytest
import torch


def test_failed_check_raises():
    from helexa_b200 import ops
    try:
        C = ops.C
    except ImportError:
        pytest.skip("extension not built")
    with pytest.raises(RuntimeError):
        C.gguf_quant_host(torch.zeros(256), 99)
    with pytest.raises(RuntimeError):
        C.embed(torch.zeros(4), torch.zeros(4), torch.zeros(4))
