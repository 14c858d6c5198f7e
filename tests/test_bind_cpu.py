"""The native binding of the serving operators: it loads, exports its calls and
refuses bad arguments with ValueError before anything is launched (no GPU needed)."""

from __future__ import annotations

from importlib.machinery import ExtensionFileLoader
from importlib.util import module_from_spec, spec_from_file_location

import pytest
import torch

from torque_mlx_b200 import _lib


@pytest.fixture(scope="module")
def bind():
    from torque_mlx_b200.build import build_library
    build_library()
    spec = spec_from_file_location("_torch_bind", _lib.BIND_PATH,
                                   loader=ExtensionFileLoader("_torch_bind", str(_lib.BIND_PATH)))
    module = module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def test_exports(bind):
    for name in ("paged_append", "paged_attend", "paged_dequantize", "gemv_w4", "verify_drafts"):
        assert callable(getattr(bind, name))


def test_argument_counts(bind):
    for name in ("paged_append", "paged_attend", "paged_dequantize", "gemv_w4", "verify_drafts"):
        with pytest.raises(ValueError, match="arguments"):
            getattr(bind, name)(None)


def test_refusals_name_what_is_wrong(bind):
    with pytest.raises(ValueError, match="target_probs must be a torch tensor"):
        bind.verify_drafts([0.5], None, None, None, None, None)
    with pytest.raises(ValueError, match="CUDA tensor"):
        bind.verify_drafts(torch.zeros(1, 2, 4), None, None, None, None, None)
    codes = torch.zeros(16, dtype=torch.uint8)
    with pytest.raises(ValueError, match=r"x must be \[tokens, 128\]"):
        bind.gemv_w4(codes, codes, 32, 128, 64, torch.zeros(2, 64, dtype=torch.bfloat16), 0, None, 0.0, None, None)
    with pytest.raises(ValueError, match="group_size must be an integer"):
        bind.gemv_w4(codes, codes, 32, 128, "64", torch.zeros(2, 64), 0, None, 0.0, None, None)


@pytest.mark.skipif(torch.cuda.is_available(), reason="checks the no-GPU failure path")
def test_serving_operators_fail_loudly_without_gpu(bind):
    import torque_mlx_b200 as tq
    with pytest.raises(RuntimeError, match="CUDA device"):
        tq.PagedKV8Cache(4, kv_heads=1, head_dim=64)
    with pytest.raises(RuntimeError, match="CUDA device"):
        tq.verify_drafts(torch.zeros(1, 1, 4), None, torch.zeros(1, 0, dtype=torch.int32), torch.zeros(1, 0),
                         torch.ones(1, 4))
    with pytest.raises(RuntimeError, match="CUDA device"):
        tq.W4Weight.quantize(torch.zeros(16, 64))
