"""CPU-only: the dynamic-quantisation entry points refuse bad arguments before any CUDA call,
and the Python operators refuse CPU tensors."""
import ctypes

import pytest
import torch

from texo_b200 import _lib, ops


@pytest.fixture(scope="module")
def lib(libs):
    return _lib.load()


PTR = ctypes.c_void_p(4096)  # never dereferenced: every call here is refused


def test_mm_entry_point_refuses(lib):
    good = [PTR, PTR, PTR, 4, 32, 16, PTR, PTR, None, 0, None, 0, None]
    for at, value in ((0, None), (1, None), (2, None), (3, 0), (3, -1), (4, 0), (5, -1), (6, None), (7, None),
                      (9, 3), (9, -1)):
        args = list(good)
        args[at] = value
        assert lib.texo_mm_int8_solve_per_token(*args) == -1, (at, value)


def test_block_norm_entry_points_refuse(lib):
    f16, bf16, f32 = 0, 1, 2
    good = [PTR, PTR, PTR, None, PTR, PTR, PTR, 6, 64, 3, 1, 1e-5, 1.0, f16, f16, 0, None]
    for at, value in ((0, None), (1, None), (2, None), (5, None), (6, None), (7, 0), (8, 0), (9, 0), (9, 4),
                      (13, 3), (14, bf16), (14, 5)):
        args = list(good)
        args[at] = value
        assert lib.texo_block_norm_solve(*args) == -1, (at, value)
        args.insert(6, None if at == 6 else PTR)  # the scales; z moves on by one
        if at == 6:
            args[7] = PTR
        assert lib.texo_block_norm_quant_solve(*args) == -1, (at, value)
    args = list(good)
    args[13], args[14] = f32, f16
    assert lib.texo_block_norm_solve(*args) == -1


def test_quantiser_entry_points_refuse(lib):
    for at, value in ((0, None), (1, None), (2, None), (3, 0), (4, 0), (5, 63), (6, 7)):
        args = [PTR, PTR, PTR, 4, 64, 64, 0, None]
        args[at] = value
        assert lib.texo_quant_per_token_solve(*args) == -1, (at, value)
        args = [PTR, PTR, PTR, 4, 32, 64, 0, 0, None]
        args[at if at < 6 else 7] = value
        assert lib.texo_swiglu_quant_per_token_solve(*args) == -1, (at, value)


def test_operators_have_no_cpu_path():
    a, s = torch.zeros((4, 16), dtype=torch.int8), torch.ones(4)
    with pytest.raises(ValueError, match="CUDA"):
        ops.mm_int8_per_token(a, a.t().contiguous(), s, s)
    x = torch.zeros((4, 16))
    for call in (lambda: ops.block_norm(x, x, x[0], 1e-5), lambda: ops.quant_per_token(x),
                 lambda: ops.block_norm_quant_per_token(x, x, x[0], 1e-5), lambda: ops.swiglu_quant_per_token(x)):
        with pytest.raises(ValueError, match="CUDA"):
            call()
