"""CPU-only: the Python operators refuse sizes that a C int does not hold, instead of passing their low
32 bits on.  Meta tensors stand in for CUDA tensors of those sizes; nothing is computed."""
import pytest
import torch

from texo_b200 import ops

BIG = 2 ** 32 + 64  # its low 32 bits make a small, valid size


def meta(*shape, dtype=torch.float16):
    return torch.empty(shape, dtype=dtype, device="meta")


def int8(*shape):
    return meta(*shape, dtype=torch.int8)


def f32(*shape):
    return meta(*shape, dtype=torch.float32)


def u8(*shape):
    return meta(*shape, dtype=torch.uint8)


Q = (1.0, 1.0, 1.0, 0, 0, 0)
CALLS = {
    "mm_int8_per_token M": lambda: ops.mm_int8_per_token(int8(BIG, 16), int8(16, 16), f32(BIG), f32(16)),
    "mm_int8_per_token N": lambda: ops.mm_int8_per_token(int8(16, 16), int8(16, BIG), f32(16), f32(BIG)),
    "mm_int8_per_token K": lambda: ops.mm_int8_per_token(int8(16, BIG), int8(BIG, 16), f32(16), f32(16)),
    "block_norm N": lambda: ops.block_norm(meta(BIG, 8), meta(BIG, 8), meta(8), 1e-5),
    "block_norm C": lambda: ops.block_norm(meta(1, BIG), meta(1, BIG), meta(BIG), 1e-5),
    "block_norm_quant_per_token C": lambda: ops.block_norm_quant_per_token(meta(1, BIG), meta(1, BIG), meta(BIG), 1e-5),
    "quant_per_token N": lambda: ops.quant_per_token(meta(BIG, 1)),
    "quant_per_token C": lambda: ops.quant_per_token(meta(1, BIG)),
    "swiglu_quant_per_token N": lambda: ops.swiglu_quant_per_token(meta(BIG, 2)),
    "swiglu_quant_per_token F": lambda: ops.swiglu_quant_per_token(meta(1, 2 * BIG)),
    "mm_int8 M": lambda: ops.mm_int8(int8(BIG, 16), int8(16, 16), *Q),
    "mm_int8_per_channel N": lambda: ops.mm_int8_per_channel(int8(1, 16), int8(16, BIG), 1.0, f32(BIG), 1.0, 0, None, 0),
    "mm_int8_per_group K": lambda: ops.mm_int8_per_group(int8(1, BIG), int8(BIG, 16), BIG, 1.0, f32(1, 16), 1.0, 0, 0, 0),
    "mm_int8_swiglu F": lambda: ops.mm_int8_swiglu(int8(1, 16), int8(16, 2 * BIG), 1.0, 1.0, 1.0, 1.0, 0, 0, 0, 0),
    "mm_int8_dequant K": lambda: ops.mm_int8_dequant(int8(1, BIG), int8(BIG, 16), 1.0, 1.0, 0, 0),
    "mm_int4 N": lambda: ops.mm_int4(meta(1, 16), u8(BIG, 8), meta(BIG, 1), 16),
    "mm_int4a8 K": lambda: ops.mm_int4a8(int8(1, BIG), u8(16, BIG // 2), *Q),
    "mm_int4a8_per_channel M": lambda: ops.mm_int4a8_per_channel(int8(BIG, 16), u8(16, 8), 1.0, f32(16), 1.0, 0, None, 0),
    "mm_int4a8_per_group M": lambda: ops.mm_int4a8_per_group(int8(BIG, 16), u8(16, 8), 16, 1.0, f32(16, 1), 1.0, 0, 0, 0),
    "dequantization M": lambda: ops.dequantization(f32(BIG, 4), f32(BIG, 4), 1),
    "dequantization T": lambda: ops.dequantization(f32(4, 4), f32(1, 1), BIG),
    "rms_norm_w_residual N": lambda: ops.rms_norm_w_residual(f32(BIG, 4), f32(BIG, 4), f32(4), 1e-5),
    "rms_norm_quant C": lambda: ops.rms_norm_quant(f32(1, BIG), f32(1, BIG), f32(BIG), 1e-5, 1.0, 0),
    "Int8Weights K": lambda: ops.Int8Weights(int8(BIG, 16)),
}


@pytest.mark.parametrize("name", CALLS)
def test_sizes_past_32_bits_are_refused(monkeypatch, name):
    monkeypatch.setattr(ops, "_check_cuda", lambda *a: None)
    monkeypatch.setattr(ops, "_check_float", lambda n, t: ops._TYPE_CODES[t.dtype])
    monkeypatch.setattr(ops, "_check_rows", lambda n, t: ops._TYPE_CODES[t.dtype])

    def unreachable(*args):
        raise AssertionError("went past the checks")

    monkeypatch.setattr(ops._lib, "load", unreachable)
    monkeypatch.setattr(ops, "_matrix", unreachable)
    monkeypatch.setattr(ops, "_vector", unreachable)
    with pytest.raises(ValueError, match="2\\^31"):
        CALLS[name]()
