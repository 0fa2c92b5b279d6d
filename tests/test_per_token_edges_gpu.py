"""GPU tests of the dynamic-quantisation operators at the ends of their ranges: values, sizes,
errors of other calls, and the paths of the product that only large problems take.  Helpers and the
counting of roundings are those of test_per_token_gpu.py."""
import os
import random
import subprocess
import sys

import pytest

from tests.test_per_token_gpu import (BF16, F16, F32, U, assert_within, check_quantised, dtype, generator, half_step,
                                      mm_expected, mm_inputs, norm_expected, norm_inputs, ops)  # noqa: F401  (ops is a fixture)

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


# ------------------------------------------------------------------ SwiGLU far from zero
def far_rows(F, x_type, seed):
    """gate, up [8, F]: rows whose outputs are finite although exp(-gate), or gate * up, is not."""
    g = generator(seed)

    def between(lo, hi):
        return (torch.rand(F, generator=g, device="cuda") * (hi - lo) + lo).to(dtype(x_type))

    big = 6e4 if x_type == F16 else 1e38  # (2^126.2; an f16 gate of -87 and this make 5e-33)
    gates = [between(-104, -86), between(-170, -100), between(-20, -1), between(-90, -84), between(-300, -87),
             between(-8, 8), between(-90, 8), between(-88.8, -86.4)]
    ups = [between(0.5 * big, big), between(0.9 * big, big), between(0.5 * big, big), between(-2, 2), between(-2, 2),
           between(-2, 2), between(-1, 1) * min(big, 1e6), between(-big, big)]
    return torch.stack(gates), torch.stack(ups)


@pytest.mark.parametrize("F", [1, 2, 9, 64, 65, 1024, 1025, 8192, 8191, 20001, 28672, 40001])
@pytest.mark.parametrize("x_type", [F16, BF16, F32])
@pytest.mark.parametrize("interleaved", [True, False])
def test_swiglu_where_the_exponential_overflows(ops, F, x_type, interleaved):
    """In U, relative to y: 1.23 |gate| + 9 as the kernel counts them; gates below -80: the exponent
    of e^(gate / 2) is exact, the function two ulps (4), two of it, three products: 11.  The absolute
    2^-114 stands for gates below -174, where e^(gate / 2) is subnormal."""
    gate, up = far_rows(F, x_type, F)
    x = torch.stack([gate, up], dim=2).reshape(8, 2 * F) if interleaved else torch.cat([gate, up], dim=1)
    g64, u64 = gate.double(), up.double()
    y = g64 / (1 + torch.exp(-g64)) * u64
    assert bool((y.abs().amax(dim=1) < 3e38).all())
    dy = y.abs() * (1.24 * g64.abs().clamp_max(90) + 12) * U + 2.0 ** -114
    q, s = ops.swiglu_quant_per_token(x.contiguous(), interleaved=interleaved)
    check_quantised(q, s, y, dy)
    if x_type != F16:
        assert bool((q[:3].abs().amax(dim=1) == 127).all())  # rows of far gates have values
    part = x[5:6].contiguous()
    q1, s1 = ops.swiglu_quant_per_token(part, interleaved=interleaved)
    assert torch.equal(q1[0], q[5]) and torch.equal(s1[0], s[5])


@pytest.mark.parametrize("F", [64, 65, 8192, 40001])
@pytest.mark.parametrize("x_type", [F16, BF16, F32])
def test_swiglu_of_values_that_are_not_finite(ops, F, x_type):
    inf, nan = float("inf"), float("nan")
    rows = [(1.0, 1.0), (nan, 1.0), (1.0, nan), (inf, 1.0), (-inf, 1.0), (1.0, inf), (-100.0, inf), (-inf, 0.0), (2.0, -3.0)]
    gate = torch.full((len(rows), F), 0.5, dtype=dtype(x_type), device="cuda")
    up = torch.full_like(gate, 0.25)
    for r, (a, b) in enumerate(rows):
        gate[r, F - 1], up[r, F - 1] = a, b
    x = torch.cat([gate, up], dim=1)
    q, s = ops.swiglu_quant_per_token(x, interleaved=False)
    assert s.isnan().tolist() == [False] + [True] * 7 + [False]
    assert not bool(q[1:8].any()) and bool((q[0] != 0).all())


# ------------------------------------------------------------------ errors of other calls
@pytest.mark.parametrize("K", [0, 40, 131072])
def test_an_error_of_the_callers_is_left_alone(ops, K):
    """An error code that an earlier CUDA call of the caller's left behind is neither taken for the
    product's own nor cleared, whichever kernel runs (K = 0 and K = 2^17: the SIMT one)."""
    import ctypes

    M, N = 3, 32
    A, B, sa, sb, bias = mm_inputs(M, N, K, 6) if K else (
        torch.empty((M, 0), dtype=torch.int8, device="cuda"), torch.empty((0, N), dtype=torch.int8, device="cuda"),
        torch.ones(M, device="cuda"), torch.ones(N, device="cuda"), torch.ones(N, device="cuda"))
    want = ops.mm_int8_per_token(A, B, sa, sb, bias, out_dtype=torch.float32)
    out = torch.full_like(want, 7.0)
    torch.cuda.synchronize()
    runtime = ctypes.CDLL("libcudart.so.12")
    value = ctypes.c_int()
    invalid_device = 101
    assert runtime.cudaGetLastError() == 0
    assert runtime.cudaDeviceGetAttribute(ctypes.byref(value), 1, 4096) == invalid_device  # no such device
    try:
        assert runtime.cudaPeekAtLastError() == invalid_device
        ops.mm_int8_per_token(A, B, sa, sb, bias, out_dtype=torch.float32, out=out)
        assert runtime.cudaPeekAtLastError() == invalid_device
    finally:
        runtime.cudaGetLastError()
    assert torch.equal(out, want)


# ------------------------------------------------------------------ several tiles per cluster
# (M, N, K), path forced, path taken; on 148 SMs: R, CTAs of a cluster, clusters, tiles
ROUNDS = [
    ((1, 38976, 2576), 0, 2),     # 16, 3, 45, 153
    ((16, 57344, 8192), 0, 2),    # 16, 3, 45, 224: a wide fused gate/up projection in decode
    ((27, 38752, 3008), 0, 2),    # 32, 3, 45, 152
    ((56, 38576, 3504), 0, 2),    # 64, 4, 33, 151
    ((73, 19520, 7040), 0, 2),    # 128, 5, 26, 77
    ((87, 19392, 6816), 0, 2),    # 128, 3, 45, 76
    ((128, 57344, 8192), 0, 2),   # 128, 3, 45, 224
    ((384, 4096, 14336), 0, 2),   # 128, 5, 26, 48: three rows of tiles
    ((1, 38422, 1424), 0, 3),     # 16, 3, 45, 151, gathering from here on
    ((8, 21730, 1514), 0, 3),     # 16, 3, 45, 85
    ((64, 13220, 3113), 0, 3),    # 64, 5, 26, 52
    ((128, 13220, 3113), 3, 3),   # 128, 5, 26, 52
    ((128, 24020, 1483), 3, 3),   # 128, 4, 33, 94
    ((200, 9988, 4453), 3, 3),    # 128, 3, 45, 80: two rows of tiles
    ((16, 21728, 1536), 3, 3),    # 16, 3, 45, 85, aligned operands
    ((64, 13216, 3120), 3, 3),    # 64, 5, 26, 52, aligned operands
]


@pytest.mark.parametrize("shape,force,path", ROUNDS)
@pytest.mark.parametrize("out_type", [BF16, F32])
def test_mm_several_tiles_per_cluster(ops, shape, force, path, out_type):
    """A cluster that splits K and joins through its ring, tile after tile: the ring fills again only once
    the partials of the tile before have been read.  Three calls in a row on different activations,
    against 64 bits and, bit for bit, the SIMT kernel."""
    from texo_b200 import _lib

    M, N, K = shape
    t = dtype(out_type)
    A, B, sa, sb, bias = mm_inputs(M, N, K, M + N + K, full_range=True)
    batches = [A, A.flip(0).contiguous(), A.flip(1).contiguous()]
    ops.mm_int8_per_token(A[:1], B, sa[:1], sb)  # the device's set-up
    lib = _lib.load()
    lib.texo_mm_int8_per_token_force_path(force)
    try:
        got = [ops.mm_int8_per_token(a, B, sa, sb, bias, out_dtype=t) for a in batches]
        assert lib.texo_mm_int8_per_token_last_path() == path
        lib.texo_mm_int8_per_token_force_path(1)
        simt = [ops.mm_int8_per_token(a, B, sa, sb, bias, out_dtype=t) for a in batches]
        assert lib.texo_mm_int8_per_token_last_path() == 1
    finally:
        lib.texo_mm_int8_per_token_force_path(0)
    for a, y, want in zip(batches, got, simt):
        assert torch.equal(y, want)
    want, bound = mm_expected(A, B, sa, sb, bias, t)
    assert_within(got[0], want, bound)
    assert ops.status() == 0


def test_mm_several_tiles_per_cluster_on_two_streams_and_replayed(ops):
    cases = [mm_inputs(16, 38976, 2576, 1), mm_inputs(8, 21730, 1514, 2)]
    want = [ops.mm_int8_per_token(*c, out_dtype=torch.float32) for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    results = [[], []]
    for _ in range(10):
        for case, stream, kept in zip(cases, streams, results):
            with torch.cuda.stream(stream):
                kept.append(ops.mm_int8_per_token(*case, out_dtype=torch.float32))
    torch.cuda.synchronize()
    for w, kept in zip(want, results):
        assert all(torch.equal(w, y) for y in kept)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = [ops.mm_int8_per_token(*c, out_dtype=torch.float32) for c in cases]
    for _ in range(3):
        for o in outs:
            o.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(w, o) for w, o in zip(want, outs))
    assert ops.status() == 0


# ------------------------------------------------------------------ the quotient y / scale
def quotients(x):
    """x / scale and its scale as IEEE divisions give them, and the quotient in 64 bits."""
    top = x.float().abs().amax(dim=1).clamp_min(2.0 ** -100)
    scale = top / torch.full_like(top, 127.0)  # (a division by a tensor; by a number it is a product)
    return scale, x.float() / scale[:, None], x.double() / scale.double()[:, None]


@pytest.mark.parametrize("x_type", [F16, BF16])
@pytest.mark.parametrize("exponent", [-14, 0, 15, 100, 120])
def test_quotients_of_16_bit_values_are_those_of_a_division(ops, x_type, exponent):
    """Every row maximum of one binade against every value of the nine binades up to it (below, q = 0)."""
    if x_type == F16 and exponent > 15:
        pytest.skip("out of FP16's range")
    bits = 10 if x_type == F16 else 7
    steps = torch.arange(2 ** bits, device="cuda", dtype=torch.float64) / 2 ** bits + 1
    tops = steps * 2.0 ** exponent
    below = (steps[None] * 2.0 ** torch.arange(exponent - 8, exponent + 1, device="cuda", dtype=torch.float64)[:, None]).flatten()
    values = torch.minimum(below[None], tops[:, None])
    values = values * (1 - 2 * (torch.arange(values.shape[1], device="cuda") % 2))  # both signs
    x = torch.cat([tops[:, None], values], dim=1).to(dtype(x_type))
    q, s = ops.quant_per_token(x)
    scale, quotient, _ = quotients(x)
    assert torch.equal(s, scale)
    assert torch.equal(q.float(), torch.round(quotient))


@pytest.mark.parametrize("exponent", [0, -90, 105, 110, 127])
def test_quotients_next_to_ties(ops, exponent):
    """FP32 values up to three ulps around every tie, for a thousand row maxima: q is rint of the FP32 quotient
    but where the true one lies within 2^-45 (twice the documented distance) of the middle between two
    FP32 values, as one in 2^20 does, less than two of these 1.8 million.  Exact ties go to the even side."""
    g = generator(exponent + 200)
    rows = 1000
    # below 2^128: the largest mantissas are left to the smaller exponents
    tops = (1 + torch.rand(rows, generator=g, device="cuda", dtype=torch.float64) * 0.999).float() * 2.0 ** exponent
    scale = tops / torch.full_like(tops, 127.0)
    halves = torch.arange(-126, 126, device="cuda", dtype=torch.float64) + 0.5
    near = (scale.double()[:, None] * halves).float()
    ulps = torch.arange(-3, 4, device="cuda", dtype=torch.int32)
    near = (near.view(torch.int32)[:, :, None] + ulps).view(torch.float32).reshape(rows, -1)
    x = torch.cat([tops[:, None], near], dim=1)
    assert bool(torch.isfinite(x).all()) and bool((x.abs() <= tops[:, None]).all())
    q, s = ops.quant_per_token(x)
    scale, quotient, exact = quotients(x)
    assert torch.equal(s, scale)
    other = q.float() != torch.round(quotient)
    up = torch.nextafter(quotient, torch.full_like(quotient, float("inf"))).double()
    down = torch.nextafter(quotient, torch.full_like(quotient, float("-inf"))).double()
    to_middle = torch.minimum((exact - (quotient.double() + up) / 2).abs(), (exact - (quotient.double() + down) / 2).abs())
    assert not bool((other & (to_middle > exact.abs() * 2.0 ** -45)).any())
    assert int(other.sum()) <= 4
    tie = exact == torch.floor(exact) + 0.5
    assert torch.equal(q[tie].double(), torch.round(exact[tie]))


@pytest.mark.parametrize("C", [64, 1001, 8192, 16385])
@pytest.mark.parametrize("size", [1.0, 2.0 ** 100, 2.0 ** 115])
def test_quantised_norm_is_the_quantiser_of_the_norm(ops, C, size):
    """In FP32 the norm's y is what its quantised form quantises, huge rows included."""
    g = generator(C)
    x, r = (torch.randn(7, C, generator=g, device="cuda") for _ in range(2))
    w = (1 + 0.2 * torch.randn(C, generator=g, device="cuda")) * size
    y, _ = ops.block_norm(x, r, w, 1e-5)
    q, s, _ = ops.block_norm_quant_per_token(x, r, w, 1e-5)
    q1, s1 = ops.quant_per_token(y)
    assert torch.equal(q, q1) and torch.equal(s, s1)
    assert bool((s > size / 127).all())


@pytest.mark.parametrize("F", [1, 7, 65, 1025, 8191])
@pytest.mark.parametrize("x_type", [F16, BF16, F32])
@pytest.mark.parametrize("interleaved", [True, False])
def test_swiglu_rows_do_not_depend_on_what_lies_behind_them(ops, F, x_type, interleaved):
    """Rows of ordinary gates (down to -86.5) whose neighbours in memory begin and end with far ones: the
    same bits as each row alone."""
    g = generator(F)
    rows = 64
    gate = torch.rand(rows, F, generator=g, device="cuda") * -5.5 - 81
    up = (torch.rand(rows, F, generator=g, device="cuda") + 0.5) * (6e4 if x_type == F16 else 1e30)
    gate[1::2] = -1e4
    up[1::2] = -6e4
    gate, up = gate.to(dtype(x_type)), up.to(dtype(x_type))
    x = torch.stack([gate, up], dim=2).reshape(rows, 2 * F) if interleaved else torch.cat([gate, up], dim=1)
    q, s = ops.swiglu_quant_per_token(x.contiguous(), interleaved=interleaved)
    for r in range(0, rows, 2):
        q1, s1 = ops.swiglu_quant_per_token(x[r:r + 1].contiguous(), interleaved=interleaved)
        # (in FP16 some rows hold an infinity: NaN scales, compared by their bits)
        assert torch.equal(s1.view(torch.int32)[0], s.view(torch.int32)[r]) and torch.equal(q1[0], q[r])


@pytest.mark.parametrize("F", [64, 1024, 1025, 8191, 28672])
@pytest.mark.parametrize("x_type", [F16, BF16, F32])
@pytest.mark.parametrize("interleaved", [True, False])
def test_swiglu_far_gates_in_large_batches(ops, F, x_type, interleaved):
    """Batches whose rows are not all at work at once lay a row out differently (four groups per thread)."""
    gate, up = far_rows(F, x_type, F)
    x = torch.stack([gate, up], dim=2).reshape(8, 2 * F) if interleaved else torch.cat([gate, up], dim=1)
    q, s = ops.swiglu_quant_per_token(x.contiguous(), interleaved=interleaved)
    copies = 160
    qs, ss = ops.swiglu_quant_per_token(x.repeat(copies, 1), interleaved=interleaved)
    assert torch.equal(ss.view(copies, 8), s.expand(copies, 8))
    assert torch.equal(qs.view(copies, 8, F), q.expand(copies, 8, F))


# ------------------------------------------------------------------ rooms about 48 KiB
@pytest.mark.parametrize("C", range(24331, 24600, 42))
def test_staged_rows_about_48_kib(ops, C):
    """A block's staged rows and its own few words together may pass the 48 KiB that a kernel has without asking
    where the rows alone do not.  C: FP16 values whose granules are 192 bytes below that to a little above."""
    g = generator(C)
    x = torch.randn(3, C, generator=g, device="cuda")
    zero = torch.zeros((), dtype=torch.float64, device="cuda")
    for part, call in ((x[:, :C].half(), ops.quant_per_token), (x[:, :C // 2], ops.quant_per_token)):
        part = part[:, :part.shape[1] - (part.shape[1] % 8 == 0)].contiguous()
        q, s = call(part)
        check_quantised(q, s, part.double(), zero.expand(part.shape))
    for dt, width in ((torch.float16, C // 2), (torch.float32, C // 4)):
        F = width - (width % 8 == 0)
        gu = torch.randn(3, 2 * F, generator=g, device="cuda").to(dt)
        for interleaved in (True, False):
            gate, up = (gu[:, 0::2], gu[:, 1::2]) if interleaved else (gu[:, :F], gu[:, F:])
            gate, up = gate.double(), up.double()
            y = gate * torch.sigmoid(gate) * up
            q, s = ops.swiglu_quant_per_token(gu, interleaved=interleaved)
            check_quantised(q, s, y, y.abs() * (12 + 1.24 * gate.abs()) * U + 2.0 ** -114)
    for types, width in (((F16, F16, F16), C // 2), ((F16, F32, F32), C // 3), ((F32, F32, F32), C // 4)):
        c = width - (width % 8 == 0)
        x2, r, w, p, gt = norm_inputs(3, c, *types, "channel", C)
        y64, dy, z64, dz = norm_expected(x2, r, w, p, gt, 1e-5, 1.0)
        y, z = ops.block_norm(x2, r, w, 1e-5, post_weight=p, gate=gt)
        assert_within(z, z64, dz + half_step(z64, z.dtype) * 1.01)
        assert_within(y, y64, dy + half_step(y64, y.dtype) * 1.01)
        q, s, _ = ops.block_norm_quant_per_token(x2, r, w, 1e-5, post_weight=p, gate=gt)
        check_quantised(q, s, y64, dy)


def test_the_first_call_about_48_kib(ops):
    """The same in a process that has made no larger call before: a kernel keeps the room that it was once given."""
    script = """
import torch
from texo_b200 import ops
x = torch.randn(3, 24499, device="cuda")
h = x.half()
ops.quant_per_token(h), ops.quant_per_token(x[:, :12249].contiguous())
for gu in (h[:, :24498].contiguous(), x[:, :12246].contiguous()):
    for interleaved in (True, False):
        ops.swiglu_quant_per_token(gu, interleaved=interleaved)
for a, b in ((h[:, :12249], h[:, :12249]), (h[:, :8166], x[:, :8166]), (x[:, :6123], x[:, :6123])):
    a, b = a.contiguous(), b.contiguous()
    ops.block_norm(a, b, a[0].contiguous(), 1e-5), ops.block_norm_quant_per_token(a, b, a[0].contiguous(), 1e-5)
torch.cuda.synchronize()
print("ran")
"""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    run = subprocess.run([sys.executable, "-c", script], cwd=root, capture_output=True, text=True, timeout=300)
    assert run.returncode == 0 and "ran" in run.stdout, run.stderr


# ------------------------------------------------------------------ random sizes, strides and addresses
def spread(rng, lo, hi):
    """An integer of [lo, hi], spread over its logarithm."""
    return min(hi, max(lo, int(round(lo * (hi / lo) ** rng.random()))))


def placed(x, by):
    """A copy of x `by` elements into a larger buffer."""
    base = torch.zeros(x.numel() + by, dtype=x.dtype, device="cuda")
    base[by:] = x.reshape(-1)
    return base[by:].view(x.shape)


class Guarded:
    """An output inside a larger buffer, 0 to 8 elements off a 16-byte boundary."""

    def __init__(self, rng, rows, columns, t):
        self.count = rows * columns
        self.start = 32 + rng.choice([0, 0, 1, 3, 8])
        self.base = torch.full((self.start + self.count + 32,), 77, dtype=t, device="cuda")
        self.out = self.base[self.start:self.start + self.count].view(rows, columns)

    def check(self):
        assert bool((self.base[:self.start] == 77).all()) and bool((self.base[self.start + self.count:] == 77).all())


@pytest.mark.parametrize("seed", range(4))
def test_random_products(ops, seed):
    rng = random.Random(seed)
    for i in range(150):
        M, N, K = spread(rng, 1, 900), spread(rng, 1, 6000), spread(rng, 1, 6000)
        if rng.random() < 0.5:
            N, K = (N + 15) // 16 * 16, (K + 15) // 16 * 16
        A, B, sa, sb, bias = mm_inputs(M, N, K, 1000 * seed + i, full_range=True)
        A, B = (placed(v, rng.randrange(16)) if rng.random() < 0.3 else v for v in (A, B))
        t = dtype(rng.choice([BF16, F32]))
        bias = bias if rng.random() < 0.5 else None
        guarded = Guarded(rng, M, N, t)
        ops.mm_int8_per_token(A, B, sa, sb, bias, out_dtype=t, out=guarded.out)
        want, bound = mm_expected(A, B, sa, sb, bias, t)
        assert_within(guarded.out, want, bound)
        guarded.check()
    assert ops.status() == 0


@pytest.mark.parametrize("seed", range(4))
def test_random_producers(ops, seed):
    rng = random.Random(100 + seed)
    for i in range(150):
        C = spread(rng, 1, 30000)
        N = spread(rng, 1, max(1, min(3000, 4000000 // C)))
        if rng.random() < 0.5:
            C = (C + 7) // 8 * 8
        x_type = rng.choice([F16, BF16, F32])
        g = generator(1000 * seed + i)
        kind = rng.choice(["plain", "pairs", "halves", "norm"])
        guarded = Guarded(rng, N, C, torch.int8)
        if kind == "norm":
            types = (x_type, rng.choice([x_type, F32]), rng.choice([x_type, F32]))
            x, r, w, p, gt = norm_inputs(N, C, *types, rng.choice(["none", "channel", "scalar", "rows", "tokens"]), i)
            p = p if rng.random() < 0.5 else None
            x, r = (placed(v, rng.randrange(8)) if rng.random() < 0.3 else v for v in (x, r))
            y64, dy, z64, dz = norm_expected(x, r, w, p, gt, 1e-5, 0.75)
            y, z = ops.block_norm(x, r, w, 1e-5, post_weight=p, gate=gt, residual_scale=0.75)
            assert_within(z, z64, dz + half_step(z64, z.dtype) * 1.01)
            assert_within(y, y64, dy + half_step(y64, y.dtype) * 1.01)
            q, s, z2 = ops.block_norm_quant_per_token(x, r, w, 1e-5, post_weight=p, gate=gt, residual_scale=0.75,
                                                      out=guarded.out)
            assert torch.equal(z, z2)
            check_quantised(q, s, y64, dy)
        else:
            width, extra = (C if kind == "plain" else 2 * C), rng.choice([0, 0, 1, 5, 8])
            wide = (torch.randn(N, width + extra, generator=g, device="cuda") * rng.choice([0.01, 3, 30])).to(dtype(x_type))
            x = wide[:, :width] if rng.random() < 0.5 else wide[:, extra:]
            if kind == "plain":
                q, s = ops.quant_per_token(x, out=guarded.out)
                check_quantised(q, s, x.double(), torch.zeros_like(x, dtype=torch.float64))
            else:
                q, s = ops.swiglu_quant_per_token(x, interleaved=kind == "pairs", out=guarded.out)
                gate, up = (x[:, 0::2], x[:, 1::2]) if kind == "pairs" else (x[:, :C], x[:, C:])
                gate, up = gate.double(), up.double()
                y = gate / (1 + torch.exp(-gate)) * up
                check_quantised(q, s, y, y.abs() * (1.24 * gate.abs().clamp_max(90) + 12) * U + 2.0 ** -114)
        guarded.check()
