"""GPU tests of the dynamic-quantisation operators (mm_int8_per_token, block_norm and the
per-token quantisers) against plain implementations in 64 bits.

Tolerances count roundings.  A rounding to a type of machine epsilon e is off by at most e / 2
relative to the value: U = 2^-24 for FP32, and `half_step` for the output's type (plus half of
its smallest subnormal).  The bounds are computed next to the values, in 64 bits.
"""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

U = 2.0 ** -24
F16, BF16, F32 = "float16", "bfloat16", "float32"


@pytest.fixture(scope="module")
def ops():
    if not torch.cuda.is_available():
        pytest.fail("no CUDA device: GPU tests need a B200")
    from texo_b200 import ops

    return ops


def dtype(name):
    return getattr(torch, name)


def half_step(want, t):
    """Largest error of rounding `want` (float64) to type t."""
    smallest = {torch.float16: 2.0 ** -24, torch.bfloat16: 2.0 ** -133, torch.float32: 2.0 ** -149}[t]
    return torch.finfo(t).eps / 2 * want.abs() + smallest / 2


def assert_within(got, want, bound):
    bad = ~((got.double() - want).abs() <= bound)
    assert not bool(bad.any()), (
        f"{int(bad.sum())} of {bad.numel()} values outside; first at {bad.nonzero()[0].tolist()}: "
        f"got {got.double()[bad][0].item()!r}, want {want[bad][0].item()!r} +- {bound[bad][0].item()!r}")


def generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


# ------------------------------------------------------------------ the product
def mm_inputs(M, N, K, seed, full_range=False):
    g = generator(seed)
    A = torch.randint(-128 if full_range else -127, 128, (M, K), generator=g, device="cuda", dtype=torch.int8)
    B = torch.randint(-128 if full_range else -127, 128, (K, N), generator=g, device="cuda", dtype=torch.int8)
    sa = torch.rand(M, generator=g, device="cuda") * 0.01 + 1e-4
    sb = torch.rand(N, generator=g, device="cuda") * 0.01 + 1e-4
    bias = torch.randn(N, generator=g, device="cuda")
    return A, B, sa, sb, bias


def mm_expected(A, B, sa, sb, bias, t):
    # int8 products are exact in 64-bit floating point, and so are their sums (K < 2^39)
    dot = A.double() @ B.double()
    scaled = dot * sa.double()[:, None] * sb.double()
    want = scaled if bias is None else scaled + bias.double()
    # the dot's rounding, its product with scale_A, the fused second product and sum; U^2 terms
    # are below a hundredth of U
    bound = 2.01 * U * scaled.abs() + 1.01 * U * want.abs()
    return want, bound + half_step(want, t) * (1 + 4 * U)


MM_SHAPES = [
    (1, 1, 1), (1, 16, 16), (1, 1024, 1024), (2, 272, 48), (5, 256, 4096), (16, 512, 1024), (17, 528, 8192),
    (31, 2048, 256), (32, 768, 2080), (33, 256, 512), (64, 512, 16), (65, 1040, 384), (100, 8192, 128),
    (127, 256, 28672), (128, 512, 1024), (129, 512, 1024), (200, 272, 4096), (256, 256, 128), (257, 1296, 144),
    (300, 4096, 2048), (512, 512, 1024), (1000, 2064, 656), (2048, 2560, 512),
]
MM_ODD = [
    (1, 3, 5), (1, 1023, 1025), (3, 17, 31), (7, 257, 129), (16, 1001, 999), (33, 255, 128), (64, 512, 100),
    (65, 67, 31), (128, 130, 1024), (130, 1000, 1000), (333, 499, 501), (300, 4104, 1999), (1030, 2050, 257),
]


@pytest.mark.parametrize("shape", MM_SHAPES + MM_ODD)
@pytest.mark.parametrize("out_type,with_bias", [(F16, False), (BF16, True), (F32, True)])
def test_mm_matches_64_bits(ops, shape, out_type, with_bias):
    M, N, K = shape
    t = dtype(out_type)
    A, B, sa, sb, bias = mm_inputs(M, N, K, M * 7 + N * 3 + K)
    if t == torch.float16:
        sa *= 0.1  # keeps the largest sums in range
    want, bound = mm_expected(A, B, sa, sb, bias if with_bias else None, t)
    out = torch.full((M, N), 99.0, dtype=t, device="cuda")
    got = ops.mm_int8_per_token(A, B, sa, sb, bias if with_bias else None, out_dtype=t, out=out)
    assert got is out
    assert_within(got, want, bound)
    assert ops.status() == 0


@pytest.mark.parametrize("path", [1, 2, 3, 4])
@pytest.mark.parametrize("shape", [(1, 16, 16), (1, 17, 15), (15, 300, 1300), (40, 528, 400), (65, 67, 31),
                                   (129, 511, 1025), (256, 512, 1024), (300, 1001, 640), (600, 272, 2047),
                                   (513, 2000, 129)])
@pytest.mark.parametrize("out_type", [F16, BF16, F32])
def test_mm_paths_agree(ops, path, shape, out_type):
    """Each path (SIMT, streaming, gathering, CTA pairs) on shapes that the choice would not send it."""
    from texo_b200 import _lib

    M, N, K = shape
    t = dtype(out_type)
    A, B, sa, sb, bias = mm_inputs(M, N, K, sum(shape), full_range=True)
    if t == torch.float16:
        sa *= 0.1
    ops.mm_int8_per_token(A[:1], B, sa[:1], sb)  # the device's set-up
    lib = _lib.load()
    lib.texo_mm_int8_per_token_force_path(path)
    try:
        got = ops.mm_int8_per_token(A, B, sa, sb, bias, out_dtype=t)
        assert lib.texo_mm_int8_per_token_last_path() == path
    finally:
        lib.texo_mm_int8_per_token_force_path(0)
    want, bound = mm_expected(A, B, sa, sb, bias, t)
    assert_within(got, want, bound)
    assert torch.equal(got, ops.mm_int8_per_token(A, B, sa, sb, bias, out_dtype=t))
    assert ops.status() == 0


def test_mm_with_less_workspace_than_it_asks_for(ops):
    """Without the workspace for padded copies the call gathers, and gives the same bits."""
    from texo_b200 import _lib

    M, N, K = 300, 1001, 2047
    A, B, sa, sb, bias = mm_inputs(M, N, K, 11)
    want = ops.mm_int8_per_token(A, B, sa, sb, bias, out_dtype=torch.float32)
    lib = _lib.load()
    lib.texo_mm_int8_per_token_force_path(2)  # streaming, which needs the copies here
    try:
        asked = lib.texo_mm_int8_per_token_workspace(A.data_ptr(), B.data_ptr(), M, N, K)
        assert asked == M * 2048 + K * 1008
        space = torch.full((asked + 16,), 3, dtype=torch.uint8, device="cuda")
        stream = torch.cuda.current_stream().cuda_stream
        for pointer, size, path in ((None, 0, 3), (space.data_ptr(), asked - 1, 3), (space.data_ptr() + 1, asked, 3),
                                    (None, asked, 3), (space.data_ptr(), asked, 2)):
            got = torch.zeros_like(want)
            assert lib.texo_mm_int8_solve_per_token(A.data_ptr(), B.data_ptr(), got.data_ptr(), M, N, K, sa.data_ptr(),
                                                    sb.data_ptr(), bias.data_ptr(), 2, pointer, size, stream) == 0
            assert torch.equal(got, want)
            assert lib.texo_mm_int8_per_token_last_path() == path
            assert path == 2 or bool((space == 3).all())
    finally:
        lib.texo_mm_int8_per_token_force_path(0)
    assert bool((space[asked:] == 3).all())


@pytest.mark.parametrize("shape", [(20, 256, 8192), (160, 512, 30000), (3, 100, 4099)])
def test_mm_extreme_values(ops, shape):
    """All -128 against all -128: the largest dots there are (2^14 K), and their rounding to FP32."""
    M, N, K = shape
    A = torch.full((M, K), -128, dtype=torch.int8, device="cuda")
    B = torch.full((K, N), -128, dtype=torch.int8, device="cuda")
    B[0] = 127  # an odd dot, which FP32 cannot hold
    B[1] = 127
    A[:, 0] = 1
    one_m, one_n = torch.ones(M, device="cuda"), torch.ones(N, device="cuda")
    got = ops.mm_int8_per_token(A, B, one_m, one_n, out_dtype=torch.float32)
    dot = 16384 * (K - 2) + 127 - 128 * 127
    assert bool((got.double() == float(np.float32(dot))).all())


@pytest.mark.parametrize("K", [131071, 131072, 140000])
def test_mm_long_sums_do_not_wrap(ops, K):
    """At K = 2^17 an int32 sum of -128 * -128 wraps."""
    M, N = 3, 32
    A = torch.full((M, K), -128, dtype=torch.int8, device="cuda")
    B = torch.full((K, N), -128, dtype=torch.int8, device="cuda")
    one_m, one_n = torch.ones(M, device="cuda"), torch.ones(N, device="cuda")
    got = ops.mm_int8_per_token(A, B, one_m, one_n, out_dtype=torch.float32)
    assert bool((got.double() == float(np.float32(16384 * K))).all())


def test_mm_without_k_and_without_rows(ops):
    M, N = 5, 33
    sa, sb = torch.ones(M, device="cuda"), torch.ones(N, device="cuda")
    bias = torch.arange(N, device="cuda", dtype=torch.float32)
    A = torch.empty((M, 0), dtype=torch.int8, device="cuda")
    B = torch.empty((0, N), dtype=torch.int8, device="cuda")
    got = ops.mm_int8_per_token(A, B, sa, sb, bias, out_dtype=torch.float32)
    assert torch.equal(got, bias.expand(M, N))
    assert not bool(ops.mm_int8_per_token(A, B, sa, sb).any())
    none = ops.mm_int8_per_token(A[:0], B, sa[:0], sb)
    assert none.shape == (0, N) and none.dtype == torch.float16


@pytest.mark.parametrize("shape,offset", [((8, 256, 256), 1), ((40, 512, 1024), 3), ((200, 512, 512), 7),
                                          ((300, 272, 144), 8)])
def test_mm_at_odd_addresses(ops, shape, offset):
    M, N, K = shape
    A, B, sa, sb, bias = mm_inputs(M, N, K, 5)

    def moved(x, by):
        base = torch.zeros(x.numel() + by, dtype=x.dtype, device="cuda")
        base[by:] = x.reshape(-1)
        return base[by:].view(x.shape)

    want, bound = mm_expected(A, B, sa, sb, bias, torch.bfloat16)
    A, B = moved(A, offset), moved(B, offset + 2)
    sa, sb, bias = moved(sa, 1), moved(sb, 1), moved(bias, 3)
    out = moved(torch.zeros((M, N), dtype=torch.bfloat16, device="cuda"), 1)
    got = ops.mm_int8_per_token(A, B, sa, sb, bias, out_dtype=torch.bfloat16, out=out)
    assert got.data_ptr() == out.data_ptr()
    assert_within(got, want, bound)


@pytest.mark.parametrize("shape", [(3, 256, 512), (40, 512, 1024), (200, 512, 2048), (70, 333, 777)])
def test_mm_writes_its_output_alone(ops, shape):
    M, N, K = shape
    A, B, sa, sb, _ = mm_inputs(M, N, K, 9)
    base = torch.full((M * N + 256,), 7.0, dtype=torch.float16, device="cuda")
    out = base[128:128 + M * N].view(M, N)
    ops.mm_int8_per_token(A, B, sa * 0.1, sb, out=out)
    assert bool((base[:128] == 7).all()) and bool((base[128 + M * N:] == 7).all())
    assert bool((out != 7).any(dim=1).all())


def test_mm_carries_nan_scales_through_their_rows(ops):
    M, N, K = 40, 512, 1024
    A, B, sa, sb, bias = mm_inputs(M, N, K, 2)
    sa[7] = float("nan")
    got = ops.mm_int8_per_token(A, B, sa, sb, bias, out_dtype=torch.bfloat16)
    assert bool(got[7].isnan().all()) and not bool(got[:7].isnan().any()) and not bool(got[8:].isnan().any())


def test_mm_rows_do_not_depend_on_the_batch(ops):
    """Every path computes the same formula on the same integer dot."""
    N, K = 1024, 2048
    A, B, sa, sb, bias = mm_inputs(700, N, K, 3)
    whole = ops.mm_int8_per_token(A, B, sa, sb, bias, out_dtype=torch.float32)
    for m in (1, 16, 33, 100, 260):
        part = ops.mm_int8_per_token(A[:m].contiguous(), B, sa[:m].contiguous(), sb, bias, out_dtype=torch.float32)
        assert torch.equal(part, whole[:m])


def test_mm_offsets_past_32_bits(ops):
    """An output of more than 2^31 elements (its bytes pass 2^32 as well)."""
    M, N, K = 70000, 32768, 16
    A, B, sa, sb, _ = mm_inputs(M, N, K, 4)
    got = ops.mm_int8_per_token(A, B, sa, sb, out_dtype=torch.float16)
    rows = torch.tensor([0, 1, 65535, 65536, 69998, 69999], device="cuda")
    want, bound = mm_expected(A[rows], B, sa[rows], sb, None, torch.float16)
    assert_within(got[rows], want, bound)


# ------------------------------------------------------------------ block norm
def norm_inputs(N, C, x_type, res_type, w_type, gate, seed):
    g = generator(seed)
    x = (torch.randn(N, C, generator=g, device="cuda") * 1.5).to(dtype(x_type))
    r = (torch.randn(N, C, generator=g, device="cuda") * 3).to(dtype(res_type))
    w = (1 + 0.3 * torch.randn(C, generator=g, device="cuda")).to(dtype(w_type))
    p = (1 + 0.3 * torch.randn(C, generator=g, device="cuda")).to(dtype(w_type))
    gates = {"none": None, "channel": (C,), "rows": (N, C), "scalar": (1, 1), "tokens": (N, 1), "half": (2, C)}
    shape = gates[gate]
    gt = None if shape is None else (0.6 * torch.randn(*shape, generator=g, device="cuda")).to(dtype(w_type))
    return x, r, w, p, gt


def rms64(v, w, eps):
    """RMSNorm in 64 bits and a bound on its error in FP32 relative to its value: a square and at
    most 32 additions per thread (or C / 1024 for rows in several passes), ten more across the
    row, the division and eps, halved by the root; rsqrtf's two ulps (4 U); two products."""
    C = v.shape[1]
    inv = 1 / torch.sqrt((v * v).mean(dim=1, keepdim=True) + eps)
    relative = ((max(32, C / 1024) + 14) / 2 + 4 + 2) * U
    return v * inv * w.double(), inv, relative


def norm_expected(x, r, w, p, gate, eps, scale):
    """y and z in 64 bits, with bounds of their errors in FP32."""
    N, C = x.shape
    u = x.double()
    du = torch.zeros_like(u)
    if p is not None:
        u, _, rel = rms64(u, p, eps)
        du = u.abs() * rel
    if gate is not None:
        gd = gate.double()
        if gd.dim() == 1:
            gd = gd[None]
        gd = gd.repeat_interleave(N // gd.shape[0], dim=0)
        u = u * gd
        du = du * gd.abs() + u.abs() * U
    z = u + scale * r.double()
    dz = du + U * z.abs()
    y, inv, rel = rms64(z, w, eps)
    # the error of z's own norm shifts all of its row
    shift = dz.norm(dim=1, keepdim=True) / z.norm(dim=1, keepdim=True).clamp_min(1e-300)
    dy = w.double().abs() * inv * dz + y.abs() * (shift + rel)
    return y, dy * 1.01, z, dz * 1.01


NORM_SHAPES = [(1, 1), (1, 8192), (2, 7), (4, 64), (3, 1000), (6, 1001), (600, 96), (514, 264), (700, 512),
               (512, 1024), (600, 1025), (34, 4096), (520, 4999), (513, 16383), (2, 16384), (514, 16384), (4, 16385),
               (2, 20002)]
NORM_TYPES = [(F16, F16, F16), (BF16, F32, BF16), (BF16, BF16, F32), (F32, F32, F32), (F16, F32, F32)]


@pytest.mark.parametrize("shape", NORM_SHAPES)
@pytest.mark.parametrize("types", NORM_TYPES)
@pytest.mark.parametrize("post,gate", [(False, "none"), (True, "channel"), (True, "rows"), (False, "scalar"),
                                       (True, "tokens")])
def test_block_norm_matches_64_bits(ops, shape, types, post, gate):
    N, C = shape
    x, r, w, p, gt = norm_inputs(N, C, *types, gate, N + C)
    p = p if post else None
    y64, dy, z64, dz = norm_expected(x, r, w, p, gt, 1e-5, 0.875)
    y, z = ops.block_norm(x, r, w, 1e-5, post_weight=p, gate=gt, residual_scale=0.875)
    assert y.dtype == x.dtype and z.dtype == r.dtype
    assert_within(z, z64, dz + half_step(z64, z.dtype) * 1.01)
    assert_within(y, y64, dy + half_step(y64, y.dtype) * 1.01)
    q, s, z2 = ops.block_norm_quant_per_token(x, r, w, 1e-5, post_weight=p, gate=gt, residual_scale=0.875)
    assert torch.equal(z2, z)
    check_quantised(q, s, y64, dy)


def check_quantised(q, s, y, dy):
    """scale: the row maximum's error, one division.  q: rint of y / scale, where y, the maximum
    (their errors dy) and two roundings (scale's, the quotient's) move the argument; an argument
    next to a tie may round either way."""
    assert q.dtype == torch.int8 and s.dtype == torch.float32
    amax = y.abs().amax(dim=1)
    damax = dy.amax(dim=1)
    top = amax.clamp_min(2.0 ** -100)
    assert_within(s, top / 127, (damax + 1.01 * U * top) / 127)
    t = y * (127 / top)[:, None]
    dt = 127 / top[:, None] * (dy + y.abs() * (damax / top)[:, None]) * 1.01 + 2.01 * U * t.abs()
    assert_within(q, t, 0.5 + dt)
    assert int(q.min()) >= -127


def test_block_norm_gate_rows_serve_consecutive_tokens(ops):
    x, r, w, p, gt = norm_inputs(6, 256, BF16, BF16, BF16, "half", 1)
    y, z = ops.block_norm(x, r, w, 1e-6, gate=gt)
    for row in (0, 1):
        part = slice(3 * row, 3 * row + 3)
        y1, z1 = ops.block_norm(x[part].contiguous(), r[part].contiguous(), w, 1e-6, gate=gt[row])
        assert torch.equal(y1, y[part]) and torch.equal(z1, z[part])


@pytest.mark.parametrize("shape", [(5, 1024), (5, 1001), (3, 16500)])
def test_block_norm_in_place(ops, shape):
    x, r, w, p, gt = norm_inputs(*shape, F16, F16, F16, "channel", 2)
    y, z = ops.block_norm(x, r, w, 1e-5, post_weight=p, gate=gt)
    q, s, _ = ops.block_norm_quant_per_token(x, r, w, 1e-5, post_weight=p, gate=gt)
    r2 = r.clone()
    q2, s2, z2 = ops.block_norm_quant_per_token(x, r2, w, 1e-5, post_weight=p, gate=gt, z_out=r2)
    assert z2 is r2 and torch.equal(r2, z) and torch.equal(q2, q) and torch.equal(s2, s)
    x3, r3 = x.clone(), r.clone()
    y3, z3 = ops.block_norm(x3, r3, w, 1e-5, post_weight=p, gate=gt, out=x3, z_out=r3)
    assert y3 is x3 and torch.equal(x3, y) and torch.equal(r3, z)


def test_block_norm_at_odd_addresses(ops):
    x, r, w, p, gt = norm_inputs(9, 512, BF16, BF16, BF16, "channel", 3)

    def moved(t):
        base = torch.zeros(t.numel() + 1, dtype=t.dtype, device="cuda")
        base[1:] = t.reshape(-1)
        return base[1:].view(t.shape)

    y64, dy, z64, dz = norm_expected(x, r, w, p, gt, 1e-5, 1.0)
    y, z = ops.block_norm(*map(moved, (x, r, w)), 1e-5, post_weight=moved(p), gate=moved(gt))
    assert_within(z, z64, dz + half_step(z64, z.dtype) * 1.01)
    assert_within(y, y64, dy + half_step(y64, y.dtype) * 1.01)


@pytest.mark.parametrize("C", [512, 513, 17000])
def test_block_norm_rows_that_are_not_finite(ops, C):
    x, r, w, _, _ = norm_inputs(6, C, BF16, BF16, BF16, "none", 4)
    x[1, C // 2] = float("nan")
    r[3, C - 1] = float("inf")
    x[4] = 0
    r[4] = 0
    q, s, z = ops.block_norm_quant_per_token(x, r, w, 1e-5)
    assert s.isnan().tolist() == [False, True, False, True, False, False]
    assert not bool(q[1].any()) and not bool(q[3].any()) and not bool(q[4].any())
    assert s[4].item() == np.float32(np.float32(2.0 ** -100) / np.float32(127))
    assert bool(z[1].isnan().any()) and bool(z[3].isinf().any())
    clean = [0, 2, 5]
    q1, s1, z1 = ops.block_norm_quant_per_token(x[clean], r[clean], w, 1e-5)
    assert torch.equal(q1, q[clean]) and torch.equal(s1, s[clean]) and torch.equal(z1, z[clean])
    y, _ = ops.block_norm(x, r, w, 1e-5)
    assert bool(y[1].isnan().all()) and bool(y[3].isnan().any()) and not bool(y[4].any())


# ------------------------------------------------------------------ quantisers
QUANT_SHAPES = [(1, 1), (1, 5), (16, 8192), (3, 64), (700, 100), (520, 128), (600, 1024), (515, 4999), (33, 16384),
                (513, 16384), (2, 16385), (600, 20001), (3, 28672), (520, 28672), (2, 40001), (515, 65536), (2, 140000)]


@pytest.mark.parametrize("shape", QUANT_SHAPES)
@pytest.mark.parametrize("x_type", [F16, BF16, F32])
def test_quant_matches_64_bits(ops, shape, x_type):
    g = generator(shape[0] + shape[1])
    x = (torch.randn(*shape, generator=g, device="cuda") * 3).to(dtype(x_type))
    q, s = ops.quant_per_token(x)
    check_quantised(q, s, x.double(), torch.zeros_like(x, dtype=torch.float64))


@pytest.mark.parametrize("shape", [(64, 512), (3, 8192), (515, 1001), (2, 140000)])
@pytest.mark.parametrize("x_type", [F16, BF16])
def test_quant_of_ties(ops, shape, x_type):
    """Values of few bits lie half way between two multiples of the scale often: the quotient in FP32
    decides, ties to even, as elementary operations do it."""
    g = generator(9)
    x = torch.randint(-254, 255, shape, generator=g, device="cuda").to(dtype(x_type))
    x[:, 0] = 254
    x[0] *= 0.37
    q, s = ops.quant_per_token(x)
    want = x.float().abs().amax(dim=1) / 127
    assert torch.equal(s, want)
    t = x.float() / want[:, None]
    assert torch.equal(q.float(), torch.round(t))
    assert bool(((t[1:] % 1).abs() == 0.5).any())


@pytest.mark.parametrize("shape", QUANT_SHAPES)
@pytest.mark.parametrize("x_type,interleaved", [(F16, True), (F16, False), (BF16, True), (F32, False), (F32, True)])
def test_swiglu_quant_matches_64_bits(ops, shape, x_type, interleaved):
    N, F = shape
    g = generator(N + F + 1)
    gu = (torch.randn(N, 2 * F, generator=g, device="cuda") * 3).to(dtype(x_type))
    gate, up = (gu[:, 0::2], gu[:, 1::2]) if interleaved else (gu[:, :F], gu[:, F:])
    gate, up = gate.double(), up.double()
    y = gate * torch.sigmoid(gate) * up
    # (in U) e^-gate = 2^(-gate log2 e): the exponent's rounding and its constant's 1.23 |gate|, the power
    # two ulps = 4; the sum 1, the reciprocal one ulp = 2, the products 1 each
    dy = y.abs() * (2 * (2 + 1.16 * gate.abs()) + 1 + 4 + 1) * U + 2.0 ** -126
    q, s = ops.swiglu_quant_per_token(gu, interleaved=interleaved)
    check_quantised(q, s, y, dy)


def test_quantisers_take_slices_of_wider_rows(ops):
    g = generator(6)
    wide = torch.randn(40, 3 * 512 + 8, generator=g, device="cuda").to(torch.float16)
    for lo, hi in ((0, 512), (512, 1024), (520, 1033), (3, 514)):
        q, s = ops.quant_per_token(wide[:, lo:hi])
        q1, s1 = ops.quant_per_token(wide[:, lo:hi].contiguous())
        assert torch.equal(q, q1) and torch.equal(s, s1)
    for inter in (True, False):
        q, s = ops.swiglu_quant_per_token(wide[:, 8:1032], interleaved=inter)
        q1, s1 = ops.swiglu_quant_per_token(wide[:, 8:1032].contiguous(), interleaved=inter)
        assert torch.equal(q, q1) and torch.equal(s, s1)


@pytest.mark.parametrize("C", [64, 65, 8192, 20000])
def test_quant_of_unusual_rows(ops, C):
    x = torch.ones(8, C, device="cuda")
    x[0] = 0
    x[1, 0] = float("nan")
    x[2, C - 1] = float("-inf")
    x[3] = 1e-40  # subnormal
    x[4] = torch.finfo(torch.float32).max
    x[5] = -x[4]
    x[6] = 2.0 ** -100
    q, s = ops.quant_per_token(x)
    assert s.isnan().tolist() == [False, True, True, False, False, False, False, False]
    for row, value in ((0, 0), (1, 0), (2, 0), (3, 0), (4, 127), (5, -127), (6, 127), (7, 127)):
        assert bool((q[row] == value).all()), row
    assert s[0].item() == s[3].item() == s[6].item()
    assert_within(s[4:8], x[4:8, 0].double().abs() / 127, x[4:8, 0].double().abs() / 127 * 1.01 * U)


@pytest.mark.parametrize("shape", [(5, 100), (3, 5001), (520, 333), (513, 4096)])
@pytest.mark.parametrize("shift", [0, 1, 3])
def test_producers_write_their_outputs_alone(ops, shape, shift):
    """Outputs inside wider buffers, at addresses aligned to no more than an element: the same values, and
    nothing around them touched."""
    N, C = shape
    x, r, w, p, gt = norm_inputs(N, C, F16, F32, F16, "channel", 5)

    def room(dt):
        base = torch.full((N * C + 128,), 77, dtype=dt, device="cuda")
        return base, base[64 + shift:64 + shift + N * C].view(N, C)

    def untouched(base):
        return bool((base[:64 + shift] == 77).all()) and bool((base[64 + shift + N * C:] == 77).all())

    for call, dt in ((ops.block_norm, torch.float16), (ops.block_norm_quant_per_token, torch.int8)):
        want = call(x, r, w, 1e-5, post_weight=p, gate=gt)
        out_base, out = room(dt)
        z_base, z = room(torch.float32)
        got = call(x, r, w, 1e-5, post_weight=p, gate=gt, out=out, z_out=z)
        assert untouched(out_base) and untouched(z_base)
        if shift == 0:  # (another path may sum in another order)
            assert all(torch.equal(a, b) for a, b in zip(want, got))
        y64, dy, z64, dz = norm_expected(x, r, w, p, gt, 1e-5, 1.0)
        assert_within(z, z64, dz + half_step(z64, torch.float32) * 1.01)
        if dt == torch.int8:
            check_quantised(got[0], got[1], y64, dy)
        else:
            assert_within(out, y64, dy + half_step(y64, torch.float16) * 1.01)
    base, out = room(torch.int8)
    q, s = ops.quant_per_token(x, out=out)
    want = ops.quant_per_token(x)
    assert untouched(base) and torch.equal(q, want[0]) and torch.equal(s, want[1])
    if C % 2 == 0:
        base = torch.full((N * (C // 2) + 128,), 77, dtype=torch.int8, device="cuda")
        out = base[64 + shift:64 + shift + N * (C // 2)].view(N, C // 2)
        for inter in (True, False):
            q, s = ops.swiglu_quant_per_token(x, interleaved=inter, out=out)
            want = ops.swiglu_quant_per_token(x, interleaved=inter)
            assert torch.equal(q, want[0]) and torch.equal(s, want[1])
            assert bool((base[:64 + shift] == 77).all()) and bool((base[64 + shift + N * (C // 2):] == 77).all())


@pytest.mark.parametrize("C", [8192, 8191])
def test_producers_past_32_bit_offsets(ops, C):
    """Rows whose elements lie beyond the 2^31st."""
    N = 270000
    x = torch.empty((N, C), dtype=torch.bfloat16, device="cuda").uniform_(-2, 2, generator=generator(1))
    rows = torch.tensor([0, 1, 131072, 262143, 262144, N - 2, N - 1], device="cuda")
    w = torch.ones(C, device="cuda", dtype=torch.bfloat16)

    def check(q, s, z):
        part = x[rows]
        q1, s1, z1 = ops.block_norm_quant_per_token(part, part, w, 1e-5)
        y64, dy, z64, dz = norm_expected(part, part, w, None, None, 1e-5, 1.0)
        check_quantised(q, s, y64, dy)
        assert_within(z, z64, dz + half_step(z64, torch.bfloat16) * 1.01)
        assert torch.equal(z, z1)

    q, s = ops.quant_per_token(x)
    assert N * C > 2 ** 31
    check_quantised(q[rows], s[rows], x[rows].double(), torch.zeros((len(rows), C), dtype=torch.float64, device="cuda"))
    q, s, z = ops.block_norm_quant_per_token(x, x, w, 1e-5)
    check(q[rows], s[rows], z[rows])


def test_swiglu_of_far_gates(ops):
    gate = torch.tensor([-1e4, -200.0, -100.0, -88.0, -87.0, 88.0, 200.0, 1e4], device="cuda")
    up = torch.full_like(gate, 2.0)
    q, s = ops.swiglu_quant_per_token(torch.cat([gate, up])[None].contiguous(), interleaved=False)
    want = torch.round(torch.relu(gate) * 2 / s[0])
    assert torch.equal(q[0].float(), want) and not bool(s.isnan().any())


# ------------------------------------------------------------------ together, streams, graphs
def mlp(ops, x, residual, weights):
    """A block's second half as a user runs it: norm and quantise, gate/up, SwiGLU and quantise,
    down, and the next block's norm."""
    a, sa, z = ops.block_norm_quant_per_token(x, residual, weights["norm"], 1e-5, post_weight=weights["post"])
    gu = ops.mm_int8_per_token(a, weights["gu"], sa, weights["gu_scale"], out_dtype=torch.bfloat16)
    h, sh = ops.swiglu_quant_per_token(gu)
    d = ops.mm_int8_per_token(h, weights["down"], sh, weights["down_scale"], out_dtype=torch.bfloat16)
    return (*ops.block_norm(d, z, weights["norm2"], 1e-5, gate=weights["gate"]), a, sa, gu, h, sh, d)


def mlp_setup(n, c, f, seed=8):
    g = generator(seed)

    def quantised(k, cols):
        w = torch.randn(k, cols, generator=g, device="cuda") / k ** 0.5
        s = w.abs().amax(dim=0) / 127
        return torch.round(w / s).to(torch.int8).contiguous(), s

    weights = {k: (1 + 0.1 * torch.randn(c, generator=g, device="cuda")).bfloat16() for k in ("norm", "post", "norm2")}
    weights["gate"] = (0.5 * torch.randn(c, generator=g, device="cuda")).bfloat16()
    weights["gu"], weights["gu_scale"] = quantised(c, 2 * f)
    weights["down"], weights["down_scale"] = quantised(f, c)
    x = torch.randn(n, c, generator=g, device="cuda").bfloat16()
    return x, torch.randn(n, c, generator=g, device="cuda"), weights


@pytest.mark.parametrize("n,c,f", [(1, 512, 1024), (16, 512, 1024), (70, 500, 333), (300, 1024, 2048)])
def test_a_block_of_them(ops, n, c, f):
    """Each call against its 64-bit definition on the values that the call before it gave."""
    x, residual, w = mlp_setup(n, c, f)
    y, z2, a, sa, gu, h, sh, d = mlp(ops, x, residual, w)
    y64, dy, z64, dz = norm_expected(x, residual, w["norm"], w["post"], None, 1e-5, 1.0)
    check_quantised(a, sa, y64, dy)
    want, bound = mm_expected(a, w["gu"], sa, w["gu_scale"], None, torch.bfloat16)
    assert_within(gu, want, bound)
    gate, up = gu[:, 0::2].double(), gu[:, 1::2].double()
    act = gate * torch.sigmoid(gate) * up
    check_quantised(h, sh, act, act.abs() * (2 * (2 + 1.16 * gate.abs()) + 6) * U + 2.0 ** -126)
    want, bound = mm_expected(h, w["down"], sh, w["down_scale"], None, torch.bfloat16)
    assert_within(d, want, bound)
    _, z = ops.block_norm(x, residual, w["norm"], 1e-5, post_weight=w["post"])
    y64, dy, z64, dz = norm_expected(d, z, w["norm2"], None, w["gate"], 1e-5, 1.0)
    assert_within(z2, z64, dz + half_step(z64, torch.float32) * 1.01)
    assert_within(y, y64, dy + half_step(y64, torch.bfloat16) * 1.01)
    # the whole block without quantisation: 8-bit steps and BF16 roundings, about one part in a
    # hundred each in a two-norm; a wrong scale or layout is off by its whole value
    def rms(v, wt):
        return v * torch.rsqrt((v * v).mean(1, keepdim=True) + 1e-5) * wt.double()

    r = residual.double() + rms(x.double(), w["post"])
    gu64 = rms(r, w["norm"]) @ (w["gu"].double() * w["gu_scale"].double())
    act = gu64[:, 0::2] * torch.sigmoid(gu64[:, 0::2]) * gu64[:, 1::2]
    z64 = r + act @ (w["down"].double() * w["down_scale"].double()) * w["gate"].double()
    assert (z2.double() - z64).norm() < 0.05 * (z64 - r).norm()


def test_two_streams_at_once(ops):
    cases = [mlp_setup(n, 512, 1024, seed) for n, seed in ((16, 1), (300, 2), (1, 3))]
    alone = [[t.clone() for t in mlp(ops, *case)] for case in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    results = [[] for _ in cases]
    for _ in range(20):
        for case, stream, kept in zip(cases, streams, results):
            with torch.cuda.stream(stream):
                kept.append(mlp(ops, *case))
    torch.cuda.synchronize()
    for want, kept in zip(alone, results):
        for got in kept:
            assert all(torch.equal(a, b) for a, b in zip(want, got))


def test_several_threads_at_once(ops):
    # more operand pairs than the library keeps tensor maps of
    from concurrent.futures import ThreadPoolExecutor

    threads, pairs = 4, 12
    sets = [[mm_inputs(8 + 16 * i, 128 + 16 * i, 256 + 32 * t, 100 * t + i) for i in range(pairs)] for t in range(threads)]
    torch.cuda.synchronize()

    def work(mine):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            results = [ops.mm_int8_per_token(*mine[k % pairs], out_dtype=torch.float32) for k in range(10 * pairs)]
        stream.synchronize()
        return results

    with ThreadPoolExecutor(threads) as pool:
        everything = list(pool.map(work, sets))
    for mine, results in zip(sets, everything):
        for i, operands in enumerate(mine):
            want = ops.mm_int8_per_token(*operands, out_dtype=torch.float32)
            for got in results[i::pairs]:
                assert torch.equal(got, want)


@pytest.mark.parametrize("n", [1, 16, 200])
def test_captured_and_replayed(ops, n):
    x, residual, w = mlp_setup(n, 512, 1024)
    mlp(ops, x, residual, w)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = mlp(ops, x, residual, w)
    for seed in (21, 22):
        x2, r2, _ = mlp_setup(n, 512, 1024, seed)
        x.copy_(x2)
        residual.copy_(r2)
        graph.replay()
        want = mlp(ops, x2, r2, w)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want))


# ------------------------------------------------------------------ refusals
def test_mm_refusals(ops):
    A, B, sa, sb, bias = mm_inputs(4, 32, 16, 1)
    f = ops.mm_int8_per_token
    bad = [
        (A.cpu(), B, sa, sb), (A.float(), B, sa, sb), (A, B.t().contiguous().t(), sa, sb), (A, B[:8], sa, sb),
        (A, B, sa[:3], sb), (A, B, sa.half(), sb), (A, B, sa, sb[:31]), (A, B, sa, sb, bias[:5]),
        (A, B, sa, sb, bias.half()), (A, B, sa, sb, bias.cpu()), (A[0], B, sa, sb), (A, B, sa[:, None], sb),
    ]
    for args in bad:
        with pytest.raises(ValueError):
            f(*args)
    with pytest.raises(ValueError):
        f(A, B, sa, sb, out_dtype=torch.float64)
    with pytest.raises(ValueError):
        f(A, B, sa, sb, out=torch.empty((4, 31), dtype=torch.float16, device="cuda"))
    with pytest.raises(ValueError):
        f(A, B, sa, sb, out=torch.empty((4, 32), dtype=torch.float32, device="cuda"))


def test_producer_refusals(ops):
    x, r, w, p, gt = norm_inputs(4, 64, F16, F16, F16, "channel", 1)
    wrong = [
        dict(x=x.cpu()), dict(x=x.double()), dict(x=x[:, ::2]), dict(residual=r[:3]), dict(residual=r.bfloat16()),
        dict(weight=w[:63]), dict(weight=w.bfloat16()), dict(post_weight=p.float()), dict(post_weight=p[:5]),
        dict(gate=gt.float()), dict(gate=gt[:7]), dict(gate=gt.expand(3, 64).contiguous()),
        dict(gate=gt.expand(4, 64)), dict(gate=gt[:8].reshape(4, 2)), dict(z_out=torch.empty_like(r, dtype=torch.float32)),
        dict(out=torch.empty_like(x, dtype=torch.float32)),
    ]
    for change in wrong:
        for f in (ops.block_norm, ops.block_norm_quant_per_token):
            with pytest.raises(ValueError):
                f(**{**dict(x=x, residual=r, weight=w, eps=1e-5), **change})
    for bad in (x.cpu(), x.double(), x[0], x.t(), x[:, :0], x[:1].expand(4, 64)):
        with pytest.raises(ValueError):
            ops.quant_per_token(bad)
        with pytest.raises(ValueError):
            ops.swiglu_quant_per_token(bad)
    with pytest.raises(ValueError):
        ops.swiglu_quant_per_token(x[:, :63])
    with pytest.raises(ValueError):
        ops.quant_per_token(x, out=torch.empty((4, 63), dtype=torch.int8, device="cuda"))
    with pytest.raises(ValueError):
        ops.quant_per_token(x, scale_out=torch.empty((5,), device="cuda"))


def test_empty_batches(ops):
    x, r, w, _, _ = norm_inputs(0, 64, F16, F32, F16, "none", 1)
    y, z = ops.block_norm(x, r, w, 1e-5)
    q, s, z = ops.block_norm_quant_per_token(x, r, w, 1e-5)
    assert y.shape == q.shape == z.shape == (0, 64) and s.shape == (0,)
    assert ops.quant_per_token(x)[0].shape == (0, 64) and ops.swiglu_quant_per_token(x)[0].shape == (0, 32)
