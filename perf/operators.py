"""The dynamic-quantisation operators of the INT8 path, as cases to be timed and compared.

One transformer block with 8-bit weights and activations makes these calls per projection: a
producer (block norm, SwiGLU or a plain quantiser) that gives int8 activations with one scale
per token, and the int8 product with one scale per token and one per output channel.  `run`
makes one such call: the operator's definition in elementary torch operations, or the
framework's operator where `own` is true.  Quantised activations are returned as the values
they stand for (q * scale, in bfloat16, whose eight significant bits hold an 8-bit integer),
together with their scales.
"""
import torch

own = False

_TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
_SIZE = {"f16": 2, "bf16": 2, "f32": 4}
EPS = 1e-5
TINY = 2.0 ** -100  # the quantisers' smallest row maximum


def listed():
    return [
        # One token through a small projection: the call's latency is all there is.
        {"name": "mm-token", "op": "mm", "M": 1, "N": 1024, "K": 1024, "out": "f16", "bias": False},
        # Sixteen sequences decoding, gate/up projection: the weights stream from memory once.
        {"name": "mm-decode-16", "op": "mm", "M": 16, "N": 28672, "K": 8192, "out": "bf16", "bias": False},
        # A batch of 128 through the down projection: a long sum, few columns.
        {"name": "mm-decode-128", "op": "mm", "M": 128, "N": 8192, "K": 28672, "out": "bf16", "bias": False},
        # A short prompt through a small layer with bias.
        {"name": "mm-512", "op": "mm", "M": 512, "N": 512, "K": 1024, "out": "f16", "bias": True},
        # A ragged batch against a weight matrix whose rows start at odd addresses, logits in f32.
        {"name": "mm-ragged", "op": "mm", "M": 333, "N": 4999, "K": 5001, "out": "f32", "bias": True},
        # A long prefill: bound by the tensor cores.
        {"name": "mm-8192", "op": "mm", "M": 8192, "N": 8192, "K": 8192, "out": "bf16", "bias": False},
        # One token between two blocks, both norms.
        {"name": "norm-token", "op": "norm", "N": 1, "C": 8192, "x": "f16", "res": "f16", "post": True,
         "gate": 0, "quant": True},
        # A prefill's worth of tokens with a residual stream in f32 and one gate per channel.
        {"name": "norm-prefill", "op": "norm", "N": 4096, "C": 8192, "x": "bf16", "res": "f32", "post": True,
         "gate": 1, "quant": False},
        # Two sequences, each with its own gate, an odd row length, quantised for the next product.
        {"name": "norm-ragged", "op": "norm", "N": 2050, "C": 4999, "x": "f16", "res": "f16", "post": False,
         "gate": 2, "quant": True},
        # The attention output of sixteen decoding sequences in front of the output projection.
        {"name": "quant-16", "op": "quant", "N": 16, "C": 8192, "x": "f16"},
        # Gate and up columns interleaved, a long prefill in front of the down projection.
        {"name": "swiglu-prefill", "op": "swiglu", "N": 4096, "C": 28672, "x": "bf16", "interleaved": True},
        # Gate and up halves side by side, an odd width.
        {"name": "swiglu-ragged", "op": "swiglu", "N": 1023, "C": 11007, "x": "f16", "interleaved": False},
    ]


def _between(rng, lo, hi):
    """An integer of [lo, hi], spread over its logarithm."""
    return min(hi, max(lo, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    op = rng.choice(["mm", "mm", "mm", "norm", "norm", "quant", "swiglu"])
    if op == "mm":
        while True:
            m, n, k = _between(rng, 1, 8192), _between(rng, 256, 28672), _between(rng, 256, 28672)
            if rng.random() < 0.7:  # rows that start at aligned addresses
                n, k = (n + 15) // 16 * 16, (k + 15) // 16 * 16
            if m * n * k <= 1 << 38:
                break
        return {"op": op, "M": m, "N": n, "K": k, "out": rng.choice(["f16", "bf16", "f32"]),
                "bias": rng.random() < 0.5}
    x = rng.choice(["f16", "bf16", "f32"])
    n, c = _between(rng, 1, 8192), _between(rng, 64, 16384)
    if rng.random() < 0.7:
        c = (c + 7) // 8 * 8
    if op == "norm":
        n = min(n, (1 << 25) // c)
        gate = rng.choice([0, 1, 1, n])
        return {"op": op, "N": n, "C": c, "x": x, "res": rng.choice([x, "f32"]), "post": rng.random() < 0.5,
                "gate": gate, "quant": rng.random() < 0.6}
    if op == "quant":
        return {"op": op, "N": min(n, (1 << 26) // c), "C": c, "x": x}
    return {"op": op, "N": min(n, (1 << 26) // c), "C": c, "x": x, "interleaved": rng.random() < 0.5}


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed * 1000003 + 17)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    s = {"op": case["op"]}
    if case["op"] == "mm":
        m, n, k = case["M"], case["N"], case["K"]
        # normal activations and weights, quantised per token and per channel at about 4 sigma
        s["A"] = normal(m, k).mul_(32).round_().clamp_(-127, 127).to(torch.int8)
        s["B"] = normal(k, n).mul_(32).round_().clamp_(-127, 127).to(torch.int8)
        s["scale_A"] = torch.rand(m, generator=g, device="cuda") * 0.045 + 0.005
        s["scale_B"] = torch.rand(n, generator=g, device="cuda") * 0.0009 + 0.0001
        s["bias"] = normal(n) if case["bias"] else None
        s["out"] = _TYPES[case["out"]]
        return s
    t = _TYPES[case["x"]]
    if case["op"] == "norm":
        n, c = case["N"], case["C"]
        s["x"] = (normal(n, c) * 1.5).to(t)
        s["residual"] = (normal(n, c) * 3).to(_TYPES[case["res"]])
        s["weight"] = (1 + 0.2 * normal(c)).to(t)
        s["post_weight"] = (1 + 0.2 * normal(c)).to(t) if case["post"] else None
        s["gate"] = (0.5 * normal(case["gate"], c)).to(t) if case["gate"] else None
        s["residual_scale"] = 0.875
        s["quant"] = case["quant"]
        return s
    wide = case["C"] * (2 if case["op"] == "swiglu" else 1)
    x = normal(case["N"], wide)
    x[:, :: max(1, wide // 16)] *= 8  # a few channels stand out, as they do in earnest
    s["x"] = x.to(t)
    s["interleaved"] = case.get("interleaved", False)
    return s


def _values(q, scale):
    """What int8 activations stand for."""
    out = torch.empty(q.shape, dtype=torch.bfloat16, device=q.device)
    return torch.mul(q, scale[:, None], out=out), scale


def _rms(v, weight):
    return v * torch.rsqrt((v * v).mean(dim=1, keepdim=True) + EPS) * weight.float()


def _quantised(y):
    scale = y.abs().amax(dim=1).clamp_min(TINY) / 127
    q = torch.round(y / scale[:, None])
    return (q * scale[:, None]).to(torch.bfloat16), scale


def _plain(s):
    if s["op"] == "mm":
        y = (s["A"].float() @ s["B"].float()) * s["scale_A"][:, None] * s["scale_B"]
        if s["bias"] is not None:
            y = y + s["bias"]
        return y.to(s["out"])
    x = s["x"].float()
    if s["op"] == "quant":
        return _quantised(x)
    if s["op"] == "swiglu":
        half = x.shape[1] // 2
        gate, up = (x[:, 0::2], x[:, 1::2]) if s["interleaved"] else (x[:, :half], x[:, half:])
        return _quantised(up * gate / (1 + torch.exp(-gate)))
    u = x if s["post_weight"] is None else _rms(x, s["post_weight"])
    if s["gate"] is not None:
        rows = x.shape[0] // s["gate"].shape[0]
        u = u * s["gate"].float().repeat_interleave(rows, dim=0)
    z = s["residual_scale"] * s["residual"].float() + u
    y = _rms(z, s["weight"])
    if s["quant"]:
        return (*_quantised(y), z.to(s["residual"].dtype))
    return y.to(s["x"].dtype), z.to(s["residual"].dtype)


def run(state):
    s = state
    if not own:
        return _plain(s)
    from texo_b200 import ops

    if s["op"] == "mm":
        return ops.mm_int8_per_token(s["A"], s["B"], s["scale_A"], s["scale_B"], s["bias"], out_dtype=s["out"])
    if s["op"] == "quant":
        return _values(*ops.quant_per_token(s["x"]))
    if s["op"] == "swiglu":
        return _values(*ops.swiglu_quant_per_token(s["x"], interleaved=s["interleaved"]))
    args = (s["x"], s["residual"], s["weight"], EPS)
    more = {"post_weight": s["post_weight"], "gate": s["gate"], "residual_scale": s["residual_scale"]}
    if s["quant"]:
        q, scale, z = ops.block_norm_quant_per_token(*args, **more)
        return (*_values(q, scale), z)
    return ops.block_norm(*args, **more)


def work(case):
    if case["op"] == "mm":
        m, n, k = case["M"], case["N"], case["K"]
        return {"bytes": m * k + k * n + 4 * m + 4 * n * (2 if case["bias"] else 1) + m * n * _SIZE[case["out"]],
                "flops": 2 * m * n * k}
    n, c, e = case["N"], case["C"], _SIZE[case["x"]]
    if case["op"] == "norm":
        rows = 1 + int(case["post"]) + case["gate"]
        out = n * c + 4 * n if case["quant"] else n * c * e
        return {"bytes": n * c * e + 2 * n * c * _SIZE[case["res"]] + rows * c * e + out, "flops": 12 * n * c}
    if case["op"] == "quant":
        return {"bytes": n * c * e + n * c + 4 * n, "flops": 3 * n * c}
    return {"bytes": 2 * n * c * e + n * c + 4 * n, "flops": 8 * n * c}


def exact(case, seed):
    """The operators' definitions in 64 bits; quantised values are the nearest multiples of the row's scale."""
    s = prepare(case, seed)
    if case["op"] == "mm":
        total = torch.matmul(s["A"].to(torch.float64), s["B"].to(torch.float64))
        total *= torch.outer(s["scale_A"].double(), s["scale_B"].double())
        return total if s["bias"] is None else total.add_(s["bias"].double())

    def levels(v):
        top = torch.maximum(v.amax(dim=-1), -v.amin(dim=-1))
        step = torch.clamp(top, min=TINY).div(127.0).unsqueeze(-1)
        return torch.round(v.div(step)).mul(step), step.squeeze(-1)

    def normed(v, w):
        return v.div(torch.sqrt(v.square().sum(dim=-1, keepdim=True).div(v.shape[-1]).add(EPS))).mul(w.double())

    x = s["x"].double()
    if case["op"] == "quant":
        return levels(x)
    if case["op"] == "swiglu":
        pairs = x.view(case["N"], case["C"], 2) if case["interleaved"] else x.view(case["N"], 2, case["C"]).transpose(1, 2)
        return levels(torch.sigmoid(pairs[..., 0]).mul(pairs[..., 0]).mul(pairs[..., 1]))
    if case["post"]:
        x = normed(x, s["post_weight"])
    if case["gate"]:
        x = x.view(case["gate"], -1, case["C"]).mul(s["gate"].double().unsqueeze(1)).view(case["N"], case["C"])
    z = x.add(s["residual"].double(), alpha=s["residual_scale"])
    y = normed(z, s["weight"])
    return (*levels(y), z) if case["quant"] else (y, z)
