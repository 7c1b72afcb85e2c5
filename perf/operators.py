"""Measured cases of the 8-bit operators around a DiT block's linear layers.

Three operators, each reached as a user's program reaches it:

* `add_norm`: the gated residual addition, RMSNorm or LayerNorm with its
  affine and modulation, and an output in e4m3 with a float32 scale for each
  128 features of a row (or in bf16);
* `quantize_fp8`: a tensor as e4m3 values with those scales;
* `linear_fp8`: the matrix product of e4m3 activations (a scale for each row
  and 128 input features) and e4m3 weights (a scale for each 128 x 128
  block), with bias and tanh GELU, its output in bf16 or again in e4m3.

`own` False computes them with elementary torch operations in float32,
`own` True with vidax_b200. The sizes are Wan2.1's (dim 1536 / 5120, FFN 8960
/ 13824, 512 text tokens of 4096 features; 4680, 32760 and 75600 video
tokens) and odd ones between them.
"""
import math

import torch

own = False

BLOCK = 128
FP8_MAX = 448.0
AMAX_FLOOR = 2.0 ** -100   # an all-zero block gets the scale 2^-100 / 448, not 0
EPS = 1e-6


# ------------------------------------------------------------------ cases


def listed():
    return [
        # a short prompt's rows: launch and latency decide
        {"name": "norm-few-rows", "op": "norm", "batch": 1, "rows": 7, "dim": 1536, "norm": "rms",
         "stream": "float32", "mod": False, "gate": False, "out": "fp8"},
        # a block's norm between two sub-layers, Wan2.1-1.3B at 480p, 81 frames
        {"name": "norm-480p", "op": "norm", "batch": 1, "rows": 32760, "dim": 1536, "norm": "layer",
         "stream": "float32", "mod": True, "gate": True, "out": "fp8"},
        # the 14B model's width at 720p, 81 frames
        {"name": "norm-720p", "op": "norm", "batch": 1, "rows": 75600, "dim": 5120, "norm": "rms",
         "stream": "float32", "mod": False, "gate": True, "out": "fp8"},
        # a bf16 residual stream, two batch items, a width that no vector divides
        {"name": "norm-odd", "op": "norm", "batch": 2, "rows": 2339, "dim": 1187, "norm": "rms",
         "stream": "bfloat16", "mod": True, "gate": False, "out": "bfloat16"},
        # the attention output before its projection
        {"name": "quantize-480p", "op": "quantize", "rows": 32760, "dim": 1536, "dtype": "bfloat16"},
        # a ragged text batch, its last block of features short
        {"name": "quantize-odd", "op": "quantize", "rows": 487, "dim": 4091, "dtype": "float32"},
        # one token (a timestep embedding) through the modulation projection: weight bytes decide
        {"name": "linear-one-token", "op": "linear", "m": 1, "k": 1536, "n": 9216, "act": False,
         "out": "bfloat16"},
        # a prompt through the text embedding
        {"name": "linear-text", "op": "linear", "m": 487, "k": 4096, "n": 1536, "act": True,
         "out": "bfloat16"},
        # three latent frames through the fused q, k, v projection
        {"name": "linear-3-frames", "op": "linear", "m": 4680, "k": 1536, "n": 4608, "act": False,
         "out": "bfloat16"},
        # the 1.3B model's FFN at 480p, up (output again in e4m3) and down
        {"name": "linear-ffn-up-480p", "op": "linear", "m": 32760, "k": 1536, "n": 8960, "act": True,
         "out": "fp8"},
        {"name": "linear-ffn-down-480p", "op": "linear", "m": 32760, "k": 8960, "n": 1536,
         "act": False, "out": "bfloat16"},
        # the 14B model's FFN at 720p: the largest product
        {"name": "linear-ffn-up-720p", "op": "linear", "m": 75600, "k": 5120, "n": 13824, "act": True,
         "out": "fp8"},
    ]


def _spread(rng, lo, hi):
    """A size between lo and hi, even over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["norm", "quantize", "linear", "linear"])
    if op == "norm":
        dim = _spread(rng, 128, 5120)
        if rng.random() < 0.6:
            dim = max(128, dim // 64 * 64)
        rows = _spread(rng, 1, min(75600, 75600 * 5120 // dim // 2))
        return {"op": op, "batch": rng.choice([1, 1, 2]), "rows": rows, "dim": dim,
                "norm": rng.choice(["rms", "layer"]), "stream": rng.choice(["float32", "float32", "bfloat16"]),
                "mod": rng.random() < 0.5, "gate": rng.random() < 0.5,
                "out": rng.choice(["fp8", "fp8", "bfloat16"])}
    if op == "quantize":
        return {"op": op, "rows": _spread(rng, 1, 75600), "dim": _spread(rng, 64, 13824),
                "dtype": rng.choice(["bfloat16", "float32"])}
    k, n = _spread(rng, 64, 13824), _spread(rng, 16, 13824)
    if rng.random() < 0.6:
        k, n = max(64, k // 64 * 64), max(64, n // 64 * 64)
    m = _spread(rng, 1, min(75600, 75600 * 5120 * 13824 // (2 * k * n)))
    return {"op": op, "m": m, "k": k, "n": n, "act": rng.random() < 0.4,
            "out": rng.choice(["bfloat16", "bfloat16", "float32", "fp8"])}


# ------------------------------------------------------------------ inputs


def _pad16(data):
    """`data` (rows, k) in rows that start on 16-byte boundaries, as the quantiser lays them out."""
    rows, k = data.shape
    buf = torch.zeros((rows, -(-k // 16) * 16), dtype=data.dtype, device=data.device)
    buf[:, :k] = data
    return buf[:, :k]


def _quantised(x, block_rows):
    """Plain quantisation: (e4m3 values, float32 scales) of (rows, k) with a scale for each
    block_rows x 128 block."""
    rows, k = x.shape
    kb, rb = -(-k // BLOCK), -(-rows // block_rows)
    padded = torch.zeros((rb * block_rows, kb * BLOCK), dtype=torch.float32, device=x.device)
    padded[:rows, :k] = x
    blocks = padded.view(rb, block_rows, kb, BLOCK)
    amax = blocks.abs().amax(dim=(1, 3)).clamp_min(AMAX_FLOOR)
    inv = FP8_MAX / amax
    q = (blocks * inv[:, None, :, None]).clamp(-FP8_MAX, FP8_MAX).to(torch.float8_e4m3fn)
    return q.view(rb * block_rows, kb * BLOCK)[:rows, :k], amax / FP8_MAX


def _dequantised(data, scale, block_rows):
    """The float32 values that e4m3 `data` with these scales stands for."""
    rows, k = data.shape
    s = scale.repeat_interleave(BLOCK, dim=1)[:, :k]
    if block_rows > 1:
        s = s.repeat_interleave(block_rows, dim=0)[:rows]
    return data.float() * s


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda")

    st = {"case": case}
    if case["op"] == "norm":
        b, rows, d = case["batch"], case["rows"], case["dim"]
        stream = getattr(torch, case["stream"])
        # a residual stream with a few strong features, as deep blocks have them
        strong = 1 + 8 * (torch.rand(d, generator=g, device="cuda") > 0.98).float()
        st["x"] = (normal(b, rows, d) * strong).to(stream)
        st["y"] = normal(b, rows, d).to(torch.bfloat16)
        st["sum"] = torch.empty_like(st["x"])
        st["gate"] = normal(b, d) * 0.3 if case["gate"] else None
        st["weight"] = 1 + 0.1 * normal(d)
        st["bias"] = 0.1 * normal(d) if case["norm"] == "layer" else None
        st["scale"] = 0.3 * normal(b, d) if case["mod"] else None
        st["shift"] = 0.3 * normal(b, d) if case["mod"] else None
    elif case["op"] == "quantize":
        r, d = case["rows"], case["dim"]
        st["x"] = (normal(r, d) * torch.exp(normal(r, 1))).to(getattr(torch, case["dtype"]))
    else:
        m, k, n = case["m"], case["k"], case["n"]
        xd, xs = _quantised(normal(m, k), 1)
        wd, ws = _quantised(0.02 * normal(n, k), BLOCK)
        st["xd"], st["wd"] = _pad16(xd), _pad16(wd)
        st["xs"] = xs.t().contiguous().t()   # scales of a block of features side by side, as the quantiser lays them out
        st["ws"] = ws
        st["bias"] = 0.1 * normal(n)
    return st


# ------------------------------------------------------------------ one pass


def _run_own(st):
    import vidax_b200 as vx
    c = st["case"]
    out = {"fp8": torch.float8_e4m3fn, "bfloat16": torch.bfloat16, "float32": torch.float32}
    if c["op"] == "norm":
        r, total = vx.add_norm(st["x"], st["y"], st["gate"], norm=c["norm"], weight=st["weight"],
                               bias=st["bias"], scale=st["scale"], shift=st["shift"], eps=EPS,
                               out_dtype=out[c["out"]], residual_out=st["sum"])
        return [total, r.data, r.scale] if c["out"] == "fp8" else [total, r]
    if c["op"] == "quantize":
        r = vx.quantize_fp8(st["x"])
        return [r.data, r.scale]
    r = vx.linear_fp8(vx.Fp8Tensor(st["xd"], st["xs"]), vx.Fp8Tensor(st["wd"], st["ws"]),
                      st["bias"], activation="gelu_tanh" if c["act"] else None,
                      out_dtype=out[c["out"]])
    return [r.data, r.scale] if c["out"] == "fp8" else r


def _gelu_tanh(x):
    return 0.5 * x * (1 + torch.tanh(math.sqrt(2 / math.pi) * (x + 0.044715 * x * x * x)))


def _rounded(y, kind):
    """float32 (rows, features) in the output's type, as a list of outputs."""
    if kind == "fp8":
        return list(_quantised(y, 1))
    return [y.to(getattr(torch, kind))]


def run(st):
    if own:
        return _run_own(st)
    c = st["case"]
    if c["op"] == "norm":
        y = st["y"].float()
        if st["gate"] is not None:
            y = y * st["gate"][:, None, :]
        total = (st["x"].float() + y).to(st["x"].dtype)
        h = total.float()
        if c["norm"] == "layer":
            h = h - h.mean(dim=-1, keepdim=True)
        h = h * torch.rsqrt((h * h).mean(dim=-1, keepdim=True) + EPS) * st["weight"]
        if st["bias"] is not None:
            h = h + st["bias"]
        if st["scale"] is not None:
            h = h * (1 + st["scale"][:, None, :]) + st["shift"][:, None, :]
        d = c["dim"]
        outs = _rounded(h.reshape(-1, d), c["out"])
        return [total] + [o.reshape(c["batch"], c["rows"], -1) for o in outs]
    if c["op"] == "quantize":
        return list(_quantised(st["x"].float(), 1))
    y = _dequantised(st["xd"], st["xs"], 1) @ _dequantised(st["wd"], st["ws"], BLOCK).t() + st["bias"]
    if c["act"]:
        y = _gelu_tanh(y)
    outs = _rounded(y, c["out"])
    return outs if c["out"] == "fp8" else outs[0]


# ------------------------------------------------------------------ bounds and exact values


def work(case):
    size = {"float32": 4, "bfloat16": 2}

    def out_bytes(rows, d, kind):
        return rows * d + 4 * rows * -(-d // BLOCK) if kind == "fp8" else rows * d * size[kind]

    if case["op"] == "norm":
        rows, d = case["batch"] * case["rows"], case["dim"]
        vectors = 1 + (case["norm"] == "layer") + case["batch"] * (2 * case["mod"] + case["gate"])
        return {"bytes": rows * d * (2 * size[case["stream"]] + 2) + out_bytes(rows, d, case["out"])
                + 4 * d * vectors, "flops": 10 * rows * d}
    if case["op"] == "quantize":
        rows, d = case["rows"], case["dim"]
        return {"bytes": rows * d * size[case["dtype"]] + out_bytes(rows, d, "fp8"),
                "flops": 3 * rows * d}
    m, k, n = case["m"], case["k"], case["n"]
    kb = -(-k // BLOCK)
    return {"bytes": m * k + n * k + 4 * (m * kb + -(-n // BLOCK) * kb + n)
            + out_bytes(m, n, case["out"]), "flops": 2 * m * n * k}


def _exact_fp8(y):
    """(values before their rounding to e4m3, scales) of float64 rows."""
    rows, d = y.shape
    blocks = torch.nn.functional.pad(y, (0, -d % BLOCK)).view(rows, -1, BLOCK)
    s = blocks.abs().amax(dim=2).clamp_min(AMAX_FLOOR) / FP8_MAX
    return [(blocks / s[:, :, None]).view(rows, -1)[:, :d], s]


def _exact_values(data, scale, block_rows):
    """float64 values of e4m3 blocks, block by block."""
    rows, k = data.shape
    kb, rb = scale.shape[1], -(-rows // block_rows)
    v = torch.nn.functional.pad(data.double(), (0, kb * BLOCK - k, 0, rb * block_rows - rows))
    v = v.view(rb, block_rows, kb, BLOCK) * scale.double()[:, None, :, None]
    return v.view(rb * block_rows, kb * BLOCK)[:rows, :k]


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "quantize":
        return _exact_fp8(st["x"].double())
    if case["op"] == "norm":
        b, rows, d = case["batch"], case["rows"], case["dim"]
        # in parts of the rows: several float64 copies of the largest stream at once are not needed
        total, outs = [], []
        part = max(1, (1 << 28) // d)
        for i in range(b):
            for r0 in range(0, rows, part):
                x, y = st["x"][i, r0:r0 + part].double(), st["y"][i, r0:r0 + part].double()
                x = x + (y if st["gate"] is None else y * st["gate"][i].double())
                # the sum is stored in the stream's type, and the norm is that of the stored sum
                h = x.to(st["x"].dtype).double()
                total.append(x)
                mean = h.mean(dim=1, keepdim=True) if case["norm"] == "layer" else 0.0
                var = ((h - mean) ** 2).mean(dim=1, keepdim=True)
                h = (h - mean) / torch.sqrt(var + EPS) * st["weight"].double()
                if st["bias"] is not None:
                    h = h + st["bias"].double()
                if st["scale"] is not None:
                    h = h * (1 + st["scale"][i].double()) + st["shift"][i].double()
                outs.append(_exact_fp8(h) if case["out"] == "fp8" else [h])
        return [torch.cat(total).view(b, rows, d)] + [
            torch.cat([o[j] for o in outs]).view(b, rows, -1) for j in range(len(outs[0]))]
    w = _exact_values(st["wd"], st["ws"], BLOCK).t()
    parts = []
    part = max(1, (1 << 28) // max(case["k"], case["n"]))
    for r0 in range(0, case["m"], part):
        y = _exact_values(st["xd"][r0:r0 + part], st["xs"][r0:r0 + part], 1) @ w
        y = y + st["bias"].double()
        if case["act"]:
            u = math.sqrt(2 / math.pi) * (y + 0.044715 * y ** 3)
            y = y * torch.sigmoid(2 * u)
        parts.append(_exact_fp8(y) if case["out"] == "fp8" else [y])
    outs = [torch.cat([p[j] for p in parts]) for j in range(len(parts[0]))]
    return outs if case["out"] == "fp8" else outs[0]
