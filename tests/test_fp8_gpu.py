"""The 8-bit linear layer's operators (vidax_b200.fp8) against their float64
restatement (oracle/fp8_ref.py).

Tolerances, derived from the formulas:

* e4m3 has 3 mantissa bits: its rounding is off by at most 2^-4 of the value,
  or half the subnormal step (2^-10, in units of the scale).
* float32 operations are off by at most 2^-24 of their result; sums of n
  terms by n of those of the sum of magnitudes, however they are ordered.
* bf16 rounding is off by at most 2^-8 of the value.
"""
import numpy as np
import pytest
import torch

from oracle import fp8_ref

pytestmark = pytest.mark.gpu

U32 = 2.0 ** -24   # float32 rounding
UBF = 2.0 ** -8    # bf16 rounding
U8 = 2.0 ** -4     # e4m3 rounding of a normal value
SUB = 2.0 ** -10   # half the e4m3 subnormal step


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _f64(t):
    return t.double().cpu().numpy()


def _ok():
    from vidax_b200 import _lib
    torch.cuda.synchronize()
    assert _lib.device_status() == 0


def _call(name, a):
    """The C entry point itself."""
    import ctypes
    from vidax_b200 import _lib, fp8
    _lib.check(fp8._entry(name, a)(ctypes.byref(a), torch.cuda.current_stream().cuda_stream))


def _check_blocks(q, want, block_rows=1, err=0.0):
    """An Fp8Tensor against the float64 values it rounds, known within `err`."""
    want = want.reshape(-1, want.shape[-1])
    data, scale = _f64(q.data).reshape(want.shape), _f64(q.scale)
    scale = scale.reshape(-1, scale.shape[-1])
    err = np.broadcast_to(err, want.shape)
    amax = np.maximum(fp8_ref.block_amax(want, block_rows), fp8_ref.AMAX_FLOOR)
    # 1/448 and the product round once each; the largest magnitude is off by err
    off = fp8_ref.block_amax(err, block_rows)
    assert (np.abs(scale * 448 - amax) <= 3 * U32 * amax + off).all()
    s = fp8_ref.expand(scale, block_rows, *want.shape)
    # the factor 448 / a, its product with x, and the scale: four roundings
    tol = (U8 + 4 * U32) * np.abs(want) + SUB * s + 1.1 * err
    assert (np.abs(data * s - want) <= tol).all()


# ------------------------------------------------------------------ quantize


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("shape", [(1, 1), (1, 128), (3, 127), (5, 129), (4, 256), (9, 1000),
                                   (130, 1536), (2, 7, 264), (257, 4091)])
def test_quantize_rows(shape, dtype):
    import vidax_b200 as vx
    x = (torch.randn(shape, generator=_gen(1), device="cuda") * 3).to(dtype)
    q = vx.quantize_fp8(x)
    _ok()
    assert q.data.shape == x.shape and q.scale.shape == (*shape[:-1], -(-shape[-1] // 128))
    _check_blocks(q, _f64(x))
    # bit for bit the float32 formula (a tensor divided by a tensor: torch turns a
    # number over a tensor into a rounded reciprocal times that number)
    a = x.float().abs()
    pad = torch.nn.functional.pad(a, (0, -shape[-1] % 128)).unflatten(-1, (-1, 128)).amax(-1)
    inv = (torch.full_like(pad, 448.0) / pad.clamp_min(2.0 ** -100)).repeat_interleave(128, -1)[..., :shape[-1]]
    assert torch.equal(q.data.float(), (x.float() * inv).to(torch.float8_e4m3fn).float())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("shape", [(1, 1), (127, 130), (128, 128), (129, 264), (300, 1000)])
def test_quantize_weight_blocks(shape, dtype):
    import vidax_b200 as vx
    w = (torch.randn(shape, generator=_gen(2), device="cuda") * 0.02).to(dtype)
    q = vx.quantize_fp8(w, block_rows=128)
    _ok()
    assert q.scale.shape == (-(-shape[0] // 128), -(-shape[1] // 128))
    _check_blocks(q, _f64(w), 128)


def test_quantize_strided_and_misaligned_rows():
    import vidax_b200 as vx
    big = torch.randn((6, 1001), generator=_gen(3), device="cuda").bfloat16()
    for x in (big[:, 1:258], big[::2, 3:], big.t()[:, :6], big[:, :256]):
        q = vx.quantize_fp8(x)
        ref = vx.quantize_fp8(x.contiguous())
        assert torch.equal(q.data.float(), ref.data.float()) and torch.equal(q.scale, ref.scale)
    _ok()


def test_quantize_zero_tiny_huge_and_nonfinite_blocks():
    import vidax_b200 as vx
    x = torch.zeros((6, 256), device="cuda")
    x[1, 3] = 1e-38          # below the floor: rounds to 0
    x[2, :128] = 3e38
    x[3, 5] = float("nan")
    x[3, 6] = 2.0
    x[4, 130] = float("inf")
    x[5, 0] = 2.0 ** -90
    q = vx.quantize_fp8(x)
    _ok()
    d, s = q.data.float(), q.scale
    assert torch.equal(d[0], torch.zeros_like(d[0])) and (s[0] > 0).all()
    assert (d[1] == 0).all() and torch.isfinite(s[1]).all()
    assert (d[2, :128] == 448).all()
    assert torch.isnan(d[3, 5]) and d[3, 6] == 448 and int(torch.isnan(d[3]).sum()) == 1
    v = q.dequantize()
    assert torch.isnan(v[4, 128:]).all() and (v[4, :128] == 0).all()
    assert d[5, 0] == 448
    assert vx.quantize_fp8(x[:0]).data.shape == (0, 256)


def test_quantize_leaves_the_padding_and_later_rows_alone():
    """Only `dim` bytes of `rows` rows are written."""
    from vidax_b200 import fp8
    x = torch.randn((5, 130), generator=_gen(4), device="cuda")
    dst = torch.full((8, 160), 77, dtype=torch.uint8, device="cuda")
    sc = torch.full((8, 2), -1.0, device="cuda")
    a = fp8.QuantizeFp8Args()
    a.src, a.dst, a.scale = x.data_ptr(), dst.data_ptr(), sc.data_ptr()
    a.src_stride, a.dst_stride = 130, 160
    a.scale_stride[:] = (2, 1)
    a.rows, a.dim, a.src_type, a.block_rows = 5, 130, 0, 1
    _call("vx_quantize_fp8", a)
    _ok()
    assert (dst[:5, 130:] == 77).all() and (dst[5:] == 77).all() and (sc[5:] == -1).all()
    assert torch.equal(dst[:5, :130], fp8.quantize_fp8(x).data.view(torch.uint8))


# ------------------------------------------------------------------ add_norm


def _norm_case(b, l, dim, stream, seed):
    g = _gen(seed)

    def r(*s):
        return torch.randn(s, generator=g, device="cuda")

    return {"x": (r(b, l, dim) * 2 + 0.5).to(stream), "y": r(b, l, dim).bfloat16(),
            "gate": r(b, dim) * 0.5, "weight": 1 + 0.2 * r(dim), "bias": 0.3 * r(dim),
            "scale": 0.4 * r(b, dim), "shift": 0.4 * r(b, dim)}


def _check_norm(c, norm, out, total, eps=1e-6, before=None):
    x0 = _f64(c["x"] if before is None else before)
    n64 = {k: None if c.get(k) is None else _f64(c[k]) for k in
           ("y", "gate", "weight", "bias", "scale", "shift")}
    bf = c["x"].dtype == torch.bfloat16
    # the stored sum: one fused multiply-add, then the stream's rounding
    if n64["y"] is not None:
        g = 1.0 if n64["gate"] is None else n64["gate"][:, None]
        exact = x0 + n64["y"] * g
        u = UBF if bf else 0.0
        assert (np.abs(_f64(total) - exact) <= (u + 2 * U32) * np.abs(exact)).all()
    h = _f64(total)  # what is normalised is what is stored
    want, _ = fp8_ref.add_norm(h, None, None, norm, n64["weight"], n64["bias"], n64["scale"],
                               n64["shift"], eps, lambda v: v)
    # Row sums: below 64 terms per lane and 8 levels across lanes and warps,
    # so mean and variance are off by < 80 U32 of the mean magnitude (the
    # variance's terms are all positive); rstd halves that and adds 4 of its
    # own; subtraction, products and sums of the epilogue add 6 of the
    # magnitudes that meet there.
    m = h.mean(-1, keepdims=True) if norm == "layer" else 0.0
    rstd = 1 / np.sqrt(((h - m) ** 2).mean(-1, keepdims=True) + eps)
    w = 1.0 if n64["weight"] is None else np.abs(n64["weight"])
    b = 0.0 if n64["bias"] is None else np.abs(n64["bias"])
    s = 1.0 if n64["scale"] is None else np.abs(1 + n64["scale"])[:, None] + U32
    t = 0.0 if n64["shift"] is None else np.abs(n64["shift"])[:, None]
    mag = (np.abs(h - m) * 50 + (80 * np.abs(h).mean(-1, keepdims=True) if norm == "layer" else 0)) * rstd
    err = U32 * ((mag * w + 6 * (np.abs(h - m) * rstd * w + b)) * s + 4 * t)
    if isinstance(out, tuple):
        _check_blocks(out, want, err=err.reshape(-1, want.shape[-1]))
    else:
        assert (np.abs(_f64(out) - want) <= UBF * (np.abs(want) + err) + err).all()


@pytest.mark.parametrize("out", ["fp8", "bf16"])
@pytest.mark.parametrize("stream", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("norm", ["rms", "layer"])
@pytest.mark.parametrize("b,l,dim", [(1, 1, 1), (1, 3, 128), (2, 5, 200), (1, 9, 1187), (2, 4, 1536),
                                     (1, 700, 512), (1, 650, 1000), (1, 600, 1536), (1, 3, 5120),
                                     (1, 2, 8000), (1, 2, 13824), (1, 2, 16392), (1, 2, 20001)])
def test_add_norm(b, l, dim, norm, stream, out):
    """Every variant by width (registers, several warps per row, re-read) and
    by row count, vector and element loads."""
    import vidax_b200 as vx
    c = _norm_case(b, l, dim, stream, dim + l)
    o, total = vx.add_norm(**c, norm=norm,
                           out_dtype=torch.float8_e4m3fn if out == "fp8" else torch.bfloat16)
    _ok()
    assert total.data_ptr() != c["x"].data_ptr() and total.dtype == stream
    _check_norm(c, norm, o, total)


@pytest.mark.parametrize("out", ["fp8", "bf16"])
@pytest.mark.parametrize("stream", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("dim", [129, 515, 1187, 1500, 2047, 2500])
def test_add_norm_odd_widths_many_rows(dim, stream, out):
    """Rows off the 16-byte boundaries, enough of them for the variants with
    few warps per row."""
    import vidax_b200 as vx
    c = _norm_case(1, 700, dim, stream, dim)
    o, total = vx.add_norm(**c, norm="layer",
                           out_dtype=torch.float8_e4m3fn if out == "fp8" else torch.bfloat16)
    _ok()
    _check_norm(c, "layer", o, total)


@pytest.mark.parametrize("missing", ["y", "gate", "weight", "bias", "scale", "shift", "all"])
def test_add_norm_optional_parts(missing):
    import vidax_b200 as vx
    c = _norm_case(2, 6, 384, torch.float32, 11)
    for k in list(c):
        if k != "x" and (missing in (k, "all") or (missing == "y" and k == "gate")):
            c[k] = None
    o, total = vx.add_norm(**c, norm="layer")
    _ok()
    if c["y"] is None:
        assert total is c["x"]
    _check_norm(c, "layer", o, total)


def test_add_norm_in_place_strided_and_misaligned():
    import vidax_b200 as vx
    c = _norm_case(2, 33, 256, torch.float32, 12)
    ref, tref = vx.add_norm(**c, norm="rms")
    # modulation rows of a (B, 6, dim) buffer, y a slice of a wider buffer, x updated in place
    mod = torch.stack([c["scale"], c["shift"], c["gate"]], 1)
    wide = torch.zeros((2, 33, 3 * 256), dtype=torch.bfloat16, device="cuda")
    wide[..., 256:512] = c["y"]
    x = c["x"].clone()
    o, t = vx.add_norm(x, wide[..., 256:512], mod[:, 2], norm="rms", weight=c["weight"],
                       bias=c["bias"], scale=mod[:, 0:1], shift=mod[:, 1:2], residual_out=x)
    _ok()
    assert t is x and torch.equal(x, tref) and torch.equal(o, ref)
    # rows that start on 4-byte boundaries only: the element path, the same numbers
    odd = torch.zeros((2 * 33 * 257 + 1,), device="cuda")[1:].view(2, 33, 257)[..., :256]
    odd.copy_(c["x"])
    c2 = dict(c, x=odd)
    o2, t2 = vx.add_norm(**c2, norm="rms")
    _ok()
    assert torch.equal(t2, tref) and torch.equal(o2, ref)


def test_add_norm_refuses_overlapping_sums():
    import vidax_b200 as vx
    buf = torch.zeros((5, 64), device="cuda")
    y = torch.zeros((4, 64), dtype=torch.bfloat16, device="cuda")
    with pytest.raises(ValueError, match="apart"):
        vx.add_norm(buf[:4], y, residual_out=buf[1:])
    x = torch.zeros((4, 64), dtype=torch.bfloat16, device="cuda")
    with pytest.raises(ValueError, match="apart"):
        vx.add_norm(x, y, residual_out=y)
    with pytest.raises(ValueError, match="evenly"):
        vx.add_norm(buf[:4], y, residual_out=torch.zeros((64, 4), device="cuda").t())
    with pytest.raises(ValueError):
        vx.add_norm(buf[:4], None, residual_out=buf[:4])
    with pytest.raises(NotImplementedError, match="gradient"):
        vx.add_norm(buf[:4], y, weight=torch.ones(64, device="cuda", requires_grad=True))
    with pytest.raises(ValueError, match="weight"):
        vx.add_norm(buf[:4], y, weight=torch.ones(63, device="cuda"))


def test_add_norm_refuses_what_it_would_overwrite_in_place():
    """residual_out=x: y and the vectors are compared with it too."""
    import vidax_b200 as vx
    buf = torch.randn((9, 64), generator=_gen(16), device="cuda")
    h = buf.bfloat16()
    y = torch.zeros((8, 64), dtype=torch.bfloat16, device="cuda")
    with pytest.raises(ValueError, match="apart"):
        vx.add_norm(h[1:], h[:-1], residual_out=h[1:])
    for x in (buf[1:], buf[:8]):
        for name in ("weight", "bias"):
            with pytest.raises(ValueError, match="apart"):
                vx.add_norm(x, y, residual_out=x, **{name: buf[3]})
        for name in ("gate", "scale", "shift"):
            with pytest.raises(ValueError, match="apart"):
                vx.add_norm(x, y, residual_out=x, **{name: buf[3:4]})
            with pytest.raises(ValueError, match="apart"):
                vx.add_norm(x.clone(), y, residual_out=x, **{name: buf[3:4]})
    assert torch.equal(buf.bfloat16(), h)
    with pytest.raises(TypeError, match="residual_out"):
        vx.add_norm(x, y, residual_out=[1])


def test_add_norm_in_place_on_columns_of_one_buffer():
    """x and y side by side in a wider buffer, y = x itself, and a copied x."""
    import vidax_b200 as vx
    wide = torch.randn((40, 3 * 128), generator=_gen(17), device="cuda").bfloat16()
    x, y = wide[:, :128], wide[:, 128:256]
    o, t = vx.add_norm(x.clone(), y.clone(), norm="layer")
    rest = wide[:, 128:].clone()
    o2, t2 = vx.add_norm(x, y, norm="layer", residual_out=x)
    assert t2 is x and torch.equal(x, t) and torch.equal(o2, o) and torch.equal(wide[:, 128:], rest)
    o, t = vx.add_norm(y.clone(), y.clone())
    o2, t2 = vx.add_norm(y, y, residual_out=y)
    assert torch.equal(t2, t) and torch.equal(o2, o)
    _ok()


@pytest.mark.parametrize("stream", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows", [3, 700])
@pytest.mark.parametrize("dim", [129, 300, 768, 1187, 1536, 2500, 4091, 5120, 8000, 13824, 16392, 20001])
def test_add_norm_in_place_is_the_same(dim, rows, stream):
    """Every variant by width and row count with residual_out=x, on rows that
    lie densely and in a wider buffer off the 16-byte boundaries (which may be
    another variant, with its own order of sums): bit for bit what the same rows
    give into a new tensor, and nothing around the rows touched."""
    import vidax_b200 as vx
    c = _norm_case(1, rows, dim, stream, dim + rows)
    for out in (torch.float8_e4m3fn, torch.bfloat16):
        wide = torch.full((rows, dim + 3), 9.0, dtype=stream, device="cuda")
        for x in (torch.empty_like(c["x"]), wide[None, :, 1:1 + dim]):
            x.copy_(c["x"])
            o, total = vx.add_norm(**dict(c, x=x), norm="layer", out_dtype=out)
            if rows == 3:
                _check_norm(c, "layer", o, total)
            o2, t2 = vx.add_norm(**dict(c, x=x), norm="layer", out_dtype=out, residual_out=x)
            _ok()
            assert t2 is x and torch.equal(x, total)
            for a, b in zip(o if isinstance(o, tuple) else (o,), o2 if isinstance(o2, tuple) else (o2,)):
                assert torch.equal(a.float(), b.float())
        assert (wide[:, 0] == 9).all() and (wide[:, 1 + dim:] == 9).all()


def test_add_norm_many_batch_items_of_one_row():
    """A CTA's run of rows crosses a batch item at every row."""
    import vidax_b200 as vx
    c = _norm_case(1500, 1, 384, torch.float32, 15)
    o, total = vx.add_norm(**c, norm="layer", out_dtype=torch.float8_e4m3fn)
    _ok()
    _check_norm(c, "layer", o, total)


def test_add_norm_large_mean_keeps_its_variance():
    """LayerNorm of rows with a mean 1000 times their deviation: E[h^2] - m^2
    in float32 would lose the variance."""
    import vidax_b200 as vx
    x = torch.randn((1, 5, 1536), generator=_gen(13), device="cuda") + 1000
    o, _ = vx.add_norm(x, norm="layer", out_dtype=torch.bfloat16)
    _ok()
    _check_norm({"x": x}, "layer", o, x)


def test_add_norm_equals_the_separate_calls():
    """gated_residual_ then ln_modulate, whose results it replaces."""
    import vidax_b200 as vx
    from vidax_b200.wan_dit import gated_residual_, ln_modulate
    c = _norm_case(2, 100, 1536, torch.float32, 14)
    x = c["x"].clone()
    gated_residual_(x, c["y"], c["gate"])
    ref = ln_modulate(x, 1e-6, scale=c["scale"], shift=c["shift"])
    o, total = vx.add_norm(c["x"], c["y"], c["gate"], norm="layer", scale=c["scale"],
                           shift=c["shift"])
    _ok()
    assert torch.allclose(total, x, rtol=2 ** -22, atol=2 ** -22)
    assert float((o.float() - ref.float()).abs().max()) <= 2 * UBF * float(ref.float().abs().max())


# ------------------------------------------------------------------ linear


def _operands(m, n, k, seed):
    import vidax_b200 as vx
    g = _gen(seed)
    x = vx.quantize_fp8(torch.randn((m, k), generator=g, device="cuda")
                        * torch.exp(torch.randn((m, 1), generator=g, device="cuda")))
    w = vx.quantize_fp8(0.05 * torch.randn((n, k), generator=g, device="cuda"), 128)
    return x, w, 0.3 * torch.randn((n,), generator=g, device="cuda")


def _check_linear(x, w, bias, gelu, out):
    xs, ws = _f64(x.scale).reshape(-1, x.scale.shape[-1]), _f64(w.scale)
    xd = _f64(x.data).reshape(xs.shape[0], -1)
    b64 = None if bias is None else _f64(bias)
    y, mag = fp8_ref.linear(xd, xs, _f64(w.data), ws, b64)
    # A block's 128 products are exact; their sum is off by at most one unit
    # (2^-23, sums may truncate) of the magnitudes per addition of 32 aligned
    # terms and per MMA; a block then costs the scales' product, the
    # multiplication and the addition to the running sum.
    err = (36 * 2 * U32 + (xs.shape[1] + 4) * U32) * mag
    if gelu:
        # |gelu'| < 1.13; the exponential's argument t = 2 u log2(e) is off by
        # 6 U32 |t|, the exponential and the reciprocal by 2^-21 of theirs;
        # below t = -60 the quotient is cut off at |y| 2^-60.
        t = np.minimum(2.31 * np.abs(y) * (1 + 0.0448 * y * y), 60)
        want = fp8_ref.gelu_tanh(y)
        err = 1.13 * err + (6 * U32 * t + 2.0 ** -20) * np.abs(want) + np.abs(y) * 2.0 ** -59
        y = want
    if isinstance(out, tuple):
        _check_blocks(out, y, err=err)
    else:
        u = UBF if out.dtype == torch.bfloat16 else U32
        got = _f64(out).reshape(y.shape)
        assert (np.abs(got - y) <= err + u * (np.abs(y) + err)).all(), float(
            (np.abs(got - y) / (err + u * np.abs(y) + 1e-300)).max())


SHAPES = [(1, 1, 1), (1, 64, 128), (3, 17, 16), (5, 130, 129), (16, 128, 1000), (33, 300, 257),
          (64, 256, 384), (100, 1536, 512), (128, 128, 128), (129, 257, 640), (257, 130, 1187),
          (300, 520, 1536), (700, 900, 300), (1000, 64, 1536)]
OUTS = {"bf16": torch.bfloat16, "f32": torch.float32, "fp8": torch.float8_e4m3fn}


@pytest.mark.parametrize("out", list(OUTS))
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_linear(m, n, k, out):
    import vidax_b200 as vx
    x, w, bias = _operands(m, n, k, m + n + k)
    got = vx.linear_fp8(x, w, bias, out_dtype=OUTS[out])
    _ok()
    _check_linear(x, w, bias, False, got)


@pytest.mark.parametrize("out", list(OUTS))
@pytest.mark.parametrize("m,n,k", [(1, 256, 128), (20, 200, 300), (300, 520, 640)])
def test_linear_gelu(m, n, k, out):
    import vidax_b200 as vx
    x, w, bias = _operands(m, n, k, 3 * m + n + k)
    bias = bias * 20  # reach both flat ends of the activation
    got = vx.linear_fp8(x, w, bias, activation="gelu_tanh", out_dtype=OUTS[out])
    _ok()
    _check_linear(x, w, bias, True, got)


@pytest.mark.parametrize("variant", [1, 2, 3, 4])
def test_linear_gelu_far_from_zero(variant):
    """Pre-activations of any size (zero products, so each is its bias): the
    function goes to 0 below and to x above; a NaN stays in its column. At and
    below -7.5 the function's value is less than 7.5 * 2^-60, and what is
    computed there is that of -7.5: together below 2^-56."""
    import vidax_b200 as vx
    inf, nan = float("inf"), float("nan")
    b = torch.tensor([-7.4, -7.5, -8.0, -20.0, -1e4, -1e10, -1e19, -2e19, -1e20, -1e30, -3.4e38, -inf, 3.0,
                      nan, 1.0, 0.0, -0.5, nan, nan, 7.0, 40.0, 1e19, 1e20, 3.4e38, 1.5, inf, -1e25, 2.0])
    n = b.numel()
    x = vx.quantize_fp8(torch.zeros((3, 128), device="cuda"))
    w = vx.quantize_fp8(torch.zeros((n, 128), device="cuda"), 128)
    y = _f64(vx.linear_fp8(x, w, b.cuda(), activation="gelu_tanh", out_dtype=torch.float32, variant=variant))
    _ok()
    v = b.double().numpy()
    assert (np.isnan(y) == np.isnan(v)).all() and (y == y[:1])[:, ~np.isnan(v)].all()
    low = v <= -7.5
    assert (np.abs(y[:, low]) <= 2.0 ** -56).all()
    assert (y[:, v == inf] == inf).all()
    mid = ~low & np.isfinite(v)
    # 0.5 x (1 + tanh u) without the cancellation that leaves 0 of it at -7.4
    with np.errstate(over="ignore"):
        want = v[mid] / (1 + np.exp(-2 * np.sqrt(2 / np.pi) * (v[mid] + 0.044715 * v[mid] ** 3)))
    t = np.minimum(2.31 * np.abs(v[mid]) * (1 + 0.0448 * v[mid] ** 2), 61)
    assert (np.abs(y[:, mid] - want) <= (7 * U32 * t + 2.0 ** -19) * np.abs(want)).all()
    if variant < 3:
        # a large negative pre-activation does not set its block's scale
        c = torch.where(b < -7, b, 0.25).nan_to_num(0.25, 0.25, -3e38).cuda()
        q = vx.linear_fp8(x, w, c, activation="gelu_tanh", out_dtype=torch.float8_e4m3fn, variant=variant)
        _ok()
        _check_blocks(q, np.repeat(fp8_ref.gelu_tanh(_f64(c).clip(-30))[None], 3, 0), err=2.0 ** -20)


@pytest.mark.parametrize("variant", [1, 2, 3])
@pytest.mark.parametrize("m,n,k", [(1, 40, 100), (128, 64, 128), (300, 700, 1000), (2100, 1300, 512)])
def test_linear_every_variant(m, n, k, variant):
    """Each tile over one and several tiles per CTA, short and full edges."""
    import vidax_b200 as vx
    x, w, bias = _operands(m, n, k, 7 * m + n + k)
    for out in ("bf16", "f32") + (("fp8",) if variant < 3 else ()):
        got = vx.linear_fp8(x, w, bias, out_dtype=OUTS[out], variant=variant)
        _ok()
        _check_linear(x, w, bias, False, got)


@pytest.mark.parametrize("gelu", [False, True])
@pytest.mark.parametrize("out", list(OUTS))
@pytest.mark.parametrize("m", [1, 2, 8, 9, 15, 16])
@pytest.mark.parametrize("n,k", [(1, 1), (16, 17), (100, 130), (640, 128), (1000, 1187), (257, 4100)])
def test_linear_few_rows(m, n, k, out, gelu):
    """The form for a few rows over its token counts, short last blocks of
    features and of columns, and (n = 1000: 63 CTAs) a last cluster with CTAs
    that have no column."""
    import vidax_b200 as vx
    x, w, bias = _operands(m, n, k, m + 3 * n + k)
    got = vx.linear_fp8(x, w, bias, activation="gelu_tanh" if gelu else None, out_dtype=OUTS[out],
                        variant=4)
    _ok()
    _check_linear(x, w, bias, gelu, got)


def test_linear_padding_behind_the_features_is_not_read_as_values():
    """NaN codes in the storage behind each row's features."""
    import vidax_b200 as vx
    for m, v in ((5, 4), (5, 3), (200, 1)):
        x, w, bias = _operands(m, 70, 133, 40 + m)
        ref = vx.linear_fp8(x, w, bias, variant=v)
        for t in (x, w):
            full = torch.as_strided(t.data.view(torch.uint8), (t.data.shape[0] - 1, 144), (144, 1))
            full[:, 133:] = 0x7F
        assert torch.equal(vx.linear_fp8(x, w, bias, variant=v), ref)
    _ok()


def test_linear_no_bias_batched_and_any_layout():
    import vidax_b200 as vx
    x, w, _ = _operands(6 * 7, 96, 200, 5)
    ref = vx.linear_fp8(x, w)
    _check_linear(x, w, None, False, ref)
    xb = vx.Fp8Tensor(x.data.unflatten(0, (6, 7)), x.scale.unflatten(0, (6, 7)))
    assert torch.equal(vx.linear_fp8(xb, w), ref.view(6, 7, 96))
    # scales in rows, operands in unpadded and misaligned storage
    raw = torch.zeros(42 * 200 + 1, dtype=torch.uint8, device="cuda")[1:].view(42, 200)
    raw.copy_(x.data.view(torch.uint8))
    xo = vx.Fp8Tensor(raw.view(torch.float8_e4m3fn), x.scale.contiguous())
    wo = vx.Fp8Tensor(w.data.contiguous(), w.scale.t().contiguous().t())
    assert torch.equal(vx.linear_fp8(xo, wo), ref)
    # a slice of the features of a wider tensor, from a block boundary on
    y = vx.linear_fp8(vx.Fp8Tensor(x.data[:, 128:], x.scale[:, 1:]),
                      vx.Fp8Tensor(w.data[:, 128:], w.scale[:, 1:]), out_dtype=torch.float32)
    _ok()
    _check_linear(vx.Fp8Tensor(x.data[:, 128:], x.scale[:, 1:]),
                  vx.Fp8Tensor(w.data[:, 128:], w.scale[:, 1:]), None, False, y)
    assert vx.linear_fp8(vx.Fp8Tensor(x.data[:0], x.scale[:0]), w).shape == (0, 96)


def test_linear_extreme_values():
    """Full-range codes, zero rows, and a NaN that stays in its row."""
    import vidax_b200 as vx
    g = _gen(6)
    m, n, k = 140, 200, 256
    codes = torch.randint(0, 256, (m + n, k), generator=g, device="cuda", dtype=torch.uint8)
    codes[(codes & 127) == 127] = 1  # no NaN codes
    data = codes.view(torch.float8_e4m3fn)
    x = vx.Fp8Tensor(data[:m], torch.rand((m, 2), generator=g, device="cuda") * 1e-3)
    w = vx.Fp8Tensor(data[m:], torch.rand((2, 2), generator=g, device="cuda") * 1e3)
    for v in (0, 1, 3):
        _check_linear(x, w, None, False, vx.linear_fp8(x, w, out_dtype=torch.float32, variant=v))
    z = torch.zeros((130, k), device="cuda")
    z[7, 3] = float("nan")
    o = vx.linear_fp8(vx.quantize_fp8(z), w, out_dtype=torch.float32)
    _ok()
    assert torch.isnan(o[7]).all()
    o[7] = 0
    assert (o == 0).all()


def test_linear_writes_only_its_rows_and_columns():
    """Odd n: rows of the output are not 32-byte multiples and the buffer
    behind the last row stays as it was."""
    from vidax_b200 import fp8
    x, w, _ = _operands(70, 100, 160, 8)
    for odt, name in ((torch.bfloat16, "bf16"), (torch.float32, "f32"), (torch.uint8, "fp8")):
        buf = torch.full((80, 111), 99, dtype=odt, device="cuda")
        sc = torch.full((80, 1), -1.0, device="cuda")
        a = fp8.LinearFp8Args()
        a.x, a.w, a.x_scale, a.w_scale = (t.data_ptr() for t in (x.data, w.data, x.scale, w.scale))
        a.out, a.out_scale, a.out_stride = buf.data_ptr(), sc.data_ptr(), 111
        a.out_scale_stride[:] = (1, 1)
        a.x_stride, a.w_stride = x.data.stride(0), w.data.stride(0)
        a.x_scale_stride[:], a.w_scale_stride[:] = x.scale.stride(), w.scale.stride()
        a.m, a.n, a.k, a.out_type = 70, 100, 160, fp8._TYPES[OUTS[name]]
        _call("vx_linear_fp8", a)
        _ok()
        assert (buf[70:] == 99).all() and (buf[:70, 100:] == 99).all()
        got = buf[:70, :100]
        _check_linear(x, w, None, False, got if name != "fp8" else
                      fp8.Fp8Tensor(got.contiguous().view(torch.float8_e4m3fn), sc[:70]))
        assert name != "fp8" or (sc[70:] == -1).all()


@pytest.mark.parametrize("variant", [0, 1, 2, 3, 4])
@pytest.mark.parametrize("stride", [111, 112, 128])
@pytest.mark.parametrize("name", list(OUTS))
def test_linear_leaves_the_rest_of_a_padded_output(name, stride, variant):
    """Rows that lie on 16-byte boundaries but end between two, by every form:
    nothing behind a row's columns or behind the last row is written."""
    from vidax_b200 import fp8
    if variant == 3 and name == "fp8":
        pytest.skip("no such variant")
    for m, n in ((70, 100), (70, 99), (13, 97)) if variant != 4 else ((13, 100), (16, 97), (1, 99)):
        x, w, bias = _operands(m, n, 160, 80 + m + n)
        odt = OUTS[name]
        buf = torch.empty((m + 3, stride), dtype=odt, device="cuda")
        buf.view(torch.uint8).fill_(85)
        sc = torch.full((m + 3, 1), -1.0, device="cuda")
        a = fp8.LinearFp8Args()
        a.x, a.w, a.x_scale, a.w_scale = (t.data_ptr() for t in (x.data, w.data, x.scale, w.scale))
        a.bias, a.out, a.out_scale, a.out_stride = bias.data_ptr(), buf.data_ptr(), sc.data_ptr(), stride
        a.out_scale_stride[:] = (1, 1)
        a.x_stride, a.w_stride = x.data.stride(0), w.data.stride(0)
        a.x_scale_stride[:], a.w_scale_stride[:] = x.scale.stride(), w.scale.stride()
        a.m, a.n, a.k, a.out_type, a.variant = m, n, 160, fp8._TYPES[odt], variant
        _call("vx_linear_fp8", a)
        _ok()
        assert (buf[m:].view(torch.uint8) == 85).all() and (sc[m:] == -1).all()
        assert (buf[:, n:].contiguous().view(torch.uint8) == 85).all()
        got = buf[:m, :n]
        _check_linear(x, w, bias, False, got if name != "fp8" else
                      fp8.Fp8Tensor(got.contiguous(), sc[:m]))


def test_linear_repeats_bit_for_bit():
    import vidax_b200 as vx
    x, w, bias = _operands(900, 700, 1536, 9)
    ref = vx.linear_fp8(x, w, bias, out_dtype=torch.float32)
    for _ in range(5):
        assert torch.equal(vx.linear_fp8(x, w, bias, out_dtype=torch.float32), ref)


@pytest.mark.parametrize("variant", [1, 2, 3])
@pytest.mark.parametrize("k", [64, 200, 300, 640])
def test_linear_few_blocks_many_tiles(k, variant):
    """One to five blocks of features per tile and several tiles per CTA: the
    rings of stages, TMEM buffers and scale groups wrap inside and across tiles."""
    import vidax_b200 as vx
    x, w, bias = _operands(9000, 700, k, 60 + k)
    for out in ("f32",) + (("fp8",) if variant < 3 else ()):
        got = vx.linear_fp8(x, w, bias, out_dtype=OUTS[out], variant=variant)
        _ok()
        _check_linear(x, w, bias, False, got)


@pytest.mark.parametrize("variant,m,n,k", [(1, 4680, 1024, 1536), (2, 2000, 1024, 1300),
                                           (3, 1000, 1500, 1536), (4, 8, 4000, 1536)])
def test_linear_cold_operands(variant, m, n, k):
    """Operands that come from HBM: their loads land late and out of order.
    Three sets in turn, and a buffer larger than L2 written in between."""
    import vidax_b200 as vx
    flush = torch.empty(256 << 20, dtype=torch.uint8, device="cuda")
    sets = [_operands(m, n, k, 50 + i) for i in range(3)]
    refs = [vx.linear_fp8(*s, out_dtype=torch.float32, variant=variant) for s in sets]
    _check_linear(*sets[0], False, refs[0])
    same = []
    for i in range(60):
        flush.fill_(i)
        out = vx.linear_fp8(*sets[i % 3], out_dtype=torch.float32, variant=variant)
        same.append((out == refs[i % 3]).all())
    _ok()
    assert bool(torch.stack(same).all())


def test_offsets_past_32_bits():
    """Tensors of more than 2^31 elements: their last rows equal the same rows
    computed alone."""
    import vidax_b200 as vx
    rows, dim = 170000, 13000
    x = torch.empty((rows, dim), dtype=torch.bfloat16, device="cuda")
    x.normal_(generator=_gen(70))
    q = vx.quantize_fp8(x)
    ref = vx.quantize_fp8(x[-9:].clone())
    assert torch.equal(q.data[-9:].float(), ref.data.float()) and torch.equal(q.scale[-9:], ref.scale)
    del q
    gate = torch.full((1, dim), 0.5, device="cuda")
    o, total = vx.add_norm(x, x, gate, out_dtype=torch.float8_e4m3fn)
    oref, tref = vx.add_norm(x[-9:].clone(), x[-9:].clone(), gate, out_dtype=torch.float8_e4m3fn)
    assert torch.equal(o.data[-9:].float(), oref.data.float()) and torch.equal(o.scale[-9:], oref.scale)
    assert torch.equal(total[-9:], tref)
    del x, o, total
    m, k = 260000, 130
    g = _gen(71)
    a = vx.quantize_fp8(torch.randn((m, k), generator=g, device="cuda"))
    tail = vx.Fp8Tensor(a.data[-200:], a.scale[-200:])
    for n, out in ((8704, torch.bfloat16), (8703, torch.bfloat16), (8703, torch.float8_e4m3fn)):
        w = vx.quantize_fp8(torch.randn((n, k), generator=g, device="cuda"), 128)
        y = vx.linear_fp8(a, w, out_dtype=out)
        ref = vx.linear_fp8(tail, w, out_dtype=out)
        _ok()
        if out == torch.bfloat16:
            assert torch.equal(y[-200:], ref)
        else:
            assert torch.equal(y.data[-200:].float(), ref.data.float())
            assert torch.equal(y.scale[-200:], ref.scale)
        del y, ref


def test_sizes_past_32_bits_are_refused_by_every_operator():
    """Views of one element, so nothing of that size exists: an error with a
    message, before anything is allocated."""
    import vidax_b200 as vx
    many = 2 ** 31
    one = torch.zeros(1, device="cuda")
    codes = one.to(torch.float8_e4m3fn)
    w = vx.quantize_fp8(torch.zeros((4, 1), device="cuda"), 128)
    held = torch.cuda.memory_allocated()
    for shape in ((many, 1), (1, many), (2, many // 2, 1)):
        big = one.expand(shape)
        for call in (lambda: vx.quantize_fp8(big), lambda: vx.add_norm(big)):
            with pytest.raises(NotImplementedError, match="2\\^31 - 1"):
                call()
    x = vx.Fp8Tensor(codes.expand(many, 1), one.expand(many, 1))
    with pytest.raises(NotImplementedError, match="2\\^31 - 1"):
        vx.linear_fp8(x, w)
    x = vx.Fp8Tensor(codes.expand(1, many), one.expand(1, many // 128))
    with pytest.raises(NotImplementedError, match="2\\^31 - 1"):
        vx.linear_fp8(x, vx.Fp8Tensor(codes.expand(1, many), one.expand(1, many // 128)))
    assert torch.cuda.memory_allocated() == held
    for eps in (-1.0, 1e39, float("inf"), float("nan")):
        with pytest.raises(ValueError, match="eps"):
            vx.add_norm(torch.zeros((2, 8), device="cuda"), eps=eps)
    x = vx.quantize_fp8(torch.zeros((4, 1), device="cuda"))
    for variant in (-1, 5, 2 ** 40, None):
        with pytest.raises(ValueError, match="variant"):
            vx.linear_fp8(x, w, variant=variant)


# ------------------------------------------------------------------ together


def _layer(x, y, gate, p):
    import vidax_b200 as vx
    h8, total = vx.add_norm(x, y, gate, norm="layer", weight=p["nw"], bias=p["nb"],
                            out_dtype=torch.float8_e4m3fn)
    u8 = vx.linear_fp8(h8, p["w1"], p["b1"], activation="gelu_tanh", out_dtype=torch.float8_e4m3fn)
    return vx.linear_fp8(u8, p["w2"], p["b2"]), total


def _layer_params(dim, ffn, seed):
    import vidax_b200 as vx
    g = _gen(seed)

    def r(*s):
        return torch.randn(s, generator=g, device="cuda")

    return {"nw": 1 + 0.1 * r(dim), "nb": 0.1 * r(dim), "w1": vx.quantize_fp8(r(ffn, dim) * dim ** -0.5, 128),
            "b1": 0.1 * r(ffn), "w2": vx.quantize_fp8(r(dim, ffn) * ffn ** -0.5, 128), "b2": 0.1 * r(dim)}


def test_feed_forward_run():
    """Norm, up projection and down projection, each step checked on the
    inputs that the step before it gave."""
    import vidax_b200 as vx
    p = _layer_params(256, 640, 20)
    c = _norm_case(2, 75, 256, torch.float32, 21)
    h8, total = vx.add_norm(c["x"], c["y"], c["gate"], norm="layer", weight=p["nw"], bias=p["nb"],
                            out_dtype=torch.float8_e4m3fn)
    _check_norm({**c, "weight": p["nw"], "bias": p["nb"], "scale": None, "shift": None}, "layer",
                h8, total)
    u8 = vx.linear_fp8(h8, p["w1"], p["b1"], activation="gelu_tanh", out_dtype=torch.float8_e4m3fn)
    _check_linear(h8, p["w1"], p["b1"], True, u8)
    o = vx.linear_fp8(u8, p["w2"], p["b2"])
    _ok()
    _check_linear(u8, p["w2"], p["b2"], False, o)
    o2, t2 = _layer(c["x"], c["y"], c["gate"], p)
    assert torch.equal(o2, o) and torch.equal(t2, total)


def test_feed_forward_on_streams_and_in_graphs():
    """Two streams at once, and a captured graph replayed on new inputs, give
    the eager results: the calls share no workspace."""
    p = _layer_params(384, 896, 22)
    cs = [_norm_case(1, 300 + 50 * i, 384, torch.float32, 30 + i) for i in range(2)]
    refs = [_layer(c["x"], c["y"], c["gate"], p)[0] for c in cs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cs]
    outs = [[], []]
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                outs[i].append(_layer(cs[i]["x"], cs[i]["y"], cs[i]["gate"], p)[0])
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(o, refs[i]) for o in outs[i])
    g = torch.cuda.CUDAGraph()
    x, y = cs[0]["x"].clone(), cs[0]["y"].clone()
    _layer(x, y, cs[0]["gate"], p)
    torch.cuda.synchronize()
    with torch.cuda.graph(g):
        o, _ = _layer(x, y, cs[0]["gate"], p)
    new = _norm_case(1, 300, 384, torch.float32, 33)
    x.copy_(new["x"])
    y.copy_(new["y"])
    g.replay()
    ref = _layer(new["x"], new["y"], cs[0]["gate"], p)[0]
    _ok()
    assert torch.equal(o, ref)


def test_single_token_run_in_a_graph():
    """One token through norm, up and down projection (the forms for few rows,
    the e4m3 one a cluster launch), captured and replayed."""
    p = _layer_params(1536, 2048, 23)
    c = _norm_case(1, 1, 1536, torch.float32, 34)
    _layer(c["x"], c["y"], c["gate"], p)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    x = c["x"].clone()
    with torch.cuda.graph(g):
        o, _ = _layer(x, c["y"], c["gate"], p)
    new = _norm_case(1, 1, 1536, torch.float32, 35)
    x.copy_(new["x"])
    g.replay()
    ref, _ = _layer(new["x"], c["y"], c["gate"], p)
    _ok()
    assert torch.equal(o, ref)


@pytest.mark.skipif(torch.cuda.device_count() < 2, reason="needs 2 GPUs")
def test_on_another_device_than_the_current_one():
    p = _layer_params(256, 384, 24)
    c = _norm_case(1, 40, 256, torch.float32, 36)
    ref, _ = _layer(c["x"], c["y"], c["gate"], p)
    import vidax_b200 as vx
    there = {k: vx.Fp8Tensor(*(t.to("cuda:1") for t in v)) if isinstance(v, tuple) else v.to("cuda:1")
             for k, v in p.items()}
    o, _ = _layer(*(c[k].to("cuda:1") for k in ("x", "y", "gate")), there)
    torch.cuda.synchronize(1)
    assert torch.equal(o.cpu(), ref.cpu())
