"""The 8-bit operators without a GPU: the oracle's e4m3 against torch's, and
every refusal, in Python and at the C ABI (which checks its arguments before
it touches a device)."""
import ctypes

import numpy as np
import pytest
import torch

from oracle import fp8_ref


def test_oracle_e4m3_is_the_format():
    codes = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double().numpy()
    v = codes[np.isfinite(codes)]
    assert np.array_equal(fp8_ref.e4m3(v), v)
    x = np.concatenate([np.random.default_rng(0).standard_normal(20000) * 60,
                        np.linspace(-0.05, 0.05, 4001), (v[:-1] + v[1:]) / 2])
    x = x[np.abs(x) <= 448]
    ref = torch.from_numpy(x.astype(np.float32)).to(torch.float8_e4m3fn).double().numpy()
    assert np.array_equal(fp8_ref.e4m3(x.astype(np.float32)), ref)


def test_oracle_quantize_round_trip():
    x = np.random.default_rng(1).standard_normal((5, 300))
    for r in (1, 128):
        q, s = fp8_ref.quantize(x, r)
        back = q * fp8_ref.expand(s, r, 5, 300)
        assert (np.abs(back - x) <= 2.0 ** -4 * np.abs(x) + 2.0 ** -10 * s.max()).all()


def test_fp8_tensor_dequantize():
    from vidax_b200 import Fp8Tensor
    d = torch.ones((130, 200)).to(torch.float8_e4m3fn)
    row = Fp8Tensor(d, torch.arange(260, dtype=torch.float32).view(130, 2)).dequantize()
    assert row[3, 5] == 6 and row[3, 199] == 7
    blk = Fp8Tensor(d, torch.arange(4, dtype=torch.float32).view(2, 2)).dequantize()
    assert blk[127, 127] == 0 and blk[127, 128] == 1 and blk[128, 0] == 2 and blk[129, 199] == 3


def test_row_strides():
    from vidax_b200.fp8 import _empty_fp8, _row_stride
    t = torch.zeros((3, 4, 32))
    assert _row_stride(t) == 32 and _row_stride(t[..., :20]) == 32 and _row_stride(t[:, 1:2]) == 128
    assert _row_stride(t[:, :3]) is None          # a gap between batch items
    assert _row_stride(t.transpose(0, 1)) is None
    assert _row_stride(t[..., ::2]) is None
    assert _row_stride(torch.zeros((1, 32)).expand(4, 32)) is None  # rows that lie on one another
    assert _row_stride(t[0, 0]) == 32
    q, ld, ls = _empty_fp8((2, 5, 130), "cpu")
    assert (ld, ls) == (144, 12)
    assert q.data.shape == (2, 5, 130) and _row_stride(q.data) == 144
    assert q.scale.shape == (2, 5, 2) and q.scale.flatten(0, 1).stride() == (1, 12)


def test_python_refusals():
    import vidax_b200 as vx
    f32, bf = torch.zeros((4, 8)), torch.zeros((4, 8), dtype=torch.bfloat16)
    with pytest.raises(TypeError):
        vx.quantize_fp8([1.0])
    with pytest.raises(NotImplementedError):
        vx.quantize_fp8(f32.half())
    with pytest.raises(ValueError, match="CUDA"):
        vx.quantize_fp8(f32)
    with pytest.raises(ValueError, match="CUDA"):
        vx.add_norm(f32, bf)
    with pytest.raises(NotImplementedError):
        vx.add_norm(f32.double())
    q = vx.Fp8Tensor(f32.to(torch.float8_e4m3fn), torch.ones((4, 1)))
    with pytest.raises(TypeError):
        vx.linear_fp8(f32, q)
    with pytest.raises(NotImplementedError):
        vx.linear_fp8(vx.Fp8Tensor(f32, q.scale), q)
    with pytest.raises(ValueError, match="CUDA"):
        vx.linear_fp8(q, q)


def test_packed_arguments_are_the_structs():
    """The layouts that the entry points pack their arguments in."""
    from vidax_b200 import fp8
    for name, cls in (("vx_quantize_fp8", fp8.QuantizeFp8Args), ("vx_add_norm", fp8.AddNormArgs),
                      ("vx_linear_fp8", fp8.LinearFp8Args)):
        flat, values = [], []
        for n, t in cls._fields_:
            flat += [(n, i) for i in range(t._length_)] if hasattr(t, "_length_") else [(n, None)]
        values = list(range(1, len(flat) + 1))
        raw = fp8._PACKED[name].pack(*values)
        assert len(raw) == ctypes.sizeof(cls)
        a = cls.from_buffer_copy(raw)
        assert [getattr(a, n) if i is None else getattr(a, n)[i] for n, i in flat] == values


def _args(cls, **kw):
    a = cls()
    for k, v in kw.items():
        if isinstance(v, tuple):
            getattr(a, k)[:] = v
        else:
            setattr(a, k, v)
    return a


P = 1 << 20  # an aligned address that no refused call reads


def _rc(name, a):
    from vidax_b200 import _lib, fp8
    rc = fp8._entry(name, a)(ctypes.byref(a), None)
    return rc, _lib.load().vx_last_error().decode()


QOK = dict(src=P, dst=P, scale=P, src_stride=200, dst_stride=208, scale_stride=(1, 4), rows=4, dim=200,
           src_type=1, block_rows=1)


@pytest.mark.parametrize("change,code", [
    (dict(rows=-1), 1), (dict(dim=0), 1), (dict(src_type=2), 2), (dict(src_type=7), 2),
    (dict(block_rows=64), 2), (dict(src=None), 1), (dict(dst=None), 1), (dict(scale=None), 1),
    (dict(src=P + 1), 1), (dict(scale=P + 2), 1), (dict(src_stride=199), 1), (dict(dst_stride=-8), 1),
    (dict(scale_stride=(-1, 1)), 1), (dict(rows=1 << 40, src_stride=200), 2)])
def test_quantize_c_refusals(change, code):
    from vidax_b200 import fp8
    rc, msg = _rc("vx_quantize_fp8", _args(fp8.QuantizeFp8Args, **{**QOK, **change}))
    assert rc == code and msg


NOK = dict(x=P, y=P, sum=P, out=P, out_scale=P, x_stride=96, y_stride=96, sum_stride=96, out_stride=96,
           out_scale_stride=(1, 4), rows=4, rows_per_batch=2, dim=96, x_type=0, out_type=2, norm=0,
           eps=1e-6)


@pytest.mark.parametrize("change,code", [
    (dict(rows=-2), 1), (dict(dim=0), 1), (dict(rows_per_batch=0), 1), (dict(rows_per_batch=3), 1),
    (dict(x_type=2), 2), (dict(out_type=0), 2), (dict(norm=2), 2), (dict(eps=-1.0), 1),
    (dict(eps=float("nan")), 1), (dict(y=None, gate=P), 1), (dict(x=None), 1), (dict(sum=None), 1),
    (dict(out=None), 1), (dict(out_scale=None), 1), (dict(x_stride=95), 1), (dict(y=P + 1), 1),
    (dict(weight=P + 2), 1), (dict(gate=P, gate_stride=-1), 1)])
def test_add_norm_c_refusals(change, code):
    from vidax_b200 import fp8
    rc, msg = _rc("vx_add_norm", _args(fp8.AddNormArgs, **{**NOK, **change}))
    assert rc == code and msg


LOK = dict(x=P, x_scale=P, w=P, w_scale=P, out=P, out_scale=P, x_stride=96, w_stride=96, out_stride=64,
           x_scale_stride=(1, 4), w_scale_stride=(1, 1), out_scale_stride=(1, 4), m=4, n=64, k=96,
           out_type=1)


@pytest.mark.parametrize("change,code", [
    (dict(m=-1), 1), (dict(n=0), 1), (dict(k=0), 1), (dict(out_type=3), 2), (dict(activation=2), 2),
    (dict(variant=-1), 1), (dict(variant=99), 1),
    (dict(variant=4, m=17), 2), (dict(variant=3, out_type=2), 2), (dict(x=None), 1), (dict(w=None), 1),
    (dict(out=None), 1), (dict(x_scale=None), 1), (dict(w_scale=None), 1),
    (dict(out_type=2, out_scale=None), 1), (dict(x=P + 8), 1), (dict(w_stride=100), 1),
    (dict(x_stride=80), 1), (dict(out_stride=63), 1), (dict(bias=P + 1), 1),
    (dict(w_scale_stride=(1, -1)), 1)])
def test_linear_c_refusals(change, code):
    from vidax_b200 import fp8
    rc, msg = _rc("vx_linear_fp8", _args(fp8.LinearFp8Args, **{**LOK, **change}))
    assert rc == code and msg


def test_c_null_and_empty_calls():
    from vidax_b200 import _lib, fp8
    lib = _lib.load()
    for name in ("vx_quantize_fp8", "vx_add_norm", "vx_linear_fp8"):
        assert getattr(lib, name)(None, None) == _lib.VX_EINVAL
    assert _rc("vx_quantize_fp8", _args(fp8.QuantizeFp8Args, **{**QOK, "rows": 0}))[0] == 0
    assert _rc("vx_add_norm", _args(fp8.AddNormArgs, **{**NOK, "rows": 0}))[0] == 0
    assert _rc("vx_linear_fp8", _args(fp8.LinearFp8Args, **{**LOK, "m": 0}))[0] == 0


@pytest.mark.parametrize("change,call,code", [
    ({}, (-1, 0, 1000), 1), ({}, (4, 0, 1000), 1), ({}, (1, -1, 1000), 1), ({}, (1, 0, 0), 1),
    ({}, (1, 0, 1 << 33), 1), (dict(variant=1), (1, 0, 1000), 2), (dict(out_type=0), (1, 0, 1000), 2),
    (dict(m=-1), (1, 0, 1000), 1), (dict(x=None), (1, 0, 1000), 1)])
def test_linear_selftest_refusals(change, call, code):
    from vidax_b200 import _lib, fp8
    fn = _lib.load().vx_selftest_linear_fp8
    a = _args(fp8.LinearFp8Args, **{**LOK, **change})
    role, after, limit = call
    assert fn(ctypes.byref(a), role, after, ctypes.c_int64(limit), None) == code
    assert fn(None, 1, 0, ctypes.c_int64(1000), None) == 1


# add_norm: sum at S, 4 rows of 96 floats (384 bytes), 512 bytes apart
S = P + (1 << 16)
IN_PLACE = dict(x=S, sum=S, x_stride=128, sum_stride=128, y=P, y_stride=96, out=P + (1 << 18), out_stride=96)


@pytest.mark.parametrize("change", [
    dict(y=S), dict(y=S + 512, y_stride=256),            # y under the stream, a row further on
    dict(y=S - 2), dict(y=S - 3 * 192 + 2, y_stride=96), # its last bytes in the first row
    dict(y=S + 380, y_stride=256),                       # the end of a row, then the gap
    dict(y=S + 512 - 190, y_stride=256),                 # the gap, then the next row's start
    dict(sum=S + 512), dict(sum=S - 512), dict(sum=S + 4), dict(sum=S, sum_stride=96),
    dict(gate=S + 64, gate_stride=0), dict(scale=S + 1000, scale_stride=96),
    dict(shift=S - 384 - 512, shift_stride=224), dict(weight=S + 3 * 512 + 380), dict(bias=S - 380),
    dict(out=S), dict(out=S + 100, out_stride=512), dict(out=P + 96, out_type=1),
    dict(weight=P + (1 << 18) + 4), dict(x_type=1, y=S + 64, y_stride=128)])
def test_add_norm_c_refuses_overlaps(change):
    """Written memory that is read for other rows, in place and not: found from
    the addresses alone, before anything is launched."""
    from vidax_b200 import fp8
    rc, msg = _rc("vx_add_norm", _args(fp8.AddNormArgs, **{**NOK, **IN_PLACE, **change}))
    assert rc == 1 and "apart" in msg


@pytest.mark.parametrize("change", [
    {}, dict(y=S + 384, y_stride=256, dim=32, out_stride=96),      # y in the gaps between the rows
    dict(y=S + 3 * 512 + 384), dict(y=S - 3 * 192 - 192),          # right behind, right before
    dict(sum=S + 4 * 512), dict(gate=S + 384, gate_stride=128, dim=32), dict(weight=S + 3 * 512 + 384),
    dict(out=S + 384, out_stride=512), dict(x_type=1, y=S, y_stride=128),
    dict(x=P + (1 << 17))])
def test_add_norm_c_takes_memory_apart(change):
    """Side by side, interleaved, in place: past the checks of the addresses,
    to the next one, of the scales (so that nothing is launched)."""
    from vidax_b200 import fp8
    rc, msg = _rc("vx_add_norm", _args(fp8.AddNormArgs, **{**NOK, **IN_PLACE, "out_scale": None, **change}))
    assert rc == 1 and "out_scale" in msg


def test_add_norm_c_overlap_is_byte_for_byte():
    """Random rows against the sets of bytes they are."""
    import random
    from vidax_b200 import fp8
    rng = random.Random(7)
    seen = [0, 0]
    for _ in range(1500):
        rows, dim = rng.randint(1, 5), rng.randint(1, 6)
        ss, ys = dim + rng.randint(0, 30), dim + rng.choice([0, rng.randint(0, 60), dim * 3])
        if rng.random() < 0.3:
            ys = 2 * ss
        y = S + 2 * rng.randint(-60, 140)
        a = _args(fp8.AddNormArgs, **{**NOK, "x": S, "sum": S, "x_stride": ss, "sum_stride": ss, "y": y,
                                      "y_stride": ys, "out": P + (1 << 19), "out_stride": dim, "rows": rows,
                                      "rows_per_batch": rows, "dim": dim, "out_scale": None})
        sum_bytes = {S + r * ss * 4 + i for r in range(rows) for i in range(4 * dim)}
        meets = any(y + r * ys * 2 + i in sum_bytes for r in range(rows) for i in range(2 * dim))
        rc, msg = _rc("vx_add_norm", a)
        assert rc == 1 and ("apart" in msg) == meets, (rows, dim, ss, ys, y - S)
        seen[meets] += 1
    assert min(seen) > 200


def test_sizes_past_32_bits_are_refused():
    from vidax_b200.fp8 import _FLT_MAX, _check_sizes
    _check_sizes(2 ** 31 - 1, 2 ** 31 - 4096)
    for sizes in ((2 ** 31, 1), (1, 2 ** 31), (1, 1, 2 ** 31), (1, 2 ** 31 - 4095)):
        with pytest.raises(NotImplementedError, match="2\\^31 - 1"):
            _check_sizes(*sizes)
    assert _FLT_MAX == float(np.finfo(np.float32).max)


@pytest.mark.parametrize("most", [2 ** 31 - 1, 2 ** 31 - 256, 2 ** 31 - 2000])
def test_features_whose_indices_would_overflow_are_refused(most):
    """The kernels step past a row's end by up to 2048 features in 32 bits; one
    that wrapped would read at a negative offset. Refused before a launch."""
    from vidax_b200 import fp8
    far = dict(x_stride=2 ** 31, out_stride=2 ** 31, y=None, sum=None)
    for rows in (1, 4):
        rc, msg = _rc("vx_add_norm", _args(fp8.AddNormArgs, **{**NOK, **far, "rows": rows, "rows_per_batch": 1,
                                                              "dim": most}))
        assert rc == 2 and "features" in msg
    for change in (dict(n=most, out_stride=2 ** 31), dict(k=most, x_stride=2 ** 31, w_stride=2 ** 31)):
        rc, msg = _rc("vx_linear_fp8", _args(fp8.LinearFp8Args, **{**LOK, **change}))
        assert rc == 2 and "features" in msg
