"""Failure detection without a GPU fault: a bounded device-side wait that can
never complete gives up, records its code in the device status word, and the
context stays usable for the next kernel."""
import pytest
import torch

from oracle.attention_ref import compare, sdpa, seeded_qkv


@pytest.mark.gpu
def test_bounded_wait_times_out_and_context_survives():
    import vidax_b200 as vx
    from vidax_b200 import _lib
    _lib.device_status(clear=True)
    status = _lib.selftest_wait_timeout(2_000_000)   # ~1 ms of SM cycles
    assert status & 16
    assert _lib.device_status(clear=True) & 16        # visible to the host, then cleared
    assert _lib.device_status(clear=False) == 0
    q, k, v = seeded_qkv((1, 256, 2, 128), 5)
    t = [torch.from_numpy(x).cuda().bfloat16() for x in (q, k, v)]
    out = vx.flash_attention(*t, 128 ** -0.5)
    torch.cuda.synchronize()
    assert _lib.device_status() == 0
    mx, mean = compare(out.float().cpu().numpy(), sdpa(q, k, v))
    assert mx <= 2e-2 and mean <= 2e-3


@pytest.mark.gpu
@pytest.mark.parametrize("after", [0, 3, 16])
@pytest.mark.parametrize("role", [1, 2, 3])
@pytest.mark.parametrize("out", ["bf16", "fp8"])
def test_linear_fp8_waits_give_up(out, role, after):
    """A role of the 8-bit product that falls silent (loads, scales, an adding
    warp), at once or in mid-stream, several tiles per CTA: waits run out, the kernel ends with a code in the status word,
    and the next product is right."""
    import ctypes
    from vidax_b200 import _lib, fp8
    m, n, k = 4000, 1312, 1000      # 192 (672) tiles of 256 (64) columns, eight blocks each
    g = torch.Generator(device="cuda").manual_seed(5)
    x = fp8.quantize_fp8(torch.randn((m, k), generator=g, device="cuda"))
    w = fp8.quantize_fp8(torch.randn((n, k), generator=g, device="cuda"), 128)
    odt = torch.bfloat16 if out == "bf16" else torch.float8_e4m3fn
    variant = 3 if out == "bf16" else 1
    want = fp8.linear_fp8(x, w, out_dtype=odt, variant=variant)
    buf = torch.empty((m + 1, 1328), dtype=odt, device="cuda").view(torch.uint8).fill_(85).view(odt)
    sc = torch.full((m + 1, 11), -1.0, device="cuda")
    a = fp8.LinearFp8Args()
    a.x, a.w, a.x_scale, a.w_scale = (t.data_ptr() for t in (x.data, w.data, x.scale, w.scale))
    a.out, a.out_scale, a.out_stride = buf.data_ptr(), sc.data_ptr(), 1328
    a.out_scale_stride[:] = (11, 1)
    a.x_stride, a.w_stride = x.data.stride(0), w.data.stride(0)
    a.x_scale_stride[:], a.w_scale_stride[:] = x.scale.stride(), w.scale.stride()
    a.m, a.n, a.k, a.out_type = m, n, k, fp8._TYPES[odt]
    fn = _lib.load().vx_selftest_linear_fp8
    stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)

    def run(role):
        _lib.check(fn(ctypes.byref(a), role, after, ctypes.c_int64(2_000_000), stream))  # ~1 ms
        return _lib.device_status(clear=True)

    def got():
        return (buf[:m, :n].float(), sc[:m]) if out == "fp8" else (buf[:m, :n].float(),)

    assert _lib.device_status(clear=True) == 0
    # scales and adding warps count a tile's eight blocks, the others a CTA's
    # (two tiles of 256 columns, five of 64)
    expires = after < (8 if role >= 2 else 16 if out == "fp8" else 40)
    status = run(role)
    assert bool(status & 7) == expires and status & ~7 == 0
    # nothing behind the output's rows and columns, whatever was computed
    assert (buf[m:].view(torch.uint8) == 85).all() and (sc[m:] == -1).all()
    assert (buf[:m, n:].contiguous().view(torch.uint8) == 85).all()
    # and the same kernel, and the ordinary one, are right afterwards
    assert run(0) == 0
    ref = want if out == "fp8" else (want,)
    assert all(torch.equal(b, r.float()) for b, r in zip(got(), ref))
    again = fp8.linear_fp8(x, w, out_dtype=odt, variant=variant)
    assert _lib.device_status() == 0
    assert all(torch.equal(b.float(), r.float())
               for b, r in zip(again if out == "fp8" else (again,), ref))
