"""The DiT step with 8-bit linear layers (wan_dit.quantize_params) against the
same steps in plain float32 torch, and against the bf16 model.

Tolerances. Against the plain steps on the same quantised values: the sums
differ in their order only, and what rounds to bf16 or e4m3 on the way differs
where a value lies within float32 rounding of a tie, as in the bf16 driver's
own comparison with the oracle: relative L2 2e-2. Against the bf16 model: a
value's e4m3 rounding is off by up to 2^-4, uniformly, so 2^-4 / sqrt(3) =
3.6 % in the root mean square at worst over a binade; a linear layer rounds
its input and its weights (independent: sqrt(2) of that, 5.1 %), a branch of
the block has at most two layers in a row after its norm (7.2 %), and the
branches add to a residual stream that is not rounded. The head's linear map
of the stream keeps that relative error: relative L2 <= 0.11 with half as much
again for the attention weights, which see the errors of q and k."""
import numpy as np
import pytest
import torch

from test_wan_dit_gpu import _inputs, _rel, _tiny

pytestmark = pytest.mark.gpu


def _plain_quantize(x, block_rows=1):
    from vidax_b200 import Fp8Tensor
    rows, k = x.reshape(-1, x.shape[-1]).shape
    v = x.reshape(rows, k).float()
    p = torch.nn.functional.pad(v, (0, -k % 128, 0, -rows % block_rows))
    p = p.view(p.shape[0] // block_rows, block_rows, -1, 128)
    a = p.abs().amax((1, 3), keepdim=True).clamp_min(2.0 ** -100)
    q = (p * (torch.full_like(a, 448.0) / a)).to(torch.float8_e4m3fn)
    q = q.reshape(p.shape[0] * block_rows, -1)[:rows, :k]
    s = (a / 448).reshape(p.shape[0], -1)
    if block_rows == 1:
        s = s.reshape(*x.shape[:-1], -1)
    return Fp8Tensor(q.reshape(x.shape), s)


def _plain_add_norm(x, y=None, gate=None, *, norm="rms", weight=None, bias=None, scale=None,
                    shift=None, eps=1e-6, out_dtype=torch.bfloat16, residual_out=None):
    def rows(t):
        return t.reshape(x.shape[0], 1, x.shape[-1])
    h = x
    if y is not None:
        h = x + (y.float() if gate is None else y.float() * rows(gate))
        residual_out.copy_(h)
        h = residual_out
    n = h - h.mean(-1, keepdim=True) if norm == "layer" else h
    n = n / torch.sqrt((n * n).mean(-1, keepdim=True) + eps)
    n = n if weight is None else n * weight
    n = n if bias is None else n + bias
    n = n if scale is None else n * (1 + rows(scale)) + rows(shift)
    return (_plain_quantize(n) if out_dtype == torch.float8_e4m3fn else n.to(out_dtype)), h


def _plain_linear(x, w, bias=None, *, activation=None, out_dtype=torch.bfloat16):
    y = x.dequantize() @ w.dequantize().t()
    y = y if bias is None else y + bias
    if activation:
        y = torch.nn.functional.gelu(y, approximate="tanh")
    return _plain_quantize(y) if out_dtype == torch.float8_e4m3fn else y.to(out_dtype)


def _run(p, cfg, seed, batch):
    from vidax_b200 import _lib
    from vidax_b200.wan_dit import wan_dit_forward
    latents, context, t = _inputs(cfg, seed, batch)
    out = wan_dit_forward(p, cfg, torch.from_numpy(latents).cuda(), torch.from_numpy(t).cuda(),
                          torch.from_numpy(context).cuda())
    torch.cuda.synchronize()
    assert _lib.device_status() == 0
    return out.float().cpu().numpy()


@pytest.mark.parametrize("head_dim,batch", [(128, 1), (64, 1), (128, 2)])
def test_wan_dit_fp8_matches_plain_steps(head_dim, batch, monkeypatch):
    from vidax_b200 import wan_dit
    cfg = _tiny(head_dim)
    p = wan_dit.init_params(cfg, "cuda", seed=3)
    q = wan_dit.quantize_params(p, cfg)
    assert "blocks_0.self_attn_q_w" not in q and q["blocks_0.norm3_w"] is p["blocks_0.norm3_w"]
    assert q["blocks_1.self_attn_norm_q"] is p["blocks_1.self_attn_norm_q"]
    got = _run(q, cfg, 5, batch)
    assert got.shape == (batch, 2, 8, 16, cfg.out_dim) and np.isfinite(got).all()
    bf16 = _run(p, cfg, 5, batch)
    monkeypatch.setattr(wan_dit, "quantize_fp8", _plain_quantize)
    monkeypatch.setattr(wan_dit, "add_norm", _plain_add_norm)
    monkeypatch.setattr(wan_dit, "linear_fp8", _plain_linear)
    plain = _run(q, cfg, 5, batch)
    assert _rel(got, plain) <= 2e-2, _rel(got, plain)
    assert _rel(got, bf16) <= 0.11, _rel(got, bf16)


def test_wan_dit_fp8_replays_in_a_graph():
    """The block stack of the step, captured and replayed on another input."""
    from vidax_b200 import quantize_fp8, wan_dit
    cfg = _tiny(128)
    q = wan_dit.quantize_params(wan_dit.init_params(cfg, "cuda", seed=4), cfg)
    g = torch.Generator(device="cuda").manual_seed(1)

    def r(*s):
        return torch.randn(s, generator=g, device="cuda")

    L = 200
    rope = wan_dit.rope3d_freqs(2, 10, 10, 128, device="cuda")
    ctx = quantize_fp8(r(1, 16, cfg.dim))
    t_mod = 0.1 * r(1, 6, cfg.dim)

    def blocks(x):
        pending = (None, None)
        for i in range(cfg.num_layers):
            x, pending = wan_dit._block_forward_fp8(q, i, cfg, x, pending, ctx, t_mod, rope)
        return wan_dit.gated_residual_(x, *pending)

    x0, x1 = r(1, L, cfg.dim), r(1, L, cfg.dim)
    ref = blocks(x1.clone())
    buf = x0.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        blocks(buf)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = blocks(buf)
    for _ in range(2):
        buf.copy_(x1)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, ref)


@pytest.mark.parametrize("head_dim,batch,P", [(128, 1, 2), (64, 2, 2), (64, 1, 4)])
def test_wan_dit_fp8_sequence_parallel(head_dim, batch, P, monkeypatch):
    """Every rank's token chunk through the 8-bit blocks, the ranks emulated as
    threads: equal to the single-GPU step but for the order of sums (2e-2 as
    above; a row is normalised and quantised by itself on either side)."""
    import vidax_b200 as vx
    from emulated_ranks import RankGroup, run_ranks
    from vidax_b200 import _lib, ulysses, wan_dit
    cfg = _tiny(head_dim)
    q = wan_dit.quantize_params(wan_dit.init_params(cfg, "cuda", seed=3), cfg)
    single = _run(q, cfg, 5, batch)
    lat, ctx, t = (torch.from_numpy(x).cuda() for x in _inputs(cfg, 5, batch))
    fake = RankGroup(P)
    monkeypatch.setattr(ulysses, "dist", fake)
    monkeypatch.setattr(wan_dit, "dist", fake)
    vx.register_axis("sp_fp8", None)
    try:
        outs = run_ranks(P, fake, lambda r: wan_dit.wan_dit_forward(
            q, cfg, lat, t, ctx, sp_axis_name="sp_fp8").float().cpu().numpy())
    finally:
        vx.unregister_axis("sp_fp8")
    assert _lib.device_status() == 0
    for o in outs:
        assert o.shape == single.shape and _rel(o, single) <= 2e-2, _rel(o, single)
