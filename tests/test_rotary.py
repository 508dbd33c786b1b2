"""Rotary positions: refusals on the CPU, numerics and gradients on a B200 against 64-bit sums."""
import ctypes

import pytest
import torch
from torch.autograd import forward_ad as fwAD

from ascend_rsfa import _capi
from ascend_rsfa import flash_attention_forward as fa
from ascend_rsfa import rotary as ro
from oracle import operators_ref as ref

lib = _capi.load()
HALF_STEP = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}     # half a step of the smallest numbers


def close(got, x, table, want, dtype, positions=None, interleaved=False, inverse=False):
    """One rounding to 16 bits, and two products and a sum in 32 bits with table entries that are rounded to 32
    bits: four roundings of 2^-24 of |a| c + |b| s at most, allowed as 2^-22 of (|a| + |b|) times the table's size."""
    ones = torch.ones_like(table)                        # turned by these, (|a|, |b|) gives |a| + |b| one way round
    size = torch.maximum(*(ref.rotary(x.abs(), ones, positions, interleaved, way) for way in (False, True)))
    bound = HALF_STEP[dtype] * want.abs() + 2.0 ** -22 * table.abs().max().double() * size + TINY[dtype]
    err = (got.double() - want).abs()
    assert bool((err <= bound).all()), float((err - bound).max())


# ------------------------------------------------------------------ without a GPU

def test_scaled_frequencies_of_the_oracle():
    f = ref.frequencies(64)
    assert f[0] == 1.0 and abs(float(f[1]) - 10000 ** (-2 / 64)) < 1e-15
    assert torch.allclose(ref.frequencies(64, scaling="linear", factor=4.0), f / 4)
    for scaling in ("yarn", "bands"):
        g = ref.frequencies(64, scaling=scaling, factor=8.0, original_length=4096)
        assert g[0] == f[0] and torch.isclose(g[-1], f[-1] / 8) and bool((g <= f).all()) and bool((g >= f / 8 * (1 - 1e-12)).all())
    # the lowest frequency of ntk scaling is the linear one
    assert torch.isclose(ref.frequencies(64, scaling="ntk", factor=8.0)[-1], f[-1] / 8)


def test_refusals_need_no_device():
    q = torch.zeros(1, 2, 4, 64, dtype=torch.float16)
    table = torch.zeros(8, 32, 2)
    with pytest.raises(RuntimeError, match="no CPU path"):
        ro.rotary(q, q, table)
    with pytest.raises(RuntimeError, match="no CPU path"):
        ro.rotary_table(8, 64, device="cpu")
    for bad in (dict(scaling="other"), dict(length=0), dict(dim=63), dict(dim=258), dict(dim=0)):
        with pytest.raises(ValueError):
            ro.rotary_table(**{**dict(length=8, dim=64, device="cuda"), **bad})
    with pytest.raises(ValueError, match="share B, S and D"):
        ro.rotary(q, q[:, :, :2], table)
    with pytest.raises(ValueError, match="D must be"):
        ro.rotary(q[..., :48], None, table)


def test_c_refusals_need_no_device():
    bad = _capi.RSFA_ERR_INVALID_ARGUMENT
    p, st = ctypes.c_void_p(4096), (ctypes.c_int64 * 16)(*([4 * 64 * 2, 4 * 64, 64, 1] * 4))

    def call(q=p, k=p, qo=p, ko=p, B=1, Hq=2, Hk=2, S=4, D=64, strides=st, table=p, length=8, dim=64, pos=None, p64=0, ps=None, dtype=0):
        return lib.rsfa_rotary(q, k, qo, ko, B, Hq, Hk, S, D, strides, table, length, dim, pos, p64, ps, 0, 0, dtype, None)

    for kw in (dict(q=None), dict(k=None), dict(qo=None), dict(Hk=0), dict(table=None), dict(strides=None), dict(B=0), dict(S=0),
               dict(D=48), dict(dim=66), dict(dim=63), dict(dim=0), dict(length=0), dict(dtype=7), dict(q=ctypes.c_void_p(4100)),
               dict(pos=p), dict(strides=(ctypes.c_int64 * 16)(*([512, 256, 60, 1] * 4))),
               dict(strides=(ctypes.c_int64 * 16)(*([512, 256, 64, 2] * 4)))):
        assert call(**kw) == bad, kw
    assert call(B=1 << 20, S=1 << 20) == _capi.RSFA_ERR_TOO_LARGE
    t = lib.rsfa_rotary_table
    for args in ((None, 8, 64, 1e4, 0, 1.0, 0, 0.0, 0.0, 1.0), (p, 0, 64, 1e4, 0, 1.0, 0, 0.0, 0.0, 1.0), (p, 8, 63, 1e4, 0, 1.0, 0, 0.0, 0.0, 1.0),
                 (p, 8, 64, 1.0, 0, 1.0, 0, 0.0, 0.0, 1.0), (p, 8, 64, float("nan"), 0, 1.0, 0, 0.0, 0.0, 1.0), (p, 8, 64, 1e4, 5, 1.0, 0, 0.0, 0.0, 1.0),
                 (p, 8, 64, 1e4, 1, 0.0, 0, 0.0, 0.0, 1.0), (p, 8, 64, 1e4, 3, 2.0, 0, 1.0, 32.0, 1.0), (p, 8, 64, 1e4, 3, 2.0, 4096, 32.0, 1.0, 1.0),
                 (p, 8, 64, 1e4, 0, 1.0, 0, 0.0, 0.0, float("inf"))):
        assert t(*args, None) == bad, args


# ------------------------------------------------------------------ on a B200

@pytest.mark.gpu
@pytest.mark.parametrize("scaling", ["none", "linear", "ntk", "yarn", "bands"])
@pytest.mark.parametrize("dim", [2, 6, 64, 128, 256])
def test_table(cuda_device, scaling, dim):
    length = 5003
    kw = dict(scaling=scaling, factor=8.0, original_length=2048) if scaling != "none" else {}
    got = ro.rotary_table(length, dim, device=cuda_device, **kw)
    mul = 1.2079441541679836 if scaling == "yarn" else 1.0           # 0.1 ln 8 + 1
    want = ref.rotary_table(length, dim, multiplier=mul, **kw)
    assert got.shape == want.shape
    # one rounding of 2^-24, the angle's own error (5003 * 2^-53 and what pow() is off, a few 2^-53 of 5003) below 2^-38
    assert float((got.double().cpu() - want).abs().max()) <= mul * 2.0 ** -24 + 2.0 ** -38


@pytest.mark.gpu
def test_table_at_far_positions(cuda_device):
    got = ro.rotary_table(131072 + 3, 128, scaling="linear", factor=4.0, device=cuda_device)[131000:]
    f = ref.frequencies(128, scaling="linear", factor=4.0)
    angle = torch.arange(131000, 131075, dtype=torch.float64)[:, None] * f
    assert float((got.double().cpu() - torch.stack((angle.cos(), angle.sin()), -1)).abs().max()) <= 2.0 ** -24 + 2.0 ** -34


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("B,Hq,Hk,S,D,R", [
    (1, 1, 1, 1, 128, 128), (2, 3, 1, 7, 64, 64), (3, 8, 2, 33, 128, 64), (1, 32, 8, 5, 256, 256), (2, 5, 5, 19, 16, 16),
    (2, 2, 1, 13, 32, 8), (1, 4, 2, 9, 128, 6), (2, 17, 3, 4, 64, 2), (1, 1, 0, 40, 256, 96), (1, 40, 8, 600, 128, 128),
])
def test_forward(cuda_device, dtype, interleaved, B, Hq, Hk, S, D, R):
    g = torch.Generator(device=cuda_device).manual_seed(B * 1000 + S)
    q = torch.randn(B, Hq, S, D, generator=g, device=cuda_device).to(dtype)
    k = torch.randn(B, Hk, S, D, generator=g, device=cuda_device).to(dtype) if Hk else None
    table = ro.rotary_table(700, R, device=cuda_device)
    per_row = torch.randint(0, 700, (B, S), generator=g, device=cuda_device)
    for pos in (None, per_row.int(), per_row, per_row[0].int(), per_row[:1], torch.stack((per_row, per_row), -1)[..., 0]):
        got = ro.rotary(q, k, table, pos, interleaved)
        for x, y in zip((q, k), got):
            if x is None:
                assert y is None
                continue
            assert y.shape == x.shape and y.dtype == dtype
            close(y, x, table, ref.rotary(x, table, pos, interleaved), dtype, pos, interleaved)
            assert torch.equal(y[..., R:], x[..., R:])
    fa.device_status()


@pytest.mark.gpu
def test_storage_orders(cuda_device):
    B, H, S, D = 2, 4, 24, 64
    g = torch.Generator(device=cuda_device).manual_seed(2)
    rand = lambda *s: torch.randn(s, generator=g, device=cuda_device).half()  # noqa: E731
    table = ro.rotary_table(64, 32, device=cuda_device)
    forms = [rand(B, H, S, D), rand(B, S, H, D).transpose(1, 2), rand(B, S, 3, H, D).permute(2, 0, 3, 1, 4)[1], rand(B, H, S, D + 8)[..., :D],
             rand(B, H, S, D + 4)[..., :D], rand(B, H, S, 2 * D)[..., ::2], rand(B, 1, S, D).expand(B, H, S, D), rand(B, H, D, S).transpose(2, 3),
             rand(B * H * S * D + 1)[1:].view(B, H, S, D), rand(S, B, H, D).permute(1, 2, 0, 3)]
    for x in forms:
        y, z = ro.rotary(x, forms[1], table)
        close(y, x, table, ref.rotary(x, table), torch.float16)
        close(z, forms[1], table, ref.rotary(forms[1], table), torch.float16)


@pytest.mark.gpu
@pytest.mark.parametrize("route", ["native", "python"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("R", [64, 24, 10])
def test_gradient(cuda_device, monkeypatch, route, interleaved, R):
    if route == "python":
        monkeypatch.setattr(ro, "_native", None)
    B, Hq, Hk, S, D = 2, 4, 2, 11, 64
    g = torch.Generator(device=cuda_device).manual_seed(3)
    rand = lambda *s: torch.randn(s, generator=g, device=cuda_device).half()  # noqa: E731
    table = ro.rotary_table(50, R, scaling="yarn", factor=4.0, original_length=16, device=cuda_device)
    pos = torch.randint(0, 50, (B, S), generator=g, device=cuda_device)
    q, k = rand(B, Hq, S, D).requires_grad_(), rand(B, 1, S, D).requires_grad_()
    dq, dk = rand(B, Hq, S, D), rand(B, Hk, S, D)
    out = ro.rotary(q, k.expand(B, Hk, S, D), table, pos, interleaved)
    gq, gk = torch.autograd.grad(out, (q, k), (dq, dk))
    close(gq, dq, table, ref.rotary(dq, table, pos, interleaved, inverse=True), torch.float16, pos, interleaved, True)
    # the gradient of shared heads is their sum, taken by torch in 16 bits: one more rounding of each part and of the sum
    want = ref.rotary(dk, table, pos, interleaved, inverse=True)
    assert bool(((gk.double() - want.sum(1, keepdim=True)).abs() <= 2.0 ** -10 * want.abs().sum(1, keepdim=True) + 2.0 ** -20 * 8).all())
    # against differences: the map is linear, so <dq, R x> is <R^T dq, x>, up to the roundings of either side
    y = ref.rotary(q.detach(), table, pos, interleaved)
    lhs, rhs = (dq.double() * y).sum(), (gq.double() * q.detach().double()).sum()
    assert abs(float(lhs - rhs)) <= 2.0 ** -10 * float((dq.double() * y).abs().sum() + (gq.double() * q.detach().double()).abs().sum())
    # one output alone, sums (gradients without strides), and the gradient's own gradient
    only_k = torch.autograd.grad(ro.rotary(q, k, table, pos, interleaved)[1].float().sum(), k)[0]
    assert only_k.shape == k.shape and bool(torch.isfinite(only_k).all())
    a = ro.rotary(q, None, table, pos, interleaved)[0]
    seed = dq.clone().requires_grad_()
    first = torch.autograd.grad(a, q, seed, create_graph=True)[0]
    dd = rand(B, Hq, S, D)
    again = torch.autograd.grad(first, seed, dd)[0]
    close(again, dd, table, ref.rotary(dd, table, pos, interleaved), torch.float16, pos, interleaved)
    # gradients that the library cannot read as they are: no strides, columns apart, an unaligned base
    flat = rand(B * Hq * S * D + 1)[1:].view(B, Hq, S, D)
    for odd in (rand(1, 1, 1, 1).expand(B, Hq, S, D), rand(B, Hq, D, S).transpose(2, 3), flat):
        got = torch.autograd.grad(ro.rotary(q, k, table, pos, interleaved)[0], q, odd)[0]
        close(got, odd, table, ref.rotary(odd, table, pos, interleaved, inverse=True), torch.float16, pos, interleaved, True)
    with torch.no_grad():
        assert not ro.rotary(q, k, table, pos, interleaved)[0].requires_grad


@pytest.mark.gpu
def test_positions_outside_the_table_are_reported(cuda_device):
    table = ro.rotary_table(16, 64, device=cuda_device)
    q = torch.ones(1, 3, 4, 64, device=cuda_device, dtype=torch.bfloat16)
    fa.device_status()
    for bad in (16, -1, 2 ** 31 - 1):
        pos = torch.tensor([0, bad, 15, 3], device=cuda_device, dtype=torch.int32)
        y = ro.rotary(q, None, table, pos)[0]
        with pytest.raises(RuntimeError, match="device status 0x20001"):
            fa.device_status()
        assert bool(y[:, :, 1].isnan().all()) and bool(torch.isfinite(y[:, :, [0, 2, 3]]).all())
    fa.device_status()


@pytest.mark.gpu
def test_refusals_on_the_device(cuda_device):
    q = torch.zeros(1, 2, 4, 64, dtype=torch.float16, device=cuda_device)
    table = ro.rotary_table(8, 64, device=cuda_device)
    pos = torch.zeros(1, 4, dtype=torch.int32, device=cuda_device)
    for args in ((q.float(), q, table), (q, q.bfloat16(), table), (q, q, table.half()), (q, q, table[:, ::2]), (q, q, table[0]), (q, q, table.cpu()),
                 (q[..., :32].contiguous(), None, table), (q, q, table, pos.float()), (q, q, table, pos[:, :3]), (q, q, table, pos.cpu()),
                 (q, q, table.clone().requires_grad_())):
        with pytest.raises(ValueError):
            ro.rotary(*args)
    assert ro.rotary(q[:, :0], q, table)[1].shape == q.shape
    assert ro.rotary(q[:0], q[:0], table)[0].shape == q[:0].shape


@pytest.mark.gpu
def test_captured_forward_and_backward(cuda_device):
    table = ro.rotary_table(64, 128, device=cuda_device)
    q = torch.randn(2, 4, 16, 128, device=cuda_device, dtype=torch.bfloat16).requires_grad_()
    dq = torch.randn_like(q)
    eager = ro.rotary(q, None, table)[0].detach()   # (a live graph of the leaf made on another stream, torch itself refuses)
    want = torch.autograd.grad(ro.rotary(q, None, table)[0], q, dq)[0]
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        torch.autograd.grad(ro.rotary(q, None, table)[0], q, dq)
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = ro.rotary(q, None, table)[0]
        gq = torch.autograd.grad(y, q, dq)[0]
    for _ in range(2):
        y.data.zero_(), gq.zero_()
        graph.replay()
        assert torch.equal(gq, want) and torch.equal(y, eager)


@pytest.mark.gpu
@pytest.mark.parametrize("route", ["native", "python"])
@pytest.mark.parametrize("interleaved", [False, True])
def test_forward_mode(cuda_device, monkeypatch, route, interleaved):
    """A tangent is turned like what it belongs to, with and without gradients recorded, and through the backward pass."""
    if route == "python":
        monkeypatch.setattr(ro, "_native", None)
    B, Hq, Hk, S, D, R = 2, 3, 1, 9, 64, 32
    g = torch.Generator(device=cuda_device).manual_seed(4)
    rand = lambda *s: torch.randn(s, generator=g, device=cuda_device).bfloat16()  # noqa: E731
    table, pos = ro.rotary_table(40, R, device=cuda_device), torch.randint(0, 40, (B, S), generator=g, device=cuda_device)
    q, tq, k, tk = rand(B, Hq, S, D), rand(B, Hq, S, D), rand(B, Hk, S, D), rand(B, Hk, S, D)
    turned = lambda x, inverse=False: ref.rotary(x, table, pos, interleaved, inverse)  # noqa: E731
    plain = ro.rotary(q, k, table, pos, interleaved)
    for grad in (False, True):
        for qs, ks in ((True, True), (True, False), (False, True)):
            with fwAD.dual_level(), torch.set_grad_enabled(grad):
                x, y = q.clone().requires_grad_(grad), k.clone().requires_grad_(grad)
                out = ro.rotary(fwAD.make_dual(x, tq) if qs else x, fwAD.make_dual(y, tk) if ks else y, table, pos, interleaved)
                for o, p, t, used in zip(out, plain, (tq, tk), (qs, ks)):
                    primal, tangent = fwAD.unpack_dual(o)
                    assert torch.equal(primal, p) and (not grad or o.requires_grad)
                    if used:
                        close(tangent, t, table, turned(t), torch.bfloat16, pos, interleaved)
                    else:
                        assert tangent is None or bool((tangent == 0).all())
                if qs:
                    one = fwAD.unpack_dual(ro.rotary(fwAD.make_dual(x, tq), None, table, pos, interleaved)[0]).tangent
                    close(one, tq, table, turned(tq), torch.bfloat16, pos, interleaved)
    # forward over reverse: the gradient's tangent is the tangent of what comes in, turned back
    dq, dk, ddq, ddk = rand(B, Hq, S, D), rand(B, Hk, S, D), rand(B, Hq, S, D), rand(B, Hk, S, D)
    x, y = q.clone().requires_grad_(), k.clone().requires_grad_()
    for both in (True, False):
        with fwAD.dual_level():
            out = ro.rotary(x, y if both else None, table, pos, interleaved)
            seeds = (fwAD.make_dual(dq, ddq), fwAD.make_dual(dk, ddk))
            got = torch.autograd.grad(out if both else out[0], (x, y) if both else x, seeds if both else seeds[0])
            for o, d, dd in zip(got, (dq, dk), (ddq, ddk)):
                primal, tangent = fwAD.unpack_dual(o)
                close(primal, d, table, turned(d, True), torch.bfloat16, pos, interleaved, True)
                close(tangent, dd, table, turned(dd, True), torch.bfloat16, pos, interleaved, True)
    fa.device_status()


@pytest.mark.gpu
@pytest.mark.parametrize("route", ["native", "python"])
def test_refusals_of_the_library_with_a_gradient_recorded(cuda_device, monkeypatch, route):
    """The same errors with and without a gradient, and by either route."""
    if route == "python":
        monkeypatch.setattr(ro, "_native", None)
    q = torch.zeros(1, 65536, 1, 16, dtype=torch.float16, device=cuda_device)
    table = ro.rotary_table(4, 16, device=cuda_device)
    for x in (q, q.clone().requires_grad_()):
        with pytest.raises(ValueError, match="rsfa_rotary failed: problem too large"):
            ro.rotary(x, None, table)
    q = torch.zeros(1, 2, 1, 16, dtype=torch.float16, device=cuda_device, requires_grad=True)
    good = ro.rotary(q, None, table)[0]
    fa.device_status()
    try:
        fa.set_option("check_status", 1)
        ro.rotary(q.detach(), None, table, torch.tensor([9], device=cuda_device))
        torch.cuda.synchronize()
        with pytest.raises(RuntimeError, match="rsfa_rotary failed: a kernel reported"):
            ro.rotary(q, None, table)
        with pytest.raises(RuntimeError, match="rsfa_rotary failed: a kernel reported"):
            good.sum().backward()
        with pytest.raises(RuntimeError, match="0x20001"):
            fa.device_status()
    finally:
        fa.set_option("check_status", 0)
    fa.device_status()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("D,R", [(64, 32), (128, 16), (64, 6), (32, 20), (256, 2), (16, 16)])
def test_the_whole_row_of_a_position_outside_the_table_is_nan(cuda_device, dtype, interleaved, D, R):
    table = ro.rotary_table(16, R, device=cuda_device)
    q, k = (torch.randn(2, h, 5, D, device=cuda_device).to(dtype) for h in (3, 18))
    pos = torch.tensor([[0, 16, 15, -1, 3], [2 ** 31 - 1, 1, 2, 3, -2 ** 31]], device=cuda_device, dtype=torch.int32)
    fa.device_status()
    lost = ((pos < 0) | (pos >= 16))[:, None, :, None]
    for x, y in zip((q, k), ro.rotary(q, k, table, pos, interleaved)):
        assert torch.equal(y.isnan(), lost.expand_as(y))
        assert torch.equal(torch.where(lost, 0, y)[..., R:], torch.where(lost, 0, x)[..., R:])
    with pytest.raises(RuntimeError, match="device status 0x20001"):
        fa.device_status()
    fa.device_status()
