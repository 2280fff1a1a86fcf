"""W8A8Linear, W8A8GatedMLP and quantize_linear_layers(scheme="w8a8") on the
GPU, against the operators they are made of and against 64 bits.

The layer's output must be the product of its own codes: exact integer sums,
four fp32 roundings, one rounding to the activation type (2^-8 bf16, 2^-11
fp16, of the value). Against the float layer the 8-bit grid shows: a row's
127th (int8) rounded to nearest, an error of uniform spread step / sqrt(12) in
each operand, below 1.5 % of the product together for Gaussian rows.
"""

import pytest
import torch
import torch.nn as nn

import pico_kernels_b200 as pk
from pico_kernels_b200 import _lib

pytestmark = pytest.mark.gpu

HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


@pytest.mark.parametrize("code", [torch.int8, torch.float8_e4m3fn])
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("bias", [True, False])
@pytest.mark.parametrize("lead", [(), (1,), (2, 3), (5, 60)])
def test_linear_is_the_product_of_its_codes(lead, bias, dt, code):
    torch.manual_seed(0)
    lin = nn.Linear(500, 333, bias=bias).cuda().to(dt)
    q = pk.W8A8Linear.from_linear(lin, code)
    x = torch.randn(*lead, 500, device="cuda").to(dt)
    y = q(x)
    assert y.shape == (*lead, 333) and y.dtype == dt
    c, s = pk.quantize_rows(x.reshape(-1, 500), code)
    ref = (c.double() * s.double()[:, None]) @ q.dequantized_weight().double().t()
    mag = (c.double().abs() * s.double()[:, None]) @ q.dequantized_weight().double().abs().t()
    b = q.bias.double() if bias else torch.zeros(333, device="cuda", dtype=torch.float64)
    # int8 sums are exact; e4m3's lose at most a last place an addition; the
    # dequantized weight itself is a rounded product (2^-24 of each term)
    err = (8 if code == torch.int8 else 1000) * 2.0 ** -24 * (mag + b.abs())
    ref = (ref + b).reshape(y.shape)
    err = err.reshape(y.shape)
    assert ((y.double() - ref).abs() <= err + HALF[dt] * (ref.abs() + err) + 2.0 ** -24).all()
    full = nn.functional.linear(x.double(), lin.weight.double(),
                                lin.bias.double() if bias else None)
    assert torch.linalg.norm(y.double() - full) <= \
        (0.02 if code == torch.int8 else 0.06) * torch.linalg.norm(full)
    assert pk.device_status() == (0, 0)


@pytest.mark.parametrize("M", [1, 40, 300])
@pytest.mark.parametrize("norm,residual", [(False, False), (True, False), (True, True)])
@pytest.mark.parametrize("act", ["silu", "gelu_tanh"])
def test_gated_mlp_is_its_operators(act, norm, residual, M):
    torch.manual_seed(M)
    K, F = 272, 700
    g, u, d = nn.Linear(K, F, bias=False), nn.Linear(K, F, bias=False), nn.Linear(F, K)
    mods = [m.cuda().bfloat16() for m in (g, u, d)]
    w = (1 + 0.1 * torch.randn(K, device="cuda")).bfloat16() if norm else None
    mlp = pk.W8A8GatedMLP.from_linears(*mods, norm_weight=w, activation=act)
    x = torch.randn(2, M, K, device="cuda").bfloat16()
    r = torch.randn(2, M, K, device="cuda").bfloat16() if residual else None
    out = mlp(x, r) if residual else mlp(x)
    y, h = out if residual else (out, None)
    assert y.shape == x.shape and y.dtype == x.dtype
    n = x.double()
    if residual:
        assert torch.equal(h, (x.float() + r.float()).bfloat16())
        n = h.double()
    if norm:
        n = n / torch.sqrt(n.square().mean(-1, keepdim=True) + 1e-6) * w.double()
    a = n @ g.weight.double().t()
    f = nn.functional.silu(a) if act == "silu" else nn.functional.gelu(a, approximate="tanh")
    ref = (f * (n @ u.weight.double().t())) @ d.weight.double().t() + d.bias.double()
    # three products of int8 operands, each off by under 1.5 %
    assert torch.linalg.norm(y.double() - ref) <= 0.05 * torch.linalg.norm(ref)
    # and exactly the chain of the public operators
    x2 = x.reshape(-1, K)
    if residual:
        q, s, _ = pk.rms_norm_quant(x2, w, 1e-6, residual=r.reshape(-1, K))
    elif norm:
        q, s = pk.rms_norm_quant(x2, w, 1e-6)
    else:
        q, s = pk.quantize_rows(x2)
    t = pk.w8a8_gated_gemm(q, s, mlp.gate.weight8, mlp.gate.scales, mlp.up.weight8,
                           mlp.up.scales, activation=act, out_dtype=torch.bfloat16)
    q, s = pk.quantize_rows(t)
    z = pk.w8a8_gemm(q, s, mlp.down.weight8, mlp.down.scales, bias=mlp.down.bias,
                     out_dtype=torch.bfloat16)
    assert torch.equal(y.reshape(-1, K), z)
    assert pk.device_status() == (0, 0)


def test_quantize_linear_layers_w8a8():
    torch.manual_seed(3)
    model = nn.Sequential(nn.Linear(200, 301), nn.GELU(), nn.Linear(301, 64)).cuda()
    x = torch.randn(70, 200, device="cuda")
    full = model(x)
    pk.quantize_linear_layers(model, scheme="w8a8")
    assert isinstance(model[0], pk.W8A8Linear) and isinstance(model[2], pk.W8A8Linear)
    y = model(x)
    assert torch.linalg.norm(y - full) <= 0.05 * torch.linalg.norm(full)
    # saved, loaded and moved over the host: the same codes, laid out as before
    other = nn.Sequential(pk.W8A8Linear(200, 301), nn.GELU(), pk.W8A8Linear(301, 64))
    other.load_state_dict(model.state_dict())
    other = other.cuda()
    assert other[2].weight8.stride(0) % 16 == 0
    assert torch.equal(other(x), y)
    # selected layers only, e4m3
    model = nn.Sequential(nn.Linear(64, 64), nn.Linear(64, 64)).cuda()
    pk.quantize_linear_layers(model, scheme="w8a8", dtype=torch.float8_e4m3fn,
                              select=lambda n, m: n == "1")
    assert type(model[0]) is nn.Linear and model[1].dtype == torch.float8_e4m3fn


def test_mlp_step_captured_in_a_graph():
    torch.manual_seed(4)
    K, F = 512, 1024
    mods = [nn.Linear(a, b, bias=False).cuda().bfloat16() for a, b in ((K, F), (K, F), (F, K))]
    w = torch.rand(K, device="cuda").bfloat16()
    mlp = pk.W8A8GatedMLP.from_linears(*mods, norm_weight=w)
    x, r = (torch.randn(3, K, device="cuda").bfloat16() for _ in range(2))
    mlp(x, r)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y, h = mlp(x, r)
    for scale in (1.0, -2.0):
        x.mul_(scale)
        g.replay()
        ye, he = mlp(x, r)
        torch.cuda.synchronize()
        assert torch.equal(y, ye) and torch.equal(h, he)


def test_refusals():
    lin = nn.Linear(64, 64).cuda()
    q = pk.W8A8Linear.from_linear(lin)
    with pytest.raises(_lib.ShapeError):
        q(torch.zeros(2, 63, device="cuda"))
    with pytest.raises(_lib.DtypeError):
        q(torch.zeros(2, 64, device="cuda", dtype=torch.float64))
    nb = pk.W8A8Linear.from_linear(nn.Linear(64, 64, bias=False).cuda())
    mlp = pk.W8A8GatedMLP(nb, nb, q)
    with pytest.raises(_lib.ShapeError):
        mlp(torch.zeros(2, 64, device="cuda"), torch.zeros(2, 64, device="cuda"))
    with pytest.raises(_lib.ShapeError):
        mlp(torch.zeros(2, 32, device="cuda"))
