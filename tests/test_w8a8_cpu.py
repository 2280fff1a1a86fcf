"""Refusals of the W8A8 operators, on the host: nothing is launched, so they
need no GPU. Tensors without storage on a device stand in for CUDA tensors
where a check comes after the one for CUDA."""

import pytest
import torch

import pico_kernels_b200 as pk
from pico_kernels_b200 import _lib, gemm_w8a8

I8, E4, BF, F32 = _lib.PK_I8, _lib.PK_E4M3, _lib.PK_BF16, _lib.PK_F32


def test_c_abi_refuses_rows():
    lib = _lib.load()
    good = dict(x=64, dtype=BF, M=4, K=100, ldx=100, q=64, q_dtype=I8, ldq=112, scale=64, stream=None)

    def call(**kw):
        return lib.pk_quantize_rows(*dict(good, **kw).values())
    for kw in (dict(x=None), dict(q=None), dict(scale=None), dict(M=0), dict(K=0), dict(ldx=99),
               dict(ldq=99), dict(K=1 << 30, ldx=1 << 30, ldq=1 << 30), dict(M=(1 << 31) - 1)):
        assert call(**kw) == _lib.PK_ERR_SHAPE, kw
    for kw in (dict(dtype=I8), dict(q_dtype=BF), dict(q_dtype=_lib.PK_U8)):
        assert call(**kw) == _lib.PK_ERR_DTYPE, kw
    assert call(x=65) == call(scale=66) == _lib.PK_ERR_ALIGN
    deq = dict(q=64, q_dtype=E4, M=4, K=100, ldq=112, scale=64, out=64, out_dtype=BF, ldo=100,
               stream=None)

    def dcall(**kw):
        return lib.pk_dequantize_rows(*dict(deq, **kw).values())
    for kw in (dict(q=None), dict(out=None), dict(scale=None), dict(ldq=99), dict(ldo=99),
               dict(M=-1)):
        assert dcall(**kw) == _lib.PK_ERR_SHAPE, kw
    assert dcall(out_dtype=I8) == _lib.PK_ERR_DTYPE
    assert dcall(q_dtype=F32) == _lib.PK_ERR_DTYPE


def test_c_abi_refuses_norms():
    lib = _lib.load()
    good = dict(x=64, dtype=BF, M=4, K=100, ldx=100, residual=64, ldr=100, weight=64, w_dtype=BF,
                eps=1e-6, h=64, ldh=100, q=64, q_dtype=I8, ldq=112, scale=64, stream=None)

    def call(**kw):
        return lib.pk_rms_norm_quant(*dict(good, **kw).values())
    for kw in (dict(x=None), dict(weight=None), dict(q=None), dict(scale=None), dict(h=None),
               dict(ldr=99), dict(ldh=99), dict(ldx=99), dict(M=0), dict(eps=0.0), dict(eps=-1e-6),
               dict(eps=float("nan")), dict(eps=float("inf")), dict(eps=1e-45)):
        assert call(**kw) == _lib.PK_ERR_SHAPE, kw
    for kw in (dict(dtype=I8), dict(w_dtype=_lib.PK_F16), dict(q_dtype=F32)):
        assert call(**kw) == _lib.PK_ERR_DTYPE, kw
    for kw in (dict(x=65), dict(residual=65), dict(h=65), dict(weight=65), dict(scale=66)):
        assert call(**kw) == _lib.PK_ERR_ALIGN, kw


@pytest.mark.parametrize("gated", [False, True])
def test_c_abi_refuses_products(gated):
    lib = _lib.load()
    good = dict(a=64, dtype=I8, lda=112, sa=64, w=64, ldw=112, sw=64)
    good |= dict(u=64, ldu=112, su=64, act=0) if gated else dict(bias=None)
    good |= dict(M=4, N=32, K=100, out=64, out_dtype=BF, ldo=32, stream=None)
    fn = lib.pk_w8a8_gated_gemm if gated else lib.pk_w8a8_gemm

    def call(**kw):
        return fn(*dict(good, **kw).values())
    shape = [dict(a=None), dict(sa=None), dict(w=None), dict(sw=None), dict(out=None), dict(M=0),
             dict(N=0), dict(K=0), dict(lda=96), dict(ldw=96), dict(ldo=31), dict(M=1 << 30),
             dict(K=131072, lda=131072, ldw=131072, **(dict(ldu=131072) if gated else {}))]
    if gated:
        shape += [dict(u=None), dict(su=None), dict(ldu=96), dict(act=2), dict(act=-1)]
    for kw in shape:
        assert call(**kw) == _lib.PK_ERR_SHAPE, kw
    for kw in (dict(dtype=BF), dict(dtype=_lib.PK_U8), dict(out_dtype=I8), dict(out_dtype=E4)):
        assert call(**kw) == _lib.PK_ERR_DTYPE, kw
    align = [dict(a=72), dict(w=65), dict(lda=104), dict(ldw=120), dict(out=65), dict(sa=66),
             dict(sw=66)]
    for kw in align + ([dict(u=72), dict(ldu=104)] if gated else []):
        assert call(**kw) == _lib.PK_ERR_ALIGN, kw
    assert _lib.last_error() != ""


def test_host_tensors_are_refused():
    x = torch.zeros(2, 32, dtype=torch.bfloat16)
    q = torch.zeros(2, 32, dtype=torch.int8)
    s = torch.ones(2)
    for call in (lambda: pk.quantize_rows(x), lambda: pk.dequantize_rows(q, s),
                 lambda: pk.rms_norm_quant(x, torch.ones(32)),
                 lambda: pk.w8a8_gemm(q, s, q, s),
                 lambda: pk.w8a8_gated_gemm(q, s, q, s, q, s)):
        with pytest.raises(_lib.DtypeError):
            call()
    with pytest.raises(_lib.DtypeError):
        pk.quantize_rows(x, torch.uint8)
    with pytest.raises(ValueError):
        pk.w8a8_gated_gemm(q, s, q, s, q, s, activation="relu")


@pytest.fixture
def as_if_on_a_gpu(monkeypatch):
    """Let host tensors past the CUDA check, and fail where a call would launch."""
    monkeypatch.setattr(_lib, "require_cuda", lambda *ts: None)
    monkeypatch.setattr(_lib, "torch_fast", lambda: None)

    def launched(*_):
        raise AssertionError("a refused call reached its launch")
    monkeypatch.setattr(_lib, "load", launched)
    monkeypatch.setattr(_lib, "on_device", launched)


def test_wrappers_refuse(as_if_on_a_gpu):
    S, D = _lib.ShapeError, _lib.DtypeError
    x, w = torch.zeros(2, 32, dtype=torch.bfloat16), torch.ones(32)
    q, s = torch.zeros(2, 32, dtype=torch.int8), torch.ones(2)
    e = q.to(torch.float8_e4m3fn)
    cases = [
        (D, lambda: pk.quantize_rows(q)), (D, lambda: pk.quantize_rows(x.double())),
        (S, lambda: pk.quantize_rows(torch.tensor(1.0))),
        (S, lambda: pk.quantize_rows(x[:, :0])),
        (D, lambda: pk.dequantize_rows(x, s)), (D, lambda: pk.dequantize_rows(q, s.double())),
        (S, lambda: pk.dequantize_rows(q, s[:1])), (D, lambda: pk.dequantize_rows(q, s, torch.int8)),
        (S, lambda: pk.rms_norm_quant(x, w[:31])), (D, lambda: pk.rms_norm_quant(x, w.half())),
        (S, lambda: pk.rms_norm_quant(x, w, residual=x[:1])),
        (D, lambda: pk.rms_norm_quant(x, w, residual=x.float())),
        (S, lambda: pk.rms_norm_quant(x, w, residual_out=x)),
        (S, lambda: pk.rms_norm_quant(x, w, residual=x, residual_out=x.float())),
        (S, lambda: pk.rms_norm_quant(x, w, residual=x, residual_out=x.t().contiguous().t())),
        (D, lambda: pk.rms_norm_quant(x, w, dtype=torch.uint8)),
        (D, lambda: pk.w8a8_gemm(q, s, e, s)), (D, lambda: pk.w8a8_gemm(x, s, q, s)),
        (S, lambda: pk.w8a8_gemm(q, s, q[:, :16], s)), (S, lambda: pk.w8a8_gemm(q[0], s, q, s)),
        (S, lambda: pk.w8a8_gemm(q, s[:1], q, s)), (S, lambda: pk.w8a8_gemm(q, s, q, w)),
        (D, lambda: pk.w8a8_gemm(q, s.half(), q, s)),
        (S, lambda: pk.w8a8_gemm(q, s, q, s, bias=w)),
        (D, lambda: pk.w8a8_gemm(q, s, q, s, bias=s.bfloat16())),
        (D, lambda: pk.w8a8_gemm(q, s, q, s, out_dtype=torch.int8)),
        (S, lambda: pk.w8a8_gemm(q, s, q, s, out=torch.zeros(2, 3))),
        (S, lambda: pk.w8a8_gemm(q, s, q, s, out=torch.zeros(2, 2).t()[:, ::2])),
        (S, lambda: pk.w8a8_gemm(q, s, q[:, :0], s)),
        (S, lambda: pk.w8a8_gated_gemm(q, s, q, s, q[:1], s[:1])),
        (S, lambda: pk.w8a8_gated_gemm(q, s, q, s, q[:, :16], s)),
        (D, lambda: pk.w8a8_gated_gemm(q, s, q, s, e, s)),
        (S, lambda: pk.w8a8_gated_gemm(q, s, q, s, q, w)),
    ]
    for i, (err, call) in enumerate(cases):
        with pytest.raises(err):
            call()
            pytest.fail(f"case {i} was not refused")


def test_tensors_of_two_devices_are_refused(as_if_on_a_gpu):
    q, s = torch.zeros(2, 32, dtype=torch.int8), torch.ones(2)
    there = torch.empty(2, 32, dtype=torch.int8, device="meta")
    with pytest.raises(_lib.DtypeError):
        pk.w8a8_gemm(q, s.to("meta"), q, s)
    with pytest.raises(_lib.DtypeError):
        pk.dequantize_rows(q, s.to("meta"))
    x = torch.zeros(2, 32, dtype=torch.bfloat16)
    with pytest.raises(_lib.DtypeError):
        pk.rms_norm_quant(x, torch.ones(32, device="meta"))
    with pytest.raises(_lib.DtypeError):
        pk.rms_norm_quant(x, torch.ones(32), residual=x.to("meta"))
    assert there.device.type == "meta"


def test_row_storage_and_layouts(as_if_on_a_gpu):
    for K in (1, 15, 16, 17, 1000):
        t = gemm_w8a8.empty_rows((3, K), torch.int8, torch.device("cpu"))
        assert t.shape == (3, K) and t.stride() == (gemm_w8a8.row_pitch(K), 1)
        assert gemm_w8a8.row_pitch(K) % 16 == 0 and 0 <= gemm_w8a8.row_pitch(K) - K < 16
    x = torch.arange(4 * 6 * 8, dtype=torch.float32).reshape(4, 6, 8)
    for v, copied in ((x, False), (x[:, :, :5], False), (x[:, ::2], True),
                      (x.transpose(1, 2), True), (x[0, :1].expand(4, 8), True), (x[:1, :1], False)):
        r, ld = gemm_w8a8.as_rows(v)
        assert torch.equal(r, v.reshape(-1, v.shape[-1])) and ld >= v.shape[-1]
        assert r.shape[0] == 1 or r.stride(0) == ld
        assert copied or r.data_ptr() == v.data_ptr()


def test_modules_refuse():
    S, D = _lib.ShapeError, _lib.DtypeError
    def lin(i, o, bias=False, dtype=torch.int8):
        return pk.W8A8Linear(i, o, bias, dtype)
    a, down = lin(32, 64), lin(64, 32, True)
    assert a.weight8.shape == (64, 32) and lin(17, 3).codes.shape == (3, 32)
    pk.W8A8GatedMLP(a, a, down)
    for err, call in [
            (D, lambda: lin(32, 64, dtype=torch.uint8)),
            (S, lambda: pk.W8A8GatedMLP(a, a, down, activation="relu")),
            (S, lambda: pk.W8A8GatedMLP(lin(32, 64, True), a, down)),
            (S, lambda: pk.W8A8GatedMLP(a, lin(32, 48), down)),
            (S, lambda: pk.W8A8GatedMLP(a, a, lin(48, 32))),
            (D, lambda: pk.W8A8GatedMLP(a, lin(32, 64, dtype=torch.float8_e4m3fn), down)),
            (S, lambda: pk.W8A8GatedMLP(a, a, down, norm_weight=torch.ones(31))),
            (D, lambda: pk.W8A8Linear.from_linear(torch.nn.Linear(4, 4))),
            (S, lambda: pk.quantize_linear_layers(torch.nn.Linear(4, 4), scheme="w2a2")),
            (S, lambda: pk.quantize_linear_layers(torch.nn.Linear(4, 4), scheme="w8a8",
                                                  calib=torch.zeros(1, 4))),
            (D, lambda: pk.quantize_linear_layers(torch.nn.Linear(4, 4), scheme="w8a8",
                                                  dtype=torch.bfloat16))]:
        with pytest.raises(err):
            call()


@pytest.mark.parametrize("gated", [False, True])
def test_c_abi_refuses_long_e4m3_sums(gated):
    lib = _lib.load()
    K = (1 << 24) + 16
    if gated:
        st = lib.pk_w8a8_gated_gemm(64, E4, K, 64, 64, K, 64, 64, K, 64, 0, 1, 1, K, 64, F32, 1, None)
    else:
        st = lib.pk_w8a8_gemm(64, E4, K, 64, 64, K, 64, None, 1, 1, K, 64, F32, 1, None)
    assert st == _lib.PK_ERR_SHAPE


@pytest.mark.parametrize("code", [torch.int8, torch.float8_e4m3fn])
def test_linear_keeps_its_types(code):
    """Casts of a module tree move the layer but change neither codes nor scales."""
    layer = pk.W8A8Linear(20, 6, dtype=code)
    layer.codes.view(torch.uint8).random_(0, 120)
    layer.scales.uniform_()
    layer.bias.uniform_()
    codes, scales, bias = (t.clone() for t in (layer.codes, layer.scales, layer.bias))
    tree = torch.nn.Sequential(torch.nn.Linear(4, 4), layer)
    for cast in (lambda m: m.half(), lambda m: m.to(torch.bfloat16), lambda m: m.double(),
                 lambda m: m.to("cpu", torch.float16)):
        cast(tree)
        assert tree[0].weight.dtype != torch.float32
        assert layer.codes.dtype == code
        assert torch.equal(layer.codes.view(torch.uint8), codes.view(torch.uint8))
        assert torch.equal(layer.scales, scales) and torch.equal(layer.bias, bias)
    loaded = pk.W8A8Linear(20, 6, dtype=code).half()
    loaded.load_state_dict(layer.state_dict())
    assert torch.equal(loaded.scales, scales)


def test_outputs_that_overlap_an_operand_are_refused(as_if_on_a_gpu):
    pool = torch.zeros(4096, dtype=torch.uint8)
    q = pool[:1024].view(torch.int8).view(32, 32)
    s, b = (pool[i:i + 128].view(torch.float32) for i in (1024, 1152))
    w, one = torch.zeros(32, 32, dtype=torch.int8), torch.ones(32)

    def out(at):
        return pool[at:at + 2048].view(torch.bfloat16).view(32, 32)

    bf = torch.bfloat16
    for at, a8, sa, w8, sw, bias in ((0, q, one, w, one, None), (1022, q, one, w, one, None),
                                     (0, w, one, q, one, None), (1022, w, one, q, one, None),
                                     (1024, w, s, w, one, None), (1150, w, one, w, s, None),
                                     (1152, w, one, w, one, b), (1278, w, one, w, one, b)):
        with pytest.raises(_lib.ShapeError):
            pk.w8a8_gemm(a8, sa, w8, sw, bias=bias, out_dtype=bf, out=out(at))
        if bias is None:
            for weights in ((w8, sw, w, one), (w, one, w8, sw)):
                with pytest.raises(_lib.ShapeError):
                    pk.w8a8_gated_gemm(a8, sa, *weights, out_dtype=bf, out=out(at))
    with pytest.raises(AssertionError):  # not refused: it gets to its launch
        pk.w8a8_gemm(q, s, w, one, bias=b, out_dtype=bf, out=out(1280))
