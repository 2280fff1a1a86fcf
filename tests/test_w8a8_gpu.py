"""The W8A8 products on the GPU against their definitions in 64 bits.

Tolerances: int8 sums are exact, so a result carries the int32 -> fp32
conversion, one product per scale and the bias's addition: four fp32 roundings
(2^-24 each) of a magnitude of at most |sum| + |bias|, then the output type's
half step. e4m3 sums are fp32: every addition may lose up to a last place
(2^-23) of the running sum of magnitudes, K * 2^-23 * sum|a||w| at most, and
the whole product stays within the framework's fp8 bar (rel-Frobenius 1e-5).
The gated form carries both products' errors through act'(g) (at most 1.2 for
SiLU and GELU) and u, and its own roundings: the exponent's relative error is
|t| * 2^-22 where t < 0, a dozen roundings elsewhere.
"""

import pytest
import torch

import pico_kernels_b200 as pk
from pico_kernels_b200 import _lib

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24}
CODES = [torch.int8, torch.float8_e4m3fn]
# single tokens, a tile's edges in every dimension, lengths of one, odd sizes,
# several waves of large tiles with a ragged last one
SHAPES = [(1, 1, 1), (1, 4096, 4096), (1, 129, 1000), (2, 64, 15), (3, 1000, 17), (7, 128, 128),
          (16, 256, 4096), (16, 8192, 1024), (17, 130, 127), (33, 1111, 1001), (64, 512, 129),
          (65, 384, 640), (128, 2048, 256), (129, 257, 511), (200, 1000, 2048), (256, 256, 384),
          (257, 31, 272), (300, 4096, 1024), (1000, 1111, 333), (1025, 8200, 192),
          (5000, 520, 144), (40, 3, 20000)]


def _codes(rows, cols, code, g, pitch=None):
    v = torch.randn(rows, pitch or (cols + 15) // 16 * 16, device="cuda", generator=g)
    most = 127 if code == torch.int8 else 448
    v = (v * most / 4).clamp(-most, most)
    return (v.round() if code == torch.int8 else v).to(code)[:, :cols]


def _operands(M, N, K, code, seed=0, weights=1):
    g = torch.Generator(device="cuda").manual_seed(seed + M + N + K)
    most = 127 if code == torch.int8 else 448
    a = _codes(M, K, code, g)
    sa = (0.5 + torch.rand(M, device="cuda", generator=g)) * 4 / most
    w = []
    for _ in range(weights):
        w += [_codes(N, K, code, g),
              (0.5 + torch.rand(N, device="cuda", generator=g)) * 4 / most / K ** 0.5]
    return a, sa, w, torch.randn(N, device="cuda", generator=g)


def _product64(a, sa, w, sw):
    """(product, its error bound before the bias and the output's rounding)."""
    s = sa.double()[:, None] * sw.double()
    y = (a.double() @ w.double().t()) * s
    if a.dtype == torch.int8:
        return y, 3 * U * y.abs()
    mag = (a.double().abs() @ w.double().abs().t()) * s
    return y, a.shape[1] * 2 * U * mag + 3 * U * y.abs()


def _assert_near(y, ref, err, rel=None):
    assert torch.isfinite(y.float()).all()
    tol = err + HALF[y.dtype] * (ref.abs() + err) + TINY[y.dtype]
    over = (y.double() - ref).abs() > tol
    assert not over.any(), (over.sum().item(), (y.double() - ref).abs().max().item())
    if rel is not None and y.dtype == torch.float32:
        assert (torch.linalg.norm(y.double() - ref) <= rel * torch.linalg.norm(ref)).item()


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("M,N,K", SHAPES)
def test_w8a8_gemm(M, N, K, code):
    a, sa, (w, sw), b = _operands(M, N, K, code)
    ref, err = _product64(a, sa, w, sw)
    y = pk.w8a8_gemm(a, sa, w, sw)
    assert y.dtype == torch.float32 and y.shape == (M, N)
    _assert_near(y, ref, err, 1e-5)
    assert torch.equal(pk.w8a8_gemm(a, sa, w, sw), y)
    for dt in (torch.bfloat16, torch.float16):
        # the fp32 result rounded once
        assert torch.equal(pk.w8a8_gemm(a, sa, w, sw, out_dtype=dt), y.to(dt))
    yb = pk.w8a8_gemm(a, sa, w, sw, bias=b)
    _assert_near(yb, ref + b.double(), err + U * (ref.abs() + b.double().abs()))
    assert pk.device_status() == (0, 0)


@pytest.mark.parametrize("M,N,K", [(1, 512, 28672), (16, 256, 28672), (300, 300, 28672),
                                   (600, 4096, 12000), (130, 130, 100000)])
def test_long_e4m3_sums_keep_fp32_precision(M, N, K):
    # no accumulator of an fp32 output takes more than 5120 of K, where a tensor
    # core's truncation (half a last place of fp32 a step of 32, towards zero, is
    # 2^-25 * 160 = 4.8e-6 at worst, and 4.5e-9 * 160 = 7e-7 of a sum of either
    # sign as measured) stays below 1e-6 of the result's norm
    for weights in (1, 2):
        a, sa, w, _ = _operands(M, N, K, torch.float8_e4m3fn, seed=5, weights=weights)
        ref = _product64(a, sa, w[0], w[1])[0]
        if weights == 1:
            y = pk.w8a8_gemm(a, sa, w[0], w[1])
        else:
            ref = _act64(ref, "silu")[0] * _product64(a, sa, w[2], w[3])[0]
            y = pk.w8a8_gated_gemm(a, sa, *w)
        assert (torch.linalg.norm(y.double() - ref) <= 1e-6 * weights * torch.linalg.norm(ref)).item()


def _act64(g, act):
    if act == "silu":
        return g * torch.sigmoid(g), g
    t = 2 * (2 / torch.pi) ** 0.5 * (g + 0.044715 * g ** 3)
    return g * torch.sigmoid(t), t


@pytest.mark.parametrize("act", ["silu", "gelu_tanh"])
@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("M,N,K", SHAPES)
def test_w8a8_gated_gemm(M, N, K, code, act):
    a, sa, (wg, sg, wu, su), _ = _operands(M, N, K, code, seed=1, weights=2)
    (g, eg), (u, eu) = _product64(a, sa, wg, sg), _product64(a, sa, wu, su)
    f, t = _act64(g, act)
    ref = f * u
    own = (12 + 4 * (-t).clamp(0, 100)) * U
    err = 1.2 * eg * (u.abs() + eu) + f.abs() * eu + own * ref.abs()
    y = pk.w8a8_gated_gemm(a, sa, wg, sg, wu, su, activation=act)
    _assert_near(y, ref, err, 1e-5)
    for dt in (torch.bfloat16, torch.float16):
        assert torch.equal(pk.w8a8_gated_gemm(a, sa, wg, sg, wu, su, activation=act,
                                              out_dtype=dt), y.to(dt))
    assert pk.device_status() == (0, 0)


def test_int8_sums_are_exact_to_the_last_unit():
    # the largest K and the largest magnitudes: 131071 * 2^14 < 2^31
    K = 131071
    a = torch.full((2, K + 1), -128, device="cuda", dtype=torch.int8)[:, :K]
    w = torch.full((3, K + 1), -128, device="cuda", dtype=torch.int8)[:, :K]
    one = torch.ones(3, device="cuda")
    for M in (2, 300):
        x = a[:1].expand(M, K).contiguous()
        x = torch.nn.functional.pad(x, (0, 1))[:, :K]
        y = pk.w8a8_gemm(x, torch.ones(M, device="cuda"), w, one)
        assert (y == float(K * 2 ** 14)).all()  # (2^17 - 1) * 2^14 is exact in fp32
        x = x.clone()
        x = torch.nn.functional.pad(x, (0, 1))[:, :K]
        x[:, ::2] = 127
        s = int((x[0].long() * w[0].long()).sum())
        y = pk.w8a8_gemm(x, torch.ones(M, device="cuda"), w, one)
        assert (y == torch.tensor(s, dtype=torch.float64).float().item()).all()


def test_gate_far_from_zero():
    # |g| from tiny to where exp leaves fp32: no NaN, act's own limits
    vals = torch.tensor([0.0, 1e-30, -1e-30, 0.1, -0.1, 20.0, -20.0, 88.0, -88.0, -89.5, -104.0,
                         3e4, -3e4, 1e12, -1e12, 1e30, -1e30], device="cuda")
    n = vals.numel()
    a = torch.ones(1, 16, device="cuda", dtype=torch.int8)
    w = torch.zeros(n, 16, device="cuda", dtype=torch.int8)
    w[:, 0] = 1
    one = torch.ones(1, device="cuda")
    for act in ("silu", "gelu_tanh"):
        y = pk.w8a8_gated_gemm(a, one, w, vals, w, torch.ones(n, device="cuda"),
                               activation=act)[0].double()
        f, t = _act64(vals.double(), act)
        assert torch.isfinite(y).all()
        # below exp's range the result is zero or a subnormal: 1e-30 covers g * exp(-|t|) there
        assert ((y - f).abs() <= (12 + 4 * (-t).clamp(0, 100)) * U * f.abs() + 1e-30).all()


def test_scales_with_nan_reach_only_their_rows_and_columns():
    a, sa, (w, sw), _ = _operands(200, 300, 256, torch.int8)
    sa, sw = sa.clone(), sw.clone()
    sa[7] = float("nan")
    sw[11] = float("nan")
    y = pk.w8a8_gemm(a, sa, w, sw)
    bad = torch.isnan(y)
    assert bad[7].all() and bad[:, 11].all()
    assert bad.sum() == 200 + 300 - 1


@pytest.mark.parametrize("code", CODES)
def test_layouts(code):
    M, N, K = 70, 96, 208
    g = torch.Generator(device="cuda").manual_seed(0)
    wide = _codes(M, 512, code, g)
    both = _codes(2 * N, K, code, g)
    s = torch.rand(2 * N, device="cuda") / 100
    sa = torch.rand(M, device="cuda") / 100
    a = wide[:, 16:16 + K]                       # rows 512 apart, aligned
    ref = pk.w8a8_gemm(a.contiguous(), sa, both[:N].clone(), s[:N].clone())
    assert torch.equal(pk.w8a8_gemm(a, sa[:, None], both[:N], s[:N]), ref)
    ug = wide[:, 7:7 + K]                        # unaligned: copied
    assert torch.equal(pk.w8a8_gemm(ug, sa, both[:N], s[:N]),
                       pk.w8a8_gemm(ug.contiguous(), sa, both[:N], s[:N]))
    t = a.t().contiguous().t()                   # column-major
    assert torch.equal(pk.w8a8_gemm(t, sa, both[:N], s[:N]), ref)
    assert torch.equal(pk.w8a8_gemm(a[:1].expand(M, K), sa, both[:N], s[:N]),
                       pk.w8a8_gemm(a[:1].repeat(M, 1), sa, both[:N], s[:N]))
    # gate and up as halves of one weight
    fused = pk.w8a8_gated_gemm(a, sa, both[:N], s[:N], both[N:], s[N:])
    apart = pk.w8a8_gated_gemm(a, sa, both[:N].clone(), s[:N].clone(), both[N:].clone(),
                               s[N:].clone())
    assert torch.equal(fused, apart)
    out = torch.empty(M, N, device="cuda", dtype=torch.bfloat16)
    assert pk.w8a8_gemm(a, sa, both[:N], s[:N], out_dtype=torch.bfloat16, out=out) is out
    assert torch.equal(out, ref.bfloat16())
    # no tokens
    assert pk.w8a8_gemm(a[:0], sa[:0], both[:N], s[:N]).shape == (0, N)
    assert pk.w8a8_gated_gemm(a[:0], sa[:0], both[:N], s[:N], both[N:], s[N:]).shape == (0, N)


@pytest.mark.parametrize("M", [1, 5, 100, 700])
def test_rows_and_columns_past_the_output_are_left_alone(M):
    lib = _lib.load()
    N, K, ldo = 200, 160, 264
    a, sa, (w, sw), _ = _operands(M, N, K, torch.int8)
    for dt, code in ((torch.float32, _lib.PK_F32), (torch.bfloat16, _lib.PK_BF16)):
        buf = torch.full((M + 2, ldo), 77.0, device="cuda", dtype=dt)
        st = lib.pk_w8a8_gemm(a.data_ptr(), _lib.PK_I8, a.stride(0), sa.data_ptr(), w.data_ptr(),
                              w.stride(0), sw.data_ptr(), None, M, N, K, buf[1:].data_ptr(), code,
                              ldo, _lib.stream_of(a))
        assert st == _lib.PK_OK, _lib.last_error()
        assert (buf[0] == 77).all() and (buf[-1] == 77).all() and (buf[:, N:] == 77).all()
        assert torch.equal(buf[1:-1, :N], pk.w8a8_gemm(a, sa, w, sw, out_dtype=dt))
        # an output whose rows are not 16-byte aligned
        odd = torch.full((M * 203 + 1,), 77.0, device="cuda", dtype=dt)
        st = lib.pk_w8a8_gemm(a.data_ptr(), _lib.PK_I8, a.stride(0), sa.data_ptr(), w.data_ptr(),
                              w.stride(0), sw.data_ptr(), None, M, N, K, odd[1:].data_ptr(), code,
                              203, _lib.stream_of(a))
        assert st == _lib.PK_OK, _lib.last_error()
        o = odd[1:].view(M, 203)
        assert odd[0] == 77 and (o[:, N:] == 77).all()
        assert torch.equal(o[:, :N], buf[1:-1, :N])


def test_what_lies_between_the_columns_and_the_pitch_is_not_read():
    for M in (3, 400):
        a, sa, (w, sw), _ = _operands(M, 300, 100, torch.float8_e4m3fn)
        ref = pk.w8a8_gemm(a, sa, w, sw)
        for t in (a, w):
            full = torch.as_strided(t.view(torch.uint8), (t.shape[0], t.stride(0)),
                                    (t.stride(0), 1))
            full[:, 100:] = 0x7F  # e4m3 NaN
        assert torch.equal(pk.w8a8_gemm(a, sa, w, sw), ref)


def test_output_offsets_past_31_bits():
    M, N, K = 66000, 32768, 32
    g = torch.Generator(device="cuda").manual_seed(0)
    a, w = _codes(M, K, torch.int8, g), _codes(N, K, torch.int8, g)
    sa, sw = torch.rand(M, device="cuda"), torch.rand(N, device="cuda")
    y = pk.w8a8_gemm(a, sa, w, sw, out_dtype=torch.bfloat16)
    tail = pk.w8a8_gemm(a[-200:], sa[-200:], w, sw, out_dtype=torch.bfloat16)
    assert torch.equal(y[-200:], tail)


def test_a_token_does_not_depend_on_its_batch_in_int8():
    a, sa, (wg, sg, wu, su), b = _operands(600, 640, 512, torch.int8, weights=2)
    y = pk.w8a8_gemm(a, sa, wg, sg, bias=b)
    z = pk.w8a8_gated_gemm(a, sa, wg, sg, wu, su)
    for rows in (slice(0, 1), slice(5, 9), slice(100, 140), slice(300, 600)):
        assert torch.equal(pk.w8a8_gemm(a[rows], sa[rows], wg, sg, bias=b), y[rows])
        assert torch.equal(pk.w8a8_gated_gemm(a[rows], sa[rows], wg, sg, wu, su), z[rows])


@pytest.mark.parametrize("M", [1, 12, 600])
def test_fast_path_equals_python_path(M):
    a, sa, (wg, sg, wu, su), b = _operands(M, 640, 520, torch.int8, weights=2)
    tf = _lib.torch_fast()
    assert tf is not None
    y = tf.w8a8_gemm(a, sa, wg, sg, b, torch.bfloat16, None)
    z = tf.w8a8_gated_gemm(a, sa, wg, sg, wu, su, 1, torch.float16, None)
    assert isinstance(y, torch.Tensor) and isinstance(z, torch.Tensor)
    saved = _lib._tfast
    _lib._tfast = False
    try:
        assert torch.equal(pk.w8a8_gemm(a, sa, wg, sg, bias=b, out_dtype=torch.bfloat16), y)
        assert torch.equal(pk.w8a8_gated_gemm(a, sa, wg, sg, wu, su, activation="gelu_tanh",
                                              out_dtype=torch.float16), z)
    finally:
        _lib._tfast = saved


def _block(x, r, w, gate, up, down):
    q, s, h = pk.rms_norm_quant(x, w, residual=r)
    y = pk.w8a8_gated_gemm(q, s, *gate, *up, out_dtype=torch.bfloat16)
    y8, sy = pk.quantize_rows(y)
    return pk.w8a8_gemm(y8, sy, *down, out_dtype=torch.bfloat16), h


def _block_weights(K, F, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    w = (1 + 0.1 * torch.randn(K, device="cuda", generator=g)).bfloat16()
    mats = [torch.randn(n, k, device="cuda", generator=g) * k ** -0.5
            for n, k in ((F, K), (F, K), (K, F))]
    return w, mats, [pk.quantize_rows(m) for m in mats]


@pytest.mark.parametrize("M", [1, 16, 150, 600])
def test_the_operators_together_as_a_feed_forward_block(M):
    K, F = 1000, 1304
    w, mats, packed = _block_weights(K, F)
    x = torch.randn(M, K, device="cuda").bfloat16()
    r = torch.randn(M, K, device="cuda").bfloat16()
    y, h = _block(x, r, w, *packed)
    assert torch.equal(h, (x.float() + r.float()).bfloat16())
    # the float block: 8-bit codes are off by at most half a step of a row's
    # 127th; with Gaussian rows (maximum ~3.5 deviations) that is ~0.8 % rms of
    # each of the two operands of each product
    n = h.double() / torch.sqrt(h.double().square().mean(-1, keepdim=True) + 1e-6) * w.double()
    g, u, d = (m.double() for m in mats)
    t = torch.nn.functional.silu(n @ g.t()) * (n @ u.t())
    ref = t @ d.t()
    assert torch.linalg.norm(y.double() - ref) <= 0.05 * torch.linalg.norm(ref)
    # the same chain of the operators' own values in 64 bits: what is left is
    # bf16's rounding of y and the codes that a rounding moved by one
    q, s = pk.rms_norm_quant(h, w)
    n = q.double() * s.double()[:, None]
    (g, u, d) = (pk.dequantize_rows(*p).double() for p in packed)
    t8, st = pk.quantize_rows((torch.nn.functional.silu(n @ g.t()) * (n @ u.t())).bfloat16())
    ref = (t8.double() * st.double()[:, None]) @ d.t()
    assert torch.linalg.norm(y.double() - ref) <= 2.0 ** -8 * 2 * torch.linalg.norm(ref)
    assert pk.device_status() == (0, 0)


def test_block_captured_twice_and_replayed_at_once():
    # nothing is shared between captured calls: two graphs of the same block run
    # on two streams at the same time and give the eager results
    w, _, packed = _block_weights(512, 768)
    xs = [torch.randn(m, 512, device="cuda").bfloat16() for m in (1, 70)]
    want = [_block(x, x, w, *packed) for x in xs]
    graphs, outs = [], []
    for x in xs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(_block(x, x, w, *packed))
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in xs]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(20):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for o, want_o in zip(outs, want):
        assert all(torch.equal(a, b) for a, b in zip(o, want_o))
    for x in xs:
        x.mul_(-1.5)
    want = [_block(x, x, w, *packed) for x in xs]
    for g in graphs:
        g.replay()
    torch.cuda.synchronize()
    for o, want_o in zip(outs, want):
        assert all(torch.equal(a, b) for a, b in zip(o, want_o))


def test_products_of_several_streams_at_once():
    """Clusters of different sizes share SMs and their tensor memory: the results
    are those of the calls one after another."""
    sizes = [(1, 512, 4096), (16, 256, 16384), (40, 384, 8192), (130, 640, 4096), (200, 512, 4096),
             (256, 256, 8192), (300, 1024, 512)]
    calls = []
    for i, (M, N, K) in enumerate(sizes):
        for code in CODES:
            g = torch.Generator(device="cuda").manual_seed(i)
            a, w, u = (_codes(r, K, code, g) for r in (M, N, N))
            sa, sw, su = (torch.rand(r, device="cuda", generator=g) for r in (M, N, N))
            calls.append(lambda a=a, sa=sa, w=w, sw=sw: pk.w8a8_gemm(a, sa, w, sw))
            calls.append(lambda a=a, sa=sa, w=w, sw=sw, u=u, su=su:
                         pk.w8a8_gated_gemm(a, sa, w, sw, u, su, out_dtype=torch.float16))
    want = [c() for c in calls]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    for turn in range(4):
        got = [[] for _ in streams]
        for j in range(len(calls)):
            for s, stream in enumerate(streams):
                k = (j * (2 * s + 1) + 5 * s + turn) % len(calls)
                with torch.cuda.stream(stream):
                    got[s].append((k, calls[k]()))
        torch.cuda.synchronize()
        for rows in got:
            for k, y in rows:
                assert torch.equal(y.nan_to_num(), want[k].nan_to_num()), sizes[k // 4]
    assert pk.device_status()[0] == 0


@pytest.mark.parametrize("M,N,K", [(17, 515, 4096), (33, 130, 8192), (50, 1, 8192), (64, 515, 4096),
                                   (100, 1000, 8192), (112, 260, 4000), (144, 130, 16384),
                                   (250, 513, 8192), (256, 1024, 8192)])
def test_sums_of_a_split_that_their_owners_fetch(M, N, K):
    """Few channel tiles and long sums: K is split over a cluster, more sums than the
    memory beside the ring holds. Ragged tokens and channels, rows of outputs on and
    off 16-byte boundaries."""
    for code in CODES:
        a, sa, (wg, sg, wu, su), b = _operands(M, N, K, code, seed=3, weights=2)
        (g, eg), (u, eu) = _product64(a, sa, wg, sg), _product64(a, sa, wu, su)
        y = pk.w8a8_gemm(a, sa, wg, sg, bias=b)
        _assert_near(y, g + b.double(), eg + U * (g.abs() + b.double().abs()))
        f, t = _act64(g, "silu")
        ref = f * u
        z = pk.w8a8_gated_gemm(a, sa, wg, sg, wu, su)
        _assert_near(z, ref, 1.2 * eg * (u.abs() + eu) + f.abs() * eu +
                     (12 + 4 * (-t).clamp(0, 100)) * U * ref.abs(), 1e-5)
        if code == torch.int8:
            for dt in (torch.bfloat16, torch.float16):
                assert torch.equal(pk.w8a8_gemm(a, sa, wg, sg, bias=b, out_dtype=dt), y.to(dt))
                assert torch.equal(pk.w8a8_gated_gemm(a, sa, wg, sg, wu, su, out_dtype=dt), z.to(dt))
    assert pk.device_status() == (0, 0)


def test_split_products_beside_the_other_kernels_of_tensor_memory():
    """Clusters of 32 to 512 columns a CTA on one stream, single CTAs, pairs and the
    int4 decode kernel on others: whoever waits for another CTA of a cluster holds no
    tensor memory that a third one needs. Results as of the calls one by one."""
    g = torch.Generator(device="cuda").manual_seed(0)
    calls = [[], [], []]
    for i, (M, N, K, s) in enumerate([(1, 512, 8192, 0), (16, 384, 16384, 0), (40, 512, 8192, 0),
                                      (100, 640, 8192, 0), (144, 256, 16384, 0), (256, 512, 8192, 0),
                                      (1, 640, 16384, 1), (130, 512, 8192, 1), (300, 2048, 1024, 1),
                                      (64, 512, 4096, 1), (1000, 2000, 512, 1), (24, 1024, 4096, 1)]):
        code = CODES[i & 1]
        a, w, u = (_codes(r, K, code, g) for r in (M, N, N))
        sa, sw = (torch.rand(r, device="cuda", generator=g) / 1000 for r in (M, N))
        calls[s].append(lambda a=a, sa=sa, w=w, sw=sw: pk.w8a8_gemm(a, sa, w, sw))
        calls[s].append(lambda a=a, sa=sa, w=w, sw=sw, u=u: pk.w8a8_gated_gemm(a, sa, w, sw, u, sw))
    w4, scales = pk.quantize_int4_grouped(torch.randn(4096, 1024, device="cuda", generator=g), 128,
                                          torch.bfloat16)
    for M in (16, 32):
        x = torch.randn(M, 4096, device="cuda", generator=g).bfloat16()
        calls[2].append(lambda x=x: pk.int4_gemm(x, w4, scales, group_size=128))
    want = [[f() for f in c] for c in calls]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in calls]
    got = [[] for _ in calls]
    for turn in range(30):
        for c, stream, out in zip(calls, streams, got):
            with torch.cuda.stream(stream):
                for j in range(6):
                    k = (turn * 5 + j) % len(c)
                    out.append((k, c[k]()))
    torch.cuda.synchronize()
    for out, ref in zip(got, want):
        assert all(torch.equal(y, ref[k]) for k, y in out)
    assert pk.device_status() == (0, 0)


def _long_product64(a, sa, w, sw):
    """_product64's value, K in pieces."""
    y = sum(a[:, k:k + 65536].double() @ w[:, k:k + 65536].double().t()
            for k in range(0, a.shape[1], 65536))
    return y * (sa.double()[:, None] * sw.double())


def _long_operands(M, N, K, weights):
    g = torch.Generator(device="cuda").manual_seed(K)

    def codes(rows):
        t = torch.empty(rows, K, device="cuda", dtype=torch.float8_e4m3fn)
        for k in range(0, K, 1 << 20):
            n = min(1 << 20, K - k)
            t[:, k:k + n] = (torch.randn(rows, n, device="cuda", generator=g) * 112).clamp_(-448, 448)
        return t
    s = [(0.5 + torch.rand(n, device="cuda", generator=g)) / 112 for n in (M, N, N)]
    return codes(M), s[0], [t for i in range(weights) for t in (codes(N), s[1 + i] / K ** 0.5)]


@pytest.mark.parametrize("weights", [1, 2])
def test_long_e4m3_sums_of_many_tokens_keep_fp32_precision(weights):
    # the bound of test_long_e4m3_sums_keep_fp32_precision for more tokens than the
    # accumulators of one wide tile could hold in pieces of 5120
    a, sa, w = _long_operands(2048, 128, 600000, weights)
    ref = _long_product64(a, sa, w[0], w[1])
    if weights == 1:
        y = pk.w8a8_gemm(a, sa, *w)
    else:
        ref = _act64(ref, "silu")[0] * _long_product64(a, sa, w[2], w[3])
        y = pk.w8a8_gated_gemm(a, sa, *w)
    assert (torch.linalg.norm(y.double() - ref) <= 1e-6 * weights * torch.linalg.norm(ref)).item()


def test_the_longest_e4m3_sums_keep_16_bit_precision():
    # An output is off by half a step, 2^-11 of itself at most, and by what its
    # accumulators truncate: 1280 K tiles of 4 steps each at 4.5e-9 of the result a
    # step as measured, 2.4e-5, a twentieth of that. One accumulator for all of K
    # would truncate 2.4e-3.
    for M in (4, 130):
        a, sa, w = _long_operands(M, 64, 1 << 24, 1)
        ref = _long_product64(a, sa, *w)
        y = pk.w8a8_gemm(a, sa, *w, out_dtype=torch.float16)
        assert (torch.linalg.norm(y.double() - ref) <= 1.1 * 2.0 ** -11 * torch.linalg.norm(ref)).item()
    assert pk.device_status() == (0, 0)


def test_out_beside_and_over_operands():
    """Memory next to an operand is served, an overlap refused, on both paths."""
    M, N, K = 32, 48, 64
    a, sa, (w, sw, u, su), b = _operands(M, N, K, torch.int8, weights=2)
    sizes = [t.numel() * t.element_size() for t in (a, sa, w, sw, u, su, b)]
    pool = torch.zeros(sum(sizes) + 2 * M * N * 2, device="cuda", dtype=torch.uint8)
    views, at = [], 0
    for t, n in zip((a, sa, w, sw, u, su, b), sizes):
        views.append(pool[at:at + n].view(t.dtype).view(t.shape).copy_(t))
        at += n
    want = (pk.w8a8_gemm(a, sa, w, sw, bias=b, out_dtype=torch.bfloat16),
            pk.w8a8_gated_gemm(a, sa, w, sw, u, su, out_dtype=torch.bfloat16))
    va, vsa, vw, vsw, vu, vsu, vb = views

    def out(at):
        return pool[at:at + M * N * 2].view(torch.bfloat16).view(M, N)

    saved = _lib._tfast
    for fast in (saved, False):
        _lib._tfast = fast
        try:
            y = pk.w8a8_gemm(va, vsa, vw, vsw, bias=vb, out_dtype=torch.bfloat16, out=out(at))
            z = pk.w8a8_gated_gemm(va, vsa, vw, vsw, vu, vsu, out_dtype=torch.bfloat16,
                                   out=out(at + M * N * 2))
            assert torch.equal(y, want[0]) and torch.equal(z, want[1])
            for i in range(len(sizes)):  # ends at, or starts in, an operand's last bytes
                o = out(max(0, sum(sizes[:i + 1]) - 4))
                with pytest.raises(_lib.ShapeError):
                    pk.w8a8_gemm(va, vsa, vw, vsw, bias=vb, out_dtype=torch.bfloat16, out=o)
            with pytest.raises(_lib.ShapeError):
                pk.w8a8_gated_gemm(va, vsa, vw, vsw, vu, vsu, out_dtype=torch.bfloat16, out=out(0))
        finally:
            _lib._tfast = saved


def test_outputs_written_in_place_are_seen_by_autograd():
    """A tensor that an earlier operation saved and a call then overwrites makes that
    operation's backward an error, on both paths; inference tensors are written
    as any other."""
    a, sa, (w, sw, u, su), _ = _operands(8, 16, 32, torch.int8, weights=2)
    x, g = torch.randn(8, 64, device="cuda").bfloat16(), torch.ones(64, device="cuda")
    calls = [((8, 64), lambda o: pk.rms_norm_quant(x, g, residual=o, residual_out=o)),
             ((8, 64), lambda o: pk.rms_norm_quant(x, g, residual=x, residual_out=o)),
             ((8, 16), lambda o: pk.w8a8_gemm(a, sa, w, sw, out_dtype=torch.bfloat16, out=o)),
             ((8, 16), lambda o: pk.w8a8_gated_gemm(a, sa, w, sw, u, su, out_dtype=torch.bfloat16,
                                                    out=o))]
    saved = _lib._tfast
    for fast in (saved, False):
        _lib._tfast = fast
        try:
            for shape, call in calls:
                p = torch.randn(shape, device="cuda").bfloat16().requires_grad_()
                h = p * 1
                loss = h.square().sum()
                version = h._version
                call(h)
                assert h._version == version + 1
                with pytest.raises(RuntimeError, match="modified by an inplace operation"):
                    loss.backward()
                with torch.inference_mode():
                    buf = torch.ones(shape, device="cuda", dtype=torch.bfloat16)
                    call(buf)
                call(buf)
        finally:
            _lib._tfast = saved
