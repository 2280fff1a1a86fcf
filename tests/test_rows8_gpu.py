"""8-bit rows on the GPU: quantize_rows, dequantize_rows and rms_norm_quant
against their definitions in 64 bits.

Tolerances count roundings, each half a step (fp32 2^-24 relative):

* a scale a / most: one rounding. The norm's scale also carries r = 1 /
  sqrt(mean + eps): the sum of K squares in fp32 has at most a chain of
  `chain` additions (a thread's values, then the tree), half of whose error
  survives the square root, and seven more roundings;
* a code: the quotient t = y / scale is within |t| * 2^-24 * (roundings on its
  way) of the fp32 one that is rounded: 3 for the quantizer, 8 for the norm
  (r cancels in it). So |code - t| <= half a step of the code + that.
"""

import pytest
import torch

import pico_kernels_b200 as pk
from pico_kernels_b200 import _lib

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
CODES = [torch.int8, torch.float8_e4m3fn]
TYPES = [torch.bfloat16, torch.float16, torch.float32]
# one column, below and at a chunk, a warp's row and past it, odd widths, the
# widest held row (32768) and one past it
WIDTHS = [1, 7, 8, 31, 128, 1000, 1024, 1032, 4096, 5001, 8192, 16392, 32768, 33000]


def _x(rows, cols, dt, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(rows, cols, device="cuda", generator=g)
    return (x * torch.exp(2 * torch.randn(rows, 1, device="cuda", generator=g))).to(dt)


def _check_codes(q, scale, y, roundings, scale_tol):
    """codes and scale of the fp64 rows y."""
    most = 127.0 if q.dtype == torch.int8 else 448.0
    s = y.abs().amax(-1).clamp_min(1e-12) / most
    assert scale.dtype == torch.float32 and scale.shape == y.shape[:-1]
    assert ((scale.double() - s).abs() <= scale_tol * s).all()
    t = y / s[..., None]
    v = q.double()
    half = torch.full_like(t, 0.5) if q.dtype == torch.int8 else \
        torch.clamp(t.abs() * 2.0 ** -4, min=2.0 ** -10)
    # the oracle's scale against the exact one costs a rounding of t as well
    assert ((v - t).abs() <= half + t.abs() * (roundings + 1) * U).all()
    assert v.abs().max() <= most


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("cols", WIDTHS)
def test_quantize_rows(cols, dt, code):
    for rows in (1, 3, 200):
        x = _x(rows, cols, dt, seed=rows)
        q, s = pk.quantize_rows(x, code)
        assert q.shape == x.shape and q.dtype == code
        assert rows == 1 or q.stride(0) == (cols + 15) // 16 * 16
        _check_codes(q, s, x.double(), 3, U)
        # the same bits on a second run and on rows of another batch
        q2, s2 = pk.quantize_rows(x[-1:].clone(), code)
        assert torch.equal(q2.view(torch.uint8)[0], q.view(torch.uint8)[-1])
        assert torch.equal(s2[0], s[-1])


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("out", TYPES)
@pytest.mark.parametrize("rows,cols", [(1, 1), (5, 16), (3, 17), (200, 1000), (70, 5001)])
def test_dequantize_rows(rows, cols, out, code):
    q, s = pk.quantize_rows(_x(rows, cols, torch.float32), code)
    y = pk.dequantize_rows(q, s, out)
    assert y.is_contiguous()
    assert torch.equal(y, (q.float() * s[:, None]).to(out))  # one product, one rounding
    assert torch.equal(pk.dequantize_rows(q, s[:, None], out), y)


def _norm64(h, w, eps):
    h = h.double()
    return h / torch.sqrt(h.square().mean(-1, keepdim=True) + eps) * w.double()


@pytest.mark.parametrize("residual", [True, False])
@pytest.mark.parametrize("dt,wt", [(torch.bfloat16, torch.bfloat16), (torch.bfloat16, torch.float32),
                                   (torch.float16, torch.float16), (torch.float32, torch.float32)])
@pytest.mark.parametrize("cols", WIDTHS)
def test_rms_norm_quant(cols, dt, wt, residual):
    g = torch.Generator(device="cuda").manual_seed(cols)
    w = (1 + 0.3 * torch.randn(cols, device="cuda", generator=g)).to(wt)
    chain = max(64, cols // 1024) + 16
    for rows, code in ((1, torch.int8), (3, torch.float8_e4m3fn), (200, torch.int8)):
        x = _x(rows, cols, dt, seed=rows)
        if residual:
            r = _x(rows, cols, dt, seed=rows + 50)
            q, s, h = pk.rms_norm_quant(x, w, 1e-5, residual=r, dtype=code)
            assert torch.equal(h, (x.float() + r.float()).to(dt))
        else:
            q, s = pk.rms_norm_quant(x, w, 1e-5, dtype=code)
            h = x
        _check_codes(q, s, _norm64(h, w, 1e-5), 8, (chain / 2 + 8) * U)
        # the same bits for a row in another batch
        alone = pk.rms_norm_quant(h[-1:].clone(), w, 1e-5, dtype=code)
        assert torch.equal(alone[1][0], s[-1])
        assert torch.equal(alone[0].view(torch.uint8)[0], q.view(torch.uint8)[-1])


def test_rows_of_zeros_and_tiny_rows():
    x = torch.zeros(3, 100, device="cuda")
    x[1] = 1e-20
    x[2] = 1e-12
    for code in CODES:
        q, s = pk.quantize_rows(x, code)
        most = 127.0 if code == torch.int8 else 448.0
        assert torch.equal(s, torch.full((3,), 1e-12, device="cuda") / most)
        assert q.float()[0].abs().max() == 0 and q.float()[1].abs().max() <= 2.0 ** -9
        assert (q.float()[2] == most).all()
        q, s = pk.rms_norm_quant(x, torch.ones(100, device="cuda"), dtype=code)
        assert q.float()[0].abs().max() == 0 and torch.isfinite(s).all()


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("cols", [100, 1001, 4096, 33000])
def test_a_row_with_a_nan_or_infinity_poisons_only_itself(cols, bad):
    x = _x(5, cols, torch.bfloat16)
    w = torch.ones(cols, device="cuda", dtype=torch.bfloat16)
    y = x.clone()
    y[2, cols // 2] = bad
    for code in CODES:
        for clean, dirty in ((pk.quantize_rows(x, code), pk.quantize_rows(y, code)),
                             (pk.rms_norm_quant(x, w, dtype=code),
                              pk.rms_norm_quant(y, w, dtype=code))):
            keep = [0, 1, 3, 4]
            assert torch.isnan(dirty[1][2]) and dirty[0].float()[2].abs().max() == 0
            assert torch.equal(dirty[1][keep], clean[1][keep])
            assert torch.equal(dirty[0].float()[keep], clean[0].float()[keep])
            assert torch.isnan(pk.dequantize_rows(*dirty)[2]).all()


@pytest.mark.parametrize("cols", [64, 1001, 8192, 33000])
def test_norm_of_values_whose_squares_leave_fp32(cols):
    x = _x(4, cols, torch.float32)
    x = x / x.abs().amax(-1, keepdim=True)
    w = torch.ones(cols, device="cuda")
    big = x * 2.0 ** 100
    q, s = pk.rms_norm_quant(big, w, 1e-6)
    _check_codes(q, s, _norm64(big, w, 1e-6), 8, (max(64, cols // 1024) / 2 + 16) * U)
    q, s = pk.rms_norm_quant(x * 2.0 ** -90, w, 2.0 ** -126)  # and below it: eps (the least) carries the sum
    assert torch.isfinite(s).all()


def test_strided_and_batched_rows():
    base = _x(40, 300, torch.bfloat16).reshape(4, 10, 300)
    w = torch.rand(256, device="cuda").bfloat16()
    for x in (base[..., 8:264],               # rows apart by 300, 16 bytes in
              base[..., 3:259],               # unaligned rows
              base.transpose(0, 1)[..., :256],  # rows no single distance describes
              base.transpose(1, 2)[:, :256, :].contiguous().transpose(1, 2),
              base[:1, :1, :256].expand(4, 10, 256)):
        c = x.contiguous()
        for a, b in zip(pk.quantize_rows(x), pk.quantize_rows(c)):
            assert a.shape == b.shape and torch.equal(a, b)
        for a, b in zip(pk.rms_norm_quant(x, w, residual=x), pk.rms_norm_quant(c, w, residual=c)):
            assert a.shape == b.shape and torch.equal(a, b)
    q, s = pk.quantize_rows(base.contiguous())
    assert s.shape == (4, 10)
    assert torch.equal(pk.dequantize_rows(q[:, ::2], s[:, ::2]), pk.dequantize_rows(q, s)[:, ::2])
    assert torch.equal(pk.dequantize_rows(q[1, :, 5:], s[1]), pk.dequantize_rows(q, s)[1, :, 5:])


def test_no_rows_and_vectors():
    for shape in ((0, 64), (3, 0, 64)):
        x = torch.zeros(shape, device="cuda", dtype=torch.bfloat16)
        q, s = pk.quantize_rows(x)
        assert q.shape == shape and s.shape == shape[:-1]
        assert pk.dequantize_rows(q, s).shape == shape
        q, s, h = pk.rms_norm_quant(x, torch.ones(64, device="cuda"), residual=x)
        assert q.shape == h.shape == shape
    v = _x(1, 77, torch.float16)[0]
    q, s = pk.quantize_rows(v)
    assert q.shape == (77,) and s.shape == ()
    assert torch.equal(pk.dequantize_rows(q, s), q.float() * s)


def test_residual_updated_in_place():
    w = torch.rand(512, device="cuda").bfloat16()
    x, r = _x(9, 512, torch.bfloat16, 1), _x(9, 512, torch.bfloat16, 2)
    q, s, h = pk.rms_norm_quant(x, w, residual=r)
    for target in ("x", "residual", "own"):
        x2, r2 = x.clone(), r.clone()
        o = {"x": x2, "residual": r2, "own": torch.empty_like(x)}[target]
        q2, s2, h2 = pk.rms_norm_quant(x2, w, residual=r2, residual_out=o)
        assert h2 is o and torch.equal(h2, h) and torch.equal(q2, q) and torch.equal(s2, s)
    buf = torch.zeros(10 * 512, device="cuda", dtype=torch.bfloat16)
    with pytest.raises(_lib.ShapeError):  # shifted by a row: each row would overwrite the next
        pk.rms_norm_quant(buf[:9 * 512].view(9, 512), w, residual=r,
                          residual_out=buf[512:].view(9, 512))


def test_columns_past_the_row_are_left_alone():
    lib = _lib.load()
    x = _x(6, 100, torch.bfloat16)
    q = torch.full((6, 128), 99, device="cuda", dtype=torch.int8)
    s = torch.full((7,), -1.0, device="cuda")
    assert lib.pk_quantize_rows(x.data_ptr(), _lib.PK_BF16, 6, 100, 100, q.data_ptr(), _lib.PK_I8,
                                128, s.data_ptr(), _lib.stream_of(x)) == _lib.PK_OK
    assert (q[:, 100:] == 99).all() and s[6] == -1
    out = torch.full((6, 120), 7.0, device="cuda")
    assert lib.pk_dequantize_rows(q.data_ptr(), _lib.PK_I8, 5, 100, 128, s.data_ptr(),
                                  out.data_ptr(), _lib.PK_F32, 120, _lib.stream_of(x)) == _lib.PK_OK
    assert (out[:, 100:] == 7).all() and (out[5] == 7).all()


def test_offsets_past_31_bits():
    rows, cols = 66000, 32768  # 2.16e9 values
    x = torch.zeros(rows, cols, device="cuda", dtype=torch.bfloat16)
    tail = _x(3, cols, torch.bfloat16)
    x[-3:] = tail
    w = torch.ones(cols, device="cuda", dtype=torch.bfloat16)
    q, s = pk.quantize_rows(x)
    qt, st = pk.quantize_rows(tail)
    assert torch.equal(q[-3:], qt) and torch.equal(s[-3:], st)
    assert torch.equal(pk.dequantize_rows(q, s, torch.bfloat16)[-3:],
                       pk.dequantize_rows(qt, st, torch.bfloat16))
    del q
    q, s, h = pk.rms_norm_quant(x, w, residual=x, residual_out=x)
    qt, st, ht = pk.rms_norm_quant(tail, w, residual=tail)
    assert torch.equal(q[-3:], qt) and torch.equal(s[-3:], st) and torch.equal(h[-3:], ht)


def test_fast_path_equals_python_path():
    assert _lib.torch_fast() is not None
    x, r = _x(33, 1000, torch.bfloat16, 3), _x(33, 1000, torch.bfloat16, 4)
    w = torch.rand(1000, device="cuda")
    calls = [lambda: pk.quantize_rows(x, torch.float8_e4m3fn),
             lambda: pk.rms_norm_quant(x, w, 1e-6, residual=r),
             lambda: (pk.dequantize_rows(*pk.quantize_rows(x)),)]
    fast = [f() for f in calls]
    saved = _lib._tfast
    _lib._tfast = False
    try:
        slow = [f() for f in calls]
    finally:
        _lib._tfast = saved
    for a, b in zip(fast, slow):
        assert len(a) == len(b)
        for t, u in zip(a, b):
            assert t.dtype == u.dtype and t.stride() == u.stride()
            assert torch.equal(t.float(), u.float())
    assert type(_lib.torch_fast().quantize_rows(x, torch.int8)) is tuple  # served, not refused
    assert type(_lib.torch_fast().rms_norm_quant(x, w, 1e-6, r, torch.int8, None)) is tuple
    assert pk.device_status() == (0, 0)


def test_captured_and_replayed_on_another_stream():
    x, r = _x(16, 2048, torch.bfloat16, 1), _x(16, 2048, torch.bfloat16, 2)
    w = torch.rand(2048, device="cuda").bfloat16()

    def step():
        q, s, h = pk.rms_norm_quant(x, w, residual=r)
        return q, s, h, pk.dequantize_rows(q, s, torch.bfloat16)

    step()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        out = step()
    x.copy_(_x(16, 2048, torch.bfloat16, 9))
    for _ in range(2):
        g.replay()
    torch.cuda.synchronize()
    for a, b in zip(out, step()):
        assert torch.equal(a, b)


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("cols", [20, 100, 200, 256, 400, 512])
def test_rows_that_share_a_warp(cols, code):
    """Rows of up to 512 columns share a warp: large ones, which the norm goes over
    twice, and one with a NaN leave their neighbours' bits alone."""
    x = _x(37, cols, torch.float32, seed=cols)
    x = x / x.abs().amax(-1, keepdim=True)
    x[::3] *= 2.0 ** 100
    x[5, cols // 3] = float("nan")
    r = x * 0.25
    w = 1 + 0.3 * torch.randn(cols, device="cuda", generator=torch.Generator("cuda").manual_seed(1))
    q, s = pk.rms_norm_quant(x, w, 1e-5, dtype=code)
    qr, sr, h = pk.rms_norm_quant(x, w, 1e-5, residual=r, dtype=code)
    good = [i for i in range(37) if i != 5]
    assert torch.equal(h[good], (x + r)[good])
    for y, a, b in ((x, q, s), (h, qr, sr)):
        assert torch.isnan(b[5]) and a.float()[5].abs().max() == 0
        _check_codes(a[good], b[good], _norm64(y[good], w, 1e-5), 8, (80 / 2 + 8) * U)
    for i in (0, 4, 6, 7, 36):
        a, b = pk.rms_norm_quant(x[i:i + 1].clone(), w, 1e-5, dtype=code)
        assert torch.equal(a.view(torch.uint8)[0], q.view(torch.uint8)[i]) and b[0] == s[i]
    q, s = pk.quantize_rows(x, code)
    assert torch.isnan(s[5]) and q.float()[5].abs().max() == 0
    _check_codes(q[good], s[good], x[good].double(), 3, U)


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("cols", [2, 9, 33, 250, 255, 1001, 1003, 2047, 5001])
def test_residual_streams_of_odd_width(cols, dt):
    """Rows off 16-byte boundaries: h is stored in blocks that span two threads'
    chunks, in place as well, and in a tensor that starts at any element."""
    x, r = _x(67, cols, dt, seed=cols), _x(67, cols, dt, seed=cols + 1)
    w = torch.ones(cols, device="cuda")
    want = (x.float() + r.float()).to(dt)
    q, s, h = pk.rms_norm_quant(x, w, residual=r)
    assert torch.equal(h, want)
    for shift in (0, 1, 3):
        flat = torch.full((67 * cols + 8,), 5.0, device="cuda", dtype=dt)
        out = flat[shift:shift + 67 * cols].view(67, cols)
        out.copy_(r)
        q2, s2, h2 = pk.rms_norm_quant(x, w, residual=out, residual_out=out)
        assert h2.data_ptr() == out.data_ptr() and torch.equal(out, want)
        assert (flat[:shift] == 5).all() and (flat[shift + 67 * cols:] == 5).all()
        assert torch.equal(q, q2) and torch.equal(s, s2)


def _tie_rows(code, dt, cols, g):
    """Rows with a largest value of 7 k 2^j (e4m3) or 127 2^j (int8), for which a
    row's half steps are numbers of its type: most / max then has no short form."""
    rows = []
    for i in range(24):
        if code == torch.int8:
            k, top = 1, 127
            v = torch.randint(-127, 127, (cols,), device="cuda", generator=g) + 0.5
        else:
            k, top = (1, 3, 5, 7)[i % 4], 448
            m = torch.randint(8, 16, (cols,), device="cuda", generator=g) + 0.5
            e = torch.randint(-6, 5, (cols,), device="cuda", generator=g)
            v = m * torch.exp2(e.float()) * (1 - 2 * torch.randint(0, 2, (cols,), device="cuda", generator=g))
        v = (v * k).clamp(-top * k, top * k)
        v[i % cols] = top * k
        rows.append(v * 2.0 ** (i // 4 - 8))
    x = torch.stack(rows)
    assert torch.equal(x.to(dt).float(), x)
    return x.to(dt)


def _nearest_codes(u, code):
    """Rows in 64 bits to their codes: u * most / max|u|, half steps to even."""
    most = 127.0 if code == torch.int8 else 448.0
    t = u * most / u.abs().amax(-1, keepdim=True)
    if code == torch.int8:
        return t.round()
    step = torch.exp2(torch.floor(torch.log2(t.abs().clamp_min(2.0 ** -6))) - 3)
    return (t / step).round() * step


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("cols", [1, 9, 100, 1000, 1001, 4096, 16392, 33000])
def test_codes_of_16_bit_rows_are_the_nearest(cols, dt, code):
    """Exactly: u and max|u| have at most 11 bits, so a quotient u * most / max|u| that
    is no half step lies at least 2^-20 of its size away from one, and 64 bits
    (2^-52) and the kernel's fp32 (2^-24) round it alike; a half step goes to even."""
    g = torch.Generator(device="cuda").manual_seed(cols)
    for x in (_tie_rows(code, dt, cols, g), _x(200, cols, dt, seed=cols)):
        q = pk.quantize_rows(x, code)[0]
        assert torch.equal(q.double(), _nearest_codes(x.double(), code))


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("residual", [True, False])
@pytest.mark.parametrize("cols", [1, 9, 100, 1000, 1001, 4096, 16392, 33000])
def test_codes_of_bf16_norms_are_the_nearest(cols, residual, code):
    """r = 1 / sqrt(mean + eps) multiplies the whole row, so the codes are those of
    h * w, which fp32 holds exactly (16 bits). A quotient that is no half step is
    off one by at least 1 / (2 * 2^16) of a row maximum of 127 (int8; farther in
    e4m3), 2^-24 of its size, which fp32 tells apart."""
    g = torch.Generator(device="cuda").manual_seed(cols)
    one = torch.ones(cols, device="cuda", dtype=torch.bfloat16)
    for x, w in ((_tie_rows(code, torch.bfloat16, cols, g), one),
                 (_x(200, cols, torch.bfloat16, seed=cols),
                  (1 + 0.3 * torch.randn(cols, device="cuda", generator=g)).bfloat16())):
        r = torch.zeros_like(x) if residual else None
        q = pk.rms_norm_quant(x, w, 1e-5, residual=r, dtype=code)[0]
        assert torch.equal(q.double(), _nearest_codes(x.double() * w.double(), code))


@pytest.fixture(scope="module")
def far_buffer():
    yield torch.zeros((1 << 32) + (1 << 18), device="cuda", dtype=torch.uint8)


def _far(buf, x):
    """x's two rows 4 GiB apart."""
    n = (1 << 32) // x.element_size()
    y = torch.as_strided(buf.view(x.dtype), x.shape, (n, 1))
    y.copy_(x)
    return y


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("cols", [1, 7, 20, 100, 128, 129, 300, 512, 1000, 1024, 1032, 2047, 4096,
                                  5001, 8192, 16384, 16385])
def test_rows_gigabytes_apart(cols, dt, far_buffer):
    """The bits of the same rows side by side: codes, scales and sums do not depend
    on strides, whichever kernel a distance needs."""
    x = _x(2, cols, dt, seed=cols)
    w = 1 + 0.3 * torch.randn(cols, device="cuda", generator=torch.Generator("cuda").manual_seed(2))
    for big in ((1.0, 2.0 ** 80) if dt != torch.float16 else (1.0,)):  # squares in and past fp32
        x = torch.stack((x[0], (x[1].float() * big).to(dt)))
        r = (x * 0.5).flip(1)
        for code in CODES:
            want = (pk.quantize_rows(x, code), pk.rms_norm_quant(x, w, dtype=code),
                    pk.rms_norm_quant(x, w, residual=r, dtype=code),
                    pk.rms_norm_quant(r, w, residual=x, dtype=code))
            y = _far(far_buffer, x)
            got = (pk.quantize_rows(y, code), pk.rms_norm_quant(y, w, dtype=code),
                   pk.rms_norm_quant(y, w, residual=r, dtype=code),
                   pk.rms_norm_quant(r, w, residual=y, dtype=code))
            for a, b in zip(want, got):
                for s, t in zip(a, b):
                    assert torch.equal(s.float(), t.float())
            q, s = want[0]
            assert torch.equal(pk.dequantize_rows(_far(far_buffer, q), s), pk.dequantize_rows(q, s))


@pytest.mark.parametrize("residual", [True, False])
@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("cols", [16376, 16383, 16384, 16385])
def test_rows_around_the_widest_that_threads_hold(cols, dt, residual):
    w = 1 + 0.3 * torch.randn(cols, device="cuda", generator=torch.Generator("cuda").manual_seed(3))
    for rows, code in ((1, torch.int8), (5, torch.float8_e4m3fn), (300, torch.int8)):
        x = _x(rows, cols, dt, seed=rows)
        q, s = pk.quantize_rows(x, code)
        _check_codes(q, s, x.double(), 3, U)
        h = x
        if residual:
            r = _x(rows, cols, dt, seed=rows + 7)
            q, s, h = pk.rms_norm_quant(x, w, 1e-5, residual=r, dtype=code)
            assert torch.equal(h, (x.float() + r.float()).to(dt))
        else:
            q, s = pk.rms_norm_quant(x, w, 1e-5, dtype=code)
        _check_codes(q, s, _norm64(h, w, 1e-5), 8, (80 / 2 + 8) * U)


@pytest.mark.parametrize("residual", [True, False])
@pytest.mark.parametrize("cols", [20, 64, 1001, 8192, 33000])
def test_norm_of_products_past_fp32(cols, residual):
    """h * w past fp32's range where h * r * w is not: the row's own sum and eps
    count, whatever is done to reach the product."""
    x = (_x(5, cols, torch.float32) * 0 + 1) * torch.linspace(-1, 1, cols, device="cuda") + 2.0
    w = torch.linspace(0.5, 1, cols, device="cuda")
    tol = (max(64, cols // 1024) / 2 + 16) * U
    for size, weight, eps in ((1e3, 1e36, 1e-6), (1e3, 1e36, 1e6), (1.0, 2e38, 1e-6), (2.0 ** 65, 1.0, 2.0 ** 127),
                              (2.0 ** 65, 1e30, 2.0 ** 127), (2.0 ** 100, 1e20, 1e-6)):
        h = x * size
        v = w * weight
        if residual:
            q, s, got = pk.rms_norm_quant(h * 0.5, v, eps, residual=h * 0.5)
            assert torch.equal(got, h)
        else:
            q, s = pk.rms_norm_quant(h, v, eps)
        _check_codes(q, s, _norm64(h, v, eps), 8, tol)


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
def test_a_nan_or_infinity_at_either_place_of_a_packed_pair(dt, bad):
    x = _x(6, 20000, dt)
    clean = pk.quantize_rows(x)
    for at in (0, 1, 7, 4098, 19998, 19999):
        y = x.clone()
        y[3, at] = bad
        y[1, at] = -y[1].abs().max() * 2  # the largest, with a sign
        q, s = pk.quantize_rows(y)
        assert torch.isnan(s[3]) and q[3].abs().max() == 0
        most = -y[1, at].item() / 127
        assert abs(s[1].item() - most) <= U * most and q[1, at] == -127
        for i in (0, 2, 4, 5):
            assert torch.equal(q[i], clean[0][i]) and s[i] == clean[1][i]
