"""Cases of the 8-bit (W8A8) operators: what a quantized transformer block runs
around its matrix products when weights and activations are both held in 8
bits with one scale per row.

* ``quantize_rows`` / ``dequantize_rows``: ``x[M, K]`` to int8 or e4m3 codes
  with one fp32 scale per row, and back;
* ``rms_norm_quant``: the residual's addition, the root-mean-square norm and
  the 8-bit output of the next product in one pass;
* ``w8a8_gemm``: ``(A8 @ W8^T) * a_scale[m] * w_scale[n] (+ bias[n])``;
* ``w8a8_gated_gemm``: ``act(gate) * up`` of two such products.

``run`` is their plain form in elementary torch operations where ``own`` is
false, and the framework's calls where it is true. 8-bit weights and
activations are [rows, K] with K contiguous and rows a multiple of 16 bytes
apart, as ``quantize_rows`` writes them.
"""

import torch

own = False

_BF16, _F16, _F32 = "bfloat16", "float16", "float32"
_I8, _E4M3 = "int8", "float8_e4m3fn"
_EPS = 1e-6
_MOST_FLOPS = 2 * 2 * 4096 * 4096 * 11008
_MOST_VALUES = 4096 * 28672


def listed():
    return [
        # one token through a 4096-wide attention projection: launch latency and a 17 MB weight stream
        {"name": "gemm_decode", "op": "gemm", "M": 1, "N": 4096, "K": 4096, "code": _I8, "out": _BF16, "bias": False},
        # 16 sequences, one token each, through a 70B-sized down projection
        {"name": "gemm_decode_wide", "op": "gemm", "M": 16, "N": 8192, "K": 28672, "code": _E4M3, "out": _F32, "bias": False},
        # a short ragged batch through a layer with odd sizes and a bias
        {"name": "gemm_ragged", "op": "gemm", "M": 333, "N": 1111, "K": 1001, "code": _I8, "out": _F16, "bias": True},
        # a 4096-token prompt through the up projection of a 7B model
        {"name": "gemm_prefill", "op": "gemm", "M": 4096, "N": 11008, "K": 4096, "code": _I8, "out": _BF16, "bias": False},
        # one token through the two input projections of a 70B-sized gated block: a 470 MB weight stream
        {"name": "gated_decode", "op": "gated", "M": 1, "N": 28672, "K": 8192, "code": _I8, "out": _BF16, "act": "silu"},
        # a mixed batch (a few prompts' last chunks and single tokens) through a 7B block with a GELU gate
        {"name": "gated_batch", "op": "gated", "M": 200, "N": 11008, "K": 4096, "code": _I8, "out": _F16, "act": "gelu_tanh"},
        # a 4096-token prompt through the gated block of a 7B model
        {"name": "gated_prefill", "op": "gated", "M": 4096, "N": 11008, "K": 4096, "code": _E4M3, "out": _BF16, "act": "silu"},
        # the norm before one token's projections: latency alone; its codes are read back as values
        {"name": "norm_decode", "op": "norm", "M": 1, "K": 4096, "x": _BF16, "w": _BF16, "code": _I8, "residual": True},
        # the norm of a 4096-token prompt in a 70B-sized block
        {"name": "norm_prefill", "op": "norm", "M": 4096, "K": 8192, "x": _BF16, "w": _BF16, "code": _E4M3, "residual": True},
        # an odd width without a residual (a first layer), fp32 norm weights; codes read back as values
        {"name": "norm_ragged", "op": "norm", "M": 1000, "K": 5001, "x": _F16, "w": _F32, "code": _I8, "residual": False},
        # the activations of a 4096-token prompt before a 70B-sized down projection
        {"name": "rows_prefill", "op": "rows", "M": 4096, "K": 28672, "x": _BF16, "code": _E4M3},
        # weights or activations of odd width in fp32, quantized and read back
        {"name": "rows_ragged", "op": "rows", "M": 77, "K": 11007, "x": _F32, "code": _I8},
    ]


def _log(rng, lo, hi):
    """A whole number between lo and hi, uniform in its logarithm; often a multiple of a tile size, often odd."""
    v = max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))
    if rng.random() < 0.5:
        for m in (128, 64, 32, 16):
            if v >= 2 * m:
                return v // m * m
    return v


def draw(rng):
    op = rng.choice(["gemm", "gated", "norm", "rows"])
    code = rng.choice([_I8, _E4M3])
    if op in ("gemm", "gated"):
        while True:
            c = {"op": op, "M": _log(rng, 1, 8192), "N": _log(rng, 32, 28672), "K": _log(rng, 64, 28672), "code": code,
                 "out": rng.choice([_BF16, _BF16, _F16, _F32])}
            if (2 if op == "gemm" else 4) * c["M"] * c["N"] * c["K"] <= _MOST_FLOPS and c["N"] * c["K"] <= 28672 * 8192:
                break
        return {**c, "bias": rng.random() < 0.5} if op == "gemm" else {**c, "act": rng.choice(["silu", "gelu_tanh"])}
    while True:
        c = {"op": op, "M": _log(rng, 1, 16384), "K": _log(rng, 32, 32768), "x": rng.choice([_BF16, _BF16, _F16, _F32]), "code": code}
        if c["M"] * c["K"] <= _MOST_VALUES:
            break
    if op == "norm":
        c["w"] = rng.choice([c["x"], _F32])
        c["residual"] = rng.random() < 0.7
    return c


def _dt(name):
    return getattr(torch, name)


def _codes(rows, cols, code, gen):
    """8-bit codes of rows that were scaled to their own largest value: [rows, cols], rows a multiple of 16 bytes apart."""
    pitch = (cols + 15) // 16 * 16
    q = torch.empty((rows, pitch), dtype=_dt(code), device="cuda")
    most = 127 if code == _I8 else 448
    step = max(1, (1 << 26) // pitch)
    for r in range(0, rows, step):
        v = torch.randn((min(step, rows - r), pitch), device="cuda", generator=gen) * (most / 4.2)
        q[r:r + step] = (v.round_() if code == _I8 else v).clamp_(-most, most).to(_dt(code))
    return q[:, :cols]


def _activations(rows, cols, dtype, gen):
    """A residual stream: most channels near one, a few larger ones, as language models have them."""
    big = torch.exp(0.5 * torch.randn(cols, device="cuda", generator=gen))
    big[torch.randint(0, cols, (max(1, cols // 512),), device="cuda", generator=gen)] *= 12.0
    return (torch.randn((rows, cols), device="cuda", generator=gen) * big).to(_dt(dtype))


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    s = dict(case)
    if case["op"] in ("gemm", "gated"):
        M, N, K = case["M"], case["N"], case["K"]
        most = 127.0 if case["code"] == _I8 else 448.0
        weight_scale = 4.2 * K ** -0.5 / most * 1.5
        s["a8"] = _codes(M, K, case["code"], gen)
        s["a_scale"] = (0.5 + torch.rand(M, device="cuda", generator=gen)) * (4.2 / most)
        for name in ("w",) if case["op"] == "gemm" else ("gate", "up"):
            s[name + "8"] = _codes(N, K, case["code"], gen)
            s[name + "_scale"] = (0.5 + torch.rand(N, device="cuda", generator=gen)) * weight_scale
        s["b"] = torch.randn(N, device="cuda", generator=gen) if case.get("bias") else None
        return s
    s["x_"] = _activations(case["M"], case["K"], case["x"], gen)
    if case["op"] == "norm":
        s["w_"] = (1 + 0.2 * torch.randn(case["K"], device="cuda", generator=gen)).to(_dt(case["w"]))
        s["r_"] = _activations(case["M"], case["K"], case["x"], gen) if case["residual"] else None
    return s


# ---------------------------------------------------------------- plain forms


def _plain_quantize(y, code):
    """fp32 rows to (the codes' values before scaling, scales): scale = max|y| / most, code = round(y / scale)."""
    most = 127.0 if code == _I8 else 448.0
    a = y.abs().amax(-1, keepdim=True).clamp_min(1e-12)
    t = y * (most / a)
    q = t.round().clamp(-most, most) if code == _I8 else t.clamp(-most, most).to(torch.float8_e4m3fn)
    return q, (a / most).squeeze(-1)


def _read_dtype(case):
    """int8 codes are read back in the input's 16-bit type (bf16 for an fp32 input)."""
    return torch.bfloat16 if case["x"] == _F32 else _dt(case["x"])


def _plain_product(s, name):
    return (s["a8"].float() @ s[name + "8"].float().t()) * s["a_scale"][:, None] * s[name + "_scale"]


def _plain(s):
    if s["op"] == "gemm":
        y = _plain_product(s, "w")
        return (y if s["b"] is None else y + s["b"]).to(_dt(s["out"]))
    if s["op"] == "gated":
        g, u = _plain_product(s, "gate"), _plain_product(s, "up")
        t = g if s["act"] == "silu" else 1.5957691216057308 * (g + 0.044715 * g * g * g)
        return (g / (1 + torch.exp(-t)) * u).to(_dt(s["out"]))
    h = None
    y = s["x_"].float()
    if s["op"] == "norm":
        if s["residual"]:
            h = (y + s["r_"].float()).to(_dt(s["x"]))  # the residual stream's own type: what the next block adds to
            y = h.float()
        y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + _EPS) * s["w_"].float()
    q, scale = _plain_quantize(y, s["code"])
    if s["code"] == _I8:
        q = (q * scale[:, None]).to(_read_dtype(s))
    return {"q": q, "scale": scale, "h": h}


# ---------------------------------------------------------- the framework's calls

_pk = None


def _own(s):
    global _pk
    if _pk is None:
        import pico_kernels_b200
        _pk = pico_kernels_b200
    if s["op"] == "gemm":
        return _pk.w8a8_gemm(s["a8"], s["a_scale"], s["w8"], s["w_scale"], bias=s["b"], out_dtype=_dt(s["out"]))
    if s["op"] == "gated":
        return _pk.w8a8_gated_gemm(s["a8"], s["a_scale"], s["gate8"], s["gate_scale"], s["up8"], s["up_scale"],
                                   activation=s["act"], out_dtype=_dt(s["out"]))
    h = None
    if s["op"] == "norm" and s["residual"]:
        q, scale, h = _pk.rms_norm_quant(s["x_"], s["w_"], _EPS, residual=s["r_"], dtype=_dt(s["code"]))
    elif s["op"] == "norm":
        q, scale = _pk.rms_norm_quant(s["x_"], s["w_"], _EPS, dtype=_dt(s["code"]))
    else:
        q, scale = _pk.quantize_rows(s["x_"], _dt(s["code"]))
    if s["code"] == _I8:
        q = _pk.dequantize_rows(q, scale, _read_dtype(s))
    return {"q": q, "scale": scale, "h": h}


def run(state):
    return _own(state) if own else _plain(state)


def work(case):
    """Bytes: inputs once, outputs once. int8 codes that are read back count as written, read, and written as 16-bit values."""
    M, K = case["M"], case["K"]
    if case["op"] in ("gemm", "gated"):
        n = 1 if case["op"] == "gemm" else 2
        N, o = case["N"], 4 if case["out"] == _F32 else 2
        return {"bytes": M * K + 4 * M + n * N * (K + 4) + (4 * N if case.get("bias") else 0) + M * N * o,
                "flops": 2 * n * M * N * K}
    e = 4 if case["x"] == _F32 else 2
    b = M * K * (e + 1) + 4 * M
    if case["code"] == _I8:
        b += M * K * 3
    if case["op"] == "norm":
        b += K * (4 if case["w"] == _F32 else 2) + (2 * M * K * e if case["residual"] else 0)
    return {"bytes": b, "flops": M * K * (8 if case["op"] == "norm" else 4)}


def exact(case, seed):
    """The operators' definitions in 64 bits."""
    s = prepare(case, seed)
    if case["op"] in ("gemm", "gated"):
        def product(codes, scales):
            y = torch.empty((case["M"], case["N"]), dtype=torch.float64, device="cuda")
            a = s["a8"].double().mul_(s["a_scale"].double().unsqueeze(1))
            for n in range(0, case["N"], 4096):
                w = codes[n:n + 4096].double() * scales[n:n + 4096].double().unsqueeze(1)
                y[:, n:n + 4096] = torch.einsum("mk,nk->mn", a, w)
            return y
        if case["op"] == "gemm":
            y = product(s["w8"], s["w_scale"])
            return y if s["b"] is None else y + s["b"].double().unsqueeze(0)
        g, u = product(s["gate8"], s["gate_scale"]), product(s["up8"], s["up_scale"])
        if case["act"] == "silu":
            return u * g * torch.special.expit(g)
        return u * g * 0.5 * (1 + torch.tanh((2 / torch.pi) ** 0.5 * (g + 0.044715 * g ** 3)))
    h, y = None, s["x_"].double()
    if case["op"] == "norm":
        if case["residual"]:
            # the sum is rounded to the stream's type by definition: the norm is that of the stored sum
            h = (y + s["r_"].double()).to(_dt(case["x"])).double()
            y = h
        y = y / torch.sqrt(y.square().sum(-1, keepdim=True) / case["K"] + _EPS) * s["w_"].double()
    top = 127.0 if case["code"] == _I8 else 448.0
    scale = torch.clamp(torch.linalg.vector_norm(y, float("inf"), dim=-1), min=1e-12) / top
    q = y / scale.unsqueeze(1)
    if case["code"] == _I8:
        q = torch.round(q) * scale.unsqueeze(1)
    else:
        # e4m3 by its definition: 3 bits after the leading one, steps of 2^-9 below 2^-6, ties to even
        step = torch.exp2(torch.floor(torch.log2(q.abs().clamp_min(2.0 ** -6))) - 3)
        q = torch.clamp(torch.round(q / step) * step, -top, top)
    return {"q": q, "scale": scale, "h": h}
