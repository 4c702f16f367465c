"""Measured cases of the 4-bit floating-point operators (``glm53.ops.fp4``): quantisation with read-back, the
projection with 4-bit weights, and the gated feed-forward block in 4 bits.

Formats.  A row of K values is cut into blocks; an element is an e2m1 code (0, .5, 1, 1.5, 2, 3, 4, 6 and the
negatives) times its block's scale, times (nvfp4) its row's scale:

* ``mxfp4``: blocks of 32; the block scale is the smallest power of two 2^e with amax <= 6 * 2^e;
* ``nvfp4``: blocks of 16; the row scale is the smallest power of two 2^k with amax(row) <= 6 * 448 * 2^k, the block
  scale is amax(block) * 2^-k / 6 rounded to e4m3 (nearest, ties to even).

Codes are rounded to nearest, ties to the even code; a block whose scale is 0 reads back as 0.

* quantize:  x -> Q(x) -> the values Q(x) stands for;
* linear:    y = a W^T, W in 4 bits, a = x, or a = Q(x) with ``act4`` (more than 16 rows);
* mlp:       y = h Wd^T, h = silu(min(g, L)) * clip(u, -L, L), [g | u] = a Wgu^T; h is held in bf16, or with ``act4``
  (more than 16 rows) in 4 bits, nvfp4 with the one row scale that fits L * L.
"""

from __future__ import annotations

import math

import torch

own = False

LIMIT = 10.0                # the model configuration's clamp of the gated block
LEVELS = 448.0 * 6.0        # largest e4m3 times the largest e2m1


# ------------------------------------------------------------------------------------------------- the cases
def listed() -> list[dict]:
    return [
        # rows of one prefill chunk at the hidden width, as the 4-bit prefill quantises them
        {"name": "quantize chunk nv", "op": "quantize", "rows": 8192, "k": 4096, "fmt": "nvfp4", "dtype": "bf16"},
        # an odd tail chunk of the dense layers' inner width
        {"name": "quantize tail mx", "op": "quantize", "rows": 777, "k": 12288, "fmt": "mxfp4", "dtype": "bf16"},
        # a few rows of a tensor-parallel shard, from f16: launch latency
        {"name": "quantize few nv f16", "op": "quantize", "rows": 5, "k": 1536, "fmt": "nvfp4", "dtype": "f16"},
        # one token through the dense layers' gate/up projection
        {"name": "linear 1 nv", "op": "linear", "m": 1, "n": 24576, "k": 4096, "fmt": "nvfp4", "act4": False,
         "out": "bf16"},
        # a verify window of 8 rows over one of eight vocabulary shards, fp32 logits
        {"name": "linear 8 head mx", "op": "linear", "m": 8, "n": 19360, "k": 4096, "fmt": "mxfp4", "act4": False,
         "out": "f32"},
        # two windows' rows over a small projection (one query up-projection shard)
        {"name": "linear 13 small nv", "op": "linear", "m": 13, "n": 2048, "k": 1536, "fmt": "nvfp4", "act4": False,
         "out": "bf16"},
        # a prefill chunk through the dense layers' down projection, 4-bit activations
        {"name": "linear chunk a4 nv", "op": "linear", "m": 8192, "n": 4096, "k": 12288, "fmt": "nvfp4",
         "act4": True, "out": "bf16"},
        # an odd chunk and an odd output width, 4-bit activations, fp32 partials
        {"name": "linear odd a4 mx", "op": "linear", "m": 1111, "n": 1000, "k": 1536, "fmt": "mxfp4", "act4": True,
         "out": "f32"},
        # one token through the shared expert: the smallest block of a decode step
        {"name": "mlp 1 shared nv", "op": "mlp", "m": 1, "k": 4096, "width": 2048, "n": 4096, "fmt": "nvfp4",
         "act4": False},
        # 16 rows (two verify windows) through a dense layer's block
        {"name": "mlp 16 dense mx", "op": "mlp", "m": 16, "k": 4096, "width": 12288, "n": 4096, "fmt": "mxfp4",
         "act4": False},
        # a short prompt with exact activations through the shared expert
        {"name": "mlp 300 shared nv", "op": "mlp", "m": 300, "k": 4096, "width": 2048, "n": 4096, "fmt": "nvfp4",
         "act4": False},
        # a prefill chunk through a dense layer's block, 4-bit activations
        {"name": "mlp chunk a4 nv", "op": "mlp", "m": 8192, "k": 4096, "width": 12288, "n": 4096, "fmt": "nvfp4",
         "act4": True},
    ]


def _log(rng, lo: int, hi: int, step: int = 1) -> int:
    """A multiple of step in [lo, hi], spread over the logarithm."""
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return min(hi // step, max(-(-lo // step), round(v / step))) * step


def draw(rng) -> dict:
    op = rng.choice(["quantize", "linear", "linear", "mlp", "mlp"])
    fmt = rng.choice(["nvfp4", "mxfp4"])
    if op == "quantize":
        return {"op": op, "rows": _log(rng, 1, 8192), "k": _log(rng, 96, 12288, 32), "fmt": fmt,
                "dtype": rng.choice(["bf16", "bf16", "f16"])}
    # decode windows, short prompts, chunks
    m, act4 = rng.choice([(_log(rng, 1, 16), False), (_log(rng, 1, 16), False), (_log(rng, 17, 700), False),
                          (_log(rng, 17, 8192), True), (_log(rng, 256, 8192), True)])
    k = _log(rng, 256, 4096, 32)
    if op == "linear":
        wide = m < 1024
        return {"op": op, "m": m, "n": _log(rng, 256, 19360 if wide else 4096),
                "k": _log(rng, 256, 12288, 32) if wide else k, "fmt": fmt, "act4": act4,
                "out": rng.choice(["bf16", "f32"])}
    return {"op": op, "m": m, "k": k, "width": _log(rng, 256, 12288, 32), "n": _log(rng, 256, 4096, 8), "fmt": fmt,
            "act4": act4}


# --------------------------------------------------------------------------------------------------- inputs
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def _device():
    return "cuda" if torch.cuda.is_available() else "cpu"


def _tensors(case: dict, seed: int) -> dict:
    """Activations as they leave a norm (unit variance, a few channels some times larger) and weights as trained ones
    are (small, one width per row), from the seed alone."""
    dev = _device()
    g = torch.Generator(device=dev).manual_seed(seed)

    def acts(rows, k, dtype):
        x = torch.randn(rows, k, generator=g, device=dev)
        x *= 1.0 + 7.0 * (torch.rand(k, generator=g, device=dev) < 0.02)
        return x.to(dtype)

    def weight(n, k):
        w = torch.randn(n, k, generator=g, device=dev)
        w *= k ** -0.5 * (0.5 + torch.rand(n, 1, generator=g, device=dev))
        return w.to(torch.bfloat16)

    if case["op"] == "quantize":
        return {"x": acts(case["rows"], case["k"], DTYPES[case["dtype"]])}
    x = acts(case["m"], case["k"], torch.bfloat16)
    if case["op"] == "linear":
        return {"x": x, "w": weight(case["n"], case["k"])}
    return {"x": x, "gate": weight(case["width"], case["k"]), "up": weight(case["width"], case["k"]),
            "down": weight(case["n"], case["width"])}


def prepare(case: dict, seed: int) -> dict:
    t = _tensors(case, seed)
    st = {"case": dict(case), "x": t["x"]}
    fmt = case["fmt"]
    if case["op"] == "quantize":
        return st
    if own:
        from glm53.ops import fp4
        if case["op"] == "linear":
            st["w"] = fp4.quantize4(t["w"], fmt)
        else:
            st["w"] = fp4.pack_mlp4(t["gate"], t["up"], t["down"], fmt)
        out = DTYPES[case.get("out", "bf16")]
        st["y"] = torch.empty(case["m"], case["n"], dtype=out, device=t["x"].device)
    else:
        for name in ("w", "gate", "up", "down"):
            if name in t:
                st[name] = _pack(*_quantize(t[name], fmt))
    return st


# ------------------------------------------------------------------------------------------------ plain form
def _pow2(e: torch.Tensor) -> torch.Tensor:
    """2^e in fp32, from its bits (normal range)."""
    return ((e.clamp(-126, 127) + 127).to(torch.int32) << 23).view(torch.float32)


def _range_exponent(amax: torch.Tensor, shift: int, top: float) -> torch.Tensor:
    """Smallest e with amax <= c * 2^e, for c = 2 * top * 2^(shift - 1) and top in [0.5, 1)."""
    f, e = torch.frexp(amax)
    return e - shift + (f > top).to(e.dtype)


def _round_e2m1(q: torch.Tensor) -> torch.Tensor:
    """|q| to the nearest of 0, .5, 1, 1.5, 2, 3, 4, 6 (ties to the even code)."""
    v = torch.full_like(q, 6.0)
    v = torch.where(q <= 5.0, 4.0, v)
    v = torch.where(q < 3.5, 3.0, v)
    v = torch.where(q <= 2.5, 2.0, v)
    v = torch.where(q < 1.75, 1.5, v)
    v = torch.where(q <= 1.25, 1.0, v)
    v = torch.where(q < 0.75, 0.5, v)
    return torch.where(q <= 0.25, 0.0, v)


def _quantize(x: torch.Tensor, fmt: str, bound: float | None = None):
    """(e2m1 values [R, K], block scales [R, K / block], row scales [R, 1]), all fp32.  bound: the row scale is the one
    that fits this bound instead of the row's own maximum (nvfp4)."""
    x = x.float()
    block = 16 if fmt == "nvfp4" else 32
    xb = x.view(x.shape[0], -1, block)
    amax = xb.abs().amax(-1)
    if fmt == "mxfp4":
        # 6 = 0.75 * 2^3; E8M0 holds exponents from -127
        s = _pow2(_range_exponent(amax, 3, 0.75).clamp_min(-126))
        r = torch.ones(x.shape[0], 1, device=x.device)
    else:
        top = amax.amax(-1, keepdim=True) if bound is None else torch.full((x.shape[0], 1), bound, device=x.device)
        # 2688 = 0.65625 * 2^12
        k = _range_exponent(top, 12, 0.65625)
        r = _pow2(k)
        six = torch.full((), 6.0, device=x.device)
        s = (amax * _pow2(-k) / six).to(torch.float8_e4m3fn).float()
        xb = xb * _pow2(-k)[..., None]
    q = torch.where(s[..., None] > 0, xb.abs() / s[..., None], 0.0)
    return (torch.sign(xb) * _round_e2m1(q)).view(x.shape), s, r


def _values(v: torch.Tensor, s: torch.Tensor, r: torch.Tensor) -> torch.Tensor:
    return (v.view(*s.shape, -1) * (s * r)[..., None]).view(v.shape)


def _pack(v: torch.Tensor, s: torch.Tensor, r: torch.Tensor):
    """The 4-bit codes two to a byte (sign, then the place among the eight magnitudes), with their scales."""
    mags = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device=v.device)
    c = torch.bucketize(v.abs(), mags).to(torch.uint8) | ((v < 0).to(torch.uint8) << 3)
    return c[:, 0::2] | (c[:, 1::2] << 4), s, r


def _unpack(p: torch.Tensor, s: torch.Tensor, r: torch.Tensor) -> torch.Tensor:
    mags = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]
    table = torch.tensor(mags + [-m for m in mags], device=p.device)
    v = torch.stack((table[(p & 15).int()], table[(p >> 4).int()]), -1).view(p.shape[0], -1)
    return _values(v, s, r)


def _gated(g: torch.Tensor, u: torch.Tensor) -> torch.Tensor:
    g, u = g.clamp(max=LIMIT), u.clamp(-LIMIT, LIMIT)
    return g / (1.0 + torch.exp(-g)) * u


def _run_plain(st: dict):
    case, fmt = st["case"], st["case"]["fmt"]
    x = st["x"]
    if case["op"] == "quantize":
        return _values(*_quantize(x, fmt)).to(x.dtype)
    act4 = case["act4"] and x.shape[0] > 16
    a = _values(*_quantize(x, fmt)) if act4 else x.float()
    if case["op"] == "linear":
        return (a @ _unpack(*st["w"]).t()).to(DTYPES[case["out"]])
    h = _gated(a @ _unpack(*st["gate"]).t(), a @ _unpack(*st["up"]).t())
    h = _values(*_quantize(h, fmt, LIMIT * LIMIT)) if act4 else h.to(torch.bfloat16).float()
    return (h @ _unpack(*st["down"]).t()).to(torch.bfloat16)


def _run_own(st: dict):
    from glm53.ops import fp4
    from glm53.ops import kernels as K
    case = st["case"]
    if case["op"] == "quantize":
        return fp4.dequantize4(fp4.quantize4(st["x"], case["fmt"]), st["x"].dtype)
    if case["op"] == "linear":
        mode = K.GEMV_F32 if case["out"] == "f32" else K.GEMV_BF16
        return fp4.linear4(st["x"], st["w"], st["y"], mode, act4=case["act4"])
    return fp4.mlp4(st["x"], st["w"], st["y"], LIMIT, K.GEMV_BF16, act4=case["act4"])


def run(state: dict):
    return _run_own(state) if own else _run_plain(state)


# ------------------------------------------------------------------------------------------------------ work
def work(case: dict) -> dict:
    per = 0.5 + (1.0 / 16 if case["fmt"] == "nvfp4" else 1.0 / 32)       # bytes of a 4-bit element
    if case["op"] == "quantize":
        n = case["rows"] * case["k"]
        return {"bytes": n * (2 + per + 2), "flops": 4 * n}
    m, n, k = case["m"], case["n"], case["k"]
    if case["op"] == "linear":
        out = 4 if case["out"] == "f32" else 2
        return {"bytes": n * k * per + 2 * m * k + out * m * n, "flops": 2 * m * n * k}
    w = case["width"]
    return {"bytes": (2 * w * k + n * w) * per + 2 * m * k + 2 * m * n, "flops": 2 * m * w * (2 * k + n)}


# -------------------------------------------------------------------------------------- the definition, 64 bits
def _exact_q(x: torch.Tensor, fmt: str, bound: float | None = None) -> torch.Tensor:
    """The values of Q(x) in 64 bits: scales by logarithms put right at their borders, codes by rounding on the
    lattice of each binade."""
    x = x.double()
    rows, k = x.shape

    def two(e):
        return ((e.to(torch.int64) + 1023) << 52).view(torch.float64)

    def ceil2(t):
        """Smallest power of two >= t, for t > 0 (1 elsewhere)."""
        p = two(torch.ceil(torch.log2(torch.where(t > 0, t, 1.0))))
        p = torch.where(p / 2 >= t, p / 2, p)
        return torch.where((t > 0) & (p < t), p * 2, p)

    if fmt == "mxfp4":
        b = x.view(rows, k // 32, 32)
        scale = ceil2(b.abs().amax(-1, keepdim=True) / 6.0).clamp_min(2.0 ** -126)
    else:
        b = x.view(rows, k // 16, 16)
        top = b.abs().amax((-1, -2), keepdim=True) if bound is None else x.new_full((rows, 1, 1), bound)
        row = ceil2(top / LEVELS)
        t = b.abs().amax(-1, keepdim=True) / row / 6.0
        lattice = ceil2(t.clamp_min(2.0 ** -6) * (1 + 2.0 ** -40)) / 16               # e4m3: 3 bits of mantissa
        scale = torch.round(t / lattice) * lattice * row
    q = torch.where(scale > 0, b.abs() / torch.where(scale > 0, scale, 1.0), 0.0)
    step = 0.5 * (1 + (q >= 2).double() + 2 * (q >= 4).double())
    return (torch.sign(b) * (torch.round(q / step) * step).clamp_max(6.0) * scale).view(rows, k)


def exact(case: dict, seed: int):
    t, fmt = _tensors(case, seed), case["fmt"]
    x = t["x"]
    if case["op"] == "quantize":
        return _exact_q(x, fmt)
    act4 = case["act4"] and x.shape[0] > 16
    a = _exact_q(x, fmt) if act4 else x.double()
    if case["op"] == "linear":
        return a @ _exact_q(t["w"], fmt).t()
    g = (a @ _exact_q(t["gate"], fmt).t()).clamp(max=LIMIT)
    u = (a @ _exact_q(t["up"], fmt).t()).clamp(-LIMIT, LIMIT)
    h = g * torch.sigmoid(g) * u
    h = _exact_q(h, fmt, LIMIT * LIMIT) if act4 else h.to(torch.bfloat16).double()
    return h @ _exact_q(t["down"], fmt).t()
