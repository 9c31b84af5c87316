"""Performance cases of the block-scaled 8-bit operators: what is timed, on which
inputs, and what it must compute.

The operators are the device-pointer entry points of the C-ABI
(`include/seeml_hip.h`) that run a frozen base in 8-bit floats and keep a step's
activations in them:

  linear  `seeml_hip_f8_quantize` of the activations, then
          `seeml_hip_gemm_f8_nt` with a frozen weight: y = x W.
  gated   the same with `seeml_hip_gated_f8_fwd`: h = act(x Wg) * (x Wu), the
          gated half of a decoder's feed-forward block, for evaluation.
  train   a training step of it: the forward pass keeping both projections in
          8 bits, then `seeml_hip_gated_f8_bwd` for the gradient of x.
  act     an activation kept in 8 bits (`seeml_hip_f8_quantize`) and its
          backward pass from there (`seeml_hip_act_bwd_f8`).
  norm    the same of an RMS norm's input (`seeml_hip_rms_norm_bwd_f8`).
  lora    the same of a LoRA layer's input: the gradient of its down projection
          (`seeml_hip_gemm_tn_f8`).

The format: a matrix [rows, cols] is one e4m3 code a value, rows padded with
zeros to whole blocks of 128, and one byte a block, of value 2^(byte - 127); the
bytes lie [blocks of a row][rows, rounded up to 128]. A block's exponent is the
least that brings its largest magnitude to 448 or below. Activations have blocks
of 1 x 128, weights of 128 x 128.

Sizes are those of the repository's own decoders (widths 512, 2048 and 4096, feed-forward
widths 1376, 5504 and 16384, batches of 32 to 8192 tokens), single tokens, and
ragged sizes between them.
"""
import math
import os
import sys

import torch

own = False

_DEV = "cuda:0"
_TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_ACTS = {"relu": 1, "gelu": 2, "silu": 3}


# ---------------------------------------------------------------- the cases

def listed():
    return [
        # One token through the d_model-2048 decoder's up projection.
        dict(name="linear_1x2048x5504_bf16", kind="linear", T=1, D=2048, F=5504, type="bf16", pad=0,
             padded=False),
        # A batch of 8 x 1024 tokens through it.
        dict(name="linear_8192x2048x5504_bf16", kind="linear", T=8192, D=2048, F=5504, type="bf16",
             pad=0, padded=True),
        # The small decoder's down projection, rows that fill no tile, float32.
        dict(name="linear_515x1376x2000", kind="linear", T=515, D=1376, F=2000, type="f32", pad=3,
             padded=True),
        # One token through the gated block.
        dict(name="gated_1x2048x5504_bf16", kind="gated", T=1, D=2048, F=5504, type="bf16",
             act="silu", pad=0, padded=False),
        # One step of 24 sequences through the small decoder's, float32.
        dict(name="gated_24x512x1376", kind="gated", T=24, D=512, F=1376, type="f32", act="silu",
             pad=0, padded=False),
        # A training batch of the d_model-2048 decoder, 8 x 1024: the largest.
        dict(name="train_8192x2048x5504_bf16", kind="train", T=8192, D=2048, F=5504, type="bf16",
             act="silu", pad=0, padded=True),
        # Sizes that divide by nothing.
        dict(name="train_777x520x1003_f16", kind="train", T=777, D=520, F=1003, type="f16",
             act="gelu", pad=5, padded=True),
        # The d_model-4096 decoder's GELU over its feed-forward width, 4 x 2048 tokens.
        dict(name="act_8192x16384", kind="act", T=8192, D=16384, type="f32", act="gelu", pad=0,
             padded=False),
        # A ragged activation, rows of a wider buffer.
        dict(name="act_333x1003_bf16", kind="act", T=333, D=1003, type="bf16", act="silu", pad=8,
             padded=True),
        # The d_model-2048 decoder's norm input over its batch.
        dict(name="norm_8192x2048", kind="norm", T=8192, D=2048, type="f32", pad=0, padded=True),
        # The adapters' input of the d_model-2048 decoder, rank 16.
        dict(name="lora_8192x2048_r16", kind="lora", T=8192, D=2048, r=16, type="f32", pad=0,
             padded=True),
        # Rank 64 of a ragged batch.
        dict(name="lora_2047x1376_r64_bf16", kind="lora", T=2047, D=1376, r=64, type="bf16", pad=0,
             padded=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["linear", "linear", "gated", "train", "act", "norm", "lora"])
    case = dict(kind=kind, type=rng.choice(["f32", "bf16", "bf16", "f16"]),
                pad=rng.choice([0, 0, 1, 8, 13]), padded=rng.random() < 0.5)
    if kind in ("linear", "gated", "train"):
        if kind == "train" and case["type"] == "f32":
            case["type"] = "bf16"
        case["D"] = rng.choice([512, 2048, _log(rng, 64, 4096), _log(rng, 64, 4096)])
        case["F"] = rng.choice([1376, 5504, _log(rng, 64, 8192), _log(rng, 64, 8192)])
        most = 8192 * 2048 * 5504 // (case["D"] * case["F"])
        case["T"] = _log(rng, 1, max(2, min(8192, most)))
        if kind != "linear":
            case["act"] = rng.choice(["silu", "silu", "gelu", "relu"])
        return case
    case["D"] = rng.choice([512, 2048, _log(rng, 64, 16384), _log(rng, 64, 16384)])
    case["T"] = _log(rng, 1, 8192)
    if kind == "act":
        case["act"] = rng.choice(["silu", "gelu", "relu"])
    if kind == "lora":
        case["r"] = rng.choice([8, 16, 64, _log(rng, 1, 128)])
    return case


# ------------------------------------------------------------------- inputs

def _up(n):
    return -(-n // 128) * 128


def _pow2(byte):
    """2^(byte - 127) of bytes below 255, exactly; byte 0 is a subnormal number."""
    return torch.where(byte > 0, (byte << 23).view(torch.float32), 2.0 ** -127)


def _blocks(x, square):
    """x [rows, cols] in float32 as blocks [rows', 128 or 1 rows, blocks, 128] (zeros
    behind its ends), and each block's scale byte."""
    rows, cols = x.shape
    tall = 128 if square else 1
    xb = torch.zeros(-(-rows // tall) * tall, _up(cols), device=x.device)
    xb[:rows, :cols] = x
    xb = xb.view(-1, tall, _up(cols) // 128, 128)
    amax = torch.where(torch.isfinite(xb), xb.abs(), 0.0).amax((1, 3), keepdim=True)
    bits = amax.view(torch.int32)
    byte = ((bits >> 23) - 8 + ((bits & 0x7FFFFF) > 0x600000).int()).clamp(min=0)
    return xb, byte


def _codes(xb, byte):
    scaled = xb * ((254 - byte) << 23).view(torch.float32)
    return scaled.to(torch.float8_e4m3fn)


def _kept(x):
    """What 8 bits keep of x [rows, cols], as float32."""
    xb, byte = _blocks(x.float(), False)
    kept = _codes(xb, byte).float() * _pow2(byte)
    return kept.view(xb.shape[0], -1)[:, :x.shape[1]]


def _weight(w):
    """A weight in 8 bits: (codes, scales), rows as they are."""
    rows, cols = w.shape
    xb, byte = _blocks(w, True)
    codes = _codes(xb, byte).view(-1, _up(cols))[:rows].view(torch.uint8).contiguous()
    scales = byte.expand(-1, 128, -1, -1).reshape(-1, _up(cols) // 128).t().to(torch.uint8)
    return codes, scales.contiguous()


def _values(weight, cols):
    """A weight's values [rows, cols] as float32."""
    codes, scales = weight
    rows = codes.shape[0]
    x = codes.view(torch.float8_e4m3fn).float().view(rows, -1, 128)
    return (x * _pow2(scales[:, :rows].t().int())[:, :, None]).view(rows, -1)[:, :cols]


def prepare(case, seed):
    g = torch.Generator(device=_DEV)
    g.manual_seed(1000003 * int(seed) + 31)
    T, D = case["T"], case["D"]
    dtype = _TYPES[case["type"]]
    randn = lambda *s: torch.randn(*s, generator=g, device=_DEV)  # noqa: E731

    def rows_of(x):  # in the case's type, in a buffer whose rows may be longer
        buf = torch.zeros(x.shape[0], x.shape[1] + case["pad"], device=_DEV, dtype=dtype)
        buf[:, :x.shape[1]] = x
        return buf[:, :x.shape[1]]

    # Activations of a decoder: a few columns much larger than the rest.
    x = randn(T, D)
    x *= 1.0 + 15.0 * (torch.rand(D, generator=g, device=_DEV) < 0.01).float()
    if case["padded"]:  # rows behind a sequence's end, the first row never
        x[1:] *= (torch.rand(T, 1, generator=g, device=_DEV)[1:] >= 0.125).float()
    s = dict(case=case, x=rows_of(x))
    if case["kind"] in ("linear", "gated", "train"):
        F = case["F"]
        names = ("w",) if case["kind"] == "linear" else ("wg", "wu")
        for name in names:  # [D, F], kept as the transpose for y = x W
            w = randn(D, F) * (0.9 / math.sqrt(D))
            s[name + "_t"] = _weight(w.t())
            if case["kind"] == "train":
                s[name] = _weight(w)
        if case["kind"] == "train":
            s["dh"] = rows_of(randn(T, F))
    elif case["kind"] == "lora":
        s["dt"] = (randn(T, case["r"]) * 0.05).to(dtype)
    else:
        s["dy"] = rows_of(randn(T, D))
        if case["kind"] == "norm":
            s["gamma"] = 1.0 + 0.1 * randn(D)
            s["rstd"] = torch.rsqrt(s["x"].double().square().mean(-1) + 1e-5).float()
    return s


# ---------------------------------------------------------------- one pass

def run(s):
    return _own(s) if own else _plain(s)


def _own(s):
    """The calls of a user's program: outputs and scratch from torch's
    allocator, the current stream."""
    path = os.path.join(os.getcwd(), "see-ml_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    from seeml_amd import lib
    L, c, x = lib(), s["case"], s["x"]
    T, D, kind = c["T"], c["D"], c["kind"]
    dtype = {"f32": 0, "bf16": 1, "f16": 2}[c["type"]]
    act = _ACTS.get(c.get("act"), 0)
    stream = torch.cuda.current_stream().cuda_stream
    at = lambda t: t.data_ptr() if t is not None else None  # noqa: E731

    def call(name, *args):
        args = [at(a) if a is None or isinstance(a, torch.Tensor) else a for a in args]
        if getattr(L, "seeml_hip_" + name)(*args, stream) != 0:
            raise RuntimeError("%s: %s" % (name, L.seeml_hip_kernel_error().decode()))

    def room(rows, cols):  # codes and scales of a [rows, cols] matrix
        return (torch.empty(rows, _up(cols), device=_DEV, dtype=torch.uint8),
                torch.empty(_up(cols) // 128, _up(rows), device=_DEV, dtype=torch.uint8))

    def scratch(nbytes):
        return torch.empty(nbytes, device=_DEV, dtype=torch.uint8) if nbytes else None

    new = lambda *shape: torch.empty(*shape, device=_DEV, dtype=x.dtype)  # noqa: E731
    x8 = room(T, D)
    call("f8_quantize", x, dtype, x.stride(0), T, D, *x8)
    if kind == "linear":
        F = c["F"]
        y = new(T, F)
        nbytes = L.seeml_hip_gemm_f8_scratch(T, F, D)
        call("gemm_f8_nt", *x8, *s["w_t"], y, dtype, F, T, F, D, scratch(nbytes), nbytes)
        return dict(y=y)
    if kind in ("gated", "train"):
        F = c["F"]
        h = new(T, F)
        g8, u8 = (room(T, F), room(T, F)) if kind == "train" else ((None, None), (None, None))
        nbytes = L.seeml_hip_gated_f8_scratch(T, D, F)
        work_ = scratch(nbytes)
        call("gated_f8_fwd", *x8, *s["wg_t"], *s["wu_t"], act, h, dtype, F, None, None, *g8, *u8,
             T, D, F, work_, nbytes)
        if kind == "gated":
            return dict(h=h)
        dh, dx = s["dh"], new(T, D)
        dg8, du8 = room(T, F), room(T, F)
        call("gated_f8_bwd", dh, dtype, dh.stride(0), *g8, *u8, act, *s["wg"], *s["wu"], *dg8,
             *du8, None, 0, dx, D, T, D, F, work_, nbytes)
        return dict(h=h, dx=dx)
    if kind == "lora":
        r = c["r"]
        out = torch.empty(D, r, device=_DEV)
        nbytes = L.seeml_hip_gemm_tn_f8_scratch(T, D, r)
        call("gemm_tn_f8", *x8, s["dt"], dtype, r, out, T, D, r, scratch(nbytes), nbytes)
        return dict(da=out)
    dy, dx = s["dy"], new(T, D)
    if kind == "act":
        call("act_bwd_f8", dy, dtype, dy.stride(0), *x8, act, dx, D, T, D)
    else:
        call("rms_norm_bwd_f8", dy, dtype, dy.stride(0), *x8, s["gamma"], s["rstd"], dx, D, T, D)
    return dict(dx=dx)


def _act(name, x):
    if name == "relu":
        return x.clamp(min=0)
    if name == "silu":
        return x / (1.0 + torch.exp(-x))
    return 0.5 * x * (1.0 + torch.tanh(0.7978845608028654 * (x + 0.044715 * x * x * x)))


def _dact(name, x):
    if name == "relu":
        return (x > 0).float()
    if name == "silu":
        p = 1.0 / (1.0 + torch.exp(-x))
        return p * (1.0 + x * (1.0 - p))
    t = torch.tanh(0.7978845608028654 * (x + 0.044715 * x * x * x))
    return 0.5 * (1.0 + t) + 0.5 * x * (1.0 - t * t) * 0.7978845608028654 * (1.0 + 0.134145 * x * x)


def _plain(s):
    c, kind = s["case"], s["case"]["kind"]
    dtype = s["x"].dtype
    x = _kept(s["x"])
    if kind == "linear":
        return dict(y=(x @ _values(s["w_t"], c["D"]).t()).to(dtype))
    if kind in ("gated", "train"):
        g = x @ _values(s["wg_t"], c["D"]).t()
        u = x @ _values(s["wu_t"], c["D"]).t()
        h = (_act(c["act"], g) * u).to(dtype)
        if kind == "gated":
            return dict(h=h)
        g, u, dh = _kept(g), _kept(u), s["dh"].float()
        dg, du = _kept(dh * u * _dact(c["act"], g)), _kept(dh * _act(c["act"], g))
        dx = dg @ _values(s["wg"], c["F"]).t() + du @ _values(s["wu"], c["F"]).t()
        return dict(h=h, dx=dx.to(dtype))
    if kind == "lora":
        return dict(da=x.t().contiguous() @ s["dt"].float())
    dy = s["dy"].float()
    if kind == "act":
        return dict(dx=(dy * _dact(c["act"], x)).to(dtype))
    r = s["rstd"][:, None]
    dyg = dy * s["gamma"]
    dot = (dyg * x).sum(-1, keepdim=True, dtype=torch.float64) / c["D"]
    return dict(dx=(r * (dyg - x * (r.double().square() * dot).float())).to(dtype))


# ------------------------------------------------- the work of one pass

def work(case):
    """Activations read and results written once in their own type, frozen weights
    read as 8 bits (in a training step as they are and as the transpose)."""
    T, D, F, kind = case["T"], case["D"], case.get("F", 0), case["kind"]
    size = 4 if case["type"] == "f32" else 2
    if kind == "linear":
        return dict(bytes=size * T * (D + F) + D * F, flops=2.0 * T * D * F)
    if kind == "gated":
        return dict(bytes=size * T * (D + F) + 2 * D * F, flops=4.0 * T * D * F)
    if kind == "train":
        return dict(bytes=size * T * 2 * (D + F) + 4 * D * F, flops=8.0 * T * D * F)
    if kind == "lora":
        r = case["r"]
        return dict(bytes=size * T * (D + r) + 4 * D * r, flops=2.0 * T * D * r)
    return dict(bytes=size * T * D * 3, flops=20.0 * T * D)


# -------------------------------------------------- the same in 64 bits

def _rounded(x):
    """x to the nearest value that its block's 8 bits have, ties to even, in 64 bits."""
    rows, cols = x.shape
    b = torch.nn.functional.pad(x, (0, _up(cols) - cols)).reshape(rows, -1, 128)
    top = b.abs().amax(-1, keepdim=True)
    mantissa, exponent = torch.frexp(top)  # top = mantissa 2^exponent, mantissa in [1/2, 1)
    e = exponent - 9 + (mantissa > 0.875).int()
    e = torch.where(top > 0, e, -127).clamp(min=-127).double()
    y = b * torch.exp2(-e)
    _, k = torch.frexp(y)
    step = torch.exp2((k - 4).clamp(min=-9).double())  # 3 bits behind the leading one; 2^-9 at least
    return (torch.round(y / step) * step * torch.exp2(e)).reshape(rows, -1)[:, :cols]


def _read(weight, cols):
    codes, scales = weight
    rows = codes.shape[0]
    factor = torch.exp2(scales[:, :rows].t().double() - 127).repeat_interleave(128, 1)
    return (codes.view(torch.float8_e4m3fn).double() * factor)[:, :cols]


def _act64(name, x):
    """An activation and its derivative."""
    if name == "relu":
        return torch.relu(x), (x > 0).double()
    if name == "silu":
        p = torch.sigmoid(x)
        return x * p, p + x * p * torch.sigmoid(-x)
    a = math.sqrt(2.0 / math.pi)
    t = torch.tanh(a * (x + 0.044715 * x ** 3))
    return x * (1 + t) / 2, (1 + t) / 2 + x * (1 - t ** 2) * a * (1 + 3 * 0.044715 * x ** 2) / 2


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    x = _rounded(s["x"].double())
    if kind == "linear":
        return dict(y=x @ _read(s["w_t"], case["D"]).t())
    if kind in ("gated", "train"):
        g = x @ _read(s["wg_t"], case["D"]).t()
        u = x @ _read(s["wu_t"], case["D"]).t()
        out = dict(h=_act64(case["act"], g)[0] * u)
        if kind == "train":
            g, u = _rounded(g), _rounded(u)
            a, d = _act64(case["act"], g)
            dh = s["dh"].double()
            out["dx"] = (_rounded(dh * u * d) @ _read(s["wg"], case["F"]).t()
                         + _rounded(dh * a) @ _read(s["wu"], case["F"]).t())
        return out
    if kind == "lora":
        return dict(da=x.t().contiguous() @ s["dt"].double())
    dy = s["dy"].double()
    if kind == "act":
        return dict(dx=dy * _act64(case["act"], x)[1])
    r, up = s["rstd"].double()[:, None], dy * s["gamma"].double()
    along = (up * x).mean(-1, keepdim=True)
    return dict(dx=up * r - x * along * r ** 3)
