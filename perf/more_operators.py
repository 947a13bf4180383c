"""The framework's operators of the 8-bit linear path, as they are timed: quantising rows to int8 with a scale each and
reading them back, the root-mean-square norm with the residual's addition and an int8 output, the matrix product of int8
rows and int8 weights, and a run of them as a layer boundary of the model has it.

``listed()`` gives the cases, ``prepare(case, seed)`` a program's inputs on the GPU, ``run(state)`` one pass: the plain
form in 32-bit torch operations (64 bits for a row's statistics and quotients, whose last bits decide between two codes),
or with ``own`` set the calls into ``mamba_tp_lite_b200``.  ``exact(case, seed)`` is the same from the definitions in 64 bits,
``work(case)`` the bytes and operations one pass cannot do without.  int8 codes are returned as the values they stand for.
"""
import math

import torch

own = False

_DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_SIZE = {"f32": 4, "bf16": 2, "f16": 2}

EPS = 1e-5


def listed():
    return [
        # one decode step's scan output in front of out_proj (1.4b shape)
        dict(name="quantize_step", op="quantize", rows=1, cols=4096, pad=0, dtype="bf16"),
        # the same for the benchmark's prompts, 32 x 1024 tokens
        dict(name="quantize_prompt", op="quantize", rows=32768, cols=4096, pad=0, dtype="bf16"),
        # an out_proj weight of the 2.8b shape, a scale for each output channel, when a model is quantised
        dict(name="quantize_weight", op="quantize", rows=2560, cols=5120, pad=0, dtype="f32"),
        # a layer's boundary in a decode step of 32 sequences: residual stream in fp32
        dict(name="norm_b32", op="norm", rows=32, cols=2048, pad=0, dtype="bf16", residual="f32"),
        # the same for the benchmark's prompts
        dict(name="norm_prompt", op="norm", rows=32768, cols=2048, pad=0, dtype="bf16", residual="f32"),
        # a ragged batch of odd width, cut out of wider rows, residual stream in fp16
        dict(name="norm_ragged", op="norm", rows=777, cols=1111, pad=5, dtype="f16", residual="f16"),
        # in_proj of one decode step
        dict(name="linear_step", op="linear", rows=1, cols=2048, out=8192, dtype="bf16", bias=False),
        # out_proj of a decode step of 64 sequences
        dict(name="linear_b64", op="linear", rows=64, cols=4096, out=2048, dtype="bf16", bias=False),
        # odd sizes, a bias, fp32 results
        dict(name="linear_odd", op="linear", rows=333, cols=1001, out=777, dtype="f32", bias=True),
        # in_proj of the benchmark's prompts
        dict(name="linear_prompt", op="linear", rows=32768, cols=2048, out=8192, dtype="bf16", bias=False),
        # from one layer's scan output to the next layer's in_proj output: one token
        dict(name="path_step", op="path", rows=1, inner=4096, cols=2048, dtype="bf16"),
        # the same for 8 x 1024 tokens
        dict(name="path_prompt", op="path", rows=8192, inner=4096, cols=2048, dtype="bf16"),
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["quantize", "norm", "norm", "linear", "linear", "path"])
    if op == "path":
        cols = 8 * _log_uniform(rng, 32, 320)
        return dict(op=op, rows=_log_uniform(rng, 1, 4096), inner=2 * cols, cols=cols, dtype=rng.choice(["bf16", "f16"]))
    if op == "linear":
        cols, out = _log_uniform(rng, 64, 5120), _log_uniform(rng, 64, 10240)
        if rng.random() < 0.5:
            cols, out = 16 * ((cols + 15) // 16), 16 * ((out + 15) // 16)
        most = max(1, min(32768, int(5e11 / (2.0 * cols * out))))
        return dict(op=op, rows=_log_uniform(rng, 1, most), cols=cols, out=out, dtype=rng.choice(["bf16", "bf16", "f16", "f32"]),
                    bias=rng.random() < 0.3)
    cols = _log_uniform(rng, 64, 8192)
    if rng.random() < 0.5:
        cols = 16 * ((cols + 15) // 16)
    rows = _log_uniform(rng, 1, max(1, min(65536, int(6e7 / cols))))
    case = dict(op=op, rows=rows, cols=cols, pad=rng.choice([0, 0, 0, 1, 8]), dtype=rng.choice(["bf16", "bf16", "f16", "f32"]))
    if op == "norm":
        case.update(residual=rng.choice(["none", "f32", "f32", case["dtype"]]))
    return case


# ------------------------------------------------------------------ inputs
def _activations(rows, cols, pad, dtype, gen, scale=1.0):
    """Activations [rows, cols] cut out of rows of cols + pad values: normal, with a size for each token and a few
    channels that are many times the others', as in a language model's hidden states."""
    x = torch.randn(rows, cols + pad, generator=gen, device="cuda")
    x.mul_(torch.exp(torch.randn(rows, 1, generator=gen, device="cuda") * 0.5) * scale)
    loud = torch.rand(cols + pad, generator=gen, device="cuda") < 0.01
    x.mul_(torch.where(loud, 12.0, 1.0))
    return x.to(_DTYPES[dtype])[:, :cols]


def _codes(x):
    """int8 rows as a program has them in hand: codes, each row on a 16-byte boundary, and a scale for each row."""
    scale = x.abs().amax(-1) / 127.0
    codes = torch.round(x / scale.unsqueeze(-1)).to(torch.int8)
    wide = (x.shape[1] + 15) // 16 * 16
    held = torch.zeros(x.shape[0], wide, device=x.device, dtype=torch.int8)
    held[:, :x.shape[1]] = codes
    return held[:, :x.shape[1]], scale


def _weight(out, cols, gen):
    return _codes(torch.randn(out, cols, generator=gen, device="cuda") / math.sqrt(cols))


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    st = dict(case=case)
    rows, cols = case["rows"], case["cols"]
    if case["op"] == "quantize":
        st["x"] = _activations(rows, cols, case["pad"], case["dtype"], gen)
    elif case["op"] == "norm":
        st["x"] = _activations(rows, cols, case["pad"], case["dtype"], gen, 0.3)
        if case["residual"] != "none":
            st["residual"] = _activations(rows, cols, case["pad"], case["residual"], gen)
        st["norm"] = (1.0 + 0.3 * torch.randn(cols, generator=gen, device="cuda")).to(_DTYPES[case["dtype"]])
    elif case["op"] == "linear":
        st["x"] = _codes(_activations(rows, cols, 0, "f32", gen))
        st["weight"] = _weight(case["out"], cols, gen)
        st["bias"] = torch.randn(case["out"], generator=gen, device="cuda").to(_DTYPES[case["dtype"]]) if case["bias"] else None
    else:
        st["x"] = _activations(rows, case["inner"], 0, case["dtype"], gen)
        st["residual"] = _activations(rows, cols, 0, "f32", gen)
        st["norm"] = (1.0 + 0.3 * torch.randn(cols, generator=gen, device="cuda")).to(_DTYPES[case["dtype"]])
        st["out_proj"] = _weight(cols, case["inner"], gen)
        st["in_proj"] = _weight(2 * case["inner"], cols, gen)
    return st


# ------------------------------------------------------------------ the plain form
def _plain_quantize(y):
    """(codes as fp32 whole numbers, scale [rows, 1] in fp32) of 64-bit rows: the multiple of the scale next to each value."""
    scale = (y.abs().amax(-1, keepdim=True).clamp(min=1e-8) / 127.0).float()
    return torch.round(y / scale.double()).clamp(-127.0, 127.0).float(), scale


def _plain_norm(x, residual, weight):
    """(codes, scale, residual stream): the sum in fp32, statistics and products in 64 bits."""
    h = x if residual is None else (x.float() + residual.float()).to(residual.dtype)
    hd = h.double()
    r = (hd.square().mean(-1, keepdim=True) + EPS).rsqrt()
    codes, scale = _plain_quantize(hd * r * weight.double())
    return codes, scale, h


def _plain_linear(codes, scale, weight, bias, dtype):
    """codes and weights as fp32 whole numbers: their products and sums stay below 2^24 in size and so are exact."""
    wq, ws = weight
    y = (codes @ wq.float().T) * scale * ws
    if bias is not None:
        y = y + bias.float()
    return y.to(dtype)


def _run_plain(st):
    case = st["case"]
    dtype = _DTYPES[case["dtype"]]
    if case["op"] == "quantize":
        codes, scale = _plain_quantize(st["x"].double())
        return {"values": (codes * scale).to(dtype), "scale": scale.squeeze(-1)}
    if case["op"] == "norm":
        codes, scale, h = _plain_norm(st["x"], st.get("residual"), st["norm"])
        out = {"values": (codes * scale).to(dtype), "scale": scale.squeeze(-1)}
        if "residual" in st:
            out["residual"] = h
        return out
    if case["op"] == "linear":
        codes, scale = st["x"]
        return {"out": _plain_linear(codes.float(), scale.unsqueeze(-1), st["weight"], st["bias"], dtype)}
    codes, scale = _plain_quantize(st["x"].double())
    branch = _plain_linear(codes, scale, st["out_proj"], None, torch.float32)  # what is added to an fp32 stream
    codes, scale, h = _plain_norm(branch, st["residual"], st["norm"])
    return {"residual": h, "out": _plain_linear(codes, scale, st["in_proj"], None, dtype)}


# ------------------------------------------------------------------ the framework's calls
def _run_own(st):
    from mamba_tp_lite_b200 import int8 as Q

    case = st["case"]
    dtype = _DTYPES[case["dtype"]]
    if case["op"] == "quantize":
        rows = Q.quantize_rows(st["x"])
        return {"values": Q.dequantize_rows(rows, dtype), "scale": rows.scale}
    if case["op"] == "norm":
        if "residual" not in st:
            rows = Q.rms_norm_int8(st["x"], st["norm"], EPS)
            return {"values": Q.dequantize_rows(rows, dtype), "scale": rows.scale}
        rows, h = Q.add_rms_norm_int8(st["x"], st["residual"], st["norm"], EPS)
        return {"values": Q.dequantize_rows(rows, dtype), "scale": rows.scale, "residual": h}
    if case["op"] == "linear":
        return {"out": Q.int8_linear(Q.Int8Rows(*st["x"]), Q.Int8Rows(*st["weight"]), st["bias"], dtype=dtype)}
    branch = Q.int8_linear(Q.quantize_rows(st["x"]), Q.Int8Rows(*st["out_proj"]), dtype=torch.float32)
    rows, h = Q.add_rms_norm_int8(branch, st["residual"], st["norm"], EPS)
    return {"residual": h, "out": Q.int8_linear(rows, Q.Int8Rows(*st["in_proj"]), dtype=dtype)}


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ------------------------------------------------------------------ the definitions in 64 bits
def _exact_rows(y):
    """What a row's codes stand for: the nearest of 255 multiples of its scale, which is held in fp32."""
    scale = torch.maximum(y.abs().amax(1), torch.full_like(y[:, 0], 1e-8)).div(127).float().double()
    q = (y / scale[:, None]).round()
    return q, scale


def _exact_norm(h, weight):
    mean = (h * h).sum(1) / h.shape[1]
    return h / torch.sqrt(mean + EPS)[:, None] * weight.double()


def _exact_product(q, scale, weight, bias):
    wq, ws = weight
    out = (q @ wq.double().t()) * (scale[:, None] * ws.double()[None, :])
    return out if bias is None else out + bias.double()


def exact(case, seed):
    st = prepare(case, seed)
    x = st["x"]
    if case["op"] == "linear":
        codes, scale = x
        return {"out": _exact_product(codes.double(), scale.double(), st["weight"], st["bias"])}
    if case["op"] == "quantize":
        q, scale = _exact_rows(x.double())
        return {"values": q * scale[:, None], "scale": scale}
    if case["op"] == "norm":
        h = x.double()
        if "residual" in st:  # the sum as it is held: rounded to the stream's type
            h = (x.float() + st["residual"].float()).to(st["residual"].dtype).double()
        q, scale = _exact_rows(_exact_norm(h, st["norm"]))
        out = {"values": q * scale[:, None], "scale": scale}
        if "residual" in st:
            out["residual"] = x.double() + st["residual"].double()
        return out
    q, scale = _exact_rows(x.double())
    h = _exact_product(q, scale, st["out_proj"], None) + st["residual"].double()
    q, scale = _exact_rows(_exact_norm(h, st["norm"]))
    return {"residual": h, "out": _exact_product(q, scale, st["in_proj"], None)}


def work(case):
    rows, cols = case["rows"], case["cols"]
    es = _SIZE[case["dtype"]]
    if case["op"] == "quantize":  # values in, values and scales out
        return {"bytes": rows * (2 * cols * es + 4), "flops": 4 * rows * cols}
    if case["op"] == "norm":
        er = 0 if case["residual"] == "none" else _SIZE[case["residual"]]
        return {"bytes": rows * (cols * (2 * es + 2 * er) + 4) + cols * es, "flops": 9 * rows * cols}
    if case["op"] == "linear":
        n = case["out"]
        return {"bytes": rows * (cols + 4) + n * (cols + 4 + (es if case["bias"] else 0)) + rows * n * es,
                "flops": 2 * rows * n * cols}
    inner = case["inner"]
    return {"bytes": rows * (inner * es + 8 * cols + 2 * inner * es) + 3 * inner * cols + 4 * (cols + 2 * inner) + cols * es,
            "flops": 6 * rows * inner * cols}
