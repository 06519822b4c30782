"""Operators on rows of 8-bit integers, in their plain form and as the framework's kernels, and the cases they are timed on.

A row of activations, or of weights, is held as integers of -127 .. 127 and one fp32 scale: ``scale = max |x| / 127``,
``q = round(x * (127 / max |x|))`` (halves to even), so that ``x`` is about ``q * scale``. The operators:

* ``norm``: what stands between two sublayers. ``h = x + add`` (fp32, the residual stream), then the RMS norm of every row of ``h``
  with ``gain``, left as such rows. Returned: ``h`` (where something was added), the rows' values in bf16 and their scales.
* ``quantize``: rows of activations, or a weight's output channels at load, made such rows. Returned: the values in bf16, the scales.
* ``product``: ``y[m, n] = a_scale[m] * w_scale[n] * sum_k a[m, k] w[n, k]``, the sum in whole numbers; plain, with a bias, with the
  gate of a feed-forward (``silu(y of w) * (y of w2)``), or added into fp32 rows (the residual stream).

Sizes are the Qwen3 dense models' layers as the benchmark names them (width 4096 / feed-forward 12288 of the 8B, 5120 / 17408 of the
14B, 5120 / 25600 of the 32B, width 2560 of the 4B), with the row counts of decode steps, mixed steps and prompts, and one product of odd sizes.
"""
import math

import torch

own = False

EPS = 1e-6
LEVELS = 127.0


# ------------------------------------------------------------------------------------------------ the cases
def _norm(name, rows, width, add, gain):
    return {"name": name, "op": "norm", "rows": rows, "width": width, "add": add, "gain": gain}


def _quantize(name, rows, width, dtype, pad=0):
    return {"name": name, "op": "quantize", "rows": rows, "width": width, "dtype": dtype, "pad": pad}


def _product(name, rows, outputs, inputs, kind="store", out="bfloat16", bias="", pad=0):
    return {"name": name, "op": "product", "rows": rows, "outputs": outputs, "inputs": inputs, "kind": kind, "out": out, "bias": bias, "pad": pad}


def listed():
    return [
        # a decode step of eight requests of the 8B: the seam in front of a sublayer, where only latency counts
        _norm("norm_8", 8, 4096, "bfloat16", "bfloat16"),
        # a step that mixes a portion of a prompt with single rows, 4B, with a sublayer's output and gains in fp32
        _norm("norm_631", 631, 2560, "float32", "float32"),
        # several prompts in one step, 14B and 32B
        _norm("norm_8192", 8192, 5120, "bfloat16", "bfloat16"),
        # the hidden rows of the 8B's feed-forward in a decode step of 64, on their way into the down product
        _quantize("quantize_64", 64, 12288, "bfloat16"),
        # the down weights of a 32B layer, when a model is loaded
        _quantize("quantize_weights", 5120, 25600, "bfloat16"),
        # decode of one request, 8B: q, k and v
        _product("product_1", 1, 6144, 4096),
        # decode of eight requests, 8B: gate and up
        _product("product_8_gated", 8, 12288, 4096, kind="gated"),
        # decode of 64 requests, 8B: down, into the residual stream
        _product("product_64_add", 64, 4096, 12288, kind="add", out="float32"),
        # sizes that no tile divides and rows that begin anywhere: small models, odd heads
        _product("product_odd", 77, 2051, 1037, out="float32", bias="float32", pad=3),
        # a mixed step of the 14B: down
        _product("product_631", 631, 5120, 17408, out="float32"),
        # a prompt of the 14B: q, k and v with biases
        _product("product_2048", 2048, 7168, 5120, bias="bfloat16"),
        # several prompts in one step, 14B: gate and up
        _product("product_8192_gated", 8192, 17408, 5120, kind="gated"),
    ]


def _spread(rng, low, high):
    """A whole number between the two, spread over its logarithm."""
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def _size(rng, low, high):
    """A width: most are multiples of 16, 64 or 128, as models have them; some are any number."""
    unit = rng.choice((1, 16, 64, 64, 128, 128))
    return max(low, _spread(rng, low, high) // unit * unit)


MOST_MULTIPLIES = 8192 * 17408 * 5120 * 2   # of the largest listed product
MOST_ENTRIES = 5120 * 25600                 # of the largest listed rows


def draw(rng):
    op = rng.choice(("norm", "quantize", "product", "product"))
    if op == "norm":
        width = _size(rng, 64, 8192)
        rows = _spread(rng, 1, min(16384, 8192 * 5120 // width))
        case = _norm("", rows, width, rng.choice(("bfloat16", "float32", "")), rng.choice(("bfloat16", "float32")))
    elif op == "quantize":
        width = _size(rng, 64, 25600)
        rows = _spread(rng, 1, min(25600, MOST_ENTRIES // width // 2))
        case = _quantize("", rows, width, rng.choice(("bfloat16", "float32")), rng.choice((0, 0, 0, 1, 8)))
    else:
        kind = rng.choice(("store", "store", "add", "gated"))
        outputs, inputs = _size(rng, 16, 25600), _size(rng, 16, 17408)
        most = MOST_MULTIPLIES // (outputs * inputs * (2 if kind == "gated" else 1))
        rows = _spread(rng, 1, max(1, min(8192, most, 8192 * 17408 // outputs)))
        case = _product("", rows, outputs, inputs, kind, "float32" if kind == "add" else rng.choice(("bfloat16", "float32")),
                        rng.choice(("", "", "bfloat16", "float32")) if kind != "gated" else "", rng.choice((0, 0, 0, 16, 5)))
    del case["name"]
    return case


# ------------------------------------------------------------------------------------------------ the inputs
def _dtype(name):
    return getattr(torch, name)


def _padded(rows, width, pad, make):
    """[rows, width] whose rows lie ``width + pad`` apart."""
    return make(rows, width + pad)[:, :width]


def _int8_rows(x):
    """What a model holds: rows of weights or activations that were made 8-bit before."""
    most = x.abs().amax(dim=1, keepdim=True)
    return (x * (LEVELS / most)).round_().to(torch.int8), (most / LEVELS).squeeze(1)


def prepare(case, seed):
    device = "cuda" if torch.cuda.is_available() else "cpu"
    gen = torch.Generator(device=device)
    gen.manual_seed(seed)

    def normal(*shape):
        return torch.randn(shape, generator=gen, device=device)

    state = {"case": case}
    if case["op"] == "norm":
        n, d = case["rows"], case["width"]
        # a residual stream: channels of different strength, a few that are far above the others, as trained models have them
        strength = torch.exp(normal(d) * 0.5)
        strength[torch.randint(0, d, (max(1, d // 512),), generator=gen, device=device)] *= 20
        state["x"] = normal(n, d) * strength
        state["gain"] = (1 + 0.1 * normal(d)).to(_dtype(case["gain"]))
        state["add"] = normal(n, d).to(_dtype(case["add"])) if case["add"] else None
        state["sum"] = torch.empty_like(state["x"]) if case["add"] else None
    elif case["op"] == "quantize":
        state["x"] = _padded(case["rows"], case["width"], case["pad"], lambda n, d: normal(n, d).to(_dtype(case["dtype"])))
    else:
        m, n, k = case["rows"], case["outputs"], case["inputs"]
        a, state["a_scale"] = _int8_rows(normal(m, k))
        state["a"] = torch.zeros((m, k + case["pad"]), dtype=torch.int8, device=device)[:, :k]
        state["a"].copy_(a)
        state["w"], state["w_scale"] = _int8_rows(normal(n, k) / math.sqrt(k))
        if case["kind"] == "gated":
            state["w2"], state["w2_scale"] = _int8_rows(normal(n, k) / math.sqrt(k))
        state["bias"] = normal(n).to(_dtype(case["bias"])) if case["bias"] else None
        if case["kind"] == "add":
            state["out"] = normal(m, n)
    return state


# ------------------------------------------------------------------------------------------------ one pass
def _plain_rows(y):
    """fp32 rows as 8-bit ones: the values that they stand for, and the scales."""
    most = y.abs().amax(dim=1, keepdim=True)
    q = torch.clamp(torch.round(y * (LEVELS / most)), -LEVELS, LEVELS)
    scale = most / LEVELS
    return (q * scale).to(torch.bfloat16), scale.squeeze(1)


def _plain_sums(a, a_scale, w, w_scale):
    return (a.float() @ w.float().t()) * a_scale[:, None] * w_scale[None, :]


def _run_plain(state):
    case = state["case"]
    if case["op"] == "quantize":
        return _plain_rows(state["x"].float())
    if case["op"] == "norm":
        h = state["x"]
        if state["add"] is not None:
            h = h + state["add"].float()
        y = h * torch.rsqrt((h * h).mean(dim=1, keepdim=True) + EPS) * state["gain"].float()
        values, scale = _plain_rows(y)
        return (values, scale) if state["add"] is None else (h, values, scale)
    y = _plain_sums(state["a"], state["a_scale"], state["w"], state["w_scale"])
    if state["bias"] is not None:
        y = y + state["bias"].float()
    if case["kind"] == "gated":
        y = y / (1 + torch.exp(-y)) * _plain_sums(state["a"], state["a_scale"], state["w2"], state["w2_scale"])
    if case["kind"] == "add":
        state["out"] += y
        return state["out"]
    return y.to(_dtype(case["out"]))


def _run_own(state):
    from jllm_serve_amd.kernels import ops
    case = state["case"]
    if case["op"] == "quantize":
        rows = ops.quantize_rows(state["x"])
        return rows.tensor(torch.bfloat16), rows.scale
    if case["op"] == "norm":
        rows = ops.rmsnorm_int8(state["x"], state["gain"], EPS, add=state["add"], out=state["sum"])
        values = rows.tensor(torch.bfloat16)
        return (values, rows.scale) if state["add"] is None else (state["sum"], values, rows.scale)
    a, w = ops.Int8Rows(state["a"], state["a_scale"]), ops.Int8Rows(state["w"], state["w_scale"])
    if case["kind"] == "gated":
        return ops.gemm_int8(a, w, w2=ops.Int8Rows(state["w2"], state["w2_scale"]), epilogue=ops.EPI_GATED, out_dtype=_dtype(case["out"]))
    if case["kind"] == "add":
        return ops.gemm_int8(a, w, bias=state["bias"], out=state["out"], epilogue=ops.EPI_ADD)
    return ops.gemm_int8(a, w, bias=state["bias"], out_dtype=_dtype(case["out"]))


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ------------------------------------------------------------------------------------------------ what it costs, what it is
def work(case):
    if case["op"] == "product":
        m, n, k = case["rows"], case["outputs"], case["inputs"]
        weights = 2 if case["kind"] == "gated" else 1
        read = m * k + 4 * m + weights * (n * k + 4 * n) + (n * _dtype(case["bias"]).itemsize if case["bias"] else 0)
        written = m * n * _dtype(case["out"]).itemsize * (2 if case["kind"] == "add" else 1)
        return {"bytes": read + written, "flops": 2 * weights * m * n * k}
    n, d = case["rows"], case["width"]
    written = n * d * 2 + 4 * n
    if case["op"] == "quantize":
        return {"bytes": n * d * _dtype(case["dtype"]).itemsize + written, "flops": 3 * n * d}
    read = n * d * 4 + d * _dtype(case["gain"]).itemsize
    if case["add"]:
        read += n * d * _dtype(case["add"]).itemsize
        written += n * d * 4
    return {"bytes": read + written, "flops": 8 * n * d}


def _exact_rows(y):
    scale = y.abs().max(dim=1).values / 127
    return torch.round(y / scale[:, None]).mul_(scale[:, None]), scale


def exact(case, seed):
    state = prepare(case, seed)
    double = torch.float64
    if case["op"] == "quantize":
        return _exact_rows(state["x"].to(double))
    if case["op"] == "norm":
        h = state["x"].to(double)
        if case["add"]:
            h += state["add"]
        y = h / torch.sqrt(torch.linalg.vecdot(h, h)[:, None] / case["width"] + EPS) * state["gain"].to(double)
        values, scale = _exact_rows(y)
        return (h, values, scale) if case["add"] else (values, scale)

    def product(w, w_scale):  # the whole numbers' sums are exact in 64 bits
        y = torch.mm(state["a"].to(double), w.to(double).t().contiguous())
        return y.mul_(torch.outer(state["a_scale"].to(double), w_scale.to(double)))

    y = product(state["w"], state["w_scale"])
    if case["bias"]:
        y += state["bias"]
    if case["kind"] == "gated":
        y = torch.sigmoid(y).mul_(y).mul_(product(state["w2"], state["w2_scale"]))
    return state["out"].to(double) + y if case["kind"] == "add" else y
