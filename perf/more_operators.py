"""Workloads of the operators that a model of tokens trains with next to its
Dense layers: the embedding (lookup with scaling, and its gradient), dropout
from a counter-based generator whose mask is never stored, and matrices in
8-bit floating point (E4M3) with one power-of-two scale for every 128 elements
along the reduced axis: quantisation, and the product of two of them.

Each case runs in two forms on the same inputs: a plain form in elementary
torch operations (``own`` false), and the calls of rgpu_b200 (``own`` true).
``exact`` gives the same results in 64 bits.
"""
import math
import random

import numpy as np
import torch

own = False

#: 8-bit floating point, E4M3
BLOCK = 128  # elements that share a scale
GROUP = 4  # scales of one row that lie side by side
TILE = 128  # rows of one scale tile
LARGEST = 448.0  # of an element

_TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
_gpu = None


# ------------------------------------------------------------------- cases
def _embedding(name, direction, tokens, width, vocabulary, table, out, spread, padding):
    """`table` and `out`: types of the embedding (its gradient is f32) and of the rows looked up (or their gradients).
    `padding`: share of positions that hold no token (an index past the vocabulary)."""
    return {"name": name, "op": "embedding", "dir": direction, "m": tokens, "n": width, "v": vocabulary, "table": table,
            "type": out, "spread": spread, "padding": padding}


def _dropout(name, direction, m, n, dtype, p, add):
    return {"name": name, "op": "dropout", "dir": direction, "m": m, "n": n, "type": dtype, "p": p, "add": add}


def _quantize(name, m, n, dtype, axis):
    return {"name": name, "op": "quantize", "m": m, "n": n, "type": dtype, "axis": axis}


def _product(name, m, n, k, out, epilogue):
    return {"name": name, "op": "product", "m": m, "n": n, "k": k, "out": out, "epilogue": epilogue}


def listed():
    return [
        # one token looked up while answering: launch latency
        _embedding("embed token bf16", "forward", 1, 4096, 32768, "bf16", "bf16", "uniform", 0.0),
        # a training batch of text: frequent tokens and rare ones, f32 master table, bf16 activations
        _embedding("embed batch bf16", "forward", 65536, 1024, 50257, "f32", "bf16", "zipf", 0.0),
        # the gradient of a small batch of categories, odd in every extent, some positions empty
        _embedding("embed back ragged f32", "backward", 2047, 1000, 1000, "f32", "f32", "uniform", 0.1),
        # the gradient of the training batch: long runs of frequent tokens, many tokens that do not occur
        _embedding("embed back batch bf16", "backward", 65536, 1024, 50257, "f32", "bf16", "zipf", 0.0),
        # hidden activations of the small network's batch
        _dropout("dropout small f32", "forward", 2048, 1024, "f32", 0.1, False),
        # a training batch of the wide model's hidden width, joined with its residual stream
        _dropout("dropout batch bf16", "forward", 8192, 8192, "bf16", 0.1, True),
        # the gradient of an odd batch, rows that start at any 2-byte boundary
        _dropout("dropout back ragged bf16", "backward", 4099, 1001, "bf16", 0.5, False),
        # a batch of activations before a product, to 8 bits and back
        _quantize("quantize batch bf16", 8192, 8192, "bf16", 1),
        # a layer's weights [inputs, outputs], scales along the inputs: laid out transposed
        _quantize("quantize weights f32", 4096, 8192, "f32", 0),
        # one token through a layer: the weights are read once
        _product("product token", 1, 8192, 8192, "bf16", "bias"),
        # logits of an odd batch over 1000 classes
        _product("product logits f32", 2047, 1000, 8192, "f32", "bias"),
        # a training batch through the widest layer
        _product("product batch", 8192, 8192, 8192, "bf16", "bias_relu"),
    ]


def _log(rng, lo, hi):
    """A whole number of [lo, hi], even over its logarithm; one time in three a multiple of 64."""
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    if rng.random() < 1 / 3 and v > 64:
        v = v // 64 * 64
    return max(lo, min(hi, v))


def draw(rng):
    op = rng.choice(("forward", "backward", "dropout", "quantize", "product", "product"))
    if op == "product":
        case = _product("", _log(rng, 1, 8192), _log(rng, 64, 8192), _log(rng, 32, 8192), rng.choice(("bf16", "f32")),
                        rng.choice(("none", "bias", "bias_relu")))
    elif op == "quantize":
        n = _log(rng, 32, 16384)
        case = _quantize("", _log(rng, 1, min(16384, (1 << 25) // n)), n, rng.choice(("bf16", "f32")), rng.choice((0, 1)))
    elif op == "dropout":
        n = _log(rng, 32, 16384)
        case = _dropout("", rng.choice(("forward", "backward")), _log(rng, 1, min(65536, (1 << 25) // n)), n,
                        rng.choice(("bf16", "f32")), rng.choice((0.05, 0.1, 0.25, 0.5)), False)
        case["add"] = case["dir"] == "forward" and rng.random() < 0.5
    else:
        n = _log(rng, 32, 8192)
        case = _embedding("", op, _log(rng, 1, min(65536, (1 << 25) // n)), n, _log(rng, 16, min(65536, (1 << 25) // n)),
                          rng.choice(("bf16", "f32")) if op == "forward" else "f32", rng.choice(("bf16", "f32")),
                          rng.choice(("uniform", "zipf")), rng.choice((0.0, 0.1)))
    del case["name"]
    return case


def _share(case):
    """How often each token of the vocabulary is met: all alike, or as its rank's inverse (the words of a text)."""
    p = np.ones(case["v"]) if case["spread"] == "uniform" else 1.0 / np.arange(1, case["v"] + 1)
    return p / p.sum()


def work(case):
    m, n = case["m"], case["n"]
    if case["op"] == "product":
        k = case["k"]
        held = (m + n) * (k + math.ceil(k / BLOCK))
        bias = 0 if case["epilogue"] == "none" else 4 * n
        return {"bytes": held + bias + m * n * (2 if case["out"] == "bf16" else 4), "flops": 2 * m * n * k}
    size = 2 if case["type"] == "bf16" else 4
    if case["op"] == "quantize":
        held = m * n + (m * math.ceil(n / BLOCK) if case["axis"] == 1 else n * math.ceil(m / BLOCK))
        return {"bytes": 2 * m * n * size + held, "flops": 4 * m * n}
    if case["op"] == "dropout":
        # ten rounds of two products and four exclusive ors for eight elements; a comparison, a product, a choice
        return {"bytes": (3 if case["add"] else 2) * m * n * size, "flops": (10 * 6 / 8 + 3) * m * n}
    full = round(m * (1.0 - case["padding"]))  # positions that hold a token
    if case["dir"] == "backward":
        return {"bytes": 4 * m + full * n * size + 4 * case["v"] * n, "flops": 2 * full * n}
    met = float((1.0 - (1.0 - _share(case)) ** full).sum())  # distinct tokens to be expected
    return {"bytes": 4 * m + met * n * (2 if case["table"] == "bf16" else 4) + m * n * size, "flops": full * n}


# ------------------------------------------------------------------ inputs
def prepare(case, seed):
    g = torch.Generator("cuda").manual_seed(seed)

    def normal(*shape, std=1.0):
        return torch.randn(*shape, device="cuda", generator=g) * std

    s = {"case": case}
    m, n = case["m"], case["n"]
    if case["op"] == "product":
        k = case["k"]
        # activations with a few strong channels, weights of a Kaiming spread
        s["a"] = _held(normal(m, k) * torch.exp(normal(1, k, std=0.7)))
        s["b"] = _held(normal(n, k, std=math.sqrt(2.0 / k)))
        if case["epilogue"] != "none":
            s["bias"] = normal(1, n, std=0.1)
    elif case["op"] == "quantize":
        spread = torch.exp(normal(1, n, std=0.7)) if case["axis"] == 1 else math.sqrt(2.0 / m)
        s["x"] = (normal(m, n) * spread).to(_TYPES[case["type"]])
    elif case["op"] == "dropout":
        t = _TYPES[case["type"]]
        # a hidden layer's activations after ReLU, or a gradient
        s["x"] = (normal(m, n).clamp_min(0) if case["dir"] == "forward" else normal(m, n, std=0.01)).to(t)
        if case["add"]:
            s["add"] = (normal(m, n) * 1.5).to(t)
        r = random.Random(seed)
        s["seed"], s["site"], s["step"], s["row"] = r.getrandbits(64), r.randrange(16), r.randrange(100000), r.randrange(8) * m
    else:
        v = case["v"]
        share = torch.from_numpy(np.cumsum(_share(case))).cuda()
        rank = torch.searchsorted(share, torch.rand(m, device="cuda", generator=g, dtype=torch.float64)).clamp_max(v - 1)
        tokens = torch.randperm(v, device="cuda", generator=g)[rank]  # frequent tokens anywhere in the table
        if case["padding"]:
            tokens = torch.where(torch.rand(m, device="cuda", generator=g) < case["padding"], v, tokens)
        s["tokens"] = tokens.to(torch.int32)
        s["scale"] = math.sqrt(n)
        if case["dir"] == "forward":
            s["table"] = normal(v, n, std=1.0 / math.sqrt(n)).to(_TYPES[case["table"]])
        else:
            s["dy"] = normal(m, n, std=0.01).to(_TYPES[case["type"]])
    if own:
        _attach(s)  # the handles and buffers that a program keeps beside its tensors
    return s


# -------------------------------------------------------------- plain form
def _power(e, dtype=torch.float32):
    """2^e of whole numbers e in [-149, 127], exactly (a power function may be a last place off, which decides ties)."""
    return torch.from_numpy(np.ldexp(1.0, np.arange(-149, 128))).to(e.device, dtype)[e.long() + 149]


def _fp8(x):
    """(E4M3 values, scale exponents) of x [rows, k] in f32, k padded with zeros to whole blocks."""
    rows, k = x.shape
    blocks = -(-k // BLOCK)
    if blocks * BLOCK != k:
        x = torch.cat([x, x.new_zeros(rows, blocks * BLOCK - k)], 1)
    x = x.view(rows, blocks, BLOCK)
    amax = x.abs().amax(2, keepdim=True)
    # the least exponent that brings amax to 448 = 1.75 * 2^8 or less, from amax's bits: a mantissa above 0.75 carries over
    e = ((amax.view(torch.int32) + 0x1FFFFF) >> 23) - 127 - 8
    e = e.clamp_min(-127)
    return (x * _power(-e)).to(torch.float8_e4m3fn), e


def _held(x):
    """x [rows, k] as it is held: a byte an element, rows of whole 16 bytes; scales in tiles of 128 rows by 4 blocks,
    byte [row % 32][row // 32 % 4][block % 4] of tile [row // 128][block // 4]."""
    q, e = _fp8(x)
    rows, blocks = q.shape[:2]
    stride = -(-x.shape[1] // 16) * 16
    groups, tiles = -(-blocks // GROUP), -(-rows // TILE)
    scales = torch.zeros(tiles * TILE, groups * GROUP, dtype=torch.uint8, device=x.device)
    scales[:rows, :blocks] = (e.view(rows, blocks) + 127).to(torch.uint8)
    scales = scales.view(tiles, 4, 32, groups, GROUP).permute(0, 3, 2, 1, 4).contiguous()
    return {"codes": q.view(torch.uint8).view(rows, -1)[:, :stride].contiguous(), "scales": scales, "rows": rows, "k": x.shape[1]}


def _values(h, dtype):
    """What a held matrix stands for, [rows, k]."""
    rows, k = h["rows"], h["k"]
    scales = h["scales"].permute(0, 3, 2, 1, 4).reshape(-1, h["scales"].shape[1] * GROUP)[:rows]
    unit = _power(scales.to(torch.int32) - 127, dtype)
    return h["codes"].view(torch.float8_e4m3fn)[:, :k].to(dtype) * unit.repeat_interleave(BLOCK, 1)[:, :k]


def _philox(c, key):
    """Ten rounds of Philox4x32 (Salmon, Moraes, Dror, Shaw 2011) on 32-bit words held in 64 bits: four counter words, two of key."""
    low = 0xFFFFFFFF

    def high(a, m):  # upper half of a 32 x 32-bit product
        return ((a >> 16) * m + (((a & 0xFFFF) * m) >> 16)) >> 16

    k0, k1 = key
    for _ in range(10):
        c = (high(c[2], 0xCD9E8D57) ^ c[1] ^ k0, (c[2] * 0xCD9E8D57) & low, high(c[0], 0xD2511F53) ^ c[3] ^ k1,
             (c[0] * 0xD2511F53) & low)
        k0, k1 = (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low
    return c


def _dropout_plain(s):
    c = s["case"]
    m, n, drop = c["m"], c["n"], round(c["p"] * 65536)
    column = torch.arange(-(-n // 8), device="cuda").view(1, -1)
    row = torch.arange(s["row"], s["row"] + m, device="cuda").view(-1, 1)
    zero = torch.zeros(m, column.shape[1], dtype=torch.int64, device="cuda")
    words = _philox((zero + column, zero + row, zero + s["step"], zero + s["site"]), (s["seed"] & 0xFFFFFFFF, s["seed"] >> 32))
    bits = torch.stack([words[i // 2] >> 16 * (i % 2) & 0xFFFF for i in range(8)], 2).view(m, -1)[:, :n]
    y = torch.where(bits >= drop, s["x"].float() * (65536.0 / (65536 - drop)), 0.0)
    if "add" in s:
        y = s["add"].float() + y
    return {"y" if c["dir"] == "forward" else "dx": y.to(s["x"].dtype)}


def _embedding_plain(s):
    c, tokens = s["case"], s["tokens"].long()
    there = (tokens < c["v"]).unsqueeze(1)
    tokens = torch.where(there[:, 0], tokens, 0)
    if c["dir"] == "forward":
        return {"y": torch.where(there, s["table"][tokens].float() * s["scale"], 0.0).to(_TYPES[c["type"]])}
    # long sums: in 64 bits
    d = torch.zeros(c["v"], c["n"], dtype=torch.float64, device="cuda")
    d.index_add_(0, tokens, torch.where(there, s["dy"].double(), 0.0))
    return {"dtable": (d * s["scale"]).float()}


def _product_plain(s):
    c = s["case"]
    v = _values(s["a"], torch.float32) @ _values(s["b"], torch.float32).T
    if "bias" in s:
        v = v + s["bias"]
    if c["epilogue"] == "bias_relu":
        v = v.clamp_min(0)
    return {"c": v.to(_TYPES[c["out"]])}


def _quantize_plain(s):
    c = s["case"]
    x = s["x"].float()
    x = x.T.contiguous() if c["axis"] == 0 else x
    q, e = _fp8(x)
    v = q.float() * _power(e)
    return {"values": v.view(x.shape[0], -1)[:, :x.shape[1]].to(s["x"].dtype)}


# ------------------------------------------------------ the framework's form
def _attach(s):
    """Handles of the state's tensors and buffers for the outputs; no input is read."""
    global _gpu
    import rgpu_b200 as rg

    if _gpu is None:
        _gpu = rg.Gpu(torch.cuda.current_device())
    c = s["case"]
    kinds = {torch.bfloat16: "bf16", torch.float32: "f32", torch.int32: "u32"}

    def wrap(t):
        return _gpu.wrap(t.data_ptr(), t.shape, kinds[t.dtype])

    def held(h):
        return _gpu.fp8_wrap(h["codes"].data_ptr(), h["scales"].data_ptr(), h["rows"], h["k"])

    def buffer(name, shape, t):
        s["out"] = {name: torch.empty(shape, dtype=t, device="cuda")}
        s["to"] = wrap(s["out"][name])

    m, n = c["m"], c["n"]
    if c["op"] == "product":
        buffer("c", (m, n), _TYPES[c["out"]])
        s["qa"], s["qb"] = held(s["a"]), held(s["b"])
        s["qbias"] = wrap(s["bias"]) if "bias" in s else None
    elif c["op"] == "quantize":
        shape = (m, n) if c["axis"] == 1 else (n, m)
        buffer("values", shape, s["x"].dtype)
        s["qx"], s["q"] = wrap(s["x"]), _gpu.fp8_zeros(*shape)
    elif c["op"] == "dropout":
        buffer("y" if c["dir"] == "forward" else "dx", (m, n), s["x"].dtype)
        s["qx"], s["qadd"] = wrap(s["x"]), wrap(s["add"]) if "add" in s else None
        s["mask"] = rg.Dropout(c["p"], s["seed"], site=s["site"], step=s["step"], first_row=s["row"])
    else:
        s["qtokens"] = wrap(s["tokens"])
        if c["dir"] == "forward":
            buffer("y", (m, n), _TYPES[c["type"]])
            s["qtable"] = wrap(s["table"])
        else:
            buffer("dtable", (c["v"], n), torch.float32)
            s["qdy"] = wrap(s["dy"])
            s["work"] = _gpu.zeros((_gpu.embedding_backward_workspace(m, c["v"], n),))


def _run_own(s):
    c = s["case"]
    if c["op"] == "product":
        _gpu.fp8_matmul(s["qa"], s["qb"], s["to"], bias=s["qbias"], relu=c["epilogue"] == "bias_relu")
    elif c["op"] == "quantize":
        _gpu.fp8_quantize(s["qx"], s["q"], axis=c["axis"])
        _gpu.fp8_dequantize(s["q"], s["to"])
    elif c["op"] == "dropout":
        _gpu.dropout(s["qx"], s["to"], s["mask"], add=s["qadd"])
    elif c["dir"] == "forward":
        _gpu.embedding_forward(s["qtable"], s["qtokens"], s["to"], scale=s["scale"])
    else:
        _gpu.embedding_backward(s["qtokens"], s["qdy"], s["to"], s["work"], scale=s["scale"])
    return s["out"]


def run(state):
    if own:
        return _run_own(state)
    return {"product": _product_plain, "quantize": _quantize_plain, "dropout": _dropout_plain,
            "embedding": _embedding_plain}[state["case"]["op"]](state)


# ------------------------------------------------------------ in 64 bits
def _exact_fp8(x):
    """The values that x [rows, k] stands for in the 8-bit form, from the definition, in 64 bits."""
    rows, k = x.shape
    whole = torch.zeros(rows, -(-k // BLOCK) * BLOCK, dtype=torch.float64, device=x.device)
    whole[:, :k] = x.double()
    b = whole.view(rows, -1, BLOCK)
    top = b.abs().max(2, keepdim=True).values
    mantissa, exponent = torch.frexp(top / LARGEST)  # top / 448 = mantissa 2^exponent, mantissa in [0.5, 1)
    exponent = torch.where(mantissa == 0.5, exponent - 1, exponent)
    unit = _power(torch.where(top > 0, exponent, -127).clamp_min(-127), torch.float64)
    a = b / unit
    # neighbours are 2^-3 of the power of two below apart, 2^-9 at least; ties go to the even one
    step = _power((torch.frexp(a).exponent - 1).clamp_min(-6) - 3, torch.float64)
    return (torch.round(a / step) * step * unit).view(rows, -1)[:, :k]


def _exact_keep(s):
    """Which elements are kept: the generator's words by numpy's unsigned integers."""
    c = s["case"]
    m, n = c["m"], c["n"]
    low, shift = np.uint64(0xFFFFFFFF), np.uint64(32)
    x = [np.broadcast_to(v, (m, -(-n // 8))).astype(np.uint64) for v in
         (np.arange(-(-n // 8))[None], np.arange(s["row"], s["row"] + m)[:, None], s["step"], s["site"])]
    k = [s["seed"] % 2 ** 32, s["seed"] // 2 ** 32]
    for _ in range(10):
        p, q = x[0] * np.uint64(0xD2511F53), x[2] * np.uint64(0xCD9E8D57)
        x = [(q >> shift) ^ x[1] ^ np.uint64(k[0]), q & low, (p >> shift) ^ x[3] ^ np.uint64(k[1]), p & low]
        k = [(k[0] + 0x9E3779B9) % 2 ** 32, (k[1] + 0xBB67AE85) % 2 ** 32]
    words = np.stack(x, 2).astype("<u4").view("<u2").reshape(m, -1)[:, :n]
    return torch.from_numpy(words >= round(c["p"] * 65536)).cuda()


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "product":
        v = _values(s["a"], torch.float64).mm(_values(s["b"], torch.float64).t())
        if "bias" in s:
            v += s["bias"].double()
        return {"c": torch.relu(v) if case["epilogue"] == "bias_relu" else v}
    if case["op"] == "quantize":
        return {"values": _exact_fp8(s["x"] if case["axis"] == 1 else s["x"].t())}
    if case["op"] == "dropout":
        keep = _exact_keep(s)
        kept = 1.0 - round(case["p"] * 65536) / 65536
        y = s["x"].double() / kept * keep
        return {"y": y + s["add"].double() if "add" in s else y} if case["dir"] == "forward" else {"dx": y}
    tokens = s["tokens"].long()
    if case["dir"] == "forward":
        table = torch.cat([s["table"].double(), torch.zeros(1, case["n"], dtype=torch.float64, device="cuda")])
        return {"y": table.index_select(0, tokens) * s["scale"]}
    # sums of runs of the sorted tokens as differences of running sums
    order = torch.argsort(tokens, stable=True)
    running = torch.zeros(case["m"] + 1, case["n"], dtype=torch.float64, device="cuda")
    torch.cumsum(s["dy"].double()[order], 0, out=running[1:])
    ends = torch.searchsorted(tokens[order], torch.arange(case["v"] + 1, device="cuda"))
    return {"dtable": (running[ends[1:]] - running[ends[:-1]]) * s["scale"]}
