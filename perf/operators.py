"""Microscaled 4-bit floating point (MXFP4): the cases whose speed is watched, and the operators in their plain form.

A block of 32 neighbouring values shares a power of two; a value is one of 0, 0.5, 1, 1.5, 2, 3, 4, 6 with a sign, times it.
Two values lie in a byte (the even one low), the exponents (plus 127) four to a word, ``[ceil(k / 128), rows]``.

Three kinds of pass:

* ``quantize``: rows of 16 or 32 bits, as they lie or gathered for their experts, into codes and exponents, and those back into
  values.
* ``linear``: rows of activations times a weight matrix, both in 4 bits, with or without a bias.
* ``experts``: rows sorted by expert times their experts' matrices; gate and up as pairs that leave as one value in 16 bits, or
  down products that leave in 32."""

import math

import torch

own = False

TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
MOST_OPERATIONS = 2 * 4096 * 14336 * 4096
MOST_VALUES = 14336 * 4096


def listed():
    return [
        # one token's activations on their way into a product: the smallest call
        {"name": "quantize f16 1 x 4096", "kind": "quantize", "type": "f16", "rows": 1, "k": 4096, "gather": 0},
        # a prompt's activations, each token's row for both of its experts
        {"name": "quantize bf16 2048 x 4096 for 2 experts each", "kind": "quantize", "type": "bf16", "rows": 2048, "k": 4096, "gather": 2},
        # a weight matrix of a checkpoint in 32 bits, when a model is loaded
        {"name": "quantize f32 14336 x 4096", "kind": "quantize", "type": "f32", "rows": 14336, "k": 4096, "gather": 0},
        # one user's token through the largest matrix of an 8B-shaped block: the weight stream
        {"name": "linear f16 1 x 4096 x 14336", "kind": "linear", "type": "f16", "m": 1, "n": 14336, "k": 4096, "bias": False},
        # eight users through its down projection: a long sum, few columns
        {"name": "linear bf16 8 x 14336 x 4096", "kind": "linear", "type": "bf16", "m": 8, "n": 4096, "k": 14336, "bias": True},
        # a short question to a small model: k is no multiple of 128
        {"name": "linear f16 33 x 576 x 1536", "kind": "linear", "type": "f16", "m": 33, "n": 1536, "k": 576, "bias": False},
        # the output projection of a full batch, logits in 32 bits
        {"name": "linear f32 32 x 4096 x 128256", "kind": "linear", "type": "f32", "m": 32, "n": 128256, "k": 4096, "bias": False},
        # a prompt of odd length through a block of width 2048
        {"name": "linear bf16 777 x 2048 x 7168", "kind": "linear", "type": "bf16", "m": 777, "n": 7168, "k": 2048, "bias": True},
        # a document through the largest matrix of an 8B-shaped block
        {"name": "linear f16 4096 x 4096 x 14336", "kind": "linear", "type": "f16", "m": 4096, "n": 14336, "k": 4096, "bias": False},
        # one token through the gate and up rows of its two experts
        {"name": "experts up bf16 1 x 2 of 16, 4096 x 7168", "kind": "experts", "type": "bf16", "tokens": 1, "top": 2, "experts": 16,
         "n": 7168, "k": 4096, "paired": True},
        # a full batch through the down rows of its experts, some of which nobody chose
        {"name": "experts down bf16 32 x 2 of 16, 1792 x 2048", "kind": "experts", "type": "bf16", "tokens": 32, "top": 2, "experts": 16,
         "n": 2048, "k": 1792, "paired": False},
        # a prompt through the gate and up rows of all experts, ragged and uneven
        {"name": "experts up f16 2048 x 2 of 16, 4096 x 7168", "kind": "experts", "type": "f16", "tokens": 2048, "top": 2, "experts": 16,
         "n": 7168, "k": 4096, "paired": True},
    ]


def _spread(rng, low, high):
    """Whole numbers spread over their logarithm."""
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def _length(rng, high):
    """A contraction's length: whole blocks, half of the time whole groups of four."""
    return 128 * _spread(rng, 1, high // 128) if rng.random() < 0.5 else 32 * _spread(rng, 2, high // 32)


def draw(rng):
    kind = rng.choice(("quantize", "linear", "linear", "experts"))
    if kind == "quantize":
        k, gather = _length(rng, 14336), rng.choice((0, 0, 1, 2, 4))
        return {"kind": kind, "type": rng.choice(("f16", "bf16", "f32")), "rows": _spread(rng, 1, max(1, min(16384, MOST_VALUES // (k * max(gather, 1))))),
                "k": k, "gather": gather}
    if kind == "linear":
        k, n = _length(rng, 14336), _spread(rng, 8, 32768)
        return {"kind": kind, "type": rng.choice(("f16", "bf16", "f32")), "m": _spread(rng, 1, max(1, min(4096, MOST_OPERATIONS // (2 * n * k)))),
                "n": n, "k": k, "bias": rng.random() < 0.5}
    experts, paired = _spread(rng, 2, 64), rng.random() < 0.5
    top, k = rng.randint(1, min(4, experts)), _length(rng, 4096)
    n = _spread(rng, 32, max(32, min(8192, (1 << 28) // (experts * k)))) // 2 * 2
    return {"kind": kind, "type": rng.choice(("f16", "bf16")), "tokens": _spread(rng, 1, max(1, min(2048, MOST_OPERATIONS // (8 * n * k * top)))),
            "top": top, "experts": experts, "n": n, "k": k, "paired": paired}


# ---- the operators in their plain form ----------------------------------------------------------------

def quantized(x):
    """Codes uint8 [rows, k / 2] and exponent words int32 [ceil(k / 128), rows] of x [rows, k]."""
    rows, k = x.shape
    blocks = x.float().reshape(rows, k // 32, 32)
    # frexp gives a fraction in [0.5, 1): the largest value's power of two is one less, and 4 to 8 is where it should lie
    shift = (torch.frexp(blocks.abs().amax(-1)).exponent - 3).clamp(-127, 127)
    scaled = torch.ldexp(blocks, -shift.unsqueeze(-1))
    size = scaled.abs()
    # steps of 0.5 up to 2, of 1 up to 4, of 2 beyond; torch.round takes ties to the even number, which is the even code
    code = torch.where(size < 2, torch.round(size * 2), torch.where(size < 4, torch.round(size) + 2, (torch.round(size / 2) + 4).clamp(max=7)))
    code = code.to(torch.uint8) | torch.where(torch.signbit(scaled), 8, 0).to(torch.uint8)
    code = code.reshape(rows, k)
    codes = code[:, 0::2] | (code[:, 1::2] << 4)
    exponents = torch.zeros(rows, (k + 127) // 128 * 4, dtype=torch.uint8, device=x.device)
    exponents[:, :k // 32] = (shift + 127).to(torch.uint8)
    words = exponents.reshape(rows, -1, 4).transpose(0, 1).contiguous().view(torch.int32).squeeze(-1)
    return codes, words


def values(codes, words):
    """The values in 32 bits, [rows, k], of codes and exponent words."""
    rows, k = codes.shape[0], codes.shape[1] * 2
    table = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0], device=codes.device)
    both = torch.stack((table[(codes & 15).int()], table[(codes >> 4).int()]), dim=-1).reshape(rows, k // 32, 32)
    exponents = words.contiguous().unsqueeze(-1).view(torch.uint8).transpose(0, 1).reshape(rows, -1)[:, :k // 32]
    return torch.ldexp(both, exponents.int().unsqueeze(-1) - 127).reshape(rows, k)


def _linear(s):
    y = values(s["x"], s["x_scales"]) @ values(s["w"], s["w_scales"]).T
    if s["bias"] is not None:
        y = y + s["bias"].float()
    return y.to(s["out"].dtype)


def _experts(s):
    x, w = values(s["x"], s["x_scales"]), values(s["w"], s["w_scales"])
    experts, n, k = s["experts"], s["n"], s["k"]
    rows = torch.zeros(experts, s["most_rows"], k, device=x.device)
    rows[s["expert_of_slot"], s["place_of_slot"]] = x
    y = torch.bmm(rows, w.reshape(experts, n, k).transpose(1, 2))[s["expert_of_slot"], s["place_of_slot"]]
    if not s["paired"]:
        return y
    gate, up = (y * s["scores"].unsqueeze(-1)).reshape(-1, n // 2, 2).unbind(-1)
    return (gate / (1 + torch.exp(-gate)) * up).to(s["out"].dtype)


# ---- inputs ---------------------------------------------------------------------------------------------

def _generator(seed):
    return torch.Generator("cuda").manual_seed(int(seed) & 0x7FFFFFFFFFFFFFFF)


def _activations(g, rows, k):
    """Rows of unlike size with a few columns that stand out, as a layer's inputs have them."""
    columns = torch.where(torch.rand(k, generator=g, device="cuda") < 0.01, 8.0, 1.0)
    sizes = torch.exp(0.5 * torch.randn(rows, 1, generator=g, device="cuda"))
    return torch.randn(rows, k, generator=g, device="cuda") * columns * sizes


def _weights(g, n, k):
    return torch.randn(n, k, generator=g, device="cuda") / math.sqrt(k)


def _routing(g, tokens, top, experts):
    """A router's choices, some experts far more often than others, sorted by expert: the row, expert, score and place of every
    slot, the tiles of at most 128 slots, and the most rows of an expert."""
    favour = 1.5 * torch.randn(experts, generator=g, device="cuda")
    logits = torch.randn(tokens, experts, generator=g, device="cuda") + favour
    best, chosen = torch.topk(logits, top, dim=1)
    expert, order = torch.sort(chosen.reshape(-1), stable=True)
    counts = torch.bincount(expert, minlength=experts)
    first = torch.cumsum(counts, 0) - counts
    tiles_of = (counts + 127) // 128
    owner = torch.repeat_interleave(torch.arange(experts, device="cuda"), tiles_of)
    turn = torch.arange(owner.numel(), device="cuda") - (torch.cumsum(tiles_of, 0) - tiles_of)[owner]
    begin = first[owner] + 128 * turn
    end = torch.minimum(begin + 128, first[owner] + counts[owner])
    pairs = tokens * top
    plan = torch.zeros(1 + pairs // 128 + min(experts, pairs), 4, dtype=torch.int32, device="cuda")
    plan[0, 0] = owner.numel()
    plan[1:1 + owner.numel()] = torch.stack((owner, begin, end, torch.zeros_like(owner)), 1).int()
    place = torch.arange(pairs, device="cuda") - first[expert]
    return (order // top).int(), expert, torch.sigmoid(best.reshape(-1))[order].contiguous(), place, plan, int(counts.max())


def prepare(case, seed):
    g, kind = _generator(seed), case["kind"]
    element = TYPES[case["type"]]
    if kind == "quantize":
        rows, k, gather = case["rows"], case["k"], case["gather"]
        out_rows = rows * max(gather, 1)
        index = None
        if gather:
            index = torch.randperm(out_rows, generator=g, device="cuda").remainder(rows).int()
        x = _activations(g, rows, k) if rows < 4096 else _weights(g, rows, k)
        return {"kind": kind, "type": case["type"], "x": x.to(element), "index": index, "rows": out_rows, "source_rows": rows, "k": k,
                "codes": torch.empty(out_rows, k // 2, dtype=torch.uint8, device="cuda"),
                "scales": torch.empty((k + 127) // 128, out_rows, dtype=torch.int32, device="cuda"),
                "out": torch.empty(out_rows, k, dtype=element, device="cuda")}
    if kind == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        x, x_scales = quantized(_activations(g, m, k))
        w, w_scales = quantized(_weights(g, n, k))
        bias = (0.1 * torch.randn(n, generator=g, device="cuda")).to(element) if case["bias"] else None
        return {"kind": kind, "type": case["type"], "x": x, "x_scales": x_scales, "w": w, "w_scales": w_scales, "bias": bias, "m": m, "n": n,
                "k": k, "out": torch.empty(m, n, dtype=element, device="cuda")}
    n, k, experts, pairs = case["n"], case["k"], case["experts"], case["tokens"] * case["top"]
    row, expert, scores, place, plan, most_rows = _routing(g, case["tokens"], case["top"], experts)
    x, x_scales = quantized(_activations(g, case["tokens"], k)[row.long()])
    w, w_scales = quantized(_weights(g, experts * n, k))
    out = torch.empty(pairs, n // 2, dtype=element, device="cuda") if case["paired"] else torch.empty(pairs, n, device="cuda")
    return {"kind": kind, "type": case["type"], "x": x, "x_scales": x_scales, "w": w, "w_scales": w_scales, "plan": plan, "scores": scores,
            "expert_of_slot": expert, "place_of_slot": place, "most_rows": most_rows, "pairs": pairs, "n": n, "k": k, "experts": experts,
            "paired": case["paired"], "out": out}


# ---- a pass -----------------------------------------------------------------------------------------------

_runtime = None


def _own(s):
    global _runtime
    if _runtime is None:
        from llmopt_b200.cuda_native import Runtime

        _runtime = Runtime(0)
    stream = torch.cuda.current_stream().cuda_stream
    out = s["out"].data_ptr()
    if s["kind"] == "quantize":
        codes, scales = s["codes"].data_ptr(), s["scales"].data_ptr()
        _runtime.mxfp4_quantize_pointers(s["type"], s["x"].data_ptr(), None if s["index"] is None else s["index"].data_ptr(), codes, scales,
                                         s["rows"], s["source_rows"], s["k"], s["k"], stream)
        _runtime.mxfp4_dequantize_pointers(s["type"], codes, scales, out, s["rows"], s["k"], stream)
    elif s["kind"] == "linear":
        _runtime.mxfp4_linear_pointers(s["type"], s["x"].data_ptr(), s["x_scales"].data_ptr(), s["w"].data_ptr(), s["w_scales"].data_ptr(),
                                       None if s["bias"] is None else s["bias"].data_ptr(), out, s["m"], s["n"], s["k"], stream)
    else:
        _runtime.mxfp4_expert_rows_pointers(s["type"], s["x"].data_ptr(), s["x_scales"].data_ptr(), s["w"].data_ptr(), s["w_scales"].data_ptr(),
                                            s["plan"].data_ptr(), s["scores"].data_ptr(), out, s["pairs"], s["n"], s["k"], s["experts"],
                                            s["paired"], stream)
    return s["out"]


def run(state):
    if own:
        return _own(state)
    if state["kind"] == "quantize":
        x = state["x"] if state["index"] is None else state["x"][state["index"].long()]
        return values(*quantized(x)).to(x.dtype)
    return _linear(state) if state["kind"] == "linear" else _experts(state)


def work(case):
    k = case["k"]
    held = k // 2 + k // 32  # bytes of a row in 4 bits
    size = 4 if case["type"] == "f32" else 2
    if case["kind"] == "quantize":
        rows = case["rows"] * max(case["gather"], 1)
        return {"bytes": case["rows"] * k * size + rows * (held + k * size + (4 if case["gather"] else 0)), "flops": 4 * rows * k}
    if case["kind"] == "linear":
        m, n = case["m"], case["n"]
        return {"bytes": (m + n) * held + m * n * size + (n * size if case["bias"] else 0), "flops": 2 * m * n * k}
    pairs, n = case["tokens"] * case["top"], case["n"]
    chosen = min(case["experts"], pairs)  # the most experts that can be read
    result = pairs * n // 2 * size if case["paired"] else pairs * n * 4
    return {"bytes": pairs * held + chosen * n * held + result + 8 * pairs, "flops": 2 * pairs * n * k}


# ---- 64 bits ----------------------------------------------------------------------------------------------

def _exact_values(codes, words, first=0, end=None):
    """The values of rows first to end from the format's definition: sign, two bits of exponent, one of fraction."""
    codes, words = codes[first:end], words[:, first:end]
    k = codes.shape[1] * 2
    nibble = torch.empty(codes.shape[0], k, dtype=torch.float64, device=codes.device)
    for half in range(2):
        n = ((codes >> (4 * half)) & 15).to(torch.int64)
        exponent, fraction = (n >> 1) & 3, (n & 1).double()
        size = torch.where(exponent == 0, fraction / 2, (1 + fraction / 2) * torch.pow(2.0, (exponent - 1).double()))
        nibble[:, half::2] = torch.where(n >= 8, -size, size)
    block = torch.arange(k, device=codes.device) // 32
    shared = (words.long()[block // 4].T >> (8 * (block % 4))) & 255
    return nibble * torch.pow(torch.tensor(2.0, dtype=torch.float64, device=codes.device), (shared - 127).double())


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "quantize":
        x = s["x"].double() if s["index"] is None else s["x"].double()[s["index"].long()]
        blocks = x.reshape(s["rows"], -1, 32)
        most = blocks.abs().amax(-1, keepdim=True)
        power = torch.floor(torch.log2(torch.where(most == 0, torch.ones_like(most), most)))
        # log2 in 64 bits of a value in 16 or 32 bits can only miss a power of two by its rounding
        power = power + (torch.pow(2.0, power + 1) <= most).double() - (torch.pow(2.0, power) > most).double() * (most > 0)
        scale = torch.pow(2.0, (power - 2).clamp(-127, 127))
        grid = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64, device=x.device)
        size = blocks.abs() / scale
        # the nearest of the eight; halfway the one with the even index
        middle = (grid[1:] + grid[:-1]) / 2
        below = torch.bucketize(size, middle)  # ties count as below
        tie = (size == middle[below.clamp(max=6)]) & (below < 7) & (below % 2 == 1)
        return torch.copysign(grid[below + tie.long()] * scale, blocks).reshape(s["rows"], s["k"])
    if case["kind"] == "linear":
        x = _exact_values(s["x"], s["x_scales"])
        out = torch.empty(s["m"], s["n"], dtype=torch.float64, device="cuda")
        for n0 in range(0, s["n"], 8192):
            out[:, n0:n0 + 8192] = x @ _exact_values(s["w"], s["w_scales"], n0, min(s["n"], n0 + 8192)).T
        return out if s["bias"] is None else out + s["bias"].double()
    n = s["n"]
    out = torch.empty(s["pairs"], n, dtype=torch.float64, device="cuda")
    for e in range(s["experts"]):
        slots = (s["expert_of_slot"] == e).nonzero().squeeze(1)
        if slots.numel():
            x = _exact_values(s["x"][slots], s["x_scales"][:, slots])
            out[slots] = x @ _exact_values(s["w"], s["w_scales"], e * n, (e + 1) * n).T
    if not s["paired"]:
        return out
    y = out * s["scores"].double().unsqueeze(1)
    gate, up = y[:, 0::2], y[:, 1::2]
    return gate * torch.sigmoid(gate) * up
