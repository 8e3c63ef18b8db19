"""MXFP4 on the GPU against its definition in 64 bits: conversions to the last bit, products within what fp32 sums and one rounding of the
output's type can be off, rows and columns outside of a result as they were."""

import numpy as np
import pytest

import mxfp4_oracle as mx

pytestmark = pytest.mark.gpu

HALF_STEP = {"float16": 2.0 ** -11, "bfloat16": 2.0 ** -8, "float32": 2.0 ** -24}
NAMES = {"float16": "f16", "bfloat16": "bf16", "float32": "f32"}
CANARY = 0xA5


def to_bits(values, dtype):
    """What a device buffer of ``dtype`` holds of float values (rounded to nearest, ties to even)."""
    with np.errstate(over="ignore"):
        values = np.ascontiguousarray(values, np.float32)
    if dtype != "bfloat16":
        with np.errstate(over="ignore"):
            return values.astype(dtype)
    bits = values.view(np.uint32)
    rounded = ((bits.astype(np.uint64) + 0x7FFF + ((bits >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(values), np.uint16(0x7FC0), rounded)


def from_bits(array, dtype):
    if dtype != "bfloat16":
        return array.view(dtype).astype(np.float64)
    return (array.view(np.uint16).astype(np.uint32) << 16).view(np.float32).astype(np.float64)


def size_of(dtype):
    return 4 if dtype == "float32" else 2


def device(runtime, array, dtype=None, offset=0):
    """A tensor whose buffer begins ``offset`` bytes into an allocation."""
    from llmopt_b200 import dispatch
    from llmopt_b200.cuda_native import Buffer

    array = np.ascontiguousarray(array)
    whole = Buffer.of_bytes(runtime, b"\x00" * offset + array.tobytes()) if array.nbytes or offset else Buffer.create(runtime, 16)
    return dispatch.Tensor(whole.view(offset, array.nbytes) if offset else whole, array.shape, dtype or str(array.dtype))


def blank(runtime, shape, dtype, behind=0):
    """A tensor of canaries, with ``behind`` more bytes of them in its buffer."""
    from llmopt_b200 import dispatch
    from llmopt_b200.cuda_native import Buffer

    itemsize = {"uint8": 1, "uint32": 4}.get(dtype) or size_of(dtype)
    nbytes = int(np.prod(shape)) * itemsize
    return dispatch.Tensor(Buffer.of_bytes(runtime, bytes([CANARY]) * max(nbytes + behind, 16)), tuple(shape), dtype)


def read(tensor, behind=0):
    """The tensor's values as they are held; the ``behind`` bytes after them must be canaries."""
    itemsize, held = {"uint8": (1, np.uint8), "uint32": (4, np.uint32), "float32": (4, np.float32)}.get(tensor.dtype) or (2, np.uint16)
    data = np.frombuffer(tensor.buffer.contents(), np.uint8)
    nbytes = int(np.prod(tensor.shape)) * itemsize
    assert (data[nbytes:nbytes + behind] == CANARY).all(), "bytes behind the result were written"
    return data[:nbytes].copy().view(held).reshape(tensor.shape)


def context(runtime, batch=None):
    from llmopt_b200 import dispatch

    return dispatch.Context(runtime, batch)


def special_rows(rng, rows, k, dtype):
    """Rows of very unlike sizes, with blocks of zeros, ties, infinities, NaN and the type's smallest and largest numbers."""
    low, high = {"float16": (-20, 12), "bfloat16": (-140, 120), "float32": (-150, 125)}[dtype]
    x = rng.standard_normal((rows, k)) * np.exp2(rng.integers(low, high, (rows, k // 32))).repeat(32, axis=1)
    blocks = x.reshape(-1, 32)
    at = rng.permutation(len(blocks))
    ties = np.array([4.0, 0.25, -0.25, 0.75, 1.25, -1.75, 2.5, 3.5, 5.0, -5.0, 6.5, 7.0, 7.5, -0.0, 0.0, 0.5])
    largest, smallest = {"float16": (65504.0, 2.0 ** -24), "bfloat16": (3.3895314e38, 2.0 ** -133), "float32": (3.4028235e38, 2.0 ** -149)}[dtype]
    fills = [np.zeros(32), np.concatenate([ties, -ties]), np.full(32, -0.0), np.where(np.arange(32) == 5, np.inf, 1.0),
             np.where(np.arange(32) == 31, np.nan, 1.0), np.where(np.arange(32) == 0, -np.inf, np.nan), np.full(32, largest),
             np.full(32, smallest), np.where(np.arange(32) % 2, largest, smallest), np.where(np.arange(32) == 17, smallest * 9, 0.0)]
    for fill, place in zip(fills, at):
        blocks[place] = fill
    return to_bits(x.astype(np.float32) if dtype != "float16" else x, dtype)


@pytest.mark.parametrize("dtype", ["float16", "bfloat16", "float32"])
@pytest.mark.parametrize("rows,k,extra,offset", [(1, 32, 0, 0), (1, 4096, 0, 0), (2, 96, 0, 0), (31, 128, 8, 0), (33, 160, 3, 0), (5, 576, 0, 4),
                                                 (64, 256, 0, 16), (70, 2080, 32, 0), (3, 14336, 0, 0)])
def test_quantization_is_exact(runtime, dtype, rows, k, extra, offset):
    from llmopt_b200 import dispatch

    rng = np.random.default_rng(rows * 131 + k)
    bits = special_rows(rng, rows, k, dtype)
    wide = np.concatenate([bits, np.full((rows, extra), 0x7F, bits.dtype)], axis=1)  # what lies between rows is not read
    x = device(runtime, wide, dtype, offset)
    codes, scales = blank(runtime, (rows, k // 2), "uint8", 64), blank(runtime, ((k + 127) // 128, rows), "uint32", 64)
    dispatch.dispatch_mxfp4_quantize(context(runtime), input=x, codes=codes, scales=scales, columns=k)
    nibbles, exponents = mx.quantize(from_bits(bits, dtype))
    assert np.array_equal(mx.exponents(read(scales, 64), k), exponents)
    assert np.array_equal(mx.unpack(read(codes, 64)), nibbles)


@pytest.mark.parametrize("dtype", ["float16", "bfloat16", "float32"])
@pytest.mark.parametrize("slots,source,k", [(1, 1, 32), (7, 3, 160), (100, 40, 576), (65, 200, 4096)])
def test_gathered_rows_are_quantized_in_the_order_of_slots(runtime, dtype, slots, source, k):
    from llmopt_b200 import dispatch

    rng = np.random.default_rng(slots)
    bits = special_rows(rng, source, k, dtype)
    index = rng.integers(0, source, slots).astype(np.uint32)
    index[-1] = source - 1
    beyond = index.copy()
    beyond[-1] = 0xFFFFFFFF  # counts as the last row
    codes, scales = blank(runtime, (slots, k // 2), "uint8", 64), blank(runtime, ((k + 127) // 128, slots), "uint32", 64)
    dispatch.dispatch_mxfp4_quantize(context(runtime), input=device(runtime, bits, dtype), codes=codes, scales=scales,
                                     row_of_slot=device(runtime, beyond))
    nibbles, exponents = mx.quantize(from_bits(bits, dtype)[index])
    assert np.array_equal(mx.exponents(read(scales, 64), k), exponents)
    assert np.array_equal(mx.unpack(read(codes, 64)), nibbles)


@pytest.mark.parametrize("dtype", ["float16", "bfloat16", "float32"])
@pytest.mark.parametrize("rows,k,offset", [(256, 32, 0), (1, 96, 0), (37, 416, 4), (40, 2080, 0)])
def test_values_of_all_codes_and_exponents(runtime, dtype, rows, k, offset):
    from llmopt_b200 import dispatch

    rng = np.random.default_rng(k)
    nibbles, exponents = rng.integers(0, 16, (rows, k)).astype(np.uint8), rng.integers(0, 256, (rows, k // 32)).astype(np.uint8)
    nibbles[0, :16] = np.arange(16)
    if rows == 256:
        exponents[:, 0] = np.arange(256)
    whole = blank(runtime, (rows * k + offset,), dtype, 64)
    out = dispatch.Tensor(whole.buffer.view(offset * size_of(dtype), rows * k * size_of(dtype) + 64), (rows, k), dtype)
    dispatch.dispatch_mxfp4_dequantize(context(runtime), codes=device(runtime, mx.pack(nibbles)), scales=device(runtime, mx.words(exponents, 255)),
                                       output=out)
    want = from_bits(to_bits(mx.values(nibbles, exponents), dtype), dtype)
    got = from_bits(read(out, 64), dtype)
    assert np.array_equal(got, want, equal_nan=True) and np.array_equal(np.signbit(got)[want == 0], np.signbit(want)[want == 0])


# ---- products -------------------------------------------------------------------------------------------

def random_operand(rng, rows, k, spread=3):
    """(nibbles, exponents) of rows whose blocks are of unlike size."""
    return rng.integers(0, 16, (rows, k)).astype(np.uint8), rng.integers(127 - spread, 128 + spread, (rows, k // 32)).astype(np.uint8)


def upload(runtime, operand, fill=0):
    nibbles, exponents = operand
    return device(runtime, mx.pack(nibbles)), device(runtime, mx.words(exponents, fill))


def allowed(x, w, want, dtype):
    """How far a product may be off: products of two elements are exact, a tensor core adds 64 of them at a time to an fp32 sum, each
    addition and each alignment of its terms off by at most a step (2^-23) of what has been summed, whose size the sum of sizes
    bounds -- k / 64 of the former, as many of the latter, and eight for the joining of partial sums --, and the result is rounded once."""
    k = x.shape[1]
    return (2 * (k / 64) + 8) * 2.0 ** -23 * (np.abs(x) @ np.abs(w).T) + HALF_STEP[dtype] * np.abs(want) * (1 + 2.0 ** -10) + 2.0 ** -25


def check(got, want, limit):
    assert np.array_equal(np.isnan(got), np.isnan(want))
    fine = ~np.isnan(want)
    error = np.abs(got - want)[fine]
    worst = np.argmax(error / limit[fine]) if error.size else 0
    assert (error <= limit[fine]).all(), (error[worst], limit[fine][worst], (error > limit[fine]).sum(), error.size)


LINEAR = [(1, 1, 32), (1, 8, 64), (1, 4096, 4096), (1, 130, 14336), (2, 127, 96), (3, 129, 160), (7, 333, 576), (8, 256, 1024), (9, 64, 14336),
          (16, 500, 2048), (17, 1000, 416), (31, 128, 4096), (32, 640, 512), (33, 1536, 576), (63, 72, 8192), (64, 128, 256), (65, 257, 288),
          (100, 384, 1056), (127, 1024, 640), (128, 130, 128), (129, 2048, 2048), (200, 96, 3200), (255, 1, 512), (256, 256, 256),
          (257, 300, 736), (400, 4100, 1024), (513, 2560, 2080), (1025, 640, 4096)]


@pytest.mark.parametrize("m,n,k", LINEAR)
def test_linear_is_the_product_of_the_values(runtime, m, n, k):
    from llmopt_b200 import dispatch

    rng = np.random.default_rng(m * 7919 + n * 31 + k)
    x, w = random_operand(rng, m, k), random_operand(rng, n, k)
    xv, wv = mx.values(*x), mx.values(*w)
    want = xv @ wv.T
    xt, wt = upload(runtime, x, 255), upload(runtime, w, 255)  # bytes behind k hold what they like
    bias = rng.standard_normal(n) * np.abs(want).max()
    for dtype, has_bias in (("float16", False), ("bfloat16", True), ("float32", True), ("float16", True)):
        scale = 2.0 ** -6 if dtype == "float16" else 1.0  # within the type's range
        x_scaled = xt if scale == 1.0 else upload(runtime, (x[0], (x[1] - 6).astype(np.uint8)), 255)
        held = to_bits(bias * scale, dtype)
        y = blank(runtime, (m, n), dtype, 256)
        dispatch.dispatch_mxfp4_linear(context(runtime), input=x_scaled[0], input_scales=x_scaled[1], weight=wt[0], weight_scales=wt[1], output=y,
                                       bias=device(runtime, held, dtype) if has_bias else None)
        exact = want * scale + (from_bits(held, dtype) if has_bias else 0.0)
        check(from_bits(read(y, 256), dtype), exact,
              allowed(xv * scale, wv, exact, dtype) + (2.0 ** -23 * np.abs(exact) if has_bias else 0.0))


def test_one_block_at_a_time_meets_its_exponents(runtime):
    """Every block of a long row alone, with its own power of two: exact, and any exchange of codes or exponents shows."""
    from llmopt_b200 import dispatch

    k, n = 1056, 140
    blocks = k // 32
    nibbles, exponents = np.zeros((blocks, k), np.uint8), np.full((blocks, blocks), 127, np.uint8)
    for b in range(blocks):
        nibbles[b, b * 32 + b % 32] = 2  # 1
        exponents[b, b] = 100 + b
    rng = np.random.default_rng(5)
    w = rng.integers(0, 16, (n, k)).astype(np.uint8), (110 + rng.integers(0, 30, (n, blocks))).astype(np.uint8)
    want = mx.values(nibbles, exponents) @ mx.values(*w).T
    for m in (1, 5, 33):
        x = nibbles[:m], exponents[:m]
        y = blank(runtime, (m, n), "float32")
        xt, wt = upload(runtime, x), upload(runtime, w)
        dispatch.dispatch_mxfp4_linear(context(runtime), input=xt[0], input_scales=xt[1], weight=wt[0], weight_scales=wt[1], output=y)
        assert np.array_equal(read(y), want[:m].astype(np.float32))


# rows and columns in other numbers than the tiles have, one to several tiles for every pair of SMs, sums shared out over a cluster's CTAs
SIZES = [(48, 8192, 8192), (17, 4096, 4096), (64, 4096, 14336), (1, 128256, 256), (33, 20000, 512), (65, 9472, 512), (224, 18944, 256), (225, 2560, 1024),
         (256, 14336, 512), (448, 4736, 288), (777, 7168, 256), (1000, 1000, 1000 // 32 * 32), (3000, 600, 128), (90, 40, 16384), (16, 123400, 160), (17, 123400, 160), (64, 128256, 256)]


@pytest.mark.parametrize("m,n,k", SIZES)
def test_linear_in_every_number_of_tiles(runtime, m, n, k):
    """Values of few bits, whose sums are whole numbers that fp32 holds: exact, whatever adds them in which order."""
    from llmopt_b200 import dispatch

    rng = np.random.default_rng(m + n + k)
    pick = np.array([0, 2, 4, 5, 10, 12, 13], np.uint8)  # 0, 1, 2, 3, -1, -2, -3
    x = rng.choice(pick, (m, k)), np.full((m, k // 32), 127, np.uint8)
    w = rng.choice(pick, (n, k)), rng.integers(127, 129, (n, k // 32)).astype(np.uint8)
    want = (mx.values(*x).astype(np.float32) @ mx.values(*w).astype(np.float32).T).astype(np.float32)  # below 2^24, so exact too
    xt, wt = upload(runtime, x, 255), upload(runtime, w, 255)
    y = blank(runtime, (m, n), "float32", 256)
    dispatch.dispatch_mxfp4_linear(context(runtime), input=xt[0], input_scales=xt[1], weight=wt[0], weight_scales=wt[1], output=y)
    got = read(y, 256)
    assert np.array_equal(got, want), np.argwhere(got != want)[:5]
    half = blank(runtime, (m, n), "float16", 256)
    dispatch.dispatch_mxfp4_linear(context(runtime), input=xt[0], input_scales=xt[1], weight=wt[0], weight_scales=wt[1], output=half)
    assert np.array_equal(read(half, 256), to_bits(want, "float16").view(np.uint16))


@pytest.mark.parametrize("m", [1, 40, 300])
def test_products_at_the_ends_of_the_exponents(runtime, m):
    """One product per sum: exact wherever fp32 holds it, subnormal numbers and infinity included.  A product of two elements has at most four
    significant bits, so fp32 fails to hold it only below 2^-126, where its numbers lie 2^-149 apart; the tensor cores cut a sum to one of
    them (as they do its last bits anywhere), so there the result is off by less than 2^-149."""
    from llmopt_b200 import dispatch

    pairs = [(254, 127), (254, 0), (254, 254), (0, 0), (0, 127), (60, 64), (50, 50), (40, 70), (63, 65), (254, 129), (253, 128), (1, 126), (0, 128)]
    n, k = 130, 64
    codes = np.arange(1, 8, dtype=np.uint8)
    for sx, sw in pairs:
        x = np.zeros((m, k), np.uint8), np.full((m, 2), 127, np.uint8)
        w = np.zeros((n, k), np.uint8), np.full((n, 2), 127, np.uint8)
        x[0][:, 5], x[1][:, 0] = np.resize(codes, m), sx
        w[0][:, 5], w[1][:, 0] = np.resize(codes[::-1], n), sw
        w[0][::2, 5] |= 8
        exact = mx.values(*x) @ mx.values(*w).T
        with np.errstate(over="ignore"):
            want = exact.astype(np.float32)
        held = np.isinf(want) | (want == exact)
        xt, wt, y = upload(runtime, x), upload(runtime, w), blank(runtime, (m, n), "float32")
        dispatch.dispatch_mxfp4_linear(context(runtime), input=xt[0], input_scales=xt[1], weight=wt[0], weight_scales=wt[1], output=y)
        got = read(y)
        assert np.array_equal(got[held], want[held]), (sx, sw)
        assert (np.abs(got.astype(np.float64) - exact)[~held] < 2.0 ** -149).all(), (sx, sw)


@pytest.mark.parametrize("m,n,k", [(1, 256, 4096), (5, 264, 96), (33, 128, 1024), (64, 1000, 512), (70, 256, 320), (300, 272, 640)])
def test_results_and_biases_at_any_multiple_of_their_element(runtime, m, n, k):
    from llmopt_b200 import dispatch

    rng = np.random.default_rng(m + n)
    x, w = random_operand(rng, m, k), random_operand(rng, n, k)
    x = x[0], (x[1] - 6).astype(np.uint8)
    xv, wv = mx.values(*x), mx.values(*w)
    want = xv @ wv.T
    bias = rng.standard_normal(n) * np.abs(want).max()
    xt, wt = upload(runtime, x, 255), upload(runtime, w, 255)
    for dtype in ("float16", "bfloat16", "float32"):
        for steps in (1, 2, 7):
            whole, held = blank(runtime, (m * n + steps,), dtype, 256), to_bits(bias, dtype)
            y = dispatch.Tensor(whole.buffer.view(steps * size_of(dtype), m * n * size_of(dtype) + 256), (m, n), dtype)
            dispatch.dispatch_mxfp4_linear(context(runtime), input=xt[0], input_scales=xt[1], weight=wt[0], weight_scales=wt[1], output=y,
                                           bias=device(runtime, held, dtype, steps * size_of(dtype)))
            exact = want + from_bits(held, dtype)
            check(from_bits(read(y, 256), dtype), exact, allowed(xv, wv, exact, dtype) + 2.0 ** -23 * np.abs(exact))
            assert (np.frombuffer(whole.buffer.contents(), np.uint8)[:steps * size_of(dtype)] == CANARY).all()


def test_offsets_beyond_32_bits(runtime):
    """More than 2^32 values: the first and last rows of conversions both ways, and of a product."""
    import torch

    torch.cuda.init()
    rows, k = 2 ** 22 + 5, 1024
    generator = torch.Generator("cuda").manual_seed(1)
    codes = torch.randint(0, 256, (rows, k // 2), dtype=torch.uint8, device="cuda", generator=generator)
    scales = torch.randint(120, 130, (k // 128, rows, 4), dtype=torch.uint8, device="cuda", generator=generator)
    values = torch.empty(rows, k, dtype=torch.float16, device="cuda")
    again, words = torch.empty_like(codes), torch.empty(k // 128, rows, dtype=torch.int32, device="cuda")
    stream = torch.cuda.current_stream().cuda_stream
    runtime.mxfp4_dequantize_pointers("f16", codes.data_ptr(), scales.data_ptr(), values.data_ptr(), rows, k, stream)
    runtime.mxfp4_quantize_pointers("f16", values.data_ptr(), None, again.data_ptr(), words.data_ptr(), rows, rows, k, k, stream)
    for part in (slice(0, 40), slice(rows - 40, rows)):
        want = mx.values(mx.unpack(codes[part].cpu().numpy()), mx.exponents(np.ascontiguousarray(scales[:, part].cpu().numpy()).view(np.uint32)[..., 0], k))
        assert np.array_equal(values[part].cpu().double().numpy(), want)
        nibbles, exponents = mx.quantize(want)
        assert np.array_equal(again[part].cpu().numpy(), mx.pack(nibbles))
        assert np.array_equal(np.ascontiguousarray(words[:, part].cpu().numpy()).view(np.uint32), mx.words(exponents))
    del values, again
    m, n = 4099, 2 ** 20 + 8
    x, w = codes.view(-1)[:m * 16], codes.view(-1)[-n * 16:]  # k of 32
    xs, ws = (torch.full((1, rows, 4), 125, dtype=torch.uint8, device="cuda")[:, :count].contiguous() for count in (m, n))
    y = torch.empty(m, n, dtype=torch.float16, device="cuda")
    runtime.mxfp4_linear_pointers("f16", x.data_ptr(), xs.data_ptr(), w.data_ptr(), ws.data_ptr(), None, y.data_ptr(), m, n, 32, stream)
    value = lambda held, count: mx.values(mx.unpack(held.cpu().numpy().reshape(count, 16)), np.full((count, 1), 125, np.uint8))
    wv = value(w, n)
    for row in (0, m // 2, m - 1):  # whole sixty-fourths of at most 72, which 16 bits hold to 11 bits of fraction
        want = (value(x[row * 16:row * 16 + 16], 1) @ wv.T)[0]
        assert np.array_equal(y[row].cpu().numpy(), want.astype(np.float16))


@pytest.mark.parametrize("m,n,k", [(3, 200, 416), (40, 130, 4096), (300, 260, 1024)])
def test_blocks_of_nan_reach_their_row_or_column_alone(runtime, m, n, k):
    from llmopt_b200 import dispatch

    rng = np.random.default_rng(9)
    x, w = random_operand(rng, m, k), random_operand(rng, n, k)
    x[1][m // 2, -1], w[1][n - 2, 3] = 255, 255
    x[0][m // 2, -32:] = 0  # elements of zero are NaN too there
    xv, wv = mx.values(*x), mx.values(*w)
    want = np.where(np.isnan(xv).any(1)[:, None] | np.isnan(wv).any(1)[None], np.nan, np.nan_to_num(xv) @ np.nan_to_num(wv).T)
    xt, wt, y = upload(runtime, x), upload(runtime, w), blank(runtime, (m, n), "float32")
    dispatch.dispatch_mxfp4_linear(context(runtime), input=xt[0], input_scales=xt[1], weight=wt[0], weight_scales=wt[1], output=y)
    check(read(y).astype(np.float64), want, allowed(np.nan_to_num(xv), np.nan_to_num(wv), np.nan_to_num(want), "float32"))


def test_linear_gives_the_same_bits_again(runtime):
    from llmopt_b200 import dispatch

    rng = np.random.default_rng(10)
    for m, n, k in ((1, 4096, 8192), (48, 700, 4096), (500, 900, 2048)):
        xt, wt = upload(runtime, random_operand(rng, m, k)), upload(runtime, random_operand(rng, n, k))
        seen = []
        for _ in range(3):
            y = blank(runtime, (m, n), "float32")
            dispatch.dispatch_mxfp4_linear(context(runtime), input=xt[0], input_scales=xt[1], weight=wt[0], weight_scales=wt[1], output=y)
            seen.append(read(y))
        assert np.array_equal(seen[0], seen[1]) and np.array_equal(seen[0], seen[2])


def expert_case(rng, counts, n, k):
    slots, experts = int(sum(counts)), len(counts)
    expert_of_slot = np.repeat(np.arange(experts), counts)
    x, w = random_operand(rng, slots, k), random_operand(rng, experts * n, k)
    return expert_of_slot, x, w, rng.uniform(0.05, 1.0, slots).astype(np.float32)


EXPERTS = [([1], 2, 32), ([0, 0, 1], 64, 160), ([1, 1], 7168, 1024), ([3, 0, 1, 0, 0, 2, 1, 1], 258, 576), ([0, 5, 11, 0], 130, 2048),
           ([128, 127, 129, 0, 1], 96, 416), ([300], 200, 256), ([0, 700, 3, 0, 65], 320, 1792), ([2] * 40, 32, 96), ([17, 33, 64, 40], 500, 736),
           ([1, 3] * 12, 5400, 96), ([40, 0, 1] + [1] * 19, 6000, 544),
           ([225, 224, 449, 1, 128], 322, 352), ([5000, 40, 0, 3000], 64, 64), ([1, 0, 400], 4736, 1056),
           ([225, 224, 449, 1, 128], 322, 2080), ([5000, 40, 0, 3000], 64, 2048), ([1, 0, 400], 4736, 2176), ([160] * 40, 34, 2048)]


@pytest.mark.parametrize("case", range(len(EXPERTS)))
def test_expert_rows_are_products_with_their_matrices(runtime, case):
    from llmopt_b200 import dispatch

    counts, n, k = EXPERTS[case]
    rng = np.random.default_rng(100 + case)
    expert_of_slot, x, w, score = expert_case(rng, counts, n, k)
    slots, experts = len(expert_of_slot), len(counts)
    x = x[0], (x[1] - 4).astype(np.uint8)  # f16 has to hold the products of two columns
    xv, wv = mx.values(*x), mx.values(*w)
    want, limit = np.zeros((slots, n)), np.zeros((slots, n))
    for e in range(experts):
        rows, mine = expert_of_slot == e, wv[e * n:(e + 1) * n]
        want[rows] = xv[rows] @ mine.T
        limit[rows] = allowed(xv[rows], mine, want[rows], "float32")
    xt, wt = upload(runtime, x, 255), upload(runtime, w, 255)
    plan = device(runtime, mx.plan_of(expert_of_slot, experts))
    operands = dict(input=xt[0], input_scales=xt[1], weight=wt[0], weight_scales=wt[1], experts=experts, plan=plan.buffer)
    y = blank(runtime, (slots, n), "float32", 256)
    dispatch.dispatch_mxfp4_expert_rows(context(runtime), **operands, output=y)
    check(read(y, 256).astype(np.float64), want, limit)
    gate, up = want[:, 0::2] * score[:, None], want[:, 1::2] * score[:, None]
    gate_off, up_off = limit[:, 0::2] * score[:, None] + 2.0 ** -24 * np.abs(gate), limit[:, 1::2] * score[:, None] + 2.0 ** -24 * np.abs(up)
    with np.errstate(over="ignore"):
        silu = gate / (1 + np.exp(-gate))
    pairs = silu * up
    # the slope of silu is below 1.1; exp, the division and two products of fp32 are a few steps of 2^-24 each, exp one of its argument
    off = 1.1 * gate_off * (np.abs(up) + up_off) + np.abs(silu) * up_off + np.abs(pairs) * 2.0 ** -24 * (8 + 2 * np.abs(gate))
    for dtype in ("float16", "bfloat16"):
        y = blank(runtime, (slots, n // 2), dtype, 256)
        dispatch.dispatch_mxfp4_expert_rows(context(runtime), **operands, output=y, score_of_slot=device(runtime, score))
        got = from_bits(read(y, 256), dtype)
        inside = np.abs(pairs) < 60000.0 if dtype == "float16" else np.ones_like(pairs, bool)
        assert inside.mean() > 0.9
        check(got[inside], pairs[inside], (off + HALF_STEP[dtype] * (np.abs(pairs) + off) + 2.0 ** -25)[inside])


def test_expert_rows_without_a_tile_stay_as_they_were(runtime):
    """Slots that no tile of the plan names (rows behind the last sequence) keep what they held, and a plan that points outside is cut."""
    from llmopt_b200 import dispatch

    rng = np.random.default_rng(12)
    n, k = 96, 256
    expert_of_slot, x, w, _ = expert_case(rng, [4, 6], n, k)
    xt, wt = upload(runtime, x), upload(runtime, w)
    plan = mx.plan_of(expert_of_slot, 2, most=2 + 1)
    plan[0, 0], plan[2] = 2, (1, 6, 8, 0)  # slots 4, 5, 8 and 9 are nobody's
    y = blank(runtime, (10, n), "float32", 256)
    operands = dict(input=xt[0], input_scales=xt[1], weight=wt[0], weight_scales=wt[1], experts=2)
    dispatch.dispatch_mxfp4_expert_rows(context(runtime), **operands, plan=device(runtime, plan).buffer, output=y)
    got = read(y, 256)
    untouched = np.full(4, CANARY, np.uint8).view(np.float32)[0]
    assert (got[[4, 5, 8, 9]] == untouched).all()
    xv, wv = mx.values(*x), mx.values(*w)
    assert np.allclose(got[:4], xv[:4] @ wv[:n].T, rtol=1e-5, atol=1e-3) and np.allclose(got[6:8], xv[6:8] @ wv[n:].T, rtol=1e-5, atol=1e-3)
    plan[0, 0], plan[2] = 1000, (7, 6, 5000, 0)  # more tiles than the plan has room for, an expert and rows that are not there
    y = blank(runtime, (10, n), "float32", 256)
    dispatch.dispatch_mxfp4_expert_rows(context(runtime), **operands, plan=device(runtime, plan).buffer, output=y)
    got = read(y, 256)
    assert np.allclose(got[6:], xv[6:] @ wv[n:].T, rtol=1e-5, atol=1e-3)


@pytest.mark.parametrize("k", [256, 2048])
def test_many_expert_rows_follow_the_plan(runtime, k):
    """Rows between the tiles stay as they were, and what points outside is cut."""
    from llmopt_b200 import dispatch

    rng = np.random.default_rng(13)
    n, slots = 96, 600
    x, w = random_operand(rng, slots, k), random_operand(rng, 2 * n, k)
    xt, wt = upload(runtime, x), upload(runtime, w)
    plan = np.zeros((1 + slots // 128 + 2, 4), np.uint32)
    plan[0, 0] = 1000  # more tiles than it has room for; an end and an expert that are not there; tiles without rows
    plan[1:5] = (0, 0, 128, 0), (0, 128, 5000, 0), (0, 270, 300, 0), (7, 590, 2 ** 32 - 1, 0)
    y = blank(runtime, (slots, n), "float32", 256)
    dispatch.dispatch_mxfp4_expert_rows(context(runtime), input=xt[0], input_scales=xt[1], weight=wt[0], weight_scales=wt[1], experts=2,
                                        plan=device(runtime, plan).buffer, output=y)
    got = read(y, 256)
    untouched = np.full(4, CANARY, np.uint8).view(np.float32)[0]
    expert = np.full(slots, -1)
    expert[:256], expert[270:300], expert[590:] = 0, 0, 1
    xv, wv = mx.values(*x), mx.values(*w)
    assert (got[expert < 0] == untouched).all()
    for e in (0, 1):
        mine = wv[e * n:(e + 1) * n]
        want = xv[expert == e] @ mine.T
        check(got[expert == e].astype(np.float64), want, allowed(xv[expert == e], mine, want, "float32"))


# ---- as they are used -------------------------------------------------------------------------------------

@pytest.mark.parametrize("rows,experts,top,width,inner", [(1, 4, 2, 160, 96), (5, 8, 2, 256, 160), (40, 6, 3, 576, 224), (300, 16, 2, 512, 288)])
def test_a_routed_layer_in_one_batch(runtime, rows, experts, top, width, inner):
    """Weights quantized on the device, a router's choices, the rows of every expert quantized, gate and up, their products quantized, down,
    and the sums of every row: each step against its own inputs."""
    from llmopt_b200 import dispatch, parameters
    from llmopt_b200.cuda_native import Batch, Buffer

    rng = np.random.default_rng(rows)
    x = to_bits(rng.standard_normal((rows, width)), "bfloat16")
    logits = rng.standard_normal((rows, experts)).astype(np.float32)
    up, down = rng.standard_normal((experts * 2 * inner, width)) / width ** 0.5, rng.standard_normal((experts * width, inner)) / inner ** 0.5
    pairs, batch = rows * top, Batch(runtime)
    ctx = context(runtime, batch)

    def held(shape_rows, k):
        return blank(runtime, (shape_rows, k // 2), "uint8"), blank(runtime, ((k + 127) // 128, shape_rows), "uint32")

    up_held, down_held, x_held, hidden_held = held(len(up), width), held(len(down), inner), held(pairs, width), held(pairs, inner)
    for source, target in ((up, up_held), (down, down_held)):
        dispatch.dispatch_mxfp4_quantize(ctx, input=device(runtime, source.astype(np.float32)), codes=target[0], scales=target[1])
    chosen, scores = blank(runtime, (rows, top), "uint32"), blank(runtime, (rows, top), "float32")
    plan, row_of_slot = Buffer.create(runtime, 16 * (1 + pairs // 128 + min(experts, pairs))), blank(runtime, (pairs,), "uint32")
    score_of_slot, slot_of_pair = blank(runtime, (pairs,), "float32"), blank(runtime, (pairs,), "uint32")
    size = parameters.route(rows=rows, experts=experts, top=top)
    run = lambda name, buffers, params: runtime.dispatch(name, buffers=buffers, parameters=params, batch=batch)
    run("llmopt_route_rows_f32", [device(runtime, logits).buffer, chosen.buffer, scores.buffer], size)
    run("llmopt_route_plan", [chosen.buffer, scores.buffer, plan, row_of_slot.buffer, score_of_slot.buffer, slot_of_pair.buffer], size)
    dispatch.dispatch_mxfp4_quantize(ctx, input=device(runtime, x, "bfloat16"), codes=x_held[0], scales=x_held[1], row_of_slot=row_of_slot)
    hidden, y = blank(runtime, (pairs, inner), "bfloat16"), blank(runtime, (pairs, width), "float32")
    dispatch.dispatch_mxfp4_expert_rows(ctx, input=x_held[0], input_scales=x_held[1], weight=up_held[0], weight_scales=up_held[1], experts=experts,
                                        plan=plan, output=hidden, score_of_slot=score_of_slot)
    dispatch.dispatch_mxfp4_quantize(ctx, input=hidden, codes=hidden_held[0], scales=hidden_held[1])
    dispatch.dispatch_mxfp4_expert_rows(ctx, input=hidden_held[0], input_scales=hidden_held[1], weight=down_held[0], weight_scales=down_held[1],
                                        experts=experts, plan=plan, output=y)
    batch.commit()

    order = np.argsort(-logits, axis=1, kind="stable")[:, :top]
    expert = order.reshape(-1)
    slots = np.argsort(expert, kind="stable")
    expert_of_slot = expert[slots]
    assert np.array_equal(read(row_of_slot), slots // top)

    def quantized(source, target):
        nibbles, exponents = mx.quantize(source)
        codes, words = read(target[0]), read(target[1])
        assert np.array_equal(mx.unpack(codes), nibbles) and np.array_equal(mx.exponents(words, source.shape[1]), exponents)
        return mx.values(nibbles, exponents)

    up_v, down_v = quantized(up.astype(np.float32), up_held), quantized(down.astype(np.float32), down_held)
    x_v = quantized(from_bits(x, "bfloat16")[slots // top], x_held)
    hidden_got, y_got = from_bits(read(hidden), "bfloat16"), read(y).astype(np.float64)
    hidden_v = quantized(hidden_got, hidden_held)
    score = read(score_of_slot).astype(np.float64)
    for e in range(experts):
        mine = expert_of_slot == e
        w = up_v[e * 2 * inner:(e + 1) * 2 * inner]
        sums = (x_v[mine] @ w.T) * score[mine, None]
        off = allowed(x_v[mine], w, np.zeros(1), "float32")
        gate, value = sums[:, 0::2], sums[:, 1::2]
        want = gate / (1 + np.exp(-gate)) * value
        limit = (1.1 * off[:, 0::2] * (np.abs(value) + off[:, 1::2]) + np.abs(gate) * off[:, 1::2] + 2.0 ** -8 * (1 + 2.0 ** -6) * np.abs(want)
                 + 2.0 ** -20 * np.abs(want) + 2.0 ** -25)
        check(hidden_got[mine], want, limit)
        w = down_v[e * width:(e + 1) * width]
        want = hidden_v[mine] @ w.T
        check(y_got[mine], want, allowed(hidden_v[mine], w, want, "float32"))


def routed_model(experts=6, top=2, inner=64, width=96):
    from mixer_models import dense_mlp, routed_mlp, sandwich_config, weights_of, window_layer

    config = sandwich_config([window_layer(mlp=routed_mlp(experts, top, inner)), window_layer(kv_from=0, mlp=dense_mlp(64)),
                              window_layer(mlp=routed_mlp(4, 1, 160))], width=width)
    return config, weights_of(config, seed=4)


@pytest.mark.parametrize("tokens", [1, 7, 60, 300])
def test_experts_of_a_decoder_in_mxfp4(runtime, tokens):
    """A prompt through an engine whose experts are quantized, replayed kernel by kernel: each against its own inputs."""
    from llmopt_b200 import mixer_engine
    from llmopt_b200.model import parse_config

    config, weights = routed_model()
    engine = mixer_engine.MixerEngine(runtime, parse_config(config), weights, capacity=320, experts="mxfp4")
    for index, (spec, inner) in ((0, (6, 64)), (2, (4, 160))):  # matrices as they were quantized
        feed = engine.layers[index].feed_forward
        for held, matrix, k in ((feed.up, None, 96), (feed.down, None, inner)):
            rows = spec * (2 * inner if held is feed.up else 96)
            name = lambda e, part: weights[f"l{index}.mlp.e{e}.{part}"]
            source = np.concatenate([np.stack([name(e, "gate"), name(e, "up")], 1).reshape(-1, k) if held is feed.up else name(e, "down")
                                     for e in range(spec)])
            nibbles, exponents = mx.quantize(source)
            assert source.shape == (rows, k) and np.array_equal(np.frombuffer(held[0].contents(), np.uint8)[:rows * k // 2].reshape(rows, -1), mx.pack(nibbles))
            words = np.frombuffer(held[1].contents(), np.uint32)[:(k + 127) // 128 * rows].reshape(-1, rows)
            assert np.array_equal(mx.exponents(words, k), exponents)
    ids = np.random.default_rng(tokens).integers(0, config["vocab"], tokens).tolist()
    first = engine.prefill(ids)
    assert first == engine.prefill(ids)
    plan = mixer_engine._Plan(engine, 1, tokens)
    engine._record_layers(plan.step)
    plan.write(ids, [0], [engine._row(0)])
    seen = []

    def held(buffers, rows, k):
        codes = np.frombuffer(buffers[0].contents(), np.uint8)[:rows * k // 2].reshape(rows, -1)
        words = np.frombuffer(buffers[1].contents(), np.uint32)[:(k + 127) // 128 * rows].reshape(-1, rows)
        return mx.unpack(codes), mx.exponents(words, k)

    for item in plan.items:
        runtime.dispatch(item.name, buffers=item.buffers, parameters=item.parameters)
        numbers, b = np.frombuffer(item.parameters, np.uint32).tolist(), item.buffers
        if item.name.startswith("llmopt_mxfp4_quantize"):
            rows, k = numbers[:2]
            x = np.frombuffer(b[0].contents(), np.uint16)
            if "rows" in item.name:
                index = np.frombuffer(b[1].contents(), np.uint32)[:rows]
                x = x[:numbers[3] * k].reshape(-1, k)[index]
            want = mx.quantize(from_bits(x[:rows * k].reshape(rows, k) if x.ndim == 1 else x, "bfloat16"))
            got = held(b[-2:], rows, k)
            assert np.array_equal(got[0], want[0]) and np.array_equal(got[1], want[1])
        elif item.name.startswith("llmopt_mxfp4_expert_rows"):
            slots, n, k, experts, paired = numbers
            xv, wv = mx.values(*held(b[0:2], slots, k)), mx.values(*held(b[2:4], experts * n, k)).reshape(experts, n, k)
            plan_words = np.frombuffer(b[4].contents(), np.uint32).reshape(-1, 4)
            covered = 0
            for expert, begin, end, _ in plan_words[1:1 + plan_words[0, 0]]:
                sums = xv[begin:end] @ wv[expert].T
                off = allowed(xv[begin:end], wv[expert], np.zeros(1), "float32")
                if paired:
                    score = np.frombuffer(b[5].contents(), np.float32)[begin:end, None].astype(np.float64)
                    got = from_bits(np.frombuffer(b[6].contents(), np.uint16)[:slots * n // 2].reshape(slots, -1)[begin:end], "bfloat16")
                    gate, value = sums[:, 0::2] * score, sums[:, 1::2] * score
                    want = gate / (1 + np.exp(-gate)) * value
                    check(got, want, 1.1 * off[:, 0::2] * (np.abs(value) + off[:, 1::2]) + np.abs(gate) * off[:, 1::2]
                          + 2.0 ** -8 * (1 + 2.0 ** -6) * np.abs(want) + 2.0 ** -20 * np.abs(want) + 2.0 ** -25)
                else:
                    got = np.frombuffer(b[6].contents(), np.float32)[:slots * n].reshape(slots, n)[begin:end].astype(np.float64)
                    check(got, sums, off + HALF_STEP["float32"] * np.abs(sums))
                covered += end - begin
            assert covered == slots
        else:
            continue
        seen.append(item.name)
    assert len(seen) == 8


def test_generation_with_experts_in_mxfp4(runtime, tmp_path, capsys):
    """Prompts, steps, chained steps and the command give the same tokens as one another."""
    from llmopt_b200 import generate, mixer_engine
    from llmopt_b200.model import parse_config
    from test_gpu_dalorax import checkpoint

    config, weights = routed_model(experts=8, top=3, inner=32, width=64)
    engine = mixer_engine.MixerEngine(runtime, parse_config(config), weights, capacity=64, experts="mxfp4")
    stream = [engine.prefill([3, 99, 41])]
    for past in range(3, 9):
        stream += engine.step(stream[-1:], past)
    engine.prefill([3, 99, 41])
    chained, _ = engine.generate_chained(stream[:1], 3, 6)
    assert chained == stream[1:]
    checkpoint(tmp_path, config, weights)
    generate.main(["--model", str(tmp_path), "--prompt", "3,99,41", "--tokens", "7", "--experts", "mxfp4"])
    assert capsys.readouterr().out.splitlines() == [",".join(map(str, stream))]


def test_a_layer_replayed_as_a_plan(runtime):
    """Quantization and product in a plan that is replayed with new inputs."""
    from llmopt_b200 import dispatch, parameters
    from llmopt_b200.cuda_native import Batch, Buffer, Prebaked

    rng = np.random.default_rng(21)
    m, n, k = 3, 200, 288
    w = random_operand(rng, n, k)
    wt = upload(runtime, w)
    x = device(runtime, np.zeros((m, k), np.float16))
    codes, scales, y = blank(runtime, (m, k // 2), "uint8"), blank(runtime, (3, m), "uint32"), blank(runtime, (m, n), "float32")
    batch = Batch(runtime)
    ctx = context(runtime, batch)
    dispatch.dispatch_mxfp4_quantize(ctx, input=x, codes=codes, scales=scales)
    dispatch.dispatch_mxfp4_linear(ctx, input=codes, input_scales=scales, weight=wt[0], weight_scales=wt[1], output=y)
    token, picked = Buffer.create(runtime, 8), Buffer.create(runtime, 16)
    plan = Prebaked(runtime, batch.pending, token, picked)
    batch.pending = []
    for _ in range(3):
        values = rng.standard_normal((m, k)).astype(np.float16)
        x.buffer.write(0, values)
        plan.execute(token=0, past_tokens=0)
        xv = mx.values(*mx.quantize(values))
        want = xv @ mx.values(*w).T
        check(read(y).astype(np.float64), want, allowed(xv, mx.values(*w), want, "float32"))


# ---- raw pointers -----------------------------------------------------------------------------------------

def test_pointers_streams_and_captured_calls(runtime):
    """The pointer forms on a stream of the caller's, two streams at once, and captured into a graph that is replayed on new inputs."""
    import torch

    torch.cuda.init()
    rng = np.random.default_rng(30)
    cases = []
    for m, n, k in ((2, 300, 1024), (70, 500, 608)):
        w = random_operand(rng, n, k)
        cases.append(dict(m=m, n=n, k=k, wv=mx.values(*w), w=torch.from_numpy(mx.pack(w[0])).cuda(),
                          ws=torch.from_numpy(mx.words(w[1]).view(np.int32)).cuda(), x=torch.zeros(m, k, dtype=torch.bfloat16, device="cuda"),
                          codes=torch.empty(m, k // 2, dtype=torch.uint8, device="cuda"),
                          scales=torch.empty((k + 127) // 128, m, dtype=torch.int32, device="cuda"), y=torch.empty(m, n, device="cuda"),
                          back=torch.empty(m, k, dtype=torch.bfloat16, device="cuda")))
    torch.cuda.synchronize()

    def layer(c, stream):
        runtime.mxfp4_quantize_pointers("bf16", c["x"].data_ptr(), None, c["codes"].data_ptr(), c["scales"].data_ptr(), c["m"], c["m"], c["k"],
                                        c["k"], stream)
        runtime.mxfp4_linear_pointers("f32", c["codes"].data_ptr(), c["scales"].data_ptr(), c["w"].data_ptr(), c["ws"].data_ptr(), None,
                                      c["y"].data_ptr(), c["m"], c["n"], c["k"], stream)
        runtime.mxfp4_dequantize_pointers("bf16", c["codes"].data_ptr(), c["scales"].data_ptr(), c["back"].data_ptr(), c["m"], c["k"], stream)

    def checked(c, x):
        values = mx.values(*mx.quantize(x.double().numpy()))
        want = values @ c["wv"].T
        check(c["y"].cpu().double().numpy(), want, allowed(values, c["wv"], want, "float32"))
        assert np.array_equal(c["back"].cpu().double().numpy(), values)

    streams = [torch.cuda.Stream() for _ in cases]
    for _ in range(2):
        inputs = [torch.randn(c["m"], c["k"]).bfloat16() for c in cases]
        for c, x, s in zip(cases, inputs, streams):
            with torch.cuda.stream(s):
                c["x"].copy_(x)
                layer(c, s.cuda_stream)
        torch.cuda.synchronize()
        for c, x in zip(cases, inputs):
            checked(c, x)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for c in cases:
            layer(c, torch.cuda.current_stream().cuda_stream)
    for _ in range(2):
        inputs = [torch.randn(c["m"], c["k"]).bfloat16() for c in cases]
        for c, x in zip(cases, inputs):
            c["x"].copy_(x)
        graph.replay()
        torch.cuda.synchronize()
        for c, x in zip(cases, inputs):
            checked(c, x)


def test_calls_on_the_default_stream_come_after_its_work(runtime):
    """A stream of 0 is torch's default one: what that still has to write is read, and what it does next reads the results."""
    import torch

    torch.cuda.init()
    rng = np.random.default_rng(32)
    for m in (2, 80):
        n, k = 256, 512
        w = random_operand(rng, n, k)
        held = torch.from_numpy(mx.pack(w[0])).cuda(), torch.from_numpy(mx.words(w[1]).view(np.int32)).cuda()
        x, codes = torch.zeros(m, k, device="cuda"), torch.zeros(m, k // 2, dtype=torch.uint8, device="cuda")
        words, y = torch.zeros(k // 128, m, dtype=torch.int32, device="cuda"), torch.zeros(m, n, device="cuda")
        values = torch.zeros(m, k, device="cuda")
        source = torch.randn(m, k, device="cuda")
        torch.cuda.synchronize()
        stream = torch.cuda.current_stream().cuda_stream
        torch.cuda._sleep(100_000_000)
        x.copy_(source)
        runtime.mxfp4_quantize_pointers("f32", x.data_ptr(), None, codes.data_ptr(), words.data_ptr(), m, m, k, k, stream)
        runtime.mxfp4_dequantize_pointers("f32", codes.data_ptr(), words.data_ptr(), values.data_ptr(), m, k, stream)
        runtime.mxfp4_linear_pointers("f32", codes.data_ptr(), words.data_ptr(), held[0].data_ptr(), held[1].data_ptr(), None, y.data_ptr(),
                                      m, n, k, stream)
        got, got_values = y.clone(), values.clone()
        for tensor in (x, codes, words, values, y):
            tensor.zero_()
        xv, wv = mx.values(*mx.quantize(source.cpu().double().numpy())), mx.values(*w)
        assert np.array_equal(got_values.cpu().double().numpy(), xv)
        check(got.cpu().double().numpy(), xv @ wv.T, allowed(xv, wv, xv @ wv.T, "float32"))


def test_calls_from_several_threads(runtime):
    """Streams with clusters and pairs of CTAs side by side, each from a thread of its own: whole numbers, which come out exactly."""
    import threading

    import torch

    torch.cuda.init()
    rng = np.random.default_rng(31)
    pick = np.array([0, 2, 4, 5, 10, 12, 13], np.uint8)
    cases = []
    for m, n, k in ((3, 4096, 4096), (64, 2048, 8192), (300, 2304, 2048), (129, 9472, 512)):
        x, w = rng.choice(pick, (m, k)), rng.choice(pick, (n, k))
        ones = [np.full((rows, k // 32), 127, np.uint8) for rows in (m, n)]
        want = torch.from_numpy((mx.values(x, ones[0]).astype(np.float32) @ mx.values(w, ones[1]).astype(np.float32).T)).cuda()
        operands = [torch.from_numpy(a).cuda() for a in (mx.pack(x), mx.words(ones[0]).view(np.int32), mx.pack(w), mx.words(ones[1]).view(np.int32))]
        cases.append((m, n, k, operands, [torch.empty(m, n, device="cuda") for _ in range(20)], want, torch.cuda.Stream()))
    torch.cuda.synchronize()
    failed = []

    def run(m, n, k, operands, results, want, stream):
        try:
            for y in results:
                runtime.mxfp4_linear_pointers("f32", *[t.data_ptr() for t in operands], None, y.data_ptr(), m, n, k, stream.cuda_stream)
        except Exception as error:
            failed.append(error)

    threads = [threading.Thread(target=run, args=case) for case in cases]
    for thread in threads:
        thread.start()
    for thread in threads:
        thread.join()
    torch.cuda.synchronize()
    assert not failed
    for _, _, _, _, results, want, _ in cases:
        assert all(torch.equal(y, want) for y in results)


def test_expert_rows_of_pointers(runtime):
    import torch

    rng = np.random.default_rng(31)
    counts, n, k = [3, 0, 9], 64, 160
    expert_of_slot, x, w, score = expert_case(rng, counts, n, k)
    to = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()
    xs, ws = to(mx.words(x[1]).view(np.int32)), to(mx.words(w[1]).view(np.int32))
    xc, wc, plan = to(mx.pack(x[0])), to(mx.pack(w[0])), to(mx.plan_of(expert_of_slot, 3).view(np.int32))
    y = torch.empty(12, n, device="cuda")
    torch.cuda.synchronize()
    runtime.mxfp4_expert_rows_pointers("bf16", xc.data_ptr(), xs.data_ptr(), wc.data_ptr(), ws.data_ptr(), plan.data_ptr(), None, y.data_ptr(), 12, n,
                                       k, 3, False, torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    xv, wv = mx.values(*x), mx.values(*w).reshape(3, n, k)
    want = np.einsum("sk,snk->sn", xv, wv[expert_of_slot])
    limit = np.stack([allowed(xv[i:i + 1], wv[e], want[i:i + 1], "float32")[0] for i, e in enumerate(expert_of_slot)])
    check(y.cpu().double().numpy(), want, limit)


def test_nothing_to_do_is_done(runtime):
    """No rows: accepted, and nothing is read."""
    runtime.mxfp4_quantize_pointers("f16", 0, None, 0, 0, 0, 0, 64, 64)
    runtime.mxfp4_quantize_pointers("f16", 0, 16, 0, 0, 0, 0, 64, 64)
    runtime.mxfp4_dequantize_pointers("f32", 0, 0, 0, 0, 64)
    with pytest.raises(ValueError):
        runtime.mxfp4_linear_pointers("f32", 0, 0, 0, 0, None, 0, 0, 8, 64)  # the weights are there all the same
    runtime.synchronize()


# ---- refusals: all on the host, before a launch --------------------------------------------------------------

def test_refusals(runtime):
    from llmopt_b200 import parameters
    from llmopt_b200.cuda_native import Buffer, NativeError

    big = Buffer.create(runtime, 1 << 16)
    short, odd = big.view(0, 32), big.view(8, 1 << 12)
    q, r, d, l = (parameters.mxfp4_quantize, parameters.mxfp4_quantize_rows, parameters.mxfp4_dequantize, parameters.mxfp4_linear)
    e = parameters.expert_rows
    refused = [
        ("quantize_f16", [big, big, big], q(rows=4, k=48, stride=48)), ("quantize_f16", [big, big, big], q(rows=4, k=0, stride=48)),
        ("quantize_f16", [big, big, big], q(rows=4, k=64, stride=63)), ("quantize_f16", [short, big, big], q(rows=4, k=64, stride=64)),
        ("quantize_f32", [big, short, big], q(rows=4, k=64, stride=64)), ("quantize_f32", [big, big, short], q(rows=40, k=64, stride=64)),
        ("quantize_f32", [big, odd, big], q(rows=4, k=64, stride=64)), ("quantize_f32", [big.view(2, 4096), big, big], q(rows=4, k=64, stride=64)),
        ("quantize_f32", [big, big], q(rows=4, k=64, stride=64)), ("quantize_f32", [big, big, big], d(rows=4, k=64)),
        ("quantize_bf16", [big, big, big], q(rows=0xFFFFFFFF, k=64, stride=64)),
        ("quantize_rows_bf16", [big, short, big, big], r(rows=9, k=64, stride=64, source_rows=4)),
        ("quantize_rows_bf16", [big, big, big, big], r(rows=9, k=64, stride=64, source_rows=0)),
        ("quantize_rows_bf16", [big, big, big, big], r(rows=9, k=64, stride=64, source_rows=1 << 20)),
        ("dequantize_f16", [short, big, big], d(rows=4, k=64)), ("dequantize_f16", [big, big, short], d(rows=4, k=64)),
        ("dequantize_f16", [big, big, big.view(1, 4096)], d(rows=4, k=64)), ("dequantize_f16", [odd, big, big], d(rows=4, k=64)),
        ("dequantize_f16", [big, big, big], d(rows=4, k=33)),
        ("linear_f16", [big, big, big, big, big, big], l(m=4, n=8, k=16, has_bias=False)),
        ("linear_f16", [big, big, big, big, big, big], l(m=4, n=0, k=64, has_bias=False)),
        ("linear_f16", [big, big, big, big, short, big], l(m=4, n=32, k=64, has_bias=True)),
        ("linear_f16", [short, big, big, big, big, big], l(m=4, n=8, k=64, has_bias=False)),
        ("linear_f16", [big, big.view(0, 4), big, big, big, big], l(m=4, n=8, k=64, has_bias=False)),
        ("linear_f16", [big, big, short, big, big, big], l(m=4, n=8, k=64, has_bias=False)),
        ("linear_f16", [big, big, big, big.view(0, 16), big, big], l(m=4, n=8, k=64, has_bias=False)),
        ("linear_f16", [big, big, big, big, big, short], l(m=4, n=8, k=64, has_bias=False)),
        ("linear_f16", [odd, big, big, big, big, big], l(m=4, n=8, k=64, has_bias=False)),
        ("linear_f16", [big, big, odd, big, big, big], l(m=4, n=8, k=64, has_bias=False)),
        ("linear_f32", [big, big, big, big, big, big.view(2, 4096)], l(m=4, n=8, k=64, has_bias=False)),
        ("linear_f16", [big] * 5, l(m=4, n=8, k=64, has_bias=False)),
        ("expert_rows_f16", [big] * 7, e(pairs=4, n=7, k=64, experts=2, paired=True)),
        ("expert_rows_f16", [big] * 7, e(pairs=4, n=8, k=64, experts=0, paired=True)),
        ("expert_rows_f16", [big] * 7, e(pairs=4, n=8, k=64, experts=9000, paired=True)),
        ("expert_rows_f16", [big] * 7, e(pairs=4, n=1 << 20, k=64, experts=4096, paired=True)),
        ("expert_rows_f16", [big, big, big, big, short, big, big], e(pairs=4, n=8, k=64, experts=2, paired=True)),
        ("expert_rows_f16", [big, big, big, big, odd, big, big], e(pairs=4, n=8, k=64, experts=2, paired=True)),
        ("expert_rows_f16", [big, big, big, big, big, short, big], e(pairs=9, n=8, k=64, experts=2, paired=True)),
        ("expert_rows_f16", [big, big, big, big, big, big, short], e(pairs=9, n=8, k=64, experts=2, paired=True)),
        ("expert_rows_bf16", [big, big, big, big, big, big, big.view(2, 4096)], e(pairs=9, n=8, k=64, experts=2, paired=False)),
    ]
    for name, buffers, params in refused:
        with pytest.raises(NativeError):
            runtime.dispatch(f"llmopt_mxfp4_{name}", buffers=buffers, parameters=params)
    runtime.synchronize()


def test_refusals_of_pointers(runtime):
    from llmopt_b200.cuda_native import Buffer

    p = Buffer.create(runtime, 1 << 16)
    at = p.device_pointer()
    for call in (lambda: runtime.mxfp4_linear_pointers("f16", at, at, at, at, None, at, -1, 8, 64),
                 lambda: runtime.mxfp4_linear_pointers("f16", at, at, at, at, None, at, 1, 1 << 31, 64),
                 lambda: runtime.mxfp4_linear_pointers("f16", at, at, at, at, None, at, 1, 8, 40),
                 lambda: runtime.mxfp4_linear_pointers("f16", at + 8, at, at, at, None, at, 1, 8, 64),
                 lambda: runtime.mxfp4_linear_pointers("f16", at, at, at, 0, None, at, 1, 8, 64),
                 lambda: runtime.mxfp4_quantize_pointers("f32", 0, None, at, at, 1, 1, 64, 64),
                 lambda: runtime.mxfp4_quantize_pointers("f32", at, None, at, at, 1, 1, 64, 32),
                 lambda: runtime.mxfp4_quantize_pointers("f32", at, at, at, at, 1, 0, 64, 64),
                 lambda: runtime.mxfp4_dequantize_pointers("f32", at, at, at + 2, 1, 64),
                 lambda: runtime.mxfp4_expert_rows_pointers("f32", at, at, at, at, at, at, at, 2, 8, 64, 2, True),
                 lambda: runtime.mxfp4_expert_rows_pointers("f16", at, at, at, at, at, 0, at, 2, 8, 64, 2, True),
                 lambda: runtime.mxfp4_expert_rows_pointers("f16", at, at, at, at, at, at, at, 2, 8, 64, 0, True)):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(KeyError):
        runtime.mxfp4_dequantize_pointers("f64", at, at, at, 1, 64)
    runtime.synchronize()
