"""Calls of the MXFP4 operators at the ends of what they take: gates far from zero, sizes, raw pointers, streams, failures."""

import numpy as np
import pytest

import mxfp4_oracle as mx
from test_gpu_mxfp4 import HALF_STEP, allowed, blank, check, context, device, expert_case, from_bits, read, special_rows, upload

pytestmark = pytest.mark.gpu


# slots and k: a tile's CTA by itself, a cluster that shares out k, pairs of CTAs with the plan's tiles and with joined ones
@pytest.mark.parametrize("slots,k", [(40, 64), (40, 4096), (200, 64), (200, 2048)])
@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
def test_pairs_with_gates_far_from_zero(runtime, dtype, slots, k):
    """silu of a gate near -88 is near 2^-120, which the other column can bring back into the range of 16 bits: the score is the gate, the
    other column a power of two times it.  In steps of 2^-23: e^(gate / 3) is off by 2 (ex2.approx) and by what its argument is, whose factor
    and product round to 1.5 of 2^-24 of gate / 3; it enters three times.  The reciprocal is off by 1, eight other operations by a half each."""
    from llmopt_b200 import dispatch

    power = 120 if dtype == "float16" else 100
    score = np.linspace(80.0, 103.0 if dtype == "float16" else 150.0, slots).astype(np.float32)
    if dtype == "bfloat16":
        score[::5] *= -1  # gates above zero
    n = 34
    x, w = (np.zeros((slots, k), np.uint8), np.full((slots, k // 32), 127, np.uint8)), (np.zeros((n, k), np.uint8), np.full((n, k // 32), 127, np.uint8))
    x[0][:, k - 40] = 2
    w[0][0::2, k - 40], w[0][1::2, k - 40], w[1][1::2, (k - 40) // 32] = 10, 2, 127 + power  # -1, 2^power
    gate, up = -score.astype(np.float64), score.astype(np.float64) * 2.0 ** power
    want = np.repeat((gate / (1 + np.exp(-gate)) * up)[:, None], n // 2, 1)
    xt, wt = upload(runtime, x), upload(runtime, w)
    y = blank(runtime, (slots, n // 2), dtype, 256)
    dispatch.dispatch_mxfp4_expert_rows(context(runtime), input=xt[0], input_scales=xt[1], weight=wt[0], weight_scales=wt[1], experts=1,
                                        plan=device(runtime, mx.plan_of(np.zeros(slots, int), 1)).buffer, output=y, score_of_slot=device(runtime, score))
    steps = 3 * (2 + 0.75 * np.abs(gate) / 3) + 1 + 8 / 2
    limit = np.abs(want) * (HALF_STEP[dtype] * (1 + 2.0 ** -10) + steps[:, None] * 2.0 ** -23) + (2.0 ** -25 if dtype == "float16" else 0.0)
    got = from_bits(read(y, 256), dtype)
    beyond = np.abs(want) - limit > (65520.0 if dtype == "float16" else np.inf)  # from there on the nearest of f16 is infinity
    assert (got[beyond] == -np.inf).all() and beyond.mean() < 0.1
    check(got[~beyond], want[~beyond], limit[~beyond])


@pytest.mark.parametrize("slots,k", [(40, 64), (200, 2048)])
@pytest.mark.parametrize("power,low,high", [(-125, 1.0, 22.6), (119, 1.0, 22.6), (0, 1.0, 22.6), (-134, 17.0, 80.0)])
def test_pairs_whose_products_lie_at_the_ends_of_bfloat16(runtime, power, low, high, slots, k):
    """Results between 2^-126 and 2^128 are normal numbers of bfloat16 with 8 bits each, whatever the factors: nothing on the way may leave
    fp32's range before they do.  Steps as above, and the other column's by which it is off where it is subnormal; results within half a
    step of the largest number are left out."""
    from llmopt_b200 import dispatch

    score = np.geomspace(low, high, slots).astype(np.float32)
    score[::3] *= -1  # gates below zero
    n = 34
    x, w = (np.zeros((slots, k), np.uint8), np.full((slots, k // 32), 127, np.uint8)), (np.zeros((n, k), np.uint8), np.full((n, k // 32), 127, np.uint8))
    x[0][:, 0], x[0][:, -1], w[0][0::2, 0], w[0][1::2, -1] = 2, 2, 2, 2  # 1 for the gate, from the other end 2^power for the other column
    x[1][:, -1], w[1][:, -1] = 127 + min(power, 0) // 2, 127 + power - min(power, 0) // 2
    gate, up = score.astype(np.float64), score.astype(np.float64) * 2.0 ** power
    want = np.repeat((gate / (1 + np.exp(-gate)) * up)[:, None], n // 2, 1)
    xt, wt = upload(runtime, x), upload(runtime, w)
    y = blank(runtime, (slots, n // 2), "bfloat16", 256)
    dispatch.dispatch_mxfp4_expert_rows(context(runtime), input=xt[0], input_scales=xt[1], weight=wt[0], weight_scales=wt[1], experts=1,
                                        plan=device(runtime, mx.plan_of(np.zeros(slots, int), 1)).buffer, output=y, score_of_slot=device(runtime, score))
    limit = np.abs(want) * (HALF_STEP["bfloat16"] * (1 + 2.0 ** -10) + (3 * (2 + 0.75 * np.abs(gate) / 3) + 5)[:, None] * 2.0 ** -23)
    limit = limit + 2.0 ** -150 * np.abs(want / up[:, None])
    got, normal = from_bits(read(y, 256), "bfloat16"), (np.abs(want) >= 2.0 ** -126) & (np.abs(want) < 2.0 ** 128 * (1 - 2.0 ** -8))
    assert normal.mean() > 0.6
    check(got[normal], want[normal], limit[normal])


@pytest.mark.parametrize("counts,n,k", [([3, 5, 0, 9], 130, 416), ([3, 5, 9], 200, 4096), ([100, 200, 40], 96, 288), ([130, 300, 20], 300, 2080)])
def test_blocks_of_nan_among_sorted_rows_reach_their_row_or_column_alone(runtime, counts, n, k):
    """Rows of another expert, and another expert's columns, lie in the same boxes."""
    from llmopt_b200 import dispatch

    rng = np.random.default_rng(len(counts) + k)
    expert_of_slot, x, w, score = expert_case(rng, counts, n, k)
    slots, ends = len(expert_of_slot), np.cumsum(counts)
    x = x[0], (x[1] - 4).astype(np.uint8)
    x[1][ends[0] - 1, -1] = x[1][ends[1], 0] = 255  # the last row of one expert, the first of the one after the next
    w[1][n, 1] = w[1][2 * n - 1, -1] = 255          # the second expert's first and last column
    xv, wv = mx.values(*x), mx.values(*w).reshape(len(counts), n, k)
    bad = np.isnan(xv).any(1)[:, None] | np.isnan(wv).any(2)[expert_of_slot]
    xn, wn = np.nan_to_num(xv), np.nan_to_num(wv)
    want, limit = np.zeros((slots, n)), np.zeros((slots, n))
    for e in range(len(counts)):
        mine = expert_of_slot == e
        want[mine] = xn[mine] @ wn[e].T
        limit[mine] = allowed(xn[mine], wn[e], want[mine], "float32")
    xt, wt = upload(runtime, x), upload(runtime, w)
    plan = device(runtime, mx.plan_of(expert_of_slot, len(counts)))
    operands = dict(input=xt[0], input_scales=xt[1], weight=wt[0], weight_scales=wt[1], experts=len(counts), plan=plan.buffer)
    y = blank(runtime, (slots, n), "float32", 256)
    dispatch.dispatch_mxfp4_expert_rows(context(runtime), **operands, output=y)
    check(read(y, 256).astype(np.float64), np.where(bad, np.nan, want), limit)
    y = blank(runtime, (slots, n // 2), "bfloat16", 256)
    dispatch.dispatch_mxfp4_expert_rows(context(runtime), **operands, output=y, score_of_slot=device(runtime, score))
    assert np.array_equal(np.isnan(from_bits(read(y, 256), "bfloat16")), bad[:, 0::2] | bad[:, 1::2])


@pytest.mark.parametrize("m", [2, 70])
def test_the_longest_rows(runtime, m):
    """k of 2^23, the most that is taken: single elements here and there, whose products fp32 holds."""
    import torch

    k, n = 1 << 23, 5
    rng = np.random.default_rng(m)
    places = np.unique(np.concatenate([[0, 1, 31, 32, 511, 512, k // 2 - 1, k // 2, k - 1], rng.integers(0, k, 40)]))
    pick = np.array([2, 4, 5, 10, 12], np.uint8)  # 1, 2, 3, -1, -2
    value = np.array([0.0, 0.0, 1.0, 0.0, 2.0, 3.0, 0.0, 0.0, 0.0, 0.0, -1.0, 0.0, -2.0])

    def rows(count):
        nibbles = rng.choice(pick, (count, len(places)))
        codes = torch.zeros(count, k // 2, dtype=torch.uint8, device="cuda")
        for column, place in enumerate(places):
            codes[:, place // 2] |= on_gpu(nibbles[:, column] << (4 * (place % 2)))
        return value[nibbles], codes, torch.full((k // 128, count), 0x7F7F7F7F, dtype=torch.int32, device="cuda")

    (xv, x, xs), (wv, w, ws) = rows(m), rows(n)
    y = torch.zeros(m, n, device="cuda")
    stream = torch.cuda.current_stream().cuda_stream
    runtime.mxfp4_linear_pointers("f32", x.data_ptr(), xs.data_ptr(), w.data_ptr(), ws.data_ptr(), None, y.data_ptr(), m, n, k, stream)
    assert np.array_equal(y.cpu().numpy(), xv @ wv.T)
    with pytest.raises(ValueError, match="too large"):
        runtime.mxfp4_linear_pointers("f32", x.data_ptr(), xs.data_ptr(), w.data_ptr(), ws.data_ptr(), None, y.data_ptr(), 1, 1, k + 32, stream)


def test_as_many_experts_as_there_can_be(runtime):
    """8192 of them, most with a row or two, some with none."""
    from llmopt_b200 import dispatch

    rng = np.random.default_rng(61)
    experts, n, k = 8192, 6, 64
    pick = np.array([0, 2, 4, 5, 10, 12, 13], np.uint8)
    counts = rng.integers(0, 3, experts)
    counts[-1] = 1
    expert_of_slot = np.repeat(np.arange(experts), counts)
    slots = len(expert_of_slot)
    x, w = ((rng.choice(pick, (rows, k)), np.full((rows, 2), 127, np.uint8)) for rows in (slots, experts * n))
    want = np.einsum("sk,snk->sn", mx.values(*x), mx.values(*w).reshape(experts, n, k)[expert_of_slot])
    xt, wt, y = upload(runtime, x), upload(runtime, w), blank(runtime, (slots, n), "float32", 256)
    dispatch.dispatch_mxfp4_expert_rows(context(runtime), input=xt[0], input_scales=xt[1], weight=wt[0], weight_scales=wt[1], experts=experts,
                                        plan=device(runtime, mx.plan_of(expert_of_slot, experts)).buffer, output=y)
    assert np.array_equal(read(y, 256), want)


# ---- raw pointers -----------------------------------------------------------------------------------------

def on_gpu(array):
    import torch

    array = np.ascontiguousarray(array)
    return torch.from_numpy(array.view(np.int32) if array.dtype == np.uint32 else array).cuda()


@pytest.mark.parametrize("element", ["f32", "f16", "bf16"])
def test_sums_of_expert_rows_are_fp32_whatever_the_type(runtime, element):
    import torch

    rng = np.random.default_rng(41)
    counts, n, k = [5, 0, 2], 66, 96
    expert_of_slot, x, w, _ = expert_case(rng, counts, n, k)
    xv, wv = mx.values(*x), mx.values(*w).reshape(len(counts), n, k)
    held = [on_gpu(a) for a in (mx.pack(x[0]), mx.words(x[1]), mx.pack(w[0]), mx.words(w[1]), mx.plan_of(expert_of_slot, len(counts)))]
    y = torch.full((7, n), float("nan"), device="cuda")
    stream = torch.cuda.current_stream().cuda_stream
    runtime.mxfp4_expert_rows_pointers(element, *[t.data_ptr() for t in held], None, y.data_ptr(), 7, n, k, len(counts), False, stream)
    want = np.einsum("sk,snk->sn", xv, wv[expert_of_slot])
    limit = np.stack([allowed(xv[i:i + 1], wv[e], want[i:i + 1], "float32")[0] for i, e in enumerate(expert_of_slot)])
    check(y.cpu().double().numpy(), want, limit)


def guarded(shape, dtype, behind=64):
    """A tensor on the GPU with bytes of canaries in it and behind it, and what says that those behind are as they were."""
    import torch

    count = int(np.prod(shape)) * torch.empty(0, dtype=dtype).element_size()
    whole = torch.full((count + behind,), 0xA5, dtype=torch.uint8, device="cuda")
    return whole[:count].view(dtype).reshape(shape), lambda: bool((whole[count:] == 0xA5).all())


@pytest.mark.parametrize("element,dtype", [("f16", "float16"), ("bf16", "bfloat16"), ("f32", "float32")])
def test_gathered_rows_of_pointers(runtime, element, dtype):
    """Fewer and more slots than rows, rows further apart than they are long, an index beyond them."""
    import torch

    rng = np.random.default_rng(51)
    stream = torch.cuda.current_stream().cuda_stream
    for slots, source, k, stride in ((9, 40, 160, 161), (70, 5, 576, 640), (1, 1, 32, 32)):
        bits = special_rows(rng, source, k, dtype)
        index = rng.integers(0, source, slots).astype(np.uint32)
        index[-1] = source - 1
        beyond = index.copy()
        beyond[-1] = source + 7
        wide = np.concatenate([bits, np.full((source, stride - k), 0x7F, bits.dtype)], axis=1)
        x, rows = on_gpu(wide.view({2: np.int16, 4: np.int32}[wide.itemsize])), on_gpu(beyond)
        (codes, codes_kept), (scales, scales_kept) = guarded((slots, k // 2), torch.uint8), guarded(((k + 127) // 128, slots), torch.int32)
        runtime.mxfp4_quantize_pointers(element, x.data_ptr(), rows.data_ptr(), codes.data_ptr(), scales.data_ptr(), slots, source, k, stride, stream)
        nibbles, exponents = mx.quantize(from_bits(bits, dtype)[index])
        assert np.array_equal(mx.exponents(scales.cpu().numpy().view(np.uint32), k), exponents) and scales_kept()
        assert np.array_equal(mx.unpack(codes.cpu().numpy()), nibbles) and codes_kept()


@pytest.mark.parametrize("element,dtype", [("f16", "float16"), ("bf16", "bfloat16")])
def test_pairs_of_pointers(runtime, element, dtype):
    """The same bits as a dispatch of the kernel, whose results are compared with the definition, and none behind them."""
    import torch

    from llmopt_b200 import dispatch

    rng = np.random.default_rng(52)
    stream = torch.cuda.current_stream().cuda_stream
    for counts, n, k in (([3, 0, 9], 64, 160), ([150, 1, 0, 60], 202, 2048)):
        expert_of_slot, x, w, score = expert_case(rng, counts, n, k)
        x = x[0], (x[1] - 4).astype(np.uint8)
        slots, plan = len(expert_of_slot), mx.plan_of(expert_of_slot, len(counts))
        xt, wt, want = upload(runtime, x), upload(runtime, w), blank(runtime, (slots, n // 2), dtype)
        dispatch.dispatch_mxfp4_expert_rows(context(runtime), input=xt[0], input_scales=xt[1], weight=wt[0], weight_scales=wt[1], experts=len(counts),
                                            plan=device(runtime, plan).buffer, output=want, score_of_slot=device(runtime, score))
        held = [on_gpu(a) for a in (mx.pack(x[0]), mx.words(x[1]), mx.pack(w[0]), mx.words(w[1]), plan, score)]
        y, kept = guarded((slots, n // 2), torch.int16)
        runtime.mxfp4_expert_rows_pointers(element, *[t.data_ptr() for t in held], y.data_ptr(), slots, n, k, len(counts), True, stream)
        assert np.array_equal(y.cpu().numpy().view(np.uint16), read(want)) and kept()


def whole_numbers(rng, m, n, k):
    """Operands of a product whose sums fp32 holds, on the GPU, and the product."""
    pick = np.array([0, 2, 4, 5, 10, 12, 13], np.uint8)
    x, w = rng.choice(pick, (m, k)), rng.choice(pick, (n, k))
    ones = [np.full((rows, k // 32), 127, np.uint8) for rows in (m, n)]
    want = mx.values(x, ones[0]).astype(np.float32) @ mx.values(w, ones[1]).astype(np.float32).T
    return [on_gpu(a) for a in (mx.pack(x), mx.words(ones[0]), mx.pack(w), mx.words(ones[1]))], want


# streams of one CTA per tile, longer and shorter than their ring, and of clusters; pairs of CTAs with one tile each and with several
SHAPES = [(3, 4096, 4096), (64, 2048, 8192), (20, 40000, 1024), (5, 300, 96), (300, 2304, 2048), (129, 18944, 1536), (100, 256, 96)]


@pytest.mark.parametrize("limit", [0, 1, 2])
def test_products_that_give_up_say_so_to_whoever_waits_for_pointers(runtime, monkeypatch, limit):
    """A context whose kernels look at a barrier ``limit`` times: products that have to wait longer are reported, by the wait for pointers
    alone, to everybody until it is cleared; the others are right, and so is everything that runs after them."""
    import torch

    from llmopt_b200.cuda_native import NativeError, Runtime

    monkeypatch.setenv("LLMOPT_CUDA_MXFP4_WAIT_LIMIT", str(limit))
    hasty = Runtime()
    rng = np.random.default_rng(limit)
    stream = torch.cuda.Stream()
    for m, n, k in SHAPES:
        operands, want = whole_numbers(rng, m, n, k)
        results = [torch.zeros(m, n, device="cuda") for _ in range(4)]
        torch.cuda.synchronize()
        call = lambda which, y, s: which.mxfp4_linear_pointers("f32", *[t.data_ptr() for t in operands], None, y.data_ptr(), m, n, k, s)
        for y in results[:3]:
            call(hasty, y, stream.cuda_stream)
        stream.synchronize()
        hasty.synchronize()  # has another stream and another word
        try:
            hasty.mxfp4_synchronize(stream.cuda_stream)
            gave_up = False
        except NativeError as error:
            assert "ran out" in str(error)
            gave_up = True
        if limit == 0:
            assert gave_up
        if gave_up:
            for clear in (False, True):
                with pytest.raises(NativeError, match="ran out"):
                    hasty.mxfp4_synchronize(0, clear=clear)
        else:
            assert all(np.array_equal(y.cpu().numpy(), want) for y in results[:3])
        hasty.mxfp4_synchronize(stream.cuda_stream)
        call(runtime, results[3], stream.cuda_stream)
        runtime.mxfp4_synchronize(stream.cuda_stream)
        assert np.array_equal(results[3].cpu().numpy(), want)


def test_a_batch_that_gives_up_says_so_to_the_context(runtime, monkeypatch):
    from llmopt_b200 import dispatch
    from llmopt_b200.cuda_native import NativeError, Runtime

    monkeypatch.setenv("LLMOPT_CUDA_MXFP4_WAIT_LIMIT", "0")
    hasty = Runtime()
    rng = np.random.default_rng(3)
    for m in (3, 300):
        x, w = ((rng.integers(0, 16, (rows, 1024)).astype(np.uint8), np.full((rows, 32), 127, np.uint8)) for rows in (m, 256))
        xt, wt, y = upload(hasty, x), upload(hasty, w), blank(hasty, (m, 256), "float32")
        with pytest.raises(NativeError, match="bounded wait"):
            dispatch.dispatch_mxfp4_linear(context(hasty), input=xt[0], input_scales=xt[1], weight=wt[0], weight_scales=wt[1], output=y)
        hasty.synchronize()
        hasty.mxfp4_synchronize()


def cudart():
    """The CUDA runtime that torch has loaded."""
    import ctypes

    with open("/proc/self/maps") as maps:
        return ctypes.CDLL(next(line.split()[-1] for line in maps if "libcudart" in line))


def test_a_launch_that_cuda_refuses_is_no_invalid_argument(runtime):
    """The stream's capture has been spoilt by a wait, so nothing can be launched on it until the capture has ended."""
    import ctypes

    import torch

    from llmopt_b200.cuda_native import NativeError

    torch.cuda.init()
    x, codes, scales = torch.ones(3, 64, device="cuda"), torch.zeros(3, 32, dtype=torch.uint8, device="cuda"), torch.zeros(1, 3, dtype=torch.int32, device="cuda")
    y = torch.zeros(3, 3, device="cuda")
    torch.cuda.synchronize()
    stream, graph, lib = torch.cuda.Stream(), ctypes.c_void_p(), cudart()
    quantize = lambda: runtime.mxfp4_quantize_pointers("f32", x.data_ptr(), None, codes.data_ptr(), scales.data_ptr(), 3, 3, 64, 64, stream.cuda_stream)
    operand = codes.data_ptr(), scales.data_ptr()
    product = lambda: runtime.mxfp4_linear_pointers("f32", *operand, *operand, None, y.data_ptr(), 3, 3, 64, stream.cuda_stream)
    assert lib.cudaStreamBeginCapture(ctypes.c_void_p(stream.cuda_stream), 2) == 0
    assert lib.cudaStreamSynchronize(ctypes.c_void_p(stream.cuda_stream)) != 0
    for call in (quantize, product):
        with pytest.raises(NativeError, match="launch failed"):
            call()
    assert lib.cudaStreamEndCapture(ctypes.c_void_p(stream.cuda_stream), ctypes.byref(graph)) != 0
    lib.cudaGetLastError()
    quantize()
    product()
    stream.synchronize()
    assert (y == 64.0).all()  # ones in four bits are ones
