"""MXFP4 on the host: the packing against the definition, the dispatchers' records and refusals, and the C entry points' refusals, which
come before anything touches a device."""

import numpy as np
import pytest

import mxfp4_oracle as mx


class Recorder:
    def __init__(self):
        self.records = []

    def dispatch(self, entry, *, buffers, parameters, grid=(1, 1, 1), batch=None):
        self.records.append((entry, list(buffers), parameters))
        return entry


def _tensor(name, shape, dtype):
    from llmopt_b200 import dispatch

    return dispatch.Tensor(name, shape, dtype)


def _context():
    from llmopt_b200 import dispatch

    return dispatch.Context(Recorder())


def test_oracle_rounds_to_the_nearest_element_and_ties_to_even():
    x = np.zeros((1, 64))
    x[0, :8] = [4.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0]
    x[0, 8:16] = [-7.99, 0.24999, 0.25001, 4.99, 5.01, -0.0, 6.5, 7.0]
    nibbles, exponents = mx.quantize(x)
    assert exponents.tolist() == [[127, 0]]
    want = [4, 0, 1, 1, 2, 2, 4, 4, -6, 0, 0.5, 4, 6, -0.0, 6, 6]
    got = mx.values(nibbles, exponents)[0, :16]
    assert got.tolist() == want and np.signbit(got[13])


@pytest.mark.parametrize("rows,k", [(1, 32), (3, 96), (5, 128), (2, 160), (7, 576)])
def test_host_packing_is_the_definition(rows, k):
    from llmopt_b200.quantize import pack_mxfp4_weight

    rng = np.random.default_rng(1)
    x = (rng.standard_normal((rows, k)) * np.exp2(rng.integers(-140, 127, (rows, 1)))).astype(np.float32)
    x[0, :5] = [0.0, -0.0, 1.5, 2.5, -3.5]
    if rows > 2:
        x[1, :32], x[2, 40], x[2, 70] = 0.0, np.inf, np.nan
    codes, words = pack_mxfp4_weight(x)
    nibbles, exponents = mx.quantize(x)
    assert np.array_equal(codes, mx.pack(nibbles)) and np.array_equal(words, mx.words(exponents))
    assert words.shape == ((k + 127) // 128, rows)


def test_packing_refuses_what_is_no_rows_of_blocks():
    from llmopt_b200 import quantize

    for shape in ((4, 48), (4, 0), (32,), (1, 2, 32)):
        with pytest.raises(ValueError):
            quantize.pack_mxfp4_weight(np.zeros(shape, np.float32))
    with pytest.raises(TypeError):
        quantize.mxfp4_scale_words(np.zeros((2, 4), np.int32))


def test_records_of_a_layer():
    from llmopt_b200 import dispatch, parameters

    context = _context()
    x, codes, scales = _tensor("x", (5, 100), "bfloat16"), _tensor("c", (5, 48), "uint8"), _tensor("s", (1, 5), "uint32")
    dispatch.dispatch_mxfp4_quantize(context, input=x, codes=codes, scales=scales, columns=96)
    slots = _tensor("i", (7,), "uint32")
    dispatch.dispatch_mxfp4_quantize(context, input=_tensor("x", (5, 96), "float32"), codes=_tensor("c", (7, 48), "uint8"),
                                     scales=_tensor("s", (1, 7), "uint32"), row_of_slot=slots)
    dispatch.dispatch_mxfp4_dequantize(context, codes=codes, scales=scales, output=_tensor("o", (5, 96), "float16"))
    w, ws = _tensor("w", (12, 48), "uint8"), _tensor("ws", (1, 12), "uint32")
    dispatch.dispatch_mxfp4_linear(context, input=codes, input_scales=scales, weight=w, weight_scales=ws, output=_tensor("y", (5, 12), "float32"))
    dispatch.dispatch_mxfp4_linear(context, input=codes, input_scales=scales, weight=w, weight_scales=ws,
                                   output=_tensor("y", (5, 12), "float16"), bias=_tensor("b", (12,), "float16"))
    dispatch.dispatch_mxfp4_expert_rows(context, input=codes, input_scales=scales, weight=w, weight_scales=ws, experts=3, plan="plan",
                                        output=_tensor("y", (5, 2), "float16"), score_of_slot=_tensor("g", (5,), "float32"))
    dispatch.dispatch_mxfp4_expert_rows(context, input=codes, input_scales=scales, weight=w, weight_scales=ws, experts=3, plan="plan",
                                        output=_tensor("y", (5, 4), "float32"))
    assert context.runtime.records == [
        ("llmopt_mxfp4_quantize_bf16", ["x", "c", "s"], parameters.u32s([5, 96, 100])),
        ("llmopt_mxfp4_quantize_rows_f32", ["x", "i", "c", "s"], parameters.u32s([7, 96, 96, 5])),
        ("llmopt_mxfp4_dequantize_f16", ["c", "s", "o"], parameters.u32s([5, 96])),
        ("llmopt_mxfp4_linear_f32", ["c", "s", "w", "ws", "y", "y"], parameters.u32s([5, 12, 96, 0])),
        ("llmopt_mxfp4_linear_f16", ["c", "s", "w", "ws", "b", "y"], parameters.u32s([5, 12, 96, 1])),
        ("llmopt_mxfp4_expert_rows_f16", ["c", "s", "w", "ws", "plan", "g", "y"], parameters.u32s([5, 4, 96, 3, 1])),
        ("llmopt_mxfp4_expert_rows_bf16", ["c", "s", "w", "ws", "plan", "plan", "y"], parameters.u32s([5, 4, 96, 3, 0])),
    ]


def test_dispatchers_refuse_inconsistent_operands():
    from llmopt_b200 import dispatch

    context = _context()
    good = dict(input=_tensor("c", (5, 48), "uint8"), input_scales=_tensor("s", (1, 5), "uint32"), weight=_tensor("w", (12, 48), "uint8"),
                weight_scales=_tensor("ws", (1, 12), "uint32"))
    y = _tensor("y", (5, 12), "float16")
    for wrong in (dict(input=_tensor("c", (5, 32), "uint8")), dict(input=_tensor("c", (5, 48), "int8")),
                  dict(input_scales=_tensor("s", (5, 1), "uint32")), dict(weight_scales=_tensor("ws", (2, 12), "uint32")),
                  dict(weight=_tensor("w", (12, 40), "uint8")), dict(output=_tensor("y", (5, 11), "float16")),
                  dict(weight=_tensor("w", (576,), "uint8")), dict(input=_tensor("c", (), "uint8")), dict(output=_tensor("y", (5, 12), "float64")), dict(bias=_tensor("b", (12,), "float32")),
                  dict(bias=_tensor("b", (11,), "float16"))):
        with pytest.raises(dispatch.DispatchError):
            dispatch.dispatch_mxfp4_linear(context, **{**good, "output": y, **wrong})
    score = _tensor("g", (5,), "float32")
    experts = dict(**good, experts=3, plan="plan", output=_tensor("y", (5, 2), "bfloat16"), score_of_slot=score)
    for wrong in (dict(experts=5), dict(experts=4), dict(experts=0), dict(weight=_tensor("w", (576,), "uint8")), dict(output=_tensor("y", (5, 2), "float32")),
                  dict(output=_tensor("y", (5, 4), "bfloat16")), dict(score_of_slot=None), dict(score_of_slot=_tensor("g", (4,), "float32"))):
        with pytest.raises(dispatch.DispatchError):
            dispatch.dispatch_mxfp4_expert_rows(context, **{**experts, **wrong})
    quantize = dict(input=_tensor("x", (5, 100), "float16"), codes=_tensor("c", (5, 48), "uint8"), scales=_tensor("s", (1, 5), "uint32"), columns=96)
    for wrong in (dict(columns=None), dict(columns=128), dict(columns=0), dict(input=_tensor("x", (500,), "float16")),
                  dict(input=_tensor("x", (5, 100), "int32")), dict(row_of_slot=_tensor("i", (6,), "uint32")),
                  dict(row_of_slot=_tensor("i", (5,), "int64")), dict(scales=_tensor("s", (1, 5), "uint8"))):
        with pytest.raises(dispatch.DispatchError):
            dispatch.dispatch_mxfp4_quantize(context, **{**quantize, **wrong})
    for wrong in (dict(output=_tensor("o", (5, 90), "float16")), dict(output=_tensor("o", (4, 96), "float16")), dict(output=_tensor("o", (480,), "float16"))):
        with pytest.raises(dispatch.DispatchError):
            dispatch.dispatch_mxfp4_dequantize(context, **{**dict(codes=quantize["codes"], scales=quantize["scales"]), **wrong})
    assert not context.runtime.records


def test_entry_points_need_a_context():
    import threading

    from llmopt_b200 import cuda_native

    lib, got = cuda_native.load_library(), []

    def call():  # messages are kept per thread
        got.append(lib.llmopt_cuda_mxfp4_quantize(None, 0, 16, None, 16, 16, 1, 1, 32, 32, None))
        got.append(lib.llmopt_cuda_mxfp4_dequantize(None, 0, 16, 16, 16, 1, 32, None))
        got.append(lib.llmopt_cuda_mxfp4_linear(None, 0, 16, 16, 16, 16, None, 16, 1, 1, 32, None))
        got.append(lib.llmopt_cuda_mxfp4_expert_rows(None, 0, 16, 16, 16, 16, 16, 16, 16, 1, 2, 32, 1, 1, None))
        got.append(lib.llmopt_cuda_last_error())

    thread = threading.Thread(target=call)
    thread.start()
    thread.join()
    assert got == [1, 1, 1, 1, b"CUDA context has been finalized"]


# ---- routed experts of a decoder ------------------------------------------------------------------------

def test_records_of_a_step_with_experts_in_mxfp4():
    """Any number of rows goes the same way: sorted, quantized, multiplied, quantized, multiplied, combined."""
    from unittest import mock

    from llmopt_b200 import mixer_engine
    from mixer_models import dense_mlp, routed_mlp, sandwich_config, window_layer
    from test_dalorax_cpu import RecordingEngine

    config = sandwich_config([window_layer(mlp=dense_mlp(64)), window_layer(kv_from=0, mlp=routed_mlp(6, 2, 32))], width=96)
    with mock.patch.object(mixer_engine.MixerEngine, "upload_matrix_mxfp4", lambda self, array: (array.shape, "scales")):
        engine = RecordingEngine(config, batch=3, capacity=256, experts="mxfp4")
    assert engine.layers[1].feed_forward.up == ((6 * 2 * 32, 96), "scales") and engine.layers[1].feed_forward.down == ((6 * 96, 32), "scales")
    routed = ["llmopt_route_rows_f32", "llmopt_route_plan", "llmopt_mxfp4_quantize_rows_bf16", "llmopt_mxfp4_expert_rows_bf16",
              "llmopt_mxfp4_quantize_bf16", "llmopt_mxfp4_expert_rows_bf16", "llmopt_expert_combine_bf16"]
    for recorded in engine.names.values():
        assert recorded[-7:] == routed and not any("mxfp4" in name for name in recorded[:-7])


def test_experts_in_mxfp4_need_whole_blocks_and_bfloat16():
    from mixer_models import dense_mlp, routed_mlp, sandwich_config, window_layer
    from test_dalorax_cpu import RecordingEngine

    routed = [window_layer(mlp=routed_mlp(4, 2, 32))]
    for config, options in ((sandwich_config(routed, width=104), {}), (sandwich_config([window_layer(mlp=routed_mlp(4, 2, 48))], width=96), {}),
                            (sandwich_config(routed, width=96), {"dtype": "float32"}), (sandwich_config([window_layer(mlp=dense_mlp(64))], width=96), {})):
        with pytest.raises(ValueError, match="multiples of 32"):
            RecordingEngine(config, capacity=64, experts="mxfp4", **options)
    with pytest.raises(ValueError, match="unsupported format"):
        RecordingEngine(sandwich_config(routed, width=96), capacity=64, experts="int4")
