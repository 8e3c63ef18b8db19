"""Calls of the MXFP4 operators at the ends of what they take, as far as they need no GPU."""

import threading

import pytest


class Recorder:
    """Keeps records, after the checks that a record of a runtime gets."""

    def __init__(self):
        self.records = []

    def dispatch(self, entry, *, buffers, parameters, grid=(1, 1, 1), batch=None):
        from llmopt_b200.cuda_native import DispatchItem, pack_records

        pack_records([DispatchItem(entry, [], bytes(parameters), tuple(grid), (1, 1, 1))])
        assert min(grid) > 0  # what the runtime refuses
        self.records.append(entry)


@pytest.mark.parametrize("m,n,k", [(0, 64, 32), (1, 8, 32), (4096, 128256, 4096), (1 << 20, 32768, 1024)])
def test_a_product_of_any_size_is_recorded(m, n, k):
    """No rows, and more results than 2^31 threads would have an eighth of."""
    from llmopt_b200 import dispatch

    tensor = lambda shape, dtype: dispatch.Tensor("buffer", shape, dtype)
    runtime, words = Recorder(), dispatch.mxfp4_scale_words(k)
    dispatch.dispatch_mxfp4_linear(dispatch.Context(runtime), input=tensor((m, k // 2), "uint8"), input_scales=tensor((words, m), "uint32"),
                                   weight=tensor((n, k // 2), "uint8"), weight_scales=tensor((words, n), "uint32"), output=tensor((m, n), "float16"))
    assert runtime.records == ["llmopt_mxfp4_linear_f16"]


def test_the_wait_for_pointers_needs_a_context():
    from llmopt_b200 import cuda_native

    lib, got = cuda_native.load_library(), []
    call = lambda: got.extend([lib.llmopt_cuda_mxfp4_synchronize(None, None, 0), lib.llmopt_cuda_last_error()])
    thread = threading.Thread(target=call)  # messages are kept per thread
    thread.start()
    thread.join()
    assert got == [1, b"CUDA context has been finalized"]
