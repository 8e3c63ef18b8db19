"""The W4A16 linear on raw device pointers: the default stream."""

import numpy as np
import pytest

from conftest import assert_close_f16
from helpers import random_w4

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("m", [1, 3, 40, 200])
def test_calls_on_the_default_stream_come_after_its_work(runtime, oracle, m):
    """A stream of 0 is torch's default one: what that still has to write is read, and what it does next reads the results."""
    import torch

    torch.cuda.init()
    rng = np.random.default_rng(m)
    n, k = 256, 512
    packed, scale = random_w4(rng, n, k)
    values = rng.standard_normal((m, k)).astype(np.float16)
    on = lambda array: torch.from_numpy(np.ascontiguousarray(array)).cuda()
    weight, scales, source = on(packed), on(scale), on(values)
    x, y = torch.zeros(m, k, dtype=torch.float16, device="cuda"), torch.zeros(m, n, dtype=torch.float16, device="cuda")
    torch.cuda.synchronize()
    assert torch.cuda.current_stream().cuda_stream == 0
    torch.cuda._sleep(50_000_000)
    x.copy_(source)
    runtime.w4a16_linear_pointers(x.data_ptr(), weight.data_ptr(), scales.data_ptr(), None, y.data_ptr(), m, n, k, 0)
    got = y.clone()
    x.zero_()
    y.zero_()
    assert_close_f16(got.cpu().numpy(), oracle.w4a16_linear(values, packed, scale, None, 0))
    runtime.synchronize()
