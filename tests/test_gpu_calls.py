"""The Python layer's calls into the library, on the GPU."""
import numpy as np
import pytest

import accelerate_b200 as A
from accelerate_b200 import sharded

pytestmark = pytest.mark.gpu


def test_a_view_of_a_result_that_is_an_input_sees_the_adopted_payload(gpu_ctx):
    ex = sharded.GpuExecutor(gpu_ctx)
    x = A.param(1, "f32")
    prog = A.build_program([x, A.map(lambda v: v + 1, x)])
    a = gpu_ctx.from_host(np.zeros(5, np.float32))
    same, more = gpu_ctx.execute(prog.text, [a], 2)
    a.adopt_host([np.full(5, 7, np.float32)])
    view = ex.tensor(same)
    gpu_ctx.sync()
    assert view.tolist() == [7.0] * 5
    assert np.array_equal(more.download(), np.ones(5, np.float32))
