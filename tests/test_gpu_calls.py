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


@pytest.mark.parametrize("alias", ["detach", "data", "view", "slice", "inference slice"])
def test_an_alias_of_a_view_keeps_the_array(gpu_ctx, alias):
    import gc
    import weakref

    import torch
    ex = sharded.GpuExecutor(gpu_ctx)
    x = A.param(1, "f32")
    prog = A.build_program([A.map(lambda v: v + 1, x)])
    out, = gpu_ctx.execute(prog.text, [gpu_ctx.from_host(np.zeros(64, np.float32))], 1)
    gpu_ctx.sync()
    alive = weakref.ref(out)
    first = ex.tensor(out)
    del out
    if alias == "inference slice":
        with torch.inference_mode():
            other = first[3:]
    else:
        other = {"detach": lambda t: t.detach(), "data": lambda t: t.data, "view": lambda t: t.view(torch.int32), "slice": lambda t: t[3:]}[alias](first)
    del first
    gc.collect()
    assert alive() is not None
    # (the next result of this size does not get that memory)
    again, = gpu_ctx.execute(prog.text, [gpu_ctx.from_host(np.full(64, 9, np.float32))], 1)
    gpu_ctx.sync()
    assert again.devptr() != alive().devptr()
    assert other.view(torch.float32).tolist() == [1.0] * other.numel()
    del other
    gc.collect()
    assert alive() is None


WITHOUT = """
import sys, warnings
warnings.simplefilter("ignore", RuntimeWarning)
sys.modules["accelerate_b200._binding"] = None
from accelerate_b200 import backend, sharded
import accelerate_b200 as A
import numpy as np
import torch
x, v = np.arange(12, dtype=np.float32).reshape(3, 4), np.ones(4, np.float32)
y, (mean, rstd) = backend.run(list(A.layerNorm(1e-5, v, v, x)))
assert np.array_equal(mean, x.mean(-1)) and y.shape == (3, 4)
ex = sharded.GpuExecutor(backend.default_context())
t = torch.arange(6, device="cuda", dtype=torch.float32)
torch.cuda.synchronize()
out = ex.run("twice", lambda a: A.map(lambda e: e * 2, a), [ex.wrap(t, "f32")])
ex.sync()
assert ex.tensor(out).tolist() == [0, 2, 4, 6, 8, 10]
try:
    backend.run(list(A.logProbs(1, np.array([9, 0, 0], np.int32), x)))
    sys.exit("no error")
except backend.B200Error as e:
    assert e.code == 5
"""


def test_runs_without_the_compiled_binding(gpu_ctx):
    import subprocess
    import sys
    r = subprocess.run([sys.executable, "-c", WITHOUT], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr


def test_the_examples_of_the_documentation(gpu_ctx):
    """Two ways to call a row operator: on host arrays, and on torch's tensors without copies."""
    import os
    import re

    import torch
    text = open(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "README.md")).read()
    names = {}
    for code in re.findall(r"```python\n(.*?)```", text, re.S):
        exec(code, names)
    logits, tokens = torch.tensor(names["logits"], device="cuda"), torch.tensor(names["tokens"], device="cuda")
    for _ in range(3):
        stats, top = names["log_probs_of"](tokens, logits)
        # (each round's results go before the next's are computed; their memory is used again)
        got = [t.cpu().numpy() for t in stats + top]
    want = [names[k] for k in ("logp", "normaliser", "entropy", "ids", "top")]
    assert all(np.array_equal(a, b) for a, b in zip(got, want))
    assert np.array_equal(got[3], np.argsort(-names["logits"].astype(np.float64), axis=-1, kind="stable")[:, :5])
