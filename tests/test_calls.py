"""The Python layer's calls into the library, without a GPU: a library that records and answers stands in for it."""
import ctypes

import numpy as np
import pytest

from accelerate_b200 import backend


class Library:
    """Every entry point succeeds; `devptr` answers with `now`."""

    now = 0

    def __getattr__(self, name):
        return lambda *a: 0

    def b200_array_devptr(self, ctx, ident, leaf, out):
        ctypes.cast(out, ctypes.POINTER(ctypes.c_void_p))[0] = self.now
        return 0


class Fast:
    """The compiled binding: a run yields one vector of two Floats at `now`."""

    def __init__(self, library):
        self.library, self.wrapped = library, []

    def execute(self, ctx, prog, ids, n_out):
        return [(9, (2,), ["f32"], (self.library.now,))]

    def wrap(self, ctx, elt, shape, ptrs):
        self.wrapped.append((elt, tuple(shape), tuple(ptrs)))
        return 10

    def free(self, ctx, ident):
        return 0


@pytest.fixture
def calls(monkeypatch):
    library = Library()
    fast = Fast(library)
    monkeypatch.setattr(backend, "lib", lambda: library)
    monkeypatch.setattr(backend, "_fast", fast)
    ctx = backend.Context(0)
    ctx._programs["p"] = ctypes.c_void_p(1)
    return ctx, library, fast


def test_a_result_that_is_an_input_asks_again_once_the_input_was_given_other_data(calls):
    """A program may hand an input on as its result: two handles of one array.  A payload adopted through one of them is
    copied when the array's pointer is next asked for, through either."""
    ctx, library, _ = calls
    a = ctx.array("f32", (2,))
    library.now = 111
    out, = ctx.execute("p", [a], 1)
    assert out.devptr() == 111
    a.adopt_host([np.ones(2, np.float32)])
    library.now = 222
    assert out.devptr() == 222, "the library was not asked, and the adopted payload stays where it is"
    after, = ctx.execute("p", [a], 1)
    library.now = 333
    assert after.devptr() == 222, "known from the run"


class Array:
    """What `GpuExecutor.tensor` looks at of a device array."""

    shape, leaf_types = (3,), ["f32"]

    def devptr(self, leaf=0):
        return 4096


def test_what_torch_keeps_of_a_view_keeps_the_array(monkeypatch):
    """A tensor's storage, and with it every alias (detach, a view of another type, a slice in inference mode), holds the
    object that described the memory, not the attributes of the tensor that was made first."""
    import gc
    import weakref

    import torch

    from accelerate_b200 import sharded
    held = []

    def as_tensor(v, device):
        held.append(v)
        assert v.__cuda_array_interface__["data"] == (4096, False)
        return torch.zeros(3)
    monkeypatch.setattr(sharded, "_as_tensor", as_tensor)
    ex = sharded.GpuExecutor.__new__(sharded.GpuExecutor)
    ex.device = torch.device("cpu")
    a = Array()
    alive = weakref.ref(a)
    t = ex.tensor(a)
    del a, t
    gc.collect()
    assert alive() is not None, "the array's memory went back to the pool under a tensor that still points at it"
    held.clear()
    gc.collect()
    assert alive() is None


COUNTER = r"""
import ctypes, importlib.machinery, importlib.util, sys, threading, time

path, which = sys.argv[1:]
spec = importlib.util.spec_from_loader("_binding", importlib.machinery.ExtensionFileLoader("_binding", path))
binding = importlib.util.module_from_spec(spec)
spec.loader.exec_module(binding)
libc = ctypes.CDLL(None)
address = lambda f: ctypes.cast(f, ctypes.c_void_p).value
# Stand-ins from the C library for what may wait for a context's lock: usleep(context), which succeeds after 0.4 s, and
# abs(x), which succeeds at once for 0 and fails for anything else (a failed description: the results are freed again).
wait, done = address(libc.usleep), address(libc.abs)
calls = {name: done for name in ("wrap", "run", "info", "devptr", "free")}
calls["free" if which == "cleanup" else which] = wait
binding.setup(calls["wrap"], calls["run"], calls["info"], calls["devptr"], calls["free"], address(libc.gnu_get_libc_version), RuntimeError, ("f32",))
# (a run's first argument is the program, the others' the context)
ctx, prog = (0, 400000) if which == "run" else (400000, 0)
call = {"cleanup": lambda: fails(lambda: binding.execute(ctx, prog, [], 1)), "wrap": lambda: binding.wrap(ctx, b"f32", (), ()), "free": lambda: binding.free(ctx, 1)}.get(which, lambda: binding.execute(ctx, prog, [], 1))
def fails(f):
    try:
        f()
        sys.exit("no error")
    except RuntimeError:
        pass


thread = threading.Thread(target=call)
longest, last = 0.0, time.perf_counter()
began = last
thread.start()
while thread.is_alive():
    time.sleep(0.001)
    now = time.perf_counter()
    longest, last = max(longest, now - last), now
print(longest, last - began)
"""


@pytest.mark.parametrize("which", ["wrap", "run", "info", "free", "cleanup"])
def test_the_interpreter_runs_while_a_call_waits_for_the_library(lib_built, which):
    """A call may wait for a context's lock as long as another thread's download takes; other threads go on meanwhile."""
    import subprocess
    import sys

    from accelerate_b200 import build
    r = subprocess.run([sys.executable, "-c", COUNTER, build.BINDING, which], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0, r.stderr
    longest, whole = map(float, r.stdout.split())
    assert whole >= 0.39 and longest < 0.3, "the interpreter stood still for as long as the call waited"


POINTERS = r"""
import ctypes, importlib.machinery, importlib.util, sys

spec = importlib.util.spec_from_loader("_binding", importlib.machinery.ExtensionFileLoader("_binding", sys.argv[1]))
binding = importlib.util.module_from_spec(spec)
spec.loader.exec_module(binding)
address = lambda f: ctypes.cast(f, ctypes.c_void_p).value
got = []


@ctypes.CFUNCTYPE(ctypes.c_int, ctypes.c_void_p, ctypes.c_char_p, ctypes.c_int, ctypes.POINTER(ctypes.c_int64), ctypes.POINTER(ctypes.c_void_p),
                  ctypes.POINTER(ctypes.c_uint64))
def wrap(ctx, elt, rank, shape, ptrs, out):
    got.append((ctx, elt, shape[:rank], ptrs[:4]))
    out[0] = 10
    return 0


a = address(ctypes.CDLL(None).abs)
binding.setup(address(wrap), a, a, a, a, a, RuntimeError, ("f32",))
assert binding.wrap(5, b"f32", (2, 3), [ctypes.c_void_p(64), 128, None, ctypes.c_void_p(None)]) == 10
assert got == [(5, b"f32", [2, 3], [64, 128, None, None])], got
for bad in (5.0, "64", ctypes.c_float(1), [64]):
    try:
        binding.wrap(5, b"f32", (2, 3), [bad])
        sys.exit(repr(bad))
    except TypeError:
        pass
assert len(got) == 1
"""


def test_pointers_may_be_numbers_or_void_pointers(lib_built):
    import subprocess
    import sys

    from accelerate_b200 import build
    r = subprocess.run([sys.executable, "-c", POINTERS, build.BINDING], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0, r.stderr


MESSAGE = r"""
import ctypes, importlib.machinery, importlib.util, sys

spec = importlib.util.spec_from_loader("_binding", importlib.machinery.ExtensionFileLoader("_binding", sys.argv[1]))
binding = importlib.util.module_from_spec(spec)
spec.loader.exec_module(binding)
text = ctypes.create_string_buffer(b"unknown name \xff")
last_error = ctypes.CFUNCTYPE(ctypes.c_void_p)(lambda: ctypes.addressof(text))
address = lambda f: ctypes.cast(f, ctypes.c_void_p).value
a = address(ctypes.CDLL(None).abs)


class Error(RuntimeError):
    pass


binding.setup(a, a, a, a, a, address(last_error), Error, ("f32",))
for call in (lambda: binding.wrap(3, b"f32", (), ()), lambda: binding.execute(0, 3, [], 1)):
    try:
        call()
        sys.exit("no error")
    except Error as e:
        assert e.args == (3, "unknown name �"), e.args
"""


def test_a_message_that_is_not_utf8_arrives_all_the_same(lib_built):
    import subprocess
    import sys

    from accelerate_b200 import build
    r = subprocess.run([sys.executable, "-c", MESSAGE, build.BINDING], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0, r.stderr


class Tensor:
    """What `GpuExecutor.wrap` looks at of a tensor."""

    def __init__(self, dtype, device=0, shape=(4, 6), contiguous=True, pinned=False):
        self.dtype, self.device_index, self.shape, self.contiguous, self.pinned = dtype, device, shape, contiguous, pinned

    def get_device(self): return self.device_index
    def element_size(self): return self.dtype.itemsize
    def numel(self): return int(np.prod(self.shape))
    def is_contiguous(self): return self.contiguous
    def is_pinned(self): return self.pinned
    def data_ptr(self): return 4096


def test_memory_that_cannot_be_the_array_is_not_wrapped(calls):
    import torch

    from accelerate_b200 import sharded
    ctx, _, fast = calls
    ex = sharded.GpuExecutor.__new__(sharded.GpuExecutor)
    ex.ctx = ctx
    for t, elt in [(Tensor(torch.float32, device=-1), "f32"), (Tensor(torch.float32, device=1), "f32"),       # host memory; another GPU's
                   (Tensor(torch.float16), "f32"), (Tensor(torch.int32), "i64"), (Tensor(torch.int64), "i32"),   # fewer or more bytes
                   (Tensor(torch.bfloat16), "f16"), (Tensor(torch.complex64), "f64"),                          # other numbers
                   (Tensor(torch.float32, contiguous=False), "f32"), (Tensor(torch.float16), ("f32",))]:
        with pytest.raises(ValueError):
            ex.wrap(t, elt)
    assert not fast.wrapped
    for t, elt in [(Tensor(torch.float32), "f32"), (Tensor(torch.bool), "u8"), (Tensor(torch.int16), "u16"), (Tensor(torch.bfloat16), "u16"),
                   (Tensor(torch.float16), ("f16",)), (Tensor(torch.int32), "f32"),
                   (Tensor(torch.float32, device=-1, pinned=True), "f32"), (Tensor(torch.float32, device=-1, shape=(0, 3)), "f32")]:
        assert ex.wrap(t, elt).shape == t.shape
    assert len(fast.wrapped) == 8


def test_the_compiled_binding_is_named_after_the_interpreter(lib_built):
    """Another Python version in the same checkout must not load a module that was built for this one."""
    import importlib.machinery
    import os

    from accelerate_b200 import _binding, build
    tagged = importlib.machinery.EXTENSION_SUFFIXES[0]
    assert "cpython" in tagged and build.BINDING.endswith("_binding" + tagged)
    assert os.path.samefile(_binding.__file__, build.BINDING)
    assert not os.path.exists(os.path.join(os.path.dirname(build.BINDING), "_binding.so")), "any version would load that one"


def test_the_library_is_built_where_python_has_no_headers(lib_built, monkeypatch, tmp_path):
    """The C ABI has other users, and the Python layer makes the same calls through ctypes where the module is missing."""
    from accelerate_b200 import build
    missing = str(tmp_path / ("_binding" + ".so"))
    monkeypatch.setattr(build, "BINDING", missing)
    monkeypatch.setattr(build.sysconfig, "get_paths", lambda: {"include": str(tmp_path)})
    with pytest.warns(RuntimeWarning, match="Python.h"):
        assert build.build() == lib_built
    assert not (tmp_path / "_binding.so").exists()


WITHOUT = """
import sys, warnings
sys.modules["accelerate_b200._binding"] = None
from accelerate_b200 import backend
import accelerate_b200 as A
import numpy as np
with warnings.catch_warnings(record=True) as said:
    warnings.simplefilter("always")
    backend.lib()
assert [w.category for w in said] == [RuntimeWarning], said
text = A.build_program([A.map(lambda v: v + 1, A.param(1, "f32"))]).text
assert "ok elementwise" in backend.compile_check(text)
"""


def test_the_backend_runs_without_the_compiled_binding(lib_built):
    import subprocess
    import sys
    r = subprocess.run([sys.executable, "-c", WITHOUT], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stderr


def test_calls_through_ctypes_make_the_same_of_the_library(monkeypatch):
    """The stand-in for the compiled binding against a library that answers: ids, shapes, types, pointers, errors."""
    class Answers(Library):
        freed = []

        def b200_array_wrap(self, ctx, elt, rank, shape, ptrs, out):
            assert ctx == 77 and elt == b"f32" and rank == 2 and list(shape[:2]) == [2, 3] and ptrs[0] == 64
            ctypes.cast(out, ctypes.POINTER(ctypes.c_uint64))[0] = 5
            return 0

        def b200_program_run(self, prog, ins, n_in, outs, n_out):
            assert prog == 88 and list(ins[:n_in]) == [5, 6]
            outs[0], outs[1] = 11, 12
            return 0

        def b200_array_info(self, ctx, ident, max_rank, rank, shape, max_leaves, leaves, types):
            ctypes.cast(rank, ctypes.POINTER(ctypes.c_int))[0] = 1
            ctypes.cast(leaves, ctypes.POINTER(ctypes.c_int))[0] = 2
            shape[0], types[0], types[1] = 7, 8, 2
            return 3 if ident == self.bad else 0

        def b200_array_devptr(self, ctx, ident, leaf, out):
            ctypes.cast(out, ctypes.POINTER(ctypes.c_void_p))[0] = 1000 * ident + leaf
            return 0

        def b200_array_free(self, ctx, ident):
            self.freed.append(ident)
            return 0

        def b200_last_error(self):
            return b"no such array"
    library = Answers()
    library.bad = None
    monkeypatch.setattr(backend, "lib", lambda: library)
    calls = backend._CtypesCalls
    assert calls.wrap(77, b"f32", (2, 3), (64,)) == 5
    assert calls.execute(77, 88, [5, 6], 2) == [(11, (7,), ["f32", "i32"], (11000, 11001)), (12, (7,), ["f32", "i32"], (12000, 12001))]
    assert calls.free(77, 11) == 0 and library.freed == [11]
    library.bad = 12
    with pytest.raises(backend.B200Error) as e:
        calls.execute(77, 88, [5, 6], 2)
    assert e.value.code == 3 and "no such array" in str(e.value) and library.freed == [11, 11, 12], "nobody else knows the results' ids"


LARGE = r"""
import ctypes, importlib.machinery, importlib.util, resource, sys

spec = importlib.util.spec_from_loader("_binding", importlib.machinery.ExtensionFileLoader("_binding", sys.argv[1]))
binding = importlib.util.module_from_spec(spec)
spec.loader.exec_module(binding)
libc = ctypes.CDLL(None)
address = lambda f: ctypes.cast(f, ctypes.c_void_p).value
a = address(libc.abs)
binding.setup(a, a, a, a, a, address(libc.gnu_get_libc_version), RuntimeError, ("f32",))
before = resource.getrusage(resource.RUSAGE_SELF).ru_maxrss
try:
    binding.execute(0, 3, [], 1 << 20)
    sys.exit("no error")
except RuntimeError:
    pass
assert resource.getrusage(resource.RUSAGE_SELF).ru_maxrss - before < 50 << 10
"""


def test_a_wrong_number_of_results_costs_no_memory(lib_built):
    """The library says that the program yields another number; nothing is described before."""
    import subprocess
    import sys

    from accelerate_b200 import build
    r = subprocess.run([sys.executable, "-c", LARGE, build.BINDING], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0, r.stderr
