"""``run`` / ``runN`` on a B200 through the C-ABI library (``libaccb200.so``).

Mirrors the reference backend interface (``Interpreter.hs:93-126``): ``run``
evaluates a closed array term, ``runN`` turns a function over arrays into a
function over host arrays that is compiled once and reused.  There is no CPU
fallback: without the built library or without a GPU every entry point raises.
"""
from __future__ import annotations

import ctypes
import os
import warnings

import numpy as np

from . import language as L

_HERE = os.path.dirname(os.path.abspath(__file__))
_LIB_PATH = os.path.join(_HERE, "libaccb200.so")
_lib = None
_fast = None          # the compiled binding of the calls that every run makes (csrc/python/binding.cpp)

ERRORS = {1: "parse", 2: "type", 3: "compile", 4: "cuda", 5: "bounds", 6: "unsupported", 7: "argument", 8: "timeout", 9: "arithmetic"}


class B200Error(RuntimeError):
    """Failure reported by the backend (the Haskell wrapper would throw the
    corresponding ``boundsError`` / ``internalError``, Error.hs:77-85)."""

    def __init__(self, code, message):
        super().__init__(f"[{ERRORS.get(code, code)}] {message}")
        self.code = code


class _CtypesCalls:
    """The compiled binding's calls through ctypes, for a Python without the headers to build it: the same library and
    kernels, some 30 us more for every run."""

    @staticmethod
    def wrap(ctx, elt, shape, ptrs):
        ident = ctypes.c_uint64()
        sh, arr = (ctypes.c_int64 * max(1, len(shape)))(*shape), (ctypes.c_void_p * max(1, len(ptrs)))(*ptrs)
        _check(lib().b200_array_wrap(ctx, elt, len(shape), sh, arr, ctypes.byref(ident)))
        return ident.value

    @staticmethod
    def execute(ctx, prog, ids, n_out):
        ins, outs = (ctypes.c_uint64 * max(1, len(ids)))(*ids), (ctypes.c_uint64 * max(1, n_out))()
        _check(lib().b200_program_run(prog, ins, len(ids), outs, n_out))
        try:
            described = [_describe(ctx, outs[k]) for k in range(n_out)]
            return [(outs[k], shape, types, tuple(_pointer(ctx, outs[k], leaf) for leaf in range(len(types))))
                    for k, (shape, types) in enumerate(described)]
        except B200Error:
            for k in range(n_out):
                lib().b200_array_free(ctx, outs[k])
            raise

    @staticmethod
    def free(ctx, ident):
        return lib().b200_array_free(ctx, ident)


def _describe(ctx, ident):
    """Shape and leaf types of an array, from the library."""
    rank, leaves = ctypes.c_int(), ctypes.c_int()
    for most_rank, most_leaves in ((8, 32), (1 << 10, 1 << 16)):
        sh, types = (ctypes.c_int64 * most_rank)(), (ctypes.c_int32 * most_leaves)()
        rc = lib().b200_array_info(ctx, ident, most_rank, ctypes.byref(rank), sh, most_leaves, ctypes.byref(leaves), types)
        if rc == 0:
            break
    _check(rc)
    return tuple(sh[:rank.value]), [L.SCALARS[k] for k in types[:leaves.value]]


def _pointer(ctx, ident, leaf):
    p = ctypes.c_void_p()
    _check(lib().b200_array_devptr(ctx, ident, leaf, ctypes.byref(p)))
    return p.value or 0


def lib():
    """The loaded C-ABI library; raises if it has not been built."""
    global _lib, _fast
    if _lib is None:
        if not os.path.exists(_LIB_PATH):
            raise B200Error(4, f"{_LIB_PATH} is missing: build it with `python -m accelerate_b200.build` (no CPU fallback exists)")
        l = ctypes.CDLL(_LIB_PATH)
        vp, cp, i64p, u64p = ctypes.c_void_p, ctypes.c_char_p, ctypes.POINTER(ctypes.c_int64), ctypes.POINTER(ctypes.c_uint64)
        l.b200_last_error.restype = cp
        l.b200_ctx_create.argtypes = [ctypes.c_int, ctypes.c_uint32, ctypes.POINTER(vp)]
        l.b200_ctx_destroy.argtypes = [vp]
        l.b200_ctx_destroy.restype = None
        l.b200_array_new.argtypes = [vp, cp, ctypes.c_int, i64p, u64p]
        l.b200_array_wrap.argtypes = [vp, cp, ctypes.c_int, i64p, ctypes.POINTER(vp), u64p]
        l.b200_array_upload.argtypes = [vp, ctypes.c_uint64, ctypes.c_int, vp, ctypes.c_size_t]
        l.b200_array_download.argtypes = [vp, ctypes.c_uint64, ctypes.c_int, vp, ctypes.c_size_t]
        l.b200_array_adopt_host.argtypes = [vp, ctypes.c_uint64, ctypes.c_int, vp, ctypes.c_size_t]
        l.b200_array_download_async.argtypes = [vp, ctypes.c_uint64, ctypes.c_int, vp, ctypes.c_size_t]
        l.b200_array_free.argtypes = [vp, ctypes.c_uint64]
        l.b200_array_intern.argtypes = [vp, ctypes.c_uint64, cp, ctypes.c_int, i64p, ctypes.POINTER(vp), u64p]
        l.b200_array_forget.argtypes = [vp, ctypes.c_uint64]
        l.b200_array_rank.argtypes = [vp, ctypes.c_uint64, ctypes.POINTER(ctypes.c_int)]
        l.b200_array_shape.argtypes = [vp, ctypes.c_uint64, i64p]
        l.b200_array_num_leaves.argtypes = [vp, ctypes.c_uint64, ctypes.POINTER(ctypes.c_int)]
        l.b200_array_leaf_type.argtypes = [vp, ctypes.c_uint64, ctypes.c_int, ctypes.POINTER(cp)]
        l.b200_array_info.argtypes = [vp, ctypes.c_uint64, ctypes.c_int, ctypes.POINTER(ctypes.c_int), i64p, ctypes.c_int,
                                      ctypes.POINTER(ctypes.c_int), ctypes.POINTER(ctypes.c_int32)]
        l.b200_array_devptr.argtypes = [vp, ctypes.c_uint64, ctypes.c_int, ctypes.POINTER(vp)]
        l.b200_program_load.argtypes = [vp, cp, ctypes.c_size_t, ctypes.POINTER(vp)]
        l.b200_program_free.argtypes = [vp]
        l.b200_program_free.restype = None
        l.b200_program_num_inputs.argtypes = [vp, ctypes.POINTER(ctypes.c_int)]
        l.b200_program_num_outputs.argtypes = [vp, ctypes.POINTER(ctypes.c_int)]
        l.b200_program_run.argtypes = [vp, u64p, ctypes.c_int, u64p, ctypes.c_int]
        l.b200_program_run_rows.argtypes = [vp, u64p, ctypes.c_int, ctypes.c_uint64, ctypes.c_int64, ctypes.c_int64]
        l.b200_program_run_rows2.argtypes = [vp, u64p, ctypes.c_int, ctypes.c_uint64, ctypes.c_int64, ctypes.c_int64, ctypes.c_int64, ctypes.c_int64]
        l.b200_group_unique_id.argtypes = [ctypes.c_char_p]
        l.b200_group_create.argtypes = [vp, ctypes.c_char_p, ctypes.c_int, ctypes.c_int, ctypes.c_double, ctypes.POINTER(vp)]
        l.b200_group_destroy.argtypes = [vp]
        l.b200_group_destroy.restype = None
        l.b200_group_all_gather.argtypes = [vp, ctypes.c_uint64, u64p]
        l.b200_group_all_reduce.argtypes = [vp, ctypes.c_uint64, ctypes.c_int]
        l.b200_group_halo_exchange.argtypes = [vp, ctypes.c_uint64, ctypes.c_int64, ctypes.c_int64, ctypes.c_int64, ctypes.c_int64,
                                               ctypes.c_int, ctypes.c_int, ctypes.c_int]
        l.b200_group_halo_wait.argtypes = [vp]
        l.b200_sync.argtypes = [vp]
        l.b200_stats.argtypes = [vp, i64p]
        l.b200_memory_stats.argtypes = [vp, i64p]
        l.b200_ctx_purge.argtypes = [vp]
        l.b200_ctx_stream.argtypes = [vp, ctypes.POINTER(vp)]
        l.b200_compile_check.argtypes = [cp, ctypes.c_size_t, ctypes.c_char_p, ctypes.c_size_t]
        l.b200_kernel_source.argtypes = [cp, ctypes.c_size_t, ctypes.c_int, ctypes.c_char_p, ctypes.c_size_t]
        l.b200_program_lowered.argtypes = [cp, ctypes.c_size_t, ctypes.c_char_p, ctypes.c_size_t]
        try:
            from . import _binding
        except ImportError as e:
            warnings.warn(f"the compiled binding is missing ({e}), so calls take longer: build it with `python -m accelerate_b200.build`",
                          RuntimeWarning, stacklevel=2)
            _binding = _CtypesCalls
        else:
            address = lambda f: ctypes.cast(f, vp).value  # noqa: E731
            _binding.setup(address(l.b200_array_wrap), address(l.b200_program_run), address(l.b200_array_info), address(l.b200_array_devptr),
                           address(l.b200_array_free), address(l.b200_last_error), B200Error, tuple(L.SCALARS))
        _lib, _fast = l, _binding
    return _lib


def _check(rc):
    if rc != 0:
        raise B200Error(rc, lib().b200_last_error().decode(errors="replace"))


def compile_check(text):
    """NVRTC-compile every kernel of ``text`` for sm_100a; needs no GPU."""
    log = ctypes.create_string_buffer(1 << 16)
    b = text.encode()
    rc = lib().b200_compile_check(b, len(b), log, len(log))
    if rc != 0:
        raise B200Error(rc, log.value.decode(errors="replace"))
    return log.value.decode()


def program_lowered(text):
    """The program text after the library's own rewriting (arrays of SIMD vectors regrouped at the boundary)."""
    buf = ctypes.create_string_buffer(len(text) * 4 + (1 << 16))
    b = text.encode()
    _check(lib().b200_program_lowered(b, len(b), buf, len(buf)))
    return buf.value.decode()


def kernel_source(text, node=0):
    buf = ctypes.create_string_buffer(1 << 20)
    b = text.encode()
    _check(lib().b200_kernel_source(b, len(b), node, buf, len(buf)))
    return buf.value.decode()


_LEAVES, _ELT_TEXT = {}, {}
_SCALAR_TEXT = {t: t.encode() for t in L.SCALARS}


def _leaf_types(elt):
    """Scalar types of an element type's leaves (remembered: asked for with every array)."""
    try:
        r = _LEAVES.get(elt)
        if r is None:
            r = _LEAVES[elt] = L.flatten_ty(elt)
        return r
    except TypeError:                    # a list in the place of a tuple
        return L.flatten_ty(elt)


def _elt_text(elt):
    try:
        r = _ELT_TEXT.get(elt)
        if r is None:
            r = _ELT_TEXT[elt] = L.ty_sx(elt).encode()
        return r
    except TypeError:
        return L.ty_sx(elt).encode()


class DeviceArray:
    """A device-resident array (struct-of-arrays) owned by a context.  Whoever made it and knows its element type and
    shape passes both; otherwise the library is asked, once."""

    def __init__(self, ctx, ident, elt=None, shape=None, leaf_types=None, ptrs=None):
        self.ctx, self.id, self._ptrs = ctx, ident, ptrs
        if ptrs is not None:
            self._since = ctx.adoptions
        if leaf_types is not None:
            self.shape, self.leaf_types = shape, leaf_types
        elif shape is not None and elt is not None:
            self.shape, self.leaf_types = shape, list(_leaf_types(elt))
        else:
            self.shape, self.leaf_types = _describe(ctx.h, ident)
        self.elt = elt if elt is not None else (self.leaf_types[0] if len(self.leaf_types) == 1 else tuple(self.leaf_types))

    def devptr(self, leaf=0):
        # (the pointers a run reported hold as long as no payload was adopted since: this may be a second handle of the
        # array that adopted it, and the library copies the payload when it is asked for the pointer)
        if self._ptrs is not None and 0 <= leaf < len(self._ptrs) and self._since is self.ctx.adoptions:
            return self._ptrs[leaf]
        return _pointer(self.ctx.h, self.id, leaf)

    def upload(self, leaves):
        for k, a in enumerate(leaves):
            a = np.ascontiguousarray(a)
            _check(lib().b200_array_upload(self.ctx.h, self.id, k, a.ctypes.data, a.nbytes))
        return self

    def adopt_host(self, leaves):
        """Lazy upload: the host arrays are copied when the array is first used on the device;
        they are kept alive by this object until then."""
        self._adopted = [np.ascontiguousarray(a) for a in leaves]
        try:
            for k, a in enumerate(self._adopted):
                _check(lib().b200_array_adopt_host(self.ctx.h, self.id, k, a.ctypes.data, a.nbytes))
        finally:
            self.ctx.adoptions = object()
        return self

    def download(self, out=None):
        """Host copy: an ndarray (scalar elements) or a tuple of ndarrays."""
        res = []
        for k, t in enumerate(self.leaf_types):
            a = out[k] if out is not None else np.empty(self.shape, dtype=L.NP_OF[t])
            _check(lib().b200_array_download(self.ctx.h, self.id, k, a.ctypes.data, a.nbytes))
            res.append(a)
        return res[0] if L.is_scalar(self.elt) else tuple(res)

    def download_async(self, out):
        """Start copying every leaf into the given (pinned) host arrays on the copy-out stream; the
        data is there after ``Context.sync()``.  The array may be freed at once."""
        for k in range(len(self.leaf_types)):
            a = out[k]
            _check(lib().b200_array_download_async(self.ctx.h, self.id, k, a.ctypes.data, a.nbytes))
        if getattr(self, "_keepalive", None) is not None:
            # a view over memory that another object owns: the library defers the release of an array
            # it is copying from, but cannot know that this view's memory belongs to a different one
            self.ctx._inflight.append(self)
        return out[0] if L.is_scalar(self.elt) else tuple(out)

    def free(self):
        if self.id is not None and self.ctx.handle:
            _fast.free(self.ctx.handle, self.id)
            self.id = self._ptrs = None

    def __del__(self):
        # (free() without its frame: every temporary array comes through here)
        try:
            if self.id is not None and self.ctx.handle:
                _fast.free(self.ctx.handle, self.id)
        except Exception:
            pass


class Context:
    """A backend handle: one GPU, one stream, a kernel cache."""

    def __init__(self, device=0):
        self.h = ctypes.c_void_p()
        _check(lib().b200_ctx_create(device, 0, ctypes.byref(self.h)))
        self.handle = self.h.value           # the same as a number; 0 once the context is closed
        self.device = device
        self._programs = {}
        self._inflight = []          # views with an asynchronous download under way (kept alive until sync)
        self._interned = {}          # host payloads registered in the memory table, by key
        self.adoptions = object()    # another one whenever a payload is adopted (DeviceArray.devptr)

    def close(self):
        if self.h:
            for p in self._programs.values():
                lib().b200_program_free(p)
            self._programs = {}
            self.handle = 0
            lib().b200_ctx_destroy(self.h)
            self.h = ctypes.c_void_p()

    # arrays ---------------------------------------------------------------
    def array(self, elt, shape):
        ident = ctypes.c_uint64()
        sh = (ctypes.c_int64 * max(1, len(shape)))(*shape)
        _check(lib().b200_array_new(self.h, _elt_text(elt), len(shape), sh, ctypes.byref(ident)))
        return DeviceArray(self, ident.value, elt, tuple(map(int, shape)))

    def from_host(self, a, elt=None):
        """Upload an ndarray, or a tuple of equal-shape ndarrays (array of tuples)."""
        leaves = [np.ascontiguousarray(x) for x in (a if isinstance(a, (tuple, list)) else [a])]
        leaves = [x.view(np.uint8) if x.dtype == np.bool_ else x for x in leaves]
        if elt is None:
            elt = tuple(L.TY_OF_NP[x.dtype] for x in leaves) if isinstance(a, (tuple, list)) else L.TY_OF_NP[leaves[0].dtype]
        return self.array(elt, leaves[0].shape).upload(leaves)

    def from_host_lazy(self, a, elt=None):
        """As ``from_host``, but the copy happens when the array is first used (``b200_array_adopt_host``)."""
        leaves = [np.ascontiguousarray(x) for x in (a if isinstance(a, (tuple, list)) else [a])]
        leaves = [x.view(np.uint8) if x.dtype == np.bool_ else x for x in leaves]
        if elt is None:
            elt = tuple(L.TY_OF_NP[x.dtype] for x in leaves) if isinstance(a, (tuple, list)) else L.TY_OF_NP[leaves[0].dtype]
        return self.array(elt, leaves[0].shape).adopt_host(leaves)

    def intern(self, key, a, elt=None):
        """The device copy of host array ``a`` under the caller's unique ``key`` (the memory table,
        ``b200_array_intern``): uploaded at most once however often it is asked for.  The caller
        guarantees that ``a`` is not modified while the key is registered."""
        leaves = [np.ascontiguousarray(x) for x in (a if isinstance(a, (tuple, list)) else [a])]
        leaves = [x.view(np.uint8) if x.dtype == np.bool_ else x for x in leaves]
        if elt is None:
            elt = tuple(L.TY_OF_NP[x.dtype] for x in leaves) if isinstance(a, (tuple, list)) else L.TY_OF_NP[leaves[0].dtype]
        shape = leaves[0].shape
        ident = ctypes.c_uint64()
        sh = (ctypes.c_int64 * max(1, len(shape)))(*shape)
        ptrs = (ctypes.c_void_p * len(leaves))(*[x.ctypes.data for x in leaves])
        _check(lib().b200_array_intern(self.h, key, L.ty_sx(elt).encode(), len(shape), sh, ptrs, ctypes.byref(ident)))
        d = DeviceArray(self, ident.value, elt)
        d._adopted = leaves
        self._interned.setdefault(key, leaves)      # the payload stays alive while the key is registered
        return d

    def forget(self, key):
        _check(lib().b200_array_forget(self.h, key))
        self._interned.pop(key, None)

    def wrap_scalars(self, elt, shape, ptr):
        """``wrap`` for a scalar element type and a tuple of ints as the shape."""
        return DeviceArray(self, _fast.wrap(self.handle, _SCALAR_TEXT[elt], shape, (ptr,)), elt, shape, [elt])

    def wrap(self, elt, shape, ptrs):
        """Adopt caller-owned device memory (one pointer per leaf: a number or a ``ctypes.c_void_p``)."""
        if len(ptrs) != len(_leaf_types(elt)):
            raise ValueError("one pointer per scalar leaf of the element type")
        shape = tuple(map(int, shape))
        return DeviceArray(self, _fast.wrap(self.handle, _elt_text(elt), shape, ptrs), elt, shape)

    # programs ---------------------------------------------------------------
    def load(self, text):
        p = self._programs.get(text)
        if p is None:
            p = ctypes.c_void_p()
            b = text.encode()
            _check(lib().b200_program_load(self.h, b, len(b), ctypes.byref(p)))
            self._programs[text] = p
        return p

    def execute(self, text, inputs, n_out):
        """Run program ``text`` on device arrays; returns device arrays."""
        p = self.load(text)
        return [DeviceArray(self, ident, None, shape, types, ptrs)
                for ident, shape, types, ptrs in _fast.execute(self.handle, p.value, [a.id for a in inputs], n_out)]

    def run_rows(self, text, inputs, out, row_lo, row_hi):
        """Rows [row_lo, row_hi) of a one-stencil-node program's result, into the existing array ``out``."""
        p = self.load(text)
        ins = (ctypes.c_uint64 * max(1, len(inputs)))(*[a.id for a in inputs])
        _check(lib().b200_program_run_rows(p, ins, len(inputs), out.id, row_lo, row_hi))

    def run_rows2(self, text, inputs, out, row_lo, row_hi, row_lo2, row_hi2):
        """The same for two ranges of rows (the second above the first) in one launch."""
        p = self.load(text)
        ins = (ctypes.c_uint64 * max(1, len(inputs)))(*[a.id for a in inputs])
        _check(lib().b200_program_run_rows2(p, ins, len(inputs), out.id, row_lo, row_hi, row_lo2, row_hi2))

    def sync(self):
        try:
            _check(lib().b200_sync(self.h))
        finally:
            self._inflight = []

    def stats(self):
        out = (ctypes.c_int64 * 8)()
        _check(lib().b200_stats(self.h, out))
        keys = ["launches", "h2d_bytes", "d2h_bytes", "compiled", "mem_hits", "disk_hits", "allocated_bytes", "runs"]
        return dict(zip(keys, [int(v) for v in out]))

    def memory_stats(self):
        """Live bytes, and the freed buffers kept for reuse (the nursery): bytes, count, allocations served."""
        out = (ctypes.c_int64 * 5)()
        _check(lib().b200_memory_stats(self.h, out))
        return dict(zip(["live_bytes", "nursery_bytes", "nursery_blocks", "nursery_hits", "inplace_permutes"], [int(v) for v in out]))

    def purge(self):
        """Hand the kept buffers back to the driver."""
        _check(lib().b200_ctx_purge(self.h))

    def stream(self):
        s = ctypes.c_void_p()
        _check(lib().b200_ctx_stream(self.h, ctypes.byref(s)))
        return s.value or 0


class Group:
    """This context's GPU as one rank of a group of GPUs (``b200_group_*``): the exchange steps of
    the sharded skeletons, enqueued on the context's streams."""

    OPS = {"add": 0, "min": 1, "max": 2, "mul": 3}

    @staticmethod
    def unique_id():
        buf = ctypes.create_string_buffer(128)
        _check(lib().b200_group_unique_id(buf))
        return buf.raw

    def __init__(self, ctx, unique_id, rank, world, deadline_s=60.0):
        self.ctx, self.rank, self.world = ctx, rank, world
        self.h = ctypes.c_void_p()
        _check(lib().b200_group_create(ctx.h, unique_id, rank, world, deadline_s, ctypes.byref(self.h)))

    def close(self):
        if self.h:
            lib().b200_group_destroy(self.h)
            self.h = ctypes.c_void_p()

    def all_gather(self, a):
        out = ctypes.c_uint64()
        _check(lib().b200_group_all_gather(self.h, a.id, ctypes.byref(out)))
        return DeviceArray(self.ctx, out.value, a.elt)

    def all_reduce(self, a, op):
        _check(lib().b200_group_all_reduce(self.h, a.id, self.OPS[op]))

    def halo_exchange(self, a, top, rows, bot, radius, up, down, overlap=False):
        _check(lib().b200_group_halo_exchange(self.h, a.id, top, rows, bot, radius, -1 if up is None else up, -1 if down is None else down,
                                              1 if overlap else 0))

    def halo_wait(self):
        _check(lib().b200_group_halo_wait(self.h))


_default = None


def default_context():
    global _default
    if _default is None:
        dev = int(os.environ.get("LOCAL_RANK", "0")) if "ACCELERATE_B200_DEVICE" not in os.environ else int(os.environ["ACCELERATE_B200_DEVICE"])
        _default = Context(dev)
    return _default


def run_program(prog, host_inputs, ctx=None):
    """Upload, execute, download.  ``host_inputs``: list of ``(shape, [leaves])``."""
    ctx = ctx or default_context()
    ins = []
    for n, (shape, leaves) in zip(prog.inputs, host_inputs):
        # (an array of SIMD vectors is, to the library, an array of the component type with one more dimension)
        ins.append(ctx.array(L.vec_parts(n.elt)[1] if L.vec_parts(n.elt) else n.elt, shape).upload(leaves))
    outs = ctx.execute(prog.text, ins, len(prog.outputs))
    res = []
    for o, (_, elt) in zip(outs, prog.outputs):
        o.elt = elt
        res.append(o.download())
    return res


def run(acc, ctx=None, embed=False):
    """``run :: Arrays a => Acc a -> a`` (Interpreter.hs:93).  With ``embed`` the arrays given to
    ``use`` travel inside the program as ``Use`` nodes, as they do in ``run (... (use xs))``;
    otherwise they are bound as program inputs (what ``runN`` does with its arguments)."""
    single = not isinstance(acc, (list, tuple))
    prog = L.build_program(acc, embed=embed)
    res = run_program(prog, [n.data for n in prog.inputs], ctx)
    return res[0] if single else res


def runN(f, ctx=None):
    """``runN`` (Interpreter.hs:110-126): the program is built and loaded on the
    first call for given argument types and reused afterwards."""
    cache = {}

    def go(*arrays):
        arrays = [a if isinstance(a, (tuple, list)) else np.ascontiguousarray(a) for a in arrays]
        sig = tuple((tuple(x.dtype.str for x in a), a[0].ndim) if isinstance(a, (tuple, list)) else (a.dtype.str, a.ndim) for a in arrays)
        ent = cache.get(sig)
        if ent is None:
            L.reset_names()
            params = []
            for a in arrays:
                if isinstance(a, (tuple, list)):
                    params.append(L.param(a[0].ndim, tuple(L.TY_OF_NP[x.dtype] for x in a)))
                else:
                    params.append(L.param(a.ndim, L.TY_OF_NP[a.dtype]))
            res = f(*params)
            single = not isinstance(res, (list, tuple))
            prog = L.build_program(res)
            order = [params.index(next(q for q in params if q.node is n)) for n in prog.inputs]
            ent = cache[sig] = (prog, order, single)
        prog, order, single = ent
        host = []
        for k in order:
            a = arrays[k]
            leaves = list(a) if isinstance(a, (tuple, list)) else [a]
            host.append((tuple(leaves[0].shape), leaves))
        out = run_program(prog, host, ctx)
        return out[0] if single else out
    return go
