"""tadma_b200: B200 (sm_100a) kernels behind TADMA's Tensor API, Python binding.

The product is the C-ABI library ``libtadma_b200.so`` built in-tree from
``tadma_b200/csrc`` (declared in ``include/tadma_b200.h``).  This module loads
it with ctypes and offers thin helpers that build descriptors from torch CUDA
tensors.  torch is used for device memory and streams only; every op runs the
library's own kernels.  There is no CPU fallback: if the library is missing the
import raises.
"""
from __future__ import annotations

import ctypes
import functools
import os

from .abi import (  # noqa: F401  (re-exported)
    MAX_INPUTS, MAX_INSTR, MAX_RANK, ROWPROG_MAX_STAGES, SRC_IMM, SRC_NONE, BINARY_OPS, TRANSCENDENTAL, UNARY_OPS,
    Compute, Dist, DType, LNMode, Op, Reduce, Status, TadmaInstr, TadmaRowProgram, TadmaRowStage, TadmaTensor,
    instr, make_tensor, program,
)

LIB_PATH = os.path.join(os.path.dirname(os.path.abspath(__file__)), "libtadma_b200.so")

_lib = None

EXPORTS = (
    "tadma_b200_eltwise", "tadma_b200_reduce", "tadma_b200_softmax", "tadma_b200_layer_norm",
    "tadma_b200_rms_norm", "tadma_b200_gather", "tadma_b200_fill", "tadma_b200_last_error",
    "tadma_b200_version", "tadma_b200_error_flags", "tadma_b200_dtype_size", "tadma_b200_reduce_noalloc",
    "tadma_b200_reduce_chain", "tadma_b200_reduce_chain_post", "tadma_b200_row_program",
    "tadma_b200_block_tables", "tadma_b200_kv4_append", "tadma_b200_kv4_read", "tadma_b200_kv4_attention",
    "tadma_b200_kv4_attention_workspace", "tadma_b200_kv4_attention_uses", "tadma_b200_matvec_q4", "tadma_b200_adjust_logits",
)


class TadmaError(RuntimeError):
    """A C-ABI call returned a non-zero status (code + the library's message)."""

    def __init__(self, code: int, msg: str):
        super().__init__(f"{Status(code).name}: {msg}")
        self.code = code


def lib() -> ctypes.CDLL:
    """Load libtadma_b200.so (raises if it has not been built)."""
    global _lib
    if _lib is not None:
        return _lib
    if not os.path.exists(LIB_PATH):
        raise ImportError(f"{LIB_PATH} is missing: build it with `python -c 'import __graft_entry__ as g; g.build()'`")
    L = ctypes.CDLL(LIB_PATH)
    P = ctypes.POINTER
    T, I = TadmaTensor, TadmaInstr
    c_int, c_void, c_double = ctypes.c_int32, ctypes.c_void_p, ctypes.c_double
    L.tadma_b200_eltwise.argtypes = [P(T), P(T), c_int, P(I), c_int, c_int, c_void]
    L.tadma_b200_reduce.argtypes = [c_int, P(T), c_int, c_int, P(T), c_void]
    L.tadma_b200_reduce_noalloc.argtypes = [c_int, P(T), c_int, c_int, P(T), c_void]
    L.tadma_b200_reduce_chain.argtypes = [c_int, P(T), c_int, P(I), c_int, c_int, c_int, P(T), c_void]
    L.tadma_b200_reduce_chain_post.argtypes = [c_int, P(T), c_int, P(I), c_int, P(I), c_int, c_int, c_int, P(T),
                                               c_void]
    L.tadma_b200_row_program.argtypes = [P(TadmaRowProgram), c_void]
    L.tadma_b200_softmax.argtypes = [P(T), c_int, P(T), c_void]
    L.tadma_b200_layer_norm.argtypes = [P(T), c_int, P(T), P(T), c_double, c_int, P(T), c_void]
    L.tadma_b200_rms_norm.argtypes = [P(T), c_int, c_double, P(T), c_void]
    L.tadma_b200_gather.argtypes = [P(T), c_int, P(T), P(T), P(T), c_void]
    L.tadma_b200_fill.argtypes = [P(T), c_int, c_double, c_double, ctypes.c_uint64, ctypes.c_uint64,
                                  ctypes.c_int64, c_void]
    L.tadma_b200_block_tables.argtypes = [P(T), P(T), P(T), P(T), c_int, P(T), P(T), P(T), P(T), P(T), c_void]
    L.tadma_b200_kv4_append.argtypes = [P(T)] * 7 + [c_void]
    L.tadma_b200_kv4_read.argtypes = [P(T)] * 7 + [c_void]
    L.tadma_b200_kv4_attention.argtypes = [P(T)] * 7 + [c_double, P(T), c_void, ctypes.c_int64, c_void]
    L.tadma_b200_kv4_attention_workspace.argtypes = [ctypes.c_int64] * 4
    L.tadma_b200_kv4_attention_uses.argtypes = [P(T)] * 4
    L.tadma_b200_matvec_q4.argtypes = [P(T)] * 6 + [c_void]
    L.tadma_b200_adjust_logits.argtypes = [P(T)] * 11 + [c_void]
    L.tadma_b200_error_flags.argtypes = [P(ctypes.c_uint32), c_int]
    L.tadma_b200_dtype_size.argtypes = [c_int]
    for name in EXPORTS:
        getattr(L, name).restype = ctypes.c_int32
    L.tadma_b200_kv4_attention_workspace.restype = ctypes.c_int64
    L.tadma_b200_kv4_attention_uses.restype = ctypes.c_int64
    L.tadma_b200_last_error.restype = ctypes.c_char_p
    L.tadma_b200_version.restype = ctypes.c_char_p
    L.tadma_b200_last_error.argtypes = []
    L.tadma_b200_version.argtypes = []
    _lib = L
    return L


def check(rc: int) -> None:
    if rc != 0:
        raise TadmaError(rc, lib().tadma_b200_last_error().decode())


def version() -> str:
    return lib().tadma_b200_version().decode()


# ---------------------------------------------------------------- torch glue --

def _torch():
    import torch
    return torch


_TORCH_DT = None


def torch_dtype_code(t) -> DType:
    global _TORCH_DT
    torch = _torch()
    if _TORCH_DT is None:
        _TORCH_DT = {torch.float32: DType.F32, torch.float16: DType.F16, torch.bfloat16: DType.BF16,
                     torch.float64: DType.F64, torch.int64: DType.I64, torch.int32: DType.I32,
                     torch.uint8: DType.U8, torch.bool: DType.BOOL, torch.int8: DType.I8}
    return _TORCH_DT[t.dtype]


def desc(t, shape=None, strides=None) -> TadmaTensor:
    """Descriptor of a torch tensor (optionally re-viewed with shape/strides in elements)."""
    return make_tensor(t.data_ptr() if t.numel() else None, torch_dtype_code(t),
                       list(t.shape) if shape is None else shape,
                       list(t.stride()) if strides is None else strides)


def none_tensor() -> TadmaTensor:
    return TadmaTensor()


def _stream(stream):
    if stream is None:
        return ctypes.c_void_p(_torch().cuda.current_stream().cuda_stream)
    if isinstance(stream, int):
        return ctypes.c_void_p(stream)
    return ctypes.c_void_p(stream.cuda_stream)


class Prepared:
    """A C-ABI call with its ctypes arguments built once (descriptors, program,
    stream): calling it costs one foreign call, for launch-bound loops.  The
    stream is fixed when the call is prepared (the current torch stream when
    none is given); prepare on the capture stream to record into a CUDA graph."""

    def __init__(self, fn, args, keep=()):
        self._fn, self._args, self._keep = fn, args, keep

    def __call__(self) -> None:
        rc = self._fn(*self._args)
        if rc != 0:
            check(rc)


def _d(t):
    return t if isinstance(t, TadmaTensor) else desc(t)


def prepare_eltwise(out, ins, prog, compute=Compute.AUTO, stream=None) -> Prepared:
    o = _d(out)
    arr = (TadmaTensor * max(1, len(ins)))(*[_d(x) for x in ins])
    p, n = program(prog)
    return Prepared(lib().tadma_b200_eltwise, (ctypes.byref(o), arr, len(ins), p, n, int(compute), _stream(stream)),
                    (o, arr, p))


def prepare_reduce(op, x, axis, out, pre_op=Op.COPY, stream=None) -> Prepared:
    i, o = _d(x), _d(out)
    return Prepared(lib().tadma_b200_reduce, (int(op), ctypes.byref(i), int(axis), int(pre_op), ctypes.byref(o),
                                              _stream(stream)), (i, o))


def prepare_reduce_chain(op, ins, prog, axis, out, compute=Compute.AUTO, stream=None, post=None) -> Prepared:
    """out = reduce `op` over `axis` of chain(ins...) in one kernel (tadma_b200_reduce_chain); with `post`
    (instructions with immediate operands), out = post(reduce(...)) (tadma_b200_reduce_chain_post)."""
    arr = (TadmaTensor * max(1, len(ins)))(*[_d(x) for x in ins])
    p, n = program(prog)
    o = _d(out)
    if post:
        q, m = program(post)
        return Prepared(lib().tadma_b200_reduce_chain_post, (int(op), arr, len(ins), p, n, q, m, int(compute),
                                                             int(axis), ctypes.byref(o), _stream(stream)),
                        (arr, p, q, o))
    return Prepared(lib().tadma_b200_reduce_chain, (int(op), arr, len(ins), p, n, int(compute), int(axis),
                                                    ctypes.byref(o), _stream(stream)), (arr, p, o))


def prepare_softmax(x, axis, out, stream=None) -> Prepared:
    i, o = _d(x), _d(out)
    return Prepared(lib().tadma_b200_softmax, (ctypes.byref(i), int(axis), ctypes.byref(o), _stream(stream)), (i, o))


def prepare_layer_norm(x, axis, gamma, beta, eps, out, mode=LNMode.ONNX, stream=None) -> Prepared:
    i, o = _d(x), _d(out)
    g = none_tensor() if gamma is None else _d(gamma)
    b = none_tensor() if beta is None else _d(beta)
    return Prepared(lib().tadma_b200_layer_norm, (ctypes.byref(i), int(axis), ctypes.byref(g), ctypes.byref(b),
                                                  float(eps), int(mode), ctypes.byref(o), _stream(stream)), (i, o, g, b))


def prepare_rms_norm(x, axis, eps, out, stream=None) -> Prepared:
    i, o = _d(x), _d(out)
    return Prepared(lib().tadma_b200_rms_norm, (ctypes.byref(i), int(axis), float(eps), ctypes.byref(o),
                                                _stream(stream)), (i, o))


def prepare_gather(table, axis, ids, out, add=None, stream=None) -> Prepared:
    t, i, o = _d(table), _d(ids), _d(out)
    a = none_tensor() if add is None else _d(add)
    return Prepared(lib().tadma_b200_gather, (ctypes.byref(t), int(axis), ctypes.byref(i), ctypes.byref(a),
                                              ctypes.byref(o), _stream(stream)), (t, i, o, a))


def prepare_fill(out, dist, p0, p1, seed, stream_id, offset=0, stream=None) -> Prepared:
    o = _d(out)
    return Prepared(lib().tadma_b200_fill, (ctypes.byref(o), int(dist), float(p0), float(p1), int(seed),
                                            int(stream_id), int(offset), _stream(stream)), (o,))


def eltwise(out, ins, prog, compute=Compute.AUTO, stream=None) -> None:
    """out = chain(ins...) (tadma_b200_eltwise).  `out`/`ins` are torch tensors or descriptors."""
    prepare_eltwise(out, ins, prog, compute, stream)()


def reduce(op, x, axis, out, pre_op=Op.COPY, stream=None) -> None:
    prepare_reduce(op, x, axis, out, pre_op, stream)()


def reduce_chain(op, ins, prog, axis, out, compute=Compute.AUTO, stream=None, post=None) -> None:
    prepare_reduce_chain(op, ins, prog, axis, out, compute, stream, post)()


def row_program(rows, cols, ins, stages, prog, out, acc=0, compute=Compute.F32, stream=None) -> None:
    """tadma_b200_row_program.  ins: descriptors (or torch tensors) viewed as
    {rows, cols}; stages: (op, chain, post, out, acc) tuples, out a {rows}
    descriptor or tensor; prog: the final chain; out: {rows, cols}."""
    rp = TadmaRowProgram()
    rp.rows, rp.cols = int(rows), int(cols)
    rp.n_ins = len(ins)
    for k, t in enumerate(ins):
        rp.ins[k] = _d(t)
    rp.n_stages = len(stages)
    for s, (op, chain, post, sout, sacc) in enumerate(stages):
        st = rp.stages[s]
        st.op, st.n_instr, st.n_post, st.acc = int(op), len(chain), len(post), int(sacc)
        for i, I in enumerate(chain):
            st.prog[i] = I
        for i, I in enumerate(post):
            st.post[i] = I
        st.out = _d(sout)
    rp.n_instr = len(prog)
    for i, I in enumerate(prog):
        rp.prog[i] = I
    rp.acc = int(acc)
    rp.compute = int(compute)
    rp.out = _d(out)
    check(lib().tadma_b200_row_program(ctypes.byref(rp), _stream(stream)))


def softmax(x, axis, out, stream=None) -> None:
    prepare_softmax(x, axis, out, stream)()


def layer_norm(x, axis, gamma, beta, eps, out, mode=LNMode.ONNX, stream=None) -> None:
    prepare_layer_norm(x, axis, gamma, beta, eps, out, mode, stream)()


def rms_norm(x, axis, eps, out, stream=None) -> None:
    prepare_rms_norm(x, axis, eps, out, stream)()


def gather(table, axis, ids, out, add=None, stream=None) -> None:
    prepare_gather(table, axis, ids, out, add, stream)()


def fill(out, dist, p0, p1, seed, stream_id, offset=0, stream=None) -> None:
    prepare_fill(out, dist, p0, p1, seed, stream_id, offset, stream)()


# ------------------------------------------------------------- token step --
# block_tables, kv4_append, kv4_read, kv4_attention, matvec_q4, adjust_logits:
# see include/tadma_b200.h for shapes, types and what each computes.

def prepare_block_tables(held, added, free_list, num_free, page_size, table, slots, starts, lens, left,
                         stream=None) -> Prepared:
    d = [_d(t) for t in (held, added, free_list, num_free, table, slots, starts, lens, left)]
    r = [ctypes.byref(t) for t in d]
    return Prepared(lib().tadma_b200_block_tables, (*r[:4], int(page_size), *r[4:], _stream(stream)), d)


def prepare_kv4_append(k, v, slots, k_codes, k_params, v_codes, v_params, stream=None) -> Prepared:
    d = [_d(t) for t in (k, v, slots, k_codes, k_params, v_codes, v_params)]
    return Prepared(lib().tadma_b200_kv4_append, (*map(ctypes.byref, d), _stream(stream)), d)


def prepare_kv4_read(k_codes, k_params, v_codes, v_params, slots, k_out, v_out, stream=None) -> Prepared:
    d = [_d(t) for t in (k_codes, k_params, v_codes, v_params, slots, k_out, v_out)]
    return Prepared(lib().tadma_b200_kv4_read, (*map(ctypes.byref, d), _stream(stream)), d)


def prepare_kv4_attention(q, k_codes, k_params, v_codes, v_params, table, lens, scale, out, workspace=None,
                          stream=None) -> Prepared:
    """`workspace`: a uint8 CUDA tensor of kv4_attention_workspace(...) bytes that no overlapping call uses.  Without
    one, a call on torch's current stream takes it from torch's allocator, a call on another stream allocates it in
    that stream's order."""
    if workspace is None and stream is None:
        workspace = _attention_workspace(q, k_codes)
    d = [_d(t) for t in (q, k_codes, k_params, v_codes, v_params, table, lens, out)]
    r = [ctypes.byref(t) for t in d]
    ws, n = (None, 0) if workspace is None else (workspace.data_ptr(), workspace.numel() * workspace.element_size())
    return Prepared(lib().tadma_b200_kv4_attention, (*r[:7], float(scale), r[7], ws, n, _stream(stream)),
                    (d, workspace))


@functools.lru_cache(maxsize=None)
def kv4_attention_workspace(requests, heads, kv_heads, dim) -> int:
    """Bytes of workspace of a call with those sizes."""
    return lib().tadma_b200_kv4_attention_workspace(int(requests), int(heads), int(kv_heads), int(dim))


def _bytes_on_gpu(n):
    torch = _torch()
    return torch.empty(n, dtype=torch.uint8, device="cuda")


def _attention_workspace(q, k_codes):
    """The workspace of a call on torch's current stream, from torch's allocator; None where the call will refuse."""
    dims, cache = (t.dims if isinstance(t, TadmaTensor) else t.shape for t in (q, k_codes))
    if len(dims) < 3 or len(cache) < 2:
        return None
    n = kv4_attention_workspace(dims[0], dims[1], cache[1], dims[2])
    return _bytes_on_gpu(n) if n else None


def prepare_matvec_q4(x, codes, scales, out, zeros=None, bias=None, stream=None) -> Prepared:
    d = [none_tensor() if t is None else _d(t) for t in (x, codes, scales, zeros, bias, out)]
    return Prepared(lib().tadma_b200_matvec_q4, (*map(ctypes.byref, d), _stream(stream)), d)


def prepare_adjust_logits(logits, ids, prompt_lens, lens, out, repetition=None, presence=None, frequency=None,
                          bias_ids=None, bias=None, mask=None, stream=None) -> Prepared:
    d = [none_tensor() if t is None else _d(t) for t in (logits, ids, prompt_lens, lens, repetition, presence,
                                                         frequency, bias_ids, bias, mask, out)]
    return Prepared(lib().tadma_b200_adjust_logits, (*map(ctypes.byref, d), _stream(stream)), d)


# One-shot calls of a token step are bound by the host, so they go through the
# extension module _pycall (csrc/pycall.c) instead of ctypes.

def _operand(t):
    if t is None or isinstance(t, TadmaTensor):
        return t
    if not hasattr(t, "data_ptr"):
        raise TypeError("expected a tensor or a tensor descriptor")
    d = TadmaTensor(data=t.data_ptr(), dtype=int(_TORCH_DT.get(t.dtype, -1)), rank=t.dim())  # the call refuses what it does not know
    for i, (n, s) in enumerate(zip(t.shape[:MAX_RANK], t.stride())):
        d.dims[i], d.strides[i] = n, s
    return d


class _CtypesCalls:
    """What _pycall offers, through ctypes (10 to 45 us more host time a call): for a Python whose headers the build did
    not have."""

    @staticmethod
    def _refs(tensors):
        return [None if t is None else ctypes.byref(t) for t in map(_operand, tensors)]

    def _call(self, name, tensors, stream):
        return getattr(lib(), "tadma_b200_" + name)(*self._refs(tensors), stream)

    def block_tables(self, *a):
        r = self._refs(a[:9])
        page = a[9] if 0 <= a[9] <= 0x7fffffff else 0
        return lib().tadma_b200_block_tables(*r[:4], page, *r[4:], a[10])

    def kv4_append(self, *a):
        return self._call("kv4_append", a[:7], a[7])

    def kv4_read(self, *a):
        return self._call("kv4_read", a[:7], a[7])

    def kv4_attention(self, *a):
        r = self._refs(a[:8])
        scale, ws, n, stream, alloc = a[8:]
        made = None
        if not ws and alloc is not None:
            n = lib().tadma_b200_kv4_attention_uses(r[0], r[1], r[2], r[5])
            if n > 0:
                made = alloc(n)
                ws = made.data_ptr()
        return lib().tadma_b200_kv4_attention(*r[:7], scale, r[7], ws, n, stream)

    def matvec_q4(self, *a):
        return self._call("matvec_q4", a[:6], a[6])

    def adjust_logits(self, *a):
        return self._call("adjust_logits", a[:11], a[11])


_calls = None        # the module (or what stands in for it), once loaded
_stream_now = None   # address of torch's current stream


def _load_steps():
    global _calls, _stream_now
    lib()  # its error where the library has not been built; and the module finds it loaded
    torch = _torch()
    torch_dtype_code(torch.empty(0))
    try:
        from . import _pycall as calls
        calls.set_dtypes({t: int(c) for t, c in _TORCH_DT.items()})
    except ImportError:
        calls = _CtypesCalls()
    raw, device = getattr(torch._C, "_cuda_getCurrentRawStream", None), torch.cuda.current_device
    if raw is None:
        _stream_now = lambda: torch.cuda.current_stream().cuda_stream  # noqa: E731
    else:
        _stream_now = lambda: raw(device())  # noqa: E731  (without the object, which takes 3 us)
    _calls = calls
    return _calls


def _raw_stream(stream):
    return stream if isinstance(stream, int) else stream.cuda_stream


def block_tables(held, added, free_list, num_free, page_size, table, slots, starts, lens, left, stream=None) -> None:
    c = _calls or _load_steps()
    rc = c.block_tables(held, added, free_list, num_free, table, slots, starts, lens, left, page_size,
                        _stream_now() if stream is None else _raw_stream(stream))
    if rc:
        check(rc)


def kv4_append(k, v, slots, k_codes, k_params, v_codes, v_params, stream=None) -> None:
    c = _calls or _load_steps()
    rc = c.kv4_append(k, v, slots, k_codes, k_params, v_codes, v_params,
                      _stream_now() if stream is None else _raw_stream(stream))
    if rc:
        check(rc)


def kv4_read(k_codes, k_params, v_codes, v_params, slots, k_out, v_out, stream=None) -> None:
    c = _calls or _load_steps()
    rc = c.kv4_read(k_codes, k_params, v_codes, v_params, slots, k_out, v_out,
                    _stream_now() if stream is None else _raw_stream(stream))
    if rc:
        check(rc)


def kv4_attention(q, k_codes, k_params, v_codes, v_params, table, lens, scale, out, workspace=None,
                  stream=None) -> None:
    """`workspace` as in prepare_kv4_attention."""
    c = _calls or _load_steps()
    ws, n = (0, 0) if workspace is None else (workspace.data_ptr(), workspace.nbytes)
    rc = c.kv4_attention(q, k_codes, k_params, v_codes, v_params, table, lens, out, scale, ws, n,
                         _stream_now() if stream is None else _raw_stream(stream),
                         _bytes_on_gpu if stream is None else None)
    if rc:
        check(rc)


def matvec_q4(x, codes, scales, out, zeros=None, bias=None, stream=None) -> None:
    c = _calls or _load_steps()
    rc = c.matvec_q4(x, codes, scales, zeros, bias, out, _stream_now() if stream is None else _raw_stream(stream))
    if rc:
        check(rc)


def adjust_logits(logits, ids, prompt_lens, lens, out, repetition=None, presence=None, frequency=None, bias_ids=None,
                  bias=None, mask=None, stream=None) -> None:
    c = _calls or _load_steps()
    rc = c.adjust_logits(logits, ids, prompt_lens, lens, repetition, presence, frequency, bias_ids, bias, mask, out,
                         _stream_now() if stream is None else _raw_stream(stream))
    if rc:
        check(rc)


def error_flags(clear: bool = True) -> int:
    w = ctypes.c_uint32(0)
    check(lib().tadma_b200_error_flags(ctypes.byref(w), 1 if clear else 0))
    return int(w.value)
