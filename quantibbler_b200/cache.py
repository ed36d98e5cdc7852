"""Key/value caches on the device in float32, bfloat16 or INT8 (codes with a float32 scale per token and kv
head), and the attention over them: of a step (one query per sequence), of a prompt's portion, and both behind
a prefix that all sequences share.

A ``KvCache`` names torch tensors; every method is C-ABI calls (``qk_cache_*``) that only launch kernels, so
that a step can be captured in a CUDA graph.  Work runs on the context's stream and is ordered with torch's
current stream on both sides.  A captured call has a workspace of its graph's; eager calls share the context's.
"""

from __future__ import annotations

import contextlib
import ctypes
import threading

from . import _lib
from ._lib import QK_BF16, QK_F32, QK_I8, KernelError, check
from .gpu import GpuContext

DTYPES = ("float32", "bfloat16", "int8")
_TAGS = {"float32": QK_F32, "bfloat16": QK_BF16, "int8": QK_I8}


class KvCacheStruct(ctypes.Structure):
    """qk_kv_cache."""
    _fields_ = [("dtype", ctypes.c_int32), ("k", ctypes.c_void_p), ("v", ctypes.c_void_p),
                ("k_scale", ctypes.c_void_p), ("v_scale", ctypes.c_void_p), ("n_seq", ctypes.c_size_t),
                ("n_kv_heads", ctypes.c_size_t), ("rows", ctypes.c_size_t), ("head_dim", ctypes.c_size_t)]


def _stream_of(torch, handle, device):
    """The stream ``handle`` as torch knows it."""
    return torch.cuda.ExternalStream(handle, device=device) if handle > 2 else torch.cuda.default_stream(device)


@contextlib.contextmanager
def _joined(torch, handle, current):
    """Orders the context's stream ``handle`` behind torch's ``current`` stream, and that behind it."""
    stream = _stream_of(torch, handle, current.device)
    stream.wait_stream(current)
    try:
        yield
    finally:
        current.wait_stream(stream)


_alone = contextlib.nullcontext()
_growing = threading.Lock()


def _raw_stream(torch):
    """Device index -> handle of torch's current stream (a tenth of the cost of the stream object)."""
    return getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
        lambda index: torch.cuda.current_stream(index).cuda_stream)


def ordered(ctx: GpuContext, device):
    """A context manager around calls on ``ctx`` whose tensors belong to torch's current stream."""
    import torch
    handle = ctx.stream_handle
    # (the legacy default stream is 0 to torch, 1 to the context)
    if handle == (_raw_stream(torch)(device.index) or 1):
        return _alone
    return _joined(torch, handle, torch.cuda.current_stream(device))


def workspace(ctx: GpuContext, size: int, device):
    """Device memory of ``size`` bytes for one call on ``ctx``: the context's own for its stream, grown and kept (calls
    follow one another there), but inside a stream capture a tensor of the graph's."""
    import torch
    if not size:
        return None
    if torch.cuda.is_current_stream_capturing():
        return torch.empty(size, dtype=torch.uint8, device=device)
    kept = ctx.workspaces.setdefault(ctx.stream_handle, [])    # (the ones outgrown stay: work in flight may use them)
    if not kept or kept[-1].numel() < size:
        with _growing:
            if not kept or kept[-1].numel() < size:
                # (of that stream's own memory: another thread's call may use it before this one has ordered the streams)
                with torch.cuda.stream(_stream_of(torch, ctx.stream_handle, device)):
                    kept.append(torch.empty(max(size, 1 << 20, 2 * kept[-1].numel() if kept else 0), dtype=torch.uint8,
                                            device=device))
    return kept[-1]


def check_tensor(what: str, t, dtype, device, shape=None) -> None:
    if t.dtype != dtype:
        raise KernelError(f"{what} must be {str(dtype).replace('torch.', '')}, got {str(t.dtype).replace('torch.', '')}")
    if t.device != device:
        raise KernelError(f"{what} is on {t.device}, not on the cache's device {device}")
    if shape is not None and tuple(t.shape) != tuple(shape):
        raise KernelError(f"{what} must have the shape {tuple(shape)}, got {tuple(t.shape)}")


class KvCache:
    """Rows of keys and values, ``[slots, kv heads, rows, head_dim]``.

    ``k`` and ``v`` are contiguous float32, bfloat16 or int8 tensors; int8 caches come with ``k_scale`` and
    ``v_scale`` ``[slots, kv heads, rows]`` (float32).  Row r of a slot holds the position
    ``first_position + r`` of its sequence (``first_position`` > 0: the rows behind a shared prefix).

    Attention over bfloat16 and int8 rows of head_dim 64 and 128 runs on the tensor cores where k, v and q lie on
    16-byte boundaries; other caches, and a q off them, take a plain kernel that is a hundred times slower."""

    def __init__(self, ctx: GpuContext, k, v, k_scale=None, v_scale=None, first_position: int = 0):
        import torch
        self._torch, self._f32, self._i32, self.ctx = torch, torch.float32, torch.int32, ctx
        names = {torch.float32: "float32", torch.bfloat16: "bfloat16", torch.int8: "int8"}
        if k.dtype not in names:
            raise KernelError(f"a cache holds float32, bfloat16 or int8, got {str(k.dtype).replace('torch.', '')}")
        self.dtype = names[k.dtype]
        if k.dim() != 4:
            raise KernelError(f"k must be [slots, kv heads, rows, head_dim], got {tuple(k.shape)}")
        if k.device.type != "cuda":
            raise KernelError(f"a cache lives on a CUDA device, got {k.device}")
        if k.device.index != ctx.device_index:
            raise KernelError(f"the cache is on {k.device}, its context on cuda:{ctx.device_index}")
        self.device = k.device
        check_tensor("v", v, k.dtype, k.device, k.shape)
        if (self.dtype == "int8") != (k_scale is not None) or (k_scale is None) != (v_scale is None):
            raise KernelError("an int8 cache comes with k_scale and v_scale, others without")
        for what, t in (("k", k), ("v", v), ("k_scale", k_scale), ("v_scale", v_scale)):
            if t is None:
                continue
            if what.endswith("scale"):
                check_tensor(what, t, torch.float32, k.device, k.shape[:3])
            if not t.is_contiguous():
                raise KernelError(f"{what} must be contiguous")
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        self._like = {name: torch.empty(0, dtype=getattr(torch, name), device=k.device) for name in ("float32", "bfloat16")}
        self.n_seq, self.n_kv_heads, self.rows, self.head_dim = (int(n) for n in k.shape)
        self.first_position = int(first_position)
        ptr = lambda t: None if t is None else t.data_ptr()  # noqa: E731
        self._c = KvCacheStruct(_TAGS[self.dtype], ptr(k), ptr(v), ptr(k_scale), ptr(v_scale), self.n_seq,
                                self.n_kv_heads, self.rows, self.head_dim)
        self._ref = ctypes.byref(self._c)
        check(_lib.lib().qk_cache_check(ctx.handle, self._ref))

    @classmethod
    def empty(cls, ctx: GpuContext, n_seq: int, n_kv_heads: int, rows: int, head_dim: int, dtype: str = "int8",
              first_position: int = 0) -> "KvCache":
        """A new cache of zeros on the context's device."""
        import torch
        if dtype not in DTYPES:
            raise KernelError(f"cache dtype must be one of {', '.join(DTYPES)}, got {dtype!r}")
        dev = torch.device("cuda", ctx.device_index)
        shape = (n_seq, n_kv_heads, rows, head_dim)
        k, v = (torch.zeros(shape, dtype=getattr(torch, dtype), device=dev) for _ in range(2))
        scales = (torch.ones(shape[:3], dtype=torch.float32, device=dev) for _ in range(2)) if dtype == "int8" else ()
        return cls(ctx, k, v, *scales, first_position=first_position)

    @property
    def nbytes(self) -> int:
        """Device bytes of the rows and scales."""
        return sum(t.numel() * t.element_size() for t in (self.k, self.v, self.k_scale, self.v_scale) if t is not None)

    def _rows(self, what: str, t, heads: int | None, tokens: int | None = None):
        """A float32 ``[tokens, heads, head_dim]`` whose tokens may lie apart; its tokens and their distance."""
        d, shape = self.head_dim, t.shape
        if (t.dtype is self._f32 and t.device == self.device and len(shape) == 3 and shape[2] == d
                and (heads is None or shape[1] == heads) and (tokens is None or shape[0] == tokens) and t.is_contiguous()):
            return shape[0], shape[1] * d
        check_tensor(what, t, self._f32, self.device)
        if t.dim() != 3 or t.shape[2] != d or (heads is not None and t.shape[1] != heads) or \
                (tokens is not None and t.shape[0] != tokens):
            want = ("tokens" if tokens is None else tokens, "heads" if heads is None else heads, d)
            raise KernelError(f"{what} must be [{', '.join(map(str, want))}], got {tuple(t.shape)}")
        if (t.stride(2) != 1 and d > 1) or (t.shape[1] > 1 and t.stride(1) != d):
            raise KernelError(f"{what}: a token's heads must lie one behind the other, got strides {t.stride()}")
        width = t.shape[1] * d
        return t.shape[0], (t.stride(0) if t.shape[0] > 1 else width)

    def _places(self, positions, seq_index, tokens: int | None = None) -> int:
        shape = positions.shape
        if (positions.dtype is self._i32 and seq_index.dtype is self._i32 and len(shape) == 1 and seq_index.shape == shape
                and (tokens is None or shape[0] == tokens) and positions.device == self.device
                and seq_index.device == self.device and positions.is_contiguous() and seq_index.is_contiguous()):
            return shape[0]
        n = shape[0] if len(shape) == 1 else -1
        for what, t in (("positions", positions), ("seq_index", seq_index)):
            check_tensor(what, t, self._i32, self.device, (n if tokens is None else tokens,))
            if not t.is_contiguous():
                raise KernelError(f"{what} must be contiguous")
        return n

    def append(self, k, v, cos_sin, positions, seq_index, q=None, q_out=None):
        """Rotates ``k`` by its position's row of ``cos_sin`` ``[positions, head_dim / 2, 2]`` and writes it and
        ``v`` (``[tokens, kv heads, head_dim]``) into row ``positions[t] - first_position`` of slot
        ``seq_index[t]`` (int32, on the device), quantised where the cache is int8.  ``q``
        ``[tokens, heads, head_dim]``, if given, is rotated into ``q_out`` (default: a new tensor; ``q`` itself is
        allowed), which is returned.  A token outside the cache is skipped and reported by
        ``ctx.synchronize()``; of several tokens that name one row the last one stays."""
        torch = self._torch
        n, k_stride = self._rows("k", k, self.n_kv_heads)
        _, v_stride = self._rows("v", v, self.n_kv_heads, n)
        self._places(positions, seq_index, n)
        check_tensor("cos_sin", cos_sin, torch.float32, self.device)
        if cos_sin.dim() != 3 or tuple(cos_sin.shape[1:]) != (self.head_dim // 2, 2) or not cos_sin.is_contiguous():
            raise KernelError(f"cos_sin must be a contiguous [positions, {self.head_dim // 2}, 2], got {tuple(cos_sin.shape)}")
        q_ptr = out_ptr = None
        q_stride = out_stride = heads = 0
        if q is not None:
            _, q_stride = self._rows("q", q, None, n)
            heads = q.shape[1]
            if q_out is None:
                q_out = q.new_empty(q.shape)
            _, out_stride = self._rows("q_out", q_out, heads, n)
            q_ptr, out_ptr = q.data_ptr(), q_out.data_ptr()
        elif q_out is not None:
            raise KernelError("q_out without q")
        if n:
            with ordered(self.ctx, self.device):
                check(_lib.lib().qk_cache_append(
                    self.ctx.handle, self._ref, q_ptr, q_stride, out_ptr, out_stride, heads, k.data_ptr(), k_stride,
                    v.data_ptr(), v_stride, cos_sin.data_ptr(), cos_sin.shape[0], positions.data_ptr(),
                    seq_index.data_ptr(), self.first_position, n))
        return q_out

    def read(self, positions, seq_index, dtype: str = "float32"):
        """The rows of the named tokens as values: k, v ``[tokens, kv heads, head_dim]`` in float32 or bfloat16.
        A row that does not exist reads as zeros and is reported by ``ctx.synchronize()``."""
        if dtype not in ("float32", "bfloat16"):
            raise KernelError(f"rows are read as float32 or bfloat16, got {dtype!r}")
        n = self._places(positions, seq_index)
        shape, like = (n, self.n_kv_heads, self.head_dim), self._like[dtype]
        k, v = like.new_empty(shape), like.new_empty(shape)
        if n:
            with ordered(self.ctx, self.device):
                check(_lib.lib().qk_cache_read(self.ctx.handle, self._ref, positions.data_ptr(), seq_index.data_ptr(),
                                               self.first_position, n, _TAGS[dtype], k.data_ptr(), v.data_ptr()))
        return k, v

    def _out(self, out, q, n: int, heads: int):
        if out is None:
            return q.new_empty(q.shape), heads * self.head_dim
        return out, self._rows("out", out, heads, n)[1]

    def _prefix(self, prefix, prefix_len: int, prefix_seq: int):
        if prefix is None:
            if prefix_len:
                raise KernelError(f"prefix_len {prefix_len} without a prefix")
            return None
        if prefix.device != self.device:
            raise KernelError(f"the prefix is on {prefix.device}, the cache on {self.device}")
        if prefix_len < 0 or prefix_seq < 0:
            raise KernelError(f"prefix_len and prefix_seq must not be negative, got {prefix_len}, {prefix_seq}")
        return prefix._ref

    def attend(self, q, kv_len, prefix: "KvCache | None" = None, prefix_len: int = 0, prefix_seq: int = 0, out=None):
        """softmax(q k^T / sqrt(head_dim)) v with one query per sequence: ``q`` ``[batch, heads, head_dim]``
        (rotated), sequence b sees the first ``kv_len[b]`` rows of slot b (int32, on the device) and the first
        ``prefix_len`` rows of slot ``prefix_seq`` of ``prefix``, a cache of the same kind.  A sequence that sees
        nothing gets zeros.  Returns ``out`` (default: a new tensor; ``q`` itself is allowed)."""
        n, q_stride = self._rows("q", q, None)
        heads = q.shape[1]
        check_tensor("kv_len", kv_len, self._i32, self.device, (n,))
        if not kv_len.is_contiguous():
            raise KernelError("kv_len must be contiguous")
        ref = self._prefix(prefix, prefix_len, prefix_seq)
        out, out_stride = self._out(out, q, n, heads)
        lib = _lib.lib()
        if n:
            scratch = workspace(self.ctx, lib.qk_cache_attend_scratch(self._ref, prefix_len, n, heads), self.device)
            with ordered(self.ctx, self.device):
                check(lib.qk_cache_attend(self.ctx.handle, self._ref, ref, prefix_seq, prefix_len, q.data_ptr(), q_stride,
                                          kv_len.data_ptr(), n, heads, None if scratch is None else scratch.data_ptr(),
                                          out.data_ptr(), out_stride))
        return out

    def portion(self, q, seq: int, first_position: int, prefix: "KvCache | None" = None, prefix_len: int = 0,
                prefix_seq: int = 0, out=None):
        """The same for consecutive tokens of one sequence: ``q`` ``[tokens, heads, head_dim]`` are the positions
        ``first_position ...`` of slot ``seq``, whose rows have been appended; each sees the rows up to its own,
        and the prefix."""
        n, q_stride = self._rows("q", q, None)
        heads = q.shape[1]
        if seq < 0 or first_position < self.first_position:
            raise KernelError(f"slot {seq}, position {first_position}: the cache begins at slot 0, position "
                              f"{self.first_position}")
        ref = self._prefix(prefix, prefix_len, prefix_seq)
        row = first_position - self.first_position
        out, out_stride = self._out(out, q, n, heads)
        lib = _lib.lib()
        if n:
            scratch = workspace(self.ctx, lib.qk_cache_portion_scratch(self._ref, row, prefix_len, n, heads),
                                self.device)
            with ordered(self.ctx, self.device):
                check(lib.qk_cache_portion(self.ctx.handle, self._ref, seq, row, ref, prefix_seq, prefix_len, q.data_ptr(),
                                           q_stride, n, heads, None if scratch is None else scratch.data_ptr(),
                                           out.data_ptr(), out_stride))
        return out
