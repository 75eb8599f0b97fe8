"""Serving what the engine converts: products with packed HiF4 weights, a paged
key/value cache in packed HiF4 and the attention that reads it.

Weights are the (meta, codes) pairs that codec.convert(packed=True) and
codec.pack give; the cache holds the same 64-element units.  Activations are
bf16: a HiF4 value is a bf16 number, so nothing is lost before the fp32 sums
(fp16 does not reach HiF4's exponents).  Every function launches kernels from
libhif4x.so on the current stream of the tensors' device, allocates with
torch and neither synchronises nor reads back, so a call can be captured into
a CUDA graph.  There is no backward pass: where gradients are recorded, tensors
that require one are refused.  linalg.check_device_status reports what a kernel found wrong
(a page table that names no page of the cache).
"""
from __future__ import annotations

import ctypes
import functools

import torch

from . import _lib as L

GROUP = 64
_I32 = (torch.int32,)
ACTIVATIONS = {"none": 0, "relu": 1, "gelu": 2, "gelu_tanh": 3, "silu": 4}


def _call(dev: torch.device, name: str, *args) -> None:
    """An entry point with the device's current stream behind its arguments, the device being the current one."""
    index = dev.index
    stream = torch._C._cuda_getCurrentRawStream(index)
    if index == torch.cuda.current_device():
        L.call(name, *args, stream)
    else:
        with torch.cuda.device(index):
            L.call(name, *args, stream)


def _cuda(t: torch.Tensor, name: str, dtypes, dim: int, dev: torch.device | None = None):
    """The tensor has one of the dtypes and `dim` dimensions, is on `dev` (None: on any GPU) and waits for no gradient."""
    if isinstance(t, torch.Tensor) and t.dtype in dtypes and t.dim() == dim and (
            t.device == dev if dev is not None else t.is_cuda):
        if t.requires_grad and torch.is_grad_enabled():
            raise ValueError(f"{name} requires a gradient and this call has none: detach it, or call under torch.no_grad()")
        return
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a tensor")
    if t.dtype not in dtypes:
        raise TypeError(f"{name} is {t.dtype}: {' or '.join(str(d) for d in dtypes)} wanted")
    if t.dim() != dim:
        raise ValueError(f"{name} has {t.dim()} dimensions: {dim} wanted")
    if not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor")
    raise ValueError(f"{name} is on {t.device}, the first tensor on {dev}")


def _row_stride(t: torch.Tensor, name: str, aligned: bool) -> int:
    """Stride of the rows of a 2-D tensor with unit inner stride (one row: its length, rounded up)."""
    rows, cols = t.shape
    if cols > 1 and t.stride(1) != 1:
        raise ValueError(f"{name} needs unit stride along its last dimension")
    ld = t.stride(0) if rows > 1 else (cols + 7) // 8 * 8
    if rows > 1 and ld < cols:
        raise ValueError(f"{name} has rows {ld} apart, shorter than the {cols} of a row")
    if aligned and (ld % 8 or t.data_ptr() % 16):
        raise ValueError(f"{name} needs a 16-byte aligned start and rows a multiple of 8 elements apart")
    return ld


def _span(t: torch.Tensor) -> tuple[int, int]:
    """The addresses from a tensor's first element to behind its last."""
    at = t.data_ptr()
    if t.is_contiguous():
        return at, at + t.nbytes
    return at, at + (sum((s - 1) * st for s, st in zip(t.shape, t.stride())) + 1) * t.element_size()


def _overlap(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether the spans of two tensors' elements meet."""
    (a0, a1), (b0, b1) = _span(a), _span(b)
    return a0 < b1 and b0 < a1


def _runs(t: torch.Tensor) -> tuple[int, int]:
    """(pitch, width) in bytes: the elements as runs of `width` that begin `pitch` apart, a run for each index of
    the dimension with the largest stride."""
    dims = sorted((st, s) for s, st in zip(t.shape, t.stride()) if s > 1)
    size = t.element_size()
    if not dims:
        return 0, size
    return dims[-1][0] * size, (sum((s - 1) * st for st, s in dims[:-1]) + 1) * size


def _beside(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether two tensors whose spans meet are ranges of columns of one buffer that do not."""
    (pa, wa), (pb, wb) = _runs(a), _runs(b)
    if pa != pb or pa == 0:
        return False
    return wa <= (b.data_ptr() - a.data_ptr()) % pa <= pa - wb


def _apart(out: torch.Tensor, name: str, *inputs) -> None:
    """`out` lies over none of the inputs, (tensor, name) each."""
    for t, what in inputs:
        if _overlap(out, t) and not _beside(out, t):
            raise ValueError(f"{name} overlaps {what}")


def linear(x: torch.Tensor, meta: torch.Tensor, codes: torch.Tensor, bias: torch.Tensor | None = None,
           activation: str = "none", residual: torch.Tensor | None = None,
           out: torch.Tensor | None = None) -> torch.Tensor:
    """activation(x W^T + bias) + residual, bf16 (T, N), with W (N, C) in packed HiF4.

    x: (T, C) bf16, unit inner stride, rows a multiple of 8 elements apart, 16-byte aligned.  meta int32
    (N, C/64) and codes uint8 (N, C/2): contiguous.  bias: (N,) fp32 or bf16.  activation: none, relu, gelu
    (by erf), gelu_tanh or silu.  residual: (T, N) bf16, unit inner stride; out: the same, and it may be the
    residual itself, but lie over no other input.  Sums are fp32 on the tensor cores, rounded once at the end.

    x is taken as it comes.  A weight that linear.calibrate_weight made, or codec.convert with smoothing or
    rotation, belongs to activations smoothed (times the activation state's s) and, where its mode is 1, rotated:
    bring x there first, by codec.convert(x, kind=SRC_VALUES, smooth=s, smooth_mode=SMOOTH_MUL, rotate=mode == 1,
    encode=ENC_NONE, out_x=True), or pass the values that linear.dynamic_activation chose."""
    _cuda(x, "x", (torch.bfloat16,), 2)
    dev = x.device
    _cuda(codes, "codes", (torch.uint8,), 2, dev)
    _cuda(meta, "meta", (torch.int32,), 2, dev)
    (T, C), N = x.shape, codes.shape[0]
    if C == 0 or C % GROUP:
        raise ValueError(f"last dimension {C} is not divisible by 64")
    if codes.shape[1] * 2 != C or meta.shape[0] != N or meta.shape[1] * GROUP != C:
        raise ValueError(f"codes {tuple(codes.shape)} and meta {tuple(meta.shape)} are no packed weight of {C} columns")
    if N == 0:
        raise ValueError("the weight has no rows")
    if not (codes.is_contiguous() and meta.is_contiguous()):
        raise ValueError("codes and meta must be contiguous")
    if codes.data_ptr() % 16 or meta.data_ptr() % 16:
        raise ValueError("codes and meta need 16-byte aligned starts")
    if activation not in ACTIVATIONS:
        raise ValueError(f"activation {activation!r}: one of {', '.join(ACTIVATIONS)} wanted")
    ldx = _row_stride(x, "x", True)
    bias_dtype = 0
    if bias is not None:
        _cuda(bias, "bias", (torch.float32, torch.bfloat16), 1, dev)
        if bias.shape[0] != N or (N > 1 and bias.stride(0) != 1):
            raise ValueError(f"bias must be {N} contiguous values")
        bias_dtype = L.dtype_code(bias.dtype)
    ldr = N
    if residual is not None:
        _cuda(residual, "residual", (torch.bfloat16,), 2, dev)
        if residual.shape != (T, N):
            raise ValueError(f"residual is {tuple(residual.shape)}: ({T}, {N}) wanted")
        ldr = _row_stride(residual, "residual", False)
    if out is None:
        out = torch.empty(T, N, dtype=torch.bfloat16, device=dev)
        ldy = N
    else:
        _cuda(out, "out", (torch.bfloat16,), 2, dev)
        if out.shape != (T, N):
            raise ValueError(f"out is {tuple(out.shape)}: ({T}, {N}) wanted")
        ldy = _row_stride(out, "out", False)
        if T:
            _apart(out, "out", (x, "x"), (meta, "meta"), (codes, "codes"), *([(bias, "bias")] if bias is not None else []))
        if T and residual is not None and _overlap(out, residual) and not _beside(out, residual) and not (
                out.data_ptr() == residual.data_ptr() and ldy == ldr):
            raise ValueError("out overlaps residual without being it")
    if T == 0:
        return out
    _call(dev, "hif4x_linear_packed", x.data_ptr(), ldx, meta.data_ptr(), codes.data_ptr(), T, N, C,
          None if bias is None else bias.data_ptr(), bias_dtype, ACTIVATIONS[activation],
          None if residual is None else residual.data_ptr(), ldr, out.data_ptr(), ldy)
    return out


class PagedKV:
    """A paged key/value cache in packed HiF4: for K and for V codes uint8 (pages, kv_heads, page_size,
    head_dim/2) and meta int32 (pages, kv_heads, page_size, head_dim/64).  head_dim 64 or 128, page_size a
    power of two from 16 to 256.  Holds the tensors, which stay the caller's; they cannot be exchanged for others."""

    def __init__(self, k_codes: torch.Tensor, k_meta: torch.Tensor, v_codes: torch.Tensor, v_meta: torch.Tensor):
        _cuda(k_codes, "k_codes", (torch.uint8,), 4)
        dev = k_codes.device
        shape = k_codes.shape
        n, h, p, half = shape
        _cuda(k_meta, "k_meta", _I32, 4, dev)
        _cuda(v_codes, "v_codes", (torch.uint8,), 4, dev)
        _cuda(v_meta, "v_meta", _I32, 4, dev)
        meta = torch.Size((n, h, p, half // 32))
        if not (v_codes.shape == shape and k_meta.shape == meta and v_meta.shape == meta):
            raise ValueError(f"v_codes {tuple(v_codes.shape)}, k_meta {tuple(k_meta.shape)} and v_meta "
                             f"{tuple(v_meta.shape)} do not go with k_codes {tuple(shape)}: {tuple(shape)} and "
                             f"{tuple(meta)} wanted")
        at = [t.data_ptr() for t in (k_codes, k_meta, v_codes, v_meta)]
        if (at[0] | at[1] | at[2] | at[3]) % 16 or not (k_codes.is_contiguous() and k_meta.is_contiguous()
                                                        and v_codes.is_contiguous() and v_meta.is_contiguous()):
            raise ValueError("the cache's tensors must be contiguous and 16-byte aligned")
        if half not in (32, 64):
            raise ValueError(f"head_dim {2 * half}: 64 or 128 wanted")
        if p not in (16, 32, 64, 128, 256):
            raise ValueError(f"page_size {p}: a power of two from 16 to 256 wanted")
        if n == 0 or h == 0:
            raise ValueError("the cache has no pages or no heads")
        desc = L.KVCacheDesc(*at, n, p, h, 2 * half)
        self.__dict__.update(k_codes=k_codes, k_meta=k_meta, v_codes=v_codes, v_meta=v_meta, num_pages=n, kv_heads=h,
                             page_size=p, head_dim=2 * half, device=dev, _desc=desc, _ref=ctypes.byref(desc))

    _FIXED = frozenset(("k_codes", "k_meta", "v_codes", "v_meta", "num_pages", "kv_heads", "page_size", "head_dim",
                        "device", "_desc", "_ref"))

    def __setattr__(self, name, value):
        if name in self._FIXED:
            raise AttributeError(f"{name} of a cache is fixed (its tensors' addresses are taken when it is made): "
                                 "make another PagedKV")
        object.__setattr__(self, name, value)

    @staticmethod
    def empty(num_pages: int, page_size: int, kv_heads: int, head_dim: int, device) -> "PagedKV":
        """A cache of zeros (every code decodes to 0)."""
        if head_dim not in (64, 128):
            raise ValueError(f"head_dim {head_dim}: 64 or 128 wanted")
        shape = (num_pages, kv_heads, page_size)
        make = lambda last, dt: torch.zeros(*shape, last, dtype=dt, device=device)  # noqa: E731
        return PagedKV(make(head_dim // 2, torch.uint8), make(head_dim // 64, torch.int32),
                       make(head_dim // 2, torch.uint8), make(head_dim // 64, torch.int32))

    def _reads(self, cu_new: torch.Tensor, kv_len: torch.Tensor, pages: torch.Tensor):
        """What a call over the cache reads besides its rows, for _apart."""
        cache = ((t, "the cache") for t in (self.k_codes, self.k_meta, self.v_codes, self.v_meta))
        return *cache, (cu_new, "cu_new"), (kv_len, "kv_len"), (pages, "pages")

    def _batch(self, cu_new: torch.Tensor, kv_len: torch.Tensor, pages: torch.Tensor) -> L.KVBatchDesc:
        dev = self.device
        _cuda(cu_new, "cu_new", _I32, 1, dev)
        _cuda(kv_len, "kv_len", _I32, 1, dev)
        _cuda(pages, "pages", _I32, 2, dev)
        B, (rows, most) = kv_len.shape[0], pages.shape
        if B == 0 or cu_new.shape[0] != B + 1 or rows != B or most == 0:
            raise ValueError(f"cu_new {tuple(cu_new.shape)}, kv_len {tuple(kv_len.shape)} and pages "
                             f"{tuple(pages.shape)} describe no batch: (B + 1,), (B,) and (B, most) wanted")
        ld, unit = pages.stride()
        if cu_new.stride(0) != 1 or (B > 1 and kv_len.stride(0) != 1):
            raise ValueError("cu_new and kv_len must be contiguous")
        if (most > 1 and unit != 1) or (B > 1 and ld < most):
            raise ValueError("pages needs unit stride along its last dimension and rows apart")
        return L.KVBatchDesc(cu_new.data_ptr(), kv_len.data_ptr(), pages.data_ptr(), B, most, ld if B > 1 else most)


def _heads(t: torch.Tensor, name: str, dtypes, cache: PagedKV, heads: int | None = None):
    _cuda(t, name, dtypes, 3, cache.device)
    if t.shape[2] != cache.head_dim or (heads is not None and t.shape[1] != heads):
        raise ValueError(f"{name} is {tuple(t.shape)}: (rows, {heads or 'heads'}, {cache.head_dim}) wanted")
    if t.stride(2) != 1:
        raise ValueError(f"{name} needs unit stride along its last dimension")


def _strides(t: torch.Tensor, name: str):
    """Row and head strides of a (rows, heads, dh) tensor whose rows take 16-byte accesses."""
    rows, heads, dh = t.shape
    sh = t.stride(1) if heads > 1 else dh
    sr = t.stride(0) if rows > 1 else heads * dh
    if sr % 8 or sh % 8 or t.data_ptr() % 16:
        raise ValueError(f"{name} needs a 16-byte aligned start and strides of multiples of 8 elements")
    return sr, sh


def kv_append(cache: PagedKV, k: torch.Tensor, v: torch.Tensor, cu_new: torch.Tensor, kv_len: torch.Tensor,
              pages: torch.Tensor) -> None:
    """Write new K and V rows (rows, kv_heads, head_dim) bf16 or fp32 into the cache, by the searched encode
    (the bits that codec.convert gives).

    Sequence s has the rows cu_new[s] .. cu_new[s + 1] - 1 and, with them, kv_len[s] tokens; pages[s, i] holds
    its tokens i * page_size and on (int32, on the device).  Row j of its n new ones goes to position
    kv_len[s] - n + j.  Rows behind the last sequence are padding.  No two rows of a call may have the same
    place.  K and V may be strided views with unit inner stride."""
    _heads(k, "k", (torch.bfloat16, torch.float32), cache, cache.kv_heads)
    _heads(v, "v", (k.dtype,), cache, cache.kv_heads)
    if v.shape != k.shape:
        raise ValueError(f"k is {tuple(k.shape)}, v {tuple(v.shape)}")
    batch = cache._batch(cu_new, kv_len, pages)
    if k.shape[0] == 0:
        return
    _call(cache.device, "hif4x_kv_append", cache._ref, ctypes.byref(batch), k.data_ptr(), k.stride(0),
          k.stride(1), v.data_ptr(), v.stride(0), v.stride(1), L.dtype_code(k.dtype), k.shape[0])


def kv_read(cache: PagedKV, cu_new: torch.Tensor, kv_len: torch.Tensor, pages: torch.Tensor, rows: int,
            dtype: torch.dtype = torch.bfloat16, out: tuple[torch.Tensor, torch.Tensor] | None = None):
    """(k, v): the values of the batch's rows as the cache holds them, (rows, kv_heads, head_dim) of `dtype`
    (bf16 or fp32, both exact): the rows that kv_append writes for the same arguments, or any run of last
    tokens that cu_new names.  out: tensors to write instead, apart from all that is read; rows that have no place
    are left as they were (undefined without out)."""
    batch = cache._batch(cu_new, kv_len, pages)
    if rows < 0:
        raise ValueError(f"rows {rows}")
    if out is None:
        L.dtype_code(dtype)
        k, v = (torch.empty(rows, cache.kv_heads, cache.head_dim, dtype=dtype, device=cache.device) for _ in range(2))
    else:
        k, v = out
        _heads(k, "out[0]", (torch.bfloat16, torch.float32), cache, cache.kv_heads)
        _heads(v, "out[1]", (k.dtype,), cache, cache.kv_heads)
        if k.shape[0] != rows or v.shape[0] != rows or not (k.is_contiguous() and v.is_contiguous()):
            raise ValueError(f"out must be two contiguous tensors of {rows} rows")
        if rows:
            if k.data_ptr() % 16 or v.data_ptr() % 16 or _overlap(k, v):
                raise ValueError("out must be two 16-byte aligned tensors apart")
            for t, name in ((k, "out[0]"), (v, "out[1]")):
                _apart(t, name, *cache._reads(cu_new, kv_len, pages))
    if rows:
        _call(cache.device, "hif4x_kv_read", cache._ref, ctypes.byref(batch), rows, k.data_ptr(),
              v.data_ptr(), L.dtype_code(k.dtype))
    return k, v


@functools.lru_cache(maxsize=1024)
def _attention_work(dev: torch.device, *sizes: int) -> int:
    """Bytes of workspace of an attention call of these sizes."""
    need = L.i64()
    with torch.cuda.device(dev):
        L.call("hif4x_paged_attention_work", *sizes, ctypes.byref(need))
    return need.value


def paged_attention(q: torch.Tensor, cache: PagedKV, cu_new: torch.Tensor, kv_len: torch.Tensor, pages: torch.Tensor,
                    scale: float | None = None, window: int = 0, sinks: int = 0, max_new: int | None = None,
                    out: torch.Tensor | None = None) -> torch.Tensor:
    """Softmax attention of the batch's new rows over the cache: bf16 (rows, q_heads, head_dim).

    The batch is kv_append's, and the new rows' K and V are in the cache already.  The row at position p sees
    the keys t <= p and, with window > 0, of these t > p - window and the first `sinks` ones.  Query head h
    reads key head h // (q_heads / kv_heads).  A row that sees nothing (a negative position) gives zeros.
    scale: head_dim ** -0.5 by default.  max_new: the most new rows of a sequence, if the program knows it
    (rows otherwise): it chooses how the work is laid out; the result holds for any.  out: a tensor to write
    instead, apart from all that is read; rows of no sequence are left as they were (undefined without out)."""
    _heads(q, "q", (torch.bfloat16,), cache)
    rows, heads, dh = q.shape
    if heads == 0 or heads % cache.kv_heads:
        raise ValueError(f"{heads} query heads over {cache.kv_heads} key heads")
    if not 0 <= window <= 1 << 30 or not 0 <= sinks <= 1 << 30:
        raise ValueError(f"window {window}, sinks {sinks}: from 0 to 2^30 wanted")
    if max_new is not None and max_new < 1:
        raise ValueError(f"max_new {max_new}")
    batch = cache._batch(cu_new, kv_len, pages)
    qr, qh = _strides(q, "q")
    if out is None:
        out = torch.empty(rows, heads, dh, dtype=torch.bfloat16, device=cache.device)
        orow, ohead = heads * dh, dh
    else:
        _heads(out, "out", (torch.bfloat16,), cache, heads)
        if out.shape[0] != rows:
            raise ValueError(f"out has {out.shape[0]} rows: {rows} wanted")
        orow, ohead = _strides(out, "out")
        by_row = ohead >= dh and orow >= (heads - 1) * ohead + dh
        by_head = orow >= dh and ohead >= (rows - 1) * orow + dh
        if rows and not (by_row or by_head):
            raise ValueError("out overlaps itself")
        if rows:
            _apart(out, "out", (q, "q"), *cache._reads(cu_new, kv_len, pages))
    if rows == 0:
        return out
    most = min(rows, max_new) if max_new is not None else rows
    need = _attention_work(cache.device, cache.page_size, cache.kv_heads, dh, batch.sequences, batch.max_pages, heads,
                           rows, window, sinks, most)
    work = torch.empty(need, dtype=torch.uint8, device=cache.device) if need else None
    _call(cache.device, "hif4x_paged_attention", cache._ref, ctypes.byref(batch), q.data_ptr(), qr, qh,
          heads, rows, dh ** -0.5 if scale is None else float(scale), window, sinks, most, out.data_ptr(), orow, ohead,
          None if work is None else work.data_ptr(), need)
    return out
