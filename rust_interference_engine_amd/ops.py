"""The batched serving operators of librie_hip.so on torch tensors: rows appended to a
cache of pages, attention of new tokens over it, attention over packed prompts, and
token log probabilities (include/rie_hip.h has their rules).

Each operator is an object that is made once over the tensors it works on, which checks
them, holds them and takes its workspace, and is then called as often as wanted: a call
only queues the kernels, on ``stream`` (a ``torch.cuda.Stream``) or else on torch's
current stream of the tensors' device, and reads the tensors as they are by then, so it
can be captured into a graph.  An object's calls share its workspace: two that may run at
the same time need an object each.  Keep the object until its calls have finished (one
that a graph has captured: as long as the graph is replayed); one that is made within a
capture belongs to that graph.  There are no gradients.

    kv = ops.PagedKv(k_pages, v_pages, table)
    seqs = ops.Seqs(starts, lens, max_new=1, max_len=4096)
    append = ops.PagedAppend(kv, seqs, k, v)
    attend = ops.PagedAttention(kv, seqs, q, out)
    append(); attend()
"""
from __future__ import annotations

import ctypes as C
import math

import torch

from . import _lib
from .backend import RieError

_TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 30}  # ggml type ids
_I8 = 24


def _current_stream(device: int) -> int:
    """the handle of torch's current stream: 0.1 us, where torch.cuda.current_stream takes 2"""
    return torch._C._cuda_getCurrentRawStream(device)


def _capturing(stream) -> bool:
    with torch.cuda.stream(stream):
        return torch.cuda.is_current_stream_capturing()


def _need(ok, what: str) -> None:
    if not ok:
        raise RieError(-5, what)


def _type(t: torch.Tensor, what: str) -> int:
    if t.dtype not in _TYPES:
        raise RieError(-3, f"{what} is {t.dtype}: f32, f16 or bf16 is wanted")
    return _TYPES[t.dtype]


def _int(x, what: str, least: int, most: int) -> int:
    _need(int(x) == x and least <= x <= most, f"{what} has to lie in {least}..{most}, got {x}")
    return int(x)


def _written(t: torch.Tensor, what: str) -> None:
    span = 1  # of the dimensions with smaller strides
    for st, n in sorted((st, n) for n, st in zip(t.shape, t.stride()) if n > 1):
        _need(st >= span, f"{what} is expanded or overlaps itself: its rows would be written over one another")
        span += (n - 1) * st


def _strides(t: torch.Tensor) -> tuple:
    """strides that count: a dimension of one entry has none"""
    return tuple(st if n > 1 else 0 for n, st in zip(t.shape, t.stride()))


def _device(*tensors) -> torch.device:
    d = tensors[0].device
    for t in tensors:
        _need(not t.requires_grad, "these operators have no gradients: detach the tensors")
        _need(t.device == d and d.type == "cuda", f"tensors have to be on one GPU: got {t.device} and {d}")
    return d


def _rows(t: torch.Tensor, what: str, last: int | None = None) -> torch.Tensor:
    """t as [rows, heads, size] with consecutive values"""
    _need(t.dim() == 3 and t.numel() > 0, f"{what} has to be [rows, heads, head size], got {tuple(t.shape)}")
    _need(t.shape[2] == 1 or t.stride(2) == 1, f"{what}: a row's values have to be consecutive")
    _need(last is None or t.shape[2] == last, f"{what} has heads of {t.shape[2]}, {last} is wanted")
    return t


def _ints(t: torch.Tensor, what: str, dim: int) -> torch.Tensor:
    _need(t.dtype == torch.int32 and t.dim() == dim, f"{what} has to be int32 with {dim} dimension(s), got {t.dtype} {tuple(t.shape)}")
    _need(t.shape[-1] <= 1 or t.stride(-1) == 1, f"{what}: values have to be consecutive")
    return t


class _Op:
    """One prepared call: function and arguments, and what they point to."""

    def _ready(self, fn, args, device, workspace: int, ws_at: int | None, keep):
        self._fn, self._device, self._keep = fn, device, keep
        self._err = C.create_string_buffer(512)
        self.workspace = torch.empty(workspace, dtype=torch.uint8, device=device) if workspace else None
        if workspace:
            # Its memory may still be in use by what the current stream has queued: a call on another one waits for that.
            made_on = torch.cuda.current_stream(device)
            self._ordered, self._captured = {made_on.cuda_stream}, _capturing(made_on)
            self._made = made_on.record_event()
        if ws_at is not None:
            args = args[:ws_at] + [self.workspace.data_ptr() if workspace else None, workspace] + args[ws_at:]
        self._args = args

    def __call__(self, stream=None) -> None:
        if stream is None:
            handle = _current_stream(self._device.index)
        else:
            _need(stream.device == self._device, f"stream of {stream.device}, tensors on {self._device}")
            handle = stream.cuda_stream
        if self.workspace is not None and handle not in self._ordered:
            self._order(torch.cuda.current_stream(self._device) if stream is None else stream)
        if handle == 0 and torch.cuda.current_device() != self._device.index:  # every device's null stream is 0
            with torch.cuda.device(self._device):
                rc = self._fn(*self._args, None, self._err, 512)
        else:
            rc = self._fn(*self._args, handle, self._err, 512)
        if rc:
            raise RieError(rc, self._err.value.decode(errors="replace"))

    def _order(self, stream) -> None:
        # a capture waits for events of its own only (torch.cuda.graph has waited for the device before it begins)
        if _capturing(stream) == self._captured:
            stream.wait_event(self._made)
            if not self._captured:
                self._ordered.add(stream.cuda_stream)


class Seqs:
    """The sequences of a batch: rows ``starts[i]..starts[i+1]`` are sequence i's new
    tokens, the last of its ``lens[i]`` positions; both int32 on the GPU.  ``max_new``
    and ``max_len`` bound any one sequence's.  ``lens`` is not needed by packed prompts."""

    def __init__(self, starts: torch.Tensor, lens: torch.Tensor | None = None, *, max_new: int, max_len: int):
        _ints(starts, "starts", 1)
        _need(starts.numel() >= 2, "starts has to hold a sequence's first row and its end at least")
        if lens is not None:
            _ints(lens, "lens", 1)
            _need(lens.numel() == starts.numel() - 1, f"{lens.numel()} lens for {starts.numel() - 1} sequences")
            _device(starts, lens)
        self.starts, self.lens = starts, lens
        self.max_new, self.max_len = _int(max_new, "max_new", 1, 1 << 30), _int(max_len, "max_len", 1, 1 << 30)

    def _struct(self, n_rows: int) -> _lib.Seqs:
        _int(n_rows, "rows", 1, (1 << 26) - 4)
        return _lib.Seqs(self.starts.numel() - 1, n_rows, self.max_new, self.max_len, self.starts.data_ptr(),
                         self.lens.data_ptr() if self.lens is not None else None)


class PagedKv:
    """A layer's keys and values in pages: ``k`` and ``v`` [pages, page size, KV heads, head
    size] of the same type and strides (a transposed view of another order of the middle
    two will do), ``table`` int32 [sequences, most pages of one].

    In 8 bits: ``k`` and ``v`` are int8 codes, and ``k_scale`` and ``v_scale`` (f32 [pages,
    blocks of a page, KV heads], of the same strides) what the codes of a block of page size /
    blocks positions are multiplied by.  A block that new tokens come to is one sequence's alone."""

    def __init__(self, k: torch.Tensor, v: torch.Tensor, table: torch.Tensor, *, k_scale: torch.Tensor | None = None,
                 v_scale: torch.Tensor | None = None):
        _need(k.dim() == 4 and k.numel() > 0, f"pages have to be [pages, page size, KV heads, head size], got {tuple(k.shape)}")
        _need(k.shape == v.shape and k.dtype == v.dtype and _strides(k) == _strides(v), "k and v have to have one shape, type and strides")
        _need(k.shape[3] == 1 or k.stride(3) == 1, "pages: a row's values have to be consecutive")
        _ints(table, "table", 2)
        _need(table.numel() > 0, "table is empty")
        self.device = _device(k, v, table)
        self.k, self.v, self.table = k, v, table
        n_pages, page, n_kv, hd = k.shape
        self.k_scale, self.v_scale = k_scale, v_scale
        self.bits8 = k.dtype == torch.int8
        _need((k_scale is not None) == (v_scale is not None) == self.bits8, "int8 pages, and no others, have k_scale and v_scale")
        pages = _lib.Pages(_I8 if self.bits8 else _type(k, "pages"), hd, n_kv, n_pages, page, table.shape[1], k.data_ptr(), v.data_ptr(),
                           k.stride(0), k.stride(1), k.stride(2), table.data_ptr(), table.stride(0))
        if not self.bits8:
            self._struct = pages
            return
        _device(k, k_scale, v_scale)
        blocks = k_scale.shape[1] if k_scale.dim() == 3 else 0
        _need(k_scale.dtype == v_scale.dtype == torch.float32, f"scales are {k_scale.dtype} and {v_scale.dtype}: f32 is wanted")
        _need(k_scale.shape == v_scale.shape == (n_pages, blocks, n_kv) and blocks > 0 and page % blocks == 0,
              f"scales have to be [{n_pages} pages, blocks of a page, {n_kv} KV heads], got {tuple(k_scale.shape)} and {tuple(v_scale.shape)}")
        _need(_strides(k_scale) == _strides(v_scale), "k_scale and v_scale have to have the same strides")
        self._struct = _lib.Pages8(pages, k_scale.data_ptr(), v_scale.data_ptr(), k_scale.stride(0), k_scale.stride(1), k_scale.stride(2), page // blocks)


def _check_seqs(seqs: Seqs, table: torch.Tensor | None) -> None:
    if table is not None:
        _need(seqs.lens is not None, "seqs has no lens")
        _need(table.shape[0] >= seqs.starts.numel() - 1, f"table of {table.shape[0]} rows for {seqs.starts.numel() - 1} sequences")


class PagedAppend(_Op):
    """The new tokens' ``k`` and ``v`` [rows, KV heads, head size] (f32 or the pages' type; to
    8-bit pages f32, f16 or bf16; one stride set) written to their pages."""

    def __init__(self, kv: PagedKv, seqs: Seqs, k: torch.Tensor, v: torch.Tensor):
        hd = kv.k.shape[3]
        _rows(k, "k", hd), _rows(v, "v", hd)
        _need(k.shape == v.shape and k.dtype == v.dtype and _strides(k) == _strides(v), "k and v have to have one shape, type and strides")
        _need(k.shape[1] == kv.k.shape[2], f"k has {k.shape[1]} heads, the pages {kv.k.shape[2]}")
        _check_seqs(seqs, kv.table)
        _written(kv.k, "pages")
        if kv.bits8:
            _written(kv.k_scale, "scales")
        dev = _device(kv.k, k, v, seqs.starts, seqs.lens)
        sq = seqs._struct(k.shape[0])
        L = _lib.lib()
        self._ready(L.rie_hip_k_paged_append8 if kv.bits8 else L.rie_hip_k_paged_append, [C.byref(kv._struct), C.byref(sq), _type(k, "k"), k.data_ptr(), v.data_ptr(),
                    k.stride(0), k.stride(1)], dev, 0, None, (kv, seqs, sq, k, v))


def _attn(q: torch.Tensor, out: torch.Tensor, n_kv: int, ty: torch.dtype, hd: int, scale, window: int, softcap: float) -> _lib.Attn:
    _rows(q, "q", hd), _rows(out, "out", hd)
    _need(q.shape == out.shape and q.dtype == out.dtype == ty, "q and out have to have one shape, and the keys' type")
    _need(q.shape[1] % n_kv == 0, f"{q.shape[1]} query heads on {n_kv} KV heads")
    _written(out, "out")
    return _lib.Attn(q.shape[1], _int(window, "window", 0, 2**31 - 1), 1 / math.sqrt(hd) if scale is None else scale, softcap, q.data_ptr(), q.stride(0), q.stride(1),
                     out.data_ptr(), out.stride(0), out.stride(1))


class PagedAttention(_Op):
    """Causal attention of every sequence's new tokens ``q`` [rows, heads, head size] over
    its pages, which hold them already, to ``out``, both of the pages' type (over 8-bit pages
    f16 or bf16)."""

    def __init__(self, kv: PagedKv, seqs: Seqs, q: torch.Tensor, out: torch.Tensor, *, scale: float | None = None, window: int = 0,
                 softcap: float = 0.0):
        _check_seqs(seqs, kv.table)
        at = _attn(q, out, kv.k.shape[2], q.dtype if kv.bits8 else kv.k.dtype, kv.k.shape[3], scale, window, softcap)
        dev = _device(kv.k, q, out, seqs.starts, seqs.lens)
        sq = seqs._struct(q.shape[0])
        L = _lib.lib()
        if kv.bits8:
            fn, ws, args = L.rie_hip_k_paged_attention8, L.rie_hip_k_paged_attention8_ws, [C.byref(kv._struct), C.byref(sq), _type(q, "q"), C.byref(at)]
        else:
            fn, ws, args = L.rie_hip_k_paged_attention, L.rie_hip_k_paged_attention_ws, [C.byref(kv._struct), C.byref(sq), C.byref(at)]
        self._ready(fn, args, dev, ws(*args), len(args), (kv, seqs, sq, at, q, out))


class PackedAttention(_Op):
    """Causal attention within each of the whole prompts that ``seqs`` packs: ``q`` and
    ``out`` [rows, heads, head size], ``k`` and ``v`` [rows, KV heads, head size]."""

    def __init__(self, seqs: Seqs, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, out: torch.Tensor, *, scale: float | None = None,
                 window: int = 0, softcap: float = 0.0):
        hd = _rows(q, "q").shape[2]
        _rows(k, "k", hd), _rows(v, "v", hd)
        _need(k.shape == v.shape and k.dtype == v.dtype and k.shape[0] == q.shape[0], "k and v have to have one shape and type, and q's rows")
        at = _attn(q, out, k.shape[1], k.dtype, hd, scale, window, softcap)
        dev = _device(q, k, v, out, seqs.starts)
        sq = seqs._struct(q.shape[0])
        ty, n_kv = _type(k, "k"), k.shape[1]
        ws = _lib.lib().rie_hip_k_packed_attention_ws(C.byref(sq), ty, hd, n_kv, C.byref(at))
        self._ready(_lib.lib().rie_hip_k_packed_attention, [C.byref(sq), ty, hd, n_kv, k.data_ptr(), v.data_ptr(), k.stride(0), k.stride(1),
                    v.stride(0), v.stride(1), C.byref(at)], dev, ws, 11, (seqs, sq, at, q, k, v, out))


class TokenLogprobs(_Op):
    """Of ``logits`` [rows, vocabulary]: ``logprob`` [rows] of the int32 ``targets``, the
    ``entropy`` [rows], and the most likely tokens ``top_ids`` (int32) with
    ``top_logprobs``, both [rows, number wanted]; results f32, any of them None."""

    def __init__(self, logits: torch.Tensor, *, targets: torch.Tensor | None = None, logprob: torch.Tensor | None = None,
                 entropy: torch.Tensor | None = None, top_ids: torch.Tensor | None = None, top_logprobs: torch.Tensor | None = None):
        _need(logits.dim() == 2 and logits.numel() > 0, f"logits have to be [rows, vocabulary], got {tuple(logits.shape)}")
        _need(logits.shape[1] == 1 or logits.stride(1) == 1, "a row's logits have to be consecutive")
        n, n_vocab = _int(logits.shape[0], "rows", 1, 1 << 22), _int(logits.shape[1], "vocabulary", 1, 1 << 21)
        _need((targets is None) == (logprob is None), "targets and logprob have to be given together")
        _need((top_ids is None) == (top_logprobs is None), "top_ids and top_logprobs have to be given together")
        top = 0
        if top_ids is not None:
            _need(top_ids.dim() == 2 and top_ids.shape[0] == n and top_ids.shape == top_logprobs.shape, "top_ids and top_logprobs have to be [rows, number wanted]")
            top = top_ids.shape[1]
        for t, what, dtype in ((targets, "targets", torch.int32), (logprob, "logprob", torch.float32), (entropy, "entropy", torch.float32),
                               (top_ids, "top_ids", torch.int32), (top_logprobs, "top_logprobs", torch.float32)):
            if t is not None:
                _need(t.dim() == (2 if what.startswith("top") else 1), f"{what} has {t.dim()} dimensions")
                _need(t.dtype == dtype and t.shape[0] == n and t.is_contiguous(), f"{what} has to be contiguous {dtype} for {n} rows")
        given = [t for t in (targets, logprob, entropy, top_ids, top_logprobs) if t is not None]
        dev = _device(logits, *given)
        ptr = [None if t is None or not t.numel() else t.data_ptr() for t in (targets, logprob, entropy, top_ids, top_logprobs)]
        self._ready(_lib.lib().rie_hip_k_token_logprobs, [_type(logits, "logits"), logits.data_ptr(), n, n_vocab, logits.stride(0),
                    ptr[0], ptr[1], ptr[2], top, ptr[3], ptr[4]], dev, _lib.lib().rie_hip_k_token_logprobs_ws(n, n_vocab), 11, (logits, given))
