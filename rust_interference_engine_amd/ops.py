"""The batched serving operators of librie_hip.so on torch tensors: rows appended to a
cache of pages (of 16 or 8 bits), attention of new tokens over it, attention over packed
prompts, token log probabilities, rotary positions, beam search's selection, and pools of
pages (include/rie_hip.h has their rules).

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

A search with beams over a pool, after the step's logits:

    pool = ops.PagePool.empty(n_pages, n_seq, most_pages_of_one, page_size, device)
    select = ops.BeamSelect(logits, scores, next_scores, parents, tokens)
    fork = ops.PageFork(pool, parents.view(-1), [k_pages, v_pages])
    reserve = ops.PageReserve(pool)
    select(); fork(); pool.lens += 1; reserve()
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
        n_pages, page, n_kv, hd = k.shape
        self.bits8 = k.dtype == torch.int8
        scales = [s for s in (k_scale, v_scale) if s is not None]
        _need(len(scales) == 2 * self.bits8, "int8 pages, and no others, have k_scale and v_scale")
        blocks = 0
        if self.bits8:
            blocks = k_scale.shape[1] if k_scale.dim() == 3 else 0
            _need(k_scale.dtype == v_scale.dtype == torch.float32, f"scales are {k_scale.dtype} and {v_scale.dtype}: f32 is wanted")
            _need(k_scale.shape == v_scale.shape == (n_pages, blocks, n_kv) and blocks > 0 and page % blocks == 0,
                  f"scales have to be [{n_pages} pages, blocks of a page, {n_kv} KV heads], got {tuple(k_scale.shape)} and {tuple(v_scale.shape)}")
            _need(_strides(k_scale) == _strides(v_scale), "k_scale and v_scale have to have the same strides")
        self.device = _device(k, v, table, *scales)
        self.k, self.v, self.table, self.k_scale, self.v_scale = k, v, table, k_scale, v_scale
        pages = _lib.Pages(_I8 if self.bits8 else _type(k, "pages"), hd, n_kv, n_pages, page, table.shape[1], k.data_ptr(), v.data_ptr(),
                           k.stride(0), k.stride(1), k.stride(2), table.data_ptr(), table.stride(0))
        self._struct = _lib.Pages8(pages, k_scale.data_ptr(), v_scale.data_ptr(), *k_scale.stride(), page // blocks) if self.bits8 else pages


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


def rotary_frequencies(dims: int, base: float = 10000.0, *, factors=None, linear: float = 1.0, parts: tuple | None = None):
    """The angles per position of ``dims`` / 2 pairs, base^(-2i / dims), as f64 on the host, and the factor of the
    rotated values.  For contexts beyond those trained on: ``factors`` divides each pair's angle by its own number (as
    ``rope_freqs.weight`` does), ``linear`` all of them by one; ``parts`` = (factor, original context) divides the
    slow ones by factor and leaves the fast ones, with a ramp, linear in the pair's number, between those that turn
    once and 32 times within the original context, and multiplies the rotated values by 0.1 ln(factor) + 1 (YaRN, arXiv 2309.00071)."""
    _need(dims >= 2 and dims % 2 == 0, f"dims has to be even and positive, got {dims}")
    _need(base > 0 and linear > 0, "base and linear have to be positive")
    f = base ** (-2 * torch.arange(dims // 2, dtype=torch.float64) / dims) / linear
    magnitude = 1.0
    if factors is not None:
        factors = torch.as_tensor(factors, dtype=torch.float64, device="cpu")
        _need(factors.shape == f.shape, f"{tuple(factors.shape)} factors for {dims // 2} pairs")
        f = f / factors
    if parts is not None:
        factor, original = parts
        _need(factor >= 1 and original > 0 and base > 1, "parts has to be (a factor of 1 or more, the original context), of a base above 1")

        def pair(turns):  # that turns so often within the original context
            return dims * math.log(original / (turns * 2 * math.pi)) / (2 * math.log(base))

        low, high = max(math.floor(pair(32)), 0), min(math.ceil(pair(1)), dims - 1)
        ramp = ((torch.arange(dims // 2, dtype=torch.float64) - low) / max(high - low, 1e-3)).clamp(0, 1)
        f = f / factor * ramp + f * (1 - ramp)
        magnitude = 0.1 * math.log(factor) + 1.0
    return f, magnitude


class Rotary(_Op):
    """Queries ``q`` and keys ``k`` [rows, heads, head size] turned by their positions, to
    ``q_out`` and ``k_out`` (of any of the types; ``q`` and ``k`` themselves will do).
    ``frequencies`` f64 [dims / 2] on the GPU: angles per position of the first dims values
    of a head.  Positions: int32 ``positions`` [rows], or those of the tokens of ``seqs``.
    ``k`` and ``k_out`` may be None."""

    def __init__(self, frequencies: torch.Tensor, q: torch.Tensor, k: torch.Tensor | None, q_out: torch.Tensor, k_out: torch.Tensor | None, *,
                 positions: torch.Tensor | None = None, seqs: Seqs | None = None, interleaved: bool = False, magnitude: float = 1.0):
        _need(frequencies.dtype == torch.float64 and frequencies.dim() == 1 and frequencies.is_contiguous() and frequencies.numel() > 0,
              f"frequencies have to be contiguous f64 [dims / 2], got {frequencies.dtype} {tuple(frequencies.shape)}")
        _need((positions is None) != (seqs is None), "positions or seqs has to be given, not both")
        _need((k is None) == (k_out is None), "k and k_out have to be given together")
        hd = _rows(q, "q").shape[2]
        pairs = [(q, q_out, "q")] + ([(k, k_out, "k")] if k is not None else [])
        n = _int(q.shape[0], "rows", 1, (1 << 26) - 4)
        x = _lib.Rotary(n, hd, 2 * frequencies.numel(), 0, 0, int(interleaved), _type(q, "q"), _type(q_out, "q_out"), magnitude, frequencies.data_ptr(),
                        positions.data_ptr() if positions is not None else None)
        for t, out, what in pairs:
            _rows(t, what, hd), _rows(out, what + "_out", hd)
            _need(t.shape == out.shape and t.shape[0] == n, f"{what} and {what}_out have to have one shape, and q's rows")
            _need(t.dtype == q.dtype and out.dtype == q_out.dtype, "q and k, and q_out and k_out, have to have one type")
            _written(out, what + "_out")
            setattr(x, "n_" + what, t.shape[1])
            for name, y in ((what, t), (what + "_out", out)):
                setattr(x, name, y.data_ptr())
                setattr(x, name + "_row_stride", y.stride(0))
                setattr(x, name + "_head_stride", y.stride(1))
        _need(2 * frequencies.numel() <= hd, f"{2 * frequencies.numel()} dims of heads of {hd}")
        tensors = [frequencies] + [t for p in pairs for t in p[:2]]
        sq = None
        if positions is not None:
            _ints(positions, "positions", 1)
            _need(positions.numel() == n, f"{positions.numel()} positions for {n} rows")
            tensors.append(positions)
        else:
            _need(seqs.lens is not None, "seqs has no lens")
            sq = seqs._struct(n)
            tensors += [seqs.starts, seqs.lens]
        dev = _device(*tensors)
        self._ready(_lib.lib().rie_hip_k_rotary, [C.byref(x), C.byref(sq) if sq else None], dev, 0, None, (x, sq, seqs, tensors))


class BeamSelect(_Op):
    """Of ``logits`` [requests * beams, vocabulary] and the beams' sums ``scores`` f32
    [requests, beams]: the best continuations of every request, in order, to ``next_scores``
    (f32), ``parents`` (int32: rows of logits) and ``tokens`` (int32), all [requests, number
    wanted].  Beams with ``finished`` (int32 [requests, beams]) other than 0 go on with the
    token ``pad`` and their own sum."""

    def __init__(self, logits: torch.Tensor, scores: torch.Tensor, next_scores: torch.Tensor, parents: torch.Tensor, tokens: torch.Tensor, *,
                 finished: torch.Tensor | None = None, pad: int = 0):
        _need(logits.dim() == 2 and logits.numel() > 0, f"logits have to be [requests * beams, vocabulary], got {tuple(logits.shape)}")
        _need(logits.shape[1] == 1 or logits.stride(1) == 1, "a row's logits have to be consecutive")
        _need(scores.dim() == 2 and scores.numel() == logits.shape[0], f"scores have to be [requests, beams] of {logits.shape[0]} rows, got {tuple(scores.shape)}")
        n, beams = scores.shape
        _need(next_scores.dim() == 2 and next_scores.shape[0] == n and next_scores.shape == parents.shape == tokens.shape,
              "next_scores, parents and tokens have to be [requests, number wanted]")
        for t, what, dtype in ((scores, "scores", torch.float32), (next_scores, "next_scores", torch.float32), (parents, "parents", torch.int32),
                               (tokens, "tokens", torch.int32), (finished, "finished", torch.int32)):
            _need(t is None or t.dtype == dtype and t.is_contiguous(), f"{what} has to be contiguous {dtype}")
        _need(finished is None or finished.shape == scores.shape, "finished has to have the shape of scores")
        n_vocab, keep = _int(logits.shape[1], "vocabulary", 1, 1 << 21), next_scores.shape[1]
        given = [scores, next_scores, parents, tokens] + ([finished] if finished is not None else [])
        dev = _device(logits, *given)
        L = _lib.lib()
        self._ready(L.rie_hip_k_beam_select, [_type(logits, "logits"), logits.data_ptr(), n, beams, n_vocab, logits.stride(0), scores.data_ptr(),
                    finished.data_ptr() if finished is not None else None, _int(pad, "pad", 0, n_vocab - 1), keep, next_scores.data_ptr(), parents.data_ptr(),
                    tokens.data_ptr()], dev, L.rie_hip_k_beam_select_ws(n, beams, n_vocab, keep), 13, (logits, given))


class PagePool:
    """The pages of a cache and the sequences that hold them, all int32 on the GPU: ``table``
    [sequences, most pages of one], the positions ``lens`` and the number of pages ``held`` of
    each, ``refs`` [pages], how many rows hold a page (0: free), and ``counts`` [2], how many
    pages the last reserve or fork lacked and how many the last compact found in use."""

    def __init__(self, table: torch.Tensor, lens: torch.Tensor, held: torch.Tensor, refs: torch.Tensor, counts: torch.Tensor, *, page_size: int):
        _ints(table, "table", 2)
        for t, what in ((lens, "lens"), (held, "held"), (refs, "refs"), (counts, "counts")):
            _ints(t, what, 1)
        n = table.shape[0]
        _need(lens.numel() == held.numel() == n, f"{lens.numel()} lens and {held.numel()} held for {n} sequences")
        _need(counts.numel() == 2, "counts has to hold two numbers")
        _written(table, "table")
        self.device = _device(table, lens, held, refs, counts)
        self.table, self.lens, self.held, self.refs, self.counts, self.page_size = table, lens, held, refs, counts, page_size
        self._struct = _lib.Pool(_int(n, "sequences", 1, 4096), _int(refs.numel(), "pages", 1, 1 << 24), _int(table.shape[1], "columns", 1, 1 << 20),
                                 _int(page_size, "page_size", 1, 4096), table.data_ptr(), table.stride(0), lens.data_ptr(), held.data_ptr(), refs.data_ptr(),
                                 counts.data_ptr())

    @classmethod
    def empty(cls, n_pages: int, n_seq: int, cols: int, page_size: int, device) -> "PagePool":
        """A pool of free pages and sequences without any."""
        def zeros(*shape):
            return torch.zeros(*shape, dtype=torch.int32, device=device)

        return cls(zeros(n_seq, cols) - 1, zeros(n_seq), zeros(n_seq), zeros(n_pages), zeros(2), page_size=page_size)

    def _workspace(self) -> int:
        return _lib.lib().rie_hip_k_page_ws(C.byref(self._struct))


def _page_bufs(caches, n_pages: int):
    """caches [pages, ...] as the library takes them: a page's values lie together, in any order"""
    caches = list(caches)
    bufs = (_lib.PageBuf * max(len(caches), 1))()
    for b, t in zip(bufs, caches):
        _need(t.dim() >= 2 and t.shape[0] == n_pages and t.numel() > 0, f"a cache has to be [{n_pages} pages, ...], got {tuple(t.shape)}")
        span = 1
        for st, n in sorted((st, n) for n, st in zip(t.shape[1:], t.stride()[1:]) if n > 1):
            _need(st == span, "a page's values have to lie together")
            span *= n
        b.base, b.page_stride, b.page_bytes = t.data_ptr(), t.stride(0) * t.element_size(), span * t.element_size()
    return caches, bufs


class PageReserve(_Op):
    """Pages for the positions that ``pool.lens`` says: the lowest free ones, row by row.  What the pool lacks is counted in
    ``pool.counts[0]``, and what a row of the table has no room for."""

    def __init__(self, pool: PagePool):
        self._ready(_lib.lib().rie_hip_k_page_reserve, [C.byref(pool._struct)], pool.device, pool._workspace(), 1, (pool,))


class PageFork(_Op):
    """Row i of the pool becomes what row ``src[i]`` (int32 [sequences], on the GPU) was, all at
    once: full pages are shared, a partial last one is copied for all but one of the rows that
    take it, and for that one too where a row beside them holds it, in the pages of all ``caches``
    [pages, ...].  A row whose src is none becomes empty."""

    def __init__(self, pool: PagePool, src: torch.Tensor, caches=()):
        _ints(src, "src", 1)
        _need(src.numel() == pool.table.shape[0], f"{src.numel()} src for {pool.table.shape[0]} sequences")
        caches, bufs = _page_bufs(caches, pool.refs.numel())
        dev = _device(pool.table, src, *caches)
        self._ready(_lib.lib().rie_hip_k_page_fork, [C.byref(pool._struct), src.data_ptr(), bufs, len(caches)], dev, pool._workspace(), 4, (pool, src, caches, bufs))


class PageFree(_Op):
    """Sequences whose ``which`` (int32 [sequences], on the GPU) is not 0 give up their pages."""

    def __init__(self, pool: PagePool, which: torch.Tensor):
        _ints(which, "which", 1)
        _need(which.numel() == pool.table.shape[0], f"{which.numel()} which for {pool.table.shape[0]} sequences")
        dev = _device(pool.table, which)
        self._ready(_lib.lib().rie_hip_k_page_free, [C.byref(pool._struct), which.data_ptr()], dev, 0, None, (pool, which))


class PageCompact(_Op):
    """The pool's n pages in use become pages 0..n-1: those numbered n and up move, with their
    contents in all ``caches`` [pages, ...]."""

    def __init__(self, pool: PagePool, caches=()):
        caches, bufs = _page_bufs(caches, pool.refs.numel())
        dev = _device(pool.table, *caches)
        self._ready(_lib.lib().rie_hip_k_page_compact, [C.byref(pool._struct), bufs, len(caches)], dev, pool._workspace(), 3, (pool, caches, bufs))


class PageCopy(_Op):
    """Page ``src[i]`` of every one of ``caches`` [pages, ...] to page ``dst[i]`` (int32, on the
    GPU).  No page may be written that another pair reads or writes."""

    def __init__(self, caches, src: torch.Tensor, dst: torch.Tensor):
        caches = list(caches)
        _need(len(caches) > 0, "no caches")
        _ints(src, "src", 1), _ints(dst, "dst", 1)
        _need(src.numel() == dst.numel() > 0, f"{src.numel()} src and {dst.numel()} dst")
        n_pages = caches[0].shape[0]
        caches, bufs = _page_bufs(caches, n_pages)
        dev = _device(src, dst, *caches)
        self._ready(_lib.lib().rie_hip_k_page_copy, [bufs, len(caches), n_pages, src.data_ptr(), dst.data_ptr(), src.numel()], dev, 0, None, (caches, src, dst, bufs))
