"""Serving-step operators on torch CUDA tensors, over the C ABI.

    PagedKV      a paged K/V cache (f16, or 8-bit codes with a scale per row) shared by many sequences
      .write     the new tokens' K and V rows into their pages, quantised as they are written
      .read      the last positions of every sequence back out of the pages
      .attend    attention of new tokens over their sequences' pages
      .check     waits, and raises if an attention gave up inside its kernel
    Seqs         the sequences of a call: page tables, new tokens, lengths
    LogitRules   repetition / frequency / presence penalties, biases and grammar masks
      .choose    the rules on logits, the greedy choice and its log-probability

Every call runs on torch's current stream of the tensors' device and returns
without waiting for it. Arguments are checked on the host and raise ValueError
(MgbError for what the library refuses); data on the device that is out of
range (page numbers, lengths, token ids) is skipped by the kernels.
"""
from __future__ import annotations

import ctypes

import torch

from . import _lib
from ._lib import check

_TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
# The quick forms of current_stream(device).cuda_stream and current_device(), where this torch has them.
_stream_of = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda device: torch.cuda.current_stream(device).cuda_stream)
_current_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device


def _need(ok: bool, what: str) -> None:
    if not ok:
        raise ValueError(what)


def _cuda(x: torch.Tensor, name: str, dtype: torch.dtype, shape: tuple | None = None, device=None) -> int:
    """Address of a contiguous CUDA tensor of that type (and shape, and device)."""
    _need(x.is_cuda and x.dtype == dtype and x.is_contiguous(), f"{name} must be a contiguous CUDA tensor of {dtype}")
    _need(shape is None or tuple(x.shape) == tuple(shape), f"{name} has shape {tuple(x.shape)}, not {shape}")
    _need(device is None or x.device == device, f"{name} is on {x.device}, not {device}")
    return x.data_ptr()


def _rows(x: torch.Tensor, name: str, index: int, dim: int) -> _lib.Rows:
    """Packed rows [tokens, heads, dim] as the library takes them: any strides of tokens and heads."""
    kind = _TYPES.get(x.dtype)
    if kind is None:
        raise ValueError(f"{name} must be float32, float16 or bfloat16")
    if x.get_device() != index:
        raise ValueError(f"{name} is on {x.device}, the cache on GPU {index}")
    shape, strides = x.shape, x.stride()
    if len(shape) != 3 or shape[2] != dim or strides[2] != 1:
        raise ValueError(f"{name} must be [tokens, heads, {dim}] with contiguous rows")
    return _lib.Rows(x.data_ptr(), strides[0], strides[1], shape[0], shape[1], kind)


def _call(index: int, fn, *args) -> None:
    """fn(*args, current stream) with GPU `index`, the tensors', current."""
    if _current_device() == index:
        code = fn(*args, _stream_of(index))
    else:
        with torch.cuda.device(index):
            code = fn(*args, _stream_of(index))
    if code:
        check(code)


class Seqs:
    """The sequences of a call, as int32 CUDA tensors.

    table [seqs, n]: page numbers; position p of sequence b is in page
        table[b, p // page] (rows may be longer than the sequence needs).
    q_start [seqs + 1]: the new tokens of sequence b are rows q_start[b] to
        q_start[b + 1] - 1 of the call's packed rows. They stand at the last
        positions of the sequence.
    kv_len [seqs]: positions of every sequence, the new tokens included.
    max_new, max_len: host-side bounds of the new tokens and positions of a
        sequence. They only size launches: a bound that is too small costs
        time, not correctness. Without them all of a call's tokens and all of
        the tables' room are assumed.
    tokens: q_start's last entry, for calls that make packed rows (read).

    The tensors are read when a call's kernels run, so a server may update them
    in place between steps.
    """

    def __init__(self, table: torch.Tensor, q_start: torch.Tensor, kv_len: torch.Tensor, max_new: int | None = None,
                 max_len: int | None = None, tokens: int | None = None):
        _need(table.dim() == 2, "table must be [seqs, pages]")
        n, device = table.size(0), table.device
        self.tensors = (table, q_start, kv_len)  # kept alive
        self.device, self.index = device, table.get_device()
        self.tokens, self.empty = tokens, n == 0
        self._c = _lib.KvSeqs(_cuda(table, "table", torch.int32), _cuda(q_start, "q_start", torch.int32, (n + 1,), device),
                              _cuda(kv_len, "kv_len", torch.int32, (n,), device), n, table.size(1),
                              max_new or 0, max_len or 0)
        self._ref = ctypes.byref(self._c)

    @classmethod
    def of(cls, tables: list[list[int]], new: list[int], lengths: list[int], device="cuda") -> "Seqs":
        """From host lists: the page numbers, new tokens and positions of every sequence."""
        _need(len(tables) == len(new) == len(lengths), "tables, new and lengths differ in length")
        width = max([len(t) for t in tables], default=0)
        table = torch.zeros(len(tables), max(width, 1), dtype=torch.int32)
        for b, t in enumerate(tables):
            table[b, : len(t)] = torch.tensor(t, dtype=torch.int32)
        start = torch.tensor([0, *new], dtype=torch.int32).cumsum(0, dtype=torch.int32)
        return cls(table.to(device), start.to(device), torch.tensor(lengths, dtype=torch.int32).to(device),
                   max(new, default=0), max(lengths, default=0), sum(new))


class PagedKV:
    """A paged K/V cache over the caller's tensors k, v [pages, heads, page, dim]:
    float16, or int8 codes with k_scale, v_scale [pages, heads, page] float32
    (row value = code * scale, scale = max|row| / 127). dim is 16, 32, 64 or
    128, page a power of two from 16 to 1024."""

    def __init__(self, k: torch.Tensor, v: torch.Tensor, k_scale: torch.Tensor | None = None,
                 v_scale: torch.Tensor | None = None):
        _need(k.dim() == 4, "k must be [pages, heads, page, dim]")
        _need(k.dtype in (torch.float16, torch.int8), "the cache must be float16 or int8")
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        self.device, self.q8 = k.device, k.dtype == torch.int8
        self.index = k.get_device()
        self.pages, self.heads, self.page, self.dim = k.shape
        _need(self.dim in (16, 32, 64, 128), f"head dim {self.dim} is not 16, 32, 64 or 128")
        _need(16 <= self.page <= 1024 and self.page & (self.page - 1) == 0,
              f"page {self.page} is not a power of two from 16 to 1024")
        _need(self.q8 == (k_scale is not None) == (v_scale is not None), "an int8 cache needs both scales, a float16 one none")
        kp, vp = _cuda(k, "k", k.dtype), _cuda(v, "v", k.dtype, k.shape, k.device)
        ks = _cuda(k_scale, "k_scale", torch.float32, k.shape[:3], k.device) if self.q8 else None
        vs = _cuda(v_scale, "v_scale", torch.float32, k.shape[:3], k.device) if self.q8 else None
        self._c = _lib.Kv(kp, vp, ks, vs, self.pages, self.heads, self.page, self.dim, int(self.q8))
        self._ref = ctypes.byref(self._c)
        self._scale = self.dim ** -0.5
        self._lib = _lib.load()

    @classmethod
    def empty(cls, pages: int, heads: int, page: int, dim: int, format: str = "f16", device="cuda") -> "PagedKV":
        """A new cache of zeros; format "f16" or "q8"."""
        _need(format in ("f16", "q8"), f"unknown cache format {format!r}")
        shape = (pages, heads, page, dim)
        dtype = torch.float16 if format == "f16" else torch.int8
        data = [torch.zeros(shape, dtype=dtype, device=device) for _ in range(2)]
        scales = [torch.zeros(shape[:3], dtype=torch.float32, device=device) for _ in range(2)] if format == "q8" else []
        return cls(*data, *scales)

    def _check(self, seqs: Seqs) -> None:
        if seqs.index != self.index:
            raise ValueError(f"the sequences are on {seqs.device}, the cache on {self.device}")

    def write(self, seqs: Seqs, k: torch.Tensor, v: torch.Tensor) -> None:
        """Writes the new tokens' rows k, v [tokens, heads, dim] into their pages."""
        self._check(seqs)
        ck, cv = _rows(k, "k", self.index, self.dim), _rows(v, "v", self.index, self.dim)
        _call(self.index, self._lib.mgb_kv_write, self._ref, seqs._ref, ctypes.byref(ck), ctypes.byref(cv))

    def read(self, seqs: Seqs, dtype: torch.dtype = torch.float16,
             out: tuple[torch.Tensor, torch.Tensor] | None = None) -> tuple[torch.Tensor, torch.Tensor]:
        """The values at every sequence's last q_start[b + 1] - q_start[b] positions, as packed rows
        [tokens, heads, dim] of K and of V (q_start = the running sum of kv_len reads everything).
        Into out = (K, V) where given, else into new tensors of seqs.tokens rows."""
        self._check(seqs)
        if out is None:
            if seqs.tokens is None:
                raise ValueError("read needs out, or sequences that know their number of tokens")
            k = self.k.new_empty((seqs.tokens, self.heads, self.dim), dtype=dtype)
            v = torch.empty_like(k)
        else:
            k, v = out
        ck, cv = _rows(k, "k", self.index, self.dim), _rows(v, "v", self.index, self.dim)
        _call(self.index, self._lib.mgb_kv_read, self._ref, seqs._ref, ctypes.byref(ck), ctypes.byref(cv))
        return k, v

    def attend(self, seqs: Seqs, q: torch.Tensor, scale: float | None = None, causal: bool = True,
               out: torch.Tensor | None = None) -> torch.Tensor:
        """Attention of the new tokens' queries q [tokens, query heads, dim] over their sequences:
        softmax(scale * q k) v, scale 1 / sqrt(dim) unless given. Query head h reads cache head
        h // (query heads / heads). causal: a token sees the positions up to its own, else all of its
        sequence. A token that sees nothing gets zeros, and so does a row of no sequence. Returns out (q's
        type and shape unless given). Sums are held in f32; with float16 or bfloat16 q each key's weight counts
        to 2^-11 of itself, with float32 q to 2^-21."""
        self._check(seqs)
        cq = _rows(q, "q", self.index, self.dim)
        if out is None:
            out = torch.empty_like(q, memory_format=torch.contiguous_format)
            heads = cq.heads
            co = _lib.Rows(out.data_ptr(), heads * self.dim, self.dim, cq.tokens, heads, cq.type)
        else:
            co = _rows(out, "out", self.index, self.dim)
        _call(self.index, self._lib.mgb_kv_attend, self._ref, seqs._ref, ctypes.byref(cq), ctypes.byref(co),
              self._scale if scale is None else scale, causal)
        if seqs.empty:  # a call that does nothing
            out.zero_()
        return out

    def check(self) -> None:
        """Waits for the current stream's work and raises MgbError if an attention on this GPU gave up a wait
        inside its kernel since the last check: some rows that it wrote are NaN then."""
        _call(self.index, self._lib.mgb_kv_status)


class LogitRules:
    """Rules on the logits of a batch of rows; every part may be absent.

    history [rows, n] int32, history_len [rows] int32 (all n if absent): the
        tokens that the penalties count. With c > 0 occurrences of a token,
        repetition[r] divides its positive logit and multiplies a negative one,
        then frequency[r] * c + presence[r] is subtracted.
    bias_ids, bias [rows, m] int32 / float32: added to those tokens' logits
        (pad with id -1; a token's several entries add up).
    allow [grammars, words] int32 bit rows, allow_row [rows] int32: row r may
        choose only tokens t with bit t % 32 of allow[allow_row[r], t // 32]
        set; -1 means any token. Without allow_row every row follows allow[0].
    """

    def __init__(self, history: torch.Tensor | None = None, history_len: torch.Tensor | None = None,
                 repetition: torch.Tensor | None = None, frequency: torch.Tensor | None = None,
                 presence: torch.Tensor | None = None, bias_ids: torch.Tensor | None = None,
                 bias: torch.Tensor | None = None, allow: torch.Tensor | None = None,
                 allow_row: torch.Tensor | None = None):
        _need((bias_ids is None) == (bias is None), "bias_ids and bias come together")
        _need(history is not None or (history_len is None and repetition is None and frequency is None and presence is None),
              "penalties need a history")
        _need(allow is not None or allow_row is None, "allow_row needs allow")
        per_row = [x for x in (history, history_len, repetition, frequency, presence, bias_ids, bias, allow_row)
                   if x is not None]
        self.rows = per_row[0].size(0) if per_row else None  # None: any number of rows
        self.device = per_row[0].device if per_row else allow.device if allow is not None else None
        self.index = None if self.device is None else (per_row[0] if per_row else allow).get_device()
        self.tensors = (history, history_len, repetition, frequency, presence, bias_ids, bias, allow, allow_row)
        n, dev = self.rows, self.device

        def vec(x, name, dtype):
            return None if x is None else _cuda(x, name, dtype, (n,), dev)

        def mat(x, name, dtype, rows):
            if x is None:
                return None
            _need(x.dim() == 2 and rows in (None, x.size(0)), f"{name} must be two-dimensional with a row for every row")
            return _cuda(x, name, dtype, None, dev)

        if bias is not None:
            _need(bias.shape == bias_ids.shape, "bias_ids and bias differ in shape")
        self.words = allow.size(1) if allow is not None else 0
        self._c = _lib.LogitRules(
            mat(history, "history", torch.int32, n), vec(history_len, "history_len", torch.int32),
            vec(repetition, "repetition", torch.float32), vec(frequency, "frequency", torch.float32),
            vec(presence, "presence", torch.float32), mat(bias_ids, "bias_ids", torch.int32, n),
            mat(bias, "bias", torch.float32, n), mat(allow, "allow", torch.int32, None),
            vec(allow_row, "allow_row", torch.int32), history.size(1) if history is not None else 0,
            bias_ids.size(1) if bias_ids is not None else 0, allow.size(0) if allow is not None else 0, self.words)
        self._ref = ctypes.byref(self._c)
        self._lib = _lib.load()

    def choose(self, logits: torch.Tensor, adjusted: torch.Tensor | None = None):
        """Applies the rules to logits [rows, vocab] (float32, float16 or bfloat16) and returns per row
        the token with the largest result (the lowest on ties; int32, -1 where nothing may be chosen)
        and its log-probability (float32) among the results. adjusted, of the logits' type and shape,
        gets the results themselves and comes back as a third value; it may be the logits."""
        kind, shape, strides = _TYPES.get(logits.dtype), logits.shape, logits.stride()
        if kind is None:
            raise ValueError("logits must be float32, float16 or bfloat16")
        if len(shape) != 2 or not logits.is_cuda or strides[1] != 1:
            raise ValueError("logits must be [rows, vocab] on a GPU with contiguous rows")
        index, (rows, vocab) = logits.get_device(), shape
        if self.rows is not None and self.rows != rows:
            raise ValueError(f"the rules are for {self.rows} rows, the logits have {rows}")
        if self.index is not None and self.index != index:
            raise ValueError(f"the rules are on GPU {self.index}, the logits on {logits.device}")
        y, y_stride = None, 0
        if adjusted is not None:
            if (adjusted.dtype != logits.dtype or adjusted.shape != shape or adjusted.get_device() != index
                    or adjusted.stride(1) != 1):
                raise ValueError("adjusted must be like the logits")
            y, y_stride = adjusted.data_ptr(), adjusted.stride(0)
        ids = logits.new_empty((rows,), dtype=torch.int32)
        logp = torch.empty_like(ids, dtype=torch.float32)
        _call(index, self._lib.mgb_logits_choose, logits.data_ptr(), kind, strides[0], rows, vocab, self._ref,
              ids.data_ptr(), logp.data_ptr(), y, y_stride)
        return (ids, logp) if adjusted is None else (ids, logp, adjusted)
