"""One step of several sequences over quantized KV pages.

The engine's ``CudaChatModel`` decodes one sequence over its own float KV
cache. This module has what a step of several requests does around the
packed projections (``Weight.gemv`` / ``Weight.gemm_rows``):

  * ``KVPool`` -- int8 or int4 KV pages in a caller-owned byte tensor:
    ``append`` (per-head RMSNorm of queries and keys, RoPE and the quantizing
    write in one pass), ``attend`` (decode rows, drafted rows and prompt
    chunks in one call; tanh cap, distance bias, window, prefix) and ``read``
    (rows back as floats);
  * ``SeqBatch`` -- the step's sequences: row offsets, lengths, page table;
  * ``adjust_logits`` -- penalties, biases, grammar mask and argmax.

The arithmetic and the pool's layout are declared in ``lumina_cuda.h``. All
calls take CUDA tensors, run on the current stream of the pool's device and
return without waiting; a batch whose device data is out of range sets bit
64 of ``cuda.fault_status``. Errors raise ``LuminaError``; there is no CPU
path.
"""
from __future__ import annotations

import ctypes

import torch

from . import cuda
from .cuda import LuminaError, check

FAULT_WAIT, FAULT_DATA = 32, 64
_TYPES = {torch.float32: 0, torch.float16: 1}
_VP, _I, _SZ, _F = ctypes.c_void_p, ctypes.c_int, ctypes.c_size_t, ctypes.c_float


class _Pool(ctypes.Structure):
    _fields_ = [("pool_dev", _VP), ("device", _I), ("bits", _I), ("n_pages", _I), ("n_kv", _I), ("head_dim", _I),
                ("page_size", _I)]


class _Batch(ctypes.Structure):
    _fields_ = [("row_start_dev", _VP), ("len_dev", _VP), ("pages_dev", _VP), ("pages_ld", _I), ("n_seq", _I),
                ("n_rows", _I), ("max_rows", _I)]


class _Attend(ctypes.Structure):
    _fields_ = [("q_dev", _VP), ("out_dev", _VP), ("ldq", _I), ("ldo", _I), ("type", _I), ("n_heads", _I),
                ("scale", _F), ("softcap", _F), ("slopes_dev", _VP), ("prefix_dev", _VP), ("window", _I),
                ("workspace_dev", _VP), ("workspace_bytes", _SZ)]


class _Logits(ctypes.Structure):
    _fields_ = [("logits_dev", _VP), ("out_dev", _VP), ("ld", _I), ("ldo", _I), ("rows", _I), ("vocab", _I),
                ("hist_start_dev", _VP), ("hist_tok_dev", _VP), ("hist_len", _I), ("repeat_dev", _VP),
                ("frequency_dev", _VP), ("presence_dev", _VP), ("bias_start_dev", _VP), ("bias_tok_dev", _VP),
                ("bias_val_dev", _VP), ("bias_len", _I), ("mask_dev", _VP), ("mask_ld", _I), ("argmax_dev", _VP),
                ("device", _I)]


def _bad(text: str):
    raise LuminaError(1, text)


def _lib(device: int) -> ctypes.CDLL:
    return _LIBS.get(device) or _LIBS.setdefault(device, cuda.ensure_device(device))


_LIBS: dict[int, ctypes.CDLL] = {}


def _stream(device: int) -> int:
    return torch._C._cuda_getCurrentRawStream(device)


def _vec(t, dtype, device, name, n=None):
    """A contiguous 1-D (or row-major) tensor of ``dtype`` on the device."""
    if t.dtype is not dtype or t.get_device() != device or not t.is_contiguous() or (n is not None and t.numel() != n):
        _bad("%s: %s%s on %s, a contiguous %s of %s elements on cuda:%d is needed"
             % (name, t.dtype, tuple(t.shape), t.device, dtype, "any" if n is None else n, device))
    return t.data_ptr()


def _rows(t, dtype, device, n, width, name):
    """Rows of ``width`` contiguous elements: (n, width) or (n, heads, dim)
    with the heads side by side. Returns the row stride."""
    if t.dim() < 2 or t.dtype is not dtype or t.get_device() != device or t.shape[0] != n:
        _bad("%s: %s%s on %s, %d rows of %s on cuda:%d are needed" % (name, t.dtype, tuple(t.shape), t.device, n, dtype, device))
    st = t.stride()
    if t.dim() == 2:
        ok = t.shape[1] == width and st[1] == 1
    else:
        ok = t.dim() == 3 and t.shape[1] * t.shape[2] == width and st[2] == 1 and (st[1] == t.shape[2] or t.shape[1] == 1)
    if not ok:
        _bad("%s: shape %s strides %s, rows of %d contiguous elements are needed" % (name, tuple(t.shape), st, width))
    return st[0] if n > 1 else width


class SeqBatch:
    """The sequences of one step. ``row_start`` (n_seq + 1) int32: sequence s
    owns activation rows row_start[s] .. row_start[s+1] - 1, its last ones;
    ``lens`` (n_seq) int32: its cached tokens, those rows included; ``pages``
    (n_seq, ld) int32: its page table. ``n_rows`` = row_start[-1] and
    ``max_rows`` (the most rows of one sequence) are host numbers, so that
    nothing here waits for the GPU. The tensors may be rewritten in place
    between steps (a captured graph reads them anew)."""

    __slots__ = ("c", "n_seq", "n_rows", "max_rows", "device", "_keep")

    def __init__(self, row_start, lens, pages, n_rows: int, max_rows: int):
        n = lens.numel()
        dev = lens.get_device()
        if dev < 0 or pages.dim() != 2 or pages.shape[0] != n:
            _bad("SeqBatch: CUDA tensors and a page table of %d rows are needed, got %s on %s" % (n, tuple(pages.shape), lens.device))
        self.c = _Batch(_vec(row_start, torch.int32, dev, "row_start", n + 1), _vec(lens, torch.int32, dev, "lens"),
                        _vec(pages, torch.int32, dev, "pages"), pages.shape[1], n, n_rows, max_rows)
        self.n_seq, self.n_rows, self.max_rows, self.device = n, n_rows, max_rows, dev
        self._keep = (row_start, lens, pages)


_WORKSPACES: dict[tuple[int, int], torch.Tensor] = {}


def _capturing(device: int) -> bool:
    """Whether the device's current stream is being captured into a graph."""
    if device == torch.cuda.current_device():
        return torch.cuda.is_current_stream_capturing()
    with torch.cuda.device(device):
        return torch.cuda.is_current_stream_capturing()


def attend_workspace(device: int = 0) -> torch.Tensor:
    """A zeroed workspace for ``KVPool.attend``: one for each stream and each
    captured graph whose calls may run at the same time as another's. Make it
    outside any capture (the zeros have to be there before the first replay)
    and keep it as long as the graph."""
    n = _SZ()
    check(_lib(device).lumina_kvq_workspace_bytes(device, ctypes.byref(n)))
    return torch.zeros(n.value, dtype=torch.uint8, device="cuda:%d" % device)


class KVPool:
    """Quantized KV pages: ``data`` is a caller-owned uint8 tensor (n_pages,
    n_kv, block_bytes) on the GPU, ``block_bytes`` from ``KVPool.block_bytes``
    (``KVPool.empty`` makes one)."""

    __slots__ = ("data", "c", "bits", "head_dim", "page_size", "n_kv", "n_pages", "device", "lib")

    def __init__(self, data: torch.Tensor, bits: int, head_dim: int, page_size: int = 16):
        if data.dtype is not torch.uint8 or data.dim() != 3 or not data.is_contiguous() or data.get_device() < 0:
            _bad("KVPool: a contiguous uint8 CUDA tensor (n_pages, n_kv, block_bytes) is needed, got %s%s on %s"
                 % (data.dtype, tuple(data.shape), data.device))
        want = page_size * (2 * (head_dim * bits // 8) + 8)
        if data.shape[2] != want:
            _bad("KVPool: blocks of %d bytes, %d for %d bits, head dim %d and %d tokens" % (data.shape[2], want, bits, head_dim, page_size))
        self.data, self.bits, self.head_dim, self.page_size = data, bits, head_dim, page_size
        self.n_pages, self.n_kv, self.device = data.shape[0], data.shape[1], data.get_device()
        self.lib = _lib(self.device)
        self.c = _Pool(data.data_ptr(), self.device, bits, self.n_pages, self.n_kv, head_dim, page_size)

    @staticmethod
    def block_bytes(bits: int, head_dim: int, page_size: int = 16) -> int:
        n = _SZ()
        check(cuda.bound_lib().lumina_kvq_block_bytes(bits, head_dim, page_size, ctypes.byref(n)))
        return n.value

    @classmethod
    def empty(cls, n_pages: int, n_kv: int, head_dim: int, bits: int = 8, page_size: int = 16, device: int = 0) -> "KVPool":
        n = cls.block_bytes(bits, head_dim, page_size)
        return cls(torch.empty(n_pages, n_kv, n, dtype=torch.uint8, device="cuda:%d" % device), bits, head_dim, page_size)

    def _batch(self, batch: SeqBatch):
        if batch.device != self.device:
            _bad("batch on cuda:%d, pool on cuda:%d" % (batch.device, self.device))
        return ctypes.byref(batch.c)

    def _type(self, t, name):
        code = _TYPES.get(t.dtype)
        if code is None:
            _bad("%s: %s, float32 or float16 is needed" % (name, t.dtype))
        return code

    def _width(self, q):
        width = q.shape[1] if q.dim() == 2 else q.shape[1] * q.shape[2] if q.dim() == 3 else 0
        if width == 0 or width % self.head_dim:
            _bad("q: shape %s, rows of a multiple of head dim %d are needed" % (tuple(q.shape), self.head_dim))
        return width

    def append(self, batch: SeqBatch, q, k, v, cos, sin, q_norm=None, k_norm=None, eps: float = 1e-6, out=None):
        """Write the batch's new rows: q (n_rows, heads, head_dim), k and v
        (n_rows, n_kv, head_dim) -- or the same as 2-D column ranges of one
        fused projection. Queries and keys are normalized per head when
        ``q_norm`` / ``k_norm`` are given and rotated with row ``position`` of
        ``cos`` / ``sin`` (n_pos, head_dim / 2). Returns the rotated queries."""
        b, hd, dev, n = self._batch(batch), self.head_dim, self.device, batch.n_rows
        dt, ty = q.dtype, self._type(q, "q")
        width = self._width(q)
        ldq = _rows(q, dt, dev, n, width, "q")
        ldk = _rows(k, dt, dev, n, self.n_kv * hd, "k")
        ldv = _rows(v, dt, dev, n, self.n_kv * hd, "v")
        if out is None:
            out = torch.empty((n, width // hd, hd), dtype=dt, device=q.device)
        ldo = _rows(out, dt, dev, n, width, "out")
        if cos.dim() != 2 or cos.shape[1] * 2 != hd or sin.shape != cos.shape:
            _bad("cos / sin: %s / %s, (n_pos, %d) is needed" % (tuple(cos.shape), tuple(sin.shape), hd // 2))
        check(self.lib.lumina_kvq_append(
            ctypes.byref(self.c), b, q.data_ptr(), ldq, k.data_ptr(), ldk, v.data_ptr(), ldv, ty, width // hd,
            None if q_norm is None else _vec(q_norm, torch.float32, dev, "q_norm", hd),
            None if k_norm is None else _vec(k_norm, torch.float32, dev, "k_norm", hd), eps,
            _vec(cos, torch.float32, dev, "cos"), _vec(sin, torch.float32, dev, "sin"), cos.shape[0],
            out.data_ptr(), ldo, _stream(dev)), self.lib)
        return out

    def read(self, batch: SeqBatch, dtype=torch.float32, out=None):
        """K and V (n_rows, n_kv, head_dim) of the batch's rows as the pool
        holds them; a batch whose sequences own ``lens`` rows reads them
        whole. ``out``: the two tensors to fill."""
        b, dev, n, w = self._batch(batch), self.device, batch.n_rows, self.n_kv * self.head_dim
        if out is None:
            out = tuple(torch.empty((n, self.n_kv, self.head_dim), dtype=dtype, device="cuda:%d" % dev) for _ in range(2))
        k, v = out
        ld = _rows(k, k.dtype, dev, n, w, "k")
        if _rows(v, k.dtype, dev, n, w, "v") != ld:
            _bad("read: k and v have different row strides")
        check(self.lib.lumina_kvq_read(ctypes.byref(self.c), b, k.data_ptr(), v.data_ptr(), ld, self._type(k, "out"),
                                       _stream(dev)), self.lib)
        return out

    def attend(self, batch: SeqBatch, q, scale: float = 0.0, softcap: float = 0.0, slopes=None, window: int = 0,
               prefix=None, out=None, workspace=None):
        """Attention of the batch's rows q (n_rows, heads, head_dim) over
        their sequences' pages (rows already appended). Key j is visible to a
        row at position p when j <= p and j > p - ``window`` (0: no limit), or
        when j < ``prefix[s]`` (n_seq, int32). ``scale`` 0 means 1 /
        sqrt(head_dim); ``softcap`` c > 0 turns scores into c tanh(x / c);
        ``slopes`` (heads, float32) subtract slope * |p - j|. A row that sees
        nothing gives zeros. ``workspace``: ``attend_workspace(device)``, by
        default one of about 50 MB that this module makes for each stream at its
        first call and keeps. While a graph is captured there is no default:
        a graph's calls need a workspace that is theirs at every replay."""
        b, hd, dev, n = self._batch(batch), self.head_dim, self.device, batch.n_rows
        dt, ty = q.dtype, self._type(q, "q")
        width = self._width(q)
        ldq = _rows(q, dt, dev, n, width, "q")
        if out is None:
            out = torch.empty((n, width // hd, hd), dtype=dt, device=q.device)
        ldo = _rows(out, dt, dev, n, width, "out")
        stream = _stream(dev)
        if workspace is None:
            if _capturing(dev):
                _bad("attend: a captured call needs a workspace of its own (attend_workspace, made outside the capture)")
            workspace = _WORKSPACES.get((dev, stream))
            if workspace is None:
                workspace = _WORKSPACES[(dev, stream)] = attend_workspace(dev)
            ws = workspace.data_ptr()
        else:
            ws = _vec(workspace, torch.uint8, dev, "workspace")
        a = _Attend(q.data_ptr(), out.data_ptr(), ldq, ldo, ty, width // hd, scale, softcap,
                    None if slopes is None else _vec(slopes, torch.float32, dev, "slopes", width // hd),
                    None if prefix is None else _vec(prefix, torch.int32, dev, "prefix", batch.n_seq), window,
                    ws, workspace.numel())
        check(self.lib.lumina_kvq_attend(ctypes.byref(self.c), b, ctypes.byref(a), stream), self.lib)
        return out


def adjust_logits(logits, history=None, repeat=None, frequency=None, presence=None, bias=None, mask=None, out=None,
                  argmax=True):
    """Shape logits rows (rows, vocab) float32 and pick the largest.

    ``history`` = (offsets (rows + 1) int32, tokens int32): for each token
    that occurs c times in the row's slice, l / ``repeat`` if l > 0 else l *
    ``repeat``, then minus ``frequency`` * c + ``presence`` (each (rows)
    float32). All three go by the same history: for a repetition over prompt
    and output and the others over the output alone, call twice, in place.
    ``bias`` = (offsets, tokens, float32 values) is added (a token listed
    twice takes its last entry). ``mask`` (rows, words) int32: bit t % 32 of
    word t // 32 is 0 for a forbidden token, which becomes -inf.
    Returns (out, argmax (rows) int32); ``out`` may be ``logits`` itself,
    ``argmax`` a tensor to fill, or False for none."""
    if logits.dim() != 2 or logits.dtype is not torch.float32 or logits.get_device() < 0:
        _bad("logits: %s%s on %s, float32 (rows, vocab) on the GPU is needed" % (logits.dtype, tuple(logits.shape), logits.device))
    R, V = logits.shape
    dev = logits.get_device()
    lib = _lib(dev)
    if out is None:
        out = torch.empty_like(logits, memory_format=torch.contiguous_format)
    if argmax is True:
        argmax = torch.empty(R, dtype=torch.int32, device=logits.device)
    a = _Logits(logits.data_ptr(), out.data_ptr(), _rows(logits, torch.float32, dev, R, V, "logits"),
                _rows(out, torch.float32, dev, R, V, "out"), R, V)
    a.device = dev
    if history is not None and history[1].numel():
        a.hist_start_dev = _vec(history[0], torch.int32, dev, "history offsets", R + 1)
        a.hist_tok_dev = _vec(history[1], torch.int32, dev, "history tokens")
        a.hist_len = history[1].numel()
    if repeat is not None:
        a.repeat_dev = _vec(repeat, torch.float32, dev, "repeat", R)
    if frequency is not None:
        a.frequency_dev = _vec(frequency, torch.float32, dev, "frequency", R)
    if presence is not None:
        a.presence_dev = _vec(presence, torch.float32, dev, "presence", R)
    if bias is not None and bias[1].numel():
        a.bias_start_dev = _vec(bias[0], torch.int32, dev, "bias offsets", R + 1)
        a.bias_tok_dev = _vec(bias[1], torch.int32, dev, "bias tokens")
        a.bias_val_dev = _vec(bias[2], torch.float32, dev, "bias values", bias[1].numel())
        a.bias_len = bias[1].numel()
    if mask is not None:
        if mask.dim() != 2 or mask.shape[0] != R:
            _bad("mask: %s, (%d, words) is needed" % (tuple(mask.shape), R))
        a.mask_dev = _vec(mask, torch.int32, dev, "mask")
        a.mask_ld = mask.shape[1]
    if argmax is not False:
        a.argmax_dev = _vec(argmax, torch.int32, dev, "argmax", R)
    check(lib.lumina_logits_adjust(ctypes.byref(a), _stream(dev)), lib)
    return out, (None if argmax is False else argmax)
