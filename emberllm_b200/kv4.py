"""The many-stream operators of include/ember_kv4.h on device arrays: the paged
4-bit KV cache (``Kv4Cache``: store, read, attention) and one draw per row of a
batch of logits (``sample_rows``).

Arrays are CUDA tensors as torch makes them (anything with ``data_ptr``,
``shape``, ``stride()``, ``dtype`` and ``device`` works; this module does not
import torch). The caller owns every buffer; a call allocates nothing and enqueues
its work on ``stream`` (a cudaStream_t as an integer; 0 is the default stream).
None, the default, is the stream that torch's own operations on these tensors would take
now (torch.cuda.current_stream), or 0 for arrays of others.
Arguments that do not fit raise ValueError; what the library refuses raises
RuntimeError with its message.
"""
import struct
import sys

from . import _lib as _libmod

# the structures of include/ember_kv4.h in native layout, packed per call: a ctypes
# Structure of 14 fields costs a call a microsecond more
_CACHE = struct.Struct("@Piiii")                # EmberKv4Cache
_BATCH = struct.Struct("@PPPiiii")              # EmberKv4Batch
_ROWS = struct.Struct("@PPi4xqqqq")             # EmberKv4Rows
_ATT = struct.Struct("@PPiiqqqqfiiiPN")       # EmberKv4Attention
_SAMPLE = struct.Struct("@PiiiqPPPPPP")         # EmberSampleRows


class _Dtypes(dict):
    """the library's code of a dtype object, by its name"""

    def __missing__(self, dtype):
        self[dtype] = code = {"torch.float32": 0, "torch.float16": 3, "torch.int32": -32}.get(str(dtype))
        return code


_DT = _Dtypes()
_F32, _I32 = 0, -32


_torch = None          # (its Tensor, its current stream of a device), once it is there


def _on(stream, t):
    """the stream a call on array t goes to"""
    global _torch
    if stream is not None:
        return stream
    if _torch is None:
        m = sys.modules.get("torch")
        if m is None:
            return 0
        # (the public call makes an object of the stream: a microsecond more)
        _torch = m.Tensor, getattr(m._C, "_cuda_getCurrentRawStream",
                                   lambda i: m.cuda.current_stream(i).cuda_stream)
    device = t.get_device() if isinstance(t, _torch[0]) else -1
    return _torch[1](device) if device >= 0 else 0


def _fail():
    raise RuntimeError(_libmod.load().ember_cuda_error().decode())


def _too_large(e):
    return ValueError(f"a number does not fit its field: {e}")


def _dtype(t, name):
    d = _DT[t.dtype]
    if d is None or d < 0:
        raise ValueError(f"{name} must be float32 or float16, not {t.dtype}")
    return d


def _array(t, name, dtype, n):
    """pointer of a contiguous array of n elements of `dtype`"""
    if _DT[t.dtype] != dtype or t.shape != (n,) or (n > 1 and t.stride(0) != 1):
        raise ValueError(f"{name} must be a contiguous {'float32' if dtype == _F32 else 'int32'} array of {n}")
    return t.data_ptr()


def _rows(t, name, heads, head_dim):
    """strides (row, head) of a [rows][heads][head_dim] tensor"""
    s = t.shape
    if len(s) != 3 or s[1] != heads or s[2] != head_dim:
        raise ValueError(f"{name} must be [rows][{heads}][{head_dim}], not {list(s)}")
    st = t.stride()
    if st[2] != 1:
        raise ValueError(f"{name}: a head's elements must be consecutive")
    return st[0], st[1]


class Kv4Cache:
    """One layer's paged cache in 4 bits over the caller's device buffer."""

    @staticmethod
    def nbytes(n_pages, page_size, n_kv_heads, head_dim):
        """bytes of the buffer such a cache needs"""
        sizes = (int(n_pages), int(page_size), int(n_kv_heads), int(head_dim))
        n = max(sizes) < 2 ** 31 and min(sizes) > 0 and _libmod.load().ember_cuda_kv4_bytes(*sizes)
        if not n:
            raise ValueError(f"a cache of {n_pages} pages of {page_size} positions, {n_kv_heads} kv heads of {head_dim} "
                             "is not supported")
        return n

    def __init__(self, buffer, n_pages, page_size, n_kv_heads, head_dim):
        n_pages, page_size, n_kv_heads, head_dim = int(n_pages), int(page_size), int(n_kv_heads), int(head_dim)
        need = Kv4Cache.nbytes(n_pages, page_size, n_kv_heads, head_dim)
        if not buffer.is_contiguous() or buffer.numel() * buffer.element_size() < need:
            raise ValueError(f"the cache needs a contiguous buffer of {need} bytes")
        self.lib = _libmod.load()
        self.buffer = buffer            # kept alive
        self.page_size, self.n_kv_heads, self.head_dim = page_size, n_kv_heads, head_dim
        self._p = _CACHE.pack(buffer.data_ptr(), n_pages, page_size, n_kv_heads, head_dim)

    def _batch(self, tokens, q_start, kv_len, block_table, max_q):
        n, ts = kv_len.shape, block_table.shape
        n = n[0] if n else -1
        if len(ts) != 2 or ts[0] != n or _DT[block_table.dtype] != _I32:
            raise ValueError(f"block_table must be an int32 [{n}][pages] array")
        if not block_table.is_contiguous():
            raise ValueError("block_table must be contiguous")
        return _BATCH.pack(0 if q_start is None else _array(q_start, "q_start", _I32, n + 1),
                           _array(kv_len, "kv_len", _I32, n), block_table.data_ptr(), n, ts[1], tokens, max_q)

    def _io(self, fn, k, v, q_start, kv_len, block_table, max_q, stream):
        k_tok, k_head = _rows(k, "k", self.n_kv_heads, self.head_dim)
        v_tok, v_head = _rows(v, "v", self.n_kv_heads, self.head_dim)
        if k.shape[0] != v.shape[0] or k.dtype != v.dtype:
            raise ValueError("k and v must have the same rows and type")
        try:
            batch = self._batch(k.shape[0], q_start, kv_len, block_table, max_q)
            rows = _ROWS.pack(k.data_ptr(), v.data_ptr(), _dtype(k, "k"), k_tok, k_head, v_tok, v_head)
        except struct.error as e:
            raise _too_large(e) from None
        if fn(self._p, batch, rows, _on(stream, k)):
            _fail()

    def store(self, k, v, q_start, kv_len, block_table, max_q=1, stream=None):
        """Quantize the rows' keys and values ([rows][kv heads][head_dim]) into the
        cache: rows q_start[i]..q_start[i+1]-1 are the last positions of sequence i's
        kv_len[i]. ``q_start`` None: one row per sequence. ``max_q``: the most rows
        any sequence has."""
        self._io(self.lib.ember_cuda_kv4_store, k, v, q_start, kv_len, block_table, max_q, stream)

    def read(self, k, v, q_start, kv_len, block_table, max_q=1, stream=None):
        """The inverse of ``store``: the cached values of the rows' positions into k
        and v."""
        self._io(self.lib.ember_cuda_kv4_read, k, v, q_start, kv_len, block_table, max_q, stream)

    def attention_workspace(self, n_heads, n_seqs, max_q, max_kv):
        """bytes of workspace an attention call of these sizes needs (may be 0)"""
        return self.lib.ember_cuda_kv4_attention_workspace(self._p, n_heads, n_seqs, max_q, max_kv)

    def attention(self, q, out, q_start, kv_len, block_table, max_q=1, max_kv=None, scale=None, window=0, sinks=0,
                  workspace=None, stream=None):
        """Causal attention of the rows' queries ([rows][heads][head_dim]) over the
        cache into ``out``; ``window`` > 0 limits it to the last ``window`` positions
        and the first ``sinks``. ``max_kv`` bounds kv_len (default: all the block table
        can hold), ``scale`` defaults to head_dim ** -0.5."""
        shape = q.shape
        heads = shape[1] if len(shape) > 1 else 0
        q_tok, q_head = _rows(q, "q", heads, self.head_dim)
        out_tok, out_head = _rows(out, "out", heads, self.head_dim)
        if shape[0] != out.shape[0] or q.dtype != out.dtype:
            raise ValueError("q and out must have the same rows and type")
        if max_kv is None:
            max_kv = min(block_table.shape[1] * self.page_size, 2 ** 31 - 1)
        ws, nws = 0, 0
        if workspace is not None:
            if not workspace.is_contiguous():      # (its bytes need not be there)
                raise ValueError("workspace must be contiguous")
            ws, nws = workspace.data_ptr(), workspace.nbytes
        try:
            batch = self._batch(shape[0], q_start, kv_len, block_table, max_q)
            att = _ATT.pack(q.data_ptr(), out.data_ptr(), _dtype(q, "q"), heads, q_tok, q_head, out_tok, out_head,
                            self.head_dim ** -0.5 if scale is None else scale, max_kv, window, sinks, ws, nws)
        except struct.error as e:
            raise _too_large(e) from None
        if self.lib.ember_cuda_kv4_attention(self._p, batch, att, _on(stream, q)):
            _fail()

    def check(self, stream=None):
        """Wait for the stream's work; RuntimeError when a device wait of an attention
        call has run out since the last check (its rows are NaN)."""
        if self.lib.ember_cuda_kv4_status(self._p, _on(stream, self.buffer)):
            _fail()


def sample_rows(logits, out, u, temperature=None, top_k=None, top_p=None, min_p=None, stream=None):
    """Draw one token per row of ``logits`` [rows][vocab] into ``out`` (int32), with
    each row's own random number ``u`` in [0, 1) and settings (float32 arrays,
    ``top_k`` int32; None: temperature 1, no truncation). See
    ember_cuda_sample_rows for the exact definition."""
    lib = _libmod.load()
    if logits.ndim != 2 or (logits.shape[1] > 1 and logits.stride()[1] != 1):
        raise ValueError("logits must be [rows][vocab] with consecutive elements")
    n = logits.shape[0]

    def opt(t, name, dtype=_F32):
        return 0 if t is None else _array(t, name, dtype, n)
    if lib.ember_cuda_sample_rows(
            _SAMPLE.pack(logits.data_ptr(), _dtype(logits, "logits"), n, logits.shape[1], logits.stride(0),
                         opt(temperature, "temperature"), opt(top_p, "top_p"), opt(min_p, "min_p"),
                         _array(u, "u", _F32, n), opt(top_k, "top_k", _I32), _array(out, "out", _I32, n)), _on(stream, logits)):
        _fail()
