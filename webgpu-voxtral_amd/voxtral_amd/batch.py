"""Operators for batches that decode together, on tensors in GPU memory
(vx_paged_append, vx_paged_attend and vx_sample_rows of
include/voxtral_engine.h): a paged key/value cache, the attention of a batch
that shares a prefix, and sampling.

Arguments are torch tensors of one GPU.  Calls are enqueued on the stream that
is current for it (`stream`: another one, an object with `cuda_stream` or its
number; the caller then keeps the arguments alive and ready for that stream,
and tensors that the call makes belong to it) and return without waiting.  They can be captured into graphs.  Wrong
shapes, types, strides or devices raise ValueError or TypeError, what the
library refuses raises VoxtralError.  There is no backward pass: tensors that
require gradients are refused while gradients are recorded."""
import ctypes
import struct

from . import VX_OK, VoxtralError, load_library

# the argument structures of the C ABI, in native layout
_KV = struct.Struct("@PPqqqiiiiii")
_APPEND = struct.Struct("@64sPPqqqqPPqqqqPPPqiiiiiidii")
_ATTEND = struct.Struct("@64sPPPqqqqPPPPqiiiiiiiif4xPN")
_SAMPLE = struct.Struct("@PqPPPPPPPPiiiifffiPN")
assert _KV.size == 64

_torch = None
_types = None  # dtype -> VX_TYPE_*
_raw_stream = None


def _load():
    global _torch, _types, _raw_stream
    if _torch is None:
        import torch
        _types = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
        # the number of the current stream, without an object around it (2 us less a call)
        _raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream",
                              lambda index: torch.cuda.current_stream(index).cuda_stream)
        _torch = torch
    return load_library()


def _pack(layout, *args):
    try:
        return layout.pack(*args)
    except struct.error as e:  # a number that its field does not hold
        raise ValueError(f"an argument is out of range: {e}") from None


def _call(fn, *args):
    rc = fn(*args)
    if rc != VX_OK:
        raise VoxtralError(rc, load_library().vx_batch_error().decode())


def _stream(index, stream):
    return _raw_stream(index) if stream is None else getattr(stream, "cuda_stream", stream)


def _made(stream, index, make):
    """make()'s tensor for a call on `stream`: memory is taken from that
    stream's own, since what the current stream has freed it may still be
    using."""
    if stream is None:
        return make()
    if not isinstance(stream, _torch.cuda.Stream):
        number = _stream(index, stream)
        stream = _torch.cuda.ExternalStream(number, index) if number else _torch.cuda.default_stream(index)
    with _torch.cuda.stream(stream):
        return make()


def _refuse(name, x, dims, index):
    """Says what is wrong with x, of which _fits() is not true."""
    if not isinstance(x, _torch.Tensor):
        raise TypeError(f"{name}: a torch tensor is needed, not {type(x).__name__}")
    if x.get_device() != index or index < 0:
        raise ValueError(f"{name} is on {x.device}, not on GPU {index}")
    if x.dim() != dims:
        raise ValueError(f"{name} has {x.dim()} dimensions, not {dims}")
    if x.requires_grad and _torch.is_grad_enabled():
        raise ValueError(f"{name} requires a gradient: this operator has no backward pass")
    raise ValueError(f"{name}: the last dimension is not contiguous")


def _fits(x, dims, index):
    """Whether x is a tensor of `dims` dimensions on GPU `index`, its last one contiguous."""
    if not isinstance(x, _torch.Tensor) or x.get_device() != index or index < 0:
        return False
    st = x.stride()
    return len(st) == dims and (st[-1] == 1 or x.shape[-1] <= 1) and not (x.requires_grad and _torch.is_grad_enabled())


def _tensor(name, x, dims, index):
    if not _fits(x, dims, index):
        _refuse(name, x, dims, index)
    return x


def _vector(name, x, dtype, n, index):
    """The address of a contiguous vector of n elements (None: any number)."""
    if not _fits(x, 1, index):
        _refuse(name, x, 1, index)
    if x.dtype != dtype:
        raise TypeError(f"{name}: {dtype} is needed, not {x.dtype}")
    if n is not None and x.shape[0] != n:
        raise ValueError(f"{name} has {x.shape[0]} elements, not {n}")
    return x.data_ptr()


class PagedKV:
    """A paged cache of one layer: K and V pools [page][kv head][slot][head_dim]
    of float32, float16 or bfloat16, with the same strides.  A sequence's slot
    s is slot s mod page_size of page table[sequence][s // page_size]; which
    pages belong to which sequence is the caller's.  Rows (q, k, v, out) are of
    the pools' type, or float32 for float16 pools."""

    def __init__(self, k_pages, v_pages):
        self._lib = _load()
        self.index = k_pages.get_device() if isinstance(k_pages, _torch.Tensor) else -1
        _tensor("k_pages", k_pages, 4, self.index)
        _tensor("v_pages", v_pages, 4, self.index)
        if v_pages.shape != k_pages.shape or v_pages.stride() != k_pages.stride() or v_pages.dtype != k_pages.dtype:
            raise ValueError("k_pages and v_pages differ in shape, strides or type")
        if k_pages.dtype not in _types:
            raise TypeError(f"k_pages: float32, float16 or bfloat16 is needed, not {k_pages.dtype}")
        self.k_pages, self.v_pages = k_pages, v_pages
        self.n_pages, self.n_kv_heads, self.page_size, self.head_dim = k_pages.shape
        self._int32 = _torch.int32
        self._head = _KV.pack(k_pages.data_ptr(), v_pages.data_ptr(), *k_pages.stride()[:3], self.n_pages, self.page_size,
                              self.n_kv_heads, self.head_dim, _types[k_pages.dtype], self.index)

    def _rows(self, name, x, tokens, heads):
        """The address and the strides of rows [tokens][heads][head_dim] (None: any number)."""
        if not _fits(x, 3, self.index):
            _refuse(name, x, 3, self.index)
        if x.dtype not in _types:
            raise TypeError(f"{name}: float32, float16 or bfloat16 is needed, not {x.dtype}")
        t, h, d = x.shape
        if d != self.head_dim or (tokens is not None and t != tokens) or (heads is not None and h != heads):
            raise ValueError(f"{name} has shape {tuple(x.shape)}, not ({tokens}, {heads}, {self.head_dim})")
        row, head, _ = x.stride()
        return x.data_ptr(), row, head

    def _table(self, table):
        if not _fits(table, 2, self.index):
            _refuse("table", table, 2, self.index)
        if table.dtype != self._int32:
            raise TypeError(f"table: int32 is needed, not {table.dtype}")
        return table.data_ptr(), table.stride(0)

    def append(self, k, v, pos, table, seq=None, base=0, q=None, q_out=None, theta=1e6, rotary_dim=None, interleaved=True,
               stream=None):
        """Writes k and v [tokens][kv heads][head_dim] to the cache, k (and q,
        into q_out) turned by their positions: token t of sequence seq[t]
        (None: t) at position pos[t] goes to the sequence's slot pos[t] -
        base.  rotary_dim: elements that turn (None: all; 0: none).  Tokens
        with a negative pos, a seq outside the table or a slot without a page
        are skipped.  Returns q_out (None without q; made, with zeros for
        skipped tokens, if not given)."""
        k_at, k_row, k_head = self._rows("k", k, None, self.n_kv_heads)
        n = k.shape[0]
        v_at, v_row, v_head = self._rows("v", v, n, self.n_kv_heads)
        table_at, table_row = self._table(table)
        seqs, width = table.shape
        dtype = k.dtype
        if v.dtype != dtype:
            raise TypeError(f"v is {v.dtype}, k is {dtype}")
        heads = q_at = q_row = q_head = o_at = o_row = o_head = 0
        if q is not None:
            q_at, q_row, q_head = self._rows("q", q, n, None)
            heads = q.shape[1]
            if q_out is None:
                q_out = _made(stream, self.index, lambda: q.new_zeros(q.shape))
            o_at, o_row, o_head = self._rows("q_out", q_out, n, heads)
            if q.dtype != dtype or q_out.dtype != dtype:
                raise TypeError(f"q is {q.dtype}, q_out is {q_out.dtype}, k is {dtype}")
        i32 = self._int32
        _call(self._lib.vx_paged_append,
              _pack(_APPEND, self._head, k_at, v_at, k_row, k_head, v_row, v_head, q_at, o_at, q_row, q_head, o_row, o_head,
                    _vector("pos", pos, i32, n, self.index), 0 if seq is None else _vector("seq", seq, i32, n, self.index),
                    table_at, table_row, width, base, n, seqs, heads, _types[dtype], theta,
                    self.head_dim if rotary_dim is None else rotary_dim, bool(interleaved)), _stream(self.index, stream))
        return q_out if q is not None else None

    def attend(self, q, lens, table, row_start=None, prefix_pages=None, prefix_len=0, max_len=None, scale=None, out=None,
               lse=None, workspace=None, stream=None):
        """Attention of a batch that shares a prefix.  q [rows][heads][head_dim]:
        one row a sequence, or rows row_start[s] .. row_start[s + 1] - 1 for
        sequence s, its last ones.  A row sees the prefix_len keys of
        prefix_pages (page ids) and the first lens[s] keys of its sequence's
        own pages, less one for each row of the sequence behind it.  max_len: a
        bound on lens (None: what the table holds); keys from there on are not
        seen.  scale None: 1 / sqrt(head_dim).  lse [rows][heads] float32
        receives the logarithms of the sums of exponentials.  Returns out
        (made if not given, with zeros in rows behind the last sequence).
        workspace: a uint8 tensor of attend_workspace() bytes for this call
        alone (None: made by this call)."""
        q_at, q_row, q_head = self._rows("q", q, None, None)
        n, heads, _ = q.shape
        table_at, table_row = self._table(table)
        seqs, width = table.shape
        i32, index = self._int32, self.index
        lens_at = _vector("lens", lens, i32, seqs, index)
        start = 0 if row_start is None else _vector("row_start", row_start, i32, seqs + 1, index)
        pages, count = 0, 0
        if prefix_pages is not None:
            pages = _vector("prefix_pages", prefix_pages, i32, None, index)
            count = prefix_pages.shape[0]
        if max_len is None:
            max_len = width * self.page_size
        if out is None:
            out = _made(stream, index, lambda: q.new_empty(q.shape) if row_start is None else q.new_zeros(q.shape))
        o_at, o_row, o_head = self._rows("out", out, n, heads)
        if out.dtype != q.dtype:
            raise TypeError(f"out is {out.dtype}, q is {q.dtype}")
        lse_at = 0
        if lse is not None:
            _tensor("lse", lse, 2, index)
            if lse.dtype != _torch.float32 or lse.shape != (n, heads) or not lse.is_contiguous():
                raise ValueError(f"lse: a contiguous float32 tensor of shape ({n}, {heads}) is needed")
            lse_at = lse.data_ptr()
        if scale is None:
            scale = 0.0
        elif scale == 0:
            raise ValueError("scale is 0")
        args = [self._head, q_at, o_at, lse_at, q_row, q_head, o_row, o_head, start, lens_at, table_at, pages, table_row, width, count,
                prefix_len, max_len, n, seqs, heads, _types[q.dtype], scale, 0, 0]
        if workspace is None:
            need = ctypes.c_size_t()
            _call(self._lib.vx_paged_attend_workspace, _pack(_ATTEND, *args), ctypes.byref(need))
            if need.value:
                workspace = _made(stream, index, lambda: table.new_empty((need.value + 3) // 4))
        else:
            _tensor("workspace", workspace, 1, index)
        if workspace is not None:
            args[-2], args[-1] = workspace.data_ptr(), workspace.numel() * workspace.element_size()
        _call(self._lib.vx_paged_attend, _pack(_ATTEND, *args), _stream(index, stream))
        return out

    def attend_workspace(self, rows, heads, seqs, width, ragged=False, prefix_len=0, max_len=None, dtype=None):
        """The bytes of workspace that attend() needs for `rows` query rows of
        `heads` heads, a table of seqs x width pages and these bounds."""
        need = ctypes.c_size_t()
        t = _types[self.k_pages.dtype if dtype is None else dtype]
        args = _pack(_ATTEND, self._head, 0, 0, 0, 0, 0, 0, 0, int(ragged), 0, 0, 0, width, width,
                     -(-prefix_len // self.page_size), prefix_len, width * self.page_size if max_len is None else max_len,
                     rows, seqs, heads, t, 0.0, 0, 0)
        _call(self._lib.vx_paged_attend_workspace, args, ctypes.byref(need))
        return need.value


def sample_rows(logits, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, out=None, stream=None):
    """Draws a token for each row of logits [rows][n] (float32, float16 or
    bfloat16; n up to 2^20) by the uniforms u [rows] (float64, in [0, 1)):
    among the top_k largest (0: all), the largest whose weights reach top_p of
    those' (1: all), and the ones of at least min_p times the largest's weight,
    weights being exp(logit / temperature).  The draw runs along the falling
    logits, equal ones by index.  Each of temperature, top_k, top_p and min_p
    is a number or a tensor [rows] (float32; int32 for top_k); temperature 0
    takes the first of the largest.  Returns (token, kept, prob): int32 ids,
    the numbers of tokens that were left to draw from, and the drawn one's
    probability among them; a row with nothing but NaN and -inf gives (-1, 0,
    0).  out: these three tensors, to write to."""
    lib = _load()
    index = logits.get_device() if isinstance(logits, _torch.Tensor) else -1
    _tensor("logits", logits, 2, index)
    if logits.dtype not in _types:
        raise TypeError(f"logits: float32, float16 or bfloat16 is needed, not {logits.dtype}")
    rows, n = logits.shape
    f32, i32, tensor = _torch.float32, _torch.int32, _torch.Tensor
    t_at = k_at = p_at = m_at = 0
    if isinstance(temperature, tensor):
        t_at, temperature = _vector("temperature", temperature, f32, rows, index), 0
    if isinstance(top_k, tensor):
        k_at, top_k = _vector("top_k", top_k, i32, rows, index), 0
    if isinstance(top_p, tensor):
        p_at, top_p = _vector("top_p", top_p, f32, rows, index), 0
    if isinstance(min_p, tensor):
        m_at, min_p = _vector("min_p", min_p, f32, rows, index), 0
    u_at = _vector("u", u, _torch.float64, rows, index)
    if out is None:
        token, kept, prob = _made(stream, index, lambda: (logits.new_empty(rows, dtype=i32), logits.new_empty(rows, dtype=i32),
                                                          logits.new_empty(rows, dtype=f32)))
        at = token.data_ptr(), kept.data_ptr(), prob.data_ptr()
    else:
        token, kept, prob = out
        at = (_vector("token", token, i32, rows, index), _vector("kept", kept, i32, rows, index),
              _vector("prob", prob, f32, rows, index))
    kind = _types[logits.dtype]
    space = _sample_space(lib, rows, n, kind, index)
    work = 0
    if space:
        held = _made(stream, index, lambda: logits.new_empty((space + 3) // 4, dtype=i32))
        work = held.data_ptr()
    _call(lib.vx_sample_rows, _pack(_SAMPLE, logits.data_ptr(), logits.stride(0), t_at, p_at, m_at, k_at, u_at, *at, rows, n, kind, index,
                                   temperature, top_p, min_p, top_k, work, space), _stream(index, stream))
    return token, kept, prob


_spaces = {}  # (rows, n, type, device) -> bytes of workspace


def _sample_space(lib, rows, n, kind, index):
    key = rows, n, kind, index
    space = _spaces.get(key)
    if space is None:
        need = ctypes.c_size_t()
        _call(lib.vx_sample_rows_workspace, _SAMPLE.pack(*(0,) * 10, *key, 0, 0, 0, 0, 0, 0), ctypes.byref(need))
        if len(_spaces) >= 4096:
            _spaces.clear()
        space = _spaces[key] = need.value
    return space
