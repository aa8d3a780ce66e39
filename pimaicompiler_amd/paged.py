"""A layer's keys and values of all served sequences in pages: appending to it, with the position rotation on the way, and attention of each
sequence's new token over it.

The reference's attention reads an encoder's outputs, all of one length (the decoder step, DecoderPlan); a language model's reads
what it has produced so far, which grows by a token a step and is of another length in every sequence.  Errors are NNRuntimeException, as
everywhere in this package; there is no CPU path and no backward pass."""
import ctypes
import math

import torch

from . import _lib as L
from .mx4 import _require
from .ops import NNRuntimeException, _check, _ensure_init, _Launch, _native, _require_no_gradient, _result

HEAD_DIM_MOST = 256
_CACHE_CODES = {torch.float16: L.PIMHIP_F16, torch.bfloat16: L.PIMHIP_BF16, torch.float8_e4m3fn: L.PIMHIP_F8E4M3}


def _overlaps(t):
    """Whether two elements of a tensor may lie in one place."""
    reach = 1
    for stride, size in sorted(zip(t.stride(), t.shape)):
        if size > 1:
            if stride < reach:
                return True
            reach = stride * (size - 1) + reach
    return False


def rotary_table(positions, dim, base=10000.0, scale=1.0, device=None):
    """The angles of PagedCache.append: [positions, dim] fp32, cosines of position / scale * base^(-2 i / dim) for i < dim / 2, then their sines,
    worked out in 64 bits."""
    if int(positions) < 1 or int(dim) < 2 or dim % 2 or not base > 0 or not scale > 0:
        raise NNRuntimeException(f"positions={positions} must be at least 1, dim={dim} even, base={base} and scale={scale} positive")
    i = torch.arange(0, int(dim), 2, dtype=torch.float64, device=device)
    angle = (torch.arange(int(positions), dtype=torch.float64, device=device) / scale).unsqueeze(1) * base ** (-i / dim)
    return torch.cat([torch.cos(angle), torch.sin(angle)], 1).float()


class PagedCache:
    """k_pages and v_pages [pages, kv_heads, page_size, head_dim] in fp16, bf16 or float8_e4m3fn, on the GPU, with any strides but for the last
    dimension (a cache laid out [pages, page_size, kv_heads, head_dim] is given as its transpose(1, 2)).  A cache in 8 bits has k_scale and
    v_scale [kv_heads] fp32: a stored value times its head's scale is what it stands for.

    The tensors are the cache's from then on and stay where they are; append writes to them.  head_dim is a multiple of 8 (16 in 8 bits)
    up to 256, page_size up to 65536.  A cache may be used on several streams, as far as its user orders writes and reads.

    Common to both calls: page_table [sequences, width] int32, a sequence's pages in order, and lengths [sequences] int32, its tokens, those of the
    current step among them.  Entries of the table behind a sequence's last page may be anything; a page outside of the cache is none: its
    tokens are not stored and not seen, nor are those of a sequence that its row of the table has no room for."""

    def __init__(self, k_pages, v_pages, k_scale=None, v_scale=None):
        for name, t in (("k_pages", k_pages), ("v_pages", v_pages)):
            _require(name, t, tuple(_CACHE_CODES))
            if t.dim() != 4 or t.stride(3) != 1 and t.size(3) > 1 or min(t.shape) < 1:
                raise NNRuntimeException(f"{name} must be [pages, kv_heads, page_size, head_dim], the values of a head next to each other; got {tuple(t.shape)}")
            if _overlaps(t):
                raise NNRuntimeException(f"{name} has elements in the same place (strides {t.stride()})")
        if k_pages.shape != v_pages.shape or k_pages.dtype != v_pages.dtype or k_pages.device != v_pages.device:
            raise NNRuntimeException(f"k_pages and v_pages differ: {tuple(k_pages.shape)} {k_pages.dtype} {k_pages.device}, {tuple(v_pages.shape)} {v_pages.dtype} "
                                     f"{v_pages.device}")
        pages, heads, size, dim = k_pages.shape
        eight = k_pages.dtype == torch.float8_e4m3fn
        if dim % (16 if eight else 8) or dim > HEAD_DIM_MOST or size > 65536 or heads > 65535:
            raise NNRuntimeException(f"head_dim={dim} must be a multiple of {16 if eight else 8} up to {HEAD_DIM_MOST}, page_size={size} at most 65536, kv_heads={heads} at most 65535")
        if eight != (k_scale is not None) or eight != (v_scale is not None):
            raise NNRuntimeException("k_scale and v_scale go with a cache in 8 bits: both or neither")
        if eight:
            for name, t in (("k_scale", k_scale), ("v_scale", v_scale)):
                _require(name, t, (torch.float32,))
                if tuple(t.shape) != (heads,) or t.device != k_pages.device:
                    raise NNRuntimeException(f"{name} must be [{heads}] on {k_pages.device}, got {tuple(t.shape)} on {t.device}")
            k_scale, v_scale = k_scale.contiguous(), v_scale.contiguous()
        _require_no_gradient(k_pages, v_pages, k_scale, v_scale)
        self.k_pages, self.v_pages, self.k_scale, self.v_scale = k_pages, v_pages, k_scale, v_scale
        self.kv_heads, self.page_size, self.head_dim, self.dtype, self.device = heads, size, dim, k_pages.dtype, k_pages.device
        ptr = lambda t: t.data_ptr() if t is not None else None  # noqa: E731
        self._keep = L.PagedCache(k_pages.data_ptr(), v_pages.data_ptr(), ptr(k_scale), ptr(v_scale), (ctypes.c_int64 * 3)(*k_pages.stride()[:3]),
                                  (ctypes.c_int64 * 3)(*v_pages.stride()[:3]), pages, heads, size, dim, _CACHE_CODES[k_pages.dtype])
        self._at = ctypes.addressof(self._keep)   # (what the native calls read the cache through)
        self._device_index = k_pages.device.index
        _ensure_init(k_pages)

    def __reduce__(self):
        """A deep copy, or one read from a file, is made of its own tensors: what the native calls read it through holds addresses."""
        return PagedCache, (self.k_pages, self.v_pages, self.k_scale, self.v_scale)

    def _require_tokens(self, name, t, heads=None):
        """[tokens, heads, head_dim] of one of the types that go with the cache."""
        _require(name, t, (torch.float16, torch.bfloat16))
        if self.dtype != torch.float8_e4m3fn and t.dtype != self.dtype:
            raise NNRuntimeException(f"{name} is {t.dtype}, the cache {self.dtype}")
        if t.dim() != 3 or t.size(2) != self.head_dim or heads is not None and t.size(1) != heads or t.device != self.device:
            raise NNRuntimeException(f"{name} must be [tokens, {'heads' if heads is None else heads}, {self.head_dim}] on {self.device}, got {tuple(t.shape)} on {t.device}")
        _require_no_gradient(t)

    def _require_batch(self, page_table, lengths):
        for name, t, dims in (("page_table", page_table, 2), ("lengths", lengths, 1)):
            _require(name, t, (torch.int32,))
            if t.dim() != dims or t.device != self.device:
                raise NNRuntimeException(f"{name} must have {dims} dimension{'s' if dims > 1 else ''} on {self.device}, got {tuple(t.shape)} on {t.device}")
        if page_table.size(0) != lengths.size(0) or page_table.size(1) < 1:
            raise NNRuntimeException(f"page_table must be [{lengths.size(0)}, 1 or more] for {lengths.size(0)} lengths, got {tuple(page_table.shape)}")

    # What the native calls take of tensors that were looked at, and the tensors it points into.  Copies are made here, so it is called inside _Launch: on the
    # stream that reads them.
    @staticmethod
    def _batch(page_table, lengths):
        if page_table.stride(1) != 1 and page_table.size(1) > 1 or page_table.size(0) > 1 and page_table.stride(0) < page_table.size(1):
            page_table = page_table.contiguous()
        lengths = lengths.contiguous()
        return L.PagedBatch(page_table.data_ptr(), lengths.data_ptr(), page_table.stride(0), lengths.size(0), page_table.size(1)), (page_table, lengths)

    @staticmethod
    def _rows(t):
        t = t if t.stride(2) == 1 else t.contiguous()   # (the values of a head next to each other)
        return L.PagedRows(t.data_ptr(), t.stride(0), t.stride(1)), t

    def append(self, k, v, page_table, lengths, starts=None, q=None, rotary=None, interleaved=False, stream=None):
        """Stores k and v [tokens, kv_heads, head_dim] (fp16 or bf16, the cache's type where that is not in 8 bits).

        starts [sequences + 1] int32, rising: tokens starts[s] .. starts[s + 1] - 1 are the last of sequence s, others nobody's and not stored;
        None: one token for each sequence.  A sequence of length 0, or shorter than its tokens, has none at the positions below 0.
        rotary [width * page_size or more, n] fp32 (rotary_table): the first n values of each key are turned in pairs by the token's
        position, in fp32, values i and n / 2 + i, or 2 i and 2 i + 1 if interleaved; so are those of q [tokens, heads, head_dim], the queries
        of the same tokens, which are returned (zeros for a token that is nobody's, or at no position of the table).  Without q the result is None.

        k, v and q lie in other memory than the cache, whose keys and values lie in memory of their own (a cache of one tensor for both is refused).
        Values are rounded once; in 8 bits x / scale is, saturating at 448.  Two tokens of a call that are given the same place (a page that two
        sequences write) leave either's values there."""
        native = _native().fast_paged_append(self._at, self._device_index, k, v, page_table, lengths, starts, q, rotary, interleaved) if stream is None else None
        if native is not None:
            return _result(native) if type(native) is int else native[0]
        self._require_tokens("k", k, self.kv_heads)
        self._require_tokens("v", v, self.kv_heads)
        if v.shape != k.shape or v.dtype != k.dtype:
            raise NNRuntimeException(f"k and v differ: {tuple(k.shape)} {k.dtype}, {tuple(v.shape)} {v.dtype}")
        tokens = k.size(0)
        if q is not None:
            if rotary is None:
                raise NNRuntimeException("q is only turned: it goes with rotary")
            self._require_tokens("q", q)
            if q.size(0) != tokens or q.dtype != k.dtype or q.size(1) < 1:
                raise NNRuntimeException(f"q must be [{tokens}, 1 or more, {self.head_dim}] in {k.dtype}, got {tuple(q.shape)} in {q.dtype}")
        self._require_batch(page_table, lengths)
        sequences = lengths.size(0)
        if starts is not None:
            _require("starts", starts, (torch.int32,))
            if tuple(starts.shape) != (sequences + 1,) or starts.device != self.device:
                raise NNRuntimeException(f"starts must be [{sequences + 1}] on {self.device}, got {tuple(starts.shape)} on {starts.device}")
        elif tokens != sequences:
            raise NNRuntimeException(f"{tokens} tokens for {sequences} sequences need starts")
        if rotary is not None:
            _require("rotary", rotary, (torch.float32,))
            _require_no_gradient(rotary)
            if rotary.dim() != 2 or rotary.size(1) % 2 or not 2 <= rotary.size(1) <= self.head_dim or rotary.device != self.device:
                raise NNRuntimeException(f"rotary must be [positions, an even number up to {self.head_dim}] on {self.device}, got {tuple(rotary.shape)} on {rotary.device}")
            if rotary.size(0) < page_table.size(1) * self.page_size:
                raise NNRuntimeException(f"rotary has {rotary.size(0)} positions, the page table room for {page_table.size(1) * self.page_size}")
        ptr = lambda t: t.data_ptr() if t is not None else None  # noqa: E731
        with _Launch(self.device, stream, k, v, q, page_table, lengths, starts, rotary, self.k_pages, self.v_pages, self.k_scale, self.v_scale) as handle:
            batch, batch_tensors = self._batch(page_table, lengths)
            (k_rows, k), (v_rows, v) = self._rows(k), self._rows(v)
            q_rows, out = None, None
            if q is not None:
                q_rows, q = self._rows(q)
                out = torch.empty(q.shape, dtype=q.dtype, device=self.device)
            if starts is not None:
                starts = starts.contiguous()
            dim = rows = pitch = 0
            if rotary is not None:
                if rotary.stride(1) != 1 or rotary.size(0) > 1 and rotary.stride(0) < rotary.size(1):
                    rotary = rotary.contiguous()
                rows, dim = rotary.shape
                pitch = rotary.stride(0) if rows > 1 else dim   # (one row may have any stride)
            _check(L.load().pimhip_paged_append(self._at, ctypes.byref(batch), ptr(starts), tokens, ctypes.byref(k_rows), ctypes.byref(v_rows),
                                                ctypes.byref(q_rows) if q is not None else None, q.size(1) if q is not None else 0, ptr(out),
                                                _CACHE_CODES[k.dtype], ptr(rotary), rows, pitch, dim, int(bool(interleaved)), handle))
        return out

    def attend(self, q, page_table, lengths, scale=None, window=0, lse=False, stream=None):
        """out [sequences, heads, head_dim] for q [sequences, heads, head_dim], a query for each sequence: softmax(scale q . k) v over its tokens, or the
        last `window` of them where that is not 0.  heads is a multiple of kv_heads, neighbouring ones share a key head; scale is 1 / sqrt(head_dim) by
        default.  With lse also [sequences, heads] fp32, the logarithm of the sum of exp(scale q . k).

        Statistics, sums and the weights of the values are fp32, out is rounded once.  A sequence without tokens: zeros, and -inf.  What lies in places
        that are not seen has no influence, NaN included.  Weights are up to 2^10 before their sum divides them: values above 2^118 / tokens may
        overflow."""
        scale = 1.0 / math.sqrt(self.head_dim) if scale is None else scale
        native = _native().fast_paged_attend(self._at, self._device_index, q, page_table, lengths, scale, window, lse) if stream is None else None
        if native is not None:
            return _result(native)
        self._require_tokens("q", q)
        self._require_batch(page_table, lengths)
        heads = q.size(1)
        if q.size(0) != lengths.size(0) or heads < 1 or heads % self.kv_heads:
            raise NNRuntimeException(f"q must be [{lengths.size(0)}, a multiple of {self.kv_heads}, {self.head_dim}], got {tuple(q.shape)}")
        if not isinstance(window, int) or not 0 <= window <= 2**31 - 1 or not isinstance(scale, (int, float)) or not abs(scale) < 3.4e38:
            raise NNRuntimeException(f"window={window!r} must be a whole number from 0 on, scale={scale!r} a finite number")
        lib = L.load()
        with _Launch(self.device, stream, q, page_table, lengths, self.k_pages, self.v_pages, self.k_scale, self.v_scale) as handle:
            (batch, batch_tensors), (rows, q) = self._batch(page_table, lengths), self._rows(q)
            n = ctypes.c_uint64()
            _check(lib.pimhip_paged_attend_workspace_bytes(self._at, ctypes.byref(batch), heads, ctypes.byref(n)))
            out = torch.empty(q.shape, dtype=q.dtype, device=self.device)
            sums = torch.empty(q.shape[:2], dtype=torch.float32, device=self.device) if lse else None
            workspace = torch.empty(n.value, dtype=torch.uint8, device=self.device)
            _check(lib.pimhip_paged_attend(self._at, ctypes.byref(batch), ctypes.byref(rows), heads, _CACHE_CODES[q.dtype], scale, window,
                                           out.data_ptr(), sums.data_ptr() if lse else None, workspace.data_ptr(), handle))
        return (out, sums) if lse else out
