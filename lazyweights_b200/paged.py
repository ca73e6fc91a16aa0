"""Keys and values of several sequences in pools of pages, and the operators that fill and read them.

`append` rotates the rows of a fused q/k/v product and writes their keys and values to the pages; `attend` is attention of
one new token per sequence, `attend_prompt` causal attention of packed prompts (or pieces of prompts).  All three take the
same description of the sequences, CUDA int32 tensors that are read when the kernel runs (a captured call can be replayed
with other contents):

  table   [n, columns]  the pages of every sequence; entries behind its length are not read
  lens    [n]           length of every sequence, the positions of the call's rows included
  starts  [n + 1]       rows starts[b] .. starts[b + 1] - 1 are the last positions of sequence b; rows outside belong to none

Every call has at least one sequence and one row, and 2^30 rows at most.  Queries, keys, values, results and attention's weights are rounded to the cache's type, scores
and sums held in 32 bits.  torch is only used for device memory and streams.  A page outside the pool, a length beyond the table or a position beyond
the rotation tables is not followed and sets bit 1 of lw_kernel_error().
"""
from . import _native as nat
from .runtime import _stream, _torch

_CODES = None


def _codes(torch):
    global _CODES
    if _CODES is None:
        _CODES = {torch.float16: 0, torch.bfloat16: 1, torch.float32: 2}
    return _CODES


def _window(window):
    """ctypes would cut it to 32 bits."""
    if not 0 <= window < 1 << 31:
        raise ValueError("window must be 0 (all positions) .. 2^31 - 1, not %r" % (window,))
    return window


class PagedCache:
    """Pools k_pages and v_pages [pages, kv_heads, page_size, head_dim], CUDA fp16 or bf16, of the same strides (any multiples of
    eight, head_dim contiguous: a pool with the heads inside the positions is passed transposed).  The tensors are kept alive."""

    def __init__(self, k_pages, v_pages):
        torch = _torch()
        self._h, self._spaces, self._lib = None, {}, nat.lib()
        if k_pages.dim() != 4 or k_pages.shape != v_pages.shape or k_pages.dtype is not v_pages.dtype or \
                k_pages.dtype not in (torch.float16, torch.bfloat16):
            raise ValueError("PagedCache wants two fp16 or bf16 pools [pages, kv_heads, page_size, head_dim] of one shape and type")
        if not k_pages.is_cuda or k_pages.device != v_pages.device:
            raise ValueError("the pools must be on one CUDA device")
        n, heads, size, dim = k_pages.shape
        sp, sh, st, sd = k_pages.stride()
        if sd != 1 or any(a != b and c > 1 for a, b, c in zip(k_pages.stride(), v_pages.stride(), k_pages.shape)):
            raise ValueError("the pools must have the same strides and a contiguous head_dim")
        self.k_pages, self.v_pages = k_pages, v_pages
        self.n_pages, self.kv_heads, self.page_size, self.head_dim = n, heads, size, dim
        self.dtype, self.device, self._index = k_pages.dtype, k_pages.device, k_pages.get_device()
        with torch.cuda.device(self._index):
            ptr = self._lib.lw_cache_create(k_pages.data_ptr(), v_pages.data_ptr(), _codes(torch)[self.dtype], n, heads, size, dim, sp, sh, st)
        if not ptr:
            raise nat.LwError(self._lib.lw_last_status() or -1, nat.last_error())
        self._h = ptr

    @classmethod
    def empty(cls, n_pages, kv_heads, page_size, head_dim, dtype=None, device="cuda"):
        """A cache with pools of its own (fp16 unless `dtype` says otherwise)."""
        torch = _torch()
        shape = (n_pages, kv_heads, page_size, head_dim)
        pools = [torch.empty(shape, dtype=dtype or torch.float16, device=device) for _ in range(2)]
        return cls(*pools)

    def close(self):
        if self._h:
            self._lib.lw_cache_destroy(self._h)
            self._h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    # ---- checks.  A call on a few rows takes the GPU 2 to 20 us, so what the checks cost counts: one call per property.
    def _sequences(self, torch, table, lens):
        i32 = torch.int32
        n = lens.shape[0] if lens.dim() == 1 else -1
        if table.dtype is not i32 or lens.dtype is not i32 or table.dim() != 2 or table.shape[0] != n or \
                table.get_device() != self._index or lens.get_device() != self._index:
            raise ValueError("table [n, columns] and lens [n] must be int32 on the cache's device")
        cols = table.shape[1]
        st, sc = table.stride()
        if cols > 1 and sc != 1 or n > 1 and lens.stride(0) != 1:
            raise ValueError("the rows of table, and lens, must be contiguous")
        return n, cols, st if n > 1 else max(cols, 1)

    def _starts(self, torch, starts, n):
        if starts.dtype is not torch.int32 or starts.dim() != 1 or starts.shape[0] != n + 1 or starts.get_device() != self._index or \
                starts.stride(0) != 1:
            raise ValueError("starts [%d] must be contiguous int32 on the cache's device" % (n + 1))

    def _rows(self, t, what, rows=None, heads=None):
        """Rows, heads and strides of a [rows, heads, head_dim] tensor of queries or results."""
        if t.dim() == 3 and t.dtype is self.dtype and t.get_device() == self._index:
            r, h, d = t.shape
            sr, sh, sd = t.stride()
            if d == self.head_dim and sd == 1 and (rows is None or r == rows) and (heads is None or h == heads):
                if h == 1:
                    sh = d
                return r, h, (sr if r > 1 else h * sh), sh
        raise ValueError("%s must be [%s, %s, %d] of the cache's type and device, head_dim contiguous"
                         % (what, "rows" if rows is None else rows, "heads" if heads is None else heads, self.head_dim))

    # ---- operators
    def append(self, qkv, n_heads, cos, sin, table, lens, starts=None, q=None):
        """Rows [n, (n_heads + 2 kv_heads) * head_dim] (fp16, bf16 or fp32) of a fused product: rotated queries [n, n_heads,
        head_dim] in the cache's type are returned (`q`: a tensor to fill), rotated keys and values go to the pages.  cos, sin: fp32
        tables [positions, r], pairs (i, i + r) are rotated, dimensions from 2 r on copied.  Without starts, row b is the last position
        of sequence b.  Rows of no sequence are left as they are, in q too."""
        torch = _torch()
        index = self._index
        n, cols, tstride = self._sequences(torch, table, lens)
        if starts is not None:
            self._starts(torch, starts, n)
        code, width = _codes(torch).get(qkv.dtype), (n_heads + 2 * self.kv_heads) * self.head_dim
        if qkv.dim() != 2 or code is None or qkv.get_device() != index or qkv.shape[1] != width or qkv.stride(1) != 1:
            raise ValueError("qkv must be [rows, %d] fp16, bf16 or fp32 on the cache's device" % width)
        f32 = torch.float32
        if cos.dtype is not f32 or sin.dtype is not f32 or cos.dim() != 2 or cos.shape != sin.shape or not cos.is_contiguous() or \
                not sin.is_contiguous() or cos.get_device() != index or sin.get_device() != index:
            raise ValueError("cos and sin must be contiguous fp32 tables [positions, pairs] on the cache's device")
        rows = qkv.shape[0]
        if q is None:
            q = torch.empty((rows, n_heads, self.head_dim), dtype=self.dtype, device=self.device)
        _, _, qt, qh = self._rows(q, "q", rows, n_heads)
        positions, pairs = cos.shape
        rc = self._lib.lw_cache_append(self._h, qkv.data_ptr(), code, qkv.stride(0) if rows > 1 else width, rows, n_heads, cos.data_ptr(),
                                       sin.data_ptr(), positions, pairs, None if starts is None else starts.data_ptr(), lens.data_ptr(),
                                       table.data_ptr(), n, cols, tstride, q.data_ptr(), qt, qh, _stream(torch, index))
        if rc < 0:
            nat.check(rc)
        return q

    def _workspace(self, torch, heads, prompt):
        """A workspace of the call's own: calls may overlap, and captured ones too."""
        need = self._spaces.get((heads, prompt))
        if need is None:
            need = self._spaces[heads, prompt] = nat.check(self._lib.lw_cache_workspace(self._h, heads, prompt))
        return torch.empty(need, dtype=torch.uint8, device=self.device), need

    def attend(self, q, table, lens, scale=None, window=0, out=None):
        """Attention of one new token per sequence: q [n, heads, head_dim] -> the same shape (`out`: a tensor to fill).  scale: of
        the scores, head_dim ** -0.5 unless given; window: positions seen, the token's own included (0: all).  A sequence of length 0
        gives zeros."""
        torch = _torch()
        n, cols, tstride = self._sequences(torch, table, lens)
        _, heads, qt, qh = self._rows(q, "q", n)
        if out is None:
            out = torch.empty((n, heads, self.head_dim), dtype=self.dtype, device=self.device)
        _, _, ot, oh = self._rows(out, "out", n, heads)
        space, size = self._workspace(torch, heads, 0)
        rc = self._lib.lw_cache_attend(self._h, q.data_ptr(), qt, qh, n, heads, lens.data_ptr(), table.data_ptr(), cols, tstride,
                                       self.head_dim ** -0.5 if scale is None else scale, _window(window), out.data_ptr(), ot, oh,
                                       space.data_ptr(), size, _stream(torch, self._index))
        if rc < 0:
            nat.check(rc)
        return out

    def attend_prompt(self, q, table, lens, starts, scale=None, window=0, out=None):
        """Causal attention of packed rows q [rows, heads, head_dim] -> the same shape: rows starts[b] .. starts[b + 1] - 1 are the last
        positions of sequence b, each sees the positions up to its own (with a window, the last `window` of them).  Rows before
        position 0 give zeros, rows of no sequence are left as they are."""
        torch = _torch()
        n, cols, tstride = self._sequences(torch, table, lens)
        self._starts(torch, starts, n)
        rows, heads, qt, qh = self._rows(q, "q")
        if out is None:
            out = torch.empty((rows, heads, self.head_dim), dtype=self.dtype, device=self.device)
        _, _, ot, oh = self._rows(out, "out", rows, heads)
        space, size = self._workspace(torch, heads, 1)
        rc = self._lib.lw_cache_attend_prompt(self._h, q.data_ptr(), qt, qh, rows, heads, starts.data_ptr(), lens.data_ptr(), table.data_ptr(), n, cols,
                                              tstride, self.head_dim ** -0.5 if scale is None else scale, _window(window), out.data_ptr(), ot, oh,
                                              space.data_ptr(), size, _stream(torch, self._index))
        if rc < 0:
            nat.check(rc)
        return out
