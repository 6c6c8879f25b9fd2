"""A KV cache for requests of different lengths, in pages of 64 positions held
in fp8 e4m3fn with a power-of-two scale per page and kv head, or (``bits=4``) in
whole numbers of 4 bits with a scale per position and 32 dims.

``PagedKVCache`` stands beside ``GroupedQueryAttention``'s own cache (one fp16
buffer per layer, one length for the whole batch, engine.py:105-109): row i is
one sequence, rows share a pool of pages, and a position takes half the bytes,
or 28 % of them.
A serving step is

    cache.extend(new_lens, plan)                    # once per step, for all layers
    q = cache.append(layer, k, v, plan, q=q, rotary=rotary)
    out = cache.attend(layer, q, plan)              # (tokens, n_q, 128)

with the step's tokens packed row after row (``plan.cu``).  Lengths, tables and
work lists live on the GPU and nothing waits on the host, so a step can be
captured into a graph.  ``rewind`` cuts rows back: rejected drafts, or the end
of a sequence.  ``fetch`` takes positions of a 4-bit cache out again as dense k
and v: a request that moves, a prefix that another cache takes over.

``extend``, ``rewind`` and ``append`` on one cache write its tables and pages:
they, and what reads the cache, have to be ordered, on one stream or by events.
``attend`` and ``fetch`` only read: of one step, for several layers or queries,
they may run on several streams at once.
"""
from __future__ import annotations

import ctypes

import torch

from . import _lib
from .rotary import Rotary

PAGE = 64
HEAD_DIM = 128
GROUP4 = 32                 # dims of a scale of the 4-bit cache
BLOCK4 = 9216               # bytes of its pages, per kv head
MAX_SEQS = 2048


class PagePlan:
    """A step's layout as ``PagedKVCache.extend`` writes it (device tensors):

    cu         (n_seqs + 1) first packed token of each row, and the total
    positions  (max_tokens) position of each token, -1 past the last one and
               for the tokens of a rejected row
    slots      (max_tokens) page * 64 + place in the page, -1 likewise
    kv_len     (n_seqs) positions of the row with the step's, 0: rejected
    rejected   (n_seqs) 1 where the row could not grow
    """

    def __init__(self, cache: "PagedKVCache", max_tokens: int, max_new: int | None = None):
        self.max_tokens = int(max_tokens)
        self.max_new = self.max_tokens if max_new is None else int(max_new)
        if self.max_tokens < 1 or self.max_new < 1:
            raise ValueError(f"a plan of {max_tokens} tokens, {max_new} a row: one at least")
        nbytes = _lib.load_library().oi2_page_plan_bytes(cache._ref, self.max_tokens, self.max_new)
        if not nbytes:
            raise ValueError(f"a plan of {max_tokens} tokens is too large")

        def ints(n):
            return torch.full((n,), -1, dtype=torch.int32, device=cache.device)

        self.cache = cache
        self.cu = torch.zeros(cache.n_seqs + 1, dtype=torch.int32, device=cache.device)
        self.positions, self.slots = ints(self.max_tokens), ints(self.max_tokens)
        self.kv_len = torch.zeros(cache.n_seqs, dtype=torch.int32, device=cache.device)
        self.rejected = torch.zeros(cache.n_seqs, dtype=torch.int32, device=cache.device)
        # its head counts the work: none before the first extend
        self.work = torch.zeros(nbytes // 4, dtype=torch.int32, device=cache.device)
        self._struct = _lib.PagePlan(self.max_tokens, self.max_new, self.cu.data_ptr(), self.positions.data_ptr(),
                                     self.slots.data_ptr(), self.kv_len.data_ptr(), self.rejected.data_ptr(),
                                     self.work.data_ptr())
        self._ref = ctypes.byref(self._struct)
        self._attend_bytes = _lib.load_library().oi2_kv_attend_workspace_bytes(
            cache._ref, self.max_tokens, self.max_new)


class PagedKVCache:
    """Pages of ``n_layers`` layers for ``n_seqs`` rows of at most ``max_len``
    positions: ``n_pages`` pages of 64 positions, ``n_kv`` kv heads of 128 for
    ``n_q`` query heads (groups of 1, 2, 4 or 8).  A page takes 16.4 KB per
    layer and kv head with ``bits`` 8, 9.2 KB with 4.

    With 4 bits a head's values are groups of 32 dims: whole numbers from -7 to 7
    times the group's largest magnitude over 7, rounded to 8 significant bits.
    Magnitudes past 65408 are held as that, a group with a NaN or an infinity as
    NaN.

    block_table (n_seqs, ceil(max_len / 64)), lens (n_seqs), free (n_pages, a
    stack) and n_free (1) are the tables, int32 on the device.  A row is
    rejected (``plan.rejected``) and stays as it was when it would pass max_len
    or the plan's sizes, or when the pool runs out of pages.  With 0 layers there
    are the tables alone, and plan.slots say where a caller's own pages of 64
    positions hold the step's tokens."""

    def __init__(self, n_layers: int, n_q: int, n_kv: int, n_seqs: int, max_len: int, n_pages: int, device="cuda",
                 bits: int = 8):
        if bits not in (4, 8):
            raise ValueError(f"{bits} bits: 4 or 8")
        self.bits = int(bits)
        self.n_layers, self.n_q, self.n_kv = int(n_layers), int(n_q), int(n_kv)
        self.n_seqs, self.max_len, self.n_pages = int(n_seqs), int(max_len), int(n_pages)
        if self.n_layers < 0:
            raise ValueError(f"{n_layers} layers")
        if self.n_kv < 1 or self.n_q % self.n_kv or self.n_q // self.n_kv not in (1, 2, 4, 8):
            raise ValueError(f"{self.n_q} query heads over {self.n_kv} kv heads: groups of 1, 2, 4 or 8")
        if not 1 <= self.n_seqs <= MAX_SEQS:
            raise ValueError(f"{self.n_seqs} rows: 1 to {MAX_SEQS}")
        if not 1 <= self.max_len <= 2 ** 31 - 1 - 2 * PAGE:
            raise ValueError(f"rows of {self.max_len} positions")
        if not 1 <= self.n_pages < 2 ** 25:
            raise ValueError(f"{self.n_pages} pages: 1 to 2^25 - 1")
        self.device = dev = _lib.gpu(device)
        self.width = -(-self.max_len // PAGE)

        def ints(shape, value):
            return torch.full(shape, value, dtype=torch.int32, device=dev)

        self.block_table = ints((self.n_seqs, self.width), -1)
        self.lens = ints((self.n_seqs,), 0)
        self.free = torch.arange(self.n_pages - 1, -1, -1, dtype=torch.int32, device=dev)
        self.n_free = ints((1,), self.n_pages)
        pool = (self.n_layers, self.n_pages, self.n_kv)
        if self.bits == 8:
            # a page and kv head's k codes and then its v codes
            self.pages = torch.zeros((*pool, 2, PAGE * HEAD_DIM), dtype=torch.uint8, device=dev)
            self._scales = torch.full((*pool, 2), 2.0 ** -40, dtype=torch.float32, device=dev)
        else:
            # k codes, v codes, k scales, v scales
            self.pages = torch.zeros((*pool, BLOCK4), dtype=torch.uint8, device=dev)
            self._scales = None
        self._views = {}
        self._struct = _lib.Paged(self.n_q, self.n_kv, self.n_seqs, self.max_len, self.n_pages, self.n_layers,
                                  self.block_table.data_ptr(), self.lens.data_ptr(), self.free.data_ptr(),
                                  self.n_free.data_ptr(), self.pages.data_ptr() or None,
                                  None if self._scales is None else self._scales.data_ptr() or None)
        self._ref = ctypes.byref(self._struct)

    # -- tables ---------------------------------------------------------------
    def new_plan(self, max_tokens: int, max_new: int | None = None) -> PagePlan:
        """Room for the layout of steps of up to max_tokens tokens, max_new of
        one row (max_tokens by default).  A plan belongs to its cache and serves
        one step at a time.  Decoding steps want max_new as small as it is:
        attention then leaves out its kernel for many rows."""
        return PagePlan(self, max_tokens, max_new)

    def _lens(self, lens) -> torch.Tensor:
        if not isinstance(lens, torch.Tensor):
            lens = torch.tensor(lens, dtype=torch.int32)
        if lens.dtype is torch.int32 and lens.shape == self.lens.shape and lens.device == self.device and lens.is_contiguous():
            return lens
        if lens.shape != (self.n_seqs,) or lens.dtype not in (torch.int32, torch.int64):
            raise ValueError(f"lengths: ({self.n_seqs},) int32, got {tuple(lens.shape)} {lens.dtype}")
        if lens.dtype == torch.int64:
            lens = lens.clamp(-1, 2 ** 31 - 1)       # not to wrap
        return lens.to(self.device, torch.int32).contiguous()

    def _plan(self, plan: PagePlan) -> PagePlan:
        if not isinstance(plan, PagePlan) or plan.cache is not self:
            raise ValueError("a plan of this cache (new_plan)")
        return plan

    def extend(self, new_lens, plan: PagePlan) -> PagePlan:
        """Row i grows by new_lens[i] positions (0 or less: not in the step); the
        plan is written and returned.  new_lens: (n_seqs) int32 on the device, or
        anything that converts to that (a list waits for its copy, and cannot be
        captured into a graph).  Rejected rows are not an error here:
        ``plan.rejected`` tells, at the price of waiting for it."""
        plan, new_lens = self._plan(plan), self._lens(new_lens)
        L = _lib.load_library()
        with _lib.on_device(self.device) as stream:
            _lib.check(L.oi2_page_extend(self._ref, plan._ref, new_lens.data_ptr(), stream))
        return plan

    def rewind(self, lens) -> None:
        """Row i is cut back to lens[i] positions where it holds more, and its
        pages past them are free again; 0 ends the sequence, a negative value
        leaves the row.  The former plan's step is not to be used after it."""
        lens = self._lens(lens)
        L = _lib.load_library()
        with _lib.on_device(self.device) as stream:
            _lib.check(L.oi2_page_rewind(self._ref, lens.data_ptr(), stream))

    # -- pages ----------------------------------------------------------------
    def _rows(self, x: torch.Tensor, heads: int, what: str, like: torch.Tensor | None = None):
        shape = x.shape
        if len(shape) != 3 or shape[1] != heads or shape[2] != HEAD_DIM:
            raise ValueError(f"{what}: (tokens, {heads}, {HEAD_DIM}), got {tuple(shape)}")
        if x.dtype not in (torch.float16, torch.bfloat16):
            raise TypeError(f"{what}: float16 or bfloat16, got {x.dtype}")
        if x.device != self.device:
            raise ValueError(f"{what} on {x.device}, the cache on {self.device}")
        if like is not None and (shape[0] != like.shape[0] or x.dtype != like.dtype):
            raise ValueError(f"{what} {tuple(x.shape)} {x.dtype} beside {tuple(like.shape)} {like.dtype}")
        return _lib.heads(x, heads)

    def _layer(self, layer: int) -> int:
        if not 0 <= int(layer) < self.n_layers:
            raise ValueError(f"layer {layer} of a cache of {self.n_layers}")
        return int(layer)

    def _tokens(self, x: torch.Tensor, plan: PagePlan) -> int:
        n = x.shape[0]
        if n > plan.max_tokens:
            raise ValueError(f"{n} tokens in a plan of {plan.max_tokens}")
        return n

    def append(self, layer: int, k: torch.Tensor, v: torch.Tensor, plan: PagePlan, q: torch.Tensor | None = None,
               rotary: Rotary | None = None, q_out: torch.Tensor | None = None):
        """k and v (tokens, n_kv, 128) of the step, fp16 or bf16 with any
        strides, into the layer's pages.  With ``rotary`` k is rotated first, to
        the bits that ``rotary`` itself gives, and so is q (tokens, heads, 128)
        if given; returns the rotated q, else None.  Tokens of rejected rows and
        past the step's last one are left out: their rows of q_out are not
        written, those of a new q are 0.  Each layer takes a step once: what a page
        of 8 bits holds is coded again when its scale grows."""
        plan, layer = self._plan(plan), self._layer(layer)
        k, hk = self._rows(k, self.n_kv, "k")
        v, hv = self._rows(v, self.n_kv, "v", k)
        n = self._tokens(k, plan)
        if rotary is None:
            if q is not None or q_out is not None:
                raise ValueError("q is rotated here: it needs the rotary")
        elif rotary.head_dim != HEAD_DIM or rotary.device != self.device:
            raise ValueError(f"a rotary of head_dim {HEAD_DIM} on {self.device}, got {rotary.head_dim} on {rotary.device}")
        if q is not None:
            q, hq = self._rows(q, q.shape[1] if q.dim() == 3 else self.n_q, "q", k)
            new = q_out is None
            q_out = rotary._output(q_out, q, "q_out")
            if q_out.data_ptr() == q.data_ptr() and not q.is_contiguous():
                raise ValueError("an output that is its own input must be contiguous")
        elif q_out is not None:
            raise ValueError("q_out without q")
        L = _lib.load_library()
        _lib.launch(self.device, L.oi2_kv4_append if self.bits == 4 else L.oi2_kv_append,
                    self._ref, plan._ref, layer, _lib.dtype_code(k.dtype) | (_lib.ZERO_LEFT_OUT if q is not None and new else 0), n,
                    ctypes.byref(hk), ctypes.byref(hv), None if rotary is None else rotary._ref,
                    None if q is None else ctypes.byref(hq), _lib.ptr(q_out))
        return q_out

    def attend(self, layer: int, q: torch.Tensor, plan: PagePlan, scale: float | None = None,
               out: torch.Tensor | None = None) -> torch.Tensor:
        """Causal attention of the step's tokens over the layer's pages, after
        the step was appended: the token at position t of a row sees positions
        [0, t] of it.  q (tokens, n_q, 128) fp16 or bf16 with any strides;
        ``scale`` of the scores 1 / sqrt(128) by default.  Returns (tokens, n_q,
        128) like q: zeros for the tokens of rejected rows; rows past the step's
        last token are 0 in a new tensor, and not written in ``out``."""
        plan, layer = self._plan(plan), self._layer(layer)
        q, hq = self._rows(q, self.n_q, "q")
        n = self._tokens(q, plan)
        dtype = _lib.dtype_code(q.dtype)
        if out is None:
            out = torch.empty_like(q, memory_format=torch.contiguous_format)
            dtype |= _lib.ZERO_LEFT_OUT
        elif out.shape != q.shape or out.dtype != q.dtype or out.device != q.device or not out.is_contiguous():
            raise ValueError("out must be a contiguous tensor like q")
        L = _lib.load_library()
        nbytes = plan._attend_bytes
        ws = q.new_empty((nbytes,), dtype=torch.uint8)
        _lib.launch(self.device, L.oi2_kv4_attend if self.bits == 4 else L.oi2_kv_attend,
                    self._ref, plan._ref, layer, dtype, n, ctypes.byref(hq),
                    HEAD_DIM ** -0.5 if scale is None else float(scale), out.data_ptr(), ws.data_ptr(), nbytes)
        return out

    def _given(self, x: torch.Tensor, what: str, n: int, dtype) -> torch.Tensor:
        if x.shape != (n, self.n_kv, HEAD_DIM) or x.dtype != dtype or x.device != self.device or x.stride(2) != 1:
            raise ValueError(f"{what}: ({n}, {self.n_kv}, {HEAD_DIM}) {dtype} on {self.device} with a dense last dimension, "
                             f"got {tuple(x.shape)} {x.dtype} on {x.device}")
        return x

    def fetch(self, layer: int, counts, max_tokens: int, first=None, dtype=torch.float16,
              k_out: torch.Tensor | None = None, v_out: torch.Tensor | None = None):
        """Positions [first[i], first[i] + counts[i]) of row i, cut to what it
        holds (first: 0 by default), of all rows one behind the other, as what
        they stand for: ``(k, v, cu)``, k and v (max_tokens, n_kv, 128) of
        ``dtype`` (fp16, exactly; bf16, fp32), cu (n_seqs + 1) int32 the first
        token of each row and the total.  counts and first: (n_seqs) int32 on the
        device, or anything that converts to that (a list waits for its copy).
        Tokens from max_tokens on are left out.  Rows past the last token are 0 in
        new tensors and not written in k_out and v_out, which may have any strides
        that keep their values apart, the same ones where they lie in one another's
        span: slices of one buffer, whichever dimension comes first.  A cache of 4
        bits; nothing waits on the host."""
        layer = self._layer(layer)
        if self.bits != 4:
            raise ValueError("fetch takes a cache of 4 bits; read() a row of either")
        n = int(max_tokens)
        if n < 0 or n > 2 ** 31 - 1:
            raise ValueError(f"{max_tokens} tokens")
        if dtype not in (torch.float16, torch.bfloat16, torch.float32):
            raise TypeError(f"{dtype}: float16, bfloat16 or float32")
        if (k_out is None) != (v_out is None):
            raise ValueError("k_out and v_out together")
        counts, first = self._lens(counts), None if first is None else self._lens(first)
        code = _lib.dtype_code(dtype)
        if k_out is None:
            code |= _lib.ZERO_LEFT_OUT
            k_out = torch.empty((n, self.n_kv, HEAD_DIM), dtype=dtype, device=self.device)
            v_out = torch.empty_like(k_out)
            st = self.n_kv * HEAD_DIM
            hk, hv = _lib.Heads(k_out.data_ptr(), self.n_kv, st, HEAD_DIM), _lib.Heads(v_out.data_ptr(), self.n_kv, st, HEAD_DIM)
        else:
            hk, hv = (_lib.heads(self._given(x, what, n, dtype), self.n_kv)[1] for x, what in ((k_out, "k_out"), (v_out, "v_out")))
        cu = counts.new_empty(self.n_seqs + 1)
        _lib.launch(self.device, _lib.load_library().oi2_kv4_fetch, self._ref, layer, _lib.ptr(first), counts.data_ptr(), code, n,
                    ctypes.byref(hk), ctypes.byref(hv), cu.data_ptr())
        return k_out, v_out, cu

    # -- views ----------------------------------------------------------------
    def codes(self, layer: int) -> tuple[torch.Tensor, torch.Tensor]:
        """The layer's k and v codes as views, float8_e4m3fn: k (n_pages, n_kv,
        4, 4, 4, 8, 16) and v (n_pages, n_kv, 4, 16, 8, 16), whose last two
        dimensions are the 128 dims and the ones before them the 64 positions of
        a page, in order; the memory holds them in the order of the attention's
        loads.  Of 4 bits, as copies: int8 (n_pages, n_kv, 64, 128)."""
        if self.bits == 4:
            return self._codes4(self._layer(layer))
        return self._layer_views(layer)[0]

    def scales(self, layer: int) -> tuple[torch.Tensor, torch.Tensor]:
        """The scales (n_pages, n_kv) of k and of v, as views: powers of two;
        v's is negative where the page holds a NaN in v.  Of 4 bits, fp16: k's
        (n_pages, n_kv, 4, 4, 4, 4) and v's (n_pages, n_kv, 64, 4), positions of a
        page and then groups of 32 dims."""
        if self.bits == 4:
            x = self.pages[self._layer(layer)].view(torch.float16)
            k, v = x[..., BLOCK4 // 2 - 512:BLOCK4 // 2 - 256], x[..., BLOCK4 // 2 - 256:]
            # k's memory: groups, places / 16, places % 4, places / 4 % 4
            return (k.unflatten(-1, (4, 4, 4, 4)).permute(0, 1, 3, 5, 4, 2), v.unflatten(-1, (4, PAGE)).transpose(2, 3))
        return self._layer_views(layer)[1]

    def _codes4(self, layer: int):
        x = self.pages[layer][..., :PAGE * HEAD_DIM].view(torch.int32)
        # k's memory: places / 4 % 4, groups, places / 16, places % 4, dwords of a
        # group; v's: places / 4 % 4, places / 16, dwords, places % 4
        k = x[..., :1024].unflatten(-1, (4, 4, 4, 4, 4)).permute(0, 1, 4, 2, 5, 3, 6)
        v = x[..., 1024:].unflatten(-1, (4, 4, 16, 4)).permute(0, 1, 3, 2, 5, 4)
        e = torch.arange(4, device=self.device, dtype=torch.int32)
        at = torch.cat([8 * e, 8 * e + 4])               # magnitudes
        sign = torch.cat([8 * e + 7, (8 * e + 11) % 32])

        def values(d):
            d = d.reshape(self.n_pages, self.n_kv, PAGE, 16, 1)
            n = (d >> at) & 7
            return torch.where(((d >> sign) & 1) != 0, -n, n).to(torch.int8).flatten(3)
        return values(k), values(v)

    def _layer_views(self, layer: int):
        layer = self._layer(layer)
        if layer not in self._views:
            x = self.pages[layer].view(torch.float8_e4m3fn)
            k = x[:, :, 0].view(self.n_pages, self.n_kv, 4, 8, 4, 4, 16).permute(0, 1, 4, 2, 5, 3, 6)
            v = x[:, :, 1].view(self.n_pages, self.n_kv, 8, 4, 16, 16).permute(0, 1, 3, 5, 2, 4)
            s = self._scales[layer]
            self._views[layer] = (k, v), (s[..., 0], s[..., 1])
        return self._views[layer]

    def read(self, layer: int, row: int, dtype=torch.float16) -> tuple[torch.Tensor, torch.Tensor]:
        """What a row's cache stands for: k and v (n_kv, length, 128), as the
        reference lays a cache out.  Waits for the row's length."""
        n = int(self.lens[row])
        if self.bits == 4:
            counts = torch.zeros(self.n_seqs, dtype=torch.int32, device=self.device)
            counts[row] = n
            k, v, _ = self.fetch(layer, counts, n, dtype=torch.float32)
            return k.transpose(0, 1).to(dtype).contiguous(), v.transpose(0, 1).to(dtype).contiguous()
        ids = self.block_table[row, :-(-n // PAGE)].long()
        out = []
        for c, s in zip(self.codes(layer), self.scales(layer)):
            x = c.view(torch.uint8)[ids].reshape(-1, self.n_kv, PAGE, HEAD_DIM).view(torch.float8_e4m3fn).float()
            x = x * s[ids].abs()[..., None, None]
            out.append(x.transpose(0, 1).reshape(self.n_kv, -1, HEAD_DIM)[:, :n].to(dtype))
        return out[0], out[1]
