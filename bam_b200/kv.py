"""A key/value cache of attention heads in the pages of a PageCache.

The rows live in an Array over the store, so a cache larger than GPU memory needs nothing special: pages that are not
resident are fetched by the call that reads them, dirty ones are written back when they are evicted (or by
PageCache.flush).  The calls are asynchronous like every other launch: what goes wrong on the device -- a wait that ran
out, an index outside its range -- is reported by Controller.status() / check_status().
"""
import ctypes as C

from . import _lib
from ._lib import KvAppend, KvAttend, KvLayout, check
from .host import REPLICATE, Array

ROPE_STYLES = {"half": 0, "pairs": 1}


class KvCache:
    """n_layers x n_blocks blocks of block_tokens tokens for n_kv_heads heads of head_dim elements.

    One page of `cache` holds the keys and the values of one block for one head; block_tokens defaults to what fits (a
    multiple of 16).  A token's slot is block * block_tokens + its place in the block.  `dist` lays the pages over the
    controllers of the cache (REPLICATE or STRIPE), store_byte_offset places them in the store."""

    def __init__(self, cache, n_blocks, n_kv_heads, head_dim, dtype=None, block_tokens=None, n_layers=1, store_byte_offset=0,
                 dist=REPLICATE):
        import torch
        dtype = torch.bfloat16 if dtype is None else dtype
        if dtype not in (torch.bfloat16, torch.float16):
            raise ValueError(f"dtype must be bfloat16 or float16, not {dtype}")
        if head_dim % 16 or not 16 <= head_dim <= 256:
            raise ValueError(f"head_dim must be a multiple of 16 up to 256, not {head_dim}")
        if n_blocks < 1 or n_kv_heads < 1 or n_layers < 1:
            raise ValueError("n_blocks, n_kv_heads and n_layers must be positive")
        row = 4 * head_dim                                       # a key and a value
        if block_tokens is None:
            block_tokens = cache.page_size // row // 16 * 16
        if block_tokens < 16 or block_tokens % 16 or block_tokens * row > cache.page_size:
            raise ValueError(f"a page of {cache.page_size} bytes does not hold a block of 16 n tokens of {row} bytes")
        self.lib, self.cache = cache.lib, cache
        self.n_blocks, self.n_kv_heads, self.head_dim, self.dtype = n_blocks, n_kv_heads, head_dim, dtype
        self.block_tokens, self.n_layers = block_tokens, n_layers
        self.device = torch.device("cuda", cache.ctrl.device)
        self.array = Array(cache, n_layers * n_blocks * n_kv_heads * (cache.page_size // 8), 8, store_byte_offset, dist)
        self._layouts = [KvLayout(0 if dtype == torch.bfloat16 else 1, head_dim, n_kv_heads, block_tokens, n_blocks,
                                  i * n_blocks * n_kv_heads) for i in range(n_layers)]
        self._scratch_bytes = self.lib.bam_kv_scratch_bytes(self.array.h, C.byref(self._layouts[0]))

    def close(self):
        self.array.close()

    # ---- arguments ----------------------------------------------------------------------------------------

    def _layout(self, layer):
        if not 0 <= layer < self.n_layers:
            raise ValueError(f"layer {layer} of {self.n_layers}")
        return C.byref(self._layouts[layer])

    def _on(self, name, t, dtype, ndim):
        if t.device != self.device:
            raise ValueError(f"{name} is on {t.device}, the cache on {self.device}")
        if t.dtype != dtype:
            raise ValueError(f"{name} must be {dtype}, not {t.dtype}")
        if t.dim() != ndim:
            raise ValueError(f"{name} must have {ndim} dimensions, not {t.dim()}")
        return t

    def _heads(self, name, t, n, heads):
        """A tensor [n, heads, head_dim] whose heads are contiguous."""
        self._on(name, t, self.dtype, 3)
        if (n is not None and t.shape[0] != n) or t.shape[1] != heads or t.shape[2] != self.head_dim:
            raise ValueError(f"{name} has shape {tuple(t.shape)}, wanted ({'n' if n is None else n}, {heads}, {self.head_dim})")
        if t.stride(2) != 1:
            raise ValueError(f"the elements of a head of {name} must be contiguous")
        return t

    def _flat(self, name, t, dtype, n):
        self._on(name, t, dtype, 1)
        if t.shape[0] != n or (n > 1 and t.stride(0) != 1):
            raise ValueError(f"{name} must be {n} contiguous values")
        return t

    def _queue(self, stream):
        """The stream the call runs on, as a context for the memory it takes: `stream` (a torch stream or a raw
        handle), or torch's current stream of the cache's device."""
        import torch
        if stream is None:
            return None
        if not isinstance(stream, torch.cuda.Stream):
            stream = torch.cuda.ExternalStream(int(stream), device=self.device)
        if stream.device != self.device:
            raise ValueError(f"the stream is on {stream.device}, the cache on {self.device}")
        return stream

    def _run(self, stream, call):
        import torch
        s = self._queue(stream)
        if s is None:
            s = torch.cuda.current_stream(self.device)
            return call(s.cuda_stream)
        with torch.cuda.stream(s):
            return call(s.cuda_stream)

    def _scratch(self):
        import torch
        return torch.empty(self._scratch_bytes, dtype=torch.uint8, device=self.device)

    # ---- operators ----------------------------------------------------------------------------------------

    def append(self, k, v, slots, layer=0, positions=None, rope=None, rope_style="half", q=None, q_norm=None, k_norm=None,
               norm_eps=1e-6, q_out=None, stream=None):
        """Write the rows k[t], v[t] ([n, n_kv_heads, head_dim], any strides of tokens and heads) to slots[t] (int64;
        negative: a padding row, nothing is written).  The other slots must be distinct: of two rows for one slot neither
        is sure to be kept whole.

        With `k_norm` ([head_dim], of the cache's dtype) every head of k is normed by its root mean square and scaled;
        with `rope` = (cos, sin), float tensors [n_positions, rotary_dim / 2], its first rotary_dim elements are then
        rotated by the angle of positions[t] (int64) in pairs (i, i + rotary_dim / 2) ("half") or (2 i, 2 i + 1)
        ("pairs").  `q` ([n, heads, head_dim]) takes the same pass with `q_norm`, into `q_out` (may be q itself) or a
        new tensor, which is returned.  All of it is computed in 32 bits and rounded once."""
        import torch
        n = k.shape[0]
        self._heads("k", k, None, self.n_kv_heads)
        self._heads("v", v, n, self.n_kv_heads)
        self._flat("slots", slots, torch.int64, n)
        a = KvAppend(k=k.data_ptr(), v=v.data_ptr(), n_tokens=n, slots=slots.data_ptr(), norm_eps=norm_eps)
        a.k_stride[:], a.v_stride[:] = k.stride()[:2], v.stride()[:2]
        if rope is not None:
            cos, sin = rope
            self._on("cos", cos, torch.float32, 2)
            self._on("sin", sin, torch.float32, 2)
            if rope_style not in ROPE_STYLES:
                raise ValueError(f"rope_style must be one of {sorted(ROPE_STYLES)}, not {rope_style!r}")
            if positions is None:
                raise ValueError("a rotation needs positions")
            self._flat("positions", positions, torch.int64, n)
            if cos.shape != sin.shape or cos.stride() != sin.stride() or cos.stride(1) != 1 or cos.shape[0] == 0:
                raise ValueError("cos and sin must be rows of the same shape and strides")
            rotary = 2 * cos.shape[1]
            if rotary % 16 or not 0 < rotary <= self.head_dim:
                raise ValueError(f"{rotary} rotated elements: a multiple of 16 up to {self.head_dim} is wanted")
            a.positions, a.cos, a.sin, a.n_positions = positions.data_ptr(), cos.data_ptr(), sin.data_ptr(), cos.shape[0]
            a.rope_stride, a.rotary_dim, a.rope_style = max(cos.stride(0), rotary // 2), rotary, ROPE_STYLES[rope_style]
        for name, w in (("q_norm", q_norm), ("k_norm", k_norm)):
            if w is not None:
                setattr(a, name, self._flat(name, w, self.dtype, self.head_dim).data_ptr())
        if q is None:
            if q_norm is not None or q_out is not None:
                raise ValueError("q_norm and q_out go with q")
        else:
            if q.dim() != 3 or q.shape[1] < 1:
                raise ValueError("q must be [n, heads, head_dim]")
            self._heads("q", q, n, q.shape[1])
            if q_out is not None:
                self._heads("q_out", q_out, n, q.shape[1])

        def call(s):
            out = q_out
            if q is not None:
                if out is None:
                    out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
                a.q, a.q_out, a.n_q_heads = q.data_ptr(), out.data_ptr(), q.shape[1]
                a.q_stride[:], a.q_out_stride[:] = q.stride()[:2], out.stride()[:2]
            scratch = self._scratch()
            check(self.lib.bam_launch_kv_append(self.array.h, self._layout(layer), C.byref(a), scratch.data_ptr(),
                                                self._scratch_bytes, s), "bam_launch_kv_append")
            return out
        if n == 0:
            self._layout(layer)
            return q_out if q is None or q_out is not None else torch.empty_like(q)
        return self._run(stream, call)

    def gather(self, slots, layer=0, out=None, stream=None):
        """The rows at `slots` (int64; negative: zeros) as (k, v), each [n, n_kv_heads, head_dim]; `out`: a pair of
        tensors of that shape, with any strides of tokens and heads, to write them to."""
        import torch
        n = slots.shape[0] if slots.dim() == 1 else -1
        self._flat("slots", slots, torch.int64, n)
        if out is not None:
            self._heads("out[0]", out[0], n, self.n_kv_heads)
            self._heads("out[1]", out[1], n, self.n_kv_heads)

        def call(s):
            k, v = out if out is not None else (torch.empty((n, self.n_kv_heads, self.head_dim), dtype=self.dtype, device=self.device)
                                                for _ in range(2))
            ks, vs = (C.c_int64 * 2)(*k.stride()[:2]), (C.c_int64 * 2)(*v.stride()[:2])
            scratch = self._scratch()
            if n:
                check(self.lib.bam_launch_kv_gather(self.array.h, self._layout(layer), n, slots.data_ptr(), k.data_ptr(), v.data_ptr(),
                                                    ks, vs, scratch.data_ptr(), self._scratch_bytes, s), "bam_launch_kv_gather")
            return k, v
        self._layout(layer)
        return self._run(stream, call)

    def attend(self, q, block_table, seq_lens, layer=0, scale=None, window=0, sinks=0, out=None, return_lse=False, stream=None):
        """Attention of one new token per sequence: q [batch, heads, head_dim] (heads a multiple of n_kv_heads) over the
        first seq_lens[b] (int32) tokens of sequence b, token j in block block_table[b, j // block_tokens] (int32).

        window > 0: only the last `window` tokens and the first `sinks` are visible; blocks without a visible token are
        not touched, their table entries may be anything.  scale defaults to head_dim ** -0.5.  Returns out, or
        (out, lse) with the logarithm of the softmax's denominator [batch, heads]; a sequence with nothing visible gets
        zeros and -inf.  The new token's own key and value have to be appended first."""
        import torch
        if q.dim() != 3 or q.shape[1] < 1 or q.shape[1] % self.n_kv_heads:
            raise ValueError(f"q must be [batch, heads, head_dim] with a multiple of {self.n_kv_heads} heads")
        n, heads = q.shape[:2]
        self._heads("q", q, n, heads)
        self._on("block_table", block_table, torch.int32, 2)
        if block_table.shape[0] != n or block_table.shape[1] < 1 or (block_table.shape[1] > 1 and block_table.stride(1) != 1):
            raise ValueError(f"block_table must be {n} rows of contiguous entries")
        self._flat("seq_lens", seq_lens, torch.int32, n)
        if window < 0 or sinks < 0:
            raise ValueError("window and sinks must not be negative")
        if out is not None:
            self._heads("out", out, n, heads)

        def call(s):
            o = torch.empty((n, heads, self.head_dim), dtype=self.dtype, device=self.device) if out is None else out
            lse = torch.empty((n, heads), dtype=torch.float32, device=self.device) if return_lse else None
            if n:
                a = KvAttend(q=q.data_ptr(), out=o.data_ptr(), lse=None if lse is None else lse.data_ptr(),
                             block_table=block_table.data_ptr(), seq_lens=seq_lens.data_ptr(), table_stride=block_table.stride(0),
                             window=window, sinks=sinks, batch=n, n_q_heads=heads, table_width=block_table.shape[1],
                             scale=self.head_dim ** -0.5 if scale is None else scale)
                a.q_stride[:], a.out_stride[:] = q.stride()[:2], o.stride()[:2]
                scratch = self._scratch()
                check(self.lib.bam_launch_kv_attend(self.array.h, self._layout(layer), C.byref(a), scratch.data_ptr(),
                                                    self._scratch_bytes, s), "bam_launch_kv_attend")
            return (o, lse) if return_lse else o
        self._layout(layer)
        return self._run(stream, call)
