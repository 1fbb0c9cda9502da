"""A key/value cache of attention heads in the pages of a PageCache.

The rows live in an Array over the store, so a cache larger than GPU memory needs nothing special: pages that are not
resident are fetched by the call that reads them, dirty ones are written back when they are evicted (or by
PageCache.flush).  The calls are asynchronous like every other launch: what goes wrong on the device -- a wait that ran
out, an index outside its range -- is reported by Controller.status() / check_status().
"""
import ctypes as C
import threading
import weakref

from . import _lib
from ._lib import KvAppend, KvAttend, KvLayout, check
from .host import REPLICATE, Array

ROPE_STYLES = {"half": 0, "pairs": 1}

_NO_STRIDE = (0, 0)
_PER_THREAD = 2     # cudaStreamPerThread
_NO_STREAM = (1 << 64) - 1
_scratch = {}       # (device, stream) -> the stream's number, the scratch memory of the launches on that stream
_open, _open_lock = weakref.WeakSet(), threading.RLock()      # (a collection in the midst of it may close another cache)


class KvCache:
    """n_layers x n_blocks blocks of block_tokens tokens for n_kv_heads heads of head_dim elements.

    One page of `cache` holds the keys and the values of one block for one head; block_tokens defaults to what fits (a
    multiple of 16).  A token's slot is block * block_tokens + its place in the block.  `dist` lays the pages over the
    controllers of the cache (REPLICATE or STRIPE), store_byte_offset places them in the store.

    While Controller.status() says that something went wrong, calls do nothing and their results are undefined.

    The calls run on the current stream of the cache's device or on `stream` (a torch stream or a raw handle), in whose
    memory pool their results are; the order between streams, and that tensors live long enough, is the caller's affair as
    for any work on another stream.  (The per-thread default stream is refused: its handle is the same number in every
    thread, and torch's memory pools take it for one stream.)  They may be captured into CUDA graphs.  Results carry no
    gradient."""

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
        if n_blocks > 0x7fffffff or n_kv_heads > 65536:
            raise ValueError("at most 2^31 - 1 blocks and 65536 heads")
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
        self._layouts = [C.byref(KvLayout(0 if dtype == torch.bfloat16 else 1, head_dim, n_kv_heads, block_tokens, n_blocks,
                                          i * n_blocks * n_kv_heads)) for i in range(n_layers)]
        with _open_lock:
            _open.add(self)
        self._scratch_bytes = self.lib.bam_kv_scratch_bytes(self.array.h, self._layouts[0])
        # what every call asks torch, by the short ways where this torch has them: a call takes 13 us in all
        self._current_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)
        self._capturing = getattr(torch._C, "_cuda_isCurrentStreamCapturing", torch.cuda.is_current_stream_capturing)
        self._raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", lambda index: torch.cuda.current_stream(index).cuda_stream)

    def close(self):
        """Waits for the device.  The streams' scratch memory (15 MB each with heads of 128) goes with its last cache."""
        self.array.close()
        with _open_lock:
            _open.discard(self)
            if not any(kv.device == self.device for kv in _open):
                for key in [key for key in _scratch if key[0] == self.device.index]:
                    _scratch.pop(key, None)

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    # ---- arguments ----------------------------------------------------------------------------------------

    def _layout(self, layer):
        if not 0 <= layer < self.n_layers:
            raise ValueError(f"layer {layer} of {self.n_layers}")
        return self._layouts[layer]

    def _on(self, name, t, dtype, ndim):
        if t.dtype is dtype and t.dim() == ndim and t.device == self.device:
            return t
        if t.device != self.device:
            raise ValueError(f"{name} is on {t.device}, the cache on {self.device}")
        if t.dtype != dtype:
            raise ValueError(f"{name} must be {dtype}, not {t.dtype}")
        raise ValueError(f"{name} must have {ndim} dimensions, not {t.dim()}")

    def _heads(self, name, t, n, heads):
        """The strides of a tensor [n, heads, head_dim] whose heads are contiguous."""
        shape, stride = t.shape, t.stride()
        if t.dtype is self.dtype and shape == (n, heads, self.head_dim) and stride[2] == 1 and t.device == self.device:
            return stride[:2]
        self._on(name, t, self.dtype, 3)
        if shape != (n, heads, self.head_dim):
            raise ValueError(f"{name} has shape {tuple(shape)}, wanted ({n}, {heads}, {self.head_dim})")
        if stride[2] != 1:
            raise ValueError(f"the elements of a head of {name} must be contiguous")
        return stride[:2]

    def _rows(self, name, t, n, heads):
        """The same of a tensor that is written."""
        stride = self._heads(name, t, n, heads)
        if (n > 1 and stride[0] < self.head_dim) or (heads > 1 and stride[1] < self.head_dim):
            raise ValueError(f"the rows of {name} lie on one another")
        return stride

    @staticmethod
    def _changed(*tensors):
        """The caller's tensors that a launch writes: autograd is to notice if it has saved them."""
        import torch
        for t in tensors:
            if not t.is_inference():
                torch.autograd.graph.increment_version(t)

    def _flat(self, name, t, dtype, n):
        """The address of n contiguous values."""
        if not (t.dtype is dtype and t.shape == (n,) and t.is_contiguous() and t.device == self.device):
            self._on(name, t, dtype, 1)
            if t.shape[0] != n or (n > 1 and t.stride(0) != 1):
                raise ValueError(f"{name} must be {n} contiguous values")
        return t.data_ptr()

    def _on_stream(self, stream):
        """`stream` (a torch stream or a raw handle) as the context the call takes its memory and runs in."""
        import torch
        if not isinstance(stream, torch.cuda.Stream):
            stream = (stream.value or 0) if isinstance(stream, C.c_void_p) else int(stream)
            if stream == _PER_THREAD:
                raise ValueError("the per-thread default stream is not supported")
            stream = torch.cuda.ExternalStream(stream, device=self.device)
        if stream.device != self.device:
            raise ValueError(f"the stream is on {stream.device}, the cache on {self.device}")
        return torch.cuda.stream(stream)

    def _new_scratch(self, stream):
        import torch
        scratch = torch.empty(self._scratch_bytes, dtype=torch.uint8, device=self.device)
        check(self.lib.bam_kv_scratch_init(self.array.h, scratch.data_ptr(), self._scratch_bytes, stream), "bam_kv_scratch_init")
        return scratch

    def _scratch_of(self, stream):
        """The scratch memory of a stream, whose launches run one after the other (and share it between all caches of the
        device).  A handle may be given out again when its stream is gone, possibly while that one's last launch still runs;
        the number of a stream is its own."""
        if stream == _PER_THREAD:
            raise ValueError("the per-thread default stream is not supported")
        number = self.lib.bam_kv_stream_id(stream)
        had, scratch = _scratch.get((self.device.index, stream), (number, None))
        if number == _NO_STREAM:
            raise RuntimeError(f"{stream:#x} is no stream")
        if had != number:
            import torch
            torch.cuda.synchronize(self.device)
            scratch = None
        if scratch is None or scratch.numel() < self._scratch_bytes:
            scratch = self._new_scratch(stream)
            _scratch[self.device.index, stream] = number, scratch
        return scratch

    def _call(self, launch, layer, *args):
        """A launch on the current stream of the cache's device, with scratch memory that no launch uses at the same time: that
        of the stream, or, for a captured launch, its own, which belongs to its graph."""
        index = self.device.index
        if self._current_device() != index:
            import torch
            with torch.cuda.device(index):
                return self._call(launch, layer, *args)
        stream = self._raw_stream(index)
        scratch = self._new_scratch(stream) if self._capturing() else self._scratch_of(stream)
        check(launch(self.array.h, layer, *args, scratch.data_ptr(), self._scratch_bytes, stream), launch.__name__)

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
        if stream is not None:
            with self._on_stream(stream):
                return self.append(k, v, slots, layer, positions, rope, rope_style, q, q_norm, k_norm, norm_eps, q_out)
        n = k.shape[0] if k.dim() else 0
        k_stride, v_stride = self._heads("k", k, n, self.n_kv_heads), self._heads("v", v, n, self.n_kv_heads)
        at = self._flat("slots", slots, torch.int64, n)
        turn = 0, 0, 0, 0, 0, 0, 0                       # positions, cos, sin, rows, their stride, rotated elements, style
        if rope is not None:
            cos, sin = rope
            self._on("cos", cos, torch.float32, 2)
            self._on("sin", sin, torch.float32, 2)
            if rope_style not in ROPE_STYLES:
                raise ValueError(f"rope_style must be one of {sorted(ROPE_STYLES)}, not {rope_style!r}")
            if positions is None:
                raise ValueError("a rotation needs positions")
            (rows, half), stride = cos.shape, cos.stride()
            if sin.shape != cos.shape or sin.stride() != stride or stride[1] != 1 or rows == 0:
                raise ValueError("cos and sin must be rows of the same shape and strides")
            if half % 8 or not 0 < 2 * half <= self.head_dim:
                raise ValueError(f"{2 * half} rotated elements: a multiple of 16 up to {self.head_dim} is wanted")
            turn = (self._flat("positions", positions, torch.int64, n), cos.data_ptr(), sin.data_ptr(), rows, stride[0], 2 * half,
                    ROPE_STYLES[rope_style])
        q_w = None if q_norm is None else self._flat("q_norm", q_norm, self.dtype, self.head_dim)
        k_w = None if k_norm is None else self._flat("k_norm", k_norm, self.dtype, self.head_dim)
        layout = self._layout(layer)
        q_at = out_at = given = None
        heads, q_stride, out_stride = 0, _NO_STRIDE, _NO_STRIDE
        if q is None:
            if q_norm is not None or q_out is not None:
                raise ValueError("q_norm and q_out go with q")
        else:
            if q.dim() != 3 or q.shape[1] < 1:
                raise ValueError("q must be [n, heads, head_dim]")
            heads = q.shape[1]
            q_stride = self._heads("q", q, n, heads)
            if q_out is None:
                q_out = torch.empty((n, heads, self.head_dim), dtype=self.dtype, device=self.device)
                out_stride = heads * self.head_dim, self.head_dim
            else:
                out_stride = self._rows("q_out", q_out, n, heads)
                given = q_out
            q_at, out_at = q.data_ptr(), q_out.data_ptr()
        if n:
            a = KvAppend(q_at, k.data_ptr(), v.data_ptr(), out_at, q_stride, k_stride, v_stride, out_stride, n, at, *turn[:5],
                         q_w, k_w, heads, turn[5], turn[6], norm_eps)
            self._call(self.lib.bam_launch_kv_append, layout, C.byref(a))
            if given is not None:
                self._changed(given)
        return q_out

    def gather(self, slots, layer=0, out=None, stream=None):
        """The rows at `slots` (int64; negative: zeros) as (k, v), each [n, n_kv_heads, head_dim]; `out`: a pair of
        tensors of that shape, with any strides of tokens and heads, to write them to."""
        import torch
        if stream is not None:
            with self._on_stream(stream):
                return self.gather(slots, layer, out)
        n = slots.shape[0] if slots.dim() == 1 else -1
        at = self._flat("slots", slots, torch.int64, n)
        layout = self._layout(layer)
        if out is None:
            k, v = torch.empty((2, n, self.n_kv_heads, self.head_dim), dtype=self.dtype, device=self.device).unbind()
            ks = vs = (C.c_int64 * 2)(self.n_kv_heads * self.head_dim, self.head_dim)
        else:
            k, v = out
            ks = (C.c_int64 * 2)(*self._rows("out[0]", k, n, self.n_kv_heads))
            vs = (C.c_int64 * 2)(*self._rows("out[1]", v, n, self.n_kv_heads))
        if n:
            self._call(self.lib.bam_launch_kv_gather, layout, n, at, k.data_ptr(), v.data_ptr(), ks, vs)
            if out is not None:
                self._changed(k, v)
        return k, v

    def attend(self, q, block_table, seq_lens, layer=0, scale=None, window=0, sinks=0, out=None, return_lse=False, stream=None):
        """Attention of one new token per sequence: q [batch, heads, head_dim] (heads a multiple of n_kv_heads) over the
        first seq_lens[b] (int32) tokens of sequence b, token j in block block_table[b, j // block_tokens] (int32).

        window > 0: only the last `window` tokens and the first `sinks` are visible; blocks without a visible token are
        not touched, their table entries may be anything.  scale defaults to head_dim ** -0.5.  Returns out, or
        (out, lse) with the logarithm of the softmax's denominator [batch, heads]; a sequence with nothing visible gets
        zeros and -inf.  A score of -infinity hides its token, +infinity or NaN make the head's row NaN; an infinite value
        makes its element infinite (a weight below 2^-126 of the largest is 0, and 0 x infinity NaN).  The new token's own
        key and value have to be appended first.  `out` may be q itself."""
        import torch
        if stream is not None:
            with self._on_stream(stream):
                return self.attend(q, block_table, seq_lens, layer, scale, window, sinks, out, return_lse)
        if q.dim() != 3 or q.shape[1] < 1 or q.shape[1] % self.n_kv_heads:
            raise ValueError(f"q must be [batch, heads, head_dim] with a multiple of {self.n_kv_heads} heads")
        n, heads = q.shape[0], q.shape[1]
        q_stride = self._heads("q", q, n, heads)
        self._on("block_table", block_table, torch.int32, 2)
        (rows, width), stride = block_table.shape, block_table.stride()
        if rows != n or width < 1 or (width > 1 and stride[1] != 1):
            raise ValueError(f"block_table must be {n} rows of contiguous entries")
        lens = self._flat("seq_lens", seq_lens, torch.int32, n)
        if window < 0 or sinks < 0:
            raise ValueError("window and sinks must not be negative")
        layout = self._layout(layer)
        given = out
        if out is None:
            out = torch.empty((n, heads, self.head_dim), dtype=self.dtype, device=self.device)
            out_stride = heads * self.head_dim, self.head_dim
        else:
            out_stride = self._rows("out", out, n, heads)
        lse = torch.empty((n, heads), dtype=torch.float32, device=self.device) if return_lse else None
        if n:
            a = KvAttend(q.data_ptr(), out.data_ptr(), lse.data_ptr() if return_lse else None, q_stride, out_stride, block_table.data_ptr(),
                         lens, stride[0], min(window, 1 << 62), min(sinks, 1 << 62), n, heads, width,
                         self.head_dim ** -0.5 if scale is None else scale)
            self._call(self.lib.bam_launch_kv_attend, layout, C.byref(a))
            if given is not None:
                self._changed(given)
        return (out, lse) if return_lse else out
