"""Key/value cache in 8 bits for the block-cached sampler, and the attention over it.

No counterpart in the reference, whose sampler recomputes every position (generate.py:80-92).  Keys and values are held
as 8-bit codes (``"e4m3"``: OCP float8, ``"int8"``) in blocks of 64 tokens and one head, each block of keys and of values
with a power-of-two scale of its own: a third of the memory of the bf16 [Q | K | V] image ``LLaDAModel.kv_cache`` keeps
otherwise, and half the bytes to read per key.  ``generate(cache="dual", kv_dtype="e4m3")`` runs on it; the methods
here are for callers with a loop of their own."""
import torch

from . import _lib

HEAD_DIM = 128


def _overlap(a, b):
    """Whether the memory two tensors span has bytes in common."""
    (a0, a1), (b0, b1) = ((t.data_ptr(), t.data_ptr() + (sum((n - 1) * s for n, s in zip(t.shape, t.stride())) + 1) * t.element_size()) for t in (a, b))
    return a0 < b1 and b0 < a1


def _output_races(out, q, q_stride):
    """Whether writing ``out`` (contiguous rows) could change queries that another workgroup has yet to read: it overlaps q's rows
    without standing exactly in their places (each query's result replaces it after it has been read)."""
    in_place = out.data_ptr() == q.data_ptr() and (q_stride == out.shape[-1] or out.shape[0] * out.shape[1] == 1)
    return _overlap(out, q) and not in_place


class KVCache8:
    """Keys and values of ``n_layers`` layers, ``n_seq`` sequences of ``seq_len`` tokens and ``n_heads`` heads of 128.

    A new cache holds zeros.  Every method enqueues on the current stream of the cache's device and returns; calls on
    one cache from several streams need the caller's own ordering, like any tensor."""

    def __init__(self, n_seq, seq_len, n_heads, n_layers=1, dtype="e4m3", device="cuda"):
        if dtype not in _lib.KV_TYPES:
            raise NotImplementedError(f"kv cache dtype {dtype!r} (one of {sorted(_lib.KV_TYPES)})")
        if min(n_seq, seq_len, n_heads, n_layers) < 1:
            raise ValueError("a cache needs at least one sequence, token, head and layer")
        if max(n_seq, seq_len, n_heads, n_layers) >= 2 ** 31 or n_seq * n_heads * -(-seq_len // 64) >= 2 ** 31:
            raise ValueError("sequences, tokens, heads and their 64-token blocks are counted in 32 bits")
        if torch.device(device).type != "cuda":
            raise ValueError(f"a KVCache8 lives in GPU memory, not on {device}")
        self.lib = _lib.load()
        self.n_seq, self.seq_len, self.n_heads, self.n_layers, self.dtype = n_seq, seq_len, n_heads, n_layers, dtype
        self.d = n_heads * HEAD_DIM
        self._type = _lib.KV_TYPES[dtype]
        self.layer_bytes = self.lib.llada_kv8_layer_bytes(n_seq, seq_len, n_heads)
        self.data = torch.zeros((n_layers, self.layer_bytes), dtype=torch.uint8, device=device)
        self.device = self.data.device
        self._index = self.device.index
        n_tiles = n_seq * n_heads * ((seq_len + 63) // 64)
        self.data[:, :n_tiles * 8].view(torch.float32).fill_(1.0)      # the scales of all-zero blocks
        self._ws_bytes = {}

    def numel_bytes(self):
        return self.data.numel()

    # -- helpers -------------------------------------------------------------------------------------------------
    def _layer(self, layer):
        if not 0 <= layer < self.n_layers:
            raise IndexError(f"layer {layer} of a cache of {self.n_layers}")
        return self.data.data_ptr() + layer * self.layer_bytes

    def _rows(self, x, n, width, what):
        """x as n rows a sequence at one row stride: (tensor kept alive, row stride)."""
        shape, st = x.shape, x.stride()
        if x.dtype != torch.bfloat16 or x.device != self.device:
            raise ValueError(f"{what}: bfloat16 on {self.device} is wanted, not {x.dtype} on {x.device}")
        if len(shape) == 3:
            ok, row = shape[0] == self.n_seq and shape[1] == n, st[1] if n > 1 else st[0]
            even = self.n_seq == 1 or st[0] == n * row
        else:
            ok, row, even = len(shape) == 2 and shape[0] == self.n_seq * n, st[0], True
        if not ok or shape[-1] < width:
            raise ValueError(f"{what}: [{self.n_seq}, {n}, >= {width}] is wanted, not {list(shape)}")
        if st[-1] != 1 or row < width or row % 8 or not even or x.data_ptr() % 16:
            x = x[..., :width].clone(memory_format=torch.contiguous_format)
            row = width
        return x, row

    def _mask(self, key_mask):
        if key_mask is None:
            return None
        if tuple(key_mask.shape) != (self.n_seq, self.seq_len) or key_mask.device != self.device:
            raise ValueError(f"key_mask: [{self.n_seq}, {self.seq_len}] on {self.device} is wanted, not {list(key_mask.shape)} on {key_mask.device}")
        if key_mask.dtype == torch.bool:
            key_mask = key_mask.view(torch.uint8)
        elif key_mask.dtype != torch.uint8:
            key_mask = (key_mask != 0).view(torch.uint8)
        return key_mask if key_mask.is_contiguous() else key_mask.contiguous()

    def _on_device(self):
        return _lib.on_device(self.device)

    # -- the operators -------------------------------------------------------------------------------------------
    def fill(self, layer, qkv, key_mask=None):
        """Writes every token of ``layer`` from the rows ``qkv`` [n_seq, seq_len, >= 3 d] (bf16 [Q | K | V], of which K and
        V are read).  ``key_mask`` [n_seq, seq_len] (non-zero = attend): a masked token is stored as zeros."""
        self._write(layer, qkv, 0, self.seq_len, key_mask)

    def update(self, layer, qkv, start, key_mask=None):
        """Writes the tokens ``start`` .. ``start + len - 1`` of every sequence from ``qkv`` [n_seq, len, >= 3 d].  The other
        tokens of a 64-token block that the range covers in part are stored anew under the block's new scale."""
        if qkv.dim() != 3:
            raise ValueError(f"update: [n_seq, len, >= {3 * self.d}] is wanted, not {list(qkv.shape)}")
        self._write(layer, qkv, start, qkv.shape[1], key_mask)

    def _write(self, layer, qkv, start, length, key_mask):
        at = self._layer(layer)
        if start < 0 or length < 1 or start + length > self.seq_len:
            raise ValueError(f"tokens {start} .. {start + length - 1} of {self.seq_len}")
        x, stride = self._rows(qkv, length, 3 * self.d, "qkv")
        m = self._mask(key_mask)
        with self._on_device():
            _lib.check(self.lib.llada_kv8_write(x.data_ptr(), stride, _lib.ptr(m), at, self._type, self.n_seq, self.seq_len,
                                                self.n_heads, start, length, _lib.stream_ptr(self._index)))

    def read(self, layer):
        """The values ``layer`` stands for: (keys, values), bf16 [n_seq, seq_len, n_heads, 128]."""
        at = self._layer(layer)
        with self._on_device():
            k, v = torch.empty((2, self.n_seq, self.seq_len, self.n_heads, HEAD_DIM), dtype=torch.bfloat16, device=self.device).unbind(0)
            _lib.check(self.lib.llada_kv8_read(at, self._type, k.data_ptr(), v.data_ptr(), self.n_seq, self.seq_len,
                                               self.n_heads, _lib.stream_ptr(self._index)))
        return k, v

    def attend(self, layer, q, key_mask=None, block=None, block_start=0, out=None):
        """softmax(q k^T / sqrt(128)) v of ``q`` [n_seq, n_q, >= d] (bf16 rows, head h at columns h * 128) over every
        unmasked token, no causal mask -> [n_seq, n_q, d] bf16.  ``block`` [n_seq, len, >= 3 d]: fresh [Q | K | V] rows
        whose keys and values stand in for the cached tokens from ``block_start`` on (the cache is only read); in a
        cached denoise step q and block are the same rows.  A sequence without an unmasked token gives zeros.  ``out`` may be
        q itself where q's rows are d wide and contiguous; any other overlap with what the call reads is refused."""
        at = self._layer(layer)
        if q.dim() != 3 or q.shape[1] < 1:
            raise ValueError(f"q: [{self.n_seq}, n_q, >= {self.d}] is wanted, not {list(q.shape)}")
        n_q = q.shape[1]
        qx, q_stride = self._rows(q, n_q, self.d, "q")
        bx, b_stride, b_len = None, 0, 0
        if block is not None:
            if block.dim() != 3:
                raise ValueError(f"block: [{self.n_seq}, len, >= {3 * self.d}] is wanted, not {list(block.shape)}")
            b_len = block.shape[1]
            if block_start < 0 or b_len < 1 or block_start + b_len > self.seq_len:
                raise ValueError(f"block tokens {block_start} .. {block_start + b_len - 1} of {self.seq_len}")
            bx, b_stride = self._rows(block, b_len, 3 * self.d, "block")
        m = self._mask(key_mask)
        with self._on_device():
            if out is None:
                out = torch.empty((self.n_seq, n_q, self.d), dtype=torch.bfloat16, device=self.device)
            elif tuple(out.shape) != (self.n_seq, n_q, self.d) or out.dtype != torch.bfloat16 or out.device != self.device or not out.is_contiguous() or out.data_ptr() % 16:
                raise ValueError(f"out: a contiguous bfloat16 [{self.n_seq}, {n_q}, {self.d}] on {self.device} is wanted")
            elif bx is not None and _overlap(out, bx):
                raise ValueError("out overlaps the block's rows, which every head's queries read")
            elif _overlap(out, self.data) or m is not None and _overlap(out, m):
                raise ValueError("out overlaps the cache or the mask, which are read meanwhile")
            elif _output_races(out, qx, q_stride):
                raise ValueError("out overlaps q's rows without being q itself: queries would be overwritten before they are read")
            need = self._ws_bytes.get(n_q)
            if need is None:
                need = self._ws_bytes[n_q] = self.lib.llada_attn_kv8_workspace_bytes(self.n_seq, n_q, self.seq_len, self.n_heads)
            # scratch of this call alone, from the caching allocator: calls on other streams and captured graphs have their own
            ws = torch.empty(need, dtype=torch.uint8, device=self.device) if need else None
            _lib.check(self.lib.llada_attn_kv8(qx.data_ptr(), q_stride, n_q, at, self._type, _lib.ptr(m), out.data_ptr(), self.n_seq,
                                               self.seq_len, self.n_heads, _lib.ptr(bx), b_stride, block_start, b_len,
                                               _lib.ptr(ws), need, _lib.stream_ptr(self._index)))
        return out
