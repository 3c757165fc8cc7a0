"""An 8-bit paged KV cache: appending to it, attention over it, and blocks to and from 16-bit caches.

A layer is a ``float8_e4m3fn`` tensor ``[2, blocks, block_size, kv_heads, head_dim]`` (0: keys, 1: values;
any strides with the last axis contiguous, so vLLM's orders are views of it) and a ``float32`` tensor
``[blocks, 2, kv_heads]``: one scale a block, side and KV head. A code ``c`` at scale ``s`` stands for
``c * s``. Scales are powers of two, the smallest with ``amax <= 448 s``; 0 for a block of zeros.

Half the bytes of the 16-bit caches the data plane saves: a session's attention reads half as much, and
``TorchBlockDataPlane(cache.codes, block_size, capacity, scales=cache.scales)`` saves and restores it over
the host link in half the time, scales included.

    cache = PagedCache8.allocate(names, blocks, 16, kv_heads=8, head_dim=128, device="cuda")
    batch = PagedBatch(block_table, query_start, lengths, max_query=1)       # one step's sequences
    query = cache.append(name, key, value, batch, query=query, rotary=rotary_table(40960, 128, 1e6))
    out = cache.attend(name, query, batch)

Every call runs on the caller's current stream of the cache's device, allocates only its outputs and
workspaces there, never waits for the GPU, and can be captured into a CUDA graph (block ids given as lists
are copied to the GPU first: both need tensors). Tables and lengths are read on the GPU; what a kernel finds
wrong with them it skips and records, and ``check()`` raises. For serving: no gradients are taken, and rows
that ask for some are refused (call under ``torch.no_grad()`` or ``torch.inference_mode()``).
"""
from __future__ import annotations

import ctypes as C

from . import _abi
from .dataplane import _dp, _load

_PROBLEMS = {
    _abi.BAD_BLOCK: "a block id outside the cache",
    _abi.C8_BAD_LENGTH: "a sequence's length or query rows that do not fit the block table, the rows or max_query",
    _abi.C8_BAD_POSITION: "a position behind the rotary table's end",
    _abi.C8_STALLED: "a wait inside a kernel ran out: its results are not valid",
}


def rotary_table(positions, rotary_dim, base=10000.0, *, device="cuda"):
    """``[positions, rotary_dim / 2, 2]`` float32: (cos, sin) of position * base ** (-2 i / rotary_dim).

    Angles are taken in 64 bits: in 32 a position of 100,000 is off by up to 0.004 radian.
    """
    import torch
    if rotary_dim <= 0 or rotary_dim % 16:
        raise ValueError("rotary_dim must be a positive multiple of 16")
    rate = float(base) ** (-torch.arange(0, rotary_dim, 2, dtype=torch.float64, device=device) / rotary_dim)
    angle = torch.arange(positions, dtype=torch.float64, device=device)[:, None] * rate
    return torch.stack((angle.cos(), angle.sin()), dim=-1).to(torch.float32)


def _type_of(dtype):
    import torch
    if dtype is torch.bfloat16:
        return _abi.C8_BF16
    if dtype is torch.float16:
        return _abi.C8_FP16
    raise ValueError(f"16-bit rows are bfloat16 or float16, not {dtype}")


def _raw_stream():
    """The function from a device's index to its current stream's handle."""
    import torch
    # current_stream() makes a Stream object a call, 2.3 us of a 12 us append.
    return getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda i: torch.cuda.current_stream(i).cuda_stream)


class PagedBatch:
    """The sequences of one model step, as the engine lays them out on the GPU.

    ``table`` int32 ``[sequences, width]``: block ids of each sequence's pages in order. ``start`` int32
    ``[sequences + 1]``: sequence s owns token rows ``start[s]:start[s + 1]`` of the step's tensors, and they
    are its last tokens. ``lengths`` int32 ``[sequences]``: tokens of each sequence with the new ones (0 for a
    padded entry). ``max_query``: an upper bound of the rows of any sequence (1 for a decode step), known to
    the host; without it, no bound. The arrays may be rewritten between steps: nothing of them is kept.
    """

    def __init__(self, table, start, lengths, *, max_query=None):
        import torch
        for name, tensor, ndim in (("table", table, 2), ("start", start, 1), ("lengths", lengths, 1)):
            if tensor.dtype != torch.int32 or tensor.ndim != ndim or tensor.device.type != "cuda":
                raise ValueError(f"{name} must be a {ndim}-D int32 CUDA tensor")
            if tensor.device != table.device:
                raise ValueError("one CUDA device required")
            if tensor.numel() and tensor.stride(-1) != 1 and tensor.shape[-1] > 1:
                raise ValueError(f"{name} must be contiguous along its last axis")
        seqs = lengths.shape[0]
        if table.shape[0] != seqs or start.shape[0] != seqs + 1:
            raise ValueError("table, start and lengths must describe the same sequences")
        if max(table.shape) >= 1 << 30:
            raise ValueError("the block table is too large")
        if max_query is not None and (type(max_query) is not int or max_query < 0):
            raise ValueError("max_query must be a non-negative int")
        self.table, self.start, self.lengths, self.max_query = table, start, lengths, max_query
        self.device, self.seqs = table.device, seqs
        self._addresses = (table.data_ptr(), start.data_ptr(), lengths.data_ptr(), table.stride(0), table.shape[1], seqs)
        self._records, self._workspaces = {}, {}

    def _for(self, rows):
        """The call's record for tensors of ``rows`` rows (a few row counts are kept: they are the caller's steps)."""
        record = self._records.get(rows)
        if record is None:
            if len(self._records) > 64:
                self._records.clear()
            record = _abi.C8Batch(*self._addresses, rows, rows if self.max_query is None else min(rows, self.max_query))
            self._records[rows] = record
        return record


class PagedCache8:
    """The 8-bit paged caches of a model's layers, by layer name (all of one geometry, on one device).

    ``codes[name]``: float8_e4m3fn ``[2, blocks, block_size, kv_heads, head_dim]``, ``scales[name]``: float32
    ``[blocks, 2, kv_heads]``. head_dim is 64 or 128, block_size a multiple of 16.
    """

    def __init__(self, codes, scales):
        import torch
        if not codes:
            raise ValueError("empty KV cache registration")
        if set(codes) != set(scales):
            raise ValueError("codes and scales must name the same layers")
        first = next(iter(codes.values()))
        shape = tuple(first.shape)
        if first.device.type != "cuda":
            raise ValueError("one CUDA device required")
        if len(shape) != 5 or shape[0] != 2 or min(shape) == 0:
            raise ValueError("codes are [2, blocks, block_size, kv_heads, head_dim]")
        if shape[4] not in (64, 128):
            raise ValueError("head_dim must be 64 or 128")
        if shape[2] % 16:
            raise ValueError("block_size must be a multiple of 16")
        self.device, self.block_size, self.kv_heads, self.head_dim = first.device, *shape[2:]
        self.codes, self.scales, self._records = dict(codes), dict(scales), {}
        for name, tensor in self.codes.items():
            scale = self.scales[name]
            if tensor.device != self.device or scale.device != self.device:
                raise ValueError("one CUDA device required")
            if tensor.dtype != torch.float8_e4m3fn or tuple(tensor.shape[2:]) != shape[2:] or tensor.ndim != 5 \
                    or tensor.shape[0] != 2:
                raise ValueError(f"layer {name}: codes must be float8_e4m3fn [2, blocks, {shape[2]}, {shape[3]}, {shape[4]}]")
            if scale.dtype != torch.float32 or tuple(scale.shape) != (tensor.shape[1], 2, shape[3]) \
                    or not scale.is_contiguous():
                raise ValueError(f"layer {name}: scales must be contiguous float32 [blocks, 2, kv_heads]")
            pitches = tensor.stride()
            if pitches[4] != 1 or tensor.data_ptr() % 16 or any(p % 16 or p < 0 for p in pitches[:4]):
                raise ValueError(f"layer {name}: codes must have a contiguous head_dim and 16-byte aligned strides")
            self._records[name] = _abi.C8Cache(tensor.data_ptr(), scale.data_ptr(), *pitches[:4], tensor.shape[1],
                                               *shape[2:], self.device.index, 0)
        self._lib, self._current_stream, self._index = _dp(_load()), _raw_stream(), first.device.index
        self._grad_enabled = torch.is_grad_enabled
        if not hasattr(self._lib, "kvsnap_c8_append"):
            raise RuntimeError("the CUDA library has no 8-bit cache kernels; rebuild with python -m kvsnap_b200.build")
        self.status = torch.zeros(1, dtype=torch.int32, device=self.device)
        self._status_at = self.status.data_ptr()

    @classmethod
    def allocate(cls, layers, blocks, block_size, kv_heads, head_dim, *, device="cuda"):
        """Empty caches (all zeros) for ``layers``, in the ``[2, blocks, block_size, kv_heads, head_dim]`` order."""
        import torch
        shape = (2, blocks, block_size, kv_heads, head_dim)
        codes = {name: torch.zeros(shape, dtype=torch.float8_e4m3fn, device=device) for name in layers}
        return cls(codes, {name: torch.zeros((blocks, 2, kv_heads), device=device) for name in layers})

    # ---- arguments -------------------------------------------------------------------------

    def _layer(self, layer):
        record = self._records.get(layer)
        if record is None:
            raise KeyError(f"no 8-bit cache layer named {layer!r}")
        return record

    def _rows(self, what, tensor, heads=None):
        """(address, token pitch, head pitch) in bytes of ``[rows, heads, head_dim]`` 16-bit rows."""
        if tensor.device != self.device:
            raise ValueError(f"{what} must be on {self.device}")
        if tensor.requires_grad and self._grad_enabled():
            raise ValueError(f"{what} requires a gradient, which the 8-bit cache does not take: call under torch.no_grad()")
        shape = tensor.shape
        if len(shape) != 3 or shape[2] != self.head_dim or (heads and shape[1] != heads):
            raise ValueError(f"{what} must be [rows, {heads or 'heads'}, {self.head_dim}]")
        token, head, element = tensor.stride()
        at = tensor.data_ptr()
        if element != 1 or token < 0 or head < 0:
            raise ValueError(f"{what} must have a contiguous head_dim")
        token = 2 * token if shape[0] > 1 else 0             # an axis of one element is never stepped along
        head = 2 * head if shape[1] > 1 else 0
        if (at | token | head) & 15:
            raise ValueError(f"{what} must be 16-byte aligned in every row")
        return at, token, head

    def _batch(self, batch, rows):
        if batch.device != self.device:
            raise ValueError(f"the batch must be on {self.device}")
        return batch._for(rows)

    def _check(self, rc):
        if rc < 0:
            raise RuntimeError(self._lib.kvsnap_cuda_error().decode())

    # ---- operators -------------------------------------------------------------------------

    def append(self, layer, key, value, batch, *, query=None, rotary=None, interleaved=False):
        """Write the step's new keys and values ``[rows, kv_heads, head_dim]`` into their pages of ``layer``.

        ``rotary``: a :func:`rotary_table` (any rotary_dim up to head_dim); keys are rotated on the way in 32
        bits, pairs (i, i + rotary_dim / 2) or, ``interleaved``, (2i, 2i + 1). ``query`` ``[rows, q_heads,
        head_dim]`` is rotated the same way, and returned as a new tensor (None without ``query``). Its rows
        that are no sequence's, or whose position would be negative or lies behind the table, are unspecified.
        Tokens behind the table are not written, and reported by :meth:`check`.

        A page's scale only grows while tokens are added to it, older codes being rounded again; a page whose
        first slot is written starts anew. Slots behind a sequence's last token keep their codes. Sequences
        of one call must not share a page that one of them appends to. Infinities become the largest value
        the page's scale holds; NaN stays NaN; neither sets a scale.
        """
        import torch
        cache, dtype = self._layer(layer), key.dtype
        rows, kind = key.shape[0], _type_of(dtype)
        k, v = self._rows("key", key, self.kv_heads), self._rows("value", value, self.kv_heads)
        if value.dtype is not dtype or value.shape[0] != rows:
            raise ValueError("key and value must have the same rows and type")
        q, q_heads, out, out_at = (None, 0, 0), 0, None, None
        if query is not None:
            q, shape = self._rows("query", query), query.shape
            if query.dtype is not dtype or shape[0] != rows or not shape[1]:
                raise ValueError("query must have the keys' rows and type, and at least one head")
            q_heads = shape[1]
        table, positions, rotary_dim = None, 0, 0
        if rotary is not None:
            if rotary.dtype is not torch.float32 or rotary.ndim != 3 or rotary.device != self.device \
                    or not rotary.is_contiguous():
                raise ValueError(f"rotary must be a contiguous float32 [positions, rotary_dim / 2, 2] on {self.device}")
            positions, half, two = rotary.shape
            table, rotary_dim = rotary.data_ptr(), 2 * half
            if two != 2:
                raise ValueError("rotary must hold (cos, sin) in its last axis")
            if rotary_dim <= 0 or rotary_dim % 16 or rotary_dim > self.head_dim or not positions:
                raise ValueError("rotary_dim must be a multiple of 16 up to head_dim, for at least one position")
            if table % 16:
                raise ValueError("rotary must be 16-byte aligned")
        elif query is not None:
            raise ValueError("query is only rotated: it needs rotary")
        record = self._batch(batch, rows)
        if query is not None:
            out = torch.empty_like(query, memory_format=torch.contiguous_format)
            out_at = out.data_ptr()
        self._check(self._lib.kvsnap_c8_append(cache, record, kind, *k, *v, *q, q_heads, out_at, table, positions,
                                               rotary_dim, bool(interleaved), self._status_at,
                                               self._current_stream(self._index)))
        return out

    def attend(self, layer, query, batch, *, scale=None, out=None):
        """Causal attention of ``query`` ``[rows, q_heads, head_dim]`` over the sequences' cached tokens of ``layer``.

        Row i of a sequence sees its positions up to its own, the new tokens' own keys (already appended)
        included. ``scale`` (not negative) multiplies the scores, 1 / sqrt(head_dim) by default. Query heads g * group to
        (g + 1) * group - 1 share KV head g. ``out``: a contiguous tensor like ``query`` to write to. A row
        that sees no token is zeros; rows that are no sequence's are left as they are in ``out`` (unspecified
        without it), and so are those of a sequence that does not fit. ``out`` may be ``query``.

        Sums and the softmax's statistics are 32-bit. A weight times its page's value scale is rounded to 16 bits
        once: by at most 2^-11 of itself or 2^-24 of the row's largest such product, whichever is more (in
        sequences of many new rows a page's scale counts for the latter as up to 2^6 more, where its neighbours' are).
        A scale that is no power of two is itself rounded to 16 bits there.

        Sequences of up to 16 rows a KV head (query heads of a group times new tokens) are read at the memory's
        rate; others, groups of more than 16 heads among them, 256 rows at a time.
        """
        import torch
        cache, dtype, shape = self._layer(layer), query.dtype, query.shape
        kind, q = _type_of(dtype), self._rows("query", query)
        rows, q_heads, _ = shape
        if not q_heads or q_heads % self.kv_heads:
            raise ValueError("query heads must be a multiple of the KV heads")
        scale = self.head_dim ** -0.5 if scale is None else float(scale)
        if not 0.0 <= scale < 3.4e38:
            raise ValueError("scale must be finite and not negative")
        if out is not None:
            if out.shape != shape or out.dtype is not dtype or out.device != self.device or not out.is_contiguous():
                raise ValueError("out must be a contiguous tensor of the query's shape, type and device")
            if out.data_ptr() % 16:
                raise ValueError("out must be 16-byte aligned")
        record = self._batch(batch, rows)
        # What a call of these sizes needs is asked once.
        sizes = (rows, q_heads, self.kv_heads, self.head_dim, self.block_size)
        size = batch._workspaces.get(sizes)
        if size is None:
            needed = C.c_size_t()
            self._check(self._lib.kvsnap_c8_attend_workspace(cache, record, q_heads, needed))
            if len(batch._workspaces) > 64:
                batch._workspaces.clear()
            size = batch._workspaces[sizes] = needed.value
        if out is None:
            out = torch.empty_like(query, memory_format=torch.contiguous_format)
        # A workspace of the call's own, from the stream's (or the capture's) memory: no two calls share one.
        workspace = self.status.new_empty(size // 4) if size else None
        self._check(self._lib.kvsnap_c8_attend(cache, record, kind, *q, q_heads, scale, out.data_ptr(),
                                               workspace.data_ptr() if size else None, size, self._status_at,
                                               self._current_stream(self._index)))
        return out

    def converter(self, caches):
        """A :class:`CacheConverter` between this cache and 16-bit ``caches`` (layer name -> tensor)."""
        return CacheConverter(self, caches)

    def check(self):
        """Wait for the calls so far, on all streams, and raise ``ValueError`` if a kernel met an argument it had to skip."""
        import torch
        torch.cuda.synchronize(self.device)
        found = int(self.status.item())
        if found:
            self.status.zero_()
            torch.cuda.synchronize(self.device)              # before a call on another stream records anew
            raise ValueError("8-bit cache: " + "; ".join(text for bit, text in _PROBLEMS.items() if found & bit))


class CacheConverter:
    """Whole blocks between an 8-bit cache and 16-bit caches of the same geometry, every layer in one launch.

    ``caches``: some of the 8-bit cache's layers by name, each bfloat16 or float16 ``[2, blocks, block_size,
    kv_heads, head_dim]`` (one type; the last axis contiguous). For a session restored from a 16-bit snapshot
    and served in 8 bits, or the other way round.
    """

    def __init__(self, cache, caches):
        import torch
        if not caches:
            raise ValueError("empty KV cache registration")
        self.cache, self.caches = cache, dict(caches)
        pairs = (_abi.C8Pair * len(self.caches))()
        kinds = set()
        geometry = (cache.block_size, cache.kv_heads, cache.head_dim)
        for pair, (name, wide) in zip(pairs, self.caches.items()):
            record = cache._layer(name)
            if wide.device != cache.device:
                raise ValueError("one CUDA device required")
            if wide.ndim != 5 or wide.shape[0] != 2 or tuple(wide.shape[2:]) != geometry:
                raise ValueError(f"layer {name}: 16-bit cache must be [2, blocks, {geometry[0]}, {geometry[1]}, {geometry[2]}]")
            kinds.add(_type_of(wide.dtype))
            pitches = [2 * p for p in wide.stride()]
            if pitches[4] != 2 or wide.data_ptr() % 16 or any(p % 16 or p < 0 for p in pitches[:4]):
                raise ValueError(f"layer {name}: 16-bit cache must have a contiguous head_dim and 16-byte aligned strides")
            pair.codes, pair.scales = record.codes, record.scales
            pair.side_pitch, pair.block_pitch = record.side_pitch, record.block_pitch
            pair.token_pitch, pair.head_pitch = record.token_pitch, record.head_pitch
            pair.wide = wide.data_ptr()
            pair.wide_side, pair.wide_block, pair.wide_token, pair.wide_head = pitches[:4]
            pair.blocks, pair.wide_blocks = record.blocks, wide.shape[1]
        if len(kinds) != 1:
            raise ValueError("16-bit caches must have one type")
        self._kind = kinds.pop()
        self._pairs = torch.frombuffer(bytearray(bytes(pairs)), dtype=torch.uint8).to(cache.device)
        self._pairs_at = self._pairs.data_ptr()

    def _ids(self, ids):
        import torch
        if not isinstance(ids, torch.Tensor):
            ids = torch.tensor(list(ids), dtype=torch.int64).to(self.cache.device)
        if ids.dtype is not torch.int64 or ids.ndim != 1 or ids.device != self.cache.device or not ids.is_contiguous():
            raise ValueError(f"block ids are a list or a contiguous 1-D int64 tensor on {self.cache.device}")
        return ids

    def _call(self, entry, source, target, *valid):
        cache = self.cache
        source, target = self._ids(source), self._ids(target)
        count = source.shape[0]
        if target.shape[0] != count:
            raise ValueError("one source per block is required")
        cache._check(entry(self._pairs_at, len(self.caches), cache.block_size, cache.kv_heads, cache.head_dim, self._kind,
                           source.data_ptr(), target.data_ptr(), count, *valid, cache._status_at, cache._index,
                           cache._current_stream(cache._index)))

    def compress(self, source_blocks, blocks, num_kv_tokens=None):
        """16-bit blocks ``source_blocks[i]`` into 8-bit blocks ``blocks[i]``, with new scales.

        ``num_kv_tokens``: tokens that the blocks hold, in order; slots behind the last become zeros, as a
        save zeroes them (None: every slot counts). Block ids are lists, or int64 tensors on the cache's
        device. A target block must not be named twice.
        """
        if num_kv_tokens is not None and (type(num_kv_tokens) is not int or num_kv_tokens < 0):
            raise ValueError("num_kv_tokens must be a non-negative int")
        self._call(self.cache._lib.kvsnap_c8_compress, source_blocks, blocks, -1 if num_kv_tokens is None else num_kv_tokens)

    def expand(self, blocks, target_blocks):
        """8-bit blocks ``blocks[i]`` into 16-bit blocks ``target_blocks[i]``: exact in bfloat16 up to its
        smallest normal number, rounded once in float16."""
        self._call(self.cache._lib.kvsnap_c8_expand, blocks, target_blocks)
