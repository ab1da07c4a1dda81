"""A KV cache in 8 bits, in blocks: tables made on the GPU, a quantising write, and the attention that reads it.

Half the bytes of a bf16 pool on the path that KV bytes bound:

* :class:`BlockTables` — which blocks a request holds and the slots of a step's new tokens
  (``qq_block_plan``, ``qq_block_trim``): free blocks wait in a ring on the device, so a step is planned
  from device lengths with no host round trip.  It also fills a ``req_to_token`` map, the table the page
  selection (:class:`~qwenquest_b200.quest.QuestAlgorithm`) translates its positions through.
* :class:`KV8Cache` — per layer e4m3 codes ``[blocks, kv_heads, block, head_dim]`` and fp32 scales
  ``[blocks, kv_heads]``: :meth:`~KV8Cache.append`, :meth:`~KV8Cache.gather`, and the attention of one token
  per request over its whole sequence (:meth:`~KV8Cache.decode_attention`) or over selected rows
  (:meth:`~KV8Cache.sparse_decode_attention`), and of a prefill batch (:meth:`~KV8Cache.extend_attention`):
  what :func:`~qwenquest_b200.kernels.sparse_decode_attention` and
  :func:`~qwenquest_b200.kernels.extend_attention` do over a bf16 pool.

A step::

    slots, offsets = tables.plan(reqs, seq_lens, prefix_lens, num_tokens)
    cache.append(layer, k, v, slots)
    out = cache.decode_attention(layer, q, tables.block_table, reqs, seq_lens, scaling)

Nothing here waits for the GPU.  What a kernel finds wrong (an index out of range, no free block) is kept in an
error word and raised by the next call on the object or by ``check_errors``; ``synchronize`` waits first.
Calls run on the current stream of the object's device.  Plans and trims of one set of tables go one after another;
appends of several streams may overlap where they write different blocks, and attention calls share nothing.
"""

from __future__ import annotations

import ctypes

import torch

from qwenquest_b200 import _lib
from qwenquest_b200._device import DeviceError, dtype_code
from qwenquest_b200._lib import check

__all__ = ["BlockTables", "KV8Cache"]

BLOCK_SIZES = (16, 32, 64, 128)


def _as_int(t: torch.Tensor, dtype: torch.dtype, name: str, device: torch.device) -> torch.Tensor:
    """Integers of another type or place.  Narrowed to 32 bits, those past them become the nearest, which the kernels
    find out of range; cut off they might be numbers in range."""
    if t.numel() and (t.dtype.is_floating_point or t.dtype.is_complex or t.dtype == torch.bool):
        raise ValueError(f"{name}: integers are wanted, got {t.dtype}")
    if dtype == torch.int32 and t.dtype.itemsize >= 4 and t.dtype != torch.int32:
        t = t.to(device=device, dtype=torch.int64).clamp(-2 ** 31, 2 ** 31 - 1)
    return t.to(device=device, dtype=dtype)


def _cuda_device(device) -> torch.device:
    device = torch.device(device)
    if device.type != "cuda":
        raise ValueError("qwenquest_b200 runs on a CUDA device only")
    if device.index is None:
        device = torch.device("cuda", torch.cuda.current_device())
    return device


class _OnDevice:
    """The device, its current stream, and the error word of an object's kernels."""

    def __init__(self, device: torch.device, what: str):
        self.device = device
        self._index = device.index
        self.lib = _lib.load()
        self._what = what
        self._err = DeviceError(torch.zeros(1, dtype=torch.int32).pin_memory())
        self._err_ptr = self._err.ptr()
        self._err_word = ctypes.c_int32.from_address(self._err.word.data_ptr())

    def check_errors(self) -> None:
        """Raise for device errors of earlier calls (no synchronisation)."""
        if self._err_word.value:
            _lib.raise_device_error(self._err.take(), self._what)

    def synchronize(self) -> None:
        """Wait for the device's current stream, then raise what its kernels reported."""
        torch.cuda.current_stream(self.device).synchronize()
        self.check_errors()

    def _call(self, fn, *args) -> None:
        """One entry point, launched on the current stream of the object's device (also when another is current)."""
        index = self._index
        if torch._C._cuda_getDevice() == index:
            rc = fn(*args, torch._C._cuda_getCurrentRawStream(index))
        else:
            with torch.cuda.device(index):
                rc = fn(*args, torch._C._cuda_getCurrentRawStream(index))
        if rc:
            check(rc, fn.__name__)

    def _call_with_scratch(self, size: int, fn, *args) -> None:
        """The same with `size` bytes of scratch, the call's own: calls on several streams, or captured graphs,
        share none.  Asked of the allocator that tensors come from, on the launching stream, and handed back as a
        tensor would be (a tensor around it takes 2 us more)."""
        if not size:
            return self._call(fn, *args, None, 0)
        index = self._index
        if torch._C._cuda_getDevice() != index:
            with torch.cuda.device(index):
                return self._call_with_scratch(size, fn, *args)
        stream = torch._C._cuda_getCurrentRawStream(index)
        scratch = torch._C._cuda_cudaCachingAllocator_raw_alloc(size, stream)
        try:
            rc = fn(*args, scratch, size, stream)
        finally:
            torch._C._cuda_cudaCachingAllocator_raw_delete(scratch)
        if rc:
            check(rc, fn.__name__)

    def _ints(self, t, dtype: torch.dtype, name: str, n: int | None = None) -> torch.Tensor:
        """A contiguous device vector of `dtype`; lists and tensors elsewhere are copied over."""
        if not isinstance(t, torch.Tensor):
            t = torch.as_tensor(t)
        if t.dtype != dtype or t.get_device() != self._index:
            t = _as_int(t, dtype, name, self.device)
        if t.dim() != 1 or (n is not None and t.shape[0] != n):
            raise ValueError(f"{name} must be [{'n' if n is None else n}], got {tuple(t.shape)}")
        return t if t.is_contiguous() else t.contiguous()


class BlockTables(_OnDevice):
    """Block tables of up to ``max_reqs`` requests over ``num_blocks`` blocks.

    ``block_table`` int32 ``[max_reqs, max_blocks]`` (-1: no block), ``held`` int32 ``[max_reqs]``,
    ``free_blocks`` int32 ``[num_blocks]`` and ``ring`` int64 ``[2]`` (blocks taken and given back, all
    time) are device tensors a caller may read.  Free blocks go out in the order they came back.
    """

    def __init__(self, num_blocks: int, max_reqs: int, max_blocks: int, device, *, block_size: int = 64):
        device = _cuda_device(device)
        if num_blocks <= 0 or max_reqs <= 0 or max_blocks <= 0:
            raise ValueError("num_blocks, max_reqs and max_blocks must be > 0")
        i32 = dict(dtype=torch.int32, device=device)
        self._setup(torch.full((max_reqs, max_blocks), -1, **i32), torch.zeros(max_reqs, **i32),
                    torch.arange(num_blocks, **i32), torch.tensor([0, num_blocks], dtype=torch.int64, device=device),
                    block_size)

    @classmethod
    def from_tensors(cls, block_table: torch.Tensor, held: torch.Tensor, free_blocks: torch.Tensor,
                     ring: torch.Tensor, block_size: int = 64) -> BlockTables:
        """Tables around a caller's own tensors (kept, not copied): for state that lives elsewhere."""
        self = cls.__new__(cls)
        self._setup(block_table, held, free_blocks, ring, block_size)
        return self

    def _setup(self, block_table, held, free_blocks, ring, block_size) -> None:
        if block_size not in BLOCK_SIZES:
            raise ValueError(f"block_size must be one of {BLOCK_SIZES}, got {block_size}")
        if block_table.dim() != 2 or block_table.dtype != torch.int32:
            raise ValueError("block_table must be int32 [max_reqs, max_blocks] with contiguous rows")
        reqs, width = block_table.shape
        # what stride() says of a dimension of size 1 is any number
        stride = block_table.stride(0) if reqs > 1 else width
        if (width > 1 and block_table.stride(1) != 1) or stride < width:
            raise ValueError("block_table must be int32 [max_reqs, max_blocks] with contiguous rows")
        for name, t, dtype, shape in (("held", held, torch.int32, (reqs,)), ("ring", ring, torch.int64, (2,)),
                                      ("free_blocks", free_blocks, torch.int32, (free_blocks.numel(),))):
            if t.dtype != dtype or tuple(t.shape) != shape or not t.is_contiguous() or t.device != block_table.device:
                raise ValueError(f"{name} must be a contiguous {dtype} {shape} on {block_table.device}")
        _OnDevice.__init__(self, _cuda_device(block_table.device), "(block tables)")
        self.block_table, self.held, self.free_blocks, self.ring = block_table, held, free_blocks, ring
        self.block_size, self.max_reqs, self.max_blocks = block_size, reqs, width
        self._claim = torch.zeros(reqs, dtype=torch.int32, device=self.device)
        self._tables = _lib.QQBlockTables(
            block_table.data_ptr(), stride, held.data_ptr(), self._claim.data_ptr(),
            free_blocks.data_ptr(), ring.data_ptr(), free_blocks.numel(), reqs, width, block_size)

    def check_errors(self) -> None:
        """Raise for device errors of earlier calls (no synchronisation)."""
        if not self._err_word.value & _lib.QQ_DEV_ERR_CAPACITY:
            return super().check_errors()
        others = self._err.take() & ~_lib.QQ_DEV_ERR_CAPACITY
        try:
            _lib.raise_device_error(others, self._what)
        except RuntimeError as other:
            raise RuntimeError(f"no free block left: some requests of an earlier plan got none; and {other}") from other
        raise RuntimeError("no free block left: some requests of an earlier plan got none")

    def available(self) -> int:
        """Free blocks (reads the device, so it waits)."""
        taken, given = self.ring.tolist()
        return given - taken

    def plan(self, req_pool_indices, seq_lens, prefix_lens, num_tokens: int, *,
             req_to_token: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
        """The blocks and slots of a step: request ``req_pool_indices[i]`` grows from ``prefix_lens[i]`` to
        ``seq_lens[i]`` tokens.

        Returns ``(slots, token_offsets)``: int64 ``[num_tokens]``, the slot of every new token in batch order
        (-1 behind the last one, and for an entry that is refused), and int64 ``[bs + 1]``, the first row of each
        entry.  An entry of ``seq_lens`` 0 is padding.  ``req_to_token`` (int32 ``[rows, max_context]``; columns
        of a wider map where they hold ``max_blocks * block_size`` positions) gets the slots by request and position.  A batch that runs out of blocks raises ``RuntimeError`` at the next
        check; the entries that no longer fit are left as they were.
        """
        if self._err_word.value:
            self.check_errors()
        reqs = self._ints(req_pool_indices, torch.int64, "req_pool_indices")
        bs = reqs.shape[0]
        seq = self._ints(seq_lens, torch.int64, "seq_lens", bs)
        prefix = self._ints(prefix_lens, torch.int64, "prefix_lens", bs)
        num_tokens = int(num_tokens)
        if num_tokens < 0:
            raise ValueError("num_tokens must be >= 0")
        made = reqs.new_empty(num_tokens + bs + 1)
        slots, offsets = made.split_with_sizes((num_tokens, bs + 1))
        mapped = (None, 0, 0)
        if req_to_token is not None:
            mapped = self._map(req_to_token)
        self._call(self.lib.qq_block_plan, self._tables, reqs.data_ptr(), seq.data_ptr(), prefix.data_ptr(), bs,
                   made.data_ptr(), num_tokens, made.data_ptr() + 8 * num_tokens, *mapped, self._err_ptr)
        return slots, offsets

    def _map(self, t: torch.Tensor) -> tuple[int, int, int]:
        """The map's address, the distance between its rows and their number.  The kernel takes the distance as a
        row's length, so rows that are part of wider ones must hold every position the tables can."""
        if t.dim() != 2 or t.dtype != torch.int32 or t.device != self.device or (t.shape[1] > 1 and t.stride(1) != 1):
            raise ValueError("req_to_token must be int32 [rows, max_context] with contiguous rows on the device")
        rows, width = t.shape
        stride = t.stride(0) if rows > 1 else width
        if stride < width or (stride > width and width < self.max_blocks * self.block_size):
            raise ValueError(f"req_to_token must be contiguous, or at least {self.max_blocks * self.block_size} wide")
        return t.data_ptr(), stride, rows

    def trim(self, req_pool_indices, keep_lens=None) -> None:
        """Requests keep the blocks of their first ``keep_lens[i]`` tokens (``None``: of none, they are finished);
        the others are free again.  A request of -1 is padding."""
        if self._err_word.value:
            self.check_errors()
        reqs = self._ints(req_pool_indices, torch.int64, "req_pool_indices")
        keep = None if keep_lens is None else self._ints(keep_lens, torch.int64, "keep_lens", reqs.shape[0])
        self._call(self.lib.qq_block_trim, self._tables, reqs.data_ptr(), None if keep is None else keep.data_ptr(),
                   reqs.shape[0], self._err_ptr)


class KV8Cache(_OnDevice):
    """Keys and values of ``num_layers`` layers as e4m3 codes with a scale per block of tokens and KV head.

    ``k[layer]``, ``v[layer]``: ``float8_e4m3fn [num_blocks, kv_heads, block_size, head_dim]``;
    ``k_scale[layer]``, ``v_scale[layer]``: fp32 ``[num_blocks, kv_heads]``.  ``head_dim`` a multiple of 8 up to
    256.  Slots are those of :class:`BlockTables` (``block * block_size + offset``).
    """

    def __init__(self, num_layers: int, num_blocks: int, kv_heads: int, head_dim: int, device, *, block_size: int = 64):
        device = _cuda_device(device)
        if min(num_layers, num_blocks, kv_heads, head_dim) <= 0:
            raise ValueError("num_layers, num_blocks, kv_heads and head_dim must be > 0")

        def codes():
            t = torch.zeros((num_blocks, kv_heads, block_size, head_dim), dtype=torch.uint8, device=device)
            return t.view(torch.float8_e4m3fn)

        def scales():
            return torch.zeros((num_blocks, kv_heads), dtype=torch.float32, device=device)

        layers = range(num_layers)
        self._setup([codes() for _ in layers], [codes() for _ in layers], [scales() for _ in layers],
                    [scales() for _ in layers])

    @classmethod
    def from_tensors(cls, k: list[torch.Tensor], v: list[torch.Tensor], k_scale: list[torch.Tensor],
                     v_scale: list[torch.Tensor]) -> KV8Cache:
        """A cache around a caller's own tensors, one of each per layer (kept, not copied).  Scales may be any
        positive numbers (calibrated ones, say); :meth:`append` keeps one that is large enough."""
        self = cls.__new__(cls)
        self._setup(list(k), list(v), list(k_scale), list(v_scale))
        return self

    def _setup(self, k, v, k_scale, v_scale) -> None:
        if not k or not len(k) == len(v) == len(k_scale) == len(v_scale):
            raise ValueError("k, v, k_scale and v_scale must have one tensor per layer")
        shape, device = tuple(k[0].shape), k[0].device
        if len(shape) != 4:
            raise ValueError(f"codes must be [blocks, kv_heads, block, head_dim], got {shape}")
        if shape[2] not in BLOCK_SIZES:
            raise ValueError(f"block_size must be one of {BLOCK_SIZES}, got {shape[2]}")
        if shape[3] % 8 or not 0 < shape[3] <= 256:
            raise ValueError(f"head_dim must be a multiple of 8 up to 256, got {shape[3]}")
        for t in k + v:
            if tuple(t.shape) != shape or t.dtype != torch.float8_e4m3fn or not t.is_contiguous() or t.device != device:
                raise ValueError(f"codes must be contiguous float8_e4m3fn {shape} on {device}")
        for t in k_scale + v_scale:
            if tuple(t.shape) != shape[:2] or t.dtype != torch.float32 or not t.is_contiguous() or t.device != device:
                raise ValueError(f"scales must be contiguous float32 {shape[:2]} on {device}")
        _OnDevice.__init__(self, _cuda_device(device), "(8-bit KV cache)")
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        self.num_layers = len(k)
        self.num_blocks, self.kv_heads, self.block_size, self.head_dim = shape
        words = _lib.QQ_KV8_STATE_WORDS + 2 * self.kv_heads * self.num_blocks
        self._state = torch.zeros((self.num_layers, words), dtype=torch.int32, device=self.device)
        self._layers = [
            _lib.QQKv8Cache(a.data_ptr(), b.data_ptr(), sa.data_ptr(), sb.data_ptr(), st.data_ptr(), self.num_blocks,
                            self.kv_heads, self.head_dim, self.block_size)
            for a, b, sa, sb, st in zip(k, v, k_scale, v_scale, self._state)
        ]
        self._ws_bytes: dict[tuple, int] = {}

    def storage_bytes(self) -> int:
        """Bytes of codes and scales over all layers."""
        return 2 * sum(a.numel() + 4 * s.numel() for a, s in zip(self.k, self.k_scale))

    # ------------------------------------------------------------------ write and read

    def _tokens(self, t: torch.Tensor, name: str) -> tuple[torch.Tensor, int, int]:
        """``[n, kv_heads, head_dim]`` with dense 16-byte aligned rows, its address and the distance between tokens."""
        shape = t.shape
        if len(shape) != 3 or shape[1] != self.kv_heads or shape[2] != self.head_dim or t.get_device() != self._index:
            raise ValueError(f"{name} must be [tokens, {self.kv_heads}, {self.head_dim}] on {self.device}, "
                             f"got {tuple(shape)} on {t.device}")
        token, head, one = t.stride()
        row = self.kv_heads * self.head_dim
        ptr = t.data_ptr()
        if one != 1 or head != self.head_dim or token < row or (token * t.element_size() | ptr) & 15:
            t = t.clone(memory_format=torch.contiguous_format)
            ptr, token = t.data_ptr(), row
        return t, ptr, token

    def append(self, layer: int, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor) -> None:
        """Quantise new tokens (``k``, ``v``: ``[tokens, kv_heads, head_dim]`` bf16 or fp32) into their slots.

        A slot of -1 skips its token.  The tokens of a block stand next to each other in ascending slots, as
        :meth:`BlockTables.plan` gives them; a block met twice in one call is an error, raised at the next
        check, and only the first stretch is written.  A block's scale is a power of two that only grows until a token is written at its offset 0.
        """
        if self._err_word.value:
            self.check_errors()
        k, k_ptr, k_stride = self._tokens(k, "k")
        v, v_ptr, v_stride = self._tokens(v, "v")
        n = k.shape[0]
        if n != v.shape[0] or k.dtype != v.dtype:
            raise ValueError("k and v must have the same tokens and dtype")
        slots = self._ints(slots, torch.int64, "slots", n)
        self._call(self.lib.qq_kv8_append, self._layers[layer], k_ptr, v_ptr, dtype_code(k.dtype), k_stride, v_stride,
                   slots.data_ptr(), n, self._err_ptr)

    def gather(self, layer: int, slots: torch.Tensor, *, dtype: torch.dtype = torch.bfloat16
               ) -> tuple[torch.Tensor, torch.Tensor]:
        """The keys and values of the slots, ``[n, kv_heads, head_dim]`` each; -1 gives zeros."""
        if self._err_word.value:
            self.check_errors()
        slots = self._ints(slots, torch.int64, "slots")
        n = slots.shape[0]
        code = dtype_code(dtype)
        k = slots.new_empty(n, self.kv_heads, self.head_dim, dtype=dtype)
        v = torch.empty_like(k)
        self._call(self.lib.qq_kv8_gather, self._layers[layer], slots.data_ptr(), n, k.data_ptr(), v.data_ptr(), code,
                   self._err_ptr)
        return k, v

    # ------------------------------------------------------------------ attention

    def _query(self, q: torch.Tensor, out: torch.Tensor | None) -> tuple[torch.Tensor, int, int, torch.Tensor, int]:
        """The queries with dense 16-byte aligned rows, their address and row distance; the result and its row distance."""
        shape = q.shape
        if len(shape) != 3 or shape[2] != self.head_dim or q.get_device() != self._index:
            raise ValueError(f"q must be [tokens, heads, {self.head_dim}] on {self.device}, got {tuple(shape)} "
                             f"on {q.device}")
        n, heads, dim = shape
        if heads == 0 or heads % self.kv_heads:
            raise ValueError(f"q_heads {heads} not divisible by kv_heads {self.kv_heads}")
        token, head, one = q.stride()
        row = heads * dim
        ptr = q.data_ptr()
        if one != 1 or head != dim or token < row or (token * q.element_size() | ptr) & 15:
            q = q.clone(memory_format=torch.contiguous_format)
            ptr, token = q.data_ptr(), row
        if out is None:
            return q, ptr, token, q.new_empty(n, row), row
        if (tuple(out.shape) != (n, row) or out.dtype != q.dtype or out.device != self.device
                or out.stride(1) != 1 or (n > 1 and out.stride(0) < row)):
            raise ValueError(f"out must be {q.dtype} [{n}, {row}] with contiguous rows on {self.device}")
        return q, ptr, token, out, max(out.stride(0), row)

    def _table(self, t: torch.Tensor) -> torch.Tensor:
        shape = t.shape
        if len(shape) != 2 or t.dtype != torch.int32 or t.get_device() != self._index or 0 in shape:
            raise ValueError(f"block_table must be int32 [requests, blocks] on {self.device}")
        # the kernels take the row's stride as its length
        return t if t.stride() == (shape[1], 1) else t.contiguous()

    def _workspace(self, heads: int, code: int, bs: int, tokens: int, max_keys: int, extend: int) -> int:
        key = (heads, code, bs, tokens, max_keys, extend)
        size = self._ws_bytes.get(key)
        if size is None:
            if len(self._ws_bytes) > 4096:  # sizes only: cheap to ask for again
                self._ws_bytes.clear()
            with torch.cuda.device(self._index):  # the size depends on the device
                size = self._ws_bytes[key] = int(self.lib.qq_kv8_workspace_bytes(
                    self._layers[0], heads, code, bs, tokens, max_keys, extend))
        return size

    def decode_attention(self, layer: int, q: torch.Tensor, block_table: torch.Tensor, req_pool_indices, seq_lens,
                         scaling: float, *, out: torch.Tensor | None = None) -> torch.Tensor:
        """Attention of one token per request over its ``seq_lens[i]`` cached tokens.

        ``q``: ``[bs, heads, head_dim]`` bf16 or fp32; ``block_table``: int32 ``[requests, blocks]``.  Returns
        ``[bs, heads * head_dim]`` in ``q``'s dtype; a length of 0 (padding) gives zeros.
        """
        if self._err_word.value:
            self.check_errors()
        q, q_ptr, q_stride, out, out_stride = self._query(q, out)
        bs, heads, _ = q.shape
        if bs == 0:
            return out
        code = dtype_code(q.dtype)
        table = self._table(block_table)
        reqs = self._ints(req_pool_indices, torch.int64, "req_pool_indices", bs)
        seq = self._ints(seq_lens, torch.int64, "seq_lens", bs)
        width = table.shape[1]
        size = self._workspace(heads, code, bs, bs, width * self.block_size, 0)
        self._call_with_scratch(size, self.lib.qq_kv8_decode_attention, self._layers[layer],
                                _lib.QQBatch(reqs.data_ptr(), seq.data_ptr(), bs), table.data_ptr(), width,
                                table.shape[0], q_ptr, code, heads, q_stride, float(scaling), out.data_ptr(),
                                out_stride, self._err_ptr)
        return out

    def sparse_decode_attention(self, layer: int, q: torch.Tensor, rows: torch.Tensor, lens, scaling: float, *,
                                out: torch.Tensor | None = None) -> torch.Tensor:
        """The same over the slots ``rows[i, :lens[i]]`` (int32 ``[bs, top_k]``; duplicates counted, a negative row
        takes no part): the rows :meth:`~qwenquest_b200.quest.QuestAlgorithm.select` writes and its ``actual_lens``."""
        if self._err_word.value:
            self.check_errors()
        q, q_ptr, q_stride, out, out_stride = self._query(q, out)
        bs, heads, _ = q.shape
        if bs == 0:
            return out
        code = dtype_code(q.dtype)
        if rows.dim() != 2 or rows.shape[0] != bs or rows.shape[1] == 0 or rows.get_device() != self._index:
            raise ValueError(f"rows must be int32 [{bs}, top_k] on {self.device}, got {tuple(rows.shape)}")
        if rows.dtype != torch.int32:
            rows = _as_int(rows, torch.int32, "rows", self.device)
        if rows.stride(1) != 1 or rows.stride(0) < rows.shape[1]:
            rows = rows.contiguous()
        lens = self._ints(lens, torch.int32, "lens", bs)
        top = rows.shape[1]
        size = self._workspace(heads, code, bs, bs, top, 0)
        self._call_with_scratch(size, self.lib.qq_kv8_sparse_attention, self._layers[layer], bs, rows.data_ptr(),
                                max(rows.stride(0), top), top, lens.data_ptr(), q_ptr, code, heads, q_stride, float(scaling),
                                out.data_ptr(), out_stride, self._err_ptr)
        return out

    def extend_attention(self, layer: int, q: torch.Tensor, block_table: torch.Tensor, req_pool_indices, seq_lens,
                         prefix_lens, token_offsets, scaling: float, *, out: torch.Tensor | None = None
                         ) -> torch.Tensor:
        """Causal attention of an extend batch: row ``token_offsets[i] + t`` of ``q`` (``[tokens, heads, head_dim]``)
        is position ``prefix_lens[i] + t`` of its request, for ``t < seq_lens[i] - prefix_lens[i]``, and attends
        to positions up to its own, its own token included (append first).

        ``token_offsets`` is what :meth:`BlockTables.plan` returns (``[bs + 1]``, or ``[bs]``).  Rows behind the
        last sequence are left as they were: pass ``out`` where they matter.
        """
        if self._err_word.value:
            self.check_errors()
        q, q_ptr, q_stride, out, out_stride = self._query(q, out)
        tokens, heads, _ = q.shape
        code = dtype_code(q.dtype)
        table = self._table(block_table)
        reqs = self._ints(req_pool_indices, torch.int64, "req_pool_indices")
        bs = reqs.shape[0]
        seq = self._ints(seq_lens, torch.int64, "seq_lens", bs)
        prefix = self._ints(prefix_lens, torch.int64, "prefix_lens", bs)
        offsets = self._ints(token_offsets, torch.int64, "token_offsets")
        if offsets.shape[0] not in (bs, bs + 1):
            raise ValueError(f"token_offsets must be [{bs}] or [{bs + 1}], got {tuple(offsets.shape)}")
        width = table.shape[1]
        size = self._workspace(heads, code, bs, tokens, width * self.block_size, 1)
        batch = _lib.QQExtendBatch(reqs.data_ptr(), seq.data_ptr(), prefix.data_ptr(), offsets.data_ptr(), None,
                                   tokens, bs, 0)
        self._call_with_scratch(size, self.lib.qq_kv8_extend_attention, self._layers[layer], batch, table.data_ptr(),
                                width, table.shape[0], q_ptr, code, heads, q_stride, float(scaling), out.data_ptr(),
                                out_stride, self._err_ptr)
        return out
