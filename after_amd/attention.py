"""Attention over sequences of different lengths: of whole prompts (`attend_packed`), and over a key / value cache that is held
in four bits (`KVCache4`), next to the attention and the streaming K/V caches inside `DenoiserV2`
(after/diffusion/networks/transformerv2.py:62-235).  fp32, bf16 and fp16 tensors; inference only, like the rest of the package
(a tensor that requires a gradient or carries a tangent is refused);
hand-written HIP kernels behind the C ABI of include/after_hip.h, no fallback.

    cache = KVCache4(rows=4, kv_heads=8, head_dim=128, capacity=16384)
    y = attend_packed(q, k, v, starts)                       # the prompts, one behind the other
    cache.append(k, v, starts)
    cache.attend(q_last, accumulate=True)                    # which slots do the last tokens look at?
    small = KVCache4(4, 8, 128, capacity=4096)
    cache.evict(small, keep=2048, recent=64)                 # keep those, and the newest
    while ...:                                               # one token per row and step
        small.append(k1, v1)                                 # [rows, 1, kv_heads, head_dim]
        y = small.attend(q1)                                 # [rows, 1, heads, head_dim]
"""
import ctypes
import functools
import math
import weakref

import torch
from torch.autograd import forward_ad

from . import _lib

_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


def _refuse_gradients(t, name):
    if t.requires_grad and torch.is_grad_enabled():
        raise NotImplementedError(f"{name} requires a gradient: after_amd is inference only (use torch.no_grad())")
    if forward_ad._current_level >= 0 and forward_ad.unpack_dual(t).tangent is not None:
        raise NotImplementedError(f"{name} carries a tangent: after_amd is inference only")


def _operand(t, name, dims, index=None, dtype=None):
    """A tensor the kernels can address: fp32 / bf16 / fp16 on the GPU, channels contiguous, strides and base multiples of 16
    bytes -- a view of a fused projection is taken as it is, anything else is copied."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if not t.is_cuda:
        raise _lib.AFTERHipError(f"{name} is on {t.device}: after_amd runs on MI355X only (HIP kernels)")
    kind, strides = t.dtype, t.stride()
    if kind not in _TYPES:
        raise TypeError(f"{name} must be float32, bfloat16 or float16, got {kind}")
    if len(strides) != dims:
        raise ValueError(f"{name} must have {dims} dimensions, got {tuple(t.shape)}")
    if index is not None and t.get_device() != index:
        raise ValueError(f"{name} is on {t.device}, expected cuda:{index}")
    if dtype is not None and kind is not dtype:
        raise TypeError(f"{name} is {kind}, expected {dtype}")
    if t.requires_grad or forward_ad._current_level >= 0:
        _refuse_gradients(t, name)
    odd = strides[0] | strides[1] | (strides[2] if dims == 4 else 0) | t.data_ptr() // t.element_size()
    # (a token's place in a tile is addressed with 32 bits; what the strides of an empty tensor are does not matter)
    if odd & (3 if kind is torch.float32 else 7) or strides[-1] != 1 or strides[-3] >= 1 << 22:
        t = t.clone(memory_format=torch.contiguous_format)
    return t


def _enqueue(name, index, *args):
    """One call of the C ABI on the current stream of device `index`."""
    fn, stream = getattr(_lib.lib(), name), torch._C._cuda_getCurrentRawStream(index)
    if torch._C._cuda_getDevice() == index:
        rc = fn(*args, stream)
    else:
        with torch.cuda.device(index):
            rc = fn(*args, stream)
    if rc:
        _lib.check(rc, name)


def _starts(t, name, n, index):
    """int32 [n + 1] on device `index` (n None: any)."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if t.dtype is not torch.int32 or t.dim() != 1 or t.get_device() != index:
        raise ValueError(f"{name} must be a one-dimensional int32 tensor on cuda:{index}, got {t.dtype} {tuple(t.shape)} on {t.device}")
    if t.numel() != n + 1 if n is not None else t.numel() < 1:
        raise ValueError(f"{name} has {t.numel()} entries, expected {'one more than sequences' if n is None else n + 1}")
    return t.contiguous()


def _ranges(tensors):
    """[first, last) address of each (contiguous or not; empty ones have none)."""
    return [(t.data_ptr(), t.data_ptr() + t.element_size() * (1 + sum((n - 1) * s for n, s in zip(t.shape, t.stride()))))
            for t in tensors if t.numel()]


def _share(a, b):
    return any(x < v and u < y for x, y in _ranges(a) for u, v in _ranges(b))


def _scale(scale, dim):
    scale = 1.0 / math.sqrt(dim) if scale is None else float(scale)
    if not abs(scale) < 2.35e38:  # (log2 e times as much is the kernels' factor)
        raise ValueError(f"scale must be within 2.35e38, got {scale}")
    return scale


@functools.lru_cache(maxsize=1024)
def _packed_workspace(*sizes):
    """Bytes of scratch that a call of these sizes takes (a function of the sizes alone)."""
    size = ctypes.c_longlong()
    _lib.check(_lib.lib().after_attend_packed_workspace(*sizes, ctypes.byref(size)), "after_attend_packed_workspace")
    return size.value


def attend_packed(q, k, v, q_starts, k_starts=None, *, causal=True, window=None, chunk=1, scale=None, out=None):
    """Attention of packed sequences (include/after_hip.h: after_attend_packed).

    q [tokens, heads, D], k / v [keys, kv_heads, D], D = 64 or 128, heads a multiple of kv_heads; sequence b's queries are the
    rows q_starts[b] .. q_starts[b + 1] - 1 and its keys the rows k_starts[b] ... (int32 device tensors from 0, ascending;
    k_starts defaults to q_starts).  A sequence's queries are the newest of its keys: with more keys than queries it continues
    what is cached, with one query it is a decoding step.

    causal: a query sees the keys up to its own position; with `chunk` > 1 also the rest of its chunk, and with `window` only the
    newest `window` keys outside its chunk: the mask of DenoiserV2's local attention (transformerv2.py:62-96).  A query that
    sees nothing gets zeros.  Sums and softmax are fp32; bf16 and fp16 products take probabilities rounded to that type.

    Rows behind the last sequence are zeros in a new tensor and left alone in `out`, which must be contiguous and must not
    overlap q, k or v; it may be q itself."""
    chunk, window = int(chunk), None if window is None else int(window)
    if not 1 <= chunk <= 1 << 24 or (window is not None and window < 1):
        raise ValueError(f"chunk must be 1 .. 2^24 and window at least 1, got {chunk} and {window}")
    if not causal and (chunk != 1 or window is not None):
        raise ValueError("chunk and window belong to causal attention")
    q = _operand(q, "q", 3)
    index, dtype = q.get_device(), q.dtype
    k = _operand(k, "k", 3, index, dtype)
    v = _operand(v, "v", 3, index, dtype)
    n, heads, dim = q.shape
    keys, kv_heads, k_dim = k.shape
    if k.shape != v.shape or k_dim != dim or kv_heads == 0 or heads == 0 or heads % kv_heads:
        raise ValueError(f"bad shapes q{tuple(q.shape)} k{tuple(k.shape)} v{tuple(v.shape)}: k and v alike, heads a multiple of kv_heads, one head_dim")
    if dim not in (64, 128):
        raise ValueError(f"head_dim must be 64 or 128, got {dim}")
    q_starts = _starts(q_starts, "q_starts", None, index)
    seqs = q_starts.numel() - 1
    if seqs >= 1 << 24:
        raise ValueError(f"at most 2^24 - 1 sequences, got {seqs}")
    k_starts = q_starts if k_starts is None else _starts(k_starts, "k_starts", seqs, index)
    scale = _scale(scale, dim)
    fresh = out is None
    if fresh:
        out = q.new_empty((n, heads, dim))
    elif not isinstance(out, torch.Tensor) or out.shape != q.shape or out.dtype != dtype or out.device != q.device \
            or not out.is_contiguous() or out.data_ptr() % 16:
        raise ValueError(f"out must be a contiguous, 16-byte aligned {dtype} tensor {tuple(q.shape)} on {q.device}")
    else:
        _refuse_gradients(out, "out")
        if _share([out], [k, v] if out.data_ptr() == q.data_ptr() and q.is_contiguous() else [q, k, v]):
            raise ValueError("out shares memory with q, k or v (it may be q itself, if that is contiguous)")
    window, kind = min(window or 0, 1 << 30), _TYPES[dtype]
    size = _packed_workspace(kind, n, keys, seqs, heads, kv_heads, dim, window)
    work = torch.empty(size, dtype=torch.uint8, device=q.device) if size else None  # (as in KVCache4.attend)
    q_at, k_at, v_at = q.stride(), k.stride(), v.stride()
    _enqueue("after_attend_packed", index, _lib.Packed.FORMAT.pack(
        q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), q_starts.data_ptr(), k_starts.data_ptr(), work.data_ptr() if size else 0, size,
        n, keys, q_at[0], q_at[1], k_at[0], k_at[1], v_at[0], v_at[1], heads * dim, dim, kind, seqs, heads, kv_heads, dim, scale,
        1 if causal else 0, window, chunk, 1 if fresh else 0))
    return out


class KVCache4:
    """Keys and values of `rows` sequences, `kv_heads` heads each, in four bits: 17 bytes per 32 channels, with the attention
    that reads them and the eviction of slots by the attention they received (include/after_hip.h: after_kv4, which states the
    format).  `capacity` slots per row (rounded up to a multiple of 32).

    The state is six tensors of the object -- `keys`, `key_scales`, `values`, `value_scales` (uint8), `weights` (fp32
    [rows, kv_heads, capacity]: attention received, summed up by `attend(accumulate=True)`), `lengths` (int32 [rows]: slots in
    use) -- which `buffers()` returns and `KVCache4(..., buffers=...)` takes over as they are.  They can be written in place, not
    replaced.

    Every call but `check` enqueues on the current stream, never synchronises and can be captured into a graph; the lengths live
    on the device.  One call at a time works on a cache: order calls on different streams with events, as for any tensor."""

    def __init__(self, rows, kv_heads, head_dim, capacity, device="cuda", buffers=None):
        rows, kv_heads, head_dim, capacity = int(rows), int(kv_heads), int(head_dim), int(capacity)
        if rows < 1 or kv_heads < 1 or rows * kv_heads > 1 << 20:
            raise ValueError(f"rows and kv_heads must be at least 1, and rows x kv_heads at most 2^20, got {rows} and {kv_heads}")
        if head_dim not in (64, 128):
            raise ValueError(f"head_dim must be 64 or 128, got {head_dim}")
        if not 1 <= capacity <= 1 << 24:
            raise ValueError(f"capacity must be 1 .. 2^24, got {capacity}")
        self.rows, self.kv_heads, self.head_dim = rows, kv_heads, head_dim
        self.capacity = C = (capacity + 31) // 32 * 32
        device = torch.device(device)
        if device.type != "cuda":
            raise _lib.AFTERHipError(f"KVCache4 on {device}: after_amd runs on MI355X only (HIP kernels)")
        self.device = torch.device("cuda", torch.cuda.current_device() if device.index is None else device.index)
        self._index = self.device.index
        layout = dict(keys=((rows, kv_heads, C, head_dim // 2), torch.uint8), key_scales=((rows, kv_heads, C, head_dim // 32), torch.uint8),
                      values=((rows, kv_heads, C // 8, head_dim, 4), torch.uint8), value_scales=((rows, kv_heads, C, head_dim // 32), torch.uint8),
                      weights=((rows, kv_heads, C), torch.float32), lengths=((rows, ), torch.int32))
        if buffers is not None and set(buffers) != set(layout):
            raise ValueError(f"buffers must hold {sorted(layout)}, got {sorted(buffers)}")
        tensors = {}
        for name, (shape, dtype) in layout.items():
            if buffers is None:
                t = torch.zeros(shape, dtype=dtype, device=self.device)
            else:
                t = buffers[name]
                if not isinstance(t, torch.Tensor) or tuple(t.shape) != shape or t.dtype != dtype or t.device != self.device \
                        or not t.is_contiguous() or t.data_ptr() % 16:
                    raise ValueError(f"buffers[{name!r}] must be a contiguous, 16-byte aligned {dtype} tensor {shape} on {self.device}")
            tensors[name] = t
        if buffers is not None and any(_share([t], [u]) for i, t in enumerate(tensors.values()) for u in list(tensors.values())[:i]):
            raise ValueError("two of the buffers share memory")
        self._failed = torch.zeros(1, dtype=torch.int32, device=self.device)
        self._tensors = tensors  # (their addresses are in _c: the attributes cannot be set to others)
        self._evicted_into = None
        self._c = _lib.KV4(*(t.data_ptr() for t in tensors.values()), self._failed.data_ptr(), rows, kv_heads, head_dim, C)
        self._ref = ctypes.byref(self._c)
        self._work = {}  # (type, heads, tokens, accumulate) -> bytes of an attend call's scratch

    keys = property(lambda self: self._tensors["keys"])
    key_scales = property(lambda self: self._tensors["key_scales"])
    values = property(lambda self: self._tensors["values"])
    value_scales = property(lambda self: self._tensors["value_scales"])
    weights = property(lambda self: self._tensors["weights"])
    lengths = property(lambda self: self._tensors["lengths"])

    def buffers(self):
        """The six tensors of the state, by name."""
        return dict(self._tensors)

    def _row_values(self, t, name):
        if not isinstance(t, torch.Tensor) or t.dtype is not torch.int32 or t.dim() != 1 or t.numel() != self.rows or t.get_device() != self._index:
            raise ValueError(f"{name} must be an int32 tensor ({self.rows},) on {self.device}")
        return t.contiguous()

    def append(self, k, v, starts=None):
        """Rounds new keys and values to four bits and puts them behind each row's slots: [rows, tokens, kv_heads, head_dim], or
        [total, kv_heads, head_dim] with `starts` (int32 [rows + 1]): those of row r are starts[r] .. starts[r + 1] - 1.  Tokens
        for which a row has no room are dropped; `check()` reports that."""
        dims = 4 if starts is None else 3
        k = _operand(k, "k", dims, self._index)
        v = _operand(v, "v", dims, self._index, k.dtype)
        *outer, heads, dim = k.shape
        if k.shape != v.shape or heads != self.kv_heads or dim != self.head_dim or (starts is None and outer[0] != self.rows):
            raise ValueError(f"bad shapes k{tuple(k.shape)} v{tuple(v.shape)} for {self.rows} rows of {self.kv_heads} heads of {self.head_dim}")
        k_at, v_at = k.stride(), v.stride()
        tokens, total = 0, outer[0]
        if starts is None:
            tokens = outer[1]
            if tokens > self.capacity:
                raise ValueError(f"{tokens} new tokens, the cache has {self.capacity} slots per row")
            total *= tokens
            # (one token of each row, as a rule: its rows are the tokens)
            if tokens == 1:
                k_at, v_at = (k_at[0], k_at[2]), (v_at[0], v_at[2])
            else:
                k, v = k.flatten(0, 1), v.flatten(0, 1)
                k_at, v_at = k.stride(), v.stride()
        else:
            starts = _starts(starts, "starts", self.rows, self._index)
        _enqueue("after_kv4_append", self._index, self._ref, k.data_ptr(), v.data_ptr(), _TYPES[k.dtype], None if starts is None else starts.data_ptr(),
                 tokens, total, k_at[0], k_at[1], v_at[0], v_at[1])

    def truncate(self, lengths=None):
        """Takes back the newest slots: row r keeps the first lengths[r] (int32 [rows] on the device); None empties the cache."""
        lengths = None if lengths is None else self._row_values(lengths, "lengths")
        _enqueue("after_kv4_truncate", self._index, self._ref, None if lengths is None else lengths.data_ptr())

    def read(self, start=None, count=None, dtype=torch.bfloat16):
        """(k, v) [rows, kv_heads, count, head_dim]: the values that the slots start[r] .. start[r] + count - 1 stand for (int32
        [rows]; default: from slot 0, the whole capacity), zeros past a row's length.  bf16 holds them exactly."""
        count = self.capacity if count is None else int(count)
        if not 0 <= count <= self.capacity:
            raise ValueError(f"count must be 0 .. {self.capacity}, got {count}")
        if dtype not in (torch.bfloat16, torch.float32):
            raise TypeError(f"values are read as bfloat16 or float32, got {dtype}")
        start = None if start is None else self._row_values(start, "start")
        k, v = (torch.empty(self.rows, self.kv_heads, count, self.head_dim, dtype=dtype, device=self.device) for _ in range(2))
        _enqueue("after_kv4_read", self._index, self._ref, k.data_ptr(), v.data_ptr(), _TYPES[dtype], None if start is None else start.data_ptr(), count)
        return k, v

    def attend(self, q, scale=None, accumulate=False, decay=1.0):
        """Attention of the newest tokens of every row, q [rows, tokens, heads, head_dim], over the cached keys and values (their
        own have been appended): token t of T sees the slots below lengths - T + t + 1; one that sees none gets zeros.  A row
        with fewer new tokens than T has its own at the end.  Returns [rows, tokens, heads, head_dim].  Sums and softmax are fp32;
        a probability is multiplied in as many bf16 pieces as hold a number of q's type: for bf16 queries it is rounded to bf16.

        accumulate: `weights` = decay * weights + the probability that each slot received, summed over the tokens and the heads
        of its group (decay = 0 replaces them).  Up to 32 queries of a row and key head keep their scores for that, in scratch of
        4 bytes x queries x rows x kv_heads x capacity."""
        q = _operand(q, "q", 4, self._index)
        rows, tokens, heads, dim = q.shape
        if rows != self.rows or dim != self.head_dim or heads == 0 or heads % self.kv_heads:
            raise ValueError(f"bad shape q{tuple(q.shape)} for {self.rows} rows of {self.kv_heads} key heads of {self.head_dim}")
        scale, decay = _scale(scale, dim), float(decay)
        if not abs(decay) < 3e38:
            raise ValueError(f"decay must be finite in 32 bits, got {decay}")
        out = torch.empty(rows, tokens, heads, dim, dtype=q.dtype, device=self.device)
        if tokens == 0:
            if accumulate and decay != 1.0:
                raise ValueError("accumulate with a decay needs at least one token")
            return out
        accumulate = int(bool(accumulate))
        key = (q.dtype, heads, tokens, accumulate)
        if key not in self._work:
            size = ctypes.c_longlong()
            _lib.check(_lib.lib().after_kv4_attend_workspace(self._ref, _TYPES[q.dtype], *key[1:], ctypes.byref(size)), "after_kv4_attend_workspace")
            self._work[key] = size.value
        # (scratch of this call: the allocator gives it to later calls of this stream only, and to a captured graph its own)
        size = self._work[key]
        work = torch.empty(size, dtype=torch.uint8, device=self.device) if size else None
        _enqueue("after_kv4_attend", self._index, self._ref, _lib.KV4Query.FORMAT.pack(
            q.data_ptr(), out.data_ptr(), work.data_ptr() if size else 0, size, *q.stride()[:3], _TYPES[q.dtype], heads, tokens, scale, accumulate, decay))
        return out

    def evict(self, into, keep, recent=0):
        """Moves min(length, keep) slots per row and head into another cache of the same rows, heads and head_dim, in their order,
        replacing its content: the `recent` newest, and of the others those that received most attention (`weights`; ties go to
        the lower slot, NaN counts as the least).  Heads choose for themselves.  This cache stays as it is.  Returns int32
        [rows, kv_heads, keep]: the slot each came from, -1 past a row's new length."""
        keep, recent = int(keep), int(recent)
        if not isinstance(into, KVCache4) or into is self:
            raise ValueError("evict moves into another KVCache4")
        if self._evicted_into is None or self._evicted_into() is not into:
            if (into.rows, into.kv_heads, into.head_dim, into.device) != (self.rows, self.kv_heads, self.head_dim, self.device):
                raise ValueError("both caches need the same rows, kv_heads, head_dim and device")
            if _share(self._tensors.values(), into._tensors.values()):
                raise ValueError("the two caches share memory")
            self._evicted_into = weakref.ref(into)  # (looked at once)
        if not 1 <= keep <= into.capacity or not 0 <= recent <= keep:
            raise ValueError(f"1 <= keep <= {into.capacity} and 0 <= recent <= keep, got {keep} and {recent}")
        slots = torch.empty(self.rows, self.kv_heads, keep, dtype=torch.int32, device=self.device)
        _enqueue("after_kv4_evict", self._index, self._ref, into._ref, keep, recent, slots.data_ptr())
        return slots

    def check(self):
        """Waits for the current stream and raises AFTERHipError if an append has dropped tokens since the last look."""
        if int(self._failed.item()):
            self._failed.zero_()
            raise _lib.AFTERHipError(f"KVCache4.append: a row had no room for all of its new tokens ({self.capacity} slots)")
