"""The paged key/value cache of a decoder and the operators around it, over libbybycuda.so: what a
decode or prompt step does between the quantised projections.

``rope_append``      rotary positions, and the new keys and values into their pages
``paged_attention``  attention of a chunk of new tokens (or one) over the cache
``copy_pages``       page copies of all layers in one launch (forks, compaction)
``beam_select``      beam search's best continuations of the LM head's logits
``PagedKvCache``     the tensors of all layers
``PagePool``         who holds which page: allocate, fork, copy-on-write, free, compact
``rope_frequencies`` turns per position of each dimension pair, stretched for long contexts

Tensors are torch device tensors, every call is asynchronous on `stream` (default: the current
one) and there is no CPU fallback: a call that cannot run raises ``BybyCudaError``.  Page ids and
lengths live on the device; the kernels check them and report through ``_lib.device_error()``.

With `stream` given the caller orders it after the stream that made the inputs, and keeps the inputs
until the work is done.  An output that the call allocates belongs to `stream`; one that is used on
another stream afterwards needs that stream to wait, and ``record_stream`` before it is dropped.

A batch is three int32 device tensors: ``page_table`` [sequences, pages], ``q_start``
[sequences + 1] (sequence b's new tokens are rows q_start[b] .. q_start[b+1]) and ``kv_lens``
[sequences] (tokens in the cache, the new ones included).
"""
from __future__ import annotations

import array
import ctypes as C
import heapq
import itertools
import math
import struct

from . import _lib
from ._lib import BybyCudaError, check, load
from .gpubackend import _dtype_code, _output

# A decode step makes several of these calls a layer, so what a call costs the host counts: the
# argument structs of include/bybycuda.h are packed in one go (bybycu_paged_kv, bybycu_rope,
# bybycu_attention, field by field), and passed as bytes.
_KV = struct.Struct("=QQqqqQqQQ8i").pack
_ROPE = struct.Struct("=QQQQ8qQQ4ifi").pack
_ATTENTION = struct.Struct("=QQ4qQQ6i2f").pack
_calls: dict = {}


def _call(name: str):
    fn = _calls.get(name)
    if fn is None:
        fn = load()[name]     # a handle of its own: raw pointers and bytes for the structs
        fn.argtypes = [C.c_void_p if a not in (C.c_int, C.c_int64) else a for a in _lib.SIGNATURES[name]]
        fn.restype = C.c_int
        _calls[name] = fn
    return fn


def _refuse(code: int, message: str):
    raise BybyCudaError(code, message)


def _pack(op: str, pack, *fields) -> bytes:
    try:
        return pack(*fields)
    except (struct.error, OverflowError) as e:
        _refuse(_lib.ERR_ARGS, f"{op}: an argument does not fit its field ({e})")


def _stream(op: str, device: int, stream) -> int:
    """The raw stream of a call on `device`, which has to be the current one and the stream's (the
    default stream has one handle on every device)."""
    import torch
    if torch._C._cuda_getDevice() != device:
        _refuse(_lib.ERR_ARGS, f"{op}: the tensors are on cuda:{device}, the current device is cuda:{torch.cuda.current_device()}")
    if stream is None:
        return torch._C._cuda_getCurrentRawStream(device)
    if stream.device_index != device:
        _refuse(_lib.ERR_ARGS, f"{op}: the stream is on cuda:{stream.device_index}, the tensors are on cuda:{device}")
    return stream.cuda_stream


def _paged(op: str, n_tokens: int, k_cache, v_cache, page_table, q_start, kv_lens):
    """The packed bybycu_paged_kv and (device, sequences, kv heads, head dim) of a call's cache and batch."""
    import torch
    if k_cache.dim() != 4 or k_cache.dtype != torch.bfloat16 or v_cache.dtype != torch.bfloat16:
        _refuse(_lib.ERR_ARGS, f"{op}: caches must be bfloat16 [pages, kv heads, page size, head dim]")
    shape, strides = k_cache.shape, k_cache.stride()
    n_pages, heads, page, dim = shape
    if v_cache.shape != shape or v_cache.stride() != strides or strides[3] != 1:
        _refuse(_lib.ERR_ARGS, f"{op}: the caches must share shape and strides, the last dimension dense")
    if page_table.dim() != 2 or page_table.dtype != torch.int32 or q_start.dtype != torch.int32 or kv_lens.dtype != torch.int32:
        _refuse(_lib.ERR_ARGS, f"{op}: page_table [sequences, pages], q_start and kv_lens must be int32")
    n_seqs, max_pages = page_table.shape
    if q_start.numel() != n_seqs + 1 or kv_lens.numel() != n_seqs:
        _refuse(_lib.ERR_SHAPE, f"{op}: {n_seqs} sequences need {n_seqs + 1} starts and {n_seqs} lengths")
    table_stride, one = page_table.stride()
    if not q_start.is_contiguous() or not kv_lens.is_contiguous() or (max_pages > 1 and one != 1):
        _refuse(_lib.ERR_ARGS, f"{op}: page_table rows, q_start and kv_lens must be contiguous")
    dev = k_cache.get_device()
    if dev < 0 or v_cache.get_device() != dev or page_table.get_device() != dev or q_start.get_device() != dev or \
            kv_lens.get_device() != dev:
        _refuse(_lib.ERR_ARGS, f"{op}: every tensor must be on the device")
    if n_seqs <= 1:
        table_stride = max_pages
    return _KV(k_cache.data_ptr(), v_cache.data_ptr(), strides[0], strides[1], strides[2], page_table.data_ptr(), table_stride,
               q_start.data_ptr(), kv_lens.data_ptr(), n_pages, page, heads, dim, max_pages, n_seqs, n_tokens, 0), dev, n_seqs, heads, dim


def _heads(op: str, name: str, t, tokens: int, heads: int, dim: int, dev: int, dtype):
    """Checks a [tokens, heads, dim] tensor and returns its (token, head) strides."""
    if t.shape != (tokens, heads, dim):
        _refuse(_lib.ERR_SHAPE, f"{op}: {name} is {tuple(t.shape)}, not [{tokens}, {heads}, {dim}]")
    if t.get_device() != dev or (dtype is not None and t.dtype != dtype):
        _refuse(_lib.ERR_ARGS, f"{op}: {name} must be a tensor on the caches' device" + (f" of {dtype}" if dtype is not None else ""))
    a, b, c = t.stride()
    if c != 1:
        _refuse(_lib.ERR_ARGS, f"{op}: the last dimension of {name} must be dense")
    return a, b


def _vector(op: str, name: str, t, n: int, dtype, dev: int) -> int:
    """The address of an optional vector, 0 for None."""
    if t is None:
        return 0
    if t.dtype != dtype or t.numel() != n or not t.is_contiguous() or t.get_device() != dev:
        _refuse(_lib.ERR_ARGS, f"{op}: {name} must be {n} contiguous {dtype} on the caches' device")
    return t.data_ptr()


def rope_frequencies(rotary_dim: int, base: float = 10000.0, *, scaling: str = "none", factor: float = 1.0,
                     original_context: int = 0, low: float = 1.0, high: float = 32.0, device=None):
    """Turns per position (frequency / 2 pi) of the rotary_dim / 2 dimension pairs, fp64 on the device.

    scaling stretches them for contexts `factor` times `original_context`:
    "none"     base ** (-2 i / rotary_dim);
    "linear"   every frequency divided by factor (positions interpolated);
    "base"     the base raised so that the slowest pair is divided by factor and the fastest kept;
    "by-parts" pairs that turn more than `high` times over original_context keep their frequency,
               those that turn less than `low` times are divided by factor, linearly in between.
    """
    import torch
    if rotary_dim < 0 or rotary_dim % 2 or not base > 0 or not factor > 0:
        _refuse(_lib.ERR_ARGS, f"rope_frequencies: rotary_dim={rotary_dim} base={base} factor={factor}")
    pairs = rotary_dim // 2
    if scaling == "base" and rotary_dim > 2:
        base = base * factor ** (rotary_dim / (rotary_dim - 2))
    f = [base ** (-2.0 * i / rotary_dim) / (2.0 * math.pi) for i in range(pairs)]
    if scaling == "linear":
        f = [x / factor for x in f]
    elif scaling == "by-parts":
        if original_context <= 0 or not high > low:
            _refuse(_lib.ERR_ARGS, f"rope_frequencies: original_context={original_context} low={low} high={high}")
        kept = [min(1.0, max(0.0, (x * original_context - low) / (high - low))) for x in f]
        f = [x * (k + (1.0 - k) / factor) for x, k in zip(f, kept)]
    elif scaling not in ("none", "base"):
        _refuse(_lib.ERR_ARGS, f"rope_frequencies: unknown scaling {scaling!r} (none, linear, base, by-parts)")
    dev = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
    return torch.tensor(f, dtype=torch.float64, device=dev)


_LAYOUTS = {"half": 0, "interleaved": 1}


def rope_append(q, k, v, k_cache, v_cache, page_table, q_start, kv_lens, turns, *, layout: str = "half",
                magnitude: float = 1.0, positions=None, q_out=None, stream=None):
    """Turns q and k [tokens, heads, dim] by their positions, writes k and v to their slots of the
    cache (bf16) and returns the turned queries (bf16).  q, k and v may be views of one fused
    projection, float32 or bfloat16.  turns: fp64 [pairs], the turns per position of each pair
    (``rope_frequencies``); 2 * pairs dimensions turn, the rest pass.  layout "half" pairs (i, i +
    pairs), "interleaved" (2i, 2i + 1).  positions (int32 [tokens]) turns by other positions than
    those in the cache.  A token at a negative position is padding: its queries come back zero.  Rows that belong to
    no sequence (before q_start[0], from q_start[-1] on) are not written: whatever the output held."""
    import torch
    if q.dim() != 3:
        _refuse(_lib.ERR_SHAPE, f"rope_append: q is {tuple(q.shape)}, not [tokens, heads, dim]")
    T, hq, _ = q.shape
    kv, dev, _, hk, dim = _paged("rope_append", T, k_cache, v_cache, page_table, q_start, kv_lens)
    if layout not in _LAYOUTS:
        _refuse(_lib.ERR_ARGS, f"rope_append: unknown layout {layout!r} (half, interleaved)")
    dtype = q.dtype
    qs = _heads("rope_append", "q", q, T, hq, dim, dev, None)
    ks = _heads("rope_append", "k", k, T, hk, dim, dev, dtype)
    vs = _heads("rope_append", "v", v, T, hk, dim, dev, dtype)
    raw = _stream("rope_append", dev, stream)
    if q_out is None:
        q_out = _output((T, hq, dim), torch.bfloat16, q.device, stream)
        os_ = hq * dim, dim
    else:
        os_ = _heads("rope_append", "q_out", q_out, T, hq, dim, dev, torch.bfloat16)
    pairs = turns.numel()
    args = _pack("rope_append", _ROPE, q.data_ptr(), k.data_ptr(), v.data_ptr(), q_out.data_ptr(), *qs, *ks, *vs, *os_,
                 _vector("rope_append", "turns", turns, pairs, torch.float64, dev),
                 _vector("rope_append", "positions", positions, T, torch.int32, dev), _dtype_code(q), hq, pairs,
                 _LAYOUTS[layout], magnitude, 0)
    check(_call("bybycu_rope_append")(kv, args, raw))
    return q_out


def paged_attention(q, k_cache, v_cache, page_table, q_start, kv_lens, *, max_q: int, max_kv: int, scale: float | None = None,
                    softcap: float = 0.0, slopes=None, window: int = 0, prefix_lens=None, out=None, out_dtype=None,
                    route: int = _lib.ROUTE_AUTO, stream=None):
    """Attention of q (bf16 [tokens, heads, dim]) over the cache, causal by position.

    max_q, max_kv: the most new tokens and cached tokens of any sequence (host numbers that size
    the launch).  scale: default dim ** -0.5.  softcap > 0 caps the scores at softcap *
    tanh(score / softcap); slopes (float32 [heads]) subtracts slope * distance; window > 0 hides
    keys `window` or more positions back; prefix_lens (int32 [sequences]) lets every row see the
    first prefix_lens[b] keys.  The output is q's shape in out_dtype (bfloat16 by default, or
    float32), its vectors apart from one another; rows that see nothing are zero, rows that belong to
    no sequence (before q_start[0], from q_start[-1] on) are not written: whatever the output held."""
    import torch
    if q.dim() != 3:
        _refuse(_lib.ERR_SHAPE, f"paged_attention: q is {tuple(q.shape)}, not [tokens, heads, dim]")
    T, hq, _ = q.shape
    kv, dev, n_seqs, _, dim = _paged("paged_attention", T, k_cache, v_cache, page_table, q_start, kv_lens)
    qs = _heads("paged_attention", "q", q, T, hq, dim, dev, torch.bfloat16)
    raw = _stream("paged_attention", dev, stream)
    if out is None:
        out = _output((T, hq, dim), torch.bfloat16 if out_dtype is None else out_dtype, q.device, stream)
        os_ = hq * dim, dim
    else:
        os_ = _heads("paged_attention", "out", out, T, hq, dim, dev, out_dtype)
    args = _pack("paged_attention", _ATTENTION, q.data_ptr(), out.data_ptr(), *qs, *os_, _vector("paged_attention", "slopes", slopes, hq, torch.float32, dev),
                      _vector("paged_attention", "prefix_lens", prefix_lens, n_seqs, torch.int32, dev), _dtype_code(out), hq,
                      max_q, max_kv, window, route, dim ** -0.5 if scale is None else scale, softcap)
    check(_call("bybycu_paged_attention")(kv, args, raw))
    return out


def _pairs(pairs):
    """The pairs of a copy as contiguous int32 [n, 2] on the host."""
    import torch
    if isinstance(pairs, torch.Tensor) and pairs.dtype == torch.int32 and pairs.is_cpu and pairs.dim() == 2 and pairs.shape[1] == 2:
        return pairs.contiguous()
    if isinstance(pairs, (list, tuple)):
        try:
            if not all(len(p) == 2 for p in pairs):
                _refuse(_lib.ERR_SHAPE, f"copy_pages: pairs are {pairs!r:.60}, not [n, 2]")
            flat = array.array("i", itertools.chain.from_iterable(pairs))
        except (TypeError, OverflowError):
            _refuse(_lib.ERR_ARGS, "copy_pages: pairs must be whole numbers that fit 32 bits, two each")
        return torch.frombuffer(flat, dtype=torch.int32).view(-1, 2) if flat else torch.empty(0, 2, dtype=torch.int32)
    p = torch.as_tensor(pairs, device="cpu")
    if (p.dim() != 2 or p.shape[1] != 2) and (p.numel() or p.dim() == 0):
        _refuse(_lib.ERR_SHAPE, f"copy_pages: pairs are {tuple(p.shape)}, not [n, 2]")
    if p.dtype != torch.int32 and p.numel():
        wide = p.to(torch.int64)
        if p.dtype.is_floating_point or p.dtype.is_complex or p.dtype == torch.bool or wide.min() < -(1 << 31) or wide.max() >= 1 << 31:
            _refuse(_lib.ERR_ARGS, "copy_pages: pairs must be whole numbers that fit 32 bits, two each")
        p = wide
    return p.to(torch.int32).contiguous()


def copy_pages(k_cache, v_cache, pairs, *, stream=None) -> None:
    """Page dst becomes page src for each (src, dst) of `pairs` (host: int32 [n, 2] tensor or
    array, or a list), in every layer of caches [layers, pages, ...] (bf16 or any other type; 4-D
    [pages, ...] for one layer), in one launch.  The pairs act at once: no destination may be in
    another pair."""
    import torch
    if v_cache is not None and (v_cache.shape != k_cache.shape or v_cache.stride() != k_cache.stride() or v_cache.dtype != k_cache.dtype):
        _refuse(_lib.ERR_ARGS, "copy_pages: the caches must share shape, strides and type")
    shape, strides = k_cache.shape, k_cache.stride()
    if len(shape) not in (4, 5):
        _refuse(_lib.ERR_SHAPE, f"copy_pages: caches are {tuple(shape)}, not [layers, pages, heads, page size, dim]")
    dev = k_cache.get_device()
    if dev < 0 or (v_cache is not None and v_cache.get_device() != dev):
        _refuse(_lib.ERR_ARGS, "copy_pages: the caches must be on the device")
    layers, layer_stride = (shape[0], strides[0]) if len(shape) == 5 else (1, 0)
    n_pages, page_stride = shape[-4], strides[-4]
    dense = shape[-3] * shape[-2] * shape[-1]
    if not k_cache.is_contiguous():
        run = 1
        for st, n in sorted((st, n) for st, n in zip(strides[-3:], shape[-3:]) if n > 1):
            if st != run:
                _refuse(_lib.ERR_ARGS, "copy_pages: a page must be one dense block")
            run *= n
    if n_pages == 1:
        page_stride = dense
    p = _pairs(pairs)
    n = p.shape[0] if p.numel() else 0
    esz = k_cache.element_size()
    check(_call("bybycu_copy_pages")(k_cache.data_ptr(), 0 if v_cache is None else v_cache.data_ptr(), layers, layer_stride * esz,
                                     page_stride * esz, dense * esz, n_pages, p.data_ptr(), n, _stream("copy_pages", dev, stream)))


def beam_select(logits, scores, keep: int, *, stream=None):
    """The `keep` best continuations of each group: logits [groups * beams, vocab] float32 or
    bfloat16, scores float32 [groups, beams] the beams' log-probabilities so far.  Returns (scores
    float32, beams int32, tokens int32), each [groups, keep], best first; equal scores by the lower
    beam, within a beam by the larger logit, then the lower token."""
    import torch
    if logits.dim() != 2 or scores.dim() != 2 or logits.shape[0] != scores.numel():
        _refuse(_lib.ERR_SHAPE, f"beam_select: logits {tuple(logits.shape)} for scores {tuple(scores.shape)}")
    rows, vocab = logits.shape
    stride, one = logits.stride()
    dev = logits.get_device()
    if scores.dtype != torch.float32 or not scores.is_contiguous() or dev < 0 or scores.get_device() != dev or (vocab > 1 and one != 1):
        _refuse(_lib.ERR_ARGS, "beam_select: scores must be contiguous float32, the rows of logits dense, both on the device")
    groups, beams = scores.shape
    if not 1 <= keep <= 64 or keep > beams * vocab:
        _refuse(_lib.ERR_SHAPE, f"beam_select: groups={groups} beams={beams} vocab={vocab} keep={keep}")
    raw = _stream("beam_select", dev, stream)
    best = _output((groups, keep), torch.float32, logits.device, stream)
    which = _output((2, groups, keep), torch.int32, logits.device, stream)
    at = which.data_ptr()
    check(_call("bybycu_beam_select")(logits.data_ptr(), _dtype_code(logits), stride if rows > 1 else max(1, vocab), scores.data_ptr(),
                                      groups, beams, vocab, keep, best.data_ptr(), at, at + 4 * groups * keep, raw))
    beam, token = which.unbind(0)
    return best, beam, token


class PagedKvCache:
    """The K and V tensors of all layers, bf16 [layers, pages, kv heads, page size, head dim]."""

    def __init__(self, n_layers: int, n_pages: int, kv_heads: int, head_dim: int, page_size: int = 64, device=None):
        import torch
        dev = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
        self.page_size = page_size
        shape = (n_layers, n_pages, kv_heads, page_size, head_dim)
        self.k = torch.zeros(shape, dtype=torch.bfloat16, device=dev)
        self.v = torch.zeros(shape, dtype=torch.bfloat16, device=dev)

    def layer(self, i: int):
        return self.k[i], self.v[i]

    def copy(self, pairs, stream=None) -> None:
        copy_pages(self.k, self.v, pairs, stream=stream)


class PagePool:
    """Which sequence holds which page (host bookkeeping).

    A page is shared by reference count: ``fork`` gives a new sequence the same pages, and
    ``extend`` gives a sequence that is about to write into a shared page one of its own first.
    Methods that need pages moved on the device return the (src, dst) pairs for ``copy_pages``;
    copy them before the next launch that writes to the cache."""

    def __init__(self, n_pages: int, page_size: int):
        if n_pages <= 0 or page_size <= 0:
            _refuse(_lib.ERR_ARGS, f"PagePool: {n_pages} pages of {page_size}")
        self.n_pages, self.page_size = n_pages, page_size
        self._free = list(range(n_pages))       # a heap: the lowest free page first
        self._refs = [0] * n_pages
        self._seqs: dict[int, tuple[list[int], int]] = {}
        self._next = 0

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def _seq(self, seq: int):
        if seq not in self._seqs:
            _refuse(_lib.ERR_ARGS, f"PagePool: unknown sequence {seq}")
        return self._seqs[seq]

    def length(self, seq: int) -> int:
        return self._seq(seq)[1]

    def pages(self, seq: int) -> list[int]:
        return list(self._seq(seq)[0])

    def new(self) -> int:
        self._next += 1
        self._seqs[self._next] = ([], 0)
        return self._next

    def _take(self) -> int:
        page = heapq.heappop(self._free)
        self._refs[page] = 1
        return page

    def _drop(self, page: int) -> None:
        self._refs[page] -= 1
        if self._refs[page] == 0:
            heapq.heappush(self._free, page)

    def extend(self, seq: int, tokens: int) -> list[tuple[int, int]]:
        """Makes room for `tokens` more; the copies that unshare the page written to first."""
        pages, n = self._seq(seq)
        if tokens < 0:
            _refuse(_lib.ERR_ARGS, f"PagePool: {tokens} tokens")
        if not tokens:
            return []
        shared = n % self.page_size != 0 and self._refs[pages[n // self.page_size]] > 1
        need = -(-(n + tokens) // self.page_size) - len(pages)
        if need + shared > len(self._free):
            _refuse(_lib.ERR_RANGE, f"PagePool: {need + shared} pages wanted, {len(self._free)} free")
        pairs = []
        if shared:
            old = pages[n // self.page_size]
            pages[n // self.page_size] = page = self._take()
            self._drop(old)
            pairs.append((old, page))
        pages.extend(self._take() for _ in range(need))
        self._seqs[seq] = (pages, n + tokens)
        return pairs

    def fork(self, seq: int) -> int:
        """A new sequence with the same tokens, all pages shared."""
        pages, n = self._seq(seq)
        for p in pages:
            self._refs[p] += 1
        new = self.new()
        self._seqs[new] = (list(pages), n)
        return new

    def reorder(self, seqs: list[int], parents: list[int]) -> list[int]:
        """Beam search's step: sequence i of the result continues seqs[parents[i]]; the old ones are freed."""
        for q in seqs:
            self._seq(q)
        if len(set(seqs)) != len(seqs) or not all(0 <= p < len(seqs) for p in parents):
            _refuse(_lib.ERR_ARGS, f"PagePool: parents {parents} of {len(seqs)} different sequences")
        new = [self.fork(seqs[p]) for p in parents]
        for s in seqs:
            self.free(s)
        return new

    def free(self, seq: int) -> None:
        pages, _ = self._seq(seq)
        del self._seqs[seq]
        for p in pages:
            self._drop(p)

    def compact(self) -> list[tuple[int, int]]:
        """Moves the pages in use into the lowest ids; the copies that this takes.  Every page table
        built before is stale after it."""
        used = self.n_pages - len(self._free)
        holes = sorted(p for p in self._free if p < used)
        high = [p for p in range(used, self.n_pages) if self._refs[p]]
        pairs = list(zip(high, holes))
        to = dict(pairs)
        for a, b in pairs:
            self._refs[b], self._refs[a] = self._refs[a], 0
        for seq, (pages, n) in self._seqs.items():
            self._seqs[seq] = ([to.get(p, p) for p in pages], n)
        self._free = list(range(used, self.n_pages))
        return pairs

    def table(self, seqs: list[int], device=None, width: int | None = None):
        """(page_table, kv_lens) of `seqs` as int32 device tensors, unused entries -1."""
        import torch
        rows = [self._seq(s) for s in seqs]
        wide = max([1] + [len(p) for p, _ in rows]) if width is None else width
        if any(len(p) > wide for p, _ in rows):
            _refuse(_lib.ERR_RANGE, f"PagePool: a sequence has more than {wide} pages")
        dev = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
        t = torch.tensor([p + [-1] * (wide - len(p)) for p, _ in rows], dtype=torch.int32).reshape(len(rows), wide)
        return t.to(dev), torch.tensor([n for _, n in rows], dtype=torch.int32).to(dev)


__all__ = ["rope_frequencies", "rope_append", "paged_attention", "copy_pages", "beam_select", "PagedKvCache", "PagePool"]
