"""Keys and values of several sequences in pages, for dense decoding beside
the routed one: `PagedCache.append` writes new rows, `attend` runs one new
query token of every sequence over its pages, and `evict` bounds a cache by
accumulated attention weight.  No counterpart in the reference.

Any head layout with head_dim 64, 128 or 256 in bf16, fp16 or fp32, and up to 64
GiB each of k and v pages (NotImplementedError otherwise); for inference, without
gradients.  As for `Native8B`: validation happens on the host before
anything is enqueued (ValueError), calls go to the current stream of the
cache's device, never synchronise and can be captured into a HIP graph after
one eager call has made their workspaces; lengths and page table are read on
the device.  An instance's buffers are shared state: one instance per stream,
and graphs captured from it are replayed on one stream.  A slot below a
sequence's length that has no page is reported at the next call
(RuntimeError); the results since then are invalid.
"""
from __future__ import annotations

import ctypes
import itertools
import math
import threading
from collections import deque

import torch

from . import _lib

DTYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
HEAD_DIMS = (64, 128, 256)
MAX_SCALE = torch.finfo(torch.float32).max / 1.4426950408889634
ERR_PAGES, ERR_ROWS = 4, 8  # codes of the error word, as the kernels write them
ERROR_MESSAGES = {ERR_PAGES: "a slot below a sequence's length has no page",
                  ERR_ROWS: "the offsets of an append did not ascend from 0 to its number of rows"}
_SCORED = ("seen", "scores", "positions")


# The current stream's handle; building a torch.cuda.Stream for it takes 1 us beside a
# call's 7.
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda index: torch.cuda.current_stream(index).cuda_stream)


def _check(cond, what):
    if not cond:
        raise ValueError(what)


def _i32(x, shape, device, what):
    _check(isinstance(x, torch.Tensor) and x.dtype == torch.int32 and tuple(x.shape) == shape and x.is_contiguous()
           and x.device == device, f"{what} must be a contiguous int32 {list(shape)} on the cache's device")
    return x


class _ErrorWord:
    """The error word of a cache, its forks and what it was resized to, in pinned
    host memory that the kernels write and a call reads without a tensor operation:
    16 bytes of a page of them, since pinning memory for each takes longer than the
    rest of a cache's set-up.  Given back when the last of the caches is gone; as
    launches that may write it can still be queued then, another cache gets it only
    after the device has been waited for, once for every PER_PAGE words."""

    PER_PAGE = 256
    homes: dict = {}  # device index -> (words that nothing enqueued writes, words given back)
    pages: list = []
    lock = threading.Lock()  # for refilling (not for giving back, which the collector may do at any time)

    def __init__(self, lib, device):
        fresh, self.home = self.homes.setdefault(device.index, (deque(), deque()))
        while not hasattr(self, "slot"):
            try:
                self.slot = fresh.popleft()
            except IndexError:
                with self.lock:
                    if not fresh:
                        self._refill(lib, device, fresh, self.home)
        self.address = self.slot[0]
        self.word = ctypes.c_int32.from_address(self.slot[1])
        self.word.value = 0

    @classmethod
    def _refill(cls, lib, device, fresh, given_back):
        count = len(given_back)
        with torch.cuda.device(device):
            if count >= cls.PER_PAGE and not torch.cuda.is_current_stream_capturing():
                torch.cuda.synchronize(device)
                fresh.extend(given_back.popleft() for _ in range(count))
                return
            page = torch.zeros(cls.PER_PAGE, 4, dtype=torch.int32, device="cpu", pin_memory=True)
            address = lib.query("prismkv_mapped_pointer", page.data_ptr())
        if not address:
            raise RuntimeError("prismkv_mapped_pointer: the pinned error word is not device-accessible")
        cls.pages.append(page)
        fresh.extend((address + 16 * i, page.data_ptr() + 16 * i) for i in range(cls.PER_PAGE))

    def __del__(self):
        if hasattr(self, "slot"):
            self.home.append(self.slot)


class PagedCache:
    """A cache of `sequences` sequences in `pages` pages of `page_size` slots;
    a sequence takes at most `max_pages` of them.

    Tensors: k, v [pages, kv_heads, page_size, head_dim]; table i32
    [sequences, max_pages] (-1: no page); lengths i32 [sequences]; and, if
    `scored`, seen i32 [sequences] (tokens appended so far), scores f32 and
    positions i32 [sequences, kv_heads, max_pages * page_size] (each slot's
    accumulated attention weight and its token's number), which eviction goes
    by.  Slots at and behind a length hold nothing of meaning.

    `reserve` and `release` hand out pages on the host; calls that take `into`
    (a `fork`) write their results there and leave this cache's own lengths,
    scores and positions, so that an `append`, an `attend` or a step can be taken
    back.  An `evict` cannot: it moves rows in the shared pages.  A fork holds what
    this cache held when it was made, and a call into it writes what that call
    changes; it is made anew when this cache has gone on by itself."""

    def __init__(self, sequences, pages, max_pages, *, page_size=64, kv_heads=8, head_dim=128, dtype=torch.bfloat16,
                 scored=False, device="cuda", library=None, _err=None):
        for value, what in ((sequences, "sequences"), (pages, "pages"), (max_pages, "max_pages"),
                            (page_size, "page_size"), (kv_heads, "kv_heads")):
            _check(int(value) >= 1, f"{what} must be positive")
        device = torch.device(device)
        _check(device.type == "cuda", "native backend requires a device tensor")
        if device.index is None:
            device = torch.device("cuda", torch.cuda.current_device())
        _native_types(int(head_dim), dtype)
        shape = (int(pages), int(kv_heads), int(page_size), int(head_dim))
        slots = int(max_pages) * int(page_size)
        _check_slots(int(sequences), slots)
        if math.prod(shape) * dtype.itemsize > 1 << 36:
            raise NotImplementedError("pages that span at most 64 GiB (of k, and of v)")
        k = torch.zeros(shape, dtype=dtype, device=device)
        v = torch.zeros(shape, dtype=dtype, device=device)
        table = torch.full((int(sequences), int(max_pages)), -1, dtype=torch.int32, device=device)
        lengths = torch.zeros(int(sequences), dtype=torch.int32, device=device)
        meta = {}
        if scored:
            meta = dict(seen=torch.zeros_like(lengths),
                        scores=torch.zeros(int(sequences), int(kv_heads), slots, dtype=torch.float32, device=device),
                        positions=torch.zeros(int(sequences), int(kv_heads), slots, dtype=torch.int32, device=device))
        self._setup(k, v, table, lengths, library=library, err=_err, **meta)
        self._free = list(range(int(pages)))[::-1]
        self._pages = [[] for _ in range(int(sequences))]

    @classmethod
    def from_tensors(cls, k, v, table, lengths, *, seen=None, scores=None, positions=None, library=None):
        """A cache over the caller's own tensors (pages of any strides of
        16-byte multiples, the same for k and v), whose page table the caller
        keeps: `reserve` and `release` are not offered.  seen, scores and
        positions are given all or none."""
        obj = cls.__new__(cls)
        obj._setup(k, v, table, lengths, seen=seen, scores=scores, positions=positions, library=library)
        return obj

    def _setup(self, k, v, table, lengths, *, seen=None, scores=None, positions=None, library=None, err=None):
        _check(isinstance(k, torch.Tensor) and k.device.type == "cuda", "native backend requires a device tensor")
        _check(k.dim() == 4 and k.shape == v.shape and k.dtype == v.dtype and k.device == v.device,
               "K and V pages [pages, kv_heads, page_size, head_dim] of one type required")
        pages, kv_heads, page_size, head_dim = k.shape
        _native_types(head_dim, k.dtype)
        _check(min(k.shape) >= 1, "K and V pages [pages, kv_heads, page_size, head_dim] of one type required")
        es = k.element_size()
        _check(k.stride() == v.stride() and k.stride(3) == 1, "K and V pages of equal strides and contiguous rows required")
        _check(not any(s * es % 16 for s in k.stride()[:3]) and not (k.data_ptr() | v.data_ptr()) % 16,
               "K/V rows must be 16-byte aligned")
        _check(k.stride(2) >= head_dim and (pages == 1 or k.stride(0) >= head_dim) and
               (kv_heads == 1 or k.stride(1) >= head_dim), "K/V rows must not overlap")
        if max(pages * k.stride(0), (pages - 1) * k.stride(0) + page_size * k.stride(2)) * es > 1 << 36:
            raise NotImplementedError("pages that span at most 64 GiB (of k, and of v)")
        _check(table.dim() == 2 and min(table.shape) >= 1, "an int32 page table [sequences, max_pages] required")
        sequences, max_pages = table.shape
        slots = max_pages * page_size
        _check_slots(sequences, slots)
        _i32(table, (sequences, max_pages), k.device, "table")
        _i32(lengths, (sequences,), k.device, "lengths")
        given = [x is not None for x in (seen, scores, positions)]
        _check(all(given) or not any(given), "seen, scores and positions are given together")
        if all(given):
            shape = (sequences, kv_heads, slots)
            _i32(seen, (sequences,), k.device, "seen")
            _i32(positions, shape, k.device, "positions")
            _check(isinstance(scores, torch.Tensor) and scores.dtype == torch.float32 and tuple(scores.shape) == shape
                   and scores.is_contiguous() and scores.device == k.device,
                   f"scores must be a contiguous float32 {list(shape)} on the cache's device")
        self.lib = _lib.load(library)
        if self.lib.missing:
            raise RuntimeError(f"{self.lib.path.name} lacks entry points {self.lib.missing}; rebuild it")
        self._tensors = (k, v, table, lengths, seen, scores, positions)
        self.device = k.device
        self._shape = (sequences, kv_heads, head_dim, page_size, max_pages)
        # the buffers that calls read and write besides the pages, as [from, to)
        self._spans = tuple((x.data_ptr(), x.data_ptr() + 4 * x.numel()) for x in self._tensors[3:] if x is not None)
        _check(not any(_overlap(x, y) for x, y in itertools.combinations(self._spans, 2)),
               "lengths, seen, scores and positions must not overlap")
        self._free = self._pages = None
        self._attend_work, self._evict_work = {}, None
        self._err = _ErrorWord(self.lib, self.device) if err is None else err
        # what the C entries read of the cache; its tensors are fixed from here on
        pointers = [0 if x is None else x.data_ptr() for x in self._tensors]
        self._desc = _lib.PagedCacheDesc(*pointers, self._err.address, pages, *k.stride()[:3], *self._shape,
                                         DTYPES[k.dtype])
        self._pointer = ctypes.c_void_p(ctypes.addressof(self._desc))

    # ------------------------------------------------------------ pages

    k, v, table, lengths, seen, scores, positions = (property(lambda self, i=i: self._tensors[i]) for i in range(7))

    @property
    def scored(self):
        return self.scores is not None

    @property
    def slots(self):
        """Slots of one sequence's table."""
        return self._shape[3] * self._shape[4]

    def fork(self):
        """A cache over the same pages and page table with copies of this
        one's lengths, scores and positions: the `into` of a step that may be
        taken back.  (Rows that `evict` moves are moved for both.)"""
        obj = PagedCache.__new__(PagedCache)
        meta = {name: getattr(self, name).clone() for name in _SCORED} if self.scored else {}
        obj._setup(self.k, self.v, self.table, self.lengths.clone(), library=self.lib.path, err=self._err, **meta)
        return obj

    def reserve(self, tokens):
        """Makes room for `tokens` slots in every sequence (an int, or one per
        sequence), from the free pages; RuntimeError when they run out, and
        nothing is then reserved.  Pages are kept until `release`."""
        self._owns_pages()
        sequences, _, _, page_size, max_pages = self._shape
        tokens = [int(tokens)] * sequences if isinstance(tokens, int) else [int(t) for t in tokens]
        _check(len(tokens) == sequences, "one token count per sequence required")
        _check(all(0 <= t <= self.slots for t in tokens), f"token counts must be in [0, {self.slots}]")
        more = [max(0, -(-t // page_size) - len(held)) for t, held in zip(tokens, self._pages)]
        if sum(more) > len(self._free):
            raise RuntimeError(f"{sum(more)} pages wanted, {len(self._free)} free")
        if not any(more):
            return
        for held, count in zip(self._pages, more):
            held.extend(self._free.pop() for _ in range(count))
        self._write_table()

    def release(self, sequence, tokens=0):
        """Gives back the pages of a sequence behind its first `tokens` slots;
        the caller sees to it that its length (and that of forks) is no larger."""
        self._owns_pages()
        _check(0 <= int(sequence) < self._shape[0] and int(tokens) >= 0, "no such sequence or slot")
        held, page_size = self._pages[int(sequence)], self._shape[3]
        keep = -(-int(tokens) // page_size)
        if keep < len(held):
            self._free.extend(reversed(held[keep:]))
            del held[keep:]
            self._write_table()

    def resized(self, pages, max_pages):
        """A new cache of `pages` pages, at most `max_pages` to a sequence, with
        this one's contents: per sequence its first max_pages pages, which the
        caller knows to hold its length, their scores and positions.  (A cut
        cache in the table of its longest prompt would keep that prompt's memory,
        and its cuts the cost of that many slots.)  Reports of this cache's launches
        go to it as well."""
        self._owns_pages()
        sequences, kv_heads, head_dim, page_size, _ = self._shape
        counts = [min(len(held), int(max_pages)) for held in self._pages]
        _check(sum(counts) <= int(pages), "the sequences' pages do not fit")
        new = PagedCache(sequences, pages, max_pages, page_size=page_size, kv_heads=kv_heads, head_dim=head_dim,
                         dtype=self.k.dtype, scored=self.scored, device=self.device, library=self.lib.path, _err=self._err)
        new.reserve([count * page_size for count in counts])
        for held, own, count in zip(self._pages, new._pages, counts):
            new.k[own] = self.k[held[:count]]
            new.v[own] = self.v[held[:count]]
        new.lengths.copy_(self.lengths)
        if self.scored:
            slots = min(new.slots, self.slots)
            new.seen.copy_(self.seen)
            new.scores[:, :, :slots] = self.scores[:, :, :slots]
            new.positions[:, :, :slots] = self.positions[:, :, :slots]
        return new

    def _owns_pages(self):
        if self._pages is None:
            raise RuntimeError("the page table of this cache is kept by the caller (or the cache it was forked from)")
        with torch.cuda.device(self.device):
            if torch.cuda.is_current_stream_capturing():
                raise RuntimeError("pages cannot be handed out inside a capture")

    def _write_table(self):
        max_pages = self._shape[4]
        rows = torch.tensor([held + [-1] * (max_pages - len(held)) for held in self._pages], dtype=torch.int32)
        self.table.copy_(rows)

    # ------------------------------------------------------------ calls

    def check_errors(self):
        """RuntimeError if an earlier launch found a slot below a sequence's
        length without a page, or offsets that do not cover an append's rows:
        the results since the last check are invalid.  Reads a host-mapped word
        (no synchronisation, launches that have not run yet are not seen) and
        clears it."""
        code = self._err.word.value
        if code:
            torch.cuda.synchronize(self.device)
            self._err.word.value = 0
            raise RuntimeError(f"paged cache: {ERROR_MESSAGES.get(code, code)}; the results of the launches since the "
                               "last check are invalid")

    def _call(self, name, *args):
        index = self.device.index
        if torch.cuda.current_device() == index:
            self.lib.call(name, *args, stream=_raw_stream(index))
        else:
            with torch.cuda.device(index):
                self.lib.call(name, *args, stream=_raw_stream(index))

    def _into(self, into):
        if into is None or into is self:
            return self
        if not isinstance(into, PagedCache) or into.device != self.device:
            raise ValueError("into must be a fork of this cache")
        a, b = self._desc, into._desc
        if (a.k != b.k or a.v != b.v or a.table != b.table or a.pages != b.pages or a.page_stride != b.page_stride
                or a.head_stride != b.head_stride or a.slot_stride != b.slot_stride or into._shape != self._shape
                or a.dtype != b.dtype or (a.scores == 0) != (b.scores == 0)):
            raise ValueError("into must be a fork of this cache")
        # (what `fork` made has buffers of its own)
        if into._err is not self._err and into._spans != self._spans and any(
                _overlap(x, y) for x in self._spans for y in into._spans):
            raise ValueError("into's lengths, seen, scores and positions must be all of this cache's or overlap none")
        return into

    def _workspace(self, nbytes, zero):
        """A new workspace (zeroed up to `zero` bytes); never inside a capture,
        whose memory would not outlive the graph and whose fill would not have run."""
        with torch.cuda.device(self.device):
            if torch.cuda.is_current_stream_capturing():
                raise RuntimeError("the first call of a kind makes its workspace: run it once before the capture")
            work = torch.empty(max(nbytes, 16), dtype=torch.uint8, device=self.device)
            work[:zero].zero_()
            return work

    def append(self, k, v, offsets=None, *, into=None):
        """Writes new rows behind every sequence's: k and v [rows, kv_heads,
        head_dim] of the cache's type, one row per sequence, or with `offsets`
        (i32 [sequences + 1], ascending from 0) rows offsets[b] .. offsets[b +
        1] for sequence b.  Advances the lengths; of a scored cache also the
        tokens seen, the rows starting with score 0.  The slots need pages
        (`reserve`); a row without one is dropped and reported."""
        to = self if into is None else self._into(into)
        sequences, kv_heads, head_dim, _, _ = self._shape
        shape, ks, vs = k.shape, k.stride(), v.stride()
        if len(shape) != 3 or v.shape != shape or shape[1] != kv_heads or shape[2] != head_dim:
            raise ValueError(f"K and V rows [rows, {kv_heads}, {head_dim}] required")
        dtype, device = self.k.dtype, self.device
        if k.dtype != dtype or v.dtype != dtype or k.device != device or v.device != device:
            raise ValueError("K and V rows of the cache's type on its device required")
        rows, es = shape[0], k.element_size()
        if rows and (ks[2] != 1 or vs[2] != 1):
            raise ValueError("contiguous head dimension required")
        kp, vp = k.data_ptr(), v.data_ptr()
        if ((ks[0] | ks[1] | vs[0] | vs[1]) * es | kp | vp) % 16:
            raise ValueError("K/V rows must be 16-byte aligned")
        if offsets is not None:
            _i32(offsets, (sequences + 1,), self.device, "offsets")
        elif rows != sequences:
            raise ValueError("one row per sequence, or offsets, required")
        self.check_errors()
        self._call("prismkv_paged_append", self._pointer, to._pointer, kp, vp,
                   0 if offsets is None else offsets.data_ptr(), rows, ks[0], ks[1], vs[0], vs[1])

    def attend(self, q, *, scale=None, accumulate=False, lse=None, into=None):
        """Softmax attention of q [sequences, heads, head_dim] (heads a
        multiple of the cache's kv_heads; consecutive heads share a KV head)
        over each sequence's slots, scaled by `scale` (default 1 /
        sqrt(head_dim)); the output has q's shape and type, 0 for an empty
        sequence.  `accumulate` adds to every slot's score its weight, summed
        over the heads that share it.  `lse`, an f32 [sequences, heads] tensor,
        receives the logarithm of each softmax's sum (-inf for an empty one)."""
        to = self if into is None else self._into(into)
        group, scale = self._check_q(q, scale, accumulate, lse)
        accumulate = bool(accumulate)
        return self._attend(q, group, scale, accumulate, lse, to, 0, self._attend_workspace(group, accumulate))

    def _check_q(self, q, scale, accumulate, lse):
        """The query heads per KV head, and the scale."""
        sequences, kv_heads, head_dim, _, _ = self._shape
        shape = q.shape
        if (len(shape) != 3 or shape[0] != sequences or shape[2] != head_dim or shape[1] < 1 or shape[1] % kv_heads
                or not q.is_contiguous()):
            raise ValueError(f"contiguous Q[{sequences}, a multiple of {kv_heads} heads, {head_dim}] required")
        if q.dtype != self.k.dtype or q.device != self.device:
            raise ValueError("Q of the cache's type on its device required")
        if q.data_ptr() % 16:
            raise ValueError("Q rows must be 16-byte aligned")
        group = shape[1] // kv_heads
        if group > 1024:
            raise NotImplementedError("at most 1024 query heads per KV head")
        if accumulate and self.scores is None:
            raise ValueError("accumulate needs a scored cache")
        scale = 1.0 / math.sqrt(head_dim) if scale is None else float(scale)
        if not abs(scale) <= MAX_SCALE:
            raise ValueError("a scale that is finite in float32, as times log2(e), required")
        if lse is not None and (lse.dtype != torch.float32 or lse.shape != q.shape[:2] or not lse.is_contiguous()
                                or lse.device != self.device):
            raise ValueError("lse must be a contiguous float32 [sequences, heads] on the cache's device")
        return group, scale

    def _attend_workspace(self, group, accumulate):
        work = self._attend_work.get((group, accumulate))
        if work is None:
            # (the leading counters are zeroed; the kernels leave them so)
            sequences, kv_heads, head_dim, _, _ = self._shape
            nbytes = self.lib.query("prismkv_paged_attend_work_bytes", sequences, kv_heads, group, head_dim, self.slots,
                                    int(accumulate), self._desc.dtype)
            if not nbytes:
                raise NotImplementedError("less than 2^31 blocks of 32 slots in all (of every sequence's table, KV head "
                                          "and 16 query heads on it)")
            work = self._attend_work[(group, accumulate)] = self._workspace(
                nbytes, 4 * sequences * kv_heads * ((group + 15) // 16))
        return work

    def _attend(self, q, group, scale, accumulate, lse, to, flags, work):
        self.check_errors()
        out = torch.empty_like(q)
        self._call("prismkv_paged_attend", self._pointer, to._pointer, q.data_ptr(), 0 if lse is None else lse.data_ptr(),
                   work.data_ptr(), out.data_ptr(), group, flags + accumulate, scale, work.numel())
        return out

    def __call__(self, q, k, v, *, scale=None, accumulate=False, lse=None, into=None):
        """A decode step: `append` one row of k and v [sequences, kv_heads,
        head_dim] to every sequence, then `attend`.  With `into` both results
        go there, the new rows into the shared pages behind this cache's
        lengths."""
        to = self if into is None else self._into(into)
        # nothing is appended for a query that is refused
        group, scale = self._check_q(q, scale, accumulate, lse)
        accumulate = bool(accumulate)
        work = self._attend_workspace(group, accumulate)
        self.append(k, v, into=into)
        return self._attend(q, group, scale, accumulate, lse, to, 2, work)

    def evict(self, keep, *, recent=0, sinks=0, into=None):
        """Cuts every sequence longer than `keep` slots (an int, or i32
        [sequences]) to them, per KV head: the `recent` newest tokens and the
        first `sinks` ones stay before all others, then the slots of the
        highest scores (NaN above all numbers), the lower slot on ties.  The
        fewest rows move: a slot that stays and lies behind the budget goes
        into one that became free, in ascending order, with its score and
        position; the order of the slots is not that of the tokens afterwards.
        The pages stay reserved (`release`).  With `into` the rows move in the
        shared pages all the same, over rows that this cache still lists: it may
        then repeat the same cut, into a fork or itself, but not be attended to,
        appended to or cut otherwise."""
        to = self if into is None else self._into(into)
        _check(self.scored, "evict needs a scored cache")
        sequences, kv_heads, _, _, _ = self._shape
        keeps = 0
        if isinstance(keep, torch.Tensor):
            keeps, keep = _i32(keep, (sequences,), self.device, "keep").data_ptr(), 0
        keep, recent, sinks = int(keep), int(recent), int(sinks)
        _check(min(keep, recent, sinks) >= 0 and max(keep, recent, sinks) < 2 ** 31,
               "keep, recent and sinks must be in [0, 2^31)")
        self.check_errors()
        if self._evict_work is None:
            self._evict_work = self._workspace(
                self.lib.query("prismkv_paged_evict_work_bytes", sequences, kv_heads, self.slots), 4 * sequences)
        self._call("prismkv_paged_evict", self._pointer, to._pointer, keeps, self._evict_work.data_ptr(), keep, recent,
                   sinks, self._evict_work.numel())

    def buffer_bytes(self):
        """Live tensors held here, by name (a fork's pages are its origin's)."""
        names = ("k", "v", "table", "lengths", "seen", "scores", "positions")
        held = {name: x for name, x in zip(names, self._tensors) if x is not None}
        if self._evict_work is not None:
            held["evict_work"] = self._evict_work
        held.update((f"attend_work{key}", x) for key, x in self._attend_work.items())
        return {name: x.numel() * x.element_size() for name, x in held.items()}


def _overlap(x, y):
    return x[0] < y[1] and y[0] < x[1]


def _native_types(head_dim, dtype):
    if head_dim not in HEAD_DIMS or dtype not in DTYPES:
        raise NotImplementedError("the paged cache holds bf16, fp16 or fp32 rows of head_dim 64, 128 or 256")


def _check_slots(sequences, slots):
    if slots > 1 << 30 or sequences * slots >= 1 << 31 or sequences > 65535:
        raise NotImplementedError("at most 2^30 slots per sequence, 2^31 in all and 65535 sequences")
