"""PagedKiviCache: a KIVI 2-bit cache of many sequences, each with a length of its own.

The reference's cache (src/kivi_sycl/cache/manager.py:52-423) and ``KiviCache`` hold one batch in lock step.
Here sequences come and go one by one and grow by any number of tokens a step; what is quantized lies in pages
of a common pool, what is not yet in a window per sequence.  Flush policy, codes, scales and zeros are those of
``KiviCache`` to the bit: a sequence of t tokens has all but its last ``R - G .. R - 1`` (fewer than ``R`` at
first) in pages.

A step of the model, over any set of its sequences::

    cache = PagedKiviCache.from_model(model, num_pages=4096, max_sequences=64)
    a, b = cache.add_sequence(), cache.add_sequence()
    batch = cache.begin([a, b], [512, 1])              # new tokens of each: rows of the step's tensors, one after the other
    for layer in range(cache.num_layers):
        out = cache.step(layer, batch, q, k, v, rotary=rotary)     # q [513, Hq, D], k and v [513, H, D]
    cache.end(batch)

``step`` is ``append`` (keys and queries turned to their positions on the way, whole groups quantized into pages) and
``attention`` (causal, over pages, window and the step's own tokens).  A sequence's tokens are attended as they
are while they are in the window or new, as their codes stand for once they are in pages.  What a step has
appended stays until its sequence is freed: tokens that a speculative decoder rejects cannot be taken back.

All kernels follow arrays in device memory, so a step can be captured: ``begin(..., max_len=...)`` with the longest
length it shall reach, and before each replay ``end(batch)`` and ``refresh(batch)``.  A layer's arrays are laid
out by its first step, which therefore is not a captured one.

``codes="e4m3"`` holds pages in 8 bits, for models that 2 bits are too coarse for: e4m3 numbers with one scale for
each block of ``group_size`` tokens and head, keys and values apart, four times the bytes.  Windows, lengths and steps are the
same.  Such a cache also takes positions on several axes (``append``) and what models do to scores
(``attention``): a cap by tanh, a bias that falls with distance, a sliding window, a prefix that all rows see.
"""
from dataclasses import dataclass, field
from typing import List, Optional, Sequence, Tuple

import torch

from .. import cabi
from ..config.model_config import detect_model_config
from ..extension.loader import kivi_native

__all__ = ["PagedKiviCache", "PagedBatch"]


@dataclass
class PagedBatch:
    """The sequences of one step: what the host knows, and the int32 arrays that the kernels follow."""
    seqs: List[int]
    new: List[int]
    held: List[int]
    max_new: int
    max_len: int
    rows: int
    page_table: torch.Tensor
    slots: torch.Tensor
    seq_lens: torch.Tensor
    cu_new: torch.Tensor
    open: bool = field(default=True)


class PagedKiviCache:
    def __init__(self, num_layers: int, head_dim: int, num_kv_heads: int, num_pages: int, max_sequences: int,
                 page_tokens: int = 256, group_size: int = 32, residual_length: int = 128, dtype=torch.bfloat16,
                 device: str = "cuda", rounding: str = "half_away", codes: str = "2bit"):
        G, R, D = group_size, residual_length, head_dim
        assert codes in ("2bit", "e4m3"), f"codes ({codes!r}) must be '2bit' or 'e4m3'"
        if codes == "2bit":
            assert D % G == 0, f"head_dim ({D}) must be divisible by group_size ({G})"
            assert G >= 4 and G % 4 == 0, f"group_size ({G}) must be >= 4 and divisible by 4"
            assert D <= 256 and (D <= 64 or D % 64 == 0), f"head_dim ({D}) must be <= 64 or a multiple of 64 up to 256"
        else:
            assert 16 <= G <= 256 and G % 16 == 0, f"group_size ({G}) must be a multiple of 16 up to 256"
            assert 16 <= D <= 256 and D % 16 == 0, f"head_dim ({D}) must be a multiple of 16 up to 256"
            assert rounding == "half_away", "rounding is of 2-bit codes: e4m3 numbers round to even"
        assert G <= R, f"group_size ({G}) must not exceed residual_length ({R})"
        assert page_tokens > 0 and page_tokens % G == 0, f"page_tokens ({page_tokens}) must be a multiple of group_size ({G})"
        assert num_pages >= 0 and max_sequences > 0 and num_kv_heads > 0
        assert dtype in (torch.bfloat16, torch.float32)
        assert rounding in ("half_away", "half_even")
        self.num_layers, self.head_dim, self.num_kv_heads, self.codes = num_layers, D, num_kv_heads, codes
        self.G, self.R, self.page_tokens, self.dtype = G, R, page_tokens, dtype
        self.num_pages, self.max_sequences = num_pages, max_sequences
        self.device = torch.device(device)
        self.rounding = cabi.ROUND_HALF_AWAY if rounding == "half_away" else cabi.ROUND_HALF_EVEN
        self._layers: List[Optional[Tuple[torch.Tensor, ...]]] = [None] * num_layers
        self._free_pages = list(range(num_pages - 1, -1, -1))
        self._free_slots = list(range(max_sequences - 1, -1, -1))
        self._pages: dict = {}                     # sequence -> its pages
        self._lens: dict = {}                      # sequence -> tokens held
        self._steps: dict = {}                     # sequence -> its step that has not ended

    @classmethod
    def from_model(cls, model, num_pages: int, max_sequences: int, **kwargs) -> "PagedKiviCache":
        cfg = detect_model_config(model)
        return cls(cfg["num_layers"], cfg["head_dim"], cfg["num_kv_heads"], num_pages, max_sequences, **kwargs)

    # ------------------------------------------------------------------ sequences
    def quantized(self, tokens: int) -> int:
        """How many of a sequence's ``tokens`` are in pages."""
        return ((tokens - self.R) // self.G + 1) * self.G if tokens >= self.R else 0

    def add_sequence(self) -> int:
        """A new, empty sequence; its number stays its until ``free``."""
        if not self._free_slots:
            raise RuntimeError(f"all {self.max_sequences} sequences are taken")
        s = self._free_slots.pop()
        self._pages[s], self._lens[s] = [], 0
        return s

    def free(self, seq: int) -> None:
        """Give a sequence's window and pages back.  Kernels queued before may still read them: later steps
        come behind those on the same stream.  A step of it that has not ended is given up, for its other
        sequences too (``begin``)."""
        self._give_up(seq)
        self._free_pages.extend(reversed(self._pages.pop(seq)))
        del self._lens[seq]
        self._free_slots.append(seq)

    def _give_up(self, seq: int) -> None:
        step = self._steps.get(seq)
        if step is not None:
            step.open = False
            for s in step.seqs:
                self._steps.pop(s, None)
                self._trim(s)

    def _pages_for(self, tokens: int) -> int:
        return -(-self.quantized(tokens) // self.page_tokens)

    def _trim(self, seq: int) -> None:
        """Give back the pages that a step took and did not come to fill."""
        pages, keep = self._pages[seq], self._pages_for(self._lens[seq])
        self._free_pages.extend(reversed(pages[keep:]))
        del pages[keep:]

    def length(self, seq: int) -> int:
        return self._lens[seq]

    @property
    def free_pages(self) -> int:
        return len(self._free_pages)

    def _layer(self, i: int) -> Tuple[torch.Tensor, ...]:
        if self._layers[i] is None:
            # (the arrays would belong to the graph, and every replay would empty them)
            if self.device.type == "cuda" and torch.cuda.is_current_stream_capturing():
                raise RuntimeError(f"layer {i} is used for the first time in a captured step: run a step outside first")
            P, H, D, G, R, T = max(1, self.num_pages), self.num_kv_heads, self.head_dim, self.G, self.R, self.page_tokens
            z = lambda *s, dtype=torch.float32: torch.zeros(*s, dtype=dtype, device=self.device)  # noqa: E731
            if self.codes == "e4m3":
                self._layers[i] = (z(P, H, T, D, dtype=torch.uint8), z(P, H, T // G), z(P, H, T, D, dtype=torch.uint8), z(P, H, T // G),
                                   z(self.max_sequences, H, R, D, dtype=self.dtype), z(self.max_sequences, H, R, D, dtype=self.dtype))
                return self._layers[i]
            self._layers[i] = (z(P, H, T // G, D * G // 4, dtype=torch.uint8), z(P, H, T // G, D), z(P, H, T // G, D),
                               z(P, H, T, D // 4, dtype=torch.uint8), z(P, H, T, D // G), z(P, H, T, D // G),
                               z(self.max_sequences, H, R, D, dtype=self.dtype), z(self.max_sequences, H, R, D, dtype=self.dtype))
        return self._layers[i]

    # ------------------------------------------------------------------ steps
    def _start(self, seqs, lens) -> None:
        """Give up the steps of ``seqs`` that have not ended and take the pages for ``lens`` tokens; raises before
        anything has changed."""
        touched = set(seqs).union(*(self._steps[s].seqs for s in seqs if s in self._steps))
        free = len(self._free_pages) + sum(len(self._pages[s]) - self._pages_for(self._lens[s]) for s in touched)
        need = {s: self._pages_for(n) - self._pages_for(self._lens[s]) for s, n in zip(seqs, lens)}
        if sum(need.values()) > free:
            raise RuntimeError(f"{sum(need.values())} pages are needed, {free} of {self.num_pages} are free")
        for s, n in need.items():
            self._give_up(s)
            self._trim(s)
        for s, n in need.items():
            self._pages[s].extend(self._free_pages.pop() for _ in range(n))

    def _table(self, seqs, width) -> torch.Tensor:
        return torch.tensor([self._pages[s] + [-1] * (width - len(self._pages[s])) for s in seqs], dtype=torch.int32).reshape(len(seqs), width)

    def begin(self, seqs: Sequence[int], new: Sequence[int], max_len: Optional[int] = None) -> PagedBatch:
        """Start a step in which sequence ``seqs[i]`` gets ``new[i]`` tokens (0 is allowed): takes the pages that the
        step fills and lays down the arrays its kernels follow.  A step of one of them that has not ended is given up and its pages
        are given back; what it has appended to some layers is not undone, so give up only what has not run.  ``max_len``: the longest length a captured step
        shall reach (default: this step's)."""
        seqs, new = [int(s) for s in seqs], [int(n) for n in new]
        assert len(seqs) == len(new) and seqs, "begin() needs at least one sequence, and new tokens for each"
        assert len(set(seqs)) == len(seqs), "a sequence appears twice in one step"
        for s in seqs:
            assert s in self._lens, f"sequence {s} is not there"
        assert all(n >= 0 for n in new), "new tokens cannot be negative"
        held = [self._lens[s] for s in seqs]
        longest = max(h + n for h, n in zip(held, new))
        assert max_len is None or max_len >= longest, f"max_len ({max_len}) is below this step's longest length ({longest})"
        self._start(seqs, [h + n for h, n in zip(held, new)])
        max_len = max_len or longest
        cu = [0]
        for n in new:
            cu.append(cu[-1] + n)
        width = max(1, -(-self.quantized(max_len) // self.page_tokens))
        dev = lambda x: torch.tensor(x, dtype=torch.int32).to(self.device)  # noqa: E731
        batch = PagedBatch(seqs, new, held, max(new), max_len, cu[-1], self._table(seqs, width).to(self.device), dev(seqs), dev(held), dev(cu))
        self._steps.update((s, batch) for s in seqs)
        return batch

    def append(self, layer: int, batch: PagedBatch, k: torch.Tensor, v: torch.Tensor, rotary: Optional[torch.Tensor] = None,
               q: Optional[torch.Tensor] = None, interleaved: bool = False, positions: Optional[torch.Tensor] = None,
               pair_axis: Optional[torch.Tensor] = None):
        """Append the step's keys and values [rows, H, D] (of the cache's dtype).  With ``rotary`` [positions, rotary_dim]
        (fp32: cosines, then sines) keys and queries are turned to their positions first; returns (q, k) as the
        attention wants them.  Once per layer and step: window slots that it has read are written again.

        ``positions`` int32 [axes, rows] and ``pair_axis`` int32 [rotary_dim / 2] (``codes="e4m3"``): pair i of a token is
        turned by its position on axis ``pair_axis[i]`` in place of its place in the sequence (images and video: time, height,
        width)."""
        assert batch.open, "the step has ended"
        q_out = k_out = None
        if rotary is not None:
            k_out = torch.empty(k.shape, dtype=k.dtype, device=k.device)
            q_out = None if q is None else torch.empty(q.shape, dtype=q.dtype, device=q.device)
        where = (batch.page_table, batch.slots, batch.seq_lens, batch.cu_new, batch.max_new, batch.max_len, self.G)
        turned = q if rotary is not None else None
        if self.codes == "e4m3":
            kivi_native.paged8_append(k, v, *self._layer(layer), *where, rotary, turned, q_out, k_out, interleaved, positions, pair_axis)
        else:
            if positions is not None or pair_axis is not None:
                raise ValueError("positions on several axes need codes='e4m3'")
            kivi_native.paged_append(k, v, *self._layer(layer), *where, rotary, turned, q_out, k_out, interleaved, self.rounding)
        return (q, k) if rotary is None else (q_out, k_out)

    def attention(self, layer: int, batch: PagedBatch, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, sm_scale: float = 0.0,
                  out: Optional[torch.Tensor] = None, softcap: float = 0.0, slopes: Optional[torch.Tensor] = None, window: int = 0,
                  prefix: Optional[torch.Tensor] = None) -> torch.Tensor:
        """Causal attention of the step's rows, after ``append`` of the same step: [rows, Hq, D].  q, k: as ``append``
        returned them.

        With ``codes="e4m3"``, x a score: ``softcap`` > 0: x becomes softcap * tanh(x / softcap); ``slopes`` fp32 [Hq]: then x gets
        slopes[head] * (place of the token - place of the row); ``window`` > 0: a row sees the last ``window`` tokens up to its
        own; ``prefix`` int32 [sequences of the batch]: and the sequence's first ``prefix`` tokens, those behind it too."""
        assert batch.open, "the step has ended"
        if out is None:
            out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
        where = (batch.page_table, batch.slots, batch.seq_lens, batch.cu_new, batch.max_new, batch.max_len)
        if self.codes == "e4m3":
            kivi_native.paged8_attention(q, k, v, *self._layer(layer), *where, out, self.G, sm_scale, softcap, slopes, window, prefix)
        else:
            if softcap or slopes is not None or window or prefix is not None:
                raise ValueError("softcap, slopes, window and prefix need codes='e4m3'")
            kivi_native.paged_attention(q, k, v, *self._layer(layer), *where, out, self.G, sm_scale)
        return out

    def step(self, layer: int, batch: PagedBatch, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, rotary: Optional[torch.Tensor] = None,
             sm_scale: float = 0.0, interleaved: bool = False, positions: Optional[torch.Tensor] = None, pair_axis: Optional[torch.Tensor] = None,
             **rules) -> torch.Tensor:
        """``append`` and ``attention`` of one layer (``rules``: softcap, slopes, window, prefix)."""
        q, k = self.append(layer, batch, k, v, rotary, q, interleaved, positions, pair_axis)
        return self.attention(layer, batch, q, k, v, sm_scale, **rules)

    def end(self, batch: PagedBatch) -> None:
        """The step is done in all layers: its tokens are the sequences' own."""
        assert batch.open, "the step has ended"
        for s, h in zip(batch.seqs, batch.held):
            assert self._lens.get(s) == h, f"sequence {s} has changed during the step"
        for s, h, n in zip(batch.seqs, batch.held, batch.new):
            self._lens[s] = h + n
            self._steps.pop(s, None)
        batch.open = False

    def refresh(self, batch: PagedBatch) -> None:
        """Open the next step of the same sequences and numbers of new tokens in the same arrays (for a captured
        step, whose kernels have their addresses)."""
        assert not batch.open, "the step has not ended"
        for s in batch.seqs:
            assert s in self._lens, f"sequence {s} is not there"
        held = [self._lens[s] for s in batch.seqs]
        lens = [h + n for h, n in zip(held, batch.new)]
        assert max(lens) <= batch.max_len, f"the step reaches {max(lens)} tokens, it was begun for {batch.max_len}"
        self._start(batch.seqs, lens)
        batch.page_table.copy_(self._table(batch.seqs, batch.page_table.shape[1]))
        batch.seq_lens.copy_(torch.tensor(held, dtype=torch.int32))
        batch.held, batch.open = held, True
        self._steps.update((s, batch) for s in batch.seqs)

    # ------------------------------------------------------------------ reading back
    def read(self, layer: int, seq: int, start: int = 0, stop: Optional[int] = None) -> Tuple[torch.Tensor, torch.Tensor]:
        """Tokens start .. stop-1 of a sequence as they are served: fp32 keys and values [tokens, H, D].  Not while a
        step of the sequence is open: the step's append has moved tokens to pages and taken their slots in the window."""
        held = self._lens[seq]
        stop = held if stop is None else stop
        assert 0 <= start <= stop <= held, f"tokens {start} .. {stop} of a sequence of {held}"
        assert seq not in self._steps, f"a step of sequence {seq} has not ended"
        k = torch.empty(stop - start, self.num_kv_heads, self.head_dim, device=self.device)
        v = torch.empty_like(k)
        if stop > start:
            dev = lambda x: torch.tensor(x, dtype=torch.int32).to(self.device)  # noqa: E731
            width = max(1, len(self._pages[seq]))
            read = kivi_native.paged8_read if self.codes == "e4m3" else kivi_native.paged_read
            read(*self._layer(layer), self._table([seq], width).to(self.device), dev([seq]), dev([held]), dev([start]), dev([0, stop - start]),
                 stop - start, k, v, self.G)
        return k, v

    def check_device_fault(self) -> None:
        """Raise if a kernel has met arrays that point outside the cache, or a wait has run out (synchronises).  The
        word is that of the cache's device, whichever is the current one."""
        with torch.cuda.device(self.device):
            word = cabi.device_fault()
            if word:
                cabi.device_fault_clear()
        if word:
            raise RuntimeError(f"kivi_cuda device fault word = {word}; outputs since the last check may be wrong")

    def __repr__(self):
        return (f"PagedKiviCache(layers={self.num_layers}, head_dim={self.head_dim}, codes={self.codes}, G={self.G}, R={self.R}, "
                f"pages={self.num_pages - len(self._free_pages)}/{self.num_pages} of {self.page_tokens}, sequences={len(self._lens)})")
