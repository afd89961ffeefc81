"""A bank of key / value rows held in 4 bits on MI355X, read by softmax attention, that drops the rows that attention uses least.

It stands next to ``MemoryBank`` (``models/memory_bank.py:35-72``: rows in whole floats, the oldest leave first, read by a dense product and
a softmax as in ``track_semi/comatch.py:187-189``) and has no reference counterpart: rows belong to ``heads`` heads of ``batch`` sequences, as
the keys and values of an attention layer do; ``heads=1, batch=1`` is a plain feature bank.

    bank = CacheBank()
    bank.register("layer0", dim=128, k=4096, heads=8, batch=64)
    bank.push("layer0", key, value)                            # [batch, heads, T, dim], quantised to 4.25 bits a value
    out = bank.attend("layer0", query, accumulate=True)        # [batch, heads * group, T, dim]; also sums what each row got
    bank.evict("layer0", keep=2048, recent=256)                # the least attended rows leave

Storage is registered buffers (``<name>_key``, ``_key_scale``, ``_value``, ``_value_scale``, ``_weight``, ``_position``, ``_length``, ``_seen``;
layouts and the number format in ``include/mi_knn.h``), so ``.to(device)`` and ``state_dict`` behave as for the other banks.  Each rank holds
its own sequences: nothing is gathered.  No gradients: the bank is memory, as the MoCo queue is.  No CPU path.

Lengths live on the device and no call waits for it, except to copy ``counts`` that are given as a list, to look at the order of rows
after an eviction (see ``attend``), and for a ``push`` that may run over: the host knows an upper bound of the lengths and reads them back
when that bound plus the new rows passes ``k``, or when torch has written to the lengths, or put others in their place, since it knew it.
(A collective or a kernel of one's own that writes to them in place goes unnoticed: load them with ``load_state_dict`` or ``copy_``.)  All
calls can be captured into a graph; a captured ``push`` cannot look, and rows that do not fit when it is replayed are dropped."""
from __future__ import annotations

import contextlib
import ctypes
import operator

import torch
from torch import nn
from torch.autograd import forward_ad

from . import _lib

__all__ = ["CacheBank"]

_CODES = {torch.float32: _lib.MI_F32, torch.bfloat16: _lib.MI_BF16, torch.float16: _lib.MI_F16}
_PARTS = ("key", "key_scale", "value", "value_scale", "weight", "position", "length", "seen")
_DTYPES = (torch.uint8, torch.uint8, torch.uint8, torch.uint8, torch.float32, torch.int32, torch.int32, torch.int32)


def _on(device: torch.device):
    """The device's context, where it is not the current one already."""
    return contextlib.nullcontext() if torch.cuda.current_device() == device.index else torch.cuda.device(device)


_ARRAYS = {}                   # strides -> the same as a C array (there are few different ones; made anew they are 2 us a call)


def _strides(t: torch.Tensor):
    """Strides of the sequence, head and row of a [batch, heads, rows, dim] tensor; a size of one has none."""
    (a, b, c, _), (x, y, z, _) = t.shape, t.stride()
    return (x if a > 1 else 0, y if b > 1 else 0, z if c > 1 else 0)


def _array(strides):
    known = _ARRAYS.get(strides)
    if known is None:
        if len(_ARRAYS) > 1024:
            _ARRAYS.clear()
        known = _ARRAYS[strides] = (ctypes.c_int64 * 3)(*strides)
    return known


def _aligned(t: torch.Tensor):
    """``t`` itself where its rows are contiguous and start on 16 bytes, else a copy that is so; and its strides."""
    step, strides = 16 // t.element_size(), _strides(t)
    if (t.stride(3) == 1 or t.shape[3] == 1) and t.data_ptr() % 16 == 0 and not (strides[0] % step or strides[1] % step or strides[2] % step):
        return t, strides
    t = t.clone(memory_format=torch.contiguous_format)
    return t, _strides(t)


def _part_shapes(k, batch, heads, dim):
    width = 64 if dim <= 64 else 128 if dim <= 128 else 256
    rows = (k + 63) // 64 * 64
    held, scales, each = (batch, heads, rows, width // 2), (batch, heads, width // 32, rows), (batch, heads, rows)
    return held, scales, held, scales, each, each, (batch,), (batch,)


class CacheBank(nn.Module):
    """Named 4-bit banks of keys and values: ``register``, ``push``, ``attend``, ``evict``, ``trim``, ``bank[name]``."""

    def __init__(self):
        super().__init__()
        self.sizes = {}            # name -> k
        self.shapes = {}           # name -> (batch, heads, dim)
        self._bounds = {}          # name -> rows that the longest sequence has at most, as far as the host knows ...
        self._marks = {}           # name -> ... and the lengths that this was said of: (buffer, torch's count of writes to it, where it starts)
        self._pushed = {}          # name -> rows pushed to every sequence since slots may have stopped telling a row's age, or None: they tell it
        self._padded = {}          # name -> more rows of that time, of which counts on the device say how many there were
        self._captured = set()     # names whose lengths a graph may change behind the host's back
        self._mixed = set()        # names whose rows a graph may put into another order
        self._loaded = set()       # names whose rows came from elsewhere, in an order that the host has not seen
        self._views = {}           # name -> (buffers, mi_cache_t over them, how to pick them, where they start)

    def __getstate__(self):
        return {**self.__dict__, "_views": {}, "_marks": {}}

    def _load_from_state_dict(self, *args, **kwargs):
        super()._load_from_state_dict(*args, **kwargs)
        self._bounds, self._loaded = dict(self.sizes), set(self.sizes)
        for name in self.sizes:
            self._doubt(name)

    def register(self, name, dim, k, heads=1, batch=1, device=None):
        """An empty bank of ``k`` rows of ``dim`` values (a multiple of 8, at most 256) for each head of each sequence, on ``device``
        (the current HIP device where there is one: such banks are large, and of no use elsewhere)."""
        if device is None and torch.cuda.is_available():
            device = torch.device("cuda", torch.cuda.current_device())
        dim, k, heads, batch = int(dim), int(k), int(heads), int(batch)
        if dim < 8 or dim > 256 or dim % 8:
            raise ValueError(f"dim must be a multiple of 8 in [8, 256], got {dim}")
        if k < 1 or heads < 1 or batch < 1:
            raise ValueError(f"k, heads and batch must be positive, got k={k} heads={heads} batch={batch}")
        for part, dtype, shape in zip(_PARTS, _DTYPES, _part_shapes(k, batch, heads, dim)):
            self.register_buffer(f"{name}_{part}", torch.zeros(shape, dtype=dtype, device=device))
        self.sizes[name], self.shapes[name] = k, (batch, heads, dim)
        self._captured.discard(name)
        self._mixed.discard(name)
        self._loaded.discard(name)
        self._doubt(name)
        self._bound(name)
        self._bounds[name], self._pushed[name] = 0, None
        self._views.pop(name, None)

    # ------------------------------------------------------------------------------------------------------------ helpers
    def _cache(self, name, what):
        if name not in self.sizes:
            raise KeyError(f"CacheBank.{what}: no bank named {name!r}")
        known = self._views.get(name)
        if known is not None and all(map(operator.is_, known[0], known[2](self._buffers))) and known[3] == [*map(torch.Tensor.data_ptr, known[0])]:
            return known[1], known[0]
        pick = operator.itemgetter(*[f"{name}_{part}" for part in _PARTS])
        held = pick(self._buffers)
        if not held[0].is_cuda:
            raise RuntimeError(f"CacheBank.{what}: buffer is on {held[0].device}; image-classification_amd moves bank rows "
                               "with HIP kernels only (no CPU fallback) -- call .to(device) first")
        batch, heads, dim = self.shapes[name]
        for part, dtype, shape, t in zip(_PARTS, _DTYPES, _part_shapes(self.sizes[name], batch, heads, dim), held):
            if t.shape != shape:
                raise RuntimeError(f"CacheBank.{what}: buffer {name}_{part} is {tuple(t.shape)}, the bank was registered with {shape}")
            if t.dtype != dtype or not t.is_contiguous() or t.device != held[0].device:
                raise RuntimeError(f"CacheBank.{what}: buffer {name}_{part} must be contiguous {dtype} on {held[0].device}, "
                                   f"got {t.dtype} on {t.device} (move banks with .to(device), not to another dtype)")
        starts = [t.data_ptr() for t in held]
        view = ctypes.pointer(_lib.Cache(*starts, batch, heads, dim, held[4].shape[2], self.sizes[name]))
        if name in self._marks and self._marks[name][2] != starts[6]:
            del self._marks[name]
        self._bound(name)
        self._views[name] = (held, view, pick, starts)
        return view, held

    @staticmethod
    def _counts(counts, batch, T, device):
        if counts is None:
            return None
        if not isinstance(counts, torch.Tensor):
            if torch.cuda.is_current_stream_capturing():
                raise RuntimeError("CacheBank: a graph cannot capture counts from the host; give them as a tensor on the device")
            values = [int(n) for n in counts]
            if len(values) != batch or any(n < 0 or n > T for n in values):
                raise ValueError(f"counts must be {batch} numbers in [0, {T}], got {values}")
            return torch.tensor(values, dtype=torch.int32, device=device)
        if counts.dtype not in (torch.int32, torch.int64) or tuple(counts.shape) != (batch,) or counts.device != device:
            raise ValueError(f"counts must be {batch} int32 or int64 on {device}, got {counts.dtype} {tuple(counts.shape)} on {counts.device}")
        return (counts if counts.dtype == torch.int32 else counts.clamp(0, T).to(torch.int32)).contiguous()

    def _rows(self, what, name, t, arg, heads, device):
        batch, _, dim = self.shapes[name]
        if not isinstance(t, torch.Tensor) or not t.is_cuda:
            raise RuntimeError(f"{arg} must be a tensor on an MI355X (HIP) device: image-classification_amd has no CPU fallback")
        if t.device != device:
            raise RuntimeError(f"CacheBank.{what}: {arg} is on {t.device}, the bank on {device}")
        if t.dtype not in _CODES:
            raise ValueError(f"CacheBank.{what}: {arg} must be float32, bfloat16 or float16, got {t.dtype}")
        if t.dim() != 4 or t.shape[0] != batch or t.shape[3] != dim or (heads is not None and t.shape[1] != heads):
            raise ValueError(f"CacheBank.{what}: {arg} {tuple(t.shape)} does not fit a bank of {batch} sequences, {self.shapes[name][1]} heads, dim {dim} "
                             "(expected [batch, heads, rows, dim])")
        return t

    def _changes(self, name) -> bool:
        """Whether the call is being captured: from then on the host knows nothing about this bank's lengths."""
        if torch.cuda.is_current_stream_capturing():
            self._captured.add(name)
            return True
        return False

    def _bound(self, name, length=None) -> int:
        """The bound, where it still speaks of the lengths that the bank has; otherwise they may be anything up to ``k``."""
        length, mark = self._buffers[f"{name}_length"] if length is None else length, self._marks.get(name)
        if mark is None or mark[0] is not length or mark[1] != length._version:
            # (writes to an inference tensor are not counted: it has no mark that holds)
            self._marks[name] = (None, 0, 0) if length.is_inference() else (length, length._version, length.data_ptr())
            self._bounds[name] = self.sizes[name]
            if self._pushed[name] is None:
                self._loaded.add(name)
            self._doubt(name)
        return self._bounds[name]

    def _set_bound(self, name, bound):
        """A bound after a call, of the lengths that :meth:`_bound` was last asked for before it."""
        self._bounds[name] = self.sizes[name] if name in self._captured else min(bound, self.sizes[name])

    def _span(self, name) -> int:
        """About how many rows are in use: what launches are sized by."""
        return max(1, self.sizes[name] if name in self._captured else self._bounds[name])

    def _in_order(self, name, view, counts, T, device) -> bool:
        """Whether the last T rows of every sequence (or ``counts`` of them) are the rows pushed last, in their order: waits for the device."""
        order = torch.empty(1, dtype=torch.int32, device=device)
        _lib.check(_lib.lib().mi_cache_in_order(view, None if counts is None else counts.data_ptr(), T, order.data_ptr(),
                                                _lib.raw_stream(device.index)), "mi_cache_in_order")
        return bool(order)

    def _doubt(self, name):
        self._pushed[name] = self._padded[name] = 0

    def _told(self, name, capturing=False, given=False):
        """How many rows of the bank's end are in the order of their pushes: None for all, as far as the host knows.  ``given``: the rows
        asked for are counted on the device, as those of their push were."""
        pushed = self._pushed[name]
        if pushed is None and (capturing or name not in self._mixed):
            return None
        if name in self._captured and not capturing:       # a replay may have come between; a graph's own pushes come before its attention
            return 0
        return pushed + self._padded[name] if given else pushed

    def _check_order(self, name, view, counts, T, device, given):
        """Refuses causal attention of T rows where slots do not say which rows were pushed before which.  They do until rows are evicted,
        and the rows pushed since then do; a look at the device says the same of others."""
        if self._pushed[name] is None and name not in self._mixed:
            return
        capturing = torch.cuda.is_current_stream_capturing()
        told = self._told(name, capturing, given)
        if told is None or T <= told:
            return
        text = (f"CacheBank.attend: the last rows of bank {name!r} are not the rows pushed last, in their order, since an evict moved rows: causal "
                "attention of several rows comes after their push and before the next evict")
        if capturing:
            if name not in self._loaded:
                raise RuntimeError(text + " (a graph cannot look; a call outside of it, before, can)")
        elif self._in_order(name, view, None, T, device):
            self._pushed[name] = T
        elif counts is None or not self._in_order(name, view, counts, T, device):
            raise RuntimeError(text)

    # --------------------------------------------------------------------------------------------------------------- calls
    def push(self, name, key, value, counts=None, held=False):
        """Appends ``key`` and ``value`` [batch, heads, T, dim] behind the last row of every sequence, quantised to 4 bits.

        ``counts`` (one whole number for each sequence, a list, which the host waits to copy, or a tensor on the device): only the first
        ``counts[b]`` of the T rows of sequence b are real; the others are not stored.  ``held=True`` returns the values that the bank now
        holds for the two, in their type and [batch, heads, T, dim], zeros where nothing was stored (a float16 above 57344 is held as 65536,
        and returned as 65504).
        Raises ``RuntimeError`` before anything is written if a sequence would pass ``k`` rows."""
        view, held_by = self._cache(name, "push")
        device = held_by[0].device
        heads = self.shapes[name][1]
        key = self._rows("push", name, key, "key", heads, device).detach()
        value = self._rows("push", name, value, "value", heads, device).detach()
        if key.shape != value.shape or key.dtype != value.dtype:
            raise ValueError(f"CacheBank.push: key {tuple(key.shape)} {key.dtype} and value {tuple(value.shape)} {value.dtype} differ")
        T, k = key.shape[2], self.sizes[name]
        least = T if counts is None else 0              # rows that every sequence gets, for all the host knows
        if counts is not None and not isinstance(counts, torch.Tensor):
            counts = [int(n) for n in counts]
            least = min(counts, default=0)
        counts = self._counts(counts, key.shape[0], T, device)
        with _on(device):
            if not self._changes(name):
                bound = k if name in self._captured else self._bound(name, held_by[6])
                if bound + T > k:                       # waits for the device
                    longest = torch.empty(1, dtype=torch.int32, device=device)
                    _lib.check(_lib.lib().mi_cache_longest(view, None if counts is None else counts.data_ptr(), T, longest.data_ptr(),
                                                           _lib.raw_stream(device.index)), "mi_cache_longest")
                    longest = int(longest)
                    if longest > k:
                        raise RuntimeError(f"CacheBank.push: {longest} rows do not fit bank {name!r} of {k}; evict or trim first")
                    bound = longest - T
                self._set_bound(name, bound + T)
            else:
                self._set_bound(name, k)
            (key, key_strides), (value, value_strides) = _aligned(key), _aligned(value)
            out = tuple(torch.empty(key.shape, dtype=key.dtype, device=device) for _ in range(2)) if held else (None, None)
            _lib.check(_lib.lib().mi_cache_push(view, key.data_ptr(), _array(key_strides),
                                                value.data_ptr(), _array(value_strides), _CODES[key.dtype], T,
                                                None if counts is None else counts.data_ptr(), None if not held else out[0].data_ptr(),
                                                None if not held else out[1].data_ptr(), _lib.raw_stream(device.index)), "mi_cache_push")
            if self._pushed[name] is not None:
                self._pushed[name] += least
                self._padded[name] += T - least
        return out if held else None

    def attend(self, name, query, counts=None, scale=None, causal=True, accumulate=False):
        """Softmax attention of ``query`` [batch, heads * group, T, dim] over the bank, in the query's type and layout: query head h
        reads head ``h // group``.

        ``causal``: the query rows are the last rows of their sequence (push first, then attend), and row t does not see the rows after
        its own; otherwise every row sees the whole sequence.  An :meth:`evict` may put rows into other slots, which then do not say who came
        before whom: causal attention of more than one row has to come before it, and is refused after it until as many rows are pushed
        again, unless the last rows are still in their order (the host then waits for the device once, as it does for a state that was
        loaded).  ``counts``: as in :meth:`push`, real rows of each sequence (after an eviction, the counts of the push).  Rows that are
        not real or see nothing give zeros.  ``scale``: positive, ``dim ** -0.5`` if not given.  ``accumulate`` adds to :meth:`weights`
        what each row of the bank got, summed over query rows and the group's heads; :meth:`evict` goes by that.  What query rows that are
        trimmed later (a rejected draft) have added to other rows stays: attend to a draft without, and to what was accepted of it with
        ``accumulate``, where that matters.

        Sums and statistics are float32; probabilities enter the second product as bf16 pieces: three for a float32 query (2^-24 of each
        is left out), two for float16 and for up to 32 rows (T times the group) of bfloat16 (2^-17), one for more rows of bfloat16 (2^-8,
        half a step of that type)."""
        view, held_by = self._cache(name, "attend")
        device = held_by[0].device
        batch, heads, dim = self.shapes[name]
        query = self._rows("attend", name, query, "query", None, device)
        if query.shape[1] == 0 or query.shape[1] % heads:
            raise ValueError(f"CacheBank.attend: {query.shape[1]} query heads are no multiple of the bank's {heads}")
        if (torch.is_grad_enabled() and query.requires_grad) or (forward_ad._current_level >= 0 and forward_ad.unpack_dual(query).tangent is not None):
            raise RuntimeError("CacheBank.attend has no gradient: call it under torch.no_grad() or with query.detach()")
        scale = dim ** -0.5 if scale is None else float(scale)
        query = query.detach()
        T, group = query.shape[2], query.shape[1] // heads
        given = isinstance(counts, torch.Tensor)
        counts = self._counts(counts, batch, T, device)
        L = _lib.lib()
        with _on(device):
            query, query_strides = _aligned(query)
            out = torch.empty_like(query)
            if T == 0:
                return out
            if causal and T > 1:
                self._check_order(name, view, counts, T, device, given)
            step, out_strides = 16 // out.element_size(), _strides(out)
            if out.stride(3) != 1 or out_strides[0] % step or out_strides[1] % step or out_strides[2] % step:
                out = torch.empty(query.shape, dtype=query.dtype, device=device)
                out_strides = _strides(out)
            span = self._span(name)
            code = _CODES[query.dtype]
            nbytes = L.mi_cache_attend_workspace_bytes(view, code, T, group, span, int(causal), int(accumulate))
            ws = torch.empty(max(int(nbytes), 16), dtype=torch.uint8, device=device)
            _lib.check(L.mi_cache_attend(view, query.data_ptr(), _array(query_strides),
                                         out.data_ptr(), _array(out_strides), code, T, group,
                                         None if counts is None else counts.data_ptr(), scale, int(causal), int(accumulate), span,
                                         ws.data_ptr(), ws.numel(), _lib.raw_stream(device.index)), "mi_cache_attend")
        return out

    def evict(self, name, keep, recent=0, into=None):
        """Cuts every head of every sequence down to ``keep`` rows: those among the last ``recent`` pushed of the sequence stay, then those
        with the largest :meth:`weights`, ties to the lower slot.  Slots below ``keep`` whose row leaves take, in ascending order, the kept
        rows from above.  ``into``: the rows that stay go to that bank (same batch, heads, dim, at least ``keep`` rows; what it held is
        gone) and this one is left as it was."""
        view, held_by = self._cache(name, "evict")
        device = held_by[0].device
        target, keep, recent = name if into is None else into, int(keep), int(recent)
        if into == name:
            raise ValueError("CacheBank.evict: into must name another bank (leave it out to evict in place)")
        other = view if into is None else self._cache(into, "evict")[0]
        if into is not None and (self.shapes[into] != self.shapes[name] or self._buffers[f"{into}_key"].device != device):
            raise ValueError(f"CacheBank.evict: bank {into!r} {self.shapes[into]} does not match bank {name!r} {self.shapes[name]} (batch, heads, dim) on {device}")
        if keep < 1 or keep > self.sizes[target]:
            raise ValueError(f"CacheBank.evict: keep={keep} outside [1, {self.sizes[target]}]")
        if recent < 0 or recent > keep:
            raise ValueError(f"CacheBank.evict: recent={recent} outside [0, keep={keep}]")
        L = _lib.lib()
        with _on(device):
            captured, bound = self._changes(target), self._bound(name, held_by[6])
            if into is not None:
                self._bound(into)
            ws = torch.empty(int(L.mi_cache_evict_workspace_bytes(view, keep)), dtype=torch.uint8, device=device)
            span = self._span(name)
            _lib.check(L.mi_cache_evict(view, other, keep, recent, span, ws.data_ptr(), ws.numel(),
                                        _lib.raw_stream(device.index)), "mi_cache_evict")
        if name in self._captured:
            bound = self.sizes[name]
        self._set_bound(target, min(keep, bound))
        # rows moved, for all the host knows, unless there are no more than `keep`: then they are as they were
        moved, told, padded = bound > keep, self._told(name), self._padded[name]
        self._doubt(target)
        if not moved:
            self._pushed[target], self._padded[target] = told, padded if told else 0
        if moved or name not in self._loaded:
            self._loaded.discard(target)
        else:
            self._loaded.add(target)
        if captured and (moved or name in self._mixed):
            self._mixed.add(target)

    def trim(self, name, lengths=0):
        """Cuts every sequence to at most ``lengths`` rows (a number for all, or one for each sequence as a tensor on the device): 0 empties
        the bank, a smaller length takes back the rows pushed last (a rejected draft), by position, wherever an eviction has put them:
        freed slots below the new length take, in ascending order, the rows that stay from above.  Positions go on from the cut; weights
        stay as they are, with what the rows that leave had added to others as queries."""
        view, held_by = self._cache(name, "trim")
        device = held_by[0].device
        each, number = None, 0
        if isinstance(lengths, torch.Tensor):
            top = torch.iinfo(torch.int32).max
            each = self._counts(lengths, self.shapes[name][0], top, device)
        else:
            number = int(lengths)
            if number < 0:
                raise ValueError(f"CacheBank.trim: lengths must not be negative, got {number}")
            number = min(number, self.sizes[name])
        with _on(device):
            captured = self._changes(name)
            _lib.check(_lib.lib().mi_cache_trim(view, None if each is None else each.data_ptr(), number,
                                                _lib.raw_stream(device.index)), "mi_cache_trim")
        if each is None:
            self._set_bound(name, min(number, self._bound(name, held_by[6])))
        if self._pushed[name] is not None:
            self._doubt(name)
            if each is None and number == 0 and not captured:      # an empty bank is in order
                self._pushed[name] = None

    def __getitem__(self, name):
        """(keys, values) as the bank holds them, bfloat16 [batch, heads, k, dim] each (exact); rows not in use are zeros."""
        view, held_by = self._cache(name, "__getitem__")
        device = held_by[0].device
        batch, heads, dim = self.shapes[name]
        with _on(device):
            out = tuple(torch.empty((batch, heads, self.sizes[name], dim), dtype=torch.bfloat16, device=device) for _ in range(2))
            _lib.check(_lib.lib().mi_cache_read(view, out[0].data_ptr(), out[1].data_ptr(), _lib.raw_stream(device.index)), "mi_cache_read")
        return out

    def lengths(self, name):
        """Rows in use of each sequence: the bank's own int32 [batch] buffer (to read, not to write)."""
        return self._buffers[f"{name}_length"]

    def weights(self, name):
        """Attention that each row got since it was pushed, float32 [batch, heads, k]; slots from the length on hold nothing of meaning."""
        return self._buffers[f"{name}_weight"][..., :self.sizes[name]]

    def positions(self, name):
        """How many rows of its sequence were pushed before each row, int32 [batch, heads, k]; as for :meth:`weights`."""
        return self._buffers[f"{name}_position"][..., :self.sizes[name]]
