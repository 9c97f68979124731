"""What the host works out once per batch for the kernels that share work among its requests; every layer's calls take the same plan.

A plan belongs to one batch. Its arrays are on the device when the constructor returns, and no call changes them: calls on any stream, and
captured graphs, may share one. It may be dropped while calls are still on their way, on whatever stream; only a captured graph does not keep it
alive: as long as that is replayed, its plans have to be kept, as its other inputs."""
from __future__ import annotations

from typing import Sequence, Tuple

import numpy as np
import torch

#: query rows of a unit, and keys of a strip, of a shared prefix' own keys
OWN_ROWS, OWN_STRIP = 8, 16
#: workers of a CTA for own keys; what beginning and end of a unit take, in strips
OWN_WORKERS, OWN_BEGIN = 12, 2
#: weights of pick_shares, in microseconds: an SM's for a strip of own keys, a CTA's for 128 keys of a prefix under one and under two tiles of rows. Fitted to
#: whole calls at an earlier state of the kernel, both parts running at once; a tile by itself takes less now (see attention_shared.cu)
T_OWN, T_ONE, T_TWO = 0.17, 1.3, 2.9
#: of a sequence: the kernels count to the end of its last tile in 32 bits
MAX_KEYS = (1 << 31) - 129
#: of attention's scores: times log2(e) it has to be a number in 32 bits
MAX_SCALE = 2.0**127
#: rows of a tile of the adapter kernels, and of the tiles that go through one kernel
ADAPTER_ROWS, ADAPTER_FEW = 64, 16


def _host_ints(values, name: str) -> np.ndarray:
    if torch.is_tensor(values):
        values = values.detach().cpu().numpy()
    a = np.asarray(values if len(values) else np.zeros(0, dtype=np.int64))
    if a.ndim != 1 or a.dtype.kind not in "iu":
        raise ValueError(f"{name} must be a list of whole numbers")
    return a.astype(np.int64)


class _Plan:
    """Where a plan's arrays are."""

    #: device number (-1: not on a GPU), its memory, the stream that this belongs to, and the others that have calls with it
    index, _dev, _stream, _others = -1, None, 0, frozenset()

    def _place(self, flat: np.ndarray, device: torch.device) -> int:
        """The int32 values ``flat`` to the GPU ``device``; where they are."""
        self._dev = torch.from_numpy(flat).to(device)
        self.index = self._dev.get_device()
        self._stream = torch._C._cuda_getCurrentRawStream(self.index)
        return self._dev.data_ptr()

    def used_on(self, stream: int) -> None:
        """A call on the current stream of the plan's device, which has that number, reads the arrays: their memory is not given to anybody else
        ahead of its end."""
        if stream != self._stream and stream not in self._others:
            self._dev.record_stream(torch.cuda.current_stream(self.index))
            self._others = self._others | {stream}

    # (a plan holds addresses: a copy's would outlive the memory behind them, and another process has none)
    def __copy__(self):
        return self

    def __deepcopy__(self, memo):
        return self

    def __getstate__(self):
        if self._dev is not None:
            raise TypeError("a plan on a GPU belongs to its process: make another one from its lists")
        return self.__dict__


class AdapterPlan(_Plan):
    """Which rows go through which adapter. ``ids[t]``: the adapter of row t, negative for none. ``device``: where the calls run (host
    memory: only the restatement in torch does)."""

    def __init__(self, ids, n_adapters: int, device=None) -> None:
        a = _host_ints(ids, "ids")
        if a.size and int(a.max()) >= n_adapters:
            raise ValueError(f"row {int(a.argmax())} has adapter {int(a.max())}, there are {n_adapters}")
        if a.size >= 1 << 26:
            raise ValueError("at most 2^26 rows")
        self.ids, self.n_adapters, self.n_rows = np.where(a < 0, -1, a).astype(np.int32), int(n_adapters), int(a.size)
        #: rows sorted by adapter, those without one first
        order = np.argsort(self.ids, kind="stable").astype(np.int32)
        names, starts, counts = np.unique(self.ids[order], return_index=True, return_counts=True)
        bounds = [(name, start, start + count) for name, start, count in zip(names.tolist(), starts.tolist(), counts.tolist())]
        cut = lambda name, start, stop: [(name, p, min(ADAPTER_ROWS, stop - p), 0) for p in range(start, stop, ADAPTER_ROWS)]  # noqa: E731
        #: (adapter, first place in the order, rows, 0); rows without an adapter (they are copied) come last
        tiles = [t for b in bounds if b[0] >= 0 for t in cut(*b)]
        self.n_tiles = len(tiles)
        self.tile_rows = max((t[2] for t in tiles), default=0)
        tiles += [t for b in bounds if b[0] < 0 for t in cut(*b)]
        self.n_tiles_and_bare = len(tiles)
        self.tiles = tiles
        self.device = None if device is None else torch.device(device)
        #: device pointers
        self.tiles_ptr, self.rows_ptr = 0, 0
        if self.device is not None and self.device.type == "cuda":
            flat = np.asarray(tiles, dtype=np.int32).reshape(-1, 4)
            places = flat[:, 1:2] + np.minimum(np.arange(ADAPTER_ROWS, dtype=np.int32), flat[:, 2:3] - 1)      # (the last row again where a tile ends)
            self.tiles_ptr = self._place(np.concatenate([flat.reshape(-1), order[places].reshape(-1)]), self.device)
            self.rows_ptr = self.tiles_ptr + 16 * len(tiles)


class SharedPrefixPlan(_Plan):
    """A batch whose sequences share prefixes. ``new_tokens[i]`` query rows of sequence i (in this order in ``q``), behind ``keys[i]`` -
    ``new_tokens[i]`` earlier tokens; ``groups``: (first sequence, sequences, prefix) - the block tables of these neighbouring sequences
    begin with the same pages, for ``prefix`` tokens (a multiple of the block size, and none of the new ones). Sequences in no group share nothing."""

    def __init__(self, new_tokens, keys, groups: Sequence[Tuple[int, int, int]], n_q_heads: int, n_kv_heads: int, head_dim: int, block_size: int,
                 device=None) -> None:
        new, kv = _host_ints(new_tokens, "new_tokens"), _host_ints(keys, "keys")
        if new.shape != kv.shape:
            raise ValueError("new_tokens and keys are lists of the same sequences")
        if n_kv_heads < 1 or n_q_heads < 1 or n_q_heads % n_kv_heads or n_q_heads // n_kv_heads > 128:
            raise ValueError(f"{n_q_heads} query heads do not share {n_kv_heads} KV heads (up to 128 each)")
        if block_size not in (16, 32, 64, 128):
            raise ValueError("block_size must be 16, 32, 64 or 128")
        if (new < 0).any() or (new > kv).any() or kv.size and int(kv.max()) > MAX_KEYS:
            raise ValueError("a sequence has at least its new tokens as keys, and fewer than 2^31 - 128")
        self.n_q_heads, self.n_kv_heads, self.head_dim, self.block_size = n_q_heads, n_kv_heads, head_dim, block_size
        self.new_tokens, self.keys, self.groups = new, kv, [tuple(map(int, g)) for g in groups]
        self.n_seqs, self.rows = int(new.size), int(new.sum())
        if self.rows >= 1 << 24 or self.n_seqs > 65535:
            raise ValueError("at most 65535 sequences with 2^24 new tokens in all")
        prefix = np.zeros(new.size, dtype=np.int64)
        row0 = np.concatenate([[0], np.cumsum(new)])
        taken = np.zeros(new.size, dtype=bool)
        tile_tokens, tiles = 2 * (128 // (n_q_heads // n_kv_heads)), []
        for first, n, length in self.groups:
            if first < 0 or n < 1 or first + n > self.n_seqs or taken[first:first + n].any():
                raise ValueError(f"group ({first}, {n}, {length}): sequences that are there, and in no other group")
            if length < 0 or length % block_size or (length > kv[first:first + n] - new[first:first + n]).any():
                raise ValueError(f"group ({first}, {n}, {length}): a prefix is whole pages ahead of the new tokens of all its sequences")
            taken[first:first + n] = True
            prefix[first:first + n] = length
            if length:
                lo, hi = int(row0[first]), int(row0[first + n])
                tiles += [(first, r, min(tile_tokens, hi - r), length) for r in range(lo, hi, tile_tokens)]
        self.prefix = prefix
        #: pages that the longest sequence needs in its block table
        self.max_blocks = -(-int(kv.max()) // block_size) if kv.size else 0
        G = n_q_heads // n_kv_heads
        self.n_tiles = len(tiles)
        # units of own keys: (sequence, KV head, 8 query rows); all their strips of 16 keys in one line, cut into pieces of equal cost for the workers
        row_tiles = -(-new * G // OWN_ROWS)
        strips = np.where(new > 0, -(-(kv - prefix) // OWN_STRIP), 0)
        per_item = row_tiles * n_kv_heads
        unit0 = np.concatenate([[0], np.cumsum(per_item)])
        of_item = np.repeat(np.arange(new.size), per_item)                     # a unit's sequence
        ends = np.concatenate([[0], np.cumsum(strips[of_item])])               # strips ahead of a unit
        self.n_units, total = int(unit0[-1]), int(ends[-1])
        if total >= 1 << 31:
            raise ValueError("too many keys for one call")
        self.device = None if device is None else torch.device(device)
        on_gpu = self.device is not None and self.device.type == "cuda"
        sms = [torch.cuda.get_device_properties(self.device).multi_processor_count] if on_gpu else []
        # a unit costs its strips and a beginning and end that take as long as OWN_BEGIN more
        costs = np.concatenate([[0], np.cumsum(np.where(strips[of_item] > 0, strips[of_item] + OWN_BEGIN, 0))])
        self.p_splits, ctas = pick_shares(self.n_tiles * n_kv_heads, max((t[3] for t in tiles), default=0),
                                          any(t[2] > tile_tokens // 2 for t in tiles), int(costs[-1]), *sms)
        self.n_workers = W = min(ctas * OWN_WORKERS, -(-total // 2))
        cost = costs[-1] * np.arange(W + 1, dtype=np.int64) // max(W, 1)
        unit = np.searchsorted(costs, cost[:-1], side="right") - 1
        cuts = np.concatenate([ends[unit] + np.maximum(cost[:-1] - costs[unit] - OWN_BEGIN, 0), [total]])
        unit = np.searchsorted(ends, cuts[:-1], side="right") - 1
        workers = np.stack([of_item[unit], unit - unit0[of_item[unit]], cuts[:-1] - ends[unit], np.diff(cuts)], axis=1) if W else np.zeros((0, 4))
        units = np.stack([np.searchsorted(cuts, ends[:-1], side="right") - 1, np.searchsorted(cuts, ends[1:], side="left") - 1], axis=1)
        items = np.zeros((new.size, 8), dtype=np.int32)
        items[:, 0], items[:, 1], items[:, 2], items[:, 3] = np.arange(new.size), row0[:-1], new, kv
        items[:, 4], items[:, 5], items[:, 6] = prefix, unit0[:-1], row_tiles
        self.items, self.workers, self.units = items, workers.astype(np.int32), units.astype(np.int32)
        #: bytes of a call's scratch (0: the library has not been asked yet)
        self.workspace_bytes = 0
        if on_gpu:
            row_items = np.repeat(np.arange(new.size), new).astype(np.int32)
            parts = [np.asarray(tiles, dtype=np.int32), items, self.workers, self.units, row_items]       # all but the last start on 16-byte boundaries
            flat = [np.concatenate([p.reshape(-1), np.zeros(-p.size % 4, dtype=np.int32)]) for p in parts]
            at = self._place(np.concatenate(flat), self.device) + 4 * np.cumsum([0] + [f.size for f in flat])
            self.tiles_ptr, self.items_ptr, self.workers_ptr, self.units_ptr, self.rows_ptr = at[:5].tolist()


def pick_shares(units: int, prefix: int, two: bool, cost: int, sms: int = 148) -> Tuple[int, int]:
    """Parts of a prefix of that many tokens, ``units`` CTAs wide, and the CTAs for own keys of that cost in strips: both begin together, on SMs of
    their own, and the later end counts. Measured at eleven batches beside 12 to 90 other pairs each (a third to three times the parts, half to twice the
    CTAs): ten of them within 4% of the best pair, one 14% behind (36 units, prefix 10496, cost 1068: 33.3 us, and 29.2 with four parts for three); the
    worst pairs took up to 2.3 times as long."""
    tiles = -(-prefix // 128)
    if units == 0 or tiles == 0:
        return 1, sms
    parts, ctas = np.arange(1, min(64, tiles) + 1)[:, None], np.arange(1, sms)[None, :]
    ends = np.maximum(-(-units * parts // (sms - ctas)) * (5.0 + (T_TWO if two else T_ONE) * -(-tiles // parts)), 4.0 + T_OWN * cost / ctas)
    best = int((ends + 0.05 * parts).argmin())      # (a part more to join)
    return best // (sms - 1) + 1, best % (sms - 1) + 1
