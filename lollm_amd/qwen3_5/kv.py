"""Qwen3_5Cache -- the family cache, batched and device-resident, with O(1) rollback.

Keeps the method names of the reference cache (src/qwen3_5/kv.py:20-58:
append_kv / read_kv / linear_state / set_linear_state / advance / seen_tokens / clone
/ nbytes) so code written against that API keeps working, but the storage is laid out
for the MI355X kernels:

  * full-attention layers: preallocated K and V of shape (B, n_kv, max_len, head_dim)
    bf16, one contiguous slab per (sequence, KV head); `lengths` (B,) int32 on the
    device holds each sequence's committed length (the reference has one scalar
    `seen_tokens`, so it cannot hold ragged batches).
  * Gated DeltaNet layers: a conv-window buffer (B, 2W, conv_dim) bf16 with W = K-1+S
    rows per half, a recurrent-state buffer (B, 2, n_v, Dk, Dv) fp32 and a replay-record
    buffer (B, 2, n_v, S, 4 Dk + 16) bytes with S = 1 + k positions per half.
    `conv_off` (B,) int32 locates each sequence's committed conv state; `rec_half` and
    `replay` (B,) int32 say that its committed recurrent state is that half's state with
    the half's first `replay` records applied.  A forward reads the committed half and
    writes the other one (the kernel derives the halves on the device); a short forward
    (T <= S) writes the committed state plus one record per position instead of T
    states, so rolling back to `a` accepted drafts only rewrites four small integers per
    sequence (`lollm_spec_commit`) -- the reference instead deep-copies the whole cache
    before every verify (kv.py:49-54, mtp.py:141) and re-runs on reject (mtp.py:156-162).

Qwen3_5PagedCache holds the full-attention layers' keys and values in pages instead, in bf16
or in 8 bits: a sequence takes the pages it fills, and gives them back.

A forward over a tree of drafts writes its nodes' rows and records behind the committed ones and
commits nothing; keep_path moves the accepted path's to the front and sets the indices.
"""

from __future__ import annotations

import torch

from .. import ops
from .config import Qwen3_5Config


def capturing() -> bool:
    """Whether the current stream is recording a HIP graph (False without a device)."""
    return torch.cuda.is_available() and torch.cuda.is_current_stream_capturing()


class Qwen3_5Cache:
    def __init__(self, cfg: Qwen3_5Config, batch: int, max_len: int, spec_slots: int = 4,
                 device="cuda"):
        self.cfg = cfg
        self.batch, self.max_len, self.spec_slots = batch, max_len, spec_slots
        self.device = torch.device(device)
        n = cfg.num_hidden_layers
        self.layers = [None] * n
        K = cfg.linear_conv_kernel_dim
        for i in range(n):
            if cfg.layer_type(i) == "full_attention":
                self.layers[i] = self._kv_layer()
            else:
                self.layers[i] = {
                    "win": torch.zeros(batch, 2 * self.win_rows, cfg.conv_dim,
                                       dtype=torch.bfloat16, device=device),
                    "rec": torch.zeros(batch, 2, cfg.linear_num_value_heads,
                                       cfg.linear_key_head_dim, cfg.linear_value_head_dim,
                                       dtype=torch.float32, device=device),
                    "rep": torch.zeros(batch, 2, cfg.linear_num_value_heads, spec_slots,
                                       4 * cfg.linear_key_head_dim + 16, dtype=torch.uint8,
                                       device=device),
                }
        self.fresh = True                 # no GDN state yet (zero initial state)
        self.lengths = torch.zeros(batch, dtype=torch.int32, device=device)
        self.rec_half = torch.zeros(batch, dtype=torch.int32, device=device)
        self.replay = torch.zeros(batch, dtype=torch.int32, device=device)
        self.conv_off = torch.zeros(batch, dtype=torch.int32, device=device)
        self.last_T = 0
        self.tree_T = 0                   # nodes of a tree that the last forward wrote, uncommitted
        # host-side upper bound of max(lengths): every forward or speculative step adds
        # its T, rollbacks leave it, so capacity is checked without reading the device
        self.len_bound = 0

    def _kv_layer(self):
        cfg = self.cfg
        shape = (self.batch, cfg.num_key_value_heads, self.max_len, cfg.head_dim)
        return {"k": torch.zeros(shape, dtype=torch.bfloat16, device=self.device),
                "v": torch.zeros(shape, dtype=torch.bfloat16, device=self.device)}

    def kv_args(self, layer):
        """What GatedAttention.core takes beside the layer's "k" and "v"."""
        return {}

    @property
    def win_rows(self):
        return self.cfg.linear_conv_kernel_dim - 1 + self.spec_slots

    # -- capacity ----------------------------------------------------------------------
    def reserve(self, T: int):
        """Raise RuntimeError unless T more rows fit every sequence (lengths + T <=
        max_len) -- the kernels would otherwise drop the KV rows past the end.  Reads the
        device lengths (a host sync) only when the host-side bound says they may not fit."""
        if self.len_bound + T <= self.max_len:
            return
        if capturing():
            raise RuntimeError(f"KV cache capacity: {self.len_bound} + {T} rows may exceed "
                               f"max_len {self.max_len} (cannot check exactly under capture)")
        self._measure()
        if self.len_bound + T > self.max_len:
            raise RuntimeError(f"KV cache capacity exceeded: a sequence holds {self.len_bound} "
                               f"tokens, {T} more do not fit max_len {self.max_len}")

    def _measure(self):
        """Set the bound to what it bounds (a host sync)."""
        self.len_bound = self.longest(self.lengths)

    def longest(self, counts: torch.Tensor) -> int:
        """The largest of a count per sequence (a host sync)."""
        return int(counts.max()) if self.batch else 0

    def grew(self, T: int):
        """Record that a call may have added up to T tokens to every sequence."""
        self.len_bound += T
        self.tree_T = 0                   # (an earlier tree's rows are no longer behind the tokens)

    # -- bookkeeping used by the model's forward -------------------------------------
    def commit_all(self, T: int):
        """After a forward over T tokens: every token is committed (the reference's
        forward + advance(T), modeling_qwen3_5.py:97).  The forward wrote the other half
        of every GDN buffer: a short forward its T records, a long one its final state."""
        S, W, K = self.spec_slots, self.win_rows, self.cfg.linear_conv_kernel_dim
        self.fresh = False
        self.last_T = T
        full = K - 1 + T <= W
        self.rec_half.bitwise_xor_(1)
        self.replay.fill_(T if T <= S else 0)
        self.conv_off.copy_(torch.where(self.conv_off >= W, 0, W) + (T if full else 0))
        self.lengths.add_(T)
        self.grew(T)

    def rollback(self, n_accepted: torch.Tensor):
        """After commit_all(T) with T <= spec_slots: keep n_accepted[b] + 1 tokens."""
        T = self.last_T
        if T > self.spec_slots:
            raise RuntimeError("rollback needs the last forward to have written replay records")
        self.tree_T = 0
        a = n_accepted.to(torch.int32).clamp(0, T - 1)
        self.lengths.sub_(T - 1 - a)
        self.replay.sub_(T - 1 - a)
        self.conv_off.sub_(T - 1 - a)

    # -- a tree of drafts --------------------------------------------------------------
    def tree_begins(self, T: int):
        """Raise unless a forward over a tree of T nodes fits this cache."""
        if not 1 <= T <= min(self.spec_slots, ops.TREE_MAX):
            raise ValueError(f"a tree of {T} nodes needs a cache with spec_slots >= {T} (this one has "
                             f"{self.spec_slots}) and at most {ops.TREE_MAX} nodes")
        self.tree_T = 0

    def tree_written(self, T: int):
        """After a forward over a tree of T nodes, which commits nothing."""
        self.tree_T = T

    def keep_path(self, path: torch.Tensor, count: torch.Tensor):
        """Commit a path of the tree that the last forward wrote: nodes path[b, :count[b]], increasing,
        (B, P) and (B,) int32 as ops.tree_accept gives them, become the sequence's next tokens."""
        T = self.tree_T
        if not T:
            raise RuntimeError("keep_path follows a forward over a tree")
        W, K = self.win_rows, self.cfg.linear_conv_kernel_dim
        for i, s in enumerate(self.layers):
            if "rep" in s:
                ops.tree_keep_gdn(s["rep"], s["win"], self.rec_half, self.conv_off, path, count, T, K)
            else:
                ops.tree_keep_kv(s["k"], s["v"], self.lengths, path, count, T, self.kv_args(i).get("table"))
        n = count.clamp(0, min(T, path.shape[1]))
        self.fresh = False
        self.rec_half.bitwise_xor_(1)
        self.replay.copy_(n)
        self.conv_off.copy_(torch.where(self.conv_off >= W, 0, W) + n)
        self.lengths.add_(n)
        self.grew(min(T, path.shape[1]))
        self.last_T = self.spec_slots + 1   # (not a call that a rollback shortens)

    # -- the reference cache API (kv.py:26-58) ---------------------------------------
    def _uniform_length(self) -> int:
        L = self.lengths.cpu()
        if not bool((L == L[0]).all()):
            raise RuntimeError("sequences have different lengths; use .lengths")
        return int(L[0])

    @property
    def seen_tokens(self) -> int:
        return self._uniform_length()

    def advance(self, n):
        self.reserve(n)
        self.lengths.add_(n)
        self.grew(n)

    def append_kv(self, layer, k, v):
        """Write k, v (B, n_kv, t, D) at the current length; return the full (K, V)."""
        s = self.layers[layer]
        L = self._uniform_length()
        t = k.shape[2]
        if L + t > self.max_len:
            raise RuntimeError("KV cache capacity exceeded")
        if t:
            self.tree_T = 0               # (written over)
        s["k"][:, :, L:L + t] = k
        s["v"][:, :, L:L + t] = v
        return s["k"][:, :, :L + t], s["v"][:, :, :L + t]

    def read_kv(self, layer):
        s = self.layers[layer]
        if s is None or "k" not in s:
            return None
        L = self._uniform_length()
        return s["k"][:, :, :L], s["v"][:, :, :L]

    def linear_state(self, layer):
        """(conv_state (B, conv_dim, K-1), recurrent_state (B, n_v, Dk, Dv)) copies, or
        (None, None) before the first forward."""
        s = self.layers[layer]
        if s is None or "win" not in s or self.fresh:
            return None, None
        K = self.cfg.linear_conv_kernel_dim
        b = torch.arange(self.batch, device=self.device)
        rows = self.conv_off[:, None].long() + torch.arange(K - 1, device=self.device)[None]
        conv = s["win"][b[:, None], rows].transpose(1, 2).contiguous()
        rec = ops.gdn_state(s["rec"], self.rec_half, s["rep"], self.replay)
        return conv, rec

    def settle(self):
        """Fold every GDN layer's pending replay records into its state: each layer's
        committed state goes to the other half, which becomes the committed one with no
        records (the cache holds the same state afterwards)."""
        if self.fresh:
            return
        self.tree_T = 0
        for s in self.layers:
            if s is not None and "rec" in s:
                ops.gdn_state(s["rec"], self.rec_half, s["rep"], self.replay, to_other_half=True)
        self.rec_half.bitwise_xor_(1)
        self.replay.zero_()

    def set_linear_state(self, layer, conv, rec):
        s = self.layers[layer]
        K = self.cfg.linear_conv_kernel_dim
        b = torch.arange(self.batch, device=self.device)
        self.tree_T = 0
        self.settle()   # the other layers keep their states; this one's is replaced whole
        rows = self.conv_off[:, None].long() + torch.arange(K - 1, device=self.device)[None]
        s["win"][b[:, None], rows] = conv.transpose(1, 2).to(torch.bfloat16)
        s["rec"][b, self.rec_half.long()] = rec.float()
        self.fresh = False   # (a new cache's other layers hold zero states, as on a first call)

    def clone(self):
        new = Qwen3_5Cache.__new__(Qwen3_5Cache)
        new.__dict__.update(self.__dict__)
        new.layers = []
        for s in self.layers:
            if s is None:
                new.layers.append(None)
            else:
                new.layers.append({n: t.clone() for n, t in s.items()})
        for n in ("lengths", "rec_half", "replay", "conv_off"):
            setattr(new, n, getattr(self, n).clone())
        return new

    def nbytes(self):
        tot = 0
        for s in self.layers:
            if s is None:
                continue
            for t in s.values():
                tot += t.numel() * t.element_size()
        return tot


class Qwen3_5PagedCache(Qwen3_5Cache):
    """The same cache with the full-attention layers' keys and values in pages of `page` rows
    (16, 32, 64 or 128) that sequences take from one pool as they grow: `table` (batch,
    ceil(max_len / page)) int32 on the device names each sequence's pages, the same ones in every
    layer's pools "k", "v" (n_pages, n_kv, page, head_dim).  kv_dtype torch.float8_e4m3fn holds
    them in 8 bits with one power-of-two scale per page and KV head ("ks", "vs"; ops.attn_append):
    half the memory and half of what a long context's attention reads.

    n_pages: pages of the pool, by default enough for every sequence at max_len.  `reserve` hands
    them out on the host, before the forward or step that fills them (a captured step is replayed
    over the same table); `release` takes a finished sequence's back."""

    def __init__(self, cfg: Qwen3_5Config, batch: int, max_len: int, spec_slots: int = 4,
                 device="cuda", page: int = 64, kv_dtype=torch.bfloat16, n_pages=None):
        if page not in ops.PAGE_SIZES:
            raise ValueError(f"page must be one of {ops.PAGE_SIZES}, got {page}")
        if kv_dtype not in (torch.bfloat16, torch.float8_e4m3fn):
            raise TypeError(f"kv_dtype must be bfloat16 or float8_e4m3fn, got {kv_dtype}")
        self.page, self.kv_dtype = page, kv_dtype
        self.live = [True] * batch       # released sequences take no more
        width = -(-max_len // page)
        self.n_pages = batch * width if n_pages is None else n_pages
        if self.n_pages < 1:
            raise ValueError("n_pages must be positive")
        super().__init__(cfg, batch, max_len, spec_slots, device)
        self.table = torch.full((batch, width), -1, dtype=torch.int32, device=self.device)
        self._host_table = torch.full((batch, width), -1, dtype=torch.int32)
        self.free = list(range(self.n_pages - 1, -1, -1))
        self.held = [0] * batch          # pages of each sequence
        self._dead = torch.zeros(batch, dtype=torch.bool, device=self.device)   # not live

    def _kv_layer(self):
        cfg = self.cfg
        shape = (self.n_pages, cfg.num_key_value_heads, self.page, cfg.head_dim)
        kv = {n: torch.zeros(shape, dtype=self.kv_dtype, device=self.device) for n in ("k", "v")}
        if self.kv_dtype != torch.bfloat16:
            kv.update({n: torch.ones(shape[:2], dtype=torch.float32, device=self.device)
                       for n in ("ks", "vs")})
        return kv

    def kv_args(self, layer):
        s = self.layers[layer]
        return {"table": self.table, "k_scale": s.get("ks"), "v_scale": s.get("vs")}

    @property
    def len_bound(self):
        return max((n for n, live in zip(self._bounds, self.live) if live), default=0)

    @len_bound.setter
    def len_bound(self, n):
        self._bounds = [n] * self.batch      # of each sequence: lengths part as drafts are rejected

    def _measure(self):
        self._bounds = self.lengths.tolist()

    def longest(self, counts):
        return max((n for n, live in zip(counts.tolist(), self.live) if live), default=0)

    def grew(self, T: int):
        self._bounds = [n + T for n in self._bounds]
        self.tree_T = 0

    def reserve(self, T: int):
        """Raise RuntimeError unless T more rows fit max_len and the pool; name their pages.  Goes
        by the host-side bounds of the lengths, and by the lengths themselves (a host sync) only
        where the pool is short of that; sequences then give back the pages that they do not need for
        their rows and T more (an earlier call's, if it reserved more and they were not filled)."""
        super().reserve(T)
        if not all(self.live) and not capturing():
            self.lengths.masked_fill_(self._dead, 0)   # what calls since have added

        def needs():
            return [-(-(n + T) // self.page) if live else 0 for n, live in zip(self._bounds, self.live)]

        def missing(need):
            return sum(max(0, n - held) for n, held in zip(need, self.held))

        need = needs()
        if not missing(need):
            return
        if capturing():
            raise RuntimeError("pages cannot be handed out under capture: reserve() before it")
        if missing(need) > len(self.free):
            self._measure()
            need = needs()
            if sum(need) > self.n_pages:
                raise RuntimeError(f"KV page pool exhausted: {sum(need)} pages needed, the pool has {self.n_pages}")
            if missing(need) > len(self.free):
                for b, n in enumerate(need):   # (past the rows to come: rolled back, or never written)
                    self._take_back(b, n)
        for b, n in enumerate(need):
            while self.held[b] < n:
                self._host_table[b, self.held[b]] = self.free.pop()
                self.held[b] += 1
        self.table.copy_(self._host_table)

    def _take_back(self, b: int, keep: int):
        """Pages of sequence b from its `keep`-th on go back to the pool (the table follows)."""
        self.free += self._host_table[b, keep:max(keep, self.held[b])].tolist()
        self._host_table[b, keep:] = -1
        self.held[b] = min(self.held[b], keep)

    def release(self, b: int):
        """Give back the pages of a finished sequence: it holds no keys from now on, takes no more
        pages, and its rows of later calls mean nothing (take a decoder's tokens before).  What calls
        add to its length is cleared by the next reserve() and counts against no capacity."""
        if capturing():
            raise RuntimeError("release() under capture")
        self._take_back(b, 0)
        self.live[b] = False
        self._dead[b] = True
        self.lengths[b] = 0
        self.table.copy_(self._host_table)

    # -- the reference cache API -------------------------------------------------------
    def tree_begins(self, T: int):
        super().tree_begins(T)
        if self.kv_dtype != torch.bfloat16:
            raise ValueError("a tree of drafts takes bf16 pages: the rows of 8-bit pages share their page's scale and "
                             "cannot be moved alone")

    def _rows(self, L):
        if not all(self.live):
            raise RuntimeError("a released sequence has no rows")
        at = torch.arange(L, device=self.device)
        return self.table[:, at // self.page].long(), at % self.page

    def append_kv(self, layer, k, v):
        """Write k, v (B, n_kv, t, D) at the current length; return the full (K, V)."""
        s = self.layers[layer]
        if "ks" in s:
            raise RuntimeError("8-bit pages are written by ops.attn_append, which keeps their scales")
        L, t = self._uniform_length(), k.shape[2]
        if L + t > self.max_len:
            raise RuntimeError("KV cache capacity exceeded")
        if t:
            self.reserve(t)
            self.tree_T = 0
            page, slot = self._rows(L + t)
            s["k"][page[:, L:], :, slot[L:]] = k.transpose(1, 2).to(torch.bfloat16)
            s["v"][page[:, L:], :, slot[L:]] = v.transpose(1, 2).to(torch.bfloat16)
        return self._read(layer, L + t)

    def _read(self, layer, L):
        s = self.layers[layer]
        page, slot = self._rows(L)
        out = []
        for n, sn in (("k", "ks"), ("v", "vs")):
            if sn in s:
                x = s[n].view(torch.uint8)[page, :, slot].view(self.kv_dtype).float()
                x = (x * s[sn][page][..., None]).to(torch.bfloat16)   # exact
            else:
                x = s[n][page, :, slot]
            out.append(x.transpose(1, 2))
        return tuple(out)

    def read_kv(self, layer):
        s = self.layers[layer]
        if s is None or "k" not in s:
            return None
        return self._read(layer, self._uniform_length())

    def clone(self):
        new = super().clone()
        new.__class__ = Qwen3_5PagedCache
        for n in ("table", "_host_table", "_dead"):
            setattr(new, n, getattr(self, n).clone())
        for n in ("free", "held", "live", "_bounds"):
            setattr(new, n, list(getattr(self, n)))
        return new

    def nbytes(self):
        return super().nbytes() + self.table.numel() * self.table.element_size()
