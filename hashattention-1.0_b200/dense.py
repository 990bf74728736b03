"""Dense attention over the paged cache and what goes with it: trees of drafted tokens, their acceptance and commit, the
attention weight that cached tokens receive, and eviction by it. (The reference's decode attends the selected tokens only;
these have no counterpart there.)

One round of speculative decoding on a model's layers, drafts by the sparse step or any other drafter:

    mask = tree_mask(parents, tree_lens)                       # once for all layers
    ...                                                        # the drafts' K / V (and codes) are in the cache, seq_lens count them
    out, lse = ctx.tree_attention(q, mask, tree_lens)          # per layer
    got = tree_accept(draft, parents, target, tree_lens, cache.seq_lens)
    ctx.attention_mass(q, lse, mass, mask, tree_lens, rows=got.accepted)   # per layer, where eviction is wanted
    ctx.tree_commit(got.accepted, tree_lens, mass=mass)        # per layer
    cache.seq_lens.copy_(got.seq_lens)                         # once: the layers of a model may share the tensor

and where a cache has grown too long

    kept, mass, lens = ctx.cache_evict(mass, keep_tokens, init_budget, recent_budget)   # per layer
    cache.seq_lens.copy_(lens)

Nothing here synchronises with the host; problems the kernels find arrive in the context's status word.
"""
from __future__ import annotations

import ctypes
import math
import threading
from dataclasses import dataclass

import torch

from . import _lib
from .cache import GROUP, HEAD_DIM, PAGE, PagedHashKVCache
from .ops import _check, _raise_on, _stream_ptr, library_call

MAX_NODES = _lib.HA_MAX_TREE_NODES
MASK_WORDS = MAX_NODES // 32


def _cuda(t, name: str) -> None:
    if not isinstance(t, torch.Tensor):
        raise ValueError(f"{name} must be a tensor")
    if t.device.type != "cuda":
        raise ValueError(f"{name} must live on a CUDA device, got {t.device}")


def _tree_size(t: torch.Tensor, name: str):
    if t.dim() != 2 or t.shape[0] < 1 or not 1 <= t.shape[1] <= MAX_NODES:
        raise ValueError(f"{name} should be of size (batch, 1 .. {MAX_NODES}), but is {tuple(t.shape)}")
    return t.shape


def pack_nodes(bits: torch.Tensor) -> torch.Tensor:
    """Truth values ``[..., n <= 128]`` as the int32 words ``[..., 4]`` of node sets and tree masks (bit j of the row in
    word j // 32); any device."""
    n = bits.shape[-1]
    if bits.dtype != torch.bool or n > MAX_NODES:
        raise ValueError(f"bits must be boolean with at most {MAX_NODES} columns, got {bits.dtype} {tuple(bits.shape)}")
    full = torch.zeros(*bits.shape[:-1], MAX_NODES, dtype=torch.bool, device=bits.device)
    full[..., :n] = bits
    words = (full.view(*bits.shape[:-1], MASK_WORDS, 32).long() << torch.arange(32, device=bits.device)).sum(-1)
    return torch.where(words >= 2 ** 31, words - 2 ** 32, words).to(torch.int32)


def unpack_nodes(words: torch.Tensor, n: int = MAX_NODES) -> torch.Tensor:
    """The inverse of :func:`pack_nodes`: ``[..., 4]`` int32 words -> ``[..., n]`` truth values."""
    if words.dtype != torch.int32 or words.shape[-1] != MASK_WORDS:
        raise ValueError(f"words must be int32 with {MASK_WORDS} columns, got {words.dtype} {tuple(words.shape)}")
    bits = (words[..., None] >> torch.arange(32, dtype=torch.int32, device=words.device)) & 1
    return bits.flatten(-2)[..., :n].bool()


def _status_ptr(status, device):
    if status is None:
        return None
    _check(status, "status", torch.int32, (1,), device)
    return status.data_ptr()


def tree_mask(parents: torch.Tensor, tree_lens: torch.Tensor | None = None, out: torch.Tensor | None = None,
              status: torch.Tensor | None = None) -> torch.Tensor:
    """``ha_tree_mask``: ``parents [B, T]`` int32 (-1: a root; a parent comes before its children) -> mask words
    ``[B, T, 4]`` int32 in which a node sees its ancestors and itself. ``status``: the int32 word that problems are
    reported in (a context's, say); without one they go unseen."""
    _cuda(parents, "parents")
    B, T = _tree_size(parents, "parents")
    dev = parents.device
    _check(parents, "parents", torch.int32, (B, T), dev)
    if tree_lens is not None:
        _check(tree_lens, "tree_lens", torch.int32, (B,), dev)
    if out is None:
        out = torch.empty(B, T, MASK_WORDS, dtype=torch.int32, device=dev)
    else:
        _check(out, "out", torch.int32, (B, T, MASK_WORDS), dev)
    status_ptr = _status_ptr(status, dev)
    with library_call(dev, "ha_tree_mask"):
        rc = _lib.load().ha_tree_mask(parents.data_ptr(), tree_lens.data_ptr() if tree_lens is not None else None, B, T,
                                      out.data_ptr(), status_ptr, _stream_ptr(dev))
    _raise_on(rc, "ha_tree_mask")
    return out


@dataclass(frozen=True)
class TreeAccept:
    """The accepted path of every sequence: its nodes as words ``[B, 4]`` int32, their number ``[B]`` int32, the token behind
    the last one ``[B]`` int64 (left as it was where a sequence has no drafts; 0 in a new one), and the sequence's length once
    the path is committed ``[B]`` int32."""

    accepted: torch.Tensor
    count: torch.Tensor
    next_token: torch.Tensor
    seq_lens: torch.Tensor

    @staticmethod
    def empty(batch: int, device) -> "TreeAccept":
        count = torch.empty(batch, dtype=torch.int32, device=device)  # (sizes as numbers: a tuple costs 1 us more)
        return TreeAccept(torch.empty(batch, MASK_WORDS, dtype=torch.int32, device=device), count,
                          torch.zeros(batch, dtype=torch.int64, device=device), torch.empty_like(count))


def tree_accept(draft: torch.Tensor, parents: torch.Tensor, target: torch.Tensor, tree_lens: torch.Tensor | None,
                seq_lens: torch.Tensor, out: TreeAccept | None = None, status: torch.Tensor | None = None) -> TreeAccept:
    """``ha_tree_accept``: greedy acceptance. ``draft [B, T]`` int64 tokens of the nodes (node 0's is certain),
    ``target [B, T]`` int64 the token the model puts behind each node, ``seq_lens [B]`` with the drafts counted."""
    _cuda(draft, "draft")
    B, T = _tree_size(draft, "draft")
    dev = draft.device
    _check(draft, "draft", torch.int64, (B, T), dev)
    _check(parents, "parents", torch.int32, (B, T), dev)
    _check(target, "target", torch.int64, (B, T), dev)
    if tree_lens is not None:
        _check(tree_lens, "tree_lens", torch.int32, (B,), dev)
    _check(seq_lens, "seq_lens", torch.int32, (B,), dev)
    if out is None:
        out = TreeAccept.empty(B, dev)
    else:
        _check(out.accepted, "accepted", torch.int32, (B, MASK_WORDS), dev)
        _check(out.count, "count", torch.int32, (B,), dev)
        _check(out.next_token, "next_token", torch.int64, (B,), dev)
        _check(out.seq_lens, "out.seq_lens", torch.int32, (B,), dev)
        if out.seq_lens.data_ptr() == seq_lens.data_ptr():
            raise ValueError("out.seq_lens must be another tensor than seq_lens, which the commits still need")
    status_ptr = _status_ptr(status, dev)
    with library_call(dev, "ha_tree_accept"):
        rc = _lib.load().ha_tree_accept(draft.data_ptr(), parents.data_ptr(), target.data_ptr(),
                                        tree_lens.data_ptr() if tree_lens is not None else None, seq_lens.data_ptr(), B, T,
                                        out.accepted.data_ptr(), out.count.data_ptr(), out.next_token.data_ptr(),
                                        out.seq_lens.data_ptr(), status_ptr, _stream_ptr(dev))
    _raise_on(rc, "ha_tree_accept")
    return out


class DenseDecodeContext:
    """Dense attention over one layer's paged cache for up to ``max_nodes`` new tokens per sequence (a tree of drafts; one
    token: the dense decode step), with its workspace. Creating it allocates; the calls do not, but for outputs that the
    caller leaves out. One context per call that may run at the same time; contexts whose calls follow one another on a stream
    (the layers of a model) may share the workspaces of the first of them (``workspace_of``). Python threads may enqueue through
    one context, or through contexts that share workspaces: their calls take turns, on a stream that they have to share too."""

    def __init__(self, cache: PagedHashKVCache, max_nodes: int = 1, sm_scale: float | None = None,
                 workspace_of: "DenseDecodeContext | None" = None):
        if cache.device.type != "cuda":
            raise ValueError("the cache must live on a CUDA device")
        if not 1 <= max_nodes <= MAX_NODES:
            raise ValueError(f"max_nodes must be in 1 .. {MAX_NODES}, got {max_nodes}")
        self.lib = _lib.load()
        self.cache = cache
        self.device = cache.k_pages.device  # (with its index)
        self.max_nodes = int(max_nodes)
        self.batch, self.num_kv_heads = cache.batch, cache.num_kv_heads
        self.num_q_heads = cache.num_kv_heads * GROUP
        self.sm_scale = 1.0 / math.sqrt(HEAD_DIM) if sm_scale is None else float(sm_scale)
        if not (self.sm_scale > 0.0 and math.isfinite(self.sm_scale)):
            raise ValueError("sm_scale must be positive")
        self.shape = _lib.HaShape(self.batch, self.num_kv_heads, GROUP, HEAD_DIM, PAGE, cache.max_pages, cache.num_pages, 1)
        self._shape_ref = ctypes.byref(self.shape)
        self._c_tree, self._c_strides = _lib.HaTree(), (ctypes.c_int64 * 3)()  # (filled in by each call)
        self.workspace_bytes = int(self.lib.ha_tree_workspace_bytes(self.max_nodes))
        self.evict_workspace_bytes = int(self.lib.ha_evict_workspace_bytes(self.shape))
        if self.evict_workspace_bytes == 0:
            raise ValueError("invalid shape for the CUDA library")
        if workspace_of is None:
            self.workspace = torch.empty(self.workspace_bytes, dtype=torch.uint8, device=self.device)
            self.evict_workspace = torch.empty(self.evict_workspace_bytes, dtype=torch.uint8, device=self.device)
        else:
            o = workspace_of
            if o.device != self.device or o.workspace_bytes < self.workspace_bytes or o.evict_workspace_bytes < self.evict_workspace_bytes:
                raise ValueError("workspace_of must be a context on the same device with workspaces at least as large")
            self.workspace, self.evict_workspace = o.workspace, o.evict_workspace
        # A call fills in the context's structs and launches two kernels that meet in the workspace, while the interpreter runs
        # other threads: whole calls take turns.
        self._turn = threading.Lock() if workspace_of is None else workspace_of._turn
        self.status = torch.zeros(1, dtype=torch.int32, device=self.device)
        # (the context's own buffers, which stay where they are as long as it lives)
        self._workspace_ptr, self._evict_workspace_ptr, self._status_ptr = (
            t.data_ptr() for t in (self.workspace, self.evict_workspace, self.status))

    @property
    def mass_shape(self):
        """Shape of the received weights: one number per sequence, kv-head and cached token."""
        return (self.batch, self.num_kv_heads, self.cache.max_pages * PAGE)

    def new_mass(self) -> torch.Tensor:
        return torch.zeros(self.mass_shape, dtype=torch.float32, device=self.device)

    def check_status(self) -> None:
        """Reads the device status word (synchronises) and raises if a kernel reported a problem."""
        code = int(self.status.item())
        if code != 0:
            self.status.zero_()
            raise RuntimeError(f"device status: {_lib.status_str(code)} (status {code})")

    # -- argument checks -----------------------------------------------------------------------------------------------
    def _tree(self, q, tree_mask, tree_lens):
        """Checks q [B, T, Hq, 128] (strided views allowed) and the tree's arrays -> (T, struct, strides)."""
        B, Hq = self.batch, self.num_q_heads
        if not isinstance(q, torch.Tensor) or q.dim() != 4 or q.shape[0] != B or q.shape[2:] != (Hq, HEAD_DIM) or \
                not 1 <= q.shape[1] <= self.max_nodes:
            raise ValueError(f"q should be of size ({B}, 1 .. {self.max_nodes}, {Hq}, {HEAD_DIM}), but is "
                             f"{tuple(q.shape) if isinstance(q, torch.Tensor) else type(q)}")
        if q.dtype != torch.bfloat16:
            raise ValueError(f"q must be torch.bfloat16, got {q.dtype}")
        if q.device != self.device:
            raise ValueError(f"q must live on {self.device}, got {q.device}")
        T = q.shape[1]
        batch, node, head, one = q.stride()
        batch, node = (0 if B == 1 else batch), (0 if T == 1 else node)  # (of a single one the stride means nothing)
        if one != 1 or (batch | node | head) % 8 or q.data_ptr() % 16:
            raise ValueError("q's rows of 128 must be contiguous and start on 16-byte boundaries")
        strides = self._c_strides
        strides[0], strides[1], strides[2] = batch, node, head
        return T, self._tree_struct(T, tree_mask, tree_lens), strides

    def _tree_struct(self, T, tree_mask, tree_lens):
        tree = self._c_tree
        tree.max_nodes, tree.tree_lens, tree.tree_mask = T, None, None
        if tree_mask is not None:
            _check(tree_mask, "tree_mask", torch.int32, (self.batch, T, MASK_WORDS), self.device)
            tree.tree_mask = tree_mask.data_ptr()
        if tree_lens is not None:
            _check(tree_lens, "tree_lens", torch.int32, (self.batch,), self.device)
            tree.tree_lens = tree_lens.data_ptr()
        return tree

    def _check_mass(self, mass, name="mass"):
        _check(mass, name, torch.float32, self.mass_shape, self.device)

    # -- operators -----------------------------------------------------------------------------------------------------
    def tree_attention(self, q, tree_mask=None, tree_lens=None, out: torch.Tensor | None = None,
                       lse: torch.Tensor | None = None):
        """``ha_tree_attention``: attention of ``q [B, T, Hq, 128]`` (a strided view will do) over the prefix and what
        ``tree_mask`` lets each node see (``None``: a chain). ``tree_lens [B]``: drafted tokens of each sequence, the
        last ones of ``cache.seq_lens`` (``None``: T of each); rows behind them are left as they were (zeros, where the
        outputs are not given). Returns ``out [B, T, Hq, 128]`` bf16 and ``lse [B, T, Hq]`` f32 (natural logarithm)."""
        with self._turn:
            T, tree, strides = self._tree(q, tree_mask, tree_lens)
            make = torch.zeros if tree_lens is not None else torch.empty
            size = (self.batch, T, self.num_q_heads)
            if out is None:
                out = make(*size, HEAD_DIM, dtype=torch.bfloat16, device=self.device)
            else:
                _check(out, "out", torch.bfloat16, (*size, HEAD_DIM), self.device)
            q_ptr, out_ptr = q.data_ptr(), out.data_ptr()
            if q_ptr == out_ptr:
                raise ValueError("out must be another tensor than q, which is read until the last row is written")
            if lse is None:
                lse = make(*size, dtype=torch.float32, device=self.device)
            else:
                _check(lse, "lse", torch.float32, size, self.device)
            c = self.cache
            with library_call(self.device, "ha_tree_attention"):
                rc = self.lib.ha_tree_attention(
                    self._shape_ref, tree, q_ptr, strides, c.k_pages.data_ptr(), c.v_pages.data_ptr(), c.page_table.data_ptr(),
                    c.seq_lens.data_ptr(), self.sm_scale, out_ptr, lse.data_ptr(), self._workspace_ptr,
                    self.workspace_bytes, self._status_ptr, _stream_ptr(self.device))
        _raise_on(rc, "ha_tree_attention")
        return out, lse

    def attention_mass(self, q, lse, mass, tree_mask=None, tree_lens=None, rows: torch.Tensor | None = None) -> torch.Tensor:
        """``ha_attention_mass``: adds to ``mass`` (:attr:`mass_shape`, f32) the attention weight each cached token has in
        the rows of ``q``, given the ``lse`` that :meth:`tree_attention` returned for them. ``rows [B, 4]`` int32: the
        nodes whose weights count (``TreeAccept.accepted``; ``None``: all)."""
        with self._turn:
            T, tree, strides = self._tree(q, tree_mask, tree_lens)
            _check(lse, "lse", torch.float32, (self.batch, T, self.num_q_heads), self.device)
            self._check_mass(mass)
            if rows is not None:
                _check(rows, "rows", torch.int32, (self.batch, MASK_WORDS), self.device)
            c = self.cache
            with library_call(self.device, "ha_attention_mass"):
                rc = self.lib.ha_attention_mass(
                    self._shape_ref, tree, q.data_ptr(), strides, lse.data_ptr(), rows.data_ptr() if rows is not None else None,
                    c.k_pages.data_ptr(), c.page_table.data_ptr(), c.seq_lens.data_ptr(), self.sm_scale, mass.data_ptr(),
                    self._status_ptr, _stream_ptr(self.device))
        _raise_on(rc, "ha_attention_mass")
        return mass

    def tree_commit(self, accepted, tree_lens=None, mass: torch.Tensor | None = None, max_nodes: int | None = None) -> None:
        """``ha_tree_commit``: moves the rows of the ``accepted [B, 4]`` nodes (K, V, codes, and ``mass``) to the front of
        the drafts. ``cache.seq_lens`` still counts all drafts and is left alone: copy ``TreeAccept.seq_lens`` into it when
        every layer has been committed. ``tree_lens`` as in :meth:`tree_attention`; where it is ``None``, ``max_nodes`` says how
        many drafts each sequence has (the ``T`` of the round's other calls, which nothing given here tells; a context for one
        node knows)."""
        _check(accepted, "accepted", torch.int32, (self.batch, MASK_WORDS), self.device)
        if max_nodes is None:
            if tree_lens is None and self.max_nodes > 1:
                raise ValueError("tree_commit needs tree_lens, or max_nodes = the drafts of each sequence in this round")
            max_nodes = self.max_nodes
        elif not 1 <= max_nodes <= self.max_nodes:
            raise ValueError(f"max_nodes must be in 1 .. {self.max_nodes}, got {max_nodes}")
        with self._turn:
            tree = self._tree_struct(int(max_nodes), None, tree_lens)
            if mass is not None:
                self._check_mass(mass)
            c = self.cache
            with library_call(self.device, "ha_tree_commit"):
                rc = self.lib.ha_tree_commit(
                    self._shape_ref, tree, accepted.data_ptr(), c.k_pages.data_ptr(), c.v_pages.data_ptr(), c.hash_pages.data_ptr(),
                    c.page_table.data_ptr(), c.seq_lens.data_ptr(), mass.data_ptr() if mass is not None else None,
                    self._status_ptr, _stream_ptr(self.device))
        _raise_on(rc, "ha_tree_commit")

    def cache_evict(self, mass, keep_tokens: int, init_budget: int = 128, recent_budget: int = 128,
                    kept: torch.Tensor | None = None, mass_out: torch.Tensor | None = None,
                    lens_out: torch.Tensor | None = None):
        """``ha_cache_evict``: cuts every sequence longer than ``keep_tokens`` to that many: the first ``init_budget``, the
        last ``recent_budget`` and the heaviest of the others by ``mass``, per kv-head and in their order; K, V and code rows
        move in place. Returns ``kept [B, Hkv, keep_tokens]`` int32 (former token numbers; -1 behind a shorter sequence's end,
        or as it was where given), the kept tokens' mass (zeros behind) and the new lengths ``[B]``, which the caller copies into
        ``cache.seq_lens`` when every layer that shares it has been cut. Rotary positions go on from the former length."""
        self._check_mass(mass)
        keep_tokens, init_budget, recent_budget = int(keep_tokens), int(init_budget), int(recent_budget)
        if keep_tokens < 1 or init_budget < 0 or recent_budget < 0 or init_budget + recent_budget > keep_tokens:
            raise ValueError(f"keep_tokens={keep_tokens} must cover init_budget={init_budget} and recent_budget={recent_budget}")
        if kept is None:
            kept = torch.full((self.batch, self.num_kv_heads, keep_tokens), -1, dtype=torch.int32, device=self.device)
        _check(kept, "kept", torch.int32, (self.batch, self.num_kv_heads, keep_tokens), self.device)
        mass_out = torch.empty_like(mass) if mass_out is None else mass_out
        self._check_mass(mass_out, "mass_out")
        c = self.cache
        lens_out = torch.empty_like(c.seq_lens) if lens_out is None else lens_out
        _check(lens_out, "lens_out", torch.int32, (self.batch,), self.device)
        if mass_out.data_ptr() == mass.data_ptr() or lens_out.data_ptr() == c.seq_lens.data_ptr():
            raise ValueError("mass_out and lens_out must be other tensors than mass and cache.seq_lens")
        with self._turn, library_call(self.device, "ha_cache_evict"):
            rc = self.lib.ha_cache_evict(
                self._shape_ref, keep_tokens, init_budget, recent_budget, mass.data_ptr(), c.k_pages.data_ptr(), c.v_pages.data_ptr(),
                c.hash_pages.data_ptr(), c.page_table.data_ptr(), c.seq_lens.data_ptr(), kept.data_ptr(), mass_out.data_ptr(),
                lens_out.data_ptr(), self._evict_workspace_ptr, self.evict_workspace_bytes, self._status_ptr,
                _stream_ptr(self.device))
        _raise_on(rc, "ha_cache_evict")
        return kept, mass_out, lens_out
