"""A Llama-3.1-architecture decoder with HashAttention on every layer, tensor-parallel over the GPUs of
one node: the host model of the full-model configuration (32 layers, hidden 4096, 32 query / 8 kv
heads of 128, SwiGLU FFN 14336, vocabulary 128256, RoPE theta 500000, random bf16 weights).

Parallel layout, as the reference's gpt-fast host shards it (efficiency/tp.py:48-98): the q / k / v
projections and w1 / w3 are split by columns (a rank owns whole heads: ``Hq / N`` query heads and
``Hkv / N`` kv-heads), wo and w2 by rows, and the partial results of wo and w2 are summed over the
ranks with an all-reduce after attention and after the MLP (efficiency/tp.py:104-134); embedding and
output head are replicated. One process per GPU; the all-reduce is the NCCL collective of
``torch.distributed`` (gloo in the CPU test) - a plain library call, the hot path stays inside a rank.

Attention: the prompt is prefilled with dense causal attention (``scaled_dot_product_attention``, a
library call), its keys / values go into this rank's paged cache and the key hashes are built once
(``ha_hash_prefill``); every decode step is one ``ha_decode_step`` per layer on the rank's
``Hkv / N`` kv-heads. Trees of drafted tokens are verified with dense attention over the same cache, and a cache
that has grown too long is cut by the attention weight its tokens received (:meth:`TPLlama.enable_trees`,
:meth:`TPLlama.verify_tree`, :meth:`TPLlama.evict`). A kv-head's keys, hash codes, hash MLPs and query heads live on one rank, so the
sparse-decode path itself needs no communication (SparseDecodeContext per layer).

Weights are drawn per block of 1/8 of every sharded dimension from seeds that depend on (layer,
matrix, block) only, so every rank count holds the same model.
"""
from __future__ import annotations

import zlib
from dataclasses import dataclass

import torch
import torch.distributed as dist
import torch.nn.functional as F

from . import _lib
from .cache import PAGE, PagedHashKVCache
from .dense import DenseDecodeContext, TreeAccept, tree_accept, tree_mask, unpack_nodes
from .ops import Budget, SparseDecodeContext, _check, rope_split
from .synthetic import make_usa

BLOCKS = 8  # the finest partition of a sharded dimension (one kv-head's worth of every matrix)


@dataclass
class LlamaTPConfig:
    n_layers: int = 32
    dim: int = 4096
    n_heads: int = 32
    n_kv_heads: int = 8
    head_dim: int = 128
    ffn_dim: int = 14336
    vocab_size: int = 128256
    rope_theta: float = 500000.0
    norm_eps: float = 1e-5
    init_budget: int = 128
    heavy_budget: float = 1.0 / 32
    recent_budget: int = 128
    max_seq_len: int = 32768 + 256


def block_range(world: int, rank: int) -> range:
    """The 1/8 blocks of every sharded dimension that ``rank`` of ``world`` owns (contiguous, rank order)."""
    if BLOCKS % world != 0 or not 0 <= rank < world:
        raise ValueError(f"{BLOCKS} blocks cannot be dealt to rank {rank} of {world}")
    per = BLOCKS // world
    return range(rank * per, (rank + 1) * per)


def _seed(*key) -> int:
    """A seed that depends on the key alone (not on the process, as Python's hash of a string would)."""
    return zlib.crc32(repr(key).encode()) & 0x7FFFFFFF


def _draw(shape, seed: int, device, dtype, std: float = 0.02) -> torch.Tensor:
    """N(0, std) values from the generator of the tensor's own device (billions of values are drawn where they
    live; CPU and GPU generators give different, equally seeded, streams)."""
    device = torch.device(device)
    g = torch.Generator(device=device).manual_seed(seed)
    return (torch.randn(shape, generator=g, device=device) * std).to(dtype)


def sharded_weight(name: str, layer: int, rows: int, cols: int, split: str, blocks, device, seed: int,
                   dtype=torch.bfloat16) -> torch.Tensor:
    """Rows x cols matrix ([out, in], as nn.Linear stores it) restricted to ``blocks`` of its output rows
    (``split == 'col'``: column-parallel in the usual naming, the outputs are divided) or of its input columns
    (``split == 'row'``). Block j is drawn from a seed of (seed, layer, name, j) alone."""
    parts = []
    for j in blocks:
        s = _seed(seed, layer, name, j)
        if split == "col":
            parts.append(_draw((rows // BLOCKS, cols), s, device, dtype))
        else:
            parts.append(_draw((rows, cols // BLOCKS), s, device, dtype))
    return torch.cat(parts, dim=0 if split == "col" else 1).contiguous()


def rms_norm(x: torch.Tensor, w: torch.Tensor, eps: float) -> torch.Tensor:
    return F.rms_norm(x, (x.shape[-1],), w, eps)


def rope(x: torch.Tensor, pos: torch.Tensor, theta: float) -> torch.Tensor:
    """x [..., T, H, D] rotated (rotate-half convention) for positions pos [T] (or broadcastable)."""
    d = x.shape[-1]
    inv = 1.0 / (theta ** (torch.arange(0, d, 2, dtype=torch.float32, device=x.device) / d))
    ang = pos.to(torch.float32)[..., None] * inv  # [T, D/2]
    cos = torch.cat([ang.cos(), ang.cos()], -1)[..., None, :]
    sin = torch.cat([ang.sin(), ang.sin()], -1)[..., None, :]
    xf = x.float()
    rot = torch.cat([-xf[..., d // 2:], xf[..., : d // 2]], -1)
    return (xf * cos + rot * sin).to(x.dtype)


class Layer:
    def __init__(self, cfg: LlamaTPConfig, idx: int, blocks, device, seed: int, dtype):
        kv_rows = cfg.n_kv_heads * cfg.head_dim
        mk = lambda name, r, c, split: sharded_weight(name, idx, r, c, split, blocks, device, seed, dtype)  # noqa: E731
        # one fused projection per rank: [local q heads | local k heads | local v heads] x dim
        self.wqkv = torch.cat([mk("wq", cfg.n_heads * cfg.head_dim, cfg.dim, "col"), mk("wk", kv_rows, cfg.dim, "col"),
                               mk("wv", kv_rows, cfg.dim, "col")], dim=0).contiguous()
        self.wo = mk("wo", cfg.dim, cfg.n_heads * cfg.head_dim, "row")
        self.w13 = torch.cat([mk("w1", cfg.ffn_dim, cfg.dim, "col"), mk("w3", cfg.ffn_dim, cfg.dim, "col")], dim=0).contiguous()
        self.w2 = mk("w2", cfg.dim, cfg.ffn_dim, "row")
        self.norm1 = torch.ones(cfg.dim, dtype=dtype, device=device)
        self.norm2 = torch.ones(cfg.dim, dtype=dtype, device=device)


class TPLlama:
    """One rank's share of the model. ``attention``: 'cuda' (the library's decode step on a paged cache) or a
    callable ``f(layer, q [B,Hq_l,D], k_all [B,Hkv_l,S,D], v_all) -> [B,Hq_l,D]`` used by CPU tests, in which
    case the keys / values are kept as plain tensors."""

    def __init__(self, cfg: LlamaTPConfig, world: int, rank: int, device, batch: int, seed: int = 0, group=None,
                 attention="cuda", dtype=torch.bfloat16):
        self.cfg, self.world, self.rank, self.device, self.group, self.batch = cfg, world, rank, torch.device(device), group, batch
        blocks = block_range(world, rank)
        self.hq = cfg.n_heads // world
        self.hkv = cfg.n_kv_heads // world
        self.layers = [Layer(cfg, i, blocks, self.device, seed, dtype) for i in range(cfg.n_layers)]
        self.embed = _draw((cfg.vocab_size, cfg.dim), _seed(seed, "embed"), self.device, dtype)
        self.head = _draw((cfg.vocab_size, cfg.dim), _seed(seed, "head"), self.device, dtype)
        self.final_norm = torch.ones(cfg.dim, dtype=dtype, device=self.device)
        self.attention = attention
        self.pos = torch.zeros(batch, dtype=torch.int64, device=self.device)  # position of the next token per sequence
        self.trees = None  # per layer, after enable_trees(): dense attention over the layer's cache
        self.mass = None   # per layer: attention weight received by each cached token
        if attention == "cuda":
            budget = Budget(cfg.init_budget, cfg.heavy_budget, cfg.recent_budget)
            h0 = rank * self.hq
            self.ctxs = []
            self.seq_lens = torch.zeros(batch, dtype=torch.int32, device=self.device)  # one copy for all layers
            for i in range(cfg.n_layers):
                cache = PagedHashKVCache(batch, self.hkv, cfg.max_seq_len, self.device)
                cache.seq_lens = self.seq_lens
                packed = make_usa(cfg.n_heads, cfg.head_dim, seed=seed * 1000 + i, bf16=True).packed(self.device)
                self.ctxs.append(SparseDecodeContext(cache, budget, packed.slice_heads(h0, h0 + self.hq)))
        else:
            self.kv = [None] * cfg.n_layers  # (k [B,Hkv_l,S,D], v)

    # -- collectives ---------------------------------------------------------------------------
    def all_reduce(self, x: torch.Tensor) -> torch.Tensor:
        """Sum of the row-parallel partial results over the ranks (efficiency/tp.py:114-115, 133-134)."""
        if self.world > 1:
            dist.all_reduce(x, op=dist.ReduceOp.SUM, group=self.group)
        return x

    # -- blocks ----------------------------------------------------------------------------------
    def _qkv(self, layer: Layer, h: torch.Tensor):
        cfg = self.cfg
        qkv = F.linear(h, layer.wqkv)
        q, k, v = qkv.split([self.hq * cfg.head_dim, self.hkv * cfg.head_dim, self.hkv * cfg.head_dim], dim=-1)
        return (q.reshape(*h.shape[:-1], self.hq, cfg.head_dim), k.reshape(*h.shape[:-1], self.hkv, cfg.head_dim),
                v.reshape(*h.shape[:-1], self.hkv, cfg.head_dim))

    def _mlp(self, layer: Layer, x: torch.Tensor) -> torch.Tensor:
        out = torch.empty_like(x)
        for s in range(0, x.shape[0], 8192):  # by blocks of tokens: the 14336-wide intermediate stays small
            h = rms_norm(x[s:s + 8192], layer.norm2, self.cfg.norm_eps)
            a, b = F.linear(h, layer.w13).chunk(2, dim=-1)
            out[s:s + 8192] = F.linear(F.silu(a) * b, layer.w2)
        return self.all_reduce(out)

    # -- prefill: one sequence at a time, dense causal attention -----------------------------------
    @torch.no_grad()
    def prefill(self, tokens: torch.Tensor, observe: int = 0) -> torch.Tensor:
        """tokens [B, S] -> next-token ids [B] (greedy). Fills the caches and builds the key hashes. ``observe``: the
        received weights (``enable_trees(..., mass=True)``) start with those of the prompt's last ``observe`` tokens."""
        cfg = self.cfg
        B, S = tokens.shape
        if observe:
            if self.mass is None or not 1 <= observe <= min(S, self.trees[0].max_nodes):
                raise ValueError(f"observe={observe} needs enable_trees(max_nodes >= observe, mass=True) and as many tokens")
            seen = [torch.empty(B, observe, self.hq, cfg.head_dim, dtype=torch.bfloat16, device=self.device) for _ in self.layers]
        nxt = torch.empty(B, dtype=torch.int64, device=self.device)
        pos = torch.arange(S, device=self.device)
        for b in range(B):
            x = self.embed[tokens[b]]
            for i, layer in enumerate(self.layers):
                h = rms_norm(x, layer.norm1, cfg.norm_eps)
                q, k, v = self._qkv(layer, h)               # [S, heads, D]
                q, k = rope(q, pos, cfg.rope_theta), rope(k, pos, cfg.rope_theta)
                qh, kh, vh = q.transpose(0, 1), k.transpose(0, 1), v.transpose(0, 1)  # [heads, S, D]
                att = F.scaled_dot_product_attention(qh[None], kh[None], vh[None], is_causal=True, enable_gqa=True)[0]
                if self.attention == "cuda":
                    self.ctxs[i].cache.write_kv(b, kh, vh)  # (stored as bf16)
                    if observe:
                        seen[i][b] = q[S - observe:]
                else:
                    if self.kv[i] is None:
                        self.kv[i] = (torch.zeros(B, self.hkv, S, cfg.head_dim, dtype=kh.dtype, device=self.device),
                                      torch.zeros(B, self.hkv, S, cfg.head_dim, dtype=kh.dtype, device=self.device))
                    self.kv[i][0][b], self.kv[i][1][b] = kh, vh
                o = F.linear(att.transpose(0, 1).reshape(S, self.hq * cfg.head_dim), layer.wo)
                x = x + self.all_reduce(o)
                x = x + self._mlp(layer, x)
            last = rms_norm(x[-1:], self.final_norm, cfg.norm_eps)
            nxt[b] = F.linear(last, self.head).float().argmax(-1)[0]
        if self.attention == "cuda":
            for ctx in self.ctxs:
                ctx.hash_prefill()
        if self.mass is not None:
            for m in self.mass:
                m.zero_()
        if observe:
            for i, tree in enumerate(self.trees):
                tree.attention_mass(seen[i], tree.tree_attention(seen[i])[1], self.mass[i])
        self.pos.fill_(S)
        return nxt

    # -- trees of drafted tokens, eviction -----------------------------------------------------------
    def enable_trees(self, max_nodes: int, mass: bool = False) -> None:
        """Prepares :meth:`verify_tree` for trees of up to ``max_nodes`` drafted tokens and, with ``mass``, keeps for every
        layer the attention weight that each cached token has received (what :meth:`evict` goes by). Allocates; the
        layers run one after another and share one workspace. The weights stay in these tensors for good: captured rounds
        hold their addresses."""
        if self.attention != "cuda":
            raise ValueError("trees are verified on the paged cache: attention='cuda'")
        self.trees = []
        for ctx in self.ctxs:
            self.trees.append(DenseDecodeContext(ctx.cache, max_nodes, workspace_of=self.trees[0] if self.trees else None))
        self.mass = [t.new_mass() for t in self.trees] if mass else None
        self._evicted_mass = self.trees[0].new_mass() if mass else None  # what an eviction leaves, on its way back into a layer's

    def _append_drafts(self, layer: int, k: torch.Tensor, v: torch.Tensor, first: torch.Tensor, tree_lens: torch.Tensor) -> None:
        """k, v [B, T, Hkv, 128] -> the cache's tokens first[b] .. first[b] + tree_lens[b] - 1, which have to fit. Rows behind a
        tree's own repeat its last one (in a sequence without drafts: put back the cache's last token)."""
        cache = self.ctxs[layer].cache
        n = tree_lens.long()[:, None]
        row = torch.minimum(torch.arange(k.shape[1], device=self.device)[None], n - 1)      # [B, T]; -1: no drafts
        token = (first.long()[:, None] + row).clamp(0, cache.max_pages * PAGE - 1)          # (an empty cache has no last token)
        page, slot = cache.page_table.long().gather(1, token // PAGE), token % PAGE
        take = row.clamp_min(0)[..., None, None].expand(-1, -1, *k.shape[2:])
        for pool, new in ((cache.k_pages, k), (cache.v_pages, v)):
            new = torch.where((n > 0)[..., None, None], new.gather(1, take), pool[page, :, slot])
            pool[page, :, slot] = new

    def _fitting_trees(self, tree_lens: torch.Tensor, nodes: int) -> torch.Tensor:
        """``tree_lens`` with 0 in the place of those out of 0 .. ``nodes`` and of those that do not fit the cache behind their
        sequence, which are reported (HA_ERR_BAD_SEQ_LEN, as the kernels do): such a sequence takes no part in the round."""
        lens, status = self.seq_lens, self.trees[0].status
        room = self.ctxs[0].cache.max_pages * PAGE - lens
        fits = (tree_lens >= 0) & (tree_lens <= nodes) & ((tree_lens == 0) | (lens >= 0) & (tree_lens <= room))
        status.copy_(torch.where((status == 0) & ~fits.all(), _lib.HA_ERR_BAD_SEQ_LEN, status))
        return torch.where(fits, tree_lens, 0)

    def _tree_forward(self, draft, mask, tree_lens):
        """Appends the drafts to every layer's cache (lengths and key hashes included) -> (logits [B, T, vocab], the layers'
        queries and log-sum-exps, where the received weights are kept)."""
        cfg = self.cfg
        B, T = draft.shape
        first = self.seq_lens.clone()
        self.seq_lens += tree_lens
        depth = unpack_nodes(mask).sum(-1) - 1                                     # ancestors of a node; -1 behind a tree
        pos = (self.pos[:, None] + depth.clamp_min(0)).reshape(-1)
        x = self.embed[torch.where(depth < 0, 0, draft).reshape(-1)]               # [B * T, dim]
        kept = []
        for i, layer in enumerate(self.layers):
            h = rms_norm(x, layer.norm1, cfg.norm_eps)
            q, k, v = rope_split(F.linear(h, layer.wqkv), pos, self.hq, self.hkv, cfg.rope_theta)
            q = q.view(B, T, self.hq, cfg.head_dim)
            self._append_drafts(i, k.view(B, T, self.hkv, -1), v.view(B, T, self.hkv, -1), first, tree_lens)
            self.ctxs[i].hash_prefill(first)
            att, lse = self.trees[i].tree_attention(q, mask, tree_lens)
            if self.mass is not None:
                kept.append((q, lse))
            x = x + self.all_reduce(F.linear(att.view(B * T, -1), layer.wo))
            x = x + self._mlp(layer, x)
        return F.linear(rms_norm(x, self.final_norm, cfg.norm_eps), self.head).view(B, T, -1), kept

    @torch.no_grad()
    def verify_tree(self, draft: torch.Tensor, parents: torch.Tensor, tree_lens: torch.Tensor | None = None) -> TreeAccept:
        """One round of speculative decoding: ``draft [B, T]`` int64 tokens of a tree per sequence (node 0: the token that is
        certain, as the previous step returned it), ``parents [B, T]`` int32 (-1: a root), ``tree_lens [B]`` int32 where trees
        are shorter than T. One pass with full attention over the cache, greedy acceptance, and the accepted path stays in the
        cache: positions and lengths advance by ``count``, ``next_token`` is the next round's node 0 (or the next
        :meth:`decode_step`'s token; where a sequence has no drafts, ``draft[:, 0]`` still is). With node 0 alone this is a
        dense decode step. A sequence whose drafts do not fit its cache (:meth:`evict` makes room) is left as it is, with a
        ``count`` of 0, and reported to :meth:`check_status`. Nothing synchronises with the host."""
        if self.trees is None or draft.dim() != 2 or not 1 <= draft.shape[1] <= self.trees[0].max_nodes:
            raise ValueError("verify_tree needs enable_trees(max_nodes) and a draft of [batch, 1 .. max_nodes] tokens")
        _check(draft, "draft", torch.int64, (self.batch, draft.shape[1]), self.trees[0].device)
        _check(parents, "parents", torch.int32, tuple(draft.shape), self.trees[0].device)
        status = self.trees[0].status
        if tree_lens is None:
            tree_lens = torch.full((self.batch,), draft.shape[1], dtype=torch.int32, device=self.device)
        _check(tree_lens, "tree_lens", torch.int32, (self.batch,), self.trees[0].device)
        tree_lens = self._fitting_trees(tree_lens, draft.shape[1])
        mask = tree_mask(parents, tree_lens, status=status)
        logits, kept = self._tree_forward(draft, mask, tree_lens)
        got = TreeAccept.empty(self.batch, draft.device)
        got.next_token.copy_(draft[:, 0])
        tree_accept(draft, parents, logits.float().argmax(-1), tree_lens, self.seq_lens, out=got, status=status)
        for i, tree in enumerate(self.trees):
            mass = None
            if self.mass is not None:
                mass = tree.attention_mass(*kept[i], self.mass[i], mask, tree_lens, rows=got.accepted)
            tree.tree_commit(got.accepted, tree_lens, mass=mass)
        self.seq_lens.copy_(got.seq_lens)
        self.pos += got.count
        return got

    @torch.no_grad()
    def evict(self, keep_tokens: int, init_budget: int | None = None, recent_budget: int | None = None) -> None:
        """Cuts every sequence longer than ``keep_tokens`` to the tokens of each layer and kv-head that received the most
        attention weight, beside the first ``init_budget`` and the last ``recent_budget`` (the decode step's, if left out).
        Positions go on. Sparse decode steps add no weight: what they appended since the last tree is best covered by
        ``recent_budget``."""
        if self.mass is None:
            raise ValueError("evict needs enable_trees(..., mass=True)")
        init_budget = self.cfg.init_budget if init_budget is None else init_budget
        recent_budget = self.cfg.recent_budget if recent_budget is None else recent_budget
        for i, tree in enumerate(self.trees):
            _, left, lens = tree.cache_evict(self.mass[i], keep_tokens, init_budget, recent_budget, mass_out=self._evicted_mass)
            self.mass[i].copy_(left)
        self.seq_lens.copy_(lens)

    # -- one greedy decode step for the whole batch ------------------------------------------------
    @torch.no_grad()
    def decode_step(self, tokens: torch.Tensor, out_tokens: torch.Tensor) -> None:
        """tokens [B] -> out_tokens [B] (written in place: the call is CUDA-graph capturable; positions and
        sequence lengths advance on the device)."""
        cfg = self.cfg
        x = self.embed[tokens]                                           # [B, dim]
        if self.attention == "cuda":
            self.seq_lens += 1  # the token being decoded counts (every layer's cache shares this tensor)
        for i, layer in enumerate(self.layers):
            h = rms_norm(x, layer.norm1, cfg.norm_eps)
            if self.attention == "cuda":
                # projection, then one kernel that splits q | k | v and rotates q and k, then the decode step
                q, k, v = rope_split(F.linear(h, layer.wqkv), self.pos, self.hq, self.hkv, cfg.rope_theta)
                att = self.ctxs[i].decode_step(q, k, v).to(x.dtype)
            else:
                q, k, v = self._qkv(layer, h)                            # [B, heads, D]
                q = rope(q[:, None], self.pos[:, None], cfg.rope_theta)[:, 0]
                k = rope(k[:, None], self.pos[:, None], cfg.rope_theta)[:, 0]
                kc = torch.cat([self.kv[i][0], k[:, :, None]], dim=2)
                vc = torch.cat([self.kv[i][1], v[:, :, None]], dim=2)
                self.kv[i] = (kc, vc)
                att = self.attention(i, q, kc, vc).to(x.dtype)
            o = F.linear(att.reshape(x.shape[0], self.hq * cfg.head_dim), layer.wo)
            x = x + self.all_reduce(o)
            x = x + self._mlp(layer, x)
        logits = F.linear(rms_norm(x, self.final_norm, cfg.norm_eps), self.head)
        out_tokens.copy_(logits.float().argmax(-1))
        self.pos += 1

    def check_status(self) -> None:
        if self.attention == "cuda":
            for ctx in self.ctxs + (self.trees or []):
                ctx.check_status()


def tokens_for(cfg: LlamaTPConfig, batch: int, length: int, seed: int = 1004) -> torch.Tensor:
    """Uniform random token ids [batch, length] from a fixed seed (the same on every rank)."""
    g = torch.Generator().manual_seed(seed)
    return torch.randint(0, cfg.vocab_size, (batch, length), generator=g)
