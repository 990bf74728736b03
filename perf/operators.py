"""Work of the operators over the paged cache beside the sparse step: dense attention of a tree of drafted tokens, the
attention weight each cached token has received, the commit of an accepted path, and eviction by accumulated weight.

A case is one pass through one of them, over a paged cache of 256-token pages in scattered order, 4 query heads per
kv-head, head dimension 128. Sizes are those of the package's own configurations and tests (8 kv-heads, or fewer where
the heads are cut over GPUs; contexts from a few hundred to 131072 tokens; 1 to 128 new tokens), or odd ones in between.

``run`` computes a pass with elementary torch operations in 32 bits, or, where ``own`` is true, with the package's
operators. ``exact`` computes the same from the definitions in 64 bits.
"""
import importlib.util
import math
import os
import random
import sys

import torch

own = False

GROUP, DIM, PAGE, WORDS = 4, 128, 256, 4
SCALE = 1.0 / math.sqrt(DIM)
ROW_BYTES = 2 * 2 * DIM  # a token's K and V of one kv-head
CODE_BYTES = 4 * GROUP   # its key codes
OUTLIERS = (3, 40, 77, 101)  # key channels of larger scale, as trained models have


def _package():
    """The package directory's name is no identifier: it is imported as ``hashattention_b200``."""
    if "hashattention_b200" not in sys.modules:
        root = os.path.join(os.getcwd(), "hashattention-1.0_b200")
        spec = importlib.util.spec_from_file_location("hashattention_b200", os.path.join(root, "__init__.py"),
                                                      submodule_search_locations=[root])
        module = importlib.util.module_from_spec(spec)
        sys.modules["hashattention_b200"] = module
        spec.loader.exec_module(module)
    return sys.modules["hashattention_b200"]


def _case(name, kind, batch, low, high, nodes=1, ragged=False, kv_heads=8, **more):
    case = dict(kind=kind, batch=batch, low=low, high=high, nodes=nodes, ragged=ragged, kv_heads=kv_heads, **more)
    return dict(case, name=name) if name else case


def listed():
    return [
        # ---- dense attention of drafted trees over the cache (one token: the dense decode step)
        # a short chat turn, one token of one sequence: all latency
        _case("attend_1x700_decode", "attend", 1, 701, 701, 1),
        # dense decode of a large ragged serving batch: the most cache that is read
        _case("attend_32x48k_decode", "attend", 32, 16384, 65536, 1),
        # small trees of odd sizes on one kv-head (the heads of a model cut over 8 GPUs); q is a view of the projection
        _case("attend_8x33k_tree13", "attend", 8, 33001, 33001, 13, True, 1, fused=True),
        # a mid-sized tree on one long document
        _case("attend_1x20k_tree32", "attend", 1, 20011, 20011, 32),
        # 64 drafts for each of four 128K sequences: the largest
        _case("attend_4x128k_tree64", "attend", 4, 131072, 131072, 64),
        # ---- weights the cached tokens receive
        # one decode step's weights, four sequences
        _case("mass_4x32k_decode", "mass", 4, 32768, 32768, 1, path=False),
        # the last 64 prompt tokens look back at two long prompts of odd lengths (an observation window before eviction)
        _case("mass_2x40k_window64", "mass", 2, 30011, 50021, 64, path=False),
        # ---- acceptance and commit of a drafted tree, all layers that hold it here
        # one sequence, 8 drafts, one layer
        _case("commit_1x8", "commit", 1, 701, 701, 8, layers=1),
        # a batch of 32 with trees of up to 64 drafts, four layers
        _case("commit_32x64", "commit", 32, 3000, 9001, 64, True, layers=4),
        # ---- eviction down to a budget
        # one 4K sequence cut to a quarter
        _case("evict_1x4k", "evict", 1, 4096, 4096, keep=1024, sink=128, recent=128),
        # a ragged batch on two kv-heads, some sequences short enough to stay whole
        _case("evict_8x15k_ragged", "evict", 8, 5000, 15000, kv_heads=2, keep=7001, sink=4, recent=257),
        # four 128K sequences cut to a quarter: the most rows moved
        _case("evict_4x128k", "evict", 4, 131072, 131072, keep=32768, sink=128, recent=128),
    ]


def _log_uniform(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(["attend", "attend", "attend", "mass", "mass", "commit", "evict", "evict"])
    kv_heads = rng.choice([1, 2, 4, 8, 8, 8])
    batch = _log_uniform(rng, 1, 32)
    high = _log_uniform(rng, 300, 131072)
    batch = min(batch, max(1, 1200000 // high))
    low = high if rng.random() < 0.4 else max(150, high - rng.randrange(high // 2 + 1))
    nodes = 1 if rng.random() < 0.25 else _log_uniform(rng, 2, 128)
    ragged = nodes > 1 and rng.random() < 0.5
    if kind in ("attend", "mass"):
        # no more products than 64 drafts for each of four 128K sequences, a few times fewer for the weights
        most = 4 * 131072 * 64 * 8 // (1 if kind == "attend" else 4)
        while batch > 1 and batch * high * nodes * kv_heads > most:
            batch -= 1
        nodes = max(1, min(nodes, most // (batch * high * kv_heads)))
        low, high = max(low, nodes), max(high, nodes)
        if kind == "attend":
            return _case(None, kind, batch, low, high, nodes, ragged and nodes > 1, kv_heads, fused=rng.random() < 0.3)
        return _case(None, kind, batch, low, high, nodes, ragged and nodes > 1, kv_heads, path=nodes > 1 and rng.random() < 0.5)
    if kind == "commit":
        high = min(high, 20000)
        return _case(None, kind, batch, min(low, high), high, nodes, ragged, kv_heads, layers=rng.choice([1, 2, 4]))
    batch = min(batch, max(1, 524288 // high))
    sink, recent = rng.choice([0, 4, 128]), rng.choice([0, 1, 128, 257])
    keep = max(sink + recent + 1, _log_uniform(rng, max(64, high // 16), high))
    return _case(None, kind, batch, low, high, kv_heads=kv_heads, keep=keep, sink=sink, recent=recent)


def _lengths(case):
    """Cached lengths (drafts included) and drafts of the sequences: part of the case, so that another seed changes
    values and not sizes."""
    rng = random.Random(case["batch"] * 1000003 + case["low"] * 31 + case["high"] * 7 + case["nodes"])
    lens = [rng.randint(case["low"], case["high"]) for _ in range(case["batch"])]
    nodes = [rng.randint(1, case["nodes"]) if case["ragged"] else case["nodes"] for _ in range(case["batch"])]
    return [max(s, n) for s, n in zip(lens, nodes)], nodes


def work(case):
    """Bytes that have to be read and written once, and multiply-adds (two each) of the products."""
    lens, nodes = _lengths(case)
    heads, kind = case["kv_heads"], case["kind"]
    rows = sum(nodes) * GROUP * heads
    pairs = sum(s * n for s, n in zip(lens, nodes)) * GROUP * heads
    if kind == "attend":
        return {"bytes": sum(lens) * heads * ROW_BYTES + rows * (2 * 2 * DIM + 4) + sum(nodes) * 16, "flops": 4.0 * DIM * pairs}
    if kind == "mass":
        return {"bytes": sum(lens) * heads * (2 * DIM + 8) + rows * (2 * DIM + 4), "flops": 2.0 * DIM * pairs}
    if kind == "commit":
        # drafts, parents, targets and words; about half of a path's rows move (the drawn paths are a few tokens long)
        moved = sum(max(1, int(math.log2(n + 1))) for n in nodes) * case["layers"] * heads
        return {"bytes": sum(nodes) * (8 + 4 + 8 + 16) + 2 * moved * (ROW_BYTES + CODE_BYTES), "flops": 0.0}
    total = 0
    for s in lens:
        if s > case["keep"]:
            total += 4 * heads * s + heads * (case["keep"] - case["sink"]) * 2 * (ROW_BYTES + CODE_BYTES) + heads * case["keep"] * 8
        else:
            total += 8 * heads * s
    return {"bytes": total, "flops": 0.0}


# ---- inputs ----------------------------------------------------------------------------------------------------------
def _words(bits):
    """[..., up to 128] truth values -> [..., 4] int32 words, bit j of the row in word j // 32."""
    pad = torch.zeros(*bits.shape[:-1], 32 * WORDS - bits.shape[-1], dtype=torch.bool, device=bits.device)
    b = torch.cat([bits, pad], -1).view(*bits.shape[:-1], WORDS, 32).long()
    w = (b << torch.arange(32, device=bits.device)).sum(-1)
    return torch.where(w >= 2 ** 31, w - 2 ** 32, w).int()


def _bits(words, n):
    """[..., 4] int32 words -> [..., n] truth values."""
    b = (words[..., None].long() >> torch.arange(32, device=words.device)) & 1
    return b.flatten(-2)[..., :n].bool()


def _reach(parents, nodes):
    """[B, T] parents -> [B, T, T]: node j is node i or one of its ancestors (rows of real nodes only)."""
    T = parents.shape[1]
    at = torch.arange(T, device=parents.device)
    up = ((parents[..., None] == at) | (at[:, None] == at)).float()
    for _ in range(max(1, (T - 1).bit_length())):
        up = (torch.matmul(up, up) > 0).float()
    return (up > 0) & (at[:, None] < nodes[:, None, None]) & (at < nodes[:, None, None])


def _layer(case, lens, gen, dev):
    """One layer's page pools: K, V, key codes."""
    pages = case["batch"] * -(-max(lens) // PAGE)
    shape = (pages, case["kv_heads"], PAGE, DIM)
    k = torch.empty(shape, dtype=torch.bfloat16, device=dev)
    v = torch.empty(shape, dtype=torch.bfloat16, device=dev)
    step = max(1, (1 << 27) // (case["kv_heads"] * PAGE * DIM))
    for i in range(0, pages, step):
        part = torch.randn(k[i:i + step].shape, generator=gen, device=dev)
        part[..., list(OUTLIERS)] *= 8.0
        k[i:i + step] = part
        v[i:i + step] = torch.randn(part.shape, generator=gen, device=dev)
    codes = torch.randint(-2 ** 31, 2 ** 31 - 1, (pages, case["kv_heads"], PAGE, GROUP), generator=gen, device=dev, dtype=torch.int32)
    return k, v, codes


def _inputs(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    lens, nodes = _lengths(case)
    B, H, T = case["batch"], case["kv_heads"], case["nodes"]
    width = -(-max(lens) // PAGE)
    x = {"case": case, "lens": lens, "nodes": nodes}
    x["layers"] = [_layer(case, lens, gen, dev) for _ in range(case.get("layers", 1))]
    x["table"] = torch.randperm(B * width, generator=gen, device=dev).int().view(B, width)
    x["seq_lens"] = torch.tensor(lens, dtype=torch.int32, device=dev)
    x["tree_lens"] = torch.tensor(nodes, dtype=torch.int32, device=dev)
    if case["kind"] != "evict":
        # every node hangs on one of the nodes before it, more often on a late one
        at = torch.arange(T, device=dev)
        x["parents"] = (torch.rand(B, T, generator=gen, device=dev).sqrt() * at).floor().clamp_max(T).int()
        x["parents"][:, 0] = -1
        x["visible"] = _reach(x["parents"], x["tree_lens"])
        x["mask"] = _words(x["visible"])
    if case["kind"] in ("attend", "mass"):
        if case.get("fused"):  # the query heads' part of a fused q | k | v projection
            x["q"] = torch.randn(B, T, (GROUP + 2) * H, DIM, generator=gen, device=dev).bfloat16()[:, :, :GROUP * H]
        else:
            x["q"] = torch.randn(B, T, GROUP * H, DIM, generator=gen, device=dev).bfloat16()
    if case["kind"] == "attend":
        x["out"] = torch.zeros(B, T, GROUP * H, DIM, dtype=torch.bfloat16, device=dev)
        x["lse"] = torch.zeros(B, T, GROUP * H, dtype=torch.float32, device=dev)
    if case["kind"] == "mass":
        x["lse"] = torch.zeros(B, T, GROUP * H, dtype=torch.float32, device=dev)
        for b in range(B):  # what the attention in front left
            x["lse"][b, :nodes[b]] = _attend_one(x, b)[1]
        # as much as a few passes like this one leave
        at = torch.arange(width * PAGE, device=dev)
        x["mass"] = torch.rand(B, H, width * PAGE, generator=gen, device=dev) * (at < x["seq_lens"][:, None, None])
        x["mass"] *= (GROUP * 4 * x["tree_lens"] / x["seq_lens"])[:, None, None]
        x["rows"] = None
        if case["path"]:  # the weights of an accepted path alone: one node and its ancestors
            last = [(n - 1) * 3 // 4 for n in nodes]
            x["rows"] = torch.stack([x["mask"][b, last[b]] for b in range(B)])
    if case["kind"] == "evict":
        x["mass"] = _masses(case, lens, width, gen, dev)
    if case["kind"] == "commit":
        # half of the drafted tokens are what the target model says behind their parent
        x["target"] = torch.randint(0, 128256, (B, T), generator=gen, device=dev)
        draft = torch.randint(0, 128256, (B, T), generator=gen, device=dev)
        right = x["target"].gather(1, x["parents"].long().clamp_min(0))
        x["draft"] = torch.where(torch.rand(B, T, generator=gen, device=dev) < 0.5, right, draft)
    return x


def _masses(case, lens, width, gen, dev):
    """Accumulated weights: few large ones, many small ones, equal ones among them, nothing behind a sequence's end."""
    m = torch.rand(case["batch"], case["kv_heads"], width * PAGE, generator=gen, device=dev)
    m = ((1.0 / (1e-3 + m)) * 64).floor() / 64
    at = torch.arange(width * PAGE, device=dev)
    return m * (at < torch.tensor(lens, device=dev)[:, None, None])


def prepare(case, seed):
    x = _inputs(case, seed)
    if own:
        ha = _package()
        x["contexts"] = []
        for k, v, codes in x["layers"]:
            cache = ha.PagedHashKVCache(case["batch"], case["kv_heads"], PAGE, k.device)
            cache.num_pages, cache.max_pages = k.shape[0], x["table"].shape[1]  # the filled pools in place of its own
            cache.k_pages, cache.v_pages, cache.hash_pages = k, v, codes
            cache.page_table, cache.seq_lens = x["table"], x["seq_lens"]
            x["contexts"].append(ha.DenseDecodeContext(cache, case["nodes"]))
    if case["kind"] == "evict":
        x["kept"] = torch.full((case["batch"], case["kv_heads"], case["keep"]), -1, dtype=torch.int32, device=x["mass"].device)
        x["mass_out"], x["lens_out"] = torch.empty_like(x["mass"]), torch.empty_like(x["seq_lens"])
    return x


# ---- the plain forms -------------------------------------------------------------------------------------------------
def _rows(pool, table, length):
    """A sequence's rows [Hkv, length, D] in 32 bits."""
    pages = pool[table[: -(-length // PAGE)].long()]
    return pages.transpose(0, 1).flatten(1, 2)[:, :length].float()


def _scores(x, b):
    """[Hkv, nodes * 4, length] scaled scores of one sequence, -inf where nothing is visible."""
    n, s, (k, _, _) = x["nodes"][b], x["lens"][b], x["layers"][0]
    heads = x["case"]["kv_heads"]
    q = x["q"][b, :n].float().view(n, heads, GROUP, DIM).transpose(0, 1).reshape(heads, n * GROUP, DIM)
    scores = torch.matmul(q, _rows(k, x["table"][b], s).transpose(1, 2)) * SCALE
    hidden = ~_bits(x["mask"][b, :n], n)
    scores[:, :, s - n:].masked_fill_(hidden.repeat_interleave(GROUP, 0), -math.inf)
    return scores


def _attend_one(x, b):
    n, heads = x["nodes"][b], x["case"]["kv_heads"]
    scores = _scores(x, b)
    top = scores.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    p = scores.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p, _rows(x["layers"][0][1], x["table"][b], x["lens"][b]))
    out = torch.where(total > 0, out / total, torch.zeros_like(out))
    lse = (top + total.log())[..., 0]

    def back(t):  # [Hkv, nodes * 4, ...] -> [nodes, Hq, ...]
        return t.view(heads, n, GROUP, *t.shape[2:]).transpose(0, 1).reshape(n, heads * GROUP, *t.shape[2:])

    return back(out).bfloat16(), back(lse)


def _attend(x):
    for b in range(x["case"]["batch"]):
        n = x["nodes"][b]
        x["out"][b, :n], x["lse"][b, :n] = _attend_one(x, b)
    return x["out"], x["lse"]


def _mass(x):
    heads = x["case"]["kv_heads"]
    for b in range(x["case"]["batch"]):
        n = x["nodes"][b]
        lse = x["lse"][b, :n].view(n, heads, GROUP).transpose(0, 1).reshape(heads, n * GROUP, 1)
        p = _scores(x, b).sub_(lse).exp_()
        if x["rows"] is not None:
            p = p * _bits(x["rows"][b], n).repeat_interleave(GROUP)[:, None].float()
        x["mass"][b, :, :x["lens"][b]] += p.sum(1)
    return x["mass"]


def _slots(x, tokens):
    """Row numbers [B, ...] of token numbers [B, n] in a pool seen as [pages * PAGE] slots of one kv-head's page."""
    page = x["table"].long().gather(1, (tokens // PAGE).flatten(1)).view(tokens.shape)
    return page, tokens % PAGE


def _commit(x):
    at = torch.arange(x["case"]["nodes"], device=x["parents"].device)
    n = x["tree_lens"][:, None]
    reach = _reach(x["parents"], x["tree_lens"])
    parent = x["parents"].long().clamp_min(0)
    same = (x["parents"][:, :, None] == x["parents"][:, None, :]) & (x["draft"][:, :, None] == x["draft"][:, None, :])
    first = ~(same & (at < at[:, None])).any(-1)  # of equal children of one node the lowest counts
    good = ((x["draft"] == x["target"].gather(1, parent)) & first) | (at == 0)
    accepted = ~(reach & ~good[:, None, :]).any(-1) & (at < n)
    count = accepted.sum(1).int()
    last = (accepted * (at + 1)).amax(1) - 1
    nxt = x["target"].gather(1, last[:, None])[:, 0]
    prefix = (x["seq_lens"] - x["tree_lens"]).long()
    order = torch.sort((~accepted).int(), dim=1, stable=True).indices  # accepted nodes first, in order
    keep = at < count[:, None]
    source = prefix[:, None] + torch.where(keep, order, torch.zeros_like(order))
    dest = prefix[:, None] + torch.where(keep, at.expand_as(order), torch.zeros_like(order))
    (sp, ss), (dp, ds) = _slots(x, source), _slots(x, dest)
    for pools in x["layers"]:
        for pool in pools:
            pool[dp, :, ds] = pool[sp, :, ss]
    return _words(reach), _words(accepted), count, nxt, (prefix + count).int(), x["layers"]


def _evict(x):
    case, dev = x["case"], x["table"].device
    B, H, keep, sink, recent = (case[k] for k in ("batch", "kv_heads", "keep", "sink", "recent"))
    kept, mass = x["kept"], x["mass_out"].zero_()
    heads = torch.arange(H, device=dev)[:, None]
    for b in range(B):
        s = x["lens"][b]
        if s <= keep:
            index = torch.arange(s, device=dev).expand(H, s)
        else:
            m = x["mass"][b, :, sink:s - recent]
            m = torch.where(m > 0, m, torch.zeros_like(m))
            best = torch.sort(m, dim=-1, descending=True, stable=True).indices[:, :keep - sink - recent] + sink
            index = torch.cat([torch.arange(sink, device=dev).expand(H, sink), torch.sort(best, dim=-1).values,
                               torch.arange(s - recent, s, device=dev).expand(H, recent)], -1)
            page, slot = x["table"][b].long()[index // PAGE], index % PAGE
            at = torch.arange(keep, device=dev)
            to, slot_to = x["table"][b].long()[at // PAGE], at % PAGE
            for pool in x["layers"][0]:
                pool[to[None], heads, slot_to[None]] = pool[page, heads, slot]
        kept[b, :, :index.shape[1]] = index
        mass[b, :, :index.shape[1]] = x["mass"][b].gather(1, index)
    return kept, mass, x["seq_lens"].clamp_max(keep), x["layers"]


# ---- the package's operators -----------------------------------------------------------------------------------------
def _own(x):
    kind, ctx = x["case"]["kind"], x["contexts"][0]
    if kind == "attend":
        return ctx.tree_attention(x["q"], x["mask"], x["tree_lens"], out=x["out"], lse=x["lse"])
    if kind == "mass":
        return ctx.attention_mass(x["q"], x["lse"], x["mass"], x["mask"], x["tree_lens"], rows=x["rows"])
    ha = _package()
    if kind == "commit":
        mask = ha.tree_mask(x["parents"], x["tree_lens"])
        got = ha.tree_accept(x["draft"], x["parents"], x["target"], x["tree_lens"], x["seq_lens"])
        for c in x["contexts"]:
            c.tree_commit(got.accepted, x["tree_lens"])
        return mask, got.accepted, got.count, got.next_token, got.seq_lens, x["layers"]
    case = x["case"]
    kept, mass, lens = ctx.cache_evict(x["mass"], case["keep"], case["sink"], case["recent"], kept=x["kept"],
                                       mass_out=x["mass_out"], lens_out=x["lens_out"])
    return kept, mass, lens, x["layers"]


def run(state):
    """One pass. Rows and entries behind a sequence's own are the buffers' as they were."""
    if own:
        return _own(state)
    return {"attend": _attend, "mass": _mass, "commit": _commit, "evict": _evict}[state["case"]["kind"]](state)


# ---- the definitions in 64 bits --------------------------------------------------------------------------------------
def exact(case, seed):
    x = _inputs(case, seed)
    dev, lens, nodes = x["table"].device, x["lens"], x["nodes"]
    if case["kind"] in ("attend", "mass"):
        out = torch.zeros(case["batch"], case["nodes"], GROUP * case["kv_heads"], DIM, dtype=torch.float64, device=dev)
        lse = torch.zeros(out.shape[:-1], dtype=torch.float64, device=dev)
        mass = x["mass"].double() if case["kind"] == "mass" else None
        for b in range(case["batch"]):
            token = torch.arange(lens[b], device=dev)
            page, slot = x["table"][b, token // PAGE].long(), token % PAGE
            for h in range(case["kv_heads"]):
                k, v = (x["layers"][0][i][page, h, slot].double() for i in (0, 1))
                for g in range(GROUP):
                    qh = h * GROUP + g
                    s = x["q"][b, :nodes[b], qh].double() @ k.T / math.sqrt(DIM)
                    s[:, lens[b] - nodes[b]:][~x["visible"][b, :nodes[b], :nodes[b]]] = -math.inf
                    if case["kind"] == "attend":
                        lse[b, :nodes[b], qh] = torch.logsumexp(s, 1)
                        out[b, :nodes[b], qh] = torch.softmax(s, 1) @ v
                    else:
                        w = torch.exp(s - x["lse"][b, :nodes[b], qh].double()[:, None])
                        if x["rows"] is not None:
                            w = w[_bits(x["rows"][b], nodes[b])]
                        mass[b, h, :lens[b]] += w.sum(0)
        return (out, lse) if case["kind"] == "attend" else mass
    if case["kind"] == "commit":
        parents, draft, target = (x[k].tolist() for k in ("parents", "draft", "target"))
        reach = torch.zeros(case["batch"], case["nodes"], 32 * WORDS, dtype=torch.bool)
        taken = torch.zeros(case["batch"], 32 * WORDS, dtype=torch.bool)
        count, nxt, new, paths = [], [], [], []
        for b in range(case["batch"]):
            for i in range(nodes[b]):
                j = i
                while j >= 0:
                    reach[b, i, j] = True
                    j = parents[b][j]
            path = [0]
            while True:
                step = [i for i in range(1, nodes[b]) if parents[b][i] == path[-1] and draft[b][i] == target[b][path[-1]]]
                if not step:
                    break
                path.append(step[0])
            taken[b, path] = True
            paths.append(path)
            count.append(len(path))
            nxt.append(target[b][path[-1]])
            new.append(lens[b] - nodes[b] + len(path))
        for pools in x["layers"]:
            for pool in pools:
                for b, path in enumerate(paths):
                    for i, a in enumerate(path):  # a node is never in front of its place on the path
                        f, t = (lens[b] - nodes[b] + j for j in (a, i))
                        pool[x["table"][b, t // PAGE].long(), :, t % PAGE] = pool[x["table"][b, f // PAGE].long(), :, f % PAGE]
        small = lambda v, t: torch.tensor(v, dtype=t, device=dev)  # noqa: E731
        return (_words(reach.to(dev)), _words(taken.to(dev)), small(count, torch.int32), small(nxt, torch.int64),
                small(new, torch.int32), x["layers"])
    kept = torch.full((case["batch"], case["kv_heads"], case["keep"]), -1, dtype=torch.int32, device=dev)
    mass = torch.zeros(x["mass"].shape, dtype=torch.float64, device=dev)
    for b in range(case["batch"]):
        for h in range(case["kv_heads"]):
            s, m = lens[b], x["mass"][b, h, :lens[b]].double()
            free = torch.ones(s, dtype=torch.bool, device=dev)
            if s > case["keep"]:
                wanted = case["keep"] - case["sink"] - case["recent"]
                value = m.clone()
                value[:case["sink"]] = value[s - case["recent"]:] = -1.0
                edge = torch.kthvalue(value, s - wanted + 1).values if wanted else math.inf
                above = value > edge
                level = (value == edge).nonzero()[:, 0][:wanted - int(above.sum())] if wanted else None
                free = above
                if wanted:
                    free[level] = True
                free[:case["sink"]] = free[s - case["recent"]:] = True
            index = free.nonzero()[:, 0]
            n = index.numel()
            kept[b, h, :n] = index.int()
            mass[b, h, :n] = m[index]
            to = torch.arange(n, device=dev)
            for pool in x["layers"][0]:
                rows = pool[x["table"][b, index // PAGE].long(), h, index % PAGE]
                pool[x["table"][b, to // PAGE].long(), h, to % PAGE] = rows
    return kept, mass, x["seq_lens"].clamp_max(case["keep"]), x["layers"]
