"""Dense attention of drafted trees over the paged cache, received attention weights, acceptance and commit of a tree,
eviction by accumulated weight: each against a plain implementation in 64 bits, at the sizes and masks where it can go wrong.

Tolerances. A score is a sum of 128 exact products in fp32, off by at most d = 128 * 2^-24 * c * sum |q k| (c: the softmax
scale); a weight's exponential, its split into two bf16 and the sums add less than 2^-15 relative. The output, an average of V by
those weights, is then off by at most (2 d + 2^-15) max|v|, and its bf16 rounding by 2^-8 of the value. The log-sum-exp is off
by d and a few ulp of its magnitude; a received weight, relative to itself, by twice d (its score's and its row's) and 2^-18."""
import ctypes
import math

import pytest
import torch

import hashattention_b200 as ha
from hashattention_b200 import _lib

D, PAGE, GROUP = 128, 256, 4


# ---- plain implementations in 64 bits ------------------------------------------------------------------------------------
def reach(parents):
    """Truth matrix [n, n] of one tree: node j is node i or one of its ancestors."""
    n = len(parents)
    m = torch.zeros(n, n, dtype=torch.bool)
    for i in range(n):
        j = i
        while j >= 0:
            m[i, j] = True
            j = parents[j]
    return m


def random_parents(n, gen):
    return [-1] + [int(torch.randint(0, i, (1,), generator=gen)) for i in range(1, n)]


def weights64(q, k, visible, scale):
    """q [n, Hq, D], k [Hkv, S, D], visible [n, S] -> softmax weights [n, Hq, S] and log-sum-exps [n, Hq]; rows that see
    nothing: zeros, -inf. A token that a row does not see does not enter, whatever its K holds."""
    k = k.double().repeat_interleave(GROUP, 0)
    s = torch.einsum("nhd,hsd->nhs", q.double(), k) * scale
    s = torch.where(visible[:, None, :], s, torch.full_like(s, -math.inf))
    top = s.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    e = torch.exp(s - top)
    total = e.sum(-1, keepdim=True)
    p = torch.where(total == 0, torch.zeros_like(e), e / total)
    return p, (top + total.log())[..., 0]


def attention64(q, k, v, visible, scale):
    p, lse = weights64(q, k, visible, scale)
    v = v.double().repeat_interleave(GROUP, 0)
    if bool(torch.isfinite(v).all()):
        return torch.einsum("nhs,hsd->nhd", p, v), lse
    out = torch.zeros(*p.shape[:2], D, dtype=torch.float64, device=p.device)
    for i in range(p.shape[0]):  # only what the row sees
        out[i] = torch.einsum("hs,hsd->hd", p[i][:, visible[i]], v[:, visible[i]])
    return out, lse


def score_error(q, k, scale):
    """d of the module's docstring."""
    big = torch.einsum("nhd,hsd->nhs", q.double().abs(), k.double().abs().repeat_interleave(GROUP, 0)).nan_to_num(0, 0, 0).amax()
    return 128 * 2.0 ** -24 * scale * float(big)


# ---- problems ----------------------------------------------------------------------------------------------------------------
class Problem:
    """A filled cache of ragged lengths over shuffled pages, its unused slots full of NaN, with drafted trees and queries."""

    def __init__(self, device, lens, nodes, kv_heads=2, width=None, mask="tree", seed=0, fused=False, extra_pages=3):
        g = torch.Generator().manual_seed(seed)
        self.lens, self.nodes, self.T, self.B, self.hkv = list(lens), list(nodes), width or max(1, max(nodes)), len(lens), kv_heads
        hq = self.hq = kv_heads * GROUP
        pages = -(-max(max(lens), 1) // PAGE)
        self.cache = ha.PagedHashKVCache(self.B, kv_heads, pages * PAGE, device, num_pages=self.B * pages + extra_pages, shuffle_seed=seed + 1)
        self.cache.k_pages.fill_(math.nan)
        self.cache.v_pages.fill_(math.nan)
        self.cache.hash_pages.copy_(torch.randint(-2 ** 31, 2 ** 31 - 1, self.cache.hash_pages.shape, generator=g, dtype=torch.int32))
        self.k = [torch.randn(kv_heads, s, D, generator=g).bfloat16().to(device) for s in lens]
        self.v = [torch.randn(kv_heads, s, D, generator=g).bfloat16().to(device) for s in lens]
        for b in range(self.B):
            self.write(b)
        whole = torch.randn(self.B, self.T, hq + (2 * kv_heads if fused else 0), D, generator=g).bfloat16().to(device)
        self.q = whole[:, :, :hq]
        self.parents = torch.full((self.B, self.T), -1, dtype=torch.int32)
        self.visible = []  # [n, n] per sequence
        for b, n in enumerate(nodes):
            tree = random_parents(n, g) if n else []
            if mask == "chain":
                tree = list(range(-1, n - 1))
            self.parents[b, :n] = torch.tensor(tree, dtype=torch.int32)
            m = reach(tree)
            if mask == "random":  # any mask, rows that see nothing of the tree among them
                m = torch.rand(n, n, generator=g) < 0.3
            self.visible.append(m)
        bits = torch.zeros(self.B, self.T, 128, dtype=torch.bool)
        for b, n in enumerate(nodes):
            bits[b, :n, :n] = self.visible[b]
            if mask == "random":
                bits[b, :n, n:] = True  # bits behind the tree's end mean nothing
        self.mask = ha.pack_nodes(bits).to(device)
        self.parents = self.parents.to(device)
        self.tree_lens = torch.tensor(nodes, dtype=torch.int32, device=device)
        self.cache.seq_lens.copy_(torch.tensor(lens, dtype=torch.int32))
        self.ctx = ha.DenseDecodeContext(self.cache, self.T)
        self.scale = self.ctx.sm_scale
        self.device = device

    def write(self, b):
        if self.lens[b]:
            self.cache.write_kv(b, self.k[b], self.v[b])

    def sees(self, b):
        n, s = self.nodes[b], self.lens[b]
        return torch.cat([torch.ones(n, s - n, dtype=torch.bool), self.visible[b]], 1).to(self.device)

    def check(self, out, lse, untouched=0.0):
        for b, n in enumerate(self.nodes):
            assert bool((out[b, n:] == untouched).all()) and bool((lse[b, n:] == untouched).all()), "rows behind the tree were written"
            if n == 0:
                continue
            want, want_lse = attention64(self.q[b, :n], self.k[b], self.v[b], self.sees(b), self.scale)
            d = score_error(self.q[b, :n], self.k[b], self.scale)
            vmax = float(self.v[b].double().nan_to_num(0, 0, 0).abs().amax())
            got, got_lse = out[b, :n].double(), lse[b, :n].double()
            same = torch.isfinite(want)
            assert torch.equal(torch.isfinite(got), same), "finite in other places than the definition"
            assert torch.equal(torch.isnan(got), torch.isnan(want))
            assert torch.equal(got[~same & ~torch.isnan(want)], want[~same & ~torch.isnan(want)])
            off = (got - want).abs()[same]
            allowed = (2.0 ** -8 * want.abs() + (2 * d + 2.0 ** -15) * vmax)[same]
            assert bool((off <= allowed).all()), (b, float((off - allowed).max()))
            fine = torch.isfinite(want_lse)
            assert torch.equal(got_lse[~fine & ~torch.isnan(want_lse)], want_lse[~fine & ~torch.isnan(want_lse)])
            assert torch.equal(torch.isnan(got_lse), torch.isnan(want_lse))
            assert bool(((got_lse - want_lse).abs()[fine] <= d + 4 * 2.0 ** -23 * (1 + want_lse.abs()[fine])).all())


TREES = [
    # lengths (drafts included), drafts, width of the arrays, kv-heads, mask
    ([1], [1], 1, 1, "tree"), ([2, 64, 65], [1, 1, 1], 1, 2, "tree"), ([255, 256, 257, 513], [1, 1, 1, 1], 1, 1, "tree"),
    ([700], [1], 1, 8, "chain"), ([5000, 1, 333], [1, 1, 1], 1, 2, "tree"),
    ([3, 130, 700], [3, 2, 4], 4, 2, "tree"), ([260, 64], [4, 1], 4, 2, "random"),
    ([8, 257, 1000], [8, 5, 7], 8, 2, "tree"), ([300, 20], [8, 0], 8, 1, "tree"),
    ([13, 500, 1030], [13, 9, 13], 13, 1, "random"), ([2049], [17], 17, 2, "chain"), ([40, 512], [31, 32], 32, 2, "tree"),
    ([33, 290, 768], [33, 1, 20], 33, 2, "tree"), ([64, 1500], [64, 64], 64, 2, "random"), ([700, 65], [65, 60], 65, 1, "tree"),
    ([128, 129, 400], [128, 127, 100], 128, 2, "tree"), ([384], [128], 128, 1, "random"), ([0, 500, 0], [0, 3, 0], 5, 1, "tree"),
    ([9000] * 3, [2, 11, 30], 30, 1, "tree"),
]


@pytest.mark.gpu
@pytest.mark.parametrize("lens,nodes,width,kv_heads,mask", TREES)
def test_tree_attention(device, lens, nodes, width, kv_heads, mask):
    x = Problem(device, lens, nodes, kv_heads, width, mask, seed=len(lens) + width, fused=width % 2 == 1)
    out = torch.zeros(x.B, x.T, x.hq, D, dtype=torch.bfloat16, device=device)
    lse = torch.zeros(x.B, x.T, x.hq, device=device)
    got = x.ctx.tree_attention(x.q, x.mask, x.tree_lens, out=out, lse=lse)
    assert got[0] is out and got[1] is lse
    x.ctx.check_status()
    x.check(out, lse)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1, 3, 8, 40, 128])
def test_no_mask_is_a_chain_and_no_lengths_are_full_trees(device, n):
    x = Problem(device, [n, 600 + n], [n, n], 1, n, "chain", seed=n)
    out, lse = x.ctx.tree_attention(x.q)
    with_words = x.ctx.tree_attention(x.q, x.mask, x.tree_lens)
    x.check(out, lse)
    assert torch.equal(out, with_words[0]) and torch.equal(lse, with_words[1])


@pytest.mark.gpu
@pytest.mark.parametrize("n", [2, 7, 20, 60, 100])
def test_rows_that_see_nothing(device, n):
    """No prefix, and nodes whose mask is empty: zeros and -inf, as the definition says."""
    x = Problem(device, [n, n + 5], [n, n], 2, n, "tree", seed=n)
    bits = ha.unpack_nodes(x.mask.cpu())
    for i in range(1, n, 2):
        bits[0, i] = False
        x.visible[0][i] = False
    x.mask = ha.pack_nodes(bits).to(device)
    out, lse = x.ctx.tree_attention(x.q, x.mask, x.tree_lens)
    x.check(out, lse)
    assert bool((out[0, 1] == 0).all()) and bool((lse[0, 1] == -math.inf).all())


@pytest.mark.gpu
@pytest.mark.parametrize("n,prefix", [(6, 0), (6, 300), (30, 250), (50, 130), (100, 40)])
@pytest.mark.parametrize("what", ["k", "v"])
@pytest.mark.parametrize("value", [math.inf, -math.inf, math.nan])
def test_infinities_and_nan_stay_with_the_branches_that_see_them(device, n, prefix, what, value):
    x = Problem(device, [prefix + n], [n], 2, n, "tree", seed=n + prefix)
    leaf = n - 1
    where = x.k if what == "k" else x.v
    where[0][0, prefix + leaf, 5] = value
    where[0][1, prefix + leaf // 2, 77] = value
    x.write(0)
    out, lse = x.ctx.tree_attention(x.q, x.mask, x.tree_lens)
    x.check(out, lse)
    blind = ~x.visible[0][:, leaf]  # rows of kv-head 0 that do not see the leaf
    assert bool(torch.isfinite(out[0, blind.to(device), :GROUP]).all())


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1, 4, 20, 64])
def test_large_scores_and_values(device, n):
    """Scores of a few hundred (one token has all the weight) and huge values."""
    x = Problem(device, [900, 300], [n, n], 1, n, "tree", seed=3 * n)
    x.q.mul_(30.0)
    for b in range(2):
        x.v[b][:, :, 3] = 2.0 ** 100
        x.write(b)
    out, lse = x.ctx.tree_attention(x.q, x.mask, x.tree_lens)
    for b in range(2):
        want, want_lse = attention64(x.q[b], x.k[b], x.v[b], x.sees(b), x.scale)
        d = score_error(x.q[b], x.k[b], x.scale)
        off, big = (out[b].double() - want).abs(), x.v[b].double().abs().amax(1).repeat_interleave(GROUP, 0)
        assert bool((off <= 2.0 ** -8 * want.abs() + (2 * d + 2.0 ** -15) * big).all())
        assert bool(((lse[b].double() - want_lse).abs() <= d + 4 * 2.0 ** -23 * (1 + want_lse.abs())).all())


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1, 8, 40, 100])
def test_many_sequences(device, n):
    """More units than CTAs, short and empty ones among them: ranges that cover several units."""
    g = torch.Generator().manual_seed(n)
    lens = [int(v) for v in torch.randint(n, 700, (70,), generator=g)]
    nodes = [int(v) for v in torch.randint(0, n + 1, (70,), generator=g)]
    x = Problem(device, lens, nodes, 4, n, "tree", seed=n)
    out, lse = x.ctx.tree_attention(x.q, x.mask, x.tree_lens)
    x.ctx.check_status()
    x.check(out, lse)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1, 6, 32, 70])
def test_long_sequence_is_cut_into_many_ranges(device, n):
    x = Problem(device, [40000], [n], 1, n, "tree", seed=n)
    out, lse = x.ctx.tree_attention(x.q, x.mask, x.tree_lens)
    x.check(out, lse)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1, 5, 24, 64])
def test_capture_streams_and_repeated_calls_change_no_bit(device, n):
    x = Problem(device, [1200, 90 + n], [n, n], 2, n, "tree", seed=n)
    out, lse = x.ctx.tree_attention(x.q, x.mask, x.tree_lens)
    mass = x.ctx.attention_mass(x.q, lse, x.ctx.new_mass(), x.mask, x.tree_lens)
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    side.wait_stream(torch.cuda.current_stream())
    o2, l2, m2 = torch.empty_like(out), torch.empty_like(lse), x.ctx.new_mass()
    with torch.cuda.stream(side):
        x.ctx.tree_attention(x.q, x.mask, x.tree_lens, out=o2, lse=l2)
        assert torch.equal(o2, out) and torch.equal(l2, lse)
        with torch.cuda.graph(graph, stream=side):
            m2.zero_()
            x.ctx.tree_attention(x.q, x.mask, x.tree_lens, out=o2, lse=l2)
            x.ctx.attention_mass(x.q, l2, m2, x.mask, x.tree_lens)
    torch.cuda.current_stream().wait_stream(side)
    for _ in range(3):
        o2.zero_()
        graph.replay()
        assert torch.equal(o2, out) and torch.equal(l2, lse) and torch.equal(m2, mass)
    # lengths and queries are read at replay
    x.lens = [v - 3 for v in x.lens] if n > 3 else [v - 1 for v in x.lens]
    x.cache.seq_lens.copy_(torch.tensor(x.lens, dtype=torch.int32))
    x.k, x.v = [k[:, :s] for k, s in zip(x.k, x.lens)], [v[:, :s] for v, s in zip(x.v, x.lens)]
    x.q.copy_(torch.randn_like(x.q.float()).bfloat16())
    graph.replay()
    x.check(o2, l2)


@pytest.mark.gpu
def test_two_contexts_on_two_streams(device):
    a, b = Problem(device, [9000], [5], 4, 5, seed=1), Problem(device, [7000, 300], [40, 40], 4, 40, seed=2)
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(5):
        with torch.cuda.stream(s1):
            r1 = a.ctx.tree_attention(a.q, a.mask, a.tree_lens)
        with torch.cuda.stream(s2):
            r2 = b.ctx.tree_attention(b.q, b.mask, b.tree_lens)
    torch.cuda.synchronize()
    a.check(*r1)
    b.check(*r2)


@pytest.mark.gpu
def test_one_token_is_the_sparse_step_with_a_full_budget(device):
    """decode_step attends everything where the budget is the whole sequence: the dense step on the same cache agrees."""
    from hashattention_b200 import synthetic
    x = Problem(device, [701, 300], [1, 1], 2, 1, seed=5)
    sparse = ha.SparseDecodeContext(x.cache, ha.Budget(128, 1.0, 128), synthetic.make_usa(8, D, seed=0, bf16=True).packed(device))
    k_new = torch.stack([k[:, -1] for k in x.k])
    v_new = torch.stack([v[:, -1] for v in x.v])
    want = sparse.decode_step(x.q[:, 0].contiguous(), k_new, v_new).double()
    out, lse = x.ctx.tree_attention(x.q)
    x.check(out, lse)
    # two bf16 outputs of the same sums, each within its half step
    assert bool(((out[:, 0].double() - want).abs() <= 2 * 2.0 ** -8 * want.abs() + 2e-4 * 5).all())


# ---- received weights -----------------------------------------------------------------------------------------------------
MASSES = [
    ([1], [1], 1, 1, False), ([700, 64, 65], [1, 1, 1], 1, 2, False), ([257, 2], [1, 1], 1, 8, False),
    ([300, 8], [5, 8], 8, 2, True), ([300, 8], [5, 8], 8, 2, False), ([1000, 40, 20], [13, 31, 0], 32, 1, True),
    ([2000], [64], 64, 1, False), ([700, 129], [100, 128], 128, 2, True), ([512], [128], 128, 1, False), ([20000], [3], 3, 1, False),
    ([5000, 333], [33, 20], 40, 2, False),
]


def accepted_words(x, seed):
    """Random node sets, one of them empty where there are several sequences."""
    g = torch.Generator().manual_seed(seed)
    sets = []
    for b, n in enumerate(x.nodes):
        s = torch.zeros(128, dtype=torch.bool)
        if b != 1:
            s[:n] = torch.rand(n, generator=g) < 0.4
            if n:
                s[n - 1] = True
        s[n:] = torch.rand(128 - n, generator=g) < 0.5  # bits behind the tree's end mean nothing
        sets.append(s)
    return torch.stack(sets)


@pytest.mark.gpu
@pytest.mark.parametrize("lens,nodes,width,kv_heads,some", MASSES)
def test_attention_mass(device, lens, nodes, width, kv_heads, some):
    x = Problem(device, lens, nodes, kv_heads, width, "tree", seed=width + 50, fused=width % 2 == 0)
    _, lse = x.ctx.tree_attention(x.q, x.mask, x.tree_lens)
    sets = accepted_words(x, width)
    rows = ha.pack_nodes(sets).to(device) if some else None
    start = torch.rand(x.ctx.mass_shape, device=device)
    mass = start.clone()
    for _ in range(2):  # it adds
        assert x.ctx.attention_mass(x.q, lse, mass, x.mask, x.tree_lens, rows=rows) is mass
    x.ctx.check_status()
    for b, n in enumerate(nodes):
        s = lens[b]
        assert torch.equal(mass[b, :, s:], start[b, :, s:]), "weights behind the sequence's end were written"
        if n == 0:
            assert torch.equal(mass[b], start[b])
            continue
        p, _ = weights64(x.q[b, :n], x.k[b], x.sees(b), x.scale)
        if some:
            p = p[sets[b, :n].to(device)]
        add = p.view(-1, kv_heads, GROUP, s).sum((0, 2)) if p.numel() else torch.zeros(kv_heads, s, dtype=torch.float64, device=device)
        want = start[b, :, :s].double() + 2 * add
        d = score_error(x.q[b, :n], x.k[b], x.scale)
        # both additions round the sum, and up to 512 weights are added up in fp32
        allowed = 2 * add * (2 * d + 2.0 ** -18 + 512 * 2.0 ** -24) + 2 * 2.0 ** -24 * want
        assert bool(((mass[b, :, :s].double() - want).abs() <= allowed).all()), b


@pytest.mark.gpu
def test_attention_mass_of_rows_that_see_nothing_and_of_masked_infinities(device):
    n = 9
    x = Problem(device, [n, 300], [n, n], 1, n, "tree", seed=8)
    bits = ha.unpack_nodes(x.mask.cpu())
    bits[0, 3:] = False
    x.visible[0][3:] = False
    x.mask = ha.pack_nodes(bits).to(device)
    x.k[0][0, n - 1, 7] = math.nan   # seen by none
    x.k[1][0, 299, 7] = math.inf     # seen by the last node alone, which is not counted
    x.write(0)
    x.write(1)
    _, lse = x.ctx.tree_attention(x.q, x.mask, x.tree_lens)
    rows = torch.ones(2, 128, dtype=torch.bool)
    rows[1, n - 1] = False
    mass = x.ctx.attention_mass(x.q, lse, x.ctx.new_mass(), x.mask, x.tree_lens, rows=ha.pack_nodes(rows).to(device))
    assert bool(torch.isfinite(mass).all())
    assert float(mass[0].sum()) == pytest.approx(3 * GROUP, rel=1e-4) and float(mass[1].sum()) == pytest.approx((n - 1) * GROUP, rel=1e-4)


# ---- trees: mask words, acceptance, commit -------------------------------------------------------------------------------------
def test_node_sets_pack_and_unpack():
    g = torch.Generator().manual_seed(1)
    for n in (1, 31, 32, 33, 64, 100, 128):
        bits = torch.rand(3, 2, n, generator=g) < 0.5
        words = ha.pack_nodes(bits)
        assert words.shape == (3, 2, 4) and torch.equal(ha.unpack_nodes(words, n), bits)
        assert not bool(ha.unpack_nodes(words)[..., n:].any())
    assert ha.pack_nodes(torch.ones(128, dtype=torch.bool)).tolist() == [-1] * 4
    with pytest.raises(ValueError):
        ha.pack_nodes(torch.ones(129, dtype=torch.bool))
    with pytest.raises(ValueError):
        ha.pack_nodes(torch.ones(5))


@pytest.mark.gpu
@pytest.mark.parametrize("nodes,width", [([1], 1), ([2, 1, 0], 2), ([31, 32, 33], 33), ([128, 64, 100], 128), ([7], 20)])
@pytest.mark.parametrize("shape", ["random", "chain", "star", "forest"])
def test_tree_mask(device, nodes, width, shape):
    g = torch.Generator().manual_seed(width)
    parents = torch.full((len(nodes), width), 99, dtype=torch.int32)  # what lies behind a tree's end means nothing
    trees = []
    for b, n in enumerate(nodes):
        tree = {"random": random_parents(n, g) if n else [], "chain": list(range(-1, n - 1)), "star": [-1] + [0] * (n - 1),
                "forest": [-1 if i % 3 == 0 else i - 1 for i in range(n)]}[shape][:n]
        trees.append(tree)
        parents[b, :n] = torch.tensor(tree, dtype=torch.int32)
    status = torch.zeros(1, dtype=torch.int32, device=device)
    words = ha.tree_mask(parents.to(device), torch.tensor(nodes, dtype=torch.int32, device=device), status=status)
    assert int(status) == 0
    bits = ha.unpack_nodes(words.cpu())
    for b, n in enumerate(nodes):
        assert torch.equal(bits[b, :n, :n], reach(trees[b]))
        assert not bool(bits[b, n:].any()) and not bool(bits[b, :, n:].any())


@pytest.mark.gpu
@pytest.mark.parametrize("bad", [3, 4, -2, 1000])
def test_tree_mask_reports_a_parent_behind_its_child(device, bad):
    parents = torch.tensor([[-1, 0, 1, bad, 3]], dtype=torch.int32, device=device)
    status = torch.zeros(1, dtype=torch.int32, device=device)
    words = ha.tree_mask(parents, status=status)
    assert int(status) == _lib.HA_ERR_BAD_ARG
    assert torch.equal(ha.unpack_nodes(words.cpu(), 5)[0], reach([-1, 0, 1, -1, 3]))


def accept64(parents, draft, target):
    path = [0] if parents else []
    while path:
        nxt = [i for i in range(path[-1] + 1, len(parents)) if parents[i] == path[-1] and draft[i] == target[path[-1]]]
        if not nxt:
            break
        path.append(nxt[0])
    return path


@pytest.mark.gpu
@pytest.mark.parametrize("nodes,width,vocab", [([1], 1, 2), ([5, 1, 0, 9], 9, 2), ([64, 33, 128, 100, 31], 128, 2), ([128] * 9, 128, 1), ([40] * 6, 50, 3)])
def test_tree_accept(device, nodes, width, vocab):
    """Few tokens in the vocabulary: long paths, and equal children of one node."""
    g = torch.Generator().manual_seed(width + vocab)
    B = len(nodes)
    parents = torch.full((B, width), -1, dtype=torch.int32)
    for b, n in enumerate(nodes):
        if n:
            parents[b, :n] = torch.tensor(random_parents(n, g) if b % 2 == 0 else list(range(-1, n - 1)), dtype=torch.int32)
    draft = torch.randint(0, vocab, (B, width), generator=g) + 2 ** 40
    target = torch.randint(0, vocab, (B, width), generator=g) + 2 ** 40
    lens = torch.tensor([n + 100 * b for b, n in enumerate(nodes)], dtype=torch.int32)
    got = ha.tree_accept(draft.to(device), parents.to(device), target.to(device), torch.tensor(nodes, dtype=torch.int32, device=device), lens.to(device))
    bits = ha.unpack_nodes(got.accepted.cpu())
    for b, n in enumerate(nodes):
        path = accept64(parents[b, :n].tolist(), draft[b].tolist(), target[b].tolist())
        assert bits[b].nonzero()[:, 0].tolist() == path and int(got.count[b]) == len(path)
        assert int(got.seq_lens[b]) == int(lens[b]) - n + len(path)
        if n:
            assert int(got.next_token[b]) == int(target[b, path[-1]])


def flat_rows(cache, b):
    """All slots of sequence b's pages: K, V, codes [Hkv, slots, ...]."""
    pages = cache.page_table[b].long()
    return [pool[pages].transpose(0, 1).flatten(1, 2) for pool in (cache.k_pages, cache.v_pages, cache.hash_pages)]


@pytest.mark.gpu
@pytest.mark.parametrize("lens,nodes,width", [([1], [1], 1), ([256, 257, 258], [3, 3, 3], 3), ([300, 20, 5], [60, 20, 0], 64),
                                              ([128, 383, 384, 600], [128, 128, 127, 100], 128), ([511, 513], [2, 33], 40)])
@pytest.mark.parametrize("kind", ["some", "all", "first", "last"])
@pytest.mark.parametrize("with_mass", [False, True])
def test_tree_commit(device, lens, nodes, width, kind, with_mass):
    x = Problem(device, lens, nodes, 2, width, seed=width)
    sets = accepted_words(x, 5)
    for b, n in enumerate(nodes):
        if kind != "some":
            sets[b] = False
            sets[b, {"all": slice(0, n), "first": slice(0, min(n, 1)), "last": slice(max(n - 1, 0), n)}[kind]] = True
    before = [flat_rows(x.cache, b) for b in range(x.B)]
    mass = torch.rand(x.ctx.mass_shape, device=device)
    old = mass.clone()
    x.ctx.tree_commit(ha.pack_nodes(sets).to(device), x.tree_lens, mass=mass if with_mass else None)
    x.ctx.check_status()
    assert x.cache.seq_lens.tolist() == lens
    for b, n in enumerate(nodes):
        P, path = lens[b] - n, sets[b, :n].nonzero()[:, 0].to(device)
        now = flat_rows(x.cache, b)
        for was, is_ in zip(before[b], now):
            want = was.clone()
            want[:, P:P + len(path)] = was[:, P + path]
            assert torch.equal(is_.view(torch.int16 if is_.dtype == torch.bfloat16 else torch.int32), want.view(torch.int16 if is_.dtype == torch.bfloat16 else torch.int32))
        want = old[b].clone()
        if with_mass and n:
            want[:, P:P + len(path)] = old[b][:, P + path]
            want[:, P + len(path):P + n] = 0
        assert torch.equal(mass[b], want)


# ---- eviction -------------------------------------------------------------------------------------------------------------------
def evict64(mass, S, keep, sink, recent):
    """Kept token numbers of one row of weights."""
    if S <= keep:
        return list(range(S))
    value = [float(v) if v > 0 else 0.0 for v in mass[sink:S - recent].tolist()]
    best = sorted(range(len(value)), key=lambda i: (-value[i], i))[:keep - sink - recent]
    return list(range(sink)) + sorted(i + sink for i in best) + list(range(S - recent, S))


EVICTIONS = [
    # lengths, keep, sink, recent
    ([700], 300, 16, 16), ([700, 300, 299, 301], 300, 4, 128), ([1, 0, 5, 6], 5, 0, 0), ([1000], 1, 0, 0), ([1000], 1, 1, 0),
    ([1000, 513], 512, 256, 256), ([3000, 2049, 800], 777, 128, 1), ([5000], 4999, 0, 0), ([257, 256, 255], 255, 0, 255),
    ([9001], 2048, 0, 128),
]


@pytest.mark.gpu
@pytest.mark.parametrize("lens,keep,sink,recent", EVICTIONS)
@pytest.mark.parametrize("weights", ["random", "ties", "odd"])
def test_cache_evict(device, lens, keep, sink, recent, weights):
    x = Problem(device, lens, [0] * len(lens), 2, 1, seed=keep)
    g = torch.Generator().manual_seed(keep + sink)
    mass = torch.rand(x.ctx.mass_shape, generator=g)
    if weights == "ties":
        mass = (mass * 3).floor() / 3  # zeros among them
    if weights == "odd":  # values that no accumulation of weights leaves, and the ends of the range
        pick = torch.randint(0, 8, mass.shape, generator=g)
        for i, v in enumerate([math.nan, -1.0, math.inf, 1e-45, 3e38, -0.0]):
            mass[pick == i] = v
    mass = mass.to(device)
    old = mass.clone()
    before = [flat_rows(x.cache, b) for b in range(x.B)]
    kept, mass_out, lens_out = x.ctx.cache_evict(mass, keep, sink, recent)
    x.ctx.check_status()
    assert torch.equal(mass.view(torch.int32), old.view(torch.int32)) and x.cache.seq_lens.tolist() == lens
    assert lens_out.tolist() == [min(s, keep) for s in lens]
    for b, s in enumerate(lens):
        now = flat_rows(x.cache, b)
        for h in range(2):
            index = evict64(old[b, h].cpu(), s, keep, sink, recent)
            n = len(index)
            assert kept[b, h, :n].tolist() == index and bool((kept[b, h, n:] == -1).all())
            at = torch.tensor(index, dtype=torch.long, device=device)
            assert torch.equal(mass_out[b, h, :n].view(torch.int32), old[b, h][at].view(torch.int32)) and bool((mass_out[b, h, n:] == 0).all())
            for was, is_ in zip(before[b], now):
                want = was[h].clone()
                want[:n] = was[h][at]
                kind = torch.int16 if is_.dtype == torch.bfloat16 else torch.int32
                assert torch.equal(is_[h].view(kind), want.view(kind)), (b, h)


@pytest.mark.gpu
@pytest.mark.parametrize("S,keep", [(40000, 10000), (400000, 50001)])
def test_cache_evict_of_long_rows(device, S, keep):
    """Rows of weights that the cluster holds in shared memory, and one that it does not; one kv-head."""
    cache = ha.PagedHashKVCache(1, 1, S, device, shuffle_seed=2)
    g = torch.Generator(device=device).manual_seed(1)
    cache.k_pages.copy_(torch.randn(cache.k_pages.shape, generator=g, device=device))
    cache.v_pages.copy_(torch.randn(cache.k_pages.shape, generator=g, device=device))
    cache.hash_pages.copy_(torch.randint(-2 ** 31, 2 ** 31 - 1, cache.hash_pages.shape, generator=g, device=device, dtype=torch.int32))
    cache.seq_lens.fill_(S)
    ctx = ha.DenseDecodeContext(cache)
    mass = (torch.rand(ctx.mass_shape, generator=g, device=device) * 5000).floor()
    before = flat_rows(cache, 0)
    kept, mass_out, lens_out = ctx.cache_evict(mass, keep, 128, 128)
    ctx.check_status()
    value = mass[0, 0, 128:S - 128]
    best = torch.sort(value, dim=0, descending=True, stable=True).indices[:keep - 256] + 128
    index = torch.cat([torch.arange(128, device=device), best.sort().values, torch.arange(S - 128, S, device=device)])
    assert torch.equal(kept[0, 0].long(), index) and torch.equal(mass_out[0, 0, :keep], mass[0, 0][index]) and lens_out.tolist() == [keep]
    for was, is_ in zip(before, flat_rows(cache, 0)):
        want = was.clone()
        want[:, :keep] = was[:, index]
        assert torch.equal(is_, want)


@pytest.mark.gpu
def test_cache_evict_repeated_and_captured(device):
    x = Problem(device, [900, 500], [0, 0], 2, 1, seed=4)
    mass = torch.rand(x.ctx.mass_shape, device=device)
    want = [t.clone() for t in x.ctx.cache_evict(mass, 400, 8, 8)]
    rows = [flat_rows(x.cache, b) for b in range(2)]
    y = Problem(device, [900, 500], [0, 0], 2, 1, seed=4)
    got = [torch.full_like(want[0], -1), torch.empty_like(mass), torch.empty_like(y.cache.seq_lens)]
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side), torch.cuda.graph(graph, stream=side):
        y.ctx.cache_evict(mass, 400, 8, 8, kept=got[0], mass_out=got[1], lens_out=got[2])
    torch.cuda.current_stream().wait_stream(side)
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    for b in range(2):
        for a, c in zip(rows[b], flat_rows(y.cache, b)):
            kind = torch.int16 if a.dtype == torch.bfloat16 else torch.int32
            assert torch.equal(a.view(kind), c.view(kind))


# ---- what is refused ----------------------------------------------------------------------------------------------------------
def test_entry_points_refuse_bad_arguments_before_launching():
    lib, N, X = _lib.load(), None, ctypes.c_void_p(256)  # X is never dereferenced: the checks come first
    good = _lib.HaShape(1, 2, 4, 128, 256, 4, 4, 1)
    tree, bad = _lib.HaTree(8, None, None), _lib.HA_ERR_BAD_ARG

    def attend(shape=good, t=tree, q=X, strides=None, scale=0.1, ws=X, n=1 << 40, out=X, mask=None):
        t = _lib.HaTree(t.max_nodes, None, mask) if mask else t
        return lib.ha_tree_attention(shape, t, q, (ctypes.c_int64 * 3)(*strides) if strides else None, X, X, X, X, scale, out, N, ws, n, X, N)

    def mass(shape=good, t=tree, q=X, lse=X, scale=0.1, m=X):
        return lib.ha_attention_mass(shape, t, q, None, lse, N, X, X, X, scale, m, X, N)

    for dim in (dict(head_dim=64), dict(gqa_group=8), dict(page_size=128)):
        s = _lib.HaShape(1, 2, 4, 128, 256, 4, 4, 1)
        for k, v in dim.items():
            setattr(s, k, v)
        assert attend(s) == mass(s) == _lib.HA_ERR_UNSUPPORTED_DIM
        assert lib.ha_tree_commit(s, tree, X, X, X, N, X, X, N, X, N) == _lib.HA_ERR_UNSUPPORTED_DIM
        assert lib.ha_cache_evict(s, 10, 1, 1, X, X, X, N, X, X, X, N, ctypes.c_void_p(512), X, 1 << 40, X, N) == _lib.HA_ERR_UNSUPPORTED_DIM
    assert attend(t=_lib.HaTree(129, None, None)) == mass(t=_lib.HaTree(129, None, None)) == _lib.HA_ERR_UNSUPPORTED_DIM
    assert attend(t=_lib.HaTree(0, None, None)) == mass(t=_lib.HaTree(-1, None, None)) == bad
    for scale in (0.0, -1.0, math.nan, math.inf):
        assert attend(scale=scale) == mass(scale=scale) == bad
    assert attend(q=N) == attend(out=N) == attend(q=ctypes.c_void_p(258)) == attend(strides=(8, 8, 4)) == attend(strides=(-8, 8, 8)) == bad
    assert attend(mask=264) == bad
    assert mass(q=N) == mass(lse=N) == mass(m=N) == bad
    assert attend(ws=N) == attend(n=100) == _lib.HA_ERR_WORKSPACE
    assert lib.ha_tree_workspace_bytes(0) == lib.ha_tree_workspace_bytes(129) == 0
    sizes = [lib.ha_tree_workspace_bytes(n) for n in (1, 4, 8, 32, 64, 128)]
    assert sizes == sorted(sizes) and sizes[0] > 0
    assert lib.ha_tree_mask(N, N, 1, 8, X, N, N) == lib.ha_tree_mask(X, N, 0, 8, X, N, N) == lib.ha_tree_mask(X, N, 1, 0, X, N, N) == bad
    assert lib.ha_tree_mask(X, N, 1, 129, X, N, N) == _lib.HA_ERR_UNSUPPORTED_DIM
    assert lib.ha_tree_accept(X, X, N, N, X, 1, 8, X, X, X, X, N, N) == bad
    assert lib.ha_tree_accept(X, X, X, N, X, 1, 129, X, X, X, X, N, N) == _lib.HA_ERR_UNSUPPORTED_DIM
    assert lib.ha_tree_commit(good, tree, N, X, X, N, X, X, N, X, N) == bad
    assert lib.ha_tree_commit(good, tree, ctypes.c_void_p(260), X, X, N, X, X, N, X, N) == bad

    def evict(keep=10, sink=1, recent=1, m=X, mo=N, lens=X, lo=ctypes.c_void_p(512), ws=X, n=1 << 40):
        return lib.ha_cache_evict(good, keep, sink, recent, m, X, X, N, X, lens, X, mo, lo, ws, n, X, N)

    assert evict(keep=0) == evict(sink=-1) == evict(recent=-1) == evict(sink=6, recent=5) == evict(mo=X) == evict(lo=X) == evict(m=N) == bad
    assert evict(ws=N) == evict(n=8) == _lib.HA_ERR_WORKSPACE
    assert evict(keep=2 ** 31 - 1, sink=2 ** 31 - 1, recent=2 ** 31 - 1) == bad


def test_python_refusals_on_cpu():
    cache = ha.PagedHashKVCache(1, 1, 256, "cpu")
    with pytest.raises(ValueError, match="CUDA"):
        ha.DenseDecodeContext(cache)
    with pytest.raises(ValueError, match="CUDA"):
        ha.tree_mask(torch.zeros(1, 4, dtype=torch.int32))
    with pytest.raises(ValueError, match="CUDA"):
        ha.tree_accept(*[torch.zeros(1, 4, dtype=torch.int64)] * 3, None, torch.zeros(1, dtype=torch.int32))


@pytest.mark.gpu
def test_python_refusals(device):
    x = Problem(device, [300, 300], [5, 5], 2, 5)
    ctx, q = x.ctx, x.q
    lse = torch.zeros(2, 5, 8, device=device)
    for bad in (q[:1], q[:, :, :4], q.float(), q.cpu(), q[..., ::2], torch.zeros(2, 6, 8, D, dtype=torch.bfloat16, device=device),
                torch.zeros(2, 5, 8, D + 4, dtype=torch.bfloat16, device=device)[..., :D],
                torch.zeros(2 * 5 * 8 * D + 1, dtype=torch.bfloat16, device=device)[1:].view(2, 5, 8, D)):
        with pytest.raises(ValueError):
            ctx.tree_attention(bad)
        with pytest.raises(ValueError):
            ctx.attention_mass(bad, lse, ctx.new_mass())
    for kw in (dict(tree_mask=x.mask[:, :4]), dict(tree_mask=x.mask.long()), dict(tree_lens=x.tree_lens[:1]), dict(tree_lens=x.tree_lens.long()),
               dict(out=torch.zeros(2, 5, 8, D, device=device)), dict(lse=lse.double()), dict(lse=lse.cpu()), dict(tree_mask=x.mask.cpu())):
        with pytest.raises(ValueError):
            ctx.tree_attention(q, **kw)
    for args in ((lse[:, :4], ctx.new_mass()), (lse, ctx.new_mass()[:, :1]), (lse, ctx.new_mass().double())):
        with pytest.raises(ValueError):
            ctx.attention_mass(q, *args)
    with pytest.raises(ValueError):
        ctx.attention_mass(q, lse, ctx.new_mass(), rows=torch.zeros(2, 3, dtype=torch.int32, device=device))
    with pytest.raises(ValueError):
        ctx.tree_commit(torch.zeros(2, 4, dtype=torch.int64, device=device))
    for args in ((0, 0, 0), (10, 6, 5), (10, -1, 0), (10, 0, -1)):
        with pytest.raises(ValueError):
            ctx.cache_evict(ctx.new_mass(), *args)
    m = ctx.new_mass()
    with pytest.raises(ValueError):
        ctx.cache_evict(m, 10, 0, 0, mass_out=m)
    with pytest.raises(ValueError):
        ctx.cache_evict(m, 10, 0, 0, lens_out=x.cache.seq_lens)
    for n in (0, 129):
        with pytest.raises(ValueError):
            ha.DenseDecodeContext(x.cache, n)
    for scale in (0.0, -1.0, math.nan, math.inf):
        with pytest.raises(ValueError):
            ha.DenseDecodeContext(x.cache, 1, sm_scale=scale)
    for parents in (torch.zeros(2, 129), torch.zeros(4), torch.zeros(0, 4), torch.zeros(2, 0)):
        with pytest.raises(ValueError):
            ha.tree_mask(parents.int().to(device))
    with pytest.raises(ValueError):
        ha.tree_accept(torch.zeros(2, 4, dtype=torch.int32, device=device), *[torch.zeros(2, 4, dtype=torch.int32, device=device)] * 2, None, x.cache.seq_lens)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1, 6, 20, 50])
def test_bad_pages_and_lengths_are_reported_and_leave_the_others_alone(device, n):
    """The kernels look at page ids and lengths before they touch memory: a bad one is reported in the status word."""
    x = Problem(device, [700, 300, 500], [n, n, n], 1, n, seed=n)
    out, lse = torch.zeros(3, n, 4, D, dtype=torch.bfloat16, device=device), torch.zeros(3, n, 4, device=device)
    for b_len, n_len in ((n - 1, n), (10 ** 9, n), (-5, n), (300, n + 1), (300, -1)):
        x.cache.seq_lens.copy_(torch.tensor([700, b_len, 500], dtype=torch.int32))
        x.tree_lens.copy_(torch.tensor([n, n_len, n], dtype=torch.int32))
        calls = [lambda: x.ctx.tree_attention(x.q, x.mask, x.tree_lens, out=out, lse=lse),
                 lambda: x.ctx.attention_mass(x.q, lse, x.ctx.new_mass(), x.mask, x.tree_lens),
                 lambda: x.ctx.tree_commit(torch.zeros(3, 4, dtype=torch.int32, device=device), x.tree_lens)]
        for call in calls:
            call()
            with pytest.raises(RuntimeError, match="status"):
                x.ctx.check_status()
        assert bool((out[1] == 0).all()) and bool((lse[1] == 0).all())
    x.cache.seq_lens.copy_(torch.tensor([700, 300, 500], dtype=torch.int32))
    x.tree_lens.fill_(n)
    for bad in (x.cache.num_pages, -1, 2 ** 31 - 1):
        table = x.cache.page_table.clone()
        x.cache.page_table[1, 0] = bad
        x.ctx.tree_attention(x.q, x.mask, x.tree_lens, out=out, lse=lse)
        with pytest.raises(RuntimeError, match="status"):
            x.ctx.check_status()
        x.ctx.attention_mass(x.q, lse, x.ctx.new_mass(), x.mask, x.tree_lens)
        with pytest.raises(RuntimeError, match="status"):
            x.ctx.check_status()
        x.cache.page_table.copy_(table)
        want, _ = attention64(x.q[0], x.k[0], x.v[0], x.sees(0), x.scale)
        assert bool(((out[0].double() - want).abs() <= 2.0 ** -8 * want.abs() + 5e-3).all())
    # eviction: a bad length is left as it is, a bad page's rows are not moved
    x.cache.seq_lens.copy_(torch.tensor([700, 10 ** 9, 500], dtype=torch.int32))
    kept, _, lens = x.ctx.cache_evict(torch.rand(x.ctx.mass_shape, device=device), 256, 4, 4)
    with pytest.raises(RuntimeError, match="status"):
        x.ctx.check_status()
    assert lens.tolist() == [256, 10 ** 9, 256] and bool((kept[1] == -1).all())
