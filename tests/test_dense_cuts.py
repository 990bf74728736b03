"""Dense attention and received weights over the paged cache where the work is cut over the CTAs in different ways: units that begin
a range of their own or not, more units than CTAs, more sequences than a warp has lanes, several groups of query rows; and what
the contexts share and refuse. Tolerances as in test_dense.py."""
import ctypes

import pytest
import torch

import hashattention_b200 as ha
from hashattention_b200 import _lib
from test_dense import D, GROUP, Problem, score_error, weights64


def check_mass(x, lse, mass):
    for b, n in enumerate(x.nodes):
        s = x.lens[b]
        assert bool((mass[b, :, s:] == 0).all())
        if n == 0:
            assert bool((mass[b] == 0).all())
            continue
        p, _ = weights64(x.q[b, :n], x.k[b], x.sees(b), x.scale)
        want = p.view(-1, x.hkv, GROUP, s).sum((0, 2))
        d = score_error(x.q[b, :n], x.k[b], x.scale)
        assert bool(((mass[b, :, :s].double() - want).abs() <= want * (2 * d + 2.0 ** -18 + 513 * 2.0 ** -24)).all()), b


def run(x):
    out, lse = x.ctx.tree_attention(x.q, x.mask, x.tree_lens)
    x.ctx.check_status()
    x.check(out, lse)
    mass = x.ctx.attention_mass(x.q, lse, x.ctx.new_mass(), x.mask, x.tree_lens)
    x.ctx.check_status()
    check_mass(x, lse, mass)


CUTS = [
    # lengths, drafts, kv-heads
    ([9001], [5], 8), ([9001], [40], 8), ([4099], [128], 8),                              # few equal units
    ([12000, 300, 5000], [9, 9, 30], 2), ([15000, 130, 64], [1, 1, 1], 8), ([12000, 129], [70, 3], 2),  # ragged ones
    ([700] * 32, [3] * 32, 4), ([700] * 32, [6] * 32, 4), ([700] * 33, [6] * 33, 4),      # nearly as many units as CTAs, 32 and 33 sequences
    ([130, 0, 2000] * 14, [40, 0, 12] * 14, 3), ([64, 65] * 40, [2, 1] * 40, 1),
    ([129] * 148, [5] * 148, 1), ([129] * 149, [5] * 149, 1),
]


@pytest.mark.gpu
@pytest.mark.parametrize("lens,nodes,kv_heads", CUTS)
def test_cuts(device, lens, nodes, kv_heads):
    run(Problem(device, lens, nodes, kv_heads, seed=len(lens) + nodes[0]))


@pytest.mark.gpu
@pytest.mark.parametrize("seed", range(24))
def test_drawn_shapes(device, seed):
    g = torch.Generator().manual_seed(1000 + seed)

    def draw(low, high):
        return int(torch.randint(low, high + 1, (1,), generator=g))

    width = draw(1, [4, 12, 32, 64, 128][seed % 5])
    batch, kv_heads = draw(1, [1, 4, 20, 40][seed % 4]), draw(1, 8)
    high = max(width, min(20000, 100000 // (batch * kv_heads)))
    nodes = [draw(0 if batch > 1 else 1, width) for _ in range(batch)]
    lens = [draw(max(n, 1), max(high, n, 1)) if n else draw(0, high) for n in nodes]
    if max(nodes) == 0:
        nodes[0], lens[0] = 1, max(lens[0], 1)
    run(Problem(device, lens, nodes, kv_heads, max(nodes), ["tree", "chain", "random"][seed % 3], seed=seed, fused=seed % 2 == 0))


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1, 5, 40])
@pytest.mark.parametrize("scale", [300.0, 5000.0])
def test_scores_of_many_thousands(device, n, scale):
    """One token has all of a row's weight: the references that weights are taken against must not be coarser than fp32's range
    allows (2^18 in powers of two here, where half an ulp of bf16 is 512)."""
    x = Problem(device, [n + 700, n], [n, n], 2, n, seed=n)
    x.ctx = ha.DenseDecodeContext(x.cache, n, sm_scale=scale)
    x.scale = x.ctx.sm_scale
    out, lse = x.ctx.tree_attention(x.q, x.mask, x.tree_lens)
    x.check(out, lse)


@pytest.mark.gpu
def test_contexts_that_share_workspaces(device):
    a, b = Problem(device, [3000], [20], 4, seed=1), Problem(device, [2500], [7], 4, seed=2)
    ctx = ha.DenseDecodeContext(b.cache, 7, workspace_of=a.ctx)
    assert ctx.workspace.data_ptr() == a.ctx.workspace.data_ptr() and ctx.evict_workspace.data_ptr() == a.ctx.evict_workspace.data_ptr()
    for _ in range(3):
        first = a.ctx.tree_attention(a.q, a.mask, a.tree_lens)
        second = ctx.tree_attention(b.q, b.mask, b.tree_lens)
    a.check(*first)
    b.check(*second)
    with pytest.raises(ValueError, match="workspace_of"):
        ha.DenseDecodeContext(a.cache, 64, workspace_of=ctx)  # (those of trees of up to 32 nodes)


@pytest.mark.gpu
def test_strides_of_single_sequences_and_nodes_mean_nothing(device):
    x = Problem(device, [500], [1], 2, seed=3)
    out, lse = x.ctx.tree_attention(x.q, x.mask, x.tree_lens)
    odd = x.q.as_strided(x.q.shape, (3, 5, D, 1))
    got = x.ctx.tree_attention(odd, x.mask, x.tree_lens)
    assert torch.equal(got[0], out) and torch.equal(got[1], lse)


def test_shapes_with_more_tiles_than_are_counted_are_refused():
    lib, X = _lib.load(), ctypes.c_void_p(256)  # (never dereferenced: the checks come first)
    tree = _lib.HaTree(128, None, None)
    for batch, heads, pages, ok in ((65535, 8, 65535, False), (4096, 8, 257, False), (1, 8, 65535, None)):
        shape = _lib.HaShape(batch, heads, 4, 128, 256, pages, 4, 1)
        # (a workspace that is too small is the next thing looked at)
        want = _lib.HA_ERR_WORKSPACE if ok is None else _lib.HA_ERR_UNSUPPORTED_DIM
        assert lib.ha_tree_attention(shape, tree, X, None, X, X, X, X, 0.1, X, None, X, 8, X, None) == want
        if ok is not None:
            assert lib.ha_attention_mass(shape, tree, X, None, X, None, X, X, X, 0.1, X, X, None) == want


@pytest.mark.gpu
def test_acceptance_does_not_write_the_lengths_that_the_commit_needs(device):
    x = Problem(device, [300], [4], 1, seed=1)
    out = ha.TreeAccept.empty(1, device)
    same = ha.TreeAccept(out.accepted, out.count, out.next_token, x.cache.seq_lens)
    tokens = torch.zeros(1, 4, dtype=torch.int64, device=device)
    with pytest.raises(ValueError, match="seq_lens"):
        ha.tree_accept(tokens, x.parents, tokens, x.tree_lens, x.cache.seq_lens, out=same)


def test_the_library_refuses_acceptance_over_the_lengths():
    lib, X, Y = _lib.load(), ctypes.c_void_p(256), ctypes.c_void_p(512)  # (never dereferenced)
    assert lib.ha_tree_accept(X, X, X, None, Y, 1, 8, X, X, X, Y, None, None) == _lib.HA_ERR_BAD_ARG
