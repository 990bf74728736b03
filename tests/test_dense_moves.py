"""What commit and eviction move, and what they leave alone: page ids and lengths that are out of range, rounds narrower than the
context, capacities far above the lengths. Rows are compared bit by bit."""
import ctypes

import pytest
import torch

import hashattention_b200 as ha
from hashattention_b200 import _lib
from test_dense import Problem, evict64, flat_rows


def pools(cache):
    """The three pools as integers (NaN compares)."""
    return [cache.k_pages.view(torch.int16).clone(), cache.v_pages.view(torch.int16).clone(), cache.hash_pages.clone()]


@pytest.mark.gpu
@pytest.mark.parametrize("bad", [-1, 2 ** 31 - 1, "num_pages"])
@pytest.mark.parametrize("which", [0, 1])
@pytest.mark.parametrize("owner", ["nobody", "a sequence"])
def test_commit_writes_nothing_where_a_page_id_is_out_of_range(device, bad, which, owner):
    """Drafts that cross from page 1 into page 2, one of the two ids out of range: no pool row changes, physical page 0 included,
    and the sequences beside it are committed."""
    n = 9
    x = Problem(device, [515, 300, 515], [n, n, n], 2, n, seed=11)
    table = x.cache.page_table
    spare = sorted(set(range(x.cache.num_pages)) - set(table.flatten().tolist()))
    # physical page 0: nobody's, or page 0 of the last sequence (the pool's pages change places with their contents)
    zero = (table == 0).nonzero()
    if owner == "a sequence":
        if len(zero):
            b, i = zero[0].tolist()
            table[b, i] = table[2, 0]
        table[2, 0] = 0
    elif len(zero):
        b, i = zero[0].tolist()
        table[b, i] = spare[0] if spare[0] != 0 else spare[1]
    for b in range(3):
        x.write(b)
    table[0, 1 + which] = x.cache.num_pages if bad == "num_pages" else bad
    bits = torch.zeros(3, 128, dtype=torch.bool)
    bits[0, [2, 5, 8]] = True   # moves in the sequence with the bad page
    bits[1, [1, 3, 7]] = True   # moves beside it
    bits[2, 0] = True           # moves nothing
    mass = torch.rand(x.ctx.mass_shape, device=device)
    before, old = pools(x.cache), mass.clone()
    x.ctx.tree_commit(ha.pack_nodes(bits).to(device), x.tree_lens, mass=mass)
    with pytest.raises(RuntimeError, match=rf"status {_lib.HA_ERR_BAD_PAGE}\)"):
        x.ctx.check_status()
    own = table[1].tolist()
    P = 300 - n
    for was, now in zip(before, pools(x.cache)):
        others = [i for i in range(x.cache.num_pages) if i not in own]
        assert torch.equal(now[others], was[others]), "rows of another sequence were moved"
        flat_was, flat_now = was[own].transpose(0, 1).flatten(1, 2), now[own].transpose(0, 1).flatten(1, 2)
        want = flat_was.clone()
        want[:, P:P + 3] = flat_was[:, [P + 1, P + 3, P + 7]]
        assert torch.equal(flat_now, want)
    assert torch.equal(mass[0], old[0]), "the received weights moved without their rows"


@pytest.mark.gpu
def test_commit_without_tree_lens_needs_the_nodes_of_the_round(device):
    """A context for 32 nodes in a round of 8 without tree_lens: attention and acceptance go by the round's width, and so does the
    commit, which cannot know it from the words of the accepted path."""
    T, S = 8, 300
    x = Problem(device, [S, 200], [T, T], 2, T, "tree", seed=3)
    ctx = ha.DenseDecodeContext(x.cache, 32)
    out, lse = ctx.tree_attention(x.q, x.mask)
    x.check(out, lse)
    bits = torch.zeros(2, 128, dtype=torch.bool)
    bits[0, [0, 2, 5]] = bits[1, [0, 7]] = True
    words, mass = ha.pack_nodes(bits).to(device), torch.rand(ctx.mass_shape, device=device)
    before, old = [flat_rows(x.cache, b) for b in range(2)], mass.clone()
    with pytest.raises(ValueError, match="max_nodes"):
        ctx.tree_commit(words, mass=mass)
    for bad in (0, 33, -1):
        with pytest.raises(ValueError, match="max_nodes"):
            ctx.tree_commit(words, mass=mass, max_nodes=bad)
    ctx.tree_commit(words, mass=mass, max_nodes=T)
    ctx.check_status()
    for b, path in enumerate(([0, 2, 5], [0, 7])):
        P = x.lens[b] - T
        path = torch.tensor(path, device=device)
        for was, now in zip(before[b], flat_rows(x.cache, b)):
            want = was.clone()
            want[:, P:P + len(path)] = was[:, P + path]
            kind = torch.int16 if now.dtype == torch.bfloat16 else torch.int32
            assert torch.equal(now.view(kind), want.view(kind))
        want = old[b].clone()
        want[:, P:P + len(path)] = old[b][:, P + path]
        want[:, P + len(path):P + T] = 0
        assert torch.equal(mass[b], want)
    # a context for one node has one width only
    one = ha.DenseDecodeContext(x.cache, 1)
    one.tree_commit(torch.ones(2, 4, dtype=torch.int32, device=device))
    one.check_status()


@pytest.mark.gpu
def test_eviction_keeps_the_weights_of_a_sequence_whose_length_is_out_of_range(device):
    x = Problem(device, [700, 300, 500], [0, 0, 0], 2, 1, seed=2)
    mass = torch.rand(x.ctx.mass_shape, device=device)
    for bad in (10 ** 9, -5):
        x.cache.seq_lens[1] = bad
        before = pools(x.cache)
        kept, mass_out, lens = x.ctx.cache_evict(mass, 600, 4, 4)  # (the others: one is cut, one is not)
        with pytest.raises(RuntimeError, match=rf"status {_lib.HA_ERR_BAD_SEQ_LEN}\)"):
            x.ctx.check_status()
        assert lens.tolist() == [600, bad, 500] and bool((kept[1] == -1).all())
        assert torch.equal(mass_out[1], mass[1])
        assert torch.equal(mass_out[2, :, :500], mass[2, :, :500]) and bool((mass_out[2, :, 500:] == 0).all())
        own = x.cache.page_table[1].tolist()
        for was, now in zip(before, pools(x.cache)):
            assert torch.equal(now[own], was[own])


@pytest.mark.gpu
@pytest.mark.parametrize("bad", [-1, 2 ** 31 - 1])
def test_eviction_moves_no_row_from_or_to_a_page_out_of_range(device, bad):
    """Page ids out of range as source and as destination: what lies there stays, all other kept rows move, and other
    sequences' pages (physical page 0 among them) are as if nothing had been wrong."""
    lens, keep = [900, 800], 300
    x = Problem(device, lens, [0, 0], 2, 1, seed=9)
    y = Problem(device, lens, [0, 0], 2, 1, seed=9)  # the same without bad ids
    mass = torch.rand(x.ctx.mass_shape, device=device)
    table = x.cache.page_table.clone()
    for page in (0, 2):  # (tokens 0 .. 255: destinations, 512 .. 767: sources)
        x.cache.page_table.copy_(table)
        for b in range(2):
            x.write(b)
            y.write(b)
        x.cache.hash_pages.copy_(y.cache.hash_pages)
        x.cache.page_table[0, page] = bad
        before = pools(x.cache)
        kept, _, _ = x.ctx.cache_evict(mass, keep, 8, 8)
        with pytest.raises(RuntimeError, match=rf"status {_lib.HA_ERR_BAD_PAGE}\)"):
            x.ctx.check_status()
        y.ctx.cache_evict(mass, keep, 8, 8)
        y.ctx.check_status()
        other = table[1].tolist()
        for was, now, good in zip(before, pools(x.cache), pools(y.cache)):
            assert torch.equal(now[other], good[other])
            rest = [i for i in range(x.cache.num_pages) if i not in table.flatten().tolist()]
            assert torch.equal(now[rest], was[rest]) and torch.equal(now[int(table[0, page])], was[int(table[0, page])])
            for h in range(2):
                rows_was = was[table[0].long(), h].flatten(0, 1)
                want = rows_was.clone()
                for i, t in enumerate(kept[0, h].tolist()):
                    if t != i and t // 256 != page and i // 256 != page:
                        want[i] = rows_was[t]
                assert torch.equal(now[table[0].long(), h].flatten(0, 1), want)


@pytest.mark.gpu
@pytest.mark.parametrize("lens,keep", [([4000], 1000), ([700, 300, 20], 256), ([9000, 8192, 100], 8000)])
def test_eviction_of_sequences_far_below_the_capacity(device, lens, keep):
    """Pages for 131072 tokens a sequence: the cluster's form of the selection on rows that fill a part of it, or one CTA of it only."""
    cache = ha.PagedHashKVCache(len(lens), 2, 131072, device, shuffle_seed=4)
    g = torch.Generator(device=device).manual_seed(1)
    for pool in (cache.k_pages, cache.v_pages):
        pool.view(torch.int16).random_(-2 ** 15, 2 ** 15, generator=g)
    cache.hash_pages.random_(-2 ** 31, 2 ** 31 - 1, generator=g)
    cache.seq_lens.copy_(torch.tensor(lens, dtype=torch.int32))
    ctx = ha.DenseDecodeContext(cache)
    mass = torch.rand(ctx.mass_shape, generator=g, device=device)
    before = [[r.clone() for r in flat_rows(cache, b)] for b in range(len(lens))]
    kept, mass_out, lens_out = ctx.cache_evict(mass, keep, 16, 16)
    ctx.check_status()
    assert lens_out.tolist() == [min(s, keep) for s in lens]
    for b, s in enumerate(lens):
        now = flat_rows(cache, b)
        for h in range(2):
            index = evict64(mass[b, h].cpu(), s, keep, 16, 16)
            n = len(index)
            assert kept[b, h, :n].tolist() == index and bool((kept[b, h, n:] == -1).all())
            at = torch.tensor(index, device=device)
            assert torch.equal(mass_out[b, h, :n], mass[b, h][at]) and bool((mass_out[b, h, n:] == 0).all())
            for was, is_ in zip(before[b], now):
                want = was[h].clone()
                want[:n] = was[h][at]
                kind = torch.int16 if is_.dtype == torch.bfloat16 else torch.int32
                assert torch.equal(is_[h].view(kind), want.view(kind))


def test_pools_with_more_rows_than_are_numbered_are_refused():
    """2^31 rows of K (512 GB): row numbers are 32 bits."""
    lib, X = _lib.load(), ctypes.c_void_p(256)  # (never dereferenced: the checks come first)
    tree = _lib.HaTree(8, None, None)
    for pages, want in ((2 ** 20, _lib.HA_ERR_UNSUPPORTED_DIM), (2 ** 20 - 1, _lib.HA_ERR_WORKSPACE)):
        shape = _lib.HaShape(1, 8, 4, 128, 256, 4, pages, 1)
        # (a workspace that is too small is the next thing looked at, by those that take one)
        assert lib.ha_tree_attention(shape, tree, X, None, X, X, X, X, 0.1, X, None, X, 8, X, None) == want
        if want == _lib.HA_ERR_UNSUPPORTED_DIM:
            assert lib.ha_attention_mass(shape, tree, X, None, X, None, X, X, X, 0.1, X, X, None) == want
            assert lib.ha_cache_evict(shape, 10, 1, 1, X, X, X, None, X, X, X, None, ctypes.c_void_p(512), X, 1 << 40, X, None) == want
