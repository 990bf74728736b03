"""What a round of drafts and an eviction leave of a model's state (llama_tp.py): sequences whose drafts do not fit their cache, lengths
that are out of range, sequences without drafts, and graphs captured before an eviction."""
import pytest
import torch


def _cfg(**more):
    from hashattention_b200 import llama_tp
    return llama_tp.LlamaTPConfig(n_layers=2, dim=256, ffn_dim=512, vocab_size=1000, max_seq_len=700, **more)  # (768 tokens)


def _model(device, batch, nodes, mass=False, **more):
    from hashattention_b200 import llama_tp
    model = llama_tp.TPLlama(_cfg(**more), 1, 0, device, batch=batch, seed=1)
    model.enable_trees(nodes, mass=mass)
    return model


def _state(model):
    """Everything a round may change, the pools as integers."""
    pools = []
    for ctx in model.ctxs:
        c = ctx.cache
        pools.append([c.k_pages.view(torch.int16).clone(), c.v_pages.view(torch.int16).clone(), c.hash_pages.clone()])
    return dict(pools=pools, mass=None if model.mass is None else [m.clone() for m in model.mass], lens=model.seq_lens.tolist(),
                pos=model.pos.tolist())


def _assert_left_alone(model, before, b):
    """Sequence b is as it was: its pages, received weights, length and position."""
    now = _state(model)
    own = model.ctxs[0].cache.page_table[b].long()
    for was, is_ in zip(before["pools"], now["pools"]):
        for p, q in zip(was, is_):
            assert torch.equal(p[own], q[own]), "a token of the cache was overwritten"
    if before["mass"] is not None:
        assert all(torch.equal(m[b], k[b]) for m, k in zip(before["mass"], now["mass"]))
    assert now["lens"][b] == before["lens"][b] and now["pos"][b] == before["pos"][b]


def _prefilled(model, lens, seed=3):
    """Prefills the longest length, then takes shorter ones for the others (their tokens are a prefix of the same prompt)."""
    from hashattention_b200 import llama_tp
    model.prefill(llama_tp.tokens_for(model.cfg, model.batch, max(lens), seed=seed).to(model.device))
    model.seq_lens.copy_(torch.tensor(lens, dtype=torch.int32))
    model.pos.copy_(torch.tensor(lens))


def _chain(B, T, device):
    return torch.arange(-1, T - 1, dtype=torch.int32, device=device).repeat(B, 1)


@pytest.mark.gpu
@pytest.mark.parametrize("full", [768, 767, 761])
def test_drafts_that_do_not_fit_are_reported_and_change_nothing(device, full):
    """8 drafts behind 761 and more of 768 tokens: that sequence takes no part in the round and can be evicted and go on; the
    sequence beside it gives, bit by bit, what it gives where the full one has no drafts."""
    from hashattention_b200 import _lib
    T = 8
    draft = torch.randint(0, 1000, (2, T), generator=torch.Generator().manual_seed(2)).to(device)
    results = []
    for tree_lens in ([T, T], [0, T]):
        model = _model(device, 2, T, mass=True, init_budget=16, recent_budget=16)
        _prefilled(model, [full, 300])
        for m in model.mass:
            m.copy_(torch.rand(m.shape, generator=torch.Generator().manual_seed(6)))
        before = _state(model)
        got = model.verify_tree(draft, _chain(2, T, device), torch.tensor(tree_lens, dtype=torch.int32, device=device))
        results.append((got, _state(model), model.ctxs[0].cache.page_table[1].long()))
        if tree_lens[0]:
            with pytest.raises(RuntimeError, match=rf"status {_lib.HA_ERR_BAD_SEQ_LEN}\)"):
                model.check_status()
            _assert_left_alone(model, before, 0)
            assert int(got.count[0]) == 0 and not bool(got.accepted[0].any()) and int(got.seq_lens[0]) == full
            assert int(got.next_token[0]) == int(draft[0, 0])  # still the token that is certain
            # after an eviction the same drafts fit
            model.evict(400)
            assert model.seq_lens.tolist()[0] == 400
            again = model.verify_tree(draft, _chain(2, T, device))
            model.check_status()
            assert int(again.count[0]) >= 1 and int(model.pos[0]) == full + int(again.count[0])
        else:
            model.check_status()
    (a, sa, own), (b, sb, _) = results
    assert torch.equal(a.accepted[1], b.accepted[1]) and int(a.next_token[1]) == int(b.next_token[1])
    assert sa["lens"][1] == sb["lens"][1] == 300 + int(a.count[1]) and sa["pos"][1] == sb["pos"][1]
    for p, q in zip(sa["pools"], sb["pools"]):
        for s, t in zip(p, q):
            assert torch.equal(s[own], t[own])


@pytest.mark.gpu
def test_drafts_that_just_fit_are_taken(device):
    model = _model(device, 1, 8)
    _prefilled(model, [760])
    got = model.verify_tree(torch.zeros(1, 8, dtype=torch.int64, device=device), _chain(1, 8, device))
    model.check_status()
    assert int(got.count[0]) >= 1 and model.seq_lens.tolist() == [760 + int(got.count[0])]


@pytest.mark.gpu
@pytest.mark.parametrize("bad", [9, -1, 2 ** 31 - 1])
def test_tree_lens_out_of_range_are_reported_and_change_nothing(device, bad):
    from hashattention_b200 import _lib
    model = _model(device, 2, 8, mass=True)
    _prefilled(model, [300, 300])
    before = _state(model)
    draft = torch.randint(0, 1000, (2, 8), generator=torch.Generator().manual_seed(2)).to(device)
    got = model.verify_tree(draft, _chain(2, 8, device), torch.tensor([bad, 5], dtype=torch.int32, device=device))
    with pytest.raises(RuntimeError, match=rf"status {_lib.HA_ERR_BAD_SEQ_LEN}\)"):
        model.check_status()
    _assert_left_alone(model, before, 0)
    assert got.count.tolist()[0] == 0 and int(got.next_token[0]) == int(draft[0, 0])
    assert int(got.count[1]) >= 1 and model.seq_lens.tolist() == [300, 300 + int(got.count[1])]
    with pytest.raises(ValueError, match="tree_lens"):
        model.verify_tree(draft, _chain(2, 8, device), torch.ones(2, dtype=torch.int64, device=device))


@pytest.mark.gpu
def test_next_token_of_a_sequence_without_drafts(device):
    """Where nothing was drafted there is no token behind the last accepted one: node 0's stays the next one in a model's round (the
    embedding takes it), and acceptance by itself gives 0 in tensors of its own and leaves given ones alone."""
    import hashattention_b200 as ha
    model = _model(device, 3, 4)
    _prefilled(model, [50, 40, 30])
    draft = torch.randint(0, 1000, (3, 4), generator=torch.Generator().manual_seed(2)).to(device)
    lens = torch.tensor([4, 0, 1], dtype=torch.int32, device=device)
    torch.full((4096,), -7, dtype=torch.int64, device=device)  # (freed: what the allocator hands out next)
    got = model.verify_tree(draft, _chain(3, 4, device), lens)
    model.check_status()
    assert got.count.tolist()[1] == 0 and int(got.next_token[1]) == int(draft[1, 0])
    nxt = torch.empty(3, dtype=torch.int64, device=device)
    model.decode_step(got.next_token, nxt)
    model.check_status()
    args = (draft, _chain(3, 4, device), draft, lens, model.seq_lens)
    for size in (1, 3, 64, 512):
        torch.full((size,), -7, dtype=torch.int64, device=device)
    assert int(ha.tree_accept(*args).next_token[1]) == 0
    out = ha.TreeAccept.empty(3, device)
    out.next_token.fill_(77)
    assert int(ha.tree_accept(*args, out=out).next_token[1]) == 77


@pytest.mark.gpu
def test_a_round_captured_before_an_eviction_goes_on_after_it(device):
    """The received weights stay in the tensors that a captured round adds to: replayed after an eviction it gives what the eager
    round gives."""
    B, T = 2, 6
    draft = torch.randint(0, 1000, (B, T), generator=torch.Generator().manual_seed(2)).to(device)
    parents, tree_lens = _chain(B, T, device), torch.tensor([T, 3], dtype=torch.int32, device=device)
    ends = []
    for captured in (False, True):
        model = _model(device, B, T, mass=True, init_budget=16, recent_budget=16)
        _prefilled(model, [500, 450])
        for m in model.mass:
            m.copy_(torch.rand(m.shape, generator=torch.Generator().manual_seed(6)))
        where = [m.data_ptr() for m in model.mass]
        if captured:
            start = [t.clone() for t in [model.seq_lens, model.pos] + model.mass]
            model.verify_tree(draft, parents, tree_lens)  # (warm-up; the drafts' rows are written again)
            graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side), torch.cuda.graph(graph, stream=side):
                got = model.verify_tree(draft, parents, tree_lens)
            torch.cuda.current_stream().wait_stream(side)
            for t, s in zip([model.seq_lens, model.pos] + model.mass, start):
                t.copy_(s)
        for keep in (300, 200):
            model.evict(keep)
            # (in front of any replay: a graph must not be run on tensors that are gone)
            assert [m.data_ptr() for m in model.mass] == where, "the received weights moved"
            assert model.seq_lens.tolist() == [keep] * B
            if captured:
                graph.replay()
            else:
                got = model.verify_tree(draft, parents, tree_lens)
        model.check_status()
        ends.append((got.accepted.tolist(), got.count.tolist(), got.next_token.tolist(), _state(model), model))
    (a, b) = ends
    assert a[:3] == b[:3] and a[3]["lens"] == b[3]["lens"] and a[3]["pos"] == b[3]["pos"]
    for m, k in zip(a[3]["mass"], b[3]["mass"]):
        assert torch.equal(m, k) and float(m.sum()) > 0


@pytest.mark.gpu
def test_an_eviction_can_be_captured_with_its_round(device):
    """Eviction and round in one graph, replayed: the cache stays at its budget and the received weights in their place."""
    B, T, keep = 2, 4, 128
    model = _model(device, B, T, mass=True, init_budget=16, recent_budget=16)
    _prefilled(model, [300, 200])
    draft = torch.randint(0, 1000, (B, T), generator=torch.Generator().manual_seed(2)).to(device)
    parents = _chain(B, T, device)
    model.verify_tree(draft, parents)
    model.evict(keep)
    where = [m.data_ptr() for m in model.mass]
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side), torch.cuda.graph(graph, stream=side):
        got = model.verify_tree(draft, parents)
        model.evict(keep)
    torch.cuda.current_stream().wait_stream(side)
    assert [m.data_ptr() for m in model.mass] == where
    pos = model.pos.tolist()
    for _ in range(3):
        graph.replay()
        pos = [p + c for p, c in zip(pos, got.count.tolist())]
        assert model.pos.tolist() == pos and model.seq_lens.tolist() == [keep] * B
    model.check_status()
    for m in model.mass:
        assert bool((m[:, :, keep:] == 0).all()) and bool(torch.isfinite(m).all())
