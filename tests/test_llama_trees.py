"""Trees of drafted tokens and eviction on the tensor-parallel Llama host (llama_tp.py): the operators of dense.py in one run, as a
serving loop uses them - prompt, verification of a tree, commit, the next tree, a sparse step, eviction - against a plain
forward pass of the same weights in 64 bits.

Tolerance of the logits. The model computes in bf16: a layer rounds its values 13 times (norm, projection, rotary, stored K and V,
attention, output projection, residual; norm, projection, silu, product, projection, residual), the embedding's norm and the
head 3 times more, each by 2^-8 of the value at most. Two layers: 29 roundings, 29 * 2^-8 = 0.113 of the norm."""
import pytest
import torch

TOL = 29 * 2.0 ** -8


def _cfg(**more):
    from hashattention_b200 import llama_tp
    return llama_tp.LlamaTPConfig(n_layers=2, dim=256, ffn_dim=512, vocab_size=1000, max_seq_len=700, **more)


def forward64(weights, cfg, tokens, pos, visible):
    """Logits [n, vocab] of one sequence in 64 bits: tokens, positions [n], visible [n, n] (row i sees column j)."""
    D, Hq, Hkv = cfg.head_dim, cfg.n_heads, cfg.n_kv_heads

    def norm(x):
        return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + cfg.norm_eps)

    def rope(x):  # [n, heads, D]
        ang = pos.double()[:, None] / cfg.rope_theta ** (torch.arange(0, D, 2).double() / D)
        cos, sin = torch.cat([ang.cos()] * 2, -1)[:, None], torch.cat([ang.sin()] * 2, -1)[:, None]
        return x * cos + torch.cat([-x[..., D // 2:], x[..., :D // 2]], -1) * sin

    x = weights["embed"][tokens]
    for wqkv, wo, w13, w2 in weights["layers"]:
        q, k, v = (norm(x) @ wqkv.T).split([Hq * D, Hkv * D, Hkv * D], -1)
        q, k, v = rope(q.view(-1, Hq, D)), rope(k.view(-1, Hkv, D)), v.view(-1, Hkv, D)
        k, v = k.repeat_interleave(Hq // Hkv, 1), v.repeat_interleave(Hq // Hkv, 1)
        s = torch.einsum("nhd,mhd->hnm", q, k) / D ** 0.5
        p = torch.softmax(torch.where(visible, s, torch.full_like(s, -torch.inf)), -1)
        x = x + torch.einsum("hnm,mhd->nhd", p, v).reshape(len(x), -1) @ wo.T
        a, b = (norm(x) @ w13.T).chunk(2, -1)
        x = x + (torch.nn.functional.silu(a) * b) @ w2.T
    return norm(x) @ weights["head"].T


def weights64(model):
    def c(w):
        return w.detach().cpu().double()
    return {"embed": c(model.embed), "head": c(model.head),
            "layers": [(c(w.wqkv), c(w.wo), c(w.w13), c(w.w2)) for w in model.layers]}


def tree_inputs(path, tree_tokens, parents):
    """Tokens, positions and sight of a sequence: the path so far, then a tree behind it."""
    S, n = len(path), len(tree_tokens)
    visible = torch.ones(S + n, S + n, dtype=torch.bool).tril()
    pos = list(range(S))
    for i, p in enumerate(parents):
        up, j = set(), i
        while j >= 0:
            up.add(j)
            j = parents[j]
        visible[S + i, S:] = torch.tensor([j in up for j in range(n)])
        pos.append(S + len(up) - 1)
    return torch.tensor(list(path) + list(tree_tokens)), torch.tensor(pos), visible


def off(got, want):
    return float((got.double().cpu() - want).norm() / want.norm())


PARENTS = [-1, 0, 0, 1, 1, 2, 5, 3, 0]


def test_trees_are_refused_on_a_model_without_a_paged_cache():
    from hashattention_b200 import llama_tp
    model = llama_tp.TPLlama(llama_tp.LlamaTPConfig(n_layers=1, dim=64, ffn_dim=128, vocab_size=64, max_seq_len=64), 1, 0, "cpu", 1,
                             attention=lambda *a: None, dtype=torch.float32)
    with pytest.raises(ValueError, match="paged cache"):
        model.enable_trees(4)
    with pytest.raises(ValueError, match="enable_trees"):
        model.verify_tree(torch.zeros(1, 1, dtype=torch.int64), torch.full((1, 1), -1, dtype=torch.int32))
    with pytest.raises(ValueError, match="enable_trees"):
        model.evict(8)
    with pytest.raises(ValueError, match="observe"):
        model.prefill(torch.zeros(1, 4, dtype=torch.int64), observe=2)


@pytest.mark.gpu
@pytest.mark.parametrize("prompt", [6, 250])
def test_tree_logits_of_two_rounds_and_the_sparse_step_between(device, prompt):
    """Logits of a tree, of a second tree behind the accepted path, and of one behind a sparse step, all against the plain model;
    with a chain's sight in place of the tree's the oracle itself is further off than the tolerance (where the tree matters)."""
    from hashattention_b200 import llama_tp, pack_nodes, tree_mask
    cfg = _cfg()
    model = llama_tp.TPLlama(cfg, 1, 0, device, batch=2, seed=1)
    model.enable_trees(len(PARENTS))
    w = weights64(model)
    prompts = llama_tp.tokens_for(cfg, 2, prompt, seed=3)
    model.prefill(prompts.to(device))
    paths = [p.tolist() for p in prompts]
    gen = torch.Generator().manual_seed(5)
    for turn, nodes in enumerate(([9, 4], [3, 9])):
        tree_lens = torch.tensor(nodes, dtype=torch.int32, device=device)
        parents = torch.tensor([PARENTS] * 2, dtype=torch.int32, device=device)
        draft = torch.randint(0, cfg.vocab_size, (2, len(PARENTS)), generator=gen)
        before = model.seq_lens.clone()
        mask = tree_mask(parents, tree_lens)
        logits, _ = model._tree_forward(draft.to(device), mask, tree_lens)
        assert model.seq_lens.tolist() == [len(p) + n for p, n in zip(paths, nodes)]
        model.seq_lens.copy_(before)
        target = []
        for b in range(2):
            n, S = nodes[b], len(paths[b])
            tokens, pos, visible = tree_inputs(paths[b], draft[b, :n].tolist(), PARENTS[:n])
            want = forward64(w, cfg, tokens, pos, visible)[S:]
            assert off(logits[b, :n], want) < TOL
            if prompt < 10 and n == 9:
                chain = forward64(w, cfg, tokens, pos, torch.ones(S + n, S + n, dtype=torch.bool).tril())[S:]
                assert off(chain, want) > 1.5 * TOL
            target.append(logits[b].float().argmax(-1).cpu())
        # drafts that agree with the model along 0 - 2 - 5 (as far as the tree goes): the path is accepted and stays
        agreed = draft.clone()
        for b in range(2):
            for node, parent in ((2, 0), (5, 2)):
                agreed[b, node] = target[b][parent]
            for node in (1, 8):
                agreed[b, node] = (target[b][0] + 1) % cfg.vocab_size
        # (node 2's token has changed, and with it what the model puts behind it: from here on what the call itself returns counts)
        got = model.verify_tree(agreed.to(device), parents, tree_lens)
        count, accepted = got.count.tolist(), got.accepted
        for b in range(2):
            bits = [j for j in range(nodes[b]) if (int(accepted[b, 0]) >> j) & 1]
            assert len(bits) == count[b] and bits[:2] == [0, 2]
            assert torch.equal(accepted[b].cpu(), pack_nodes(torch.tensor([[j in bits for j in range(9)]]))[0])
            paths[b] += [int(agreed[b, j]) for j in bits]
        assert model.seq_lens.tolist() == model.pos.tolist() == [len(p) for p in paths]
        # a sparse step: with these lengths its budget covers every token
        nxt = torch.empty(2, dtype=torch.int64, device=device)
        model.decode_step(got.next_token, nxt)
        for b in range(2):
            paths[b].append(int(got.next_token[b]))
    model.check_status()
    # one node: the dense step
    one = torch.full((2, 1), -1, dtype=torch.int32, device=device)
    draft = nxt[:, None].contiguous()
    logits, _ = model._tree_forward(draft, tree_mask(one), torch.ones(2, dtype=torch.int32, device=device))
    for b in range(2):
        tokens, pos, visible = tree_inputs(paths[b], [int(nxt[b])], [-1])
        assert off(logits[b], forward64(w, cfg, tokens, pos, visible)[-1:]) < TOL
    model.check_status()


@pytest.mark.gpu
def test_received_weights_and_eviction_in_a_serving_loop(device):
    """Every counted row hands out a weight of one per query head; after eviction the lengths are the budget's, positions go on,
    the next rounds run, and a captured round gives the eager one's result."""
    from hashattention_b200 import llama_tp
    cfg = _cfg(init_budget=16, recent_budget=16)
    B, W, S, keep = 3, 32, 500, 300
    model = llama_tp.TPLlama(cfg, 1, 0, device, batch=B, seed=2)
    model.enable_trees(W, mass=True)
    with pytest.raises(ValueError, match="observe"):
        model.prefill(llama_tp.tokens_for(cfg, B, 4).to(device), observe=5)
    cur = model.prefill(llama_tp.tokens_for(cfg, B, S, seed=4).to(device), observe=W)
    rows = torch.full((B,), float(W), device=device)
    parents = torch.tensor([PARENTS] * B, dtype=torch.int32, device=device)
    tree_lens = torch.tensor([9, 0, 5], dtype=torch.int32, device=device)

    def draft_of(first, seed):
        d = torch.randint(0, cfg.vocab_size, (B, len(PARENTS)), generator=torch.Generator().manual_seed(seed)).to(device)
        d[:, 0] = first
        return d

    def check_mass():
        for m in model.mass:
            # sums of S + 9 weights of W + 9 rows, each off by 2^-16 of itself at most
            assert float((m.sum(-1) - 4 * rows[:, None]).abs().max()) < 4 * (W + 18) * 2.0 ** -16
            for b in range(B):
                assert bool((m[b, :, int(model.seq_lens[b]):] == 0).all())

    check_mass()
    got = model.verify_tree(draft_of(cur, 1), parents, tree_lens)
    rows += got.count
    assert got.count.tolist()[1] == 0 and model.seq_lens.tolist()[1] == S
    check_mass()
    pos = model.pos.tolist()
    model.evict(keep)
    assert model.seq_lens.tolist() == [keep] * B and model.pos.tolist() == pos
    first = torch.where(got.count > 0, got.next_token, cur)
    # a round on the cut cache, eagerly and as a graph of the same state
    state = [model.seq_lens.clone(), model.pos.clone()] + [m.clone() for m in model.mass]
    draft = draft_of(first, 2)
    eager = model.verify_tree(draft, parents, tree_lens)
    after = [model.seq_lens.clone(), model.pos.clone()] + [m.clone() for m in model.mass]

    def restore():
        for t, s in zip([model.seq_lens, model.pos] + model.mass, state):
            t.copy_(s)

    restore()
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        with torch.cuda.graph(graph, stream=side):
            got = model.verify_tree(draft, parents, tree_lens)
    torch.cuda.current_stream().wait_stream(side)
    restore()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(got.accepted, eager.accepted) and torch.equal(got.count, eager.count)
    assert torch.equal(got.next_token[eager.count > 0], eager.next_token[eager.count > 0])
    for t, s in zip([model.seq_lens, model.pos] + model.mass, after):
        assert torch.equal(t, s)
    nxt = torch.empty(B, dtype=torch.int64, device=device)
    model.decode_step(torch.where(got.count > 0, got.next_token, first), nxt)
    model.check_status()
    assert bool(((nxt >= 0) & (nxt < cfg.vocab_size)).all())


@pytest.mark.gpu
def test_drafts_behind_the_cache_are_reported(device):
    from hashattention_b200 import llama_tp
    cfg = _cfg()
    model = llama_tp.TPLlama(cfg, 1, 0, device, batch=1, seed=1)
    model.enable_trees(8)
    model.prefill(llama_tp.tokens_for(cfg, 1, 760, seed=3).to(device))  # (three pages of 256)
    parents = torch.arange(-1, 7, dtype=torch.int32, device=device)[None].contiguous()
    draft = torch.zeros(1, 8, dtype=torch.int64, device=device)
    model.verify_tree(draft, parents)  # 768 tokens: just as many as fit
    model.check_status()
    model.seq_lens.fill_(761)
    model.verify_tree(draft, parents)
    with pytest.raises(RuntimeError, match="status"):
        model.check_status()
