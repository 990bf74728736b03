"""Dense attention over the paged cache at the ends of the value range: infinities in the V rows of the prefix, scores of up to 2^29 in
powers of two with one clear winner per row."""
import math

import pytest
import torch

import hashattention_b200 as ha
from test_dense import D, GROUP, Problem, score_error, weights64


def plant(x, b, spots):
    """(kv-head, token, channel, value) into V of sequence b."""
    for h, token, channel, value in spots:
        x.v[b][h, token, channel] = value
    x.write(b)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1, 4, 6, 30, 50, 100])
@pytest.mark.parametrize("prefix", [40, 700, 9000])
def test_infinities_in_the_prefix(device, n, prefix):
    """The output is an average with weights above zero: infinite where V is, NaN where V is or where both infinities meet, and
    finite in all other channels. Units of one CTA, and units that many CTAs share."""
    x = Problem(device, [prefix + n, 300 + n], [n, n], 2, n, "tree", seed=n + prefix)
    last = prefix - 1
    plant(x, 0, [(0, 3, 0, math.inf), (0, last, 5, -math.inf), (0, 0, 31, math.inf), (0, last, 31, math.inf),   # one sign
                 (0, 7, 64, math.inf), (0, last - 5, 64, -math.inf),                                              # both
                 (0, 20, 127, math.nan), (0, 21, 90, math.inf), (0, 30, 90, math.nan),
                 (1, prefix // 2, 17, -math.inf)])
    out, lse = x.ctx.tree_attention(x.q, x.mask, x.tree_lens)
    x.check(out, lse)
    assert bool((out[0, :, :GROUP, 0] == math.inf).all()) and bool((out[0, :, :GROUP, 5] == -math.inf).all())
    assert bool((out[0, :, :GROUP, 31] == math.inf).all()) and bool(out[0, :, :GROUP, [64, 90, 127]].isnan().all())
    assert bool((out[0, :, GROUP:, 17] == -math.inf).all())
    assert int((~torch.isfinite(out[0, :, :GROUP])).sum()) == 6 * GROUP * n and bool(torch.isfinite(out[1]).all())


@pytest.mark.gpu
@pytest.mark.parametrize("n", [4, 6, 40])
def test_infinities_in_the_prefix_and_in_drafts(device, n):
    """An infinity of the prefix meets those of drafts in the rows that see them only."""
    prefix, leaf = 500, n - 1
    x = Problem(device, [prefix + n], [n], 1, n, "tree", seed=7)
    plant(x, 0, [(0, 9, 1, math.inf), (0, prefix + leaf, 1, -math.inf),   # opposite signs
                 (0, 9, 2, math.inf), (0, prefix + leaf, 2, math.inf),    # the same one
                 (0, 9, 3, -math.inf), (0, prefix + leaf, 3, math.nan),
                 (0, prefix + leaf, 4, -math.inf)])
    out, lse = x.ctx.tree_attention(x.q, x.mask, x.tree_lens)
    x.check(out, lse)
    sees = x.visible[0][:, leaf].to(device)
    assert bool(out[0, sees][:, :, [1, 3]].isnan().all()) and bool((out[0, ~sees][:, :, [1, 2]] == math.inf).all())
    assert bool((out[0, sees][:, :, 4] == -math.inf).all()) and bool(torch.isfinite(out[0, ~sees][:, :, 4]).all())


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1, 4, 6, 40])
@pytest.mark.parametrize("prefix", [300, 9000])
def test_infinities_whose_weight_fp32_holds_as_zero(device, n, prefix):
    """Scores thousands apart: every weight but one is zero in fp32 (and in 64 bits), but none is by its definition."""
    x = Problem(device, [prefix + n, 200 + n], [n, n], 2, n, "tree", seed=n + prefix)
    x.ctx, leaf = ha.DenseDecodeContext(x.cache, n, sm_scale=300.0), n - 1
    spots = [(0, 3, 0, math.inf), (0, prefix - 1, 5, -math.inf), (0, prefix // 2, 77, math.inf), (0, prefix // 3, 100, math.inf),
             (0, 9, 100, -math.inf), (0, 40, 101, math.nan)]
    if n > 1:
        spots += [(0, prefix + leaf, 20, math.inf), (0, prefix + leaf, 77, -math.inf)]
    plant(x, 0, spots)
    out, lse = x.ctx.tree_attention(x.q, x.mask, x.tree_lens)
    sees = x.visible[0][:, leaf].to(device) if n > 1 else torch.zeros(n, dtype=torch.bool, device=device)
    want = torch.zeros(n, GROUP, D, device=device)
    want[:, :, 0], want[:, :, 5], want[:, :, 77], want[:, :, [100, 101]] = math.inf, -math.inf, math.inf, math.nan
    want[sees, :, 20] = math.inf
    want[sees, :, 77] = math.nan
    got = out[0, :, :GROUP].float()
    assert torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(torch.isfinite(got), torch.isfinite(want))
    assert torch.equal(got == math.inf, want == math.inf)
    assert bool(torch.isfinite(out[0, :, GROUP:]).all()) and bool(torch.isfinite(out[1]).all()) and bool(torch.isfinite(lse).all())


@pytest.mark.gpu
@pytest.mark.parametrize("what", ["k", "q"])
@pytest.mark.parametrize("n", [1, 30, 50])
def test_scores_that_are_not_finite_stay_nan_beside_infinite_values(device, what, n):
    """NaN scores make their whole row NaN, infinite V or not."""
    x = Problem(device, [600 + n], [n], 1, n, "chain", seed=n)
    if what == "k":
        x.k[0][0, 11, 3] = math.nan
    else:
        x.q[0, n - 1, 2, 8] = math.nan
    plant(x, 0, [(0, 50, 9, math.inf)])
    out, lse = x.ctx.tree_attention(x.q, x.mask, x.tree_lens)
    x.check(out, lse)


@pytest.mark.gpu
@pytest.mark.parametrize("n,prefix,kv_heads", [(1, 700, 2), (1, 20000, 2), (4, 3000, 4), (5, 700, 2), (9, 9000, 8), (32, 20000, 4), (40, 700, 2), (60, 9000, 2), (128, 2000, 1)])
@pytest.mark.parametrize("power", [0, 8, 15, 17, 19, 22])
def test_one_clear_winner_per_row(device, n, prefix, kv_heads, power):
    """Entries of q and K are +1 and -1 and the softmax scale 2^power, so a score is an integer times a power of two. Each node has one
    token of the prefix, or itself, whose K is its q but for one channel: a score of 126, all others being 72 at most (asserted).
    The weights of the others are below e^-54, so the output is the winner's V row, a bf16 number: against half a step of bf16
    (2^-9), e^-54 * 20000 and the 2^-16 of the weight's split are nothing, and rounding gives that very number. Winners lie all
    over the prefix, in every tile and every CTA's range. The reference of a row's weights is its score in powers of two, rounded
    (up to 2^29.5, where half an ulp is 16): the winner's weight is not 1 but a power of two, which has to cancel. The log-sum-exp is
    126 * 2^power up to the roundings of log2(e), ln(2), a sum and two products, each 2^-24 of it, and the correction for cut
    sums, 2^-23."""
    x = Problem(device, [prefix + n, n + 3], [n, n], kv_heads, n, "tree", seed=power)
    g = torch.Generator().manual_seed(100 * n + power)

    def signs(*size):
        return (torch.randint(0, 2, size, generator=g) * 2 - 1).to(torch.bfloat16).to(device)

    u = signs(2, n, kv_heads, D)
    x.q.copy_(u.repeat_interleave(GROUP, 2))
    winner = []
    for b in range(2):
        S, P = x.lens[b], x.lens[b] - n
        x.k[b] = signs(kv_heads, S, D)
        at = P + torch.arange(n)                                     # itself ...
        if b == 0:
            spread = 1 + torch.randperm(P - 2, generator=g)[:n]
            at = torch.where(torch.arange(n) % 4 == 3, at, spread)   # ... or a token of the prefix, its ends among them
            at[0], at[n // 2] = P - 1, 0
        assert len(set(at.tolist())) == n
        at = at.to(device)
        for h in range(kv_heads):
            near = u[b, :, h].clone()
            near[:, 77] *= -1
            x.k[b][h, at] = near
            s = x.k[b][h].double() @ u[b, :, h].double().T           # [S, n]
            assert bool((s[at, torch.arange(n, device=device)] == 126).all())
            s[at, torch.arange(n, device=device)] = -128
            assert float(s.amax()) <= 72
        winner.append(at)
        x.write(b)
    x.ctx = ha.DenseDecodeContext(x.cache, n, sm_scale=2.0 ** power)
    out, lse = x.ctx.tree_attention(x.q, x.mask, x.tree_lens)
    x.ctx.check_status()
    for b in range(2):
        want = x.v[b][:, winner[b]].transpose(0, 1).repeat_interleave(GROUP, 1)  # [n, Hq, D]
        assert torch.equal(out[b], want)
        assert bool(((lse[b].double() / (126 * 2.0 ** power) - 1).abs() <= 5 * 2.0 ** -24 + 2.0 ** -23).all())


@pytest.mark.gpu
def test_the_output_in_the_place_of_the_queries_is_refused(device):
    """Queries are read again behind the first written rows where a draft's V has an infinity."""
    x = Problem(device, [300], [6], 1, 6, seed=1)
    q = x.q.contiguous()
    with pytest.raises(ValueError, match="another tensor"):
        x.ctx.tree_attention(q, x.mask, x.tree_lens, out=q)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1, 3, 6, 40])
@pytest.mark.parametrize("prefix", [0, 500, 9000])
def test_infinite_values_under_scores_of_minus_infinity(device, n, prefix):
    """K of -inf against q above zero: a weight of zero, and zero times an infinity is NaN. A row whose scores are all -inf is zeros."""
    x = Problem(device, [prefix + n, 200 + n], [n, n], 2, n, "chain", seed=n + prefix)
    x.q[..., 7] = x.q[..., 7].abs() + 0.5
    S, leaf = prefix + n, prefix + n - 1
    if prefix:
        x.k[0][0, 30, 7], x.v[0][0, 30, 3] = -math.inf, math.inf           # weightless: NaN
        x.k[0][0, prefix - 1, 7] = -math.inf                                # weightless beside finite values: nothing
        x.v[0][0, 60, 9] = math.inf                                         # infinite
        x.v[0][0, 61, 3] = math.inf
    x.k[0][0, leaf, 7], x.v[0][0, leaf, 11] = -math.inf, -math.inf
    x.k[1][1, :, 7], x.v[1][1, ::3, 20] = -math.inf, math.inf               # every score of a kv-head
    x.write(0)
    x.write(1)
    out, lse = x.ctx.tree_attention(x.q, x.mask, x.tree_lens)
    assert bool((out[1, :, GROUP:] == 0).all()) and bool((lse[1, :, GROUP:] == -math.inf).all())
    x.lens, x.nodes = [S, 0], [n, 0]  # (the definition's 0 / 0 of the second one has been looked at)
    out[1] = lse[1] = 0
    if S > 1:
        x.check(out, lse)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1, 5, 20, 64, 128])
@pytest.mark.parametrize("prefix", [0, 300, 3000])
def test_received_weights_of_rows_that_are_nan(device, n, prefix):
    """A row whose log-sum-exp is NaN gives NaN to the tokens it sees and nothing to the others."""
    x = Problem(device, [prefix + n, 100 + n], [n, n], 2, n, "tree", seed=n + prefix)
    leaf, mid = n - 1, n // 2
    x.k[0][0, prefix + leaf, 5] = math.nan   # kv-head 0: the rows that see the leaf (itself)
    x.q[0, mid, GROUP + 1, 3] = math.nan     # kv-head 1: one row of one node
    x.write(0)
    _, lse = x.ctx.tree_attention(x.q, x.mask, x.tree_lens)
    mass = x.ctx.attention_mass(x.q, lse, x.ctx.new_mass(), x.mask, x.tree_lens)
    x.ctx.check_status()
    sees, S = x.sees(0), prefix + n
    p, _ = weights64(x.q[0], x.k[0], sees, x.scale)           # [n, Hq, S], NaN in the rows that are
    nan_rows = torch.isnan(lse[0])                             # [n, Hq]
    assert nan_rows.nonzero().tolist() == sorted([[leaf, h] for h in range(GROUP)] + [[mid, GROUP + 1]])
    p = torch.where(nan_rows[..., None], torch.where(sees[:, None], math.nan, 0.0).double(), p)
    want = p.view(n, 2, GROUP, S).sum((0, 2))
    got = mass[0, :, :S].double()
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    d = score_error(x.q[0].nan_to_num(), x.k[0].nan_to_num(), x.scale)
    fine = ~torch.isnan(want)
    assert bool(((got - want).abs()[fine] <= (want * (2 * d + 2.0 ** -18 + 513 * 2.0 ** -24))[fine]).all())
    assert bool(torch.isfinite(mass[1]).all()) and bool((mass[0, :, S:] == 0).all())
