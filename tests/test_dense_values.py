"""Dense attention over the paged cache at the ends of the value range: infinities in the V rows of the prefix, scores of up to 2^29 in
powers of two with one clear winner per row."""
import math

import pytest
import torch

import hashattention_b200 as ha
from test_dense import D, GROUP, Problem


def plant(x, b, spots):
    """(kv-head, token, channel, value) into V of sequence b."""
    for h, token, channel, value in spots:
        x.v[b][h, token, channel] = value
    x.write(b)


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
