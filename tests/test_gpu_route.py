"""Routing by scores on the GPU against the float64 oracle: indices equal, weights and gradients within float32 rounding.

Tolerances.  u = 2^-24.  A weight is exp of a difference (argument rounded: u |argument| relative, arguments up to 2 max|z|), a
sum of at most E terms in a tree over lanes with chains of at most 16, a division and a product: relative error at most
u (2 max|z| + 64).  A routing entry is that, rounded once to the storage type.  A gradient is a product of a weight with a
difference of gradients, each of whose terms carries that error."""
import math

import numpy as np
import pytest
import torch

from oracle import norm_route as R

pytestmark = pytest.mark.gpu

DEV = 'cuda:0'
U = 2.0 ** -24


def _ops():
    from d2dmoe_amd import ops
    return ops


def _half(t):
    return torch.finfo(t).eps / 2


def _logits(n, e, t, seed, ties=False, masks=False):
    g = torch.Generator().manual_seed(seed)
    z = torch.randn(n, e, generator=g) * 1.5 + torch.randn(e, generator=g) * 0.5
    if ties:
        z = (z * 2).round() / 2
    if masks:
        z[torch.rand(n, e, generator=g) < 0.2] = -math.inf
        z[::7] = -math.inf                                # rows that a padding mask emptied
        z[3::11, e // 2] = math.nan
        z[5::13, 0] = math.inf
        z[4::17] = torch.finfo(t).min                     # masked with the type's lowest value: ordinary, equal logits
    return z.to(t)


def _check(z, k, scoring, bias, kw, t, got):
    routing, indices, weights, counts = got
    want, idx, w = R.route(z.double().numpy(), k, scoring, bias=None if bias is None else bias.double().numpy(), **kw)
    assert indices.dtype == torch.int32 and np.array_equal(indices.cpu().numpy(), idx)
    big = z.float()[torch.isfinite(z.float()) & (z.float() > -1e4)]
    tol = U * (2 * big.abs().max().item() + 64 if big.numel() else 64)
    err = np.abs(weights.double().cpu().numpy() - w)
    assert weights.dtype == torch.float32 and (err <= tol * w + 1e-37).all(), (err / (w + 1e-37)).max()
    err = np.abs(routing.double().cpu().numpy() - want)
    assert routing.dtype == t and (err <= (tol + _half(t)) * want + 2.0 ** -25 * (t == torch.float16) + 1e-37).all()
    if counts is not None:
        assert np.array_equal(counts.cpu().numpy(), np.bincount(idx[idx >= 0], minlength=z.size(1)))
    return idx, tol


def _check_grad(z, idx, q, scoring, renormalise, scale, t, grad, tol):
    zz = z.double().numpy()
    want = R.route_grads(zz, idx, q, scoring, renormalise, scale)
    # every term is a product of scores (<= 1) with gradients; the row's largest gradient bounds the terms that cancel
    size = np.abs(q).max(1, initial=0.0)[:, None] * scale
    if renormalise:
        w = R.route_grads(zz, idx, np.ones_like(q), scoring, False, 1.0)    # where a gradient can be at all
        bound = 4 * tol * size * (np.abs(want) + np.abs(w) > 0)
    else:
        bound = 4 * tol * size
    err = np.abs(grad.double().cpu().numpy() - want)
    assert grad.dtype == t and (err <= bound + _half(t) * np.abs(want) + 2.0 ** -25 * (t == torch.float16)).all(), (err - bound).max()


EXPERTS = [1, 2, 3, 7, 8, 13, 16, 24, 60, 64, 65, 100, 128, 129, 160, 256, 320, 512, 513, 1000, 1024]


@pytest.mark.parametrize('t', [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize('e', EXPERTS)
def test_plain_choice(e, t):
    for k in sorted({1, 2, 8, min(e, 33), e if e <= 129 else 70}):
        if k > e:
            continue
        for scoring in ('softmax', 'sigmoid'):
            for renormalise in (True, False):
                print('route', e, k, t, scoring, renormalise, flush=True)
                z = _logits(29, e, t, seed=e + k, ties=k % 2 == 0, masks=True)
                kw = dict(renormalise=renormalise, scale=1.0 if renormalise else 2.5)
                got = _ops().route_topk(z.to(DEV), k, scoring, want_counts=True, **kw)
                idx, tol = _check(z, k, scoring, None, kw, t, got)
                g = torch.Generator().manual_seed(k)
                q, dense = torch.randn(29, k, generator=g), torch.randn(29, e, generator=g).to(t)
                grad = _ops().route_topk_backward(z.to(DEV), got[1], scoring, grad_weights=q.to(DEV), **kw)
                _check_grad(z, idx, q.double().numpy(), scoring, renormalise, kw['scale'], t, grad, tol)
                by_place = np.where(idx >= 0, np.take_along_axis(dense.double().numpy(), np.maximum(idx, 0), 1), 0.0)
                grad = _ops().route_topk_backward(z.to(DEV), got[1], scoring, grad_routing=dense.to(DEV), **kw)
                _check_grad(z, idx, by_place, scoring, renormalise, kw['scale'], t, grad, tol)
                grad = _ops().route_topk_backward(z.to(DEV), got[1], scoring, grad_routing=dense.to(DEV), grad_weights=q.to(DEV), **kw)
                _check_grad(z, idx, by_place + q.double().numpy(), scoring, renormalise, kw['scale'], t, grad, tol)


@pytest.mark.parametrize('t', [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize('e,groups,kept,k', [(4, 2, 1, 2), (8, 4, 3, 2), (12, 3, 2, 4), (16, 2, 1, 4), (16, 8, 3, 2), (8, 2, 1, 3), (8, 4, 2, 4), (8, 8, 3, 2), (12, 3, 2, 5), (24, 3, 1, 8), (60, 5, 2, 6), (64, 8, 4, 8),
                                             (96, 8, 3, 6), (128, 4, 2, 8), (128, 64, 9, 8), (160, 8, 3, 6), (256, 8, 4, 8), (256, 1, 1, 8),
                                             (320, 10, 5, 8), (512, 2, 1, 4), (512, 16, 4, 12), (1000, 10, 4, 8), (1024, 32, 4, 8),
                                             (1024, 1024, 40, 33)])
def test_groups_and_bias(e, groups, kept, k, t):
    for scoring in ('softmax', 'sigmoid'):
        for score in ('top2', 'max'):
            for biased in (True, False):
                print('groups', e, groups, kept, k, t, scoring, score, biased, flush=True)
                z = _logits(23, e, t, seed=e + groups, ties=score == 'max', masks=True)
                bias = torch.randn(e, generator=torch.Generator().manual_seed(3)) * (0.1 if scoring == 'sigmoid' else 0.5 / e) if biased else None
                if biased and e > 8:
                    bias[1] = -math.inf                  # an expert the bias switches off
                kw = dict(n_groups=groups, kept_groups=kept, group_score=score, renormalise=True, scale=2.5)
                got = _ops().route_topk(z.to(DEV), k, scoring, None if bias is None else bias.to(DEV), want_counts=True, **kw)
                _check(z, k, scoring, bias, kw, t, got)


@pytest.mark.parametrize('t', [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize('e,groups,k', [(5, 1, 5), (16, 2, 8), (18, 3, 5), (32, 4, 8), (33, 3, 9), (20, 2, 16), (48, 8, 12), (60, 5, 9), (64, 8, 16), (65, 5, 12),
                                        (64, 4, 32), (100, 10, 30), (128, 4, 32), (130, 2, 20), (66, 3, 33), (200, 8, 50), (256, 8, 64), (257, 1, 40)])
def test_many_places(e, groups, k, t):
    """Nearly as many places as the experts, and the lanes of their teams, leave room for."""
    for scoring in ('softmax', 'sigmoid'):
        for biased in (False, True):
            for kept in sorted({groups, -(-k * groups // e)}):
                print('places', e, groups, kept, k, t, scoring, biased, flush=True)
                z = _logits(21, e, t, seed=e + k, masks=True)
                bias = torch.randn(e, generator=torch.Generator().manual_seed(k)) * 0.1 if biased else None
                kw = dict(n_groups=groups, kept_groups=kept, group_score='top2' if biased else 'max', renormalise=True, scale=1.5)
                got = _ops().route_topk(z.to(DEV), k, scoring, None if bias is None else bias.to(DEV), want_counts=True, **kw)
                _check(z, k, scoring, bias, kw, t, got)


@pytest.mark.parametrize('t', [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize('e,groups,kept,k', [(65, 1, 1, 65), (66, 33, 33, 66), (130, 2, 2, 65), (130, 2, 1, 65), (140, 70, 40, 66),
                                             (256, 8, 4, 100), (513, 1, 1, 128), (1000, 10, 4, 333), (1024, 32, 16, 200),
                                             (1024, 1024, 500, 70), (1024, 1, 1, 1024)])
def test_more_places_than_a_wave_has_lanes(e, groups, kept, k, t):
    """k > 64 runs on a kernel of its own: scores, biases, groups, masked and NaN rows, and the gradient of what it chose."""
    n = 23 if k <= 66 else 8                                   # (the oracle's gradient takes k^2 steps a row)
    for scoring in ('softmax', 'sigmoid'):
        for score in ('top2', 'max'):
            for biased in (True, False):
                print('far', e, groups, kept, k, t, scoring, score, biased, flush=True)
                z = _logits(n, e, t, seed=e + k, ties=score == 'max', masks=True)
                bias = torch.randn(e, generator=torch.Generator().manual_seed(k)) * (0.1 if scoring == 'sigmoid' else 0.5 / e) if biased else None
                if biased:
                    bias[1] = -math.inf
                    bias[e // 2] = torch.finfo(torch.float32).min
                how = dict(renormalise=biased, scale=2.5)
                kw = dict(n_groups=groups, kept_groups=kept, group_score=score, **how)
                got = _ops().route_topk(z.to(DEV), k, scoring, None if bias is None else bias.to(DEV), want_counts=True, **kw)
                idx, tol = _check(z, k, scoring, bias, kw, t, got)
                q = torch.randn(n, k, generator=torch.Generator().manual_seed(e))
                grad = _ops().route_topk_backward(z.to(DEV), got[1], scoring, grad_weights=q.to(DEV), **how)
                _check_grad(z, idx, q.double().numpy(), scoring, how['renormalise'], 2.5, t, grad, tol)


def test_more_places_than_lanes_with_biases_of_any_size():
    g = torch.Generator().manual_seed(4)
    e, lowest = 160, torch.finfo(torch.float32).min
    z, some = _logits(40, e, torch.float32, seed=e), torch.rand(160, generator=g)
    for bias in (torch.full((e,), 1000.0), some * 1e30, some * 1e-30, torch.where(some < 0.7, lowest, 0.0),
                 torch.where(some < 0.5, 1e5, -1e5), torch.where(some < 0.3, math.inf, 0.0), torch.full((e,), -math.inf),
                 torch.where(some < 0.9, 0.0, math.nan)):
        for scoring in ('softmax', 'sigmoid'):
            for kw in ({}, dict(n_groups=4, kept_groups=2, group_score='top2'), dict(n_groups=4, kept_groups=2, group_score='max')):
                got = _ops().route_topk(z.to(DEV), 70, scoring, bias.to(DEV), want_counts=True, **kw)
                _check(z, 70, scoring, bias, kw, torch.float32, got)


def test_bias_that_is_not_a_number_routes_nothing():
    z = _logits(9, 32, torch.float32, seed=1)
    bias = torch.zeros(32)
    bias[4] = math.nan
    routing, indices, weights, counts = _ops().route_topk(z.to(DEV), 4, 'sigmoid', bias.to(DEV), want_counts=True)
    assert (indices == -1).all() and not routing.any() and not weights.any() and not counts.any()


@pytest.mark.parametrize('scoring', ['softmax', 'sigmoid'])
def test_neighbours_that_float32_scores_do_not_tell_apart(scoring):
    """Choices whose difference lies below float32's step at the score: pairs of experts whose scores plus bias differ by a few
    2^-40 (the bias takes back what the logits differ by, up to its own rounding), in every row."""
    g = torch.Generator().manual_seed(6)
    z = torch.randn(4000, 64, generator=g)
    z = z + 0.0
    z[:, 1::2] = z[:, ::2]                               # equal pairs ...
    z[:, 1::2] *= 1 + 2.0 ** -22                         # ... a step or two apart
    bias = torch.full((64,), 0.25)
    for k, kw in ((8, {}), (6, dict(n_groups=8, kept_groups=3, group_score='top2')), (6, dict(n_groups=8, kept_groups=3, group_score='max'))):
        got = _ops().route_topk(z.to(DEV), k, scoring, bias.to(DEV), **kw)
        _check(z[:400], k, scoring, bias, kw, torch.float32, (got[0][:400], got[1][:400], got[2][:400], None))
    # zero bias, 16-bit logits: ties in nearly every row
    zb = z.bfloat16()
    got = _ops().route_topk(zb.to(DEV), 8, scoring, torch.zeros(64, device=DEV))
    _check(zb[:400], 8, scoring, torch.zeros(64), {}, torch.bfloat16, (got[0][:400], got[1][:400], got[2][:400], None))


@pytest.mark.parametrize('e,k', [(8, 3), (16, 12), (64, 8), (200, 8), (256, 24), (1024, 8)])
def test_masks_in_the_bias(e, k):
    """Low values that switch experts off, also so many that some of those have to be chosen, and choices a little above and below
    a distance of four from the best."""
    g = torch.Generator().manual_seed(e)
    z = _logits(60 if e <= 256 else 20, e, torch.float32, seed=e)
    z[1::3] = z[1::3, :1]                                      # rows of equal logits
    some = torch.rand(e, generator=g)
    for off in (torch.finfo(torch.float32).min, -1e9, -1e4, -65.0, -4.0, -3.0):
        for share in (0.1, 0.9, 1.0):
            bias = torch.where(some < share, off, 0.0)
            bias[e // 2] = -62.0 if off < -65 else 0.5
            bias[e // 3] = max(off, -1e4) + 61.0
            for scoring in ('softmax', 'sigmoid'):
                for kw in ({}, dict(n_groups=4, kept_groups=3, group_score='top2')):
                    print('mask', e, k, off, share, scoring, kw, flush=True)
                    got = _ops().route_topk(z.to(DEV), k, scoring, bias.to(DEV), want_counts=True, **kw)
                    _check(z, k, scoring, bias, kw, torch.float32, got)


@pytest.mark.parametrize('scoring', ['softmax', 'sigmoid'])
@pytest.mark.parametrize('e,k', [(2, 1), (4, 2), (8, 4), (16, 4), (24, 4), (64, 8), (128, 8), (256, 8), (256, 32), (512, 8), (1000, 20), (1024, 64)])
def test_one_pair_that_float32_scores_do_not_tell_apart(e, k, scoring):
    """Row p: the choices lie far apart but for places p and p + 1, whose logits are neighbouring float32 numbers, the larger one at
    the higher index.  Every place has its turn, the last one with the first that is left out among them."""
    g = torch.Generator().manual_seed(e + k)
    z = torch.empty(k, e)
    for p in range(k):
        falling = 1.0 - torch.arange(e) * 2.0 / e          # by place
        falling[p] = torch.nextafter(falling[p + 1], torch.tensor(9.0))
        at = torch.randperm(e, generator=g)
        if at[p] < at[p + 1]:
            at[p], at[p + 1] = at[p + 1].clone(), at[p].clone()
        z[p, at] = falling
    for groups in (1, 2):
        kw = dict(n_groups=groups, kept_groups=groups, group_score='top2')
        got = _ops().route_topk(z.to(DEV), k, scoring, torch.zeros(e, device=DEV), want_counts=True, **kw)
        _check(z, k, scoring, torch.zeros(e), kw, torch.float32, got)
        one = torch.cat([_ops().route_topk(z[p:p + 1].to(DEV), k, scoring, torch.zeros(e, device=DEV), **kw)[1] for p in range(k)])
        assert torch.equal(one, got[1])                    # (alone in its wave)


@pytest.mark.parametrize('e', [4, 8, 16, 64, 200, 1024])
def test_biases_of_any_size(e):
    """What the choice goes by spans anything from a float32 step of a large offset to the ends of the type: the choice is still
    that of the float64 sums."""
    g = torch.Generator().manual_seed(e)
    z = _logits(150 if e <= 64 else 20, e, torch.float32, seed=e)
    lowest, some = torch.finfo(torch.float32).min, torch.rand(e, generator=g)
    biases = {'offset': torch.full((e,), 1000.0), 'two steps of an offset': 1000.0 + (some > 0.5) * 2.0 ** -13,
              'far': some * 1e30, 'tiny': some * 1e-30, 'lowest': torch.where(some < 0.7, lowest, 0.0), 'all lowest': torch.full((e,), lowest),
              'ends': torch.where(some < 0.4, lowest, torch.where(some < 0.6, 3e38, 3.2e38)), 'two low ones': torch.where(some < 0.5, lowest, -3.3e38),
              'inf': torch.where(some < 0.3, math.inf, 0.0), 'infs': torch.where(some < 0.3, math.inf, torch.where(some < 0.6, -math.inf, lowest)),
              'none': torch.full((e,), -math.inf), 'one': torch.where(torch.arange(e) == e // 2, 0.0, -math.inf)}
    for name, bias in biases.items():
        for scoring in ('softmax', 'sigmoid'):
            for kw in ({}, dict(n_groups=4, kept_groups=2, group_score='top2'), dict(n_groups=4, kept_groups=2, group_score='max')):
                k = min(4, e // 2)
                print('bias', e, name, scoring, kw, flush=True)
                got = _ops().route_topk(z.to(DEV), k, scoring, bias.to(DEV), want_counts=True, **kw)
                _check(z, k, scoring, bias, kw, torch.float32, got)


@pytest.mark.parametrize('e,groups', [(8, 2), (24, 4), (64, 4), (256, 8), (1024, 16)])
def test_large_biases_that_cancel_in_a_group(e, groups):
    """In every group one expert that a bias of +B forces and one that -B masks, as its two best: the sum is a few units, each
    addend's float32 rounding B 2^-24, so the order of two sums may only come from the float64 ones."""
    g = torch.Generator().manual_seed(e)
    size = e // groups
    n = max(300, 24000 // e)
    for large in (1e2, 1e3, 1e4, 1e5, 1e7):
        for spread in (1.5, 0.02):
            z = torch.randn(n, e, generator=g) * spread
            bias = torch.full((e,), -2.0 * large)
            for i in range(groups):
                at = torch.randperm(size, generator=g)[:2] + i * size
                own = large * (1 + 0.25 * (i % 2))
                bias[at[0]], bias[at[1]] = own, -own
            for scoring in ('softmax', 'sigmoid'):
                for kept, k in ((1, 1), (groups // 2, min(2, groups // 2))):
                    kw = dict(n_groups=groups, kept_groups=kept, group_score='top2')
                    print('cancel', e, groups, large, spread, scoring, kept, k, flush=True)
                    got = _ops().route_topk(z.to(DEV), k, scoring, bias.to(DEV), want_counts=True, **kw)
                    _check(z, k, scoring, bias, kw, torch.float32, got)


def test_scores_that_underflow_still_share_their_weight():
    """Chosen scores of 1e-60 and less: renormalised weights go by their ratio."""
    z = torch.tensor([[-140.0, -139.0, -150.0, -400.0], [-3e38, -3e38, -3e38, -3e38]])
    for scoring in ('softmax', 'sigmoid'):
        got = _ops().route_topk(z.to(DEV), 2, scoring)
        # (row 1: equal logits; the arguments are differences of the logits, so the bound of the other tests holds)
        assert got[1].tolist() == [[1, 0], [0, 1]]
        want = [[1 / (1 + math.exp(-1)), 1 / (1 + math.exp(1))], [0.5, 0.5]]
        assert np.abs(got[2].cpu().numpy() - want).max() < 64 * U
    # a bias that chooses experts far below the row's best
    bias = torch.tensor([0.0, 0.0, 5.0, 6.0])
    got = _ops().route_topk(torch.tensor([[0.0, 1.0, -200.0, -201.0]], device=DEV), 2, 'softmax', bias.to(DEV))
    assert got[1].tolist() == [[3, 2]] and abs(got[2][0, 1].item() - 1 / (1 + math.exp(-1))) < 64 * U


def test_no_tokens_and_many():
    ops = _ops()
    e = torch.empty(0, 16, device=DEV)
    routing, indices, weights, counts = ops.route_topk(e, 3, want_counts=True)
    assert routing.shape == (0, 16) and indices.shape == weights.shape == (0, 3) and not counts.any()
    assert ops.route_topk_backward(e, indices, grad_weights=weights).shape == (0, 16)
    # more than 2^31 logits
    n = (1 << 21) + 5
    z = torch.zeros(n, 1024, dtype=torch.bfloat16, device=DEV)
    tail = _logits(5, 1024, torch.bfloat16, seed=4)
    z[-5:] = tail.to(DEV)
    routing, indices, weights, _ = ops.route_topk(z, 4)
    _check(tail, 4, 'softmax', None, {}, torch.bfloat16, (routing[-5:], indices[-5:], weights[-5:], None))
    assert (indices[:-5] == torch.arange(4, device=DEV)).all() and (weights[:-5] == 0.25).all()
    q = torch.ones(n, 4, device=DEV)
    q[-5:, 0] = 2.0
    grad = ops.route_topk_backward(z, indices, grad_weights=q)
    assert not grad[:-5].any() and grad[-5:].any()
    del z, routing, grad


def test_more_tokens_than_one_launch_takes():
    """Sixteen tokens per wave, four waves per workgroup: the launches are cut at 2^22 workgroups."""
    ops = _ops()
    n = (1 << 28) + 77
    z = torch.zeros(n, 4, dtype=torch.bfloat16, device=DEV)
    z[:, 2] = 1.0
    tail = _logits(100, 4, torch.bfloat16, seed=8)
    z[-100:] = tail.to(DEV)
    routing, indices, weights, counts = ops.route_topk(z, 1, 'sigmoid', renormalise=False, want_counts=True)
    _check(tail, 1, 'sigmoid', None, dict(renormalise=False), torch.bfloat16, (routing[-100:], indices[-100:], weights[-100:], None))
    assert (indices[:-100] == 2).all() and int(counts.sum()) == n
    grad = ops.route_topk_backward(z, indices, 'sigmoid', False, grad_weights=torch.ones_like(weights))
    assert (grad[:-100, 2] == grad[0, 2]).all() and not grad[:-100, 3].any()
    ref = R.route_grads(tail.double().numpy(), indices[-100:].cpu().numpy(), np.ones((100, 1)), 'sigmoid', False, 1.0)
    assert np.abs(grad[-100:].double().cpu().numpy() - ref).max() <= _half(torch.bfloat16)
    del z, routing, indices, weights, grad


def test_places_that_are_no_experts_are_left_out():
    """Indices of the caller's own making: out of range counts as left over, the same expert twice adds up."""
    z = _logits(6, 40, torch.float32, seed=2)
    idx = torch.tensor([[3, -1, 7], [40, 5, 2], [1 << 30, -5, 0], [9, 9, 4], [-1, -1, -1], [39, 0, 38]], dtype=torch.int32)
    q = torch.randn(6, 3, generator=torch.Generator().manual_seed(1))
    for scoring in ('softmax', 'sigmoid'):
        for renormalise in (True, False):
            grad = _ops().route_topk_backward(z.to(DEV), idx.to(DEV), scoring, renormalise, 1.5, grad_weights=q.to(DEV))
            _check_grad(z, idx.numpy(), q.double().numpy(), scoring, renormalise, 1.5, torch.float32, grad, U * 80)


@pytest.mark.parametrize('off', [1, 3])
def test_rows_that_start_anywhere_and_bytes_around_them(off):
    import ctypes
    from d2dmoe_amd import hip_abi as abi
    lib = abi.load()
    for t, code in ((torch.bfloat16, abi.BF16), (torch.float32, abi.F32)):
        for n, e, k in ((7, 128, 8), (9, 60, 5), (5, 31, 31), (3, 700, 20)):
            z = _logits(n, e, t, seed=n)
            q = torch.randn(n, e, generator=torch.Generator().manual_seed(7)).to(t)

            def place(v):
                buf = torch.full((off + v.numel() + 64,), 7.0, dtype=v.dtype, device=DEV)
                buf[off:off + v.numel()] = v.reshape(-1).to(DEV)
                return buf

            ins = [place(z), place(q)]
            outs = [torch.full((off + c + 64,), 7, dtype=ty, device=DEV) for c, ty in
                    ((n * e, t), (n * k, torch.int32), (n * k, torch.float32), (e, torch.int32), (n * e, t))]
            at = [v.data_ptr() + off * v.element_size() for v in ins + outs]
            rs = abi.RouteShape(n, e, k, code, 0, 1, 1, 0, 1, 1.0)
            s = torch.cuda.current_stream().cuda_stream
            abi.check(lib.d2dmoe_route_topk(ctypes.byref(rs), at[0], None, at[2], at[3], at[4], at[5], s), 'forward')
            abi.check(lib.d2dmoe_route_topk_backward(ctypes.byref(rs), at[0], at[3], at[1], None, at[6], s), 'backward')
            sizes = (n * e, n * k, n * k, e, n * e)
            for v, c in zip(outs, sizes):
                assert (v[:off] == 7).all() and (v[off + c:] == 7).all()
            cut = [v[off:off + c] for v, c in zip(outs, sizes)]
            idx, tol = _check(z, k, 'softmax', None, {}, t, (cut[0].view(n, e), cut[1].view(n, k), cut[2].view(n, k), cut[3]))
            by_place = np.take_along_axis(q.double().numpy(), idx, 1)
            _check_grad(z, idx, by_place, 'softmax', True, 1.0, t, cut[4].view(n, e), tol)
            # each output alone
            alone = torch.full_like(outs[1], 7)
            abi.check(lib.d2dmoe_route_topk(ctypes.byref(rs), at[0], None, None, alone.data_ptr() + off * 4, None, None, s), 'indices')
            assert torch.equal(alone, outs[1])


def test_on_a_stream_of_its_own_and_captured():
    ops = _ops()
    cases = []
    for seed, (n, e) in enumerate(((900, 128), (500, 320))):
        z = _logits(n, e, torch.bfloat16, seed=seed).to(DEV)
        q = torch.randn(n, e, generator=torch.Generator().manual_seed(seed)).bfloat16().to(DEV)
        bias = torch.randn(e, device=DEV) * 0.05

        def step(z=z, q=q, bias=bias):
            routing, indices, weights, counts = ops.route_topk(z, 6, 'sigmoid', bias, want_counts=True)
            return routing, indices, weights, counts, ops.route_topk_backward(z, indices, 'sigmoid', grad_routing=q)

        eager = [v.clone() for v in step()]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            for a, c in zip(step(), eager):
                assert torch.equal(a, c)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = step()
        cases.append((graph, got, eager, step))
    for _ in range(4):
        for graph, got, eager, step in cases:
            for v in got:
                v.fill_(3)
            graph.replay()
            step()
            torch.cuda.synchronize()
            for a, c in zip(got, eager):
                assert torch.equal(a, c)


def test_gradient_is_the_difference_quotient():
    """float32, central differences of step 2^-7 of the weights' sum with q: truncation 2^-14 / 6 of a third derivative of order
    one, rounding 2^-24 of weights below 2.5 over the step (4e-5)."""
    ops = _ops()
    z = _logits(3, 20, torch.float32, seed=12).to(DEV)
    q = torch.randn(3, 4, generator=torch.Generator().manual_seed(2)).to(DEV)
    step = 2.0 ** -7
    for scoring in ('softmax', 'sigmoid'):
        for renormalise in (True, False):
            _, idx, _, _ = ops.route_topk(z, 4, scoring, renormalise=renormalise, scale=2.5)
            grad = ops.route_topk_backward(z, idx, scoring, renormalise, 2.5, grad_weights=q)
            for j in range(20):
                sums = []
                for sign in (1, -1):
                    v = z.clone()
                    v[:, j] += sign * step
                    _, i2, w2, _ = ops.route_topk(v, 20, scoring, renormalise=False, scale=1.0)
                    s = torch.zeros_like(z).scatter_(1, i2.long(), w2).gather(1, idx.long()).double()      # scores of the same experts
                    w = 2.5 * (s / s.sum(1, keepdim=True) if renormalise else s)
                    sums.append((w * q.double()).sum(1))
                quotient = (sums[0] - sums[1]) / (2 * step)
                assert (quotient - grad[:, j].double()).abs().max() < 1e-3


@pytest.mark.parametrize('t', [torch.float32, torch.bfloat16])
def test_differentiable_function_and_layer(t):
    """The MoE layer's gates by scores: routing equal to the composition in PyTorch, router gradients through both experts modes
    that can be trained, and the weighted routing honoured by the HIP experts."""
    from d2dmoe_amd import MoeficationMoE, MoeficationRouter, functional
    from d2dmoe_amd.layer import route_topk_torch
    torch.manual_seed(3)
    moe = MoeficationMoE('m', 256, 32, True, 16, torch.nn.ReLU)
    moe.router = MoeficationRouter(256, 32, width=64, depth=2, activation='relu', output_activation='identity')
    moe = moe.to(DEV).to(t)
    x = torch.randn(3, 50, 256, device=DEV).to(t)
    moe.k, moe.collect_counts = 5, True
    for mode, scoring in (('softmax_topk', 'softmax'), ('sigmoid_topk', 'sigmoid')):
        moe.forward_mode = mode
        moe.n_groups, moe.kept_groups = (4, 2) if scoring == 'sigmoid' else (1, 1)
        moe.balance_bias = 0.05 * torch.randn(32, device=DEV) if scoring == 'sigmoid' else None
        logits = moe.router(x)
        bias = None if moe.balance_bias is None else moe.balance_bias.float()
        args = (5, scoring, bias, moe.n_groups, moe.kept_groups)
        routing, indices, weights, counts = functional.route_topk(logits, *args, want_counts=True)
        ref, ref_idx, ref_w = route_topk_torch(logits, *args)
        assert indices.shape == weights.shape == (3, 50, 5) and torch.equal(indices, ref_idx)
        assert (weights - ref_w).abs().max() <= 128 * U
        q, g = torch.randn_like(weights), torch.randn_like(routing)
        a = torch.autograd.grad((routing, weights), logits, (g, q), retain_graph=True)[0]
        c = torch.autograd.grad((ref, ref_w), logits, (g, q), retain_graph=True)[0]
        # the composition rounds routing's gradient and the sum of the two once more
        assert (a - c).abs().max() <= 4 * _half(t) * c.abs().max() + 1e-5
        assert torch.equal(counts.long(), torch.bincount(indices.flatten().long(), minlength=32))
        # the layer: masked experts train, HIP experts answer; both see the same weighted routing
        moe.experts.forward_mode = 'masked'
        out, gating = moe(x)
        out.float().square().mean().backward()
        grad = moe.router.layers[0].weight.grad
        assert torch.isfinite(grad).all() and grad.abs().sum() > 0
        assert torch.equal(moe.last_expert_counts.long(), (gating['m'][0] != 0).sum((0, 1)))
        moe.zero_grad()
        moe.experts.forward_mode = 'hip'
        with torch.no_grad():
            moe.router_logits = None
            got, gating2 = moe(x)
            want = moe.experts.forward_all(x.view(-1, 256).double() if t == torch.float64 else x.view(-1, 256),
                                           gating2['m'][0].view(-1, 32)) + moe.last_bias
        err = (got.view(-1, 256).float() - want.float()).abs().max() / want.float().abs().max()
        assert err < (1e-5 if t == torch.float32 else 2e-2)


def test_together_as_a_block_uses_them():
    """GPT-2 with expert layers routed by scores and every norm on the HIP kernels: one training step in float32 against the same
    model composed in PyTorch, then the served model (norm, router, choice, weighted experts all on the HIP kernels)."""
    from d2dmoe_amd import add_routers, gpt2, set_norm_mode
    from d2dmoe_amd.layer import route_topk_torch
    import d2dmoe_amd.layer as layer_module
    torch.manual_seed(5)
    base = gpt2.GPT(gpt2.GPTConfig(block_size=64, vocab_size=128, n_layer=2, n_head=4, n_embd=256))
    moe, names = gpt2.replace_with_moes(base, num_experts=16)
    gpt2.split_original_parameters(base, moe, names)
    add_routers(moe, dict(width=64, depth=2, bias=False, activation='relu', output_activation='identity'))
    moe = moe.to(DEV)
    idx = torch.randint(0, 128, (2, 64), device=DEV)
    layers = [gpt2.get_module_by_name(moe, n) for n in names]
    for lay in layers:
        lay.forward_mode, lay.k = 'softmax_topk', 4
        lay.experts.forward_mode = 'masked'

    def step():
        moe.zero_grad()
        logits = moe(idx)
        torch.nn.functional.cross_entropy(logits.view(-1, 128).float(), idx.roll(-1, 1).view(-1)).backward()
        return logits.detach().clone(), {k: v.grad.clone() for k, v in moe.named_parameters() if v.grad is not None}

    set_norm_mode(moe, 'hip')
    hip = step()
    kept = functional_route = layer_module.functional.route_topk
    try:
        layer_module.functional.route_topk = lambda z, *a, want_counts=False: (*route_topk_torch(z, *a), None)
        set_norm_mode(moe, 'torch')
        plain = step()
    finally:
        layer_module.functional.route_topk = kept
    assert functional_route is kept
    assert (hip[0] - plain[0]).abs().max() <= 1e-4 * plain[0].abs().max()
    assert set(hip[1]) == set(plain[1]) and any('router' in k for k in hip[1])
    for k in plain[1]:
        assert (hip[1][k] - plain[1][k]).norm() <= 1e-3 * plain[1][k].norm() + 1e-9, k
    # served: everything on the HIP kernels
    set_norm_mode(moe, 'hip')
    for lay in layers:
        lay.experts.forward_mode = 'hip'
    with torch.no_grad():
        served, gating = moe(idx, return_gating_data=True)
    assert (served - plain[0]).abs().max() <= 1e-4 * plain[0].abs().max()
    assert all(((g[0] > 0).sum(-1) == 4).all() for g in gating.values())


def test_the_layer_calls_the_routing_function_once(monkeypatch):
    """On the GPU a gate by scores is functional.route_topk, once per layer and pass; a substitute in its place is what runs."""
    from d2dmoe_amd import add_routers, gpt2
    from d2dmoe_amd.layer import route_topk_torch
    import d2dmoe_amd.layer as layer_module
    torch.manual_seed(6)
    base = gpt2.GPT(gpt2.GPTConfig(block_size=16, vocab_size=32, n_layer=2, n_head=2, n_embd=64))
    moe, names = gpt2.replace_with_moes(base, num_experts=8)
    gpt2.split_original_parameters(base, moe, names)
    add_routers(moe, dict(width=16, depth=2, bias=False, activation='relu', output_activation='identity'))
    moe = moe.to(DEV)
    for name in names:
        lay = gpt2.get_module_by_name(moe, name)
        lay.forward_mode, lay.k, lay.experts.forward_mode = 'sigmoid_topk', 2, 'masked'
    calls = []
    real = layer_module.functional.route_topk

    def counted(run):
        def call(z, *a, want_counts=False):
            calls.append(run)
            return real(z, *a, want_counts=want_counts) if run == 'hip' else (*route_topk_torch(z, *a), None)
        return call

    idx = torch.randint(0, 32, (2, 16), device=DEV)
    found = {}
    for run in ('hip', 'torch'):
        with monkeypatch.context() as m:
            m.setattr(layer_module.functional, 'route_topk', counted(run))
            with torch.no_grad():
                found[run] = moe(idx)
    assert calls == ['hip'] * len(names) + ['torch'] * len(names) and layer_module.functional.route_topk is real
    assert (found['hip'] - found['torch']).abs().max() <= 1e-4 * found['torch'].abs().max()
