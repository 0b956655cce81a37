"""Layer norm and routing by scores without a GPU: the oracle against independent statements, the PyTorch compositions that
run off the GPU, the modules' modes, and every refusal (none of which may reach a device)."""
import contextlib
import ctypes
import math

import numpy as np
import pytest
import torch
from torch.nn import functional as F

from oracle import norm_route as R


def _gen(seed):
    return torch.Generator().manual_seed(seed)


# ------------------------------------------------------------------------------------------------------------ oracle
def test_oracle_layer_norm_is_the_definition_and_its_derivative():
    g = _gen(1)
    h = (torch.randn(5, 33, generator=g, dtype=torch.float64) * 2 + 1).requires_grad_()
    w = torch.randn(33, generator=g, dtype=torch.float64).requires_grad_()
    b = torch.randn(33, generator=g, dtype=torch.float64).requires_grad_()
    go = torch.randn(5, 33, generator=g, dtype=torch.float64)
    want = F.layer_norm(h, (33,), w, b, 1e-5)
    grads = torch.autograd.grad(want, (h, w, b), go)
    out, mean, rstd = R.layer_norm(h.detach().numpy(), w.detach().numpy(), b.detach().numpy(), 1e-5)
    assert np.abs(out - want.detach().numpy()).max() < 1e-12
    got = R.layer_norm_grads(go.numpy(), None, h.detach().numpy(), w.detach().numpy(), 1e-5)
    for a, c in zip(got, grads):
        assert np.abs(a - c.numpy()).max() < 1e-12


def _differences(f, z, step=1e-6):
    """Central differences of the scalar f at every entry of z (float64)."""
    out = np.zeros_like(z)
    for i in np.ndindex(z.shape):
        up, down = z.copy(), z.copy()
        up[i] += step
        down[i] -= step
        out[i] = (f(up) - f(down)) / (2 * step)
    return out


@pytest.mark.parametrize('scoring', ['softmax', 'sigmoid'])
@pytest.mark.parametrize('renormalise', [True, False])
def test_oracle_route_gradient_is_the_difference_quotient(scoring, renormalise):
    g = np.random.RandomState(3)
    z, q = g.randn(4, 9), g.randn(4, 3)
    idx = R.route(z, 3, scoring, renormalise=renormalise, scale=2.5)[1]

    def loss(v):                                     # the choice held fixed: small steps do not change it
        d, i, w = R.route(v, 3, scoring, renormalise=renormalise, scale=2.5)
        assert np.array_equal(i, idx)
        return float((w * q).sum())

    # central differences of step 1e-6: truncation 1e-12 times a third derivative of order 1, rounding 1e-16 / 1e-6
    assert np.abs(R.route_grads(z, idx, q, scoring, renormalise, 2.5) - _differences(loss, z)).max() < 1e-8


def test_oracle_route_by_hand():
    # two groups of two; sums of the two best: 0.9 + 0.1 < 0.6 + 0.5 -> the second group alone stays
    s = np.array([[0.9, 0.1, 0.6, 0.5]])
    z = np.log(s / (1 - s))
    dense, idx, w = R.route(z, 2, 'sigmoid', n_groups=2, kept_groups=1, group_score='top2')
    assert idx.tolist() == [[2, 3]] and np.allclose(w, [[0.6 / 1.1, 0.5 / 1.1]])
    assert R.route(z, 2, 'sigmoid', n_groups=2, kept_groups=1, group_score='max')[1].tolist() == [[0, 1]]
    # the bias decides the choice and not the weights
    assert R.route(z, 1, 'sigmoid', bias=np.array([0, 1.0, 0, 0]), renormalise=False)[1].tolist() == [[1]]
    assert np.allclose(R.route(z, 1, 'sigmoid', bias=np.array([0, 1.0, 0, 0]), renormalise=False)[2], 0.1)
    # ties to the lowest index, masked experts never, rows with nothing
    inf = math.inf
    assert R.route(np.array([[1.0, 2.0, 2.0, -inf]]), 4, 'softmax')[1].tolist() == [[1, 2, 0, -1]]
    assert R.route(np.array([[-inf] * 3, [1, math.nan, 2], [1, inf, 2]]), 2, 'softmax')[1].tolist() == [[-1, -1]] * 3
    assert R.route(np.array([[1, inf, 2.0]]), 2, 'sigmoid')[1].tolist() == [[1, 2]]


# ------------------------------------------------------------------------------------- the compositions off the GPU
ROUTES = [dict(k=1), dict(k=3), dict(k=4, renormalise=False, scale=2.5), dict(k=2, bias=True),
          dict(k=3, bias=True, n_groups=4, kept_groups=2), dict(k=5, n_groups=2, kept_groups=2, group_score='max'),
          dict(k=2, n_groups=6, kept_groups=3, renormalise=False), dict(k=12)]


@pytest.mark.parametrize('scoring', ['softmax', 'sigmoid'])
@pytest.mark.parametrize('kw', ROUTES)
@pytest.mark.parametrize('dtype', [torch.float64, torch.float32, torch.bfloat16])
def test_composed_route_matches_the_oracle_with_its_gradient(scoring, kw, dtype):
    from d2dmoe_amd.layer import route_topk_torch
    kw = dict(kw)
    g = _gen(11)
    z = (torch.randn(40, 12, generator=g) * 1.5).to(dtype)
    z[3] = float('-inf')
    z[5, 4] = float('nan')
    z[7, 2:9] = float('-inf')
    z[9] = z[9, 0]
    bias = torch.randn(12, generator=g) * 0.2 if kw.pop('bias', False) else None
    k = kw.pop('k')
    want, idx, w = R.route(z.double().numpy(), k, scoring, bias=None if bias is None else bias.numpy(), **kw)
    z.requires_grad_()
    routing, indices, weights = route_topk_torch(z, k, scoring, bias, **kw)
    assert routing.dtype == dtype and np.array_equal(indices.numpy(), idx)
    # float32: logsumexp, exp and a division, a few roundings each; one more for the storage type
    half = torch.finfo(dtype).eps / 2 if dtype != torch.float64 else 0.0
    scale = kw.get('scale', 1.0)
    tol = 16 * (2.0 ** -24 if dtype != torch.float64 else 2.0 ** -52) * scale
    assert np.abs(weights.detach().double().numpy() - w).max() <= tol
    assert (np.abs(routing.detach().double().numpy() - want) <= tol + half * np.abs(want)).all()
    q = torch.randn(40, k, generator=g, dtype=weights.dtype)
    grad, = torch.autograd.grad(weights, z, q)
    ref = R.route_grads(z.detach().double().numpy(), idx, q.double().numpy(), scoring, kw.get('renormalise', True), scale)
    bound = 8 * tol * q.abs().max().item() * k
    assert (np.abs(grad.double().numpy() - ref) <= bound + half * np.abs(ref)).all()


def test_layer_gates_by_scores_on_the_cpu():
    from d2dmoe_amd import MoeficationMoE, MoeficationRouter
    torch.manual_seed(0)
    moe = MoeficationMoE('m', 16, 8, True, 4, torch.nn.ReLU)
    keys = set(moe.state_dict())
    moe.router = MoeficationRouter(16, 8, width=16, depth=2, activation='relu', output_activation='identity')
    assert 'balance_bias' not in keys
    x = torch.randn(2, 5, 16)
    moe.k = 3
    for mode, scoring in (('softmax_topk', 'softmax'), ('sigmoid_topk', 'sigmoid')):
        moe.forward_mode = mode
        moe.collect_counts = True
        routing = moe.gate(x)
        want, idx, _ = R.route(moe.router(x).detach().double().view(10, 8).numpy(), 3, scoring)
        assert np.abs(routing.detach().double().view(10, 8).numpy() - want).max() < 1e-6
        assert np.array_equal(moe.last_expert_counts.numpy(), np.bincount(idx.ravel(), minlength=8))
        moe.experts.forward_mode = 'masked'
        out, gating = moe(x)
        masked = moe.experts.forward_all(x.view(-1, 16), routing.view(-1, 8)) + moe.last_bias
        assert torch.allclose(out.view(-1, 16), masked, atol=1e-6) and torch.equal(gating['m'][0], routing)
        out.sum().backward()
        assert moe.router.layers[0].weight.grad.abs().sum() > 0
    # the balance bias is saved with the layer once it is set, and moves the choice only
    moe.balance_bias = torch.zeros(8)
    moe.balance_bias[6] = 10.0
    assert 'balance_bias' in moe.state_dict()
    assert (moe.gate(x)[..., 6] > 0).all()
    fresh = MoeficationMoE('m', 16, 8, True, 4, torch.nn.ReLU)
    fresh.router = MoeficationRouter(16, 8, width=16, depth=2, activation='relu', output_activation='identity')
    fresh.load_state_dict(moe.state_dict())
    assert torch.equal(fresh.balance_bias, moe.balance_bias)
    with pytest.raises(ValueError):
        fresh.forward_mode = 'softmax_topk'
        fresh.gate(x)


def test_norm_modules_off_the_gpu():
    from d2dmoe_amd import D2DMoEError, gpt2, set_norm_mode, vit
    torch.manual_seed(1)
    m = gpt2.GPT(gpt2.GPTConfig(block_size=8, vocab_size=32, n_layer=2, n_head=2, n_embd=16)).eval()
    v = vit.VisionTransformer(image_size=32, num_layers=1, num_heads=2, hidden_dim=16, mlp_dim=32, num_classes=4).eval()
    idx = torch.randint(0, 32, (2, 8), generator=_gen(2))
    ln = m.transformer.h[0].ln_1
    x = torch.randn(3, 16)
    assert torch.equal(ln(x), F.layer_norm(x, (16,), ln.weight, ln.bias, 1e-5))
    vn = v.encoder.ln
    assert torch.equal(vn(x), F.layer_norm(x, (16,), vn.weight, vn.bias, 1e-6))
    assert set_norm_mode(m, 'hip') == 5 and set_norm_mode(v, 'hip') == 3
    with pytest.raises(D2DMoEError):
        m(idx)                                        # there is no CPU fallback behind 'hip'
    with pytest.raises(D2DMoEError):
        ln(x, x)
    set_norm_mode(m, 'torch')
    assert torch.isfinite(m(idx)).all()
    out, h = ln(x, x)
    assert torch.equal(h, x + x) and torch.equal(out, ln(h))
    with pytest.raises(ValueError):
        set_norm_mode(m, 'fast')
    ln.forward_mode = 'fast'
    with pytest.raises(NotImplementedError):
        ln(x)
    # a block whose second norm was replaced by another module still adds the residual
    m.transformer.h[0].ln_1.forward_mode = 'torch'
    m.transformer.h[0].ln_2 = torch.nn.Identity()
    assert torch.isfinite(m(idx)).all()


# ---------------------------------------------------------------------------------------------------------- refusals
def test_c_entry_points_refuse_before_anything_is_launched():
    """Dummy pointers: a call that passed its checks would fault, so every status below is a host-side refusal."""
    from d2dmoe_amd import hip_abi as abi
    lib = abi.load()
    p = 4096

    def norm(n=4, d=8, dtype=abi.BF16, param=abi.BF16, eps=1e-5, x=p, out=p, residual=None, weight=None, mean=None, total=None):
        sh = abi.NormShape(n, d, dtype, param, eps)
        return lib.d2dmoe_layer_norm(ctypes.byref(sh), x, residual, weight, None, total, out, mean, None, None)

    assert lib.d2dmoe_layer_norm(None, p, None, None, None, None, p, None, None, None) == -1
    assert norm(x=None) == norm(out=None) == norm(total=p) == -1
    assert norm(n=-1) == -2 and norm(d=0) == -2 and norm(d=(1 << 24) + 1) == -2 and norm(n=1 << 62) == -2
    assert norm(dtype=7) == -3 and norm(param=abi.F16) == -3 and norm(dtype=abi.F32, param=abi.BF16) == -3
    assert norm(eps=-1.0) == norm(eps=math.nan) == norm(eps=math.inf) == abi.E_VALUE
    assert norm(x=p + 1) == norm(residual=p + 1) == norm(weight=p + 1) == norm(mean=p + 2) == -7
    assert norm(param=abi.F32, weight=p + 2) == -7
    assert norm(n=0, x=None, out=None) == 0
    assert b'scalar' in lib.d2dmoe_status_string(abi.E_VALUE)

    def back(n=4, go=p, h=p, mean=p, rstd=p, grad=p, gw=p, gb=p, ws=p, nbytes=1 << 30, gs=None, weight=None):
        sh = abi.NormShape(n, 8, abi.BF16, abi.BF16, 0.0)
        return lib.d2dmoe_layer_norm_backward(ctypes.byref(sh), go, gs, h, weight, mean, rstd, grad, gw, gb, ws, nbytes, None)

    assert back(go=None) == back(h=None) == back(mean=None) == back(rstd=None) == back(grad=None, gw=None, gb=None) == -1
    assert back(ws=None) == back(nbytes=4) == back(ws=p + 16) == -5
    assert back(grad=p + 1) == back(gs=p + 1) == back(mean=p + 2) == back(gb=p + 1) == -7
    assert back(n=0, gw=None, gb=None) == 0
    sh = abi.NormShape(1000, 768, abi.BF16, abi.F32, 0.0)
    ws = lib.d2dmoe_layer_norm_workspace_bytes(ctypes.byref(sh))
    assert ws >= 2 * 768 * 4 and ws % 256 == 0
    assert lib.d2dmoe_layer_norm_workspace_bytes(ctypes.byref(abi.NormShape(0, 768, abi.BF16, abi.F32, 0.0))) == 0
    assert lib.d2dmoe_layer_norm_workspace_bytes(ctypes.byref(abi.NormShape(9, 0, abi.BF16, abi.F32, 0.0))) == 0

    def route(n=4, e=8, k=2, dtype=abi.F32, scoring=0, groups=1, kept=1, score=1, renorm=1, scale=1.0, logits=p, bias=None,
              routing=p, indices=p, weights=p, counts=None):
        rs = abi.RouteShape(n, e, k, dtype, scoring, groups, kept, score, renorm, scale)
        return lib.d2dmoe_route_topk(ctypes.byref(rs), logits, bias, routing, indices, weights, counts, None)

    assert lib.d2dmoe_route_topk(None, p, None, p, p, p, None, None) == -1
    assert route(logits=None) == route(routing=None, indices=None, weights=None) == route(indices=None, counts=p) == -1
    assert route(n=-1) == route(e=0) == route(e=1025) == route(k=0) == route(k=9) == -2
    assert route(groups=3, kept=1) == route(groups=0) == route(groups=4, kept=5) == route(groups=4, kept=0) == -2
    assert route(groups=4, kept=1, k=3) == -2
    assert route(dtype=5) == -3
    assert route(scoring=2) == route(renorm=2) == route(scale=math.nan) == route(scale=math.inf) == abi.E_VALUE
    assert route(groups=4, kept=2, score=2) == abi.E_VALUE
    assert route(logits=p + 2) == route(bias=p + 1) == route(indices=p + 2) == route(weights=p + 2) == route(counts=p + 2) == -7
    assert route(n=0, logits=None, routing=None, indices=None, weights=None) == 0

    def grad(n=4, k=2, logits=p, indices=p, gr=p, gw=None, out=p, scoring=0):
        rs = abi.RouteShape(n, 8, k, abi.F32, scoring, 0, 0, 9, 1, 1.0)     # the fields of the choice are not read
        return lib.d2dmoe_route_topk_backward(ctypes.byref(rs), logits, indices, gr, gw, out, None)

    assert grad(logits=None) == grad(indices=None) == grad(gr=None) == grad(out=None) == -1
    assert grad(k=9) == -2 and grad(scoring=4) == abi.E_VALUE
    assert grad(gr=p + 2) == grad(gw=p + 2) == grad(out=p + 1) == -7
    assert grad(n=0) == 0


def test_a_call_runs_on_its_tensors_device(monkeypatch):
    """The current device is another one than the tensors': the call switches to theirs and takes that device's stream."""
    from d2dmoe_amd import ops
    seen = []

    class Device:
        def __init__(self, dev):
            self.dev = dev

        def __enter__(self):
            seen.append(('enter', self.dev))

        def __exit__(self, *_):
            seen.append(('leave', self.dev))

    monkeypatch.setattr(torch.cuda, 'current_device', lambda: 0)
    monkeypatch.setattr(torch.cuda, 'device', Device)
    monkeypatch.setattr(ops, '_raw_stream', lambda index: 1000 + index)

    def call(*args):
        seen.append(args)
        return 0

    ops._launch(3, call, 'call', 7)
    assert seen == [('enter', 3), (7, 1003), ('leave', 3)]
    seen.clear()
    ops._launch(0, call, 'call', 7)
    assert seen == [(7, 1000)]


def test_numbers_beyond_32_bits_are_refused_not_cut():
    """The C records hold 32-bit fields, and ctypes drops what does not fit: 2^32 + 1 groups would run as one."""
    from d2dmoe_amd import D2DMoEError, ops
    x = torch.randn(4, 8)
    for far in (1 << 32, (1 << 32) + 1, (1 << 31), -(1 << 32) + 1):
        for args in (dict(n_groups=far), dict(kept_groups=far), dict(k=far)):
            with pytest.raises(D2DMoEError, match='32 bits'):
                ops._route_shape('route_topk', x, **{**dict(k=2, scoring='softmax', renormalise=True, scale=1.0), **args})
    with pytest.raises(D2DMoEError, match='32 bits'):
        ops._route_record(4, (1 << 32) + 8, 2, 0, 0, 1, 1, 0, 1, 1.0)
    with pytest.raises(D2DMoEError, match='32 bits'):
        ops._norm_shape(1, (1 << 32) + 8, 1, 1, 1e-5)
    assert ops._norm_shape(1 << 40, 8, 1, 1, 1e-5)[0]._obj.n_rows == 1 << 40      # (rows and tokens are 64-bit)


def test_forward_mode_derivatives_are_refused_not_lost(monkeypatch):
    """A dual tensor that asks for no reverse-mode gradient must not come out without its tangent.  The kernel calls are replaced:
    what is tested is what stands in front of them."""
    from d2dmoe_amd import functional, ops
    from torch.autograd import forward_ad
    monkeypatch.setattr(ops, 'layer_norm', lambda x, w, b, eps, r, want_stats=False: (x * 1.0, None if r is None else x + r, None, None))
    monkeypatch.setattr(ops, 'route_topk', lambda z, k, *args: (z * 1.0, torch.zeros(z.size(0), k, dtype=torch.int32),
                                                               torch.ones(z.size(0), k), None))
    x, w = torch.randn(4, 8), torch.ones(8)
    with forward_ad.dual_level():
        dual, dual_w = forward_ad.make_dual(x, torch.ones_like(x)), forward_ad.make_dual(w, w)
        for grad in (True, False):
            with torch.set_grad_enabled(grad):
                for call in (lambda: functional.layer_norm(dual, w), lambda: functional.layer_norm(x, w, residual=dual),
                             lambda: functional.layer_norm(x, dual_w), lambda: functional.layer_norm(x, w, dual_w),
                             lambda: functional.route_topk(dual, 2)):
                    with pytest.raises(NotImplementedError):
                        call()
        # tensors without a tangent pass as ever
        assert functional.layer_norm(x, w).shape == (4, 8) and functional.route_topk(x, 2)[1].shape == (4, 2)


def _norm_calls(monkeypatch):
    """The 'hip' mode off the GPU: the kernel call replaced by its formula, with the refusal of two element types that it has."""
    from d2dmoe_amd import D2DMoEError, norm, ops
    seen = []

    def layer_norm(x, w=None, b=None, eps=1e-5, residual=None, want_stats=False):
        if residual is not None and residual.dtype != x.dtype:
            raise D2DMoEError('two element types')
        ops._norm_params('layer_norm', x.size(1), x.dtype, w, b)
        seen.append((x.dtype, None if residual is None else residual.dtype))
        h = x if residual is None else x + residual
        out = F.layer_norm(h.float(), (h.size(1),), None if w is None else w.float(), None if b is None else b.float(), eps).to(x.dtype)
        return out, None if residual is None else h, None, None

    monkeypatch.setattr(ops, 'layer_norm', layer_norm)
    monkeypatch.setattr(norm.NormModes, '_hip', lambda self, x: self.forward_mode == 'hip')
    return seen


@pytest.mark.parametrize('bias', [True, False])
def test_hip_norm_takes_the_element_types_of_the_torch_mode(bias, monkeypatch):
    """Two element types, and autocast: the sum has the wider type, and under autocast the norm is float32."""
    from d2dmoe_amd import gpt2
    from d2dmoe_amd.norm import add_norm
    seen = _norm_calls(monkeypatch)
    n = gpt2.LayerNorm(16, bias)
    n.forward_mode = 'hip'
    x, r = torch.randn(3, 16), torch.randn(3, 16)

    @contextlib.contextmanager
    def autocast():                                              # (torch's own switches itself off where there is no GPU)
        with monkeypatch.context() as m:
            m.setattr(torch, 'is_autocast_enabled', lambda kind: kind == 'cuda')
            yield

    with torch.no_grad():
        for tx in (torch.bfloat16, torch.float16, torch.float32):
            for tr in (torch.bfloat16, torch.float16, torch.float32):
                wide = torch.promote_types(tx, tr)
                a, b = x.to(tx), r.to(tr)
                out, h = add_norm(n, a, b)
                assert out.dtype == h.dtype == wide and torch.equal(h, a + b) and seen[-1] == (wide, wide)
                with autocast():
                    out, h = add_norm(n, a, b)
                    alone = n(a)
                # what F.layer_norm gives there on a GPU, and an addition: float32, and the wider type
                assert out.dtype == alone.dtype == torch.float32 and h.dtype == wide and torch.equal(h, a + b)
                assert torch.equal(out, F.layer_norm((a + b).float(), (16,), n.weight, n.bias, 1e-5))
        # 16-bit parameters under autocast, as F.layer_norm takes them
        n.bfloat16()
        with autocast():
            assert n(x).dtype == torch.float32


@pytest.mark.parametrize('mode', ['softmax_topk', 'sigmoid_topk'])
def test_layer_refuses_a_scale_that_routes_nothing(mode):
    """The experts count an entry of the routing tensor as routed where it is above zero: with a scale that is not, the containers
    would disagree ('masked' applies such weights, the others drop every token)."""
    from d2dmoe_amd import MoeficationMoE, MoeficationRouter
    moe = MoeficationMoE('m', 16, 8, True, 4, torch.nn.ReLU)
    moe.router = MoeficationRouter(16, 8, width=16, depth=2, activation='relu', output_activation='identity')
    moe.forward_mode, moe.k = mode, 3
    x = torch.randn(2, 5, 16)
    for scale in (0.0, -1.0, math.nan, -math.inf, math.inf):
        moe.route_scale = scale
        with pytest.raises(ValueError, match='route_scale'):
            moe.gate(x)
    moe.route_scale = 0.5
    assert ((moe.gate(x) > 0).sum(-1) == 3).all()


def test_composed_route_refuses_what_the_kernel_call_refuses():
    """The same settings of a gate must not answer on the CPU and raise on the GPU (or answer otherwise: any group_score but 'top2'
    went as 'max', k beyond the kept groups left places over)."""
    from d2dmoe_amd import D2DMoEError
    from d2dmoe_amd.layer import route_topk_torch
    z = torch.randn(2, 3, 8)
    for kw in (dict(k=0), dict(k=9), dict(k=2, scoring='tanh'), dict(k=2, group_score='mean'), dict(k=2, n_groups=3), dict(k=2, n_groups=0),
               dict(k=2, n_groups=4, kept_groups=0), dict(k=2, n_groups=4, kept_groups=5), dict(k=3, n_groups=4, kept_groups=1),
               dict(k=2, kept_groups=2), dict(k=2, choice_bias=torch.zeros(1)), dict(k=2, choice_bias=torch.zeros(3, 8)),
               dict(k=2, scale=math.inf), dict(k=2, scale=math.nan)):
        with pytest.raises(D2DMoEError):
            route_topk_torch(z, **kw)
    assert route_topk_torch(z, 2, n_groups=4, kept_groups=1)[1].shape == (2, 3, 2)


def test_differentiable_route_copies_a_strided_bias(monkeypatch):
    """As it does strided logits: a column of a table of biases is a bias."""
    from d2dmoe_amd import functional, ops
    got = []
    monkeypatch.setattr(ops, 'route_topk', lambda z, k, scoring, bias, *args: (got.append((z, bias)), z, z[:, :k], z[:, :k], None)[1:])
    table = torch.randn(8, 3)
    z = torch.randn(8, 4).t()
    functional.route_topk(z, 2, 'sigmoid', table[:, 1])
    assert got[0][0].is_contiguous() and torch.equal(got[0][0], z)
    assert got[0][1].is_contiguous() and torch.equal(got[0][1], table[:, 1])


@pytest.mark.parametrize('shape', [(4, 8), (2, 2, 8), (8,), (0, 3, 8)])
@pytest.mark.parametrize('strided', [False, True])
def test_gradients_of_x_and_residual_are_tensors_of_their_own(shape, strided, monkeypatch):
    """Both are the same numbers, computed once.  As two views of one tensor they became the .grad of two leaves in the same
    memory, and a second backward pass added itself to it twice.  (Kernel calls replaced by a stream of ones.)"""
    from d2dmoe_amd import functional, ops

    def forward(x, w, b, eps, r, want_stats=False):
        assert x.dim() == 2 and x.is_contiguous() and (r is None or r.is_contiguous())
        return x * 1.0, None if r is None else x + r, torch.zeros(x.size(0)), torch.ones(x.size(0))

    def backward(g, h, w, mean, rstd, gs=None, want_grad=True, want_weight=True, want_bias=True, param_dtype=None):
        assert g.shape == h.shape and g.is_contiguous() and (gs is None or gs.shape == h.shape and gs.is_contiguous())
        return g.clone() if gs is None else g + gs, None, None

    monkeypatch.setattr(ops, 'layer_norm', forward)
    monkeypatch.setattr(ops, 'layer_norm_backward', backward)

    def leaf():
        t = torch.randn(shape)
        return (t.transpose(0, -1).contiguous().transpose(0, -1) if strided else t).requires_grad_()

    for use in ('both', 'out', 'sum'):
        x, r = leaf(), leaf()
        for i in range(1, 4):
            out, h = functional.layer_norm(x, residual=r)
            assert out.shape == h.shape == shape
            loss = (out.sum() if use != 'sum' else 0) + (h.sum() if use != 'out' else 0)
            loss.backward()
            each = 2.0 * i if use == 'both' else float(i)
            assert (x.grad == each).all() and (r.grad == each).all()
        if x.numel():
            assert x.grad.data_ptr() != r.grad.data_ptr()
    # what comes back may be changed in place, and what the backward pass needs may not unseen
    x, r = leaf(), leaf()
    out, h = functional.layer_norm(x, residual=r)
    out.mul_(2.0)
    (out.sum() + h.sum()).backward()
    assert (x.grad == 3.0).all() and (r.grad == 3.0).all()
    out, h = functional.layer_norm(x, residual=r)
    h.add_(1.0)
    with pytest.raises(RuntimeError):
        out.sum().backward()
    # one tensor in both places
    x = leaf()
    for i in range(1, 3):
        out, h = functional.layer_norm(x, residual=x)
        out.sum().backward()
        assert (x.grad == 2.0 * i).all()


def test_a_saved_bias_of_another_number_of_experts_does_not_load():
    """A layer without a balance bias takes a saved one, of its own number of experts only."""
    from d2dmoe_amd import MoeficationMoE
    moe, other = (MoeficationMoE('m', 16, 8, True, 4, torch.nn.ReLU) for _ in range(2))
    state = moe.state_dict()
    state['balance_bias'] = torch.zeros(7)
    with pytest.raises(RuntimeError, match='balance_bias'):
        other.load_state_dict(state)
    state['balance_bias'] = torch.arange(8.0)
    other.load_state_dict(state)
    assert torch.equal(other.balance_bias, torch.arange(8.0))


class _Standin:
    """A tensor as far as the device check goes; -1: on the CPU."""

    def __init__(self, index, contiguous=True):
        self.index, self.contiguous = index, contiguous

    def get_device(self):
        return self.index

    def is_contiguous(self):
        return self.contiguous


def test_device_check_in_any_order():
    """A tensor on the CPU is refused wherever it stands among tensors on a GPU: its address would reach the kernel."""
    from d2dmoe_amd import D2DMoEError, ops
    for where in ((-1, 0), (0, -1), (-1, -1), (None, -1, 0), (-1, None, 0, 0), (0, None, -1), (0, 1), (1, 0), (None, 2, 2, 3), (None,), ()):
        with pytest.raises(D2DMoEError):
            ops._gpu_index(*(None if i is None else _Standin(i) for i in where))
    for where, index in (((0,), 0), ((None, 3, None, 3), 3), ((1, 1, 1), 1)):
        assert ops._gpu_index(*(None if i is None else _Standin(i) for i in where)) == index
    with pytest.raises(D2DMoEError):
        ops._gpu_index(_Standin(0), _Standin(0, contiguous=False))


def test_tensor_level_refusals():
    from d2dmoe_amd import D2DMoEError, functional, ops
    x = torch.randn(4, 8)
    ok = torch.ones(8)
    stats = torch.zeros(4)
    idx = torch.zeros(4, 2, dtype=torch.int32)
    for call in (
            lambda: ops.layer_norm(x, ok),                                            # CPU tensors
            lambda: ops.layer_norm(x.double()),                                       # element type
            lambda: ops.layer_norm(x.view(2, 2, 8), ok),                              # dimensions
            lambda: ops.layer_norm(x, torch.ones(7)),                                 # parameter width
            lambda: ops.layer_norm(x, ok.bfloat16()),                                 # parameter narrower than the rows
            lambda: ops.layer_norm(x.bfloat16(), ok, ok.bfloat16()),                  # two parameter types
            lambda: ops.layer_norm(x, ok, residual=x[:2]),                            # residual shape
            lambda: ops.layer_norm(x, ok, residual=x.half()),                         # residual type
            lambda: ops.layer_norm_backward(x, x, ok, stats[:3], stats),              # statistics of other rows
            lambda: ops.layer_norm_backward(x.half(), x, ok, stats, stats),           # gradient type
            lambda: ops.layer_norm_backward(x, x, ok, stats, stats, x[:, :4]),        # shape of the residual's gradient
            lambda: ops.layer_norm_backward(x, x, None, stats, stats, param_dtype=torch.float16),
            lambda: ops.layer_norm_backward(x, x, ok, stats, stats),                  # CPU tensors
            lambda: ops.route_topk(x, 2),                                             # CPU tensors
            lambda: ops.route_topk(x, 2, scoring='tanh'),
            lambda: ops.route_topk(x, 2, group_score='mean'),
            lambda: ops.route_topk(x, 2, choice_bias=torch.zeros(7)),
            lambda: ops.route_topk(x, 2, choice_bias=torch.zeros(8, dtype=torch.float64)),
            lambda: ops.route_topk(x[0], 2),
            lambda: ops.route_topk_backward(x, idx),                                  # no gradient given
            lambda: ops.route_topk_backward(x, idx.long(), grad_weights=torch.zeros(4, 2)),
            lambda: ops.route_topk_backward(x, idx[:3], grad_weights=torch.zeros(3, 2)),
            lambda: ops.route_topk_backward(x, idx, grad_weights=torch.zeros(4, 3)),
            lambda: ops.route_topk_backward(x, idx, grad_routing=x.half()),
            lambda: functional.layer_norm(x, ok, residual=x[0]),
            lambda: functional.route_topk(x, 2)):
        with pytest.raises(D2DMoEError):
            call()
