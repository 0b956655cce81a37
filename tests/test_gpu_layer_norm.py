"""Layer norm on the GPU against the float64 oracle.

Tolerances.  u = 2^-24 (half a float32 step), t = half a step of the storage type.  With n = (h - m) r and K roundings in a
row's sums (a thread adds at most D / 64 + 8 values in a chain, the rest are trees), the kernel's n is off by at most
u (K + 8) (|n| + 1) -- the centred value, the variance under the root, the product -- so out by
u (K + 8) (|n| + 1) |w| + 2 u (|out| + |b|), and the stored value by t |out| more.  The backward pass adds the stored
float32 mean's rounding, u |m| r in n.  A column sum of N products in any order is off by u (N + 64) times the sum of their sizes.
2^-25 is half of float16's smallest step."""
import ctypes

import numpy as np
import pytest
import torch
from torch.nn import functional as F

from oracle import norm_route as R

pytestmark = pytest.mark.gpu

DEV = 'cuda:0'
U = 2.0 ** -24
TINY = 2.0 ** -25
SHAPES = [(1, 1), (2, 2), (5, 3), (3, 7), (4, 8), (5, 64), (17, 253), (2, 1001), (67, 768), (300, 1280), (33, 2048), (21, 2056), (9, 4096),
          (5, 4100), (3, 8200), (2, 16384), (2, 20001), (1, 70000), (1030, 96), (4099, 40), (71, 65), (333, 121),
          (129, 128), (77, 200), (1500, 256), (3, 30000)]
TYPES = [(torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16), (torch.bfloat16, torch.float32),
         (torch.float16, torch.float16), (torch.float16, torch.float32)]


def _ops():
    from d2dmoe_amd import ops
    return ops


def _half(t):
    return torch.finfo(t).eps / 2


def _inputs(n, d, t, p, seed, residual=True, spread=1.0, mean=0.3):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(n, d, generator=g) * spread + mean).to(t)
    r = (torch.randn(n, d, generator=g) * 0.5).to(t) if residual else None
    w = (1 + 0.3 * torch.randn(d, generator=g)).to(p)
    b = (0.2 * torch.randn(d, generator=g)).to(p)
    go = torch.randn(n, d, generator=g).to(t)
    gs = torch.randn(n, d, generator=g).to(t) if residual else None
    return x, r, w, b, go, gs


def _dev(*ts):
    return [None if t is None else t.to(DEV) for t in ts]


def _np(t):
    return None if t is None else t.detach().double().cpu().numpy()


def _check_forward(out, h, w, b, eps, t):
    want, mean, rstd = R.layer_norm(_np(h), _np(w), _np(b), eps)
    d = h.size(1)
    n = np.abs((_np(h) - mean[:, None]) * rstd[:, None])
    wa = np.abs(_np(w)) if w is not None else 1.0
    ba = np.abs(_np(b)) if b is not None else 0.0
    tol = U * (d / 64 + 16) * (n + 1) * wa + 2 * U * (np.abs(want) + ba)
    tol = tol * (1 + _half(t)) + _half(t) * np.abs(want) + TINY
    err = np.abs(_np(out) - want)
    assert out.dtype == t and (err <= tol).all(), (err - tol).max()
    return mean, rstd


def _check_backward(got, go, gs, h, w, eps, t, p):
    grad, gw, gb = got
    want, want_w, want_b = R.layer_norm_grads(_np(go), _np(gs), _np(h), _np(w), eps)
    _, mean, rstd = R.layer_norm(_np(h), None, None, eps)
    n_rows, d = h.shape
    m, r = mean[:, None], rstd[:, None]
    n = (_np(h) - m) * r
    u = _np(go) * (_np(w) if w is not None else 1.0)
    A, B = np.abs(u).mean(1)[:, None], np.abs(u * n).mean(1)[:, None]
    K = d / 64 + 24
    M = np.abs(m) * r
    off = r * (np.abs(u) + A + (np.abs(n) + 1) * (B + A)) * K + 4 * r * M * (B + np.abs(n) * A)
    if gs is not None:
        off = off + np.abs(_np(gs))
    tol = U * off * (1 + _half(t)) + _half(t) * np.abs(want) + TINY
    err = np.abs(_np(grad) - want)
    assert grad.dtype == t and (err <= tol).all(), (err - tol).max()
    a = np.abs(_np(go))
    tol_w = U * ((n_rows + 64) * (a * np.abs(n)).sum(0) + 8 * (a * (np.abs(n) + 1 + M)).sum(0) * (1 + d / 64))
    tol_b = U * (n_rows + 64) * a.sum(0)
    for g, w_, tl in ((gw, want_w, tol_w), (gb, want_b, tol_b)):
        if g is None:
            continue
        err = np.abs(_np(g) - w_)
        assert g.dtype == p and (err <= tl * (1 + _half(p)) + _half(p) * np.abs(w_) + TINY).all(), err.max()


@pytest.mark.parametrize('t,p', TYPES)
@pytest.mark.parametrize('n,d', SHAPES)
def test_forward_and_backward(n, d, t, p):
    print('layer norm', n, d, t, p, flush=True)
    for residual in (True, False):
        x, r, w, b, go, gs = _inputs(n, d, t, p, seed=n + d, residual=residual)
        dx, dr, dw, db, dgo, dgs = _dev(x, r, w, b, go, gs)
        out, total, mean, rstd = _ops().layer_norm(dx, dw, db, 1e-5, dr, want_stats=True)
        h = x if r is None else (x.float() + r.float()).to(t)
        if residual:
            assert torch.equal(total.cpu(), h)
        else:
            assert total is None
        m, rs = _check_forward(out, h, w, b, 1e-5, t)
        assert np.abs(_np(mean) - m).max() <= U * (2 * np.abs(m).max() + (d / 64 + 16) * (1 / rs).max())
        assert (np.abs(_np(rstd) - rs) <= U * (d / 64 + 16) * rs).all()
        got = _ops().layer_norm_backward(dgo, dx if total is None else total, dw, mean, rstd, dgs)
        _check_backward(got, go, gs, h, w, 1e-5, t, p)
        # same inputs, same bits
        again = _ops().layer_norm_backward(dgo, dx if total is None else total, dw, mean, rstd, dgs)
        assert all(torch.equal(a, c) for a, c in zip(got, again))


@pytest.mark.parametrize('t,p', TYPES)
@pytest.mark.parametrize('n,d', [(270, 12288), (259, 10001), (258, 16381), (3, 8193), (262, 4100), (260, 7383)])
def test_wide_rows_in_turn(n, d, t, p):
    """More wide rows than workgroups: each takes several, one after the other."""
    test_forward_and_backward(n, d, t, p)


@pytest.mark.parametrize('d', [768, 77])
def test_optional_operands(d):
    """Each of weight, bias and the outputs may be missing; what is there does not change."""
    x, r, w, b, go, _ = _inputs(40, d, torch.bfloat16, torch.bfloat16, seed=5)
    dx, dr, dw, db, dgo = _dev(x, r, w, b, go)
    for w_, b_ in ((None, None), (w, None), (None, b)):
        out = _ops().layer_norm(dx, *_dev(w_, b_), 1e-5)[0]
        _check_forward(out, x, w_, b_, 1e-5, torch.bfloat16)
    _, total, mean, rstd = _ops().layer_norm(dx, dw, db, 1e-5, dr, want_stats=True)
    full = _ops().layer_norm_backward(dgo, total, dw, mean, rstd)
    for want in ((True, False, False), (False, True, False), (False, False, True), (False, True, True), (False, False, False)):
        part = _ops().layer_norm_backward(dgo, total, dw, mean, rstd, None, *want)
        for on, a, c in zip(want, part, full):
            assert (a is None) == (not on) and (a is None or torch.equal(a, c))
    grad, gw, gb = _ops().layer_norm_backward(dgo, total, None, mean, rstd, param_dtype=torch.float32)
    assert gw is None
    _check_backward((grad, None, gb), go, None, total.cpu(), None, 1e-5, torch.bfloat16, torch.float32)


def test_no_rows():
    e = torch.empty(0, 24, dtype=torch.bfloat16, device=DEV)
    w = torch.ones(24, device=DEV)
    out, total, mean, rstd = _ops().layer_norm(e, w, w, 1e-5, e, want_stats=True)
    assert out.shape == total.shape == (0, 24) and mean.shape == rstd.shape == (0,)
    grad, gw, gb = _ops().layer_norm_backward(e, e, w, mean, rstd, e)
    assert grad.shape == (0, 24) and not gw.any() and not gb.any()      # a sum of no rows is zero, not what was there


@pytest.mark.parametrize('t', [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize('d', [768, 1001])
def test_rows_that_are_not_numbers_stay_alone(t, d):
    x, _, w, b, go, _ = _inputs(9, d, t, t, seed=2, residual=False)
    x[2, 5] = float('nan')
    x[4, d - 1] = float('inf')
    x[6] = 0.25                                      # a constant row: variance zero
    dx, dw, db, dgo = _dev(x, w, b, go)
    out, _, mean, rstd = _ops().layer_norm(dx, dw, db, 1e-5, want_stats=True)
    assert out[2].isnan().all() and out[4].isnan().all()
    keep = [0, 1, 3, 5, 6, 7, 8]
    _check_forward(out[keep], x[keep], w, b, 1e-5, t)
    grad, gw, _ = _ops().layer_norm_backward(dgo, dx, dw, mean, rstd)
    assert grad[2].isnan().all() and torch.isfinite(grad[keep]).all() and gw.isnan().any()


def test_a_mean_far_larger_than_the_spread():
    """h = 1000 + N(0, 1) in float32: the values themselves hold the spread to 2^-15 of it, and the norm loses nothing more.
    The centred values' own sum corrects the mean, so the bound of the other tests holds unchanged."""
    x, _, w, b, _, _ = _inputs(50, 768, torch.float32, torch.float32, seed=8, residual=False, mean=1000.0)
    out = _ops().layer_norm(*_dev(x, w, b), 1e-5)[0]
    _check_forward(out, x, w, b, 1e-5, torch.float32)


@pytest.mark.parametrize('off', [1, 3, 8])
def test_rows_that_start_anywhere_and_bytes_around_them(off):
    """Operands that begin `off` elements into their allocations; the elements before and behind every output stay."""
    from d2dmoe_amd import hip_abi as abi
    lib = abi.load()
    for t, code in ((torch.bfloat16, abi.BF16), (torch.float32, abi.F32)):
        for n, d in ((7, 768), (5, 333), (3, 9000), (2, 40000)):
            print('guards', t, off, n, d, flush=True)
            x, r, w, b, go, gs = _inputs(n, d, t, t, seed=off, residual=True)

            def place(v):
                buf = torch.full((off + v.numel() + 64,), 7.0, dtype=v.dtype, device=DEV)
                buf[off:off + v.numel()] = v.reshape(-1).to(DEV)
                return buf

            bufs = [place(v) for v in (x, r, w, b, go, gs)]
            outs = [torch.full((off + k + 64,), 7.0, dtype=ty, device=DEV)
                    for k, ty in ((n * d, t), (n * d, t), (n, torch.float32), (n, torch.float32), (n * d, t), (d, t), (d, t))]
            at = [v.data_ptr() + off * v.element_size() for v in bufs + outs]
            sh = abi.NormShape(n, d, code, code, 1e-5)
            s = torch.cuda.current_stream().cuda_stream
            abi.check(lib.d2dmoe_layer_norm(ctypes.byref(sh), at[0], at[1], at[2], at[3], at[6], at[7], at[8], at[9], s), 'forward')
            nb = lib.d2dmoe_layer_norm_workspace_bytes(ctypes.byref(sh))
            ws = torch.full((nb + 256,), 7, dtype=torch.uint8, device=DEV)
            abi.check(lib.d2dmoe_layer_norm_backward(ctypes.byref(sh), at[4], at[5], at[6], at[2], at[8], at[9], at[10], at[11], at[12],
                                                     ws.data_ptr(), nb, s), 'backward')
            for v, k in zip(outs, (n * d, n * d, n, n, n * d, d, d)):
                assert (v[:off] == 7.0).all() and (v[off + k:] == 7.0).all()
            assert (ws[nb:] == 7).all()
            cut = [v[off:off + k] for v, k in zip(outs, (n * d, n * d, n, n, n * d, d, d))]
            h = (x.float() + r.float()).to(t)
            assert torch.equal(cut[0].view(n, d).cpu(), h)
            _check_forward(cut[1].view(n, d), h, w, b, 1e-5, t)
            _check_backward((cut[4].view(n, d), cut[5], cut[6]), go, gs, h, w, 1e-5, t, t)


def test_more_than_two_to_the_31_elements():
    n, d = (1 << 21) + 3, 1032
    x = torch.zeros(n, d, dtype=torch.bfloat16, device=DEV)
    tail = torch.randn(5, d, generator=torch.Generator().manual_seed(1)).bfloat16()
    x[-5:] = tail.to(DEV)
    w = torch.ones(d, device=DEV)
    out, _, mean, rstd = _ops().layer_norm(x, w, None, 1e-5, want_stats=True)
    _check_forward(out[-5:], tail, None, None, 1e-5, torch.bfloat16)
    assert not out[:-5].any()
    grad, gw, gb = _ops().layer_norm_backward(x, x, w, mean, rstd)
    _check_backward((grad[-5:], None, None), tail, None, tail, None, 1e-5, torch.bfloat16, torch.float32)
    # the other rows are zero: the column sums are those of the last five
    _, want_w, want_b = R.layer_norm_grads(_np(tail), None, _np(tail), None, 1e-5)
    assert np.abs(_np(gw) - want_w).max() < 1e-4 and np.abs(_np(gb) - want_b).max() < 1e-5
    del x, out, grad


def test_on_a_stream_of_its_own_and_captured():
    """Two captured graphs of forward and backward, replayed in turn with eager work between them, against eager results."""
    ops = _ops()
    side = torch.cuda.Stream()
    cases = []
    for seed, (n, d) in enumerate(((700, 768), (300, 4096))):
        x, r, w, b, go, gs = _dev(*_inputs(n, d, torch.bfloat16, torch.float32, seed=seed))

        def step(x=x, r=r, w=w, b=b, go=go, gs=gs):
            out, total, mean, rstd = ops.layer_norm(x, w, b, 1e-5, r, want_stats=True)
            return (out, total) + ops.layer_norm_backward(go, total, w, mean, rstd, gs)

        eager = [v.clone() for v in step()]
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
                v.fill_(3.0)
            graph.replay()
            step()
            torch.cuda.synchronize()
            for a, c in zip(got, eager):
                assert torch.equal(a, c)


@pytest.mark.parametrize('t,p', [(torch.float32, torch.float32), (torch.bfloat16, torch.float32), (torch.float16, torch.float16)])
def test_differentiable_function(t, p):
    """Through autograd, with strided inputs, broadcast-free leading dimensions, and each leaf alone."""
    from d2dmoe_amd import functional
    x, r, w, b, go, gs = _inputs(24, 320, t, p, seed=4)
    leaves = [v.to(DEV).requires_grad_() for v in (x, r, w, b)]
    X = leaves[0].view(4, 6, 320).transpose(0, 1)             # strided: copied by the function
    Rr = leaves[1].view(4, 6, 320).transpose(0, 1)
    out, h = functional.layer_norm(X, leaves[2], leaves[3], 1e-5, Rr)
    assert out.shape == h.shape == (6, 4, 320)
    go_, gs_ = (v.view(4, 6, 320).transpose(0, 1).to(DEV) for v in (go, gs))
    grads = torch.autograd.grad((out, h), leaves, (go_, gs_), retain_graph=True)
    total = (x.float() + r.float()).to(t)
    _check_backward((grads[0], grads[2], grads[3]), go, gs, total, w, 1e-5, t, p)
    assert torch.equal(grads[0], grads[1])
    for i, leaf in enumerate(leaves):
        alone, = torch.autograd.grad((out, h), leaf, (go_, gs_), retain_graph=True)
        assert torch.equal(alone, grads[i])
    # only the stream used, only the norm used
    only_h, = torch.autograd.grad(h, leaves[1], gs_, retain_graph=True)
    assert torch.equal(only_h, gs.to(DEV))
    only_out = torch.autograd.grad(out, leaves, go_)
    _check_backward((only_out[0], only_out[2], only_out[3]), go, None, total, w, 1e-5, t, p)
    with torch.no_grad():
        assert not functional.layer_norm(leaves[0], leaves[2], leaves[3]).requires_grad


def test_gradient_is_the_difference_quotient():
    """float32, central differences of step 2^-6: the truncation is 2^-12 / 6 of a third derivative of order r^3, the rounding
    of the loss 2^-24 sqrt(96) of sums near 10 over the step."""
    ops = _ops()
    x, _, w, b, go, _ = _inputs(2, 48, torch.float32, torch.float32, seed=9, residual=False)
    dx, dw, db, dgo = _dev(x, w, b, go)
    _, _, mean, rstd = ops.layer_norm(dx, dw, db, 1e-5, want_stats=True)
    grad = ops.layer_norm_backward(dgo, dx, dw, mean, rstd)[0]
    step = 2.0 ** -6
    worst = 0.0
    for j in range(48):
        up, down = dx.clone(), dx.clone()
        up[:, j] += step
        down[:, j] -= step
        a, c = (ops.layer_norm(v, dw, db, 1e-5)[0].double() for v in (up, down))
        quotient = ((a - c) * dgo.double()).sum(1) / (2 * step)
        worst = max(worst, (quotient - grad[:, j].double()).abs().max().item())
    assert worst < 2e-3


def test_models_run_on_it():
    """GPT-2 and ViT with every norm on the HIP kernels: logits within the storage type's noise of the PyTorch norms', the
    default mode's untouched, and a training step whose gradients agree."""
    from d2dmoe_amd import gpt2, set_norm_mode, vit
    torch.manual_seed(0)
    gpt = gpt2.GPT(gpt2.GPTConfig(block_size=64, vocab_size=256, n_layer=2, n_head=4, n_embd=128)).to(DEV).eval()
    img = vit.VisionTransformer(image_size=32, num_layers=2, num_heads=4, hidden_dim=128, mlp_dim=256, num_classes=8).to(DEV).eval()
    idx = torch.randint(0, 256, (2, 64), device=DEV)
    pic = torch.randn(2, 3, 32, 32, device=DEV)
    for model, data in ((gpt, idx), (img, pic)):
        results = {}
        for mode in ('torch', 'hip', 'torch'):
            set_norm_mode(model, mode)
            model.zero_grad()
            out = model(data)
            out.float().square().mean().backward()
            got = (out.detach().clone(), {k: v.grad.clone() for k, v in model.named_parameters() if v.grad is not None})
            if mode in results:
                assert torch.equal(results[mode][0], got[0])
            results[mode] = got
        a, c = results['torch'], results['hip']
        # float32 throughout: a few hundred roundings of 2^-24 along the model
        assert (a[0] - c[0]).abs().max() <= 1e-4 * a[0].abs().max()
        assert set(a[1]) == set(c[1])
        for k in a[1]:
            assert (a[1][k] - c[1][k]).norm() <= 1e-3 * a[1][k].norm() + 1e-9, k


class _Mix(torch.nn.Module):
    """In the place of an attention: a projection, which autocast runs in 16 bits."""

    def __init__(self, d, pair):
        super().__init__()
        self.project, self.pair = torch.nn.Linear(d, d), pair

    def forward(self, x, *_, **__):
        out = self.project(x)
        return (out, None) if self.pair else out


@pytest.mark.parametrize('t', [torch.bfloat16, torch.float16])
def test_models_under_autocast(t):
    """A training step under autocast: the blocks see a 16-bit branch and a float32 residual stream.  Every norm's input, and with
    it the stream, has the element type that the PyTorch mode gives it.  The norms' float32 rows differ in their last bits, so a
    few of the 16-bit roundings behind them flip; were it all of them, a step (twice `half`) each in four norms and as many
    products, outputs and gradients would be off by 16 `half` of their size.

    A gradient's size is that of the terms it adds up.  The encoder ends in a norm, whose squares add up to D v / (v + eps) in
    every row: the terms 2 n r of the loss's gradient cancel down to eps of them, the roundings do not.  So the size is
    taken from the backward pass of a gradient at the output with the same entries under random signs, which keeps every
    term's size and cancels nothing."""
    from d2dmoe_amd import gpt2, set_norm_mode, vit
    torch.manual_seed(0)
    gpt = gpt2.GPT(gpt2.GPTConfig(block_size=32, vocab_size=64, n_layer=2, n_head=4, n_embd=128)).to(DEV).eval()
    img = vit.VisionTransformer(image_size=32, num_layers=2, num_heads=4, hidden_dim=128, mlp_dim=256, num_classes=8).to(DEV).eval()
    for block in gpt.transformer.h:
        block.attn = _Mix(128, False).to(DEV)
    for block in img.encoder.layers:
        block.self_attention = _Mix(128, True).to(DEV)
    idx = torch.randint(0, 64, (2, 32), device=DEV)
    tokens = torch.randn(2, 5, 128, device=DEV)
    for model, data in ((gpt, idx), (img.encoder, tokens)):
        blocks = list(gpt.transformer.h if model is gpt else img.encoder.layers)
        results = {}
        for mode in ('torch', 'hip'):
            set_norm_mode(model, mode)
            model.zero_grad()
            types = []
            hooks = [b.register_forward_hook(lambda _, i, o: types.append((i[0].dtype, o.dtype))) for b in blocks]
            with torch.autocast('cuda', t):
                out = model(data)
                loss = out.float().square().sum()
            loss.backward(retain_graph=True)
            for h in hooks:
                h.remove()
            grads = {k: v.grad.clone() for k, v in model.named_parameters() if v.grad is not None}
            model.zero_grad()
            signs = torch.randint(0, 2, out.shape, generator=torch.Generator().manual_seed(1)).to(DEV) * 2 - 1
            out.backward((2 * out.detach().float() * signs).to(out.dtype))
            sizes = {k: v.grad.norm() for k, v in model.named_parameters() if v.grad is not None}
            results[mode] = (out.detach().float(), grads, types, sizes)
        a, c = results['torch'], results['hip']
        assert a[2] == c[2] and a[2][0][1] == torch.float32
        bound = 16 * _half(t)
        assert (a[0] - c[0]).abs().max() <= bound * a[0].abs().max()
        assert set(a[1]) == set(c[1])
        for k in a[1]:
            assert a[1][k].dtype == c[1][k].dtype and torch.isfinite(c[1][k]).all()
            assert (a[1][k] - c[1][k]).norm() <= bound * torch.maximum(a[1][k].norm(), a[3][k]), k


def test_gradients_add_up_over_backward_passes():
    """Leaves with leading dimensions, three passes: the same gradients three times (float32; two additions of a half step each)."""
    from d2dmoe_amd import functional
    x, r, w, b, go, gs = _inputs(12, 64, torch.float32, torch.float32, seed=11)
    leaves = [v.view(3, 4, 64).to(DEV).requires_grad_() for v in (x, r)] + [v.to(DEV).requires_grad_() for v in (w, b)]
    go, gs = go.view(3, 4, 64).to(DEV), gs.view(3, 4, 64).to(DEV)
    once = torch.autograd.grad(functional.layer_norm(leaves[0], leaves[2], leaves[3], 1e-5, leaves[1]), leaves, (go, gs))
    for _ in range(3):
        torch.autograd.backward(functional.layer_norm(leaves[0], leaves[2], leaves[3], 1e-5, leaves[1]), (go, gs))
    assert len({v.grad.data_ptr() for v in leaves}) == 4
    for v, g in zip(leaves, once):
        assert ((v.grad - 3 * g).abs() <= 8 * U * g.abs()).all()
