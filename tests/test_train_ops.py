"""linear_cross_entropy, orthogonalize, muon_step_ / FlowMuon against plain implementations in 64 bits.

Every numerical test runs on the GPU (`-m gpu`) and, at its smaller sizes, over the host-executed kernel sources (tests/train_on_host.py).

Tolerances.  u(t) = finfo(t).eps / 2 is a rounding to type t.
  z        a logit is a sum of D products in fp32, of numbers of 22 bits (fp32 inputs) or exact (16-bit inputs):
           dz <= scale (D 2^-24 + 2^-20) max sum_d |h||w|
  loss     two exponents / logarithms of arguments up to Z = max |z| and sums of up to 128 terms in a row: 2 dz + (2 Z + 128) 2^-23
  dh, dw   an element is a sum over K of G times a number.  G = p - [v = t] is off by dp = p (2 dz + (2 Z + 128) 2^-23) + 2^-23, then rounded to
           u(fp16) of itself (2^-21 for two planes) or to 2^-39; the sum adds K 2^-24, the result is rounded to its type.
  orthogonalize   three matrices a step are rounded to 22 bits where fp32 rounds to 24: four times the error of the same iteration in fp32, plus
           the 16 roundings 2^-22 themselves, plus the output's own rounding; in the Frobenius norm."""
import contextlib
import copy
import math
import os
import sys

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, os.path.join(ROOT, 'tests'))

from unopticalflow_amd import ops, optim  # noqa: E402

DTYPES = [torch.float32, torch.bfloat16, torch.float16]
COEFFICIENTS = (3.4445, -4.7750, 2.0315)


@pytest.fixture(params=['host', pytest.param('cuda', marks=pytest.mark.gpu)])
def device(request):
    if request.param == 'cuda':
        yield 'cuda'
        return
    import train_on_host
    with train_on_host.patched():
        yield 'cpu'


def _u(dtype):
    return torch.finfo(dtype).eps / 2


# ------------------------------------------------------------------------------------------ linear_cross_entropy
def _inputs(rows, vocab, dim, dtype, device, seed=0, ignored=0.2, spread=1.0):
    g = torch.Generator().manual_seed(seed)
    h = spread * torch.randn(rows, dim, generator=g)
    w = torch.randn(vocab, dim, generator=g) / math.sqrt(dim)
    t = torch.randint(vocab, (rows,), generator=g)
    t[torch.rand(rows, generator=g) < ignored] = -100
    return h.to(dtype).to(device), w.to(dtype).to(device), t.to(device)


def _check_lce(h, w, t, dtype, reduction='mean', scale=1.0, ignore=-100, upstream=None, want=(True, True), **more):
    """Runs forward and backward and compares loss, dh, dw with 64 bits under the bounds of the module's docstring."""
    device = h.device
    h, w = h.detach().requires_grad_(want[0]), w.detach().requires_grad_(want[1])
    n, d = t.numel(), h.shape[-1]
    if upstream is None:
        gen = torch.Generator().manual_seed(5)
        upstream = (torch.rand(t.shape, generator=gen) if reduction == 'none' else torch.tensor(1.7)).to(device)
    loss = ops.linear_cross_entropy(h, w, t, ignore_index=ignore, scale=scale, reduction=reduction, **more)
    assert loss.dtype == torch.float32 and loss.shape == (t.shape if reduction == 'none' else ())
    grads = torch.autograd.grad(loss, [x for x, need in ((h, want[0]), (w, want[1])) if need], upstream) if any(want) else ()
    hd, wd, td, up = h.detach().double().reshape(-1, d), w.detach().double(), t.reshape(-1), upstream.double().reshape(-1)
    used = td != ignore
    hd = hd.where(used[:, None], 0)
    count = max(1, int(used.sum()))
    z = scale * (hd @ wd.T)
    lse = z.logsumexp(1)
    at = td.where(used, 0)
    losses = (lse - z.gather(1, at[:, None])[:, 0]).where(used, 0)
    exact = {'none': losses.view(t.shape), 'sum': losses.sum(), 'mean': losses.sum() / count}[reduction]
    dz = abs(scale) * (d * 2**-24 + 2**-20) * float((hd.abs() @ wd.abs().T).max())
    top = float(z.abs().max())
    loose = 2 * dz + (2 * top + 128) * 2**-23
    bound = loose * (n if reduction == 'sum' else 1) + n * 2**-24 * exact.abs()
    assert bool(((loss.detach().double() - exact).abs() <= bound).all()), (loss, exact)
    p = z.softmax(1)
    onehot = torch.zeros_like(p).scatter_(1, at[:, None], 1.0)
    weight = (up if reduction == 'none' else up / count if reduction == 'mean' else up).expand(n) * used * scale
    g = (p - onehot) * weight[:, None]
    rounding = 2**-21 if dtype == torch.float32 else _u(torch.float16)
    off = ((p * loose + 2**-23) + (p - onehot).abs() * rounding + 2**-39) * weight.abs()[:, None]
    if reduction == 'none':                              # (rows are packed relative to the largest upstream gradient)
        off = off + 2**-38 * float(weight.abs().max())
    got = iter(grads)
    out = []
    for need, exact, magnitude, error, k, largest in ((want[0], g @ wd, g.abs() @ wd.abs(), off @ wd.abs(), len(wd), float(wd.abs().max()) * g.abs().sum(1, keepdim=True)),
                                                      (want[1], g.T @ hd, g.abs().T @ hd.abs(), off.T @ hd.abs(), n, float(hd.abs().max()) * g.abs().sum(0)[:, None])):
        if not need:
            continue
        x = next(got)
        assert x.dtype == dtype and x.shape == (h.shape if exact.shape[0] == n and x.shape == h.shape else exact.shape)
        x = x.double().reshape(exact.shape)
        bound = error + magnitude * (k * 2**-24 + 2**-20) + largest * 2**-39 + _u(dtype) * exact.abs() + torch.finfo(dtype).smallest_normal * _u(dtype) * 2
        assert bool(((x - exact).abs() <= bound).all()), float(((x - exact).abs() / bound).max())
        out.append(x)
    return loss.detach(), out


@pytest.mark.parametrize('dtype', DTYPES, ids=str)
@pytest.mark.parametrize('rows,vocab,dim,reduction,scale', [
    (1, 1, 1, 'mean', 1.0), (1, 3, 1, 'sum', 1.0), (2, 5, 8, 'none', -2.0), (5, 70, 40, 'mean', 1.0), (64, 64, 64, 'sum', 1.0),
    (65, 257, 33, 'none', 0.5), (67, 130, 96, 'mean', 1 / 0.07), (3, 200, 520, 'none', 1.0), (20, 77, 16, 'mean', 3.0), (33, 64, 4, 'sum', 1.0), (17, 300, 200, 'sum', 1.0), (130, 31, 72, 'mean', 1.0)])
def test_loss_and_gradients(device, dtype, rows, vocab, dim, reduction, scale):
    h, w, t = _inputs(rows, vocab, dim, dtype, device, ignored=0.2 if rows > 4 else 0.0)
    _check_lce(h, w, t, dtype, reduction, scale)


@pytest.mark.parametrize('dtype', DTYPES, ids=str)
@pytest.mark.parametrize('rows,dim', [(1, 3), (1, 4), (2, 7), (3, 8), (16, 9), (5, 31), (17, 65), (1, 250), (32, 257), (33, 515), (64, 130), (65, 37), (7, 1023)])
def test_rows_that_start_and_end_anywhere(device, dtype, rows, dim):
    """Rows cut out of wider ones, off 16 bytes and with NaN on both sides of them."""
    h, w, t = _inputs(rows, 100, dim, dtype, device, ignored=0.2 if rows > 4 else 0.0)
    for before, behind in ((1, 0), (0, 1), (3, 5)):
        cut = []
        for x in (h, w):
            wide = torch.full((len(x), before + dim + behind), float('nan'), dtype=dtype, device=device)
            wide[:, before:before + dim] = x
            cut.append(wide[:, before:before + dim])
        _check_lce(*cut, t, dtype, 'none')
        with torch.no_grad():
            assert torch.equal(ops.linear_cross_entropy(*cut, t, reduction='none').isnan(), torch.zeros(rows, dtype=torch.bool, device=device))


@pytest.mark.parametrize('rows,vocab,dim,scale', [(60, 90, 16, 14.0), (33, 200, 100, 1.0), (3, 40, 8, 2.0), (20, 50, 33, -3.0)])
@pytest.mark.parametrize('spread', [1.0, 2.0**-60, 2.0**60])
def test_gradients_of_bf16_inputs_are_rounded_to_bf16_once(device, rows, vocab, dim, scale, spread):
    """What is summed holds 11 bits (two factors: 2^-11 of a term each at most, and 2^-39 of the largest), whatever the inputs' magnitudes: the
    output's own eps / 2 = 2^-8 is the only rounding to bf16."""
    h, w, t = _inputs(rows, vocab, dim, torch.bfloat16, device, ignored=0.2 if rows > 4 else 0.0)
    h, w = h * spread, w / spread
    h[t < 0] = 3e38                                       # (an ignored row has no part in any scale)
    h.requires_grad_()
    w.requires_grad_()
    dh, dw = torch.autograd.grad(ops.linear_cross_entropy(h, w, t, scale=scale, reduction='sum'), (h, w))
    hd, wd, used = h.detach().double().where((t >= 0)[:, None], 0), w.detach().double(), t >= 0
    z = scale * (hd @ wd.T)
    dz = abs(scale) * (dim * 2**-24 + 2**-20) * float((hd.abs() @ wd.abs().T).max())
    loose = 2 * dz + (2 * float(z.abs().max()) + 128) * 2**-23
    p = z.softmax(1)
    g = (p - torch.zeros_like(p).scatter_(1, t.where(used, 0)[:, None], 1.0)) * used[:, None] * scale
    off = ((p * loose + 2**-23) * abs(scale) + g.abs() * _u(torch.float16) + 2**-39 * abs(scale)) * used[:, None]
    for got, a, b, error in ((dh, g, wd, off), (dw, g.T, hd, off.T)):
        exact, size = a @ b, a.abs() @ b.abs()
        bound = error @ b.abs() + size * (a.shape[1] * 2**-24 + _u(torch.float16)) + a.abs().sum(1, keepdim=True) * float(b.abs().max()) * 2**-38 + _u(torch.bfloat16) * exact.abs()
        assert bool(((got.double() - exact).abs() <= bound).all()), float(((got.double() - exact).abs() / (bound + 2.0**-200)).max())


@pytest.mark.parametrize('rows,vocab,reduction', [(1024, 40, 'mean'), (1025, 40, 'mean'), (5, 2200, 'sum'), (300, 2200, 'mean'), (40, 2048, 'sum')])
def test_rows_and_tiles_joined_in_one_launch_or_two(device, rows, vocab, reduction):
    """Up to 1024 rows of up to 32 tiles, and more of either."""
    h, w, t = _inputs(rows, vocab, 8, torch.bfloat16, device)
    _check_lce(h, w, t, torch.bfloat16, reduction)


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', DTYPES, ids=str)
@pytest.mark.parametrize('rows,vocab,dim', [(1, 32000, 2048), (7, 50257, 129), (513, 3001, 777), (832, 832, 96), (2100, 2200, 200), (3700, 4000, 264),
                                            (300, 70001, 64), (20000, 9000, 40)])
def test_loss_and_gradients_at_size(dtype, rows, vocab, dim):
    """Every tile size, sums cut into shares, and classes in several pieces (70001 classes; 20000 rows)."""
    h, w, t = _inputs(rows, vocab, dim, dtype, 'cuda', ignored=0.1 if rows > 4 else 0.0)
    _check_lce(h, w, t, dtype, 'none' if rows < 1000 else 'mean')


@pytest.mark.parametrize('dtype', DTYPES, ids=str)
def test_layouts(device, dtype):
    """Rows further apart than they are long, columns that are not adjacent, a start off 16 bytes, three dimensions, one row repeated."""
    base, w, t = _inputs(24, 50, 64, dtype, device)
    plain = [x.clone() for x in (base[:, :40], w[:, :40])]
    want = _check_lce(*plain, t, dtype)
    for h2, w2 in ((base[:, :40], w[:, :40]), (plain[0].T.contiguous().T, plain[1].T.contiguous().T)):
        loss, grads = _check_lce(h2, w2, t, dtype)
        assert torch.equal(loss, want[0]) and all(torch.equal(a, b) for a, b in zip(grads, want[1]))
    odd = torch.zeros(24 * 40 + 1, dtype=dtype, device=device)
    odd[1:] = plain[0].reshape(-1)
    _check_lce(odd[1:].view(24, 40), plain[1], t, dtype)
    _check_lce(plain[0].view(2, 12, 40), plain[1], t.view(2, 12), dtype, 'none')
    _check_lce(plain[0][:1].expand(24, 40), plain[1], t, dtype)


@pytest.mark.parametrize('want', [(True, False), (False, True), (False, False)])
def test_one_gradient_only(device, want):
    h, w, t = _inputs(33, 70, 24, torch.bfloat16, device)
    _check_lce(h, w, t, torch.bfloat16, want=want)


@pytest.mark.parametrize('dtype', DTYPES, ids=str)
@pytest.mark.parametrize('reduction', ['mean', 'sum', 'none'])
def test_all_rows_ignored(device, dtype, reduction):
    h, w, t = _inputs(9, 20, 16, dtype, device, ignored=2.0)
    h.fill_(float('nan'))
    loss, (dh, dw) = _check_lce(h, w, t, dtype, reduction)
    assert not loss.any() and not dh.any() and not dw.any()


@pytest.mark.parametrize('dtype', DTYPES, ids=str)
@pytest.mark.parametrize('bad', [float('nan'), float('inf'), -float('inf'), 'largest'])
def test_ignored_rows_may_hold_anything(device, dtype, bad):
    h, w, t = _inputs(40, 33, 24, dtype, device, ignored=0.4)
    h[t == -100] = torch.finfo(dtype).max if bad == 'largest' else bad
    _check_lce(h, w, t, dtype)


@pytest.mark.parametrize('dtype', DTYPES, ids=str)
def test_targets_outside_the_classes(device, dtype):
    h, w, t = _inputs(20, 33, 24, dtype, device, ignored=0.0)
    t[3], t[7], t[11] = 33, -1, 1 << 40
    losses = ops.linear_cross_entropy(h, w, t, reduction='none')
    bad = torch.zeros(20, dtype=torch.bool, device=device)
    bad[[3, 7, 11]] = True
    assert bool(torch.isnan(losses[bad]).all()) and bool(torch.isfinite(losses[~bad]).all())
    h.requires_grad_()
    dh, = torch.autograd.grad(ops.linear_cross_entropy(h, w, t, reduction='sum'), h)
    assert bool(torch.isnan(dh[bad]).all()) and bool(torch.isfinite(dh[~bad]).all())
    _check_lce(h, w, t.where(~bad, 33), dtype, ignore=33)                # any value may be the ignored one
    t = t.where(~bad, 5)
    _check_lce(h, w, t, dtype, ignore=5)


@pytest.mark.parametrize('dtype', DTYPES, ids=str)
def test_extreme_logits(device, dtype):
    """Logits of +-thousands, equal logits, and hidden rows that differ by 2^20 in size."""
    h, w, t = _inputs(20, 130, 24, dtype, device, ignored=0.0, spread=2000.0)
    _check_lce(h, w, t, dtype, 'none')
    h, w, t = _inputs(20, 130, 24, dtype, device, ignored=0.0)
    _check_lce(torch.zeros_like(h), w, t, dtype, 'none')
    h[:10] *= 2.0**-10
    h[15:] *= 2.0**8
    _check_lce(h, w, t, dtype, 'none')


def test_a_row_of_infinities_is_nan_and_stays_alone(device):
    for dtype in DTYPES:
        h, w, t = _inputs(20, 70, 24, dtype, device, ignored=0.0)
        clean = ops.linear_cross_entropy(h, w, t, reduction='none')
        h[4], h[9, 3] = float('inf'), float('nan')
        losses = ops.linear_cross_entropy(h, w, t, reduction='none')
        others = torch.ones(20, dtype=torch.bool, device=device)
        others[[4, 9]] = False
        assert bool(torch.isnan(losses[[4, 9]]).all()) and torch.equal(losses[others], clean[others])


def test_no_rows(device):
    for reduction in ('mean', 'sum', 'none'):
        h, w, t = _inputs(4, 7, 8, torch.float32, device)
        h, w = h[:0].requires_grad_(), w.requires_grad_()
        loss = ops.linear_cross_entropy(h, w, t[:0], reduction=reduction)
        assert loss.shape == ((0,) if reduction == 'none' else ())
        dh, dw = torch.autograd.grad(loss.sum(), (h, w))
        assert dh.shape == (0, 8) and not dw.any() and not loss.any()


def test_gradient_against_differences(device):
    """Central differences of the loss itself (fp32, step 2^-6: the loss is off by 2^-21 of itself, third derivatives are below 1)."""
    h, w, t = _inputs(6, 11, 5, torch.float32, device, ignored=0.2)
    h, w = h.requires_grad_(), w.requires_grad_()
    grads = torch.autograd.grad(ops.linear_cross_entropy(h, w, t, scale=1.5, reduction='sum'), (h, w))
    step, f = 2.0**-6, lambda: float(ops.linear_cross_entropy(h, w, t, scale=1.5, reduction='sum'))
    for x, g in zip((h, w), grads):
        for i in range(0, x.numel(), 7):
            with torch.no_grad():
                flat = x.view(-1)
                old = float(flat[i])
                flat[i] = old + step
                up = f()
                flat[i] = old - step
                down = f()
                flat[i] = old
            assert abs((up - down) / (2 * step) - float(g.reshape(-1)[i])) < 20 * step**2 + 20 * 2**-21 / step


@pytest.mark.parametrize('dtype', DTYPES, ids=str)
def test_results_are_reproducible_bit_for_bit(device, dtype):
    h, w, t = _inputs(150, 333, 72, dtype, device)
    h, w = h.requires_grad_(), w.requires_grad_()

    def once():
        loss = ops.linear_cross_entropy(h, w, t)
        return (loss.detach(), *torch.autograd.grad(loss, (h, w)))
    first = once()
    assert all(torch.equal(a, b) for a, b in zip(first, once()))


@pytest.mark.gpu
def test_offsets_beyond_32_bits():
    """A weight of 2.4 G numbers: the last classes are found, and get their gradient."""
    v, d = 600_000, 4096
    w = torch.zeros(v, d, dtype=torch.bfloat16, device='cuda')
    g = torch.Generator('cuda').manual_seed(0)
    h = torch.randn(3, d, generator=g, device='cuda').bfloat16()
    w[-2:] = torch.randn(2, d, generator=g, device='cuda').bfloat16() / 64
    t = torch.tensor([v - 1, v - 2, 0], device='cuda')
    h.requires_grad_()
    w.requires_grad_()
    loss = ops.linear_cross_entropy(h, w, t, reduction='none')
    dh, dw = torch.autograd.grad(loss.sum(), (h, w))
    z = h.detach().double() @ w.detach()[-2:].double().T
    lse = (z.exp().sum(1) + (v - 2)).log()
    exact = lse - torch.stack([z[0, 1], z[1, 0], torch.zeros_like(z[0, 0])])
    assert torch.allclose(loss.detach().double(), exact, rtol=0, atol=(2 * 4096 * 2**-24 + 2**-19) * 64 + 140 * 2**-23)
    p = (z - lse[:, None]).exp()
    p[0, 1] -= 1
    p[1, 0] -= 1
    tail = p.T @ h.detach().double()
    assert bool(((dw[-2:].double() - tail).abs() <= 2 * 2**-8 * (p.abs().T @ h.detach().double().abs())).all())
    assert bool(((dh.double() - p @ w.detach()[-2:].double()).abs() <= 2 * 2**-8 * (p.abs() @ w.detach()[-2:].double().abs()) + 2**-30).all())


def test_no_second_derivative(device):
    """The gradients are values: asking for theirs is an error, not a zero."""
    h, w, t = _inputs(4, 7, 8, torch.float32, device)
    h.requires_grad_()
    loss = ops.linear_cross_entropy(h, w, t)
    g, = torch.autograd.grad(loss, h, create_graph=True)
    with pytest.raises(RuntimeError):
        g.square().sum().backward()


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', DTYPES, ids=str)
def test_captured_and_replayed(dtype):
    """Two graphs of the same leaves, replayed in turn with eager calls between them; every replay equals the eager result."""
    h, w, t = _inputs(300, 700, 72, dtype, 'cuda')
    h2, w2, t2 = _inputs(90, 700, 72, dtype, 'cuda', seed=1)

    def make(h, w, t, reduction):
        h, w = h.detach().clone().requires_grad_(), w.detach().clone().requires_grad_()
        up = torch.rand(t.shape, device='cuda') if reduction == 'none' else torch.ones((), device='cuda')

        def once():
            loss = ops.linear_cross_entropy(h, w, t, reduction=reduction)
            return (loss.detach(), *torch.autograd.grad(loss, (h, w), up))
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            once()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = once()
        return h, w, once, graph, out
    pair = [make(h, w, t, 'mean'), make(h2, w2, t2, 'none')]
    for k in range(3):
        for x, y, once, graph, out in pair:
            with torch.no_grad():
                x.mul_(0.9)
                y.mul_(1.05)
            graph.replay()
            kept = [o.clone() for o in out]
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(kept, once())), k


@pytest.mark.gpu
def test_on_another_stream():
    h, w, t = _inputs(500, 3000, 136, torch.bfloat16, 'cuda')
    want = _check_lce(h, w, t, torch.bfloat16)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = _check_lce(h, w, t, torch.bfloat16)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got[0], want[0]) and all(torch.equal(a, b) for a, b in zip(got[1], want[1]))


def test_refusals_of_the_loss():
    h, w, t = _inputs(4, 7, 8, torch.float32, 'cpu')
    with pytest.raises(RuntimeError, match='MI355X'):
        ops.linear_cross_entropy(h, w, t)
    import train_on_host
    with train_on_host.patched():
        for bad in (dict(reduction='avg'),):
            with pytest.raises(ValueError):
                ops.linear_cross_entropy(h, w, t, **bad)
        for args in ((h, w[:, :7], t), (h, w[0], t), (h, w, t[:3]), (h, w, t.int()), (h, w[:0], t), (h[:, :0], w[:, :0], t), (h[0, 0], w, t)):
            with pytest.raises(ValueError):
                ops.linear_cross_entropy(*args)
        with pytest.raises(TypeError):
            ops.linear_cross_entropy(h.double(), w.double(), t)
        with pytest.raises(TypeError):
            ops.linear_cross_entropy(h.bfloat16(), w, t)


def test_entry_points_check_their_arguments():
    """The C entries refuse what they do not take before anything is launched."""
    import ctypes
    import __graft_entry__ as ge
    ge.build()
    from unopticalflow_amd import _lib
    lib = _lib.load()
    ok, k, a, b = 4096, ctypes.c_longlong(), ctypes.c_longlong(), ctypes.c_longlong()
    size = lambda *v: lib.unflow_linear_ce_workspace(ok, v[2], ok, v[2], *v, 1, 1, ctypes.byref(k), ctypes.byref(a), ctypes.byref(b))  # noqa: E731
    assert size(5, 7, 8, 0) == 0 and a.value > 0 and b.value > 0 and k.value > 0
    for bad in ((0, 7, 8, 0), (5, 0, 8, 0), (5, 7, 0, 0), (5, 7, 8, 3), (5, 7, 8, -1), ((1 << 20) + 1, 7, 8, 0), (5, (1 << 30) + 1, 8, 0), (5, 7, (1 << 20) + 1, 0)):
        assert size(*bad) == -22, bad
    fwd = lambda ws, n, red=0, loss=ok, kept=ok: lib.unflow_linear_ce_fwd(ok, 8, ok, 8, ok, 5, 7, 8, 0, 1.0, -100, red, loss, kept, ws, n, None)  # noqa: E731
    assert fwd(ok, 16) == -22 and fwd(None, 1 << 30) == -22 and fwd(ok, 1 << 30, 3) == -22 and fwd(ok, 1 << 30, 0, None) == -22 and fwd(ok, 1 << 30, 0, ok, None) == -22
    assert lib.unflow_linear_ce_bwd(ok, 8, ok, 8, ok, ok, 5, 7, 8, 0, 1.0, -100, 0, None, None, ok, ok, 1 << 30, None) == -22
    assert lib.unflow_linear_ce_fwd(ok, 7, ok, 8, ok, 5, 7, 8, 0, 1.0, -100, 0, ok, ok, ok, 1 << 30, None) == -22
    m = lambda *v: (ops._Matrix * 1)(v)  # noqa: E731
    need = ctypes.c_longlong()
    assert lib.unflow_orthogonalize_workspace(m(ok, ok, None, 5, 7), 1, 0, ctypes.byref(need)) == 0 and need.value > 0
    for bad in ((ok, ok, None, 0, 7), (ok, ok, None, 5, -1), (ok, ok, None, 5, (1 << 18) + 1)):
        assert lib.unflow_orthogonalize_workspace(m(*bad), 1, 0, ctypes.byref(need)) == -22
    orth = lambda mat, steps=5, c=COEFFICIENTS, n=1 << 30, count=1, dtype=0: lib.unflow_orthogonalize(mat, count, dtype, steps, *c, 1e-7, ok, n, None)  # noqa: E731
    good = m(ok, ok, None, 5, 7)
    assert orth(good, steps=0) == -22 and orth(good, steps=65) == -22 and orth(good, n=64) == -22 and orth(good, count=0) == -22 and orth(good, dtype=3) == -22
    assert orth(good, c=(9.0, 9.0, 9.0)) == -22 and orth(m(None, ok, None, 5, 7)) == -22 and orth(m(ok, None, None, 5, 7)) == -22
    assert lib.unflow_muon_step(good, 1, 0, 0.1, 0.9, 0.0, 1, 5, *COEFFICIENTS, 1e-7, ok, 1 << 30, None) == -22          # no momentum


# ------------------------------------------------------------------------------------------ orthogonalize
def _iterate(x, steps=5, coefficients=COEFFICIENTS, eps=1e-7):
    """The iteration in x's own type."""
    a, b, c = coefficients
    turned = x.shape[-2] > x.shape[-1]
    x = x.mT if turned else x
    x = x / (x.norm(dim=(-2, -1), keepdim=True) + eps)
    for _ in range(steps):
        s = x @ x.mT.contiguous()
        x = a * x + (b * s + c * (s @ s)) @ x
    return x.mT if turned else x


def _check_orthogonal(got, x, **how):
    assert got.dtype == x.dtype and got.shape == x.shape
    exact = _iterate(x.double(), **how)
    plain = _iterate(x.float(), **how).double()
    norm = float(exact.norm())
    tolerance = (4 * float((plain - exact).norm()) + 16 * 2**-22 * norm) + (_u(x.dtype) * norm if x.dtype != torch.float32 else 0)
    assert float((got.double() - exact).norm()) <= tolerance, (float((got.double() - exact).norm()) / norm, tolerance / norm)


def _matrix(*shape, dtype, device, seed=0, rank=None):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(shape, generator=g)
    if rank is not None:
        x = torch.randn(*shape[:-1], rank, generator=g) @ torch.randn(*shape[:-2], rank, shape[-1], generator=g)
    return (1e-3 * x).to(dtype).to(device)


@pytest.mark.parametrize('dtype', DTYPES, ids=str)
@pytest.mark.parametrize('shape', [(1, 1), (1, 9), (9, 1), (5, 7), (2, 864), (40, 40), (33, 90), (90, 33), (3, 2, 70, 65), (64, 64), (130, 300), (64, 2100)])
def test_orthogonalize(device, dtype, shape):
    x = _matrix(*shape, dtype=dtype, device=device)
    _check_orthogonal(ops.orthogonalize(x), x)


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', DTYPES, ids=str)
@pytest.mark.parametrize('shape', [(2, 4096, 1024), (1027, 1999), (4096, 4096), (8, 128, 1152), (300, 20000), (2, 2600, 2500)])
def test_orthogonalize_at_size(dtype, shape):
    x = _matrix(*shape, dtype=dtype, device='cuda')
    _check_orthogonal(ops.orthogonalize(x), x)


@pytest.mark.parametrize('shape,rank', [((1, 1), None), ((1, 300), None), ((300, 1), None), ((2, 8), None), ((4, 512), None), ((15, 175), None), ((175, 15), None),
                                        ((31, 129), None), ((32, 32), None), ((3, 32, 127), None), ((257, 32), None), ((20, 60), 3), ((13, 8400), None), ((8400, 7), 2)])
def test_few_rows(device, shape, rank):
    """Up to 32 rows or columns: all sums in 64 bits (n 2^-53, times a^10 = 2^18, and the steps' rounding), one rounding of the result to 2^-24."""
    x = _matrix(*shape, dtype=torch.float32, device=device, rank=rank)
    got = ops.orthogonalize(x)
    g = x.double().mT if shape[-2] > shape[-1] else x.double()
    m, n = g.shape[-2:]
    g = g / (g.norm(dim=(-2, -1), keepdim=True) + 1e-7)
    a, b, c = COEFFICIENTS
    s, p = g @ g.mT.contiguous(), torch.eye(m, dtype=torch.float64, device=x.device)
    for _ in range(5):
        q = a * torch.eye(m, dtype=torch.float64, device=x.device) + b * s + c * (s @ s)
        p, s = q @ p, q @ s @ q
    exact = p @ g
    bound = exact.abs() * 2**-24 + (n + 1000) * 2**-53 * 2**18 * float(g.abs().max()) * m + 2**-149
    got = got.double().mT if shape[-2] > shape[-1] else got.double()
    assert bool(((got - exact).abs() <= bound).all()), float(((got - exact).abs() / bound).max())


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', DTYPES, ids=str)
def test_captured_orthogonalize(dtype):
    """A graph of the tiles, one of the kernels for few rows and one of a Muon step, replayed in turn with eager calls between them."""
    wide, few = ([_matrix(*s, dtype=dtype, device='cuda', seed=i) for i, s in enumerate(shapes)] for shapes in (((40, 300), (130, 70), (20, 9)), ((31, 700), (5, 5))))
    weights, grads = ([_matrix(*s, dtype=dtype, device='cuda', seed=9 + i) for s in ((60, 90), (33, 8))] for i in range(2))
    momenta = [torch.zeros_like(w, dtype=torch.float32) for w in weights]

    def step():
        optim.muon_step_(weights, grads, momenta, lr=0.1)
        return weights + momenta
    graphs = []
    for call in (lambda: ops.orthogonalize(wide), lambda: ops.orthogonalize(few), step):
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            call()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            graphs.append((graph, call, call()))
    for k in range(3):
        for x in wide + few + grads:
            x.mul_(0.5).add_(1e-4)
        for graph, call, out in graphs:
            before = [t.clone() for t in weights + momenta]
            graph.replay()
            kept = [t.clone() for t in out]
            torch.cuda.synchronize()
            for t, old in zip(weights + momenta, before):
                t.copy_(old)
            assert all(torch.equal(a, b) for a, b in zip(kept, call())), k


@pytest.mark.parametrize('dtype', DTYPES, ids=str)
def test_orthogonalize_low_rank(device, dtype):
    """Rank 3 of 60: the directions that only rounding fills are multiplied by 485 and must be the input's, not the kernel's."""
    x = _matrix(60, 80, dtype=dtype, device=device, rank=3)
    _check_orthogonal(ops.orthogonalize(x), x)


def test_orthogonalize_steps_coefficients_and_scale(device):
    x = _matrix(20, 30, dtype=torch.float32, device=device)
    for how in (dict(steps=1), dict(steps=2), dict(steps=12, coefficients=(1.5, -0.5, 0.0)), dict(steps=6, coefficients=(2.0, -1.5, 0.5)), dict(eps=0.5)):
        _check_orthogonal(ops.orthogonalize(x, **how), x, **how)
    tiny, huge = x * 1e-12, x * 1e12                       # the norm's squares leave fp32 (eps is 0 where it would swamp the matrix)
    _check_orthogonal(ops.orthogonalize(tiny, eps=0.0), tiny, eps=0.0)
    _check_orthogonal(ops.orthogonalize(huge), huge)
    # x 1e30: the plain form in fp32 overflows; a power of two changes no bit of the normalised matrix but eps' share of its norm
    assert torch.allclose(ops.orthogonalize(x * 2.0**100, eps=0.0), ops.orthogonalize(x, eps=0.0), rtol=0, atol=2**-20)


def test_orthogonalize_lists_zeros_and_nan(device):
    """Matrices of a list do not touch each other: a zero matrix stays zero, one with a NaN is NaN throughout, the others are as alone."""
    xs = [_matrix(*s, dtype=torch.float32, device=device, seed=i) for i, s in enumerate([(5, 7), (70, 20), (2, 33, 40), (1, 3), (20, 20), (0, 5), (64, 65)])]
    alone = [ops.orthogonalize(x) for x in xs]
    xs[4].zero_()
    xs[0][2, 3] = float('nan')
    together = ops.orthogonalize(xs)
    assert isinstance(together, list) and len(together) == len(xs)
    assert bool(torch.isnan(together[0]).all()) and not together[4].any() and together[5].shape == (0, 5)
    for i in (1, 2, 3, 6):
        assert float((together[i] - alone[i]).norm()) <= 2 * 16 * 2**-22 * float(alone[i].norm()) + 1e-5 * float(alone[i].norm())
    assert ops.orthogonalize([]) == []
    many = [_matrix(2, 3, dtype=torch.bfloat16, device=device, seed=i) for i in range(1100)]      # more than one table holds
    for x, y in list(zip(many, ops.orthogonalize(many)))[::97]:
        _check_orthogonal(y, x)


def test_orthogonalize_strides(device):
    x = _matrix(40, 64, dtype=torch.bfloat16, device=device)
    want = ops.orthogonalize(x[:, :30].contiguous())
    assert torch.equal(ops.orthogonalize(x[:, :30]), want)
    assert torch.equal(ops.orthogonalize(x[:, :30].T.contiguous().T), want)
    before = x.clone()
    ops.orthogonalize(x)
    assert torch.equal(x, before)


def test_refusals_of_orthogonalize():
    x = torch.zeros(4, 5)
    with pytest.raises(RuntimeError, match='MI355X'):
        ops.orthogonalize(x)
    import train_on_host
    with train_on_host.patched():
        for bad in (dict(steps=0), dict(steps=65), dict(eps=-1.0), dict(coefficients=(1.0, 2.0)), dict(coefficients=(5.0, 5.0, 5.0)), dict(eps=float('nan'))):
            with pytest.raises(ValueError):
                ops.orthogonalize(x, **bad)
        for bad in (x[0], [x, x[0]], [x, 3.0], torch.zeros(1, (1 << 18) + 1)):
            with pytest.raises(ValueError):
                ops.orthogonalize(bad)
        for bad in (x.double(), [x, x.bfloat16()], x.int()):
            with pytest.raises(TypeError):
                ops.orthogonalize(bad)


# ------------------------------------------------------------------------------------------ muon_step_, FlowMuon
SHAPES = [(16, 3, 3, 3), (33, 20), (20, 33), (2, 32, 3, 3), (1, 7), (70, 64), (64, 4, 3, 3)]


def _weights(dtype, device, seed=0, shapes=SHAPES):
    g = torch.Generator().manual_seed(seed)
    made = []
    for s in shapes:
        p, d, m = (torch.randn(s, generator=g) * k for k in (1.0, 1e-3, 1e-3))
        if len(s) == 4:
            p, d, m = (t.contiguous(memory_format=torch.channels_last) for t in (p, d, m))
        made.append((p.to(dtype).to(device), d.to(dtype).to(device), m.to(device)))
    return [list(v) for v in zip(*made)]


def _muon(p, g, m, lr, mu, decay, nesterov, dtype=torch.float64):
    p, g, m = p.to(dtype), g.to(dtype), m.to(dtype)
    m = m + (1 - mu) * (g - m)
    u = g + mu * (m - g) if nesterov else m
    o = _iterate(u.reshape(len(u), -1)).reshape(p.shape)
    return p * (1 - lr * decay) - lr * max(1.0, len(p) / (p.numel() / len(p))) ** 0.5 * o, m


@pytest.mark.parametrize('dtype', DTYPES, ids=str)
@pytest.mark.parametrize('nesterov,decay', [(True, 0.0), (False, 0.1)])
def test_muon_step(device, dtype, nesterov, decay):
    params, grads, momenta = _weights(dtype, device)
    want = [_muon(*v, 0.05, 0.9, decay, nesterov) for v in zip(params, grads, momenta)]
    plain = [_muon(*v, 0.05, 0.9, decay, nesterov, torch.float32) for v in zip(params, grads, momenta)]
    strides = [p.stride() for p in params]
    before = [g.clone() for g in grads]
    assert optim.muon_step_(params, grads, momenta, lr=0.05, momentum=0.9, weight_decay=decay, nesterov=nesterov) is None
    for p, m, (ep, em), (fp, _), s in zip(params, momenta, want, plain, strides):
        assert p.dtype == dtype and p.stride() == s and m.dtype == torch.float32
        assert bool(((m.double() - em).abs() <= 4 * 2**-24 * (em.abs() + 1e-3 * 8)).all())
        step = 0.05 * max(1.0, len(p) / (p.numel() / len(p))) ** 0.5 * math.sqrt(p.numel()) * 1.3
        tolerance = 4 * float((fp.double() - ep).norm()) + 16 * 2**-22 * step + _u(dtype) * float(ep.norm()) + 4 * 2**-24 * float(ep.norm())
        assert float((p.double() - ep).norm()) <= tolerance
    assert all(torch.equal(a, b) for a, b in zip(grads, before))


def test_muon_step_takes_gradients_in_another_layout(device):
    params, grads, momenta = _weights(torch.float32, device)
    again = [[t.clone(memory_format=torch.preserve_format) for t in v] for v in (params, grads, momenta)]
    optim.muon_step_(params, grads, momenta, lr=0.1)
    again[1] = [g.contiguous() if g.dim() == 4 else g.T.contiguous().T for g in again[1]]
    optim.muon_step_(*again, lr=0.1)
    assert all(torch.equal(a, b) for a, b in zip(params + momenta, again[0] + again[2]))


def test_refusals_of_muon_step():
    import train_on_host
    params, grads, momenta = _weights(torch.float32, 'cpu')
    with pytest.raises(RuntimeError, match='MI355X'):
        optim.muon_step_(params, grads, momenta, lr=0.1)
    with train_on_host.patched():
        kept = [t.clone() for t in params + momenta]
        for bad in ((params, grads[:-1], momenta), (params + params[:1], grads + grads[:1], momenta + [momenta[0].clone()]),
                    ([p.clone() for p in params] + [params[0].clone()], grads + grads[:1], momenta + momenta[:1]),
                    ([torch.zeros(5)], [torch.zeros(5)], [torch.zeros(5)]), ([params[1]], [grads[2]], [momenta[1]]),
                    ([params[1].T], [grads[1].T], [momenta[1].T]), ([torch.zeros(4, 8)[:, :5]],) * 2 + ([torch.zeros(4, 5)],), ([params[0]], [grads[0]], [momenta[0].contiguous()])):
            with pytest.raises(ValueError):
                optim.muon_step_(*bad, lr=0.1)
        with pytest.raises(TypeError):
            optim.muon_step_([p.bfloat16() for p in params], [g.bfloat16() for g in grads], [m.bfloat16() for m in momenta], lr=0.1)
        with pytest.raises(TypeError):
            optim.muon_step_(params, [g.bfloat16() for g in grads], momenta, lr=0.1)
        with pytest.raises(ValueError):
            optim.muon_step_(params, grads, momenta, lr=0.1, coefficients=(5.0, 5.0, 5.0))
        optim.muon_step_([], [], [], lr=0.1)
        assert all(torch.equal(a, b) for a, b in zip(params + momenta, kept))
    with pytest.raises(ValueError):
        optim.FlowMuon([])
    opt = optim.FlowMuon([torch.nn.Parameter(torch.zeros(3, 4))])
    with pytest.raises(ValueError):
        opt.add_param_group({'params': [torch.nn.Parameter(torch.zeros(4))]})


def test_flow_muon_groups(device):
    """A group of its own step size, and a schedule on both: the weights move by lr sqrt(max(1, rows / cols)) times the same matrix."""
    g = torch.Generator().manual_seed(0)
    a, b = (torch.nn.Parameter(torch.randn(12, 20, generator=g).to(device)) for _ in range(2))
    a.grad, b.grad = torch.randn(12, 20, generator=g).to(device), torch.randn(12, 20, generator=g).to(device)
    opt = optim.FlowMuon([a], lr=0.25, momentum=0.0)
    opt.add_param_group({'params': [b], 'lr': 0.5})
    opt.param_groups[0]['lr'] = 0.125
    before = [p.detach().clone() for p in (a, b)]
    opt.step()
    for p, old, lr in zip((a, b), before, (0.125, 0.5)):
        assert torch.allclose((old - p.detach()) / lr, ops.orthogonalize(p.grad), rtol=0, atol=16 * 2**-24 * 4 / lr + 2**-20)


class _Head(torch.nn.Module):
    """A convolution, a projection and biases: what FlowMuon tells apart."""

    def __init__(self, dim=24, classes=50):
        super().__init__()
        self.conv = torch.nn.Conv2d(3, dim, 3, padding=1)
        self.proj = torch.nn.Linear(dim, dim)
        self.classes = torch.nn.Parameter(torch.randn(classes, dim) / dim**0.5)

    def forward(self, x):
        return self.proj(torch.relu(self.conv(x)).flatten(2).mT)


def _train(model, opt, x, t, loss_of, steps):
    losses = []
    for _ in range(steps):
        opt.zero_grad()
        loss = loss_of(model(x), model.classes, t)
        loss.backward()
        opt.step()
        losses.append(loss.detach().clone())
    return losses


@pytest.mark.gpu
def test_loss_and_optimiser_together():
    """The loss, its gradients and the step as a training run uses them: three steps against the same three steps in 64 bits."""
    torch.manual_seed(0)
    model = _Head().cuda()
    x = torch.randn(2, 3, 8, 8, device='cuda')
    t = torch.randint(50, (2, 64), device='cuda')
    t[0, :9] = -100
    exact = copy.deepcopy(model).double()
    opt = optim.FlowMuon(list(model.parameters()), lr=0.02, adam_lr=1e-3, weight_decay=0.01)
    losses = _train(model, opt, x, t, lambda h, w, t: ops.linear_cross_entropy(h, w, t, scale=2.0), 3)

    class Plain:
        def __init__(self, params):
            self.params = list(params)
            self.momenta = [torch.zeros_like(p) for p in self.params]
            self.adam = torch.optim.Adam([p for p in self.params if p.dim() < 2], lr=1e-3)

        def zero_grad(self):
            for p in self.params:
                p.grad = None

        @torch.no_grad()
        def step(self):
            for p, m in zip(self.params, self.momenta):
                if p.dim() >= 2:
                    new, mom = _muon(p, p.grad, m, 0.02, 0.95, 0.01, True)
                    p.copy_(new)
                    m.copy_(mom)
            self.adam.step()
    want = _train(exact, Plain(exact.parameters()), x.double(), t, lambda h, w, t: torch.nn.functional.cross_entropy(2.0 * (h @ w.T).flatten(0, 1), t.flatten()), 3)
    # fp32 convolutions and projections around the operators: a relative 2^-19 of each step's gradient, times the 485 of the iteration in its weakest
    # directions (2^-10); the first loss has seen no step
    assert abs(float(losses[0] - want[0])) <= 2**-18 * float(want[0])
    for a, b in zip(losses[1:], want[1:]):
        assert abs(float(a - b)) <= 2**-9 * float(b)
    for p, q in zip(model.parameters(), exact.parameters()):
        assert float((p.detach().double() - q.detach()).norm()) <= 3 * 0.02 * 2**-9 * math.sqrt(p.numel()) + 2**-20 * float(q.detach().norm())


@pytest.mark.gpu
def test_flow_muon_state_capture_and_checkpoint():
    """prepare() makes a capture possible; replays equal eager steps; a checkpoint goes on where it was; a missing gradient is passed over."""
    torch.manual_seed(0)
    base = _Head().cuda()
    grads = [torch.randn_like(p) * 1e-2 for p in base.parameters()]

    def fresh():
        m = copy.deepcopy(base)
        for p, g in zip(m.parameters(), grads):
            p.grad = g.clone()
        return m, optim.FlowMuon(list(m.parameters()), lr=0.02, adam_lr=1e-3)
    eager, opt = fresh()
    for _ in range(4):
        opt.step()
    captured, copt = fresh()
    with pytest.raises(RuntimeError, match='prepare'):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            copt.step()
    torch.cuda.synchronize()
    assert copt.prepare()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        copt.step()
    for _ in range(4):
        graph.replay()
        torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(eager.parameters(), captured.parameters()))
    half, hopt = fresh()
    for _ in range(2):
        hopt.step()
    state = copy.deepcopy(hopt.state_dict())
    resumed, ropt = fresh()
    resumed.load_state_dict(half.state_dict())
    ropt.load_state_dict(state)
    for _ in range(2):
        ropt.step()
    assert all(torch.equal(a, b) for a, b in zip(eager.parameters(), resumed.parameters()))
    part, popt = fresh()
    part.proj.weight.grad = None
    popt.step()
    assert torch.equal(part.proj.weight, base.proj.weight) and not torch.equal(part.classes, base.classes)


def test_flow_muon_checkpoint_of_bf16_weights(device):
    """The momentum of a bf16 weight goes through a checkpoint in its 32 bits."""
    g = torch.Generator().manual_seed(0)
    p = torch.nn.Parameter(torch.randn(9, 14, generator=g).bfloat16().to(device))
    p.grad = torch.randn(9, 14, generator=g).bfloat16().to(device)
    opt = optim.FlowMuon([p], lr=0.02)
    opt.step()
    q = torch.nn.Parameter(p.detach().clone())
    resumed = optim.FlowMuon([q], lr=0.02)
    resumed.load_state_dict(copy.deepcopy(opt.state_dict()))
    momentum = opt.state[p]['momentum_buffer']
    assert momentum.dtype == torch.float32 and not torch.equal(momentum, momentum.bfloat16().float())
    assert torch.equal(resumed.state[q]['momentum_buffer'], momentum)
    q.grad = p.grad.clone()
    opt.step()
    resumed.step()
    assert torch.equal(p, q)


def test_a_momentum_is_not_its_parameter():
    import train_on_host
    with train_on_host.patched():
        p, g = torch.ones(3, 4), torch.ones(3, 4)
        with pytest.raises(ValueError):
            optim.muon_step_([p], [g], [p], lr=0.1)
        assert torch.equal(p, torch.ones(3, 4))


@pytest.mark.gpu
@pytest.mark.parametrize('graph', [False, True])
def test_trainer_with_muon(graph):
    """The flow network's own train step with --optimizer muon: two steps, eager and replayed, whose every weight moves by what the step's formula
    allows (lr sqrt(max(1, rows / cols)) times a matrix of spectral norm below 1.3)."""
    from oracle import ref_cpu as R
    from unopticalflow_amd import get_model
    from unopticalflow_amd.trainer import FlowTrainer
    cfg = R.default_cfg()
    x = R.synthetic_triplets(2, 64, 128, seed=0, structured=True).cuda()
    torch.manual_seed(0)
    model = get_model('flow')(cfg).cuda()
    trainer = FlowTrainer(cfg, model, use_graph=graph, optimizer='muon', muon_lr=0.01)
    for k in range(2):
        before = {n: p.detach().clone() for n, p in model.named_parameters()}
        loss, _ = trainer.step(x)
        assert torch.isfinite(loss)
        for n, p in model.named_parameters():
            moved = (p.detach() - before[n]).flatten(1) if p.dim() > 1 else None
            if moved is None:
                continue
            limit = 0.01 * max(1.0, moved.shape[0] / moved.shape[1]) ** 0.5
            size = float(torch.linalg.matrix_norm(moved.double(), 2))
            assert 0.2 * limit < size < 1.3 * limit, (n, size, limit)


def test_train_command_offers_muon():
    from unopticalflow_amd.trainer import FlowTrainer
    from types import SimpleNamespace
    with pytest.raises(ValueError):
        FlowTrainer(SimpleNamespace(lr=1e-4, **_loss_weights()), torch.nn.Linear(3, 3), optimizer='sgd')
    text = open(os.path.join(ROOT, 'unopticalflow_amd', 'train.py')).read()
    assert "'--optimizer'" in text and "'--muon_lr'" in text


def _loss_weights():
    from oracle import ref_cpu as R
    return {k: v for k, v in vars(R.default_cfg()).items() if k != 'lr'}
