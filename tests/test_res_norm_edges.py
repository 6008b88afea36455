"""Calls of the residual norm at the ends of their range: gates that are shut or open for good, rows of many waves, maps without rows,
entries of the C interface that ask for a gradient nothing computes, and the module under autograd's own tools."""
import ctypes
import gc
import weakref

import pytest
import torch

from oracle import res_norm as oracle

U, K = 2.0 ** -24, 512                   # as derived in test_res_norm.py
BF, H, F = torch.bfloat16, torch.float16, torch.float32
VECS = ('scale', 'w_post', 'b_post', 'w_pre', 'b_pre')


def _close(got, want, what, floor=0.0):
    val, mag = want
    g = got.detach().cpu().double()
    tol = torch.finfo(got.dtype).eps / 2 * val.abs() + K * U * mag + floor
    if got.dtype == H:
        tol = tol + 2.0 ** -25           # below 2^-14 fp16 has a fixed step of 2^-24
    assert g.shape == val.shape and bool(torch.isfinite(g).all()), what
    worst = float(((g - val).abs() / tol.clamp_min(1e-40)).max()) if g.numel() else 0.0
    assert worst <= 1, (what, worst)


# ------------------------------------------------------------------------------------------------------------ gates shut and open
@pytest.mark.parametrize('act', ['sigmoid', 'tanh'])
def test_oracle_gate_ends(act):
    """values and slopes where 1 - a rounds to 0 or e^g overflows, against the exponential series' leading term"""
    g = torch.tensor([float('inf'), float('-inf'), 3.3e38, -3.3e38, 1e4, -1e4, 40.0, -40.0], dtype=torch.float64)
    a, slope = oracle._act(g, act)
    low = 0.0 if act == 'sigmoid' else -1.0
    e = torch.exp(torch.tensor(-40.0 if act == 'sigmoid' else -80.0, dtype=torch.float64))
    assert a[:6].tolist() == [1.0, low] * 3 and slope[:6].tolist() == [0.0] * 6
    assert bool((slope[6:] / (e if act == 'sigmoid' else 4 * e) - 1).abs().max() < 1e-15)


@pytest.mark.gpu
@pytest.mark.parametrize('xt,ft', [(BF, BF), (H, H), (F, F), (F, BF)])
@pytest.mark.parametrize('rows,C,gates', [(24, 48, 24), (96, 48, 3), (8192, 16, 1024), (6, 5000, 6), (6, 5000, 2), (3, 9000, 3)])
@pytest.mark.parametrize('act', ['sigmoid', 'tanh'])
def test_saturated_gates(act, rows, C, gates, xt, ft, dev):
    """Logits of +-inf, of the type's largest and lowest value, and every order of magnitude down to 1, among ordinary ones: for each row, for
    long and for short runs of rows.  The exponential flushes what lies below 2^-126, so a value or slope of a gate is off by that much
    besides; the terms that it multiplies are summed to less than 2^10 here: 2^-116."""
    from mscl_amd import kernels as K_
    gen = torch.Generator().manual_seed(rows + C + gates)
    ends = torch.tensor([float('inf'), float('-inf'), torch.finfo(ft).max, torch.finfo(ft).min] +
                        [s * m for s in (1, -1) for m in (6e4, 1e4, 1e3, 150.0, 104.0, 103.0, 89.0, 87.0, 60.0, 30.0, 17.0, 9.0, 4.0, 1.0)])
    gate = 2 * torch.randn(gates, C, generator=gen)
    pick = torch.randint(0, 2 * len(ends), (gates, C), generator=gen)
    gate = torch.where(pick < len(ends), ends[pick.clamp_max(len(ends) - 1)], gate).to(ft)
    assert bool(torch.isinf(gate).any())
    x, f = torch.randn(rows, C, generator=gen).to(xt), torch.randn(rows, C, generator=gen).to(ft)
    dy, dh = torch.randn(rows, C, generator=gen).to(xt), torch.randn(rows, C, generator=gen).to(ft)
    vec = {k: torch.randn(C, generator=gen) * 0.2 + (1.0 if k.startswith('w') else 0.3) for k in VECS}
    d = {k: v.double() for k, v in vec.items()}
    want = oracle.run(x.double(), f.double(), gate.double(), act, d['scale'], 'rms', d['w_post'], d['b_post'], 'layer', d['w_pre'], d['b_pre'], 1e-6,
                      dy.double(), dh.double())
    y, h, saved = K_.res_norm_fwd(x.to(dev), f.to(dev), gate=gate.to(dev), gate_act=act, post_norm='rms', pre_norm='layer', save=True,
                                  **{k: v.to(dev) for k, v in vec.items()})
    got = dict(K_.res_norm_bwd(saved, dy.to(dev), dh.to(dev)), y=y, h=h)
    for k, v in got.items():
        _close(v, want[k if k in ('y', 'h') else 'd' + k], (k, act), 2.0 ** -116)


@pytest.mark.gpu
@pytest.mark.parametrize('act', ['sigmoid', 'tanh'])
def test_nan_gates_stay_nan(act, dev):
    """a logit that is no number is not taken for a shut gate"""
    from mscl_amd import kernels as K_
    x = torch.randn(6, 64, device=dev)
    gate = torch.zeros(6, 64, device=dev)
    gate[2, 5] = float('nan')
    for g, rows in ((gate, [2]), (gate[1:4:2].contiguous(), []), (gate[2:4].contiguous(), [0, 1, 2])):
        y, _, saved = K_.res_norm_fwd(x, x, gate=g, gate_act=act, save=True)
        bad = torch.isnan(y)
        assert sorted(bad.nonzero()[:, 0].tolist()) == rows and bool((bad.nonzero()[:, 1] == 5).all())
        out = K_.res_norm_bwd(saved, x)
        assert torch.equal(torch.isnan(out['gate']), torch.isnan(g))


# ------------------------------------------------------------------------------------------------------------ no rows
@pytest.mark.gpu
@pytest.mark.parametrize('dtype', [F, BF])
def test_gates_of_an_empty_batch_get_zero_gradients(dtype, dev):
    """gates may outnumber the rows of an empty batch: their gradient is a sum over no rows"""
    from mscl_amd import kernels as K_
    x = torch.zeros(0, 16, dtype=dtype, device=dev)
    gate, w = torch.randn(3, 16, device=dev).to(dtype), torch.ones(16, device=dev)
    _, _, saved = K_.res_norm_fwd(x, x, gate=gate, scale=w, save=True)
    for _ in range(3):
        held = [torch.full((3, 16), float('nan'), dtype=dtype, device=dev) for _ in range(8)]        # what the allocator hands out next
        del held
        g = K_.res_norm_bwd(saved, x)
        assert g['gate'].shape == gate.shape and not g['gate'].any() and not g['scale'].any() and g['x'].shape == x.shape


# ------------------------------------------------------------------------------------------------------------ the module
def _module(dev, C=16, **kw):
    from mscl_amd.arena import ParamArena
    from mscl_amd.nn import ResNormHip
    from mscl_amd.recognizers import bind_module
    m = ResNormHip(C, 'rms', 'layer', scale=0.5, bias=True, **kw)
    ar = ParamArena(dev)
    plan = [(ar.add(n, p.shape), p) for n, p in m.named_parameters()]
    ar.allocate(with_key=False)
    for slot, p in plan:
        v = ar.view('Q', slot)
        v.copy_(p.data)
        p.data, p.grad, p._mscl_slot = v, ar.view('G', slot), slot
    bind_module(m, ar, False, m)
    return m, ar


@pytest.mark.gpu
def test_second_derivatives_are_refused(dev):
    """the backward pass is no graph of its own: differentiating through it would leave terms out"""
    m, _ = _module(dev)
    x, f = (torch.randn(5, 16, device=dev, requires_grad=True) for _ in range(2))
    y, h = m(x, f)
    g, = torch.autograd.grad((y * y).sum() + (h * h).sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match='once_differentiable'):
        torch.autograd.grad((g * g).sum() + (x * x).sum(), x)


class _Offload:
    """hooks that keep saved tensors on the host, densely packed"""

    def __init__(self, dev):
        self.dev, self.packed = dev, 0

    def pack(self, t):
        self.packed += 1
        return t.to('cpu', copy=True).contiguous()

    def unpack(self, t):
        return t.to(self.dev)


@pytest.mark.gpu
@pytest.mark.parametrize('strided', [False, True])
def test_saved_tensor_hooks_move_the_inputs(strided, dev):
    """under saved-tensor hooks nothing but the hooks' copies stays; gradients are the same bits, also where a copy is laid out otherwise"""
    torch.manual_seed(0)
    shape = (40, 32) if strided else (40, 16)
    x0, f0, gate0 = torch.randn(shape, device=dev), torch.randn(shape, device=dev), torch.randn(4, 16, device=dev)
    dy, dh = torch.randn(40, 16, device=dev), torch.randn(40, 16, device=dev)
    want = None
    for hooked in (False, True):
        m, ar = _module(dev)
        x, f, gate = (t.clone().requires_grad_() for t in (x0, f0, gate0))
        off = _Offload(dev)

        def forward():
            a, b, c = x * 1.0, f * 1.0, gate * 1.0
            y, h = m(a[:, 8:24], b[:, 8:24], c) if strided else m(a, b, c)
            return y, h, [weakref.ref(t) for t in (a, b, c)]
        if hooked:
            with torch.autograd.graph.saved_tensors_hooks(off.pack, off.unpack):
                y, h, refs = forward()
            gc.collect()
            assert off.packed >= 3 and all(r() is None for r in refs)
        else:
            y, h, refs = forward()
        torch.autograd.backward([y, h], [dy, dh], retain_graph=True)
        got = [x.grad.clone(), f.grad.clone(), gate.grad.clone(), ar.G.clone()]
        if want is not None:
            assert all(torch.equal(a, b) for a, b in zip(want, got))
        want = got
        torch.autograd.backward([y, h], [dy, dh])           # a second pass over the same graph accumulates
        assert torch.equal(x.grad, 2 * got[0]) and torch.equal(ar.G, 2 * got[3])


# ------------------------------------------------------------------------------------------------------------ C interface
def test_gradients_without_their_input_are_refused():
    """a bias gradient without that bias, or a gate gradient without a gate, is computed by no kernel: asked for, it is refused before any
    launch"""
    from mscl_amd import lib
    d = lib.ResNormDesc(x=16, f=16, dy=16, dh=16, rstd_f=16, rstd_y=16, ws=16, rows=4, C=8, ld_x=8, ld_f=8, rows_per_gate=4, x_type=2, f_type=2,
                        post=1, pre=1, eps=1e-6)
    d.ws_floats = lib.call_raw('mscl_res_norm_ws', ctypes.byref(d))
    for name in ('db_post', 'db_pre', 'dgate'):
        e = lib.ResNormDesc.from_buffer_copy(d)
        setattr(e, name, 16)
        assert lib.call_raw('mscl_res_norm_bwd', ctypes.byref(e), None) == -1, name


@pytest.mark.gpu
def test_captured_beside_a_living_eager_graph(dev):
    """a forward and backward pass captured while the graph of an eager pass over the same module lives; three replays against eager passes"""
    m, ar = _module(dev)
    x, f, dy = torch.randn(12, 16, device=dev), torch.randn(12, 16, device=dev), torch.randn(12, 16, device=dev)
    keep, _ = m(x.clone(), f.clone())         # never differentiated before the capture; no input needs a gradient
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ar.G.zero_()
        y, _ = m(x, f)
        torch.autograd.backward([y], [dy])
    for k in range(3):
        graph.replay()
        torch.cuda.synchronize()
        got, out = ar.G.clone(), y.detach().clone()
        ar.G.zero_()
        y2, _ = m(x, f)
        torch.autograd.backward([y2], [dy])
        torch.cuda.synchronize()
        assert torch.equal(got, ar.G) and torch.equal(out, y2) and got.any()
        x.mul_(0.7)
        dy.add_(0.1)
    first = ar.G.clone()
    torch.autograd.backward([keep], [torch.zeros_like(dy)])          # the eager graph is still whole
    assert torch.equal(first, ar.G)


@pytest.mark.gpu
def test_recomputed_in_a_checkpoint(dev):
    """activation checkpointing throws the saved tensors away and makes them again: the same gradients, added to the arena once"""
    from torch.utils.checkpoint import checkpoint
    torch.manual_seed(1)
    x0, f0, gate, dy = torch.randn(40, 16, device=dev), torch.randn(40, 16, device=dev), torch.randn(4, 16, device=dev), torch.randn(40, 16, device=dev)
    want = None
    for recompute in (False, True):
        m, ar = _module(dev)
        x, f = x0.clone().requires_grad_(), f0.clone().requires_grad_()

        def block(a, b):
            y, h = m(a * 2.0, b, gate)
            return y + h.tanh()
        out = checkpoint(block, x, f, use_reentrant=False) if recompute else block(x, f)
        out.backward(dy)
        got = [x.grad.clone(), f.grad.clone(), ar.G.clone()]
        assert want is None or all(torch.equal(a, b) for a, b in zip(want, got))
        want = got


@pytest.mark.gpu
def test_inputs_of_any_layout(dev):
    """permuted, strided and broadcast inputs of the module against dense copies of them: outputs and gradients, bit for bit"""
    torch.manual_seed(2)
    base = torch.randn(3, 16, 5, 4, device=dev)
    forms = dict(permuted=lambda t: t.permute(0, 2, 3, 1), part=lambda t: t.permute(0, 2, 3, 1)[:, 1:4], row=lambda t: t[:, :, :1, :1].permute(0, 2, 3, 1),
                 spread=lambda t: t[:1, :, :1].permute(0, 2, 3, 1).expand(3, 5, 4, 16))
    for name, form in forms.items():
        got = []
        for dense in (False, True):
            m, ar = _module(dev)
            x, f, gate = base.clone().requires_grad_(), (base * 0.5 + 1).requires_grad_(), torch.linspace(-2, 2, 48, device=dev).view(16, 3).requires_grad_()
            a, b, c = form(x), form(f), gate.t()
            y, h = m(*(t.contiguous() for t in (a, b, c))) if dense else m(a, b, c)
            gx, gf, gg = torch.autograd.grad((y * 1.5).sum() + (h * h).sum(), [x, f, gate], create_graph=True)
            assert gx.shape == x.shape and gg.shape == gate.shape
            with pytest.raises(RuntimeError, match='once_differentiable'):
                torch.autograd.grad(gx.square().sum() + x.sum(), x)
            got.append([y.detach().clone(), h.detach().clone(), gx.detach(), gf.detach(), gg.detach(), ar.G.clone()])
        assert all(torch.equal(p, q) for p, q in zip(*got)), name
