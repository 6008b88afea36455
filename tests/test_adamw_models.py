"""AdamW and the residual norm as a model uses them: blocks of norms, gates and linear / convolution layers bound to a parameter arena, their
backward pass into its gradients, and optimizer steps over it; the optimizer on the framework's own models, captured and resumed."""
import os

import numpy as np
import pytest
import torch
import torch.nn as nn
import torch.nn.functional as F

from oracle import adamw as oracle

U = 2.0 ** -24


class _Rows(nn.Module):
    """two residual blocks over (N, T, C) rows: linear branches, a gate per clip, a classifier over the mean row"""

    def __init__(self, C, classes):
        super().__init__()
        from mscl_amd.nn import LinearHip, ResNormHip
        self.norm0 = ResNormHip(C, post=None, pre='rms')
        self.fc1, self.fc2, self.head = LinearHip(C, C), LinearHip(C, C), LinearHip(C, classes)
        self.norm1 = ResNormHip(C, 'rms', 'layer', scale=0.1, bias=True)
        self.norm2 = ResNormHip(C, 'layer', 'rms', scale=0.2, gate_act='tanh')

    def forward(self, x, gate):
        from mscl_amd.recognizer3d import _LinearFn
        lin = lambda t, m: _LinearFn.apply(t.reshape(-1, t.shape[-1]), m).view(*t.shape[:-1], -1)          # noqa: E731
        x, h = self.norm0(x)
        x, h = self.norm1(x, lin(h, self.fc1), gate)
        x, h = self.norm2(x, lin(h, self.fc2), gate)
        return lin(h.mean(1), self.head)

    def sync_streams(self):
        pass

    def refresh_after_optimizer(self):
        pass


def _rows_ref(p, x, gate):
    """the same in plain torch at the parameters' precision"""
    def norm(v, kind, w, b=None):
        if kind == 'layer':
            v = v - v.mean(-1, keepdim=True)
        v = v / torch.sqrt((v * v).mean(-1, keepdim=True) + 1e-6) * w
        return v if b is None else v + b
    g = gate[:, None]
    h = norm(x, 'rms', p['norm0.w_pre'])
    f = norm(h @ p['fc1.weight'].t() + p['fc1.bias'], 'rms', p['norm1.w_post'], p['norm1.b_post'])
    x = x + p['norm1.scale'] * torch.sigmoid(g) * f
    h = norm(x, 'layer', p['norm1.w_pre'], p['norm1.b_pre'])
    f = norm(h @ p['fc2.weight'].t() + p['fc2.bias'], 'layer', p['norm2.w_post'])
    x = x + p['norm2.scale'] * torch.tanh(g) * f
    h = norm(x, 'rms', p['norm2.w_pre'])
    return h.mean(1) @ p['head.weight'].t() + p['head.bias']


def _materialize(model, dev):
    from mscl_amd.arena import ParamArena
    from mscl_amd.recognizers import bind_module
    ar = ParamArena(dev)
    plan = [(ar.add(n, p.shape), p) for n, p in model.named_parameters()]
    ar.allocate(with_key=False)
    for slot, p in plan:
        v = ar.view('Q', slot)
        v.copy_(p.data)
        p.data, p.grad, p._mscl_slot = v, ar.view('G', slot), slot
    model.arena = ar
    for m in model.modules():
        bind_module(m, ar, False, model)
    return model


def test_unbound_module_and_argument_errors():
    from mscl_amd import build_optimizer
    from mscl_amd.lib import MsclError
    from mscl_amd.nn import ResNormHip
    m = ResNormHip(8, 'rms', 'layer', scale=0.5, bias=True)
    assert {n: tuple(p.shape) for n, p in m.named_parameters()} == {k: (8,) for k in ('scale', 'w_post', 'b_post', 'w_pre', 'b_pre')}
    assert float(m.scale[0]) == 0.5 and float(m.w_post[0]) == 1 and float(m.b_pre[0]) == 0
    assert [n for n, _ in ResNormHip(8, None, 'rms').named_parameters()] == ['w_pre']
    with pytest.raises(MsclError):
        m(torch.zeros(2, 8))
    with pytest.raises(ValueError):
        ResNormHip(8, 'batch')
    with pytest.raises(NotImplementedError, match='Adagrad'):
        build_optimizer(None, dict(type='Adagrad', lr=1))
    with pytest.raises(NotImplementedError, match='amsgrad'):
        build_optimizer(None, dict(type='AdamW', lr=1, amsgrad=True))


def _expect_step(opt, before, grads, max_norm, t, lr, wd):
    """checks every slot of a ClipAdamW step against the formula in 64 bits on the states and gradients from before"""
    inner = opt._inner
    coef, norm = oracle.coefficient(list(grads.values()), max_norm)
    if max_norm:
        assert abs(float(opt.grad_norm()) - norm) <= 2 * U * norm
    for i, slot in enumerate(opt._slots):
        a, b = opt._mult.get(slot, (1.0, 1.0))
        o, n = inner.offsets[i], slot.numel
        m0, v0 = (s[o:o + n] for s in before['states'])
        G, P = grads[slot.name], before['Q'][slot.off:slot.off + n]
        rate = lr * a
        new, m, v = oracle.step(P, G, m0, v0, t, coef, rate, decay=wd * b)
        M = np.abs(0.9 * m0) + np.abs(0.1 * coef * G)
        upd = rate / (1 - 0.9 ** t) * M / (np.sqrt(v / (1 - 0.999 ** t)) + 1e-8)
        got = opt.arena.Q[slot.off:slot.off + n].cpu().double().numpy()
        tol = 4 * U * np.maximum(np.abs(P), np.abs(new)) + 24 * U * upd + 1e-38
        assert (np.abs(got - new) <= tol).all(), slot.name
        assert torch.equal(opt.arena.Qb[slot.off:slot.off + n], opt.arena.Q[slot.off:slot.off + n].bfloat16())


def _snapshot(opt):
    inner = opt._inner
    return dict(Q=opt.arena.Q.cpu().double().numpy(),
                states=None if inner is None else [s.cpu().double().numpy() for s in inner.state_values()])


@pytest.mark.gpu
@pytest.mark.parametrize('bits', [32, 8])
def test_residual_rows_train(bits, dev):
    """three steps; per step the gradients against autograd in 64 bits at the same parameters, then the update against the formula.
    A gradient passes five stages (norms, linear layers of 48 terms), each within 512 u of its terms: 5 * 512 u = 1.5e-4 of a tensor's
    norm."""
    from mscl_amd import build_optimizer
    torch.manual_seed(0)
    N, T, C, classes = 6, 9, 48, 5
    model = _materialize(_Rows(C, classes), dev)
    opt = build_optimizer(model, dict(type='AdamW', lr=2e-3, weight_decay=0.1, state_bits=bits, paramwise_cfg=dict(norm_decay_mult=0.0, custom_keys={
        'head': dict(lr_mult=10.0)})), dict(grad_clip=dict(max_norm=0.5, norm_type=2)))
    gen = torch.Generator().manual_seed(3)
    for t in range(1, 4):
        x, gate = torch.randn(N, T, C, generator=gen), torch.randn(N, C, generator=gen)
        label = torch.randint(0, classes, (N,), generator=gen)
        p64 = {n: p.detach().cpu().double().requires_grad_() for n, p in model.named_parameters()}
        gate64 = gate.double().requires_grad_()
        loss64 = F.cross_entropy(_rows_ref(p64, x.double(), gate64), label)
        loss64.backward()
        gd = gate.to(dev).requires_grad_()
        opt.zero_grad()
        loss = F.cross_entropy(model(x.to(dev), gd), label.to(dev))
        loss.backward()
        assert abs(float(loss.detach()) - float(loss64.detach())) <= 1.5e-4 * max(1.0, float(loss64.detach()))
        for n, p in list(model.named_parameters()) + [('gate', gd)]:
            want = gate64.grad if n == 'gate' else p64[n].grad
            off, size = float((p.grad.cpu().double() - want).norm()), float(want.norm())
            assert off <= 1.5e-4 * size + 1e-9, (n, off / size)
        before = _snapshot(opt)
        if before['states'] is None:
            before['states'] = [np.zeros(sum(-(-s.numel // 256) * 256 for s in model.arena.slots))] * 2
        grads = {s.name: model.arena.G[s.off:s.off + s.numel].cpu().double().numpy() for s in model.arena.slots}
        opt.param_groups[0]['lr'] = 2e-3 / t
        opt.step()
        assert all(s.touched for s in model.arena.slots)
        _expect_step(opt, before, grads, 0.5, t, float(np.float32(2e-3 / t)), 0.1)
    assert opt.steps == opt._inner.device_step() == 3
    norm_slots = [s for s in opt._slots if s.name.startswith('norm')]
    assert norm_slots and all(opt._mult[s] == (1.0, 0.0) for s in norm_slots)
    assert [opt._mult[s] for s in opt._slots if s.name.startswith('head')] == [(10.0, 1.0)] * 2


@pytest.mark.gpu
def test_residual_norm_around_a_convolution(dev):
    """a bottleneck-like block on an NDHWC bf16 map: norm, 1x1x1 convolution, gated residual, norm.  Against autograd in fp32 on the
    same values: h, f, y and the gradients of h, f and x are rounded to bf16 on the way, at most 6 half steps of 2^-8 of the terms: 2.4 %."""
    from mscl_amd import kernels as K
    from mscl_amd.nn import Conv3dHip, ResNormHip, conv_bias
    torch.manual_seed(1)
    C = 64

    class Block(nn.Module):
        def __init__(self):
            super().__init__()
            self.a, self.conv, self.b = ResNormHip(C, None, 'rms'), Conv3dHip(C, C, 1, 1, 0), ResNormHip(C, 'rms', 'layer', scale=0.5)

        def forward(self, x, gate):
            x, h = self.a(x)
            return self.b(x, conv_bias(self.conv, h), gate)
    block = Block()
    nn.init.normal_(block.conv.weight, 0.0, 0.1)                # (the module leaves its weight uninitialised)
    m = _materialize(block, dev)
    K.cast_bf16(m.arena.Q, m.arena.Qb)
    m.conv._rt['wT'].copy_(m.arena.packed('Qb', m.conv.weight._mscl_slot).permute(4, 1, 2, 3, 0))
    x = torch.randn(2, 3, 8, 8, C).bfloat16()
    gate, dy, dh = torch.randn(2, C).bfloat16(), torch.randn(2, 3, 8, 8, C).bfloat16(), torch.randn(2, 3, 8, 8, C).bfloat16()
    xd, gd = x.to(dev).requires_grad_(), gate.to(dev).requires_grad_()
    y, h = m(xd, gd)
    torch.autograd.backward([y, h], [dy.to(dev), dh.to(dev)])
    torch.cuda.synchronize()
    p = {n: v.detach().cpu().float().requires_grad_() for n, v in m.named_parameters()}
    p['conv.weight'] = p['conv.weight'].detach().bfloat16().float().requires_grad_()
    xr, gr = x.float().requires_grad_(), gate.float().requires_grad_()

    def rms(v):
        return v / torch.sqrt((v * v).mean(-1, keepdim=True) + 1e-6)
    f = (rms(xr) * p['a.w_pre']) @ p['conv.weight'].reshape(C, C).t()
    yr = xr + p['b.scale'] * torch.sigmoid(gr)[:, None, None, None] * rms(f) * p['b.w_post']
    c = yr - yr.mean(-1, keepdim=True)
    hr = rms(c) * p['b.w_pre']
    torch.autograd.backward([yr, hr], [dy.float(), dh.float()])
    for got, want, what in [(y, yr, 'y'), (h, hr, 'h'), (xd.grad, xr.grad, 'dx'), (gd.grad, gr.grad, 'dgate')] + \
            [(dict(m.named_parameters())[n].grad, v.grad, n) for n, v in p.items()]:
        off, size = float((got.detach().cpu().float() - want.detach()).norm()), float(want.detach().norm())
        assert off <= 0.024 * size, (what, off / size)


@pytest.mark.gpu
def test_module_edges(dev):
    """unused outputs, no grad mode, inputs without gradients, double use, an input changed before the backward pass"""
    from mscl_amd.nn import ResNormHip, _ResNormFn
    m = _materialize(nn.Sequential(ResNormHip(16, 'rms', 'rms', scale=1.0)), dev)
    n, ar = m[0], m.arena
    x, f = torch.randn(5, 16, device=dev), torch.randn(5, 16, device=dev)
    with torch.no_grad():
        y0, h0 = n(x, f)
    assert not y0.requires_grad
    y, h = n(x, f)                                   # no input needs a gradient: the module's parameters still do
    assert torch.equal(y, y0) and torch.equal(h, h0)
    y.sum().backward()
    by = {s.name: s for s in ar.slots}
    assert by['0.scale'].touched and by['0.w_post'].touched and not by['0.w_pre'].touched
    assert ar.view('G', by['0.scale']).any() and not ar.view('G', by['0.w_pre']).any()
    once = ar.G.clone()
    y, h = n(x, f)
    y2, h2 = n(x, f)
    (y.sum() + y2.sum()).backward()                  # accumulated
    assert torch.equal(ar.G, once + once + once) or torch.allclose(ar.G, 3 * once, rtol=4 * U, atol=0)
    y, h = n(x, f)
    h.sum().backward()
    assert by['0.w_pre'].touched
    x2 = x.clone().requires_grad_()
    y, h = n(x2 * 1.0, f)
    f.add_(1.0)
    with pytest.raises(RuntimeError, match='modified by an inplace operation'):
        y.sum().backward()
    _, h = n(x)
    h.sum().backward()                               # no branch: the pre-norm alone
    from mscl_amd.lib import MsclError
    y, h = n(x, f)
    dy = torch.ones_like(y)
    with pytest.raises(MsclError, match='capture'):              # an eager forward's backward inside a capture
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            _ResNormFn.backward(y.grad_fn, dy, None)


@pytest.mark.gpu
def test_finetune_with_adamw_and_its_state(dev):
    """Recognizer3D: clip + AdamW against the formula; the state goes into a second model, whose next step is the same bits; so does a state
    of torch.optim.AdamW, by parameter index"""
    from mscl_amd import build_model, build_optimizer
    from mscl_amd.fill import fill_module
    from mscl_amd.lib import MsclError
    cfg = dict(type='AdamW', lr=1e-3, weight_decay=0.05, paramwise_cfg=dict(norm_decay_mult=0.0, bias_decay_mult=0.0))
    clip = dict(grad_clip=dict(max_norm=5.0, norm_type=2))

    def make(bits):
        m = build_model(dict(type='Recognizer3D', backbone=dict(type='torchvision.r3d_18'),
                             cls_head=dict(type='I3DHead', num_classes=5, in_channels=512, spatial_type='none', dropout_ratio=0.0)))
        fill_module(m)
        m.materialize(dev).train()
        return m, build_optimizer(m, dict(cfg, state_bits=bits), clip)
    imgs, label = torch.randn(2, 1, 3, 8, 32, 32, device=dev), torch.tensor([[1], [3]], device=dev)
    for bits in (32, 8):
        m, opt = make(bits)
        with pytest.raises(MsclError):
            opt.step()                                # nothing has a gradient yet
        m.train_step(dict(imgs=imgs, label=label))['loss'].backward()
        total = sum(-(-s.numel // 256) * 256 for s in m.arena.slots if s.touched)
        before = dict(Q=m.arena.Q.cpu().double().numpy(), states=[np.zeros(total)] * 2)
        grads = {s.name: m.arena.G[s.off:s.off + s.numel].cpu().double().numpy() for s in m.arena.slots if s.touched}
        opt.step()
        _expect_step(opt, before, grads, 5.0, 1, float(np.float32(1e-3)), 0.05)
        state = {k: v.cpu() if torch.is_tensor(v) else v for k, v in opt.state_dict().items()}
        m2, opt2 = make(bits)
        m2.arena.Q.copy_(m.arena.Q)
        opt2.load_state_dict(state)
        m2.arena.G.copy_(m.arena.G)
        opt.step()
        opt2.step()
        assert opt2.steps == 2 and torch.equal(m.arena.Q, m2.arena.Q) and torch.equal(m.arena.Qb, m2.arena.Qb)
        assert torch.equal(opt._inner.exp_avg, opt2._inner.exp_avg) and torch.equal(opt._inner.exp_avg_sq, opt2._inner.exp_avg_sq)
        with pytest.raises(MsclError):
            make(40 - bits)[1].load_state_dict(state)
    # torch.optim.AdamW's own state
    m, opt = make(32)
    ref = [p.detach().clone().requires_grad_() for p in m.parameters()]
    topt = torch.optim.AdamW(ref, lr=3e-3, weight_decay=0.05)
    for p in ref:
        p.grad = torch.randn_like(p) * 0.01
    topt.step()
    opt.load_state_dict(topt.state_dict())
    assert opt.steps == opt._inner.device_step() == 1 and opt.param_groups[0]['lr'] == 3e-3
    from mscl_amd.arena import _physical_view
    at = dict(zip(opt._slots, opt._inner.offsets))
    for p, r in zip(m.parameters(), ref):
        assert torch.equal(_physical_view(opt._inner.exp_avg, at[p._mscl_slot], p._mscl_slot.shape), topt.state[r]['exp_avg'])
        assert torch.equal(_physical_view(opt._inner.exp_avg_sq, at[p._mscl_slot], p._mscl_slot.shape), topt.state[r]['exp_avg_sq'])


@pytest.mark.gpu
@pytest.mark.parametrize('bits', [32, 8])
def test_pretraining_step_captured_and_resumed(bits, dev, tmp_path):
    """the whole MSCL step with AdamW: graph replays are the eager steps bit for bit (deterministic mode); a checkpoint goes on as the run does"""
    from mscl_amd import Config, build_model, build_optimizer, lib, train as tr
    from mscl_amd.fill import fill_module
    from mscl_amd.graph import GraphedStep
    from mscl_amd.synthetic import synthetic_batch
    B, T, H, Kq = 2, 8, 32, 64
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

    def build():
        cfg = Config.fromfile(os.path.join(root, 'configs/recognition/moco/mscl_r18_cosm_lr2e-2.py'))
        cfg.model.sup_head.t = T // 2
        cfg.model.recognizer.K = cfg.model.recognizer_flow.K = Kq
        torch.manual_seed(0)
        m = build_model(cfg.model)
        fill_module(m)
        m.materialize(dev).train()
        return m, build_optimizer(m, dict(type='AdamW', lr=1e-3, weight_decay=0.05, state_bits=bits), dict(grad_clip=dict(max_norm=40, norm_type=2)))
    batches = [synthetic_batch(B, T, H, H, 0, s, device=dev) for s in range(3)]

    def eager(m, opt, batch):
        out = m.train_step(batch, sync_logs=False)
        opt.zero_grad()
        out['loss'].backward()
        opt.step()
        return float(out['loss'].detach())
    lib.set_deterministic(True)
    try:
        m, opt = build()
        ref = []
        path = str(tmp_path / 'ck.pth')
        for i, s in enumerate((0, 0, 0, 1, 2)):
            if i == 4:
                tr.save_checkpoint(path, m, opt, epoch=1, it=4)
            opt.param_groups[0]['lr'] = 1e-3 / (i + 1)
            ref.append(eager(m, opt, batches[s]))
        g, gopt = build()
        gopt.param_groups[0]['lr'] = 1e-3
        step = GraphedStep(g, gopt, batches[0], warmup=2)
        got = []
        for i, s in enumerate((0, 1, 2)):
            gopt.param_groups[0]['lr'] = 1e-3 / (i + 3)
            got.append(float(step.step(batches[s])[0]))
        assert gopt._inner.device_step() == gopt.steps == 5
        r2, r2opt = build()                       # the graph's warm-up steps both ran at 1e-3
        want = []
        for i, s in enumerate((0, 0, 0, 1, 2)):
            r2opt.param_groups[0]['lr'] = 1e-3 if i < 2 else 1e-3 / (i + 1)
            want.append(eager(r2, r2opt, batches[s]))
        assert got == want[2:]
        assert torch.equal(g.arena.Q, r2.arena.Q) and torch.equal(gopt._inner.exp_avg_sq, r2opt._inner.exp_avg_sq)
        c, copt = build()
        c.arena.Q.zero_()
        tr.resume(path, c, copt)
        assert copt.steps == copt._inner.device_step() == 4
        copt.param_groups[0]['lr'] = 1e-3 / 5
        assert eager(c, copt, batches[2]) == ref[4]
        assert torch.equal(c.arena.Q, m.arena.Q) and torch.equal(copt._inner.exp_avg, opt._inner.exp_avg)
    finally:
        lib.set_deterministic(False)
