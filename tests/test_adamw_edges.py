"""Calls of the AdamW step at the ends of their range, its checkpoints across other parameters and other optimizers, and what autograd sees of
it."""
import ctypes
import os
import re

import numpy as np
import pytest
import torch
import torch.nn as nn

U = 2.0 ** -24
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_a_clip_that_is_no_number_is_refused_by_the_library():
    """without a clip `partials` and `grad_norm` may be NULL, so a max_norm that compares neither way must not get to the kernels"""
    from mscl_amd import lib
    d = lib.AdamWDesc(tensors=16, grads=16, chunk_tensor=16, m=16, v=16, words=16, lr=16, beta1=0.9, beta2=0.999, eps=1e-8, max_norm=float('nan'),
                      n_chunks=1, state_bits=32, grad_type=1)
    assert lib.call_raw('mscl_adamw_step', ctypes.byref(d), None) == -1


def test_eps_below_the_normal_range_is_refused():
    """the reciprocal of a subnormal is infinite, and an element with no gradient yet would be 0 * inf"""
    from mscl_amd import lib, optim
    from mscl_amd.lib import MsclError
    for eps in (1e-38, 1e-45):
        with pytest.raises(MsclError, match='eps'):
            optim.AdamW([torch.zeros(3)], eps=eps)
    with pytest.raises(MsclError, match='no CPU fallback'):
        optim.AdamW([torch.zeros(3)], eps=1.2e-38)
    d = lib.AdamWDesc(tensors=16, grads=16, chunk_tensor=16, m=16, v=16, words=16, lr=16, beta1=0.9, beta2=0.999, eps=1e-38, n_chunks=1,
                      state_bits=32, grad_type=1)
    assert lib.call_raw('mscl_adamw_step', ctypes.byref(d), None) == -1


@pytest.mark.gpu
@pytest.mark.parametrize('bits', [32, 8])
@pytest.mark.parametrize('eps', [1e-8, 1e-15, 1e-20, 1e-30, 2e-38])
def test_second_moments_below_the_normal_range(eps, bits, dev):
    """gradients whose squares are subnormal, beside zeros and ordinary ones: the first step against the formula on the second moment as fp32
    holds it.  24 u of the update and 4 u of p (as derived in test_adamw.py), whatever eps is."""
    from mscl_amd import AdamW
    g = torch.cat([torch.zeros(5)] + [torch.full((7,), 10.0 ** -k) * (1 + torch.arange(7) / 7) for k in (2, 8, 14, 17, 18, 19, 20, 21)])
    p = torch.zeros(g.numel(), device=dev)
    opt = AdamW([p], lr=1.0, eps=eps, weight_decay=0.0, state_bits=bits)
    opt.step([g.to(dev)])
    G = g.numpy()
    v = (G * G) * np.float32(1 - 0.999)
    assert v.dtype == np.float32 and ((v > 0) & (v < 2.0 ** -126)).sum() > 10
    m = G.astype(np.float64) * 0.1
    want = -(m / (1 - 0.9)) / (np.sqrt(v.astype(np.float64) / (1 - 0.999)) + float(np.float32(eps)))
    got = p.cpu().double().numpy()
    assert (np.abs(got - want) <= 28 * U * np.abs(want) + 1e-38).all(), (got / np.where(want == 0, 1, want)).tolist()


def test_kernel_constants_are_the_headers():
    """chunk, block, number of partial sums and the layout of the words buffer are written once, in the header"""
    src = open(os.path.join(ROOT, 'mscl_amd', 'csrc', 'adamw.hip')).read()
    for name in ('CHUNK', 'PARTS'):
        assert re.search(rf'constexpr int {name} = MSCL_ADAMW_{name};', src), name
    assert 'sizeof(Words) == MSCL_ADAMW_WORDS' in src and 'MSCL_ADAMW_BLOCK ==' in src


@pytest.mark.gpu
def test_a_step_invalidates_graphs_of_before(dev):
    """a backward pass over a graph from before the step would use the new weights in the place of the saved ones: refused, as after any
    other in-place change; shadows count too"""
    from mscl_amd import AdamW
    net = nn.Sequential(nn.Linear(8, 8), nn.Linear(8, 3)).to(dev)
    opt = AdamW(net.parameters(), lr=1e-2)
    x = torch.randn(4, 8, device=dev)
    loss = net(x).square().sum()
    loss.backward(retain_graph=True)
    opt.step()
    with pytest.raises(RuntimeError, match='modified by an inplace operation'):
        loss.backward()
    opt.zero_grad()
    net(x).square().sum().backward()
    opt.step()
    master = torch.randn(8, 8, device=dev)
    shadow = master.bfloat16().requires_grad_()
    opt = AdamW([master], shadows=[shadow.detach()])
    x16 = x.bfloat16().requires_grad_()
    out = (x16 @ shadow).float().sum()
    opt.step([torch.ones(8, 8, device=dev)])
    with pytest.raises(RuntimeError, match='modified by an inplace operation'):
        out.backward()
    with torch.inference_mode():
        p = torch.zeros(5, device=dev)
    AdamW([p]).step([torch.ones(5, device=dev)])          # (a tensor without a version counter is stepped as before)
    assert bool((p < 0).all())


@pytest.mark.gpu
def test_changed_settings_are_refused(dev):
    """lr is read at every step; a change of the others would be ignored"""
    from mscl_amd import AdamW
    from mscl_amd.lib import MsclError
    p, g = torch.zeros(5, device=dev), torch.ones(5, device=dev)
    opt = AdamW([p], lr=1e-2)
    opt.step([g])
    for key, v in (('weight_decay', 0.5), ('eps', 1e-3), ('betas', (0.5, 0.9))):
        old = opt.param_groups[0][key]
        opt.param_groups[0][key] = v
        before = p.clone()
        with pytest.raises(MsclError, match='param_groups'):
            opt.step([g])
        with pytest.raises(MsclError, match='param_groups'):
            opt.sync_lr()
        assert torch.equal(p, before) and opt.device_step() == 1
        opt.param_groups[0][key] = list(old) if key == 'betas' else old
    opt.step([g])
    assert opt.device_step() == 2


@pytest.mark.gpu
def test_gradients_of_another_type_at_the_same_address(dev):
    """wider gradients at the address of narrow ones reach further: their memory is looked at again"""
    from mscl_amd import AdamW
    from mscl_amd.lib import MsclError
    buf = torch.zeros(64, device=dev)
    p = buf[16:48]                                         # bytes 64 .. 191
    g16 = buf.view(torch.bfloat16)[:32]                    # bytes 0 .. 63
    opt = AdamW([p])
    opt.step([g16])
    with pytest.raises(MsclError, match='share memory'):
        opt.step([buf[:32]])                               # bytes 0 .. 127
    opt.step([g16])
    assert opt.device_step() == 2


@pytest.mark.gpu
@pytest.mark.parametrize('bits', [32, 8])
def test_states_of_other_tensors_are_refused(bits, dev):
    """the flat states belong to a list of tensors: another list that pads to as many blocks does not take them"""
    from mscl_amd import AdamW
    from mscl_amd.lib import MsclError

    def make(sizes):
        ps = [torch.zeros(n, device=dev) for n in sizes]
        opt = AdamW(ps, state_bits=bits)
        opt.step([torch.ones_like(p) for p in ps])
        return opt
    a = make([300, 10, 77])
    state = a.state_dict()
    for sizes in ([10, 300, 77], [300, 77, 10], [300, 256, 256], [768, 256]):
        b = make(sizes)
        assert b.numel == a.numel
        before = b.state_dict()
        with pytest.raises(MsclError, match='other parameters'):
            b.load_state_dict(state)
        after = b.state_dict()
        assert all(torch.equal(v, after[k]) if torch.is_tensor(v) else v == after[k] for k, v in before.items())
    c = make([300, 10, 77])
    c.load_state_dict(state)
    old = {k: v for k, v in state.items() if k in ('step', 'state_bits', 'lr', 'seed', 'exp_avg', 'exp_avg_sq', 'exponents')}
    c.load_state_dict(old)                                 # a state written without the sizes


class _Net(nn.Module):
    """three norms bound to an arena; `first` and `last` may have rates of their own"""

    def __init__(self):
        super().__init__()
        from mscl_amd.nn import ResNormHip
        self.first, self.mid, self.last = ResNormHip(24, None, 'rms'), ResNormHip(24, 'rms', None, scale=0.5), ResNormHip(24, 'layer', None, bias=True)

    def forward(self, x, upto=3):
        x, h = self.first(x)
        if upto > 1:
            x, _ = self.mid(x, h)
        if upto > 2:
            x, _ = self.last(x, h)
        return x if upto > 1 else h

    def sync_streams(self):
        pass

    def refresh_after_optimizer(self):
        pass


def _net(dev, bits=32, **cfg):
    from mscl_amd import build_optimizer
    from mscl_amd.arena import ParamArena
    from mscl_amd.recognizers import bind_module
    model, ar = _Net(), ParamArena(dev)
    plan = [(ar.add(n, p.shape), p) for n, p in model.named_parameters()]
    ar.allocate(with_key=False)
    for slot, p in plan:
        v = ar.view('Q', slot)
        v.copy_(p.data)
        p.data, p.grad, p._mscl_slot = v, ar.view('G', slot), slot
    model.arena = ar
    for m in model.modules():
        bind_module(m, ar, False, model)
    return model, build_optimizer(model, dict(type='AdamW', lr=1e-3, state_bits=bits, **cfg))


def _train(model, opt, steps=1, upto=3):
    for s in range(steps):
        opt.zero_grad()
        x = torch.randn(6, 24, generator=torch.Generator().manual_seed(s)).to(model.arena.device)
        model(x, upto).square().sum().backward()
        opt.step()


def _torch_state(model, lrs, steps=1, skip=()):
    """torch.optim.AdamW's state over the model's parameters, a group for each"""
    ref = [p.detach().clone().requires_grad_() for p in model.parameters()]
    groups = [dict(params=[p], lr=lr) for p, lr in zip(ref, lrs)]
    opt = torch.optim.AdamW(groups)
    for _ in range(steps):
        for i, p in enumerate(ref):
            p.grad = None if i in skip else torch.randn_like(p)
        opt.step()
    return opt.state_dict()


@pytest.mark.gpu
def test_paramwise_rates_of_a_torch_state(dev):
    """torch's groups hold lr times the parameter's multiplier: the base rate is what is left without it, from whichever group; groups that
    disagree, as under another paramwise_cfg, are refused and change nothing"""
    from mscl_amd.lib import MsclError
    from mscl_amd.optim import _param_mults
    cfg = dict(custom_keys=dict(first=dict(lr_mult=0.1), last=dict(lr_mult=0.0)))
    model, opt = _net(dev, paramwise_cfg=cfg)
    mult, _ = _param_mults(list(model.named_parameters()), set(), cfg)
    assert mult[0] == 0.1 and 1.0 in mult and mult[-1] == 0.0
    opt.load_state_dict(_torch_state(model, [3e-4 * m for m in mult]))
    assert abs(opt.param_groups[0]['lr'] / 3e-4 - 1) < 1e-12
    one = _torch_state(model, [3e-4] * len(mult))
    m2, o2 = _net(dev, paramwise_cfg=cfg)
    with pytest.raises(MsclError, match='rate'):
        o2.load_state_dict(one)
    assert o2._inner is None and o2.param_groups[0]['lr'] == 1e-3 and not any(s.touched for s in m2.arena.slots)
    m3, o3 = _net(dev)
    o3.load_state_dict(one)
    assert o3.param_groups[0]['lr'] == 3e-4
    m4, o4 = _net(dev, paramwise_cfg=dict(norm_decay_mult=0.0, custom_keys=dict(first=dict(lr_mult=0.0), mid=dict(lr_mult=0.0), last=dict(lr_mult=0.0))))
    o4.load_state_dict(_torch_state(m4, [0.0] * len(mult)))
    assert o4.param_groups[0]['lr'] == 1e-3               # no group tells: as configured


@pytest.mark.gpu
def test_moments_that_a_torch_state_lacks_start_at_zero(dev):
    """loaded into an optimizer that has stepped: parameters without an entry have no moments, as in torch"""
    model, opt = _net(dev)
    _train(model, opt, 3)
    n = len(list(model.parameters()))
    state = _torch_state(model, [1e-3] * n, steps=2, skip=(1, n - 1))
    opt.load_state_dict(state)
    assert opt.steps == opt._inner.device_step() == 2
    at = dict(zip(opt._slots, opt._inner.offsets))
    for i, p in enumerate(model.parameters()):
        for flat, key in ((opt._inner.exp_avg, 'exp_avg'), (opt._inner.exp_avg_sq, 'exp_avg_sq')):
            got = flat[at[p._mscl_slot]:at[p._mscl_slot] + p.numel()].view(p.shape)
            want = state['state'][i][key] if i in state['state'] else torch.zeros_like(p)
            assert torch.equal(got, want.detach()), (i, key)


@pytest.mark.gpu
def test_amsgrad_states_are_refused(dev):
    """a maximum of second moments is no part of this step"""
    model, opt = _net(dev)
    ref = [p.detach().clone().requires_grad_() for p in model.parameters()]
    topt = torch.optim.AdamW(ref, lr=1e-3, amsgrad=True)
    for p in ref:
        p.grad = torch.randn_like(p)
    topt.step()
    with pytest.raises(NotImplementedError, match='amsgrad'):
        opt.load_state_dict(topt.state_dict())
    assert opt._inner is None


@pytest.mark.gpu
@pytest.mark.parametrize('bits', [32, 8])
def test_the_state_from_before_the_first_step(bits, dev):
    """loaded into an optimizer that has stepped, it takes that one back to its beginning"""
    model, opt = _net(dev, bits)
    first = opt.state_dict()
    q = model.arena.Q.clone()
    _train(model, opt, 2)
    want = model.arena.Q.clone()
    opt.load_state_dict(first)
    assert opt.steps == 0 and opt._inner.device_step() == 0
    assert not any(v.any() for v in opt._inner.state_values())
    model.arena.Q.copy_(q)
    _train(model, opt, 2)
    assert torch.equal(model.arena.Q, want)


@pytest.mark.gpu
def test_a_refused_state_changes_nothing(dev):
    """states of another model, of other parameters or damaged ones: parameters that take part, moments, counter and rate stay"""
    from mscl_amd.lib import MsclError
    model, opt = _net(dev)
    _train(model, opt, 2)
    whole = opt.state_dict()
    part, popt = _net(dev)
    _train(part, popt, 1, upto=2)                          # `last` has received no gradient
    before = popt.state_dict()
    inner, slots = popt._inner, list(popt._slots)
    bad = [dict(whole, slots=[0, 99]), dict(whole, exp_avg=whole['exp_avg'][:256]), dict(whole, exp_avg_sq=whole['exp_avg_sq'].double()),
           dict(whole, slots=whole['slots'][1:]), dict(whole, step=-1), dict(whole, state_bits=8)]
    other = _torch_state(part, [1e-3] * len(list(part.parameters())))
    worse = {k: dict(v) for k, v in other['state'].items()}
    worse[4] = dict(worse[4], exp_avg_sq=worse[4]['exp_avg_sq'][:3])
    for state in bad + [dict(other, state=worse)]:
        with pytest.raises((MsclError, ValueError)):
            popt.load_state_dict(state)
        assert popt._inner is inner and popt._slots == slots and [s for s in part.arena.slots if s.touched] == slots
        after = popt.state_dict()
        assert all(torch.equal(v, after[k]) if torch.is_tensor(v) else v == after[k] for k, v in before.items()), state.get('slots')
    for state in bad:                                      # the same before the first step
        fresh, fopt = _net(dev)
        with pytest.raises(MsclError):
            fopt.load_state_dict(state)
        assert fopt._inner is None and not any(s.touched for s in fresh.arena.slots) and fopt.param_groups[0]['lr'] == 1e-3
    popt.load_state_dict(whole)                            # a whole one for more parameters is taken: nothing of it is captured
    assert popt._slot_indices() == whole['slots'] and popt.steps == 2


@pytest.mark.gpu
def test_a_captured_step_keeps_its_memory(dev):
    """a captured step reads and writes the optimizer's buffers: a state that would need others is refused, one that fits goes into them"""
    from mscl_amd.lib import MsclError
    model, opt = _net(dev)
    _train(model, opt, 2)
    whole = opt.state_dict()
    part, popt = _net(dev)
    _train(part, popt, 1, upto=2)
    own = popt.state_dict()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        popt.step()
    inner = popt._inner
    for state in (whole, _torch_state(part, [1e-3] * len(list(part.parameters())))):
        with pytest.raises(MsclError, match='captured'):
            popt.load_state_dict(state)
        assert popt._inner is inner and not all(s.touched for s in part.arena.slots)
    q = part.arena.Q.clone()
    graph.replay()
    torch.cuda.synchronize()
    want = part.arena.Q.clone()
    popt.load_state_dict(own)
    part.arena.Q.copy_(q)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(part.arena.Q, want) and popt._inner is inner and inner.device_step() == 2


def test_rates_of_a_schedule_with_a_floor():
    """mmcv's schedules start from initial_lr and may end at one min_lr for all groups: their rates then differ by more than the multipliers, but
    the groups agree on where they started, and one without a multiplier tells the rate"""
    from mscl_amd.lib import MsclError
    from mscl_amd.optim import _base_lr
    mult, low, c = [0.1, 1.0, 0.0, 10.0], 1e-5, 0.3

    def groups(start):
        return [dict(params=[i], initial_lr=s, lr=low + (s - low) * c) for i, s in enumerate(start)]
    assert abs(_base_lr(groups([2e-3 * m for m in mult]), mult) / (low + (2e-3 - low) * c) - 1) < 1e-12
    with pytest.raises(MsclError, match='rate'):
        _base_lr(groups([2e-3] * 4), mult)
    half = groups([2e-3 * m for m in mult])
    del half[1]['initial_lr']
    with pytest.raises(MsclError, match='rate'):
        _base_lr(half, mult)
    assert _base_lr([dict(params=[0, 1, 2, 3], lr=3e-4)], [1.0] * 4) == 3e-4
    assert _base_lr([dict(lr=3e-4)], mult) == 3e-4 and _base_lr([{}], mult) is None and _base_lr([dict(params=[2], lr=0.0)], mult) is None
    with pytest.raises(MsclError, match='has not'):
        _base_lr([dict(params=[4], lr=1.0)], mult)
