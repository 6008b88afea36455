"""The residual norm (csrc/res_norm.hip, kernels.res_norm_fwd / _bwd) against oracle/res_norm.py in 64 bits.

Tolerances, with u = 2^-24 (a rounding of fp32): a result is off by one rounding to its type -- half a step: 2^-8, 2^-11 of the value for
bf16, fp16 (1/2 of eps; 2^-24 for fp32) -- plus K u times the magnitude that the oracle gives beside it (the formula with every term
positive).  K counts fp32 roundings on the longest path: a row sum is 16 values in a lane, up to 10 steps in a wave and 16 over the
waves (42), then mean, + eps, square root, division (4): 1 / deviation is good to 46 u / 2 + 4, a normalised value to ~30 u and 4 more for
the mean of a layer norm (42 again): n 80 u;  w, b, scale, act (the kernels' exponential 2 ulp, 1 + e, the 1-ulp reciprocal and a product: 8 u;
tanhf 2 ulp), add: y 95 u;  the second norm on top: yhat 95 + 80, h 180 u;  its backward: product, row sum, 3 more: dx 180 + 50 = 230 u;  the
branch's: 230 + 5 + 50 + 80: df 365 u;  column sums: 230 + 90 per term (90: n and a gate's value or slope), one rounding per row in a thread and one
for each of a block's 256 / T teams of T lanes (the second launch adds in 64 bits): 320 + rows_in_a_thread + 32 for T >= 8.  Up to 32 channels T is
1 .. 4, with up to 256 teams, but a row sum is 8 values and 2 steps: n 20 u, y 35, yhat 60, dx 85, a column's term 125: 125 + rows_in_a_thread + 256.
K = 512 covers all of them while a thread adds up to 128 rows; the tests stay below (at most 6000 rows over teams of 16 .. 1024 lanes, 1024 blocks
or fewer rows)."""
import itertools
import random

import pytest
import torch

from oracle import res_norm as oracle

U, K = 2.0 ** -24, 512
BF, H, F = torch.bfloat16, torch.float16, torch.float32
VECS = ('scale', 'w_post', 'b_post', 'w_pre', 'b_pre')


def _case(seed, rows, C, xt=BF, ft=BF, post='rms', pre='rms', gates=0, act='sigmoid', vecs=VECS, pad=0, f=True, dy=True, dh=True):
    return dict(seed=seed, rows=rows, C=C, xt=xt, ft=ft, post=post if f else None, pre=pre, gates=gates if f else 0, act=act, vecs=vecs, pad=pad,
                f=f, dy=dy, dh=dh and pre is not None)


def _inputs(c):
    gen = torch.Generator().manual_seed(c['seed'])

    def rnd(*s):
        return torch.randn(s, generator=gen)
    R, C = c['rows'], c['C']
    t = dict(x=rnd(R, C).to(c['xt']), f=None, gate=None)
    if c['f']:
        t['f'] = (rnd(R, C) * (0.3 + torch.rand(C, generator=gen)) + 0.3).to(c['ft'])
        if c['gates']:
            t['gate'] = (2 * rnd(c['gates'], C)).to(c['ft'])
    for k in VECS:
        live = k in c['vecs'] and (c['post'] if k.endswith('post') else c['pre'] if k.endswith('pre') else c['f'])
        t[k] = (rnd(C) * 0.2 + (1.0 if k.startswith('w') else 0.3)) if live else None
    t['dy'] = rnd(R, C).to(c['xt']) * 0.5 if c['dy'] else None
    t['dh'] = rnd(R, C).to(c['ft'] if c['f'] else c['xt']) if c['dh'] else None
    return t


def _want(c, t):
    d = {k: (v.double() if v is not None else None) for k, v in t.items()}
    return oracle.run(d['x'], d['f'], d['gate'], c['act'], d['scale'], c['post'], d['w_post'], d['b_post'], c['pre'], d['w_pre'], d['b_pre'], 1e-6,
                      d['dy'], d['dh'])


def _close(got, want, what):
    val, mag = want
    g = got.detach().cpu().double()
    tol = torch.finfo(got.dtype).eps / 2 * val.abs() + K * U * mag
    if got.dtype == H:
        tol = tol + 2.0 ** -25                  # below 2^-14 fp16 has a fixed step of 2^-24
    err = (g - val).abs()
    assert g.shape == val.shape and bool(torch.isfinite(g).all()), what
    worst = float((err / tol.clamp_min(1e-40)).max()) if err.numel() else 0.0
    assert worst <= 1, (what, worst)


def _run(c, dev, **kw):
    from mscl_amd import kernels as K_
    t = _inputs(c)
    g = {}
    for k, v in t.items():
        if v is None:
            g[k] = None
        elif c['pad'] and k in ('x', 'f'):           # rows of a wider tensor
            wide = torch.full((c['rows'], c['C'] + c['pad']), 7.0, dtype=v.dtype, device=dev)
            wide[:, c['pad'] // 2:c['pad'] // 2 + c['C']] = v.to(dev)
            g[k] = wide[:, c['pad'] // 2:c['pad'] // 2 + c['C']]
        else:
            g[k] = v.to(dev)
    y, h, saved = K_.res_norm_fwd(g['x'], g['f'], gate=g['gate'], gate_act=c['act'], post_norm=c['post'], pre_norm=c['pre'], save=True,
                                  **{k: g[k] for k in VECS})
    grads = K_.res_norm_bwd(saved, g['dy'], g['dh'], **kw) if c['dy'] or c['dh'] else {}
    return t, g, y, h, saved, grads


def _check(c, dev):
    t, g, y, h, saved, grads = _run(c, dev)
    want = _want(c, t)
    if c['f']:
        assert y.dtype == c['xt']
        _close(y, want['y'], (c, 'y'))
    if c['pre']:
        _close(h, want['h'], (c, 'h'))
    names = {'x'} | ({'f'} if c['f'] else set()) | ({'gate'} if c['gates'] else set()) | {k for k in VECS if t[k] is not None}
    if c['dy'] or c['dh']:
        assert set(grads) == names, (c, set(grads))
    for k, v in grads.items():
        if 'd' + k in want:
            _close(v, want['d' + k], (c, 'd' + k))
        else:
            assert not v.any(), (c, k)                # no dh: nothing reaches the pre-norm's vectors


# ------------------------------------------------------------------------------------------------------------ CPU
@pytest.mark.parametrize('post,pre,act', list(itertools.product([None, 'rms', 'layer'], [None, 'rms', 'layer'], ['sigmoid', 'tanh', 'linear'])))
def test_oracle_gradients_against_differences(post, pre, act):
    """the formulas of the backward pass against central differences of the forward one, step 1e-6 in 64 bits: 1e-9 of the terms'"""
    c = _case(3, 6, 5, F, F, post, pre, 3, act)
    t = {k: (v.double() if v is not None else None) for k, v in _inputs(c).items()}

    def loss(d):
        o = oracle.run(d['x'], d['f'], d['gate'], act, d['scale'], post, d['w_post'], d['b_post'], pre, d['w_pre'], d['b_pre'])
        return (o['y'][0] * t['dy']).sum() + ((o['h'][0] * t['dh']).sum() if pre else 0)
    want = _want(c, t)
    for k in ('x', 'f', 'gate') + VECS:
        if t[k] is None:
            continue
        num = torch.zeros_like(t[k])
        for i in range(t[k].numel()):
            for sign in (1, -1):
                d = dict(t)
                d[k] = t[k].clone()
                d[k].view(-1)[i] += sign * 1e-6
                num.view(-1)[i] += sign * loss(d) / 2e-6
        assert float((num - want['d' + k][0]).abs().max()) <= 1e-7 * (1 + float(want['d' + k][1].max())), k


def test_refusals_on_the_host():
    from mscl_amd import kernels as K_, lib
    x, v = torch.zeros(6, 8), torch.zeros(8)

    def bad(match, *a, **kw):
        with pytest.raises(lib.MsclError, match=match):
            K_.res_norm_fwd(*a, **kw)
    bad('no channels', torch.zeros(3, 0), pre_norm='rms')
    bad('up to', torch.zeros(2, 16385), pre_norm='rms')
    bad('norms are', x, x, post_norm='batch')
    bad('norms are', x, x, pre_norm='rms', gate_act='relu')
    bad('eps', x, x, pre_norm='rms', eps=0.0)
    bad('eps', x, x, pre_norm='rms', eps=float('nan'))
    bad('without a branch', x)
    bad('without a branch', x, pre_norm='rms', scale=v)
    bad('without a branch', x, pre_norm='rms', gate=x)
    bad('equal for x and f', x, x.double())
    bad('equal for x and f', x.half(), x.bfloat16())
    bad('equal for x and f', x.half(), x)
    bad('does not fit', x, torch.zeros(6, 4))
    bad('fp32 vector', x, x, scale=torch.zeros(7))
    bad('fp32 vector', x, x, scale=v.half())
    bad('fp32 vector', x, x, scale=torch.zeros(16)[::2])
    bad('without its norm', x, x, w_post=v)
    bad('without its norm', x, x, b_pre=v)
    bad('gate is', x, x, gate=torch.zeros(6, 4))
    bad('gate is', x, x, gate=x.half())
    bad('gate is', x, x, gate=torch.zeros(8))
    bad('divide', x, x, gate=torch.zeros(4, 8))
    bad('divide', x, x, gate=torch.zeros(0, 8))
    bad('no CPU fallback', x, x, pre_norm='rms')
    assert lib.load() and lib.call_raw('mscl_res_norm_fwd', None, None) == -1 and lib.call_raw('mscl_res_norm_bwd', None, None) == -1
    import ctypes
    d = lib.ResNormDesc(x=16, f=16, y=16, rows=4, C=8, ld_x=8, ld_f=8, x_type=2, f_type=2, eps=1e-6)
    for field, v, rc in (('C', 16385, -2), ('rows', 1 << 31, -2), ('ld_x', 7, -3), ('ld_f', 7, -3), ('x_type', 3, -2), ('f_type', 0, -2), ('post', 3, -1),
                         ('gate_act', 3, -1), ('eps', 0.0, -1), ('rows', 0, -1), ('y', None, -1), ('pre', 1, -1)):
        e = lib.ResNormDesc.from_buffer_copy(d)
        setattr(e, field, v)
        assert lib.call_raw('mscl_res_norm_fwd', ctypes.byref(e), None) == rc, field
    e = lib.ResNormDesc.from_buffer_copy(d)
    e.gate, e.rows_per_gate = 16, 3
    assert lib.call_raw('mscl_res_norm_fwd', ctypes.byref(e), None) == -2
    d.dy = 16                                                  # a workspace that is too small is refused, not overrun
    n = lib.call_raw('mscl_res_norm_ws', ctypes.byref(d))
    assert n == 4 * 8 * 1
    d.ws, d.ws_floats = 16, n - 1
    assert lib.call_raw('mscl_res_norm_bwd', ctypes.byref(d), None) == -1


def test_rows_of_strided_tensors():
    from mscl_amd import kernels as K_
    base = torch.arange(4 * 5 * 12).float().view(4, 5, 12)
    for t, ld in ((base, 12), (base[..., 2:10], 12), (base[:, 0], 60), (base[:, 0, 3:7], 60), (base[1, 2:3, 4:], 8), (base[..., :1], 12)):
        r, got = K_._rows_of(t, t.shape[-1])
        assert got == ld and r.data_ptr() == t.data_ptr(), (t.shape, got)
    for t in (base[:, 1:4], base[..., ::2], base.transpose(1, 2), base[:1, :1].expand(4, 5, 12)):
        r, got = K_._rows_of(t, t.shape[-1])
        assert got == t.shape[-1] and r.is_contiguous() and torch.equal(r, t)


# ------------------------------------------------------------------------------------------------------------ GPU
WIDTHS = [1, 2, 3, 7, 8, 9, 16, 17, 31, 32, 64, 65, 96, 128, 129, 136, 200, 256, 257, 320, 333, 512, 513, 520, 777, 1000, 1024, 1025, 1032, 2040, 2048,
          2500, 4096, 4099, 8192, 8193, 8200, 10000, 16376, 16383, 16384]


@pytest.mark.gpu
@pytest.mark.parametrize('C', WIDTHS)
def test_every_width(C, dev):
    rows = 41 if C <= 4096 else 5
    _check(_case(C, rows, C, BF, BF, 'rms', 'rms', 0), dev)
    _check(_case(C + 1, rows, C, F, F, 'layer', 'layer', rows, 'tanh'), dev)
    _check(_case(C + 2, 2 * rows, C, H, H, 'layer', 'rms', 2), dev)


def _mixed():
    rng = random.Random(11)
    out = []
    for i in range(60):
        xt, ft = rng.choice([(BF, BF), (H, H), (F, F), (F, BF), (F, H)])
        rows = rng.choice([1, 2, 3, 5, 16, 37, 64, 100, 700])
        C = rng.choice([5, 8, 16, 24, 64, 100, 128, 192, 256, 264, 500, 512, 640, 1024, 1100, 2048])
        gates = rng.choice([0, 0, 1, rows] + [g for g in (2, 4, 5, 10, 20, 50, 350) if rows % g == 0])
        vecs = tuple(v for v in VECS if rng.random() < 0.6)
        f = rng.random() < 0.85
        pre = rng.choice(['rms', 'layer', None]) if f else rng.choice(['rms', 'layer'])
        dh = rng.random() < 0.8
        out.append(_case(100 + i, rows, C, xt, ft if f else xt, rng.choice(['rms', 'layer', None]), pre, gates, rng.choice(['sigmoid', 'tanh', 'linear']),
                         vecs, rng.choice([0, 0, 8, 6]), f, rng.random() < 0.8 or not (dh and pre), dh))
    return out


@pytest.mark.gpu
@pytest.mark.parametrize('i', range(60))
def test_mixed_forms(i, dev):
    _check(_mixed()[i], dev)


@pytest.mark.gpu
@pytest.mark.parametrize('rows,C,gates', [(6000, 64, 8), (6000, 64, 6000), (6000, 32, 375), (6000, 16, 400), (5985, 128, 1), (2048, 256, 128), (4000, 72, 250),
                                          (1500, 1024, 3), (1500, 1032, 100), (600, 2048, 30), (300, 9000, 15), (300, 9000, 150)])
def test_gate_runs(rows, C, gates, dev):
    """long runs of rows per gate (shared by several blocks) and short ones (a team each), on each kind of team"""
    _check(_case(rows + C, rows, C, BF, BF, 'rms', 'rms', gates), dev)
    _check(_case(rows + C, rows, C, F, H, 'layer', 'layer', gates, 'tanh'), dev)


@pytest.mark.gpu
@pytest.mark.parametrize('vecs', [VECS, ('scale', 'w_post', 'w_pre')])
@pytest.mark.parametrize('gates', [0, 2, 150, 300])
@pytest.mark.parametrize('C', [5000, 6144, 6145, 7000, 8191, 9001])
def test_wide_rows(C, gates, vecs, dev):
    """a block of 9 .. 16 waves a row, column sums in registers and in LDS: no gate, long and short runs, a gate for every row"""
    _check(_case(C + gates, 300, C, BF, BF, 'rms', 'layer', gates, 'sigmoid', vecs), dev)
    _check(_case(C + gates + 1, 300, C, F, *((BF, 'layer', 'rms') if C % 2 else (F, 'rms', 'rms')), gates, 'tanh', vecs), dev)


@pytest.mark.gpu
def test_whole_gates_past_8192_channels(dev):
    """so many short runs that a team takes whole gates there too; the 64-bit reference runs on the GPU for its size"""
    c = _case(77, 3680, 8200, BF, BF, 'rms', 'layer', 1840)
    t, g, y, h, saved, grads = _run(c, dev)
    want = _want(c, g)
    for k, v in dict(grads, y=y, h=h).items():
        val, mag = want[k if k in ('y', 'h') else 'd' + k]
        _close(v, (val.cpu(), mag.cpu()), k)


@pytest.mark.gpu
def test_bit_reproducible_accumulating_and_partial(dev):
    from mscl_amd import kernels as K_
    c = _case(5, 3000, 96, BF, BF, 'layer', 'rms', 30)
    t, g, y, h, saved, grads = _run(c, dev)
    again = K_.res_norm_bwd(saved, g['dy'], g['dh'])
    assert all(torch.equal(a, again[k]) for k, a in grads.items())
    into = {k: torch.full((96,), 2.0, device=dev) for k in VECS}
    added = K_.res_norm_bwd(saved, g['dy'], g['dh'], into=into)
    want = _want(c, t)
    for k in VECS:
        assert added[k] is into[k]
        _close(into[k] - 0.0, (want['d' + k][0] + 2, want['d' + k][1] + 2), k)
    some = K_.res_norm_bwd(saved, g['dy'], g['dh'], need=('f', 'w_pre'))
    assert set(some) == {'f', 'w_pre'} and torch.equal(some['f'], grads['f']) and torch.equal(some['w_pre'], grads['w_pre'])
    assert set(K_.res_norm_bwd(saved, g['dy'], need=('x',))) == {'x'}
    for kw, match in ((dict(), 'needs dy or dh'), (dict(dy=g['dy'].half()), 'dy is'), (dict(dh=g['dh'][:2]), 'dh is'),
                      (dict(dy=g['dy'], into={'scale': into['scale']}), 'into')):
        with pytest.raises(Exception, match=match):
            K_.res_norm_bwd(saved, **kw)


@pytest.mark.gpu
def test_maps_empty_rows_and_strides(dev):
    """an NDHWC map with a gate per clip; no rows at all; a permuted input; zero and constant rows"""
    from mscl_amd import kernels as K_
    x = torch.randn(2, 3, 4, 5, 16, device=dev).bfloat16()
    f = torch.randn(2, 3, 4, 16, 5, device=dev).bfloat16().transpose(3, 4)
    gate = torch.randn(2, 16, device=dev).bfloat16()
    y, h, s = K_.res_norm_fwd(x, f, gate=gate, pre_norm='rms', post_norm='layer', save=True)
    y2, h2, s2 = K_.res_norm_fwd(x.view(-1, 16), f.contiguous().view(-1, 16), gate=gate, pre_norm='rms', post_norm='layer', save=True)
    assert y.shape == x.shape and torch.equal(y.view(-1, 16), y2) and torch.equal(h.view(-1, 16), h2)
    a, b = K_.res_norm_bwd(s, x, f), K_.res_norm_bwd(s2, x.view(-1, 16), f.contiguous().view(-1, 16))
    assert a['x'].shape == x.shape and a['gate'].shape == gate.shape and all(torch.equal(a[k].reshape(-1), b[k].reshape(-1)) for k in a)
    e = torch.zeros(0, 16, device=dev)
    w = torch.ones(16, device=dev)
    y, h, s = K_.res_norm_fwd(e, e, gate=e, scale=w, pre_norm='rms', w_pre=w, save=True)
    g = K_.res_norm_bwd(s, e, e)
    assert y.shape == h.shape == g['x'].shape == g['gate'].shape == (0, 16) and not g['scale'].any() and not g['w_pre'].any()
    z = torch.zeros(3, 40, device=dev)
    z[1] = 3.0
    y, h, s = K_.res_norm_fwd(z, z, post_norm='layer', pre_norm='layer', save=True)
    assert torch.equal(y, z) and not h.any()                       # a constant row has no deviation: eps alone
    g = K_.res_norm_bwd(s, z, torch.ones_like(z))
    assert torch.isfinite(g['f']).all() and torch.isfinite(g['x']).all()


@pytest.mark.gpu
def test_non_finite_rows_stay_apart(dev):
    from mscl_amd import kernels as K_
    for C in (64, 1024, 4096):
        x = torch.randn(9, C, device=dev)
        f = torch.randn(9, C, device=dev)
        f[3, 1], f[5, 0], x[7, 2] = float('nan'), float('inf'), float('-inf')
        y, h, _ = K_.res_norm_fwd(x, f, post_norm='rms', pre_norm='rms')
        bad = ~torch.isfinite(h).all(1)
        assert bad.tolist() == [i in (3, 5, 7) for i in range(9)]
        x2, f2 = x.clone(), f.clone()
        x2[7], f2[3], f2[5] = 0, 0, 0
        y2, h2, _ = K_.res_norm_fwd(x2, f2, post_norm='rms', pre_norm='rms')
        assert torch.equal(h[~bad], h2[~bad])


@pytest.mark.gpu
def test_offsets_past_32_bits(dev):
    """a map of 2^31 + elements: the last rows, against the same rows alone"""
    from mscl_amd import kernels as K_
    rows, C = (1 << 25) + 17, 64
    f = torch.empty(rows, C, dtype=BF, device=dev)
    f.normal_()
    x = f
    y, h, s = K_.res_norm_fwd(x, f, post_norm='rms', pre_norm='layer', save=True)
    y2, h2, s2 = K_.res_norm_fwd(x[-40:], f[-40:], post_norm='rms', pre_norm='layer', save=True)
    assert torch.equal(y[-40:], y2) and torch.equal(h[-40:], h2)
    g = K_.res_norm_bwd(s, f, f, need=('x', 'f'))
    g2 = K_.res_norm_bwd(s2, f[-40:], f[-40:], need=('x', 'f'))
    assert torch.equal(g['x'][-40:], g2['x']) and torch.equal(g['f'][-40:], g2['f'])


@pytest.mark.gpu
def test_one_gate_for_over_a_billion_rows(dev):
    from mscl_amd import kernels as K_
    rows = (1 << 30) + 40
    x = torch.ones(rows, 1, dtype=BF, device=dev)
    gate = torch.full((1, 1), 0.5, dtype=BF, device=dev)
    x[-40:] = torch.arange(40, dtype=BF, device=dev)[:, None]
    y, _, s = K_.res_norm_fwd(x, x, gate=gate, save=True)
    a = torch.sigmoid(torch.tensor(0.5))
    want = (x[-45:].float() * (1 + float(a))).bfloat16()
    assert float((y[-45:].float() - want.float()).abs().max()) <= 2.0 ** -7 * 64          # one step of the largest value, 39 a
    g = K_.res_norm_bwd(s, x)
    assert float((g['x'][-45:].float() - x[-45:].float()).abs().max()) == 0
    total = float(a * (1 - a)) * (float(rows - 40) + sum(i * i for i in range(40)))
    assert abs(float(g['gate']) / total - 1) <= 2.0 ** -8 + 1e-3                          # bf16, and fp32 sums over 2^30 ones


@pytest.mark.gpu
def test_captured_and_on_another_stream(dev):
    from mscl_amd import kernels as K_
    c = _case(9, 500, 128, BF, BF, 'rms', 'rms', 10)
    _, g, y, h, _, grads = _run(c, dev)
    args = dict(gate=g['gate'], post_norm='rms', pre_norm='rms', save=True, **{k: g[k] for k in VECS})
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y1, h1, s1 = K_.res_norm_fwd(g['x'], g['f'], **args)
        g1 = K_.res_norm_bwd(s1, g['dy'], g['dh'])
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(y, y1) and torch.equal(h, h1) and all(torch.equal(grads[k], g1[k]) for k in grads)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y2, h2, s2 = K_.res_norm_fwd(g['x'], g['f'], **args)
        g2 = K_.res_norm_bwd(s2, g['dy'], g['dh'])
    for k in range(3):
        graph.replay()
        torch.cuda.synchronize()
        yk, hk, sk = K_.res_norm_fwd(g['x'], g['f'], **args)
        gk = K_.res_norm_bwd(sk, g['dy'], g['dh'])
        torch.cuda.synchronize()
        assert torch.equal(yk, y2) and torch.equal(hk, h2) and all(torch.equal(gk[n], g2[n]) for n in gk)
        g['x'].mul_(0.7)
        g['f'].add_(0.1)
