"""AdamW over many tensors, moments in 32 and in 8 bits (mscl_amd/optim.py, csrc/adamw.hip), against oracle/adamw.py in 64 bits.

Tolerances.  u = 2^-24 is a rounding of fp32.  m = b1 m + (c g) a1 takes roundings of b1, a1, c g, two products and a sum: 6 u of the
larger term's magnitude; with M = |b1 m| + |a1 c g| that is |err| <= 6 u M.  v likewise, 8 u of its (positive) terms.  The update
lr c1 m / (sqrt(v) c2 + eps): m is off by 6 u M, sqrt(v) by 4 u + 1 ulp, the reciprocal by 1 ulp, five more products, so
24 u (M / |m|) relative; p adds lr wd p (2 u of p) and two roundings: |err| <= 4 u |p| + 24 u * update(M)."""
import numpy as np
import pytest
import torch

from oracle import adamw as oracle

U = 2.0 ** -24


# ------------------------------------------------------------------------------------------------------------ CPU
def test_refusals_on_the_host():
    from mscl_amd import optim
    from mscl_amd.lib import MsclError
    a, b = torch.zeros(300), torch.zeros(7)
    buf = torch.zeros(1000)

    def bad(match, params, **kw):
        with pytest.raises((MsclError, NotImplementedError), match=match):
            optim.AdamW(params, **kw)

    bad('no parameters', [])
    bad('32 or 8', [a], state_bits=16)
    bad('betas', [a], betas=(1.0, 0.9))
    bad('betas', [a], betas=(0.9, float('nan')))
    bad('eps', [a], eps=0.0)
    bad('eps', [a], eps=1e-60)
    bad('weight_decay', [a], weight_decay=-1.0)
    bad('L2', [a], grad_clip=dict(max_norm=1.0, norm_type=1))
    bad('max_norm', [a], grad_clip=dict(max_norm=0.0))
    bad('max_norm', [a], grad_clip=dict(max_norm=float('nan')))
    bad('one entry', [a, b], lr_mult=[1.0])
    bad('one entry', [a, b], shadows=[a.bfloat16()])
    bad('fp32 masters', [a.bfloat16()])
    bad('empty', [torch.zeros(0)])
    bad('gaps', [torch.zeros(8, 4)[:, :3]])
    bad('gaps', [torch.zeros(4)[:1].expand(4)])
    bad('share memory', [a, a])
    bad('share memory', [buf[:500], buf[499:]])
    bad('shadows are', [a], shadows=[a.clone()])
    bad('laid out', [a], shadows=[b.bfloat16()])
    bad('laid out', [torch.zeros(3, 4)], shadows=[torch.zeros(4, 3, dtype=torch.bfloat16).t()])
    bad('no CPU fallback', [a, b, buf[:10], buf[10:20], torch.zeros(2, 3, 4, 5, 6).to(memory_format=torch.channels_last_3d)])


def test_gradient_refusals_on_the_host():
    from mscl_amd import optim
    from mscl_amd.lib import MsclError
    p = [torch.zeros(4, 6), torch.zeros(5)]
    good = [torch.zeros(4, 6), torch.zeros(5)]
    optim._check_grads(good, p)
    optim._check_grads([g.half() for g in good], p)
    for grads, match in (([good[0]], 'one gradient'), ([good[0], None], 'no gradient'), ([good[0], good[1].half()], 'type'),
                         ([good[0], torch.zeros(6)], 'shape'), ([torch.zeros(6, 4).t(), good[1]], 'laid out'),
                         ([g.double() for g in good], 'fp32, bf16 or fp16')):
        with pytest.raises(MsclError, match=match):
            optim._check_grads(grads, p)
    # gradients may share memory among themselves, never with what is written
    spans = [(1000, 400, 'parameter 0'), (2000, 100, 'parameter 1')]
    optim._check_grad_memory([1400, 1400, 0, 2100], [600, 600, 1000, 50], spans)
    for ptr, n in ((1399, 4), (999, 2), (900, 2000), (2050, 1), (0, 1001)):
        with pytest.raises(MsclError, match='share memory'):
            optim._check_grad_memory([ptr], [n], spans)


def test_layout_and_multipliers():
    from mscl_amd import optim
    off, first, total, n_chunks, chunks = optim._layout([1, 256, 257, 4096, 4097, 1 << 33])
    assert off.tolist() == [0, 256, 512, 1024, 5120, 9472] and total == 9472 + (1 << 33)
    assert first.tolist() == [0, 1, 2, 3, 4, 6] and n_chunks == 6 + (1 << 21) and chunks.sum() == n_chunks
    ps = [torch.zeros(2) for _ in range(6)]
    named = list(zip(['a.weight', 'a.bias', 'bn.weight', 'bn.bias', 'head.fc.weight', 'head.fc.bias'], ps))
    lr, wd = optim._param_mults(named, {id(ps[2]), id(ps[3])}, dict(bias_lr_mult=2, bias_decay_mult=0.5, norm_decay_mult=0,
                                custom_keys={'head': dict(lr_mult=10), 'head.fc': dict(lr_mult=3, decay_mult=0.25)}))
    assert lr == [1, 2, 1, 1, 3, 3] and wd == [1, 0.5, 0, 0, 0.25, 0.25]
    with pytest.raises(NotImplementedError):
        optim._param_mults(named, set(), dict(dwconv_decay_mult=0))


def test_constants_match_the_header():
    import os
    import re
    from mscl_amd import lib, optim
    header = open(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), 'include', 'mscl_hip.h')).read()
    for name, v in dict(BLOCK=optim.BLOCK, CHUNK=optim.CHUNK, PARTS=optim.PARTS, WORDS=optim.WORDS).items():
        assert int(re.search(rf'#define MSCL_ADAMW_{name}\s+(\d+)', header).group(1)) == v
    assert optim._TENSOR.itemsize == 48 and oracle.BLOCK == optim.BLOCK
    import ctypes
    assert ctypes.sizeof(lib.AdamWDesc) == 6 * 8 + 8 + 4 * 8 + 4 * 8 + 4 * 4
    if lib._lib is None:
        lib.load()
    assert lib.call_raw('mscl_adamw_step', None, None) == -1
    assert lib.call_raw('mscl_adamw_values', None, None, None, None, None, 1, None) == -1


def test_oracle_quantisation_is_unbiased_and_keeps_positive():
    rng = np.random.default_rng(0)
    x = rng.standard_normal(256) * 10.0 ** rng.uniform(-6, 0, 256)
    x[0] = np.abs(x).max() * 1.5
    mean = np.zeros(256)
    N = 2000
    for t in range(N):
        lo, _ = oracle.random_bits(256, 0, 1, t)
        q, a, b = oracle.quantise(x, lo, 4)
        mean += q / N
    spread = np.abs(b - a) / 2 / np.sqrt(N) * 6 + np.abs(b - a) / 65536      # 6 sigma of a two-point variable's mean, 16 random bits
    assert (np.abs(mean - x) <= spread + 1e-30).all()
    v = np.array([1.0] + [2.0 ** -k for k in range(1, 60)])
    q, _, _ = oracle.quantise(v, np.zeros(60), 5)
    assert (q > 0).all()


# ------------------------------------------------------------------------------------------------------------ GPU
def _make(sizes, dev, seed, gtype=torch.float32, skew=0, shadow=None, sigma=0.01):
    gen = torch.Generator().manual_seed(seed)
    ps, gs, ss = [], [], []
    for i, n in enumerate(sizes):
        buf = torch.zeros(n + skew, device=dev)
        p = buf[skew:]
        p.copy_(torch.randn(n, generator=gen) * 0.05)
        g = torch.zeros(n + skew, dtype=gtype, device=dev)[skew:]
        g.copy_(torch.randn(n, generator=gen) * sigma * 4.0 ** (i % 3))
        ps.append(p)
        gs.append(g)
        if shadow is not None:
            ss.append(torch.full((n + skew,), 9.0, dtype=shadow, device=dev)[skew:])
    return ps, gs, (ss if shadow is not None else None)


def _check_p(got, p, m, v, M, t, lr, wd, betas, eps, where):
    rate = lr / (1 - betas[0] ** t)
    upd = rate * M / (np.sqrt(v / (1 - betas[1] ** t)) + eps)
    new = p * (1 - lr * wd) - rate * m / (np.sqrt(v / (1 - betas[1] ** t)) + eps)
    tol = 4 * U * np.maximum(np.abs(p), np.abs(new)) + 24 * U * upd + 1e-38
    err = np.abs(got - new)
    assert (err <= tol).all(), (where, float((err / tol).max()))
    return new


SIZES = [[1], [255, 256, 257], [4095, 4096, 4097, 3, 64, 9001], [300000, 1, 5]]


@pytest.mark.gpu
@pytest.mark.parametrize('gtype', [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize('skew', [0, 1])
@pytest.mark.parametrize('sizes', SIZES, ids=['one', 'blocks', 'chunks', 'long'])
def test_fp32_states(sizes, skew, gtype, dev):
    from mscl_amd import AdamW
    shadow = {torch.float32: torch.bfloat16, torch.bfloat16: torch.float16, torch.float16: None}[gtype]
    clip = {0: dict(max_norm=0.05, norm_type=2), 1: None}[skew]
    ps, gs, ss = _make(sizes, dev, 3, gtype, skew, shadow)
    lrm, wdm = [1.0 + 0.5 * (i % 2) for i in range(len(sizes))], [float(i % 3) for i in range(len(sizes))]
    opt = AdamW(ps, lr=3e-3, betas=(0.8, 0.99), eps=1e-7, weight_decay=0.1, lr_mult=lrm, decay_mult=wdm, grad_clip=clip, shadows=ss)
    guard = [(p._base.clone(), g._base.clone()) for p, g in zip(ps, gs)] if skew else None
    P = [p.cpu().double().numpy() for p in ps]
    M, V = [np.zeros(n) for n in sizes], [np.zeros(n) for n in sizes]
    for t in range(1, 4):
        if t == 2:
            opt.param_groups[0]['lr'] = 1e-3
        lr = float(np.float32(opt.param_groups[0]['lr']))
        for i, g in enumerate(gs):
            g.copy_((torch.randn(sizes[i], generator=torch.Generator().manual_seed(50 * t + i)) * 0.01))
        G = [g.cpu().double().numpy() for g in gs]
        coef, norm = oracle.coefficient(G, 0.05 if clip else 0.0)
        opt.step(gs)
        if clip:
            assert abs(float(opt.grad_norm()) - norm) <= 2 * U * norm
        for i, n in enumerate(sizes):
            # the oracle goes on from the kernel's own states, so that tolerances do not accumulate
            o = opt.offsets[i]
            Mt = np.abs(0.8 * M[i]) + np.abs(0.2 * G[i] * coef)
            _, m, v = oracle.step(P[i], G[i], M[i], V[i], t, coef, lr, (0.8, 0.99), 1e-7)
            got_m, got_v = (s[o:o + n].cpu().double().numpy() for s in (opt.exp_avg, opt.exp_avg_sq))
            assert (np.abs(got_m - m) <= 6 * U * Mt + 1e-44).all()
            assert (np.abs(got_v - v) <= 8 * U * v + 1e-44).all()
            _check_p(ps[i].cpu().double().numpy(), P[i], m, v, Mt, t, lr * lrm[i], 0.1 * wdm[i], (0.8, 0.99), 1e-7, (t, i))
            if ss:
                assert torch.equal(ss[i], ps[i].to(shadow))
            P[i], M[i], V[i] = ps[i].cpu().double().numpy(), got_m, got_v
    for i, n in enumerate(sizes):                # padding of the states stays zero, memory in front of a skewed tensor stays as it was
        o = opt.offsets[i]
        assert not opt.exp_avg[o + n:o + -(-n // 256) * 256].any()
        if skew:
            assert torch.equal(ps[i]._base[:1], guard[i][0][:1])
    assert opt.device_step() == opt.steps == 3


@pytest.mark.gpu
@pytest.mark.parametrize('gtype,skew,clip', [(torch.float32, 0, True), (torch.bfloat16, 0, False), (torch.float16, 1, True)])
@pytest.mark.parametrize('sizes', SIZES, ids=['one', 'blocks', 'chunks', 'long'])
def test_8bit_states(sizes, gtype, skew, clip, dev):
    """p against the formula on the decoded states; the new codes are the oracle's but where the fp32 value (off by 8 u) and the 64-bit
    one fall on different sides of the random threshold: at most 8 u / (2^-4 step) = 2^-17 of them in the mean, and then neighbours."""
    from mscl_amd import AdamW
    ps, gs, ss = _make(sizes, dev, 4, gtype, skew, torch.bfloat16)
    opt = AdamW(ps, lr=1e-3, betas=(0.9, 0.999), weight_decay=0.05, grad_clip=dict(max_norm=0.03) if clip else None, state_bits=8,
                shadows=ss, seed=77)
    lr, N = float(np.float32(1e-3)), opt.numel
    off_m = off_v = 0
    for t in range(1, 5):
        for i, g in enumerate(gs):       # magnitudes spread over many octaves inside a block, zeros among them
            gen = torch.Generator().manual_seed(90 * t + i)
            x = torch.randn(sizes[i], generator=gen) * 10 ** (-3 * torch.rand(sizes[i], generator=gen))
            x[::17] = 0
            g.copy_(x * 0.1)
        codes = [s.cpu().numpy() for s in (opt.exp_avg, opt.exp_avg_sq)]
        ex = opt.exponents.cpu().numpy()
        m0, v0 = oracle.decode(codes[0], ex[0], 4), oracle.decode(codes[1], ex[1], 5)
        P = [p.cpu().double().numpy() for p in ps]
        G = [g.cpu().double().numpy() for g in gs]
        coef, _ = oracle.coefficient(G, 0.03 if clip else 0.0)
        opt.step(gs)
        gm, gv = (s.cpu().double().numpy() for s in opt.state_values())
        ex1 = opt.exponents.cpu().numpy()
        assert np.array_equal(gm, oracle.decode(opt.exp_avg.cpu().numpy(), ex1[0], 4))
        assert np.array_equal(gv, oracle.decode(opt.exp_avg_sq.cpu().numpy(), ex1[1], 5))
        for i, n in enumerate(sizes):
            o = opt.offsets[i]
            M = np.abs(0.9 * m0[o:o + n]) + np.abs(0.1 * G[i] * coef)
            _, m, v = oracle.step(P[i], G[i], m0[o:o + n], v0[o:o + n], t, coef, lr)
            _check_p(ps[i].cpu().double().numpy(), P[i], m, v, M, t, lr, 0.05, (0.9, 0.999), 1e-8, (t, i))
            assert torch.equal(ss[i], ps[i].bfloat16())
            lo, hi = oracle.random_bits(n, o, 77, t)
            for got, want, r, bits in ((gm, m, lo, 4), (gv, v, hi, 5)):
                q, a, b = oracle.quantise(want, r, bits)
                bad = got[o:o + n] != q
                near = np.isin(np.abs(got[o:o + n][bad]), np.concatenate([np.abs(a[bad]), np.abs(b[bad])]))
                assert near.all()
                if bits == 4:
                    off_m += int(bad.sum())
                else:
                    off_v += int(bad.sum())
                    assert ((got[o:o + n] > 0) == (want > 0)).all()
    assert off_m <= 4 + 4 * N * 2.0 ** -16 and off_v <= 4 + 4 * N * 2.0 ** -16, (off_m, off_v)


@pytest.mark.gpu
def test_8bit_second_moment_follows_the_gradient(dev):
    """b2 = 0.999: a step moves v by at most 0.1 %, a 3-bit code by 6 % or more.  With unbiased rounding the mean over 65536 elements
    still follows the formula: after 300 steps of a constant gradient, v / v0 = 0.999^300 + (1 - 0.999^300) g^2 / v0.  The mean's spread:
    300 roundings, each of variance <= 1/4 of a step (12.5 %) squared, over 65536 elements: sqrt(300) * 0.0625 / 256 = 0.4 % (6 sigma: 2.6 %)."""
    from mscl_amd import AdamW
    n = 65536
    p, g = torch.zeros(n, device=dev), torch.full((n,), 2e-3, device=dev)
    opt = AdamW([p], lr=0.0, state_bits=8, weight_decay=0.0)
    g0 = torch.full((n,), 1e-3, device=dev)
    v = 0.0
    for k in range(300):
        opt.step([g0 if k < 150 else g])
        v = 0.999 * v + 0.001 * (1e-6 if k < 150 else 4e-6)
    got = float(opt.state_values()[1].double().mean())
    assert abs(got / v - 1) < 0.026, got / v
    assert not p.any()


@pytest.mark.gpu
def test_non_finite_gradients_and_zero_blocks(dev):
    from mscl_amd import AdamW
    n = 1024
    for bits in (32, 8):
        ps, gs, _ = _make([n, 300], dev, 8)
        gs[0][:] = 0
        gs[1][5] = float('inf')
        gs[0][700] = float('nan')
        before = ps[0].clone()
        opt = AdamW(ps, lr=1e-3, weight_decay=0.0, state_bits=bits)
        opt.step(gs)
        m, v = opt.state_values()
        assert torch.isnan(ps[0][700]) and torch.isnan(ps[1][5])
        keep = torch.ones(n, dtype=torch.bool, device=dev)
        keep[700] = False
        assert torch.equal(ps[0][keep], before[keep])         # a zero gradient with zero moments moves nothing
        assert torch.isfinite(ps[1][6:]).all()
        poisoned = m[512:768] if bits == 8 else m[700:701]    # 8 bits: the block of 256 that holds it
        assert torch.isnan(poisoned).all() and torch.isfinite(m[:512]).all() and not m[768:1024].any()
        with_clip = AdamW(ps[1:], lr=1e-3, grad_clip=dict(max_norm=1.0), state_bits=bits)
        gs[1][5] = float('nan')
        with_clip.step(gs[1:])
        assert torch.isnan(ps[1]).all()                       # the norm is a NaN, as clip_grad_norm_ has it


@pytest.mark.gpu
def test_matches_torch_adamw_and_reads_grad_attributes(dev):
    """20 steps of a small net beside torch.optim.AdamW on the same gradients.  Each side is off by 4 u |p| + 24 u lr M' per step, where
    M' = c1 M / (c2 sqrt(v)) <= sqrt(sum w^2 / w') <= 1.2 for t <= 20 (Cauchy-Schwarz; w, w': the weights of the two moving averages)."""
    from mscl_amd import AdamW
    torch.manual_seed(0)
    net = torch.nn.Sequential(torch.nn.Linear(37, 53), torch.nn.GELU(), torch.nn.Linear(53, 11)).to(dev)
    ref = torch.nn.Sequential(torch.nn.Linear(37, 53), torch.nn.GELU(), torch.nn.Linear(53, 11)).to(dev)
    ref.load_state_dict(net.state_dict())
    opt = AdamW(net.parameters(), lr=1e-3, weight_decay=0.1, grad_clip=dict(max_norm=0.5))
    topt = torch.optim.AdamW(ref.parameters(), lr=1e-3, weight_decay=0.1)
    gen = torch.Generator().manual_seed(1)
    for _ in range(20):
        x, dy = torch.randn(16, 37, generator=gen).to(dev), torch.randn(16, 11, generator=gen).to(dev)
        opt.zero_grad()
        topt.zero_grad()
        ref(x).backward(dy)
        for p, r in zip(net.parameters(), ref.parameters()):
            p.grad = r.grad.clone()                            # another tensor every step: the address table follows
        torch.nn.utils.clip_grad_norm_(ref.parameters(), 0.5)
        opt.step()
        topt.step()
    for p, r in zip(net.parameters(), ref.parameters()):
        assert float((p - r).abs().max()) <= 20 * 2 * U * (4 * float(r.abs().max() + 0.02) + 24 * 1.2e-3)
    with pytest.raises(Exception, match='no gradient'):
        net[0].bias.grad = None
        opt.step()


@pytest.mark.gpu
@pytest.mark.parametrize('bits', [32, 8])
def test_captured_step_replays(bits, dev):
    """graph replays == eager steps bit for bit, with eager work and other gradients of an eager step in between"""
    from mscl_amd import AdamW
    sizes = [5000, 77, 70000]
    runs = []
    for graphed in (False, True):
        ps, gs, ss = _make(sizes, dev, 5, shadow=torch.bfloat16)
        opt = AdamW(ps, lr=1e-2, grad_clip=dict(max_norm=0.1), state_bits=bits, shadows=ss, seed=3)
        opt.step(gs)
        others = [g * 0.5 for g in gs]
        graph = None
        if graphed:
            graph = torch.cuda.CUDAGraph()
            torch.cuda.synchronize()
            with torch.cuda.graph(graph):
                opt.step(gs)
            assert opt.device_step() == 1
        for k in range(4):
            opt.param_groups[0]['lr'] = 1e-2 / (k + 1)
            if graphed:
                opt.sync_lr()
                graph.replay()
            else:
                opt.step(gs)
            torch.cuda.synchronize()
            if k == 1:
                opt.step(others)              # an eager step between replays, with its own gradients' addresses
            for g in gs:
                g.mul_(0.9)
        runs.append([t.clone() for t in ps + ss] + [opt.exp_avg.clone(), opt.exp_avg_sq.clone(), torch.tensor(opt.device_step())])
    assert int(runs[0][-1]) == 6
    for a, b in zip(*runs):
        assert torch.equal(a, b)
    from mscl_amd.lib import MsclError
    ps, gs, _ = _make(sizes, dev, 6)
    opt = AdamW(ps)
    with pytest.raises(MsclError, match='capture'):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            opt.step(gs)                      # no eager step before: the addresses cannot be uploaded inside a capture
    # the same after a captured step; the refused one leaves eager and captured steps as they were
    twin = AdamW([p.clone() for p in ps], state_bits=bits)
    opt = AdamW(ps, state_bits=bits)
    opt.step(gs)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        opt.step(gs)
    others = [g.clone() for g in gs]
    with pytest.raises(MsclError, match='capture'):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            opt.step(others)
    opt.step(gs)
    graph.replay()
    for _ in range(3):
        twin.step(gs)
    assert opt.device_step() == 3 and all(torch.equal(a, b) for a, b in zip(ps, twin.params))


@pytest.mark.gpu
def test_other_stream_state_dict_and_layouts(dev):
    from mscl_amd import AdamW
    from mscl_amd.lib import MsclError
    w = torch.randn(8, 6, 1, 3, 3, device=dev).contiguous(memory_format=torch.channels_last_3d)
    g = torch.randn(8, 6, 1, 3, 3, device=dev).contiguous(memory_format=torch.channels_last_3d)
    twin, gt = w.contiguous().clone(), g.contiguous().clone()
    for bits in (32, 8):
        a, b = AdamW([w], state_bits=bits, seed=1), AdamW([twin], state_bits=bits, seed=1)
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            a.step([g])
        torch.cuda.current_stream().wait_stream(s)
        b.step([gt])
        if bits == 32:
            assert torch.equal(w, twin)       # dense in another dimension order: the same numbers
        with pytest.raises(MsclError):
            a.step([gt])
        c = AdamW([twin.clone()], state_bits=bits)
        c.load_state_dict({k: v.cpu() if torch.is_tensor(v) else v for k, v in b.state_dict().items()})
        c.params[0].copy_(twin)
        b.step([gt])
        c.step([gt])
        assert torch.equal(twin, c.params[0]) and torch.equal(b.exp_avg, c.exp_avg) and c.device_step() == 2
        with pytest.raises(MsclError):
            c.load_state_dict(dict(b.state_dict(), state_bits=40 - bits))
        with pytest.raises(MsclError):
            AdamW([twin[:4].clone()], state_bits=bits).load_state_dict(dict(b.state_dict(), exp_avg=b.exp_avg[:1]))
    p = torch.nn.Parameter(torch.zeros(10, device=dev))
    o = AdamW([p])
    p.data = torch.zeros(10, device=dev)
    with pytest.raises(MsclError, match='moved'):
        o.step([torch.zeros(10, device=dev)])
    with pytest.raises(MsclError, match='share memory'):
        AdamW([twin], lr=1e-3).step([twin])


@pytest.mark.gpu
@pytest.mark.parametrize('bits', [32, 8])
def test_offsets_past_32_bits(bits, dev):
    """one tensor of 2^32 + 1000 elements (34 to 60 GB): its last elements against the formula, and a tensor behind it"""
    from mscl_amd import AdamW
    n, tail = (1 << 32) + 1000, 3000
    p, g = torch.zeros(n, device=dev), torch.zeros(n, dtype=torch.bfloat16, device=dev)
    gen = torch.Generator().manual_seed(2)
    p[-tail:].copy_(torch.randn(tail, generator=gen))
    g[-tail:].copy_(torch.randn(tail, generator=gen) * 0.01)
    p2, g2 = torch.ones(77, device=dev), torch.full((77,), 0.01, dtype=torch.bfloat16, device=dev)
    P, G = p[-tail:].cpu().double().numpy(), g[-tail:].cpu().double().numpy()
    opt = AdamW([p, p2], lr=1e-2, weight_decay=0.1, grad_clip=dict(max_norm=0.05), state_bits=bits, seed=5)
    opt.step([g, g2])
    coef, norm = oracle.coefficient([G, g2.cpu().double().numpy()], 0.05)
    assert coef < 1 and abs(float(opt.grad_norm()) - norm) <= 2 * U * norm
    lr = float(np.float32(1e-2))
    _, m, v = oracle.step(P, G, np.zeros(tail), np.zeros(tail), 1, coef, lr)
    _check_p(p[-tail:].cpu().double().numpy(), P, m, v, np.abs(m), 1, lr, 0.1, (0.9, 0.999), 1e-8, 'tail')
    assert not p[:n - tail].any()
    if bits == 32:
        assert (np.abs(opt.exp_avg[n - tail:n].cpu().double().numpy() - m) <= 6 * U * np.abs(m)).all()
    else:                                   # whole blocks only: from the first block boundary inside the tail
        o = -(-(n - tail) // 256) * 256
        k = o - (n - tail)
        lo, hi = oracle.random_bits(n - o, o, 5, 1)
        for got, want, r, b in ((opt.exp_avg, m[k:], lo, 4), (opt.exp_avg_sq, v[k:], hi, 5)):
            e = opt.exponents[b - 4, o // 256:-(-n // 256)].cpu().numpy()
            q, _, _ = oracle.quantise(want, r, b)
            assert (oracle.decode(got[o:n].cpu().numpy(), e, b) != q).sum() <= 2
    assert opt.offsets == [0, -(-n // 256) * 256] and bool((p2 < 1).all())
