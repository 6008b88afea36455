"""Rows of more than eight waves: every lane of the block has to arrive at the same sums, or the lanes that share a channel (the last vector of
a row that is no multiple of 8 wide repeats channels of the one before it) store different bits for it."""
import numpy as np
import pytest
import torch

BF, H, F = torch.bfloat16, torch.float16, torch.float32
VECS = ('scale', 'w_post', 'b_post', 'w_pre', 'b_pre')


def _totals(parts, order):
    """what each of 16 lanes holds after a row's butterfly over `parts`: two steps inside the quads, then one between neighbouring quads --
    'ror' takes the quad before a lane's own, 'mirror' its partner in the half row -- and one between the half rows"""
    v = np.zeros(16, np.float32)
    v[:len(parts)] = parts
    lane = np.arange(16)
    v = v + v[lane ^ 1]
    v = v + v[lane ^ 2]
    v = v + (v[(lane - 4) % 16] if order == 'ror' else v[(lane & 8) | (7 - (lane & 7))])
    return v + v[(lane + 8) % 16]


@pytest.mark.parametrize('waves', [9, 11, 13, 16])
def test_order_of_a_rows_total(waves):
    """the order in which a block adds its waves' sums gives one value in all lanes; a rotation by a quad would not"""
    rng = np.random.default_rng(waves)
    differ = 0
    for _ in range(200):
        parts = rng.random(waves).astype(np.float32) * 512
        assert len(set(_totals(parts, 'mirror').tolist())) == 1
        differ += len(set(_totals(parts, 'ror').tolist())) > 1
    assert differ > 10


def _inputs(rows, C, gates, xt, ft, dev, level):
    """rows that are random up to channel C - level and one value from there on, gates, per-channel vectors and gradients likewise"""
    gen = torch.Generator().manual_seed(C + gates)

    def rnd(*shape, dtype=F):
        t = torch.randn(*shape, generator=gen)
        t[..., C - level:] = t[..., :1]
        return t.to(dtype).to(dev)
    t = dict(x=rnd(rows, C, dtype=xt), f=rnd(rows, C, dtype=ft), gate=rnd(gates, C, dtype=ft) if gates else None,
             dy=rnd(rows, C, dtype=xt), dh=rnd(rows, C, dtype=ft))
    t.update({k: rnd(C) * 0.2 + 1.0 for k in VECS})
    return t


@pytest.mark.gpu
@pytest.mark.parametrize('xt,ft,norm', [(BF, BF, 'rms'), (F, F, 'layer'), (F, H, 'rms')])
@pytest.mark.parametrize('gates', [0, 1, 16, 64])
@pytest.mark.parametrize('C', [4097, 4099, 4131, 5001, 6145, 7005, 8193, 8227, 12001])
def test_equal_channels_get_equal_bits(C, gates, xt, ft, norm, dev):
    """Channels that hold the same values in every row, gate and vector have the same results, bit for bit, whichever lane computes them; and a
    second call repeats the first.  The level stretch spans more than two waves and ends the row."""
    from mscl_amd import kernels as K_
    t = _inputs(64, C, gates, xt, ft, dev, 1300)
    args = dict(gate=t['gate'], post_norm=norm, pre_norm='rms', save=True, **{k: t[k] for k in VECS})
    y, h, saved = K_.res_norm_fwd(t['x'], t['f'], **args)
    out = dict(K_.res_norm_bwd(saved, t['dy'], t['dh']), y=y, h=h)
    for k, v in out.items():
        tail = v[..., C - 1300:]
        assert bool((tail == tail[..., :1]).all()), (k, int((tail != tail[..., :1]).sum()))
    y2, h2, saved2 = K_.res_norm_fwd(t['x'], t['f'], **args)
    again = dict(K_.res_norm_bwd(saved2, t['dy'], t['dh']), y=y2, h=h2)
    assert all(torch.equal(v, again[k]) for k, v in out.items())


@pytest.mark.gpu
@pytest.mark.parametrize('C', [4099, 6145, 8193])
def test_wide_odd_rows_captured(C, dev):
    """replays of a captured forward and backward pass are the eager ones, bit for bit"""
    from mscl_amd import kernels as K_
    t = _inputs(64, C, 64, BF, BF, dev, 1)
    args = dict(gate=t['gate'], post_norm='layer', pre_norm='rms', save=True, **{k: t[k] for k in VECS})
    K_.res_norm_bwd(K_.res_norm_fwd(t['x'], t['f'], **args)[2], t['dy'], t['dh'])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, h, saved = K_.res_norm_fwd(t['x'], t['f'], **args)
        g = K_.res_norm_bwd(saved, t['dy'], t['dh'])
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        y2, h2, s2 = K_.res_norm_fwd(t['x'], t['f'], **args)
        g2 = K_.res_norm_bwd(s2, t['dy'], t['dh'])
        torch.cuda.synchronize()
        assert torch.equal(y, y2) and torch.equal(h, h2) and all(torch.equal(v, g2[k]) for k, v in g.items())
        t['x'].mul_(0.7)


def test_wide_backward_without_a_device():
    """the entry point reports what the runtime says to it before the launch, too (here: that there is no GPU), instead of launching on"""
    import ctypes

    from mscl_amd import lib
    if torch.cuda.is_available():
        pytest.skip('needs a host without a GPU')
    d = lib.ResNormDesc(x=16, f=16, dy=16, dh=16, rstd_f=16, rstd_y=16, ws=16, rows=4, C=8192, ld_x=8192, ld_f=8192, x_type=2, f_type=2, post=1, pre=1,
                        eps=1e-6)
    d.ws_floats = lib.call_raw('mscl_res_norm_ws', ctypes.byref(d))
    assert lib.call_raw('mscl_res_norm_bwd', ctypes.byref(d), None) > 0


@pytest.mark.gpu
def test_wide_backward_from_several_threads(dev):
    """calls from four threads at once, a stream each, the first calls of these forms in the process or not: the results of one thread"""
    import threading

    from mscl_amd import kernels as K_
    C = 8000
    t = _inputs(8, C, 8, F, H, dev, 1)
    _, _, saved = K_.res_norm_fwd(t['x'], t['f'], gate=t['gate'], post_norm='rms', pre_norm='layer', save=True, **{k: t[k] for k in VECS})
    torch.cuda.synchronize()
    got, streams = [None] * 4, [torch.cuda.Stream() for _ in range(4)]

    def work(i):
        with torch.cuda.stream(streams[i]):
            got[i] = K_.res_norm_bwd(saved, t['dy'], t['dh'])
    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for th in threads:
        th.start()
    for th in threads:
        th.join()
    torch.cuda.synchronize()
    want = K_.res_norm_bwd(saved, t['dy'], t['dh'])
    torch.cuda.synchronize()
    assert all(torch.equal(v, g[k]) for g in got for k, v in want.items())
