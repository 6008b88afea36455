"""The residual norm from its definition, in 64 bits (test infrastructure), with the magnitudes that a rounding analysis needs: beside each
result stands the same formula with every term's absolute value, i.e. what the results of its additions can be off by, in units of the
relative error of a term.

  y = x + s a(g) (w N(f) + b);   h = w' N'(y) + b'       N: rms / layer over the last dimension, None: identity
gradients for dy, dh as in csrc/res_norm.hip."""
import torch


def _act(g, act):
    # slopes from the exponential: a (1 - a) and 1 - a^2 cancel where a gate saturates
    if act == 'sigmoid':
        e = torch.exp(-g.abs())
        return 1 / (1 + torch.exp(-g)), e / (1 + e) ** 2
    if act == 'tanh':
        e = torch.exp(-2 * g.abs())
        return torch.tanh(g), 4 * e / (1 + e) ** 2
    return g, torch.ones_like(g)


def _norm(v, mag, kind, eps):
    """(normalised v, its magnitude, 1 / deviation)"""
    if kind is None:
        return v, mag, None
    if kind == 'layer':
        v = v - v.mean(1, keepdim=True)
        mag = mag + mag.mean(1, keepdim=True)
    r = 1 / torch.sqrt((v * v).mean(1, keepdim=True) + eps)
    n = v * r
    # the deviation's own error: mean(v dv) r^2 <= mean(|n| mag) r, relative
    return n, mag * r + n.abs() * (1 + (n.abs() * mag).mean(1, keepdim=True) * r), r


def _norm_bwd(d, dmag, n, nmag, r, kind):
    if kind is None:
        return d, dmag
    g = d - n * (d * n).mean(1, keepdim=True)
    m = dmag + n.abs() * (dmag * n.abs() + d.abs() * nmag).mean(1, keepdim=True) + nmag * (d * n).mean(1, keepdim=True).abs()
    if kind == 'layer':
        g = g - d.mean(1, keepdim=True)
        m = m + dmag.mean(1, keepdim=True)
    return g * r, m * r + (g * r).abs()


def run(x, f=None, gate=None, act='sigmoid', scale=None, post=None, w_post=None, b_post=None, pre=None, w_pre=None, b_pre=None, eps=1e-6,
        dy=None, dh=None):
    """{name: (value, magnitude)} of y, h and, with dy / dh, of the gradients; all inputs (rows, C) doubles, gate (gates, C)"""
    one = torch.ones(x.shape[1], dtype=torch.float64)
    zero = torch.zeros_like(one)
    R, C = x.shape
    out = {}
    y, ymag = x, x.abs()
    if f is not None:
        w, b, s = (one if w_post is None else w_post), (zero if b_post is None else b_post), (one if scale is None else scale)
        n, nmag, r = _norm(f, f.abs(), post, eps)
        z, zmag = w * n + b, w.abs() * nmag + b.abs()
        a = slope = torch.ones_like(x)
        if gate is not None:
            a, slope = (t.repeat_interleave(R // gate.shape[0], 0) for t in _act(gate, act))
        y, ymag = x + s * a * z, x.abs() + (s * a).abs() * zmag
        out['y'] = (y, ymag)
    if pre is not None:
        w2, b2 = (one if w_pre is None else w_pre), (zero if b_pre is None else b_pre)
        yh, yhmag, r2 = _norm(y, ymag, pre, eps)
        out['h'] = (w2 * yh + b2, w2.abs() * yhmag + b2.abs())
    if dy is None and dh is None:
        return out
    t, tmag = (torch.zeros_like(x), torch.zeros_like(x)) if dy is None else (dy, dy.abs())
    if dh is not None:
        g, gmag = _norm_bwd(dh * w2, (dh * w2).abs(), yh, yhmag, r2, pre)
        t, tmag = t + g, tmag + gmag
        out['dw_pre'] = ((dh * yh).sum(0), (dh.abs() * yhmag).sum(0))
        out['db_pre'] = (dh.sum(0), dh.abs().sum(0))
    out['dx'] = (t, tmag)
    if f is not None:
        sa = s * a
        out['dscale'] = ((t * a * z).sum(0), (a.abs() * (tmag * z.abs() + t.abs() * zmag)).sum(0))
        out['dw_post'] = ((t * sa * n).sum(0), (sa.abs() * (tmag * n.abs() + t.abs() * nmag)).sum(0))
        out['db_post'] = ((t * sa).sum(0), (sa.abs() * tmag).sum(0))
        if gate is not None:
            G = gate.shape[0]
            out['dgate'] = tuple(v.view(G, R // G, C).sum(1) for v in (slope * s * z * t, slope.abs() * s.abs() * (tmag * z.abs() + t.abs() * zmag)))
        out['df'] = _norm_bwd(t * sa * w, tmag * (sa * w).abs(), n, nmag, r, post)
    return out
