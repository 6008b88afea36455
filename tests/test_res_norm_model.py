"""ResNormHip inside one of the framework's own models: bound by that model's materialize(), trained and saved with it."""
import pytest
import torch


def _model(dev):
    from mscl_amd import build_model
    from mscl_amd.fill import fill_module
    from mscl_amd.nn import ResNormHip
    m = build_model(dict(type='Recognizer3D', backbone=dict(type='torchvision.r3d_18'),
                         cls_head=dict(type='I3DHead', num_classes=5, in_channels=512, spatial_type='none', dropout_ratio=0.0)))
    fill_module(m)
    m.tail = ResNormHip(512, 'rms', 'layer', scale=0.1, bias=True)
    return m.materialize(dev).train()


def _loss(m, imgs, label, gate):
    from mscl_amd import kernels as K
    from mscl_amd.recognizer3d import pool
    K.ZEROS.reset(imgs.device)
    x = m.backbone(K.pack_input(imgs))[-1]
    y, h = m.tail(x, x * 0.5, gate)
    for t in (y, h):
        t.retain_grad()
    feat = pool(h, h.shape[0], h.shape[1] * h.shape[2] * h.shape[3])
    return torch.nn.functional.cross_entropy(m.cls_head(feat), label) + y.float().square().mean(), x, y, h


@pytest.mark.gpu
@pytest.mark.parametrize('bits', [32, 8])
def test_bound_by_materialize_trained_and_resumed(bits, dev):
    """gradients in the arena are those of the plain calls, bit for bit; AdamW steps them with no decay on the norm; the state dict and the
    optimizer's state go into a second model, whose next step is the same bits"""
    from mscl_amd import build_optimizer
    from mscl_amd import kernels as K
    torch.manual_seed(0)
    cfg = dict(type='AdamW', lr=1e-3, weight_decay=0.05, state_bits=bits, paramwise_cfg=dict(norm_decay_mult=0.0))
    imgs, label = torch.randn(2, 3, 8, 32, 32, device=dev), torch.tensor([1, 3], device=dev)
    gate = torch.randn(2, 512, device=dev).bfloat16()
    gate[0, 3], gate[1, 4] = float('-inf'), float('inf')
    m = _model(dev)
    opt = build_optimizer(m, cfg, dict(grad_clip=dict(max_norm=5.0, norm_type=2)))
    names = [n for n, _ in m.tail.named_parameters()]
    assert names == ['scale', 'w_post', 'b_post', 'w_pre', 'b_pre']
    for step in range(2):
        opt.zero_grad()
        loss, x, y, h = _loss(m, imgs, label, gate)
        loss.backward()
        vec = {n: getattr(m.tail, n).detach().clone() for n in names}
        _, _, saved = K.res_norm_fwd(x.detach(), (x * 0.5).detach(), gate=gate, post_norm='rms', pre_norm='layer', save=True, **vec)
        want = K.res_norm_bwd(saved, y.grad, h.grad)
        for n in names:
            slot = getattr(m.tail, n)._mscl_slot
            assert torch.equal(m.arena.view('G', slot), want[n]) and want[n].any() and torch.isfinite(want[n]).all(), n
        opt.step()
        for n in names:
            assert opt._mult[getattr(m.tail, n)._mscl_slot] == (1.0, 0.0) and not torch.equal(getattr(m.tail, n), vec[n])
    twin = _model(dev)
    topt = build_optimizer(twin, cfg, dict(grad_clip=dict(max_norm=5.0, norm_type=2)))
    twin.load_state_dict(m.state_dict())
    topt.load_state_dict({k: v.cpu() if torch.is_tensor(v) else v for k, v in opt.state_dict().items()})
    twin.arena.G.copy_(m.arena.G)
    opt.step()
    topt.step()
    assert torch.equal(m.arena.Q, twin.arena.Q) and topt._inner.device_step() == 3
