"""grad-clip + SGD-momentum over the flat arena.  ref: mmcv OptimizerHook.after_train_iter wired at
mmaction/apis/train.py:111-119 with optimizer / optimizer_config of mscl_r18_cosm_lr2e-2.py:114-119:
clip_grad_norm_(params with grad, max_norm=40, L2) then torch.optim.SGD(lr, momentum 0.9, wd 1e-4).
Three kernels per step (sum of squares, fused clip+decay+momentum+update+bf16 shadow per active range,
kernel re-layout for the input-gradient GEMM) instead of ~600 tiny ones.

AdamW (`optimizer=dict(type='AdamW', ...)`, which the reference's build_optimizer hands to torch.optim.AdamW): `AdamW` steps any list of
GPU tensors in two or three launches, with moments in 32 or in 8 bits; `ClipAdamW` is the same over a model's arena, beside `ClipSGD`.
`build_optimizer` picks by the config's `type`."""
import ctypes
import math

import numpy as np
import torch

from . import kernels as K
from . import lib
from . import parallel
from .arena import _physical_view
from .lib import AdamWDesc, MsclError
from .nn import BatchNorm3dHip
from .staging import StagingRing


def cosine_lr(base_lr, epoch, max_epochs, min_lr=0.0):
    """mmcv CosineAnnealingLrUpdaterHook by epoch (lr_config at mscl_r18_cosm_lr2e-2.py:123; the config has
    no `warmup=` key, so mmcv applies no warm-up -- SURVEY.md §5)."""
    return min_lr + 0.5 * (base_lr - min_lr) * (1 + math.cos(math.pi * epoch / max_epochs))


class ClipSGD:
    def __init__(self, model, lr=0.02, momentum=0.9, weight_decay=1e-4, grad_clip=dict(max_norm=40, norm_type=2)):
        if grad_clip is not None and grad_clip.get('norm_type', 2) != 2:
            raise NotImplementedError('only the L2 norm is used (optimizer_config.grad_clip.norm_type=2)')
        self.model, self.arena = model, model.arena
        self.lr, self.momentum, self.wd = lr, momentum, weight_decay
        self.max_norm = float(grad_clip['max_norm']) if grad_clip else 0.0
        self.steps = 0
        self._ranges = None
        self._sumsq = torch.zeros(1, dtype=torch.float32, device=self.arena.device)
        self.param_groups = [dict(lr=lr, momentum=momentum, weight_decay=weight_decay)]
        # lr is read from a device word, so a captured graph sees schedule changes; the word is fed through a ring of
        # pinned slots (staging.py) so that the host, which runs steps ahead of the GPU, never rewrites a word in flight
        self._lr = StagingRing((1,), torch.float32, self.arena.device)
        self._lr_cpu = torch.full((1,), float(lr), dtype=torch.float32)
        self._lr.push(self._lr_cpu)

    @classmethod
    def from_cfg(cls, model, optimizer, optimizer_config=None):
        o = dict(optimizer)
        if o.pop('type', 'SGD') != 'SGD':
            raise NotImplementedError('ClipSGD is built from type=SGD (build_optimizer takes SGD and AdamW)')
        clip = (optimizer_config or {}).get('grad_clip')
        return cls(model, grad_clip=clip, **o)

    def zero_grad(self):
        self.model.sync_streams()
        self.arena.G.zero_()

    def grad_norm(self):
        """device scalar: L2 norm of the (all-reduced) gradient before clipping"""
        return self._sumsq.sqrt()

    @torch.no_grad()
    def step(self):
        ar = self.arena
        self.model.sync_streams()
        if getattr(self.model, 'reducer', None) is not None:
            self.model.reducer.finish()         # buckets were launched from backward; wait for them
        else:
            parallel.allreduce_mean_(ar.G)
        ranges = ar.active_ranges()
        if self._ranges is None:
            self._ranges = ranges
        elif ranges != self._ranges:
            raise RuntimeError('the set of parameters receiving gradients changed between steps')
        self._sumsq.zero_()
        K.sumsq(ar.G, self._sumsq)
        if not torch.cuda.is_current_stream_capturing():        # a captured step publishes before each replay (graph.py)
            self.sync_lr()
        for a, b in ranges:     # momentum buffers start at zero: buf = mom*0 + d == torch's first-step buf = d
            K.sgd_step_dev(ar.Q[a:b], ar.G[a:b], ar.MOM[a:b], ar.Qb[a:b], self._sumsq, self.max_norm, self._lr.dev,
                           self.momentum, self.wd)
        self.model.refresh_after_optimizer()
        self.steps += 1

    def sync_lr(self):
        """publish param_groups[0]['lr'] to the device word the SGD kernel reads, in stream order (eager steps: from
        step(); captured steps: before each graph replay).  Unchanged values are not re-sent."""
        lr = float(self.param_groups[0]['lr'])
        if self._lr.pushes and float(self._lr_cpu[0]) == torch.tensor(lr, dtype=torch.float32).item():
            return
        self._lr_cpu[0] = lr
        self._lr.push(self._lr_cpu)

    @property
    def _lr_dev(self):
        return self._lr.dev


BLOCK, CHUNK, PARTS, WORDS = 256, 4096, 2048, 32        # = MSCL_ADAMW_* (include/mscl_hip.h)
_TYPES = {torch.float32: 1, torch.bfloat16: 2, torch.float16: 3}        # = MSCL_F32 / BF16 / F16
_TENSOR = np.dtype([('p', '<u8'), ('shadow', '<u8'), ('n', '<i8'), ('off', '<i8'), ('lr_mult', '<f4'), ('decay', '<f4'),
                    ('first_chunk', '<i4'), ('pad', '<i4')])             # = mscl_adamw_tensor


def _dense(t):
    """whether the tensor's elements fill one stretch of memory without gaps or overlap (in any dimension order)"""
    if t.is_contiguous():
        return True
    want = 1
    for stride, size in sorted((st, sz) for st, sz in zip(t.stride(), t.shape) if sz != 1):
        if stride != want:
            return False
        want *= size
    return True


def _layout(sizes):
    """(state offset, first chunk) of each tensor, elements of the state buffers, number of chunks"""
    n = np.asarray(sizes, dtype=np.int64)
    padded, chunks = -(-n // BLOCK) * BLOCK, -(-n // CHUNK)
    off, first = np.concatenate([[0], np.cumsum(padded)]), np.concatenate([[0], np.cumsum(chunks)])
    return off[:-1], first[:-1], int(off[-1]), int(first[-1]), chunks


def _check_disjoint(spans):
    """spans: [(first byte, bytes, name)] of memory a step writes; the kernel runs them all at once"""
    spans = sorted(spans)
    for (a, n, what), (b, _, other) in zip(spans, spans[1:]):
        if a + n > b:
            raise MsclError(f'AdamW: {what} and {other} share memory')


def _check_params(params, shadows):
    """refuses what a step over these tensors cannot do; returns the memory that it writes"""
    if not params:
        raise MsclError('AdamW: no parameters')
    spans = []
    for i, p in enumerate(params):
        if p.device != params[0].device:
            raise MsclError('AdamW: parameters live on one device')
        if p.dtype != torch.float32:
            raise MsclError(f'AdamW: parameter {i} is {p.dtype}: pass fp32 masters, and 16-bit copies as shadows')
        if p.numel() == 0 or not _dense(p):
            raise MsclError(f'AdamW: parameter {i} is empty or has gaps between its elements')
        spans.append((p.data_ptr(), 4 * p.numel(), f'parameter {i}'))
    for i, (s, p) in enumerate(zip(shadows or (), params)):
        if s.dtype != shadows[0].dtype or s.dtype not in (torch.bfloat16, torch.float16) or s.device != p.device:
            raise MsclError("AdamW: shadows are all bf16 or all fp16, on the parameters' device")
        if s.shape != p.shape or s.stride() != p.stride():
            raise MsclError(f'AdamW: shadow {i} is not laid out like its parameter')
        spans.append((s.data_ptr(), 2 * s.numel(), f'shadow {i}'))
    _check_disjoint(spans)
    return sorted(spans)


def _check_grads(grads, params):
    """refuses gradients that do not fit the parameters one by one"""
    if len(grads) != len(params):
        raise MsclError('AdamW: one gradient per parameter')
    for i, (g, p) in enumerate(zip(grads, params)):
        if g is None:
            raise MsclError(f'AdamW: parameter {i} has no gradient')
        if g.dtype != grads[0].dtype or g.device != p.device or g.shape != p.shape:
            raise MsclError(f"AdamW: gradient {i} has another type, device or shape than its parameter's")
        if g.stride() != p.stride() and not (g.is_contiguous() and p.is_contiguous()):
            raise MsclError(f'AdamW: gradient {i} is not laid out like its parameter')
    if grads[0].dtype not in _TYPES:
        raise MsclError(f'AdamW: gradients are fp32, bf16 or fp16, not {grads[0].dtype}')


def _check_grad_memory(ptrs, nbytes, spans):
    """a gradient may share memory with another one, never with what the step writes (spans: sorted, disjoint, so only the last one that
    starts below a gradient's end can reach into it)"""
    at, end = np.asarray([a for a, _, _ in spans]), np.asarray([a + n for a, n, _ in spans])
    a = np.asarray(ptrs)
    j = np.searchsorted(at, a + np.asarray(nbytes)) - 1
    hit = np.nonzero((j >= 0) & (end[np.maximum(j, 0)] > a))[0]
    if len(hit):
        raise MsclError(f'AdamW: gradient {hit[0]} and {spans[j[hit[0]]][2]} share memory')


def _check_args(lr, betas, eps, weight_decay, grad_clip, state_bits, seed=0):
    if state_bits not in (32, 8):
        raise MsclError(f'AdamW: state_bits is 32 or 8, not {state_bits}')
    if not (0 <= betas[0] < 1 and 0 <= betas[1] < 1 and np.float32(eps) >= np.finfo(np.float32).tiny and lr >= 0 and weight_decay >= 0):
        raise MsclError('AdamW: needs 0 <= betas < 1, eps of at least 2^-126 (the least normal fp32 number), lr >= 0, weight_decay >= 0')
    if grad_clip is not None and grad_clip.get('norm_type', 2) != 2:
        raise NotImplementedError('only the L2 norm is used (optimizer_config.grad_clip.norm_type=2)')
    if grad_clip is not None and not grad_clip['max_norm'] > 0:
        raise MsclError('AdamW: grad_clip needs max_norm > 0 (None: no clip)')


def _check_state(state, state_bits, sizes):
    """refuses a state that does not belong to tensors of these sizes"""
    if state['state_bits'] != state_bits:
        raise MsclError(f"AdamW: a state of {state['state_bits']} bits does not fit state_bits={state_bits}")
    if state['step'] < 0:
        raise MsclError('AdamW: a negative step')
    total = _layout(sizes)[2]
    want = dict(exp_avg=(total,), exp_avg_sq=(total,))
    if state_bits == 8:
        want['exponents'] = (2, total // BLOCK)
    if (list(state.get('sizes', sizes)) != list(sizes) or          # (states written without them are told by the total alone)
            any(tuple(state[k].shape) != shape or state[k].dtype != (torch.float32 if state_bits == 32 else torch.uint8) for k, shape in want.items())):
        raise MsclError('AdamW: the state belongs to other parameters')


_raise_version = getattr(torch._C, '_increment_version', None) or torch.autograd.graph.increment_version          # (raw: 4 / 62 tensors 0.6 / 4.0 us, not 1.2 / 5.6)


class AdamW:
    """AdamW with decoupled decay over a list of fp32 GPU tensors, two or three launches per step whatever their number.

    params       fp32 tensors (masters), dense in any dimension order, on one device; no two may share memory
    lr_mult, decay_mult   a factor per tensor on lr / weight_decay (None: 1)
    grad_clip    dict(max_norm=, norm_type=2): clip by the 2-norm over all tensors, as clip_grad_norm_; None: no clip
    state_bits   32: two fp32 moments (8 bytes per element); 8: block-wise 8-bit moments (2 bytes), rounded without bias by a hash of
                 (seed, step, element) -- formats in include/mscl_hip.h
    shadows      bf16 or fp16 tensors (one type), one per parameter, that receive the rounded parameters

    `step(grads)` takes one gradient per parameter -- fp32, bf16 or fp16, one type for all, laid out like the parameter -- or reads
    `p.grad`; a parameter whose gradient is None is refused (build the optimizer over the parameters that train).  lr is
    `param_groups[0]['lr']`, read from a device word: set it between steps, and call sync_lr() before replaying a captured step (betas, eps >=
    2^-126 and weight_decay are fixed: a change of them is refused).  The
    step counter lives on the device, so a captured step counts its replays; capture a step only after an eager one with the same
    gradient tensors (their addresses are uploaded by the eager one)."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.01, lr_mult=None, decay_mult=None, grad_clip=None,
                 state_bits=32, shadows=None, seed=0):
        self._leaves = list(params)
        self.params = [p.detach() for p in self._leaves]
        self.shadows = None if shadows is None else list(shadows)
        _check_args(lr, betas, eps, weight_decay, grad_clip, state_bits)
        n = len(self.params)
        lr_mult, decay_mult = ([1.0] * n if m is None else [float(v) for v in m] for m in (lr_mult, decay_mult))
        if len(lr_mult) != n or len(decay_mult) != n or (self.shadows is not None and len(self.shadows) != n):
            raise MsclError('AdamW: lr_mult, decay_mult and shadows have one entry per parameter')
        self._spans = _check_params(self.params, self.shadows)
        self.device = self.params[0].device
        if not self.params[0].is_cuda:
            raise MsclError('mscl_amd kernels run on the GPU only (got a CPU tensor); there is no CPU fallback')
        self._param_ptrs = [p.data_ptr() for p in self.params]
        self._shapes, self._strides = [p.shape for p in self.params], [p.stride() for p in self.params]
        self.betas, self.eps, self.wd, self.state_bits, self.seed = (float(betas[0]), float(betas[1])), float(eps), float(weight_decay), state_bits, int(seed)
        self.max_norm = float(grad_clip['max_norm']) if grad_clip else 0.0
        self.param_groups = [dict(lr=lr, betas=self.betas, eps=self.eps, weight_decay=self.wd)]
        self.steps = 0
        sizes = [p.numel() for p in self.params]
        off, first, total, n_chunks, chunks = _layout(sizes)
        if n_chunks >= 1 << 31:
            raise MsclError('AdamW: too many elements for one step')
        self.sizes, self.offsets, self.numel = sizes, off.tolist(), total
        with torch.cuda.device(self.device):
            table = np.zeros(n, dtype=_TENSOR)
            table['p'] = [p.data_ptr() for p in self.params]
            table['shadow'] = [s.data_ptr() for s in self.shadows] if self.shadows else 0
            table['n'], table['off'], table['first_chunk'] = sizes, off, first
            table['lr_mult'], table['decay'] = lr_mult, [self.wd * m for m in decay_mult]
            self._table = torch.from_numpy(table.view(np.uint8).copy()).to(self.device)
            self._chunk_tensor = torch.from_numpy(np.repeat(np.arange(n, dtype=np.int32), chunks)).to(self.device)
            kind = torch.float32 if state_bits == 32 else torch.uint8
            self.exp_avg = torch.zeros(total, dtype=kind, device=self.device)
            self.exp_avg_sq = torch.zeros(total, dtype=kind, device=self.device)
            self.exponents = None
            if state_bits == 8:        # 1: the smallest exponent, a block of zeros
                self.exponents = torch.ones((2, total // BLOCK), dtype=torch.uint8, device=self.device)
            self._words = torch.zeros(WORDS // 4, dtype=torch.int32, device=self.device)
            self._set_seed(self.seed)
            self._partials = torch.zeros(PARTS, dtype=torch.float64, device=self.device)
            self._norm = torch.zeros(1, dtype=torch.float32, device=self.device)
            self._lr = StagingRing((1,), torch.float32, self.device)
            self._lr_cpu = torch.full((1,), float(lr), dtype=torch.float32)
            self._lr.push(self._lr_cpu)
            self._lr_sent = float(lr)
            self._grad_ring = StagingRing((n,), torch.int64, self.device)
        self._grad_ptrs, self._in_graph, self._kept = None, False, []
        self._written = [t for t in self._leaves + (self.shadows or []) if not t.is_inference()]
        P = lib.ptr
        self._desc = AdamWDesc(P(self._table), P(self._grad_ring.dev), P(self._chunk_tensor), P(self.exp_avg), P(self.exp_avg_sq),
                               P(self.exponents), total // BLOCK, P(self._words), P(self._partials), P(self._norm), P(self._lr.dev),
                               self.betas[0], self.betas[1], self.eps, self.max_norm, n_chunks, state_bits, 0,
                               _TYPES[self.shadows[0].dtype] if self.shadows else 0)

    def zero_grad(self):
        for p in self._leaves:
            p.grad = None

    def grad_norm(self):
        """device scalar: L2 norm of the gradients of the last step before clipping (kept only with grad_clip)"""
        return self._norm[0]

    def _set_grads(self, grads):
        T = torch.Tensor
        if list(map(T.data_ptr, self._leaves)) != self._param_ptrs:
            raise MsclError('AdamW: a parameter has moved to other memory since the optimizer was built')
        grads = [p.grad for p in self._leaves] if grads is None else list(grads)
        try:            # all at once for many tensors (hundreds of them cost more host time than a small step takes)
            alike = ([g.shape for g in grads] == self._shapes and list(map(T.stride, grads)) == self._strides and
                     len({g.dtype for g in grads}) == 1 and grads[0].dtype in _TYPES and set(map(T.get_device, grads)) == {self.device.index})
        except (AttributeError, TypeError):
            alike = False
        if not alike:   # one by one: names what does not fit, or finds that it does
            _check_grads(grads, self.params)
        ptrs, kind = list(map(T.data_ptr, grads)), _TYPES[grads[0].dtype]
        moved = ptrs != self._grad_ptrs
        if moved and torch.cuda.is_current_stream_capturing():
            raise MsclError('AdamW: a step is captured with the gradient tensors of the eager step before it (a capture cannot upload other addresses)')
        if moved or kind != self._desc.grad_type:
            _check_grad_memory(ptrs, [g.numel() * g.element_size() for g in grads], self._spans)
        if moved:
            if self._in_graph:                  # a captured step reads the old table: leave it as it is, with its gradients' addresses
                self._kept.append(self._grad_ring)
                self._grad_ring, self._in_graph = StagingRing((len(ptrs),), torch.int64, self.device), False
                self._desc.grads = lib.ptr(self._grad_ring.dev)
            self._grad_ring.push(torch.tensor(ptrs, dtype=torch.int64))
            self._grad_ptrs = ptrs
        self._desc.grad_type = kind

    def step(self, grads=None):
        if torch.cuda.current_device() != self.device.index:
            with torch.cuda.device(self.device):
                return self.step(grads)
        self._set_grads(grads)
        self._launch()
        _raise_version(self._written)          # a backward pass over a graph from before the step is refused

    def _check_groups(self):
        g = self.param_groups[0]
        if (len(self.param_groups) > 1 or g.get('weight_decay', self.wd) != self.wd or g.get('eps', self.eps) != self.eps
                or tuple(g.get('betas', self.betas)) != self.betas):
            raise MsclError('AdamW: betas, eps and weight_decay are fixed when the optimizer is built, of param_groups[0] lr alone is read')

    def _launch(self):
        capturing = torch.cuda.is_current_stream_capturing()
        if capturing:
            self._check_groups()
            self._in_graph = True
        else:                                               # a captured step publishes before each replay
            self.sync_lr()
        lib.call('mscl_adamw_step', ctypes.byref(self._desc), lib.stream_ptr())
        self.steps += not capturing

    def sync_lr(self):
        """publish param_groups[0]['lr'] to the device word the kernel reads, in stream order.  Unchanged values are not re-sent."""
        self._check_groups()
        lr = float(self.param_groups[0]['lr'])
        if lr == self._lr_sent:
            return
        if torch.cuda.current_device() != self.device.index:
            with torch.cuda.device(self.device):
                return self.sync_lr()
        self._lr_cpu[0] = lr
        self._lr.push(self._lr_cpu)
        self._lr_sent = lr

    def state_values(self):
        """(exp_avg, exp_avg_sq) as numbers, flat: the fp32 states themselves, or what the 8-bit codes stand for, in bf16 (exact)"""
        if self.state_bits == 32:
            return self.exp_avg, self.exp_avg_sq
        if torch.cuda.current_device() != self.device.index:
            with torch.cuda.device(self.device):
                return self.state_values()
        m, v = torch.empty((2, self.numel), dtype=torch.bfloat16, device=self.device).unbind(0)
        lib.call('mscl_adamw_values', self.exp_avg.data_ptr(), self.exp_avg_sq.data_ptr(), self.exponents.data_ptr(), m.data_ptr(), v.data_ptr(),
                 self.numel // BLOCK, lib.stream_ptr())
        return m, v

    def device_step(self):
        """the step counter on the device (counts the replays of a captured step too); synchronises"""
        return int(self._words[:2].cpu().view(torch.int64))

    def set_step(self, step):
        self._words[:2].copy_(torch.tensor([int(step)], dtype=torch.int64).view(torch.int32))
        self.steps = int(step)

    def _set_seed(self, seed):
        self.seed = int(seed)
        self._words[5] = ((self.seed & 0xFFFFFFFF) ^ 0x80000000) - 0x80000000          # 32 bits of the seed as an int32

    def reset(self, seed):
        """as before the first step, in the same memory"""
        self.exp_avg.zero_()
        self.exp_avg_sq.zero_()
        if self.exponents is not None:
            self.exponents.fill_(1)                        # the smallest exponent, a block of zeros
        self._set_seed(seed)
        self.set_step(0)

    def state_dict(self):
        """flat states (tensor i at self.offsets[i], sizes[i] elements), on the device; synchronises for the step counter"""
        out = dict(step=self.device_step(), state_bits=self.state_bits, lr=self.param_groups[0]['lr'], seed=self.seed, sizes=list(self.sizes),
                   exp_avg=self.exp_avg.clone(), exp_avg_sq=self.exp_avg_sq.clone())
        if self.state_bits == 8:
            out['exponents'] = self.exponents.clone()
        return out

    def load_state_dict(self, state):
        _check_state(state, self.state_bits, self.sizes)
        pairs = [(self.exp_avg, state['exp_avg']), (self.exp_avg_sq, state['exp_avg_sq'])]
        if self.state_bits == 8:
            pairs.append((self.exponents, state['exponents']))
        for dst, src in pairs:
            dst.copy_(src)
        self.set_step(state['step'])
        if 'seed' in state:
            self._set_seed(state['seed'])
        if 'lr' in state:
            self.param_groups[0]['lr'] = state['lr']


def _param_mults(named_params, norm_params, cfg):
    """(lr_mult, decay_mult) per parameter from mmcv's `paramwise_cfg` (DefaultOptimizerConstructor): custom_keys first -- the longest
    matching key, ties by alphabet -- else the bias / norm multipliers"""
    cfg = dict(cfg or {})
    custom = dict(cfg.pop('custom_keys', {}))
    bias_lr, bias_decay, norm_decay = (float(cfg.pop(k, 1.0)) for k in ('bias_lr_mult', 'bias_decay_mult', 'norm_decay_mult'))
    if cfg:
        raise NotImplementedError(f'paramwise_cfg: {sorted(cfg)} is not supported')
    keys = sorted(sorted(custom), key=len, reverse=True)
    lr_mult, decay_mult = [], []
    for name, p in named_params:
        key = next((k for k in keys if k in name), None)
        if key is not None:
            a, b = custom[key].get('lr_mult', 1.0), custom[key].get('decay_mult', 1.0)
        else:
            norm, bias = id(p) in norm_params, name.rsplit('.', 1)[-1] == 'bias'
            a = bias_lr if bias and not norm else 1.0
            b = norm_decay if norm else bias_decay if bias else 1.0
        lr_mult.append(float(a))
        decay_mult.append(float(b))
    return lr_mult, decay_mult


def _base_lr(groups, mult):
    """the rate that every one of torch's parameter groups gives for a parameter of multiplier 1 (mmcv's constructor writes a group for each
    parameter, lr times its multiplier); None where no group tells.  mult: lr multiplier of each parameter index"""
    if any(not 0 <= i < len(mult) for g in groups for i in g.get('params', ())):
        raise MsclError("ClipAdamW: the state's groups hold parameters that the model has not")
    known = [(i, g) for g in groups if 'lr' in g for i in g.get('params', ()) if mult[i] > 0]
    if not known:
        return float(groups[0]['lr']) if 'lr' in groups[0] and 'params' not in groups[0] else None
    key = 'initial_lr' if all('initial_lr' in g for _, g in known) else 'lr'          # a schedule's floor is the same for all groups
    rates = [float(g[key]) / mult[i] for i, g in known]
    if max(rates) - min(rates) > 1e-6 * max(rates):
        raise MsclError(f'ClipAdamW: the state holds rates from {min(rates)} to {max(rates)} without their lr_mult: built with another paramwise_cfg')
    i, g = min(known, key=lambda e: abs(mult[e[0]] - 1))
    return float(g['lr']) / mult[i]


class ClipAdamW:
    """Clip + AdamW over a model's arena: what ClipSGD is, with `AdamW` in place of the SGD pass.  The parameters that have received a
    gradient by the first step take part (those that never do are left alone, as torch leaves a parameter without .grad)."""

    def __init__(self, model, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.01, grad_clip=None, state_bits=32, paramwise_cfg=None, seed=0):
        self.model, self.arena = model, model.arena
        self.state_bits, self._inner, self._slots = state_bits, None, None
        self._args = dict(betas=tuple(betas), eps=eps, weight_decay=weight_decay, grad_clip=grad_clip, state_bits=state_bits, seed=seed)
        _check_args(lr=lr, **self._args)
        norms = {id(p) for m in model.modules() if getattr(m, 'is_norm', False) or isinstance(m, BatchNorm3dHip) for p in m.parameters(recurse=False)}
        named = [(n, p) for n, p in model.named_parameters() if getattr(p, '_mscl_slot', None) is not None and p.requires_grad]
        self._mult = {p._mscl_slot: (a, b) for (n, p), a, b in zip(named, *_param_mults(named, norms, paramwise_cfg))}
        self.param_groups = [dict(lr=lr, betas=tuple(betas), eps=eps, weight_decay=weight_decay)]
        self.steps = 0

    @classmethod
    def from_cfg(cls, model, optimizer, optimizer_config=None):
        o = dict(optimizer)
        if o.pop('type', 'AdamW') != 'AdamW':
            raise NotImplementedError('ClipAdamW is built from type=AdamW (build_optimizer takes SGD and AdamW)')
        if o.pop('amsgrad', False):
            raise NotImplementedError('amsgrad is not built')
        return cls(model, grad_clip=(optimizer_config or {}).get('grad_clip'), **o)

    def zero_grad(self):
        self.model.sync_streams()
        self.arena.G.zero_()

    def grad_norm(self):
        """device scalar: L2 norm of the (all-reduced) gradient before clipping (kept only with grad_clip)"""
        return self._inner.grad_norm()

    def _build(self):
        ar = self.arena
        slots = [s for s in ar.slots if s.touched]
        if self._inner is not None and slots == self._slots:
            return
        self._slots = slots
        if not self._slots:
            raise MsclError('ClipAdamW: no parameter has received a gradient yet')
        cut = lambda which: [getattr(ar, which)[s.off:s.off + s.numel] for s in self._slots]          # noqa: E731
        mult = [self._mult.get(s, (1.0, 1.0)) for s in self._slots]
        self._inner = AdamW(cut('Q'), lr=self.param_groups[0]['lr'], shadows=cut('Qb'), lr_mult=[a for a, _ in mult],
                            decay_mult=[b for _, b in mult], **self._args)
        self._inner.param_groups = self.param_groups
        self._inner._set_grads(cut('G'))

    @torch.no_grad()
    def step(self):
        ar = self.arena
        self.model.sync_streams()
        if getattr(self.model, 'reducer', None) is not None:
            self.model.reducer.finish()         # buckets were launched from backward; wait for them
        else:
            parallel.allreduce_mean_(ar.G)
        if self._inner is None:
            if torch.cuda.is_current_stream_capturing():
                raise MsclError('ClipAdamW: take one eager step before capturing one')
            self._build()
        elif [s for s in ar.slots if s.touched] != self._slots:
            raise RuntimeError('the set of parameters receiving gradients changed between steps')
        self._inner._launch()
        self.model.refresh_after_optimizer()
        self.steps += 1

    def sync_lr(self):
        if self._inner is not None:
            self._inner.sync_lr()

    def _check_rebuild(self, loaded):
        """refuses a state whose parameters, beside those that take part by now, need another optimizer while a captured step uses this one"""
        inner = self._inner
        if inner is not None and (inner._in_graph or inner._kept) and any(s not in self._slots for s in loaded):
            raise MsclError('ClipAdamW: the state has parameters that a captured step does not update: load it into an optimizer that is not captured')

    def _slot_indices(self):
        return [i for i, s in enumerate(self.arena.slots) if any(s is t for t in self._slots)]

    def state_dict(self):
        if self._inner is None:
            return dict(type='AdamW', lr=self.param_groups[0]['lr'], state_bits=self.state_bits, slots=[])
        return dict(self._inner.state_dict(), type='AdamW', slots=self._slot_indices())

    def load_state_dict(self, state):
        """a state_dict() of this class, or torch.optim.AdamW's own (the reference's checkpoints; 32-bit states only), whose entries are
        keyed by the parameter's index in model.parameters() and whose groups hold lr times the parameter's multiplier (one step counter: the
        largest of the entries').  A state that is refused changes nothing"""
        if 'slots' in state:
            held, slots = list(state['slots']), self.arena.slots
            if state['state_bits'] != self.state_bits or any(not 0 <= i < len(slots) for i in held):
                raise MsclError('ClipAdamW: the state belongs to another model or another state_bits')
            if held:                                       # all of it is looked at before anything is changed
                _check_state(state, self.state_bits, [slots[i].numel for i in held])
                if held != sorted(set(held) | {i for i, s in enumerate(slots) if s.touched}):
                    raise MsclError('ClipAdamW: other parameters receive gradients than in the state')
                self._check_rebuild([slots[i] for i in held])
            self.param_groups[0]['lr'] = state['lr']
            if not held:                                   # from before the first step
                if self._inner is not None:
                    self._inner.reset(self._args['seed'])
                self.steps = 0
                return
            for i in held:
                slots[i].touched = True                    # as at the step that wrote the state
            self._build()
            self._inner.load_state_dict(state)
            self.steps = self._inner.steps
            return
        if self.state_bits != 32:
            raise MsclError('ClipAdamW: a torch.optim.AdamW state loads into state_bits=32')
        if any(g.get('amsgrad') for g in state.get('param_groups') or ()):
            raise NotImplementedError('amsgrad is not built')
        found, step, params = [], 0, list(self.model.parameters())
        for idx, p in enumerate(params):
            st = state['state'].get(idx, state['state'].get(str(idx)))
            if st is None:
                continue
            slot = getattr(p, '_mscl_slot', None)
            if slot is None or not p.requires_grad or any(tuple(st[k].shape) != tuple(p.shape) for k in ('exp_avg', 'exp_avg_sq')):
                raise ValueError(f'optimizer state {idx} does not belong to trainable parameter {idx} of this model')
            step = max(step, int(st['step']))
            found.append((slot, st))
        if not found:
            raise MsclError('ClipAdamW: the checkpoint holds no AdamW moments')
        mult = [self._mult.get(getattr(p, '_mscl_slot', None), (1.0, 1.0))[0] if p.requires_grad else 1.0 for p in params]
        lr = _base_lr(state.get('param_groups') or [{}], mult)
        self._check_rebuild([slot for slot, _ in found])
        for slot, _ in found:
            slot.touched = True
        self._build()
        at = dict(zip(self._slots, self._inner.offsets))
        for flat in (self._inner.exp_avg, self._inner.exp_avg_sq):          # parameters without an entry have no moments
            flat.zero_()
        for slot, st in found:
            for flat, key in ((self._inner.exp_avg, 'exp_avg'), (self._inner.exp_avg_sq, 'exp_avg_sq')):
                _physical_view(flat, at[slot], slot.shape).copy_(st[key])
        if lr is not None:
            self.param_groups[0]['lr'] = lr
        self._inner.set_step(step)
        self.steps = step


def build_optimizer(model, optimizer, optimizer_config=None):
    """the config's `optimizer` dict -> ClipSGD or ClipAdamW (ref: build_optimizer at mmaction/apis/train.py:94)"""
    kinds = dict(SGD=ClipSGD, AdamW=ClipAdamW)
    if optimizer.get('type', 'SGD') not in kinds:
        raise NotImplementedError(f"optimizer type {optimizer['type']}: SGD and AdamW are built")
    return kinds[optimizer.get('type', 'SGD')].from_cfg(model, optimizer, optimizer_config)
