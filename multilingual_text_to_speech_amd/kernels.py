"""Thin Python wrappers over the C-ABI: argument packing + torch.autograd glue.

Every compute step goes through libmtts_hip.so; torch is used for device memory, streams and
autograd bookkeeping only.  Activations are channel-last ([N, L, C]).
"""
import ctypes
import os

import torch
from torch.autograd import forward_ad

from . import _C
from ._C import check, lib, ptr, require_gpu, stream_of, stream_ptr

ACT = {'identity': 0, 'relu': 1, 'tanh': 2, 'sigmoid': 3}


def _f32(*shape, device):
    return torch.empty(*shape, dtype=torch.float32, device=device)


def keep_mask(shape, p, device, generator=None):
    """uint8 keep flags for dropout probability p (1 = keep)."""
    return (torch.rand(shape, device=device, generator=generator) >= p).to(torch.uint8)


# ------------------------------------------------------------------------------------------------
# GEMM
# ------------------------------------------------------------------------------------------------

def gemm(A, B, C, M, N, K, lda, ldb, ldc, transA=False, transB=False, alpha=1.0, beta=0.0, bias=None, act=0,
         mask=None, mask_scale=1.0, **kw):
    """C = epilogue(alpha * A(m,k) B(n,k) + beta C).  Extra GemmArgs fields via **kw (conv / batch modes)."""
    _C.ensure_workspace(C.device)
    g = _C.GemmArgs()
    g.A, g.B, g.C, g.bias, g.mask = ptr(A), ptr(B), ptr(C), ptr(bias), ptr(mask)
    g.M, g.N, g.K, g.lda, g.ldb, g.ldc = M, N, K, lda, ldb, ldc
    g.ldmask = kw.pop('ldmask', N)
    g.transA, g.transB = int(transA), int(transB)
    g.taps, g.Kc, g.batch, g.zt = 1, K, 1, 1
    g.alpha, g.beta, g.act, g.mask_scale = alpha, beta, act, mask_scale
    for k, v in kw.items():
        setattr(g, k, v)
    check(lib().mtts_gemm_ex(ctypes.byref(g), stream_ptr()), 'mtts_gemm_ex')
    return C


def colsum(x2):
    """Column sums of a contiguous [R, C] matrix (deterministic two-stage reduction, mtts_colsum): bias gradients."""
    R, C = x2.shape
    out = _f32(C, device=x2.device)
    ws = _f32(int(lib().mtts_colsum_workspace_floats(C)), device=x2.device)
    check(lib().mtts_colsum(ptr(x2), ptr(out), R, C, C, ptr(ws), stream_ptr()), 'mtts_colsum')
    return out


def linear_fwd(x, weight, bias=None, act=0, mask=None, mask_scale=1.0):
    """y = act(x W^T + b) [* dropout]; x [..., K] contiguous, weight [N, K] (torch Linear layout)."""
    require_gpu(x, weight)
    K = x.shape[-1]
    N = weight.shape[0]
    x2 = x.reshape(-1, K)
    y = _f32(x2.shape[0], N, device=x.device)
    gemm(x2, weight, y, x2.shape[0], N, K, K, K, N, bias=bias, act=act, mask=mask, mask_scale=mask_scale)
    return y.reshape(*x.shape[:-1], N)


def linear_bwd(x, weight, dy, need_dx=True):
    """Gradients of y = x W^T + b given dy (pre-activation gradient)."""
    K = x.shape[-1]
    N = weight.shape[0]
    x2, dy2 = x.reshape(-1, K), dy.reshape(-1, N)
    R = x2.shape[0]
    dW = _f32(N, K, device=x.device)
    gemm(dy2, x2, dW, N, K, R, N, K, K, transA=True, transB=True)
    db = colsum(dy2.contiguous())
    dx = None
    if need_dx:
        dx = _f32(R, K, device=x.device)
        gemm(dy2, weight, dx, R, K, N, N, K, K, transB=True)
        dx = dx.reshape(x.shape)
    return dx, dW, db


def _linear_bwd8(held, weight, dy, need_dx):
    """linear_bwd with the input held as a Checkpoint8."""
    N, K = weight.shape
    dy2 = dy.reshape(-1, N)
    dW = conv1d_weight_grad8(Checkpoint8._of(held.values.view(-1, K), held.scales.view(-1, held.scales.shape[-1])), dy2, 1).view(N, K)
    db = colsum(dy2)
    dx = None
    if need_dx:
        dx = _f32(dy2.shape[0], K, device=dy.device)
        gemm(dy2, weight, dx, dy2.shape[0], K, N, N, K, K, transB=True)
        dx = dx.view(held.values.shape)
    return dx, dW, db


class LinearFn(torch.autograd.Function):
    """Linear (+ReLU +dropout) through the MFMA GEMM.  mask: uint8 keep flags or None.  checkpoint: the input is saved in 8 bits (and
    of the output only which values are positive)."""

    @staticmethod
    def forward(ctx, x, weight, bias, act, mask, mask_scale, checkpoint=False):
        x = x.contiguous()
        y = linear_fwd(x, weight, bias, act, mask, mask_scale)
        if checkpoint:
            held = checkpoint8(x)
            ctx.save_for_backward(held.values, held.scales, weight, y > 0 if act == 1 else None, mask)
        else:
            ctx.save_for_backward(x, None, weight, y, mask)
        ctx.act, ctx.mask_scale, ctx.has_bias, ctx.checkpoint = act, mask_scale, bias is not None, checkpoint
        return y

    @staticmethod
    def backward(ctx, dy):
        if ctx.checkpoint:
            _first_derivative_only('linear')
        x, scales, weight, y, mask = ctx.saved_tensors
        dz = dy.contiguous()
        if mask is not None:
            dz = dz * mask.view_as(dz) * ctx.mask_scale
        if ctx.act == 1:
            dz = dz * (y if ctx.checkpoint else y > 0)
        elif ctx.act != 0:
            raise NotImplementedError('LinearFn backward supports identity/relu')
        if ctx.checkpoint:
            dx, dW, db = _linear_bwd8(Checkpoint8._of(x, scales), weight, dz, ctx.needs_input_grad[0])
        else:
            dx, dW, db = linear_bwd(x, weight, dz, ctx.needs_input_grad[0])
        return dx, dW, (db if ctx.has_bias else None), None, None, None, None


def linear(x, weight, bias=None, act='identity', mask=None, mask_scale=1.0, checkpoint=False):
    """y = act(x W^T + b) [* dropout].  checkpoint=True saves x for the backward as a `Checkpoint8` (a quarter of its bytes): the weight
    gradient is the one of the 8-bit values, everything else is unchanged (a second derivative is refused)."""
    return LinearFn.apply(x, weight, bias, ACT[act], mask, mask_scale, checkpoint and _recorded(x, weight, bias))


# ------------------------------------------------------------------------------------------------
# Embedding
# ------------------------------------------------------------------------------------------------

_ERR_FLAGS = {}


class _PinnedRing:
    """Small host -> device copies WITHOUT a stream synchronisation.  `cpu_tensor.to(device)` of pageable memory is hipMemcpyAsync +
    hipStreamSynchronize: the host waits until everything queued on the stream has finished - a train step did that nine times (sequence
    lengths in the encoder, the decoder, the output mask and the loss; the optimizer's pointer table), each one ending the host's run-ahead
    and leaving the GPU idle until the next launch arrives (scripts/dbg_sync_points.py).  Here the values go through a ring of pinned
    staging buffers: a CPU copy into the slot, an asynchronous copy to the device, an event that guards the slot's reuse."""
    SLOTS, BYTES = 32, 1 << 16

    def __init__(self):
        import threading
        self.slots, self.next, self.lock = [], 0, threading.Lock()

    def copy(self, src, device, dtype=None):
        dtype = dtype or src.dtype
        src = src.detach().to(dtype=dtype).contiguous().reshape(-1)
        nbytes = src.numel() * src.element_size()
        if nbytes > self.BYTES or nbytes == 0:
            return src.to(device)
        with self.lock:                                  # host threads driving different streams share the ring
            return self._copy_locked(src, device, dtype, nbytes)

    def _copy_locked(self, src, device, dtype, nbytes):
        if len(self.slots) < self.SLOTS:
            self.slots.append(dict(buf=torch.empty(self.BYTES, dtype=torch.uint8).pin_memory(), event=None))
            slot = self.slots[-1]
        else:
            slot = self.slots[self.next]
            self.next = (self.next + 1) % self.SLOTS
            if slot['event'] is not None:
                slot['event'].synchronize()              # the copy out of this slot was queued 32 copies ago: long done
        view = slot['buf'][:nbytes].view(dtype)
        view.copy_(src)
        out = torch.empty(src.numel(), dtype=dtype, device=device)
        with torch.cuda.device(device):
            out.copy_(view, non_blocking=True)
            if slot['event'] is None:
                slot['event'] = torch.cuda.Event()
            slot['event'].record()
        return out


_H2D = _PinnedRing()
_H2D_BLOCKING = os.environ.get('MTTS_H2D_BLOCKING', '0') == '1'      # A/B: the synchronising copies of round 5


def to_device_async(t, device, dtype=None):
    """`t.to(device=device, dtype=dtype)` for the small host tensors of a step (lengths, ids, pointer tables) without synchronising the
    stream; tensors that already live on the device are converted in place of a copy."""
    if t is None:
        return None
    if t.is_cuda or _H2D_BLOCKING:
        return t.to(device=device, dtype=dtype or t.dtype)
    shape = t.shape
    return _H2D.copy(t, torch.device(device), dtype).reshape(shape)


def _err_flag(device):
    """Two device ints per GPU: [0] raised by kernels that met invalid input (an embedding id outside its table), [1] by a persistent
    decoder kernel whose grid barrier gave up (DecoderArgs.persist_err)."""
    key = torch.device(device).index or 0
    if key not in _ERR_FLAGS:
        _ERR_FLAGS[key] = torch.zeros(2, dtype=torch.int32, device=device)
    return _ERR_FLAGS[key]


def check_device_errors(device=None):
    """Raise if a kernel flagged invalid input since the last check, or if a persistent decoder kernel gave up on a grid barrier
    (synchronises; call once per step / synthesis call)."""
    for key, flag in list(_ERR_FLAGS.items()):
        if device is not None and (torch.device(device).index or 0) != key:
            continue
        v = flag.tolist()
        if v[1] != 0:
            flag.zero_()
            raise _C.MttsError(f'a persistent decoder kernel reported error {v[1]} (2 = a grid barrier timed out: the decode of that call '
                               'is invalid); set MTTS_PERSIST=0 to run the per-step launch schedule')
        if v[0] != 0:
            flag.zero_()
            raise _C.MttsError('an embedding id was outside its table (symbol id >= symbols_count()+3, speaker id >= '
                               'hp.speaker_number or language id >= hp.language_number); the row was read as zeros')


_ERR_POLL = {}


def poll_device_errors(device=None):
    """check_device_errors without stalling the stream: enqueues a copy of this GPU's error words into pinned host memory and raises
    for what the PREVIOUS poll fetched (if that copy has completed - after a whole train step it has).  Called once per optimizer step
    by bench.train_step: a persistent decoder kernel that gave up is reported one step later, and the guarded optimizer step
    (AdamArgs.guard) has kept the invalid step away from the weights in the meantime."""
    for key, flag in list(_ERR_FLAGS.items()):
        if device is not None and (torch.device(device).index or 0) != key:
            continue
        st = _ERR_POLL.get(key)
        if st is None:
            st = _ERR_POLL[key] = dict(host=torch.zeros(2, dtype=torch.int32).pin_memory(), event=None)
        if st['event'] is not None:
            if not st['event'].query():
                continue                               # the previous copy is still in flight: look again at the next call
            st['event'] = None
            if int(st['host'][0]) != 0 or int(st['host'][1]) != 0:
                check_device_errors(flag.device)       # synchronises, clears the words and raises with the full message
        with torch.cuda.device(flag.device):
            st['host'].copy_(flag, non_blocking=True)
            st['event'] = torch.cuda.Event()
            st['event'].record()


class EmbeddingFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, table, ids, padding_idx):
        require_gpu(table, ids)
        ids = ids.contiguous()
        D = table.shape[1]
        out = _f32(*ids.shape, D, device=table.device)
        check(lib().mtts_embedding_fwd(ptr(table), ptr(ids), ptr(out), ids.numel(), D, D, 0, ctypes.c_long(table.shape[0]),
                                       ptr(_err_flag(table.device)), stream_ptr()), 'embedding_fwd')
        ctx.save_for_backward(ids)
        ctx.shape, ctx.padding_idx = table.shape, padding_idx
        return out

    @staticmethod
    def backward(ctx, dout):
        (ids,) = ctx.saved_tensors
        dout = dout.contiguous()
        D = ctx.shape[1]
        dtable = torch.zeros(ctx.shape, dtype=torch.float32, device=dout.device)
        check(lib().mtts_embedding_bwd(ptr(dout), ptr(ids), ptr(dtable), ids.numel(), D, D, 0,
                                       -1 if ctx.padding_idx is None else ctx.padding_idx, ctypes.c_long(ctx.shape[0]),
                                       stream_ptr()), 'embedding_bwd')
        return dtable, None, None


def embedding(table, ids, padding_idx=None):
    return EmbeddingFn.apply(table, ids, padding_idx)


# ------------------------------------------------------------------------------------------------
# Conv1d (+BN +act +dropout +highway), channel-last
# ------------------------------------------------------------------------------------------------

def pack_conv_weight(weight):
    """torch [O, I, k] -> implicit-GEMM layout [O, k, I]."""
    O, I, k = weight.shape
    out = _f32(O, k, I, device=weight.device)
    check(lib().mtts_conv_weight_pack(ptr(weight.contiguous()), ptr(out), O, I, k, 1, stream_ptr()), 'conv_weight_pack')
    return out


def unpack_conv_weight(packed, O, I, k):
    out = _f32(O, I, k, device=packed.device)
    check(lib().mtts_conv_weight_pack(ptr(packed), ptr(out), O, I, k, 0, stream_ptr()), 'conv_weight_pack')
    return out


def conv1d_fwd(x, wp, k, dilation, groups):
    """x [N, L, Cin] channel-last, wp packed [O, k, Cin/G] -> [N, L, O] ('same' zero padding)."""
    N_, L, Cin = x.shape
    O = wp.shape[0]
    Cg, Og = Cin // groups, O // groups
    y = _f32(N_, L, O, device=x.device)
    p = (k - 1) * dilation // 2
    gemm(x, wp, y, N_ * L, Og, k * Cg, Cin, k * Cg, O, taps=k, Kc=Cg, seq_len=L, shift_mode=1, shift0=-p, dshift=dilation,
         batch=groups, a_z=Cg, b_z=Og * k * Cg, c_z=Og)
    return y


def conv1d_bwd(x, wp, dy, k, dilation, groups, need_dx=True):
    """Gradients of conv1d_fwd: dx [N,L,Cin], dwp packed [O,k,Cin/G]."""
    N_, L, Cin = x.shape
    O = wp.shape[0]
    Cg, Og = Cin // groups, O // groups
    R = N_ * L
    p = (k - 1) * dilation // 2
    dwp = _f32(O, k, Cg, device=x.device)
    # dW[o, t, c] = sum_r dy[r, o] * x[r + shift_t, c]   (one TN GEMM per tap through grid.z)
    gemm(dy, x, dwp, Og, Cg, R, O, Cin, k * Cg, transA=True, transB=True, seq_len=L, shift_mode=2, shift0=-p,
         dshift=dilation, batch=groups, zt=k, a_z=Og, b_z=Cg, c_z=Og * k * Cg, c_ztap=Cg)
    return conv1d_input_grad(wp, dy, Cin, k, dilation, groups) if need_dx else None, dwp


def conv1d_input_grad(wp, dy, Cin, k, dilation, groups):
    """Input gradient of conv1d_fwd: dx [N, L, Cin]."""
    N_, L, O = dy.shape
    Cg, Og = Cin // groups, O // groups
    dx = _f32(N_, L, Cin, device=dy.device)
    # dx[r, c] = sum_t sum_o dy[r - shift_t, o] * w[o, t, c]
    gemm(dy, wp, dx, N_ * L, Cg, k * Og, O, k * Cg, Cin, transB=True, taps=k, Kc=Og, seq_len=L, shift_mode=1, shift0=(k - 1) * dilation // 2,
         dshift=-dilation, b_tap=Cg, batch=groups, a_z=Og, b_z=Og * k * Cg, c_z=Cg)
    return dx


def _bn_args(x2, gamma, beta, rmean, rvar, smean, srstd, mask, resid, y, ws, training, momentum, eps, act, mask_scale,
             hw_groups):
    a = _C.BnArgs()
    a.x, a.gamma, a.beta = ptr(x2), ptr(gamma), ptr(beta)
    a.running_mean, a.running_var, a.save_mean, a.save_rstd = ptr(rmean), ptr(rvar), ptr(smean), ptr(srstd)
    a.mask, a.resid, a.y, a.ws = ptr(mask), ptr(resid), ptr(y), ptr(ws)
    a.R, a.C = x2.shape[0], x2.shape[1]
    a.training, a.momentum, a.eps, a.act, a.mask_scale, a.hw_groups = int(training), momentum, eps, act, mask_scale, hw_groups
    return a


class ConvBnActFn(torch.autograd.Function):
    """pad -> conv1d(groups, dilation, no bias) -> BatchNorm -> act -> dropout [-> highway gate], channel-last.

    reference: ConvBlock modules/layers.py:50-86, HighwayConvBlock :134-153 and the generated variants :89-178
    (the generated kernel / affine tensors are passed in as `weight`, `gamma`, `beta`)."""

    @staticmethod
    def forward(ctx, x, weight, gamma, beta, rmean, rvar, mask, cfg):
        k, dilation, groups, act, training, momentum, eps, mask_scale, highway = cfg[:9]
        packed = len(cfg) > 9 and cfg[9]          # weight already in the implicit-GEMM layout [O, k, I/G] (generated kernels)
        require_gpu(x, weight)
        x = x.contiguous()
        N_, L, Cin = x.shape
        O = weight.shape[0]
        wp = weight.contiguous() if packed else pack_conv_weight(weight)
        conv = conv1d_fwd(x, wp, k, dilation, groups)
        conv2 = conv.view(N_ * L, O)
        dev = x.device
        smean, srstd = _f32(O, device=dev), _f32(O, device=dev)
        ws = _f32(int(lib().mtts_bn_workspace_floats(O)), device=dev)
        Cy = O // 2 if highway else O
        y = _f32(N_, L, Cy, device=dev)
        a = _bn_args(conv2, gamma.contiguous(), beta.contiguous(), rmean, rvar, smean, srstd, mask, x if highway else None, y, ws,
                     training, momentum, eps, act, mask_scale, groups if highway else 0)
        check(lib().mtts_bn_act_fwd(ctypes.byref(a), stream_ptr()), 'bn_act_fwd')
        ctx.checkpoint = len(cfg) > 10 and cfg[10]
        held_x, held_conv = (checkpoint8(x), checkpoint8(conv)) if ctx.checkpoint else (None, None)
        ctx.save_for_backward(held_x.values if held_x else x, wp, held_conv.values if held_conv else conv, gamma, beta, smean, srstd, mask,
                              held_x.scales if held_x else None, held_conv.scales if held_conv else None)
        ctx.cfg, ctx.wshape = cfg, tuple(weight.shape)
        return y

    @staticmethod
    def backward(ctx, dy):
        x, wp, conv, gamma, beta, smean, srstd, mask, x_scales, conv_scales = ctx.saved_tensors
        k, dilation, groups, act, training, momentum, eps, mask_scale, highway = ctx.cfg[:9]
        packed = len(ctx.cfg) > 9 and ctx.cfg[9]
        held_x = None
        if ctx.checkpoint:
            _first_derivative_only('conv_bn_act')
            held_x = Checkpoint8._of(x, x_scales)
            conv = Checkpoint8._of(conv, conv_scales).unpack()
            x = held_x.unpack() if highway else x
        N_, L, Cin = x.shape
        O = conv.shape[2]
        dev = x.device
        dy = dy.contiguous()
        dconv = _f32(N_, L, O, device=dev)
        dgamma, dbeta = _f32(O, device=dev), _f32(O, device=dev)
        dresid = _f32(N_, L, O // 2, device=dev) if highway else None
        ws = _f32(int(lib().mtts_bn_workspace_floats(O)), device=dev)
        a = _bn_args(conv.view(N_ * L, O), gamma.contiguous(), beta.contiguous(), None, None, smean, srstd, mask,
                     x if highway else None, None, ws, training, momentum, eps, act, mask_scale, groups if highway else 0)
        a.dy, a.dx, a.dgamma, a.dbeta, a.dresid = ptr(dy), ptr(dconv), ptr(dgamma), ptr(dbeta), ptr(dresid)
        check(lib().mtts_bn_act_bwd(ctypes.byref(a), stream_ptr()), 'bn_act_bwd')
        if ctx.checkpoint:
            dx = conv1d_input_grad(wp, dconv, Cin, k, dilation, groups) if ctx.needs_input_grad[0] or highway else None
            dw = conv1d_weight_grad8(held_x, dconv, k, dilation, groups, packed=packed)
        else:
            dx, dwp = conv1d_bwd(x, wp, dconv, k, dilation, groups, ctx.needs_input_grad[0] or highway)
            dw = dwp if packed else unpack_conv_weight(dwp, *ctx.wshape)
        if highway:
            dx = dx + dresid
        return dx, dw, dgamma, dbeta, None, None, None, None


def conv_bn_act(x, weight, gamma, beta, rmean, rvar, mask, *, kernel, dilation=1, groups=1, act='identity', training=True,
                momentum=0.1, eps=1e-5, mask_scale=1.0, highway=False, packed=False, checkpoint=False):
    """checkpoint=True saves the block's input and the convolution's output for the backward as `Checkpoint8` (a quarter of their bytes); a
    second derivative is refused then."""
    cfg = (kernel, dilation, groups, ACT[act], training, momentum, eps, mask_scale, highway, packed,
           checkpoint and _recorded(x, weight, gamma, beta))
    return ConvBnActFn.apply(x, weight, gamma, beta, rmean, rvar, mask, cfg)


# ------------------------------------------------------------------------------------------------
# 8-bit activation checkpoints, the weight gradient that reads them, group norm, channel-last
# ------------------------------------------------------------------------------------------------

CHECKPOINT_BLOCK = 32                      # neighbouring channels of a row that share an exponent
_DTYPE = {torch.float32: 0, torch.bfloat16: 1}
GN_ACT = {**ACT, 'silu': 4}


_MOST_ROWS = 0x7fff0000                    # row and channel numbers are 32-bit


def _refuse(what, why):
    raise _C.MttsError(f'{what}: {why}')


def _check_sizes(what, **sizes):
    """The kernels count in 32 bits, with room for a workgroup's rows behind the last one; ctypes would cut a larger number off."""
    for name, n in sizes.items():
        if n > _MOST_ROWS:
            _refuse(what, f'{n} {name} are too many for one call')


def _check_storage(what, t, name):
    if t.dtype not in _DTYPE:
        _refuse(what, f'{name} is {t.dtype}: float32 or bfloat16 is expected')


def _first_derivative_only(what):
    if torch.is_grad_enabled():            # a backward under create_graph=True: its outputs would look like constants
        _refuse(what, 'there is no second derivative (create_graph=True)')


def _recorded(*tensors):
    """Whether a graph is being recorded: nobody reads what a call saves otherwise."""
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


def _differentiated(x, gamma, beta):
    """Whether autograd follows the call: a graph is being recorded, or an operand carries a forward-mode tangent (such an operand need
    not require a gradient; autograd.Function refuses it where there is no jvp)."""
    if torch.is_grad_enabled() and (x.requires_grad or gamma.requires_grad or beta.requires_grad):
        return True
    if forward_ad.unpack_dual(x).primal is x:      # outside of forward-mode differentiation: nothing has a tangent
        return False
    return any(forward_ad.unpack_dual(t).tangent is not None for t in (x, gamma, beta))


def _same_device(what, device, *tensors):
    for t in tensors:
        if t is not None and t.device != device:
            _refuse(what, f'the input is on {device}, another operand on {t.device}')


def _at(t):
    return None if t is None else t.data_ptr()


class _On:
    """The launch's device is the tensors' own, whatever device is current."""
    __slots__ = ('guard',)

    def __init__(self, device):
        self.guard = torch.cuda.device(device) if device.index != torch.cuda.current_device() else None

    def __enter__(self):
        if self.guard is not None:
            self.guard.__enter__()

    def __exit__(self, *exc):
        if self.guard is not None:
            self.guard.__exit__(*exc)


def _check_lengths(what, lengths, N, L, device):
    """Lengths [N], int32 or int64.  Host values are checked; values that already live on the device are clamped to [0, L] by the kernels."""
    if lengths is None:
        return None
    if not isinstance(lengths, torch.Tensor):
        lengths = torch.tensor(lengths)
        if not (lengths.numel() and lengths.is_floating_point()):            # fractions are refused below, not cut off
            lengths = lengths.to(torch.int64)
    if tuple(lengths.shape) != (N,) or lengths.dtype not in (torch.int32, torch.int64):
        _refuse(what, f'lengths is {lengths.dtype} {tuple(lengths.shape)}: int32 or int64 of shape ({N},) is expected')
    if lengths.is_cuda:
        _same_device(what, device, lengths)
    elif N and (int(lengths.min()) < 0 or int(lengths.max()) > L):
        _refuse(what, f'lengths run from {int(lengths.min())} to {int(lengths.max())}: 0 to {L} is expected')
    return lengths


def _device_lengths(what, lengths, device):
    if lengths is None:
        return None
    if not lengths.is_cuda and torch.cuda.is_current_stream_capturing():
        _refuse(what, 'lengths have to be on the device while a graph is captured')
    if lengths.is_cuda and lengths.dtype == torch.int64:
        lengths = lengths.clamp(-1, 2 ** 31 - 1)              # the kernels' clamp to [0, L] must not see a wrapped value
    return to_device_async(lengths, device, torch.int32).contiguous()


class Checkpoint8:
    """An activation in 8 bits: `values` int8 [..., C] and `scales` uint8 [..., ceil(C / 32)], biased exponents of one power of two per 32
    neighbouring channels of a row.  It stands for values * 2^(scales - 127), which is exact in float32 and in bfloat16; a block with an
    infinity or a NaN (exponent 255) stands for NaN.  `dtype` is the type that unpack() returns unless told otherwise."""
    __slots__ = ('values', 'scales', 'dtype')

    def __init__(self, values, scales, dtype=torch.float32):
        if values.dtype != torch.int8 or scales.dtype != torch.uint8 or values.dim() < 1:
            _refuse('Checkpoint8', f'values {values.dtype}, scales {scales.dtype}: int8 and uint8 are expected')
        want = (*values.shape[:-1], -(-values.shape[-1] // CHECKPOINT_BLOCK))
        if scales.shape != want:
            _refuse('Checkpoint8', f'scales have shape {tuple(scales.shape)}: {want} is expected for values of shape {tuple(values.shape)}')
        if dtype not in _DTYPE:
            _refuse('Checkpoint8', f'dtype is {dtype}: float32 or bfloat16 is expected')
        _same_device('Checkpoint8', values.device, scales)
        self.values, self.scales, self.dtype = values.contiguous(), scales.contiguous(), dtype

    @classmethod
    def _of(cls, values, scales, dtype=torch.float32):
        """Around tensors that this module made: nothing to check."""
        held = cls.__new__(cls)
        held.values, held.scales, held.dtype = values, scales, dtype
        return held

    @property
    def shape(self):
        return self.values.shape

    @property
    def nbytes(self):
        return self.values.numel() + self.scales.numel()

    def unpack(self, dtype=None):
        """The values it stands for, [..., C]."""
        dtype = dtype or self.dtype
        if dtype not in _DTYPE:
            _refuse('Checkpoint8.unpack', f'dtype is {dtype}: float32 or bfloat16 is expected')
        _check_sizes('Checkpoint8.unpack', channels=self.shape[-1])
        require_gpu(self.values)
        out = torch.empty(self.values.shape, dtype=dtype, device=self.values.device)
        if out.numel():
            C = out.shape[-1]
            with _On(out.device):
                check(lib().mtts_checkpoint8_unpack(self.values.data_ptr(), self.scales.data_ptr(), out.data_ptr(), out.numel() // C, C,
                                                    _DTYPE[dtype], stream_of(out.device)), 'checkpoint8_unpack')
        return out


def checkpoint8(x, lengths=None):
    """`Checkpoint8` of an activation [..., C] (float32 or bfloat16).  With `lengths` [N] for x [N, L, C] the rows behind a sample's length
    are not read and stand for zeros.  The error is at most half of a step of the block's power of two: 1/127.5 of the block's largest
    magnitude, 2^-127 where that is below 2^-120; magnitudes of 255/128 * 2^127 and more stop at 63/32 * 2^127.  To autograd what
    unpack() returns is a constant."""
    what = 'checkpoint8'
    _check_storage(what, x, 'x')
    if lengths is not None and x.dim() != 3:
        _refuse(what, f'lengths need an input [N, L, C], not {tuple(x.shape)}')
    if x.dim() < 1 or x.shape[-1] < 1:
        _refuse(what, f'x has shape {tuple(x.shape)}: at least one channel is expected')
    if lengths is not None:
        lengths = _check_lengths(what, lengths, x.shape[0], x.shape[1], x.device)
    _check_sizes(what, rows=x.numel() // x.shape[-1], channels=x.shape[-1])
    require_gpu(x)
    if not x.is_contiguous():
        x = x.detach().contiguous()
    C = x.shape[-1]
    values = torch.empty(x.shape, dtype=torch.int8, device=x.device)
    scales = torch.empty((*x.shape[:-1], -(-C // CHECKPOINT_BLOCK)), dtype=torch.uint8, device=x.device)
    if x.numel():
        N, L = (x.shape[0], x.shape[1]) if lengths is not None else (1, x.numel() // C)
        with _On(x.device):
            lens = _device_lengths(what, lengths, x.device)
            check(lib().mtts_checkpoint8_pack(x.data_ptr(), _at(lens), values.data_ptr(), scales.data_ptr(), N, L, C, _DTYPE[x.dtype], stream_of(x.device)), what)
    return Checkpoint8._of(values, scales, x.dtype)


def conv1d_weight_grad8(held, dy, kernel, dilation=1, groups=1, packed=False):
    """Weight gradient of a 'same'-padded 1-D convolution from the `Checkpoint8` of its input [N, L, I] and dy [N, L, O] (float32 or
    bfloat16): dW[o, c, t] = sum_{n, l} dy[n, l, o] x[n, l + t * dilation - (kernel - 1) * dilation // 2, c], float32 [O, I / groups, kernel]
    (packed: [O, kernel, I / groups]).  kernel 1 takes inputs [..., I] of any shape: a linear layer.  A float32 dy keeps its bits down
    to 2^-133 (all 24 from magnitudes of 2^-110 on) unless set_precision('bf16') is on; an infinity in it makes its output channel NaN.  To
    autograd the result is a constant."""
    what = 'conv1d_weight_grad8'
    _check_storage(what, dy, 'dy')
    if kernel < 1 or dilation < 1 or groups < 1:
        _refuse(what, f'kernel {kernel}, dilation {dilation}, groups {groups}: whole numbers of 1 and more are expected')
    if held.shape[:-1] != dy.shape[:-1] or dy.dim() < 1 or (kernel > 1 and dy.dim() != 3):
        _refuse(what, f'input {tuple(held.shape)} and gradient {tuple(dy.shape)} do not belong to one convolution of kernel {kernel}')
    _same_device(what, dy.device, held.values)
    I, O = held.shape[-1], dy.shape[-1]
    if I % groups or O % groups or not I or not O:
        _refuse(what, f'{I} x {O} channels are not a multiple of {groups} groups')
    _check_sizes(what, rows=dy.numel() // O, channels=max(I, O), taps=max(kernel, (kernel - 1) * dilation))
    require_gpu(held.values, dy)
    shape = (O, kernel, I // groups) if packed else (O, I // groups, kernel)
    rows = dy.numel() // O
    if not rows:
        return torch.zeros(shape, dtype=torch.float32, device=dy.device)
    if not dy.is_contiguous():
        dy = dy.detach().contiguous()
    dw = _f32(shape, device=dy.device)
    N, L = (dy.shape[0], dy.shape[1]) if kernel > 1 else (1, rows)
    a = _C.Wgrad8Args(held.values.data_ptr(), held.scales.data_ptr(), dy.data_ptr(), dw.data_ptr(), None, N, L, I, O, kernel, dilation if kernel > 1 else 1, groups,
                      _DTYPE[dy.dtype], int(packed), 0)
    with _On(dy.device):
        n = lib().mtts_conv_weight_grad8_workspace_floats(ctypes.byref(a))
        if n < 0:
            _refuse(what, lib().mtts_last_error().decode())
        ws = _f32(n, device=dy.device) if n else None
        a.ws = _at(ws)
        check(lib().mtts_conv_weight_grad8(ctypes.byref(a), stream_of(dy.device)), what)
    return dw


def _gn_fwd(x, gamma, beta, groups, lengths, mask, act, eps, mask_scale, checkpoint):
    """y, mean and rstd [2, N, G], checkpoint values / scales (or None) of contiguous operands."""
    N, L, C = x.shape
    dev = x.device
    y = torch.empty_like(x)
    stats = torch.empty((2, N, groups), dtype=torch.float32, device=dev)
    q = code = None
    if checkpoint:
        q = torch.empty(x.shape, dtype=torch.int8, device=dev)
        code = torch.empty(N, L, -(-C // CHECKPOINT_BLOCK), dtype=torch.uint8, device=dev)
    if x.numel():
        at = stats.data_ptr()
        a = _C.GroupNormArgs(x.data_ptr(), gamma.data_ptr(), beta.data_ptr(), _at(lengths), _at(mask), y.data_ptr(), at, at + 4 * N * groups,
                             _at(q), _at(code), None, N, L, C, groups, _DTYPE[x.dtype], act, eps, mask_scale)
        _gn_launch(lib().mtts_group_norm_act_fwd, 'group_norm_act_fwd', a, 0, dev)
    return y, stats, q, code


def _gn_launch(entry, what, a, backward, device):
    at = ctypes.addressof(a)
    n = lib().mtts_group_norm_workspace_floats(at, backward)
    if n < 0:
        _refuse(what, lib().mtts_last_error().decode())
    if n:
        ws = _f32(n, device=device)
        a.ws = ws.data_ptr()
    check(entry(at, stream_of(device)), what)


def _gn_bwd(x, q, code, gamma, beta, stats, lengths, mask, dy, groups, act, eps, mask_scale):
    """dx, dgamma, dbeta; x may be None where the checkpoint (q, code) holds it."""
    N, L, C = dy.shape
    dx = torch.empty_like(dy)
    if not dy.numel():
        return dx, torch.zeros_like(gamma), torch.zeros_like(beta)
    dgamma, dbeta = torch.empty_like(gamma), torch.empty_like(beta)
    at = stats.data_ptr()
    a = _C.GroupNormArgs(_at(x), gamma.data_ptr(), beta.data_ptr(), _at(lengths), _at(mask), None, at, at + 4 * N * groups, _at(q), _at(code), None,
                         N, L, C, groups, _DTYPE[dy.dtype], act, eps, mask_scale, dy.data_ptr(), dx.data_ptr(), dgamma.data_ptr(), dbeta.data_ptr())
    _gn_launch(lib().mtts_group_norm_act_bwd, 'group_norm_act_bwd', a, 1, dy.device)
    return dx, dgamma, dbeta


class GroupNormActFn(torch.autograd.Function):
    """Group norm + activation + dropout (mtts_group_norm_act_fwd / _bwd)."""

    @staticmethod
    def forward(ctx, x, gamma, beta, lengths, mask, cfg):
        groups, act, eps, mask_scale, checkpoint = cfg
        y, stats, q, code = _gn_fwd(x, gamma, beta, groups, lengths, mask, act, eps, mask_scale, checkpoint)
        ctx.save_for_backward(None if checkpoint else x, q, code, gamma, beta, stats, lengths, mask)
        ctx.cfg = cfg
        return y

    @staticmethod
    def backward(ctx, dy):
        _first_derivative_only('group_norm_act')
        x, q, code, gamma, beta, stats, lengths, mask = ctx.saved_tensors
        groups, act, eps, mask_scale, _ = ctx.cfg
        with _On(dy.device):
            dx, dgamma, dbeta = _gn_bwd(x, q, code, gamma, beta, stats, lengths, mask, dy.contiguous(), groups, act, eps, mask_scale)
        return dx, dgamma, dbeta, None, None, None


def _gn_check(what, shape, device, gamma, beta, groups, lengths, mask, act):
    """Contiguous gamma, beta, lengths (where they are) and uint8 flags, or a refusal."""
    N, L, C = shape
    if max(N, L, C) > _MOST_ROWS:
        _check_sizes(what, samples=N, rows=L, channels=C)
    if groups < 1 or C < 1 or C % groups:
        _refuse(what, f'{C} channels are not a multiple of {groups} groups')
    if act not in GN_ACT:
        _refuse(what, f'unknown activation {act!r}: one of {", ".join(GN_ACT)} is expected')
    if gamma.dtype != torch.float32 or gamma.shape != (C,):
        _refuse(what, f'gamma is {gamma.dtype} {tuple(gamma.shape)}: float32 of shape ({C},) is expected')
    if beta.dtype != torch.float32 or beta.shape != (C,):
        _refuse(what, f'beta is {beta.dtype} {tuple(beta.shape)}: float32 of shape ({C},) is expected')
    if mask is not None:
        if mask.dtype not in (torch.uint8, torch.bool) or mask.shape != (N, L, C):
            _refuse(what, f'mask is {mask.dtype} {tuple(mask.shape)}: uint8 keep flags of shape {(N, L, C)} are expected')
        mask = mask.contiguous()
        if mask.dtype == torch.bool:
            mask = mask.view(torch.uint8)
    _same_device(what, device, gamma, beta, mask)
    return gamma.contiguous(), beta.contiguous(), _check_lengths(what, lengths, N, L, device), mask


def group_norm_act(x, gamma, beta, groups, lengths=None, mask=None, *, act='identity', eps=1e-5, mask_scale=1.0, checkpoint=False):
    """y = dropout(act(gamma * (x - mean) / sqrt(var + eps) + beta)) over x [N, L, C] channel-last, float32 or bfloat16 (gamma, beta:
    float32).  Mean and (biased) variance of a sample's group run over its lengths[n] valid rows and the group's C / groups channels; rows
    behind the length are never read, and y and the gradient of x are zero there.  act: identity, relu, tanh, sigmoid or silu;
    mask: uint8 keep flags [N, L, C] with the factor mask_scale, as in conv_bn_act.  First derivatives in reverse mode only.
    checkpoint=True saves x for the backward as a `Checkpoint8`: mean and deviation stay those of x, the gradients are those of the
    8-bit values.  A backward that is captured into a graph has to be the only live graph of its leaves (torch's own rule: release the
    eager one first)."""
    what = 'group_norm_act'
    _check_storage(what, x, 'x')
    if x.dim() != 3:
        _refuse(what, f'x has shape {tuple(x.shape)}: [N, L, C] is expected')
    gamma, beta, lengths, mask = _gn_check(what, x.shape, x.device, gamma, beta, groups, lengths, mask, act)
    require_gpu(x)
    with _On(x.device):
        lens, x = _device_lengths(what, lengths, x.device), x.contiguous()
        if _differentiated(x, gamma, beta):
            return GroupNormActFn.apply(x, gamma, beta, lens, mask, (groups, GN_ACT[act], eps, mask_scale, checkpoint))
        return _gn_fwd(x, gamma, beta, groups, lens, mask, GN_ACT[act], eps, mask_scale, False)[0]


class ConvGnActFn(torch.autograd.Function):
    """pad -> conv1d(groups, dilation, no bias) -> group norm -> act -> dropout, channel-last: ConvBnActFn with statistics per sample."""

    @staticmethod
    def forward(ctx, x, weight, gamma, beta, lengths, mask, cfg):
        k, dilation, groups, norm_groups, act, eps, mask_scale, checkpoint = cfg
        with _On(x.device):
            wp = pack_conv_weight(weight)
            conv = conv1d_fwd(x, wp, k, dilation, groups)
            y, stats, q, code = _gn_fwd(conv, gamma, beta, norm_groups, lengths, mask, act, eps, mask_scale, checkpoint)
            held = checkpoint8(x) if checkpoint else None
        if checkpoint:
            ctx.save_for_backward(held.values, held.scales, None, q, code, wp, gamma, beta, stats, lengths, mask)
        else:
            ctx.save_for_backward(x, None, conv, None, None, wp, gamma, beta, stats, lengths, mask)
        ctx.cfg, ctx.wshape = cfg, tuple(weight.shape)
        return y

    @staticmethod
    def backward(ctx, dy):
        _first_derivative_only('conv_gn_act')
        x, x_scales, conv, q, code, wp, gamma, beta, stats, lengths, mask = ctx.saved_tensors
        k, dilation, groups, norm_groups, act, eps, mask_scale, checkpoint = ctx.cfg
        with _On(dy.device):
            dconv, dgamma, dbeta = _gn_bwd(conv, q, code, gamma, beta, stats, lengths, mask, dy.contiguous(), norm_groups, act, eps, mask_scale)
            need_dx = ctx.needs_input_grad[0]
            if checkpoint:
                dx = conv1d_input_grad(wp, dconv, x.shape[2], k, dilation, groups) if need_dx else None
                dw = conv1d_weight_grad8(Checkpoint8._of(x, x_scales), dconv, k, dilation, groups)
            else:
                dx, dwp = conv1d_bwd(x, wp, dconv, k, dilation, groups, need_dx)
                dw = unpack_conv_weight(dwp, *ctx.wshape)
        return dx, dw, dgamma, dbeta, None, None, None


def conv_gn_act(x, weight, gamma, beta, lengths=None, mask=None, *, kernel, norm_groups, dilation=1, groups=1, act='identity', eps=1e-5,
                mask_scale=1.0, checkpoint=False):
    """The block of conv_bn_act with group norm over norm_groups groups in place of batch norm: x float32 [N, L, I], weight [O, I / groups,
    kernel] -> [N, L, O].  The rows behind a sample's length take part in the convolution as they are (zeros, where the previous block was
    this one) and are zeros in the output.  checkpoint=True saves the input and the convolution's output in 8 bits, and the weight
    gradient is computed from the 8-bit input."""
    what = 'conv_gn_act'
    if x.dtype != torch.float32 or weight.dtype != torch.float32 or x.dim() != 3 or weight.dim() != 3:
        _refuse(what, f'x {x.dtype} {tuple(x.shape)}, weight {weight.dtype} {tuple(weight.shape)}: float32 [N, L, I] and [O, I / groups, kernel] are expected')
    if not x.numel():
        _refuse(what, f'x has shape {tuple(x.shape)}: at least one value is expected')
    if min(kernel, dilation, groups) < 1 or tuple(weight.shape[1:]) != (x.shape[2] // groups, kernel) or x.shape[2] % groups or weight.shape[0] % groups:
        _refuse(what, f'input {tuple(x.shape)} and weight {tuple(weight.shape)} do not belong to one convolution of kernel {kernel} with {groups} groups')
    _check_sizes(what, rows=x.shape[0] * x.shape[1] + (kernel - 1) * dilation)      # a tap's place among them
    _same_device(what, x.device, weight)
    gamma, beta, lengths, mask = _gn_check(what, (x.shape[0], x.shape[1], weight.shape[0]), x.device, gamma, beta, norm_groups, lengths, mask, act)
    require_gpu(x)
    with _On(x.device):
        lens = _device_lengths(what, lengths, x.device)
        cfg = (kernel, dilation, groups, norm_groups, GN_ACT[act], eps, mask_scale, checkpoint and _recorded(x, weight, gamma, beta))
        return ConvGnActFn.apply(x.contiguous(), weight, gamma, beta, lens, mask, cfg)


class GenKernelFn(torch.autograd.Function):
    """Generated convolution kernel straight into the implicit-GEMM layout (reference Conv1dGenerated.forward,
    modules/generated.py:34-42): hidden [G, bott] x w_kernel [(O/G)(I/G)k, bott]^T + b_kernel -> packed [O, k, I/G].
    One bandwidth-bound kernel each way (mtts_gen_params_fwd / _bwd) instead of a padded MFMA GEMM + view + repack."""

    @staticmethod
    def forward(ctx, hidden, w_kernel, b_kernel, dims):
        Og, Cg, k = dims
        require_gpu(hidden, w_kernel)
        hidden, w_kernel = hidden.contiguous(), w_kernel.contiguous()
        G, bott = hidden.shape
        wp = _f32(G * Og, k, Cg, device=hidden.device)
        a = _C.GenParamsArgs()
        a.hidden, a.w_kernel, a.b_kernel, a.w_packed = ptr(hidden), ptr(w_kernel), ptr(b_kernel), ptr(wp)
        a.G, a.bott, a.Og, a.Cg, a.k = G, bott, Og, Cg, k
        check(lib().mtts_gen_params_fwd(ctypes.byref(a), stream_ptr()), 'mtts_gen_params_fwd')
        ctx.save_for_backward(hidden, w_kernel)
        ctx.dims, ctx.has_bias = dims, b_kernel is not None
        return wp

    @staticmethod
    def backward(ctx, dwp):
        hidden, w_kernel = ctx.saved_tensors
        Og, Cg, k = ctx.dims
        G, bott = hidden.shape
        dev = hidden.device
        dwp = dwp.contiguous()
        nslab = int(lib().mtts_gen_params_slabs(Og, Cg))
        dwk = _f32(*w_kernel.shape, device=dev)
        dbk = _f32(w_kernel.shape[0], device=dev) if ctx.has_bias else None
        slab = _f32(nslab, G * bott, device=dev)
        a = _C.GenParamsArgs()
        a.hidden, a.w_kernel, a.d_w_packed, a.d_w_kernel, a.d_b_kernel, a.d_hidden_slab = ptr(hidden), ptr(w_kernel), ptr(dwp), ptr(dwk), ptr(dbk), ptr(slab)
        a.G, a.bott, a.Og, a.Cg, a.k = G, bott, Og, Cg, k
        check(lib().mtts_gen_params_bwd(ctypes.byref(a), stream_ptr()), 'mtts_gen_params_bwd')
        dhid = _f32(G * bott, device=dev)
        ws = _f32(int(lib().mtts_colsum_workspace_floats(G * bott)), device=dev)
        check(lib().mtts_colsum(ptr(slab), ptr(dhid), nslab, G * bott, G * bott, ptr(ws), stream_ptr()), 'mtts_colsum')
        return dhid.view(G, bott), dwk, dbk, None


def generated_kernel(hidden, w_kernel, b_kernel, Og, Cg, k):
    return GenKernelFn.apply(hidden, w_kernel, b_kernel, (Og, Cg, k))


# ------------------------------------------------------------------------------------------------
# BiLSTM (packed-sequence semantics)
# ------------------------------------------------------------------------------------------------

class BiLstmFn(torch.autograd.Function):
    """Bidirectional LSTM with packed-sequence semantics (reference modules/encoder.py:41-44); x [B, L, C]."""

    @staticmethod
    def forward(ctx, x, lengths, w_ih, w_hh, b_ih, b_hh, w_ih_r, w_hh_r, b_ih_r, b_hh_r):
        require_gpu(x, w_ih)
        B, L, Cin = x.shape
        x_tm = x.transpose(0, 1).contiguous()            # time-major [L, B, C]
        H = w_hh.shape[1]
        dev = x.device
        a = _C.BiLstmArgs()
        a.B, a.L, a.Cin, a.H = B, L, Cin, H
        lengths32 = to_device_async(lengths, dev, torch.int32).contiguous()
        a.x, a.lengths = ptr(x_tm), ptr(lengths32)
        ws = [(w_ih.contiguous(), w_hh.contiguous(), b_ih.contiguous(), b_hh.contiguous()),
              (w_ih_r.contiguous(), w_hh_r.contiguous(), b_ih_r.contiguous(), b_hh_r.contiguous())]
        lib().mtts_bilstm_buffer_elems.restype = ctypes.c_long
        n = lambda field: int(lib().mtts_bilstm_buffer_elems(ctypes.byref(a), 0, field.encode()))      # sizes come from the library
        xproj = [_f32(n('xproj'), device=dev).view(L, B, 4 * H) for _ in range(2)]
        h = [torch.zeros(n('h'), device=dev).view(L + 1, B, H) for _ in range(2)]
        c = [torch.zeros(n('c'), device=dev).view(L + 1, B, H) for _ in range(2)]
        gates = [_f32(n('gates'), device=dev).view(L, B, 4 * H) for _ in range(2)]
        y = _f32(n('y'), device=dev).view(B, L, 2 * H)
        for d in range(2):
            a.w_ih[d], a.w_hh[d], a.b_ih[d], a.b_hh[d] = (t.data_ptr() for t in ws[d])
            a.xproj[d], a.h[d], a.c[d], a.gates[d] = xproj[d].data_ptr(), h[d].data_ptr(), c[d].data_ptr(), gates[d].data_ptr()
        a.y = ptr(y)
        check(lib().mtts_bilstm_fwd(ctypes.byref(a), stream_ptr()), 'bilstm_fwd')
        ctx.save_for_backward(x_tm, lengths32, *ws[0], *ws[1], *h, *c, *gates)
        return y

    @staticmethod
    def backward(ctx, dy):
        from .backward import bilstm_bwd
        return bilstm_bwd(ctx, dy)


def bilstm(x, lengths, params):
    return BiLstmFn.apply(x, lengths, *params)


def grad_reverse_clamp(g, l, c):
    """clamp(g, -c, c) * (-l): gradient-reversal backward (reference modules/classifier.py:16-18)."""
    require_gpu(g)
    g = g.contiguous()
    out = torch.empty_like(g)
    check(lib().mtts_grad_reverse_clamp(ptr(g), ptr(out), ctypes.c_long(g.numel()), ctypes.c_float(l), ctypes.c_float(c),
                                        stream_ptr()), 'grad_reverse_clamp')
    return out
