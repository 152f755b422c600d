"""Refusals of the group norm / 8-bit checkpoint operators (no GPU needed: nothing may be launched), and the 64-bit definitions
that their GPU tests use, against torch and against differences."""
import ctypes

import pytest
import torch

from multilingual_text_to_speech_amd import _C
from multilingual_text_to_speech_amd import kernels as K
from tests import operator_refs as R


@pytest.fixture(scope='module')
def library():
    import os
    if not os.path.exists(_C.LIB_PATH):
        from multilingual_text_to_speech_amd.build import build
        build()
    return _C.lib()


def refused(match, f, *a, **kw):
    with pytest.raises(_C.MttsError, match=match):
        f(*a, **kw)


def test_struct_mirrors_of_the_new_blocks(library):
    assert library.mtts_sizeof_struct(16) == ctypes.sizeof(_C.GroupNormArgs)
    assert library.mtts_sizeof_struct(17) == ctypes.sizeof(_C.Wgrad8Args)


def test_group_norm_refusals():
    x, g = torch.zeros(2, 3, 8), torch.ones(8)
    refused('CPU', K.group_norm_act, x, g, g, 2)
    refused('float16', K.group_norm_act, x.half(), g, g, 2)
    refused(r'\[N, L, C\]', K.group_norm_act, x[0], g, g, 2)
    refused('groups', K.group_norm_act, x, g, g, 3)
    refused('groups', K.group_norm_act, x, g, g, 0)
    refused('activation', K.group_norm_act, x, g, g, 2, act='gelu')
    refused('gamma', K.group_norm_act, x, g[:4], g, 2)
    refused('beta', K.group_norm_act, x, g, g.bfloat16(), 2)
    refused('mask', K.group_norm_act, x, g, g, 2, None, torch.ones(2, 3, 1, dtype=torch.uint8))
    refused('mask', K.group_norm_act, x, g, g, 2, None, torch.ones(2, 3, 8))
    refused('lengths', K.group_norm_act, x, g, g, 2, torch.tensor([1, 2, 3]))
    refused('lengths', K.group_norm_act, x, g, g, 2, torch.tensor([1., 2.]))
    refused('lengths run', K.group_norm_act, x, g, g, 2, torch.tensor([1, 4]))
    refused('lengths run', K.group_norm_act, x, g, g, 2, [-1, 2])


def test_checkpoint_refusals():
    x = torch.zeros(2, 3, 40)
    v, s = torch.zeros(2, 3, 40, dtype=torch.int8), torch.ones(2, 3, 2, dtype=torch.uint8)
    refused('CPU', K.checkpoint8, x)
    refused('float64', K.checkpoint8, x.double())
    refused('lengths need', K.checkpoint8, x[0], [1, 1])
    refused('lengths run', K.checkpoint8, x, [1, 5])
    refused('one channel', K.checkpoint8, torch.zeros(3, 0))
    refused('too many', K.checkpoint8, torch.zeros(1, 1).expand(2 ** 31, 1))
    refused('too many', K.conv1d_weight_grad8, K.Checkpoint8(torch.empty(2 ** 31, 1, dtype=torch.int8, device='meta'), torch.empty(2 ** 31, 1, dtype=torch.uint8, device='meta')),
            torch.empty(2 ** 31, 1, device='meta'), 1)
    refused('int8', K.Checkpoint8, v.to(torch.uint8), s)
    refused('int8', K.Checkpoint8, v, s.to(torch.int8))
    refused('shape', K.Checkpoint8, v, s[..., :1])
    refused('dtype', K.Checkpoint8, v, s, torch.float16)
    held = K.Checkpoint8(v, s)
    assert held.nbytes == 2 * 3 * 42 and held.shape == (2, 3, 40)
    refused('CPU', held.unpack)
    refused('dtype', held.unpack, torch.float64)


def test_weight_grad_refusals():
    held = K.Checkpoint8(torch.zeros(2, 3, 40, dtype=torch.int8), torch.ones(2, 3, 2, dtype=torch.uint8))
    dy = torch.zeros(2, 3, 10)
    refused('CPU', K.conv1d_weight_grad8, held, dy, 3)
    refused('float16', K.conv1d_weight_grad8, held, dy.half(), 3)
    refused('belong', K.conv1d_weight_grad8, held, dy[:, :2], 3)
    refused('groups', K.conv1d_weight_grad8, held, dy, 3, groups=4)
    for bad in (dict(kernel=0), dict(kernel=3, dilation=0), dict(kernel=3, groups=0)):
        refused('whole numbers', K.conv1d_weight_grad8, held, dy, **bad)
    flat = K.Checkpoint8(held.values[0], held.scales[0])
    refused('belong', K.conv1d_weight_grad8, flat, dy[0], 3)            # a kernel needs to know where a sample ends


def test_conv_gn_refusals():
    x, w, g = torch.zeros(2, 3, 8), torch.zeros(6, 8, 5), torch.ones(6)
    refused('CPU', K.conv_gn_act, x, w, g, g, kernel=5, norm_groups=2)
    refused('belong', K.conv_gn_act, x, w, g, g, kernel=3, norm_groups=2)
    refused('belong', K.conv_gn_act, x, w, g, g, kernel=5, norm_groups=2, groups=2)
    refused('float32', K.conv_gn_act, x.bfloat16(), w, g, g, kernel=5, norm_groups=2)
    refused('groups', K.conv_gn_act, x, w, g, g, kernel=5, norm_groups=4)


def test_entry_points_refuse_before_they_launch(library):
    """The C entries check shapes, types and pointers themselves: error text, nothing launched (there is no GPU here)."""
    err = lambda: library.mtts_last_error().decode()  # noqa: E731
    p = ctypes.c_void_p(4096)
    a = _C.GroupNormArgs(gamma=4096, beta=4096, mean=4096, rstd=4096, ws=4096, x=4096, y=4096, N=2, L=3, C=8, G=3)
    assert library.mtts_group_norm_act_fwd(ctypes.byref(a), None) and 'multiple of 3 groups' in err()
    a.G, a.dtype = 2, 7
    assert library.mtts_group_norm_act_fwd(ctypes.byref(a), None) and 'dtype 7' in err()
    a.dtype, a.act = 0, 9
    assert library.mtts_group_norm_act_bwd(ctypes.byref(a), None) and 'activation 9' in err()
    a.act, a.y = 0, None
    assert library.mtts_group_norm_act_fwd(ctypes.byref(a), None) and 'missing tensor' in err()
    assert library.mtts_group_norm_act_bwd(ctypes.byref(a), None) and 'missing tensor' in err()
    a.y, a.q = 4096, 4096                                           # values without their exponents
    assert library.mtts_group_norm_act_fwd(ctypes.byref(a), None) and 'missing tensor' in err()
    a.N, a.q = 0, None
    assert library.mtts_group_norm_act_fwd(ctypes.byref(a), None) and 'empty' in err()
    assert library.mtts_group_norm_workspace_floats(ctypes.byref(a), 0) == -1
    a.N, a.L, a.ws = 2, 100000, None                                # too long for one workgroup: a workspace is needed
    assert library.mtts_group_norm_workspace_floats(ctypes.byref(a), 0) > 0
    assert library.mtts_group_norm_act_fwd(ctypes.byref(a), None) and 'workspace' in err()
    a.dy = a.dx = 4096
    assert library.mtts_group_norm_act_bwd(ctypes.byref(a), None) and 'workspace' in err()
    a.N, a.C, a.G = 1 << 30, 64, 1
    assert library.mtts_group_norm_act_fwd(ctypes.byref(a), None) and 'too many' in err()
    assert library.mtts_checkpoint8_pack(p, None, p, None, 1, 1, 1, 0, None) and 'missing tensor' in err()
    assert library.mtts_checkpoint8_pack(p, None, p, p, 1, 0, 1, 0, None) and 'bad shape' in err()
    assert library.mtts_checkpoint8_pack(p, None, p, p, 2 ** 30, 2 ** 30, 64, 0, None) and 'too many' in err()
    assert library.mtts_checkpoint8_unpack(p, p, p, ctypes.c_long(1), 1, 5, None) and 'bad shape' in err()
    w = _C.Wgrad8Args(q=4096, q_code=4096, dy=4096, dw=4096, N=1, L=4, I=6, O=6, kernel=3, dilation=1, groups=4)
    assert library.mtts_conv_weight_grad8_workspace_floats(ctypes.byref(w)) == -1 and '4 groups' in err()
    assert library.mtts_conv_weight_grad8(ctypes.byref(w), None) and '4 groups' in err()
    w.groups, w.dilation = 1, 0
    assert library.mtts_conv_weight_grad8(ctypes.byref(w), None) and 'dilation 0' in err()
    w.dilation, w.dw = 1, None
    assert library.mtts_conv_weight_grad8(ctypes.byref(w), None) and 'missing tensor' in err()
    w.dw, w.kernel, w.dilation = 4096, 2 ** 20, 2 ** 20
    assert library.mtts_conv_weight_grad8(ctypes.byref(w), None) and 'too large' in err()


def test_block_option_refuses_other_widths(monkeypatch):
    from multilingual_text_to_speech_amd.modules import layers
    from multilingual_text_to_speech_amd.params.params import Params as hp
    assert not layers._checkpoint()
    monkeypatch.setattr(hp, 'activation_checkpoint_bits', 8, raising=False)
    assert layers._checkpoint()
    monkeypatch.setattr(hp, 'activation_checkpoint_bits', 4, raising=False)
    with pytest.raises(ValueError, match='8 or 32'):
        layers._checkpoint()


# ---- the definitions ------------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize('act', list(R.ACTS))
def test_definition_equals_torch_and_differences(act):
    gen = torch.Generator().manual_seed(3)
    N, L, C, G = 2, 5, 12, 3
    x = torch.randn(N, L, C, generator=gen, dtype=torch.float64).requires_grad_()
    gamma = torch.randn(C, generator=gen, dtype=torch.float64).requires_grad_()
    beta = torch.randn(C, generator=gen, dtype=torch.float64).requires_grad_()
    dy = torch.randn(N, L, C, generator=gen, dtype=torch.float64)
    y = R.ACTS[act](torch.nn.functional.group_norm(x.transpose(1, 2), G, gamma, beta, 1e-5)).transpose(1, 2)
    grads = torch.autograd.grad(y, (x, gamma, beta), dy)
    ref = R.group_norm(x, gamma, beta, G, act=act, dy=dy)
    torch.testing.assert_close(ref['y'], y.detach(), rtol=0, atol=1e-13)
    for name, g in zip(('dx', 'dgamma', 'dbeta'), grads):
        torch.testing.assert_close(ref[name], g, rtol=0, atol=1e-11)
    # along one direction: (f(x + h v) - f(x - h v)) / 2h = <dx, v> + O(h^2)
    v, h = torch.randn(x.shape, generator=gen, dtype=torch.float64), 1e-5
    f = lambda t: (R.group_norm(t, gamma, beta, G, act=act)['y'] * dy).sum()  # noqa: E731
    assert abs((f(x + h * v) - f(x - h * v)) / (2 * h) - (ref['dx'] * v).sum()) < 1e-6


def test_definition_ignores_what_lies_behind_the_lengths():
    x = torch.randn(3, 6, 8)
    lengths = torch.tensor([6, 0, 2])
    a = R.group_norm(x, torch.ones(8), torch.zeros(8), 2, lengths, dy=torch.ones_like(x))
    x[1], x[2, 2:] = float('nan'), float('inf')
    b = R.group_norm(x, torch.ones(8), torch.zeros(8), 2, lengths, dy=torch.ones_like(x))
    for k in ('y', 'dx', 'dgamma', 'dbeta'):
        assert torch.equal(a[k], b[k]) and torch.isfinite(a[k]).all()
    assert not a['y'][1].any() and not a['dx'][2, 2:].any()


def test_round_trip_definition():
    x = torch.tensor([[127.4, -127.5, 1.0, 0.5, 1.5, 0.0]])
    q, code, v = R.round_trip(x)
    assert code.tolist() == [[128]] and q.tolist() == [[64, -64, 0, 0, 1, 0]]           # 127.5 rounds to 128: the step doubles
    q, code, v = R.round_trip(x[:, :1])
    assert code.tolist() == [[127]] and q.tolist() == [[127]]
    q, code, v = R.round_trip(torch.tensor([[1.0, float('inf')]]))
    assert code.tolist() == [[255]] and v.isnan().all() and not q.any()
    q, code, v = R.round_trip(torch.tensor([[torch.finfo(torch.float32).max, -1.0]]))
    assert code.tolist() == [[249]] and q.tolist() == [[63, 0]]
    y = torch.randn(40, 77)
    q, code, v = R.round_trip(y)
    assert ((v - y).abs() <= torch.pow(2.0, code.double() - 128).repeat_interleave(32, -1)[:, :77]).all()
    assert torch.equal(v.bfloat16().double(), v)                                         # exact in bfloat16


def test_entry_points_take_whole_addresses(library):
    """Addresses are passed as Python numbers: every entry that takes one has to say that it is a pointer (a bare number is a C int)."""
    for name in ('mtts_group_norm_workspace_floats', 'mtts_group_norm_act_fwd', 'mtts_group_norm_act_bwd', 'mtts_conv_weight_grad8',
                 'mtts_conv_weight_grad8_workspace_floats', 'mtts_checkpoint8_pack', 'mtts_checkpoint8_unpack'):
        f = getattr(library, name)
        assert f.argtypes is not None and f.argtypes[0] is ctypes.c_void_p, name
    a = _C.GroupNormArgs(gamma=4096, beta=4096, mean=4096, rstd=4096, x=4096, y=4096, N=2, L=3, C=8, G=2)
    assert library.mtts_group_norm_workspace_floats(ctypes.addressof(a), 0) == 0
