"""Limits of the group norm / 8-bit checkpoint operators and the bounds of their GPU tests (no GPU needed: nothing may be launched)."""
import ctypes

import pytest
import torch

from multilingual_text_to_speech_amd import _C
from multilingual_text_to_speech_amd import kernels as K
from tests import operator_bounds as B
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


def meta(*shape, dtype=torch.float32):
    return torch.empty(*shape, dtype=dtype, device='meta')


def held(*shape):
    return K.Checkpoint8(meta(*shape, dtype=torch.int8), meta(*shape[:-1], -(-shape[-1] // 32), dtype=torch.uint8))


@pytest.mark.parametrize('big', [2 ** 31 - 1, 2 ** 32 + 1, 2 ** 32 + 5])
def test_sizes_that_pass_32_bits_are_refused(big):
    """2^31 - 1 rows leave no room for a workgroup's row numbers; a C int would take 2^32 + 5 for 5."""
    one = meta(1)
    refused('rows are too many', K.group_norm_act, meta(1, big, 1), one, one, 1)
    refused('samples are too many', K.group_norm_act, meta(big, 1, 1), one, one, 1)
    refused('channels are too many', K.group_norm_act, meta(1, 1, big), meta(big), meta(big), 1)
    refused('channels are too many', K.checkpoint8, meta(1, big))
    refused('rows are too many', K.checkpoint8, meta(big, 1))
    refused('channels are too many', held(1, big).unpack)
    refused('channels are too many', K.conv1d_weight_grad8, held(1, big), meta(1, 1), 1)
    refused('channels are too many', K.conv1d_weight_grad8, held(1, 1), meta(1, big), 1)
    refused('taps are too many', K.conv1d_weight_grad8, held(1, 4, 1), meta(1, 4, 1), 3, dilation=big)
    refused('taps are too many', K.conv1d_weight_grad8, held(1, 4, 1), meta(1, 4, 1), big)
    refused('rows are too many', K.conv_gn_act, meta(1, 4, 1), meta(1, 1, 3), one, one, kernel=3, norm_groups=1, dilation=big)
    refused('rows are too many', K.conv_gn_act, meta(1, big, 1), meta(1, 1, 3), one, one, kernel=3, norm_groups=1)


def test_entry_points_refuse_rows_without_room(library):
    err = lambda: library.mtts_last_error().decode()  # noqa: E731
    a = _C.GroupNormArgs(gamma=4096, beta=4096, mean=4096, rstd=4096, ws=4096, x=4096, y=4096, dy=4096, dx=4096, N=1, L=2 ** 31 - 1, C=1, G=1)
    for f in (library.mtts_group_norm_act_fwd, library.mtts_group_norm_act_bwd):
        assert f(ctypes.byref(a), None) and 'rows are too many' in err()
    assert library.mtts_group_norm_workspace_floats(ctypes.byref(a), 0) == -1
    w = _C.Wgrad8Args(q=4096, q_code=4096, dy=4096, dw=4096, ws=4096, N=1, L=2 ** 31 - 1, I=1, O=1, kernel=1, dilation=1, groups=1)
    assert library.mtts_conv_weight_grad8(ctypes.byref(w), None) and 'rows are too many' in err()
    assert library.mtts_conv_weight_grad8_workspace_floats(ctypes.byref(w)) == -1


def test_lengths_that_are_no_whole_numbers_are_refused():
    x, g = torch.zeros(2, 3, 8), torch.ones(8)
    for lengths in ([1.5, 2.9], [1.0, 2.0], (0.5, 3)):
        refused('int32 or int64', K.group_norm_act, x, g, g, 2, lengths)
        refused('int32 or int64', K.checkpoint8, x, lengths)
    refused('CPU', K.group_norm_act, x, g, g, 2, [1, 3])                      # whole ones get as far as the device
    refused('CPU', K.group_norm_act, x, g, g, 2, (0, 3))
    refused('CPU', K.group_norm_act, x[:0], g, g, 2, [])
    import numpy
    refused('CPU', K.group_norm_act, x, g, g, 2, numpy.array([1, 3]))
    refused('CPU', K.group_norm_act, x, g, g, 2, numpy.array([1, 3], dtype=numpy.uint8))


def test_an_empty_block_input_is_named():
    one = torch.ones(6)
    for shape in ((0, 3, 8), (2, 0, 8), (2, 3, 0)):
        refused('at least one value', K.conv_gn_act, torch.zeros(shape), torch.zeros(6, 8, 5), one, one, kernel=5, norm_groups=2)


# ---- the cases and bounds of the GPU tests --------------------------------------------------------------------------------------------

@pytest.mark.parametrize('case,fp32,bf16', B.FORMS, ids=lambda v: str(v))
def test_the_listed_shapes_reach_their_form(library, case, fp32, bf16):
    assert (B.splits_of(case, torch.float32), B.splits_of(case, torch.bfloat16)) == (fp32, bf16)


@pytest.mark.parametrize('kind', ['dense', 'bits', 'one'])
def test_whole_number_cases_miss_nothing(kind):
    """In float32 the sums are exact; a lost row, and with 17 and 24 bits a lost third plane of dy, changes them."""
    case = (3, 50, 64, 40, 3, 2, 1)
    v, s, dy = B.whole_numbers(case, torch.float32, kind, 1, 'cpu')
    want = B.whole_weight_grad(v, s, dy, 3, 2, 1)
    x = K.Checkpoint8(v, s)
    x = x.values.float() * torch.pow(2.0, x.scales.float() - 127).repeat_interleave(32, -1)[..., :64]
    assert torch.equal(R.weight_grad(x, dy, 3, 2, 1)[0], want) and torch.equal(want.float().double(), want)
    one = torch.einsum('nlo,nlc->oc', dy, x)                                  # in float32
    assert torch.equal(one.double(), want[:, :, 1])
    for r in range(0, 50, 7):
        lost = v.clone()
        lost[1, r] = 0
        assert kind == 'one' and not v[1, r].any() or not torch.equal(B.whole_weight_grad(lost, s, dy, 3, 2, 1), want)
    if kind != 'dense':
        a1 = (dy.view(torch.int32) & -65536).view(torch.float32)
        a2 = ((dy - a1).view(torch.int32) & -65536).view(torch.float32)
        assert not torch.equal(B.whole_weight_grad(v, s, a1 + a2, 3, 2, 1), want)


@pytest.mark.parametrize('offset', [0.0, 100.0, 3000.0])
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('shape', B.LONG, ids=str)
def test_the_bounds_of_group_norm_miss_nothing(shape, dtype, offset):
    """The definition's own result passes; one without either mean, without one of 64 chunks in them, or with one lost in the sums for scale and
    offset does not."""
    if offset and dtype != torch.float32:
        return                                    # the spread is gone in bfloat16
    N, L, C, G = shape
    x, gamma, beta, keep, dy, lens = B.norm_case(shape, dtype, 'tanh', 'cpu', offset=offset)
    ref = B.norm_reference(x, gamma, beta, G, lens, keep, 'tanh', 1.0, dy, False)
    ey, edx, edg, edb = B.norm_bounds(x, gamma, beta, G, ref, dy)
    r = ref['rstd'].repeat_interleave(C // G, -1)[:, None, :]
    assert not B.outside(ref['dx'].to(dtype), ref['dx'], edx).any()
    assert not B.outside(ref['dgamma'].float(), ref['dgamma'], edg).any()
    chunk = torch.arange(L) >= -(-L // 64)                                    # the first of 64 chunks is lost
    m1, m2 = B.norm_means(ref, gamma, G, chunk)
    wrong = {'m1': r * ref['m1'], 'm2': r * ref['xhat_b'] * ref['m2'], 'both': r * (ref['m1'] + ref['xhat_b'] * ref['m2'])}
    if offset < 3000:
        wrong['chunk'] = r * (ref['m1'] - m1 + ref['xhat_b'] * (ref['m2'] - m2))
    for name, off in wrong.items():
        assert B.outside((ref['dx'] + off).to(dtype), ref['dx'], edx).float().mean() > 0.05, name
    if offset == 0:
        for rows in (slice(L // 2, L // 2 + -(-L // 64)), slice(0, L, 100)):          # a chunk, a hundredth of the rows
            assert B.outside((ref['dbeta'] - ref['dz'][0, rows].sum(0)).float(), ref['dbeta'], edb).float().mean() > 0.5
            assert B.outside((ref['dgamma'] - (ref['dz'] * ref['xhat_b'])[0, rows].sum(0)).float(), ref['dgamma'], edg).float().mean() > 0.5
