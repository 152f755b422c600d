"""Group norm, 8-bit checkpoints and their weight gradient on the GPU: what autograd is told, empty inputs, limits, and every form of the
kernels with bounds close enough to miss nothing (tests/operator_bounds.py)."""
import ctypes

import pytest
import torch
from torch.autograd import forward_ad

from multilingual_text_to_speech_amd import _C
from multilingual_text_to_speech_amd import kernels as K
from tests import operator_bounds as B

pytestmark = pytest.mark.gpu
DEV = 'cuda'
F32, BF16 = torch.float32, torch.bfloat16


# ---- autograd -------------------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize('dual', ['x', 'gamma', 'beta'])
@pytest.mark.parametrize('recording', [True, False])
def test_a_forward_mode_tangent_is_refused(dual, recording):
    """There is no forward-mode derivative: the call raises, as linear does, and does not return a result without a tangent."""
    t = {'x': torch.randn(2, 9, 32, device=DEV), 'gamma': torch.rand(32, device=DEV), 'beta': torch.randn(32, device=DEV)}
    plain = K.group_norm_act(t['x'], t['gamma'], t['beta'], 4, act='silu')
    w = torch.randn(8, 32, device=DEV)
    with torch.set_grad_enabled(recording), forward_ad.dual_level():
        assert torch.equal(K.group_norm_act(t['x'], t['gamma'], t['beta'], 4, act='silu'), plain)
        t[dual] = forward_ad.make_dual(t[dual], torch.ones_like(t[dual]))
        with pytest.raises(RuntimeError, match='jvp'):
            K.group_norm_act(t['x'], t['gamma'], t['beta'], 4, act='silu')
        with pytest.raises(RuntimeError, match='jvp'):
            K.linear(forward_ad.make_dual(w, w), w)


def _calls(checkpoint):
    gen = torch.Generator(device=DEV).manual_seed(3)
    normal = lambda *s: torch.randn(*s, generator=gen, device=DEV)  # noqa: E731
    x, w, k, one, zero = normal(2, 9, 32), normal(8, 32), normal(8, 32, 3), torch.ones(8, device=DEV), torch.zeros(8, device=DEV)
    return {'linear': ((x, w), lambda x, w: K.linear(x, w, checkpoint=checkpoint)),
            'conv_bn_act': ((x, k), lambda x, w: K.conv_bn_act(x, w, one, zero, zero.clone(), one.clone(), None, kernel=3, checkpoint=checkpoint)),
            'conv_gn_act': ((x, k), lambda x, w: K.conv_gn_act(x, w, one, zero, kernel=3, norm_groups=2, checkpoint=checkpoint))}


@pytest.mark.parametrize('name', ['linear', 'conv_bn_act', 'conv_gn_act'])
def test_no_second_derivative_from_a_checkpoint(name):
    """Gradients that were asked for with create_graph=True would look like constants."""
    leaves, f = _calls(True)[name]
    leaves = [t.requires_grad_() for t in leaves]
    with pytest.raises(_C.MttsError, match='second derivative'):
        torch.autograd.grad(f(*leaves).square().sum(), leaves, create_graph=True)
    assert all(torch.isfinite(g).all() for g in torch.autograd.grad(f(*leaves).square().sum(), leaves))


@pytest.mark.parametrize('name', ['linear', 'conv_bn_act', 'conv_gn_act'])
def test_nothing_is_packed_where_nothing_is_recorded(name, monkeypatch):
    leaves, f = _calls(True)[name]
    want = f(*[t.clone().requires_grad_() for t in leaves]).detach()
    packs = []
    real = K.checkpoint8
    monkeypatch.setattr(K, 'checkpoint8', lambda *a: packs.append(a) or real(*a))
    assert torch.equal(f(*leaves), want) and not packs                     # no operand requires a gradient
    with torch.no_grad():
        assert torch.equal(f(*[t.clone().requires_grad_() for t in leaves]), want) and not packs
    f(*[t.clone().requires_grad_() for t in leaves])
    assert packs


# ---- empty inputs ---------------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize('shape', [(0, 80), (3, 0, 80)], ids=str)
@pytest.mark.parametrize('act', ['identity', 'relu'])
def test_linear_of_no_rows_from_a_checkpoint(shape, act):
    x, w, b = (torch.randn(*s, device=DEV, requires_grad=True) for s in (shape, (36, 80), (36,)))
    keep = torch.ones(*shape[:-1], 36, dtype=torch.uint8, device=DEV)
    y = K.linear(x, w, b, act, keep, 2.0, checkpoint=True)
    assert y.shape == (*shape[:-1], 36)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), torch.zeros_like(y))
    assert dx.shape == x.shape and dw.shape == w.shape and db.shape == b.shape
    assert not dw.any() and not db.any()


# ---- limits of the weight gradient's three terms ----------------------------------------------------------------------------------------

@pytest.mark.parametrize('dtype', [F32, BF16])
@pytest.mark.parametrize('value', [float('inf'), float('-inf'), float('nan')])
@pytest.mark.parametrize('rows', [40, 7680])                # 128- and 256-wide tiles
def test_a_non_finite_gradient_stays_in_its_output_channel(rows, value, dtype):
    """An infinity: NaN in three terms, the products' own infinities in one; the other channels keep their bits."""
    O, I = (96, 64) if rows == 40 else (512, 2560)
    gen = torch.Generator(device=DEV).manual_seed(5)
    held = K.checkpoint8(torch.randint(1, 100, (1, rows, I), generator=gen, device=DEV).float())
    dy = torch.randn(1, rows, O, generator=gen, device=DEV).to(dtype)
    clean = K.conv1d_weight_grad8(held, dy, 1)
    dy[0, rows - 9, 17] = value
    got = K.conv1d_weight_grad8(held, dy, 1)
    if dtype == BF16 and value == value:
        assert torch.equal(got[17], torch.full_like(got[17], value))          # no 8-bit value of this row is zero
    else:
        assert got[17].isnan().all()
    others = torch.arange(O, device=DEV) != 17
    assert torch.equal(got[others], clean[others]) and torch.isfinite(clean).all()


def test_bits_of_small_gradients():
    """One product per output, with x = 2^106.  The three terms are whole multiples of 2^-133: nothing is lost at magnitudes of 2^-110 and
    more (24 bits), less than 2^-133 below, also where dy is subnormal; a bfloat16 dy is taken as it is."""
    held = K.checkpoint8(torch.full((1, 1, 32), 2.0 ** 106, device=DEV))
    gen = torch.Generator(device=DEV).manual_seed(6)
    for e in range(-149, -100):
        bits = torch.randint(2 ** 23, 2 ** 24, (1, 1, 2048), generator=gen, device=DEV).double()
        dy = (bits * 2.0 ** (e - 23)).float()
        error = K.conv1d_weight_grad8(held, dy, 1)[:, 0, 0].double() * 2.0 ** -106 - dy.double()[0, 0]
        assert error.abs().max() < 2.0 ** -133 and (e < -110 or not error.any())
        half = dy.bfloat16()
        assert torch.equal(K.conv1d_weight_grad8(held, half, 1)[:, 0, 0].double() * 2.0 ** -106, half.double()[0, 0])


# ---- the weight gradient, exactly ---------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize('kind,dtype', [('dense', F32), ('dense', BF16), ('bits', F32), ('one', F32)], ids=lambda v: str(v))
@pytest.mark.parametrize('case', [c for c, _, _ in B.FORMS], ids=str)
def test_weight_grad_of_whole_numbers_is_exact(case, kind, dtype):
    """Every form of the kernel, at split borders and remainders: no row, tap, term or slab may be lost."""
    k, d, g = case[4:]
    v, s, dy = B.whole_numbers(case, dtype, kind, 7, DEV)
    want = B.whole_weight_grad(v, s, dy, k, d, g)
    held = K.Checkpoint8(v, s)
    assert torch.equal(K.conv1d_weight_grad8(held, dy, k, dilation=d, groups=g).double(), want)
    packed = K.conv1d_weight_grad8(held, dy, k, dilation=d, groups=g, packed=True)
    assert torch.equal(packed.double().permute(0, 2, 1), want)


@pytest.mark.parametrize('dtype', [F32, BF16])
@pytest.mark.parametrize('case', [(41, 201, 512, 512, 5, 2, 1), (33, 301, 256, 260, 3, 2, 1)], ids=str)
def test_weight_grad_of_whole_numbers_at_odd_addresses_and_in_bf16_mode(case, dtype):
    """Tensors that start one element behind an aligned address, in both tiles; bf16 mode rounds nothing of small whole numbers."""
    k, d, g = case[4:]
    v, s, dy = B.whole_numbers(case, dtype, 'dense', 8, DEV)
    want = B.whole_weight_grad(v, s, dy, k, d, g)

    def off(t):
        o = torch.empty(t.numel() + 1, dtype=t.dtype, device=DEV)[1:].view(t.shape)
        return o.copy_(t)
    try:
        for mode in ('fp32', 'bf16'):
            _C.set_precision(mode)
            for vv, dd in ((v, dy), (off(v), dy), (v, off(dy)), (off(v), off(dy))):
                assert torch.equal(K.conv1d_weight_grad8(K.Checkpoint8(vv, off(s)), dd, k, dilation=d, groups=g).double(), want)
    finally:
        _C.set_precision('fp32')


@pytest.mark.parametrize('dilation', [1 << 20, 2 ** 31 - 1, 2 ** 32, 2 ** 32 + 1])
def test_one_tap_has_no_dilation(dilation):
    v, s, dy = B.whole_numbers((2, 37, 64, 96, 1, 1, 1), F32, 'dense', 9, DEV)
    got = K.conv1d_weight_grad8(K.Checkpoint8(v, s), dy, 1, dilation=dilation)
    assert torch.equal(got.double(), B.whole_weight_grad(v, s, dy, 1, 1, 1))


def among(t, poison, lead=0):
    """t, lead elements behind an aligned address, with the poison in front of it and behind it."""
    store = torch.full((t.numel() + 64 + lead,), poison, dtype=t.dtype, device=DEV)
    o = store[32 + lead:32 + lead + t.numel()].view(t.shape)
    return o.copy_(t)


@pytest.mark.parametrize('lead', [0, 1])
@pytest.mark.parametrize('dtype', [F32, BF16])
@pytest.mark.parametrize('case', [(1, 7, 64, 33, 1, 1, 1), (1, 6, 81, 559, 1, 3, 1), (3, 5, 35, 33, 3, 1, 1), (5, 17, 60, 45, 3, 2, 3), (33, 301, 257, 259, 3, 2, 1),
                                  (23, 357, 510, 511, 5, 1, 1), (41, 201, 512, 512, 5, 2, 1), (1, 9001, 40, 35, 2, 1, 1)], ids=str)
def test_weight_grad_reads_nothing_of_its_neighbours(case, dtype, lead):
    """NaN next to the gradient, exponents that stand for NaN next to the checkpoint's: also where a tensor ends inside a word."""
    k, d, g = case[4:]
    v, s, dy = B.whole_numbers(case, dtype, 'dense', 11, DEV)
    want = B.whole_weight_grad(v, s, dy, k, d, g)
    got = K.conv1d_weight_grad8(K.Checkpoint8(among(v, 127, lead), among(s, 255, lead)), among(dy, float('nan'), lead), k, dilation=d, groups=g)
    assert torch.equal(got.double(), want)


# ---- group norm, with bounds that a missing mean, chunk or row exceeds ------------------------------------------------------------------------

def close(got, want, bound, what):
    bad = B.outside(got, want, bound)
    assert not bad.any(), f'{what}: {int(bad.sum())} of {bad.numel()} values are off, the first by {(got.double() - want).abs()[bad][0].item():.3g}, bound {bound.expand_as(bad)[bad][0].item():.3g}'


def check_norm(shape, dtype, act, ckpt, lengths, mask, offset=0.0):
    G, scale = shape[3], 2.0 if mask else 1.0
    x, gamma, beta, keep, dy, lens = B.norm_case(shape, dtype, act, DEV, 3, lengths, mask, offset)
    ref = B.norm_reference(x, gamma, beta, G, lens, keep, act, scale, dy, ckpt)
    ey, edx, edg, edb = B.norm_bounds(x, gamma, beta, G, ref, dy, scale)
    leaves = [t.requires_grad_() for t in (x, gamma, beta)]
    y = K.group_norm_act(*leaves, G, lens, keep, act=act, mask_scale=scale, checkpoint=ckpt)
    dx, dgamma, dbeta = torch.autograd.grad(y, leaves, dy)
    close(y.detach(), ref['y'], ey, 'y')
    close(dx, ref['dx'], edx, 'dx')
    close(dgamma, ref['dgamma'], edg, 'dgamma')
    close(dbeta, ref['dbeta'], edb, 'dbeta')


@pytest.mark.parametrize('ckpt', [False, True])
@pytest.mark.parametrize('dtype', [F32, BF16])
@pytest.mark.parametrize('shape', B.NORMS, ids=str)
def test_every_form_of_group_norm(shape, dtype, ckpt):
    """Ragged where there are several samples; dropout without a checkpoint."""
    N, L = shape[:2]
    act = ('tanh', 'silu')[B.NORMS.index(shape) % 2]
    check_norm(shape, dtype, act, ckpt, [L, L - L // 3, 1][:N] if N > 1 else None, not ckpt)


@pytest.mark.parametrize('offset', [100.0, 3000.0])
@pytest.mark.parametrize('shape', [s for s in B.LONG if s[0] * s[1] * s[2] < 300000], ids=str)
def test_group_norm_of_an_offset(shape, offset):
    check_norm(shape, F32, 'tanh', False, None, False, offset)


@pytest.mark.parametrize('kind', ['plain', 'highway', 'generated', 'generated highway'])
def test_every_model_block_trains_from_checkpoints(kind, monkeypatch):
    """activation_checkpoint_bits = 8: the same output; gradients within the rounding of the 8-bit values, 2 * 2^-7 of a block's largest value
    in one element and far less over a tensor (bounded as in the batch norm block's test)."""
    from multilingual_text_to_speech_amd.modules import layers as M
    from multilingual_text_to_speech_amd.params.params import Params as hp
    torch.manual_seed(2)
    cls = {'plain': M.ConvBlock, 'highway': M.HighwayConvBlock, 'generated': M.ConvBlockGenerated, 'generated highway': M.HighwayConvBlockGenerated}[kind]
    generated = 'generated' in kind
    block = cls(*((6, 4) if generated else ()), 60, 60, 3, 0.0, 'tanh', 2, 3 if generated else 1).to(DEV)
    x, dy = torch.randn(5, 31, 60, device=DEV), torch.randn(5, 31, 60, device=DEV)
    e = (torch.randn(3, 6, device=DEV),) if generated else ()
    out = {}
    for bits in (32, 8):
        monkeypatch.setattr(hp, 'activation_checkpoint_bits', bits, raising=False)
        xr = x.clone().requires_grad_()
        y = block(*e, xr)
        out[bits] = (y.detach(), torch.autograd.grad(y, [xr, *block.parameters()], dy, allow_unused=True))
    assert torch.equal(out[32][0], out[8][0])
    seen = 0
    for a, b in zip(out[8][1], out[32][1]):
        assert (a is None) == (b is None)
        if a is not None:
            seen += 1
            rel = ((a - b).norm() / b.norm()).item()
            assert a.shape == b.shape and 0 < rel < 0.06, rel
    assert seen >= 4


# ---- neighbours in memory: nothing is read of them, nothing is written to them -------------------------------------------------------------

GUARD = 64


def hidden(*shape, dtype, lead, fill):
    """A tensor to write to, GUARD elements of `fill` in front of it and behind it, and a check that they are still there."""
    n = 1
    for v in shape:
        n *= v
    store = torch.full((n + 2 * GUARD + lead,), fill, dtype=dtype, device=DEV)
    view = store[GUARD + lead:GUARD + lead + n].view(shape)
    rest = torch.ones(store.shape, dtype=torch.bool, device=DEV)
    rest[GUARD + lead:GUARD + lead + n] = False

    def untouched():
        torch.cuda.synchronize()
        return torch.equal(store[rest], torch.full_like(store[rest], fill))
    return view, untouched


# widths of whole vectors and odd ones, rows that end inside a checkpoint block, strips that cut groups, long samples
@pytest.mark.parametrize('lead', [0, 1])
@pytest.mark.parametrize('dtype', [F32, BF16])
@pytest.mark.parametrize('shape', [(3, 5, 80, 8), (2, 61, 33, 3), (3, 300, 80, 8), (2, 70, 48, 2), (2, 600, 64, 4), (1, 3001, 40, 2), (1, 3001, 37, 1), (2, 17, 4100, 2), (5, 1, 7, 7)], ids=str)
def test_group_norm_keeps_to_its_tensors(shape, dtype, lead):
    N, L, C, G = shape
    x, gamma, beta, keep, dy, lens = B.norm_case(shape, dtype, 'tanh', DEV, 4, [L, L - L // 3, 0, 1, 1][:N], True)
    nan, nb = float('nan'), -(-C // 32)
    plain = [t.clone().requires_grad_() for t in (x, gamma, beta)]
    y = K.group_norm_act(*plain, G, lens, keep, act='tanh', mask_scale=2.0)
    want = (y.detach(), *torch.autograd.grad(y, plain, dy))
    held = K.checkpoint8(x, lens)
    xs, gs, bs, ks, ds = among(x, nan, lead), among(gamma, nan, lead), among(beta, nan, lead), among(keep, 1, lead), among(dy, nan, lead)
    outs = {'y': hidden(N, L, C, dtype=dtype, lead=lead, fill=7), 'dx': hidden(N, L, C, dtype=dtype, lead=lead, fill=7),
            'mean': hidden(N, G, dtype=F32, lead=lead, fill=7), 'rstd': hidden(N, G, dtype=F32, lead=lead, fill=7),
            'q': hidden(N, L, C, dtype=torch.int8, lead=lead, fill=7), 'code': hidden(N, L, nb, dtype=torch.uint8, lead=lead, fill=7),
            'dgamma': hidden(C, dtype=F32, lead=lead, fill=7), 'dbeta': hidden(C, dtype=F32, lead=lead, fill=7)}
    at = {k: v[0].data_ptr() for k, v in outs.items()}
    li = among(lens.int(), 2 ** 30, lead)
    a = _C.GroupNormArgs(xs.data_ptr(), gs.data_ptr(), bs.data_ptr(), li.data_ptr(), ks.data_ptr(), at['y'], at['mean'], at['rstd'], at['q'], at['code'], None,
                         N, L, C, G, K._DTYPE[dtype], K.GN_ACT['tanh'], 1e-5, 2.0, ds.data_ptr(), at['dx'], at['dgamma'], at['dbeta'])

    def call(entry, backward):
        n = _C.lib().mtts_group_norm_workspace_floats(ctypes.byref(a), backward)
        ws, intact = hidden(n, dtype=F32, lead=0, fill=7)
        a.ws = ws.data_ptr()
        _C.check(entry(ctypes.byref(a), _C.stream_ptr()), 'group norm')
        assert intact() and all(u() for _, u in outs.values())
    call(_C.lib().mtts_group_norm_act_fwd, 0)
    if lead == 0:                                # another alignment may sum in another order
        assert torch.equal(outs['y'][0], want[0])
    ref = B.norm_reference(x, gamma, beta, G, lens, keep, 'tanh', 2.0, dy, False)
    bounds = B.norm_bounds(x, gamma, beta, G, ref, dy, 2.0)
    close(outs['y'][0], ref['y'], bounds[0], 'y')
    assert torch.equal(outs['q'][0], held.values) and torch.equal(outs['code'][0], held.scales)
    a.q = a.q_code = None                        # the backward from x
    call(_C.lib().mtts_group_norm_act_bwd, 1)
    for got, w, e in zip(('dx', 'dgamma', 'dbeta'), want[1:], bounds[1:]):
        assert lead or torch.equal(outs[got][0], w)
        close(outs[got][0], ref[got], e, got)
    qs, cs = among(held.values, 127, lead), among(held.scales, 255, lead)
    a.q, a.q_code, a.x = qs.data_ptr(), cs.data_ptr(), None
    call(_C.lib().mtts_group_norm_act_bwd, 1)
    ref = B.norm_reference(x, gamma, beta, G, lens, keep, 'tanh', 2.0, dy, True)
    for got, e in zip(('dx', 'dgamma', 'dbeta'), B.norm_bounds(x, gamma, beta, G, ref, dy, 2.0)[1:]):
        close(outs[got][0], ref[got], e, got)


@pytest.mark.parametrize('lead', [0, 1, 3])
@pytest.mark.parametrize('dtype', [F32, BF16])
@pytest.mark.parametrize('shape', [(1, 1, 1), (2, 3, 33), (5, 37, 80), (3, 11, 31), (2, 100, 512), (130, 1, 39), (3, 211, 1285)], ids=str)
def test_checkpoints_keep_to_their_tensors(shape, dtype, lead):
    N, L, C = shape
    gen = torch.Generator(device=DEV).manual_seed(12)
    x = torch.randn(*shape, generator=gen, device=DEV).to(dtype)
    lens = torch.randint(0, L + 1, (N,), generator=gen, device=DEV, dtype=torch.int32)
    held = K.checkpoint8(x, lens)
    q, q_intact = hidden(*shape, dtype=torch.int8, lead=lead, fill=7)
    code, code_intact = hidden(N, L, -(-C // 32), dtype=torch.uint8, lead=lead, fill=7)
    back, back_intact = hidden(*shape, dtype=dtype, lead=lead, fill=7)
    xs, li = among(x, float('nan'), lead), among(lens, 2 ** 30, lead)
    _C.check(_C.lib().mtts_checkpoint8_pack(xs.data_ptr(), li.data_ptr(), q.data_ptr(), code.data_ptr(), N, L, C, K._DTYPE[dtype], _C.stream_ptr()), 'pack')
    _C.check(_C.lib().mtts_checkpoint8_unpack(q.data_ptr(), code.data_ptr(), back.data_ptr(), N * L, C, K._DTYPE[dtype], _C.stream_ptr()), 'unpack')
    assert q_intact() and code_intact() and back_intact()
    assert torch.equal(q, held.values) and torch.equal(code, held.scales) and torch.equal(back, held.unpack())


@pytest.mark.parametrize('packed', [0, 1])
@pytest.mark.parametrize('dtype', [F32, BF16])
@pytest.mark.parametrize('case', [(1, 7, 64, 33, 1, 1, 1), (5, 17, 60, 45, 3, 2, 3), (33, 301, 257, 259, 3, 2, 1), (23, 357, 510, 511, 5, 1, 1), (64, 120, 512, 512, 5, 1, 1),
                                  (64, 600, 32, 64, 3, 1, 1), (2, 400, 8, 8, 2500, 1, 1)], ids=str)
def test_weight_grad_keeps_to_its_tensors(case, dtype, packed):
    N, L, I, O, k, d, g = case
    v, s, dy = B.whole_numbers(case, dtype, 'dense', 13, DEV)
    want = B.whole_weight_grad(v, s, dy, k, d, g)
    dw, intact = hidden(*((O, k, I // g) if packed else (O, I // g, k)), dtype=F32, lead=1, fill=7)
    a = _C.Wgrad8Args(v.data_ptr(), s.data_ptr(), dy.data_ptr(), dw.data_ptr(), None, N, L, I, O, k, d, g, K._DTYPE[dtype], packed, 0)
    ws, ws_intact = hidden(_C.lib().mtts_conv_weight_grad8_workspace_floats(ctypes.byref(a)), dtype=F32, lead=0, fill=7)
    a.ws = ws.data_ptr()
    _C.check(_C.lib().mtts_conv_weight_grad8(ctypes.byref(a), _C.stream_ptr()), 'weight gradient')
    assert intact() and ws_intact()
    assert torch.equal((dw.permute(0, 2, 1) if packed else dw).double(), want)


@pytest.mark.parametrize('name', ['linear', 'conv_bn_act', 'conv_gn_act'])
def test_blocks_from_checkpoints_captured_and_replayed(name):
    """Forward and backward in one graph, replayed with eager work between: the eager bits each time."""
    (x, w), f = _calls(True)[name]

    def step(a, b):
        leaves = [a.detach().requires_grad_(), b.detach().requires_grad_()]
        y = f(*leaves)
        return [y.detach(), *torch.autograd.grad(y, leaves, torch.ones_like(y))]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(x, w)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(x, w)
    gen = torch.Generator(device=DEV).manual_seed(14)
    for _ in range(4):
        x.copy_(torch.randn(x.shape, generator=gen, device=DEV))
        w.copy_(torch.randn(w.shape, generator=gen, device=DEV))
        want = step(x, w)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))
        assert all(torch.equal(a, b) for a, b in zip(step(x, w), want))
