"""Cases and bounds of the group norm / 8-bit checkpoint operators that leave no room for a lost row, a lost term or an untested form:
integers whose sums are exact, and elementwise bounds from the roundings that an element's own terms make."""
import ctypes

import torch

from multilingual_text_to_speech_amd import _C
from multilingual_text_to_speech_amd import kernels as K

# ---- weight gradient: sums of whole numbers below 2^24 are exact in fp32, in any order ---------------------------------------------------

# (N, L, I, O, kernel, dilation, groups), splits for fp32 and for bf16 gradients (they tell the forms apart: see the comments)
FORMS = [
    # 256 x 256 tiles (128 x 128 would take 3, 3, 16, 1, 1, 2, 1, 6 and 1 splits)
    ((64, 120, 512, 512, 5, 1, 1), 12, 12),
    ((41, 201, 512, 512, 5, 2, 1), 12, 12),          # 8241 rows: the last split ends inside a step
    ((64, 600, 512, 512, 1, 1, 1), 64, 64),
    ((13, 1000, 1022, 1022, 3, 1, 1), 4, 4),         # quads at any byte
    ((7, 1171, 511, 1278, 3, 3, 1), 7, 7),
    ((64, 119, 1024, 1280, 3, 9, 2), 7, 7),          # groups
    ((11, 1001, 1021, 509, 5, 2, 1), 6, 6),
    ((5, 3000, 252, 500, 5, 1, 1), 25, 25),
    ((16, 433, 1280, 2560, 5, 9, 5), 5, 5),
    # 128 x 128 tiles: one split, a few, more than sixteen slabs to a sum
    ((16, 120, 512, 512, 5, 1, 1), 3, 3),
    ((2, 37, 64, 96, 5, 1, 1), 1, 1),
    ((12, 133, 1280, 2560, 3, 9, 5), 2, 2),
    ((33, 301, 257, 259, 3, 2, 1), 12, 12),
    ((64, 600, 32, 64, 3, 1, 1), 200, 200),
    ((1, 9001, 40, 36, 2, 1, 1), 47, 47),
    # no pipeline: taps far apart (only one of them inside a sample), rows too wide for 32-bit offsets in a split (1100000 channels: fp32)
    ((6, 70, 100, 72, 3, 1 << 23, 1), 2, 2),
    ((2, 40, 4, 1100000, 3, 1, 1), 1, 1),
    ((2, 40, 4400000, 2, 3, 1, 1), 1, 1),
]


def splits_of(case, dtype):
    """Partial tiles that a call with aligned tensors asks its workspace for."""
    N, L, I, O, k, d, g = case
    a = _C.Wgrad8Args(q=4096, q_code=4096, dy=4096, dw=4096, N=N, L=L, I=I, O=O, kernel=k, dilation=d, groups=g, dtype=K._DTYPE[dtype])
    n = _C.lib().mtts_conv_weight_grad8_workspace_floats(ctypes.byref(a))
    assert n >= 0 and n % (O * k * (I // g)) == 0
    return n // (O * k * (I // g)) or 1


def whole_numbers(case, dtype, kind, seed, device):
    """values, scales, dy.  dense: every row has its products, scales of 1/2, 1 and 2; sums stay below 3 * 2 * 7 rows, half units.
    bits: dy of 17 bits (three planes of eight), 120 values of +-1 to a column of x.  one: dy of 24 bits, one value of +-1 to a column."""
    N, L, I, O, k, d, g = case
    rows = N * L
    gen = torch.Generator(device=device).manual_seed(seed)
    blocks = -(-I // 32)
    draw = lambda lo, hi, *shape, **kw: torch.randint(lo, hi, shape, generator=gen, device=device, **kw)  # noqa: E731
    if kind == 'dense':
        assert 2 * 42 * rows < 2 ** 24
        return draw(-3, 4, N, L, I, dtype=torch.int8), draw(126, 129, N, L, blocks, dtype=torch.uint8), draw(-7, 8, N, L, O).to(dtype)
    assert dtype == torch.float32
    n, bits = (min(120, rows), 17) if kind == 'bits' else (1, 24)
    assert n * 2 ** bits <= 2 ** 24
    values = torch.zeros(rows, I, dtype=torch.int8, device=device)
    at = (draw(0, rows, 1, I) + torch.arange(n, device=device)[:, None] * (rows // n)) % rows          # n rows of a column, spread evenly
    values.scatter_(0, at, 2 * draw(0, 2, n, I, dtype=torch.int8) - 1)
    dy = (draw(2 ** (bits - 1), 2 ** bits, N, L, O) | 1) * (2 * draw(0, 2, N, L, O) - 1)
    return values.view(N, L, I), torch.full((N, L, blocks), 127, dtype=torch.uint8, device=device), dy.float()


def whole_weight_grad(values, scales, dy, k, d, g):
    """The definition tap by tap in 64 bits: exact."""
    N, L, I = values.shape
    O, Og, Cg = dy.shape[-1], dy.shape[-1] // g, I // g
    x = values.double() * torch.tensor([2.0 ** (e - 127) for e in range(120, 136)], dtype=torch.float64, device=values.device)[scales.long() - 120].repeat_interleave(32, -1)[..., :I]
    dy = dy.double()
    out = torch.zeros(O, Cg, k, dtype=torch.float64, device=values.device)
    for t in range(k):
        shift = t * d - (k - 1) * d // 2
        lo, hi = max(0, -shift), min(L, L - shift)
        for i in range(g if lo < hi else 0):
            a = dy[:, lo:hi, i * Og:(i + 1) * Og].reshape(-1, Og).t().contiguous()
            out[i * Og:(i + 1) * Og, :, t] = a @ x[:, lo + shift:hi + shift, i * Cg:(i + 1) * Cg].reshape(-1, Cg).contiguous()
    return out


# ---- group norm ---------------------------------------------------------------------------------------------------------------------------

# (N, L, C, G).  Resident strips of 1, 4, 8, 10, 12 and 16 rows a thread in both types and directions, with vectors that straddle groups (ten
# channels to a group) and without; two passes with chunks, with a group wider than a workgroup, one value at a time
NORMS = [(3, 5, 80, 8), (2, 200, 80, 8), (2, 230, 80, 8), (2, 250, 80, 8), (3, 300, 80, 8), (2, 480, 80, 8), (2, 700, 80, 8), (3, 800, 80, 8),
         (2, 900, 80, 8), (2, 1100, 80, 8), (3, 1400, 80, 8), (1, 1800, 80, 8), (2, 7000, 80, 8), (1, 5000, 40, 2),
         (2, 400, 512, 16), (2, 500, 512, 16), (2, 600, 512, 16), (2, 700, 512, 16), (2, 1000, 512, 16), (2, 1300, 512, 16), (2, 2000, 512, 16),
         (1, 2049, 256, 2), (2, 1025, 128, 4), (1, 1500, 64, 4), (2, 600, 511, 7), (1, 70, 4100, 2), (1, 20, 4101, 1)]
LONG = [s for s in NORMS if s[1] >= 1000 or s[2] % 4]
ADDS = 256          # additions that a term of any of these sums passes through, at most (a thread's rows, its workgroup's, its chunks')


def norm_case(shape, dtype, act, device, seed=1, lengths=None, mask=False, offset=0.0):
    """As an activation: every channel has its own offset and width.  dy has a mean and a part along xhat in every group, so that both means
    of the backward are about as large as the rest of it."""
    N, L, C, G = shape
    gen = torch.Generator(device=device).manual_seed(seed)
    normal = lambda *s: torch.randn(*s, generator=gen, device=device)  # noqa: E731
    x = (normal(N, L, C) * torch.exp(0.3 * normal(C)) + 0.5 * normal(C) + offset).to(dtype)
    gamma, beta = 1 + 0.2 * normal(C), 0.2 * normal(C)
    keep = (torch.rand(N, L, C, generator=gen, device=device) < 0.6).to(torch.uint8) if mask else None
    dy = (normal(N, L, C) + 2 + (x.float() - offset)).to(dtype)
    return x, gamma, beta, keep, dy, None if lengths is None else torch.tensor(lengths, device=device)


def norm_bounds(x, gamma, beta, G, ref, dy, mask_scale=1.0):
    """Elementwise bounds of an fp32 evaluation (u = 2^-24), for y, dx and, per channel, dgamma and dbeta.

    xhat = (x - mean) r.  Pieces of at most 32 values are averaged and merged pairwise (or all are averaged and the mean is corrected by that
    of the deviations): the mean is off by 64 u of the values and ADDS u of the deviations, r by ADDS u of itself and by what a wrong mean
    of a piece adds, 64 u max|x| r.  So ex = u (64 max|x| r + ADDS) (1 + |xhat|), max|x| over the group.
    z = gamma xhat + beta: ez = |gamma| ex + 4 u (|gamma xhat| + |beta|).  The activations have slopes of at most 1.1 and second derivatives
    of at most 1; their own evaluation and that of their slopes is off by 16 u of 1 + |z|, of 1.
    gamma dz: e = |gamma dy| (ez + 16 u) + 4 u |gamma dz|.  m1 and m2 are means of such terms, ADDS u of the terms' magnitudes off; and
    dx = r (gamma dz - m1 - xhat m2) takes each part's error, 8 u of the parts for the four operations, and r's own."""
    from tests import operator_refs as R
    u, (N, L, C) = R.U, x.shape
    valid = ref['valid']
    group = lambda t: t.reshape(N, L, G, C // G)  # noqa: E731
    spread = lambda v: v.repeat_interleave(C // G, -1)[:, None, :]  # noqa: E731
    count = (valid.sum(1).double() * (C // G)).clamp_min(1)
    mean = lambda t: spread(group(torch.where(valid, t, 0.0)).sum((1, 3)) / count)  # noqa: E731
    gamma, beta, r = gamma.detach().double().abs(), beta.detach().double().abs(), spread(ref['rstd'])
    top = spread(group(torch.where(valid, x.detach().double().abs(), 0.0)).amax((1, 3))) * r
    own = u * (64 * top + ADDS)

    def through(xhat, z):
        ex = own * (1 + xhat.abs())
        return ex, gamma * ex + 4 * u * (gamma * xhat.abs() + beta)
    _, ez = through(ref['xhat'], ref['z'])
    ey = torch.where(valid, 1.1 * ez + 16 * u * (1 + ref['z'].abs()), 0.0) * mask_scale
    xhat, dz = ref['xhat_b'].abs(), ref['dz']
    ex, ez = through(ref['xhat_b'], ref['z_b'])
    edz = torch.where(valid, dy.detach().double().abs() * mask_scale * (ez + 16 * u) + 3 * u * dz.abs(), 0.0)
    gdz, e = gamma * dz.abs(), gamma * edz + u * gamma * dz.abs()
    m1, m2 = ref['m1'].abs(), ref['m2'].abs()
    em1 = mean(e) + ADDS * u * mean(gdz)
    em2 = mean(e * xhat + gdz * ex) + ADDS * u * mean(gdz * xhat)
    edx = r * (e + em1 + xhat * em2 + ex * m2 + 8 * u * (gdz + m1 + xhat * m2)) + own * ref['dx'].abs()
    edgamma = (edz * xhat + dz.abs() * ex).sum((0, 1)) + ADDS * u * (dz * xhat).abs().sum((0, 1))
    edbeta = edz.sum((0, 1)) + ADDS * u * dz.abs().sum((0, 1))
    return ey, torch.where(valid, edx, 0.0), edgamma, edbeta


def norm_reference(x, gamma, beta, G, lengths, keep, act, mask_scale, dy, checkpoint):
    """operator_refs.group_norm, and the two means of its backward."""
    from tests import operator_refs as R
    ref = R.group_norm(x, gamma, beta, G, lengths, keep, act, 1e-5, mask_scale, dy=dy, checkpoint=checkpoint)
    ref['m1'], ref['m2'] = norm_means(ref, gamma, G)
    return ref


def norm_means(ref, gamma, G, rows=None):
    """mean(gamma dz) and mean(gamma dz xhat), spread over the channels; rows: only these are added (a planted mistake)."""
    dz = ref['dz'] * gamma.detach().double()
    if rows is not None:
        dz = dz * rows.to(dz.dtype)[None, :, None]
    N, L, C = dz.shape
    n = (ref['valid'].sum(1).double() * (C // G)).clamp_min(1)
    means = [(t.reshape(N, L, G, C // G).sum((1, 3)) / n).repeat_interleave(C // G, -1)[:, None, :] for t in (dz, dz * ref['xhat_b'])]
    return [torch.where(ref['valid'], m, 0.0) for m in means]


def outside(got, want, bound):
    """Elements that a result of got's type would have off by more than the bound and half a step."""
    from tests import operator_refs as R
    return ~((got.double() - want).abs() <= bound + 1.01 * R.HALF[got.dtype] * (want.abs() + bound))
