"""Plain 64-bit definitions of the group norm / 8-bit checkpoint operators on the CPU or the GPU, and the bounds that their tests use."""
import torch

U = 2.0 ** -24                     # half a step of float32, relative
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}
BLOCK = 32

ACTS = {'identity': lambda z: z, 'relu': torch.relu, 'tanh': torch.tanh, 'sigmoid': torch.sigmoid, 'silu': lambda z: z * torch.sigmoid(z)}


def round_trip(x, lengths=None):
    """(q int8, biased exponent uint8, the float64 values) of x [..., C], by definition: e the smallest whole number >= -126 with
    |round(x / 2^e)| <= 127 for the block's 32 channels.  Blocks with an infinity or a NaN stand for NaN."""
    C = x.shape[-1]
    nb = -(-C // BLOCK)
    x64 = x.detach().double()
    if lengths is not None:
        behind = torch.arange(x.shape[1], device=x.device)[None, :] >= lengths.to(x.device)[:, None]
        x64 = torch.where(behind[..., None], 0.0, x64)
    b = torch.nn.functional.pad(x64, (0, nb * BLOCK - C)).unflatten(-1, (nb, BLOCK))
    finite = torch.isfinite(b).all(-1)
    clean = torch.where(finite[..., None], b, 0.0)
    top = clean.abs().amax(-1)
    e = torch.where(top > 0, torch.frexp(top)[1] - 7, -126).clamp_min(-126)
    two = lambda k: ((k.long() + 1023) << 52).view(torch.float64)  # noqa: E731  (exact: pow may be off in its last bit)
    e = e + (torch.round(top / two(e)) > 127).to(e.dtype)
    limit = torch.where(e == 122, 63.0, 127.0)[..., None]
    q = torch.minimum(torch.maximum(torch.round(clean / two(e)[..., None]), -limit), limit)
    values = torch.where(finite[..., None], q * two(e)[..., None], float('nan')).flatten(-2)[..., :C]
    code = torch.where(finite, e + 127, 255)
    return q.flatten(-2)[..., :C].to(torch.int8), code.to(torch.uint8), values


def rows_valid(x, lengths):
    L = x.shape[1]
    if lengths is None:
        return torch.ones(x.shape[0], L, 1, dtype=torch.bool, device=x.device)
    return (torch.arange(L, device=x.device)[None, :] < lengths.to(x.device).clamp(0, L)[:, None])[..., None]


def group_norm(x, gamma, beta, G, lengths=None, mask=None, act='identity', eps=1e-5, mask_scale=1.0, dy=None, checkpoint=False):
    """dict of float64 results: y, z, xhat, rstd, and with dy: dz, dx, dgamma, dbeta (with checkpoint those of the 8-bit values)."""
    N, L, C = x.shape
    valid = rows_valid(x, lengths)
    x64 = torch.where(valid, x.detach().double(), 0.0)
    g64, b64 = gamma.detach().double(), beta.detach().double()
    count = valid.sum(1).double() * (C // G)                                            # [N, 1]
    grp = lambda t: t.reshape(N, L, G, C // G)  # noqa: E731
    spread = lambda v: v.repeat_interleave(C // G, -1)[:, None, :]  # noqa: E731
    n = count.clamp_min(1)
    mean = grp(x64).sum((1, 3)) / n
    var = torch.where(valid, (x64 - spread(mean)) ** 2, 0.0)
    rstd = 1 / torch.sqrt(grp(var).sum((1, 3)) / n + eps)
    factor = torch.ones_like(x64) if mask is None else (mask != 0).double() * mask_scale

    def through(held):
        xhat = torch.where(valid, (held - spread(mean)) * spread(rstd), 0.0)
        return xhat, xhat * g64 + b64
    xhat, z = through(x64)
    out = {'y': torch.where(valid, ACTS[act](z) * factor, 0.0), 'z': z, 'xhat': xhat, 'mean': mean, 'rstd': rstd, 'valid': valid}
    if dy is None:
        return out
    if checkpoint:
        xhat, z = through(torch.where(valid, round_trip(x, lengths)[2], 0.0))
    zr = z.clone().requires_grad_()
    slope, = torch.autograd.grad(ACTS[act](zr).sum(), zr)
    dz = torch.where(valid, torch.where(valid, dy.detach().double(), 0.0) * factor * slope, 0.0)
    m1 = spread(grp(dz * g64).sum((1, 3)) / n)
    m2 = spread(grp(dz * g64 * xhat).sum((1, 3)) / n)
    dx = torch.where(valid, spread(rstd) * (dz * g64 - m1 - xhat * m2), 0.0)
    out.update(dz=dz, dx=dx, dgamma=(dz * xhat).sum((0, 1)), dbeta=dz.sum((0, 1)), xhat_b=xhat, z_b=z)
    return out


def norm_bounds(x, gamma, ref, dy=None, mask_scale=1.0):
    """Elementwise bounds of a float32 evaluation, from the roundings it makes (u = 2^-24).  The mean is merged from partial means in at
    most 32 steps, each off by u of the values: 32 u max|x|; so xhat is off by ex = 32 u (max|x| rstd + max|xhat|) (the deviation's own
    32 roundings are relative to xhat), z by ez = max|gamma| ex + 2 u max|z|; the activations' slopes stay below 1.1 and their own
    evaluation within 8 u.  dz is off by |dy| (ez + 8 u) (second derivatives stay below 1); dx = rstd (gamma dz - m1 - xhat m2) with
    mean |xhat| <= 1, sums of 64 roundings deep.  Returns ey, and with dy: edx, edgamma, edbeta."""
    valid = ref['valid']
    xm = torch.where(valid, x.detach().double().abs(), 0.0).max()
    r, g = ref['rstd'].max(), gamma.detach().double().abs().max()
    X = max(ref['xhat'].abs().max().item(), ref.get('xhat_b', ref['xhat']).abs().max().item())
    ex = 32 * U * (xm * r + X)
    ez = g * ex + 2 * U * ref['z'].abs().max()
    ey = 1.1 * ez + 8 * U * (1 + ref['z'].abs().max())
    if dy is None:
        return ey * mask_scale
    top = torch.where(valid, dy.detach().double().abs(), 0.0).max() * mask_scale
    edz = top * (1.1 * ez + 16 * U)
    D = 1.1 * top * max(g, 1.0)
    edx = r * (2 + 2 * X) * (edz * max(g, 1.0) + D * (ex + 64 * U))
    rows = valid.sum().double()
    edbeta = rows * edz + 64 * U * ref['dz'].abs().sum((0, 1))
    edgamma = rows * (edz * X + 1.1 * top * ex) + 64 * U * (ref['dz'] * ref['xhat_b']).abs().sum((0, 1))
    return ey * mask_scale, edx, edgamma, edbeta


def shifted(x, k, d):
    """[N, L, C] -> [N, L, k, C]: the rows that the taps of a 'same' convolution see."""
    N, L, C = x.shape
    pad = (k - 1) * d // 2
    xp = torch.nn.functional.pad(x, (0, 0, pad, (k - 1) * d - pad))
    at = torch.arange(L, device=x.device)[:, None] + torch.arange(k, device=x.device) * d
    return xp[:, at]


def conv(x, w, d=1, groups=1):
    """'same' convolution of float64 x [N, L, I] with w [O, I / groups, k] -> [N, L, O]."""
    N, L, I = x.shape
    O, Cg, k = w.shape
    taps = shifted(x, k, d)
    out = [torch.matmul(taps[..., g * Cg:(g + 1) * Cg].reshape(N * L, k * Cg), w[g * (O // groups):(g + 1) * (O // groups)].permute(2, 1, 0).reshape(k * Cg, O // groups))
           for g in range(groups)]
    return torch.cat(out, 1).reshape(N, L, O)


def weight_grad(x, dy, k, d=1, groups=1):
    """dW [O, I / groups, k] in 64 bits, and the sum of the products' magnitudes."""
    N, L, I = x.shape
    O, Cg = dy.shape[-1], I // groups
    taps, dy = shifted(x.double(), k, d), dy.detach().double()

    def product(a, b):
        out = [torch.matmul(a[..., g * (O // groups):(g + 1) * (O // groups)].reshape(N * L, -1).t().contiguous(),
                            b[..., g * Cg:(g + 1) * Cg].reshape(N * L, k * Cg)) for g in range(groups)]
        return torch.cat(out, 0).reshape(O, k, Cg).permute(0, 2, 1)
    return product(dy, taps), product(dy.abs(), taps.abs())
