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
