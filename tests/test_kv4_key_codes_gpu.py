"""Keys written to the 4-bit cache, to the byte: a code is a decision, so a key is worked out in 64 bits and its codes and numbers are those of the
formulas wherever the formulas themselves leave no doubt."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def turned(x, angle, half):
    c, s = torch.cos(angle)[:, None], torch.sin(angle)[:, None]
    y, h = torch.empty_like(x), x.shape[-1] // 2
    a, b = (slice(0, h), slice(h, None)) if half else (slice(0, None, 2), slice(1, None, 2))
    y[..., a], y[..., b] = x[..., a] * c - x[..., b] * s, x[..., a] * s + x[..., b] * c
    return y


def made(x, w, eps, angle, half):
    """Normed and rotated, in x's precision."""
    y = x * torch.rsqrt(x.pow(2).mean(-1, keepdim=True) + eps) * w.to(x.dtype)
    return turned(y, angle.to(x.dtype), half)


def bf16(x):
    return x.float().bfloat16().to(x.dtype)


def held(y):
    zero = bf16(y.amin(-1, keepdim=True))
    step = bf16((y.amax(-1, keepdim=True) - zero).clamp_min(0) / 15)
    return torch.round((y - zero) / step).clamp(0, 15).long(), step, zero


def check(qkv, w, inv, nh, nkv, hd, half, first, doubtful=2):
    from mivi_v4_b200.ops import kernels as K
    page, n = 64, qkv.shape[0]
    pages = -(-(first + n) // page)
    pool = torch.zeros(pages, nkv, page * (hd + 8), dtype=torch.uint8, device=DEV)
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)          # noqa: E731
    K.kv4_prepare(qkv.to(DEV), w.to(DEV), w.to(DEV), 1e-5, inv.to(DEV), half, ints(list(range(first, first + n))), ints([0] * n), ints([list(range(pages))]), pool,
                  torch.empty(n, nh * hd, device=DEV), nh, nkv, hd)
    got = pool.cpu()

    def rows(x):                                                 # [pages, kv heads, page, ...] -> [n, kv heads, ...]
        return x.transpose(1, 2).flatten(0, 1)[first:first + n]
    codes = rows(got[..., :page * hd // 2].unflatten(-1, (page, hd // 2))).long()
    codes = torch.stack([codes & 15, codes >> 4], -1).flatten(-2)
    numbers = rows(got[..., page * hd:].contiguous().view(torch.bfloat16).unflatten(-1, (page, 4))).double()
    step, zero = numbers[..., 0:1], numbers[..., 1:2]
    y = made(qkv.view(n, -1, hd)[:, nh:nh + nkv].double(), w, EPS, angles(first, n, inv), half)
    # What 64 bits leave open: an angle below 2^11.1 is 2^10.5 quarter turns, whose own last place is 2^-54, so 2^-43.5 of the row's largest element; all
    # else is some 2^-50.  An element within 2^-40 of its row's largest of a border may fall on either side.
    doubt = 2.0 ** -40 * y.abs().amax(-1, keepdim=True)
    low, high = y.amin(-1, keepdim=True), y.amax(-1, keepdim=True)
    assert ((zero == bf16(low)) | (zero == bf16(low - doubt)) | (zero == bf16(low + doubt))).all()
    span = lambda d: bf16((high + d - zero).clamp_min(0) / 15)   # noqa: E731
    assert ((step == span(0)) | (step == span(-doubt)) | (step == span(doubt))).all()
    t = (y - zero) / step
    want = torch.round(t).clamp(0, 15).long()
    near = ((t - torch.floor(t)) - 0.5).abs() * step <= doubt
    wrong = (codes != want) & ~near
    assert int(near.sum()) <= doubtful and not wrong.any(), (int(wrong.sum()), int(near.sum()))


EPS = float(torch.tensor(1e-5, dtype=torch.float32))             # (handed over in 32 bits)


def angles(first, n, inv):
    return torch.arange(first, first + n).double()[:, None] * inv.double()


def inputs(nh, nkv, hd, n, seed):
    g = torch.Generator().manual_seed(seed)
    qkv = 3 * torch.randn(n, (nh + 2 * nkv) * hd, generator=g)
    return qkv, 1 + 0.3 * torch.randn(hd, generator=g), (1e6 ** (-torch.arange(0, hd, 2).double() / hd)).float()


@pytest.mark.parametrize("nh,nkv,hd,half,n", [(4, 8, 64, False, 2048), (4, 8, 64, True, 2048), (2, 16, 32, False, 2048), (2, 4, 128, True, 2048),
                                              (1, 2, 256, False, 2048), (8, 20, 64, False, 200), (1, 5, 96, True, 1500)])
def test_key_codes_are_those_of_64_bits(nh, nkv, hd, half, n):
    qkv, w, inv = inputs(nh, nkv, hd, n, hd + n + half)
    check(qkv, w, inv, nh, nkv, hd, half, 37)


def next_to_borders(nh, nkv, hd, half, n, first):
    """Rows whose first pair's first element is moved, by float32 numbers, as near as those come to the border between two codes."""
    qkv, w, inv = inputs(nh, nkv, hd, n, 5 * hd + half)
    x, partner = qkv.view(n, -1, hd)[:, nh:nh + nkv], hd // 2 if half else 1
    angle = angles(first, n, inv)
    c, s = torch.cos(angle[:, :1]), torch.sin(angle[:, :1])
    x[..., 0] = 0.1                                              # (not an end of its row)
    for _ in range(6):                                           # each move changes the row's norm, and with it the border, a little less
        y = made(x.double(), w, EPS, angle, half)
        _, step, zero = held(y)
        t = (y[..., 0] - zero[..., 0]) / step[..., 0]
        border = zero[..., 0] + step[..., 0] * (torch.floor(t) + 0.5)
        norm = torch.rsqrt(x.double().pow(2).mean(-1) + EPS)
        fine = (c.abs() > 0.3).expand_as(border)
        x[..., 0] = torch.where(fine, ((border / norm + w.double()[partner] * x.double()[..., partner] * s) / (w.double()[0] * c)).float(), x[..., 0])
    return qkv, w, inv


BORDERS = [(4, 8, 64, False, 1024), (2, 4, 128, True, 1024), (2, 16, 32, False, 1024), (1, 3, 256, True, 600), (2, 6, 96, False, 290)]


@pytest.mark.parametrize("nh,nkv,hd,half,n", BORDERS)
def test_keys_next_to_a_border(nh, nkv, hd, half, n):
    # (float32 numbers come within 2^-30 of a border or so, and within 2^-40 of it once in some hundred to a thousand rows)
    check(*next_to_borders(nh, nkv, hd, half, n, 37), nh, nkv, hd, half, 37, doubtful=2 + n * nkv // 50)


def test_32_bits_would_be_seen():
    """The rows next to a border in 32 bits, with sines and cosines of 64: many codes differ from those of 64 bits."""
    for nh, nkv, hd, half, n in BORDERS:
        qkv, w, inv = next_to_borders(nh, nkv, hd, half, n, 37)
        x = qkv.view(n, -1, hd)[:, nh:nh + nkv]
        angle = angles(37, n, inv)
        c64 = held(made(x.double(), w, EPS, angle, half))[0]
        y = x * torch.rsqrt(x.pow(2).mean(-1, keepdim=True) + 1e-5) * w
        c, s = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]
        z, h = torch.empty_like(y), hd // 2
        a, b = (slice(0, h), slice(h, None)) if half else (slice(0, None, 2), slice(1, None, 2))
        z[..., a], z[..., b] = y[..., a] * c - y[..., b] * s, y[..., a] * s + y[..., b] * c
        differ = int((held(z)[0] != c64).sum())
        assert differ >= n * nkv // 20, (hd, differ)
