"""The 4-bit cache's kernels against plain expressions in float64 (plain_kv4.py), at the sizes, masks and rows where they can go wrong."""
import math

import pytest
import torch

import plain_kv4 as Q
import plain_lfm2 as P

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def K():
    from mivi_v4_b200.ops import kernels
    return kernels


def workspace():
    from mivi_v4_b200.engine import Workspace
    return Workspace(DEV)


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def tables(lengths, page, seed, spare=3):
    """A shuffled page table for sequences of these lengths: (rows as lists, total pages)."""
    g = torch.Generator().manual_seed(seed)
    blocks = [-(-n // page) for n in lengths]
    total = sum(blocks) + spare
    perm = torch.randperm(total, generator=g).tolist()
    rows, at = [], 0
    for n in blocks:
        rows.append(perm[at:at + n] + [0] * (max(blocks) - n))
        at += n
    return rows, total


def filled(total, nkv, page, hd, seed, loud=True):
    """Random rows for every page, the spare ones too: (pool bytes on the device, keys, values as they stand in float64)."""
    g = torch.Generator().manual_seed(seed)
    k = torch.randn(total, nkv, page, hd, generator=g)
    v = torch.randn(total, nkv, page, hd, generator=g) * torch.exp(torch.randn(total, nkv, page, 1, generator=g))
    if loud:
        k[..., 0] *= 4
    pool = Q.pool_bytes(k, v)
    rk, rv = Q.rows_of(pool, page, hd)
    return pool, rk, rv


def allowed(q, k, v, pos, scale, window, want, dtype, pages):
    """How far a result may be off: [nh, hd] float64.

    float32: sums of hd products for a score and of T weighted values, each off by 2^-24 of the sum of magnitudes a step (two factors
    of 4: the exponential's own last places and the merging of parts).  bfloat16: the result's own rounding, half a step of 2^-7 and so 2^-8 of it, and the
    weights' rounding to 11 bits, 2^-11 of the largest value.  Read back in bfloat16 (``pages``), keys, values and weights are rounded
    by 2^-8: a score is off by 2^-8 scale sum |q||k|, the weights by twice that, values and weights by 2^-8 each."""
    nh, hd = q.shape
    nkv = k.shape[1]
    lo = max(0, pos - window + 1) if window > 0 else 0
    out = torch.zeros(nh, hd, dtype=torch.float64)
    for h in range(nh):
        g = h // (nh // nkv)
        kk, vv = k[lo:pos + 1, g], v[lo:pos + 1, g]
        top = float(vv.abs().max())
        mags = float((kk.abs() @ q[h].abs()).max()) * scale
        spare = 4 * 2.0 ** -24 * (mags * hd ** 0.5 + 8) * 2 * top + 4 * 2.0 ** -24 * kk.shape[0] ** 0.5 * top
        if dtype == torch.bfloat16:
            spare += 2.0 ** -11 * top
            if pages:
                spare += (math.expm1(2 * 2.0 ** -8 * mags) + 2 * 2.0 ** -8) * top
        out[h] = spare
    return out + (2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -23) * want.abs()


def attend_all(q, pool, rows, lengths, lens, nh, nkv, hd, page, window, ws=None, splits=None):
    """The step that brings ``lens`` tokens to sequences that are ``lengths`` long with them."""
    starts = [n - m for n, m in zip(lengths, lens)]
    cu = [sum(lens[:b]) for b in range(len(lens) + 1)]
    qd = q.reshape(sum(lens), nh * hd).contiguous().to(DEV)
    out = torch.full_like(qd, float("nan"))
    K().attention_kv4(qd, pool, ints(rows), ints([s + i for s, m in zip(starts, lens) for i in range(m)]),
                      ints([b for b, m in enumerate(lens) for _ in range(m)]), ints(cu), ints(starts), out, nh, nkv, hd, hd ** -0.5, window,
                      ws or workspace(), starts, lens, splits=splits)
    return out.reshape(-1, nh, hd)


def check(out, q, rk, rv, rows, lengths, lens, page, window, dtype, pages=None, only=None):
    from mivi_v4_b200.ops import kernels
    n = 0
    for b, (L, m) in enumerate(zip(lengths, lens)):
        k, v = Q.sequence(rk, rows[b], L), Q.sequence(rv, rows[b], L)
        back = (m > kernels.KV4_DIRECT_TOKENS) if pages is None else pages
        for i in range(m):
            if only is None or (b, i) in only or i in (0, m - 1) or i % 37 == 5:
                pos = L - m + i
                qi = q[n].double()
                want = Q.attend(qi, k, v, pos, q.shape[-1] ** -0.5, window)
                got = out[n].double().cpu()
                room = allowed(qi, k, v, pos, q.shape[-1] ** -0.5, window, want, dtype, back)
                bad = (got - want).abs() > room
                assert not bad.any() and torch.isfinite(got).all(), (b, i, pos, ((got - want).abs() / room).max())
            n += 1


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("nh,nkv,hd,page,window", [
    (4, 2, 16, 16, 0), (3, 1, 32, 64, 0), (5, 5, 48, 32, 0), (32, 8, 64, 64, 0), (12, 1, 128, 64, 0), (2, 2, 256, 8, 0), (8, 2, 64, 64, 37),
    (6, 3, 80, 16, 64), (7, 1, 8, 1, 0), (24, 8, 64, 16, 1), (16, 1, 64, 128, 100), (20, 1, 96, 2, 0), (4, 4, 40, 4, 3), (9, 3, 128, 32, 200)])
@pytest.mark.parametrize("splits", [None, 1, 7])
def test_single_tokens(dtype, nh, nkv, hd, page, window, splits):
    lengths = [1, 33, 300, 64, 129, 2, 65, 127]
    rows, total = tables(lengths, page, seed=hd)
    pool, rk, rv = filled(total, nkv, page, hd, seed=nh + hd)
    g = torch.Generator().manual_seed(5)
    q = (2 * torch.randn(len(lengths), nh, hd, generator=g)).to(dtype)
    # one far key of the longest sequence stands out for head 0: a kernel that loses it cannot pass
    far = Q.sequence(rk, rows[2], 300)[5, 0]
    if window == 0:
        q[2, 0] = (far / far.norm() * 8.0 * hd ** 0.25).to(dtype)
    ws = workspace()
    for _ in range(2):                                           # twice: counters are back at zero
        out = attend_all(q, pool.to(DEV), rows, lengths, [1] * len(lengths), nh, nkv, hd, page, window, ws, splits)
        check(out, q, rk, rv, rows, lengths, [1] * len(lengths), page, window, dtype)
    again = attend_all(q, pool.to(DEV), rows, lengths, [1] * len(lengths), nh, nkv, hd, page, window, ws, splits)
    assert torch.equal(out, again)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("nh,nkv,hd,page,window", [(32, 8, 64, 64, 0), (3, 1, 64, 64, 0), (6, 2, 128, 16, 0), (5, 5, 48, 32, 50), (8, 2, 64, 64, 70),
                                                   (4, 2, 40, 8, 0), (2, 1, 256, 64, 0), (16, 8, 96, 64, 0)])
@pytest.mark.parametrize("lens", [[2, 1, 5], [16, 3, 7], [17, 1, 300], [260, 140], [3, 64, 16, 17, 1]])
def test_several_tokens(dtype, nh, nkv, hd, page, window, lens):
    """Short runs, long ones and both in one step, over caches that held tokens before."""
    lengths = [m + [0, 200, 63, 64, 1][b] for b, m in enumerate(lens)]
    rows, total = tables(lengths, page, seed=hd + len(lens))
    pool, rk, rv = filled(total, nkv, page, hd, seed=nh + sum(lens))
    g = torch.Generator().manual_seed(6)
    q = torch.randn(sum(lens), nh, hd, generator=g).to(dtype)
    out = attend_all(q, pool.to(DEV), rows, lengths, lens, nh, nkv, hd, page, window)
    check(out, q, rk, rv, rows, lengths, lens, page, window, dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("hd,lens,window", [(64, [1, 1, 1], 0), (64, [6, 2, 1], 0), (64, [150, 300, 140], 0), (64, [40, 20, 17], 30), (48, [1, 20, 3], 0),
                                            (128, [9, 1, 1], 9), (40, [30, 1, 18], 0)])
def test_rows_that_are_not_finite(dtype, hd, lens, window):
    """A key or value row that is not finite makes the queries that see it NaN and no others: not those before it, not those whose window
    has left it behind, not other sequences; what stands behind a sequence's last row counts for nobody."""
    nh, nkv, page = 4, 2, 64 if hd == 64 else 16
    lengths = [m + 90 for m in lens]
    rows, total = tables(lengths, page, seed=3, spare=1)
    g = torch.Generator().manual_seed(8)
    k, v = torch.randn(total, nkv, page, hd, generator=g), torch.randn(total, nkv, page, hd, generator=g)
    first = {}
    for b, (L, m) in enumerate(zip(lengths, lens)):              # a bad key row of kv head 0, a bad value row of kv head 1, in mid-run
        for head, x in ((0, k), (1, v)):
            t = L - 1 - m // 2 if b < 2 else 20                  # (the last sequence: one that all of its queries see, or none behind a window)
            first[b, head] = t
            x[rows[b][t // page], head, t % page, 3] = [math.inf, math.nan, -math.inf][b]
    for b, L in enumerate(lengths):                              # stale rows behind the last one
        for t in range(L, -(-L // page) * page):
            k[rows[b][t // page], :, t % page] = math.nan
            v[rows[b][t // page], :, t % page] = math.inf
    spare = (set(range(total)) - {p for b, L in enumerate(lengths) for p in rows[b][:-(-L // page)]}).pop()
    k[spare], v[spare] = math.nan, math.nan
    rows = [[p if i * page < L else spare for i, p in enumerate(r)] for r, L in zip(rows, lengths)]
    pool = Q.pool_bytes(k, v)
    rk, rv = Q.rows_of(pool, page, hd)
    q = torch.randn(sum(lens), nh, hd, generator=g).to(dtype)
    out = attend_all(q, pool.to(DEV), rows, lengths, lens, nh, nkv, hd, page, window).double().cpu()
    n = 0
    for b, (L, m) in enumerate(zip(lengths, lens)):
        kk, vv = Q.sequence(rk, rows[b], L), Q.sequence(rv, rows[b], L)
        for i in range(m):
            pos = L - m + i
            for head in range(2):
                t = first[b, head]
                sees = t <= pos and (window <= 0 or t > pos - window)
                got = out[n, 2 * head:2 * head + 2]
                assert bool(torch.isnan(got).all()) == sees and bool(torch.isnan(got).any()) == sees, (b, i, head, sees)
                if not sees:
                    want = Q.attend(q[n].double(), kk[:, [head]], vv[:, [head]], pos, hd ** -0.5, window)[2 * head:2 * head + 2]
                    assert (got - want).abs().max() < 0.05
            n += 1


def test_values_and_queries_of_any_size():
    """Rows near the largest and the smallest floats, rows of one value, a query row far larger than its neighbour's."""
    nh, nkv, hd, page = 4, 1, 64, 64
    g = torch.Generator().manual_seed(9)
    for big, qs in ((1e30, 1e-30), (1e-30, 1e30), (3e38, 1e-38), (1e-36, 1e36)):
        k = torch.randn(3, nkv, page, hd, generator=g).clamp(-1, 1) * big
        v = torch.randn(3, nkv, page, hd, generator=g).clamp(-1, 1) * torch.tensor([1e-20, 1.0, 1e20]).view(3, 1, 1, 1)
        v[1, 0, :8] = 0.0
        v[1, 0, 8:16] = -7.0
        pool = Q.pool_bytes(k, v)
        rk, rv = Q.rows_of(pool, page, hd)
        for order in ([0, 1, 2], [2, 1, 0], [1, 0, 2]):
            rows, lengths = [order], [150]
            for dtype in (torch.float32, torch.bfloat16):
                q = torch.randn(1, nh, hd, generator=g)
                q[0, 1] *= 1e-3
                q = (q * qs).to(dtype)
                out = attend_all(q, pool.to(DEV), rows, lengths, [1], nh, nkv, hd, page, 0)
                check(out, q, rk, rv, rows, lengths, [1], page, 0, dtype)


def test_offsets_beyond_32_bits():
    """A pool of more than 4 GB: the last pages are written, read back and attended to."""
    nh, nkv, hd, page = 8, 8, 64, 64
    total = (1 << 32) // (nkv * page * (hd + 8)) + 9
    pool = torch.zeros((total, nkv, page * (hd + 8)), dtype=torch.uint8, device=DEV)
    assert pool.numel() > 1 << 32
    lens, rows = [70], [[total - 1, total - 2]]
    g = torch.Generator().manual_seed(10)
    qkv = torch.randn(70, (nh + 2 * nkv) * hd, generator=g)
    positions, seq_of = ints(list(range(70))), ints([0] * 70)
    for dtype in (torch.float32, torch.bfloat16):
        q = torch.empty(70, nh * hd, dtype=dtype, device=DEV)
        K().kv4_prepare(qkv.to(DEV), None, None, 0.0, None, False, positions, seq_of, ints(rows), pool, q, nh, nkv, hd)
        k, v = torch.empty(2, 70, nkv, hd, device=DEV).unbind(0)
        K().kv4_read(pool, ints(rows), positions, seq_of, k, v, nkv, hd)
        want = Q.held(qkv.view(70, -1, hd)[:, nh:])
        assert torch.allclose(k.double().cpu(), want[:, :nkv], rtol=1e-6, atol=1e-6)
        assert torch.allclose(v.double().cpu(), want[:, nkv:], rtol=1e-6, atol=1e-6)
        small = pool[total - 9:].cpu()
        rk, rv = Q.rows_of(small, page, hd)
        near = [[8, 7]]
        for lens in ([70], [2]):
            out = attend_all(q.view(70, nh, hd)[70 - lens[0]:].cpu(), pool, rows, [70], lens, nh, nkv, hd, page, 0)
            check(out, q.view(70, nh, hd)[70 - lens[0]:].cpu(), rk, rv, near, [70], lens, page, 0, dtype)
    assert int(pool[:1000].max()) == 0 and int(pool[total - 9:total - 2].max()) == 0


# ---------------------------------------------------------------------------------------------- writing and reading
def prepared(nh, nkv, hd, page, lens, starts, dtype, wq, wk, eps, inv, half, qkv, pool, rows):
    q = torch.full((sum(lens), nh * hd), float("nan"), dtype=dtype, device=DEV)
    pos = [s + i for s, m in zip(starts, lens) for i in range(m)]
    seq = [b for b, m in enumerate(lens) for _ in range(m)]
    dev = lambda t: None if t is None else t.to(DEV)             # noqa: E731
    K().kv4_prepare(qkv.to(DEV), dev(wq), dev(wk), eps, dev(inv), half, ints(pos), ints(seq), ints(rows), pool, q, nh, nkv, hd)
    return q.view(-1, nh, hd), torch.tensor(pos), seq


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("style", ["interleaved", "half_split"])
@pytest.mark.parametrize("nh,nkv,hd,page,normed,rotated,lens,starts", [
    (32, 8, 64, 64, True, True, [1, 1, 1], [0, 63, 30000]), (4, 2, 16, 16, True, True, [1, 40, 5], [7, 0, 14]), (5, 5, 48, 32, True, False, [3], [1]),
    (3, 1, 32, 64, False, True, [70, 2], [0, 120000]), (7, 7, 8, 2, True, True, [9], [0]), (2, 1, 256, 8, True, True, [20], [3]),
    (24, 8, 64, 64, True, True, [130, 66], [5, 64]), (16, 4, 128, 1, False, False, [3], [0]), (1, 3, 40, 4, True, True, [11], [2]),
    (32, 8, 64, 64, False, True, [90], [0]), (16, 8, 96, 32, True, True, [65], [31])])
def test_written_rows(dtype, style, nh, nkv, hd, page, normed, rotated, lens, starts):
    lengths = [s + m for s, m in zip(starts, lens)]
    rows, total = tables(lengths, page, seed=hd, spare=2)
    g = torch.Generator().manual_seed(hd + nh)
    N = sum(lens)
    qkv = 2 * torch.randn(N, (nh + 2 * nkv) * hd, generator=g)
    wq, wk = ((1 + 0.3 * torch.randn(hd, generator=g)) if normed else None for _ in range(2))
    wk = (1 + 0.3 * torch.randn(hd, generator=g)) if normed else None
    inv = (10000.0 ** (-torch.arange(0, hd, 2).double() / hd)).float() if rotated else None
    before = torch.randint(0, 256, (total, nkv, page * (hd + 8)), generator=g, dtype=torch.uint8)
    pool = before.to(DEV)
    q, pos, seq = prepared(nh, nkv, hd, page, lens, starts, dtype, wq, wk, 1e-5, inv, style == "half_split", qkv, pool, rows)
    after = pool.cpu()

    def made(x, w):
        x = x.double()
        if w is not None:
            x = P.plain_rms_norm(x, w.double(), 1e-5)
        if inv is not None:
            ang = pos.double()[:, None, None] * inv.double()
            c, s, half = torch.cos(ang), torch.sin(ang), hd // 2
            y = torch.empty_like(x)
            a, b = (x[..., 0::2], x[..., 1::2]) if style == "interleaved" else (x[..., :half], x[..., half:])
            ra, rb = a * c - b * s, a * s + b * c
            if style == "interleaved":
                y[..., 0::2], y[..., 1::2] = ra, rb
            else:
                y[..., :half], y[..., half:] = ra, rb
            x = y
        return x

    heads = qkv.view(N, nh + 2 * nkv, hd)
    want_q, want_k, want_v = made(heads[:, :nh], wq), made(heads[:, nh:nh + nkv], wk), heads[:, nh + nkv:]
    # an element goes through a sum of hd squares, a root, two products and two more with a sine and cosine of one turn: some 10
    # roundings of 2^-24 of its row's largest; then its own rounding where q is bfloat16
    slack = 16 * 2.0 ** -24
    room = slack * want_q.abs().amax(-1, keepdim=True) + (2.0 ** -8 * want_q.abs() if dtype == torch.bfloat16 else 0)
    assert ((q.double().cpu() - want_q).abs() <= room).all()
    # the rows, byte by byte: values exactly; keys exactly unless a code or number lies within the slack of a border
    params = after[..., page * hd:].reshape(total, nkv, page, 8)
    touched = torch.zeros(total, page, dtype=torch.bool)
    free = 0
    for n in range(N):
        p, r = rows[seq[n]][int(pos[n]) // page], int(pos[n]) % page
        touched[p, r] = True
        for j, x in ((0, want_k), (1, want_v)):
            for h in range(nkv):
                row = after[p, h, (j * page + r) * hd // 2:(j * page + r + 1) * hd // 2].long()
                code = torch.stack([row & 15, row >> 4], -1).flatten()
                step, zero = params[p, h, r, 4 * j:4 * j + 4].contiguous().view(torch.bfloat16).double()
                if j == 1:                                       # float32 arithmetic, as torch does it
                    y = x[n, h]
                    z = y.min().bfloat16().float()
                    s = ((y.max() - z).clamp_min(0) / 15).bfloat16().float()
                    c = torch.round((y - z) / s).clamp(0, 15) if s > 0 else torch.zeros_like(y)
                    assert step == s and zero == z and torch.equal(code, c.long())
                    continue
                y = x[n, h].double()
                eps = slack * float(y.abs().max())
                lo, hi = float(y.min()), float(y.max())
                zs = {float(Q.bf16(torch.tensor(lo + d, dtype=torch.float64))) for d in (-eps, 0, eps)}
                assert float(zero) in zs
                ss = {float(Q.bf16(torch.tensor(max(0.0, hi + d - float(zero)) / 15, dtype=torch.float64))) for d in (-eps, 0, eps)}
                assert float(step) in ss
                t = (y - zero) / step
                want = torch.round(t).clamp(0, 15).long()
                near = ((t - torch.floor(t)) - 0.5).abs() * step <= 2 * eps
                assert ((code == want) | (near & ((code - want).abs() <= 1))).all(), (n, h)
                free += int((code != want).sum())
    assert free <= 2 + N * nkv * hd // 1000
    # nothing else is touched
    for j in range(2):
        a, b = ((x[..., j * page * hd // 2:(j + 1) * page * hd // 2].reshape(total, nkv, page, hd // 2).movedim(2, 1)[~touched]) for x in (after, before))
        assert torch.equal(a, b)
    a, b = (x[..., page * hd:].reshape(total, nkv, page, 8).movedim(2, 1)[~touched] for x in (after, before))
    assert torch.equal(a, b)


def test_rows_of_one_value_and_of_no_finite_value():
    nh, nkv, hd, page = 1, 2, 64, 16
    qkv = torch.randn(7, (nh + 2 * nkv) * hd, generator=torch.Generator().manual_seed(2))
    kv = qkv.view(7, nh + 2 * nkv, hd)[:, nh:]
    kv[0, 0] = 0.0
    kv[1, 1] = -3.7
    kv[2, 2, 5] = math.nan
    kv[3, 3, 63] = -math.inf
    kv[4, 0, 0] = math.inf
    kv[5, 1] = torch.linspace(-3.4e38, 3.4e38, hd, dtype=torch.float64).float()   # a span beyond the largest float
    kv[5, 2] = 3.4028234e38
    kv[6, 3] = torch.linspace(1000.0, 1001.0, hd)                # far from zero: as exact as bfloat16 is there
    kv[6, 0] = torch.linspace(0, 1e-39, hd)                      # below the normal numbers
    assert torch.isfinite(kv).sum() == kv.numel() - 3
    pool = torch.zeros(1, nkv, page * (hd + 8), dtype=torch.uint8, device=DEV)
    prepared(nh, nkv, hd, page, [7], [0], torch.float32, None, None, 0.0, None, False, qkv, pool, [[0]])
    k, v = torch.empty(2, 7, nkv, hd, device=DEV).unbind(0)
    K().kv4_read(pool, ints([[0]]), ints(list(range(7))), ints([0] * 7), k, v, nkv, hd)
    got = torch.cat([k, v], dim=1).cpu()
    for n, h in ((2, 2), (3, 3), (4, 0)):
        assert got[n, h].isnan().all()
        got[n, h] = kv[n, h] = 0.0
    assert torch.isfinite(got).all()
    # one value: zero is its bfloat16 (-3.703125), what is missing is the 15th of 15 steps
    assert (got[0, 0] == 0).all() and (got[1, 1] == got[1, 1, 0]).all() and abs(float(got[1, 1, 0]) + 3.7) <= 2.0 ** -8 * 0.003125 + 2.0 ** -22
    span = kv.double().amax(-1) - kv.double().amin(-1)
    room = span / 30 + span * 2.0 ** -8 + 2.0 ** -8 * kv.double().abs().amax(-1) + 1e-40
    assert ((got.double() - kv.double()).abs().amax(-1) <= room).all()


@pytest.mark.parametrize("nkv,hd,page", [(8, 64, 64), (1, 8, 1), (3, 40, 16), (2, 256, 2), (5, 128, 128)])
def test_read_back(nkv, hd, page):
    lengths = [1, 130, 77]
    rows, total = tables(lengths, page, seed=hd)
    pool, rk, rv = filled(total, nkv, page, hd, seed=1)
    which = [(0, 0), (1, 129), (1, 0), (2, 76), (2, 63), (1, 64), (1, 129)]
    for dtype in (torch.float32, torch.bfloat16):
        k, v = torch.full((2, len(which), nkv, hd), float("nan"), dtype=dtype, device=DEV).unbind(0)
        K().kv4_read(pool.to(DEV), ints(rows), ints([p for _, p in which]), ints([b for b, _ in which]), k, v, nkv, hd)
        for i, (b, p) in enumerate(which):
            for got, x in ((k, rk), (v, rv)):
                want = x[rows[b][p // page], :, p % page]
                assert torch.equal(got[i].cpu(), want.float().to(dtype))
    K().kv4_read(pool.to(DEV), ints(rows), ints([]), ints([]), k[:0], v[:0], nkv, hd)     # no rows: nothing happens


# ---------------------------------------------------------------------------------------------- together, as a program uses them
def test_written_then_attended_cut_anywhere():
    """The rows of three sequences written and attended to in one step, in two and token by token: the same rows to the byte, and results
    that differ by their last places only."""
    nh, nkv, hd, page = 8, 2, 64, 64
    lengths = [150, 40, 3]
    rows, total = tables(lengths, page, seed=4)
    g = torch.Generator().manual_seed(4)
    qkv = [torch.randn(n, (nh + 2 * nkv) * hd, generator=g) for n in lengths]
    w = 1 + 0.1 * torch.randn(hd, generator=g)
    inv = (1e6 ** (-torch.arange(0, hd, 2).double() / hd)).float()
    done = {}
    for cut in ("whole", "halves", "tokens"):
        pool = torch.zeros(total, nkv, page * (hd + 8), dtype=torch.uint8, device=DEV)
        pieces = [torch.zeros(0, nh, hd) for _ in lengths]
        ws, at = workspace(), [0] * 3
        while any(a < n for a, n in zip(at, lengths)):
            size = {"whole": 10 ** 6, "halves": 75, "tokens": 1}[cut]
            lens = [min(size, n - a) for a, n in zip(at, lengths)]
            live = [b for b in range(3) if lens[b]]
            x = torch.cat([qkv[b][at[b]:at[b] + lens[b]] for b in live])
            table = [rows[b] for b in live]
            q, _, _ = prepared(nh, nkv, hd, page, [lens[b] for b in live], [at[b] for b in live], torch.bfloat16, w, w, 1e-5, inv, False, x, pool, table)
            out = attend_all(q, pool, table, [at[b] + lens[b] for b in live], [lens[b] for b in live], nh, nkv, hd, page, 0, ws)
            n = 0
            for b in live:
                pieces[b] = torch.cat([pieces[b], out[n:n + lens[b]].float().cpu()])
                n += lens[b]
                at[b] += lens[b]
        done[cut] = (pool.cpu(), torch.cat(pieces))
    for cut in ("halves", "tokens"):
        assert torch.equal(done[cut][0], done["whole"][0])
        a, b = done[cut][1], done["whole"][1]
        # read back in bfloat16 or straight from the codes: 2^-8 a rounding, of scores, weights, values and the result
        assert (a - b).norm() <= 4 * 2.0 ** -8 * b.norm() and (a - b).abs().max() <= 0.06 * b.abs().max()


def test_another_stream_and_recorded_launches():
    """A decode step's launches recorded once and replayed with other lengths, queries and pages; two recordings that share a workspace; a
    stream of the caller's."""
    nh, nkv, hd, page, B = 32, 8, 64, 64, 5
    ws = workspace()
    g = torch.Generator().manual_seed(12)
    recorded = []
    cases = [[70, 300, 1, 64, 500], [512, 2, 65, 128, 129]]
    total = 60
    pool, rk, rv = filled(total, nkv, page, hd, seed=12)
    pool = pool.to(DEV)
    for n_seq in (B, 2):
        q = torch.zeros(n_seq, nh * hd, dtype=torch.bfloat16, device=DEV)
        pos, table, out = ints([0] * n_seq), torch.zeros(n_seq, 8, dtype=torch.int32, device=DEV), torch.zeros_like(q)
        seq, cu = ints(list(range(n_seq))), ints(list(range(n_seq + 1)))

        def go(q=q, pos=pos, table=table, seq=seq, cu=cu, out=out, n_seq=n_seq):
            K().attention_kv4(q, pool, table, pos, seq, cu, pos, out, nh, nkv, hd, hd ** -0.5, 0, ws, [0] * n_seq, [1] * n_seq)
        recorded.append((q, pos, table, out, go))
    for _, _, _, _, go in recorded:                              # the buffers take their sizes
        go()
    graphs = []
    for r in recorded:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            r[4]()
        graphs.append(graph)
    side = torch.cuda.Stream()
    for lengths in cases:
        rows, used = tables(lengths, page, seed=sum(lengths), spare=0)
        assert used <= total
        x = torch.randn(B, nh, hd, generator=g).bfloat16()
        with torch.cuda.stream(side):
            for (q, pos, table, out, _), graph, n_seq in zip(recorded, graphs, (B, 2)):
                q.copy_(x[:n_seq].reshape(n_seq, -1))
                pos.copy_(torch.tensor([n - 1 for n in lengths[:n_seq]], dtype=torch.int32))
                table.zero_()
                table[:, :len(rows[0])] = torch.tensor(rows[:n_seq], dtype=torch.int32, device=DEV)
                out.fill_(float("nan"))
                graph.replay()
        side.synchronize()
        for (q, pos, table, out, _), n_seq in zip(recorded, (B, 2)):
            check(out.view(n_seq, nh, hd), x[:n_seq], rk, rv, rows, lengths[:n_seq], [1] * n_seq, page, 0, torch.bfloat16)
        # the same without a recording, on the caller's stream
        with torch.cuda.stream(side):
            got = attend_all(x, pool, rows, lengths, [1] * B, nh, nkv, hd, page, 0)
        side.synchronize()
        check(got, x, rk, rv, rows, lengths, [1] * B, page, 0, torch.bfloat16)


def test_refusals_on_the_device():
    from mivi_v4_b200.ops.kernels import KernelError
    nh, nkv, hd, page = 4, 2, 64, 16
    pool = torch.zeros(4, nkv, page * (hd + 8), dtype=torch.uint8, device=DEV)
    q = torch.zeros(2, nh * hd, device=DEV)
    a = dict(q=q, pool=pool, page_table=ints([[0, 1]]), positions=ints([0, 1]), seq_of=ints([0, 0]), cu=ints([0, 2]), starts=ints([0]), out=torch.zeros_like(q),
             nh=nh, nkv=nkv, hd=hd, scale=0.1, window=0, ws=workspace(), host_starts=[0], host_lens=[2])
    for over, match in ((dict(host_starts=[40]), "reaches 32"), (dict(page_table=ints([0, 1])), "page table"), (dict(positions=ints([0])), "positions"),
                        (dict(out=torch.zeros(nh * hd, 2, device=DEV).t()), "contiguous"), (dict(q=q.half(), out=q.half()), "float32 and bfloat16"),
                        (dict(splits=0), "key splits"), (dict(cu=ints([0, 2, 2])), "cu"), (dict(pool=pool.cpu()), "CUDA devices only"),
                        (dict(q=torch.zeros(2 * nh * hd + 1, device=DEV)[1:].view(2, -1)), "16 bytes"), (dict(page_table=ints([[0, 1]])[:0]), "sequences")):
        with pytest.raises(KernelError, match=match):
            K().attention_kv4(**{**a, **over})
    with pytest.raises(KernelError, match="16 bytes"):
        K().kv4_read(pool, ints([[0]]), ints([0]), ints([0]), torch.zeros(nkv * hd + 1, device=DEV)[1:].view(1, nkv, hd), torch.zeros(1, nkv, hd, device=DEV), nkv, hd)
    with pytest.raises(KernelError, match="16 bytes"):
        K().kv4_prepare(torch.zeros((nh + 2 * nkv) * hd + 1, device=DEV)[1:].view(1, -1), None, None, 0.0, None, False, ints([0]), ints([0]), ints([[0]]), pool,
                        torch.zeros(1, nh * hd, device=DEV), nh, nkv, hd)
    # a step of nothing
    K().attention_kv4(q[:0], pool, ints([[0, 1]]), ints([]), ints([]), ints([0]), ints([]), q[:0], nh, nkv, hd, 0.1, 0, workspace(), [], [])
