"""Attention over the 4-bit cache, held to what each query weighs: a result may be off by a share of the sum of weight times value size, so a row
that a query does not see, or gives no weight, has no say in how far off it may be, however large its values or keys are."""
import pytest
import torch

import plain_kv4 as Q
from test_kv4_gpu import DEV, K, attend_all, tables

pytestmark = pytest.mark.gpu


def kernel_of(dtype, hd, page, lens, m):
    """How a sequence of ``m`` tokens in a step of ``lens`` is attended to: "core" (CUDA cores), "codes" (few tokens), "half" (many tokens), "back"
    (read back in the model's dtype)."""
    fused = dtype == torch.bfloat16 and hd <= 64
    if max(lens) > 16 and fused:
        return "half" if m > 16 else "codes"
    if dtype == torch.bfloat16 and page >= 16:
        return "codes"
    return "back" if m > 256 and hd <= 128 else "core"


def weighed(q, k, v, first, window, dtype, form):
    """(wanted, how far off a result may be, whether the mean of what is seen is out of that) of the queries [m, nh, hd] at positions first, first + 1, ...

    A score of query q and key k may be off by scale times: the query's rounding (codes: whole numbers of 16 bits whose largest is 2^14 or more, so
    2^-15 of the largest element an element; half, back: none to speak of), the key's (half: 2^-11 of an element and, below half's normal numbers, 15 * 2^-25 for a
    row whose largest is 2 or more, rows of 2^12 times its size sharing its power of two: 2^-22 of it; query elements 2^-11; back in bfloat16: 2^-8), and sums in 32 bits, hd
    steps of 2^-24 of sum |q| (|zero| + 15 step), taken as twice sum |q| max |k|.  A score off by e makes its weight off by exp(e) - 1.  Weights are rounded
    by 2^-11 (codes, half) or 2^-8 (back in bfloat16), values by 2^-11 + 2^-22 of the row's largest (half) or 2^-8 (back); sums of T weighted
    values and T weights in 32 bits, 4 sqrt(T) 2^-24, the exponential's last places 2^-20.  The result's own rounding is 2^-8 or 2^-24 of it, and below
    bfloat16's or float32's normal numbers nothing is asked for."""
    m, nh, hd = q.shape
    T, nkv = k.shape[:2]
    G, scale = nh // nkv, hd ** -0.5
    q, k, v = q.double(), k.double(), v.double()
    bf = dtype == torch.bfloat16
    at, t = torch.arange(first, first + m)[:, None], torch.arange(T)[None, :]
    hidden = (t > at) | ((t <= at - window) if window > 0 else torch.zeros_like(t > at))
    want, room, mean = (torch.zeros(m, nh, hd, dtype=torch.float64) for _ in range(3))
    seen = (~hidden).double()
    for h in range(nh):
        kk, vv, qq = k[:, h // G], v[:, h // G], q[:, h]
        s = (qq @ kk.T * scale).masked_fill(hidden, -torch.inf)
        logp = s - torch.logsumexp(s, -1, keepdim=True)
        p = logp.exp()
        mags, k_top, q_sum, q_top = qq.abs() @ kk.abs().T, kk.abs().amax(-1), qq.abs().sum(-1, keepdim=True), qq.abs().amax(-1, keepdim=True)
        e = 2 * hd * 2.0 ** -24 * 2 * q_sum * k_top
        if form == "codes":
            e = e + 2.0 ** -15 * q_top * kk.abs().sum(-1)
        if form == "half":
            e = e + 2 * 2.0 ** -11 * mags + 2.0 ** -22 * q_sum * k_top
        if form == "back" and bf:
            e = e + 2.0 ** -8 * mags
        off = ((logp + e * scale).exp() - p).clamp_max(1.0) + 2.0 ** -20 * p
        v_top = vv.abs().amax(-1)
        want[:, h] = p @ vv
        lost = off.sum(-1, keepdim=True)
        open_ = lost > 0.5                                       # (scores too large to be told apart: only a mean of what is seen is asked for)
        lost = lost.clamp_max(0.5)
        weight = {"core": 0.0, "codes": 2.0 ** -11, "half": 2 * 2.0 ** -11 + 2.0 ** -22, "back": 2 * 2.0 ** -8 if bf else 0.0}[form] + 4 * T ** 0.5 * 2.0 ** -24
        room[:, h] = (off @ vv.abs() + lost * want[:, h].abs()) / (1 - lost) + weight * (p @ v_top)[:, None]
        room[:, h] += open_ * 2 * (seen * v_top).amax(-1, keepdim=True)
        mean[:, h] = (seen @ vv) / seen.sum(-1, keepdim=True)
    room += (2.0 ** -8 if bf else 2.0 ** -23) * want.abs() + 2.0 ** -125
    return want, room, (((mean - want).abs() > room) & (want.abs() > room)).flatten(1).any(-1)


def hold_to_weights(out, q, ks, vs, lens, before, window, dtype, page, teeth=0.9, forms=None):
    """Every row of the step against the formula; ks, vs: what the sequences' rows stand for; forms: a sequence's kernel where it is not the usual one."""
    n = telling = 0
    for b, (m, first) in enumerate(zip(lens, before)):
        form = forms or kernel_of(dtype, q.shape[-1], page, lens, m)
        want, room, tells = weighed(q[n:n + m], ks[b], vs[b], first, window, dtype, form)
        got = out[n:n + m].double().cpu()
        assert torch.isfinite(got).all(), (b, form)
        share = (got - want).abs() / room
        assert (share <= 1).all(), (b, form, "row %d head %d" % divmod(int(share.amax(-1).argmax()), q.shape[1]), float(share.max()))
        telling += int(tells.sum()) + (1 if first == 0 else 0)   # (a query that sees one row gets that row)
        n += m
    assert telling >= teeth * n, (telling, n)                    # zeros, or the mean of the values, would not have passed


def in_pages(xs, page, seed, spare=2):
    """Sequences' rows (keys, values) [L, nkv, hd] -> pool, page table, what the rows stand for."""
    rows, total = tables([k.shape[0] for k, _ in xs], page, seed, spare)
    nkv, hd = xs[0][0].shape[1:]
    whole = torch.full((2, total, nkv, page, hd), 3.0)           # spare pages and stale rows: other values
    for (k, v), row in zip(xs, rows):
        for j, x in enumerate((k, v)):
            for i in range(0, x.shape[0], page):
                whole[j, row[i // page], :, :len(x[i:i + page])] = x[i:i + page].transpose(0, 1)
    pool = Q.pool_bytes(whole[0], whole[1])
    rk, rv = Q.rows_of(pool, page, hd)
    return pool, rows, [Q.sequence(rk, r, k.shape[0]) for (k, _), r in zip(xs, rows)], [Q.sequence(rv, r, k.shape[0]) for (k, _), r in zip(xs, rows)]


# name: dtype, heads, kv heads, head size, page, window, tokens, cached before, ways to share (of the many-token kernel)
SHAPES = {
    "one token": (torch.bfloat16, 8, 2, 64, 64, 0, [1, 1], [300, 70], None),
    "one token, small head": (torch.bfloat16, 4, 4, 40, 16, 0, [1, 1], [300, 70], None),
    "one token, wide heads": (torch.bfloat16, 32, 1, 128, 32, 0, [1] * 20, [90 + 7 * b for b in range(20)], None),
    "one token, widest heads": (torch.bfloat16, 16, 1, 256, 16, 0, [1] * 40, [70 + b for b in range(40)], None),
    "one token, window": (torch.bfloat16, 8, 2, 64, 64, 50, [1, 1], [300, 71], None),
    "short runs": (torch.bfloat16, 8, 2, 64, 64, 0, [4, 16, 1], [100, 3, 260], None),
    "short runs, window": (torch.bfloat16, 4, 4, 64, 16, 10, [14, 9], [200, 3], None),
    "short runs, many": (torch.bfloat16, 8, 1, 64, 64, 0, [13] * 24, [5 * b for b in range(24)], None),
    "many tokens": (torch.bfloat16, 8, 2, 64, 64, 0, [200, 33, 7], [0, 300, 20], "planned"),
    "many tokens, whole": (torch.bfloat16, 4, 2, 64, 16, 0, [270], [130], "whole"),
    "many tokens, shared": (torch.bfloat16, 4, 2, 64, 64, 0, [270, 40], [130, 500], "shared"),
    "many tokens, few blocks": (torch.bfloat16, 6, 2, 64, 64, 30, [270, 40], [130, 500], "few blocks"),
    "many tokens, window": (torch.bfloat16, 3, 1, 64, 1, 40, [300], [100], "planned"),
    "many tokens, small head": (torch.bfloat16, 6, 2, 48, 64, 0, [100, 140], [200, 0], "shared"),
    "many tokens, large head": (torch.bfloat16, 4, 2, 128, 64, 0, [90, 200], [200, 0], None),
    "many tokens, large head, window": (torch.bfloat16, 6, 2, 96, 32, 45, [150], [100], None),
    "small pages": (torch.bfloat16, 4, 2, 96, 8, 0, [60, 20], [40, 90], None),
    "small pages, read back": (torch.bfloat16, 4, 2, 96, 8, 0, [270, 20], [40, 90], None),
    "small pages, read back, window": (torch.bfloat16, 4, 2, 80, 1, 40, [270, 300], [40, 0], None),
    "float32": (torch.float32, 8, 2, 64, 64, 0, [1, 5, 40], [300, 20, 0], None),
    "float32, read back": (torch.float32, 3, 1, 64, 64, 70, [270, 3], [60, 100], None),
    "float32, read back, large head": (torch.float32, 2, 1, 128, 16, 0, [270], [60], None),
}


def shared_out(monkeypatch, way):
    plan = K().attention_kv4_prefill_plan

    def forced(starts, ms, group, kv_heads, w):
        blocks = lambda tiles: {"whole": min(148, tiles * kv_heads), "shared": 148, "few blocks": 7}[way]      # noqa: E731
        return [(n, tiles, way == "whole", blocks(tiles)) for n, tiles, _, _ in plan(starts, ms, group, kv_heads, w)]
    if way not in (None, "planned"):
        monkeypatch.setattr(K(), "attention_kv4_prefill_plan", forced)


def queries_and_rows(shape, seed):
    """Queries that all lean one way (u): a key against it scores some 80 below the others, one with it some 30 above."""
    dtype, nh, nkv, hd, page, window, lens, before, _ = shape
    g = torch.Generator().manual_seed(seed)
    u = torch.sign(torch.randn(hd, generator=g)) / hd ** 0.5
    lean = (80 * hd ** 0.5) ** 0.5
    q = (lean * u + 0.5 * torch.randn(sum(lens), nh, hd, generator=g)).to(dtype)
    xs = [(0.5 * torch.randn(m + c, nkv, hd, generator=g), torch.randn(m + c, nkv, hd, generator=g)) for m, c in zip(lens, before)]
    return q, xs, lean * u


def run(shape, q, xs, seed=1):
    dtype, nh, nkv, hd, page, window, lens, before, _ = shape
    pool, rows, ks, vs = in_pages(xs, page, seed)
    out = attend_all(q, pool.to(DEV), rows, [m + c for m, c in zip(lens, before)], lens, nh, nkv, hd, page, window)
    return out, ks, vs


@pytest.mark.parametrize("name", SHAPES)
def test_ordinary_rows(monkeypatch, name):
    """Rows of ordinary sizes, and values whose sizes change a lot from row to row."""
    shape = SHAPES[name]
    dtype, nh, nkv, hd, page, window, lens, before, way = shape
    shared_out(monkeypatch, way)
    q, xs, _ = queries_and_rows(shape, 1)
    for spread in (0.0, 1.0, 4.0):
        g = torch.Generator().manual_seed(2)
        ys = [(k, v * torch.exp(spread * torch.randn(v.shape[0], nkv, 1, generator=g))) for k, v in xs]
        out, ks, vs = run(shape, q, ys)
        hold_to_weights(out, q, ks, vs, lens, before, window, dtype, page)


@pytest.mark.parametrize("power", [12, 16, 20, 24, 60, 100])
@pytest.mark.parametrize("name,where", [(n, w) for n, x in SHAPES.items() for w in ("later", "behind", "unweighted")
                                        if not (w == "later" and max(x[6]) == 1) and not (w == "behind" and not x[5])])
def test_one_large_value_row(monkeypatch, name, where, power):
    """One value row of each sequence, 2^power times as large as the others: the last token's (those before it do not see it) and one in mid-run; one that
    is behind some or all windows; one that every query sees with a score some 80 below the best."""
    shape = SHAPES[name]
    dtype, nh, nkv, hd, page, window, lens, before, way = shape
    shared_out(monkeypatch, way)
    q, xs, along = queries_and_rows(shape, 3)
    for (k, v), m, c in zip(xs, lens, before):
        if where == "later":
            big = [c + m - 1] + ([c + m // 2] if m > 2 and power > 60 else [])
            if m == 1:
                continue
        elif where == "behind":
            big = [max(0, c - window)]
        else:
            big = [min(c + m - 1, 33) if c > 40 else 0]
            k[big] = -along
        v[big] *= 2.0 ** power
    out, ks, vs = run(shape, q, xs)
    hold_to_weights(out, q, ks, vs, lens, before, window, dtype, page, teeth=0.5)


# (2^60: scores that 32 bits round by more than an exponential takes.  The kernels that rows read back in bfloat16 go to, those of a bfloat16
# cache, are not made for them.)
@pytest.mark.parametrize("name,power", [(n, p) for n, x in SHAPES.items() for p in (12, 20, 40, 60)
                                        if not (p > 20 and x[0] == torch.bfloat16 and n.startswith("small pages, read back"))])
def test_one_large_key_row(monkeypatch, name, power):
    """One key row 2^power times as large as the others: the last token's, or one behind a window, whose value is small; and one that every query sees far
    below the best."""
    shape = SHAPES[name]
    dtype, nh, nkv, hd, page, window, lens, before, way = shape
    shared_out(monkeypatch, way)
    q, xs, along = queries_and_rows(shape, 4)
    for (k, v), m, c in zip(xs, lens, before):
        k[c + m - 1 if m > 1 else 0] *= 2.0 ** power
        k[max(0, c - 1)] = -along * 2.0 ** power
    out, ks, vs = run(shape, q, xs)
    # (whose own score is of the large row's size cannot be told by 32 bits, or by anybody's rounding: they are held to that)
    hold_to_weights(out, q, ks, vs, lens, before, window, dtype, page, teeth=0.4)


@pytest.mark.parametrize("below", [8, 25, 40])
@pytest.mark.parametrize("name", SHAPES)
def test_most_weight_on_a_row_of_zeros(monkeypatch, name, below):
    """One row of each sequence takes nearly all of the weight, the others score ``below`` under it, and its values are zero: what is left is
    the others', as exact as ever."""
    shape = SHAPES[name]
    dtype, nh, nkv, hd, page, window, lens, before, way = shape
    shared_out(monkeypatch, way)
    q, xs, along = queries_and_rows(shape, 5)
    for (k, v), m, c in zip(xs, lens, before):
        at = 0 if not window else max(0, c - 3)
        k *= 0.2
        k[at] = along * below / 80
        v[at] = 0.0
    out, ks, vs = run(shape, q, xs)
    hold_to_weights(out, q, ks, vs, lens, before, window, dtype, page)


@pytest.mark.parametrize("name", SHAPES)
def test_values_of_every_size(monkeypatch, name):
    """Values from 2^-100 to 2^100, row by row, in every order, and a row of zeros now and then."""
    shape = SHAPES[name]
    dtype, nh, nkv, hd, page, window, lens, before, way = shape
    shared_out(monkeypatch, way)
    q, xs, along = queries_and_rows(shape, 6)
    g = torch.Generator().manual_seed(7)
    for seed in range(3):
        ys = []
        for k, v in xs:
            powers = torch.randint(-100, 101, (v.shape[0], nkv, 1), generator=g).float()
            if seed == 1:
                powers = powers.sort(dim=0).values
            if seed == 2:
                powers = powers.sort(dim=0, descending=True).values
            v = v * torch.exp2(powers)
            v[torch.rand(v.shape[0], generator=g) < 0.05] = 0.0
            ys.append((k, v))
        out, ks, vs = run(shape, q, ys)
        hold_to_weights(out, q, ks, vs, lens, before, window, dtype, page, teeth=0.5)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("nh,nkv,hd,page,window", [(32, 8, 64, 64, 0), (3, 1, 64, 64, 0), (6, 2, 128, 16, 0), (5, 5, 48, 32, 50), (8, 2, 64, 64, 70),
                                                   (4, 2, 40, 8, 0), (2, 1, 256, 64, 0), (16, 8, 96, 64, 0), (4, 2, 96, 8, 0), (3, 1, 80, 1, 60), (2, 1, 256, 8, 0)])
@pytest.mark.parametrize("lens", [[17, 1, 300], [260, 140], [3, 64, 16, 17, 1]])
def test_runs_of_all_lengths(dtype, nh, nkv, hd, page, window, lens):
    """More than 16 tokens, and steps with both, of every head size, type and page size: over the codes, on tcgen05 and read back."""
    before = [0, 200, 63, 64, 1][:len(lens)]
    shape = (dtype, nh, nkv, hd, page, window, lens, before, None)
    g = torch.Generator().manual_seed(nh + sum(lens))
    xs = []
    for m, c in zip(lens, before):                               # keys with a channel that stands out, values whose size changes from row to row
        k, v = torch.randn(2, m + c, nkv, hd, generator=g)
        k[..., 0] *= 4
        xs.append((k, v * torch.exp(torch.randn(m + c, nkv, 1, generator=g))))
    q = torch.randn(sum(lens), nh, hd, generator=g).to(dtype)
    out, ks, vs = run(shape, q, xs)
    hold_to_weights(out, q, ks, vs, lens, before, window, dtype, page)


def test_more_rows_than_the_tables_of_the_many_token_kernel_hold(monkeypatch):
    """Such a step goes over the codes."""
    monkeypatch.setattr(K(), "KV4_PREFILL_MOST", 4)
    monkeypatch.setattr(K(), "_attention_kv4_prefill", None)
    shape = (torch.bfloat16, 8, 1, 64, 64, 0, [130], [0], None)
    q, xs, _ = queries_and_rows(shape, 8)
    out, ks, vs = run(shape, q, xs)
    hold_to_weights(out, q, ks, vs, [130], [0], 0, torch.bfloat16, 64, forms="codes")


def test_the_bound_has_teeth():
    """Zeros, and the mean of what is seen, are out of it by far; a result that is right to its last place is within it."""
    for dtype, hd, form in ((torch.bfloat16, 128, "codes"), (torch.bfloat16, 64, "half"), (torch.bfloat16, 96, "back"), (torch.float32, 64, "core"),
                            (torch.float32, 96, "back")):
        shape = (dtype, 4, 2, hd, 64, 0, [40], [460], None)
        q, xs, _ = queries_and_rows(shape, 9)
        _, _, (k,), (v,) = in_pages(xs, 64, 1)
        want, room, tells = weighed(q, k, v, 460, 0, dtype, form)
        assert tells.all() and ((want.to(dtype).double() - want).abs() <= room).all()
        assert float(room.max()) < (0.5 if form == "back" else 0.1) * float(want.abs().max())
