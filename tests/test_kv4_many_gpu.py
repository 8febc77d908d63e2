"""Attention of many tokens a step over the 4-bit cache: the tcgen05 kernel of heads of 64 in both of its ways to share the work, long runs of
head sizes that only the kernel for few tokens takes, and short runs behind long contexts."""
import math

import pytest
import torch

import plain_kv4 as Q
from test_kv4_gpu import DEV, K, attend_all, check, filled, ints, tables, workspace

pytestmark = pytest.mark.gpu


def held_to_half(out, q, rk, rv, rows, lengths, lens, page, window, which):
    """Against the formula in float64, as exact as operands of 11 bits allow.  Queries and keys are rounded by 2^-11 each, so a score is off by
    2^-10 scale sum |q||k| and a weight by as much again for the sum; weights are rounded by 2^-11 and values by 2^-11, and a value's powers of
    two are of 32 neighbours, below which half precision's subnormal numbers are 2^-24 apart; sums in float32 add a few 2^-24.  The result's
    own rounding is 2^-8 of it."""
    nh, hd = q.shape[1:]
    nkv = rk.shape[1]
    first = [sum(lens[:b]) for b in range(len(lens))]
    for b, i in which:
        L, m = lengths[b], lens[b]
        k, v = Q.sequence(rk, rows[b], L), Q.sequence(rv, rows[b], L)
        pos, n = L - m + i, first[b] + i
        want = Q.attend(q[n].double(), k, v, pos, hd ** -0.5, window)
        lo = max(0, pos - window + 1) if window > 0 else 0
        for h in range(nh):
            kk, vv = k[lo:pos + 1, h // (nh // nkv)], v[lo:pos + 1, h // (nh // nkv)]
            mags = float((kk.abs() @ q[n, h].double().abs()).max()) * hd ** -0.5
            top = float(vv.abs().max())
            room = (2 * math.expm1(2.0 ** -10 * mags) + 2 * 2.0 ** -11 + 16 * 2.0 ** -24 * (mags + 8)) * top + 2.0 ** -8 * want[h].abs()
            got = out[n, h].double().cpu()
            assert torch.isfinite(got).all() and ((got - want[h]).abs() <= room).all(), (b, i, h, float(((got - want[h]).abs() / room).max()))


def some(lens, every=41):
    return [(b, i) for b, m in enumerate(lens) for i in range(m) if i in (0, m - 1) or i % every == 7]


@pytest.mark.parametrize("way", ["planned", "whole", "shared", "few blocks", "one block"])
@pytest.mark.parametrize("nh,nkv,page,window,lens,before", [
    (8, 2, 64, 0, [300, 17, 64], [0, 1000, 129]), (5, 1, 1, 0, [70], [63]), (3, 3, 16, 0, [129, 128], [0, 127]), (32, 1, 128, 0, [40, 19], [200, 0]),
    (14, 2, 32, 90, [200, 33], [700, 0]), (8, 8, 256, 1, [65, 300], [0, 63]), (6, 2, 64, 500, [513], [1024]), (1, 1, 64, 0, [1000], [24])])
def test_both_ways_to_share_the_work(monkeypatch, way, nh, nkv, page, window, lens, before):
    """Tiles cut in mid-key by any number of blocks, tiles of several blocks, halves without a row, and whole tiles back and forth."""
    lengths = [a + m for a, m in zip(before, lens)]
    rows, total = tables(lengths, page, seed=nh + page)
    pool, rk, rv = filled(total, nkv, page, 64, seed=nh + sum(lens))
    q = torch.randn(sum(lens), nh, 64, generator=torch.Generator().manual_seed(6)).bfloat16()
    plan = K().attention_kv4_prefill_plan

    def forced(starts, ms, group, kv_heads, w):
        made = []
        for n, tiles, _, _ in plan(starts, ms, group, kv_heads, w):
            blocks = {"whole": min(148, tiles * kv_heads), "shared": 148, "few blocks": 7, "one block": 1}[way]
            made.append((n, tiles, way == "whole", blocks))
        return made
    if way != "planned":
        monkeypatch.setattr(K(), "attention_kv4_prefill_plan", forced)
    ws, dev_pool = workspace(), pool.to(DEV)
    out = attend_all(q, dev_pool, rows, lengths, lens, nh, nkv, 64, page, window, ws)
    held_to_half(out, q, rk, rv, rows, lengths, lens, page, window, some(lens))
    for _ in range(3):                                           # counters are back at zero, and the order of blocks changes nothing
        assert torch.equal(out, attend_all(q, dev_pool, rows, lengths, lens, nh, nkv, 64, page, window, ws))


@pytest.mark.parametrize("whole", [True, False])
@pytest.mark.parametrize("nh,nkv,hd,page,window", [(8, 2, 48, 64, 0), (3, 1, 8, 1, 0), (4, 4, 16, 2, 70), (6, 2, 40, 16, 0), (5, 1, 56, 1, 100), (16, 8, 32, 64, 0),
                                                   (24, 1, 24, 128, 0)])
def test_smaller_heads(monkeypatch, whole, nh, nkv, hd, page, window):
    lens, before = [20, 300, 150], [500, 0, 77]
    lengths = [a + m for a, m in zip(before, lens)]
    rows, total = tables(lengths, page, seed=hd)
    pool, rk, rv = filled(total, nkv, page, hd, seed=nh + hd)
    q = torch.randn(sum(lens), nh, hd, generator=torch.Generator().manual_seed(9)).bfloat16()
    plan = K().attention_kv4_prefill_plan
    monkeypatch.setattr(K(), "attention_kv4_prefill_plan", lambda *a: [(n, tiles, whole, min(148, tiles * nkv) if whole else 13) for n, tiles, _, _ in plan(*a)])
    out = attend_all(q, pool.to(DEV), rows, lengths, lens, nh, nkv, hd, page, window)
    held_to_half(out, q, rk, rv, rows, lengths, lens, page, window, some(lens))


def test_a_run_of_more_rows_than_the_tables_hold(monkeypatch):
    """Such a step takes the other kernels."""
    nh, nkv, hd, page, lens, lengths = 8, 1, 64, 64, [130], [130]
    monkeypatch.setattr(K(), "KV4_PREFILL_MOST", 4)
    monkeypatch.setattr(K(), "_attention_kv4_prefill", None)
    rows, total = tables(lengths, page, seed=hd)
    pool, rk, rv = filled(total, nkv, page, hd, seed=nh + hd)
    q = torch.randn(130, nh, hd, generator=torch.Generator().manual_seed(9)).bfloat16()
    check(attend_all(q, pool.to(DEV), rows, lengths, lens, nh, nkv, hd, page, 0), q, rk, rv, rows, lengths, lens, page, 0, torch.bfloat16)


def test_more_sequences_than_a_launch_takes():
    nh, nkv, page, n_seqs = 2, 1, 16, 1100
    lens = [17 + b % 3 for b in range(n_seqs)]
    lengths = [m + (5 * b) % 40 for b, m in enumerate(lens)]
    rows, total = tables(lengths, page, seed=1)
    pool, rk, rv = filled(total, nkv, page, 64, seed=2)
    q = torch.randn(sum(lens), nh, 64, generator=torch.Generator().manual_seed(3)).bfloat16()
    out = attend_all(q, pool.to(DEV), rows, lengths, lens, nh, nkv, 64, page, 0)
    held_to_half(out, q, rk, rv, rows, lengths, lens, page, 0, [(b, b % 17) for b in list(range(0, n_seqs, 29)) + [1022, 1023, 1024, 1025, n_seqs - 1]])
    assert torch.isfinite(out.float()).all()


@pytest.mark.parametrize("nh,nkv,hd,page,window", [(4, 1, 72, 16, 0), (2, 2, 256, 64, 0), (12, 2, 40, 64, 100), (6, 1, 24, 32, 0)])
@pytest.mark.parametrize("lens,before", [([600], [3]), ([7, 255, 1, 300], [10, 5, 0, 64]), ([3] * 120, [1] * 120)])
def test_more_rows_than_a_launch_takes(monkeypatch, nh, nkv, hd, page, window, lens, before):
    """Launches of the kernel for few tokens begin and end within runs, and within what one block takes of a run."""
    monkeypatch.setattr(K(), "attention_kv4_prefill_supported", lambda dtype, hd: False)
    lengths = [a + m for a, m in zip(before, lens)]
    rows, total = tables(lengths, page, seed=hd)
    pool, rk, rv = filled(total, nkv, page, hd, seed=hd + 1)
    q = torch.randn(sum(lens), nh, hd, generator=torch.Generator().manual_seed(7)).bfloat16()
    ends = [n for n in range(sum(lens)) if n % K().KV4_DIRECT_ROWS in (0, 1, 254, 255)]
    first = [sum(lens[:b]) for b in range(len(lens))]
    only = {(b, n - f) for n in ends for b, (f, m) in enumerate(zip(first, lens)) if f <= n < f + m}
    ws = workspace()
    for _ in range(2):
        out = attend_all(q, pool.to(DEV), rows, lengths, lens, nh, nkv, hd, page, window, ws)
        check(out, q, rk, rv, rows, lengths, lens, page, window, torch.bfloat16, pages=False, only=only)


@pytest.mark.parametrize("lens,before", [([40], [1280]), ([17, 60, 2], [544, 1920, 0]), ([40], [1279]), ([20, 200, 30], [700, 100, 1000])])
def test_short_runs_behind_long_contexts(lens, before):
    """Heads of 128: more rows than a launch takes, and fewer."""
    nh, nkv, hd, page = 4, 2, 128, 64
    lengths = [a + m for a, m in zip(before, lens)]
    rows, total = tables(lengths, page, seed=5)
    pool, rk, rv = filled(total, nkv, page, hd, seed=6)
    q = torch.randn(sum(lens), nh, hd, generator=torch.Generator().manual_seed(8)).bfloat16()
    out = attend_all(q, pool.to(DEV), rows, lengths, lens, nh, nkv, hd, page, 0)
    check(out, q, rk, rv, rows, lengths, lens, page, 0, torch.bfloat16, pages=False)


def test_recorded_prompts_and_two_recordings_of_one_workspace():
    """Two steps of many tokens, one whole and one shared, recorded over one workspace and replayed in turn with other queries."""
    nh, nkv, page = 8, 2, 64
    ws, g = workspace(), torch.Generator().manual_seed(4)
    steps = []
    for lens, before in (([300, 40], [0, 2000]), ([700], [100])):
        lengths = [a + m for a, m in zip(before, lens)]
        rows, total = tables(lengths, page, seed=sum(lens))
        pool, rk, rv = filled(total, nkv, page, 64, seed=sum(lens))
        q = torch.zeros(sum(lens), nh * 64, dtype=torch.bfloat16, device=DEV)
        args = (q, pool.to(DEV), ints(rows), ints([s + i for s, m in zip(before, lens) for i in range(m)]),
                ints([b for b, m in enumerate(lens) for _ in range(m)]), ints([sum(lens[:b]) for b in range(len(lens) + 1)]), ints(before),
                torch.empty_like(q), nh, nkv, 64, 0.125, 0, ws, before, lens)
        K().attention_kv4(*args)
        steps.append((args, lens, lengths, rows, rk, rv))
    graphs = []
    for args, *_ in steps:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            K().attention_kv4(*args)
        graphs.append(graph)
    for _ in range(2):
        for (args, lens, lengths, rows, rk, rv), graph in zip(steps, graphs):
            x = torch.randn(sum(lens), nh, 64, generator=g).bfloat16()
            args[0].copy_(x.reshape(sum(lens), -1))
            args[7].fill_(float("nan"))
            graph.replay()
        torch.cuda.synchronize()
        out = args[7].view(-1, nh, 64)
        held_to_half(out, x, rk, rv, rows, lengths, lens, page, 0, some(lens, 97))
    K().check_device_errors()


@pytest.mark.parametrize("qs,ks,vs", [(1e3, 1e3, 1e6), (1e-6, 1.0, 1e-30), (1e20, 1e-20, 1e30), (1e-30, 1e30, 3e37)])
def test_rows_of_any_size(qs, ks, vs):
    """Queries, keys and values far outside half precision's range, values whose sizes change from page to page, equal scores."""
    nh, nkv, page, m = 4, 1, 64, 150
    g = torch.Generator().manual_seed(3)
    total = 5
    k = torch.randn(total, nkv, page, 64, generator=g).clamp(-2, 2) * ks
    v = torch.randn(total, nkv, page, 64, generator=g).clamp(-2, 2) * vs * torch.tensor([1.0, 2.0 ** -9, 1.0, 2.0 ** -20, 4.0]).view(5, 1, 1, 1)
    if qs * ks > 1e3:
        k = k * 1e-6                                             # (scores of some hundreds are as far as they can be told apart)
    pool = Q.pool_bytes(k, v)
    rk, rv = Q.rows_of(pool, page, 64)
    q = (torch.randn(m, nh, 64, generator=g).clamp(-2, 2) * qs).bfloat16()
    out = attend_all(q, pool.to(DEV), [[3, 0, 1, 4, 2]], [300], [m], nh, nkv, 64, page, 0)
    held_to_half(out, q, rk, rv, [[3, 0, 1, 4, 2]], [300], [m], page, 0, some([m], 19))


@pytest.mark.parametrize("dtype,nh,nkv,hd,page,window", [(torch.float32, 4, 2, 64, 64, 0), (torch.float32, 3, 1, 96, 8, 90), (torch.float32, 2, 1, 256, 16, 0),
                                                         (torch.bfloat16, 4, 2, 96, 8, 0), (torch.bfloat16, 2, 2, 80, 1, 40)])
@pytest.mark.parametrize("lens,before", [([256, 3, 257], [70, 0, 10]), ([300], [0]), ([30, 200, 90], [3, 500, 0])])
def test_float32_and_small_pages(dtype, nh, nkv, hd, page, window, lens, before):
    """Over the codes, read back, and both in one step."""
    lengths = [a + m for a, m in zip(before, lens)]
    rows, total = tables(lengths, page, seed=hd)
    pool, rk, rv = filled(total, nkv, page, hd, seed=hd + 2)
    q = torch.randn(sum(lens), nh, hd, generator=torch.Generator().manual_seed(8)).to(dtype)
    out = attend_all(q, pool.to(DEV), rows, lengths, lens, nh, nkv, hd, page, window)
    check(out, q, rk, rv, rows, lengths, lens, page, window, dtype, pages=max(lens) > K().KV4_DIRECT_INSTEAD)


@pytest.mark.parametrize("nh,nkv,hd,page,window", [(16, 1, 64, 64, 0), (32, 1, 64, 16, 0), (12, 1, 48, 32, 70), (20, 1, 96, 64, 0), (16, 2, 128, 64, 0),
                                                   (24, 1, 256, 16, 0), (64, 4, 64, 64, 1 << 40), (6, 1, 16, 64, -1)])
@pytest.mark.parametrize("splits", [None, 3])
def test_many_single_tokens(nh, nkv, hd, page, window, splits):
    """Enough columns of queries for wide tiles: many heads of a kv head, in one tile or several."""
    lengths = [1 + (37 * b) % 400 for b in range(70)]
    lens = [1] * len(lengths)
    rows, total = tables(lengths, page, seed=hd)
    pool, rk, rv = filled(total, nkv, page, hd, seed=nh)
    q = (2 * torch.randn(len(lengths), nh, hd, generator=torch.Generator().manual_seed(2))).bfloat16()
    out = attend_all(q, pool.to(DEV), rows, lengths, lens, nh, nkv, hd, page, window, splits=splits)
    check(out, q, rk, rv, rows, lengths, lens, page, 0 if window > 10 ** 6 else window, torch.bfloat16)
