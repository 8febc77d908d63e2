"""The 4-bit cache without a GPU: its layout, its bookkeeping, how a step's sequences are dealt out, and what is refused."""
import pytest
import torch

import plain_kv4 as Q
from mivi_v4_b200.cache import CacheError, KVNeed, SequenceCache, plan_cache
from mivi_v4_b200.cache.cache import rows_of_4_bits
from mivi_v4_b200.ops import kernels as K
from mivi_v4_b200.ops.kernels import KernelError


def ints(v):
    return torch.tensor(v, dtype=torch.int32)


@pytest.mark.parametrize("nkv,hd,page", [(1, 8, 1), (2, 64, 64), (3, 40, 4), (1, 256, 2)])
def test_rows_of_pages(nkv, hd, page):
    g = torch.Generator().manual_seed(hd)
    k, v = torch.randn(5, nkv, page, hd, generator=g), 3 * torch.randn(5, nkv, page, hd, generator=g)
    v[1, 0, 0] = 2.5                                             # a row of one value: step 0
    k[2, 0, 0, 3] = float("inf")                                 # stands for NaN throughout
    pool = Q.pool_bytes(k, v)
    assert pool.shape == (5, nkv, K.kv4_page_bytes(page, hd))
    got = rows_of_4_bits(pool, page, hd)
    wk, wv = Q.rows_of(pool, page, hd)
    # float32: step * code is exact in 12 bits, one rounding of the sum
    assert torch.equal(got[:, 0].isnan(), wk.isnan()) and got[2, 0, 0, 0].isnan().all() and got[:, 0].isnan().sum() == hd
    assert torch.allclose(got.double(), torch.stack([wk, wv], 1), rtol=2.0 ** -23, atol=1e-30, equal_nan=True)
    assert float((got[1, 1, 0, 0] - 2.5).abs().max()) == 0.0
    # a row is off by half a step, or where a number's own rounding (2^-8 of it) moves its ends
    for x, y in ((k, wk), (v, wv)):
        code, step, zero = Q.hold(x)
        fine = torch.isfinite(step).expand_as(y)
        room = (0.5 * step + 15 * 2.0 ** -8 * step + 2.0 ** -8 * zero.abs()).expand_as(y)
        assert ((x.double() - y).abs() <= room)[fine].all()


def test_storage_bookkeeping_and_dump():
    needs = [KVNeed(2, 16, bits=4), KVNeed(2, 16), KVNeed(2, 16, bits=4), KVNeed(2, 16, 3, bits=4)]
    c = SequenceCache(plan_cache(needs, [None] * 4), n_slots=2, n_pages=6, page_size=4, dtype=torch.float32, device="cpu")
    assert len(c.plan.groups) == 3 and c.storage[0].shape == (2, 6, 2, 4 * 24) and c.storage[0].dtype == torch.uint8
    assert c.storage[1].dtype == torch.float32 and c.bytes() == 2 * 6 * 2 * 96 + 6 * 2 * 2 * 4 * 16 * 4 + 6 * 2 * 96
    s = c.assign()
    c.reserve(s, 7)
    g = torch.Generator().manual_seed(1)
    rows = torch.randn(2, 6, 2, 4, 16, generator=g)              # K or V
    for layer in range(2):
        c.storage[0][layer] = Q.pool_bytes(rows[0] + layer, rows[1] - layer)
    c.advance(s, 7)
    got = c.dump_slot(s)[0]
    assert got.shape == (2, 2, 7, 2, 16) and got.dtype == torch.float32
    for layer in range(2):
        for j, x in enumerate((rows[0] + layer, rows[1] - layer)):
            want = Q.sequence(Q.held(x), c.page_rows(0, [s])[0], 7)
            assert torch.allclose(got[layer, j].double(), want, rtol=1e-6, atol=1e-6)
    # the group behind a window gives pages back like any other
    assert c.page_rows(2, [s])[0][0] == 0 and c._seq[s].pages[2][0] is None
    c.check()
    c.release(s)
    c.check()


def test_a_model_says_which_caches_it_can_hold():
    from mivi_v4_b200.engine.model import Model, describe_config
    from mivi_v4_b200.cache import StateNeed
    from tiny_configs import TINY_A
    from votavik_configs import CONFIGS as VOTAVIK
    m = Model(describe_config(TINY_A)[1])
    plan = m.cache_plan("int4")
    assert [g.need.bits for g in plan.groups if isinstance(g.need, KVNeed)] == [4]
    assert [g.need for g in plan.groups if isinstance(g.need, StateNeed)] == [g.need for g in m.cache_plan().groups if isinstance(g.need, StateNeed)]
    assert [g.need.bits for g in m.cache_plan().groups if isinstance(g.need, KVNeed)] == [0]
    with pytest.raises(ValueError, match="known"):
        m.cache_plan("int3")
    with pytest.raises(CacheError, match="model's dtype only"):
        Model(describe_config(VOTAVIK["P"][0])[1]).cache_plan("int4")


def test_bytes_a_token_of_the_measurement():
    from mivi_v4_b200.engine.model import Model, describe_config
    from mivi_v4_b200.measure import model_numbers
    from tiny_configs import TINY_F
    m = Model(describe_config(TINY_F)[1])
    m.dtype = torch.bfloat16
    assert model_numbers(m)["kv_bytes_per_token"] == 2 * 1 * 2 * 64 * 2
    assert model_numbers(m, "int4")["kv_bytes_per_token"] == 2 * 1 * (64 + 8)


def test_command_line_takes_the_cache_dtype():
    from mivi_v4_b200.cli import build_parser
    p = build_parser()
    assert p.parse_args(["generate", "-m", "x", "--cache-dtype", "int4"]).cache_dtype == "int4"
    assert p.parse_args(["bench", "-m", "x"]).cache_dtype is None
    assert p.parse_args(["replay", "--model", "x", "--dtype", "float32", "--out", "o", "--max-tokens", "4", "--cache-dtype", "int4"]).cache_dtype == "int4"
    with pytest.raises(SystemExit):
        p.parse_args(["generate", "-m", "x", "--cache-dtype", "int3"])


def test_how_sequences_are_dealt_out(monkeypatch):
    few, many = K.KV4_DIRECT_TOKENS, K.KV4_DIRECT_TOKENS + 1
    assert K.kv4_runs([], [], 0, 64, 100) == []
    assert K.kv4_runs([5, 0, 900], [1, few, 3], 0, 64, 100) == [(0, 3, 0)]
    # 64-row pages: 100 + 17 rows are 2 pages, 0 + 65 are 2
    assert K.kv4_runs([100, 0, 7, 100], [many, 65, 1, many], 0, 64, 100) == [(0, 2, 4), (2, 3, 0), (3, 4, 2)]
    # behind a window of 10 the pages before the first query's first key stay out: 129 - 9 = 120 lies in page 1 of 0..2
    assert K.kv4_runs([129], [many], 10, 64, 100) == [(0, 1, 2)]
    # what is read back together is bounded; one sequence alone may be more
    monkeypatch.setattr(K, "KV4_READ_BYTES", 500)
    assert K.kv4_runs([640, 64, 64], [many] * 3, 0, 64, 100) == [(0, 1, 11), (1, 3, 4)]


def test_work_of_many_tokens_is_shared_out():
    """Launches take all sequences in order, no more tiles or sequences than one launch can, and no more blocks than there is work."""
    plan, most = K.attention_kv4_prefill_plan, K.KV4_PREFILL_MOST
    for starts, lens, group, nkv, window in (((0,), (2048,), 4, 8, 0), ((6000, 12000), (700, 400), 4, 8, 0), ((0,), (17,), 1, 1, 0), ((9, 0), (20, 300), 3, 2, 50),
                                             ((0,) * 3000, (17,) * 3000, 2, 1, 0), ((0,) * 9, (200 * 256,) * 9, 1, 1, 0)):
        made, b = plan(starts, lens, group, nkv, window), 0
        for n, tiles, whole, blocks in made:
            assert 1 <= n <= most and 1 <= tiles <= most and tiles == sum(-(-m * group // 256) for m in lens[b:b + n])
            assert 1 <= blocks <= (min(K.n_sms(), tiles * nkv) if whole else K.n_sms())
            b += n
        assert b == len(lens)
    assert plan((0,), (2048,), 4, 8, 0)[0][2] and not plan((6000, 12000), (700, 400), 4, 8, 0)[0][2]


def _args(nh=4, nkv=2, hd=16, page=4, n=3, pages=5, **over):
    a = dict(qkv=torch.zeros(n, (nh + 2 * nkv) * hd), wq=torch.ones(hd), wk=torch.ones(hd), eps=1e-5, inv_freq=torch.ones(hd // 2),
             half_split=False, positions=ints(list(range(n))), seq_of=ints([0] * n), page_table=ints([[1, 2]]),
             pool=torch.zeros(pages, nkv, page * (hd + 8), dtype=torch.uint8), q_out=torch.zeros(n, nh * hd), nh=nh, nkv=nkv, hd=hd)
    a.update(over)
    return a


@pytest.mark.parametrize("over,match", [
    (dict(hd=20), "multiple of 8"), (dict(hd=264), "at most 256"), (dict(nkv=0), "kv heads"), (dict(pool=torch.zeros(5, 3, 96, dtype=torch.uint8)), "uint8"), (dict(nh=0), "heads"),
    (dict(pool=torch.zeros(5, 2, 4 * 24)), "uint8"), (dict(pool=torch.zeros(5, 2, 100, dtype=torch.uint8)), "uint8"),
    (dict(pool=torch.zeros(5, 2, 3 * 24, dtype=torch.uint8)), "power of two"), (dict(pool=torch.zeros(5, 2, 0, dtype=torch.uint8)), "uint8"),
    (dict(), "CUDA devices only")])
def test_prepare_refuses(over, match):
    with pytest.raises(KernelError, match=match):
        K.kv4_prepare(**_args(**over))


@pytest.mark.parametrize("over,match", [
    (dict(hd=12), "multiple of 8"), (dict(nkv=1), "uint8"), (dict(v_out=torch.zeros(3, 2, 16, dtype=torch.bfloat16)), "v out"), (dict(), "CUDA devices only")])
def test_read_refuses(over, match):
    a = dict(pool=torch.zeros(5, 2, 4 * 24, dtype=torch.uint8), page_table=ints([[1, 2]]), positions=ints([0, 1, 2]), seq_of=ints([0, 0, 0]),
             k_out=torch.zeros(3, 2, 16), v_out=torch.zeros(3, 2, 16), nkv=2, hd=16)
    a.update(over)
    with pytest.raises(KernelError, match=match):
        K.kv4_read(**a)


@pytest.mark.parametrize("over,match", [
    (dict(hd=20), "multiple of 8"), (dict(nh=3), "not a multiple"), (dict(nh=0), "not a multiple"), (dict(out=torch.zeros(3, 64).bfloat16()), "agree"),
    (dict(host_lens=[4]), "3 rows"), (dict(host_lens=[3, 0], host_starts=[0, 0]), "a token or more"), (dict(host_starts=[0, 1]), "2 starts"),
    (dict(scale=0.0), "positive"), (dict(scale=-0.1), "positive"), (dict(scale=float("nan")), "positive"), (dict(splits=0), "key splits"),
    (dict(), "CUDA devices only")])
def test_attention_refuses(over, match):
    a = dict(q=torch.zeros(3, 64), pool=torch.zeros(5, 2, 4 * 24, dtype=torch.uint8), page_table=ints([[1, 2]]), positions=ints([0, 1, 2]),
             seq_of=ints([0, 0, 0]), cu=ints([0, 3]), starts=ints([0]), out=torch.zeros(3, 64), nh=4, nkv=2, hd=16, scale=0.25, window=0,
             ws=None, host_starts=[0], host_lens=[3])
    a.update(over)
    with pytest.raises(KernelError, match=match):
        K.attention_kv4(**a)
