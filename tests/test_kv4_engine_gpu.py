"""Whole models over the 4-bit cache: what is held, the logits that follow from it, cuts, recordings, generation, the programs."""
import json
import os
import subprocess
import sys

import pytest
import torch

import plain_kv4 as Q
import plain_lfm2 as P
from helpers import assert_close, plain_view64, write_model
from tiny_configs import CONFIGS, LOUD_CONFIGS, config_of, prompts

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def with_held_rows(model_dir, tokens, kv, dtype=torch.float64, rnd=P._same):
    """The plain model's logits, every attention layer reading the rows of ``kv`` [layers, 2, T, kv heads, hd] in place of its own; and the
    keys and values that it would have had itself (after norm and rotation)."""
    cfg, weights = plain_view64(model_dir)
    plain, own = P.plain_attention, []

    def attention(u, *w, **kw):
        kw = {k: v for k, v in kw.items() if k not in ("return_kv", "kv")}
        _, mine = plain(u, *w, **dict(kw, rnd=P._same), return_kv=True)
        own.append(torch.stack(mine))
        rows = kv[len(own) - 1].to(u.dtype)
        return plain(u, *w, **kw, kv=(rows[0], rows[1]), return_kv=True)
    P.plain_attention = attention
    try:
        logits = P.plain_forward(cfg, {k: v.to(dtype) for k, v in weights.items()}, list(tokens), dtype=dtype, rnd=rnd)
    finally:
        P.plain_attention = plain
    return logits.double(), torch.stack(own).double()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("name", ["AL", "BL", "C", "D", "E", "FL"])
def test_logits_follow_from_what_is_held(tmp_path, name, dtype):
    from mivi_v4_b200 import Engine, load_model
    cfg, seed = (CONFIGS.get(name) or LOUD_CONFIGS[name])
    d = write_model(tmp_path, cfg, seed, init="loud" if name in LOUD_CONFIGS else "baseline")
    eng = Engine(load_model(d, dtype, DEV), max_tokens=2048, cache_dtype="int4")
    ps = prompts(cfg["vocab_size"], [150, 5, 70, 1], seed=1)
    slots = [eng.open() for _ in ps]
    got = [[] for _ in ps]
    # prompts in unequal pieces, then token by token
    at = [0] * 4
    for takes in ([100, 2, 17, 1], [30, 1, 16, 0], [1] * 4, [1] * 4, [200] * 4):
        items = [(slots[b], ps[b][at[b]:at[b] + t]) for b, t in enumerate(takes) if ps[b][at[b]:at[b] + t]]
        if not items:
            continue
        lg = eng.step(items, "all")
        n = 0
        for b, t in enumerate(takes):
            m = len(ps[b][at[b]:at[b] + t])
            got[b].append(lg[n:n + m])
            n += m
            at[b] += m
    eng.check_errors()
    g = eng.cache.kv_groups[0]
    for b, p in enumerate(ps):
        kv = eng.cache.dump_slot(slots[b])[g].cpu()
        want, own = with_held_rows(d, p, kv)
        rnd = P.round_to(torch.bfloat16) if dtype == torch.bfloat16 else P._same
        sim, _ = with_held_rows(d, p, kv, torch.float64 if dtype == torch.bfloat16 else torch.float32, rnd)
        noise = float((sim - want).pow(2).mean().sqrt())
        assert_close(torch.cat(got[b]), want, dtype, f"{name} sequence {b}", noise=noise)
        # what is held is what a row of these values is held as: half a step, the numbers' own rounding, and the run's noise in x
        step = Q.hold(own)[1]
        slack = 2.0 ** -5 if dtype == torch.bfloat16 else 1e-4
        room = 0.5 * step + 15 * 2.0 ** -8 * step + (2.0 ** -8 + slack) * own.abs().amax(-1, keepdim=True)
        assert ((kv.double() - own).abs() <= room).all()
    eng.cache.check()


def test_generation_recorded_and_not(tmp_path):
    """Greedy generation replays recorded decode steps; without recordings the same tokens come out, and the cache takes 36 bytes where it took 128."""
    from mivi_v4_b200 import Engine, SamplingParams, load_model
    cfg = config_of("FL")
    d = write_model(tmp_path, cfg, 5, init="loud")
    ps = prompts(cfg["vocab_size"], [130, 3, 64, 20], seed=2)
    model = load_model(d, torch.float32, DEV)
    outs = []
    for graphs in (True, False):
        eng = Engine(model, max_tokens=2048, cuda_graphs=graphs, cache_dtype="int4")
        outs.append(eng.generate(ps, 40, SamplingParams.greedy(), stop_token_ids=[]))
        assert (eng.graph_replays > 20) == graphs
        eng.cache.check()
        held = sum(eng.cache.storage[g].numel() for g in eng.cache.kv_groups)
        bf = Engine(load_model(d, torch.bfloat16, DEV), max_tokens=2048)
        assert held * 128 == 36 * sum(bf.cache.storage[g].numel() * 2 for g in bf.cache.kv_groups)
    assert outs[0] == outs[1] and all(len(o) == 40 for o in outs[0])


def test_slots_are_used_again(tmp_path):
    """A sequence that takes over another's slot and pages sees nothing of it."""
    from mivi_v4_b200 import Engine, load_model
    cfg = config_of("AL")
    d = write_model(tmp_path, cfg, 0, init="loud")
    eng = Engine(load_model(d, torch.float32, DEV), max_tokens=128, max_batch=1, cache_dtype="int4")
    a, b = prompts(cfg["vocab_size"], [100, 90], seed=3)
    s = eng.open()
    eng.step([(s, a)], None)
    eng.close(s)
    s = eng.open()
    used = eng.step([(s, b)], "all")
    fresh = Engine(load_model(d, torch.float32, DEV), max_tokens=128, max_batch=1, cache_dtype="int4")
    assert torch.equal(used, fresh.step([(fresh.open(), b)], "all"))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_windowed_and_shared_layers(dtype):
    """Parts alone: a layer with a window over a 4-bit cache, and a layer with queries only that reads it."""
    from mivi_v4_b200.cache import SequenceCache, plan_cache
    from mivi_v4_b200.engine import StepContext, Workspace
    from mivi_v4_b200.parts.mixers import GroupedQueryAttention
    from dataclasses import replace
    H, nh, nkv, hd, win = 128, 4, 2, 32, 20
    g = torch.Generator().manual_seed(7)

    class NoRotation:
        def rotary(self, device):
            return None
    mats = {n: (torch.randn(*s, generator=g) / H ** 0.5).to(torch.bfloat16) for n, s in
            (("q_proj.weight", (nh * hd, H)), ("k_proj.weight", (nkv * hd, H)), ("v_proj.weight", (nkv * hd, H)), ("out_proj.weight", (H, nh * hd)))}
    dev = {n: m.to(DEV, dtype) for n, m in mats.items()}
    own = GroupedQueryAttention(H, nh, nkv, hd, NoRotation(), window=win)
    own.load(dev)
    other = GroupedQueryAttention(H, nh, nkv, hd, NoRotation(), window=win, shared_kv=True)
    other.load({k: dev[k] for k in ("q_proj.weight", "out_proj.weight")})
    need = replace(own.cache_need(), bits=4)
    plan = plan_cache([need, replace(other.cache_need(), bits=4)], [None, 0])
    ws = Workspace(DEV)
    cache = SequenceCache(plan, n_slots=1, n_pages=4, page_size=16, dtype=dtype, device=DEV)
    s = cache.assign()
    T = 75
    u = torch.randn(T, H, generator=g).to(torch.bfloat16)
    got = [torch.zeros(0, H), torch.zeros(0, H)]
    done, kept = 0, []
    for take in (1, 18, 1, 1, 14, 30, 10):
        cache.reserve(s, take)
        ctx = StepContext(slots=[s], starts=[done], token_lists=[[0] * take], out_rows=[], page_rows={0: cache.page_rows(0, [s])}, dtype=dtype, ws=ws)
        for i, part in enumerate((own, other)):
            resid = torch.zeros(take, H, device=DEV)
            part.forward(u[done:done + take].to(DEV, dtype), resid, ctx, cache.view(i, ctx.page_tables))
            got[i] = torch.cat([got[i], resid.cpu()])
        cache._len[s] += take                                    # (the rows as they are before pages go back)
        kept.append(cache.dump_slot(s)[0].cpu()[0, :, done:done + take])
        cache._len[s] -= take
        cache.advance(s, take)
        done += take
    kv = torch.cat(kept, dim=1).double()
    w = {n: m.double() for n, m in mats.items()}
    x = u.double()
    q = (x @ w["q_proj.weight"].T).view(T, nh, hd)
    tol = 1e-4 if dtype == torch.float32 else 3e-2
    want = torch.stack([Q.attend(q[t], kv[0], kv[1], t, hd ** -0.5, win) for t in range(T)]).reshape(T, -1) @ w["out_proj.weight"].T
    for i in range(2):
        assert (got[i].double() - want).norm() <= tol * want.norm(), i
    cache.check()


def test_programs(tmp_path):
    """``generate`` and ``replay`` with --cache-dtype int4 give what the library gives; a model that cannot be held so is refused in one line."""
    from mivi_v4_b200 import Engine, SamplingParams, load_model, write_random_model
    from votavik_configs import CONFIGS as VOTAVIK
    cfg = config_of("FL")
    d = write_model(tmp_path, cfg, 5, init="loud")
    p = prompts(cfg["vocab_size"], [40], seed=4)[0]
    eng = Engine(load_model(d, "float32", DEV), max_tokens=256, cache_dtype="int4")
    want = eng.generate([p], 12, SamplingParams.greedy(), stop_token_ids=[])[0]
    cmd = [sys.executable, "-m", "mivi_v4_b200"]
    r = subprocess.run(cmd + ["generate", "-m", d, "--prompt-ids", ",".join(map(str, p)), "-n", "12", "-t", "0", "-r", "1", "--dtype", "float32", "--cache-dtype",
                              "int4", "--stop-ids", "", "--json"], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr
    assert json.loads(r.stdout)["outputs"][0] == want
    out = tmp_path / "out"
    r = subprocess.run(cmd + ["replay", "--model", d, "--dtype", "float32", "--out", str(out), "--max-tokens", "200", "--cache-dtype", "int4"], cwd=ROOT,
                       input=json.dumps({"step": 0, "entries": [{"id": "a", "tokens": p, "want": [39]}], "end": ["a"]}) + "\n", capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr
    s = eng.open()
    row = eng.step([(s, p)], "last").cpu().numpy()
    assert (out / "0.f32").read_bytes() == row.astype("<f4").tobytes()
    v = write_random_model(str(tmp_path / "v"), VOTAVIK["P"][0], 1, "float32")
    r = subprocess.run(cmd + ["generate", "-m", v, "--prompt-ids", "1,2", "-n", "2", "--dtype", "float32", "--cache-dtype", "int4"], cwd=ROOT, capture_output=True,
                       text=True, timeout=300)
    assert r.returncode == 1 and "CacheError" in r.stderr and "Traceback" not in r.stderr
