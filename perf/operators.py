"""What the 4-bit cache is measured on: keys and values quantised as they are written into the pages of the cache, read back,
and attention over them, for single tokens, short runs of tokens and whole prompts.

A row is one token's key or value of one kv head, x of ``head_dim`` elements.  It is held as 4-bit codes and two bfloat16
numbers: zero = bf16(min x), step = bf16(max(0, max x - zero) / 15), code = clamp(rint((x - zero) / step), 0, 15), and stands for
zero + step * code.  The pool is uint8 [pages, kv heads, page_size * (head_dim + 8)]: of one kv head in one page the keys' codes
[row][head_dim / 2] (element d in byte d / 2, the even one in the low four bits), the values' codes in the same way, then (key
step, key zero, value step, value zero) as bfloat16 [row][4].

Sizes are those of the library's models and benchmark (heads of 64, 32, 24 or 16 heads on 8 kv heads) and of its tests' small
models; contexts go from one token to the benchmark's 32,768.  Lengths of a batch are in equal ratios from the shortest to the
longest.
"""
import math

import torch

own = False
DEVICE = "cuda:0"


def _case(name, kind, heads, kv_heads, head_dim, batch, cached, new, window=0, dtype="bfloat16", page=64, half=False):
    return {"name": name, "kind": kind, "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim, "batch": batch,
            "cached_lo": cached[0], "cached_hi": cached[1], "new_lo": new[0], "new_hi": new[1], "window": window, "dtype": dtype,
            "page": page, "half_split": half}


def listed():
    return [
        # one user's reply early on: the smallest call, all latency
        _case("attend_reply_1", "attend", 32, 8, 64, 1, (300, 300), (1, 1)),
        # the benchmark's batch of eight replies, unequal contexts
        _case("attend_replies_8", "attend", 32, 8, 64, 8, (511, 4095), (1, 1)),
        # a busy server: 64 replies side by side (the 700M-parameter heads)
        _case("attend_replies_64", "attend", 24, 8, 64, 64, (130, 2047), (1, 1)),
        # eight replies over the benchmark's longest contexts: the cache's bytes are everything
        _case("attend_long_8", "attend", 32, 8, 64, 8, (32767, 32767), (1, 1)),
        # a few tokens each (the tail of a chunked prompt, drafted tokens to verify), the 350M-parameter heads
        _case("attend_short_runs", "attend", 16, 8, 64, 16, (200, 3000), (1, 6)),
        # the 32-bit path
        _case("attend_float32", "attend", 16, 8, 64, 4, (100, 900), (1, 1), dtype="float32"),
        # wide heads behind a window, small pages
        _case("attend_window_wide", "attend", 16, 4, 128, 8, (700, 5000), (1, 1), window=1000, page=16),
        # a whole prompt's attention over its own rows
        _case("attend_prompt", "attend", 32, 8, 64, 1, (0, 0), (2048, 2048)),
        # later pieces of two long prompts
        _case("attend_pieces", "attend", 32, 8, 64, 2, (6000, 12000), (400, 700)),
        # what a decode step of eight replies writes, read back
        _case("store_replies_8", "store", 32, 8, 64, 8, (48, 4000), (1, 1)),
        # what a 2,048-token prompt writes, read back
        _case("store_prompt", "store", 32, 8, 64, 1, (0, 0), (2048, 2048)),
        # unequal prompts in one step (the 700M-parameter heads), the other pairing of the rotation
        _case("store_prompts_12", "store", 24, 8, 64, 12, (0, 37), (64, 1024), half=True),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    heads, kv = rng.choice([(32, 8), (24, 8), (16, 8), (8, 2), (3, 1), (5, 5), (7, 7), (16, 1), (10, 5), (12, 4)])
    hd = rng.choice([64, 64, 64, 128, 32, 96, 16, 48, 80, 40, 256])
    page = rng.choice([64, 64, 64, 16, 32, 128])
    dtype = rng.choice(["bfloat16"] * 5 + ["float32"])
    if rng.random() < 0.3:                                       # rows written and read back, in bfloat16
        batch = _log_int(rng, 1, 32)
        top = _log_int(rng, 1, max(1, 4096 // batch))
        case = _case("", "store", heads, kv, hd, batch, (0, _log_int(rng, 1, 8000)), (max(1, top // 4), top), 0, "bfloat16", page,
                     rng.random() < 0.3)
    else:
        window = rng.choice([0, 0, 0, _log_int(rng, 1, 3000)])
        shape = rng.random()
        if shape < 0.5:                                          # a token each
            batch, new = _log_int(rng, 1, 96), (1, 1)
            hi = _log_int(rng, 1, min(16000, 120000000 // (batch * kv * (hd + 8))))
        elif shape < 0.75:                                       # a few tokens each
            batch = _log_int(rng, 1, 24)
            new = (1, rng.randint(2, 24))
            hi = _log_int(rng, 1, min(8000, 60000000 // (batch * kv * (hd + 8))))
        else:                                                    # prompts and pieces of prompts
            batch = _log_int(rng, 1, 4)
            top = _log_int(rng, 130, max(130, 1500 * 2048 // (batch * max(2048, heads * hd))))
            new = (max(1, top // 3), top)
            hi = _log_int(rng, 1, 8000 // batch)
        if dtype == "float32":
            hi = min(hi, 2000)
        case = _case("", "attend", heads, kv, hd, batch, (max(0, hi // rng.randint(1, 8) - 1), hi), new, window, dtype, page)
    del case["name"]
    return case


def _spread(lo, hi, n):
    """n whole numbers in equal ratios from lo to hi (in equal steps from 0)."""
    if n == 1:
        return [hi]
    if lo <= 0:
        return [int(round(lo + (hi - lo) * i / (n - 1))) for i in range(n)]
    return [int(round(lo * (hi / lo) ** (i / (n - 1)))) for i in range(n)]


def _lengths(case):
    starts = _spread(case["cached_lo"], case["cached_hi"], case["batch"])
    lens = _spread(case["new_lo"], case["new_hi"], case["batch"])[::-1]
    return starts, lens


def _pack4(codes):
    codes = codes.to(torch.uint8)
    return codes[..., 0::2] | (codes[..., 1::2] << 4)


def _held(x):
    """Codes, step and zero of rows x [..., head_dim] (in x's precision; step and zero are values of bfloat16)."""
    zero = x.amin(-1, keepdim=True).to(torch.bfloat16).to(x.dtype)
    step = ((x.amax(-1, keepdim=True) - zero).clamp_min(0) / 15).to(torch.bfloat16).to(x.dtype)
    code = torch.where(step > 0, torch.round((x - zero) / torch.where(step > 0, step, torch.ones_like(step))), torch.zeros_like(x))
    return code.clamp(0, 15), step, zero


def _values(x):
    """What the rows x stand for once they are held in 4 bits."""
    code, step, zero = _held(x)
    return zero + step * code


def prepare(case, seed):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(seed)
    nh, nkv, hd, page, B = case["heads"], case["kv_heads"], case["head_dim"], case["page"], case["batch"]
    starts, lens = _lengths(case)
    N = sum(lens)
    blocks = [-(-(s + n) // page) for s, n in zip(starts, lens)]
    W = max(blocks)
    total = sum(blocks) + 3
    perm = torch.randperm(total, generator=g, device=DEVICE)
    table = torch.zeros((B, W), dtype=torch.int32, device=DEVICE)
    at = 0
    for b, n in enumerate(blocks):
        table[b, :n] = perm[at:at + n].int()
        at += n

    def ints(v):
        return torch.tensor(v, dtype=torch.int32, device=DEVICE)

    state = {"case": dict(case), "starts": starts, "lens": lens, "table": table, "scale": 1.0 / math.sqrt(hd),
             "positions": ints([s + i for s, n in zip(starts, lens) for i in range(n)]),
             "seq_of": ints([b for b, n in enumerate(lens) for _ in range(n)]),
             "cu": ints([sum(lens[:b]) for b in range(B + 1)]), "starts_dev": ints(starts), "keep": {}}
    dt = getattr(torch, case["dtype"])
    if case["kind"] == "store":
        state["qkv"] = torch.randn((N, (nh + 2 * nkv) * hd), generator=g, device=DEVICE)
        state["wq"] = 1 + 0.2 * torch.randn(hd, generator=g, device=DEVICE)
        state["wk"] = 1 + 0.2 * torch.randn(hd, generator=g, device=DEVICE)
        state["eps"] = 1e-5
        state["inv_freq"] = (1000000.0 ** (-torch.arange(0, hd, 2, dtype=torch.float64, device=DEVICE) / hd)).float()
        # what earlier sequences left in the pages
        state["pool"] = torch.randint(0, 256, (total, nkv, page * (hd + 8)), generator=g, device=DEVICE, dtype=torch.uint8)
        state["q"] = torch.empty((N, nh * hd), dtype=dt, device=DEVICE)
        state["k"] = torch.empty((N, nkv, hd), dtype=dt, device=DEVICE)
        state["v"] = torch.empty((N, nkv, hd), dtype=dt, device=DEVICE)
        return state
    # a full pool, the pages of other sequences and the rows behind the last token too: keys of a norm near sqrt(head_dim) with a few
    # channels that stand out, values whose size changes from row to row
    loud = 1 + 2 * (torch.rand(hd, generator=g, device=DEVICE) < 0.06).float()
    parts = []
    for first in range(0, total, 256):
        n = min(256, total - first)
        k = torch.randn((n, nkv, page, hd), generator=g, device=DEVICE) * loud
        v = torch.randn((n, nkv, page, hd), generator=g, device=DEVICE) * torch.exp(0.5 * torch.randn((n, nkv, page, 1), generator=g, device=DEVICE))
        kc, ks, kz = _held(k)
        vc, vs, vz = _held(v)
        params = torch.cat([ks, kz, vs, vz], dim=-1).to(torch.bfloat16).contiguous().view(torch.uint8)
        parts.append(torch.cat([_pack4(kc).flatten(2), _pack4(vc).flatten(2), params.flatten(2)], dim=-1))
    state["pool"] = torch.cat(parts)
    state["q"] = (1.5 * torch.randn((N, nh * hd), generator=g, device=DEVICE)).to(dt)
    state["out"] = torch.empty((N, nh * hd), dtype=dt, device=DEVICE)
    return state


def _unpack(state, dtype):
    """Keys and values of the pages of every sequence: [batch, kv heads, width * page, head_dim] each."""
    case, table = state["case"], state["table"]
    hd, page = case["head_dim"], case["page"]
    got = state["pool"][table.long()]                                        # [B, W, kv heads, bytes]
    codes, params = got[..., :page * hd], got[..., page * hd:].contiguous().view(torch.bfloat16)
    codes = codes.unflatten(-1, (2, page, hd // 2))
    codes = torch.stack([codes & 15, codes >> 4], dim=-1).flatten(-2).to(dtype)  # [B, W, kv heads, 2, page, hd]
    params = params.unflatten(-1, (page, 2, 2)).to(dtype)                    # [B, W, kv heads, page, (K, V), (step, zero)]
    k = codes[..., 0, :, :] * params[..., 0, 0:1] + params[..., 0, 1:2]
    v = codes[..., 1, :, :] * params[..., 1, 0:1] + params[..., 1, 1:2]
    return [x.transpose(1, 2).flatten(2, 3) for x in (k, v)]


def _attend_plain(state):
    case = state["case"]
    nh, nkv, hd, B, window = case["heads"], case["kv_heads"], case["head_dim"], case["batch"], case["window"]
    k, v = _unpack(state, torch.float32)
    seq, pos = state["seq_of"].long(), state["positions"].long()
    local = pos - state["starts_dev"].long()[seq]
    most = max(state["lens"])
    q = torch.zeros((B, most, nkv, nh // nkv, hd), dtype=torch.float32, device=DEVICE)
    q[seq, local] = state["q"].float().view(-1, nkv, nh // nkv, hd)
    at = torch.zeros((B, most), dtype=torch.long, device=DEVICE)
    at[seq, local] = pos
    rows = q.permute(0, 2, 1, 3, 4).reshape(B, nkv, most * (nh // nkv), hd)
    s = (rows @ k.transpose(-1, -2)).mul_(state["scale"]).view(B, nkv, most, nh // nkv, -1)
    t = torch.arange(k.shape[2], device=DEVICE)
    seen = t <= at[:, :, None]
    if window > 0:
        seen = seen & (t > at[:, :, None] - window)
    s.masked_fill_(~seen[:, None, :, None, :], float("-inf"))
    s = s.sub_(s.amax(-1, keepdim=True)).exp_()
    o = (s.view(B, nkv, most * (nh // nkv), -1) @ v).view(B, nkv, most, nh // nkv, hd) / s.sum(-1, keepdim=True)
    return {"out": o.permute(0, 2, 1, 3, 4)[seq, local].reshape(-1, nh * hd).to(state["q"].dtype)}


def _rotated(x, state, half):
    """x [N, heads, head_dim] in 64 bits, rotated by the angles of its tokens' positions."""
    a = state["positions"].double()[:, None, None] * state["inv_freq"].double()
    c, s = torch.cos(a), torch.sin(a)
    if half:
        x0, x1 = x.chunk(2, dim=-1)
        return torch.cat([x0 * c - x1 * s, x0 * s + x1 * c], dim=-1)
    x0, x1 = x[..., 0::2], x[..., 1::2]
    return torch.stack([x0 * c - x1 * s, x0 * s + x1 * c], dim=-1).flatten(-2)


def _store_plain(state):
    case = state["case"]
    nh, nkv, hd = case["heads"], case["kv_heads"], case["head_dim"]
    q, k, v = state["qkv"].view(-1, nh + 2 * nkv, hd).split([nh, nkv, nkv], dim=1)

    def normed(x, w):                                            # in 64 bits: a code next to a border goes by the last places
        x = x.double()
        return _rotated(x * torch.rsqrt(x.pow(2).mean(-1, keepdim=True) + state["eps"]) * w.double(), state, case["half_split"])

    dt = state["q"].dtype
    return {"q": normed(q, state["wq"]).flatten(1).to(dt), "k": _values(normed(k, state["wk"])).to(dt), "v": _values(v).to(dt)}


def run(state):
    case = state["case"]
    if not own:
        return _attend_plain(state) if case["kind"] == "attend" else _store_plain(state)
    from mivi_v4_b200.engine import Workspace
    from mivi_v4_b200.ops import kernels as K
    nh, nkv, hd = case["heads"], case["kv_heads"], case["head_dim"]
    if case["kind"] == "store":
        K.kv4_prepare(state["qkv"], state["wq"], state["wk"], state["eps"], state["inv_freq"], case["half_split"], state["positions"],
                      state["seq_of"], state["table"], state["pool"], state["q"], nh, nkv, hd)
        K.kv4_read(state["pool"], state["table"], state["positions"], state["seq_of"], state["k"], state["v"], nkv, hd)
        return {"q": state["q"], "k": state["k"], "v": state["v"]}
    if "ws" not in state["keep"]:
        state["keep"]["ws"] = Workspace(DEVICE)                  # the scratch that an engine keeps
    K.attention_kv4(state["q"], state["pool"], state["table"], state["positions"], state["seq_of"], state["cu"], state["starts_dev"],
                    state["out"], nh, nkv, hd, state["scale"], case["window"], state["keep"]["ws"], state["starts"], state["lens"])
    return {"out": state["out"]}


def work(case):
    nh, nkv, hd, window = case["heads"], case["kv_heads"], case["head_dim"], case["window"]
    starts, lens = _lengths(case)
    N, size = sum(lens), 2 if case["dtype"] == "bfloat16" else 4
    if case["kind"] == "store":
        held = N * nkv * (hd + 8)                                # written, then read
        return {"bytes": N * (nh + 2 * nkv) * hd * 4 + N * nh * hd * size + 2 * held + 2 * N * nkv * hd * size,
                "flops": N * ((nh + nkv) * hd * 10 + 2 * nkv * hd * 6)}
    rows = pairs = 0
    for s, n in zip(starts, lens):
        first = max(0, s - window + 1) if window > 0 else 0
        rows += s + n - first
        pairs += sum(min(s + i + 1, window) for i in range(n)) if window > 0 else n * s + n * (n + 1) // 2
    return {"bytes": rows * nkv * (hd + 8) + 2 * N * nh * hd * size, "flops": 4 * nh * hd * pairs}


def exact(case, seed):
    state = prepare(case, seed)
    nh, nkv, hd, page, window = case["heads"], case["kv_heads"], case["head_dim"], case["page"], case["window"]
    G = nh // nkv
    if case["kind"] == "store":
        x = state["qkv"].double().view(-1, nh + 2 * nkv, hd)
        angle = state["positions"].double()[:, None] * state["inv_freq"].double()[None, :]
        turn = torch.polar(torch.ones_like(angle), angle)[:, None, :]
        got = {}
        for name, lo, n, w in (("q", 0, nh, state["wq"]), ("k", nh, nkv, state["wk"]), ("v", nh + nkv, nkv, None)):
            y = x[:, lo:lo + n]
            if w is not None:
                y = y / torch.sqrt((y * y).sum(-1, keepdim=True) / hd + state["eps"]) * w.double()
                if case["half_split"]:
                    r = torch.complex(y[..., :hd // 2], y[..., hd // 2:]) * turn
                    y = torch.cat([r.real, r.imag], dim=-1)
                else:
                    y = torch.view_as_real(torch.view_as_complex(y.reshape(*y.shape[:-1], hd // 2, 2).contiguous()) * turn).flatten(-2)
            if name != "q":
                lowest = y.min(-1, keepdim=True).values.float().bfloat16().double()
                unit = ((y.max(-1, keepdim=True).values - lowest).clamp_min(0) / 15).float().bfloat16().double()
                y = torch.where(unit > 0, lowest + unit * ((y - lowest) / unit).round().clamp(0, 15), lowest.expand_as(y))
            got[name] = y.flatten(1) if name == "q" else y
        return got
    out = torch.empty((sum(state["lens"]), nh, hd), dtype=torch.float64, device=DEVICE)
    shifts = torch.tensor([0, 4], device=DEVICE, dtype=torch.uint8)
    row = 0
    for b, (s, n) in enumerate(zip(state["starts"], state["lens"])):
        T = s + n
        pages = state["pool"][state["table"][b, :-(-T // page)].long()]
        rest = pages[:, :, page * hd:].contiguous().view(torch.bfloat16).double().view(-1, nkv, page, 4)
        kv = []
        for j in (0, 1):
            c = pages[:, :, j * page * hd // 2:(j + 1) * page * hd // 2].unflatten(2, (page, hd // 2))
            c = ((c[..., None] >> shifts) & 15).flatten(-2).double()
            kv.append((c * rest[..., 2 * j:2 * j + 1] + rest[..., 2 * j + 1:2 * j + 2]).transpose(0, 1).flatten(1, 2)[:, :T])
        q = state["q"][row:row + n].double().view(n, nkv, G, hd)
        at = torch.arange(s, T, device=DEVICE)[:, None]
        t = torch.arange(T, device=DEVICE)[None, :]
        hidden = (t > at) | ((t <= at - window) if window > 0 else torch.zeros_like(t > at))
        for h in range(nkv):
            w = torch.einsum("ngd,td->gnt", q[:, h], kv[0][h]) * state["scale"]
            w = torch.softmax(w.masked_fill(hidden, -math.inf), dim=-1)
            out[row:row + n, h * G:(h + 1) * G] = torch.einsum("gnt,td->ngd", w, kv[1][h])
        row += n
    return {"out": out.flatten(1)}
